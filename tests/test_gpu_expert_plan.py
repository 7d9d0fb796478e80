"""One ExpertPlan for several products: indices overwritten after plan_experts, products on two streams, and CUDA graphs that hold
the plan or only use it."""
import pytest
import torch

from mace_onegpu import experts as X

pytestmark = pytest.mark.gpu

T, K, E, D, O = 500, 2, 6, 64, 40


def _case(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, D, device="cuda", generator=g)
    w = torch.randn(E, O, D, device="cuda", generator=g) / 8
    ex = torch.randint(-1, E, (T, K), device="cuda", generator=g, dtype=torch.int32)
    return x, w, ex


def _want(x, w, ex):
    z = torch.einsum("td,tkod->tko", x.double(), w.double()[ex.long().clamp(min=0)])
    return z * (ex >= 0)[..., None]


def _close(got, want):
    assert (got.double() - want).abs().max() <= 2e-5


@pytest.fixture(params=["few", "sorted"])
def form(request, monkeypatch):
    if request.param == "sorted":
        monkeypatch.setattr(X, "FEW_SLOTS", 0)
    return request.param


@pytest.mark.parametrize("early", [False, True])
def test_indices_overwritten_after_the_plan(early, form):
    """Copied (64-bit) indices: the plan stays what it was.  The caller's own: it is refused, whichever form the size takes."""
    x, w, ex = _case(1)
    want = _want(x, w, ex)
    wide = ex.long()
    mine, theirs = X.plan_experts(wide, E), X.plan_experts(ex, E)
    if early:
        _close(X.expert_linear(x, w, mine), want)
        _close(X.expert_linear(x, w, theirs), want)
    wide.fill_(0)
    ex.fill_(0)
    _close(X.expert_linear(x, w, mine), want)
    mine.check()
    with pytest.raises(RuntimeError, match="changed in place"):
        X.expert_linear(x, w, theirs)
    _close(X.expert_linear(x, w, X.plan_experts(ex, E)), _want(x, w, ex))


def test_two_streams_share_a_plan(form):
    """The sort sits behind a long kernel on the first stream; the second one's product comes at once."""
    x, w, ex = _case(2)
    want = _want(x, w, ex)
    plan = X.plan_experts(ex, E)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (a, b):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(a):
        torch.cuda._sleep(50_000_000)              # about 25 ms
        ya = X.expert_linear(x, w, plan)
    with torch.cuda.stream(b):
        yb = X.expert_linear(x, w, plan)
    a.synchronize()
    b.synchronize()
    _close(ya, want)
    _close(yb, want)


def test_a_captured_plan_follows_its_indices_and_stays_inside(form):
    """route's part is played by additions to a buffer: the graph sorts what it holds at each replay; eager products with the
    same plan, before and after, take what the plan's indices hold then."""
    x, w, ex = _case(3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        X.expert_linear(x, w, X.plan_experts(ex, E))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan = X.plan_experts(ex + 0, E)
        y1 = X.expert_linear(x, w, plan)
        y2 = X.expert_linear(y1[:, 0].contiguous() @ torch.eye(O, D, device="cuda"), w, plan)
    X.expert_linear(x, w, plan)                    # nothing of the graph has run: whatever its copy holds, in bounds
    torch.cuda.synchronize()
    for seed in (4, 5):
        ex.copy_(_case(seed)[2])
        graph.replay()
        torch.cuda.synchronize()
        want = _want(x, w, ex)
        _close(y1, want)
        first = torch.zeros(T, D, device="cuda")
        first[:, :O] = y1[:, 0]
        _close(y2, _want(first, w, ex))
        _close(X.expert_linear(x, w, plan), want)
        plan.check()


def test_an_eager_plan_used_by_a_graph(form):
    """The graph sorts the plan's indices itself, whether the plan was sorted before or not."""
    x, w, ex = _case(6)
    want = _want(x, w, ex)
    for warm in (False, True):
        plan = X.plan_experts(ex, E)
        if warm:
            X.expert_linear(x, w, plan)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = X.expert_linear(x, w, plan)
        _close(X.expert_linear(x, w, plan), want)  # before the first replay
        x2 = torch.randn(T, D, device="cuda")
        old = x.clone()
        x.copy_(x2)
        graph.replay()
        torch.cuda.synchronize()
        _close(y, _want(x2, w, ex))
        x.copy_(old)


def test_a_captured_training_step():
    """Forward and backward of one plan in one capture: two products, one sort, gradients that follow new inputs."""
    x, w, ex = _case(7)
    w = w.requires_grad_()
    dy = torch.randn(T, K, O, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        plan = X.plan_experts(ex, E)
        return torch.autograd.grad(X.expert_linear(x, w, plan), w, dy)[0]

    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        dw = step()
    for seed in (8, 9):
        n, _, e = _case(seed)
        x.copy_(n)
        ex.copy_(e)
        graph.replay()
        torch.cuda.synchronize()
        want = torch.zeros(E, O, D, dtype=torch.float64, device="cuda")
        for i in range(E):
            for j in range(K):
                t = torch.nonzero(e[:, j] == i)[:, 0]
                want[i] += dy[t, j].double().T @ n[t].double()
        assert (dw.double() - want).abs().max() <= 2e-5 * want.abs().max()


def test_the_capture_number():
    from mace_onegpu import _native as N

    s = torch.cuda.Stream()
    assert N.lib().mace_b200_capture_id(s.cuda_stream) == 0
    seen = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            torch.zeros(1, device="cuda")
            seen.append(N.lib().mace_b200_capture_id(s.cuda_stream))
            assert N.lib().mace_b200_capture_id(torch.cuda.default_stream().cuda_stream) == 0
    assert seen[0] != 0 and seen[1] != 0 and seen[0] != seen[1]
    assert N.lib().mace_b200_capture_id(s.cuda_stream) == 0


def test_a_plan_and_a_block_can_be_copied_and_saved(form, tmp_path):
    """After calls, too (a block keeps its last plan): the copy sorts for itself."""
    import copy
    import pickle

    x, w, ex = _case(10)
    want = _want(x, w, ex)
    plan = X.plan_experts(ex, E)
    X.expert_linear(x, w, plan)
    for other in (copy.deepcopy(plan), copy.copy(plan), pickle.loads(pickle.dumps(plan))):
        _close(X.expert_linear(x, w, other), want)
        other.check()
    ex.fill_(0)
    with pytest.raises(RuntimeError, match="changed in place"):
        X.expert_linear(x, w, plan)
    block = X.ExpertBlock(D, 32, 8, E, K)
    y = block(x)
    torch.save(block, tmp_path / "block.pt")
    for other in (copy.deepcopy(block), torch.load(tmp_path / "block.pt", weights_only=False)):
        assert torch.equal(other(x), y)
        assert torch.equal(other.balance(), block.balance(0.0))
