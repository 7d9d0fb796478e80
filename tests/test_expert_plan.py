"""When ExpertPlan sorts, on the CPU with the sort and the place (stream, capture) replaced: indices that change, one sort per place,
no table of one CUDA graph capture used outside of it, and an order between streams."""
import pytest
import torch

from mace_onegpu import experts as X


class Place:
    """Stands for the current stream and the number of the capture it is in (0: none)."""

    def __init__(self, monkeypatch):
        self.stream, self.capture, self.sorts, self.waits = 1, 0, [], []
        monkeypatch.setattr(X, "_op", lambda name: self.sort)
        monkeypatch.setattr(X, "_place", lambda index: (self.stream, self.capture), raising=False)
        monkeypatch.setattr(X, "_ready", lambda device: ("event", self.stream), raising=False)
        monkeypatch.setattr(X, "_after", lambda device, event, *tensors: self.waits.append((event, self.stream)), raising=False)

    def sort(self, experts, n):
        self.sorts.append((self.stream, self.capture, experts.clone()))
        return torch.full((8,), len(self.sorts), dtype=torch.int32)


@pytest.fixture
def place(monkeypatch):
    return Place(monkeypatch)


COPIED = [lambda e: e.long(), lambda e: e.t().contiguous().t(), lambda e: e[:, 1], lambda e: e.long()[:, 0]]


@pytest.mark.parametrize("make", COPIED)
def test_copied_indices_stay_as_they_were(place, make):
    ex = make(torch.tensor([[0, 1], [2, 0], [1, 1]], dtype=torch.int32))
    plan = X.plan_experts(ex, 3)
    was = plan.experts.clone()
    ex.fill_(2)
    assert torch.equal(plan.experts, was)
    plan.words
    ex.fill_(0)
    plan.words
    assert len(place.sorts) == 1 and torch.equal(place.sorts[0][2], was)


@pytest.mark.parametrize("sorted_before", [False, True])
@pytest.mark.parametrize("view", [lambda e: e, lambda e: e.view(-1), lambda e: e[1:3]])
def test_a_plan_whose_indices_were_changed_is_refused(place, view, sorted_before):
    ex = torch.tensor([[0, 1], [2, 0], [1, 1]], dtype=torch.int32)
    plan = X.plan_experts(view(ex), 3)
    assert plan.experts.data_ptr() == view(ex).data_ptr()
    if sorted_before:
        plan.words
    ex[2, 0] = 0                                   # through the base: a view shares its version
    with pytest.raises(RuntimeError, match="changed in place"):
        plan.words
    w = torch.zeros(3, 4, 5)
    with pytest.raises(RuntimeError, match="changed in place"):          # the form without a sort, too
        X.expert_linear(torch.zeros(len(plan.experts), 5), w, plan)
    assert len(place.sorts) == sorted_before


def test_inference_tensors_are_copied(place):
    with torch.inference_mode():
        ex = torch.zeros(3, 1, dtype=torch.int32)
        plan = X.plan_experts(ex, 2)
        ex.fill_(1)
        assert not plan.experts.any()
        plan.words
    assert not place.sorts[0][2].any()


def test_another_stream_waits_for_the_sort(place):
    plan = X.plan_experts(torch.zeros(4, 1, dtype=torch.int32), 2)
    a = plan.words
    assert plan.words is a and not place.waits
    place.stream = 2
    assert plan.words is a
    assert [w for w in place.waits if w[0] is not None] == [(("event", 1), 2)]
    assert len(place.sorts) == 1


def test_no_table_crosses_a_capture(place):
    plan = X.plan_experts(torch.zeros(4, 1, dtype=torch.int32), 2)
    place.capture = 7
    inside = plan.words
    assert plan.words is inside                    # one sort serves the whole capture
    place.capture = 0
    eager = plan.words                             # nothing of the capture has run yet
    assert eager is not inside
    assert plan.words is eager
    place.capture = 8                              # a later capture sorts for itself: its replays need memory of their own
    assert plan.words is not eager
    assert [c for _, c, _ in place.sorts] == [7, 0, 8]


def test_a_plan_made_in_a_capture_is_sorted_at_every_eager_use(place):
    place.capture = 3
    plan = X.plan_experts(torch.zeros(4, 1, dtype=torch.int32), 2)
    inside = plan.words
    assert plan.words is inside
    place.capture = 0                              # each replay writes the plan's indices anew
    assert plan.words is not plan.words
    assert [c for _, c, _ in place.sorts] == [3, 0, 0]
