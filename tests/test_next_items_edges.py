"""evaluate.next_items where its arguments leave the catalogue: on the CPU, with plain forms in the place of the product and of the log probabilities."""
import math

import pytest
import torch

from legommenders_amd import functional as F
from legommenders_amd._lib import LegoHipError
from legommenders_amd.evaluate import next_items


def _probs(x, t=None, k=0, mask=None):
    lp = torch.log_softmax(x if mask is None else x.masked_fill(~mask, -math.inf), 1)
    has = torch.zeros(len(x), dtype=torch.bool) if t is None else (t >= 0) & (t < x.shape[1])
    at = torch.zeros(len(x), 1, dtype=torch.int64) if t is None else torch.where(has, t, 0)[:, None]
    p = lp.exp()
    top, index = lp.topk(k, 1)
    return torch.where(has, lp.gather(1, at)[:, 0], 0.0), -torch.where(p > 0, p * lp, 0.0).sum(1), top, index.int()


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request, monkeypatch):
    if request.param == "cpu":
        monkeypatch.setattr(F, "linear", lambda x, w: x @ w.t())
        monkeypatch.setattr(F, "token_logprobs", _probs)
    return request.param


def _world(dev):
    g = torch.Generator().manual_seed(1)
    users, items = torch.randn(6, 8, generator=g).to(dev), torch.randn(10, 8, generator=g).to(dev)
    hist = torch.tensor([[1, 2, 3], [4, 4, -1], [9, 0, 5], [7, -1, -1], [2, 2, 2], [-1, -1, -1]], dtype=torch.int32, device=dev)
    return users, items, (hist, torch.tensor([3, 2, 3, 1, 2, 0], dtype=torch.int32, device=dev))


def test_a_target_outside_the_catalogue_is_none(dev):
    users, items, seen = _world(dev)
    who = [0, 1, 2, 3]
    for s in (None, seen):
        a = next_items(users, items, who, [3, 10, -7, 1 << 40], k=2, seen=s)
        b = next_items(users, items, who, [3, -1, -1, -1], k=2, seen=s)
        assert all(torch.equal(a[n], b[n]) for n in a) and bool((a["logp"][1:] == 0).all()) and float(a["logp"][0]) < 0


def test_a_click_outside_the_catalogue_hides_nothing(dev):
    users, items, (hist, lens) = _world(dev)
    far = hist.clone()
    far[0, 2], far[2, 0] = 10, -1
    want = hist.clone()
    want[0, 2], want[2, 0] = 1, 0                                                            # (items that are hidden already)
    a, b = (next_items(users, items, [0, 2], k=3, seen=(h, lens)) for h in (far, want))
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_users_that_are_not_there_are_refused(dev):
    users, items, seen = _world(dev)
    for who in ([0, 6], [-1], torch.tensor([0, 1 << 40]), torch.tensor([-6], device=dev)):
        with pytest.raises(LegoHipError, match="users"):
            next_items(users, items, who, k=2)


def test_targets_that_are_not_one_a_user_are_refused(dev):
    users, items, _ = _world(dev)
    for t in ([0], [0, 1, 2], [[0, 1]]):
        with pytest.raises(LegoHipError, match="targets"):
            next_items(users, items, [0, 1], t, k=2)
