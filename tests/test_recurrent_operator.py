"""The recurrent user encoder (model/operators/recurrent_operator.py) and what is scored over the whole catalogue (functional.next_item_loss,
evaluate.next_items, tester --next_items): configuration and discovery on the CPU; on the GPU against a plain 64-bit restatement, click by
click against the whole history, and through the trainer and tester."""
import math
import os

import numpy as np
import pytest
import torch

from legommenders_amd.trainer import get_configurations

COMMON = dict(data="config/data/synthetic.yaml", model="config/model/naml-recurrent.yaml", embed="config/embed/glove.yaml", batch_size=32,
              hidden_size=64, lr=0.001, cuda=0, world="small")


def test_configuration_and_discovery():
    from legommenders_amd.loader.class_hub import ClassHub
    from legommenders_amd.model.operators.recurrent_operator import RecurrentOperator, RecurrentOperatorConfig
    c = get_configurations(dict(COMMON, num_recurrent_layers=3))
    assert c.model.meta.item == "CNN" and c.model.meta.user == "Recurrent" and c.model.meta.predictor == "Dot"
    assert c.model.config()["user_config"]["num_recurrent_layers"] == 3
    assert ClassHub.operators()["Recurrent"] is RecurrentOperator
    with pytest.raises(ValueError, match="at least 1"):
        RecurrentOperatorConfig(hidden_size=8, input_dim=8, num_recurrent_layers=0)


def test_refusals():
    from legommenders_amd import functional as F
    from legommenders_amd._lib import LegoHipError
    with pytest.raises(LegoHipError):
        F.next_item_loss(torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64))       # CPU tensors


# ----------------------------------------------------------------------------------------------- GPU
def _operator(layers=2, **over):
    from legommenders_amd.loader.env import Env
    from legommenders_amd.trainer import build_model, load_world
    cfg = get_configurations(dict(COMMON, num_recurrent_layers=layers, **over))
    dev = Env.set_device(0)
    torch.manual_seed(11)
    model, kind = build_model(cfg, load_world(cfg.data, 5), dev)
    assert kind == "plugin" and type(model.user_op).__name__ == "RecurrentOperator" and len(model.user_op.blocks) == layers
    g = torch.Generator().manual_seed(3)
    with torch.no_grad():
        for p in model.user_op.parameters():
            if p.dim() == 1:                                                                 # not only ones and zeros
                p.add_((0.1 * torch.randn(p.shape, generator=g)).to(p))
    return model, cfg


def _plain(op, x, live, c):
    """the operator in 64 bits, step by step"""
    P = {k: v.detach().double().cpu().requires_grad_() for k, v in op.named_parameters()}
    sig = torch.sigmoid
    norm = lambda t, w: t / (t.square().mean(-1, keepdim=True) + c.norm_eps).sqrt() * w      # noqa: E731
    B, S, D = x.shape
    y, n = x, norm(x, P["blocks.0.pre_norm"])
    layers = len(op.blocks)
    for q in range(layers):
        b = f"blocks.{q}."
        v, r, i, g = (n @ P[b + "in_proj.weight"].t() + P[b + "in_proj.bias"]).chunk(4, -1)
        a = torch.exp(-c.sharpness * torch.nn.functional.softplus(P[b + "decay"]) * sig(r))
        u = torch.sqrt(1 - a * a) * sig(i) * v
        h, hs = torch.zeros(B, D, dtype=torch.float64), []
        for t in range(S):
            h = torch.where(live[:, t, None], a[:, t] * h + u[:, t], h)
            hs.append(torch.where(live[:, t, None], h, torch.zeros_like(h)))
        o = torch.stack(hs, 1) @ P[b + "out_proj.weight"].t()
        y = y + P[b + "scale"] * g * sig(g) * norm(o, P[b + "post_norm"])
        n = norm(y, P[f"blocks.{q + 1}.pre_norm"] if q + 1 < layers else P["norm"])
    at = (live * torch.arange(1, S + 1)).amax(1)
    out = n[torch.arange(B), (at - 1).clamp(min=0)]
    return torch.where((at > 0)[:, None], out, torch.zeros_like(out)), P


@pytest.mark.gpu
def test_operator_and_its_gradients_in_64_bits():
    model, _ = _operator()
    op = model.user_op
    g = torch.Generator().manual_seed(1)
    B, S, D = 5, 50, op.config.input_dim
    x = torch.randn(B, S, D, generator=g)
    lens = torch.tensor([50, 1, 0, 17, 33])
    live = torch.arange(S)[None] < lens[:, None]
    live[4, 3:9] = False                                                                     # a hole
    want, P = _plain(op, x.double(), live, op.config)
    pick = torch.randn(B, D, generator=g)
    gw = torch.autograd.grad((want * pick.double()).sum(), list(P.values()))
    got = op(x.cuda(), mask=live.long().cuda())
    # products of up to 256 terms in fp32 and two blocks with norms between them: 1e-5 of the largest value is some 170 roundings of it
    assert float((got.detach().cpu().double() - want.detach()).abs().max()) <= 1e-5 * float(want.detach().abs().max())
    assert float(got[2].abs().max()) == 0.0
    grads = torch.autograd.grad((got * pick.cuda()).sum(), [dict(op.named_parameters())[k] for k in P])
    for k, a, b in zip(P, grads, gw):
        err = float((a.cpu().double() - b).norm()) / max(float(b.norm()), 1e-30)
        assert err <= 5e-5, (k, err)


@pytest.mark.gpu
def test_click_by_click_equals_the_whole_history():
    model, _ = _operator()
    op = model.user_op.eval()
    g = torch.Generator().manual_seed(2)
    B, S, D = 7, 23, op.config.input_dim
    x = torch.randn(B, S, D, generator=g).cuda()
    lens = torch.tensor([23, 0, 1, 12, 5, 23, 8], device="cuda")
    live = torch.arange(S, device="cuda")[None] < lens[:, None]
    with torch.no_grad():
        want = op(x, mask=live.long())
    states, user = op.initial_state(B), torch.zeros(B, D, device="cuda")
    kept = [s.clone() for s in states]
    for t in range(S):
        vec, new = op.step(x[:, t], states, mask=live[:, t])
        assert all(torch.equal(a, b) for a, b in zip(states, kept))                          # the old states are left as they were
        user = torch.where(live[:, t, None], vec, user)
        states, kept = new, [s.clone() for s in new]
    assert torch.allclose(user, want, rtol=2e-5, atol=2e-5)


@pytest.mark.gpu
def test_next_item_loss_and_its_gradients():
    from legommenders_amd import functional as F
    g = torch.Generator().manual_seed(4)
    B, N, D = 9, 501, 64
    u, it = torch.randn(B, D, generator=g), torch.randn(N, D, generator=g) * 0.3
    t = torch.randint(0, N, (B,), generator=g)
    t[3] = -1
    mask = torch.rand(N, generator=g) < 0.8
    mask[t.clamp(min=0)] = True
    u64, i64 = u.double().requires_grad_(), it.double().requires_grad_()
    lp = torch.log_softmax((u64 @ i64.t()).masked_fill(~mask, -math.inf), 1)
    want = -lp[torch.arange(B), t.clamp(min=0)][t >= 0].mean()
    gw = torch.autograd.grad(want, (u64, i64))
    ud, idv = u.cuda().requires_grad_(), it.cuda().requires_grad_()
    got = F.next_item_loss(ud, idv, t.cuda(), mask=mask.cuda())
    assert abs(float(got) - float(want)) <= 2e-6 * float(want)
    for a, b in zip(torch.autograd.grad(got, (ud, idv)), gw):
        assert float((a.cpu().double() - b).norm()) <= 1e-5 * float(b.norm())
    assert float(F.next_item_loss(ud, idv, torch.full((B,), -1, device="cuda"))) == 0.0


@pytest.mark.gpu
def test_next_items_over_the_catalogue():
    from legommenders_amd.evaluate import next_items
    g = torch.Generator().manual_seed(6)
    users, items, S, k = 40, 2002, 50, 5
    ur, ir = torch.randn(users, 64, generator=g), torch.randn(items, 64, generator=g)
    hist, lens = torch.randint(0, items, (users, S), generator=g).int(), torch.randint(0, S + 1, (users,), generator=g).int()
    who = torch.randint(0, users, (23,), generator=g)
    t = torch.randint(0, items, (23,), generator=g)
    t[5] = int(hist[who[5], 0])                                                              # a target that was clicked before stays in
    t[7] = -1
    r = next_items(ur.cuda(), ir.cuda(), who, t, k=k, seen=(hist.cuda(), lens.cuda()), page=8)
    s = ur.double()[who] @ ir.double().t()
    for q in range(23):
        seen = hist[who[q], :lens[who[q]]].long()
        keep = s[q, t[q]].clone() if t[q] >= 0 else None
        s[q, seen] = -math.inf
        if keep is not None:
            s[q, t[q]] = keep
    lp = torch.log_softmax(s, 1)
    want = torch.where(t >= 0, lp[torch.arange(23), t.clamp(min=0)], 0.0)
    # scores of 64 terms in fp32: off by some 64 roundings of their size (|u||i| <= 200)
    assert float((r["logp"].cpu().double() - want).abs().max()) <= 64 * 200 * 2.0 ** -24
    top, index = lp.topk(k, 1)
    assert torch.equal(r["items"].cpu().long(), index) and float((r["top"].cpu().double() - top).abs().max()) <= 64 * 200 * 2.0 ** -24
    none = next_items(ur.cuda(), ir.cuda(), who[:0], k=k)
    assert none["items"].shape == (0, k) and none["logp"].shape == (0,)


@pytest.mark.gpu
def test_trains_and_tests_through_the_command_line(tmp_path, monkeypatch):
    from legommenders_amd import tester
    from legommenders_amd.trainer import Trainer
    monkeypatch.chdir(tmp_path)
    tr = Trainer(get_configurations(dict(COMMON, epoch=1, patience=2, interval=0, epoch_batch=6, num_recurrent_layers=2)))
    assert tr.kind == "plugin"
    before = tr.legommender.user_op.blocks[1].decay.detach().clone()
    res = tr.run()
    assert set(res) == {"GAUC", "MRR", "NDCG@1", "NDCG@5", "NDCG@10"} and all(np.isfinite(v) for v in res.values())
    assert not torch.equal(before, tr.legommender.user_op.blocks[1].decay)                   # the decays are trained
    state = torch.load(os.path.join("checkpoints", "synthetic", tr.config.model.name, tr.signature + ".pt"))
    assert set(state["model"]) == set(tr.legommender.state_dict())
    te = tester.Tester(tester.get_configurations(dict(COMMON, load_sign=tr.signature, next_items=10, num_recurrent_layers=2)))
    out = te.run()
    n = te.world["n_items"]
    assert set(out) == {"LogProb", "Entropy", "HitRatio@10"}
    assert out["LogProb"] < 0 and 0 < out["Entropy"] <= math.log(n) + 1e-3 and 0 <= out["HitRatio@10"] <= 1
    r = te.evaluator.next_items([0, 1, 2], k=3, exclude_seen=True)
    hist = te.data.user_hist[:3].cpu()
    for q in range(3):
        assert not set(r["items"][q].tolist()) & set(hist[q, :int(te.data.user_hist_len[q])].tolist())
