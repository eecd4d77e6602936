"""The sequence operators under torch's transforms: forward-mode derivatives are refused, never answered with zeros, and the public functions are traced whole.

Without a GPU the registered ops get a stand-in on the CPU (plain torch forms), so that the Python above the kernels is what runs."""
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from legommenders_amd import functional as F
from legommenders_amd import kernels as K
from legommenders_amd._lib import LegoHipError

L = torch.ops.lego_hip


def _scan(x, r, i, lam, state, c):
    a = torch.exp(-c * torch.nn.functional.softplus(lam) * torch.sigmoid(r.float()))
    b = torch.sqrt(1 - a * a) * torch.sigmoid(i.float()) * x.float()
    now, hs = torch.zeros(x.shape[0], x.shape[2]) if state is None else state, []
    for t in range(x.shape[1]):
        now = a[:, t] * now + b[:, t]
        hs.append(now)
    return torch.stack(hs, 1).to(x.dtype), now


def _norm(x, w, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w


def _scan_impl(x, r, i, lam, mask, state, c, keep):
    h, last = _scan(x, r, i, lam, state, c)
    return h, last.clone(), torch.zeros(x.shape[0], -(-x.shape[1] // K.SCAN_TILE) if keep else 0, x.shape[2])


def _with_autograd(f):
    """a kernel is called below autograd; a stand-in that differentiates a plain form does so on a thread of its own"""
    def g(*args):
        with ThreadPoolExecutor(1) as pool:
            return pool.submit(f, *args).result()
    return g


@_with_autograd
def _scan_bwd_impl(gh, glast, x, r, i, lam, mask, tiles, c):
    with torch.enable_grad():
        leaves = [t.detach().requires_grad_() for t in (x, r, i, lam, torch.zeros(x.shape[0], x.shape[2]))]
        h, last = _scan(*leaves, c)
        return torch.autograd.grad((h, last), leaves, (gh, torch.zeros_like(last) if glast is None else glast))


def _norm_impl(x, o, gate, post_w, scale, next_w, eps, act, keep):
    y = x if o is None else x + scale * torch.nn.functional.silu(gate) * _norm(o, post_w, eps)
    stat = torch.ones((o is not None) + (next_w is not None), x.shape[0] if keep else 0)
    return x.new_empty(0) if o is None else y, x.new_empty(0) if next_w is None else _norm(y, next_w, eps), stat


@_with_autograd
def _norm_bwd_impl(dy, dn, x, o, gate, post_w, scale, next_w, stat, eps, act):
    with torch.enable_grad():
        leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, o, gate, post_w, scale, next_w)]
        y, n, _ = _norm_impl(*leaves, eps, act, False)
        outs = [(t, g) for t, g in ((y, dy), (n, dn)) if g is not None]
        there = [t for t in leaves if t is not None]
        grads = iter(torch.autograd.grad([t for t, _ in outs], there, [g for _, g in outs]))
    return tuple(x.new_empty(0) if t is None else next(grads) for t in leaves)


def _probs_impl(logits, targets, mask, k):
    lp = torch.log_softmax(logits.float(), 1)
    top, index = lp.topk(k, 1)
    at = torch.zeros(len(lp), 1, dtype=torch.int64) if targets is None else targets.long()[:, None]
    return lp.gather(1, at)[:, 0], -(lp.exp() * lp).sum(1), torch.zeros(len(lp), 2), top, index.int()


@_with_autograd
def _probs_bwd_impl(gl, ge, gt, logits, targets, mask, stat, entropy, index):
    with torch.enable_grad():
        x = logits.detach().requires_grad_()
        outs = [(t, g) for t, g in zip(_probs_impl(x, targets, mask, index.shape[1]), (gl, ge, None, gt)) if g is not None]
        return torch.autograd.grad([t for t, _ in outs], x, [g for _, g in outs])[0]


@pytest.fixture
def on_the_cpu(monkeypatch):
    lib = torch.library.Library("lego_hip", "IMPL")
    for name, f in dict(gated_scan=_scan_impl, gated_scan_bwd=_scan_bwd_impl, block_norm=_norm_impl, block_norm_bwd=_norm_bwd_impl, token_logprobs=_probs_impl,
                        token_logprobs_bwd=_probs_bwd_impl,
                        gated_scan_step=lambda x, r, i, lam, st, mask, c: tuple(t[:, 0] if t.dim() == 3 else t for t in _scan(x[:, None], r[:, None], i[:, None], lam, st, c))
                        ).items():
        lib.impl(name, f, "CPU")
    monkeypatch.setattr(F, "_need_gpu", lambda t, what: None)
    yield "cpu"
    lib._destroy()
    torch.compiler.reset()


def _calls(dev):
    """name -> (a public function of one tensor, that tensor), every operator in each of its operands' places that a derivative can enter by"""
    g = torch.Generator().manual_seed(1)
    x, r, i = (torch.randn(2, 5, 8, generator=g).to(dev) for _ in range(3))
    lam, st, w = torch.randn(8, generator=g).to(dev), torch.randn(2, 8, generator=g).to(dev), torch.ones(8, device=dev)
    t = torch.tensor([1, 0], device=dev)
    return {
        "scan x": (lambda v: F.gated_scan(v, r, i, lam), x), "scan lam": (lambda v: F.gated_scan(x, r, i, v)[0], lam),
        "scan state": (lambda v: F.gated_scan(x, r, i, lam, state=v)[1], st),
        "step x": (lambda v: F.gated_scan_step(v, r[:, 0], i[:, 0], lam, st)[0], x[:, 0]), "step state": (lambda v: F.gated_scan_step(x[:, 0], r[:, 0], i[:, 0], lam, v), st),
        "rms": (lambda v: F.rms_norm(v, w), x), "rms w": (lambda v: F.rms_norm(x, v), w),
        "tail o": (lambda v: F.gated_residual_norm(x, v, i, w, w, w), r), "tail gate": (lambda v: F.gated_residual_norm(x, r, v, w, w)[0], i),
        "probs": (lambda v: F.token_logprobs(v, t, k=3)[:3], st),
    }


NAMES = list(_calls("cpu"))


def _jvp(f, v):
    return torch.func.jvp(f, (v,), (torch.ones_like(v),))


def _dual(f, v):
    with torch.autograd.forward_ad.dual_level():
        f(torch.autograd.forward_ad.make_dual(v, torch.ones_like(v)))


def _dual_beside_a_leaf(f, v):
    with torch.autograd.forward_ad.dual_level():
        f(torch.autograd.forward_ad.make_dual(v.clone().requires_grad_(), torch.ones_like(v)))


@pytest.mark.parametrize("how", [_jvp, _dual])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(on_the_cpu, name, how):
    f, v = _calls(on_the_cpu)[name]
    with pytest.raises(LegoHipError, match="forward-mode"):
        how(f, v)
    with torch.autograd.forward_ad.dual_level():                                             # nothing dual among the operands: nothing to refuse
        f(v)


@pytest.mark.gpu
@pytest.mark.parametrize("how", [_jvp, _dual, _dual_beside_a_leaf])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused_on_the_gpu(name, how):
    f, v = _calls("cuda")[name]
    with pytest.raises(LegoHipError, match="forward-mode|no gradient"):
        how(f, v)


def test_forward_mode_is_refused_below_the_public_functions(on_the_cpu):
    x, lam, st, w = torch.randn(2, 5, 8), torch.randn(8), torch.randn(2, 8), torch.ones(8)
    tiles, stat, index = torch.zeros(2, 1, 8), torch.ones(1, 2), torch.zeros(2, 1, dtype=torch.int32)
    t = torch.zeros(2, dtype=torch.int64)
    for f, v in [(lambda v: L.gated_scan(v, x, x, lam, None, None, 8.0, False), x), (lambda v: L.gated_scan_step(st, st, st, lam, v, None, 8.0), st),
                 (lambda v: L.gated_scan_bwd(v, None, x, x, x, lam, None, tiles, 8.0), x), (lambda v: L.block_norm(v, None, None, None, None, w, 1e-6, 0, False), st),
                 (lambda v: L.block_norm_bwd(None, v, st, None, None, None, None, w, stat, 1e-6, 0), st), (lambda v: L.token_logprobs(v, t, None, 1), st),
                 (lambda v: L.token_logprobs_bwd(v, None, None, st, t, None, st[:, :2], st[:, 0], index), st[:, 1])]:
        for how in (_jvp, _dual):
            with pytest.raises(LegoHipError, match="forward-mode"):
                how(f, v)


def _compiled_calls(dev):
    """name -> (a function of leaves that require a gradient, the leaves)"""
    g = torch.Generator().manual_seed(2)
    x, r, i = (torch.randn(2, 70, 8, generator=g).to(dev) for _ in range(3))
    lam, st, w, s = torch.randn(8, generator=g).to(dev), torch.randn(2, 8, generator=g).to(dev), torch.ones(8, device=dev), torch.randn(8, generator=g).to(dev)
    t = torch.tensor([1, 0], device=dev)
    return {
        "scan": (lambda x, r, i, lam, st: F.gated_scan(x, r, i, lam, state=st), (x, r, i, lam, st)),
        "rms": (lambda x, w: (F.rms_norm(x, w),), (x, w)),
        "tail": (lambda x, o, g, w, s: F.gated_residual_norm(x, o, g, w, s, w), (x, r, i, w, s)),
        "tail alone": (lambda x, o, g, w, s: F.gated_residual_norm(x, o, g, w, s)[:1], (x, r, i, w, s)),
        "probs": (lambda x: F.token_logprobs(x, t, k=3)[:3], (st,)),
        "probs of a batch": (lambda x: F.token_logprobs(x, k=2)[1:3], (x,)),
    }


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("name", list(_compiled_calls("cpu")))
def test_public_functions_compile_whole(request, name, dev):
    if dev == "cpu":
        request.getfixturevalue("on_the_cpu")
    f, leaves = _compiled_calls(dev)[name]
    whole = torch.compile(f, fullgraph=True, backend="aot_eager")
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(whole(*leaves), f(*leaves)))
    live = [t.clone().requires_grad_() for t in leaves]
    want, got = f(*live), whole(*live)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    up = [torch.ones_like(t) for t in want]
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, live, up), torch.autograd.grad(want, live, up)))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_the_single_step_compiles_whole(request, dev):
    if dev == "cpu":
        request.getfixturevalue("on_the_cpu")
    x, r, i, st = (torch.randn(3, 8, generator=torch.Generator().manual_seed(q)).to(dev) for q in range(4))
    lam = torch.randn(8, generator=torch.Generator().manual_seed(9)).to(dev)
    f = lambda *a: F.gated_scan_step(*a)      # noqa: E731
    whole = torch.compile(f, fullgraph=True, backend="aot_eager")
    assert all(torch.equal(a, b) for a, b in zip(whole(x, r, i, lam, st), f(x, r, i, lam, st)))


def test_ops_without_a_gradient_say_so_in_the_backward_pass(on_the_cpu):
    st, lam = torch.randn(2, 8), torch.randn(8)
    h, new = L.gated_scan_step(st, st, st, lam.requires_grad_(), st, None, 8.0)
    with pytest.raises(LegoHipError, match="gated_scan_step has no gradient"):
        h.sum().backward()
    with torch.no_grad():
        assert not L.gated_scan_step(st, st, st, lam, st, None, 8.0)[0].requires_grad
