"""The sequence operators -- gated_scan / gated_scan_step, rms_norm / gated_residual_norm, token_logprobs -- against plain 64-bit forms on the CPU,
and their refusals.

Tolerances: an output is off by at most half a step of its type (torch.finfo(t).eps / 2, relative) from its one rounding, plus what fp32 arithmetic
adds: U = 2^-24 a rounding, against the sum of the ABSOLUTE values of the terms that make the number (cancellation costs nothing in that
measure).  The number of roundings is counted beside each test."""
import ctypes
import math

import pytest
import torch

from legommenders_amd import _lib, functional as F
from legommenders_amd import kernels as K
from legommenders_amd._lib import LegoHipError

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
L = torch.ops.lego_hip


def check(got, want, terms, roundings, floor=0.0):
    """|got - want| <= half a step of got's type + roundings * U * terms + floor (+ the type's smallest subnormal) where want is finite; equal elsewhere.
    What is larger than the type's largest number rounds to infinity (fp16: 65504)."""
    t = torch.finfo(got.dtype)
    got, want = got.detach().cpu().double(), want.double()
    want = torch.where(want.abs() > t.max, want.sign() * math.inf, want)
    assert got.shape == want.shape, (got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)) and torch.equal(torch.isnan(want), torch.isnan(got))
    rest = ~fine & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest])
    terms = torch.as_tensor(terms, dtype=torch.float64).expand_as(want)
    slack = (t.eps / 2) * want.abs() + roundings * U * terms + t.smallest_normal * t.eps + 2.0 ** -126 + floor
    bad = ((got - want).abs() > slack) & fine
    worst = ((got - want).abs() / slack)[fine].max() if fine.any() else 0.0
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, the worst {float(worst):.3g} times its bound"


# --------------------------------------------------------------------------------------------------------------- 64-bit forms
def scan_64(x, r, i, lam, mask, state, c, gh=None, glast=None):
    """loops over the steps; returns outputs, gradients, and for each the sum of the absolute values of its terms"""
    n, length, width = x.shape
    x, r, i, lam = x.double(), r.double(), i.double(), lam.double()
    live = torch.ones(n, length, dtype=torch.bool) if mask is None else mask != 0
    m = live[..., None]
    x, r, i = (torch.where(m, t, torch.zeros((), dtype=torch.float64)) for t in (x, r, i))
    sp = torch.nn.functional.softplus(lam, threshold=1000)
    sr, si = torch.sigmoid(r), torch.sigmoid(i)
    l = torch.where(m, -c * sp * sr, torch.zeros((), dtype=torch.float64))
    a, beta = torch.exp(l), torch.sqrt(-torch.expm1(2 * l))
    u = si * x
    now = torch.zeros(n, width, dtype=torch.float64) if state is None else state.double()
    size = now.abs()
    h, hs, before, befores = (torch.zeros(n, length, width, dtype=torch.float64) for _ in range(4))
    for t in range(length):
        before[:, t], befores[:, t] = now, size
        now, size = a[:, t] * now + beta[:, t] * u[:, t], a[:, t] * size + (beta[:, t] * u[:, t]).abs()
        h[:, t], hs[:, t] = now, size
    zero = torch.zeros((), dtype=torch.float64)
    out = {"h": (torch.where(m, h, zero), torch.where(m, hs, zero)), "last": (now, size)}
    if gh is None:
        return out
    gh = torch.where(m, gh.double(), zero)
    C, Cs = glast.double(), glast.double().abs()
    dx, dr, di, dxs, drs, dis, q, qs = (torch.zeros(n, length, width, dtype=torch.float64) for _ in range(8))
    ratio = torch.where(beta > 0, l / torch.where(beta > 0, beta, 1.0), zero)
    for t in range(length - 1, -1, -1):
        G, Gs = gh[:, t] + C, gh[:, t].abs() + Cs
        du, dus = G * beta[:, t], Gs * beta[:, t]
        q[:, t] = G * a[:, t] * (before[:, t] * l[:, t] - u[:, t] * a[:, t] * ratio[:, t])
        qs[:, t] = Gs * a[:, t] * (befores[:, t] * l[:, t].abs() + (u[:, t] * a[:, t] * ratio[:, t]).abs())
        dx[:, t], dxs[:, t] = du * si[:, t], dus * si[:, t]
        di[:, t], dis[:, t] = du * u[:, t] * (1 - si[:, t]), (dus * u[:, t] * (1 - si[:, t])).abs()
        dr[:, t], drs[:, t] = q[:, t] * (1 - sr[:, t]), qs[:, t] * (1 - sr[:, t])
        C, Cs = a[:, t] * G, a[:, t] * Gs
    hide = lambda t: torch.where(m, t, zero)      # noqa: E731
    k = torch.sigmoid(lam) / sp
    out.update(dx=(hide(dx), hide(dxs)), dr=(hide(dr), hide(drs)), di=(hide(di), hide(dis)), dlam=(hide(q).sum((0, 1)) * k, hide(qs).sum((0, 1)) * k),
               dstate=(C, Cs))
    return out


def norm_64(x, o, gate, wp, sc, wn, eps, act):
    """autograd in 64 bits; o None: a plain norm"""
    y = x
    if o is not None:
        g = 1.0 if act is None else torch.sigmoid(gate) if act == "sigmoid" else torch.nn.functional.silu(gate)
        y = x + sc * g * (o / (o.square().mean(-1, keepdim=True) + eps).sqrt() * wp)
    return y, None if wn is None else y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * wn


def logprobs_64(x, targets, k, mask):
    x = x.double()
    rows, items = x.shape
    live = torch.ones_like(x, dtype=torch.bool) if mask is None else (mask != 0).expand(rows, items)
    x = torch.where(live, x, -math.inf)
    bad = (torch.isnan(x) | (x == math.inf)).any(1, keepdim=True)
    some = (x > -math.inf).any(1, keepdim=True)
    lp = torch.where(some, torch.log_softmax(torch.where(some, x, 0.0), 1), -math.inf)
    lp = torch.where(bad, math.nan, lp)
    p = torch.exp(lp)
    entropy = -torch.where(p > 0, p * lp, torch.zeros(())).sum(1)
    entropy = torch.where(bad[:, 0], math.nan, entropy)
    has = torch.zeros(rows, dtype=torch.bool) if targets is None else (targets >= 0) & (targets < items)
    at = torch.where(has, targets, 0).long()[:, None] if targets is not None else torch.zeros(rows, 1, dtype=torch.long)
    logp = torch.where(has, torch.where(live.gather(1, at)[:, 0] | bad[:, 0], lp.gather(1, at)[:, 0], -math.inf), 0.0)
    top, index = torch.sort(torch.where(bad, 0.0, lp), dim=1, descending=True, stable=True)
    top, index = top[:, :k], index[:, :k]
    index = torch.where((top == -math.inf) | bad, -1, index)
    return dict(lp=lp, p=p, entropy=entropy, logp=logp, top=torch.where(bad, math.nan, top), index=index, has=has, at=at, live=live, some=some[:, 0])


# --------------------------------------------------------------------------------------------------------------- without a GPU
def test_refusals_of_the_recurrence():
    x, lam, st = torch.zeros(2, 5, 8), torch.zeros(8), torch.zeros(2, 8)
    bad = [
        ((x, x, x[:, :4], lam), {}), ((x, x, x.half(), lam), {}), ((x.double(), x.double(), x.double(), lam), {}), ((x, x, x, lam[:4]), {}),
        ((x, x, x, lam.half()), {}), ((x, x, x, lam), dict(state=st[:1])), ((x, x, x, lam), dict(state=st.half())),
        ((x, x, x, lam), dict(mask=torch.ones(2, 4))), ((x, x, x, lam), dict(sharpness=0.0)), ((x[0], x[0], x[0], lam), {}),
        ((x, x, None, lam), {}), ((x, x, x, lam), {}),                                       # the last: right, but on the CPU
    ]
    for args, kw in bad:
        with pytest.raises(LegoHipError, match="gated_scan"):
            F.gated_scan(*args, **kw)
    s = x[:, 0]
    for args, kw in [((s, s, s, lam, st[:1]), {}), ((s, s, s, lam, None), {}), ((x, x, x, lam, st), {}), ((s, s, s, lam, st), dict(mask=torch.ones(3))),
                     ((s, s, s.clone().requires_grad_(), lam, st), {}), ((s, s, s, lam, st), {})]:
        with pytest.raises(LegoHipError, match="gated_scan_step"):
            F.gated_scan_step(*args, **kw)


def test_refusals_of_the_norms():
    x, w = torch.zeros(3, 8), torch.zeros(8)
    for args, kw in [((x, x[:2], x, w, w), {}), ((x, x, x.half(), w, w), {}), ((x, x, None, w, w), {}), ((x, x, x, w, w), dict(act=None)),
                     ((x, x, x, w, w), dict(act="relu")), ((x, x, x, w[:4], w), {}), ((x, x, x, w, w.half()), {}), ((x, x, x, w, w, w[:1]), {}),
                     ((x, x, x, w, w), {})]:
        with pytest.raises(LegoHipError, match="gated_residual_norm"):
            F.gated_residual_norm(*args, **kw)
    for args in [(x, w[:4]), (x.double(), w.double()), (torch.zeros(2, 0), torch.zeros(0)), (torch.zeros(1, 16385), torch.zeros(16385)), (x, w)]:
        with pytest.raises(LegoHipError, match="rms_norm"):
            F.rms_norm(*args)


def test_refusals_of_the_log_probabilities():
    x, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    for args, kw in [((x, t[:2]), {}), ((x, t.float()), {}), ((x, t), dict(k=9)), ((x, t), dict(k=-1)), ((x, t), dict(k=2.0)),
                     ((torch.zeros(3, 500), t), dict(k=129)), ((x, t), dict(mask=torch.ones(3, 7))), ((x, t), dict(mask=torch.ones(1, 8))),
                     ((torch.zeros(3, 0), t), {}), ((x.double(), t), {}), ((x, t), {})]:
        with pytest.raises(LegoHipError, match="token_logprobs"):
            F.token_logprobs(*args, **kw)


def test_refusals_at_the_c_entry():
    h = _lib.lib()
    one = ctypes.c_void_p(64)
    z64 = ctypes.c_int64(0)
    err = lambda: h.lego_last_error().decode()      # noqa: E731
    fwd = lambda dt, n, length, width, x=one, ws=z64: h.lego_gated_scan_fwd(      # noqa: E731
        x, z64, z64, one, z64, z64, one, z64, z64, dt, one, ctypes.c_float(8.0), None, z64, None, one, one, None, None, ws, n, length, width, None)
    for dt, n, length, width, why in [(3, 1, 1, 4, "dtype"), (0, 65536, 1, 4, "sizes"), (0, 1, -1, 4, "sizes"), (0, 1, 0, 4, "length 0"),
                                      (0, 1, 4096, 64, "workspace")]:
        assert fwd(dt, n, length, width) != 0 and why in err(), (dt, n, length, width, err())
    assert fwd(0, 1, 1, 4, x=None) != 0 and "NULL" in err()
    assert fwd(0, 0, 5, 4) == 0 and fwd(0, 3, 5, 0) == 0                                      # nothing to do
    assert h.lego_gated_scan_bwd(one, z64, z64, one, z64, z64, one, z64, z64, one, z64, z64, 0, one, ctypes.c_float(8.0), None, z64, one, None, one, one,
                                 one, one, None, None, z64, 1, 5, 4, None) != 0 and "workspace" in err()
    far = ctypes.c_int64(1 << 24)
    assert h.lego_gated_scan_fwd(one, z64, far, one, z64, z64, one, z64, z64, 0, one, ctypes.c_float(8.0), None, z64, None, one, one, None, one,
                                 ctypes.c_int64(1 << 20), 1, 5, 4, None) != 0 and "strides" in err()
    assert h.lego_gated_scan_step(one, z64, one, z64, one, z64, 0, one, ctypes.c_float(8.0), None, None, one, one, 1, 4, None) != 0 and "NULL" in err()
    norm = lambda o, wn, act, rows, width: h.lego_block_norm_fwd(one, z64, o, z64, None, z64, 0, act, one, one, wn, ctypes.c_float(1e-6), one, one,      # noqa: E731
                                                                 None, rows, width, None)
    assert norm(None, None, 0, 3, 8) != 0 and "neither" in err()
    assert norm(one, one, 3, 3, 8) != 0 and "activation" in err()
    assert norm(one, one, 2, 3, 8) != 0 and "NULL" in err()                                   # a gate's activation without a gate
    assert norm(one, one, 0, 3, 16385) != 0 and "width" in err()
    assert norm(one, one, 0, 0, 8) == 0
    lp = lambda k, items, rows=3, dt=0: h.lego_token_logprobs_fwd(one, z64, dt, None, z64, one, 1, k, one, one, one, None, None, None, z64, rows, items, None)      # noqa: E731
    assert lp(129, 500) != 0 and "k=129" in err()
    assert lp(9, 8) != 0 and "k=9" in err()
    assert lp(2, 8) != 0 and "NULL" in err()
    assert lp(0, 0) != 0 and "sizes" in err()
    assert lp(0, 400000) != 0 and "workspace" in err()
    assert lp(0, 8, rows=0) == 0


def test_refusals_below_the_public_functions():
    """the registered ops end here: what the pointers rely on is looked at for them too, before anything is launched"""
    x, w, bad = torch.zeros(2, 70, 8), torch.zeros(8), torch.zeros(8, dtype=torch.float64)
    st, tiles = torch.zeros(2, 8), torch.zeros(2, 2, 8)
    for call in [lambda: K.gated_scan_fwd(x, x, x, bad), lambda: K.gated_scan_fwd(x, x[:1], x, w), lambda: K.gated_scan_fwd(x, x, x.half(), w),
                 lambda: K.gated_scan_fwd(x, x, x, w, torch.ones(2, 69)), lambda: K.gated_scan_fwd(x, x, x, w, None, st[:1]),
                 lambda: K.gated_scan_bwd(x, None, x, x, x, w, None, tiles[:, :1]), lambda: K.gated_scan_bwd(x[:, :1], None, x, x, x, w, None, tiles),
                 lambda: K.gated_scan_step(st, st, st, w[:4], st), lambda: K.gated_scan_step(st, st, st, w, st.half()),
                 lambda: K.gated_scan_step(st, st, st, w, st, torch.ones(3)), lambda: K.gated_scan_fwd(x, x, x, w)]:
        with pytest.raises(LegoHipError, match="gated_scan"):
            call()
    stat = torch.zeros(2, 2)
    for call in [lambda: K.block_norm_fwd(st, st, None, w, w, bad, 1e-6, 0), lambda: K.block_norm_fwd(st, st[:1], None, w, w, w, 1e-6, 0),
                 lambda: K.block_norm_bwd(st, st, st, st, None, w, w, w, 1e-6, 0, stat[:1]), lambda: K.block_norm_fwd(st, st, st, w, w, w, 1e-6, 2),
                 lambda: K.block_norm_fwd(torch.empty(1 << 31, 1, device="meta"), None, None, None, None, w[:1], 1e-6, 0)]:
        with pytest.raises(LegoHipError, match="block_norm"):
            call()
    t, index = torch.zeros(2, dtype=torch.int64), torch.zeros(2, 3, dtype=torch.int32)
    for call in [lambda: K.token_logprobs_fwd(st, t[:1]), lambda: K.token_logprobs_fwd(st, t.float()), lambda: K.token_logprobs_fwd(st, t, 3, st[:1]),
                 lambda: K.token_logprobs_fwd(st.double(), t), lambda: K.token_logprobs_fwd(torch.empty(1 << 31, 1, device="meta"), None),
                 lambda: K.token_logprobs_bwd(None, None, torch.zeros(2, 2), st, t, None, stat, w[:2], index),
                 lambda: K.token_logprobs_bwd(w[:2], None, None, st, t, None, stat, w[:2], index.long()), lambda: K.token_logprobs_fwd(st, t, 3)]:
        with pytest.raises(LegoHipError, match="token_logprobs"):
            call()


def test_workspaces_cover_what_the_kernels_index():
    h = _lib.lib()
    for n, length, width in [(1, 1, 1), (1, 10007, 301), (2, 32768, 768), (64, 50, 256), (65535, 3, 4), (1, 64 * 5 + 1, 1 << 12)]:
        slices, tiles = -(-width // 64), -(-length // 64)
        floats = h.lego_gated_scan_workspace(n, length, width)
        assert floats >= width and floats <= (2 * n * tiles + max(n, 1) * tiles) * width
        if n * slices >= 512 or tiles < 4:
            assert floats <= n * width                                                       # not cut: the partial sums of d lam alone
    assert h.lego_gated_scan_workspace(0, 5, 5) == h.lego_block_norm_workspace(0, 8) == h.lego_token_logprobs_workspace(0, 8, 0, 1) == 0
    assert h.lego_token_logprobs_workspace(4096, 30522, 1, 5) == 0                            # as many rows as fill the GPU: one chunk each
    assert h.lego_token_logprobs_workspace(1, 400000, 0, 20) >= 42


def test_shapes_without_a_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 130, 24, device="cuda", dtype=torch.bfloat16)
        lam = torch.empty(24, device="cuda")
        h, last, tiles = L.gated_scan(x, x, x, lam, None, None, 8.0, True)
        assert h.shape == x.shape and h.dtype == x.dtype and last.shape == (3, 24) and last.dtype == torch.float32 and tiles.shape == (3, 3, 24)
        y, n, stat = L.block_norm(x[0], x[0], x[0], lam, lam, None, 1e-6, 2, False)
        assert y.shape == (130, 24) and n.numel() == 0 and stat.shape == (1, 0)
        out = L.token_logprobs(x[0], None, None, 5)
        assert [tuple(t.shape) for t in out] == [(130,), (130,), (130, 2), (130, 5), (130, 5)] and out[4].dtype == torch.int32


# --------------------------------------------------------------------------------------------------------------- GPU: the recurrence
def _rand(seed, *shape, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _lam(width, seed=9, lo=0.6, hi=0.9999):
    g = torch.Generator().manual_seed(seed)
    d = lo + (hi - lo) * torch.rand(width, generator=g)
    return torch.log(torch.expm1(-torch.log(d) / 8.0))


def _mask(kind, n, length, seed=3):
    g = torch.Generator().manual_seed(seed)
    if kind is None:
        return None
    if kind == "prefix":
        lens = torch.randint(0, length + 1, (n,), generator=g)
        lens[0] = 0
        return torch.arange(length)[None] < lens[:, None]
    if kind == "holes":
        return torch.rand(n, length, generator=g) < 0.5
    return torch.zeros(n, length, dtype=torch.bool)


def _scan_case(n, length, width, dtype, mask, state, packed=False, seed=1):
    if packed:
        rows = _rand(seed, n, length, 3 * width, dtype=dtype)
        x, r, i = rows[..., :width], rows[..., width:2 * width], rows[..., 2 * width:]
    else:
        x, r, i = (_rand(seed + q, n, length, width, dtype=dtype) for q in range(3))
    m = _mask(mask, n, length)
    if m is not None:                                                                        # what a mask hides must not matter
        junk = torch.tensor([math.nan, math.inf, -math.inf, 3e38])
        for q, t in enumerate((x, r, i)):
            t[~m] = junk[(torch.arange(width) + q) % 4].to(dtype)
    return x, r, i, _lam(width), m, _rand(seed + 7, n, width) if state else None


def _memory(length):
    """steps whose errors can add up: 1 / (1 - a) at the slowest decay of _lam, at most the length"""
    return min(length, 2000)


# Roundings a value: l = k sigmoid(r) -- softplus 6, exponential 2 + |r| for its argument (|r| <= 6), sum and reciprocal 3, products 2: 20, weighed by
# |l| <= 8 softplus(lam) <= 0.52 in a, plus its own rounding, one product and one sum a step: 12 a step of memory.  beta 12, sigmoid(i) 12, products
# 4: 30.  Gradients pass through both: 2 x.
SCAN_STEP, SCAN_CELL = 12, 30
SHAPES = [(1, 1, 1), (2, 3, 5), (3, 63, 64), (2, 64, 68), (5, 65, 100), (1, 130, 257), (2, 1003, 72), (1, 300, 33)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", [None, "prefix", "holes", "nothing"])
@pytest.mark.parametrize("shape", SHAPES)
def test_scan_and_its_gradients(shape, mask, dtype):
    n, length, width = shape
    packed, state = width % 2 == 0, (n + length) % 2 == 0
    x, r, i, lam, m, st = _scan_case(n, length, width, dtype, mask, state, packed)
    gh, glast = _rand(20, n, length, width, dtype=dtype), _rand(21, n, width)
    want = scan_64(x, r, i, lam, m, st, 8.0, gh, glast)
    if packed:
        rows = torch.cat((x, r, i), -1).cuda()
        leaves = [t.detach().requires_grad_() for t in (rows[..., :width], rows[..., width:2 * width], rows[..., 2 * width:])]
    else:
        leaves = [t.cuda().requires_grad_() for t in (x, r, i)]
    leaves.append(lam.cuda().requires_grad_())
    if st is not None:
        leaves.append(st.cuda().requires_grad_())
    md = None if m is None else m.cuda()
    h, last = F.gated_scan(*leaves[:4], mask=md, state=leaves[4] if st is not None else None)
    with torch.no_grad():
        h2, last2 = F.gated_scan(*leaves[:4], mask=md, state=leaves[4] if st is not None else None)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    many = SCAN_STEP * _memory(length) + SCAN_CELL
    check(h, *want["h"], many)
    check(last, *want["last"], many)
    grads = torch.autograd.grad((h, last), leaves, (gh.cuda(), glast.cuda()))
    for name, g in zip(("dx", "dr", "di", "dlam", "dstate"), grads):
        check(g, *want[name], 2 * many + (n * length if name == "dlam" else 0))
    again = torch.autograd.grad(F.gated_scan(*leaves[:4], mask=md, state=leaves[4] if st is not None else None), leaves, (gh.cuda(), glast.cuda()))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,mask,dtype",
                         [((200, 260, 24), m, t) for m in (None, "prefix", "holes") for t in TYPES] +          # forward: a workgroup a sequence, 5 tiles each
                         [((230, 260, 24), m, t) for m in (None, "holes") for t in TYPES] +                    # backward too
                         [((190, 1280, 24), m, torch.bfloat16) for m in (None, "prefix")] +                    # chunks of 4 tiles
                         [((52, 193, 2561), "prefix", torch.float16), ((52, 193, 2561), None, torch.float32)])    # backward: workgroups with two sequences
def test_scan_of_many_sequences(shape, mask, dtype):
    test_scan_and_its_gradients(shape, mask, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("mask_type", [torch.bool, torch.uint8, torch.int32, torch.int64, torch.float32])
def test_scan_takes_masks_of_any_type_and_strided_everything(mask_type):
    n, length, width = 3, 70, 12
    x, r, i, lam, m, st = _scan_case(n, length, width, torch.float32, "prefix", True)
    want = scan_64(x, r, i, lam, m, st, 8.0)
    wide = torch.zeros(n, length, 2, dtype=mask_type, device="cuda")
    wide[..., 0] = m.cuda().to(mask_type)
    turned = [t.cuda().transpose(0, 1).contiguous().transpose(0, 1) for t in (x, r)] + [i.cuda().transpose(1, 2).contiguous().transpose(1, 2)]
    h, last = F.gated_scan(*turned, lam.cuda()[:, None].expand(width, 2)[:, 0], mask=wide[..., 0], state=st.cuda().t().contiguous().t())
    many = SCAN_STEP * length + SCAN_CELL
    check(h, *want["h"], many)
    check(last, *want["last"], many)


@pytest.mark.gpu
def test_scan_without_steps_channels_or_sequences():
    lam = _lam(8).cuda()
    for n, length, width in [(2, 0, 8), (0, 5, 8), (2, 5, 0)]:
        x = torch.zeros(n, length, width, device="cuda", requires_grad=True)
        st = torch.ones(n, width, device="cuda", requires_grad=True)
        h, last = F.gated_scan(x, x, x, lam[:width], state=st)
        assert h.shape == x.shape and (length > 0 or torch.equal(last, st))
        gx, gs = torch.autograd.grad(last.sum() + h.sum(), (x, st))
        assert gx.shape == x.shape and gs.shape == st.shape and (length > 0 or bool((gs == 1).all()))
    assert float(F.gated_scan(*(torch.zeros(2, 0, 8, device="cuda"),) * 3, lam)[1].abs().max()) == 0.0


@pytest.mark.gpu
def test_scan_at_the_ends_of_its_gates():
    """open and closed gates: no NaN where 1 - a^2 or softplus underflow, and the state passes through untouched"""
    n, length, width = 1, 9, 8
    r = torch.tensor([0.0, 200.0, -200.0, -90.0, 30.0, -30.0, 0.0, 0.0]).expand(n, length, width).contiguous()
    i = torch.tensor([200.0, -200.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0]).expand(n, length, width).contiguous()
    lam = torch.tensor([0.0, 3.0, 0.0, 3.0, 30.0, -3.0, -200.0, 90.0])
    x, st, gh, gl = _rand(1, n, length, width), _rand(2, n, width), _rand(3, n, length, width), _rand(4, n, width)
    want = scan_64(x, r, i, lam, None, st, 8.0, gh, gl)
    leaves = [t.cuda().requires_grad_() for t in (x, r, i, lam, st)]
    h, last = F.gated_scan(*leaves[:4], state=leaves[4])
    grads = torch.autograd.grad((h, last), leaves, (gh.cuda(), gl.cuda()))
    # arguments up to 720: the exponential's argument adds 720 roundings
    for got, name in zip((h, last, *grads), ("h", "last", "dx", "dr", "di", "dlam", "dstate")):
        assert torch.isfinite(got).all(), name
        # A gate below 2^-126 counts as closed (fp32 has no normal number for it).  Then l is off by |k| 2^-126, k = 8 softplus(lam) <= 720, and what
        # goes by its root -- beta = sqrt(-2 l), l / beta = -sqrt(-l / 2) -- by sqrt(2 k) 2^-63 <= 38 * 2^-63, times |G| |u| < 64 and 9 steps' sum.
        check(got, want[name][0], want[name][1], 800 * length, floor=38 * 2.0 ** -63 * 64 * length)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,width", [(1, 1), (64, 256), (5, 301), (513, 64)])
def test_steps_follow_the_scan(n, width, dtype):
    x, r, i, lam, m, st = _scan_case(n, 4, width, dtype, "holes", True, packed=width % 2 == 0)
    want = scan_64(x, r, i, lam, m, st, 8.0)
    rows = torch.cat((x, r, i), -1).cuda()
    state, kept = st.cuda(), st.cuda()
    md = m.cuda()
    for t in range(4):
        h, new = F.gated_scan_step(*(rows[:, t, q * width:(q + 1) * width] for q in range(3)), lam.cuda(), state, mask=md[:, t])
        check(h, want["h"][0][:, t], want["h"][1][:, t], 4 * SCAN_STEP + SCAN_CELL)
        state = new
    check(state, *want["last"], 4 * SCAN_STEP + SCAN_CELL)
    assert torch.equal(kept, st.cuda())
    h, last = F.gated_scan(*(rows[..., q * width:(q + 1) * width] for q in range(3)), lam.cuda(), mask=md, state=st.cuda())
    assert torch.allclose(last, state, rtol=1e-5, atol=1e-5)


# --------------------------------------------------------------------------------------------------------------- GPU: the norms
NORM_SHAPES = [(1, 1), (3, 5), (7, 64), (130, 256), (9, 300), (65, 768), (4099, 68), (5, 1024), (3, 1025), (6, 2048), (2, 4096), (2, 4100), (2, 16384), (1, 8191)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("half", ["both", "block", "norm"])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_norms_and_their_gradients(shape, half, dtype):
    rows, width = shape
    act = [None, "sigmoid", "silu"][(rows + width) % 3]
    x, o, g = (_rand(q, rows, width, dtype=dtype, scale=2.0) for q in (1, 2, 3))
    if rows > 2:
        x[1], o[1] = 0, 0                                                                    # a row of zeros: its norm is 0, not NaN
    wp, sc, wn = 1 + _rand(4, width, scale=0.3), _rand(5, width), 1 + _rand(6, width, scale=0.3)
    gy, gn = _rand(7, rows, width, dtype=dtype), _rand(8, rows, width, dtype=dtype)
    block, norm = half != "norm", half != "block"
    ops = {"x": x, **({"o": o, "post_w": wp, "scale": sc} if block else {}), **({"gate": g} if block and act else {}), **({"next_w": wn} if norm else {})}
    wide = {k: v.double().requires_grad_() for k, v in ops.items()}
    eps = 1e-5
    y64, n64 = norm_64(wide["x"], wide.get("o"), wide.get("gate"), wide.get("post_w"), wide.get("scale"), wide.get("next_w"), eps, act)
    outs = [(t, gg) for t, gg, on in ((y64, gy, block), (n64, gn, norm)) if on]
    g64 = dict(zip(wide, torch.autograd.grad([t for t, _ in outs], list(wide.values()), [gg.double() for _, gg in outs])))
    dev = {k: v.cuda().requires_grad_() for k, v in ops.items()}
    if block:
        y, n = F.gated_residual_norm(dev["x"], dev["o"], dev.get("gate"), dev["post_w"], dev["scale"], dev.get("next_w"), eps=eps, act=act)
        assert (n is None) == (not norm)
    else:
        y, n = None, F.rms_norm(dev["x"], dev["next_w"], eps=eps)
    # A sum of `width` squares in four-fold lanes and a tree: at most width / 256 + 12 roundings of its terms, halved by the root; 20 more a value.
    many = width / 256 + 40
    ok = lambda t, want, terms, m: check(t, want.detach(), terms.detach(), m)      # noqa: E731
    size = y64.detach().abs() + (0 if not block else x.double().abs())
    if block:
        ok(y, y64, size, many)
    if norm:
        r64 = 1 / (y64.detach().square().mean(-1, keepdim=True) + eps).sqrt()
        ok(n, n64, size * r64 * wn.double().abs(), many)
    grads = dict(zip(dev, torch.autograd.grad([t for t in (y, n) if t is not None], list(dev.values()), [gg.cuda() for _, gg in outs])))
    # the terms of the gradients: d = gy + r (t - yh mean(t yh)), and the block's from d
    d = gy.double().abs() if block else torch.zeros(rows, width, dtype=torch.float64)
    if norm:
        yh, t = size * r64, gn.double().abs() * wn.double().abs()
        d = d + r64 * (t + yh * (t * yh).mean(-1, keepdim=True))
        ok(grads["next_w"], g64["next_w"], (gn.double().abs() * yh).sum(0), many + rows)
    ok(grads["x"], g64["x"], d, 3 * many)
    if block:
        ro = 1 / (o.double().square().mean(-1, keepdim=True) + eps).sqrt()
        oh, gd = o.double().abs() * ro, g.double()
        sig = torch.sigmoid(gd)
        a = torch.ones_like(gd) if act is None else sig if act == "sigmoid" else (gd * sig).abs()
        slope = sig * (1 - sig) if act == "sigmoid" else sig + a * (1 - sig)
        e = d * sc.double().abs() * a * wp.double().abs()
        ok(grads["o"], g64["o"], ro * (e + oh * (e * oh).mean(-1, keepdim=True)), 4 * many)
        z = (d * a * oh).sum(0)
        ok(grads["post_w"], g64["post_w"], z * sc.double().abs(), 4 * many + rows)
        ok(grads["scale"], g64["scale"], z * wp.double().abs(), 4 * many + rows)
        if act:
            ok(grads["gate"], g64["gate"], d * sc.double().abs() * oh * wp.double().abs() * slope, 4 * many)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_norms_of_strided_rows(dtype):
    rows, width = 21, 36
    packed = _rand(1, rows, 3, width + 4, dtype=dtype).cuda()
    x, o, g = (packed[:, q, :width] for q in range(3))
    w = torch.ones(width, device="cuda")
    y, n = F.gated_residual_norm(x, o, g, w, 0.5 * w, w)
    y2, n2 = F.gated_residual_norm(x.contiguous(), o.contiguous(), g.contiguous(), w, 0.5 * w, w)
    assert torch.equal(y, y2) and torch.equal(n, n2)
    odd = packed.view(-1)[1:1 + rows * width].view(rows, width)                               # rows that are not aligned
    assert torch.equal(F.rms_norm(odd, w), F.rms_norm(odd.clone(), w))
    turned = x.t().contiguous().t()
    assert torch.equal(F.rms_norm(turned, w), F.rms_norm(x.contiguous(), w))
    one = x[0].float()
    assert F.rms_norm(one.expand(4, 5, width), w).shape == (4, 5, width)
    lead = one.clone().requires_grad_()
    g1 = torch.autograd.grad(F.rms_norm(lead.expand(4, 5, width), w).sum(), lead)[0]         # a broadcast input: its rows' gradients add up
    g2 = torch.autograd.grad(F.rms_norm(lead[None], w).sum(), lead)[0]
    assert torch.allclose(g1, 20 * g2, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_norms_of_no_rows():
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y, n = F.gated_residual_norm(x, x, x, w, w, w)
    g = torch.autograd.grad(y.sum() + n.sum(), (x, w))
    assert y.shape == n.shape == g[0].shape == (0, 8) and float(g[1].abs().max()) == 0.0


# --------------------------------------------------------------------------------------------------------------- GPU: log probabilities
def _logits(rows, items, dtype, kind, seed=1):
    x = _rand(seed, rows, items, scale=3.0)
    if kind == "ties":
        x = x.round()
    if kind == "constant":
        x = torch.full((rows, items), -1.25)
    if kind == "edges":                                                                      # -inf, the type's lowest value, huge and tiny
        x.view(-1)[::3] = -math.inf
        x[:, 1::5] = torch.finfo(dtype).min
        x[0] = -math.inf
        if rows > 1:
            x[1] = torch.finfo(dtype).min
        if rows > 2:
            x[2] = -math.inf
            x[2, items // 2] = 4.0
        if rows > 3:
            x[3] = torch.finfo(dtype).max
    return x.to(dtype)


LP_SHAPES = [(1, 1), (3, 2), (5, 7), (4, 1000), (2, 1023), (6, 4097), (33, 30522), (1, 65238), (2100, 257)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["plain", "ties", "constant", "edges", "masked"])
@pytest.mark.parametrize("shape", LP_SHAPES)
def test_log_probabilities_and_their_gradients(shape, kind, dtype):
    rows, items = shape
    k = min(items, [0, 1, 5, 20, 128][(rows + items) % 5])
    x = _logits(rows, items, dtype, kind)
    g = torch.Generator().manual_seed(5)
    targets = torch.randint(-1, items, (rows,), generator=g)
    mask = None
    if kind == "masked":
        mask = torch.rand(rows, items, generator=g) < 0.6
        mask[rows // 2] = False
        if rows > 4:
            mask[0] = False
            mask[0, items // 3] = True
        x[~mask] = math.nan
        x[:, ::7] = torch.where(mask[:, ::7], x[:, ::7], math.inf)
    w = logprobs_64(x, targets, k, mask)
    xd = x.cuda().requires_grad_()
    logp, entropy, top, index = F.token_logprobs(xd, targets.cuda() if rows % 2 else targets.int().cuda(), k=k, mask=None if mask is None else mask.cuda())
    # x - m is exact to a rounding of its size; 2 a term of S and T, log 2, and the sum of up to items / 256 + 12 terms, over S >= 1.
    # Terms: |x| + |lse| for a log probability; the entropy's are sum p |ln p| + ln S (d up to 200 by its own rounding).
    many = items / 256 + 40
    xm = torch.where(torch.isfinite(x.double()) & w["live"], x.double().abs(), 0.0)
    big = torch.where(w["p"] > 0, xm, 0.0).amax(1) + 12.0
    check(logp, w["logp"], big, many)
    check(entropy, w["entropy"], big, many)
    check(top, w["top"], big[:, None], many)
    assert torch.equal(index.cpu().long(), w["index"].long())
    gl, ge, gt = _rand(6, rows), _rand(7, rows), _rand(8, rows, k)
    out, grads = [logp, entropy], [gl.cuda(), ge.cuda()]
    if k:
        out, grads = out + [top], grads + [gt.cuda()]
    dx = torch.autograd.grad(out, xd, grads)[0]
    p, lp = w["p"], w["lp"]
    has = w["has"].double()
    some = w["some"][:, None]
    taken = torch.where(w["index"] >= 0, gt.double(), 0.0) if k else torch.zeros(rows, 1, dtype=torch.float64)
    a = torch.where(p > 0, lp + w["entropy"][:, None], 0.0)
    G = (gl.double() * has + taken.sum(1))[:, None]
    d = -p * (G + ge.double()[:, None] * a)
    d.scatter_add_(1, w["at"], (gl.double() * has)[:, None])
    if k:
        d.scatter_add_(1, w["index"].clamp(min=0).long(), taken)
    d = torch.where(w["live"] & some, d, 0.0)
    size = p * (gl.double().abs() * has + taken.abs().sum(1))[:, None] + p * ge.double().abs()[:, None] * (a.abs() + big[:, None])
    size.scatter_add_(1, w["at"], (gl.double().abs() * has)[:, None])
    if k:
        size.scatter_add_(1, w["index"].clamp(min=0).long(), taken.abs())
    # p = exp(x - lse): its exponent is off by `many` roundings of its terms
    check(dx, d, size * (1 + big[:, None]), many)


@pytest.mark.gpu
def test_a_row_that_is_not_a_distribution():
    x = _rand(1, 6, 5000)
    x[1, 77], x[2, 4999], x[3, 0] = math.nan, math.inf, -math.inf
    x[4] = math.nan
    xd = x.cuda().requires_grad_()
    t = torch.tensor([3, 3, -1, 0, -1, 5])
    logp, entropy, top, index = F.token_logprobs(xd, t.cuda(), k=4)
    w = logprobs_64(x, t, 4, None)
    check(logp, w["logp"], 20.0, 100)
    check(entropy, w["entropy"], 20.0, 100)
    check(top, w["top"], 20.0, 100)
    assert torch.equal(index.cpu().long(), w["index"].long())
    d = torch.autograd.grad((logp.sum(), entropy.sum()), xd)[0]
    assert torch.isfinite(d[0]).all() and torch.isfinite(d[3]).all() and torch.isfinite(d[5]).all() and torch.isnan(d[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_the_largest_where_one_lane_owns_them_all(dtype):
    """rows whose large elements repeat with the lanes' stride: the list of candidates overflows, and the items come one at a time"""
    vec = 128 // torch.finfo(dtype).bits
    items, k = 256 * vec * 40, 100
    x = torch.zeros(3, items)
    for row, lanes in enumerate((1, 40, 128)):
        for lane in range(lanes):
            x[row].view(-1, 256, vec)[:, lane] = 1 + _rand(row, 40, vec).abs()
    x = x.to(dtype)
    w = logprobs_64(x, None, k, None)
    logp, entropy, top, index = F.token_logprobs(x.cuda(), k=k)
    assert torch.equal(index.cpu().long(), w["index"].long()) and float(logp.abs().max()) == 0.0
    check(top, w["top"], 20.0, 300)
    check(entropy, w["entropy"], 20.0, 300)


@pytest.mark.gpu
def test_log_probabilities_of_strided_rows_and_one_mask_for_all():
    wide = _rand(1, 9, 1301, dtype=torch.bfloat16).cuda()
    x = wide[:, 3:1203]
    mask = torch.rand(1200, generator=torch.Generator().manual_seed(1)) < 0.5
    t = torch.arange(9, device="cuda") * 100
    a = F.token_logprobs(x, t, k=7, mask=mask.cuda())
    b = F.token_logprobs(x.contiguous(), t, k=7, mask=mask.expand(9, 1200).contiguous().cuda())
    assert all(torch.allclose(p, q, rtol=1e-5, atol=1e-6) for p, q in zip(a, b)) and torch.equal(a[3], b[3])
    xl, xc = x.detach().requires_grad_(), x.contiguous().requires_grad_()
    ga = torch.autograd.grad(F.token_logprobs(xl, t, mask=mask.cuda())[0].sum(), xl)[0]
    gb = torch.autograd.grad(F.token_logprobs(xc, t, mask=mask.cuda())[0].sum(), xc)[0]
    assert torch.equal(ga != 0, gb != 0) and torch.allclose(ga.float(), gb.float(), rtol=2 ** -7, atol=1e-6)
    lead = F.token_logprobs(x.contiguous().view(3, 3, 1200), t.view(3, 3), k=2)
    assert lead[0].shape == (3, 3) and lead[2].shape == (3, 3, 2)
    turned = F.token_logprobs(x.t().contiguous().t(), t, k=7, mask=mask.cuda())
    assert torch.equal(turned[3], a[3])


@pytest.mark.gpu
def test_log_probabilities_of_no_rows():
    x = torch.zeros(0, 9, device="cuda", requires_grad=True)
    out = F.token_logprobs(x, torch.zeros(0, dtype=torch.int64, device="cuda"), k=3)
    assert [tuple(t.shape) for t in out] == [(0,), (0,), (0, 3), (0, 3)]
    assert torch.autograd.grad(out[0].sum(), x)[0].shape == (0, 9)


# --------------------------------------------------------------------------------------------------------------- GPU: all of them
def _differences(f, leaves, seed, eps=1e-2):
    """(f(x + eps v) - f(x - eps v)) / (2 eps) in a random direction, f summed in 64 bits"""
    vs = [_rand(seed + q, *t.shape).cuda() for q, t in enumerate(leaves)]
    with torch.no_grad():
        hi = f(*[t + eps * v for t, v in zip(leaves, vs)])
        lo = f(*[t - eps * v for t, v in zip(leaves, vs)])
    return (float(hi) - float(lo)) / (2 * eps), vs


@pytest.mark.gpu
def test_gradients_against_differences():
    # a central difference is off by eps^2 / 6 of the third derivative (a few times the slope here: 1e-3) and by f's roundings over eps
    n, length, width = 2, 70, 20
    pick = [_rand(40 + q, n, length, width).cuda().double() for q in range(2)]
    seqs = [_rand(q, n, length, width).cuda() for q in range(3)] + [_lam(width, lo=0.6, hi=0.95).cuda(), _rand(5, n, width).cuda()]
    scan = lambda x, r, i, lam, st: (F.gated_scan(x, r, i, lam, state=st)[0].double() * pick[0]).sum()      # noqa: E731
    rows = [_rand(q, n * length, width).cuda() for q in range(3)] + [1 + _rand(6, width, scale=0.1).cuda(), _rand(7, width).cuda(), 1 + _rand(8, width, scale=0.1).cuda()]
    pick2 = [p.view(-1, width) for p in pick]

    def norms(*a):
        y, nx = F.gated_residual_norm(*a, act="silu")
        return (y.double() * pick2[0] + nx.double() * pick2[1]).sum()
    logits = [_rand(9, 12, 333).cuda()]
    t = (torch.arange(12, device="cuda") * 7) % 333

    def probs(x):
        logp, entropy, top, _ = F.token_logprobs(x, t, k=3)
        return (logp.double() + 0.5 * entropy.double()).sum() + 0.3 * top.double()[:, 0].sum()
    for f, leaves in ((scan, seqs), (norms, rows), (probs, logits)):
        slope, vs = _differences(f, leaves, 60)
        live = [x.clone().requires_grad_() for x in leaves]
        grads = torch.autograd.grad(f(*live), live)
        got = sum(float((g.double() * v.double()).sum()) for g, v in zip(grads, vs))
        size = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
        assert abs(got - slope) <= 2e-2 * size + 1e-2, (got, slope, size)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["gated_scan", "gated_scan_bwd", "gated_scan_step", "block_norm", "block_norm_plain", "block_norm_bwd", "token_logprobs",
                                  "token_logprobs_bwd"])
def test_opcheck(name):
    x, r, i = (_rand(q, 2, 70, 12).cuda() for q in range(3))
    lam, st, w = _lam(12).cuda(), _rand(5, 2, 12).cuda(), torch.ones(12, device="cuda")
    mask = torch.ones(2, 70, dtype=torch.bool, device="cuda")
    a, b, c = (t.view(-1, 12) for t in (x, r, i))
    req = lambda *ts: tuple(t.clone().requires_grad_() for t in ts)      # noqa: E731
    ent = torch.zeros(140, device="cuda")
    args = {
        "gated_scan": (*req(x, r, i, lam), mask, *req(st), 8.0, True),
        "gated_scan_bwd": (x, st, x, r, i, lam, mask, torch.zeros(2, 2, 12, device="cuda"), 8.0),
        "gated_scan_step": (x[:, 0], r[:, 0], i[:, 0], lam, st, mask[:, 0], 8.0),
        "block_norm": (*req(a, b, c, w, w, w), 1e-6, 2, True),
        "block_norm_plain": (*req(a), None, None, None, None, *req(w), 1e-6, 0, True),
        "block_norm_bwd": (a, b, a, b, c, w, w, w, torch.ones(2, 140, device="cuda"), 1e-6, 2),
        "token_logprobs": (*req(a), torch.zeros(140, dtype=torch.int64, device="cuda"), None, 3),
        "token_logprobs_bwd": (ent, ent, None, a, torch.zeros(140, dtype=torch.int64, device="cuda"), None, torch.zeros(140, 2, device="cuda"), ent,
                               torch.zeros(140, 3, dtype=torch.int32, device="cuda")),
    }[name]
    torch.library.opcheck(getattr(L, name.replace("_plain", "")).default, args,
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic"))


def _all_of_them(rows, lam, st, mask, w, scale, table, targets):
    """the operators as an encoder uses them: norm, recurrence, tail, log probabilities over a catalogue, and the gradients of all of it"""
    n, length, width = rows.shape
    x = rows.detach().requires_grad_()
    a = F.rms_norm(x, w)
    h, last = F.gated_scan(a, a * 0.5, -a, lam, mask=mask, state=st)
    y, nx = F.gated_residual_norm(x, h, a, w, scale, w)
    logits = F.linear(nx[:, -1].contiguous(), table)
    logp, entropy, top, index = F.token_logprobs(logits, targets, k=4)
    return (h, last, y, nx, logp, entropy, top, index) + torch.autograd.grad((logp.sum() + 0.1 * entropy.sum() + y.sum(), last), (x,), (None, st))


def _stack(seed=1, n=3, length=140, width=32, items=5000):
    return (_rand(seed, n, length, width).cuda(), _lam(width).cuda(), _rand(seed + 1, n, width).cuda(), _mask("prefix", n, length).cuda(),
            (1 + _rand(seed + 2, width, scale=0.1)).cuda(), _rand(seed + 3, width).cuda(), _rand(seed + 4, items, width).cuda(),
            torch.tensor([5, -1, 4999], device="cuda"))


@pytest.mark.gpu
def test_scan_steps_that_lie_far_apart():
    """steps 2^24 elements apart, further than a tile's 32-bit offsets reach (one tensor of three is), and a single step with such a stride"""
    far = torch.zeros((1 << 24) * 2 + 8, dtype=torch.float16, device="cuda").as_strided((1, 3, 8), (0, 1 << 24, 1))
    x, r, i = (_rand(50 + q, 1, 3, 8, dtype=torch.float16).cuda() for q in range(3))
    lam = _rand(53, 8).cuda()
    far.copy_(x)
    for length in (3, 1):
        want, last = F.gated_scan(x[:, :length], r[:, :length], i[:, :length], lam)
        got, state = F.gated_scan(far[:, :length], r[:, :length], i[:, :length], lam)
        assert torch.equal(got, want) and torch.equal(state, last)


@pytest.mark.gpu
def test_operands_of_another_device_are_refused():
    x, w, t = _rand(1, 2, 3, 8).cuda(), _rand(2, 8).cuda(), torch.zeros(2, 3, dtype=torch.int64)
    for grad in (False, True):
        x = x.detach().requires_grad_(grad)
        for call in [lambda: F.gated_scan(x, x, x, w.cpu()), lambda: F.gated_scan(x, x.detach().cpu(), x, w), lambda: F.rms_norm(x, w.cpu()),
                     lambda: F.gated_scan(x, x, x, w, mask=torch.ones(2, 3)), lambda: F.gated_residual_norm(x, x, x, w, w.cpu(), w),
                     lambda: F.token_logprobs(x, t), lambda: F.token_logprobs(x, mask=torch.ones(8)),
                     lambda: F.gated_scan_step(x.detach()[0], x.detach()[0], x.detach()[0], w, torch.zeros(3, 8))]:
            with pytest.raises(LegoHipError):
                call()


@pytest.mark.gpu
def test_together_on_another_stream():
    args = _stack()
    want = _all_of_them(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _all_of_them(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_together_in_two_graphs_replayed_in_turn():
    """captured, replayed with new inputs and eager work between the replays; two graphs share nothing"""
    one, two = _stack(1), _stack(50)
    inputs = [[t.clone() for t in one], [t.clone() for t in two]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in inputs:
            _all_of_them(*a)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for a in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_all_of_them(*a))
        graphs.append(g)
    for seed in (1, 7, 13):
        fresh = [_stack(seed), _stack(seed + 100)]
        want = [_all_of_them(*f) for f in fresh]
        for a, f in zip(inputs, fresh):
            for dst, src in zip(a, f):
                dst.copy_(src)
        graphs[0].replay()
        graphs[1].replay()
        _all_of_them(*one)
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(o, w))


@pytest.mark.gpu
def test_nothing_is_written_outside_the_outputs():
    """outputs laid inside a larger buffer through the tensor-level wrappers' own allocations would hide a stray store: the C entries write into a
    buffer with guard bands"""
    n, length, width, rows, items, k = 2, 67, 7, 5, 1001, 3
    guard = 64

    def banded(count, dtype=torch.float32):
        t = torch.full((count + 2 * guard,), 7.0 if dtype.is_floating_point else 7, dtype=dtype, device="cuda")
        return t, ctypes.c_void_p(t.data_ptr() + guard * t.element_size())

    x, r, i = (_rand(q, n, length, width).cuda() for q in range(3))
    lam, p, st = _lam(width).cuda(), K._ptr, K._stream()
    h, hp = banded(n * length * width)
    last, lp = banded(n * width)
    tiles, tp = banded(n * 2 * width)
    size = _lib.lib().lego_gated_scan_workspace(n, length, width)
    ws, wp = banded(size)
    s = (length * width, width)
    _lib.call("lego_gated_scan_fwd", p(x), *s, p(r), *s, p(i), *s, 0, p(lam), 8.0, None, 0, None, hp, lp, tp, wp, size, n, length, width, st)
    outs = [banded(n * length * width) for _ in range(3)] + [banded(width), banded(n * width)]
    _lib.call("lego_gated_scan_bwd", p(x), *s, p(r), *s, p(i), *s, p(x), *s, 0, p(lam), 8.0, None, 0, tp, None, *(o[1] for o in outs), wp, size, n,
              length, width, st)
    w = torch.ones(width, device="cuda")
    m = n * length
    y, nx, stat = banded(m * width), banded(m * width), banded(2 * m)
    _lib.call("lego_block_norm_fwd", p(x), width, p(r), width, p(i), width, 0, 2, p(w), p(w), p(w), 1e-6, y[1], nx[1], stat[1], m, width, st)
    size = _lib.lib().lego_block_norm_workspace(m, width)
    ws2, wp2 = banded(size)
    more = [banded(m * width) for _ in range(3)] + [banded(width) for _ in range(3)]
    _lib.call("lego_block_norm_bwd", p(x), width, p(r), width, p(i), width, 0, 2, p(w), p(w), p(w), 1e-6, p(x), width, p(r), width, stat[1],
              *(o[1] for o in more), wp2, size, m, width, st)
    logits = _rand(4, rows, items).cuda()
    size = _lib.lib().lego_token_logprobs_workspace(rows, items, 0, k)
    ws3, wp3 = banded(max(size, 1), torch.int64)
    row = [banded(rows), banded(rows), banded(2 * rows)] + [banded(rows * k), banded(rows * k, torch.int32)]
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    _lib.call("lego_token_logprobs_fwd", p(logits), items, 0, None, 0, p(t), 1, k, *(o[1] for o in row), wp3, size, rows, items, st)
    d = banded(rows * items)
    _lib.call("lego_token_logprobs_bwd", p(logits), items, 0, None, 0, p(t), 1, k, row[2][1], row[1][1], row[4][1], row[0][1], row[1][1], row[3][1], d[1], rows,
              items, st)
    torch.cuda.synchronize()
    for b, _ in [(h, 0), (last, 0), (tiles, 0), (ws, 0), (ws2, 0), (ws3, 0), y, nx, stat, d] + outs + more + row:
        assert bool((b[:guard] == 7).all()) and bool((b[-guard:] == 7).all())
