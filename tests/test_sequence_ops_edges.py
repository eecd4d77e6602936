"""The sequence operators at the ends of their ranges: saturated and overflowing gates, operands that a mode has no use for, very many rows, the forms that cut
sequences and rows, against the plain 64-bit forms of test_sequence_ops.py and with its tolerances."""
import math

import pytest
import torch

from legommenders_amd import _lib, functional as F
from legommenders_amd import kernels as K
from legommenders_amd._lib import LegoHipError
from tests.test_sequence_ops import SCAN_CELL, SCAN_STEP, TYPES, _lam, _memory, _rand, check, logprobs_64, scan_64


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("side", [1, -1, 0])
def test_gradients_of_saturated_gates(side, dtype):
    """1 - sigmoid(v) = e^-v sigmoid(v) has its bits for large v too, where 1 minus a rounded sigmoid has lost them (0.9 % at 12, all from 17 on)"""
    n, length, width = 2, 70, 24
    g = torch.Generator().manual_seed(5)
    r, i = ((8 + 17 * torch.rand(n, length, width, generator=g)) for _ in range(2))
    if side <= 0:
        r = torch.where(torch.rand(r.shape, generator=g) < (0.5 if side == 0 else 1.0), -r, r)
        i = torch.where(torch.rand(i.shape, generator=g) < (0.5 if side == 0 else 1.0), -i, i)
    x, r, i = (t.to(dtype) for t in (_rand(1, n, length, width), r, i))
    lam, st, gh, gl = _lam(width, lo=0.9, hi=0.999), _rand(2, n, width), _rand(3, n, length, width, dtype=dtype), _rand(4, n, width)
    want = scan_64(x, r, i, lam, None, st, 8.0, gh, gl)
    for name, v in (("dr", r.double()), ("di", i.double())):                                 # that form's 1 - sigmoid loses bits in 64 bits as well
        want[name] = tuple(t * torch.sigmoid(-v) / (1 - torch.sigmoid(v)) for t in want[name])
    leaves = [t.cuda().requires_grad_() for t in (x, r, i, lam, st)]
    h, last = F.gated_scan(*leaves[:4], state=leaves[4])
    grads = torch.autograd.grad((h, last), leaves, (gh.cuda(), gl.cuda()))
    many = SCAN_STEP * _memory(length) + SCAN_CELL + 2 * 25                                  # the exponentials' arguments are up to 25 in size: a rounding each
    # closed gates: sqrt(2 k) 2^-63 for each step where sigmoid(r) would be below 2^-126 -- none here (r >= -25)
    for got, name in zip((h, last, *grads), ("h", "last", "dx", "dr", "di", "dlam", "dstate")):
        check(got, *want[name], 2 * many + (n * length if name == "dlam" else 0))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["lam", "sharpness"])
@pytest.mark.parametrize("length", [5, 64, 300])
def test_decays_that_overflow(kind, length):
    """a rate beyond fp32 (lam infinite, or a huge sharpness): a live step forgets the state, a masked one and the places behind the sequence keep it"""
    n, width = 3, 24
    x, r, i, st, gh, gl = _rand(1, n, length, width), _rand(2, n, length, width), _rand(3, n, length, width), 1e3 * _rand(4, n, width), _rand(5, n, length, width), _rand(6, n, width)
    m = torch.rand(n, length, generator=torch.Generator().manual_seed(7)) < 0.5
    m[1] = False
    lam = _lam(width)
    lam[::3] = math.inf if kind == "lam" else 3.0                                            # 3e38 softplus(3) is beyond fp32, 3e38 softplus(the others) is not
    far = torch.where(torch.isinf(lam), 1e4, lam)                                            # there a is 0 in 64 bits too, and every term is finite
    want = scan_64(x, r, i, far, m, st, 8.0, gh, gl) if kind == "lam" else scan_64(x, r, i, torch.full((width,), 1e4), m, st, 8.0, gh, gl)
    leaves = [t.cuda().requires_grad_() for t in (x, r, i, lam, st)]
    h, last = F.gated_scan(*leaves[:4], mask=m.cuda(), state=leaves[4], sharpness=8.0 if kind == "lam" else 3e38)
    grads = torch.autograd.grad((h, last), leaves, (gh.cuda(), gl.cuda()))
    many = SCAN_STEP * _memory(length) + SCAN_CELL
    for got, name in zip((h, last, *grads), ("h", "last", "dx", "dr", "di", "dlam", "dstate")):
        check(got, *want[name], 2 * many + (n * length if name == "dlam" else 0))


@pytest.fixture
def filled():
    """fresh memory is full of NaN"""
    torch.use_deterministic_algorithms(True)
    yield
    torch.use_deterministic_algorithms(False)


UNUSED = [dict(o=1, post_w=1, scale=1, next_w=1, gate=1), dict(o=1, post_w=1, scale=1, gate=1), dict(next_w=1, gate=1), dict(next_w=1, post_w=1), dict(next_w=1, scale=1)]


@pytest.mark.parametrize("given", UNUSED)
def test_nothing_uninitialised_comes_back_for_what_a_norm_does_not_use(given, filled, monkeypatch):
    """the kernels write no gradient of a gate without an activation, or of a block's operands without a block: the registered op's are zeros"""
    wrote = []
    monkeypatch.setattr(K, "_agree", lambda *a, **k: None)
    monkeypatch.setattr(K, "_launch", lambda t, name, *a: wrote.append(name))
    x, w = torch.ones(3, 8), torch.ones(8)
    o, gate = (x if given.get(k) else None for k in ("o", "gate"))
    pw, sc, nw = (w if given.get(k) else None for k in ("post_w", "scale", "next_w"))
    out = K.block_norm_bwd(x, x if nw is not None else None, x, o, gate, pw, sc, nw, 1e-6, 0, torch.ones(2, 3))
    assert wrote == ["lego_block_norm_bwd"]
    for name, t in zip(("gate", "post_w", "scale"), (out[2], out[3], out[4])):
        used = name != "gate" and o is not None
        assert t is None or used or bool((t == 0).all()), name


@pytest.mark.gpu
@pytest.mark.parametrize("given", UNUSED)
def test_operands_that_a_norm_does_not_use(given, filled):
    block_norm = torch.ops.lego_hip.block_norm
    names = ("o", "gate", "post_w", "scale", "next_w")
    x = _rand(1, 5, 12).cuda().requires_grad_()
    ops = [None if not given.get(k) else _rand(2 + q, *((5, 12) if q < 2 else (12,))).cuda().requires_grad_() for q, k in enumerate(names)]
    used = [t if given.get("o") or k == "next_w" else None for k, t in zip(names, ops)]
    used[1] = None
    grads = []
    for a in (ops, used):
        out = [t for t in block_norm(x, *a, 1e-6, 0, True)[:2] if t.numel()]
        there = [x] + [t for t in ops if t is not None]
        grads.append(torch.autograd.grad(out, there, [torch.ones_like(t) for t in out], allow_unused=True))
    for got, want in zip(*grads):
        assert torch.equal(got, torch.zeros_like(got) if want is None else want)


@pytest.mark.gpu
def test_more_rows_than_a_launch_has_workgroups():
    """2^24 rows of a workgroup of 256 lanes each are 2^32 lanes, one more than a launch takes"""
    rows, items, k = (1 << 24) + 5, 3, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, items, generator=g, device="cuda").half().requires_grad_()
    t = torch.randint(-1, items, (rows,), generator=g, device="cuda").int()
    m = torch.rand(rows, items, generator=g, device="cuda") < 0.9
    m[:, 1] = True
    logp, entropy, top, index = F.token_logprobs(x, t, k=k, mask=m)
    gl, ge, gt = torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, k, generator=g, device="cuda")
    dx, = torch.autograd.grad((logp, entropy, top), x, (gl, ge, gt))
    for a in range(0, rows, 1 << 22):                                                        # each row against a call of its own part, and both sides of the border
        s = slice(a, min(a + (1 << 22), rows))
        p = x.detach()[s].requires_grad_()
        part = F.token_logprobs(p, t[s], k=k, mask=m[s])
        assert all(torch.equal(u[s], v) for u, v in zip((logp, entropy, top, index), part))
        assert torch.equal(dx[s], torch.autograd.grad(part[:3], p, (gl[s], ge[s], gt[s]))[0])
    w = logprobs_64(x.detach()[-7:].cpu(), t[-7:].cpu().long(), k, m[-7:].cpu())
    for got, name in ((logp, "logp"), (entropy, "entropy"), (top, "top")):
        check(got[-7:], w[name], 20.0, 100)
    assert torch.equal(index[-7:].cpu().long(), w["index"])


class _Bands:
    """tensors inside larger buffers: what surrounds an input is NaN (all bits set, where whole numbers are), what surrounds an output has to stay"""

    def __init__(self, guard=256):
        self.guard, self.outs = guard, []

    def input(self, t):
        t = t.contiguous()
        fill = math.nan if t.dtype.is_floating_point else (255 if t.dtype == torch.uint8 else -1)
        buf = torch.full((t.numel() + 2 * self.guard,), fill, dtype=t.dtype, device="cuda")
        inside = buf[self.guard:self.guard + t.numel()].view(t.shape)
        inside.copy_(t)
        return inside

    def output(self, *shape, dtype=torch.float32):
        count = math.prod(shape)
        buf = torch.full((count + 2 * self.guard,), 7, dtype=dtype, device="cuda")
        self.outs.append(buf)
        return buf[self.guard:self.guard + count].view(shape)

    def check(self):
        torch.cuda.synchronize()
        assert all(bool((b[:self.guard] == 7).all()) and bool((b[-self.guard:] == 7).all()) for b in self.outs)


DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,masked", [((1, 1030, 33), False), ((1, 10007, 301), False), ((2, 4096, 64), True), ((3, 705, 1), True), ((190, 1280, 24), False), ((52, 193, 2561), True)])
def test_cut_scans_stay_inside_their_buffers(shape, masked, dtype):
    n, length, width = shape
    b, p, st = _Bands(), K._ptr, K._stream()
    x, r, i, gh = (b.input(_rand(q, n, length, width, dtype=dtype)) for q in range(4))
    lam, state, glast = b.input(_lam(width)), b.input(_rand(5, n, width)), b.input(_rand(6, n, width))
    m = None
    if masked:
        m = (torch.rand(n, length, generator=torch.Generator().manual_seed(1)) < 0.7).to(torch.uint8)
        m[0, : length // 2] = 0
        m = b.input(m)
    want = F.gated_scan(*(t.clone() for t in (x, r, i, lam)), mask=None if m is None else m.clone(), state=state.clone())
    h, last, tiles = b.output(n, length, width, dtype=dtype), b.output(n, width), b.output(n, -(-length // 64), width)
    size = _lib.lib().lego_gated_scan_workspace(n, length, width)
    ws = b.output(size)
    s, ms = (length * width, width), 0 if m is None else length
    _lib.call("lego_gated_scan_fwd", p(x), *s, p(r), *s, p(i), *s, DT[dtype], p(lam), 8.0, p(m), ms, p(state), p(h), p(last), p(tiles), p(ws), size, n, length, width, st)
    assert torch.equal(h, want[0]) and torch.equal(last, want[1])
    d = [b.output(n, length, width, dtype=dtype) for _ in range(3)] + [b.output(width), b.output(n, width)]
    ws.fill_(math.nan)                                                                       # (nothing in it is taken over)
    _lib.call("lego_gated_scan_bwd", p(x), *s, p(r), *s, p(i), *s, p(gh), *s, DT[dtype], p(lam), 8.0, p(m), ms, p(tiles.clone()), p(glast), *(p(t) for t in d), p(ws), size,
              n, length, width, st)
    leaves = [t.clone().requires_grad_() for t in (x, r, i, lam, state)]
    out = F.gated_scan(*leaves[:4], mask=None if m is None else m.clone(), state=leaves[4])
    for got, g in zip(d, torch.autograd.grad(out, leaves, (gh.clone(), glast.clone()))):
        assert torch.equal(got, g) and bool(torch.isfinite(got).all())
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,k,masked", [((1, 400001), 20, False), ((1, 400001), 128, True), ((5, 65238), 50, True), ((3, 131075), 0, False), ((300, 16411), 7, True), ((600, 65239), 10, False)])
def test_cut_rows_stay_inside_their_buffers(shape, k, masked, dtype):
    rows, items = shape
    b, p, st = _Bands(), K._ptr, K._stream()
    g = torch.Generator(device="cuda").manual_seed(2)
    x = b.input(torch.randn(rows, items, generator=g, device="cuda").to(dtype))
    t = b.input(torch.randint(-1, items, (rows,), generator=g, device="cuda"))
    m = b.input((torch.rand(rows, items, generator=g, device="cuda") < 0.7).to(torch.uint8)) if masked else None
    gl, ge, gt = (b.input(torch.randn(*s, generator=g, device="cuda")) for s in ((rows,), (rows,), (rows, k)))
    leaf = x.clone().requires_grad_()
    want = F.token_logprobs(leaf, t.clone(), k=k, mask=None if m is None else m.clone())
    logp, entropy, stat, top, index = b.output(rows), b.output(rows), b.output(rows, 2), b.output(rows, k), b.output(rows, k, dtype=torch.int32)
    size = _lib.lib().lego_token_logprobs_workspace(rows, items, DT[dtype], k)
    ws = b.output(max(size, 2), dtype=torch.int64)
    ms = 0 if m is None else items
    _lib.call("lego_token_logprobs_fwd", p(x), items, DT[dtype], p(m), ms, p(t), 1, k, p(logp), p(entropy), p(stat), p(top), p(index), p(ws), size, rows, items, st)
    assert all(torch.equal(u, v) for u, v in zip((logp, entropy, top, index), want))
    assert not bool(torch.isnan(logp).any()) and bool(torch.isfinite(entropy).all())             # (a masked target's logp is -inf)
    d = b.output(rows, items, dtype=dtype)
    _lib.call("lego_token_logprobs_bwd", p(x), items, DT[dtype], p(m), ms, p(t), 1, k, p(stat), p(entropy), p(index), p(gl), p(ge), p(gt) if k else None, p(d), rows, items, st)
    assert torch.equal(d, torch.autograd.grad(want[:3] if k else want[:2], leaf, (gl, ge, gt)[:3 if k else 2])[0]) and bool(torch.isfinite(d).all())
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(9, 1), (130, 33), (2049, 257), (7, 1025), (5, 2051), (5, 4099), (3, 5120), (3, 8193), (2, 16384), (600, 4100)])
def test_norms_stay_inside_their_buffers(rows, width, dtype):
    b, p, st = _Bands(), K._ptr, K._stream()
    x, o, g, gy, gn = (b.input(_rand(q, rows, width, dtype=dtype)) for q in range(5))
    pw, sc, nw = (b.input(_rand(5 + q, width)) for q in range(3))
    leaves = [t.clone().requires_grad_() for t in (x, o, g, pw, sc, nw)]
    want = F.gated_residual_norm(*leaves, act="silu")
    y, n, stat = b.output(rows, width, dtype=dtype), b.output(rows, width, dtype=dtype), b.output(2, rows)
    _lib.call("lego_block_norm_fwd", p(x), width, p(o), width, p(g), width, DT[dtype], 2, p(pw), p(sc), p(nw), 1e-6, p(y), p(n), p(stat), rows, width, st)
    assert torch.equal(y, want[0]) and torch.equal(n, want[1])
    d = [b.output(rows, width, dtype=dtype) for _ in range(3)] + [b.output(width) for _ in range(3)]
    size = _lib.lib().lego_block_norm_workspace(rows, width)
    ws = b.output(size)
    _lib.call("lego_block_norm_bwd", p(x), width, p(o), width, p(g), width, DT[dtype], 2, p(pw), p(sc), p(nw), 1e-6, p(gy), width, p(gn), width, p(stat), *(p(t) for t in d),
              p(ws), size, rows, width, st)
    for got, w in zip(d, torch.autograd.grad(want, leaves, (gy.clone(), gn.clone()))):
        assert torch.equal(got, w) and bool(torch.isfinite(got).all())
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,items", [(520, 65536), (513, 70001)])
@pytest.mark.parametrize("kind", ["plain", "rounded", "constant", "lowest", "two"])
def test_the_largest_of_uncut_rows_of_1024_lanes(kind, rows, items, dtype):
    """k up to 16 (64 groups of lanes) and above (256), rows in which more elements are equal than the list of candidates holds"""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(rows, items, generator=g, device="cuda")
    x = dict(plain=x, rounded=x.round(), constant=torch.full_like(x, -0.5), lowest=torch.where(x > 3, x, torch.finfo(dtype).min), two=(x > 0).float())[kind].to(dtype)
    order = torch.sort(x.float(), dim=1, descending=True, stable=True)
    lp = torch.log_softmax(x.double(), 1)
    for k in (1, 10, 16, 17, 65, 128):
        logp, entropy, top, index = F.token_logprobs(x, order.indices[:, 0], k=k)
        assert torch.equal(index.long(), order.indices[:, :k])
        want = lp.gather(1, order.indices[:, :k]).cpu()
        finite = x.double().masked_fill(x == torch.finfo(dtype).min, 0).abs().amax(1).cpu() + 12.0
        some = want > -1e30                                                                  # (behind a row's large elements come the lowest ones)
        check(torch.where(some.cuda(), top, 0.0), torch.where(some, want, 0.0), finite[:, None], items / 256 + 40)
        check(logp, lp.gather(1, order.indices[:, :1])[:, 0].cpu(), finite, items / 256 + 40)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 8), (2, 0, 8), (0, 3, 5)])
@pytest.mark.parametrize("next_norm", [False, True])
@pytest.mark.parametrize("grad", [False, True])
def test_tails_of_no_rows(shape, next_norm, grad):
    x, o, g = (torch.zeros(shape, device="cuda", requires_grad=grad) for _ in range(3))
    w = torch.ones(shape[-1], device="cuda", requires_grad=grad)
    y, n = F.gated_residual_norm(x, o, g, w, w, w if next_norm else None)
    assert y.shape == shape and (n.shape == shape if next_norm else n is None)
    if grad:
        dx, dw = torch.autograd.grad(y.sum() + (n.sum() if next_norm else 0), (x, w))
        assert dx.shape == shape and bool((dw == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("length", [1, 70, 300])
def test_decays_of_one(length):
    """softplus(-inf) is 0: the channel keeps its state for ever, takes nothing in, and has no gradient but the state's"""
    n, width = 2, 24
    x, r, i, st, gh, gl = _rand(1, n, length, width), _rand(2, n, length, width), _rand(3, n, length, width), _rand(4, n, width), _rand(5, n, length, width), _rand(6, n, width)
    lam = _lam(width)
    lam[::4] = -math.inf
    want = scan_64(x, r, i, lam, None, st, 8.0, gh, gl)
    dlam, terms = want["dlam"]                                                               # (that form's sigmoid / softplus is 0 / 0 there)
    want["dlam"] = tuple(torch.where(torch.isinf(lam), 0.0, t) for t in (dlam, terms))
    leaves = [t.cuda().requires_grad_() for t in (x, r, i, lam, st)]
    h, last = F.gated_scan(*leaves[:4], state=leaves[4])
    grads = torch.autograd.grad((h, last), leaves, (gh.cuda(), gl.cuda()))
    many = SCAN_STEP * _memory(length) + SCAN_CELL
    for got, name in zip((h, last, *grads), ("h", "last", "dx", "dr", "di", "dlam", "dstate")):
        check(got, *want[name], 2 * many + (n * length if name == "dlam" else 0))
    assert torch.equal(last.cpu()[:, ::4], st[:, ::4])
    h1, new = F.gated_scan_step(*(t.detach()[:, 0] for t in leaves[:3]), leaves[3].detach(), leaves[4].detach())
    assert torch.equal(new.cpu()[:, ::4], st[:, ::4]) and bool(torch.isfinite(new).all())


@pytest.mark.parametrize("sharpness", [1e39, 1e300, 1e-300, math.inf, math.nan, 0.0, -8.0])
def test_a_sharpness_that_fp32_does_not_hold_is_refused(sharpness):
    """the kernels take it in 32 bits: beyond them it would be infinite there, and 0 below"""
    x, lam, st = torch.zeros(2, 5, 8), torch.zeros(8), torch.zeros(2, 8)
    with pytest.raises(LegoHipError, match="sharpness"):
        F.gated_scan(x, x, x, lam, sharpness=sharpness)
    with pytest.raises(LegoHipError, match="sharpness"):
        F.gated_scan_step(st, st, st, lam, st, sharpness=sharpness)
