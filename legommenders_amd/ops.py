"""`torch.ops.lego_hip.*`: the HIP kernels of liblego_hip.so registered with the PyTorch dispatcher as custom ops
(SURVEY.md section 8b "Native/FFI layer"; north star: "hand-written CDNA4 HIP kernels registered as PyTorch-ROCm
custom ops").

Every forward op has a CUDA (= ROCm) implementation only -- a CPU tensor finds no kernel and raises, there is no
fallback -- a fake (meta) implementation so that `torch.compile` / `make_fx` / `torch.library.opcheck` can trace it, and
an autograd formula whose backward is itself built from registered ops (`*_bwd`), so the backward traces too.
Randomness is explicit: a dropout op takes `(p, seed, site)` and draws its keep bits from that Philox stream, forward
and backward alike; nothing reads hidden state.  The plug-in classes (`model/operators/*`, `model/predictors/*`,
`loader/embedding_hub`) reach the kernels through `legommenders_amd.functional`, which calls these ops; the fused
ragged engines (`engine.py`) stay the training fast path and call the same C ABI directly.

Reference call sites each op replaces are cited on the op.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.library import custom_op, register_autograd, register_fake

from . import kernels as K
from ._lib import LegoHipError, call

NS = "lego_hip"


def _drop(p: float, seed: int, site: int):
    return (float(p), int(seed), int(site)) if p > 0.0 else None


def _f(t: torch.Tensor) -> torch.Tensor:
    return t.detach().to(torch.float32).contiguous()


def _cuda(name, **kw):
    return custom_op(f"{NS}::{name}", mutates_args=kw.pop("mutates_args", ()), device_types="cuda", **kw)


# =============================================================================== embedding look-ups (a4)
@_cuda("gather_rows")
def gather_rows(table: torch.Tensor, idx: torch.Tensor) -> torch.Tensor:
    """out[r,:] = table[idx[r],:], idx < 0 -> zero row (nn.Embedding look-up behind the inputers' pad handling,
    loader/embedding_hub.py:73-96; the coalesced HBM row gather of the hot path)"""
    return K.gather_rows(_f(table), idx.to(torch.int32).contiguous())


@register_fake(f"{NS}::gather_rows")
def _(table, idx):
    return table.new_empty(idx.numel(), table.shape[1], dtype=torch.float32)


@_cuda("scatter_add_rows")
def scatter_add_rows(g: torch.Tensor, idx: torch.Tensor, rows: int) -> torch.Tensor:
    """dense [rows, W] gradient of gather_rows (embedding_hub.py:325-335: nn.Embedding's dense gradient)"""
    out = torch.zeros(rows, g.shape[1], dtype=torch.float32, device=g.device)
    return K.scatter_add_rows(out, idx.to(torch.int32).contiguous(), _f(g))


@register_fake(f"{NS}::scatter_add_rows")
def _(g, idx, rows):
    return g.new_empty(rows, g.shape[1], dtype=torch.float32)


def _gather_setup(ctx, inputs, output):
    table, idx = inputs
    ctx.save_for_backward(idx)
    ctx.rows = table.shape[0]


def _gather_bwd(ctx, g):
    (idx,) = ctx.saved_tensors
    return torch.ops.lego_hip.scatter_add_rows(g.contiguous(), idx, ctx.rows), None


register_autograd(f"{NS}::gather_rows", _gather_bwd, setup_context=_gather_setup)


# =============================================================================== nn.Linear (a4 / a5 / a8)
@_cuda("linear")
def linear(x: torch.Tensor, W: torch.Tensor, b: Optional[torch.Tensor]) -> torch.Tensor:
    """y = x W^T + b on the fp32 MFMA kernels (x: [M,K], W: [N,K]; nn.Linear of cnn_operator.py:58-60,
    attention_operator.py:52, embedding_hub.py:95)"""
    return K.linear_fwd(_f(x), _f(W), None if b is None else _f(b), act=0)


@register_fake(f"{NS}::linear")
def _(x, W, b):
    return x.new_empty(x.shape[0], W.shape[0], dtype=torch.float32)


@_cuda("linear_bwd")
def linear_bwd(g: torch.Tensor, x: torch.Tensor, W: torch.Tensor, has_bias: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    g, x, W = _f(g), _f(x), _f(W)
    gW = torch.zeros_like(W)
    K.linear_bwd_weight(g, x, gW)
    gb = torch.zeros(W.shape[0], dtype=torch.float32, device=W.device)
    if has_bias:
        K.colsum(g, gb)
    return K.linear_bwd_data(g, W), gW, gb


@register_fake(f"{NS}::linear_bwd")
def _(g, x, W, has_bias):
    return torch.empty_like(x, dtype=torch.float32), torch.empty_like(W, dtype=torch.float32), W.new_empty(W.shape[0], dtype=torch.float32)


def _linear_setup(ctx, inputs, output):
    x, W, b = inputs
    ctx.save_for_backward(x, W)
    ctx.has_b = b is not None


def _linear_bwd(ctx, g):
    x, W = ctx.saved_tensors
    gx, gW, gb = torch.ops.lego_hip.linear_bwd(g.contiguous(), x, W, ctx.has_b)
    return gx, gW, (gb if ctx.has_b else None)


register_autograd(f"{NS}::linear", _linear_bwd, setup_context=_linear_setup)


# =============================================================================== frozen table -> projection (a3 / a4)
@_cuda("glove_project")
def glove_project(ids: torch.Tensor, table: torch.Tensor, W: torch.Tensor, b: torch.Tensor, p: float, seed: int,
                  site: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Transformation.forward + SimpleInputer masking: Dropout(Linear(Embedding(ids))) * (ids >= 0)
    (loader/embedding_hub.py:95-96, model/inputer/simple_inputer.py:55-63); ids flat [R], table frozen.
    Returns (H [R,D], X [R,E0] the gathered rows, kept for the weight gradient)."""
    flat = ids.to(torch.int32).contiguous()
    X = K.gather_rows(_f(table), flat)
    rowinfo = torch.where(flat >= 0, torch.full_like(flat, 4), torch.zeros_like(flat))
    H = K.linear_fwd(X, _f(W), _f(b), act=0, rowinfo=rowinfo, drop=_drop(p, seed, site))
    return H, X


@register_fake(f"{NS}::glove_project")
def _(ids, table, W, b, p, seed, site):
    return W.new_empty(ids.numel(), W.shape[0], dtype=torch.float32), W.new_empty(ids.numel(), table.shape[1], dtype=torch.float32)


@_cuda("glove_project_bwd")
def glove_project_bwd(gH: torch.Tensor, X: torch.Tensor, ids: torch.Tensor, W: torch.Tensor, p: float, seed: int,
                      site: int) -> Tuple[torch.Tensor, torch.Tensor]:
    D = W.shape[0]
    flat = ids.to(torch.int32).contiguous()
    rowinfo = torch.where(flat >= 0, torch.full_like(flat, 4), torch.zeros_like(flat))
    g = _f(gH).clone()
    call("lego_mask_dropout_rows", K._ptr(g), D, g.shape[0], None, D, K._ptr(rowinfo), K._drop(_drop(p, seed, site)), None, K._stream())
    gW = torch.zeros(W.shape, dtype=torch.float32, device=W.device)
    K.linear_bwd_weight(g, _f(X), gW)
    gb = torch.zeros(D, dtype=torch.float32, device=W.device)
    K.colsum(g, gb)
    return gW, gb


@register_fake(f"{NS}::glove_project_bwd")
def _(gH, X, ids, W, p, seed, site):
    return torch.empty_like(W, dtype=torch.float32), W.new_empty(W.shape[0], dtype=torch.float32)


@_cuda("glove_project_bwd_table")
def glove_project_bwd_table(gH: torch.Tensor, ids: torch.Tensor, W: torch.Tensor, rows: int, p: float, seed: int, site: int) -> torch.Tensor:
    """gradient of an UN-FROZEN pre-trained table under Transformation (`load_pretrained_embedding(..., frozen=False)`,
    loader/embedding_hub.py:171,262: nn.Embedding.from_pretrained with requires_grad switched on): the mask + Dropout backward of
    gH (the same Philox bits as the forward), dX = g W, rows added to the DENSE [rows, E0] gradient the reference's autograd
    produces (pad ids -1 contribute nothing: the reference's masked positions look up row 0 and are zeroed after the projection)"""
    D = W.shape[0]
    flat = ids.to(torch.int32).contiguous()
    rowinfo = torch.where(flat >= 0, torch.full_like(flat, 4), torch.zeros_like(flat))
    g = _f(gH).clone()
    call("lego_mask_dropout_rows", K._ptr(g), D, g.shape[0], None, D, K._ptr(rowinfo), K._drop(_drop(p, seed, site)), None, K._stream())
    gX = K.linear_bwd_data(g, _f(W))
    gT = torch.zeros(rows, W.shape[1], dtype=torch.float32, device=W.device)
    return K.scatter_add_rows(gT, flat, gX)


@register_fake(f"{NS}::glove_project_bwd_table")
def _(gH, ids, W, rows, p, seed, site):
    return W.new_empty(rows, W.shape[1], dtype=torch.float32)


def _gp_setup(ctx, inputs, output):
    ids, table, W, b, p, seed, site = inputs
    ctx.save_for_backward(output[1], ids, W)
    ctx.rng = (p, seed, site)
    ctx.table_rows = table.shape[0]


def _gp_bwd(ctx, gH, gX):
    X, ids, W = ctx.saved_tensors
    gW, gb = torch.ops.lego_hip.glove_project_bwd(gH.contiguous(), X, ids, W, *ctx.rng)
    gT = None
    if ctx.needs_input_grad[1]:                  # un-frozen pre-trained table
        gT = torch.ops.lego_hip.glove_project_bwd_table(gH.contiguous(), ids, W, ctx.table_rows, *ctx.rng)
    return None, gT, gW, gb, None, None, None


register_autograd(f"{NS}::glove_project", _gp_bwd, setup_context=_gp_setup)


# =============================================================================== CNNOperator title branch (a5)
@_cuda("conv3_relu_mask")
def conv3_relu_mask(h: torch.Tensor, mask: torch.Tensor, w: torch.Tensor, b: torch.Tensor, p: float, seed: int,
                    site: int) -> torch.Tensor:
    """Conv1d(k=3, 'same') -> ReLU -> * mask -> Dropout on [n,L,Din] (model/operators/cnn_operator.py:54-57)"""
    n, L, Din = h.shape
    plan = K.plan_dense(mask)
    y = K.conv3_fwd(_f(h).view(n * L, Din), K.conv3_pack(w), b, plan, drop=_drop(p, seed, site))
    return y.view(n, L, w.shape[0])


@register_fake(f"{NS}::conv3_relu_mask")
def _(h, mask, w, b, p, seed, site):
    return h.new_empty(h.shape[0], h.shape[1], w.shape[0], dtype=torch.float32)


@_cuda("conv3_relu_mask_bwd")
def conv3_relu_mask_bwd(gy: torch.Tensor, h: torch.Tensor, y: torch.Tensor, mask: torch.Tensor, w: torch.Tensor,
                        p: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    n, L, Din = h.shape
    Dout = w.shape[0]
    plan = K.plan_dense(mask)
    wt = K.conv3_pack(w)
    g = _f(gy).reshape(n * L, Dout).clone()
    scale = 1.0 / (1.0 - p) if p > 0.0 else 1.0          # y > 0 <=> kept and pre-activation > 0: the mask is in y itself
    y2 = _f(y).view(n * L, Dout)
    call("lego_relu_bwd", K._ptr(g), Dout, K._ptr(y2), Dout, n * L, Dout, float(scale), K._stream())
    gb = torch.zeros(Dout, dtype=torch.float32, device=g.device)
    K.colsum(g, gb)
    dwt = torch.zeros(3, Dout, Din, dtype=torch.float32, device=g.device)
    K.conv3_bwd_weight(g, _f(h).view(n * L, Din), plan, dwt)
    gw = torch.zeros(w.shape, dtype=torch.float32, device=g.device)
    K.conv3_unpack_add(dwt, gw)
    # d h: rows are NOT re-masked here (the live factor belongs to the producer of h)
    gh = K.conv3_bwd_data(g, wt, K.DensePlan(None, n, L, g.device), Din)
    return gh.view(n, L, Din), gw, gb


@register_fake(f"{NS}::conv3_relu_mask_bwd")
def _(gy, h, y, mask, w, p):
    return torch.empty_like(h, dtype=torch.float32), torch.empty_like(w, dtype=torch.float32), w.new_empty(w.shape[0], dtype=torch.float32)


def _conv_setup(ctx, inputs, output):
    h, mask, w, b, p, seed, site = inputs
    ctx.save_for_backward(h, output, mask, w)
    ctx.p = p


def _conv_bwd(ctx, gy):
    h, y, mask, w = ctx.saved_tensors
    gh, gw, gb = torch.ops.lego_hip.conv3_relu_mask_bwd(gy.contiguous(), h, y, mask, w, ctx.p)
    return gh, None, gw, gb, None, None, None


register_autograd(f"{NS}::conv3_relu_mask", _conv_bwd, setup_context=_conv_setup)


# =============================================================================== AdditiveAttention (a6 / a7)
@_cuda("additive_pool")
def additive_pool(x: torch.Tensor, mask: torch.Tensor, W1: torch.Tensor, b1: torch.Tensor,
                  w2: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """AdditiveAttention.forward on [n,L,D] + mask [n,L] (model/common/attention.py:31-38): tanh hidden on the MFMA
    kernel, LDS-staged pool with wavefront-shuffle softmax reductions.  Returns (out [n,D], tanh hidden [n*L,A],
    attention weights [n*L]) -- the last two are what the backward needs."""
    out, c = K.additive_attention_fwd(x, mask, W1, b1, w2)
    return out, c.t, c.wrow


@register_fake(f"{NS}::additive_pool")
def _(x, mask, W1, b1, w2):
    n, L, D = x.shape
    return x.new_empty(n, D, dtype=torch.float32), x.new_empty(n * L, W1.shape[0], dtype=torch.float32), x.new_empty(n * L, dtype=torch.float32)


@_cuda("additive_pool_bwd")
def additive_pool_bwd(gout: torch.Tensor, x: torch.Tensor, mask: torch.Tensor, W1: torch.Tensor, w2: torch.Tensor,
                      t: torch.Tensor, wrow: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    n, L, D = x.shape
    c = K._AddCtx()
    c.x, c.t, c.wrow, c.plan = _f(x).view(n * L, D), t.clone(), wrow, K.plan_dense(mask)     # the pool backward overwrites t
    c.W1, c.w2, c.shape = _f(W1), _f(w2).view(-1), (n, L, D, W1.shape[0])
    gx, gW1, gb1, gw2 = K.additive_attention_bwd(c, _f(gout))
    return gx, gW1, gb1, gw2


@register_fake(f"{NS}::additive_pool_bwd")
def _(gout, x, mask, W1, w2, t, wrow):
    A = W1.shape[0]
    return (torch.empty_like(x, dtype=torch.float32), torch.empty_like(W1, dtype=torch.float32), W1.new_empty(A, dtype=torch.float32),
            W1.new_empty(1, A, dtype=torch.float32))


def _add_setup(ctx, inputs, output):
    x, mask, W1, b1, w2 = inputs
    ctx.save_for_backward(x, mask, W1, w2, output[1], output[2])
    ctx.w2_shape = w2.shape


def _add_bwd(ctx, gout, gt, gw):
    x, mask, W1, w2, t, wrow = ctx.saved_tensors
    gx, gW1, gb1, gw2 = torch.ops.lego_hip.additive_pool_bwd(gout.contiguous(), x, mask, W1, w2, t, wrow)
    return gx, None, gW1, gb1, gw2.view(ctx.w2_shape)


register_autograd(f"{NS}::additive_pool", _add_bwd, setup_context=_add_setup)


# =============================================================================== nn.MultiheadAttention (a8)
@_cuda("mhsa")
def mhsa(x: torch.Tensor, mask: torch.Tensor, in_w: torch.Tensor, in_b: torch.Tensor, out_w: torch.Tensor,
         out_b: torch.Tensor, heads: int, p: float, seed: int, site: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """nn.MultiheadAttention(q=k=v=x, key_padding_mask=1-mask) (model/operators/attention_operator.py:46-50): MFMA in/out
    projections + the attention core.  Returns (y [n,L,D], compact x rows, qkv, head outputs, log-sum-exp of the score rows);
    the saved activations hold the R live rows first inside n*L-row buffers the kernels wrote in place, so every output shape
    is static and nothing is copied (the probabilities are not saved: the backward pass recomputes them)."""
    y, c = K.mhsa_fwd(x, mask, in_w, in_b, out_w, out_b, heads, drop=_drop(p, seed, site), padded=True)
    return (y,) + c.saved


@register_fake(f"{NS}::mhsa")
def _(x, mask, in_w, in_b, out_w, out_b, heads, p, seed, site):
    n, L, D = x.shape
    R = n * L
    f = dict(dtype=torch.float32)
    return (x.new_empty(n, L, D, **f), x.new_empty(R, D, **f), x.new_empty(R, 3 * D, **f), x.new_empty(R, D, **f),
            x.new_empty(R, heads, **f))


@_cuda("mhsa_bwd")
def mhsa_bwd(gy: torch.Tensor, mask: torch.Tensor, in_w: torch.Tensor, out_w: torch.Tensor, xc: torch.Tensor,
             qkv: torch.Tensor, o: torch.Tensor, lse: torch.Tensor, heads: int, p: float, seed: int,
             site: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    n, L, D = gy.shape
    c = K._MhsaCtx()
    c.idx, c.seg_off = K._compact(mask)
    R = c.idx.numel()
    c.xc, c.qkv, c.o, c.lse = xc[:R], qkv[:R], o[:R], lse[:R]
    c.in_w, c.out_w, c.heads, c.shape, c.drop = _f(in_w), _f(out_w), heads, (n, L, D), _drop(p, seed, site)
    return K.mhsa_bwd(c, _f(gy))


@register_fake(f"{NS}::mhsa_bwd")
def _(gy, mask, in_w, out_w, xc, qkv, o, lse, heads, p, seed, site):
    f = dict(dtype=torch.float32)
    D = gy.shape[2]
    return (torch.empty_like(gy, **f), torch.empty_like(in_w, **f), in_w.new_empty(3 * D, **f), torch.empty_like(out_w, **f),
            in_w.new_empty(D, **f))


def _mhsa_setup(ctx, inputs, output):
    x, mask, in_w, in_b, out_w, out_b, heads, p, seed, site = inputs
    ctx.save_for_backward(mask, in_w, out_w, *output[1:])
    ctx.args = (heads, p, seed, site)


def _mhsa_bwd(ctx, gy, *unused):
    mask, in_w, out_w, xc, qkv, o, lse = ctx.saved_tensors
    gx, gin_w, gin_b, gout_w, gout_b = torch.ops.lego_hip.mhsa_bwd(gy.contiguous(), mask, in_w, out_w, xc, qkv, o, lse, *ctx.args)
    return gx, None, gin_w, gin_b, gout_w, gout_b, None, None, None, None


register_autograd(f"{NS}::mhsa", _mhsa_bwd, setup_context=_mhsa_setup)


# =============================================================================== predictors / loss (a9 / a10)
@_cuda("rowdot")
def rowdot(u: torch.Tensor, it: torch.Tensor) -> torch.Tensor:
    """DotPredictor: sum(u * i, -1) on [n,D] pairs (model/predictors/dot_predictor.py:7-10)"""
    u2, i2 = _f(u), _f(it)
    n, D = u2.shape
    out = torch.empty(n, dtype=torch.float32, device=u.device)
    call("lego_rowdot_fwd", K._ptr(u2), D, K._ptr(i2), D, n, D, K._ptr(out), K._stream())
    return out


@register_fake(f"{NS}::rowdot")
def _(u, it):
    return u.new_empty(u.shape[0], dtype=torch.float32)


@_cuda("rowdot_bwd")
def rowdot_bwd(g: torch.Tensor, u: torch.Tensor, it: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    u2, i2, g2 = _f(u), _f(it), _f(g)
    n, D = u2.shape
    gu, gi = torch.empty_like(u2), torch.empty_like(i2)
    call("lego_rowdot_bwd", K._ptr(u2), D, K._ptr(i2), D, K._ptr(g2), n, D, K._ptr(gu), D, K._ptr(gi), D, K._stream())
    return gu, gi


@register_fake(f"{NS}::rowdot_bwd")
def _(g, u, it):
    return torch.empty_like(u, dtype=torch.float32), torch.empty_like(it, dtype=torch.float32)


register_autograd(f"{NS}::rowdot", lambda ctx, g: torch.ops.lego_hip.rowdot_bwd(g.contiguous(), *ctx.saved_tensors),
                  setup_context=lambda ctx, inputs, output: ctx.save_for_backward(*inputs))


@_cuda("dot_ce")
def dot_ce(user: torch.Tensor, items: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """batched user x candidate scoring + CrossEntropy(label 0): scores[b,c] = <user[b], items[b,c]>, loss = mean_b
    (model/legommender.py:254,263 with the Dot predictor).  Returns (loss [], scores [B,C])."""
    scores, loss = K.dot_ce_fwd(user, items)
    return loss.view(()), scores


@register_fake(f"{NS}::dot_ce")
def _(user, items):
    return user.new_empty((), dtype=torch.float32), user.new_empty(items.shape[0], items.shape[1], dtype=torch.float32)


@_cuda("dot_ce_bwd")
def dot_ce_bwd(gloss: torch.Tensor, user: torch.Tensor, items: torch.Tensor, scores: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    gu, gi = K.dot_ce_bwd(user, items, scores, gloss=1.0)
    s = gloss.to(torch.float32).reshape(())
    return gu * s, gi * s


@register_fake(f"{NS}::dot_ce_bwd")
def _(gloss, user, items, scores):
    return torch.empty_like(user, dtype=torch.float32), torch.empty_like(items, dtype=torch.float32)


def _dotce_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[0], inputs[1], output[1])
    ctx.set_materialize_grads(True)


def _dotce_bwd(ctx, gloss, gscores):
    user, items, scores = ctx.saved_tensors
    return torch.ops.lego_hip.dot_ce_bwd(gloss, user, items, scores)


register_autograd(f"{NS}::dot_ce", _dotce_bwd, setup_context=_dotce_setup)


# =============================================================================== optimiser / sampler (a11 / a13)
@_cuda("adam_step", mutates_args=("p", "g", "m", "v"))
def adam_step(p: torch.Tensor, g: torch.Tensor, m: torch.Tensor, v: torch.Tensor, lr: float, step: int, grad_scale: float,
              zero_grad: bool) -> None:
    """torch.optim.Adam defaults (base_lego.py:201-204) over one flat fp32 buffer, gradient scaled by grad_scale first
    (1/world after the all-reduce) and optionally cleared as it is consumed"""
    call("lego_adam_step", K._ptr(p), K._ptr(g), K._ptr(m), K._ptr(v), p.numel(), float(lr), 0.9, 0.999, 1e-8, int(step),
         float(grad_scale), 1 if zero_grad else 0, K._stream())


@_cuda("sample_negatives")
def sample_negatives(row_user: torch.Tensor, row_item: torch.Tensor, neg_list: torch.Tensor, neg_len: torch.Tensor, K_neg: int,
                     n_items: int, seed: int, step: int, row_base: int, row_stride: int) -> torch.Tensor:
    """Resampler.rebuild_candidates (loader/resampler.py:159-171) on device: [B, K+1] candidates, positive first"""
    B = row_user.numel()
    cand = torch.empty(B, K_neg + 1, dtype=torch.int32, device=row_user.device)
    call("lego_sample_negatives", K._ptr(row_user), K._ptr(row_item), K._ptr(neg_list), K._ptr(neg_len), neg_list.shape[1], B, K_neg,
         n_items, int(seed), int(step), int(row_base), int(row_stride), None, K._ptr(cand), K._stream())
    return cand


@register_fake(f"{NS}::sample_negatives")
def _(row_user, row_item, neg_list, neg_len, K_neg, n_items, seed, step, row_base, row_stride):
    return row_user.new_empty(row_user.numel(), K_neg + 1, dtype=torch.int32)


@_cuda("gather_history")
def gather_history(row_user: torch.Tensor, user_hist: torch.Tensor, user_hist_len: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """the DataSet row copy (loader/data_set.py:61-85): click history and its length of each row's user"""
    B, S = row_user.numel(), user_hist.shape[1]
    hist = torch.empty(B, S, dtype=torch.int32, device=row_user.device)
    hl = torch.empty(B, dtype=torch.int32, device=row_user.device)
    call("lego_gather_history", K._ptr(row_user), K._ptr(user_hist), K._ptr(user_hist_len), B, S, K._ptr(hist), K._ptr(hl), K._stream())
    return hist, hl


@register_fake(f"{NS}::gather_history")
def _(row_user, user_hist, user_hist_len):
    return row_user.new_empty(row_user.numel(), user_hist.shape[1], dtype=torch.int32), row_user.new_empty(row_user.numel(), dtype=torch.int32)


# =============================================================================== sequence operators
# A recurrent encoder of click histories, the norms around its blocks, next-item log probabilities.  No counterpart in the reference.  They keep
# the activations' type; an output that a call does not make is an empty tensor (an op's outputs are tensors).
#
# Registered through torch.library's definitions themselves, not custom_op: the autograd formula is a plain autograd.Function, which costs the host
# about half of what custom_op's generic one does (84 against 167 us for a forward and backward pass of three tensors, CPU-bound) -- these
# operators run for tens of microseconds.  `functional` enters at the Function (a gradient is wanted) or below the autograd key (it is not).
_LIB = torch.library.Library(NS, "FRAGMENT")
below_autograd = torch._C._AutoDispatchBelowAutograd


def _define(name, schema, impl, fake):
    _LIB.define(name + schema, tags=(torch.Tag.pt2_compliant_tag,))
    _LIB.impl(name, impl, "CUDA")
    register_fake(f"{NS}::{name}", fake, lib=_LIB)
    return getattr(torch.ops.lego_hip, name).default


def refuse_tangents(what, operands):
    """forward-mode derivatives: a dual operand need not require a gradient, and the kernels would answer as if it had no tangent"""
    if forward_ad._current_level >= 0:                       # (outside a dual level nothing is looked at)
        for t in operands:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise LegoHipError(f"{what}: no forward-mode derivative; reverse mode (backward, torch.autograd.grad) differentiates it")


def _differentiable(name, function, wants):
    """the Autograd entry of an op: `function` where one of its operands (those at the places `wants`) requires a gradient"""
    op = getattr(torch.ops.lego_hip, name).default

    def entry(*args):
        refuse_tangents(name, args)
        if torch.is_grad_enabled() and any(args[q] is not None and args[q].requires_grad for q in wants):
            return function.apply(*args)
        with below_autograd():
            return op(*args)
    _LIB.impl(name, entry, "Autograd")


def _not_differentiable(name):
    """the Autograd entry of an op that has no gradient: its outputs say so where a backward pass reaches them"""
    op = getattr(torch.ops.lego_hip, name).default

    class NoGradient(torch.autograd.Function):
        @staticmethod
        def forward(ctx, *args):
            with below_autograd():
                return op(*args)

        @staticmethod
        def backward(ctx, *grads):
            raise LegoHipError(f"lego_hip::{name} has no gradient")
    _differentiable(name, NoGradient, [q for q, a in enumerate(op._schema.arguments) if "Tensor" in str(a.type)])


def _once(what):
    if torch.is_grad_enabled():              # create_graph: what these backward passes return has no graph of its own
        raise RuntimeError(f"{what} is differentiable once (create_graph=True is not supported)")


def _or_empty(t, like, dtype=None):
    return like.new_empty(0, dtype=dtype or like.dtype) if t is None else t


# ---- gated_scan: h_t = a_t h_(t-1) + sqrt(1 - a_t^2) sigmoid(i_t) x_t, a_t = exp(-sharpness softplus(lam) sigmoid(r_t)), over [n, length, width]
# -> (h, the last state [n, width], the tiles' states -- empty unless `keep`: the backward pass starts from them)
def _scan_fake(x, r, i, lam, mask, state, sharpness, keep):
    n, length, width = x.shape
    f = dict(dtype=torch.float32)
    tiles = (length + K.SCAN_TILE - 1) // K.SCAN_TILE if keep else 0
    return x.new_empty(n, length, width), x.new_empty(n, width, **f), x.new_empty(n, tiles, width, **f)


def _scan_bwd_fake(gh, glast, x, r, i, lam, mask, tiles, sharpness):
    n, length, width = x.shape
    f = dict(dtype=torch.float32)
    return (x.new_empty(n, length, width), x.new_empty(n, length, width), x.new_empty(n, length, width), x.new_empty(width, **f),
            x.new_empty(n, width, **f))


scan_op = _define("gated_scan", "(Tensor x, Tensor r, Tensor i, Tensor lam, Tensor? mask, Tensor? state, float sharpness, bool keep) -> (Tensor, Tensor, Tensor)",
                K.gated_scan_fwd, _scan_fake)
scan_bwd_op = _define("gated_scan_bwd", "(Tensor gh, Tensor? glast, Tensor x, Tensor r, Tensor i, Tensor lam, Tensor? mask, Tensor tiles, float sharpness)"
                    " -> (Tensor, Tensor, Tensor, Tensor, Tensor)", K.gated_scan_bwd, _scan_bwd_fake)
scan_step_op = _define("gated_scan_step", "(Tensor x, Tensor r, Tensor i, Tensor lam, Tensor state, Tensor? mask, float sharpness) -> (Tensor, Tensor)",
                     K.gated_scan_step, lambda x, r, i, lam, state, mask, sharpness: (x.new_empty(x.shape), x.new_empty(x.shape, dtype=torch.float32)))


class GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, i, lam, mask, state, sharpness, keep):
        with below_autograd():
            h, last, tiles = scan_op(x, r, i, lam, mask, state, sharpness, True)
        ctx.save_for_backward(x, r, i, lam, mask, tiles)
        ctx.mark_non_differentiable(tiles)
        ctx.set_materialize_grads(False)
        ctx.sharpness, ctx.has_state = sharpness, state is not None
        return h, last, tiles

    @staticmethod
    def backward(ctx, gh, glast, gtiles):
        _once("lego_hip::gated_scan")
        x, r, i, lam, mask, tiles = ctx.saved_tensors
        if gh is None:
            gh = torch.zeros_like(x, memory_format=torch.contiguous_format)
        with below_autograd():
            dx, dr, di, dlam, dstate = scan_bwd_op(gh, glast, x, r, i, lam, mask, tiles, ctx.sharpness)
        return dx, dr, di, dlam, None, dstate if ctx.has_state else None, None, None


_differentiable("gated_scan", GatedScan, (0, 1, 2, 3, 5))
_not_differentiable("gated_scan_bwd")
_not_differentiable("gated_scan_step")


# ---- block_norm: y = x + scale act(gate) rmsnorm(o) post_w, next = rmsnorm(y) next_w, over rows [rows, width] -> (y, next, the rows'
# 1 / root mean squares [halves, rows]); y is empty without o, next without next_w, the last unless `keep`
def _norm_impl(x, o, gate, post_w, scale, next_w, eps, act, keep):
    y, nxt, stat = K.block_norm_fwd(x, o, gate, post_w, scale, next_w, eps, act, keep)
    return _or_empty(y, x), _or_empty(nxt, x), stat


def _norm_fake(x, o, gate, post_w, scale, next_w, eps, act, keep):
    rows, width = x.shape
    return (x.new_empty(0) if o is None else x.new_empty(rows, width), x.new_empty(0) if next_w is None else x.new_empty(rows, width),
            x.new_empty((o is not None) + (next_w is not None), rows if keep else 0, dtype=torch.float32))


def _norm_bwd_impl(dy, dn, x, o, gate, post_w, scale, next_w, stat, eps, act):
    out = K.block_norm_bwd(dy, dn, x, o, gate, post_w, scale, next_w, eps, act, stat)
    return tuple(_or_empty(t, x, torch.float32 if q >= 3 else None) for q, t in enumerate(out))


def _norm_bwd_fake(dy, dn, x, o, gate, post_w, scale, next_w, stat, eps, act):
    rows = [x.new_empty(0) if t is None else x.new_empty(x.shape) for t in (x, o, gate)]
    return tuple(rows + [x.new_empty(0 if t is None else x.shape[1], dtype=torch.float32) for t in (post_w, scale, next_w)])


norm_op = _define("block_norm", "(Tensor x, Tensor? o, Tensor? gate, Tensor? post_w, Tensor? scale, Tensor? next_w, float eps, int act, bool keep)"
                " -> (Tensor, Tensor, Tensor)", _norm_impl, _norm_fake)
norm_bwd_op = _define("block_norm_bwd", "(Tensor? dy, Tensor? dn, Tensor x, Tensor? o, Tensor? gate, Tensor? post_w, Tensor? scale, Tensor? next_w, Tensor stat,"
                    " float eps, int act) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)", _norm_bwd_impl, _norm_bwd_fake)


class BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, o, gate, post_w, scale, next_w, eps, act, keep):
        with below_autograd():
            y, nxt, stat = norm_op(x, o, gate, post_w, scale, next_w, eps, act, True)
        ctx.save_for_backward(x, o, gate, post_w, scale, next_w, stat)
        ctx.mark_non_differentiable(*(t for t in (y, nxt, stat) if t is stat or t.numel() == 0 and x.numel() > 0))
        ctx.set_materialize_grads(False)
        ctx.eps, ctx.act = eps, act
        return y, nxt, stat

    @staticmethod
    def backward(ctx, gy, gn, gstat):
        _once("lego_hip::block_norm")
        x, o, gate, post_w, scale, next_w, stat = ctx.saved_tensors
        if next_w is not None and gn is None:
            gn = torch.zeros_like(x, memory_format=torch.contiguous_format)
        if next_w is None and gy is None:
            gy = torch.zeros_like(x, memory_format=torch.contiguous_format)
        with below_autograd():
            out = norm_bwd_op(gy if o is not None else None, gn if next_w is not None else None, x, o, gate, post_w, scale, next_w, stat, ctx.eps, ctx.act)
        return tuple(None if t is None else g for g, t in zip(out, (x, o, gate, post_w, scale, next_w))) + (None, None, None)


_differentiable("block_norm", BlockNorm, range(6))
_not_differentiable("block_norm_bwd")


# ---- token_logprobs: rows of logits [rows, items] -> (log probability of the target, entropy, [rows, 2] maximum and ln of the sum of
# exp(x - maximum), the k largest log probabilities, their indices)
def _lp_fake(logits, targets, mask, k):
    rows, f = logits.shape[0], dict(dtype=torch.float32)
    return (logits.new_empty(rows, **f), logits.new_empty(rows, **f), logits.new_empty(rows, 2, **f), logits.new_empty(rows, k, **f),
            logits.new_empty(rows, k, dtype=torch.int32))


logprobs_op = _define("token_logprobs", "(Tensor logits, Tensor? targets, Tensor? mask, SymInt k) -> (Tensor, Tensor, Tensor, Tensor, Tensor)",
              lambda logits, targets, mask, k: K.token_logprobs_fwd(logits, targets, k, mask), _lp_fake)
logprobs_bwd_op = _define("token_logprobs_bwd", "(Tensor? g_logp, Tensor? g_entropy, Tensor? g_top, Tensor logits, Tensor? targets, Tensor? mask, Tensor stat,"
                  " Tensor entropy, Tensor index) -> Tensor", K.token_logprobs_bwd,
                  lambda g_logp, g_entropy, g_top, logits, targets, mask, stat, entropy, index: logits.new_empty(logits.shape))


class TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, k):
        with below_autograd():
            logp, entropy, stat, top, index = logprobs_op(logits, targets, mask, k)
        ctx.save_for_backward(logits, targets, mask, stat, entropy, index)
        ctx.mark_non_differentiable(stat, index)
        ctx.set_materialize_grads(False)
        return logp, entropy, stat, top, index

    @staticmethod
    def backward(ctx, g_logp, g_entropy, g_stat, g_top, g_index):
        _once("lego_hip::token_logprobs")
        logits, targets, mask, stat, entropy, index = ctx.saved_tensors
        with below_autograd():
            return logprobs_bwd_op(g_logp, g_entropy, g_top, logits, targets, mask, stat, entropy, index), None, None, None


_differentiable("token_logprobs", TokenLogprobs, (0,))
_not_differentiable("token_logprobs_bwd")


OPS = ("gather_rows", "scatter_add_rows", "linear", "linear_bwd", "glove_project", "glove_project_bwd", "glove_project_bwd_table", "conv3_relu_mask",
       "conv3_relu_mask_bwd", "additive_pool", "additive_pool_bwd", "mhsa", "mhsa_bwd", "rowdot", "rowdot_bwd", "dot_ce",
       "dot_ce_bwd", "adam_step", "sample_negatives", "gather_history", "gated_scan", "gated_scan_bwd", "gated_scan_step", "block_norm",
       "block_norm_bwd", "token_logprobs", "token_logprobs_bwd")
