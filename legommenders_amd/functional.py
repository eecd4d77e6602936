"""The reference's dense operator shapes on `torch.ops.lego_hip.*` (legommenders_amd/ops.py: the HIP kernels registered
with the PyTorch dispatcher, autograd and fake implementations included).

This is the layer the plug-in classes (`model/operators/*`, `model/predictors/*`, `loader/embedding_hub`) call, so
third-party operators written against the reference's interface keep working while every arithmetic step runs in
liblego_hip.so.  The functions here only reshape to the ops' 2-D / 3-D layouts and hand each dropout call its Philox
stream `(p, seed, site)`.  The training fast path (`engine.py`) bypasses autograd entirely.  No CPU fallback: the ops have
ROCm implementations only, and CPU tensors raise `LegoHipError` here before they reach the dispatcher.
"""
from __future__ import annotations

import itertools

import torch

from . import ops as _ops  # noqa: F401  (registers torch.ops.lego_hip)
from ._lib import LegoHipError

_site = itertools.count(1)
SEED = 2023
L = torch.ops.lego_hip


def seed_streams(seed: int):
    """seed of the Philox dropout streams of this process (data parallel: train_step.rank_seed(seed, rank))"""
    global SEED
    SEED = int(seed)


def _rng(p, training):
    """(p, seed, site): a fresh Philox stream per call; p = 0 in eval"""
    if not training or p <= 0:
        return 0.0, 0, 0
    return float(p), SEED, 1000 + next(_site)


def _need_gpu(t, what):
    if not t.is_cuda:
        raise LegoHipError(f"{what}: CPU tensors are not supported -- the MI355X path has no CPU fallback "
                           "(use the reference for --cuda -1)")


def linear(x, W, b=None, act=0):
    _need_gpu(x, "linear")
    if act != 0:
        raise LegoHipError("functional.linear implements nn.Linear only; tanh is fused inside additive_attention")
    shape = x.shape
    y = L.linear(x.reshape(-1, shape[-1]), W, b)
    return y.view(*shape[:-1], W.shape[0])


def glove_project(ids, table, W, b, p=0.0, training=False):
    """Transformation.forward + SimpleInputer masking (loader/embedding_hub.py:95-96, simple_inputer.py:55-63)"""
    _need_gpu(ids, "embedding")
    H, _ = L.glove_project(ids.reshape(-1), table, W, b, *_rng(p, training))
    return H.view(*ids.shape, W.shape[0])


def embedding(ids, table):
    """trainable nn.Embedding look-up with the inputer's pad handling (id -1 -> zero row), dense gradient"""
    _need_gpu(ids, "embedding")
    return L.gather_rows(table, ids.reshape(-1)).view(*ids.shape, table.shape[1])


def conv3_relu_mask(h, mask, w, b, p=0.0, training=False):
    """CNNOperator title branch: Conv1d(k=3,'same') -> ReLU -> *mask -> Dropout (cnn_operator.py:54-57)"""
    _need_gpu(h, "conv3")
    if w.shape[2] != 3:
        raise LegoHipError("the HIP conv kernel implements kernel_size=3 (config/model/naml.yaml:14)")
    return L.conv3_relu_mask(h, mask, w, b, *_rng(p, training))


def additive_attention(x, mask, W1, b1, w2):
    _need_gpu(x, "additive_attention")
    return L.additive_pool(x, mask, W1, b1, w2)[0]


def multi_head_self_attention(x, mask, in_w, in_b, out_w, out_b, heads, p=0.0, training=False):
    _need_gpu(x, "multi_head_attention")
    return L.mhsa(x, mask, in_w, in_b, out_w, out_b, int(heads), *_rng(p, training))[0]


def rowdot(u, it):
    _need_gpu(u, "dot predictor")
    return L.rowdot(u, it)


def dot_ce(user, items):
    """fused DotPredictor + CrossEntropy(label 0) on [B,D] users x [B,C,D] candidates -> (loss, scores)"""
    _need_gpu(user, "dot_ce")
    return L.dot_ce(user, items)


# ------------------------------------------------------------------------------------------ sequence operators
# fp32, bf16 or fp16 activations (kept), fp32 weights and states; strided rows are taken as they are.  A step that a mask (0 / False) hides is
# never used, whatever it holds.  (The checks run on every call of operators that take microseconds: they build no message unless they refuse.)
_LEAST, _MOST = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max
_TYPES = frozenset((torch.float32, torch.bfloat16, torch.float16))


def _refuse(what, why):
    raise LegoHipError(f"{what}: {why}")


def _activations(what, first, *others):
    """same shape and type for every activation (the device of every operand is looked at where the pointers are taken)"""
    if not isinstance(first, torch.Tensor) or first.dtype not in _TYPES:
        _refuse(what, "activations are float32, bfloat16 or float16 tensors")
    for t in others:
        if not isinstance(t, torch.Tensor) or t.shape != first.shape or t.dtype is not first.dtype:
            _refuse(what, f"every activation has to match the first: {tuple(first.shape)}, {first.dtype}")


def _weights(what, like, shape, *weights):
    for t in weights:
        if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype is not torch.float32:
            _refuse(what, f"weights and states are float32 tensors on {like.device}, here of shape {tuple(shape)}")


def _mask_of(what, mask, shape, like):
    if not isinstance(mask, torch.Tensor) or mask.shape != shape:
        _refuse(what, f"mask has to be of shape {tuple(shape)} on {like.device}")


def _run(what, function, op, operands, *rest):
    """the op on its operands and the rest of its arguments: through its autograd.Function where a gradient is wanted, else below the autograd key"""
    if torch.compiler.is_compiling():                # traced: the registered op, whose autograd entry does the rest
        return op(*rest)
    _ops.refuse_tangents(what, operands)
    if torch.is_grad_enabled():
        for t in operands:
            if t is not None and t.requires_grad:
                return function.apply(*rest)
    with _ops.below_autograd():
        return op(*rest)


def gated_scan(x, r, i, lam, mask=None, state=None, sharpness=8.0):
    """Gated linear recurrence over [n, length, width], a channel at a time:

        a_t = exp(-sharpness softplus(lam) sigmoid(r_t)),   h_t = a_t h_(t-1) + sqrt(1 - a_t^2) sigmoid(i_t) x_t,   h_0 = state (default 0)

    -> (h in the activations' type, the state behind the last step [n, width] fp32).  `mask` [n, length]: a masked step keeps the state, its
    row of h is zeros and its gradients are zeros.  Differentiable (once) in x, r, i, lam and state.  For one more step of many states without a
    gradient: `gated_scan_step`.  A gate below 2^-126 counts as closed."""
    what = "gated_scan"
    _activations(what, x, r, i)
    if x.dim() != 3 or x.shape[0] > 65535:
        _refuse(what, f"x is [n, length, width] with n <= 65535, not {tuple(x.shape)}")
    n, length, width = x.shape
    _weights(what, x, (width,), lam)
    if state is not None:
        _weights(what, x, (n, width), state)
    if mask is not None:
        _mask_of(what, mask, (n, length), x)
    if not _LEAST <= sharpness <= _MOST:
        _refuse(what, f"sharpness {sharpness} is not a positive number of fp32")
    _need_gpu(x, what)
    h, last, _ = _run(what, _ops.GatedScan, _ops.scan_op, (x, r, i, lam, state), x, r, i, lam, mask, state, float(sharpness), False)
    return h, last


def gated_scan_step(x, r, i, lam, state, mask=None, sharpness=8.0):
    """`gated_scan` for one step: x, r, i [n, width], state [n, width] fp32 -> (h [n, width], the new state).  The form that serves: no
    gradient (operands that require one are refused under grad mode), `state` is left as it is.  A masked row keeps its state, its h is zeros."""
    what = "gated_scan_step"
    _activations(what, x, r, i)
    if x.dim() != 2:
        _refuse(what, f"x is [n, width], not {tuple(x.shape)}")
    _weights(what, x, x.shape[1:], lam)
    _weights(what, x, x.shape, state)
    if mask is not None:
        _mask_of(what, mask, x.shape[:1], x)
    if not _LEAST <= sharpness <= _MOST:
        _refuse(what, f"sharpness {sharpness} is not a positive number of fp32")
    if torch.is_grad_enabled() and (x.requires_grad or r.requires_grad or i.requires_grad or lam.requires_grad or state.requires_grad):
        _refuse(what, "has no gradient; use gated_scan, or call it under torch.no_grad()")
    _need_gpu(x, what)
    if torch.compiler.is_compiling():
        return _ops.scan_step_op(x, r, i, lam, state, mask, float(sharpness))
    _ops.refuse_tangents(what, (x, r, i, lam, state))
    with _ops.below_autograd():
        return _ops.scan_step_op(x, r, i, lam, state, mask, float(sharpness))


def _rows2(t):
    return t if t is None or t.dim() == 2 else t.reshape(-1, t.shape[-1])


def _norm_width(what, x):
    if x.dim() < 1 or not 0 < x.shape[-1] <= _ops.K.BLOCK_NORM_MAX_WIDTH:
        _refuse(what, f"the last dimension is 1 to {_ops.K.BLOCK_NORM_MAX_WIDTH} wide, not {tuple(x.shape)}")


def rms_norm(x, w, eps=1e-6):
    """x (mean x^2 + eps)^-1/2 w over the last dimension (at most 16384 wide); x in fp32, bf16 or fp16 (kept), w fp32.  Differentiable (once)."""
    what = "rms_norm"
    _activations(what, x)
    _norm_width(what, x)
    _weights(what, x, x.shape[-1:], w)
    _need_gpu(x, what)
    n = _run(what, _ops.BlockNorm, _ops.norm_op, (x, w), _rows2(x), None, None, None, None, w, float(eps), 0, False)[1]
    return n if x.dim() == 2 else n.view(x.shape)


def gated_residual_norm(x, o, gate, post_w, scale, next_w=None, eps=1e-6, act="silu"):
    """The norms around a residual block with its gate and residual scale, in one pass over the rows:

        y = x + scale * act(gate) * (o (mean o^2 + eps)^-1/2 post_w),     n = y (mean y^2 + eps)^-1/2 next_w

    x: the residual stream, o: the block's output, gate: its gate's logits (act "silu" or "sigmoid"; None with act=None: no gate), all of one
    shape [..., width] and type; post_w, scale, next_w [width] fp32.  -> (y, n): n is the norm before the next block (None without next_w),
    taken from y before its rounding.  Differentiable (once) in every operand."""
    what = "gated_residual_norm"
    if act not in _ops.K.GATE_ACTS or (gate is None) != (act is None):
        _refuse(what, f"act {act!r} has to be 'silu' or 'sigmoid' with a gate, None without")
    if gate is None:
        _activations(what, x, o)
    else:
        _activations(what, x, o, gate)
    _norm_width(what, x)
    _weights(what, x, x.shape[-1:], post_w, scale)
    if next_w is not None:
        _weights(what, x, x.shape[-1:], next_w)
    _need_gpu(x, what)
    y, n, _ = _run(what, _ops.BlockNorm, _ops.norm_op, (x, o, gate, post_w, scale, next_w), _rows2(x), _rows2(o), _rows2(gate), post_w, scale, next_w,
                   float(eps), _ops.K.GATE_ACTS[act], False)
    if x.dim() != 2:
        y, n = y.view(x.shape), n if next_w is None else n.view(x.shape)
    return y, None if next_w is None else n


def token_logprobs(logits, targets=None, k=0, mask=None):
    """Log probabilities over rows of logits [..., items] (fp32, bf16 or fp16; rows may be strided), all fp32:

        -> (logp [...] of `targets`, entropy [...], top [..., k] the largest log probabilities, index [..., k] int32)

    targets int32 / int64 [...]: an item outside [0, items) -- the pad id -1 -- is no target: logp 0, no gradient.  top is sorted, equal values by
    index; k <= 128.  `mask` [..., items] or [items]: items that are 0 / False there do not exist (the clicks a user has made already).  A row
    with nothing left has logp and top -inf, entropy 0, index -1, and a zero gradient; one with NaN or +inf among its items has NaN.
    Differentiable (once) in logits through logp, entropy and top; a masked target's logp is -inf."""
    what = "token_logprobs"
    _activations(what, logits)
    if logits.dim() < 1 or not 0 < logits.shape[-1] <= 1 << 30:
        _refuse(what, f"logits are [..., items] with at least one item, not {tuple(logits.shape)}")
    items = logits.shape[-1]
    if not isinstance(k, int) or not 0 <= k <= min(_ops.K.LOGPROBS_MAX_K, items):
        _refuse(what, f"k = {k} is not 0 to {min(_ops.K.LOGPROBS_MAX_K, items)}")
    if targets is not None and (not isinstance(targets, torch.Tensor) or targets.dtype not in (torch.int32, torch.int64)
                                or targets.shape != logits.shape[:-1]):
        _refuse(what, f"targets are int32 or int64 of shape {tuple(logits.shape[:-1])} on {logits.device}")
    if mask is not None and (not isinstance(mask, torch.Tensor) or (mask.shape != logits.shape and mask.shape != (items,))):
        _refuse(what, f"mask has to be of shape {tuple(logits.shape)} or ({items},) on {logits.device}")
    _need_gpu(logits, what)
    flat = logits.dim() == 2
    rows = logits if flat else logits.reshape(-1, items)
    if mask is not None and mask.dim() != 2:
        mask = mask.reshape(-1, items) if mask.dim() > 2 else mask.expand(rows.shape)
    if targets is not None and not flat:
        targets = targets.reshape(-1)
    logp, entropy, _, top, index = _run(what, _ops.TokenLogprobs, _ops.logprobs_op, (logits,), rows, targets, mask, k)
    if flat:
        return logp, entropy, top, index
    lead = logits.shape[:-1]
    return logp.view(lead), entropy.view(lead), top.view(*lead, k), index.view(*lead, k)


def catalogue_scores(user, items):
    """<user, item> of every pair: user [B, D] x items [N, D] -> [B, N] on the product kernels.  Their rows are multiples of 4 elements: other
    catalogues are padded by zero items, and the result is a view without them (`token_logprobs` takes such rows)."""
    n = items.shape[0]
    return linear(user, torch.nn.functional.pad(items, (0, 0, 0, -n % 4)) if n % 4 else items)[:, :n]


def next_item_loss(user, items, targets, mask=None):
    """-mean log probability of each user's next item over a whole catalogue: user [B, D] x items [N, D] -> scalar; targets [B] (outside
    [0, N): the row does not count).  The full-softmax sibling of `dot_ce`'s sampled one: the scores are one product, their softmax and its
    gradient one pass each.  Where 4 does not divide N, the items and the scores' gradient are copied once more into padded ones (512 users x 65 238
    items: 5 % of the step)."""
    if targets.dim() != 1 or user.dim() != 2 or targets.shape[0] != user.shape[0]:
        _refuse("next_item_loss", f"targets are one item a user: {tuple(targets.shape)} for users {tuple(user.shape)}")
    _need_gpu(user, "next_item_loss")
    logp = token_logprobs(catalogue_scores(user, items), targets, mask=mask)[0]
    return -logp.sum() / ((targets >= 0) & (targets < items.shape[0])).sum().clamp(min=1)
