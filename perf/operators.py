"""Work of the sequence operators on the GPU, case by case: the gated linear recurrence of a click-history encoder, the norms, gate and
residual scale around its blocks, and the log probabilities of the next item over a catalogue (with entropy and the likeliest items).

`own` chooses what `run` calls: the plain form (elementary torch operations in 32 bits) or `legommenders_amd.functional`."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SHARPNESS, EPS = 8.0, 1e-6


# ------------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new click for each of 64 users: the serving form, where only latency counts
        {"name": "step_64x256_f32", "op": "step", "n": 64, "width": 256, "type": "f32"},
        # the user-cache page of the evaluators: 512 users, histories of 0 to 50 clicks, inference
        {"name": "history_512x50x256_f32", "op": "scan", "n": 512, "length": 50, "width": 256, "type": "f32", "ragged": True, "train": False},
        # a training batch of 64 users at the default width
        {"name": "history_64x50x256_f32_train", "op": "scan", "n": 64, "length": 50, "width": 256, "type": "f32", "ragged": True, "train": True},
        # one long event stream of odd sizes that goes on from a state, inference in half precision
        {"name": "stream_1x10007x301_f16", "op": "scan", "n": 1, "length": 10007, "width": 301, "type": "f16", "ragged": False, "train": False},
        # long sequences at the transformer width, two a GPU, training
        {"name": "stream_2x32768x768_bf16_train", "op": "scan", "n": 2, "length": 32768, "width": 768, "type": "bf16", "ragged": False, "train": True},
        # the norms around a block for one training batch of histories (64 x 50 rows), forward only
        {"name": "norms_3200x256_f32", "op": "norms", "rows": 3200, "width": 256, "type": "f32", "train": False},
        # the rows of a batch of encoded titles at the transformer width, training
        {"name": "norms_29600x768_f32_train", "op": "norms", "rows": 29600, "width": 768, "type": "f32", "train": True},
        # the same for long sequences in 16 bits
        {"name": "norms_65536x1024_bf16_train", "op": "norms", "rows": 65536, "width": 1024, "type": "bf16", "train": True},
        # one user's next item over a vocabulary of 400 000, 20 alternatives: latency
        {"name": "next_1x400000_f32_top20", "op": "logprobs", "rows": 1, "items": 400000, "type": "f32", "k": 20, "mask": False, "train": False},
        # a page of 512 users over the whole catalogue, 10 alternatives
        {"name": "next_512x65238_f32_top10", "op": "logprobs", "rows": 512, "items": 65238, "type": "f32", "k": 10, "mask": False, "train": False},
        # a training batch over the catalogue without the items that a user knows already (one row has none left), 50 alternatives
        {"name": "next_64x65238_f32_top50_masked_train", "op": "logprobs", "rows": 64, "items": 65238, "type": "f32", "k": 50, "mask": True, "train": True},
        # masked-token training rows over the word-piece vocabulary in 16 bits, where values tie
        {"name": "next_2048x30522_bf16_train", "op": "logprobs", "rows": 2048, "items": 30522, "type": "bf16", "k": 5, "mask": False, "train": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "norms", "norms", "logprobs", "logprobs"])
    kind = rng.choice(["f32", "f32", "bf16", "f16"])
    if op == "step":
        return {"op": op, "n": _log(rng, 1, 8192), "width": _log(rng, 16, 1024), "type": kind}
    if op == "scan":
        width = _log(rng, 16, 1024)
        length = _log(rng, 1, 32768)
        n = _log(rng, 1, max(1, min(4096, (1 << 25) // (width * length))))
        return {"op": op, "n": n, "length": length, "width": width, "type": kind, "ragged": rng.random() < 0.5, "train": rng.random() < 0.6}
    if op == "norms":
        width = _log(rng, 16, 2048)
        return {"op": op, "rows": _log(rng, 1, max(1, min(65536, (1 << 25) // width))), "width": width, "type": kind, "train": rng.random() < 0.6}
    items = _log(rng, 100, 400000)
    return {"op": op, "rows": _log(rng, 1, max(1, min(4096, (1 << 25) // items))), "items": items, "type": kind, "k": _log(rng, 1, 64),
            "mask": rng.random() < 0.4, "train": rng.random() < 0.6}


# ------------------------------------------------------------------------------------------------------------------- inputs
def _randn(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = TYPES[case["type"]]
    s = {"op": case["op"], "train": case.get("train", False)}
    if case["op"] in ("step", "scan"):
        n, width, length = case["n"], case["width"], case.get("length", 1)
        # values, both gates' logits: three thirds of one projection's rows, as the encoder's product writes them
        rows = _randn(g, (n, length, 3 * width), dtype)
        rows = rows[:, 0] if case["op"] == "step" else rows
        s["x"], s["r"], s["i"] = rows[..., :width], rows[..., width:2 * width], rows[..., 2 * width:]
        decay = 0.9 + 0.099 * torch.rand(width, generator=g, device="cuda")                 # of a fully open gate
        s["lam"] = torch.log(torch.expm1(-torch.log(decay) / SHARPNESS))
        s["state"] = _randn(g, (n, width))
        s["mask"] = None
        if case.get("ragged"):                                                               # lengths about 0.4 of the full one; some users have none
            u = torch.rand(n, generator=g, device="cuda")
            lens = torch.clamp((-torch.log1p(-u) * 0.4 * length).to(torch.int64), 0, length)
            s["mask"] = torch.arange(length, device="cuda")[None] < lens[:, None]
        leaves = ("x", "r", "i", "lam", "state")
        if s["train"]:
            s["g_h"], s["g_last"] = _randn(g, (n, length, width), dtype), _randn(g, (n, width))
    elif case["op"] == "norms":
        rows, width = case["rows"], case["width"]
        s["x"], s["o"], s["gate"] = _randn(g, (rows, width), dtype, 2.0), _randn(g, (rows, width), dtype), _randn(g, (rows, width), dtype)
        s["post_w"], s["next_w"] = 1 + _randn(g, (width,), scale=0.2), 1 + _randn(g, (width,), scale=0.2)
        s["scale"] = _randn(g, (width,), scale=0.3)
        leaves = ("x", "o", "gate", "post_w", "scale", "next_w")
        if s["train"]:
            s["g_y"], s["g_n"] = _randn(g, (rows, width), dtype), _randn(g, (rows, width), dtype)
    else:
        rows, items = case["rows"], case["items"]
        s["logits"] = _randn(g, (rows, items), dtype, 2.5)
        s["targets"] = torch.randint(0, items, (rows,), generator=g, device="cuda")
        s["targets"][rows // 3:rows // 3 + rows // 8] = -1                                   # rows without a target
        s["k"], s["mask"] = min(case["k"], items), None
        if case["mask"]:
            s["mask"] = torch.rand((rows, items), generator=g, device="cuda") < 0.97
            s["mask"].scatter_(1, s["targets"].clamp(min=0)[:, None], True)
            s["mask"][rows // 2] = rows == 1                                                 # nothing left for this row
            s["targets"][rows // 2] = -1
        leaves = ("logits",)
        if s["train"]:
            s["g_logp"], s["g_entropy"] = _randn(g, (rows,)), _randn(g, (rows,), scale=0.1)
    if s["train"]:
        for k in leaves:
            s[k] = s[k].detach().requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    from legommenders_amd import functional as F
    if s["op"] == "step":
        h, state = F.gated_scan_step(s["x"], s["r"], s["i"], s["lam"], s["state"], sharpness=SHARPNESS)
        return {"h": h, "state": state}
    if s["op"] == "scan":
        h, last = F.gated_scan(s["x"], s["r"], s["i"], s["lam"], mask=s["mask"], state=s["state"], sharpness=SHARPNESS)
        if not s["train"]:
            return {"h": h, "last": last}
        d = torch.autograd.grad((h, last), (s["x"], s["r"], s["i"], s["lam"], s["state"]), (s["g_h"], s["g_last"]))
        return {"h": h, "last": last, "dx": d[0], "dr": d[1], "di": d[2], "dlam": d[3], "dstate": d[4]}
    if s["op"] == "norms":
        y, n = F.gated_residual_norm(s["x"], s["o"], s["gate"], s["post_w"], s["scale"], s["next_w"], eps=EPS, act="silu")
        if not s["train"]:
            return {"y": y, "n": n}
        d = torch.autograd.grad((y, n), (s["x"], s["o"], s["gate"], s["post_w"], s["scale"], s["next_w"]), (s["g_y"], s["g_n"]))
        return {"y": y, "n": n, "dx": d[0], "do": d[1], "dgate": d[2], "dpost_w": d[3], "dscale": d[4], "dnext_w": d[5]}
    logp, entropy, top, index = F.token_logprobs(s["logits"], s["targets"], k=s["k"], mask=s["mask"])
    out = {"logp": logp, "entropy": entropy, "top": top, "index": index}
    if s["train"]:
        out["dlogits"] = torch.autograd.grad((logp, entropy), (s["logits"],), (s["g_logp"], s["g_entropy"]))[0]
    return out


# ------------------------------------------------------------------------------------------------------------------- the plain forms
def _scan(a, b):
    """h_t = a_t h_(t-1) + b_t along dimension 1, by doubling"""
    step, length = 1, a.shape[1]
    while step < length:
        b = torch.cat((b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]), 1)
        a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    return b


def _plain_scan(s):
    dtype = s["x"].dtype
    step = s["op"] == "step"
    x, r, i = ((t[:, None] if step else t).float() for t in (s["x"], s["r"], s["i"]))
    soft = torch.log1p(torch.exp(s["lam"]))
    gr, gi = 1 / (1 + torch.exp(-r)), 1 / (1 + torch.exp(-i))
    log_a = -SHARPNESS * soft * gr
    a, beta = torch.exp(log_a), torch.sqrt(-torch.expm1(2 * log_a))
    u = gi * x
    b = beta * u
    live = None if s["mask"] is None else s["mask"][..., None]
    if live is not None:
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)
    first = b.clone()
    first[:, 0] += a[:, 0] * s["state"]
    h = _scan(a, first)
    last = h[:, -1].clone()
    seen = (h if live is None else torch.where(live, h, 0.0)).to(dtype)
    if step:
        return {"h": seen[:, 0], "state": last}
    if not s["train"]:
        return {"h": seen, "last": last}
    gh = s["g_h"].float()
    if live is not None:
        gh = torch.where(live, gh, 0.0)
    gh = gh.clone() if live is None else gh
    gh[:, -1] += s["g_last"]
    # G_t = gh_t + a_(t+1) G_(t+1): the same scan from the other end
    back = torch.cat((torch.ones_like(a[:, :1]), a.flip(1)[:, :-1]), 1)
    G = _scan(back, gh.flip(1)).flip(1)
    before = torch.cat((s["state"][:, None], h[:, :-1]), 1)
    du = G * beta
    q = G * (before * a - u * a * a / beta) * log_a
    if live is not None:
        du, q = torch.where(live, du, 0.0), torch.where(live, q, 0.0)
    dlam = q.sum((0, 1)) / (soft * (1 + torch.exp(-s["lam"])))
    return {"h": seen, "last": last, "dx": (du * gi).to(dtype), "dr": (q * (1 - gr)).to(dtype), "di": (du * u * (1 - gi)).to(dtype),
            "dlam": dlam, "dstate": a[:, 0] * G[:, 0]}


def _plain_norms(s):
    dtype = s["x"].dtype
    x, o, g = s["x"].float(), s["o"].float(), s["gate"].float()
    wp, sc, wn = s["post_w"], s["scale"], s["next_w"]
    ro = torch.rsqrt((o * o).mean(1, keepdim=True) + EPS)
    oh, sig = o * ro, 1 / (1 + torch.exp(-g))
    act = g * sig
    y = x + sc * act * oh * wp
    ry = torch.rsqrt((y * y).mean(1, keepdim=True) + EPS)
    yh = y * ry
    out = {"y": y.to(dtype), "n": (yh * wn).to(dtype)}
    if not s["train"]:
        return out
    gy, gn = s["g_y"].float(), s["g_n"].float()
    t = gn * wn
    d = gy + ry * (t - yh * (t * yh).mean(1, keepdim=True))
    z = (d * act * oh).sum(0)
    t = d * sc * act * wp
    out.update(dx=d.to(dtype), do=(ro * (t - oh * (t * oh).mean(1, keepdim=True))).to(dtype),
               dgate=(d * sc * oh * wp * (sig + act * (1 - sig))).to(dtype), dpost_w=z * sc, dscale=z * wp, dnext_w=(gn * yh).sum(0))
    return out


def _plain_logprobs(s):
    x = s["logits"].float()
    rows, items = x.shape
    if s["mask"] is not None:
        x = torch.where(s["mask"], x, -math.inf)
    m = x.amax(1, keepdim=True)
    empty = m == -math.inf
    e = torch.exp(x - torch.where(empty, 0.0, m))
    total = e.sum(1, keepdim=True)
    lse = torch.where(empty, -math.inf, m + torch.log(total))
    p = e / torch.where(empty, 1.0, total)
    lp = torch.where(empty, -math.inf, x - torch.where(empty, 0.0, lse))
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(1)
    wanted = s["targets"] >= 0
    logp = torch.where(wanted, lp.gather(1, s["targets"].clamp(min=0)[:, None])[:, 0], 0.0)
    # the largest first, ties to the lowest index: whole keys that order as the values do, with the index behind
    bits = (x + 0.0).view(torch.int32).long()
    key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32) + (items - 1 - torch.arange(items, device=x.device))
    index = items - 1 - (key.topk(s["k"], 1)[0] & 0xFFFFFFFF)
    top = lp.gather(1, index)
    out = {"logp": logp, "entropy": entropy, "top": top, "index": torch.where(top == -math.inf, -1, index).to(torch.int32)}
    if s["train"]:
        gl, ge = (s["g_logp"] * wanted)[:, None], s["g_entropy"][:, None]
        d = -p * gl - ge * torch.where(p > 0, p * (lp + entropy[:, None]), 0.0)
        d.scatter_add_(1, s["targets"].clamp(min=0)[:, None], gl)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"step": _plain_scan, "scan": _plain_scan, "norms": _plain_norms, "logprobs": _plain_logprobs}[state["op"]](state)


# ------------------------------------------------------------------------------------------------------------------- in 64 bits
def _exact_scan(s):
    step = s["op"] == "step"
    x, r, i = ((t.detach()[:, None] if step else t.detach()).double() for t in (s["x"], s["r"], s["i"]))
    lam, state = s["lam"].detach().double(), s["state"].detach().double()
    n, length, width = x.shape
    live = torch.ones(n, length, 1, dtype=torch.bool, device=x.device) if s["mask"] is None else s["mask"][..., None]
    soft = torch.nn.functional.softplus(lam, threshold=1000)
    gr, gi = torch.sigmoid(r), torch.sigmoid(i)
    log_a = -SHARPNESS * soft * gr
    a = torch.exp(log_a)
    beta = torch.sqrt(-torch.expm1(2 * log_a))
    A, Bu = a.masked_fill(~live, 1.0), (beta * gi * x).masked_fill(~live, 0.0)
    h = torch.empty_like(x)
    now = state
    for t in range(length):
        now = torch.addcmul(Bu[:, t], A[:, t], now)
        h[:, t] = now
    seen = h.masked_fill(~live, 0.0)
    if step:
        return {"h": seen[:, 0], "state": now}
    if not s["train"]:
        return {"h": seen, "last": now}
    gh = s["g_h"].double().masked_fill(~live, 0.0)
    G = torch.empty_like(x)
    carry = s["g_last"].double()
    for t in range(length - 1, -1, -1):
        carry = carry + gh[:, t]
        G[:, t] = carry
        carry = carry * A[:, t]
    before = torch.cat((state[:, None], h[:, :-1]), 1)
    dlog = (G * (before * a - gi * x * (a * a) / beta)).masked_fill(~live, 0.0)
    du = (G * beta).masked_fill(~live, 0.0)
    dlam = -SHARPNESS * torch.sigmoid(lam) * (dlog * gr).sum((0, 1))
    return {"h": seen, "last": now, "dx": du * gi, "dr": dlog * (-SHARPNESS) * soft * gr * (1 - gr), "di": du * x * gi * (1 - gi),
            "dlam": dlam, "dstate": carry}


def _exact_norms(s):
    names = ("x", "o", "gate", "post_w", "scale", "next_w")
    x, o, g, wp, sc, wn = v = [s[k].detach().double().requires_grad_(s["train"]) for k in names]
    p = o / (o.square().mean(-1, keepdim=True) + EPS).sqrt() * wp
    y = x + sc * (torch.nn.functional.silu(g) * p)
    n = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * wn
    if not s["train"]:
        return {"y": y, "n": n}
    d = torch.autograd.grad((y, n), v, (s["g_y"].double(), s["g_n"].double()))
    return dict(zip(("y", "n", "dx", "do", "dgate", "dpost_w", "dscale", "dnext_w"), (y.detach(), n.detach(), *d)))


def _exact_logprobs(s):
    x = s["logits"].detach().double()
    if s["mask"] is not None:
        x = x.masked_fill(~s["mask"], -math.inf)
    some = (x > -math.inf).any(1)
    lp = torch.log_softmax(x, 1).masked_fill(~some[:, None], -math.inf)
    p = torch.exp(lp)
    entropy = torch.special.entr(p).sum(1)
    wanted = s["targets"] >= 0
    one = torch.zeros_like(p).scatter_(1, s["targets"].clamp(min=0)[:, None], 1.0) * wanted[:, None]
    logp = torch.where(wanted, lp.gather(1, s["targets"].clamp(min=0)[:, None]).squeeze(1), 0.0)
    top, index = (t[:, :s["k"]] for t in torch.sort(lp, dim=1, descending=True, stable=True))
    out = {"logp": logp, "entropy": entropy, "top": top, "index": index.masked_fill(top == -math.inf, -1).to(torch.int32)}
    if s["train"]:
        d = (one - p * wanted[:, None]) * s["g_logp"].double()[:, None]
        out["dlogits"] = d - s["g_entropy"].double()[:, None] * torch.special.xlogy(p, p * torch.exp(entropy)[:, None])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"step": _exact_scan, "scan": _exact_scan, "norms": _exact_norms, "logprobs": _exact_logprobs}[case["op"]](s)


# ------------------------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    """`flops`: an exponential, a root or a division counts as one operation"""
    es = 4 if case["type"] == "f32" else 2
    train = case.get("train", False)
    if case["op"] in ("step", "scan"):
        n, width, length = case["n"], case["width"], case.get("length", 1)
        share = 0.4 if case.get("ragged") else 1.0                       # the masked rows need not be read; the outputs' zeros are written
        cells, states = n * length * width, n * width * 4
        size = cells * es * (3 * share + 1) + 2 * states + 4 * width + (n * length if case.get("ragged") else 0)
        if train:
            size += cells * es * (4 * share + 3) + 2 * states + 8 * width
        return {"bytes": int(size), "flops": int(cells * share * (16 if not train else 56))}
    if case["op"] == "norms":
        cells, width = case["rows"] * case["width"], case["width"]
        size = 5 * cells * es + 12 * width + (8 * cells * es + 24 * width if train else 0)
        return {"bytes": int(size), "flops": int(cells * (14 if not train else 50))}
    rows, items = case["rows"], case["items"]
    size = rows * items * es + (rows * items if case["mask"] else 0) + rows * (8 + 8 + 8 * case["k"])
    if train:
        size += 2 * rows * items * es + (rows * items if case["mask"] else 0) + 8 * rows
    return {"bytes": int(size), "flops": int(rows * items * (6 if not train else 14))}
