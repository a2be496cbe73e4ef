"""Workloads of the layer-norm, differential-attention and AdamW operators, with their plain forms.

A workload is a dict of plain values (listed(), draw()); prepare() makes its inputs on the GPU, run()
makes one pass: through elementary torch operations while `own` is false, through the package's
operators when it is true.  exact() computes the same outputs in 64 bits, written apart from the
plain form, and work() counts the bytes and operations a pass cannot do without.

  layer_norm       y = w (s - mean) / sqrt(var + eps) + b over the last axis, s = x (+ residual, rounded
                   to the inputs' type, which is what the next layer reads)
  diff_attention   o = (softmax(c q1 k1^T) - lam softmax(c q2 k2^T)) v per head: q [B,Tq,H,2,d],
                   k [B,Tk,Hk,2,d], v [B,Tk,Hk,2d], lam [H]; causal (aligned at the last key) and
                   per-sample key counts; rows that see no key give zero
  adamw            decoupled weight decay over many tensors, moments in f32 or in 8 bits: blocks of 256
                   share the exponent E of their largest value, the first moment is a sign, 4 exponent
                   and 3 mantissa bits below it, the second 5 and 3; stochastic rounding from an integer
                   hash of (seed, step, tensor, element)
"""
import importlib
import math
import random

import torch

own = False

PACKAGE = "tcn-transformer-gan-hybrid-model-for-predicting-streamflow-in-ungauged-basins_amd"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256


def _functional():
    return importlib.import_module(PACKAGE).functional


# ------------------------------------------------------------------------------ the cases
def _model_sizes():
    """Parameter tensors of the forecasting model at hidden 128 with 10 input channels: two conv +
    BatchNorm layers, two 262144-wide Linear layers, two Transformer layers, the decoder."""
    layer = [384 * 128, 384, 128 * 128, 128, 512 * 128, 512, 128 * 512, 128, 128, 128, 128, 128]
    return ([128 * 10 * 9, 128, 128, 256 * 128 * 9, 256, 256, 128 * 262144, 128] + layer + layer
            + [262144 * 128, 262144, 64 * 256 * 9, 64, 64 * 64 * 9, 64, 64, 1])


def _patchgan_sizes():
    """Parameter tensors of the PatchGAN discriminator (1 -> 64 -> 128 -> 256 -> 512 -> 1)."""
    out = [64 * 16, 64]
    for i, o in ((64, 128), (128, 256), (256, 512)):
        out += [o * i * 16, o, o, o]
    return out + [512 * 16, 1]


def _text(sizes):
    return ",".join(str(n) for n in sizes)


def listed():
    return [
        # the smallest call: the tokens of one training batch (32 windows of 5 days) at the model's width
        {"name": "norm train 160x128", "op": "norm", "rows": 160, "dim": 128, "dtype": "bf16", "residual": True, "train": True},
        # inference over the 32 x 32 map tokens of 5 frames of 32 windows
        {"name": "norm infer 163840x256", "op": "norm", "rows": 163840, "dim": 256, "dtype": "bf16", "residual": True, "train": False},
        # a wide training layer
        {"name": "norm train 16384x4096", "op": "norm", "rows": 16384, "dim": 4096, "dtype": "bf16", "residual": True, "train": True},
        # full precision, a width that no vector access divides
        {"name": "norm train 30011x999 f32", "op": "norm", "rows": 30011, "dim": 999, "dtype": "f32", "residual": False, "train": True},
        # one new token per sequence against its keys and values, heads shared four to one, ragged lengths
        {"name": "attn token 16x8192", "op": "attn", "batch": 16, "tq": 1, "tk": 8192, "heads": 16, "kv_heads": 4, "d": 64,
         "dtype": "bf16", "causal": False, "pad": True, "train": False},
        # a year of daily tokens at the model's width (4 heads of 2 x 16), padded samples
        {"name": "attn train 32x365", "op": "attn", "batch": 32, "tq": 365, "tk": 365, "heads": 4, "kv_heads": 4, "d": 16,
         "dtype": "bf16", "causal": True, "pad": True, "train": True},
        # the 5 x 32 x 32 map tokens of a window
        {"name": "attn train 2x5120", "op": "attn", "batch": 2, "tq": 5120, "tk": 5120, "heads": 8, "kv_heads": 8, "d": 64,
         "dtype": "bf16", "causal": False, "pad": False, "train": True},
        # a long causal sequence read once, heads shared
        {"name": "attn infer 1x8191", "op": "attn", "batch": 1, "tq": 8191, "tk": 8191, "heads": 8, "kv_heads": 2, "d": 64,
         "dtype": "bf16", "causal": True, "pad": False, "train": False},
        # full precision at an odd length
        {"name": "attn train 4x777 f32", "op": "attn", "batch": 4, "tq": 777, "tk": 777, "heads": 4, "kv_heads": 2, "d": 32,
         "dtype": "f32", "causal": True, "pad": True, "train": True},
        # the discriminator's small tensors, packed as the flat optimiser lays them out
        {"name": "adamw patchgan f32", "op": "adamw", "sizes": _text(_patchgan_sizes()), "align": 64, "bits": 32, "grad": "f32"},
        # the whole generator, both kinds of state
        {"name": "adamw model f32", "op": "adamw", "sizes": _text(_model_sizes()), "align": 64, "bits": 32, "grad": "f32"},
        {"name": "adamw model 8 bit", "op": "adamw", "sizes": _text(_model_sizes()), "align": BLOCK, "bits": 8, "grad": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_norm(rng):
    dim = _log(rng, 8, 8192)
    if rng.random() < 0.5:
        dim = max(8, dim // 8 * 8)
    return {"op": "norm", "rows": _log(rng, 1, max(1, min(500000, 16384 * 4096 // dim))), "dim": dim,
            "dtype": rng.choice(["bf16", "f32"]), "residual": rng.random() < 0.5, "train": rng.random() < 0.7}


def _draw_attn(rng):
    dtype = rng.choice(["bf16", "bf16", "f32"])
    d = 8 * rng.randint(1, 8)
    kv = rng.choice([1, 2, 3, 4])
    heads = kv * rng.choice([1, 1, 2, 4])
    batch = rng.randint(1, 8)
    most = (2 * 8 * 5120 * 5120 * 64 if dtype == "bf16" else 4 * 8 * 777 * 777 * 64) // (batch * heads * d)
    form = rng.choice(["self", "self", "cross", "token"])
    tq = _log(rng, 1, 5120) if form != "token" else rng.randint(1, 4)
    tk = tq if form == "self" else _log(rng, 1, 8192)
    while tq * tk > most:
        tq, tk = (max(1, tq * 2 // 3), max(1, tk * 2 // 3)) if form != "token" else (tq, max(1, tk * 2 // 3))
    # (a softmax over one key has no gradient at all: nothing to measure against)
    train = min(tq, tk) >= 8 and rng.random() < 0.6
    return {"op": "attn", "batch": batch, "tq": tq, "tk": tk, "heads": heads, "kv_heads": kv, "d": d, "dtype": dtype,
            "causal": rng.random() < 0.5, "pad": rng.random() < 0.5, "train": train}


def _draw_adamw(rng):
    bits = rng.choice([32, 8])
    sizes, left = [], 1 << 25
    for _ in range(rng.randint(1, 60)):
        n = _log(rng, 1, 1 << 22)
        if n <= left:
            sizes.append(n)
            left -= n
    return {"op": "adamw", "sizes": _text(sizes), "align": BLOCK if bits == 8 else rng.choice([1, 64]), "bits": bits,
            "grad": rng.choice(["f32", "bf16"])}


def draw(rng):
    return rng.choice([_draw_norm, _draw_attn, _draw_adamw])(rng)


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _prepare_norm(case, g):
    dt, rows, dim = DTYPES[case["dtype"]], case["rows"], case["dim"]
    s = {"x": _normal(g, (rows, dim), dt) + _normal(g, (rows, 1), dt),
         "w": 1.0 + 0.1 * torch.randn(dim, generator=g, device="cuda"), "b": 0.1 * torch.randn(dim, generator=g, device="cuda"),
         "res": _normal(g, (rows, dim), dt) if case["residual"] else None}
    if case["train"]:
        s["dy"] = _normal(g, (rows, dim), dt)
        s["ds"] = _normal(g, (rows, dim), dt) if case["residual"] else None
        for k in ("x", "w", "b", "res"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


def _lengths(case, g):
    """Key counts of a padded batch: evenly spread from nothing to everything, in an order of the seed."""
    B, tk = case["batch"], case["tk"]
    if not case["pad"]:
        return None
    even = torch.tensor([tk * (i + (B == 1)) // max(1, B - 1) for i in range(B)], dtype=torch.int32, device="cuda")
    return even[torch.randperm(B, generator=g, device="cuda")].contiguous()


def _prepare_attn(case, g):
    dt, B, H, Hk, d = DTYPES[case["dtype"]], case["batch"], case["heads"], case["kv_heads"], case["d"]
    s = {"q": _normal(g, (B, case["tq"], H, 2, d), dt, 1.5), "k": _normal(g, (B, case["tk"], Hk, 2, d), dt, 1.5),
         "v": _normal(g, (B, case["tk"], Hk, 2 * d), dt),
         "lam": (0.2 + 0.6 * torch.rand(H, generator=g, device="cuda")).to(dt), "lengths": _lengths(case, g)}
    if case["train"]:
        s["do"] = _normal(g, (B, case["tq"], H, 2 * d), dt)
        for k in ("q", "k", "v", "lam"):
            s[k].requires_grad_(True)
    return s


def _layout(case):
    """Sizes, starts and the whole length of the tensors in their flat buffer."""
    sizes, starts, at = [int(t) for t in case["sizes"].split(",")], [], 0
    for n in sizes:
        starts.append(at)
        at += (n + case["align"] - 1) // case["align"] * case["align"]
    return sizes, starts, at


def _views(flat, sizes, starts):
    return [flat[o:o + n] for n, o in zip(sizes, starts)]


def _nearest_codes(x, signed):
    """Codes and block exponents of f32 values, rounded toward zero: how prepare() fills the 8-bit moments."""
    bits = x.abs().view(-1, BLOCK).view(torch.int32)
    e = ((bits.amax(1) + 0xFFFFF) >> 23).clamp(16 if signed else 32, 255)
    c = ((bits >> 20) - 8 * e[:, None] + (120 if signed else 248)).clamp(0, 127 if signed else 255)
    if signed:
        c = c | ((x.view(-1, BLOCK) < 0).int() << 7)
    return c.to(torch.uint8).reshape(-1), e.to(torch.uint8)


def _prepare_adamw(case, g):
    sizes, starts, total = _layout(case)
    live = torch.zeros(total, dtype=torch.bool, device="cuda")
    for t in _views(live, sizes, starts):
        t.fill_(True)
    p = torch.randn(total, generator=g, device="cuda") * 0.05 * live
    mag = torch.exp(torch.randn(total, generator=g, device="cuda") * 1.5 - 6.0) * live
    grad = torch.randn(total, generator=g, device="cuda") * mag
    m, v = torch.randn(total, generator=g, device="cuda") * mag * 0.3, mag * mag
    s = {"p": p, "g": grad.to(DTYPES[case["grad"]]), "sizes": sizes, "starts": starts, "seed": 20240229,
         "state": torch.tensor([100, 0], dtype=torch.int32, device="cuda"),
         "decay": [DECAY if i % 2 == 0 else 0.0 for i in range(len(sizes))]}
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        s["m"], s["me"] = _nearest_codes(m, True)
        s["v"], s["ve"] = _nearest_codes(v, False)
        s["m_out"], s["v_out"] = (torch.zeros(total, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    names = ["p", "g", "m", "v"] + (["m_out", "v_out"] if case["bits"] == 8 else [])
    s["lists"] = {k: _views(s[k], sizes, starts) for k in names}
    if case["bits"] == 8:
        for k in ("m", "v"):
            e = [s[k + "e"][o // BLOCK:(o + n + BLOCK - 1) // BLOCK] for n, o in zip(sizes, starts)]
            s["lists"][k] = list(zip(s["lists"][k], e))
    return s


def prepare(case, seed):
    s = {"norm": _prepare_norm, "attn": _prepare_attn, "adamw": _prepare_adamw}[case["op"]](case, _gen(seed))
    s["case"] = case
    return s


# ------------------------------------------------------------------------------ one pass
def _plain_norm(x, res, w, b):
    dt = x.dtype
    s = x if res is None else (x.float() + res.float()).to(dt)
    f = s.float()
    c = f - f.mean(-1, keepdim=True)
    y = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * w + b
    return (y.to(dt), None) if res is None else (y.to(dt), s)


def _run_norm(s):
    x, res, w, b = s["x"], s["res"], s["w"], s["b"]
    if own:
        got = _functional().layer_norm(x, w, b, EPS, residual=res)
        y, total = got if res is not None else (got, None)
    else:
        y, total = _plain_norm(x, res, w, b)
    if not s["case"]["train"]:
        return {"y": y, "s": total}
    if res is None:
        grads = torch.autograd.grad(y, [x, w, b], s["dy"])
        return {"y": y, "dx": grads[0], "dw": grads[1], "db": grads[2]}
    grads = torch.autograd.grad([y, total], [x, res, w, b], [s["dy"], s["ds"]])
    return {"y": y, "s": total, "dx": grads[0], "dres": grads[1], "dw": grads[2], "db": grads[3]}


def _mask(B, tq, tk, causal, lengths, device):
    """[B, 1, 1, tq, tk] (or None): which keys a query sees."""
    key = torch.arange(tk, device=device)
    seen = None
    if causal:
        seen = (key <= torch.arange(tq, device=device)[:, None] + (tk - tq)).view(1, 1, 1, tq, tk)
    if lengths is not None:
        short = (key < lengths.view(B, 1)).view(B, 1, 1, 1, tk)
        seen = short if seen is None else seen & short
    return seen


def _plain_attn(q, k, v, lam, causal, lengths):
    B, tq, H, _, d = q.shape
    tk, Hk = k.shape[1], k.shape[2]
    qf = q.float().permute(0, 2, 3, 1, 4)
    kf = k.float().permute(0, 2, 3, 1, 4).repeat_interleave(H // Hk, 1)
    vf = v.float().permute(0, 2, 1, 3).repeat_interleave(H // Hk, 1)
    z = qf @ kf.transpose(-1, -2) * (1.0 / math.sqrt(d))
    seen = _mask(B, tq, tk, causal, lengths, q.device)
    if seen is not None:
        z = z.masked_fill(~seen, -math.inf)
    top = z.detach().amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    o = (p[:, :, 0] - lam.float().view(1, H, 1, 1) * p[:, :, 1]) @ vf
    return o.permute(0, 2, 1, 3).to(q.dtype)


def _run_attn(s):
    c = s["case"]
    args = (s["q"], s["k"], s["v"], s["lam"])
    if own:
        o = _functional().diff_attention(*args, causal=c["causal"], lengths=s["lengths"])
    else:
        o = _plain_attn(*args, c["causal"], s["lengths"])
    if not c["train"]:
        return {"o": o}
    dq, dk, dv, dlam = torch.autograd.grad(o, args, s["do"])
    return {"o": o, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def _mix(x):
    """32-bit integer mixing on int64 tensors that hold 32-bit values."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_bits(s, step, total):
    """The 32 random bits of every element: the upper 16 round the first moment, the lower 16 the second."""
    sizes = torch.tensor(s["sizes"], device="cuda")
    starts = torch.tensor(s["starts"], device="cuda")
    room = torch.diff(torch.cat([starts, torch.tensor([total], device="cuda")]))
    key = _mix((((s["seed"] & 0xFFFFFFFF) + step.long() * 0x9E3779B1) & 0xFFFFFFFF) ^ (s["seed"] >> 32))
    keys = _mix((key + torch.arange(len(sizes), device="cuda") * 0x85EBCA6B) & 0xFFFFFFFF)
    i = torch.arange(total, device="cuda") - torch.repeat_interleave(starts, room)
    at = ((i & 0xFFFFFFFF) * 0x9E3779B1 + (i >> 32) * 0xC2B2AE35) & 0xFFFFFFFF
    return _mix((at + torch.repeat_interleave(keys, room)) & 0xFFFFFFFF)


def _plain_decode(codes, e, signed):
    c = codes.int().view(-1, BLOCK)
    low = c & 127 if signed else c
    x = ((low + 8 * e.int()[:, None] - (120 if signed else 248)) << 20).view(torch.float32)
    x = torch.where(low == 0, 0.0, x)
    return (torch.where(c > 127, -x, x) if signed else x).reshape(-1)


def _plain_encode(x, r, signed):
    """Stochastic rounding to the block's codes: r holds 16 random bits per value."""
    bits = x.abs().view(-1, BLOCK).view(torch.int32).long()
    r = r.view(-1, BLOCK)
    e = ((bits.amax(1, keepdim=True) + 0xFFFFF) >> 23).clamp(16 if signed else 32, 255)
    base = 8 * e - (120 if signed else 248)
    c = ((bits + r * 16) >> 20) - base
    least = ((base + 1) << 20).int().view(torch.float32)
    a = x.abs().view(-1, BLOCK)
    low = (a > r.float() / 65536 * least).long() if signed else (a > 0).long()
    c = torch.where(a < least, low, c.clamp(1, 127 if signed else 255))
    if signed:
        c = c + 128 * (x.view(-1, BLOCK) < 0).long()
    return c.to(torch.uint8).reshape(-1), e.to(torch.uint8).reshape(-1)


def _plain_adamw(s):
    bits8, total = s["case"]["bits"] == 8, s["p"].numel()
    room = torch.diff(torch.tensor(s["starts"] + [total])).cuda()
    decay = torch.repeat_interleave(torch.tensor(s["decay"], device="cuda"), room)
    s["state"][0] += 1
    t = s["state"][0].double()
    g = s["g"].float()
    m = _plain_decode(s["m"], s["me"], True) if bits8 else s["m"]
    v = _plain_decode(s["v"], s["ve"], False) if bits8 else s["v"]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    step = m / (torch.sqrt(v) / torch.sqrt(1 - BETA2 ** t) + ADAM_EPS)
    s["p"].copy_(s["p"] * (1 - LR * decay) - LR / (1 - BETA1 ** t) * step)
    if not bits8:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return
    r = _random_bits(s, s["state"][0], total)
    for k, x, part in (("m", m, r >> 16), ("v", v, r & 0xFFFF)):
        codes, e = _plain_encode(x, part, k == "m")
        s[k].copy_(codes)
        s[k + "e"].copy_(e)
        s[k + "_out"].copy_(_plain_decode(codes, e, k == "m"))


def _run_adamw(s):
    bits8, lists = s["case"]["bits"] == 8, s["lists"]
    if own:
        F = _functional()
        F.adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], s["state"], LR, (BETA1, BETA2), ADAM_EPS, s["decay"],
                     seed=s["seed"])
        if bits8:
            F.adamw_moments(lists["m"], lists["v"], out=(lists["m_out"], lists["v_out"]))
    else:
        _plain_adamw(s)
    return {"p": s["p"], "m": s["m_out"], "v": s["v_out"]} if bits8 else {"p": s["p"], "m": s["m"], "v": s["v"]}


def run(state):
    return {"norm": _run_norm, "attn": _run_attn, "adamw": _run_adamw}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------ what a pass cannot do without
def _pairs(case):
    """Query-key pairs of one head over the batch (padded batches: the sum over the evenly spread lengths)."""
    B, tq, tk = case["batch"], case["tq"], case["tk"]
    counts = [tk * (i + (B == 1)) // max(1, B - 1) for i in range(B)] if case["pad"] else [tk] * B
    if not case["causal"]:
        return sum(counts) * tq
    total = 0
    for n in counts:
        first = tk - tq + 1                       # keys that query 0 sees
        rise = max(0, min(tq, n - first))         # queries whose reach still grows below n
        skip = min(rise, max(0, -first))          # of these, queries that see nothing
        total += (rise - skip) * (first + skip + first + rise - 1) // 2 + (tq - rise) * (n if first + tq - 1 >= n else 0)
    return total


def work(case):
    if case["op"] == "norm":
        e, n = (2 if case["dtype"] == "bf16" else 4), case["rows"] * case["dim"]
        arrays = 2 + 2 * case["residual"] + (2 + 2 * case["residual"] if case["train"] else 0)
        return {"bytes": n * e * arrays + 8 * case["dim"] * (2 if case["train"] else 1), "flops": n * (20 if case["train"] else 8)}
    if case["op"] == "attn":
        e, B, H, Hk, d = (2 if case["dtype"] == "bf16" else 4), case["batch"], case["heads"], case["kv_heads"], case["d"]
        nq, nk = B * case["tq"] * H * 2 * d, B * case["tk"] * Hk * 2 * d
        keys = nk * (0.5 if case["pad"] and B > 1 else 1.0)
        if not case["train"]:
            return {"bytes": e * (2 * nq + 2 * keys), "flops": 8 * d * H * _pairs(case)}
        return {"bytes": e * (4 * nq + 2 * keys + 2 * nk), "flops": 28 * d * H * _pairs(case)}
    n = sum(_layout(case)[0])
    g = 2 if case["grad"] == "bf16" else 4
    return {"bytes": n * (8 + g + (16 if case["bits"] == 32 else 8)), "flops": 16 * n}


# ------------------------------------------------------------------------------ 64 bits
def _exact_norm(s):
    x, w, b = (s[k].detach().double() for k in ("x", "w", "b"))
    dim, res = x.shape[1], s["res"]
    total = x if res is None else (x + res.detach().double()).to(s["x"].dtype).double()
    mean = total.sum(1, keepdim=True) / dim
    var = (total - mean).square().sum(1, keepdim=True) / dim
    inv = 1.0 / torch.sqrt(var + EPS)
    xhat = (total - mean) * inv
    out = {"y": xhat * w + b}
    if res is not None:
        out["s"] = total
    if not s["case"]["train"]:
        return out if res is not None else {"y": out["y"], "s": None}
    dy = s["dy"].double()
    out["db"], out["dw"] = dy.sum(0), (dy * xhat).sum(0)
    g = dy * w
    out["dx"] = inv * (g - g.sum(1, keepdim=True) / dim - xhat * (g * xhat).sum(1, keepdim=True) / dim)
    if res is not None:
        out["dx"] = out["dx"] + s["ds"].double()
        out["dres"] = out["dx"]
    return out


def _exact_attn(s):
    c = s["case"]
    q, k, v, lam = (s[n].detach().double() for n in ("q", "k", "v", "lam"))
    B, tq, H, _, d = q.shape
    tk, group = k.shape[1], H // k.shape[2]
    out = {"o": torch.zeros_like(q).view(B, tq, H, 2 * d)}
    if c["train"]:
        out |= {"dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v), "dlam": torch.zeros_like(lam)}
        do = s["do"].double()
    scale = d ** -0.5
    for b in range(B):
        n = tk if s["lengths"] is None else int(s["lengths"][b])
        hide = torch.arange(tk, device=q.device)[None, :].expand(tq, tk) >= n
        if c["causal"]:
            hide = hide | torch.ones(tq, tk, device=q.device, dtype=torch.bool).triu(tk - tq + 1)
        dead = hide.all(1)
        for h in range(H):
            j = h // group
            maps = []
            for half in (0, 1):
                z = (q[b, :, h, half] @ k[b, :, j, half].T * scale).masked_fill(hide, -math.inf)
                z[dead] = 0.0
                p = torch.softmax(z, 1)
                p[dead] = 0.0
                maps.append(p)
            a = maps[0] - lam[h] * maps[1]
            out["o"][b, :, h] = a @ v[b, :, j]
            if not c["train"]:
                continue
            da = do[b, :, h] @ v[b, :, j].T
            out["dv"][b, :, j] += a.T @ do[b, :, h]
            out["dlam"][h] -= (maps[1] * da).sum()
            for half, f in ((0, 1.0), (1, -lam[h])):
                p = maps[half]
                dz = f * p * (da - (p * da).sum(1, keepdim=True)) * scale
                out["dq"][b, :, h, half] = dz @ k[b, :, j, half]
                out["dk"][b, :, j, half] += dz.T @ q[b, :, h, half]
    return out


def _exact_values(codes, e, mant_exp_bits):
    """Values of 8-bit codes in 64 bits: exponent and mantissa taken apart."""
    top = 2 ** mant_exp_bits - 1
    low = (codes.long() & top).view(-1, BLOCK)
    up = e.double()[:, None] - 127 - (top // 8) + (low // 8).double()
    x = torch.where(low == 0, 0.0, torch.exp2(up) * (1 + (low % 8).double() / 8))
    return torch.where(codes.view(-1, BLOCK) > top, -x, x).reshape(-1)


def _exact_round(x, u, reach):
    """x (64 bits) stochastically rounded to three mantissa bits, `reach` binades below its block's largest."""
    a, u = x.abs().view(-1, BLOCK), u.view(-1, BLOCK)
    big = a.amax(1, keepdim=True)
    floor = torch.floor(torch.log2(big.clamp_min(1e-300)))
    top = floor + (big > 1.875 * torch.exp2(floor)).double()
    top = top.clamp_min((16 if reach == 15 else 32) - 127)
    least = 1.125 * torch.exp2(top - reach)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(1e-300))) - 3)
    y = torch.floor(a / step + u) * step
    small = torch.where(a > u * least, least, 0.0) if reach == 15 else torch.where(a > 0, least, 0.0)
    return (torch.where(a < least, small, y) * torch.sign(x.view(-1, BLOCK))).reshape(-1)


def _exact_adamw(s):
    bits8, total = s["case"]["bits"] == 8, s["p"].numel()
    t = int(s["state"][0]) + 1
    g = s["g"].double()
    m = _exact_values(s["m"], s["me"], 7) if bits8 else s["m"].double()
    v = _exact_values(s["v"], s["ve"], 8) if bits8 else s["v"].double()
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g * g - v)
    p = s["p"].double()
    for w, view in zip(s["decay"], _views(p, s["sizes"], s["starts"])):
        view *= 1 - LR * w
    p -= LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
    if not bits8:
        return {"p": p, "m": m, "v": v}
    r = _random_bits(s, torch.tensor(t, device="cuda"), total)
    return {"p": p, "m": _exact_round(m, (r >> 16).double() / 65536, 15), "v": _exact_round(v, (r & 0xFFFF).double() / 65536, 31)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "attn": _exact_attn, "adamw": _exact_adamw}[case["op"]](s)
