"""Differential attention, forward and backward, against the formula in 64 bits: lengths, heads, masks that leave
rows empty, strides, single tokens, refusals.

Tolerances.  f32: sums of up to a few thousand products of values of order one, exponentials of arguments of a few
tens: each probability is off by (|argument| <= 64) f32 half-steps from the argument's rounding and a few from the
sums of d products; 2^-24 * 256 of the sum of the terms' magnitudes bounds every output.  bf16: inputs are exact in
both; each probability (and score gradient) enters the second product rounded by half a step 2^-9 * 2 = u of its
size at most u = 2^-8 (the bound is per element, the sums below add the magnitudes), outputs are rounded once more (u of
the value), delta carries the rounding of the probabilities in the saved maps (u of the sum of |do| |o| terms).  So an output is within
u * (|value| + 2.5 * sum of the magnitudes of its terms), where the terms of dS hold |dP| + |delta| and the rounding
of delta; the factor 2.5 covers probability, delta and score-gradient rounding, one u each being the worst
case of a whole row rounded the same way, at half weight as 2^-8 is twice the half step bf16 has."""
import math

import pytest
import torch

from conftest import load_pkg

BF, F = torch.bfloat16, torch.float32


def oracle(q, k, v, lam, causal, lengths, scale, do=None):
    """Outputs and, per output, the sum of the magnitudes of its terms."""
    q, k, v, lam = (x.detach().double().cpu() for x in (q, k, v, lam))
    B, Tq, H, _, d = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    g = H // Hk
    out = {n: torch.zeros(s, dtype=torch.float64) for n, s in (
        ("o", (B, Tq, H, 2 * d)), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape), ("dlam", lam.shape))}
    mag = {n: torch.zeros_like(x) for n, x in out.items()}
    do = None if do is None else do.detach().double().cpu()
    for b in range(B):
        n = Tk if lengths is None else max(0, min(Tk, int(lengths[b])))
        see = torch.arange(Tk)[None, :].expand(Tq, Tk) < n
        if causal:
            see = see & (torch.arange(Tk)[None, :] <= torch.arange(Tq)[:, None] + (Tk - Tq))
        kb, vb = k[b].clone(), v[b].clone()
        kb[n:], vb[n:] = 0, 0                       # whatever lies behind the length does not count
        for h in range(H):
            j = h // g
            P = []
            for i in (0, 1):
                z = (q[b, :, h, i] @ kb[:, j, i].T * scale).masked_fill(~see, -math.inf)
                top = z.amax(1, keepdim=True)
                e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
                P.append(e / e.sum(1, keepdim=True).clamp_min(1e-300))
            A, M = P[0] - lam[h] * P[1], P[0] + lam[h].abs() * P[1]
            out["o"][b, :, h] = A @ vb[:, j]
            mag["o"][b, :, h] = M @ vb[:, j].abs()
            if do is None:
                continue
            G = do[b, :, h]
            dP = G @ vb[:, j].T
            dPm = G.abs() @ vb[:, j].abs().T
            out["dv"][b, :, j] += A.T @ G
            mag["dv"][b, :, j] += M.T @ G.abs()
            out["dlam"][h] -= (P[1] * dP).sum()
            mag["dlam"][h] += (G.abs() * (P[1] @ vb[:, j].abs())).sum()
            for i, f in ((0, 1.0), (1, -lam[h])):
                delta = (P[i] * dP).sum(1, keepdim=True)
                # delta carries the rounding of the probabilities: |do| . (P_1 + |lam| 2 P_2) |v| in magnitude
                dm = (G.abs() * ((P[0] + lam[h].abs() * 2 * P[1]) @ vb[:, j].abs())).sum(1, keepdim=True)
                dS = f * P[i] * (dP - delta) * scale
                dSm = abs(f) * P[i] * (dP.abs() + dm) * scale
                out["dq"][b, :, h, i] = dS @ kb[:, j, i]
                mag["dq"][b, :, h, i] = dSm @ kb[:, j, i].abs()
                out["dk"][b, :, j, i] += dS.T @ q[b, :, h, i]
                mag["dk"][b, :, j, i] += dSm.T @ q[b, :, h, i].abs()
            del dPm
    return out, mag


def bound(want, mag, dtype):
    if dtype == F:
        return 2.0 ** -24 * 256 * (want.abs() + mag)
    return 2.0 ** -8 * (want.abs() + 2.5 * mag)


def check(got, want, mag, dtype, what):
    got = got.detach().double().cpu()
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    lim = bound(want, mag, dtype) + 1e-30
    err = (got - want).abs()
    assert bool((err <= lim).all()), f"{what}: off by {float((err / lim).max()):.2f} times the bound"
    # and as a whole, where roundings average out: 2-norm within 8 steps of f32 times sqrt-free margin, 1.5 % for bf16
    ref = float(want.norm())
    if ref > 0 and want.numel() > 200:
        assert float((got - want).norm()) <= (2e-5 if dtype == F else 1.5e-2) * ref + 1e-3 * float(lim.norm()), what


def make(B, Tq, Tk, H, Hk, d, dtype, seed=0, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(B, Tq, H, 2, d, generator=g) * spread).to(dtype)
    k = (torch.randn(B, Tk, Hk, 2, d, generator=g) * spread).to(dtype)
    v = torch.randn(B, Tk, Hk, 2 * d, generator=g).to(dtype)
    lam = 0.2 + 0.6 * torch.rand(H, generator=g)
    do = torch.randn(B, Tq, H, 2 * d, generator=g).to(dtype)
    return q, k, v, lam, do


def run(sf, q, k, v, lam, do=None, **kw):
    xs = [t.detach().cuda().requires_grad_(True) for t in (q, k, v, lam)]
    o = sf.functional.diff_attention(*xs, **kw)
    if do is None:
        return o, None
    return o, dict(zip(("dq", "dk", "dv", "dlam"), torch.autograd.grad(o, xs, do.cuda())))


def compare(sf, q, k, v, lam, do, causal=False, lengths=None, scale=None):
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    o, g = run(sf, q, k, v, lam, do, causal=causal, lengths=None if ln is None else ln.cuda(), scale=scale)
    want, mag = oracle(q, k, v, lam, causal, ln, q.shape[-1] ** -0.5 if scale is None else scale, do)
    check(o, want["o"], mag["o"], q.dtype, "o")
    for n in ("dq", "dk", "dv"):
        check(g[n], want[n], mag[n], q.dtype, n)
    check(g["dlam"], want["dlam"], mag["dlam"], q.dtype, "dlam")
    with torch.no_grad():           # the inference call keeps nothing and gives the same bits
        o2 = sf.functional.diff_attention(*(t.cuda() for t in (q, k, v, lam)), causal=causal,
                                          lengths=None if ln is None else ln.cuda(), scale=scale)
    assert torch.equal(o2, o)
    return o, g


SHAPES = [  # B, Tq, Tk, H, Hk, d
    (1, 1, 1, 1, 1, 8), (2, 5, 5, 4, 4, 16), (1, 32, 32, 1, 1, 32), (1, 33, 31, 2, 1, 64), (2, 64, 65, 2, 2, 24),
    (1, 127, 129, 3, 3, 40), (1, 200, 200, 4, 2, 64), (3, 129, 257, 4, 1, 56), (1, 300, 40, 2, 2, 48), (1, 2, 700, 8, 2, 32),
    (1, 31, 513, 1, 1, 64), (2, 1, 300, 6, 3, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF, F])
def test_shapes(shape, causal, dtype):
    compare(load_pkg(), *make(*shape, dtype, seed=sum(shape)), causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(dtype, causal):
    """Every way a length can fall: none, one key, inside a tile, at its edges, all, and out of range."""
    x = make(8, 150, 150, 2, 1, 32, dtype, seed=3)
    compare(load_pkg(), *x, causal=causal, lengths=[0, 1, 31, 32, 33, 64, 150, 149])
    o, g = run(load_pkg(), *x, causal=causal, lengths=torch.tensor([-5, 1000, 150, 2 ** 31 - 1, 0, 0, 0, 150], dtype=torch.int32).cuda())
    o2, g2 = run(load_pkg(), *x, causal=causal, lengths=torch.tensor([0, 150, 150, 150, 0, 0, 0, 150], dtype=torch.int32).cuda())
    assert torch.equal(o, o2) and all(torch.equal(g[n], g2[n]) for n in g)
    assert float(o[0].detach().abs().max()) == 0 and float(g["dk"][0].abs().max()) == 0 and float(g["dq"][4].abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F])
def test_garbage_behind_the_lengths(dtype):
    """NaN and infinities in keys and values that no query may see do not reach any output."""
    sf = load_pkg()
    for Tq, d in ((70, 64), (1, 16)):
        q, k, v, lam, do = make(3, Tq, 200, 4, 2, d, dtype, seed=7)
        lengths = torch.tensor([0, 77, 160], dtype=torch.int32).cuda()
        o, g = run(sf, q, k, v, lam, do, lengths=lengths)
        for b, n in enumerate((0, 77, 160)):
            k[b, n:], v[b, n:] = float("nan"), float("inf")
        o2, g2 = run(sf, q, k, v, lam, do, lengths=lengths)
        assert torch.equal(o, o2)
        for n in g:
            assert torch.equal(g[n], g2[n]), n
        assert float(g2["dk"][1, 77:].abs().max()) == 0 and float(g2["dv"][2, 160:].abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("shape", [(2, 1, 4000, 8, 2, 64), (1, 4, 2049, 2, 1, 16), (1, 40, 3000, 1, 1, 32), (3, 1, 130, 4, 4, 64),
                                   (1, 1, 127, 32, 1, 8), (1, 1, 1000, 33, 1, 24)], ids=str)
def test_few_queries_many_keys(shape, dtype):
    """The key axis is split and joined again; with lengths, whole parts are empty."""
    sf = load_pkg()
    x = make(*shape, dtype, seed=1)
    compare(sf, *x)
    compare(sf, *x, causal=True, lengths=[shape[2] // (3 * b + 1) for b in range(shape[0])])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F])
def test_large_scores(dtype):
    """Scores of hundreds: the running maximum has to follow, rows are decided by one key."""
    q, k, v, lam, do = make(1, 100, 300, 2, 2, 32, dtype, seed=5, spread=1.0)
    k = k * torch.linspace(0.1, 12, 300).view(1, 300, 1, 1, 1).to(dtype)      # later keys score higher
    q = (q * 4).to(dtype)
    # the arguments reach +-1500 here instead of 64: 24 times the rounding of the argument in f32, which is
    # within the bf16 bound (2^-24 * 1500 * 2 < 2^-12) and is taken into account for f32
    ln = None
    o, g = run(load_pkg(), q, k, v, lam, do)
    want, mag = oracle(q, k, v, lam, False, ln, 32 ** -0.5, do)
    for n, x in {"o": o, **g}.items():
        lim = bound(want[n], mag[n], dtype) * (24 if dtype == F else 1) + 1e-30
        assert bool(((x.detach().double().cpu() - want[n]).abs() <= lim).all()), n


@pytest.mark.gpu
@pytest.mark.parametrize("Tq", [1, 40])
def test_scores_near_the_end_of_the_range(Tq):
    """All of a row's scores are hugely negative, or hugely positive: the softmax only knows their differences.  Scores
    of -+ 2^110 and -+ 2^111 exactly: one key takes all, in bf16 and in f32, forward and backward."""
    sf = load_pkg()
    for dtype in (BF, F):
        for sign in (-1.0, 1.0):
            q = torch.zeros(1, Tq, 1, 2, 8)
            k = torch.zeros(1, 300, 1, 2, 8)
            q[..., 0], k[..., 0] = sign * 2.0 ** 55, 2.0 ** 56
            best = 77 if sign < 0 else 211
            k[:, best, :, :, 0] = 2.0 ** 55 if sign < 0 else 2.0 ** 57
            v = torch.randn(1, 300, 1, 16)
            q, k, v = (t.to(dtype) for t in (q, k, v))
            o, g = run(sf, q, k, v, torch.tensor([0.25]), torch.ones(1, Tq, 1, 16).to(dtype), scale=1.0)
            want = (0.75 * v[:, best:best + 1].double()).expand(1, Tq, 1, 16)
            assert bool(((o.detach().double().cpu() - want).abs() <= 2.0 ** -8 * want.abs()).all())
            dv = g["dv"].double().cpu()
            assert bool((dv[:, best] == 0.75 * Tq).all()) and float(dv.abs().sum()) == 0.75 * Tq * 16
            # P is one-hot, so dP - delta is 0 in exact numbers.  In f32 both are sums of the same 16 products dO V, in orders of
            # their own: each is off by at most 16 half steps of 2^-24 of sum |V|, their difference by 32, and two more for
            # its own rounding and its rounding to the operand type (2^-8 of it).  It is multiplied by the key (dq) or, over
            # the Tq rows, by the query (dk).
            off = 34 * 2.0 ** -24 * float(v[0, best].double().abs().sum())
            assert float(g["dq"].abs().max()) <= off * float(k[0, best].double().abs().max())
            assert float(g["dk"].abs().max()) <= off * Tq * float(q.double().abs().max())


@pytest.mark.gpu
def test_lam_zero_one_negative_and_types():
    sf = load_pkg()
    q, k, v, _, do = make(2, 60, 60, 4, 4, 16, BF, seed=2)
    for lam in (torch.zeros(4), torch.ones(4), torch.tensor([-0.5, 0.3, 2.0, 0.0]), torch.tensor([0.5, 0.25, 1.5, -1.0]).to(BF)):
        o, g = run(sf, q, k, v, lam, do)
        want, mag = oracle(q, k, v, lam, False, None, 0.25, do)
        check(o, want["o"], mag["o"], BF, "o")
        check(g["dq"], want["dq"], mag["dq"], BF, "dq")
        assert g["dlam"].dtype == lam.dtype
        check(g["dlam"], want["dlam"], mag["dlam"], BF, "dlam")
    # both maps equal and lam one: nothing is left but the f32 rounding of one of two equal products (|O_i| <= 4 here)
    same = torch.stack([q[:, :, :, 0], q[:, :, :, 0]], 3), torch.stack([k[:, :, :, 0], k[:, :, :, 0]], 3)
    o, _ = run(sf, *same, v, torch.ones(4))
    assert float(o.detach().abs().max()) <= 4 * 2.0 ** -24


@pytest.mark.gpu
def test_scale():
    compare(load_pkg(), *make(1, 50, 50, 2, 2, 24, F, seed=4), scale=0.37)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F])
def test_strides(dtype):
    """Slices of one projection, transposed heads, odd offsets: same bits as contiguous copies."""
    sf = load_pkg()
    B, T, H, d = 2, 77, 4, 16
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(B, T, 3 * H * 2 * d, generator=g).to(dtype).cuda()
    q = qkv[..., :H * 2 * d].view(B, T, H, 2, d)
    k = qkv[..., H * 2 * d:2 * H * 2 * d].view(B, T, H, 2, d)
    v = qkv[..., 2 * H * 2 * d:].view(B, T, H, 2 * d)
    lam = torch.tensor([0.2, 0.4, 0.6, 0.8]).cuda()
    do = torch.randn(B, T, H, 2 * d, generator=g).to(dtype).cuda()
    want = run(sf, q.contiguous(), k.contiguous(), v.contiguous(), lam, do)
    variants = {"slices": (q, k, v),
                "heads first": tuple(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)),
                "halves outside": (q.transpose(3, 4).contiguous().transpose(3, 4), k, v)}
    odd = torch.zeros(qkv.numel() + 1, dtype=dtype, device="cuda")[1:].view(qkv.shape)
    odd.copy_(qkv)
    variants["odd address"] = (odd[..., :H * 2 * d].view(B, T, H, 2, d), k, v)
    for name, (a, b, c) in variants.items():
        xs = [t.requires_grad_(True) if t.is_leaf else t.detach().requires_grad_(True) for t in (a, b, c, lam.clone())]
        xs = [t.detach().as_strided(t.shape, t.stride(), t.storage_offset()).requires_grad_(True) for t in xs]
        o = sf.functional.diff_attention(*xs)
        grads = torch.autograd.grad(o, xs, do)
        assert torch.equal(o, want[0]), name
        for n, x in zip(("dq", "dk", "dv", "dlam"), grads):
            assert torch.equal(x, want[1][n]), (name, n)
    # a shared key / value set expanded over the batch
    e = run(sf, q, k[:1].expand(B, T, H, 2, d).contiguous(), v[:1].expand(B, T, H, 2 * d).contiguous(), lam)[0]
    assert torch.equal(sf.functional.diff_attention(q, k[:1].expand(B, T, H, 2, d), v[:1].expand(B, T, H, 2 * d), lam), e)
    # one token, one sample: strides of axes of length one mean nothing
    one = torch.randn(1, 1, 1, 2, d, device="cuda").to(dtype).as_strided((1, 1, 1, 2, d), (3, 5, 7, d, 1))
    assert torch.equal(sf.functional.diff_attention(one, k[:1, :, :1], v[:1, :, :1], lam[:1]),
                       sf.functional.diff_attention(one.clone(memory_format=torch.contiguous_format), k[:1, :, :1], v[:1, :, :1], lam[:1]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Tq", [1, 300])
def test_offsets_beyond_32_bits(Tq, dtype):
    """Tokens and samples so far apart that their byte offsets pass 2^32 (a long cache): the same bits as packed ones."""
    sf = load_pkg()
    q, k, v, lam, do = (t.cuda() for t in make(2, Tq, 700, 2, 1, 64, dtype, seed=14))
    step = (1 << 22) - 64                               # elements between two tokens, just below what the kernels take

    def far(t, n):
        buf = torch.empty(n, device="cuda", dtype=dtype)
        gap = t.shape[1] * step                         # between the samples
        strides = (gap, step, *t.contiguous().stride()[2:])
        x = buf.as_strided(t.shape, strides)
        x.copy_(t)
        return x
    xs = [far(t, 2 * t.shape[1] * step) for t in (q, k, v)]
    if Tq > 1:
        assert all(t.stride(0) * t.element_size() > 1 << 31 for t in xs)
    assert all(2 * t.shape[1] * step * t.element_size() > 1 << 32 for t in xs[1:])
    assert all(sf.ops.kernel_layout(t) is t for t in xs)
    o, g = run(sf, q, k, v, lam, do, causal=True)
    leaves = [t.requires_grad_(True) for t in (*xs, lam)]
    of = sf.functional.diff_attention(*leaves, causal=True)
    gf = torch.autograd.grad(of, leaves, do)
    assert torch.equal(of, o)
    for x, n in zip(gf, ("dq", "dk", "dv", "dlam")):
        assert torch.equal(x, g[n])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 130, 300, 4, 2, 64), (1, 40, 3000, 1, 1, 32), (2, 1, 300, 6, 3, 8), (2, 700, 700, 2, 1, 16),
                                   (1, 700, 900, 2, 2, 64)], ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_lam_gradient_in_bf16(shape, causal):
    """dlam takes part in no rounding to bf16 but that of the inputs: its sums are of f32 probabilities and f32 dP, so it
    meets the bound of the f32 form."""
    q, k, v, lam, do = make(*shape, BF, seed=15)
    _, g = run(load_pkg(), q, k, v, lam, do, causal=causal)
    want, mag = oracle(q, k, v, lam, causal, None, q.shape[-1] ** -0.5, do)
    check(g["dlam"], want["dlam"], mag["dlam"], F, "dlam")


@pytest.mark.gpu
def test_shared_heads_gradient_is_the_sum():
    """Shared key / value heads against the same call with the heads repeated: gradients add up over the group."""
    sf = load_pkg()
    q, k, v, lam, do = make(2, 90, 110, 6, 2, 32, F, seed=6)
    _, g = run(sf, q, k, v, lam, do)
    _, r = run(sf, q, k.repeat_interleave(3, 2), v.repeat_interleave(3, 2), lam, do)
    _, mag = oracle(q, k, v, lam, False, None, 32 ** -0.5, do)
    for n in ("dk", "dv"):
        s = r[n].double().cpu()
        s = s.view(*s.shape[:2], 2, 3, *s.shape[3:]).sum(3)
        assert bool(((g[n].double().cpu() - s).abs() <= 2 * 2.0 ** -24 * 256 * mag[n] + 1e-30).all()), n


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the 64-bit formula along random directions (h = 1e-5: truncation h^2, cancellation
    1e-16 / h) against the f32 kernel's gradient, 1e-5 of the sum of the magnitudes of its terms."""
    sf = load_pkg()
    q, k, v, lam, do = make(1, 20, 30, 2, 1, 8, F, seed=8)
    ln = torch.tensor([25], dtype=torch.int32)
    _, g = run(sf, q, k, v, lam, do, causal=True, lengths=ln.cuda())
    base = [x.double() for x in (q, k, v, lam)]
    gen = torch.Generator().manual_seed(3)
    h = 1e-5
    for i, n in enumerate(("dq", "dk", "dv", "dlam")):
        e = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + h * e, base[i] - h * e
        f = [float((oracle(*x, True, ln, 8 ** -0.5)[0]["o"] * do.double()).sum()) for x in (up, dn)]
        ana = (g[n].double().cpu() * e).sum()
        assert abs((f[0] - f[1]) / (2 * h) - float(ana)) <= 1e-5 * float((g[n].double().cpu() * e).abs().sum()) + 1e-8, n


@pytest.mark.gpu
def test_empty_axes():
    sf = load_pkg()
    for B, Tq, Tk in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        xs = [torch.zeros(s, device="cuda", requires_grad=True) for s in ((B, Tq, 2, 2, 8), (B, Tk, 1, 2, 8), (B, Tk, 1, 16), (2,))]
        o = sf.functional.diff_attention(*xs)
        assert o.shape == (B, Tq, 2, 16) and (o.numel() == 0 or float(o.detach().abs().max()) == 0)
        o.sum().backward()
        for x in xs:
            assert x.grad.shape == x.shape and (x.numel() == 0 or float(x.grad.abs().max()) == 0)


@pytest.mark.gpu
def test_same_bits_every_time_and_on_another_stream():
    sf = load_pkg()
    for shape in ((2, 300, 300, 4, 2, 64), (4, 1, 2000, 4, 1, 64)):
        x = make(*shape, BF, seed=9)
        o0, g0 = run(sf, *x)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            o1, g1 = run(sf, *x)
        torch.cuda.current_stream().wait_stream(st)
        torch.cuda.synchronize()
        assert torch.equal(o0, o1) and all(torch.equal(g0[n], g1[n]) for n in g0)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 130, 130, 4, 2, 32), (2, 1, 3000, 4, 2, 64)], ids=str)
def test_captured_forward_replays(shape):
    """With changing inputs and lengths between the replays; two graphs on one set of inputs do not share a workspace."""
    sf = load_pkg()
    q, k, v, lam, _ = (t.cuda() for t in make(*shape, BF, seed=10))
    lengths = torch.full((2,), shape[2], dtype=torch.int32, device="cuda")
    sf.functional.diff_attention(q, k, v, lam, lengths=lengths)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sf.functional.diff_attention(q, k, v, lam, lengths=lengths))
        graphs.append(g)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        lengths.copy_(torch.tensor([shape[2] // (i + 1), i * 7], dtype=torch.int32))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        want = sf.functional.diff_attention(q, k, v, lam, lengths=lengths)
        assert torch.equal(outs[i % 2], want)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 100, 100, 4, 2, 64), (1, 260, 300, 2, 2, 16)], ids=str)
def test_captured_training_pass_replays(shape):
    """Forward and backward in one graph, replayed with other inputs, against the eager pass."""
    sf = load_pkg()
    for dtype in (BF, F):
        q, k, v, lam, do = (t.cuda() for t in make(*shape, dtype, seed=12))

        def passes():
            xs = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
            o = sf.functional.diff_attention(*xs, causal=True)
            return (o.detach(), *torch.autograd.grad(o, xs, do))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            passes()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = passes()
        for i in range(4):
            for t in (q, k, v, do):
                t.copy_(torch.randn_like(t) * (1 + i))
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(got, passes()):
                assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F])
def test_saved_tensors_in_another_layout(dtype):
    """Slices of one projection, saved on the host meanwhile: what comes back for the backward pass is contiguous, and
    the gradients have the same bits."""
    sf = load_pkg()
    x = torch.randn(2, 70, 3 * 2 * 32, device="cuda").to(dtype)
    lam, do = torch.tensor([0.3, 0.6], device="cuda"), torch.randn(2, 70, 2, 32, device="cuda").to(dtype)

    def grads():
        leaf = x.clone().requires_grad_(True)
        q, k, v = (t.view(2, 70, 2, 32) for t in leaf.split(64, -1))
        q, k = q.view(2, 70, 2, 2, 16), k.view(2, 70, 2, 2, 16)
        assert all(sf.ops.kernel_layout(t) is t and not t.is_contiguous() for t in (q, k, v))
        return torch.autograd.grad(sf.functional.diff_attention(q, k, v, lam, causal=True), leaf, do)[0]
    want = grads()
    with torch.autograd.graph.save_on_cpu():
        assert torch.equal(grads(), want)


@pytest.mark.gpu
def test_second_derivative_is_refused():
    sf = load_pkg()
    q, k, v, lam, do = (t.cuda() for t in make(1, 9, 9, 1, 1, 8, F))
    q.requires_grad_(True)
    g, = torch.autograd.grad(sf.functional.diff_attention(q, k, v, lam), q, do, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q)


def test_refusals():
    sf = load_pkg()
    with pytest.raises(RuntimeError, match="GPU"):
        sf.functional.diff_attention(torch.zeros(1, 2, 1, 2, 8), torch.zeros(1, 2, 1, 2, 8), torch.zeros(1, 2, 1, 16), torch.zeros(1))


def test_library_refusals():
    """Bad descriptors and pointers are turned away before anything is launched (no GPU needed)."""
    import ctypes
    sf = load_pkg()
    L, D = sf.ops.lib(), sf.ops.DiffAttnDesc
    ll3 = ctypes.c_longlong * 3

    def desc(**kw):
        f = dict(dtype=1, lam_dtype=0, B=1, Tq=4, Tk=4, H=2, Hk=1, d=16, causal=0, scale=0.25, q=(256, 64, 32), k=(128, 32, 32), v=(128, 32, 32))
        f.update(kw)
        return D(f["dtype"], f["lam_dtype"], f["B"], f["Tq"], f["Tk"], f["H"], f["Hk"], f["d"], f["causal"], f["scale"],
                 ll3(*f["q"]), ll3(*f["k"]), ll3(*f["v"]))
    a = ctypes.c_void_p(4096)

    def fwd(d, q=a, lam=a, maps=None, lse=None, ws=None, nbytes=0):
        return L.sf_diff_attn_fwd(ctypes.byref(d), q, a, a, lam, None, a, maps, lse, ws, ctypes.c_size_t(nbytes), None)
    for bad in (dict(dtype=2), dict(lam_dtype=5), dict(B=0), dict(Tq=0), dict(Tk=0), dict(H=3, Hk=2), dict(Hk=0), dict(d=12), dict(d=72),
                dict(d=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(q=(256, 68, 32)), dict(k=(128, 16, 32)),
                dict(v=(128, 1 << 22, 32)), dict(q=(-256, 64, 32)), dict(Tq=(1 << 24) + 1)):
        assert fwd(desc(**bad)) == -22, bad
        assert int(L.sf_diff_attn_fwd_workspace_bytes(ctypes.byref(desc(**bad)))) == 0
    assert fwd(desc(), q=ctypes.c_void_p(4104)) == -22 and fwd(desc(), q=None) == -22
    assert fwd(desc(), lam=None) == -22 and fwd(desc(), maps=a) == -22 and fwd(desc(), lse=a) == -22
    long = desc(Tq=1, Tk=4000)
    need = int(L.sf_diff_attn_fwd_workspace_bytes(ctypes.byref(long)))
    assert need > 0 and fwd(long) == -22 and fwd(long, ws=a, nbytes=need - 1) == -22
    nb = int(L.sf_diff_attn_bwd_workspace_bytes(ctypes.byref(desc())))
    assert nb >= 1 * 2 * 4 * 16

    def bwd(ws=a, n=nb, do=a):
        return L.sf_diff_attn_bwd(ctypes.byref(desc()), a, a, a, a, None, a, a, do, a, a, a, a, ws, ctypes.c_size_t(n), None)
    assert bwd(ws=None) == -22 and bwd(n=nb - 1) == -22 and bwd(do=None) == -22
    # more work than one launch has threads for
    for many in (dict(B=1 << 23, H=4, Hk=2), dict(B=1 << 10, Tk=1 << 20), dict(B=1 << 12, H=8, Hk=1, Tq=1 << 16)):
        assert fwd(desc(**many)) == -22, many
    wide = desc(B=1 << 21, H=1, Hk=1)
    assert int(L.sf_diff_attn_bwd_workspace_bytes(ctypes.byref(wide))) == 0


@pytest.mark.gpu
def test_gpu_refusals():
    sf = load_pkg()
    att = sf.functional.diff_attention
    z = lambda *s, dt=F: torch.zeros(*s, device="cuda", dtype=dt)
    q, k, v, lam = z(2, 3, 4, 2, 8), z(2, 5, 2, 2, 8), z(2, 5, 2, 16), z(4)
    att(q, k, v, lam)
    with pytest.raises(TypeError):
        att(q, k.bfloat16(), v, lam)
    with pytest.raises(TypeError):
        att(q.half(), k.half(), v.half(), lam)
    with pytest.raises(TypeError):
        att(q, k, v, lam.double())
    with pytest.raises(RuntimeError, match="fit"):
        att(q, k[:1], v, lam)
    with pytest.raises(RuntimeError, match="fit"):
        att(q, k, v[:, :4], lam)
    with pytest.raises(RuntimeError, match="fit"):
        att(q, z(2, 5, 3, 2, 8), z(2, 5, 3, 16), lam)
    with pytest.raises(RuntimeError, match="lam"):
        att(q, k, v, lam[:2])
    with pytest.raises(NotImplementedError):
        att(z(2, 3, 4, 2, 12), z(2, 5, 2, 2, 12), z(2, 5, 2, 24), lam)
    with pytest.raises(NotImplementedError):
        att(z(2, 3, 4, 2, 72), z(2, 5, 2, 2, 72), z(2, 5, 2, 144), lam)
    with pytest.raises(RuntimeError, match="lengths"):
        att(q, k, v, lam, lengths=torch.zeros(2, device="cuda", dtype=torch.int64))
    with pytest.raises(RuntimeError, match="lengths"):
        att(q, k, v, lam, lengths=torch.zeros(3, device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError, match="device"):
        att(q, k, v, lam, lengths=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="scale"):
        att(q, k, v, lam, scale=-1.0)
    with pytest.raises(RuntimeError, match="q \\["):
        att(q[0], k, v, lam)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F])
def test_gradients_at_any_address(dtype):
    """A contiguous gradient that starts between two 16-byte pieces (a slice of a flat buffer, what the backward pass of a concatenation
    hands over) and saved tensors that come back at such an address: the same bits."""
    sf = load_pkg()
    x = make(2, 33, 50, 4, 2, 16, dtype, seed=16)
    want = run(sf, *x)[1]
    leaves = [t.cuda().requires_grad_(True) for t in x[:4]]
    do = x[4].cuda()

    def odd(t):
        buf = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
        view = buf[1:].view(t.shape)
        view.copy_(t)
        return view
    assert odd(do).is_contiguous() and odd(do).data_ptr() % 16
    got = torch.autograd.grad(sf.functional.diff_attention(*leaves), leaves, odd(do))
    assert all(torch.equal(a, want[n]) for a, n in zip(got, ("dq", "dk", "dv", "dlam")))
    flat = torch.cat([torch.zeros(3, dtype=dtype, device="cuda"), sf.functional.diff_attention(*leaves).flatten()])
    got = torch.autograd.grad(flat, leaves, torch.cat([torch.zeros(3, dtype=dtype, device="cuda"), do.flatten()]))
    assert all(torch.equal(a, want[n]) for a, n in zip(got, ("dq", "dk", "dv", "dlam")))
    with torch.autograd.graph.saved_tensors_hooks(odd, lambda t: t):
        got = torch.autograd.grad(sf.functional.diff_attention(*leaves), leaves, do)
    assert all(torch.equal(a, want[n]) for a, n in zip(got, ("dq", "dk", "dv", "dlam")))


def oracle_on_gpu(q, k, v, lam, causal, lengths, scale, do):
    """oracle() with the heads of a sample at once, in 64 bits on the GPU: outputs and the sums of their terms' magnitudes."""
    q, k, v, lam, do = (x.detach().double().cuda() for x in (q, k, v, lam, do))
    B, Tq, H, _, d = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    g = H // Hk
    out = {n: torch.zeros(s, dtype=torch.float64, device="cuda") for n, s in (
        ("o", (B, Tq, H, 2 * d)), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape), ("dlam", lam.shape))}
    mag = {n: torch.zeros_like(x) for n, x in out.items()}
    key = torch.arange(Tk, device="cuda")
    w = lam.view(H, 1, 1)

    def shared(x):          # gradients of the group's heads add up in their key / value head
        return x.view(Hk, g, *x.shape[1:]).sum(1).transpose(0, 1)
    for b in range(B):
        n = Tk if lengths is None else max(0, min(Tk, int(lengths[b])))
        hide = (key[None, :] >= n).expand(Tq, Tk)
        if causal:
            hide = hide | (key[None, :] > torch.arange(Tq, device="cuda")[:, None] + (Tk - Tq))
        live = (key < n).double()
        kb = (k[b] * live.view(Tk, 1, 1, 1)).permute(1, 2, 0, 3).repeat_interleave(g, 0)        # [H, 2, Tk, d]
        vb = (v[b] * live.view(Tk, 1, 1)).transpose(0, 1).repeat_interleave(g, 0)               # [H, Tk, 2 d]
        qb, G = q[b].permute(1, 2, 0, 3), do[b].transpose(0, 1)                                 # [H, 2, Tq, d], [H, Tq, 2 d]
        z = (qb @ kb.transpose(-1, -2).contiguous() * scale).masked_fill(hide, -math.inf)
        top = z.amax(-1, keepdim=True)
        e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
        P = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
        A, M = P[:, 0] - w * P[:, 1], P[:, 0] + w.abs() * P[:, 1]
        va, Ga = vb.abs(), G.abs()
        out["o"][b], mag["o"][b] = (A @ vb).transpose(0, 1), (M @ va).transpose(0, 1)
        dP, dPm = G @ vb.transpose(-1, -2).contiguous(), G.abs()
        out["dv"][b] = shared(A.transpose(-1, -2).contiguous() @ G)
        mag["dv"][b] = shared(M.transpose(-1, -2).contiguous() @ Ga)
        out["dlam"] -= (P[:, 1] * dP).sum((1, 2))
        mag["dlam"] += (dPm * (P[:, 1] @ va)).sum((1, 2))
        dm = (Ga * ((P[:, 0] + w.abs() * 2 * P[:, 1]) @ va)).sum(-1, keepdim=True)
        for i, f in ((0, torch.ones_like(w)), (1, -w)):
            delta = (P[:, i] * dP).sum(-1, keepdim=True)
            dS = f * P[:, i] * (dP - delta) * scale
            dSm = f.abs() * P[:, i] * (dP.abs() + dm) * scale
            out["dq"][b, :, :, i], mag["dq"][b, :, :, i] = (dS @ kb[:, i]).transpose(0, 1), (dSm @ kb[:, i].abs()).transpose(0, 1)
            out["dk"][b, :, :, i] = shared(dS.transpose(-1, -2).contiguous() @ qb[:, i])
            mag["dk"][b, :, :, i] = shared(dSm.transpose(-1, -2).contiguous() @ qb[:, i].abs())
    return out, mag


def within_terms(sf, q, k, v, lam, do, causal=False, lengths=None):
    """Every output of a forward and backward pass within the bound of its terms; returns the passes' outputs."""
    o, g = run(sf, q, k, v, lam, do, causal=causal, lengths=lengths)
    want, mag = oracle_on_gpu(q, k, v, lam, causal, lengths, q.shape[-1] ** -0.5, do)
    for n, x in {"o": o, **g}.items():
        err, lim = (x.detach().double() - want[n]).abs(), bound(want[n], mag[n], q.dtype) + 1e-30
        assert bool((err <= lim).all()), f"{n}: off by {float((err / lim).max()):.3g} times the bound"     # (NaN fails too)
    return o, g


@pytest.mark.gpu
@pytest.mark.parametrize("power", [8, 13, 20, 24, 27, 33, 100])
@pytest.mark.parametrize("d", [8, 32, 64])
@pytest.mark.parametrize("dtype", [BF, F])
def test_finite_scores_of_any_size(power, d, dtype):
    """Scores of about 2.25 * 2^power, positive in the first map and negative in the second, that differ by 0 to 12 small
    steps: the softmax only knows the differences.  Ties for the largest lie in different tiles and parts.  The scores are exact
    in f32: two products, one of two numbers of two bits, the other step n, the sum of at most 24 bits since a step is at least
    2^(power - 22).  Queries are larger and smaller by powers of two, so rows of all sizes share a wave, down to a zero one whose
    scores are the steps alone.  In the second form the scores climb by a factor 2^15 along the keys.
    Bounds as for other scores: an exponent is a difference of scores times the scale in two roundings, 2^-23 of itself, and
    a probability 2^-x has at most 2^-x x 2^-23 <= 2^-23 of an error from it (x 2^-x < 1), below the 2^-24 * 256 of its terms."""
    sf = load_pkg()
    e = power // 2
    for (B, Tq, Tk, H, Hk), causal, lengths in (((2, 70, 300, 2, 1), True, [300, 77]), ((1, 1, 4000, 2, 2), False, None),
                                                ((1, 300, 300, 2, 2), False, None), ((16, 260, 260, 8, 8), False, None)):
        for climb in (False, True):
            q, k, v, lam, do = make(B, Tq, Tk, H, Hk, d, F, seed=power + d)
            gen = torch.Generator().manual_seed(power)
            q.zero_()
            k.zero_()
            size = torch.tensor([1.0, 2.0 ** -4, 2.0 ** -8, 0.0])[torch.arange(Tq) % 4].view(1, Tq, 1)
            n = torch.randint(0, 13, (B, Tk, Hk, 2), generator=gen).float()
            n[:, [3, Tk // 2, Tk - 1]] = 0
            rise = torch.ldexp(torch.ones(Tk), (torch.arange(Tk) * 16 // Tk if climb else torch.full((Tk,), 15)) - 15).view(1, Tk, 1)
            for i, sign in ((0, 1.0), (1, -1.0)):
                q[..., i, 0], q[..., i, 1] = sign * 1.5 * 2.0 ** e * size, 1.0
                k[..., i, 0], k[..., i, 1] = 1.5 * 2.0 ** (power - e) * rise, -n[..., i] * 2.0 ** max(0, power - 22)
            ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
            within_terms(sf, *(t.to(dtype) for t in (q, k, v)), lam, do.to(dtype), causal, ln)


# Shapes whose work items are more than one round of the chip and whose last ones are cut into parts (forward or query
# gradients: by rows and by keys; key gradients: by keys and by rows), and causal ones of more than 512 items, every other 256 of
# which are taken in reverse.  (B, Tq, Tk, H, Hk, d, causal)
MANY = [(16, 775, 1191, 8, 2, 8, False), (33, 48, 231, 16, 16, 24, False), (33, 86, 720, 16, 8, 64, False), (33, 17, 1517, 16, 16, 64, False),
        (33, 24, 1626, 16, 8, 8, False), (33, 652, 699, 4, 4, 8, False), (64, 1527, 398, 4, 1, 8, False), (33, 350, 130, 16, 8, 64, False),
        (33, 98, 98, 16, 16, 8, True), (33, 70, 1773, 16, 2, 8, True), (33, 133, 866, 16, 2, 64, True), (33, 202, 1444, 8, 4, 24, True),
        (33, 399, 399, 4, 4, 24, True), (64, 39, 1219, 8, 1, 64, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", MANY, ids=str)
@pytest.mark.parametrize("dtype", [BF, F])
def test_many_items(shape, dtype):
    *sizes, causal = shape
    B, Tk = shape[0], shape[2]
    x = make(*sizes, dtype, seed=21)
    within_terms(load_pkg(), *x, causal=causal)
    lengths = (torch.arange(B) * 37 % (Tk + 1)).to(torch.int32).cuda()
    lengths[-1] = Tk
    within_terms(load_pkg(), *x, causal=causal, lengths=lengths)


def test_plans_of_many_items():
    """The shapes above reach what they are for: a cut forward pass has a workspace, and a cut backward pass one
    beyond its statistics (no GPU needed)."""
    import ctypes
    sf = load_pkg()
    L, D = sf.ops.lib(), sf.ops.DiffAttnDesc
    cut = {"fwd": 0, "bwd": 0}
    for B, Tq, Tk, H, Hk, d, causal in MANY:
        for code in (0, 1):
            ll3 = ctypes.c_longlong * 3
            w = 2 * d
            desc = D(code, 0, B, Tq, Tk, H, Hk, d, int(causal), 0.25, ll3(Tq * H * w, H * w, w), ll3(Tk * Hk * w, Hk * w, w),
                     ll3(Tk * Hk * w, Hk * w, w))
            least = B * H * ((Tq + 127) // 128 * 128) * 9 * 4       # nine values of a row
            cut["fwd"] += int(L.sf_diff_attn_fwd_workspace_bytes(ctypes.byref(desc))) > 0
            cut["bwd"] += int(L.sf_diff_attn_bwd_workspace_bytes(ctypes.byref(desc))) > least
    assert cut["fwd"] >= 8 and cut["bwd"] >= 16, cut


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("scale", [2e-38, 1e-30, 1e-6, 1e4, 1e12, 1e25])
def test_any_scale(scale, dtype):
    """The smallest scales leave all probabilities equal, the largest decide every row by one key; rows without a key among the others (more
    queries than keys, causal; an empty sample).  Scores are sums of 8 products of values of order one: two keys of a row
    whose scores differ by less than the rounding of these sums, 2^-21 or so, would be told apart in 64 bits alone; values of
    few bits make the scores exact instead.  Bounds as in the module's docstring, exponents being differences of scores times
    the scale (2^-23 of themselves)."""
    sf = load_pkg()
    for B, Tq, Tk, H, Hk in ((2, 150, 70, 2, 1), (2, 40, 300, 4, 2), (2, 1, 3000, 2, 2)):
        q, k, v, lam, do = make(B, Tq, Tk, H, Hk, 8, F, seed=31)
        q, k = (torch.round(t * 4) / 4 for t in (q, k))
        lengths = torch.tensor([Tk, 0], dtype=torch.int32, device="cuda")
        for ln in (None, lengths):
            xs = [t.to(dtype) for t in (q, k, v)]
            o, g = run(sf, *xs, lam, do.to(dtype), causal=True, lengths=ln, scale=scale)
            want, mag = oracle_on_gpu(*xs, lam, True, ln, scale, do.to(dtype))
            for n, x in {"o": o, **g}.items():
                err, lim = (x.detach().double() - want[n]).abs(), bound(want[n], mag[n], dtype) + 1e-30
                assert bool((err <= lim).all()), (n, float((err / lim).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F])
def test_rows_without_keys_beside_far_ones(dtype):
    """Queries that see no key share waves with queries whose scores are of the order of 2^33."""
    sf = load_pkg()
    for d in (8, 64):
        q, k, v, lam, do = make(2, 150, 70, 2, 1, d, F, seed=33)
        q.zero_()
        k.zero_()
        q[..., 0], k[..., 0] = 1.5 * 2.0 ** 16, 1.5 * 2.0 ** 17
        q[..., 1], k[..., 1] = 1.0, -2048.0 * torch.randint(0, 3, k.shape[:-1], generator=torch.Generator().manual_seed(1))
        within_terms(sf, *(t.to(dtype) for t in (q, k, v)), lam, do.to(dtype), True, torch.tensor([70, 33], dtype=torch.int32, device="cuda"))
