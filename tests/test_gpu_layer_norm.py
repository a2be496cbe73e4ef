"""LayerNorm over the last axis (forward, fused residual add, backward with the weight gradients) against
the formula in 64 bits and against differences; shapes, alignments and refusals.

Tolerances.  u = eps(type) / 2 is half a step of the output's type.  An output value is rounded once
from f32 (u of its own size); before that it is a handful of f32 operations on sums of D values, whose
pairwise order keeps the error of a mean below a few f32 steps of the row's largest term: 16 f32 steps of
the largest magnitude of the row's terms cover the chain.  dw and db are f32 sums over the rows: every
partial sum is rounded to f32, (64 + sqrt(rows)) steps of the sum of magnitudes / sqrt(rows) bound a random walk of
them with room to spare; the bound used is rows-independent in the worst case: 2^-24 * 64 * sum |terms|."""
import math

import pytest
import torch

from conftest import load_pkg

BF, F = torch.bfloat16, torch.float32
U32 = torch.finfo(F).eps / 2


def oracle(x, res, w, b, eps, dy=None, ds=None):
    """The formula in 64 bits; s is rounded to the inputs' type, as the operator defines it."""
    s = x.double() if res is None else (x.double() + res.double()).to(x.dtype).double()
    D = s.shape[-1]
    mean = s.mean(-1, keepdim=True)
    var = (s - mean).square().mean(-1, keepdim=True)
    r = (var + eps).rsqrt()
    xh = (s - mean) * r
    wd = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    bd = torch.zeros(D, dtype=torch.float64) if b is None else b.double()
    out = {"y": xh * wd + bd, "s": s, "xh": xh, "r": r}
    if dy is not None:
        g = dy.double() * wd
        dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        out["dx"] = dx if ds is None else dx + ds.double()
        # the size of the terms dx is made of (for the tolerance: they cancel)
        out["dx_terms"] = r * (g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
        if ds is not None:
            out["dx_terms"] = out["dx_terms"] + ds.double().abs()
        red = tuple(range(dy.dim() - 1))
        out["dw"], out["dw_mag"] = (dy.double() * xh).sum(red), (dy.double() * xh).abs().sum(red)
        out["db"], out["db_mag"] = dy.double().sum(red), dy.double().abs().sum(red)
    return out


def check(got, want, bound, what):
    err = (got.detach().double().cpu() - want).abs()
    assert bool((err <= bound).all()), f"{what}: off by {float((err / bound.clamp_min(1e-300)).max()):.2f} times the bound"


def tol(want, terms, dtype):
    """Half a step of the output's type, 1 % more for the double rounding, and 16 f32 steps of the row's terms.  The
    centred values inherit the rounding of the mean: the row's largest magnitude over its spread."""
    return want.abs() * (torch.finfo(dtype).eps / 2) * 1.01 + 16 * U32 * terms


def make(rows, D, dtype, residual, seed, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, D, generator=g) + offset).to(dtype)
    res = torch.randn(rows, D, generator=g).to(dtype) if residual else None
    w, b = 1 + 0.3 * torch.randn(D, generator=g), 0.3 * torch.randn(D, generator=g)
    dy = torch.randn(rows, D, generator=g).to(dtype)
    ds = torch.randn(rows, D, generator=g).to(dtype) if residual else None
    return x, res, w, b, dy, ds


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def run(sf, x, res, w, b, dy, ds, eps=1e-5):
    xs = [None if t is None else t.detach().clone().requires_grad_(True) for t in cuda(x, res, w, b)]
    out = sf.functional.layer_norm(xs[0], xs[2], xs[3], eps, residual=xs[1])
    outs = list(out) if res is not None else [out]
    live = [t for t in xs if t is not None]
    grads = torch.autograd.grad(outs, live, cuda(dy, ds)[:len(outs)])
    by = dict(zip([n for n, t in zip(("dx", "dres", "dw", "db"), xs) if t is not None], grads))
    return outs[0], (outs[1] if res is not None else None), by


def compare(sf, x, res, w, b, dy, ds, eps=1e-5):
    y, s, g = run(sf, x, res, w, b, dy, ds, eps)
    o = oracle(x, res, w, b, eps, dy, ds)
    big = o["s"].abs().amax(-1, keepdim=True) * o["r"] + 1      # rounding of the mean, in units of the spread
    wd = 1.0 if w is None else w.double().abs()
    bd = 0.0 if b is None else b.double().abs()
    check(y, o["y"], tol(o["y"], big * wd + o["xh"].abs() * wd + bd, x.dtype), "y")
    if res is not None:
        assert torch.equal(s.cpu().double(), o["s"]), "the sum is one rounding of x + residual"
        assert torch.equal(g["dx"], g["dres"])
    # an error of `big` steps in xh enters dx through the projection on xh
    check(g["dx"], o["dx"], tol(o["dx"], o["dx_terms"] * (1 + big), x.dtype), "dx")
    rows = x.shape[0]
    if "dw" in g:
        check(g["dw"], o["dw"], 64 * U32 * (o["dw_mag"] + (dy.double().abs() * big).sum(0)), "dw")
    if "db" in g:
        check(g["db"], o["db"], 64 * U32 * o["db_mag"] + 1e-300, "db")
    assert y.dtype == x.dtype and g["dx"].dtype == x.dtype and rows == y.shape[0]


# widths around every change of layout: below one piece, pieces that end inside the row, one lane group to the
# next, a wave's registers to a workgroup's, beyond a workgroup's registers
WIDTHS = [1, 3, 7, 8, 9, 64, 65, 128, 129, 255, 257, 513, 768, 1000, 1024, 1100, 1300, 1536, 2047, 2049, 4095, 4096, 5000, 6144, 8192, 8195]


@pytest.mark.gpu
@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype,residual", [(BF, True), (BF, False), (F, True), (F, False)])
def test_widths(D, dtype, residual):
    compare(load_pkg(), *make(37, D, dtype, residual, seed=D))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 31, 33, 1025, 20011])
@pytest.mark.parametrize("dtype", [BF, F])
def test_row_counts(rows, dtype):
    compare(load_pkg(), *make(rows, 72, dtype, True, seed=rows))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F])
def test_rows_far_from_zero(dtype):
    compare(load_pkg(), *make(64, 200, dtype, False, seed=5, offset=100.0))


@pytest.mark.gpu
def test_constant_rows_and_no_affine():
    sf = load_pkg()
    x, _, _, _, dy, _ = make(6, 96, F, False, seed=3)
    x[2] = 4.0                       # no spread: the output is the bias, the gradient finite
    compare(sf, x, None, None, None, dy, None)
    w = torch.full((96,), 2.0)
    compare(sf, x, None, w, None, dy, None)
    compare(sf, x, None, None, w, dy, None)


@pytest.mark.gpu
def test_offset_views_and_strides():
    """Buffers that start at an odd element, transposed and sliced inputs, expanded gradients."""
    sf = load_pkg()
    for dtype in (BF, F):
        x, res, w, b, dy, ds = make(50, 130, dtype, True, seed=9)
        buf = torch.zeros(50 * 130 + 1, dtype=dtype, device="cuda")
        xv = buf[1:].view(50, 130)
        xv.copy_(x)
        wb = torch.zeros(131, device="cuda")
        wv = wb[1:]
        wv.copy_(w)
        y0, s0 = sf.functional.layer_norm(x.cuda(), w.cuda(), b.cuda(), residual=res.cuda())
        y1, s1 = sf.functional.layer_norm(xv, wv, b.cuda(), residual=res.cuda().t().contiguous().t())
        assert torch.equal(y0, y1) and torch.equal(s0, s1)
        xg = x.cuda().requires_grad_(True)
        y = sf.functional.layer_norm(xg, w.cuda(), b.cuda())
        y.sum().backward()               # an expanded gradient
        o = oracle(x, None, w, b, 1e-5, torch.ones_like(dy))
        check(xg.grad, o["dx"], tol(o["dx"], o["dx_terms"] * 8, dtype), "dx")


@pytest.mark.gpu
def test_only_one_output_used():
    sf = load_pkg()
    x, res, w, b, dy, ds = make(20, 40, F, True, seed=2)
    xs = [t.cuda().requires_grad_(True) for t in (x, res, w, b)]
    y, s = sf.functional.layer_norm(xs[0], xs[2], xs[3], residual=xs[1])
    g = torch.autograd.grad(s, xs[:2], ds.cuda(), retain_graph=True)
    assert torch.equal(g[0].cpu(), ds) and torch.equal(g[1].cpu(), ds)
    g = torch.autograd.grad(y, xs, dy.cuda())
    o = oracle(x, res, w, b, 1e-5, dy)
    check(g[0], o["dx"], tol(o["dx"], o["dx_terms"] * 8, F), "dx without a gradient at the sum")


@pytest.mark.gpu
def test_gradient_against_differences():
    """f(x + h e) - f(x - h e) over 2 h of the 64-bit formula, along random directions: the analytic gradient
    of the kernel agrees to the differences' own error (h^2 of a smooth function, f32 values of the gradient)."""
    sf = load_pkg()
    x, res, w, b, dy, ds = make(5, 24, F, True, seed=11)
    _, _, g = run(sf, x, res, w, b, dy, ds)

    def f(x, res, w, b):
        o = oracle(x, None, w, b, 1e-5)
        return (o["y"] * dy.double()).sum() + (o["s"] * ds.double()).sum()
    gen = torch.Generator().manual_seed(1)
    h = 1e-5
    base = (x.double() + res.double(), w.double(), b.double())
    for k, name in enumerate(("dx", "dw", "db")):
        e = torch.randn(base[k].shape, generator=gen, dtype=torch.float64)
        up, dn = [list(base) for _ in range(2)]
        up[k], dn[k] = base[k] + h * e, base[k] - h * e
        num = (f(up[0], None, up[1], up[2]) - f(dn[0], None, dn[1], dn[2])) / (2 * h)
        ana = (g[name].double().cpu() * e).sum()
        scale = (g[name].double().cpu() * e).abs().sum()
        assert abs(float(num - ana)) <= 1e-5 * float(scale), name


@pytest.mark.gpu
def test_non_finite_rows_stay_apart():
    sf = load_pkg()
    x, _, w, b, dy, _ = make(9, 100, F, False, seed=4)
    ref = sf.functional.layer_norm(x.cuda(), w.cuda(), b.cuda())
    x[3, 7], x[5, 1] = float("nan"), float("inf")
    y = sf.functional.layer_norm(x.cuda(), w.cuda(), b.cuda())
    keep = [0, 1, 2, 4, 6, 7, 8]
    assert torch.equal(y[keep], ref[keep])
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[5]).all())


@pytest.mark.gpu
def test_empty_batch():
    sf = load_pkg()
    x = torch.zeros(0, 5, 32, device="cuda", requires_grad=True)
    w = torch.ones(32, device="cuda", requires_grad=True)
    y = sf.functional.layer_norm(x, w, None)
    assert y.shape == (0, 5, 32)
    y.sum().backward()
    assert x.grad.shape == x.shape and float(w.grad.abs().sum()) == 0.0


@pytest.mark.gpu
def test_same_bits_every_time_and_on_another_stream():
    sf = load_pkg()
    args = make(3000, 320, BF, True, seed=8)
    y0, s0, g0 = run(sf, *args)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y1, s1, g1 = run(sf, *args)
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    assert torch.equal(y0, y1) and torch.equal(s0, s1)
    for k in g0:
        assert torch.equal(g0[k], g1[k]), k


@pytest.mark.gpu
def test_captured_forward_replays():
    sf = load_pkg()
    x, res, w, b, _, _ = cuda(*make(640, 128, BF, True, seed=6))
    sf.functional.layer_norm(x, w, b, residual=res)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, s = sf.functional.layer_norm(x, w, b, residual=res)
    for k in range(4):
        x.copy_(torch.randn(640, 128, device="cuda") + k)
        graph.replay()
        torch.cuda.synchronize()
        ye, se = sf.functional.layer_norm(x, w, b, residual=res)
        assert torch.equal(y, ye) and torch.equal(s, se)


@pytest.mark.gpu
def test_module_follows_autocast_and_matches_torch_keys():
    sf = load_pkg()
    m, t = sf.LayerNorm(48).cuda(), torch.nn.LayerNorm(48).cuda()
    assert list(m.state_dict()) == list(t.state_dict())
    x = torch.randn(4, 6, 48, device="cuda")
    with torch.no_grad():
        m.weight.normal_()
        m.bias.normal_()
    t.load_state_dict(m.state_dict())
    o = oracle(x.cpu(), None, m.weight.detach().cpu(), m.bias.detach().cpu(), 1e-5)
    check(m(x), o["y"], 64 * U32 * (1 + o["y"].abs() + m.weight.detach().cpu().double().abs() * 8), "module")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y, s = m(x, residual=x)
    assert y.dtype == BF and s.dtype == BF


def test_refusals():
    sf = load_pkg()
    with pytest.raises(RuntimeError, match="GPU"):
        sf.functional.layer_norm(torch.zeros(2, 4), None, None)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sf.LayerNorm(4)(torch.zeros(2, 4))
    with pytest.raises(NotImplementedError):
        sf.LayerNorm((3, 4))


def test_library_refusals():
    """Bad arguments are turned away before anything is launched (no GPU needed)."""
    import ctypes
    sf = load_pkg()
    L = sf.ops.lib()
    ll, f, vp = ctypes.c_longlong, ctypes.c_float, ctypes.c_void_p
    a = vp(4096)

    def fwd(rows=4, D=8, dtype=0, res=None, total=None, mean=None, rstd=None, eps=1e-5, x=a):
        return L.sf_layer_norm_fwd(x, res, total, None, None, a, mean, rstd, ll(rows), D, f(eps), dtype, None)
    for bad in (dict(rows=0), dict(D=0), dict(D=(1 << 24) + 1), dict(dtype=2), dict(res=a), dict(total=a), dict(mean=a),
                dict(rstd=a), dict(eps=-1.0), dict(x=None)):
        assert fwd(**bad) == -22, bad
    need = int(L.sf_layer_norm_bwd_workspace_bytes(ll(100), 64, 0))
    assert need > 0 and int(L.sf_layer_norm_bwd_workspace_bytes(ll(0), 64, 0)) == 0

    def bwd(ws=a, nbytes=need, dw=a, rows=100, D=64, dtype=0, mean=a):
        return L.sf_layer_norm_bwd(a, None, a, None, mean, a, a, dw, None, ws, ctypes.c_size_t(nbytes), ll(rows), D, dtype, None)
    for bad in (dict(ws=None), dict(nbytes=need - 1), dict(rows=0), dict(dtype=7), dict(mean=None)):
        assert bwd(**bad) == -22, bad


@pytest.mark.gpu
def test_gpu_refusals():
    sf = load_pkg()
    x = torch.zeros(2, 4, device="cuda")
    ln = sf.functional.layer_norm
    with pytest.raises(TypeError):
        ln(x.half(), None, None)
    with pytest.raises(RuntimeError, match="residual"):
        ln(x, None, None, residual=x.bfloat16())
    with pytest.raises(RuntimeError, match="residual"):
        ln(x, None, None, residual=x[:1])
    with pytest.raises(RuntimeError, match="weight"):
        ln(x, torch.ones(5, device="cuda"), None)
    with pytest.raises(RuntimeError, match="bias"):
        ln(x, None, torch.ones(4))
    with pytest.raises(RuntimeError, match="no axis"):
        ln(torch.zeros(3, 0, device="cuda"), None, None)


@pytest.mark.gpu
def test_captured_training_pass_replays():
    sf = load_pkg()
    x, res, w, b, dy, ds = cuda(*make(700, 200, BF, True, seed=7))

    def passes():
        xs = [t.detach().requires_grad_(True) for t in (x, res, w, b)]
        y, s = sf.functional.layer_norm(*xs[:1], *xs[2:], residual=xs[1])
        return (y.detach(), s.detach(), *torch.autograd.grad([y, s], xs, [dy, ds]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = passes()
    for k in range(4):
        for t in (x, res, dy, ds):
            t.copy_(torch.randn_like(t) + k)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(got, passes()):
            assert torch.equal(a, e)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """2^20 + 3 rows of 2056 bf16 values, 4.3 GB: a row's result does not depend on the rows before it, so the last ones have
    the bits that they have alone."""
    sf = load_pkg()
    x = torch.empty((1 << 20) + 3, 2056, device="cuda", dtype=BF).normal_().requires_grad_(True)
    w = torch.randn(2056, device="cuda")
    y = sf.functional.layer_norm(x, w, None)
    dx, = torch.autograd.grad(y, x, x.detach())
    tail = x.detach()[-1000:].clone().requires_grad_(True)
    yt = sf.functional.layer_norm(tail, w, None)
    dt, = torch.autograd.grad(yt, tail, tail.detach())
    assert torch.equal(y[-1000:], yt) and torch.equal(dx[-1000:], dt)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [96, 999, 1000, 4095, 8191, 8195, 50001, (1 << 20) + 3])
@pytest.mark.parametrize("dtype", [BF, F])
def test_rows_without_spread(D, dtype):
    """Rows of one value, far from zero: the centred values are zero, so y is the bias and dx is r (g - mean(g)), r = 1 / sqrt(eps).
    The kernel's first mean is off by k steps of the value, k below the 32 + 8 roundings of its sum; k, k^2 and their sums over D
    values are whole numbers below 2^24 of those steps (D <= 8192; wider rows are summed in 64 bits), hence exact, and so the second mean
    takes all of the first one's error out: y is w * 0 + b exactly.  dx: mean(g) is off by at most 64 f32 half steps
    of the mean magnitude, r by 4 of itself, and dx is rounded once."""
    sf = load_pkg()
    vals = torch.tensor([1e3, -3.3e4, 1e5, -1e6, 7.0, 0.0]).to(dtype)
    x = vals.view(-1, 1).expand(-1, D).contiguous()
    g = torch.Generator().manual_seed(D)
    w, b = 1 + 0.3 * torch.randn(D, generator=g), 0.3 * torch.randn(D, generator=g)
    dy = torch.randn(len(vals), D, generator=g).to(dtype)
    y, _, grads = run(sf, x, None, w, b, dy, None)
    assert torch.equal(y.detach().cpu(), b.to(dtype).expand(len(vals), D))
    gw = dy.double() * w.double()
    r = 1e-5 ** -0.5
    want = r * (gw - gw.mean(1, keepdim=True))
    check(grads["dx"], want, want.abs() * (torch.finfo(dtype).eps / 2 * 1.01 + 4 * U32) + r * 64 * U32 * (gw.abs().mean(1, keepdim=True) + gw.abs()), "dx")
    assert float(grads["dw"].abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("D", [999, 1000, 8192, 8195, (1 << 20) + 3])
@pytest.mark.parametrize("offset", [1e3, 3e4, 1e6])
@pytest.mark.parametrize("dtype", [BF, F])
def test_rows_of_few_values_far_from_zero(D, offset, dtype):
    """Rows that differ by single steps of their type around a large value: the deviations are exact, so y is known to their
    precision, not to that of the offset.  In steps s of f32 at the offset: the first mean is off by at most 40 s (1/2 s for wide rows,
    in 64 bits), the centred values are exact multiples of s / 2 or so, rounded to U32 of their size (at most 44 s or the spread), their mean
    likewise: 40 U32 of (44 s + the largest deviation) for all of it.  The variance loses as much again, relative to itself
    or, where the correction is the larger part, 40 U32 of (44 s)^2."""
    sf = load_pkg()
    g = torch.Generator().manual_seed(D)
    base = torch.full((4, D), offset).to(dtype)
    step = torch.finfo(dtype).eps * 2.0 ** torch.floor(torch.log2(base.float().abs()))
    x = (base.double() + torch.randint(-1, 3, (4, D), generator=g) * step.double()).to(dtype)
    w, b = 1 + 0.3 * torch.randn(D, generator=g), 0.3 * torch.randn(D, generator=g)
    y = sf.functional.layer_norm(x.cuda(), w.cuda(), b.cuda())
    o = oracle(x, None, w, b, 1e-5)
    s = torch.finfo(F).eps * 2.0 ** math.floor(math.log2(offset))
    dev = (o["s"] - o["s"].mean(1, keepdim=True)).abs().amax(1, keepdim=True)
    off = 40 * U32 * (44 * s + dev) * o["r"]                      # of the normalised value
    rel = 40 * U32 * (1 + (44 * s * o["r"]) ** 2)                 # of r
    check(y, o["y"], o["y"].abs() * (torch.finfo(dtype).eps / 2 * 1.01) + w.double().abs() * (off + rel * o["xh"].abs()) + 4 * U32 * (b.double().abs() + o["xh"].abs() * w.double().abs()), "y")
