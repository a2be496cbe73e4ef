"""AdamW over many tensors, moments in 32 and in 8 bits, against the update in 64 bits; the 8-bit codec
against its definition; sizes, alignments, skips, captures and refusals.

Tolerances (u = 2^-24, half an f32 step).  m' = b1 m + a1 g: two products, one sum and the rounding of both
factors: 5 u of |b1 m| + |a1 g|.  v' the same with one more product: 6 u of the positive sum.  p' = p keep -
step m' / (sqrt(v') root + eps): the quotient collects m' (5 u of its terms' sizes), v' / 2 (3 u), square root,
product, sum, division, step and product (1 u each, step and root are rounded from 64 bits): 16 u of
step (|b1 m| + |a1 g|) / denominator, plus 3 u of |p| (factor, product, difference).  8-bit moments: the f32
value before rounding is off by the bounds above, so the code may differ from that of the 64-bit value only where
the two lie on either side of a rounding threshold; then the values differ by one code step, at most 1/8 of
the value (2^-3: three mantissa bits), or by the smallest code."""
import importlib

import pytest
import torch

from conftest import load_pkg

U = 2.0 ** -24
BLOCK = 256


def mix(x):
    """The 32-bit integer mixing of the rounding's hash, on int64 tensors."""
    M = 0xFFFFFFFF
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & M
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & M
    return x ^ (x >> 16)


def hash_bits(seed, step, ordinal, n):
    M = 0xFFFFFFFF
    t = torch.tensor
    key = mix(t((((seed & M) + step * 0x9E3779B1) & M) ^ (seed >> 32)))
    key = mix((key + ordinal * 0x85EBCA6B) & M)
    i = torch.arange(n)
    return mix(((i & M) * 0x9E3779B1 + (i >> 32) * 0xC2B2AE35 + key) & M)


def codec_values(signed):
    """The positive values of a code, in units of 2 ** (E - 127): zero, then three mantissa bits per binade, from
    15 (first moment) or 31 binades below the block's exponent."""
    reach, top = (15, 127) if signed else (31, 255)
    c = torch.arange(1, top + 1)
    return torch.cat([torch.zeros(1, dtype=torch.float64),
                      torch.ldexp(1 + (c % 8).double() / 8, (c // 8) - reach)])


def decode(codes, exps, signed):
    c = codes.cpu().long()
    low = c & 127 if signed else c
    e = exps.cpu().long().repeat_interleave(BLOCK)[:c.numel()]
    x = torch.ldexp(codec_values(signed)[low], e - 127)
    return torch.where(c > 127, -x, x) if signed else x


def pad_blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def block_exps(x, signed):
    """E of each block: the f32 exponent of the largest magnitude, one more above 1.875 times its power of two."""
    big = pad_blocks(x.abs()).amax(1)
    e = torch.floor(torch.log2(big.clamp_min(1e-300)))
    e = e + (big > 1.875 * torch.exp2(e)).double()
    return (e + 127).clamp(16 if signed else 32, 255).long()


def encode(x, r16, signed):
    """Values (64 bits) after stochastic rounding with 16 random bits each, and the block exponents."""
    e = block_exps(x, signed)
    unit = torch.exp2((e - 127).double()).repeat_interleave(BLOCK)[:x.numel()]
    grid = codec_values(signed)
    a = x.abs() / unit
    lo = (torch.searchsorted(grid, a, right=True) - 1).clamp(0, len(grid) - 1)
    hi = (lo + 1).clamp(max=len(grid) - 1)
    f = (a - grid[lo]) / (grid[hi] - grid[lo]).clamp_min(1e-300)
    u = r16.double() / 65536
    up = f + u >= 1
    if signed:
        up = torch.where(lo == 0, a > u * grid[1], up)
    else:
        up = torch.where(lo == 0, a > 0, up)
    up = up & (lo < len(grid) - 1)
    return torch.where(up, grid[hi], grid[lo]) * unit * torch.sign(x), e


def oracle(p, g, m, v, t, lr, b1, b2, eps, wd, scale=1.0):
    p, g, m, v = (x.double().cpu() for x in (p, g, m, v))
    g = g * scale
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    den = (v2 / (1 - b2 ** t)).sqrt() + eps
    step = lr / (1 - b1 ** t)
    p2 = p * (1 - lr * wd) - step * m2 / den
    terms = b1 * m.abs() + (1 - b1) * g.abs()
    return p2, m2, v2, 16 * U * step * terms / den + 3 * U * p.abs(), 5 * U * terms, 6 * U * v2


def check(got, want, bound, what):
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound + 1e-300).all()), f"{what}: off by {float((err / (bound + 1e-300)).max()):.2f} times the bound"


def check_codes(pair, exact, bound, r16, signed, what):
    """8-bit moments against the codes of the 64-bit values: exponents and values equal, but where the f32 error
    moves a value across a threshold (the codes of exact - bound and exact + bound bracket the result)."""
    codes, exps = pair
    got = decode(codes, exps, signed)
    lo_e, hi_e = block_exps(exact.abs() - bound, signed), block_exps(exact.abs() + bound, signed)
    e = exps.cpu().long()
    assert bool(((e >= lo_e) & (e <= hi_e)).all()), f"{what}: block exponents"
    same = (lo_e == hi_e).repeat_interleave(BLOCK)[:exact.numel()]
    want, _ = encode(exact, r16, signed)
    below, _ = encode(exact.abs() - torch.minimum(bound, exact.abs()), r16, signed)
    above, _ = encode(exact.abs() + bound, r16, signed)
    ok = (got == want) | ((got.abs() >= below) & (got.abs() <= above)) | ~same
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} codes off"
    flips = float((got != want)[same].double().mean()) if bool(same.any()) else 0.0
    assert flips <= 1e-3 + 2.0 / max(1, int(same.sum())), f"{what}: {flips:.2e} of the codes differ"


def make(sizes, bits, gdtype, seed=0, align=1):
    g = torch.Generator().manual_seed(seed)
    out = {"p": [], "g": [], "m": [], "v": []}
    for n in sizes:
        mag = torch.exp(1.5 * torch.randn(n, generator=g) - 5)
        vals = {"p": 0.1 * torch.randn(n, generator=g), "g": (torch.randn(n, generator=g) * mag).to(gdtype),
                "m": torch.randn(n, generator=g) * mag * 0.3, "v": mag * mag}
        for k, x in vals.items():
            if bits == 8 and k in "mv":
                e = block_exps(x.double(), k == "m")
                unit = torch.exp2((e - 127).double()).repeat_interleave(BLOCK)[:n]
                c = torch.searchsorted(codec_values(k == "m"), x.double().abs() / unit, right=True) - 1
                c = c + (128 * (x < 0) if k == "m" else 0)
                out[k].append((c.to(torch.uint8).cuda(), e.to(torch.uint8).cuda()))
            else:
                buf = torch.zeros(n + align, dtype=x.dtype, device="cuda")
                view = buf[align:align + n]
                view.copy_(x)
                out[k].append(view)
    return out


def values(x, signed):
    return decode(*x, signed) if isinstance(x, tuple) else x.double().cpu()


SIZES = [[1], [255, 256, 257], [4095, 4096, 4097, 1, 3, 5], [100003], [17] * 41 + [5000] * 43, [0, 12, 0, 300]]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES, ids=[f"{len(s)}x{max(s)}" for s in SIZES])
@pytest.mark.parametrize("bits,gdtype", [(32, torch.float32), (32, torch.bfloat16), (8, torch.float32), (8, torch.bfloat16)])
def test_against_64_bits(sizes, bits, gdtype):
    """Three steps; lr and decay per tensor; buffers at odd elements; each step held against the formula from the
    state before it."""
    sf = load_pkg()
    x = make(sizes, bits, gdtype, seed=len(sizes))
    state = torch.tensor([4, 0], dtype=torch.int32, device="cuda")
    lrs = [1e-3 * (1 + i % 3) for i in range(len(sizes))]
    wds = [0.0 if i % 2 else 0.05 for i in range(len(sizes))]
    for t in (5, 6, 7):
        before = [(p.clone(), values(m, True), values(v, False)) for p, m, v in zip(x["p"], x["m"], x["v"])]
        sf.functional.adamw_step(x["p"], x["g"], x["m"], x["v"], state, lrs, (0.9, 0.99), 1e-8, wds, seed=77 + (5 << 32),
                                 grad_scale=0.5)
        for i, (p, m, v) in enumerate(before):
            p2, m2, v2, bp, bm, bv = oracle(p, x["g"][i], m, v, t, lrs[i], 0.9, 0.99, 1e-8, wds[i], 0.5)
            check(x["p"][i], p2, bp, f"p[{i}]")
            if bits == 32:
                check(x["m"][i], m2, bm, f"m[{i}]")
                check(x["v"][i], v2, bv, f"v[{i}]")
            elif sizes[i]:
                r = hash_bits(77 + (5 << 32), t, i, sizes[i])
                check_codes(x["m"][i], m2, bm, r >> 16, True, f"m[{i}]")
                check_codes(x["v"][i], v2, bv, r & 0xFFFF, False, f"v[{i}]")
    assert state.tolist() == [7, 0]


@pytest.mark.gpu
def test_neighbours_are_left_alone():
    """Tensors inside larger buffers: nothing before or behind them is written."""
    sf = load_pkg()
    for bits in (32, 8):
        bufs = {k: torch.full((1000,), 7.0, device="cuda") for k in "pg"}
        n, o = 515, 131
        p, g = bufs["p"][o:o + n], bufs["g"][o:o + n]
        if bits == 32:
            mb, vb = torch.full((1000,), 3.0, device="cuda"), torch.full((1000,), 3.0, device="cuda")
            m, v, extra = mb[o:o + n], vb[o:o + n], []
        else:
            mb, vb, eb, fb = (torch.full((1000,), 9, dtype=torch.uint8, device="cuda") for _ in range(4))
            for t in (mb, vb):
                t[o:o + n] = 0
            for t in (eb, fb):
                t[5:8] = 0
            m, v, extra = (mb[o:o + n], eb[5:8]), (vb[o:o + n], fb[5:8]), [(eb, 5, 3, 9), (fb, 5, 3, 9)]
        sh = torch.full((1000,), 5.0, dtype=torch.bfloat16, device="cuda")
        state = torch.zeros(2, dtype=torch.int32, device="cuda")
        sf.functional.adamw_step([p], [g], [m], [v], state, 1e-2, shadows=[sh[o:o + n]])
        fill = 3.0 if bits == 32 else 9
        for buf, at, k, want in [(bufs["p"], o, n, 7.0), (mb, o, n, fill), (vb, o, n, fill), (sh, o, n, 5.0)] + extra:
            assert bool((buf[:at] == want).all()) and bool((buf[at + k:] == want).all())
        assert torch.equal(sh[o:o + n], p.bfloat16())
        assert bool((p != 7.0).all())


@pytest.mark.gpu
def test_moment_values_are_exact_and_whole():
    sf = load_pkg()
    n = 5001
    g = torch.Generator().manual_seed(0)
    pairs = {}
    for name, least in (("m", 16), ("v", 32)):
        codes = torch.randint(0, 256, (n,), generator=g).to(torch.uint8)
        exps = torch.randint(least, 250, ((n + 255) // 256,), generator=g).to(torch.uint8)
        pairs[name] = (codes.cuda(), exps.cuda())
    mv, vv = sf.functional.adamw_moments([pairs["m"]], [pairs["v"]])
    assert torch.equal(mv[0].double().cpu(), decode(*pairs["m"], True))
    assert torch.equal(vv[0].double().cpu(), decode(*pairs["v"], False))


@pytest.mark.gpu
def test_rounding_is_unbiased_and_second_moments_decay():
    """Ten thousand elements with one value, one step each: the mean code value is the value, to 5 standard
    deviations of the rounding (a step is 1/8 of the value at most: sigma <= value / 16 / sqrt(n)).  And with no
    gradient, 1000 steps at b2 = 0.999 take the second moment from 1 to 0.999^1000 = 0.37 in the mean, where
    rounding to nearest would leave it at 1: within 5 sigma, sigma of one element being at most 0.25 (see
    below), so 0.25 / sqrt(n)."""
    sf = load_pkg()
    n = 1 << 14
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 0.77, device="cuda")
    g[::BLOCK] = 1.3                    # another value is the block's largest
    m, v = ((torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(n // BLOCK, dtype=torch.uint8, device="cuda"))
            for _ in range(2))
    state = torch.zeros(2, dtype=torch.int32, device="cuda")
    sf.functional.adamw_step([p], [g], [m], [v], state, 0.0, (0.9, 0.999), weight_decay=0.0, seed=3)
    rest = torch.ones(n, dtype=torch.bool)
    rest[::BLOCK] = False
    for pair, signed, want in ((m, True, 0.1 * 0.77), (v, False, 0.001 * 0.77 ** 2)):
        got = decode(*pair, signed)[rest]
        assert len(got.unique()) == 2
        assert abs(float(got.mean()) - want) <= 5 * want / 16 / got.numel() ** 0.5
    # decay: per step the value loses 1e-3 of itself through rounding events of at most 1/8 of the value, variance
    # 1e-3 * (1/8) * value^2; over 1000 steps (values fall from 1) at most 1000 * 1.25e-4 / 2 = 0.0625 = 0.25^2
    zero = torch.zeros(n, device="cuda")
    v0 = float(decode(*v, False)[rest].mean())
    for _ in range(1000):
        sf.functional.adamw_step([p], [zero], [m], [v], state, 0.0, (0.9, 0.999), weight_decay=0.0, seed=3)
    v1 = float(decode(*v, False)[rest].mean())
    assert abs(v1 / v0 - 0.999 ** 1000) <= 5 * 0.25 / int(rest.sum()) ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_extreme_values(bits):
    """Gradients from the smallest f32 to large ones, zeros, and blocks of zeros: finite results, zero moments stay
    zero, the second moment of a small non-zero gradient is never rounded to zero."""
    sf = load_pkg()
    n = 1024
    g = torch.zeros(n, device="cuda")
    g[:256] = torch.logspace(-44, 0, 256, device="cuda")
    g[256:512] = torch.logspace(0, 15, 256, device="cuda")
    g[512] = 1e-30
    p = torch.ones(n, device="cuda")
    x = [torch.zeros(n, device="cuda") if bits == 32 else (torch.zeros(n, dtype=torch.uint8, device="cuda"),
                                                           torch.zeros(4, dtype=torch.uint8, device="cuda")) for _ in range(2)]
    state = torch.zeros(2, dtype=torch.int32, device="cuda")
    for _ in range(3):
        sf.functional.adamw_step([p], [g], [x[0]], [x[1]], state, 1e-3, weight_decay=0.0)
        assert bool(torch.isfinite(p).all())
    if bits == 8:
        m, v = decode(*x[0], True), decode(*x[1], False)
        assert bool((m[513:] == 0).all()) and bool((v[513:] == 0).all()) and bool((p[513:] == 1).all())
        sq = (g[:513].float() * g[:513]).cpu() * 0.001
        assert bool((v[:513][sq > 1e-37] > 0).all())
        assert x[0][1].tolist()[3] == 16 and x[1][1].tolist()[3] == 32


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_found_inf_skips_on_the_device(bits):
    sf = load_pkg()
    x = make([300, 5000], bits, torch.float32)
    x["g"][1][17] = float("nan")
    state = torch.zeros(2, dtype=torch.int32, device="cuda")
    flag = torch.ones(1, dtype=torch.int32, device="cuda")
    flat = [t for k in "pmv" for y in x[k] for t in (y if isinstance(y, tuple) else (y,))]
    before = [t.clone() for t in flat]
    sf.functional.adamw_step(x["p"], x["g"], x["m"], x["v"], state, 1e-3, found_inf=flag)
    assert state.tolist() == [0, 1] and all(torch.equal(a, b) for a, b in zip(before, flat))
    flag.zero_()
    x["g"][1][17] = 0.0
    sf.functional.adamw_step(x["p"], x["g"], x["m"], x["v"], state, 1e-3, found_inf=flag)
    assert state.tolist() == [1, 1] and not torch.equal(before[0], flat[0])


@pytest.mark.gpu
def test_matches_torch_adamw_with_missing_gradients():
    """The optimiser class against torch.optim.AdamW over ten steps, a parameter sitting out some of them: both f32,
    so each step adds the bounds of the module's docstring, 16 u of lr * (ratio <= 1 / (1 - b1)) plus 3 u of |p|."""
    sf = load_pkg()
    training = importlib.import_module(sf.__name__ + ".training")
    torch.manual_seed(1)
    ps = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((7, 5), (300,), (64, 33))]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    ours = training.AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 3e-3, "weight_decay": 0.0}], lr=1e-3, weight_decay=0.1)
    ref = torch.optim.AdamW([{"params": qs[:2]}, {"params": qs[2:], "lr": 3e-3, "weight_decay": 0.0}], lr=1e-3, weight_decay=0.1)
    for k in range(10):
        for i, (p, q) in enumerate(zip(ps, qs)):
            g = torch.randn_like(p)
            p.grad, q.grad = (None, None) if i == 1 and k in (0, 3, 4) else (g.clone(), g.clone())
        ours.step()
        ref.step()
    assert ours.t == 10
    for p, q in zip(ps, qs):
        assert float((p - q).detach().abs().max()) <= 10 * (16 * U * 3e-3 * 10 + 6 * U * float(q.detach().abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_round_trip_and_reproducibility(bits, tmp_path):
    sf = load_pkg()
    training = importlib.import_module(sf.__name__ + ".training")

    def fresh():
        torch.manual_seed(2)
        ps = [torch.nn.Parameter(torch.randn(n, device="cuda")) for n in (1000, 33, 4100)]
        return ps, training.AdamW(ps, lr=1e-2, state_bits=bits, seed=9)

    def steps(ps, opt, ks):
        for k in ks:
            for i, p in enumerate(ps):
                p.grad = torch.sin(torch.arange(p.numel(), device="cuda") * (k + 1.3) + i)
            opt.step()
    a, oa = fresh()
    steps(a, oa, range(6))
    b, ob = fresh()
    steps(b, ob, range(3))
    torch.save(ob.state_dict(), tmp_path / "o.pt")
    c, oc = fresh()
    for x, y in zip(c, b):
        x.data.copy_(y.data)
    oc.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
    steps(c, oc, range(3, 6))
    for x, y in zip(a, c):
        assert torch.equal(x, y)
    for x, y in zip(oa.moments(), oc.moments()):
        assert all(torch.equal(s, t) for s, t in zip(x, y)) and x[0].shape == a[0].shape
    other = training.AdamW([torch.nn.Parameter(torch.zeros(5, device="cuda"))], state_bits=bits)
    with pytest.raises(RuntimeError):
        other.load_state_dict(oc.state_dict())


@pytest.mark.gpu
def test_derived_copies_go_stale():
    sf = load_pkg()
    training = importlib.import_module(sf.__name__ + ".training")
    p = torch.nn.Parameter(torch.randn(64, 8, device="cuda"))
    sh = sf.ops.weight_shadow(p)
    p.grad = torch.ones_like(p)
    training.AdamW([p], lr=0.1).step()
    assert sf.ops.shadow_if_current(p) is None
    assert torch.equal(sf.ops.weight_shadow(p), p.detach().bfloat16()) and not torch.equal(sh, p.detach().bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays(bits):
    sf = load_pkg()
    sizes = [513, 40, 9000]
    a, b = make(sizes, bits, torch.float32, seed=4), make(sizes, bits, torch.float32, seed=4)
    sa, sb = (torch.zeros(2, dtype=torch.int32, device="cuda") for _ in range(2))
    w, sw = make(sizes, bits, torch.float32, seed=5), torch.zeros(2, dtype=torch.int32, device="cuda")
    sf.functional.adamw_step(w["p"], w["g"], w["m"], w["v"], sw, 1e-2, seed=1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sf.functional.adamw_step(a["p"], a["g"], a["m"], a["v"], sa, 1e-2, seed=1)
    for k in range(4):
        for x in (a, b):
            for i, g in enumerate(x["g"]):
                g.copy_(torch.cos(torch.arange(g.numel(), device="cuda") * (k + 0.7) + i))
        graph.replay()
        torch.cuda.synchronize()
        sf.functional.adamw_step(b["p"], b["g"], b["m"], b["v"], sb, 1e-2, seed=1)
        for key in "pmv":
            for x, y in zip(a[key], b[key]):
                for s, t in zip(*((x, y) if isinstance(x, tuple) else ((x,), (y,)))):
                    assert torch.equal(s, t), (k, key)
    assert sa.tolist() == [4, 0]


def tiny_config(**train):
    return {"data": {"image_size": [64, 64], "window_size": 5, "upscale_factor": 2},
            "model": {"input_channels": 3, "hidden_dim": 16, "num_layers": 2, "temporal_module": "Transformer", "use_gan": True},
            "loss": {"metric": "MSE", "weights": {"image": 1.0, "station": 0.5}}, "stations": {"kernel_size": 5, "metric": "MSE"},
            "train": {"lr": 1e-3, **train}, "system": {"mixed_precision": False}}


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_trainer_option(bits, tmp_path):
    """train.optimizer AdamW: the step moves every parameter as the formula says from its gradient, decay on weight
    matrices alone; checkpoints carry the state."""
    sf = load_pkg()
    training = importlib.import_module(sf.__name__ + ".training")
    torch.manual_seed(0)
    tr = training.Trainer(tiny_config(optimizer="AdamW", weight_decay=0.1, optimizer_state_bits=bits), device="cuda:0")
    tr.model.temporal_module.dropout = 0.0
    x, y = torch.randn(2, 5, 3, 64, 64), torch.randn(2, 1, 64, 64)
    pos, run = [torch.tensor([[5, 7]])] * 2, [torch.tensor([0.3])] * 2
    seen = {}
    step = training.FlatAdamW.step

    def spy(self, *a, **k):
        ns = len(self.small)
        seen[id(self)] = [(p.detach().clone(), (self._small_views[i] if i < ns else p.grad).clone())
                          for i, p in enumerate(self.params)]
        return step(self, *a, **k)
    training.FlatAdamW.step = spy
    try:
        tr.train_step(x, y, pos, run)
    finally:
        training.FlatAdamW.step = step
    for opt, lr, betas in ((tr.opt_g, 1e-3, (0.9, 0.999)), (tr.opt_d, 2e-4, (0.5, 0.999))):
        assert opt.t == 1
        for p, (before, g) in zip(opt.params, seen[id(opt)]):
            z = torch.zeros_like(before)
            p2, _, _, bp, _, _ = oracle(before, g, z, z, 1, lr, *betas, 1e-8, 0.1 if p.dim() > 1 else 0.0)
            check(p.detach(), p2, bp, tuple(p.shape))
    tr.save_checkpoint(str(tmp_path / "c.pt"))
    tr2 = training.Trainer(tiny_config(optimizer="AdamW", weight_decay=0.1, optimizer_state_bits=bits), device="cuda:0")
    assert tr2.load_checkpoint(str(tmp_path / "c.pt")) == "resume"
    for (m, v), (m2, v2) in zip(tr.opt_g.moment_pairs, tr2.opt_g.moment_pairs):
        for s, t in zip((*m, *v) if bits == 8 else (m, v), (*m2, *v2) if bits == 8 else (m2, v2)):
            assert torch.equal(s, t)
    other = training.Trainer(tiny_config(optimizer="AdamW", optimizer_state_bits=40 - bits), device="cuda:0")
    with pytest.raises(RuntimeError, match="bits"):
        other.load_checkpoint(str(tmp_path / "c.pt"))


@pytest.mark.gpu
def test_trainer_without_the_option(caplog):
    """Adam as before, with any other value of a key that was not read before."""
    sf = load_pkg()
    training = importlib.import_module(sf.__name__ + ".training")
    for value, warns in ((None, False), ("adam", False), ("SGD", True)):
        caplog.clear()
        tr = training.Trainer(tiny_config(**({} if value is None else {"optimizer": value})), device="cuda:0")
        assert type(tr.opt_g) is training.FlatAdam and type(tr.opt_d) is training.FlatAdam
        assert any("neither Adam nor AdamW" in r.getMessage() for r in caplog.records) == warns


def test_hash_spreads():
    """The rounding bits over 2^16 consecutive elements, per tensor and step: each half's mean and variance are
    those of a uniform number to 5 standard deviations, and different steps, tensors and halves do not correlate."""
    n = 1 << 16
    streams = []
    for step, ordinal in ((1, 0), (2, 0), (1, 1)):
        r = hash_bits(12345, step, ordinal, n)
        streams += [(r >> 16).double() / 65536, (r & 0xFFFF).double() / 65536]
    for u in streams:
        assert abs(float(u.mean()) - 0.5) < 5 * (1 / 12) ** 0.5 / n ** 0.5
        assert abs(float(u.var()) - 1 / 12) < 5 * (1 / 180) ** 0.5 / n ** 0.5
    for i in range(len(streams)):
        for j in range(i):
            c = float(((streams[i] - 0.5) * (streams[j] - 0.5)).mean()) * 12
            assert abs(c) < 5 / n ** 0.5
        c = float(((streams[i][1:] - 0.5) * (streams[i][:-1] - 0.5)).mean()) * 12
        assert abs(c) < 5 / n ** 0.5


def test_refusals():
    sf = load_pkg()
    training = importlib.import_module(sf.__name__ + ".training")
    z = torch.zeros(4)
    with pytest.raises(RuntimeError, match="GPU"):
        sf.functional.adamw_step([z], [z], [z], [z], torch.zeros(2, dtype=torch.int32), 1e-3)
    with pytest.raises(ValueError, match="bits"):
        training.AdamW([torch.nn.Parameter(z)], state_bits=16)
    with pytest.raises(ValueError, match="betas"):
        training.AdamW([torch.nn.Parameter(z)], betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="twice"):
        p = torch.nn.Parameter(z)
        training.AdamW([p, p])
    with pytest.raises(TypeError):
        training.AdamW([torch.nn.Parameter(z.bfloat16())])
    with pytest.raises(ValueError, match="no parameters"):
        training.AdamW([])


def test_library_refusals():
    """Bad arguments are turned away before anything is launched (no GPU needed)."""
    import ctypes
    L = load_pkg().ops.lib()
    vp, ll, d, i32 = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_double, ctypes.c_int
    a = (vp * 1)(4096)

    def call(n=4, bits=32, b1=0.9, b2=0.999, eps=1e-8, p=a, e=None, gd=0, off=None, state=vp(4096)):
        return L.sf_adamw_step(1, p, a, a, a, e, e, None, (ll * 1)(n), (d * 1)(1e-3), (d * 1)(0.0), (i32 * 1)(gd),
                               None if off is None else (i32 * 1)(off), bits, d(b1), d(b2), ctypes.c_float(eps),
                               ctypes.c_float(1.0), ctypes.c_ulonglong(0), state, None, None)
    for bad in (dict(n=-1), dict(n=(1 << 41) + 1), dict(bits=16), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(p=(vp * 1)(None)),
                dict(bits=8), dict(bits=8, e=(vp * 1)(None)), dict(gd=3), dict(off=1), dict(state=None), dict(p=None)):
        assert call(**bad) == -22, bad


@pytest.mark.gpu
def test_gpu_refusals():
    sf = load_pkg()
    step = sf.functional.adamw_step
    z = lambda n=4, dt=torch.float32: torch.zeros(n, dtype=dt, device="cuda")
    state = z(2, torch.int32)
    p = z()
    with pytest.raises(RuntimeError, match="twice"):
        step([p, p], [z(), z()], [z(), z()], [z(), z()], state, 1e-3)
    with pytest.raises(RuntimeError, match="found_inf"):
        step([p], [z()], [z()], [z()], state, 1e-3, found_inf=torch.zeros(0, device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError, match="twice"):
        m = z()
        step([p, z()], [z(), z()], [m, m], [z(), z()], state, 1e-3)
    with pytest.raises(RuntimeError, match="gradient 0"):
        step([p], [z(5)], [z()], [z()], state, 1e-3)
    with pytest.raises(RuntimeError, match="moment"):
        step([p], [z()], [z(5)], [z()], state, 1e-3)
    with pytest.raises(RuntimeError, match="block exponents"):
        step([p], [z()], [(z(4, torch.uint8), z(2, torch.uint8))], [(z(4, torch.uint8), z(1, torch.uint8))], state, 1e-3)
    with pytest.raises(TypeError, match="mixed"):
        step([p], [z()], [z()], [(z(4, torch.uint8), z(1, torch.uint8))], state, 1e-3)
    with pytest.raises(TypeError):
        step([z(4, torch.bfloat16)], [z()], [z()], [z()], state, 1e-3)
    with pytest.raises(TypeError):
        step([p], [z(4, torch.float16)], [z()], [z()], state, 1e-3)
    with pytest.raises(RuntimeError, match="contiguous"):
        step([z(8)[::2]], [z()], [z()], [z()], state, 1e-3)
    with pytest.raises(ValueError, match="betas"):
        step([p], [z()], [z()], [z()], state, 1e-3, betas=(0.9, 1.0))
    with pytest.raises(RuntimeError, match="weight_decay"):
        step([p], [z()], [z()], [z()], state, 1e-3, weight_decay=[0.1, 0.1])
    with pytest.raises(RuntimeError, match="state"):
        step([p], [z()], [z()], [z()], z(3, torch.int32), 1e-3)
    assert state.tolist() == [0, 0]


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A tensor of 2^30 + 5001 elements (4.3 GB each of values, gradients and f32 moments), between two small ones: its last
    elements take the step that they take alone."""
    sf = load_pkg()
    n, k = (1 << 30) + 5001, 7001
    big = [torch.full((n,), x, device="cuda") for x in (0.5, 0.25, 0.125, 0.0625)]
    for t in big:
        t[-k:].normal_()
    big[3].abs_()
    alone = [t[-k:].clone() for t in big]
    lists = [[torch.ones(5, device="cuda"), t, torch.ones(3, device="cuda")] for t in big]
    for xs in (lists, [[t] for t in alone]):
        state = torch.zeros(2, device="cuda", dtype=torch.int32)
        sf.functional.adamw_step(*xs, state, 1e-2)
    for t, a in zip(big, alone):
        assert torch.equal(t[-k:], a)
    head = [torch.full((100,), x, device="cuda") for x in (0.5, 0.25, 0.125, 0.0625)]
    sf.functional.adamw_step(*([t] for t in head), torch.zeros(2, device="cuda", dtype=torch.int32), 1e-2)
    for t, a in zip(big, head):
        assert bool((t[:-k] == a[0]).all())


@pytest.mark.gpu
def test_derived_copies_go_stale_for_an_iterator():
    """The parameters may come as an iterator (module.parameters()), as any other list of the call."""
    sf = load_pkg()
    lin = torch.nn.Linear(16, 8).cuda()
    shadow = sf.ops.weight_shadow(lin.weight).clone()
    gs, ms, vs = ([torch.ones_like(p) for p in lin.parameters()] for _ in range(3))
    state = torch.zeros(2, dtype=torch.int32, device="cuda")
    sf.functional.adamw_step(lin.parameters(), iter(gs), iter(ms), iter(vs), state, 0.1)
    assert sf.ops.shadow_if_current(lin.weight) is None
    assert torch.equal(sf.ops.weight_shadow(lin.weight), lin.weight.detach().bfloat16())
    assert not torch.equal(shadow, lin.weight.detach().bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("decay", [1e-6, 2e-7, 1e-7, 2e-8])
def test_small_decay_counts(decay, bits):
    """lr * weight_decay far below a step of f32 at one still takes part in the sum that is rounded into p.  Of the new value only that
    last rounding is of the size of p: half a step of f32, 2^-24 in [1, 2) and less below one, 2^-23 where it ends above
    two.  Everything before is of the size of the change, |step| <= lr: 16 u of it (the module's docstring), u of the decay's rounding
    and u of the sum's, 18 u (lr + 2 decay) together.  (A factor 1 - lr * weight_decay, rounded to f32, is off by up to 2^-25 of the
    value and its product by half a step more.)"""
    sf = load_pkg()
    n, lr = 1 << 20, 1e-3
    gen = torch.Generator().manual_seed(6)
    p0 = 1 + torch.rand(n, generator=gen)
    g = torch.randn(n, generator=gen)
    p = p0.cuda()
    m, v = ([torch.zeros(n, device="cuda")] if bits == 32 else
            [(torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(n // BLOCK, dtype=torch.uint8, device="cuda"))] for _ in range(2))
    sf.functional.adamw_step([p], [g.cuda()], m, v, torch.zeros(2, dtype=torch.int32, device="cuda"), lr, weight_decay=decay / lr)
    z = torch.zeros(n)
    want = oracle(p0, g, z, z, 1, lr, 0.9, 0.999, 1e-8, decay / lr)[0]
    half = torch.exp2(torch.floor(torch.log2(want + 2.0 ** -22)) - 24)
    check(p, want, half + 18 * U * (lr + 2 * decay), "p")


def test_group_options_that_are_not_per_group():
    """betas and eps are those of the optimiser: a group that brings others is turned away, not ignored; so are torch's variants
    of the update.  Equal values, and keys that are no options, are fine."""
    training = importlib.import_module(load_pkg().__name__ + ".training")
    p = torch.nn.Parameter(torch.zeros(4))
    for extra in ({"betas": (0.5, 0.9)}, {"eps": 1e-6}, {"amsgrad": True}, {"maximize": True}):
        with pytest.raises(ValueError, match=next(iter(extra))):
            training.AdamW([{"params": [p], **extra}])
    opt = training.AdamW([{"params": [p], "lr": 1e-2, "weight_decay": 0.0, "betas": [0.9, 0.999], "eps": 1e-8, "amsgrad": False,
                           "maximize": False, "name": "all"}])
    opt.param_groups[0]["betas"] = (0.5, 0.9)
    p.grad = torch.zeros(4)
    with pytest.raises(ValueError, match="betas"):
        opt.step()


def test_8_bit_state_is_not_read_as_adam():
    """A checkpoint of 8-bit moments says so when plain Adam is asked to resume from it."""
    training = importlib.import_module(load_pkg().__name__ + ".training")
    net = torch.nn.Linear(4, 4)
    opt = training.FlatAdam(net, 1e-3)
    with pytest.raises(RuntimeError, match="8 bits"):
        opt.load_state_by_name(net, {"t": 3, "state_bits": 8, "seed": 0, "moments": {}})


@pytest.mark.gpu
def test_shadows_and_exponents_listed_twice_are_refused():
    sf = load_pkg()
    z = lambda n=300, dt=torch.float32: torch.zeros(n, dtype=dt, device="cuda")
    byte = lambda n=300: z(n, torch.uint8)
    state, sh, e = z(2, torch.int32), z(300, torch.bfloat16), byte(2)
    with pytest.raises(RuntimeError, match="twice"):
        sf.functional.adamw_step([z(), z()], [z(), z()], [z(), z()], [z(), z()], state, 1e-3, shadows=[sh, sh])
    for ms, vs in (([(byte(), e), (byte(), e)], [(byte(), byte(2)), (byte(), byte(2))]),
                   ([(byte(), byte(2)), (byte(), byte(2))], [(byte(), e), (byte(), e)]), ([(byte(), e)], [(byte(), e)])):
        n = len(ms)
        with pytest.raises(RuntimeError, match="twice"):
            sf.functional.adamw_step([z() for _ in range(n)], [z() for _ in range(n)], ms, vs, state, 1e-3)
    with pytest.raises(RuntimeError, match="twice"):
        sf.functional.adamw_moments([(byte(), byte(2))] * 2, [(byte(), byte(2))] * 2, out=([sh, sh], [z(300, torch.bfloat16) for _ in range(2)]))
    assert state.tolist() == [0, 0]
    sf.functional.adamw_step([z(), z()], [z(), z()], [z(), z()], [z(), z()], state, 1e-3, shadows=[None, None])


@pytest.mark.gpu
def test_captured_step_and_derived_copies():
    """A replay updates the parameters without a call of Python: copies derived from them (shadows, packed weights) are never
    taken for current once a step has been captured, copies built inside a graph are the graph's own, and a step is not captured
    while a copy from outside is current, since what came before it in the graph may read that copy at every replay."""
    sf = load_pkg()
    p, q = (torch.nn.Parameter(torch.randn(64, 8, device="cuda")) for _ in range(2))
    new = lambda: [torch.zeros(64, 8, device="cuda")]
    copy = lambda x: sf.ops.derived(x, "copy", lambda: x.detach().clone())
    state = torch.zeros(2, dtype=torch.int32, device="cuda")
    grads, ms, vs = [torch.ones(64, 8, device="cuda")], new(), new()
    sf.functional.adamw_step([p], grads, ms, vs, state, 0.1)
    copy(p)
    sf.ops.weight_shadow(p)
    sf.ops.touch([p])                                   # (announced: the copies from outside are stale)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = copy(p)
        sf.functional.adamw_step([p], grads, ms, vs, state, 0.1)
    for _ in range(3):
        before = p.detach().clone()
        assert torch.equal(sf.ops.weight_shadow(p), before.bfloat16()) and torch.equal(copy(p), before)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(inside, before) and not torch.equal(p.detach(), before)
    sf.functional.adamw_step([p], grads, ms, vs, state, 0.1)
    assert torch.equal(sf.ops.weight_shadow(p), p.detach().bfloat16()) and torch.equal(copy(p), p.detach())
    assert state.tolist() == [5, 0]
    more = (new(), new())
    for make_copy in (sf.ops.weight_shadow, copy):
        q = torch.nn.Parameter(q.detach().clone())
        make_copy(q)
        with pytest.raises(RuntimeError, match="derived"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                sf.functional.adamw_step([q], grads, *more, state, 0.1)
        torch.cuda.synchronize()
        assert state.tolist() == [5, 0] and torch.equal(make_copy(q).float(), q.detach().to(make_copy(q).dtype).float())


def test_copies_of_host_parameters_are_kept():
    """Without a GPU the cache of derived copies asks no stream."""
    ops = load_pkg().ops
    p = torch.nn.Parameter(torch.zeros(4))
    first = ops.derived(p, "copy", lambda: p.detach().clone())
    assert ops.derived(p, "copy", lambda: p.detach().clone()) is first
    ops.touch([p])
    assert ops.derived(p, "copy", lambda: p.detach().clone()) is not first


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("wd", [0.0, 0.1])
def test_infinite_parameters_stay(bits, wd):
    """A parameter that holds infinities (a learned mask) keeps them, as p (1 - lr wd) - step does; its other values step."""
    sf = load_pkg()
    p = torch.tensor([1.0, float("inf"), -2.0, float("-inf")], device="cuda")
    m, v = ([torch.zeros(4, device="cuda")] if bits == 32 else
            [(torch.zeros(4, dtype=torch.uint8, device="cuda"), torch.zeros(1, dtype=torch.uint8, device="cuda"))] for _ in range(2))
    g = torch.tensor([1.0, 0.0, 1.0, 0.5], device="cuda")
    sf.functional.adamw_step([p], [g], m, v, torch.zeros(2, dtype=torch.int32, device="cuda"), 1e-2, weight_decay=wd)
    assert p[1] == float("inf") and p[3] == float("-inf")
    assert bool(torch.isfinite(p[::2]).all()) and float(p[0]) < 1.0 and float(p[2]) < -1.99
