"""LayerNorm, differential attention and AdamW together, as a training step of a pre-norm attention block uses them,
against the same block in 64 bits (plain torch operations, autograd and torch.optim.AdamW on the CPU)."""
import importlib
import math

import pytest
import torch
import torch.nn as nn

from conftest import load_pkg

E, H, KV, T, B = 64, 2, 1, 83, 3


class Block(nn.Module):
    """x + attention(norm(x)), then a norm over the sum and a linear read-out (the residual add fused into the norm)."""

    def __init__(self, sf, causal):
        super().__init__()
        self.norm1, self.norm2 = sf.LayerNorm(E), sf.LayerNorm(E)
        self.attn = sf.DifferentialAttention(E, H, KV, causal=causal)

    def forward(self, x, lengths):
        a = self.attn(self.norm1(x), lengths)
        y, s = self.norm2(a.to(x.dtype), residual=x)
        return y, s


def plain_norm(x, w, b):
    c = x - x.mean(-1, keepdim=True)
    return c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * w + b


def plain_block(p, x, lengths, causal, lambda_init=0.8):
    d = E // (2 * H)
    h = plain_norm(x, p["norm1.weight"], p["norm1.bias"])
    qkv = h @ p["attn.in_proj.weight"].T + p["attn.in_proj.bias"]
    q, k, v = torch.split(qkv, [H * 2 * d, KV * 2 * d, KV * 2 * d], -1)
    q = q.view(B, T, H, 2, d).permute(0, 2, 3, 1, 4)
    k = k.view(B, T, KV, 2, d).permute(0, 2, 3, 1, 4).repeat_interleave(H // KV, 1)
    v = v.view(B, T, KV, 2 * d).permute(0, 2, 1, 3).repeat_interleave(H // KV, 1)
    see = (torch.arange(T) < lengths.view(B, 1)).view(B, 1, 1, 1, T)
    if causal:
        see = see & torch.ones(T, T, dtype=torch.bool).tril().view(1, 1, 1, T, T)
    z = (q @ k.transpose(-1, -2) / math.sqrt(d)).masked_fill(~see, -math.inf)
    top = z.detach().amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    m = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    lam = (torch.exp((p["attn.lambda_q1"] * p["attn.lambda_k1"]).sum(-1)) - torch.exp((p["attn.lambda_q2"] * p["attn.lambda_k2"]).sum(-1))
           + lambda_init)
    o = ((m[:, :, 0] - lam.view(1, H, 1, 1) * m[:, :, 1]) @ v).permute(0, 2, 1, 3)
    o = plain_norm(o, p["attn.norm.weight"], p["attn.norm.bias"]) * (1 - lambda_init)
    a = o.reshape(B, T, -1) @ p["attn.out_proj.weight"].T + p["attn.out_proj.bias"]
    s = a + x
    return plain_norm(s, p["norm2.weight"], p["norm2.bias"]), s


def rel(a, b):
    return float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm().clamp_min(1e-300))


@pytest.mark.gpu
@pytest.mark.parametrize("causal,bits", [(False, 32), (True, 8)])
def test_training_steps_in_f32(causal, bits):
    """Three steps.  f32 against 64 bits: every stage is a few f32 roundings of sums of up to a few hundred terms, some
    1e-6 of a tensor's norm, and the norm over a head's difference of two maps multiplies what lies before it by the
    spread it divides by (a tenth and more here): 1e-4 of the norm covers the chain.  The first two AdamW steps move
    an entry by lr in the direction of its gradient, whatever its size: where a gradient is below its own rounding the
    direction is noise.  Those entries (gradients under 1e-4 of the tensor's largest) are left out of the parameters'
    comparison; the others differ by the relative error of the gradient (1e-4 / 1e-4 at most, 2 lr) in the worst entry and
    a hundredth of that in the norm.  The state's width does not matter to the first steps' parameters beyond the
    rounding of a moment to three mantissa bits (1/16 of it) in the second and third, 1/8 of lr per step."""
    sf = load_pkg()
    training = importlib.import_module(sf.__name__ + ".training")
    torch.manual_seed(0)
    blk = Block(sf, causal).cuda()
    ref = {n: p.detach().cpu().double().clone().requires_grad_(True) for n, p in blk.named_parameters()}
    names = list(ref)
    lr = 1e-3
    opt = training.AdamW(blk.parameters(), lr=lr, weight_decay=0.1, state_bits=bits)
    ropt = torch.optim.AdamW([ref[n] for n in names], lr=lr, weight_decay=0.1)
    lengths = torch.tensor([T, 41, 0], dtype=torch.int32)
    live = {n: torch.ones_like(p, dtype=torch.bool) for n, p in ref.items()}
    for step in range(3):
        x, gy, gs = torch.randn(B, T, E), torch.randn(B, T, E), torch.randn(B, T, E)
        xc = x.cuda().requires_grad_(True)
        xr = x.double().requires_grad_(True)
        y, s = blk(xc, lengths.cuda())
        yr, sr = plain_block(ref, xr, lengths, causal)
        tol = 1e-4 if step == 0 else 3e-2          # (from the second step on the parameters differ as said above)
        assert rel(y, yr) <= tol and rel(s, sr) <= tol
        torch.autograd.backward([y, s], [gy.cuda(), gs.cuda()])
        torch.autograd.backward([yr, sr], [gy.double(), gs.double()])
        assert rel(xc.grad, xr.grad) <= tol
        if step == 0:
            for n, p in blk.named_parameters():
                big = ref[n].grad.abs().max()
                # (a key bias shifts all scores of a row alike: its gradient is zero but for rounding)
                if float(big) > 1e-9:
                    assert float((p.grad.double().cpu() - ref[n].grad).abs().max()) <= 1e-4 * float(big) + 1e-4, n
        for n, p in ref.items():
            live[n] &= p.grad.abs() > 1e-4 * p.grad.abs().max() + 1e-5
        opt.step()
        ropt.step()
        opt.zero_grad()
        ropt.zero_grad()
        for n, p in blk.named_parameters():
            d = ((p.detach().double().cpu() - ref[n].detach()).abs() * live[n])
            assert float(d.max()) <= 2 * lr * (step + 1), n
            if int(live[n].sum()) > 50:
                rms = float(d.square().sum().div(live[n].sum()).sqrt())
                assert rms <= lr * (step + 1) * (0.02 if bits == 32 or step == 0 else 0.125), (n, step, rms / lr)
    assert opt.t == 3


@pytest.mark.gpu
def test_bf16_block_runs_and_follows_f32():
    """Inside autocast the same block computes in bf16: outputs within 3 % of f32 in the norm (2^-8 per stage, the head
    norm multiplying what the difference of the maps leaves), gradients of the same direction."""
    sf = load_pkg()
    torch.manual_seed(1)
    blk = Block(sf, True).cuda()
    x = torch.randn(B, T, E, device="cuda")
    lengths = torch.tensor([T, 41, 7], dtype=torch.int32, device="cuda")
    y, s = blk(x, lengths)
    g = torch.randn_like(y)
    y.backward(g)
    ref = {n: p.grad.clone() for n, p in blk.named_parameters()}
    blk.zero_grad()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        yb, sb = blk(x, lengths)
    assert yb.dtype == torch.bfloat16
    assert float((yb.float() - y.detach()).norm() / y.detach().norm()) <= 0.03
    yb.backward(g.bfloat16())
    for n, p in blk.named_parameters():
        a, b = p.grad.float().flatten(), ref[n].flatten()
        if float(b.norm()) > 1e-3 * float(g.norm()):
            assert float(torch.dot(a, b) / (a.norm() * b.norm())) >= 0.98, n


def test_refusals():
    sf = load_pkg()
    with pytest.raises(NotImplementedError):
        sf.DifferentialAttention(60, 2)
    with pytest.raises(NotImplementedError):
        sf.DifferentialAttention(512, 2)
    with pytest.raises(ValueError):
        sf.DifferentialAttention(64, 2, 3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sf.DifferentialAttention(64, 2)(torch.zeros(1, 2, 64))


@pytest.mark.gpu
@pytest.mark.parametrize("amp", [False, True])
@pytest.mark.parametrize("shape", [(0, 5), (3, 0)])
def test_no_tokens(shape, amp):
    """A batch without samples and samples without tokens: an empty result, gradients of zero."""
    sf = load_pkg()
    m = sf.DifferentialAttention(E, H, KV).cuda()
    x = torch.zeros(*shape, E, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=amp):
        y = m(x, torch.zeros(shape[0], dtype=torch.int32, device="cuda"))
    assert y.shape == x.shape and y.dtype == torch.float32
    y.sum().backward()
    assert x.grad.shape == x.shape
    assert all(p.grad is None or float(p.grad.abs().sum()) == 0 for p in m.parameters())
