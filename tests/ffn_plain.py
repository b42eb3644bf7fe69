"""64-bit forms of the feed-forward operators and the error bounds that their
tests use.

Bounds.  bf16 rounding is off by at most 2^-8 of the value (half a step), fp32
by 2^-24.  A sum of K products is accumulated in fp32 by the tensor cores, 16
products a step, each step rounding (or truncating) the running sum and the
products aligned to it: at most (K / 16 + 16) * 2^-22 * sum |products|.  The
activations use fast e^x and reciprocals, whose relative error stays below
2^-18 for the |x| < 20 of these tests: 2^-17 (1 + |x|) bounds the absolute
error of act(x) and act'(x)."""
import math

import torch

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
BF16 = 2.0 ** -8
F32 = 2.0 ** -24


def act(x, kind):
    """act(x) and act'(x) in x's type."""
    if kind == "silu":
        s = torch.sigmoid(x)
        return x * s, s + x * s * torch.sigmoid(-x)
    if kind == "gelu":
        phi = 0.5 * torch.special.erfc(-x / math.sqrt(2.0))
        return x * phi, phi + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (x + 0.044715 * x ** 3))
        return 0.5 * x * (1 + th), 0.5 * (1 + th) + 0.5 * x * (1 - th * th) * c * (1 + 3 * 0.044715 * x * x)
    if kind == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x)), (x > 0).to(x.dtype)
    return x, torch.ones_like(x)


def fn_err(x):
    return 2.0 ** -17 * (1 + x.abs())


def sum_err(K):
    return (K / 16 + 16) * 2.0 ** -22


def product(a, b):
    """a @ b^T in 64 bits and the bound of its fp32 sum."""
    a, b = a.double(), b.double()
    return a @ b.t(), sum_err(a.shape[1]) * (a.abs() @ b.abs().t())


def gated(g, eg, u, eu, kind):
    """act(g) * u and its bound, from g and u with their bounds."""
    a, _ = act(g, kind)
    ea = 1.2 * eg + fn_err(g) + 2.0 ** -22 * a.abs()  # |act'| < 1.2
    h = a * u
    return h, ea * u.abs() + a.abs() * eu + ea * eu


def grads(dh, g, u, kind):
    """dG, dU in 64 bits and the bounds of their bf16 values."""
    dh, g, u = dh.double(), g.double(), u.double()
    a, da = act(g, kind)
    dg, du = dh * u * da, dh * a
    return (dg, BF16 * dg.abs() + 1.01 * fn_err(g) * (dh * u).abs() + 1e-38,
            du, BF16 * du.abs() + 1.01 * fn_err(g) * dh.abs() + 1e-38)


def close(got, ref, err, rounding=BF16):
    """Whether every element is its reference within `err` and one rounding."""
    got = got.double()
    bound = err * (1 + rounding) + rounding * ref.abs() + 1e-38
    ok = (got - ref).abs() <= bound
    if not ok.all():
        worst = ((got - ref).abs() / bound).nan_to_num(nan=float("inf")).max()
        raise AssertionError(f"{int((~ok).sum())} of {ok.numel()} elements off, worst {worst:.3g} of the bound")


def rows(M, N, seed, std=1.0, pad=0, fill=float("nan"), device="cuda"):
    """A bf16 [M, N] view of a wider buffer whose other columns hold `fill`."""
    gen = torch.Generator().manual_seed(seed)
    pitch = 8 * ((N + 7) // 8) + pad
    full = torch.full((M, pitch), fill, dtype=torch.bfloat16)
    full[:, :N] = (torch.randn(M, N, generator=gen) * std).to(torch.bfloat16)
    return full.to(device)[:, :N]


def w4_values(codes, scales):
    """The weights that 4-bit codes stand for, in 64 bits."""
    N, K = codes.shape[0], 2 * codes.shape[1]
    q = torch.stack((codes % 16, codes // 16), dim=2).reshape(N, K).double() - 8
    return q * scales.double().t().repeat_interleave(K // scales.shape[0], dim=1)


def w4_quantize(w, group):
    """(codes, scales) by the definition, in 64 bits."""
    N, K = w.shape
    b = w.double().reshape(N, K // group, group)
    scales = (b.abs().amax(dim=2) / 7).to(torch.bfloat16)
    s = scales.double().unsqueeze(2)
    q = torch.where(s > 0, torch.round(b / s), torch.zeros_like(b)).nan_to_num(nan=0.0).clamp(-8, 7)
    q = (q + 8).to(torch.uint8).reshape(N, K)
    return q[:, 0::2] | (q[:, 1::2] << 4), scales.t().contiguous()


def w4_random(N, K, group, seed, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (N, K // 2), generator=gen, dtype=torch.uint8)
    scales = (torch.randn(K // group, N, generator=gen).abs() * 0.02 + 0.01).to(torch.bfloat16)
    return codes.to(device), scales.to(device)
