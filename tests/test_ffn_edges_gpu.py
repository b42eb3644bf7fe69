"""Feed-forward operators on the GPU where their values or sizes are at an
edge: gates far in the lower tail, NaN and infinities, sizes past a kernel's
grid, parts of a gradient on their own.

Bounds are relative and counted in steps of fp32 (2^-23, `ULP`), plus one
rounding of the result to bf16 (plain.BF16).  A weight matrix of one non-zero
column makes a gate of every chosen value without any rounding."""
import math

import pytest

from b200_gemm_b200 import _lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ffn_plain as plain  # noqa: E402

BF = torch.bfloat16
ULP = 2.0 ** -23


def _gates():
    """Every gate of 96 between -9 and -1/16, and the few around the derivative's zero."""
    g = torch.cat([torch.linspace(-9, -0.0625, 96), torch.tensor([-0.75, -0.7539, -5.25, -5.5, -5.75])])
    return g.to(BF).cuda()


def _tail(g, kind):
    """act(g), act'(g) for g < 0 in 64 bits without cancellation, and the bounds
    of their fp32 forms.

    gelu: Phi(g) = e^-a t P(t) with a = g^2 / 2: the fitted polynomial with its
    roundings is within 10.7 steps (by evaluation in fp32 over a fine grid), the
    reciprocal t within one, which counts 2.42 times; a's rounding a / 2, the
    fast exponential 2 + 1.173 a; four more products: 0.85 g^2 + 18 steps.  The
    derivative's second term has the exponential, its factors and the sum.
    gelu_tanh and silu: s = 1 / (1 + e^a), a's six roundings (3 a steps), the
    exponential, the sum and the reciprocal: 4.2 a + 4 steps; for g < 0 1 - s
    is at least 1/2, so its relative error is no larger."""
    g = g.double()
    if kind == "gelu":
        phi = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
        pdf = torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        r = (0.85 * g * g + 18) * ULP
        return g * phi, (g * phi).abs() * r, phi + g * pdf, phi * r + (g * pdf).abs() * (0.85 * g * g + 5) * ULP
    c = math.sqrt(8 / math.pi)
    z, dz = (c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g * g)) if kind == "gelu_tanh" else (g, torch.ones_like(g))
    s = torch.sigmoid(z)
    r = (4.2 * z.abs() + 5) * ULP
    second = g * s * torch.sigmoid(-z) * dz
    return g * s, (g * s).abs() * r, s + second, s * r + second.abs() * (2 * r + 8 * ULP)


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M", [1, 20, 140])
def test_lower_tail(gpu_handle, M, kind):
    """H keeps its relative accuracy where the activation is nearly 0: the
    kernel for few rows and the tiled one."""
    g = _gates()
    F = g.numel()
    x = torch.zeros(M, 8, dtype=BF, device="cuda")
    x[:, 0] = 1
    wg, wu = (torch.zeros(F, 8, dtype=BF, device="cuda") for _ in range(2))
    wg[:, 0], wu[:, 0] = g, 1
    a, ea, _, _ = _tail(g, kind)
    plain.close(gpu_handle.gated(x, wg, wu, activation=kind), a.expand(M, F), ea.expand(M, F))


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M", [1, 20])
def test_lower_tail_4bit(gpu_handle, M, kind):
    """The same with 4-bit weights: a gate is its group's scale times one."""
    g = _gates()
    F = g.numel()
    x = torch.zeros(M, 32, dtype=BF, device="cuda")
    x[:, 0] = 1
    codes = torch.full((F, 16), 0x88, dtype=torch.uint8, device="cuda")  # q - 8 = 0
    codes[:, 0] = 0x89
    a, ea, _, _ = _tail(g, kind)
    H = gpu_handle.w4_gated(x, codes, g[None].contiguous(), codes, torch.ones_like(g)[None].contiguous(), activation=kind)
    plain.close(H, a.expand(M, F), ea.expand(M, F))


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
def test_lower_tail_gradient(gpu_handle, kind):
    """dG and dU of one row, which dWg and dWu show as they are."""
    g = _gates()
    F = g.numel()
    G = torch.zeros(1, 8 * ((F + 7) // 8), dtype=BF, device="cuda")[:, :F]
    G[0] = g
    one = torch.ones_like(G)
    x = torch.zeros(1, 8, dtype=BF, device="cuda")
    x[:, 0] = 1
    w = torch.zeros(F, 8, dtype=BF, device="cuda")
    _, dwg, dwu = gpu_handle.gated_backward(one, x, w, w, G, one, activation=kind)
    a, ea, da, eda = _tail(g, kind)
    plain.close(dwu[:, 0], a, ea)
    plain.close(dwg[:, 0], da, eda)
