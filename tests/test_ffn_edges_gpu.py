"""Feed-forward operators on the GPU where their values or sizes are at an
edge: gates far in the lower tail, NaN and infinities, sizes past a kernel's
grid, parts of a gradient on their own.

Bounds are relative and counted in steps of fp32 (2^-23, `ULP`), plus one
rounding of the result to bf16 (plain.BF16).  A weight matrix of one non-zero
column makes a gate of every chosen value without any rounding."""
import math
import subprocess
import sys
from pathlib import Path

import pytest

from b200_gemm_b200 import _lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ffn_plain as plain  # noqa: E402

BF = torch.bfloat16
ULP = 2.0 ** -23
ROOT = Path(__file__).resolve().parent.parent


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


def _others_equal(got, ref, bad_rows=(), bad_cols=()):
    rows = [r for r in range(got.shape[0]) if r not in bad_rows]
    cols = [c for c in range(got.shape[1]) if c not in bad_cols]
    assert torch.equal(got[rows][:, cols], ref[rows][:, cols])


@pytest.mark.parametrize("kind", plain.ACTS)
@pytest.mark.parametrize("M", [5, 70])
def test_bad_values_of_the_gated_block(gpu_handle, M, kind):
    """A NaN among the weights or the activations is a NaN in every result that
    it is part of, under each activation, an infinity is nothing finite; the
    other results keep their bits."""
    x = plain.rows(M, 128, 1)
    wg, wu = (plain.rows(101, 128, i, 0.1) for i in (2, 3))
    H, G, U = gpu_handle.gated(x, wg, wu, activation=kind, save=True)
    for which, col in ((0, 7), (1, 100)):
        w = [wg.clone(), wu.clone()]
        w[which][col, 5] = float("nan")
        h, g, u = gpu_handle.gated(x, *w, activation=kind, save=True)
        assert h[:, col].isnan().all() and (g, u)[which][:, col].isnan().all()
        _others_equal(h, H, bad_cols=(col,))
        _others_equal((g, u)[1 - which], (G, U)[1 - which])
    y = x.clone()
    y[1, 9], y[4, 127] = float("nan"), float("-inf")
    h = gpu_handle.gated(y, wg, wu, activation=kind)
    assert h[1].isnan().all() and not h[4].isfinite().any()
    _others_equal(h, H, bad_rows=(1, 4))


@pytest.mark.parametrize("kind", plain.ACTS)
@pytest.mark.parametrize("M,F,K", [(40, 70, 64), (17, 1100, 72)])
def test_bad_values_of_the_gradients(gpu_handle, M, F, K, kind):
    """The same backward, for dX of one range and of several: a bad dH, G or U
    at (m, f) reaches row m of dX and row f of dWg or dWu."""
    args = {"dH": plain.rows(M, F, 0), "X": plain.rows(M, K, 1), "Wg": plain.rows(F, K, 2), "Wu": plain.rows(F, K, 3),
            "G": plain.rows(M, F, 4), "U": plain.rows(M, F, 5)}
    ref = gpu_handle.gated_backward(**args, activation=kind)
    m, f = 16, F - 1
    for name, value in (("dH", "nan"), ("G", "nan"), ("U", "nan"), ("dH", "inf"), ("U", "-inf")):
        bad = dict(args)
        t = plain.rows(M, F, {"dH": 0, "G": 4, "U": 5}[name])
        t[m, f] = float(value)
        bad[name] = t
        dx, dwg, dwu = gpu_handle.gated_backward(**bad, activation=kind)
        in_dg, in_du = name != "G" or kind != "none", name != "U"
        reached = [dx[m]] + ([dwg[f]] if in_dg else []) + ([dwu[f]] if in_du else [])
        assert all(r.isnan().all() if value == "nan" else not r.isfinite().any() for r in reached)
        _others_equal(dx, ref[0], bad_rows=(m,))
        _others_equal(dwg, ref[1], bad_rows=(f,) if in_dg else ())
        _others_equal(dwu, ref[2], bad_rows=(f,) if in_du else ())


@pytest.mark.parametrize("kind", plain.ACTS)
@pytest.mark.parametrize("M,group", [(3, 32), (3, 128), (12, 32), (12, 64), (40, 32), (40, 128)])
def test_bad_values_of_the_4bit_gated_block(gpu_handle, M, group, kind):
    x = plain.rows(M, 384, 1)
    gate, up = (plain.w4_random(150, 384, group, i) for i in (2, 3))
    H = gpu_handle.w4_gated(x, *gate, *up, activation=kind)
    for which, value in ((0, "nan"), (1, "nan"), (0, "inf"), (1, "-inf")):
        w = [gate, up]
        s = w[which][1].clone()
        s[-1, 149] = s[0, 3] = float(value)
        w[which] = (w[which][0], s)
        h = gpu_handle.w4_gated(x, *w[0], *w[1], activation=kind)
        assert h[:, [3, 149]].isnan().all()
        _others_equal(h, H, bad_cols=(3, 149))
    y = x.clone()
    y[0, 380], y[2, 0] = float("nan"), float("inf")
    h = gpu_handle.w4_gated(y, *gate, *up, activation=kind)
    assert h[0].isnan().all() and not h[2].isfinite().any()
    _others_equal(h, H, bad_rows=(0, 2))


@pytest.mark.parametrize("F", [65535 * 32, 65535 * 32 + 1])
def test_gated_few_rows_of_very_many_columns(gpu_handle, F):
    """The last width that the kernel for few rows can take, and the next one."""
    x = plain.rows(2, 8, 0)
    wg, wu = (torch.randn(F, 8, generator=torch.Generator("cuda").manual_seed(i), device="cuda").to(BF) for i in (1, 2))
    H = gpu_handle.gated(x, wg, wu, activation="relu")
    assert gpu_handle.last_device_status()[0] == 0
    g, eg = plain.product(x, wg)
    u, eu = plain.product(x, wu)
    plain.close(H, *plain.gated(g, eg, u, eu, "relu"))


@pytest.mark.parametrize("gated", [False, True])
def test_4bit_products_of_very_many_rows(gpu_handle, gated):
    """More rows of X than one launch's grid takes: 65535 blocks of 64."""
    M, N, K = 65535 * 64 + 5, 3, 32
    x = torch.randn(M, K, generator=torch.Generator("cuda").manual_seed(0), device="cuda").to(BF)
    gate, up = plain.w4_random(N, K, 32, 1), plain.w4_random(N, K, 32, 2)
    buf = torch.full((M + 1, N), 7.0, dtype=BF, device="cuda")
    if gated:
        gpu_handle.w4_gated(x, *gate, *up, activation="none", out=buf[:M])
    else:
        gpu_handle.w4_nt(x, *gate, out=buf[:M])
    assert gpu_handle.last_device_status()[0] == 0

    def product(codes, scales):
        # Two steps of 16 products of (q - 8) x, each of 17 terms truncated to
        # 2^-22 of the largest, at most 8 sum|x|; scaled, with a few roundings.
        w = plain.w4_values(codes, scales)
        x64 = x.double()
        err = 2 * 17 * 8 * 2.0 ** -22 * x64.abs().sum(1, keepdim=True) * scales.double() + 4 * ULP * (x64.abs() @ w.abs().t())
        return x64 @ w.t(), err

    g, eg = product(*gate)
    if gated:
        plain.close(buf[:M], *plain.gated(g, eg, *product(*up), "none"))
    else:
        plain.close(buf[:M], g, eg)
    assert (buf[M] == 7.0).all()


@pytest.mark.parametrize("M,F,K", [(500, 3000, 1000), (300, 4100, 520), (17, 1100, 72), (1, 5003, 2056), (640, 8200, 264)])
def test_input_gradient_on_its_own(gpu_handle, M, F, K):
    """dX has the same bits whether the weights' gradients are asked for or
    not, where its sum is split into ranges too."""
    size = _lib.load().b200gemm_gated_backward_workspace(gpu_handle._h, M, F, K)
    assert size > 4 * M * 8 * ((F + 7) // 8)  # a case that is split
    dh, g, u = (plain.rows(M, F, i) for i in range(3))
    x, wg, wu = plain.rows(M, K, 3), plain.rows(F, K, 4), plain.rows(F, K, 5)
    dx, dwg, dwu = gpu_handle.gated_backward(dh, x, wg, wu, g, u)
    assert torch.equal(gpu_handle.gated_backward(dh, x, wg, wu, g, u, weight_grad=False)[0], dx)
    parts = gpu_handle.gated_backward(dh, x, wg, wu, g, u, input_grad=False)
    assert torch.equal(parts[1], dwg) and torch.equal(parts[2], dwu)


_FIRST_CALLS = """
import sys
import torch
import b200_gemm_b200 as b200

BF = torch.bfloat16
g = torch.Generator("cuda").manual_seed(0)
r = lambda m, n: torch.randn(m, n, generator=g, device="cuda").to(BF)
h = b200.Gemm(0)
x, w, v, dh, gu = r(300, 256), r(520, 256), r(520, 256), r(300, 520), r(300, 520)
codes = torch.randint(0, 256, (520, 128), generator=g, device="cuda", dtype=torch.uint8)
scales = torch.full((2, 520), 0.01, dtype=BF, device="cuda")
calls = [
    lambda: h.gated(x[:2], w, v),
    lambda: h.gated(x, w, v, save=True)[0],
    lambda: torch.cat(h.gated_backward(dh, x, w, v, gu, gu)),
    lambda: torch.cat(h.gated_backward(dh[:17], x[:17], w, v, gu[:17], gu[:17])),
    lambda: h.w4_nt(x[:2], codes, scales),
    lambda: h.w4_nt(x[:40], codes, scales),
    lambda: h.w4_gated(x[:12], codes, scales, codes, scales),
    lambda: h.w4_quantize(w)[1],
    lambda: h.w4_dequantize(codes, scales),
]
for i in [int(a) for a in sys.argv[1:]]:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls[i]()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, calls[i]()), i
    del graph
assert h.last_device_status()[0] == 0
"""


@pytest.mark.parametrize("order", ["012345678", "876543210", "360"])
def test_first_calls_are_captured(order):
    """The first call of every kind in a process, made while a stream is
    captured: it loads its kernels and is replayed like any other."""
    run = subprocess.run([sys.executable, "-c", _FIRST_CALLS, *order], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("M", [1, 12, 20, 70])
def test_scales_of_both_signs(gpu_handle, M, group):
    """Scales of either sign and exactly zero; the bound is that of the sums of
    (q - 8) x over at most 128 k's: 8 steps of 16 products, each of 17 terms
    truncated to 2^-22 of the largest, at most 8 sum|x|; scaled and added up
    over K / 32 such sums."""
    N, K = 210, 1280
    x = plain.rows(M, K, 1)
    codes, scales = plain.w4_random(N, K, group, 2)
    gen = torch.Generator("cuda").manual_seed(3)
    scales = scales * (torch.randint(0, 3, scales.shape, generator=gen, device="cuda") - 1).to(BF)
    w, x64 = plain.w4_values(codes, scales), x.double()
    s = scales.double().abs().t().repeat_interleave(group, dim=1)
    err = 8 * 17 * 8 * 2.0 ** -22 * (x64.abs() @ s.t()) + (K / 32 + 16) * ULP * (x64.abs() @ w.abs().t())
    plain.close(gpu_handle.w4_nt(x, codes, scales, out_dtype=torch.float32), x64 @ w.t(), err, plain.F32)
    assert torch.equal(gpu_handle.w4_dequantize(codes, scales), w.to(BF))


def test_dequantize_among_subnormals(gpu_handle):
    """Scales down to the smallest bf16 subnormal: the scaled codes as they are."""
    codes, _ = plain.w4_random(64, 256, 32, 1)
    scales = (2.0 ** torch.linspace(-133, -120, 8 * 64, device="cuda").round()).reshape(8, 64).to(BF)
    assert torch.equal(gpu_handle.w4_dequantize(codes, scales), plain.w4_values(codes, scales).to(BF))
