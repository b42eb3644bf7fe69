"""Gated feed-forward block (Gemm.gated, Gemm.gated_backward) on the GPU
against 64-bit forms, with the bounds derived in ffn_plain.py."""
import ctypes

import pytest

from b200_gemm_b200 import _lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ffn_plain as plain  # noqa: E402

BF = torch.bfloat16


def _check_gated(h, M, F, K, kind, save, pad=0, seed=0):
    x = plain.rows(M, K, seed, pad=pad)
    wg, wu = (plain.rows(F, K, seed + i, K ** -0.5, pad=pad) for i in (1, 2))
    pitch = 8 * ((F + 7) // 8) + 8
    # two rows below and the columns beside the results must stay as they are
    bufs = [torch.full((M + 2, pitch), 7.0, dtype=BF, device="cuda") for _ in range(3 if save else 1)]
    outs = [b[:M, :F] for b in bufs]
    if save:
        h.gated(x, wg, wu, activation=kind, out=outs[0], gate_out=outs[1], up_out=outs[2])
    else:
        h.gated(x, wg, wu, activation=kind, out=outs[0])
    assert h.last_device_status()[0] == 0
    g, eg = plain.product(x, wg)
    u, eu = plain.product(x, wu)
    plain.close(outs[0], *plain.gated(g, eg, u, eu, kind))
    if save:
        plain.close(outs[1], g, eg)
        plain.close(outs[2], u, eu)
    for b in bufs:
        assert (b[M:] == 7.0).all() and (b[:, F:] == 7.0).all()


# rows at and around the few-rows limit (32) and the 128-row halves and 256-row
# tiles; widths that end inside a 16-byte group, a 32-column chunk, a tile
@pytest.mark.parametrize("kind", plain.ACTS)
@pytest.mark.parametrize("M,F,K", [(1, 64, 64), (3, 1, 8), (8, 33, 136), (9, 257, 512), (17, 130, 1032), (32, 300, 264),
                                   (33, 131, 200), (129, 255, 64), (257, 520, 328)])
def test_gated(gpu_handle, M, F, K, kind):
    _check_gated(gpu_handle, M, F, K, kind, save=kind == "gelu", seed=M + F)


@pytest.mark.parametrize("M,F,K", [(1, 14000, 4096), (8, 5001, 2056), (12, 3001, 4096), (32, 6000, 2048), (1, 40, 8192),
                                   (100, 300, 4104), (65, 70, 2048), (20, 9500, 520)])
def test_gated_few_rows_long(gpu_handle, M, F, K):
    """Few rows against many and long weights: every ring goes around many
    times, every SM holds several blocks; and a width that splits K."""
    _check_gated(gpu_handle, M, F, K, "silu", save=M % 2 == 0, seed=M)


@pytest.mark.parametrize("width", [512, 256, 192, 128])
@pytest.mark.parametrize("save", [False, True])
@pytest.mark.parametrize("M,F,K", [(1, 7, 8), (300, 1001, 520), (2, 128, 64)])
def test_gated_tiled(gpu_handle, M, F, K, width, save):
    """Every tile width of the tiled kernel, whatever the rule would pick."""
    gpu_handle.set_tile_width(width)
    try:
        _check_gated(gpu_handle, M, F, K, "silu", save, pad=24, seed=K)
    finally:
        gpu_handle.set_tile_width(0)


@pytest.mark.parametrize("M", [1, 32, 100])
def test_gated_row_strides(gpu_handle, M):
    """Activations and weights that are slices of wider matrices, whose other
    columns hold NaN."""
    _check_gated(gpu_handle, M, 200, 104, "gelu_tanh", save=M == 100, pad=64, seed=9)


def test_gated_many_tiles(gpu_handle):
    """More tiles than clusters, several bands of tile rows."""
    _check_gated(gpu_handle, 4500, 1100, 136, "silu", save=True, seed=4)


@pytest.mark.parametrize("M", [5, 70])
def test_gated_bad_rows_stay_alone(gpu_handle, M):
    """A row with an infinity or NaN does not touch the others."""
    h = gpu_handle
    x = plain.rows(M, 128, 1)
    wg, wu = (plain.rows(96, 128, i, 0.1) for i in (2, 3))
    ref = h.gated(x, wg, wu)
    y = x.clone()
    y[1, 5] = float("nan")
    y[3, 7] = float("inf")
    got = h.gated(y, wg, wu)
    keep = [r for r in range(M) if r not in (1, 3)]
    assert torch.equal(got[keep].view(torch.int16), ref[keep].view(torch.int16))
    assert got[1].isnan().all() and not got[3].isfinite().all()


def test_gated_far_rows(gpu_handle):
    """Row offsets past 2^31 elements, for the TMA and the element stores."""
    M, F, K, ld = 300, 37, 64, 1 << 23
    x = plain.rows(M, K, 1)
    wg, wu = (plain.rows(F, K, i, 0.1) for i in (2, 3))
    buf = torch.empty(M * ld, dtype=BF, device="cuda")
    out = buf.as_strided((M, F), (ld, 1))
    gpu_handle.gated(x, wg, wu, out=out)
    assert torch.equal(out.contiguous().view(torch.int16), gpu_handle.gated(x, wg, wu).contiguous().view(torch.int16))


def _backward_raw(h, dh, x, wg, wu, g, u, kind, workspace, dx, dwg, dwu):
    M, F = dh.shape
    K = x.shape[1]
    lib = _lib.load()
    rc = lib.b200gemm_bf16_gated_backward(
        h._h, M, F, K, dh.data_ptr(), dh.stride(0), x.data_ptr(), x.stride(0), wg.data_ptr(), wu.data_ptr(),
        wg.stride(0), g.data_ptr(), u.data_ptr(), g.stride(0),
        {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}[kind], dx.data_ptr(), dx.stride(0),
        dwg.data_ptr(), dwu.data_ptr(), dwg.stride(0), workspace.data_ptr(), workspace.numel(),
        torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert h.last_device_status()[0] == 0


def _check_backward(h, M, F, K, kind, pad=0, seed=0, small_workspace=False):
    dh = plain.rows(M, F, seed, 0.1, pad=pad)
    g, u = (plain.rows(M, F, seed + i, 1.5, pad=pad) for i in (1, 2))
    x = plain.rows(M, K, seed + 3, pad=pad)
    wg, wu = (plain.rows(F, K, seed + i, K ** -0.5, pad=pad) for i in (4, 5))
    f8 = 8 * ((F + 7) // 8)
    base = 4 * M * f8
    size = _lib.load().b200gemm_gated_backward_workspace(h._h, M, F, K)
    assert size >= base
    buf = torch.full((base if small_workspace else size,), 255, dtype=torch.uint8, device="cuda")  # NaN, as it happens
    ws = buf[:base].view(BF).view(2, M, f8)
    outs = [torch.full((r + 2, K + 8), 7.0, dtype=BF, device="cuda") for r in (M, F, F)]
    dx, dwg, dwu = (b[:r, :K] for b, r in zip(outs, (M, F, F)))
    _backward_raw(h, dh, x, wg, wu, g, u, kind, buf, dx, dwg, dwu)
    # dG and dU element by element, then the products of what they were rounded to
    rdg, edg, rdu, edu = plain.grads(dh, g, u, kind)
    dg, du = ws[0, :, :F].double(), ws[1, :, :F].double()
    assert ((dg - rdg).abs() <= edg).all()
    assert ((du - rdu).abs() <= edu).all()
    assert (ws[:, :, F:] == 0).all()
    ref = dg @ wg.double() + du @ wu.double()
    err = plain.sum_err(2 * f8) * (dg.abs() @ wg.double().abs() + du.abs() @ wu.double().abs())
    plain.close(dx, ref, err)
    for d, got in ((dg, dwg), (du, dwu)):
        plain.close(got, *plain.product(d.t(), x.t()))
    for b, r in zip(outs, (M, F, F)):
        assert (b[r:] == 7.0).all() and (b[:, K:] == 7.0).all()


@pytest.mark.parametrize("kind", plain.ACTS)
@pytest.mark.parametrize("M,F,K", [(1, 1, 8), (1, 300, 72), (63, 65, 64), (200, 131, 520), (513, 257, 264)])
def test_backward(gpu_handle, M, F, K, kind):
    _check_backward(gpu_handle, M, F, K, kind, seed=M + F)


@pytest.mark.parametrize("width", [512, 256, 128])
@pytest.mark.parametrize("M,F,K", [(130, 70, 136), (700, 1030, 1160)])
def test_backward_tiled(gpu_handle, M, F, K, width):
    gpu_handle.set_tile_width(width)
    try:
        _check_backward(gpu_handle, M, F, K, "silu", pad=16, seed=3)
    finally:
        gpu_handle.set_tile_width(0)


@pytest.mark.parametrize("M,F,K", [(1, 5003, 2056), (40, 9000, 264), (300, 4100, 520), (17, 1100, 72)])
@pytest.mark.parametrize("small_workspace", [False, True])
def test_backward_split(gpu_handle, M, F, K, small_workspace):
    """dX of few tiles: its sum in ranges, with partial sums in the workspace;
    and without, when the workspace has no room for them."""
    size = _lib.load().b200gemm_gated_backward_workspace(gpu_handle._h, M, F, K)
    assert size > 4 * M * 8 * ((F + 7) // 8)  # a case that is split
    _check_backward(gpu_handle, M, F, K, "silu", seed=M, small_workspace=small_workspace)


def test_backward_many_tiles(gpu_handle):
    _check_backward(gpu_handle, 4400, 2100, 1288, "gelu", seed=8)


def test_backward_parts(gpu_handle):
    """Only the input's or only the weights' gradient: the same values."""
    h = gpu_handle
    M, F, K = 90, 130, 264
    dh, g, u = (plain.rows(M, F, i) for i in range(3))
    x, wg, wu = plain.rows(M, K, 3), plain.rows(F, K, 4), plain.rows(F, K, 5)
    dx, dwg, dwu = h.gated_backward(dh, x, wg, wu, g, u)
    a = h.gated_backward(dh, x, wg, wu, g, u, weight_grad=False)
    b = h.gated_backward(dh, x, wg, wu, g, u, input_grad=False)
    assert a[1] is None and a[2] is None and b[0] is None
    assert torch.equal(a[0], dx) and torch.equal(b[1], dwg) and torch.equal(b[2], dwu)


def test_backward_empty_sums(gpu_handle):
    h = gpu_handle
    e = lambda *s: torch.empty(*s, dtype=BF, device="cuda")  # noqa: E731
    dx, dwg, dwu = h.gated_backward(e(0, 24), e(0, 16), e(24, 16), e(24, 16), e(0, 24), e(0, 24))
    assert dx.shape == (0, 16) and (dwg == 0).all() and (dwu == 0).all()
    dx, dwg, dwu = h.gated_backward(e(5, 0), e(5, 16), e(0, 16), e(0, 16), e(5, 0), e(5, 0))
    assert (dx == 0).all() and dwg.shape == (0, 16)
    assert h.gated(e(0, 16), e(24, 16), e(24, 16)).shape == (0, 24)
    assert h.gated(e(5, 16), e(0, 16), e(0, 16)).shape == (5, 0)


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_backward_extreme_gates(gpu_handle, kind):
    """Gates far out in both tails: act' is 1 above and 0 below, no NaN."""
    M, F, K = 4, 16, 8
    g = torch.zeros(M, F, dtype=BF, device="cuda")
    g[0], g[1], g[2], g[3] = 1e4, -1e4, 3e38, -3e38
    one = torch.ones(M, F, dtype=BF, device="cuda")
    x, w = torch.ones(M, K, dtype=BF, device="cuda"), torch.full((F, K), 2.0 ** -130, dtype=BF, device="cuda")
    buf = torch.empty(4 * M * F, dtype=torch.uint8, device="cuda")
    ws = buf.view(BF).view(2, M, F)
    dx, dwg, dwu = (torch.empty(r, K, dtype=BF, device="cuda") for r in (M, F, F))
    _backward_raw(gpu_handle, one, x, w, w, g, one, kind, buf, dx, dwg, dwu)
    assert torch.equal(ws[0, :, 0].float().cpu(), torch.tensor([1.0, 0.0, 1.0, 0.0]))
    assert (ws[1, 1] == 0).all() and (ws[1, 3] == 0).all()
    assert torch.equal(ws[1, 0], g[0]) and torch.equal(ws[1, 2], g[2])


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_training_step_against_differences(gpu_handle, kind):
    """Forward and backward as a training step runs them: the slope of
    sum(dH * H) along random directions of X, Wg and Wu against central
    differences of the 64-bit block.

    Bound: G, U, dG and dU are each rounded to bf16 and so are the results:
    relative errors of at most 2^-8 of every term |dH U act'(G) (dG)| and
    |dH act(G) (dU)| from dG or dU, from U or act(G), and from the result
    itself, and act'' < 1.1 turns G's rounding into at most 2^-8 |G| 1.1 of
    act'.  5 * 2^-8 of the terms' absolute sums (products of the direction
    with |weights|, |inputs|) covers them; the differences' own error, of the
    order of 1e-6, is far below."""
    h = gpu_handle
    M, F, K = 40, 72, 64
    x = plain.rows(M, K, 0)
    wg, wu = (plain.rows(F, K, i, K ** -0.5) for i in (1, 2))
    dh = plain.rows(M, F, 3)
    H, G, U = h.gated(x, wg, wu, activation=kind, save=True)
    dx, dwg, dwu = h.gated_backward(dh, x, wg, wu, G, U, activation=kind)
    x64, wg64, wu64, dh64 = x.double(), wg.double(), wu.double(), dh.double()

    def loss(a, b, c):
        return (dh64 * plain.act(a @ b.t(), kind)[0] * (a @ c.t())).sum()

    g, u = x64 @ wg64.t(), x64 @ wu64.t()
    a, da = plain.act(g, kind)
    tg = (dh64 * u).abs() * (da.abs() + 1.1 * g.abs())   # weight of an error in a column of G
    tu = dh64.abs() * (a.abs() + 1.2 * g.abs())
    for seed in range(3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        v = [torch.randn(t.shape, generator=gen, device="cuda", dtype=torch.float64) for t in (x, wg, wu)]
        eps = 1e-4
        slope = (loss(x64 + eps * v[0], wg64 + eps * v[1], wu64 + eps * v[2]) -
                 loss(x64 - eps * v[0], wg64 - eps * v[1], wu64 - eps * v[2])) / (2 * eps)
        got = sum((d.double() * w).sum() for d, w in zip((dx, dwg, dwu), v))
        terms = (tg * (v[0].abs() @ wg64.abs().t() + x64.abs() @ v[1].abs().t()) +
                 tu * (v[0].abs() @ wu64.abs().t() + x64.abs() @ v[2].abs().t())).sum()
        assert abs(got - slope) <= 5 * 2.0 ** -8 * terms
        # and far tighter on average: errors of 40 * 72 * 64 terms of random sign
        assert abs(got - slope) <= 0.1 * (5 * 2.0 ** -8 * terms)


def test_streams_and_graphs(gpu_handle):
    """On a side stream, on two at once, and captured from the first call on;
    two graphs of the same handle replayed in turn."""
    h = gpu_handle
    M, F, K = 280, 136, 192
    sets = []
    for s in range(2):
        x, dh = plain.rows(M, K, 10 * s), plain.rows(M, F, 10 * s + 1)
        wg, wu = plain.rows(F, K, 10 * s + 2, 0.1), plain.rows(F, K, 10 * s + 3, 0.1)
        sets.append((x, wg, wu, dh))

    def step(x, wg, wu, dh, stream=None):
        H, G, U = h.gated(x, wg, wu, save=True, stream=stream)
        return (H, *h.gated_backward(dh, x, wg, wu, G, U, stream=stream), h.gated(x[:3], wg, wu, stream=stream))

    ref = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = [step(*s, stream=st) for s, st in zip(sets, streams)]
    raw = step(*sets[0], stream=streams[1].cuda_stream)
    torch.cuda.synchronize()
    for r, o in zip(ref, got):
        assert all(torch.equal(a, b) for a, b in zip(r, o))
    assert all(torch.equal(a, b) for a, b in zip(ref[0], raw))
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*s))
        graphs.append(graph)
    for _ in range(3):
        for o in outs:
            for t in o:
                t.fill_(float("nan"))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for r, o in zip(ref, outs):
            assert all(torch.equal(a, b) for a, b in zip(r, o))
    assert h.last_device_status()[0] == 0
    del graphs


@pytest.mark.parametrize("mode", [_lib.PDL_ON, _lib.PDL_WEIGHTS_EARLY])
def test_launch_overlap_chain(gpu_handle, mode):
    """Few-row calls that read the previous call's output, with launch overlap."""
    h = gpu_handle
    x = plain.rows(4, 512, 0)
    w = [(plain.rows(512, 512, 2 * i + 1, 0.05), plain.rows(512, 512, 2 * i + 2, 0.05)) for i in range(6)]

    def chain():
        y = x
        for wg, wu in w:
            y = h.gated(y, wg, wu, activation="none")
        return y

    ref = chain()
    h.set_pdl(mode)
    try:
        for _ in range(10):
            assert torch.equal(chain(), ref)
    finally:
        h.set_pdl(_lib.PDL_OFF)


def test_same_result_twice(gpu_handle):
    h = gpu_handle
    x, wg, wu = plain.rows(20, 2048, 0), plain.rows(100, 2048, 1, 0.02), plain.rows(100, 2048, 2, 0.02)
    ref = h.gated(x, wg, wu)
    for _ in range(5):
        assert torch.equal(h.gated(x, wg, wu), ref)


def test_refusals(gpu_handle):
    h = gpu_handle
    x, w = plain.rows(4, 64, 0), plain.rows(16, 64, 1)
    hh = plain.rows(4, 16, 2)
    with pytest.raises(TypeError):
        h.gated(x.float(), w, w)
    with pytest.raises(ValueError):
        h.gated(x.cpu(), w, w)
    with pytest.raises(ValueError):
        h.gated(x, w, w[:, :32])
    with pytest.raises(ValueError):
        h.gated(x, w, w, activation="tanh")
    with pytest.raises(ValueError):
        h.gated(x, w, plain.rows(16, 64, 1, pad=8))       # another row stride
    with pytest.raises(ValueError):
        h.gated(x, w.t().contiguous().t(), w)
    with pytest.raises(ValueError):
        h.gated(x, w, w, out=torch.empty(4, 17, dtype=BF, device="cuda"))
    with pytest.raises(_lib.B200GemmError) as e:
        h.gated(x[:, :60], w[:, :60], w[:, :60])          # K % 8
    assert e.value.code == _lib.ERR_UNSUPPORTED
    with pytest.raises(_lib.B200GemmError) as e:
        h.gated(x, w, w, out=x[:, :16])                   # writes over X
    assert e.value.code == _lib.ERR_INVALID_ARG
    with pytest.raises(_lib.B200GemmError) as e:
        h.gated(x, w, w, out=hh, gate_out=hh, up_out=hh.clone())
    assert e.value.code == _lib.ERR_INVALID_ARG
    both = torch.empty(4, 32, dtype=BF, device="cuda")    # halves of one buffer are fine
    h.gated(x, w, w, gate_out=both[:, :16], up_out=both[:, 16:])
    with pytest.raises(ValueError):
        h.gated_backward(hh, x, w, w, hh, plain.rows(4, 16, 2, pad=8))
    with pytest.raises(ValueError):
        h.gated_backward(hh, x[:3], w, w, hh, hh)
    assert ctypes.sizeof(ctypes.c_longlong) == 8
