"""4-bit weights (Gemm.w4_quantize, w4_dequantize, w4_nt, w4_gated) on the GPU
against 64-bit forms, with the bounds derived in ffn_plain.py."""
import pytest

from b200_gemm_b200 import _lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ffn_plain as plain  # noqa: E402

BF = torch.bfloat16


def _w4_product(x, codes, scales):
    """X W^T in 64 bits and the bound of the kernel's sum.

    The kernels sum (q - 8) x, times a power of two, over at most 128 k's with
    at most 8 steps of 16 products: a step adds 17 terms, each truncated to
    2^-22 of a largest one of at most 8 sum|x|, so a scaled sum is off by at
    most 8 * 17 * 8 * 2^-22 s sum|x|.  Then one fp32 multiply-add per such sum
    (at least 32 k's), a few more over the warps and the cluster."""
    w = plain.w4_values(codes, scales)
    x = x.double()
    s = scales.double().t().repeat_interleave(x.shape[1] // scales.shape[0], dim=1)
    err = 8 * 2.0 ** -22 * 136 * (x.abs() @ s.t()) + (x.shape[1] / 32 + 16) * 2.0 ** -23 * (x.abs() @ w.abs().t())
    return x @ w.t(), err


def _check_nt(h, M, N, K, group, dtype=BF, seed=0, pad=0):
    x = plain.rows(M, K, seed, pad=pad)
    codes, scales = plain.w4_random(N, K, group, seed + 1)
    buf = torch.full((M + 2, N + 3), 7.0, dtype=dtype, device="cuda")
    out = buf[:M, :N]
    h.w4_nt(x, codes, scales, out=out)
    assert h.last_device_status()[0] == 0
    ref, err = _w4_product(x, codes, scales)
    plain.close(out, ref, err, plain.BF16 if dtype == BF else plain.F32)
    assert (buf[M:] == 7.0).all() and (buf[:, N:] == 7.0).all()


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("M,N,groups", [(1, 1, 1), (1, 64, 3), (2, 65, 5), (8, 130, 8), (9, 63, 9), (16, 200, 2),
                                        (17, 64, 7), (32, 257, 4), (33, 96, 3), (100, 70, 4)])
def test_nt(gpu_handle, M, N, groups, group):
    _check_nt(gpu_handle, M, N, groups * group, group, seed=M + N)


@pytest.mark.parametrize("M", [1, 12, 32])
def test_nt_f32(gpu_handle, M):
    _check_nt(gpu_handle, M, 200, 1024, 64, dtype=torch.float32, seed=M)


@pytest.mark.parametrize("M,N,K,group", [(1, 40, 16384, 32), (5, 3000, 8192, 128), (1, 10000, 512, 32),
                                         (30, 12000, 256, 256), (2, 100, 16416, 32)])
def test_nt_long(gpu_handle, M, N, K, group):
    """Long sums (K split over a cluster, more groups than are held at once),
    many rows of weights."""
    _check_nt(gpu_handle, M, N, K, group, seed=K, pad=16)


@pytest.mark.parametrize("kind", plain.ACTS)
@pytest.mark.parametrize("M,F,K,group", [(1, 33, 96, 32), (7, 100, 512, 128), (20, 1001, 320, 64), (64, 40, 256, 256)])
def test_gated(gpu_handle, M, F, K, group, kind):
    x = plain.rows(M, K, 1, pad=8)
    gate, up = plain.w4_random(F, K, group, 2), plain.w4_random(F, K, group, 3)
    buf = torch.full((M + 2, F + 1), 7.0, dtype=BF, device="cuda")
    gpu_handle.w4_gated(x, *gate, *up, activation=kind, out=buf[:M, :F])
    assert gpu_handle.last_device_status()[0] == 0
    g, eg = _w4_product(x, *gate)
    u, eu = _w4_product(x, *up)
    plain.close(buf[:M, :F], *plain.gated(g, eg, u, eu, kind))
    assert (buf[M:] == 7.0).all() and (buf[:, F:] == 7.0).all()


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("N,groups", [(1, 1), (31, 3), (33, 9), (200, 17)])
def test_quantize_and_back(gpu_handle, N, groups, group):
    """Codes and scales equal the definition's, and the values are the scaled
    codes rounded once."""
    K = groups * group
    w = plain.rows(N, K, N + K, K ** -0.5, pad=8)
    w[0, :group] = 0  # a group of zeros
    w[-1, -1] = 100.0
    codes, scales = gpu_handle.w4_quantize(w, group)
    ref_codes, ref_scales = plain.w4_quantize(w.cpu(), group)
    assert torch.equal(codes.cpu(), ref_codes)
    assert torch.equal(scales.cpu(), ref_scales)
    buf = torch.full((N + 1, K + 8), 7.0, dtype=BF, device="cuda")
    gpu_handle.w4_dequantize(codes, scales, out=buf[:N, :K])
    assert torch.equal(buf[:N, :K].cpu(), plain.w4_values(ref_codes, ref_scales).to(BF))
    assert (buf[N:] == 7.0).all() and (buf[:, K:] == 7.0).all()


def test_quantize_ties_and_tiny(gpu_handle):
    """w / s half way between two codes goes to the even one; scales among the
    subnormals; a scale that rounds to zero."""
    w = torch.zeros(4, 32, dtype=BF)
    w[0] = torch.tensor([7.0] + [v + 0.5 for v in range(-7, 7)] * 2 + [0.0, 1.0, 2.0])
    w[1] = torch.linspace(-1, 1, 32) * 2.0 ** -128
    w[2] = torch.linspace(-1, 1, 32) * 2.0 ** -132
    w[3, 0] = 2.0 ** -133                       # s = 2^-133 / 7 rounds to 0
    codes, scales = gpu_handle.w4_quantize(w.cuda(), 32)
    ref_codes, ref_scales = plain.w4_quantize(w, 32)
    assert torch.equal(scales.cpu(), ref_scales) and float(scales[0, 3]) == 0.0
    assert torch.equal(codes.cpu(), ref_codes)


def test_bad_groups_come_back_as_nan(gpu_handle):
    w = plain.rows(3, 128, 0)
    w[0, 3] = float("nan")
    w[1, 70] = float("inf")
    codes, scales = gpu_handle.w4_quantize(w, 64)
    v = gpu_handle.w4_dequantize(codes, scales)
    assert v[0, :64].isnan().all() and v[1, 64:].isnan().all()
    assert v[0, 64:].isfinite().all() and v[1, :64].isfinite().all() and v[2].isfinite().all()
    y = gpu_handle.w4_nt(plain.rows(2, 128, 1), codes, scales)
    assert y[:, :2].isnan().all() and y[:, 2].isfinite().all()


def test_bad_rows_stay_alone(gpu_handle):
    x = plain.rows(6, 256, 1)
    codes, scales = plain.w4_random(80, 256, 64, 2)
    ref = gpu_handle.w4_nt(x, codes, scales)
    y = x.clone()
    y[2, 9] = float("nan")
    y[4, 0] = float("inf")
    got = gpu_handle.w4_nt(y, codes, scales)
    keep = [0, 1, 3, 5]
    assert torch.equal(got[keep], ref[keep]) and got[2].isnan().all() and not got[4].isfinite().any()


def test_block_as_it_is_served(gpu_handle):
    """A trained block quantised, then decoded: gated and down projection on 4
    bits against the bf16 kernels on the dequantised weights.

    The two differ by roundings alone: each side's H by its sums' bounds and
    one rounding, carried through the down projection, and its own."""
    h = gpu_handle
    M, D, F = 3, 256, 320
    x = plain.rows(M, D, 0)
    wg, wu, wd = plain.rows(F, D, 1, D ** -0.5), plain.rows(F, D, 2, D ** -0.5), plain.rows(D, F, 3, F ** -0.5)
    q = [h.w4_quantize(w, 32) for w in (wg, wu, wd)]
    H = h.w4_gated(x, *q[0], *q[1])
    y = h.w4_nt(H, *q[2])
    g, eg = _w4_product(x, *q[0])
    u, eu = _w4_product(x, *q[1])
    r, er = plain.gated(g, eg, u, eu, "silu")
    plain.close(H, r, er)
    ref, err = _w4_product(H, *q[2])
    plain.close(y, ref, err)
    # prefill: the values back as bf16 (rounded: 2^-8 each) through the bf16 kernels
    d = [h.w4_dequantize(*p) for p in q]
    Hb = h.gated(x, d[0], d[1])
    g2, eg2 = plain.product(x, d[0])
    u2, eu2 = plain.product(x, d[1])
    plain.close(Hb, *plain.gated(g2, eg2, u2, eu2, "silu"))


def test_streams_graphs_and_overlap(gpu_handle):
    h = gpu_handle
    x = plain.rows(2, 1024, 0)
    gate, up, down = (plain.w4_random(1024, 1024, 128, s) for s in (1, 2, 3))

    def step(stream=None):
        y = x
        for _ in range(3):
            y = h.w4_nt(h.w4_gated(y, *gate, *up, activation="silu", stream=stream), *down, stream=stream)
            y = y.clamp(-4, 4) if stream is None else y
        return y

    def chain(stream=None):
        y = x
        for _ in range(4):
            y = h.w4_nt(y, *down, stream=stream)
        return y

    ref, cref = step(), chain()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = chain(side)
    torch.cuda.synchronize()
    assert torch.equal(got, cref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
    del graph
    for mode in (_lib.PDL_ON, _lib.PDL_WEIGHTS_EARLY):
        h.set_pdl(mode)
        try:
            for _ in range(10):
                assert torch.equal(chain(), cref)
        finally:
            h.set_pdl(_lib.PDL_OFF)


def test_refusals(gpu_handle):
    h = gpu_handle
    x = plain.rows(2, 128, 0)
    codes, scales = plain.w4_random(64, 128, 32, 1)
    e = lambda *s, t=BF: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731
    with pytest.raises(ValueError):
        h.w4_quantize(plain.rows(4, 96, 0), 64)           # 64 does not divide 96
    with pytest.raises(ValueError):
        h.w4_quantize(plain.rows(4, 96, 0), 48)
    with pytest.raises(TypeError):
        h.w4_nt(x, codes.to(torch.int8), scales)
    with pytest.raises(TypeError):
        h.w4_nt(x, codes, scales.float())
    with pytest.raises(ValueError):
        h.w4_nt(x, codes, scales[:3])
    with pytest.raises(ValueError):
        h.w4_nt(x, codes, scales.t().contiguous().t())
    with pytest.raises(ValueError):
        h.w4_nt(x[:, :64], codes, scales)
    with pytest.raises(ValueError):
        h.w4_nt(x, codes.cpu(), scales.cpu())
    with pytest.raises(TypeError):
        h.w4_nt(x, codes, scales, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        h.w4_gated(x, codes, scales, *plain.w4_random(64, 128, 64, 1))
    with pytest.raises(ValueError):
        h.w4_gated(x, codes, scales, *plain.w4_random(32, 128, 32, 1))
    with pytest.raises(_lib.B200GemmError) as err:
        h.w4_nt(x, codes, scales, out=x[:, :64])          # writes over A
    assert err.value.code == _lib.ERR_INVALID_ARG
    assert h.w4_nt(e(0, 128), codes, scales).shape == (0, 64)
    assert h.w4_dequantize(e(0, 64, t=torch.uint8), e(4, 0)).shape == (0, 128)


@pytest.mark.parametrize("group", [32, 64, 256])
@pytest.mark.parametrize("M,N,K", [(17, 1, 256), (32, 129, 768), (25, 8192, 1024), (40, 30000, 512), (33, 400, 8448),
                                   (300, 130, 256)])
def test_nt_more_rows(gpu_handle, M, N, K, group):
    """17 rows and more: blocks of 128 rows of weights that end anywhere, one
    and two of them per CTA, K split over clusters, several blocks of rows of X."""
    _check_nt(gpu_handle, M, N, K, group, seed=N, pad=8)


@pytest.mark.parametrize("M,F,K,group", [(17, 1, 32, 32), (32, 130, 4096, 64), (31, 14000, 256, 128), (50, 300, 8192, 32)])
def test_gated_more_rows(gpu_handle, M, F, K, group):
    x = plain.rows(M, K, 1)
    gate, up = plain.w4_random(F, K, group, 2), plain.w4_random(F, K, group, 3)
    out = gpu_handle.w4_gated(x, *gate, *up, activation="gelu")
    assert gpu_handle.last_device_status()[0] == 0
    plain.close(out, *plain.gated(*_w4_product(x, *gate), *_w4_product(x, *up), "gelu"))


def test_more_rows_bad_values(gpu_handle):
    """The same as with a few rows: a bad row of X or group of W reaches its own results only."""
    x = plain.rows(40, 256, 1)
    codes, scales = plain.w4_random(300, 256, 64, 2)
    ref = gpu_handle.w4_nt(x, codes, scales)
    y = x.clone()
    y[2, 9] = float("nan")
    y[35, 0] = float("inf")
    got = gpu_handle.w4_nt(y, codes, scales)
    keep = [i for i in range(40) if i not in (2, 35)]
    assert torch.equal(got[keep], ref[keep]) and got[2].isnan().all() and not got[35].isfinite().any()
    bad = scales.clone()
    bad[3, 7], bad[0, 299], bad[1, 140] = float("nan"), float("inf"), float("-inf")
    got = gpu_handle.w4_nt(x, codes, bad)
    keep = [n for n in range(300) if n not in (7, 299, 140)]
    assert torch.equal(got[:, keep], ref[:, keep]) and got[:, [7, 299, 140]].isnan().all()


@pytest.mark.parametrize("M", [3, 20])
def test_scales_of_any_size(gpu_handle, M):
    """Scales and activations that are powers of two shift the results by their
    exponents and nothing else: 2^120 * 2^-110 as 1 * 1, and 2^-100 * 2^90."""
    x = plain.rows(M, 512, 1)
    codes, scales = plain.w4_random(70, 512, 128, 2)
    ref = gpu_handle.w4_nt(x, codes, scales)
    for s, v in ((110, -100), (-100, 90)):
        got = gpu_handle.w4_nt(x * 2.0 ** v, codes, scales * 2.0 ** s)
        assert torch.equal(got.float() * 2.0 ** -(s + v), ref.float())


def test_more_rows_repeat_exactly(gpu_handle):
    """No atomics: the same call gives the same bits."""
    x = plain.rows(70, 8192, 1)
    codes, scales = plain.w4_random(900, 8192, 32, 2)
    ref = gpu_handle.w4_nt(x, codes, scales, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(gpu_handle.w4_nt(x, codes, scales, out_dtype=torch.float32), ref)


def test_more_rows_streams_graphs_and_overlap(gpu_handle):
    """Calls at once on two streams (kernels that take a whole SM each, in
    clusters), a captured and replayed one, and launches that overlap."""
    h = gpu_handle
    sets = [(plain.rows(m, k, m), plain.w4_random(n, k, 64, n)) for m, n, k in
            ((20, 400, 8192), (32, 9000, 1024), (24, 2048, 4096), (70, 30000, 512))]
    ref = [h.w4_nt(x, *w) for x, w in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = [[torch.empty_like(r) for r in ref] for _ in range(2)]
    for _ in range(25):
        for s, results in zip(streams, out):
            for i in (0, 1, 2, 3) if s is streams[0] else (2, 0, 3, 1):
                h.w4_nt(sets[i][0], *sets[i][1], out=results[i], stream=s)
    torch.cuda.synchronize()
    assert h.last_device_status()[0] == 0
    for results in out:
        assert all(torch.equal(a, b) for a, b in zip(results, ref))

    x = plain.rows(24, 2048, 5)
    gate, up, down = (plain.w4_random(2048, 2048, 32, s) for s in (1, 2, 3))

    def step():
        y = x
        for _ in range(3):
            y = h.w4_nt(h.w4_gated(y, *gate, *up, activation="gelu"), *down).mul_(2.0 ** -12)
        return y

    def chain():
        y = x
        for _ in range(4):
            y = h.w4_nt(y, *down)
        return y

    want, cwant = step(), chain()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        got.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    del graph
    for mode in (_lib.PDL_ON, _lib.PDL_WEIGHTS_EARLY):
        h.set_pdl(mode)
        try:
            for _ in range(10):
                assert torch.equal(chain(), cwant)
        finally:
            h.set_pdl(_lib.PDL_OFF)


@pytest.mark.parametrize("M", [16, 20])
def test_nt_far_rows(gpu_handle, M):
    """A result whose last rows lie past 2^31 elements."""
    x, w = plain.rows(M, 128, 0), plain.w4_random(40, 128, 32, 1)
    pitch = 2 ** 31 // (M - 2)
    buf = torch.empty((M - 1) * pitch + 40, dtype=BF, device="cuda")
    out = torch.as_strided(buf, (M, 40), (pitch, 1))
    gpu_handle.w4_nt(x, *w, out=out)
    assert torch.equal(out, gpu_handle.w4_nt(x, *w))


@pytest.mark.parametrize("M,F,K,group", [(9, 13000, 256, 64), (16, 14336, 384, 128), (12, 12500, 512, 32),
                                         (16, 20000, 256, 256)])
def test_gated_many_rows_of_weights(gpu_handle, M, F, K, group):
    """More rows of weights than the kernel for a few rows holds at once."""
    x = plain.rows(M, K, 1)
    gate, up = plain.w4_random(F, K, group, 2), plain.w4_random(F, K, group, 3)
    out = gpu_handle.w4_gated(x, *gate, *up, activation="silu")
    assert gpu_handle.last_device_status()[0] == 0
    plain.close(out, *plain.gated(*_w4_product(x, *gate), *_w4_product(x, *up), "silu"))


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("M,N,K", [(64, 300, 2304), (65, 100, 256), (128, 7000, 1280)])
def test_nt_blocks_of_64_rows(gpu_handle, M, N, K, group):
    _check_nt(gpu_handle, M, N, K, group, dtype=torch.float32, seed=M, pad=8)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_gated_blocks_of_64_rows(gpu_handle, group):
    x = plain.rows(90, 1536, 1)
    gate, up = plain.w4_random(3000, 1536, group, 2), plain.w4_random(3000, 1536, group, 3)
    out = gpu_handle.w4_gated(x, *gate, *up, activation="relu")
    plain.close(out, *plain.gated(*_w4_product(x, *gate), *_w4_product(x, *up), "relu"))
