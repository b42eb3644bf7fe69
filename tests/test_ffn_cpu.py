"""Refusals of the feed-forward entry points, without a GPU: a call that is
refused returns before any CUDA call, so a zeroed stand-in serves as the
handle and made-up addresses as the matrices."""
import ctypes

import pytest

from b200_gemm_b200 import _lib

OK, INVALID, UNSUPPORTED, TOO_LARGE = _lib.OK, _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED, _lib.ERR_TOO_LARGE
HANDLE = ctypes.create_string_buffer(1 << 16)
H = ctypes.cast(HANDLE, ctypes.c_void_p)


def _at(i):
    return (i + 1) << 36  # far apart


def _gated(handle=H, M=4, F=16, K=64, X=_at(0), ldx=64, Wg=_at(1), Wu=_at(2), ldw=64, act=4, out=_at(3), ldh=16, G=None,
           U=None, ldgu=16):
    return _lib.load().b200gemm_bf16_gated(handle, M, F, K, X, ldx, Wg, Wu, ldw, act, out, ldh, G, U, ldgu, None)


@pytest.mark.parametrize("change,code", [
    (dict(handle=None), INVALID), (dict(M=-1), INVALID), (dict(F=-1), INVALID), (dict(K=-8), INVALID),
    (dict(act=5), INVALID), (dict(act=-1), INVALID), (dict(G=_at(4)), INVALID), (dict(U=_at(4)), INVALID),
    (dict(X=None), INVALID), (dict(Wg=None), INVALID), (dict(Wu=None), INVALID), (dict(out=None), INVALID),
    (dict(M=0), OK), (dict(F=0), OK), (dict(K=0), UNSUPPORTED), (dict(K=60), UNSUPPORTED),
    (dict(ldx=56), UNSUPPORTED), (dict(ldx=68), UNSUPPORTED), (dict(ldw=60), UNSUPPORTED), (dict(ldh=12), UNSUPPORTED),
    (dict(ldh=20), UNSUPPORTED), (dict(G=_at(4), U=_at(5), ldgu=8), UNSUPPORTED), (dict(X=_at(0) + 8), UNSUPPORTED),
    (dict(out=_at(3) + 2), UNSUPPORTED), (dict(M=2 ** 31 - 1), TOO_LARGE), (dict(ldx=2 ** 62), TOO_LARGE),
    (dict(ldw=2 ** 39), TOO_LARGE), (dict(ldh=2 ** 39), TOO_LARGE),
    (dict(out=_at(0)), INVALID), (dict(out=_at(1) + 15 * 128), INVALID), (dict(G=_at(3), U=_at(5)), INVALID),
    (dict(G=_at(4), U=_at(4)), INVALID), (dict(G=_at(4), U=_at(4) + 16, ldgu=24), INVALID),
])
def test_gated(change, code):
    assert _gated(**change) == code


def test_column_slices_of_one_matrix_are_apart():
    """Not refused: the call gets as far as the device, which is not there."""
    try:
        import torch

        if torch.cuda.is_available():
            pytest.skip("a GPU is present")
    except ImportError:
        pass
    assert _gated(G=_at(4), U=_at(4) + 32, ldgu=32) == _lib.ERR_CUDA
    assert _gated(out=_at(4) + 64, ldh=48, G=_at(4), U=_at(4) + 32, ldgu=48) == _lib.ERR_CUDA


def _backward(handle=H, M=4, F=16, K=64, dH=_at(0), lddh=16, X=_at(1), ldx=64, Wg=_at(2), Wu=_at(3), ldw=64, G=_at(4),
              U=_at(5), ldgu=16, act=4, dX=_at(6), lddx=64, dWg=_at(7), dWu=_at(8), lddw=64, ws=_at(9), ws_bytes=4 * 4 * 16):
    return _lib.load().b200gemm_bf16_gated_backward(handle, M, F, K, dH, lddh, X, ldx, Wg, Wu, ldw, G, U, ldgu, act, dX,
                                                    lddx, dWg, dWu, lddw, ws, ws_bytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(handle=None), INVALID), (dict(M=-1), INVALID), (dict(act=9), INVALID), (dict(dWg=None), INVALID),
    (dict(dWu=None), INVALID), (dict(dX=None, dWg=None, dWu=None), OK), (dict(M=0, F=0), OK), (dict(K=0), OK),
    (dict(K=12), UNSUPPORTED), (dict(lddx=60), UNSUPPORTED), (dict(lddw=8), UNSUPPORTED), (dict(lddh=8), UNSUPPORTED),
    (dict(ldgu=17), UNSUPPORTED), (dict(ldx=65), UNSUPPORTED), (dict(dX=_at(6) + 2), UNSUPPORTED),
    (dict(ws=_at(9) + 4), UNSUPPORTED), (dict(dH=None), INVALID), (dict(G=None), INVALID), (dict(ws=None), INVALID),
    (dict(K=2 ** 31 - 8), UNSUPPORTED), (dict(lddx=2 ** 62), TOO_LARGE), (dict(ldgu=2 ** 39), TOO_LARGE),
    (dict(dX=_at(1)), INVALID), (dict(dX=_at(0)), INVALID),
    (dict(dWg=_at(2)), INVALID), (dict(dWg=_at(7), dWu=_at(7)), INVALID), (dict(ws=_at(6)), INVALID),
    (dict(ws=_at(4)), INVALID), (dict(ws_bytes=4 * 4 * 16 - 1), UNSUPPORTED),
    (dict(ws=_at(6) - 4096, ws_bytes=4097), INVALID), (dict(F=9, ws_bytes=4 * 4 * 16 - 1), UNSUPPORTED),
])
def test_backward(change, code):
    assert _backward(**change) == code


def test_workspace_size_of_nothing():
    size = _lib.load().b200gemm_gated_backward_workspace
    assert size(H, 0, 5, 8) == 0 and size(H, 5, 0, 8) == 0 and size(H, -1, 4, 8) == 0 and size(None, 4, 4, 8) == 0


def _nt(handle=H, M=2, N=64, K=128, A=_at(0), lda=128, codes=_at(1), scales=_at(2), group=32, C=_at(3), ldc=64, out=0):
    return _lib.load().b200gemm_w4_nt(handle, M, N, K, A, lda, codes, scales, group, C, ldc, out, None)


@pytest.mark.parametrize("change,code", [
    (dict(handle=None), INVALID), (dict(N=-1), INVALID), (dict(out=2), INVALID), (dict(M=0), OK), (dict(N=0), OK),
    (dict(K=0), UNSUPPORTED), (dict(A=None), INVALID), (dict(codes=None), INVALID), (dict(scales=None), INVALID),
    (dict(C=None), INVALID), (dict(group=16), UNSUPPORTED), (dict(group=48), UNSUPPORTED), (dict(group=0), UNSUPPORTED),
    (dict(group=512), UNSUPPORTED), (dict(K=96, group=64), UNSUPPORTED), (dict(lda=120), UNSUPPORTED),
    (dict(lda=132), UNSUPPORTED), (dict(ldc=63), UNSUPPORTED), (dict(A=_at(0) + 2), UNSUPPORTED),
    (dict(codes=_at(1) + 8), UNSUPPORTED), (dict(scales=_at(2) + 1), UNSUPPORTED), (dict(C=_at(3) + 1), UNSUPPORTED),
    (dict(C=_at(3) + 2, out=1), UNSUPPORTED), (dict(N=2 ** 31 - 1, ldc=2 ** 31), TOO_LARGE), (dict(lda=2 ** 40), TOO_LARGE), (dict(ldc=2 ** 62), TOO_LARGE),
    (dict(C=_at(0)), INVALID), (dict(C=_at(1) + 64 * 64 - 2), INVALID), (dict(C=_at(2)), INVALID),
])
def test_w4_nt(change, code):
    assert _nt(**change) == code


def _w4_gated(handle=H, M=2, F=64, K=128, X=_at(0), ldx=128, gc=_at(1), gs=_at(2), uc=_at(3), us=_at(4), group=64, act=4,
              out=_at(5), ldh=64):
    return _lib.load().b200gemm_w4_gated(handle, M, F, K, X, ldx, gc, gs, uc, us, group, act, out, ldh, None)


@pytest.mark.parametrize("change,code", [
    (dict(handle=None), INVALID), (dict(act=7), INVALID), (dict(F=0), OK), (dict(K=0), UNSUPPORTED),
    (dict(uc=None), INVALID), (dict(group=31), UNSUPPORTED), (dict(ldh=62), UNSUPPORTED), (dict(gs=_at(2) + 1), UNSUPPORTED),
    (dict(uc=_at(3) + 4), UNSUPPORTED), (dict(out=_at(0) + 128), INVALID), (dict(out=_at(4)), INVALID),
])
def test_w4_gated(change, code):
    assert _w4_gated(**change) == code


def _convert(back, handle=H, N=8, K=64, W=_at(0), ldw=64, group=32, codes=_at(1), scales=_at(2)):
    lib = _lib.load()
    if back:
        return lib.b200gemm_w4_dequantize(handle, N, K, codes, scales, group, W, ldw, None)
    return lib.b200gemm_w4_quantize(handle, N, K, W, ldw, group, codes, scales, None)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("change,code", [
    (dict(handle=None), INVALID), (dict(N=-1), INVALID), (dict(N=0), OK), (dict(K=0), OK), (dict(group=33), UNSUPPORTED),
    (dict(K=48), UNSUPPORTED), (dict(W=None), INVALID), (dict(codes=None), INVALID), (dict(ldw=56), UNSUPPORTED),
    (dict(ldw=66), UNSUPPORTED), (dict(W=_at(0) + 2), UNSUPPORTED), (dict(codes=_at(1) + 2), UNSUPPORTED),
    (dict(scales=_at(2) + 1), UNSUPPORTED), (dict(N=2 ** 22), TOO_LARGE), (dict(codes=_at(0)), INVALID),
    (dict(scales=_at(0) + 8 * 128 - 2), INVALID),
])
def test_w4_convert(back, change, code):
    assert _convert(back, **change) == code


def test_python_checks_need_no_handle():
    torch = pytest.importorskip("torch")
    import b200_gemm_b200 as b200

    for call in (lambda t: b200.gated(t, t, t), lambda t: b200.w4_quantize(t),
                 lambda t: b200.gated_backward(t, t, t, t, t, t), lambda t: b200.w4_nt(t, t, t),
                 lambda t: b200.w4_dequantize(t, t), lambda t: b200.w4_gated(t, t, t, t, t)):
        with pytest.raises(ValueError):
            call(torch.zeros(4, 64, dtype=torch.bfloat16))
