"""Feed-forward operators of a `Gemm` handle: the gated block forward and
backward, and its 4-bit-weight serving form (include/b200gemm.h,
b200gemm_bf16_gated and after).

Activations are 2-D bf16 CUDA tensors whose rows may be slices of wider ones
(stride(1) == 1, row stride a multiple of 8 elements, 16-byte aligned); all
tensors of a call live on the handle's device.  A call runs on `stream` (a
torch stream or a raw pointer; default: the current stream of the handle's
device); tensors that it allocates are allocated for that stream.  Autograd
records none of these calls, whatever their inputs require: `gated_backward` is
called by hand, or from a torch.autograd.Function of the caller's."""
from __future__ import annotations

from . import _lib

ACTIVATIONS = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU,
               "gelu_tanh": _lib.ACT_GELU_TANH, "silu": _lib.ACT_SILU}
W4_GROUPS = (32, 64, 128, 256)


class _NoContext:
    """contextlib.nullcontext without its cost."""

    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return None


_NO_CONTEXT = _NoContext()
_torch_module = None


def _torch():
    """torch, imported when a call first needs it."""
    global _torch_module
    if _torch_module is None:
        import torch

        _torch_module = torch
    return _torch_module


def _activation(name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}") from None


class FfnOps:
    """Mixin of `Gemm` (uses its `_lib`, `_h` and `device`).  A call's checks
    are kept to a few microseconds: at one token they are a good part of it."""

    # --------------------------------------------------------------- helpers
    def _check(self, t, name: str, dtype, rows=None, cols=None) -> int:
        """Checks a row-major matrix argument; returns its row pitch."""
        shape = t.shape
        if (t.dtype is dtype and t.get_device() == self.device and len(shape) == 2
                and (rows is None or shape[0] == rows) and (cols is None or shape[1] == cols)):
            pitch, step = t.stride()
            if step == 1 or shape[1] <= 1:
                return pitch if shape[0] > 1 else 8 * ((shape[1] + 7) // 8)  # (one row's stride means nothing)
            raise ValueError(f"{name} must be row-major (stride(1) == 1)")
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}")
        if t.get_device() != self.device:
            raise ValueError(f"{name} must be on cuda:{self.device}")
        want = f"[{'*' if rows is None else rows}, {'*' if cols is None else cols}]"
        raise ValueError(f"{name} must have shape {want}, not {list(shape)}")

    def _where(self, stream):
        """(stream pointer, context in which the call's tensors are allocated)."""
        torch = _torch()
        if stream is None:
            return torch._C._cuda_getCurrentRawStream(self.device), _NO_CONTEXT
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device=self.device)
        if stream.device.index != self.device:
            raise ValueError(f"stream must belong to cuda:{self.device}")
        return int(stream.cuda_stream), torch.cuda.stream(stream)

    @staticmethod
    def _empty(like, rows: int, cols: int, dtype=None):
        """A [rows, cols] matrix on `like`'s device (of its type, or `dtype`)
        whose rows start on 16-byte boundaries, and its row pitch."""
        pitch = cols + -cols % 8
        t = like.new_empty((rows, pitch)) if dtype is None else like.new_empty((rows, pitch), dtype=dtype)
        return (t if pitch == cols else t[:, :cols]), pitch

    # ------------------------------------------------------------ gated block
    def gated(self, X, Wg, Wu, activation: str = "silu", save: bool = False, out=None, gate_out=None, up_out=None,
              stream=None):
        """H = act(X Wg^T) * (X Wu^T) in one kernel.

        X: bf16 [M, K]; Wg, Wu: bf16 [F, K] with equal row strides.  Returns H
        (bf16 [M, F]); with `save` (H, G, U), G = X Wg^T and U = X Wu^T rounded
        to bf16, which `gated_backward` takes.  `out`, `gate_out` and `up_out`
        may be given, the last two with one row stride; nothing may overlap
        what is written.  activation: none, relu, gelu, gelu_tanh, silu."""
        torch = _torch()
        act = _activation(activation)
        bf16 = torch.bfloat16
        ldx = self._check(X, "X", bf16)
        M, K = X.shape
        ldw = self._check(Wg, "Wg", bf16, None, K)
        F = Wg.shape[0]
        if self._check(Wu, "Wu", bf16, F, K) != ldw:
            raise ValueError("Wg and Wu must have the same row stride")
        ptr, where = self._where(stream)
        ldgu = 0
        with where:
            H, ldh = self._empty(X, M, F) if out is None else (out, self._check(out, "out", bf16, M, F))
            G = U = None
            if save or gate_out is not None or up_out is not None:
                G, ldgu = (self._empty(X, M, F) if gate_out is None
                           else (gate_out, self._check(gate_out, "gate_out", bf16, M, F)))
                U, ldu = (self._empty(X, M, F) if up_out is None
                          else (up_out, self._check(up_out, "up_out", bf16, M, F)))
                if ldu != ldgu:
                    raise ValueError("gate_out and up_out must have the same row stride")
            rc = self._lib.b200gemm_bf16_gated(
                self._h, M, F, K, X.data_ptr(), ldx, Wg.data_ptr(), Wu.data_ptr(), ldw, act, H.data_ptr(), ldh,
                None if G is None else G.data_ptr(), None if U is None else U.data_ptr(), ldgu, ptr)
        _lib.check(rc, "b200gemm_bf16_gated")
        return H if G is None else (H, G, U)

    def gated_backward(self, dH, X, Wg, Wu, G, U, activation: str = "silu", input_grad: bool = True,
                       weight_grad: bool = True, stream=None):
        """Gradients of H = act(G) * U, G = X Wg^T, U = X Wu^T: (dX, dWg, dWu),
        bf16, from dH and the G and U that `gated(..., save=True)` returned.

        dU = dH act(G) and dG = dH U act'(G) are rounded to bf16 before the
        products (they are tensor-core operands); sums are fp32.  With
        `input_grad` or `weight_grad` off the matching results are None."""
        torch = _torch()
        act = _activation(activation)
        bf16 = torch.bfloat16
        lddh = self._check(dH, "dH", bf16)
        M, F = dH.shape
        ldx = self._check(X, "X", bf16, M)
        K = X.shape[1]
        ldw = self._check(Wg, "Wg", bf16, F, K)
        if self._check(Wu, "Wu", bf16, F, K) != ldw:
            raise ValueError("Wg and Wu must have the same row stride")
        ldgu = self._check(G, "G", bf16, M, F)
        if self._check(U, "U", bf16, M, F) != ldgu:
            raise ValueError("G and U must have the same row stride")
        ptr, where = self._where(stream)
        with where:
            dX = dWg = dWu = None
            lddx = lddw = 0
            if input_grad:
                dX, lddx = self._empty(X, M, K)
            if weight_grad:
                dWg, lddw = self._empty(X, F, K)
                dWu, lddw = self._empty(X, F, K)
            # Freed when this returns: the allocator hands it on in the order of
            # the stream that it was allocated for, which is the call's.
            ws_bytes = self._lib.b200gemm_gated_backward_workspace(self._h, M, F, K)
            ws = X.new_empty(ws_bytes + 16, dtype=torch.uint8)
            rc = self._lib.b200gemm_bf16_gated_backward(
                self._h, M, F, K, dH.data_ptr(), lddh, X.data_ptr(), ldx, Wg.data_ptr(), Wu.data_ptr(), ldw,
                G.data_ptr(), U.data_ptr(), ldgu, act, None if dX is None else dX.data_ptr(), lddx,
                None if dWg is None else dWg.data_ptr(), None if dWu is None else dWu.data_ptr(), lddw,
                ws.data_ptr(), ws_bytes, ptr)
        _lib.check(rc, "b200gemm_bf16_gated_backward")
        return dX, dWg, dWu

    # --------------------------------------------------------- 4-bit weights
    def _w4(self, codes, scales, name: str, K=None, N=None):
        """Checks 4-bit weights; returns (N, K, group)."""
        torch = _torch()
        if codes.dtype is not torch.uint8 or scales.dtype is not torch.bfloat16:
            raise TypeError(f"{name}: codes must be torch.uint8 and scales torch.bfloat16")
        if codes.get_device() != self.device or scales.get_device() != self.device:
            raise ValueError(f"{name} must be on cuda:{self.device}")
        cs, ss = codes.shape, scales.shape
        if len(cs) != 2 or len(ss) != 2 or not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError(f"{name}: codes [N, K / 2] and scales [K / group, N] must be contiguous")
        n, k, groups = cs[0], 2 * cs[1], ss[0]
        if (N is not None and n != N) or (K is not None and k != K):
            raise ValueError(f"{name}: codes of a [{n}, {k}] weight where [{n if N is None else N}, "
                             f"{k if K is None else K}] is needed")
        if ss[1] != n or groups == 0 or k % groups != 0 or k // groups not in W4_GROUPS:
            raise ValueError(f"{name}: scales {list(ss)} do not fit codes {list(cs)} with a group "
                             f"of {', '.join(map(str, W4_GROUPS))}")
        return n, k, k // groups

    def w4_quantize(self, W, group: int = 128, stream=None):
        """bf16 weights [N, K] -> (codes, scales): per `group` (32, 64, 128 or
        256) consecutive k of a row s = bf16(max|w| / 7) and
        q = clamp(rint(w / s), -8, 7) + 8.  codes: uint8 [N, K / 2], the even k
        in the low four bits; scales: bf16 [K / group, N]."""
        torch = _torch()
        ldw = self._check(W, "W", torch.bfloat16)
        N, K = W.shape
        if group not in W4_GROUPS or K % group != 0 or K == 0:
            raise ValueError(f"group must be one of {W4_GROUPS} and divide K = {K}")
        ptr, where = self._where(stream)
        with where:
            codes = torch.empty(N, K // 2, dtype=torch.uint8, device=W.device)
            scales = torch.empty(K // group, N, dtype=torch.bfloat16, device=W.device)
            rc = self._lib.b200gemm_w4_quantize(self._h, N, K, W.data_ptr(), ldw, group, codes.data_ptr(),
                                                scales.data_ptr(), ptr)
        _lib.check(rc, "b200gemm_w4_quantize")
        return codes, scales

    def w4_dequantize(self, codes, scales, out=None, stream=None):
        """The bf16 [N, K] weights that the codes stand for, bf16(s (q - 8)).
        For long prompts: `bf16_nt` with these beats `w4_nt` from about 65
        rows on, from about 160 where they are made for that one call."""
        torch = _torch()
        N, K, group = self._w4(codes, scales, "weights")
        ptr, where = self._where(stream)
        with where:
            bf16 = torch.bfloat16
            W, ldw = self._empty(scales, N, K) if out is None else (out, self._check(out, "out", bf16, N, K))
            rc = self._lib.b200gemm_w4_dequantize(self._h, N, K, codes.data_ptr(), scales.data_ptr(), group,
                                                  W.data_ptr(), ldw, ptr)
        _lib.check(rc, "b200gemm_w4_dequantize")
        return W

    def w4_nt(self, A, codes, scales, out=None, out_dtype=None, stream=None):
        """out = A W^T for 4-bit weights W (see `w4_quantize`): bf16 A [M, K],
        out [M, N] bf16 (default) or fp32.  No weight is rounded: group sums of
        A (q - 8) are scaled in fp32."""
        torch = _torch()
        N, K, group = self._w4(codes, scales, "weights")
        lda = self._check(A, "A", torch.bfloat16, None, K)
        M = A.shape[0]
        if out_dtype is None:
            out_dtype = torch.bfloat16 if out is None else out.dtype
        if out_dtype not in (torch.bfloat16, torch.float32):
            raise TypeError("out_dtype must be torch.bfloat16 or torch.float32")
        ptr, where = self._where(stream)
        with where:
            C, ldc = (self._empty(A, M, N, None if out_dtype is A.dtype else out_dtype) if out is None
                      else (out, self._check(out, "out", out_dtype, M, N)))
            rc = self._lib.b200gemm_w4_nt(self._h, M, N, K, A.data_ptr(), lda, codes.data_ptr(), scales.data_ptr(),
                                          group, C.data_ptr(), ldc,
                                          _lib.OUT_F32 if out_dtype == torch.float32 else _lib.OUT_BF16, ptr)
        _lib.check(rc, "b200gemm_w4_nt")
        return C

    def w4_gated(self, X, gate_codes, gate_scales, up_codes, up_scales, activation: str = "silu", out=None,
                 stream=None):
        """H = act(X Wg^T) * (X Wu^T) for 4-bit Wg and Wu [F, K] of one group."""
        torch = _torch()
        act = _activation(activation)
        F, K, group = self._w4(gate_codes, gate_scales, "gate weights")
        if self._w4(up_codes, up_scales, "up weights", K, F)[2] != group:
            raise ValueError("gate and up weights must have the same group")
        ldx = self._check(X, "X", torch.bfloat16, None, K)
        M = X.shape[0]
        ptr, where = self._where(stream)
        with where:
            bf16 = torch.bfloat16
            H, ldh = self._empty(X, M, F) if out is None else (out, self._check(out, "out", bf16, M, F))
            rc = self._lib.b200gemm_w4_gated(self._h, M, F, K, X.data_ptr(), ldx, gate_codes.data_ptr(),
                                             gate_scales.data_ptr(), up_codes.data_ptr(), up_scales.data_ptr(), group,
                                             act, H.data_ptr(), ldh, ptr)
        _lib.check(rc, "b200gemm_w4_gated")
        return H
