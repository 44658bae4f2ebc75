"""Matrix products beside ``tb.matmul``: rows grouped by expert, and 8-bit
operands with a scale per block of 128.

    grouped_matmul        C[r] = beta·C[r] + A[r] · B[e]       r in [offsets[e], offsets[e + 1])
    grouped_matmul_wgrad  G[e] = beta·G[e] + A[rows of e]^T · D[rows of e]
    quantize_fp8          S = max|block| / 448, Q = e4m3(X / S)
    matmul_fp8            C = beta·C + Σ_b SA[:, b] SB[b, :] (A_b · B_b), b = blocks of 128 along k
    grouped_matmul_fp8    the same for the rows of each expert

As ``tb.matmul``, they update their output in place (``beta=1``, the default,
adds to it; ``beta=0`` overwrites) on the current stream of its device, and
return it. Offsets stay on the device: no call waits for the GPU, and a captured
CUDA graph follows their contents. Operands are strided views; rows that
do not begin on 16-byte boundaries are copied first (into ``workspace``, or a
buffer from torch's allocator). An output may not overlap an operand.

The gradients of ``C = grouped_matmul(A, B)`` for a gradient D of C are
``grouped_matmul(D, B.transpose(1, 2), dA, offsets)`` and
``grouped_matmul_wgrad(A, D, dB, offsets)``; those of ``matmul_fp8`` are
``matmul_fp8`` of D quantised along n with B.t(), and of A^T with D, both
quantised in blocks of 128 rows (``block=(128, 1)``). The gradient of the rows
of ``grouped_matmul_fp8`` is the same call on ``B.transpose(1, 2)`` and
``SB.transpose(1, 2)``; that of its weights takes 16-bit rows
(``grouped_matmul_wgrad``).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import TBError, _check, _lib
from . import _capi
from ._capi import TB_BF16, TB_E4M3, TB_ERR_INVALID_ARGUMENT, TB_ERR_UNSUPPORTED, TB_F16, TB_F32

__all__ = ["grouped_matmul", "grouped_matmul_wgrad", "quantize_fp8", "matmul_fp8", "grouped_matmul_fp8"]

_HALF = {torch.float16: TB_F16, torch.bfloat16: TB_BF16}
_OUT = {torch.float32: TB_F32, torch.float16: TB_F16, torch.bfloat16: TB_BF16}
_FP8 = torch.float8_e4m3fn


def _load_calls():
    """Module _tbtorch (csrc/tb_torch.cpp), given the library's entry points."""
    try:
        from . import _tbtorch
    except ImportError as e:
        raise ImportError("_tbtorch.so is missing or of another torch: build it with "
                          "`python -m mini_triton_nvgpu_v1_b200.build`") from e
    _tbtorch.library(*(C.cast(f, C.c_void_p).value for f in (
        _lib.tb_grouped_matmul, _lib.tb_grouped_matmul_wgrad, _lib.tb_quantize_blocks, _lib.tb_matmul_blockscaled,
        _lib.tb_grouped_matmul_blockscaled, _lib.tb_grouped_matmul_workspace_bytes,
        _lib.tb_grouped_matmul_wgrad_workspace_bytes)))
    return _tbtorch


# Calls like an earlier one, by the tensors' sizes, strides, types and device:
# _call0(op, tensors..., x, y) is 0 when it ran them, -1 when it knows no such
# call or has to leave the copy of its operands in the caller's workspace to the
# long way.
_calls = _load_calls()
_call0, _remember = _calls.call, _calls.remember
_ROWS, _WGRAD, _QUANTIZE, _BYTES, _ROWS_BYTES = range(5)


def _bad(message: str, code: int = TB_ERR_INVALID_ARGUMENT):
    return TBError(code, message)


def _same_device(**tensors) -> int:
    device = None
    for name, t in tensors.items():
        if not t.is_cuda:
            raise _bad(f"{name} must be a CUDA tensor")
        if device is None:
            device = t.device
        elif t.device != device:
            raise _bad(f"{name} is on {t.device}, the others on {device}")
    return device.index


def _rows(t, name: str) -> int:
    """Leading dimension of the row-major matrices t (…, rows, cols)."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise _bad(f"{name} must have a unit stride along its columns", TB_ERR_UNSUPPORTED)
    return t.stride(-2) if t.shape[-2] > 1 else max(1, t.shape[-1])


def _either(t, name: str) -> tuple[bool, int]:
    """(column-major?, leading dimension) of the matrices t (…, rows, cols)."""
    r, c = t.shape[-2:]
    by_row = c <= 1 or t.stride(-1) == 1
    by_col = r <= 1 or t.stride(-2) == 1
    if by_col and (c <= 1 or not by_row):
        return True, t.stride(-1) if c > 1 else max(1, r)
    if not by_row:
        raise _bad(f"{name} must have a unit stride along its rows or its columns", TB_ERR_UNSUPPORTED)
    return False, t.stride(-2) if r > 1 else max(1, c)


def _batch(t, name: str) -> int:
    """Stride between the matrices of t (groups, rows, cols), which may not overlap."""
    e, r, c = t.shape
    if e <= 1 or t.numel() == 0:
        return max(1, r * c)
    _apart(t, name)
    return t.stride(0)


def _apart(t, name: str) -> None:
    """Refuses a t with two entries in one place."""
    spans = sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1)
    reach = 1
    for st, sz in spans:
        if st < reach:
            raise _bad(f"entries of {name} overlap", TB_ERR_UNSUPPORTED)
        reach = st * (sz - 1) + reach


def _check_offsets(offsets, groups: int) -> int:
    if offsets.dim() != 1 or offsets.shape[0] != groups + 1:
        raise _bad(f"offsets must hold {groups + 1} entries, one more than there are groups")
    if offsets.dtype not in (torch.int32, torch.int64):
        raise _bad("offsets must be int32 or int64")
    if not offsets.is_contiguous():
        raise _bad("offsets must be contiguous")
    return 1 if offsets.dtype == torch.int64 else 0


def _desc(groups, rows, n, k, ab, c, beta, a_col, b_col, long_) -> _capi.tb_grouped_desc:
    if beta not in (0, 1):
        raise _bad("beta must be 0 or 1")
    d = _capi.tb_grouped_desc()
    d.groups, d.rows, d.n, d.k = groups, rows, n, k
    d.ab_dtype, d.c_dtype, d.beta = ab, c, int(beta)
    d.a_col_major, d.b_col_major, d.offsets_long = int(a_col), int(b_col), long_
    return d


def _empty(shape, dtype, device, stream):
    """Memory of the stream it is used on: the allocator orders reuse by stream."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _scratch(need: int, workspace, device, stream):
    """(address, bytes, tensor to keep) of a call's workspace."""
    if not need:
        return None, 0, None
    if workspace is None:
        workspace = _empty((need,), torch.uint8, device, stream)
    elif not workspace.is_cuda or workspace.device != device or not workspace.is_contiguous():
        raise _bad("workspace must be a contiguous CUDA tensor on the operands' device")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace


def _call(dev: int, stream, fn, *args) -> None:
    """fn(*args, stream) with `dev` current."""
    s = stream if stream is not None else torch.cuda.current_stream(dev)
    if torch.cuda.current_device() == dev:
        code = fn(*args, s.cuda_stream or None)
    else:
        with torch.cuda.device(dev):
            code = fn(*args, s.cuda_stream or None)
    _check(code)


def _setup_grouped(A, B, Cm, offsets, beta, eight_bit: bool):
    """(desc, lda, ldb, stride_b, ldc)."""
    if A.dim() != 2 or B.dim() != 3 or Cm.dim() != 2:
        raise _bad("grouped products take A [rows, k], B [groups, k, n] and C [rows, n]")
    rows, k = A.shape
    groups, kb, n = B.shape
    if kb != k or tuple(Cm.shape) != (rows, n):
        raise _bad("operand shapes disagree: A [rows, k], B [groups, k, n], C [rows, n]")
    if eight_bit:
        if A.dtype != _FP8 or B.dtype != _FP8:
            raise _bad("A and B must be float8_e4m3fn")
        ab = TB_E4M3
    else:
        if A.dtype not in _HALF or B.dtype != A.dtype:
            raise _bad("A and B must both be f16 or both be bf16")
        ab = _HALF[A.dtype]
    if Cm.dtype not in _OUT:
        raise _bad("C must be f32, f16 or bf16")
    long_ = _check_offsets(offsets, groups)
    b_col, ldb = _either(B, "B")
    lda, ldc = _rows(A, "A"), _rows(Cm, "C")
    d = _desc(groups, rows, n, k, ab, _OUT[Cm.dtype], beta, False, b_col, long_)
    return d, lda, ldb, _batch(B, "B"), ldc


def _need(d, A, lda, B, ldb, stride_b) -> int:
    return _lib.tb_grouped_matmul_workspace_bytes(C.byref(d), A.data_ptr(), lda, B.data_ptr(), ldb, stride_b)


def grouped_matmul(A, B, Cm, offsets, *, beta: int = 1, workspace=None, stream=None):
    """C[r] ← beta·C[r] + A[r] · B[e] for the rows r in [offsets[e],
    offsets[e + 1]) of every group e. A [rows, k] and B [groups, k, n] f16 or
    bf16 (B row-major, or a transposed view of weights kept as n × k), C
    [rows, n] f32, f16 or bf16, offsets groups + 1 int32 or int64 on the
    device. Rows outside every group keep what C held. Returns C."""
    if stream is None:
        code = _call0(_ROWS, A, B, Cm, offsets, beta, workspace is not None)
        if code >= 0:
            if code:
                _check(code)
            return Cm
    dev = _same_device(A=A, B=B, C=Cm, offsets=offsets)
    d, lda, ldb, stride_b, ldc = _setup_grouped(A, B, Cm, offsets, beta, False)
    ws, nbytes, _kept = _scratch(_need(d, A, lda, B, ldb, stride_b), workspace, Cm.device, stream)
    _call(dev, stream, _lib.tb_grouped_matmul, d, A.data_ptr(), lda, B.data_ptr(), ldb, stride_b, Cm.data_ptr(), ldc,
          offsets.data_ptr(), ws, nbytes)
    _remember(_ROWS, A, B, Cm, offsets, int(beta), 0, d, (lda, ldb, stride_b, ldc), None, None)
    return Cm


def grouped_matmul_wgrad(A, D, G, offsets, *, beta: int = 1, workspace=None, stream=None):
    """G[e] ← beta·G[e] + A[rows of e]^T · D[rows of e]: the gradient of the
    weights of :func:`grouped_matmul` from the gradient D of its output.
    A [rows, k] and D [rows, n] f16 or bf16, G [groups, k, n] f32, f16 or
    bf16. A group without rows gets beta·G[e]. Returns G."""
    if stream is None:
        code = _call0(_WGRAD, A, D, G, offsets, beta, workspace is not None)
        if code >= 0:
            if code:
                _check(code)
            return G
    dev = _same_device(A=A, D=D, G=G, offsets=offsets)
    if A.dim() != 2 or D.dim() != 2 or G.dim() != 3:
        raise _bad("the weight gradient takes A [rows, k], D [rows, n] and G [groups, k, n]")
    rows, k = A.shape
    groups, n = G.shape[0], D.shape[1]
    if D.shape[0] != rows or tuple(G.shape) != (groups, k, n):
        raise _bad("operand shapes disagree: A [rows, k], D [rows, n], G [groups, k, n]")
    if A.dtype not in _HALF or D.dtype != A.dtype:
        raise _bad("A and D must both be f16 or both be bf16")
    if G.dtype not in _OUT:
        raise _bad("G must be f32, f16 or bf16")
    long_ = _check_offsets(offsets, groups)
    lda, ldd, ldg = _rows(A, "A"), _rows(D, "D"), _rows(G, "G")
    stride_g = _batch(G, "G")
    d = _desc(groups, rows, n, k, _HALF[A.dtype], _OUT[G.dtype], beta, False, False, long_)
    need = _lib.tb_grouped_matmul_wgrad_workspace_bytes(C.byref(d), A.data_ptr(), lda, D.data_ptr(), ldd)
    ws, nbytes, _kept = _scratch(need, workspace, G.device, stream)
    _call(dev, stream, _lib.tb_grouped_matmul_wgrad, d, A.data_ptr(), lda, D.data_ptr(), ldd, G.data_ptr(), ldg,
          stride_g, offsets.data_ptr(), ws, nbytes)
    _remember(_WGRAD, A, D, G, offsets, int(beta), 0, d, (lda, ldd, ldg, stride_g), None, None)
    return G


def _blocks(n: int) -> int:
    return (n + 127) // 128


def quantize_fp8(X, Q=None, S=None, *, block=(1, 128), stream=None):
    """Q ← e4m3(448 · X / m), S ← m / 448 with m = max(max|block|, 448 · 2^-63)
    for every block (1, 128), (128, 1) or (128, 128) of X [rows, cols] or
    [batch, rows, cols] (f32, f16 or bf16). The exact quotient of f16 and bf16
    values is rounded to nearest, ties to even; of f32 values one within 2^-22
    of the border of two e4m3 values may go to either. Q: float8_e4m3fn of X's shape; S:
    f32 [(batch,) ceil(rows / block[0]), ceil(cols / block[1])]. A Q that is
    not given is made with rows that begin on 16-byte boundaries, as the
    8-bit products read them without a copy; what is not given belongs to
    ``stream``. Returns (Q, S)."""
    br, bc = block
    if Q is not None and S is not None and stream is None:
        code = _call0(_QUANTIZE, X, Q, S, br, bc)
        if code >= 0:
            if code:
                _check(code)
            return Q, S
    if (br, bc) not in ((1, 128), (128, 1), (128, 128)):
        raise _bad("blocks are (1, 128), (128, 1) or (128, 128)")
    if X.dim() not in (2, 3):
        raise _bad("X must be [rows, cols] or [batch, rows, cols]")
    if not X.is_cuda:
        raise _bad("X must be a CUDA tensor")
    if X.dtype not in _OUT:
        raise _bad("X must be f32, f16 or bf16")
    rows, cols = X.shape[-2:]
    if Q is None:
        Q = _empty((*X.shape[:-1], (cols + 15) // 16 * 16), torch.uint8, X.device, stream).view(_FP8)[..., :cols]
    if S is None:
        S = _empty((*X.shape[:-2], -(-rows // br), -(-cols // bc)), torch.float32, X.device, stream)
    dev = _same_device(X=X, Q=Q, S=S)
    if Q.dtype != _FP8 or Q.shape != X.shape:
        raise _bad("Q must be float8_e4m3fn of X's shape")
    if S.dtype != torch.float32 or tuple(S.shape) != (*X.shape[:-2], -(-rows // br), -(-cols // bc)):
        raise _bad("S must be f32 with one entry for each block")
    batched = X.dim() == 3
    d = _capi.tb_quantize_desc()
    d.batch, d.rows, d.cols = (X.shape[0] if batched else 1), rows, cols
    d.block_rows, d.block_cols, d.x_dtype = int(br), int(bc), _OUT[X.dtype]
    if X.numel():
        _apart(Q, "Q")
        _apart(S, "S")
    ints = (_rows(X, "X"), X.stride(0) if batched else 0, _rows(Q, "Q"), Q.stride(0) if batched else 0,
            S.stride(0) if batched else 0, S.stride(-2), S.stride(-1))
    _call(dev, stream, _lib.tb_quantize_blocks, d, X.data_ptr(), *ints[:2], Q.data_ptr(), *ints[2:4], S.data_ptr(),
          *ints[4:])
    _remember(_QUANTIZE, X, Q, S, int(br), int(bc), d, ints, None, None)
    return Q, S


def _scales(s, name: str, mn: int, k: int, mn_axis: int, k_axis: int, lead: tuple) -> _capi.tb_scales:
    if s.dtype != torch.float32 or s.dim() != len(lead) + 2 or tuple(s.shape[:-2]) != lead:
        raise _bad(f"{name} must be f32 with one entry for each block")
    per = s.shape[mn_axis]
    if s.shape[k_axis] != _blocks(k) or per not in (mn, _blocks(mn)):
        raise _bad(f"{name} must hold one scale for 1 or 128 rows or columns and 128 elements along k")
    sc = _capi.tb_scales()
    sc.ptr = s.data_ptr()
    sc.stride_group = s.stride(0) if lead else 0
    sc.stride_mn, sc.stride_k = s.stride(mn_axis), s.stride(k_axis)
    sc.block = 1 if per == mn else 128
    return sc


def matmul_fp8(A, SA, B, SB, Cm, *, beta: int = 1, workspace=None, stream=None):
    """C ← beta·C + Σ_b SA[:, b] SB[b, :] (A_b · B_b), b = blocks of 128 along
    k. A [m, k] and B [k, n] float8_e4m3fn, each row-major or a transposed
    view; SA f32 [m or ceil(m / 128), ceil(k / 128)]; SB f32 [ceil(k / 128),
    n or ceil(n / 128)]; C [m, n] f32, f16 or bf16. The sum over a block and
    over the blocks is in f32. Returns C."""
    if stream is None:
        code = _call0(_BYTES, A, SA, B, SB, Cm, beta, workspace is not None)
        if code >= 0:
            if code:
                _check(code)
            return Cm
    dev = _same_device(A=A, SA=SA, B=B, SB=SB, C=Cm)
    if A.dim() != 2 or B.dim() != 2 or Cm.dim() != 2:
        raise _bad("matmul_fp8 takes A [m, k], B [k, n] and C [m, n]")
    m, k = A.shape
    n = B.shape[1]
    if B.shape[0] != k or tuple(Cm.shape) != (m, n):
        raise _bad("operand shapes disagree: A [m, k], B [k, n], C [m, n]")
    if A.dtype != _FP8 or B.dtype != _FP8:
        raise _bad("A and B must be float8_e4m3fn")
    if Cm.dtype not in _OUT:
        raise _bad("C must be f32, f16 or bf16")
    a_col, lda = _either(A, "A")
    b_col, ldb = _either(B, "B")
    ldc = _rows(Cm, "C")
    d = _desc(1, m, n, k, TB_E4M3, _OUT[Cm.dtype], beta, a_col, b_col, 0)
    sa, sb = _scales(SA, "SA", m, k, 0, 1, ()), _scales(SB, "SB", n, k, 1, 0, ())
    ws, nbytes, _kept = _scratch(_need(d, A, lda, B, ldb, 0), workspace, Cm.device, stream)
    _call(dev, stream, _lib.tb_matmul_blockscaled, d, A.data_ptr(), lda, sa, B.data_ptr(), ldb, sb, Cm.data_ptr(), ldc,
          ws, nbytes)
    _remember(_BYTES, A, SA, B, SB, Cm, int(beta), 0, d, (lda, ldb, ldc), sa, sb)
    return Cm


def grouped_matmul_fp8(A, SA, B, SB, Cm, offsets, *, beta: int = 1, workspace=None, stream=None):
    """:func:`matmul_fp8` for the rows of each group (:func:`grouped_matmul`):
    A [rows, k] with SA [rows, ceil(k / 128)], B [groups, k, n] (row-major, or a
    transposed view) with SB [groups, ceil(k / 128), n or ceil(n / 128)].
    Returns C."""
    if stream is None:
        code = _call0(_ROWS_BYTES, A, SA, B, SB, Cm, offsets, beta, workspace is not None)
        if code >= 0:
            if code:
                _check(code)
            return Cm
    dev = _same_device(A=A, SA=SA, B=B, SB=SB, C=Cm, offsets=offsets)
    d, lda, ldb, stride_b, ldc = _setup_grouped(A, B, Cm, offsets, beta, True)
    rows, k = A.shape
    groups, _, n = B.shape
    if SA.dim() != 2 or SA.shape[0] != rows:
        raise _bad("SA must hold a scale for each row of A and 128 elements along k")
    sa, sb = _scales(SA, "SA", rows, k, 0, 1, ()), _scales(SB, "SB", n, k, 2, 1, (groups,))
    ws, nbytes, _kept = _scratch(_need(d, A, lda, B, ldb, stride_b), workspace, Cm.device, stream)
    _call(dev, stream, _lib.tb_grouped_matmul_blockscaled, d, A.data_ptr(), lda, sa, B.data_ptr(), ldb, stride_b, sb,
          Cm.data_ptr(), ldc, offsets.data_ptr(), ws, nbytes)
    _remember(_ROWS_BYTES, A, SA, B, SB, Cm, offsets, int(beta), 0, d, (lda, ldb, stride_b, ldc), sa, sb)
    return Cm
