"""CPU: what the grouped and 8-bit products refuse, before any CUDA call."""
from __future__ import annotations

import ctypes as C

import pytest

from mini_triton_nvgpu_v1_b200 import _capi

OK, INVALID, UNSUPPORTED, WORKSPACE = 0, _capi.TB_ERR_INVALID_ARGUMENT, _capi.TB_ERR_UNSUPPORTED, _capi.TB_ERR_WORKSPACE
FAKE = C.c_void_p(0x10000)


@pytest.fixture(scope="module")
def lib():
    return _capi.load()


def desc(lib, **kw):
    d = _capi.tb_grouped_desc()
    assert lib.tb_grouped_desc_init(C.byref(d)) == OK
    assert (d.groups, d.ab_dtype, d.c_dtype, d.beta) == (1, _capi.TB_F16, _capi.TB_F32, 1)
    for key, v in dict(dict(groups=4, rows=64, n=64, k=64), **kw).items():
        setattr(d, key, v)
    return d


def scales(block=1, ptr=0x10000):
    s = _capi.tb_scales()
    s.ptr, s.stride_mn, s.stride_k, s.block = ptr, 1, 1, block
    return s


def rows(lib, d, A=FAKE, lda=64, B=FAKE, ldb=64, stride=4096, Cm=FAKE, ldc=64, off=FAKE):
    return lib.tb_grouped_matmul(d and C.byref(d), A, lda, B, ldb, stride, Cm, ldc, off, None, 0, None)


def wgrad(lib, d, A=FAKE, lda=64, D=FAKE, ldd=64, G=FAKE, ldg=64, off=FAKE):
    return lib.tb_grouped_matmul_wgrad(d and C.byref(d), A, lda, D, ldd, G, ldg, 4096, off, None, 0, None)


def bytes_(lib, d, A=FAKE, lda=64, sa=None, B=FAKE, ldb=64, sb=None):
    return lib.tb_matmul_blockscaled(d and C.byref(d), A, lda, sa, B, ldb, sb, FAKE, 64, None, 0, None)


def test_descs_are_checked(lib):
    assert lib.tb_grouped_desc_init(None) == INVALID
    for call in (rows, wgrad):
        assert call(lib, None) == INVALID
        assert call(lib, desc(lib, rows=-1)) == INVALID
        assert call(lib, desc(lib, beta=2)) == INVALID
        assert call(lib, desc(lib, ab_dtype=_capi.TB_F32)) == INVALID
        assert call(lib, desc(lib, ab_dtype=_capi.TB_E4M3)) == INVALID
        assert call(lib, desc(lib, c_dtype=_capi.TB_E4M3)) == INVALID
        assert call(lib, desc(lib, groups=1025)) == UNSUPPORTED
        assert call(lib, desc(lib, n=1 << 32)) == UNSUPPORTED
        assert call(lib, desc(lib, rows=1 << 30, n=1 << 30)) == UNSUPPORTED
        assert call(lib, desc(lib, a_col_major=1)) == UNSUPPORTED
    assert wgrad(lib, desc(lib, b_col_major=1)) == UNSUPPORTED
    assert bytes_(lib, desc(lib, groups=1)) == INVALID            # f16 operands
    assert bytes_(lib, desc(lib, ab_dtype=_capi.TB_E4M3)) == INVALID  # four groups


def test_operands_are_checked(lib):
    d = desc(lib)
    for name in ("A", "B", "Cm", "off"):
        assert rows(lib, d, **{name: None}) == INVALID
    for name in ("A", "D", "G", "off"):
        assert wgrad(lib, d, **{name: None}) == INVALID
    for name in ("lda", "ldb", "ldc"):
        assert rows(lib, d, **{name: 63}) == INVALID
    for name in ("lda", "ldd", "ldg"):
        assert wgrad(lib, d, **{name: 63}) == INVALID
    assert b"leading dimension" in lib.tb_last_error()
    assert rows(lib, d, Cm=C.c_void_p(0x10002)) == INVALID        # f32 C on a 2-byte boundary
    assert rows(lib, d, off=C.c_void_p(0x10002)) == INVALID


def test_scales_are_checked(lib):
    d = desc(lib, groups=1, ab_dtype=_capi.TB_E4M3)
    good = scales()
    assert bytes_(lib, d, sa=None, sb=C.byref(good)) == INVALID
    assert bytes_(lib, d, sa=C.byref(good), sb=C.byref(scales(ptr=None))) == INVALID
    assert bytes_(lib, d, sa=C.byref(scales(64)), sb=C.byref(good)) == INVALID
    g = desc(lib, ab_dtype=_capi.TB_E4M3)
    assert lib.tb_grouped_matmul_blockscaled(C.byref(g), FAKE, 64, C.byref(scales(128)), FAKE, 64, 4096,
                                             C.byref(good), FAKE, 64, FAKE, None, 0, None) == UNSUPPORTED


def test_repacking_asks_for_its_workspace(lib):
    d = desc(lib)
    need = lib.tb_grouped_matmul_workspace_bytes
    assert need(C.byref(d), FAKE, 64, FAKE, 64, 4096) == 0
    assert need(C.byref(d), FAKE, 65, FAKE, 64, 4096) == 64 * 64 * 2           # A alone
    assert need(C.byref(d), FAKE, 64, FAKE, 64, 4097) == 4 * 64 * 64 * 2       # B alone
    assert need(C.byref(d), C.c_void_p(0x10002), 64, FAKE, 65, 65 * 64) == 5 * 64 * 64 * 2
    odd = desc(lib, k=37, n=51)
    assert need(C.byref(odd), FAKE, 37, FAKE, 51, 37 * 51) == 64 * 40 * 2 + (4 * 37 * 56 * 2 + 255) // 256 * 256
    assert rows(lib, d, lda=65) == WORKSPACE
    assert b"8192" in lib.tb_last_error()
    assert wgrad(lib, d, ldd=65) == WORKSPACE
    assert lib.tb_grouped_matmul_wgrad_workspace_bytes(C.byref(d), FAKE, 64, FAKE, 65) == 8192


def test_nothing_to_do_is_ok_without_operands(lib):
    for kw in (dict(rows=0), dict(n=0), dict(groups=0)):
        assert rows(lib, desc(lib, **kw), A=None, B=None, Cm=None) == OK
    for kw in (dict(k=0), dict(n=0), dict(groups=0)):
        assert wgrad(lib, desc(lib, **kw), A=None, D=None, G=None) == OK


def test_quantize_refusals(lib):
    def call(X=FAKE, ldx=64, Q=FAKE, S=FAKE, ldq=64, **kw):
        d = _capi.tb_quantize_desc()
        for key, v in dict(dict(batch=1, rows=8, cols=64, block_rows=1, block_cols=128, x_dtype=_capi.TB_F16),
                           **kw).items():
            setattr(d, key, v)
        return lib.tb_quantize_blocks(C.byref(d), X, ldx, 0, Q, ldq, 0, S, 0, 1, 1, None)
    assert lib.tb_quantize_blocks(None, FAKE, 64, 0, FAKE, 64, 0, FAKE, 0, 1, 1, None) == INVALID
    assert call(rows=-1) == INVALID
    assert call(block_rows=1, block_cols=64) == INVALID
    assert call(block_rows=1, block_cols=1) == INVALID
    assert call(x_dtype=_capi.TB_E4M3) == INVALID
    for name in ("X", "Q", "S"):
        assert call(**{name: None}) == INVALID
    assert call(ldx=63) == INVALID and call(ldq=63) == INVALID
    assert call(X=C.c_void_p(0x10001)) == INVALID
    assert call(batch=1 << 20, rows=1 << 20, cols=1 << 20, ldx=1 << 20, ldq=1 << 20) == UNSUPPORTED
    assert call(rows=0, X=None, Q=None, S=None) == OK


def test_python_refusals():
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    h = torch.float16
    A, B, Cm, off = torch.ones(4, 8, dtype=h), torch.ones(2, 8, 16, dtype=h), torch.ones(4, 16), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(tb.TBError, match="CUDA tensor"):
        tb.grouped_matmul(A, B, Cm, off)
    with pytest.raises(tb.TBError, match="CUDA tensor"):
        tb.grouped_matmul_wgrad(A, Cm, B, off)
    with pytest.raises(tb.TBError, match="CUDA tensor"):
        tb.quantize_fp8(A)
    with pytest.raises(tb.TBError, match="blocks are"):
        tb.quantize_fp8(A, block=(1, 64))
    with pytest.raises(tb.TBError, match="CUDA tensor"):
        tb.matmul_fp8(A, A, A, A, A)
    from mini_triton_nvgpu_v1_b200 import grouped
    with pytest.raises(tb.TBError, match="entries"):
        grouped._check_offsets(off, 3)
    with pytest.raises(tb.TBError, match="int32 or int64"):
        grouped._check_offsets(off.float(), 2)
    with pytest.raises(tb.TBError, match="contiguous"):
        grouped._check_offsets(torch.zeros(6, dtype=torch.int32)[::2], 2)
    with pytest.raises(tb.TBError, match="overlap"):
        grouped._batch(torch.zeros(8, 16).expand(2, 8, 16), "B")
    with pytest.raises(tb.TBError, match="unit stride"):
        grouped._rows(torch.zeros(8, 32)[:, ::2], "A")
    with pytest.raises(tb.TBError, match="unit stride"):
        grouped._either(torch.zeros(16, 32)[::2, ::2], "B")
    with pytest.raises(tb.TBError, match="for each block"):
        grouped._scales(torch.zeros(4, 2, dtype=torch.float64), "SA", 4, 256, 0, 1, ())
    with pytest.raises(tb.TBError, match="1 or 128"):
        grouped._scales(torch.zeros(4, 3), "SA", 4, 256, 0, 1, ())


def test_layouts_of_views():
    import torch
    from mini_triton_nvgpu_v1_b200 import grouped
    x = torch.zeros(6, 10)
    assert grouped._either(x, "x") == (False, 10)
    assert grouped._either(x.t(), "x") == (True, 10)
    assert grouped._either(x[:, :1], "x") == (False, 10)   # one column: a row-major view with its row stride
    assert grouped._either(x[:1], "x") == (False, 10)
    assert grouped._either(x[:1, :1], "x") in ((False, 1), (True, 1))
    assert grouped._batch(torch.zeros(3, 4, 5), "x") == 20
    assert grouped._batch(torch.zeros(4, 3, 5).transpose(0, 1), "x") == 5


def test_outputs_do_not_overlap():
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    from mini_triton_nvgpu_v1_b200 import grouped
    for t in (torch.zeros(4, 1).expand(4, 3), torch.zeros(3).expand(4, 3), torch.zeros(5).as_strided((2, 3), (2, 1)),
              torch.zeros(1, 4, 3).expand(2, 4, 3)):
        with pytest.raises(tb.TBError, match="overlap"):
            grouped._apart(t, "S")
    for t in (torch.zeros(4, 3), torch.zeros(4, 3).t(), torch.zeros(6, 8)[::2, ::3], torch.zeros(1).expand(1, 1)):
        grouped._apart(t, "S")


def test_known_calls_take_whole_numbers_only():
    """A beta or block that is no whole number is left to the checks, not answered by a TypeError."""
    import torch
    from mini_triton_nvgpu_v1_b200 import grouped
    t = torch.zeros(2, 2)
    for beta in (0.5, 1.0, None, 1 << 80, "1"):
        assert grouped._call0(grouped._ROWS, t, t, t, t, beta, 0) == -1


def test_selftest_budget_is_validated(lib):
    assert lib.tb_selftest_grouped_wait(None, 0) == INVALID
    assert lib.tb_selftest_grouped_wait(None, 3_000_000_000) == INVALID
