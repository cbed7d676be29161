"""Refusals of the int8 and expert-grouped entry points, answered on the host before any
device work (no GPU needed), and the argument checks of their allocating forms."""
import ctypes

import numpy as np
import pytest

INVALID, UNSUPPORTED, MISALIGNED, ARCH = 1001, 1002, 1003, 1005
PTR = 1 << 20  # never dereferenced: every call below is refused on the host
BF16, F16, F32 = 1, 2, 0


def _grouped(L, A=PTR, lda=64, B=PTR, ldb=64, layout=0, ab=BF16, D=PTR, d=BF16, ldd=64, off=PTR, E=2, M=8, N=64,
             K=64):
    return L.mpk_gemm_grouped(A, lda, B, ldb, layout, ab, D, d, ldd, off, E, M, N, K, None)


def _wgrad(L, A=PTR, lda=64, G=PTR, ldg=64, ab=BF16, D=PTR, d=BF16, ldd=64, off=PTR, E=2, M=8, N=64, K=64):
    return L.mpk_gemm_grouped_wgrad(A, lda, G, ldg, ab, D, d, ldd, off, E, M, N, K, None)


def _int8(L, A=PTR, lda=64, sa=PTR, B=PTR, ldb=64, layout=0, sb=PTR, bias=None, D=PTR, d=BF16, ldd=64, M=8, N=64,
          K=64):
    return L.mpk_gemm_int8(A, lda, sa, B, ldb, layout, sb, bias, D, d, ldd, M, N, K, None)


def _linear(L, x=PTR, t=BF16, ldx=64, B=PTR, ldb=64, layout=0, sb=PTR, bias=None, D=PTR, d=BF16, ldd=64, M=8, N=64,
            K=64):
    return L.mpk_linear_int8(x, t, ldx, B, ldb, layout, sb, bias, D, d, ldd, M, N, K, None)


def _grouped_int8(L, A=PTR, lda=64, sa=PTR, B=PTR, ldb=64, layout=0, sb=PTR, D=PTR, d=BF16, ldd=64, off=PTR, E=2,
                  M=8, N=64, K=64):
    return L.mpk_gemm_grouped_int8(A, lda, sa, B, ldb, layout, sb, D, d, ldd, off, E, M, N, K, None)


def _mxfp8(L, A=PTR, sa=PTR, B=PTR, ldb=64, D=PTR, sd=PTR, off=PTR, E=2, M=8, N=64, K=64):
    return L.mpk_gemm_grouped_mxfp8(A, sa, B, ldb, D, sd, off, E, M, N, K, None)


@pytest.mark.parametrize("call", [_grouped, _wgrad, _int8, _linear, _grouped_int8, _mxfp8])
def test_sizes_and_pointers_are_refused(mpk_lib, call):
    L = mpk_lib.lib()
    for size in ("M", "N", "K"):
        assert call(L, **{size: -1}) == INVALID
        assert call(L, **{size: 2 ** 31 - 1}) == UNSUPPORTED
    assert call(L, B=None) == INVALID if call is not _wgrad else call(L, G=None) == INVALID
    assert call(L, D=None) == INVALID
    if call is _linear:
        assert call(L, x=None) == INVALID
    else:
        assert call(L, A=None) == INVALID
    assert b"null" in L.mpk_last_error_string()
    # nothing to do: success without a look at the pointers
    assert call(L, N=0, D=None, **({"G": None} if call is _wgrad else {"B": None})) == 0
    empty = {"K": 0} if call is _wgrad else {"M": 0}
    assert call(L, D=None, **empty) == 0


@pytest.mark.parametrize("call", [_grouped, _wgrad, _grouped_int8, _mxfp8])
def test_groups_are_checked(mpk_lib, call):
    L = mpk_lib.lib()
    assert call(L, E=-1) == INVALID
    assert call(L, E=mpk_lib.MAX_GROUPS + 1) == UNSUPPORTED
    assert call(L, off=None) == INVALID
    assert call(L, off=PTR + 2) == MISALIGNED
    assert call(L, E=0, off=None, D=None) == 0


@pytest.mark.parametrize("call", [_grouped, _wgrad, _int8, _linear, _grouped_int8])
def test_types_layouts_and_strides_are_refused(mpk_lib, call):
    L = mpk_lib.lib()
    for d in (-1, 3, 16, 17):
        assert call(L, d=d) == INVALID
    assert call(L, ldd=63) == INVALID
    assert call(L, ldd=1 << 62) == UNSUPPORTED
    if call is not _linear:
        assert call(L, lda=63) == INVALID
    else:
        assert call(L, ldx=63) == INVALID
        for t in (-1, 3, 16):
            assert call(L, t=t) == INVALID
    if call is _wgrad:
        assert call(L, ldg=63) == INVALID
    else:
        assert call(L, ldb=63) == INVALID
        assert call(L, layout=2) == INVALID and call(L, layout=-1) == INVALID
        # the stride is of rows of K elements in the other layout
        assert call(L, layout=1, N=128, ldd=128, K=65, **({"lda": 65} if call is not _linear else {"ldx": 65})) == INVALID
    if call in (_grouped, _wgrad):
        for ab in (F32, 3, 16, 17, -1):
            assert call(L, ab=ab) == INVALID
        assert call(L, A=PTR + 1) == MISALIGNED
    assert call(L, D=PTR + 1) == MISALIGNED


def test_int8_limits(mpk_lib):
    L = mpk_lib.lib()
    for call in (_int8, _linear, _grouped_int8):
        stride = {"ldx": 131072} if call is _linear else {"lda": 131072}
        assert call(L, K=131072, ldb=64, **stride) == UNSUPPORTED
        assert call(L, sb=None) == INVALID
        assert call(L, sb=PTR + 1) == MISALIGNED
    assert _int8(L, sa=None) == INVALID and _grouped_int8(L, sa=None) == INVALID
    assert _int8(L, bias=PTR + 2) == MISALIGNED
    assert _linear(L, x=PTR + 1) == MISALIGNED
    assert _mxfp8(L, sa=None) == INVALID and _mxfp8(L, sd=None) == INVALID


def test_quantizers_refuse(mpk_lib):
    L = mpk_lib.lib()

    def rows(x=PTR, t=BF16, ldx=64, codes=PTR, ldc=64, s=PTR, M=8, K=64):
        return L.mpk_int8_quantize_rows(x, t, ldx, codes, ldc, s, M, K, None)

    def cols(x=PTR, t=BF16, ldx=64, codes=PTR, ldc=64, s=PTR, E=2, K=8, N=64):
        return L.mpk_int8_quantize_cols(x, t, ldx, codes, ldc, s, E, K, N, None)

    for call in (rows, cols):
        assert call(K=-1) == INVALID
        assert call(t=3) == INVALID and call(t=-1) == INVALID
        assert call(x=None) == INVALID and call(codes=None) == INVALID and call(s=None) == INVALID
        assert call(ldx=63) == INVALID and call(ldc=63) == INVALID
        assert call(ldx=1 << 50) == UNSUPPORTED
        assert call(x=PTR + 1) == MISALIGNED and call(s=PTR + 2) == MISALIGNED
        assert call(t=F32, x=PTR + 2) == MISALIGNED
    assert rows(M=-1) == INVALID and rows(M=0, x=None, codes=None, s=None) == 0
    assert cols(E=-1) == INVALID and cols(N=-1) == INVALID
    assert cols(E=0, x=None, s=None) == 0 and cols(N=0, x=None, s=None) == 0


def test_a_checked_call_reaches_the_device_check(mpk_lib):
    """The defaults above are sound: without a GPU they are refused for the architecture
    (or by the CUDA runtime), and not for an argument."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("the defaults hold no device memory")
    L = mpk_lib.lib()
    for call in (_grouped, _wgrad, _int8, _linear, _grouped_int8, _mxfp8):
        assert call(L) == ARCH


def test_allocating_forms_check_their_tensors(mpk_lib):
    import torch

    m = mpk_lib
    x = torch.zeros((4, 8))
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        m.quantize_int8(x)
    with pytest.raises(ValueError, match="CUDA"):
        m.gemm_grouped(x.bfloat16(), torch.zeros((2, 8, 8)), off)
    with pytest.raises(ValueError, match="CUDA"):
        m.gemm_grouped_wgrad(x.bfloat16(), x.bfloat16(), off)
    # row strides
    assert m._row_stride(torch.zeros((4, 8)), "x") == 8
    assert m._row_stride(torch.zeros((4, 16))[:, :8], "x") == 16
    assert m._row_stride(torch.zeros((1, 8)), "x") == 8
    assert m._row_stride(torch.zeros((3, 4, 16))[..., :8], "x") == 16
    assert m._row_stride(torch.zeros((3, 5, 8))[:, :1], "x") == 40
    for bad in (torch.zeros((8, 4)).t(), torch.zeros((4, 1, 8)).expand(4, 3, 8), torch.zeros((3, 5, 8))[:, :2],
                torch.zeros((1, 8)).expand(4, 8), torch.zeros((4, 16))[:, ::2]):
        with pytest.raises(ValueError):
            m._row_stride(bad, "x")


def test_sizes_past_32_bits_are_refused(mpk_lib):
    """Sizes that a C int cannot hold raise; 2^32 + 5 rows are not taken for 5."""
    from types import SimpleNamespace

    import torch

    m = mpk_lib
    big = (1 << 32) + 5
    for sizes in ((big, 1, 1, 1), (1, big, 1, 1), (1, 1, big, 1), (1, 1, 1, big), (1, 1, 1, -big), (1, 1 << 31, 1, 1)):
        E, M, N, K = sizes
        for call in (lambda: m.gemm_grouped_gpu(PTR, K, PTR, N, m.B_KN, m.TYPE_BF16, PTR, m.TYPE_BF16, N, PTR, *sizes),
                     lambda: m.gemm_grouped_wgrad_gpu(PTR, K, PTR, N, m.TYPE_BF16, PTR, m.TYPE_BF16, N, PTR, *sizes),
                     lambda: m.gemm_grouped_int8_gpu(PTR, K, PTR, PTR, N, m.B_KN, PTR, PTR, m.TYPE_BF16, N, PTR,
                                                     *sizes),
                     lambda: m.gemm_grouped_mxfp8_gpu(PTR, PTR, PTR, N, PTR, PTR, PTR, *sizes)):
            with pytest.raises(ValueError, match="32-bit"):
                call()
    for M, N, K in ((big, 1, 1), (1, big, 1), (1, 1, big)):
        with pytest.raises(ValueError, match="32-bit"):
            m.gemm_int8_gpu(PTR, K, PTR, PTR, N, m.B_KN, PTR, None, PTR, m.TYPE_BF16, N, M, N, K)
        with pytest.raises(ValueError, match="32-bit"):
            m.int8_quantize_cols_gpu(PTR, m.TYPE_BF16, K, PTR, K, PTR, M, N, K)
        with pytest.raises(ValueError, match="32-bit"):
            m.linear_int8_gpu(PTR, m.TYPE_BF16, K, PTR, N, m.B_KN, PTR, None, PTR, m.TYPE_BF16, N, M, N, K)
    with pytest.raises(ValueError, match="32-bit"):
        m.int8_quantize_rows_gpu(PTR, m.TYPE_BF16, 1, PTR, 1, PTR, big, 1)
    # the allocating forms look at their tensors' shapes
    t = SimpleNamespace(shape=(big, 1), dtype=torch.int8, is_cuda=True, get_device=lambda: 0)
    with pytest.raises(ValueError, match="32-bit"):
        m._matrix(t, "x", 2, torch.int8)
