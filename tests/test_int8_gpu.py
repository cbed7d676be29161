"""int8 quantizers and int8 products against plain 64-bit forms.

The quantizers' codes and scales are compared exactly: their FP32 operations are single
correctly rounded ones, and a 64-bit quotient or product of two FP32 values rounded to
FP32 is the correctly rounded FP32 result (64-bit has more than twice the digits).  The
products' sums are exact integers, so D equals the same three FP32 operations done on
them elementwise, bit for bit; against 64 bits it is off by at most 2^-24 for each of
the conversion, two products and the sum, and half a step of D's type."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ("float32", "bfloat16", "float16")


def _codes_64(x, axis):
    """Codes and scales along `axis` of x (numpy float32), in 64 bits rounded to FP32 per step."""
    a = np.max(np.abs(x), axis=axis, keepdims=True, initial=2.0 ** -100).astype(np.float32)
    bad = ~np.isfinite(x).all(axis=axis, keepdims=True)
    a = np.where(bad, np.float32(1), a).astype(np.float64)
    scale = (a / 127.0).astype(np.float32)
    inv = (127.0 / a).astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        t = (x.astype(np.float64) * inv).astype(np.float32)
    codes = np.where(bad, 0.0, np.rint(t)).astype(np.int8)
    return codes, np.where(bad, np.float32("nan"), scale).squeeze(axis)


def _same(a, b):
    return bool(np.all((a == b) | (np.isnan(a) & np.isnan(b))))


def _values(rng, shape, kind):
    x = rng.standard_normal(shape).astype(np.float32)
    if kind == "wide":
        x *= np.exp(rng.uniform(-40, 40, shape[:-1] + (1,))).astype(np.float32)
    elif kind == "ties":  # multiples of half a code step where the largest value is 127
        x = (rng.integers(-254, 255, shape) / 2).astype(np.float32)
        x[..., :1] = 127.0
    elif kind == "special":
        x[rng.random(shape) < 0.02] = np.nan
        x[rng.random(shape) < 0.02] = np.inf
        x[rng.random(shape) < 0.02] = -np.inf
    elif kind == "zeros":
        x[::2] = 0.0
        x[1::2] = -0.0
    elif kind == "tiny":
        x *= np.float32(2.0 ** -120)
    return x


def _tensor(x, dtype, pad=0, shift=0):
    """x on the GPU with `pad` extra elements per row (garbage NaN) and its base `shift`
    elements off the allocation's."""
    import torch

    t = torch.from_numpy(np.ascontiguousarray(x)).cuda().to(getattr(torch, dtype))
    shape = tuple(t.shape[:-1]) + (t.shape[-1] + pad,)
    flat = torch.full((int(np.prod(shape)) + shift,), float("nan"), dtype=t.dtype, device="cuda")
    view = flat[shift:].view(shape)[..., :t.shape[-1]]
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["normal", "wide", "ties", "special", "zeros", "tiny"])
@pytest.mark.parametrize("M,K,pad,shift", [(1, 1, 0, 0), (3, 7, 0, 0), (5, 4096, 0, 0), (2, 2051, 0, 0),
                                           (33, 520, 8, 0), (4, 129, 3, 1), (1, 20000, 0, 0), (2500, 64, 0, 0)])
def test_rows(mpk_lib, cuda, dtype, kind, M, K, pad, shift):
    import torch

    rng = np.random.default_rng(M * 7 + K)
    x = _tensor(_values(rng, (M, K), kind), dtype, pad, shift)
    codes, scales = mpk_lib.quantize_int8(x)
    want_c, want_s = _codes_64(x.float().cpu().numpy(), 1)
    assert np.array_equal(codes.cpu().numpy(), want_c)
    assert _same(scales.cpu().numpy(), want_s)
    assert codes.stride(0) % 16 == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["normal", "special", "zeros"])
@pytest.mark.parametrize("E,K,N,pad,shift", [(1, 1, 1, 0, 0), (1, 5, 8, 0, 0), (3, 515, 130, 0, 0), (2, 64, 4096, 0, 0),
                                             (2, 300, 72, 8, 0), (2, 33, 31, 0, 1), (1, 9000, 16, 0, 0)])
def test_cols(mpk_lib, cuda, dtype, kind, E, K, N, pad, shift):
    rng = np.random.default_rng(E + K * 3 + N)
    w = _tensor(_values(rng, (E, K, N), kind), dtype, pad, shift)
    want_c, want_s = _codes_64(w.float().cpu().numpy(), 1)
    codes, scales = mpk_lib.quantize_int8_cols(w)
    assert np.array_equal(codes.cpu().numpy(), want_c)
    assert _same(scales.cpu().numpy(), want_s)
    if E == 1:
        codes, scales = mpk_lib.quantize_int8_cols(w[0])
        assert np.array_equal(codes.cpu().numpy(), want_c[0]) and _same(scales.cpu().numpy(), want_s[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,K,N", [(160, 40, 128), (160, 513, 128), (150, 1025, 128), (40, 2049, 512), (64, 2100, 100),
                                   (1, 700, 320), (1, 8, 24), (300, 17, 5), (9, 1, 2048)])
def test_cols_of_every_split(mpk_lib, cuda, dtype, E, K, N):
    """Many strips and few: one to eight blocks share a strip's rows, some of them without a row."""
    rng = np.random.default_rng(E * 5 + K + N)
    x = _values(rng, (E, K, N), "normal")
    x[::3, -1] = np.inf  # the last block's row alone spoils every column of some matrices
    w = _tensor(x, dtype)
    want_c, want_s = _codes_64(w.float().cpu().numpy(), 1)
    codes, scales = mpk_lib.quantize_int8_cols(w)
    assert np.array_equal(codes.cpu().numpy(), want_c)
    assert _same(scales.cpu().numpy(), want_s)


def test_quantizers_leave_the_padding_and_take_no_rows(mpk_lib, cuda):
    import torch

    x = torch.randn((6, 20), device="cuda")
    codes = torch.full((6, 32), 99, dtype=torch.int8, device="cuda")
    s = torch.empty(6, device="cuda")
    mpk_lib.int8_quantize_rows_gpu(x, mpk_lib.TYPE_F32, 20, codes, 32, s, 6, 20)
    assert bool((codes[:, 20:] == 99).all()) and bool((codes[:, :20] == mpk_lib.quantize_int8(x)[0]).all())
    codes.fill_(99)
    s = torch.empty(20, device="cuda")
    mpk_lib.int8_quantize_cols_gpu(x, mpk_lib.TYPE_F32, 20, codes, 32, s, 1, 6, 20)
    assert bool((codes[:, 20:] == 99).all())
    codes, s = mpk_lib.quantize_int8(torch.empty((0, 8), device="cuda"))
    assert codes.shape == (0, 8) and s.shape == (0,)
    codes, s = mpk_lib.quantize_int8(torch.empty((3, 0), device="cuda"))
    assert codes.shape == (3, 0) and bool((s == np.float32(np.float32(2.0 ** -100) / np.float32(127))).all())


# ------------------------------- products -----------------------------------

HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _random_codes(rng, shape):
    return rng.integers(-128, 128, shape, dtype=np.int64).astype(np.int8)


def _padded(x, pad, shift=0):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    shape = tuple(t.shape[:-1]) + (t.shape[-1] + pad,)
    flat = torch.full((int(np.prod(shape)) + shift,), 77, dtype=torch.int8, device="cuda")
    view = flat[shift:].view(shape)[..., :t.shape[-1]]
    view.copy_(t)
    return view


def _check(D, acc, sa, sb, bias, dtype):
    """D against the elementwise FP32 operations (exactly) and against 64 bits."""
    import torch

    v = (acc.astype(np.float32) * sa[:, None]) * sb
    d64 = acc.astype(np.float64) * sa[:, None].astype(np.float64) * sb.astype(np.float64)
    scale = np.abs(d64)
    if bias is not None:
        v = v + bias
        d64 = d64 + bias.astype(np.float64)
        scale = scale + np.abs(d64)
    want = torch.from_numpy(v).to(getattr(torch, dtype))
    got = D.cpu()
    assert got.dtype == want.dtype and torch.equal(got, want)
    # three roundings of the scaled sum, one of the sum with the bias, one to D's type
    bound = 4 * 2.0 ** -24 * scale + HALF[dtype] * (1 + 2.0 ** -20) * np.abs(d64)
    assert np.all(np.abs(got.double().numpy() - d64) <= bound)


SHAPES = [(1, 1, 1), (1, 16, 16), (3, 5, 7), (1, 4096, 512), (37, 1003, 515), (128, 128, 128), (129, 257, 130),
          (300, 520, 1024), (256, 256, 4096), (513, 768, 2000), (2, 130, 8192), (700, 300, 48)]


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(mpk_lib, cuda, M, N, K, layout):
    rng = np.random.default_rng(M + 3 * N + 7 * K)
    a, b = _random_codes(rng, (M, K)), _random_codes(rng, (K, N))
    if M > 2:
        a[0], b[:, 0] = -128, -128  # the largest sums
    sa = (rng.uniform(0.5, 2.0, M) * 2.0 ** -10).astype(np.float32)
    sb = (rng.uniform(0.5, 2.0, N) * 2.0 ** -8).astype(np.float32)
    acc = a.astype(np.int64) @ b.astype(np.int64)
    import torch

    SA, SB = torch.from_numpy(sa).cuda(), torch.from_numpy(sb).cuda()
    for pad, shift, dtype, with_bias in ((0, 0, "bfloat16", False), ((-K) % 16 + 16, 0, "float32", True),
                                         (3, 1, "float16", True)):
        A = _padded(a, pad, shift)
        if layout == "kn":
            B = _padded(b, (-N) % 16 if shift == 0 else 5, shift)
        else:
            B = _padded(b.T, (-K) % 16 if shift == 0 else 5, shift)
        bias = rng.standard_normal(N).astype(np.float32) if with_bias else None
        D = mpk_lib.gemm_int8(A, SA, B, SB, None if bias is None else torch.from_numpy(bias).cuda(),
                              getattr(torch, dtype), mpk_lib.B_KN if layout == "kn" else mpk_lib.B_NK)
        _check(D, acc, sa, sb, bias, dtype)
    assert mpk_lib.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 256, 512), (5, 77, 130), (200, 384, 1024), (600, 1000, 264)])
def test_linear_is_the_quantizer_and_the_product(mpk_lib, cuda, dtype, M, N, K):
    import torch

    rng = np.random.default_rng(M + N + K)
    x = _tensor(_values(rng, (M, K), "normal"), dtype)
    w = _tensor(_values(rng, (K, N), "normal"), "bfloat16")
    bias = torch.randn(N, device="cuda")
    B, sb = mpk_lib.quantize_int8_cols(w)
    D = mpk_lib.linear_int8(x, B, sb, bias)
    q, s = mpk_lib.quantize_int8(x)
    assert torch.equal(D, mpk_lib.gemm_int8(q, s, B, sb, bias, x.dtype))
    acc = q.cpu().numpy().astype(np.int64) @ B.cpu().numpy().astype(np.int64)
    _check(D, acc, s.cpu().numpy(), sb.cpu().numpy(), bias.cpu().numpy(), dtype)
    # against the product of the unquantized operands: a code is off by half a step, that is
    # by at most scale / 2 (and 127 * 2^-23 of a step where x * (127 / a) was rounded)
    X, W, S, T = x.double(), w.double(), s.double()[:, None] * 0.5001, sb.double() * 0.5001
    # |xw - (x + dx)(w + dw)| <= |x||dw| + |dx||w| + |dx||dw|, plus the FP32 and output roundings
    off = X.abs().sum(1, keepdim=True) * T + S * W.abs().sum(0) + K * S * T
    exact = X @ W + bias.double()
    off = off + (HALF[dtype] + 2.0 ** -20) * (exact.abs() + off)
    assert bool(((D.double() - exact).abs() <= off).all())


def test_nan_rows_and_columns_show(mpk_lib, cuda):
    import torch

    x = torch.randn((4, 64), device="cuda", dtype=torch.bfloat16)
    w = torch.randn((64, 48), device="cuda", dtype=torch.bfloat16)
    x[1, 3], x[2, 5], w[7, 9] = float("nan"), float("inf"), float("-inf")
    B, sb = mpk_lib.quantize_int8_cols(w)
    D = mpk_lib.linear_int8(x, B, sb)
    bad = torch.zeros((4, 48), dtype=torch.bool, device="cuda")
    bad[1:3] = True
    bad[:, 9] = True
    assert torch.equal(torch.isnan(D), bad)


def test_empty_sizes_and_strided_results(mpk_lib, cuda):
    import torch

    m = mpk_lib
    A, sa = torch.zeros((5, 0), dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda")
    B, sb = torch.zeros((0, 9), dtype=torch.int8, device="cuda"), torch.ones(9, device="cuda")
    bias = torch.arange(9.0, device="cuda")
    assert torch.equal(m.gemm_int8(A, sa, B, sb, bias, torch.float32), bias.expand(5, 9))
    assert bool((m.gemm_int8(A, sa, B, sb) == 0).all())
    assert m.gemm_int8(A[:0], sa[:0], B, sb).shape == (0, 9)
    assert m.gemm_int8(A, sa, B[:, :0], sb[:0]).shape == (5, 0)
    x = torch.zeros((3, 0), device="cuda")
    assert torch.equal(m.linear_int8(x, B, sb, bias), bias.expand(3, 9))
    A = torch.ones((5, 32), dtype=torch.int8, device="cuda")
    B = torch.ones((32, 9), dtype=torch.int8, device="cuda")
    for width, first in ((16, 0), (17, 3), (64, 32)):
        whole = torch.full((5, width + 9), 7.0, device="cuda")
        m.gemm_int8(A, sa, B, sb, bias, out=whole[:, first:first + 9])
        assert torch.equal(whole[:, first:first + 9], bias.expand(5, 9) + 32)
        assert bool((whole[:, :first] == 7).all()) and bool((whole[:, first + 9:] == 7).all())


def test_largest_reduction_is_exact(mpk_lib, cuda):
    """K = 131071 of -128 * -128: the largest sum, 2^31 - 2^14, whose FP32 value is 2^31."""
    import torch

    K = 131071
    A = _padded(np.full((2, K), -128, np.int8), 1)
    B = _padded(np.full((16, K), -128, np.int8), 1)
    B[1, 1:] = 0
    one = torch.ones(16, device="cuda")
    D = mpk_lib.gemm_int8(A, one[:2], B, one, out_dtype=torch.float32, b_layout=mpk_lib.B_NK)
    want = torch.full((2, 16), float(np.float32(K * 16384)), device="cuda")
    want[:, 1] = 16384.0
    assert torch.equal(D, want)


def test_streams_and_graphs(mpk_lib, cuda):
    """Two streams at once, and two captured graphs that both need a workspace, replayed
    with new inputs while eager calls run."""
    import torch

    m = mpk_lib
    g = torch.Generator(device="cuda").manual_seed(5)
    w = torch.randn((520, 1003), device="cuda", generator=g)
    B, sb = m.quantize_int8_cols(w)
    Bt = B.t().contiguous()  # rows of 520: TMA reads it in place; the odd B below is copied
    odd = torch.empty((520 * 1003 + 1,), dtype=torch.int8, device="cuda")[1:].view(520, 1003)
    odd.copy_(B)
    xs = [torch.randn((n, 520), device="cuda", generator=g) for n in (3, 300)]
    want = [m.linear_int8(x, B, sb).clone() for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                outs.append(m.linear_int8(x, odd, sb))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want[i % 2])
    graphs = []
    ins = [torch.zeros_like(x) for x in xs]
    for x in ins:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = m.linear_int8(x, odd, sb)
            z = m.linear_int8(x, Bt, sb, b_layout=m.B_NK)
        graphs.append((gr, y, z))
    for rep in range(2):
        for x, i in zip(xs, ins):
            i.copy_(x * (1 + rep))
        torch.cuda.synchronize()
        for (gr, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        eager = m.linear_int8(xs[0], B, sb)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        for (gr, y, z), v in zip(graphs, want):
            assert torch.equal(y, z) and torch.equal(y, v * (1 + rep))
    assert m.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 17, 700])
def test_linear_of_unaligned_and_strided_rows(mpk_lib, cuda, dtype, M):
    """Rows of x off a 16-byte boundary and apart, weights off it too, D odd columns wide and
    inside a larger tensor; the same result as from contiguous operands."""
    import torch

    m = mpk_lib
    rng = np.random.default_rng(M)
    K, N = 333, 65
    x = _values(rng, (M, K), "normal")
    B, sb = m.quantize_int8_cols(_tensor(_values(rng, (K, N), "normal"), "float32"))
    plain = m.linear_int8(_tensor(x, dtype), B, sb)
    odd = torch.empty((K * N + 3,), dtype=torch.int8, device="cuda")[3:].view(K, N)
    odd.copy_(B)
    whole = torch.full((M, 2 * N + 1), 5.0, dtype=plain.dtype, device="cuda")
    for pad, shift in ((3, 1), (8, 0), (5, 7)):
        for w in (B, odd):
            D = m.linear_int8(_tensor(x, dtype, pad, shift), w, sb, out=whole[:, 1:N + 1])
            assert torch.equal(D, plain)
            assert bool((whole[:, 0] == 5).all()) and bool((whole[:, N + 1:] == 5).all())
    assert m.device_status() == 0


def test_fused_and_separate_quantizers_agree(mpk_lib, cuda):
    """Few rows are quantized inside the product (up to 16 of 512, 1 of 8192), more in a kernel
    of their own: a row's result does not depend on how many others come with it."""
    import torch

    m = mpk_lib
    for K in (64, 512, 1000, 4096, 8192, 8200, 20000):
        x = torch.randn((33, K), device="cuda").bfloat16()
        x[1, K // 2] = float("nan")
        B, sb = m.quantize_int8_cols(torch.randn((K, 300), device="cuda"))
        all_rows = m.linear_int8(x, B, sb, out_dtype=torch.float32)
        for n in (1, 2, 3, 4, 7, 8, 9, 16, 17):
            got = m.linear_int8(x[:n], B, sb, out_dtype=torch.float32)
            assert torch.equal(got.nan_to_num(7.0), all_rows[:n].nan_to_num(7.0))
            assert torch.equal(got.isnan(), all_rows[:n].isnan())
    assert m.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 4096), (1, 8192), (2, 4096), (16, 512), (7, 500), (17, 1024), (300, 264)])
def test_linear_in_place_of_its_input(mpk_lib, cuda, dtype, M, K):
    """D written over x, or a row further down in x's tensor, is the D of a call that keeps x,
    for rows that the product quantizes itself as for more."""
    import torch

    m = mpk_lib
    rng = np.random.default_rng(M + K)
    x = _tensor(_values(rng, (M, K), "normal"), dtype)
    B, sb = m.quantize_int8_cols(_tensor(_values(rng, (K, K), "normal"), "float32"))
    want = m.linear_int8(x, B, sb)
    for down in (0, 1):
        for _ in range(5):
            whole = torch.zeros((M + 1, K), dtype=x.dtype, device="cuda")
            whole[:M] = x
            m.linear_int8(whole[:M], B, sb, out=whole[down:M + down])
            assert torch.equal(whole[down:M + down], want)
    assert m.device_status() == 0


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("M,N,K", [(1030, 2570, 200), (2100, 2570, 200), (4500, 1300, 130), (40, 19500, 64)])
def test_product_of_many_tiles(mpk_lib, cuda, M, N, K, layout):
    """Sizes at which pairs of CTAs share a tile (the first three), a CTA has more tiles than one,
    so that its second accumulator and both accumulators' row scales come into use (the
    last three), and a row's tiles make more than one panel (4500 rows)."""
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(M + N + K)
    a = torch.randint(-128, 128, (M, K), generator=gen, device="cuda").to(torch.int8)
    b = torch.randint(-128, 128, (K, N), generator=gen, device="cuda").to(torch.int8)
    sa = (torch.rand(M, generator=gen, device="cuda") + 0.5) * 2.0 ** -10
    sb = (torch.rand(N, generator=gen, device="cuda") + 0.5) * 2.0 ** -8
    sa[3 % M], sa[M - 1], sb[N - 2] = float("nan"), float("inf"), float("nan")
    bias = torch.randn(N, generator=gen, device="cuda")
    acc = a.double() @ b.double()
    want = acc.float() * sa[:, None] * sb
    kept = b if layout == "kn" else b.t()
    for pad, dtype, add in ((16 - kept.shape[1] % 16, torch.bfloat16, None), (16 - kept.shape[1] % 16, torch.float32, bias),
                            (1, torch.float16, bias)):
        B = torch.full((kept.shape[0], kept.shape[1] + pad), 77, dtype=torch.int8, device="cuda")[:, :kept.shape[1]]
        B.copy_(kept)
        A = torch.full((M, K + (-K) % 16 + 16), 77, dtype=torch.int8, device="cuda")[:, :K]
        A.copy_(a)
        whole = torch.full((M + 1, N + 6), 5.0, dtype=dtype, device="cuda")
        D = m.gemm_int8(A, sa, B, sb, add, b_layout=m.B_KN if layout == "kn" else m.B_NK, out=whole[:M, :N])
        full = (want if add is None else want + add).to(dtype)
        assert bool(((D == full) | (D.isnan() & full.isnan())).all())
        assert bool((whole[M:] == 5).all()) and bool((whole[:, N:] == 5).all())
    assert m.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 19500, 130), (1, 40000, 64), (16, 19500, 72), (3, 38000, 2048)])
def test_fused_codes_serve_many_tiles(mpk_lib, cuda, dtype, M, N, K):
    """More columns than the SMs take at once: a CTA multiplies the codes that it made with the
    weights of its second and third tile too."""
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(M + N + K)
    x = torch.randn((M, K), generator=gen, device="cuda").to(getattr(torch, dtype))
    x[M - 1, K // 2] = float("nan") if M > 1 else 9.0
    B = torch.randint(-127, 128, (K, N), generator=gen, device="cuda").to(torch.int8)
    sb = torch.rand(N, generator=gen, device="cuda")
    q, s = m.quantize_int8(x)
    want = (q.double() @ B.double()).float() * s[:, None] * sb
    D = m.linear_int8(x, B, sb, out_dtype=torch.float32)
    assert bool(((D == want) | (D.isnan() & want.isnan())).all())
    assert m.device_status() == 0
