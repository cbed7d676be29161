"""Products grouped by expert and their gradients against plain 64-bit forms.

Most inputs are small integers: every product and partial sum is then exact in FP32, so D
has to equal the 64-bit result rounded once to D's type, whatever the order of the sums.
Random inputs are held to the bound of FP32 summation: products of 16-bit floats are
exact, and each of the K additions is off by at most one unit in the last place of a
partial sum, so |D - exact| <= K * 2^-23 * sum|a b|, plus half a step of D's type.  That
half step is relative to the value (2^-11 of it in FP16) only down to the smallest normal
number: below 2^-14 FP16's steps stay 2^-24, so a rounding there is off by up to 2^-25
however small the value, and the products of two normal variates reach below 2^-14."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
SUBNORMAL = {"float32": 0.0, "bfloat16": 0.0, "float16": 2.0 ** -25}


def _offsets(sizes, first=0):
    import torch

    return torch.tensor(np.concatenate([[first], first + np.cumsum(sizes)]), dtype=torch.int32, device="cuda")


def _ints(shape, gen, dtype, pad=0, shift=0, fill=float("nan"), span=3):
    """Integers of -span..span in a tensor whose rows have `pad` more elements (holding
    `fill`) and whose base is `shift` elements off its allocation's."""
    import torch

    t = torch.randint(-span, span + 1, shape, generator=gen, device="cuda").to(dtype)
    full = tuple(shape[:-1]) + (shape[-1] + pad,)
    flat = torch.full((int(np.prod(full)) + shift,), fill, dtype=dtype, device="cuda")
    view = flat[shift:].view(full)[..., :shape[-1]]
    view.copy_(t)
    return view


def _product_64(A, B, sizes, first=0):
    """[M, N] float64, NaN outside the groups; B [E, K, N]."""
    import torch

    out = torch.full((A.shape[0], B.shape[2]), float("nan"), dtype=torch.float64, device="cuda")
    lo = first
    for e, n in enumerate(sizes):
        out[lo:lo + n] = A[lo:lo + n].double() @ B[e].double()
        lo += n
    return out


def _wgrad_64(A, G, sizes, first=0):
    import torch

    out, lo = [], first
    for n in sizes:
        out.append(A[lo:lo + n].double().t() @ G[lo:lo + n].double())
        lo += n
    return torch.stack(out)


def _equal(got, want64, dtype):
    import torch

    want = want64.to(dtype)
    assert got.dtype == dtype
    bad = ~((got == want) | (got.isnan() & want.isnan()))
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())


SIZES = [[1], [0, 1, 0], [128, 128], [127, 129, 1, 0, 65], [256], [257, 0, 255, 300], [700], [0, 0, 0],
         [16, 15, 17, 64, 63], [513, 900]]
SHAPES = [(8, 8), (64, 64), (256, 128), (250, 72), (33, 100), (1, 1), (520, 264)]


@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("N,K", SHAPES)
def test_product_is_exact(mpk_lib, cuda, sizes, N, K):
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(N * 31 + K + len(sizes))
    E, M = len(sizes), sum(sizes)
    for layout, dtype, out, pad, shift in ((m.B_KN, torch.bfloat16, torch.bfloat16, 0, 0),
                                           (m.B_NK, torch.float16, torch.float32, 8, 0),
                                           (m.B_KN, torch.float16, torch.float16, 3, 1),
                                           (m.B_NK, torch.bfloat16, torch.float32, 0, 1)):
        A = _ints((M, K), gen, dtype, pad, shift)
        B = _ints((E, K, N) if layout == m.B_KN else (E, N, K), gen, dtype, pad, shift)
        D = m.gemm_grouped(A, B, _offsets(sizes), out, layout)
        _equal(D, _product_64(A, B if layout == m.B_KN else B.transpose(1, 2), sizes), out)
    assert m.device_status() == 0


@pytest.mark.parametrize("first,sizes,behind", [(0, [5, 0, 130, 9], 40), (7, [300, 64, 3], 200), (130, [0, 0], 5),
                                                (3, [900, 2], 1)], ids=str)
def test_rows_outside_the_groups(mpk_lib, cuda, first, sizes, behind):
    """Rows before, behind and of other groups: D's are left as they were, and NaN or
    infinity in A's, in other experts' weights or behind K does not reach a group."""
    import torch

    m = mpk_lib
    K, N = 72, 136
    gen = torch.Generator(device="cuda").manual_seed(first)
    M, E = first + sum(sizes) + behind, len(sizes)
    for layout in (m.B_KN, m.B_NK):
        for poisoned in range(E + 1):  # a group whose rows and weights are not finite; E: the rows outside
            A = _ints((M, K), gen, torch.bfloat16, 8)
            B = _ints((E, K, N) if layout == m.B_KN else (E, N, K), gen, torch.bfloat16, 8)
            lo = first + sum(sizes[:poisoned]) if poisoned < E else 0
            if poisoned < E:
                A[lo:lo + sizes[poisoned]] = float("nan")
                B[poisoned] = float("inf")
            else:
                A[:first] = float("inf")
                A[M - behind:] = float("nan")
            whole = torch.full((M, N + 8), 5.0, dtype=torch.bfloat16, device="cuda")
            D = m.gemm_grouped(A, B, _offsets(sizes, first), b_layout=layout, out=whole[:, :N])
            want = _product_64(A, B if layout == m.B_KN else B.transpose(1, 2), sizes, first)
            want[:first] = 5.0
            want[M - behind:] = 5.0
            _equal(D, want, torch.bfloat16)
            assert bool((whole[:, N:] == 5).all())


def test_many_groups_and_any_offsets(mpk_lib, cuda):
    """The most groups there can be, and offsets that are out of range or out of order: they
    are clamped, and nothing outside the operands is touched."""
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(2)
    rng = np.random.default_rng(3)
    sizes = rng.integers(0, 4, m.MAX_GROUPS).tolist()
    M = sum(sizes)
    A, B = _ints((M, 32), gen, torch.bfloat16), _ints((len(sizes), 32, 24), gen, torch.bfloat16)
    _equal(m.gemm_grouped(A, B, _offsets(sizes)), _product_64(A, B, sizes), torch.bfloat16)
    G = _ints((M, 24), gen, torch.bfloat16)
    _equal(m.gemm_grouped_wgrad(A, G, _offsets(sizes), torch.float32), _wgrad_64(A, G, sizes), torch.float32)
    sizes = [1] * 5 + [0] * 1000 + [290]
    A, B = _ints((295, 32), gen, torch.bfloat16), _ints((len(sizes), 32, 24), gen, torch.bfloat16)
    _equal(m.gemm_grouped(A, B, _offsets(sizes)), _product_64(A, B, sizes), torch.bfloat16)
    big = 2 ** 31 - 1
    for values, rows in (([-5, 3, 1 << 20], [(0, 3), (3, 20)]), ([big, big, big], [(20, 20), (20, 20)]),
                         ([-big, -1, 7], [(0, 0), (0, 7)]), ([10, 4, 9], [(10, 10), (4, 9)])):
        off = torch.tensor(values, dtype=torch.int32, device="cuda")
        A, B = _ints((20, 32), gen, torch.bfloat16), _ints((2, 32, 24), gen, torch.bfloat16)
        want = torch.full((20, 24), 9.0, dtype=torch.float64, device="cuda")
        for e, (lo, hi) in enumerate(rows):
            want[lo:hi] = A[lo:hi].double() @ B[e].double()
        D = m.gemm_grouped(A, B, off, out=torch.full((20, 24), 9.0, dtype=torch.bfloat16, device="cuda"))
        _equal(D, want, torch.bfloat16)
        G = _ints((20, 24), gen, torch.bfloat16)
        dB = m.gemm_grouped_wgrad(A, G, off, torch.float32)
        for e, (lo, hi) in enumerate(rows):
            _equal(dB[e], A[lo:hi].double().t() @ G[lo:hi].double(), torch.float32)
    assert m.device_status() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("sizes,N,K", [([100, 0, 300, 1], 200, 520), ([600, 601], 328, 2048), ([5], 64, 4096)],
                         ids=str)
def test_random_values(mpk_lib, cuda, dtype, sizes, N, K):
    import torch

    m = mpk_lib
    t = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(K)
    M, E = sum(sizes), len(sizes)
    A = torch.randn((M, K), generator=gen, device="cuda").to(t)
    B = torch.randn((E, K, N), generator=gen, device="cuda").to(t)
    off = _offsets(sizes)
    want, size = _product_64(A, B, sizes), _product_64(A.abs(), B.abs(), sizes)
    for out in ("float32", dtype):
        D = m.gemm_grouped(A, B, off, getattr(torch, out))
        bound = K * 2.0 ** -23 * size * (1 + HALF[out]) + HALF[out] * want.abs() + SUBNORMAL[out]
        over = int(((D.double() - want).abs() > bound).sum())
        assert over == 0
    G = torch.randn((M, N), generator=gen, device="cuda").to(t)
    want, size = _wgrad_64(A, G, sizes), _wgrad_64(A.abs(), G.abs(), sizes)
    for out in ("float32", dtype):
        dB = m.gemm_grouped_wgrad(A, G, off, getattr(torch, out))
        bound = max(sizes) * 2.0 ** -23 * size * (1 + HALF[out]) + HALF[out] * want.abs() + SUBNORMAL[out]
        over = int(((dB.double() - want).abs() > bound).sum())
        assert over == 0


@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("N,K", SHAPES)
def test_weight_gradient_is_exact(mpk_lib, cuda, sizes, N, K):
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(N * 13 + K + len(sizes))
    M = sum(sizes)
    for dtype, out, pad, shift in ((torch.bfloat16, torch.float32, 0, 0), (torch.float16, torch.float16, 8, 0),
                                   (torch.bfloat16, torch.bfloat16, 3, 1)):
        A, G = _ints((M, K), gen, dtype, pad, shift), _ints((M, N), gen, dtype, pad, shift)
        _equal(m.gemm_grouped_wgrad(A, G, _offsets(sizes), out), _wgrad_64(A, G, sizes), out)
    assert m.device_status() == 0


@pytest.mark.parametrize("first,sizes,behind", [(0, [5, 0, 130, 9], 40), (7, [300, 64, 3], 200), (2, [17, 31], 0)],
                         ids=str)
def test_weight_gradient_of_poisoned_neighbours(mpk_lib, cuda, first, sizes, behind):
    """NaN and infinity in the rows of other groups, and outside all, in either operand."""
    import torch

    m = mpk_lib
    K, N, E = 136, 72, len(sizes)
    gen = torch.Generator(device="cuda").manual_seed(first + 1)
    M = first + sum(sizes) + behind
    bounds = np.concatenate([[first], first + np.cumsum(sizes)])
    for clean in range(E):
        A, G = _ints((M, K), gen, torch.bfloat16), _ints((M, N), gen, torch.bfloat16)
        lo, hi = int(bounds[clean]), int(bounds[clean + 1])
        want = A[lo:hi].double().t() @ G[lo:hi].double()
        for t, v in ((A, float("nan")), (G, float("inf"))):
            t[:lo] = v
            t[hi:] = v
        _equal(m.gemm_grouped_wgrad(A, G, _offsets(sizes, first), torch.float32)[clean], want, torch.float32)


def test_results_with_strides_and_empty_operands(mpk_lib, cuda):
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(9)
    sizes = [40, 0, 25]
    A, G = _ints((65, 48), gen, torch.bfloat16), _ints((65, 40), gen, torch.bfloat16)
    off = _offsets(sizes)
    for extra in (1, 8, 24):
        whole = torch.full((3, 48, 40 + extra), 3.0, device="cuda")
        m.gemm_grouped_wgrad(A, G, off, out=whole[..., :40])
        _equal(whole[..., :40], _wgrad_64(A, G, sizes), torch.float32)
        assert bool((whole[..., 40:] == 3).all())
    # no rows at all: every gradient is zeros, and the product has nothing to do
    none = _offsets([0, 0])
    dB = m.gemm_grouped_wgrad(A[:0], G[:0], none, out=torch.ones((2, 48, 40), device="cuda"))
    assert bool((dB == 0).all())
    assert m.gemm_grouped(A[:0], _ints((2, 48, 8), gen, torch.bfloat16), none).shape == (0, 8)
    # nothing to sum over: the groups' rows become zeros
    D = torch.full((65, 16), 2.0, dtype=torch.bfloat16, device="cuda")
    m.gemm_grouped(A[:, :0], torch.empty((2, 0, 16), dtype=torch.bfloat16, device="cuda"), _offsets([10, 20]), out=D)
    assert bool((D[:30] == 0).all()) and bool((D[30:] == 2).all())
    assert m.gemm_grouped_wgrad(A, G, torch.zeros(1, dtype=torch.int32, device="cuda")).shape == (0, 48, 40)
    with pytest.raises(ValueError):
        m.gemm_grouped(A, _ints((3, 48, 8), gen, torch.float16), off)
    with pytest.raises(ValueError):
        m.gemm_grouped(A, _ints((3, 40, 8), gen, torch.bfloat16), off)
    with pytest.raises(ValueError):
        m.gemm_grouped(A, _ints((3, 48, 8), gen, torch.bfloat16), off.long())
    with pytest.raises(ValueError):
        m.gemm_grouped(A, _ints((4, 48, 8), gen, torch.bfloat16), off)
    with pytest.raises(ValueError):
        m.gemm_grouped_wgrad(A, G[:64], off)
    with pytest.raises(ValueError):
        m.gemm_grouped(A.float(), _ints((3, 48, 8), gen, torch.float32), off)


@pytest.mark.parametrize("sizes", [[1], [100, 0, 300, 1], [257, 255], [700, 5]], ids=str)
@pytest.mark.parametrize("N,K", [(64, 64), (256, 96), (100, 72), (33, 31), (520, 264)])
def test_mxfp8_matches_the_oracle(mpk_lib, cuda, sizes, N, K):
    """A's values are integers times a power of two per block, so the sums are exact, and D
    is the oracle's quantization of them, code for code and scale for scale."""
    import torch

    import oracle as O

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(N + K)
    rng = np.random.default_rng(N)
    M, E = sum(sizes), len(sizes)
    values = rng.integers(-8, 9, (M, K)).astype(np.float32) * np.exp2(rng.integers(-2, 3, (M, 1))).astype(np.float32)
    codes, scales = O.quantize(values)
    assert np.array_equal(O.dequantize(codes, scales), values)
    B = _ints((E, K, N), gen, torch.bfloat16, pad=8)
    off = _offsets(sizes)
    D, Ds = m.gemm_grouped_mxfp8(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), B, off)
    exact = _product_64(torch.from_numpy(values).cuda(), B, sizes).float().cpu().numpy()
    want, want_s = O.quantize(np.ascontiguousarray(exact))
    assert np.array_equal(Ds.cpu().numpy(), want_s)
    # the sums' zeros carry no sign to speak of
    got = D.cpu().numpy()
    assert np.all((got == want) | ((got & 0x7F == 0) & (want & 0x7F == 0)))
    # rows outside the groups stay as they were
    D2, Ds2 = torch.full_like(D, 0xEE), torch.full_like(Ds, 0xEE)
    m.gemm_grouped_mxfp8(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), B[:1],
                         _offsets([max(M // 2, 1)]), out=(D2, Ds2))
    assert bool((D2[max(M // 2, 1):] == 0xEE).all()) and bool((Ds2[max(M // 2, 1):] == 0xEE).all())
    assert m.device_status() == 0


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("sizes", [[1], [100, 0, 300, 1], [257, 255], [700, 5, 0]], ids=str)
@pytest.mark.parametrize("N,K", [(64, 64), (256, 130), (100, 515), (33, 31)])
def test_int8_groups(mpk_lib, cuda, sizes, N, K, layout):
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(N + K)
    M, E = sum(sizes), len(sizes)
    x = torch.randn((M, K), generator=gen, device="cuda").bfloat16()
    w = torch.randn((E, K, N), generator=gen, device="cuda")
    A, sa = m.quantize_int8(x)
    B, sb = m.quantize_int8_cols(w)
    stored = B
    if layout == "nk":
        stored = torch.zeros((E, N, K + (-K) % 16), dtype=torch.int8, device="cuda")[..., :K]
        stored.copy_(B.transpose(1, 2))
    out = torch.full((M + 3, N), 6.0, device="cuda")
    D = m.gemm_grouped_int8(A, sa, stored, sb, _offsets(sizes), b_layout=m.B_KN if layout == "kn" else m.B_NK,
                            out=out[:M])
    acc = _product_64(A, B, sizes)
    expert = torch.repeat_interleave(torch.arange(E, device="cuda"), torch.tensor(sizes, device="cuda"))
    assert torch.equal(D, acc.float() * sa[:, None] * sb[expert])
    assert bool((out[M:] == 6).all())
    # one group of all rows is the plain product
    assert torch.equal(m.gemm_grouped_int8(A, sa, B[:1], sb[:1], _offsets([M])), m.gemm_int8(A, sa, B[0], sb[0]))
    assert m.device_status() == 0


def test_offsets_past_32_bits(mpk_lib, cuda):
    """Weights and gradients of more than 2^31 elements (more than 2^32 bytes)."""
    import torch

    m = mpk_lib
    E, K, N = 9, 16384, 16384
    gen = torch.Generator(device="cuda").manual_seed(4)
    B = torch.zeros((E, K, N), dtype=torch.bfloat16, device="cuda")
    B[E - 1] = torch.randint(-2, 3, (K, N), generator=gen, device="cuda").bfloat16()
    sizes = [3] * (E - 1) + [40]
    A = _ints((sum(sizes), K), gen, torch.bfloat16, span=1)
    off = _offsets(sizes)
    D = m.gemm_grouped(A, B, off, torch.float32)
    assert bool((D[:24] == 0).all())
    assert torch.equal(D[24:], (A[24:].float() @ B[E - 1].float()))
    G = _ints((sum(sizes), N), gen, torch.bfloat16, span=1)
    m.gemm_grouped_wgrad(A, G, off, out=B)
    for e in (0, E - 2, E - 1):
        lo, hi = int(off[e]), int(off[e + 1])
        assert torch.equal(B[e], (A[lo:hi].float().t() @ G[lo:hi].float()).bfloat16())


def test_graphs_follow_new_offsets(mpk_lib, cuda):
    """A captured product and its gradients, replayed with other groups: nothing of the
    router's result was baked in.  Two graphs and eager calls run side by side."""
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(8)
    E, M, K, N = 4, 500, 104, 200
    A, G = _ints((M, K), gen, torch.bfloat16), _ints((M, N), gen, torch.bfloat16)
    B = _ints((E, K, N), gen, torch.bfloat16)
    odd = _ints((E, K, N), gen, torch.bfloat16, 1, 1)  # needs a workspace
    codes, scales = m.quantize(torch.randint(-4, 5, (M, K), generator=gen, device="cuda").float())
    offs = [_offsets([M, 0, 0, 0]), _offsets([M, 0, 0, 0])]

    def step(off):
        return (m.gemm_grouped(A, B, off), m.gemm_grouped(A, odd, off), m.gemm_grouped(G, B, off, b_layout=m.B_NK),
                m.gemm_grouped_wgrad(A, G, off, torch.float32), *m.gemm_grouped_mxfp8(codes, scales, B, off))

    step(offs[0])
    graphs = []
    for off in offs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphs_out = step(off)
        graphs.append((gr, graphs_out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for all_sizes in (([100, 200, 150, 50], [1, 0, 499, 0]), ([0, 0, 0, M], [125, 125, 125, 125])):
        for off, sizes in zip(offs, all_sizes):
            off.copy_(_offsets(sizes))
        torch.cuda.synchronize()
        for (gr, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        eager = [step(off) for off in offs]
        torch.cuda.synchronize()
        for (_, outs), mine, sizes in zip(graphs, eager, all_sizes):
            for a, b in zip(outs, mine):
                assert torch.equal(a, b)
            _equal(outs[0], _product_64(A, B, sizes), torch.bfloat16)
            _equal(outs[3], _wgrad_64(A, G, sizes), torch.float32)
    assert m.device_status() == 0


def test_repeated_calls_give_the_same_bits(mpk_lib, cuda):
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(6)
    A = torch.randn((777, 1000), generator=gen, device="cuda").bfloat16()
    B = torch.randn((5, 1000, 304), generator=gen, device="cuda").bfloat16()
    G = torch.randn((777, 304), generator=gen, device="cuda").bfloat16()
    for sizes in ([100, 0, 300, 377, 0], [777, 0, 0, 0, 0], [1, 2, 3, 4, 5]):
        off = _offsets(sizes)
        n = sum(sizes)
        first = m.gemm_grouped(A, B, off, torch.float32)[:n], m.gemm_grouped_wgrad(A, G, off, torch.float32)
        for _ in range(5):
            assert torch.equal(first[0], m.gemm_grouped(A, B, off, torch.float32)[:n])
            assert torch.equal(first[1], m.gemm_grouped_wgrad(A, G, off, torch.float32))


def _experts(m, x, w1, w2, off):
    """A mixture-of-experts feed-forward block with squared-ReLU, in BF16 and FP32 sums."""
    h = m.gemm_grouped(x, w1, off)
    a = h.float().relu().square().to(h.dtype)
    return h, a, m.gemm_grouped(a, w2, off)


def test_experts_forward_and_backward_together(mpk_lib, cuda):
    """A step through two grouped products and back, against 64-bit autograd on the same
    inputs, and the weights' gradients against differences of the loss."""
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(11)
    M, E, K, H = 300, 5, 96, 160
    sizes = [90, 0, 150, 1, 59]
    off = _offsets(sizes)
    x = torch.randn((M, K), generator=gen, device="cuda").bfloat16()
    w1 = (torch.randn((E, K, H), generator=gen, device="cuda") / K ** 0.5).bfloat16()
    w2 = (torch.randn((E, H, K), generator=gen, device="cuda") / H ** 0.5).bfloat16()
    dy = torch.randn((M, K), generator=gen, device="cuda").bfloat16()

    h, a, y = _experts(m, x, w1, w2, off)
    da = m.gemm_grouped(dy, w2, off, b_layout=m.B_NK)
    dw2 = m.gemm_grouped_wgrad(a, dy, off, torch.float32)
    dh = (da.float() * 2 * h.float().relu()).bfloat16()
    dx = m.gemm_grouped(dh, w1, off, b_layout=m.B_NK)
    dw1 = m.gemm_grouped_wgrad(x, dh, off, torch.float32)

    X, W1, W2 = (t.double().requires_grad_() for t in (x, w1, w2))

    def forward(w1_, w2_):
        rows, lo = [], 0
        for e, n in enumerate(sizes):
            hh = X[lo:lo + n] @ w1_[e]
            rows.append(hh.relu().square() @ w2_[e])
            lo += n
        return torch.cat(rows)

    Y = forward(W1, W2)
    loss = (Y * dy.double()).sum()
    loss.backward()
    # Each chain passes at most four roundings to BF16 (2^-8 each) on the way, entering sums of
    # terms of either sign: relative to the norm, independent roundings add in squares, and
    # squaring doubles one of them.  4 * 2 * 2^-8 = 2^-5 bounds the norm of the difference.
    for got, want in ((y, Y), (dx, X.grad), (dw1, W1.grad), (dw2, W2.grad)):
        off_by = float((got.double() - want.detach()).norm() / want.detach().norm())
        assert off_by <= 2.0 ** -5, off_by
    assert bool((dw1[1] == 0).all()) and bool((dw2[1] == 0).all())
    # differences of the 64-bit loss along random directions: its second derivative is bounded,
    # the central difference's error falls with step^2
    for grad, which in ((dw1, 0), (dw2, 1)):
        u = torch.randn(grad.shape, generator=gen, device="cuda").double()
        u = u * grad.double().sign()  # so that the slope is not a difference of large terms
        u = u.abs() * grad.double().sign()
        step = 1e-5
        with torch.no_grad():
            plus = forward(W1 + step * u, W2) if which == 0 else forward(W1, W2 + step * u)
            minus = forward(W1 - step * u, W2) if which == 0 else forward(W1, W2 - step * u)
            slope = float(((plus - minus) * dy.double()).sum() / (2 * step))
        mine = float((grad.double() * u).sum())
        assert abs(mine - slope) <= 2.0 ** -5 * abs(slope)

    # the same experts served in int8 and in the framework's MXFP8: as near as their codes allow
    q1, s1 = m.quantize_int8_cols(w1)
    q2, s2 = m.quantize_int8_cols(w2)
    xq, xs = m.quantize_int8(x)
    h8 = m.gemm_grouped_int8(xq, xs, q1, s1, off)
    aq, as_ = m.quantize_int8(h8.float().relu().square())
    y8 = m.gemm_grouped_int8(aq, as_, q2, s2, off)
    # a code's error is at most 1/254 of the row's largest value; eight times the rms of normal
    # rows bounds that value, so each of the four quantizations is within 8/254 of the norm, and
    # squaring doubles the first two
    assert float((y8.double() - Y.detach()).norm() / Y.detach().norm()) <= 6 * 8 / 254
    d, s = m.quantize(x.float())
    hd, hs = m.gemm_grouped_mxfp8(d, s, w1, off)
    # E4M3 with power-of-two block scales: 2^-4 of each value, for A and again for D
    H64 = torch.cat([x[lo:lo + n].double() @ w1[e].double()
                     for e, (lo, n) in enumerate(zip(np.concatenate([[0], np.cumsum(sizes)]).tolist(), sizes))])
    assert float((m.dequantize(hd, hs).double() - H64).norm() / H64.norm()) <= 2 * 2.0 ** -4


@pytest.mark.parametrize("sizes", [[3000], [1000, 0, 3, 2500], [2048, 64, 17, 1], [4097]], ids=str)
@pytest.mark.parametrize("N,K", [(64, 72), (200, 371), (256, 256)])
def test_long_groups_with_small_weights(mpk_lib, cuda, sizes, N, K):
    """Few tiles and a long ragged reduction: it is shared by a cluster, of which short and
    empty groups leave some blocks nothing."""
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(N + len(sizes))
    M = sum(sizes) + 5
    for dtype, out in ((torch.bfloat16, torch.float32), (torch.float16, torch.float16)):
        A, G = _ints((M, K), gen, dtype, 8, span=1), _ints((M, N), gen, dtype, 8, span=1)
        A[M - 5:] = float("nan")
        G[M - 5:] = float("nan")
        _equal(m.gemm_grouped_wgrad(A, G, _offsets(sizes), out), _wgrad_64(A, G, sizes), out)
    assert m.device_status() == 0


def test_operands_written_just_before(mpk_lib, cuda):
    """Back to back on one stream, without a pause: weights, codes, offsets and activations
    are rewritten between the calls that read them, by the library's own kernels and by
    others, and results are overwritten at once.  Every call sees its own operands."""
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(21)
    E, M, K, N = 3, 64, 512, 1024
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    w = torch.empty((E, K, N), dtype=torch.bfloat16, device="cuda")
    x = torch.empty((M, K), dtype=torch.bfloat16, device="cuda")
    d = torch.empty((M, N), dtype=torch.float32, device="cuda")
    q = torch.empty((M, N), dtype=torch.float32, device="cuda")
    dw = torch.empty((E, K, N), dtype=torch.float32, device="cuda")
    rounds = 12
    ws = [torch.randint(-2, 3, (E, K, N), generator=gen, device="cuda").bfloat16() for _ in range(rounds)]
    xs = [torch.randint(-2, 3, (M, K), generator=gen, device="cuda").bfloat16() for _ in range(rounds)]
    splits = [[0, 10 + i, 30 + i, M] for i in range(rounds)]
    offs = [torch.tensor(s, dtype=torch.int32, device="cuda") for s in splits]
    got = []
    torch.cuda.synchronize()
    for i in range(rounds):
        off.copy_(offs[i])
        w.copy_(ws[i])
        x.copy_(xs[i])
        m.gemm_grouped(x, w, off, out=d)
        codes, scales = m.quantize_int8_cols(w[0])
        m.linear_int8(x, codes, scales, out=q)
        m.gemm_grouped_wgrad(x, d.bfloat16(), off, out=dw)
        got.append((d.clone(), q.clone(), dw.clone()))
    torch.cuda.synchronize()
    for i in range(rounds):
        sizes = np.diff(splits[i]).tolist()
        _equal(got[i][0], _product_64(xs[i], ws[i], sizes), torch.float32)
        c, s = m.quantize_int8_cols(ws[i][0])
        torch.cuda.synchronize()
        assert torch.equal(got[i][1], m.linear_int8(xs[i], c, s, out_dtype=torch.float32))
        torch.cuda.synchronize()
        bound = M * 2.0 ** -23 * _wgrad_64(xs[i].abs(), got[i][0].bfloat16().abs(), sizes)
        diff = (got[i][2].double() - _wgrad_64(xs[i], got[i][0].bfloat16(), sizes)).abs()
        assert int((diff > bound).sum()) == 0


@pytest.mark.parametrize("M,E,K", [(1, 64, 4096), (40, 3, 2048), (300, 16, 512)])
def test_overlapping_groups_stay_inside(mpk_lib, cuda, M, E, K):
    """Offsets that run back and forth, so that groups overlap and there are more tiles than
    disjoint groups could have: nothing outside the groups is written and no wait gives up."""
    import torch

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(M)
    rows = 8 + M
    off = torch.tensor([0 if e % 2 == 0 else M for e in range(E + 1)], dtype=torch.int32, device="cuda")
    A, B = _ints((rows, K), gen, torch.bfloat16, span=1), _ints((E, K, 128), gen, torch.bfloat16, span=1)
    whole = torch.full((rows, 160), 4.0, dtype=torch.bfloat16, device="cuda")
    m.gemm_grouped(A, B, off, out=whole[:, :128])
    assert bool((whole[M:] == 4).all()) and bool((whole[:, 128:] == 4).all())
    dB = m.gemm_grouped_wgrad(A, A[:, :128], off, torch.float32)
    want = A[:M].double().t() @ A[:M, :128].double()
    _equal(dB[0], want, torch.float32)
    assert m.device_status() == 0


@pytest.mark.parametrize("K", [1, 7, 16, 33, 100, 515, 4099])
def test_operands_at_every_address(mpk_lib, cuda, K):
    """Bases and rows of A and B at all 16 places within 16 bytes, NaN all around 16-bit ones."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(K)
    M, N, E = 21, 40, 2
    off = torch.tensor([0, 9, M], dtype=torch.int32, device="cuda")

    def at(values, shift, fill):
        shape, pad = values.shape, 1 + shift % 3
        flat = torch.full((values.numel() // K * (K + pad) + 32,), fill, dtype=values.dtype, device="cuda")
        view = flat[shift:shift + values.numel() // K * (K + pad)].view(*shape[:-1], K + pad)[..., :K]
        view.copy_(values)
        return view

    a = torch.randint(-4, 5, (M, K), generator=gen, device="cuda")
    b = torch.randint(-4, 5, (E, N, K), generator=gen, device="cuda")
    want = torch.cat([a[:9].double() @ b[0].double().t(), a[9:].double() @ b[1].double().t()])
    one, ones = torch.ones(M, device="cuda"), torch.ones((E, N), device="cuda")
    for shift in range(16):
        # sums of at most 16 * 4099 < 2^24 are exact in FP32
        got = mpk_lib.gemm_grouped_int8(at(a.to(torch.int8), shift, 77), one, at(b.to(torch.int8), 15 - shift, 77),
                                        ones, off, out_dtype=torch.float32, b_layout=mpk_lib.B_NK)
        assert torch.equal(got.double(), want)
        nan = float("nan")
        got = mpk_lib.gemm_grouped(at(a.bfloat16(), shift % 8, nan), at(b.bfloat16(), (shift + 3) % 8, nan), off,
                                   out_dtype=torch.float32, b_layout=mpk_lib.B_NK)
        assert torch.equal(got.double(), want)


@pytest.mark.parametrize("M,K,N", [(4000000, 64, 64), (1000000, 2048, 2048)], ids=["cluster", "pairs"])
def test_a_wait_that_runs_out_is_reported(mpk_lib, cuda, M, K, N):
    """Reductions of milliseconds under a wait budget of a microsecond: the epilogue's waits give
    up (a wait parks for up to a millisecond per test, and tests twice), in a cluster that
    shares one tile's reduction and in pairs with a tile each.  The call returns, nothing of D is
    written, the status word says so, and the next call with the usual budget is right."""
    import torch

    m = mpk_lib
    A = torch.ones((M, K), dtype=torch.bfloat16, device="cuda")
    G = torch.ones((M, N), dtype=torch.bfloat16, device="cuda")
    G[M // 2:] = -1.0
    off = _offsets([M])
    dB = torch.full((1, K, N), 7.0, device="cuda")
    torch.cuda.synchronize()
    m.set_wait_timeout_ns(1000)
    try:
        m.gemm_grouped_wgrad(A, G, off, out=dB)
        torch.cuda.synchronize()
    finally:
        m.set_wait_timeout_ns(2_000_000_000)
    assert m.device_status() == 0x124
    assert bool((dB == 7).all())
    m.gemm_grouped_wgrad(A, G, off, out=dB)
    assert m.device_status() == 0
    # M / 2 ones and M / 2 minus ones: whole numbers below 2^24
    assert bool((dB == 0).all())


# Groups whose tiles are shared by pairs of CTAs (more than 48 rows per group, enough tiles),
# with more tiles than pairs and, in the longest group, more than one panel of row tiles.
MANY = [4500, 3, 700]


@pytest.mark.parametrize("poisoned", [None, 0, 1, 2])
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("N,K", [(1304, 200), (1003, 131)])
def test_many_tiles_are_exact(mpk_lib, cuda, dtype, layout, poisoned, N, K):
    """The kernels of long batches, with a group whose rows and weights are not finite beside
    groups that must not see them, and rows in front of and behind all groups."""
    import torch

    m = mpk_lib
    t = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(N)
    first, behind = 5, 9
    M, E = first + sum(MANY) + behind, len(MANY)
    for out, pad in ((t, 8), (torch.float32, 3)):
        A = _ints((M, K), gen, t, pad)
        B = _ints((E, K, N) if layout == "kn" else (E, N, K), gen, t, pad)
        A[:first], A[M - behind:] = float("inf"), float("nan")
        if poisoned is not None:
            lo = first + sum(MANY[:poisoned])
            A[lo:lo + MANY[poisoned]] = float("nan")
            B[poisoned] = float("inf")
        whole = torch.full((M, N + 8), 5.0, dtype=out, device="cuda")
        D = m.gemm_grouped(A, B, _offsets(MANY, first), b_layout=m.B_KN if layout == "kn" else m.B_NK,
                           out=whole[:, :N])
        want = _product_64(A, B if layout == "kn" else B.transpose(1, 2), MANY, first)
        want[:first] = 5.0
        want[M - behind:] = 5.0
        _equal(D, want, out)
        assert bool((whole[:, N:] == 5).all())
    assert m.device_status() == 0


def _mx_values(rng, M, K):
    """FP32 values that MXFP8 holds exactly: integers times a power of two per row."""
    return rng.integers(-8, 9, (M, K)).astype(np.float32) * np.exp2(rng.integers(-2, 3, (M, 1))).astype(np.float32)


def _check_mxfp8(D, Ds, exact64, rows):
    """Codes and scales of `rows` against the oracle's quantization of the exact sums."""
    import oracle as O

    want, want_s = O.quantize(np.ascontiguousarray(exact64.float().cpu().numpy()[rows]))
    got, got_s = D.cpu().numpy()[rows], Ds.cpu().numpy()[rows]
    assert np.array_equal(got_s, want_s)
    bad = (got != want) & ~((got & 0x7F == 0) & (want & 0x7F == 0))  # zeros carry no sign to speak of
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist())


@pytest.mark.parametrize("sizes,K", [(MANY, 256), (MANY, 200), ([40], 2048), ([33, 0, 7], 2048), ([1], 4096),
                                     ([300], 1024)], ids=str)
@pytest.mark.parametrize("N", [1304, 1280, 77, 256])
def test_mxfp8_of_every_kernel_with_nan_and_infinity(mpk_lib, cuda, sizes, K, N):
    """Tiles of pairs, of single CTAs and of clusters that share a reduction make the same codes
    and scales: NaN does not enter a block's largest magnitude and becomes the code 0x7F; an
    infinity gives its block the scale 255, whose inverse is 0.  Both in rows of A (every
    value of those rows of D) and in single weights (a column of D, beside finite ones)."""
    import torch

    import oracle as O

    m = mpk_lib
    rng = np.random.default_rng(K + N + len(sizes))
    gen = torch.Generator(device="cuda").manual_seed(K + N)
    M, E = sum(sizes), len(sizes)
    values = _mx_values(rng, M, K)
    codes, scales = O.quantize(values)
    codes[M // 3, K // 2] = 0x7F  # NaN
    scales[M // 2, K // 64] = 255  # 0 * inf and x * inf
    values = O.dequantize(codes, scales)
    B = _ints((E, K, N), gen, torch.bfloat16, pad=8)
    B[0, K // 3, 5], B[0, 1, 40], B[0, 2, 41] = float("inf"), float("nan"), float("-inf")
    D, Ds = m.gemm_grouped_mxfp8(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), B, _offsets(sizes))
    _check_mxfp8(D, Ds, _product_64(torch.from_numpy(values).cuda(), B, sizes), slice(0, M))
    assert m.device_status() == 0


@pytest.mark.parametrize("shift", range(8))
@pytest.mark.parametrize("K", [64, 96, 200, 33])
def test_mxfp8_codes_at_every_address(mpk_lib, cuda, K, shift):
    """Codes and scales anywhere, with the bytes around them holding NaN: whole blocks take the
    codec's pre-pass where they are aligned and the product's own unpacking elsewhere.  Scale
    bytes 0 (the value 0) and 255 (infinity) and NaN codes among them."""
    import torch

    import oracle as O

    m = mpk_lib
    rng = np.random.default_rng(K + shift)
    gen = torch.Generator(device="cuda").manual_seed(K)
    sizes = [9, 0, 50]
    M, N = sum(sizes), 72
    values = _mx_values(rng, M, K)
    codes, scales = O.quantize(values)
    codes[4, K - 1], codes[20, 0] = 0x7F, 0xFF
    scales[7, :], scales[30, -1] = 0, 255
    values = O.dequantize(codes, scales)

    def at(x):
        flat = torch.full((x.size + 16,), 0xFF, dtype=torch.uint8, device="cuda")
        view = flat[shift:shift + x.size].view(x.shape)
        view.copy_(torch.from_numpy(x))
        return view

    B = _ints((3, K, N), gen, torch.bfloat16, pad=8)
    D, Ds = m.gemm_grouped_mxfp8(at(codes), at(scales), B, _offsets(sizes))
    _check_mxfp8(D, Ds, _product_64(torch.from_numpy(values).cuda(), B, sizes), slice(0, M))
    assert m.device_status() == 0


@pytest.mark.parametrize("K", [512, 500])
def test_mxfp8_operands_written_just_before(mpk_lib, cuda, K):
    """The grouped MXFP8 product reads its offsets and loads weights while its own unpacking kernel
    runs.  Back to back on one stream: offsets, weights, codes and scales rewritten just in
    front of it, then weights that the gradient's kernel (which lets its successor start early)
    has just written; the codec's pre-pass (K = 512) and the product's unpacking (K = 500)."""
    import torch

    import oracle as O

    m = mpk_lib
    gen = torch.Generator(device="cuda").manual_seed(K)
    rng = np.random.default_rng(K)
    E, M, N, rounds = 3, 600, 1024, 10
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    w = torch.empty((E, K, N), dtype=torch.bfloat16, device="cuda")
    codes = torch.empty((M, K), dtype=torch.uint8, device="cuda")
    scales = torch.empty((M, m.nblk(K)), dtype=torch.uint8, device="cuda")
    values = [_mx_values(rng, M, K) for _ in range(rounds)]
    quantized = [[torch.from_numpy(t).cuda() for t in O.quantize(v)] for v in values]
    ws = [_ints((E, K, N), gen, torch.bfloat16) for _ in range(rounds)]
    xs = [_ints((M, K), gen, torch.bfloat16, span=1) for _ in range(rounds)]
    gs = [_ints((M, N), gen, torch.bfloat16, span=1) for _ in range(rounds)]
    splits = [[0, 60 + 11 * i, 300 + 7 * i, M] for i in range(rounds)]
    offs = [torch.tensor(s, dtype=torch.int32, device="cuda") for s in splits]
    first = [(torch.empty((M, N), dtype=torch.uint8, device="cuda"),
              torch.empty((M, m.nblk(N)), dtype=torch.uint8, device="cuda")) for _ in range(rounds)]
    second = [tuple(torch.empty_like(t) for t in pair) for pair in first]
    w_grad = []
    torch.cuda.synchronize()
    for i in range(rounds):
        codes.copy_(quantized[i][0])
        scales.copy_(quantized[i][1])
        w.copy_(ws[i])
        off.copy_(offs[i])
        m.gemm_grouped_mxfp8(codes, scales, w, off, out=first[i])
        m.gemm_grouped_wgrad(xs[i], gs[i], off, out=w)
        m.gemm_grouped_mxfp8(codes, scales, w, off, out=second[i])
        w_grad.append(w.clone())
    torch.cuda.synchronize()
    for i in range(rounds):
        sizes = np.diff(splits[i]).tolist()
        v = torch.from_numpy(values[i]).cuda()
        _check_mxfp8(*first[i], _product_64(v, ws[i], sizes), slice(0, M))
        _equal(w_grad[i], _wgrad_64(xs[i], gs[i], sizes), torch.bfloat16)
        # |w| <= 390 and 512 terms of at most 32 * 390 in steps of 1/4: exact in FP32
        _check_mxfp8(*second[i], _product_64(v, w_grad[i], sizes), slice(0, M))
    assert m.device_status() == 0
