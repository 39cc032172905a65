"""GPU: quantisation to MXFP4 and back, and products of MXFP4 matrices, against their definition in 64 bits (mx_ref.py,
where the tolerances are derived)."""
import math

import numpy as np
import pytest
import torch

import mx_ref as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def check_quantize(gpu, x):
    m = gpu.mxfp4_quantize(x)
    torch.cuda.synchronize()
    code, scales = ref.quantize(x)
    assert m.shape == tuple(x.shape)
    assert torch.equal(m.scales.cpu(), scales)
    assert torch.equal(ref.unpack(m.packed), code)
    return m


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows, K", [(1, 32), (1, 2880), (3, 64), (7, 96), (64, 160), (65, 1024), (130, 4096), (1000, 224),
                                     (2, 40000)])
def test_quantize(gpu, rows, K, dtype):
    x = torch.randn((rows, K), device="cuda", generator=gen_of(rows + K))
    x *= torch.exp2(torch.randint(-20, 20, (rows, K // 32, 1), device="cuda", generator=gen_of(K))).expand(-1, -1, 32).flatten(1)
    check_quantize(gpu, x.to(dtype))


def test_quantize_every_bf16(gpu):
    """All 65536 patterns, with neighbours of their size and with ones of any size."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).cuda()
    mixed = bits[torch.randperm(65536, device="cuda", generator=gen_of(1))]
    for b in (bits, mixed):
        check_quantize(gpu, b.view(BF16).view(-1, 64))


def test_quantize_float_patterns(gpu):
    bits = torch.randint(-2 ** 31, 2 ** 31, (512, 96), device="cuda", generator=gen_of(2)).to(torch.int32)
    check_quantize(gpu, bits.view(F32))  # every exponent, some blocks with NaN
    small = bits & 0x81ffffff  # below 2^-123: where the scale ends, and denormal numbers
    check_quantize(gpu, small.view(F32))
    check_quantize(gpu, (bits & -2147483648 | (bits & 0x7fffff)).to(torch.int32).view(F32))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantize_borders(gpu, dtype):
    """Half way between neighbours, next to it, and powers of two next to each other."""
    mids = torch.tensor([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.9375], device="cuda")
    for e in (-126, -60, 0, 1, 60, 124):
        v = torch.cat((mids, -mids, mids.new_zeros(30)))
        up = torch.nextafter(v.to(dtype), torch.full_like(v, 100).to(dtype)).float()
        down = torch.nextafter(v.to(dtype), torch.full_like(v, -100).to(dtype)).float()
        x = torch.stack((v, up, down)).double()
        x[:, 0] = 7.9375  # the block's largest: its scale is 1
        x[:, 32] = -4
        check_quantize(gpu, torch.ldexp(x, torch.tensor(e, device="cuda")).to(dtype))


def test_quantize_rows_that_are_apart(gpu):
    wide = torch.randn((40, 512), device="cuda", generator=gen_of(3))
    for x in (wide[:, 64:320], wide[::3, 4:100], wide.to(BF16)[:, 8:200], wide.to(BF16)[1::2], wide[7:8, 32:64]):
        m = check_quantize(gpu, x)
        out = gpu.MXFP4Matrix(torch.zeros_like(m.packed), torch.zeros_like(m.scales))
        assert gpu.mxfp4_quantize(x, out=out) is out
        assert torch.equal(out.packed, m.packed) and torch.equal(out.scales, m.scales)
    for bad in (wide[:, 1:33], wide.to(BF16)[:, 4:36]):
        with pytest.raises(ValueError, match="aligned"):
            gpu.mxfp4_quantize(bad)
    assert gpu.mxfp4_quantize(wide[:0]).shape == (0, 512)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows, K", [(1, 32), (5, 2880), (256, 32), (33, 192), (700, 1024)])
def test_dequantize(gpu, rows, K, dtype):
    m = ref.random_matrix(gpu, gen_of(rows), rows, K, low=0, high=256)
    want = ref.of_matrix(m)
    # past the types' range: infinities; bf16 ends at 2^-133
    want = want.to(dtype).double()
    got = gpu.mxfp4_dequantize(m, dtype=dtype)
    assert got.dtype == dtype and torch.equal(got.cpu().double().nan_to_num(-7.25), want.nan_to_num(-7.25))
    wide = torch.full((rows, K + 64), 3.0, device="cuda", dtype=dtype)
    assert gpu.mxfp4_dequantize(m, out=wide[:, 32:K + 32]).data_ptr() == wide[:, 32:].data_ptr()
    assert torch.equal(wide[:, 32:K + 32].cpu().double().nan_to_num(-7.25), want.nan_to_num(-7.25))
    assert bool((wide[:, :32] == 3).all()) and bool((wide[:, K + 32:] == 3).all())


def test_dequantize_a_stack(gpu):
    m = ref.random_matrix(gpu, gen_of(4), 3, 5, 64)
    got = gpu.mxfp4_dequantize(m)
    assert got.shape == (3, 5, 64) and torch.equal(got.cpu().double(), ref.of_matrix(m))
    assert gpu.mxfp4_dequantize(ref.random_matrix(gpu, gen_of(4), 0, 64)).shape == (0, 64)


def test_quantised_weights_are_the_layers_format(gpu):
    """What mxfp4_quantize makes is what pack_tiled takes."""
    x = torch.randn((128, 320), device="cuda", generator=gen_of(5))
    m = gpu.mxfp4_quantize(x)
    nib, sc = gpu.pack_tiled(m.packed, m.scales, 128, 320)
    assert torch.equal(gpu.dequant(nib, sc, 128, 320), gpu.mxfp4_dequantize(m))


def test_offsets_past_32_bits(gpu):
    """2^32 + values: the last rows are in their places."""
    rows, K = 65537, 65568
    x = torch.zeros((rows, K), dtype=BF16, device="cuda")
    x[-3:] = torch.randn((3, K), device="cuda", generator=gen_of(6)).to(BF16)
    x[1] = x[-1]
    m = gpu.mxfp4_quantize(x)
    last = gpu.mxfp4_quantize(x[-3:])
    assert torch.equal(m.packed[-3:], last.packed) and torch.equal(m.scales[-3:], last.scales)
    assert torch.equal(m.packed[1], last.packed[-1]) and not m.packed[2:-3].any()
    x.fill_(1)
    gpu.mxfp4_dequantize(m, out=x)
    assert torch.equal(x[-3:], gpu.mxfp4_dequantize(last)) and torch.equal(x[1], x[-1]) and not x[2:-3].any()


# -- products -----------------------------------------------------------------
SHAPES = [(1, 1, 32), (1, 64, 32), (2, 63, 96), (1, 5120, 2880), (8, 200, 2880), (17, 1024, 512), (31, 65, 64), (32, 64, 160),
          (33, 127, 2880), (64, 320, 4096), (100, 1001, 2016), (129, 257, 1056), (300, 513, 4096), (257, 640, 8192),
          (513, 258, 32), (1025, 770, 224)]


def operands(gpu, M, N, K, seed=0, **kw):
    a, w = ref.random_matrix(gpu, gen_of(seed), M, K, **kw), ref.random_matrix(gpu, gen_of(seed + 1), N, K, **kw)
    bias = (20 * torch.randn(N, device="cuda", generator=gen_of(seed + 2))).to(BF16)
    return a, w, bias


@pytest.mark.parametrize("M, N, K", SHAPES)
def test_product(gpu, M, N, K):
    a, w, bias = operands(gpu, M, N, K, M + N)
    for b in (None, bias):
        want, tol = ref.product(ref.of_matrix(a), ref.of_matrix(w), b)
        for dtype in (BF16, F32):
            got = gpu.mxfp4_matmul(a, w, bias=b, dtype=dtype)
            assert got.dtype == dtype
            ref.assert_values(got, want, tol, (M, N, K, b is not None, dtype))


@pytest.mark.parametrize("M, N, K", SHAPES)
def test_product_quantized(gpu, M, N, K):
    N = (N + 31) // 32 * 32
    a, w, bias = operands(gpu, M, N, K, M + N)
    want, tol = ref.product(ref.of_matrix(a), ref.of_matrix(w), bias)
    got = gpu.mxfp4_matmul(a, w, bias=bias, quantize=True)
    assert got.shape == (M, N)
    ref.assert_quantized(got, want, tol)


@pytest.mark.parametrize("M, N, K", SHAPES)
@pytest.mark.parametrize("with_bias", [False, True])
def test_product_swiglu(gpu, M, N, K, with_bias):
    N = (N + 63) // 64 * 64
    a, w, bias = operands(gpu, M, N, K, M + N, low=119, high=124)
    bias = bias / 8 if with_bias else None
    y, tol = ref.product(ref.of_matrix(a), ref.of_matrix(w), bias)
    want, tol = ref.swiglu(y, tol)
    ref.assert_quantized(gpu.mxfp4_matmul(a, w, bias=bias, swiglu=True, quantize=True), want, tol)
    for dtype in (BF16, F32):
        ref.assert_values(gpu.mxfp4_matmul(a, w, bias=bias, swiglu=True, dtype=dtype), want, tol, (M, N, K))


def test_product_refusals(gpu):
    a, w, _ = operands(gpu, 3, 64, 64)
    for kw, text in ((dict(alpha=1e300), "alpha"), (dict(alpha=math.inf), "alpha"), (dict(alpha=math.nan), "alpha"),
                     (dict(alpha="1"), "alpha"), (dict(limit=-1.0), "limit"), (dict(limit=-1e300), "limit"),
                     (dict(limit=math.nan), "limit"), (dict(dtype=torch.float16), "dtype"),
                     (dict(out=torch.empty((3, 33), device="cuda")), "shape"),
                     (dict(out=torch.empty((3, 32), device="cuda", dtype=torch.float16)), "dtype")):
        for quantize in (False, True):
            if not quantize or "dtype" not in kw and "out" not in kw:
                with pytest.raises(ValueError, match=text):
                    gpu.mxfp4_matmul(a, w, swiglu=True, quantize=quantize, **kw)
    with pytest.raises(ValueError, match="K="):
        gpu.mxfp4_matmul(a, operands(gpu, 3, 64, 96)[1])


@pytest.mark.parametrize("M, N, K", [(1, 96, 4096), (5, 2880, 4128), (17, 130, 4640), (40, 992, 512), (1100, 1920, 64),
                                     (1031, 1985, 288), (2950, 2944, 96), (2817, 2946, 320)])
def test_product_of_many_tiles(gpu, M, N, K):
    """Long rows that several waves share, and calls with tiles enough for the larger ones."""
    a, w, bias = operands(gpu, M, N, K, M + N, low=119, high=124)
    want, tol = ref.product(ref.of_matrix(a), ref.of_matrix(w), bias)
    for dtype in (BF16, F32):
        ref.assert_values(gpu.mxfp4_matmul(a, w, bias=bias, dtype=dtype), want, tol)
    if N % 32 == 0:
        ref.assert_quantized(gpu.mxfp4_matmul(a, w, bias=bias, quantize=True), want, tol)
    if N % 2 == 0:
        want, tol = ref.swiglu(want, tol)
        ref.assert_values(gpu.mxfp4_matmul(a, w, bias=bias, swiglu=True), want, tol)
        if N % 64 == 0:
            ref.assert_quantized(gpu.mxfp4_matmul(a, w, bias=bias, swiglu=True, quantize=True), want, tol)


@pytest.mark.parametrize("M, N", [(5, 6), (40, 2), (200, 130), (70, 1002)])
def test_product_swiglu_of_few_columns(gpu, M, N):
    a, w, bias = operands(gpu, M, N, 96, M, low=119, high=124)
    y, tol = ref.product(ref.of_matrix(a), ref.of_matrix(w), bias)
    for alpha, limit in ((1.702, 7.0), (1.0, math.inf), (0.0, 0.0), (-2.0, 3.0)):
        want, off = ref.swiglu(y, tol, alpha, limit)
        # alpha scales the slope's second part: |g sigmoid'(alpha g) alpha| is at most max(1.1, |alpha| |g| / 4)
        off = off + (y[:, 1::2].clamp(-limit, limit) + 1).abs() * tol[:, ::2] * (1 + (alpha * y[:, ::2]).abs())
        ref.assert_values(gpu.mxfp4_matmul(a, w, bias=bias, swiglu=True, alpha=alpha, limit=limit, dtype=F32), want, off)


@pytest.mark.parametrize("M, N, K", [(3, 70, 96), (40, 129, 320), (300, 300, 1024)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_product_into_a_part_of_a_buffer(gpu, M, N, K, dtype):
    """Rows any distance apart, on no more than their element's alignment; what lies around stays."""
    a, w, bias = operands(gpu, M, N, K)
    want, tol = ref.product(ref.of_matrix(a), ref.of_matrix(w), bias)
    for before, after in ((0, 0), (1, 0), (3, 5), (8, 8), (4, 64)):
        wide = torch.full((M + 2, before + N + after), 7.0, device="cuda", dtype=dtype)
        out = wide[1:-1, before:before + N]
        assert gpu.mxfp4_matmul(a, w, bias=bias, out=out) is out
        ref.assert_values(out, want, tol)
        assert bool((wide[0] == 7).all()) and bool((wide[-1] == 7).all())
        assert bool((wide[:, :before] == 7).all()) and bool((wide[:, before + N:] == 7).all())


@pytest.mark.parametrize("M, N, K", [(3, 70, 96), (70, 129, 320), (300, 300, 1024)])
def test_product_of_scales_of_any_size(gpu, M, N, K):
    """Sums of blocks whose scales differ by 2^40; scales at both ends of their range."""
    a, w, _ = operands(gpu, M, N, K, 3, low=107, high=148)
    want, tol = ref.product(ref.of_matrix(a), ref.of_matrix(w))
    ref.assert_values(gpu.mxfp4_matmul(a, w, dtype=F32), want, tol)
    a, w, _ = operands(gpu, M, N, K, 4, low=0, high=4)
    w = gpu.MXFP4Matrix(w.packed, 248 + w.scales)
    want, tol = ref.product(ref.of_matrix(a), ref.of_matrix(w))
    ref.assert_values(gpu.mxfp4_matmul(a, w, dtype=F32), want, tol)
    ref.assert_values(gpu.mxfp4_matmul(w, a, dtype=F32), want.T, tol.T)


@pytest.mark.parametrize("M, N, K", [(3, 70, 96), (70, 129, 320), (300, 300, 1056)])
def test_nan_blocks_stay_in_their_rows(gpu, M, N, K):
    a, w, bias = operands(gpu, M, N, K, 5)
    a.scales[M // 2, 0] = 255
    a.scales[0, -1] = 255
    a.packed[0, -16:] = 0  # NaN whatever the nibbles say
    w.scales[N - 1, K // 64] = 255
    A, W = ref.of_matrix(a), ref.of_matrix(w)
    want, tol = ref.product(A, W, bias)
    assert torch.isnan(want).sum() == 2 * N + M - 2
    for dtype in (BF16, F32):
        ref.assert_values(gpu.mxfp4_matmul(a, w, bias=bias, dtype=dtype), want, tol.nan_to_num())
    # results as MXFP4: a block with a NaN is one
    w = ref.random_matrix(gpu, gen_of(6), 128, K)
    w.scales[40, 0] = 255
    for swiglu in (False, True):
        got = gpu.mxfp4_matmul(a, w, swiglu=swiglu, quantize=True)
        cols = 64 if swiglu else 128
        bad = torch.zeros((M, cols // 32), dtype=torch.bool)
        bad[0], bad[M // 2], bad[:, 0 if swiglu else 1] = True, True, True
        assert torch.equal(got.scales.cpu() == 255, bad)
        assert not got.packed.view(M, -1, 16)[bad.cuda()].any()


def test_a_product_that_overflows(gpu):
    """Past the range: infinities of the sum's sign."""
    a, w = (gpu.MXFP4Matrix(torch.full((2, 32), 0x77, dtype=torch.uint8, device="cuda"),
                            torch.full((2, 2), 254, dtype=torch.uint8, device="cuda")) for _ in range(2))
    w.packed[1] = 0xff
    got = gpu.mxfp4_matmul(a, w, dtype=F32).cpu()
    assert got.tolist() == [[math.inf, -math.inf]] * 2


def test_rows_give_the_same_in_any_call(gpu):
    """A result is that of its row and column: calls that take the same way give the same bits, and repeats do."""
    a, w, bias = operands(gpu, 600, 512, 1024, 8)
    first = gpu.mxfp4_matmul(a, w, bias=bias)
    for _ in range(3):
        assert torch.equal(gpu.mxfp4_matmul(a, w, bias=bias), first)


def test_quantise_and_multiply(gpu):
    """As a projection runs: activations to MXFP4, then the product."""
    x = torch.randn((70, 2880), device="cuda", generator=gen_of(9)).to(BF16)
    w = gpu.mxfp4_quantize(torch.randn((200, 2880), device="cuda", generator=gen_of(10)) / 50)
    code, s = ref.quantize(x)
    want, tol = ref.product(ref.values(code, s), ref.of_matrix(w))
    ref.assert_values(gpu.mxfp4_matmul(gpu.mxfp4_quantize(x), w), want, tol)


def test_streams_and_graphs(gpu):
    x = torch.randn((64, 1024), device="cuda", generator=gen_of(11)).to(BF16)
    _, w, bias = operands(gpu, 1, 512, 1024, 12)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = gpu.mxfp4_matmul(gpu.mxfp4_quantize(x, stream=side), w, bias=bias, stream=side)
    side.synchronize()
    assert torch.equal(got, gpu.mxfp4_matmul(gpu.mxfp4_quantize(x), w, bias=bias))
    q = gpu.MXFP4Matrix(torch.empty((64, 512), dtype=torch.uint8, device="cuda"),
                        torch.empty((64, 32), dtype=torch.uint8, device="cuda"))
    out, back = torch.empty((64, 512), dtype=BF16, device="cuda"), torch.empty((64, 1024), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.mxfp4_matmul(gpu.mxfp4_quantize(x, out=q), w, bias=bias, out=out)
        gpu.mxfp4_dequantize(q, out=back)
    for seed in range(3):
        x.copy_(torch.randn((64, 1024), device="cuda", generator=gen_of(seed)))
        fresh = gpu.mxfp4_quantize(x)
        want = gpu.mxfp4_matmul(fresh, w, bias=bias)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(back, gpu.mxfp4_dequantize(fresh, dtype=F32))


def test_bf16_patterns_survive_the_trip(gpu):
    """Values that MXFP4 holds come back as they were."""
    m = ref.random_matrix(gpu, gen_of(13), 64, 256, low=4, high=250)
    m.packed[:, ::16] = 0x77  # the largest code in every block, so that the scale is found again
    v = gpu.mxfp4_dequantize(m)
    again = gpu.mxfp4_quantize(v)
    assert torch.equal(again.scales, m.scales) and torch.equal(gpu.mxfp4_dequantize(again), v)
    assert np.isfinite(v.float().cpu().numpy()).all()


def rows_of(gpu, m, at):
    return gpu.MXFP4Matrix(m.packed[at].contiguous(), m.scales[at].contiguous())


def test_quantize_past_32_bits(gpu):
    """Values, packed bytes and results at offsets beyond 2^32."""
    rows, K = (1 << 21) + 5, 4128
    x = torch.empty((rows, K), device="cuda", dtype=BF16)
    x.view(torch.int16).random_(-17000, 17000)  # with NaN among the negative ones
    m = gpu.mxfp4_quantize(x)
    back = gpu.mxfp4_dequantize(m)
    assert m.packed.numel() > 1 << 32
    at = torch.tensor([0, 1, 520287, 1040575, 2080895, rows - 2, rows - 1], device="cuda")
    few = x[at]
    want = ref.quantize(few)
    got = rows_of(gpu, m, at)
    assert torch.equal(ref.unpack(got.packed), want[0]) and torch.equal(got.scales.cpu(), want[1])
    assert torch.equal(back[at].cpu().double().nan_to_num(-7.25), ref.of_matrix(got).to(BF16).double().nan_to_num(-7.25))


def test_products_past_32_bits(gpu):
    """Weights, and results, at offsets beyond 2^32."""
    E, N, K = 290, 4096, 8192
    w = ref.random_matrix(gpu, gen_of(1), E, N, K, low=119, high=124)
    a = ref.random_matrix(gpu, gen_of(2), 200, K, low=119, high=124)
    W = ref.of_matrix(gpu.MXFP4Matrix(w.packed[E - 2], w.scales[E - 2]))
    for n in (3, 40, 200):
        offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        offsets[E - 1:] = n
        want, tol = ref.product(ref.of_matrix(gpu.MXFP4Matrix(a.packed[:n], a.scales[:n])), W)
        ref.assert_values(gpu.grouped_mxfp4_matmul(a, w, offsets, n), want, tol)
        all_rows = torch.tensor([0] * E + [n], dtype=torch.int32, device="cuda")
        last = gpu.grouped_mxfp4_matmul(a, w, all_rows, n)
        want, tol = ref.product(ref.of_matrix(gpu.MXFP4Matrix(a.packed[:n], a.scales[:n])),
                                ref.of_matrix(gpu.MXFP4Matrix(w.packed[E - 1], w.scales[E - 1])))
        ref.assert_values(last, want, tol)
    flat = gpu.MXFP4Matrix(w.packed.view(E * N, -1), w.scales.view(E * N, -1))  # tiles, by its many columns
    for n in (2, 8, 40, 200):
        few = gpu.MXFP4Matrix(a.packed[:n], a.scales[:n])
        want, tol = ref.product(ref.of_matrix(few), W)
        ref.assert_values(gpu.mxfp4_matmul(few, flat)[:, (E - 2) * N:(E - 1) * N], want, tol)
    del w, flat
    M, N, K = 70001, 32768, 64
    a, w, _ = operands(gpu, M, N, K, 3, low=119, high=124)
    got = gpu.mxfp4_matmul(a, w, dtype=F32)
    packed = gpu.mxfp4_matmul(a, w, quantize=True)
    at = torch.tensor([0, 16383, 32768, 65535, 65536, M - 2, M - 1], device="cuda")
    want, tol = ref.product(ref.of_matrix(rows_of(gpu, a, at)), ref.of_matrix(w))
    ref.assert_values(got[at], want, tol)
    ref.assert_quantized(rows_of(gpu, packed, at), want, tol)


@pytest.mark.parametrize("M, N", [(5, 6), (40, 2), (200, 130), (70, 1002), (650, 3206), (2900, 2946)])
def test_swiglu_of_few_columns_in_bf16(gpu, M, N):
    """In rows that begin on no more than an element: the same as the fp32 results, rounded."""
    a, w, bias = operands(gpu, M, N, 96, M, low=119, high=124)
    want = gpu.mxfp4_matmul(a, w, bias=bias, swiglu=True, dtype=F32).to(BF16)
    y, tol = ref.product(ref.of_matrix(a), ref.of_matrix(w), bias)
    ref.assert_values(want, *ref.swiglu(y, tol))
    for before, after in ((0, 0), (1, 0), (3, 4), (2, 1)):
        buf = torch.full((M, before + N // 2 + after), 7.0, device="cuda", dtype=BF16)
        out = buf[:, before:before + N // 2]
        gpu.mxfp4_matmul(a, w, bias=bias, swiglu=True, out=out)
        assert torch.equal(out, want), (before, after)
        assert bool((buf[:, :before] == 7).all()) and bool((buf[:, before + N // 2:] == 7).all())


@pytest.mark.parametrize("M, N, K", [(1, 64, 512), (3, 64, 4096), (40, 64, 32), (650, 3200, 32), (2900, 2944, 32)])
def test_swiglu_of_the_steepest_alpha(gpu, M, N, K):
    """alpha of 2^127: the sigmoid is 0 or 1, and 1/2 of a gate of zero; gates and ups are the biases."""
    a, w, _ = operands(gpu, M, N, K)
    a.packed.zero_()
    gate = torch.tensor([0.0, 1.0, -1.0, 0.5, -8.0, 8.0, -0.0, 2.0], device="cuda").repeat(N // 16)
    up = torch.linspace(-8, 8, N // 2, device="cuda").to(BF16).float()
    bias = torch.stack((gate, up), 1).flatten().to(BF16)
    g, u = gate.clamp(max=7), up.clamp(-7, 7)
    for alpha in (2.0 ** 127, -2.0 ** 127):
        on = (g * alpha) > 0
        got = gpu.mxfp4_matmul(a, w, bias=bias, swiglu=True, alpha=alpha, dtype=F32)
        assert torch.equal(got, torch.where(on, (u + 1) * g, torch.zeros_like(g)).expand(M, -1))
