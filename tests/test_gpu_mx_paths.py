"""GPU: MXFP4 products on each of their kernels, with K of several turns of its loop and every kind of rest, dense and by
expert.  test_mx_paths_cpu.py holds which kernel each call takes.

fp32 results are compared with 64 bits (mx_ref.py, where the tolerances are derived); the same call's results in bf16 and in
MXFP4 are those of the fp32 ones, rounded or quantised, bit for bit: every kernel sums a result in one order."""
import pytest
import torch

import mx_ref as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32

# (kernel, rows of each expert or of the one matrix, N, K).  Tiles take K in chunks of 256 and loop over four of them: 1056 is
# a loop, a chunk and of that one block; 1760 a loop and three, the last one a part; 2880 three loops, whose last chunk is a part.
LARGE = [300, 120, 200, 60, 0]  # tiles of 256, 44, 120, 200 and 60 rows
MIDDLE = [30, 90, 65, 128, 1, 0, 64, 33, 260, 77, 40, 50, 66, 31, 32, 96]
LOW = [4, 24, 0, 33, 17, 1, 8, 12, 40, 3, 16, 5, 32, 9, 7, 11, 20, 0, 14, 6, 2, 65, 10, 13]
FEW = [2, 1, 0, 3, 2, 2, 17, 0, 1, 2, 4, 1, 0, 0, 3, 1, 2, 2, 0, 1, 2, 1, 0, 1]
CASES = [("large", LARGE, 6720, K) for K in (1056, 1760, 2880)] + \
        [("middle", MIDDLE, 1472, K) for K in (1056, 1760, 2880)] + \
        [("low", LOW, 704, K) for K in (1056, 1760, 2880)] + \
        [("large", [2817], 2946, 1760), ("large", [2900], 2944, 2880), ("middle", [700], 2946, 1056), ("middle", [650], 3200, 2880),
         ("low", [300], 1001, 2080), ("low", [200], 1344, 2880)] + \
        [("stream", FEW, 1984, K) for K in (544, 2880, 8224)] + \
        [("stream", [130, 1], 192, 8224), ("wide stream", [2] * 56 + [0] * 72, 2304, 2880)] + \
        [("split stream", [5, 0, 4], 256, K) for K in (4096, 4128, 17056)] + \
        [("split stream", [16], 96, 17056), ("split stream", [1], 2048, 8224)]
IDS = [f"{way.replace(' ', '_')}-{sum(counts)}of{len(counts)}-{N}-{K}" for way, counts, N, K in CASES]


def edges(counts):
    """Rows before the first expert's and after the last one's: none of a dense product."""
    return (0, 0) if len(counts) == 1 else (1, 1) if sum(counts) < 16 else (3, 5)


def values(m):
    """As mx_ref's, on the GPU."""
    table = torch.cat((ref.GRID, -ref.GRID)).cuda()
    code = torch.stack((m.packed & 15, m.packed >> 4), dim=-1).flatten(-2).int()
    return table[code] * torch.exp2(m.scales.double() - 127).repeat_interleave(32, dim=-1)


class Case:
    def __init__(self, gpu, counts, N, K):
        self.gpu, E = gpu, len(counts)
        gen = torch.Generator(device="cuda").manual_seed(N + K + E)
        before, after = edges(counts)
        ends = [before]
        for n in counts:
            ends.append(ends[-1] + n)
        self.rows, self.lo, self.hi, self.ends = ends[-1] + after, before, ends[-1], ends
        self.grouped = E > 1
        a_rows = self.rows // 2 + 1 if self.grouped else self.rows
        self.a = ref.random_matrix(gpu, gen, a_rows, K, low=119, high=124)
        self.w = ref.random_matrix(gpu, gen, *((E, N) if self.grouped else (N,)), K, low=119, high=124)
        self.bias = torch.randn((E, N) if self.grouped else N, device="cuda", generator=gen).to(BF16)
        self.offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
        self.index = torch.randint(0, a_rows, (self.rows,), device="cuda", generator=gen).to(torch.int32)

    def want(self, bias):
        A, outs = values(self.a), []
        for e, (lo, hi) in enumerate(zip(self.ends, self.ends[1:])):
            if lo < hi:
                m = self.gpu.MXFP4Matrix(self.w.packed[e], self.w.scales[e]) if self.grouped else self.w
                W, rows = values(m), A[self.index[lo:hi].long()] if self.grouped else A
                y, size = rows @ W.T, rows.abs() @ W.abs().T
                tol = A.shape[1] * 2.0 ** -24 * size
                if bias:
                    y = y + (self.bias[e] if self.grouped else self.bias).double()
                    tol = tol + 2.0 ** -24 * y.abs()
                outs.append((y.cpu(), tol.cpu() + 2.0 ** -140))
        return [torch.cat(t) for t in zip(*outs)]

    def __call__(self, **kw):
        if self.grouped:
            return self.gpu.grouped_mxfp4_matmul(self.a, self.w, self.offsets, self.rows, row_index=self.index, **kw)
        return self.gpu.mxfp4_matmul(self.a, self.w, **kw)


@pytest.mark.parametrize("way, counts, N, K", CASES, ids=IDS)
def test_products(gpu, way, counts, N, K):
    c = Case(gpu, counts, N, K)
    lo, hi = c.lo, c.hi
    for with_bias in (True, False):
        y, tol = c.want(with_bias)
        for swiglu in (False, True) if N % 2 == 0 else (False,):
            want, off = ref.swiglu(y, tol) if swiglu else (y, tol)
            cols = want.shape[1]
            kw = dict(bias=c.bias if with_bias else None, swiglu=swiglu)
            out = torch.full((c.rows, cols), 9.0, device="cuda")
            assert c(out=out, **kw) is out
            ref.assert_values(out[lo:hi], want, off, (way, with_bias, swiglu))
            assert bool((out[:lo] == 9).all()) and bool((out[hi:] == 9).all())
            # in bf16; in rows that begin on no more than an element, and in ones on 16 bytes
            short = c(dtype=BF16, **kw)
            assert torch.equal(short[lo:hi], out[lo:hi].to(BF16))
            for dtype in (BF16, F32):
                for before, after in ((1, 2 - cols % 2), (8, 16 - cols % 8)):
                    buf = torch.full((c.rows, before + cols + after), 9.0, device="cuda", dtype=dtype)
                    part = buf[:, before:before + cols]
                    c(out=part, **kw)
                    assert torch.equal(part[lo:hi], out[lo:hi].to(dtype)), (dtype, before)
                    part[lo:hi] = 9
                    assert bool((buf == 9).all())
            if cols % 32 == 0:
                m = gpu.MXFP4Matrix(torch.full((c.rows, cols // 2), 99, dtype=torch.uint8, device="cuda"),
                                    torch.full((c.rows, cols // 32), 88, dtype=torch.uint8, device="cuda"))
                assert c(quantize=True, out=m, **kw) is m
                q = gpu.mxfp4_quantize(out[lo:hi].contiguous())
                assert torch.equal(m.packed[lo:hi], q.packed) and torch.equal(m.scales[lo:hi], q.scales)
                m.packed[lo:hi], m.scales[lo:hi] = 99, 88
                assert bool((m.packed == 99).all()) and bool((m.scales == 88).all())


# (kernel, N, K): the first rows of larger calls, and other numbers of rows, on the same kernel
PREFIXES = [("large", 6720, 1056, (2300, 1409, 1300)), ("middle", 1472, 1056, (1500, 1441, 1400)),
            ("low", 704, 1056, (500, 401, 388)), ("stream", 192, 2880, (130, 1, 17, 64)), ("split stream", 256, 4128, (16, 1, 7))]


@pytest.mark.parametrize("way, N, K, rows", PREFIXES, ids=[p[0].replace(" ", "_") for p in PREFIXES])
def test_a_prefix_gives_the_same(gpu, way, N, K, rows):
    """A result is that of its row and column: the same bits in a call of fewer rows on the same kernel, and in another place."""
    c = Case(gpu, [rows[0]], N, K)
    first = c(bias=c.bias)
    for n in rows[1:]:
        for at in (slice(0, n), slice(rows[0] - n, rows[0])):
            a = gpu.MXFP4Matrix(c.a.packed[at].contiguous(), c.a.scales[at].contiguous())
            assert torch.equal(gpu.mxfp4_matmul(a, c.w, bias=c.bias), first[at]), n


@pytest.mark.parametrize("M, N, K", [(3, 64, 512), (40, 128, 32), (40, 256, 512), (16, 128, 4096), (300, 264, 64),
                                     (650, 3200, 96), (2900, 2944, 64), (2900, 2944, 288)])
def test_sums_keep_24_bits(gpu, M, N, K):
    """Sums whose every part, in any order, is a whole number below 2^24 of one unit: fp32 holds each of them, so the result is
    exact.  One block is 2^p larger than the others, as far as that goes."""
    gen = torch.Generator(device="cuda").manual_seed(K)
    a = ref.random_matrix(gpu, gen, M, K, low=127, high=128)
    w = ref.random_matrix(gpu, gen, N, K, low=127, high=128)
    # products are multiples of 2^-2 up to 36: (36 * 32 * 2^p + 36 * (K - 32)) * 4 < 2^24
    p = 0
    while (36 * 32 * 2 ** (p + 1) + 36 * (K - 32)) * 4 < 1 << 24:
        p += 1
    for block in {0, K // 64, K // 32 - 1}:
        a.scales.fill_(127)
        a.scales[:, block] = 127 + p
        want = values(a) @ values(w).T
        assert float((values(a).abs() @ values(w).abs().T).max()) * 4 < 1 << 24
        got = gpu.mxfp4_matmul(a, w, dtype=F32)
        assert torch.equal(got.double(), want), (block, p, float((got - want).abs().max()))
