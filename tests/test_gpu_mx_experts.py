"""GPU: the grouped MXFP4 products, and routing, quantisation and products together as a mixture of experts runs them,
against their definition in 64 bits (mx_ref.py, where the tolerances are derived)."""
import pytest
import torch

import mx_ref as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Case:
    def __init__(self, gpu, counts, N, K, seed=0, gather=True, before=0, after=0):
        self.gpu, E = gpu, len(counts)
        ends = [before]
        for n in counts:
            ends.append(ends[-1] + n)
        self.rows = ends[-1] + after
        self.lo, self.hi = before, ends[-1]
        gen = gen_of(seed)
        a_rows = max(1, self.rows // 3 if gather else self.rows)
        self.a = ref.random_matrix(gpu, gen, a_rows, K, low=119, high=124)
        self.w = ref.random_matrix(gpu, gen, E, N, K, low=119, high=124)
        self.bias = torch.randn((E, N), device="cuda", generator=gen).to(BF16)
        self.offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
        self.index = torch.randint(0, a_rows, (self.rows,), device="cuda", generator=gen).to(torch.int32) if gather else None
        self.ends = ends

    def want(self, swiglu=False, bias=True):
        A, W = ref.of_matrix(self.a), ref.of_matrix(self.w)
        outs, tols = [], []
        for e, (lo, hi) in enumerate(zip(self.ends, self.ends[1:])):
            at = torch.arange(lo, hi) if self.index is None else self.index[lo:hi].cpu().long()
            rows = torch.where((at >= 0)[:, None] & (at < A.shape[0])[:, None], A[at.clamp(0, A.shape[0] - 1)], 0.0)
            y, tol = ref.product(rows, W[e], self.bias[e] if bias else None)
            y, tol = ref.swiglu(y, tol) if swiglu else (y, tol)
            outs.append(y), tols.append(tol)
        return torch.cat(outs), torch.cat(tols)

    def check(self, swiglu=False, bias=True, dtype=BF16):
        want, tol = self.want(swiglu, bias)
        out = torch.full((self.rows, want.shape[1]), 9.0, device="cuda", dtype=dtype)
        got = self.gpu.grouped_mxfp4_matmul(self.a, self.w, self.offsets, self.rows, row_index=self.index,
                                            bias=self.bias if bias else None, swiglu=swiglu, out=out)
        torch.cuda.synchronize()
        assert got is out
        ref.assert_values(out[self.lo:self.hi], want, tol)
        assert bool((out[:self.lo] == 9).all()) and bool((out[self.hi:] == 9).all())
        if want.shape[1] % 32 == 0 and self.rows:
            m = self.gpu.MXFP4Matrix(torch.full((self.rows, want.shape[1] // 2), 99, dtype=torch.uint8, device="cuda"),
                                     torch.full((self.rows, want.shape[1] // 32), 88, dtype=torch.uint8, device="cuda"))
            self.gpu.grouped_mxfp4_matmul(self.a, self.w, self.offsets, self.rows, row_index=self.index,
                                          bias=self.bias if bias else None, swiglu=swiglu, quantize=True, out=m)
            lo, hi = self.lo, self.hi
            if hi > lo:
                ref.assert_quantized(self.gpu.MXFP4Matrix(m.packed[lo:hi], m.scales[lo:hi]), want, tol)
            assert bool((m.packed[:lo] == 99).all()) and bool((m.packed[hi:] == 99).all())
            assert bool((m.scales[:lo] == 88).all()) and bool((m.scales[hi:] == 88).all())


COUNTS = [[1], [0, 0, 0], [5], [0, 3, 0, 1, 0], [1] * 20, [16, 17, 15], [31, 32, 33, 0, 64], [100, 0, 1, 260, 7],
          [300, 513, 2], [0, 0, 1000], [129, 127, 128, 255, 257]]


@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("N, K", [(64, 96), (128, 2880), (192, 512), (321, 64), (640, 1056)])
def test_grouped(gpu, counts, N, K):
    for gather in (True, False):
        c = Case(gpu, counts, N, K, seed=N + len(counts), gather=gather, before=3 if gather else 0, after=5 if gather else 0)
        c.check(dtype=F32 if gather else BF16)
        if N % 2 == 0:
            c.check(swiglu=True, bias=gather)


@pytest.mark.parametrize("counts, N, K", [([300, 100, 40, 129, 64, 65], 8192, 96), ([700, 0, 3], 9026, 64)])
def test_many_tiles(gpu, counts, N, K):
    """Tiles of 256 rows and their smaller ones."""
    c = Case(gpu, counts, N, K, before=2, after=3)
    c.check(dtype=F32)
    c.check(swiglu=True)


@pytest.mark.parametrize("N, K", [(256, 512), (258, 608)])
def test_few_rows_of_many_experts(gpu, N, K):
    E, used = 1024, {0: 3, 7: 17, 8: 1, 500: 40, 1023: 2}
    counts = [used.get(e, 0) for e in range(E)]
    offsets = torch.tensor([sum(counts[:e]) for e in range(E + 1)], dtype=torch.int32, device="cuda")
    rows = E  # as the call says; those behind the last offset stay as they are
    gen = gen_of(N)
    a = ref.random_matrix(gpu, gen, rows, K, low=119, high=124)
    w = ref.random_matrix(gpu, gen, E, N, K, low=119, high=124)
    bias = torch.randn((E, N), device="cuda", generator=gen).to(BF16)
    want, tol = [], []
    for e, n in used.items():
        lo = sum(counts[:e])
        y, t = ref.product(ref.of_matrix(gpu.MXFP4Matrix(a.packed[lo:lo + n], a.scales[lo:lo + n])),
                           ref.of_matrix(gpu.MXFP4Matrix(w.packed[e], w.scales[e])), bias[e])
        want.append(y), tol.append(t)
    want, tol, live = torch.cat(want), torch.cat(tol), sum(counts)
    out = torch.full((rows, N), 9.0, device="cuda", dtype=BF16)
    gpu.grouped_mxfp4_matmul(a, w, offsets, rows, bias=bias, out=out)
    ref.assert_values(out[:live], want, tol)
    assert bool((out[live:] == 9).all())
    want, tol = ref.swiglu(want, tol)
    out = torch.full((rows, N // 2), 9.0, device="cuda", dtype=F32)
    gpu.grouped_mxfp4_matmul(a, w, offsets, rows, bias=bias, swiglu=True, out=out)
    ref.assert_values(out[:live], want, tol)
    assert bool((out[live:] == 9).all())
    if N % 64 == 0:
        m = gpu.grouped_mxfp4_matmul(a, w, offsets, rows, bias=bias, swiglu=True, quantize=True)
        ref.assert_quantized(gpu.MXFP4Matrix(m.packed[:live], m.scales[:live]), want, tol)


def test_many_experts(gpu):
    """1024 experts, some of them with tokens."""
    g = torch.Generator().manual_seed(1)
    counts = (torch.randint(0, 40, (1024,), generator=g) * (torch.rand(1024, generator=g) < 0.1)).tolist()
    Case(gpu, counts, 64, 32).check()
    counts = [0] * 1023 + [70]
    Case(gpu, counts, 64, 32).check()


def test_row_numbers_outside_of_a(gpu):
    """They stand for rows of zeros: the bias alone."""
    c = Case(gpu, [40, 3, 100], 96, 160, before=2, after=2)
    c.index[5], c.index[20], c.index[44], c.index[60] = -1, c.a.rows, -2 ** 31, 2 ** 31 - 1
    c.check()
    c.check(swiglu=True)
    c.index.fill_(-1)
    c.check()


@pytest.mark.parametrize("offsets", [[-5, 4, 20, 40], [0, 30, 10, 40], [0, 10, 50, 70], [60, 60, 60, 60], [-9, -8, -7, -6],
                                     [-2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]])
def test_offsets_out_of_range_write_nothing_else(gpu, offsets):
    """Offsets that are no offsets: rows within the call are written or not, and nothing else is."""
    c = Case(gpu, [10, 20, 10], 64, 96, gather=False)
    around = torch.full((3 * 40, 64), 9.0, device="cuda", dtype=F32)
    c.gpu.grouped_mxfp4_matmul(c.a, c.w, torch.tensor(offsets, dtype=torch.int32, device="cuda"), 40,
                               out=around[40:80])
    torch.cuda.synchronize()
    assert bool((around[:40] == 9).all()) and bool((around[80:] == 9).all())


def test_empty_call(gpu):
    c = Case(gpu, [0, 0], 64, 96)
    assert gpu.grouped_mxfp4_matmul(c.a, c.w, c.offsets, 0).shape == (0, 64)
    assert gpu.mxfp4_matmul(gpu.mxfp4_quantize(torch.zeros((0, 96), device="cuda")), ref.random_matrix(gpu, gen_of(1), 64, 96)
                            ).shape == (0, 64)


class Block:
    """A mixture of experts on MXFP4 activations: router logits to the residual's sum."""

    def __init__(self, gpu, T, E, k, H, I, seed=0, groups=4):
        self.gpu, self.T, self.E, self.k, self.H, self.groups = gpu, T, E, k, H, groups
        gen = gen_of(seed)
        self.gen = gen
        self.bias = 0.1 * torch.randn(E, device="cuda", generator=gen)
        self.w1 = ref.random_matrix(gpu, gen, E, 2 * I, H, low=119, high=122)
        self.w2 = ref.random_matrix(gpu, gen, E, H, I, low=119, high=122)
        self.b1 = (0.1 * torch.randn((E, 2 * I), device="cuda", generator=gen)).to(BF16)
        self.b2 = (0.1 * torch.randn((E, H), device="cuda", generator=gen)).to(BF16)
        self.logits, self.x, self.residual = (torch.empty((T, n), device="cuda", dtype=BF16) for n in (E, H, H))
        self.fill()

    def fill(self):
        for t in (self.logits, self.x, self.residual):
            t.copy_(torch.randn(t.shape, device="cuda", generator=self.gen))

    def __call__(self):
        g = self.gpu
        idx, w = g.select_experts(self.logits, self.k, score="sigmoid", bias=self.bias, num_groups=self.groups,
                                  top_groups=self.groups // 2, scale=2.5)
        plan = g.permute_plan(idx, self.E)
        rows = self.T * self.k
        act = g.grouped_mxfp4_matmul(g.mxfp4_quantize(self.x), self.w1, plan["offsets"], rows, row_index=plan["perm_token"],
                                     bias=self.b1, swiglu=True, quantize=True)
        y = g.grouped_mxfp4_matmul(act, self.w2, plan["offsets"], rows, bias=self.b2)
        return g.combine(y, plan["gather_map"], w, self.residual, self.T, self.H, self.k), act, idx, plan

    def check(self):
        out, act, idx, plan = self()
        torch.cuda.synchronize()
        want_idx, w, _ = ref.select(self.logits, self.k, "sigmoid", self.bias, self.groups, self.groups // 2, 2, True, 2.5)
        assert torch.equal(idx.cpu(), want_idx)
        code, s = ref.quantize(self.x)
        x, A = ref.values(code, s), ref.of_matrix(act)
        W1, W2 = ref.of_matrix(self.w1), ref.of_matrix(self.w2)
        gm = plan["gather_map"].cpu().view(self.T, self.k)
        total, room = self.residual.cpu().double(), torch.zeros((self.T, self.H), dtype=torch.float64)
        for i in range(self.k):
            for e in want_idx[:, i].unique().tolist():
                t = (want_idx[:, i] == e).nonzero()[:, 0]
                y, tol = ref.swiglu(*ref.product(x[t], W1[e], self.b1[e]))
                m = self.gpu.MXFP4Matrix(act.packed[gm[t, i].cuda()].contiguous(), act.scales[gm[t, i].cuda()].contiguous())
                ref.assert_quantized(m, y, tol)
                # the activations that were made, through the second product; its rounding to bf16, the weights' and
                # the sum's in fp32
                z, tol = ref.product(A[gm[t, i]], W2[e], self.b2[e])
                p = w[t, i, None].double()
                total[t] += p * z
                room[t] += p * (tol + 2.0 ** -8 * z.abs()) + 20 * 2.0 ** -23 * (p * z).abs()
        ref.assert_values(out, total, room + (self.k + 1) * 2.0 ** -24 * total.abs() + 2.0 ** -20)


@pytest.mark.parametrize("T, E, k, H, I", [(1, 16, 4, 96, 64), (7, 32, 4, 320, 192), (200, 8, 2, 512, 256), (33, 64, 8, 224, 96)])
def test_the_operators_together(gpu, T, E, k, H, I):
    Block(gpu, T, E, k, H, I, seed=T).check()


def test_the_operators_together_in_a_graph(gpu):
    """Captured, replayed with other inputs (and so another routing), beside eager calls."""
    b = Block(gpu, 48, 32, 4, 320, 192)
    b()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b()[0]
    for _ in range(3):
        b.fill()
        want = b()[0]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_two_streams_at_once(gpu):
    """Nothing is shared between calls."""
    blocks = [Block(gpu, 64, 32, 4, 320, 192, seed=s) for s in range(2)]
    want = [b()[0] for b in blocks]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in blocks]
    for _ in range(5):
        got = []
        for b, s in zip(blocks, streams):
            with torch.cuda.stream(s):
                got.append(b()[0])
        torch.cuda.synchronize()
        for a, w in zip(got, want):
            assert torch.equal(a, w)


@pytest.mark.parametrize("counts, N, K", [([3, 0, 5], 96, 512), ([2, 3], 64, 4096), ([40, 3, 100], 96, 160),
                                          ([40] * 12, 1472, 64), ([300, 100, 40, 129, 64, 65], 8192, 96)])
def test_rows_of_zeros_and_weights_of_nan(gpu, counts, N, K):
    """A row number outside of a gives the bias alone, whatever the weights hold; other rows are NaN in such columns."""
    c = Case(gpu, counts, N, K, seed=3, before=1, after=1)
    c.w.scales[:, ::3, 0] = 255
    c.index[::2] = -1
    c.index[1::4] = c.a.rows
    expert = torch.cat([torch.full((n,), e) for e, n in enumerate(counts)])
    got = gpu.grouped_mxfp4_matmul(c.a, c.w, c.offsets, c.rows, row_index=c.index, bias=c.bias, dtype=F32)[c.lo:c.hi].cpu()
    index, bias = c.index[c.lo:c.hi].cpu(), c.bias.float().cpu()[expert]
    zero = (index < 0) | (index >= c.a.rows)
    assert bool(zero.any()) and bool((~zero).any())
    assert torch.equal(got[zero], bias[zero])
    nan = torch.isnan(got[~zero])
    assert bool(nan[:, ::3].all()) and not nan[:, 1::3].any() and not nan[:, 2::3].any()
