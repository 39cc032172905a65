"""GPU: attention over caches whose scores or values lie at the ends of their range, against 64 bits (attn_ref.py)."""
import pytest
import torch

import attn_ref as ref
from test_gpu_attention import BF16, GPT, Case, randn, say

pytestmark = pytest.mark.gpu

GQA4 = (32, 8, 128, 32)


@pytest.mark.parametrize("shape", [GPT, GQA4, (5, 1, 64, 64)])
@pytest.mark.parametrize("n", [20, 100, 1000, 5000])
def test_large_values_without_weight(gpu, shape, n):
    """A visible value of 1e38 counts for nothing where its weight is below 2^-126 of the largest: with exact weights
    below 2^-300 it adds less than 1e-52."""
    say("large values", shape, n)
    H, Hk, D, bs = shape
    c = Case(gpu, 71, [n, n], *shape)
    q = (randn(c.gen, 2, H * D, scale=1.5).float() + 2.0).to(BF16)  # all heads against a key of -4 in every dim
    for b in range(2):
        for t in (3, n // 2, n - 1):
            page = c.tables[b, t // bs].long()
            c.pages[0][page, :, t % bs] = -4.0
            c.pages[1][page, :, t % bs] = 1e38
    # every head's score of these tokens is far enough below its best
    for b in range(2):
        for h in range(H):
            k = ref.load(c.pages, c.scales, c.tables[b], bs, n, h // (H // Hk))[0]
            s = 8.0 * (k @ q[b].double().view(H, D)[h])
            assert s.max() - max(s[3], s[n // 2], s[n - 1]) > 300 * 0.6932, (b, h)
    want, tol = c.want(q, [1, 1], scale=8.0)
    off = torch.arange(3, dtype=torch.int32, device="cuda")
    for name, got in (("decode", gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens, scale=8.0)),
                      ("prefill", gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens, scale=8.0))):
        bad = ref.within(got, want, tol)
        assert bad is None, (name, bad)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("scale", [1e-44, 1e-40, 1e-20])
def test_smallest_scales(gpu, e4m3, scale):
    """Scales so small that the product with an 8-bit cache's underflows: every seen token counts alike."""
    c = Case(gpu, 72, [50, 333, 3], *GPT, e4m3=e4m3)
    if e4m3:
        c.scales[0].fill_(0.01)
    for window in (0, 20):
        c.check_decode(window=window, scale=scale)
        c.check_prefill([50, 70, 1], window=window, scale=scale)


@pytest.mark.parametrize("shape,e4m3,new,n", [(GPT, False, 2048, 2048), (GPT, False, 60, 9000), (GQA4, True, 300, 6000)])
def test_what_lies_past_the_end_costs_nothing(gpu, shape, e4m3, new, n):
    """NaN in the last page's slots past the end, as memory that nothing was written to may hold: the same results, in
    about the same time (looking at every token took 13 to 18 times as long)."""
    H, Hk, D, bs = shape
    c = Case(gpu, 73, [n - 3], *shape, e4m3=e4m3)
    pages = [p.clone() for p in c.pages]
    raw = pages[1].view(torch.uint8) if e4m3 else pages[1]
    page = c.tables[0, -1].long()
    raw[page, :, (n - 3) % bs:] = 0
    clean = gpu.KVCache(pages[0], pages[1], *c.scales)
    q = randn(c.gen, new, H * D, scale=1.5)
    off = torch.tensor([0, new], dtype=torch.int32, device="cuda")

    def took(cache):
        best = float("inf")
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(10):
                out = gpu.paged_attention_prefill(q, off, cache, c.tables, c.seq_lens)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return out, best

    (want, fast), (got, slow) = took(clean), took(c.cache)
    say("past the end", shape, e4m3, new, n, f"{100 * fast:.1f} us, with NaN {100 * slow:.1f}")
    assert torch.equal(got, want) and want.isfinite().all()
    assert slow < 3 * fast


@pytest.mark.parametrize("shape,e4m3", [(GPT, False), (GPT, True), (GQA4, False), (GQA4, True), ((128, 4, 64, 16), False)])
@pytest.mark.parametrize("window,first", [(0, 0), (1200, 0), (5000, 70)])
def test_values_of_far_tiles_reach_only_who_sees_them(gpu, shape, e4m3, window, first):
    """NaN and infinities among the values of a long context, 64 tiles apart and in one tile, in seen places, between
    window and first tokens and past the end: in the rows that see them and in no other."""
    say("far values", shape, e4m3, window, first)
    H, Hk, D, bs = shape
    n, new, G = 9000, 4200 if H == 128 else 150, H // Hk
    c = Case(gpu, 74, [n], *shape, e4m3=e4m3)
    q = randn(c.gen, new, H * D, scale=1.5)
    off = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    call = lambda: gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens, window=window,  # noqa: E731
                                               first_tokens=first).view(new, H, D)
    want = call().clone()
    assert want.isfinite().all()
    pos = torch.arange(n - new, n, device="cuda")
    bad = torch.zeros((new, H, D), dtype=torch.bool, device="cuda")
    for i, t in enumerate([2, 69, 70, 4850, 4850 - 4096, n - 1 - 4096, n - 130, n - 130 + 1, n - 100, n - 64, n - 1, n - 1]):
        d = 5 * i % D
        page = c.tables[0, t // bs].long()
        if e4m3:
            c.pages[1].view(torch.uint8)[page, 1, t % bs, d] = 0x7f
        else:
            c.pages[1][page, 1, t % bs, d] = float("inf") if i % 2 else float("nan")
        sees = (t <= pos) & ((window == 0) | (pos - t < window) | (t < first))
        bad[:, G:2 * G, d] |= sees[:, None]
    got = call()
    assert (~got[bad].isfinite()).all()
    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("shape", [GPT, GQA4])
@pytest.mark.parametrize("lens", [[40, 500], [9000]])
def test_values_up_to_the_limit(gpu, shape, lens):
    """Values times tokens up to 2^115 give no infinities on the way: 4.5 * 1.5 sigma * 2^98 * 9000 is below it."""
    c = Case(gpu, 75, lens, *shape)
    for b, n in enumerate(lens):  # NaN past the ends stays NaN
        c.pages[1][c.tables[b, : (n + shape[3] - 1) // shape[3]].long()] *= 2.0 ** 98
    c.check_decode(sinks=randn(c.gen, shape[0]))
    c.check_prefill([min(n, 70) for n in lens])
    c.check_prefill([min(n, 5) for n in lens], window=200, first=10)


@pytest.mark.parametrize("shape", [GPT, GQA4])
@pytest.mark.parametrize("n", [2, 300, 3000])
def test_large_values_of_small_weights(gpu, shape, n):
    """The largest values where their weights are the smallest powers of two: as precise as any.  With a scale of ln 2 a
    key of -g in one dim of a query of ones is a weight of 2^-g; the other tokens but one have none at all."""
    H, Hk, D, bs = shape
    gaps = [90, 100, 110, 116, 118, 120, 122, 124, 125]
    c = Case(gpu, 76, [n] * len(gaps), *shape)
    for b, gap in enumerate(gaps):
        for t in range(n):
            page = c.tables[b, t // bs].long()
            c.pages[0][page, :, t % bs] = -4.0
            if t in (0, n // 2):
                c.pages[0][page, :, t % bs] = 0.0
        page = c.tables[b, n // 2 // bs].long()
        c.pages[0][page, :, n // 2 % bs, 5] = -float(gap)
        c.pages[1][page, :, n // 2 % bs] = 3.25e38
    q = torch.ones((len(gaps), H * D), dtype=BF16, device="cuda")
    want, tol = c.want(q, [1] * len(gaps), scale=0.6931471805599453)
    off = torch.arange(len(gaps) + 1, dtype=torch.int32, device="cuda")
    for name, got in (("decode", gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens, scale=0.6931471805599453)),
                      ("prefill", gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens, scale=0.6931471805599453))):
        bad = ref.within(got, want, tol)
        assert bad is None, (name, bad)
    # an infinite value is infinite with all of these weights
    for b, gap in enumerate(gaps):
        c.pages[1][c.tables[b, n // 2 // bs].long(), :, n // 2 % bs, 7] = float("inf")
    for name, call in (("decode", lambda: gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens, scale=0.6931471805599453)),
                       ("prefill", lambda: gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens,
                                                                       scale=0.6931471805599453))):
        got = call().view(len(gaps), H, D)
        say(name, [(gap, got[b, 0, 7].item()) for b, gap in enumerate(gaps)])
        assert (got[..., 7] == float("inf")).all() and got[..., :7].isfinite().all() and got[..., 8:].isfinite().all()
