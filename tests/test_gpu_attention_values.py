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
