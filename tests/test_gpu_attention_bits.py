"""GPU: decode's weights meet the values with 16 significant bits (attn_bits.py; test_attention_bits_cpu.py shows that
bf16 weights do not pass)."""
import pytest
import torch

import attn_bits as bits
import attn_ref as ref
from test_gpu_attention import GPT, GQA4, Case, randn, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [GPT, GQA4, (17, 1, 64, 256), (6, 6, 128, 16)])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[600], [2, 17, 100, 600], [600, 33, 100, 17, 64, 350] * 12])
@pytest.mark.parametrize("wide", [False, True])
def test_weights_of_16_bits(gpu, shape, e4m3, lens, wide):
    """In one launch, and cut into pieces that are joined (the wide table)."""
    say("bits", shape, e4m3, len(lens), wide)
    H, Hk, D, bs = shape
    c = Case(gpu, 95, lens, *shape, e4m3=e4m3, width=8192 // bs if wide else None)
    q = randn(c.gen, len(lens), H * D, scale=0.5)
    got = gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens)
    for b, n in enumerate(lens):
        out, tol, _ = bits.decode64(q[b].view(H, D), n, c.pages, c.scales, c.tables[b], bs, D ** -0.5)
        bad = ref.within(got[b].view(H, D), out, tol)
        assert bad is None, (b, bad)
