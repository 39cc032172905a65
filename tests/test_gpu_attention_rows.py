"""GPU: attention operators whose inputs and results are columns of one buffer."""
import pytest
import torch

import attn_ref as ref
from test_gpu_attention import BF16, GPT, Case, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_first", [False, True])
def test_results_beside_the_queries(gpu, out_first):
    """q and out as the halves of a buffer's rows: the bits of separate tensors, and q as it was."""
    c = Case(gpu, 91, [100, 37, 1500], *GPT)
    new = [30, 1, 5]
    off = torch.tensor([0, 30, 31, 36], dtype=torch.int32, device="cuda")
    for rows, call in ((36, lambda q, **k: gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens, **k)),
                       (3, lambda q, **k: gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens, **k))):
        both = randn(c.gen, rows, 2 * 4096 + 16)
        q, out = both[:, :4096], both[:, 4096 + 8:4096 + 8 + 4096]
        if out_first:
            q, out = out, q
        was, edge = q.clone(), both[:, 4096:4096 + 8].clone()
        want = call(was)
        assert call(q, out=out).data_ptr() == out.data_ptr()
        assert torch.equal(out, want) and torch.equal(q, was) and torch.equal(both[:, 4096:4096 + 8], edge)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("pairs", [False, True])
def test_queries_beside_their_rows(gpu, e4m3, pairs):
    gen = torch.Generator(device="cuda").manual_seed(92)
    H, Hk, D, bs = GPT
    table = gpu.rope_table()
    T, cols = 70, (H + 2 * Hk) * D
    both = randn(gen, T, cols + H * D)
    pos = torch.randint(0, 131072, (T,), device="cuda", generator=gen).to(torch.int32)
    slots = torch.randperm(T + 10, device="cuda", generator=gen)[:T].to(torch.int32)
    got = []
    for qkv, q_out in ((both[:, :cols].clone(), torch.zeros((T, H * D), dtype=BF16, device="cuda")),
                       (both[:, :cols], both[:, cols:])):
        pages, scales = ref.make_cache(torch.Generator(device="cuda").manual_seed(93), 5, Hk, bs, D, e4m3, fill=0.5)
        was = qkv.clone()
        gpu.rope_kv_append(qkv, pos, slots, table, gpu.KVCache(*pages, *scales), H, interleaved=pairs, q_out=q_out)
        assert torch.equal(qkv, was)
        got.append([q_out] + [p.view(torch.uint8) for p in pages])
    for a, b in zip(*got):
        assert torch.equal(a, b)
