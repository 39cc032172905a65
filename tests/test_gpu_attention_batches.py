"""GPU: attention calls of very many sequences, and of tables much wider than their sequences, against 64 bits
(attn_ref.py)."""
import pytest
import torch

import attn_ref as ref
from test_gpu_attention import BF16, GPT, GQA4, Case, gen_of, randn, say

pytestmark = pytest.mark.gpu


def shared(gpu, seed, B, width, Hk=1, D=64, bs=16, blocks=300):
    """A cache whose pages all sequences share: tables of any pages."""
    gen = gen_of(seed)
    pages = [randn(gen, blocks, Hk, bs, D, scale=1.5) for _ in range(2)]
    tables = torch.randint(0, blocks, (B, width), device="cuda", generator=gen).to(torch.int32)
    return gen, pages, gpu.KVCache(*pages), tables


@pytest.mark.parametrize("B,D,H,Hk", [(8193, 64, 8, 1), (20000, 64, 8, 1), (17000, 128, 2, 2)])
def test_tens_of_thousands_of_sequences(gpu, B, D, H, Hk):
    """Short sequences with long ones among them, which are cut; in a prompt call most have no new token."""
    say("sequences", B, D, H, Hk)
    gen, pages, cache, tables = shared(gpu, 81, B, 130, Hk, D)
    lens = [1 + 37 * b % 90 for b in range(B)]
    marks = sorted({k * x // 12 for x in (B, B - 1) for k in range(13)} - {B} | {4095, 4096, 4097, 6666, 6667, 8191, 8192})
    for i, b in enumerate(marks):
        lens[b] = (2070, 1, 0, 1300, 33)[i % 5]
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = randn(gen, B, H * D, scale=1.5)
    want = torch.full((B, H * D), 7.0, dtype=BF16, device="cuda")
    got = gpu.paged_attention_decode(q, cache, tables, seq_lens, out=want)
    new = [0] * B
    for b in marks:
        new[b] = min(lens[b], 20)
    rows = sum(new)
    p = randn(gen, rows, H * D, scale=1.5)
    off = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    chunk = gpu.paged_attention_prefill(p, off, cache, tables, seq_lens)
    off = off.tolist()
    torch.cuda.synchronize()
    assert got.isfinite().all() and not (got == 7).all(1).any()  # every row is written
    for b in marks + [b + 1 for b in marks if b + 1 < B]:
        n, at = lens[b], off[b]
        for x, out, pos in ((q[b:b + 1], got[b:b + 1], [n - 1]),
                            (p[at:at + new[b]], chunk[at:at + new[b]], range(n - new[b], n))):
            o, tol = ref.attend64(x.view(-1, H, D), list(pos), n, pages, [None, None], tables[b], 16, D ** -0.5)
            bad = ref.within(out.view(-1, H, D), o, tol)
            assert bad is None, (b, bad)


def test_time_grows_with_the_sequences(gpu):
    """Eight times as many sequences take about eight times as long (45 and 80 times where every work-group looked
    through all of them)."""
    took = {}
    for B in (8192, 65536):
        gen, pages, cache, tables = shared(gpu, 82, B, 80)
        seq_lens = torch.full((B,), 3, dtype=torch.int32, device="cuda")
        q, out = randn(gen, B, 512), torch.empty((B, 512), dtype=BF16, device="cuda")
        off = torch.arange(B + 1, dtype=torch.int32, device="cuda")
        for name, call in (("decode", lambda: gpu.paged_attention_decode(q, cache, tables, seq_lens, out=out)),
                           ("prefill", lambda: gpu.paged_attention_prefill(q, off, cache, tables, seq_lens, out=out))):
            best = float("inf")
            for _ in range(4):
                a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
                a.record()
                call()
                b.record()
                torch.cuda.synchronize()
                best = min(best, a.elapsed_time(b))
            took[name, B] = best
            say(name, B, f"{best:.2f} ms")
    for name in ("decode", "prefill"):
        assert took[name, 65536] < 24 * took[name, 8192]


# tables as a serving engine has them, of the longest context that it allows
WIDE = [(GPT, [680], [680]), (GPT, [512], [512]), (GPT, [1120, 900, 500, 300], [120, 110, 60, 40]),
        (GPT, [1028, 900, 800, 700, 500, 300, 200, 128], [128, 100, 60, 40, 100, 20, 30, 28]), (GQA4, [680], [680]),
        (GPT, [1], [1]), (GPT, [17, 0, 2], [5, 0, 2]), (GQA4, [100, 3000], [1, 1]), ((6, 6, 128, 16), [300, 20], [31, 20])]


@pytest.mark.parametrize("shape,lens,new", WIDE)
@pytest.mark.parametrize("e4m3", [False, True])
def test_wide_tables(gpu, shape, lens, new, e4m3):
    """Tables of 131072 tokens over short sequences."""
    say("wide tables", shape, lens, new, e4m3)
    c = Case(gpu, 83, lens, *shape, e4m3=e4m3, width=131072 // shape[3])
    sinks = randn(c.gen, shape[0])
    c.check_prefill(new, sinks=sinks)
    c.check_prefill(new, window=100, first=3)
    c.check_decode(sinks=sinks)
    c.check_decode(window=100, first=3)


@pytest.mark.parametrize("B,L", [(1, 1000), (1, 500), (64, 1000), (40, 30)])
def test_wide_tables_of_single_tokens(gpu, B, L):
    c = Case(gpu, 84, [L - 3 * b for b in range(min(B, L // 3))], *GPT, width=131072 // 16)
    c.check_decode(sinks=randn(c.gen, 64))


@pytest.mark.parametrize("shape,new", [(GPT, 210), (GQA4, 340)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_prefill_two_groups_in_two_pieces(gpu, shape, new, e4m3):
    say("two groups in two pieces", shape, new, e4m3)
    c = Case(gpu, 85, [4090], *shape, e4m3=e4m3)
    c.tables[0, 20] = -1
    c.check_prefill([new], sinks=randn(c.gen, shape[0], scale=2.0))
    c.check_prefill([new], window=3500, first=70)
