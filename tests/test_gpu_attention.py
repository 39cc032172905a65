"""GPU: position rotation with the append to the paged cache, and attention of single tokens and of prompt chunks over
it, against their definition in 64 bits (attn_ref.py, where the tolerances are derived)."""
import math

import pytest
import torch

import attn_ref as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def say(*a):
    print(*a, flush=True)


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(gen, *shape, scale=1.0):
    return (scale * torch.randn(shape, device="cuda", generator=gen)).to(BF16)


class Case:
    """Sequences of lens tokens in a cache whose other slots hold NaN."""

    def __init__(self, gpu, seed, lens, H, Hk, D, bs, e4m3=False, layout="heads", spare=2, width=None):
        self.gpu, self.lens, self.H, self.Hk, self.D, self.bs = gpu, lens, H, Hk, D, bs
        self.gen = gen_of(seed)
        blocks = sum((n + bs - 1) // bs for n in lens) + spare
        self.pages, self.scales = ref.make_cache(self.gen, blocks, Hk, bs, D, e4m3, layout)
        self.tables = ref.page_tables(self.gen, lens, bs, blocks, width)
        for b, n in enumerate(lens):
            if n:
                ref.store(self.pages, self.scales, self.tables[b], bs,
                          [randn(self.gen, n, Hk, D, scale=1.5) for _ in range(2)])
        self.cache = gpu.KVCache(self.pages[0], self.pages[1], self.scales[0], self.scales[1])
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def want(self, q, new, window=0, first=0, sinks=None, scale=None):
        """q [sum(new), H * D]: the last new[b] tokens of each sequence."""
        scale = scale or self.D ** -0.5
        outs, tols, row = [], [], 0
        for b, (n, m) in enumerate(zip(self.lens, new)):
            o, t = ref.attend64(q[row:row + m].view(m, self.H, self.D), list(range(n - m, n)), n, self.pages, self.scales,
                                self.tables[b], self.bs, scale, window, first, sinks)
            outs.append(o), tols.append(t)
            row += m
        return torch.cat(outs).view(row, -1), torch.cat(tols).view(row, -1)

    def check_decode(self, window=0, first=0, sinks=None, **kw):
        q = randn(self.gen, len(self.lens), self.H * self.D, scale=1.5)
        want, tol = self.want(q, [1] * len(self.lens), window, first, sinks, kw.get("scale"))
        got = self.gpu.paged_attention_decode(q, self.cache, self.tables, self.seq_lens, window=window,
                                              first_tokens=first, sinks=sinks, **kw)
        torch.cuda.synchronize()
        bad = ref.within(got, want, tol)
        assert bad is None, bad
        return q, got

    def check_prefill(self, new, window=0, first=0, sinks=None, **kw):
        q = randn(self.gen, sum(new), self.H * self.D, scale=1.5)
        offsets = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
        want, tol = self.want(q, new, window, first, sinks, kw.get("scale"))
        got = self.gpu.paged_attention_prefill(q, offsets, self.cache, self.tables, self.seq_lens, window=window,
                                               first_tokens=first, sinks=sinks, **kw)
        torch.cuda.synchronize()
        bad = ref.within(got, want, tol)
        assert bad is None, bad
        return q, offsets, got


# heads, kv heads, head_dim, page size
GPT = (64, 8, 64, 16)
LAYOUTS = [
    (GPT, False, "heads"),
    (GPT, True, "heads"),
    ((32, 8, 128, 32), False, "tokens"),
    ((32, 8, 128, 32), True, "tokens"),
    ((5, 1, 64, 64), False, "slab"),       # one kv head, an odd group
    ((6, 6, 128, 16), True, "slab"),       # every head its own
    ((17, 1, 64, 256), False, "heads"),    # more heads per kv head than a tile has columns
    ((80, 2, 128, 128), False, "tokens"),  # 40 heads per kv head
]
MASKS = [(0, 0, False), (0, 0, True), (128, 0, True), (1, 0, False), (33, 4, True), (200, 70, False)]


@pytest.mark.parametrize("shape,e4m3,layout", LAYOUTS)
@pytest.mark.parametrize("window,first,sink", MASKS)
def test_decode(gpu, shape, e4m3, layout, window, first, sink):
    say("decode", shape, e4m3, layout, window, first, sink)
    c = Case(gpu, 11, [1, 2, 15, 16, 17, 31, 33, 64, 100, 257, 640, 0, 1023], *shape, e4m3=e4m3, layout=layout)
    sinks = randn(c.gen, shape[0], scale=2.0) if sink else None
    _, got = c.check_decode(window, first, sinks)
    assert not got[11].any()  # nothing to see: zeros


@pytest.mark.parametrize("shape,e4m3,layout", LAYOUTS)
@pytest.mark.parametrize("window,first,sink", MASKS)
def test_prefill(gpu, shape, e4m3, layout, window, first, sink):
    say("prefill", shape, e4m3, layout, window, first, sink)
    c = Case(gpu, 12, [1, 40, 129, 300, 77, 210], *shape, e4m3=e4m3, layout=layout)
    sinks = randn(c.gen, shape[0], scale=2.0) if sink else None
    c.check_prefill([1, 40, 1, 33, 70, 17], window, first, sinks)


@pytest.mark.parametrize("B,L", [(1, 1), (1, 5000), (1, 40000), (3, 9000), (70, 300), (200, 40)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_decode_batches_and_long_caches(gpu, B, L, e4m3):
    say("decode", B, L, e4m3)
    lens = [L] + [max(0, (L * (7 * b % 11)) // 11 - 3) for b in range(1, B)]
    c = Case(gpu, 13, lens, *GPT, e4m3=e4m3)
    c.check_decode(sinks=randn(c.gen, 64))
    c.check_decode(window=128)


@pytest.mark.parametrize("B,L", [(63, 3000), (64, 3000), (65, 3000), (257, 2100), (520, 1300)])
def test_decode_ragged_batches(gpu, B, L):
    """Lengths from nothing to L in no order, as many as are found in one, four and more reads."""
    c = Case(gpu, 47, [L * (37 * b % 101) // 101 // (1 + b % 7) + (b == B - 1) * L for b in range(B)], 16, 2, 64, 16)
    c.check_decode(sinks=randn(c.gen, 16))


@pytest.mark.parametrize("B,L", [(1, 1), (1, 6000), (3, 200), (9, 3000), (30, 700)])
@pytest.mark.parametrize("H,Hk", [(8, 8), (40, 2), (64, 8)])
def test_decode_rows_of_half_a_line(gpu, B, L, H, Hk):
    """Token-major rows of 64 bytes, whose lines two heads share."""
    c = Case(gpu, 51, [max(1, L - 97 * b) for b in range(B)], H, Hk, 64, 32, e4m3=True, layout="tokens")
    c.check_decode(sinks=randn(c.gen, H))
    c.check_decode(window=100)


@pytest.mark.parametrize("B,L", [(40, 0), (40, 1500), (100, 1300), (300, 0)])
def test_decode_uniform_batches(gpu, B, L):
    """Many sequences of one length, nothing at all among them, with a table that would hold more."""
    c = Case(gpu, 46, [L] * B, *GPT, width=200)
    q, got = c.check_decode(sinks=randn(c.gen, 64))
    if L:
        c.check_decode()


def test_window_of_every_token_is_none(gpu):
    """A window no sequence can outgrow, up to the largest number, gives the bits of no window."""
    lens = [70, 0, 1000, 2048]
    c = Case(gpu, 61, lens, *GPT)
    for window in (2048, 2 ** 31 - 1):
        q, got = c.check_decode()
        assert got.equal(gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens, window=window, first_tokens=2 ** 31 - 1))
        q, offsets, got = c.check_prefill([70, 0, 90, 1])
        assert got.equal(gpu.paged_attention_prefill(q, offsets, c.cache, c.tables, c.seq_lens, window=window,
                                                     first_tokens=2 ** 31 - 1))


def test_one_workspace_for_fewer_rows(gpu):
    """A workspace sized once for the largest call serves every smaller one."""
    c = Case(gpu, 62, [3000, 900, 2200], *GPT)
    ws = torch.zeros(gpu.paged_attention_workspace_bytes(9000, 3, 64, c.cache), dtype=torch.uint8, device="cuda")
    for new in ([1, 1, 1], [700, 0, 2], [3000, 900, 2200], [40, 40, 40]):
        c.check_prefill(new, workspace=ws)
    c.check_decode(workspace=ws)


@pytest.mark.parametrize("lens,new", [([1000], [1000]), ([2300], [260]), ([700, 5000], [700, 9]), ([64], [64]),
                                      ([300] * 9, [3] * 9), ([4100], [1]), ([90, 0, 91], [0, 0, 91])])
@pytest.mark.parametrize("shape,e4m3", [(GPT, False), (GPT, True), ((32, 8, 128, 32), False), ((4, 4, 64, 16), False),
                                        ((12, 4, 128, 64), True)])
def test_prefill_lengths(gpu, lens, new, shape, e4m3):
    say("prefill", lens, new, shape, e4m3)
    c = Case(gpu, 14, lens, *shape, e4m3=e4m3)
    c.check_prefill(new, sinks=randn(c.gen, shape[0]))
    c.check_prefill(new, window=100, first=5)


def test_weights_of_far_apart_scores(gpu):
    """Scores of a thousand and more: the running maximum moves late, early and not at all."""
    c = Case(gpu, 15, [700, 700, 700], *GPT)
    for b, at in enumerate((0, 350, 699)):
        page = c.tables[b, at // 16].long()
        c.pages[0][page, :, at % 16] *= 300
    c.check_decode(scale=1.0)
    c.check_prefill([700, 20, 1], scale=1.0)


def test_hidden_places_hold_anything(gpu):
    """Pages given back (-1, or a number of no page) and what lies outside of the window or past the end, NaN and
    infinities among it, have no effect; a row that sees nothing is zero, with and without sinks."""
    shape = GPT
    for sink in (False, True):
        c = Case(gpu, 16, [400, 400, 64, 100], *shape)
        sinks = randn(c.gen, 64) if sink else None
        c.tables[0, : 400 // 16 - 9] = -1          # a window's old pages
        c.tables[1, 3] = 1 << 30                   # one page in the middle, of no page's number
        c.tables[1, 7] = -5
        c.tables[2, :] = -1                        # nothing is left
        q, got = c.check_decode(window=128, sinks=sinks)
        assert not got[2].any()
        c.check_decode(sinks=sinks)
        c.check_prefill([30, 100, 64, 1], sinks=sinks)
        _, _, got = c.check_prefill([30, 100, 64, 1], window=50, first=20, sinks=sinks)
        assert not got[130:194].any()
        # infinities beyond the end of a sequence and before its window
        page = c.tables[3, 100 // 16].long()
        c.pages[0][page, :, 100 % 16:] = math.inf
        c.pages[1][page, :, 100 % 16:] = -math.inf
        c.pages[1][c.tables[3, 0].long(), :, :8] = math.inf
        for got in (c.check_decode(window=90, sinks=sinks)[1], c.check_prefill([1, 1, 1, 2], window=91, sinks=sinks)[2]):
            assert torch.isfinite(got).all()


def test_visible_nan_and_infinities_follow_the_formula(gpu):
    c = Case(gpu, 17, [50, 50, 50], *GPT)
    c.pages[0][c.tables[0, 1].long(), 2, 3] = math.nan    # a NaN score: its heads only
    c.pages[1][c.tables[1, 1].long(), 3, 3, 5] = math.inf  # an infinite value: its dim only
    sinks = torch.zeros(64, dtype=BF16, device="cuda")
    sinks[8] = -math.inf                                    # no sink at all
    q = randn(c.gen, 3, 4096)
    off = torch.arange(4, dtype=torch.int32, device="cuda")
    for got in (gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens, sinks=sinks),
                gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens, sinks=sinks)):
        got = got.view(3, 8, 8, 64)
        assert got[0, 2].isnan().all() and got[0, :2].isfinite().all() and got[0, 3:].isfinite().all()
        assert got[1, 3, :, 5].isinf().all() and got[1, 3].isinf().sum() == 8 and got[1].isnan().sum() == 0
        assert got[2].isfinite().all()


@pytest.mark.parametrize("shape,e4m3", [(GPT, False), (GPT, True), ((32, 8, 128, 32), False), ((32, 8, 128, 32), True)])
@pytest.mark.parametrize("window", [0, 30])
def test_values_reach_only_who_sees_them(gpu, shape, e4m3, window):
    """NaN (and, in bf16, infinities) among the values of a prompt: in the rows that see their tokens and in no other,
    also where both lie in one tile."""
    H, Hk, D, bs = shape
    n = 150
    c = Case(gpu, 45, [n], *shape, e4m3=e4m3)
    q = randn(c.gen, n, H * D, scale=1.5)
    off = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    want = gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens, window=window).view(n, H, D).clone()
    marks = [(0, 3, math.nan), (70, 7, math.nan), (100, 5, math.nan if e4m3 else math.inf), (149, 9, math.nan)]
    for t, d, x in marks:
        page = c.tables[0, t // bs].long()
        raw = c.pages[1]
        if e4m3:
            raw.view(torch.uint8)[page, 1, t % bs, d] = 0x7f
        else:
            raw[page, 1, t % bs, d] = x
    got = gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens, window=window).view(n, H, D)
    G = H // Hk
    bad = torch.zeros((n, H, D), dtype=torch.bool, device="cuda")
    for t, d, x in marks:
        rows = slice(t, n if not window else min(n, t + window))
        bad[rows, G:2 * G, d] = True
        if math.isinf(x):
            assert (got[rows, G:2 * G, d] == math.inf).all()
    assert (~got[bad].isfinite()).all()
    assert torch.equal(got[~bad], want[~bad])


# few rows over many tokens: 1, 3 and 4 pieces of the tokens, each shared by two groups of waves
GQA4 = (32, 8, 128, 32)
FEW = [(GPT, 270), (GPT, 90), (GQA4, 540), (GQA4, 180), ((34, 2, 64, 64), 500), ((9, 3, 128, 16), 2700)]


@pytest.mark.parametrize("shape,new", FEW)
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("window,first,sink", [(0, 0, False), (1500, 0, True), (1501, 70, False)])
def test_prefill_few_rows_over_many_tokens(gpu, shape, new, e4m3, window, first, sink):
    say("prefill, few rows", shape, new, e4m3, window, first, sink)
    c = Case(gpu, 48, [2900, 40, max(2101, new)], *shape, e4m3=e4m3)
    c.tables[0, 20] = -1
    c.check_prefill([new // 2, 7, new // 2 + 1], window, first, randn(c.gen, shape[0], scale=2.0) if sink else None)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("window,first,sink", [(0, 0, True), (100, 20, False), (700, 0, True)])
def test_prefill_many_rows(gpu, e4m3, window, first, sink):
    """Enough rows for a wave to take 64 of them."""
    c = Case(gpu, 50, [2000, 1, 1501, 1500], 128, 4, 64, 16, e4m3=e4m3)
    c.tables[2, 5] = -1
    c.check_prefill([1990, 1, 1501, 700], window, first, randn(c.gen, 128, scale=2.0) if sink else None)


@pytest.mark.parametrize("shape,new", FEW[:4] + [((128, 4, 64, 16), 4120)])
def test_values_reach_only_who_sees_them_in_few_rows(gpu, shape, new):
    H, Hk, D, bs = shape
    n, G, window = max(2000, new + 100), H // Hk, 1200
    c = Case(gpu, 49, [n], *shape)
    q = randn(c.gen, new, H * D, scale=1.5)
    off = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    want = gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens, window=window).view(new, H, D).clone()
    bad = torch.zeros((new, H, D), dtype=torch.bool, device="cuda")
    for t, d, x in [(10, 1, math.nan), (max(0, n - new - 1190), 3, math.nan), (n - 1200, 5, math.inf), (n - 60, 7, math.nan),
                    (n - 1, 9, math.inf)]:
        c.pages[1][c.tables[0, t // bs].long(), 1, t % bs, d] = x
        rows = slice(max(0, t - n + new), max(0, min(new, t + window - n + new)))
        bad[rows, G:2 * G, d] = True
    got = gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens, window=window).view(new, H, D)
    assert bad.any() and (~got[bad].isfinite()).all()
    assert torch.equal(got[~bad], want[~bad])


def test_lengths_outside_the_table(gpu):
    """A length past the table's pages is cut to them, a negative one is 0."""
    c = Case(gpu, 18, [64, 48], *GPT)
    q = randn(c.gen, 2, 4096)
    whole = gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens)
    lens = torch.tensor([1 << 30, -7], dtype=torch.int32, device="cuda")
    got = gpu.paged_attention_decode(q, c.cache, c.tables, lens)
    assert torch.equal(got[0], whole[0]) and not got[1].any()
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    got = gpu.paged_attention_prefill(q, off, c.cache, c.tables, lens)
    want, tol = c.want(q, [1, 1])
    assert ref.within(got[:1], want[:1], tol[:1]) is None and not got[1].any()


def test_prefill_rows_outside_and_before(gpu):
    """Rows of no sequence stay as they were; more new rows than tokens: the first ones see nothing."""
    c = Case(gpu, 19, [20, 5], *GPT)
    q = randn(c.gen, 40, 4096)
    out = torch.full((40, 4096), 7.0, dtype=BF16, device="cuda")
    off = torch.tensor([3, 15, 25], dtype=torch.int32, device="cuda")
    gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens, out=out)
    assert (out[:3] == 7).all() and (out[25:] == 7).all()
    assert not out[15:20].any()
    want, tol = c.want(torch.cat((q[3:15], q[20:25])), [12, 5])
    assert ref.within(torch.cat((out[3:15], out[20:25])), want, tol) is None


def test_strided_rows_and_tables(gpu):
    c = Case(gpu, 20, [100, 37, 16], *GPT)
    wide = randn(c.gen, 3, 5120)
    q = wide[:, :4096]
    tables = torch.full((3, c.tables.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    tables[:, : c.tables.shape[1]] = c.tables
    big = torch.full((3, 4096 + 24), 3.0, dtype=BF16, device="cuda")
    want, tol = c.want(q, [1, 1, 1])
    gpu.paged_attention_decode(q, c.cache, tables[:, : c.tables.shape[1]], c.seq_lens, out=big[:, 8:8 + 4096])
    assert ref.within(big[:, 8:8 + 4096], want, tol) is None
    assert (big[:, :8] == 3).all() and (big[:, 8 + 4096:] == 3).all()
    off = torch.arange(4, dtype=torch.int32, device="cuda")
    big.fill_(3.0)
    gpu.paged_attention_prefill(q, off, c.cache, tables[:, : c.tables.shape[1]], c.seq_lens, out=big[:, 8:8 + 4096])
    assert ref.within(big[:, 8:8 + 4096], want, tol) is None
    assert (big[:, :8] == 3).all() and (big[:, 8 + 4096:] == 3).all()


def test_offsets_past_32_bits(gpu):
    """Pages that begin past 2^32 bytes and past 2^31 elements of the cache."""
    H, Hk, D, bs = GPT
    blocks = (1 << 31) // (Hk * bs * D) + 40
    gen = gen_of(21)
    pages = [torch.empty((blocks, Hk, bs, D), dtype=BF16, device="cuda") for _ in range(2)]
    lens = [100, 300]
    tables = torch.full((2, 19), -1, dtype=torch.int32, device="cuda")
    tables[0, :7] = blocks - 1 - torch.arange(7, device="cuda")
    tables[1] = blocks - 9 - torch.arange(19, device="cuda")
    tables[1, 0] = 5
    cache = gpu.KVCache(*pages)
    table = gpu.rope_table()
    for b, n in enumerate(lens):
        qkv = randn(gen, n, (H + 2 * Hk) * D)
        t = torch.arange(n, device="cuda")
        slots = (tables[b, t // bs] * bs + t % bs).to(torch.int32)
        gpu.rope_kv_append(qkv, t.to(torch.int32), slots, table, cache, H)
        assert torch.equal(pages[1][tables[b, t // bs].long(), :, t % bs].reshape(n, -1), qkv[:, (H + Hk) * D:])
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = randn(gen, 40, H * D)
    off = torch.tensor([0, 3, 40], dtype=torch.int32, device="cuda")
    dec = gpu.paged_attention_decode(q[:2].contiguous(), cache, tables, seq_lens)
    pre = gpu.paged_attention_prefill(q, off, cache, tables, seq_lens)
    row = 0
    for b, (n, m) in enumerate(zip(lens, (3, 37))):
        o, t = ref.attend64(q[row:row + m].view(m, H, D), list(range(n - m, n)), n, pages, [None, None], tables[b], bs,
                            D ** -0.5)
        assert ref.within(pre[row:row + m].view(m, H, D), o, t) is None
        o, t = ref.attend64(q[b:b + 1].view(1, H, D), [n - 1], n, pages, [None, None], tables[b], bs, D ** -0.5)
        assert ref.within(dec[b:b + 1].view(1, H, D), o, t) is None
        row += m


def test_results_repeat(gpu):
    """The same call gives the same bits, whatever the workspace held."""
    c = Case(gpu, 22, [9000, 100, 2500], *GPT)
    q = randn(c.gen, 3, 4096)
    need = gpu.paged_attention_workspace_bytes(3, 3, 64, c.cache)
    off = torch.arange(4, dtype=torch.int32, device="cuda")
    for call in (lambda **k: gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens, **k),
                 lambda **k: gpu.paged_attention_prefill(q, off, c.cache, c.tables, c.seq_lens, **k)):
        first = call()
        for fill in (0, 255):
            ws = torch.full((max(need, 1),), fill, dtype=torch.uint8, device="cuda")
            assert torch.equal(call(workspace=ws), first)


# ---------------------------------------------------------------------------
# the rotation and the append
# ---------------------------------------------------------------------------
def yarn64(cfg, pos):
    """cos and sin [n, rotary / 2] in 64 bits."""
    half = cfg.rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    f = cfg.theta ** (-2 * i / cfg.rotary_dim)
    m = 1.0
    if cfg.scaling_factor != 1:
        turn = lambda r: half * math.log(cfg.original_positions / (r * 2 * math.pi)) / math.log(cfg.theta)  # noqa: E731
        low, high = turn(cfg.beta_fast), turn(cfg.beta_slow)
        ramp = ((i - low) / (high - low)).clamp(0, 1)
        f = (1 - ramp) * f + ramp * f / cfg.scaling_factor
        m = 0.1 * math.log(cfg.scaling_factor) + 1
    a = pos.double()[:, None] * f
    return a.cos() * m, a.sin() * m


@pytest.mark.parametrize("rotary,factor,theta,positions", [(64, 32.0, 150000.0, 131072), (128, 1.0, 10000.0, 5000),
                                                           (16, 8.0, 500000.0, 33)])
def test_rope_table(gpu, rotary, factor, theta, positions):
    cfg = gpu.default_rope_config()
    cfg.rotary_dim, cfg.scaling_factor, cfg.theta, cfg.max_positions = rotary, factor, theta, positions
    table = gpu.rope_table(cfg)
    cos, sin = yarn64(cfg, torch.arange(positions, device="cuda"))
    m = 0.1 * math.log(factor) + 1
    # one fp32 rounding of a value up to m, and 64-bit angles (up to 131072 rad, to 2^-53 of that, twice over)
    tol = 2.0 ** -24 * m * 1.01 + 4 * positions * 2.0 ** -53
    assert (table[:, 0].double() - cos).abs().max() <= tol
    assert (table[:, 1].double() - sin).abs().max() <= tol


@pytest.mark.parametrize("T", [1, 2, 63, 300])
@pytest.mark.parametrize("shape,e4m3,layout,rotary,pairs", [
    (GPT, False, "heads", 64, False), (GPT, True, "heads", 64, False), ((32, 8, 128, 32), True, "tokens", 128, True),
    ((32, 8, 128, 32), False, "tokens", 32, False), ((5, 1, 64, 64), False, "slab", 16, True),
    ((6, 6, 128, 16), True, "slab", 48, False), ((7, 7, 64, 16), True, "heads", 64, True)])
def test_append(gpu, T, shape, e4m3, layout, rotary, pairs):
    say("append", T, shape, e4m3, layout, rotary, pairs)
    H, Hk, D, bs = shape
    gen = gen_of(31)
    blocks = (T + bs - 1) // bs + 3
    # finite codes everywhere, so that what is kept can be compared
    pages, scales = ref.make_cache(gen, blocks, Hk, bs, D, e4m3, layout, fill=0.5)
    before = [p.clone() for p in pages]
    cache = gpu.KVCache(pages[0], pages[1], scales[0], scales[1])
    cfg = gpu.default_rope_config()
    cfg.rotary_dim = rotary
    table = gpu.rope_table(cfg)
    wide = randn(gen, T, (H + 2 * Hk) * D + 16)
    qkv = wide[:, : (H + 2 * Hk) * D]
    qkv[0, H * D] = 1000.0  # past an 8-bit cache's largest value
    pos = torch.randint(0, cfg.max_positions, (T,), generator=gen, device="cuda").to(torch.int32)
    slots = torch.randperm(blocks * bs, generator=gen, device="cuda")[:T].to(torch.int32)
    if T > 60:
        slots[5], slots[7], slots[9] = -1, blocks * bs, -(1 << 31)
        pos[11], pos[13] = -1, cfg.max_positions
    q_out = torch.full((T, H * D), 9.0, dtype=BF16, device="cuda")
    got = gpu.rope_kv_append(qkv, pos, slots, table, cache, H, interleaved=pairs, q_out=q_out)
    torch.cuda.synchronize()
    assert got is q_out
    turned = (pos >= 0) & (pos < cfg.max_positions)
    cos, sin = yarn64(cfg, pos)
    x = qkv.double().view(T, H + 2 * Hk, D)
    y, slack = x.clone(), torch.zeros_like(x)
    half = torch.arange(rotary // 2, device="cuda")
    ia, ib = (2 * half, 2 * half + 1) if pairs else (half, half + rotary // 2)
    a, b = x[:, : H + Hk, ia], x[:, : H + Hk, ib]
    c, s = cos[:, None], sin[:, None]
    y[:, : H + Hk, ia], y[:, : H + Hk, ib] = a * c - b * s, b * c + a * s
    # table, products and their sum: three fp32 roundings of terms up to |a c| + |b s|
    for i, v in ((ia, a.abs() * c.abs() + b.abs() * s.abs()), (ib, b.abs() * c.abs() + a.abs() * s.abs())):
        slack[:, : H + Hk, i] = 4 * 2.0 ** -24 * v + 2.0 ** -30 * (a.abs() + b.abs())
    want = y[:, :H].reshape(T, -1)
    tol = want.abs() * 2.0 ** -8 + slack[:, :H].reshape(T, -1)
    bad = ref.within(q_out[turned], want[turned], tol[turned])
    assert bad is None, bad
    assert (q_out[~turned] == 9).all()
    stored = turned & (slots >= 0) & (slots < blocks * bs)
    page, place = (slots[stored] // bs).long(), (slots[stored] % bs).long()
    for n, (p, was, sc) in enumerate(zip(pages, before, scales)):
        want, sl = y[stored, H + n * Hk:H + (n + 1) * Hk], slack[stored, H + n * Hk:H + (n + 1) * Hk]
        raw = p.view(torch.uint8) if e4m3 else p
        got = raw[page, :, place].view(p.dtype).double()
        if e4m3:
            want, sl = want / sc.double()[:, None], sl / sc.double()[:, None]
            # half a step of three mantissa bits, or of the smallest values' 2^-9; the division rounds in fp32
            tol = (want.abs() * (2.0 ** -4 + 2.0 ** -22)).clamp(min=2.0 ** -10) + 1.1 * sl
            want = want.clamp(-448, 448)
        else:
            tol = want.abs() * 2.0 ** -8 + sl
        bad = ref.within(got, want, tol)
        assert bad is None, bad
        keep = torch.ones((blocks, bs), dtype=torch.bool, device="cuda")
        keep[page, place] = False
        same = (raw == (was.view(torch.uint8) if e4m3 else was)).all(3).transpose(1, 2)  # [block][slot][head]
        assert same[keep].all()


def test_append_in_place(gpu):
    """The queries may be turned where they lie."""
    gen = gen_of(33)
    H, Hk, D, bs = GPT
    pages, _ = ref.make_cache(gen, 4, Hk, bs, D, False, fill=0.0)
    cache, table = gpu.KVCache(*pages), gpu.rope_table()
    for T in (1, 40):
        qkv = randn(gen, T, (H + 2 * Hk) * D)
        pos = torch.arange(T, dtype=torch.int32, device="cuda") + 70000
        slots = torch.arange(T, dtype=torch.int32, device="cuda")
        for pairs in (False, True):
            apart = gpu.rope_kv_append(qkv.clone(), pos, slots, table, cache, H, interleaved=pairs)
            k = pages[0].clone()
            mine = qkv.clone()
            got = gpu.rope_kv_append(mine, pos, slots, table, cache, H, interleaved=pairs, q_out=mine[:, :H * D])
            assert got.data_ptr() == mine.data_ptr()
            assert torch.equal(got, apart) and torch.equal(mine[:, H * D:], qkv[:, H * D:]) and torch.equal(pages[0], k)


def test_append_keeps_nan(gpu):
    gen = gen_of(34)
    H, Hk, D, bs = GPT
    pages, scales = ref.make_cache(gen, 2, Hk, bs, D, True, fill=0.0)
    cache = gpu.KVCache(pages[0], pages[1], scales[0], None)
    qkv = randn(gen, 1, (H + 2 * Hk) * D)
    v = qkv.view(-1, D)[H + Hk:]
    v[0, 3], v[0, 4], v[0, 5] = math.nan, math.inf, -math.inf
    one = torch.tensor([3], dtype=torch.int32, device="cuda")
    gpu.rope_kv_append(qkv, one, one, gpu.rope_table(), cache, H)
    got = pages[1].float()[0, 0, 3]
    assert got[3].isnan() and got[4] == 448 and got[5] == -448


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("shape,e4m3,window", [(GPT, False, 0), (GPT, False, 40), ((32, 8, 128, 32), True, 0)])
def test_prompt_then_steps(gpu, shape, e4m3, window):
    """A prompt in chunks, then single tokens: every step's attention over what the appends stored."""
    H, Hk, D, bs = shape
    gen = gen_of(41)
    lens = [0, 0, 0]
    chunks = [[70, 1, 33], [50, 20, 0], [1, 1, 1], [1, 1, 1]]
    blocks, width = 40, 13
    pages, scales = ref.make_cache(gen, blocks, Hk, bs, D, e4m3)
    tables = torch.randperm(blocks, generator=gen, device="cuda")[:39].view(3, 13).to(torch.int32).contiguous()
    cache = gpu.KVCache(pages[0], pages[1], scales[0], scales[1])
    cfg = gpu.default_rope_config()
    cfg.rotary_dim = D
    table = gpu.rope_table(cfg)
    sinks = randn(gen, H)
    for step in chunks:
        rows = sum(step)
        qkv = randn(gen, rows, (H + 2 * Hk) * D)
        seq = torch.tensor([b for b, n in enumerate(step) for _ in range(n)], device="cuda")
        pos = torch.tensor([lens[b] + i for b, n in enumerate(step) for i in range(n)], device="cuda")
        slots = tables[seq, pos // bs] * bs + pos % bs
        q = gpu.rope_kv_append(qkv, pos.to(torch.int32), slots.to(torch.int32), table, cache, H)
        lens = [a + n for a, n in zip(lens, step)]
        seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        off = torch.tensor([0] + step, device="cuda").cumsum(0).to(torch.int32)
        outs = [gpu.paged_attention_prefill(q, off, cache, tables, seq_lens, window=window, sinks=sinks)]
        if step == [1, 1, 1]:
            outs.append(gpu.paged_attention_decode(q, cache, tables, seq_lens, window=window, sinks=sinks))
        row = 0
        for b, n in enumerate(step):
            o, t = ref.attend64(q[row:row + n].view(n, H, D), list(range(lens[b] - n, lens[b])), lens[b], pages, scales,
                                tables[b], bs, D ** -0.5, window, 0, sinks)
            for out in outs:
                bad = ref.within(out[row:row + n].view(n, H, D), o, t)
                assert bad is None, (step, b, bad)
            row += n


def test_captured_step_follows_its_buffers(gpu):
    """Append and decode captured once: replays follow positions, slots and lengths, with eager work and
    synchronizations in between; two graphs with a workspace each may run at the same time."""
    H, Hk, D, bs = GPT
    B, n0 = 3, [5, 2000, 130]
    c = Case(gpu, 42, [n + 40 for n in n0], *GPT)
    table = gpu.rope_table()
    need = gpu.paged_attention_workspace_bytes(B, B, H, c.cache)

    class Step:
        def __init__(self):
            self.qkv = torch.zeros((B, (H + 2 * Hk) * D), dtype=BF16, device="cuda")
            self.pos, self.slots, self.lens = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(3))
            self.q, self.out = (torch.zeros((B, H * D), dtype=BF16, device="cuda") for _ in range(2))
            self.ws = torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda")

        def run(self):
            gpu.rope_kv_append(self.qkv, self.pos, self.slots, table, c.cache, H, q_out=self.q)
            gpu.paged_attention_decode(self.q, c.cache, c.tables, self.lens, out=self.out, workspace=self.ws)

        def set(self, step, seed):
            pos = torch.tensor([n + step for n in n0], device="cuda")
            self.qkv.copy_(randn(gen_of(seed), B, (H + 2 * Hk) * D))
            self.pos.copy_(pos)
            self.slots.copy_(c.tables[torch.arange(B, device="cuda"), pos // bs] * bs + pos % bs)
            self.lens.copy_(pos + 1)

    a, eager = Step(), Step()
    a.set(0, 100)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.run()
    for step in range(5):
        a.set(step, 100 + step)
        graph.replay()
        torch.cuda.synchronize()
        got = a.out.clone()
        eager.set(step, 100 + step)
        eager.run()
        assert torch.equal(got, eager.out), step
        q64, tol = ref.attend64(a.q[1:2].view(1, H, D), [n0[1] + step], n0[1] + step + 1, c.pages, c.scales, c.tables[1],
                                bs, D ** -0.5)
        assert ref.within(got[1:2].view(1, H, D), q64, tol) is None
    # two decodes at once, each with its workspace
    other = Step()
    other.set(4, 104)
    other.q.copy_(a.q)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(20):
            gpu.paged_attention_decode(other.q, c.cache, c.tables, other.lens, out=other.out, workspace=other.ws)
    for _ in range(20):
        gpu.paged_attention_decode(a.q, c.cache, c.tables, a.lens, out=a.out, workspace=a.ws)
    torch.cuda.synchronize()
    assert torch.equal(a.out, other.out) and torch.equal(a.out, got)


def test_captured_prompt_follows_its_buffers(gpu):
    """A captured prompt chunk: replays follow offsets and lengths, whatever its pieces were joined from before; eager
    calls of the same workspace's size run between them and on another stream beside them."""
    c = Case(gpu, 52, [2600, 1900, 700], *GPT)
    rows = 100
    ws, beside = (torch.zeros(gpu.paged_attention_workspace_bytes(rows, 3, 64, c.cache), dtype=torch.uint8, device="cuda")
                  for _ in range(2))
    q, off = torch.zeros((rows, 4096), dtype=BF16, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    lens, out = c.seq_lens.clone(), torch.zeros((rows, 4096), dtype=BF16, device="cuda")

    def run(out, ws):
        gpu.paged_attention_prefill(q, off, c.cache, c.tables, lens, window=0, out=out, workspace=ws)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        run(out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(out, ws)
    for step, (new, ends) in enumerate([([100, 0, 0], [2600, 5, 5]), ([1, 98, 1], [2600, 1900, 700]),
                                        ([40, 40, 20], [64, 1900, 20]), ([0, 0, 100], [1, 1, 700]),
                                        ([33, 33, 34], [2600, 1900, 700])]):
        q.copy_(randn(gen_of(300 + step), rows, 4096))
        off.copy_(torch.tensor([0] + new).cumsum(0))
        lens.copy_(torch.tensor(ends))
        torch.cuda.synchronize()
        want = torch.zeros_like(out)
        with torch.cuda.stream(s):
            run(want, beside)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), step
        c.lens = ends
        o, tol = c.want(q, new)
        assert ref.within(out, o, tol) is None, step


def test_many_sequences(gpu):
    """Thousands of sequences in one call, most of them without a new token in a prompt's."""
    B = 5000
    lens = [1 + 37 * b % 90 for b in range(B)]
    lens[77], lens[4321] = 2000, 1100
    c = Case(gpu, 53, lens, 8, 1, 64, 16)
    q = randn(c.gen, B, 512, scale=1.5)
    got = gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens)
    new = [0] * B
    picked = [0, 63, 64, 77, 255, 256, 1000, 4321, B - 1]
    for b in picked:
        new[b] = min(lens[b], 20)
    rows = sum(new)
    p = randn(c.gen, rows, 512, scale=1.5)
    off = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    chunk = gpu.paged_attention_prefill(p, off, c.cache, c.tables, c.seq_lens)
    torch.cuda.synchronize()
    for b in picked:
        n, at = lens[b], int(off[b])
        for x, out, pos in ((q[b:b + 1], got[b:b + 1], [n - 1]), (p[at:at + new[b]], chunk[at:at + new[b]], range(n - new[b], n))):
            o, tol = ref.attend64(x.view(-1, 8, 64), list(pos), n, c.pages, c.scales, c.tables[b], 16, 0.125)
            assert ref.within(out.view(-1, 8, 64), o, tol) is None, b


def test_on_a_given_stream(gpu):
    """stream= runs the call there, on buffers that it allocates there."""
    c = Case(gpu, 43, [3000, 100], *GPT)
    q = randn(c.gen, 2, 4096)
    want = gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream, 0):
        got = gpu.paged_attention_decode(q, c.cache, c.tables, c.seq_lens, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_empty_calls(gpu):
    c = Case(gpu, 44, [10], *GPT)
    none = torch.empty((0, 4096), dtype=BF16, device="cuda")
    no = torch.empty((0,), dtype=torch.int32, device="cuda")
    tables = torch.empty((0, 4), dtype=torch.int32, device="cuda")
    assert gpu.paged_attention_decode(none, c.cache, tables, no).shape == (0, 4096)
    off = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert gpu.paged_attention_prefill(none, off, c.cache, c.tables, c.seq_lens).shape == (0, 4096)
    qkv = torch.empty((0, 5120), dtype=BF16, device="cuda")
    assert gpu.rope_kv_append(qkv, no, no, gpu.rope_table(), c.cache, 64).shape == (0, 4096)
