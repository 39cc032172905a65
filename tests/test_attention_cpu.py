"""CPU tests of the attention operators: what the C ABI and the Python binding refuse.  None of these calls
reaches a kernel launch."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def g():
    import gptoss_moe
    return gptoss_moe


A = 1 << 20  # an aligned address that no call here reads


def cache(g, **kw):
    d = g.KvCacheDesc(A, 2 * A, None, None, 0, 0, 0, g.GPTOSS_KV_BF16, 100, 16, 8, 64)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def decode(g, desc, cfg=None, **kw):
    a = dict(q=4 * A, q_stride=4096, tables=8 * A, table_stride=10, max_blocks=10, lens=9 * A, B=3, H=64, out=5 * A,
             out_stride=4096, ws=16 * A, ws_bytes=1 << 40)
    a.update(kw)
    c = g.AttentionConfig(0.125, 0, 0, None) if cfg is None else cfg
    return g.lib.gptoss_paged_attention_decode(a["q"], a["q_stride"], ctypes.byref(desc) if desc else None, a["tables"],
                                               a["table_stride"], a["max_blocks"], a["lens"], a["B"], a["H"],
                                               ctypes.byref(c) if c else None, a["out"], a["out_stride"], a["ws"],
                                               a["ws_bytes"], None)


def prefill(g, desc, cfg=None, **kw):
    a = dict(q=4 * A, q_stride=4096, off=7 * A, T=20, tables=8 * A, table_stride=10, max_blocks=10, lens=9 * A, B=3, H=64,
             out=5 * A, out_stride=4096, ws=16 * A, ws_bytes=1 << 40)
    a.update(kw)
    c = g.AttentionConfig(0.125, 0, 0, None) if cfg is None else cfg
    return g.lib.gptoss_paged_attention_prefill(a["q"], a["q_stride"], a["off"], a["T"], ctypes.byref(desc), a["tables"],
                                                a["table_stride"], a["max_blocks"], a["lens"], a["B"], a["H"],
                                                ctypes.byref(c), a["out"], a["out_stride"], a["ws"], a["ws_bytes"], None)


def append(g, desc, **kw):
    a = dict(qkv=4 * A, stride=5120, pos=8 * A, slots=9 * A, table=10 * A, rotary=64, positions=1000, pairs=0, T=7, H=64,
             q=6 * A, q_stride=4096)
    a.update(kw)
    return g.lib.gptoss_rope_kv_append(a["qkv"], a["stride"], a["pos"], a["slots"], a["table"], a["rotary"], a["positions"],
                                       a["pairs"], a["T"], a["H"], a["q"], a["q_stride"], ctypes.byref(desc), None)


CACHES = [
    (dict(dtype=7), "INVALID", b"dtype"),
    (dict(head_dim=96), "UNSUPPORTED", b"head_dim"),
    (dict(block_size=24), "UNSUPPORTED", b"block_size"),
    (dict(block_size=8), "UNSUPPORTED", b"block_size"),
    (dict(block_size=512), "UNSUPPORTED", b"block_size"),
    (dict(num_kv_heads=0), "INVALID", b"num_kv_heads"),
    (dict(num_blocks=0), "INVALID", b"num_blocks"),
    (dict(num_blocks=1 << 28), "UNSUPPORTED", b"slots"),
    (dict(k=None), "INVALID", b"null cache"),
    (dict(v=A + 8), "INVALID", b"aligned"),
    (dict(k_scale=A), "INVALID", b"no scales"),
    (dict(block_stride=8192, head_stride=1024, token_stride=32), "INVALID", b"strides"),
    (dict(block_stride=8192, head_stride=1028, token_stride=64), "INVALID", b"strides"),
    (dict(block_stride=-8192, head_stride=1024, token_stride=64), "INVALID", b"strides"),
    (dict(dtype=1, block_stride=8192, head_stride=1032, token_stride=64), "INVALID", b"strides"),
    (dict(num_kv_heads=7), "INVALID", b"num_heads"),
]


@pytest.mark.parametrize("change,code,message", CACHES)
def test_caches_refused(g, change, code, message):
    for call in (decode, prefill, append):
        assert call(g, cache(g, **change)) == getattr(g, "GPTOSS_ERR_" + code)
        assert message in g.lib.gptoss_last_error()


def test_null_cache_and_config(g):
    assert decode(g, None) == g.GPTOSS_ERR_INVALID and b"cache" in g.lib.gptoss_last_error()
    rc = g.lib.gptoss_paged_attention_decode(4 * A, 4096, ctypes.byref(cache(g)), 8 * A, 10, 10, 9 * A, 3, 64, None, 5 * A,
                                             4096, 16 * A, 1 << 40, None)
    assert rc == g.GPTOSS_ERR_INVALID and b"cfg" in g.lib.gptoss_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(q=None), b"null q"), (dict(q=4 * A + 2), b"aligned"), (dict(q_stride=4088), b"q: rows"),
    (dict(q_stride=4100), b"multiple of 8"), (dict(out=None), b"null out"), (dict(out_stride=64), b"out: rows"),
    (dict(out=4 * A), b"overlaps"), (dict(out=4 * A + 4096), b"overlaps"), (dict(tables=None), b"null block_tables"),
    (dict(lens=None), b"seq_lens"), (dict(max_blocks=0), b"max_blocks"), (dict(table_stride=9), b"table_stride"),
    (dict(B=-1), b"num_seqs"), (dict(H=0), b"num_heads"), (dict(H=60), b"num_heads")])
def test_attention_arguments_refused(g, change, message):
    for call in (decode, prefill):
        assert call(g, cache(g), **change) == g.GPTOSS_ERR_INVALID, change
        assert message in g.lib.gptoss_last_error()


def test_prefill_arguments_refused(g):
    assert prefill(g, cache(g), T=-1) == g.GPTOSS_ERR_INVALID
    assert prefill(g, cache(g), off=None) == g.GPTOSS_ERR_INVALID and b"query_offsets" in g.lib.gptoss_last_error()
    assert prefill(g, cache(g), T=1 << 26, q=1 << 44, out=1 << 50, ws_bytes=1 << 62) == g.GPTOSS_ERR_UNSUPPORTED
    assert decode(g, cache(g, num_kv_heads=1), H=129, q_stride=129 * 64, out_stride=129 * 64) == g.GPTOSS_ERR_UNSUPPORTED


@pytest.mark.parametrize("cfg", [(0.0, 0, 0), (-1.0, 0, 0), (float("nan"), 0, 0), (float("inf"), 0, 0), (3e38, 0, 0), (1.0, -1, 0),
                                 (1.0, 4, -1)])
def test_attention_config_refused(g, cfg):
    for call in (decode, prefill):
        assert call(g, cache(g), g.AttentionConfig(*cfg, None)) == g.GPTOSS_ERR_INVALID


def test_nothing_to_do(g):
    assert decode(g, cache(g), B=0, q=None, out=None, tables=None, lens=None, max_blocks=0, ws=None) == g.GPTOSS_OK
    assert prefill(g, cache(g), T=0, q=None, out=None, off=None, ws=None) == g.GPTOSS_OK
    assert prefill(g, cache(g), B=0, tables=None, lens=None, off=None, ws=None) == g.GPTOSS_OK
    assert append(g, cache(g), T=0, qkv=None, q=None, pos=None, slots=None) == g.GPTOSS_OK


@pytest.mark.parametrize("change,message", [
    (dict(T=-1), b"num_tokens"), (dict(rotary=0), b"rotary_dim"), (dict(rotary=24), b"rotary_dim"),
    (dict(rotary=80), b"rotary_dim"), (dict(positions=0), b"max_positions"), (dict(qkv=None), b"null qkv"),
    (dict(stride=5112), b"qkv: rows"), (dict(stride=5124), b"multiple of 8"), (dict(q_stride=4090), b"q_out: rows"),
    (dict(pos=None), b"positions"), (dict(slots=None), b"slots"), (dict(table=None), b"rope_table"),
    (dict(table=A + 4), b"aligned"), (dict(q=4 * A), b"overlaps"), (dict(q=4 * A + 16, q_stride=5120), b"overlaps"),
    (dict(H=60), b"num_heads")])
def test_append_arguments_refused(g, change, message):
    assert append(g, cache(g), **change) == g.GPTOSS_ERR_INVALID, change
    assert message in g.lib.gptoss_last_error()


@pytest.mark.parametrize("change", [dict(rotary_dim=0), dict(rotary_dim=20), dict(max_positions=0), dict(theta=1.0),
                                    dict(theta=float("nan")), dict(scaling_factor=0.5), dict(original_positions=0.0),
                                    dict(beta_fast=-1.0), dict(beta_slow=float("nan"))])
def test_rope_table_refused(g, change):
    cfg = g.default_rope_config()
    assert (cfg.rotary_dim, cfg.max_positions, cfg.theta, cfg.scaling_factor) == (64, 131072, 150000.0, 32.0)
    assert (cfg.original_positions, cfg.beta_fast, cfg.beta_slow) == (4096.0, 32.0, 1.0)
    for k, v in change.items():
        setattr(cfg, k, v)
    assert g.lib.gptoss_rope_table(ctypes.byref(cfg), A, None) == g.GPTOSS_ERR_INVALID
    assert g.lib.gptoss_rope_table(ctypes.byref(g.default_rope_config()), None, None) == g.GPTOSS_ERR_INVALID
    assert g.lib.gptoss_rope_config_default(None) == g.GPTOSS_ERR_INVALID


def test_workspace_refused(g):
    """Calls that are cut: less than they need, none, and one that is not aligned."""
    wide = dict(max_blocks=2000, table_stride=2000)
    for call, T in ((decode, 0), (prefill, 20)):
        need = g.lib.gptoss_paged_attention_call_bytes(T, 3, 64, 8, 64, 32000, 0, 0)
        assert 0 < need <= g.lib.gptoss_paged_attention_workspace_bytes(max(T, 3), 3, 64, 8, 64)
        assert call(g, cache(g), ws_bytes=need - 1, **wide) == g.GPTOSS_ERR_INVALID and b"workspace" in g.lib.gptoss_last_error()
        assert call(g, cache(g), ws=None, **wide) == g.GPTOSS_ERR_INVALID
        assert call(g, cache(g), ws=16 * A + 8, **wide) == g.GPTOSS_ERR_INVALID and b"aligned" in g.lib.gptoss_last_error()


@pytest.mark.parametrize("H,Hk,D", [(64, 8, 64), (32, 8, 128), (5, 1, 64), (128, 1, 128), (6, 6, 128), (1, 1, 64)])
def test_call_bytes(g, H, Hk, D):
    """No call needs more than the workspace for its counts; short ones need none."""
    one, top = g.lib.gptoss_paged_attention_call_bytes, g.lib.gptoss_paged_attention_workspace_bytes
    for B in (1, 2, 7, 64, 700):
        for tokens in (1, 512, 513, 1024, 1025, 4000, 131072, 1 << 30):
            for window, first in ((0, 0), (128, 0), (3000, 4), (2 ** 31 - 1, 2 ** 31 - 1)):
                assert one(0, B, H, Hk, D, tokens, window, first) <= top(B, B, H, Hk, D)
                for T in (1, B, 90, 680, 5000):
                    assert one(T, B, H, Hk, D, tokens, window, first) <= top(T, B, H, Hk, D)
    assert one(0, 3, H, Hk, D, 512, 0, 0) == one(20, 3, H, Hk, D, 400, 0, 0) == 0
    for bad in ((-1, 1, H, Hk, D, 9, 0, 0), (0, 0, H, Hk, D, 9, 0, 0), (0, 1, H, 0, D, 9, 0, 0), (0, 1, H, Hk, D, 0, 0, 0),
                (0, 1, H, Hk, D, 9999, -1, 0), (0, 1, H, Hk, D, 1 << 40, 0, 0)):
        assert one(*bad) == 0


@pytest.mark.parametrize("H,Hk,D", [(64, 8, 64), (32, 8, 128), (5, 1, 64), (128, 1, 128), (6, 6, 128), (1, 1, 64)])
def test_workspace_is_enough_for_smaller_calls(g, H, Hk, D):
    size = lambda T, B: g.lib.gptoss_paged_attention_workspace_bytes(T, B, H, Hk, D)
    sizes = [size(T, 1) for T in range(1, 3000)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert [size(4096, B) for B in range(1, 300)] == sorted(size(4096, B) for B in range(1, 300))
    assert size(0, 1) == size(1, 0) == 0
    big = 2 ** 31 - 1
    assert g.lib.gptoss_paged_attention_workspace_bytes(big, big, big, big, D) == 0
    assert g.lib.gptoss_paged_attention_workspace_bytes(big, big, big, 1, D) == 0
    assert size(big, big) > 0


def test_limits_refused(g):
    def refused(rc, message):
        assert rc == g.GPTOSS_ERR_UNSUPPORTED and message in g.lib.gptoss_last_error()

    far = dict(out=1 << 60, ws=1 << 62, ws_bytes=1 << 62)
    refused(decode(g, cache(g), B=(1 << 16) + 1, **far), b"sequences of 64 heads")
    refused(prefill(g, cache(g), T=(1 << 20) + 1, **far), b"rows and")
    refused(prefill(g, cache(g), B=(1 << 16) + 1, **far), b"sequences of 64 heads")
    for call in (decode, prefill):
        refused(call(g, cache(g), max_blocks=(1 << 26) + 1, table_stride=1 << 27, B=1, T=1, **far), b"tables of")
        refused(call(g, cache(g), max_blocks=1 << 26, table_stride=1 << 27, B=33, T=33, **far), b"tables of")
        refused(call(g, cache(g, token_stride=(1 << 24) + 64, head_stride=64, block_stride=64), **far), b"token_stride")
    refused(append(g, cache(g), T=(1 << 25) + 1, q=1 << 60), b"rows in one call")


# ---------------------------------------------------------------------------
# the binding
# ---------------------------------------------------------------------------
def pages(dtype=torch.bfloat16, shape=(6, 8, 16, 64)):
    return torch.zeros(shape).to(dtype)


def test_kv_cache_tensors(g):
    e4m3 = torch.float8_e4m3fn
    ones = torch.ones(8)
    c = g.KVCache(pages(e4m3), pages(e4m3), ones, None)
    assert (c.desc.block_stride, c.desc.head_stride, c.desc.token_stride) == (8192, 1024, 64)
    tok = pages(shape=(6, 16, 8, 64)).permute(0, 2, 1, 3), pages(shape=(6, 16, 8, 64)).permute(0, 2, 1, 3)
    c = g.KVCache(*tok)
    assert (c.num_blocks, c.kv_heads, c.block_size, c.head_dim) == (6, 8, 16, 64)
    assert (c.desc.block_stride, c.desc.head_stride, c.desc.token_stride) == (8192, 64, 512)
    slab = pages(shape=(6, 2, 8, 16, 64))
    assert g.KVCache(slab[:, 0], slab[:, 1]).desc.block_stride == 16384
    one = g.KVCache(pages(shape=(1, 1, 16, 64)), pages(shape=(1, 1, 16, 64)))
    assert one.desc.token_stride == 64
    for bad in [
        (pages(torch.float32), pages(torch.float32)), (pages(), pages(e4m3)), (pages(), pages(shape=(5, 8, 16, 64))),
        (pages(), tok[0]), (pages()[0], pages()[0]), (pages(shape=(0, 8, 16, 64)),) * 2,
        (pages(shape=(6, 8, 64, 16)).transpose(2, 3),) * 2, (pages(shape=(1, 8, 16, 64)).expand(6, 8, 16, 64),) * 2,
        (pages(), pages(), ones), (pages(e4m3), pages(e4m3), torch.ones(7)), (pages(e4m3), pages(e4m3), ones.double()),
        (torch.as_strided(pages(), (6, 8, 16, 64), (8192, 512, 64, 1)),) * 2,
    ]:
        with pytest.raises(ValueError):
            g.KVCache(*bad)


def test_binding_refuses(g):
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    c = g.KVCache(pages(), pages())
    q, t, n = bf(3, 4096), i32(3, 5), i32(3)
    cases = [
        (lambda: g.paged_attention_decode(q, c, t, n), "GPU is needed"),
        (lambda: g.paged_attention_prefill(q, i32(4), c, t, n), "GPU is needed"),
        (lambda: g.rope_kv_append(bf(3, 5120), n, n, torch.zeros(9, 2, 32), c, 64), "GPU is needed"),
        (lambda: g.paged_attention_decode(q.float(), c, t, n), "dtype"),
        (lambda: g.paged_attention_decode(bf(3, 4095), c, t, n), "num_heads"),
        (lambda: g.paged_attention_decode(bf(4096, 3).T, c, t, n), "contiguous"),
        (lambda: g.paged_attention_decode(bf(1, 4096).expand(3, 4096), c, t, n), "contiguous"),
        (lambda: g.paged_attention_decode(bf(2, 4096), c, t, n), "rows"),
        (lambda: g.paged_attention_decode(q, c, t.long(), n), "dtype"),
        (lambda: g.paged_attention_decode(q, c, i32(5, 3).T, n), "contiguous"),
        (lambda: g.paged_attention_decode(q, c, t, i32(4)), "entries"),
        (lambda: g.paged_attention_decode(q, c, t, i32(6)[::2]), "contiguous"),
        (lambda: g.paged_attention_decode(q, c, t, n, sinks=bf(8)), "entries"),
        (lambda: g.paged_attention_decode(q, c, t, n, sinks=torch.zeros(64)), "dtype"),
        (lambda: g.paged_attention_decode(q, c, t, n, out=bf(2, 4096)), "rows"),
        (lambda: g.paged_attention_decode(q, c, t, n, out=bf(3, 64)), "shape"),
        (lambda: g.paged_attention_prefill(q, None, c, t, n), "query_offsets"),
        (lambda: g.paged_attention_prefill(q, i32(3), c, t, n), "entries"),
        (lambda: g.rope_kv_append(bf(3, 4096), n, n, torch.zeros(9, 2, 32), c, 64), "shape"),
        (lambda: g.rope_kv_append(bf(3, 5120), n, i32(2), torch.zeros(9, 2, 32), c, 64), "entries"),
        (lambda: g.rope_kv_append(bf(3, 5120), n, n, torch.zeros(9, 64), c, 64), "3-D"),
        (lambda: g.rope_kv_append(bf(3, 5120), n, n, torch.zeros(9, 3, 32), c, 64), "table"),
        (lambda: g.rope_kv_append(bf(3, 5120), n, n, torch.zeros(9, 2, 32), c, 64, q_out=bf(2, 4096)), "rows"),
    ]
    for call, message in cases:
        with pytest.raises(ValueError, match=message):
            call()
