"""CPU tests: further calls that the attention operators refuse, and what their host side answers.  None of these calls
reaches a kernel launch."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def g():
    import gptoss_moe
    return gptoss_moe


A = 1 << 20  # an aligned address that no call here reads


@pytest.mark.parametrize("change", [dict(beta_fast=float("inf")), dict(beta_fast=1e308),
                                    dict(beta_fast=1e300, original_positions=1e-30),
                                    dict(beta_fast=float("inf"), original_positions=float("inf"))])
def test_rope_ramp_without_a_beginning_refused(g, change):
    """Frequencies would be NaN: the ramp begins infinitely far away."""
    cfg = g.default_rope_config()
    for k, v in change.items():
        setattr(cfg, k, v)
    assert g.lib.gptoss_rope_table(ctypes.byref(cfg), A + 4, None) == g.GPTOSS_ERR_INVALID
    assert b"beta_fast" in g.lib.gptoss_last_error()
    cfg.scaling_factor = 1.0  # unused then: what is refused is the table's alignment
    assert g.lib.gptoss_rope_table(ctypes.byref(cfg), A + 4, None) == g.GPTOSS_ERR_INVALID
    assert b"aligned" in g.lib.gptoss_last_error()


def cache(g, **kw):
    d = g.KvCacheDesc(64 * A, 80 * A, None, None, 0, 0, 0, g.GPTOSS_KV_BF16, 100, 16, 8, 64)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


SPAN = 100 * 16 * 8 * 64 * 2  # bytes of K, and of V


def attend(g, desc, prefill=False, **kw):
    a = dict(q=4 * A, q_stride=4096, off=7 * A, T=3, tables=8 * A, table_stride=10, max_blocks=10, lens=9 * A, B=3, H=64,
             out=5 * A, out_stride=4096, ws=16 * A + 8, ws_bytes=0)
    a.update(kw)
    c = g.AttentionConfig(0.125, 0, 0, None)
    head = (a["q"], a["q_stride"]) + ((a["off"], a["T"]) if prefill else ())
    f = g.lib.gptoss_paged_attention_prefill if prefill else g.lib.gptoss_paged_attention_decode
    return f(*head, ctypes.byref(desc), a["tables"], a["table_stride"], a["max_blocks"], a["lens"], a["B"], a["H"],
             ctypes.byref(c), a["out"], a["out_stride"], a["ws"], a["ws_bytes"], None)


def append(g, desc, **kw):
    a = dict(qkv=4 * A, stride=5120, pos=8 * A, slots=9 * A, table=10 * A, rotary=64, positions=1000, pairs=0, T=7, H=64,
             q=6 * A, q_stride=4096)
    a.update(kw)
    return g.lib.gptoss_rope_kv_append(a["qkv"], a["stride"], a["pos"], a["slots"], a["table"], a["rotary"], a["positions"],
                                       a["pairs"], a["T"], a["H"], a["q"], a["q_stride"], ctypes.byref(desc), None)


@pytest.mark.parametrize("at", [64 * A, 64 * A + SPAN - 16, 64 * A - 16, 80 * A + 4096, 80 * A - 2 * 8192 - 8192 + 16])
def test_results_in_the_cache_refused(g, at):
    for prefill in (False, True):
        assert attend(g, cache(g), prefill, out=at) == g.GPTOSS_ERR_INVALID
        assert g.lib.gptoss_last_error() == b"out overlaps the cache"
    for kw in (dict(q=at), dict(qkv=at, q=at, q_stride=5120), dict(qkv=at, T=3)):
        assert append(g, cache(g), **kw) == g.GPTOSS_ERR_INVALID
        assert b"overlaps the cache" in g.lib.gptoss_last_error()


def test_results_beside_the_cache(g):
    """Right before and behind K and V (what is refused is the next argument); strides past any address do not wrap."""
    for at in (64 * A - 3 * 8192, 64 * A + SPAN, 80 * A - 3 * 8192, 80 * A + SPAN):
        for prefill in (False, True):
            assert attend(g, cache(g), prefill, out=at, tables=None) == g.GPTOSS_ERR_INVALID
            assert b"null block_tables" in g.lib.gptoss_last_error()
    far = cache(g, num_blocks=1 << 20, block_stride=1 << 60, head_stride=1 << 40, token_stride=64)
    for prefill in (False, True):
        assert attend(g, far, prefill, out=128 * A) == g.GPTOSS_ERR_INVALID
        assert g.lib.gptoss_last_error() == b"out overlaps the cache"


@pytest.mark.parametrize("at,fits", [(4096, True), (4096 + 96, True), (-4096 - 96, True), (4096 - 8, False), (4096 + 104, False),
                                     (8, False), (-8, False), (2 * 8288 - 8, False), (2 * 8288 + 4096, True), (-4096 - 104, False)])
def test_rows_between_rows(g, at, fits):
    """q and out as columns of one buffer: rows of either lie between the other's (what is refused then is the next
    argument).  `at`: elements from q to out; a buffer's row has 8288, each of the two 4096."""
    for prefill in (False, True):
        kw = dict(q=20 * A, q_stride=8288, out=20 * A + 2 * at, out_stride=8288, B=3, T=3, tables=None)
        assert attend(g, cache(g), prefill, **kw) == g.GPTOSS_ERR_INVALID
        assert (b"null block_tables" if fits else b"out overlaps q") in g.lib.gptoss_last_error()


@pytest.mark.parametrize("at,fits", [(5120, True), (5120 + 128, True), (-4096, True), (-4096 - 128, True), (5112, False),
                                     (5120 + 136, False), (8, False), (-8, False)])
def test_queries_between_rows(g, at, fits):
    kw = dict(qkv=20 * A, stride=9344, q=20 * A + 2 * at, q_stride=9344)
    if fits:  # accepted as far as the cache, which is made to hold it
        d = cache(g, k=20 * A)
        assert append(g, d, **kw) == g.GPTOSS_ERR_INVALID and b"overlaps the cache" in g.lib.gptoss_last_error()
    else:
        assert append(g, cache(g), **kw) == g.GPTOSS_ERR_INVALID and b"overlaps qkv" in g.lib.gptoss_last_error()


# ---------------------------------------------------------------------------
# the binding
# ---------------------------------------------------------------------------
def pages(blocks=6):
    import torch
    return torch.zeros((blocks, 8, 16, 64), dtype=torch.bfloat16)


def test_kv_cache_is_fixed(g):
    """Another tensor would not be what calls use: their descriptor holds the addresses of the first."""
    k, v = pages(), pages()
    c = g.KVCache(k, v)
    for name, x in (("k", pages(9)), ("v", pages(9)), ("k_scale", None), ("num_blocks", 9), ("desc", None), ("other", 1)):
        with pytest.raises(AttributeError, match="fixed"):
            setattr(c, name, x)
    with pytest.raises(AttributeError, match="fixed"):
        del c.k
    assert c.k is k and c.v is v and c.desc.k == k.data_ptr() and c.desc.num_blocks == c.num_blocks == 6


def test_numbers_past_32_bits_refused(g):
    """A window of 2^32 + 128 is not one of 128."""
    import torch
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    c, q = g.KVCache(pages(), pages()), torch.zeros((3, 4096), dtype=torch.bfloat16)
    for bad in (2 ** 32 + 128, 2 ** 31, -1, -2 ** 32):
        for kw in (dict(window=bad), dict(window=4, first_tokens=bad)):
            with pytest.raises(ValueError, match="2\\^31"):
                g.paged_attention_decode(q, c, i32(3, 5), i32(3), **kw)
            with pytest.raises(ValueError, match="2\\^31"):
                g.paged_attention_prefill(q, i32(4), c, i32(3, 5), i32(3), **kw)
    with pytest.raises(ValueError, match="GPU is needed"):
        g.paged_attention_decode(q, c, i32(3, 5), i32(3), window=2 ** 31 - 1, first_tokens=2 ** 31 - 1)
    for bad in ((2 ** 32 + 5, 3, 64), (5, 2 ** 32 + 3, 64), (5, 3, 2 ** 32 + 64)):
        with pytest.raises(ValueError, match="2\\^31"):
            g.paged_attention_workspace_bytes(*bad, c)


def test_engine_names_the_attention_there_is():
    """The engine's refusal to generate points to the attention operators instead of denying them."""
    import torch  # noqa: F401  (first: the library binds to torch's HIP runtime)
    import gptoss
    with pytest.raises(RuntimeError, match="gptoss_moe's rope_kv_append and paged_attention_decode"):
        gptoss.InferenceEngine().generate([1, 2, 3])
    assert "does not contain" not in gptoss.InferenceEngine.generate.__doc__
