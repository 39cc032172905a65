"""CPU tests: which way the attention calls of the GPU tests go, by the workspace that they need (none: not cut), so
that a changed rule that leaves a way untested fails here."""
import pytest

from test_gpu_attention import FEW, GPT, GQA4


@pytest.fixture(scope="module")
def g():
    import gptoss_moe
    return gptoss_moe


def pieces(g, rows, B, shape, tokens, window=0, first=0):
    """Pieces of a prompt call's tokens: partial results of every row in each, and a count for every row."""
    H, Hk, D, _ = shape
    size = g.lib.gptoss_paged_attention_call_bytes(rows, B, H, Hk, D, tokens, window, first)
    if size == 0:
        return 1
    n, rest = divmod(size - (4 * rows + 15) // 16 * 16, 4 * rows * H * (D + 4))
    assert rest == 0 and n > 1
    return n


@pytest.mark.parametrize("case,want", zip(FEW, [(1, 1, 1), (3, 3, 3), (1, 1, 1), (4, 3, 3), (1, 1, 1), (1, 1, 1)]))
def test_few_rows(g, case, want):
    """test_prefill_few_rows_over_many_tokens: all with two groups of waves."""
    shape, new = case
    bs = shape[3]
    tokens = (max(2900, new) + bs - 1) // bs * bs
    for (window, first), n in zip(((0, 0), (1500, 0), (1501, 70)), want):
        assert pieces(g, new // 2 + 7 + new // 2 + 1, 3, shape, tokens, window, first) == n


def test_two_groups_in_two_pieces(g):
    """test_prefill_two_groups_in_two_pieces."""
    for window, first in ((0, 0), (3500, 70)):
        assert pieces(g, 210, 1, GPT, 4096, window, first) == pieces(g, 340, 1, GQA4, 4096, window, first) == 2


def test_wide_tables(g):
    """Of test_wide_tables, which calls are cut with the table that they need and with one of 131072 tokens."""
    for shape, rows, lens, tight, wide in [(GPT, 680, [680], 1, 2), (GPT, 512, [512], 1, 1), (GPT, 330, [1120, 900, 500, 300], 1, 4),
                                           (GPT, 506, [1028, 900, 800, 700, 500, 300, 200, 128], 1, 2),
                                           (GQA4, 680, [680], 1, 1)]:
        bs = shape[3]
        need = max((n + bs - 1) // bs for n in lens) * bs
        assert pieces(g, rows, len(lens), shape, need) == tight
        assert pieces(g, rows, len(lens), shape, 131072) == wide
    for shape, B in ((GPT, 1), (GPT, 64)):
        H, Hk, D, _ = shape
        size = g.lib.gptoss_paged_attention_call_bytes
        assert size(0, B, H, Hk, D, 1008, 0, 0) == 0 < size(0, B, H, Hk, D, 131072, 0, 0)
