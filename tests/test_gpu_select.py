"""GPU: the expert selection against its definition in 64 bits (mx_ref.py, where the tolerances are derived)."""
import math

import pytest
import torch

import mx_ref as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def check(gpu, logits, k, **kw):
    got = gpu.select_experts(logits, k, score=kw.get("score", "softmax"), bias=kw.get("bias"),
                             num_groups=kw.get("groups", 1), top_groups=kw.get("top_groups", 1),
                             group_rank=kw.get("rank", 2), renormalize=kw.get("renormalize", True),
                             scale=kw.get("scale", 1.0))
    torch.cuda.synchronize()
    ref.assert_selected(got, ref.select(logits, k, **kw), (tuple(logits.shape), k, kw.get("score"), kw.get("groups")))
    return got


GROUPS = [(1, 1, 2), (4, 2, 2), (4, 3, 1), (4, 4, 2)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups, top_groups, rank", GROUPS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("E, k", [(4, 1), (8, 2), (60, 5), (64, 8), (128, 4), (192, 6), (256, 8), (512, 10), (1000, 7),
                                  (1024, 32)])
def test_against_64_bits(gpu, E, k, bias, groups, top_groups, rank, score, dtype):
    gen = gen_of(E + k)
    logits = (2 * torch.randn((37, E), device="cuda", generator=gen)).to(dtype)
    b = 0.1 * torch.randn(E, device="cuda", generator=gen) if bias else None
    check(gpu, logits, min(k, top_groups * (E // groups)), score=score, bias=b, groups=groups, top_groups=top_groups, rank=rank,
          renormalize=E % 128 != 0, scale=2.5 if E % 3 else 1.0)


@pytest.mark.parametrize("T", [1, 2, 3, 5, 63, 64, 65, 257, 2000])
@pytest.mark.parametrize("E, groups", [(256, 8), (128, 1), (24, 3)])
def test_token_counts(gpu, T, E, groups):
    logits = (2 * torch.randn((T, E), device="cuda", generator=gen_of(T))).to(BF16)
    bias = 0.1 * torch.randn(E, device="cuda", generator=gen_of(T + 1))
    check(gpu, logits, 6, score="sigmoid", bias=bias, groups=groups, top_groups=(groups + 1) // 2, scale=2.5)
    check(gpu, logits, 4)


@pytest.mark.parametrize("E", [1, 2, 3, 7, 33, 65, 127, 130, 257, 1023])
def test_odd_expert_counts(gpu, E):
    logits = torch.randn((9, E), device="cuda", generator=gen_of(E))
    for k in {1, min(E, 5), min(E, 32)}:
        for score in ("softmax", "sigmoid"):
            check(gpu, logits, k, score=score)
            check(gpu, logits.to(BF16), k, score=score, renormalize=False)
            check(gpu, logits, k, score=score, bias=torch.linspace(-1, 1, E, device="cuda"))


@pytest.mark.parametrize("groups, top_groups", [(2, 1), (8, 3), (16, 5), (32, 32), (64, 17)])
@pytest.mark.parametrize("rank", [1, 2])
def test_group_sizes(gpu, groups, top_groups, rank):
    for size in (1, 2, 3, 16):
        E = groups * size
        logits = (3 * torch.randn((21, E), device="cuda", generator=gen_of(E + rank))).to(BF16)
        k = min(top_groups * size, 8)
        for score in ("softmax", "sigmoid"):
            check(gpu, logits, k, score=score, groups=groups, top_groups=top_groups, rank=rank)
            check(gpu, logits, k, score=score, groups=groups, top_groups=top_groups, rank=rank,
                  bias=torch.randn(E, device="cuda", generator=gen_of(E)))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_ties_go_to_the_lower_index(gpu, score, bias, groups):
    E = 64
    b = torch.full((E,), 0.25, device="cuda") if bias else None
    few = torch.randint(0, 3, (50, E), device="cuda", generator=gen_of(1)).float()  # three different values
    for logits in (torch.zeros((3, E), device="cuda"), few, few.to(BF16), -few):
        check(gpu, logits, 8, score=score, bias=b, groups=groups, top_groups=(groups + 1) // 2)
    zeros = torch.zeros((2, E), device="cuda")
    zeros[:, ::2] = -0.0
    idx, _ = check(gpu, zeros, 4, score=score, bias=b)
    assert idx.cpu().tolist() == [[0, 1, 2, 3]] * 2


@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_choices_that_32_bits_do_not_tell_apart(gpu, score, groups):
    """The order is that of the exact choices: the bias makes up for the score but for a few 1e-9."""
    E, T = 64, 40
    logits = torch.randn((T, E), device="cuda", generator=gen_of(3))
    logits = logits[:1].expand(T, E).contiguous()  # one row, so that one bias nearly evens it out
    x = logits[0].double()
    s = torch.softmax(x, 0) if score == "softmax" else torch.sigmoid(x)
    bias = (0.9 - s).float()
    # what rounding the bias to 32 bits leaves is of the size of 2^-26 to 2^-25, and never a tie
    left = s + bias.double()
    assert 0 < float((left.sort().values.diff()).min()) < 1e-8 and float(left.max() - left.min()) < 1e-6
    check(gpu, logits, 8, score=score, bias=bias, groups=groups, top_groups=(groups + 1) // 2)


@pytest.mark.parametrize("E, groups", [(129, 1), (256, 1), (256, 8), (300, 3), (1000, 1), (1024, 16)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_many_chosen_of_many(gpu, E, groups, score):
    """Ties on the border of what is chosen and within it, choices of all sizes and signs, few left, infinite and NaN ones."""
    gen = gen_of(E)
    kw = dict(score=score, groups=groups, top_groups=(groups + 1) // 2)
    few = torch.randint(0, 3, (12, E), device="cuda", generator=gen).float()
    some = torch.randint(0, 60, (12, E), device="cuda", generator=gen).float() / 16
    plain = torch.randn((12, E), device="cuda", generator=gen)
    size = torch.exp2(torch.randint(-100, 100, (E,), device="cuda", generator=gen).float())
    wide = torch.randn(E, device="cuda", generator=gen) * size
    two = torch.where(torch.rand(E, device="cuda", generator=gen) < 0.02, 1e30, -1e-30)
    left = torch.full((E,), -math.inf, device="cuda")
    left[::E // 9] = 0.25
    odd = wide.clone()
    odd[3], odd[E // 2], odd[E - 1] = math.inf, math.nan, -math.inf
    for k in (6, 8, 32):
        for logits in (few, some, some.to(BF16), plain):
            check(gpu, logits, k, **kw)
            check(gpu, logits, k, bias=torch.full((E,), 0.5, device="cuda"), **kw)
        for bias in (wide, -wide.abs(), two, left, odd):
            check(gpu, plain, k, bias=bias, renormalize=False, **kw)


def test_close_choices_among_others(gpu):
    """Pairs of nearly equal choices here and there in ordinary rows."""
    E, T = 256, 64
    gen = gen_of(5)
    logits = 2 * torch.randn((T, E), device="cuda", generator=gen)
    top = logits.argsort(1, descending=True)
    for t in range(T):  # the eighth and ninth, or two in the middle of the chosen
        a, b = top[t, 7 if t % 2 else 3], top[t, 8 if t % 2 else 4]
        logits[t, a] = torch.nextafter(logits[t, b], torch.tensor(math.inf, device="cuda"))
    bias = torch.full((E,), 0.125, device="cuda")
    for score in ("softmax", "sigmoid"):
        check(gpu, logits, 8, score=score, bias=bias)
        check(gpu, logits, 8, score=score, bias=bias, groups=8, top_groups=4)
        check(gpu, logits, 8, score=score, groups=8, top_groups=4)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_experts_switched_off(gpu, score, groups):
    E, k = 32, 8
    gen = gen_of(7)
    logits = torch.randn((60, E), device="cuda", generator=gen)
    keep = torch.rand((60, E), device="cuda", generator=gen) < torch.linspace(0, 1, 60, device="cuda")[:, None]
    masked = torch.where(keep, logits, -math.inf)  # the first rows have few or none left
    masked[0], masked[1] = -math.inf, -math.inf
    masked[1, E - 1] = 0.5
    kw = dict(score=score, groups=groups, top_groups=(groups + 1) // 2)
    for dtype in (F32, BF16):
        idx, w = check(gpu, masked.to(dtype), k, **kw)
        assert idx.sort(1).values.diff(dim=1).min() > 0 and idx.min() >= 0 and idx.max() < E  # distinct and valid
        assert not w[0].any()
    for off in (1, 20, 31, 32):
        bias = 0.1 * torch.randn(E, device="cuda", generator=gen)
        bias[torch.randperm(E, device="cuda", generator=gen)[:off]] = -math.inf
        check(gpu, logits, k, bias=bias, **kw)
        check(gpu, masked, k, bias=bias, renormalize=False, **kw)
    check(gpu, torch.full((2, E), torch.finfo(BF16).min, device="cuda", dtype=BF16), k, **kw)  # the lowest value is one
    check(gpu, torch.full((2, E), -1e38, device="cuda"), k, bias=torch.linspace(0, 1, E, device="cuda"), **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("bias", [False, True])
def test_infinite_and_nan_logits(gpu, score, groups, bias):
    E = 32
    logits = torch.randn((8, E), device="cuda", generator=gen_of(9))
    logits[0, 5] = math.inf
    logits[1, 5], logits[1, 29] = math.inf, math.inf
    logits[2, 7] = math.nan
    logits[3] = math.nan
    logits[4, 3], logits[4, 4], logits[4, 20] = math.nan, -math.inf, math.inf
    logits[5] = math.inf
    logits[6, :8] = math.nan
    b = 0.1 * torch.randn(E, device="cuda", generator=gen_of(10)) if bias else None
    if bias:
        b[11] = math.nan
        b[12] = math.inf
    for dtype in (F32, BF16):
        check(gpu, logits.to(dtype), 6, score=score, groups=groups, top_groups=(groups + 1) // 2, bias=b)


def test_wide_logits(gpu):
    """Far apart, and all far below zero: shares of a vanishing sum."""
    for scale in (30.0, 100.0):
        logits = scale * torch.randn((40, 64), device="cuda", generator=gen_of(11))
        check(gpu, logits, 4)
        check(gpu, logits, 4, renormalize=False)
    check(gpu, torch.randn((40, 64), device="cuda", generator=gen_of(12)) - 300, 4, score="sigmoid")
    check(gpu, torch.randn((40, 64), device="cuda", generator=gen_of(12)) - 95, 4, score="sigmoid", groups=4, top_groups=2)


def test_strided_logits_and_given_results(gpu):
    wide = torch.randn((33, 300), device="cuda", generator=gen_of(13))
    idx = torch.empty((33, 4), dtype=torch.int32, device="cuda")
    w = torch.empty((33, 4), device="cuda")
    for view in (wide[:, 100:228], wide[:, 1:129], wide[::2, 3:131], wide.to(BF16)[:, 7:135]):
        n = view.shape[0]
        got = gpu.select_experts(view, 4, out=(idx[:n], w[:n]))
        assert got[0].data_ptr() == idx.data_ptr()
        ref.assert_selected(got, ref.select(view, 4))
    one = wide[5:6, 200:264]
    ref.assert_selected(gpu.select_experts(one, 3), ref.select(one, 3))
    assert gpu.select_experts(wide[:0], 4)[0].shape == (0, 4)


def test_the_largest_call(gpu):
    """2^26 tokens: more threads than one launch holds."""
    T = 1 << 26
    logits = torch.zeros((T, 2), device="cuda", dtype=BF16)
    for t in (0, 12345, (1 << 25) - 1, 1 << 25, T - 2):
        logits[t, 1] = 1.0 + t % 7
    idx, w = gpu.select_experts(logits, 1, renormalize=False)
    torch.cuda.synchronize()
    assert torch.equal(idx[:, 0].long(), (logits[:, 1] > 0).long())
    for t in (0, 1, 12345, (1 << 25) - 1, 1 << 25, (1 << 25) + 1, T - 2, T - 1):
        want = 1 / (1 + math.exp(-float(logits[t, 1])))
        assert abs(float(w[t]) - want) < 2.0 ** -23 * want


def test_a_prefix_gives_the_same(gpu):
    """A token's choice is its own: the same bits in a smaller call, and in another place of it."""
    logits = (2 * torch.randn((3000, 256), device="cuda", generator=gen_of(14))).to(BF16)
    bias = 0.1 * torch.randn(256, device="cuda", generator=gen_of(15))
    kw = dict(score="sigmoid", bias=bias, num_groups=8, top_groups=4, scale=2.5)
    idx, w = gpu.select_experts(logits, 8, **kw)
    for n in (1, 7, 64, 1000):
        a, b = gpu.select_experts(logits[:n], 8, **kw)
        assert torch.equal(a, idx[:n]) and torch.equal(b, w[:n])
        a, b = gpu.select_experts(logits[-n:], 8, **kw)
        assert torch.equal(a, idx[-n:]) and torch.equal(b, w[-n:])


@pytest.mark.parametrize("E, k", [(32, 4), (128, 4), (128, 8), (256, 2)])
def test_like_the_top_k_softmax(gpu, E, k):
    """Softmax scores, renormalised: what gptoss_topk_softmax_forward computes."""
    for dtype in (BF16, F32):
        logits = (2 * torch.randn((300, E), device="cuda", generator=gen_of(16))).to(dtype)
        idx, w = gpu.select_experts(logits, k)
        idx2, w2 = gpu.topk_softmax(logits, k)
        assert torch.equal(idx, idx2)
        assert float(((w - w2).abs() / w).max()) < 40 * 2.0 ** -23  # arguments up to 16, both off by 2^-23 of them


def test_streams_and_graphs(gpu):
    logits = 2 * torch.randn((64, 256), device="cuda", generator=gen_of(17))
    bias = 0.1 * torch.randn(256, device="cuda", generator=gen_of(18))
    kw = dict(score="sigmoid", bias=bias, num_groups=8, top_groups=4)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = gpu.select_experts(logits, 8, stream=side, **kw)
    side.synchronize()
    want = gpu.select_experts(logits, 8, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out = (torch.empty_like(want[0]), torch.empty_like(want[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.select_experts(logits, 8, out=out, **kw)
    for seed in range(3):
        logits.copy_(2 * torch.randn((64, 256), device="cuda", generator=gen_of(seed)))
        want = gpu.select_experts(logits, 8, **kw)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("groups", [1, 4])
def test_a_bias_that_switches_off_a_nan(gpu, groups, dtype):
    """A bias of -inf switches its expert off whatever the score is: weight 0 beside NaN, and nothing in the sum."""
    E, off = 8, (2, 5)
    bias = torch.zeros(E, device="cuda")
    bias[list(off)] = -math.inf
    logits = torch.linspace(-2, 2, 3 * E, device="cuda").view(3, E).to(dtype)
    logits[0, 2] = math.nan  # of an expert that is off
    logits[1, 2], logits[1, 6] = math.nan, math.nan  # and of one that is not
    logits[2, 6] = math.nan
    kw = dict(bias=bias, num_groups=groups, top_groups=groups)
    x = logits.double().cpu()

    def order(nan):  # finite choices, the larger first, then the others by index
        last = sorted(set(off) | set(nan))
        return sorted(set(range(E)) - set(last), reverse=True) + last

    # sigmoid: each score is its own
    idx, w = gpu.select_experts(logits, E, score="sigmoid", renormalize=False, **kw)
    for t, nan in enumerate(((), (6,), (6,))):
        assert idx[t].tolist() == order(nan)
        for e, got in zip(idx[t].tolist(), w[t].tolist()):
            if e in off:
                assert got == 0.0, (t, e, got)
            elif e in nan:
                assert math.isnan(got)
            else:
                assert abs(got - float(torch.sigmoid(x[t, e]))) <= (2.0 ** -24 + 2.0 ** -48) * got  # rounded once from 64 bits
    idx, w = gpu.select_experts(logits, E, score="sigmoid", **kw)
    s = torch.sigmoid(x[0])
    s[list(off)] = 0
    want = (s / s.sum())[idx[0].cpu().long()]
    assert bool(((w[0].cpu().double() - want).abs() <= (2.0 ** -24 + 2.0 ** -48) * want).all())
    # softmax over a row with a NaN: the scores are NaN, but of experts that are off
    idx, w = gpu.select_experts(logits, E, renormalize=False, **kw)
    for t in range(3):
        assert idx[t].tolist() == list(range(E))
        assert [e for e in range(E) if not math.isnan(float(w[t, e]))] == list(off)
        assert not w[t, list(off)].any()


def weights_of_64_bits(logits, k, score="softmax", **kw):
    """mx_ref's selection, and how far 64-bit arithmetic with one rounding at the end may be from it.  The exponential's
    argument is a difference of fp32 values, off by 2^-53 of its size, the exponential by two units of 2^-52; sums of up to
    1024 terms by lanes and then across them, two divisions and the scale have fewer than 40 roundings of 2^-53; the
    oracle's own arithmetic has no more.  Then half a unit of fp32, 2^-24 of a normal number and 2^-150 below."""
    idx, w, _ = ref.select(logits, k, score, **kw)
    x = logits.detach().cpu().double()
    far = (x - x.amax(1, keepdim=True) if score == "softmax" else x).abs().amax(1, keepdim=True)
    return idx, w, w.abs() * (2.0 ** -24 + (far + 64) * 2.0 ** -51) + 2.0 ** -150


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E, k, groups", [(8, 2, 1), (32, 4, 1), (64, 8, 4), (128, 4, 1), (128, 8, 8), (256, 8, 8), (384, 6, 1),
                                          (1000, 32, 1), (1024, 32, 16)])
@pytest.mark.parametrize("spread", [0.01, 2.0, 60.0])
def test_weights_are_rounded_once(gpu, E, k, groups, score, dtype, spread):
    gen = gen_of(E + k)
    logits = (spread * torch.randn((50, E), device="cuda", generator=gen)).to(dtype)
    bias = 0.1 * torch.randn(E, device="cuda", generator=gen) if groups > 1 else None
    for renormalize, scale in ((True, 1.0), (True, 2.5), (False, 0.75)):
        kw = dict(score=score, bias=bias, renormalize=renormalize, scale=scale)
        got = gpu.select_experts(logits, k, num_groups=groups, top_groups=(groups + 1) // 2, **kw)
        ref.assert_selected(got, weights_of_64_bits(logits, k, groups=groups, top_groups=(groups + 1) // 2, **kw),
                            (renormalize, scale))
