"""The expert selection and the MXFP4 operators in 64 bits, from their definition, and how far results may be off.

Tolerances.  Products of e2m1 values with their scales are exact, so a sum of K of them in fp32 is within
K * 2^-24 * sum|a w| of the exact one in whatever order, the bias adds one rounding (2^-24 of what it is then), and a
bf16 result one of 2^-8 of its value.  SwiGLU's slope is at most 1.1 |up + 1| along the gate (x sigmoid(x) rises at
most 1.1 per 1, and so does its scaled form) and |g sigmoid| along up; its own arithmetic has an exponential whose
argument is off by 2^-23 |alpha g| and seven further roundings of at most 2^-22."""
import math

import torch

F64 = torch.float64
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=F64)


def nearest(v):
    """Codes 0..7 of magnitudes: the nearest grid value, half way the even code, above 6 the last."""
    d = (v.cpu().unsqueeze(-1) - GRID).abs()
    best = d.amin(-1, keepdim=True)
    tied = d == best
    even = tied & (torch.arange(8) % 2 == 0)
    return torch.where(even.any(-1), even.int().argmax(-1), tied.int().argmax(-1))


def scale_bytes(top):
    """Of the largest magnitudes: floor(log2) - 2, at least -126, plus 127; 255 without a finite one."""
    e = (torch.frexp(top.double()).exponent - 3).clamp(min=-126)
    e = torch.where(top == 0, torch.full_like(e, -126), e)
    return torch.where(torch.isfinite(top), e + 127, torch.full_like(e, 255))


def quantize(x):
    """(codes [rows, K], scale bytes [rows, K / 32]) of x, on the host."""
    v = x.detach().cpu().double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(v).all(-1)
    top = torch.where(bad, torch.full_like(v[..., 0], math.inf), v.abs().amax(-1))
    s = scale_bytes(top)
    y = torch.ldexp(v, (127 - s).unsqueeze(-1))
    code = nearest(y.abs().nan_to_num(0, 0, 0)) + 8 * torch.signbit(v).int()
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code)
    return code.flatten(-2).to(torch.uint8), s.to(torch.uint8)


def unpack(packed):
    p = packed.cpu()
    return torch.stack((p & 15, p >> 4), dim=-1).flatten(-2)


def pack(code):
    return code[..., ::2] | (code[..., 1::2] << 4)


def values(code, scales):
    """In 64 bits on the host: e2m1 * 2^(byte - 127), NaN for byte 255."""
    v = GRID[(code & 7).long()] * torch.where(code >= 8, -1.0, 1.0).double()
    s = torch.exp2(scales.cpu().double() - 127)
    s = torch.where(scales.cpu() == 255, torch.full_like(s, math.nan), s)
    return v * s.repeat_interleave(32, dim=-1)


def of_matrix(m):
    return values(unpack(m.packed), m.scales)


def random_matrix(gpu, gen, *shape, low=120, high=134):
    """Uniform codes, scale bytes in [low, high)."""
    K = shape[-1]
    return gpu.MXFP4Matrix(
        torch.randint(0, 256, (*shape[:-1], K // 2), device="cuda", generator=gen, dtype=torch.uint8),
        torch.randint(low, high, (*shape[:-1], K // 32), device="cuda", generator=gen, dtype=torch.uint8))


def product(a, w, bias=None):
    """(y, tolerance of the fp32 sums) of a [M, K] and w [N, K] in 64 bits."""
    y, size = a @ w.T, a.abs() @ w.abs().T
    tol = a.shape[1] * 2.0 ** -24 * size
    if bias is not None:
        y = y + bias.cpu().double()
        tol = tol + 2.0 ** -24 * y.abs()
    return y, tol + 2.0 ** -140


def swiglu(y, tol, alpha=1.702, limit=7.0):
    g, u = y[:, ::2].clamp(max=limit), y[:, 1::2].clamp(-limit, limit)
    s = g * torch.sigmoid(alpha * g)
    act = (u + 1) * s
    off = 1.1 * (u + 1).abs() * tol[:, ::2] + s.abs() * tol[:, 1::2] + 2.0 * tol[:, ::2] * tol[:, 1::2]
    return act, off + act.abs() * ((alpha * g).abs() * 2.0 ** -23 + 7 * 2.0 ** -22) + s.abs() * 2.0 ** -24


def assert_values(got, want, tol, what=""):
    """Values of bf16 or fp32; NaN and infinities where the definition has them."""
    half = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[got.dtype]
    g = got.cpu().double()
    assert g.shape == want.shape, what
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(g), torch.isnan(want)), what
    assert torch.equal(g[~fine].nan_to_num(), want[~fine].nan_to_num()), what
    room = tol[fine] * (1 + half) + half * want[fine].abs()
    bad = (g[fine] - want[fine]).abs() > room
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, most " \
                          f"{float(((g[fine] - want[fine]).abs() / room).max()):.2f} of the tolerance"


def assert_quantized(m, want, tol, what=""):
    """An MXFP4Matrix of results that are within tol of want: scale bytes and codes that such results have."""
    code, s = unpack(m.packed), m.scales.cpu().int()
    w, t = want.unflatten(-1, (-1, 32)), tol.unflatten(-1, (-1, 32))
    lo = scale_bytes((w.abs() - t).clamp(min=0).amax(-1))
    hi = scale_bytes((w.abs() + t).amax(-1))
    assert bool(((s >= lo) & (s <= hi)).all()), what
    e = (127 - s).unsqueeze(-1)

    def rounded(v):
        v = torch.ldexp(v, e.expand_as(v))
        return torch.copysign(GRID[nearest(v.abs())], v)

    v = values(code, torch.full_like(m.scales.cpu(), 127)).unflatten(-1, (-1, 32))
    assert bool(((v >= rounded(w - t)) & (v <= rounded(w + t))).all()), what


def select(logits, k, score="softmax", bias=None, groups=1, top_groups=1, rank=2, renormalize=True, scale=1.0):
    """(indices, weights, how far weights may be off) in 64 bits, a token at a time."""
    x = logits.detach().cpu().double()
    T, E = x.shape
    b = torch.zeros(E, dtype=F64) if bias is None else bias.detach().cpu().double()
    size = E // groups
    idx, wts = torch.zeros((T, k), dtype=torch.int32), torch.zeros((T, k), dtype=F64)
    tol = torch.zeros((T, k), dtype=F64)
    for t in range(T):
        l = x[t].tolist()
        m = max((v for v in l if v == v), default=-math.inf)
        if score == "softmax":
            ex = [math.nan if v != v else 0.0 if v == -math.inf else 1.0 if v == m else math.exp(v - m) for v in l]
            total = math.fsum(ex) if all(v == v for v in ex) else math.nan
            s = [v / total if total != 0 else 0.0 for v in ex]
            far = [abs(v - m) if 0 < e < 1 else 0.0 for v, e in zip(l, ex)]
        else:
            s = [math.nan if v != v else 0.0 if v < -745 else 1 / (1 + math.exp(-v)) for v in l]
            far = [abs(v) if abs(v) < 1e3 else 0.0 for v in l]
        c = [a + d for a, d in zip(s, b.tolist())]
        off = [v == -math.inf or d == -math.inf for v, d in zip(l, c)]
        s = [0.0 if o else v for v, o in zip(s, off)]
        c = [-math.inf if o or not v > -math.inf else v for v, o in zip(c, off)]
        kept = range(groups)
        if groups > 1:
            sums = []
            for g in range(groups):
                best = [v for v in sorted(c[g * size:(g + 1) * size], reverse=True)[:rank] if v > -math.inf]
                sums.append(sum(best) if best else -math.inf)
            kept = sorted(range(groups), key=lambda g: (-sums[g], g))[:top_groups]
        order = sorted(range(E), key=lambda e: (e // size not in kept, -c[e], e))[:k]
        chosen = [s[e] for e in order]
        total = sum(chosen)
        for i, e in enumerate(order):
            w = chosen[i]
            if renormalize:
                w = w / total if total != 0 else 0.0
            idx[t, i], wts[t, i] = e, w * scale
            # fp32 scores: their argument off by 2^-23 of its size (the largest of the row's where it is divided by
            # their sum), eight roundings
            tol[t, i] = abs(w * scale) * (max(far, default=0.0) + 8) * 2.0 ** -23 + 2.0 ** -149
    return idx, wts, tol


def assert_selected(got, want, what=""):
    idx, w = got
    assert torch.equal(idx.cpu(), want[0]), what
    w = w.cpu().double()
    assert torch.equal(torch.isnan(w), torch.isnan(want[1])), what
    fine = ~torch.isnan(w)
    assert bool(((w - want[1]).abs()[fine] <= want[2][fine]).all()), what
