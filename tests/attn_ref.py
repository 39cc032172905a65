"""The attention operators in 64 bits, from their definition, with how far fp32 sums, bf16 weights and one
rounding of the result may be off; and the inputs of their tests."""
import math

import torch


def make_cache(gen, blocks, Hk, bs, D, e4m3, layout="heads", device="cuda", fill=float("nan")):
    """K and V pages as [blocks, Hk, bs, D] (a permuted view when token-major), and scales."""
    shape = (blocks, Hk, bs, D) if layout == "heads" else (blocks, bs, Hk, D)
    dtype = torch.float8_e4m3fn if e4m3 else torch.bfloat16
    if layout == "slab":
        slab = torch.full((blocks, 2, Hk, bs, D), fill, device=device).to(dtype)
        pages = [slab[:, 0], slab[:, 1]]
    else:
        pages = [torch.full(shape, fill, device=device).to(dtype) for _ in range(2)]
        if layout == "tokens":
            pages = [p.permute(0, 2, 1, 3) for p in pages]
    scales = [torch.rand(Hk, device=device, generator=gen) * 0.05 + 0.01 for _ in range(2)] if e4m3 else [None, None]
    return pages, scales


def store(pages, scales, table, bs, rows):
    """Writes rows [n, Hk, D] (k, v) as tokens 0.. of the sequence whose pages are `table`."""
    n = rows[0].shape[0]
    t = torch.arange(n, device=rows[0].device)
    page = table[: (n + bs - 1) // bs].long().to(rows[0].device)[t // bs]
    for p, s, r in zip(pages, scales, rows):
        if s is None:
            p[page, :, t % bs] = r.to(torch.bfloat16)
        else:
            code = (r.float() / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
            p.view(torch.uint8)[page, :, t % bs] = code.view(torch.uint8)


def load(pages, scales, table, bs, n, h):
    """Tokens 0..n-1 of kv head h in 64 bits, [n, D] of K and of V."""
    out = []
    t = torch.arange(n, device=pages[0].device)
    for p, s in zip(pages, scales):
        raw = p.view(torch.uint8) if s is not None else p
        x = raw[table[t // bs].long(), h, t % bs].view(p.dtype).double()
        out.append(x if s is None else x * s[h].double())
    return out


def attend64(q, pos, length, pages, scales, table, bs, scale, window=0, first=0, sinks=None):
    """q [n, H, D] at positions pos (list) over the first `length` tokens; table entries outside the pages hide
    their tokens.  Returns (out, tol) [n, H, D]: the result and the largest error that the kernels' arithmetic
    allows.  With A = sum p |v| / l and half a bf16 step h = 2^-8 relative: the weights' rounding moves the result by
    up to h A (where the sum is of the rounded weights too the bound is h sum p |v - out| / l, at most h (A + |out|);
    that is counted as h A all the same), the result's own by h |out|; the scores' fp32 sums of D products (and the product with the scale) by a
    relative 2 (D + 8) 2^-24 max sum |q k| scale of each weight, and the fp32 sums over the tokens by L 2^-23."""
    n, H, D = q.shape
    Hk = pages[0].shape[1]
    dev = q.device
    out = torch.zeros(n, H, D, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    if length == 0 or n == 0:
        return out, tol
    t = torch.arange(length, device=dev)
    p = torch.tensor(pos, device=dev)[:, None]
    page = table[t // bs]
    seen = (t <= p) & (page >= 0) & (page < pages[0].shape[0])
    if window:
        seen &= (p - t < window) | (t < first)
    safe = table.clamp(0, pages[0].shape[0] - 1)
    any_seen = seen.any(1)
    h = 2.0 ** -8
    for g in range(Hk):
        k, v = load(pages, scales, safe, bs, length, g)
        used = seen.any(0)
        k, v = k.masked_fill(~used[:, None], 0.0), v.masked_fill(~used[:, None], 0.0)
        for i in range(g * (H // Hk), (g + 1) * (H // Hk)):
            x = q[:, i].double()
            s = (x @ k.T * scale).masked_fill(~seen, -math.inf)
            norm = torch.logsumexp(s, 1, keepdim=True)
            if sinks is not None:
                norm = torch.logaddexp(norm, sinks[i].double().expand_as(norm))
            w = (s - norm).exp().masked_fill(~any_seen[:, None], 0.0)
            o, a = w @ v, w @ v.abs()
            smax = ((x.abs() @ k.abs().T) * scale).max()
            out[:, i] = o
            tol[:, i] = a * (1.01 * h + 2 * (D + 8) * 2.0 ** -24 * smax + (length + 64) * 2.0 ** -23) + h * o.abs() + 1e-30
    return out, tol


def page_tables(gen, lens, bs, blocks, width=None, device="cuda"):
    """Distinct pages for each sequence, -1 past them."""
    used = [(n + bs - 1) // bs for n in lens]
    assert sum(used) <= blocks
    perm = torch.randperm(blocks, generator=gen, device=device).to(torch.int32)
    tables = torch.full((len(lens), width or max(max(used), 1)), -1, dtype=torch.int32, device=device)
    at = 0
    for b, n in enumerate(used):
        tables[b, :n] = perm[at:at + n]
        at += n
    return tables


def within(got, want, tol):
    """None, or what is off: every element within its tolerance, and neither NaN nor infinite."""
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    if not bad.any():
        return None
    i = int(bad.flatten().nonzero()[0])
    return (f"{int(bad.sum())} of {bad.numel()} off; first at {i}: got {got.flatten()[i].item()}, want "
            f"{want.flatten()[i].item()}, tol {tol.flatten()[i].item()}")
