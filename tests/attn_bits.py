"""How far decode's results may be off: its weights meet the values with 16 significant bits."""
import torch

import attn_ref as ref


def decode64(q, length, pages, scales, table, bs, scale):
    """q [H, D], one new token over `length` tokens, all seen.  Returns (out, tol, parts): out and tol
    [H, D], and for each kv head the softmax's weights [H / Hk, length] and the values [length, D].  With
    A = sum p |v|: the weights' two bf16 leave half a step of 16 bits, 2^-16 A; scores and fp32 sums as in
    attn_ref.attend64; the result's own rounding 2^-8 |out|."""
    H, D = q.shape
    Hk = pages[0].shape[1]
    G = H // Hk
    outs, tols, parts = [], [], []
    for g in range(Hk):
        k, v = ref.load(pages, scales, table, bs, length, g)
        x = q[g * G:(g + 1) * G].double()
        p = torch.softmax(x @ k.T * scale, 1)
        a, o = p @ v.abs(), p @ v
        smax = (x.abs() @ k.abs().T * scale).amax(1, keepdim=True)
        outs.append(o)
        tols.append(a * (1.01 * 2.0 ** -16 + 2 * (D + 8) * 2.0 ** -24 * smax + (length + 64) * 2.0 ** -23) + 2.0 ** -8 * o.abs()
                    + 1e-30)
        parts.append((p, v))
    return torch.cat(outs), torch.cat(tols), parts


def bf16_cut(x):
    """x without the bits that bf16 has no room for."""
    return (x.float().view(torch.int32) & -65536).view(torch.float32).double()
