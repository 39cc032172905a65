"""CPU test: the bound of decode's results (attn_bits.py) holds weights of 16 bits and fails weights of bf16."""
import pytest
import torch

import attn_bits as bits
import attn_ref as ref


@pytest.mark.parametrize("length", [2, 17, 100, 600])
@pytest.mark.parametrize("H,Hk,D,bs", [(64, 8, 64, 16), (32, 8, 128, 32)])
def test_bound_tells_the_weights_apart(length, H, Hk, D, bs):
    gen = torch.Generator().manual_seed(5)
    blocks = (length + bs - 1) // bs
    pages = [torch.randn((blocks, Hk, bs, D), generator=gen).to(torch.bfloat16) for _ in range(2)]
    table = torch.randperm(blocks, generator=gen)
    q = (0.5 * torch.randn((H, D), generator=gen)).to(torch.bfloat16)
    out, tol, parts = bits.decode64(q, length, pages, [None, None], table, bs, D ** -0.5)
    over = {}
    for name, form in (("16 bits", lambda p: bits.bf16_cut(p) + (p - bits.bf16_cut(p)).to(torch.bfloat16).double()),
                       ("cut to bf16", bits.bf16_cut), ("rounded to bf16", lambda p: p.to(torch.bfloat16).double()),
                       ("second part swapped", lambda p: bits.bf16_cut(p) + (p - bits.bf16_cut(p)).roll(1, 1))):
        got = torch.cat([form(p) @ v for p, v in parts]).to(torch.bfloat16)
        over[name] = ((got.double() - out).abs() > tol).double().mean().item()
    assert over.pop("16 bits") == 0
    assert min(over.values()) > 0.005, over  # dozens of elements in every case
