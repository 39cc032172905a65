"""GPU: the layer stack's decode step with attention from this library in its hook.  Per layer the hook runs
the input norm, the MXFP4 projection to queries, keys and values, the rotation with the append to the layer's
paged cache, attention of the new tokens over it (a window in every other layer) and the output projection, all
on the stack's stream, so that the whole step is one captured graph."""
import ctypes

import numpy as np
import pytest

import attn_ref as ref
import ckpt_data
import moe_data
from test_gpu_parity import dev, say

pytestmark = pytest.mark.gpu

E, K, H, I, NL = 8, 4, 256, 128, 3
NH, HK, D, BS, WINDOW = 8, 2, 64, 16, 24
QKV = (NH + 2 * HK) * D
MAX_T = 4


@pytest.fixture(scope="module")
def torch_mod():
    import torch
    return torch


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    ws = [moe_data.make_layer(700 + l, E, H, I, bias="random") for l in range(NL)]
    norms = [moe_data.bf16(np.random.default_rng(710 + l).normal(1.0, 0.1, H)) for l in range(NL)]
    t = {}
    for l in range(NL):
        t.update(ckpt_data.layer_tensors(l, ws[l], E, H, I, norm_w=norms[l]))
    d = tmp_path_factory.mktemp("attn_stack_ckpt")
    ckpt_data.write_shards(str(d), t, n_shards=1)
    return str(d)


class Attention:
    """The attention halves of NL layers: weights, caches, and buffers with fixed addresses."""

    def __init__(self, gpu, torch, like=None):
        """With `like` a second one of the same weights, whose caches hold the same."""
        self.gpu, self.lib, gen = gpu, gpu.lib, torch.Generator(device="cuda").manual_seed(5)
        bf, i32 = (lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")), \
            (lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda"))

        def mxfp4(N, K_):
            codes = torch.randint(0, 256, (N, K_ // 2), dtype=torch.uint8, device="cuda", generator=gen)
            scales = torch.randint(119, 122, (N, K_ // 32), dtype=torch.uint8, device="cuda", generator=gen)
            return gpu.pack_tiled(codes, scales, N, K_)

        def randn(*s, scale):
            return (scale * torch.randn(s, device="cuda", generator=gen)).to(torch.bfloat16)

        self.w = like.w if like else [dict(qkv=mxfp4(QKV, H), o=mxfp4(H, NH * D), norm=randn(H, scale=0.1) + 1,
                                  bias=randn(QKV, scale=0.1), sinks=randn(NH, scale=1.0)) for _ in range(NL)]
        self.caches = []
        for layer in range(NL):
            if like:
                c = like.caches[layer]
                pages, scales = (c.k.clone(), c.v.clone()), (c.k_scale, c.v_scale)
            else:
                pages, scales = ref.make_cache(gen, 40, HK, BS, D, e4m3=layer == 1)
            self.caches.append(gpu.KVCache(pages[0], pages[1], scales[0], scales[1]))
        self.tables = torch.arange(40, dtype=torch.int32, device="cuda").view(MAX_T, 10).flip(1).contiguous()
        self.rope = gpu.rope_table()
        self.pos, self.slots, self.lens = i32(MAX_T), i32(MAX_T), i32(MAX_T)
        self.zeros, self.normed, self.proj = bf(MAX_T, H), bf(MAX_T, H), bf(MAX_T, QKV)
        self.q = [bf(MAX_T, NH * D) for _ in range(NL)]
        self.out = [bf(MAX_T, NH * D) for _ in range(NL)]
        need = gpu.paged_attention_workspace_bytes(MAX_T, MAX_T, NH, self.caches[0])
        self.ws = torch.zeros(need, dtype=torch.uint8, device="cuda")

    def at(self, torch, pos):
        p = torch.tensor(pos, dtype=torch.int32, device="cuda")
        rows = torch.arange(len(pos), device="cuda")
        self.pos[: len(pos)].copy_(p)
        self.slots[: len(pos)].copy_(self.tables[rows, (p // BS).long()] * BS + p % BS)
        self.lens[: len(pos)].copy_(p + 1)

    def hook(self, layer, residual, delta, T, stream):
        g, w, check = self.gpu, self.w[layer], self.gpu.check
        check(self.lib.gptoss_fused_residual_rmsnorm_forward(residual, self.zeros.data_ptr(), w["norm"].data_ptr(),
                                                             self.normed.data_ptr(), None, T, H, ctypes.c_float(1e-5), stream))
        check(self.lib.gptoss_mxfp4_gemv_forward(self.normed.data_ptr(), T, w["qkv"][0].data_ptr(), w["qkv"][1].data_ptr(),
                                                 w["bias"].data_ptr(), self.proj.data_ptr(), QKV, H, stream))
        g.rope_kv_append(self.proj[:T], self.pos[:T], self.slots[:T], self.rope, self.caches[layer], NH,
                         q_out=self.q[layer][:T], stream=stream)
        g.paged_attention_decode(self.q[layer][:T], self.caches[layer], self.tables[:T], self.lens[:T],
                                 window=WINDOW if layer % 2 == 0 else 0, sinks=w["sinks"], out=self.out[layer][:T],
                                 workspace=self.ws, stream=stream)
        check(self.lib.gptoss_mxfp4_gemv_forward(self.out[layer].data_ptr(), T, w["o"][0].data_ptr(), w["o"][1].data_ptr(),
                                                 None, delta, H, NH * D, stream))


def test_stack_step_with_attention(gpu, torch_mod, model):
    torch = torch_mod
    cfg = gpu.default_config(E, MAX_T, decode_exact=True)
    cfg.hidden_size, cfg.intermediate_size, cfg.top_k = H, I, K
    with gpu.Checkpoint(model) as ck:
        eager_stack, graph_stack = (gpu.MoEStack.from_checkpoint(cfg, 0, ck) for _ in range(2))
    eager = Attention(gpu, torch)
    graph = Attention(gpu, torch, like=eager)
    T, start = 3, [0, 5, 31]
    for a in (eager, graph):  # what the sequences hold already
        gen = torch.Generator(device="cuda").manual_seed(9)
        for c in a.caches:
            for b, n in enumerate(start):
                if n:
                    ref.store((c.k, c.v), (c.k_scale, c.v_scale), a.tables[b], BS,
                              [torch.randn((n, HK, D), device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2)])
    hooks = (eager.hook, graph.hook)
    for step in range(6):
        pos = [n + step for n in start]
        x, _ = moe_data.make_tokens(800 + step, T, H)
        outs = []
        for st, a, hook, use_graph in ((eager_stack, eager, hooks[0], False), (graph_stack, graph, hooks[1], True)):
            a.at(torch, pos)
            st.residual[:T].copy_(dev(x, torch))
            outs.append(st.decode_step(T, hook=hook, use_graph=use_graph).clone())
            torch.cuda.synchronize()
        say("stack step with attention", step)
        assert torch.equal(outs[0], outs[1]), step
        assert torch.isfinite(outs[0].float()).all()
        for layer in range(NL):
            assert torch.equal(eager.q[layer], graph.q[layer]) and torch.equal(eager.out[layer], graph.out[layer])
            c = graph.caches[layer]
            for b in range(T):
                o, tol = ref.attend64(graph.q[layer][b:b + 1].view(1, NH, D), [pos[b]], pos[b] + 1, (c.k, c.v),
                                      (c.k_scale, c.v_scale), graph.tables[b], BS, D ** -0.5,
                                      WINDOW if layer % 2 == 0 else 0, 0, graph.w[layer]["sinks"])
                bad = ref.within(graph.out[layer][b:b + 1].view(1, NH, D), o, tol)
                assert bad is None, (step, layer, b, bad)
    eager_stack.destroy()
    graph_stack.destroy()
