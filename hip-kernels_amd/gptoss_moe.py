"""Python host binding of libgptoss_moe.so (the gfx950 GPT-OSS MoE block).

Mirrors the reference's MoE operator interface (src/model/moe_layer.cu:
1556-1615: moe_layer_create / init / forward / forward_prenormed /
get_ffn_norm_weight / destroy) and its kernel launchers, over the C ABI
declared in include/gptoss_moe.h; attention over a paged key-value cache
(KVCache, rope_kv_append, paged_attention_decode, paged_attention_prefill); routing by scores, bias and groups
(select_experts); and MXFP4 matrices (MXFP4Matrix, mxfp4_quantize, mxfp4_dequantize, mxfp4_matmul,
grouped_mxfp4_matmul).  Device memory is held in torch tensors
(plumbing only); every computation runs in the HIP library, and importing
this module without the built library raises immediately.

bf16 tensors are passed as torch.bfloat16 (or their int16/uint16 bit views).
"""
from __future__ import annotations

import ctypes
import functools
import os
import struct
from dataclasses import dataclass

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
# GPTOSS_MOE_LIB: another build of the same library (the sanitizer build of
# tests/sanitize loads its instrumented copy this way)
LIB_PATH = os.environ.get("GPTOSS_MOE_LIB") or os.path.join(HERE, "libgptoss_moe.so")

if not os.path.exists(LIB_PATH):
    raise ImportError(f"{LIB_PATH} is not built; run __graft_entry__.build() (make -C hip-kernels_amd)")

_lib = ctypes.CDLL(LIB_PATH)

_P = ctypes.c_void_p
_I = ctypes.c_int
_F = ctypes.c_float
_SZ = ctypes.c_size_t

GPTOSS_OK = 0
GPTOSS_ERR_INVALID = 1
GPTOSS_ERR_UNSUPPORTED = 2
GPTOSS_ERR_HIP = 3
GPTOSS_ERR_STATE = 4
GPTOSS_ERR_OOM = 5
GPTOSS_ERR_NOT_FOUND = 6
GPTOSS_ERR_IO = 7


class GptossError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"[gptoss_moe status {code}] {msg}")
        self.code = code


class ValueErrorG(GptossError, ValueError):
    """Invalid argument (status GPTOSS_ERR_INVALID); also a ValueError, as the
    reference bindings map argument errors to ValueError (bindings.cpp:105-116)."""


class MoeConfig(ctypes.Structure):
    _fields_ = [("hidden_size", _I), ("num_experts", _I), ("top_k", _I), ("intermediate_size", _I),
                ("swiglu_alpha", _F), ("swiglu_limit", _F), ("rms_norm_eps", _F), ("logits_fp32", _I),
                ("max_tokens", _I), ("prefill_min_tokens", _I), ("decode_exact", _I),
                ("prefill_block_scaled", _I)]


class MoeWeights(ctypes.Structure):
    _fields_ = [("moe_norm_weight", _P), ("router_weight", _P), ("router_bias", _P),
                ("gate_up_bias", _P), ("down_bias", _P),
                ("mlp1_packed", ctypes.POINTER(_P)), ("mlp1_scales", ctypes.POINTER(_P)),
                ("mlp2_packed", ctypes.POINTER(_P)), ("mlp2_scales", ctypes.POINTER(_P)),
                ("mlp1_tiled_nibbles", _P), ("mlp1_tiled_scales", _P),
                ("mlp2_tiled_nibbles", _P), ("mlp2_tiled_scales", _P)]


class MoeTrace(ctypes.Structure):
    _fields_ = [("logits", _P), ("expert_indices", _P), ("expert_weights", _P), ("expert_counts", _P),
                ("expert_offsets", _P), ("gather_map", _P), ("perm_token", _P), ("active_experts", _P),
                ("n_active", _P), ("gate_up", _P), ("act", _P), ("expert_out", _P)]


class TensorInfo(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char_p), ("dtype", ctypes.c_char_p), ("ndim", _I),
                ("shape", ctypes.c_int64 * 8), ("nbytes", ctypes.c_uint64), ("data", _P), ("shard", _I)]


class ProfRecord(ctypes.Structure):
    _fields_ = [("host_us", ctypes.c_double), ("num_tokens", _I), ("prefill", _I),
                ("start_ms", _F * 4), ("dur_ms", _F * 4)]


class KvCacheDesc(ctypes.Structure):
    _fields_ = [("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P),
                ("block_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("dtype", _I), ("num_blocks", _I), ("block_size", _I), ("num_kv_heads", _I), ("head_dim", _I)]


class RopeConfig(ctypes.Structure):
    _fields_ = [("rotary_dim", _I), ("max_positions", _I), ("theta", ctypes.c_double),
                ("scaling_factor", ctypes.c_double), ("original_positions", ctypes.c_double),
                ("beta_fast", ctypes.c_double), ("beta_slow", ctypes.c_double)]


class AttentionConfig(ctypes.Structure):
    _fields_ = [("scale", _F), ("window", _I), ("first_tokens", _I), ("sinks", _P)]


class RoutingConfig(ctypes.Structure):
    _fields_ = [("score", _I), ("top_k", _I), ("num_groups", _I), ("top_groups", _I), ("group_rank", _I),
                ("renormalize", _I), ("scale", _F)]


class Mxfp4Result(ctypes.Structure):
    _fields_ = [("swiglu", _I), ("alpha", _F), ("limit", _F), ("out_fp32", _I), ("out", _P),
                ("out_stride", ctypes.c_int64), ("out_packed", _P), ("out_scales", _P)]


_pack_result = struct.Struct("@iffiPqPP").pack  # an Mxfp4Result's bytes, in a third of its time


def _sig(name, args, res=_I):
    f = getattr(_lib, name)
    f.argtypes = args
    f.restype = res
    return f


_sig("gptoss_last_error", [], ctypes.c_char_p)
_sig("gptoss_abi_version", [])
_sig("gptoss_moe_config_default", [ctypes.POINTER(MoeConfig), _I, _I])
_sig("gptoss_mxfp4_tiled_size", [_I, _I, ctypes.POINTER(_SZ), ctypes.POINTER(_SZ)])
_sig("gptoss_mxfp4_pack_tiled", [_P, _P, _I, _I, _P, _P, _P])
_sig("gptoss_moe_layer_create", [], _P)
_sig("gptoss_moe_layer_init", [_P, ctypes.POINTER(MoeConfig), _I, ctypes.POINTER(MoeWeights)])
_sig("gptoss_moe_layer_workspace_bytes", [ctypes.POINTER(MoeConfig)], _SZ)
_sig("gptoss_moe_layer_init_with_workspace", [_P, ctypes.POINTER(MoeConfig), _I, ctypes.POINTER(MoeWeights), _P,
                                               _SZ])
_sig("gptoss_moe_layer_forward", [_P, _P, _P, _I, _P])
_sig("gptoss_moe_layer_forward_prenormed", [_P, _P, _P, _P, _I, _P])
_sig("gptoss_moe_layer_forward_residual", [_P, _P, _P, _P, _P, _I, _P])
_sig("gptoss_moe_layer_forward_routed", [_P, _P, _P, _P, _P, _P, _I, _P])
_sig("gptoss_moe_layer_forward_prenormed_noalloc", [_P, _P, _P, _P, _I, _P])
_sig("gptoss_moe_layer_get_ffn_norm_weight", [_P], _P)
_sig("gptoss_moe_layer_destroy", [_P], None)
_sig("gptoss_moe_layer_init_from_checkpoint", [_P, ctypes.POINTER(MoeConfig), _I, _P, _I])
_sig("gptoss_checkpoint_open", [ctypes.c_char_p, ctypes.POINTER(_P)])
_sig("gptoss_checkpoint_close", [_P], None)
_sig("gptoss_checkpoint_num_tensors", [_P])
_sig("gptoss_checkpoint_tensor_at", [_P, _I, ctypes.POINTER(TensorInfo)])
_sig("gptoss_checkpoint_find", [_P, ctypes.c_char_p, ctypes.POINTER(TensorInfo)])
_sig("gptoss_checkpoint_set_staging_bytes", [_P, _SZ])
_sig("gptoss_moe_layer_get_config", [_P, ctypes.POINTER(MoeConfig), ctypes.POINTER(_I)])
_HOOK = ctypes.CFUNCTYPE(None, _P, _I, _P, _P, _I, _P)
_sig("gptoss_moe_stack_create", [ctypes.POINTER(MoeConfig), _I, _P, _I, _I, ctypes.POINTER(_P)])
_sig("gptoss_moe_stack_create_from_layers", [ctypes.POINTER(_P), _I, ctypes.POINTER(_P)])
_sig("gptoss_moe_stack_io", [_P, ctypes.POINTER(_P), ctypes.POINTER(_P), ctypes.POINTER(_I), ctypes.POINTER(_I)])
_sig("gptoss_moe_stack_bind", [_P, _P, _P])
_sig("gptoss_moe_stack_layer", [_P, _I, ctypes.POINTER(_P)])
_sig("gptoss_moe_stack_decode_step", [_P, _I, _HOOK, _P, _I, _P])
_sig("gptoss_moe_stack_destroy", [_P], None)
_sig("gptoss_moe_layer_trace", [_P, ctypes.POINTER(MoeTrace)])
_sig("gptoss_moe_layer_set_trace_gate_up", [_P, _I])
_sig("gptoss_moe_layer_set_profiling", [_P, _I])
_sig("gptoss_moe_layer_profile_read", [_P, ctypes.POINTER(_F), ctypes.POINTER(_F), ctypes.POINTER(_F),
                                        ctypes.POINTER(_F), ctypes.POINTER(_I)])
_sig("gptoss_moe_layer_profile_records", [_P, ctypes.POINTER(ProfRecord), _I, ctypes.POINTER(_I)])
_sig("gptoss_moe_route_scratch_bytes", [_I, _I, _I], _SZ)
_sig("gptoss_moe_route", [_P, _P, _P, _I, _I, _I, _I, _I, _P, _P, _P, _P, _P])
_sig("gptoss_topk_softmax_forward", [_P, _I, _P, _P, _P, _I, _I, _I, _P])
_sig("gptoss_moe_permute_plan", [_P, _I, _I, _I, _P, _P, _P, _P, _P, _P, _P])
_sig("gptoss_moe_scatter_tokens", [_P, _P, _P, _I, _I, _I, _P])
_sig("gptoss_mxfp4_gemv_forward", [_P, _I, _P, _P, _P, _P, _I, _I, _P])
_sig("gptoss_swiglu_forward", [_P, _P, _I, _I, _F, _F, _P])
_sig("gptoss_fused_residual_rmsnorm_forward", [_P, _P, _P, _P, _P, _I, _I, _F, _P])
_sig("gptoss_moe_combine_forward", [_P, _P, _P, _P, _P, _I, _I, _I, _P])
_sig("gptoss_mxfp4_dequant", [_P, _P, _I, _I, _P, _P])
_sig("gptoss_moe_grouped_mxfp4_gemm", [_P, _P, _P, _I, _I, _P, _P, _P, _I, _I, _I, _F, _F, _P, _P, _P])
_L = ctypes.c_int64
_sig("gptoss_rope_config_default", [ctypes.POINTER(RopeConfig)])
_sig("gptoss_rope_table", [ctypes.POINTER(RopeConfig), _P, _P])
_sig("gptoss_rope_kv_append", [_P, _L, _P, _P, _P, _I, _I, _I, _I, _I, _P, _L, _P, _P])
_sig("gptoss_paged_attention_workspace_bytes", [_I, _I, _I, _I, _I], _SZ)
_sig("gptoss_paged_attention_call_bytes", [_I, _I, _I, _I, _I, ctypes.c_int64, _I, _I], _SZ)
_sig("gptoss_paged_attention_decode", [_P, _L, _P, _P, _L, _I, _P, _I, _I, _P, _P, _L, _P, _SZ, _P])
_sig("gptoss_paged_attention_prefill", [_P, _L, _P, _I, _P, _P, _L, _I, _P, _I, _I, _P, _P, _L, _P, _SZ, _P])
_sig("gptoss_moe_select_experts", [_P, _L, _I, _P, _I, _I, _P, _P, _P, _P])
_sig("gptoss_mxfp4_quantize", [_P, _L, _I, _I, _I, _P, _P, _P])
_sig("gptoss_mxfp4_dequantize", [_P, _P, _I, _I, _P, _L, _I, _P])
_sig("gptoss_mxfp4_matmul", [_P, _P, _I, _P, _P, _P, _I, _I, _P, _P])
_sig("gptoss_moe_grouped_mxfp4_matmul", [_P, _P, _I, _P, _P, _I, _I, _P, _P, _P, _I, _I, _P, _P])

lib = _lib


def check(rc: int) -> None:
    if rc != GPTOSS_OK:
        msg = _lib.gptoss_last_error().decode()
        if rc == GPTOSS_ERR_INVALID:
            raise ValueErrorG(rc, msg)
        raise GptossError(rc, msg)


def _ptr(t):
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


def _bad(msg: str):
    raise ValueErrorG(GPTOSS_ERR_INVALID, msg)


def _check_tensor(name: str, t, device: int, dtype_size: int, cols: int, rows: int | None = None,
                  dtypes=None) -> None:
    """A contiguous 2-D tensor on cuda:`device` with `cols` columns (and
    `rows` rows when given) of `dtype_size`-byte elements; dtypes, when given,
    is the set of accepted torch dtypes.  The kernels read and write raw rows
    of that shape, so anything else is refused before the library sees it."""
    if not isinstance(t, torch.Tensor):
        _bad(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dim() != 2:
        _bad(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    if t.shape[1] != cols or (rows is not None and t.shape[0] != rows):
        want = f"[{rows if rows is not None else 'T'}, {cols}]"
        _bad(f"{name} has shape {tuple(t.shape)}, expected {want}")
    if dtypes is not None and t.dtype not in dtypes:
        _bad(f"{name} has dtype {t.dtype}, expected one of {sorted(str(d) for d in dtypes)}")
    if t.element_size() != dtype_size:
        _bad(f"{name} has {t.element_size()}-byte elements, expected {dtype_size}")
    if not t.is_contiguous():
        _bad(f"{name} must be contiguous")
    if t.device.type != "cuda" or t.device.index != device:
        _bad(f"{name} is on {t.device}, the layer is on cuda:{device}")


_BF16 = (torch.bfloat16, torch.int16, torch.uint16)


def _stream(stream):
    if stream is None:
        return torch.cuda.current_stream().cuda_stream if torch.cuda.is_available() else None
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def default_config(num_experts: int = 128, max_tokens: int = 64, logits_fp32: bool = False,
                   prefill_min_tokens: int | None = None, decode_exact: bool = False,
                   prefill_block_scaled: int | None = None) -> MoeConfig:
    cfg = MoeConfig()
    check(_lib.gptoss_moe_config_default(ctypes.byref(cfg), num_experts, max_tokens))
    cfg.logits_fp32 = 1 if logits_fp32 else 0
    if prefill_min_tokens is not None:
        cfg.prefill_min_tokens = prefill_min_tokens
    cfg.decode_exact = 1 if decode_exact else 0
    if prefill_block_scaled is not None:
        cfg.prefill_block_scaled = int(prefill_block_scaled)
    return cfg


def workspace_bytes(cfg: MoeConfig) -> int:
    """Bytes of forward scratch a layer of this config needs (0: invalid config)."""
    return _lib.gptoss_moe_layer_workspace_bytes(ctypes.byref(cfg))


def tiled_size(N: int, K: int):
    nb = _SZ()
    sb = _SZ()
    check(_lib.gptoss_mxfp4_tiled_size(N, K, ctypes.byref(nb), ctypes.byref(sb)))
    return nb.value, sb.value


def pack_tiled(packed: torch.Tensor, scales: torch.Tensor, N: int, K: int, out_nib=None, out_sc=None, stream=None):
    """Reference-layout MXFP4 [N][K/2] + [N][K/32] (uint8, device) -> tiled layout."""
    nb, sb = tiled_size(N, K)
    if out_nib is None:
        out_nib = torch.empty(nb, dtype=torch.uint8, device=packed.device)
    if out_sc is None:
        out_sc = torch.empty(sb, dtype=torch.uint8, device=packed.device)
    check(_lib.gptoss_mxfp4_pack_tiled(_ptr(packed), _ptr(scales), N, K, _ptr(out_nib), _ptr(out_sc),
                                       _stream(stream)))
    return out_nib, out_sc


@dataclass
class Trace:
    logits: int
    expert_indices: int
    expert_weights: int
    expert_counts: int
    expert_offsets: int
    gather_map: int
    perm_token: int
    active_experts: int
    n_active: int
    gate_up: int
    act: int
    expert_out: int


class MoELayer:
    """gptoss::MoELayer replacement (moe_layer.cu:607-1549) on one GPU.

    init() takes either the reference per-expert MXFP4 tables (lists of device
    tensors, packed and tiled by the library) or pre-tiled expert-major
    buffers (borrowed).  Tensors passed to init() must outlive the layer."""

    def __init__(self):
        self._h = _lib.gptoss_moe_layer_create()
        if not self._h:
            raise GptossError(GPTOSS_ERR_OOM, "gptoss_moe_layer_create failed")
        self._keep = []
        self._owned = True
        self.cfg = None
        self.device = None

    @classmethod
    def _borrow(cls, handle: int) -> "MoELayer":
        """A view of a layer owned elsewhere (a stack's); destroy() is a no-op."""
        self = cls.__new__(cls)
        self._h, self._keep, self._owned = handle, [], False
        self.cfg = MoeConfig()
        dev = _I()
        check(_lib.gptoss_moe_layer_get_config(handle, ctypes.byref(self.cfg), ctypes.byref(dev)))
        self.device = dev.value
        return self

    def init(self, cfg: MoeConfig, device_id: int, router_weight, router_bias=None, gate_up_bias=None,
             down_bias=None, moe_norm_weight=None, mlp1=None, mlp2=None, tiled=None,
             workspace=None) -> "MoELayer":
        """mlp1/mlp2: (list of packed tensors, list of scale tensors) per expert.
        tiled: (w1_nibbles, w1_scales, w2_nibbles, w2_scales) expert-major buffers.
        workspace: a device tensor of at least workspace_bytes(cfg) bytes for
        the forward scratch, shareable by layers run one after another on one
        stream (None: the layer allocates its own)."""
        wt = MoeWeights()
        wt.moe_norm_weight = _ptr(moe_norm_weight)
        wt.router_weight = _ptr(router_weight)
        wt.router_bias = _ptr(router_bias)
        wt.gate_up_bias = _ptr(gate_up_bias)
        wt.down_bias = _ptr(down_bias)
        if tiled is not None:
            wt.mlp1_tiled_nibbles, wt.mlp1_tiled_scales, wt.mlp2_tiled_nibbles, wt.mlp2_tiled_scales = (
                _ptr(t) for t in tiled)
        else:
            arrs = []
            for lst in (mlp1[0], mlp1[1], mlp2[0], mlp2[1]):
                a = (_P * len(lst))(*[_ptr(t) for t in lst])
                arrs.append(a)
            self._keep.append(arrs)
            wt.mlp1_packed = ctypes.cast(arrs[0], ctypes.POINTER(_P))
            wt.mlp1_scales = ctypes.cast(arrs[1], ctypes.POINTER(_P))
            wt.mlp2_packed = ctypes.cast(arrs[2], ctypes.POINTER(_P))
            wt.mlp2_scales = ctypes.cast(arrs[3], ctypes.POINTER(_P))
        if workspace is None:
            check(_lib.gptoss_moe_layer_init(self._h, ctypes.byref(cfg), device_id, ctypes.byref(wt)))
        else:
            nbytes = workspace.numel() * workspace.element_size()
            check(_lib.gptoss_moe_layer_init_with_workspace(self._h, ctypes.byref(cfg), device_id, ctypes.byref(wt),
                                                            _ptr(workspace), nbytes))
            self._keep.append(workspace)
        self.cfg = cfg
        self.device = device_id
        return self

    def init_from_checkpoint(self, cfg: MoeConfig, device_id: int, ckpt: "Checkpoint",
                             layer_index: int) -> "MoELayer":
        """Layer `layer_index` of a safetensors checkpoint (WeightLoader's MoE
        part, weight_loader.cu:1083-1165): the layer owns one device
        allocation with every weight, the experts already tiled."""
        check(_lib.gptoss_moe_layer_init_from_checkpoint(self._h, ctypes.byref(cfg), device_id, ckpt._h,
                                                         layer_index))
        self.cfg = cfg
        self.device = device_id
        return self

    def _rows(self, name: str, t, T: int | None = None) -> int:
        """Checks a bf16 [T, hidden_size] activation tensor on the layer's
        device; returns T."""
        if self.cfg is None:
            raise GptossError(GPTOSS_ERR_STATE, "layer not initialised")
        _check_tensor(name, t, self.device, 2, self.cfg.hidden_size, T, _BF16)
        return t.shape[0]

    def _out(self, out, like, T: int):
        if out is None:
            return torch.empty_like(like)
        self._rows("out", out, T)
        return out

    def forward(self, x, out=None, stream=None):
        """out = x + MoE(RMSNorm(x)) (moe_layer_forward)."""
        T = self._rows("x", x)
        out = self._out(out, x, T)
        check(_lib.gptoss_moe_layer_forward(self._h, _ptr(x), _ptr(out), T, _stream(stream)))
        return out

    def forward_prenormed(self, normed, residual=None, out=None, stream=None):
        """out = residual + MoE(normed) (moe_layer_forward_prenormed)."""
        T = self._rows("normed", normed)
        if residual is not None:
            self._rows("residual", residual, T)
        out = self._out(out, normed, T)
        check(_lib.gptoss_moe_layer_forward_prenormed(self._h, _ptr(normed), _ptr(residual), _ptr(out), T,
                                                      _stream(stream)))
        return out

    def forward_prenormed_noalloc(self, normed, residual=None, out=None, stream=None):
        """forward_prenormed with the forward scratch in the library's static
        device array (no allocation; up to 64 tokens; calls overlapping on one
        GPU race).  `out` must be given: this call allocates nothing."""
        if out is None:
            _bad("forward_prenormed_noalloc needs an output tensor (it allocates nothing)")
        T = self._rows("normed", normed)
        if residual is not None:
            self._rows("residual", residual, T)
        self._rows("out", out, T)
        check(_lib.gptoss_moe_layer_forward_prenormed_noalloc(self._h, _ptr(normed), _ptr(residual), _ptr(out), T,
                                                              _stream(stream)))
        return out

    def forward_residual(self, residual, delta, residual_out=None, out=None, stream=None):
        """The decode step's residual add + RMSNorm + MoE in one call:
        s = residual + delta; residual_out (optional) = bf16(s);
        out = bf16(s) + MoE(RMSNorm(s)).  residual_out must not share memory
        with residual or delta.  Returns out."""
        T = self._rows("residual", residual)
        self._rows("delta", delta, T)
        if residual_out is not None:
            self._rows("residual_out", residual_out, T)
        out = self._out(out, residual, T)
        check(_lib.gptoss_moe_layer_forward_residual(self._h, _ptr(residual), _ptr(delta), _ptr(residual_out),
                                                     _ptr(out), T, _stream(stream)))
        return out

    def forward_routed(self, normed, expert_indices, expert_weights, residual=None, out=None, stream=None):
        """out = residual + sum_k w * FFN_idx(normed) with the routing given
        (int32 [T][k] indices, fp32 [T][k] weights, on the device)."""
        T = self._rows("normed", normed)
        if residual is not None:
            self._rows("residual", residual, T)
        k = self.cfg.top_k
        _check_tensor("expert_indices", expert_indices, self.device, 4, k, T, (torch.int32,))
        _check_tensor("expert_weights", expert_weights, self.device, 4, k, T, (torch.float32,))
        out = self._out(out, normed, T)
        check(_lib.gptoss_moe_layer_forward_routed(self._h, _ptr(normed), _ptr(residual), _ptr(expert_indices),
                                                   _ptr(expert_weights), _ptr(out), T, _stream(stream)))
        return out

    def get_ffn_norm_weight(self) -> int:
        return _lib.gptoss_moe_layer_get_ffn_norm_weight(self._h) or 0

    def set_trace_gate_up(self, enable: bool) -> None:
        check(_lib.gptoss_moe_layer_set_trace_gate_up(self._h, 1 if enable else 0))

    def set_profiling(self, max_forwards: int) -> None:
        check(_lib.gptoss_moe_layer_set_profiling(self._h, max_forwards))

    def profile_read(self):
        """(route_ms, w1_ms, w2_ms, combine_ms, n_forwards) summed over the
        recorded forwards (route_ms is the plan launch for forward_routed)."""
        r, a, b, c, n = _F(), _F(), _F(), _F(), _I()
        check(_lib.gptoss_moe_layer_profile_read(self._h, ctypes.byref(r), ctypes.byref(a), ctypes.byref(b),
                                                 ctypes.byref(c), ctypes.byref(n)))
        return r.value, a.value, b.value, c.value, n.value

    def profile_records(self):
        """Per recorded forward: dict(host_us, num_tokens, prefill, start_ms[4],
        dur_ms[4]) for the route (or plan), gate_up, down and combine launches."""
        n = _I()
        check(_lib.gptoss_moe_layer_profile_records(self._h, None, 0, ctypes.byref(n)))
        recs = (ProfRecord * max(n.value, 1))()
        check(_lib.gptoss_moe_layer_profile_records(self._h, recs, n.value, ctypes.byref(n)))
        return [dict(host_us=r.host_us, num_tokens=r.num_tokens, prefill=r.prefill,
                     start_ms=list(r.start_ms), dur_ms=list(r.dur_ms)) for r in recs[:n.value]]

    def trace(self) -> Trace:
        t = MoeTrace()
        check(_lib.gptoss_moe_layer_trace(self._h, ctypes.byref(t)))
        return Trace(*[getattr(t, f[0]) or 0 for f in MoeTrace._fields_])

    def destroy(self) -> None:
        if self._h:
            if self._owned:
                _lib.gptoss_moe_layer_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


class Checkpoint:
    """A safetensors checkpoint (a directory of shards or one file), mapped
    read-only: WeightLoader's shard scan, header parse and name index
    (weight_loader.cu:297-345, 456-575).  Host-only: opening and reading
    tensors needs no GPU."""

    _NP = {"BF16": "<u2", "F16": "<f2", "F32": "<f4", "F64": "<f8", "U8": "u1", "I8": "i1", "BOOL": "u1",
           "I16": "<i2", "U16": "<u2", "I32": "<i4", "U32": "<u4", "I64": "<i8", "U64": "<u8"}

    def __init__(self, path: str):
        h = _P()
        check(_lib.gptoss_checkpoint_open(os.fsencode(path), ctypes.byref(h)))
        self._h = h.value

    def __len__(self) -> int:
        return _lib.gptoss_checkpoint_num_tensors(self._h)

    @staticmethod
    def _info(ti: TensorInfo) -> dict:
        return {"name": ti.name.decode(), "dtype": ti.dtype.decode(), "shape": tuple(ti.shape[:ti.ndim]),
                "nbytes": ti.nbytes, "data": ti.data or 0, "shard": ti.shard}

    def names(self):
        out = []
        ti = TensorInfo()
        for i in range(len(self)):
            check(_lib.gptoss_checkpoint_tensor_at(self._h, i, ctypes.byref(ti)))
            out.append(ti.name.decode())
        return out

    def info(self, name: str):
        """dict(name, dtype, shape, nbytes, data, shard), or None when absent."""
        ti = TensorInfo()
        rc = _lib.gptoss_checkpoint_find(self._h, name.encode(), ctypes.byref(ti))
        if rc == GPTOSS_ERR_NOT_FOUND:
            return None
        check(rc)
        return self._info(ti)

    def numpy(self, name: str):
        """A copy of the tensor as a numpy array (bf16 as uint16; dtypes
        outside the safetensors list as flat bytes)."""
        import numpy as np
        inf = self.info(name)
        if inf is None:
            raise KeyError(name)
        raw = ctypes.string_at(inf["data"], inf["nbytes"]) if inf["nbytes"] else b""
        dt = self._NP.get(inf["dtype"])
        a = np.frombuffer(raw, dtype=dt or "u1")
        return (a.reshape(inf["shape"]) if dt else a).copy()

    def _router_weight(self, layer: int):
        for n in ("mlp.gate.weight", "mlp.router.weight"):
            inf = self.info(f"model.layers.{layer}.{n}")
            if inf is not None:
                return inf
        return None

    def num_moe_layers(self) -> int:
        """Layers 0, 1, ... that have a router weight."""
        n = 0
        while self._router_weight(n) is not None:
            n += 1
        return n

    def moe_shape(self, layer: int = 0):
        """(E, H, I) of a layer, from its router weight [E][H] and its gate_up
        blocks or biases ([E][2I]...)."""
        rw = self._router_weight(layer)
        if rw is None:
            raise GptossError(GPTOSS_ERR_NOT_FOUND, f"no router weight for layer {layer}")
        E, H = rw["shape"]
        P = f"model.layers.{layer}.mlp.experts."
        for n in ("gate_up_proj_blocks", "gate_up_proj_bias", "0.mlp1.weight", "0.gate_up_proj.weight",
                  "0.w1.weight"):
            inf = self.info(P + n)
            if inf is not None:
                return E, H, inf["shape"][1 if n.startswith("gate_up") else 0] // 2
        raise GptossError(GPTOSS_ERR_NOT_FOUND, f"no gate_up tensor for layer {layer}")

    def set_staging_bytes(self, nbytes: int) -> None:
        check(_lib.gptoss_checkpoint_set_staging_bytes(self._h, nbytes))

    def close(self) -> None:
        if getattr(self, "_h", None):
            _lib.gptoss_checkpoint_close(self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class MoEStack:
    """The MoE half of the engine's decode step over a stack of layers
    (transformer.cu:653-753): per layer, an optional hook writes the layer's
    delta from the current residual (the engine's attention), then
    residual = bf16(residual + delta) + MoE(RMSNorm(residual + delta)),
    in place.  decode_step(use_graph=True) replays one hipGraph per token
    count, captured on first use.  The residual and deltas live in torch
    tensors bound to the stack: `residual` [max_tokens][H] and `deltas`
    [num_layers][max_tokens][H], bf16."""

    def __init__(self, handle: int, layers=None):
        self._h = handle
        self._layers = layers  # layers borrowed by the stack, kept alive here
        self._hooks = {}
        r, d, mt, nl = _P(), _P(), _I(), _I()
        check(_lib.gptoss_moe_stack_io(self._h, ctypes.byref(r), ctypes.byref(d), ctypes.byref(mt), ctypes.byref(nl)))
        self.max_tokens, self.num_layers = mt.value, nl.value
        L0 = _P()
        check(_lib.gptoss_moe_stack_layer(self._h, 0, ctypes.byref(L0)))
        cfg, dev = MoeConfig(), _I()
        check(_lib.gptoss_moe_layer_get_config(L0.value, ctypes.byref(cfg), ctypes.byref(dev)))
        self.cfg, self.device = cfg, dev.value
        H = cfg.hidden_size
        device = torch.device("cuda", self.device)
        self.residual = torch.zeros((self.max_tokens, H), dtype=torch.bfloat16, device=device)
        self.deltas = torch.zeros((self.num_layers, self.max_tokens, H), dtype=torch.bfloat16, device=device)
        check(_lib.gptoss_moe_stack_bind(self._h, _ptr(self.residual), _ptr(self.deltas)))

    @classmethod
    def from_checkpoint(cls, cfg: MoeConfig, device_id: int, ckpt: "Checkpoint", first_layer: int = 0,
                        num_layers: int | None = None) -> "MoEStack":
        if num_layers is None:
            num_layers = ckpt.num_moe_layers() - first_layer
        h = _P()
        check(_lib.gptoss_moe_stack_create(ctypes.byref(cfg), device_id, ckpt._h, first_layer, num_layers,
                                           ctypes.byref(h)))
        return cls(h.value)

    @classmethod
    def from_layers(cls, layers) -> "MoEStack":
        arr = (_P * len(layers))(*[L._h for L in layers])
        h = _P()
        check(_lib.gptoss_moe_stack_create_from_layers(arr, len(layers), ctypes.byref(h)))
        return cls(h.value, layers=list(layers))

    def layer(self, i: int) -> MoELayer:
        h = _P()
        check(_lib.gptoss_moe_stack_layer(self._h, i, ctypes.byref(h)))
        return MoELayer._borrow(h.value)

    def _c_hook(self, hook):
        """One C function pointer per Python hook, so that the same hook
        finds its captured graph again."""
        if hook is None:
            return _HOOK()
        key = id(hook)
        if key not in self._hooks:
            def tramp(_user, layer, residual, delta, T, stream, _hook=hook):
                _hook(layer, residual or 0, delta or 0, T, stream or 0)
            self._hooks[key] = (hook, _HOOK(tramp))
        return self._hooks[key][1]

    def decode_step(self, T: int, hook=None, use_graph: bool = True, stream=None) -> torch.Tensor:
        """One step on residual[:T] with deltas[:, :T].  hook(layer,
        residual_ptr, delta_ptr, T, stream_ptr) runs before each layer (only
        while a graph is captured when use_graph).  Returns residual[:T]."""
        check(_lib.gptoss_moe_stack_decode_step(self._h, T, self._c_hook(hook), None, 1 if use_graph else 0,
                                                _stream(stream)))
        return self.residual[:T]

    def destroy(self) -> None:
        if getattr(self, "_h", None):
            _lib.gptoss_moe_stack_destroy(self._h)
            self._h = None
        self._layers = None

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


class ModelConfig:
    """The MoE constants of GPT-OSS-120B, as the reference's read-only
    gptoss.ModelConfig exposes them (bindings.cpp:317-400, config.h)."""
    num_layers = 36
    hidden_size = 2880
    num_experts = 128
    num_active_experts = 4
    expert_intermediate_size = 2880
    rms_norm_eps = 1e-5
    swiglu_alpha = 1.702
    swiglu_limit = 7.0


class MoEEngine:
    """The InferenceEngine lifecycle (bindings.cpp:221-311: init(weights_dir),
    shutdown(), is_initialized) over the MoE half of the model: init() loads
    every MoE layer of a safetensors checkpoint into one stack on one GPU;
    decode_step() runs the per-layer residual add + RMSNorm + MoE of the
    decode step for all layers, as one cached hipGraph per batch size.  The
    attention that produces each layer's delta is the caller's (a hook, or
    deltas written beforehand)."""

    def __init__(self):
        self._stack = None

    def init(self, weights_dir: str, max_tokens: int = 64, device_id: int = 0, num_layers: int | None = None,
             top_k: int = ModelConfig.num_active_experts) -> "MoEEngine":
        if self._stack is not None:
            raise GptossError(GPTOSS_ERR_STATE, "[MoEEngine] Already initialized")
        with Checkpoint(weights_dir) as ck:
            E, H, I = ck.moe_shape(0)
            cfg = default_config(E, max_tokens)
            cfg.hidden_size, cfg.intermediate_size, cfg.top_k = H, I, top_k
            self._stack = MoEStack.from_checkpoint(cfg, device_id, ck, 0, num_layers)
        return self

    @property
    def is_initialized(self) -> bool:
        return self._stack is not None

    @property
    def stack(self) -> MoEStack:
        if self._stack is None:
            raise GptossError(GPTOSS_ERR_STATE, "[MoEEngine] Not initialized")
        return self._stack

    def decode_step(self, hidden: torch.Tensor, deltas: torch.Tensor | None = None, hook=None,
                    use_graph: bool = True) -> torch.Tensor:
        """hidden [T][H] bf16 (the residual stream entering layer 0); deltas
        [num_layers][T][H] (or a hook).  Returns the residual after the last
        layer, [T][H]."""
        st = self.stack
        T = hidden.shape[0]
        st.residual[:T].copy_(hidden)
        if deltas is not None:
            st.deltas[:, :T].copy_(deltas)
        return st.decode_step(T, hook=hook, use_graph=use_graph).clone()

    def shutdown(self) -> None:
        if self._stack is not None:
            self._stack.destroy()
            self._stack = None

    def __repr__(self) -> str:
        n = self._stack.num_layers if self._stack is not None else 0
        return f"<gptoss_moe.MoEEngine initialized={self.is_initialized} layers={n}>"


# ---------------------------------------------------------------------------
# device buffer readback (for traces, which are raw device pointers)
# ---------------------------------------------------------------------------
_hip = None


def copy_device_to_tensor(ptr: int, nbytes: int, dtype=torch.uint8, device="cuda") -> torch.Tensor:
    """Copy `nbytes` at device pointer `ptr` into a new device tensor (hipMemcpy D2D)."""
    global _hip
    if _hip is None:
        # same SONAME as the runtime torch loaded, so this binds to that instance
        _hip = ctypes.CDLL("libamdhip64.so.7")
        _hip.hipMemcpy.argtypes = [_P, _P, _SZ, _I]
        _hip.hipMemcpy.restype = _I
    out = torch.empty(nbytes, dtype=torch.uint8, device=device)
    if nbytes:
        rc = _hip.hipMemcpy(out.data_ptr(), ptr, nbytes, 3)  # hipMemcpyDeviceToDevice
        if rc != 0:
            raise GptossError(GPTOSS_ERR_HIP, f"hipMemcpy failed ({rc})")
    return out.view(dtype)


# ---------------------------------------------------------------------------
# stage entry points
# ---------------------------------------------------------------------------
def route_scratch(T: int, E: int, top_k: int, device="cuda") -> torch.Tensor:
    """Zero-filled scratch for route() (the call leaves its counters zero)."""
    return torch.zeros(_lib.gptoss_moe_route_scratch_bytes(T, E, top_k), dtype=torch.uint8, device=device)


def route(x, router_w, router_b, top_k: int, logits_fp32: bool = False, stream=None, out=None, scratch=None):
    """Router GEMV + top-k softmax (gptoss_moe_route): (logits, idx, weights).
    out: preallocated (logits, idx, weights); scratch: from route_scratch()."""
    T, H = x.shape
    E = router_w.shape[0]
    dev = x.device
    if out is None:
        logits = torch.empty((T, E), dtype=torch.float32 if logits_fp32 else torch.bfloat16, device=dev)
        idx = torch.empty((T, top_k), dtype=torch.int32, device=dev)
        w = torch.empty((T, top_k), dtype=torch.float32, device=dev)
    else:
        logits, idx, w = out
    if scratch is None:
        scratch = route_scratch(T, E, top_k, dev)
    check(_lib.gptoss_moe_route(_ptr(x), _ptr(router_w), _ptr(router_b), T, E, H, top_k, 1 if logits_fp32 else 0,
                                _ptr(logits), _ptr(idx), _ptr(w), _ptr(scratch), _stream(stream)))
    return logits, idx, w


def topk_softmax(logits, top_k: int, tokens_per_expert=None, stream=None):
    T, E = logits.shape
    idx = torch.empty((T, top_k), dtype=torch.int32, device=logits.device)
    w = torch.empty((T, top_k), dtype=torch.float32, device=logits.device)
    check(_lib.gptoss_topk_softmax_forward(_ptr(logits), 1 if logits.dtype == torch.float32 else 0, _ptr(idx),
                                           _ptr(w), _ptr(tokens_per_expert), T, E, top_k, _stream(stream)))
    return idx, w


def permute_plan(idx, num_experts: int, stream=None):
    T, k = idx.shape
    dev = idx.device
    S = T * k
    counts = torch.empty(num_experts, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    gmap = torch.empty(S, dtype=torch.int32, device=dev)
    ptok = torch.full((S,), -1, dtype=torch.int32, device=dev)
    active = torch.full((num_experts,), -1, dtype=torch.int32, device=dev)
    n_active = torch.empty(1, dtype=torch.int32, device=dev)
    check(_lib.gptoss_moe_permute_plan(_ptr(idx), T, k, num_experts, _ptr(counts), _ptr(offsets), _ptr(gmap),
                                       _ptr(ptok), _ptr(active), _ptr(n_active), _stream(stream)))
    return dict(counts=counts, offsets=offsets, gather_map=gmap, perm_token=ptok, active=active, n_active=n_active)


def scatter_tokens(x, gather_map, top_k: int, stream=None):
    T, H = x.shape
    out = torch.zeros((T * top_k, H), dtype=x.dtype, device=x.device)
    check(_lib.gptoss_moe_scatter_tokens(_ptr(x), _ptr(gather_map), _ptr(out), T, H, top_k, _stream(stream)))
    return out


def mxfp4_gemv(x, tiled_nib, tiled_sc, bias, N: int, K: int, stream=None):
    M = x.shape[0]
    y = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    check(_lib.gptoss_mxfp4_gemv_forward(_ptr(x), M, _ptr(tiled_nib), _ptr(tiled_sc), _ptr(bias), _ptr(y), N, K,
                                         _stream(stream)))
    return y


def swiglu(gate_up, alpha: float = 1.702, limit: float = 7.0, stream=None):
    T, N2 = gate_up.shape
    out = torch.empty((T, N2 // 2), dtype=gate_up.dtype, device=gate_up.device)
    check(_lib.gptoss_swiglu_forward(_ptr(gate_up), _ptr(out), T, N2 // 2, alpha, limit, _stream(stream)))
    return out


def fused_residual_rmsnorm(residual, delta, weight, eps: float = 1e-5, normed=None, sum_out=None, stream=None):
    """fused_residual_rmsnorm_forward: returns (normed, sum_out)."""
    T, H = residual.shape
    if normed is None:
        normed = torch.empty_like(residual)
    if sum_out is None:
        sum_out = torch.empty_like(residual)
    check(_lib.gptoss_fused_residual_rmsnorm_forward(_ptr(residual), _ptr(delta), _ptr(weight), _ptr(normed),
                                                     _ptr(sum_out), T, H, eps, _stream(stream)))
    return normed, sum_out


def combine(expert_out, gather_map, weights, residual, T: int, H: int, top_k: int, stream=None):
    out = torch.empty((T, H), dtype=torch.bfloat16, device=expert_out.device)
    check(_lib.gptoss_moe_combine_forward(_ptr(out), _ptr(expert_out), _ptr(gather_map), _ptr(weights),
                                          _ptr(residual), T, H, top_k, _stream(stream)))
    return out


def dequant(tiled_nib, tiled_sc, N: int, K: int, stream=None):
    out = torch.empty((N, K), dtype=torch.bfloat16, device=tiled_nib.device)
    check(_lib.gptoss_mxfp4_dequant(_ptr(tiled_nib), _ptr(tiled_sc), N, K, _ptr(out), _stream(stream)))
    return out


def grouped_mxfp4_gemm(x, offsets, tiled_nib, tiled_sc, N: int, K: int, rows: int, bias=None, row_index=None,
                       swiglu: bool = False, alpha: float = 1.702, limit: float = 7.0, gate_up=None, out=None,
                       stream=None):
    """Grouped expert product on the matrix cores: rows p of expert e (offsets,
    int32 [E+1] on the device) times W_e (expert-major tiled buffers); x rows
    gathered through row_index when given.  swiglu: out is [rows][N/2]."""
    E = offsets.numel() - 1
    if out is None:
        out = torch.empty((rows, N // 2 if swiglu else N), dtype=torch.bfloat16, device=x.device)
    check(_lib.gptoss_moe_grouped_mxfp4_gemm(_ptr(x), _ptr(row_index), _ptr(offsets), E, rows, _ptr(tiled_nib),
                                             _ptr(tiled_sc), _ptr(bias), N, K, 1 if swiglu else 0, alpha, limit,
                                             _ptr(out), _ptr(gate_up), _stream(stream)))
    return out


# ---------------------------------------------------------------------------
# attention over a paged key-value cache
# ---------------------------------------------------------------------------
GPTOSS_KV_BF16 = 0
GPTOSS_KV_E4M3 = 1


def default_rope_config() -> RopeConfig:
    """GPT-OSS's rotary positions (config.h:29-36)."""
    cfg = RopeConfig()
    check(_lib.gptoss_rope_config_default(ctypes.byref(cfg)))
    return cfg


def rope_table(cfg: RopeConfig | None = None, device="cuda", stream=None) -> torch.Tensor:
    """fp32 [max_positions][2][rotary_dim / 2]: the cosines of each position, then its sines."""
    cfg = cfg or default_rope_config()
    if cfg.rotary_dim < 2 or cfg.max_positions < 1:
        _bad(f"rotary_dim={cfg.rotary_dim} and max_positions={cfg.max_positions} must be positive")
    table = _empty((cfg.max_positions, 2, cfg.rotary_dim // 2), torch.float32, torch.device(device), stream)
    _needs_gpu(table.device)
    _launch(table.device, stream, _lib.gptoss_rope_table, ctypes.byref(cfg), table.data_ptr())
    return table


class _on:
    """The device of index `to` as the current one within the block."""

    def __init__(self, to: int):
        self._to = to

    def __enter__(self):
        self._was = torch.cuda.current_device()
        torch.cuda.set_device(self._to)

    def __exit__(self, *exc):
        torch.cuda.set_device(self._was)


def _launch(device, stream, fn, *args) -> None:
    """Calls fn on `stream` (None: the current one) of `device`."""
    index = device.index
    if stream is None:
        handle = torch._C._cuda_getCurrentRawStream(index)
    else:
        handle = stream if isinstance(stream, int) else stream.cuda_stream
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, handle)
    else:
        with _on(index):
            rc = fn(*args, handle)
    if rc:
        check(rc)


def _on_device(name: str, t, device, dtype=None, dim: int | None = None) -> None:
    if not isinstance(t, torch.Tensor):
        _bad(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if dtype is not None and t.dtype is not dtype:
        _bad(f"{name} has dtype {t.dtype}, expected {dtype}")
    if dim is not None and t.dim() != dim:
        _bad(f"{name} must be {dim}-D, got shape {tuple(t.shape)}")
    if t.device != device:
        _bad(f"{name} is on {t.device}, expected {device}")


def _row_tensor(name: str, t, device, cols: int) -> int:
    """bf16 [rows, cols] on `device`, rows any distance apart: the distance."""
    if not (isinstance(t, torch.Tensor) and t.dtype is torch.bfloat16 and t.dim() == 2 and t.device == device):
        _on_device(name, t, device, torch.bfloat16, 2)
    rows, width = t.shape
    step, one = t.stride()
    if width != cols:
        _bad(f"{name} has shape {tuple(t.shape)}, expected [rows, {cols}]")
    if rows < 2:
        step = (cols + 7) // 8 * 8  # torch gives a single row any stride
    if one != 1 or step < cols:
        _bad(f"{name} must have contiguous rows, strides are {t.stride()}")
    return step


def _vector(name: str, t, device, n: int, dtype) -> None:
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.dim() == 1 and t.numel() == n and t.is_contiguous() \
            and t.device == device:
        return
    _on_device(name, t, device, dtype, 1)
    if t.shape[0] != n:
        _bad(f"{name} has {t.shape[0]} entries, expected {n}")
    if not t.is_contiguous():
        _bad(f"{name} must be contiguous")


def _needs_gpu(device) -> None:
    if device.type != "cuda":
        _bad(f"the cache is on {device}, a GPU is needed")


def _empty(shape, dtype, device, stream):
    """torch.empty in the memory of `stream` (None: the current one), where the kernels that use it run: torch hands
    a freed block out again in the order of its own stream only."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if isinstance(stream, int):
        stream = torch.cuda.default_stream(device) if stream == 0 else torch.cuda.ExternalStream(stream, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


class KVCache:
    """A paged key-value cache over the caller's tensors (borrowed): k and v of
    [num_blocks, kv_heads, block_size, head_dim], bfloat16 or float8_e4m3fn with
    the last dim contiguous and the same strides, so a permuted view covers
    token-major pages and k = slab[:, 0], v = slab[:, 1] an interleaved slab.
    8-bit caches stand for code * scale, scales float32 [kv_heads], positive (None: 1).
    Fixed once made: other tensors need another KVCache."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        for name, t in (("k", k), ("v", v)):
            if not isinstance(t, torch.Tensor) or t.dim() != 4:
                _bad(f"{name} must be a 4-D tensor [num_blocks, kv_heads, block_size, head_dim]")
            if t.dtype not in (torch.bfloat16, torch.float8_e4m3fn):
                _bad(f"{name} has dtype {t.dtype}, expected torch.bfloat16 or torch.float8_e4m3fn")
        if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.stride() != v.stride():
            _bad("k and v differ in shape, dtype, device or strides")
        if k.numel() == 0:
            _bad(f"empty cache of shape {tuple(k.shape)}")
        if k.stride(3) != 1:
            _bad("k and v must be contiguous along head_dim")
        blocks, heads, size, dim = k.shape
        # strides of dims of size 1 are never used, and torch gives them any value
        stride = [st if n > 1 else dim for n, st in zip(k.shape[:3], k.stride()[:3])]
        # slots must not share memory: each stride covers what lies within it
        reach = dim
        for n, st in sorted((m for m in zip(k.shape[:3], stride) if m[0] > 1), key=lambda m: m[1]):
            if st < reach:
                _bad(f"k and v overlap themselves: strides {k.stride()} of shape {tuple(k.shape)}")
            reach = st * (n - 1) + reach
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t is None:
                continue
            if k.dtype == torch.bfloat16:
                _bad(f"{name}: a bfloat16 cache has no scales")
            _vector(name, t, k.device, heads, torch.float32)
        desc = KvCacheDesc(k.data_ptr(), v.data_ptr(), _ptr(k_scale), _ptr(v_scale), stride[0], stride[1], stride[2],
                           GPTOSS_KV_BF16 if k.dtype == torch.bfloat16 else GPTOSS_KV_E4M3, blocks, size, heads, dim)
        vars(self).update(k=k, v=v, k_scale=k_scale, v_scale=v_scale, device=k.device, num_blocks=blocks, kv_heads=heads,
                          block_size=size, head_dim=dim, desc=desc, _desc=ctypes.addressof(desc))

    def __setattr__(self, name, value):
        raise AttributeError(f"KVCache.{name} is fixed: calls use the tensors it was made with")

    def __delattr__(self, name):
        raise AttributeError(f"KVCache.{name} is fixed: calls use the tensors it was made with")


def rope_kv_append(qkv, positions, slots, table, cache: KVCache, num_heads: int, interleaved: bool = False, q_out=None,
                   stream=None):
    """Turns the queries and keys of qkv [T, (num_heads + 2 kv_heads) * head_dim] by their positions (int32
    [T]) and stores keys and values in the cache's slots (int32 [T], page * block_size + place; -1: not stored).
    Rows whose position is outside the table (rope_table()) write nothing.  Returns the queries
    [T, num_heads * head_dim]; q_out may be qkv[:, :num_heads * head_dim]."""
    dev, D = cache.device, cache.head_dim
    stride = _row_tensor("qkv", qkv, dev, (num_heads + 2 * cache.kv_heads) * D)
    T = qkv.shape[0]
    _vector("positions", positions, dev, T, torch.int32)
    _vector("slots", slots, dev, T, torch.int32)
    if not (isinstance(table, torch.Tensor) and table.dtype is torch.float32 and table.dim() == 3 and table.device == dev):
        _on_device("table", table, dev, torch.float32, 3)
    max_positions, two, half = table.shape
    if two != 2 or not table.is_contiguous():
        _bad(f"table must be contiguous [max_positions, 2, rotary_dim / 2], got {tuple(table.shape)}")
    cols = q_stride = num_heads * D
    if q_out is None:
        _needs_gpu(dev)
        q_out = qkv.new_empty((T, cols)) if stream is None else _empty((T, cols), torch.bfloat16, dev, stream)
    else:
        q_stride = _row_tensor("q_out", q_out, dev, cols)
        if q_out.shape[0] != T:
            _bad(f"q_out has {q_out.shape[0]} rows, expected {T}")
        _needs_gpu(dev)
        if T == 1 and q_out.data_ptr() == qkv.data_ptr():
            q_stride = stride
    _launch(dev, stream, _lib.gptoss_rope_kv_append, qkv.data_ptr(), stride, positions.data_ptr(), slots.data_ptr(),
            table.data_ptr(), 2 * half, max_positions, 1 if interleaved else 0, T, num_heads, q_out.data_ptr(), q_stride,
            cache._desc)
    return q_out


def paged_attention_workspace_bytes(num_tokens: int, num_seqs: int, num_heads: int, cache: KVCache) -> int:
    """Bytes of workspace that suffice for any call on up to num_tokens rows of up to num_seqs sequences; a decode call
    has a row for each sequence, so a caller that only decodes gives num_tokens = num_seqs."""
    if max(num_tokens, num_seqs, num_heads) > _INT_MAX:
        _bad(f"num_tokens={num_tokens}, num_seqs={num_seqs} and num_heads={num_heads} must be below 2^31")
    return _lib.gptoss_paged_attention_workspace_bytes(num_tokens, num_seqs, num_heads, cache.kv_heads, cache.head_dim)


_INT_MAX = 2 ** 31 - 1  # of the library's int arguments: ctypes would cut larger numbers

# (rows, 0 for decode; sequences; heads; kv heads; head_dim; tokens of a table; window; first tokens)
_call_bytes = functools.lru_cache(maxsize=4096)(_lib.gptoss_paged_attention_call_bytes)


def _attend(q, offsets, cache, block_tables, seq_lens, scale, window, first_tokens, sinks, out, workspace, stream):
    dev, D = cache.device, cache.head_dim
    if not isinstance(q, torch.Tensor) or q.dim() != 2:
        _bad(f"q must be [rows, num_heads * {D}]")
    rows, cols = q.shape
    H, rest = divmod(cols, D)
    if rest or not H:
        _bad(f"q must be [rows, num_heads * {D}]")
    q_stride = _row_tensor("q", q, dev, cols)
    if not (isinstance(block_tables, torch.Tensor) and block_tables.dtype is torch.int32 and block_tables.dim() == 2
            and block_tables.device == dev):
        _on_device("block_tables", block_tables, dev, torch.int32, 2)
    B, blocks = block_tables.shape
    table_stride, one = block_tables.stride()
    if B < 2:
        table_stride = blocks
    if blocks > 1 and one != 1:
        _bad("block_tables must have contiguous rows")
    _vector("seq_lens", seq_lens, dev, B, torch.int32)
    if (window | first_tokens) >> 31:  # negative, or past _INT_MAX
        _bad(f"window={window} and first_tokens={first_tokens} must not be negative and below 2^31")
    if sinks is not None:
        _vector("sinks", sinks, dev, H, torch.bfloat16)
        sinks = sinks.data_ptr()
    if offsets is None:
        if rows != B:
            _bad(f"q has {rows} rows for {B} sequences")
    else:
        _vector("query_offsets", offsets, dev, B + 1, torch.int32)
    if out is None:
        _needs_gpu(dev)
        out_stride = cols
        out = torch.empty_like(q) if stream is None and q.is_contiguous() else _empty((rows, cols), torch.bfloat16, dev, stream)
    else:
        out_stride = _row_tensor("out", out, dev, cols)
        if out.shape[0] != rows:
            _bad(f"out has {out.shape[0]} rows, expected {rows}")
        _needs_gpu(dev)
    where = None
    if workspace is None:
        size = _call_bytes(rows if offsets is not None else 0, B, H, cache.kv_heads, D, blocks * cache.block_size, window,
                           first_tokens) if rows else 0
        if size:
            workspace = _empty((size,), torch.uint8, dev, stream)
            where = workspace.data_ptr()
    else:
        _on_device("workspace", workspace, dev)
        if not workspace.is_contiguous():
            _bad("workspace must be contiguous")
        size = workspace.numel() * workspace.element_size()
        where = workspace.data_ptr()
    cfg = AttentionConfig(D ** -0.5 if scale is None else scale, window, first_tokens, sinks)
    tail = (cache._desc, block_tables.data_ptr(), table_stride, blocks, seq_lens.data_ptr(), B, H, ctypes.addressof(cfg),
            out.data_ptr(), out_stride, where, size)
    if offsets is None:
        _launch(dev, stream, _lib.gptoss_paged_attention_decode, q.data_ptr(), q_stride, *tail)
    else:
        _launch(dev, stream, _lib.gptoss_paged_attention_prefill, q.data_ptr(), q_stride, offsets.data_ptr(), rows, *tail)
    return out


def paged_attention_decode(q, cache: KVCache, block_tables, seq_lens, scale: float | None = None, window: int = 0,
                           first_tokens: int = 0, sinks=None, out=None, workspace=None, stream=None):
    """Attention of one new token per sequence (already appended): q [B, num_heads * head_dim] over the pages
    block_tables (int32 [B, max_blocks], -1: none) of seq_lens (int32 [B]) tokens.  scale: head_dim ** -0.5 when
    None.  window: 0, or how many of the last tokens are seen, besides the first first_tokens.  sinks: bf16
    [num_heads], a logit that joins the softmax's sum.  workspace: of paged_attention_workspace_bytes(); when None what
    the call needs is allocated, like out."""
    return _attend(q, None, cache, block_tables, seq_lens, scale, window, first_tokens, sinks, out, workspace, stream)


def paged_attention_prefill(q, query_offsets, cache: KVCache, block_tables, seq_lens, scale: float | None = None,
                            window: int = 0, first_tokens: int = 0, sinks=None, out=None, workspace=None, stream=None):
    """Causal attention of prompt chunks: rows query_offsets[b] (int32 [B + 1]) to query_offsets[b + 1] - 1 of
    q are the last tokens of sequence b, already appended.  Rows of no sequence are left as they were in `out`
    (unset when it is allocated here).  Otherwise as paged_attention_decode."""
    if query_offsets is None:
        _bad("query_offsets must be a tensor")
    return _attend(q, query_offsets, cache, block_tables, seq_lens, scale, window, first_tokens, sinks, out, workspace,
                   stream)


# ---------------------------------------------------------------------------
# routing by scores, bias and groups
# ---------------------------------------------------------------------------
GPTOSS_SCORE_SOFTMAX = 0
GPTOSS_SCORE_SIGMOID = 1
_SCORES = {"softmax": GPTOSS_SCORE_SOFTMAX, "sigmoid": GPTOSS_SCORE_SIGMOID}


@functools.lru_cache(maxsize=256)
def _routing_config(score, top_k, num_groups, top_groups, group_rank, renormalize, scale):
    if score not in _SCORES:
        _bad(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    for name, n in (("top_k", top_k), ("num_groups", num_groups), ("top_groups", top_groups), ("group_rank", group_rank)):
        if n >> 31:
            _bad(f"{name}={n} must not be negative and below 2^31")
    cfg = RoutingConfig(_SCORES[score], top_k, num_groups, top_groups, group_rank, 1 if renormalize else 0, scale)
    return cfg, ctypes.addressof(cfg)


def _strided_rows(name: str, t, dtypes, device=None):
    """[rows, cols] of one of dtypes with contiguous rows: rows, cols and the distance between rows in elements."""
    if not isinstance(t, torch.Tensor):
        _bad(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        _bad(f"{name} has dtype {t.dtype}, expected one of {', '.join(str(d) for d in dtypes)}")
    if t.dim() != 2:
        _bad(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    if device is not None and t.device != device:
        _bad(f"{name} is on {t.device}, expected {device}")
    rows, cols = t.shape
    step, one = t.stride()
    if (one != 1 and cols > 1) or (step < cols and rows > 1):
        _bad(f"{name} must have contiguous rows, strides are {t.stride()}")
    if rows > _INT_MAX or cols > _INT_MAX:
        _bad(f"{name} of shape {tuple(t.shape)} is too large")
    return rows, cols, step if rows > 1 else 0  # torch gives a single row any stride


def _gpu(name: str, device) -> None:
    if device.type != "cuda":
        _bad(f"{name} is on {device}, a GPU is needed")


def select_experts(logits, top_k: int, score: str = "softmax", bias=None, num_groups: int = 1, top_groups: int = 1,
                   group_rank: int = 2, renormalize: bool = True, scale: float = 1.0, out=None, stream=None):
    """The top_k experts of each token and their weights, (int32 [T, top_k], float32 [T, top_k]), from the router's
    logits [T, E] (bfloat16 or float32, rows any distance apart).  score: "softmax" over the experts or "sigmoid" of
    each.  bias (float32 [E]): added for the choice, not to the weights.  num_groups > 1: of that many groups of
    neighbours only the top_groups stay whose group_rank (1 or 2) best choices sum highest.  renormalize: weights over
    their sum; scale: a factor of them.  Ties go to the lower index; a logit or bias of -inf switches an expert off (it
    has weight 0 and comes after the others).  out: preallocated (indices, weights)."""
    if isinstance(logits, torch.Tensor) and logits.dim() == 2 and logits.is_contiguous() \
            and (logits.dtype is torch.bfloat16 or logits.dtype is torch.float32):
        T, E = logits.shape
        if T >> 31 or E >> 31:
            _bad(f"logits of shape {tuple(logits.shape)} is too large")
        stride = E
    else:
        T, E, stride = _strided_rows("logits", logits, (torch.bfloat16, torch.float32))
    dev = logits.device
    _, cfg = _routing_config(score, top_k, num_groups, top_groups, group_rank, bool(renormalize), float(scale))
    if bias is not None:
        _vector("bias", bias, dev, E, torch.float32)
        bias = bias.data_ptr()
    if out is None:
        if not logits.is_cuda:
            _gpu("logits", dev)
        if top_k > E:
            _bad(f"top_k={top_k} of {E} experts")
        if stream is None:
            idx = logits.new_empty(T, top_k, dtype=torch.int32)
            w = logits.new_empty(T, top_k, dtype=torch.float32)
        else:
            idx = _empty((T, top_k), torch.int32, dev, stream)
            w = _empty((T, top_k), torch.float32, dev, stream)
    else:
        idx, w = out
        for name, t, dtype in (("indices", idx, torch.int32), ("weights", w, torch.float32)):
            _on_device(name, t, dev, dtype, 2)
            if tuple(t.shape) != (T, top_k) or not t.is_contiguous():
                _bad(f"{name} must be contiguous of shape {(T, top_k)}, got {tuple(t.shape)}")
        _gpu("logits", dev)
    _launch(dev, stream, _lib.gptoss_moe_select_experts, logits.data_ptr(), stride or E,
            1 if logits.dtype is torch.float32 else 0, bias, T, E, cfg, idx.data_ptr(), w.data_ptr())
    return idx, w


# ---------------------------------------------------------------------------
# MXFP4 matrices
# ---------------------------------------------------------------------------
class MXFP4Matrix:
    """A matrix of [rows, K] values, or a stack of them for [experts], in the reference layout: packed uint8
    [.., rows, K / 2] (low nibble = even k) and scales uint8 [.., rows, K / 32], both contiguous.  Value = e2m1 *
    2^(scale - 127).  Fixed once made."""

    __slots__ = ("_held", "_tensors", "_device", "_experts", "_rows", "_K", "_packed", "_scales")

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor):
        for name, t in (("packed", packed), ("scales", scales)):
            if not isinstance(t, torch.Tensor) or t.dtype is not torch.uint8:
                _bad(f"{name} must be a torch.uint8 tensor")
            if not t.is_contiguous():
                _bad(f"{name} must be contiguous")
        if packed.dim() not in (2, 3) or packed.shape[:-1] != scales.shape[:-1] or packed.shape[-1] != 16 * scales.shape[-1]:
            _bad(f"packed must be [.., rows, K / 2] and scales [.., rows, K / 32], got {tuple(packed.shape)} and "
                 f"{tuple(scales.shape)}")
        if packed.shape[-1] == 0:
            _bad("K must be positive")
        if any(n > _INT_MAX for n in (*packed.shape[:-1], 2 * packed.shape[-1])):
            _bad(f"packed of shape {tuple(packed.shape)} is too large")
        if packed.device != scales.device:
            _bad(f"packed is on {packed.device}, scales are on {scales.device}")
        self._held, self._tensors, self._device = None, (packed, scales), packed.device
        self._experts = packed.shape[0] if packed.dim() == 3 else None
        self._rows, self._K = packed.shape[-2], 2 * packed.shape[-1]
        self._packed, self._scales = packed.data_ptr(), scales.data_ptr()

    @classmethod
    def _empty(cls, rows, K, like, device, stream):
        """A new [rows, K]: one allocation, whose tensors are made when they are asked for."""
        n = rows * K
        self = cls.__new__(cls)
        if stream is None and like is not None:
            self._held = like.new_empty(n // 32 * 17, dtype=torch.uint8)
        else:
            self._held = _empty((n // 32 * 17,), torch.uint8, device, stream)
        self._tensors, self._device, self._experts, self._rows, self._K = None, device, None, rows, K
        self._packed = where = self._held.data_ptr()
        self._scales = where + n // 2
        return self

    def _both(self):
        if self._tensors is None:
            n = self._rows * self._K
            self._tensors = (self._held[:n // 2].view(self._rows, self._K // 2),
                             self._held[n // 2:].view(self._rows, self._K // 32))
        return self._tensors

    def _fixed(self, *_):
        raise AttributeError("an MXFP4Matrix is fixed: calls use the tensors it was made with")

    packed = property(lambda self: self._both()[0], _fixed, _fixed)
    scales = property(lambda self: self._both()[1], _fixed, _fixed)
    device = property(lambda self: self._device, _fixed, _fixed)
    experts = property(lambda self: self._experts, _fixed, _fixed, "of a stack; None of a single matrix")
    rows = property(lambda self: self._rows, _fixed, _fixed)
    K = property(lambda self: self._K, _fixed, _fixed)

    @property
    def shape(self):
        return (self._rows, self._K) if self._experts is None else (self._experts, self._rows, self._K)

    def __repr__(self):
        return f"<gptoss_moe.MXFP4Matrix {'x'.join(str(n) for n in self.shape)} on {self.device}>"


def _matrix(name: str, m, device=None) -> "MXFP4Matrix":
    if not isinstance(m, MXFP4Matrix):
        _bad(f"{name} must be an MXFP4Matrix, got {type(m).__name__}")
    if device is not None and m._device != device:
        _bad(f"{name} is on {m._device}, expected {device}")
    return m


def mxfp4_quantize(x, out: MXFP4Matrix | None = None, stream=None) -> MXFP4Matrix:
    """x [rows, K] (bfloat16 or float32, rows a multiple of 16 bytes apart, K a multiple of 32) as MXFP4: each 32 values
    share the power of two 2^(floor(log2(largest)) - 2) and are rounded to the nearest e2m1 value, at most 6 of it.  A
    block with an infinity or NaN becomes NaN.  out: a matrix of that shape to write to."""
    if isinstance(x, torch.Tensor) and x.dim() == 2 and x.is_contiguous() \
            and (x.dtype is torch.bfloat16 or x.dtype is torch.float32):
        rows, K = x.shape
        if rows >> 31 or K >> 31:
            _bad(f"x of shape {tuple(x.shape)} is too large")
        stride = K
    else:
        rows, K, stride = _strided_rows("x", x, (torch.bfloat16, torch.float32))
        stride = stride or K
    dev = x.device
    if K & 31 or not K:
        _bad(f"x has {K} columns, a positive multiple of 32 is needed")
    if out is None:
        if not x.is_cuda:
            _gpu("x", dev)
        out = MXFP4Matrix._empty(rows, K, x, dev, stream)
    else:
        _matrix("out", out, dev)
        if out.shape != (rows, K):
            _bad(f"out has shape {out.shape}, expected {(rows, K)}")
        _gpu("x", dev)
    _launch(dev, stream, _lib.gptoss_mxfp4_quantize, x.data_ptr(), stride, 1 if x.dtype is torch.float32 else 0, rows, K,
            out._packed, out._scales)
    return out


def mxfp4_dequantize(m: MXFP4Matrix, dtype=torch.bfloat16, out=None, stream=None):
    """The values of m, [rows, K] ([experts, rows, K] of a stack), bfloat16 or float32 (exact in both).  out: a 2-D
    tensor [experts * rows, K], rows a multiple of 16 bytes apart."""
    _matrix("m", m)
    dev, K = m._device, m._K
    rows = m._rows if m._experts is None else m._experts * m._rows
    if rows > _INT_MAX:
        _bad(f"a stack of shape {m.shape} is too large")
    if out is None:
        if dtype is not torch.bfloat16 and dtype is not torch.float32:
            _bad(f"dtype must be torch.bfloat16 or torch.float32, got {dtype}")
        if dev.type != "cuda":
            _gpu("m", dev)
        like, stride = m._held, K
        out = like.new_empty(rows, K, dtype=dtype) if stream is None and like is not None \
            else _empty(m.shape, dtype, dev, stream)
    else:
        have, cols, stride = _strided_rows("out", out, (torch.bfloat16, torch.float32), dev)
        if (have, cols) != (rows, K):
            _bad(f"out has shape {tuple(out.shape)}, expected {(rows, K)}")
        stride, dtype = stride or K, out.dtype
        _gpu("m", dev)
    _launch(dev, stream, _lib.gptoss_mxfp4_dequantize, m._packed, m._scales, rows, K, out.data_ptr(), stride,
            1 if dtype is torch.float32 else 0)
    return out


def _product(a, w, rows, offsets, row_index, bias, swiglu, alpha, limit, dtype, quantize, out, stream):
    dev = a._device
    if w._device != dev:
        _bad(f"w is on {w._device}, expected {dev}")
    if a._experts is not None:
        _bad(f"a must be one matrix, got a stack of shape {a.shape}")
    K = a._K
    if K != w._K:
        _bad(f"a has K={K}, w has K={w._K}")
    N, E = w._rows, w._experts
    cols = N // 2 if swiglu else N
    if bias is not None:
        want = (N,) if E is None else (E, N)
        if not (isinstance(bias, torch.Tensor) and bias.dtype is torch.bfloat16 and bias.shape == want
                and bias.is_contiguous() and bias.device == dev):
            _on_device("bias", bias, dev, torch.bfloat16)
            _bad(f"bias must be contiguous of shape {want}, got {tuple(bias.shape)}")
        bias = bias.data_ptr()
    if quantize:
        if cols & 31 or not cols:
            _bad(f"MXFP4 results of {cols} columns, a positive multiple of 32 is needed")
        if out is None:
            if dev.type != "cuda":
                _gpu("a", dev)
            out = MXFP4Matrix._empty(rows, cols, a._held, dev, stream)
        else:
            _matrix("out", out, dev)
            if out.shape != (rows, cols):
                _bad(f"out has shape {out.shape}, expected {(rows, cols)}")
            _gpu("a", dev)
        fp32, where, stride, packed, scales = 0, 0, 0, out._packed, out._scales
    else:
        if out is None:
            if dtype is not torch.bfloat16 and dtype is not torch.float32:
                _bad(f"dtype must be torch.bfloat16 or torch.float32, got {dtype}")
            if dev.type != "cuda":
                _gpu("a", dev)
            like = a._held
            if stream is None and like is not None:
                out = like.new_empty(rows, cols, dtype=dtype)
            else:
                out = _empty((rows, cols), dtype, dev, stream)
            stride = cols
        else:
            have, wide, stride = _strided_rows("out", out, (torch.bfloat16, torch.float32), dev)
            if (have, wide) != (rows, cols):
                _bad(f"out has shape {tuple(out.shape)}, expected {(rows, cols)}")
            stride, dtype = stride or cols, out.dtype
            _gpu("a", dev)
        fp32, where, packed, scales = 1 if dtype is torch.float32 else 0, out.data_ptr(), 0, 0
    try:
        res = _pack_result(1 if swiglu else 0, alpha, limit, fp32, where, stride, packed, scales)
    except (OverflowError, struct.error) as e:
        _bad(f"alpha={alpha!r}, limit={limit!r}: {e}")
    if offsets is None:
        _launch(dev, stream, _lib.gptoss_mxfp4_matmul, a._packed, a._scales, rows, w._packed, w._scales, bias, N, K, res)
    else:
        _launch(dev, stream, _lib.gptoss_moe_grouped_mxfp4_matmul, a._packed, a._scales, a._rows, row_index,
                offsets.data_ptr(), E, rows, w._packed, w._scales, bias, N, K, res)
    return out


def mxfp4_matmul(a: MXFP4Matrix, w: MXFP4Matrix, bias=None, swiglu: bool = False, alpha: float = 1.702, limit: float = 7.0,
                 dtype=torch.bfloat16, quantize: bool = False, out=None, stream=None):
    """a [M, K] times w [N, K] transposed, plus bias (bfloat16 [N]): [M, N], summed in fp32.  swiglu: column pairs (gate,
    up) through the clamped SwiGLU, [M, N / 2].  The result is of dtype (bfloat16 or float32), or with quantize an
    MXFP4Matrix.  out: a tensor (rows any distance apart; its dtype counts) or an MXFP4Matrix."""
    if _matrix("w", w)._experts is not None:
        _bad(f"w is a stack of shape {w.shape}: grouped_mxfp4_matmul takes these")
    return _product(a, w, _matrix("a", a)._rows, None, None, bias, swiglu, alpha, limit, dtype, quantize, out, stream)


def grouped_mxfp4_matmul(a: MXFP4Matrix, w: MXFP4Matrix, offsets, rows: int, row_index=None, bias=None,
                         swiglu: bool = False, alpha: float = 1.702, limit: float = 7.0, dtype=torch.bfloat16,
                         quantize: bool = False, out=None, stream=None):
    """mxfp4_matmul of each expert's rows with its own matrix: w is a stack [E, N, K], bias bfloat16 [E, N], and result
    row p of [rows, N], offsets[e] <= p < offsets[e + 1] (int32 [E + 1], permute_plan's), that of row row_index[p] (int32
    [rows], its perm_token; None: p) of a.  Rows of no expert are left as they were (unset where out is allocated
    here)."""
    if _matrix("w", w)._experts is None:
        _bad(f"w must be a stack [experts, N, K], got shape {w.shape}")
    dev = _matrix("a", a)._device
    if not 0 <= rows <= _INT_MAX:
        _bad(f"rows={rows} must not be negative and below 2^31")
    _vector("offsets", offsets, dev, w._experts + 1, torch.int32)
    if row_index is not None:
        _vector("row_index", row_index, dev, rows, torch.int32)
        row_index = row_index.data_ptr()
    return _product(a, w, rows, offsets, row_index, bias, swiglu, alpha, limit, dtype, quantize, out, stream)
