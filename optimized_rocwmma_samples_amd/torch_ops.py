"""The path as PyTorch operators: `torch.library` custom ops under the
namespace `w8a8`, each calling the same C ABI (libw8a8.so, through this
package's ctypes layer) on torch's current stream, with a fake kernel for
shape and dtype inference, so torch.compile and torch.export trace through
them without a graph break.

    import optimized_rocwmma_samples_amd.torch_ops  # registers the ops
    q, r = torch.ops.w8a8.smoothquant(x, s, 127.0)
    c = torch.ops.w8a8.gemm(q, w, r, sb)
    c, q, r = torch.ops.w8a8.fused_sq_gemm(x, s, w, sb)
    x_out, q, r = torch.ops.w8a8.add_rmsnorm_smoothquant(x, residual, gamma, s, 1e-5, 127.0)
    pw = w8a8.pack_weights(w)                        # once; the op takes pw.data and pw.n
    c, q, r = torch.ops.w8a8.fused_sq_gemm_packed(x, s, pw.data, pw.n, sb)
    out = torch.ops.w8a8.moe_ffn(x, logits, s, w_gu, sb_gu, w_d, sb_d, 2)
    out = torch.ops.w8a8.moe_ffn_decode(x, logits, s, w_gu, sb_gu, w_d, sb_d, 2)  # <= 16 tokens
    out = torch.ops.w8a8.attention(q, k, v, seq_starts)
    torch.ops.w8a8.kv4_store(k, v, slots, kc, vc, ks, vs)   # a KV4Cache's four tensors
    out = torch.ops.w8a8.attention_kv4(q, kc, vc, ks, vs, block_table, seq_lens)

The ops are functional (every output is a new tensor), as torch.library
custom ops must be, but for kv4_store, which writes the cache it is given; the
package functions keep the in-place and preallocated-output forms.  They run only on device tensors: a CPU tensor
raises, as everywhere in the package (there is no CPU path).

Reference kernels: smoothquant <- kernel_smoothquant
(rocwmma_smoothquant.cpp:58-122); gemm <- gemm_quant_tensor_scale
(rocwmma_gemm_quantized.cpp:127-195) with per-token x per-channel scales;
gemm_packed / fused_sq_gemm_packed <- the pre-shuffled weight format of
rocwmma_flatmm.cpp:12-16 and the decode role of rocwmma_gemm_splitk.cpp:
104-201; add_rmsnorm_smoothquant <- kernel_add_rmsnorm2d_fwd
(rocwmma_rmsnorm2d.cpp:127-186) feeding the quantizer; moe_ffn <- the
route / sort / quantize / expert GEMM / combine chain of
rocwmma_fused_moe.cpp:96-211.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import KV4Cache, PackedWeights
from . import add_rmsnorm_smoothquant as _add_rmsnorm_smoothquant
from . import attention as _attention
from . import attention_kv4 as _attention_kv4
from . import fused_sq_gemm as _fused_sq_gemm
from . import fused_sq_gemm_packed as _fused_sq_gemm_packed
from . import gemm as _gemm
from . import gemm_packed as _gemm_packed
from . import kv4_load as _kv4_load
from . import kv4_store as _kv4_store
from . import moe_ffn as _moe_ffn
from . import moe_ffn_decode as _moe_ffn_decode
from . import smoothquant as _smoothquant

Tensor = torch.Tensor


@torch.library.custom_op("w8a8::smoothquant", mutates_args=())
def smoothquant(x: Tensor, smooth_scale: Tensor, quant_max: float = 127.0) -> Tuple[Tensor, Tensor]:
    """(q int8 [M, N], row_scale fp32 [M]) of fp16 x [M, N]."""
    return _smoothquant(x, smooth_scale, quant_max)


@smoothquant.register_fake
def _(x, smooth_scale, quant_max=127.0):
    m, n = x.shape
    return x.new_empty((m, n), dtype=torch.int8), x.new_empty((m,), dtype=torch.float32)


@torch.library.custom_op("w8a8::gemm", mutates_args=())
def gemm(a: Tensor, b: Tensor, scale_a: Optional[Tensor] = None,
         scale_b: Optional[Tensor] = None, tensor_scale_a: float = 1.0,
         tensor_scale_b: float = 1.0) -> Tensor:
    """fp16 C [M, N] = dequant(a [M, K] . b [N, K]^T): per-row / per-column
    scales where given, else the tensor scales."""
    return _gemm(a, b, scale_a, scale_b, tensor_scale_a, tensor_scale_b)


@gemm.register_fake
def _(a, b, scale_a=None, scale_b=None, tensor_scale_a=1.0, tensor_scale_b=1.0):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=torch.float16)


@torch.library.custom_op("w8a8::gemm_i32", mutates_args=())
def gemm_i32(a: Tensor, b: Tensor) -> Tensor:
    """int32 accumulators a [M, K] . b [N, K]^T."""
    return _gemm(a, b, out_dtype=torch.int32)


@gemm_i32.register_fake
def _(a, b):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=torch.int32)


@torch.library.custom_op("w8a8::fused_sq_gemm", mutates_args=())
def fused_sq_gemm(x: Tensor, smooth_scale: Tensor, w: Tensor,
                  scale_w: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    """SmoothQuant of x [M, K] then C = dequant(q . w^T): (c fp16 [M, N], q, row_scale)."""
    return _fused_sq_gemm(x, smooth_scale, w, scale_w)


@fused_sq_gemm.register_fake
def _(x, smooth_scale, w, scale_w):
    m, k = x.shape
    return (x.new_empty((m, w.shape[0]), dtype=torch.float16),
            x.new_empty((m, k), dtype=torch.int8), x.new_empty((m,), dtype=torch.float32))


@torch.library.custom_op("w8a8::add_rmsnorm_smoothquant", mutates_args=())
def add_rmsnorm_smoothquant(x: Tensor, residual: Tensor, gamma: Tensor, smooth_scale: Tensor,
                            eps: float = 1e-5,
                            quant_max: float = 127.0) -> Tuple[Tensor, Tensor, Tensor]:
    """(x_out = half(x + residual), q int8, row_scale) of RMSNorm(x_out) fed
    to the quantizer; x and residual are left unchanged."""
    x_out, _, q, r = _add_rmsnorm_smoothquant(x, gamma, smooth_scale, residual=residual, eps=eps,
                                              quant_max=quant_max)
    return x_out, q, r


@add_rmsnorm_smoothquant.register_fake
def _(x, residual, gamma, smooth_scale, eps=1e-5, quant_max=127.0):
    m, n = x.shape
    return (torch.empty_like(x), x.new_empty((m, n), dtype=torch.int8),
            x.new_empty((m,), dtype=torch.float32))


@torch.library.custom_op("w8a8::gemm_packed", mutates_args=())
def gemm_packed(a: Tensor, packed: Tensor, n: int, scale_a: Optional[Tensor] = None,
                scale_b: Optional[Tensor] = None) -> Tensor:
    """fp16 C [M, n] = dequant(a [M, K] . W^T) with W [n, K] given packed
    (`pack_weights(w).data`); split-K workspace allocated as the shape needs."""
    return _gemm_packed(a, PackedWeights(packed, n, a.shape[1]), scale_a, scale_b)


@gemm_packed.register_fake
def _(a, packed, n, scale_a=None, scale_b=None):
    return a.new_empty((a.shape[0], n), dtype=torch.float16)


@torch.library.custom_op("w8a8::fused_sq_gemm_packed", mutates_args=())
def fused_sq_gemm_packed(x: Tensor, smooth_scale: Tensor, packed: Tensor, n: int,
                         scale_w: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    """SmoothQuant of x [M, K] then C = dequant(q . W^T), W [n, K] packed:
    (c fp16 [M, n], q, row_scale)."""
    return _fused_sq_gemm_packed(x, smooth_scale, PackedWeights(packed, n, x.shape[1]), scale_w)


@fused_sq_gemm_packed.register_fake
def _(x, smooth_scale, packed, n, scale_w):
    m, k = x.shape
    return (x.new_empty((m, n), dtype=torch.float16), x.new_empty((m, k), dtype=torch.int8),
            x.new_empty((m,), dtype=torch.float32))


@torch.library.custom_op("w8a8::moe_ffn", mutates_args=())
def moe_ffn(x: Tensor, logits: Tensor, smooth_scale: Tensor, w_gate_up: Tensor,
            sb_gate_up: Tensor, w_down: Tensor, sb_down: Tensor, topk: int,
            smooth_scale_down: Optional[Tensor] = None, unit_size: int = 32,
            gate_up_interleaved: bool = False) -> Tensor:
    """The expert FFN of x [T, H] (fp16 out [T, H]): routing, sort, quantize,
    gate_up, SiLU(gate)*up requant, down, combine.  gate_up_interleaved: the
    gate_up weights and scales come from moe_interleave_gate_up, and the
    gate_up GEMM runs with the SiLU epilogue."""
    if gate_up_interleaved:
        out, _ = _moe_ffn(x, logits, smooth_scale, None, None, w_down, sb_down, topk,
                          smooth_scale_down, unit_size, (w_gate_up, sb_gate_up))
    else:
        out, _ = _moe_ffn(x, logits, smooth_scale, w_gate_up, sb_gate_up, w_down, sb_down, topk,
                          smooth_scale_down, unit_size)
    return out


@moe_ffn.register_fake
def _(x, logits, smooth_scale, w_gate_up, sb_gate_up, w_down, sb_down, topk,
      smooth_scale_down=None, unit_size=32, gate_up_interleaved=False):
    return torch.empty_like(x, dtype=torch.float16)


@torch.library.custom_op("w8a8::moe_ffn_decode", mutates_args=())
def moe_ffn_decode(x: Tensor, logits: Tensor, smooth_scale: Tensor, w_gate_up: Tensor,
                   sb_gate_up: Tensor, w_down: Tensor, sb_down: Tensor, topk: int,
                   smooth_scale_down: Optional[Tensor] = None,
                   quant_max: float = 127.0) -> Tensor:
    """The expert FFN of at most 16 tokens x [T, H] (fp16 out [T, H]) in three launches."""
    return _moe_ffn_decode(x, logits, smooth_scale, w_gate_up, sb_gate_up, w_down, sb_down, topk,
                           smooth_scale_down, quant_max)


@moe_ffn_decode.register_fake
def _(x, logits, smooth_scale, w_gate_up, sb_gate_up, w_down, sb_down, topk,
      smooth_scale_down=None, quant_max=127.0):
    return x.new_empty(x.shape, dtype=torch.float16)


@torch.library.custom_op("w8a8::attention", mutates_args=())
def attention(q: Tensor, k: Tensor, v: Tensor, seq_starts: Tensor,
              scale: Optional[float] = None) -> Tensor:
    """Causal attention of packed prompts: fp16 [tokens, heads, head_dim]; rows of no
    sequence are undefined."""
    return _attention(q, k, v, seq_starts, scale)


@attention.register_fake
def _(q, k, v, seq_starts, scale=None):
    return q.new_empty(q.shape)


@torch.library.custom_op("w8a8::kv4_store",
                         mutates_args=("k_codes", "v_codes", "k_scales", "v_scales"))
def kv4_store(k: Tensor, v: Tensor, slots: Tensor, k_codes: Tensor, v_codes: Tensor,
              k_scales: Tensor, v_scales: Tensor) -> None:
    """Quantizes k, v [tokens, kv_heads, head_dim] into the slots of a KV4Cache's tensors."""
    _kv4_store(k, v, slots, KV4Cache(k_codes, v_codes, k_scales, v_scales))


@kv4_store.register_fake
def _(k, v, slots, k_codes, v_codes, k_scales, v_scales):
    return None


@torch.library.custom_op("w8a8::kv4_load", mutates_args=())
def kv4_load(slots: Tensor, k_codes: Tensor, v_codes: Tensor, k_scales: Tensor,
             v_scales: Tensor) -> Tuple[Tensor, Tensor]:
    """(k, v) fp16 [n, kv_heads, head_dim] of the slots; undefined for slots outside."""
    return _kv4_load(KV4Cache(k_codes, v_codes, k_scales, v_scales), slots)


@kv4_load.register_fake
def _(slots, k_codes, v_codes, k_scales, v_scales):
    shape = (slots.shape[0], k_codes.shape[1], k_codes.shape[3] * 2)
    return k_scales.new_empty(shape), k_scales.new_empty(shape)


@torch.library.custom_op("w8a8::attention_kv4", mutates_args=())
def attention_kv4(q: Tensor, k_codes: Tensor, v_codes: Tensor, k_scales: Tensor, v_scales: Tensor,
                  block_table: Tensor, seq_lens: Tensor, scale: Optional[float] = None) -> Tensor:
    """Attention of one token per sequence, q [seqs, heads, head_dim], over a KV4Cache's
    tensors; workspace allocated for the table's columns."""
    return _attention_kv4(q, KV4Cache(k_codes, v_codes, k_scales, v_scales), block_table, seq_lens,
                          scale)


@attention_kv4.register_fake
def _(q, k_codes, v_codes, k_scales, v_scales, block_table, seq_lens, scale=None):
    return q.new_empty(q.shape)
