"""GPU operators (hand-written sm_100a kernels behind a C ABI) and their PyTorch references."""

from . import reference
from .kernels import (argmax, decode_advance, embed, fp8_gemm, paged_attn_decode, quant_rows, rmsnorm_quant,
                      rope_kv_write, silu_mul_quant)
from .kernels import attn_prefill
from .kernels import ACT_NORM, ACT_PLAIN, ACT_SWIGLU, act_gemv_ok, act_gemv_pays, fp8_gemv_act
from .batch import BatchPlan, plan_batch
from .logits import MAX_BIASES, count_tokens, process_logits
from .shared_attn import paged_attn_decode_shared
from .lib import Workspace, available, count_launches, launch_count

__all__ = ["reference", "argmax", "decode_advance", "embed", "fp8_gemm", "paged_attn_decode", "quant_rows",
           "rmsnorm_quant", "rope_kv_write", "silu_mul_quant", "Workspace", "available", "attn_prefill", "count_launches", "launch_count",
           "BatchPlan", "MAX_BIASES", "plan_batch", "count_tokens", "process_logits", "paged_attn_decode_shared"]
