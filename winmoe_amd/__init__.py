"""winmoe_amd -- MI355X-native MoE expert-layer path of WinMoE.

Router softmax/top-K, raw GGUF block dequantisation (Q8_0, Q2_K, Q3_K, Q4_K,
Q5_K, Q6_K) fused into the gate/up/down expert products, SwiGLU and the
routing-weighted combine with the shared expert, as hand-written gfx950 HIP
kernels behind the C-ABI of include/winmoe_hip.h; and the same layer with
fp16 or bf16 weights, forward and backward, out of products that also stand
alone (dense.py).
"""
from ._lib import (BF16, BLOCK_BYTES, BLOCK_ELEMS, F16, F32, Q2_K, Q3_K, Q4_K, Q5_K, Q6_K, Q8_0, QUANT_TYPES,  # noqa: F401
                   TYPE_IDS, TYPE_NAMES, WinMoEError, load)
from .moe import (ExpertPool, MoELayer, SharedExpert, decode_stack, dequant_q4k_block, dequant_q8_0_row, dequantize,  # noqa: F401
                  expert_ffn,
                  matrix_bytes, q8_0_matvec, quant_matvec, quantize, quantize_into, router_logits,
                  router_topk)
from .dense import (FloatMoELayer, act_backward, combine, combine_backward, group_by_expert, grouped_matmul,  # noqa: F401
                    grouped_matmul_backward, linear, linear_backward)

__version__ = "0.1.0"
