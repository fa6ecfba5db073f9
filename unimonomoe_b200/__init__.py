"""B200-native (sm_100a) single-launch FP8 MoE prefill layer behind the reference's
loader / C-ABI surface. See loader.py for the host API and csrc/ for the kernel; attention.py has the
attention half of the layer over a paged cache held in 4 bits, linear.py the block-FP8 products outside of the MoE launch."""
from .attention import (BatchPlan, KV4Cache, kv4_append, kv4_attention, kv4_read, plan_batch,  # noqa: F401
                        qk_norm_rope)
from .linear import (ExpertPlan, combine_experts, fp8_expert_linear, fp8_linear, fp8_quantize, moe_experts,  # noqa: F401
                     plan_experts)
from .loader import (MOE_MONOKERNEL_PREFILL_MAX_TOKENS, MonoKernel, moe_monokernel_prefill,  # noqa: F401
                     moe_monokernel_prefill_out, monokernel_validate, prefill_monokernel_geometry,
                     prefill_monokernel_tp_caps, prefill_monokernel_tp_pad_words, variant_path)
