"""B200-native fused-MoE operator behind the call surface of tingqli/pyhip's quantised MoE path."""
from .fused_moe import (ActivationType, QuantType, PreparedWeights, fused_moe, fused_topk, moe_sorting,  # noqa: F401
                        prepare_weights, release_prepared)

from .linear import int8_status, linear_fp8_128x128, linear_int8, linear_mxfp4, quantize_int8  # noqa: F401,E402
from .norm import fused_post_norm, fused_pre_norm  # noqa: F401,E402
from .router import RouterOutput, fused_router  # noqa: F401,E402

__all__ = ["ActivationType", "QuantType", "PreparedWeights", "fused_moe", "moe_sorting", "prepare_weights",
           "linear_mxfp4", "linear_fp8_128x128", "fused_topk", "release_prepared", "linear_int8", "quantize_int8", "int8_status",
           "fused_pre_norm", "fused_post_norm", "fused_router", "RouterOutput"]
