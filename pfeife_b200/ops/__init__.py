"""Differentiable ops on the sm_100a kernels (see functional.py) and raw kernel wrappers
(kernels.py)."""
from .functional import (  # noqa: F401
    ParamSlot, PolicyLoss, PreferenceLoss, RopeScaling, attention, conv2d, group_norm, upsample_nearest2x, attention_qkv, compute_dtype, cross_entropy, embedding, geglu, gelu, layer_norm, linear, mlp,
    gated_mlp, linear_cross_entropy, mse_loss, policy_loss, preference_loss, qk_norm_rope, qk_norm_rope_qkv, register_param, rms_norm, rope, rope_qkv, rope_qkv_in_one, rope_tables, scaled_embedding, silu, swiglu, unregister_params,
)
