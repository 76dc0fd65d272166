from .fused import (fused_gelu_mlp, gate_residual, fused_qkv_norm_rottary, layernorm_modulate, linearattn_vk_mul_q, litela_attention,
                    qk_norm_rope, qkv_proj_norm_rope)
from .attention import attention, attention_fp16, cross_attention
from .gemm import svdq_gemm_w4a4_cuda
from .quantize import svdq_quantize_w4a4_act_fuse_lora_cuda, svdq_quantize_w4a4_wgt
from .w8a8 import dequantize_w8a8, gemm_w8a8, quantize_w8a8, rms_norm_quantize_w8a8

__all__ = ["svdq_quantize_w4a4_act_fuse_lora_cuda", "svdq_quantize_w4a4_wgt", "svdq_gemm_w4a4_cuda", "fused_gelu_mlp", "fused_qkv_norm_rottary",
           "qk_norm_rope", "qkv_proj_norm_rope", "layernorm_modulate", "gate_residual", "litela_attention", "linearattn_vk_mul_q", "attention", "attention_fp16",
           "cross_attention", "quantize_w8a8", "dequantize_w8a8", "rms_norm_quantize_w8a8", "gemm_w8a8"]
