from .attention import attn_varlen, paged_decode_attn, sparse_attn_varlen
from .fp8 import (Fp8Rows, dequantize_fp8, fp8_linear, fp8_linear_multi, pack_fp8, quantize_fp8,
                  quantize_rows_fp8, rms_norm_fp8, silu_mul_fp8)
from .int4 import dequantize_int4, int4_linear, int4_linear_multi, pack_int4, quantize_int4
from .kv_fp8 import paged_decode_attn_fp8, paged_kv_append_fp8, paged_kv_build_fp8
from .logprobs import TokenLogprobs, TokenLogprobsFn, token_logprobs
from .selective_mha import (PagedSelectiveAttnCache, PagedSelectiveAttnCacheFP8, ScoreStdFn, cross_attention_train,
                           gated_attention_train, selective_mha_prefill)
from .ssd_scan import SSDScanFn
from .ssm_io import SSDScanGatedFn, SSMConvFn, SSMGateFn, build_conv_ctx, ssm_conv_step
from .ssu import SSUFn

__all__ = ["SSDScanFn", "SSUFn", "sparse_attn_varlen", "paged_decode_attn", "SSMConvFn",
           "SSMGateFn", "SSDScanGatedFn", "build_conv_ctx", "ssm_conv_step",
           "selective_mha_prefill", "PagedSelectiveAttnCache", "attn_varlen", "ScoreStdFn",
           "gated_attention_train", "cross_attention_train", "paged_decode_attn_fp8",
           "paged_kv_append_fp8", "paged_kv_build_fp8", "int4_linear", "int4_linear_multi",
           "pack_int4", "quantize_int4", "dequantize_int4", "token_logprobs", "TokenLogprobs",
           "TokenLogprobsFn", "PagedSelectiveAttnCacheFP8", "Fp8Rows", "fp8_linear", "fp8_linear_multi",
           "pack_fp8", "quantize_fp8", "dequantize_fp8", "quantize_rows_fp8", "rms_norm_fp8",
           "silu_mul_fp8"]
