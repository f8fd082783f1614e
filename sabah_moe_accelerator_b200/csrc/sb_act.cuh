// Activation and cache element types of the attention-side operators
// (sb_norm_rope.cu, sb_attend.cu, sb_route.cu): ggml's codes for them and the
// conversions to and from fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sb_common.cuh"

#define SABAH_API extern "C" __attribute__((visibility("default")))

enum sb_acttype : int { SB_F32 = 0, SB_F16 = 1, SB_BF16 = 30 };   // ggml.h enum values

inline int sb_act_bytes(int type) {
    return type == SB_F32 ? 4 : type == SB_F16 || type == SB_BF16 ? 2 : 0;
}

__device__ inline float sb_to_float(float v) { return v; }
__device__ inline float sb_to_float(__half v) { return __half2float(v); }
__device__ inline float sb_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ inline T sb_from_float(float v);
template <>
__device__ inline float sb_from_float<float>(float v) { return v; }
template <>
__device__ inline __half sb_from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ inline __nv_bfloat16 sb_from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
