// The router's choice for the routed block: from each token's logits the
// n_used largest experts and their softmax weights, in the layout that the
// block's entry points take (ids int32, w fp32, [n_tokens][n_used]).
//
//   p_e = exp(x_e - m) / sum_j exp(x_j - m),  m = max_j x_j
//   ids = the n_used largest x, ties to the lower index, in descending order
//   w   = scale * p_ids, divided by their own sum when renorm is set (the
//         denominator over all experts cancels, so only the chosen are summed)
//
// The choice compares logits, not probabilities: exp would round neighbours
// together. One warp holds a token's logits in registers as order-preserving
// 32-bit keys; n_used times the warp takes the largest key (redux.sync) and,
// among the lanes that hold it, the lowest expert.
#include <cuda_bf16.h>

#include "sb_act.cuh"
#include "sb_kernels.h"

namespace {

constexpr int kWarps = 4;
constexpr int kMaxExperts = 2048;
constexpr int kMaxUsed = 32;

struct RouteParams {
    const uint8_t* x;
    size_t row_stride;
    int n_tokens, n_experts, n_used, renorm;
    float scale;
    int32_t* ids;
    float* w;
};

// Larger float <=> larger key; 0 is free for "taken", NaN ranks below -inf.
__device__ inline uint32_t order_key(float f) {
    const uint32_t u = __float_as_uint(f);
    if (f != f) return 1;
    if (f == 0.f) return 0x80000000u;   // -0 ties with +0
    return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ inline float key_value(uint32_t k) {
    return k == 1 ? __int_as_float(0x7fc00000) : __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

// NV: logits per lane (n_experts <= 32 * NV); expert e is lane e % 32's
template <class Act, int NV>
__global__ void __launch_bounds__(kWarps * 32) k_route(RouteParams p) {
    const int lane = threadIdx.x & 31, t = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (t >= p.n_tokens) return;
    const Act* row = (const Act*)(p.x + (size_t)t * p.row_stride);
    uint32_t key[NV];
    uint32_t top = 0;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = lane + 32 * i;
        key[i] = e < p.n_experts ? order_key(sb_to_float(row[e])) : 0;
        nan |= key[i] == 1;
        top = max(top, key[i]);
    }
    nan = __any_sync(~0u, nan);
    const float m = key_value(__reduce_max_sync(~0u, top));
    float all = 0.f;
    if (!p.renorm) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (key[i]) all += __expf(key_value(key[i]) - m);
#pragma unroll
        for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(~0u, all, o);
    }
    float mine = 0.f, chosen = 0.f;   // lane j keeps choice j
    int my_id = 0;
    for (int j = 0; j < p.n_used; ++j) {
        uint32_t best = 0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (key[i] > best) {
                best = key[i];
                at = i;
            }
        const uint32_t k = __reduce_max_sync(~0u, best);
        const int e = __reduce_min_sync(~0u, best == k ? lane + 32 * at : 0x7fffffff);
        if (lane == (e & 31)) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (i == (e >> 5)) key[i] = 0;
        }
        const float v = expf(key_value(k) - m);
        chosen += v;
        if (lane == j) {
            mine = v;
            my_id = e;
        }
    }
    // a row with a NaN has NaN weights (its ids stay in range); a row whose
    // logits are all -inf chooses nothing: zero weights
    float w = p.scale * (mine / (p.renorm ? chosen : all));
    if (m == -INFINITY) w = 0.f;
    if (nan) w = __int_as_float(0x7fc00000);
    if (lane < p.n_used) {
        p.ids[(size_t)t * p.n_used + lane] = my_id;
        p.w[(size_t)t * p.n_used + lane] = w;
    }
}

template <class Act>
void launch_route(const RouteParams& p, cudaStream_t st) {
    const int grid = (p.n_tokens + kWarps - 1) / kWarps;
    if (p.n_experts <= 128)
        k_route<Act, 4><<<grid, kWarps * 32, 0, st>>>(p);
    else if (p.n_experts <= 512)
        k_route<Act, 16><<<grid, kWarps * 32, 0, st>>>(p);
    else
        k_route<Act, 64><<<grid, kWarps * 32, 0, st>>>(p);
}

}  // namespace

SABAH_API int sabah_route_topk(const void* d_logits, size_t row_stride, int act_type, int n_tokens, int n_experts,
                               int n_used, int renorm, float scale, int32_t* d_ids, float* d_w, void* stream) {
    int* err;
    cudaStream_t st;
    if (!sb_op_begin(stream, &st, &err)) return -1;
    const int eb = sb_act_bytes(act_type);
    if (n_tokens < 0 || n_experts <= 0 || n_experts > kMaxExperts || n_used <= 0 || n_used > kMaxUsed ||
        n_used > n_experts || !eb) {
        sb_set_error("invalid route geometry (tokens %d, experts %d of at most %d, used %d of at most %d, type %d)",
                     n_tokens, n_experts, kMaxExperts, n_used, kMaxUsed, act_type);
        return -1;
    }
    if (n_tokens == 0) return 0;
    if (!d_logits || !d_ids || !d_w || row_stride % eb || (uintptr_t)d_logits % eb ||
        ((uintptr_t)d_ids | (uintptr_t)d_w) % 4) {
        sb_set_error("invalid route arguments (a null or misaligned pointer, or a row stride of %zu bytes)", row_stride);
        return -1;
    }
    const RouteParams p{(const uint8_t*)d_logits, row_stride, n_tokens, n_experts, n_used, renorm, scale, d_ids, d_w};
    const int slot = sb_timing_begin("route_topk", st);
    if (act_type == SB_F32)
        launch_route<float>(p, st);
    else if (act_type == SB_F16)
        launch_route<__half>(p, st);
    else
        launch_route<__nv_bfloat16>(p, st);
    sb_timing_end(slot, st);
    return sb_cuda_ok(cudaGetLastError(), "route launch") ? 0 : -1;
}
