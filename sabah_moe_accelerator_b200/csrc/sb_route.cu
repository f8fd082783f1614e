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
// 32-bit keys, read 16 bytes at a time where rows allow it.
//
// Bound: for many tokens the instructions that a logit costs, else latency, so
// the choice is made without n_used rounds over all logits. The n_used-th
// largest of the 32 lanes' largest keys is a key that at least n_used logits
// reach, and few more do (about 13 of 512 for the 10 largest). Those are
// gathered one per lane, and each lane counts how many beat its own: its rank.
// 16-bit logits are compared two to a register, the lanes' largest are sorted for
// the bound, and (key, expert) of a gathered one fits 32 bits.
// Where more than 32 logits reach the bound (many equal ones), the warp takes
// the largest n_used times instead.
//
// Measured (one B200): 16384 tokens x 512 bf16 logits, the 10 largest: 12.3 us
// (1.4 TB/s, 505 instructions a token, issue slots 69%), 35 us with n_used rounds;
// 131,072 tokens: 76 us (1.8 TB/s; 82 with the gathered ones sorted by the warp and
// every lane looking at all its logits to gather them); one token: 5 us, the launch
// and the call.
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

// Larger float <=> larger key. 0 stands for "taken" and "none"; a NaN is below
// -inf once sink_nan() has seen it (until then it may have any key, 0 too).
__device__ inline uint32_t order_key(float f) {
    const int u = __float_as_int(f + 0.f);   // -0 ties with +0
    return (uint32_t)u ^ ((uint32_t)(u >> 31) | 0x80000000u);
}
__device__ inline float key_value(uint32_t k) {
    return k == 1 ? __int_as_float(0x7fc00000) : __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}
__device__ inline uint32_t sink_nan(uint32_t k) {   // beyond the keys of +-inf lie the NaNs
    return k > 0xff800000u || k < 0x007fffffu ? 1 : k;
}

// NV: logits per lane (n_experts <= 32 * NV), V of them side by side
template <class Act, int NV, int V>
__global__ void __launch_bounds__(kWarps * 32) k_route(const __grid_constant__ RouteParams p) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, t = blockIdx.x * kWarps + wid;
    __shared__ uint2 picked[kWarps][32];
    if (t >= p.n_tokens) return;
    const Act* row = (const Act*)(p.x + (size_t)t * p.row_stride);
    auto expert = [&](int i) { return (i / V * 32 + lane) * V + i % V; };
    uint32_t key[NV];
    float odd = 0.f;   // a NaN once a NaN or an infinity went in
#pragma unroll
    for (int c = 0; c < NV / V; ++c) {
        struct alignas(V * sizeof(Act)) Chunk { Act x[V]; };
        const int e = expert(c * V);
        Chunk u;
        if (e < p.n_experts) u = *(const Chunk*)(row + e);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float x = e < p.n_experts ? sb_to_float(u.x[i]) : 0.f;
            key[c * V + i] = e < p.n_experts ? order_key(x) : 0;
            odd += x * 0.f;
        }
    }
    bool nan = __any_sync(~0u, odd != 0.f);
    if (nan) {   // only then the keys are looked at one by one
        nan = false;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (expert(i) < p.n_experts) key[i] = sink_nan(key[i]);
            nan |= key[i] == 1;
        }
        nan = __any_sync(~0u, nan);
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) top = max(top, key[i]);
    const uint32_t first = __reduce_max_sync(~0u, top);
    const float m = key_value(first);
    // of all, where the weights are over all experts. __expf errs by 2 + 1.2 |x| ulp, and
    // the mean of -x under the weights is at most ln(experts): 11 ulp of the sum at 2048
    // experts (1.3e-6) at worst, 2e-7 measured
    float total = 0.f;
    if (!p.renorm) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (key[i]) total += __expf(key_value(key[i]) - m);
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
    }

    // a key that at least n_used logits reach, and who reaches it
    uint32_t bound = first, left = top;
    for (int lanes = 0;;) {
        lanes += __popc(__ballot_sync(~0u, left == bound));
        if (lanes >= p.n_used) break;
        if (left == bound) left = 0;
        const uint32_t k = __reduce_max_sync(~0u, left);
        if (k == 0) {   // fewer lanes with logits than choices: all of them count
            bound = 1;
            break;
        }
        bound = k;
    }
    int here = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) here += key[i] >= bound;
    int upto = here;   // in the lanes before and this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += x;
    }
    const int n = __shfl_sync(~0u, upto, 31);
    if (n <= 32) {
        uint2* next = &picked[wid][upto - here];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (key[i] >= bound) *next++ = make_uint2(key[i], expert(i));
    }
    uint32_t mine = 0;   // this lane's choice: its key, expert and rank
    int my_id = 0, rank = p.n_used;
    if (n <= 32) {
        __syncwarp();
        if (lane < n) {
            const uint2 u = picked[wid][lane];
            mine = u.x, my_id = u.y, rank = 0;
        }
        for (int j = 0; j < n; ++j) {
            const uint2 u = picked[wid][j];
            rank += u.x > mine || (u.x == mine && (int)u.y < my_id);
        }
    } else {
        for (int j = 0; j < p.n_used; ++j) {
            uint32_t best = 0;
            int at = 0;   // the lowest expert of the lane's largest keys: expert() grows with i
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (key[i] > best) {
                    best = key[i];
                    at = expert(i);
                }
            const uint32_t k = __reduce_max_sync(~0u, best);
            const int e = __reduce_min_sync(~0u, best == k ? at : 0x7fffffff);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (expert(i) == e) key[i] = 0;
            if (lane == j) mine = k, my_id = e, rank = j;
        }
    }
    const bool chosen = mine && rank < p.n_used;
    const float v = chosen ? expf(key_value(mine) - m) : 0.f;
    if (p.renorm) {
        total = v;
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
    }
    // a row with a NaN has NaN weights (its ids stay in range); a row whose
    // logits are all -inf chooses nothing: zero weights
    float w = p.scale * (v / total);
    if (m == -INFINITY) w = 0.f;
    if (nan) w = __int_as_float(0x7fc00000);
    if (chosen) {
        p.ids[(size_t)t * p.n_used + rank] = my_id;
        p.w[(size_t)t * p.n_used + rank] = w;
    }
}

// descending over the lanes
__device__ inline uint32_t sort_lanes(uint32_t v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k / 2; j; j >>= 1) {
            const uint32_t x = __shfl_xor_sync(~0u, v, j);
            v = ((lane & k) == 0) == ((lane & j) == 0) ? max(v, x) : min(v, x);
        }
    return v;
}

// 16-bit logits in rows of whole 16-byte chunks: as above, in 16-bit keys
template <class Act, int NV>
__global__ void __launch_bounds__(kWarps * 32, NV <= 16 ? 40 / kWarps : 1) k_route16(const __grid_constant__ RouteParams p) {
    constexpr bool kF16 = std::is_same<Act, __half>::value;
    using Act2 = typename std::conditional<kF16, __half2, __nv_bfloat162>::type;
    using Mask = typename std::conditional<NV <= 32, uint32_t, unsigned long long>::type;   // a bit per logit
    constexpr uint32_t kInf = kF16 ? 0xfc00 : 0xff80, kNegInf = kF16 ? 0x03ff : 0x007f;   // keys of +-inf
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, t = blockIdx.x * kWarps + wid;
    __shared__ alignas(16) uint32_t picked[kWarps][32];
    __shared__ uint4 kept[kWarps][NV / 8][32];   // the keys, where a lane can take one by number
    if (t >= p.n_tokens) return;
    const uint4* row = (const uint4*)(p.x + (size_t)t * p.row_stride);
    auto expert = [&](int i) { return (i / 8 * 32 + lane) * 8 + i % 8; };
    auto value = [&](uint32_t k) {
        const uint16_t u = k >> 15 ? k & 0x7fff : ~k;
        return k == 1 ? __int_as_float(0x7fc00000) : sb_to_float(*(const Act*)&u);
    };
    uint4 raw[NV / 8];
#pragma unroll
    for (int c = 0; c < NV / 8; ++c)
        raw[c] = expert(8 * c) < p.n_experts ? __ldg(row + c * 32 + lane) : make_uint4(0, 0, 0, 0);
    uint32_t key[NV / 2];   // two each; pairs beyond the experts stay 0
    Act2 odd = Act2(sb_from_float<Act>(0.f), sb_from_float<Act>(0.f));
    const Act2 zero = odd;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV / 2; ++i) {
        const uint32_t u = ((const uint32_t*)raw)[i];
        odd = __hfma2(*(const Act2*)&u, zero, odd);        // a NaN once a NaN or an infinity went in
        const Act2 plus = __hadd2(*(const Act2*)&u, zero);   // -0 ties with +0
        const uint32_t v = *(const uint32_t*)&plus;
        uint32_t negative;   // all ones in the halves that are
        asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(negative) : "r"(v));
        key[i] = expert(2 * i) < p.n_experts ? v ^ (negative | 0x80008000u) : 0;
    }
    bool nan = __any_sync(~0u, *(const uint32_t*)&odd & 0x7fff7fffu);
    if (nan) {   // only then the keys are looked at one by one
        nan = false;
#pragma unroll
        for (int i = 0; i < NV / 2; ++i) {
            if (expert(2 * i) >= p.n_experts) continue;
            uint32_t lo = key[i] & 0xffff, hi = key[i] >> 16;
            if (lo > kInf || lo < kNegInf) lo = 1, nan = true;
            if (hi > kInf || hi < kNegInf) hi = 1, nan = true;
            key[i] = hi << 16 | lo;
        }
        nan = __any_sync(~0u, nan);
    }
#pragma unroll
    for (int i = 0; i < NV / 2; ++i) top = __vmaxu2(top, key[i]);
    const uint32_t sorted = sort_lanes(max(top & 0xffff, top >> 16), lane);
    const uint32_t bound = max(__shfl_sync(~0u, sorted, p.n_used - 1), 1u);   // 1: fewer lanes with logits than choices
    const float m = value(__shfl_sync(~0u, sorted, 0));
    float total = 0.f;   // of all, where the weights are over all experts; __expf as above
    if (!p.renorm) {
#pragma unroll
        for (int i = 0; i < NV / 2; ++i)
            if (key[i]) total += __expf(value(key[i] & 0xffff) - m) + __expf(value(key[i] >> 16) - m);
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
    }
#pragma unroll
    for (int c = 0; c < NV / 8; ++c)
        kept[wid][c][lane] = make_uint4(key[4 * c], key[4 * c + 1], key[4 * c + 2], key[4 * c + 3]);
    // who reaches the bound, as (key, 65535 - expert): larger is earlier
    Mask mask = 0;
#pragma unroll
    for (int i = 0; i < NV / 2; ++i) {
        if ((key[i] & 0xffff) >= bound) mask |= Mask(1) << (2 * i);
        if (key[i] >= bound << 16) mask |= Mask(1) << (2 * i + 1);
    }
    const int here = __popcll(mask);
    int upto = here;   // in the lanes before and this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += x;
    }
    const int n = __shfl_sync(~0u, upto, 31);
    uint32_t mine = 0;
    int rank = lane;
    if (n <= 32) {
        uint32_t* next = &picked[wid][upto - here];
        for (; mask; mask &= mask - 1) {
            const int i = sizeof(Mask) == 4 ? __ffs((int)mask) - 1 : __ffsll((long long)mask) - 1;
            const uint32_t two = ((const uint32_t*)&kept[wid][i / 8][lane])[i % 8 / 2];
            *next++ = (i & 1 ? two & 0xffff0000u : two << 16) | (0xffff - expert(i));
        }
        if (lane >= n) picked[wid][lane] = 0;
        __syncwarp();
        mine = picked[wid][lane];
        rank = mine ? 0 : p.n_used;
        for (int j = 0; j < n; j += 4) {
            const uint4 u = *(const uint4*)&picked[wid][j];
            rank += (u.x > mine) + (u.y > mine) + (u.z > mine) + (u.w > mine);
        }
    } else {
        mask = 0;   // taken
        for (int j = 0; j < p.n_used; ++j) {
            uint32_t best = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const uint32_t k = i & 1 ? key[i / 2] & 0xffff0000u : key[i / 2] << 16;
                if (k && !(mask >> i & 1)) best = max(best, k | (0xffff - expert(i)));
            }
            const uint32_t k = __reduce_max_sync(~0u, best);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (expert(i) == 0xffff - (int)(k & 0xffff)) mask |= Mask(1) << i;
            if (lane == j) mine = k;
        }
    }
    const bool chosen = rank < p.n_used;
    const float v = chosen ? expf(value(mine >> 16) - m) : 0.f;
    if (p.renorm) {
        total = v;
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
    }
    float w = p.scale * (v / total);
    if (m == -INFINITY) w = 0.f;   // the same rules as above
    if (nan) w = __int_as_float(0x7fc00000);
    if (chosen) {
        p.ids[(size_t)t * p.n_used + rank] = 0xffff - (int)(mine & 0xffff);
        p.w[(size_t)t * p.n_used + rank] = w;
    }
}

// Two 16-bit logits to a register pay from 8 logits per lane on (131,072 tokens of
// bf16, 256 experts, the 8 largest: 62 us, singly 66; 128 experts: 64, singly 56,
// and the 2 largest of them 58 and 40).
template <class Act, int NV>
void launch_width(const RouteParams& p, bool wide, cudaStream_t st) {
    const int grid = (p.n_tokens + kWarps - 1) / kWarps;
    if constexpr (sizeof(Act) == 2 && NV > 4)
        if (wide && p.n_experts % 8 == 0) {
            k_route16<Act, NV><<<grid, kWarps * 32, 0, st>>>(p);
            return;
        }
    if (wide && p.n_experts % 4 == 0)
        k_route<Act, NV, 4><<<grid, kWarps * 32, 0, st>>>(p);
    else
        k_route<Act, NV, 1><<<grid, kWarps * 32, 0, st>>>(p);
}
template <class Act>
void launch_route(const RouteParams& p, cudaStream_t st) {
    const bool wide = ((uintptr_t)p.x | p.row_stride) % 16 == 0;
    if (p.n_experts <= 128)
        launch_width<Act, 4>(p, wide, st);
    else if (p.n_experts <= 256)
        launch_width<Act, 8>(p, wide, st);
    else if (p.n_experts <= 512)
        launch_width<Act, 16>(p, wide, st);
    else if (p.n_experts <= 1024)
        launch_width<Act, 32>(p, wide, st);
    else
        launch_width<Act, 64>(p, wide, st);
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
