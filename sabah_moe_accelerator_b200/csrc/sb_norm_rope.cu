// Per-head norms of queries and keys, the position rotation and the write of
// keys and values into the paged cache, in one pass over the projected rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * weight        (a null weight: y = x)
//   pair i < rope_dim / 2 is (i, i + rope_dim / 2) ("halves") or (2i, 2i + 1)
//   ("pairs"):  (a, b) -> (a c - b s, a s + b c),  (c, s) = table[pos(i)][i]
//   pos(i) = positions[pair_axis ? pair_axis[i] : 0][token]
//
// Sums, norms and the rotation are fp32; each output value is rounded once.
// The cosines come from a table: pos * frequency in fp32 would lose a radian's
// third decimal at positions of 1e5.
//
// Bound: DRAM, each row read once and written once. A row is a lane group of
// LPR lanes; a lane owns both halves of its pairs (W consecutive pairs, as two
// chunks of W values), so the rotation needs no exchange and only the sum of
// squares is shuffled. A warp takes several rows of one token and reads the
// token's cosines once for all of them.
#include "sb_act.cuh"
#include "sb_kernels.h"

namespace {

constexpr int kWarps = 8;
constexpr int kMaxDim = 256, kMaxAxes = 4;

struct NormRopeParams {
    const uint8_t *q, *k, *v;
    size_t q_token, q_head, k_token, k_head, v_token, v_head;   // bytes
    int n_q, n_kv, n_tokens, dim;
    const float *q_weight, *k_weight;
    float eps, over_dim;
    const float2* table;
    int n_positions, rope, pairs_mode;
    const int32_t* positions;
    const uint8_t* pair_axis;
    int n_axes;
    uint8_t *q_out, *k_out;
    uint8_t *k_cache, *v_cache;
    size_t kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;   // bytes
    int page_size;
    unsigned n_slots;
    const int64_t* slots;
    int* err;
    int rows, blocks;   // rows of a token; warp tasks of a token
};

template <class T, int W>
__device__ inline void load_chunk(const T* p, float* f) {
    if constexpr (W == 4 && sizeof(T) == 4) {
        const float4 u = *(const float4*)p;
        f[0] = u.x, f[1] = u.y, f[2] = u.z, f[3] = u.w;
    } else if constexpr (W == 4) {
        const uint2 u = *(const uint2*)p;
        const T* h = (const T*)&u;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = sb_to_float(h[i]);
    } else {
        f[0] = sb_to_float(*p);
    }
}
template <class T, int W>
__device__ inline void store_chunk(T* p, const float* f) {
    if constexpr (W == 4 && sizeof(T) == 4) {
        *(float4*)p = make_float4(f[0], f[1], f[2], f[3]);
    } else if constexpr (W == 4) {
        uint2 u;
        T* h = (T*)&u;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = sb_from_float<T>(f[i]);
        *(uint2*)p = u;
    } else {
        *p = sb_from_float<T>(f[0]);
    }
}

// LPR lanes per row, NP chunk pairs of W values per lane, ITER rows per lane group
template <class Act, class Cache, int W, int LPR, int NP, int ITER>
__global__ void __launch_bounds__(kWarps * 32) k_norm_rope(const __grid_constant__ NormRopeParams p) {
    constexpr int kRows = 32 / LPR;
    const unsigned task = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, sub = lane % LPR, grp = lane / LPR;
    const int t = (int)(task / (unsigned)p.blocks);
    if (t >= p.n_tokens) return;
    const int row0 = (int)(task - (unsigned)t * (unsigned)p.blocks) * kRows * ITER + grp;
    const int half = p.rope / 2;

    // where this lane's chunk pairs lie in a row
    int at[NP][2];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int cp = sub + n * LPR;
        const bool split = !p.pairs_mode && cp * 2 * W < p.rope;
        at[n][0] = cp * 2 * W >= p.dim ? -1 : split ? cp * W : cp * 2 * W;
        at[n][1] = split ? cp * W + half : cp * 2 * W + W;
    }
    // all of the task's rows are on their way before anything waits
    float x[ITER][NP][2][W];
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        const int r = row0 + it * kRows;
        const uint8_t* src = r < p.n_q            ? p.q + (size_t)t * p.q_token + (size_t)r * p.q_head
                             : r < p.n_q + p.n_kv ? p.k + (size_t)t * p.k_token + (size_t)(r - p.n_q) * p.k_head
                                                  : p.v + (size_t)t * p.v_token + (size_t)(r - p.n_q - p.n_kv) * p.v_head;
#pragma unroll
        for (int n = 0; n < NP; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (r < p.rows && at[n][0] >= 0)
                    load_chunk<Act, W>((const Act*)src + at[n][h], x[it][n][h]);
                else
#pragma unroll
                    for (int i = 0; i < W; ++i) x[it][n][h][i] = 0.f;
            }
    }
    long long slot = p.slots ? p.slots[t] : -1;
    // the cosines of this lane's pairs, once for all of its rows
    float c[NP][W], s[NP][W];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int pair0 = (sub + n * LPR) * W;
        const bool turned = pair0 * 2 < p.rope;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            c[n][i] = 1.f;
            s[n][i] = 0.f;
        }
        if (!turned) continue;
        if (p.pair_axis == nullptr) {
            const int pos = p.positions[t];
            const bool out = pos < 0 || pos >= p.n_positions;
            if (out) atomicExch(p.err, SB_DERR_BAD_INDEX);
            float cs[2 * W];
            const float* src = (const float*)(p.table + (size_t)(out ? 0 : pos) * half + pair0);
            if constexpr (W == 4) {
                load_chunk<float, W>(src, cs);
                load_chunk<float, W>(src + W, cs + W);
            } else {
                cs[0] = __ldg(src), cs[1] = __ldg(src + 1);
            }
#pragma unroll
            for (int i = 0; i < W; ++i) {
                c[n][i] = out ? __int_as_float(0x7fc00000) : cs[2 * i];
                s[n][i] = out ? __int_as_float(0x7fc00000) : cs[2 * i + 1];
            }
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const int axis = p.pair_axis[pair0 + i];
                const int pos = axis < p.n_axes ? p.positions[(size_t)axis * p.n_tokens + t] : -1;
                const bool out = pos < 0 || pos >= p.n_positions;
                if (out) atomicExch(p.err, SB_DERR_BAD_INDEX);
                const float2 cs = __ldg(p.table + (size_t)(out ? 0 : pos) * half + pair0 + i);
                c[n][i] = out ? __int_as_float(0x7fc00000) : cs.x;
                s[n][i] = out ? __int_as_float(0x7fc00000) : cs.y;
            }
        }
    }
    if (slot >= (long long)p.n_slots) {
        if (lane == 0) atomicExch(p.err, SB_DERR_BAD_INDEX);
        slot = -1;
    }
    const unsigned page = slot < 0 ? 0 : (unsigned)slot / p.page_size;
    const unsigned in_page = slot < 0 ? 0 : (unsigned)slot - page * p.page_size;

#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        const int r = row0 + it * kRows;
        const bool here = r < p.rows;
        const bool is_q = r < p.n_q, is_v = r >= p.n_q + p.n_kv;
        const float* weight = is_v ? nullptr : is_q ? p.q_weight : p.k_weight;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NP; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < W; ++i) sum += x[it][n][h][i] * x[it][n][h][i];
#pragma unroll
        for (int o = LPR / 2; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (!here) continue;
        const float inv = rsqrtf(sum * p.over_dim + p.eps);
        const int kv = is_v ? r - p.n_q - p.n_kv : r - p.n_q;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            if (at[n][0] < 0) continue;
            float y[2][W];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float w[W];
                if (weight) load_chunk<float, W>(weight + at[n][h], w);
#pragma unroll
                for (int i = 0; i < W; ++i) y[h][i] = weight ? x[it][n][h][i] * inv * w[i] : x[it][n][h][i];
            }
            if (!is_v && (sub + n * LPR) * 2 * W < p.rope) {
                float z[2][W];
                if (p.pairs_mode && W > 1) {   // (2i, 2i + 1): neighbours in the lane's 2 W values
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        const float a = (&y[0][0])[2 * i], b = (&y[0][0])[2 * i + 1];
                        (&z[0][0])[2 * i] = a * c[n][i] - b * s[n][i];
                        (&z[0][0])[2 * i + 1] = a * s[n][i] + b * c[n][i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        z[0][i] = y[0][i] * c[n][i] - y[1][i] * s[n][i];
                        z[1][i] = y[0][i] * s[n][i] + y[1][i] * c[n][i];
                    }
                }
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    y[0][i] = z[0][i];
                    y[1][i] = z[1][i];
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (is_q) {
                    store_chunk<Act, W>((Act*)p.q_out + ((size_t)t * p.n_q + r) * p.dim + at[n][h], y[h]);
                    continue;
                }
                if (!is_v && p.k_out)
                    store_chunk<Act, W>((Act*)p.k_out + ((size_t)t * p.n_kv + kv) * p.dim + at[n][h], y[h]);
                if (slot >= 0) {
                    uint8_t* dst = is_v ? p.v_cache + page * p.vc_page + in_page * p.vc_slot + kv * p.vc_head
                                        : p.k_cache + page * p.kc_page + in_page * p.kc_slot + kv * p.kc_head;
                    store_chunk<Cache, W>((Cache*)dst + at[n][h], y[h]);
                }
            }
        }
    }
}

template <class Act, class Cache, int W, int LPR, int NP, int ITER>
void launch(NormRopeParams p, cudaStream_t st) {
    const int per_task = 32 / LPR * ITER;
    p.blocks = (p.rows + per_task - 1) / per_task;
    const long long tasks = (long long)p.n_tokens * p.blocks;
    k_norm_rope<Act, Cache, W, LPR, NP, ITER><<<(unsigned)((tasks + kWarps - 1) / kWarps), kWarps * 32, 0, st>>>(p);
}

// Four rows per lane group once the rows of one would fill the chip twice over
// (148 SMs x 64 warps): the cosines, positions and indexes are then a fourth of
// the work, where few rows want all the warps there are.
template <class Act, class Cache, int LPR>
void launch_wide(const NormRopeParams& p, cudaStream_t st) {
    if ((long long)p.n_tokens * p.rows * LPR / 32 > 2 * 148 * 64)
        launch<Act, Cache, 4, LPR, 1, 4>(p, st);
    else
        launch<Act, Cache, 4, LPR, 1, 1>(p, st);
}

template <class Act, class Cache>
void launch_shape(const NormRopeParams& p, bool wide, cudaStream_t st) {
    if (!wide)
        launch<Act, Cache, 1, 32, kMaxDim / 64, 1>(p, st);
    else if (p.dim <= 64)
        launch_wide<Act, Cache, 8>(p, st);
    else if (p.dim <= 128)
        launch_wide<Act, Cache, 16>(p, st);
    else
        launch_wide<Act, Cache, 32>(p, st);
}

}  // namespace

SABAH_API int sabah_qk_norm_rope(const void* d_q, size_t q_token_stride, size_t q_head_stride, int n_q_heads,
                                 const void* d_k, size_t k_token_stride, size_t k_head_stride, const void* d_v,
                                 size_t v_token_stride, size_t v_head_stride, int n_kv_heads, int n_tokens,
                                 int head_dim, int act_type, const float* d_q_weight, const float* d_k_weight,
                                 float eps, const float* d_table, int n_positions, int rope_dim, int pairs_mode,
                                 const int32_t* d_positions, int n_axes, const uint8_t* d_pair_axis, void* d_q_out,
                                 void* d_k_out, void* d_k_cache, size_t k_page_stride, size_t k_slot_stride,
                                 size_t k_cache_head_stride, void* d_v_cache, size_t v_page_stride,
                                 size_t v_slot_stride, size_t v_cache_head_stride, int n_pages, int page_size,
                                 int cache_type, const int64_t* d_slots, void* stream) {
    int* err;
    cudaStream_t st;
    if (!sb_op_begin(stream, &st, &err)) return -1;
    const size_t ab = sb_act_bytes(act_type), cb = sb_act_bytes(cache_type);
    const bool cache = d_slots != nullptr;
    if (n_tokens < 0 || n_q_heads < 0 || n_kv_heads < 0 || n_q_heads > 65536 || n_kv_heads > 65536 || head_dim <= 0 ||
        head_dim > kMaxDim || head_dim % 2 || rope_dim < 0 || rope_dim > head_dim || rope_dim % 2 || !ab) {
        sb_set_error("invalid norm_rope geometry (tokens %d, heads %d / %d, head size %d of an even number to %d, "
                     "rotated %d, type %d)", n_tokens, n_q_heads, n_kv_heads, head_dim, kMaxDim, rope_dim, act_type);
        return -1;
    }
    if (n_tokens == 0) return 0;
    if (rope_dim && (!d_table || !d_positions || n_positions <= 0 || n_axes < 1 || n_axes > kMaxAxes)) {
        sb_set_error("invalid norm_rope rotation (positions %d, axes %d of at most %d, or no table)", n_positions,
                     n_axes, kMaxAxes);
        return -1;
    }
    if (cache && (!d_v || !d_k_cache || !d_v_cache || n_pages <= 0 || page_size <= 0 || (cb != 2) ||
                  (long long)n_pages * page_size > 0x7fffffffll)) {
        sb_set_error("invalid norm_rope cache (%d pages of %d, type %d: f16 or bf16)", n_pages, page_size, cache_type);
        return -1;
    }
    const int rows = n_q_heads + n_kv_heads * (cache ? 2 : 1);
    if ((long long)n_tokens * rows > 0x7fffffffll) {
        sb_set_error("norm_rope: %d tokens of %d rows are too many for one call", n_tokens, rows);
        return -1;
    }
    if (rows == 0) return 0;
    if ((n_q_heads && (!d_q || !d_q_out)) || (n_kv_heads && (!d_k || (!cache && !d_k_out)))) {
        sb_set_error("invalid norm_rope arguments (a null row or output pointer)");
        return -1;
    }
    // every row pointer and stride in use, for a given element size and vector width
    size_t act_bits = (uintptr_t)d_q_out | (uintptr_t)d_k_out, cache_bits = 0, f32_bits = 0;
    if (n_q_heads) act_bits |= (uintptr_t)d_q | q_token_stride | q_head_stride;
    if (n_kv_heads) act_bits |= (uintptr_t)d_k | k_token_stride | k_head_stride;
    if (cache) {
        act_bits |= (uintptr_t)d_v | v_token_stride | v_head_stride;
        cache_bits = (uintptr_t)d_k_cache | (uintptr_t)d_v_cache | k_page_stride | k_slot_stride | k_cache_head_stride |
                     v_page_stride | v_slot_stride | v_cache_head_stride;
    }
    f32_bits = (uintptr_t)d_q_weight | (uintptr_t)d_k_weight;
    if (act_bits % ab || cache_bits % 2 || f32_bits % 4 || (uintptr_t)d_table % 4 || (uintptr_t)d_positions % 4 ||
        (uintptr_t)d_slots % 8) {
        sb_set_error("invalid norm_rope arguments (a pointer or stride is not a whole number of elements)");
        return -1;
    }
    NormRopeParams p{};
    p.q = (const uint8_t*)d_q, p.k = (const uint8_t*)d_k, p.v = (const uint8_t*)d_v;
    p.q_token = q_token_stride, p.q_head = q_head_stride;
    p.k_token = k_token_stride, p.k_head = k_head_stride;
    p.v_token = v_token_stride, p.v_head = v_head_stride;
    p.n_q = n_q_heads, p.n_kv = n_kv_heads, p.n_tokens = n_tokens, p.dim = head_dim;
    p.q_weight = d_q_weight, p.k_weight = d_k_weight, p.eps = eps, p.over_dim = 1.f / head_dim;
    p.table = (const float2*)d_table, p.n_positions = n_positions, p.rope = rope_dim, p.pairs_mode = pairs_mode;
    p.positions = d_positions, p.pair_axis = d_pair_axis, p.n_axes = n_axes;
    p.q_out = (uint8_t*)d_q_out, p.k_out = (uint8_t*)d_k_out;
    p.k_cache = (uint8_t*)d_k_cache, p.v_cache = (uint8_t*)d_v_cache;
    p.kc_page = k_page_stride, p.kc_slot = k_slot_stride, p.kc_head = k_cache_head_stride;
    p.vc_page = v_page_stride, p.vc_slot = v_slot_stride, p.vc_head = v_cache_head_stride;
    p.page_size = cache ? page_size : 1, p.n_slots = cache ? (unsigned)n_pages * (unsigned)page_size : 0;
    p.slots = d_slots, p.err = err, p.rows = rows;
    // four values at a time where rows, pairs and pointers allow it
    const bool wide = head_dim % 8 == 0 && rope_dim % 8 == 0 && act_bits % (4 * ab) == 0 && cache_bits % 8 == 0 &&
                      (f32_bits | (uintptr_t)d_table) % 16 == 0;
    const int slot = sb_timing_begin("qk_norm_rope", st);
    const bool bf = cache ? cache_type == SB_BF16 : true;
    if (act_type == SB_F32)
        bf ? launch_shape<float, __nv_bfloat16>(p, wide, st) : launch_shape<float, __half>(p, wide, st);
    else if (act_type == SB_F16)
        bf ? launch_shape<__half, __nv_bfloat16>(p, wide, st) : launch_shape<__half, __half>(p, wide, st);
    else
        bf ? launch_shape<__nv_bfloat16, __nv_bfloat16>(p, wide, st) : launch_shape<__nv_bfloat16, __half>(p, wide, st);
    sb_timing_end(slot, st);
    return sb_cuda_ok(cudaGetLastError(), "norm_rope launch") ? 0 : -1;
}
