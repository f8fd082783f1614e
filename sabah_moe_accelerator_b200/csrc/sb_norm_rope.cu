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
// Bound: DRAM, each row read once and written once, with the instructions per
// row not far behind. A row is a lane group of LPR lanes; a lane owns both
// halves of its pairs (W consecutive pairs, as two chunks of W values), so the
// rotation needs no exchange and only the sum of squares is shuffled. A warp
// takes several rows of one token and one kind (queries, keys or values), reads
// the token's cosines once for all of them and multiplies them by the weights:
// a turned value is then two products and one by the norm.
//
// Measured (one B200): 8191 tokens x (32 + 8 + 8) heads of 128, bf16: 42.7 us in a
// graph (4.8 TB/s), 45 called one by one; the same rows only copied take 35 us. What
// is left is the chain position -> cosines of a short task, which more warps would
// hide and registers do not allow: issue slots 69%, DRAM 46%, warps 44%. The kind of
// row is the CTA's, so that its tests and pointers are uniform (a flat index over all
// tasks of a token: 55 us), and place and position are read before the rows (after
// them: 45). Slower: one, three or six rows per task (68, 52, 60), 9 CTAs an SM for 8
// (47); with the flat index 8 values at a time (71), tasks in a loop with the next
// one's rows ahead (59), a CTA per token with the turn in shared memory (68).
#include "sb_act.cuh"
#include "sb_kernels.h"

namespace {

constexpr int kWarps = 4;
constexpr int kMaxDim = 256, kMaxAxes = 4, kMaxHeads = 16384;   // tasks of a token are a grid dimension

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
    unsigned q_blocks, kv_blocks;   // warp tasks of a token: for queries, for keys or values
};

// W consecutive values, loaded and stored at once
template <class T, int W>
struct alignas(sizeof(T) * W) Chunk {
    T v[W];
    __device__ void load(const T* p) { *this = *(const Chunk*)p; }
    __device__ static void store(T* p, const float* f) {
        Chunk c;
#pragma unroll
        for (int i = 0; i < W; ++i) c.v[i] = sb_from_float<T>(f[i]);
        *(Chunk*)p = c;
    }
};

// LPR lanes per row, NP chunk pairs of W values per lane, ITER rows per lane group
template <class Act, class Cache, int W, int LPR, int NP, int ITER>
__global__ void __launch_bounds__(kWarps * 32, 8) k_norm_rope(const __grid_constant__ NormRopeParams p) {
    constexpr int kRows = 32 / LPR;
    const int lane = threadIdx.x & 31, sub = lane % LPR, grp = lane / LPR;
    // a warp per token; the kind of row and which of them are the CTA's
    const int t = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (t >= p.n_tokens) return;
    const int kind = blockIdx.y < p.q_blocks ? 0 : blockIdx.y < p.q_blocks + p.kv_blocks ? 1 : 2;   // queries, keys, values
    const int block = blockIdx.y - (kind == 0 ? 0 : kind == 1 ? p.q_blocks : p.q_blocks + p.kv_blocks);
    const int row0 = block * kRows * ITER + grp, rows = kind == 0 ? p.n_q : p.n_kv;
    const size_t head = kind == 0 ? p.q_head : kind == 1 ? p.k_head : p.v_head;
    const uint8_t* src = kind == 0   ? p.q + (size_t)t * p.q_token
                         : kind == 1 ? p.k + (size_t)t * p.k_token
                                     : p.v + (size_t)t * p.v_token;
    src += row0 * head;
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
    // the token's place and position, then all of the task's rows are on their
    // way before anything waits
    const bool plain = kind != 2 && half && !p.pair_axis;
    const int pos = plain ? __ldg(p.positions + t) : 0;
    const long long slot = kind != 0 && p.slots ? __ldg((const long long*)p.slots + t) : -1;
    Chunk<Act, W> raw[ITER][NP][2];
#pragma unroll
    for (int it = 0; it < ITER; ++it)
#pragma unroll
        for (int n = 0; n < NP; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (row0 + it * kRows < rows && at[n][0] >= 0)
                    raw[it][n][h].load((const Act*)(src + it * kRows * head) + at[n][h]);
                else
#pragma unroll
                    for (int i = 0; i < W; ++i) raw[it][n][h].v[i] = sb_from_float<Act>(0.f);

    // where the rows go
    uint8_t* cache = nullptr;
    size_t cache_head = 0;
    if (slot >= (long long)p.n_slots) {
        if (lane == 0) atomicExch(p.err, SB_DERR_BAD_INDEX);
    } else if (slot >= 0) {
        const unsigned page = (unsigned)slot / (unsigned)p.page_size, in_page = (unsigned)slot - page * p.page_size;
        cache_head = kind == 1 ? p.kc_head : p.vc_head;
        cache = (kind == 1 ? p.k_cache + page * p.kc_page + in_page * p.kc_slot
                           : p.v_cache + page * p.vc_page + in_page * p.vc_slot) + row0 * cache_head;
    }
    if (kind == 2) {
        if (cache)
#pragma unroll
            for (int it = 0; it < ITER; ++it)
#pragma unroll
                for (int n = 0; n < NP; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (row0 + it * kRows >= rows || at[n][0] < 0) continue;
                        float f[W];
#pragma unroll
                        for (int i = 0; i < W; ++i) f[i] = sb_to_float(raw[it][n][h].v[i]);
                        Chunk<Cache, W>::store((Cache*)(cache + it * kRows * cache_head) + at[n][h], f);
                    }
        return;
    }
    Act* dst = (Act*)(kind == 0 ? p.q_out : p.k_out);
    if (dst) dst += ((size_t)t * rows + row0) * p.dim;

    // the turn of this lane's pairs (a, b) -> (a ca - b sb, a sa + b cb), with
    // the weights in it; a value that is not turned has (weight, 0, 0, weight)
    const float* weight = kind == 0 ? p.q_weight : p.k_weight;
    float ca[NP][W], sb[NP][W], sa[NP][W], cb[NP][W];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int pair0 = (sub + n * LPR) * W;
        const bool turned = pair0 * 2 < p.rope;
        float cs[2 * W];
#pragma unroll
        for (int i = 0; i < W; ++i) cs[2 * i] = 1.f, cs[2 * i + 1] = 0.f;
        if (turned && p.pair_axis == nullptr) {
            const bool out = pos < 0 || pos >= p.n_positions;
            if (out) atomicExch(p.err, SB_DERR_BAD_INDEX);
            const float* from = (const float*)(p.table + (size_t)(out ? 0 : pos) * half + pair0);
            Chunk<float, W> u[2];
            u[0].load(from), u[1].load(from + W);
#pragma unroll
            for (int i = 0; i < 2 * W; ++i) cs[i] = out ? __int_as_float(0x7fc00000) : u[i / W].v[i % W];
        } else if (turned) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const int axis = p.pair_axis[pair0 + i];
                const int pos = axis < p.n_axes ? p.positions[(size_t)axis * p.n_tokens + t] : -1;
                const bool out = pos < 0 || pos >= p.n_positions;
                if (out) atomicExch(p.err, SB_DERR_BAD_INDEX);
                const float* from = (const float*)(p.table + (size_t)(out ? 0 : pos) * half + pair0 + i);
                cs[2 * i] = out ? __int_as_float(0x7fc00000) : __ldg(from);
                cs[2 * i + 1] = out ? __int_as_float(0x7fc00000) : __ldg(from + 1);
            }
        }
        Chunk<float, W> w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (weight && at[n][0] >= 0)
                w[h].load(weight + at[n][h]);
            else
#pragma unroll
                for (int i = 0; i < W; ++i) w[h].v[i] = 1.f;
        // the lane's 2 W values in memory order; pair i is (i, i + W), or (2i, 2i + 1) in pairs mode
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const bool next = p.pairs_mode && W > 1;
            const float wa = next ? w[2 * i / W].v[2 * i % W] : w[0].v[i];
            const float wb = next ? w[(2 * i + 1) / W].v[(2 * i + 1) % W] : w[1].v[i];
            ca[n][i] = wa * cs[2 * i], sa[n][i] = wa * cs[2 * i + 1];
            sb[n][i] = wb * cs[2 * i + 1], cb[n][i] = wb * cs[2 * i];
        }
    }

#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        float x[NP][2 * W], sum = 0.f;
#pragma unroll
        for (int n = 0; n < NP; ++n)
#pragma unroll
            for (int i = 0; i < 2 * W; ++i) {
                x[n][i] = sb_to_float(raw[it][n][i / W].v[i % W]);
                sum += x[n][i] * x[n][i];
            }
#pragma unroll
        for (int o = LPR / 2; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (row0 + it * kRows >= rows) continue;
        const float inv = weight ? rsqrtf(sum * p.over_dim + p.eps) : 1.f;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            if (at[n][0] < 0) continue;
            // a value that is not turned leaves its partner's product with zero out: an
            // infinity or NaN there is none of its business (a predicate per product; a
            // branch for such lanes: 8191 tokens with half of each head turned 45.3 us, this 44.0)
            const bool turned = (sub + n * LPR) * 2 * W < p.rope;
            float y[2 * W];
            auto turn = [&](int i, int a, int b) {   // pair i, the lane's values a and b
                float u = x[n][a] * ca[n][i], v = x[n][b] * cb[n][i];
                if (turned) u -= x[n][b] * sb[n][i], v += x[n][a] * sa[n][i];
                y[a] = u * inv, y[b] = v * inv;
            };
            if (p.pairs_mode && W > 1) {
#pragma unroll
                for (int i = 0; i < W; ++i) turn(i, 2 * i, 2 * i + 1);
            } else {
#pragma unroll
                for (int i = 0; i < W; ++i) turn(i, i, i + W);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (dst) Chunk<Act, W>::store(dst + it * kRows * p.dim + at[n][h], y + h * W);
                if (cache) Chunk<Cache, W>::store((Cache*)(cache + it * kRows * cache_head) + at[n][h], y + h * W);
            }
        }
    }
}

template <class Act, class Cache, int W, int LPR, int NP, int ITER>
void launch(NormRopeParams p, cudaStream_t st) {
    const int per_task = 32 / LPR * ITER;
    p.q_blocks = (p.n_q + per_task - 1) / per_task;
    p.kv_blocks = (p.n_kv + per_task - 1) / per_task;
    const dim3 grid((p.n_tokens + kWarps - 1) / kWarps, p.q_blocks + p.kv_blocks * (p.slots ? 2 : 1));
    k_norm_rope<Act, Cache, W, LPR, NP, ITER><<<grid, kWarps * 32, 0, st>>>(p);
}

// Four rows per lane group once the rows of one would fill the chip twice over
// (148 SMs x 64 warps): the cosines, positions and indexes are then a fourth of
// the work (8191 tokens: 45 us, with one row 68; 2049 patches of 24 + 4 heads of
// 80: 10.4 and 16.5), where few rows want all the warps there are (64 tokens: 5.0
// us either way, the launch).
template <class Act, class Cache, int LPR>
void launch_wide(const NormRopeParams& p, cudaStream_t st) {
    if ((long long)p.n_tokens * (p.n_q + 2 * p.n_kv) * LPR / 32 > 2 * 148 * 64)
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
    if (n_tokens < 0 || n_q_heads < 0 || n_kv_heads < 0 || n_q_heads > kMaxHeads || n_kv_heads > kMaxHeads || head_dim <= 0 ||
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
    p.slots = d_slots, p.err = err;
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
