// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale * <q, k_j>,  lo <= j < len,  lo = window ? max(0, len - window) : 0
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  lse = m + ln sum_j exp(s_j - m)
//
// Key j of sequence b is row j % page_size of page block_table[b][j / page_size].
// A sequence of length zero gives zeros and lse = -inf. Nothing outside
// [lo, len) is read: not a key, not a table entry.
#include "sb_act.cuh"
#include "sb_kernels.h"

namespace {

constexpr int kMaxDim = 256;

struct AttendParams {
    const uint8_t* q;
    size_t q_seq, q_head;   // bytes
    const uint8_t *k, *v;
    size_t k_page, k_slot, k_head, v_page, v_slot, v_head;   // bytes
    int n_pages, page_size;
    const int32_t* table;
    size_t table_stride;    // elements
    int table_width;
    const int32_t* lens;
    int n_seqs, n_q, n_kv, dim, window;
    float scale_log2;       // scale * log2(e)
    uint8_t* out;
    float* lse;
    int* err;
};

// one warp per (sequence, query head), one key at a time
template <class Act, class Cache>
__global__ void k_attend(AttendParams p) {
    const int lane = threadIdx.x, b = blockIdx.x / p.n_q, h = blockIdx.x % p.n_q, kv = h / (p.n_q / p.n_kv);
    int len = p.lens[b];
    bool bad = len < 0 || len > (long long)p.table_width * p.page_size;
    if (bad) len = 0;
    const int lo = p.window > 0 ? max(0, len - p.window) : 0;
    constexpr int N = kMaxDim / 32;
    // sums of kBlock keys are added up among themselves first: one running fp32
    // sum over 10^5 keys would lose half its digits
    constexpr int kBlock = 64;
    float q[N], o[N], ob[N], m = -INFINITY, l = 0.f, lb = 0.f;
    for (int i = 0; i < N; ++i) {
        const int d = lane + 32 * i;
        q[i] = d < p.dim ? sb_to_float(((const Act*)(p.q + b * p.q_seq + h * p.q_head))[d]) : 0.f;
        o[i] = ob[i] = 0.f;
    }
    for (int j = lo; j < len; ++j) {
        const int page = p.table[b * p.table_stride + j / p.page_size];
        if (page < 0 || page >= p.n_pages) {
            bad = true;
            break;
        }
        const Cache* k = (const Cache*)(p.k + page * p.k_page + (j % p.page_size) * p.k_slot + kv * p.k_head);
        const Cache* v = (const Cache*)(p.v + page * p.v_page + (j % p.page_size) * p.v_slot + kv * p.v_head);
        float s = 0.f;
        for (int i = 0; i < N; ++i)
            if (lane + 32 * i < p.dim) s += q[i] * sb_to_float(k[lane + 32 * i]);
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
        s *= p.scale_log2;
        const float top = fmaxf(m, s), a = m == -INFINITY ? 0.f : exp2f(m - top), e = exp2f(s - top);
        m = top;
        l *= a;
        lb = lb * a + e;
        for (int i = 0; i < N; ++i)
            if (lane + 32 * i < p.dim) {
                o[i] *= a;
                ob[i] = ob[i] * a + e * sb_to_float(v[lane + 32 * i]);
            }
        if ((j - lo) % kBlock == kBlock - 1 || j == len - 1) {
            l += lb;
            lb = 0.f;
            for (int i = 0; i < N; ++i) {
                o[i] += ob[i];
                ob[i] = 0.f;
            }
        }
    }
    if (bad && lane == 0) atomicExch(p.err, SB_DERR_BAD_INDEX);
    const float nan = __int_as_float(0x7fc00000);
    for (int i = 0; i < N; ++i)
        if (lane + 32 * i < p.dim)
            ((Act*)p.out)[((size_t)b * p.n_q + h) * p.dim + lane + 32 * i] =
                sb_from_float<Act>(bad ? nan : len == lo ? 0.f : o[i] / l);
    if (p.lse && lane == 0)
        p.lse[(size_t)b * p.n_q + h] = bad ? nan : len == lo ? -INFINITY : 0.69314718f * (m + log2f(l));
}

}  // namespace

SABAH_API size_t sabah_attend_paged_workspace(int n_q_heads, int n_kv_heads, int head_dim) {
    (void)n_q_heads;
    (void)n_kv_heads;
    (void)head_dim;
    return 0;
}

SABAH_API int sabah_attend_paged(const void* d_q, size_t q_seq_stride, size_t q_head_stride, int act_type,
                                 const void* d_k_cache, size_t k_page_stride, size_t k_slot_stride,
                                 size_t k_head_stride, const void* d_v_cache, size_t v_page_stride,
                                 size_t v_slot_stride, size_t v_head_stride, int cache_type, int n_pages,
                                 int page_size, const int32_t* d_block_table, size_t table_stride, int table_width,
                                 const int32_t* d_lens, int n_seqs, int n_q_heads, int n_kv_heads, int head_dim,
                                 float scale, int window, void* d_out, float* d_lse, void* d_workspace,
                                 size_t workspace_bytes, void* stream) {
    int* err;
    cudaStream_t st;
    if (!sb_op_begin(stream, &st, &err)) return -1;
    const size_t ab = sb_act_bytes(act_type);
    const bool pair = (cache_type == SB_F16 || cache_type == SB_BF16) && (act_type == SB_F32 || act_type == cache_type);
    if (n_seqs < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads || n_q_heads > 65536 ||
        head_dim <= 0 || head_dim > kMaxDim || head_dim % 8 || !pair) {
        sb_set_error("invalid attend geometry (sequences %d, heads %d / %d, head size %d: a multiple of 8 to %d, "
                     "types %d over %d)", n_seqs, n_q_heads, n_kv_heads, head_dim, kMaxDim, act_type, cache_type);
        return -1;
    }
    if (n_pages < 0 || page_size <= 0 || table_width < 0 || window < 0 ||
        (long long)table_width * page_size > 0x7fffffffll) {
        sb_set_error("invalid attend cache (%d pages of %d, %d per sequence, window %d)", n_pages, page_size,
                     table_width, window);
        return -1;
    }
    if (n_seqs == 0) return 0;
    if (!d_q || !d_lens || !d_out || (table_width && (!d_k_cache || !d_v_cache || !d_block_table)) ||
        ((uintptr_t)d_q | q_seq_stride | q_head_stride | (uintptr_t)d_out) % ab ||
        ((uintptr_t)d_k_cache | (uintptr_t)d_v_cache | k_page_stride | k_slot_stride | k_head_stride | v_page_stride |
         v_slot_stride | v_head_stride) % 16 ||
        ((uintptr_t)d_block_table | (uintptr_t)d_lens | (uintptr_t)d_lse | table_stride) % 4) {
        sb_set_error("invalid attend arguments (a null pointer, or one that is not aligned: cache rows to 16 bytes)");
        return -1;
    }
    AttendParams p{};
    p.q = (const uint8_t*)d_q, p.q_seq = q_seq_stride, p.q_head = q_head_stride;
    p.k = (const uint8_t*)d_k_cache, p.v = (const uint8_t*)d_v_cache;
    p.k_page = k_page_stride, p.k_slot = k_slot_stride, p.k_head = k_head_stride;
    p.v_page = v_page_stride, p.v_slot = v_slot_stride, p.v_head = v_head_stride;
    p.n_pages = n_pages, p.page_size = page_size;
    p.table = d_block_table, p.table_stride = table_stride / 4, p.table_width = table_width;
    p.lens = d_lens, p.n_seqs = n_seqs, p.n_q = n_q_heads, p.n_kv = n_kv_heads, p.dim = head_dim, p.window = window;
    p.scale_log2 = scale * 1.44269504088896341f;
    p.out = (uint8_t*)d_out, p.lse = d_lse, p.err = err;
    (void)d_workspace;
    (void)workspace_bytes;
    const int slot = sb_timing_begin("attend_paged", st);
    const unsigned grid = (unsigned)n_seqs * (unsigned)n_q_heads;
    if (act_type == SB_F32)
        cache_type == SB_F16 ? k_attend<float, __half><<<grid, 32, 0, st>>>(p)
                             : k_attend<float, __nv_bfloat16><<<grid, 32, 0, st>>>(p);
    else if (act_type == SB_F16)
        k_attend<__half, __half><<<grid, 32, 0, st>>>(p);
    else
        k_attend<__nv_bfloat16, __nv_bfloat16><<<grid, 32, 0, st>>>(p);
    sb_timing_end(slot, st);
    return sb_cuda_ok(cudaGetLastError(), "attend launch") ? 0 : -1;
}
