// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale * <q, k_j>,  lo <= j < len,  lo = window ? max(0, len - window) : 0
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  lse = m + ln sum_j exp(s_j - m)
//
// Key j of sequence b is row j % page_size of page block_table[b][j / page_size].
// A sequence of length zero gives zeros and lse = -inf. Nothing outside
// [lo, len) is read: not a key, not a table entry.
//
// Bound: DRAM, every key and value row once. A key-value head's query heads
// (up to 16: the rows of an MMA tile) are taken together, so the rows are read
// once for all of them; the arithmetic is 16-row mma.sync on 16 keys at a time,
// a fraction of the tensor rate and well under the time the rows take to
// arrive. tcgen05's 128-row tiles would be 87-99% padding here.
//
// The work is a list of steps of 16 keys over all (sequence, key-value head)
// rows. Each warp takes an equal, contiguous part of it, whatever the lengths:
// one long sequence spreads over the whole chip, and many short ones stay whole
// within a warp. Warps never wait for one another; each streams its own keys
// and values through its own ring in shared memory (cp.async, rows padded by 16
// bytes so that ldmatrix meets no bank twice). A row that ends in a part is
// left as (m, l, unnormalised out) in the workspace, and a second, small launch
// (a programmatic dependent of the first) joins the pieces of each cut row in
// a fixed order. Rows of at most kWhole steps are never cut; where the block
// table cannot hold a longer sequence the second launch is left out.
//
// Precision: scores, m, l and out are fp32. The MMA takes 16-bit factors, so
// fp32 queries and the softmax weights are split into a sum of 16-bit parts
// (f16: 2 parts, 22 bits; bf16: 3 parts, 24 bits), each multiplied exactly.
// With 16-bit outputs the weights take two parts, which leaves the output's
// own rounding as the only one. f16 parts keep their bits only in f16's normal
// range: a query row is scaled to below 2 by a power of two, and the weights
// are computed times 2^12. The parts but the last are cut off rather than
// rounded, so all of a number's parts have its sign, and the first part's
// products are summed apart from the others': where an infinite key or value
// makes the others infinite or NaN (0 * inf), add_rest() leaves the first.
#include <algorithm>

#include "sb_act.cuh"
#include "sb_kernels.h"

namespace {

constexpr int kMaxDim = 256;
constexpr int kMaxSeqs = 1024;   // per launch: the scan of the lengths sits in shared memory
constexpr int kStep = 16;        // keys per step
constexpr int kWhole = 8;        // rows of at most this many steps are never cut
constexpr int kMinSteps = 4;     // and a part is at least this long
constexpr int kRowCost = 2;      // what a row costs besides its steps, in steps
constexpr int kSmemLimit = 227 * 1024;

struct AttendParams {
    const uint8_t* q;
    size_t q_seq, q_head;   // bytes
    int q_pairs;            // pairs of query values are aligned
    const uint8_t *k, *v;
    size_t k_page, k_slot, k_head, v_page, v_slot, v_head;   // bytes
    int n_pages, page_size, page_shift;   // shift: log2(page_size), or -1
    const int32_t* table;
    size_t table_stride;    // elements
    int table_width;
    const int32_t* lens;
    int n_seqs, n_q, n_kv, dim, window;
    int group, tiles;       // query heads per key-value head; 16-row tiles of them
    float scale_log2;       // scale * log2(e)
    uint8_t* out;
    float* lse;
    int* err;
    int2* cuts;             // per warp: the row cut in its part (-1: none) and its number of pieces
    float* pieces;          // per warp two: the row it enters in the middle of, the row it leaves early
    int piece_floats, piece_rows;
};

// ------------------------------------------------------------ PTX helpers
__device__ inline uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ inline void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ inline void copy16_or_zero(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ inline void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ inline void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ inline void ldsm4(uint32_t* r, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ inline void ldsm4t(uint32_t* r, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <class T>
__device__ inline void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ inline float exp2_fast(float x) {   // 2 ulp; exp2(-inf) = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two values as 16-bit ones, cut off (CUT) or rounded to nearest
template <class T, bool CUT>
__device__ inline uint32_t pack2(float a, float b) {
    uint32_t u;
    if constexpr (std::is_same<T, __half>::value && CUT)
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(b), "f"(a));
    else if constexpr (std::is_same<T, __half>::value)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(b), "f"(a));
    else if constexpr (CUT)
        u = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(b), "f"(a));
    return u;
}
// first + rest, where rest counts only if it is a number: first is infinite or
// NaN whenever rest is, and of the same sign (fmaxf takes a NaN's other side)
__device__ inline float add_rest(float first, float rest) { return first + fmaxf(rest, -3.402823466e38f); }
template <class T>
__device__ inline float2 unpack2(uint32_t u) {
    if constexpr (std::is_same<T, __half>::value)
        return __half22float2(*(const __half2*)&u);
    else
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// the next part of (a, b), which keep what it leaves
template <class T>
__device__ inline uint32_t take_part(float& a, float& b, bool last) {
    const uint32_t u = last ? pack2<T, false>(a, b) : pack2<T, true>(a, b);
    const float2 f = unpack2<T>(u);
    a -= f.x;
    b -= f.y;
    return u;
}
// e with 2^e <= x < 2^(e + 1); 0 for zero, infinity and NaN
__device__ inline int exponent(float x) {
    return x > 0.f && x < INFINITY ? min(max((__float_as_int(x) >> 23) - 127, -126), 126) : 0;
}
__device__ inline float power_of_two(int e) { return __int_as_float((127 + e) << 23); }

// ------------------------------------------------------------ shapes
// DP: head size rounded up to a tile width. Each warp has a ring of kStages
// steps of 16 keys and 16 values.
template <int DP>
struct Shape {
    static constexpr int kRow = DP * 2 + 16;                  // bytes of a padded row
    static constexpr int kStage = 2 * kStep * kRow;
    static constexpr int kStages = DP <= 64 ? 6 : DP <= 96 ? 4 : 3;
    static constexpr int kLanes = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;   // lanes that copy one row
    static constexpr int kWarps = 8;                          // at most
};

// The scan of the lengths: cost of the sequences before b, for one row of each.
// A row takes its steps, then kRowCost idle places in the list, so that parts
// of many short rows and parts of one long row take as long.
struct Seqs {
    long long* pre;   // [n_seqs + 1]
    int* len;         // [n_seqs], -1 where out of range
};
__device__ inline int window_start(int len, int window) { return window > 0 ? max(0, len - window) : 0; }
__device__ inline int seq_steps(int len, int window) {
    return len <= 0 ? 1 : (len + kStep - 1) / kStep - window_start(len, window) / kStep;
}
// a / b of non-negative numbers; the 64-bit division is a long subroutine
__device__ inline long long div_fast(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

// A place in the list of steps; each warp has one that loads and one that computes.
struct Cursor {
    int b, h;            // sequence, row of it (key-value head and tile)
    int j, end, steps;   // step in the row, where this warp leaves it, the row's steps
    int len, lo;
    long long row_at;    // the row's first step in the list
};

// starts the row at c.b, c.h; the warp takes its steps from j on
__device__ inline void enter_row(Cursor& c, const Seqs& s, const AttendParams& p, int j, long long until) {
    c.len = s.len[c.b];
    c.lo = window_start(max(c.len, 0), p.window);
    c.steps = (int)(s.pre[c.b + 1] - s.pre[c.b]) - kRowCost;
    c.j = j;
    c.end = c.steps <= kWhole ? c.steps : (int)min((long long)c.steps, until - c.row_at);
}
// false at the end of the warp's part
__device__ inline bool next_row(Cursor& c, const Seqs& s, const AttendParams& p, long long until) {
    c.row_at += c.steps + kRowCost;
    if (c.row_at >= until) return false;
    if (++c.h == p.n_kv * p.tiles) {
        c.h = 0;
        if (++c.b == p.n_seqs) return false;
    }
    enter_row(c, s, p, 0, until);
    return true;
}

// ------------------------------------------------------------ the loading side
// One warp's copies into its ring, kStages - 1 steps ahead of its arithmetic.
// Block table entries are held 32 to a register, one per lane, and the register
// after the current one is always on its way, as are the first entries of this
// sequence (the next key-value head starts there again) and of the next.
template <int DP>
struct Loader {
    using S = Shape<DP>;
    const AttendParams& p;
    const Seqs& seqs;
    const long long until;
    const int lane;
    const uint32_t ring;
    Cursor c;
    bool more = true;
    uint32_t bad_steps = 0;             // bit per stage: the step met a page out of range
    int first, cur, next, head, ahead;  // cur: entries first ..; next: the 32 after them

    __device__ Loader(const AttendParams& p_, const Seqs& s_, long long until_, int lane_, uint32_t ring_, const Cursor& c_)
        : p(p_), seqs(s_), until(until_), lane(lane_), ring(ring_), c(c_) {
        first = entry_of((c.lo / kStep + c.j) * kStep);
        cur = entries(c.b, first);
        next = entries(c.b, first + 32);
        head = entries(c.b, entry_of(c.lo / kStep * kStep));
        ahead = c.b + 1 < p.n_seqs ? first_entries(c.b + 1) : -1;
    }
    __device__ int entry_of(int key) const {
        return p.page_shift >= 0 ? key >> p.page_shift : (int)((unsigned)key / (unsigned)p.page_size);
    }
    // table entries e .. e + 31 of sequence b that its window needs, -1 for the others
    __device__ int entries(int b, int e) const {
        const int len = seqs.len[b], lo = window_start(max(len, 0), p.window);
        return len > lo && e + lane >= entry_of(lo) && e + lane <= entry_of(len - 1)
                   ? __ldg(p.table + b * p.table_stride + e + lane) : -1;
    }
    __device__ int first_entries(int b) const {
        const int lo = window_start(max(seqs.len[b], 0), p.window);
        return entries(b, entry_of(lo / kStep * kStep));
    }
    __device__ int page_of(int e) const {   // e: per lane, first <= e < first + 64
        const int a = __shfl_sync(~0u, cur, e - first), b = __shfl_sync(~0u, next, e - first);
        return e - first < 32 ? a : b;
    }
    __device__ void advance() {
        if (++c.j < c.end) return;
        const int b = c.b;
        more = next_row(c, seqs, p, until);
        if (!more) return;
        if (c.b != b) {
            head = ahead;
            ahead = c.b + 1 < p.n_seqs ? first_entries(c.b + 1) : -1;
        }
        first = entry_of(c.lo / kStep * kStep);
        cur = head;
        next = entries(c.b, first + 32);
    }
    __device__ void issue(int stage) {
        if (more) {
            const int key0 = (c.lo / kStep + c.j) * kStep, kv = p.tiles == 1 ? c.h : c.h / p.tiles;
            const int e0 = entry_of(key0);
            if (e0 >= first + 32) {
                first += 32;
                cur = next;
                next = entries(c.b, first + 32);
            }
            const int copy_lane = lane % S::kLanes, copy_row = lane / S::kLanes;
            const bool copies = copy_lane * 8 < p.dim;
            const uint32_t dst = ring + stage * S::kStage + copy_row * S::kRow + copy_lane * 16;
            constexpr int kAtOnce = 32 / S::kLanes, kTimes = kStep / kAtOnce;
            const uint8_t* nowhere = (const uint8_t*)p.pieces;   // an address for copies of no bytes
            bool bad;
            if (p.page_size % kStep == 0) {   // the step lies in one page
                const int page = page_of(e0);
                bad = (page < 0 || page >= p.n_pages) && c.len > c.lo;
                const bool none = page < 0 || page >= p.n_pages;
                const long long slot = key0 - e0 * p.page_size + copy_row;
                const uint8_t* k = p.k + (none ? 0 : page) * p.k_page + slot * p.k_slot + kv * p.k_head + copy_lane * 16;
                const uint8_t* v = p.v + (none ? 0 : page) * p.v_page + slot * p.v_slot + kv * p.v_head + copy_lane * 16;
                if (!none && key0 >= c.lo && key0 + kStep <= c.len) {
                    if (copies) {
#pragma unroll
                        for (int i = 0; i < kTimes; ++i, k += kAtOnce * p.k_slot) copy16(dst + i * kAtOnce * S::kRow, k);
#pragma unroll
                        for (int i = 0; i < kTimes; ++i, v += kAtOnce * p.v_slot)
                            copy16(dst + (kStep + i * kAtOnce) * S::kRow, v);
                    }
                } else if (copies) {
#pragma unroll
                    for (int i = 0; i < kTimes; ++i, k += kAtOnce * p.k_slot, v += kAtOnce * p.v_slot) {
                        const int key = key0 + i * kAtOnce + copy_row;
                        const bool real = !none && key >= c.lo && key < c.len;
                        copy16_or_zero(dst + i * kAtOnce * S::kRow, real ? k : nowhere, real);
                        copy16_or_zero(dst + (kStep + i * kAtOnce) * S::kRow, real ? v : nowhere, real);
                    }
                }
            } else {   // lane i finds key i's place, the lanes that copy it ask that lane
                const int key = key0 + (lane & 15), inside = min(max(key, c.lo), max(c.len - 1, c.lo));
                const int e = entry_of(inside), page = page_of(e);
                const bool valid = key >= c.lo && key < c.len, out = page < 0 || page >= p.n_pages;
                bad = __any_sync(~0u, valid && out);
                const unsigned slot = (unsigned)inside - (unsigned)e * (unsigned)p.page_size;
                const bool real = valid && !out;
                const long long ko = real ? (long long)(page * p.k_page + slot * p.k_slot + kv * p.k_head) : -1;
                const long long vo = real ? (long long)(page * p.v_page + slot * p.v_slot + kv * p.v_head) : -1;
#pragma unroll
                for (int i = 0; i < kTimes; ++i) {
                    const int r = i * kAtOnce + copy_row;
                    const long long a = __shfl_sync(~0u, ko, r), b = __shfl_sync(~0u, vo, r);
                    if (!copies) continue;
                    copy16_or_zero(dst + i * kAtOnce * S::kRow, a < 0 ? nowhere : p.k + a + copy_lane * 16, a >= 0);
                    copy16_or_zero(dst + (kStep + i * kAtOnce) * S::kRow, a < 0 ? nowhere : p.v + b + copy_lane * 16, a >= 0);
                }
            }
            bad_steps &= ~(1u << stage);
            if (bad) {
                bad_steps |= 1u << stage;
                if (lane == 0) atomicExch(p.err, SB_DERR_BAD_INDEX);
            }
            advance();
        }
        copy_commit();
    }
};

// ------------------------------------------------------------ the kernel
// QP: parts of a query value (1: it has the cache's type); the weights take as
// many, and at least two. HALF: at most 8 query heads per key-value head; the
// tile's rows 8-15 then hold the second parts of rows 0-7, so one MMA multiplies
// both parts, and the query fragments stay in registers. With 9-16 heads each
// part is an MMA of its own and the queries lie in shared memory.
template <class Cache, int DP, int QP, bool HALF>
__global__ void __launch_bounds__(Shape<DP>::kWarps * 32, 1) k_attend(const AttendParams p) {
    using S = Shape<DP>;
    using Act = typename std::conditional<QP == 1, Cache, float>::type;
    constexpr int PP = QP == 1 ? 2 : QP;
    constexpr int R = HALF ? 1 : 2;          // row halves with heads of their own
    constexpr int ND = DP / 16;
    constexpr float kUp = std::is_same<Cache, __half>::value ? 12.f : 0.f;
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, n_warps = blockDim.x >> 5;

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- the scan of the lengths
    Seqs seqs{(long long*)smem, (int*)(smem + 8 * (p.n_seqs + 1))};
    __shared__ long long warp_sum[32];
    {
        const int per = (p.n_seqs + blockDim.x - 1) / blockDim.x, b0 = threadIdx.x * per;
        long long sum = 0;
        for (int b = b0; b < min(b0 + per, p.n_seqs); ++b) {
            int len = p.lens[b];
            if (len < 0 || len > (long long)p.table_width * p.page_size) {
                len = -1;
                if (blockIdx.x == 0) atomicExch(p.err, SB_DERR_BAD_INDEX);
            }
            seqs.len[b] = len;
            sum += seq_steps(len, p.window) + kRowCost;
        }
        long long run = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(~0u, run, o);
            if (lane >= o) run += x;
        }
        if (lane == 31) warp_sum[wid] = run;
        __syncthreads();
        run -= sum;
        for (int w = 0; w < wid; ++w) run += warp_sum[w];
        for (int b = b0; b < min(b0 + per, p.n_seqs); ++b) {
            seqs.pre[b] = run;
            run += seq_steps(seqs.len[b], p.window) + kRowCost;
        }
        if (b0 < p.n_seqs && b0 + per >= p.n_seqs) seqs.pre[p.n_seqs] = run;
        __syncthreads();
    }

    // ---- this warp's part of the list; neighbours in it sit on different SMs
    const int w = wid * gridDim.x + blockIdx.x, n_rows = p.n_kv * p.tiles;
    const long long total = seqs.pre[p.n_seqs] * n_rows, all_warps = (long long)gridDim.x * n_warps;
    const long long part = max(div_fast(total + all_warps - 1, all_warps), (long long)kMinSteps);
    const long long from = w * part, until = min(from + part, total);
    if (lane == 0) p.cuts[w] = make_int2(-1, 0);
    if (from >= total) return;
    Cursor cc;
    {
        // the last sequence that starts at or before `from`: 32 probes at a time
        int a = 0, span = p.n_seqs;   // it is in [a, a + span)
        while (span > 1) {
            const int hop = (span + 31) / 32, at = a + lane * hop;
            const unsigned hit = __ballot_sync(~0u, at < a + span && seqs.pre[min(at, p.n_seqs)] * n_rows <= from);
            const int last = 31 - __clz(hit);
            span = min(hop, a + span - (a + last * hop));
            a += last * hop;
        }
        cc.b = a;
        const long long at = from - seqs.pre[a] * n_rows, cost = seqs.pre[a + 1] - seqs.pre[a];
        cc.h = (int)div_fast(at, cost);
        const int j = (int)(at - cc.h * cost);
        cc.row_at = from - j;
        enter_row(cc, seqs, p, j, until);
        // a whole row is its first step's warp's
        if ((j >= cc.steps || (cc.steps <= kWhole && j > 0)) && !next_row(cc, seqs, p, until)) return;
    }

    // ---- shared memory of this warp: the ring, then (not HALF) the query rows
    const int rows = min(p.group, 16), q_rows = HALF ? 0 : rows * QP;
    const uint32_t head = (12 * p.n_seqs + 8 + 15) / 16 * 16;
    uint8_t* mine = smem + head + wid * (S::kStages * S::kStage + q_rows * S::kRow);
    uint8_t* q_mem = mine + S::kStages * S::kStage;
    const uint32_t ring = smem_addr(mine);
    const int g = lane >> 2, quad = lane & 3;
    Act qx[HALF ? ND : 1][4];   // the row's query values 16 d + 2 quad + {0, 1, 8, 9}, as they are
    auto fetch_queries = [&](const Cursor& c) {
        if constexpr (HALF) {
            const int first = c.h * p.group, heads = p.group;
            const Act* src = (const Act*)(p.q + c.b * p.q_seq + (first + min(g, heads - 1)) * p.q_head);
            if (p.q_pairs) {
                struct alignas(2 * sizeof(Act)) Pair { Act a, b; };
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int at = 16 * d + 2 * quad + i * 8;
                        const Pair u = *(const Pair*)(src + (at < p.dim ? at : 0));
                        qx[d][2 * i] = u.a, qx[d][2 * i + 1] = u.b;
                    }
            } else {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = 16 * d + 2 * quad + (i & 1) + (i >> 1) * 8;
                        qx[d][i] = src[at < p.dim ? at : 0];
                    }
            }
        }
    };
    fetch_queries(cc);
    Loader<DP> loader(p, seqs, until, lane, ring, cc);
    if (p.dim < DP) {   // columns past the head size stay zero
        const int pad = (DP - p.dim) / 8, n = (S::kStages * 2 * kStep + q_rows) * pad;
        for (int i = lane; i < n; i += 32)
            *(uint4*)(mine + i / pad * S::kRow + (p.dim + i % pad * 8) * 2) = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) loader.issue(i);

    // ---- the computing side
    float o[DP / 8][2 * R], m[R], l[R], unscale[R];
    uint32_t qf[HALF ? ND : 1][QP == 1 ? 2 : 2 * QP];   // HALF: per 16 dimensions, the parts of both 8s
    const uint32_t k_lane = ((lane >> 4) * 8 + (lane & 7)) * S::kRow + ((lane >> 3) & 1) * 16;
    const uint32_t v_lane = kStep * S::kRow + (((lane >> 3) & 1) * 8 + (lane & 7)) * S::kRow + (lane >> 4) * 16;
    int stage = 0;
    for (bool live = true; live;) {
        const int tile = p.tiles == 1 ? 0 : cc.h % p.tiles, kv = p.tiles == 1 ? cc.h : cc.h / p.tiles;
        const int first_head = kv * p.group + tile * 16, heads = min(16, p.group - tile * 16);
        const uint8_t* q_row0 = p.q + cc.b * p.q_seq + first_head * p.q_head;

        // ---- this row's queries, split into parts
#pragma unroll
        for (int r = 0; r < R; ++r) unscale[r] = 1.f;
        if constexpr (HALF) {
            // values past the head size are zero
            auto value = [&](int d, int i) {
                return 16 * d + 2 * quad + (i >> 1) * 8 < p.dim ? sb_to_float(qx[d][i]) : 0.f;
            };
            if constexpr (QP == 1) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float a = value(d, 2 * i), b = value(d, 2 * i + 1);
                        qf[d][i] = take_part<Cache>(a, b, true);
                    }
            } else {
                float top = 0.f;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(value(d, i)));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                const int e = exponent(top);
                unscale[0] = power_of_two(e);
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float a = value(d, 2 * i) * power_of_two(-e), b = value(d, 2 * i + 1) * power_of_two(-e);
#pragma unroll
                        for (int s = 0; s < QP; ++s) qf[d][i * QP + s] = take_part<Cache>(a, b, s == QP - 1);
                    }
            }
        } else {
            __syncwarp();
            for (int r = 0; r < heads; ++r) {
                const Act* src = (const Act*)(q_row0 + r * p.q_head);
                float x[(DP + 31) / 32], top = 0.f;
#pragma unroll
                for (int i = 0; i < (DP + 31) / 32; ++i) {
                    const int d = lane + 32 * i;
                    x[i] = d < p.dim ? sb_to_float(src[d]) : 0.f;
                    top = fmaxf(top, fabsf(x[i]));
                }
                int e = 0;
                if constexpr (QP > 1) {
#pragma unroll
                    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, s));
                    e = exponent(top);
                    if (r == g) unscale[0] = power_of_two(e);
                    if (r == g + 8) unscale[R - 1] = power_of_two(e);
                }
#pragma unroll
                for (int i = 0; i < (DP + 31) / 32; ++i) {
                    const int d = lane + 32 * i;
                    float rest = x[i] * power_of_two(-e), zero = 0.f;
#pragma unroll
                    for (int s = 0; s < QP; ++s) {
                        const uint32_t u = take_part<Cache>(rest, zero, s == QP - 1);
                        if (d < p.dim) ((uint16_t*)(q_mem + (s * rows + r) * S::kRow))[d] = (uint16_t)u;
                    }
                }
            }
            __syncwarp();
        }
        const uint32_t q_lane = smem_addr(q_mem) + min(lane & 15, heads - 1) * S::kRow + (lane >> 4) * 16;

#pragma unroll
        for (int t = 0; t < DP / 8; ++t)
#pragma unroll
            for (int i = 0; i < 2 * R; ++i) o[t][i] = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
        }
        bool row_bad = cc.len < 0;
        const int first_j = cc.j;
        for (; cc.j < cc.end; ++cc.j) {
            copy_wait<S::kStages - 2>();
            __syncwarp();   // and every lane has read the stage before, which the next copy fills
            row_bad |= (loader.bad_steps >> stage) & 1;
            const uint32_t at = ring + stage * S::kStage;
            loader.issue(stage == 0 ? S::kStages - 1 : stage - 1);

            // ---- scores of the tile's rows and 16 keys: first the products of
            // the first parts, and apart from them those of the rest
            float sc[R][2][2];   // [row half][key tile][pair]
            if constexpr (HALF) {
                float c[2][2][4] = {}, e[2][4] = {};
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    uint32_t kf[4];
                    ldsm4(kf, at + k_lane + d * 32);
                    const uint32_t qa[4] = {qf[d][0], qf[d][QP == 1 ? 0 : 1], qf[d][QP == 1 ? 1 : QP], qf[d][QP == 1 ? 1 : QP + 1]};
                    mma16816<Cache>(c[d & 1][0], qa, kf[0], kf[1]);
                    mma16816<Cache>(c[d & 1][1], qa, kf[2], kf[3]);
                    if constexpr (QP == 3) {
                        const uint32_t q3[4] = {qf[d][2], qf[d][2], qf[d][5], qf[d][5]};
                        mma16816<Cache>(e[0], q3, kf[0], kf[1]);
                        mma16816<Cache>(e[1], q3, kf[2], kf[3]);
                    }
                }
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        sc[0][t][i] = c[0][t][i] + c[1][t][i];
                        if constexpr (QP > 1)
                            sc[0][t][i] = add_rest(sc[0][t][i], (c[0][t][2 + i] + c[1][t][2 + i]) + e[t][i]);
                    }
            } else {
                float c[2][2][4] = {};
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    uint32_t kf[4];
                    ldsm4(kf, at + k_lane + d * 32);
#pragma unroll
                    for (int s = 0; s < QP; ++s) {
                        uint32_t qa[4];
                        ldsm4(qa, q_lane + s * rows * S::kRow + d * 32);
                        const int chain = QP == 1 ? d & 1 : s != 0;
                        mma16816<Cache>(c[chain][0], qa, kf[0], kf[1]);
                        mma16816<Cache>(c[chain][1], qa, kf[2], kf[3]);
                    }
                }
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float a = c[0][t][2 * r + i], b = c[1][t][2 * r + i];
                            sc[r][t][i] = QP == 1 ? a + b : add_rest(a, b);
                        }
            }

            // ---- the running softmax
            const int key0 = (cc.lo / kStep + cc.j) * kStep;
            const bool edge = key0 < cc.lo || key0 + kStep > cc.len;
            float alpha[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float f = p.scale_log2 * unscale[r];
                float top = m[r];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        sc[r][t][i] *= f;
                        const int key = key0 + 8 * t + 2 * quad + i;
                        if (edge && (key < cc.lo || key >= cc.len)) sc[r][t][i] = -INFINITY;
                        top = fmaxf(top, sc[r][t][i]);
                    }
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                const float base = top == -INFINITY ? 0.f : top;
                alpha[r] = exp2_fast(m[r] - base);
                m[r] = top;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) sc[r][t][i] = exp2_fast(sc[r][t][i] - base + kUp);
                l[r] = l[r] * alpha[r] + ((sc[r][0][0] + sc[r][0][1]) + (sc[r][1][0] + sc[r][1][1]));
            }

            // ---- weights as the A operand, in parts, times the values; the
            // running sums are fp32 fmas, rounded to nearest
            if constexpr (HALF) {
                uint32_t w1[4], w2[4];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    w1[2 * t] = take_part<Cache>(sc[0][t][0], sc[0][t][1], false);
                    w1[2 * t + 1] = take_part<Cache>(sc[0][t][0], sc[0][t][1], PP == 2);
                    if constexpr (PP == 3) w2[2 * t] = w2[2 * t + 1] = take_part<Cache>(sc[0][t][0], sc[0][t][1], true);
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    uint32_t vf[4];
                    ldsm4t(vf, at + v_lane + d * 32);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        float x[4] = {}, y[4] = {};
                        mma16816<Cache>(x, w1, vf[2 * t], vf[2 * t + 1]);
                        if constexpr (PP == 3) mma16816<Cache>(y, w2, vf[2 * t], vf[2 * t + 1]);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            o[2 * d + t][i] = o[2 * d + t][i] * alpha[0] + add_rest(x[i], PP == 3 ? x[2 + i] + y[i] : x[2 + i]);
                    }
                }
            } else {
                uint32_t wf[PP][4];
#pragma unroll
                for (int s = 0; s < PP; ++s)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        wf[s][x] = take_part<Cache>(sc[x & (R - 1)][x >> 1][0], sc[x & (R - 1)][x >> 1][1], s == PP - 1);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    uint32_t vf[4];
                    ldsm4t(vf, at + v_lane + d * 32);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        float x[4] = {}, y[4] = {};
                        mma16816<Cache>(x, wf[0], vf[2 * t], vf[2 * t + 1]);
#pragma unroll
                        for (int s = 1; s < PP; ++s) mma16816<Cache>(y, wf[s], vf[2 * t], vf[2 * t + 1]);
#pragma unroll
                        for (int i = 0; i < 2 * R; ++i)
                            o[2 * d + t][i] = o[2 * d + t][i] * alpha[i >> 1] + add_rest(x[i], y[i]);
                    }
                }
            }
            stage = stage + 1 == S::kStages ? 0 : stage + 1;
        }

        // ---- the end of the row, or of this warp's part of it; the next row's
        // queries are on their way meanwhile, where there are registers for them
        const Cursor done = cc;
        live = next_row(cc, seqs, p, until);
        if (DP <= 128 && live) fetch_queries(cc);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] += __shfl_xor_sync(~0u, l[r], 1);
            l[r] += __shfl_xor_sync(~0u, l[r], 2);
            if (row_bad) l[r] = __int_as_float(0x7fc00000);
        }
        const bool whole = first_j == 0 && done.end == done.steps;
        float* piece = p.pieces + (size_t)(2 * w + (first_j == 0)) * p.piece_floats;
        if (!whole && first_j == 0 && lane == 0)
            p.cuts[w] = make_int2(done.b * n_rows + done.h, (int)(div_fast(done.row_at + done.steps - 1, part) - w + 1));
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = g + 8 * r;
            if (row >= heads) continue;
            if (whole) {
                const size_t at = (size_t)done.b * p.n_q + first_head + row;
                const bool none = done.len == done.lo;
                const float inv = 1.f / l[r];
                Act* dst = (Act*)p.out + at * p.dim;
#pragma unroll
                for (int t = 0; t < DP / 8; ++t)
                    if (t * 8 < p.dim) {
                        dst[t * 8 + 2 * quad] = sb_from_float<Act>(none ? 0.f : o[t][2 * r] * inv);
                        dst[t * 8 + 2 * quad + 1] = sb_from_float<Act>(none ? 0.f : o[t][2 * r + 1] * inv);
                    }
                if (p.lse && quad == 0)
                    p.lse[at] = none ? -INFINITY : 0.69314718055994531f * (m[r] + (log2f(l[r]) - kUp));
            } else {
                if (quad == 0) *(float2*)(piece + 2 * row) = make_float2(m[r], l[r]);
#pragma unroll
                for (int t = 0; t < DP / 8; ++t)
                    *(float2*)(piece + 32 + row * DP + t * 8 + 2 * quad) = make_float2(o[t][2 * r], o[t][2 * r + 1]);
            }
        }
        if (DP > 128 && live) fetch_queries(cc);
    }
}

// ------------------------------------------------------------ the join
// Pieces of a cut row, in the order of the keys: weights from their m and l,
// then the weighted sum of their rows. A unit is a query head of a cut row and
// 32 of its columns, one per lane. Latency is all there is to it, so a unit is
// joined by one warp where its row has at most 32 pieces and by the eight warps
// of a CTA where it has more, with the pieces' loads in flight together.
constexpr int kJoinWarps = 8, kJoinThreads = kJoinWarps * 32, kMaxWarps = 148 * 2 * 8, kFew = 32;

template <class Act, int DP>
__global__ void __launch_bounds__(kJoinThreads) k_attend_join(const AttendParams p, int n_warps, float up) {
    constexpr int kSlices = DP / 32, kPer = kMaxWarps / kJoinThreads + 1;
    __shared__ short few[kMaxWarps], many[kMaxWarps];   // the warps that begin a cut row
    __shared__ int counts[2][kPer * kJoinWarps];
    __shared__ float red[2][kJoinWarps], sums[kJoinWarps][32];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- the cut rows, in the order of the warps that begin them
    int n_few = 0, n_many = 0;
    {
        const int per = (n_warps + kJoinThreads - 1) / kJoinThreads, chunks = per * kJoinWarps;
        for (int i = 0; i < per; ++i) {
            const int w = i * kJoinThreads + threadIdx.x, n = w < n_warps ? p.cuts[w].y : 0;
            const unsigned f = __ballot_sync(~0u, n > 0 && n <= kFew), y = __ballot_sync(~0u, n > kFew);
            if (lane == 0) counts[0][i * kJoinWarps + wid] = __popc(f), counts[1][i * kJoinWarps + wid] = __popc(y);
        }
        __syncthreads();
        for (int i = 0; i < per; ++i) {
            int at_few = 0, at_many = 0;   // in the chunks before this warp's
            n_few = n_many = 0;
            for (int c = lane; c < chunks; c += 32) {
                n_few += counts[0][c], n_many += counts[1][c];
                if (c < i * kJoinWarps + wid) at_few += counts[0][c], at_many += counts[1][c];
            }
            n_few = __reduce_add_sync(~0u, n_few), n_many = __reduce_add_sync(~0u, n_many);
            at_few = __reduce_add_sync(~0u, at_few), at_many = __reduce_add_sync(~0u, at_many);
            if (n_few + n_many == 0) return;
            const int w = i * kJoinThreads + threadIdx.x, n = w < n_warps ? p.cuts[w].y : 0;
            const unsigned f = __ballot_sync(~0u, n > 0 && n <= kFew), y = __ballot_sync(~0u, n > kFew);
            const unsigned before = (1u << lane) - 1;
            if (f >> lane & 1) few[at_few + __popc(f & before)] = (short)w;
            if (y >> lane & 1) many[at_many + __popc(y & before)] = (short)w;
        }
        __syncthreads();
    }
    const int n_rows = p.n_kv * p.tiles, units = p.piece_rows * kSlices;
    auto place = [&](int row, int head, bool& real) -> size_t {   // of the output row
        const int b = row / n_rows, h = row % n_rows, tile = h % p.tiles;
        real = head < min(16, p.group - tile * 16);
        return (size_t)b * p.n_q + h / p.tiles * p.group + tile * 16 + head;
    };
    auto piece = [&](int w, int k) { return p.pieces + (size_t)(2 * (w + k) + (k == 0)) * p.piece_floats; };
    auto finish = [&](size_t at, int col, float a, float top, float l) {
        if (col < p.dim) ((Act*)p.out)[at * p.dim + col] = sb_from_float<Act>(a / l);
        if (p.lse && col == 0) p.lse[at] = 0.69314718055994531f * (top + (log2f(l) - up));
    };

    // ---- rows of more than kFew pieces
    for (int u = blockIdx.x; u < n_many * units; u += gridDim.x) {
        const int w = many[u / units], head = u / kSlices % p.piece_rows, col = u % kSlices * 32 + lane;
        const int2 cut = p.cuts[w];
        const int n = cut.y;
        bool real;
        const size_t at = place(cut.x, head, real);
        if (!real) continue;
        // this warp's pieces: wid, wid + 8, ..; 32 at a time, one per lane
        float top = -INFINITY, l = 0.f, a = 0.f;
        for (int k0 = wid; k0 < n; k0 += kJoinThreads) {
            const int k = k0 + lane * kJoinWarps;
            const float2 ml = k < n ? *(const float2*)(piece(w, k) + 2 * head) : make_float2(-INFINITY, 0.f);
            float t = fmaxf(top, ml.x);
#pragma unroll
            for (int s = 16; s; s >>= 1) t = fmaxf(t, __shfl_xor_sync(~0u, t, s));
            const float base = t == -INFINITY ? 0.f : t, old = exp2_fast(top - base), f = exp2_fast(ml.x - base);
            top = t;
            l = l * old + f * ml.y;   // of this lane's pieces
            a *= old;
            const int here = min(32, (n - k0 + kJoinWarps - 1) / kJoinWarps);
#pragma unroll 16
            for (int i = 0; i < here; ++i)
                a += __shfl_sync(~0u, f, i) * piece(w, k0 + i * kJoinWarps)[32 + head * DP + col];
        }
#pragma unroll
        for (int s = 16; s; s >>= 1) l += __shfl_xor_sync(~0u, l, s);
        if (lane == 0) red[0][wid] = top, red[1][wid] = l;
        sums[wid][lane] = a;
        __syncthreads();
        if (wid == 0) {
            top = red[0][0];
            for (int i = 1; i < kJoinWarps; ++i) top = fmaxf(top, red[0][i]);
            const float base = top == -INFINITY ? 0.f : top;
            a = l = 0.f;
            for (int i = 0; i < kJoinWarps; ++i) {
                const float f = exp2_fast(red[0][i] - base);
                l += f * red[1][i];
                a += f * sums[i][lane];
            }
            finish(at, col, a, top, l);
        }
        __syncthreads();
    }

    // ---- the others
    for (int u = blockIdx.x * kJoinWarps + wid; u < n_few * units; u += gridDim.x * kJoinWarps) {
        const int w = few[u / units], head = u / kSlices % p.piece_rows, col = u % kSlices * 32 + lane;
        const int2 cut = p.cuts[w];
        const int n = cut.y;
        bool real;
        const size_t at = place(cut.x, head, real);
        if (!real) continue;
        const float2 ml = lane < n ? *(const float2*)(piece(w, lane) + 2 * head) : make_float2(-INFINITY, 0.f);
        float top = ml.x;
#pragma unroll
        for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, s));
        const float f = exp2_fast(ml.x - (top == -INFINITY ? 0.f : top));
        float l = lane < n ? f * ml.y : 0.f, a = 0.f;
#pragma unroll
        for (int s = 16; s; s >>= 1) l += __shfl_xor_sync(~0u, l, s);
#pragma unroll 16
        for (int k = 0; k < n; ++k) a += __shfl_sync(~0u, f, k) * piece(w, k)[32 + head * DP + col];
        finish(at, col, a, top, l);
    }
}

// ------------------------------------------------------------ launches
int sm_count() {
    static int sms = 0;
    if (!sms) {
        int dev = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        if (sms < 1) sms = 148;
        sms = std::min(sms, kMaxWarps / 8);
    }
    return sms;
}
int tile_width(int dim) { return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256; }
size_t cuts_bytes() { return ((size_t)sm_count() * 8 * sizeof(int2) + 255) / 256 * 256; }
int piece_floats(int group, int dim) { return 32 + std::min(group, 16) * tile_width(dim); }

template <class Cache, int DP, int QP, bool HALF>
int launch(AttendParams p, cudaStream_t st) {
    using S = Shape<DP>;
    using Act = typename std::conditional<QP == 1, Cache, float>::type;
    const int rows = std::min(p.group, 16);
    const size_t per_warp = S::kStages * S::kStage + (HALF ? 0 : (size_t)rows * QP * S::kRow);
    const size_t head = (12 * (size_t)p.n_seqs + 8 + 15) / 16 * 16;
    // static shared memory (the scan's warp sums) is 256 bytes
    const int warps = (int)std::min<size_t>(S::kWarps, (kSmemLimit - 512 - head) / per_warp);
    const size_t bytes = head + warps * per_warp;
    static bool opted = false;
    if (!opted) {
        if (!sb_cuda_ok(cudaFuncSetAttribute(k_attend<Cache, DP, QP, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kSmemLimit - 512), "attend shared memory"))
            return -1;
        opted = true;
    }
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = sm_count();
    cfg.blockDim = warps * 32;
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (!sb_cuda_ok(cudaLaunchKernelEx(&cfg, k_attend<Cache, DP, QP, HALF>, (const AttendParams)p), "attend launch")) return -1;
    const long long longest = std::min((long long)p.table_width * p.page_size,
                                       p.window > 0 ? p.window + kStep - 1ll : 1ll << 40);
    if (longest <= kWhole * kStep) return 0;   // no row can be cut
    const int n_warps = sm_count() * warps;
    cfg.gridDim = 2 * sm_count();
    cfg.blockDim = kJoinThreads;
    cfg.dynamicSmemBytes = 0;
    const float up = std::is_same<Cache, __half>::value ? 12.f : 0.f;
    return sb_cuda_ok(cudaLaunchKernelEx(&cfg, k_attend_join<Act, DP>, (const AttendParams)p, n_warps, up), "attend join launch")
               ? 0 : -1;
}

template <class Cache, int QP, bool HALF>
int launch_dim(const AttendParams& p, cudaStream_t st) {
    switch (tile_width(p.dim)) {
    case 64: return launch<Cache, 64, QP, HALF>(p, st);
    case 96: return launch<Cache, 96, QP, HALF>(p, st);
    case 128: return launch<Cache, 128, QP, HALF>(p, st);
    case 192: return launch<Cache, 192, QP, HALF>(p, st);
    default: return launch<Cache, 256, QP, HALF>(p, st);
    }
}
template <class Cache, int QP>
int launch_group(const AttendParams& p, cudaStream_t st) {
    return p.group <= 8 ? launch_dim<Cache, QP, true>(p, st) : launch_dim<Cache, QP, false>(p, st);
}

}  // namespace

SABAH_API size_t sabah_attend_paged_workspace(int n_q_heads, int n_kv_heads, int head_dim) {
    if (n_kv_heads <= 0 || n_q_heads <= 0 || head_dim <= 0 || head_dim > kMaxDim) return 0;
    return cuts_bytes() + (size_t)sm_count() * 8 * 2 * piece_floats(n_q_heads / n_kv_heads, head_dim) * sizeof(float);
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
    p.q_pairs = ((uintptr_t)d_q | q_seq_stride | q_head_stride) % (2 * ab) == 0;
    p.k = (const uint8_t*)d_k_cache, p.v = (const uint8_t*)d_v_cache;
    p.k_page = k_page_stride, p.k_slot = k_slot_stride, p.k_head = k_head_stride;
    p.v_page = v_page_stride, p.v_slot = v_slot_stride, p.v_head = v_head_stride;
    p.n_pages = n_pages, p.page_size = page_size;
    p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
    p.table = d_block_table, p.table_stride = table_stride / 4, p.table_width = table_width;
    p.lens = d_lens, p.n_seqs = n_seqs, p.n_q = n_q_heads, p.n_kv = n_kv_heads, p.dim = head_dim, p.window = window;
    p.scale_log2 = scale * 1.44269504088896341f;
    p.out = (uint8_t*)d_out, p.lse = d_lse, p.err = err;
    if (!d_workspace || (uintptr_t)d_workspace % 16 ||
        workspace_bytes < sabah_attend_paged_workspace(n_q_heads, n_kv_heads, head_dim)) {
        sb_set_error("attend workspace of %zu bytes: %zu, 16-byte aligned, are needed", workspace_bytes,
                     sabah_attend_paged_workspace(n_q_heads, n_kv_heads, head_dim));
        return -1;
    }
    p.group = n_q_heads / n_kv_heads;
    p.tiles = (p.group + 15) / 16;
    p.piece_rows = std::min(p.group, 16);
    p.piece_floats = piece_floats(p.group, head_dim);
    p.cuts = (int2*)d_workspace;
    p.pieces = (float*)((uint8_t*)d_workspace + cuts_bytes());
    const int slot = sb_timing_begin("attend_paged", st);
    int rc = 0;
    for (int b = 0; b < n_seqs && rc == 0; b += kMaxSeqs) {
        AttendParams a = p;
        a.n_seqs = std::min(kMaxSeqs, n_seqs - b);
        a.q += (size_t)b * q_seq_stride;
        a.table += (size_t)b * p.table_stride;
        a.lens += b;
        a.out += (size_t)b * n_q_heads * head_dim * ab;
        if (a.lse) a.lse += (size_t)b * n_q_heads;
        if (act_type == SB_F32)
            rc = cache_type == SB_F16 ? launch_group<__half, 2>(a, st) : launch_group<__nv_bfloat16, 3>(a, st);
        else
            rc = cache_type == SB_F16 ? launch_group<__half, 1>(a, st) : launch_group<__nv_bfloat16, 1>(a, st);
    }
    sb_timing_end(slot, st);
    return rc;
}
