// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale * <q, k_j>,  lo <= j < len,  lo = window ? max(0, len - window) : 0
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  lse = m + ln sum_j exp(s_j - m)
//
// Key j of sequence b is row j % page_size of page block_table[b][j / page_size].
// A sequence of length zero gives zeros and lse = -inf. Nothing outside
// [lo, len) counts, and no table entry outside it is read.
//
// Bound: DRAM, every key and value row once. A key-value head's query heads
// (up to 16) are taken together, so the rows are read once for all of them. The
// arithmetic is mma.sync with keys (then value columns) as the 16 rows of the
// tile and 8 query heads as its columns, a fraction of the tensor rate and under
// the time the rows take to arrive: with the heads as rows half the tile or more
// would be padding, and tcgen05's 128 rows would be 87-99% of it.
//
// The work is a list of steps of 32 keys over all (sequence, key-value head)
// rows, cut into equal parts, one per warp, whatever the lengths: one long
// sequence spreads over the whole chip, and many short ones stay whole within a
// warp. Warps never wait for one another; each streams its own keys and values
// through its own ring in shared memory, filled by TMA: boxes of as many rows as
// divide both a page and 16, in tiles of 64 columns in the 128-byte swizzle that
// lets ldmatrix meet no bank twice; one box has all tiles of 16 rows where whole
// tiles make up a row. Rows of a box past the window's ends are masked (keys) or
// zeroed (values), so that nothing they hold counts. A row of the list that ends
// in another part is left as (m, l, unnormalised out) in the workspace, and a
// second, small launch (a programmatic dependent of the first) joins the pieces
// of each cut row in the order of its keys. Rows of at most kWhole steps are
// never cut; where the block table cannot hold a longer sequence the second
// launch is left out. (Smaller last parts, taken by the warps that finish first,
// measured slower: 106 us against 98 on 64 ragged sequences of to 8192 keys,
// 8 key-value heads of 128: a part's start and end cost more than the waiting.)
//
// Precision: scores, m, l and out are fp32. The MMA takes 16-bit factors, so
// fp32 queries and the softmax weights are split into a sum of 16-bit parts
// (f16: 2 parts, 22 bits; bf16: 3 parts, 24 bits), each multiplied exactly.
// With 16-bit outputs the weights take two parts, which leaves the output's own
// rounding as the only one. f16 parts keep their bits only in f16's normal
// range: a query row is scaled to below 2 by a power of two, and the weights
// are computed times 2^11. The reference m of a running sum moves only when a
// score exceeds it by 2^4, which leaves most steps without a rescaling. The
// MMA's accumulation cuts off instead of rounding (measured: 1 + 1.75 * 2^-24
// gives 1), half a unit per step and always toward zero, so its sums are added
// to rounded fp32 sums every kFold steps.
//
// Measured (one B200, the inputs in turn larger than L2): 131,071 keys of one
// sequence, 2 heads of 256, bf16: 59 us, 4.5 TB/s, of which about 7 us pass before
// the first keys arrive and 6 in the join; 64 sequences of 128-8192 keys, 8
// heads of 128, f16 with fp32 queries: 99 us, 5.1 TB/s (the steady part 7.2); 256
// of 16-512 keys, 8 heads of 64: 29 us, 2.5 TB/s; 37 keys: 9.6 us. The start is
// a chain of dependent reads (lengths, block table, rows) and code that runs for
// the first time; what bounds the long calls is DRAM.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cstdlib>

#include "sb_act.cuh"
#include "sb_kernels.h"
#include "sb_split.cuh"

namespace {

constexpr int kMaxDim = 256;
constexpr int kMaxSeqs = 1024;   // per launch: the scan of the lengths sits in shared memory
// What the split is made of, each measured against its neighbours on one kernel, us a
// call in a graph. S: 256 sequences of 16-512 keys, 8 heads of 64, f16; L: the same
// lengths, 16 over 2 heads of 256, bf16; M: 64 of 64-2048, 32 over 8 of 128, f32 over bf16.
constexpr int kStep = 32;        // keys per step
constexpr int kWhole = 3;        // rows of at most this many steps are never cut (S 27.5, L 30.8, M 39.8; 2: 27.4, 28.7, 38.8; 4: 29.0, 31.1, 40.3; 8: 33.9, 35.9, 46.1)
constexpr int kMinSteps = 1;     // and a part is at least this long (1000 keys, 16 over 2 heads of 128: 13.8; 2: 14.3, 4: 16.8)
constexpr int kRowCost = 2;      // what a row costs besides its steps, in steps (S 27.5, L 30.8, M 39.8; 1: 29.1, 34.1, 42.1; 3: 29.5, 30.2, 39.4)
constexpr int kMaxWarps = 148 * 8;
constexpr int kSmemLimit = 227 * 1024;
constexpr float kLazy = 4.f;     // how far, in powers of two, a score may exceed the reference

struct AttendParams {
    const uint8_t* q;
    size_t q_seq, q_head;   // bytes
    int q_pairs;            // pairs of query values are aligned
    const uint8_t *k, *v;
    size_t k_page, k_slot, k_head, v_page, v_slot, v_head;   // bytes
    int n_pages, page_size, page_shift;   // shift: log2(page_size), or -1
    int box;                // rows of a TMA box: a power of two to 16 that divides the page
    int box_tiles;          // its tiles of 64 columns: all of a row's, or one
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
    uint16_t* cut_pieces;   // per warp: the pieces of the row that is cut at its part's end (0: none)
    int* cut_row;           // and which row
    float* pieces;          // per warp two: the row it enters in the middle of, the row it leaves early
    float* sums;            // per warp one: its rounded sums, where registers have no room for them
    int piece_floats, piece_rows;
    int stalled;            // test only (SABAH_TEST_ATTEND_STALL): the warp whose first wait nothing ends; -1: none
};

// ------------------------------------------------------------ PTX helpers
__device__ inline uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ inline void bar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ inline void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ inline void bar_expect_more(uint32_t bar, uint32_t bytes) {   // without arriving
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Bounded: false after 2^24 tries, under a second.
__device__ inline bool bar_wait(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < 1 << 24; ++i) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
    }
    return false;
}
// The rows pass through L2 once: they are the first to go there, so that the
// pieces, the tables and the queries stay.
__device__ inline unsigned long long pass_through() {
    unsigned long long policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ inline void tile_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int col, int slot, int head, int page,
                                 unsigned long long policy) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cta.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
                 "[%0], [%1, {%3, %4, %8, %5, %6}], [%2], %7;" ::"r"(dst), "l"(map), "r"(bar), "r"(col), "r"(slot), "r"(head),
                 "r"(page), "l"(policy), "r"(0) : "memory");
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
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ inline float exp2_fast(float x) {   // 2 ulp, less than the rounding of a score; exp2(-inf) = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// the next 16-bit part of (a, b), which keep what it leaves
template <class T>
__device__ inline uint32_t take_part(float& a, float& b) {
    uint32_t u;
    if constexpr (std::is_same<T, __half>::value) {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(b), "f"(a));
        const float2 f = __half22float2(*(const __half2*)&u);
        a -= f.x, b -= f.y;
    } else {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(b), "f"(a));
        a -= __uint_as_float(u << 16), b -= __uint_as_float(u & 0xffff0000u);
    }
    return u;
}
// e with 2^e <= x < 2^(e + 1); 0 for zero, infinity and NaN
__device__ inline int exponent(float x) {
    return x > 0.f && x < INFINITY ? min(max((__float_as_int(x) >> 23) - 127, -126), 126) : 0;
}
__device__ inline float power_of_two(int e) { return __int_as_float((127 + e) << 23); }
__device__ inline bool is_finite(float x) { return fabsf(x) <= 3.402823466e38f; }
// the reference that a score or another reference is taken relative to
__device__ inline float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

// ------------------------------------------------------------ shapes
// DP: head size rounded up to a tile width. A slot of a ring is the keys or the
// values of a step: twice kTiles tiles of 16 rows x 64 columns (128 swizzled bytes).
// As many slots as shared memory has, in as few rings as hide a warp's own
// latency (131,071 keys of 256: 4 rings of 3 slots 57.9 us, 6 of 2 59.9).
template <int DP>
struct Shape {
    static constexpr int kTiles = (DP + 63) / 64;
    static constexpr int kTileBytes = 16 * 128, kHalf = kTiles * kTileBytes, kSlot = 2 * kHalf;
    static constexpr int kSlots = DP <= 64 ? 6 : 3;
    static constexpr int kWarps = DP <= 128 ? 8 : DP <= 192 ? 5 : 4;
};
constexpr float up_of(bool f16) { return f16 ? 11.f : 0.f; }

// ------------------------------------------------------------ the list of steps
// The scan of the lengths: cost of the sequences before b, for one row of each.
// A row takes its steps, then kRowCost idle places in the list, so that parts
// of many short rows and parts of one long row take as long.
struct Seqs {
    int* pre;         // [n_seqs + 1]
    int* len;         // [n_seqs], -1 where out of range
};
__device__ inline int window_start(int len, int window) { return window > 0 ? max(0, len - window) : 0; }
__device__ inline int seq_steps(int len, int window) {
    return len <= 0 ? 1 : (len + kStep - 1) / kStep - window_start(len, window) / kStep;
}
// A place in the list; each warp has one that loads and one that computes.
struct Cursor {
    int b, h;            // sequence, row of it (key-value head and tile)
    int j, end, steps;   // step in the row, where the part leaves it, the row's steps
    int len, lo;
    int row_at, until;   // the row's first place in the list, the part's end
};
// starts the row at c.b, c.h, from its step j on
__device__ inline void enter_row(Cursor& c, const Seqs& s, const AttendParams& p, int j) {
    c.len = s.len[c.b];
    c.lo = window_start(max(c.len, 0), p.window);
    c.steps = s.pre[c.b + 1] - s.pre[c.b] - kRowCost;
    c.j = j;
    c.end = c.steps <= kWhole ? c.steps : min(c.steps, c.until - c.row_at);
}
// false at the end of the part
__device__ inline bool next_row(Cursor& c, const Seqs& s, const AttendParams& p) {
    c.row_at += c.steps + kRowCost;
    if (c.row_at >= c.until) return false;
    if (++c.h == p.n_kv * p.tiles) {
        c.h = 0;
        if (++c.b == p.n_seqs) return false;
    }
    enter_row(c, s, p, 0);
    return true;
}
// the first step of the part [from, until); b = -1 where it has none of its own
__device__ inline Cursor enter_part(const Seqs& s, const AttendParams& p, int from, int until, int lane) {
    const int n_rows = p.n_kv * p.tiles;
    Cursor c;
    c.until = until;
    int a = 0, span = p.n_seqs;   // the last sequence that starts at or before `from` is in [a, a + span)
    while (span > 1) {            // 32 probes at a time
        const int hop = (span + 31) / 32, at = a + lane * hop;
        const unsigned hit = __ballot_sync(~0u, at < a + span && s.pre[min(at, p.n_seqs)] * n_rows <= from);
        const int last = 31 - __clz(hit);
        span = min(hop, span - last * hop);
        a += last * hop;
    }
    c.b = a;
    const int at = from - s.pre[a] * n_rows, cost = s.pre[a + 1] - s.pre[a];
    c.h = div_fast(at, cost);
    const int j = at - c.h * cost;
    c.row_at = from - j;
    enter_row(c, s, p, j);
    // a whole row is its first step's part's; past a row's steps are its idle places
    if (!(j < c.steps && (c.steps > kWhole || j == 0)) && !next_row(c, s, p)) c.b = -1;
    return c;
}

// ------------------------------------------------------------ the loading side
// One warp's loads into its ring: every slot is filled again as soon as it has
// been read. Block table entries are held 32 to a register, one per lane, and
// the register after the current one is always on its way, as are the first
// entries of this sequence (the next key-value head starts there again) and of
// the next.
template <int DP>
struct Loader {
    using S = Shape<DP>;
    const AttendParams& p;
    const CUtensorMap *kmap, *vmap;
    const Seqs& seqs;
    const int lane;
    const uint32_t ring, bars;
    const unsigned long long policy;
    Cursor c;
    bool more = true, values = false;   // values: the next slot is the step's values
    uint32_t bad = 0, dirty = 0;        // bits per slot: the step met a page out of range; zeros were stored to it
    int first, cur, next, start, ahead; // cur: table entries first ..; next: the 32 after them
    int page = -1, row = 0;             // lane i: where box i of the step lies; page -1: it is not loaded

    __device__ Loader(const AttendParams& p_, const CUtensorMap* km, const CUtensorMap* vm, const Seqs& s_, int lane_,
                      uint32_t ring_, uint32_t bars_, const Cursor& c_)
        : p(p_), kmap(km), vmap(vm), seqs(s_), lane(lane_), ring(ring_), bars(bars_), policy(pass_through()), c(c_) {
        first = entry_of((c.lo / kStep + c.j) * kStep);
        cur = entries(c.b, first);
        next = entries(c.b, first + 32);
        start = first_entries(c.b);
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
    __device__ void advance() {
        if (++c.j < c.end) return;
        const int b = c.b;
        more = next_row(c, seqs, p);
        if (!more) return;
        if (c.b != b) {
            start = ahead;
            ahead = c.b + 1 < p.n_seqs ? first_entries(c.b + 1) : -1;
        }
        first = entry_of(c.lo / kStep * kStep);
        cur = start;
        next = entries(c.b, first + 32);
    }
    // fills a slot with the next keys or values
    __device__ void issue(int slot) {
        if (!more) return;
        if (!values) {
            const int key0 = (c.lo / kStep + c.j) * kStep, key = key0 + lane * p.box;
            if (entry_of(key0) >= first + 32) {
                first += 32;
                cur = next;
                next = entries(c.b, first + 32);
            }
            const int e = entry_of(key), at = e - first;   // a step has at most 32 entries: at < 64
            const int x = __shfl_sync(~0u, cur, at), y = __shfl_sync(~0u, next, at);
            page = at < 32 ? x : y;
            row = key - e * p.page_size;
            const bool in = lane * p.box < kStep && key < c.len && key + p.box > c.lo;
            const bool out = in && (page < 0 || page >= p.n_pages);
            if (!in || out) page = -1;
            bad &= ~(1u << slot);
            if (__any_sync(~0u, out)) {
                bad |= 1u << slot;
                if (lane == 0) atomicExch(p.err, SB_DERR_BAD_INDEX);
            }
        }
        if (dirty >> slot & 1) {   // order the zeros before the TMA's writes
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            dirty &= ~(1u << slot);
        }
        const int first_row = lane * p.box;
        const uint32_t bar = bars + slot * 8, dst = ring + slot * S::kSlot + first_row / 16 * S::kHalf + first_row % 16 * 128;
        const unsigned boxes = __popc(__ballot_sync(~0u, page >= 0));
        if (lane == 0) bar_expect(bar, boxes * p.box * (128 * S::kTiles));
        if (page >= 0) {
            const CUtensorMap* map = values ? vmap : kmap;
            const int kv = p.tiles == 1 ? c.h : c.h / p.tiles;
#pragma unroll 1
            for (int t = 0; t < S::kTiles; t += p.box_tiles)
                tile_load(dst + t * S::kTileBytes, map, bar, 64 * t, row, kv, page, policy);
        }
        if (values) advance();
        values = !values;
    }
};

// ------------------------------------------------------------ pieces
// m and l of each head, then the running sums as the lanes hold them: for 8
// heads and 16 columns a float4 per lane, of (column, head) = (lane / 4, 2 (lane
// % 4)), the next head, and both at column + 8.
constexpr int kPieceHead = 32;
// the row c, which part w begins and does not end, for the join
__device__ inline void cut(const AttendParams& p, const Cursor& c, int w, int part) {
    p.cut_row[w] = c.b * p.n_kv * p.tiles + c.h;
    p.cut_pieces[w] = (uint16_t)(div_fast(c.row_at + c.steps - 1, part) - w + 1);
}
__host__ __device__ inline int frag_at(int head, int col, int dp) {
    const int lane = col % 8 * 4 + head % 8 / 2;
    return ((head / 8 * (dp / 16) + col / 16) * 32 + lane) * 4 + col % 16 / 8 * 2 + head % 2;
}

// ------------------------------------------------------------ infinities
// Products of parts make NaN of what is an infinity in the formula (0 * inf,
// inf - inf between parts). Where a row's result is not finite, its columns that
// are not are computed again here, key by key in fp32, for this warp's keys
// [from, to); all of them where the softmax's own sum is not finite. A score of
// -inf weighs nothing, also where no finite one came before it; a NaN stays one,
// whatever the weights that follow.
template <class Cache, class Act>
__device__ __noinline__ void redo_row(const AttendParams& p, int b, int kv, int head, int from, int to, float m, float l,
                                      float up, bool whole, float* piece, int row, int dp, int lane) {
    constexpr int N = kMaxDim / 32;
    const Act* q = (const Act*)(p.q + b * p.q_seq + head * p.q_head);
    float o[N] = {}, top = -INFINITY, sum = 0.f;
    for (int j = from; j < to; ++j) {
        const int page = p.table[b * p.table_stride + j / p.page_size];
        if (page < 0 || page >= p.n_pages) return;   // NaN, as it is
        const Cache* k = (const Cache*)(p.k + page * p.k_page + (j % p.page_size) * p.k_slot + kv * p.k_head);
        const Cache* v = (const Cache*)(p.v + page * p.v_page + (j % p.page_size) * p.v_slot + kv * p.v_head);
        float s = 0.f;
        for (int i = 0; i < N; ++i)
            if (lane + 32 * i < p.dim) s += sb_to_float(q[lane + 32 * i]) * sb_to_float(k[lane + 32 * i]);
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
        s *= p.scale_log2;
        const float t = fmaxf(top, s), a = top == -INFINITY ? 1.f : exp2f(top - t), e = exp2f(s - finite_or_zero(t));
        top = t;
        sum = sum * a + e;
        for (int i = 0; i < N; ++i)
            if (lane + 32 * i < p.dim) o[i] = o[i] * a + e * sb_to_float(v[lane + 32 * i]);
    }
    const bool all = !is_finite(l);
    const size_t at = (size_t)b * p.n_q + head;
    Act* out = (Act*)p.out + at * p.dim;
    const float scale = all ? exp2f(up) : exp2f(finite_or_zero(top) - finite_or_zero(m) + up);
    for (int i = 0; i < N; ++i) {
        const int d = lane + 32 * i;
        if (d >= p.dim) break;
        if (whole) {
            if (all || !is_finite(sb_to_float(out[d]))) out[d] = sb_from_float<Act>(o[i] / sum);
        } else {
            float* x = piece + kPieceHead + frag_at(row, d, dp);
            if (all || !is_finite(*x)) *x = o[i] * scale;
        }
    }
    if (all && lane == 0) {
        if (!whole)
            piece[2 * row] = top, piece[2 * row + 1] = sum * scale;
        else if (p.lse)
            p.lse[at] = 0.69314718055994531f * (top + log2f(sum));
    }
}

// ------------------------------------------------------------ giving up
// A wait that never ends: the error word, then the loads in flight get their time
// (`left` of this row's are still to be used, and the ring has no more than its
// slots), and what this warp still owes becomes NaN: whole rows, and the sums of
// pieces, which the join carries on to their rows.
template <class Act>
__device__ __noinline__ void give_up(const AttendParams& p, const Seqs& seqs, Cursor c, int first_j, int left, uint32_t bars,
                                     int slot, uint32_t parity, int slots) {
    // found anew, so that the kernel keeps nothing for a call that it hardly ever makes
    const int lane = threadIdx.x & 31, n_warps = blockDim.x >> 5, w = (threadIdx.x >> 5) * gridDim.x + blockIdx.x;
    const int part = part_of(seqs.pre[p.n_seqs] * p.n_kv * p.tiles, gridDim.x * n_warps, kMinSteps);
    const float nan = __int_as_float(0x7fc00000);
    if (lane == 0) atomicExch(p.err, SB_DERR_TIMEOUT);
    int ahead = left;
    for (Cursor x = c; ahead < slots && next_row(x, seqs, p);) ahead += 2 * (x.end - x.j);
    for (int i = 0; i < min(ahead, slots); ++i) bar_wait(bars + (slot + i) % slots * 8, parity ^ (slot + i >= slots));
    for (bool live = true; live; live = next_row(c, seqs, p), first_j = 0) {
        const int tile = c.h % p.tiles, head0 = c.h / p.tiles * p.group + tile * 16, heads = min(16, p.group - tile * 16);
        if (first_j == 0 && c.end == c.steps) {
            const size_t at = (size_t)c.b * p.n_q + head0;
            for (int i = lane; i < heads * p.dim; i += 32) ((Act*)p.out)[at * p.dim + i] = sb_from_float<Act>(nan);
            if (p.lse && lane < heads) p.lse[at + lane] = nan;
            continue;
        }
        if (lane < heads) *(float2*)(p.pieces + (size_t)(2 * w + (first_j == 0)) * p.piece_floats + 2 * lane) = make_float2(0.f, nan);
        if (first_j == 0 && lane == 0) cut(p, c, w, part);
    }
}

// ------------------------------------------------------------ the kernel
// QP: parts of a query value (1: it has the cache's type); the weights take as
// many, and at least two. NT: tiles of 8 query heads. With one, the query
// fragments stay in registers; with two they are read from shared memory.
template <class Cache, int DP, int QP, int NT>
__global__ void __launch_bounds__(Shape<DP>::kWarps * 32, 1)
    k_attend(const __grid_constant__ AttendParams p, const __grid_constant__ CUtensorMap kmap,
             const __grid_constant__ CUtensorMap vmap) {
    using S = Shape<DP>;
    using Act = typename std::conditional<QP == 1, Cache, float>::type;
    constexpr int PP = QP == 1 ? 2 : QP;
    constexpr int ND = DP / 16;
    constexpr float kUp = up_of(std::is_same<Cache, __half>::value);
    // rounded sums stay in registers where there is room for them
    constexpr bool kKeep = ND * (8 * NT + (NT == 1 ? 2 * QP : 0)) <= 160;
    // A cut-off loses up to 2^-23 of the running sum, 2 PP of them a step: before a fold
    // 48 at most with fp32 outputs (6e-6; three parts), 128 with 16-bit ones (1.5e-5,
    // under a tenth of f16's half unit). More folds cost time, one is 4 ND NT adds a lane.
    constexpr int kFold = QP == 1 ? 32 : 8;
    constexpr int kQRow = DP * 2 + 16;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
    const int rows = min(p.group, 16), q_rows = NT == 1 ? 0 : rows * QP;
    uint8_t* q_mem = smem + n_warps * S::kSlots * S::kSlot + wid * q_rows * kQRow;
    uint8_t* tail = smem + n_warps * (S::kSlots * S::kSlot + q_rows * kQRow);
    const uint32_t bars = smem_addr(tail) + wid * S::kSlots * 8;
    tail += n_warps * S::kSlots * 8;
    Seqs seqs{(int*)tail, (int*)tail + p.n_seqs + 1};

    if (lane < S::kSlots) bar_init(bars + lane * 8, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (threadIdx.x == 0 && p.n_pages > 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // ---- the scan of the lengths
    __shared__ int warp_sum[32];
    {
        const int per = (p.n_seqs + blockDim.x - 1) / blockDim.x, b0 = threadIdx.x * per;
        int sum = 0;
        for (int b = b0; b < min(b0 + per, p.n_seqs); ++b) {
            int len = p.lens[b];
            if (len < 0 || len > (long long)p.table_width * p.page_size) {
                len = -1;
                if (blockIdx.x == 0) atomicExch(p.err, SB_DERR_BAD_INDEX);
            }
            seqs.len[b] = len;
            sum += seq_steps(len, p.window) + kRowCost;
        }
        int run = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(~0u, run, o);
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

    // ---- this warp's own part; neighbours in the list sit on different SMs
    const int w = wid * gridDim.x + blockIdx.x, n_rows = p.n_kv * p.tiles;
    const int cost = seqs.pre[p.n_seqs] * n_rows, all_warps = gridDim.x * n_warps;
    const int part = part_of(cost, all_warps, kMinSteps);
    if (lane == 0) p.cut_pieces[w] = 0;
    if (w >= parts_in(cost, part)) return;
    Cursor cc = enter_part(seqs, p, w * part, part_end(cost, part, w), lane);
    if (cc.b < 0) return;

    // ---- table entries and queries on their way, then keys and values
    const int g = lane >> 2, quad = lane & 3;
    Act qx[NT == 1 ? ND : 1][4];   // the row's query values 16 d + 2 quad + {0, 1, 8, 9}, as they are
    auto fetch_queries = [&](const Cursor& c) {
        if constexpr (NT == 1) {
            const Act* src = (const Act*)(p.q + c.b * p.q_seq + (c.h * p.group + min(g, p.group - 1)) * p.q_head);
            if (p.q_pairs) {
                struct alignas(2 * sizeof(Act)) Pair { Act a, b; };
                const bool full = p.dim == DP;   // then every offset is a constant
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int at = 16 * d + i * 8;
                        const Pair u = *(const Pair*)(src + 2 * quad + (full || at < p.dim ? at : 0));
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
    uint8_t* ring_mem = smem + wid * S::kSlots * S::kSlot;
    const uint32_t ring = smem_addr(ring_mem);
    if (w == p.stalled && lane == 0) bar_expect_more(bars, 16);   // test only: bytes that no load brings
    Loader<DP> loader(p, &kmap, &vmap, seqs, lane, ring, bars, cc);
    fetch_queries(cc);
#pragma unroll 1
    for (int i = 0; i < S::kSlots; ++i) loader.issue(i);

    // ---- the computing side. A lane's columns are heads 8 u + 2 quad and the
    // next; of a 16-row tile it holds rows g and g + 8.
    float acc[NT][ND][4];                          // the MMA's sums: 16 columns of the values x 8 heads
    float o[kKeep ? NT : 1][kKeep ? ND : 1][4];    // the rounded ones
    float m[2 * NT], l[2 * NT], l_sum[2 * NT], unscale[2 * NT], m_fold[2 * NT];
    uint32_t qf[NT == 1 ? ND : 1][2 * QP];         // per 16 dimensions the parts of both 8s, as the B operand
    uint32_t wf[2][NT][PP][2];                     // the weights as the B operand, per 16 keys and part
    const int k_row = ((lane >> 3) & 1) * 8 + (lane & 7), v_row = (lane >> 4) * 8 + (lane & 7);
    const uint32_t k_lane = k_row * 128 + (((lane >> 4) ^ (k_row & 7)) << 4);
    const uint32_t v_lane = v_row * 128 + ((((lane >> 3) & 1) ^ (v_row & 7)) << 4);
    float* sums = p.sums + (size_t)w * p.piece_floats;
    int slot = 0;
    uint32_t parity = 0;
    for (bool live = true; live;) {
        const int tile = p.tiles == 1 ? 0 : cc.h % p.tiles, kv = p.tiles == 1 ? cc.h : cc.h / p.tiles;
        const int first_head = kv * p.group + tile * 16, heads = min(16, p.group - tile * 16);

        // ---- this row's queries, split into parts
#pragma unroll
        for (int c = 0; c < 2 * NT; ++c) unscale[c] = p.scale_log2;
        if constexpr (NT == 1) {   // of head g
            // values past the head size are zero
            auto value = [&](int d, int i) {
                return 16 * d + 2 * quad + (i >> 1) * 8 < p.dim ? sb_to_float(qx[d][i]) : 0.f;
            };
            float down = 1.f;
            if constexpr (QP > 1) {
                float top = 0.f;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(value(d, i)));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                const int e = exponent(top);
                down = power_of_two(-e);
#pragma unroll
                for (int c = 0; c < 2; ++c) unscale[c] *= power_of_two(__shfl_sync(~0u, e, 4 * (2 * quad + c)));
            }
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float a = value(d, 2 * i) * down, b = value(d, 2 * i + 1) * down;
#pragma unroll
                    for (int s = 0; s < QP; ++s) qf[d][i * QP + s] = take_part<Cache>(a, b);
                }
        } else {
            __syncwarp();
            for (int r = 0; r < heads; ++r) {
                const Act* src = (const Act*)(p.q + cc.b * p.q_seq + (first_head + r) * p.q_head);
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
#pragma unroll
                    for (int c = 0; c < 2 * NT; ++c)
                        if (r == c / 2 * 8 + 2 * quad + c % 2) unscale[c] *= power_of_two(e);
                }
#pragma unroll
                for (int i = 0; i < (DP + 31) / 32; ++i) {
                    const int d = lane + 32 * i;
                    float rest = x[i] * power_of_two(-e), zero = 0.f;
#pragma unroll
                    for (int s = 0; s < QP; ++s) {
                        const uint32_t u = take_part<Cache>(rest, zero);
                        if (d < DP) ((uint16_t*)(q_mem + (s * rows + r) * kQRow))[d] = (uint16_t)u;
                    }
                }
            }
            __syncwarp();
        }
        const uint32_t q_lane = smem_addr(q_mem) + min((lane >> 4) * 8 + (lane & 7), heads - 1) * kQRow + ((lane >> 3) & 1) * 16;

#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int t = 0; t < ND; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    acc[u][t][i] = 0.f;
                    if constexpr (kKeep) o[u][t][i] = 0.f;
                }
#pragma unroll
        for (int c = 0; c < 2 * NT; ++c) {
            m[c] = -INFINITY;
            l[c] = l_sum[c] = 0.f;
        }
        bool row_bad = cc.len < 0;
        const int first_j = cc.j;
        int fold = kFold, folds = 0;
        // keys on even counts, then values; one copy of the code that waits and loads
#pragma unroll 1
        for (int n = 2 * (cc.end - cc.j); n > 0; --n) {
            if (!bar_wait(bars + slot * 8, parity)) {
                give_up<Act>(p, seqs, cc, first_j, n, bars, slot, parity, S::kSlots);
                return;
            }
            const uint32_t at = ring + slot * S::kSlot;
            const int key0 = (cc.lo / kStep + cc.j) * kStep;
            const bool edge = key0 < cc.lo || key0 + kStep > cc.len;
            if (!(n & 1)) {
                row_bad |= (loader.bad >> slot) & 1;
                // ---- scores of 32 keys and the tile's heads
                // fragments are read a block ahead of the MMAs, which then find
                // their factors ready and as many sums apart as hide their latency
                float ch[2][2][NT][4] = {};   // two chains over the dimensions
                uint32_t kf[2][2][2][4];      // [buffer][16 dimensions][16 keys]
                auto load_keys = [&](int d) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            ldsm4(kf[d / 2 & 1][i][h], ((at + k_lane) ^ (((d + i) & 3) << 5)) + ((d + i) >> 2) * S::kTileBytes + h * S::kHalf);
                };
                load_keys(0);
#pragma unroll
                for (int d = 0; d < ND; d += 2) {
                    if (d + 2 < ND) load_keys(d + 2);
#pragma unroll
                    for (int s = 0; s < QP; ++s) {
                        uint32_t qb[2][4];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            if constexpr (NT == 1)
                                qb[i][0] = qf[d + i][s], qb[i][1] = qf[d + i][QP + s];
                            else
                                ldsm4(qb[i], q_lane + s * rows * kQRow + (d + i) * 32);
                        }
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int u = 0; u < NT; ++u)
                                    mma16816<Cache>(ch[i][h][u], kf[d / 2 & 1][i][h], qb[i][2 * u], qb[i][2 * u + 1]);
                    }
                }
                float (&c)[2][NT][4] = ch[0];

                // ---- the running softmax
                bool move = false;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int u = 0; u < NT; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float& s = c[h][u][i];
                            s = (s + ch[1][h][u][i]) * unscale[2 * u + i % 2];
                            if (edge) {
                                const int key = key0 + 16 * h + g + i / 2 * 8;
                                if (key < cc.lo || key >= cc.len) s = -INFINITY;
                            }
                            move |= s > m[2 * u + i % 2] + kLazy;
                        }
                if (__any_sync(~0u, move)) {
#pragma unroll
                    for (int x = 0; x < 2 * NT; ++x) {
                        const int u = x / 2, i = x % 2;
                        float top = fmaxf(fmaxf(c[0][u][i], c[0][u][i + 2]), fmaxf(c[1][u][i], c[1][u][i + 2]));
#pragma unroll
                        for (int s = 4; s <= 16; s <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, s));
                        top = fmaxf(top, m[x]);
                        const float a = top == -INFINITY ? 1.f : exp2_fast(m[x] - top);
                        m[x] = top;
                        if (cc.j == first_j) continue;   // nothing to rescale yet
                        l[x] *= a, l_sum[x] *= a;
#pragma unroll
                        for (int t = 0; t < ND; ++t) {
                            acc[u][t][i] *= a, acc[u][t][i + 2] *= a;
                            if constexpr (kKeep) o[u][t][i] *= a, o[u][t][i + 2] *= a;
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < NT; ++u) {
                    float base[2], sum[2] = {};
#pragma unroll
                    for (int i = 0; i < 2; ++i) base[i] = finite_or_zero(m[2 * u + i]) - kUp;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {   // rows g, then g + 8
                            float a = exp2_fast(c[h][u][2 * i] - base[0]), b = exp2_fast(c[h][u][2 * i + 1] - base[1]);
                            sum[0] += a, sum[1] += b;
                            // in parts, each what the ones before leave; transposed to the B operand
#pragma unroll
                            for (int s = 0; s < PP; ++s)
                                asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;"
                                             : "=r"(wf[h][u][s][i]) : "r"(take_part<Cache>(a, b)));
                        }
                    l[2 * u] += sum[0], l[2 * u + 1] += sum[1];
                }
            } else {
                if (edge) {   // zeros for the values outside the window
                    uint8_t* mem = ring_mem + slot * S::kSlot;
                    const int row = lane >> 3;   // 4 rows of a tile at a time
                    for (int r = row; r < kStep; r += 4) {
                        if (key0 + r >= cc.lo && key0 + r < cc.len) continue;
#pragma unroll
                        for (int t = 0; t < S::kTiles; ++t)
                            *(uint4*)(mem + r / 16 * S::kHalf + t * S::kTileBytes + r % 16 * 128 + (lane & 7) * 16) =
                                make_uint4(0, 0, 0, 0);
                    }
                    loader.dirty |= 1u << slot;
                    __syncwarp();
                }
                // ---- values, transposed, times weights
                constexpr int kAhead = ND % 4 == 0 ? 4 : 2;   // tiles of 16 columns per block
                uint32_t vf[2][kAhead][4];
                auto load_values = [&](int blk) {   // blocks of the first 16 keys, then of the others
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) {
                        const int t = blk * kAhead % ND + i, h = blk * kAhead / ND;
                        ldsm4t(vf[blk & 1][i], ((at + v_lane) ^ ((t & 3) << 5)) + (t >> 2) * S::kTileBytes + h * S::kHalf);
                    }
                };
                load_values(0);
#pragma unroll
                for (int blk = 0; blk < 2 * ND / kAhead; ++blk) {
                    if (blk + 1 < 2 * ND / kAhead) load_values(blk + 1);
                    const int h = blk * kAhead / ND;
#pragma unroll
                    for (int s = 0; s < PP; ++s)
#pragma unroll
                        for (int i = 0; i < kAhead; ++i)
#pragma unroll
                            for (int u = 0; u < NT; ++u)
                                mma16816<Cache>(acc[u][blk * kAhead % ND + i], vf[blk & 1][i], wf[h][u][s][0], wf[h][u][s][1]);
                }

                // ---- the MMA's sums to the rounded ones
                if (--fold == 0) {
                    fold = kFold;
                    float a[2 * NT];
#pragma unroll
                    for (int x = 0; x < 2 * NT; ++x) {
                        l_sum[x] += l[x];
                        l[x] = 0.f;
                        if constexpr (!kKeep) {   // in memory, with the reference that they were added at
                            a[x] = folds ? exp2_fast(m_fold[x] - finite_or_zero(m[x])) : 0.f;
                            m_fold[x] = m[x];
                        }
                    }
#pragma unroll
                    for (int u = 0; u < NT; ++u)
#pragma unroll
                        for (int t = 0; t < ND; ++t) {
                            if constexpr (kKeep) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) o[u][t][i] += acc[u][t][i];
                            } else {
                                float4* mem = (float4*)sums + (u * ND + t) * 32 + lane;
                                float4 y = folds ? *mem : make_float4(0.f, 0.f, 0.f, 0.f);
                                y.x = y.x * a[2 * u] + acc[u][t][0], y.y = y.y * a[2 * u + 1] + acc[u][t][1];
                                y.z = y.z * a[2 * u] + acc[u][t][2], y.w = y.w * a[2 * u + 1] + acc[u][t][3];
                                *mem = y;
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[u][t][i] = 0.f;
                        }
                    ++folds;
                }
                ++cc.j;
            }
            __syncwarp();   // every lane has read the slot
            loader.issue(slot);
            if (++slot == S::kSlots) slot = 0, parity ^= 1;
        }

        // ---- the end of the row, or of this part of it; the next row's queries
        // are on their way meanwhile, where there are registers for them
        const Cursor done = cc;
        live = next_row(cc, seqs, p);
        if (DP <= 128 && live) fetch_queries(cc);
        const bool whole = first_j == 0 && done.end == done.steps, none = done.len == done.lo;
        float* piece = p.pieces + (size_t)(2 * w + (first_j == 0)) * p.piece_floats;
        if (!whole && first_j == 0 && lane == 0) cut(p, done, w, part);
        unsigned odd[2 * NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            float a[2], inv[2], check[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int x = 2 * u + i, head = 8 * u + 2 * quad + i;
                l[x] += l_sum[x];
#pragma unroll
                for (int s = 4; s <= 16; s <<= 1) l[x] += __shfl_xor_sync(~0u, l[x], s);
                if (row_bad) l[x] = __int_as_float(0x7fc00000);
                a[i] = !kKeep && folds ? exp2_fast(m_fold[x] - finite_or_zero(m[x])) : 0.f;
                inv[i] = !whole ? 1.f : none ? 0.f : 1.f / l[x];
                check[i] = l[x] * 0.f;   // a NaN once anything infinite or NaN went in
                if (g == 0 && head < heads) {
                    if (!whole)
                        *(float2*)(piece + 2 * head) = make_float2(m[x], l[x]);
                    else if (p.lse)
                        p.lse[(size_t)done.b * p.n_q + first_head + head] =
                            none ? -INFINITY : 0.69314718055994531f * (m[x] + (log2f(l[x]) - kUp));
                }
            }
            // where this lane stores: 16-bit results as pairs of columns of head g,
            // others as it holds them
            Act* out = (Act*)p.out + ((size_t)done.b * p.n_q + first_head + 8 * u) * p.dim;
#pragma unroll
            for (int t = 0; t < ND; ++t) {
                float4 x = make_float4(acc[u][t][0], acc[u][t][1], acc[u][t][2], acc[u][t][3]);
                if constexpr (kKeep) {
                    x.x += o[u][t][0], x.y += o[u][t][1], x.z += o[u][t][2], x.w += o[u][t][3];
                } else if (folds) {
                    const float4 y = ((const float4*)sums)[(u * ND + t) * 32 + lane];
                    x.x += y.x * a[0], x.y += y.y * a[1], x.z += y.z * a[0], x.w += y.w * a[1];
                }
                check[0] += x.x * 0.f, check[1] += x.y * 0.f, check[0] += x.z * 0.f, check[1] += x.w * 0.f;
                if (!whole) {
                    if (8 * u + 2 * quad < heads) ((float4*)(piece + kPieceHead))[(u * ND + t) * 32 + lane] = x;
                    continue;
                }
                x.x *= inv[0], x.y *= inv[1], x.z *= inv[0], x.w *= inv[1];
                if (none) x = make_float4(0.f, 0.f, 0.f, 0.f);
                if constexpr (QP == 1) {
                    uint32_t lo = take_part<Cache>(x.x, x.y), hi = take_part<Cache>(x.z, x.w);
                    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(lo));
                    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(hi));
                    uint32_t* dst = (uint32_t*)(out + (size_t)g * p.dim + t * 16 + 2 * quad);
                    if (8 * u + g < heads && t * 16 < p.dim) dst[0] = lo;
                    if (8 * u + g < heads && t * 16 + 8 < p.dim) dst[4] = hi;
                } else {
                    float* dst = (float*)out + (size_t)2 * quad * p.dim + t * 16 + g;
                    const bool even = 8 * u + 2 * quad < heads, next = 8 * u + 2 * quad + 1 < heads;
                    if (t * 16 < p.dim) {
                        if (even) dst[0] = x.x;
                        if (next) dst[p.dim] = x.y;
                    }
                    if (t * 16 + 8 < p.dim) {
                        if (even) dst[8] = x.z;
                        if (next) dst[p.dim + 8] = x.w;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
                odd[2 * u + i] = __ballot_sync(~0u, 8 * u + 2 * quad + i < heads && check[i] != 0.f && !row_bad && !none);
        }
#pragma unroll
        for (int x = 0; x < 2 * NT; ++x)
            while (odd[x]) {
                const int src = __ffs(odd[x]) - 1, row = x / 2 * 8 + src % 4 * 2 + x % 2;
                odd[x] &= ~(0x11111111u << src % 4);
                const float mr = __shfl_sync(~0u, m[x], src), lr = __shfl_sync(~0u, l[x], src);
                __syncwarp();
                const int base = done.lo / kStep;
                redo_row<Cache, Act>(p, done.b, kv, first_head + row, max(done.lo, (base + first_j) * kStep),
                                     min(done.len, (base + done.end) * kStep), mr, lr, kUp, whole, piece, row, DP, lane);
            }
        if (DP > 128 && live) fetch_queries(cc);
    }
}

// ------------------------------------------------------------ the join
// Pieces of a cut row, in the order of the keys: weights from their m and l,
// then the weighted sum. A unit is 8 query heads of a cut row and 16 of its
// columns, as a lane holds them in a piece. Latency is all there is to it, so a
// unit is joined by one warp where its row has few pieces, by 4 or by the 32 of
// a CTA where it has more, with kBatch pieces' loads in flight together.
constexpr int kJoinWarps = 32, kJoinThreads = kJoinWarps * 32;
constexpr int kBatch = 4, kGroup = 4;                      // pieces in flight per warp; warps for some pieces
constexpr int kFew = kBatch, kSome = 2 * kGroup * kBatch;   // most pieces for one warp, for kGroup
constexpr int kChunk = 512;                                // pieces whose weights are in shared memory

// The weighted sum of pieces first, first + every, .. below n, in this lane's
// (column, head) places, with its heads' reference and sum.
struct Joined {
    float top[2], l[2];
    float4 x;
};
// adds n parts to j: the common reference first, then exps that do not wait for one another
template <int N>
__device__ inline void join_add(Joined& j, const float4 (&ml)[N], const float4 (&x)[N]) {   // ml: (m, l) of both heads
    float top[2] = {j.top[0], j.top[1]};
#pragma unroll
    for (int i = 0; i < N; ++i) top[0] = fmaxf(top[0], ml[i].x), top[1] = fmaxf(top[1], ml[i].z);
    const float base[2] = {finite_or_zero(top[0]), finite_or_zero(top[1])};
    const float old[2] = {exp2_fast(j.top[0] - base[0]), exp2_fast(j.top[1] - base[1])};
#pragma unroll
    for (int h = 0; h < 2; ++h) j.l[h] *= old[h], j.top[h] = top[h];
    j.x.x *= old[0], j.x.y *= old[1], j.x.z *= old[0], j.x.w *= old[1];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float f = exp2_fast(ml[i].x - base[0]), g = exp2_fast(ml[i].z - base[1]);
        j.l[0] += ml[i].y * f, j.l[1] += ml[i].w * g;
        j.x.x += x[i].x * f, j.x.y += x[i].y * g, j.x.z += x[i].z * f, j.x.w += x[i].w * g;
    }
}
__device__ inline const float* piece_at(const AttendParams& p, int warp, int k) {   // piece k of the row cut by this warp first
    return p.pieces + (size_t)(2 * (warp + k) + (k == 0)) * p.piece_floats;
}
__device__ inline Joined join_pieces(const AttendParams& p, int part, int n, int first, int every, int heads_at, int unit_at, bool real) {
    Joined j{{-INFINITY, -INFINITY}, {0.f, 0.f}, make_float4(0.f, 0.f, 0.f, 0.f)};
    for (int k0 = first; k0 < n; k0 += every * kBatch) {
        float4 ml[kBatch], x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int k = k0 + i * every;
            ml[i] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < n && real) {
                const float* src = piece_at(p, part, k);
                ml[i] = *(const float4*)(src + heads_at);
                x[i] = *(const float4*)(src + unit_at);
            }
        }
        join_add<kBatch>(j, ml, x);
    }
    return j;
}

template <class Act>
__global__ void __launch_bounds__(kJoinThreads) k_attend_join(const __grid_constant__ AttendParams p, int n_warps, int dp, float up) {
    // the warps that begin a cut row, with its pieces, and the row: those of few
    // pieces, then of some, then of many
    __shared__ uint2 list[kMaxWarps];
    __shared__ int counts[2][kJoinWarps];
    __shared__ union {
        Joined sums[kJoinWarps / 2][32];
        struct {
            float weight[8][kChunk];
            float red[8][4];   // 8 heads, 4 warps each
        };
    } sh;
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- the cut rows, in the order of the keys: those of two warps per thread
    static_assert(kMaxWarps <= kJoinThreads * 2, "one pass");
    const int first = threadIdx.x * 2;
    unsigned raw = 0;
    int2 row_of = make_int2(0, 0);
    if (first < n_warps) {   // the arrays are padded to 8
        raw = *(const unsigned*)(p.cut_pieces + first);
        row_of = *(const int2*)(p.cut_row + first);
    }
    const unsigned n[2] = {raw & 0xffff, first + 1 < n_warps ? raw >> 16 : 0};
    auto kind = [&](int i) { return n[i] == 0 ? -1 : n[i] <= kFew ? 0 : n[i] <= kSome ? 1 : 2; };
    int a = 0, b = 0;   // few and some in one number; many
#pragma unroll
    for (int i = 0; i < 2; ++i) a += kind(i) == 0 ? 1 : kind(i) == 1 ? 1 << 16 : 0, b += kind(i) == 2;
    int a_to = a, b_to = b;   // in the lanes before and this one
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int x = __shfl_up_sync(~0u, a_to, s), y = __shfl_up_sync(~0u, b_to, s);
        if (lane >= s) a_to += x, b_to += y;
    }
    if (lane == 31) counts[0][wid] = a_to, counts[1][wid] = b_to;
    __syncthreads();
    const int ca = counts[0][lane], cb = counts[1][lane];
    const int a_all = __reduce_add_sync(~0u, ca), b_all = __reduce_add_sync(~0u, cb);
    a_to += __reduce_add_sync(~0u, lane < wid ? ca : 0) - a, b_to += __reduce_add_sync(~0u, lane < wid ? cb : 0) - b;
    const int count[3] = {a_all & 0xffff, a_all >> 16, b_all};
    int to[3] = {a_to & 0xffff, count[0] + (a_to >> 16), count[0] + count[1] + b_to};
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (kind(i) >= 0)
            list[kind(i) == 0 ? to[0]++ : kind(i) == 1 ? to[1]++ : to[2]++] = make_uint2((first + i) | n[i] << 16, i ? row_of.y : row_of.x);
    __syncthreads();

    const int n_rows = p.n_kv * p.tiles, tiles_d = dp / 16, units = (p.piece_rows + 7) / 8 * tiles_d;
    const int g = lane >> 2, quad = lane & 3;
    auto finish = [&](int row, int unit, const Joined& j) {
        const int b = row / n_rows, h = row % n_rows, tile = h % p.tiles, heads = min(16, p.group - tile * 16);
        const int t = unit % tiles_d;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int head = unit / tiles_d * 8 + 2 * quad + i;
            if (head >= heads) continue;
            const size_t at = (size_t)b * p.n_q + h / p.tiles * p.group + tile * 16 + head;
            Act* dst = (Act*)p.out + at * p.dim + t * 16 + g;
            if (t * 16 < p.dim) dst[0] = sb_from_float<Act>((i ? j.x.y : j.x.x) / j.l[i]);
            if (t * 16 + 8 < p.dim) dst[8] = sb_from_float<Act>((i ? j.x.w : j.x.z) / j.l[i]);
            if (p.lse && t == 0 && g == 0) p.lse[at] = 0.69314718055994531f * (j.top[i] + (log2f(j.l[i]) - up));
        }
    };

    auto join = [&](uint2 cut, int unit, int from, int every) {
        const bool real = unit / tiles_d * 8 + 2 * quad < p.piece_rows;
        return join_pieces(p, cut.x & 0xffff, cut.x >> 16, from, every, 2 * (unit / tiles_d * 8 + 2 * quad),
                           kPieceHead + (unit * 32 + lane) * 4, real);
    };
    // ---- rows of many pieces, by the CTA: weights of all heads first, then the sums
    for (int u = blockIdx.x; u < count[2] * units; u += gridDim.x) {
        const uint2 cut = list[count[0] + count[1] + u / units];
        const int part = cut.x & 0xffff, pieces = cut.x >> 16, unit = u % units, h0 = unit / tiles_d * 8;
        const bool real = h0 + 2 * quad < p.piece_rows;
        const int head = wid / 4, slot = threadIdx.x % 128;   // of the weights: a head, and every 128th piece
        float top = -INFINITY, l = 0.f;                       // of that head
        Joined j{{0.f, 0.f}, {0.f, 0.f}, make_float4(0.f, 0.f, 0.f, 0.f)};
        for (int k0 = 0; k0 < pieces; k0 += kChunk) {
            float2 ml[kChunk / 128];
            float t = top;
#pragma unroll
            for (int i = 0; i < kChunk / 128; ++i) {
                const int k = k0 + slot + 128 * i;
                ml[i] = k < pieces && h0 + head < p.piece_rows ? *(const float2*)(piece_at(p, part, k) + 2 * (h0 + head))
                                                               : make_float2(-INFINITY, 0.f);
                t = fmaxf(t, ml[i].x);
            }
#pragma unroll
            for (int s = 16; s; s >>= 1) t = fmaxf(t, __shfl_xor_sync(~0u, t, s));
            __syncthreads();
            if (lane == 0) sh.red[head][wid % 4] = t;
            __syncthreads();
            t = fmaxf(fmaxf(sh.red[head][0], sh.red[head][1]), fmaxf(sh.red[head][2], sh.red[head][3]));
            const float old = exp2_fast(top - finite_or_zero(t));
            top = t;
            l *= old;
#pragma unroll
            for (int i = 0; i < kChunk / 128; ++i) {
                const float f = exp2_fast(ml[i].x - finite_or_zero(t));
                sh.weight[head][slot + 128 * i] = f;
                l += f * ml[i].y;
            }
            __syncthreads();
            // the sums so far, at the new reference
            float now[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                now[i] = fmaxf(fmaxf(sh.red[2 * quad + i][0], sh.red[2 * quad + i][1]), fmaxf(sh.red[2 * quad + i][2], sh.red[2 * quad + i][3]));
                const float f = k0 ? exp2_fast(j.top[i] - finite_or_zero(now[i])) : 0.f;
                j.top[i] = now[i];
                if (i == 0) j.x.x *= f, j.x.z *= f;
                if (i == 1) j.x.y *= f, j.x.w *= f;
            }
            const int end = min(kChunk, pieces - k0);
            for (int i0 = wid; i0 < end; i0 += kJoinWarps * 2 * kBatch) {
                float4 x[2 * kBatch];
#pragma unroll
                for (int i = 0; i < 2 * kBatch; ++i) {
                    const int k = i0 + i * kJoinWarps;
                    x[i] = k < end && real ? *(const float4*)(piece_at(p, part, k0 + k) + kPieceHead + (unit * 32 + lane) * 4)
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int i = 0; i < 2 * kBatch; ++i) {
                    const int k = min(i0 + i * kJoinWarps, kChunk - 1);
                    const float f = sh.weight[2 * quad][k], g = sh.weight[2 * quad + 1][k];
                    if (i0 + i * kJoinWarps < end)
                        j.x.x += x[i].x * f, j.x.y += x[i].y * g, j.x.z += x[i].z * f, j.x.w += x[i].w * g;
                }
            }
        }
        // the heads' sums, then the warps' columns
#pragma unroll
        for (int s = 16; s; s >>= 1) l += __shfl_xor_sync(~0u, l, s);
        __syncthreads();
        if (lane == 0) sh.red[head][wid % 4] = l;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
            j.l[i] = (sh.red[2 * quad + i][0] + sh.red[2 * quad + i][1]) + (sh.red[2 * quad + i][2] + sh.red[2 * quad + i][3]);
        __syncthreads();
        for (int half = kJoinWarps / 2; half; half /= 2) {
            if (wid >= half && wid < 2 * half) sh.sums[wid - half][lane].x = j.x;
            __syncthreads();
            if (wid < half) {
                const float4 x = sh.sums[wid][lane].x;
                j.x.x += x.x, j.x.y += x.y, j.x.z += x.z, j.x.w += x.w;
            }
            __syncthreads();
        }
        if (wid == 0) finish(cut.y, unit, j);
    }
    // ---- of some: by groups of warps; two groups share a place for their sums, in turn
    {
        const int group = wid / kGroup, per = kJoinWarps / kGroup;
        for (int u0 = blockIdx.x * per; u0 < count[1] * units; u0 += gridDim.x * per) {
            const int u = u0 + group;
            const bool here = u < count[1] * units;
            Joined j;
            uint2 cut = make_uint2(0, 0);
            if (here) cut = list[count[0] + u / units], j = join(cut, u % units, wid % kGroup, kGroup);
            for (int turn = 0; turn < 2; ++turn) {
                const bool on = here && group % 2 == turn;
                if (on) sh.sums[group / 2 * kGroup + wid % kGroup][lane] = j;
                __syncthreads();
                if (on && wid % kGroup == 0) {
                    float4 ml[kGroup - 1], x[kGroup - 1];
#pragma unroll
                    for (int i = 1; i < kGroup; ++i) {
                        const Joined& k = sh.sums[group / 2 * kGroup + i][lane];
                        ml[i - 1] = make_float4(k.top[0], k.l[0], k.top[1], k.l[1]), x[i - 1] = k.x;
                    }
                    join_add<kGroup - 1>(j, ml, x);
                    finish(cut.y, u % units, j);
                }
                __syncthreads();
            }
        }
    }
    // ---- of few
    for (int u = blockIdx.x * kJoinWarps + wid; u < count[0] * units; u += gridDim.x * kJoinWarps) {
        const uint2 cut = list[u / units];
        finish(cut.y, u % units, join(cut, u % units, 0, 1));
    }
}

// ------------------------------------------------------------ launches
// What is kept of a device holds for that device alone. A number beyond the table is asked anew.
constexpr int kMaxDevices = 64;
int device_index() {
    int dev = -1;
    return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kMaxDevices ? dev : -1;
}
int sm_count() {
    static std::atomic<int> kept[kMaxDevices];
    const int at = device_index();
    int sms = at >= 0 ? kept[at].load(std::memory_order_relaxed) : 0;
    if (sms) return sms;
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    sms = std::min(sms < 1 ? 148 : sms, kMaxWarps / 8);
    if (at >= 0) kept[at].store(sms, std::memory_order_relaxed);
    return sms;
}
int tile_width(int dim) { return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256; }
int most_warps(int dim) { return dim <= 128 ? 8 : dim <= 192 ? 5 : 4; }   // Shape<>::kWarps
int piece_floats(int group, int dim) { return kPieceHead + (group <= 8 ? 8 : 16) * tile_width(dim); }
// The workspace: which rows are cut, their pieces, the warps' rounded sums.
struct Layout {
    size_t cut_row, pieces, sums, bytes;
    Layout(int group, int dim) {
        const size_t warps = (size_t)sm_count() * most_warps(dim), padded = (warps + 7) / 8 * 8;
        const size_t piece = piece_floats(group, dim) * sizeof(float);
        cut_row = (padded * sizeof(uint16_t) + 255) / 256 * 256;
        pieces = cut_row + (padded * sizeof(int) + 255) / 256 * 256;
        sums = pieces + 2 * warps * piece;
        bytes = sums + warps * piece;
    }
};

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) == cudaSuccess &&
                        found == cudaDriverEntryPointSuccess;
        cudaGetLastError();
        return ok ? (EncodeTiled)f : nullptr;
    }();
    return fn;
}
// [pages][heads][tiles of 64 columns][slots][columns] with a box of p.box slots and
// p.box_tiles tiles; with one tile the columns are the whole head and TMA fills
// with zeros what lies past it
bool cache_map(CUtensorMap* map, const void* base, int type, const AttendParams& p, size_t page, size_t slot, size_t head) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    const bool all = p.box_tiles > 1;
    const cuuint64_t dims[5] = {(cuuint64_t)(all ? 64 : p.dim), (cuuint64_t)p.page_size, (cuuint64_t)p.box_tiles,
                                (cuuint64_t)p.n_kv, (cuuint64_t)p.n_pages};
    // the stride of a dimension of one is never used, whatever the caller's
    const cuuint64_t strides[4] = {p.page_size == 1 ? 16 : slot, 128, p.n_kv == 1 ? 16 : head, p.n_pages == 1 ? 16 : page};
    const cuuint32_t box[5] = {64, (cuuint32_t)p.box, (cuuint32_t)p.box_tiles, 1, 1}, ones[5] = {1, 1, 1, 1, 1};
    return encode(map, type == SB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                  const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class Cache, int DP, int QP, int NT>
int launch(AttendParams p, cudaStream_t st) {
    using S = Shape<DP>;
    using Act = typename std::conditional<QP == 1, Cache, float>::type;
    constexpr bool kF16 = std::is_same<Cache, __half>::value;
    const int q_rows = NT == 1 ? 0 : std::min(p.group, 16) * QP;
    const size_t per_warp = S::kSlots * (S::kSlot + 8) + (size_t)q_rows * (DP * 2 + 16);
    const size_t seqs = 8 * (size_t)p.n_seqs + 4;
    // static shared memory (the scan's warp sums) takes 1024 bytes, the rings' alignment
    const int warps = (int)std::min<size_t>(S::kWarps, (kSmemLimit - 1024 - seqs) / per_warp);
    static std::atomic<bool> opted[kMaxDevices];
    const int dev = device_index();
    if (dev < 0 || !opted[dev].load(std::memory_order_relaxed)) {
        if (!sb_cuda_ok(cudaFuncSetAttribute(k_attend<Cache, DP, QP, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kSmemLimit - 1024), "attend shared memory"))
            return -1;
        if (dev >= 0) opted[dev].store(true, std::memory_order_relaxed);
    }
    const int type = kF16 ? SB_F16 : SB_BF16;
    p.box = 16;
    while (p.page_size % p.box) p.box /= 2;
    p.box_tiles = p.box == 16 && p.dim == S::kTiles * 64 ? S::kTiles : 1;
    CUtensorMap kmap{}, vmap{};
    if (p.n_pages > 0 && (!cache_map(&kmap, p.k, type, p, p.k_page, p.k_slot, p.k_head) ||
                          !cache_map(&vmap, p.v, type, p, p.v_page, p.v_slot, p.v_head))) {
        sb_set_error("attend: no tensor map for a cache of %d pages of %d, strides %zu / %zu / %zu and %zu / %zu / %zu bytes",
                     p.n_pages, p.page_size, p.k_page, p.k_slot, p.k_head, p.v_page, p.v_slot, p.v_head);
        return -1;
    }
    // steps of the longest row that fits; none is cut where that is short
    const long long longest = std::min((long long)p.table_width * p.page_size,
                                       p.window > 0 ? p.window + kStep - 1ll : 1ll << 40);
    const bool cuts = longest > kWhole * kStep;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = sm_count();
    cfg.blockDim = warps * 32;
    cfg.dynamicSmemBytes = warps * per_warp + seqs;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (!sb_cuda_ok(cudaLaunchKernelEx(&cfg, k_attend<Cache, DP, QP, NT>, (const AttendParams)p, (const CUtensorMap)kmap,
                                       (const CUtensorMap)vmap), "attend launch"))
        return -1;
    if (!cuts) return 0;
    cfg.gridDim = sm_count();
    cfg.blockDim = kJoinThreads;
    cfg.dynamicSmemBytes = 0;
    return sb_cuda_ok(cudaLaunchKernelEx(&cfg, k_attend_join<Act>, (const AttendParams)p, sm_count() * warps, DP, up_of(kF16)), "attend join launch")
               ? 0 : -1;
}

template <class Cache, int QP, int NT>
int launch_dim(const AttendParams& p, cudaStream_t st) {
    switch (tile_width(p.dim)) {
    case 64: return launch<Cache, 64, QP, NT>(p, st);
    case 96: return launch<Cache, 96, QP, NT>(p, st);
    case 128: return launch<Cache, 128, QP, NT>(p, st);
    case 192: return launch<Cache, 192, QP, NT>(p, st);
    default: return launch<Cache, 256, QP, NT>(p, st);
    }
}
template <class Cache, int QP>
int launch_group(const AttendParams& p, cudaStream_t st) {
    return p.group <= 8 ? launch_dim<Cache, QP, 1>(p, st) : launch_dim<Cache, QP, 2>(p, st);
}

}  // namespace

SABAH_API size_t sabah_attend_paged_workspace(int n_q_heads, int n_kv_heads, int head_dim) {
    if (n_kv_heads <= 0 || n_q_heads <= 0 || head_dim <= 0 || head_dim > kMaxDim) return 0;
    return Layout(n_q_heads / n_kv_heads, head_dim).bytes;
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
        (long long)table_width * page_size > 0x7fffff00ll) {   // a step past the last key is still an int
        sb_set_error("invalid attend cache (%d pages of %d, %d per sequence, window %d)", n_pages, page_size,
                     table_width, window);
        return -1;
    }
    if (n_seqs == 0) return 0;
    if (!d_q || !d_lens || !d_out || (table_width && !d_block_table) || (n_pages && (!d_k_cache || !d_v_cache)) ||
        ((uintptr_t)d_q | q_seq_stride | q_head_stride) % ab || (uintptr_t)d_out % 4 ||
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
    static const bool test = std::getenv("SABAH_TEST_ATTEND_STALL") != nullptr;   // at the first call; then by call
    const char* stall = test ? std::getenv("SABAH_TEST_ATTEND_STALL") : nullptr;
    p.stalled = stall ? std::atoi(stall) : -1;
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
    const Layout lay(p.group, head_dim);
    uint8_t* ws = (uint8_t*)d_workspace;
    p.cut_pieces = (uint16_t*)ws;
    p.cut_row = (int*)(ws + lay.cut_row);
    p.pieces = (float*)(ws + lay.pieces);
    p.sums = (float*)(ws + lay.sums);
    // the list of a launch has fewer than 2^31 places
    const long long most = (long long)n_kv_heads * p.tiles * ((long long)table_width * page_size / kStep + 2 + kRowCost);
    if (most > 0x7fffffffll) {
        sb_set_error("attend: %d pages of %d per sequence are too many for %d key-value heads", table_width, page_size,
                     n_kv_heads);
        return -1;
    }
    const int per_launch = (int)std::min<long long>(kMaxSeqs, 0x7fffffffll / most);
    const int slot = sb_timing_begin("attend_paged", st);
    int rc = 0;
    for (int b = 0; b < n_seqs && rc == 0; b += per_launch) {
        AttendParams a = p;
        a.n_seqs = std::min(per_launch, n_seqs - b);
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
