// What the kernels of tree attention share: arguments, the split of the
// batch's work between CTAs, visibility masks and partial results.
//
// Work is counted in units of one page of one KV head: item (s, h) is what head
// h of sequence s reads, SEG units for its start and end (queries, output) and
// then npages(s) for its pages.  The units of the whole batch, in order
// (s, h, page), are cut into equal ranges, one per worker, so a batch of any
// lengths keeps every SM busy for the same time.  A worker walks the segments
// of its range (the pages of one item that lie in it); a segment that is a
// whole item is written to the output, any other leaves a partial result
// (unnormalised output, maximum and sum of every row) in the workspace, and
// k_tree_combine adds an item's partials in page order.  A worker has at most
// two partials: the item its range starts in (slot 0) and the item its range
// ends in (slot 1).  Until such a result is there, its place holds the sum over
// the runs of pages so far (tc_run); without partials a CTA has one place for
// that.  The first worker w whose pages start inside an item says
// in ws_join[w] what there is to add: the partial of worker w - 1 (slot 1) and
// those of w, w + 1 .. (slot 0).
// Where no sequence can have many pages (`whole`), an item is one unit: none is
// cut by ranges, and nothing is joined.  If there are few items, each goes to a
// cluster of `parts` CTAs instead of one: CTA r takes the r-th part of the
// item's pages and leaves its rows' partial results in its shared memory, and
// every CTA adds and writes every parts-th row.
//
// The query rows of an item are node * group + head of the group, cut into
// tiles of `tile_rows`; a worker is `lanes` CTAs, one per tile, that walk the
// same range at the same time, so the tiles after the first find K/V in L2.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "jl_internal.h"
#include "kernels.cuh"

namespace jl {
namespace tree {

// Units of a segment's start and end: about two pages' time on a B200 (4 us
// against 1.5 us a page with two CTAs an SM).
constexpr int SEG = 2;
constexpr int ST_PAGE = 1, ST_RANGE = 2, ST_TIMEOUT = 4;  // status bits

struct Args {
    const void* q;
    void* out;
    float* lse;
    long long q_ld, out_ld;
    int rows, q_heads, kv_heads, group, seqs, max_nodes;
    const int32_t* row_start;
    const int32_t* ctx;
    const uint64_t* mask;
    int mask_words;
    const int32_t* page_table;
    int max_pages, pages;
    const void* k;
    const void* v;
    float c2;          // scale * log2(e)
    int4* ws_join;     // [worker]
    float* ws_o;       // [CTA along x][lane][slot][tile_rows][HEAD]
    float* ws_ml;      // [worker][lane][slot][tile_rows][2]: maximum (scores times c2), sum
    int workers, lanes, tile_rows, min_units;
    int slots;         // 2: partial results; 1: only runs (tc_run) are added in ws_o
    int whole;         // items are not split over workers
    int parts;         // CTAs of a cluster that share a worker's only item; 1: none
    int q_tma;         // the tensor-core kernel's queries come by TMA
    int32_t* status;
};

__device__ __forceinline__ void flag(int32_t* status, int bit) {
    if (status) atomicOr(status, bit);
}

// One sequence's rows and positions, with lengths out of range cut (and
// flagged): nodes 0..n-1 in rows lo.., committed positions ctx, np pages.
struct Seq {
    int lo, n, ctx, np;
};
__device__ __forceinline__ Seq seq_of(const Args& a, int s) {
    Seq q;
    const int lo = a.row_start[s], hi = a.row_start[s + 1], c = a.ctx[s];
    const long long most = (long long)a.max_pages * PAGE;
    long long n = (long long)hi - lo, cc = c;
    if (lo < 0 || n < 0) n = 0;
    n = min(min(n, (long long)a.max_nodes), max(0ll, (long long)a.rows - lo));
    cc = min(max(cc, 0ll), most);
    const long long np = min((cc + n + PAGE - 1) / PAGE, (long long)a.max_pages);
    if (n != (long long)hi - lo || cc != c || cc + n > most) flag(a.status, ST_RANGE);
    q.lo = lo;
    q.n = (int)n;
    q.ctx = (int)cc;
    q.np = n > 0 ? (int)np : 0;
    return q;
}

// The units (fewer than 2^31, checked on the host) cut over the workers that
// have about min_units each: the first `more` of them get `each` + 1 units.
struct Split {
    int used, each, more;
    __device__ int at(int w) const { return each * min(w, used) + min(w, more); }
    __device__ int worker_of(int u) const {
        const int cut = (each + 1) * more;
        return u < cut ? u / (each + 1) : more + (u - cut) / each;
    }
};
__device__ __forceinline__ Split split_of(const Args& a, int total) {
    Split s;
    s.used = min(a.workers, max((total + a.min_units - 1) / a.min_units, 1));
    s.each = total / s.used;
    s.more = total - s.each * s.used;
    return s;
}

__device__ __forceinline__ int item_units(const Args& a, const Seq& q) { return a.whole ? 1 : q.np + SEG; }
__device__ __forceinline__ int units_of(const Args& a, const Seq& q) { return q.np ? a.kv_heads * item_units(a, q) : 0; }

struct Found {     // the sequence a worker's range starts in
    Seq q;
    int s, first;  // its index and its first unit
};
struct LocateScratch {  // in shared memory
    int sum[16];
    Found found;
};

// Finds the sequence that worker w's range starts in (found.s == seqs: none).
// Called by all `T` threads of the block (a multiple of 32, at most 512).
template <int T>
__device__ __forceinline__ Split locate(const Args& a, int w, LocateScratch& sc) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int per = (a.seqs + T - 1) / T;
    const int s0 = min(a.seqs, t * per), s1 = min(a.seqs, s0 + per);
    Seq q{0, 0, 0, 0};
    int mine = 0;
    for (int i = s0; i < s1; ++i) {
        q = seq_of(a, i);
        mine += units_of(a, q);
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) sc.sum[warp] = inc;
    if (t == 0) sc.found.s = a.seqs;
    __syncthreads();
    int from = inc - mine, total = 0;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) {
        if (i < warp) from += sc.sum[i];
        total += sc.sum[i];
    }
    const Split sp = split_of(a, total);
    const int u = sp.at(w);
    if (mine > 0 && u >= from && u < from + mine) {
        int i = s0;
        if (per > 1)
            for (;; ++i) {
                q = seq_of(a, i);
                const int len = units_of(a, q);
                if (u < from + len) break;
                from += len;
            }
        sc.found.q = q;
        sc.found.s = i;
        sc.found.first = from;
    }
    __syncthreads();
    return sp;
}

// Walks the segments of a range: pages p0 .. p1 - 1 (at least one) of item
// (s, h).
struct Walk {
    Seq q;
    int s, h, p0, p1;
    int item, end;  // the item's first unit; the end of the range
    __device__ bool start(const Args& a, const Found& f, int from, int to) {
        s = f.s;
        end = to;
        if (from >= end || s >= a.seqs) return false;
        q = f.q;
        h = (from - f.first) / item_units(a, q);
        item = f.first + h * item_units(a, q);
        p0 = a.whole ? 0 : max(0, from - item - SEG);
        p1 = a.whole ? q.np : min(q.np, end - item - SEG);
        return p1 > p0 || next(a);
    }
    // Keeps part `rank` of the item's pages; false: it has none.
    __device__ bool part(int rank, int parts) {
        p0 = q.np * rank / parts;
        p1 = q.np * (rank + 1) / parts;
        return p1 > p0;
    }
    __device__ bool next(const Args& a) {
        item += item_units(a, q);
        if (item + (a.whole ? 0 : SEG) >= end) return false;  // no page of the next item
        if (++h >= a.kv_heads) {
            h = 0;
            do {
                if (++s >= a.seqs) return false;
                q = seq_of(a, s);
            } while (q.np == 0);
        }
        p0 = 0;
        p1 = a.whole ? q.np : min(q.np, end - item - SEG);
        return true;
    }
    // Worker w's entry of ws_join, (row of node 0, nodes, KV head, partials), from
    // its first segment (`work`: it has one).
    __device__ int4 join(const Split& sp, int w, bool work) const {
        if (!work || p0 == 0) return make_int4(0, 0, 0, 0);
        if (sp.at(w - 1) > item + SEG) return make_int4(0, 0, 0, 0);  // an earlier worker says it
        return make_int4(q.lo, q.n, h, sp.worker_of(item + q.np + SEG - 1) - w + 2);
    }
    __device__ bool whole() const { return p0 == 0 && p1 == q.np; }
    __device__ int slot() const { return p0 > 0 ? 0 : 1; }
};

// The first word of a node's mask, to be on its way before it is needed.
__device__ __forceinline__ uint64_t first_word(const Args& a, const Seq& q, int node) {
    return a.mask ? a.mask[(size_t)(q.lo + node) * a.mask_words] : 0;
}

// The positions of page p that node `node` (row `lo + node`) sees, bit i =
// position 64 p + i; m0: its mask's first word.
__device__ __forceinline__ uint64_t visible(const Args& a, const Seq& q, int node, int p, uint64_t m0) {
    const long long first = (long long)p * PAGE;
    const long long base = first - q.ctx;  // node index of bit 0
    if (base + PAGE <= 0) return ~0ull;    // committed positions only
    uint64_t v;
    if (a.mask) {
        const uint64_t* m = a.mask + (size_t)(q.lo + node) * a.mask_words;
        if (base >= 0) {
            const int w = (int)(base >> 6), sh = (int)(base & 63);
            v = w == 0 ? m0 >> sh : w < a.mask_words ? m[w] >> sh : 0;
            if (sh && w + 1 < a.mask_words) v |= m[w + 1] << (64 - sh);
        } else {
            v = (m0 << (int)-base) | ((1ull << (int)-base) - 1);
        }
        const long long left = q.n - base;  // nodes past the tree are not seen
        if (left < PAGE) v &= (1ull << (int)max(left, 0ll)) - 1;
    } else {
        const long long left = node + 1 - base;
        v = left >= PAGE ? ~0ull : (1ull << (int)max(left, 0ll)) - 1;
    }
    return v;
}

// 2^x (ex2.approx.ftz: relative error about 2^-22, results below 2^-126 zero).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// i / d for 0 <= i < 256 d, 1 <= d <= 128, inv = 1 / d in f32: (i + 0.5) / d is at
// least 0.5 / 128 away from a whole number, the rounding at most 256 * 2^-23.
__device__ __forceinline__ int div_small(int i, float inv) { return (int)(((float)i + 0.5f) * inv); }

constexpr float LN2 = 0.6931471805599453f;

__device__ __forceinline__ void store4(float* p, float4 v) { *(float4*)p = v; }
__device__ __forceinline__ void store4(uint16_t* p, float4 v) {
    *(uint2*)p = make_uint2(f2bf16(v.x) | (uint32_t)f2bf16(v.y) << 16, f2bf16(v.z) | (uint32_t)f2bf16(v.w) << 16);
}

// A row's sum over partial results, each (maximum, sum, sums of 4 dims).
struct RowSum {
    float top, sum;
    float4 o;
};
__device__ __forceinline__ void add_part(RowSum& t, float m, float l, float4 v) {
    if (l == 0.f) return;  // nothing seen there
    const float top = fmaxf(t.top, m), ref = top == -INFINITY ? 0.f : top;
    const float f = ex2(t.top - ref), g = ex2(m - ref);
    t.top = top;
    t.sum = fmaf(t.sum, f, l * g);
    t.o = make_float4(fmaf(t.o.x, f, v.x * g), fmaf(t.o.y, f, v.y * g), fmaf(t.o.z, f, v.z * g), fmaf(t.o.w, f, v.w * g));
}
// Query row g of an item with first row lo and KV head h: writes dims 4 l .. and
// (lane 0) the lse.
template <typename T>
__device__ __forceinline__ void finish_row(const Args& a, int lo, int h, int g, int l, const RowSum& sum, float inv_group) {
    const float inv = sum.sum == 0.f ? 0.f : __fdiv_rn(1.f, sum.sum);
    const int node = div_small(g, inv_group), head = h * a.group + g - node * a.group;
    store4((T*)a.out + (size_t)(lo + node) * a.out_ld + (size_t)head * HEAD + 4 * l,
           make_float4(sum.o.x * inv, sum.o.y * inv, sum.o.z * inv, sum.o.w * inv));
    if (a.lse && l == 0) a.lse[(size_t)(lo + node) * a.q_heads + head] = sum.sum == 0.f ? -INFINITY : (sum.top + log2f(sum.sum)) * LN2;
}

// The attention kernel (tree_attn_tc.cu): query rows of a tile, CTAs per SM, and
// the launch, by the types of the rows (q and out) and of the pool.
constexpr int tc_tile_rows(bool rows_f32) { return rows_f32 ? 32 : 128; }
constexpr int tc_ctas(bool pool_f32) { return pool_f32 ? 1 : 2; }
// Pages of a run: what is added in TMEM before it is added to ws_o.  The tensor
// core's additions cut off, always towards zero, 2^-25 to 2^-24 of the sum for each
// on average, and there are 4 a page for every product of pieces: 64 (72 with a
// rest) and 72 in a run of f32 rows; 512 (576) of bf16 rows, whose rounding is 2^-9.
constexpr int tc_run(bool rows_f32, bool pool_f32) { return rows_f32 ? (pool_f32 ? 6 : 16) : (pool_f32 ? 32 : 64); }
struct TcLimits {
    static constexpr int SIZES = 3;
    int clusters[2][2][SIZES];  // of 2, 4, 8 CTAs that run at once, by [rows f32][pool f32]
};
jl_status tc_configure(TcLimits& limits);
jl_status tc_launch(Args a, bool rows_f32, bool pool_f32, cudaStream_t st);

}  // namespace tree
}  // namespace jl
