// What the kernels of tree attention share: arguments, the split of the
// batch's work between CTAs, visibility masks and partial results.
//
// Work is counted in units of one page of one KV head: sequence s has
// kv_heads * npages(s) units, item (s, h) the npages(s) of them that head h
// reads.  The units of the whole batch, in order (s, h, page), are cut into
// equal ranges, one per worker, so a batch of any lengths keeps every SM busy
// for the same time.  A worker walks the segments of its range (the part of
// one item that lies in it); a segment that is a whole item is written to the
// output, any other leaves a partial result (unnormalised output, maximum and
// sum of every row) in the workspace, and k_tree_combine adds an item's
// partials in page order.  A worker has at most two partials: the item its
// range starts in (slot 0) and the item its range ends in (slot 1).
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
    float* ws_o;       // [worker][lane][slot][tile_rows][HEAD]
    float* ws_ml;      // [worker][lane][slot][tile_rows][2]: maximum (scores times c2), sum
    int workers, lanes, tile_rows, min_units;
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

// First unit of worker w's range: the units cut evenly over the workers that
// have at least min_units each.
struct Split {
    long long total;
    int used;  // workers with a range
    __device__ long long at(int w) const { return w >= used ? total : total * w / used; }
};
__device__ __forceinline__ Split split_of(const Args& a, long long total) {
    Split s;
    s.total = total;
    const long long want = (total + a.min_units - 1) / a.min_units;
    s.used = (int)min((long long)a.workers, max(want, 1ll));
    return s;
}

struct LocateScratch {  // in shared memory
    long long sum[16];
    long long first;
    int s;
};

// Finds the sequence that unit `at(w)` lies in.  Called by all `T` threads of
// the block (a multiple of 32, at most 512); returns the split and leaves the
// sequence and its first unit in *s, *first (s == seqs: no work).
template <int T>
__device__ __forceinline__ Split locate(const Args& a, int w, LocateScratch& sc, int* s, long long* first) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int per = (a.seqs + T - 1) / T;
    const int s0 = min(a.seqs, t * per), s1 = min(a.seqs, s0 + per);
    long long mine = 0;
    for (int i = s0; i < s1; ++i) mine += (long long)a.kv_heads * seq_of(a, i).np;
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) sc.sum[warp] = inc;
    if (t == 0) {
        sc.s = a.seqs;
        sc.first = 0;
    }
    __syncthreads();
    long long from = inc - mine, total = 0;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) {
        if (i < warp) from += sc.sum[i];
        total += sc.sum[i];
    }
    const Split sp = split_of(a, total);
    const long long u = sp.at(w);
    if (mine > 0 && u >= from && u < from + mine) {
        int i = s0;
        for (;; ++i) {
            const long long len = (long long)a.kv_heads * seq_of(a, i).np;
            if (u < from + len) break;
            from += len;
        }
        sc.s = i;
        sc.first = from;
    }
    __syncthreads();
    *s = sc.s;
    *first = sc.first;
    return sp;
}

// Walks the segments of a range.
struct Walk {
    Seq q;
    int s, h;         // item
    int p0, p1;       // its pages in this range
    long long u, end;
    __device__ bool start(const Args& a, int s_, long long first, long long from, long long to) {
        s = s_;
        u = from;
        end = to;
        if (u >= end || s >= a.seqs) return false;
        q = seq_of(a, s);
        h = (int)((u - first) / q.np);
        p0 = (int)((u - first) - (long long)h * q.np);
        p1 = (int)min((long long)q.np, p0 + (end - u));
        return true;
    }
    __device__ bool next(const Args& a) {
        u += p1 - p0;
        if (u >= end) return false;
        if (++h >= a.kv_heads) {
            h = 0;
            do {
                if (++s >= a.seqs) return false;
                q = seq_of(a, s);
            } while (q.np == 0);
        }
        p0 = 0;
        p1 = (int)min((long long)q.np, end - u);
        return true;
    }
    __device__ bool whole() const { return p0 == 0 && p1 == q.np; }
    __device__ int slot() const { return p0 > 0 ? 0 : 1; }
};

// The positions of page p that node `node` (row `lo + node`) sees, bit i =
// position 64 p + i.
__device__ __forceinline__ uint64_t visible(const Args& a, const Seq& q, int node, int p) {
    const long long first = (long long)p * PAGE;
    const long long base = first - q.ctx;  // node index of bit 0
    if (base + PAGE <= 0) return ~0ull;    // committed positions only
    uint64_t v;
    if (a.mask) {
        const uint64_t* m = a.mask + (size_t)(q.lo + node) * a.mask_words;
        if (base >= 0) {
            const int w = (int)(base >> 6), sh = (int)(base & 63);
            v = w < a.mask_words ? m[w] >> sh : 0;
            if (sh && w + 1 < a.mask_words) v |= m[w + 1] << (64 - sh);
        } else {
            v = (m[0] << (int)-base) | ((1ull << (int)-base) - 1);
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

constexpr float LN2 = 0.6931471805599453f;

// Tensor-core kernel (tree_attn_tc.cu): query rows of a tile, CTAs per SM, and
// the launch over a pool of bf16 pages; `f32`: the type of the q and out rows.
constexpr int TC_CTAS_PER_SM = 2;
constexpr int tc_tile_rows(bool f32) { return f32 ? 64 : 128; }
jl_status tc_configure();
jl_status tc_launch(const Args& a, bool f32, cudaStream_t st);

}  // namespace tree
}  // namespace jl
