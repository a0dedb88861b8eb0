// Tree attention on tensor cores.
//
// A CTA walks its worker's range (tree_attn.cuh) page by page with six warps:
// warp 5 brings K and V pages into two rings by TMA, warp 4 issues the MMAs,
// and warps 0-3 do the softmax, a thread per query row (MMA row = TMEM lane).
//   * S = Q K^T (128 x 64 f32) goes to TMEM.  bf16 queries are exact.
//   * The softmax thread reads its row's 64 scores, masks those it does not
//     see (only on pages past the committed positions), and writes the weights
//     2^(s c2 - m) back over the scores as bf16 pieces, the A operand of the
//     next MMA: two for bf16 outputs, each rounded to nearest, which leaves 2^-17
//     of a weight at most and no bias (cut off they left up to 2^-15, always low,
//     and twice as many outputs rounded to the wrong neighbour, in the same time).
//   * O += P V accumulates in TMEM over a run of pages (tc_run) and is then added
//     in the workspace: the tensor core's additions cut off, so over a whole long
//     segment O came out too small, by 4.7e-5 for f32 rows at 12000 positions and
//     values of one sign, 1.3e-4 over an f32 pool; by 2.3e-6 and 3.9e-6 in runs.  A
//     run's end costs 2 to 3 us (24 sequences of 4 f32 nodes at 8000 positions 174 ->
//     186 us, f32 pool 638 -> 710).  m is the maximum when it was last moved: it moves, and O is rescaled, only when a row's
//     maximum has grown by more than 2^8, so that pages seldom touch O.
//   * The scores of page j + 1 are computed while page j's weights are (two S
//     buffers).
// f32 rows are stacked: a tile has 32 rows, and lanes 32 p + r hold piece p of
// row r's three bf16 pieces (24 bits), so that one MMA of 128 rows multiplies
// all pieces.  Warps 0-2 exchange their parts of S through shared memory; each
// adds them for a window of the keys and writes the pieces of their weights;
// then warp p takes piece p of all keys to TMEM.  The three parts of O are added
// at the end.  16 sequences of 8 nodes and 4 heads a KV head at 2000 positions:
// 55 us; 66 when each warp added all parts and computed all weights, 86 with
// three MMAs a product and every piece in the columns of 64 rows.
// Sums, maxima and O are f32.  V rows past the sequence, and values of tree
// nodes that are not finite, are cleared in shared memory before P V (zero
// times them would be NaN in rows that do not see them); rows that do see such
// a value get it added from global memory at the end.
// A page outside the pool is read as rows past the end of the tensor map,
// which arrive as zeros, and masked.
//
// Pools of f32 pages: eight warps take the place of the TMA warp.  They load a
// head's K or V rows into registers, two items ahead, and write them to the rings
// as bf16 pieces, which S and O then sum: three (24 bits, exact), but two of V for
// bf16 rows, the second rounded (2^-16 of a value at most, far below the output's
// rounding).  Every piece of a weight meets every piece of V: the product of the
// two second pieces alone may reach 2^-15.  One CTA fills an SM.  Clearing V happens on the way.
//
// B200, GPU times of calls in a graph with the joining kernel, bf16 rows and
// pools, 32 heads over 8: 32 sequences of 64 nodes at 4096 positions 240 us in a
// burst of 20 calls (580 TFLOP/s of the attention's own products, 860 with the
// second piece) and 282 us in a loop of seconds, where the power cap takes the
// clock from 1.9 to 1.55 GHz; one of 16 nodes at 40000 positions 46 to 52 us; 37 of
// one node at 4096 positions 118 us (5.3 TB/s, 80% of the copy rate).  Small trees
// over long contexts are bound by the pages' bytes (1.45 us a page and CTA is the
// copy rate); large ones by the chain of a page, with two CTAs an SM to overlap it
// (tensor pipe 48% of active cycles, exponentials 33%; 8 sequences of 64 nodes at
// 8192 positions); short ones by the chain of lookups, copies and first
// instructions (about 6 us) and by the joining kernel (5 us).
// Tried and not kept: eight softmax warps, two threads a row (272 -> 297 us for
// the first case: exchanging the maxima costs more than it saves); the scores of
// two pages as one MMA group of 128 columns (227 -> 252 us: the next scores no
// longer overlap the softmax); output rows written as whole lines by way of
// shared memory (44 -> 48 us for the second); half of the exponentials left out
// changed nothing.
#include <cuda.h>
#include <cuda_bf16.h>

#include "kernels.cuh"
#include "launch.cuh"
#include "mx_pieces.cuh"
#include "ptx.cuh"
#include "tree_attn.cuh"

namespace jl {
namespace tree {
namespace {

using mx::swz128;

constexpr int W_MMA = 4, W_LOAD = 5;
constexpr uint32_t PAGE_BYTES = PAGE * HEAD * 2;  // one head's K or V of a page: two boxes of 64 dims
constexpr uint32_t BOX_BYTES = PAGE_BYTES / 2;
constexpr uint32_t COL_O = 128, TMEM_COLS = 256;
constexpr uint32_t WAIT_POLLS = 1u << 20;
constexpr float MOVE = 8.f;  // log2 of how far a row's maximum may grow before it is moved

// T: type of the rows, KV: of the pool.  SPLIT: warps that hold the pieces of the
// same rows.  NP: pieces of the weights in a row's columns.  KP, VP: pieces
// of a page.  LOADERS: warps that bring the pages.
template <typename T, typename KV>
struct Cfg {
    static constexpr bool ROWS_F32 = sizeof(T) == 4, POOL_F32 = sizeof(KV) == 4;
    static constexpr int SPLIT = ROWS_F32 ? 3 : 1, NP = SPLIT > 1 ? 1 : 2, KP = POOL_F32 ? 3 : 1, VP = !POOL_F32 ? 1 : ROWS_F32 ? 3 : 2;
    static constexpr int ROWS = tc_tile_rows(ROWS_F32), Q_ROWS = SPLIT > 1 ? SPLIT * ROWS : 128;
    static constexpr int NK = SPLIT > 1 || POOL_F32 ? 2 : 3, NV = POOL_F32 && ROWS_F32 ? 1 : 2;
    static constexpr int XCH = SPLIT > 1 ? SPLIT * ROWS * 64 * 4 : 0;  // the exchange: 64 floats of every row and part
    static constexpr int LOADERS = POOL_F32 ? 8 : 1, THREADS = 32 * (5 + LOADERS), CTAS = tc_ctas(POOL_F32);
    static constexpr uint32_t KSLOT = KP * PAGE_BYTES, VSLOT = VP * PAGE_BYTES;
    static constexpr int RUN = tc_run(ROWS_F32, POOL_F32), REST = RUN / 8;
};
constexpr int SB = 2;   // S buffers
constexpr int WIN = 24;  // keys of a warp that exchanges

template <typename C>
struct Ctl {
    uint64_t kfull[C::NK], kempty[C::NK], vfull[C::NV], vempty[C::NV];
    uint64_t sfull[2], pfull[2], odone[2];  // by page parity
    uint64_t qfull, ofree, drain;
    uint32_t tmem;
    int stop;    // a wait gave up: every role leaves
    // The loader warps of an f32 pool took a value out of segment s: odd[s % 4] is
    // s + 1 (they are less than four segments ahead: the rings hold three pages)
    int odd[4];
    float tops[C::SPLIT > 1 ? 96 : 1];  // of a page's windows
    LocateScratch locate;
};

template <typename C>
constexpr uint32_t q_bytes() { return C::Q_ROWS * HEAD * 2; }
template <typename C>
constexpr size_t tc_smem() { return q_bytes<C>() + (size_t)C::NK * C::KSLOT + (size_t)C::NV * C::VSLOT + C::XCH + 1024; }
static_assert(sizeof(Ctl<Cfg<uint16_t, uint16_t>>) <= 1024 && sizeof(Ctl<Cfg<float, float>>) <= 1024, "control block");
static_assert(tc_smem<Cfg<float, uint16_t>>() <= 113 * 1024 && tc_smem<Cfg<uint16_t, uint16_t>>() <= 113 * 1024, "two CTAs an SM");
static_assert(tc_smem<Cfg<float, float>>() <= 227 * 1024 && tc_smem<Cfg<uint16_t, float>>() <= 227 * 1024, "one CTA an SM");

// Waits for a phase, for WAIT_POLLS polls or until another role stops.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* stop) {
    for (uint32_t i = 0; i < WAIT_POLLS; ++i) {
        if (ptx::mbar_try_wait(bar, parity)) return true;
        if ((i & 63) == 63 && *stop) return false;
    }
    *stop = 1;
    return false;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}

__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Query rows of a tile into shared memory, by the 128 softmax threads:
// [64-dim block][lane][128 B], swizzled.  Unstacked bf16 rows of groups that
// divide the tile come by TMA instead.
template <typename C, typename T>
__device__ __forceinline__ void load_q(const Args& a, const Walk& w, int row0, int live, float inv_group, uint8_t* sm, int tid) {
    const T* q = (const T*)a.q + (size_t)w.q.lo * a.q_ld + (size_t)w.h * a.group * HEAD;
    auto row = [&](int r) {
        const int node = div_small(row0 + r, inv_group);
        return q + node * a.q_ld + (row0 + r - node * a.group) * HEAD;
    };
    if constexpr (C::SPLIT == 1) {
#pragma unroll 8
        for (int i = tid; i < live * 16; i += 128) {
            const int r = i >> 4, c = i & 15;
            *(uint4*)(sm + (c >> 3) * (C::Q_ROWS * 128) + swz128((uint32_t)r, (uint32_t)(c & 7) * 16)) = *(const uint4*)(row(r) + 8 * c);
        }
    } else {
#pragma unroll
        for (int i = tid; i < C::ROWS * 32; i += 128) {
            const int r = i >> 5, c = i & 31;
            if (r >= live) break;
            float4 v = *(const float4*)(row(r) + 4 * c);
#pragma unroll
            for (int p = 0; p < C::SPLIT; ++p) {  // lanes ROWS p + r
                const uint32_t x = pack_bf16(v.x, v.y), y = pack_bf16(v.z, v.w);
                *(uint2*)(sm + (c >> 4) * (C::Q_ROWS * 128) + swz128((uint32_t)(p * C::ROWS + r), (uint32_t)(c & 15) * 8)) = make_uint2(x, y);
                v = make_float4(v.x - lo_f(x), v.y - hi_f(x), v.z - lo_f(y), v.w - hi_f(y));
            }
        }
    }
}

// Shared-memory matrix descriptors of 128-byte-swizzled operands (ptx::smem_desc
// with a stride of 1024 bytes).  Only the low word depends on the address, so
// the issuing thread adds constants to it: building each descriptor from its
// address costs more than the MMA takes.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return ((saddr & 0x3ffff) >> 4) | ((lbo >> 4) << 16); }
__device__ __forceinline__ uint64_t desc(uint32_t lo) { return (uint64_t)DESC_HI << 32 | lo; }

// S = Q K^T of one page, its pieces smallest first; q, k: low words.
template <typename C>
__device__ __forceinline__ void issue_scores(uint32_t q, uint32_t k, uint32_t tmem_s) {
    const uint32_t idesc = ptx::bf16_idesc(128, PAGE);
#pragma unroll
    for (int p = C::KP - 1; p >= 0; --p)
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
            for (int s = 0; s < 4; ++s)
                ptx::mma_bf16(tmem_s, desc(q + ((db * C::Q_ROWS * 128 + 32 * s) >> 4)),
                              desc(k + ((p * PAGE_BYTES + db * BOX_BYTES + 32 * s) >> 4)), idesc, (p < C::KP - 1 || db || s) ? 1u : 0u);
}

// The exchange between the warps that hold the pieces of 32 f32 rows: floats
// c .. c + 3 (c a multiple of 4 below 64) of a row's part, swizzled so that eight
// rows' float4s lie on all banks; and the sum of a row's three parts.
__device__ __forceinline__ float4* xch_at(uint8_t* xch, int part, int row, int c) {
    return (float4*)(xch + (part * 32 + row) * 256 + (((c >> 2) ^ (row & 7)) << 4));
}
__device__ __forceinline__ float4 xch_sum(uint8_t* xch, int row, int c) {
    const float4 u = *xch_at(xch, 0, row, c), v = *xch_at(xch, 1, row, c), y = *xch_at(xch, 2, row, c);
    return make_float4(u.x + (v.x + y.x), u.y + (v.y + y.y), u.z + (v.z + y.z), u.w + (v.w + y.w));
}

// O += P V of one page: P from TMEM, V (low word v) as an MN-major operand
// (64-dim blocks BOX_BYTES apart, groups of 8 keys 1024 bytes apart).
template <typename C>
__device__ __forceinline__ void issue_pv(uint32_t tmem_p, uint32_t v, uint32_t tmem_o, bool first) {
    const uint32_t idesc = ptx::bf16_idesc(128, HEAD) | (1u << 16);
#pragma unroll
    for (int vp = C::VP - 1; vp >= 0; --vp)
#pragma unroll
        for (int p = C::NP - 1; p >= 0; --p) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {  // keys 16 s ..
                ptx::mma_bf16_ta(tmem_o, tmem_p + 32 * p + 8 * s, desc(v + ((vp * PAGE_BYTES + 2048 * s) >> 4)), idesc, first ? 0u : 1u);
                first = false;
            }
        }
}

__device__ __forceinline__ bool odd_bf16(uint32_t h) { return (h & 0x7f80u) == 0x7f80u; }  // infinite or NaN

// Clears rows of a V page that lie past the sequence, and values of the tree's
// rows that are not finite; true if there was one of those.  Thread t of 128:
// row t / 2, dims of block t % 2.
__device__ __forceinline__ bool clean_v(uint8_t* v, int tree_row, int used, int t) {
    bool odd = false;
    const int r = t >> 1;
    uint8_t* row = v + (t & 1) * BOX_BYTES + r * 128;
    if (r >= used) {
#pragma unroll
        for (int c = 0; c < 8; ++c) *(uint4*)(row + 16 * c) = make_uint4(0u, 0u, 0u, 0u);
    } else if (r >= tree_row) {
        for (int c = 0; c < 8; ++c) {
            uint4 x = *(const uint4*)(row + 16 * c);
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
            bool hit = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (odd_bf16(w[i])) w[i] &= 0xffff0000u, hit = true;
                if (odd_bf16(w[i] >> 16)) w[i] &= 0x0000ffffu, hit = true;
            }
            if (hit) {
                *(uint4*)(row + 16 * c) = make_uint4(w[0], w[1], w[2], w[3]);
                odd = true;
            }
        }
    }
    return odd;
}

// A barrier of the first N softmax threads that tells whether `ok` holds for all.
template <int N>
__device__ __forceinline__ bool all_of(bool ok) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n"
        " setp.ne.u32 p, %1, 0;\n"
        " barrier.cta.red.and.pred q, %2, %3, p;\n"
        " selp.u32 %0, 1, 0, q;\n}"
        : "=r"(r)
        : "r"((uint32_t)ok), "n"(N / 32), "n"(N)
        : "memory");
    return r != 0;
}

// Whether a run ends before page i > 0 of a segment's n; a rest of an eighth of a
// run at most stays with the last.
template <typename C>
__device__ __forceinline__ bool run_ends(int i, int n) { return i % C::RUN == 0 && n - i > C::REST; }

// A run's end (tc_run): O is added to acc, in order of the runs, which first gets
// the factor f for what the rows' maxima have moved since (`add`: it is not the
// first).  acc: the tile's rows of HEAD floats, in the workspace.
template <typename C>
__device__ __noinline__ void save_run(float* acc, uint8_t* xch, uint32_t t_o, int warp, int lane, int live, float f, bool add) {
    float o[32];
    if constexpr (C::SPLIT == 1) {
        acc += (size_t)(32 * warp + lane) * HEAD;
#pragma unroll 1
        for (int c = 0; c < HEAD; c += 32) {
            __syncwarp();
            ptx::tmem_ld32_sync(t_o + c, o);
            if (32 * warp + lane >= live) continue;
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                const float4 v = add ? *(const float4*)(acc + c + e) : make_float4(0.f, 0.f, 0.f, 0.f);
                *(float4*)(acc + c + e) = make_float4(fmaf(v.x, f, o[e]), fmaf(v.y, f, o[e + 1]), fmaf(v.z, f, o[e + 2]), fmaf(v.w, f, o[e + 3]));
            }
        }
    } else {  // the three parts of 64 dims at a time; then a half warp adds a row
        constexpr int STEPS = (C::ROWS / 2 + C::SPLIT - 1) / C::SPLIT;
        const int first = 2 * warp + (lane >> 4), rows = min(live, C::ROWS);
#pragma unroll 1
        for (int c = 0; c < HEAD; c += 64) {
            float4* at = (float4*)(acc + (size_t)first * HEAD + c) + (lane & 15);
            float4 v[STEPS];
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
                v[k] = add && first + 2 * C::SPLIT * k < rows ? at[2 * C::SPLIT * k * (HEAD / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
            __syncwarp();
#pragma unroll 1
            for (int d = 0; d < 64; d += 32) {
                ptx::tmem_ld32_sync(t_o + c + d, o);
#pragma unroll
                for (int e = 0; e < 32; e += 4) *xch_at(xch, warp, lane, d + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
            all_of<32 * C::SPLIT>(true);
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                const int r = first + 2 * C::SPLIT * k;
                const float g = __shfl_sync(0xffffffffu, f, r & 31);
                if (r < rows) {
                    const float4 u = xch_sum(xch, r, 4 * (lane & 15));
                    at[2 * C::SPLIT * k * (HEAD / 4)] = make_float4(fmaf(v[k].x, g, u.x), fmaf(v[k].y, g, u.y), fmaf(v[k].z, g, u.z), fmaf(v[k].w, g, u.w));
                }
            }
            __syncwarp();
            all_of<32 * C::SPLIT>(true);
        }
    }
}

// The last run's end: O gets f times acc added, in the rows of the one warp of a
// row's that calls this.
__device__ __noinline__ void load_runs(const float* acc, uint32_t t_o, bool mine, float f) {
#pragma unroll 1
    for (int c = 0; c < HEAD; c += 32) {
        float o[32];
        uint32_t bits[32];
        ptx::tmem_ld32_sync(t_o + c, o);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            const float4 v = mine ? *(const float4*)(acc + c + e) : make_float4(0.f, 0.f, 0.f, 0.f);
            bits[e] = __float_as_uint(fmaf(v.x, f, o[e])), bits[e + 1] = __float_as_uint(fmaf(v.y, f, o[e + 1]));
            bits[e + 2] = __float_as_uint(fmaf(v.z, f, o[e + 2])), bits[e + 3] = __float_as_uint(fmaf(v.w, f, o[e + 3]));
        }
        __syncwarp();
        ptx::tmem_st32(t_o + c, bits);
    }
    ptx::tmem_wait_st();
}

// Adds what clean_v took out to a warp's rows of O: for every node of this
// segment's pages that a row sees, its weight times the values that are not
// finite.  Arguments by value: nothing of the caller's moves to the stack.
__device__ __forceinline__ float value(uint16_t h) { return bf16f(h); }
__device__ __forceinline__ float value(float f) { return f; }
template <typename T, typename KV>
__device__ __noinline__ void add_odd(const Args a, const Walk w, int g, bool mine, float m, uint32_t t_o) {
    const int32_t* pt = a.page_table + (size_t)w.s * a.max_pages;
    const int node = g / a.group;
    const T* q = (const T*)a.q + (size_t)(w.q.lo + (mine ? node : 0)) * a.q_ld + (size_t)(w.h * a.group + g % a.group) * HEAD;
#pragma unroll 1
    for (int d0 = 0; d0 < HEAD; d0 += 32) {
        float o[32];
        uint32_t bits[32];
        ptx::tmem_ld32_sync(t_o + d0, o);
        for (int p = max(w.p0, w.q.ctx / PAGE); mine && p < w.p1; ++p) {
            const int page = pt[p];
            if ((unsigned)page >= (unsigned)a.pages) continue;
            const uint64_t vis = visible(a, w.q, node, p, first_word(a, w.q, node));
            for (int r = 0; r < PAGE; ++r) {
                const long long pos = (long long)p * PAGE + r;
                if (!(vis >> r & 1) || pos < w.q.ctx) continue;
                const KV* k = (const KV*)a.k + kv_index(page, w.h, r, a.kv_heads);
                const KV* v = (const KV*)a.v + kv_index(page, w.h, r, a.kv_heads) + d0;
                float weight = -1.f;
#pragma unroll
                for (int d = 0; d < 32; ++d) {
                    if (isfinite(value(v[d]))) continue;
                    if (weight < 0.f) {
                        float s = 0.f;
                        for (int e = 0; e < HEAD; ++e) s = fmaf(value(q[e]), value(k[e]), s);
                        weight = ex2(fmaf(s, a.c2, -m));
                    }
                    o[d] += weight * value(v[d]);
                }
            }
        }
        __syncwarp();
#pragma unroll
        for (int d = 0; d < 32; ++d) bits[d] = __float_as_uint(o[d]);
        ptx::tmem_st32(t_o + d0, bits);
    }
    ptx::tmem_wait_st();
}

// The loader warps of an f32 pool.  A segment's items, in the order in which the
// MMAs take them: K 0, K 1, V 0, K 2, V 1, .., V n - 1.
struct Item {
    uint32_t it;  // page count of the CTA, for the rings
    int seg;      // segment count of the CTA
    bool is_v;
    int used, tree_row;  // rows of the sequence; those from tree_row on are tree nodes
};
struct Items {
    Walk w;
    uint32_t it0 = 0;
    int seg = 0, step = 0;
    bool more;
    __device__ bool skip(const Args& a, int row0) const { return w.q.n * a.group <= row0; }
    __device__ void start(const Args& a, const Walk& from, int row0) {
        w = from;
        more = true;
        while (more && skip(a, row0)) more = w.next(a);
    }
    // Loads the next item's rows cw, cw + 8, .. of a warp (lane: 16 bytes of each).
    __device__ Item fetch(const Args& a, int row0, int cw, int lane, float4 (&x)[PAGE / 8]) {
        const int n = w.p1 - w.p0;
        const bool is_v = step >= 2 * n - 1 || (step && step % 2 == 0);
        const int j = !is_v ? (step + 1) / 2 : step == 2 * n - 1 ? n - 1 : step / 2 - 1, p = w.p0 + j;
        const int page = a.page_table[(size_t)w.s * a.max_pages + p];
        const bool there = (unsigned)page < (unsigned)a.pages;
        if (!there && !is_v && cw == 0 && lane == 0) flag(a.status, ST_PAGE);
        Item i{it0 + j, seg, is_v, there ? w.q.ctx + w.q.n - p * PAGE : 0, max(0, w.q.ctx - p * PAGE)};
        const float* src = (const float*)(is_v ? a.v : a.k) + kv_index(there ? page : 0, w.h, 0, a.kv_heads) + 4 * lane;
#pragma unroll
        for (int k = 0; k < PAGE / 8; ++k) {
            const int r = cw + 8 * k;
            x[k] = r < i.used ? *(const float4*)(src + (size_t)r * HEAD) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (++step == 2 * n) {
            it0 += n;
            step = 0;
            ++seg;
            do more = w.next(a);
            while (more && skip(a, row0));
        }
        return i;
    }
};

// One float4 of a row as n <= N pieces, each the next 8 bits by truncation; three
// hold all 24.  The second of two is rounded by adding half of what it drops: an
// addition more costs nothing that was measured (141 us with and without for 8
// sequences of 24 nodes, 32 bf16 heads over 8, at 4096 positions; conversions that
// round held the loaders up, 552 -> 716 us for 4 sequences of 60 nodes, 64 f32 heads
// over 8, at 2000).
template <int N>
__device__ __forceinline__ void store_pieces(uint8_t* dst, float4 x, int n) {
#pragma unroll
    for (int p = 0; p < N; ++p) {
        if (p >= n) break;
        const uint32_t up = p == 1 && n == 2 ? 0x8000u : 0u;  // half of what the last of two drops
        const uint32_t u0 = __float_as_uint(x.x) + up, u1 = __float_as_uint(x.y) + up, u2 = __float_as_uint(x.z) + up, u3 = __float_as_uint(x.w) + up;
        *(uint2*)(dst + p * PAGE_BYTES) = make_uint2(__byte_perm(u0, u1, 0x7632), __byte_perm(u2, u3, 0x7632));
        x = make_float4(x.x - hi_f(u0), x.y - hi_f(u1), x.z - hi_f(u2), x.w - hi_f(u3));
    }
}

template <typename T>
__device__ __forceinline__ void store_row32(T* dst, const float (&o)[32], float f);
template <>
__device__ __forceinline__ void store_row32<float>(float* dst, const float (&o)[32], float f) {
#pragma unroll
    for (int i = 0; i < 32; i += 4)
        *(float4*)(dst + i) = make_float4(o[i] * f, o[i + 1] * f, o[i + 2] * f, o[i + 3] * f);
}
template <>
__device__ __forceinline__ void store_row32<uint16_t>(uint16_t* dst, const float (&o)[32], float f) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        *(uint4*)(dst + i) = make_uint4(pack_bf16(o[i] * f, o[i + 1] * f), pack_bf16(o[i + 2] * f, o[i + 3] * f),
                                        pack_bf16(o[i + 4] * f, o[i + 5] * f), pack_bf16(o[i + 6] * f, o[i + 7] * f));
}

// The parts of an item that the CTAs of a cluster hold in shared memory: 128
// floats of each row, 16-byte units swizzled so that 8 rows lie on all banks.
__device__ __forceinline__ uint32_t part_at(int row, int unit) { return row * (HEAD * 4) + ((unit ^ (row & 31)) << 4); }
__device__ __forceinline__ void store_part(float* part, int row, int c, const float (&o)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 4)
        *(float4*)((uint8_t*)part + part_at(row, (c + i) >> 2)) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
}
// Adds them, in the order of the parts: each CTA takes every parts-th row, a
// warp a row, lane l its dims 4 l ..
template <typename T, int THREADS>
__device__ __forceinline__ void add_parts(const Args& a, const Walk& w, int rank, int row0, int rows, uint32_t o, uint32_t ml) {
    constexpr int AT_ONCE = 8;
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31;
    const float inv_group = 1.f / a.group;
    for (int r = rank + a.parts * warp; r < rows; r += a.parts * (THREADS / 32)) {
        RowSum sum{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
        for (int x = 0; x < a.parts; x += AT_ONCE) {
            float2 s[AT_ONCE];
            float4 v[AT_ONCE];
#pragma unroll
            for (int e = 0; e < AT_ONCE; ++e) {
                s[e] = make_float2(-INFINITY, 0.f);
                v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (x + e < a.parts) {
                    const uint32_t at = ptx::mapa(ml + 8 * r, x + e);
                    s[e] = make_float2(ptx::ld_shared_cluster(at), ptx::ld_shared_cluster(at + 4));
                    v[e] = ptx::ld_shared_cluster_v4(ptx::mapa(o + part_at(r, l), x + e));
                }
            }
#pragma unroll
            for (int e = 0; e < AT_ONCE; ++e) add_part(sum, s[e].x, s[e].y, v[e]);
        }
        finish_row<T>(a, w.q.lo, w.h, row0 + r, l, sum, inv_group);
    }
}

template <typename T, typename KV>
__global__ void __launch_bounds__(Cfg<T, KV>::THREADS, Cfg<T, KV>::CTAS)
    k_tree_attn_tc(Args a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                   const __grid_constant__ CUtensorMap qmap) {
    using C = Cfg<T, KV>;
    constexpr int ROWS = C::ROWS, NK = C::NK, NV = C::NV, NP = C::NP, SPLIT = C::SPLIT;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint8_t* kring = sm + q_bytes<C>();
    uint8_t* vring = kring + NK * C::KSLOT;
    uint8_t* xch = vring + NV * C::VSLOT;
    Ctl<C>& ctl = *(Ctl<C>*)(xch + C::XCH);
    volatile int* stop = &ctl.stop;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int worker = blockIdx.x / a.parts, rank = blockIdx.x % a.parts, tile = blockIdx.y;
    if (tid == 0) {
        for (int i = 0; i < NK; ++i) {
            ptx::mbar_init(&ctl.kfull[i], C::LOADERS);
            ptx::mbar_init(&ctl.kempty[i], 1);
        }
        for (int i = 0; i < NV; ++i) {
            ptx::mbar_init(&ctl.vfull[i], C::LOADERS);
            ptx::mbar_init(&ctl.vempty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&ctl.sfull[i], 1);
            ptx::mbar_init(&ctl.pfull[i], 4);
            ptx::mbar_init(&ctl.odone[i], 1);
        }
        ptx::mbar_init(&ctl.qfull, a.q_tma ? 1 : 4);
        ptx::mbar_init(&ctl.ofree, 4);
        ptx::mbar_init(&ctl.drain, 1);
        ptx::fence_barrier_init();
        ctl.stop = 0;
        for (int i = 0; i < 4; ++i) ctl.odd[i] = 0;
        if (!C::POOL_F32) {
            ptx::prefetch_tensormap(&kmap);
            ptx::prefetch_tensormap(&vmap);
        }
        if (a.q_tma) ptx::prefetch_tensormap(&qmap);
    }
    if (warp == W_MMA) {
        ptx::tmem_alloc(&ctl.tmem, TMEM_COLS);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    const Split sp = locate<C::THREADS>(a, worker, ctl.locate);
    Walk w;
    bool work = w.start(a, ctl.locate.found, sp.at(worker), sp.at(worker + 1)) && !(ptx::smem_u32(sm) & 1023);
    const int row0 = tile * ROWS;
    // a cluster's rows to add; the part of one without pages adds nothing
    const int shared_rows = a.parts > 1 && work ? min(ROWS, w.q.n * a.group - row0) : 0;
    float* part_o = (float*)sm;  // over Q and the rings, once they were read
    float2* part_ml = (float2*)(sm + ROWS * HEAD * 4);
    if (a.parts > 1 && work && !(work = w.part(rank, a.parts)))
        for (int i = tid; i < shared_rows; i += C::THREADS) part_ml[i] = make_float2(-INFINITY, 0.f);
    if (tid == 0 && tile == 0 && a.workers > 1 && !a.whole) a.ws_join[worker] = w.join(sp, worker, work);

    if (C::POOL_F32 && work && warp >= W_LOAD) {
        const int cw = warp - W_LOAD;
        Items items;
        items.start(a, w, row0);
        float4 x[2][PAGE / 8];  // two items on their way
        Item at[2];
        bool have[2] = {false, false}, ok = true;
#pragma unroll
        for (int b = 0; b < 2; ++b)
            if ((have[b] = items.more)) at[b] = items.fetch(a, row0, cw, lane, x[b]);
        while (ok && have[0]) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if (!ok || !have[b]) break;
                const Item& i = at[b];
                const uint32_t slot = i.is_v ? i.it % NV : i.it % NK, round = i.is_v ? i.it / NV : i.it / NK;
                ok = wait_phase(i.is_v ? &ctl.vempty[slot] : &ctl.kempty[slot], (round + 1) & 1, stop);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                uint8_t* dst = (i.is_v ? vring + slot * C::VSLOT : kring + slot * C::KSLOT) + (lane >> 4) * BOX_BYTES;
                bool odd = false;
#pragma unroll
                for (int k = 0; k < PAGE / 8; ++k) {
                    const int r = cw + 8 * k;
                    float4 v = x[b][k];
                    if (i.is_v && r >= i.tree_row && !(isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w))) {
                        odd = true;
                        v = make_float4(isfinite(v.x) ? v.x : 0.f, isfinite(v.y) ? v.y : 0.f, isfinite(v.z) ? v.z : 0.f, isfinite(v.w) ? v.w : 0.f);
                    }
                    store_pieces<C::KP>(dst + swz128((uint32_t)r, (uint32_t)(lane & 15) * 8), v, i.is_v ? C::VP : C::KP);
                }
                if (odd) *(volatile int*)&ctl.odd[i.seg & 3] = i.seg + 1;
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(i.is_v ? &ctl.vfull[slot] : &ctl.kfull[slot]);
                if ((have[b] = items.more)) at[b] = items.fetch(a, row0, cw, lane, x[b]);
            }
        }
    } else if (!C::POOL_F32 && work && warp == W_LOAD && lane == 0) {
        const int none = a.pages * a.kv_heads * PAGE;  // the row after the pool's last
        uint32_t it = 0, seg = 0;
        bool ok = true;
        auto queries = [&]() {
            const int node = row0 / a.group;
            ptx::mbar_arrive_expect_tx(&ctl.qfull, ROWS * HEAD * 2);
            ptx::tma_load_3d(sm, &qmap, 0, w.h * a.group, w.q.lo + node, &ctl.qfull);
            ptx::tma_load_3d(sm + ROWS * 128, &qmap, 64, w.h * a.group, w.q.lo + node, &ctl.qfull);
            ++seg;
        };
        do {
            if (w.q.n * a.group <= row0) continue;
            if (a.q_tma && it == 0) queries();
            const int32_t* pt = a.page_table + (size_t)w.s * a.max_pages;
            for (int p = w.p0; ok && p < w.p1; ++p, ++it) {
                const int page = pt[p];
                const bool there = (unsigned)page < (unsigned)a.pages;
                if (!there) flag(a.status, ST_PAGE);
                const int y = there ? (page * a.kv_heads + w.h) * PAGE : none;
                const uint32_t ks = it % NK, vs = it % NV;
                if (!wait_phase(&ctl.kempty[ks], (it / NK + 1) & 1, stop)) ok = false;
                if (ok) {
                    ptx::mbar_arrive_expect_tx(&ctl.kfull[ks], PAGE_BYTES);
                    ptx::tma_load_2d(kring + ks * PAGE_BYTES, &kmap, 0, y, &ctl.kfull[ks]);
                    ptx::tma_load_2d(kring + ks * PAGE_BYTES + BOX_BYTES, &kmap, 64, y, &ctl.kfull[ks]);
                    if (!wait_phase(&ctl.vempty[vs], (it / NV + 1) & 1, stop)) {
                        ok = false;
                        ptx::mbar_wait(&ctl.kfull[ks], (it / NK) & 1, WAIT_POLLS);
                    }
                }
                if (ok) {
                    ptx::mbar_arrive_expect_tx(&ctl.vfull[vs], PAGE_BYTES);
                    ptx::tma_load_2d(vring + vs * PAGE_BYTES, &vmap, 0, y, &ctl.vfull[vs]);
                    ptx::tma_load_2d(vring + vs * PAGE_BYTES + BOX_BYTES, &vmap, 64, y, &ctl.vfull[vs]);
                }
                if (ok && a.q_tma && p == w.p0 && it > 0) {  // once the last segment's scores are done
                    const uint32_t j = it - 1;
                    ok = wait_phase(&ctl.kempty[j % NK], (j / NK) & 1, stop);
                    if (ok) queries();
                }
            }
        } while (ok && w.next(a));
        // every copy in flight lands before the shared memory is given up
        for (uint32_t i = it > NK ? it - NK : 0; i < it; ++i) ptx::mbar_wait(&ctl.kfull[i % NK], (i / NK) & 1, WAIT_POLLS);
        for (uint32_t i = it > NV ? it - NV : 0; i < it; ++i) ptx::mbar_wait(&ctl.vfull[i % NV], (i / NV) & 1, WAIT_POLLS);
        if (seg > 0) ptx::mbar_wait(&ctl.qfull, (seg - 1) & 1, WAIT_POLLS);
    } else if (work && warp == W_MMA && lane == 0) {
        const uint32_t q = desc_lo(ptx::smem_u32(sm), 16), kr = desc_lo(ptx::smem_u32(kring), 16);
        const uint32_t vr = desc_lo(ptx::smem_u32(vring), BOX_BYTES);
        uint32_t it = 0, seg = 0, run = 0;
        bool ok = true;
        // A wait costs a few hundred cycles even when it is over: those that are
        // over early are made while the weights are still being computed.
        bool k_here = false;  // the next page's K was seen
        auto scores = [&](uint32_t i) {
            if (!k_here) ok = wait_phase(&ctl.kfull[i % NK], (i / NK) & 1, stop);
            k_here = false;
            if (!ok) return;
            ptx::tc_fence_after();
            issue_scores<C>(q, kr + (i % NK) * (C::KSLOT >> 4), tmem + 64 * (i % SB));
            ptx::tc_commit(&ctl.kempty[i % NK]);
            ptx::tc_commit(&ctl.sfull[i & 1]);
        };
        do {
            if (w.q.n * a.group <= row0) continue;
            const int n = w.p1 - w.p0;
            ok = wait_phase(&ctl.qfull, seg & 1, stop);
            if (ok) scores(it);
            for (int i = 0; ok && i < n; ++i, ++it) {
                if (i + 1 < n) scores(it + 1);
                ok = ok && wait_phase(&ctl.vfull[it % NV], (it / NV) & 1, stop);
                const bool fresh = i == 0 || run_ends<C>(i, n);  // the last run's O was read
                if (fresh && run++ > 0) ok = ok && wait_phase(&ctl.ofree, run & 1, stop);
                if (i + 2 < n) k_here = ptx::mbar_try_wait(&ctl.kfull[(it + 2) % NK], ((it + 2) / NK) & 1);
                ok = ok && wait_phase(&ctl.pfull[it & 1], (it >> 1) & 1, stop);
                if (!ok) break;
                ptx::tc_fence_after();
                issue_pv<C>(tmem + 64 * (it % SB), vr + (it % NV) * (C::VSLOT >> 4), tmem + COL_O, fresh);
                ptx::tc_commit(&ctl.vempty[it % NV]);
                ptx::tc_commit(&ctl.odone[it & 1]);
            }
            ++seg;
        } while (ok && w.next(a));
        // every MMA is done before TMEM and the shared memory are given up
        ptx::tc_commit(&ctl.drain);
        ptx::mbar_wait(&ctl.drain, 0, WAIT_POLLS);
    } else if (work && warp < 4) {
        const uint32_t t_lane = tmem + ((uint32_t)(warp * 32) << 16);
        const float inv_group = 1.f / a.group;
        const int r = SPLIT > 1 ? lane : tid;  // row of the tile
        uint32_t it = 0;
        int seg = 0;
        bool ok = true;
        do {
            const int live = min(ROWS, w.q.n * a.group - row0);
            if (live <= 0) continue;
            const int g = row0 + r, n = w.p1 - w.p0;
            const bool active = SPLIT > 1 ? warp < SPLIT : warp * 32 < live, mine = active && r < live;
            const int node = div_small(g, inv_group), head = w.h * a.group + g - node * a.group;
            if (!a.q_tma) {
                load_q<C, T>(a, w, row0, live, inv_group, sm, tid);
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&ctl.qfull);
            }
            const int32_t* pt = a.page_table + (size_t)w.s * a.max_pages;
            float m = -INFINITY, l = 0.f, m_run = -INFINITY;  // m_run: m at the end of the last run
            float* acc = a.ws_o + (((size_t)blockIdx.x * a.lanes + tile) * a.slots + (w.slot() & (a.slots - 1))) * (size_t)(ROWS * HEAD);
            auto runs_factor = [&]() {
                const float f = ex2(m_run - (m == -INFINITY ? 0.f : m));
                m_run = m;
                return f;
            };
            bool odd = false;  // this thread took a value out
            int page = pt[w.p0];
            const uint64_t m0 = mine ? first_word(a, w.q, node) : 0;
            // Warps that exchange leave the loop together: a wait that gives up
            // only clears ok, until the exchange tells all of them.
            for (int i = 0; i < n; ++i, ++it) {
                const int p = w.p0 + i;
                const bool there = (unsigned)page < (unsigned)a.pages;
                const bool edge = !there || (p + 1) * PAGE > w.q.ctx;
                if (i + 1 < n) page = pt[p + 1];
                ok = ok && wait_phase(&ctl.sfull[it & 1], (it >> 1) & 1, stop);
                // V only now: these threads do not wait for every page's V, and a phase
                // is told from the one before the last by the order of the waits alone.
                // The scores of page `it` are issued after page it - NV's V was waited
                // for, so the slot's phase cannot be two behind here.
                if (!C::POOL_F32 && edge && ok) {
                    static_assert(C::POOL_F32 || NV == 2, "scores are two pages ahead of the products at most");
                    ok = wait_phase(&ctl.vfull[it % NV], (it / NV) & 1, stop);
                    if (ok) {
                        odd |= clean_v(vring + (it % NV) * PAGE_BYTES, max(0, w.q.ctx - p * PAGE),
                                       there ? w.q.ctx + w.q.n - p * PAGE : 0, tid);
                        ptx::fence_proxy_async_smem();
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                if (!ok && !(SPLIT > 1 && active)) break;
                ptx::tc_fence_after();
                if (active) {
                    const uint32_t t_s = t_lane + 64 * (it % SB);
                    // moves the row's maximum to `top` where that is due, and O and l with it
                    auto move = [&](float top) {
                        float f = 1.f;
                        if (m == -INFINITY) {
                            m = top;  // nothing was seen before: O and l are zero
                        } else if (top > m + MOVE) {
                            f = ex2(m - top);
                            m = top;
                            l *= f;
                        }
                        if (i > 0 && !run_ends<C>(i, n) && __any_sync(0xffffffffu, mine && f != 1.f)) {
                            const uint32_t j = it - 1;  // every earlier P V is done
                            ok = __all_sync(0xffffffffu, wait_phase(&ctl.odone[j & 1], (j >> 1) & 1, stop));
                            ptx::tc_fence_after();
#pragma unroll 1
                            for (int c = 0; ok && c < HEAD; c += 32) {
                                float o[32];
                                uint32_t b[32];
                                ptx::tmem_ld32_sync(t_lane + COL_O + c, o);
#pragma unroll
                                for (int e = 0; e < 32; ++e) b[e] = __float_as_uint(o[e] * f);
                                ptx::tmem_st32(t_lane + COL_O + c, b);
                            }
                        }
                        return m == -INFINITY ? 0.f : m;
                    };
                    const uint64_t vis = !edge ? ~0ull : mine && there ? visible(a, w.q, node, p, m0) : 0;
                    // three pieces by truncation: each takes the next 8 bits, exactly
                    auto piece = [](float x, float y) { return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632); };
                    auto rest = [](float x, float y) {
                        return add2(make_float2(x, y), make_float2(-hi_f(__float_as_uint(x)), -hi_f(__float_as_uint(y))));
                    };
                    const float2 c2 = make_float2(a.c2, a.c2);
                    if constexpr (SPLIT > 1) {
                        // The windows have 24 keys; the last one's first 8 are the second's too.
                        // Code and registers are kept short here: S in halves and all
                        // of it sent took 55 us (case above), S at once 63, and only what
                        // others need, chosen by warp, more than the old exchange.
                        const int c0 = warp == 2 ? 40 : 24 * warp;
                        ok = all_of<32 * SPLIT>(ok);  // and the last page's pieces were read
                        if (!ok) break;
#pragma unroll
                        for (int h = 0; h < 64; h += 32) {
                            float s[32];
                            ptx::tmem_ld32_sync(t_s + h, s);
#pragma unroll
                            for (int c = 0; c < 32; c += 4) *xch_at(xch, warp, lane, h + c) = make_float4(s[c], s[c + 1], s[c + 2], s[c + 3]);
                        }
                        all_of<32 * SPLIT>(true);
                        float x[WIN];
#pragma unroll
                        for (int c = 0; c < WIN; c += 4) {
                            const float4 u = xch_sum(xch, lane, c0 + c);
                            x[c] = u.x, x[c + 1] = u.y, x[c + 2] = u.z, x[c + 3] = u.w;
                        }
                        if (edge) {
                            const uint32_t v = (uint32_t)(vis >> c0);
#pragma unroll
                            for (int c = 0; c < WIN; ++c)
                                if (!(v >> c & 1)) x[c] = -INFINITY;
                        }
                        float t0 = max3(x[0], x[1], x[2]), t1 = max3(x[3], x[4], x[5]);
#pragma unroll
                        for (int c = 6; c < WIN - 2; c += 4) t0 = max3(t0, x[c], x[c + 1]), t1 = max3(t1, x[c + 2], x[c + 3]);
                        ctl.tops[warp * 32 + lane] = fmaxf(max3(t0, x[WIN - 2], x[WIN - 1]), t1);
                        all_of<32 * SPLIT>(true);  // and every part was read
                        const float ref = move(max3(ctl.tops[lane], ctl.tops[32 + lane], ctl.tops[64 + lane]) * a.c2);
                        const float2 nref = make_float2(-ref, -ref);
                        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                        for (int q = 0; q < WIN / 8; ++q) {
                            const bool own = q > 0 || warp < 2;
                            uint32_t b[SPLIT][4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float2 y = fma2(make_float2(x[8 * q + 2 * e], x[8 * q + 2 * e + 1]), c2, nref);
                                y = make_float2(ex2(y.x), ex2(y.y));
                                if (own) sum = add2(sum, y);
#pragma unroll
                                for (int k = 0; k < SPLIT; ++k) {
                                    if (k) y = rest(y.x, y.y);
                                    b[k][e] = piece(y.x, y.y);
                                }
                            }
                            const uint32_t at = lane * 128 + (((c0 / 8 + q) ^ (lane & 7)) << 4);
#pragma unroll
                            for (int k = 0; k < SPLIT; ++k)
                                if (own) *(uint4*)(xch + k * 4096 + at) = make_uint4(b[k][0], b[k][1], b[k][2], b[k][3]);
                        }
                        l += sum.x + sum.y;
                        all_of<32 * SPLIT>(true);
                        uint32_t b[32];
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            const uint4 u = *(const uint4*)(xch + warp * 4096 + lane * 128 + ((q ^ (lane & 7)) << 4));
                            b[4 * q] = u.x, b[4 * q + 1] = u.y, b[4 * q + 2] = u.z, b[4 * q + 3] = u.w;
                        }
                        ptx::tmem_st32(t_s, b);
                    } else {
                        float x[64];
                        ptx::tmem_ld64_sync(t_s, x);
                        if (edge) {
                            const uint32_t v0 = (uint32_t)vis, v1 = (uint32_t)(vis >> 32);
#pragma unroll
                            for (int c = 0; c < 32; ++c) {
                                if (!(v0 >> c & 1)) x[c] = -INFINITY;
                                if (!(v1 >> c & 1)) x[32 + c] = -INFINITY;
                            }
                        }
                        float t0 = max3(x[0], x[1], x[2]), t1 = max3(x[3], x[4], x[5]);
                        float t2 = max3(x[6], x[7], x[8]), t3 = max3(x[9], x[10], x[11]);
#pragma unroll
                        for (int c = 12; c < 60; c += 8) {
                            t0 = max3(t0, x[c], x[c + 1]);
                            t1 = max3(t1, x[c + 2], x[c + 3]);
                            t2 = max3(t2, x[c + 4], x[c + 5]);
                            t3 = max3(t3, x[c + 6], x[c + 7]);
                        }
                        t0 = max3(t0, x[60], x[61]);
                        t1 = max3(t1, x[62], x[63]);
                        t0 = max3(t0, t1, t2);
                        const float ref = move(fmaxf(t0, t3) * a.c2);
                        const float2 nref = make_float2(-ref, -ref);
                        float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
                        for (int c = 0; c < 64; c += 4) {
                            float2 y = fma2(make_float2(x[c], x[c + 1]), c2, nref);
                            float2 z = fma2(make_float2(x[c + 2], x[c + 3]), c2, nref);
                            y = make_float2(ex2(y.x), ex2(y.y));
                            z = make_float2(ex2(z.x), ex2(z.y));
                            s0 = add2(s0, y);
                            s1 = add2(s1, z);
                            x[c] = y.x, x[c + 1] = y.y, x[c + 2] = z.x, x[c + 3] = z.y;
                        }
                        s0 = add2(s0, s1);
                        l += s0.x + s0.y;
#pragma unroll
                        for (int pc = 0; pc < NP; ++pc) {
                            uint32_t b[32];
#pragma unroll
                            for (int c = 0; c < 32; ++c) {
                                b[c] = pack_bf16(x[2 * c], x[2 * c + 1]);
                                if (pc + 1 < NP) {
                                    const float2 d = add2(make_float2(x[2 * c], x[2 * c + 1]), make_float2(-lo_f(b[c]), -hi_f(b[c])));
                                    x[2 * c] = d.x, x[2 * c + 1] = d.y;
                                }
                            }
                            ptx::tmem_st32(t_s + 32 * pc, b);
                        }
                    }
                    ptx::tmem_wait_st();
                }
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&ctl.pfull[it & 1]);
                if (run_ends<C>(i + 1, n)) {
                    if (active) {
                        ok = ok && wait_phase(&ctl.odone[it & 1], (it >> 1) & 1, stop);
                        ok = SPLIT > 1 ? all_of<32 * SPLIT>(ok) : __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        ptx::tc_fence_after();
                        const float f = runs_factor();
                        save_run<C>(acc, xch, t_lane + COL_O, warp, lane, live, f, i >= C::RUN);
                        ptx::tc_fence_before();
                        __syncwarp();
                    }
                    if (lane == 0) ptx::mbar_arrive(&ctl.ofree);
                }
            }
            if (ok) {
                const uint32_t j = it - 1;
                ok = wait_phase(&ctl.odone[j & 1], (j >> 1) & 1, stop);
            }
            ok = all_of<128>(ok);
            if (!ok) break;
            ptx::tc_fence_after();
            if (C::POOL_F32) odd = *(volatile int*)&ctl.odd[seg & 3] == seg + 1;
            ++seg;
            odd = !all_of<128>(!odd);
            if (active) {
                if (odd && (SPLIT == 1 || warp == 0)) add_odd<T, KV>(a, w, g, mine, m == -INFINITY ? 0.f : m, t_lane + COL_O);
                if (n > C::RUN + C::REST) {
                    const float f = runs_factor();
                    if (SPLIT == 1 || warp == 0) load_runs(acc + (size_t)r * HEAD, t_lane + COL_O, mine, f);
                }
                if constexpr (SPLIT > 1) {  // the windows' sums
                    ctl.tops[warp * 32 + lane] = l;
                    all_of<32 * SPLIT>(true);
                    l = ctl.tops[lane] + (ctl.tops[32 + lane] + ctl.tops[64 + lane]);
                }
                const bool whole = w.whole();
                const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);  // 0: nothing seen
                const size_t part = (((size_t)worker * a.lanes + tile) * 2 + w.slot()) * ROWS + r;  // partial results only
                T* out = (T*)a.out + (size_t)(w.q.lo + node) * a.out_ld + (size_t)head * HEAD;
                auto store = [&](int c, const float (&o)[32]) {
                    if (!mine) return;
                    if (a.parts > 1) store_part(part_o, r, c, o);
                    else if (whole) store_row32<T>(out + c, o, inv);
                    else store_row32<float>(a.ws_o + part * HEAD + c, o, 1.f);
                };
                if constexpr (SPLIT > 1) {  // 64 dims at a time: warp p adds the parts of dims 32 p ..
#pragma unroll 1
                    for (int c = 0; c < HEAD; c += 64) {
#pragma unroll 1
                        for (int d = 0; d < 64; d += 32) {
                            float o[32];
                            ptx::tmem_ld32_sync(t_lane + COL_O + c + d, o);
#pragma unroll
                            for (int e = 0; e < 32; e += 4) *xch_at(xch, warp, lane, d + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                        }
                        all_of<32 * SPLIT>(true);
                        if (warp < 2) {
                            float o[32];
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                const float4 u = xch_sum(xch, lane, 32 * warp + e);
                                o[e] = u.x, o[e + 1] = u.y, o[e + 2] = u.z, o[e + 3] = u.w;
                            }
                            store(c + 32 * warp, o);
                        }
                        all_of<32 * SPLIT>(true);
                    }
                } else {
#pragma unroll 1
                    for (int c = 0; c < HEAD; c += 32) {
                        float o[32];
                        ptx::tmem_ld32_sync(t_lane + COL_O + c, o);
                        store(c, o);
                    }
                }
                if (mine && (SPLIT == 1 || warp == 0)) {
                    if (a.parts > 1) part_ml[r] = make_float2(m, l);
                    else if (!whole) *(float2*)(a.ws_ml + part * 2) = make_float2(m, l);
                    else if (a.lse) a.lse[(size_t)(w.q.lo + node) * a.q_heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
                }
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&ctl.ofree);
        } while (w.next(a));
    }
    __syncwarp();
    __syncthreads();
    if (a.parts > 1) {
        ptx::cluster_sync();
        add_parts<T, C::THREADS>(a, w, rank, row0, shared_rows, ptx::smem_u32(part_o), ptx::smem_u32(part_ml));
        __syncwarp();
        ptx::cluster_sync();  // no CTA leaves while its parts are read
    }
    if (tid == 0 && (ctl.stop || (ptx::smem_u32(sm) & 1023))) flag(a.status, ST_TIMEOUT);
    ptx::tc_fence_after();
    if (warp == W_MMA) ptx::tmem_dealloc(tmem, TMEM_COLS);
}

template <typename T, typename KV>
jl_status launch(const Args& a, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& q, cudaStream_t st) {
    using C = Cfg<T, KV>;
    return launch_pdl_cluster(k_tree_attn_tc<T, KV>, a.parts, dim3(a.workers * a.parts, a.lanes), dim3(C::THREADS), tc_smem<C>(), st, a, k, v, q);
}

template <typename T, typename KV>
jl_status configure(TcLimits& limits) {
    using C = Cfg<T, KV>;
    auto kernel = k_tree_attn_tc<T, KV>;
    JL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tc_smem<C>()));
    // The call counts one CTA an SM: n of two an SM take the place of n / 2.
    for (int i = 0; i < TcLimits::SIZES; ++i) {
        const int n = (2 << i) / C::CTAS;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(n);
        cfg.blockDim = dim3(C::THREADS);
        cfg.dynamicSmemBytes = tc_smem<C>();
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = n;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        JL_CUDA(cudaOccupancyMaxActiveClusters(&limits.clusters[C::ROWS_F32][C::POOL_F32][i], kernel, &cfg));
    }
    return JL_OK;
}

}  // namespace

jl_status tc_configure(TcLimits& limits) {
    JL_TRY((configure<float, uint16_t>(limits)));
    JL_TRY((configure<uint16_t, uint16_t>(limits)));
    JL_TRY((configure<float, float>(limits)));
    return configure<uint16_t, float>(limits);
}

jl_status tc_launch(Args a, bool rows_f32, bool pool_f32, cudaStream_t st) {
    CUtensorMap k{}, v{}, q{};
    a.q_tma = 0;
    if (pool_f32) return rows_f32 ? launch<float, float>(a, k, v, q, st) : launch<uint16_t, float>(a, k, v, q, st);
    const uint64_t rows = (uint64_t)a.pages * a.kv_heads * PAGE;
    JL_TRY(kv_page_map(&k, a.k, rows));
    JL_TRY(kv_page_map(&v, a.v, rows));
    if (rows_f32) return launch<float, uint16_t>(a, k, v, q, st);
    // bf16 queries by TMA: rows (node, head of the group) of a tile are one box
    const int tile = tc_tile_rows(false);
    a.q_tma = tile % a.group == 0;
    if (a.q_tma) JL_TRY(q_row_map(&q, a.q, a.q_heads, a.rows, a.q_ld, a.group, tile / a.group));
    return launch<uint16_t, uint16_t>(a, k, v, q, st);
}

}  // namespace tree
}  // namespace jl
