// Attention of the nodes of drafted trees over the paged cache
// (jl_tree_attention): host checks, the CUDA-core kernel and the kernel that
// adds the partial results of items that several workers share.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "jl_internal.h"
#include "launch.cuh"
#include "ops_host.h"
#include "ptx.cuh"
#include "tree_attn.cuh"

namespace jl {
namespace tree {
namespace {

__device__ __forceinline__ float4 load4(const float* p) { return *(const float4*)p; }
__device__ __forceinline__ float4 load4(const uint16_t* p) {
    const uint2 w = *(const uint2*)p;
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
}
__device__ __forceinline__ void store4(float* p, float4 v) { *(float4*)p = v; }
__device__ __forceinline__ void store4(uint16_t* p, float4 v) {
    *(uint2*)p = make_uint2(f2bf16(v.x) | (uint32_t)f2bf16(v.y) << 16, f2bf16(v.z) | (uint32_t)f2bf16(v.w) << 16);
}

// ---- CUDA cores: pools of f32 pages -----------------------------------------------
//
// A CTA holds a tile of 16 * RT query rows and walks its range page by page:
// K and V of a page go to shared memory as f32; thread (ty, tx) scores keys
// tx + 16 i of rows ty + 16 j, the 16 threads of a row share its running
// maximum and sum (online softmax, base 2), and each keeps dims 4 tx .. and
// 64 + 4 tx .. of the row's output.
constexpr int CC_T = 256;
constexpr int CC_KLD = HEAD + 4;  // K rows padded: 8 rows' float4s on all banks
constexpr int CC_PLD = PAGE + 4;

template <int RT>
constexpr size_t cc_smem() {
    return sizeof(float) * ((size_t)16 * RT * CC_KLD + PAGE * CC_KLD + PAGE * HEAD + 16 * RT * CC_PLD);
}

template <typename T, int RT>
__global__ void __launch_bounds__(CC_T, RT <= 2 ? 2 : 1) k_tree_attn_cc(Args a) {
    extern __shared__ __align__(16) float cc_smem_raw[];
    float* qs = cc_smem_raw;                  // [16 RT][CC_KLD]
    float* ks = qs + 16 * RT * CC_KLD;        // [PAGE][CC_KLD]
    float* vs = ks + PAGE * CC_KLD;           // [PAGE][HEAD]
    float* ps = vs + PAGE * HEAD;             // [16 RT][CC_PLD]
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int worker = blockIdx.x, lane = blockIdx.y;
    constexpr int R = 16 * RT;
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    __shared__ LocateScratch scratch;
    const Split sp = locate<CC_T>(a, worker, scratch);
    Walk w;
    const bool work = w.start(a, scratch.found, sp.at(worker), sp.at(worker + 1));
    if (tid == 0 && lane == 0 && a.workers > 1 && !a.whole) a.ws_join[worker] = w.join(sp, worker, work);
    if (!work) return;
    do {
        const int live = min(R, w.q.n * a.group - lane * R);  // rows of this tile
        if (live <= 0) continue;
        __syncthreads();  // the previous segment's tiles are no longer read
        for (int i = tid; i < R * 32; i += CC_T) {
            const int r = i >> 5, c = i & 31, g = lane * R + r;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < live)
                v = load4((const T*)a.q + (size_t)(w.q.lo + g / a.group) * a.q_ld +
                          (size_t)(w.h * a.group + g % a.group) * HEAD + 4 * c);
            *(float4*)(qs + r * CC_KLD + 4 * c) = v;
        }
        float m[RT], l[RT], acc[RT][8];
        uint64_t m0[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            m[j] = -INFINITY;
            l[j] = 0.f;
            m0[j] = ty + 16 * j < live ? first_word(a, w.q, (lane * R + ty + 16 * j) / a.group) : 0;
#pragma unroll
            for (int d = 0; d < 8; ++d) acc[j][d] = 0.f;
        }
        const int32_t* pt = a.page_table + (size_t)w.s * a.max_pages;
        for (int p = w.p0; p < w.p1; ++p) {
            const int page = pt[p];
            const bool there = (unsigned)page < (unsigned)a.pages;
            if (!there && tid == 0) flag(a.status, ST_PAGE);
            const int used = there ? (int)min((long long)PAGE, (long long)w.q.ctx + w.q.n - (long long)p * PAGE) : 0;
            __syncthreads();  // the previous page's tiles are no longer read
            const size_t at = kv_index(there ? page : 0, w.h, 0, a.kv_heads);
            constexpr int LOADS = PAGE * 32 / CC_T;
            float4 kk[LOADS], vv[LOADS];  // all in flight
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = (tid + i * CC_T) >> 5, c = tid & 31;
                kk[i] = vv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < used) {  // rows past the sequence may hold anything
                    kk[i] = load4((const float*)a.k + at + (size_t)r * HEAD + 4 * c);
                    vv[i] = load4((const float*)a.v + at + (size_t)r * HEAD + 4 * c);
                }
            }
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = (tid + i * CC_T) >> 5, c = tid & 31;
                *(float4*)(ks + r * CC_KLD + 4 * c) = kk[i];
                *(float4*)(vs + r * HEAD + 4 * c) = vv[i];
            }
            __syncthreads();
            const bool edge = (long long)(p + 1) * PAGE > w.q.ctx || !there;
            uint64_t vis[RT];
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                const int r = ty + 16 * j;
                vis[j] = 0;
                if (16 * j + (ty & ~1) >= live) break;  // neither row of the warp is live
                vis[j] = !there || r >= live ? 0 : edge ? visible(a, w.q, (lane * R + r) / a.group, p, m0[j]) : ~0ull;
                float sc[4] = {0.f, 0.f, 0.f, 0.f};
                const float* qr = qs + r * CC_KLD;
#pragma unroll 8
                for (int c = 0; c < 32; ++c) {
                    const float4 q4 = *(const float4*)(qr + 4 * c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 k4 = *(const float4*)(ks + (tx + 16 * i) * CC_KLD + 4 * c);
                        sc[i] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, sc[i]))));
                    }
                }
                float top = m[j];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[i] = vis[j] >> (tx + 16 * i) & 1 ? __fmul_rn(sc[i], a.c2) : -INFINITY;
                    top = fmaxf(top, sc[i]);
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float ref = top == -INFINITY ? 0.f : top;
                const float corr = ex2(m[j] - ref);  // 0 while nothing was seen
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = vis[j] >> (tx + 16 * i) & 1 ? ex2(sc[i] - ref) : 0.f;
                    ps[r * CC_PLD + tx + 16 * i] = e;
                    sum += e;
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                l[j] = fmaf(l[j], corr, sum);
                m[j] = top;
#pragma unroll
                for (int d = 0; d < 8; ++d) acc[j][d] *= corr;
            }
            __syncwarp();  // a row's weights are read by the half warp that wrote them
            for (int key = 0; key < PAGE; ++key) {
                const float4 v0 = *(const float4*)(vs + key * HEAD + 4 * tx);
                const float4 v1 = *(const float4*)(vs + key * HEAD + 64 + 4 * tx);
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    if (16 * j + (ty & ~1) >= live) break;
                    // not seen: skipped, not multiplied by zero (V may be infinite)
                    if (edge && !(vis[j] >> key & 1)) continue;
                    const float e = ps[(ty + 16 * j) * CC_PLD + key];
                    acc[j][0] = fmaf(e, v0.x, acc[j][0]);
                    acc[j][1] = fmaf(e, v0.y, acc[j][1]);
                    acc[j][2] = fmaf(e, v0.z, acc[j][2]);
                    acc[j][3] = fmaf(e, v0.w, acc[j][3]);
                    acc[j][4] = fmaf(e, v1.x, acc[j][4]);
                    acc[j][5] = fmaf(e, v1.y, acc[j][5]);
                    acc[j][6] = fmaf(e, v1.z, acc[j][6]);
                    acc[j][7] = fmaf(e, v1.w, acc[j][7]);
                }
            }
        }
        const bool whole = w.whole();
        const size_t part = (((size_t)worker * a.lanes + lane) * 2 + w.slot()) * R;
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            const int r = ty + 16 * j, g = lane * R + r;
            if (r >= live) continue;
            float4 o0 = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
            float4 o1 = make_float4(acc[j][4], acc[j][5], acc[j][6], acc[j][7]);
            if (whole) {
                const float inv = l[j] == 0.f ? 0.f : __fdiv_rn(1.f, l[j]);  // 0: nothing seen
                const int row = w.q.lo + g / a.group, head = w.h * a.group + g % a.group;
                T* dst = (T*)a.out + (size_t)row * a.out_ld + (size_t)head * HEAD;
                store4(dst + 4 * tx, make_float4(o0.x * inv, o0.y * inv, o0.z * inv, o0.w * inv));
                store4(dst + 64 + 4 * tx, make_float4(o1.x * inv, o1.y * inv, o1.z * inv, o1.w * inv));
                if (a.lse && tx == 0)
                    a.lse[(size_t)row * a.q_heads + head] =
                        l[j] == 0.f ? -INFINITY : (m[j] + log2f(l[j])) * LN2;
            } else {
                store4(a.ws_o + (part + r) * HEAD + 4 * tx, o0);
                store4(a.ws_o + (part + r) * HEAD + 64 + 4 * tx, o1);
                if (tx == 0) *(float2*)(a.ws_ml + (part + r) * 2) = make_float2(m[j], l[j]);
            }
        }
    } while (w.next(a));
}

// ---- partial results -----------------------------------------------------------------
//
// The rows to add (query rows of the items that ws_join names) are dealt out
// over all blocks: each block scans the at most CB_MOST entries into a list of
// items and the groups of rows before each, then takes every gridDim.x-th
// group.  Lane l of a warp holds dims 4 l .. of a row, and all partials it adds
// are in flight at once where they are few: an item of fewer than CB_SHARE
// partials has groups of CB_ROWS rows, CB_RPW to a warp; one of more has groups
// of one row, whose partials the warps share and add in order.
constexpr int CB_WARPS = 4, CB_T = 32 * CB_WARPS, CB_PER_SM = 5;
constexpr int CB_MOST = 512, CB_EACH = CB_MOST / CB_T;  // workers at most; of them to a thread
constexpr int CB_SHARE = 8;    // partials from which the warps share a row
constexpr int CB_RPW = 2, CB_ROWS = CB_RPW * CB_WARPS;

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

template <typename T>
__global__ void __launch_bounds__(CB_T, CB_PER_SM) k_tree_combine(Args a) {
    __shared__ float4 share_o[CB_WARPS][32];
    __shared__ float2 share_ml[CB_WARPS];
    __shared__ int before[CB_MOST + 1];  // groups of CB_WARPS rows before item i
    __shared__ short who[CB_MOST];       // item i is ws_join[who[i]]
    __shared__ int2 warp_sums[CB_WARPS];
    const int t = threadIdx.x, warp = t >> 5, l = t & 31;
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    // items and their groups of rows: thread t's workers are CB_EACH t ..
    int some = 0, groups = 0, mine[CB_EACH];
#pragma unroll
    for (int e = 0; e < CB_EACH; ++e) {
        const int w = t * CB_EACH + e;
        const int4 join = w > 0 && w < a.workers ? a.ws_join[w] : make_int4(0, 0, 0, 0);
        const int rows = join.w > 0 ? join.y * a.group : 0;
        mine[e] = join.w >= CB_SHARE ? rows : (rows + CB_ROWS - 1) / CB_ROWS;
    }
#pragma unroll
    for (int e = 0; e < CB_EACH; ++e) {
        some += mine[e] > 0;
        groups += mine[e];
    }
    int item = some, sum = groups;  // up to and with this thread's
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, item, o), up2 = __shfl_up_sync(0xffffffffu, sum, o);
        if (l >= o) item += up, sum += up2;
    }
    if (l == 31) warp_sums[warp] = make_int2(item, sum);
    __syncthreads();
    item -= some;
    sum -= groups;
    groups = 0;
#pragma unroll
    for (int i = 0; i < CB_WARPS; ++i) {
        if (i < warp) item += warp_sums[i].x, sum += warp_sums[i].y;
        groups += warp_sums[i].y;
    }
#pragma unroll
    for (int e = 0; e < CB_EACH; ++e)
        if (mine[e] > 0) {
            who[item] = (short)(t * CB_EACH + e);
            before[item++] = sum;
            sum += mine[e];
        }
    if (t == CB_T - 1) before[item] = groups;
    __syncthreads();
    const float inv_group = 1.f / a.group;
    const int R = a.tile_rows;
    item = 0;
    for (int i = blockIdx.x; i < groups; i += gridDim.x) {
        while (before[item + 1] <= i) ++item;
        const int w = who[item];
        const int4 join = a.ws_join[w];
        const int rows = join.y * a.group, parts = join.w, at = i - before[item];
        // partial x of query row g: worker w - 1's slot 1, then slot 0 of the workers from w on
        auto slot = [&](int x, int g) {
            const int lane = g / R;
            return ((size_t)((w - 1 + x) * a.lanes + lane) * 2 + (x == 0 ? 1 : 0)) * R + (g - lane * R);
        };
        auto finish = [&](const RowSum& sum, int g) {
            const float inv = sum.sum == 0.f ? 0.f : __fdiv_rn(1.f, sum.sum);
            const int node = div_small(g, inv_group), head = join.z * a.group + g - node * a.group;
            store4((T*)a.out + (size_t)(join.x + node) * a.out_ld + (size_t)head * HEAD + 4 * l,
                   make_float4(sum.o.x * inv, sum.o.y * inv, sum.o.z * inv, sum.o.w * inv));
            if (a.lse && l == 0)
                a.lse[(size_t)(join.x + node) * a.q_heads + head] =
                    sum.sum == 0.f ? -INFINITY : (sum.top + log2f(sum.sum)) * LN2;
        };
        if (parts < CB_SHARE) {
            float2 ml[CB_RPW][CB_SHARE - 1];
            float4 v[CB_RPW][CB_SHARE - 1];
#pragma unroll
            for (int r = 0; r < CB_RPW; ++r) {
                const int g = at * CB_ROWS + r * CB_WARPS + warp;
#pragma unroll
                for (int x = 0; x < CB_SHARE - 1; ++x) {
                    ml[r][x] = make_float2(-INFINITY, 0.f);
                    v[r][x] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (x < parts && g < rows) {
                        const size_t p = slot(x, g);
                        ml[r][x] = *(const float2*)(a.ws_ml + p * 2);
                        v[r][x] = *(const float4*)(a.ws_o + p * HEAD + 4 * l);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < CB_RPW; ++r) {
                const int g = at * CB_ROWS + r * CB_WARPS + warp;
                RowSum sum{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
                for (int x = 0; x < CB_SHARE - 1; ++x)
                    if (x < parts) add_part(sum, ml[r][x].x, ml[r][x].y, v[r][x]);
                if (g < rows) finish(sum, g);
            }
            continue;
        }
        const int x0 = parts * warp / CB_WARPS, x1 = parts * (warp + 1) / CB_WARPS;
        RowSum sum{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
        for (int x = x0; x < x1; x += CB_SHARE) {
            float2 ml[CB_SHARE];
            float4 v[CB_SHARE];
#pragma unroll
            for (int e = 0; e < CB_SHARE; ++e) {
                ml[e] = make_float2(-INFINITY, 0.f);
                v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (x + e < x1) {
                    const size_t p = slot(x + e, at);
                    ml[e] = *(const float2*)(a.ws_ml + p * 2);
                    v[e] = *(const float4*)(a.ws_o + p * HEAD + 4 * l);
                }
            }
#pragma unroll
            for (int e = 0; e < CB_SHARE; ++e) add_part(sum, ml[e].x, ml[e].y, v[e]);
        }
        __syncthreads();  // the last row's sums were read
        share_o[warp][l] = sum.o;
        if (l == 0) share_ml[warp] = make_float2(sum.top, sum.sum);
        __syncthreads();
        if (warp != 0) continue;
        sum = RowSum{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
        for (int e = 0; e < CB_WARPS; ++e) add_part(sum, share_ml[e].x, share_ml[e].y, share_o[e][l]);
        finish(sum, at);
    }
}

// ---- host ----------------------------------------------------------------------------

// The kernel that a call takes and how it cuts the work.
struct Plan {
    int tile_rows, lanes, workers, min_units, whole;
    size_t bytes;
};

Plan plan_of(const jl_tree_attn& a, int sms) {
    Plan p;
    const int rows = a.max_nodes * (a.q_heads / a.pool.kv_heads);
    const bool tc = a.pool.dtype == JL_KV_BF16;
    p.tile_rows = tc ? tc_tile_rows(a.dtype == JL_KV_F32) : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    p.lanes = (rows + p.tile_rows - 1) / p.tile_rows;
    p.workers = std::min(CB_MOST, std::max(1, (tc ? TC_CTAS_PER_SM : p.tile_rows <= 32 ? 2 : 1) * sms / p.lanes));
    // Whole items or split ones: whole, a worker's longest item sets the time (in
    // waves of all workers); split, the mean does, and the join is added.  The
    // times, in us on a B200 with every SM busy, are a page's (tensor cores: 1.5
    // for bf16 rows, 2 for f32; CUDA cores: 8), a segment's start and end (6) and
    // the join (5).  Measured whole / split, 8 bf16 nodes, 32 heads over 8: one
    // sequence of 300 positions 10.6 / 14.7 us, 32 of them 15.3 / 30.4 us, 32 of up
    // to 700 23.6 / 34.5 us; f32 rows, one sequence of 700 29.6 / 20.9 us.
    const double page = !tc ? 8.0 : a.dtype == JL_KV_F32 ? 2.0 : 1.5;
    const double ctas = (double)a.seqs * a.pool.kv_heads * p.lanes, slots = (double)p.workers * p.lanes;
    const double whole = std::ceil(ctas / slots) * (a.max_pages * page + 6);
    const double split = std::max(ctas * (a.max_pages + SEG) / slots, 1.0 + SEG) * page + 6 + 5;
    // sizes of 0 ask for the workspace of any call
    p.whole = a.seqs > 0 && a.max_pages > 0 && whole <= split;
    p.min_units = p.whole ? 1 : 1 + SEG;
    p.bytes = p.workers == 1 || p.whole ? 0 : (size_t)p.workers * (sizeof(int4) + (size_t)p.lanes * 2 * p.tile_rows * (HEAD + 2) * sizeof(float));
    return p;
}

template <typename T>
jl_status launch_cc(const Args& a, cudaStream_t st) {
    const dim3 grid(a.workers, a.lanes);
    if (a.tile_rows == 16) return launch_pdl(k_tree_attn_cc<T, 1>, grid, dim3(CC_T), cc_smem<1>(), st, a);
    if (a.tile_rows == 32) return launch_pdl(k_tree_attn_cc<T, 2>, grid, dim3(CC_T), cc_smem<2>(), st, a);
    return launch_pdl(k_tree_attn_cc<T, 4>, grid, dim3(CC_T), cc_smem<4>(), st, a);
}

template <typename T>
jl_status configure_cc() {
    JL_CUDA(cudaFuncSetAttribute(k_tree_attn_cc<T, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cc_smem<1>()));
    JL_CUDA(cudaFuncSetAttribute(k_tree_attn_cc<T, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cc_smem<2>()));
    JL_CUDA(cudaFuncSetAttribute(k_tree_attn_cc<T, 4>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cc_smem<4>()));
    return JL_OK;
}

jl_status configure(int device) {  // once per device
    static std::mutex mu;
    static bool done[64] = {};
    std::lock_guard<std::mutex> g(mu);
    if (device < 64 && done[device]) return JL_OK;
    JL_TRY((configure_cc<float>()));
    JL_TRY((configure_cc<uint16_t>()));
    JL_TRY(tc_configure());
    if (device < 64) done[device] = true;
    return JL_OK;
}

jl_status check_sizes(const jl_tree_attn& a) {
    JL_REFUSE(a.rows < 0 || a.seqs < 0, "tree attention: rows and seqs must not be negative");
    JL_TRY(check_pages(a.pool, true));
    JL_REFUSE(a.q_heads < 1 || a.q_heads % a.pool.kv_heads || a.q_heads / a.pool.kv_heads > 128,
              "tree attention: %d query heads over %d kv heads (a multiple, at most 128 per kv head)", a.q_heads,
              a.pool.kv_heads);
    JL_REFUSE(a.max_nodes < 1 || a.max_nodes > JL_TREE_MAX_NODES, "tree attention: max_nodes must be 1..%d, got %d",
              JL_TREE_MAX_NODES, a.max_nodes);
    JL_REFUSE(a.dtype != JL_KV_BF16 && a.dtype != JL_KV_F32, "tree attention: dtype must be bf16 or f32");
    return JL_OK;
}

}  // namespace

jl_status tree_attention(const jl_tree_attn& a, cudaStream_t st) {
    JL_TRY(check_sizes(a));
    JL_REFUSE(!a.q || !a.out || !a.row_start || !a.ctx || !a.page_table,
              "tree attention: q, out, row_start, ctx and page_table must be non-null");
    const size_t width = (size_t)a.q_heads * HEAD;
    JL_REFUSE(a.q_ld < width || a.out_ld < width || a.q_ld % 8 || a.out_ld % 8,
              "tree attention: q_ld and out_ld must be multiples of 8 and at least %zu", width);
    JL_REFUSE(misaligned(a.q) || misaligned(a.out), "tree attention: q and out must be 16-byte aligned");
    JL_REFUSE(a.q == a.out && a.q_ld != a.out_ld, "tree attention: out over q needs out_ld == q_ld");
    JL_REFUSE(a.mask && (long long)a.mask_words * 64 < a.max_nodes, "tree attention: %d mask words hold fewer than %d nodes",
              a.mask_words, a.max_nodes);
    JL_REFUSE(a.max_pages < 1 || a.max_pages > MAX_TABLE, "tree attention: max_pages must be 1..%d", MAX_TABLE);
    JL_REFUSE((long long)a.seqs * a.pool.kv_heads * (a.max_pages + SEG) >= (1ll << 31),
              "tree attention: seqs * kv heads * max_pages must stay below 2^31");
    JL_REFUSE(!(a.scale >= 0.f) || std::isinf(a.scale), "tree attention: scale must be finite and not negative");
    if (a.rows == 0 || a.seqs == 0) return JL_OK;
    DeviceOf on;
    JL_TRY(on.enter(a.pool.k, "tree attention: pool.k"));
    JL_TRY(configure(on.device));
    const Plan p = plan_of(a, on.sms);
    JL_REFUSE(p.bytes && (!a.workspace || ((uintptr_t)a.workspace & 255)),
              "tree attention: the workspace must be 256-byte aligned device memory");
    JL_REFUSE(a.workspace_bytes < p.bytes, "tree attention: workspace of %zu bytes, %zu needed", a.workspace_bytes, p.bytes);
    Args k{};
    k.q = a.q;
    k.out = a.out;
    k.lse = a.lse;
    k.q_ld = (long long)a.q_ld;
    k.out_ld = (long long)a.out_ld;
    k.rows = a.rows;
    k.q_heads = a.q_heads;
    k.kv_heads = a.pool.kv_heads;
    k.group = a.q_heads / a.pool.kv_heads;
    k.seqs = a.seqs;
    k.max_nodes = a.max_nodes;
    k.row_start = a.row_start;
    k.ctx = a.ctx;
    k.mask = a.mask;
    k.mask_words = a.mask_words;
    k.page_table = a.page_table;
    k.max_pages = a.max_pages;
    k.pages = a.pool.pages;
    k.k = a.pool.k;
    k.v = a.pool.v;
    k.c2 = (float)((a.scale == 0.f ? 1.0 / std::sqrt((double)HEAD) : (double)a.scale) * 1.4426950408889634);
    k.workers = p.workers;
    k.lanes = p.lanes;
    k.tile_rows = p.tile_rows;
    k.min_units = p.min_units;
    k.whole = p.whole;
    k.ws_join = (int4*)a.workspace;
    k.ws_o = (float*)(k.ws_join + p.workers);
    k.ws_ml = k.ws_o + (size_t)p.workers * p.lanes * 2 * p.tile_rows * HEAD;
    k.status = a.status;
    const bool f = a.dtype == JL_KV_F32;
    if (a.pool.dtype == JL_KV_BF16) JL_TRY(tc_launch(k, f, st));
    else JL_TRY((f ? launch_cc<float>(k, st) : launch_cc<uint16_t>(k, st)));
    if (p.bytes) {
        // all blocks resident, at most one per row there may be
        const long long most = (long long)(p.workers - 1) * a.max_nodes * k.group;
        const dim3 grid((unsigned)std::min<long long>((long long)CB_PER_SM * on.sms, most));
        JL_TRY((f ? launch_pdl(k_tree_combine<float>, grid, dim3(CB_T), 0, st, k)
                  : launch_pdl(k_tree_combine<uint16_t>, grid, dim3(CB_T), 0, st, k)));
    }
    return JL_OK;
}

jl_status tree_attention_workspace(const jl_tree_attn& a, size_t* bytes) {
    JL_TRY(check_sizes(a));
    DeviceOf on;
    JL_TRY(on.enter(a.pool.k, "tree attention: pool.k"));
    *bytes = plan_of(a, on.sms).bytes;
    return JL_OK;
}

}  // namespace tree
}  // namespace jl
