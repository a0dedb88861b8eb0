// Attention of the nodes of drafted trees over the paged cache
// (jl_tree_attention): host checks and the kernel that adds the partial results
// of items that several workers share.  The attention itself: tree_attn_tc.cu.
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

template <typename T>
__global__ void __launch_bounds__(CB_T, CB_PER_SM) k_tree_combine(Args a) {
    __shared__ float4 share_o[CB_WARPS][32];
    __shared__ float2 share_ml[CB_WARPS];
    __shared__ int before[CB_MOST + 1];  // groups of rows (CB_ROWS or one) before item i
    __shared__ short who[CB_MOST];       // item i is ws_join[who[i]], kept in joins[i]
    __shared__ int4 joins[CB_MOST];
    __shared__ int2 warp_sums[CB_WARPS];
    const int t = threadIdx.x, warp = t >> 5, l = t & 31;
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    // items and their groups of rows: thread t's workers are CB_EACH t ..
    int some = 0, groups = 0, mine[CB_EACH];
    int4 join[CB_EACH];
#pragma unroll
    for (int e = 0; e < CB_EACH; ++e) {
        const int w = t * CB_EACH + e;
        join[e] = w > 0 && w < a.workers ? a.ws_join[w] : make_int4(0, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < CB_EACH; ++e) {
        const int rows = join[e].w > 0 ? join[e].y * a.group : 0;
        mine[e] = join[e].w >= CB_SHARE ? rows : (rows + CB_ROWS - 1) / CB_ROWS;
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
            joins[item] = join[e];
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
        const int4 join = joins[item];
        const int rows = join.y * a.group, parts = join.w, at = i - before[item];
        // partial x of query row g: worker w - 1's slot 1, then slot 0 of the workers from w on
        auto slot = [&](int x, int g) {
            const int lane = g / R;
            return ((size_t)((w - 1 + x) * a.lanes + lane) * 2 + (x == 0 ? 1 : 0)) * R + (g - lane * R);
        };
        auto finish = [&](const RowSum& sum, int g) { finish_row<T>(a, join.x, join.z, g, l, sum, inv_group); };
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

// What a device allows, found once.
jl_status limits_of(int device, TcLimits& out) {
    static std::mutex mu;
    static TcLimits found[64];
    static bool done[64] = {};
    std::lock_guard<std::mutex> g(mu);
    if (device >= 64 || !done[device]) {
        JL_TRY(tc_configure(out));
        if (device >= 64) return JL_OK;
        found[device] = out;
        done[device] = true;
    }
    out = found[device];
    return JL_OK;
}

// How a call cuts the work: whole items (parts 1), items shared by clusters of
// `parts` CTAs, or even ranges of units.
struct Plan {
    int tile_rows, lanes, workers, min_units, whole, parts;
    int slots;  // of ws_o for each CTA: 2 partial results, 1 for sums over runs of pages, 0 none
    size_t bytes;
};

Plan plan_of(const jl_tree_attn& a, int sms, const TcLimits& limits) {
    Plan p;
    const int rows = a.max_nodes * (a.q_heads / a.pool.kv_heads);
    const bool rows_f32 = a.dtype == JL_KV_F32, pool_f32 = a.pool.dtype == JL_KV_F32;
    p.tile_rows = tc_tile_rows(rows_f32);
    p.lanes = (rows + p.tile_rows - 1) / p.tile_rows;
    p.workers = std::min(CB_MOST, std::max(1, tc_ctas(pool_f32) * sms / p.lanes));
    p.parts = 1;
    // Whole items or shared ones: the longest item sets the time, whose parts are
    // added within a cluster.  Even ranges: the mean does (of a batch it is taken as
    // 0.8 of the longest), but the join is a kernel of its own, and starts and ends
    // of segments add up.  Times in us on a B200, fitted to calls of 32 heads over 8:
    // of a page with one CTA an SM and with two, of a CTA's start and end, and of
    // even ranges, which grow with the rows of a tile.  Measured, whole / 8 parts /
    // even: one sequence of 8 bf16 nodes at 100 positions 7.5 / 9.0 / 13.0 us, at 300
    // 11.0 / 8.6 / 14.5, at 1500 35.5 / 11.0 / 14.3, at 12000 257 / 41 / 24; four of 32
    // nodes at 4096 97 / 30 / 44; eight of 8 nodes at 1500, four parts, 39 / 20 / 28;
    // f32 rows and pool, four of 8 nodes at 1500, four parts, 84 / 32 / 44.
    const double one = pool_f32 ? 3.0 : rows_f32 ? 1.4 : 1.35, two = pool_f32 ? 3.0 : rows_f32 ? 2.0 : 1.65;
    const int r = std::min(rows, p.tile_rows);
    const double start = (pool_f32 ? 6.0 : rows_f32 ? 7.2 : 5.2) + 0.025 * r;
    const double ctas = (double)a.seqs * a.pool.kv_heads * p.lanes, slots = (double)p.workers * p.lanes;
    const double units = std::max(ctas * (a.max_pages + SEG) / slots * (a.seqs > 1 ? 0.8 : 1.0), 1.0 + SEG);
    const double even = (pool_f32 ? 12.0 : rows_f32 ? 10.5 : 9.0) + 0.12 * r + units * (pool_f32 ? 4.4 : rows_f32 ? 2.2 : 1.9);
    double best = std::ceil(ctas / slots) * (start + a.max_pages * (ctas > sms ? two : one));
    p.whole = best <= even;
    for (int i = 0, n = 2; i < TcLimits::SIZES; ++i, n *= 2) {
        const double shared = start + 1.5 + std::ceil((double)a.max_pages / n) * (ctas * n > sms ? two : one);
        if (ctas > limits.clusters[rows_f32][pool_f32][i] || shared >= std::min(best, even)) continue;
        best = shared;
        p.parts = n;
        p.whole = 1;
    }
    const bool any = a.seqs == 0 || a.max_pages == 0;  // the workspace of any call is asked for
    if (any) p.whole = 0, p.parts = 1;
    if (p.parts > 1) p.workers = a.seqs * a.pool.kv_heads;
    p.min_units = p.whole ? 1 : 1 + SEG;
    const size_t tile = (size_t)p.tile_rows * sizeof(float);
    p.slots = p.workers > 1 && !p.whole ? 2 : (a.max_pages + p.parts - 1) / p.parts > tc_run(rows_f32, pool_f32) ? 1 : 0;
    p.bytes = p.slots == 2   ? (size_t)p.workers * (sizeof(int4) + p.lanes * 2 * tile * (HEAD + 2))
              : p.slots == 1 ? (size_t)p.workers * p.parts * p.lanes * tile * HEAD
                             : 0;
    if (any) p.bytes = std::max(p.bytes, (size_t)std::max(p.workers * p.lanes, tc_ctas(pool_f32) * sms) * tile * HEAD);
    return p;
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
    if (a.rows == 0 || a.seqs == 0) return JL_OK;
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
    JL_REFUSE(misaligned(a.mask, 8) || words_misaligned(a.lse, a.row_start, a.ctx, a.page_table, a.status),
              "tree attention: mask must be 8-byte aligned, lse, row_start, ctx, page_table and status 4-byte aligned");
    DeviceOf on;
    JL_TRY(on.enter(a.pool.k, "tree attention: pool.k"));
    TcLimits limits;
    JL_TRY(limits_of(on.device, limits));
    const Plan p = plan_of(a, on.sms, limits);
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
    k.parts = p.parts;
    k.slots = std::max(p.slots, 1);
    k.ws_join = (int4*)a.workspace;
    k.ws_o = (float*)(k.ws_join + (p.slots == 2 ? p.workers : 0));
    k.ws_ml = k.ws_o + (size_t)p.workers * p.lanes * 2 * p.tile_rows * HEAD;
    k.status = a.status;
    const bool f = a.dtype == JL_KV_F32;
    JL_TRY(tc_launch(k, f, a.pool.dtype == JL_KV_F32, st));
    if (p.slots == 2) {
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
    TcLimits limits;
    JL_TRY(limits_of(on.device, limits));
    *bytes = plan_of(a, on.sms, limits).bytes;
    return JL_OK;
}

}  // namespace tree
}  // namespace jl
