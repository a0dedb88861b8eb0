// Moving rows and pages of the paged cache on the device: compaction after a
// tree of drafted tokens was verified (jl_kv_compact) and copies of pages
// (jl_kv_copy_pages).  Both move every layer in one launch and are bound by
// the bytes they read and write.
#include <algorithm>
#include <cstring>
#include <vector>

#include "kernels.cuh"
#include "launch.cuh"
#include "ops_host.h"
#include "ptx.cuh"

namespace jl {

jl_status check_pages(const jl_kv_pages& p, bool one) {
    JL_REFUSE(!p.k || !p.v, "pool: k and v must be non-null");
    JL_REFUSE(misaligned(p.k) || misaligned(p.v), "pool: k and v must be 16-byte aligned");
    JL_REFUSE(p.dtype != JL_KV_BF16 && p.dtype != JL_KV_F32, "pool: dtype must be bf16 or f32");
    JL_REFUSE(p.pages < 1 || p.kv_heads < 1 || p.kv_heads > 1024, "pool: at least one page and 1..1024 kv heads");
    JL_REFUSE((long long)p.pages * p.kv_heads * PAGE >= (1ll << 31), "pool: pages * kv_heads * 64 must stay below 2^31");
    JL_REFUSE(one ? p.layers != 1 : p.layers < 1 || p.layers > 4096,
              one ? "pool: this call works on one layer" : "pool: 1..4096 layers");
    const size_t bytes = (size_t)p.pages * p.kv_heads * PAGE * HEAD * (p.dtype == JL_KV_F32 ? 4 : 2);
    JL_REFUSE(p.layers > 1 && (p.layer_stride % 16 || p.layer_stride < bytes),
              "pool: layer_stride must be a multiple of 16 and at least one layer's %zu bytes", bytes);
    return JL_OK;
}

jl_status DeviceOf::enter(const void* p, const char* what) {
    cudaPointerAttributes at;
    JL_CUDA(cudaPointerGetAttributes(&at, p));
    JL_REFUSE(at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged, "%s is not device memory", what);
    device = at.device;
    int now = 0;
    JL_CUDA(cudaGetDevice(&now));
    if (now != device) {
        JL_CUDA(cudaSetDevice(device));
        prev = now;
    }
    JL_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    return JL_OK;
}

namespace {

struct CompactArgs {
    uint8_t* k;
    uint8_t* v;
    size_t layer_stride;
    int kv_heads, pages, seqs, path_ld, max_pages, row_bytes;
    const int32_t* ctx;
    const int32_t* path;
    const int32_t* path_len;
    const int32_t* page_table;
    int32_t* status;
};

// Offset of a sequence's position within a layer's pages (head 0), or -1.
__device__ __forceinline__ long long place(const CompactArgs& a, int s, long long p, int* bad) {
    if (p < 0 || p >= (long long)a.max_pages * PAGE) {
        *bad |= 2;
        return -1;
    }
    const int page = a.page_table[(size_t)s * a.max_pages + p / PAGE];
    if ((unsigned)page >= (unsigned)a.pages) {
        *bad |= 1;
        return -1;
    }
    return ((long long)page * a.kv_heads * PAGE + p % PAGE) * a.row_bytes;
}

// Block (y, sequence): a warp moves the rows of one slab (a kv head's K or V of
// one layer) after the other.  BATCH rows are read into registers before any of
// them is written; with at most BATCH rows the order of the path and repeated
// entries then do not matter.  A longer path is moved batch by batch, which is
// right as long as no batch reads a row that an earlier one wrote (a tree's
// path: entry i is node i or later); a path that does (or may) goes through
// shared memory whole, slab by slab.  The places of the rows are looked up once
// a block.  Bound by memory for many slabs and by the lookups' latency for few:
// B200, 36 layers of 8 heads, 32 sequences of 5 to 9 rows 16.3 us (4.3 TB/s of
// scattered 256-byte rows), one sequence of 4 rows 2.6 us.
constexpr int CP_WARPS = 4, CP_T = 32 * CP_WARPS, CP_BATCH = 16;

template <int ROW_BYTES>
__global__ void __launch_bounds__(CP_T) k_kv_compact(CompactArgs a, int slabs, int per_block) {
    constexpr int CHUNKS = ROW_BYTES / 16, REGS = CP_BATCH * CHUNKS / 32;
    extern __shared__ uint4 cp_rows[];
    __shared__ long long from[JL_TREE_MAX_NODES], to[JL_TREE_MAX_NODES];
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    const int s = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int n = a.path_len[s];
    int bad = n < 0 || n > a.path_ld ? 2 : 0;
    n = min(max(n, 0), a.path_ld);
    bool back = false;  // an entry reads what an earlier batch may write
    for (int i = threadIdx.x; i < n; i += CP_T) {
        const long long c = a.ctx[s], p = a.path[(size_t)s * a.path_ld + i];
        const bool neg = c < 0 || p < 0;
        if (neg) bad |= 2;
        from[i] = neg ? -1 : place(a, s, c + p, &bad);
        to[i] = neg || p == i ? -1 : place(a, s, c + i, &bad);
        if (from[i] < 0 || to[i] < 0) from[i] = -1;
        // never within the first batch, so paths of one batch need no shared memory
        back |= from[i] >= 0 && p < i / CP_BATCH * CP_BATCH;
    }
    if (bad && a.status) atomicOr(a.status, bad);
    back = __syncthreads_or(back);
    const int slab0 = blockIdx.x * per_block, slab1 = min(slabs, slab0 + per_block);
    auto base_of = [&](int slab) {  // slab = (2 * layer + K|V) * kv_heads + head
        const int lk = slab / a.kv_heads;
        return (lk & 1 ? a.v : a.k) + (size_t)(lk >> 1) * a.layer_stride + (size_t)(slab - lk * a.kv_heads) * PAGE * ROW_BYTES;
    };
    if (back) {
        for (int slab = slab0; slab < slab1; ++slab) {
            uint8_t* base = base_of(slab);
            for (int i = threadIdx.x; i < n * CHUNKS; i += CP_T)
                if (from[i / CHUNKS] >= 0) cp_rows[i] = *(const uint4*)(base + from[i / CHUNKS] + 16 * (i % CHUNKS));
            __syncthreads();
            for (int i = threadIdx.x; i < n * CHUNKS; i += CP_T)
                if (from[i / CHUNKS] >= 0) *(uint4*)(base + to[i / CHUNKS] + 16 * (i % CHUNKS)) = cp_rows[i];
            __syncthreads();
        }
        return;
    }
    for (int slab = slab0 + warp; slab < slab1; slab += CP_WARPS) {
        uint8_t* base = base_of(slab);
        for (int r0 = 0; r0 < n; r0 += CP_BATCH) {
            uint4 v[REGS];
#pragma unroll
            for (int k = 0; k < REGS; ++k) {
                const int i = k * 32 + lane, r = r0 + i / CHUNKS;
                if (r < n && from[r] >= 0) v[k] = *(const uint4*)(base + from[r] + 16 * (i % CHUNKS));
            }
            __syncwarp();  // all lanes have read before one writes
#pragma unroll
            for (int k = 0; k < REGS; ++k) {
                const int i = k * 32 + lane, r = r0 + i / CHUNKS;
                if (r < n && from[r] >= 0) *(uint4*)(base + to[r] + 16 * (i % CHUNKS)) = v[k];
            }
            __syncwarp();
        }
    }
}

// Pairs of one launch, in kernel parameters: nothing to upload or to keep
// alive, and a captured launch carries its own.
template <int N>
struct CopyList {
    int2 pair[N];
    uint8_t rows[N];
};

constexpr int CY_T = 256;
// Block (kv head, pair, 2 * layer + K|V): one head's rows of a page, which lie
// together (16 KB in bf16).  Bound by memory: B200, 64 pages of 8 heads in 36
// layers, 166 us (6.8 TB/s read and written, the measured copy rate).
template <int N>
__global__ void __launch_bounds__(CY_T) k_kv_copy(uint8_t* k, uint8_t* v, size_t layer_stride, int kv_heads, int row_bytes,
                                                  const __grid_constant__ CopyList<N> list) {
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    const int2 pr = list.pair[blockIdx.y];
    const int chunks = list.rows[blockIdx.y] * row_bytes / 16;
    uint8_t* base = (blockIdx.z & 1 ? v : k) + (size_t)(blockIdx.z >> 1) * layer_stride;
    const size_t slab = (size_t)PAGE * row_bytes;
    const uint4* src = (const uint4*)(base + ((size_t)pr.x * kv_heads + blockIdx.x) * slab);
    uint4* dst = (uint4*)(base + ((size_t)pr.y * kv_heads + blockIdx.x) * slab);
#pragma unroll 4
    for (int i = threadIdx.x; i < chunks; i += CY_T) dst[i] = src[i];
}

template <int N>
jl_status copy_some(const jl_kv_pages& p, const int32_t* src, const int32_t* dst, const int32_t* rows, int n, cudaStream_t st) {
    CopyList<N> list;
    for (int i = 0; i < n; ++i) {
        list.pair[i] = make_int2(src[i], dst[i]);
        list.rows[i] = (uint8_t)(rows ? rows[i] : PAGE);
    }
    const int row_bytes = HEAD * (p.dtype == JL_KV_F32 ? 4 : 2);
    return launch_pdl(k_kv_copy<N>, dim3(p.kv_heads, n, 2 * p.layers), dim3(CY_T), 0, st, (uint8_t*)p.k, (uint8_t*)p.v,
                      p.layer_stride, p.kv_heads, row_bytes, list);
}

}  // namespace

jl_status kv_compact(const jl_kv_compaction& a, cudaStream_t st) {
    JL_TRY(check_pages(a.pool, false));
    JL_REFUSE(a.seqs < 0 || a.seqs > 65535, "compaction: 0..65535 sequences");
    JL_REFUSE(a.path_ld < 1 || a.path_ld > JL_TREE_MAX_NODES, "compaction: path_ld must be 1..%d", JL_TREE_MAX_NODES);
    if (a.seqs == 0) return JL_OK;
    JL_REFUSE(!a.ctx || !a.path || !a.path_len || !a.page_table,
              "compaction: ctx, path, path_len and page_table must be non-null");
    JL_REFUSE(a.max_pages < 1 || a.max_pages > MAX_TABLE, "compaction: max_pages must be 1..%d", MAX_TABLE);
    JL_REFUSE(words_misaligned(a.ctx, a.path, a.path_len, a.page_table, a.status),
              "compaction: ctx, path, path_len, page_table and status must be 4-byte aligned");
    DeviceOf on;
    JL_TRY(on.enter(a.pool.k, "compaction: pool.k"));
    const int row_bytes = HEAD * (a.pool.dtype == JL_KV_F32 ? 4 : 2);
    CompactArgs k{(uint8_t*)a.pool.k, (uint8_t*)a.pool.v, a.pool.layer_stride, a.pool.kv_heads, a.pool.pages, a.seqs,
                  a.path_ld, a.max_pages, row_bytes, a.ctx, a.path, a.path_len, a.page_table, a.status};
    // paths of one batch need no shared memory
    const size_t smem = a.path_ld > CP_BATCH ? (size_t)a.path_ld * row_bytes : 0;
    const int slabs = 2 * a.pool.layers * a.pool.kv_heads;
    // a slab a warp for few slabs; for many, what the resident warps share
    const long long warps = (long long)on.sms * 8 * CP_WARPS;
    const int per_warp = (int)std::max<long long>(1, (long long)slabs * a.seqs / warps);
    const int per_block = per_warp * CP_WARPS;
    const dim3 grid((slabs + per_block - 1) / per_block, a.seqs);
    auto go = [&](auto kernel) -> jl_status {
        if (smem > 40 * 1024)  // the default limit is 48 KB with the static arrays
            JL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, JL_TREE_MAX_NODES * HEAD * 4));
        return launch_pdl(kernel, grid, dim3(CP_T), smem, st, k, slabs, per_block);
    };
    return row_bytes == 256 ? go(k_kv_compact<256>) : go(k_kv_compact<512>);
}

jl_status kv_copy_pages(const jl_kv_pages& pool, const int32_t* src, const int32_t* dst, const int32_t* rows, size_t n,
                        cudaStream_t st) {
    JL_TRY(check_pages(pool, false));
    JL_REFUSE(n && (!src || !dst), "page copy: src and dst must be non-null");
    JL_REFUSE(n > (size_t)pool.pages, "page copy: %zu copies into a pool of %d pages", n, pool.pages);
    std::vector<uint8_t> role(n ? pool.pages : 0);  // 1 source, 2 destination
    for (size_t i = 0; i < n; ++i) {
        JL_REFUSE((unsigned)src[i] >= (unsigned)pool.pages || (unsigned)dst[i] >= (unsigned)pool.pages,
                  "page copy: page %d or %d outside the pool of %d", src[i], dst[i], pool.pages);
        JL_REFUSE(rows && (rows[i] < 1 || rows[i] > PAGE), "page copy: rows must be 1..%d, got %d", PAGE, rows[i]);
        JL_REFUSE(role[dst[i]] & 2, "page copy: page %d is the destination of two copies", dst[i]);
        role[dst[i]] |= 2;
        role[src[i]] |= 1;
    }
    for (size_t i = 0; i < n; ++i)
        JL_REFUSE(role[dst[i]] & 1, "page copy: page %d is both source and destination", dst[i]);
    if (n == 0) return JL_OK;
    DeviceOf on;
    JL_TRY(on.enter(pool.k, "page copy: pool.k"));
    for (size_t at = 0; at < n;) {
        const int32_t* r = rows ? rows + at : nullptr;
        if (n - at <= 64) {
            JL_TRY(copy_some<64>(pool, src + at, dst + at, r, (int)(n - at), st));
            break;
        }
        const int take = (int)std::min<size_t>(n - at, 1024);
        JL_TRY(copy_some<1024>(pool, src + at, dst + at, r, take, st));
        at += take;
    }
    return JL_OK;
}

}  // namespace jl
