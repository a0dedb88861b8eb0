// Norms of queries and keys for each head, their rotation and the append to
// the pages of the cache, in one pass over q|k|v rows the caller owns
// (jl_qk_norm_rope; lib.rs:291-321, 363-396).  k_qk_rope_kv does the same
// inside the engine's own passes, where a row's rotation position is also its
// place in the cache.
#include <algorithm>

#include "kernels.cuh"
#include "launch.cuh"
#include "ops_host.h"
#include "ptx.cuh"

namespace jl {
namespace {

struct RowArgs {
    const void* qkv;
    void* q;
    long long qkv_ld, q_ld;
    int rows, q_heads, kv_heads, seqs, max_pages, pages, positions;
    const uint16_t* qn;
    const uint16_t* kn;
    float eps;
    const float* rope;
    const int32_t* pos;
    const int32_t* slot;
    const int32_t* seq;
    const int32_t* page_table;
    void* k;
    void* v;
    int32_t* status;
};

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

constexpr int NR_WARPS = 8;

// Block (row, y): the row's heads 8 y + warp, then every 8 * gridDim.y on.
// Lane l holds dims 4 l .. 4 l + 3 of a head; the dim 64 away that its
// rotation needs is in lane l ^ 16.
template <typename T, typename KV>
__global__ void __launch_bounds__(32 * NR_WARPS) k_norm_rope_rows(RowArgs a) {
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pos = a.pos[row];
    if (pos < 0 || pos >= a.positions) {
        if (threadIdx.x == 0 && a.status) atomicOr(a.status, 2);
        return;
    }
    // where the row's keys and values go (place < 0: nowhere)
    const int slot = a.slot ? a.slot[row] : pos, seq = a.seq ? a.seq[row] : 0;
    long long place = -1;
    if (slot >= 0) {
        int bad = 0;
        if ((unsigned)seq >= (unsigned)a.seqs || slot / PAGE >= a.max_pages) {
            bad = 2;
        } else {
            const int page = a.page_table[(size_t)seq * a.max_pages + slot / PAGE];
            if ((unsigned)page < (unsigned)a.pages) place = ((long long)page * a.kv_heads * PAGE + slot % PAGE) * HEAD;
            else bad = 1;
        }
        if (bad && threadIdx.x == 0 && a.status) atomicOr(a.status, bad);
    }
    const float4* rope = (const float4*)(a.rope + (size_t)pos * 2 * HALF) + 2 * (lane & 15);
    const float4 r0 = rope[0], r1 = rope[1];  // (cos, sin) of four angles
    const float sign = lane < 16 ? -1.f : 1.f;
    const float4 one = make_float4(1.f, 1.f, 1.f, 1.f);
    const float4 wq = a.qn ? load4(a.qn + 4 * lane) : one, wk = a.kn ? load4(a.kn + 4 * lane) : one;
    const T* src = (const T*)a.qkv + (size_t)row * a.qkv_ld + 4 * lane;
    T* dst = (T*)a.q + (size_t)row * a.q_ld + 4 * lane;
    const int heads = a.q_heads + (place >= 0 ? 2 * a.kv_heads : 0);
    for (int h = blockIdx.y * NR_WARPS + warp; h < heads; h += NR_WARPS * gridDim.y) {
        float4 x = load4(src + (size_t)h * HEAD);
        const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
        if (!is_v) {
            if (is_q ? a.qn != nullptr : a.kn != nullptr) {
                const float ss = warp_sum(fmaf(x.x, x.x, fmaf(x.y, x.y, fmaf(x.z, x.z, x.w * x.w))));
                const float inv = __fdiv_rn(1.f, sqrtf(__fadd_rn(ss * (1.f / HEAD), a.eps)));
                const float4 w = is_q ? wq : wk;
                x = make_float4(x.x * inv * w.x, x.y * inv * w.y, x.z * inv * w.z, x.w * inv * w.w);
            }
            float4 o;
            o.x = __shfl_xor_sync(0xffffffffu, x.x, 16);
            o.y = __shfl_xor_sync(0xffffffffu, x.y, 16);
            o.z = __shfl_xor_sync(0xffffffffu, x.z, 16);
            o.w = __shfl_xor_sync(0xffffffffu, x.w, 16);
            x.x = fmaf(x.x, r0.x, sign * o.x * r0.y);
            x.y = fmaf(x.y, r0.z, sign * o.y * r0.w);
            x.z = fmaf(x.z, r1.x, sign * o.z * r1.y);
            x.w = fmaf(x.w, r1.z, sign * o.w * r1.w);
        }
        if (is_q) {
            store4(dst + (size_t)h * HEAD, x);
        } else {
            const int kvh = is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads;
            store4((KV*)(is_v ? a.v : a.k) + place + (size_t)kvh * PAGE * HEAD + 4 * lane, x);
        }
    }
}

template <typename T, typename KV>
jl_status launch_rows(const RowArgs& a, int sms, cudaStream_t st) {
    // few rows: a warp per head; many: a block per row
    const int heads = a.q_heads + 2 * a.kv_heads, most = (heads + NR_WARPS - 1) / NR_WARPS;
    const int y = std::max(1, std::min(most, 8 * sms / a.rows));
    return launch_pdl(k_norm_rope_rows<T, KV>, dim3(a.rows, y), dim3(32 * NR_WARPS), 0, st, a);
}

}  // namespace

jl_status qk_norm_rope(const jl_norm_rope& a, cudaStream_t st) {
    JL_REFUSE(a.rows < 0, "norm and rotation: rows must not be negative");
    JL_TRY(check_pages(a.pool, true));
    JL_REFUSE(a.q_heads < 1, "norm and rotation: at least one query head");
    JL_REFUSE(a.dtype != JL_KV_BF16 && a.dtype != JL_KV_F32, "norm and rotation: dtype must be bf16 or f32");
    JL_REFUSE(!a.qkv || !a.q || !a.rope || !a.pos || !a.page_table,
              "norm and rotation: qkv, q, rope, pos and page_table must be non-null");
    const size_t in = ((size_t)a.q_heads + 2 * (size_t)a.pool.kv_heads) * HEAD, out = (size_t)a.q_heads * HEAD;
    JL_REFUSE(a.qkv_ld < in || a.qkv_ld % 8, "norm and rotation: qkv_ld must be a multiple of 8 and at least %zu", in);
    JL_REFUSE(a.q_ld < out || a.q_ld % 8, "norm and rotation: q_ld must be a multiple of 8 and at least %zu", out);
    JL_REFUSE(misaligned(a.qkv) || misaligned(a.q) || misaligned(a.rope),
              "norm and rotation: qkv, q and rope must be 16-byte aligned");
    JL_REFUSE(((uintptr_t)a.q_norm & 7) || ((uintptr_t)a.k_norm & 7),
              "norm and rotation: the norm weights must be 8-byte aligned");
    JL_REFUSE(a.q == a.qkv && a.q_ld != a.qkv_ld, "norm and rotation: q over qkv needs q_ld == qkv_ld");
    JL_REFUSE(a.seqs < 1 || a.max_pages < 1 || a.max_pages > MAX_TABLE,
              "norm and rotation: at least one sequence and 1..%d pages each", MAX_TABLE);
    JL_REFUSE(a.positions < 1, "norm and rotation: at least one position in the rotation table");
    JL_REFUSE(!(a.eps >= 0.f), "norm and rotation: eps must not be negative");
    if (a.rows == 0) return JL_OK;
    DeviceOf on;
    JL_TRY(on.enter(a.pool.k, "norm and rotation: pool.k"));
    RowArgs k{a.qkv,  a.q,        (long long)a.qkv_ld, (long long)a.q_ld, a.rows, a.q_heads, a.pool.kv_heads, a.seqs, a.max_pages,
              a.pool.pages, a.positions, a.q_norm,       a.k_norm,          a.eps,  a.rope,    a.pos,           a.slot, a.seq,
              a.page_table, a.pool.k, a.pool.v, a.status};
    const bool kf = a.pool.dtype == JL_KV_F32;
    if (a.dtype == JL_KV_F32)
        return kf ? launch_rows<float, float>(k, on.sms, st) : launch_rows<float, uint16_t>(k, on.sms, st);
    return kf ? launch_rows<uint16_t, float>(k, on.sms, st) : launch_rows<uint16_t, uint16_t>(k, on.sms, st);
}

}  // namespace jl
