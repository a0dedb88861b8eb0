// Norms of queries and keys for each head, their rotation and the append to
// the pages of the cache, in one pass over q|k|v rows the caller owns
// (jl_qk_norm_rope; lib.rs:291-321, 363-396).  k_qk_rope_kv does the same
// inside the engine's own passes, where a row's rotation position is also its
// place in the cache.
#include <cuda_bf16.h>

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

// Four values as they lie in memory.
template <typename T>
struct Quad;
template <>
struct Quad<float> {
    float4 v;
    __device__ float4 get() const { return v; }
    __device__ static Quad of(float4 x) { return {x}; }
};
template <>
struct Quad<uint16_t> {
    uint2 v;
    __device__ float4 get() const {
        return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                           __uint_as_float(v.y & 0xffff0000u));
    }
    __device__ static Quad of(float4 x) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
        return {make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b))};
    }
};
template <typename T>
__device__ __forceinline__ Quad<T> load(const T* p) {
    return *(const Quad<T>*)p;
}
template <typename T>
__device__ __forceinline__ void store(T* p, float4 x) {
    *(Quad<T>*)p = Quad<T>::of(x);
}

__device__ __forceinline__ float4 mul(float4 a, float4 b) { return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w); }
__device__ __forceinline__ float4 fma4(float4 a, float4 b, float4 c) {
    return make_float4(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y), fmaf(a.z, b.z, c.z), fmaf(a.w, b.w, c.w));
}
__device__ __forceinline__ float square(float4 a, float s) {
    return fmaf(a.x, a.x, fmaf(a.y, a.y, fmaf(a.z, a.z, fmaf(a.w, a.w, s))));
}

// A warp takes 2 * STEPS heads of a row, two side by side: lane p of a head's 16
// holds dims 4 p .. and 64 + 4 p .., the two halves of four rotations, so that
// only the sum of squares crosses lanes.  All heads are loaded before the first
// is used: the row's position, slot, page and angles are looked up while they
// are on their way.  Bound by memory: B200, 12001 f32 rows of 32 heads, 56.3 us
// (6.2 TB/s, 95% of the measured copy rate); 2048 bf16 rows of 48 heads, 14.1 us
// (3.7 TB/s: the lookups' two trips to memory are a good part of it).
constexpr int NR_WARPS = 8;

template <typename T, typename KV, int STEPS>
__global__ void __launch_bounds__(32 * NR_WARPS, 4) k_norm_rope_rows(RowArgs a) {
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    const int lane = threadIdx.x & 31, d = 4 * (lane & 15);
    const int heads = a.q_heads + 2 * a.kv_heads, per_row = (heads + 2 * STEPS - 1) / (2 * STEPS);
    const unsigned unit = blockIdx.x * NR_WARPS + (threadIdx.x >> 5);
    const int row = (int)(unit / (unsigned)per_row), h0 = (int)(unit - (unsigned)row * per_row) * (2 * STEPS) + (lane >> 4);
    if (row >= a.rows) return;
    const T* src = (const T*)a.qkv + (size_t)row * a.qkv_ld + (size_t)h0 * HEAD + d;
    Quad<T> lo[STEPS], hi[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
        if (h0 + 2 * s < heads) {
            lo[s] = load(src + 2 * s * HEAD);
            hi[s] = load(src + 2 * s * HEAD + HALF);
        }
    const int pos = a.pos[row];
    const int slot = a.slot ? a.slot[row] : pos, seq = a.seq ? a.seq[row] : 0;
    const bool first = h0 == 0 && lane == 0;
    if (pos < 0 || pos >= a.positions) {
        if (first && a.status) atomicOr(a.status, 2);
        return;
    }
    const float4 t0 = *(const float4*)(a.rope + (size_t)pos * 2 * HALF + 2 * d), t1 = *(const float4*)(a.rope + (size_t)pos * 2 * HALF + 2 * d + 4);
    // where the row's keys and values go (place < 0: nowhere)
    long long place = -1;
    if (slot >= 0) {
        int bad = 0;
        if ((unsigned)seq >= (unsigned)a.seqs || slot / PAGE >= a.max_pages) {
            bad = 2;
        } else {
            const int page = a.page_table[(size_t)seq * a.max_pages + slot / PAGE];
            if ((unsigned)page < (unsigned)a.pages) place = ((long long)page * a.kv_heads * PAGE + slot % PAGE) * HEAD + d;
            else bad = 1;
        }
        if (bad && first && a.status) atomicOr(a.status, bad);
    }
    const float4 c = make_float4(t0.x, t0.z, t1.x, t1.z), sn = make_float4(t0.y, t0.w, t1.y, t1.w);
    const float4 ns = make_float4(-sn.x, -sn.y, -sn.z, -sn.w);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int h = h0 + 2 * s;
        const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
        if (h < heads) x = lo[s].get(), y = hi[s].get();
        float ss = square(x, square(y, 0.f));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (h >= heads) continue;
        if (!is_v) {
            const uint16_t* w = is_q ? a.qn : a.kn;
            if (w) {
                const float inv = rsqrtf(fmaf(ss, 1.f / HEAD, a.eps));
                const float4 i4 = make_float4(inv, inv, inv, inv);
                x = mul(mul(x, i4), load(w + d).get());
                y = mul(mul(y, i4), load(w + d + HALF).get());
            }
            const float4 u = fma4(x, c, mul(y, ns));
            y = fma4(y, c, mul(x, sn));
            x = u;
        }
        if (is_q) {
            T* q = (T*)a.q + (size_t)row * a.q_ld + (size_t)h * HEAD + d;
            store(q, x);
            store(q + HALF, y);
        } else if (place >= 0) {
            KV* to = (KV*)(is_v ? a.v : a.k) + place + (size_t)(is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads) * PAGE * HEAD;
            store(to, x);
            store(to + HALF, y);
        }
    }
}

template <typename T, typename KV>
jl_status launch_rows(const RowArgs& a, int sms, cudaStream_t st) {
    const int heads = a.q_heads + 2 * a.kv_heads;
    // Few rows: a step of heads to a warp, for latency; many: four steps, so that
    // a warp has 2 KB on the way and looks a row's places up less often.
    auto go = [&](auto kernel, int steps) {
        const long long per_row = (heads + 2 * steps - 1) / (2 * steps);
        const long long blocks = (a.rows * per_row + NR_WARPS - 1) / NR_WARPS;
        JL_REFUSE(blocks >= (1ll << 28), "norm and rotation: too many rows and heads");
        return launch_pdl(kernel, dim3((unsigned)blocks), dim3(32 * NR_WARPS), 0, st, a);
    };
    if ((long long)a.rows * heads < 64ll * sms) return go(k_norm_rope_rows<T, KV, 1>, 1);
    return go(k_norm_rope_rows<T, KV, 4>, 4);
}

}  // namespace

jl_status qk_norm_rope(const jl_norm_rope& a, cudaStream_t st) {
    JL_REFUSE(a.rows < 0, "norm and rotation: rows must not be negative");
    JL_TRY(check_pages(a.pool, true));
    JL_REFUSE(a.q_heads < 1, "norm and rotation: at least one query head");
    JL_REFUSE(a.dtype != JL_KV_BF16 && a.dtype != JL_KV_F32, "norm and rotation: dtype must be bf16 or f32");
    if (a.rows == 0) return JL_OK;
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
    JL_REFUSE(words_misaligned(a.pos, a.slot, a.seq, a.page_table, a.status),
              "norm and rotation: pos, slot, seq, page_table and status must be 4-byte aligned");
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
