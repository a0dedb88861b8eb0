// Host checks of the operators that work on device memory the caller owns.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "jl_internal.h"

namespace jl {

// Refuses a call's arguments with a message.
#define JL_REFUSE(cond, ...)           \
    do {                               \
        if (cond) {                    \
            ::jl::set_error(__VA_ARGS__); \
            return JL_ERR_INVALID_ARG; \
        }                              \
    } while (0)

constexpr int MAX_TABLE = 1 << 24;  // pages of one sequence: positions fit 32 bits

inline bool misaligned(const void* p, uintptr_t to = 16) { return ((uintptr_t)p & (to - 1)) != 0; }
// Whether any of the arrays of 32-bit numbers is not aligned as such.
template <typename... P>
bool words_misaligned(P... p) {
    return (misaligned(p, 4) || ...);
}

// A pool's description; `one` for calls that work on one layer.
jl_status check_pages(const jl_kv_pages& p, bool one);

// Makes the device of a device pointer current for the call and restores the
// previous one when it goes out of scope.
struct DeviceOf {
    int device = 0, prev = -1, sms = 148;
    jl_status enter(const void* p, const char* what);
    ~DeviceOf() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

jl_status qk_norm_rope(const jl_norm_rope& a, cudaStream_t st);
jl_status kv_compact(const jl_kv_compaction& a, cudaStream_t st);
jl_status kv_copy_pages(const jl_kv_pages& pool, const int32_t* src, const int32_t* dst, const int32_t* rows, size_t n,
                        cudaStream_t st);

namespace tree {
jl_status tree_attention(const jl_tree_attn& a, cudaStream_t st);
jl_status tree_attention_workspace(const jl_tree_attn& a, size_t* bytes);
}  // namespace tree

}  // namespace jl
