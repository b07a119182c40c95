// ebx_kv_check.h -- what the extern "C" entries of the cache and of rotary positions have in common: errors,
// the device that a call is for, and the checks of its pools and rows.
#pragma once

#include <cuda_runtime.h>

#include <string>

#include "../../include/ebx.h"
#include "ebx_internal.h"
#include "ebx_kv.h"

namespace {

inline ebx_status invalid(const char* msg) {
    ebx::set_error(msg);
    return EBX_ERR_INVALID;
}

inline ebx_status launched(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return EBX_OK;
    ebx::set_error(std::string("CUDA error: ") + cudaGetErrorString(e) + " in " + what);
    return EBX_ERR_CUDA;
}

// Makes `dev` current and restores the caller's device on scope exit.
struct Device {
    int prev = -1;
    cudaError_t err;
    explicit Device(int dev) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != dev) err = cudaSetDevice(dev);
        else if (err == cudaSuccess) prev = -1;
    }
    ~Device() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

inline int log2_of(int block_size) {
    for (int s = 4; s <= 7; ++s)
        if (block_size == 1 << s) return s;
    return -1;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Null on success, else what is wrong with the pool.
inline const char* pool_of(const ebx_kv_pool* p, ebx::KvPool& out) {
    if (!p || !p->k_codes || !p->k_scales || !p->v_codes || !p->v_scales) return "null argument";
    if (log2_of(p->block_size) < 0) return "kv pool: block_size must be 16, 32, 64 or 128";
    if (p->head_dim != 32 && p->head_dim != 64 && p->head_dim != 128)
        return "kv pool: head_dim must be 32, 64 or 128";
    if (p->blocks < 1 || p->kv_heads < 1 ||
        int64_t(p->blocks) * p->kv_heads > int64_t(INT32_MAX) / p->block_size)
        return "kv pool: need blocks, kv_heads >= 1 and blocks * kv_heads * block_size < 2^31";
    if (!aligned16(p->k_codes) || !aligned16(p->v_codes)) return "kv pool: codes must be 16-byte aligned";
    out = ebx::KvPool{static_cast<int8_t*>(p->k_codes), p->k_scales, static_cast<int8_t*>(p->v_codes),
                      p->v_scales, p->blocks, p->kv_heads, p->block_size, p->head_dim,
                      log2_of(p->block_size)};
    return nullptr;
}

inline const char* rows_of(const void* p, int64_t token_stride, int64_t head_stride, ebx::KvRows& out) {
    if (!p) return "null argument";
    if (!aligned16(p) || token_stride % 8 != 0 || head_stride % 8 != 0)
        return "kv rows: need a 16-byte aligned base and strides that are multiples of 8 elements";
    out = ebx::KvRows{static_cast<const uint16_t*>(p), token_stride, head_stride};
    return nullptr;
}

}  // namespace
