// Operators over a caller-owned paged KV pool: what their files share.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <initializer_list>
#include <stdexcept>
#include <string>

#include "q3_common.cuh"

namespace q3 {

// The device that holds a call's pointers, made current for the call's launches. The free operators
// take raw pointers, so this is where a host pointer, or pointers of two devices, are refused before
// a kernel would fault on them. (The look-ups cost well under a microsecond and are allowed while a
// stream is being captured.)
class OnDevice {
public:
    explicit OnDevice(std::initializer_list<const void*> ptrs) {
        int dev = -1;
        for (const void* p : ptrs) {
            if (!p) continue;
            cudaPointerAttributes a{};
            const cudaError_t e = cudaPointerGetAttributes(&a, p);
            if (e != cudaSuccess) {
                cudaGetLastError();  // not left behind for the next call's check
                throw CudaError(std::string("cudaPointerGetAttributes: ") + cudaGetErrorString(e));
            }
            if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) {
                throw std::invalid_argument("a pointer is not device memory");
            }
            if (dev >= 0 && a.device != dev) {
                throw std::invalid_argument("pointers lie on different devices");
            }
            dev = a.device;
        }
        Q3_CUDA(cudaGetDevice(&previous_));
        if (dev >= 0 && dev != previous_) {
            Q3_CUDA(cudaSetDevice(dev));
            switched_ = true;
        }
        device_ = dev >= 0 ? dev : previous_;
    }
    ~OnDevice() {
        if (switched_) cudaSetDevice(previous_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    int device() const { return device_; }
    int sm_count() const {
        int n = 0;
        Q3_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device_));
        return n;
    }

private:
    int device_ = 0, previous_ = 0;
    bool switched_ = false;
};

inline bool aligned(const void* p, size_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

inline void check_pool(const q3_kv_pool* pool) {
    if (!pool) throw std::invalid_argument("KV pool: null");
    if (pool->type != Q3_TYPE_BF16 && pool->type != Q3_TYPE_E4M3) {
        throw std::invalid_argument("KV pool: type must be Q3_TYPE_BF16 or Q3_TYPE_E4M3");
    }
    if (pool->head_dim != 64 && pool->head_dim != 128) {
        throw std::invalid_argument("KV pool: head_dim must be 64 or 128");
    }
    if (pool->n_kv_heads <= 0 || pool->n_kv_heads > 65535) {
        throw std::invalid_argument("KV pool: n_kv_heads out of range");
    }
    if (pool->n_pages <= 0 || pool->n_pages > (int64_t(1) << 27) - 1) {
        throw std::invalid_argument("KV pool: n_pages out of range");
    }
    if (!pool->k || !pool->v) throw std::invalid_argument("KV pool: null pointer");
    if ((pool->type == Q3_TYPE_E4M3) != (pool->exps != nullptr)) {
        throw std::invalid_argument("KV pool: exps belong to an e4m3 pool and to no other");
    }
    if (!aligned(pool->k, 16) || !aligned(pool->v, 16) || !aligned(pool->exps, 4)) {
        throw std::invalid_argument("KV pool: k and v must be 16-byte aligned, exps 4-byte");
    }
}

// 2^(byte - 127); a float's exponent field, but for byte 0 (2^-127 is subnormal).
__device__ __forceinline__ float exp_of_byte(uint32_t byte) {
    return __uint_as_float(max(byte << 23, 0x00400000u));
}

// Two e4m3 codes (the low 16 bits of `pair`) as packed fp16: every e4m3 value is an fp16 value.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t pair) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}"
        : "=r"(r) : "r"(pair));
    return r;
}
// The same for the high 16 bits.
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t pair) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}"
        : "=r"(r) : "r"(pair));
    return r;
}

}  // namespace q3
