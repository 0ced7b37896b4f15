// Rows of fp32, fp16 and bf16 in device memory: loads and stores through fp32,
// and the checks that the entry points taking such rows share.
#pragma once

#include <cuda_bf16.h>

#include "kv_internal.cuh"
#include "row_span.h"

namespace qkv {
namespace {

// four consecutive values of a row, in fp32
__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load4(const __half *p) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    return make_float4(h2f((uint16_t)w.x), h2f((uint16_t)(w.x >> 16)), h2f((uint16_t)w.y), h2f((uint16_t)(w.y >> 16)));
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16 *p) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xFFFF0000u));
}
__device__ __forceinline__ void store4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store4(__half *p, float4 v) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack_h2(v.x, v.y), pack_h2(v.z, v.w));
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, float4 v) {
    __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
}

// Two fp32 values in one instruction.  A packed sum of packed products may be
// contracted to one rounding, so sums that must not be are made one by one.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p));
}
__device__ __forceinline__ void unpair(uint64_t p, uint32_t &lo, uint32_t &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(p));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2_down(uint64_t a, uint64_t b) {  // towards zero
    uint64_t r;
    asm("add.rz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// launch a kernel that may start while the stream's previous one still runs (it
// waits for it itself) and lets the next one start
template <typename... Params, typename... Args>
cudaError_t launch_next(void (*kernel)(Params...), dim3 grid, dim3 block, cudaStream_t s, Args &&...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    note_early_trigger();
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
    if (e == cudaSuccess) count_launch();
    else cudaGetLastError();  // reported here, not by a later launch
    return e;
}

inline bool dtype_ok(uint32_t d) { return d == QWN_DTYPE_F32 || d == QWN_DTYPE_F16 || d == QWN_DTYPE_BF16; }
inline uint64_t value_bytes(uint32_t dtype) { return dtype == QWN_DTYPE_F32 ? 4 : 2; }
// rows start on `values` values
inline bool rows_aligned(const void *p, uint64_t stride, uint32_t dtype, uint64_t values = 4) {
    return (uintptr_t)p % (value_bytes(dtype) * values) == 0 && stride % values == 0;
}
// 16-byte accesses
inline bool rows_wide(const void *p, uint64_t stride, uint32_t dtype) {
    return rows_aligned(p, stride, dtype, 16 / value_bytes(dtype));
}
inline int invalid(const char *msg) {
    set_error(msg);
    return QWN_CUDA_STATUS_INVALID_ARGUMENT;
}

}  // namespace
}  // namespace qkv
