// Residual addition, root-mean-square norm and int8 quantisation of rows
// (qwn_rmsnorm_q8), one pass over the data:
//     h = x + r,  y = h / sqrt(mean h^2 + eps) * w,  s = max|y| / 127,
//     code = y / s rounded to nearest even.
// The reference quantises its activations on the host with the same rule
// (c/qwanto_turboquant.c:555-586).
//
// One CTA per row keeps the row in registers between its two reductions (the
// sum of squares, then the largest |y|), so x and r are read once and each
// output is written once; bound by HBM, or by the launch for a few rows.
#include "kv_internal.cuh"
#include "rows.cuh"

namespace qkv {
namespace {

struct NormArgs {
    const void *x, *residual, *weight;
    void *residual_out, *rows_out;
    int8_t *codes;
    float *scales;
    uint64_t x_stride, residual_stride, residual_out_stride, codes_stride, rows_stride;
    uint32_t width, rows_dtype;
    float eps;
    bool norm;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float &d, float x) { d = x; }
__device__ __forceinline__ void from_f(__half &d, float x) { d = __float2half_rn(x); }
__device__ __forceinline__ void from_f(__nv_bfloat16 &d, float x) { d = __float2bfloat16_rn(x); }

// the n values from p on (n < V at the row's end), V in one access where VEC
template <bool VEC, int V, typename T>
__device__ __forceinline__ void load_chunk(float (&v)[V], const T *p, int n) {
    if (VEC && n >= V) {
        T t[V];
        *reinterpret_cast<uint4 *>(t) = *reinterpret_cast<const uint4 *>(p);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = to_f(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = i < n ? to_f(p[i]) : 0.f;
    }
}
template <bool VEC, int V, typename T>
__device__ __forceinline__ void store_chunk(T *p, const float (&v)[V], int n) {
    T t[V];
#pragma unroll
    for (int i = 0; i < V; i++) from_f(t[i], v[i]);
    if (VEC && n >= V) {
        constexpr int W = V * (int)sizeof(T) / 4;
        if constexpr (W % 4 == 0) {
#pragma unroll
            for (int i = 0; i < W / 4; i++) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(t)[i];
        } else {
            *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(t);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) p[i] = t[i];
    }
}

template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float *sm) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmaxf(v, u) : v + u;
    }
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    // every warp adds the warps' results in the same order: all threads agree
    v = (threadIdx.x & 31) < warps ? sm[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmaxf(v, u) : v + u;
    }
    return v;
}

// CH chunks of 16 bytes per thread hold the row; VEC: every row and the weight
// start on 16 bytes (codes and rows_out on a chunk's part)
template <typename T, int CH, bool VEC>
__global__ void __launch_bounds__(1024) rmsnorm_q8_kernel(NormArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ float sm[2][32];
    const int width = (int)a.width;
    const size_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *r = a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
    float h[CH][V];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int at = ((int)threadIdx.x + c * (int)blockDim.x) * V;
        load_chunk<VEC>(h[c], x + at, width - at);
        if (r) {
            float d[V];
            load_chunk<VEC>(d, r + at, width - at);
#pragma unroll
            for (int i = 0; i < V; i++) h[c][i] += d[i];
        }
#pragma unroll
        for (int i = 0; i < V; i++) ss = fmaf(h[c][i], h[c][i], ss);
    }
    if (a.residual_out) {
        T *out = static_cast<T *>(a.residual_out) + row * a.residual_out_stride;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int at = ((int)threadIdx.x + c * (int)blockDim.x) * V;
            store_chunk<VEC>(out + at, h[c], width - at);
        }
    }
    float inv = 1.f;
    if (a.norm) inv = __frsqrt_rn(__fdiv_rn(block_reduce<false>(ss, sm[0]), (float)width) + a.eps);
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int at = ((int)threadIdx.x + c * (int)blockDim.x) * V;
        float w[V];
        if (a.weight) load_chunk<VEC>(w, static_cast<const T *>(a.weight) + at, width - at);
#pragma unroll
        for (int i = 0; i < V; i++) {
            h[c][i] = h[c][i] * inv;
            if (a.weight) h[c][i] *= w[i];
            const float m = fabsf(h[c][i]);
            if (m < INFINITY) top = fmaxf(top, m);
        }
    }
    top = block_reduce<true>(top, sm[1]);
    const float scale = top > 0.f ? __fdiv_rn(top, 127.f) : 1.f;
    if (threadIdx.x == 0) a.scales[row] = scale;
    int8_t *codes = a.codes + row * a.codes_stride;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int at = ((int)threadIdx.x + c * (int)blockDim.x) * V, n = width - at;
        uint32_t q[V / 4];
        float back[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float m = fabsf(h[c][i]);
            const int code = m < INFINITY ? max(-127, min(127, __float2int_rn(__fdiv_rn(h[c][i], scale)))) : 0;
            back[i] = (float)code * scale;
            if (i % 4 == 0) q[i / 4] = (uint32_t)code & 0xFFu;
            else q[i / 4] |= ((uint32_t)code & 0xFFu) << (8 * (i % 4));
        }
        if (VEC && n >= V) {
            if constexpr (V == 8) *reinterpret_cast<uint2 *>(codes + at) = make_uint2(q[0], q[1]);
            else *reinterpret_cast<uint32_t *>(codes + at) = q[0];
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (i < n) codes[at + i] = (int8_t)(q[i / 4] >> (8 * (i % 4)));
        }
        if (a.rows_out) {
            const size_t o = row * a.rows_stride + at;
            if (a.rows_dtype == QWN_DTYPE_F32) store_chunk<VEC>(static_cast<float *>(a.rows_out) + o, back, n);
            else if (a.rows_dtype == QWN_DTYPE_F16) store_chunk<VEC>(static_cast<__half *>(a.rows_out) + o, back, n);
            else store_chunk<VEC>(static_cast<__nv_bfloat16 *>(a.rows_out) + o, back, n);
        }
    }
}

template <typename T, bool VEC>
cudaError_t launch_norm(const NormArgs &a, uint32_t rows, cudaStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    const uint32_t chunks = (a.width + V - 1) / V;
    auto threads = [&](uint32_t ch) { return ((chunks + ch - 1) / ch + 31) / 32 * 32; };
    if (threads(1) <= 256) rmsnorm_q8_kernel<T, 1, VEC><<<rows, threads(1), 0, s>>>(a);
    else if (threads(2) <= 256) rmsnorm_q8_kernel<T, 2, VEC><<<rows, threads(2), 0, s>>>(a);
    else if (threads(4) <= 512) rmsnorm_q8_kernel<T, 4, VEC><<<rows, threads(4), 0, s>>>(a);
    else rmsnorm_q8_kernel<T, 8, VEC><<<rows, threads(8), 0, s>>>(a);
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_norm_type(const NormArgs &a, uint32_t rows, bool vec, cudaStream_t s) {
    return vec ? launch_norm<T, true>(a, rows, s) : launch_norm<T, false>(a, rows, s);
}

}  // namespace
}  // namespace qkv

using namespace qkv;

QWN_CUDA_ABI_API int qwn_rmsnorm_q8(const QwnRmsNormQ8Request *r) {
    if (!r || !header_ok(r->header, sizeof(*r))) {
        set_error("qwn_rmsnorm_q8: bad header");
        return QWN_CUDA_STATUS_ABI_MISMATCH;
    }
    if (!dtype_ok(r->dtype) || r->mode > QWN_NORM_NONE || (r->rows_out_dev && !dtype_ok(r->rows_dtype)))
        return invalid("qwn_rmsnorm_q8: unknown type or mode");
    if (!(r->eps >= 0.f) || !(r->eps < INFINITY)) return invalid("qwn_rmsnorm_q8: eps must be finite and not negative");
    if (r->width == 0 || r->width > QWN_RMSNORM_MAX_WIDTH || r->rows > 0x7FFFFFFFu)
        return invalid("qwn_rmsnorm_q8: width must be 1..32768");
    if (r->rows == 0) return QWN_CUDA_STATUS_OK;
    if (!r->x_dev || !r->codes_dev || !r->scales_dev) return invalid("qwn_rmsnorm_q8: x, codes and scales are needed");
    NormArgs a{};
    auto stride = [&](uint64_t s) { return s ? s : (uint64_t)r->width; };
    a.x = r->x_dev, a.x_stride = stride(r->x_stride);
    a.residual = r->residual_dev, a.residual_stride = stride(r->residual_stride);
    a.residual_out = r->residual_out_dev, a.residual_out_stride = stride(r->residual_out_stride);
    a.codes = r->codes_dev, a.codes_stride = stride(r->codes_stride);
    a.rows_out = r->rows_out_dev, a.rows_stride = stride(r->rows_stride);
    a.weight = r->weight_dev;
    a.scales = r->scales_dev;
    a.width = r->width;
    a.rows_dtype = r->rows_dtype;
    a.eps = r->eps;
    a.norm = r->mode == QWN_NORM_RMS;
    if (a.x_stride < r->width || a.residual_stride < r->width || a.residual_out_stride < r->width ||
        a.codes_stride < r->width || a.rows_stride < r->width)
        return invalid("qwn_rmsnorm_q8: a row stride is shorter than the row");
    const uint64_t es = r->dtype == QWN_DTYPE_F32 ? 4 : 2, re = r->rows_dtype == QWN_DTYPE_F32 ? 4 : 2;
    const uint64_t v = 16 / es;  // values of a 16-byte chunk: its codes and rows_out values are one access each
    if ((uintptr_t)r->x_dev % es || (uintptr_t)r->residual_dev % es || (uintptr_t)r->weight_dev % es ||
        (uintptr_t)r->residual_out_dev % es || (uintptr_t)r->scales_dev % 4 ||
        (r->rows_out_dev && (uintptr_t)r->rows_out_dev % re))
        return invalid("qwn_rmsnorm_q8: a pointer is not aligned to its type");
    auto on = [](const void *p, uint64_t s, uint64_t bytes) {  // rows of s bytes start on multiples of `bytes`
        return !p || ((uintptr_t)p % bytes == 0 && s % bytes == 0);
    };
    const uint64_t ro = v * re < 16 ? v * re : 16;
    const bool vec = on(r->x_dev, a.x_stride * es, 16) && on(r->residual_dev, a.residual_stride * es, 16) &&
                     on(r->residual_out_dev, a.residual_out_stride * es, 16) && on(r->weight_dev, 0, 16) &&
                     on(r->codes_dev, a.codes_stride, v) && on(r->rows_out_dev, a.rows_stride * re, ro);
    DeviceScope scope(r->device_id);
    if (!scope.ok) return scope.fail("qwn_rmsnorm_q8");
    cudaStream_t s = static_cast<cudaStream_t>(r->stream);
    cudaError_t e;
    if (r->dtype == QWN_DTYPE_F32) e = launch_norm_type<float>(a, r->rows, vec, s);
    else if (r->dtype == QWN_DTYPE_F16) e = launch_norm_type<__half>(a, r->rows, vec, s);
    else e = launch_norm_type<__nv_bfloat16>(a, r->rows, vec, s);
    if (e != cudaSuccess) { set_cuda_error("qwn_rmsnorm_q8", e); return QWN_CUDA_STATUS_RUNTIME_ERROR; }
    return QWN_CUDA_STATUS_OK;
}
