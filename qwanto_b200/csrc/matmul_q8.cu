// int8 products with a scale per token and per output (qwn_matmul_q8_*):
//     out[m][n] = (sum_k X[m][k] W[n][k]) * sx[m] * sw[n] + b[n]
// The sum is exact in int32; the scales and the bias are applied in fp32 and
// the result is rounded once.  The reference's only device product takes
// host activations and 2-bit weights (c/cuda/qwn_hypervsq2_cuda_abi.cu); this
// one keeps both sides on the device.
//
// Weights are copied once into rows of a multiple of 128 bytes, zero past
// in_features, so a product never branches on in_features' remainder.
#include <cstring>
#include <new>

#include "kv_internal.cuh"
#include "rows.cuh"

namespace qkv {
namespace {

constexpr uint32_t kMmK = 128;  // bytes of a weight row's granule

struct MatmulQ8 {
    int device = 0;
    uint32_t n = 0, k = 0, kpad = 0;
    int8_t *w = nullptr;
    float *scales = nullptr, *bias = nullptr;
    uint32_t *status = nullptr;
};

MatmulQ8 *matmul_from(const QwnMatmulQ8Handle *h) {
    if (!h || !header_ok(h->header, sizeof(*h)) || !h->opaque) return nullptr;
    return static_cast<MatmulQ8 *>(h->opaque);
}

void matmul_release(MatmulQ8 *m) {
    cudaFree(m->w);
    cudaFree(m->scales);
    cudaFree(m->bias);
    cudaFree(m->status);
    delete m;
}

struct MmArgs {
    const int8_t *x, *w;
    const float *sx, *sw, *bias;
    void *out;
    uint64_t x_stride, out_stride;
    uint32_t m, n, k, kpad, out_dtype;
};

__device__ __forceinline__ void store_out(const MmArgs &a, uint32_t row, uint32_t col, float v) {
    const size_t o = (size_t)row * a.out_stride + col;
    if (a.out_dtype == QWN_DTYPE_F32) static_cast<float *>(a.out)[o] = v;
    else if (a.out_dtype == QWN_DTYPE_F16) static_cast<__half *>(a.out)[o] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(a.out)[o] = __float2bfloat16_rn(v);
}

// 64 x 64 outputs per CTA, 4 x 4 per thread, dot products of four codes at a time
constexpr int kSimpleTile = 64, kSimpleK = 64;
__global__ void __launch_bounds__(256) matmul_q8_simple_kernel(MmArgs a) {
    __shared__ int xs[kSimpleTile][kSimpleK / 4 + 1], ws[kSimpleTile][kSimpleK / 4 + 1];
    const uint32_t m0 = blockIdx.y * kSimpleTile, n0 = blockIdx.x * kSimpleTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (uint32_t k0 = 0; k0 < a.kpad; k0 += kSimpleK) {
        for (int i = threadIdx.x; i < kSimpleTile * kSimpleK / 4; i += 256) {
            const int r = i / (kSimpleK / 4), c = i % (kSimpleK / 4);
            const uint32_t kk = k0 + 4 * c;
            int xv = 0, wv = 0;
            if (m0 + r < a.m && kk < a.k) {
                const int8_t *p = a.x + (size_t)(m0 + r) * a.x_stride + kk;
                if (kk + 4 <= a.k) xv = *reinterpret_cast<const int *>(p);
                else
                    for (uint32_t j = 0; kk + j < a.k; j++) xv |= (int)((uint32_t)(uint8_t)p[j] << (8 * j));
            }
            if (n0 + r < a.n) wv = *reinterpret_cast<const int *>(a.w + (size_t)(n0 + r) * a.kpad + kk);
            xs[r][c] = xv;
            ws[r][c] = wv;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kSimpleK / 4; c++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(xs[ty + 16 * i][c], ws[tx + 16 * j][c], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t row = m0 + ty + 16 * i;
        if (row >= a.m) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t col = n0 + tx + 16 * j;
            if (col >= a.n) continue;
            const float v = (float)acc[i][j] * a.sx[row] * a.sw[col];
            store_out(a, row, col, a.bias ? v + a.bias[col] : v);
        }
    }
}

cudaError_t launch_matmul(const MmArgs &a, cudaStream_t s) {
    const dim3 grid((a.n + kSimpleTile - 1) / kSimpleTile, (a.m + kSimpleTile - 1) / kSimpleTile);
    matmul_q8_simple_kernel<<<grid, 256, 0, s>>>(a);
    count_launch();
    return cudaGetLastError();
}

}  // namespace
}  // namespace qkv

using namespace qkv;

QWN_CUDA_ABI_API int qwn_matmul_q8_create(const QwnMatmulQ8Options *o, QwnMatmulQ8Handle *out) {
    if (!o || !out || !header_ok(o->header, sizeof(*o)) || !header_ok(out->header, sizeof(*out))) {
        set_error("qwn_matmul_q8_create: bad header");
        return QWN_CUDA_STATUS_ABI_MISMATCH;
    }
    out->opaque = nullptr;
    if (o->out_features == 0 || o->out_features > 0x7FFFFFFFu || o->in_features == 0 ||
        o->in_features > QWN_MATMUL_Q8_MAX_IN)
        return invalid("qwn_matmul_q8_create: in_features must be 1..131071, out_features at least 1");
    const uint64_t stride = o->weight_stride ? o->weight_stride : o->in_features;
    if (!o->weight_dev || !o->scales_dev || stride < o->in_features)
        return invalid("qwn_matmul_q8_create: weight and scales are needed, and a stride of a whole row");
    DeviceScope scope(o->device_id);
    if (!scope.ok) return scope.fail("qwn_matmul_q8_create");
    MatmulQ8 *m = new (std::nothrow) MatmulQ8();
    if (!m) return QWN_CUDA_STATUS_OUT_OF_MEMORY;
    m->device = o->device_id;
    m->n = o->out_features;
    m->k = o->in_features;
    m->kpad = (o->in_features + kMmK - 1) / kMmK * kMmK;
    cudaStream_t s = static_cast<cudaStream_t>(o->stream);
    const size_t wb = (size_t)m->n * m->kpad, fb = (size_t)m->n * sizeof(float);
    if (cudaMalloc(&m->w, wb) != cudaSuccess || cudaMalloc(&m->scales, fb) != cudaSuccess ||
        (o->bias_dev && cudaMalloc(&m->bias, fb) != cudaSuccess) ||
        cudaMalloc(&m->status, sizeof(uint32_t)) != cudaSuccess) {
        set_cuda_error("qwn_matmul_q8_create: allocation", cudaGetLastError());
        matmul_release(m);
        return QWN_CUDA_STATUS_OUT_OF_MEMORY;
    }
    cudaError_t e = m->kpad == m->k ? cudaSuccess : cudaMemsetAsync(m->w, 0, wb, s);
    if (e == cudaSuccess)
        e = cudaMemcpy2DAsync(m->w, m->kpad, o->weight_dev, stride, m->k, m->n, cudaMemcpyDeviceToDevice, s);
    if (e == cudaSuccess) e = cudaMemcpyAsync(m->scales, o->scales_dev, fb, cudaMemcpyDeviceToDevice, s);
    if (e == cudaSuccess && m->bias) e = cudaMemcpyAsync(m->bias, o->bias_dev, fb, cudaMemcpyDeviceToDevice, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(m->status, 0, sizeof(uint32_t), s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) {
        set_cuda_error("qwn_matmul_q8_create: copy", e);
        matmul_release(m);
        return QWN_CUDA_STATUS_RUNTIME_ERROR;
    }
    std::memset(out, 0, sizeof(*out));
    qwn_cuda_abi_header_init(&out->header, sizeof(*out));
    out->opaque = m;
    return QWN_CUDA_STATUS_OK;
}

QWN_CUDA_ABI_API int qwn_matmul_q8_destroy(QwnMatmulQ8Handle *h) {
    MatmulQ8 *m = matmul_from(h);
    if (!m) return invalid("qwn_matmul_q8_destroy: bad handle");
    DeviceScope scope(m->device);
    cudaDeviceSynchronize();
    matmul_release(m);
    h->opaque = nullptr;
    return QWN_CUDA_STATUS_OK;
}

QWN_CUDA_ABI_API int qwn_matmul_q8(QwnMatmulQ8Handle *h, const QwnMatmulQ8Request *r) {
    MatmulQ8 *m = matmul_from(h);
    if (!m || !r || !header_ok(r->header, sizeof(*r))) return invalid("qwn_matmul_q8: bad handle or header");
    if (!dtype_ok(r->out_dtype)) return invalid("qwn_matmul_q8: unknown output type");
    const uint64_t xs = r->codes_stride ? r->codes_stride : m->k, os = r->out_stride ? r->out_stride : m->n;
    if (xs < m->k || os < m->n) return invalid("qwn_matmul_q8: a row stride is shorter than the row");
    if (r->rows == 0) return QWN_CUDA_STATUS_OK;
    if (r->rows > 0x7FFFFFFFu || !r->codes_dev || !r->scales_dev || !r->out_dev)
        return invalid("qwn_matmul_q8: codes, scales and out are needed");
    if ((uintptr_t)r->codes_dev % 16 || (xs % 16 && r->rows > 1))
        return invalid("qwn_matmul_q8: rows of codes must start on 16 bytes (pointer and stride)");
    if ((uintptr_t)r->scales_dev % 4 || (uintptr_t)r->out_dev % (r->out_dtype == QWN_DTYPE_F32 ? 4 : 2))
        return invalid("qwn_matmul_q8: a pointer is not aligned to its type");
    DeviceScope scope(m->device);
    if (!scope.ok) return scope.fail("qwn_matmul_q8");
    MmArgs a{};
    a.x = r->codes_dev, a.w = m->w;
    a.sx = r->scales_dev, a.sw = m->scales, a.bias = m->bias;
    a.out = r->out_dev, a.out_stride = os, a.x_stride = xs;
    a.m = r->rows, a.n = m->n, a.k = m->k, a.kpad = m->kpad, a.out_dtype = r->out_dtype;
    const cudaError_t e = launch_matmul(a, static_cast<cudaStream_t>(r->stream));
    if (e != cudaSuccess) { set_cuda_error("qwn_matmul_q8", e); return QWN_CUDA_STATUS_RUNTIME_ERROR; }
    return QWN_CUDA_STATUS_OK;
}

QWN_CUDA_ABI_API int qwn_matmul_q8_check(QwnMatmulQ8Handle *h, uint32_t *bits) {
    MatmulQ8 *m = matmul_from(h);
    if (!m || !bits) return invalid("qwn_matmul_q8_check: bad handle");
    DeviceScope scope(m->device);
    cudaError_t e = cudaDeviceSynchronize();
    uint32_t st = 0;
    if (e == cudaSuccess) e = cudaMemcpy(&st, m->status, sizeof(st), cudaMemcpyDeviceToHost);
    if (e == cudaSuccess) e = cudaMemset(m->status, 0, sizeof(uint32_t));
    if (e != cudaSuccess) { set_cuda_error("qwn_matmul_q8_check", e); return QWN_CUDA_STATUS_RUNTIME_ERROR; }
    *bits = st;
    return QWN_CUDA_STATUS_OK;
}
