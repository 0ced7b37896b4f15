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
// The quotient y / s is y x (1 / s), corrected once by its residual y - q s
// (Markstein 1990: with a correctly rounded inverse the corrected quotient is the
// rounded one; tested where a quotient is hardest to round), so that codes are the
// Q8 codecs' own, ties among them.  Without the residual, one code in some
// thousands of 16-bit rows differed; with it 8192 x 4096 bf16 takes 39.2 us
// instead of 39.0, quantised alone 22.6 instead of 21.6.  Adding 1.5 x 2^23 leaves
// the rounded code in the sum's low byte, and the sum less that number is the code
// in fp32: no division or conversion per value.  What can be done on two values in
// one instruction is, and values that are no numbers are looked for once per thread
// (a maximum that keeps NaN), so that 16-bit rows are not bound by instruction
// issue (4096 x 12288 bf16: 71 us; 103 one by one).  All loads of x and r are
// issued before the first is used: 8191 x 6144 fp16 with residual and rows_out
// takes 69 us, 6.5 TB/s (131 us with divisions and loads as they are needed).
// What is not given is added as -0 or multiplied as 1, which changes no value:
// conditions per value had cost as much (1000 x 6144 bf16: 9.5 us, 10.3).  Rows
// without a residual have kernels of their own; they are bound by instruction issue
// and by fewer bytes in flight between a row's reductions (8192 x 4096 bf16: 30
// us, 5.5 TB/s; 46 and 6.5 with a residual; 4.5 to 4.6 TB/s at 2560, 8960 and 12288
// wide).  Rows over 16384 wide leave one CTA's registers per SM (bf16: 2048 x 32768
// with a residual 114 us, 5.3 TB/s; 2048 x 28672 without 83 us, 3.5 TB/s).
// Rows that are not whole 16-byte chunks, or start off them, are read value by
// value (8192 x 4095 bf16: 75 us, 4096 wide 46; fp32 85).
#include <type_traits>

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
    uint32_t rows, width, rows_dtype;
    float eps;
    bool norm;
};

// V values, the first at `at`: 16 bytes that follow one another (STEP 1), or every
// STEP-th value for a CTA of that many threads, so that a warp's accesses are
// consecutive whatever the alignment.  Beyond the row's end any numbers.  No
// branch: the loads of all chunks are in flight together.
template <typename T>
struct Chunk {
    uint32_t w[4];
    __device__ __forceinline__ float get(int i) const {  // i is known at compile time
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (std::is_same_v<T, __half>) return h2f((uint16_t)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1]));
        else return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
    }
    __device__ __forceinline__ uint64_t two(int i) const { return pair(get(2 * i), get(2 * i + 1)); }
};
// what leaves every value as it is when added, or multiplied with
template <typename T>
__device__ __forceinline__ Chunk<T> minus_zeros() {
    constexpr uint32_t b = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
    return {{b, b, b, b}};
}
template <typename T>
__device__ __forceinline__ Chunk<T> ones() {
    constexpr uint32_t b = sizeof(T) == 4 ? 0x3F800000u : std::is_same_v<T, __half> ? 0x3C003C00u : 0x3F803F80u;
    return {{b, b, b, b}};
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t raw_bits(float x) { return __float_as_uint(x); }
__device__ __forceinline__ uint32_t raw_bits(__half x) { return __half_as_ushort(x); }
__device__ __forceinline__ uint32_t raw_bits(__nv_bfloat16 x) { return __bfloat16_as_ushort(x); }
template <int STEP, typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T *p, int at, int width) {
    Chunk<T> c;
    if constexpr (STEP == 1) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p + (at < width ? at : 0));
        c.w[0] = v.x, c.w[1] = v.y, c.w[2] = v.z, c.w[3] = v.w;
    } else {
        constexpr int V = 16 / (int)sizeof(T), per = V / 4;
        const T *q = p + at;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t b = at + i * STEP < width ? raw_bits(q[i * STEP]) : 0u;
            if (i % per == 0) c.w[i / per] = b;
            else c.w[i / per] |= b << 16;
        }
    }
    return c;
}
__device__ __forceinline__ uint32_t pack2(const float *, float a, float) { return __float_as_uint(a); }
__device__ __forceinline__ uint32_t pack2(const __half *, float a, float b) { return pack_h2(a, b); }
__device__ __forceinline__ uint32_t pack2(const __nv_bfloat16 *, float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
// the same values back, those before the row's end
template <int STEP, int PAIRS, typename T>
__device__ __forceinline__ void store_chunk(T *p, int at, const uint64_t (&pairs)[PAIRS], int width) {
    constexpr int V = 2 * PAIRS, per = 4 / (int)sizeof(T), W = V / per;
    float v[V];
#pragma unroll
    for (int i = 0; i < PAIRS; i++) unpair(pairs[i], v[2 * i], v[2 * i + 1]);
    uint32_t w[W];
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = pack2(p, v[per * i], v[per * i + per - 1]);
    if (STEP == 1) {
        if (at < width) {
            if constexpr (W % 4 == 0) {
#pragma unroll
                for (int i = 0; i < W; i += 4)
                    *reinterpret_cast<uint4 *>(p + at + per * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
            } else {
                *reinterpret_cast<uint2 *>(p + at) = make_uint2(w[0], w[1]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (at + i * STEP >= width) continue;
            if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t *>(p + at)[i * STEP] = w[i];
            else reinterpret_cast<uint16_t *>(p + at)[i * STEP] = (uint16_t)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1]);
        }
    }
}

// 1.5 x 2^23: a small number's sum with it is rounded to a whole one, ties to
// even, and has that number's byte at its low end
constexpr float kMagic = 12582912.f;

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

// CH chunks of 16 bytes per thread hold the row.  STEP 1: rows are whole chunks,
// and every row and the weight start on 16 bytes (codes and rows_out on a chunk's
// part); otherwise STEP is the CTA's threads.  CTAS: how many the compiler fits
// the registers of an SM for.  RES: there may be a residual.
template <typename T, int CH, int STEP, int CTAS = 0, bool RES = true>
__global__ void __launch_bounds__(CH <= 2 ? 1024 : 512, CTAS) rmsnorm_q8_kernel(NormArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    // the weight's chunks are held from the start, or come from L1 or L2 between the reductions where
    // their registers would cost a CTA per SM (4096 x 14336 bf16 without residual: 59 us, 96; 2048 x
    // 10240 fp32: 50, 76); 16-bit rows over 16384 wide have one CTA either way (2048 x 32768: 113, 116)
    constexpr bool kLateWeight = CH * V >= 32 && !(V == 8 && CH == 8);
    __shared__ float sm[2][32];
    const int width = (int)a.width;
    const size_t row = (size_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= a.rows) return;  // only with one warp per row, which waits for no other
    auto at = [](int c) {
        return STEP == 1 ? ((int)threadIdx.x + c * (int)blockDim.x) * V : (int)threadIdx.x + c * V * STEP;
    };
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *r = RES && a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
    const T *w = static_cast<const T *>(a.weight);
    uint64_t h[CH][V / 2];  // pairs of values
    Chunk<T> wc[CH];
    // values past the row's end: any numbers in whole chunks, zeros otherwise
    auto live = [&](int c) { return STEP != 1 || at(c) < width; };
    uint64_t ss = 0;
    launch_dependents();
    wait_previous();
    {
        Chunk<T> xc[CH], rc[CH];
#pragma unroll
        for (int c = 0; c < CH; c++) xc[c] = load_chunk<STEP>(x, at(c), width);
#pragma unroll
        for (int c = 0; c < CH; c++) rc[c] = minus_zeros<T>();
        if (r) {
#pragma unroll
            for (int c = 0; c < CH; c++) rc[c] = load_chunk<STEP>(r, at(c), width);
        }
#pragma unroll
        for (int c = 0; c < CH; c++) wc[c] = ones<T>();
        if (w && !kLateWeight) {
#pragma unroll
            for (int c = 0; c < CH; c++) wc[c] = load_chunk<STEP>(w, at(c), width);
        }
#pragma unroll
        for (int c = 0; c < CH; c++) {
            uint64_t sum = ss;
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                h[c][i] = xc[c].two(i);
                if (RES) h[c][i] = add2(h[c][i], rc[c].two(i));
                sum = fma2(h[c][i], h[c][i], sum);
            }
            ss = live(c) ? sum : ss;
        }
    }
    if (a.residual_out) {
        T *out = static_cast<T *>(a.residual_out) + row * a.residual_out_stride;
#pragma unroll
        for (int c = 0; c < CH; c++) store_chunk<STEP>(out, at(c), h[c], width);
    }
    float inv = 1.f;
    if (a.norm) {
        float even, odd;
        unpair(ss, even, odd);
        inv = __frsqrt_rn(__fdiv_rn(block_reduce<false>(even + odd, sm[0]), (float)width) + a.eps);
    }
    float top = 0.f;  // NaN once a value is
#pragma unroll
    for (int c = 0; c < CH; c++) {
        if (w && kLateWeight) wc[c] = load_chunk<STEP>(w, at(c), width);
        float most = top;
#pragma unroll
        for (int i = 0; i < V / 2; i++) {
            h[c][i] = mul2(mul2(h[c][i], pair(inv, inv)), wc[c].two(i));
            float even, odd;
            unpair(h[c][i], even, odd);
            most = max_or_nan(max_or_nan(most, fabsf(even)), fabsf(odd));
        }
        top = live(c) ? most : top;
    }
    if (!(top < INFINITY)) {  // what is no number has code 0
        top = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                float even, odd;
                unpair(h[c][i], even, odd);
                even = fabsf(even) < INFINITY ? even : 0.f, odd = fabsf(odd) < INFINITY ? odd : 0.f;
                h[c][i] = pair(even, odd);
                if (live(c)) top = fmaxf(top, fmaxf(fabsf(even), fabsf(odd)));
            }
    }
    top = block_reduce<true>(top, sm[1]);
    float scale = __fdiv_rn(top, 127.f);
    if (scale == 0.f) scale = 1.f;
    if (threadIdx.x == 0) a.scales[row] = scale;
    float divisor = scale;
    if (top < 0x1p-90f) {  // near the smallest numbers: scaled up by 2^60, and a scale of few bits may give more than 127
        divisor = scale * 0x1p60f;
        const float most = 127.f * divisor;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                float even, odd;
                unpair(mul2(h[c][i], pair(0x1p60f, 0x1p60f)), even, odd);
                h[c][i] = pair(fminf(fmaxf(even, -most), most), fminf(fmaxf(odd, -most), most));
            }
    }
    const float inverse = __fdiv_rn(1.f, divisor);
    int8_t *codes = a.codes + row * a.codes_stride;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int first = at(c);
        uint32_t q[V / 4];
        uint64_t back[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; i += 2) {
            uint32_t bits[4];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint64_t y = h[c][i + j], near = mul2(y, pair(inverse, inverse));
                const uint64_t rest = fma2(near, pair(-divisor, -divisor), y);
                const uint64_t sum = add2(fma2(rest, pair(inverse, inverse), near), pair(kMagic, kMagic));
                unpair(sum, bits[2 * j], bits[2 * j + 1]);
                back[i + j] = mul2(add2(sum, pair(-kMagic, -kMagic)), pair(scale, scale));
            }
            q[i / 2] = prmt(prmt(bits[0], bits[1], 0x0040u), prmt(bits[2], bits[3], 0x0040u), 0x5410u);
        }
        if (STEP == 1) {
            if (first < width) {
                if constexpr (V == 8) *reinterpret_cast<uint2 *>(codes + first) = make_uint2(q[0], q[1]);
                else *reinterpret_cast<uint32_t *>(codes + first) = q[0];
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (first + i * STEP < width) (codes + first)[i * STEP] = (int8_t)(q[i / 4] >> (8 * (i % 4)));
        }
        if (a.rows_out) {
            const size_t o = row * a.rows_stride;
            if (a.rows_dtype == QWN_DTYPE_F32) store_chunk<STEP>(static_cast<float *>(a.rows_out) + o, first, back, width);
            else if (a.rows_dtype == QWN_DTYPE_F16) store_chunk<STEP>(static_cast<__half *>(a.rows_out) + o, first, back, width);
            else store_chunk<STEP>(static_cast<__nv_bfloat16 *>(a.rows_out) + o, first, back, width);
        }
    }
}

// CTAS steers the compiler's use of registers: "at least one" gives 16-bit rows 44
// instead of 48 (4096 x 1536 bf16: 9.3 us, 9.9), and is worse for fp32 rows value by
// value (8192 x 4095: 102 us, 87)
template <typename T>
constexpr int kCtas = sizeof(T) == 2 ? 1 : 0;

template <typename T, int STEP>
cudaError_t launch_narrow(const NormArgs &a, uint32_t rows, uint32_t chunks, cudaStream_t s) {
    const dim3 grid((rows + 7) / 8), block(32, 8);
    if (chunks <= 32) return launch_next(rmsnorm_q8_kernel<T, 1, STEP, kCtas<T>>, grid, block, s, a);
    if (chunks <= 64) return launch_next(rmsnorm_q8_kernel<T, 2, STEP, kCtas<T>>, grid, block, s, a);
    return launch_next(rmsnorm_q8_kernel<T, 4, STEP>, grid, block, s, a);
}

template <typename T, int CH, int CTAS>
cudaError_t launch_row(const NormArgs &a, uint32_t rows, uint32_t threads, cudaStream_t s) {
    if (a.residual) return launch_next(rmsnorm_q8_kernel<T, CH, 1, CTAS>, dim3(rows), threads, s, a);
    return launch_next(rmsnorm_q8_kernel<T, CH, 1, CTAS, false>, dim3(rows), threads, s, a);
}
template <typename T>
cudaError_t launch_chunks(const NormArgs &a, uint32_t rows, cudaStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    const uint32_t chunks = (a.width + V - 1) / V;
    auto threads = [&](uint32_t ch) { return ((chunks + ch - 1) / ch + 31) / 32 * 32; };
    // Up to two rows per SM: wide CTAs answer sooner (1 x 1536 fp32: 1.9 us with
    // one chunk per thread, 2.3 with four).  More: small CTAs with several
    // chunks each keep more loads in flight per SM (8191 x 6144 fp16: 69 us with
    // four chunks, 94 with one; 4096 x 1536 bf16: 9.0 with two, 11.2 with one).
    // Without a residual a row is less to load and instructions count more, of
    // which four chunks need fewer each (8192 x 4096 bf16: 30 us, 37 with two).
    // Many narrow rows go eight to a CTA, a warp each (8192 x 256 bf16: 4.2 us, 9.0
    // with a CTA each; 8192 x 640: 10.2 and 11.8; 1000 x 1000: 4.5 and 4.1).
    const bool few = rows <= 296;
    if (rows >= 2048 && chunks <= 96) return launch_narrow<T, 1>(a, rows, chunks, s);
    if (few && threads(1) <= 1024) return launch_row<T, 1, kCtas<T>>(a, rows, threads(1), s);
    if (threads(2) <= (few ? 1024u : a.residual ? 256u : 96u))
        return launch_row<T, 2, kCtas<T>>(a, rows, threads(2), s);
    if (threads(4) <= (V == 4 ? 512u : 448u)) return launch_row<T, 4, 0>(a, rows, threads(4), s);
    // 16-bit rows past 448 threads: 72 registers leave one CTA per SM, 64 two (4096 x 16384 bf16: 119 us, 91)
    if constexpr (V == 8)
        if (threads(4) <= 512) return launch_row<T, 4, 2>(a, rows, threads(4), s);
    if constexpr (V == 4)  // 2048 x 16384 fp32: 56 us, 75
        if (threads(8) > 448 && threads(8) <= 512 && !a.residual)
            return launch_next(rmsnorm_q8_kernel<T, 8, 1, 2, false>, dim3(rows), threads(8), s, a);
    if (V == 8 || threads(8) <= 512) return launch_row<T, 8, 0>(a, rows, threads(8), s);
    return launch_row<T, 64 / V, 0>(a, rows, threads(64 / V), s);
}

// rows off the 16-byte grid: CTAs of 128, 256 or 512 threads
template <typename T, int CH>
cudaError_t launch_values_ch(const NormArgs &a, uint32_t rows, uint32_t threads, cudaStream_t s) {
    constexpr int ctas = CH <= 2 ? kCtas<T> : 0;
    if constexpr (CH <= 2)  // launch_values gives 128 threads up to two chunks each, 256 two at least
        if (threads == 128) return launch_next(rmsnorm_q8_kernel<T, CH, 128, ctas>, dim3(rows), dim3(128), s, a);
    if constexpr (CH >= 2)
        if (threads == 256) return launch_next(rmsnorm_q8_kernel<T, CH, 256, ctas>, dim3(rows), dim3(256), s, a);
    return launch_next(rmsnorm_q8_kernel<T, CH, 512, ctas>, dim3(rows), dim3(512), s, a);
}
template <typename T>
cudaError_t launch_values(const NormArgs &a, uint32_t rows, cudaStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    const uint32_t chunks = (a.width + V - 1) / V;
    if (rows >= 2048 && chunks <= 96) return launch_narrow<T, 32>(a, rows, chunks, s);
    uint32_t threads = rows <= 296 ? 512 : chunks <= 256 ? 128 : 256;
    if (chunks > threads * (64 / V)) threads = 512;
    if (chunks <= threads) return launch_values_ch<T, 1>(a, rows, threads, s);
    if (chunks <= threads * 2) return launch_values_ch<T, 2>(a, rows, threads, s);
    if (chunks <= threads * 4) return launch_values_ch<T, 4>(a, rows, threads, s);
    if (V == 8 || chunks <= threads * 8) return launch_values_ch<T, 8>(a, rows, threads, s);
    return launch_values_ch<T, 64 / V>(a, rows, threads, s);
}

template <typename T>
cudaError_t launch_norm_type(const NormArgs &a, uint32_t rows, bool vec, cudaStream_t s) {
    return vec ? launch_chunks<T>(a, rows, s) : launch_values<T>(a, rows, s);
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
    a.rows = r->rows;
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
    if (r->residual_out_dev) {
        const RowSpan out = {(uintptr_t)r->residual_out_dev, a.residual_out_stride * es, r->width * es, r->rows};
        auto met = [&](const void *p, uint64_t stride, uint64_t rows) {  // in place is none: a row's CTA reads it first
            const RowSpan in = {(uintptr_t)p, stride * es, out.bytes, rows};
            return p && !(in.at == out.at && (in.stride == out.stride || r->rows == 1)) && rows_meet(in, out);
        };
        if (met(r->x_dev, a.x_stride, r->rows) || met(r->residual_dev, a.residual_stride, r->rows) ||
            (r->weight_dev && rows_meet({(uintptr_t)r->weight_dev, out.bytes, out.bytes, 1}, out)))
            return invalid("qwn_rmsnorm_q8: residual_out overlaps an input that it does not equal, row for row");
    }
    auto on = [](const void *p, uint64_t s, uint64_t bytes) {  // rows of s bytes start on multiples of `bytes`
        return !p || ((uintptr_t)p % bytes == 0 && s % bytes == 0);
    };
    const uint64_t ro = v * re < 16 ? v * re : 16;
    const bool vec = r->width % v == 0 && on(r->x_dev, a.x_stride * es, 16) && on(r->residual_dev, a.residual_stride * es, 16) &&
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
