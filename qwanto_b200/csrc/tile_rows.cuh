// Rows of a ragged batch, and rows of a cached tile as the values that their codes
// stand for: 8 lanes per row, lane j holds dims 8j..8j+7 and 64+8j..64+8j+7.
#pragma once

#include <type_traits>

#include "kv_internal.cuh"
#include "rows.cuh"
#include "kv_store.cuh"

namespace qkv {
namespace {

// rows of a ragged batch: row -> (sequence, position)
struct RowMap {
    const int32_t *seq_ids;    // [num_seqs] or null
    const int32_t *row_begin;  // [num_seqs + 1] or null: one row per sequence
    const int32_t *first_pos;  // [num_seqs] or null: the sequence's last rows
    uint32_t num_seqs, num_rows;
};

struct Row16 {
    float v[16];
    __device__ __forceinline__ static int dim(int i, int j) { return i < 8 ? 8 * j + i : 56 + 8 * j + i; }
};

// a Row16 as it is in memory: loads that are issued long before their use
template <typename T>
struct Raw16 {
    uint4 w[sizeof(T) == 4 ? 4 : 2];
    __device__ __forceinline__ void load(const T *row, int j) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int q = 0; q < 4; q++) w[q] = *reinterpret_cast<const uint4 *>(row + Row16::dim(4 * q, j));
        } else {
            w[0] = *reinterpret_cast<const uint4 *>(row + 8 * j);
            w[1] = *reinterpret_cast<const uint4 *>(row + 64 + 8 * j);
        }
    }
    __device__ __forceinline__ Row16 row() const {
        Row16 r;
#pragma unroll
        for (int q = 0; q < (int)(sizeof(w) / 16); q++) {
            const uint32_t u[4] = {w[q].x, w[q].y, w[q].z, w[q].w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (sizeof(T) == 4) {
                    r.v[4 * q + i] = __uint_as_float(u[i]);
                } else if constexpr (std::is_same_v<T, __half>) {
                    r.v[8 * q + 2 * i] = h2f((uint16_t)u[i]);
                    r.v[8 * q + 2 * i + 1] = h2f((uint16_t)(u[i] >> 16));
                } else {
                    r.v[8 * q + 2 * i] = __uint_as_float(u[i] << 16);
                    r.v[8 * q + 2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
                }
            }
        }
        return r;
    }
};
// where the codes of dims 2m, 2m + 1 of both halves are (tq35_put's layout): the
// even ones in nibble n of words `even` and `even + even_step`, the odd ones' low
// bits in nibble n of word `odd`, half 1's two high bits in field n of `plane`
struct TqPlace {
    uint32_t even, even_step, odd, plane, n;
};
__device__ __forceinline__ TqPlace tq_place(int which, int t, int m) {
    if (!which) {
        const uint32_t tig = m >> 3;
        return {32u * t + 8 * tig, 4, 512u + 16 * t + 4 * tig, 768u + 8 * t + 2 * tig, (uint32_t)lb_k_nibble(m)};
    }
    const int r = m & 15;
    const uint32_t lv = ((r & 7) << 2) | ((t & 7) >> 1), b = m >> 4;
    return {16 * lv + 4 * b, 8, 512 + 8 * lv + 4 * b, 768 + 4 * lv + 2 * b,
            (uint32_t)((r >> 3) + 2 * (t >> 3) + 4 * (t & 1))};
}
template <int CODEC>
__device__ Row16 take_row(const uint8_t *tile, int t, int which, int j);

__device__ __forceinline__ Row16 take_q8(const uint8_t *tile, int t, int which, int j, float s0, float s1) {
    Row16 x;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int d = 64 * h + 8 * j;
        uint32_t b[8];
        if (!which) {
            const uint2 w = *reinterpret_cast<const uint2 *>(tile + k8_off(t, d));
#pragma unroll
            for (int i = 0; i < 8; i++) b[i] = prmt(i < 4 ? w.x : w.y, 0x4B000000u, 0x7650u | (uint32_t)(i & 3));
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) b[i] = 0x4B000000u | tile[v8_off(t, d + i)];
        }
#pragma unroll
        for (int i = 0; i < 8; i++)  // 2^23 + code + 128, less that
            x.v[8 * h + i] = (__uint_as_float(b[i]) - 8388736.f) * (h ? s1 : s0);
    }
    return x;
}
template <>
__device__ __forceinline__ Row16 take_row<QWN_KV_CODEC_Q8_HEAD_F16>(const uint8_t *tile, int t, int which, int j) {
    const float s = h2f(*reinterpret_cast<const uint16_t *>(tile + (which ? 4128 : 4096) + s16_off(t)));
    return take_q8(tile, t, which, j, s, s);
}
template <>
__device__ __forceinline__ Row16 take_row<QWN_KV_CODEC_Q8_B64_F32>(const uint8_t *tile, int t, int which, int j) {
    const uint8_t *s = tile + (which ? 4224 : 4096);
    return take_q8(tile, t, which, j, *reinterpret_cast<const float *>(s + s32_off(t, 0)),
                   *reinterpret_cast<const float *>(s + s32_off(t, 1)));
}
template <>
__device__ __forceinline__ Row16 take_row<QWN_KV_CODEC_F16>(const uint8_t *tile, int t, int which, int j) {
    Row16 x;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint4 w = *reinterpret_cast<const uint4 *>(tile + f16_off(which, t, 64 * h + 8 * j));
        const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 8; i++) x.v[8 * h + i] = h2f((uint16_t)(q[i >> 1] >> (16 * (i & 1))));
    }
    return x;
}
__device__ __forceinline__ float code_value(uint32_t code, float step, float mn) {
    return fmaf(__uint_as_float(0x4B000000u | code) - 8388608.f, step, mn);
}
template <>
__device__ __forceinline__ Row16 take_row<QWN_KV_CODEC_Q4_G32>(const uint8_t *tile, int t, int which, int j) {
    Row16 x;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int c = 2 * h + (j >> 2), mb = 4 * h + (j >> 1);
        const uint32_t par = *reinterpret_cast<const uint32_t *>(tile + (which ? 2304 : 2048) + 32 * (t & 7) + 8 * c +
                                                                 4 * (t >> 3));
        const float step = __fdiv_rn(h2f((uint16_t)par), 15.f), mn = h2f((uint16_t)(par >> 16));
        const uint32_t w = which ? 0u : *reinterpret_cast<const uint32_t *>(tile + 64 * t + 16 * (j & 3) + 4 * c);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint32_t q;
            if (!which) {
                q = w >> (8 * (i & 3) + 4 * (i >> 2));
            } else {
                const int lv = 4 * i + ((t & 7) >> 1), chunk = (mb >> 2) ^ ((lv >> 2) & 1);
                q = (uint32_t)tile[1024 + 32 * lv + 16 * chunk + 4 * (mb & 3) + (t >> 3) + 2 * (t & 1)] >> (4 * (j & 1));
            }
            x.v[8 * h + i] = code_value(q & 15u, step, mn);
        }
    }
    return x;
}
template <>
__device__ __forceinline__ Row16 take_row<QWN_KV_CODEC_TQ35_G64>(const uint8_t *tile, int t, int which, int j) {
    const uint8_t *half = tile + which * 1024;
    float mn[2], even[2], odd[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t par = *reinterpret_cast<const uint32_t *>(half + 896 + 16 * (t & 7) + 8 * h + 4 * (t >> 3));
        mn[h] = h2f((uint16_t)(par >> 16));
        even[h] = __fdiv_rn(h2f((uint16_t)par), 15.f);
        odd[h] = __fdiv_rn(h2f((uint16_t)par), 7.f);
    }
    auto word = [&](uint32_t at) { return *reinterpret_cast<const uint32_t *>(half + at); };
    Row16 x;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const TqPlace p = tq_place(which, t, 4 * j + i);
        const uint32_t o = word(p.odd) >> (4 * p.n), hi = word(p.plane & ~3u) >> (2 * p.n + 8 * (p.plane & 3u));
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t code = h ? ((o >> 3) & 1u) | ((hi & 3u) << 1) : o & 7u;
            x.v[8 * h + 2 * i] = code_value((word(p.even + h * p.even_step) >> (4 * p.n)) & 15u, even[h], mn[h]);
            x.v[8 * h + 2 * i + 1] = code_value(code, odd[h], mn[h]);
        }
    }
    return x;
}

}  // namespace
}  // namespace qkv
