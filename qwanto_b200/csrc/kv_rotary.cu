// Rows into the paged cache with the position rotation applied on the way
// (qwn_kv_append_rotary) and cached rows back out (qwn_kv_load_tokens).
//
// The reference rotates on the host before it stores
// (c/qwanto_decode.c:1657-1927); here the projection's rows go to pages in
// one pass: K is rotated in registers and quantised straight into its tile,
// V is quantised beside it, Q is rotated to rows for the attention.
//
// Rotation of a head's first rotary_dim dims, with the angles' cosines c and
// sines s from a table row [c(0..r/2-1), s(0..r/2-1)], over the pairs (i, j) =
// (p, p + r/2), or (2p, 2p + 1):
//     x'[i] = x[i] c[p] - x[j] s[p],   x'[j] = x[j] c[p] + x[i] s[p]
// in fp32 with every product and sum rounded by itself, so that K's codes do
// not depend on how the compiler contracts.
//
// Bound by HBM: rows in, rotated Q and pages out (prompts), by the launch for
// one token per sequence.  Two ways through the data:
//  - one warp per row and head, four dims per lane (store_token's layout): one
//    token per sequence, and the tiles that a prompt fills in part;
//  - one CTA per tile and kv head where all 16 tokens of the tile are new: 8
//    lanes per row, which hold dims 8j.. and 64 + 8j.., so that a pair of
//    halves meets in one lane and a maximum over a head takes 3 shuffles for 4
//    rows (with 4 dims per lane, 4 + 5 per row); the tile is put together in
//    shared memory and leaves in 16-byte stores.
// 16384 rows of 32 + 2 x 8 bf16 heads with their rotation into 4-bit pages: 69 us
// (5.1 TB/s; all rows by the first way 289), into int8 75; fp32 rows 128 and 133
// (5.4 and 5.3 TB/s); 131072 cached int8 rows of 8 heads back to bf16: 132 us (6.1
// TB/s).  One row of 12 + 2 x 2 heads: 2.9 us, back 1.9.  Six CTAs per SM: 72 us,
// four 78, measured for bf16 into 4-bit pages; under that bound (80 registers)
// every type spills, 16-bit rows 64 to 80 bytes per thread, fp32 rows up to 192.
#include <algorithm>
#include <type_traits>

#include "kv_internal.cuh"
#include "kv_store.cuh"
#include "rows.cuh"

namespace qkv {
namespace {

// rows of a ragged batch: row -> (sequence, position)
struct RowMap {
    const int32_t *seq_ids;    // [num_seqs] or null
    const int32_t *row_begin;  // [num_seqs + 1] or null: one row per sequence
    const int32_t *first_pos;  // [num_seqs] or null: the sequence's last rows
    uint32_t num_seqs, num_rows;
};

// whether a position of a sequence holds a token; latches what is wrong with it
__device__ __forceinline__ bool place_ok(const StoreGeo &g, int32_t seq, int64_t pos, bool tell) {
    if (seq < 0 || (uint32_t)seq >= g.max_seqs) {
        if (tell) latch(g.status, QWN_KV_STATUS_BAD_SEQUENCE);
        return false;
    }
    if (pos < 0 || pos >= g.seq_lens[seq]) {
        if (tell) latch(g.status, QWN_KV_STATUS_BAD_LENGTH);
        return false;
    }
    return true;
}

// the same for a unit's row
__device__ __forceinline__ bool unit_row_ok(const StoreGeo &g, int32_t seq, int32_t len, int64_t pos, bool tell) {
    if (seq >= 0 && pos >= 0 && pos < len) return true;
    if (tell) latch(g.status, seq < 0 ? QWN_KV_STATUS_BAD_SEQUENCE : QWN_KV_STATUS_BAD_LENGTH);
    return false;
}

// the sequence of a row and its position in the cache; false where there is none
__device__ __forceinline__ bool find_row(const StoreGeo &g, const RowMap &m, uint32_t row, int32_t &seq, int64_t &pos,
                                         bool tell) {
    uint32_t i = row;
    int64_t b = row, e = b + 1;
    if (m.row_begin) {
        uint32_t lo = 0, hi = m.num_seqs;  // the last i with row_begin[i] <= row
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (m.row_begin[mid] <= (int32_t)row) lo = mid;
            else hi = mid;
        }
        i = lo;
        b = m.row_begin[i];
        e = m.row_begin[i + 1];
        if ((int64_t)row < b || (int64_t)row >= e) {
            if (tell) latch(g.status, QWN_KV_STATUS_BAD_LENGTH);
            return false;
        }
    }
    seq = m.seq_ids ? m.seq_ids[i] : (int32_t)i;
    const bool known = seq >= 0 && (uint32_t)seq < g.max_seqs;
    pos = (m.first_pos ? (int64_t)m.first_pos[i] : known ? (int64_t)g.seq_lens[seq] - (e - b) : 0) + (row - b);
    return place_ok(g, seq, pos, tell);
}

// the lane's part of a position's rotation: its four dims' cosines and sines,
// the lane that holds the pairs' other halves
struct Turn {
    float c[4], s[4];
    int partner;
    bool on, second;  // this lane rotates; it holds the pairs' second members
};
__device__ __forceinline__ Turn load_turn(const float *row, int rot, bool neighbours, int lane) {
    Turn t;
    const int half = rot >> 1;
    t.on = 4 * lane < rot;
    t.second = !neighbours && 4 * lane >= half;
    t.partner = t.on ? (t.second ? lane - half / 4 : lane + half / 4) : lane;
    if (!t.on) return t;
    if (neighbours) {
        const float2 c = *reinterpret_cast<const float2 *>(row + 2 * lane);
        const float2 s = *reinterpret_cast<const float2 *>(row + half + 2 * lane);
        t.c[0] = t.c[1] = c.x;
        t.c[2] = t.c[3] = c.y;
        t.s[0] = t.s[1] = s.x;
        t.s[2] = t.s[3] = s.y;
    } else {
        const int p = 4 * lane - (t.second ? half : 0);
        const float4 c = *reinterpret_cast<const float4 *>(row + p), s = *reinterpret_cast<const float4 *>(row + half + p);
        t.c[0] = c.x, t.c[1] = c.y, t.c[2] = c.z, t.c[3] = c.w;
        t.s[0] = s.x, t.s[1] = s.y, t.s[2] = s.z, t.s[3] = s.w;
    }
    return t;
}
__device__ __forceinline__ float turn_first(float a, float b, float c, float s) {
    return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
}
__device__ __forceinline__ float turn_second(float b, float a, float c, float s) {
    return __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
}
__device__ __forceinline__ float4 rotate(float4 x, const Turn &t, bool neighbours) {
    if (neighbours) {
        if (!t.on) return x;
        return make_float4(turn_first(x.x, x.y, t.c[0], t.s[0]), turn_second(x.y, x.x, t.c[1], t.s[1]),
                           turn_first(x.z, x.w, t.c[2], t.s[2]), turn_second(x.w, x.z, t.c[3], t.s[3]));
    }
    float4 y;  // every lane takes part in the exchange
    y.x = __shfl_sync(0xffffffffu, x.x, t.partner);
    y.y = __shfl_sync(0xffffffffu, x.y, t.partner);
    y.z = __shfl_sync(0xffffffffu, x.z, t.partner);
    y.w = __shfl_sync(0xffffffffu, x.w, t.partner);
    if (!t.on) return x;
    if (t.second)
        return make_float4(turn_second(x.x, y.x, t.c[0], t.s[0]), turn_second(x.y, y.y, t.c[1], t.s[1]),
                           turn_second(x.z, y.z, t.c[2], t.s[2]), turn_second(x.w, y.w, t.c[3], t.s[3]));
    return make_float4(turn_first(x.x, y.x, t.c[0], t.s[0]), turn_first(x.y, y.y, t.c[1], t.s[1]),
                       turn_first(x.z, y.z, t.c[2], t.s[2]), turn_first(x.w, y.w, t.c[3], t.s[3]));
}

// ---------------------------------------------------------------------------
// whole tiles: 8 lanes per row, lane j holds dims 8j..8j+7 and 64+8j..64+8j+7
// ---------------------------------------------------------------------------
struct Row16 {
    float v[16];
    __device__ __forceinline__ static int dim(int i, int j) { return i < 8 ? 8 * j + i : 56 + 8 * j + i; }
};

// the same as it is in memory: loads that are issued long before their use
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
template <typename T>
__device__ __forceinline__ void store16(T *row, int j, const Row16 &r) {
#pragma unroll
    for (int q = 0; q < 4; q++)
        store4(row + Row16::dim(4 * q, j), make_float4(r.v[4 * q], r.v[4 * q + 1], r.v[4 * q + 2], r.v[4 * q + 3]));
}
__device__ __forceinline__ void store16(__half *row, int j, const Row16 &r) {
#pragma unroll
    for (int q = 0; q < 2; q++)
        *reinterpret_cast<uint4 *>(row + 64 * q + 8 * j) =
            make_uint4(pack_h2(r.v[8 * q], r.v[8 * q + 1]), pack_h2(r.v[8 * q + 2], r.v[8 * q + 3]),
                       pack_h2(r.v[8 * q + 4], r.v[8 * q + 5]), pack_h2(r.v[8 * q + 6], r.v[8 * q + 7]));
}
__device__ __forceinline__ uint32_t pack_b2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ void store16(__nv_bfloat16 *row, int j, const Row16 &r) {
#pragma unroll
    for (int q = 0; q < 2; q++)
        *reinterpret_cast<uint4 *>(row + 64 * q + 8 * j) =
            make_uint4(pack_b2(r.v[8 * q], r.v[8 * q + 1]), pack_b2(r.v[8 * q + 2], r.v[8 * q + 3]),
                       pack_b2(r.v[8 * q + 4], r.v[8 * q + 5]), pack_b2(r.v[8 * q + 6], r.v[8 * q + 7]));
}

// A row's rotation for this lane.  All 128 dims as halves: the pairs are (v[i],
// v[i + 8]).  Neighbours: (v[2i], v[2i + 1]), where the eight dims are below
// rotary_dim.  Both keep their angles for all heads of the row; halves of fewer
// dims read angles and the partner's values again for each head (from L1).
enum { kTurnWhole, kTurnNeighbours, kTurnPart };
template <int MODE>
struct Turn16 {
    float c[8], s[8];
    const float *row;
    __device__ __forceinline__ void load(const float *r, int j, int rot) {
        row = r;
        if constexpr (MODE != kTurnPart) {
#pragma unroll
            for (int q = 0; q < 2; q++) {
                if (MODE == kTurnNeighbours && 64 * q + 8 * j >= rot) continue;
                const float *at = MODE == kTurnWhole ? r + 8 * j + 4 * q : r + 32 * q + 4 * j;
                const float4 x = *reinterpret_cast<const float4 *>(at);
                const float4 y = *reinterpret_cast<const float4 *>(at + (rot >> 1));
                c[4 * q] = x.x, c[4 * q + 1] = x.y, c[4 * q + 2] = x.z, c[4 * q + 3] = x.w;
                s[4 * q] = y.x, s[4 * q + 1] = y.y, s[4 * q + 2] = y.z, s[4 * q + 3] = y.w;
            }
        }
    }
    template <typename T>
    __device__ __forceinline__ void apply(Row16 &x, const T *from, int j, int rot) const {
        if (MODE == kTurnWhole) {  // turn_first and turn_second, the products two at a time
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const uint64_t a = pair(x.v[i], x.v[i + 1]), b = pair(x.v[i + 8], x.v[i + 9]);
                const uint64_t cc = pair(c[i], c[i + 1]), ss = pair(s[i], s[i + 1]);
                float ac[2], bs[2], bc[2], as[2];
                unpair(mul2(a, cc), ac[0], ac[1]);
                unpair(mul2(b, ss), bs[0], bs[1]);
                unpair(mul2(b, cc), bc[0], bc[1]);
                unpair(mul2(a, ss), as[0], as[1]);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    x.v[i + e] = __fsub_rn(ac[e], bs[e]);
                    x.v[i + 8 + e] = __fadd_rn(bc[e], as[e]);
                }
            }
            return;
        }
        if (MODE == kTurnNeighbours) {
#pragma unroll
            for (int q = 0; q < 2; q++) {
                if (64 * q + 8 * j >= rot) continue;
#pragma unroll
                for (int i = 4 * q; i < 4 * q + 4; i++) {
                    const uint64_t ab = pair(x.v[2 * i], x.v[2 * i + 1]);
                    float ac, bc, as, bs;
                    unpair(mul2(ab, pair(c[i], c[i])), ac, bc);
                    unpair(mul2(ab, pair(s[i], s[i])), as, bs);
                    x.v[2 * i] = __fsub_rn(ac, bs);
                    x.v[2 * i + 1] = __fadd_rn(bc, as);
                }
            }
            return;
        }
        const int half = rot >> 1;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            float *v = x.v + 4 * q;
            const int d = Row16::dim(4 * q, j);
            if (d >= rot) continue;
            const bool second = d >= half;
            const int p = second ? d - half : d;
            const float4 cc = *reinterpret_cast<const float4 *>(row + p);
            const float4 ss = *reinterpret_cast<const float4 *>(row + half + p);
            const float4 o = load4(from + (second ? p : d + half));
            const float cs[4] = {cc.x, cc.y, cc.z, cc.w}, sn[4] = {ss.x, ss.y, ss.z, ss.w}, y[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int i = 0; i < 4; i++)
                v[i] = second ? turn_second(v[i], y[i], cs[i], sn[i]) : turn_first(v[i], y[i], cs[i], sn[i]);
        }
    }
};

template <int LANES, bool MIN>
__device__ __forceinline__ float lanes_extreme(float v) {
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, v, o);
        v = MIN ? fminf(v, u) : fmaxf(v, u);
    }
    return v;
}
__device__ __forceinline__ void put2(uint8_t *p, uint32_t a, uint32_t b) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(a, b);
}

// K (which 0) or V of the row of token t into the tile's image, by
// store_token's rules and layout.  Returns false, in every lane that sees it,
// for what those rules take in an order of their own: a NaN, or a minimum of
// zero (whose sign is the first zero's); the tile then goes row by row.
template <int CODEC>
__device__ bool put_row(uint8_t *tile, int t, int which, const Row16 &x, int j);

// Eight codes as two words of biased bytes.  q8_pack4 divides; here the product
// with 1 / s decides unless it lies within 1e-4 of a tie or no number is (then
// false): its error is below 127 x 2^-22.  The sum with 1.5 x 2^23 + 128 rounds
// to the nearest whole number, ties to even, and has the byte at its low end.
__device__ __forceinline__ bool q8_words(const float *v, float per, uint32_t &lo, uint32_t &hi) {
    const float magic = 12583040.f;
    const uint64_t m2 = pair(magic, magic), n2 = pair(-magic, -magic), r2 = pair(per, per);
    uint32_t bits[8];
    bool sure = true;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint64_t y = mul2(pair(v[i], v[i + 1]), r2), t = add2(y, m2);
        float y0, y1, n0, n1;
        unpair(y, y0, y1);
        unpair(add2(t, n2), n0, n1);
        sure &= fabsf(y0 - n0) < 0.4999f && fabsf(y1 - n1) < 0.4999f;
        unpair(t, bits[i], bits[i + 1]);
    }
    lo = prmt(prmt(bits[0], bits[1], 0x0040u), prmt(bits[2], bits[3], 0x0040u), 0x5410u);
    hi = prmt(prmt(bits[4], bits[5], 0x0040u), prmt(bits[6], bits[7], 0x0040u), 0x5410u);
    return sure;
}
// `top` is the largest finite value that s was made for
__device__ __forceinline__ void put_q8(uint8_t *tile, int t, int which, const Row16 &x, int j, float s0, float s1,
                                       float top0, float top1) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const float s = h ? s1 : s0, top = h ? top1 : top0;
        const float *v = x.v + 8 * h;
        const float per = __fdiv_rn(1.f, s);
        uint32_t lo, hi;
        if (!q8_words(v, per, lo, hi) || !(top * per < 127.4f)) {
            lo = q8_pack4(make_float4(v[0], v[1], v[2], v[3]), s);
            hi = q8_pack4(make_float4(v[4], v[5], v[6], v[7]), s);
        }
        const int d = 64 * h + 8 * j;
        if (!which) {
            put2(tile + k8_off(t, d), lo, hi);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) tile[v8_off(t, d + i)] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
        }
    }
}
__device__ __forceinline__ float finite_top(const float *v) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float a = fabsf(v[i]);
        if (a < INFINITY) m = fmaxf(m, a);
    }
    return m;
}
template <>
__device__ __forceinline__ bool put_row<QWN_KV_CODEC_Q8_HEAD_F16>(uint8_t *tile, int t, int which, const Row16 &x, int j) {
    const float top = lanes_extreme<8, false>(fmaxf(finite_top(x.v), finite_top(x.v + 8)));
    const uint16_t h = head_scale16(top);
    const float s = h2f(h);
    put_q8(tile, t, which, x, j, s, s, top, top);
    if (j == 0) *reinterpret_cast<uint16_t *>(tile + (which ? 4128 : 4096) + s16_off(t)) = h;
    return true;
}
template <>
__device__ __forceinline__ bool put_row<QWN_KV_CODEC_Q8_B64_F32>(uint8_t *tile, int t, int which, const Row16 &x, int j) {
    float s[2], m[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        m[h] = lanes_extreme<8, false>(finite_top(x.v + 8 * h));
        s[h] = m[h] > 0.f ? __fdiv_rn(m[h], 127.f) : 1.f;
    }
    put_q8(tile, t, which, x, j, s[0], s[1], m[0], m[1]);
    if (j < 2) *reinterpret_cast<float *>(tile + (which ? 4224 : 4096) + s32_off(t, j)) = j ? s[1] : s[0];
    return true;
}
template <>
__device__ __forceinline__ bool put_row<QWN_KV_CODEC_F16>(uint8_t *tile, int t, int which, const Row16 &x, int j) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const float *v = x.v + 8 * h;
        *reinterpret_cast<uint4 *>(tile + f16_off(which, t, 64 * h + 8 * j)) =
            make_uint4(f16_bits(v[0]) | (f16_bits(v[1]) << 16), f16_bits(v[2]) | (f16_bits(v[3]) << 16),
                       f16_bits(v[4]) | (f16_bits(v[5]) << 16), f16_bits(v[6]) | (f16_bits(v[7]) << 16));
    }
    return true;
}
// smallest value and range of a group held by LANES lanes' halves, and the
// range's inverse.  False where store_token's order or special cases matter: a
// NaN, a minimum of zero (its sign is the first zero's), parameters beyond fp16.
struct Span {
    float mn, range, inv;
};
__device__ __forceinline__ float min_nan(float a, float b) {  // NaN where either is one
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <int LANES>
__device__ __forceinline__ bool group_span(const float *v, Span &g) {
    float mn = v[0], mx = v[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
        mn = min_nan(mn, v[i]);
        mx = fmaxf(mx, v[i]);
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
        mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    g.mn = mn;
    g.range = __fsub_rn(mx, mn);
    g.inv = g.range > 1e-8f ? __fdiv_rn(1.0f, g.range) : 0.f;
    return fabsf(mn) > 0.f && fabsf(mn) < 65536.f && g.range < 65536.f;
}
// both parameters cut off to fp16 (as tq_f32_to_f16 does below 65536): range low, minimum high
__device__ __forceinline__ uint32_t span_params(const Span &g) {
    uint32_t r;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(g.mn), "f"(g.range));
    return r;
}
// tq_code of eight numbers of the span's group: the two sums towards zero are
// floor(y + 1/2) without roundf's exceptions (y is in [0, levels + 2^-19]), left
// in the low bits; the number on top of them is 0x4B000000
__device__ __forceinline__ void span_codes(const float *v, const Span &g, float even, float odd, uint32_t (&c)[8]) {
    const uint64_t mn = pair(-g.mn, -g.mn), inv = pair(g.inv, g.inv), levels = pair(even, odd);
    const uint64_t whole = pair(8388608.f, 8388608.f);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float y0, y1;
        unpair(mul2(mul2(add2(pair(v[i], v[i + 1]), mn), inv), levels), y0, y1);
        unpair(add2_down(pair(__fadd_rz(y0, 0.5f), __fadd_rz(y1, 0.5f)), whole), c[i], c[i + 1]);
    }
}
constexpr uint32_t kCodeBase = 0x4B000000u;
template <>
__device__ __forceinline__ bool put_row<QWN_KV_CODEC_Q4_G32>(uint8_t *tile, int t, int which, const Row16 &x, int j) {
    bool ok = true;
    uint32_t nib[2];  // the half's eight codes: K in byte i dims i and i + 4, V in nibble i dim i
#pragma unroll
    for (int h = 0; h < 2; h++) {
        Span g;
        uint32_t code[8];
        ok &= group_span<4>(x.v + 8 * h, g);
        span_codes(x.v + 8 * h, g, 15.f, 15.f, code);
        nib[h] = 0;
        uint32_t base = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int at = which ? 4 * i : i < 4 ? 8 * i : 8 * (i - 4) + 4;
            nib[h] += code[i] << at;
            base += kCodeBase << at;
        }
        nib[h] -= base;
        const int c = 2 * h + (j >> 2);
        if ((j & 3) == 0)
            *reinterpret_cast<uint32_t *>(tile + (which ? 2304 : 2048) + 32 * (t & 7) + 8 * c + 4 * (t >> 3)) =
                span_params(g);
        if (!which) *reinterpret_cast<uint32_t *>(tile + 64 * t + 16 * (j & 3) + 4 * c) = nib[h];
    }
    if (which) {
        // a byte holds dims gid and gid + 8 of a block of 16: lanes j and j + 1; the even one writes half 0
        const uint32_t other = __shfl_xor_sync(0xffffffffu, j & 1 ? nib[0] : nib[1], 1);
        const int h = j & 1, mb = 4 * h + (j >> 1);
        const uint32_t low = h ? other : nib[0], high = h ? nib[1] : other;
        const uint32_t even = (low & 0x0F0F0F0Fu) | ((high << 4) & 0xF0F0F0F0u);
        const uint32_t odd = ((low >> 4) & 0x0F0F0F0Fu) | (high & 0xF0F0F0F0u);
#pragma unroll
        for (int gid = 0; gid < 8; gid++) {
            const int lv = 4 * gid + ((t & 7) >> 1);
            const int chunk = (mb >> 2) ^ ((lv >> 2) & 1);
            tile[1024 + 32 * lv + 16 * chunk + 4 * (mb & 3) + (t >> 3) + 2 * (t & 1)] =
                (uint8_t)((gid & 1 ? odd : even) >> (8 * (gid >> 1)));
        }
    }
    return ok;
}
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
// the image starts as zeros: a word holds codes of several lanes
template <>
__device__ __forceinline__ bool put_row<QWN_KV_CODEC_TQ35_G64>(uint8_t *tile, int t, int which, const Row16 &x, int j) {
    uint8_t *half = tile + which * 1024;
    bool ok = true;
    uint32_t code[16];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        Span g;
        uint32_t c[8];
        ok &= group_span<8>(x.v + 8 * h, g);
        span_codes(x.v + 8 * h, g, 15.f, 7.f, c);
#pragma unroll
        for (int i = 0; i < 8; i++) code[8 * h + i] = c[i] & 15u;
        if (j == 0)
            *reinterpret_cast<uint32_t *>(half + 896 + 16 * (t & 7) + 8 * h + 4 * (t >> 3)) = span_params(g);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {  // dims 2i and 2i + 1 of both halves
        const TqPlace p = tq_place(which, t, 4 * j + i);
        auto put = [&](uint32_t at, uint32_t v) { atomicOr(reinterpret_cast<uint32_t *>(half + at), v); };
        const uint32_t o0 = code[2 * i + 1], o1 = code[9 + 2 * i];
        put(p.even, code[2 * i] << (4 * p.n));
        put(p.even + p.even_step, code[8 + 2 * i] << (4 * p.n));
        put(p.odd, (o0 | ((o1 & 1u) << 3)) << (4 * p.n));
        put(p.plane & ~3u, (o1 >> 1) << (2 * p.n + 8 * (p.plane & 3u)));
    }
    return ok;
}

struct RotaryArgs {
    RowMap rows;
    const int32_t *rotary_pos;
    const float *table;
    uint32_t layer, query_heads, rot, max_position, query_out_dtype;
    bool neighbours;
    uint64_t query_stride, key_stride, value_stride;
};

// whether a row's angles are in the table
__device__ __forceinline__ bool angle_ok(const StoreGeo &g, const RotaryArgs &a, int64_t pos, uint32_t row,
                                         int32_t &angle, bool tell) {
    if (!a.rot) return true;
    angle = a.rotary_pos ? a.rotary_pos[row] : (int32_t)pos;
    if (angle >= 0 && (uint32_t)angle < a.max_position) return true;
    if (tell) latch(g.status, QWN_KV_STATUS_BAD_LENGTH);
    return false;
}

__device__ __forceinline__ void store_any(void *out, uint32_t dtype, size_t at, float4 v) {
    if (dtype == QWN_DTYPE_F32) store4(static_cast<float *>(out) + at, v);
    else if (dtype == QWN_DTYPE_F16) store4(static_cast<__half *>(out) + at, v);
    else store4(static_cast<__nv_bfloat16 *>(out) + at, v);
}

// one row and head by a warp: rotate and store
template <int CODEC, typename T>
__device__ __forceinline__ void append_row(const StoreGeo &g, const RotaryArgs &a, bool ok, int32_t seq, int32_t pos,
                                           int32_t angle, uint32_t row, uint32_t slot, float4 x, float4 v,
                                           void *query_out, int lane) {
    if (ok && a.rot) {
        const Turn t = load_turn(a.table + (size_t)angle * a.rot, (int)a.rot, a.neighbours, lane);
        x = rotate(x, t, a.neighbours);
    }
    if (slot < g.kv_heads) {
        uint8_t *tile = ok ? tile_for(g, seq, a.layer, slot, pos) : nullptr;
        if (tile) store_token<CODEC>(tile, pos & 15, x, v, lane);
    } else {
        store_any(query_out, a.query_out_dtype,
                  ((size_t)row * a.query_heads + slot - g.kv_heads) * kHeadDim + 4 * lane,
                  ok ? x : make_float4(0.f, 0.f, 0.f, 0.f));
    }
}

// one warp per (row, head): the kv heads (K and V together), then the query heads
template <int CODEC, typename T>
__global__ void __launch_bounds__(128) append_rotary_kernel(StoreGeo g, RotaryArgs a, const T *query, const T *key,
                                                            const T *value, void *query_out) {
    const uint64_t wg = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const uint32_t slots = g.kv_heads + a.query_heads;
    const uint32_t row = (uint32_t)(wg / slots), slot = (uint32_t)(wg % slots);
    launch_dependents();
    wait_previous();
    if (row >= a.rows.num_rows) return;
    const bool is_kv = slot < g.kv_heads;
    const float4 x = is_kv ? load4(key + (size_t)row * a.key_stride + slot * kHeadDim + 4 * lane)
                           : load4(query + (size_t)row * a.query_stride + (slot - g.kv_heads) * kHeadDim + 4 * lane);
    const float4 v = is_kv ? load4(value + (size_t)row * a.value_stride + slot * kHeadDim + 4 * lane) : x;
    int32_t seq = 0, angle = 0;
    int64_t pos = 0;
    const bool tell = lane == 0 && slot == 0;
    const bool ok = find_row(g, a.rows, row, seq, pos, tell) && angle_ok(g, a, pos, row, angle, tell);
    append_row<CODEC, T>(g, a, ok, seq, (int32_t)pos, angle, row, slot, x, v, query_out, lane);
}

// the rows of a batch by tiles of the cache: unit u is tile u - base_i of
// sequence i, base_i = row_begin[i] / 16 + 2 i.  n rows touch at most n / 16 + 2
// tiles, so that num_rows / 16 + 2 num_seqs units cover them all without a
// table; some stay empty.
struct Unit {
    uint32_t first, count;  // rows; none where count is 0
    int32_t seq, len;       // -1 and 0: no such sequence
    int64_t pos;            // of the first row
};
// by one warp; the other warps of the CTA wait for it (with every warp doing
// this, half of the kernel's instructions were these)
__device__ __forceinline__ Unit find_unit(const StoreGeo &g, const RowMap &m, uint32_t u) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, n = m.num_seqs;  // the last of sequences lo .. lo + n - 1 whose base is not beyond u
    while (n > 1) {                   // 32 at a time
        const uint32_t step = (n + 31) / 32, i = lo + lane * step;
        const bool below = lane * step < n && (uint32_t)max(m.row_begin[i], 0) / 16 + 2 * i <= u;
        const uint32_t last = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1u);
        n = min(step, n - last * step);
        lo += last * step;
    }
    Unit t = {0, 0, -1, 0, 0};
    const int64_t b = max(m.row_begin[lo], 0), e = m.row_begin[lo + 1];
    const int64_t n_rows = min(e, (int64_t)m.num_rows) - b;
    const uint32_t base = (uint32_t)b / 16 + 2 * lo;
    const int32_t seq = m.seq_ids ? m.seq_ids[lo] : (int32_t)lo;
    if (seq >= 0 && (uint32_t)seq < g.max_seqs) {
        t.seq = seq;
        t.len = g.seq_lens[seq];
    }
    if (n_rows <= 0 || u < base) return t;
    const int64_t p0 = m.first_pos ? m.first_pos[lo] : t.seq < 0 ? 0 : t.len - (e - b);
    const int64_t tile = (p0 >> 4) + (u - base);
    const int64_t from = max(p0, tile << 4), to = min(p0 + n_rows, (tile + 1) << 4);
    if (from >= to) return t;
    t.first = (uint32_t)(b + (from - p0));
    t.count = (uint32_t)(to - from);
    t.pos = from;
    return t;
}
// the tile of a unit's rows for one head and the layer, whose page one of their
// positions finds; null where none of them exists
__device__ __forceinline__ uint8_t *unit_tile(const StoreGeo &g, const Unit &u, uint32_t layer, uint32_t head) {
    const int64_t some = max(u.pos, (int64_t)0);
    if (u.seq < 0 || some >= min(u.pos + u.count, (int64_t)u.len)) return nullptr;
    return tile_for(g, u.seq, layer, head, (int32_t)some);
}
// rows before the first sequence's and after the last one's: unit 0 looks at them
struct Gaps {
    int64_t before, after, count;
    __device__ __forceinline__ explicit Gaps(const RowMap &m) {
        const int64_t n = m.num_rows;
        before = min(max((int64_t)m.row_begin[0], (int64_t)0), n);
        after = min(max((int64_t)m.row_begin[m.num_seqs], before), n);
        count = before + n - after;
    }
    __device__ __forceinline__ uint32_t row(int64_t i) const { return (uint32_t)(i < before ? i : after + i - before); }
};

constexpr int kTileThreads = 128;  // 16 rows of 8 lanes

// one CTA per (tile, kv head): its K and V, and the query heads that read it
template <int CODEC, typename T, int MODE>
__global__ void __launch_bounds__(kTileThreads, 6) append_tiles_kernel(StoreGeo g, RotaryArgs a, const T *query,
                                                                    const T *key, const T *value, void *query_out) {
    constexpr int kImage = (int)tile_bytes_of(CODEC), kAhead = sizeof(T) == 4 ? 2 : 4;  // query heads in flight
    __shared__ __align__(16) uint8_t buf[2 * 16 * kHeadDim * 4];  // the tile's image, or K and V of its rows in fp32
    __shared__ uint8_t stored[16];
    const uint32_t head = blockIdx.y, group = a.query_heads / g.kv_heads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int j = threadIdx.x & 7, r = threadIdx.x >> 3;
    launch_dependents();
    wait_previous();
    const Row16 zero = {};
    auto put_query = [&](uint32_t row, uint32_t q, const Row16 &x) {
        const size_t at = ((size_t)row * a.query_heads + head * group + q) * kHeadDim;
        if (a.query_out_dtype == QWN_DTYPE_F32) store16(static_cast<float *>(query_out) + at, j, x);
        else if (a.query_out_dtype == QWN_DTYPE_F16) store16(static_cast<__half *>(query_out) + at, j, x);
        else store16(static_cast<__nv_bfloat16 *>(query_out) + at, j, x);
    };
    if (blockIdx.x == 0) {  // rows of no sequence
        const Gaps gaps(a.rows);
        if (gaps.count > 0 && head == 0 && threadIdx.x == 0) latch(g.status, QWN_KV_STATUS_BAD_LENGTH);
        for (int64_t i = r; i < gaps.count; i += 16)
            for (uint32_t q = 0; q < group; q++) put_query(gaps.row(i), q, zero);
    }
    __shared__ Unit unit;
    __shared__ uint8_t *unit_at;
    if (warp == 0) {
        const Unit t = find_unit(g, a.rows, blockIdx.x);
        if (lane == 0) unit = t;
    }
    __syncthreads();
    const Unit u = unit;
    if (u.count == 0) return;
    const bool have = (uint32_t)r < u.count;
    const uint32_t row = u.first + (have ? (uint32_t)r : 0);
    const T *kr = key + (size_t)row * a.key_stride + head * kHeadDim;
    const T *vr = value + (size_t)row * a.value_stride + head * kHeadDim;
    const T *qr = query + (size_t)row * a.query_stride + (size_t)head * group * kHeadDim;
    Raw16<T> kw, vw, qw[kAhead];
    kw.load(kr, j);
    vw.load(vr, j);
#pragma unroll
    for (uint32_t q = 0; q < kAhead; q++)
        if (q < group) qw[q].load(qr + q * kHeadDim, j);
    if (threadIdx.x == 0) unit_at = unit_tile(g, u, a.layer, head);
    int32_t angle = 0;
    const bool tell = have && j == 0 && head == 0;
    const bool ok = have && unit_row_ok(g, u.seq, u.len, u.pos + r, tell) && angle_ok(g, a, u.pos + r, row, angle, tell);
    const bool turns = ok && (MODE != kTurnPart || a.rot);
    Turn16<MODE> turn;
    if (turns) turn.load(a.table + (size_t)angle * a.rot, j, (int)a.rot);
    for (uint32_t q0 = 0; q0 < group; q0 += kAhead) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; i++) {
            const uint32_t q = q0 + i;
            if (q >= group) break;
            if (ok) {
                Row16 x = qw[i].row();
                if (MODE != kTurnPart || a.rot) turn.apply(x, qr + q * kHeadDim, j, (int)a.rot);
                // query_out may be query: the row's lanes have read their partners' values
                if (MODE == kTurnPart) __syncwarp(0xFFu << (8 * (lane >> 3)));
                put_query(row, q, x);
            } else if (have) {
                put_query(row, q, zero);
            }
            if (q + kAhead < group) qw[i].load(qr + (q + kAhead) * kHeadDim, j);
        }
    }
    Row16 k = kw.row();
    const Row16 v = vw.row();
    if (turns) turn.apply(k, kr, j, (int)a.rot);
    if (CODEC == QWN_KV_CODEC_TQ35_G64)
        for (int i = threadIdx.x; i < kImage / 16; i += kTileThreads)
            reinterpret_cast<uint4 *>(buf)[i] = make_uint4(0, 0, 0, 0);
    // 16 new tokens: the whole tile is put together here
    const bool whole = __syncthreads_and(ok && u.count == 16);
    uint8_t *tile = unit_at;
    if (whole && tile) {
        const bool fine = put_row<CODEC>(buf, r, 0, k, j) & put_row<CODEC>(buf, r, 1, v, j);
        if (__syncthreads_and(fine)) {
            for (int i = threadIdx.x; i < kImage / 16; i += kTileThreads)
                reinterpret_cast<uint4 *>(tile)[i] = reinterpret_cast<const uint4 *>(buf)[i];
            return;
        }
    }
    // a tile filled in part, or one whose codes depend on its values' order: token by token
    if (j == 0) stored[r] = ok;
    float *rows = reinterpret_cast<float *>(buf);
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int d = Row16::dim(4 * q, j);
        store4(rows + r * kHeadDim + d, make_float4(k.v[4 * q], k.v[4 * q + 1], k.v[4 * q + 2], k.v[4 * q + 3]));
        store4(rows + (16 + r) * kHeadDim + d, make_float4(v.v[4 * q], v.v[4 * q + 1], v.v[4 * q + 2], v.v[4 * q + 3]));
    }
    __syncthreads();
    if (!tile) return;
    for (uint32_t i = warp; i < u.count; i += kTileThreads / 32)
        if (stored[i])
            store_token<CODEC>(tile, (int)((u.pos + i) & 15), load4(rows + i * kHeadDim + 4 * lane),
                               load4(rows + (16 + i) * kHeadDim + 4 * lane), lane);
}

// ---------------------------------------------------------------------------
// the way back, by tiles: the tile into shared memory in 16-byte loads, its
// rows out of it by 8 lanes each
// ---------------------------------------------------------------------------
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

// one CTA per tile and `heads` kv heads: the next head's tile is on its way into
// shared memory while this one's rows go out
template <int CODEC, typename T>
__global__ void __launch_bounds__(kTileThreads) load_tiles_kernel(StoreGeo g, RowMap m, uint32_t layer, uint32_t heads,
                                                                  uint64_t key_stride, uint64_t value_stride, T *key,
                                                                  T *value) {
    constexpr int kImage = (int)tile_bytes_of(CODEC);
    __shared__ __align__(16) uint8_t image[2][kImage];
    const uint32_t h0 = blockIdx.y * heads, h1 = min(h0 + heads, g.kv_heads);
    launch_dependents();
    wait_previous();
    const int j = threadIdx.x & 7, r = threadIdx.x >> 3;
    const Row16 zero = {};
    auto put = [&](uint32_t row, uint32_t head, const Row16 &k, const Row16 &v) {
        if (key) store16(key + (size_t)row * key_stride + head * kHeadDim, j, k);
        if (value) store16(value + (size_t)row * value_stride + head * kHeadDim, j, v);
    };
    if (blockIdx.x == 0) {  // rows of no sequence
        const Gaps gaps(m);
        if (gaps.count > 0 && h0 == 0 && threadIdx.x == 0) latch(g.status, QWN_KV_STATUS_BAD_LENGTH);
        for (int64_t i = r; i < gaps.count; i += 16)
            for (uint32_t h = h0; h < h1; h++) put(gaps.row(i), h, zero, zero);
    }
    __shared__ Unit unit;
    __shared__ const uint8_t *unit_at;
    if (threadIdx.x < 32) {
        const Unit t = find_unit(g, m, blockIdx.x);
        if (threadIdx.x == 0) {
            unit = t;
            unit_at = t.count ? unit_tile(g, t, layer, h0) : nullptr;
        }
    }
    __syncthreads();
    const Unit u = unit;
    if (u.count == 0) return;
    const uint8_t *tile = unit_at;
    const size_t next = (size_t)g.tpp * g.tile_bytes;  // the following head's tile
    auto fetch = [&](uint32_t h) {
        if (tile && h < h1)
            for (int i = threadIdx.x; i < kImage / 16; i += kTileThreads)
                cp_async16(image[(h - h0) & 1] + 16 * i, tile + (h - h0) * next + 16 * i);
        cp_async_commit();
    };
    fetch(h0);
    const int64_t pos = u.pos + r;
    const bool have = (uint32_t)r < u.count;
    const bool ok = have && unit_row_ok(g, u.seq, u.len, pos, j == 0 && h0 == 0) && tile;
    const int t = (int)(pos & 15);
    for (uint32_t h = h0; h < h1; h++) {
        fetch(h + 1);
        cp_async_wait1();
        __syncthreads();
        const uint8_t *in = image[(h - h0) & 1];
        if (ok) put(u.first + r, h, take_row<CODEC>(in, t, 0, j), take_row<CODEC>(in, t, 1, j));
        else if (have) put(u.first + r, h, zero, zero);
        __syncthreads();  // before the tile after the next lands here
    }
}

// one warp per (row, head): K and V of a cached token back to rows (one token
// per sequence, and rows that are not 16-byte aligned)
template <int CODEC, typename T>
__global__ void __launch_bounds__(128) load_rows_kernel(StoreGeo g, RowMap m, uint32_t layer, uint64_t key_stride,
                                                        uint64_t value_stride, T *key, T *value) {
    const uint64_t wg = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const uint32_t row = (uint32_t)(wg / g.kv_heads), h = (uint32_t)(wg % g.kv_heads);
    launch_dependents();
    wait_previous();
    if (row >= m.num_rows) return;
    int32_t seq = 0;
    int64_t pos = 0;
    const uint8_t *tile = nullptr;
    if (find_row(g, m, row, seq, pos, lane == 0 && h == 0)) tile = tile_for(g, seq, layer, h, (int32_t)pos);
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    const size_t at = h * kHeadDim + 4 * lane;
    const int t = (int)(pos & 15);
    if (key) store4(key + (size_t)row * key_stride + at, tile ? load_token<CODEC>(tile, t, 0, lane) : zero);
    if (value) store4(value + (size_t)row * value_stride + at, tile ? load_token<CODEC>(tile, t, 1, lane) : zero);
}

// f.operator()<CODEC, T>() for the pool's codec and the rows' type
template <int CODEC, class F>
cudaError_t with_type(uint32_t dtype, F &&f) {
    switch (dtype) {
        case QWN_DTYPE_F32: return f(std::integral_constant<int, CODEC>(), (float *)nullptr);
        case QWN_DTYPE_F16: return f(std::integral_constant<int, CODEC>(), (__half *)nullptr);
        case QWN_DTYPE_BF16: return f(std::integral_constant<int, CODEC>(), (__nv_bfloat16 *)nullptr);
        default: return cudaErrorNotSupported;
    }
}
template <class F>
cudaError_t with_codec(uint32_t codec, uint32_t dtype, F &&f) {
    switch (codec) {
        case QWN_KV_CODEC_Q8_B64_F32: return with_type<QWN_KV_CODEC_Q8_B64_F32>(dtype, f);
        case QWN_KV_CODEC_Q8_HEAD_F16: return with_type<QWN_KV_CODEC_Q8_HEAD_F16>(dtype, f);
        case QWN_KV_CODEC_TQ35_G64: return with_type<QWN_KV_CODEC_TQ35_G64>(dtype, f);
        case QWN_KV_CODEC_Q4_G32: return with_type<QWN_KV_CODEC_Q4_G32>(dtype, f);
        case QWN_KV_CODEC_F16: return with_type<QWN_KV_CODEC_F16>(dtype, f);
        default: return cudaErrorNotSupported;
    }
}

uint64_t value_bytes(uint32_t dtype) { return dtype == QWN_DTYPE_F32 ? 4 : 2; }
// rows start on `values` values
bool rows_aligned(const void *p, uint64_t stride, uint32_t dtype, uint64_t values = 4) {
    return (uintptr_t)p % (value_bytes(dtype) * values) == 0 && stride % values == 0;
}
// 16-byte accesses, which the tile kernels make
bool rows_wide(const void *p, uint64_t stride, uint32_t dtype) {
    return rows_aligned(p, stride, dtype, 16 / value_bytes(dtype));
}
// units of find_unit for a batch
uint64_t unit_count(uint32_t rows, uint32_t seqs) { return (uint64_t)rows / 16 + 2 * (uint64_t)seqs; }
}  // namespace
}  // namespace qkv

using namespace qkv;

QWN_CUDA_ABI_API int qwn_kv_append_rotary(QwnKvPoolHandle *h, const QwnKvAppendRotaryRequest *r) {
    Pool *p = pool_from(h);
    if (!p || !r || !header_ok(r->header, sizeof(*r))) {
        set_error("qwn_kv_append_rotary: bad handle or header");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    const uint64_t kv_width = (uint64_t)p->kv_heads * kHeadDim, q_width = (uint64_t)r->query_heads * kHeadDim;
    const uint64_t ks = r->key_stride ? r->key_stride : kv_width, vs = r->value_stride ? r->value_stride : kv_width;
    const uint64_t qs = r->query_stride ? r->query_stride : q_width;
    if (r->layer >= p->layers || r->num_seqs > p->max_seqs || !dtype_ok(r->dtype))
        return invalid("qwn_kv_append_rotary: layer, num_seqs or dtype out of range");
    if (r->num_rows > 0x7FFFFFFFu || (!r->row_begin_dev && r->num_rows != r->num_seqs))
        return invalid("qwn_kv_append_rotary: without row_begin_dev there is one row per sequence");
    if (r->rotary_dim % 8 || r->rotary_dim > (uint32_t)kHeadDim || r->rotary_style > QWN_ROTARY_NEIGHBOURS ||
        (r->rotary_dim && (!r->rotations_dev || r->max_position == 0 || (uintptr_t)r->rotations_dev % 16)))
        return invalid("qwn_kv_append_rotary: rotary_dim must be a multiple of 8 up to 128 with a 16-byte aligned table");
    if (r->query_heads && (r->query_heads % p->kv_heads || r->query_heads > p->max_query_heads || !r->query_dev ||
                           !r->query_out_dev || !dtype_ok(r->query_out_dtype)))
        return invalid("qwn_kv_append_rotary: query heads need query_dev, query_out_dev and the pool's limits");
    if (r->num_rows == 0) return QWN_CUDA_STATUS_OK;
    if (r->num_seqs == 0) return invalid("qwn_kv_append_rotary: rows without a sequence");
    if (!r->key_dev || !r->value_dev) return invalid("qwn_kv_append_rotary: key_dev and value_dev are needed");
    if (ks < kv_width || vs < kv_width || (r->query_heads && qs < q_width))
        return invalid("qwn_kv_append_rotary: a row stride is shorter than the row");
    if (!rows_aligned(r->key_dev, ks, r->dtype) || !rows_aligned(r->value_dev, vs, r->dtype) ||
        (r->query_heads && (!rows_aligned(r->query_dev, qs, r->dtype) ||
                            !rows_aligned(r->query_out_dev, q_width, r->query_out_dtype))))
        return invalid("qwn_kv_append_rotary: rows must start on four values (pointers and strides)");
    if (r->query_heads) {
        const uint64_t in = value_bytes(r->dtype), ob = value_bytes(r->query_out_dtype);
        const RowSpan out = {(uintptr_t)r->query_out_dev, q_width * ob, q_width * ob, r->num_rows};
        auto met = [&](const void *p, uint64_t stride, uint64_t width) {
            return rows_meet({(uintptr_t)p, stride * in, width * in, r->num_rows}, out);
        };
        // in place a row's output lies on its own input, which the writing threads have read
        const bool in_place = r->query_out_dev == r->query_dev && in == ob && (qs == q_width || r->num_rows == 1);
        if ((!in_place && met(r->query_dev, qs, q_width)) || met(r->key_dev, ks, kv_width) || met(r->value_dev, vs, kv_width))
            return invalid("qwn_kv_append_rotary: query_out overlaps rows that are still read");
    }
    cudaSetDevice(p->device);
    RotaryArgs a{};
    a.rows = {r->seq_ids_dev, r->row_begin_dev, r->first_pos_dev, r->num_seqs, r->num_rows};
    a.rotary_pos = r->rotary_pos_dev;
    a.table = r->rotations_dev;
    a.layer = r->layer;
    a.query_heads = r->query_heads;
    a.rot = r->rotary_dim;
    a.max_position = r->max_position;
    a.query_out_dtype = r->query_out_dtype;
    a.neighbours = r->rotary_style == QWN_ROTARY_NEIGHBOURS;
    a.query_stride = qs;
    a.key_stride = ks;
    a.value_stride = vs;
    const StoreGeo g = store_geo(p);
    cudaStream_t s = stream_of(p, r->stream);
    // runs of rows go by tiles; one row per sequence, or rows off the 16-byte grid, one by one
    // (16384 rows of 32 + 2 x 8 bf16 heads into 4-bit pages: 69 us by tiles, 289 one by one)
    const bool tiles = r->row_begin_dev && rows_wide(r->key_dev, ks, r->dtype) && rows_wide(r->value_dev, vs, r->dtype) &&
                       (!r->query_heads || (rows_wide(r->query_dev, qs, r->dtype) &&
                                            rows_wide(r->query_out_dev, q_width, r->query_out_dtype)));
    const uint64_t ctas = tiles ? unit_count(r->num_rows, r->num_seqs)
                                : ((uint64_t)r->num_rows * (p->kv_heads + r->query_heads) + 3) / 4;
    if (ctas > 0x7FFFFFFFull || (tiles && p->kv_heads > 65535u))
        return invalid("qwn_kv_append_rotary: too many rows for one call");
    const cudaError_t e = with_codec(p->codec, r->dtype, [&](auto codec, auto *type) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int C = decltype(codec)::value;
        const T *q = static_cast<const T *>(r->query_dev), *k = static_cast<const T *>(r->key_dev),
                *v = static_cast<const T *>(r->value_dev);
        const dim3 grid((unsigned)ctas, tiles ? p->kv_heads : 1);
        if (!tiles) return launch_next(append_rotary_kernel<C, T>, grid, 128, s, g, a, q, k, v, r->query_out_dev);
        const auto kernel = a.neighbours && a.rot                 ? append_tiles_kernel<C, T, kTurnNeighbours>
                            : a.rot == (uint32_t)kHeadDim ? append_tiles_kernel<C, T, kTurnWhole>
                                                          : append_tiles_kernel<C, T, kTurnPart>;
        return launch_next(kernel, grid, kTileThreads, s, g, a, q, k, v, r->query_out_dev);
    });
    if (e != cudaSuccess) { set_cuda_error("qwn_kv_append_rotary", e); return QWN_CUDA_STATUS_RUNTIME_ERROR; }
    return QWN_CUDA_STATUS_OK;
}

QWN_CUDA_ABI_API int qwn_kv_load_tokens(QwnKvPoolHandle *h, const QwnKvLoadTokensRequest *r) {
    Pool *p = pool_from(h);
    if (!p || !r || !header_ok(r->header, sizeof(*r))) {
        set_error("qwn_kv_load_tokens: bad handle or header");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    const uint64_t width = (uint64_t)p->kv_heads * kHeadDim;
    const uint64_t ks = r->key_stride ? r->key_stride : width, vs = r->value_stride ? r->value_stride : width;
    if (r->layer >= p->layers || r->num_seqs > p->max_seqs || !dtype_ok(r->dtype))
        return invalid("qwn_kv_load_tokens: layer, num_seqs or dtype out of range");
    if (r->num_rows > 0x7FFFFFFFu || (!r->row_begin_dev && r->num_rows != r->num_seqs))
        return invalid("qwn_kv_load_tokens: without row_begin_dev there is one row per sequence");
    if (r->num_rows == 0) return QWN_CUDA_STATUS_OK;
    if (r->num_seqs == 0) return invalid("qwn_kv_load_tokens: rows without a sequence");
    if (!r->key_out_dev && !r->value_out_dev) return invalid("qwn_kv_load_tokens: no output");
    if (ks < width || vs < width) return invalid("qwn_kv_load_tokens: a row stride is shorter than the row");
    if (!rows_aligned(r->key_out_dev, ks, r->dtype) || !rows_aligned(r->value_out_dev, vs, r->dtype))
        return invalid("qwn_kv_load_tokens: rows must start on four values (pointers and strides)");
    cudaSetDevice(p->device);
    const RowMap m = {r->seq_ids_dev, r->row_begin_dev, r->first_pos_dev, r->num_seqs, r->num_rows};
    const bool tiles = r->row_begin_dev && rows_wide(r->key_out_dev, ks, r->dtype) &&
                       rows_wide(r->value_out_dev, vs, r->dtype);
    const uint64_t ctas = tiles ? unit_count(r->num_rows, r->num_seqs) : ((uint64_t)r->num_rows * p->kv_heads + 3) / 4;
    if (ctas > 0x7FFFFFFFull || (tiles && p->kv_heads > 65535u))
        return invalid("qwn_kv_load_tokens: too many rows for one call");
    const StoreGeo g = store_geo(p);
    cudaStream_t s = stream_of(p, r->stream);
    const cudaError_t e = with_codec(p->codec, r->dtype, [&](auto codec, auto *type) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int C = decltype(codec)::value;
        T *k = static_cast<T *>(r->key_out_dev), *v = static_cast<T *>(r->value_out_dev);
        // as many heads per CTA as leave every SM a few CTAs
        uint32_t heads = p->kv_heads;
        while (heads > 1 && ctas * ((p->kv_heads + heads - 1) / heads) < 16 * 148) heads = (heads + 1) / 2;
        const dim3 grid((unsigned)ctas, tiles ? (p->kv_heads + heads - 1) / heads : 1);
        if (tiles) return launch_next(load_tiles_kernel<C, T>, grid, kTileThreads, s, g, m, r->layer, heads, ks, vs, k, v);
        return launch_next(load_rows_kernel<C, T>, grid, 128, s, g, m, r->layer, ks, vs, k, v);
    });
    if (e != cudaSuccess) { set_cuda_error("qwn_kv_load_tokens", e); return QWN_CUDA_STATUS_RUNTIME_ERROR; }
    return QWN_CUDA_STATUS_OK;
}
