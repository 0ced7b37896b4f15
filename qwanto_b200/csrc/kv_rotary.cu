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

// the position in the cache of row r and its sequence; false (and the status
// latched) when the row belongs to none or lies outside its sequence
__device__ __forceinline__ bool find_row(const StoreGeo &g, const RowMap &m, uint32_t row, int32_t &seq, int32_t &pos,
                                         bool tell) {
    uint32_t i = row;
    int32_t b = (int32_t)row, e = b + 1;
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
        if ((int32_t)row < b || (int32_t)row >= e) {
            if (tell) latch(g.status, QWN_KV_STATUS_BAD_LENGTH);
            return false;
        }
    }
    seq = m.seq_ids ? m.seq_ids[i] : (int32_t)i;
    if (seq < 0 || (uint32_t)seq >= g.max_seqs) {
        if (tell) latch(g.status, QWN_KV_STATUS_BAD_SEQUENCE);
        return false;
    }
    const int32_t len = g.seq_lens[seq];
    const int64_t p = (m.first_pos ? (int64_t)m.first_pos[i] : (int64_t)len - ((int64_t)e - b)) + ((int64_t)row - b);
    if (p < 0 || p >= len) {
        if (tell) latch(g.status, QWN_KV_STATUS_BAD_LENGTH);
        return false;
    }
    pos = (int32_t)p;
    return true;
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

struct RotaryArgs {
    RowMap rows;
    const int32_t *rotary_pos;
    const float *table;
    uint32_t layer, query_heads, rot, max_position, query_out_dtype;
    bool neighbours;
    uint64_t query_stride, key_stride, value_stride;
};

__device__ __forceinline__ void store_any(void *out, uint32_t dtype, size_t at, float4 v) {
    if (dtype == QWN_DTYPE_F32) store4(static_cast<float *>(out) + at, v);
    else if (dtype == QWN_DTYPE_F16) store4(static_cast<__half *>(out) + at, v);
    else store4(static_cast<__nv_bfloat16 *>(out) + at, v);
}

// one warp per (row, head): the kv heads (K and V together), then the query heads
template <int CODEC, typename T>
__global__ void __launch_bounds__(128) append_rotary_kernel(StoreGeo g, RotaryArgs a, const T *query, const T *key,
                                                            const T *value, void *query_out) {
    const uint64_t wg = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const uint32_t slots = g.kv_heads + a.query_heads;
    const uint32_t row = (uint32_t)(wg / slots), slot = (uint32_t)(wg % slots);
    if (row >= a.rows.num_rows) return;
    int32_t seq, pos = 0;
    bool ok = find_row(g, a.rows, row, seq, pos, lane == 0 && slot == 0);
    const int32_t angle = ok && a.rotary_pos ? a.rotary_pos[row] : pos;
    if (ok && a.rot && (angle < 0 || (uint32_t)angle >= a.max_position)) {
        if (lane == 0 && slot == 0) latch(g.status, QWN_KV_STATUS_BAD_LENGTH);
        ok = false;
    }
    Turn t;
    if (ok && a.rot) t = load_turn(a.table + (size_t)angle * a.rot, (int)a.rot, a.neighbours, lane);
    if (slot < g.kv_heads) {
        if (!ok) return;
        uint8_t *tile = tile_for(g, seq, a.layer, slot, pos);
        if (!tile) return;
        float4 k = load4(key + (size_t)row * a.key_stride + slot * kHeadDim + 4 * lane);
        const float4 v = load4(value + (size_t)row * a.value_stride + slot * kHeadDim + 4 * lane);
        if (a.rot) k = rotate(k, t, a.neighbours);
        store_token<CODEC>(tile, pos & 15, k, v, lane);
    } else {
        const uint32_t h = slot - g.kv_heads;
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
        if (ok) {
            q = load4(query + (size_t)row * a.query_stride + h * kHeadDim + 4 * lane);
            if (a.rot) q = rotate(q, t, a.neighbours);
        }
        store_any(query_out, a.query_out_dtype, ((size_t)row * a.query_heads + h) * kHeadDim + 4 * lane, q);
    }
}

// one warp per (row, head): K and V of a cached token back to rows
template <int CODEC, typename T>
__global__ void __launch_bounds__(128) load_tokens_kernel(StoreGeo g, RowMap m, uint32_t layer, uint64_t key_stride,
                                                          uint64_t value_stride, T *key, T *value) {
    const uint64_t wg = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const uint32_t row = (uint32_t)(wg / g.kv_heads), h = (uint32_t)(wg % g.kv_heads);
    if (row >= m.num_rows) return;
    int32_t seq, pos;
    const uint8_t *tile = nullptr;
    if (find_row(g, m, row, seq, pos, lane == 0 && h == 0)) tile = tile_for(g, seq, layer, h, pos);
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    if (key)
        store4(key + (size_t)row * key_stride + h * kHeadDim + 4 * lane,
               tile ? load_token<CODEC>(tile, pos & 15, 0, lane) : zero);
    if (value)
        store4(value + (size_t)row * value_stride + h * kHeadDim + 4 * lane,
               tile ? load_token<CODEC>(tile, pos & 15, 1, lane) : zero);
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

// four values of a row are one access: rows start on four values
bool rows_aligned(const void *p, uint64_t stride, uint32_t dtype) {
    return (uintptr_t)p % (dtype == QWN_DTYPE_F32 ? 16 : 8) == 0 && stride % 4 == 0;
}
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
    const uint64_t ctas = ((uint64_t)r->num_rows * (p->kv_heads + r->query_heads) + 3) / 4;
    if (ctas > 0x7FFFFFFFull) return invalid("qwn_kv_append_rotary: too many rows for one call");
    const StoreGeo g = store_geo(p);
    cudaStream_t s = stream_of(p, r->stream);
    const cudaError_t e = with_codec(p->codec, r->dtype, [&](auto codec, auto *type) {
        using T = std::remove_pointer_t<decltype(type)>;
        append_rotary_kernel<decltype(codec)::value, T><<<(unsigned)ctas, 128, 0, s>>>(
            g, a, static_cast<const T *>(r->query_dev), static_cast<const T *>(r->key_dev),
            static_cast<const T *>(r->value_dev), r->query_out_dev);
        count_launch();
        return cudaGetLastError();
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
    const uint64_t ctas = ((uint64_t)r->num_rows * p->kv_heads + 3) / 4;
    if (ctas > 0x7FFFFFFFull) return invalid("qwn_kv_load_tokens: too many rows for one call");
    const StoreGeo g = store_geo(p);
    cudaStream_t s = stream_of(p, r->stream);
    const cudaError_t e = with_codec(p->codec, r->dtype, [&](auto codec, auto *type) {
        using T = std::remove_pointer_t<decltype(type)>;
        load_tokens_kernel<decltype(codec)::value, T><<<(unsigned)ctas, 128, 0, s>>>(
            g, m, r->layer, ks, vs, static_cast<T *>(r->key_out_dev), static_cast<T *>(r->value_out_dev));
        count_launch();
        return cudaGetLastError();
    });
    if (e != cudaSuccess) { set_cuda_error("qwn_kv_load_tokens", e); return QWN_CUDA_STATUS_RUNTIME_ERROR; }
    return QWN_CUDA_STATUS_OK;
}
