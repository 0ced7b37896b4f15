// Attention of a chunk of new tokens over the paged cache (qwn_kv_chunk_attention).
//
// The reference attends token by token (c/qwn_paged_kv.c:225-382,
// c/qwanto_turboquant.c:648-705, :707-768); a prompt's chunk, a batch of drafted
// tokens or a decode step in 16-bit rows goes through the tile kernel of
// prompt_tile.cuh here.  Where there are too few row tiles to fill the GPU, the
// tokens are cut into one run per SM and join_kernel puts the pieces of a row
// together:
//     M = max M_i,   out = sum_i 2^(M_i - M) o_i / sum_i 2^(M_i - M) l_i
// 33 fp16 rows of 48/8 heads over 131105 int8 tokens (8 tiles, 148 SMs): 225 us, of
// which the operations take 64; a single row of 12/2 heads over 2048 tokens: 26 us,
// all of it latency.
#include <algorithm>

#include "prompt_tile.cuh"

namespace qkv {
namespace {

// Four warps per row and query head share its pieces; four dims per lane.
template <int SRC, int PARTS, int TILES>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ AtArgs a, uint32_t grid) {
    using W = AtWork<SRC, PARTS, TILES>;
    using S = AtShape<SRC, PARTS, TILES>;
    constexpr uint32_t kRows = W::kRows;
    __shared__ float best[4], sums[4];
    __shared__ float4 rows[4][32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t row = blockIdx.x / a.query_heads, qh = blockIdx.x - row * a.query_heads;
    launch_dependents();
    wait_previous();
    if (row >= a.rows.num_rows) return;
    uint32_t i = row;
    if (a.rows.row_begin) {
        uint32_t lo = 0, hi = a.rows.num_seqs;  // the last sequence that begins at the row or before
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (a.rows.row_begin[mid] <= (int32_t)row) lo = mid;
            else hi = mid;
        }
        i = lo;
    }
    const AtSequence s = at_sequence(a, true, i);
    if ((int64_t)row < s.begin || (int64_t)row >= s.begin + s.rows) return;  // of no sequence
    int32_t first;
    const uint32_t span = at_span(a, s, AtShape<SRC, PARTS, TILES>::kBlock, first);
    const uint32_t total = a.prefix[a.rows.num_seqs];
    const AtRuns runs(total, at_runs<TILES>(total, grid));
    const uint32_t kv = qh / a.group, r = (row - (uint32_t)s.begin) * a.group + qh - kv * a.group;
    const uint32_t tile = r / kRows, item = tile * a.kv_heads + kv, u0 = a.prefix[i] + item * span;
    const uint32_t b0 = runs.owner(u0), b1 = runs.owner(u0 + span - 1);
    const bool quarters = S::kQuarters && (uint64_t)s.rows * a.group - tile * kRows <= 32;
    if (b0 == b1 && !quarters) return;  // finished by its CTA
    const uint32_t at = r % kRows;
    const uint32_t parts = (b1 - b0 + 1) << (quarters ? 2 : 0), step = a.slot_rows / 4;
    const uint32_t first_slot = S::kQuarters ? a.prefix[a.rows.num_seqs + 1 + i] + item + b0 : 0;
    // sequences that overlap have pieces that were not written (the tile kernel tells)
    if (b1 < b0 || b1 >= grid || (uint64_t)first_slot + (S::kQuarters ? b1 - b0 : 2 * b1 + 1) >= a.slot_count) return;
    const bool second = u0 > runs.begin(b0);
    // the k-th piece of the row: a CTA's, or one quarter of a CTA's
    auto piece = [&](uint32_t k, uint32_t &place) {
        const uint32_t n = quarters ? k >> 2 : k;
        place = quarters ? (k & 3) * step + at : at;
        // (without quarters: a CTA's first segment, or its second slot)
        const uint32_t slot = S::kQuarters ? first_slot + n : 2 * (b0 + n) + (n == 0 && second ? 1 : 0);
        return a.slots + (size_t)slot * at_slot_floats(a.slot_rows);
    };
    float M = -INFINITY;
    for (uint32_t k = 4 * lane + warp; k < parts; k += 128) {
        uint32_t place;
        const float *p = piece(k, place);
        M = fmaxf(M, p[a.slot_rows * kHeadDim + place]);
    }
    M = warp_max(M);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (uint32_t k = warp; k < parts; k += 4) {
        uint32_t place;
        const float *p = piece(k, place);
        const float m = p[a.slot_rows * kHeadDim + place], sum = p[a.slot_rows * (kHeadDim + 1) + place];
        const float4 v = *reinterpret_cast<const float4 *>(p + (size_t)place * kHeadDim + 4 * lane);
        if (m == -INFINITY) continue;
        const float w = ex2(m - M);
        l = fmaf(w, sum, l);
        o.x = fmaf(w, v.x, o.x);
        o.y = fmaf(w, v.y, o.y);
        o.z = fmaf(w, v.z, o.z);
        o.w = fmaf(w, v.w, o.w);
    }
    if (lane == 0) best[warp] = M, sums[warp] = l;
    rows[warp][lane] = o;
    __syncthreads();
    if (warp) return;
    M = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (best[k] == -INFINITY) continue;
        const float w = ex2(best[k] - M);
        const float4 v = rows[k][lane];
        l = fmaf(w, sums[k], l);
        o.x = fmaf(w, v.x, o.x);
        o.y = fmaf(w, v.y, o.y);
        o.z = fmaf(w, v.z, o.z);
        o.w = fmaf(w, v.w, o.w);
    }
    const float per = l > 0.f || l != l ? 1.f / l : 0.f;
    if (per == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);
    const uint64_t to = (uint64_t)row * a.out_stride + qh * kHeadDim + 4 * lane;
    const float4 y = make_float4(o.x * per, o.y * per, o.z * per, o.w * per);
    if (a.dtype == QWN_DTYPE_F32) store4(static_cast<float *>(a.out) + to, y);
    else if (a.dtype == QWN_DTYPE_F16) store4(static_cast<__half *>(a.out) + to, y);
    else store4(static_cast<__nv_bfloat16 *>(a.out) + to, y);
}

// How a call is cut: two tiles of 128 rows per CTA or one, and into runs or not.
constexpr uint64_t kMaxWorkspace = 128ull << 20;  // for pieces of rows; beyond, there are tiles for every SM
struct ChunkPlan {
    uint32_t tiles, slot_rows, slot_count;
    uint64_t units, prefix_bytes, workspace;
    bool split;  // given a workspace
};
ChunkPlan plan_chunk(const Pool *p, uint32_t num_seqs, uint32_t num_rows, uint32_t query_heads, uint32_t dtype, bool runs) {
    ChunkPlan c{};
    const uint64_t group = query_heads / p->kv_heads, rows = (uint64_t)num_rows * group;
    c.tiles = dtype != QWN_DTYPE_F32 && rows > 128ull * num_seqs ? 2 : 1;
    const uint64_t tile = 128ull * c.tiles;
    c.units = runs ? rows / tile + num_seqs : num_seqs * ((group + tile - 1) / tile);
    c.prefix_bytes = 2 * ((uint64_t)num_seqs + 1) * 4 + 255 & ~255ull;
    const bool quarters = c.tiles == 1 && dtype != QWN_DTYPE_F32 && p->codec != QWN_KV_CODEC_F16;
    // one row per sequence is a kv head's group, in each quarter
    c.slot_rows = quarters && !runs ? 4 * (uint32_t)group : 128 * c.tiles;
    const uint64_t items = c.units * p->kv_heads, slots = quarters ? items + p->sms : 2ull * p->sms;
    const uint64_t bytes = slots * at_slot_floats(c.slot_rows) * sizeof(float);
    // blocks are counted in 32 bits
    const uint64_t most = (uint64_t)p->max_pages_per_seq * p->page_tokens / 64 + 2;
    c.slot_count = (uint32_t)std::min<uint64_t>(slots, 0x7FFFFFFFu);
    c.split = (quarters ? bytes <= kMaxWorkspace : items < 8ull * p->sms) && items * most < 1ull << 31;
    c.workspace = c.split ? c.prefix_bytes + bytes : 0;
    return c;
}

// What no plan of these sizes or smaller ones goes beyond: a plan's own need is not monotone, as the largest calls
// have tiles enough and go without runs.
uint64_t most_workspace(const Pool *p, uint32_t num_seqs, uint32_t num_rows, uint32_t query_heads) {
    const uint64_t group = query_heads / p->kv_heads, rows = (uint64_t)num_rows * group, seqs = num_seqs, sms = p->sms;
    // with quarters: a slot per tile and per SM, of one tile or of a group in each quarter
    const uint64_t runs = (std::min(rows, 128 * seqs) / 128 + seqs) * p->kv_heads + sms;
    const uint64_t ones = seqs * p->kv_heads + sms, one = 4 * std::min<uint64_t>(group, 128);
    const uint64_t with = std::max(runs * at_slot_floats(128), ones * at_slot_floats((uint32_t)one)) * sizeof(float);
    const uint64_t without = 2 * sms * at_slot_floats(rows > 128 ? 256 : 128) * sizeof(float);
    return (2 * (seqs + 1) * 4 + 255) / 256 * 256 + std::max(std::min(with, kMaxWorkspace), without);
}

template <int SRC>
cudaError_t launch_chunk(const Pool *p, const ChunkPlan &c, AtArgs &a, cudaStream_t s) {
    const uint32_t ctas = a.slots ? (uint32_t)p->sms : (uint32_t)std::min<uint64_t>(c.units * p->kv_heads, (uint64_t)p->sms);
    const CUtensorMap none{};
    auto run = [&](auto parts, auto tiles) {
        constexpr int P = decltype(parts)::value, T = decltype(tiles)::value;
        cudaError_t e = launch_tile_kernel<SRC, P, T, P == 3>(p->device, ctas, s, none, none, a);
        if (e != cudaSuccess || !a.slots) return e;
        return launch_next(join_kernel<SRC, P, T>, dim3(a.rows.num_rows * a.query_heads), 128, s, a, ctas);
    };
    using One = std::integral_constant<int, 1>;
    if (a.dtype == QWN_DTYPE_F32) return run(std::integral_constant<int, 3>(), One());
    return c.tiles == 2 ? run(One(), std::integral_constant<int, 2>()) : run(One(), One());
}

}  // namespace
}  // namespace qkv

using namespace qkv;

QWN_CUDA_ABI_API int qwn_kv_chunk_workspace(const QwnKvPoolHandle *h, uint32_t num_seqs, uint32_t num_rows,
                                            uint32_t query_heads, uint64_t *bytes) {
    const Pool *p = pool_from(h);
    if (!p || !bytes) return invalid("qwn_kv_chunk_workspace: bad handle");
    if (query_heads == 0 || query_heads % p->kv_heads || query_heads > p->max_query_heads || num_seqs > p->max_seqs ||
        num_rows > 0x7FFFFFFFu)
        return invalid("qwn_kv_chunk_workspace: heads, sequences or rows out of the pool's range");
    *bytes = num_seqs && num_rows ? most_workspace(p, num_seqs, num_rows, query_heads) : 0;
    return QWN_CUDA_STATUS_OK;
}

QWN_CUDA_ABI_API int qwn_kv_chunk_attention(QwnKvPoolHandle *h, const QwnKvChunkAttentionRequest *r) {
    Pool *p = pool_from(h);
    if (!p || !r || !header_ok(r->header, sizeof(*r))) return invalid("qwn_kv_chunk_attention: bad handle or header");
    if (r->layer >= p->layers || r->num_seqs > p->max_seqs || !dtype_ok(r->dtype))
        return invalid("qwn_kv_chunk_attention: layer, num_seqs or dtype out of range");
    if (r->num_rows > 0x7FFFFFFFu || (!r->row_begin_dev && r->num_rows != r->num_seqs))
        return invalid("qwn_kv_chunk_attention: without row_begin_dev there is one row per sequence");
    if (r->query_heads == 0 || r->query_heads % p->kv_heads || r->query_heads > p->max_query_heads)
        return invalid("qwn_kv_chunk_attention: query heads must be a multiple of the kv heads within the pool's limit");
    if (!(r->scale >= 0.f) || !(r->scale < INFINITY) || r->window > 0x7FFFFFFFu)
        return invalid("qwn_kv_chunk_attention: scale must be finite and not negative, window below 2^31");
    const uint64_t width = (uint64_t)r->query_heads * kHeadDim;
    const uint64_t qs = r->query_stride ? r->query_stride : width, os = r->output_stride ? r->output_stride : width;
    if (r->num_rows == 0) return QWN_CUDA_STATUS_OK;
    if (r->num_seqs == 0) return invalid("qwn_kv_chunk_attention: rows without a sequence");
    if (!r->query_dev || !r->output_dev) return invalid("qwn_kv_chunk_attention: query and output are needed");
    if (qs < width || os < width) return invalid("qwn_kv_chunk_attention: a row stride is shorter than the row");
    if (!rows_wide(r->query_dev, qs, r->dtype) || !rows_wide(r->output_dev, os, r->dtype))
        return invalid("qwn_kv_chunk_attention: rows must start on 16 bytes (pointers and strides)");
    const uint64_t es = value_bytes(r->dtype);
    if (rows_meet({(uintptr_t)r->query_dev, qs * es, width * es, r->num_rows},
                  {(uintptr_t)r->output_dev, os * es, width * es, r->num_rows}))
        return invalid("qwn_kv_chunk_attention: output overlaps query rows that are still read");
    const ChunkPlan c = plan_chunk(p, r->num_seqs, r->num_rows, r->query_heads, r->dtype, r->row_begin_dev != nullptr);
    if (r->workspace_dev && ((uintptr_t)r->workspace_dev % 16 || r->workspace_bytes < c.workspace))
        return invalid("qwn_kv_chunk_attention: workspace must be 16-byte aligned and as large as qwn_kv_chunk_workspace tells");
    if (c.units * p->kv_heads > 0x7FFFFFFFull || (uint64_t)r->num_rows * r->query_heads > 0x7FFFFFFFull ||
        (uint64_t)r->num_rows * (r->query_heads / p->kv_heads) > 0xFFFFFFFFull)
        return invalid("qwn_kv_chunk_attention: too many rows for one call");
    DeviceScope scope(p->device);
    if (!scope.ok) return scope.fail("qwn_kv_chunk_attention");
    AtArgs a{};
    a.rows = {r->seq_ids_dev, r->row_begin_dev, r->first_pos_dev, r->num_seqs, r->num_rows};
    a.group = r->query_heads / p->kv_heads;
    a.kv_heads = p->kv_heads;
    a.query_heads = r->query_heads;
    a.window = r->window;
    a.causal = 1;
    a.layer = r->layer;
    a.dtype = r->dtype;
    set_scale(a, r->scale);
    a.query_stride = qs;
    a.out_stride = os;
    a.query = r->query_dev;
    a.out = r->output_dev;
    a.geo = store_geo(p);
    a.status = p->status;
    a.units = (uint32_t)c.units;
    if (c.split && r->workspace_dev) {
        a.slot_rows = c.slot_rows;
        a.slot_count = c.slot_count;
        a.prefix = static_cast<uint32_t *>(r->workspace_dev);
        a.slots = reinterpret_cast<float *>(static_cast<uint8_t *>(r->workspace_dev) + c.prefix_bytes);
    }
    cudaStream_t s = stream_of(p, r->stream);
    cudaError_t e;
    switch (p->codec) {
        case QWN_KV_CODEC_Q8_B64_F32: e = launch_chunk<QWN_KV_CODEC_Q8_B64_F32>(p, c, a, s); break;
        case QWN_KV_CODEC_Q8_HEAD_F16: e = launch_chunk<QWN_KV_CODEC_Q8_HEAD_F16>(p, c, a, s); break;
        case QWN_KV_CODEC_TQ35_G64: e = launch_chunk<QWN_KV_CODEC_TQ35_G64>(p, c, a, s); break;
        case QWN_KV_CODEC_Q4_G32: e = launch_chunk<QWN_KV_CODEC_Q4_G32>(p, c, a, s); break;
        case QWN_KV_CODEC_F16: e = launch_chunk<QWN_KV_CODEC_F16>(p, c, a, s); break;
        default: e = cudaErrorNotSupported;
    }
    if (e != cudaSuccess) { set_cuda_error("qwn_kv_chunk_attention", e); return QWN_CUDA_STATUS_RUNTIME_ERROR; }
    return QWN_CUDA_STATUS_OK;
}
