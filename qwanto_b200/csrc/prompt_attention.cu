// Attention of packed prompts over their own rows (qwn_prompt_attention), by the
// tile kernel of prompt_tile.cuh.  16-bit keys and values go from the rows into
// operand tiles by TMA; fp32 ones are cut into three bf16 parts on the way.  37 rows
// of 12/2 heads: 10.3 us, which is latency; 4099 fp32 rows with a window of 1000: 200.
#include <algorithm>

#include "prompt_tile.cuh"

namespace qkv {
namespace {

// K or V heads of 16-bit rows, in tiles of 64 dims x 128 tokens
bool encode_rows(CUtensorMap *map, const void *p, bool bf16, uint64_t width, uint64_t rows, uint64_t stride) {
    const EncodeFn fn = encoder();
    if (!fn) return false;
    const cuuint64_t dims[2] = {width, rows}, strides[1] = {stride * 2};
    const cuuint32_t box[2] = {64, 128}, steps[2] = {1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(p), dims,
              strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// multiprocessors of a device
int device_sms(int device) {
    static std::mutex mu;
    static int sms[64];
    if (device < 0 || device >= 64) return 0;
    std::lock_guard<std::mutex> lk(mu);
    if (!sms[device] && cudaDeviceGetAttribute(&sms[device], cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
    return sms[device];
}

}  // namespace
}  // namespace qkv

using namespace qkv;

QWN_CUDA_ABI_API int qwn_prompt_attention(const QwnPromptAttentionRequest *r) {
    if (!r || !header_ok(r->header, sizeof(*r))) return invalid("qwn_prompt_attention: bad header");
    if (!dtype_ok(r->dtype) || r->num_rows > 0x7FFFFFFFu) return invalid("qwn_prompt_attention: dtype or num_rows out of range");
    if (r->kv_heads == 0 || r->query_heads == 0 || r->query_heads % r->kv_heads || r->query_heads > 65535u)
        return invalid("qwn_prompt_attention: query heads must be a multiple of the kv heads");
    if (r->num_seqs > 0x7FFFFFFFu || (!r->row_begin_dev && r->num_seqs > 1))
        return invalid("qwn_prompt_attention: without row_begin_dev there is one sequence");
    if (!(r->scale >= 0.f) || !(r->scale < INFINITY) || r->window > 0x7FFFFFFFu || (r->window && !r->causal))
        return invalid("qwn_prompt_attention: scale must be finite and not negative, and a window is causal");
    const uint64_t qw = (uint64_t)r->query_heads * kHeadDim, kw = (uint64_t)r->kv_heads * kHeadDim;
    const uint64_t qs = r->query_stride ? r->query_stride : qw, ks = r->key_stride ? r->key_stride : kw;
    const uint64_t vs = r->value_stride ? r->value_stride : kw, os = r->output_stride ? r->output_stride : qw;
    if (r->num_rows == 0) return QWN_CUDA_STATUS_OK;
    if (r->num_seqs == 0) return invalid("qwn_prompt_attention: rows without a sequence");
    if (!r->query_dev || !r->key_dev || !r->value_dev || !r->output_dev)
        return invalid("qwn_prompt_attention: query, key, value and output are needed");
    if (qs < qw || ks < kw || vs < kw || os < qw) return invalid("qwn_prompt_attention: a row stride is shorter than the row");
    if (!rows_wide(r->query_dev, qs, r->dtype) || !rows_wide(r->key_dev, ks, r->dtype) ||
        !rows_wide(r->value_dev, vs, r->dtype) || !rows_wide(r->output_dev, os, r->dtype))
        return invalid("qwn_prompt_attention: rows must start on 16 bytes (pointers and strides)");
    const uint64_t es = value_bytes(r->dtype);
    if ((ks | vs) * es >= 1ull << 40) return invalid("qwn_prompt_attention: a row stride is too long");
    const RowSpan out = {(uintptr_t)r->output_dev, os * es, qw * es, r->num_rows};
    auto met = [&](const void *p, uint64_t stride, uint64_t width) {
        return rows_meet({(uintptr_t)p, stride * es, width * es, r->num_rows}, out);
    };
    if (met(r->query_dev, qs, qw) || met(r->key_dev, ks, kw) || met(r->value_dev, vs, kw))
        return invalid("qwn_prompt_attention: output overlaps rows that are still read");
    DeviceScope scope(r->device_id);
    if (!scope.ok) return scope.fail("qwn_prompt_attention");
    const int sms = device_sms(r->device_id);
    if (sms <= 0) return scope.fail("qwn_prompt_attention");
    AtArgs a{};
    a.rows = {nullptr, r->row_begin_dev, nullptr, r->num_seqs, r->num_rows};
    a.group = r->query_heads / r->kv_heads;
    a.kv_heads = r->kv_heads;
    a.query_heads = r->query_heads;
    a.window = r->window;
    a.causal = r->causal ? 1 : 0;
    a.dtype = r->dtype;
    set_scale(a, r->scale);
    a.query_stride = qs, a.key_stride = ks, a.value_stride = vs, a.out_stride = os;
    a.query = r->query_dev, a.key = r->key_dev, a.value = r->value_dev, a.out = r->output_dev;
    a.status = r->status_dev;
    const uint64_t rows = (uint64_t)r->num_rows * a.group;
    if (rows > 0xFFFFFFFFull) return invalid("qwn_prompt_attention: too many rows for one call");
    // units of 256 rows for 16-bit types, of 128 where that leaves SMs without any
    auto units = [&](uint64_t tile) { return r->row_begin_dev ? rows / tile + r->num_seqs : (rows + tile - 1) / tile; };
    const bool two = r->dtype != QWN_DTYPE_F32 && units(256) * r->kv_heads > (uint64_t)sms;
    const uint64_t ctas = units(two ? 256 : 128) * r->kv_heads;
    if (ctas > 0x7FFFFFFFull) return invalid("qwn_prompt_attention: too many rows for one call");
    a.units = (uint32_t)units(two ? 256 : 128);
    CUtensorMap kmap{}, vmap{};
    if (r->dtype != QWN_DTYPE_F32 &&
        (!encode_rows(&kmap, r->key_dev, r->dtype == QWN_DTYPE_BF16, kw, r->num_rows, ks) ||
         !encode_rows(&vmap, r->value_dev, r->dtype == QWN_DTYPE_BF16, kw, r->num_rows, vs))) {
        set_error("qwn_prompt_attention: the driver takes no tensor map of these rows");
        return QWN_CUDA_STATUS_UNSUPPORTED;
    }
    cudaStream_t s = static_cast<cudaStream_t>(r->stream);
    const int d = r->device_id;
    const uint32_t n = (uint32_t)std::min<uint64_t>(ctas, (uint64_t)sms);
    cudaError_t e;
    if (r->dtype == QWN_DTYPE_F32) e = launch_tile_kernel<0, 3, 1, true>(d, n, s, kmap, vmap, a);
    else if (r->dtype == QWN_DTYPE_BF16)
        e = two ? launch_tile_kernel<0, 1, 2, true>(d, n, s, kmap, vmap, a) : launch_tile_kernel<0, 1, 1, true>(d, n, s, kmap, vmap, a);
    else e = two ? launch_tile_kernel<0, 1, 2, false>(d, n, s, kmap, vmap, a) : launch_tile_kernel<0, 1, 1, false>(d, n, s, kmap, vmap, a);
    if (e != cudaSuccess) { set_cuda_error("qwn_prompt_attention", e); return QWN_CUDA_STATUS_RUNTIME_ERROR; }
    return QWN_CUDA_STATUS_OK;
}
