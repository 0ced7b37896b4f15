// int8 products with a scale per token and per output (qwn_matmul_q8_*):
//     out[m][n] = (sum_k X[m][k] W[n][k]) * sx[m] * sw[n] + b[n]
// The sum is exact in int32; the scales and the bias are applied in fp32 and
// the result is rounded once.  The reference's only device product takes
// host activations and 2-bit weights (c/cuda/qwn_hypervsq2_cuda_abi.cu); this
// one keeps both sides on the device.
//
// Both kernels give the tensor core the weights as its A operand (128 outputs
// per CTA on TMEM's lanes) and the tokens as B (the columns), so that a few
// tokens cost a narrow MMA and a warp's lanes write consecutive outputs.
// Operand tiles are 128 codes deep, loaded by TMA with 128-byte swizzle.
// The handle keeps the weights as [in/128][out][128], zero past in_features:
// a tile is 16 KB in a row of HBM (with the caller's row order its 128-byte
// pieces are in_features apart, and a large weight streamed at 4.7 TB/s
// instead of 6.6), and a product never branches on in_features' remainder;
// TMA fills what lies outside the codes with zeros.
//
// Both kernels start while the stream's previous kernel still runs
// (programmatic launch), fetch weights, and wait for it before they read codes
// or scales or write anything.
//
// Tensor memory is taken so that no allocation waits for a CTA that waits for
// it.  A kernel lets the next one start only when all its CTAs hold theirs; at
// most four CTAs of the split kernel fit an SM, by their shared memory, with a
// quarter of its columns each; a CTA of the pair kernel, which takes all
// columns, shares an SM with no other CTA of either kernel.
#include <algorithm>
#include <cstring>
#include <mutex>
#include <new>
#include <type_traits>
#include <utility>

#include "kv_internal.cuh"
#include "rows.cuh"
#include "tcgen05.cuh"

namespace qkv {
namespace {

constexpr uint32_t kMmK = 128;       // codes per operand tile row: one swizzled row
constexpr uint32_t kMmRows = 128;    // outputs per CTA: the lanes of its accumulator
constexpr uint32_t kWBytes = kMmRows * kMmK;
constexpr uint32_t kMaxStages = 12;
constexpr uint32_t kOutWarps = 8;    // read TMEM and write: two for each quarter of its lanes
constexpr uint32_t kMmThreads = 64 + 32 * kOutWarps; // TMA warp, MMA warp, those
constexpr uint32_t kMaxSplit = 8;    // CTAs of a cluster that share an output tile
constexpr uint32_t kColumns = 512;   // of an SM's tensor memory
constexpr uint32_t kSplitColumns = 128, kSplitTokens = 128;
// shared memory: of an SM, what a CTA takes beside its own, dynamic at most (beside the static part) and at least
constexpr uint32_t kSmSmem = 228 * 1024, kCtaSmem = 1024, kMmSmem = 227 * 1024 - 4096;
constexpr uint32_t kSplitSmem = 46 * 1024, kPairSmem = 182 * 1024;
static_assert(kSplitTokens <= kSplitColumns, "a column per token");
static_assert((kColumns / kSplitColumns + 1) * (kSplitSmem + kCtaSmem) > kSmSmem, "an SM has columns for all its split CTAs");
static_assert(kPairSmem + kSplitSmem + 2 * kCtaSmem > kSmSmem && kPairSmem <= kMmSmem, "a pair's CTA is alone");

struct MatmulQ8 {
    int device = 0, sms = 148;
    uint32_t n = 0, k = 0, kblocks = 0;
    int8_t *w = nullptr;
    float *scales = nullptr, *bias = nullptr;
    uint32_t *status = nullptr;
    uint32_t clusters[kMaxSplit + 1] = {};  // clusters of each size that run at once, one CTA per SM
    CUtensorMap wmap;
};

MatmulQ8 *matmul_from(const QwnMatmulQ8Handle *h) {
    if (!h || !header_ok(h->header, sizeof(*h)) || !h->opaque) return nullptr;
    return static_cast<MatmulQ8 *>(h->opaque);
}

void matmul_release(MatmulQ8 *m) {
    cudaFree(m->w);
    delete m;
}

// weight [n][k] (rows `stride` apart) into [k / 128][n][128], zeros outside; a thread moves 16 codes
__global__ void __launch_bounds__(256) pack_weight_kernel(const int8_t *w, uint64_t stride, uint32_t n, uint32_t k,
                                                          uint64_t chunks, int8_t *out) {
    const uint64_t step = (uint64_t)gridDim.x * blockDim.x;
    const bool wide = ((uintptr_t)w | stride) % 16 == 0;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < chunks; i += step) {
        const uint64_t row = i >> 3;
        const uint32_t col = (uint32_t)(row / n) * kMmK + (uint32_t)(i & 7) * 16;
        const int8_t *p = w + (row % n) * stride + col;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (wide && col + 16 <= k) {
            v = *reinterpret_cast<const uint4 *>(p);
        } else {
            uint32_t q[4] = {};
            for (uint32_t j = 0; j < 16 && col + j < k; j++) q[j >> 2] |= (uint32_t)(uint8_t)p[j] << (8 * (j & 3));
            v = make_uint4(q[0], q[1], q[2], q[3]);
        }
        reinterpret_cast<uint4 *>(out)[i] = v;
    }
}

struct MmArgs {
    const float *sx, *sw, *bias;
    void *out;
    uint64_t out_stride;
    uint32_t m, n, kblocks;
    uint32_t *status;
};

template <typename T>
__device__ __forceinline__ void store_out(T *p, float v) {
    if constexpr (std::is_same_v<T, float>) *p = v;
    else if constexpr (std::is_same_v<T, __half>) *p = __float2half_rn(v);
    else *p = __float2bfloat16_rn(v);
}
// one rounding for the sum (beyond 2^24) and one for each factor, in fp32; then the output's
__device__ __forceinline__ float scaled(int sum, float sx, float sw, float bias) {
    return fmaf((float)sum * sx, sw, bias);
}

// ---------------------------------------------------------------------------
// Few tokens: bound by the weights' bytes.  One CTA per 128 outputs, tile of
// `nt` tokens and share of k; the cluster's CTAs take a share of k each, so
// that a few hundred outputs already load from every SM.  Their int32 sums
// meet in shared memory: CTA r receives the others' sums of its share of the
// tokens, adds them (exact in any order) and writes them.
// ---------------------------------------------------------------------------
// bytes that CTA r receives: [splits][its tokens][128 outputs]
__host__ __device__ constexpr uint32_t share_tokens(uint32_t nt, uint32_t splits) { return (nt + splits - 1) / splits; }
__host__ __device__ constexpr uint32_t share_bytes(uint32_t nt, uint32_t splits) {
    return splits > 1 ? splits * share_tokens(nt, splits) * kMmRows * 4 : 0;
}

template <typename T>
__global__ void __launch_bounds__(kMmThreads, 1) matmul_q8_split_kernel(const __grid_constant__ CUtensorMap wmap,
                                                                        const __grid_constant__ CUtensorMap xmap,
                                                                        MmArgs a, uint32_t nt, uint32_t splits,
                                                                        uint32_t stages) {
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], done;
    __shared__ uint32_t tmem_at;
    __shared__ float sx[256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    const uint32_t rank = splits > 1 ? cluster_rank() : 0;
    const uint32_t n0 = blockIdx.x / splits * kMmRows, m0 = blockIdx.y * nt;
    const uint32_t kb0 = (uint32_t)((uint64_t)a.kblocks * rank / splits);
    const uint32_t kb1 = (uint32_t)((uint64_t)a.kblocks * (rank + 1) / splits);
    const uint32_t stage_bytes = 2 * (kWBytes + nt * kMmK), count = kb1 - kb0;
    const uint32_t valid = min(nt, a.m - m0);  // tokens of this tile that exist
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < stages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(&done, 1);
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc<1>(&tmem_at, kSplitColumns);
    tc_fence_before();
    __syncthreads();
    launch_dependents();  // not before: what starts may want tensor memory too
    if (splits > 1) cluster_arrive();  // this CTA runs: the others may write to it from their wait on
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    bool ok = true;
    // a stage is two tiles of 128 codes, the last one perhaps one: a barrier's round trip per eight MMAs
    // (1 x 4096 x 6144: 6.4 us with one tile per stage, 5.5 with two)
    const uint32_t steps = (count + 1) / 2, tile_bytes = kWBytes + nt * kMmK;
    if (warp == 0) {
        const bool one = elect_one();
        const uint32_t ahead = min(steps, stages);
        auto load_w = [&](uint32_t i, uint32_t st) {
            const uint32_t two = min(count - 2 * i, 2u);
            mbar_expect_tx(&full[st], two * tile_bytes);
            for (uint32_t e = 0; e < two; e++)
                tma_load(base + st * stage_bytes + e * tile_bytes, &wmap, 0, (int)((kb0 + 2 * i + e) * a.n + n0),
                         smem_u32(&full[st]));
        };
        auto load_x = [&](uint32_t i, uint32_t st) {
            const uint32_t two = min(count - 2 * i, 2u);
            for (uint32_t e = 0; e < two; e++)
                tma_load(base + st * stage_bytes + e * tile_bytes + kWBytes, &xmap, (int)((kb0 + 2 * i + e) * kMmK), (int)m0,
                         smem_u32(&full[st]));
        };
        for (uint32_t i = 0; i < ahead; i++)
            if (one) load_w(i, i);
        wait_previous();
        for (uint32_t i = 0; i < ahead; i++)
            if (one) load_x(i, i);
        Ring r;
        uint32_t i = ahead;
        for (; i < steps; i++) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[r.stage], r.parity));
            if (!ok) break;
            if (one) {
                load_w(i, r.stage);
                load_x(i, r.stage);
            }
            r.next(stages);
        }
        // the copies in flight land before the memory goes, whichever warp gave up
        if (one)
            for (uint32_t j = i - min(i, stages); j < i; j++) ok &= mbar_wait_bounded(&full[j % stages], (j / stages) & 1);
    } else if (warp == 1) {
        const bool one = elect_one();
        const uint32_t desc = i8_desc(kMmRows, nt);
        const uint64_t first = smem_desc(base);
        Ring r;
        wait_previous();  // the tokens come after it: its time does not count as waiting for them
        for (uint32_t i = 0; i < steps; i++) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[r.stage], r.parity));
            if (!ok) break;
            tc_fence_after();
            const uint64_t wd = first + ((r.stage * stage_bytes) >> 4);
            if (one) {
                mma_tile<1>(tmem, wd, wd + (kWBytes >> 4), desc, i > 0);
                if (2 * i + 1 < count)
                    mma_tile<1>(tmem, wd + (tile_bytes >> 4), wd + ((tile_bytes + kWBytes) >> 4), desc, true);
                mma_commit(&empty[r.stage]);
            }
            r.next(stages);
        }
        if (one) mma_commit(&done);
        __syncwarp();
        ok &= mbar_wait_bounded(&done, 0);  // no product in flight when the memory goes
    }
    const uint32_t quarter = warp & 3, feature = quarter * 32 + lane;  // TMEM lanes this warp may read
    const uint32_t lanes = tmem + (quarter << 21);
    const uint32_t second = warp >= 2 ? (uint32_t)(warp - 2) >> 2 : 0;  // every other 16 tokens
    const uint32_t n = n0 + feature;
    const bool in = n < a.n;
    float sw = 0.f, bias = 0.f;
    T *out = static_cast<T *>(a.out) + (uint64_t)m0 * a.out_stride + n;
    if (warp >= 2) {
        if (in) sw = a.sw[n];
        if (in && a.bias) bias = a.bias[n];
        wait_previous();
        for (uint32_t c = threadIdx.x - 64; c < valid; c += 32 * kOutWarps) sx[c] = a.sx[m0 + c];
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kOutWarps) : "memory");
        ok = mbar_wait_bounded(&done, 0);
        tc_fence_after();
    }
    if (!ok) latch(a.status, QWN_KV_STATUS_WAIT_TIMEOUT);
    __syncwarp();
    if (splits == 1) {
        if (warp >= 2) {
            for (uint32_t c0 = 16 * second; c0 < valid; c0 += 32) {
                uint32_t v[16];
                tmem_load16(v, lanes + c0);
                T *to = out + c0 * a.out_stride;
#pragma unroll
                for (uint32_t i = 0; i < 16; i++) {
                    if (in && c0 + i < valid) store_out(to, scaled((int)v[i], sx[c0 + i], sw, bias));
                    to += a.out_stride;
                }
            }
        }
    } else {
        const uint32_t share = share_tokens(valid, splits);
        const uint32_t region = base + stages * stage_bytes;
        cluster_wait();
        if (warp >= 2) {
            // this CTA's sums of token c go to the CTA of c's share
            const uint32_t mine = region + (rank * share * kMmRows + feature) * 4;
            for (uint32_t c0 = 16 * second; c0 < valid; c0 += 32) {
                uint32_t v[16];
                tmem_load16(v, lanes + c0);
                uint32_t owner = c0 / share, at = c0 - owner * share, to = cluster_addr(mine, owner);
#pragma unroll
                for (uint32_t i = 0; i < 16; i++) {
                    if (c0 + i >= valid) break;
                    if (at == share) {
                        at = 0;
                        to = cluster_addr(mine, ++owner);
                    }
                    st_cluster(to + at++ * kMmRows * 4, v[i]);
                }
            }
        }
        cluster_sync();
        if (warp >= 2 && in) {
            const uint32_t first = rank * share, mine = first < valid ? min(share, valid - first) : 0;
            for (uint32_t c = second; c < mine; c += 2) {
                int sum = 0;
#pragma unroll
                for (uint32_t p = 0; p < kMaxSplit; p++)
                    if (p < splits) sum += ld_shared(region + ((p * share + c) * kMmRows + feature) * 4);
                store_out(out + (first + c) * a.out_stride, scaled(sum, sx[first + c], sw, bias));
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free<1>(tmem, kSplitColumns);
    }
}

// ---------------------------------------------------------------------------
// Many tokens: bound by the tensor core.  A pair of CTAs on two SMs shares
// 256 outputs x `nt` tokens: each CTA brings its 128 weight rows and half of
// the tokens, one tcgen05.mma of both SMs multiplies them, and each CTA's TMEM
// receives its 128 outputs.  Pairs stay resident and walk over the tiles; two
// accumulators let the TMEM warps write one tile while the next is multiplied.
// ---------------------------------------------------------------------------
constexpr uint32_t kPairStages = 6;
constexpr uint32_t kPairTokens = 256;

// Tile t of a walk in groups of 16 token tiles, the outputs outside them: the
// pairs that run together share 16 tiles of tokens and a few of weights
// (8192 x 6144 x 8192: 246 us, 253 with all 32 token tiles in one group).
struct PairTile {
    uint32_t n, m;
};
__device__ __forceinline__ PairTile pair_tile(uint32_t t, uint32_t m_tiles, uint32_t n_tiles) {
    constexpr uint32_t kGroup = 16;
    const uint32_t group = t / (kGroup * n_tiles), in = t - group * kGroup * n_tiles;
    const uint32_t wide = min(kGroup, m_tiles - group * kGroup);
    return {in / wide, group * kGroup + in % wide};
}

template <typename T>
__global__ void __launch_bounds__(kMmThreads, 1) matmul_q8_pair_kernel(const __grid_constant__ CUtensorMap wmap,
                                                                       const __grid_constant__ CUtensorMap xmap,
                                                                       MmArgs a, uint32_t nt, uint32_t m_tiles,
                                                                       uint32_t tiles) {
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_at;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    const uint32_t rank = cluster_rank(), pairs = gridDim.x >> 1, n_tiles = tiles / m_tiles;
    const uint32_t half = nt / 2, stage_bytes = kWBytes + half * kMmK;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kPairStages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 2 * kOutWarps);  // of both CTAs
        }
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc<2>(&tmem_at, kColumns);
    tc_fence_before();
    __syncthreads();
    launch_dependents();
    cluster_sync();  // both CTAs' barriers exist
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    bool ok = true;
    if (warp == 0) {
        const bool one = elect_one();
        const uint32_t bars = cluster_addr(smem_u32(full), 0);  // the first CTA's barriers count both CTAs' bytes
        auto load_w = [&](uint32_t kb, uint32_t row, uint32_t st) {
            if (rank == 0) mbar_expect_tx(&full[st], 2 * stage_bytes);
            tma_load_pair(base + st * stage_bytes, &wmap, 0, (int)(kb * a.n + row), bars + 8 * st);
        };
        auto load_x = [&](uint32_t kb, uint32_t row, uint32_t st) {
            tma_load_pair(base + st * stage_bytes + kWBytes, &xmap, (int)(kb * kMmK), (int)row, bars + 8 * st);
        };
        const uint32_t ahead = min(a.kblocks, kPairStages);  // weights of the first tile
        uint32_t t = blockIdx.x >> 1, i = 0;
        const uint32_t first = (pair_tile(t, m_tiles, n_tiles).n * 2 + rank) * kMmRows;
        for (uint32_t j = 0; j < ahead; j++)
            if (one) load_w(j, first, j);
        wait_previous();
        Ring r;
        for (; t < tiles && ok; t += pairs) {
            const PairTile tile = pair_tile(t, m_tiles, n_tiles);
            const uint32_t n0 = (tile.n * 2 + rank) * kMmRows, m0 = tile.m * nt + rank * half;
            for (uint32_t kb = 0; kb < a.kblocks; kb++, i++) {
                if (i >= kPairStages) {
                    ok = __all_sync(0xffffffffu, mbar_wait_cluster(&empty[r.stage], r.parity ^ 1));
                    if (!ok) break;
                }
                if (one) {
                    if (i >= ahead) load_w(kb, n0, r.stage);
                    load_x(kb, m0, r.stage);
                }
                r.next(kPairStages);
            }
        }
        // the copies in flight land before the memory goes, whichever warp gave up; where it was this one,
        // the other CTA may be up to a ring of stages ahead (it fills them in order: the first half that
        // does not come is the last)
        if (one && rank == 0) {
            const uint32_t walk = (tiles - (blockIdx.x >> 1) + pairs - 1) / pairs * a.kblocks;
            const uint32_t ahead_of = ok ? i : min(i + kPairStages, walk);
            for (uint32_t j = i - min(i, kPairStages); j < ahead_of; j++) {
                if (j >= i) mbar_expect_tx(&full[j % kPairStages], stage_bytes);
                if (!mbar_wait_cluster(&full[j % kPairStages], (j / kPairStages) & 1)) {
                    ok = false;
                    break;
                }
            }
        }
    } else if (warp == 1 && rank == 0) {
        const bool one = elect_one();
        const uint32_t desc = i8_desc(2 * kMmRows, nt);
        const uint64_t first = smem_desc(base);
        Ring r;
        uint32_t n = 0;
        wait_previous();  // the tokens come after it: its time does not count as waiting for them
        for (uint32_t t = blockIdx.x >> 1; t < tiles && ok; t += pairs, n++) {
            const uint32_t buf = n & 1, d = tmem + buf * kPairTokens;
            if (n >= 2) {
                ok = __all_sync(0xffffffffu, mbar_wait_cluster(&acc_empty[buf], (n / 2 - 1) & 1));
                if (!ok) break;
            }
            tc_fence_after();
            for (uint32_t kb = 0; kb < a.kblocks; kb++) {
                ok = __all_sync(0xffffffffu, mbar_wait_cluster(&full[r.stage], r.parity));
                if (!ok) break;
                tc_fence_after();
                const uint64_t wd = first + ((r.stage * stage_bytes) >> 4);
                if (one) {
                    mma_tile<2>(d, wd, wd + (kWBytes >> 4), desc, kb > 0);
                    mma_commit_pair(&empty[r.stage]);
                }
                r.next(kPairStages);
            }
            if (one) mma_commit_pair(&acc_full[buf]);
        }
        __syncwarp();
        if (n > 0) ok &= mbar_wait_cluster(&acc_full[(n - 1) & 1], ((n - 1) / 2) & 1);  // none in flight when the memory goes
    } else if (warp >= 2) {
        const uint32_t quarter = warp & 3, second = (uint32_t)(warp - 2) >> 2;
        uint32_t n = 0;
        wait_previous();
        for (uint32_t t = blockIdx.x >> 1; t < tiles; t += pairs, n++) {
            const PairTile tile = pair_tile(t, m_tiles, n_tiles);
            const uint32_t buf = n & 1, m0 = tile.m * nt, valid = min(nt, a.m - m0);
            const uint32_t col = (tile.n * 2 + rank) * kMmRows + quarter * 32 + lane;
            const bool in = col < a.n;
            const float sw = in ? a.sw[col] : 0.f, bias = a.bias && in ? a.bias[col] : 0.f;
            constexpr uint32_t kChunks = kPairTokens / 64;  // this warp's: every other 32 tokens
            float sx[kChunks];
#pragma unroll
            for (uint32_t j = 0; j < kChunks; j++) {
                const uint32_t c = (2 * j + second) * 32 + lane;
                sx[j] = c < valid ? a.sx[m0 + c] : 0.f;
            }
            if (!mbar_wait_cluster(&acc_full[buf], (n / 2) & 1)) { ok = false; break; }
            tc_fence_after();
            T *out = static_cast<T *>(a.out) + (uint64_t)m0 * a.out_stride + col;
#pragma unroll
            for (uint32_t j = 0; j < kChunks; j++) {
                const uint32_t c0 = (2 * j + second) * 32;
                if (c0 < valid) {
                    uint32_t v[32];
                    tmem_load32(v, tmem + (quarter << 21) + buf * kPairTokens + c0);
                    T *to = out + c0 * a.out_stride;
#pragma unroll
                    for (uint32_t i = 0; i < 32; i++) {
                        const float s = __shfl_sync(0xffffffffu, sx[j], i);
                        if (in && c0 + i < valid) store_out(to, scaled((int)v[i], s, sw, bias));
                        to += a.out_stride;
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(cluster_addr(smem_u32(&acc_empty[buf]), 0));
        }
    }
    if (!ok) latch(a.status, QWN_KV_STATUS_WAIT_TIMEOUT);
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    cluster_sync();  // neither CTA's memory or barriers go while the other may still use them
    if (warp == 1) {
        tc_fence_after();
        tmem_free<2>(tmem, kColumns);
    }
}

// ---- host ---------------------------------------------------------------------

// codes [rows][width], `stride` bytes apart, in tiles of box x 128
bool encode_codes(CUtensorMap *map, const int8_t *p, uint64_t width, uint64_t rows, uint64_t stride, uint32_t box) {
    const EncodeFn fn = encoder();
    if (!fn) return false;
    const cuuint64_t dims[2] = {width, rows}, strides[1] = {stride};
    const cuuint32_t tile[2] = {kMmK, box}, steps[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(p), dims, strides, tile, steps,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// dynamic shared memory above 48 KB is opted into per kernel and device
template <typename K>
cudaError_t allow_all_smem(K kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMmSmem);
}
template <typename T>
cudaError_t allow_all_smem() {
    const cudaError_t e = allow_all_smem(matmul_q8_split_kernel<T>);
    return e == cudaSuccess ? allow_all_smem(matmul_q8_pair_kernel<T>) : e;
}

template <typename K, typename... Args>
cudaError_t launch_clusters(K kernel, dim3 grid, uint32_t cluster, size_t smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kMmThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    note_early_trigger();
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) count_launch();
    else cudaGetLastError();  // reported here, not by a later launch
    return e;
}

// how a product is cut up: tokens per tile, and for the split kernel the CTAs
// that share k
struct MmPlan {
    bool pair;
    uint32_t nt, splits;
};

// The cut with the lowest estimate of its microseconds.  What the estimates are
// made of, measured on B200:
//  - the weights come out of HBM at 6.5 KB per ns at best, and all SMs together
//    read 11 KB per ns out of L2: a tile's weights once per token tile, its
//    tokens once per 128 outputs;
//  - the split kernel spends 0.12 us on 128 codes of a CTA's share of k (four
//    narrow MMAs), 0.18 when the CTAs fill the GPU, starts and ends in 2.2 us,
//    writes a token in 20 ns, and joins a cluster's sums in 0.1 us and 25 ns per
//    token.  Shares only as long as all clusters run at once with the largest
//    shared memory that a CTA may ask for (74 of two CTAs, 45 of three, 33 of
//    four, 15 of eight): beyond, a share costs a whole CTA's time (48 clusters of
//    three took 1.5 times what 48 of two took).  With shorter rings more would
//    run (93 of three at 100 KB), which the plan does not weigh;
//  - a pair spends 0.13 us + 1.05 ns per token of its tile on 128 codes, at
//    least 10.5 ns per token on a tile (its output), and starts and ends in
//    2.6 us.
// A few tokens thus go to the split kernel with as many shares as run at once
// (1 x 1536 x 2048: 2.8 us in 4 shares, 4.3 in one; 32 x 4096 x 6144: 6.3 us
// in 2 shares, 7.3 in one), more to pairs with the widest tile that still
// reaches all of them (257 x 4099 x 4095: 10.7 us with 96 tokens a tile, 14.1
// with 256; 8192 x 6144 x 8192 before its walk in groups: 253 us with 256, 278
// with 192).
MmPlan plan_matmul(const MatmulQ8 &mm, uint32_t m) {
    MmPlan best{};
    float least = INFINITY;
    const uint32_t n_tiles = (mm.n + kMmRows - 1) / kMmRows, n_pairs = (n_tiles + 1) / 2, pairs = (uint32_t)mm.sms / 2;
    const float kb = (float)mm.kblocks, hbm = (float)mm.n * kb * (float)kMmK / 6.5e6f;
    auto l2 = [&](uint64_t ctas, uint32_t tokens) { return (float)ctas * kb * (float)((kMmRows + tokens) * kMmK) / 11e6f; };
    for (uint32_t nt = 32; nt <= kPairTokens; nt += 32) {
        const uint64_t tiles = (uint64_t)n_pairs * ((m + nt - 1) / nt), waves = (tiles + pairs - 1) / pairs;
        const float w = (float)nt, tile = std::max(kb * (0.13f + 0.00105f * w), 0.25f + 0.0105f * w);
        const float t = 2.6f + std::max({(float)waves * tile, l2(2 * tiles, nt / 2), hbm}) + 0.006f * w;
        if (t < least) {
            least = t;
            best = {true, nt, 1};
        }
    }
    if (m > 1024) return best;
    for (uint32_t m_tiles = (m + kSplitTokens - 1) / kSplitTokens; m_tiles <= 8 && (m_tiles - 1) * 16 < m; m_tiles++) {
        const uint32_t nt = ((m + m_tiles - 1) / m_tiles + 15) / 16 * 16, count = (m + nt - 1) / nt;
        const uint64_t tiles = (uint64_t)n_tiles * count;
        const float tokens = (float)std::min(m, nt);
        for (uint32_t splits = 1; splits <= kMaxSplit && splits <= mm.kblocks; splits++) {
            if (splits > 1 && tiles > mm.clusters[splits]) break;
            const uint64_t waves = splits > 1 ? 1 : (tiles + mm.sms - 1) / mm.sms;
            const float busy = (float)std::min<uint64_t>(tiles * splits, (uint64_t)mm.sms);
            float cta = (float)((mm.kblocks + splits - 1) / splits) * (0.12f + 0.0004f * (float)nt + 0.0004f * busy);
            if (waves > 1) cta += 1.f + 0.02f * tokens;
            const float out = splits > 1 ? 0.1f + 0.025f * tokens : 0.02f * tokens;
            const float t = 2.2f + std::max({(float)waves * cta, l2(tiles, nt), hbm}) + out;
            if (t < least) {
                least = t;
                best = {false, nt, splits};
            }
        }
    }
    return best;
}

template <typename T>
cudaError_t launch_matmul(const MatmulQ8 &mm, const MmArgs &a, const int8_t *x, uint64_t x_stride, cudaStream_t s) {
    const MmPlan p = plan_matmul(mm, a.m);
    const uint32_t m_tiles = (a.m + p.nt - 1) / p.nt, n_tiles = (a.n + kMmRows - 1) / kMmRows;
    CUtensorMap xmap;
    if (!encode_codes(&xmap, x, mm.k, a.m, x_stride, p.pair ? p.nt / 2 : p.nt)) return cudaErrorInvalidValue;
    if (p.pair) {
        const uint32_t tiles = (n_tiles + 1) / 2 * m_tiles, pairs = std::min(tiles, (uint32_t)mm.sms / 2);
        const uint32_t smem = std::max(kPairSmem, 1024 + kPairStages * (kWBytes + p.nt / 2 * kMmK));
        return launch_clusters(matmul_q8_pair_kernel<T>, dim3(2 * pairs), 2, smem, s, mm.wmap, xmap, a, p.nt, m_tiles, tiles);
    }
    const uint32_t stage = 2 * (kWBytes + p.nt * kMmK), extra = 1024 + share_bytes(p.nt, p.splits);
    const uint32_t stages = std::min({kMaxStages, (kMmSmem - extra) / stage, (mm.kblocks + 2 * p.splits - 1) / (2 * p.splits)});
    return launch_clusters(matmul_q8_split_kernel<T>, dim3(n_tiles * p.splits, m_tiles), p.splits,
                           std::max(kSplitSmem, extra + stages * stage), s, mm.wmap, xmap, a, p.nt, p.splits, stages);
}

// Prepares the kernels on a device (the current one), once, and tells how many
// clusters of each size it runs at once with one CTA per SM.
cudaError_t prepare_device(MatmulQ8 *mm) {
    struct Device {
        bool ready = false;
        int sms = 0;
        uint32_t clusters[kMaxSplit + 1] = {};
    };
    static std::mutex mu;
    static Device devices[64];
    if (mm->device < 0 || mm->device >= 64) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> lk(mu);
    Device &d = devices[mm->device];
    if (!d.ready) {
        cudaError_t e = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, mm->device);
        if (e == cudaSuccess) e = allow_all_smem<float>();
        if (e == cudaSuccess) e = allow_all_smem<__half>();
        if (e == cudaSuccess) e = allow_all_smem<__nv_bfloat16>();
        for (uint32_t c = 1; c <= kMaxSplit && e == cudaSuccess; c++) {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(c);
            cfg.blockDim = dim3(kMmThreads);
            cfg.dynamicSmemBytes = kMmSmem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = c;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int n = 0;
            e = cudaOccupancyMaxActiveClusters(&n, matmul_q8_split_kernel<float>, &cfg);
            d.clusters[c] = (uint32_t)n;
        }
        if (e != cudaSuccess) return e;
        d.ready = true;
    }
    mm->sms = d.sms;
    std::copy(d.clusters, d.clusters + kMaxSplit + 1, mm->clusters);
    return cudaSuccess;
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
    m->kblocks = (o->in_features + kMmK - 1) / kMmK;
    cudaStream_t s = static_cast<cudaStream_t>(o->stream);
    cudaError_t e = prepare_device(m);
    if (e != cudaSuccess) {
        set_cuda_error("qwn_matmul_q8_create", e);
        matmul_release(m);
        return QWN_CUDA_STATUS_RUNTIME_ERROR;
    }
    // one allocation: the weights, then scales, bias and the status word
    const size_t wb = (size_t)m->kblocks * m->n * kMmK, fb = (size_t)m->n * sizeof(float);
    if (cudaMalloc(&m->w, wb + 2 * fb + sizeof(uint32_t)) != cudaSuccess) {
        set_cuda_error("qwn_matmul_q8_create: allocation", cudaGetLastError());
        matmul_release(m);
        return QWN_CUDA_STATUS_OUT_OF_MEMORY;
    }
    m->scales = reinterpret_cast<float *>(m->w + wb);
    m->bias = o->bias_dev ? m->scales + m->n : nullptr;
    m->status = reinterpret_cast<uint32_t *>(m->scales + 2 * (size_t)m->n);
    const uint64_t chunks = wb / 16;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)std::min<uint64_t>((chunks + 255) / 256, (uint64_t)m->sms * 16));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    e = cudaLaunchKernelEx(&cfg, pack_weight_kernel, o->weight_dev, stride, m->n, m->k, chunks, m->w);
    if (e == cudaSuccess) count_launch();
    if (e == cudaSuccess) e = cudaMemcpyAsync(m->scales, o->scales_dev, fb, cudaMemcpyDeviceToDevice, s);
    if (e == cudaSuccess && m->bias) e = cudaMemcpyAsync(m->bias, o->bias_dev, fb, cudaMemcpyDeviceToDevice, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(m->status, 0, sizeof(uint32_t), s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) {
        set_cuda_error("qwn_matmul_q8_create: copy", e);
        matmul_release(m);
        return QWN_CUDA_STATUS_RUNTIME_ERROR;
    }
    if (!encode_codes(&m->wmap, m->w, kMmK, (uint64_t)m->kblocks * m->n, kMmK, kMmRows)) {
        set_error("qwn_matmul_q8_create: the driver has no tensor maps");
        matmul_release(m);
        return QWN_CUDA_STATUS_UNSUPPORTED;
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
    a.sx = r->scales_dev, a.sw = m->scales, a.bias = m->bias;
    a.out = r->out_dev, a.out_stride = os;
    a.m = r->rows, a.n = m->n, a.kblocks = m->kblocks;
    a.status = m->status;
    cudaStream_t s = static_cast<cudaStream_t>(r->stream);
    const uint64_t stride = (xs + 15) / 16 * 16;  // of a single row: any
    cudaError_t e;
    if (r->out_dtype == QWN_DTYPE_F32) e = launch_matmul<float>(*m, a, r->codes_dev, stride, s);
    else if (r->out_dtype == QWN_DTYPE_F16) e = launch_matmul<__half>(*m, a, r->codes_dev, stride, s);
    else e = launch_matmul<__nv_bfloat16>(*m, a, r->codes_dev, stride, s);
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
