// Causal attention of many query rows on the tensor core: the kernel behind
// qwn_kv_chunk_attention (keys and values in the paged cache) and
// qwn_prompt_attention (keys and values as rows).
//
// Per query row q at position p, over the tokens t that it sees (t <= p, and
// t > p - window where there is one):
//     s_t = scale q.k_t,   out = sum_t 2^(c s_t - M) v_t / sum_t 2^(c s_t - M)
// with c = log2 e and M near the largest c s_t so far.  M moves, and with it the
// sums, only when a row's largest score has outgrown it by kSlack (as factors of
// two): then the sums of the 128 rows are read from tensor memory, scaled and put
// back; otherwise they stay where the MMAs add to them.
//
// The rows of one kv head's query heads are one matrix: row r of a sequence is
// token r / group, head r % group, so that a tile of 128 rows reads each key and
// value once for all heads that share it.  Both products run on tcgen05 (M = 128
// rows): S = Q K^T from shared memory, then O += P V with P as the A operand out
// of tensor memory, where it lies over the S that it came from.
//
// A CTA has 16 warps, or 20:
//   0-3, 4-7   softmax, one thread per row: S out of tensor memory, P back into it
//   8-11       helpers: Q into shared memory; cached tiles into operand tiles;
//              whatever a sequence's ends ask for.  8-15 where rows do not come by
//              TMA: four warps make K's tiles, four V's
//   then       MMAs, loads, the list of work
// The two softmax groups take turns with the tensor core.  TILES = 2: each has 128
// of the CTA's 256 rows and both read the same keys.  TILES = 1: both work on the
// same 128 rows, one on the even blocks of tokens and one on the odd ones, and
// join at the end; for few rows, where the keys are what costs.
//
// PARTS = 1: 16-bit operands.  PARTS = 3: fp32 values as three bf16 parts (8 bits
// each, exact) whose products down to 2^-16 of the largest are all taken: six
// MMAs instead of one, fp32 accuracy.  int8 codes of one scale are exact in one
// part (three MMAs), fp16 values in two (five).
//
// Measured on B200, 32 query and 8 kv heads: 8192 bf16 rows of one prompt 475 us
// (1.16 PFLOP/s of visible products; not causal 963 us, 1.14), 16384 rows of 13
// prompts 304 us; 2048 rows over 34816 tokens of 4-bit pages 1.48 ms (0.76), of fp16
// pages 1.31; 32 x 4 rows over up to 8192 int8 tokens 171 us (1.6 TB/s).  fp32 rows:
// 3.0 ms, 1.5, 10.1, 5.4 and 0.34.  Long prompts are bound by the way from scores to
// probabilities to the next scores, 3700 cycles of which the products take 2048;
// cached tiles by the instructions that convert them beside the softmax (an issue
// slot in two); few rows by the tiles in flight; three parts by one stage of K and V.
#pragma once

#include <cmath>
#include <mutex>

#include "kv_internal.cuh"
#include "kv_store.cuh"
#include "rows.cuh"
#include "tcgen05.cuh"
#include "tile_rows.cuh"

namespace qkv {
namespace {

constexpr int kAtRows = 128;  // rows of a tile: the lanes of tensor memory
// one CTA's piece of work: rows of one sequence and kv head, and the blocks of tokens that it takes
struct AtSegment {
    int32_t valid;             // 0: no more work
    int32_t rows;              // of the CTA's tiles
    uint32_t row0;             // the first, among the sequence's rows (token x group + head)
    uint32_t token_row;        // the sequence's first token among the call's rows
    int32_t seq, head;         // sequence slot (-1: unknown), kv head
    int32_t len;               // tokens that exist
    int64_t pos0;              // position of the sequence's first row
    int32_t block0, blocks;    // blocks of tokens
    int32_t whole_lo, whole_hi;// blocks in [whole_lo, whole_hi) are seen whole by every row
    int32_t slot;              // of the workspace, -1: the rows are finished here
    int32_t quarters;          // the rows, 32 at most, are in each quarter of the tile (AtShape::kQuarters)
};

struct AtArgs {
    RowMap rows;
    uint32_t group, kv_heads, query_heads, window, causal, layer;
    uint32_t dtype;            // of query and output
    float scale2, scale2_low;  // scale x log2 e, and what fp32 lacks of it
    uint64_t query_stride, key_stride, value_stride, out_stride;  // values
    const void *query, *key, *value;
    void *out;
    StoreGeo geo;              // paged
    uint32_t *status;
    uint32_t units;            // row tiles, without a split
    uint32_t *prefix;          // split: blocks before each sequence and in all, then
    float *slots;              // the partial results, of
    uint32_t slot_rows;        // rows each
    uint32_t slot_count;       // what there is room for
};
// a partial result: o[rows][128], then M[rows], l[rows]
__host__ __device__ constexpr uint32_t at_slot_floats(uint32_t rows) { return rows * (kHeadDim + 2); }

template <int SRC, int PARTS, int TILES>
struct AtShape {
    static constexpr bool kPaged = SRC != 0;
    static constexpr bool kTma = !kPaged && PARTS == 1;            // operand tiles straight from the rows
    static constexpr bool kRaw = kPaged && SRC != QWN_KV_CODEC_F16;// cached tiles by way of shared memory
    // Codes of a cache in one operand: values by dims (a row per dim, the tokens along it), as the cache's
    // tiles have them, and the tokens of a tile in the order of cached_order(), K's alike.
    static constexpr bool kByDims = kRaw && (PARTS == 1 || SRC == QWN_KV_CODEC_Q8_HEAD_F16);
    // Parts of a key or value with fp32 rows: int8 codes of one scale are exact in one, fp16 values in two.  They leave
    // room for more stages.
    static constexpr int kKvParts = PARTS == 1 || SRC == QWN_KV_CODEC_Q8_HEAD_F16 ? 1 : SRC == QWN_KV_CODEC_F16 ? 2 : 3;
    // the operands are codes, the tokens' scales go to scores and probabilities
    static constexpr bool kTokenScales = SRC == QWN_KV_CODEC_Q8_HEAD_F16 || (PARTS == 1 && SRC == QWN_KV_CODEC_Q8_B64_F32);
    // Registers per thread after the split, no more in all than the block starts with.  The softmax warps hold a
    // row's 128 scores; what they lack goes to memory (16384 rows of 13 prompts: 334 us with 184, 299 with 200).
    // Where one tile's rows read the keys, the cached codes' conversion is what counts: the scores are read twice out
    // of tensor memory instead, and twice as many helpers have the registers.
    static constexpr int kHelpers = kTma ? 4 : 8, kThreads = 384 + 32 * kHelpers;
    static constexpr int kLaunchRegs = kHelpers == 8 ? 96 : 128, kSoftmaxRegs = kTma ? 200 : 112;
    static constexpr int kHelperRegs = kTma ? 64 : 96, kOtherRegs = kHelpers == 8 ? 64 : 48;
    static_assert(2 * kSoftmaxRegs + kHelpers / 4 * kHelperRegs + kOtherRegs <= kThreads / 128 * kLaunchRegs, "registers");
    // 32 rows or fewer, as a decode step or a few drafts have, would leave three warps of a softmax group idle.  They
    // are then in the tile four times, and each warp takes a quarter of a block's tokens: its rows of P are zero
    // elsewhere, and its rows of O a partial result like those of other CTAs.  Not for fp16 pages, whose values may
    // be infinite: their product with a zero of P is not a number.
    static constexpr bool kQuarters = kByDims && PARTS == 1 && TILES == 1;
    static constexpr int kBlock = PARTS == 1 ? 128 : 64;           // tokens
    static constexpr int kTiles = kBlock / kTileTokens;            // of the cache
    static constexpr uint32_t kQBytes = (uint32_t)kAtRows * 256 * PARTS, kKvPart = (uint32_t)kBlock * 256;
    static constexpr uint32_t kKvBytes = kKvPart * kKvParts;
    // Stages of K and V: loaded ones are a ring that both go through in turn, K0 V0 K1 V1 ..; converted ones
    // are apart, so that K of the next block does not wait behind V of this one.
    // Two of V where there is room (32 x 4 rows over 4-bit pages 233 us with one, 226 with two; int8 ones the same).
    static constexpr uint32_t kRing = kTma ? 5 : 0;
    static constexpr uint32_t kStagesK = kKvParts < 3 ? 2 : 1;
    static constexpr bool kRoom = PARTS == 1 ? !kRaw || TILES == 1 : kKvParts == 1;
    static constexpr uint32_t kStagesV = kTma || kRoom ? 2 : 1;
    static constexpr uint32_t kStages = kRing ? kRing : kStagesK + kStagesV;
    static constexpr uint32_t kOperands = TILES * kQBytes + kStages * kKvBytes;
    static constexpr uint32_t kSmem = (227 - (!kTma ? 12 : TILES == 2 ? 2 : 8)) * 1024;  // the rest is static
    // where K and V of the d-th block go, and for which time
    __device__ static constexpr uint32_t k_slot(uint32_t d) { return kRing ? 2 * d % (kRing ? kRing : 1) : d % kStagesK; }
    __device__ static constexpr uint32_t k_turn(uint32_t d) { return kRing ? 2 * d / (kRing ? kRing : 1) : d / kStagesK; }
    __device__ static constexpr uint32_t v_slot(uint32_t d) {
        return kRing ? (2 * d + 1) % (kRing ? kRing : 1) : kStagesK + d % kStagesV;
    }
    __device__ static constexpr uint32_t v_turn(uint32_t d) { return kRing ? (2 * d + 1) / (kRing ? kRing : 1) : d / kStagesV; }
    static constexpr uint32_t kTileBytes = (uint32_t)tile_bytes_of(SRC);
    static constexpr uint32_t kRawAll = kRaw ? (kSmem - 1024 - kOperands) / (kRaw ? kTileBytes : 1) : 0;
    // (by four, so that a slot's tiles are always the same warps': one that had not seen each turn of a barrier
    // could take the last turn but one for the last)
    static constexpr uint32_t kRawTiles = (kRawAll > 32 ? 32 : kRawAll) & ~3u;
    static_assert(kOperands + (kTma ? 0 : 1024) <= kSmem, "operands fit");
    // With one stage of V, a block's V waits in its tiles for the last block's products.  K's bytes and V's are then
    // copied and given back apart, so that the next block's K does not wait behind them (48/8 heads, 33 fp32 rows over
    // 131105 tokens of two scales: 17000 cycles a block otherwise).  The barriers of V are kRawV further.
    static constexpr uint32_t kSides = kRaw && kKvParts == 3 ? 2 : 1, kRawV = kSides == 2 ? 16 : 0;
    static_assert(kRawTiles + kRawV <= 32, "barriers");
    static constexpr uint32_t kCodeBytes = SRC == QWN_KV_CODEC_Q8_HEAD_F16 || SRC == QWN_KV_CODEC_Q8_B64_F32 ? 2048 : 1024;
    static constexpr uint32_t kRestBytes = kRaw ? kTileBytes / 2 - kCodeBytes : 0;  // of K or V, behind both's codes
    // K of a block is converted before its V, so all its tiles are there at once
    static_assert(!kRaw || kRawTiles >= (uint32_t)kTiles, "a block's cached tiles fit");
    // tensor memory: S and P share columns; P has 16-bit pairs, PARTS of them
    static constexpr uint32_t kSColumns = PARTS == 1 ? 128 : 96, kOColumn = 2 * kSColumns;
    static_assert(kOColumn + 2 * 128 <= 512, "tensor memory");
};

constexpr uint32_t kAtStages = 5;
template <int SRC, int PARTS, int TILES>
struct alignas(1024) AtShared {  // the operands behind it start on 1024 bytes
    static constexpr bool kTokens = AtShape<SRC, PARTS, TILES>::kTokenScales;
    static constexpr int kRaw = SRC == 0 ? 1 : 32;
    // operands of K and V have landed, are free again; V of a block seen in part (loaded ones only): has landed, is ready
    uint64_t full[kAtStages], empty[kAtStages], part[kAtStages], fixed[kAtStages];
    uint64_t qfull, qempty, sfull[2], pready[2][2], ofull[2], oempty[2], joined, helped, cleared, drained;
    uint64_t segfull[2], segempty[2], rawfull[kRaw], rawempty[kRaw];
    AtSegment seg[2];
    alignas(16) float kscale[kTokens ? 4 : 1][kTokens ? 128 : 4];  // of a block's tokens; read four at a time
    alignas(16) float vscale[kTokens ? 4 : 1][kTokens ? 128 : 4];
    alignas(16) float vtop[4][8];                  // log2 of a bound on a cached tile's value scales
    float ml[2][2][TILES == 1 ? kAtRows : 1][2];   // M and l of both groups' rows, by segment parity
    float qscale[2][SRC && PARTS == 1 ? TILES * kAtRows : 1];  // what a row of Q was divided by, by segment parity
    uint32_t odd_v[4][2][16];                      // tokens with values that are not finite, in blocks seen in part
    uint32_t tmem;
    int give_up;
};

// Bounded waits that also end when another role of the CTA has given up.  The
// answer is the whole warp's, so that its loops stay uniform: the roles that issue
// copies and MMAs then have counters and descriptors in uniform registers (8192
// rows of 32/8 heads: 570 us without, 500 with it, the rest as it was then).
__device__ __forceinline__ bool at_wait(volatile int &give_up, uint64_t *bar, uint32_t parity) {
    bool ok = false;
    for (uint32_t it = 0; it < kWaitLimit; ++it) {
        ok = mbar_try_wait(bar, parity);
        if (ok || ((it & 63) == 63 && give_up)) break;
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) give_up = 1;
    return ok;
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// all lanes' work is done: one arrival for the warp
__device__ __forceinline__ void warp_arrive(uint64_t *bar, int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

// ---- tensor memory and MMAs of 16-bit operands ------------------------------
__host__ __device__ constexpr uint32_t f16_desc(bool bf16, uint32_t n, bool b_by_rows) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_by_rows ? 1u : 0u) << 16) | ((n >> 3) << 17) |
           ((128u >> 4) << 24);
}
// D += A B^T, both from shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
        : "memory");
}
// the same with A in tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
        : "memory");
}
// B by rows of K (values: a token's dims side by side), 64-wide columns of 128-byte
// rows: the columns' distance, and 8 rows to the next 8
__device__ __forceinline__ uint64_t rows_desc(uint32_t addr, uint32_t column_bytes) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(column_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
#define QKV_R8(r, b) "=r"(r[b]), "=r"(r[b + 1]), "=r"(r[b + 2]), "=r"(r[b + 3]), "=r"(r[b + 4]), "=r"(r[b + 5]), "=r"(r[b + 6]), "=r"(r[b + 7])
#define QKV_R64(r, b) QKV_R8(r, b), QKV_R8(r, b + 8), QKV_R8(r, b + 16), QKV_R8(r, b + 24), QKV_R8(r, b + 32), QKV_R8(r, b + 40), QKV_R8(r, b + 48), QKV_R8(r, b + 56)
// 64 columns of the warp's 32 lanes, complete on return; in two loads, as one may
// not take more registers than a thread has at launch
__device__ __forceinline__ void tmem_load64(uint32_t *r, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31" "}, [%64];\n"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63" "}, [%65];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : QKV_R64(r, 0)
        : "r"(addr), "r"(addr + 32)
        : "memory");
}
// the same for 128 columns, in two loads behind one wait
__device__ __forceinline__ void tmem_load128(uint32_t *r, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63" "}, [%128];\n"
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
        "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
        "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,"
        "%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127" "}, [%129];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : QKV_R64(r, 0), QKV_R64(r, 64)
        : "r"(addr), "r"(addr + 64)
        : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// ---- the work ----------------------------------------------------------------

// sequence i of the batch
struct AtSequence {
    int64_t begin, rows;   // its tokens' rows
    int32_t seq, len;
    int64_t pos0;
};
__device__ __forceinline__ AtSequence at_sequence(const AtArgs &a, bool paged, uint32_t i) {
    AtSequence s;
    int64_t b = i, e = (int64_t)i + 1;
    if (a.rows.row_begin) {
        b = a.rows.row_begin[i];
        e = a.rows.row_begin[i + 1];
    } else if (!paged) {
        b = 0;
        e = a.rows.num_rows;
    }
    s.begin = max(b, (int64_t)0);
    s.rows = max(min(e, (int64_t)a.rows.num_rows) - s.begin, (int64_t)0);
    if (paged) {
        const int32_t id = a.rows.seq_ids ? a.rows.seq_ids[i] : (int32_t)i;
        const bool known = id >= 0 && (uint32_t)id < a.geo.max_seqs;
        s.seq = known ? id : -1;
        s.len = known ? min((int64_t)max(a.geo.seq_lens[id], 0), (int64_t)a.geo.mp * a.geo.page_tokens) : 0;
        s.pos0 = (a.rows.first_pos ? (int64_t)a.rows.first_pos[i] : known ? (int64_t)a.geo.seq_lens[id] - (e - b) : 0) +
                 (s.begin - b);
    } else {
        s.seq = (int32_t)i;
        s.len = (int32_t)s.rows;
        s.pos0 = 0;
    }
    return s;
}
// the tokens [lo, hi) that a row at a position sees; none where the position does not exist
struct Seen {
    int32_t lo, hi;
};
__device__ __forceinline__ Seen at_seen(const AtArgs &a, int64_t pos, int32_t len) {
    Seen s = {0, 0};
    if (pos < 0 || pos >= len) return s;
    s.hi = a.causal ? (int32_t)pos + 1 : len;
    if (a.window && pos + 1 > (int64_t)a.window) s.lo = (int32_t)(pos + 1 - a.window);
    return s;
}
// the blocks that rows at positions p0 .. p1 see some of
__device__ __forceinline__ void at_blocks(const AtArgs &a, int64_t p0, int64_t p1, int32_t len, int block, int32_t &b0,
                                          int32_t &b1) {
    p0 = max(p0, (int64_t)0);
    p1 = min(p1, (int64_t)len - 1);
    b0 = b1 = 0;
    if (p0 > p1) return;
    b0 = at_seen(a, p0, len).lo / block;
    b1 = (at_seen(a, p1, len).hi + block - 1) / block;
}
// the tile of `rows` rows that starts at row0 of a sequence, its blocks first .. first + count - 1 (count < 0: all)
__device__ __forceinline__ AtSegment at_segment(const AtArgs &a, const AtSequence &s, uint32_t row0, uint32_t most,
                                                int32_t head, int block) {
    AtSegment t;
    t.valid = 1;
    t.row0 = row0;
    t.rows = (int32_t)min((uint64_t)most, (uint64_t)s.rows * a.group - row0);
    t.token_row = (uint32_t)s.begin;
    t.seq = s.seq;
    t.head = head;
    t.len = s.len;
    t.pos0 = s.pos0;
    // rows that do not exist count for nothing
    const int64_t p0 = max(s.pos0 + row0 / a.group, (int64_t)0);
    const int64_t p1 = min(s.pos0 + (row0 + (uint32_t)t.rows - 1) / a.group, (int64_t)s.len - 1);
    const Seen first = at_seen(a, p0, s.len), last = at_seen(a, p1, s.len);
    t.block0 = first.lo / block;
    t.blocks = p0 > p1 ? 0 : (last.hi + block - 1) / block - t.block0;
    t.whole_lo = (last.lo + block - 1) / block;
    t.whole_hi = first.hi / block;
    t.slot = -1;
    t.quarters = 0;
    return t;
}
__device__ __forceinline__ uint64_t at_row_tiles(const AtArgs &a, const AtSequence &s, uint32_t tile_rows) {
    return ((uint64_t)s.rows * a.group + tile_rows - 1) / tile_rows;
}
// blocks of a sequence's last tile up to its first tile's begin: what each of its tiles counts as
__device__ __forceinline__ uint32_t at_span(const AtArgs &a, const AtSequence &s, int block, int32_t &first) {
    int32_t b1;
    at_blocks(a, s.pos0, s.pos0 + s.rows - 1, s.len, block, first, b1);
    return (uint32_t)max(b1 - first, 1);  // a tile without tokens still writes its rows
}

// The CTA's segments, one after another, by one whole warp.
//
// Without a split the CTAs take row tiles in turn, forth and back: tile u of
// (sequence, tile) pairs counted by base_i = begin_i group / R + i, which covers
// any ragged batch without a table.  A sequence's last tiles see the most tokens
// and go first.
//
// With one, the blocks of all tiles in a row (sequence, tile, head, block) are cut
// into as many equal runs as there are CTAs; a tile that a cut goes through is
// finished by the join kernel.
// The runs of `total` blocks over `ctas` CTAs: the first `more` of them have one block more than `each`.
struct AtRuns {
    uint32_t each, more;
    __device__ __forceinline__ AtRuns(uint32_t total, uint32_t ctas) : each(total / ctas), more(total % ctas) {}
    __device__ __forceinline__ uint32_t begin(uint32_t cta) const { return cta * each + min(cta, more); }
    __device__ __forceinline__ uint32_t owner(uint32_t block) const {
        const uint32_t longer = more * (each + 1);
        return block < longer ? block / (each + 1) : more + (block - longer) / each;
    }
};
// CTAs that work: each with a block at least, or one for each of its two groups
template <int TILES>
__device__ __forceinline__ uint32_t at_runs(uint32_t total, uint32_t ctas) {
    return min(ctas, TILES == 1 ? (total + 1) / 2 : total);
}
template <int SRC, int PARTS, int TILES>
struct AtWork {
    using S = AtShape<SRC, PARTS, TILES>;
    static constexpr uint32_t kRows = TILES * kAtRows;
    const AtArgs &a;
    uint32_t at, end;      // run of blocks
    uint32_t i, span, n;   // sequence, its blocks per tile, segments so far
    int32_t first;
    uint32_t item, from;   // (row tile, head) of the sequence, block of it
    uint32_t item0;        // those of the sequences before
    AtSequence s;
    // of 32 sequences, one per lane: read once and handed round, as code that runs once costs its fetch
    uint32_t held, my_items, my_span;
    int32_t my_first;
    AtSequence my;

    __device__ __forceinline__ explicit AtWork(const AtArgs &args) : a(args) {
        at = end = i = span = n = item = from = item0 = 0;
        first = 0;
        if (!a.slots) return;
        const uint32_t lane = threadIdx.x & 31;
        uint32_t total = 0;
        for (uint32_t k = 0; k < a.rows.num_seqs; k += 32) {
            hold(k);
            total += __reduce_add_sync(0xffffffffu, my_items * my_span);
        }
        const uint32_t ctas = at_runs<TILES>(total, gridDim.x);
        if (blockIdx.x >= ctas) return;
        const AtRuns runs(total, ctas);
        at = runs.begin(blockIdx.x);
        end = runs.begin(blockIdx.x + 1);
        uint32_t before = 0, within = 0, items_before = 0;
        bool found = false;
        for (uint32_t k = 0; k < a.rows.num_seqs; k += 32) {
            if (held != k) hold(k);
            const uint32_t w = my_items * my_span;
            uint32_t upto = w, items_upto = my_items;
#pragma unroll 1
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o), z = __shfl_up_sync(0xffffffffu, items_upto, o);
                if (lane >= (uint32_t)o) upto += y, items_upto += z;
            }
            if (blockIdx.x == 0) {  // the tables for the join kernel
                if (k + lane < a.rows.num_seqs) {
                    a.prefix[k + lane] = before + upto - w;
                    a.prefix[a.rows.num_seqs + 1 + k + lane] = items_before + items_upto - my_items;
                }
                if (lane == 0) a.prefix[a.rows.num_seqs] = total;
            }
            const uint32_t has = __ballot_sync(0xffffffffu, before + upto > at);
            if (has && !found) {
                const int l = __ffs(has) - 1;
                i = k + l;
                within = at - (before + __shfl_sync(0xffffffffu, upto - w, l));
                item0 = items_before + __shfl_sync(0xffffffffu, items_upto - my_items, l);
                found = true;
                if (blockIdx.x != 0) break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
            items_before += __shfl_sync(0xffffffffu, items_upto, 31);
        }
        open();
        item = within / span;
        from = within - item * span;
    }
    __device__ __noinline__ void hold(uint32_t k) {
        const uint32_t lane = threadIdx.x & 31;
        held = k;
        my_items = 0;
        my_span = 1;
        my_first = 0;
        if (k + lane >= a.rows.num_seqs) return;
        my = at_sequence(a, S::kPaged, k + lane);
        my_span = at_span(a, my, S::kBlock, my_first);
        my_items = (uint32_t)at_row_tiles(a, my, kRows) * a.kv_heads;
    }
    uint32_t items;  // of the sequence
    __device__ __noinline__ void open() {
        if (held != (i & ~31u)) hold(i & ~31u);
        const int l = i & 31;
        auto from_lane = [&](auto v) { return __shfl_sync(0xffffffffu, v, l); };
        s.begin = from_lane(my.begin);
        s.rows = from_lane(my.rows);
        s.seq = from_lane(my.seq);
        s.len = from_lane(my.len);
        s.pos0 = from_lane(my.pos0);
        span = from_lane(my_span);
        first = from_lane(my_first);
        items = from_lane(my_items);
    }
    __device__ __forceinline__ AtSegment next() {
        AtSegment t{};
        if (!a.slots) {
            const uint32_t all = a.units * a.kv_heads;
            for (;;) {
                if (n >= (all + gridDim.x - 1) / gridDim.x) return t;
                const uint32_t k = n * gridDim.x + (n & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                n++;
                if (k < all) t = single(a.units - 1 - k / a.kv_heads, k % a.kv_heads);
                if (t.valid) return t;
            }
        }
        while (at < end) {
            if (item >= items) {  // the next sequence
                item0 += items;
                if (++i >= a.rows.num_seqs) return t;
                item = from = 0;
                open();
                continue;
            }
            const uint32_t count = min(span - from, end - at);
            t = at_segment(a, s, item / a.kv_heads * kRows, kRows, (int32_t)(item % a.kv_heads), S::kBlock);
            // of the tile's own blocks those in the run
            const int32_t b0 = max(t.block0, first + (int32_t)from), b1 = min(t.block0 + t.blocks, first + (int32_t)(from + count));
            // A slot for each (tile, CTA): their indexes' sum grows along the work.  Only a run's first and last tile can
            // be cut, so that two slots per CTA do without quarters.
            t.quarters = S::kQuarters && t.rows <= 32;
            if (S::kQuarters && (t.quarters || count != span)) t.slot = (int32_t)(item0 + item + blockIdx.x);
            else if (count != span) t.slot = (int32_t)(2 * blockIdx.x + (n ? 1 : 0));
            // (more tiles than the rows make: sequences that overlap)
            if (t.slot >= (int32_t)a.slot_count || t.slot < -1) {
                latch(a.status, QWN_KV_STATUS_BAD_LENGTH);
                return AtSegment{};
            }
            t.block0 = b0;
            t.blocks = max(b1 - b0, 0);
            at += count;
            n++;
            item++;  // the run ends here, or the tile does
            from = 0;
            return t;
        }
        return t;
    }
    __device__ __forceinline__ AtSegment single(uint32_t u, uint32_t head) const {
        AtSegment t{};
        const uint32_t lane = threadIdx.x & 31;
        uint32_t lo = 0, count = a.rows.num_seqs;  // the last sequence whose base is not beyond u
        while (count > 1 && a.rows.row_begin) {
            const uint32_t step = (count + 31) / 32, k = lo + lane * step;
            const bool below = lane * step < count && base(k) <= u;
            const uint32_t last = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1u);
            count = min(step, count - last * step);
            lo += last * step;
        }
        if (!a.rows.row_begin && S::kPaged) lo = u / max(base(1), 1u);  // as many rows each
        if (lo >= a.rows.num_seqs) return t;
        const AtSequence q = at_sequence(a, S::kPaged, lo);
        const uint64_t first_unit = base(lo);
        if (u < first_unit || u - first_unit >= at_row_tiles(a, q, kRows)) return t;
        return at_segment(a, q, (uint32_t)(u - first_unit) * kRows, kRows, (int32_t)head, S::kBlock);
    }
    // the first unit of a sequence
    __device__ __forceinline__ uint32_t base(uint32_t k) const {
        if (a.rows.row_begin) return (uint32_t)((uint64_t)max(a.rows.row_begin[k], 0) * a.group / kRows) + k;
        return k * ((a.group + kRows - 1) / kRows);
    }
};

// ---- Q ------------------------------------------------------------------------

// bf16 parts of eight fp32 values: each takes the next 8 bits, so that three are exact
template <int N>
__device__ __forceinline__ void split(const float *v, uint4 (&part)[N]) {
    uint32_t w[N][4];
    float x[8];
    uint64_t zero = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        zero = fma2(pair(v[i], v[i + 1]), 0, zero);  // NaN where one is not finite
        const uint32_t a = __float_as_uint(v[i]), b = __float_as_uint(v[i + 1]);
        w[0][i >> 1] = prmt(a, b, 0x7632u);
        if constexpr (N > 1)
            unpair(add2(pair(v[i], v[i + 1]), pair(__uint_as_float((a & 0xFFFF0000u) ^ 0x80000000u),
                                                   __uint_as_float((b & 0xFFFF0000u) ^ 0x80000000u))), x[i], x[i + 1]);
    }
    float z0, z1;
    unpair(zero, z0, z1);
    if (z0 + z1 != 0.f) {  // they stay whole in the first part (a NaN keeps a bit set)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t u = __float_as_uint(v[i]);
            if ((u & 0x7F800000u) == 0x7F800000u && (u & 0xFFFFu)) w[0][i >> 1] |= 1u << (16 * (i & 1));
            if (N > 1 && !isfinite(v[i])) x[i] = 0.f;
        }
    }
#pragma unroll
    for (int k = 1; k < N; k++)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const uint32_t a = __float_as_uint(x[i]), b = __float_as_uint(x[i + 1]);
            w[k][i >> 1] = prmt(a, b, 0x7632u);
            if (k + 1 < N)
                unpair(add2(pair(x[i], x[i + 1]), pair(__uint_as_float((a & 0xFFFF0000u) ^ 0x80000000u),
                                                       __uint_as_float((b & 0xFFFF0000u) ^ 0x80000000u))), x[i], x[i + 1]);
        }
#pragma unroll
    for (int k = 0; k < N; k++) part[k] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cp_async16_at(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16-byte chunk c (of 16) of row r in an operand tile of `rows` rows: two columns of 128-byte rows, swizzled
__device__ __forceinline__ uint32_t chunk_at(uint32_t base, uint32_t rows, uint32_t r, uint32_t c) {
    return base + (c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}
// The 32 rows of a warp in a tile of Q, two at a time: 16 lanes read a row side by
// side (a lane per row took 7 us for 256 rows, 32 lines to an instruction).  For a
// cache, whose codes are f16 operands, a row of bf16 is brought into f16's range by
// a power of two.
template <int SRC, int PARTS>
__device__ __forceinline__ void put_q(const AtArgs &a, const AtSegment &t, uint32_t row0, uint32_t tile, float *unit) {
    const uint32_t lane = threadIdx.x & 31, c = lane & 15, w0 = threadIdx.x & 96;  // the warp's first row in the tile
    const uint32_t first = t.quarters ? 0 : w0;                                    // and of the segment
    uint64_t mine = 0;  // where the lane's row starts
    const bool have = (int32_t)(row0 + first + lane) < t.rows;
    if (have) {
        const uint32_t row = t.row0 + row0 + first + lane, token = row / a.group;
        mine = (uint64_t)(t.token_row + token) * a.query_stride + (t.head * a.group + row - token * a.group) * kHeadDim;
    }
    const uint32_t rows = __ballot_sync(0xffffffffu, have);
    if constexpr (SRC == 0 && PARTS == 1) {  // as it is
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) {
            const uint32_t r = 2 * i + (lane >> 4);
            const uint64_t at = __shfl_sync(0xffffffffu, mine, r) + 8 * c;
            if (rows >> r & 1) cp_async16_at(chunk_at(tile, kAtRows, w0 + r, c), static_cast<const uint16_t *>(a.query) + at);
        }
        return;
    }
    constexpr int kAhead = 4;  // loads in flight (few, as a first time through code costs its fetch)
#pragma unroll 1
    for (uint32_t i0 = 0; i0 < 16; i0 += kAhead) {
        if (!(rows >> (2 * i0))) break;
        uint4 w[kAhead][PARTS == 3 ? 2 : 1];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; i++) {
            const uint32_t r = 2 * (i0 + i) + (lane >> 4);
            const uint64_t at = __shfl_sync(0xffffffffu, mine, r) + 8 * c;
#pragma unroll
            for (int k = 0; k < (PARTS == 3 ? 2 : 1); k++) w[i][k] = make_uint4(0, 0, 0, 0);
            if (rows >> r & 1) {
                if constexpr (PARTS == 3) {
                    const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const float *>(a.query) + at);
                    w[i][0] = q[0];
                    w[i][1] = q[1];
                } else {
                    w[i][0] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.query) + at);
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kAhead; i++) {
            const uint32_t r = w0 + 2 * (i0 + i) + (lane >> 4);
            if constexpr (PARTS == 3) {
                uint4 p[3];
                split(reinterpret_cast<const float *>(w[i]), p);
#pragma unroll
                for (uint32_t k = 0; k < 3; k++) st_shared16(chunk_at(tile + k * kAtRows * 256, kAtRows, r, c), p[k]);
            } else {
                uint32_t u[4] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w};
                if (SRC != 0) {
                    float scale = 1.f;
                    if (a.dtype == QWN_DTYPE_BF16) {
                        uint32_t top = 0;  // largest exponent of a finite value
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint32_t e0 = u[k] & 0x7F80u, e1 = (u[k] >> 16) & 0x7F80u;
                            top = max(top, max(e0 == 0x7F80u ? 0u : e0, e1 == 0x7F80u ? 0u : e1));
                        }
#pragma unroll
                        for (int o = 1; o < 16; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                        // the largest value to 2^8 .. 2^9: what is below 2^-22 of it loses bits
                        const int e = max(-100, min((int)(top >> 7) - 127 - 8, 119));
                        scale = __uint_as_float((uint32_t)(e + 127) << 23);
                        const float per = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            u[k] = pack_h2(__uint_as_float(u[k] << 16) * per, __uint_as_float(u[k] & 0xFFFF0000u) * per);
                    }
                    if (c == 0) unit[row0 + r] = scale;
                }
                // dims in the order that K's words give them
                if constexpr (SRC == QWN_KV_CODEC_Q4_G32) {
                    const uint32_t v[4] = {u[0], u[1], u[2], u[3]};
                    u[0] = prmt(v[0], v[1], 0x5410u), u[1] = prmt(v[2], v[3], 0x5410u);
                    u[2] = prmt(v[0], v[1], 0x7632u), u[3] = prmt(v[2], v[3], 0x7632u);
                } else if constexpr (SRC == QWN_KV_CODEC_TQ35_G64) {  // even dims of 16 to the first chunk, odd ones to the second
                    uint32_t o[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) o[k] = __shfl_xor_sync(0xffffffffu, u[k], 1);
                    const bool odd = c & 1;
                    const uint32_t sel = odd ? 0x7632u : 0x5410u;
                    const uint32_t x[4] = {odd ? o[0] : u[0], odd ? o[1] : u[1], odd ? o[2] : u[2], odd ? o[3] : u[3]};
                    const uint32_t y[4] = {odd ? u[0] : o[0], odd ? u[1] : o[1], odd ? u[2] : o[2], odd ? u[3] : o[3]};
                    u[0] = prmt(x[0], x[2], sel), u[1] = prmt(y[0], y[2], sel);
                    u[2] = prmt(x[1], x[3], sel), u[3] = prmt(y[1], y[3], sel);
                }
                st_shared16(chunk_at(tile, kAtRows, r, c), make_uint4(u[0], u[1], u[2], u[3]));
            }
        }
    }
}

// ---- keys and values ------------------------------------------------------------

// Where token t of a cached tile goes among its 16 operand columns, and back: the four tokens that a lane's words
// of V hold (2a, 2a + 1, 2a + 8, 2a + 9) are neighbours.  Scores and probabilities are in this order.
__host__ __device__ constexpr int cached_order(int t) { return 4 * ((t & 7) >> 1) + (t & 1) + 2 * (t >> 3); }
__host__ __device__ constexpr int cached_token(int column) {
    return (column & ~15) + 2 * ((column & 15) >> 2) + (column & 1) + 8 * ((column >> 1) & 1);
}
// the page that holds a token, as the table has it
__device__ __forceinline__ int32_t at_page(const AtArgs &a, int32_t seq, int32_t token) {
    return a.geo.page_table[(size_t)seq * a.geo.mp + (uint32_t)token / a.geo.page_tokens];
}
// a cached tile's address in it, for a token that exists; a bad page latches and reads page 0
__device__ __forceinline__ const uint8_t *at_tile_in(const AtArgs &a, int32_t page, int32_t head, int32_t token) {
    const StoreGeo &g = a.geo;
    if (page < 0 || (uint32_t)page >= g.total_pages) {
        latch(a.status, QWN_KV_STATUS_BAD_PAGE);
        page = 0;
    }
    return g.pages + (size_t)page * g.page_bytes +
           ((size_t)(a.layer * g.kv_heads + head) * g.tpp + (uint32_t)token % g.page_tokens / kTileTokens) * g.tile_bytes;
}
__device__ __forceinline__ const uint8_t *at_tile(const AtArgs &a, int32_t seq, int32_t head, int32_t token) {
    return at_tile_in(a, at_page(a, seq, token), head, token);
}

// What the operands hold of a cached value, so that f16 holds it without loss of range: int8 codes by
// themselves (per 64 channels: times the half's share of the token's larger scale), with the token's scale
// applied to its score and its probability; 4- and 3.5-bit values halved (at most 65504 + 65504); fp16 as it is.
template <int SRC>
struct AtScale {
    static constexpr float kFixed = SRC == QWN_KV_CODEC_TQ35_G64 || SRC == QWN_KV_CODEC_Q4_G32 ? 2.f : 1.f;
};
// the scale of K (which 0) or V of token t
template <int SRC>
__device__ __forceinline__ float token_scale(const uint8_t *tile, int t, int which) {
    if constexpr (SRC == QWN_KV_CODEC_Q8_HEAD_F16) {
        return h2f(*reinterpret_cast<const uint16_t *>(tile + (which ? 4128 : 4096) + s16_off(t)));
    } else {
        const uint8_t *s = tile + (which ? 4224 : 4096);
        return fmaxf(*reinterpret_cast<const float *>(s + s32_off(t, 0)), *reinterpret_cast<const float *>(s + s32_off(t, 1)));
    }
}
// a row's 16 values of this lane as bf16 parts, and into an operand tile
template <int N>
struct RowParts {
    uint4 p[2][N];
    __device__ __forceinline__ void set(const Row16 &x) {
#pragma unroll
        for (int h = 0; h < 2; h++) split(x.v + 8 * h, p[h]);
    }
    __device__ __forceinline__ void put(uint32_t base, uint32_t rows, uint32_t r, int j) const {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (uint32_t k = 0; k < N; k++) st_shared16(chunk_at(base + k * rows * 256, rows, r, 8 * h + j), p[h][k]);
    }
};

// Cached tiles as f16 operands, by one warp: codes to f16 by exponent tricks (exact), then one rounded step for
// what is not exact.
__device__ __forceinline__ void st_shared8(uint32_t addr, uint32_t a, uint32_t b) {
    asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
// Halved values of low-bit codes.  V: in f16, where the step's own rounding is up to range x 2^-12 in the value of
// the largest code, too little to see beside P's.  K: in fp32 and rounded once, since that error is the same for
// all of a group's dims, and a query's outlier multiplies it (2048 rows over a 4-bit cache with outliers: outputs
// off by 3.0 to 3.8e-3 of their norm with f16 steps, where bf16's own rounding makes 1.6e-3).
template <int LEVELS>
__device__ __forceinline__ uint32_t half_steps(uint32_t ranges) {  // a pair of ranges over 2 LEVELS, rounded once
    constexpr float f = 0.5f / LEVELS, near = LEVELS == 15 ? 1092.f / 32768.f : 1170.f / 16384.f;  // f16's nearest, and
    return hfma2(ranges, pack_h2(near, near), hmul2(ranges, pack_h2(f - near, f - near)));         // what that lacks
}
__device__ __forceinline__ uint32_t key_pair(uint32_t codes, float step, float low) {
    float a, b;
    unpair(fma2(pair(h2f((uint16_t)codes), h2f((uint16_t)(codes >> 16))), pair(step, step), pair(low, low)), a, b);
    return pack_h2(a, b);
}
__device__ __forceinline__ uint4 ld16(const uint8_t *p) { return *reinterpret_cast<const uint4 *>(p); }
// eight codes of 3.5-bit words: odd dims of half 1 have their lowest bit above half 0's and two in a plane
__device__ __forceinline__ uint32_t odd_codes(uint32_t odd, uint32_t plane, int x) {
    if (x == 0) return odd & 0x77777777u;
    uint32_t p = (plane | (plane << 8)) & 0x00FF00FFu;
    p = (p | (p << 4)) & 0x0F0F0F0Fu;
    p = (p | (p << 2)) & 0x33333333u;
    return ((odd >> 3) & 0x11111111u) | (p << 1);
}
// four int8 codes as pairs of f16 or bf16, exact; bf16's seven bits take all but the sign, which picks what is too much
template <bool BF16>
__device__ __forceinline__ void codes_to_pairs(uint32_t w, uint32_t &b01, uint32_t &b23) {
    if constexpr (BF16) {
        auto take = [](uint32_t x) {
            uint32_t d;
            asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"((x & 0x007F007Fu) | 0x43004300u), "r"((x & 0x00800080u) ^ 0x43804380u));
            return d;
        };
        b01 = take(prmt(w, 0u, 0x4140u));
        b23 = take(prmt(w, 0u, 0x4342u));
    } else {
        u8x4_to_h2x2(w, b01, b23);
    }
}
// K of a tile: rows of 128 dims (in the order that put_q gives the queries).  What
// a lane converts is loaded before it stores anything.
template <int SRC, bool BF16>
struct KeyWords {
    static constexpr bool kInt8 = SRC == QWN_KV_CODEC_Q8_HEAD_F16 || SRC == QWN_KV_CODEC_Q8_B64_F32;
    uint4 w[4];   // int8: 16 codes of rows t, t + 4, ..; 4-bit: words of t and t + 8, their parameters; 3.5-bit: likewise
    __device__ __forceinline__ void load(const uint8_t *tile) {
        const int lane = threadIdx.x & 31;
        if constexpr (kInt8) {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = ld16(tile + 512 * i + 16 * lane);
        } else if constexpr (SRC == QWN_KV_CODEC_Q4_G32) {
            w[0] = ld16(tile + 16 * lane);
            w[1] = ld16(tile + 512 + 16 * lane);
            w[2] = ld16(tile + 2048 + 32 * (lane >> 2));
            w[3] = ld16(tile + 2048 + 32 * (lane >> 2) + 16);
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint2 e = *reinterpret_cast<const uint2 *>(tile + 256 * i + 8 * lane);
                w[i] = make_uint4(e.x, e.y, *reinterpret_cast<const uint32_t *>(tile + 512 + 128 * i + 4 * lane),
                                  *reinterpret_cast<const uint16_t *>(tile + 768 + 64 * i + 2 * lane));
            }
            w[2] = ld16(tile + 896 + 16 * (lane >> 2));
        }
    }
    // `tile` still holds the scales of int8 codes per 64 channels
    template <int BLOCK>
    __device__ __forceinline__ void store(const uint8_t *tile, int ti, uint32_t base) const {
        const int lane = threadIdx.x & 31;
        if constexpr (kInt8) {
            const int at = lane & 7;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = 4 * i + (lane >> 3), d16 = at ^ ((t & 1) << 2), half = d16 >> 2;
                uint32_t h[8];
                codes_to_pairs<BF16>(w[i].x, h[0], h[1]);
                codes_to_pairs<BF16>(w[i].y, h[2], h[3]);
                codes_to_pairs<BF16>(w[i].z, h[4], h[5]);
                codes_to_pairs<BF16>(w[i].w, h[6], h[7]);
                if constexpr (SRC == QWN_KV_CODEC_Q8_B64_F32) {
                    const float s0 = *reinterpret_cast<const float *>(tile + 4096 + s32_off(t, 0));
                    const float s1 = *reinterpret_cast<const float *>(tile + 4096 + s32_off(t, 1));
                    const float share = __fdividef(half ? s1 : s0, fmaxf(s0, s1));
                    const uint32_t f = pack_h2(share, share);
#pragma unroll
                    for (int k = 0; k < 8; k++) h[k] = hmul2(h[k], f);
                }
                const uint32_t r = ti * kTileTokens + cached_order(t);
                // the halves' lanes write their two chunks in opposite order: eight lanes, eight banks of 16 bytes
                const uint32_t first = chunk_at(base, BLOCK, r, 2 * d16 + half);
                const uint4 lo = make_uint4(h[0], h[1], h[2], h[3]), hi = make_uint4(h[4], h[5], h[6], h[7]);
                st_shared16(first, half ? hi : lo);
                st_shared16(first ^ 16, half ? lo : hi);
            }
        } else {
            const int tig = lane & 3;
#pragma unroll
            for (int pass = 0; pass < 2; pass++) {
                const int t = (lane >> 2) + 8 * pass;
                const uint32_t r = ti * kTileTokens + cached_order(t);
                if constexpr (SRC == QWN_KV_CODEC_Q4_G32) {
                    const uint32_t par[4] = {pass ? w[2].y : w[2].x, pass ? w[2].w : w[2].z, pass ? w[3].y : w[3].x, pass ? w[3].w : w[3].z};
                    const uint32_t word[4] = {w[pass].x, w[pass].y, w[pass].z, w[pass].w};
                    const bool odd = t & 1;
#pragma unroll
                    for (int k = 0; k < 4; k++) {  // odd tokens in another order, for the banks
                        const uint32_t c = odd ? k ^ 1 : k, p = odd ? par[k ^ 1] : par[k];
                        const float step = h2f((uint16_t)p) * (0.5f / 15.f), low = h2f((uint16_t)(p >> 16)) * 0.5f;
                        uint32_t v[4];
                        nib8_to_h2x4(odd ? word[k ^ 1] : word[k], v);
#pragma unroll
                        for (int i = 0; i < 4; i++) v[i] = key_pair(v[i], step, low);
                        st_shared16(chunk_at(base, BLOCK, r, 4 * c + tig), make_uint4(v[0], v[1], v[2], v[3]));
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const uint32_t p = x ? (pass ? w[2].w : w[2].z) : (pass ? w[2].y : w[2].x);
                        const float range = h2f((uint16_t)p), low = h2f((uint16_t)(p >> 16)) * 0.5f;
#pragma unroll
                        for (int o = 0; o < 2; o++) {
                            const float step = range * (o ? 0.5f / 7.f : 0.5f / 15.f);
                            uint32_t v[4];
                            nib8_to_h2x4(o ? odd_codes(w[pass].z, w[pass].w, x) : x ? w[pass].y : w[pass].x, v);
#pragma unroll
                            for (int i = 0; i < 4; i++) v[i] = key_pair(v[i], step, low);
                            st_shared16(chunk_at(base, BLOCK, r, 8 * x + 2 * tig + o), make_uint4(v[0], v[1], v[2], v[3]));
                        }
                    }
                }
            }
        }
    }
};
// V of a tile: of each dim the 16 tokens.  Lane 4 r + a has the tokens 2a, 2a + 1, 2a + 8, 2a + 9 of the dims with
// index r (and r + 8) in its classes of 16.  All is loaded before the tile's room is given back.
template <int SRC, bool BF16>
struct ValueWords {
    static constexpr bool kInt8 = SRC == QWN_KV_CODEC_Q8_HEAD_F16 || SRC == QWN_KV_CODEC_Q8_B64_F32;
    static constexpr int kPar = SRC == QWN_KV_CODEC_Q8_HEAD_F16 ? 0 : SRC == QWN_KV_CODEC_Q4_G32 ? 4 : 2;
    uint4 w[kInt8 ? 4 : 2], p[kPar ? kPar : 1];
    __device__ __forceinline__ void load(const uint8_t *tile) {
        const int lane = threadIdx.x & 31, a = lane & 3;
        if constexpr (kInt8) {
#pragma unroll
            for (int q = 0; q < 4; q++) w[q] = ld16(tile + 2048 + 64 * lane + 16 * (q ^ ((lane >> 1) & 3)));
#pragma unroll
            for (int i = 0; i < kPar; i++) p[i] = ld16(tile + 4224 + 32 * a + 16 * i);
        } else if constexpr (SRC == QWN_KV_CODEC_Q4_G32) {
#pragma unroll
            for (int i = 0; i < 2; i++) w[i] = ld16(tile + 1024 + 32 * lane + 16 * (i ^ ((lane >> 2) & 1)));
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = ld16(tile + 2304 + 64 * a + 16 * i);  // t = 2a: groups 0, 1; 2, 3; t = 2a + 1
        } else {
            w[0] = ld16(tile + 1024 + 16 * lane);
            const uint2 o = *reinterpret_cast<const uint2 *>(tile + 1536 + 8 * lane);
            w[1] = make_uint4(o.x, o.y, *reinterpret_cast<const uint32_t *>(tile + 1792 + 4 * lane), 0);
#pragma unroll
            for (int i = 0; i < 2; i++) p[i] = ld16(tile + 1920 + 32 * a + 16 * i);
        }
    }
    __device__ __forceinline__ void store(int ti, uint32_t base) const {
        const int lane = threadIdx.x & 31, a = lane & 3, r = lane >> 2;
        const uint32_t chunk = 2 * (ti & 3) + (a >> 1), to = base + (ti >> 2) * 16384 + 8 * (a & 1);
        auto put = [&](uint32_t d, uint32_t first, uint32_t second) {
            st_shared8(to + d * 128 + ((chunk ^ (d & 7)) << 4), first, second);
        };
        if constexpr (kInt8) {
            uint32_t share[2][2];  // of the dims' half, the tokens 2a, 2a + 1 and those plus 8
            if constexpr (SRC == QWN_KV_CODEC_Q8_B64_F32) {
                // (half 0 of t, of t + 8, half 1 of t, of t + 8) for t = 2a and 2a + 1
                const float s[4] = {__uint_as_float(p[0].x), __uint_as_float(p[0].y), __uint_as_float(p[0].z), __uint_as_float(p[0].w)};
                const float n[4] = {__uint_as_float(p[1].x), __uint_as_float(p[1].y), __uint_as_float(p[1].z), __uint_as_float(p[1].w)};
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        share[h][e] = pack_h2(__fdividef(s[2 * h + e], fmaxf(s[e], s[2 + e])), __fdividef(n[2 * h + e], fmaxf(n[e], n[2 + e])));
            }
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    uint32_t lo[2], hi[2];  // dims r and r + 8 of the class, tokens below and from 8
                    codes_to_pairs<BF16>(i ? w[q].z : w[q].x, lo[0], lo[1]);
                    codes_to_pairs<BF16>(i ? w[q].w : w[q].y, hi[0], hi[1]);
                    const uint32_t d = 32 * q + 16 * i + r;
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        if constexpr (SRC == QWN_KV_CODEC_Q8_B64_F32) {
                            lo[k] = hmul2(lo[k], share[q >> 1][0]);
                            hi[k] = hmul2(hi[k], share[q >> 1][1]);
                        }
                        put(d + 8 * k, lo[k], hi[k]);
                    }
                }
        } else if constexpr (SRC == QWN_KV_CODEC_Q4_G32) {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint4 s = p[c >> 1], n = p[2 + (c >> 1)];
                const uint32_t s0 = c & 1 ? s.z : s.x, s8 = c & 1 ? s.w : s.y, n0 = c & 1 ? n.z : n.x, n8 = c & 1 ? n.w : n.y;
                const uint32_t step0 = half_steps<15>(prmt(s0, n0, 0x5410u)), step8 = half_steps<15>(prmt(s8, n8, 0x5410u));
                const uint32_t low0 = hmul2(prmt(s0, n0, 0x7632u), 0x38003800u), low8 = hmul2(prmt(s8, n8, 0x7632u), 0x38003800u);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint4 y = w[c >> 1];
                    const int k = 2 * (c & 1) + i;
                    uint32_t v[4];
                    nib8_to_h2x4(k == 0 ? y.x : k == 1 ? y.y : k == 2 ? y.z : y.w, v);
                    const uint32_t d = 32 * c + 16 * i + r;
                    put(d, hfma2(v[0], step0, low0), hfma2(v[2], step8, low8));
                    put(d + 8, hfma2(v[1], step0, low0), hfma2(v[3], step8, low8));
                }
            }
        } else {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t s0 = x ? p[0].z : p[0].x, s8 = x ? p[0].w : p[0].y, n0 = x ? p[1].z : p[1].x, n8 = x ? p[1].w : p[1].y;
                const uint32_t r0 = prmt(s0, n0, 0x5410u), r8 = prmt(s8, n8, 0x5410u);
                const uint32_t low0 = hmul2(prmt(s0, n0, 0x7632u), 0x38003800u), low8 = hmul2(prmt(s8, n8, 0x7632u), 0x38003800u);
#pragma unroll
                for (int odd = 0; odd < 2; odd++) {
                    const uint32_t step0 = odd ? half_steps<7>(r0) : half_steps<15>(r0), step8 = odd ? half_steps<7>(r8) : half_steps<15>(r8);
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        const uint32_t codes = odd ? odd_codes(b ? w[1].y : w[1].x, (w[1].z >> (16 * b)) & 0xFFFFu, x)
                                                   : x ? (b ? w[0].w : w[0].z) : (b ? w[0].y : w[0].x);
                        uint32_t v[4];
                        nib8_to_h2x4(codes, v);
                        const uint32_t d = 64 * x + 32 * b + 2 * r + odd;
                        put(d, hfma2(v[0], step0, low0), hfma2(v[2], step8, low8));
                        put(d + 16, hfma2(v[1], step0, low0), hfma2(v[3], step8, low8));
                    }
                }
            }
        }
    }
};

// ---- values that a sequence's ends ask for ---------------------------------------
//
// A masked token must not matter, but 0 x inf is NaN in an MMA.  In blocks that
// some rows see only in part, values that are not finite are therefore taken out of
// the operand tile (tokens past the end altogether) and noted; the rows that do see
// them get them added at the end (odd_sum).  A CTA's rows span 256 tokens at most,
// so that such blocks span 512 from the first block on and 512 from `zone` on.
__device__ __forceinline__ int32_t odd_zone(const AtSegment &t, int block) {
    return max(t.whole_hi, max(t.whole_lo, t.block0)) * block;
}
__device__ __forceinline__ bool odd_word(uint32_t w, bool bf16, uint32_t &out) {
    const uint32_t e = bf16 ? 0x7F80u : 0x7C00u;
    const bool lo = (w & e) == e, hi = ((w >> 16) & e) == e;
    out = (lo ? 0u : w & 0xFFFFu) | (hi ? 0u : w & 0xFFFF0000u);
    return lo || hi;
}
// the same where the values lie by dims: a thread has a dim
__device__ __forceinline__ void note_odd(uint32_t (&noted)[2][16], const AtSegment &seg, int block, int32_t token) {
    const int32_t z = odd_zone(seg, block);
    const uint32_t i = (uint32_t)(token < z ? token - seg.block0 * block : token - z);
    if (i < 512) atomicOr(&noted[token < z ? 0 : 1][i >> 5], 1u << (i & 31));
}
__device__ __noinline__ void clear_odd_by_dims(uint32_t (&noted)[2][16], const AtSegment &seg, int32_t token0, uint32_t base) {
    const uint32_t d = threadIdx.x & 127;
    const int32_t left = seg.len - token0;  // tokens of the block that exist
#pragma unroll 1
    for (uint32_t c = 0; c < 16; c++) {  // eight tokens each
        const uint32_t at = base + (c >> 3) * 16384 + d * 128 + (((c & 7) ^ (d & 7)) << 4);
        const uint4 w = ld_shared16(at);
        uint32_t u[4] = {w.x, w.y, w.z, w.w};
        bool change = false;
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int32_t t = cached_token((int)(8 * c) + 2 * k + h);
                const bool odd = ((u[k] >> (16 * h)) & 0x7C00u) == 0x7C00u;
                if (odd && t < left) note_odd(noted, seg, 128, token0 + t);
                if (odd || t >= left) {
                    u[k] &= h ? 0x0000FFFFu : 0xFFFF0000u;
                    change = true;
                }
            }
        if (change) st_shared16(at, make_uint4(u[0], u[1], u[2], u[3]));
    }
}
template <int PARTS, int BLOCK>
__device__ void clear_odd(uint32_t (&noted)[2][16], const AtSegment &seg, int32_t token0, uint32_t base, bool bf16) {
    const uint32_t tid = threadIdx.x & 127, r = tid % BLOCK, c0 = tid / BLOCK * (BLOCK / 8);
    const int32_t token = token0 + (int32_t)r;
    const bool past = token >= seg.len;
    bool odd = false;
#pragma unroll 4
    for (uint32_t c = c0; c < c0 + BLOCK / 8; c++) {
        const uint32_t at = chunk_at(base, BLOCK, r, c);
        if (past) {
#pragma unroll
            for (uint32_t k = 0; k < PARTS; k++) st_shared16(at + k * BLOCK * 256, make_uint4(0, 0, 0, 0));
            continue;
        }
        const uint4 w = ld_shared16(at);
        uint4 y;
        const bool o = odd_word(w.x, bf16, y.x) | odd_word(w.y, bf16, y.y) | odd_word(w.z, bf16, y.z) | odd_word(w.w, bf16, y.w);
        if (o) st_shared16(at, y);
        odd |= o;
    }
    if (odd) note_odd(noted, seg, BLOCK, token);
}
// value d of a token
template <int SRC, int PARTS>
__device__ float at_value(const AtArgs &a, const AtSegment &seg, int32_t token, int d) {
    if constexpr (SRC != 0) {
        const float4 v = load_token<SRC>(at_tile(a, seg.seq, seg.head, token), token & 15, 1, d >> 2);
        return (d & 2) ? ((d & 1) ? v.w : v.z) : ((d & 1) ? v.y : v.x);
    } else {
        const uint64_t at = (uint64_t)(seg.token_row + token) * a.value_stride + seg.head * kHeadDim + d;
        if constexpr (PARTS == 3) return static_cast<const float *>(a.value)[at];
        if (a.dtype == QWN_DTYPE_F16) return __half2float(static_cast<const __half *>(a.value)[at]);
        return __bfloat162float(static_cast<const __nv_bfloat16 *>(a.value)[at]);
    }
}
// what the noted tokens that a row sees add to its sum in column d
template <int SRC, int PARTS, int BLOCK>
__device__ __noinline__ float odd_sum(const AtArgs &a, const uint32_t (&noted)[2][16], const AtSegment &seg, Seen seen, int d) {
    float sum = 0.f;
#pragma unroll 1
    for (int z = 0; z < 2; z++) {
        const int32_t from = z ? odd_zone(seg, BLOCK) : seg.block0 * BLOCK;
#pragma unroll 1
        for (int w = 0; w < 16; w++)
            for (uint32_t bits = noted[z][w]; bits; bits &= bits - 1) {
                const int32_t token = from + 32 * w + __ffs(bits) - 1;
                if (token < seen.lo || token >= seen.hi) continue;
                const float v = at_value<SRC, PARTS>(a, seg, token, d);
                if (!isfinite(v)) sum += v;
            }
    }
    return sum;
}

// ---- softmax -------------------------------------------------------------------

// P is 2^kBias near the largest score and grows by 2^kSlack at most before M moves:
// f16 holds 2^14 down to 2^-24, so that a probability is lost below 2^-32 of the
// largest; bf16 and fp32 have room.
template <bool BF16>
struct AtRange {
    static constexpr float kBias = BF16 ? 0.f : 8.f, kSlack = BF16 ? 8.f : 6.f;
};

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where either is one
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// 2^t of two values without the special function unit, which does 16 a cycle and
// SM: a block of 256 x 128 scores keeps it as busy as the tensor core.  t = n + f
// with n whole and |f| <= 1/2; 2^f by the polynomial of least relative error on
// that interval (found by exchange; degree 3: 7.5e-5, below bf16's half step of
// 3.9e-3; degree 4: 2.6e-6, below fp16's 4.9e-4), times 2^n put together from its
// exponent, which is zero at -127 and below.
template <bool BF16>
__device__ __forceinline__ uint64_t exp2_pair(uint64_t t) {
    float a, b;
    unpair(t, a, b);
    t = pair(max_nan(a, -127.f), max_nan(b, -127.f));
    constexpr float kWhole = 12582912.f + 127.f;  // 1.5 x 2^23: the sum's low bits are n + 127
    const uint64_t w = add2(t, pair(kWhole, kWhole));
    const uint64_t f = add2(t, mul2(add2(w, pair(-kWhole, -kWhole)), pair(-1.f, -1.f)));
    uint64_t y;
    if constexpr (BF16) {
        y = fma2(f, pair(0.05517166853f, 0.05517166853f), pair(0.2426111251f, 0.2426111251f));
        y = fma2(y, f, pair(0.6932609677f, 0.6932609677f));
        y = fma2(y, f, pair(0.9999280572f, 0.9999280572f));
    } else {
        y = fma2(f, pair(0.009570102207f, 0.009570102207f), pair(0.05591785908f, 0.05591785908f));
        y = fma2(y, f, pair(0.2402474433f, 0.2402474433f));
        y = fma2(y, f, pair(0.6931217909f, 0.6931217909f));
        y = fma2(y, f, pair(0.9999992847f, 0.9999992847f));
    }
    uint32_t n0, n1;
    unpair(w, n0, n1);
    return mul2(y, pair(__uint_as_float(n0 << 23), __uint_as_float(n1 << 23)));
}

// Four 16-byte pieces of each lane's row to memory: the four lanes of a group
// exchange them, so that they write 64 bytes of a row side by side, eight rows to an
// instruction (a lane per row: 32 rows, 7 us a tile).  `row` is where the lane's row
// starts, `have` the lanes that have one.
__device__ __forceinline__ void store_rows(uint8_t *row, uint32_t have, const uint4 (&piece)[4]) {
    const uint32_t lane = threadIdx.x & 31, q = lane & 3;
    uint32_t w[4][4];
#pragma unroll
    for (int k = 0; k < 4; k++) w[k][0] = piece[k].x, w[k][1] = piece[k].y, w[k][2] = piece[k].z, w[k][3] = piece[k].w;
    // a 4 x 4 transposition: pieces (0, 1), (2, 3) with the neighbour, then (0, 2), (1, 3) with the lane two on
#pragma unroll
    for (int s = 1; s <= 2; s <<= 1)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (k & s) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t give = q & s ? w[k][e] : w[k | s][e], got = __shfl_xor_sync(0xffffffffu, give, s);
                if (q & s) w[k][e] = got;
                else w[k | s][e] = got;
            }
        }
#pragma unroll
    for (int k = 0; k < 4; k++) {  // piece q of the group's row k
        const uint32_t from = (lane & ~3u) | k;
        uint8_t *p = reinterpret_cast<uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), from));
        if (have >> from & 1) *reinterpret_cast<uint4 *>(p + 16 * q) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
    }
}
// 16 values of the lane's row as 16-bit pieces 0 and 1, or as fp32 pieces 0 to 3
__device__ __forceinline__ uint4 pack8(const float *v, bool f16) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (f16) {
            w[k] = pack_h2(v[2 * k], v[2 * k + 1]);
        } else {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
            w[k] = *reinterpret_cast<const uint32_t *>(&b);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int SRC, int PARTS, int TILES, bool BF16>
struct AtRoles {
    using S = AtShape<SRC, PARTS, TILES>;
    using Scale = AtScale<SRC>;
    static constexpr bool kTokenScales = S::kTokenScales;
    // the operands' own scaling: of scores and of outputs
    static constexpr float kUnit = PARTS == 1 ? Scale::kFixed : 1.f;
    static constexpr bool kHold = PARTS == 3 || S::kTma;  // a row's scores stay in registers
    static constexpr int kStep = 32;  // columns at a time where they do not
    static constexpr uint32_t kFmaPairs = 0x10;  // of eight pairs of powers, those that FMAs compute
    const AtArgs &a;
    AtShared<SRC, PARTS, TILES> &sh;
    uint32_t q_at, kv_at, raw_at;  // shared memory
    int warp, lane;

    __device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity) const {
        return at_wait(*(volatile int *)&sh.give_up, bar, parity);
    }
    __device__ __forceinline__ uint32_t slot_at(uint32_t slot) const { return kv_at + slot * S::kKvBytes; }

    // the next segment, for a warp that works on all of them
    struct Feed {
        uint32_t n = 0;
    };
    __device__ __forceinline__ bool take(Feed &f, AtSegment &seg) {
        const uint32_t s = f.n & 1;
        if (!wait(&sh.segfull[s], (f.n >> 1) & 1)) return false;
        seg = sh.seg[s];
        warp_arrive(&sh.segempty[s], lane);
        f.n++;
        // the same in all lanes, as the compiler can tell from this
        auto one = [](int32_t &v) { v = __shfl_sync(0xffffffffu, v, 0); };
        one(seg.valid), one(seg.rows), one(seg.seq), one(seg.head), one(seg.len), one(seg.block0), one(seg.blocks);
        one(seg.whole_lo), one(seg.whole_hi), one(seg.slot), one(seg.quarters);
        return seg.valid != 0;
    }

    __device__ __forceinline__ void plan() {
        AtWork<SRC, PARTS, TILES> work(a);
        for (uint32_t n = 0;; n++) {
            const uint32_t s = n & 1;
            const AtSegment seg = work.next();
            if (!wait(&sh.segempty[s], ((n >> 1) & 1) ^ 1)) return;
            if (lane == 0) sh.seg[s] = seg;
            warp_arrive(&sh.segfull[s], lane);
            if (!seg.valid) return;
        }
    }

    __device__ __forceinline__ void load(const CUtensorMap *kmap, const CUtensorMap *vmap) {
        Feed f;
        AtSegment seg;
        uint32_t done = 0;  // blocks, or cached tiles
        uint32_t phase[2] = {}, issued[2] = {};  // a bit per slot: of full and part, the phase that the next copy fills
        bool ok = true;
        while (ok && take(f, seg)) {
            if constexpr (S::kTma) {
                for (int b = 0; b < seg.blocks && ok; b++, done++) {
                    const int y = (int)seg.token_row + (seg.block0 + b) * S::kBlock, x = seg.head * kHeadDim;
                    auto fetch = [&](uint64_t *full, uint32_t slot, uint32_t turn, const CUtensorMap *map) {
                        if (!wait(&sh.empty[slot], (turn & 1) ^ 1)) return false;
                        if (lane == 0) {
                            mbar_expect_tx(&full[slot], S::kKvBytes);
                            tma_load(slot_at(slot), map, x, y, smem_u32(&full[slot]));
                            tma_load(slot_at(slot) + S::kBlock * 128, map, x + 64, y, smem_u32(&full[slot]));
                        }
                        __syncwarp();
                        const uint32_t kind = full == sh.part;
                        phase[kind] ^= 1u << slot;
                        issued[kind] |= 1u << slot;
                        return true;
                    };
                    ok = fetch(sh.full, S::k_slot(done), S::k_turn(done), kmap) &&
                         fetch(whole(seg, seg.block0 + b) ? sh.full : sh.part, S::v_slot(done), S::v_turn(done), vmap);
                }
            } else if constexpr (S::kRaw) {
                // A lane has a tile of each block, or its K or V.  The page is looked up two blocks ahead, and nothing asks for it before
                // its turn; lanes issue as their slots become free.
                const bool tiles = lane < S::kSides * S::kTiles;
                const uint32_t side = lane / S::kTiles, mine = lane % S::kTiles;
                auto page_of = [&](int b) {
                    const int32_t token = (seg.block0 + b) * S::kBlock + mine * kTileTokens;
                    return tiles && b < seg.blocks && token < seg.len ? at_page(a, seg.seq, token) : -1;
                };
                int32_t ahead[2] = {page_of(0), page_of(1)};
                for (int b = 0; b < seg.blocks && ok; b++, done += S::kTiles) {
                    const int32_t token = (seg.block0 + b) * S::kBlock + mine * kTileTokens, page = ahead[0];
                    ahead[0] = ahead[1];
                    ahead[1] = page_of(b + 2);
                    const bool have = tiles && token < seg.len;
                    const uint32_t g = done + mine, s = g % S::kRawTiles, parity = ((g / S::kRawTiles) & 1) ^ 1;
                    const uint32_t bar = s + (S::kSides == 2 ? side * S::kRawV : 0);
                    auto copy = [&](const uint8_t *from, uint32_t at, uint32_t bytes) {
                        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
                                         "r"(raw_at + s * S::kTileBytes + at),
                                     "l"(from + at), "r"(bytes), "r"(smem_u32(&sh.rawfull[bar]))
                                     : "memory");
                    };
                    bool waits = tiles;
                    for (uint32_t it = 0;; ++it) {
                        if (waits && mbar_try_wait(&sh.rawempty[bar], parity)) {
                            waits = false;
                            if (have) {
                                const uint8_t *from = at_tile_in(a, page, seg.head, token);
                                mbar_expect_tx(&sh.rawfull[bar], S::kTileBytes / S::kSides);
                                if constexpr (S::kSides == 1) {
                                    copy(from, 0, S::kTileBytes);
                                } else {
                                    copy(from, side * S::kCodeBytes, S::kCodeBytes);
                                    if (S::kRestBytes) copy(from, 2 * S::kCodeBytes + side * S::kRestBytes, S::kRestBytes);
                                }
                            } else {
                                mbar_arrive(&sh.rawfull[bar]);
                            }
                        }
                        if (!__any_sync(0xffffffffu, waits)) break;
                        if (it >= kWaitLimit || ((it & 63) == 63 && *(volatile int *)&sh.give_up)) {
                            issued[0] = __ballot_sync(0xffffffffu, tiles && !waits);  // of this block
                            *(volatile int *)&sh.give_up = 1;
                            ok = false;
                            break;
                        }
                    }
                    ok = __all_sync(0xffffffffu, ok);
                }
            }
        }
        // copies in flight end before the CTA's memory goes, whoever gave up
        if constexpr (S::kTma) {
            for (uint32_t v = 0; v < S::kRing; v++) {
                if (issued[0] >> v & 1) mbar_wait_bounded(&sh.full[v], (phase[0] >> v & 1) ^ 1);
                if (issued[1] >> v & 1) mbar_wait_bounded(&sh.part[v], (phase[1] >> v & 1) ^ 1);
            }
        } else if constexpr (S::kRaw) {
            for (uint32_t side = 0; side < S::kSides; side++) {
                uint64_t *full = sh.rawfull + side * S::kRawV;
                const uint32_t gone = issued[0] >> (side * S::kTiles);
                for (uint32_t d = done > S::kRawTiles ? done - S::kRawTiles : 0; d < done; d++) {
                    // (after giving up, the slots that its block has filled already are a turn further)
                    const uint32_t s = d % S::kRawTiles, t = (s + S::kRawTiles - done % S::kRawTiles) % S::kRawTiles;
                    if (!ok || t >= S::kTiles || !(gone >> t & 1)) mbar_wait_bounded(&full[s], (d / S::kRawTiles) & 1);
                }
                for (uint32_t t = 0; t < S::kTiles; t++)
                    if (gone >> t & 1)
                        mbar_wait_bounded(&full[(done + t) % S::kRawTiles], ((done + t) / S::kRawTiles) & 1);
            }
        }
    }

    __device__ __forceinline__ static bool whole(const AtSegment &seg, int blk) { return blk >= seg.whole_lo && blk < seg.whole_hi; }

    // the helpers' four warps meet; a wait like the others, so that it ends when one of them has given up
    __device__ __forceinline__ bool helpers_sync(uint32_t &syncs) {
        warp_arrive(&sh.helped, lane);
        return wait(&sh.helped, syncs++ & 1);
    }
    // Operands out of cached tiles, and out of fp32 rows: four warps make K, four make V, so that the next blocks'
    // scores do not wait for the room of this one's values.  A tile of codes is in its warp's registers before its
    // room is given back.  fp16 tiles go as they are, in asynchronous copies of 16 bytes (their chunks are swizzled as the operands'
    // are); a block's are on their way while the next block's start.
    // The scales of a tile's tokens, which are read when the block's scores are there.
    __device__ __forceinline__ void put_scales(const uint8_t *tile, int ti, int32_t token0, int32_t len, uint32_t d) {
        const int t = lane & 15, v = lane >> 4;
        const float sc = token0 + ti * kTileTokens + t < len ? token_scale<SRC>(tile, t, v) : 0.f;
        (v ? sh.vscale : sh.kscale)[d & 3][ti * kTileTokens + (S::kByDims ? cached_order(t) : t)] = sc;
        const uint32_t top = __reduce_max_sync(0xffffffffu, v ? __float_as_uint(sc) : 0u);
        if (lane == 0) sh.vtop[d & 3][ti] = (float)((int)(top >> 23) - 126);
    }
    __device__ __forceinline__ bool convert_side(const AtSegment &seg, uint32_t done, uint32_t segment, uint32_t &meetings) {
        const int w = warp & 3;
        const int which = (warp - 8) >> 2;  // K or V
        auto slot_of = [&](uint32_t d) { return which ? S::v_slot(d) : S::k_slot(d); };
        auto free_slot = [&](uint32_t d) { return wait(&sh.empty[slot_of(d)], ((which ? S::v_turn(d) : S::k_turn(d)) & 1) ^ 1); };
        auto ready = [&](uint32_t d, int blk) {  // the block's operands are written
            if (which && !whole(seg, blk) && !(PARTS == 3 && S::kKvParts == 1)) {  // (codes are finite)
                warp_arrive(&sh.cleared, lane);
                if (!wait(&sh.cleared, meetings++ & 1)) return false;
                if constexpr (S::kByDims) clear_odd_by_dims(sh.odd_v[segment & 3], seg, blk * S::kBlock, slot_at(slot_of(d)));
                else clear_odd<S::kKvParts, S::kBlock>(sh.odd_v[segment & 3], seg, blk * S::kBlock, slot_at(slot_of(d)), PARTS == 3);
            }
            fence_proxy_async_shared();
            warp_arrive(&sh.full[slot_of(d)], lane);
            return true;
        };
        // Cached tiles' room for the next copies.  They write through the async proxy: without the fence they were
        // seen to overtake loads whose warp had arrived.
        auto give_back = [&](const auto &ring) {
            fence_proxy_async_shared();
            for (const uint32_t r : ring) warp_arrive(&sh.rawempty[r], lane);
        };
        if constexpr (S::kByDims) {
            extern __shared__ uint8_t dynamic[];
            constexpr int kEach = S::kTiles / 4;  // tiles of a warp
            for (int b = 0; b < seg.blocks; b++) {
                const uint32_t d = done + b, dst = slot_at(slot_of(d));
                const int32_t token0 = (seg.block0 + b) * S::kBlock;
                uint32_t ring[kEach];
                const uint8_t *tile[kEach];
#pragma unroll
                for (int i = 0; i < kEach; i++) {
                    const uint32_t g = d * S::kTiles + w + 4 * i;
                    ring[i] = g % S::kRawTiles;
                    tile[i] = dynamic + (raw_at - smem_u32(dynamic)) + ring[i] * S::kTileBytes;
                    if (!wait(&sh.rawfull[ring[i]], (g / S::kRawTiles) & 1)) return false;
                }
                if (which) {
                    ValueWords<SRC, PARTS == 3> v[kEach];
#pragma unroll
                    for (int i = 0; i < kEach; i++) v[i].load(tile[i]);
                    give_back(ring);
                    if (!free_slot(d)) return false;
#pragma unroll
                    for (int i = 0; i < kEach; i++) v[i].store(w + 4 * i, dst);
                } else {
                    KeyWords<SRC, PARTS == 3> k[kEach];
#pragma unroll
                    for (int i = 0; i < kEach; i++) k[i].load(tile[i]);
                    if (!free_slot(d)) return false;
                    if constexpr (kTokenScales) {
#pragma unroll
                        for (int i = 0; i < kEach; i++) put_scales(tile[i], w + 4 * i, token0, seg.len, d);
                    }
#pragma unroll
                    for (int i = 0; i < kEach; i++) k[i].template store<S::kBlock>(tile[i], w + 4 * i, dst);
                    give_back(ring);
                }
                if (!ready(d, seg.block0 + b)) return false;
            }
            return true;
        } else if constexpr (PARTS == 1) {
            auto address = [&](int b, int ti) -> const uint8_t * {
                const int32_t token = (seg.block0 + b) * S::kBlock + ti * kTileTokens;
                return b < seg.blocks && token < seg.len ? at_tile(a, seg.seq, seg.head, token) : nullptr;
            };
            const uint8_t *ahead[2] = {address(0, w), address(0, w + 4)};
            for (int b = 0; b < seg.blocks; b++) {
                if (!free_slot(done + b)) return false;
                const uint32_t dst = slot_at(slot_of(done + b));
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint8_t *tile = ahead[i];
                    ahead[i] = address(b + 1, w + 4 * i);
                    if (tile) {
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const int n = 32 * k + lane, t = n >> 4, c = n & 15;
                            cp_async16_at(dst + (c >> 3) * S::kBlock * 128 + ((w + 4 * i) * kTileTokens + t) * 128 + (c & 7) * 16,
                                          tile + which * 4096 + 16 * n);
                        }
                    }
                }
                cp_async_commit();
                if (b) {
                    cp_async_wait1();
                    if (!ready(done + b - 1, seg.block0 + b - 1)) return false;
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            return ready(done + seg.blocks - 1, seg.block0 + seg.blocks - 1);
        } else {
            // A warp has a tile of each block, a lane 16 dims of four of its rows.  Rows that no copy brings are read
            // ahead, two at least while the warp waits for the operands' room.
            using Value = std::conditional_t<S::kPaged, __half, float>;
            constexpr int kAhead = S::kPaged ? 4 : 2;
            // Half of them are in parts by then too (8192 fp32 rows 3200 -> 3020 us, 33 rows over 131105 4-bit tokens
            // 1239 -> 1180); not int8 codes, whose gathered bytes hold the next copy up (1116 -> 1160).
            constexpr int kEarly = SRC == QWN_KV_CODEC_Q8_B64_F32 ? 0 : 2;
            Raw16<Value> ahead[S::kRaw ? 1 : kAhead];
            const uint8_t *page = nullptr;  // of the next block's tile
            auto first = [&](int b) { return (seg.block0 + b) * S::kBlock + w * kTileTokens; };
            auto look = [&](int b) {
                if constexpr (S::kPaged)
                    page = b < seg.blocks && first(b) < seg.len ? at_tile(a, seg.seq, seg.head, first(b)) : nullptr;
            };
            auto fetch = [&](int b, int pass) {
                Raw16<Value> &to = ahead[pass % kAhead];
                const int t = 4 * pass + (lane >> 3);
                to = Raw16<Value>{};
                if (b >= seg.blocks || first(b) + t >= seg.len) return;
                if constexpr (S::kPaged) {
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        to.w[h] = *reinterpret_cast<const uint4 *>(page + f16_off(which, t, 64 * h + 8 * (lane & 7)));
                } else {
                    const float *rows = static_cast<const float *>(which ? a.value : a.key) + (size_t)seg.head * kHeadDim;
                    to.load(rows + (uint64_t)(seg.token_row + first(b) + t) * (which ? a.value_stride : a.key_stride), lane & 7);
                }
            };
            if constexpr (!S::kRaw) {
                look(0);
#pragma unroll
                for (int pass = 0; pass < kAhead; pass++) fetch(0, pass);
                look(1);
            }
            for (int b = 0; b < seg.blocks; b++) {
                const uint32_t d = done + b, dst = slot_at(slot_of(d));
                RowParts<S::kKvParts> part[kEarly ? kEarly : 1];
                auto put = [&](int pass, const RowParts<S::kKvParts> &x) {
                    x.put(dst, S::kBlock, (uint32_t)(w * kTileTokens + 4 * pass + (lane >> 3)), lane & 7);
                };
                if constexpr (S::kRaw) {
                    extern __shared__ uint8_t dynamic[];
                    const uint32_t g = d * S::kTiles + w, r = g % S::kRawTiles;
                    const uint32_t ring[1] = {r + which * S::kRawV};
                    const uint8_t *tile = dynamic + (raw_at - smem_u32(dynamic)) + r * S::kTileBytes;
                    auto row = [&](int pass) {
                        const int t = 4 * pass + (lane >> 3);
                        Row16 x = {};
                        if (first(b) + t < seg.len) x = take_row<SRC>(tile, t, which, lane & 7);
                        return x;
                    };
                    if (!wait(&sh.rawfull[ring[0]], (g / S::kRawTiles) & 1)) return false;
#pragma unroll
                    for (int pass = 0; pass < kEarly; pass++) part[pass].set(row(pass));
                    if (!free_slot(d)) return false;
#pragma unroll
                    for (int pass = 0; pass < 4; pass++) {
                        if (pass >= kEarly) part[0].set(row(pass));
                        put(pass, part[pass < kEarly ? pass : 0]);
                    }
                    give_back(ring);
                } else {
#pragma unroll
                    for (int pass = 0; pass < kEarly; pass++) {
                        part[pass].set(ahead[pass % kAhead].row());
                        fetch(b + (pass + kAhead) / 4, (pass + kAhead) % 4);
                    }
                    if (!free_slot(d)) return false;
#pragma unroll
                    for (int pass = 0; pass < 4; pass++) {
                        if (pass >= kEarly) {
                            part[0].set(ahead[pass % kAhead].row());
                            fetch(b + (pass + kAhead) / 4, (pass + kAhead) % 4);
                        }
                        put(pass, part[pass < kEarly ? pass : 0]);
                    }
                    look(b + 2);
                }
                if (!ready(d, seg.block0 + b)) return false;
            }
            return true;
        }
    }

    __device__ __forceinline__ void help() {
        Feed f;
        AtSegment seg;
        uint32_t done = 0, used = 0, syncs = 0;  // blocks, segments with any
        uint32_t phase = 0, meetings = 0;  // of part, a bit per slot; of the warps that make V
        const uint32_t tid = threadIdx.x & 127, wg = (warp - 8) >> 2;
        while (take(f, seg)) {
            if (seg.blocks == 0) continue;
            if (!wait(&sh.qempty, (used & 1) ^ 1)) return;
            if (wg == 0 && tid < 32) sh.odd_v[used & 3][tid >> 4][tid & 15] = 0;
#pragma unroll 1
            for (int t = wg; t < TILES; t += S::kHelpers / 4) put_q<SRC, PARTS>(a, seg, t * kAtRows, q_at + t * S::kQBytes, sh.qscale[used & 1]);
            if constexpr (S::kTma) asm volatile("cp.async.wait_all;" ::: "memory");
            fence_proxy_async_shared();
            if (!helpers_sync(syncs)) return;  // odd_v is empty before any warp notes a token
            warp_arrive(&sh.qfull, lane);
            if constexpr (!S::kTma) {
                if (!convert_side(seg, done, used, meetings)) return;
            } else {
                for (int b = 0; b < seg.blocks; b++) {
                    const int blk = seg.block0 + b;
                    if (whole(seg, blk)) continue;
                    const uint32_t s = S::v_slot(done + b);
                    if (!wait(&sh.part[s], phase >> s & 1)) return;
                    phase ^= 1u << s;
                    clear_odd<S::kKvParts, S::kBlock>(sh.odd_v[used & 3], seg, blk * S::kBlock, slot_at(s), BF16);
                    fence_proxy_async_shared();
                    warp_arrive(&sh.fixed[s], lane);
                }
            }
            done += seg.blocks;
            used++;
        }
    }

    // one warp; its elected lane issues
    __device__ __forceinline__ void multiply() {
        Feed f;
        AtSegment seg;
        const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
        const bool leader = elect_one();
        uint32_t done = 0, used = 0, o_uses[2] = {0, 0}, p_uses[2] = {0, 0};
        uint32_t phase[2] = {};  // loaded operands: of full and fixed, a bit per slot
        constexpr uint32_t kQk = f16_desc(BF16 || PARTS == 3, S::kBlock, false), kPv = f16_desc(BF16 || PARTS == 3, 128, !S::kByDims);
        // the products of parts that count, the small ones first
        constexpr int kPairs = PARTS == 1 ? 1 : 6;
        constexpr int kFirst[6] = {PARTS == 1 ? 0 : 2, 0, 1, 1, 0, 0}, kSecond[6] = {0, 2, 1, 0, 1, 0};
        auto scores = [&](int t, uint32_t slot) {  // S_t = Q K^T
            const uint32_t q = q_at + (TILES == 2 ? t * S::kQBytes : 0), k = slot_at(slot);
#pragma unroll
            for (int p = 0; p < kPairs; p++) {
                if (kSecond[p] >= S::kKvParts) continue;
                const uint64_t qd = smem_desc(q + kFirst[p] * kAtRows * 256), kd = smem_desc(k + kSecond[p] * S::kKvPart);
                if (leader)
#pragma unroll
                    for (int c = 0; c < 8; c++)
                        mma_ss(tmem + t * S::kSColumns, qd + (c >> 2) * (kAtRows * 128 / 16) + (c & 3) * 2,
                               kd + (c >> 2) * (S::kBlock * 128 / 16) + (c & 3) * 2, kQk, p + c > 0);
            }
        };
        // O_t += P_t V for half the tokens (16-bit operands, so that the products start while the other half's
        // powers are computed) or all
        constexpr int kHalves = PARTS == 1 ? 2 : 1, kSteps = S::kBlock / 16 / kHalves;
        auto values = [&](int t, uint32_t slot, bool add, int half) {
            const uint32_t v = slot_at(slot);
#pragma unroll
            for (int p = 0; p < kPairs; p++) {
                if (kSecond[p] >= S::kKvParts) continue;
                const uint64_t vd = S::kByDims ? smem_desc(v) : rows_desc(v + kSecond[p] * S::kKvPart, S::kBlock * 128);
                if (leader)
#pragma unroll
                    for (int c = half * kSteps; c < (half + 1) * kSteps; c++)
                        mma_ts(tmem + S::kOColumn + t * 128, tmem + t * S::kSColumns + kFirst[p] * (S::kBlock / 2) + c * 8,
                               vd + (S::kByDims ? (c >> 2) * (16384 / 16) + (c & 3) * 2 : c * (2048 / 16)), kPv, add || p + c > 0);
            }
        };
        auto commit = [&](uint64_t *bar) {
            if (leader) mma_commit(bar);
        };
        auto wait_k = [&](uint32_t d) {
            const uint32_t s = S::k_slot(d);
            if constexpr (S::kTma) {
                const bool ok = wait(&sh.full[s], phase[0] >> s & 1);
                phase[0] ^= 1u << s;
                return ok;
            }
            return wait(&sh.full[s], S::k_turn(d) & 1);
        };
        auto wait_v = [&](uint32_t d, bool all) {
            const uint32_t s = S::v_slot(d);
            if constexpr (S::kTma) {
                const bool ok = wait(all ? &sh.full[s] : &sh.fixed[s], phase[all ? 0 : 1] >> s & 1);
                phase[all ? 0 : 1] ^= 1u << s;
                return ok;
            }
            return wait(&sh.full[s], S::v_turn(d) & 1);
        };
        bool ok = true;
        while (ok && take(f, seg)) {
            const int nb = seg.blocks;
            if (nb == 0) continue;
            ok = wait(&sh.qfull, used & 1);
            // block b's scores for group t, and what becomes free behind them
            auto do_scores = [&](int b, int t) {
                if (TILES == 1 || t == 0) ok = ok && wait_k(done + b);
                if (!ok) return;
                tc_fence_after();
                scores(t, S::k_slot(done + b));
                commit(&sh.sfull[t]);
                if (TILES == 1 || t == 1) {
                    commit(&sh.empty[S::k_slot(done + b)]);
                    if (b == nb - 1) commit(&sh.qempty);
                }
            };
            for (int t = 0; t < 2; t++)
                if (TILES == 2) do_scores(0, t);
                else if (t < nb) do_scores(t, t);
            for (int b = 0; b < nb && ok; b++) {
                const uint32_t vs = S::v_slot(done + b);
                ok = wait_v(done + b, whole(seg, seg.block0 + b));
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    if (TILES == 1 && t != (b & 1)) continue;
                    const bool first = TILES == 2 ? b == 0 : b < 2;
                    if (first) ok = ok && wait(&sh.oempty[t], (o_uses[t]++ & 1) ^ 1);
#pragma unroll
                    for (int half = 0; half < kHalves; half++) {
                        ok = ok && wait(&sh.pready[t][half], p_uses[t] & 1);
                        if (!ok) break;
                        tc_fence_after();
                        values(t, vs, !first, half);
                    }
                    p_uses[t]++;
                    if (!ok) break;
                    if (TILES == 1 || t == 1) commit(&sh.empty[vs]);
                    const int nextb = b + (TILES == 2 ? 1 : 2);
                    if (nextb < nb) do_scores(nextb, t);
                    else commit(&sh.ofull[t]);
                }
            }
            done += nb;
            used++;
        }
        if (*(volatile int *)&sh.give_up) {  // products in flight end before the CTA's memory goes
            commit(&sh.drained);
            mbar_wait_bounded(&sh.drained, 0);
        }
    }

    __device__ __forceinline__ void soften() {
        Feed f;
        AtSegment seg;
        const int g = warp >> 2, w = warp & 3;
        const uint32_t lanes = sh.tmem + ((uint32_t)(w * 32) << 16);
        const uint32_t s_col = lanes + g * S::kSColumns, o_col = lanes + S::kOColumn + g * 128;
        uint32_t done = 0, used = 0, s_uses = 0, o_uses[2] = {0, 0}, joins = 0;
        const uint32_t r = (TILES == 2 ? g * kAtRows : 0) + w * 32 + lane;
        while (take(f, seg)) {
            const bool quarters = S::kQuarters && seg.quarters;
            const uint32_t mine = quarters ? lane : r;  // of the segment's rows
            const bool have = (int32_t)mine < seg.rows, any = quarters || (int32_t)(r - lane) < seg.rows;
            const int64_t pos = seg.pos0 + (have ? (seg.row0 + mine) / a.group : 0);
            const Seen seen = have ? at_seen(a, pos, seg.len) : Seen{0, 0};
            if (have && S::kPaged && (pos < 0 || pos >= seg.len))
                latch(a.status, seg.seq < 0 ? QWN_KV_STATUS_BAD_SEQUENCE : QWN_KV_STATUS_BAD_LENGTH);
            float M = -INFINITY, l = 0.f, c = 0.f;
            for (int b = TILES == 2 ? 0 : g; b < seg.blocks; b += TILES == 2 ? 1 : 2) {
                if (!wait(&sh.sfull[g], s_uses++ & 1)) return;
                tc_fence_after();
                if (!any) {
                    if (PARTS == 1) warp_arrive(&sh.pready[g][0], lane);
                } else {
                    const bool first = b < (TILES == 2 ? 1 : 2);
                    if (first) c = a.scale2 * kUnit * (SRC != 0 && PARTS == 1 && have ? sh.qscale[used & 1][r] : 1.f);
                    if (S::kQuarters && quarters) quarter(seg, seg.block0 + b, (done + b) & 3, first, have, seen, c, s_col, o_col, M, l);
                    else block(seg, seg.block0 + b, (done + b) & 3, first, have, seen, c, s_col, o_col, M, l);
                }
                tc_fence_before();
                warp_arrive(&sh.pready[g][PARTS == 1 ? 1 : 0], lane);
            }
            if (seen.lo >= seen.hi) {  // a row that does not exist: blocks seen whole by the others are no business of its
                M = -INFINITY;
                l = 0.f;
            }
            if (!finish(seg, used, have, any, r, mine, seen, g, lanes, M, l, o_uses, joins)) return;
            done += seg.blocks;
            if (seg.blocks) used++;
        }
    }

    // a block's scores to probabilities; M, l and, where M moves, the sums so far
    __device__ __forceinline__ void block(const AtSegment &seg, int blk, uint32_t slot, bool first, bool have, const Seen &seen,
                                          float c, uint32_t s_col, uint32_t o_col, float &M, float &l) {
        constexpr int N = S::kBlock;
        using Range = AtRange<BF16 || PARTS == 3>;
        const bool full = whole(seg, blk);
        const int lo = seen.lo - blk * S::kBlock, hi = seen.hi - blk * S::kBlock;
        float vtop = 0.f;
        if constexpr (kTokenScales) {
            const float4 v0 = *reinterpret_cast<const float4 *>(&sh.vtop[slot][0]);
            const float4 v1 = *reinterpret_cast<const float4 *>(&sh.vtop[slot][N == 128 ? 4 : 0]);
            vtop = fmaxf(fmaxf(fmaxf(v0.x, v0.y), fmaxf(v0.z, v0.w)), fmaxf(fmaxf(v1.x, v1.y), fmaxf(v1.z, v1.w)));
        }
        float t[8];
        uint32_t held[kHold ? N : 1];
        const float *x = reinterpret_cast<const float *>(held);
        if constexpr (kHold) {
            if constexpr (N == 128) tmem_load128(held, s_col);
            else tmem_load64(held, s_col);
            if constexpr (kTokenScales) {
                float *y = reinterpret_cast<float *>(held);
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(&sh.kscale[slot][i]);
                    unpair(mul2(pair(y[i], y[i + 1]), pair(f.x, f.y)), y[i], y[i + 1]);
                    unpair(mul2(pair(y[i + 2], y[i + 3]), pair(f.z, f.w)), y[i + 2], y[i + 3]);
                }
            }
            if (!full) hide(held, lo, hi);
#pragma unroll
            for (int i = 0; i < 8; i++) t[i] = x[i];
#pragma unroll
            for (int i = 8; i < N; i += 8)
#pragma unroll
                for (int k = 0; k < 8; k++) t[k] = fmaxf(t[k], x[i + k]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) t[k] = -INFINITY;
#pragma unroll 1
            for (int i = 0; i < N; i += kStep) {
                uint32_t u[kStep];
                tmem_load_step(u, s_col + i);
                adjust(u, i, slot, full, lo, hi);
#pragma unroll
                for (int k = 0; k < kStep; k++) t[k & 7] = fmaxf(t[k & 7], __uint_as_float(u[k]));
            }
        }
        const float top = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
        const float reach = top * c + vtop;
        follow<Range>(reach, first, have, o_col, M, l);
        const float off = Range::kBias - (M == -INFINITY ? 0.f : M);
        // P follows on S's columns, half as many (three parts: all of them).  Masked scores are -inf, whose power is
        // exactly zero in the special function unit only.
        if constexpr (kHold) {
            if (PARTS == 1 && full) l += powers<true, N>(held, 0, slot, c, off, s_col);
            else l += powers<false, N>(held, 0, slot, c, off, s_col);
        } else {
#pragma unroll 1
            for (int i = 0; i < N; i += kStep) {
                uint32_t u[kStep];
                tmem_load_step(u, s_col + i);
                adjust(u, i, slot, full, lo, hi);
                if (full) l += powers<true, kStep>(u, i, slot, c, off, s_col);
                else l += powers<false, kStep>(u, i, slot, c, off, s_col);
            }
        }
        tmem_store_wait();
    }

    // M to `reach` where that is far beyond it, and the row's sums with it
    template <class Range>
    __device__ __forceinline__ void follow(float reach, bool first, bool have, uint32_t o_col, float &M, float &l) {
        const bool grows = have && reach > M + Range::kSlack;  // true for the first that is not -inf
        if (__any_sync(0xffffffffu, grows)) {
            const float factor = grows && M != -INFINITY ? ex2(M - reach) : 1.f;
            if (grows) {
                l *= factor;
                M = reach;
            }
            if (!first) {
#pragma unroll 1
                for (int i = 0; i < 128; i += 16) {
                    uint32_t o[16];
                    tmem_load16(o, o_col + i);
#pragma unroll
                    for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * factor);
                    tmem_store16(o_col + i, o);
                }
            }
        }
    }
    // The quarter of a block's tokens that is this warp's, for its copy of the rows.
    __device__ __forceinline__ void quarter(const AtSegment &seg, int blk, uint32_t slot, bool first, bool have, const Seen &seen,
                                            float c, uint32_t s_col, uint32_t o_col, float &M, float &l) {
        using Range = AtRange<BF16>;
        const bool full = whole(seg, blk);
        const int lo = seen.lo - blk * S::kBlock, hi = seen.hi - blk * S::kBlock, at = 32 * (warp & 3);
        float vtop = 0.f;
        if constexpr (kTokenScales) {  // of the two cached tiles
            const float2 v = *reinterpret_cast<const float2 *>(&sh.vtop[slot][2 * (warp & 3)]);
            vtop = fmaxf(v.x, v.y);
        }
        uint32_t u[32];
        tmem_load32(u, s_col + at);
        adjust(u, at, slot, full, lo, hi);
        float t[8];
#pragma unroll
        for (int k = 0; k < 8; k++) t[k] = __uint_as_float(u[k]);
#pragma unroll
        for (int k = 8; k < 32; k++) t[k & 7] = fmaxf(t[k & 7], __uint_as_float(u[k]));
        const float top = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
        follow<Range>(top * c + vtop, first, have, o_col, M, l);
        const float off = Range::kBias - (M == -INFINITY ? 0.f : M);
        const uint32_t none[16] = {};
#pragma unroll
        for (int q = 0; q < 4; q++)
            if (q != (warp & 3)) tmem_store16(s_col + 16 * q, none);
        l += powers<false, 32, false>(u, at, slot, c, off, s_col);
        tmem_store_wait();
        tc_fence_before();
        warp_arrive(&sh.pready[warp >> 2][0], lane);
    }
    // -inf where a row does not see the token of a column
    template <int N>
    __device__ __forceinline__ void hide(uint32_t (&u)[N], int lo, int hi) const {
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int t = S::kByDims ? cached_token(k) : k;
            if (t < lo || t >= hi) u[k] = 0xFF800000u;
        }
    }
    // 32 columns of scores from column i on: times the tokens' scales, -inf where a row does not see the token
    static __device__ __forceinline__ void tmem_load_step(uint32_t (&u)[kStep], uint32_t addr) {
        if constexpr (kStep == 64) tmem_load64(u, addr);
        else tmem_load32(*reinterpret_cast<uint32_t (*)[32]>(u), addr);
    }
    template <int N>
    __device__ __forceinline__ void adjust(uint32_t (&u)[N], int i, uint32_t slot, bool full, int lo, int hi) {
        float *x = reinterpret_cast<float *>(u);
        if constexpr (kTokenScales) {
#pragma unroll
            for (int k = 0; k < N; k += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(&sh.kscale[slot][i + k]);
                unpair(mul2(pair(x[k], x[k + 1]), pair(f.x, f.y)), x[k], x[k + 1]);
                unpair(mul2(pair(x[k + 2], x[k + 3]), pair(f.z, f.w)), x[k + 2], x[k + 3]);
            }
        }
        if (!full) hide(u, lo - i, hi - i);
    }
    // P = 2^(c x + off) of N columns from column at0 on into tensor memory; returns their sum.  With MIXED some pairs
    // of eight are computed by FMAs.
    template <bool MIXED, int N, bool HALVES = true>
    __device__ __forceinline__ float powers(const uint32_t (&u)[N], int at0, uint32_t slot, float c, float off, uint32_t s_col) {
        const float *x = reinterpret_cast<const float *>(u);
        const uint64_t cc = pair(c, c), oo = pair(off, off);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < N; i += 32) {
            uint32_t p[PARTS][16];
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
                uint64_t t = fma2(pair(x[i + k], x[i + k + 1]), cc, oo);
                if constexpr (PARTS == 3) t = fma2(pair(x[i + k], x[i + k + 1]), pair(a.scale2_low, a.scale2_low), t);
                uint64_t e;
                if (MIXED && (kFmaPairs >> ((k >> 1) & 7) & 1)) {
                    e = exp2_pair<BF16>(t);
                } else {
                    float t0, t1;
                    unpair(t, t0, t1);
                    e = pair(ex2(t0), ex2(t1));
                }
                sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], e);
                float e0, e1;
                if constexpr (kTokenScales) {
                    const float2 v = *reinterpret_cast<const float2 *>(&sh.vscale[slot][at0 + i + k]);
                    e = mul2(e, pair(v.x, v.y));
                }
                unpair(e, e0, e1);
                if constexpr (PARTS == 3) {
                    const uint32_t a0 = __float_as_uint(e0), a1 = __float_as_uint(e1);
                    const float f0 = e0 - __uint_as_float(a0 & 0xFFFF0000u), f1 = e1 - __uint_as_float(a1 & 0xFFFF0000u);
                    const uint32_t b0 = __float_as_uint(f0), b1 = __float_as_uint(f1);
                    const float g0 = f0 - __uint_as_float(b0 & 0xFFFF0000u), g1 = f1 - __uint_as_float(b1 & 0xFFFF0000u);
                    p[0][k >> 1] = prmt(a0, a1, 0x7632u);
                    p[1][k >> 1] = prmt(b0, b1, 0x7632u);
                    p[2][k >> 1] = prmt(__float_as_uint(g0), __float_as_uint(g1), 0x7632u);
                } else if constexpr (BF16) {
                    const __nv_bfloat162 v = __floats2bfloat162_rn(e0, e1);
                    p[0][k >> 1] = *reinterpret_cast<const uint32_t *>(&v);
                } else {
                    p[0][k >> 1] = pack_h2(e0, e1);
                }
            }
#pragma unroll
            for (int k = 0; k < PARTS; k++) tmem_store16(s_col + k * (S::kBlock / 2) + (at0 + i) / 2, p[k]);
            if (HALVES && PARTS == 1 && at0 + i == S::kBlock / 2 - 32) {  // the products of half the tokens may start
                tmem_store_wait();
                tc_fence_before();
                warp_arrive(&sh.pready[warp >> 2][0], lane);
            }
        }
        float l[4];
        unpair(sum[0], l[0], l[1]);
        unpair(sum[1], l[2], l[3]);
        return (l[0] + l[1]) + (l[2] + l[3]);
    }

    // the rows of a segment: to the output, or to the workspace where other CTAs have a share of them
    __device__ __forceinline__ bool finish(const AtSegment &seg, uint32_t used, bool have, bool any, uint32_t r, uint32_t mine, const Seen &seen,
                                           int g, uint32_t lanes, float M, float l, uint32_t (&o_uses)[2], uint32_t &joins) {
        constexpr int kWide = 16;  // columns at a time
        const uint32_t o_at = lanes + S::kOColumn;
        float w0 = 1.f, w1 = 0.f;
        const bool two = TILES == 1 && seg.blocks > 1;
        if (TILES == 1) {  // both groups' rows are the same ones: each group finishes half of the columns
            const uint32_t row = r, turn = joins & 1;
            sh.ml[turn][g][row][0] = M;
            sh.ml[turn][g][row][1] = l;
            warp_arrive(&sh.joined, lane);
            if (!wait(&sh.joined, joins & 1)) return false;
            joins++;
            const float M0 = sh.ml[turn][0][row][0], M1 = sh.ml[turn][1][row][0];
            M = fmaxf(M0, M1);
            w0 = M0 == -INFINITY ? 0.f : ex2(M0 - M);
            w1 = M1 == -INFINITY ? 0.f : ex2(M1 - M);
            l = w0 * sh.ml[turn][0][row][1] + w1 * sh.ml[turn][1][row][1];
        }
        if (seg.blocks) {
            if (TILES == 2) {
                if (!wait(&sh.ofull[g], o_uses[0]++ & 1)) return false;
            } else {
                if (!wait(&sh.ofull[0], o_uses[0]++ & 1)) return false;
                if (two && !wait(&sh.ofull[1], o_uses[1]++ & 1)) return false;
            }
            tc_fence_after();
        }
        if (any) {
            uint32_t odd = 0;
            if (seg.blocks) {
                for (int z = 0; z < 2; z++) odd |= sh.odd_v[used & 3][z][lane & 15];
                odd = __any_sync(0xffffffffu, odd != 0);
            }
            const uint32_t row = seg.row0 + (have ? mine : 0), token = row / a.group, h = seg.head * a.group + row - token * a.group;
            const uint64_t at = (uint64_t)(seg.token_row + token) * a.out_stride + h * kHeadDim;
            float *slot = seg.slot < 0 ? nullptr : a.slots + (size_t)seg.slot * at_slot_floats(a.slot_rows);
            const uint32_t place = seg.quarters ? (r >> 5) * (a.slot_rows / 4) + lane : r;  // in it
            const bool floats = slot || PARTS == 3;  // what a row's values are written as
            uint8_t *to = slot ? reinterpret_cast<uint8_t *>(slot + (size_t)place * kHeadDim)
                               : static_cast<uint8_t *>(a.out) + at * (PARTS == 3 ? 4 : 2);
            const uint32_t rows = __ballot_sync(0xffffffffu, have);
            const float per = slot ? kUnit : l > 0.f || l != l ? kUnit / l : 0.f;
            const int part = TILES == 1 ? g : 0;
            const int from = part * 64, to_col = TILES == 1 ? from + 64 : 128;
            // a short loop: this code runs once a segment, and a long one waits for its instructions
            uint4 piece[4];
#pragma unroll 1
            for (int col = from; col < to_col; col += kWide) {
                float o[kWide];
                if (seg.blocks) {
                    uint32_t u[kWide];
                    tmem_load16(u, o_at + (TILES == 2 ? g * 128 : 0) + col);
#pragma unroll
                    for (int k = 0; k < kWide; k++) o[k] = TILES == 2 ? __uint_as_float(u[k]) : w0 == 0.f ? 0.f : __uint_as_float(u[k]) * w0;
                    if (two) {
                        tmem_load16(u, o_at + 128 + col);
#pragma unroll
                        for (int k = 0; k < kWide; k++)
                            if (w1 != 0.f) o[k] = fmaf(__uint_as_float(u[k]), w1, o[k]);
                    }
                    if (odd)
#pragma unroll
                        for (int k = 0; k < kWide; k++) o[k] += odd_sum<SRC, PARTS, S::kBlock>(a, sh.odd_v[used & 3], seg, seen, col + k);
                } else {
#pragma unroll
                    for (int k = 0; k < kWide; k++) o[k] = 0.f;
                }
#pragma unroll
                for (int k = 0; k < kWide; k++) o[k] = per == 0.f ? 0.f : o[k] * per;
                if (S::kQuarters && seg.quarters) {  // few rows: as they are, in a few instructions
                    if (have)
#pragma unroll
                        for (int k = 0; k < 16; k += 4)
                            store4(reinterpret_cast<float *>(to) + col + k, make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
                } else if (floats) {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        piece[k] = make_uint4(__float_as_uint(o[4 * k]), __float_as_uint(o[4 * k + 1]), __float_as_uint(o[4 * k + 2]),
                                              __float_as_uint(o[4 * k + 3]));
                    store_rows(to + 4 * col, rows, piece);
                } else {  // two steps make 64 bytes
                    const bool f16 = a.dtype == QWN_DTYPE_F16;
                    if (col & kWide) {
                        piece[2] = pack8(o, f16);
                        piece[3] = pack8(o + 8, f16);
                        store_rows(to + 2 * (col - kWide), rows, piece);
                    } else {
                        piece[0] = pack8(o, f16);
                        piece[1] = pack8(o + 8, f16);
                    }
                }
            }
            if (slot && have && part == 0) {
                slot[a.slot_rows * kHeadDim + place] = M;
                slot[a.slot_rows * (kHeadDim + 1) + place] = l;
            }
        }
        if (seg.blocks) {
            tc_fence_before();
            if (TILES == 2) {
                warp_arrive(&sh.oempty[g], lane);
            } else {
                warp_arrive(&sh.oempty[0], lane);
                if (two) warp_arrive(&sh.oempty[1], lane);
            }
        }
        return true;
    }
};

template <int SRC, int PARTS, int TILES, bool BF16>
__global__ void __launch_bounds__(AtShape<SRC, PARTS, TILES>::kThreads, 1) prompt_tile_kernel(const __grid_constant__ CUtensorMap kmap,
                                                                    const __grid_constant__ CUtensorMap vmap,
                                                                    const __grid_constant__ AtArgs a) {
    using S = AtShape<SRC, PARTS, TILES>;
    extern __shared__ uint8_t dynamic[];
    __shared__ AtShared<SRC, PARTS, TILES> sh;
    constexpr int kFirst = 8;  // the helpers' first warp
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(dynamic) + 1023u) & ~1023u;  // the host has seen that this leaves room
    if (base + S::kOperands + S::kRawTiles * S::kTileBytes > smem_u32(dynamic) + S::kSmem) {  // cannot be
        latch(a.status, QWN_KV_STATUS_WAIT_TIMEOUT);
        return;
    }
    AtRoles<SRC, PARTS, TILES, BF16> roles = {a, sh, base, base + TILES * S::kQBytes, base + S::kOperands, warp, lane};
    if (threadIdx.x == 0) {
        const uint32_t helpers = S::kTma ? 1 : 4, finishers = TILES == 2 ? 4 : 8;
        for (uint32_t i = 0; i < kAtStages; i++) {
            mbar_init(&sh.full[i], helpers);
            mbar_init(&sh.empty[i], 1);
            mbar_init(&sh.part[i], 1);
            mbar_init(&sh.fixed[i], 4);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.sfull[i], 1);
            mbar_init(&sh.pready[i][0], 4);
            mbar_init(&sh.pready[i][1], 4);
            mbar_init(&sh.ofull[i], 1);
            mbar_init(&sh.oempty[i], finishers);
            mbar_init(&sh.segfull[i], 1);
            mbar_init(&sh.segempty[i], kFirst + S::kHelpers + 2);
        }
        mbar_init(&sh.qfull, S::kHelpers);
        mbar_init(&sh.qempty, 1);
        mbar_init(&sh.joined, 8);
        mbar_init(&sh.helped, S::kHelpers);
        mbar_init(&sh.cleared, 4);
        mbar_init(&sh.drained, 1);
        for (int i = 0; i < AtShared<SRC, PARTS, TILES>::kRaw; i++) {
            mbar_init(&sh.rawfull[i], 1);
            mbar_init(&sh.rawempty[i], S::kSides == 2 ? 1 : 2);
        }
        sh.give_up = 0;
        fence_barrier_init();
    }
    if (warp == kFirst + S::kHelpers) tmem_alloc<1>(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    launch_dependents();
    wait_previous();
    if (warp < kFirst) {
        take_registers<S::kSoftmaxRegs>();
        roles.soften();
    } else if (warp < kFirst + S::kHelpers) {
        if (S::kHelperRegs < S::kLaunchRegs) give_registers<S::kHelperRegs>();
        roles.help();
    } else {
        give_registers<S::kOtherRegs>();
        if (warp == kFirst + S::kHelpers) roles.multiply();
        else if (warp == kFirst + S::kHelpers + 1) roles.load(&kmap, &vmap);
        else if (warp == kFirst + S::kHelpers + 2) roles.plan();
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && sh.give_up) latch(a.status, QWN_KV_STATUS_WAIT_TIMEOUT);
    if (warp == kFirst + S::kHelpers) {
        tc_fence_after();
        tmem_free<1>(sh.tmem, 512);
    }
}

// ---- host ----------------------------------------------------------------------

// a call's softmax scale (0: 1/sqrt(128)) times log2 e
inline void set_scale(AtArgs &a, float scale) {
    const double s = (scale > 0.f ? (double)scale : 0.08838834764831844055) * 1.44269504088896340736;
    a.scale2 = (float)s;
    // the rest is positive: times a masked score, -inf, it is to stay that
    if (a.scale2 >= s) a.scale2 = nextafterf(a.scale2, 0.f);
    a.scale2_low = (float)(s - (double)a.scale2);
}

// Prepares a kernel on the current device, once.  Refuses one whose block does not
// start with the registers that its warps share out: it would wait for them for good.
template <int SRC, int PARTS, int TILES, bool BF16>
cudaError_t prepare_tile_kernel(int device) {
    static std::mutex mu;
    static bool ready[64];
    if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> lk(mu);
    if (ready[device]) return cudaSuccess;
    const auto kernel = prompt_tile_kernel<SRC, PARTS, TILES, BF16>;
    cudaFuncAttributes at;
    cudaError_t e = cudaFuncGetAttributes(&at, kernel);
    if (e == cudaSuccess && at.numRegs < AtShape<SRC, PARTS, TILES>::kLaunchRegs) return cudaErrorInvalidConfiguration;
    // operands start on 1024 bytes behind the static part; the window itself does
    using S = AtShape<SRC, PARTS, TILES>;
    if (e == cudaSuccess && (1024 - at.sharedSizeBytes % 1024) % 1024 + S::kOperands + S::kRawTiles * S::kTileBytes > S::kSmem)
        return cudaErrorInvalidConfiguration;
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)AtShape<SRC, PARTS, TILES>::kSmem);
    ready[device] = e == cudaSuccess;
    return e;
}
template <int SRC, int PARTS, int TILES, bool BF16>
cudaError_t launch_tile_kernel(int device, uint32_t ctas, cudaStream_t s, const CUtensorMap &kmap, const CUtensorMap &vmap,
                               const AtArgs &a) {
    cudaError_t e = prepare_tile_kernel<SRC, PARTS, TILES, BF16>(device);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(AtShape<SRC, PARTS, TILES>::kThreads);
    cfg.dynamicSmemBytes = AtShape<SRC, PARTS, TILES>::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    note_early_trigger();
    e = cudaLaunchKernelEx(&cfg, prompt_tile_kernel<SRC, PARTS, TILES, BF16>, kmap, vmap, a);
    if (e == cudaSuccess) count_launch();
    else cudaGetLastError();  // reported here, not by a later launch
    return e;
}

}  // namespace
}  // namespace qkv
