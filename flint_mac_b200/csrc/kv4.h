// K/V caches held in 4 bits: the block format, and the launchers of the kernels that write and read it.
//
// A cache row is the 128 values x of one token and KV head, K or V, rounded to half, in four groups of 32.  A group keeps
//   lo = min x,   d = half((max x - lo) / 15),   code = round-half-even((x - lo) / d) limited to 0..15   (0 where d = 0)
// and stands for lo + code * d.  Differences and quotients are those of 32 bits, so a value within 2^-19 of a step of the border
// between two codes may get either: where one of x and lo is far smaller than the other, their difference has more bits than a
// float.  A group that holds an infinity or a NaN gets d = NaN and reads back as NaN throughout.
// Codes are 64 bytes a row, d and lo 2 + 2 bytes a group: 80 bytes, where the half-precision cache takes 256.
//
// 64 consecutive positions of one sequence and KV head make one block of 10240 bytes, K and V together, so that one bulk
// copy brings a tile in:
//   [0, 4096)       K codes: 64 rows of 64 bytes, dim i in nibble i (low nibble first); the 16-byte chunk c of row r lies
//                   at chunk c ^ ((r >> 1) & 3), which spreads the rows that one ldmatrix reads over all banks
//   [4096, 5120)    K groups: 64 rows of 4 x {half d, half lo}
//   [5120, 9216)    V codes, like K's
//   [9216, 10240)   V groups: 32 pairs of rows (2i, 2i + 1), each 4 x {d of row 2i, d of row 2i + 1}, then 4 x {lo, lo}:
//                   the two rows side by side are the operand pairs of the product with the probabilities
// Sequences own their blocks one after the other ([max_seqs][4][blocks], ring layers 16 blocks) or take them from a page
// pool ([pages][4]).  A ring layer whose first tokens stay visible has one more block, which keeps those.
#pragma once

#include "attn_common.h"
#include "kv4_plan.h"

namespace flint {

constexpr int kKv4Group = 32;
constexpr int kKv4Groups = kHeadDim / kKv4Group;
constexpr int kKv4BlockKeys = 64;
constexpr int kKv4RowBytes = kHeadDim / 2;
constexpr int kKv4KCodes = 0;
constexpr int kKv4KGroups = kKv4KCodes + kKv4BlockKeys * kKv4RowBytes;
constexpr int kKv4VCodes = kKv4KGroups + kKv4BlockKeys * kKv4Groups * 4;
constexpr int kKv4VGroups = kKv4VCodes + kKv4BlockKeys * kKv4RowBytes;
constexpr int kKv4BlockBytes = kKv4VGroups + kKv4BlockKeys * kKv4Groups * 4;
static_assert(kKv4BlockBytes == 10240, "block layout");
constexpr int kKv4RingBlocks = kSwaRing / kKv4BlockKeys;
static_assert(kMaxFirstTokens == kKv4BlockKeys, "one block keeps them");

// Where a layer's blocks are.
struct Kv4Cache {
    unsigned char *blocks = nullptr;
    int blocks_per_seq = 0;               // contiguous: blocks of one (sequence, KV head)
    uint32_t block_mask = 0xFFFFFFFFu;    // ring layers: 15
    int first_tokens = 0;                 // ring layers: positions below this one are kept in block kKv4RingBlocks too
    const int32_t *block_table = nullptr; // paged: block b of sequence s is page block_table[s * table_stride + b]
    int table_stride = 0;
};

// One decode launch over 4-bit caches (the fields that DecParams has mean the same).
struct Dec4Params {
    const void *qkv;
    void *out;
    const float *q_norm, *k_norm, *sinks, *inv_freq;
    Kv4Cache cache;
    float *scratch, *scratch2;  // split-K records of both merge levels, [n_records][4 KV heads][8][kRecStride]
    int *tickets, *tickets2;    // arrival counters, [n_records][4][8]; zero between launches (and graph replays)
    int tok0;                   // row of qkv and out that the launch's token 0 has
    int is_swa, has_rope, qkv_dtype, out_dtype;
    int *error_flag;
};
cudaError_t decode_kv4_setup();
// The work list (kv4_plan.h; at most kDec4MaxPieces) travels in the kernel's parameters.
cudaError_t launch_decode_kv4(const Dec4Params &p, const Dec4Piece *pieces, int n_pieces, int n_warps, cudaStream_t stream);

// Rows of K and V between a cache and dense arrays [n][4][n_rows][128]: row r of sequence i is position pos0[i] + r.
constexpr int kKvRowsSeqs = 128;  // sequences a launch names in its parameters
struct KvRowsSeqs {
    int32_t seq[kKvRowsSeqs], pos0[kKvRowsSeqs];
    int32_t held[kKvRowsSeqs];  // paged layers: pages of the sequence (the table's entries past them may be another's by now)
};
struct KvRowsParams {
    Kv4Cache cache;             // 4-bit caches, or
    __half *k_cache = nullptr, *v_cache = nullptr;  // half-precision ones (cache.blocks is null then)
    __half *first_k = nullptr, *first_v = nullptr;  // their first tokens' rows (cache.first_tokens > 0), [max_seqs][4][64][128]
    int n_slots = 0;
    int is_swa = 0;
    int raw_slots = 0;          // ring layers: pos0 counts slots (the first tokens' rows from kSwaRing on), not positions
    int dtype = 0;              // of k and v
    int staging = 0;            // load: V without infinities and NaN, K rows beside those NaN, for the products of a prefill
    int n_rows = 0;
    long long seq_stride = 0, head_stride = 0;  // elements of k and v
    void *k = nullptr, *v = nullptr;
};
cudaError_t kv_rows_setup();
cudaError_t launch_kv_store(const KvRowsParams &p, const KvRowsSeqs &seqs, int n, cudaStream_t stream);
cudaError_t launch_kv_load(const KvRowsParams &p, const KvRowsSeqs &seqs, int n, cudaStream_t stream);

}  // namespace flint
