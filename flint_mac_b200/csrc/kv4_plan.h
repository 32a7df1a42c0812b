// The work list of a decode launch over 4-bit caches (host side, and what host and device share).
//
// The visible keys of a (token, KV head) group are tiles of 64; a token's tiles are cut into equal pieces, and the launch
// has one CTA per piece and KV head, longest first.  Where there are more than the GPU holds at a time, the hardware starts
// the next one on the SM that is through first, so that an SM that gets less of the memory's bandwidth than others takes
// fewer pieces.  (CTAs that stay and take over the pieces of those that have not started, the next piece's rows fetched
// ahead, were slower on every batch: 256 windows of a mixed batch 27.4 against 20.7 us, 128 sequences of 8192 keys 137
// against 130, 400 of 0 to 3000 46.1 against 43.1.)
#pragma once

#include <algorithm>
#include <vector>

#include "attn_common.h"

namespace flint {

constexpr int kDec4CtasPerSm = 2;     // CTAs of eight warps that an SM holds at a time (of four: four, of sixteen: one)
constexpr int kDec4MaxPieces = 1300;  // of one launch (the list travels in the kernel's parameters)

// Tiles [t0, t0 + n) of a token, part `split` of n_split, for each of the four KV heads.
struct Dec4Piece {
    int32_t seq, pos, t0, n;
    uint16_t tok;              // row of the launch
    uint16_t split, n_split;
    uint16_t part0;            // cut tokens: pieces of those before it, where its records and counters begin
};
static_assert(sizeof(Dec4Piece) == 24, "pieces travel in the kernel's parameters");

// What a token at `pos` sees of its cache.
struct Dec4Range {
    int j0;       // first key of the contiguous range [j0, pos)
    int n_first;  // keys [0, n_first) in front of it that stay visible
    int tiles;    // 64-key tiles: the first tokens' one if n_first > 0, then those of the range
};
__host__ __device__ inline Dec4Range dec4_range(int pos, int is_swa, int first_tokens) {
    Dec4Range r;
    r.j0 = is_swa && pos > kNSwa - 1 ? pos - (kNSwa - 1) : 0;
    r.n_first = is_swa ? (first_tokens < r.j0 ? first_tokens : r.j0) : 0;
    r.tiles = (r.n_first > 0 ? 1 : 0) + (pos > r.j0 ? ((pos - 1) >> 6) - (r.j0 >> 6) + 1 : 0);
    return r;
}

// Splits folded by one warp in the first merge level: all of them while one trip to memory holds their records, else two
// levels of about equal size.
constexpr int kDec4MergeTrip = 10;  // records whose loads are in flight together
__host__ __device__ inline int dec4_fan(int n_split) {
    if (n_split <= kDec4MergeTrip) return n_split;
    int f = kDec4MergeTrip;
    while (f * f < n_split) f++;
    return f;
}

// Pieces of the first tokens of a batch, as many tokens as one launch takes (returned); tiles[i]: tiles of token i.
// `slots`: CTAs of eight warps that the GPU holds at a time.  n_records: pieces that leave a record (one for each KV head
// and query head); n_warps: warps of a CTA.
//
// While every token's four groups fit the slots the launch is one round: the tokens are cut so that the longest piece is as
// short as the slots allow.  A piece costs some 5 us beside its tiles (rows, norm and rotation, the merges), so nothing is
// cut below kLeast tiles, and a window never.  Larger batches go in several rounds, cut only where a token is longer than a
// slot's share.  Warps of a CTA (each the others' time in long runs): eight, as 64 x 8192 keys take 66.7 us (four 110, sixteen
// 67.1), one 131072-key sequence 22.0 (28, 28.6), 32 sequences of 0 to 32768 keys 23.7 (45, 27).  Many short pieces are over
// sooner with four, whose CTAs overlap each other's beginnings and ends: 256 windows 28.6 (eight 34.6), 256 x 600 keys 28.3
// (33.4).  Pieces that leave half of the GPU idle have sixteen, if they have tiles for them: 32 windows 7.2 (eight 10.0, four
// 14.6), 4 x 8192 keys 9.7 (12.8, 21.7).
inline int plan_decode_kv4(int n, const int32_t *seqs, const int32_t *pos, const int *tiles, int slots,
                           std::vector<Dec4Piece> &pieces, int &n_records, int &n_warps) {
    constexpr int kLeast = 16;
    n = std::min(n, kDec4MaxPieces / 2);
    slots = std::max(slots, 1);
    long long total = 0;
    int longest = 0;
    for (int i = 0; i < n; i++) {
        total += kNHeadKv * (long long)tiles[i];
        longest = std::max(longest, tiles[i]);
    }
    auto parts = [&](int t, int piece) { return std::max(1, int((t + (long long)piece - 1) / piece)); };
    const long long share = (total + slots - 1) / slots;
    const bool one_round = n * kNHeadKv <= slots;
    const long long room = one_round ? std::min(slots / kNHeadKv, kDec4MaxPieces) : kDec4MaxPieces;
    int piece = int(std::max<long long>(kLeast, share));
    for (;; piece += std::max(1, piece / 32)) {  // (piece = longest always fits: one part a token)
        long long count = 0;
        for (int i = 0; i < n; i++) count += parts(tiles[i], piece);
        if (count <= room) break;
    }
    pieces.clear();
    n_records = 0;
    int largest = 0;
    for (int i = 0; i < n; i++) {
        const int k = parts(tiles[i], piece), each = parts(tiles[i], k);  // k nearly equal parts
        const int n_split = std::max(1, parts(tiles[i], each));
        for (int s = 0, at = 0; s < n_split; s++, at += each)
            pieces.push_back(Dec4Piece{seqs[i], pos[i], at, std::min(each, tiles[i] - at), uint16_t(i), uint16_t(s), uint16_t(n_split), uint16_t(n_records)});
        largest = std::max(largest, std::min(each, tiles[i]));
        if (n_split > 1) n_records += n_split;
    }
    std::stable_sort(pieces.begin(), pieces.end(), [](const Dec4Piece &a, const Dec4Piece &b) { return a.n > b.n; });
    n_warps = !one_round && largest <= kLeast ? 4 : int(pieces.size()) * kNHeadKv * 2 <= slots && largest > 8 ? 16 : 8;
    return n;
}

}  // namespace flint
