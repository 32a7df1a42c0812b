// Device side of the 4-bit cache format (see kv4.h): addresses, and quantising a group.
#pragma once

#include "kv4.h"
#include "ptx.cuh"

namespace flint {

// Block `b` (64 positions) of a sequence's KV head; null where a paged sequence has no page there.
__device__ __forceinline__ unsigned char *kv4_block(const Kv4Cache &c, int seq, int kvh, int b) {
    if (c.block_table) {
        const int page = c.block_table[size_t(seq) * c.table_stride + b];
        return page < 0 ? nullptr : c.blocks + (size_t(page) * kNHeadKv + kvh) * kKv4BlockBytes;
    }
    return c.blocks + ((size_t(seq) * kNHeadKv + kvh) * c.blocks_per_seq + (uint32_t(b) & c.block_mask)) * kKv4BlockBytes;
}
__device__ __forceinline__ unsigned char *kv4_first_block(const Kv4Cache &c, int seq, int kvh) {
    return c.blocks + ((size_t(seq) * kNHeadKv + kvh) * c.blocks_per_seq + kKv4RingBlocks) * kKv4BlockBytes;
}

// Byte offset of 16-byte chunk `ch` (0..3: the codes of group ch) of row `row` among the codes of a block.
__device__ __forceinline__ int kv4_chunk(int row, int ch) { return row * kKv4RowBytes + ((ch ^ ((row >> 1) & 3)) << 4); }
// Byte offsets of a group's d and lo in a block.
__device__ __forceinline__ int kv4_k_group(int row, int g) { return kKv4KGroups + row * 16 + g * 4; }
__device__ __forceinline__ int kv4_v_group(int row, int g) { return kKv4VGroups + (row >> 1) * 32 + g * 4 + (row & 1) * 2; }

// Quantises one group held by eight neighbouring lanes, four values a lane (in order; already values of type half).
// Returns the lane's four codes, first one lowest; `dl` gets {d, lo}.  Whole warps call this.
__device__ __forceinline__ uint32_t kv4_quantise4(const float (&x)[4], __half2 &dl) {
    float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    const bool fine = fabsf(x[0]) <= 65504.f && fabsf(x[1]) <= 65504.f && fabsf(x[2]) <= 65504.f && fabsf(x[3]) <= 65504.f;
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
    }
    const uint32_t group = 0xffu << (threadIdx.x & 24);
    if ((__ballot_sync(0xffffffffu, fine) & group) != group) {
        dl = __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0));
        return 0;
    }
    const __half dh = __float2half_rn((hi - lo) / 15.0f);
    const float d = __half2float(dh);
    dl = __halves2half2(dh, __float2half_rn(lo));  // (exact: lo is one of the halves)
    uint32_t codes = 0;
    if (d > 0.f) {
#pragma unroll
        for (int i = 0; i < 4; i++) codes |= uint32_t(fminf(rintf((x[i] - lo) / d), 15.f)) << (4 * i);
    }
    return codes;
}

// Writes a lane's share (dims 4 * lane .. + 3) of a quantised K or V row.  Whole warps call this.
__device__ __forceinline__ void kv4_store_lane(unsigned char *block, int row, bool is_v, int lane, const float (&x)[4]) {
    __half2 dl;
    const uint32_t codes = kv4_quantise4(x, dl);
    const int g = lane >> 3;
    *reinterpret_cast<uint16_t *>(block + (is_v ? kKv4VCodes : kKv4KCodes) + kv4_chunk(row, g) + (lane & 7) * 2) = uint16_t(codes);
    if ((lane & 7) == 0) {
        if (is_v) {
            *reinterpret_cast<__half *>(block + kv4_v_group(row, g)) = __low2half(dl);
            *reinterpret_cast<__half *>(block + kv4_v_group(row, g) + 16) = __high2half(dl);
        } else {
            *reinterpret_cast<__half2 *>(block + kv4_k_group(row, g)) = dl;
        }
    }
}

// A lane's share (dims 4 * lane .. + 3) of a row, as values.
__device__ __forceinline__ float4 kv4_load_lane(const unsigned char *block, int row, bool is_v, int lane) {
    const int g = lane >> 3;
    const uint32_t c = *reinterpret_cast<const uint16_t *>(block + (is_v ? kKv4VCodes : kKv4KCodes) + kv4_chunk(row, g) + (lane & 7) * 2);
    float d, lo;
    if (is_v) {
        d = __half2float(*reinterpret_cast<const __half *>(block + kv4_v_group(row, g)));
        lo = __half2float(*reinterpret_cast<const __half *>(block + kv4_v_group(row, g) + 16));
    } else {
        const float2 dl = __half22float2(*reinterpret_cast<const __half2 *>(block + kv4_k_group(row, g)));
        d = dl.x;
        lo = dl.y;
    }
    return make_float4(fmaf(float(c & 15), d, lo), fmaf(float((c >> 4) & 15), d, lo), fmaf(float((c >> 8) & 15), d, lo),
                       fmaf(float(c >> 12), d, lo));
}

}  // namespace flint
