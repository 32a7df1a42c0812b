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

// A half-precision row's K and V, four values of each a lane, for the products of a prefill (see its prologue): infinities and
// NaN of V become zeros, and the K row beside them NaN.
__device__ __forceinline__ void half_row_staged(uint2 &k, uint2 &v) {
    auto odd = [](uint32_t w) {  // 0xffff in each half that is an infinity or a NaN
        return ((w & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((w & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
    };
    const uint32_t a = odd(v.x), b = odd(v.y);
    if (!__any_sync(0xffffffffu, (a | b) != 0)) return;
    v = make_uint2(v.x & ~a, v.y & ~b);
    k = make_uint2(0x7fff7fffu, 0x7fff7fffu);
}

// d and lo of a group, packed {d, lo}, and 1 / d, from its least and largest value (halves; NaN if a value was one).  A group
// that holds an infinity or a NaN gets d = NaN.  The quotient by 15, like those by d below, is the product with the
// reciprocal and one correction step, which rounds it as a division does (Markstein 1990).  32 bits, not exact, because exact
// codes would ask each value how near it is to a border, some 15 % more instructions of a store by count, for one code in billions.
struct Kv4Scale {
    uint32_t dl;
    float d, lo, inv;
};
__device__ __forceinline__ Kv4Scale kv4_scale(__half least, __half largest) {
    Kv4Scale s;
    s.lo = __half2float(least);
    const float hi = __half2float(largest);
    if (!(fabsf(s.lo) <= 65504.f && fabsf(hi) <= 65504.f)) {
        s.dl = 0x00007fffu;
        s.d = s.inv = s.lo = 0.f;
        return s;
    }
    constexpr float k15 = 1.0f / 15.0f;
    const float range = hi - s.lo;
    float q = range * k15;
    q = fmaf(fmaf(-q, 15.f, range), k15, q);
    const __half2 dl = __halves2half2(__float2half_rn(q), least);
    s.dl = *reinterpret_cast<const uint32_t *>(&dl);
    s.d = __low2float(dl);
    s.inv = s.d > 0.f ? __frcp_rn(s.d) : 0.f;
    return s;
}
// Two floats at a time
__device__ __forceinline__ uint64_t kv4_pack(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint64_t kv4_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t kv4_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t kv4_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// Codes of N values (pairs of floats x, at most eight), first one lowest.  Adding 1.5 * 2^23 rounds a quotient to the nearest
// whole number, ties to even, and leaves that in the low bits of the sum, whose next bits are zeros.
template <int N, bool kLimit>
__device__ __forceinline__ uint32_t kv4_codes(const float2 (&x)[N / 2], const Kv4Scale &s) {
    const uint64_t lo2 = kv4_pack(-s.lo, -s.lo), inv2 = kv4_pack(s.inv, s.inv), nd2 = kv4_pack(-s.d, -s.d), magic = kv4_pack(12582912.f, 12582912.f);
    uint32_t c[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
        uint64_t q[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const float2 v = x[2 * i + j];
            const uint64_t a = kv4_add(kv4_pack(v.x, v.y), lo2), q0 = kv4_mul(a, inv2);
            q[j] = kv4_fma(kv4_fma(q0, nd2, a), inv2, q0);
            if (kLimit) {
                float r0, r1;
                asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r0), "=f"(r1) : "l"(q[j]));
                q[j] = kv4_pack(fminf(r0, 15.f), fminf(r1, 15.f));
            }
            q[j] = kv4_add(q[j], magic);
        }
        c[i] = uint32_t(q[0]) + (uint32_t(q[0] >> 32) << 4) + (uint32_t(q[1]) << 8) + (uint32_t(q[1] >> 32) << 12);
    }
    return N == 4 ? c[0] & 0xffffu : __byte_perm(c[0], c[N / 4 - 1], 0x5410);
}
// d = 0: the codes are 0.  A subnormal d may lie well below (max - lo) / 15, so its quotients are limited to 15 (else 15.01
// is the most).
template <int N>
__device__ __forceinline__ uint32_t kv4_codes(const float2 (&x)[N / 2], const Kv4Scale &s) {
    if (s.inv == 0.f) return 0;
    return s.d < 6.103515625e-5f ? kv4_codes<N, true>(x, s) : kv4_codes<N, false>(x, s);
}
__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2 *>(&w); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }

// Quantises a group held by eight neighbouring lanes, four half-precision values a lane, in order.  Returns the lane's four
// codes; `dl` gets {d, lo}.  Whole warps call this.
__device__ __forceinline__ uint32_t kv4_quantise4(uint2 h, uint32_t &dl) {
    __half2 lo = __hmin2_nan(as_half2(h.x), as_half2(h.y)), hi = __hmax2_nan(as_half2(h.x), as_half2(h.y));
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
        lo = __hmin2_nan(lo, as_half2(__shfl_xor_sync(0xffffffffu, as_u32(lo), off)));
        hi = __hmax2_nan(hi, as_half2(__shfl_xor_sync(0xffffffffu, as_u32(hi), off)));
    }
    const Kv4Scale s = kv4_scale(__hmin_nan(__low2half(lo), __high2half(lo)), __hmax_nan(__low2half(hi), __high2half(hi)));
    dl = s.dl;
    const float2 x[2] = {__half22float2(as_half2(h.x)), __half22float2(as_half2(h.y))};
    return kv4_codes<4>(x, s);
}
// The same for two neighbouring lanes with sixteen values each.
__device__ __forceinline__ uint2 kv4_quantise16(uint4 h, uint4 k, uint32_t &dl) {
    auto least = [](uint4 w) { return __hmin2_nan(__hmin2_nan(as_half2(w.x), as_half2(w.y)), __hmin2_nan(as_half2(w.z), as_half2(w.w))); };
    auto largest = [](uint4 w) { return __hmax2_nan(__hmax2_nan(as_half2(w.x), as_half2(w.y)), __hmax2_nan(as_half2(w.z), as_half2(w.w))); };
    __half2 lo = __hmin2_nan(least(h), least(k)), hi = __hmax2_nan(largest(h), largest(k));
    lo = __hmin2_nan(lo, as_half2(__shfl_xor_sync(0xffffffffu, as_u32(lo), 1)));
    hi = __hmax2_nan(hi, as_half2(__shfl_xor_sync(0xffffffffu, as_u32(hi), 1)));
    const Kv4Scale s = kv4_scale(__hmin_nan(__low2half(lo), __high2half(lo)), __hmax_nan(__low2half(hi), __high2half(hi)));
    dl = s.dl;
    const float2 x[4] = {__half22float2(as_half2(h.x)), __half22float2(as_half2(h.y)), __half22float2(as_half2(h.z)), __half22float2(as_half2(h.w))};
    const float2 y[4] = {__half22float2(as_half2(k.x)), __half22float2(as_half2(k.y)), __half22float2(as_half2(k.z)), __half22float2(as_half2(k.w))};
    if (s.inv == 0.f) return make_uint2(0, 0);
    if (s.d < 6.103515625e-5f) return make_uint2(kv4_codes<8, true>(x, s), kv4_codes<8, true>(y, s));
    return make_uint2(kv4_codes<8, false>(x, s), kv4_codes<8, false>(y, s));
}

// Writes {d, lo} of a group of one row.
__device__ __forceinline__ void kv4_store_group(unsigned char *block, int row, int g, bool is_v, uint32_t dl) {
    if (is_v) {
        *reinterpret_cast<uint16_t *>(block + kv4_v_group(row, g)) = uint16_t(dl);
        *reinterpret_cast<uint16_t *>(block + kv4_v_group(row, g) + 16) = uint16_t(dl >> 16);
    } else {
        *reinterpret_cast<uint32_t *>(block + kv4_k_group(row, g)) = dl;
    }
}

// Writes a lane's share (dims 4 * lane .. + 3) of a K or V row, quantised.  Whole warps call this.
__device__ __forceinline__ void kv4_store_lane(unsigned char *block, int row, bool is_v, int lane, uint2 h) {
    uint32_t dl;
    const uint32_t codes = kv4_quantise4(h, dl);
    const int g = lane >> 3;
    *reinterpret_cast<uint16_t *>(block + (is_v ? kKv4VCodes : kKv4KCodes) + kv4_chunk(row, g) + (lane & 7) * 2) = uint16_t(codes);
    if ((lane & 7) == 0) kv4_store_group(block, row, g, is_v, dl);
}

}  // namespace flint
