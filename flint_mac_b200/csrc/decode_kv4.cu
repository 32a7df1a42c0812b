// Decode attention over K/V caches held in 4 bits (format: kv4.h), full layers and sliding-window layers whose first
// tokens stay visible.
//
// With x = lo + c d per group of 32 dims, scores and outputs of one query head are
//   s_j = sum_g (d_jg sum_{i in g} q_i c_ji + lo_jg sum_{i in g} q_i),   p_j = e^(s_j),
//   O_i = sum_j p_j (d_jg c_ji + lo_jg) / (e^sink + sum_j p_j)
// over the keys j that the query sees: [0, pos) on a full layer, [pos - 512, pos) and the first tokens [0, F) on a
// sliding-window layer, and the token itself.  The token itself enters at half precision, as its own record of the final
// merge; its row is quantised into the cache by the same launch.
//
// The codes go to the tensor cores as they are: bits masked out of the low byte of a 16-bit lane are a half-precision
// number, their value times 2^-24, which the products take exactly.  Of the four codes n0 .. n3 of a lane the operands are
// n0, n0 + 16 n1, n2 and n2 + 16 n3: four logical operations for the eight codes of a register.  On the K side
//   q0 n0 + q1 n1 = (q0 - q1 / 16) n0 + (q1 / 16) (n0 + 16 n1),
// so Q is stored with those factors (times four, away from half's subnormals); on the V side the output of n1 is a sixteenth
// of the difference of two outputs.  On the K side d multiplies the 32-dim partial scores (4 groups per key), on the V side
// it multiplies the probabilities (4 operand pairs per 16 keys), and lo enters through one more product each.
//
// A CTA works on one piece (kv4_plan.h).  Its warps (four, eight or sixteen) take the piece's tiles in turn and work alone: a
// tile is one 5 KB bulk copy for K and one for V, on mbarriers of the warp's own; the next tile's K comes in while this one's
// V is worked on, and the other way round.
//
// Roundings to half, 2^-11 relative each, which the products' operands need: the rows of q after norm, rotation and scale;
// their operands q0 - q1 / 16 once more; the probabilities (the denominator adds them up unrounded); a probability times d.
// Sums, maxima, records and the parts of lo are in 32 bits.
//
// Bytes per tile of 64 keys: 10240, against 885 instructions of the warp, 72 of them products.  64 x 8192 keys (337 MB) take
// 58.2 us, 5.8 TB/s or 0.90 of a copy's rate, in short runs, and 66.7 us when the GPU's power limit holds the clocks down in
// a long one: the SMs issue 2.1 instructions a cycle (46 % of the logical unit's rate, 35 % of the tensor pipe's) and DRAM is
// 69 % busy, so memory and issue bound it together.  Shorter launches are bound by latency: about 1.8 us from the wait to the
// first tile (rows, norm, rotation), 2 us a tile and warp, 1.2 us for the merge of the warps, 4 to 5 us for that of the
// splits.  One 131072-key sequence takes 22.0 us (its bytes 13), 32 windows 7.2, 256 windows of a mixed batch 21, 317 keys 5.7.
#include <cstring>

#include "decode_common.cuh"
#include "kv4.cuh"

namespace flint {

namespace {

constexpr int kHalf = kKv4VCodes;    // a block's K part, and its V part: 5120 bytes each
static_assert(kKv4BlockBytes == 2 * kHalf, "K and V part of a block are alike");
constexpr int kORow = kHeadDim + 4;  // floats between heads of the merge buffer: the eight lanes of a store hit different banks

template <int kWarps>
struct __align__(128) Dec4Smem {
    unsigned char k[kWarps][kHalf];
    union {
        unsigned char v[kWarps][kHalf];
        float o[kWarps][kGqa][kORow];  // the warps' outputs of a piece, once all are through with its tiles
    };
    alignas(8) unsigned long long full_bar[kWarps][2];  // the K part, the V part has landed
    alignas(16) unsigned char raw[kGqa + 2][kHeadDim * 4];  // raw rows: q heads, new k, new v
    alignas(16) __half q[kGqa][kHeadDim];  // normalised, rotated, scaled by log2(e) / sqrt(128)
    float red_m[kWarps][kGqa], red_l[kWarps][kGqa];
    alignas(16) __half knew[kHeadDim];
    alignas(16) __half vnew[kHeadDim];
    alignas(16) float rope_cos[kHeadDim / 2], rope_sin[kHeadDim / 2];
    alignas(16) float q_norm[kHeadDim], k_norm[kHeadDim], sinks[kNHead];
};
static_assert(sizeof(Dec4Smem<16>) <= 225 * 1024 && sizeof(Dec4Smem<4>) * 4 <= 223 * 1024 && sizeof(Dec4Smem<8>) * 2 <= 225 * 1024, "CTAs of an SM");

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ void lds128(uint32_t (&v)[4], uint32_t addr) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// The operands n0, n0 + 16 n1, n2, n2 + 16 n3 of a register of eight codes.
struct Codes {
    uint32_t n0, n01, n2, n23;
};
__device__ __forceinline__ Codes split_codes(uint32_t w) {
    Codes c;
    c.n0 = w & 0x000f000fu;
    c.n01 = w & 0x00ff00ffu;
    c.n23 = __byte_perm(w, 0u, 0x4341);
    c.n2 = c.n23 & 0x000f000fu;
    return c;
}
// D(16x8, f32) = A(16x16, f16, row) * B(16x8, f16, col)
__device__ __forceinline__ void mma_16816_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Packed two-float arithmetic
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void fma2(float &a, float &b, uint64_t m, float c0, float c1) {  // (a, b) = (a, b) * m + (c0, c1)
    asm("{\n.reg .b64 x, y;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%3, %4};\nfma.rn.f32x2 x, x, %2, y;\nmov.b64 {%0, %1}, x;\n}\n"
        : "+f"(a), "+f"(b)
        : "l"(m), "f"(c0), "f"(c1));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void sub2(float &a, float &b, uint64_t m) {  // (a, b) -= m
    asm("{\n.reg .b64 x;\nmov.b64 x, {%0, %1};\nsub.rn.f32x2 x, x, %2;\nmov.b64 {%0, %1}, x;\n}\n" : "+f"(a), "+f"(b) : "l"(m));
}
__device__ __forceinline__ void add2(uint64_t &acc, float a, float b) {
    asm("{\n.reg .b64 x;\nmov.b64 x, {%1, %2};\nadd.rn.f32x2 %0, %0, x;\n}\n" : "+l"(acc) : "f"(a), "f"(b));
}

__device__ __forceinline__ float low_half(uint32_t a) { return __low2float(*reinterpret_cast<const __half2 *>(&a)); }

// Bounded by a count of polls (a quarter of a second or more), not by the clock: the loop is four instructions.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity) {
#pragma unroll 1
    for (uint32_t n = 0; n < (1u << 24); n++)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}

// Folds n partial records of one head into (M, L, a): the lane's four dims d0 .. d0 + 3.  Record i lies at rec(i).
// kDec4MergeTrip records a trip, their loads in flight together.
struct Merged4 {
    float M, L, a[4];
};
template <typename Rec>
__device__ __forceinline__ Merged4 merge_records4(Rec rec, int n, int d0) {
    constexpr int kTrip = kDec4MergeTrip;
    Merged4 r;
    r.M = -INFINITY;
    r.L = r.a[0] = r.a[1] = r.a[2] = r.a[3] = 0.f;
#pragma unroll 1
    for (int s0 = 0; s0 < n; s0 += kTrip) {
        float2 ml[kTrip];
        float4 x[kTrip];
#pragma unroll
        for (int i = 0; i < kTrip; i++) {
            const float *q = rec(min(s0 + i, n - 1));  // past the end: the last one again, unused
            ml[i] = __ldcg(reinterpret_cast<const float2 *>(q + kHeadDim));
            x[i] = __ldcg(reinterpret_cast<const float4 *>(q + d0));
            if (s0 + i >= n) ml[i] = make_float2(-INFINITY, 0.f);
        }
        float cm = r.M;
#pragma unroll
        for (int i = 0; i < kTrip; i++) cm = fmaxf(cm, ml[i].x);
        const float keep = r.M == -INFINITY ? 0.f : fast_exp2(r.M - cm);
        r.L *= keep;
#pragma unroll
        for (int j = 0; j < 4; j++) r.a[j] *= keep;
        r.M = cm;
#pragma unroll
        for (int i = 0; i < kTrip; i++) {
            const float c = ml[i].y == 0.f ? 0.f : fast_exp2(ml[i].x - cm);
            r.L += ml[i].y * c;
            r.a[0] += x[i].x * c; r.a[1] += x[i].y * c; r.a[2] += x[i].z * c; r.a[3] += x[i].w * c;
        }
    }
    return r;
}

__device__ __forceinline__ void store_out4(void *out, int dtype, size_t idx, float a, float b, float c, float d) {
    if (dtype == kDtypeF32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(out) + idx) = make_float4(a, b, c, d);
    } else {
        const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
        *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(out) + idx) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
    }
}

__device__ __forceinline__ void cp_async8(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(dst), "l"(src) : "memory");
}

template <int kWarps>
__device__ __forceinline__ void decode_piece(const Dec4Params &p, const Dec4Piece &piece, int kvh) {
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Dec4Smem<kWarps> &sm = *reinterpret_cast<Dec4Smem<kWarps> *>(smem_raw);
    constexpr int kThreads = kWarps * 32;
    constexpr int kHeads = kWarps < kGqa ? kGqa / kWarps : 1;  // query heads of the group that a warp looks after in the prologue and the merge
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t4 = lane & 3, d0 = 4 * lane;
    // Which warps do what beside: the first eight have heads; the last two have the new token's k and v (their tiles come
    // last, if they have any), two others the rotation table.
    const bool has_heads = kWarps <= kGqa || warp < kGqa;
    const int nw = warp - (kWarps - 2), rope_at = tid - (kWarps / 2 - 2) * 32;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const bool rope = p.has_rope != 0;
    float freq = 0.f;
    const bool rope_warp = rope && rope_at >= 0 && rope_at < kHeadDim / 2;
    if (rope_warp) freq = p.inv_freq[rope_at];
    // the layer's constants, early: a load past a busy memory system takes microseconds
    for (int i = tid; i < kHeadDim; i += kThreads) {
        sm.q_norm[i] = p.q_norm[i];
        sm.k_norm[i] = p.k_norm[i];
        if (i < kNHead) sm.sinks[i] = p.sinks[i];
    }
    const uint32_t k_tile = smem_u32(&sm.k[warp][0]), v_tile = smem_u32(&sm.v[warp][0]);
    const uint32_t k_bar = smem_u32(&sm.full_bar[warp][0]), v_bar = k_bar + 8;
    if (lane == 0) {
        mbar_init(k_bar, 1);
        mbar_init(v_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }

    // ldmatrix addresses of a lane in the K and V codes of 16 rows (the chunk swizzle depends on the row mod 8 alone)
    const int sw = (lane & 7) >> 1;
    const uint32_t k_at = k_tile + (lane & 7) * kKv4RowBytes + (((lane >> 3) ^ sw) << 4);
    const uint32_t v_at = v_tile + (((lane >> 3) & 1) * 8 + (lane & 7)) * kKv4RowBytes + (((lane >> 4) ^ sw) << 4);
    const uint32_t kg_at = k_tile + kKv4KGroups + g * 16, vg_at = v_tile + (kKv4VGroups - kHalf) + t4 * 32;

    const Dec4Piece pc = piece;
    const Dec4Range rg = dec4_range(pc.pos, p.is_swa, p.cache.first_tokens);
    const int ta = pc.t0, tb = ta + pc.n;
    const bool ends = pc.split == pc.n_split - 1;  // the piece ends its group: it also takes the new token
    const int extra = rg.n_first > 0 ? 1 : 0;
    const unsigned char *seq_blocks = p.cache.blocks + (size_t(pc.seq) * kNHeadKv + kvh) * p.cache.blocks_per_seq * kKv4BlockBytes;  // contiguous caches: the group's first block
    auto load_part = [&](int t, int is_v) {  // one lane
        const int b = (rg.j0 >> 6) + t - extra;
        const unsigned char *block;
        if (p.cache.block_table) block = kv4_block(p.cache, pc.seq, kvh, b);
        else block = seq_blocks + size_t(t < extra ? uint32_t(kKv4RingBlocks) : uint32_t(b) & p.cache.block_mask) * kKv4BlockBytes;
        const uint32_t bar = is_v ? v_bar : k_bar;
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // earlier accesses to the buffer come first
        mbar_expect_tx(bar, kHalf);
        bulk_load(is_v ? v_tile : k_tile, block + is_v * kHalf, kHalf, bar);
    };
    // Raw rows: its heads of the group by each warp, the new k and v by the last two warps too.  A warp reads what it fetched.
    auto fetch_rows = [&] {
        const int head0 = kvh * kGqa, tok = p.tok0 + pc.tok;
        const size_t es = p.qkv_dtype == kDtypeF32 ? 4 : 2;
        const unsigned char *row = static_cast<const unsigned char *>(p.qkv) + size_t(tok) * kQkvDim * es;
        auto fetch = [&](int at, int i) {
            const uint32_t dst = smem_u32(&sm.raw[i][0]) + d0 * uint32_t(es);
            if (es == 4) cp_async16(dst, row + (at + d0) * es, 16);
            else cp_async8(dst, row + (at + d0) * es);
        };
#pragma unroll
        for (int i = 0; i < kHeads; i++)
            if (has_heads) fetch((head0 + warp * kHeads + i) * kHeadDim, warp * kHeads + i);
        if (ends && nw >= 0) fetch(kQDim + nw * kKvDim + kvh * kHeadDim, kGqa + nw);
        cp_async_commit();
    };
    auto rope_table = [&] {
        if (!rope_warp) return;
        float sn, cs;
        sincos_reduced(float(pc.pos) * freq, &sn, &cs);
        sm.rope_cos[rope_at] = cs;
        sm.rope_sin[rope_at] = sn;
    };
    auto finish_rows = [&] {  // raw rows (and the rotation table, visible already) -> sm.q, the new token's rows, the cache
        cp_async_wait<0>();
        __syncwarp();
        float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
        if (rope) {
            cs = reinterpret_cast<const float4 *>(sm.rope_cos)[lane & 15];
            sn = reinterpret_cast<const float4 *>(sm.rope_sin)[lane & 15];
        }
        const float qscale = rsqrtf(float(kHeadDim)) * kLog2e;  // softmax runs in base 2
#pragma unroll
        for (int i = 0; i < kHeads; i++) {
            if (!has_heads) break;
            const int h = warp * kHeads + i;
            float4 x = norm_rope(load_row4(&sm.raw[h][0], p.qkv_dtype, 0, lane), reinterpret_cast<const float4 *>(sm.q_norm)[lane], cs, sn, lane, rope);
            x.x *= qscale; x.y *= qscale; x.z *= qscale; x.w *= qscale;
            store_half4(&sm.q[h][d0], x);
        }
        if (ends && nw >= 0) {
            float4 x = load_row4(&sm.raw[kGqa + nw][0], p.qkv_dtype, 0, lane);
            if (nw == 0) x = norm_rope(x, reinterpret_cast<const float4 *>(sm.k_norm)[lane], cs, sn, lane, rope);
            const uint2 h = make_uint2(pack_half2(x.x, x.y), pack_half2(x.z, x.w));
            *reinterpret_cast<uint2 *>(nw == 0 ? &sm.knew[d0] : &sm.vnew[d0]) = h;
        }
    };
    auto store_new = [&] {  // the new token's rows -> the cache
        if (!ends || nw < 0) return;
        const uint2 h = *reinterpret_cast<const uint2 *>(nw == 0 ? &sm.knew[d0] : &sm.vnew[d0]);
        kv4_store_lane(kv4_block(p.cache, pc.seq, kvh, pc.pos >> 6), pc.pos & 63, nw == 1, lane, h);
        if (p.is_swa && pc.pos < p.cache.first_tokens)
            kv4_store_lane(kv4_first_block(p.cache, pc.seq, kvh), pc.pos, nw == 1, lane, h);
    };
    // Nothing an earlier kernel of the stream produces (rows, cache contents, split-K records and counters) is read or
    // written before this wait.
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    fetch_rows();
    if (lane == 0 && ta + warp < tb) load_part(ta + warp, 0);
    rope_table();
    __syncthreads();
    finish_rows();
    __syncthreads();

    const uint64_t two22 = pack2(4194304.f, 4194304.f);
    int used = 0;  // tiles this warp has been through: the phase of its barriers
    if (lane == 0 && ta + warp < tb) load_part(ta + warp, 1);
    store_new();
    float s_new[kHeads];  // the new token's score with the warp's heads
#pragma unroll
    for (int i = 0; i < kHeads; i++) s_new[i] = -INFINITY;
    if (ends && has_heads) {
        const uint2 h = *reinterpret_cast<const uint2 *>(&sm.knew[d0]);
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&h.y));
#pragma unroll
        for (int i = 0; i < kHeads; i++) {
            const uint2 w = *reinterpret_cast<const uint2 *>(&sm.q[warp * kHeads + i][d0]);
            const float2 c = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), d = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
            s_new[i] = warp_sum(c.x * a.x + c.y * a.y + d.x * b.x + d.y * b.y);
        }
    }

    // ---- operands of Q: group c's 32 dims are the words t4 of its four 16-byte chunks, dims 32 c + 8 t4 + nibble
    uint32_t bq[kKv4Groups][4], qs_hi, qs_lo;
    {
        const __half2 up = __float2half2_rn(4.f), down = __float2half2_rn(0.25f);
        float own = 0.f;  // sum of q over the 32 dims of group t4, for head g: the factor of lo
#pragma unroll
        for (int c = 0; c < kKv4Groups; c++) {
            const uint4 w = *reinterpret_cast<const uint4 *>(&sm.q[g][32 * c + 8 * t4]);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint32_t lo = j == 0 ? w.x : w.y, hi = j == 0 ? w.z : w.w;  // nibbles 2 j, 2 j + 1 and those four further on
                const uint32_t e = __byte_perm(lo, hi, 0x5410), f = __byte_perm(lo, hi, 0x7632);
                const __half2 r1 = __hmul2(*reinterpret_cast<const __half2 *>(&f), down);                 // of n1: 4 q1 / 16
                const __half2 c0 = __hfma2(*reinterpret_cast<const __half2 *>(&e), up, __hneg2(r1));  // of n0: 4 (q0 - q1 / 16)
                bq[c][2 * j] = *reinterpret_cast<const uint32_t *>(&c0);
                bq[c][2 * j + 1] = *reinterpret_cast<const uint32_t *>(&r1);
                const float2 fc = __half22float2(c0), fr = __half22float2(r1);
                sum += 0.25f * (fc.x + fc.y) + 4.25f * (fr.x + fr.y);  // q0 + q1 as the operands have them
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (c == t4) own = sum;
        }
        // as two halves, high and low part, in the operand's places of lo (the other places belong to d and count 0)
        const __half hi = __float2half_rn(own);
        const __half2 h2 = __halves2half2(__ushort_as_half(0), hi);
        const __half2 l2 = __halves2half2(__ushort_as_half(0), __float2half_rn(own - __half2float(hi)));
        qs_hi = *reinterpret_cast<const uint32_t *>(&h2);
        qs_lo = *reinterpret_cast<const uint32_t *>(&l2);
    }

    // Per lane: reference maximum (replicated over g) and partial sum of heads 2 t4 and 2 t4 + 1; outputs o[2c] = dims
    // 32 c + 4 g (n0) and + 1 (n0 + 16 n1), o[2c + 1] = dims + 2 and + 3, each for the two heads; om = the part of lo, group
    // g & 3.
    // The reference lies kUp + 1 under a maximum (base 2) and stays until one exceeds it by kUp + 2, so that few tiles have
    // outputs to rescale; probabilities are then at most 2^(kUp + 2) = 2^13.  Their products with d are operands in half
    // precision, and below 2^-14 a half loses bits, below 2^-25 all of them: a key would count as the least value of its
    // group.  So the outputs o are kept times 2^b: d takes the factor where b > 0, which is exact, the probabilities where
    // b < 0.  b stays while the largest d of a tile's visible rows, times 2^b, lies between 2^-6 and 4 (V rows whose groups
    // span 0.25 to 60: b = 0, and nothing is multiplied), and goes back into [1/2, 1) or below 4 when it does not.  Products
    // are then below 2^15, and normal halves for every row whose probability times d is above 2^-19 of the largest d times P,
    // with P the probability that lies kUp above the reference, which some key seen exceeds twofold; where b < 0, the
    // probabilities themselves lose bits below 2^(-25 - b) P (b >= -12).
    float m0 = -INFINITY, m1 = -INFINITY;
    int b_exp = 0;
    uint64_t l01 = 0;  // (two zeros)
    float o[2 * kKv4Groups][4], om[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2 * kKv4Groups; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    bool late = false;  // a wait ran out
    for (int t = ta + warp; t < tb; t += kWarps) {
        if (!__all_sync(0xffffffffu, wait_bar(k_bar, uint32_t(used) & 1u))) {
            late = true;
            break;
        }
        const int r0 = 64 * ((rg.j0 >> 6) + t - extra);
        const int r_lo = t < extra ? 0 : max(rg.j0 - r0, 0), r_hi = t < extra ? rg.n_first : min(pc.pos - r0, 64);
        const bool edge = r_lo > 0 || r_hi < 64;

        // S^T (64 keys x 8 heads)
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t ra[4], rb[4], ga[4], gb[4];
            ldmatrix_x4(ra, k_at + i * 16 * kKv4RowBytes);
            ldmatrix_x4(rb, k_at + (i * 16 + 8) * kKv4RowBytes);
            lds128(ga, kg_at + i * 256);
            lds128(gb, kg_at + i * 256 + 128);
            float lo[4];
            {
                const uint32_t oa = lds32(kg_at + i * 256 + 4 * t4), ob = lds32(kg_at + i * 256 + 128 + 4 * t4);
                const uint32_t a[4] = {oa, ob, oa, ob};
                mma_16816_new(lo, a, qs_hi, qs_lo);
            }
#pragma unroll
            for (int c = 0; c < kKv4Groups; c++) {
                float acc[4];
                const Codes x = split_codes(ra[c]), y = split_codes(rb[c]);
                const uint32_t a0[4] = {x.n0, y.n0, x.n01, y.n01}, a1[4] = {x.n2, y.n2, x.n23, y.n23};
                mma_16816_new(acc, a0, bq[c][0], bq[c][1]);
                mma_16816(acc, a1, bq[c][2], bq[c][3]);
                const float da = low_half(ga[c]), db = low_half(gb[c]);
                s[i][0] = c == 0 ? da * acc[0] : fmaf(da, acc[0], s[i][0]);
                s[i][1] = c == 0 ? da * acc[1] : fmaf(da, acc[1], s[i][1]);
                s[i][2] = c == 0 ? db * acc[2] : fmaf(db, acc[2], s[i][2]);
                s[i][3] = c == 0 ? db * acc[3] : fmaf(db, acc[3], s[i][3]);
            }
            fma2(s[i][0], s[i][1], two22, lo[0], lo[1]);
            fma2(s[i][2], s[i][3], two22, lo[2], lo[3]);
        }
        if (edge) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int ka = 16 * i + g, kb = ka + 8;
                if (ka < r_lo || ka >= r_hi) s[i][0] = s[i][1] = -INFINITY;
                if (kb < r_lo || kb >= r_hi) s[i][2] = s[i][3] = -INFINITY;
            }
        }
        __syncwarp();  // the whole warp is done with the K part
        if (lane == 0 && t + kWarps < tb) load_part(t + kWarps, 0);

        // running maximum (each block has a key that the query sees, so it gets finite), probabilities
        float mx0 = max3(fmaxf(s[0][0], s[0][2]), max3(s[1][0], s[1][2], s[2][0]), max3(s[2][2], s[3][0], s[3][2]));
        float mx1 = max3(fmaxf(s[0][1], s[0][3]), max3(s[1][1], s[1][3], s[2][1]), max3(s[2][3], s[3][1], s[3][3]));
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
        }
        constexpr float kUp = 11.f;
        if (__any_sync(0xffffffffu, mx0 > m0 + (kUp + 2.f) || mx1 > m1 + (kUp + 2.f))) {
            const float n0 = mx0 > m0 + (kUp + 2.f) ? mx0 - (kUp + 1.f) : m0, n1 = mx1 > m1 + (kUp + 2.f) ? mx1 - (kUp + 1.f) : m1;
            const float c0 = fast_exp2(m0 - n0), c1 = fast_exp2(m1 - n1);
            l01 = mul2(l01, pack2(c0, c1));
#pragma unroll
            for (int i = 0; i < 2 * kKv4Groups; i++) {
                o[i][0] *= c0; o[i][1] *= c1; o[i][2] *= c0; o[i][3] *= c1;
            }
            om[0] *= c0;
            om[1] *= c1;
            m0 = n0;
            m1 = n1;
        }
        const uint64_t m01 = pack2(m0, m1);
        uint32_t pb[4][2];  // P^T as the B operand: keys 2 t4, 2 t4 + 1 (and + 8) of the 16, head g
#pragma unroll
        for (int i = 0; i < 4; i++) {
            sub2(s[i][0], s[i][1], m01);
            sub2(s[i][2], s[i][3], m01);
            const float p0 = fast_exp2(s[i][0]), p1 = fast_exp2(s[i][1]), p2 = fast_exp2(s[i][2]), p3 = fast_exp2(s[i][3]);
            add2(l01, p0, p1);
            add2(l01, p2, p3);
            pb[i][0] = movmatrix_trans(pack_half2(p0, p1));
            pb[i][1] = movmatrix_trans(pack_half2(p2, p3));
        }
        if (!__all_sync(0xffffffffu, wait_bar(v_bar, uint32_t(used) & 1u))) {
            late = true;
            break;
        }
        used++;
        auto seen = [&](int r) {  // rows r and r + 1, as a mask of their halves
            return (r >= r_lo && r < r_hi ? 0xffffu : 0u) | (r + 1 >= r_lo && r + 1 < r_hi ? 0xffff0000u : 0u);
        };
        {  // the largest d: a lane looks at two rows, a maximum passes over NaN
            uint32_t w[4];
            lds128(w, v_tile + (kKv4VGroups - kHalf) + lane * 32);
            uint32_t top = as_u32(__hmax2(__hmax2(__hmax2(as_half2(w[0]), as_half2(w[1])), __hmax2(as_half2(w[2]), as_half2(w[3]))), as_half2(0u)));
            if (edge) top &= seen(2 * lane);
            top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
            const int e = int(top >> 10);  // d is in [2^(e - 15), 2^(e - 14)), for e = 0 below
            if (top != 0 && (e + b_exp < 9 || e + b_exp > 16)) {
                const int to = e + b_exp > 16 ? 16 - e : 14 - e;
                const float c = __int_as_float((127 + to - b_exp) << 23);
#pragma unroll
                for (int i = 0; i < 2 * kKv4Groups; i++) {
                    o[i][0] *= c; o[i][1] *= c; o[i][2] *= c; o[i][3] *= c;
                }
                b_exp = to;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t pb0 = pb[i][0], pb1 = pb[i][1];
            uint32_t ps0 = pb0, ps1 = pb1;  // those that meet d
            uint32_t da[4], db[4];
            // d and lo of rows 16 i + 2 t4 and the next, and of those 8 rows on
            lds128(da, vg_at + i * 256);
            lds128(db, vg_at + i * 256 + 128);
            uint32_t la = lds32(vg_at + i * 256 + 16 + 4 * (g & 3)), lb = lds32(vg_at + i * 256 + 144 + 4 * (g & 3));
            if (edge) {  // rows that the query does not see may hold anything: their d and lo count 0
                const int ka = 16 * i + 2 * t4;
                const uint32_t va = seen(ka), vb = seen(ka + 8);
#pragma unroll
                for (int c = 0; c < kKv4Groups; c++) {
                    da[c] &= va;
                    db[c] &= vb;
                }
                la &= va;
                lb &= vb;
            }
            if (b_exp != 0) {
                const uint32_t fd = uint32_t(15 + max(b_exp, 0)) * 0x04000400u, fp = uint32_t(15 + min(b_exp, 0)) * 0x04000400u;  // powers of two
                ps0 = mul_half2(ps0, fp);
                ps1 = mul_half2(ps1, fp);
#pragma unroll
                for (int c = 0; c < kKv4Groups; c++) {
                    da[c] = mul_half2(da[c], fd);
                    db[c] = mul_half2(db[c], fd);
                }
            }
            {
                const uint32_t a[4] = {la, 0u, lb, 0u};
                mma_16816(om, a, pb0, pb1);
            }
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {  // two chunks (groups) of the 16 rows: rows 0-7 and 8-15 of each
                uint32_t w[4];
                ldmatrix_x4_trans(w, (v_at ^ (hf * 32)) + i * 16 * kKv4RowBytes);
#pragma unroll
                for (int q2 = 0; q2 < 2; q2++) {
                    const int c = 2 * hf + q2;
                    const uint32_t b0v = mul_half2(ps0, da[c]), b1v = mul_half2(ps1, db[c]);
                    const Codes x = split_codes(w[2 * q2]), y = split_codes(w[2 * q2 + 1]);
                    const uint32_t a0[4] = {x.n0, x.n01, y.n0, y.n01}, a1[4] = {x.n2, x.n23, y.n2, y.n23};
                    mma_16816(o[2 * c], a0, b0v, b1v);
                    mma_16816(o[2 * c + 1], a1, b0v, b1v);
                }
            }
        }
        __syncwarp();  // the whole warp is done with the V part
        if (lane == 0 && t + kWarps < tb) load_part(t + kWarps, 1);
    }
    if (__syncthreads_or(late)) {  // (and every warp is through with its V part: they become the merge buffer)
        if (tid == 0 && p.error_flag) atomicExch(p.error_flag, 4);
        if (lane == 0)
            for (int i = 0; i < 4; i++) wait_bar(i & 1 ? v_bar : k_bar, uint32_t(i >> 1) & 1u);
        return;
    }
    float l0, l1;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(l0), "=f"(l1) : "l"(l01));
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, off);
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    }
    if (g == 0) {
        sm.red_m[warp][2 * t4] = m0; sm.red_m[warp][2 * t4 + 1] = m1;
        sm.red_l[warp][2 * t4] = l0; sm.red_l[warp][2 * t4 + 1] = l1;
    }
    const float k0 = __int_as_float((127 + 24 - b_exp) << 23), k1 = __int_as_float((127 + 20 - b_exp) << 23);  // 2^24 / 2^b, and 2^20 / 2^b for the differences
#pragma unroll
    for (int c = 0; c < kKv4Groups; c++) {
        const float lo0 = __shfl_sync(0xffffffffu, om[0], 4 * c + t4), lo1 = __shfl_sync(0xffffffffu, om[1], 4 * c + t4);
        const float *e = o[2 * c], *f = o[2 * c + 1];
        *reinterpret_cast<float4 *>(&sm.o[warp][2 * t4][32 * c + 4 * g]) =
            make_float4(fmaf(e[0], k0, lo0), fmaf(e[2] - e[0], k1, lo0), fmaf(f[0], k0, lo0), fmaf(f[2] - f[0], k1, lo0));
        *reinterpret_cast<float4 *>(&sm.o[warp][2 * t4 + 1][32 * c + 4 * g]) =
            make_float4(fmaf(e[1], k0, lo1), fmaf(e[3] - e[1], k1, lo1), fmaf(f[1], k0, lo1), fmaf(f[3] - f[1], k1, lo1));
    }
    __syncthreads();

    // ---- merge of the warps and the new token: a lane owns four dims of each of the warp's heads
    const int n_split = pc.n_split, split = pc.split, rec0 = pc.part0 * kNHeadKv + kvh;  // this KV head's records: every fourth
    const size_t out_row = size_t(p.tok0 + pc.tok) * kQDim;
#pragma unroll
    for (int i = 0; i < kHeads; i++) {
        if (!has_heads) break;
        const int h = warp * kHeads + i, head = kvh * kGqa + h;
        float M = s_new[i];
#pragma unroll
        for (int w = 0; w < kWarps; w++) M = fmaxf(M, sm.red_m[w][h]);
        float L = ends ? fast_exp2(s_new[i] - M) : 0.f, A[4] = {0.f, 0.f, 0.f, 0.f};
        if (ends) {
            const uint2 hv = *reinterpret_cast<const uint2 *>(&sm.vnew[d0]);
            const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&hv.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&hv.y));
            A[0] = L * a.x; A[1] = L * a.y; A[2] = L * b.x; A[3] = L * b.y;
        }
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float lw = sm.red_l[w][h];
            const float c = lw == 0.f ? 0.f : fast_exp2(sm.red_m[w][h] - M);  // (a warp without a tile: m = -inf, l = 0)
            const float4 x = *reinterpret_cast<const float4 *>(&sm.o[w][h][d0]);
            L += lw * c;
            A[0] += x.x * c; A[1] += x.y * c; A[2] += x.z * c; A[3] += x.w * c;
        }
        if (n_split == 1) {
            const float sink2 = sm.sinks[head] * kLog2e;
            const float Mf = fmaxf(M, sink2), cf = fast_exp2(M - Mf);
            const float inv = cf / (L * cf + fast_exp2(sink2 - Mf));
            store_out4(p.out, p.out_dtype, out_row + head * kHeadDim + d0, A[0] * inv, A[1] * inv, A[2] * inv, A[3] * inv);
        } else {  // this piece's record: acc, m (base 2), l
            float *rec = p.scratch + (size_t(rec0 + split * kNHeadKv) * kGqa + h) * kRecStride;
            *reinterpret_cast<float4 *>(rec + d0) = make_float4(A[0], A[1], A[2], A[3]);
            if (lane == 0) *reinterpret_cast<float2 *>(rec + kHeadDim) = make_float2(M, L);
        }
    }
    if (n_split == 1 || !has_heads) return;

    // ---- split-K, per query head: a warp that has written its record of a head counts it; the one that finds itself the last of
    // its run of records merges the run, and if that was the last run of the head, the runs.  (The record's stores are ordered
    // before lane 0's ticket by the warp's barrier; the ticket is an acquire-release atomic at device scope, cumulative over
    // them; the readers go past L1.)
    const int fan = dec4_fan(n_split), sub = split / fan, n_sub = (n_split + fan - 1) / fan, n = min(fan, n_split - sub * fan);
    int arrived[kHeads];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kHeads; i++)
        if (lane == 0) arrived[i] = ticket_acq_rel(&p.tickets[(rec0 + sub * kNHeadKv) * kGqa + warp * kHeads + i]);
    __syncwarp();  // lane 0's tickets come before the other lanes' reads
#pragma unroll
    for (int i = 0; i < kHeads; i++) {
        const int h = warp * kHeads + i, head = kvh * kGqa + h;
        auto record = [&](float *base, int k) { return base + (size_t(rec0 + k * kNHeadKv) * kGqa + h) * kRecStride; };
        if (__shfl_sync(0xffffffffu, arrived[i], 0) != n - 1) continue;
        if (lane == 0) p.tickets[(rec0 + sub * kNHeadKv) * kGqa + h] = 0;  // ready for the next launch
        Merged4 r = merge_records4([&](int k) { return record(p.scratch, sub * fan + k); }, n, d0);
        if (n_sub > 1) {
            float *rec = record(p.scratch2, sub);
            *reinterpret_cast<float4 *>(rec + d0) = make_float4(r.a[0], r.a[1], r.a[2], r.a[3]);
            if (lane == 0) *reinterpret_cast<float2 *>(rec + kHeadDim) = make_float2(r.M, r.L);
            __syncwarp();
            int last = 0;
            int *ticket = &p.tickets2[rec0 * kGqa + h];
            if (lane == 0) {
                last = ticket_acq_rel(ticket) == n_sub - 1;
                if (last) *ticket = 0;
            }
            __syncwarp();
            if (!__shfl_sync(0xffffffffu, last, 0)) continue;
            r = merge_records4([&](int k) { return record(p.scratch2, k); }, n_sub, d0);
        }
        const float sink2 = sm.sinks[head] * kLog2e;
        const float Mf = fmaxf(r.M, sink2), cf = fast_exp2(r.M - Mf);
        const float inv = cf / (r.L * cf + fast_exp2(sink2 - Mf));
        store_out4(p.out, p.out_dtype, out_row + head * kHeadDim + d0, r.a[0] * inv, r.a[1] * inv, r.a[2] * inv, r.a[3] * inv);
    }
}

template <int kCap>
struct Dec4List {
    Dec4Piece pieces[kCap];
};

template <int kCap, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, 16 / kWarps)
    k_decode_kv4(const __grid_constant__ Dec4Params p, const __grid_constant__ Dec4List<kCap> list) {
    decode_piece<kWarps>(p, list.pieces[blockIdx.x >> 2], int(blockIdx.x & 3));
}

// The parameter block is copied at every launch, so the kernel comes in three capacities and a launch takes the smallest
// that fits (the smallest one stays inside the classic 4 KiB parameter space).
constexpr int kSmallPieces = 160, kMidPieces = 512;
static_assert(sizeof(Dec4Params) + sizeof(Dec4List<kSmallPieces>) <= 4096, "small variant");
static_assert(sizeof(Dec4Params) + sizeof(Dec4List<kDec4MaxPieces>) <= 32764, "largest variant fits the limit");

template <int kCap, int kWarps>
cudaError_t launch_list(const Dec4Params &p, const Dec4Piece *pieces, int n_pieces, cudaStream_t stream) {
    static thread_local Dec4List<kCap> list;  // copied into the launch by the runtime before this returns
    memcpy(list.pieces, pieces, sizeof(Dec4Piece) * size_t(n_pieces));
    return launch_pdl(k_decode_kv4<kCap, kWarps>, n_pieces * kNHeadKv, kWarps * 32, sizeof(Dec4Smem<kWarps>), stream, p, list);
}

template <int kCap, int kWarps>
cudaError_t setup_list() { return allow_smem(k_decode_kv4<kCap, kWarps>, sizeof(Dec4Smem<kWarps>)); }

}  // namespace

cudaError_t decode_kv4_setup() {
    cudaError_t e = setup_list<kSmallPieces, 16>();
    if (e == cudaSuccess) e = setup_list<kSmallPieces, 8>();
    if (e == cudaSuccess) e = setup_list<kMidPieces, 8>();
    if (e == cudaSuccess) e = setup_list<kDec4MaxPieces, 8>();
    if (e == cudaSuccess) e = setup_list<kMidPieces, 4>();
    if (e == cudaSuccess) e = setup_list<kDec4MaxPieces, 4>();
    return e;
}

cudaError_t launch_decode_kv4(const Dec4Params &p, const Dec4Piece *pieces, int n_pieces, int n_warps, cudaStream_t stream) {
    if (n_pieces <= 0) return cudaSuccess;
    if (n_pieces > kDec4MaxPieces) return cudaErrorInvalidValue;
    // (sixteen warps only where the launch leaves half of the GPU idle, four only where it has several rounds: see the plan)
    if (n_warps == 16 && n_pieces <= kSmallPieces) return launch_list<kSmallPieces, 16>(p, pieces, n_pieces, stream);
    if (n_warps >= 8 && n_pieces <= kSmallPieces) return launch_list<kSmallPieces, 8>(p, pieces, n_pieces, stream);
    if (n_warps == 8 && n_pieces <= kMidPieces) return launch_list<kMidPieces, 8>(p, pieces, n_pieces, stream);
    if (n_warps == 8) return launch_list<kDec4MaxPieces, 8>(p, pieces, n_pieces, stream);
    if (n_pieces <= kMidPieces) return launch_list<kMidPieces, 4>(p, pieces, n_pieces, stream);
    return launch_list<kDec4MaxPieces, 4>(p, pieces, n_pieces, stream);
}

}  // namespace flint
