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
// The codes go to the tensor cores as they are: a nibble masked out of a 16-bit lane is the half-precision number
// c * 2^-24 (or c * 2^-20 for the second nibble: the lane holds c * 16 subnormal steps), which the products take exactly.
// Q is stored for the first and second nibbles with factors 4 and 1/4, so that both come out as q c 2^-22; outputs of
// the second nibbles are 16 times too large and are put right at the end.  That is 5 logical operations for 8 codes.
// On the K side d multiplies the 32-dim partial scores (4 groups per key), on the V side it multiplies the
// probabilities (4 operand pairs per 16 keys), and lo enters through one more product each.
//
// A warp works on whole blocks of 64 positions by itself, the four warps of a CTA on every fourth one; a block is one
// 10 KB bulk copy on the warp's own mbarrier.
#include <cstring>

#include "decode_common.cuh"
#include "kv4.cuh"

namespace flint {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 2;       // blocks of a warp in flight or in use
constexpr int kORow = kHeadDim + 4;  // floats between heads of the merge buffer: the eight lanes of a store hit different banks
constexpr uint32_t kNib0 = 0x000f000fu, kNib1 = 0x00f000f0u;

struct __align__(128) Dec4Smem {
    unsigned char tile[kWarps][kStages][kKv4BlockBytes];
    alignas(8) unsigned long long full_bar[kWarps][kStages];
    alignas(16) __half q[kGqa][kHeadDim];  // normalised, rotated, scaled by log2(e) / sqrt(128)
    float red_m[kWarps][kGqa], red_l[kWarps][kGqa], s_new[kGqa];
    alignas(16) __half knew[kHeadDim];
    alignas(16) __half vnew[kHeadDim];
    alignas(16) float rope_cos[kHeadDim / 2], rope_sin[kHeadDim / 2];
    int is_last;
};
// The per-warp outputs are merged through the (by then idle) tiles.
static_assert(sizeof(float) * kWarps * kGqa * kORow <= sizeof(Dec4Smem::tile), "merge buffer aliases the tiles");

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
__device__ __forceinline__ float low_half(uint32_t a) { return __low2float(*reinterpret_cast<const __half2 *>(&a)); }

__device__ __forceinline__ void decode_item(const Dec4Params &p, const DecItem &it) {
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Dec4Smem &sm = *reinterpret_cast<Dec4Smem *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int mh = tid >> 4, md = (tid & 15) * 8;
    const int head = it.kvh * kGqa + mh;
    const float sink = p.sinks[head];
    const bool rope = p.has_rope != 0;
    const bool fold_k = it.fold && warp == 0, fold_v = it.fold && warp == 1;
    const float4 wq = reinterpret_cast<const float4 *>(p.q_norm)[lane];
    float4 wk = wq;
    if (fold_k) wk = reinterpret_cast<const float4 *>(p.k_norm)[lane];
    float freq = 0.f;
    if (rope && tid < kHeadDim / 2) freq = p.inv_freq[tid];
    // the cached keys, 64 positions at a time: the block of first tokens if some lie before the window, then the range
    const int n_first = p.is_swa ? min(p.cache.first_tokens, it.j0) : 0;
    const int extra = n_first > 0 ? 1 : 0, b0 = it.j0 >> 6;
    const int n_tiles = extra + (it.j1 > it.j0 ? ((it.j1 + 63) >> 6) - b0 : 0);
    const uint32_t tiles = smem_u32(&sm.tile[warp][0][0]), bars = smem_u32(&sm.full_bar[warp][0]);
    auto load_tile = [&](int t, int stage) {  // one lane
        const unsigned char *block = t < extra ? kv4_first_block(p.cache, it.seq, it.kvh)
                                               : kv4_block(p.cache, it.seq, it.kvh, b0 + t - extra);
        mbar_expect_tx(bars + 8 * stage, kKv4BlockBytes);
        bulk_load(tiles + stage * kKv4BlockBytes, block, kKv4BlockBytes, bars + 8 * stage);
    };
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kStages; i++) mbar_init(bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    // Nothing an earlier kernel of the stream produces (rows, cache contents, split-K records and counters) is read or
    // written before this wait.
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kStages; i++)
            if (warp + i * kWarps < n_tiles) load_tile(warp + i * kWarps, i);
    }

    // ---- prologue: the group's q heads, and the new token's k and v
    const size_t row0 = size_t(it.tok) * kQkvDim;
    float4 q[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        q[i] = load_row4(p.qkv, p.qkv_dtype, row0 + size_t(it.kvh * kGqa + warp * 2 + i) * kHeadDim, lane);
    float4 kv_new = make_float4(0.f, 0.f, 0.f, 0.f);
    if (fold_k) kv_new = load_row4(p.qkv, p.qkv_dtype, row0 + kQDim + size_t(it.kvh) * kHeadDim, lane);
    if (fold_v) kv_new = load_row4(p.qkv, p.qkv_dtype, row0 + kQDim + kKvDim + size_t(it.kvh) * kHeadDim, lane);
    const float qscale = rsqrtf(float(kHeadDim)) * kLog2e;  // softmax runs in base 2
    if (rope && tid < kHeadDim / 2) {
        float sn, cs;
        sincos_reduced(float(it.pos) * freq, &sn, &cs);
        sm.rope_cos[tid] = cs;
        sm.rope_sin[tid] = sn;
    }
    __syncthreads();
    float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
    if (rope) {
        cs = reinterpret_cast<const float4 *>(sm.rope_cos)[lane & 15];
        sn = reinterpret_cast<const float4 *>(sm.rope_sin)[lane & 15];
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        q[i] = norm_rope(q[i], wq, cs, sn, lane, rope);
        q[i].x *= qscale; q[i].y *= qscale; q[i].z *= qscale; q[i].w *= qscale;
        store_half4(&sm.q[warp * 2 + i][4 * lane], q[i]);
    }
    if (fold_k || fold_v) {
        if (fold_k) kv_new = norm_rope(kv_new, wk, cs, sn, lane, rope);
        const uint2 h = make_uint2(pack_half2(kv_new.x, kv_new.y), pack_half2(kv_new.z, kv_new.w));
        *reinterpret_cast<uint2 *>(fold_k ? &sm.knew[4 * lane] : &sm.vnew[4 * lane]) = h;
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&h.y));
        const float x[4] = {a.x, a.y, b.x, b.y};
        kv4_store_lane(kv4_block(p.cache, it.seq, it.kvh, it.pos >> 6), it.pos & 63, fold_v, lane, x);
        if (p.is_swa && it.pos < p.cache.first_tokens)
            kv4_store_lane(kv4_first_block(p.cache, it.seq, it.kvh), it.pos, fold_v, lane, x);
    }
    __syncthreads();
    if (it.fold) {
        const uint2 h = *reinterpret_cast<const uint2 *>(&sm.knew[4 * lane]);
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&h.y));
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float s = warp_sum(q[i].x * a.x + q[i].y * a.y + q[i].z * b.x + q[i].w * b.y);
            if (lane == 0) sm.s_new[warp * 2 + i] = s;
        }
    }

    // ---- operands of Q: group c's 32 dims are the words t4 of its four 16-byte chunks, dims 32 c + 8 t4 + nibble
    const int g = lane >> 2, t4 = lane & 3;
    uint32_t bq[kKv4Groups][4], qs_hi, qs_lo;
    {
        const __half2 up = __float2half2_rn(4.f), down = __float2half2_rn(0.25f);
        float own = 0.f;  // sum of q over the 32 dims of group t4, for head g: the factor of lo
#pragma unroll
        for (int c = 0; c < kKv4Groups; c++) {
            const uint4 w = *reinterpret_cast<const uint4 *>(&sm.q[g][32 * c + 8 * t4]);
            const uint32_t pair[4] = {__byte_perm(w.x, w.z, 0x5410), __byte_perm(w.x, w.z, 0x7632),   // nibbles 0 4, 1 5
                                      __byte_perm(w.y, w.w, 0x5410), __byte_perm(w.y, w.w, 0x7632)};  // nibbles 2 6, 3 7
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const __half2 v = *reinterpret_cast<const __half2 *>(&pair[j]);
                const __half2 r = __hmul2(v, (j & 1) ? down : up);
                bq[c][j] = *reinterpret_cast<const uint32_t *>(&r);
                const float2 f = __half22float2(v);
                sum += f.x + f.y;
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
    // 32 c + 4 g and + 1, o[2c + 1] = dims + 2 and + 3, each for the two heads; om = the part of lo, group g & 3.
    // The reference lies 2 under the maximum (base 2), so that probabilities times d keep two more bits above half's
    // subnormal steps; d is at most 8736, so four times that still fits a half.
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float o[2 * kKv4Groups][4], om[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2 * kKv4Groups; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    bool late = false;
    int waited = 0;
    for (int t = warp, k = 0; t < n_tiles; t += kWarps, k++) {
        const int stage = k % kStages;
        waited = k + 1;
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(bars + 8 * stage, uint32_t(k / kStages) & 1u))) {
            late = true;
            break;
        }
        const uint32_t tile = tiles + stage * kKv4BlockBytes;
        const int r0 = 64 * (b0 + t - extra);
        const int r_lo = t < extra ? 0 : max(it.j0 - r0, 0), r_hi = t < extra ? n_first : min(it.j1 - r0, 64);
        const bool edge = r_lo > 0 || r_hi < 64;

        // S^T (64 keys x 8 heads)
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t ra[4], rb[4], ga[4], gb[4];
            const int row = 16 * i + (lane & 7), ch = (lane >> 3) ^ ((row >> 1) & 3);
            ldmatrix_x4(ra, tile + kKv4KCodes + row * kKv4RowBytes + ch * 16);
            ldmatrix_x4(rb, tile + kKv4KCodes + (row + 8) * kKv4RowBytes + ch * 16);  // ((row + 8) >> 1 & 3 is the same)
            lds128(ga, tile + kKv4KGroups + (16 * i + g) * 16);
            lds128(gb, tile + kKv4KGroups + (16 * i + g + 8) * 16);
            const uint32_t oa = lds32(tile + kKv4KGroups + (16 * i + g) * 16 + 4 * t4);
            const uint32_t ob = lds32(tile + kKv4KGroups + (16 * i + g + 8) * 16 + 4 * t4);
            float lo[4] = {0.f, 0.f, 0.f, 0.f};
            {
                const uint32_t a[4] = {oa, ob, oa, ob};
                mma_16816(lo, a, qs_hi, qs_lo);
            }
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < kKv4Groups; c++) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t x = ra[c], y = rb[c];
                const uint32_t a0[4] = {x & kNib0, y & kNib0, x & kNib1, y & kNib1};
                mma_16816(acc, a0, bq[c][0], bq[c][1]);
                x >>= 8;
                y >>= 8;
                const uint32_t a1[4] = {x & kNib0, y & kNib0, x & kNib1, y & kNib1};
                mma_16816(acc, a1, bq[c][2], bq[c][3]);
                const float da = low_half(ga[c]), db = low_half(gb[c]);
                sum[0] = fmaf(da, acc[0], sum[0]);
                sum[1] = fmaf(da, acc[1], sum[1]);
                sum[2] = fmaf(db, acc[2], sum[2]);
                sum[3] = fmaf(db, acc[3], sum[3]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) s[i][j] = fmaf(sum[j], 4194304.f, lo[j]);
            if (edge) {
                const int ka = 16 * i + g, kb = ka + 8;
                if (ka < r_lo || ka >= r_hi) s[i][0] = s[i][1] = -INFINITY;
                if (kb < r_lo || kb >= r_hi) s[i][2] = s[i][3] = -INFINITY;
            }
        }

        // running maximum (each block has a key that the query sees, so it gets finite), probabilities
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            mx0 = fmaxf(mx0, fmaxf(s[i][0], s[i][2]));
            mx1 = fmaxf(mx1, fmaxf(s[i][1], s[i][3]));
        }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
        }
        mx0 -= 2.f;
        mx1 -= 2.f;
        if (__any_sync(0xffffffffu, mx0 > m0 || mx1 > m1)) {
            const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
            const float c0 = fast_exp2(m0 - n0), c1 = fast_exp2(m1 - n1);
            l0 *= c0;
            l1 *= c1;
#pragma unroll
            for (int i = 0; i < 2 * kKv4Groups; i++) {
                o[i][0] *= c0; o[i][1] *= c1; o[i][2] *= c0; o[i][3] *= c1;
            }
            om[0] *= c0;
            om[1] *= c1;
            m0 = n0;
            m1 = n1;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float p0 = fast_exp2(s[i][0] - m0), p1 = fast_exp2(s[i][1] - m1);
            const float p2 = fast_exp2(s[i][2] - m0), p3 = fast_exp2(s[i][3] - m1);
            l0 += p0 + p2;
            l1 += p1 + p3;
            // P^T as the B operand: keys 2 t4, 2 t4 + 1 (and + 8) of the 16, head g
            const uint32_t pb0 = movmatrix_trans(pack_half2(p0, p1)), pb1 = movmatrix_trans(pack_half2(p2, p3));
            uint32_t da[4], db[4];
            const uint32_t pair = tile + kKv4VGroups + (8 * i + t4) * 32;  // rows 16 i + 2 t4 and the next; + 8: 128 bytes on
            lds128(da, pair);
            lds128(db, pair + 128);
            uint32_t la = lds32(pair + 16 + 4 * (g & 3)), lb = lds32(pair + 128 + 16 + 4 * (g & 3));
            if (edge) {  // rows that the query does not see may hold anything: their d and lo count 0
                const int ka = 16 * i + 2 * t4;
                auto seen = [&](int r) {
                    return (r >= r_lo && r < r_hi ? 0xffffu : 0u) | (r + 1 >= r_lo && r + 1 < r_hi ? 0xffff0000u : 0u);
                };
                const uint32_t va = seen(ka), vb = seen(ka + 8);
#pragma unroll
                for (int c = 0; c < kKv4Groups; c++) {
                    da[c] &= va;
                    db[c] &= vb;
                }
                la &= va;
                lb &= vb;
            }
            {
                const uint32_t a[4] = {la, 0u, lb, 0u};
                mma_16816(om, a, pb0, pb1);
            }
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {  // two chunks (groups) of the 16 rows: rows 0-7 and 8-15 of each
                uint32_t w[4];
                const int j = lane >> 3, row = 16 * i + (j & 1) * 8 + (lane & 7), ch = (2 * hf + (j >> 1)) ^ ((row >> 1) & 3);
                ldmatrix_x4_trans(w, tile + kKv4VCodes + row * kKv4RowBytes + ch * 16);
#pragma unroll
                for (int q2 = 0; q2 < 2; q2++) {
                    const int c = 2 * hf + q2;
                    const uint32_t b0v = mul_half2(pb0, da[c]), b1v = mul_half2(pb1, db[c]);
                    uint32_t x = w[2 * q2], y = w[2 * q2 + 1];
                    const uint32_t a0[4] = {x & kNib0, x & kNib1, y & kNib0, y & kNib1};
                    mma_16816(o[2 * c], a0, b0v, b1v);
                    x >>= 8;
                    y >>= 8;
                    const uint32_t a1[4] = {x & kNib0, x & kNib1, y & kNib0, y & kNib1};
                    mma_16816(o[2 * c + 1], a1, b0v, b1v);
                }
            }
        }
        __syncwarp();  // the whole warp is done with the stage
        if (lane == 0 && t + kStages * kWarps < n_tiles) {
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // order the reads above before the next copy
            load_tile(t + kStages * kWarps, stage);
        }
    }
    if (late) {  // a copy never came: wait (bounded) for the others in flight before the CTA's memory goes back
        for (int k = waited; warp + k * kWarps < n_tiles && k < waited - 1 + kStages; k++)
            mbar_wait_bounded(bars + 8 * (k % kStages), uint32_t(k / kStages) & 1u);
    }
    if (__syncthreads_or(late)) {  // (and every warp is done with its tiles: they become the merge buffer)
        if (tid == 0 && p.error_flag) atomicExch(p.error_flag, 4);
        return;
    }
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, off);
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    }
    float *obuf = reinterpret_cast<float *>(&sm.tile[0][0][0]);  // [warp][head][kORow]
    if (g == 0) {
        sm.red_m[warp][2 * t4] = m0; sm.red_m[warp][2 * t4 + 1] = m1;
        sm.red_l[warp][2 * t4] = l0; sm.red_l[warp][2 * t4 + 1] = l1;
    }
#pragma unroll
    for (int c = 0; c < kKv4Groups; c++) {
        constexpr float k0 = 16777216.f, k1 = 1048576.f;  // 2^24 and, for the second nibbles, 2^20
        const float lo0 = __shfl_sync(0xffffffffu, om[0], 4 * c + t4), lo1 = __shfl_sync(0xffffffffu, om[1], 4 * c + t4);
        float *row0 = obuf + (warp * kGqa + 2 * t4) * kORow + 32 * c + 4 * g;
        const float *e = o[2 * c], *f = o[2 * c + 1];
        *reinterpret_cast<float4 *>(row0) = make_float4(fmaf(e[0], k0, lo0), fmaf(e[2], k1, lo0), fmaf(f[0], k0, lo0), fmaf(f[2], k1, lo0));
        *reinterpret_cast<float4 *>(row0 + kORow) =
            make_float4(fmaf(e[1], k0, lo1), fmaf(e[3], k1, lo1), fmaf(f[1], k0, lo1), fmaf(f[3], k1, lo1));
    }
    __syncthreads();

    // ---- merge with the new token; a thread owns 8 dims of one head from here on
    const bool direct = it.n_split == 1;
    {
        const float s_new = it.fold ? sm.s_new[mh] : -INFINITY;
        float M = s_new;
#pragma unroll
        for (int w = 0; w < kWarps; w++) M = fmaxf(M, sm.red_m[w][mh]);
        const float cn = it.fold ? fast_exp2(s_new - M) : 0.f;
        float L = cn, A[8];
#pragma unroll
        for (int j = 0; j < 8; j++) A[j] = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float lw = sm.red_l[w][mh];
            const float c = lw == 0.f ? 0.f : fast_exp2(sm.red_m[w][mh] - M);  // (a warp without a block: m = -inf, l = 0)
            const float4 x = *reinterpret_cast<const float4 *>(obuf + (w * kGqa + mh) * kORow + md);
            const float4 y = *reinterpret_cast<const float4 *>(obuf + (w * kGqa + mh) * kORow + md + 4);
            L += lw * c;
            A[0] += x.x * c; A[1] += x.y * c; A[2] += x.z * c; A[3] += x.w * c;
            A[4] += y.x * c; A[5] += y.y * c; A[6] += y.z * c; A[7] += y.w * c;
        }
        if (it.fold) {
#pragma unroll
            for (int j = 0; j < 8; j++) A[j] = fmaf(cn, __half2float(sm.vnew[md + j]), A[j]);
        }
        if (direct) {
            const float sink2 = sink * kLog2e;
            const float Mf = fmaxf(M, sink2), cf = fast_exp2(M - Mf);
            const float inv = cf / (L * cf + fast_exp2(sink2 - Mf));
#pragma unroll
            for (int j = 0; j < 8; j++) A[j] *= inv;
            store_out8(p.out, p.out_dtype, size_t(it.tok) * kQDim + head * kHeadDim + md, A);
            return;
        }
        float *rec = p.scratch + ((size_t(it.part0) + it.split) * kGqa + mh) * kRecStride;
        *reinterpret_cast<float4 *>(rec + md) = make_float4(A[0], A[1], A[2], A[3]);
        *reinterpret_cast<float4 *>(rec + md + 4) = make_float4(A[4], A[5], A[6], A[7]);
        if (md == 0) { rec[kHeadDim] = M * kLn2; rec[kHeadDim + 1] = L; }
    }

    // ---- split-K merge by the last CTA of the group, in two levels (the half-precision kernel has the reasons)
    const int sub = it.split / kMergeFan, n_sub = (it.n_split + kMergeFan - 1) / kMergeFan;
    const int sub_size = min(kMergeFan, it.n_split - sub * kMergeFan);
    __syncthreads();
    if (tid == 0) {
        const bool last = ticket_acq_rel(&p.tickets[it.sub0 + sub]) == sub_size - 1;
        if (last) p.tickets[it.sub0 + sub] = 0;
        sm.is_last = last;
    }
    __syncthreads();
    if (!sm.is_last) return;
    const float *src = p.scratch + ((size_t(it.part0) + sub * kMergeFan) * kGqa + mh) * kRecStride;
    int n_src = sub_size;
    bool final_level = n_sub == 1;
    Merged r;
    for (;;) {
        r = merge_records(src, n_src, md, final_level, sink);
        if (final_level) break;
        float *rec2 = p.scratch2 + ((size_t(it.sub0) + sub) * kGqa + mh) * kRecStride;
        *reinterpret_cast<float4 *>(rec2 + md) = make_float4(r.a[0], r.a[1], r.a[2], r.a[3]);
        *reinterpret_cast<float4 *>(rec2 + md + 4) = make_float4(r.a[4], r.a[5], r.a[6], r.a[7]);
        if (md == 0) { rec2[kHeadDim] = r.M; rec2[kHeadDim + 1] = r.L; }
        __syncthreads();
        if (tid == 0) {
            const bool last = ticket_acq_rel(&p.tickets2[it.group]) == n_sub - 1;
            if (last) p.tickets2[it.group] = 0;
            sm.is_last = last;
        }
        __syncthreads();
        if (!sm.is_last) return;
        src = p.scratch2 + (size_t(it.sub0) * kGqa + mh) * kRecStride;
        n_src = n_sub;
        final_level = true;
    }
    const float inv = 1.0f / r.L;
#pragma unroll
    for (int j = 0; j < 8; j++) r.a[j] *= inv;
    store_out8(p.out, p.out_dtype, size_t(it.tok) * kQDim + head * kHeadDim + md, r.a);
}

__global__ void __launch_bounds__(kThreads, 2) k_decode_kv4(const Dec4Params p) {
    const DecItem it = p.items[blockIdx.x];
    decode_item(p, it);
}

template <int kCap>
__global__ void __launch_bounds__(kThreads, 2)
    k_decode_kv4_p(const __grid_constant__ Dec4Params p, const __grid_constant__ DecItemsParam<kCap> ip) {
    const DecItem it = ip.items[blockIdx.x];
    decode_item(p, it);
}

template <int kCap>
cudaError_t launch_inline(const Dec4Params &p, const DecItem *host_items, int n_items, cudaStream_t stream) {
    static thread_local DecItemsParam<kCap> ip;  // copied into the launch by the runtime before this returns
    memcpy(ip.items, host_items, sizeof(DecItem) * size_t(n_items));
    return launch_pdl(k_decode_kv4_p<kCap>, n_items, kThreads, sizeof(Dec4Smem), stream, p, ip);
}

}  // namespace

cudaError_t decode_kv4_setup() {
    cudaError_t e = allow_smem(k_decode_kv4, sizeof(Dec4Smem));
    if (e == cudaSuccess) e = allow_smem(k_decode_kv4_p<kCapSmall>, sizeof(Dec4Smem));
    if (e == cudaSuccess) e = allow_smem(k_decode_kv4_p<kCapMid>, sizeof(Dec4Smem));
    if (e == cudaSuccess) e = allow_smem(k_decode_kv4_p<kMaxParamItems>, sizeof(Dec4Smem));
    return e;
}

cudaError_t launch_decode_kv4(const Dec4Params &p, const DecItem *inline_items, int n_items, cudaStream_t stream) {
    if (n_items <= 0) return cudaSuccess;
    if (!inline_items) return launch_pdl(k_decode_kv4, n_items, kThreads, sizeof(Dec4Smem), stream, p);
    if (n_items > kMaxParamItems) return cudaErrorInvalidValue;
    if (n_items <= kCapSmall) return launch_inline<kCapSmall>(p, inline_items, n_items, stream);
    if (n_items <= kCapMid) return launch_inline<kCapMid>(p, inline_items, n_items, stream);
    return launch_inline<kMaxParamItems>(p, inline_items, n_items, stream);
}

}  // namespace flint
