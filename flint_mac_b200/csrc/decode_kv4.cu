// Decode attention over K/V caches held in 4 bits (format: kv4.h), full layers and sliding-window layers whose first
// tokens stay visible.
//
// With x = lo + c d per group, scores and outputs of one query head are
//   s_j = sum_i q_i (lo_j + c_ji d_j),   O = sum_j p_j (lo_j + c_j d_j) / (e^sink + sum_j p_j),   p_j = e^(s_j)
// over the keys j that the query sees: [0, pos) on a full layer, [pos - 512, pos) and the first tokens [0, F) on a
// sliding-window layer, and the token itself.  The token itself enters at half precision, as its own record of the final
// merge; its row is quantised into the cache by the same launch.
#include <cstring>

#include "decode_common.cuh"
#include "kv4.cuh"

namespace flint {

namespace {

constexpr int kThreads = 128;

struct __align__(128) Dec4Smem {
    float q[kGqa][kHeadDim];  // normalised, rotated, pre-scaled by log2(e) / sqrt(128)
    float o[kGqa][kHeadDim + 4];
    float p[kGqa][kKv4BlockKeys];
    float corr[kGqa], red_m[kGqa], red_l[kGqa], s_new[kGqa];
    alignas(16) __half knew[kHeadDim];
    alignas(16) __half vnew[kHeadDim];
    float rope_cos[kHeadDim / 2], rope_sin[kHeadDim / 2];
    int is_last;
};

__device__ __forceinline__ void decode_item(const Dec4Params &p, const DecItem &it) {
    __shared__ Dec4Smem sm;
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
    asm volatile("griddepcontrol.wait;\n" ::: "memory");

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
        *reinterpret_cast<float4 *>(&sm.q[warp * 2 + i][4 * lane]) = q[i];
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
    if (tid < kGqa) {
        sm.red_m[tid] = -INFINITY;
        sm.red_l[tid] = 0.f;
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

    // ---- the cached keys, 64 positions at a time: the block of first tokens if some lie before the window, then the range
    const int n_first = p.is_swa ? min(p.cache.first_tokens, it.j0) : 0;
    const int extra = n_first > 0 ? 1 : 0, b0 = it.j0 >> 6;
    const int n_tiles = extra + (it.j1 > it.j0 ? ((it.j1 + 63) >> 6) - b0 : 0);
    float o[kGqa];
#pragma unroll
    for (int h = 0; h < kGqa; h++) o[h] = 0.f;
    for (int t = 0; t < n_tiles; t++) {
        const int b = b0 + t - extra;
        const bool is_first = t < extra;
        const unsigned char *block = is_first ? kv4_first_block(p.cache, it.seq, it.kvh) : kv4_block(p.cache, it.seq, it.kvh, b);
        const int r_lo = is_first ? 0 : max(it.j0 - 64 * b, 0), r_hi = is_first ? n_first : min(it.j1 - 64 * b, 64);
        {   // scores: two threads a key, 64 dims each
            const int r = tid >> 1, hf = tid & 1;
            float s[kGqa];
#pragma unroll
            for (int h = 0; h < kGqa; h++) s[h] = 0.f;
            for (int g = 2 * hf; g < 2 * hf + 2; g++) {
                const float2 dl = __half22float2(*reinterpret_cast<const __half2 *>(block + kv4_k_group(r, g)));
                const uint4 c4 = *reinterpret_cast<const uint4 *>(block + kKv4KCodes + kv4_chunk(r, g));
                const uint32_t w[4] = {c4.x, c4.y, c4.z, c4.w};
                for (int i = 0; i < 32; i++) {
                    const float x = fmaf(float((w[i >> 3] >> (4 * (i & 7))) & 15), dl.x, dl.y);
#pragma unroll
                    for (int h = 0; h < kGqa; h++) s[h] = fmaf(x, sm.q[h][32 * g + i], s[h]);
                }
            }
#pragma unroll
            for (int h = 0; h < kGqa; h++) {
                s[h] += __shfl_xor_sync(0xffffffffu, s[h], 1);
                if (hf == 0) sm.p[h][r] = r >= r_lo && r < r_hi ? s[h] : -INFINITY;
            }
        }
        __syncthreads();
        for (int h = 2 * warp; h < 2 * warp + 2; h++) {  // two heads a warp: running maximum and sum
            const float s0 = sm.p[h][lane], s1 = sm.p[h][lane + 32];
            float mx = fmaxf(s0, s1);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const float m = sm.red_m[h], mn = fmaxf(m, mx), c = fast_exp2(m - mn);  // (at least one key of the tile is seen)
            const float p0 = fast_exp2(s0 - mn), p1 = fast_exp2(s1 - mn);
            sm.p[h][lane] = p0;
            sm.p[h][lane + 32] = p1;
            const float l = warp_sum(p0 + p1);
            if (lane == 0) {
                sm.corr[h] = c;
                sm.red_m[h] = mn;
                sm.red_l[h] = sm.red_l[h] * c + l;
            }
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < kGqa; h++) o[h] *= sm.corr[h];
        const int g = tid >> 5, nib = tid & 31;  // thread = dim
        for (int r = r_lo; r < r_hi; r++) {
            const uint32_t c = block[kKv4VCodes + kv4_chunk(r, g) + (nib >> 1)] >> (4 * (nib & 1)) & 15;
            const float d = __half2float(*reinterpret_cast<const __half *>(block + kv4_v_group(r, g)));
            const float lo = __half2float(*reinterpret_cast<const __half *>(block + kv4_v_group(r, g) + 16));
            const float x = fmaf(float(c), d, lo);
#pragma unroll
            for (int h = 0; h < kGqa; h++) o[h] = fmaf(sm.p[h][r], x, o[h]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int h = 0; h < kGqa; h++) sm.o[h][tid] = o[h];
    __syncthreads();

    // ---- merge with the new token; a thread owns 8 dims of one head from here on
    const bool direct = it.n_split == 1;
    {
        const float s_new = it.fold ? sm.s_new[mh] : -INFINITY;
        const float M = fmaxf(sm.red_m[mh], s_new);
        const float c = sm.red_l[mh] == 0.f ? 0.f : fast_exp2(sm.red_m[mh] - M);
        const float cn = it.fold ? fast_exp2(s_new - M) : 0.f;
        float L = sm.red_l[mh] * c + cn, A[8];
#pragma unroll
        for (int j = 0; j < 8; j++) A[j] = sm.o[mh][md + j] * c;
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

__global__ void __launch_bounds__(kThreads) k_decode_kv4(const Dec4Params p) {
    const DecItem it = p.items[blockIdx.x];
    decode_item(p, it);
}

template <int kCap>
__global__ void __launch_bounds__(kThreads)
    k_decode_kv4_p(const __grid_constant__ Dec4Params p, const __grid_constant__ DecItemsParam<kCap> ip) {
    const DecItem it = ip.items[blockIdx.x];
    decode_item(p, it);
}

template <int kCap>
cudaError_t launch_inline(const Dec4Params &p, const DecItem *host_items, int n_items, cudaStream_t stream) {
    static thread_local DecItemsParam<kCap> ip;  // copied into the launch by the runtime before this returns
    memcpy(ip.items, host_items, sizeof(DecItem) * size_t(n_items));
    return launch_pdl(k_decode_kv4_p<kCap>, n_items, kThreads, 0, stream, p, ip);
}

}  // namespace

cudaError_t decode_kv4_setup() { return cudaSuccess; }

cudaError_t launch_decode_kv4(const Dec4Params &p, const DecItem *inline_items, int n_items, cudaStream_t stream) {
    if (n_items <= 0) return cudaSuccess;
    if (!inline_items) return launch_pdl(k_decode_kv4, n_items, kThreads, 0, stream, p);
    if (n_items > kMaxParamItems) return cudaErrorInvalidValue;
    if (n_items <= kCapSmall) return launch_inline<kCapSmall>(p, inline_items, n_items, stream);
    if (n_items <= kCapMid) return launch_inline<kCapMid>(p, inline_items, n_items, stream);
    return launch_inline<kMaxParamItems>(p, inline_items, n_items, stream);
}

}  // namespace flint
