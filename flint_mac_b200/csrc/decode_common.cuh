// Pieces the decode kernels share: mbarriers, the norm / rotation of a head row, output stores, the merge of split-K
// records, and the launch with the work list in the kernel's parameters.
#pragma once

#include <cstdlib>

#include "attn_common.h"
#include "ptx.cuh"

namespace flint {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.b32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded: gives up after ~2^28 SM cycles, far beyond anything a healthy launch needs.
__device__ __forceinline__ bool mbar_wait_bounded(uint32_t bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; i++)
            if (mbar_try_wait(bar, parity)) return true;
        if (clock64() - t0 > (1ll << 28)) return false;
    }
}
// sin and cos of a float angle of any size.  The angle is brought into [-pi, pi] in double first (exact to ~1e-11 for
// the 1e5-radian angles of a 131072-token context), which keeps sincosf off its long-argument path: that path alone
// cost the CTAs of such a context about two microseconds before their first tile could be used.
__device__ __forceinline__ void sincos_reduced(float x, float *sn, float *cs) {
    const double xd = double(x);
    const double k = rint(xd * 0.15915494309189535);
    double r = fma(-k, 6.283185307179586, xd);
    r = fma(-k, 2.4492935982947064e-16, r);
    sincosf(float(r), sn, cs);
}

__device__ __forceinline__ float4 load_row4(const void *base, int dtype, size_t elem0, int lane) {
    if (dtype == kDtypeF32) return reinterpret_cast<const float4 *>(static_cast<const float *>(base) + elem0)[lane];
    const uint2 u = reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(base) + elem0)[lane];
    const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162 *>(&u.x);
    const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162 *>(&u.y);
    return make_float4(__low2float(a), __high2float(a), __low2float(b), __high2float(b));
}

// One 128-wide head row spread over a warp, lane owning dims 4*lane..4*lane+3: RMSNorm with weight, then NEOX RoPE
// pairing dim i with i+64, i.e. lane with lane^16 (same arithmetic as src/ref/ref_model.cpp:45-61).  cs/sn hold
// cos/sin of pos * inv_freq[4*(lane&15) .. +3], computed once per CTA.
__device__ __forceinline__ float4 norm_rope(float4 v, float4 wv, float4 cs, float4 sn, int lane, bool rope) {
    const float ss = warp_sum(v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w);
    const float scale = 1.0f / sqrtf(ss / kHeadDim + kRmsEps);
    v.x = v.x * scale * wv.x;
    v.y = v.y * scale * wv.y;
    v.z = v.z * scale * wv.z;
    v.w = v.w * scale * wv.w;
    if (!rope) return v;
    const float x[4] = {v.x, v.y, v.z, v.w}, c[4] = {cs.x, cs.y, cs.z, cs.w}, sv[4] = {sn.x, sn.y, sn.z, sn.w};
    float out[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float partner = __shfl_xor_sync(0xffffffffu, x[j], 16);
        out[j] = lane < 16 ? x[j] * c[j] - partner * sv[j] : partner * sv[j] + x[j] * c[j];
    }
    return make_float4(out[0], out[1], out[2], out[3]);
}

__device__ __forceinline__ void store_half4(__half *dst, float4 v) {
    const uint2 u = make_uint2(pack_half2(v.x, v.y), pack_half2(v.z, v.w));
    *reinterpret_cast<uint2 *>(dst) = u;
}

__device__ __forceinline__ void store_out(void *out, int dtype, size_t idx, float v) {
    if (dtype == kDtypeF32) static_cast<float *>(out)[idx] = v;
    else static_cast<__nv_bfloat16 *>(out)[idx] = __float2bfloat16_rn(v);
}

// 8 consecutive outputs of one head as one or two 16-byte stores.
__device__ __forceinline__ void store_out8(void *out, int dtype, size_t idx, const float (&v)[8]) {
    if (dtype == kDtypeF32) {
        float4 *dst = reinterpret_cast<float4 *>(static_cast<float *>(out) + idx);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t *>(&b);
        }
        *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(out) + idx) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

struct Merged {
    float M, L;
    float a[8];
};

// Takes a ticket: returns the old count.  Acquire-release at device scope (see the split-K merge).
__device__ __forceinline__ int ticket_acq_rel(int *counter) {
    int old;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;\n" : "=r"(old) : "l"(counter) : "memory");
    return old;
}

// Fold n partial records of one head (fused.metal:332-350) into the running state (M, L, a): M = max m_s,
// L = sum l_s e^(m_s - M), a = sum acc_s e^(m_s - M); the sink enters as a record with m = sink, l = 1, acc = 0.
// `rec` points at record 0 of this thread's head; consecutive records of the same head are kGqa * kRecStride floats
// apart.  The thread owns dims [d0, d0 + 8).  Eight records per trip: their 24 loads are in flight together (a trip costs about a microsecond), and
// the loop stays small -- this code runs once per group, from a cold instruction cache, so its size is its cost.
__device__ __forceinline__ Merged merge_records(const float *rec, int n, int d0, bool with_sink, float sink) {
    constexpr int kStep = kGqa * kRecStride;
    constexpr int kTrip = 8;  // records per round trip to L2
    Merged r;
    float M = with_sink ? sink : -INFINITY, L = with_sink ? 1.f : 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) r.a[j] = 0.f;
#pragma unroll 1
    for (int s0 = 0; s0 < n; s0 += kTrip) {
        float2 ml[kTrip];
        float4 x[kTrip], y[kTrip];
#pragma unroll
        for (int i = 0; i < kTrip; i++) {
            const float *q = rec + size_t(min(s0 + i, n - 1)) * kStep;  // past the end: re-read the last one, unused
            ml[i] = __ldcg(reinterpret_cast<const float2 *>(q + kHeadDim));
            x[i] = __ldcg(reinterpret_cast<const float4 *>(q + d0));
            y[i] = __ldcg(reinterpret_cast<const float4 *>(q + d0 + 4));
            if (s0 + i >= n) ml[i] = make_float2(-INFINITY, 0.f);
        }
        float cm = M;
#pragma unroll
        for (int i = 0; i < kTrip; i++) cm = fmaxf(cm, ml[i].x);
        const float keep = M == -INFINITY ? 0.f : __expf(M - cm);
        L *= keep;
#pragma unroll
        for (int j = 0; j < 8; j++) r.a[j] *= keep;
        M = cm;
#pragma unroll
        for (int i = 0; i < kTrip; i++) {
            // an empty part has m = -inf, l = 0 (fused.metal:344)
            const float c = ml[i].y == 0.f ? 0.f : __expf(ml[i].x - M);
            L += ml[i].y * c;
            r.a[0] += x[i].x * c; r.a[1] += x[i].y * c; r.a[2] += x[i].z * c; r.a[3] += x[i].w * c;
            r.a[4] += y[i].x * c; r.a[5] += y[i].y * c; r.a[6] += y[i].z * c; r.a[7] += y[i].w * c;
        }
    }
    r.M = M;
    r.L = L;
    return r;
}

// The work list either sits in device memory (any length) or, when it is short enough, travels in the kernel's
// parameter space (large kernel parameters, up to 32 KiB): one wave on a 148-SM part is ~300 items of 48 bytes, so the
// usual launch needs no host-to-device copy in front of it.  The parameter block is copied by the driver at every
// launch, so the kernel comes in three capacities and a launch takes the smallest that fits (the smallest one stays
// inside the classic 4 KiB parameter space).
template <int kCap>
struct DecItemsParam {
    DecItem items[kCap];
};

constexpr int kCapSmall = 76, kCapMid = 304;  // 304: one wave of items on a 148-SM part (two CTAs per SM) and a little more

// Launch with programmatic stream serialization: the kernel may be scheduled before its predecessor in the stream
// has finished (it waits inside, see decode_item), which hides launch latency between the short kernels of a decode
// step.  FLINT_ATTN_NO_PDL=1 in the environment turns it off.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, int n_threads, size_t smem_bytes,
                       cudaStream_t stream, const Args &...args) {
    static const bool off = [] {
        const char *v = getenv("FLINT_ATTN_NO_PDL");
        return v && v[0] == '1';
    }();
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(n_threads));
    cfg.dynamicSmemBytes = smem_bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = off ? 0 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename K>
inline cudaError_t allow_smem(K kernel, size_t bytes) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
}

}  // namespace flint
