// Rows of K and V in and out of a layer's cache on the device (4-bit caches, and half-precision ones).
#include "decode_common.cuh"
#include "kv4.cuh"

namespace flint {

namespace {

// Four neighbouring values of a row of `dtype`, as floats / stored.
__device__ __forceinline__ float4 row_load4(const void *base, int dtype, size_t elem) {
    if (dtype == kDtypeF32) return *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + elem);
    const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(base) + elem);
    if (dtype == kDtypeF16) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ void row_store4(void *base, int dtype, size_t elem, float4 v) {
    if (dtype == kDtypeF32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(base) + elem) = v;
        return;
    }
    uint2 u;
    if (dtype == kDtypeF16) {
        u = make_uint2(pack_half2(v.x, v.y), pack_half2(v.z, v.w));
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        u = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(base) + elem) = u;
}

// Element offset of a position's row in a half-precision cache; -1: no such row here.
__device__ __forceinline__ long long half_row(const KvRowsParams &p, int seq, int kvh, int pos) {
    if (p.cache.block_table) {
        const int page = p.cache.block_table[size_t(seq) * p.cache.table_stride + (pos >> 6)];
        return page < 0 ? -1 : ((long long)(page * kNHeadKv + kvh) * kPageKeys + (pos & (kPageKeys - 1))) * kHeadDim;
    }
    const int slot = p.is_swa ? pos & (kSwaRing - 1) : pos;
    return (((long long)seq * kNHeadKv + kvh) * p.n_slots + slot) * kHeadDim;
}

// One warp per (sequence, row, KV head): K's row, then V's.
__global__ void __launch_bounds__(256) k_kv_store(const KvRowsParams p, const __grid_constant__ KvRowsSeqs seqs, int n) {
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (w >= (long long)n * p.n_rows * kNHeadKv) return;
    const int kvh = int(w % kNHeadKv), r = int(w / kNHeadKv % p.n_rows), i = int(w / kNHeadKv / p.n_rows);
    const int seq = seqs.seq[i], pos = seqs.pos0[i] + r;
    // positions r and r + 1024 of one call share a slot of a ring: only the last one of a slot is stored, whatever the order
    // in which the warps run
    const bool to_ring = !p.is_swa || p.raw_slots || r + kSwaRing >= p.n_rows;
    const bool raw_first = p.is_swa && p.raw_slots && pos >= kSwaRing;
    const bool to_first = p.is_swa && !p.raw_slots && pos < p.cache.first_tokens;
    const size_t at = size_t(i) * p.seq_stride + size_t(kvh) * p.head_stride + size_t(r) * kHeadDim + 4 * lane;
    if (!to_ring && !to_first) return;
#pragma unroll
    for (int is_v = 0; is_v < 2; is_v++) {
        const float4 f = row_load4(is_v ? p.v : p.k, p.dtype, at);
        const uint2 h = make_uint2(pack_half2(f.x, f.y), pack_half2(f.z, f.w));
        if (!p.cache.blocks) {
            *reinterpret_cast<uint2 *>((is_v ? p.v_cache : p.k_cache) + half_row(p, seq, kvh, pos) + 4 * lane) = h;
            continue;
        }
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&h.y));
        const float x[4] = {a.x, a.y, b.x, b.y};
        if (to_ring) {
            unsigned char *block = raw_first ? kv4_first_block(p.cache, seq, kvh) : kv4_block(p.cache, seq, kvh, pos >> 6);
            kv4_store_lane(block, pos & 63, is_v, lane, x);
        }
        if (to_first) kv4_store_lane(kv4_first_block(p.cache, seq, kvh), pos, is_v, lane, x);
    }
}

__global__ void __launch_bounds__(256) k_kv_load(const KvRowsParams p, const __grid_constant__ KvRowsSeqs seqs, int n) {
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (w >= (long long)n * p.n_rows * kNHeadKv) return;
    const int kvh = int(w % kNHeadKv), r = int(w / kNHeadKv % p.n_rows), i = int(w / kNHeadKv / p.n_rows);
    const int seq = seqs.seq[i], pos = seqs.pos0[i] + r;
    const bool first = p.is_swa && (p.raw_slots ? pos >= kSwaRing : pos < p.cache.first_tokens);
    const size_t at = size_t(i) * p.seq_stride + size_t(kvh) * p.head_stride + size_t(r) * kHeadDim + 4 * lane;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.cache.blocks) {
        const unsigned char *block = first ? kv4_first_block(p.cache, seq, kvh) : kv4_block(p.cache, seq, kvh, pos >> 6);
        row_store4(p.k, p.dtype, at, block ? kv4_load_lane(block, pos & 63, false, lane) : zero);
        row_store4(p.v, p.dtype, at, block ? kv4_load_lane(block, pos & 63, true, lane) : zero);
    } else {
        const long long row = half_row(p, seq, kvh, pos);
        row_store4(p.k, p.dtype, at, row < 0 ? zero : row_load4(p.k_cache, kDtypeF16, size_t(row) + 4 * lane));
        row_store4(p.v, p.dtype, at, row < 0 ? zero : row_load4(p.v_cache, kDtypeF16, size_t(row) + 4 * lane));
    }
}

}  // namespace

// The SM's memory is split as the decode kernel wants it: a kernel in between that wants another split makes the next one wait
// for the SMs to be set up again.
cudaError_t kv_rows_setup() {
    cudaError_t e = cudaFuncSetAttribute(k_kv_store, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_kv_load, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    return e;
}

cudaError_t launch_kv_store(const KvRowsParams &p, const KvRowsSeqs &seqs, int n, cudaStream_t stream) {
    const long long warps = (long long)n * p.n_rows * kNHeadKv;
    if (warps <= 0) return cudaSuccess;
    return launch_pdl(k_kv_store, int((warps + 7) / 8), 256, 0, stream, p, seqs, n);
}

cudaError_t launch_kv_load(const KvRowsParams &p, const KvRowsSeqs &seqs, int n, cudaStream_t stream) {
    const long long warps = (long long)n * p.n_rows * kNHeadKv;
    if (warps <= 0) return cudaSuccess;
    return launch_pdl(k_kv_load, int((warps + 7) / 8), 256, 0, stream, p, seqs, n);
}

}  // namespace flint
