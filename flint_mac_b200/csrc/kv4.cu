// Rows of K and V in and out of a layer's cache on the device (4-bit caches, and half-precision ones).
#include <climits>

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
__device__ __forceinline__ long long half_row(const KvRowsParams &p, int seq, int kvh, int pos, int held) {
    if (p.cache.block_table) {
        if ((pos >> 6) >= held) return -1;
        const int page = p.cache.block_table[size_t(seq) * p.cache.table_stride + (pos >> 6)];
        return page < 0 ? -1 : ((long long)(page * kNHeadKv + kvh) * kPageKeys + (pos & (kPageKeys - 1))) * kHeadDim;
    }
    const int slot = p.is_swa ? pos & (kSwaRing - 1) : pos;
    return (((long long)seq * kNHeadKv + kvh) * p.n_slots + slot) * kHeadDim;
}

// Element offset of one of the first tokens' rows beside a half-precision ring.
__device__ __forceinline__ size_t half_first_row(int seq, int kvh, int pos) {
    return ((size_t(seq) * kNHeadKv + kvh) * kMaxFirstTokens + pos) * kHeadDim;
}

// ---- half-precision caches: one warp per (sequence, row, KV head).  Bound by memory: 131071 rows of one sequence from half
// (537 MB read and written) are stored in 115 us and read back in 118, 0.72 and 0.70 of a copy's rate (one or two loads in
// flight a lane); 16384 rows in 14.2 and 12.9 us (their bytes 10.4), 64 rows in 4.2 and 4.0.
__global__ void __launch_bounds__(256) k_half_store(const KvRowsParams p, const __grid_constant__ KvRowsSeqs seqs, int n) {
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // (after the wait: see the prefill prologue)
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (w >= (long long)n * p.n_rows * kNHeadKv) return;
    const int kvh = int(w % kNHeadKv), r = int(w / kNHeadKv % p.n_rows), i = int(w / kNHeadKv / p.n_rows);
    // positions r and r + 1024 of one call share a slot of a ring: only the last one of a slot is stored, whatever the order
    // in which the warps run
    const size_t at = size_t(i) * p.seq_stride + size_t(kvh) * p.head_stride + size_t(r) * kHeadDim + 4 * lane;
    if (p.is_swa && seqs.pos0[i] + r < p.cache.first_tokens) {
        const size_t to = half_first_row(seqs.seq[i], kvh, seqs.pos0[i] + r) + 4 * lane;
        row_store4(p.first_k, kDtypeF16, to, row_load4(p.k, p.dtype, at));
        row_store4(p.first_v, kDtypeF16, to, row_load4(p.v, p.dtype, at));
    }
    if (p.is_swa && r + kSwaRing < p.n_rows) return;
    const long long row = half_row(p, seqs.seq[i], kvh, seqs.pos0[i] + r, seqs.held[i]);
    row_store4(p.k_cache, kDtypeF16, size_t(row) + 4 * lane, row_load4(p.k, p.dtype, at));
    row_store4(p.v_cache, kDtypeF16, size_t(row) + 4 * lane, row_load4(p.v, p.dtype, at));
}

__global__ void __launch_bounds__(256) k_half_load(const KvRowsParams p, const __grid_constant__ KvRowsSeqs seqs, int n) {
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // (after the wait: see the prefill prologue)
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (w >= (long long)n * p.n_rows * kNHeadKv) return;
    const int kvh = int(w % kNHeadKv), r = int(w / kNHeadKv % p.n_rows), i = int(w / kNHeadKv / p.n_rows);
    const size_t at = size_t(i) * p.seq_stride + size_t(kvh) * p.head_stride + size_t(r) * kHeadDim + 4 * lane;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.staging) {  // first tokens of a prefill
        const size_t from = half_first_row(seqs.seq[i], kvh, seqs.pos0[i] + r) + 4 * lane;
        uint2 k = *reinterpret_cast<const uint2 *>(p.first_k + from), v = *reinterpret_cast<const uint2 *>(p.first_v + from);
        half_row_staged(k, v);
        *reinterpret_cast<uint2 *>(static_cast<__half *>(p.k) + at) = k;
        *reinterpret_cast<uint2 *>(static_cast<__half *>(p.v) + at) = v;
        return;
    }
    if (p.is_swa && seqs.pos0[i] + r < p.cache.first_tokens) {
        const size_t from = half_first_row(seqs.seq[i], kvh, seqs.pos0[i] + r) + 4 * lane;
        row_store4(p.k, p.dtype, at, row_load4(p.first_k, kDtypeF16, from));
        row_store4(p.v, p.dtype, at, row_load4(p.first_v, kDtypeF16, from));
        return;
    }
    const long long row = half_row(p, seqs.seq[i], kvh, seqs.pos0[i] + r, seqs.held[i]);
    row_store4(p.k, p.dtype, at, row < 0 ? zero : row_load4(p.k_cache, kDtypeF16, size_t(row) + 4 * lane));
    row_store4(p.v, p.dtype, at, row < 0 ? zero : row_load4(p.v_cache, kDtypeF16, size_t(row) + 4 * lane));
}

// ---- 4-bit caches: one CTA per (sequence, KV head, block of 64 positions), so that a block's codes are written or read by
// one CTA.  Eight neighbouring values a lane (one 16-byte access in half precision, four bytes of codes): 16 lanes a row,
// four lanes a group, two neighbouring rows a warp; a thread's loads are all in flight before the first is used.
// Loading is bound by memory: 131071 rows of one sequence to half (84 MB read, 268 MB written) take 57.0 us, 6.2 TB/s or
// 0.95 of a copy's rate.
constexpr int kRowThreads = 256;
constexpr int kRowSteps = kKv4BlockKeys * 16 / kRowThreads;  // rows of a lane in a block

template <int kType>
struct Eight;  // eight values of a row as they lie in memory
template <>
struct Eight<kDtypeF32> {
    float4 a, b;
    __device__ __forceinline__ void load(const void *base, size_t elem) {
        a = __ldcs(reinterpret_cast<const float4 *>(static_cast<const float *>(base) + elem));
        b = __ldcs(reinterpret_cast<const float4 *>(static_cast<const float *>(base) + elem) + 1);
    }
    // the values, rounded to half
    __device__ __forceinline__ uint4 get() const {
        return make_uint4(pack_half2(a.x, a.y), pack_half2(a.z, a.w), pack_half2(b.x, b.y), pack_half2(b.z, b.w));
    }
    template <bool>
    static __device__ __forceinline__ void store(void *base, size_t elem, const float (&x)[8]) {
        float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(base) + elem);
        __stcs(p, make_float4(x[0], x[1], x[2], x[3]));
        __stcs(p + 1, make_float4(x[4], x[5], x[6], x[7]));
    }
};
template <>
struct Eight<kDtypeBf16> {
    uint4 a;
    __device__ __forceinline__ void load(const void *base, size_t elem) {
        a = __ldcs(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + elem));
    }
    __device__ __forceinline__ uint4 get() const {
        auto half2_of = [](uint32_t w) { return pack_half2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); };
        return make_uint4(half2_of(a.x), half2_of(a.y), half2_of(a.z), half2_of(a.w));
    }
    template <bool>
    static __device__ __forceinline__ void store(void *base, size_t elem, const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        __stcs(reinterpret_cast<uint4 *>(static_cast<uint16_t *>(base) + elem), make_uint4(w[0], w[1], w[2], w[3]));
    }
};
template <>
struct Eight<kDtypeF16> {
    uint4 a;
    __device__ __forceinline__ void load(const void *base, size_t elem) {
        a = __ldcs(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + elem));
    }
    __device__ __forceinline__ uint4 get() const { return a; }
    // kLimit: values past the largest finite one become it (lo + 15 d can be, by half a step of d, where the row reaches it)
    template <bool kLimit>
    static __device__ __forceinline__ void store(void *base, size_t elem, const float (&x)[8]) {
        auto pack = [](float a, float b) {
            if (!kLimit) return pack_half2(a, b);
            uint32_t h;
            asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;\n" : "=r"(h) : "f"(b), "f"(a));
            return h;
        };
        __stcs(reinterpret_cast<uint4 *>(static_cast<uint16_t *>(base) + elem), make_uint4(pack(x[0], x[1]), pack(x[2], x[3]), pack(x[4], x[5]), pack(x[6], x[7])));
    }
};

// The rows of a block that a call has: positions (slots, when p.raw_slots) p0 .. p0 + n_rows - 1.
struct BlockRows {
    int seq, kvh, first, block;  // first: position of the block's row 0
    size_t base;                 // element of position 0's row in k and v
    int p0, p1;
    __device__ __forceinline__ BlockRows(const KvRowsParams &p, const KvRowsSeqs &seqs) {
        const int i = blockIdx.z;
        kvh = blockIdx.y % kNHeadKv;
        seq = seqs.seq[i];
        p0 = seqs.pos0[i];
        p1 = p0 + p.n_rows;
        block = (p0 >> 6) + int(blockIdx.x);
        first = block * kKv4BlockKeys;
        base = size_t(i) * p.seq_stride + size_t(kvh) * p.head_stride - size_t(p0) * kHeadDim;  // (wraps; added to p0 or more)
    }
    __device__ __forceinline__ bool has(int r) const { return first + r >= p0 && first + r < p1; }
};
// A block by position, or by slot (the first tokens' block follows the ring's).
__device__ __forceinline__ unsigned char *block_of(const KvRowsParams &p, const BlockRows &b) {
    if (!p.raw_slots || p.cache.block_table) return kv4_block(p.cache, b.seq, b.kvh, b.block);
    return p.cache.blocks + ((size_t(b.seq) * kNHeadKv + b.kvh) * p.cache.blocks_per_seq + b.block) * kKv4BlockBytes;
}

// Storing takes most instructions per byte, so a lane has sixteen values here (half a group: one exchange between lanes, d and
// lo worked out by two lanes instead of four: 13.1 instead of 17 us for 16384 rows, 10.4 with whole blocks apart), eight lanes
// a row, and K and V of a block are separate CTAs.  16384 rows of one sequence from half (34 MB read, 10 MB written) take
// 10.0 us: 4.4 TB/s, 0.68 of a copy's rate.  No unit is full (2.6 instructions a cycle of 4, the logical unit 45 %, DRAM 33 %,
// as what is written stays in L2): 2056 CTAs are 2.3 times what the GPU holds, and each waits for its rows once.
constexpr int kStoreSteps = kKv4BlockKeys * 8 / kRowThreads;
template <int kType>
__global__ void __launch_bounds__(kRowThreads, kType == kDtypeF32 ? 4 : 6) k_kv4_store(const KvRowsParams p, const __grid_constant__ KvRowsSeqs seqs) {
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // (after the wait: see the prefill prologue)
    const bool is_v = blockIdx.y >= kNHeadKv;
    const BlockRows b(p, seqs);
    if (b.first >= b.p1) return;
    const int sub = threadIdx.x & 7, g = sub >> 1, r0 = threadIdx.x >> 3;  // rows r0, r0 + 32: a warp has rows 4 i .. 4 i + 3
    const void *src = is_v ? p.v : p.k;
    unsigned char *block = block_of(p, b);
    // positions of one call that share a slot of a ring: only the last one of a slot is stored, whatever the order of CTAs
    const int kept = p.is_swa && !p.raw_slots ? b.p1 - kSwaRing : INT_MIN;
    const bool front = p.is_swa && !p.raw_slots && b.first < p.cache.first_tokens;
    Eight<kType> x[kStoreSteps][2];
    if (!front && b.first >= b.p0 && b.first + kKv4BlockKeys <= b.p1 && b.first >= kept) {  // a whole block: the usual one of a long call
        const size_t at = b.base + size_t(b.first + r0) * kHeadDim + 16 * sub;
#pragma unroll
        for (int i = 0; i < kStoreSteps; i++) {
            x[i][0].load(src, at + i * 32 * kHeadDim);
            x[i][1].load(src, at + i * 32 * kHeadDim + 8);
        }
        // (32 rows further on the chunk's swizzle and the place in the pair are the same)
        unsigned char *codes_at = block + (is_v ? kKv4VCodes : kKv4KCodes) + kv4_chunk(r0, g) + (sub & 1) * 8;
        unsigned char *group_at = block + (is_v ? kv4_v_group(r0 & ~1, g) + (r0 & 1) * 16 : kv4_k_group(r0, g));
#pragma unroll
        for (int i = 0; i < kStoreSteps; i++) {
            uint32_t mine;
            const uint2 codes = kv4_quantise16(x[i][0].get(), x[i][1].get(), mine);
            *reinterpret_cast<uint2 *>(codes_at + i * 32 * kKv4RowBytes) = codes;
            const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 8);
            if (is_v) mine = (r0 & 1) ? __byte_perm(other, mine, 0x7632) : __byte_perm(mine, other, 0x5410);  // {lo, lo} or {d, d} of the pair
            if ((sub & 1) == 0) *reinterpret_cast<uint32_t *>(group_at + i * 32 * 16) = mine;
        }
        return;
    }
    unsigned char *first_block = front ? kv4_first_block(p.cache, b.seq, b.kvh) : nullptr;
#pragma unroll 1
    for (int r = r0; r < kKv4BlockKeys; r += 32) {
        const bool in = b.has(r);
        if (!__any_sync(0xffffffffu, in)) continue;
        uint4 h[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (in) {
            const size_t at = b.base + size_t(b.first + r) * kHeadDim + 16 * sub;
            x[0][0].load(src, at);
            x[0][1].load(src, at + 8);
            h[0] = x[0][0].get();
            h[1] = x[0][1].get();
        }
        uint32_t dl;
        const uint2 codes = kv4_quantise16(h[0], h[1], dl);
        auto put = [&](unsigned char *blk) {
            *reinterpret_cast<uint2 *>(blk + (is_v ? kKv4VCodes : kKv4KCodes) + kv4_chunk(r, g) + (sub & 1) * 8) = codes;
            if ((sub & 1) == 0) kv4_store_group(blk, r, g, is_v, dl);
        };
        if (in && b.first + r >= kept) put(block);
        if (in && first_block && b.first + r < p.cache.first_tokens) put(first_block);
    }
}

// kStaging: see KvRowsParams.
template <int kType, bool kStaging = false>
__global__ void __launch_bounds__(kRowThreads) k_kv4_load(const KvRowsParams p, const __grid_constant__ KvRowsSeqs seqs) {
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // (after the wait: see the prefill prologue)
    const BlockRows b(p, seqs);
    if (b.first >= b.p1) return;
    const int sub = threadIdx.x & 15, r0 = threadIdx.x >> 4, g = sub >> 2;
    const unsigned char *block = p.cache.block_table && b.block >= seqs.held[blockIdx.z] ? nullptr : block_of(p, b);
    const unsigned char *front = p.is_swa && !p.raw_slots && b.first < p.cache.first_tokens ? kv4_first_block(p.cache, b.seq, b.kvh) : nullptr;
    uint32_t kc[kRowSteps], vc[kRowSteps], kg[kRowSteps];
    uint16_t vd[kRowSteps], vl[kRowSteps];
#pragma unroll
    for (int i = 0; i < kRowSteps; i++) {
        const int r = r0 + 16 * i;
        kc[i] = vc[i] = kg[i] = 0;  // (rows on pages that the sequence does not hold read as zeros)
        vd[i] = vl[i] = 0;
        const unsigned char *blk = front && b.first + r < p.cache.first_tokens ? front : block;
        if (!blk || !b.has(r)) continue;
        // (ordinary loads, which the wait above orders behind the stream's earlier kernels: one that writes the block may run
        // beside this grid's beginning, so the block is not read-only for the grid's whole life, as __ldg takes it to be)
        kc[i] = *reinterpret_cast<const uint32_t *>(blk + kKv4KCodes + kv4_chunk(r, g) + (sub & 3) * 4);
        kg[i] = *reinterpret_cast<const uint32_t *>(blk + kv4_k_group(r, g));
        vc[i] = *reinterpret_cast<const uint32_t *>(blk + kKv4VCodes + kv4_chunk(r, g) + (sub & 3) * 4);
        vd[i] = *reinterpret_cast<const uint16_t *>(blk + kv4_v_group(r, g));
        vl[i] = *reinterpret_cast<const uint16_t *>(blk + kv4_v_group(r, g) + 16);
    }
#pragma unroll
    for (int i = 0; i < kRowSteps; i++) {
        const int r = r0 + 16 * i;
        const bool odd = kStaging && (vd[i] & 0x7c00u) == 0x7c00u;  // (the row's sixteen lanes are half a warp)
        const bool bad = kStaging && (__ballot_sync(0xffffffffu, odd) >> (threadIdx.x & 16) & 0xffffu) != 0;
        if (!b.has(r)) continue;
        const size_t at = b.base + size_t(b.first + r) * kHeadDim + 8 * sub;
        float x[8];
        const float2 dl = __half22float2(*reinterpret_cast<const __half2 *>(&kg[i]));
        const float k_lo = bad ? __uint_as_float(0x7fc00000u) : dl.y;
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = fmaf(float((kc[i] >> (4 * j)) & 15u), dl.x, k_lo);
        Eight<kType>::template store<kStaging>(p.k, at, x);
        const float d = odd ? 0.f : __half2float(__ushort_as_half(vd[i])), lo = odd ? 0.f : __half2float(__ushort_as_half(vl[i]));
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = fmaf(float((vc[i] >> (4 * j)) & 15u), d, lo);
        Eight<kType>::template store<kStaging>(p.v, at, x);
    }
}

dim3 block_grid(const KvRowsParams &p, int n, int parts) {  // a range that starts inside a block touches one more
    return dim3(unsigned((p.n_rows + 2 * kKv4BlockKeys - 2) / kKv4BlockKeys), unsigned(kNHeadKv * parts), unsigned(n));
}

}  // namespace

// The SM's memory is split as the decode kernel wants it: a kernel in between that wants another split makes the next one wait
// for the SMs to be set up again.
template <typename K>
cudaError_t max_shared(K kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
}
cudaError_t kv_rows_setup() {
    cudaError_t e = max_shared(k_half_store);
    if (e == cudaSuccess) e = max_shared(k_half_load);
    if (e == cudaSuccess) e = max_shared(k_kv4_store<kDtypeF32>);
    if (e == cudaSuccess) e = max_shared(k_kv4_store<kDtypeBf16>);
    if (e == cudaSuccess) e = max_shared(k_kv4_store<kDtypeF16>);
    if (e == cudaSuccess) e = max_shared(k_kv4_load<kDtypeF32>);
    if (e == cudaSuccess) e = max_shared(k_kv4_load<kDtypeBf16>);
    if (e == cudaSuccess) e = max_shared(k_kv4_load<kDtypeF16>);
    if (e == cudaSuccess) e = max_shared(k_kv4_load<kDtypeF16, true>);
    return e;
}

cudaError_t launch_kv_store(const KvRowsParams &p, const KvRowsSeqs &seqs, int n, cudaStream_t stream) {
    if (n <= 0 || p.n_rows <= 0) return cudaSuccess;
    if (!p.cache.blocks) return launch_pdl(k_half_store, dim3(unsigned(((long long)n * p.n_rows * kNHeadKv + 7) / 8)), 256, 0, stream, p, seqs, n);
    const dim3 grid = block_grid(p, n, 2);
    if (p.dtype == kDtypeF32) return launch_pdl(k_kv4_store<kDtypeF32>, grid, kRowThreads, 0, stream, p, seqs);
    if (p.dtype == kDtypeBf16) return launch_pdl(k_kv4_store<kDtypeBf16>, grid, kRowThreads, 0, stream, p, seqs);
    return launch_pdl(k_kv4_store<kDtypeF16>, grid, kRowThreads, 0, stream, p, seqs);
}

cudaError_t launch_kv_load(const KvRowsParams &p, const KvRowsSeqs &seqs, int n, cudaStream_t stream) {
    if (n <= 0 || p.n_rows <= 0) return cudaSuccess;
    if (!p.cache.blocks) return launch_pdl(k_half_load, dim3(unsigned(((long long)n * p.n_rows * kNHeadKv + 7) / 8)), 256, 0, stream, p, seqs, n);
    const dim3 grid = block_grid(p, n, 1);
    if (p.dtype == kDtypeF32) return launch_pdl(k_kv4_load<kDtypeF32>, grid, kRowThreads, 0, stream, p, seqs);
    if (p.dtype == kDtypeBf16) return launch_pdl(k_kv4_load<kDtypeBf16>, grid, kRowThreads, 0, stream, p, seqs);
    if (p.staging) return launch_pdl(k_kv4_load<kDtypeF16, true>, grid, kRowThreads, 0, stream, p, seqs);
    return launch_pdl(k_kv4_load<kDtypeF16>, grid, kRowThreads, 0, stream, p, seqs);
}

}  // namespace flint
