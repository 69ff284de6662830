// What the decode and the prefill attention over the block-scaled paged cache share: the cache's view, the page math on
// warp-level matrix instructions, and the checks of their C entries.
//
// With x_j = scale * log2(e) * ks_j * (q . kcode_j) the output of a row is sum_j 2^x_j vs_j vcode_j / sum_j 2^x_j.  The
// scales never touch the codes: ks_j multiplies a score, and vs_j is a power of two that goes into the exponent,
//   P_j = 2^(x_j + log2 vs_j - M),  out = sum_j P_j vcode_j / l,  l = sum_j P_j / vs_j,
// so that P is always fit for 16 bits whatever the blocks' magnitudes are, and a block with small values does not
// disturb one with large ones.  Scales lie in [2^-60, 2^40] (what the store writes), which keeps l inside float32.
// M is set so that the weights so far lie well above 1 (decode: the largest at 2^7; prefill: the sum of 32 at 2^6 to 2^7) and
// follows them only when one might leave f16: P stays at or below 2^15 in decode, below 61440 in prefill.  So far above
// 1, because f16 has no finer step than 2^-24: what rounds to zero lies below 2^-31 of the weights it stands beside, and the quiet
// keys of a long row count behind a loud one.
//
// Codes are converted to f16 (exact) in registers.  A query row is brought to a power of two of its own before it goes to
// f16 (largest element in [2^14, 2^15)), so that bf16's range does not matter: elements that lose bits there are below
// 2^-28 of the row's largest.  P is rounded to f16, off by 2^-11 of a weight or by 2^-25 at most (for f16 outputs the
// rest of a weight is a second f16 operand: 2^-22 or 2^-25); scores, M, l and the output are float32.
#pragma once

#include <atomic>

#include "common.cuh"

namespace fdms {

constexpr int kCachePage = 16;                  // rows per step of a warp; a block is 1, 2, 4 or 8 of them
constexpr float kPagedLog2e = 1.4426950408889634f;
constexpr float kPagedLn2 = 0.6931471805599453f;

struct PagedCache {
    const uint8_t* k;
    const uint8_t* v;
    int64_t k_sb, k_sh, k_sr, v_sb, v_sh, v_sr;     // block, head and row stride in bytes
    const float* k_scale;                           // [blocks, heads]
    const float* v_scale;
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* kv_lens;
    int32_t* status;
    int32_t num_blocks, max_blocks, heads, shift;   // shift: log2(block size)
};

__device__ __forceinline__ float paged_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float paged_lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Four e4m3 bytes as two f16x2: bytes 0,1 and bytes 2,3.
__device__ __forceinline__ void e4m3x4_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ uint32_t f16x2_of(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t*)&h;
}

// Rows of a sequence that the cache really holds room for; an impossible length raises the status bit.
__device__ __forceinline__ int paged_len(const PagedCache& c, int b) {
    int len = c.kv_lens[b];
    const int64_t room = (int64_t)c.max_blocks << c.shift;
    if (len < 0 || len > room) {
        if (c.status) atomicOr(c.status, FDMS_DEV_BAD_INDEX);
        len = len < 0 ? 0 : (int)room;
    }
    return len;
}

// A block's V scale as the weights can carry it.  The store writes 2^-60 and more; a block that nothing was stored into may hold 0,
// whose logarithm no sum of exponents survives: it counts as 2^-60.  What is negative or NaN gives NaN.
__device__ __forceinline__ float paged_v_scale(float vs) { return vs >= 0.0f ? fmaxf(vs, 0x1p-60f) : vs; }

// Power of two that brings a row with largest magnitude `top` to [2^14, 2^15), and its inverse.
__device__ __forceinline__ void row_power(float top, float& up, float& down) {
    const int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;      // -127 for zero and subnormals, 128 for inf
    const int k = min(14 - e, 126);             // both powers are normal numbers for every e
    up = __uint_as_float((uint32_t)(127 + k) << 23);
    down = __uint_as_float((uint32_t)(127 - k) << 23);
}

template <bool BF16>
__device__ __forceinline__ void unpack_pair(uint32_t w, float& a, float& b) {
    if (BF16) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    } else {
        const __half2 h = *(const __half2*)&w;
        a = __low2float(h);
        b = __high2float(h);
    }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *(const uint32_t*)&h;
    }
    return f16x2_of(a, b);
}

// D(16x8, f32) += A(16x16, f16) B(16x8, f16).
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8x8 matrix of 16-bit values, lane (g, t) holding row g, columns 2t and 2t + 1, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// SM count of the current device.
inline int paged_sms() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev >= 0 && dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (dev >= 0 && dev < 64) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

// Checks of a cache that every entry makes; `idle`: the call has nothing to do, so its pointers may be null.
inline int32_t paged_cache_check(const char* name, const fdms_paged_cache& c, int64_t dtype, bool idle, int32_t& shift) {
    FDMS_REQUIRE(dtype == FDMS_BF16 || dtype == FDMS_F16, FDMS_E_DTYPE, "%s: bf16 or f16 activations only", name);
    FDMS_REQUIRE(c.head_dim == 64 || c.head_dim == 128, FDMS_E_ARG, "%s: head_dim must be 64 or 128, got %lld", name, (long long)c.head_dim);
    shift = c.block_size == 16 ? 4 : c.block_size == 32 ? 5 : c.block_size == 64 ? 6 : c.block_size == 128 ? 7 : -1;
    FDMS_REQUIRE(shift > 0, FDMS_E_ARG, "%s: block_size must be 16, 32, 64 or 128, got %lld", name, (long long)c.block_size);
    FDMS_REQUIRE(c.num_blocks >= 0 && c.kv_heads > 0, FDMS_E_ARG, "%s: negative size, or no KV heads", name);
    FDMS_REQUIRE(c.num_blocks <= (0x7fffffff >> shift) && c.kv_heads <= 4096, FDMS_E_CAPACITY,
                 "%s: slot numbers must fit in 31 bits, and at most 4096 KV heads", name);
    if (idle || c.num_blocks == 0) return FDMS_OK;
    FDMS_REQUIRE(c.k && c.v && c.k_scale && c.v_scale, FDMS_E_ARG, "%s: null pointer", name);
    const int64_t strides = c.k_stride[0] | c.k_stride[1] | c.k_stride[2] | c.v_stride[0] | c.v_stride[1] | c.v_stride[2];
    FDMS_REQUIRE(strides >= 0, FDMS_E_ARG, "%s: negative stride of the cache", name);
    FDMS_REQUIRE((((uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)strides) & 15) == 0 && c.k_stride[3] == 1 && c.v_stride[3] == 1, FDMS_E_ARG,
                 "%s: the cache must be contiguous in its last dimension and aligned to 16 bytes in the others", name);
    return FDMS_OK;
}

// Checks that both attention entries make, and the cache's view.
inline int32_t paged_attn_check(const char* name, const fdms_paged_attn_args* args, PagedCache& view, bool idle) {
    FDMS_REQUIRE(args, FDMS_E_ARG, "%s: null pointer", name);
    const fdms_paged_attn_args& p = *args;
    const fdms_paged_cache& c = p.cache;
    int32_t shift = 0;
    const int32_t rc = paged_cache_check(name, c, p.dtype, idle, shift);
    if (rc != FDMS_OK) return rc;
    FDMS_REQUIRE(p.tokens >= 0 && p.num_seqs >= 0 && p.max_blocks >= 0 && p.num_q_heads > 0, FDMS_E_ARG, "%s: negative size", name);
    FDMS_REQUIRE(p.num_q_heads % c.kv_heads == 0 && p.num_q_heads / c.kv_heads <= 64, FDMS_E_ARG, "%s: q_heads=%lld must be kv_heads=%lld times 1 to 64",
                 name, (long long)p.num_q_heads, (long long)c.kv_heads);
    FDMS_REQUIRE(p.max_blocks <= (0x7fffffff >> shift) && p.tokens < 0x7fffffff && p.num_seqs < 0x7fffffff, FDMS_E_CAPACITY,
                 "%s: token and slot numbers must fit in 31 bits", name);
    if (!idle) {
        FDMS_REQUIRE(p.q && p.out && p.kv_lens && (p.block_tables || p.max_blocks == 0), FDMS_E_ARG, "%s: null pointer", name);
        const int64_t strides = p.q_stride[0] | p.q_stride[1] | p.out_stride[0] | p.out_stride[1];
        FDMS_REQUIRE((((uintptr_t)p.q | (uintptr_t)p.out | (uintptr_t)(2 * strides)) & 15) == 0 && p.q_stride[2] == 1 && p.out_stride[2] == 1, FDMS_E_ARG,
                     "%s: q and out must be contiguous in their last dimension and aligned to 16 bytes in the others", name);
    }
    FDMS_REQUIRE(c.num_blocks == 0 || (c.k_stride[0] < (1ll << 32) && c.v_stride[0] < (1ll << 32) && c.k_stride[2] <= (1 << 24) && c.v_stride[2] <= (1 << 24)),
                 FDMS_E_CAPACITY, "%s: a block's stride must fit in 32 bits, a row's in 24", name);
    view = {c.k, c.v, c.k_stride[0], c.k_stride[1], c.k_stride[2], c.v_stride[0], c.v_stride[1], c.v_stride[2], c.k_scale, c.v_scale,
            p.block_tables, p.bt_stride, p.kv_lens, p.dev_status, (int32_t)c.num_blocks, (int32_t)p.max_blocks, (int32_t)c.kv_heads, shift};
    return FDMS_OK;
}

}  // namespace fdms
