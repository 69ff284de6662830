// Prefill attention over the block-scaled paged cache: the tokens of a step, packed sequence by sequence, against their
// sequence's cached rows.  Token i of a sequence with n tokens in the step and kv rows in the cache sees rows
// 0 .. kv - n + i; a token that sees no row gets zeros and a log-sum-exp of -inf.
//
// A CTA takes two tiles of 128 rows ((token, q head) pairs of one KV head, the heads of a token together), or one where there
// are few, and walks the sequence's rows, or its part of them, in tiles of 128 keys:
//   warps 0-3, 4-7   softmax of tile 0 and 1, a thread per row: scores out of tensor memory, weights P back into it as f16
//   warps 8-11       convert the keys' K and V codes to f16 (exact) in shared memory, two stages of each
//   warps 12, 13     issue a tile's tensor-core products S = Q K^T and O += P V (tcgen05, accumulators in tensor memory),
//                    one warp per tile: one for both spent more on waiting and issuing (800 cycles for each of the eight
//                    batches of 128 keys) than the products take
// Tensor memory holds O of both tiles (2 x D columns) and for each two (D = 64: three) buffers of S, 64 keys wide, P over the
// S it comes from: the scores of 64 keys are computed while the 64 before them are weighed, so that the softmax does not wait for
// their product.  Two tiles per CTA halve the conversions.  Every wait is bounded; when one runs out the CTA raises
// FDMS_DEV_WAIT_TIMEOUT, lets what it issued complete, gives its tensor memory back and returns.
//
// Measured (32 q heads on 8 KV heads, a B200): 2048 tokens over 16384 rows at head_dim 128 take 579 us in bf16 (890 TFLOP/s) and 741 in
// f16, whose weights take a second product; 7 ragged prompts of up to 3001 tokens at head_dim 64 355 and 431 us.  No unit bounds
// it: of the SMs' active time the tensor pipe works 48 %, the unit of the exponential 48 %, and an instruction issues in 45 % of the
// cycles.  A step of 128 keys takes about 2.4 us at both head sizes, where its exponentials need 1.1: each softmax warp goes through
// load, weights, store and arrival in turn, and the two of a scheduler do not fill each other's waits.  256 equal CTAs on 148 SMs
// run in two waves and leave 14 % of them idle.
//
// Few tokens over many rows would leave most SMs idle: the rows are then cut into parts for a CTA each, whose results go to a
// workspace and are joined by a second launch.
#include "paged_attn.cuh"

namespace fdms {

constexpr int kTileRows = 128;                  // query rows per tile, keys per step
constexpr int kHalf = kTileRows / 2;            // keys per buffer of scores
constexpr int kPreThreads = 14 * 32;
constexpr int kConvWarp = 8, kMmaWarp = 12;
constexpr int kConstRing = 4;                   // steps whose page constants are held: the softmax may lag two behind
constexpr uint64_t kPreWaitNs = 1000000000;     // a wait gives up after a second
constexpr int kDrainPolls = 10000000;           // of 100 ns: the wait for what was issued gives up after a second too
constexpr uint32_t kTmemCols = 512;

struct PrefillArgs {
    PagedCache c;
    const uint16_t* q;
    uint16_t* out;
    float* lse;                                 // optional [q_heads, tokens]
    const int32_t* cu;                          // [seqs + 1]
    int64_t q_st, q_sh, o_st, o_sh, lse_sh, lse_st;
    int64_t tokens;
    float* parts;                               // [splits][tokens][q_heads][D + 4]: O, M, l of a part of the rows
    int32_t seqs, group;
    int32_t tiles, splits;                      // tiles of rows per CTA (1 or 2), parts that the cached rows are cut into
    float scale;
};

// Sequence and first token (within the sequence) of tile x, tiles of `per` tokens; false beyond the last tile.  Every warp
// finds it for itself: 32 sequences at a time.
__device__ __forceinline__ bool find_tile(const PrefillArgs& a, int64_t x, int per, int& seq, int64_t& first, int64_t& begin, int64_t& count) {
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < a.seqs; base += 32) {
        const int s = base + lane;
        int64_t b = 0, e = 0;
        if (s < a.seqs) {
            b = min(max((int64_t)a.cu[s], (int64_t)0), a.tokens);
            e = min(max((int64_t)a.cu[s + 1], b), a.tokens);
        }
        const int64_t tiles = (e - b + per - 1) / per;
        int64_t sum = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        const unsigned m = __ballot_sync(0xffffffffu, sum > x);
        if (m) {
            const int l = __ffs(m) - 1;
            seq = base + l;
            first = (x - __shfl_sync(0xffffffffu, sum - tiles, l)) * per;
            begin = __shfl_sync(0xffffffffu, b, l);
            count = __shfl_sync(0xffffffffu, e - b, l);
            return true;
        }
        x -= __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
}

// ---- barriers, tensor memory, matrix instructions --------------------------------------------------------------
__device__ __forceinline__ uint32_t s_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* b, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s_addr(b)) : "memory");
}
__device__ __forceinline__ bool bar_test(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(s_addr(b)), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded wait; gives up when another warp has, or after kPreWaitNs of its own.
__device__ __noinline__ bool bar_wait_long(uint64_t* b, uint32_t parity, volatile int* give_up) {
    uint64_t t0, t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    for (;;) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(s_addr(b)), "r"(parity) : "memory");
        if (ok) return true;
        if (*give_up) return false;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
        if (t - t0 > kPreWaitNs) break;
    }
    *give_up = 1;
    return false;
}
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, volatile int* give_up) {
    return bar_test(b, parity) || bar_wait_long(b, parity, give_up);
}
// The same by a warp, with one answer for all of it.
__device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t parity, volatile int* give_up) {
    return __all_sync(0xffffffffu, bar_wait(b, parity, give_up));
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s_addr(b)) : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D (tensor memory, f32) (+)= A B: A and B in shared memory, or A in tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}

#define FDMS_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define FDMS_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// Pairs of float32 values in one 64-bit register.
__device__ __forceinline__ uint64_t pair(float a, float b) { return (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32; }
__device__ __forceinline__ uint64_t both(float a) { return pair(a, a); }
__device__ __forceinline__ float low(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float high(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 32, 16 or 8 columns of the thread's lane.  What a load brings is there after a wait that names it: the wait takes the
// registers as operands, so that nothing that uses them moves ahead of it.
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
        "%27,%28,%29,%30,%31}, [%32];"
        : FDMS_R8(r, 0), FDMS_R8(r, 8), FDMS_R8(r, 16), FDMS_R8(r, 24) : "r"(addr) : "memory");
}
#define FDMS_RW8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
__device__ __forceinline__ void tc_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : FDMS_RW8(r, 0), FDMS_RW8(r, 8), FDMS_RW8(r, 16), FDMS_RW8(r, 24) : : "memory");
}
__device__ __forceinline__ void tc_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : FDMS_RW8(r, 0), FDMS_RW8(r, 8) : : "memory");
}
__device__ __forceinline__ void tc_wait_ld(uint32_t (&r)[8]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : FDMS_RW8(r, 0) : : "memory"); }
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : FDMS_R8(r, 0), FDMS_R8(r, 8) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), FDMS_W8(r, 0), FDMS_W8(r, 8) : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : FDMS_R8(r, 0) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), FDMS_W8(r, 0) : "memory");
}

constexpr float kMostWeight = 61440.0f;         // a sum of weights below this keeps each inside f16
// log2 of what the sum of 32 weights is brought to, or up to a half below, when M is set.  Higher keeps more of the weights that f16
// cannot hold and leaves less room until M has to move again: 2048 tokens over 16384 rows take 568 us with 7 and 571 with 8, 7 ragged
// prompts 352 and 352 (head_dim 64), 392 and 394 (128).  Less than 8, so that where float32's steps at M are 16 the largest weight
// ends up at 1 and not at 2^16.
constexpr float kSetWeight = 7.0f;
// From here on whole numbers are not all float32 numbers, and M would differ from s * factor * ks, which a multiply-add takes
// exactly, by a rounding that no weight survives.  Such a row gets M = inf, under which all its weights are 0, and is computed by itself
// in the end.
constexpr float kCoarse = 0x1p24f;

// Exponents of 32 scores: x = s * factor * ks + log2 vs - ref, keys behind `seen` masked.
__device__ __forceinline__ void exponents(const uint32_t (&s)[32], float factor, const float4& p0, const float4& p1, float ref, bool cut, int seen,
                                          uint64_t (&x)[16]) {
    const uint64_t f0 = both(factor * p0.x), b0 = both(p0.y - ref), f1 = both(factor * p1.x), b1 = both(p1.y - ref);
#pragma unroll
    for (int i = 0; i < 16; ++i)
        x[i] = fma2((uint64_t)s[2 * i] | (uint64_t)s[2 * i + 1] << 32, i < 8 ? f0 : f1, i < 8 ? b0 : b1);
    if (cut) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = pair(2 * i > seen ? -INFINITY : low(x[i]), 2 * i + 1 > seen ? -INFINITY : high(x[i]));
    }
}
// Weights of 32 scores as f16 and their sums over each of the two pages; with FINE also what the rounding to f16 left.
template <bool FINE>
__device__ __forceinline__ void weigh(const uint32_t (&s)[32], float factor, const float4& p0, const float4& p1, float m, bool cut, int seen,
                                      uint32_t (&p)[16], uint32_t (&rest)[16], float& sum0, float& sum1) {
    uint64_t x[16];
    exponents(s, factor, p0, p1, m == -INFINITY ? 0.0f : m, cut, seen, x);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float e = paged_ex2(low(x[i])), f = paged_ex2(high(x[i]));
        x[i] = pair(e, f);
        p[i] = f16x2_of(e, f);
        if (FINE) {
            const __half2 h = *(const __half2*)&p[i];
            const uint64_t left = add2(x[i], pair(-__low2float(h), -__high2float(h)));
            rest[i] = f16x2_of(low(left), high(left));
        }
    }
#pragma unroll
    for (int n = 4; n > 0; n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) {
            x[i] = add2(x[i], x[i + n]);
            x[8 + i] = add2(x[8 + i], x[8 + i + n]);
        }
    sum0 = low(x[0]) + high(x[0]);
    sum1 = low(x[8]) + high(x[8]);
}
// The rare paths of the softmax, kept out of its loop: the largest exponent of 32 scores; a row of O, or a page of P, times a power
// of two.
__device__ __noinline__ float largest(uint32_t at, float factor, const float4* page, int seen) {
    uint32_t s[32];
    uint64_t x[16];
    tmem_load(at, s);
    tc_wait_ld(s);
    exponents(s, factor, page[0], page[1], 0.0f, true, seen, x);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaxf(low(x[i]), high(x[i])));
    return top;
}
template <int D>
__device__ __noinline__ void rescale_o(uint32_t at, float r) {
    for (int c = 0; c < D / 16; ++c) {
        uint32_t o[16];
        tmem_load(at + 16 * c, o);
        tc_wait_ld(o);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * r);
        tmem_store(at + 16 * c, o);
    }
}
// The factor may lie below what f16 holds while the product does not.
__device__ __forceinline__ uint32_t f16x2_times(uint32_t x, float r) {
    const __half2 h = *(const __half2*)&x;
    return f16x2_of(__low2float(h) * r, __high2float(h) * r);
}
__device__ __noinline__ void rescale_p(uint32_t at, float r) {
    uint32_t p[8];
    tmem_load(at, p);
    tc_wait_ld(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = f16x2_times(p[i], r);
    tmem_store(at, p);
}

// Operands in shared memory lie in slabs of 64 elements (128 bytes) per row, rows one after the other, 16-byte chunks
// permuted by the row's last three bits (the 128-byte swizzle).  Q and K are read along their rows (K-major), V across
// them (its channels are the product's columns); both see the same layout.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t leading, uint32_t stride) {
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// f16 operands, float32 result, 128 rows, n columns; `across`: B is read across its rows.
__host__ __device__ constexpr uint32_t instruction(int n, bool across) {
    return 1u << 4 | (across ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(kTileRows >> 4) << 24;
}
constexpr uint32_t kSlab = kTileRows * 128;     // bytes

template <int D>
struct PrefillSmem {
    static constexpr uint32_t kTile = kTileRows * D * 2;        // one operand tile
    static constexpr int kBufs = D == 64 ? 3 : 2;               // what the tensor memory has room for
    static constexpr uint32_t kO = 2 * kBufs * kHalf;           // columns: S of tile i from i * kBufs * kHalf on, O at kO + i * D
    static constexpr uint32_t kQ = 0, kK = 2 * kTile, kV = 4 * kTile, kEnd = 6 * kTile;
    // 1 KB for the alignment of the tiles; D = 64 asks for more than half of the SM's shared memory all the same, because a
    // second CTA would wait for tensor memory that the first holds
    static constexpr uint32_t kBytes = (kEnd + 1024 + 1024) > 120 * 1024 ? kEnd + 2048 : 120 * 1024;
};

struct PrefillShared {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2][3], p_full[2][3], pv_done[2][3], drain[2];
    float4 page[kConstRing][kTileRows / kCachePage];            // ks, log2 vs, 1 / vs of the step's pages
    uint32_t tmem;
    int give_up, nan_lo, nan_hi;
};

__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Scores of tile ti against the half h of the keys in stage st; the weights of tile ti times the values of that half.  `again`: the stage
// will be filled again, and that waits for the products; an arrival that nobody waits for might come after the CTA's end.
template <int D>
__device__ __forceinline__ void issue_scores(uint32_t base, uint32_t tmem, int ti, int st, int h, int buf, bool again, PrefillShared& sh) {
    using L = PrefillSmem<D>;
    const uint64_t q = operand(base + L::kQ + ti * L::kTile, 16, 1024), k = operand(base + L::kK + st * L::kTile + h * (kHalf * 128), 16, 1024);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        const uint32_t step = ((i >> 2) * kSlab + (i & 3) * 32) >> 4;      // addresses are in units of 16 bytes
        mma_ss(tmem + (L::kBufs * ti + buf) * kHalf, q + step, k + step, instruction(kHalf, false), i > 0);
    }
    tc_commit(&sh.s_full[ti][buf]);
    if (again) tc_commit(&sh.k_empty[st]);
}
template <int D, bool FINE>
__device__ __forceinline__ void issue_values(uint32_t base, uint32_t tmem, int ti, int st, int h, int buf, bool add, bool again, PrefillShared& sh) {
    using L = PrefillSmem<D>;
    const uint64_t v = operand(base + L::kV + st * L::kTile + h * (kHalf * 128), kSlab, 1024);
#pragma unroll
    for (int i = 0; i < kHalf / 16; ++i)
        mma_ts(tmem + L::kO + D * ti, tmem + (L::kBufs * ti + buf) * kHalf + 8 * i, v + (i * 2048 >> 4), instruction(D, true), i > 0 || add);
    if (FINE)
#pragma unroll
        for (int i = 0; i < kHalf / 16; ++i)
            mma_ts(tmem + L::kO + D * ti, tmem + (L::kBufs * ti + buf) * kHalf + 32 + 8 * i, v + (i * 2048 >> 4), instruction(D, true), true);
    tc_commit(&sh.pv_done[ti][buf]);
    if (again) tc_commit(&sh.v_empty[st]);
}

// One row by a warp, its weights in float32: the first `keys` cached rows from row `from` of the sequence on.  `q`: the row's f16
// elements in shared memory, of row r of its tile; a lane has a key, then D / 32 channels.
template <int D>
__device__ __forceinline__ void whole_row(const PagedCache& c, const uint8_t* q, int r, float factor, int seq, int head, int from, int keys,
                                          float (&acc)[D / 32], float& m, float& l) {
    const int lane = threadIdx.x & 31;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
    for (int base = 0; base < keys; base += 32) {
        const int at = from + base + lane, in_block = at & ((1 << c.shift) - 1);
        int blk = base + lane < keys ? c.tables[seq * c.table_stride + (at >> c.shift)] : -1;
        if (blk >= c.num_blocks) blk = -1;
        float x = -INFINITY, inv = 1.0f;
        if (blk >= 0) {
            const uint8_t* k = c.k + blk * c.k_sb + head * c.k_sh + in_block * c.k_sr;
            const float vs = paged_v_scale(c.v_scale[(int64_t)blk * c.heads + head]);
            float dot = 0.0f;
#pragma unroll 1
            for (int i = 0; i < D / 8; ++i) {
                const uint4 w = *(const uint4*)(q + (i >> 3) * kSlab + (((i & 7) ^ (r & 7)) << 4));
                const uint2 b = *(const uint2*)(k + 8 * i);
                const uint32_t y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const __half2 h = *(const __half2*)&y[e >> 1];
                    dot = fmaf(e & 1 ? __high2float(h) : __low2float(h), e4m3_to_float((uint8_t)((e < 4 ? b.x : b.y) >> (8 * (e & 3)))), dot);
                }
            }
            x = fmaf(dot, factor * c.k_scale[(int64_t)blk * c.heads + head], paged_lg2(vs));
            inv = __frcp_rn(vs);
        }
        float top = x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float next = fmaxf(m, top), ref = next == -INFINITY ? 0.0f : next, scale = paged_ex2(m - ref), p = paged_ex2(x - ref);
        m = next;
        l = fmaf(l, scale, p * inv);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] *= scale;
#pragma unroll 8
        for (int j = 0; j < 32; ++j) {
            const int b = __shfl_sync(0xffffffffu, blk, j);
            const float w = __shfl_sync(0xffffffffu, p, j);
            if (b < 0) continue;
            const uint8_t* v = c.v + b * c.v_sb + head * c.v_sh + ((from + base + j) & ((1 << c.shift) - 1)) * c.v_sr + lane * (D / 32);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(w, e4m3_to_float(v[i]), acc[i]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kPreThreads, 1) paged_prefill_kernel(PrefillArgs a) {
    extern __shared__ uint8_t dyn[];
    __shared__ PrefillShared sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (a.splits > 1) pdl_trigger();
    const int per = kTileRows / a.group;        // tokens per tile
    int seq;
    int64_t first, begin, count;
    // the last tiles of a sequence see the most rows: they start first
    if (!find_tile(a, (int64_t)gridDim.x - 1 - blockIdx.x, a.tiles * per, seq, first, begin, count)) return;
    const int head = blockIdx.y;
    const int kv = paged_len(a.c, seq);
    const int64_t end = min(first + a.tiles * per, count);
    const int tiles = a.tiles > 1 && first + per < count ? 2 : 1;
    // the CTA's part of the rows begins at row `from`; from here on rows count from there
    const int64_t sees = max((int64_t)kv - count + end, (int64_t)0);
    const int all = (int)((sees + kTileRows - 1) / kTileRows), part = (all + a.splits - 1) / a.splits;
    const int from = min((int)blockIdx.z * part, all) * kTileRows;
    const int64_t here = min(max(sees - from, (int64_t)0), (int64_t)part * kTileRows);
    const int64_t shift = (int64_t)kv - count - from;       // token j of the sequence's step sees rows 0 .. shift + j
    const int rows = kv - from;
    const int steps = (int)((here + kTileRows - 1) / kTileRows), halves = (int)((here + kHalf - 1) / kHalf);
    // keys below `open` are seen by every row of the CTA
    const int64_t open = max(shift + first + 1, (int64_t)0);
    uint8_t* tile = (uint8_t*)(((uintptr_t)dyn + 1023) & ~(uintptr_t)1023);
    using L = PrefillSmem<D>;
    // A weight in f16 is 2^-12 off on the average, as much as the rounding of an f16 output: there the rest of each weight
    // goes through a product of its own.
    constexpr bool kFine = !BF16;

    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(&sh.tmem)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (threadIdx.x == 0) {
        bar_init(&sh.q_full, 8);
        for (int i = 0; i < 2; ++i) {
            bar_init(&sh.k_full[i], 4);
            bar_init(&sh.v_full[i], 4);
            bar_init(&sh.k_empty[i], 2 * tiles);
            bar_init(&sh.v_empty[i], 2 * tiles);
            bar_init(&sh.drain[i], 1);
            for (int k = 0; k < 3; ++k) {
                bar_init(&sh.s_full[i][k], 1);
                bar_init(&sh.p_full[i][k], 4);
                bar_init(&sh.pv_done[i][k], 1);
            }
        }
        sh.give_up = 0;
        sh.nan_lo = 0x7fffffff;
        sh.nan_hi = -1;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    volatile int* give_up = &sh.give_up;

    if (warp < kConvWarp) {
        // ---- softmax: a thread per row ----
        const int ti = warp >> 2, r = threadIdx.x & 127;
        const int64_t j = first + ti * per + r / a.group;
        const bool live = r < per * a.group && j < count;
        const int hq = head * a.group + (live ? r % a.group : 0);
        const int64_t tok = begin + (live ? j : first);
        const int64_t last = live ? shift + j : (int64_t)1 << 40;          // a row that nobody reads is not worth a mask
        float factor;
        {
            const uint16_t* q = a.q + tok * a.q_st + (int64_t)hq * a.q_sh;
            uint4 w[D / 8];                     // the whole row at once: one latency
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) w[i] = make_uint4(0, 0, 0, 0);
            if (live) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) w[i] = __ldg((const uint4*)(q + 8 * i));
            }
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float e, f;
                    unpack_pair<BF16>(x[k], e, f);
                    top = fmaxf(top, fmaxf(fabsf(e), fabsf(f)));
                }
            }
            float up;
            row_power(top, up, factor);
            factor *= a.scale * kPagedLog2e;
            uint8_t* dst = tile + L::kQ + ti * L::kTile + r * 128;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                uint32_t y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float e, f;
                    unpack_pair<BF16>(x[k], e, f);
                    y[k] = f16x2_of(e * up, f * up);
                }
                *(uint4*)(dst + (i >> 3) * kSlab + (((i & 7) ^ (r & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
            }
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) bar_arrive(&sh.q_full);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                  // the warp's 32 lanes of tensor memory
        const uint32_t o_at = tmem + lanes + L::kO + D * ti;
        float m = -INFINITY, l = 0.0f;
        bool ok = ti < tiles;
        int buf = 0, turn = 0;                  // buffer of the half, and how often it has been used before (mod 2)
        for (int half = 0; ok && half < halves; ++half) {
            ok = warp_wait(&sh.s_full[ti][buf], turn, give_up);
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_at = tmem + lanes + (L::kBufs * ti + buf) * kHalf;
            const float4* page = &sh.page[(half >> 1) & (kConstRing - 1)][(half & 1) * (kHalf / kCachePage)];
            const int seen = (int)min(last - (int64_t)half * kHalf, (int64_t)kHalf);         // last key of the half that the row sees
            const bool cut = __any_sync(0xffffffffu, seen < kHalf - 1);
            // 32 keys at a time.  P takes the columns of scores that have been read.  M follows the weights only when one
            // might leave f16 (the sum of 32 tells, and says where M goes) and is a whole number: O, l and the earlier weights of
            // the half then follow by an exact factor.  Most keys need no maximum at all.
            uint32_t sc[2][32];
            tmem_load(s_at, sc[0]);
            tmem_load(s_at + 32, sc[1]);
            uint32_t rest[2][16];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                tc_wait_ld(sc[c]);
                const float4 p0 = page[2 * c], p1 = page[2 * c + 1];
                uint32_t p[16];
                float sum0, sum1;
                weigh<kFine>(sc[c], factor, p0, p1, m, cut, seen - 32 * c, p, rest[c], sum0, sum1);
                const bool moves = m == -INFINITY || sum0 + sum1 > kMostWeight;         // rows do not follow their neighbours
                if (__any_sync(0xffffffffu, moves)) {
                    if (c == 0) tc_wait_ld(sc[1]);
                    const float sum = sum0 + sum1;
                    const bool known = sum > 0x1p-100f && sum < 0x1p100f;       // else the maximum has to say
                    float to = (m == -INFINITY ? 0.0f : m) + (float)((int)(__float_as_uint(sum) >> 23) - 126);
                    if (__any_sync(0xffffffffu, moves && !known)) {
                        const float top = largest(s_at + 32 * c, factor, page + 2 * c, seen - 32 * c);
                        if (!known) to = ceilf(top);
                    }
                    float next = moves ? fmaxf(m, to - kSetWeight) : m;
                    if (fabsf(next) >= kCoarse && next != -INFINITY) next = INFINITY;
                    const float r = next == m ? 1.0f : paged_ex2(m - next);
                    m = next;
                    l *= r;
                    if (half > 0) {             // the products of the half before must be complete before O is touched
                        ok = warp_wait(&sh.pv_done[ti][buf ? buf - 1 : L::kBufs - 1], buf ? turn : turn ^ 1, give_up);
                        tc_fence_after();
                        rescale_o<D>(o_at, r);
                    }
                    tc_wait_st();
                    for (int e = 0; e < 2 * c; ++e) rescale_p(s_at + 8 * e, r);
                    if (kFine && c == 1) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) rest[0][i] = f16x2_times(rest[0][i], r);
                    }
                    tmem_load(s_at + 32 * c, sc[c]);
                    tc_wait_ld(sc[c]);
                    weigh<kFine>(sc[c], factor, p0, p1, m, cut, seen - 32 * c, p, rest[c], sum0, sum1);
                }
                tmem_store(s_at + 16 * c, p);
                l = fmaf(sum0, p0.z, l);
                l = fmaf(sum1, p1.z, l);
            }
            if (kFine) {                        // over scores that are not needed any more
                tmem_store(s_at + 32, rest[0]);
                tmem_store(s_at + 48, rest[1]);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.p_full[ti][buf]);
            if (++buf == L::kBufs) { buf = 0; turn ^= 1; }
        }
        if (ti < tiles) {
            if (halves > 0 && ok) ok = warp_wait(&sh.pv_done[ti][(halves - 1) % L::kBufs], ((halves - 1) / L::kBufs) & 1, give_up);
            tc_fence_after();
            const float inv = l > 0.0f || l != l ? __frcp_rn(l) : 0.0f;
            const bool again = live && m == INFINITY, write = live && !again;
            uint16_t* out = a.out + tok * a.o_st + (int64_t)hq * a.o_sh;
            float* mine = a.parts + (((int64_t)blockIdx.z * a.tokens + tok) * (a.c.heads * a.group) + hq) * (D + 4);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = 0;
                if (halves > 0) {
                    tmem_load(o_at + 16 * c, o);
                    tc_wait_ld(o);
                }
                if (write && a.splits > 1) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) *(uint4*)(mine + 16 * c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                } else if (write) {
#pragma unroll
                    for (int i = 0; i < 16; i += 8) {
                        uint32_t y[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            y[k] = pack_pair<BF16>(__uint_as_float(o[i + 2 * k]) * inv, __uint_as_float(o[i + 2 * k + 1]) * inv);
                        *(uint4*)(out + 16 * c + i) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                }
            }
            if (write && a.splits > 1) *(float2*)(mine + D) = make_float2(m, l);
            else if (write && a.lse) a.lse[(int64_t)hq * a.lse_sh + tok * a.lse_st] = kPagedLn2 * (m + paged_lg2(l));
            for (unsigned todo = __ballot_sync(0xffffffffu, again); todo; todo &= todo - 1) {
                const int src = __ffs(todo) - 1, row = (r & ~31) + src;
                const int keys = (int)min(max(__shfl_sync(0xffffffffu, last, src) + 1, (int64_t)0), here);
                float acc[D / 32], rm, rl;
                whole_row<D>(a.c, tile + L::kQ + ti * L::kTile + row * 128, row, __shfl_sync(0xffffffffu, factor, src), seq, head, from, keys, acc, rm, rl);
                const int64_t row_tok = __shfl_sync(0xffffffffu, tok, src);
                const int row_hq = __shfl_sync(0xffffffffu, hq, src);
                if (a.splits > 1) {
                    float* part = a.parts + (((int64_t)blockIdx.z * a.tokens + row_tok) * (a.c.heads * a.group) + row_hq) * (D + 4);
#pragma unroll
                    for (int i = 0; i < D / 32; i += 2) *(float2*)(part + lane * (D / 32) + i) = make_float2(acc[i], acc[i + 1]);
                    if (lane == 0) *(float2*)(part + D) = make_float2(rm, rl);
                } else {
                    const float by = rl > 0.0f || rl != rl ? __frcp_rn(rl) : 0.0f;
                    uint16_t* to = a.out + row_tok * a.o_st + (int64_t)row_hq * a.o_sh + lane * (D / 32);
#pragma unroll
                    for (int i = 0; i < D / 32; i += 2) *(uint32_t*)(to + i) = pack_pair<BF16>(acc[i] * by, acc[i + 1] * by);
                    if (lane == 0 && a.lse) a.lse[(int64_t)row_hq * a.lse_sh + row_tok * a.lse_st] = kPagedLn2 * (rm + paged_lg2(rl));
                }
            }
            __syncwarp();
            // NaN codes of V in steps that not every row sees whole were left out of the products: into the rows that see them
            const int lo = *(volatile int*)&sh.nan_lo, hi = *(volatile int*)&sh.nan_hi;
            if (live && lo <= hi)
                for (int64_t key = (int64_t)lo * kTileRows; key < (int64_t)(hi + 1) * kTileRows && key <= last; ++key) {
                    const int blk = a.c.tables[seq * a.c.table_stride + ((from + key) >> a.c.shift)];
                    if (blk < 0 || blk >= a.c.num_blocks) continue;
                    const uint8_t* v = a.c.v + (int64_t)blk * a.c.v_sb + head * a.c.v_sh + ((from + key) & ((1 << a.c.shift) - 1)) * a.c.v_sr;
                    for (int ch = 0; ch < D; ++ch)
                        if ((v[ch] & 0x7f) == 0x7f) {
                            if (a.splits > 1) mine[ch] = NAN; else out[ch] = 0x7fff;        // a NaN in bf16 and in f16
                        }
                }
        }
    } else if (warp < kMmaWarp) {
        // ---- codes to f16 in shared memory ----
        constexpr int kPer = D / 16;                                        // 16-byte vectors per thread, K and V each
        constexpr int kPass = 128 / kPer;                                   // rows per pass
        // A thread's vector is 16 channels of a row and becomes two 16-byte chunks.  Eight lanes in a row take four
        // vectors of two rows, whose chunks fall into different banks.
        const int ct = threadIdx.x - kConvWarp * 32;
        const int piece = D == 128 ? (ct & 3) | (ct >> 1 & 4) : ct & 3, row0 = D == 128 ? (ct >> 2 & 1) | (ct >> 4 << 1) : ct >> 2;
        uint8_t* chunk0 = tile + (piece >> 2) * kSlab + row0 * 128 + ((((piece & 3) * 2) ^ (row0 & 7)) << 4);
        uint8_t* chunk1 = tile + (piece >> 2) * kSlab + row0 * 128 + ((((piece & 3) * 2 + 1) ^ (row0 & 7)) << 4);
        const int32_t* table = a.c.tables + seq * a.c.table_stride;
        const int pages = (kv + kCachePage - 1) / kCachePage, ppb = a.c.shift - 4, in_block = (1 << a.c.shift) - 1;
        // block of page `lane` of a step, -1 where there is none
        auto look_up = [&](int step) {
            const int p = (from + step * kTileRows) / kCachePage + lane;
            int b = -1;
            if (lane < kTileRows / kCachePage && p < pages) {
                b = table[p >> ppb];
                if (b < 0 || b >= a.c.num_blocks) {
                    b = -1;
                    if (a.c.status) atomicOr(a.c.status, FDMS_DEV_BAD_INDEX);
                }
            }
            return b;
        };
        auto fetch = [&](uint4 (&x)[kPer], const uint8_t* base, uint32_t sb, uint32_t sr, int step, int blocks, int left) {
            const bool whole = left >= kTileRows && (__ballot_sync(0xffffffffu, blocks >= 0) & 0xff) == 0xff;
            const uint8_t* at[kPer];
            bool use[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int row = i * kPass + row0;
                const int blk = __shfl_sync(0xffffffffu, blocks, i * (kPass / kCachePage) + row0 / kCachePage);
                use[i] = blk >= 0 && row < left;
                at[i] = base + (uint64_t)(uint32_t)blk * sb + (uint32_t)((step * kTileRows + row) & in_block) * sr;
            }
            if (whole) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) x[i] = __ldg((const uint4*)at[i]);
            } else {
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    x[i] = make_uint4(0, 0, 0, 0);
                    if (use[i]) x[i] = __ldg((const uint4*)at[i]);
                }
            }
        };
        auto put = [&](uint32_t at, const uint4 (&x)[kPer]) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                uint32_t y[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) e4m3x4_f16(w[k], y[2 * k], y[2 * k + 1]);
                *(uint4*)(chunk0 + at + i * kPass * 128) = make_uint4(y[0], y[1], y[2], y[3]);
                *(uint4*)(chunk1 + at + i * kPass * 128) = make_uint4(y[4], y[5], y[6], y[7]);
            }
        };
        const uint8_t* kb = a.c.k + head * a.c.k_sh + 16 * piece;
        const uint8_t* vb = a.c.v + head * a.c.v_sh + 16 * piece;
        const uint32_t k_sb = (uint32_t)a.c.k_sb, k_sr = (uint32_t)a.c.k_sr, v_sb = (uint32_t)a.c.v_sb, v_sr = (uint32_t)a.c.v_sr;
        // one step ahead: the codes and scales of the next step; two ahead: its blocks
        uint4 xk[kPer], xv[kPer];
        float ks = 0.0f, vs = 0.0f;
        bool held = false;                      // a page that is left out has every score -inf
        int blocks = look_up(0);
        auto scales = [&]() {
            held = blocks >= 0;
            if (warp == kConvWarp && held) {
                ks = __ldg(a.c.k_scale + (int64_t)blocks * a.c.heads + head);
                vs = __ldg(a.c.v_scale + (int64_t)blocks * a.c.heads + head);
            }
        };
        scales();
        fetch(xk, kb, k_sb, k_sr, 0, blocks, rows);
        fetch(xv, vb, v_sb, v_sr, 0, blocks, rows);
        blocks = look_up(1);
        bool ok = true;
        for (int step = 0; ok && step < steps; ++step) {
            const int st = step & 1;
            const bool more = step + 1 < steps;
            if (step >= 2) ok = warp_wait(&sh.k_empty[st], ((step >> 1) - 1) & 1, give_up);
            if (!ok) break;
            put(L::kK + st * L::kTile, xk);
            if (warp == kConvWarp && lane < kTileRows / kCachePage) {
                const float v = paged_v_scale(vs);          // a NaN is in the scores; 1 / vs also meets rows that do not see the page
                sh.page[step & (kConstRing - 1)][lane] = held ? make_float4(ks, paged_lg2(v), v == v ? __frcp_rn(v) : 1.0f, 0.0f)
                                                              : make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.k_full[st]);
            if (more) {
                scales();
                fetch(xk, kb, k_sb, k_sr, step + 1, blocks, rows - (step + 1) * kTileRows);
            }
            if (step >= 2) ok = warp_wait(&sh.v_empty[st], ((step >> 1) - 1) & 1, give_up);
            if (!ok) break;
            if ((int64_t)(step + 1) * kTileRows > open) {
                bool odd = false;
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    uint32_t* w = (uint32_t*)&xv[i];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t nan = ((w[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;      // top bit of each NaN byte
                        odd = odd || nan != 0;
                        w[k] &= ~((nan >> 7) * 0xffu);
                    }
                }
                if (odd) {
                    atomicMin(&sh.nan_lo, step);
                    atomicMax(&sh.nan_hi, step);
                }
            }
            put(L::kV + st * L::kTile, xv);
            fence_async_shared();
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.v_full[st]);
            if (more) {
                fetch(xv, vb, v_sb, v_sr, step + 1, blocks, rows - (step + 1) * kTileRows);
                blocks = look_up(step + 2);
            }
        }
    } else if (steps > 0 && warp - kMmaWarp < tiles) {
        // ---- products of a tile ----  The whole warp runs this, one elected thread issues: what the instructions take is then the same
        // for all lanes and stays in uniform registers.
        const int ti = __shfl_sync(0xffffffffu, warp - kMmaWarp, 0);
        const uint32_t base = s_addr(tile), t0 = __shfl_sync(0xffffffffu, tmem, 0);
        bool ok = warp_wait(&sh.q_full, 0, give_up);
        auto scores = [&](int h, int buf) {
            const bool again = (h >> 1) + 2 < steps;
            if (elected()) {
                if (h & 2) { if (h & 1) issue_scores<D>(base, t0, ti, 1, 1, buf, again, sh); else issue_scores<D>(base, t0, ti, 1, 0, buf, again, sh); }
                else { if (h & 1) issue_scores<D>(base, t0, ti, 0, 1, buf, again, sh); else issue_scores<D>(base, t0, ti, 0, 0, buf, again, sh); }
            }
            __syncwarp();
        };
        for (int h = 0; ok && h < L::kBufs && h < halves; ++h) {
            ok = warp_wait(&sh.k_full[(h >> 1) & 1], 0, give_up);
            tc_fence_after();
            if (ok) scores(h, h);
        }
        int buf = 0, turn = 0;
        for (int h = 0; ok && h < halves; ++h) {
            ok = warp_wait(&sh.v_full[(h >> 1) & 1], (h >> 2) & 1, give_up) && warp_wait(&sh.p_full[ti][buf], turn, give_up);
            if (!ok) break;
            tc_fence_after();
            const bool again = (h >> 1) + 2 < steps;
            if (elected()) {
                if (h & 2) {
                    if (h & 1) issue_values<D, kFine>(base, t0, ti, 1, 1, buf, true, again, sh);
                    else issue_values<D, kFine>(base, t0, ti, 1, 0, buf, true, again, sh);
                } else {
                    if (h & 1) issue_values<D, kFine>(base, t0, ti, 0, 1, buf, true, again, sh);
                    else issue_values<D, kFine>(base, t0, ti, 0, 0, buf, h > 0, again, sh);
                }
            }
            __syncwarp();
            const int next = h + L::kBufs;
            if (next < halves) {                // its scores go where the weights of this half are: they must have been read
                ok = warp_wait(&sh.k_full[(next >> 1) & 1], (next >> 2) & 1, give_up) && warp_wait(&sh.pv_done[ti][buf], turn, give_up);
                if (!ok) break;
                tc_fence_after();
                scores(next, buf);
            }
            if (++buf == L::kBufs) { buf = 0; turn ^= 1; }
        }
        // nothing of this CTA may be in flight when its memory goes, after a wait that ran out neither
        if (elected()) tc_commit(&sh.drain[ti]);
        for (int i = 0; i < kDrainPolls && !bar_test(&sh.drain[ti], 0); ++i) __nanosleep(100);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0 && sh.give_up && a.c.status) atomicOr(a.c.status, FDMS_DEV_WAIT_TIMEOUT);
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

// Joins the parts that the same tiles left: a CTA per (tile, KV head, eight of its rows), a warp per row.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(PrefillArgs a) {
    const int lane = threadIdx.x & 31, per = kTileRows / a.group;
    int seq;
    int64_t first, begin, count;
    pdl_wait();
    if (!find_tile(a, (int64_t)blockIdx.x, a.tiles * per, seq, first, begin, count)) return;
    const int hq = a.c.heads * a.group;
    const int64_t n = min((int64_t)a.tiles * per, count - first) * a.group;
    const int r = blockIdx.z * 8 + (threadIdx.x >> 5);
    if (r < n) {
        const int64_t tok = begin + first + r / a.group;
        const int h = blockIdx.y * a.group + r % a.group;
        auto part = [&](int z) { return a.parts + (((int64_t)z * a.tokens + tok) * hq + h) * (D + 4); };
        float m = lane < a.splits ? part(lane)[D] : -INFINITY, pl = lane < a.splits ? part(lane)[D + 1] : 0.0f;
        const float pm = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        // a part without a row that this one sees holds nothing
        const unsigned held = __ballot_sync(0xffffffffu, pm != -INFINITY || pl != 0.0f);
        const float w = pm == -INFINITY ? 0.0f : paged_ex2(pm - m);
        float l = pl * w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        float acc[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
#pragma unroll 4
        for (int z = 0; z < a.splits; ++z) {
            const float wz = __shfl_sync(0xffffffffu, w, z);
            if (!(held >> z & 1)) continue;
            const float* p = part(z) + lane * (D / 32);
#pragma unroll
            for (int i = 0; i < D / 32; i += 2) {
                const float2 x = *(const float2*)(p + i);
                acc[i] = fmaf(x.x, wz, acc[i]);
                acc[i + 1] = fmaf(x.y, wz, acc[i + 1]);
            }
        }
        const float inv = l > 0.0f || l != l ? __frcp_rn(l) : 0.0f;
        uint16_t* out = a.out + tok * a.o_st + (int64_t)h * a.o_sh + lane * (D / 32);
#pragma unroll
        for (int i = 0; i < D / 32; i += 2) *(uint32_t*)(out + i) = pack_pair<BF16>(acc[i] * inv, acc[i + 1] * inv);
        if (a.lse && lane == 0) a.lse[(int64_t)h * a.lse_sh + tok * a.lse_st] = kPagedLn2 * (m + paged_lg2(l));
    }
}

}  // namespace fdms

using namespace fdms;

// Tiles of rows per CTA and parts of the cached rows: the combination with the least time by what was measured, in half
// microseconds: a step of 128 keys takes 4 with one tile and 5 with two, a CTA 8 besides, the join 8 and its traffic.  The
// longest sequence that the tables can hold stands for all.
struct PrefillPlan {
    int64_t ctas;                               // per KV head
    int tiles, splits;
};
static PrefillPlan prefill_plan(int64_t tokens, int64_t seqs, int64_t heads, int group, int64_t head_dim, int64_t max_rows, int sms) {
    PrefillPlan best = {0, 0, 0};
    const int per = kTileRows / group;
    const int64_t steps = (max_rows + kTileRows - 1) / kTileRows;
    double least = 0.0;
    for (int tiles = 1; tiles <= 2; ++tiles)
        for (int splits = 1; splits <= 16 && (splits == 1 || splits * 2 <= steps); ++splits) {
            const int64_t ctas = tokens / (tiles * per) + seqs, waves = (ctas * heads * splits + sms - 1) / sms;
            const double join = splits > 1 ? 8.0 + splits * (double)tokens * heads * group * (head_dim + 4) * 8.0 / 2.5e6 : 0.0;
            const double time = waves * (8.0 + (double)((steps + splits - 1) / splits) * (3 + tiles)) + join;
            if (best.tiles == 0 || time < least) {
                best = {ctas, tiles, splits};
                least = time;
            }
        }
    return best;
}

extern "C" int64_t fdms_paged_attn_prefill_workspace_bytes(int64_t tokens, int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                                           int64_t max_rows) {
    if (tokens < 0 || num_seqs < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || num_q_heads / num_kv_heads > kTileRows / 2 ||
        head_dim <= 0 || max_rows < 0)
        return -1;
    if (tokens == 0 || num_seqs == 0) return 0;
    const int sms = paged_sms();
    if (sms <= 0) return -1;
    const int splits = prefill_plan(tokens, num_seqs, num_kv_heads, (int)(num_q_heads / num_kv_heads), head_dim, max_rows, sms).splits;
    return splits == 1 ? 0 : splits * tokens * num_q_heads * (head_dim + 4) * (int64_t)sizeof(float);
}

extern "C" int32_t fdms_paged_attn_prefill(const fdms_paged_attn_args* args, void* stream) {
    clear_error();
    PagedCache c;
    const bool idle = args && (args->num_seqs == 0 || args->tokens == 0);
    const int32_t rc = paged_attn_check("fdms_paged_attn_prefill", args, c, idle);
    if (rc != FDMS_OK) return rc;
    if (idle) return FDMS_OK;
    const fdms_paged_attn_args& p = *args;
    FDMS_REQUIRE(p.cu_seqlens_q, FDMS_E_ARG, "fdms_paged_attn_prefill: null pointer");
    const int group = (int)p.num_q_heads / c.heads, sms = paged_sms();
    FDMS_REQUIRE(sms > 0, FDMS_E_CUDA, "fdms_paged_attn_prefill: cannot read the device's SM count");
    const PrefillPlan plan = prefill_plan(p.tokens, p.num_seqs, c.heads, group, p.cache.head_dim, p.max_blocks * p.cache.block_size, sms);
    FDMS_REQUIRE(plan.ctas < (1ll << 31), FDMS_E_CAPACITY, "fdms_paged_attn_prefill: too many tokens");
    if (plan.splits > 1) {
        const int64_t need = plan.splits * p.tokens * p.num_q_heads * (p.cache.head_dim + 4) * (int64_t)sizeof(float);
        FDMS_REQUIRE(p.workspace && ((uintptr_t)p.workspace & 15) == 0 && p.workspace_bytes >= need, FDMS_E_WORKSPACE,
                     "fdms_paged_attn_prefill: workspace missing, unaligned or smaller than %lld bytes", (long long)need);
    }
    PrefillArgs a = {c, (const uint16_t*)p.q, (uint16_t*)p.out, p.lse_out, p.cu_seqlens_q, p.q_stride[0], p.q_stride[1], p.out_stride[0],
                     p.out_stride[1], p.lse_stride[0], p.lse_stride[1], p.tokens, (float*)p.workspace, (int32_t)p.num_seqs, group, plan.tiles,
                     plan.splits, (float)p.scale};
    const dim3 grid((unsigned)plan.ctas, (unsigned)c.heads, (unsigned)plan.splits), jgrid((unsigned)plan.ctas, (unsigned)c.heads, (unsigned)(plan.tiles * kTileRows / 8));
    cudaStream_t st = (cudaStream_t)stream;
    const bool bf = p.dtype == FDMS_BF16;
#define FDMS_PREFILL(DIM, BF)                                                                                                           \
    do {                                                                                                                                \
        constexpr int bytes = (int)PrefillSmem<DIM>::kBytes;                                                                            \
        FDMS_CUDA_OK(cudaFuncSetAttribute(paged_prefill_kernel<DIM, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));           \
        paged_prefill_kernel<DIM, BF><<<grid, kPreThreads, bytes, st>>>(a);                                                             \
        FDMS_CHECK_LAUNCH("paged_prefill_kernel");                                                                                      \
        if (plan.splits > 1) FDMS_CUDA_OK(launch_chained(paged_prefill_join_kernel<DIM, BF>, jgrid, dim3(256), st, true, a));             \
    } while (0)
    if (p.cache.head_dim == 64) {
        if (bf) FDMS_PREFILL(64, true); else FDMS_PREFILL(64, false);
    } else {
        if (bf) FDMS_PREFILL(128, true); else FDMS_PREFILL(128, false);
    }
#undef FDMS_PREFILL
    FDMS_CHECK_LAUNCH("paged_prefill_join_kernel");
    return FDMS_OK;
}
