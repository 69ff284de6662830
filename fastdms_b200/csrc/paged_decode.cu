// Decode attention over the block-scaled paged cache: one new token per sequence, its q heads against the sequence's
// cached rows (the new one among them).
//
// The work is the cache's bytes, each to be read once: the pages (16 rows) of all (sequence, KV head) units are laid end to
// end and every CTA takes an equal share of them, so that ragged lengths leave no SM idle and no host has to know a
// length.  A CTA walks the units its share touches; its eight warps take every eighth page and keep (M, l, O) of the
// unit's q heads in registers, merged through shared memory at the end of a unit.  A unit that one CTA holds whole is
// written at once; parts of a unit that is cut go to a workspace, and a second launch, started while this one runs, joins
// them.
#include "paged_attn.cuh"

namespace fdms {

constexpr int kDecWarps = 8;
constexpr int kDecThreads = kDecWarps * 32;
constexpr int kDecHeads = 8;                    // q heads of a KV head that one unit takes
constexpr int kDecMaxBatch = 2048;              // prefix sums of the pages live in shared memory
constexpr int kDecCtasPerSm = 2;

struct DecodeArgs {
    PagedCache c;
    const uint16_t* q;
    uint16_t* out;
    float* lse;                                 // optional [batch, q_heads]
    int64_t q_sb, q_sh, o_sb, o_sh, lse_sb, lse_sh;
    float* parts;                               // [ctas][2][kDecHeads][D + 2]: O, M, l
    int2* cuts;                                 // [units] first part and last CTA of a unit that is cut, (0, -1) of others
    int32_t batch, group, splits;               // splits: units per (sequence, KV head), each of up to 8 q heads
    float scale;
};

// Pages before sequence b for all b (and in total), in shared memory; by all threads of the CTA.
__device__ __forceinline__ void page_prefix(const DecodeArgs& a, int32_t* s_first, int32_t* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int32_t before = 0;
    for (int base = 0; base < a.batch; base += kDecThreads) {
        const int b = base + threadIdx.x;
        const int pages = b < a.batch ? (int)(((int64_t)paged_len(a.c, b) + kCachePage - 1) / kCachePage) : 0;
        int sum = pages;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        if (lane == 31) s_warp[warp] = sum;
        __syncthreads();
        int add = before, total = 0;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
            if (w < warp) add += s_warp[w];
            total += s_warp[w];
        }
        if (b < a.batch) s_first[b] = add + sum - pages;
        before += total;
        __syncthreads();
    }
    if (threadIdx.x == 0) s_first[a.batch] = before;
    __syncthreads();
}

// The share of CTA `c` of `n` in `total` pages begins at share(c); page x belongs to CTA owner(x).
__device__ __forceinline__ int64_t share(int64_t c, int64_t n, int64_t total) { return c * total / n; }
__device__ __forceinline__ int owner(int64_t x, int64_t n, int64_t total) { return (int)(((x + 1) * n - 1) / total); }

template <int D, bool BF16>
__global__ void __launch_bounds__(kDecThreads, kDecCtasPerSm) paged_decode_kernel(DecodeArgs a) {
    extern __shared__ int32_t s_first[];        // batch + 1
    __shared__ int32_t s_warp[kDecWarps];
    __shared__ float s_o[kDecWarps][kDecHeads][D];
    __shared__ float s_m[kDecWarps][kDecHeads], s_l[kDecWarps][kDecHeads];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    pdl_trigger();
    page_prefix(a, s_first, s_warp);
    const int per_seq = a.c.heads * a.splits;
    const int64_t total = (int64_t)s_first[a.batch] * per_seq;
    // fewer CTAs than the grid has where there are not two pages for each warp
    const int64_t ctas = min((int64_t)gridDim.x, max((int64_t)1, (total + 2 * kDecWarps - 1) / (2 * kDecWarps)));
    if (blockIdx.x == 0) {                      // sequences without rows: zeros
        for (int b = warp; b < a.batch; b += kDecWarps) {
            if (s_first[b + 1] != s_first[b]) continue;
            const int hq = a.c.heads * a.group;
            for (int i = lane; i < hq * (D / 8); i += 32)
                *(uint4*)(a.out + b * a.o_sb + (i / (D / 8)) * a.o_sh + (i % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
            if (a.lse)
                for (int i = lane; i < hq; i += 32) a.lse[b * a.lse_sb + i * a.lse_sh] = -INFINITY;
            for (int i = lane; i < per_seq; i += 32) a.cuts[(int64_t)b * per_seq + i] = make_int2(0, -1);
        }
    }
    if (blockIdx.x >= ctas) return;
    const int64_t begin = share(blockIdx.x, ctas, total), end = share((int64_t)blockIdx.x + 1, ctas, total);
    int seq = 0;                                // last sequence whose pages begin at or before `begin`, and has any
    {
        int lo = 0, hi = a.batch;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if ((int64_t)s_first[mid + 1] * per_seq > begin) hi = mid; else lo = mid + 1;
        }
        seq = lo;
    }
    const int ppb = a.c.shift - 4;              // log2(pages per block)
    int64_t at = begin;
    while (at < end) {
        while ((int64_t)s_first[seq + 1] * per_seq <= at) ++seq;
        const int pages = s_first[seq + 1] - s_first[seq];
        const int64_t seq_begin = (int64_t)s_first[seq] * per_seq;
        const int u = (int)((at - seq_begin) / pages);          // unit of the sequence
        const int64_t unit_begin = seq_begin + (int64_t)u * pages;
        const int p0 = (int)(at - unit_begin), p1 = (int)min((int64_t)pages, end - unit_begin);
        const int head = u / a.splits, h0 = (u % a.splits) * kDecHeads, nh = min(kDecHeads, a.group - h0);
        const int len = min(paged_len(a.c, seq), pages * kCachePage);

        // query fragments: row g of the unit's heads
        uint32_t qa[D / 16][2];
        float factor = 0.0f;
        {
            const uint16_t* q = a.q + seq * a.q_sb + (int64_t)(head * a.group + h0 + min(g, nh - 1)) * a.q_sh;
            uint4 w[D / 64][2];
            float top = 0.0f;
#pragma unroll
            for (int n = 0; n < D / 64; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    w[n][i] = *(const uint4*)(q + 64 * n + 16 * t + 8 * i);
                    const uint32_t x[4] = {w[n][i].x, w[n][i].y, w[n][i].z, w[n][i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float e, f;
                        unpack_pair<BF16>(x[j], e, f);
                        top = fmaxf(top, fmaxf(fabsf(e), fabsf(f)));
                    }
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            float up;
            row_power(top, up, factor);
            factor *= a.scale * kPagedLog2e;
#pragma unroll
            for (int n = 0; n < D / 64; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t x[4] = {w[n][i].x, w[n][i].y, w[n][i].z, w[n][i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float e, f;
                        unpack_pair<BF16>(x[j], e, f);
                        // element 16 t + 8 i + 2 j of the chunk: step 2 i + j / 2, half j % 2
                        qa[4 * n + 2 * i + (j >> 1)][j & 1] = f16x2_of(e * up, f * up);
                    }
                }
        }
        float o[D / 8][2], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = 0.0f;

        // the warp's pages: p0 + warp + 8 i; 32 of them at a time, one per lane, are looked up in the table
        const int mine = p1 - p0 > warp ? (p1 - p0 - warp + kDecWarps - 1) / kDecWarps : 0;
        for (int base = 0; base < mine; base += 32) {
            int my_block = -1;
            float my_ks = 0.0f, my_vs = 1.0f;
            if (base + lane < mine) {
                const int p = p0 + warp + kDecWarps * (base + lane);
                my_block = a.c.tables[seq * a.c.table_stride + (p >> ppb)];
                if (my_block < 0 || my_block >= a.c.num_blocks) {
                    my_block = -1;
                    if (a.c.status) atomicOr(a.c.status, FDMS_DEV_BAD_INDEX);
                } else {
                    my_ks = a.c.k_scale[(int64_t)my_block * a.c.heads + head];
                    my_vs = a.c.v_scale[(int64_t)my_block * a.c.heads + head];
                }
            }
            const float my_lvs = paged_lg2(my_vs), my_ivs = __frcp_rn(my_vs);
            const int n = min(32, mine - base);
            PageRegs<D> pg;
            auto fetch_k = [&](int i) {
                const int blk = __shfl_sync(0xffffffffu, my_block, i);
                const int p = p0 + warp + kDecWarps * (base + i);
                const int row = (p & ((1 << ppb) - 1)) * kCachePage;
                if (blk >= 0) load_k<D>(pg, a.c.k + (int64_t)blk * a.c.k_sb + head * a.c.k_sh + row * a.c.k_sr, a.c.k_sr, lane);
            };
            auto fetch_v = [&](int i) {
                const int blk = __shfl_sync(0xffffffffu, my_block, i);
                const int p = p0 + warp + kDecWarps * (base + i);
                const int row = (p & ((1 << ppb) - 1)) * kCachePage;
                if (blk >= 0) load_v<D>(pg, a.c.v + (int64_t)blk * a.c.v_sb + head * a.c.v_sh + row * a.c.v_sr, a.c.v_sr, lane);
            };
            zero_page<D>(pg);
            fetch_k(0);
            fetch_v(0);
            for (int i = 0; i < n; ++i) {
                const int blk = __shfl_sync(0xffffffffu, my_block, i);
                const float ks = __shfl_sync(0xffffffffu, my_ks, i) * factor;
                const float lvs = __shfl_sync(0xffffffffu, my_lvs, i), ivs = __shfl_sync(0xffffffffu, my_ivs, i);
                const int p = p0 + warp + kDecWarps * (base + i);
                const int rows = blk < 0 ? 0 : min(kCachePage, len - p * kCachePage);
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < D / 64; ++c) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t b0, b1;
                        e4m3x4_f16(j == 0 ? pg.k[0][c].x : j == 1 ? pg.k[0][c].y : j == 2 ? pg.k[0][c].z : pg.k[0][c].w, b0, b1);
                        mma_816(s[0], s[1], qa[4 * c + j][0], qa[4 * c + j][1], b0, b1);
                        e4m3x4_f16(j == 0 ? pg.k[1][c].x : j == 1 ? pg.k[1][c].y : j == 2 ? pg.k[1][c].z : pg.k[1][c].w, b0, b1);
                        mma_816(s[2], s[3], qa[4 * c + j][0], qa[4 * c + j][1], b0, b1);
                    }
                }
                if (i + 1 < n) fetch_k(i + 1);
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[j] = 4 * t + j < rows ? fmaf(s[j], ks, lvs) : -INFINITY;
                    top = fmaxf(top, s[j]);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // M follows the maximum only when it lags by more than 2^8: P stays below 256, and most pages rescale nothing
                if (__any_sync(0xffffffffu, top > m + 8.0f)) {
                    const float next = fmaxf(m, top);
                    const float r = next == -INFINITY ? 1.0f : paged_ex2(m - next);
                    m = next;
                    l *= r;
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) { o[j][0] *= r; o[j][1] *= r; }
                }
                const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] = paged_ex2(s[j] - ref);
                l = fmaf((s[0] + s[1]) + (s[2] + s[3]), ivs, l);
                const uint32_t a0 = f16x2_of(s[0], s[1]), a2 = f16x2_of(s[2], s[3]);
                if (rows < kCachePage) mask_v<D>(pg, rows, lane);
#pragma unroll
                for (int w = 0; w < D / 32; ++w) {
                    const uint32_t k0 = v_word<D>(pg, 0, w), k1 = v_word<D>(pg, 1, w), k2 = v_word<D>(pg, 2, w), k3 = v_word<D>(pg, 3, w);
                    uint32_t b0[4], b1[4];
                    e4m3x4_f16(__byte_perm(k0, k1, 0x5140), b0[0], b0[1]);
                    e4m3x4_f16(__byte_perm(k0, k1, 0x7362), b0[2], b0[3]);
                    e4m3x4_f16(__byte_perm(k2, k3, 0x5140), b1[0], b1[1]);
                    e4m3x4_f16(__byte_perm(k2, k3, 0x7362), b1[2], b1[3]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma_816(o[4 * w + j][0], o[4 * w + j][1], a0, a2, b0[j], b1[j]);
                }
                if (i + 1 < n) fetch_v(i + 1);
            }
        }
        // merge the warps: lane (g, t) holds head g, channels (D/8) (2t) + j and (D/8) (2t + 1) + j
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) { s_m[warp][g] = m; s_l[warp][g] = l; }
#pragma unroll
        for (int j = 0; j < D / 8; j += 4)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                *(float4*)&s_o[warp][g][(D / 8) * (2 * t + i) + j] = make_float4(o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]);
        __syncthreads();
        const bool whole = p0 == 0 && p1 == pages;
        const int slot = blockIdx.x * 2 + (at == begin ? 0 : 1);
        constexpr int kVec = kDecHeads * D / kDecThreads;       // channels per thread: a head is D / kVec threads
        const int hd = threadIdx.x / (D / kVec), ch = (threadIdx.x % (D / kVec)) * kVec;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) mm = fmaxf(mm, s_m[w][hd]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float ll = 0.0f, acc[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) acc[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
            const float r = paged_ex2(s_m[w][hd] - ref);
            ll = fmaf(s_l[w][hd], r, ll);
#pragma unroll
            for (int i = 0; i < kVec; ++i) acc[i] = fmaf(s_o[w][hd][ch + i], r, acc[i]);
        }
        if (whole) {
            if (hd < nh) {
                const float inv = ll > 0.0f || ll != ll ? 1.0f / ll : 0.0f;
                uint16_t* out = a.out + seq * a.o_sb + (int64_t)(head * a.group + h0 + hd) * a.o_sh + ch;
#pragma unroll
                for (int i = 0; i < kVec; i += 2) *(uint32_t*)(out + i) = pack_pair<BF16>(acc[i] * inv, acc[i + 1] * inv);
                if (a.lse && ch == 0)
                    a.lse[seq * a.lse_sb + (int64_t)(head * a.group + h0 + hd) * a.lse_sh] = kPagedLn2 * (mm + paged_lg2(ll));
            }
        } else {
            float* part = a.parts + ((int64_t)slot * kDecHeads + hd) * (D + 4);
#pragma unroll
            for (int i = 0; i < kVec; i += 2) *(float2*)(part + ch + i) = make_float2(acc[i], acc[i + 1]);
            if (ch == 0) *(float2*)(part + D) = make_float2(mm, ll);
        }
        if (p0 == 0 && threadIdx.x == 0) {
            const int2 cut = whole ? make_int2(0, -1) : make_int2(slot, owner(unit_begin + pages - 1, ctas, total));
            a.cuts[(int64_t)seq * per_seq + u] = cut;
        }
        __syncthreads();
        at = unit_begin + p1;
    }
}

// Joins the parts of the units that were cut: one warp per (sequence, q head), D / 32 channels a lane.  The first part is
// where the unit's first CTA put it; every later CTA's share begins inside the unit, so its part is its first one.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) paged_decode_join_kernel(DecodeArgs a, int64_t rows) {
    const int lane = threadIdx.x & 31;
    const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_wait();
    if (r >= rows) return;
    const int hq = a.c.heads * a.group, per_seq = a.c.heads * a.splits;
    const int64_t seq = r / hq;
    const int h = (int)(r - seq * hq), head = h / a.group, j = h % a.group, u = head * a.splits + j / kDecHeads, hd = j % kDecHeads;
    const int2 cut = a.cuts[seq * per_seq + u];
    const int first = cut.x >> 1;
    if (cut.y < first) return;
    auto part = [&](int c) { return a.parts + ((int64_t)(c == first ? cut.x : 2 * c) * kDecHeads + hd) * (D + 4); };
    float m = -INFINITY;
    for (int c = first + lane; c <= cut.y; c += 32) m = fmaxf(m, part(c)[D]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float ref = m == -INFINITY ? 0.0f : m;
    constexpr int kVec = D / 32;
    float l = 0.0f, acc[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) acc[i] = 0.0f;
#pragma unroll 4
    for (int c = first; c <= cut.y; ++c) {
        const float* p = part(c);
        const float2 ml = *(const float2*)(p + D);
        const float w = paged_ex2(ml.x - ref);
        l = fmaf(ml.y, w, l);
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const float2 x = *(const float2*)(p + lane * kVec + i);
            acc[i] = fmaf(x.x, w, acc[i]);
            acc[i + 1] = fmaf(x.y, w, acc[i + 1]);
        }
    }
    const float inv = l > 0.0f || l != l ? __frcp_rn(l) : 0.0f;
    uint16_t* out = a.out + seq * a.o_sb + (int64_t)h * a.o_sh + lane * kVec;
#pragma unroll
    for (int i = 0; i < kVec; i += 2) *(uint32_t*)(out + i) = pack_pair<BF16>(acc[i] * inv, acc[i + 1] * inv);
    if (a.lse && lane == 0) a.lse[seq * a.lse_sb + (int64_t)h * a.lse_sh] = kPagedLn2 * (m + paged_lg2(l));
}

}  // namespace fdms

using namespace fdms;

static int paged_sms() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    return n;
}

static int64_t decode_parts_bytes(int sms, int head_dim) {
    return (int64_t)sms * kDecCtasPerSm * 2 * kDecHeads * (head_dim + 4) * (int64_t)sizeof(float);
}

extern "C" int64_t fdms_paged_attn_decode_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim) {
    if (batch < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || head_dim <= 0) return -1;
    const int sms = paged_sms();
    if (sms <= 0) return -1;
    const int group = num_q_heads / num_kv_heads;
    return decode_parts_bytes(sms, head_dim) + (int64_t)batch * num_kv_heads * ((group + kDecHeads - 1) / kDecHeads) * (int64_t)sizeof(int2);
}

extern "C" int32_t fdms_paged_attn_decode(const fdms_paged_attn_args* args, void* stream) {
    clear_error();
    DecodeArgs a;
    const bool idle = args && args->num_seqs == 0;
    const int32_t rc = paged_attn_check("fdms_paged_attn_decode", args, a.c, idle);
    if (rc != FDMS_OK) return rc;
    const fdms_paged_attn_args& p = *args;
    const int num_q_heads = (int)p.num_q_heads, num_kv_heads = a.c.heads, head_dim = (int)p.cache.head_dim;
    FDMS_REQUIRE(p.tokens == p.num_seqs, FDMS_E_ARG, "fdms_paged_attn_decode: one token per sequence, got %lld for %lld", (long long)p.tokens,
                 (long long)p.num_seqs);
    FDMS_REQUIRE(p.num_seqs <= kDecMaxBatch, FDMS_E_CAPACITY, "fdms_paged_attn_decode: at most %d sequences a call, got %lld", kDecMaxBatch,
                 (long long)p.num_seqs);
    if (idle) return FDMS_OK;
    const int batch = (int)p.num_seqs;
    const int sms = paged_sms();
    FDMS_REQUIRE(sms > 0, FDMS_E_CUDA, "fdms_paged_attn_decode: cannot read the device's SM count");
    const int64_t need = fdms_paged_attn_decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim);
    FDMS_REQUIRE(p.workspace && ((uintptr_t)p.workspace & 15) == 0 && p.workspace_bytes >= need, FDMS_E_WORKSPACE,
                 "fdms_paged_attn_decode: workspace missing, unaligned or smaller than %lld bytes", (long long)need);
    a.q = (const uint16_t*)p.q;
    a.out = (uint16_t*)p.out;
    a.lse = p.lse_out;
    a.q_sb = p.q_stride[0]; a.q_sh = p.q_stride[1]; a.o_sb = p.out_stride[0]; a.o_sh = p.out_stride[1];
    a.lse_sb = p.lse_stride[0]; a.lse_sh = p.lse_stride[1];
    a.parts = (float*)p.workspace;
    a.cuts = (int2*)((char*)p.workspace + decode_parts_bytes(sms, head_dim));
    a.batch = batch;
    a.group = num_q_heads / num_kv_heads;
    a.splits = (a.group + kDecHeads - 1) / kDecHeads;
    a.scale = (float)p.scale;
    const int64_t rows_held = (int64_t)batch * p.max_blocks * (p.cache.block_size / kCachePage);
    FDMS_REQUIRE(rows_held < (1ll << 31), FDMS_E_CAPACITY, "fdms_paged_attn_decode: the block tables hold too many rows");
    const int64_t useful = (rows_held * num_kv_heads * a.splits + 2 * kDecWarps - 1) / (2 * kDecWarps);
    const unsigned grid = (unsigned)(useful < 1 ? 1 : useful < (int64_t)sms * kDecCtasPerSm ? useful : (int64_t)sms * kDecCtasPerSm);
    const size_t smem = (size_t)(batch + 1) * sizeof(int32_t);
    cudaStream_t st = (cudaStream_t)stream;
    const bool bf = p.dtype == FDMS_BF16;
    const int64_t rows = (int64_t)batch * num_q_heads;
    const dim3 jgrid((unsigned)((rows + 7) / 8));
#define FDMS_DECODE(DIM, BF)                                                                                        \
    do {                                                                                                            \
        paged_decode_kernel<DIM, BF><<<grid, kDecThreads, smem, st>>>(a);                                           \
        FDMS_CHECK_LAUNCH("paged_decode_kernel");                                                                   \
        FDMS_CUDA_OK(launch_chained(paged_decode_join_kernel<DIM, BF>, jgrid, dim3(256), st, true, a, rows));       \
    } while (0)
    if (head_dim == 64) {
        if (bf) FDMS_DECODE(64, true); else FDMS_DECODE(64, false);
    } else {
        if (bf) FDMS_DECODE(128, true); else FDMS_DECODE(128, false);
    }
#undef FDMS_DECODE
    FDMS_CHECK_LAUNCH("paged_decode_join_kernel");
    return FDMS_OK;
}
