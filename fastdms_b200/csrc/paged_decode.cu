// Decode attention over the block-scaled paged cache: one new token per sequence, its q heads against the sequence's
// cached rows (the new one among them).
//
// The work is the cache's bytes, each to be read once.  A unit is a (sequence, KV head), with up to eight of its q heads; the
// eight warps of a CTA take pages (16 rows) in turn, keep (M, l, O) in registers and merge them through shared memory.
// Two kernels hand out the pages:
//   clusters  a cluster of 1 to 16 CTAs per unit, whose parts meet in distributed shared memory: one launch, no workspace.  For
//             tables that cannot hold long sequences, and for work that is small altogether.
//   shares    the pages of all units laid end to end, every CTA taking an equal share of them, so that ragged lengths leave
//             no SM idle and no host has to know a length.  A unit that one CTA holds whole is written at once; parts of a
//             unit that is cut go to a workspace, and a second launch, started while this one runs, joins them.
// Measured from memory (32 q heads on 8 KV heads): 64 sequences ragged up to 16384 rows at head_dim 128 read their 1.08 GB in
// 190 us (5.7 TB/s) in bf16 and 199 in f16; 8 sequences at head_dim 64 take about 6 us and then read at 4.9 TB/s (8192 rows: 67 MB in
// 20 us, f16 21); one sequence of 200 rows takes 5.7 us, a chain of latencies.
#include "paged_attn.cuh"

#include <algorithm>
#include <climits>
#include <mutex>

namespace fdms {

constexpr int kDecWarps = 8;
constexpr int kDecThreads = kDecWarps * 32;
constexpr int kDecHeads = 8;                    // q heads of a KV head that one unit takes
constexpr int kDecMaxBatch = 2048;              // prefix sums of the pages live in shared memory
constexpr int kDecCtasPerSm = 2;
constexpr int kClusterSizes = 5, kMaxCluster = 1 << (kClusterSizes - 1), kMaxDevices = 64;

struct DecodeArgs {
    PagedCache c;
    const uint16_t* q;
    uint16_t* out;
    float* lse;                                 // optional [tokens, q_heads]
    const int32_t* cu;                          // [batch + 1] where each sequence's token lies, or null: token b is sequence b's
    int64_t q_sb, q_sh, o_sb, o_sh, lse_sb, lse_sh;
    float* parts;                               // [ctas][2][kDecHeads][D + 4]: O, M, l
    int2* cuts;                                 // [units] first part and last CTA of a unit that is cut, (0, -1) of others
    int32_t batch, tokens, group, splits;       // splits: units per (sequence, KV head), each of up to 8 q heads
    int32_t cluster;                            // CTAs per unit (clusters)
    float scale;
};

// Row of q and out that holds sequence b's token; -1 where it has none in this step, or not exactly one.
__device__ __forceinline__ int token_of(const DecodeArgs& a, int b) {
    if (!a.cu) return b;
    const int at = a.cu[b], end = a.cu[b + 1];
    if (at >= 0 && at < a.tokens && end == at + 1) return at;
    if (end != at && a.c.status) atomicOr(a.c.status, FDMS_DEV_BAD_INDEX);
    return -1;
}

// One 16-row page as matrix operands; lane (g, t) = (lane / 4, lane % 4).  Both products run transposed, the page's codes
// being the 16-row operand and up to 8 q heads the 8 columns, so that no row of a fragment is idle:
//   S^T = K Q^T: A holds keys g and g + 8; in chunk n (64 bytes of a row) lane t brings bytes 64 n + 16 t + [0, 16), four of
//   them for each of four steps of 16 channels, and the query fragment is loaded in the same order.
//   O^T = V^T P^T: A holds channels; of keys 2t, 2t + 1, 2t + 8, 2t + 9 a lane loads D / 8 consecutive bytes, tile j taking
//   channels (D / 8) g + 2j and + 1 as its rows g and g + 8.  P^T comes out of S^T's layout by an 8x8 transpose in the warp.
template <int D>
struct PageRegs {
    uint4 k[2][D / 64];         // keys g, g + 8; chunks
    uint4 v[D == 128 ? 4 : 2];  // keys 2t, 2t + 1, 2t + 8, 2t + 9 (D = 64: two keys per vector)
};

template <int D>
__device__ __forceinline__ void load_k(PageRegs<D>& p, const uint8_t* k, uint32_t sr) {     // k: the lane's first vector
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < D / 64; ++n) p.k[i][n] = __ldg((const uint4*)(k + 8 * i * sr + 64 * n));
}
template <int D>
__device__ __forceinline__ void load_v(PageRegs<D>& p, const uint8_t* v, uint32_t sr) {
    if (D == 128) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p.v[i] = __ldg((const uint4*)(v + ((i & 1) + 8 * (i >> 1)) * sr));
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint2 a = __ldg((const uint2*)(v + 8 * i * sr)), b = __ldg((const uint2*)(v + (8 * i + 1) * sr));
            p.v[i] = make_uint4(a.x, a.y, b.x, b.y);
        }
    }
}
// Word w (channels 4w .. 4w + 3 of the lane's) of the lane's key i.
template <int D>
__device__ __forceinline__ uint32_t v_word(const PageRegs<D>& p, int i, int w) {
    const uint4& x = D == 128 ? p.v[i] : p.v[i >> 1];
    const int n = D == 128 ? w : (i & 1) * 2 + w;
    return n == 0 ? x.x : n == 1 ? x.y : n == 2 ? x.z : x.w;
}
// Rows at and beyond `rows` hold whatever the memory held: zero, so that P = 0 leaves no trace of them.
template <int D>
__device__ __forceinline__ void mask_v(PageRegs<D>& p, int rows, int t) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (2 * t + (i & 1) + 8 * (i >> 1) >= rows) {
            if (D == 128) p.v[i] = make_uint4(0, 0, 0, 0);
            else if (i & 1) p.v[i >> 1].z = p.v[i >> 1].w = 0;
            else p.v[i >> 1].x = p.v[i >> 1].y = 0;
        }
}

// What a warp keeps of a unit: lane (g, t) holds heads 2t and 2t + 1, channels (D / 8) g + [0, D / 8) in o (o[j]: channel
// 2j of both heads, channel 2j + 1 of both), M of the two heads and its share of l.
template <int D>
struct UnitState {
    float o[D / 16][4];
    float m[2], l[2];
};

template <int D>
__device__ __forceinline__ void clear(UnitState<D>& u) {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) u.o[j][0] = u.o[j][1] = u.o[j][2] = u.o[j][3] = 0.0f;
    u.m[0] = u.m[1] = -INFINITY;
    u.l[0] = u.l[1] = 0.0f;
}

// Query fragments of head `row` (column g of the products), brought to a power of two; the factor of the scores of heads
// 2t and 2t + 1 comes from the lanes that loaded them.
template <int D, bool BF16>
__device__ __forceinline__ void load_q(const uint16_t* q, float scale, uint32_t (&qb)[D / 16][2], float (&factor)[2], int lane) {
    const int t = lane & 3;
    uint4 w[D / 64][2];
    float top = 0.0f;
#pragma unroll
    for (int n = 0; n < D / 64; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) w[n][i] = *(const uint4*)(q + 64 * n + 16 * t + 8 * i);
#pragma unroll
    for (int n = 0; n < D / 64; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
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
    float up, down;
    row_power(top, up, down);
    down *= scale * kPagedLog2e;
    factor[0] = __shfl_sync(0xffffffffu, down, 8 * t);
    factor[1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
#pragma unroll
    for (int n = 0; n < D / 64; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t x[4] = {w[n][i].x, w[n][i].y, w[n][i].z, w[n][i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {       // element 16 t + 8 i + 2 j of the chunk: step 2 i + j / 2, half j % 2
                float e, f;
                unpack_pair<BF16>(x[j], e, f);
                qb[4 * n + 2 * i + (j >> 1)][j & 1] = f16x2_of(e * up, f * up);
            }
        }
}

// S^T of a page.
template <int D>
__device__ __forceinline__ void page_scores(const PageRegs<D>& p, const uint32_t (&qb)[D / 16][2], float (&s)[4]) {
    s[0] = s[1] = s[2] = s[3] = 0.0f;
#pragma unroll
    for (int n = 0; n < D / 64; ++n) {
        const uint32_t x[4] = {p.k[0][n].x, p.k[0][n].y, p.k[0][n].z, p.k[0][n].w}, y[4] = {p.k[1][n].x, p.k[1][n].y, p.k[1][n].z, p.k[1][n].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t a0, a1, a2, a3;
            e4m3x4_f16(x[j], a0, a2);
            e4m3x4_f16(y[j], a1, a3);
            mma_16816(s, a0, a1, a2, a3, qb[4 * n + j][0], qb[4 * n + j][1]);
        }
    }
}

// log2 of the largest weight when M is set, and of the most that one may be until M moves.  With 11 and 15 more of the quiet weights
// count, and 64 sequences ragged up to 16384 take 191.5 us in place of 190.2.  What a weight may be is judged by the difference to M,
// which is exact, while M +- a few is not where float32's steps are wider than these; 7, less than half a step of 16, is then
// rounded away from or up to 8, and a weight's power never passes 15.
constexpr float kTopWeight = 7.0f, kMostWeight = 15.0f;

// Scores to weights, l, and P^T; `rows` of the page count.  M follows the maximum only when that is ahead by more than 2^8:
// P stays at or below 2^15 and most pages need no maximum over the keys and rescale nothing.
// With FINE, for f16 outputs, whose own rounding is no larger than that of a weight to f16, also what that rounding left.
template <int D, bool FINE>
__device__ __forceinline__ void page_weights(UnitState<D>& u, float (&s)[4], float ks, float lvs, float ivs, const float (&factor)[2], int rows,
                                             int lane, uint32_t (&b)[4]) {
    const int g = lane >> 2;
    const float f0 = ks * factor[0], f1 = ks * factor[1];
    float x[4] = {fmaf(s[0], f0, lvs), fmaf(s[1], f1, lvs), fmaf(s[2], f0, lvs), fmaf(s[3], f1, lvs)};
    if (rows < kCachePage) {
        if (g >= rows) x[0] = x[1] = -INFINITY;
        if (g + 8 >= rows) x[2] = x[3] = -INFINITY;
    }
    const float t0 = fmaxf(x[0], x[2]), t1 = fmaxf(x[1], x[3]);
    if (__any_sync(0xffffffffu, t0 - u.m[0] > kMostWeight || t1 - u.m[1] > kMostWeight)) {
        float top[2] = {t0, t1};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
            const float next = top[i] - u.m[i] > kMostWeight ? top[i] - kTopWeight : u.m[i];      // heads do not follow their neighbours
            const float r = next == u.m[i] ? 1.0f : paged_ex2(u.m[i] - next);
            u.m[i] = next;
            u.l[i] *= r;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) { u.o[j][i] *= r; u.o[j][2 + i] *= r; }
        }
    }
    const float r0 = u.m[0] == -INFINITY ? 0.0f : u.m[0], r1 = u.m[1] == -INFINITY ? 0.0f : u.m[1];
    x[0] = paged_ex2(x[0] - r0);
    x[2] = paged_ex2(x[2] - r0);
    x[1] = paged_ex2(x[1] - r1);
    x[3] = paged_ex2(x[3] - r1);
    u.l[0] = fmaf(x[0] + x[2], ivs, u.l[0]);
    u.l[1] = fmaf(x[1] + x[3], ivs, u.l[1]);
    const uint32_t p0 = f16x2_of(x[0], x[1]), p1 = f16x2_of(x[2], x[3]);
    b[0] = transpose_8x8(p0);
    b[1] = transpose_8x8(p1);
    if (FINE) {
        const __half2 h0 = *(const __half2*)&p0, h1 = *(const __half2*)&p1;
        b[2] = transpose_8x8(f16x2_of(x[0] - __low2float(h0), x[1] - __high2float(h0)));
        b[3] = transpose_8x8(f16x2_of(x[2] - __low2float(h1), x[3] - __high2float(h1)));
    }
}

// O^T of a page.
template <int D, bool FINE>
__device__ __forceinline__ void page_values(UnitState<D>& u, const PageRegs<D>& p, const uint32_t (&b)[4]) {
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
        const uint32_t k0 = v_word<D>(p, 0, w), k1 = v_word<D>(p, 1, w), k2 = v_word<D>(p, 2, w), k3 = v_word<D>(p, 3, w);
        uint32_t a[2][4];
        e4m3x4_f16(__byte_perm(k0, k1, 0x5140), a[0][0], a[0][1]);
        e4m3x4_f16(__byte_perm(k0, k1, 0x7362), a[1][0], a[1][1]);
        e4m3x4_f16(__byte_perm(k2, k3, 0x5140), a[0][2], a[0][3]);
        e4m3x4_f16(__byte_perm(k2, k3, 0x7362), a[1][2], a[1][3]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            mma_16816(u.o[2 * w + j], a[j][0], a[j][1], a[j][2], a[j][3], b[0], b[1]);
            if (FINE) mma_16816(u.o[2 * w + j], a[j][0], a[j][1], a[j][2], a[j][3], b[2], b[3]);
        }
    }
}

// Table entry of page first + step * (base + lane), read ahead of everything that says whether the page exists: any column
// of the sequence's row may be read.
__device__ __forceinline__ int entry_ahead(const PagedCache& c, int seq, int first, int step, int base) {
    const int64_t col = ((int64_t)first + (int64_t)step * (base + (int)(threadIdx.x & 31))) >> (c.shift - 4);
    return col < c.max_blocks ? c.tables[seq * c.table_stride + col] : -1;
}

// The warp's pages first, first + step, ... (`count` of them) of a sequence's KV head, whose first `len` rows count.  Their
// table entries and scales are held 32 pages at a time, one per lane: `entry` are the first 32, the next are requested while
// these are walked.
template <int D, bool FINE>
__device__ __forceinline__ void walk_pages(const PagedCache& c, UnitState<D>& u, const uint32_t (&qb)[D / 16][2], const float (&factor)[2],
                                           int seq, int head, int first, int step, int count, int len, int entry) {
    if (count <= 0) return;
    if (c.num_blocks == 0) {                    // a needed page that no block is
        if (c.status) atomicOr(c.status, FDMS_DEV_BAD_INDEX);
        return;
    }
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int in_block = (1 << (c.shift - 4)) - 1;
    const uint32_t k_sr = (uint32_t)c.k_sr, v_sr = (uint32_t)c.v_sr;
    const uint8_t* kb = c.k + head * c.k_sh + g * c.k_sr + 16 * t;
    const uint8_t* vb = c.v + head * c.v_sh + 2 * t * c.v_sr + (D / 8) * g;
    // a usable block, or -1: such a page reads block 0, and none of its rows count
    auto block_in = [&](int e, int base) {
        if (base + lane >= count) return -1;
        if (e >= 0 && e < c.num_blocks) return e;
        if (c.status) atomicOr(c.status, FDMS_DEV_BAD_INDEX);
        return -1;
    };
    auto scale_of = [&](const float* s, int block) { return block >= 0 ? __ldg(s + (int64_t)block * c.heads + head) : 1.0f; };
    float lvs, ivs;
    auto take_vs = [&](float x) {
        x = paged_v_scale(x);
        lvs = paged_lg2(x);
        ivs = __frcp_rn(x);
    };
    int block = block_in(entry, 0), next = entry_ahead(c, seq, first, step, 32);
    float ks = scale_of(c.k_scale, block), vs = scale_of(c.v_scale, block), next_ks = 1.0f, next_vs = 1.0f;
    // Pages in registers: two at D = 64, where one is only 2 KB (8 x 8192 rows from memory 22.3 -> 19.4 us, 64 ragged up to 16384
    // 150 -> 128).  Asking the L2 cache for pages further on was slower everywhere, three pages spill.
    constexpr int kDepth = D == 64 ? 2 : 1;
    PageRegs<D> pg[kDepth];
    auto block_of = [&](int i, int j) {         // of page i + j, i in the 32 pages of `block`
        const int k = (i & 31) + j;
        return k < 32 ? __shfl_sync(0xffffffffu, block, k) : __shfl_sync(0xffffffffu, next, k - 32);
    };
    auto page_at = [&](const uint8_t* base, uint32_t sb, uint32_t sr, int blk, int i) {
        return base + (uint64_t)(uint32_t)max(blk, 0) * sb + (uint32_t)((first + step * i) & in_block) * kCachePage * sr;
    };
    const uint32_t k_sb = (uint32_t)c.k_sb, v_sb = (uint32_t)c.v_sb;
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
        if (d < count) {
            const int blk = __shfl_sync(0xffffffffu, block, d);
            load_k<D>(pg[d], page_at(kb, k_sb, k_sr, blk, d), k_sr);
            load_v<D>(pg[d], page_at(vb, v_sb, v_sr, blk, d), v_sr);
        }
    take_vs(vs);
    for (int i0 = 0; i0 < count; i0 += kDepth) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            const int i = i0 + d, j = i & 31;
            if (i >= count) break;
            if (j == 8) next = block_in(next, i + 24);
            if (j == 16) { next_ks = scale_of(c.k_scale, next); next_vs = scale_of(c.v_scale, next); }
            const int rows = __shfl_sync(0xffffffffu, block, j) < 0 ? 0 : min(kCachePage, len - (first + step * i) * kCachePage);
            const bool more = i + kDepth < count;
            const int then = block_of(i, kDepth);
            float s[4];
            page_scores<D>(pg[d], qb, s);
            if (more) load_k<D>(pg[d], page_at(kb, k_sb, k_sr, then, i + kDepth), k_sr);
            uint32_t b[4];
            page_weights<D, FINE>(u, s, __shfl_sync(0xffffffffu, ks, j), __shfl_sync(0xffffffffu, lvs, j), __shfl_sync(0xffffffffu, ivs, j), factor, rows, lane, b);
            if (rows < kCachePage) mask_v<D>(pg[d], rows, t);
            page_values<D, FINE>(u, pg[d], b);
            if (more) load_v<D>(pg[d], page_at(vb, v_sb, v_sr, then, i + kDepth), v_sr);
            if (j == 31) {
                block = next;
                ks = next_ks;
                take_vs(next_vs);
                next = entry_ahead(c, seq, first, step, i + 33);
            }
        }
    }
}

// What a unit costs its CTA before its first page and after its last, in pages: loads that wait for one another and the merge of
// the warps.  The shares count it, so that short sequences among long ones do not pile up in one CTA: from
// memory, 24 / 8 / 0 pages, 64 sequences ragged up to 16384 188 / 207 / 213 us, 3 up to 30000 30.5 / 44 / 54; 48 pages was slower again
// for many short sequences (300 up to 2000 rows 151 against 142).
constexpr int kUnitPages = 24;

// The weight (a unit's pages and kUnitPages, 0 without rows or without a token) of the sequences before b for all b, and in total, in shared memory; by
// all threads of the CTA.
__device__ __forceinline__ void weight_prefix(const DecodeArgs& a, int32_t* s_first, int32_t* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int32_t before = 0;
    for (int base = 0; base < a.batch; base += kDecThreads) {
        const int b = base + threadIdx.x;
        const int pages = b < a.batch && token_of(a, b) >= 0 ? (int)(((int64_t)paged_len(a.c, b) + kCachePage - 1) / kCachePage) : 0;
        const int weight = pages ? pages + kUnitPages : 0;
        int sum = weight;
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
        if (b < a.batch) s_first[b] = add + sum - weight;
        before += total;
        __syncthreads();
    }
    if (threadIdx.x == 0) s_first[a.batch] = before;
    __syncthreads();
}

// The share of CTA `c` of `n` in a weight of `total` begins at share(c); place x belongs to CTA owner(x).
__device__ __forceinline__ int64_t share(int64_t c, int64_t n, int64_t total) { return c * total / n; }
__device__ __forceinline__ int owner(int64_t x, int64_t n, int64_t total) { return (int)(((x + 1) * n - 1) / total); }

// The merge of a CTA's warps: every warp puts its state down, then warp h takes head h, D / 32 channels a lane.
template <int D>
struct MergeSmem {
    float o[kDecWarps][kDecHeads][D];
    float m[kDecWarps][kDecHeads], l[kDecWarps][kDecHeads];
};
static_assert(kDecWarps == kDecHeads, "the merge gives a head to a warp");

template <int D>
__device__ __forceinline__ void put_state(MergeSmem<D>& s, const UnitState<D>& st, int nh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float l = st.l[i];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (g == 0) { s.m[warp][2 * t + i] = st.m[i]; s.l[warp][2 * t + i] = l; }
        if (2 * t + i < nh)
#pragma unroll
            for (int j = 0; j < D / 16; j += 2)
                *(float4*)&s.o[warp][2 * t + i][(D / 8) * g + 2 * j] = make_float4(st.o[j][i], st.o[j][2 + i], st.o[j + 1][i], st.o[j + 1][2 + i]);
    }
}
template <int D>
__device__ __forceinline__ void merge_warps(const MergeSmem<D>& s, float (&acc)[D / 32], float& m, float& l) {
    const int hd = threadIdx.x >> 5, ch = (threadIdx.x & 31) * (D / 32);
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) m = fmaxf(m, s.m[w][hd]);
    const float ref = m == -INFINITY ? 0.0f : m;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
        const float r = paged_ex2(s.m[w][hd] - ref);
        l = fmaf(s.l[w][hd], r, l);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(s.o[w][hd][ch + i], r, acc[i]);
    }
}
template <int D, bool BF16>
__device__ __forceinline__ void write_row(const DecodeArgs& a, int tok, int hq, const float (&acc)[D / 32], float m, float l) {
    const int lane = threadIdx.x & 31;
    const float inv = l > 0.0f || l != l ? __frcp_rn(l) : 0.0f;
    uint16_t* out = a.out + tok * a.o_sb + (int64_t)hq * a.o_sh + lane * (D / 32);
#pragma unroll
    for (int i = 0; i < D / 32; i += 2) *(uint32_t*)(out + i) = pack_pair<BF16>(acc[i] * inv, acc[i + 1] * inv);
    if (a.lse && lane == 0) a.lse[tok * a.lse_sb + (int64_t)hq * a.lse_sh] = kPagedLn2 * (m + paged_lg2(l));
}

// Clusters: unit blockIdx.x / cluster, page p of it with warp p % 8 of the cluster's CTA p / 8 % cluster.
template <int D, bool BF16>
__global__ void __launch_bounds__(kDecThreads, kDecCtasPerSm) paged_decode_cluster_kernel(DecodeArgs a) {
    __shared__ MergeSmem<D> s;
    __shared__ float s_part[kDecHeads][D + 4];  // this CTA's part of the unit: O, M, l
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
    const int unit = blockIdx.x / a.cluster, rank = blockIdx.x - unit * a.cluster;
    const int per_seq = a.c.heads * a.splits, seq = unit / per_seq, u = unit - seq * per_seq;
    const int head = u / a.splits, h0 = (u % a.splits) * kDecHeads, nh = min(kDecHeads, a.group - h0);
    const int first = rank * kDecWarps + warp, step = a.cluster * kDecWarps;
    // length, table entries and queries are requested together
    const int entry = entry_ahead(a.c, seq, first, step, 0);
    const int tok = token_of(a, seq);
    if (tok < 0) return;                        // the whole cluster
    const int len = paged_len(a.c, seq), pages = (int)(((int64_t)len + kCachePage - 1) / kCachePage);
    uint32_t qb[D / 16][2];
    float factor[2];
    load_q<D, BF16>(a.q + tok * a.q_sb + (int64_t)(head * a.group + h0 + min(g, nh - 1)) * a.q_sh, a.scale, qb, factor, lane);
    UnitState<D> st;
    clear<D>(st);
    walk_pages<D, !BF16>(a.c, st, qb, factor, seq, head, first, step, first < pages ? (pages - first + step - 1) / step : 0, len, entry);
    put_state<D>(s, st, nh);
    __syncthreads();
    float acc[D / 32], m, l;
    if (warp < nh) {
        merge_warps<D>(s, acc, m, l);
        if (a.cluster == 1) write_row<D, BF16>(a, tok, head * a.group + h0 + warp, acc, m, l);
        else {
#pragma unroll
            for (int i = 0; i < D / 32; i += 2) *(float2*)&s_part[warp][lane * (D / 32) + i] = make_float2(acc[i], acc[i + 1]);
            if (lane == 0) *(float2*)&s_part[warp][D] = make_float2(m, l);
        }
    }
    if (a.cluster == 1) return;
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp < nh && warp % a.cluster == rank) {                // heads are shared out among the cluster's CTAs
        const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&s_part[warp][0]);
        float pm[kMaxCluster], pl[kMaxCluster];
        m = -INFINITY;
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
            pm[r] = -INFINITY;
            pl[r] = 0.0f;
            if (r < a.cluster) {
                uint32_t at;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mine + D * 4), "r"(r));
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(pm[r]), "=f"(pl[r]) : "r"(at) : "memory");
            }
            m = fmaxf(m, pm[r]);
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
            if (r < a.cluster) {
                uint32_t at;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mine + lane * (D / 8)), "r"(r));
                const float w = paged_ex2(pm[r] - ref);
                l = fmaf(pl[r], w, l);
#pragma unroll
                for (int i = 0; i < D / 32; i += 2) {
                    float x, y;
                    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x), "=f"(y) : "r"(at + 4 * i) : "memory");
                    acc[i] = fmaf(x, w, acc[i]);
                    acc[i + 1] = fmaf(y, w, acc[i + 1]);
                }
            }
        write_row<D, BF16>(a, tok, head * a.group + h0 + warp, acc, m, l);
    }
    // a CTA's shared memory stays until every other has read it
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kDecThreads, kDecCtasPerSm) paged_decode_kernel(DecodeArgs a) {
    extern __shared__ int32_t s_first[];        // batch + 1
    __shared__ int32_t s_warp[kDecWarps];
    __shared__ MergeSmem<D> s;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
    pdl_trigger();
    weight_prefix(a, s_first, s_warp);
    const int per_seq = a.c.heads * a.splits;
    const int64_t total = (int64_t)s_first[a.batch] * per_seq;
    // fewer CTAs than the grid has where there are not two pages for each warp
    const int64_t ctas = min((int64_t)gridDim.x, max((int64_t)1, total / (2 * kDecWarps + kUnitPages)));
    if (blockIdx.x == 0) {                      // sequences without rows: zeros
        for (int b = warp; b < a.batch; b += kDecWarps) {
            if (s_first[b + 1] != s_first[b]) continue;
            const int hq = a.c.heads * a.group, tok = token_of(a, b);
            for (int i = lane; i < hq * (D / 8) && tok >= 0; i += 32)
                *(uint4*)(a.out + tok * a.o_sb + (i / (D / 8)) * a.o_sh + (i % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
            if (a.lse)
                for (int i = lane; i < hq && tok >= 0; i += 32) a.lse[tok * a.lse_sb + i * a.lse_sh] = -INFINITY;
            for (int i = lane; i < per_seq; i += 32) a.cuts[(int64_t)b * per_seq + i] = make_int2(0, -1);
        }
    }
    if (blockIdx.x >= ctas) return;
    const int64_t begin = share(blockIdx.x, ctas, total), end = share((int64_t)blockIdx.x + 1, ctas, total);
    int seq = 0;                                // last sequence that begins at or before `begin`, and has any weight
    {
        int lo = 0, hi = a.batch;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if ((int64_t)s_first[mid + 1] * per_seq > begin) hi = mid; else lo = mid + 1;
        }
        seq = lo;
    }
    int64_t at = begin;
    while (at < end) {
        while ((int64_t)s_first[seq + 1] * per_seq <= at) ++seq;
        const int weight = s_first[seq + 1] - s_first[seq], pages = weight - kUnitPages;
        const int64_t seq_begin = (int64_t)s_first[seq] * per_seq;
        const int u = (int)((at - seq_begin) / weight);         // unit of the sequence
        const int64_t unit_begin = seq_begin + (int64_t)u * weight, unit_end = unit_begin + weight;
        const int64_t from = at;
        at = min(unit_end, end);
        // page p lies at unit_begin + kUnitPages + p; a share that ends before the first page leaves the unit to the next CTA
        const int p0 = (int)max((int64_t)0, from - unit_begin - kUnitPages), p1 = (int)(at - unit_begin) - kUnitPages;
        if (p1 <= 0) break;
        const int head = u / a.splits, h0 = (u % a.splits) * kDecHeads, nh = min(kDecHeads, a.group - h0);
        const int tok = max(token_of(a, seq), 0);       // a sequence with weight has one
        const int len = min(paged_len(a.c, seq), pages * kCachePage);
        const int entry = entry_ahead(a.c, seq, p0 + warp, kDecWarps, 0);
        uint32_t qb[D / 16][2];
        float factor[2];
        load_q<D, BF16>(a.q + tok * a.q_sb + (int64_t)(head * a.group + h0 + min(g, nh - 1)) * a.q_sh, a.scale, qb, factor, lane);
        UnitState<D> st;
        clear<D>(st);
        walk_pages<D, !BF16>(a.c, st, qb, factor, seq, head, p0 + warp, kDecWarps, p1 - p0 > warp ? (p1 - p0 - warp + kDecWarps - 1) / kDecWarps : 0, len, entry);
        put_state<D>(s, st, nh);
        __syncthreads();
        const bool whole = p0 == 0 && p1 == pages;
        const int slot = blockIdx.x * 2 + (from == begin ? 0 : 1);
        if (warp < nh) {
            float acc[D / 32], m, l;
            merge_warps<D>(s, acc, m, l);
            if (whole) write_row<D, BF16>(a, tok, head * a.group + h0 + warp, acc, m, l);
            else {
                float* part = a.parts + ((int64_t)slot * kDecHeads + warp) * (D + 4);
#pragma unroll
                for (int i = 0; i < D / 32; i += 2) *(float2*)(part + lane * (D / 32) + i) = make_float2(acc[i], acc[i + 1]);
                if (lane == 0) *(float2*)(part + D) = make_float2(m, l);
            }
        }
        if (p0 == 0 && threadIdx.x == 0) {
            const int2 cut = whole ? make_int2(0, -1) : make_int2(slot, owner(unit_end - 1, ctas, total));
            a.cuts[(int64_t)seq * per_seq + u] = cut;
        }
        __syncthreads();
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
    float l = 0.0f, acc[D / 32];
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
    write_row<D, BF16>(a, max(token_of(a, (int)seq), 0), h, acc, m, l);
}

}  // namespace fdms

using namespace fdms;

static int64_t decode_parts_bytes(int sms, int head_dim) {
    return (int64_t)sms * kDecCtasPerSm * 2 * kDecHeads * (head_dim + 4) * (int64_t)sizeof(float);
}

using ClusterKernel = void (*)(DecodeArgs);
static ClusterKernel cluster_kernel(int head_dim, bool bf16) {
    return head_dim == 64 ? (bf16 ? paged_decode_cluster_kernel<64, true> : paged_decode_cluster_kernel<64, false>)
                          : (bf16 ? paged_decode_cluster_kernel<128, true> : paged_decode_cluster_kernel<128, false>);
}
static void cluster_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute& attr, int64_t ctas, int cluster, cudaStream_t stream) {
    cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kDecThreads);
    cfg.stream = stream;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
}
// How many clusters of 2^i CTAs the current device holds at once, the least over the kernel's forms; 0 where it takes none.  The
// SMs of a partition that do not make up a cluster stay empty, so that wide clusters hold fewer CTAs than the SMs would.
struct ClusterRoom {
    int held[kClusterSizes];
};
static ClusterRoom read_cluster_room() {
    ClusterRoom room;
    for (int i = 0; i < kClusterSizes; ++i) {
        room.held[i] = INT_MAX;
        for (int form = 0; form < 4; ++form) {
            ClusterKernel kern = cluster_kernel(form & 1 ? 64 : 128, (form & 2) != 0);
            cudaLaunchConfig_t cfg;
            cudaLaunchAttribute attr;
            cluster_config(cfg, attr, 1 << i, 1 << i, nullptr);
            int n = 0;
            if ((i > 3 && cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) ||
                cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
                cudaGetLastError();
                n = 0;
            }
            room.held[i] = std::min(room.held[i], n);
        }
    }
    return room;
}
static const ClusterRoom& cluster_room() {
    static ClusterRoom rooms[kMaxDevices];
    static std::once_flag once[kMaxDevices];
    static const ClusterRoom none = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return none;
    std::call_once(once[dev], [dev] { rooms[dev] = read_cluster_room(); });
    return rooms[dev];
}

// CTAs per unit of the cluster kernel for sequences of up to `rows` rows, 0: the shares.  As many as one wave of the GPU
// holds, each with a page for every warp.  The clusters save the join and the walk over all lengths, but a long sequence among
// short ones keeps its CTAs while others are idle, the more so the fewer waves follow; so the pages that a warp may get are
// limited, by the waves.  Measured (head_dim 128, 8 KV heads, from memory, clusters / shares, us): one sequence of 2000 rows 7.7 / 12.4,
// 8000 11.2 / 14.2, 24000 23.8 / 25.9, 48000 39.0 / 34.8; 5 ragged up to 8000 24.5 / 19.2, 16 up to 3000 21.4 / 20.1 (all of 3000
// 24.4 / 29.0), 64 up to 1000 24.5 / 27.0, 64 up to 3000 53.7 / 49.2, 100 up to 4000 89 / 88, 600 up to 1000 156 / 172.  At head_dim 64 a
// page is half the work: 8 of 8192 20.0 / 23.4, 8 ragged up to 8192 18.2 / 18.4 and up to 10000 21.1 / 19.6, 2 of 24000 25.7 / 21.9.
constexpr int kClusterWaves = 4;
static int decode_cluster(int64_t units, int64_t rows, int64_t head_dim, int sms) {
    const int64_t most = head_dim == 64 ? 20 : 12;      // pages of a warp in a wave
    const int64_t pages = (rows + kCachePage - 1) / kCachePage, wave = (int64_t)sms * kDecCtasPerSm;
    const ClusterRoom& room = cluster_room();
    int n = 1;
    for (int i = 1; i < kClusterSizes && units <= room.held[i] && pages > (int64_t)n * kDecWarps; ++i) n *= 2;
    const int64_t work = std::min(std::max(units * n, wave), wave * kClusterWaves);
    return pages * wave <= work * n * kDecWarps * most && units * n < (1ll << 31) ? n : 0;
}

extern "C" int64_t fdms_paged_attn_decode_workspace_bytes(int64_t batch, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t max_rows) {
    if (batch < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || head_dim <= 0 || max_rows < 0) return -1;
    const int sms = paged_sms();
    if (sms <= 0) return -1;
    const int64_t units = batch * num_kv_heads * ((num_q_heads / num_kv_heads + kDecHeads - 1) / kDecHeads);
    return decode_cluster(units, max_rows, head_dim, sms) ? 0 : decode_parts_bytes(sms, (int)head_dim) + units * (int64_t)sizeof(int2);
}

extern "C" int32_t fdms_paged_attn_decode(const fdms_paged_attn_args* args, void* stream) {
    clear_error();
    DecodeArgs a;
    const bool idle = args && (args->num_seqs == 0 || (args->cu_seqlens_q && args->tokens == 0));
    const int32_t rc = paged_attn_check("fdms_paged_attn_decode", args, a.c, idle);
    if (rc != FDMS_OK) return rc;
    const fdms_paged_attn_args& p = *args;
    const int num_q_heads = (int)p.num_q_heads, num_kv_heads = a.c.heads, head_dim = (int)p.cache.head_dim;
    FDMS_REQUIRE(p.tokens == p.num_seqs || (p.cu_seqlens_q && p.tokens < p.num_seqs), FDMS_E_ARG,
                 "fdms_paged_attn_decode: one token per sequence, got %lld for %lld", (long long)p.tokens, (long long)p.num_seqs);
    FDMS_REQUIRE(p.num_seqs <= kDecMaxBatch, FDMS_E_CAPACITY, "fdms_paged_attn_decode: at most %d sequences a call, got %lld", kDecMaxBatch,
                 (long long)p.num_seqs);
    if (idle) return FDMS_OK;
    const int batch = (int)p.num_seqs;
    const int sms = paged_sms();
    FDMS_REQUIRE(sms > 0, FDMS_E_CUDA, "fdms_paged_attn_decode: cannot read the device's SM count");
    a.q = (const uint16_t*)p.q;
    a.out = (uint16_t*)p.out;
    a.lse = p.lse_out;
    a.cu = p.cu_seqlens_q;
    a.tokens = (int)p.tokens;
    a.q_sb = p.q_stride[0]; a.q_sh = p.q_stride[1]; a.o_sb = p.out_stride[0]; a.o_sh = p.out_stride[1];
    a.lse_sb = p.lse_stride[0]; a.lse_sh = p.lse_stride[1];
    a.batch = batch;
    a.group = num_q_heads / num_kv_heads;
    a.splits = (a.group + kDecHeads - 1) / kDecHeads;
    a.scale = (float)p.scale;
    cudaStream_t st = (cudaStream_t)stream;
    const bool bf = p.dtype == FDMS_BF16;
    const int64_t units = (int64_t)batch * num_kv_heads * a.splits;
    a.cluster = decode_cluster(units, p.max_blocks * p.cache.block_size, head_dim, sms);
    a.parts = nullptr;
    a.cuts = nullptr;
    if (a.cluster) {
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute attr;
        cluster_config(cfg, attr, units * a.cluster, a.cluster, st);
        FDMS_CUDA_OK(cudaLaunchKernelEx(&cfg, cluster_kernel(head_dim, bf), a));
        FDMS_CHECK_LAUNCH("paged_decode_cluster_kernel");
        return FDMS_OK;
    }
    const int64_t need = decode_parts_bytes(sms, head_dim) + units * (int64_t)sizeof(int2);
    FDMS_REQUIRE(p.workspace && ((uintptr_t)p.workspace & 15) == 0 && p.workspace_bytes >= need, FDMS_E_WORKSPACE,
                 "fdms_paged_attn_decode: workspace missing, unaligned or smaller than %lld bytes", (long long)need);
    a.parts = (float*)p.workspace;
    a.cuts = (int2*)((char*)p.workspace + decode_parts_bytes(sms, head_dim));
    const int64_t pages_held = (int64_t)batch * p.max_blocks * (p.cache.block_size / kCachePage);
    FDMS_REQUIRE(pages_held + (int64_t)batch * kUnitPages <= 0x7fffffff, FDMS_E_CAPACITY, "fdms_paged_attn_decode: the block tables hold too many rows");
    const int64_t useful = (pages_held * num_kv_heads * a.splits + 2 * kDecWarps - 1) / (2 * kDecWarps);
    const unsigned grid = (unsigned)(useful < 1 ? 1 : useful < (int64_t)sms * kDecCtasPerSm ? useful : (int64_t)sms * kDecCtasPerSm);
    const size_t smem = (size_t)(batch + 1) * sizeof(int32_t);
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
