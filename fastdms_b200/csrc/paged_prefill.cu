// Prefill attention over the block-scaled paged cache: the tokens of a step, packed sequence by sequence, against their
// sequence's cached rows.  Token i of a sequence with n tokens in the step and kv rows in the cache sees rows
// 0 .. kv - n + i; a token that sees no row gets zeros and a log-sum-exp of -inf.
#include "paged_attn.cuh"

namespace fdms {

constexpr int kPreWarps = 4;
constexpr int kPreRows = kPreWarps * 16;        // (token, q head) rows of a CTA, heads of a token together

// One 16-row page as matrix operands.  Lane (g, t) = (lane / 4, lane % 4).
//   Scores: B holds K^T.  Column c of the two 8-column tiles is key 4 (c / 2) + c % 2 and the same + 2, so that a lane's
//   four scores are keys 4t .. 4t + 3, which is what the second product wants from it.  The k index is permuted: in chunk
//   n (64 bytes of a row) lane t brings bytes 64 n + 16 t + [0, 16), four of them for each of four steps; a query fragment
//   is loaded in the same order.
//   Output: A holds P, its k index the keys in the order above; B holds V, column g of tile j being channel (D / 8) g + j,
//   so that a lane loads D / 8 consecutive bytes of keys 4t .. 4t + 3 and ends up with consecutive channels.
template <int D>
struct PageRegs {
    uint4 k[2][D / 64];         // keys a, a + 2; chunks
    uint4 v[D == 128 ? 4 : 2];  // keys 4t .. 4t + 3, D / 8 bytes each (D = 64: two keys per vector)
};

template <int D>
__device__ __forceinline__ void load_k(PageRegs<D>& p, const uint8_t* k, int64_t sr, int lane) {
    const int g = lane >> 2, t = lane & 3, key = 4 * (g >> 1) + (g & 1);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < D / 64; ++n) p.k[i][n] = __ldg((const uint4*)(k + (key + 2 * i) * sr + 64 * n + 16 * t));
}
template <int D>
__device__ __forceinline__ void load_v(PageRegs<D>& p, const uint8_t* v, int64_t sr, int lane) {
    const int g = lane >> 2, t = lane & 3;
    if (D == 128) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p.v[i] = __ldg((const uint4*)(v + (4 * t + i) * sr + 16 * g));
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint2 a = __ldg((const uint2*)(v + (4 * t + 2 * i) * sr + 8 * g));
            const uint2 b = __ldg((const uint2*)(v + (4 * t + 2 * i + 1) * sr + 8 * g));
            p.v[i] = make_uint4(a.x, a.y, b.x, b.y);
        }
    }
}
template <int D>
__device__ __forceinline__ void zero_page(PageRegs<D>& p) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < D / 64; ++n) p.k[i][n] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < (D == 128 ? 4 : 2); ++i) p.v[i] = make_uint4(0, 0, 0, 0);
}
// Word w (channels 4w .. 4w + 3 of the lane's) of key 4t + i.
template <int D>
__device__ __forceinline__ uint32_t v_word(const PageRegs<D>& p, int i, int w) {
    const uint4& x = D == 128 ? p.v[i] : p.v[i >> 1];
    const int n = D == 128 ? w : (i & 1) * 2 + w;
    return n == 0 ? x.x : n == 1 ? x.y : n == 2 ? x.z : x.w;
}
// Rows at and beyond `rows` hold whatever the memory held: zero, so that P = 0 leaves no trace of them.
template <int D>
__device__ __forceinline__ void mask_v(PageRegs<D>& p, int rows, int lane) {
    const int t = lane & 3;
    if (D == 128) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * t + i >= rows) p.v[i] = make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (4 * t + 2 * i >= rows) p.v[i].x = p.v[i].y = 0;
            if (4 * t + 2 * i + 1 >= rows) p.v[i].z = p.v[i].w = 0;
        }
    }
}

struct PrefillArgs {
    PagedCache c;
    const uint16_t* q;
    uint16_t* out;
    float* lse;                                 // optional [q_heads, tokens]
    const int32_t* cu;                          // [seqs + 1]
    int64_t q_st, q_sh, o_st, o_sh, lse_sh, lse_st;
    int64_t tokens;
    int32_t seqs, group;
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

template <int D, bool BF16>
__global__ void __launch_bounds__(kPreWarps * 32) paged_prefill_kernel(PrefillArgs a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int per = kPreRows / a.group;         // tokens per tile
    int seq;
    int64_t first, begin, count;
    // the last tiles of a sequence see the most rows: they start first
    if (!find_tile(a, (int64_t)gridDim.x - 1 - blockIdx.x, per, seq, first, begin, count)) return;
    const int head = blockIdx.y;
    const int kv = paged_len(a.c, seq);
    // this lane's rows
    int64_t tok[2], last[2];                    // token of the step, last cached row it sees
    int hq[2];
    bool live[2];
    float up[2], factor[2];
    uint32_t qa[D / 16][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = warp * 16 + g + 8 * i;
        const int64_t j = first + r / a.group;
        live[i] = r < per * a.group && j < count;
        tok[i] = begin + (live[i] ? j : first);
        hq[i] = head * a.group + (live[i] ? r % a.group : 0);
        last[i] = live[i] ? (int64_t)kv - count + j : -1;
        const uint16_t* q = a.q + tok[i] * a.q_st + (int64_t)hq[i] * a.q_sh;
        uint4 w[D / 64][2];
        float top = 0.0f;
#pragma unroll
        for (int n = 0; n < D / 64; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                w[n][k] = *(const uint4*)(q + 64 * n + 16 * t + 8 * k);
                const uint32_t x[4] = {w[n][k].x, w[n][k].y, w[n][k].z, w[n][k].w};
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    float e, f;
                    unpack_pair<BF16>(x[v], e, f);
                    top = fmaxf(top, fmaxf(fabsf(e), fabsf(f)));
                }
            }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        row_power(top, up[i], factor[i]);
        factor[i] *= a.scale * kPagedLog2e;
#pragma unroll
        for (int n = 0; n < D / 64; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t x[4] = {w[n][k].x, w[n][k].y, w[n][k].z, w[n][k].w};
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    float e, f;
                    unpack_pair<BF16>(x[v], e, f);
                    qa[4 * n + 2 * k + (v >> 1)][2 * (v & 1) + i] = f16x2_of(e * up[i], f * up[i]);
                }
            }
    }
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    int64_t most = max(last[0], last[1]);
    int64_t least = min(live[0] ? last[0] : (int64_t)kv, live[1] ? last[1] : (int64_t)kv);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        most = max(most, __shfl_xor_sync(0xffffffffu, most, s));
        least = min(least, __shfl_xor_sync(0xffffffffu, least, s));
    }
    const int pages = (int)((most + kCachePage) / kCachePage);
    const int ppb = a.c.shift - 4;
    for (int p = 0; p < pages; ++p) {
        const int blk = a.c.tables[seq * a.c.table_stride + (p >> ppb)];
        if (blk < 0 || blk >= a.c.num_blocks) {
            if (lane == 0 && a.c.status) atomicOr(a.c.status, FDMS_DEV_BAD_INDEX);
            continue;
        }
        const int row = (p & ((1 << ppb) - 1)) * kCachePage;
        PageRegs<D> pg;
        const uint8_t* vp = a.c.v + (int64_t)blk * a.c.v_sb + head * a.c.v_sh + row * a.c.v_sr;
        load_k<D>(pg, a.c.k + (int64_t)blk * a.c.k_sb + head * a.c.k_sh + row * a.c.k_sr, a.c.k_sr, lane);
        load_v<D>(pg, vp, a.c.v_sr, lane);
        const float ks = a.c.k_scale[(int64_t)blk * a.c.heads + head], vs = a.c.v_scale[(int64_t)blk * a.c.heads + head];
        const float lvs = paged_lg2(vs), ivs = __frcp_rn(vs);
        float s0[4] = {0, 0, 0, 0}, s1[4] = {0, 0, 0, 0};       // keys 4t, 4t + 1 and 4t + 2, 4t + 3 of rows g and g + 8
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t(&q4)[4] = qa[4 * c + j];
                uint32_t b0, b1;
                e4m3x4_f16(j == 0 ? pg.k[0][c].x : j == 1 ? pg.k[0][c].y : j == 2 ? pg.k[0][c].z : pg.k[0][c].w, b0, b1);
                mma_16816(s0, q4[0], q4[1], q4[2], q4[3], b0, b1);
                e4m3x4_f16(j == 0 ? pg.k[1][c].x : j == 1 ? pg.k[1][c].y : j == 2 ? pg.k[1][c].z : pg.k[1][c].w, b0, b1);
                mma_16816(s1, q4[0], q4[1], q4[2], q4[3], b0, b1);
            }
        uint32_t pa[4];
        const int key = p * kCachePage + 4 * t;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float s[4] = {s0[2 * i], s0[2 * i + 1], s1[2 * i], s1[2 * i + 1]}, top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[j] = key + j <= last[i] ? fmaf(s[j], ks * factor[i], lvs) : -INFINITY;
                top = fmaxf(top, s[j]);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (__any_sync(0xffffffffu, top > m[i] + 8.0f)) {
                const float next = fmaxf(m[i], top);
                const float r = next == -INFINITY ? 1.0f : paged_ex2(m[i] - next);
                m[i] = next;
                l[i] *= r;
#pragma unroll
                for (int j = 0; j < D / 8; ++j) { o[j][2 * i] *= r; o[j][2 * i + 1] *= r; }
            }
            const float ref = m[i] == -INFINITY ? 0.0f : m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] = paged_ex2(s[j] - ref);
            l[i] = fmaf((s[0] + s[1]) + (s[2] + s[3]), ivs, l[i]);
            pa[i] = f16x2_of(s[0], s[1]);
            pa[2 + i] = f16x2_of(s[2], s[3]);
        }
        if ((p + 1) * kCachePage > least + 1) {
            // Some row does not see all of the page.  What it does not see may be anything, a NaN code among it: such
            // codes count as zero in the product and are put into the rows that do see them.
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int w = 0; w < D / 32; ++w) {
                    const uint32_t x = v_word<D>(pg, i, w) & 0x7f7f7f7fu;
                    odd = odd || ((x + 0x01010101u) & 0x80808080u) != 0;
                }
            if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
                for (int i = 0; i < (D == 128 ? 4 : 2); ++i) {
                    uint32_t* x = (uint32_t*)&pg.v[i];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t nan = ((x[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;      // top bit of each NaN byte
                        x[w] &= ~((nan >> 7) * 0xffu);
                    }
                }
                for (int k = 0; k < kCachePage; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (p * kCachePage + k <= last[i])
#pragma unroll
                            for (int j = 0; j < D / 8; ++j)
#pragma unroll
                                for (int n = 0; n < 2; ++n)
                                    if ((vp[k * a.c.v_sr + (D / 8) * (2 * t + n) + j] & 0x7f) == 0x7f) o[j][2 * i + n] = NAN;
            }
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
            const uint32_t k0 = v_word<D>(pg, 0, w), k1 = v_word<D>(pg, 1, w), k2 = v_word<D>(pg, 2, w), k3 = v_word<D>(pg, 3, w);
            uint32_t b0[4], b1[4];
            e4m3x4_f16(__byte_perm(k0, k1, 0x5140), b0[0], b0[1]);
            e4m3x4_f16(__byte_perm(k0, k1, 0x7362), b0[2], b0[3]);
            e4m3x4_f16(__byte_perm(k2, k3, 0x5140), b1[0], b1[1]);
            e4m3x4_f16(__byte_perm(k2, k3, 0x7362), b1[2], b1[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) mma_16816(o[4 * w + j], pa[0], pa[1], pa[2], pa[3], b0[j], b1[j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (!live[i]) continue;
        const float inv = l[i] > 0.0f || l[i] != l[i] ? __frcp_rn(l[i]) : 0.0f;
        uint16_t* out = a.out + tok[i] * a.o_st + (int64_t)hq[i] * a.o_sh;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < D / 8; j += 2)
                *(uint32_t*)(out + (D / 8) * (2 * t + n) + j) = pack_pair<BF16>(o[j][2 * i + n] * inv, o[j + 1][2 * i + n] * inv);
        if (a.lse && t == 0) a.lse[(int64_t)hq[i] * a.lse_sh + tok[i] * a.lse_st] = kPagedLn2 * (m[i] + paged_lg2(l[i]));
    }
}

}  // namespace fdms

using namespace fdms;

extern "C" int32_t fdms_paged_attn_prefill(const fdms_paged_attn_args* args, void* stream) {
    clear_error();
    PagedCache c;
    const bool idle = args && (args->num_seqs == 0 || args->tokens == 0);
    const int32_t rc = paged_attn_check("fdms_paged_attn_prefill", args, c, idle);
    if (rc != FDMS_OK) return rc;
    if (idle) return FDMS_OK;
    const fdms_paged_attn_args& p = *args;
    FDMS_REQUIRE(p.cu_seqlens_q, FDMS_E_ARG, "fdms_paged_attn_prefill: null pointer");
    const int group = (int)p.num_q_heads / c.heads;
    PrefillArgs a = {c, (const uint16_t*)p.q, (uint16_t*)p.out, p.lse_out, p.cu_seqlens_q, p.q_stride[0], p.q_stride[1], p.out_stride[0],
                     p.out_stride[1], p.lse_stride[0], p.lse_stride[1], p.tokens, (int32_t)p.num_seqs, group, (float)p.scale};
    const int64_t tiles = p.tokens / (kPreRows / group) + p.num_seqs;
    FDMS_REQUIRE(tiles < (1ll << 31), FDMS_E_CAPACITY, "fdms_paged_attn_prefill: too many tokens");
    const dim3 grid((unsigned)tiles, (unsigned)c.heads);
    cudaStream_t st = (cudaStream_t)stream;
    const bool bf = p.dtype == FDMS_BF16;
    if (p.cache.head_dim == 64) {
        if (bf) paged_prefill_kernel<64, true><<<grid, kPreWarps * 32, 0, st>>>(a);
        else paged_prefill_kernel<64, false><<<grid, kPreWarps * 32, 0, st>>>(a);
    } else {
        if (bf) paged_prefill_kernel<128, true><<<grid, kPreWarps * 32, 0, st>>>(a);
        else paged_prefill_kernel<128, false><<<grid, kPreWarps * 32, 0, st>>>(a);
    }
    FDMS_CHECK_LAUNCH("paged_prefill_kernel");
    return FDMS_OK;
}
