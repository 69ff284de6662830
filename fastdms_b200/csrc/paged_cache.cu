// Block-scaled paged KV cache: block tables and slot maps of a step, release of blocks, and the quantising store.
//
// The cache holds K and V in e4m3, [blocks, kv_heads, block_size, head_dim] (block_size 16, 32, 64 or 128), with one
// float32 scale per (block, KV head): value = code * scale.  Scales are powers of two, 2^k with k in [-60, 40], so
// that dividing by one is exact and a code is ONE rounding of the value; a block whose later rows are louder than its
// earlier ones moves the earlier codes to the larger scale, which is an exponent shift (exact down to e4m3's
// subnormals).
//
// Measured: tables of a decode step of 256 requests 5.7 us, of 64 prompts of up to 32768 tokens (a million slots) 8.5 us; a store
// of 256 tokens into as many blocks 5 us (8 KV heads of 128), of 16 K prompt tokens 21 us: 101.6 MB read and written, 4.8 TB/s.
#include "paged_attn.cuh"

namespace fdms {

// ---------------------------------------------------------------------------------------------------------------
// Tables.  held = ceil(kv / bs), need = ceil((kv + new) / bs) - held; request i takes the blocks
// free[count - 1 - (sum of need before i) - j], j < need, if the stack reaches that far (requests are served in
// order).  A token whose position is a multiple of bs is the first of a newly opened block, and every opened block has
// exactly one such token: it writes the table entry, so that tokens are the only unit of work after the scan.
// ---------------------------------------------------------------------------------------------------------------
constexpr int kScanThreads = 1024;
constexpr int kFillThreads = 256;
constexpr int kFillTokens = 4;                 // consecutive tokens per thread: one 16-byte store of slots
constexpr int kFusedRequests = 1024;           // the one-launch form keeps its requests in shared memory

struct MetaArgs {
    const int32_t* new_lens;
    const int32_t* kv_lens;
    int32_t* kv_lens_out;
    int32_t* tables;
    int64_t table_stride;
    const int32_t* free_blocks;
    int64_t free_capacity;
    const int32_t* free_count;
    int32_t* free_count_out;
    int32_t* cu_seqlens;
    int32_t* slots;
    int64_t* positions;
    int32_t* status;
    int64_t total;
    int32_t n, max_blocks, shift;
};

// What a token needs to know of its request: rows stored before the step, and the stack index of its first block
// (-1: the request is not served).
struct Served {
    int32_t kv;
    int32_t top;
};

// Exclusive prefix sums of (blocks, tokens) over the CTA; returns the totals.
__device__ __forceinline__ void block_scan2(int64_t& a, int64_t& b, int64_t& ta, int64_t& tb, int64_t* s_a, int64_t* s_b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t ia = a, ib = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t xa = __shfl_up_sync(0xffffffffu, ia, o), xb = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) { ia += xa; ib += xb; }
    }
    __syncthreads();                            // the previous use of s_a / s_b is over
    if (lane == 31) { s_a[warp] = ia; s_b[warp] = ib; }
    __syncthreads();
    if (warp == 0) {
        int64_t wa = s_a[lane], wb = s_b[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t xa = __shfl_up_sync(0xffffffffu, wa, o), xb = __shfl_up_sync(0xffffffffu, wb, o);
            if (lane >= o) { wa += xa; wb += xb; }
        }
        s_a[lane] = wa;
        s_b[lane] = wb;
    }
    __syncthreads();
    const int64_t ea = warp ? s_a[warp - 1] : 0, eb = warp ? s_b[warp - 1] : 0;
    ta = s_a[31];
    tb = s_b[31];
    a = ea + ia - a;
    b = eb + ib - b;
}

// Slots, positions and table entries of tokens [t0, t0 + kFillTokens).  `cu` (n + 1 prefix sums) and `req` may be in
// shared or in global memory.
__device__ __forceinline__ void fill_tokens(const MetaArgs& a, const int32_t* cu, const Served* req, int64_t t0) {
    if (t0 >= a.total) return;
    int lo = 0, hi = a.n;                       // first request whose end is beyond t0
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid + 1] > t0) hi = mid; else lo = mid + 1;
    }
    int32_t slot[kFillTokens];
    int64_t pos[kFillTokens];
    int r = lo;
    const int mask = (1 << a.shift) - 1;
#pragma unroll
    for (int i = 0; i < kFillTokens; ++i) {
        const int64_t t = t0 + i;
        slot[i] = -1;
        pos[i] = 0;
        while (r < a.n && cu[r + 1] <= t) ++r;
        if (r >= a.n || t >= a.total) continue;
        const Served s = req[r];
        pos[i] = (int64_t)s.kv + (t - cu[r]);
        if (s.top < 0) continue;
        const int32_t p = (int32_t)pos[i];      // a served request fits into its row of the table
        const int held = (s.kv + mask) >> a.shift, col = p >> a.shift;
        int32_t block;
        if (col < held) {
            block = a.tables[(int64_t)r * a.table_stride + col];
        } else {
            block = a.free_blocks[s.top - (col - held)];
            if ((p & mask) == 0) a.tables[(int64_t)r * a.table_stride + col] = block;
        }
        slot[i] = block < 0 ? -1 : (block << a.shift) + (p & mask);
    }
    if (t0 + kFillTokens <= a.total) {          // slots and positions are 16-byte aligned (checked by the caller)
        *(int4*)(a.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        *(longlong2*)(a.positions + t0) = make_longlong2(pos[0], pos[1]);
        *(longlong2*)(a.positions + t0 + 2) = make_longlong2(pos[2], pos[3]);
    } else {
        for (int i = 0; i < kFillTokens && t0 + i < a.total; ++i) {
            a.slots[t0 + i] = slot[i];
            a.positions[t0 + i] = pos[i];
        }
    }
}

// One CTA: the scan over the requests, and with FUSED the tokens too.
template <bool FUSED>
__global__ void __launch_bounds__(kScanThreads) paged_scan_kernel(MetaArgs a, Served* req_out) {
    __shared__ int64_t s_a[32], s_b[32];
    __shared__ int32_t s_cu[FUSED ? kFusedRequests + 1 : 1];
    __shared__ Served s_req[FUSED ? kFusedRequests : 1];
    if (!FUSED) pdl_trigger();
    const int64_t room = (int64_t)a.max_blocks << a.shift;
    const int mask = (1 << a.shift) - 1;
    int32_t count = *a.free_count;
    bool bad = count < 0 || count > a.free_capacity;
    if (bad) count = 0;
    int64_t blocks_before = 0, tokens_before = 0, taken = 0;
    int32_t* cu = FUSED ? s_cu : a.cu_seqlens;
    Served* req = FUSED ? s_req : req_out;
    for (int base = 0; base < a.n; base += kScanThreads) {
        const int i = base + threadIdx.x;
        int64_t kv = 0, add = 0, need = 0;
        int32_t before = 0;
        bool fits = false;
        if (i < a.n) {
            kv = before = a.kv_lens[i];
            add = a.new_lens[i];
            fits = kv >= 0 && add >= 0 && kv + add <= room;
            if (add < 0) add = 0;
            if (kv < 0) kv = 0;
            if (fits) need = ((kv + add + mask) >> a.shift) - ((kv + mask) >> a.shift);
        }
        int64_t b0 = need, t0 = add, tb, tt;
        block_scan2(b0, t0, tb, tt, s_a, s_b);
        b0 += blocks_before;
        t0 += tokens_before;
        if (i < a.n) {
            const bool served = fits && t0 + add <= a.total && (need == 0 || b0 + need <= count);
            bad = bad || !fits || t0 + add > a.total;     // running out of blocks is an answer, not an error
            req[i] = {(int32_t)kv, served ? (need ? (int32_t)(count - 1 - b0) : 0) : -1};
            cu[i + 1] = (int32_t)min(t0 + add, a.total);
            if (FUSED) a.cu_seqlens[i + 1] = cu[i + 1];
            a.kv_lens_out[i] = served ? (int32_t)(kv + add) : before;
            if (served && need) taken = max(taken, b0 + need);
        }
        blocks_before += tb;
        tokens_before += tt;
    }
    if (threadIdx.x == 0) {
        cu[0] = 0;
        if (FUSED) a.cu_seqlens[0] = 0;
    }
    // the served requests that take blocks are the first ones that do, so the largest end is what the stack loses
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) taken = max(taken, __shfl_xor_sync(0xffffffffu, taken, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_a[threadIdx.x >> 5] = taken;
    __syncthreads();
    if (threadIdx.x < 32) {
        taken = s_a[threadIdx.x];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) taken = max(taken, __shfl_xor_sync(0xffffffffu, taken, o));
        if (threadIdx.x == 0) *a.free_count_out = count - (int32_t)taken;
    }
    if (bad && a.status) atomicOr(a.status, FDMS_DEV_BAD_INDEX);
    if (FUSED)
        for (int64_t t = (int64_t)threadIdx.x * kFillTokens; t < a.total; t += kScanThreads * kFillTokens)
            fill_tokens(a, s_cu, s_req, t);
}

__global__ void __launch_bounds__(kFillThreads) paged_fill_kernel(MetaArgs a, const Served* req) {
    pdl_wait();
    fill_tokens(a, a.cu_seqlens, req, ((int64_t)blockIdx.x * kFillThreads + threadIdx.x) * kFillTokens);
}

// ---------------------------------------------------------------------------------------------------------------
// Release: the blocks of the listed rows go back onto the stack in the order of the list, a row's last block lowest,
// so that admitting a request and releasing it again leaves the stack as it was.
// ---------------------------------------------------------------------------------------------------------------
constexpr int kReleaseThreads = 1024;
constexpr int kReleaseRows = 4096;

__global__ void __launch_bounds__(kReleaseThreads) paged_release_kernel(
    const int32_t* rows, int n, int32_t* kv_lens, int num_rows, int32_t* tables, int64_t table_stride, int max_blocks,
    int shift, int32_t* free_blocks, int64_t free_capacity, int64_t num_blocks, int32_t* free_count, int32_t* status) {
    __shared__ int32_t s_row[kReleaseRows];     // row of each entry, -1 where it is out of range or listed before
    __shared__ int32_t s_held[kReleaseRows];    // usable blocks of the entry, then their place on the stack
    __shared__ int32_t s_end;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kReleaseThreads / 32;
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += kReleaseThreads) {
        const int r = rows ? rows[i] : i;
        s_row[i] = r >= 0 && r < num_rows ? r : -1;
        bad = bad || s_row[i] < 0;
    }
    __syncthreads();
    for (int i = warp; i < n; i += warps) {     // a row listed twice is released once
        const int r = s_row[i];
        bool twice = false;
        if (r >= 0 && rows)
            for (int j = lane; j < i; j += 32) twice = twice || rows[j] == r;
        twice = __any_sync(0xffffffffu, twice);
        bad = bad || twice;
        int held = 0;
        if (r >= 0 && !twice) {
            const int64_t len = max(kv_lens[r], 0);
            const int cols = (int)min((len + (1 << shift) - 1) >> shift, (int64_t)max_blocks);
            for (int c = lane; c < cols; c += 32) {
                const int b = tables[(int64_t)r * table_stride + c];
                if (b >= 0 && b < num_blocks) ++held; else bad = true;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) held += __shfl_xor_sync(0xffffffffu, held, o);
        }
        if (lane == 0) s_held[i] = twice ? -1 : held;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int64_t at = min((int64_t)max(*free_count, 0), free_capacity);
        for (int i = 0; i < n; ++i) {
            const int held = s_held[i];
            if (held < 0) continue;
            s_held[i] = (int32_t)at;
            at += held;
        }
        if (at > free_capacity) { bad = true; at = free_capacity; }
        s_end = (int32_t)at;
    }
    __syncthreads();
    for (int i = warp; i < n; i += warps) {
        const int r = s_row[i];
        if (r < 0 || s_held[i] < 0) continue;
        int64_t at = s_held[i];
        const int64_t len = max(kv_lens[r], 0);
        const int cols = (int)min((len + (1 << shift) - 1) >> shift, (int64_t)max_blocks);
        for (int base = ((cols - 1) >> 5) << 5; base >= 0 && cols > 0; base -= 32) {        // last block first
            const int c = base + 31 - lane;
            int b = -1;
            if (c < cols) {
                b = tables[(int64_t)r * table_stride + c];
                tables[(int64_t)r * table_stride + c] = -1;
            }
            const bool use = b >= 0 && b < num_blocks;
            const unsigned m = __ballot_sync(0xffffffffu, use);
            const int64_t to = at + __popc(m & ((1u << lane) - 1));
            if (use && to < free_capacity) free_blocks[to] = b;
            at += __popc(m);
        }
        __syncwarp();
        if (lane == 0) kv_lens[r] = 0;
    }
    if (threadIdx.x == 0) *free_count = s_end;
    if (bad && status) atomicOr(status, FDMS_DEV_BAD_INDEX);
}

// ---------------------------------------------------------------------------------------------------------------
// Store.  A token begins a run when its slot opens a block or does not follow the token before it; a run ends with its
// block, so that a (run, head) of K or of V is one piece of work with a scale of its own: amax over the run's rows,
// 2^k the least with amax <= 448 * 2^k, the maximum with the block's scale where it holds earlier rows.
// A warp keeps 16 rows of the block in registers between the two passes (amax, rounding).  Steps of many tokens give
// every 16 rows of a block a warp of their own, so that each row is read once, and exchange the maxima through shared
// memory; in small steps, where one token per block is the rule, a warp takes the whole block.
// ---------------------------------------------------------------------------------------------------------------
constexpr int kStoreWarps = 8;
constexpr int64_t kStoreSmall = 512;            // tokens
constexpr int kScaleExpMin = -60, kScaleExpMax = 40;

struct StoreArgs {
    const uint16_t* src[2];                     // K, V
    int64_t src_st[2], src_sh[2];               // token and head stride in elements
    uint8_t* cache[2];
    int64_t sb[2], sh[2], sr[2];                // block, head and row stride in bytes
    float* scale[2];                            // [blocks, heads]
    const int32_t* slots;
    int32_t* status;
    int64_t tokens;
    int64_t num_slots;
    int32_t heads, shift, group, warps;         // tokens per CTA, warps per (run, head)
};

// Exponent k of the scale for a largest magnitude.
__device__ __forceinline__ int scale_exponent(float amax) {
    if (!(amax > 0.0f)) return kScaleExpMin;
    const uint32_t u = __float_as_uint(amax);
    // amax = 1.f * 2^e <= 448 * 2^k = 1.75 * 2^(k + 8); subnormal magnitudes read as e = -127 and land on the least k
    const int e = (int)(u >> 23) - 127;
    const int k = e - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(k, kScaleExpMin), kScaleExpMax);
}

__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

template <bool BF16>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
    if (BF16) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    } else {
        const __half2 h = *(const __half2*)&w;
        a = __low2float(h);
        b = __high2float(h);
    }
}

// The larger of each half of two words; of a number and a NaN the number.
template <bool BF16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    if (BF16) {
        const __nv_bfloat162 m = __hmax2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
        return *(const uint32_t*)&m;
    }
    const __half2 m = __hmax2(*(const __half2*)&a, *(const __half2*)&b);
    return *(const uint32_t*)&m;
}

// The nearest slot before the lane's token that is not negative, -1 if there is none; the lanes hold the slots of tokens first + lane,
// `prev` the slot before each.  By the whole warp.
__device__ __noinline__ int32_t slot_before(const int32_t* slots, int64_t first, int32_t my_slot, int32_t prev) {
    const int lane = threadIdx.x & 31;
    const unsigned below = __ballot_sync(0xffffffffu, my_slot >= 0) & ((1u << lane) - 1);
    const int32_t near = __shfl_sync(0xffffffffu, my_slot, below ? 31 - __clz(below) : 0);
    int32_t before = __shfl_sync(0xffffffffu, prev, 0);
    for (int64_t end = first - 1; before < 0 && end > 0; end -= 256) {
        int32_t x[8];                           // 256 slots, the nearest first
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t t = end - 32 * (i + 1) + lane;
            x[i] = t >= 0 ? __ldg(slots + t) : -1;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned m = __ballot_sync(0xffffffffu, x[i] >= 0);
            if (m && before < 0) before = __shfl_sync(0xffffffffu, x[i], 31 - __clz(m));
        }
    }
    return below ? near : before;
}

// D: head_dim.  A lane holds 8 elements of every (32 / (D / 8))-th row of the warp's 16.
template <int D, bool BF16>
__global__ void __launch_bounds__(kStoreWarps * 32, 4) paged_store_kernel(StoreArgs a) {
    constexpr int kLanes = D / 8;               // lanes per row
    constexpr int kRows = 32 / kLanes;          // rows per step
    constexpr int kSteps = 16 / kRows;
    __shared__ float s_max[kStoreWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int W = a.warps, per_cta = kStoreWarps / W;
    const int item = blockIdx.y * per_cta + warp / W, part = warp % W;
    const bool have = item < 2 * a.heads;
    const int which = have && item >= a.heads ? 1 : 0, head = have ? item - which * a.heads : 0;
    const int bs = 1 << a.shift;

    // the slots of 32 tokens, of which those of this CTA may begin a run
    const int64_t first = (int64_t)blockIdx.x * a.group;
    const int32_t my_slot = first + lane < a.tokens ? __ldg(a.slots + first + lane) : -1;
    int32_t prev = lane == 0 && first > 0 ? __ldg(a.slots + first - 1) : -1;
    {
        const int32_t up = __shfl_up_sync(0xffffffffu, my_slot, 1);
        if (lane > 0) prev = up;
    }
    bool begins = lane < a.group && my_slot >= 0 && ((my_slot & (bs - 1)) == 0 || prev != my_slot - 1);
    // A slot map lists a block's tokens in order and together: two runs in one block would move its scale and its codes side by
    // side.  So what a token begins a run after is the nearest one before it that is not skipped, however far back.
    if (__any_sync(0xffffffffu, begins && prev < 0)) prev = slot_before(a.slots, first, my_slot, prev);
    if (begins && (my_slot >= a.num_slots || (prev >= 0 && (prev >> a.shift) == (my_slot >> a.shift)))) {
        begins = false;
        if (a.status) atomicOr(a.status, FDMS_DEV_BAD_INDEX);
    }
    unsigned todo = __ballot_sync(0xffffffffu, begins);
    const int col = (lane % kLanes) * 8, row0 = lane / kLanes;
    while (todo) {
        const int src_lane = __ffs(todo) - 1;
        todo &= todo - 1;
        const int64_t t0 = first + src_lane;
        const int32_t slot = __shfl_sync(0xffffffffu, my_slot, src_lane);
        const int block = slot >> a.shift, off = slot & (bs - 1);
        float* scale = a.scale[which] + (int64_t)block * a.heads + head;
        const float old = have && off > 0 ? *scale : 0.0f;
        // rows of the run: slots that follow one another, inside the block
        int count;
        {
            const int d = lane - src_lane;
            const unsigned m = __ballot_sync(0xffffffffu, d > 0 && d < bs - off && my_slot == slot + d) >> src_lane >> 1;
            count = __ffs(~m);
            for (int base = count; base == count && base >= 32 - src_lane && base < bs - off; base += 32) {    // beyond the 32
                const int i = base + lane;
                const bool on = i < bs - off && t0 + i < a.tokens && a.slots[t0 + i] == slot + i;
                const unsigned more = __ballot_sync(0xffffffffu, on);
                count += more == 0xffffffffu ? 32 : __ffs(~more) - 1;
            }
        }
        // the 16-row parts of the block that this warp writes
        const int lo = W > 1 ? part : off >> 4, hi = W > 1 ? part : (off + count - 1) >> 4;
        const uint16_t* src = a.src[which] + t0 * a.src_st[which] + (int64_t)head * a.src_sh[which] + col;
        uint8_t* dst = a.cache[which] + (int64_t)block * a.sb[which] + (int64_t)head * a.sh[which] + col;
        uint4 x[kSteps];
        auto load = [&](int p) {
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                const int r = p * 16 + j * kRows + row0 - off;      // row of the run
                x[j] = make_uint4(0, 0, 0, 0);
                if (have && r >= 0 && r < count) x[j] = __ldg((const uint4*)(src + r * a.src_st[which]));
            }
        };
        uint32_t most = 0;                      // largest magnitudes of the even and the odd elements, as they are
        for (int p = lo; p <= hi; ++p) {
            load(p);
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) most = max2<BF16>(most, w[i] & 0x7fff7fffu);      // a NaN does not count
            }
        }
        float top, odd;
        unpack2<BF16>(most, top, odd);
        top = fmaxf(top, odd);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (W > 1) {
            if (lane == 0) s_max[warp] = top;
            __syncthreads();
            for (int i = 0; i < W; ++i) top = fmaxf(top, s_max[warp - part + i]);
            __syncthreads();
        }
        if (!have) continue;
        const float now = fmaxf(old, pow2(scale_exponent(top)));
        const float inv = __frcp_rn(now);       // exact for a power of two
        for (int p = lo; p <= hi; ++p) {
            if (lo < hi) load(p);
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                const int br = p * 16 + j * kRows + row0, r = br - off;
                if (r < 0 || r >= count) continue;
                const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
                float f[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) unpack2<BF16>(w[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] *= inv;
                *(uint2*)(dst + br * a.sr[which]) = make_uint2(pack_e4m3x4(f[0], f[1], f[2], f[3]), pack_e4m3x4(f[4], f[5], f[6], f[7]));
            }
        }
        if (old > 0.0f && old < now) {          // the earlier rows of the block move to the larger scale
            const float ratio = old * inv;
            const int end = min(off, W > 1 ? 16 * part + 16 : off);
            for (int br = (W > 1 ? 16 * part : 0) + row0; br < end; br += kRows) {
                uint2* p = (uint2*)(dst + br * a.sr[which]);
                const uint2 c = *p;
                float f[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    f[i] = e4m3_to_float((uint8_t)(c.x >> (8 * i))) * ratio;
                    f[4 + i] = e4m3_to_float((uint8_t)(c.y >> (8 * i))) * ratio;
                }
                *p = make_uint2(pack_e4m3x4(f[0], f[1], f[2], f[3]), pack_e4m3x4(f[4], f[5], f[6], f[7]));
            }
        }
        __syncwarp();                           // every lane has read the old scale
        if (lane == 0 && part == 0) *scale = now;
    }
}

}  // namespace fdms

using namespace fdms;

static int32_t block_shift(int64_t block_size) {
    return block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : block_size == 128 ? 7 : -1;
}

// One CTA does all of a decode step in one launch (256 requests: 5.7 us).  Beyond kFusedTokens its writes are what takes time,
// and a second launch spreads them over the GPU: 2 K tokens take 5.0 us with one and 5.7 with two, 8 K 8.1 and 5.7, 16 K 12
// and 5.7; the second launch and its workspace cost 6 us of host time.
constexpr int64_t kFusedTokens = 4 * kScanThreads * kFillTokens;
static bool metadata_fused(int64_t num_seqs, int64_t total_tokens) { return num_seqs <= kFusedRequests && total_tokens <= kFusedTokens; }

extern "C" int64_t fdms_paged_metadata_workspace_bytes(int64_t num_seqs, int64_t total_tokens) {
    if (num_seqs < 0 || total_tokens < 0) return -1;
    return metadata_fused(num_seqs, total_tokens) ? 0 : num_seqs * (int64_t)sizeof(Served);
}

extern "C" int32_t fdms_paged_metadata(const fdms_paged_metadata_args* args, void* stream) {
    clear_error();
    FDMS_REQUIRE(args, FDMS_E_ARG, "fdms_paged_metadata: null pointer");
    const fdms_paged_metadata_args& p = *args;
    FDMS_REQUIRE(p.free_count && p.free_count_out && p.cu_seqlens && (p.free_blocks || p.free_capacity == 0) &&
                     ((p.new_lens && p.kv_lens && p.kv_lens_out && (p.block_tables || p.max_blocks == 0)) || p.num_seqs == 0) &&
                     ((p.slot_mapping && p.positions) || p.total_tokens == 0),
                 FDMS_E_ARG, "fdms_paged_metadata: null pointer");
    const int32_t shift = block_shift(p.block_size);
    FDMS_REQUIRE(shift > 0, FDMS_E_ARG, "fdms_paged_metadata: block_size must be 16, 32, 64 or 128, got %lld", (long long)p.block_size);
    FDMS_REQUIRE(p.num_seqs >= 0 && p.max_blocks >= 0 && p.total_tokens >= 0 && p.free_capacity >= 0 && p.bt_stride >= p.max_blocks, FDMS_E_ARG,
                 "fdms_paged_metadata: negative size, or rows of the block table overlap");
    FDMS_REQUIRE((((uintptr_t)p.slot_mapping | (uintptr_t)p.positions) & 15) == 0, FDMS_E_ARG,
                 "fdms_paged_metadata: slot_mapping and positions must be 16-byte aligned");
    // The scan reads the lengths of kScanThreads requests and then writes theirs: what it writes must not lie ahead of what it reads.
    auto ahead = [&](const int32_t* in) { return (const int32_t*)p.kv_lens_out > in && p.kv_lens_out < in + p.num_seqs; };
    FDMS_REQUIRE(p.num_seqs <= kScanThreads || (!ahead(p.new_lens) && !ahead(p.kv_lens)), FDMS_E_ARG,
                 "fdms_paged_metadata: kv_lens_out begins inside new_lens or kv_lens, behind their first element");
    FDMS_REQUIRE(p.total_tokens < 0x7fffffff && p.num_seqs < 0x7fffffff && p.free_capacity <= (0x7fffffff >> shift) && p.max_blocks <= (0x7fffffff >> shift),
                 FDMS_E_CAPACITY, "fdms_paged_metadata: token and slot numbers must fit in 31 bits");
    const MetaArgs a = {p.new_lens, p.kv_lens, p.kv_lens_out, p.block_tables, p.bt_stride, p.free_blocks, p.free_capacity, p.free_count,
                        p.free_count_out, p.cu_seqlens, p.slot_mapping, p.positions, p.dev_status, p.total_tokens, (int32_t)p.num_seqs,
                        (int32_t)p.max_blocks, shift};
    cudaStream_t st = (cudaStream_t)stream;
    if (metadata_fused(p.num_seqs, p.total_tokens)) {
        paged_scan_kernel<true><<<1, kScanThreads, 0, st>>>(a, nullptr);
        FDMS_CHECK_LAUNCH("paged_scan_kernel");
        return FDMS_OK;
    }
    const int64_t need = fdms_paged_metadata_workspace_bytes(p.num_seqs, p.total_tokens);
    FDMS_REQUIRE((p.workspace || need == 0) && ((uintptr_t)p.workspace & 7) == 0 && p.workspace_bytes >= need, FDMS_E_WORKSPACE,
                 "fdms_paged_metadata: workspace missing, unaligned or smaller than %lld bytes", (long long)need);
    paged_scan_kernel<false><<<1, kScanThreads, 0, st>>>(a, (Served*)p.workspace);
    FDMS_CHECK_LAUNCH("paged_scan_kernel");
    if (p.total_tokens == 0) return FDMS_OK;
    const int64_t per = kFillThreads * kFillTokens;
    FDMS_CUDA_OK(launch_chained(paged_fill_kernel, dim3((unsigned)((p.total_tokens + per - 1) / per)), dim3(kFillThreads), st, true, a,
                                (const Served*)p.workspace));
    FDMS_CHECK_LAUNCH("paged_fill_kernel");
    return FDMS_OK;
}

extern "C" int32_t fdms_paged_release_pool(
    const int32_t* rows, int32_t num_listed, int32_t* kv_lens, int32_t num_rows, int32_t* block_tables, int64_t bt_stride,
    int32_t max_blocks, int32_t block_size, int32_t* free_blocks, int64_t free_capacity, int64_t num_blocks, int32_t* free_count,
    int32_t* dev_status, void* stream) {
    clear_error();
    FDMS_REQUIRE(free_count && (free_blocks || free_capacity == 0) && ((kv_lens && (block_tables || max_blocks == 0)) || num_rows == 0), FDMS_E_ARG,
                 "fdms_paged_release: null pointer");
    const int32_t shift = block_shift(block_size);
    FDMS_REQUIRE(shift > 0, FDMS_E_ARG, "fdms_paged_release: block_size must be 16, 32, 64 or 128, got %d", block_size);
    FDMS_REQUIRE(num_listed >= 0 && num_rows >= 0 && max_blocks >= 0 && free_capacity >= 0 && num_blocks >= 0 && bt_stride >= max_blocks, FDMS_E_ARG,
                 "fdms_paged_release: negative size, or rows of the block table overlap");
    FDMS_REQUIRE(rows || num_listed <= num_rows, FDMS_E_ARG, "fdms_paged_release: more rows than the block table has");
    FDMS_REQUIRE(num_listed <= kReleaseRows && free_capacity <= (0x7fffffffll >> shift) && num_blocks <= (0x7fffffffll >> shift), FDMS_E_CAPACITY,
                 "fdms_paged_release: at most %d rows a call, and slot numbers must fit in 31 bits", kReleaseRows);
    if (num_listed == 0) return FDMS_OK;
    paged_release_kernel<<<1, kReleaseThreads, 0, (cudaStream_t)stream>>>(rows, num_listed, kv_lens, num_rows, block_tables, bt_stride, max_blocks,
                                                                         shift, free_blocks, free_capacity, num_blocks, free_count, dev_status);
    FDMS_CHECK_LAUNCH("paged_release_kernel");
    return FDMS_OK;
}

extern "C" int32_t fdms_paged_release(
    const int32_t* rows, int32_t num_listed, int32_t* kv_lens, int32_t num_rows, int32_t* block_tables, int64_t bt_stride,
    int32_t max_blocks, int32_t block_size, int32_t* free_blocks, int64_t free_capacity, int32_t* free_count,
    int32_t* dev_status, void* stream) {
    return fdms_paged_release_pool(rows, num_listed, kv_lens, num_rows, block_tables, bt_stride, max_blocks, block_size, free_blocks, free_capacity,
                                   free_capacity, free_count, dev_status, stream);
}

extern "C" int32_t fdms_paged_store(const fdms_paged_store_args* args, void* stream) {
    clear_error();
    FDMS_REQUIRE(args, FDMS_E_ARG, "fdms_paged_store: null pointer");
    const fdms_paged_store_args& p = *args;
    const fdms_paged_cache& c = p.cache;
    int32_t shift = 0;
    const int32_t rc = paged_cache_check("fdms_paged_store", c, p.act_dtype, p.tokens == 0, shift);
    if (rc != FDMS_OK) return rc;
    FDMS_REQUIRE(p.tokens >= 0, FDMS_E_ARG, "fdms_paged_store: negative size");
    if (p.tokens == 0 || c.num_blocks == 0) return FDMS_OK;
    FDMS_REQUIRE(p.k && p.v && p.slot_mapping, FDMS_E_ARG, "fdms_paged_store: null pointer");
    const uintptr_t act = (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)(2 * (p.k_stride[0] | p.k_stride[1] | p.v_stride[0] | p.v_stride[1]));
    FDMS_REQUIRE((act & 15) == 0 && p.k_stride[2] == 1 && p.v_stride[2] == 1, FDMS_E_ARG,
                 "fdms_paged_store: key and value must be contiguous in their last dimension and aligned to 16 bytes in the others");
    // Small steps: a warp per (run, head); large ones: one per 16 rows of it.  256 tokens for as many blocks of 64 take 4.9 us
    // with the first and 12.9 with the second, 8000 prompt tokens 15.9 and 14.7.
    const int W = p.tokens <= kStoreSmall ? 1 : (int)c.block_size / 16, per_cta = kStoreWarps / W;
    const int64_t columns = (2 * c.kv_heads + per_cta - 1) / per_cta;
    // Tokens per CTA: a run begins at every token of a decode batch, but only once in a block of a prompt, and a CTA without one
    // is not free: at most 32 tokens, a block's worth, until the CTAs are two rounds of what the GPU holds.
    int group = 1;
    while (group < (c.block_size > 16 ? 32 : 16) && (p.tokens + group - 1) / group * columns > 1184) group *= 2;
    StoreArgs a = {{(const uint16_t*)p.k, (const uint16_t*)p.v}, {p.k_stride[0], p.v_stride[0]}, {p.k_stride[1], p.v_stride[1]}, {c.k, c.v},
                   {c.k_stride[0], c.v_stride[0]}, {c.k_stride[1], c.v_stride[1]}, {c.k_stride[2], c.v_stride[2]}, {c.k_scale, c.v_scale},
                   p.slot_mapping, p.dev_status, p.tokens, c.num_blocks << shift, (int32_t)c.kv_heads, shift, group, W};
    const int64_t ctas = (p.tokens + group - 1) / group;
    FDMS_REQUIRE(ctas < (1ll << 31), FDMS_E_CAPACITY, "fdms_paged_store: too many tokens");
    const dim3 grid((unsigned)ctas, (unsigned)columns);
    cudaStream_t st = (cudaStream_t)stream;
    const bool bf = p.act_dtype == FDMS_BF16;
    if (c.head_dim == 64) {
        if (bf) paged_store_kernel<64, true><<<grid, kStoreWarps * 32, 0, st>>>(a);
        else paged_store_kernel<64, false><<<grid, kStoreWarps * 32, 0, st>>>(a);
    } else {
        if (bf) paged_store_kernel<128, true><<<grid, kStoreWarps * 32, 0, st>>>(a);
        else paged_store_kernel<128, false><<<grid, kStoreWarps * 32, 0, st>>>(a);
    }
    FDMS_CHECK_LAUNCH("paged_store_kernel");
    return FDMS_OK;
}
