// btl_evict.hip -- gfx950 kernels that cut sequences of a paged Q8 cache down to their
// positions of most weight.
//
// Kernels:
//   k_evict_choose   per (sequence, KV head): which positions stay, where each goes.
//   k_evict_move     the moved positions' codes and scales.
//
// Of a head's `len` positions the `keep` first in the order (protected, weight, position)
// stay.  Those below `keep` stay where they are; the n-th evicted one below `keep` (a
// hole) takes the n-th that stays from `keep` on.  So sources and holes share no slot,
// and moves need no order.
#include <hip/hip_runtime.h>

#include "btl_paged.hpp"

namespace btl {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kEach = 8;                 // positions of a thread at a time
constexpr int kSpan = kThreads * kEach;  // positions of the workgroup at a time
constexpr int kBins = 4096;              // of the first 12 bits; the next two digits have 10

// What a sequence is cut down to.
struct Cut {
    int len, keep;
    bool ok;
};

__device__ __forceinline__ Cut cut_of(const PagedEvict& a, int s)
{
    const Seq q = seq_at(a.c, s);
    const int keep = a.keep[s];
    Cut x;
    x.len = q.p0 + q.n;
    x.ok = q.ok && (keep < 0 || keep >= x.len || keep <= a.max_keep);
    x.keep = keep < 0 ? x.len : min(keep, x.len);
    return x;
}

// Whole numbers in the order of the weights: NaN below everything, -0 as +0.
__device__ __forceinline__ uint32_t order_of(float w)
{
    const uint32_t b = __float_as_uint(w);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0;
    return b << 1 == 0 ? 0x80000000u : (b >> 31 ? ~b : b | 0x80000000u);
}

// sum of v over the lanes below, and over all
__device__ __forceinline__ int wave_before(int v, int lane, int& all)
{
    int upto = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(upto, off, 64);
        upto += lane >= off ? o : 0;
    }
    all = __builtin_amdgcn_readlane(upto, 63);
    return upto - v;
}

}  // namespace

// ---------------------------------------------------------------------------
// k_evict_choose
// ---------------------------------------------------------------------------
// A workgroup a (sequence, KV head).  The keep-th largest weight is found by counting
// digits of 12, 10 and 10 bits; then one pass in order ranks holes and sources, and one
// joins them.  grid nkv * n_seqs, block 1024.
__global__ __launch_bounds__(kThreads) void k_evict_choose(PagedEvict a)
{
    __shared__ uint32_t s_bin[kBins];
    __shared__ int s_wave[2][kWaves];
    __shared__ uint32_t s_found[2];
    const Paged& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = (int)(blockIdx.x % (unsigned)c.nkv), s = (int)(blockIdx.x / (unsigned)c.nkv);
    const Cut cut = cut_of(a, s);
    if (!cut.ok) return;
    const int len = cut.len, keep = cut.keep;
    const int64_t head = (int64_t)s * c.nkv + h;
    const float* weight = a.weight + head * a.ld;
    const int32_t* token = a.token + head * a.ld;
    float* weight_out = a.weight_out + head * a.ld_out;
    int32_t* token_out = a.token_out + head * a.ld_out;
    const int filled = a.filled[s], shift = a.shift[s];
    const int64_t sink = a.sink ? a.sink[s] : 0, late = (int64_t)len + shift - (a.recent ? max(a.recent[s], 0) : 0);
    auto token_at = [&](int j) { return j < filled ? token[j] : (int)((uint32_t)j + (uint32_t)shift); };
    if (keep == len) {
        for (int j = tid; j < len; j += kThreads) {
            const float w = weight[j];
            const int t = token_at(j);
            weight_out[j] = w;
            token_out[j] = t;
        }
        return;
    }
    int32_t* from = a.from + head * a.from_ld;  // [keep]: a hole's rank, then its source; -1: stays
    int32_t* movers = a.movers + head * c.cap;  // the sources, behind as many places as there are holes

    // the keys of this thread's positions of a span: wave by wave, 64 neighbours at a time
    uint32_t key[kEach];
    auto load = [&](int base) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int j = base + 64 * (kEach * wave + e) + lane;
            key[e] = 0;
            if (j < len) {
                const int64_t t = token_at(j);
                key[e] = t < sink || t >= late ? 0xFFFFFFFFu : order_of(weight[j]);
            }
        }
    };
    const bool one = len <= kSpan;  // one span: loaded once
    if (one) load(0);

    // the keep-th largest key, digit by digit from the top; `left`: its rank among those that
    // share the digits so far
    uint32_t found = 0, left = (uint32_t)keep;
    for (int digit = 0; digit < 3 && keep > 0; ++digit) {
        const int low = digit == 0 ? 20 : (digit == 1 ? 10 : 0), bins = digit == 0 ? kBins : 1024;
        for (int i = tid; i < bins; i += kThreads) s_bin[i] = 0;
        __syncthreads();
        for (int base = 0; base < len; base += kSpan) {
            if (!one) load(base);
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int j = base + 64 * (kEach * wave + e) + lane;
                const bool mine = digit == 0 || key[e] >> (low + 10) == found >> (low + 10);
                if (j < len && mine) atomicAdd(&s_bin[key[e] >> low & (uint32_t)(bins - 1)], 1u);
            }
        }
        __syncthreads();
        // thread i has the bins from the top: per thread, then over the threads
        const int per = bins / kThreads;
        uint32_t count[kBins / kThreads];
        int mine = 0;
#pragma unroll
        for (int i = 0; i < kBins / kThreads; ++i) {
            count[i] = i < per ? s_bin[bins - 1 - (per * tid + i)] : 0;
            mine += (int)count[i];
        }
        int all;
        int before = wave_before(mine, lane, all);
        if (lane == 0) s_wave[0][wave] = all;
        __syncthreads();
        for (int w = 0; w < wave; ++w) before += s_wave[0][w];
        uint32_t run = (uint32_t)before;
#pragma unroll
        for (int i = 0; i < kBins / kThreads; ++i) {
            if (run < left && run + count[i] >= left) {
                s_found[0] = (uint32_t)(bins - 1 - (per * tid + i)) << low;
                s_found[1] = left - run;
            }
            run += count[i];
        }
        __syncthreads();
        found |= s_found[0];
        left = s_found[1];
    }

    // in order: what is above the key stays, and the first `left` of its equals
    int equal = 0, moved = 0;  // so far
    for (int base = 0; base < len; base += kSpan) {
        if (!one) load(base);
        uint64_t same[kEach];
        int sum = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int j = base + 64 * (kEach * wave + e) + lane;
            same[e] = __ballot(keep > 0 && j < len && key[e] == found);
            sum += __popcll(same[e]);
        }
        if (lane == 0) s_wave[0][wave] = sum;
        __syncthreads();
        int ties = equal;
        for (int w = 0; w < kWaves; ++w) {
            ties += w < wave ? s_wave[0][w] : 0;
            equal += s_wave[0][w];
        }
        uint64_t flag[kEach];
        const uint64_t below = ((uint64_t)1 << lane) - 1;
        sum = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int j = base + 64 * (kEach * wave + e) + lane;
            const bool tie = same[e] >> lane & 1;
            const bool stays = keep > 0 && j < len && (tie ? ties + __popcll(same[e] & below) < (int)left : key[e] > found);
            ties += __popcll(same[e]);
            flag[e] = __ballot(j < keep ? !stays : stays);  // a hole, or a source
            sum += __popcll(flag[e]);
        }
        if (lane == 0) s_wave[1][wave] = sum;
        __syncthreads();
        int rank = moved;
        for (int w = 0; w < kWaves; ++w) {
            rank += w < wave ? s_wave[1][w] : 0;
            moved += s_wave[1][w];
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int j = base + 64 * (kEach * wave + e) + lane;
            const bool is = flag[e] >> lane & 1;
            const int at = rank + __popcll(flag[e] & below);
            rank += __popcll(flag[e]);
            if (j < keep) from[j] = is ? at : -1;
            else if (is) movers[at] = j;
        }
    }
    __syncthreads();
    // as many sources as holes, behind them in the count
    const int holes = moved / 2;
    for (int j = tid; j < keep; j += kThreads) {
        const int r = from[j];
        const int src = r < 0 ? j : movers[holes + r];
        if (r >= 0) from[j] = src;
        const float w = weight[src];
        const int t = token_at(src);
        weight_out[j] = w;
        token_out[j] = t;
    }
}

// ---------------------------------------------------------------------------
// k_evict_move
// ---------------------------------------------------------------------------
// A wave a block of 16 slots below `keep` of a (sequence, KV head): the holes' keys row by
// row, and its values' block made anew from the bytes of the slots that are to lie in it
// (a slot that stays gives its own).  grid nkv * ceil(max_keep / 64) * n_seqs, block 256.
__global__ __launch_bounds__(256) void k_evict_move(PagedEvict a, int blocks)
{
    const Paged& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = (int)(blockIdx.x % (unsigned)c.nkv);
    const unsigned at = blockIdx.x / (unsigned)c.nkv;
    const int block = 4 * (int)(at % (unsigned)blocks) + wave, s = (int)(at / (unsigned)blocks);
    const Cut cut = cut_of(a, s);
    if (h == 0 && block == 0 && lane == 0) {
        a.held[s] = cut.ok ? cut.keep : -1;
        if (cut.ok) {
            const int shift = a.shift[s];
            a.filled_out[s] = cut.keep;
            a.shift_out[s] = (int)((uint32_t)shift + (uint32_t)(cut.len - cut.keep));
        }
    }
    const int j0 = 16 * block;
    if (!cut.ok || cut.keep == cut.len || j0 >= cut.keep) return;
    const int hd = c.hd;
    const int32_t* table = c.pages + (int64_t)s * c.max_pages;
    // lane r < 16: where the slot j0 + r comes from (-1: stays)
    const int r = lane & 15;
    const int src = j0 + r < cut.keep ? a.from[((int64_t)s * c.nkv + h) * a.from_ld + j0 + r] : -1;
    if (!__any(src >= 0)) return;
    int in;
    const int page = page_of(c, table, block, &in);
    if (page < 0) return;  // no slot to write
    const int64_t blk = ((int64_t)page * c.nkv + h) * c.ps + 16 * in;
    int src_in;
    const int src_page = page_of(c, table, src >= 0 ? src >> 4 : block, &src_in);
    // the slot in the pool that r's bytes are taken from; a page outside the pool has none
    const bool lost = src_page < 0;
    const int64_t slot = lost || src < 0 ? blk + r : ((int64_t)src_page * c.nkv + h) * c.ps + 16 * src_in + (src & 15);
    const uint64_t holes = __ballot(lane < 16 && src >= 0);
    if (lane < 16 && src >= 0) {
        const float ks = c.ks[slot], vs = c.vs[slot];
        c.ks[blk + r] = lost ? __builtin_nanf("") : ks;  // whoever sees it is NaN
        c.vs[blk + r] = lost ? __builtin_nanf("") : vs;
    }
    auto slot_of = [&](int x) { return (int64_t)__shfl((long long)slot, x, 64); };
    const int D = hd >> 4, mul = (1024 + D - 1) / D;  // x / D = x * mul >> 10 for x < 192
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int x = lane + 64 * e, row = min(x * mul >> 10, 15);  // 16-byte piece x, of slot j0 + row
        const int64_t k0 = slot_of(row);
        if (x < hd && (holes >> row & 1)) *(uint4*)(c.k + blk * hd + 16 * x) = *(const uint4*)(c.k + k0 * hd + 16 * (x - row * D));
    }
    uint32_t lo[4] = {}, hi[4] = {};
    const bool act = 2 * lane < hd;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
        const int64_t v0 = slot_of(x);
        const uint8_t* p = c.v + (v0 & ~(int64_t)15) * hd + (v0 & 15) + 32 * lane;
        const uint32_t b0 = act ? p[0] : 0, b1 = act ? p[16] : 0;
        lo[x >> 2] |= b0 << (8 * (x & 3));
        hi[x >> 2] |= b1 << (8 * (x & 3));
    }
    if (!act) return;
    uint4* o = (uint4*)(c.v + blk * hd + 32 * lane);
    o[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    o[1] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
}

hipError_t launch_paged_evict(const PagedEvict& a, hipStream_t st)
{
    if (a.c.cap) hipLaunchKernelGGL(k_evict_choose, dim3((unsigned)(a.c.nkv * a.c.n_seqs)), dim3(kThreads), 0, st, a);
    const int blocks = evict_blocks(a);
    hipLaunchKernelGGL(k_evict_move, dim3((unsigned)(a.c.nkv * blocks * a.c.n_seqs)), dim3(256), 0, st, a, blocks);
    return hipGetLastError();
}

}  // namespace btl
