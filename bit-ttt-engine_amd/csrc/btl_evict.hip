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
constexpr int kHeld = 8192;              // keys that LDS holds

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
// joins them.  Heads of up to kSpan positions (ONE, by the host's bound) are held in
// registers between the passes; longer ones are read for each, and what shares the first
// digit of the sought weight, few of many, is held in LDS after the second.
// grid nkv * n_seqs, block 1024.
template <bool ONE>
__global__ __launch_bounds__(kThreads) void k_evict_choose(PagedEvict a)
{
    // the counts of a digit; the keys that share the first one; the sources that move
    __shared__ uint32_t s_bin[kBins];
    __shared__ uint32_t s_key[ONE ? 1 : kHeld];
    __shared__ int s_wave[2][kWaves];
    __shared__ uint32_t s_found[2], s_count;
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
    const int sink = a.sink ? a.sink[s] : 0;
    // the first token of the last ones (tokens are int32, so a bound past them is the bound)
    const int64_t first_late = (int64_t)len + shift - (a.recent ? max(a.recent[s], 0) : 0);
    const int late = (int)max(min(first_late, (int64_t)INT_MAX), (int64_t)INT_MIN);
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
    int32_t* from = a.from + head * a.from_ld;  // [keep]: where a hole's bytes come from; -1: it is none
    int32_t* movers = a.movers + head * c.cap;  // the sources, behind as many places as there are holes

    // A thread's positions of a span: four neighbours at a time, a wave 256 of them.
    auto place = [&](int base, int e) { return base + 256 * ((kEach / 4) * wave + e / 4) + 4 * lane + e % 4; };
    struct Each {
        float w[kEach];
        int t[kEach];
    };
    auto load = [&](int base, Each& x) {
#pragma unroll
        for (int e = 0; e < kEach; e += 4) {
            const int j = place(base, e);
            if (j + 4 <= len) {
                const Four w = *(const Four*)(weight + j);
#pragma unroll
                for (int i = 0; i < 4; ++i) x.w[e + i] = __uint_as_float(w.v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) x.w[e + i] = j + i < len ? weight[j + i] : 0.0f;
            }
        }
        if (base < filled) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int j = place(base, e);
                x.t[e] = j < min(filled, len) ? token[j] : (int)((uint32_t)j + (uint32_t)shift);
            }
        } else {
#pragma unroll
            for (int e = 0; e < kEach; ++e) x.t[e] = (int)((uint32_t)place(base, e) + (uint32_t)shift);
        }
    };
    auto key_of = [&](const Each& x, int e) {
        return x.t[e] < sink || x.t[e] >= late ? 0xFFFFFFFFu : order_of(x.w[e]);
    };
    // f(key, position) of every position, a span's loads ahead of the work on the one before
    Each x;
    if (ONE) load(0, x);
    auto each = [&](auto f) {
        if (ONE) {
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (place(0, e) < len) f(key_of(x, e), place(0, e));
            return;
        }
        load(0, x);
        for (int base = 0; base < len; base += kSpan) {
            uint32_t key[kEach];
#pragma unroll
            for (int e = 0; e < kEach; ++e) key[e] = key_of(x, e);
            if (base + kSpan < len) load(base + kSpan, x);
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (place(base, e) < len) f(key[e], place(base, e));
        }
    };

    // the keep-th largest key, digit by digit from the top; `left`: its rank among those that
    // share the digits so far
    uint32_t found = 0, left = (uint32_t)keep;
    int held = -1;  // keys in LDS that share the first digit (-1: they are looked for)
    for (int digit = 0; digit < 3 && keep > 0; ++digit) {
        const int low = digit == 0 ? 20 : (digit == 1 ? 10 : 0), bins = digit == 0 ? kBins : 1024;
        for (int i = tid; i < bins; i += kThreads) s_bin[i] = 0;
        if (tid == 0) s_count = 0;
        __syncthreads();
        auto count = [&](uint32_t key) { atomicAdd(&s_bin[key >> low & (uint32_t)(bins - 1)], 1u); };
        if (digit == 0) {
            each([&](uint32_t key, int) { count(key); });
        } else if (held >= 0) {
            for (int i = tid; i < held; i += kThreads)
                if (s_key[i] >> (low + 10) == found >> (low + 10)) count(s_key[i]);
        } else {
            each([&](uint32_t key, int) {
                if (key >> (low + 10) != found >> (low + 10)) return;
                count(key);
                if (!ONE && digit == 1) {
                    const uint32_t at = atomicAdd(&s_count, 1u);
                    if (at < kHeld) s_key[at] = key;
                }
            });
        }
        __syncthreads();
        if (!ONE && digit == 1 && s_count <= kHeld) held = (int)s_count;
        // thread i has the bins from the top: per thread, then over the threads
        const int per = bins / kThreads;
        uint32_t mine[kBins / kThreads];
        int sum = 0;
#pragma unroll
        for (int i = 0; i < kBins / kThreads; ++i) {
            mine[i] = i < per ? s_bin[bins - 1 - (per * tid + i)] : 0;
            sum += (int)mine[i];
        }
        int all;
        int before = wave_before(sum, lane, all);
        if (lane == 0) s_wave[0][wave] = all;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) before += w < wave ? s_wave[0][w] : 0;
        uint32_t run = (uint32_t)before;
#pragma unroll
        for (int i = 0; i < kBins / kThreads; ++i) {
            if (run < left && run + mine[i] >= left) {
                s_found[0] = (uint32_t)(bins - 1 - (per * tid + i)) << low;
                s_found[1] = left - run;
            }
            run += mine[i];
        }
        __syncthreads();
        found |= s_found[0];
        left = s_found[1];
    }

    // in order: what is above the key stays, and the first `left` of its equals
    int equal = 0, moved = 0;  // so far
    if (!ONE) load(0, x);
    for (int base = 0; base < len; base += kSpan) {
        uint32_t same = 0, above = 0;  // bit e: of this thread's positions
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const uint32_t key = key_of(x, e);
            const bool in = keep > 0 && place(base, e) < len;
            same |= (uint32_t)(in && key == found) << e;
            above |= (uint32_t)(in && key > found) << e;
        }
        if (!ONE && base + kSpan < len) load(base + kSpan, x);
        int all = 0, ties[kEach / 4];  // equals ahead of each four
#pragma unroll
        for (int e = 0; e < kEach; e += 4) {
            int sum;
            ties[e / 4] = all + wave_before(__popc(same >> e & 15u), lane, sum);
            all += sum;
        }
        if (lane == 0) s_wave[0][wave] = all;
        __syncthreads();
        int ahead = equal;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int n = s_wave[0][w];
            ahead += w < wave ? n : 0;
            equal += n;
        }
        uint32_t is = 0;  // a hole, or a source
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int j = place(base, e), t = ahead + ties[e / 4] + __popc(same >> (e & ~3) & ((1u << (e & 3)) - 1));
            const bool stays = (above >> e & 1) || ((same >> e & 1) && t < (int)left);
            is |= (uint32_t)(j < keep ? !stays : stays) << e;
        }
        int before[kEach / 4];
        all = 0;
#pragma unroll
        for (int e = 0; e < kEach; e += 4) {
            int sum;
            before[e / 4] = all + wave_before(__popc(is >> e & 15u), lane, sum);
            all += sum;
        }
        if (lane == 0) s_wave[1][wave] = all;
        __syncthreads();
        int rank = moved;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int n = s_wave[1][w];
            rank += w < wave ? n : 0;
            moved += n;
        }
        // the n-th hole or source in order
        auto nth = [&](int e) { return rank + before[e / 4] + __popc(is >> (e & ~3) & ((1u << (e & 3)) - 1)); };
        if (ONE) {
            // the sources are joined with the holes through LDS
            const int holes = moved / 2;  // the sources stand behind as many holes
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (place(0, e) >= keep && (is >> e & 1)) s_bin[nth(e) - holes] = (uint32_t)place(0, e);
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int j = place(0, e);
                if (j >= keep) continue;
                if (is >> e & 1) {
                    const int src = (int)s_bin[nth(e)];
                    from[j] = src;
                    weight_out[j] = weight[src];
                    token_out[j] = token_at(src);
                } else {
                    from[j] = -1;
                    weight_out[j] = x.w[e];
                    token_out[j] = x.t[e];
                }
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int j = place(base, e);
            if (j < keep) from[j] = is >> e & 1 ? nth(e) : -1;
            else if (is >> e & 1) movers[nth(e)] = j;
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
    // The values' block is put together from the blocks that its slots' bytes lie in, each
    // loaded once, whole: a lane has 16 slots of its values 2 lane and 2 lane + 1.  A byte
    // permute picks four slots' bytes out of eight at a time.
    const bool act = 2 * lane < hd;
    const int mine = (int)(slot >> 4);  // below 2^31: the host checks it
    u4 lo = {0, 0, 0, 0}, hi = lo;
    uint32_t todo = 0xFFFFu;
    while (todo) {
        constexpr int U = 4;  // blocks in flight
        u4 b0[U], b1[U];
        uint32_t who[U];
#pragma unroll
        for (int x = 0; x < U; ++x) {
            who[x] = 0;
            if (todo) {
                const int group = __builtin_amdgcn_readlane(mine, __ffs(todo) - 1);
                who[x] = (uint32_t)__ballot(mine == group) & todo;
                todo &= ~who[x];
                const u4* p = (const u4*)(c.v + 16 * (int64_t)group * hd + (act ? 32 * lane : 0));
                b0[x] = p[0];
                b1[x] = p[1];
            }
        }
#pragma unroll
        for (int x = 0; x < U; ++x)
            if (who[x]) {
                // lane r: which byte of the first and of the last eight slots r takes (12: zero)
                const int at = (int)(slot & 15);
                const bool in = who[x] >> r & 1;
                uint32_t first = (uint32_t)(in && at < 8 ? at : 12) << (8 * (r & 3));
                uint32_t last = (uint32_t)(in && at >= 8 ? at - 8 : 12) << (8 * (r & 3));
                first |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)first, 0xB1, 0xF, 0xF, true);  // quad [1,0,3,2]
                last |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)last, 0xB1, 0xF, 0xF, true);
                first |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)first, 0x4E, 0xF, 0xF, true);  // quad [2,3,0,1]
                last |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)last, 0x4E, 0xF, 0xF, true);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const uint32_t f = (uint32_t)__builtin_amdgcn_readlane((int)first, 4 * d);
                    const uint32_t l = (uint32_t)__builtin_amdgcn_readlane((int)last, 4 * d);
                    lo[d] |= __builtin_amdgcn_perm(b0[x].y, b0[x].x, f) | __builtin_amdgcn_perm(b0[x].w, b0[x].z, l);
                    hi[d] |= __builtin_amdgcn_perm(b1[x].y, b1[x].x, f) | __builtin_amdgcn_perm(b1[x].w, b1[x].z, l);
                }
            }
    }
    if (!act) return;
    u4* o = (u4*)(c.v + blk * hd + 32 * lane);
    o[0] = lo;
    o[1] = hi;
}

hipError_t launch_paged_evict(const PagedEvict& a, hipStream_t st)
{
    const dim3 heads((unsigned)(a.c.nkv * a.c.n_seqs));
    if (a.c.cap > kSpan) hipLaunchKernelGGL(k_evict_choose<false>, heads, dim3(kThreads), 0, st, a);
    else if (a.c.cap) hipLaunchKernelGGL(k_evict_choose<true>, heads, dim3(kThreads), 0, st, a);
    const int blocks = evict_blocks(a);
    hipLaunchKernelGGL(k_evict_move, dim3((unsigned)(a.c.nkv * blocks * a.c.n_seqs)), dim3(256), 0, st, a, blocks);
    return hipGetLastError();
}

}  // namespace btl
