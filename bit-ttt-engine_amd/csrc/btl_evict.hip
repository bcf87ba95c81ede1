// btl_evict.hip -- gfx950 kernels that cut sequences of a paged Q8 cache down to their
// positions of most weight.
//
// Kernels:
//   k_evict_choose   per (sequence, KV head): which positions stay, where each goes;
//   k_evict_count, k_evict_collect, k_evict_rank   the same for long sequences.
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

constexpr int kThreads = 1024, kWaves = kThreads / 64;  // of the largest workgroups
constexpr int kEach = 8;                 // positions of a thread at a time
constexpr int kSpan = kThreads * kEach;  // positions of a workgroup at a time
static_assert(kSpan == kEvictSpan, "the host sizes the workspace by it");
constexpr int kBins = kEvictBins;        // of a digit: 11, 11 and 10 bits

// What a sequence is cut down to, and what its arguments say: all read at once.
struct Cut {
    int len, keep, filled, shift, sink, recent;
    bool ok;
};

__device__ __forceinline__ Cut cut_of(const PagedEvict& a, int s, const int32_t* filled, const int32_t* shift)
{
    const Seq q = seq_at(a.c, s);
    const int keep = a.keep[s];
    Cut x;
    x.filled = filled[s];
    x.shift = shift[s];
    x.sink = a.sink ? a.sink[s] : 0;
    x.recent = a.recent ? max(a.recent[s], 0) : 0;
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

// the sum of v over the lanes up to this one
__device__ __forceinline__ int wave_upto(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);  // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);  // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);  // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, true);  // row_bcast:15
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, true);  // row_bcast:31
    return v;
}

// its sum over the lanes below, and over all
__device__ __forceinline__ int wave_before(int v, int& all)
{
    const int upto = wave_upto(v);
    all = __builtin_amdgcn_readlane(upto, 63);
    return upto - v;
}

// One head of a sequence.
struct Head {
    const float* weight;
    const int32_t* token;
    float* weight_out;
    int32_t* token_out;
    int32_t* from;  // [keep]: -1 where a position stays
    int len, keep, filled, shift;
    int sink, last;  // tokens below the first and above the second are protected

    __device__ __forceinline__ Head(const PagedEvict& a, const Cut& cut, int64_t head)
        : weight(a.weight + head * a.ld), token(a.token + head * a.ld), weight_out(a.weight_out + head * a.ld_out),
          token_out(a.token_out + head * a.ld_out), from(a.from + head * a.c.cap), len(cut.len), keep(cut.keep),
          filled(cut.filled), shift(cut.shift), sink(cut.sink)
    {
        // the recent ones: a bound past every token leaves none, one at or below the least all
        const int64_t bound = (int64_t)len + shift - cut.recent;
        last = bound <= INT_MIN ? INT_MAX - 1 : (int)min(bound - 1, (int64_t)INT_MAX);
        if (bound <= INT_MIN) sink = INT_MAX;
    }
    __device__ __forceinline__ int in_order(int j) const { return (int)((uint32_t)j + (uint32_t)shift); }
    __device__ __forceinline__ int token_at(int j) const { return j < filled ? token[j] : in_order(j); }
    // position `to` takes what position `src` has
    __device__ __forceinline__ void put(int to, int src) const
    {
        const float w = weight[src];
        const int t = token_at(src);
        weight_out[to] = w;
        token_out[to] = t;
    }
};

// A thread's positions of a span: four neighbours at a time, a wave 256 of them.
struct Each {
    float w[kEach];
    int t[kEach];
    int first;  // position of element 0

    __device__ __forceinline__ int at(int e) const { return first + 256 * (e >> 2) + (e & 3); }

    __device__ __forceinline__ void load(const Head& h, int base, int tid)
    {
        first = base + 64 * kEach * (tid >> 6) + 4 * (tid & 63);
#pragma unroll
        for (int e = 0; e < kEach; e += 4) {
            const int j = at(e);
            if (j + 4 <= h.len) {
                const Four x = *(const Four*)(h.weight + j);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[e + i] = __uint_as_float(x.v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[e + i] = j + i < h.len ? h.weight[j + i] : 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) t[e] = h.in_order(at(e));
        if (base >= h.filled) return;
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            if (at(e) < min(h.filled, h.len)) t[e] = h.token[at(e)];
    }
    // protected positions are above every weight
    __device__ __forceinline__ uint32_t key(const Head& h, int e) const
    {
        return t[e] < h.sink || t[e] > h.last ? 0xFFFFFFFFu : order_of(w[e]);
    }
};

// What a workgroup of T threads counts with.
template <int T = kThreads>
struct Lds {
    uint32_t bin[kBins];
    int wave[2][T / 64];
    uint32_t found[3];
};

// The sought key, digit by digit from the top: it lies among those whose bits from `low` on
// are `top`'s, as the left-th largest of them.
struct Sought {
    uint32_t top;
    int left, low;
    bool all;  // all of those stay
};

// count(f) hands every key to f.  Narrows x down by one digit.
template <int T, typename F>
__device__ __forceinline__ void narrow(Lds<T>& s, Sought& x, int tid, F count)
{
    constexpr int B = kBins / T;  // of a thread
    const int low = x.low == 32 ? 21 : (x.low == 21 ? 10 : 0), bins = 1 << (x.low - low);
    const int lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < bins; i += T) s.bin[i] = 0;
    __syncthreads();
    count([&](uint32_t key) {
        if (x.low == 32 || key >> x.low == x.top >> x.low) atomicAdd(&s.bin[key >> low & (uint32_t)(bins - 1)], 1u);
    });
    __syncthreads();
    // thread i has the bins B i .. B i + B - 1 from the top
    uint32_t n[B];
    int mine = 0;
#pragma unroll
    for (int b = 0; b < B; ++b) {
        n[b] = B * tid < bins ? s.bin[bins - 1 - B * tid - b] : 0;
        mine += (int)n[b];
    }
    int all;
    int before = wave_before(mine, all);
    if (lane == 0) s.wave[0][wave] = all;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; ++w) before += w < wave ? s.wave[0][w] : 0;
    uint32_t run = (uint32_t)before;
    const uint32_t left = (uint32_t)x.left;
    if (run < left && run + (uint32_t)mine >= left) {
        bool open = true;
#pragma unroll
        for (int b = 0; b < B; ++b) {
            if (open && run + n[b] >= left) {
                s.found[0] = (uint32_t)(bins - 1 - B * tid - b) << low;
                s.found[1] = left - run;
                s.found[2] = n[b];
                open = false;
            }
            run += n[b];
        }
    }
    __syncthreads();
    x.top |= s.found[0];
    x.left = (int)s.found[1];
    x.low = low;
    x.all = s.found[1] == s.found[2];
}

// Which of a thread's positions stay, and their places in the order, over a workgroup.
// equal: equals of the sought key ahead of the span.
struct Flags {
    uint32_t same, stays;  // bit e
};

template <int T>
__device__ __forceinline__ Flags flags_of(Lds<T>& s, const Head& h, const Each& v, const Sought& x, int equal, int tid)
{
    const int lane = tid & 63, wave = tid >> 6;
    Flags f = {0, 0};
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const bool in = v.at(e) < h.len;
        const uint32_t key = v.key(h, e) >> x.low, top = x.top >> x.low;
        f.same |= (uint32_t)(in && key == top) << e;
        f.stays |= (uint32_t)(in && key > top) << e;
    }
    if (x.all) {  // no equals to tell apart
        f.stays |= f.same;
        return f;
    }
    int all = 0, ties[kEach / 4];
#pragma unroll
    for (int e = 0; e < kEach; e += 4) {
        int sum;
        ties[e / 4] = all + wave_before(__popc(f.same >> e & 15u), sum);
        all += sum;
    }
    if (lane == 0) s.wave[0][wave] = all;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; ++w) equal += w < wave ? s.wave[0][w] : 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int t = equal + ties[e / 4] + __popc(f.same >> (e & ~3) & ((1u << (e & 3)) - 1));
        f.stays |= (f.same >> e & 1u) && t < x.left ? 1u << e : 0u;
    }
    return f;
}

// The places of the marked positions (bit e of is) in the order, over the workgroup.
struct Ranks {
    int before[kEach / 4], all;

    template <int T>
    __device__ __forceinline__ Ranks(Lds<T>& s, uint32_t is, int tid)
    {
        const int lane = tid & 63, wave = tid >> 6;
        int mine = 0;
#pragma unroll
        for (int e = 0; e < kEach; e += 4) {
            int sum;
            before[e / 4] = mine + wave_before(__popc(is >> e & 15u), sum);
            mine += sum;
        }
        if (lane == 0) s.wave[1][wave] = mine;
        __syncthreads();
        int ahead = 0;
        all = 0;
#pragma unroll
        for (int w = 0; w < T / 64; ++w) {
            const int n = s.wave[1][w];
            ahead += w < wave ? n : 0;
            all += n;
        }
#pragma unroll
        for (int e = 0; e < kEach; e += 4) before[e / 4] += ahead;
    }
    __device__ __forceinline__ int of(uint32_t is, int e) const
    {
        return before[e / 4] + __popc(is >> (e & ~3) & ((1u << (e & 3)) - 1));
    }
};

}  // namespace

// ---------------------------------------------------------------------------
// k_evict_choose
// ---------------------------------------------------------------------------
// Heads of up to kSpan positions, a workgroup each, the positions in registers.  The
// keep-th largest weight is found by counting digits of 11, 11 and 10 bits; then holes and
// sources are ranked in order and joined through LDS.  grid nkv * n_seqs, block T.
//
// Bound by latency: one reading, and a barrier after each of some fifteen steps; 9.4 us for
// 64 heads of 1025, 15.4 for 256 of up to 8192.  Counting stops where all that share the
// digits so far stay.  Read from memory once a digit the latter took 5 us more.
//
// T is 512 where that takes sequences of the batch's bounds, up to 4096: fewer waves meet at a
// barrier, and two workgroups share a CU.  An eviction and its reading back, 64 heads of 1025
// cut by one 27.6 us so and 28.6 with 1024; 512 heads of 4000 cut down to 40 29.2 and 34.6
// (256 threads, up to 2048: 28.0 the first).
template <int T>
__global__ __launch_bounds__(T) void k_evict_choose(PagedEvict a)
{
    constexpr int kMoves = kEach * T / 2;
    __shared__ Lds<T> lds;
    __shared__ int s_source[kMoves], s_token[kMoves];  // of the positions that move: where, and what lies there
    __shared__ float s_weight[kMoves];
    const int tid = threadIdx.x;
    const int s = (int)(blockIdx.x / (unsigned)a.c.nkv);
    const Cut cut = cut_of(a, s, a.filled, a.shift);
    if (!cut.ok) return;
    const Head h(a, cut, blockIdx.x);
    if (h.keep == h.len) {
        for (int j = tid; j < h.len; j += T) h.put(j, j);
        return;
    }
    if (h.keep == 0) return;
    Each v;
    v.load(h, 0, tid);
    Sought x = {0, h.keep, 32, false};
    while (x.low > 0 && !x.all)
        narrow(lds, x, tid, [&](auto f) {
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (v.at(e) < h.len) f(v.key(h, e));
        });
    const Flags f = flags_of(lds, h, v, x, 0, tid);
    uint32_t is = 0;  // holes, and behind as many of them the sources
#pragma unroll
    for (int e = 0; e < kEach; ++e) is |= (v.at(e) < h.keep ? ~f.stays : f.stays) & 1u << e;
    const Ranks r(lds, is, tid);
    const int holes = r.all / 2;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (v.at(e) >= h.keep && (is >> e & 1u)) {
            const int at = r.of(is, e) - holes;
            s_source[at] = v.at(e);
            s_token[at] = v.t[e];
            s_weight[at] = v.w[e];
        }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int j = v.at(e);
        if (j >= h.keep) continue;
        const bool hole = is >> e & 1u;
        const int at = hole ? r.of(is, e) : 0;
        h.from[j] = hole ? s_source[at] : -1;
        h.weight_out[j] = hole ? s_weight[at] : v.w[e];
        h.token_out[j] = hole ? s_token[at] : v.t[e];
    }
}

// ---------------------------------------------------------------------------
// k_evict_count, k_evict_collect, k_evict_rank
// ---------------------------------------------------------------------------
// Longer heads, a workgroup a span of kSpan positions, block 1024, grid spans * nkv *
// n_seqs each.  k_evict_count counts the first digit; k_evict_collect finds the sought
// key's from all spans' counts and puts down the keys that share it; k_evict_rank finds
// the key among those and ranks its span's holes from the first on and its sources from
// the last back, which it knows from what stays in the spans before and behind.  The span
// that `keep` falls into puts down how many holes there are; k_evict_move joins them.
//
// Bound by latency: 8 heads of 100001, 104 workgroups, 4.8, 7.1 and 10.1 us (one workgroup a
// head, which goes through its head span by span, took 101 for all three).  A launch between
// them is the cheapest way to have all spans' counts; a wait inside one kernel would need all
// its workgroups to be resident.
//
// Every workgroup goes through all spans' counts, and through all keys that share the sought
// one's first digit, up to three times: where many do, the work grows with the square of the
// head's length.  With the move, weights spread; 95 % of them zero and the cut among those; all
// of one first digit: 8 heads of 100001 55, 228 and 126 us; 8 of 10^6 0.33, 7.0 and 2.2 ms; one of
// 2^23 1.1, 62 and 28 ms.
namespace {

struct Span {
    int h, s, part, base;
    int64_t head;
};

__device__ __forceinline__ Span span_of(const PagedEvict& a)
{
    Span p;
    p.h = (int)(blockIdx.x % (unsigned)a.c.nkv);
    const unsigned b = blockIdx.x / (unsigned)a.c.nkv;
    p.part = (int)(b % (unsigned)a.spans);
    p.s = (int)(b / (unsigned)a.spans);
    p.base = kSpan * p.part;
    p.head = (int64_t)p.s * a.c.nkv + p.h;
    return p;
}

}  // namespace

__global__ __launch_bounds__(kThreads) void k_evict_count(PagedEvict a)
{
    __shared__ uint32_t s_bin[kBins];
    const int tid = threadIdx.x;
    const Span p = span_of(a);
    const Cut cut = cut_of(a, p.s, a.filled, a.shift);
    if (!cut.ok || p.base >= cut.len || cut.keep == cut.len || cut.keep == 0) return;
    const Head h(a, cut, p.head);
    // k_evict_move may put out over what came in
    if (p.h == 0 && p.part == 0 && tid == 0) {
        a.was[p.s] = h.filled;
        a.was[a.c.n_seqs + p.s] = h.shift;
    }
    Each v;
    v.load(h, p.base, tid);
    for (int i = tid; i < kBins; i += kThreads) s_bin[i] = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (v.at(e) < h.len) atomicAdd(&s_bin[v.key(h, e) >> 21], 1u);
    __syncthreads();
    // two counts of at most kSpan a word
    uint32_t* to = a.counts + (p.head * a.spans + p.part) * (kBins / 2);
    for (int i = tid; i < kBins / 2; i += kThreads) to[i] = s_bin[2 * i] | s_bin[2 * i + 1] << 16;
}

__global__ __launch_bounds__(kThreads) void k_evict_collect(PagedEvict a)
{
    __shared__ Lds<> lds;
    __shared__ int s_above, s_count;
    const int tid = threadIdx.x;
    const Span p = span_of(a);
    const Cut cut = cut_of(a, p.s, a.filled, a.shift);
    if (!cut.ok || p.base >= cut.len || cut.keep == cut.len || cut.keep == 0) return;
    const Head h(a, cut, p.head);
    Each v;
    v.load(h, p.base, tid);
    const int spans = (h.len + kSpan - 1) / kSpan;
    if (tid == 0) s_above = s_count = 0;
    // the first digit of the sought key, from the sums of the spans' counts
    Sought x = {0, h.keep, 32, false};
    {
        const uint32_t* from = a.counts + p.head * a.spans * (kBins / 2) + tid;
        uint32_t n0 = 0, n1 = 0;
        for (int i0 = 0; i0 < spans; i0 += 16) {
            uint32_t n[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) n[i] = from[(int64_t)min(i0 + i, spans - 1) * (kBins / 2)];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                n0 += i0 + i < spans ? n[i] & 0xFFFFu : 0;
                n1 += i0 + i < spans ? n[i] >> 16 : 0;
            }
        }
        // thread i has the bins 2 i and 2 i + 1
        const int mine = (int)(n0 + n1), upto = wave_upto(mine), all = __builtin_amdgcn_readlane(upto, 63);
        if ((tid & 63) == 0) lds.wave[0][tid >> 6] = all;
        __syncthreads();
        int above = all - upto;  // in bins above this thread's
#pragma unroll
        for (int w = 0; w < kWaves; ++w) above += w > tid >> 6 ? lds.wave[0][w] : 0;
        if (above < h.keep && above + mine >= h.keep) {
            const bool high = above + (int)n1 >= h.keep;
            lds.found[0] = (uint32_t)(2 * tid + (high ? 1 : 0)) << 21;
            lds.found[1] = (uint32_t)(h.keep - above - (high ? 0 : (int)n1));
        }
        __syncthreads();
        x.top = lds.found[0];
        x.left = (int)lds.found[1];
    }
    uint32_t* keys = a.keys + p.head * a.c.cap + p.base;
    int above = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        if (v.at(e) >= h.len) continue;
        const uint32_t key = v.key(h, e);
        above += key >> 21 > x.top >> 21;
        // in no order: of equals only the number counts
        if (key >> 21 == x.top >> 21) keys[atomicAdd(&s_count, 1)] = key;
    }
    above = wave_upto(above);
    if ((tid & 63) == 63) atomicAdd(&s_above, above);
    __syncthreads();
    if (tid) return;
    int32_t* to = a.spanned + 4 * (p.head * a.spans + p.part);
    to[0] = s_above;
    to[1] = s_count;
    to[2] = (int)x.top;
    to[3] = x.left;
}

__global__ __launch_bounds__(kThreads) void k_evict_rank(PagedEvict a)
{
    __shared__ Lds<> lds;
    __shared__ int s_ahead[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Span p = span_of(a);
    const Cut cut = cut_of(a, p.s, a.filled, a.shift);
    if (!cut.ok || p.base >= cut.len || cut.keep == 0) return;
    const Head h(a, cut, p.head);
    const int end = min(p.base + kSpan, h.len);
    if (h.keep == h.len) {
        for (int j = p.base + tid; j < end; j += kThreads) h.put(j, j);
        return;
    }
    Each v;
    v.load(h, p.base, tid);
    const int spans = (h.len + kSpan - 1) / kSpan;
    const int32_t* spanned = a.spanned + 4 * p.head * a.spans;
    const uint32_t* keys = a.keys + p.head * a.c.cap;
    Sought x = {(uint32_t)spanned[2], spanned[3], 21, false};
    while (x.low > 0 && !x.all)
        narrow(lds, x, tid, [&](auto f) {
            for (int i = wave; i < spans; i += kWaves)
                for (int n = spanned[4 * i + 1], y = lane; y < n; y += 64) f(keys[(int64_t)i * kSpan + y]);
        });
    // what is above the key ahead of this span, and its equals
    if (tid < 2) s_ahead[tid] = 0;
    __syncthreads();
    for (int i = wave; i < p.part; i += kWaves) {
        int above = 0, same = 0;
        for (int n = spanned[4 * i + 1], y = lane; y < n; y += 64) {
            const uint32_t key = keys[(int64_t)i * kSpan + y] >> x.low, top = x.top >> x.low;
            above += key > top;
            same += key == top;
        }
        above = __builtin_amdgcn_readlane(wave_upto(above), 63) + spanned[4 * i];
        same = __builtin_amdgcn_readlane(wave_upto(same), 63);
        if (lane == 0) {
            atomicAdd(&s_ahead[0], above);
            atomicAdd(&s_ahead[1], same);
        }
    }
    __syncthreads();
    const int equal = s_ahead[1], stay_ahead = s_ahead[0] + min(equal, x.left);
    const Flags f = flags_of(lds, h, v, x, equal, tid);
    uint32_t hole = 0, source = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const bool below = v.at(e) < h.keep;
        hole |= (below ? ~f.stays : 0u) & 1u << e;
        source |= (below ? 0u : f.stays) & 1u << e;
    }
    const Ranks holes(lds, hole, tid);
    __syncthreads();
    const Ranks sources(lds, source, tid);
    // ahead of a span that has holes all positions lie below keep; behind one that has sources
    // all that stays is a source
    const int holes_ahead = p.base - stay_ahead, below = max(min(h.keep, end) - p.base, 0);
    const int behind = h.keep - stay_ahead - (below - holes.all + sources.all);
    int32_t* movers = a.movers + p.head * a.c.cap;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int j = v.at(e);
        if (j < h.keep) h.from[j] = hole >> e & 1u ? holes_ahead + holes.of(hole, e) : -1;
        else if (source >> e & 1u) movers[behind + sources.all - 1 - sources.of(source, e)] = j;
    }
    if (tid == 0 && p.base < h.keep && h.keep <= end) a.holes[p.head] = holes_ahead + holes.all;
}

// ---------------------------------------------------------------------------
// k_evict_move
// ---------------------------------------------------------------------------
// A wave a block of 16 slots below `keep` of a (sequence, KV head): the holes' keys row by
// row, and its values' block made anew from the bytes of the slots that are to lie in it
// (a slot that stays gives its own).  LONG: after k_evict_rank, whose holes and sources are
// joined here, with their weights and tokens.  grid nkv * ceil(max_keep / 64) * n_seqs,
// block 256.
//
// A value's bytes of 16 slots lie together, so a moved slot is a byte in each of hd lines:
// bytes one by one were 160 us for 32 sequences of up to 8192 cut down to 2048 (8 heads of
// 128); whole blocks, each loaded once and picked from by byte permutes, four in flight, 82
// (64 at best).  Up to 17 blocks of 2 KB are read for one that is put out, which is the bound
// there: nearly every block behind `keep` has a slot that stays.
template <bool LONG>
__global__ __launch_bounds__(256) void k_evict_move(PagedEvict a, int blocks)
{
    const Paged& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = (int)(blockIdx.x % (unsigned)c.nkv);
    const unsigned at = blockIdx.x / (unsigned)c.nkv;
    const int block = 4 * (int)(at % (unsigned)blocks) + wave, s = (int)(at / (unsigned)blocks);
    const int hd = c.hd, j0 = 16 * block, r = lane & 15;
    const int64_t head = (int64_t)s * c.nkv + h;
    // asked for beside the sequence's size, not after it: where the slot j0 + r comes from (-1:
    // stays), if it is one that is held, and the page of the block
    const int32_t* table = c.pages + (int64_t)s * c.max_pages;
    int src = -1, in = 0, page = -1;
    if (j0 < c.cap) {
        src = a.from[head * c.cap + min(j0 + r, c.cap - 1)];
        page = page_of(c, table, block, &in);
    }
    // (over the account that came in: what k_evict_count has put by)
    const Cut cut = cut_of(a, s, LONG ? a.was : a.filled, LONG ? a.was + c.n_seqs : a.shift);
    if (h == 0 && block == 0 && lane == 0) {
        a.held[s] = cut.ok ? cut.keep : -1;
        if (cut.ok) {
            const int shift = a.shift[s];
            a.filled_out[s] = cut.keep;
            a.shift_out[s] = (int)((uint32_t)shift + (uint32_t)(cut.len - cut.keep));
        }
    }
    if (!cut.ok || cut.keep == cut.len || j0 >= cut.keep) return;
    if (j0 + r >= cut.keep) src = -1;
    if (LONG) {
        if (src >= 0) src = a.movers[head * c.cap + a.holes[head] - 1 - src];
        if (lane < 16 && j0 + r < cut.keep) Head(a, cut, head).put(j0 + r, src >= 0 ? src : j0 + r);
    }
    if (!__any(src >= 0)) return;
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
    const unsigned heads = (unsigned)(a.c.nkv * a.c.n_seqs);
    const int blocks = evict_blocks(a);
    const dim3 move(heads * blocks);
    if (a.spans > 1) {
        const dim3 spans(heads * a.spans);
        hipLaunchKernelGGL(k_evict_count, spans, dim3(kThreads), 0, st, a);
        hipLaunchKernelGGL(k_evict_collect, spans, dim3(kThreads), 0, st, a);
        hipLaunchKernelGGL(k_evict_rank, spans, dim3(kThreads), 0, st, a);
        hipLaunchKernelGGL(k_evict_move<true>, move, dim3(256), 0, st, a, blocks);
    } else {
        if (a.c.cap > kSpan / 2) hipLaunchKernelGGL(k_evict_choose<kThreads>, dim3(heads), dim3(kThreads), 0, st, a);
        else if (a.spans) hipLaunchKernelGGL(k_evict_choose<kThreads / 2>, dim3(heads), dim3(kThreads / 2), 0, st, a);
        hipLaunchKernelGGL(k_evict_move<false>, move, dim3(256), 0, st, a, blocks);
    }
    return hipGetLastError();
}

}  // namespace btl
