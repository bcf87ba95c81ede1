// btl_sample.hip -- gfx950 kernels that choose next tokens from logits: temperature,
// min-p, top-k, top-p, and a given random number (the pick of stream_completion,
// crates/rust_engine/src/model/llama.rs:496-530, with filters).
//
// A token's weight is a whole number, w = rint(2^40 exp((l - max) / T)) with the
// exponential in f64, so every sum of weights is exact in 64 bits (n <= 2^22) and
// any split of the row gives the same token.  Tokens are ordered by one 54-bit
// word, unique in its row: the logit's key (32 bits that order floats), then the
// complement of the index; "larger word" is "comes first".  top-k, top-p and the
// draw each ask for one place in that order, by count or by running weight.  No row
// is sorted: a histogram over bins of (max - l) / T -- in the order's direction --
// says which bin holds the place, and only the tokens of that bin, or of the bins
// up to it where they are few, are brought together and ordered.
//
// Kernels:
//   k_sample_max   per slice of a row the first token in the order; clears the
//                  row's histogram.
//   k_sample_hist  counts and weights of the row's bins: in LDS per slice, then
//                  added to the row's (whole numbers: any order, the same sums).
//   k_sample_pick  per row: the places in turn.
//
// One row of 128256 is latency: 3.1 + 4.9 + 17 us, the last one workgroup that reads
// the row once more (0.5 MB at some 100 GB/s a CU) and meets at some 30 barriers.  64
// rows (33 MB, 5 us at the rate of reading): 8.8 us, 24 (f64 exponentials and two LDS
// atomics a token; 13 where top-k <= 1024 asks for counts only) and 46, the slowest
// row's: a top-p whose cut lies among more than 2048 tokens reads its row twice.  Rows
// of equal or nearly equal logits are the worst: all of 128256 tokens in one bin, so in one
// LDS counter and in several readings of the row by its one workgroup, 0.37 ms without
// filters and 0.65 to 0.84 with top-k or top-p (64 rows: 0.44, and 0.71 to 0.89).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "btl_device.hpp"
#include "btl_serve.hpp"

namespace btl {

namespace {

constexpr int kBins = kSampleBins;
constexpr int kFewK = 1024;
constexpr float kSpan = 28.5f;  // weights are 0 past (max - l) / T = 41 ln 2 = 28.42
constexpr double kOne = 1099511627776.0;  // 2^40
constexpr float kMaxF = 3.40282346638528859812e38f;
constexpr uint32_t kMinusInf = 0x007FFFFFu;  // the key of -inf
constexpr uint32_t kPlusInf = 0xFF800000u;

// floats in order as u32; -0 as +0, NaN as -inf
__device__ __forceinline__ uint32_t key_of(float f)
{
    uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) == 0u) u = 0u;
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) u = 0xFF800000u;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float value_of(uint32_t key)
{
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

__device__ __forceinline__ uint64_t word_of(uint32_t key, uint32_t idx)
{
    return (uint64_t)key << 32 | (uint32_t)~idx;
}

// A row's weights: its maximum and temperature (T > 0).
struct Weigh {
    double top, per_t;
    float topf, per_bin;
    bool inf;  // the maximum is +inf: those tokens alone, alike
};

__device__ __forceinline__ Weigh weigh_at(uint32_t top_key, float t)
{
    Weigh w;
    w.topf = value_of(top_key);
    w.inf = top_key >= kPlusInf;
    w.top = w.inf ? 0.0 : (double)w.topf;
    w.per_t = __ddiv_rn(1.0, (double)t);
    w.per_bin = fminf(__fdiv_rn((float)kBins / kSpan, t), kMaxF);  // finite: 0 times it is 0
    return w;
}

// e^x for -30 < x <= 0 in f64: x = n ln 2 + r with ln 2 in two parts, n * hi exact;
// e^r, |r| <= ln 2 / 2, by its Taylor polynomial to r^13 / 13! (what is left out is
// 4e-18 of it) in Horner form; times 2^n.
__device__ __forceinline__ double exp_f64(double x)
{
    const double n = __builtin_rint(__dmul_rn(x, 1.4426950408889634074));
    const double r = __fma_rn(n, -0x1.ef35793c7673p-45, __fma_rn(n, -0x1.62e42fefa38p-1, x));
    double p = 1.0 / 6227020800.0;
    p = __fma_rn(p, r, 1.0 / 479001600.0);
    p = __fma_rn(p, r, 1.0 / 39916800.0);
    p = __fma_rn(p, r, 1.0 / 3628800.0);
    p = __fma_rn(p, r, 1.0 / 362880.0);
    p = __fma_rn(p, r, 1.0 / 40320.0);
    p = __fma_rn(p, r, 1.0 / 5040.0);
    p = __fma_rn(p, r, 1.0 / 720.0);
    p = __fma_rn(p, r, 1.0 / 120.0);
    p = __fma_rn(p, r, 1.0 / 24.0);
    p = __fma_rn(p, r, 1.0 / 6.0);
    p = __fma_rn(p, r, 0.5);
    p = __fma_rn(p, r, 1.0);
    p = __fma_rn(p, r, 1.0);
    return __builtin_ldexp(p, (int)n);
}

// the weight of a logit (2^40 for the largest); 0 for -inf and NaN
__device__ __forceinline__ uint64_t weight(const Weigh& w, float l)
{
    if (w.inf) return l == w.topf ? (uint64_t)1 << 40 : 0;
    const double x = __dmul_rn((double)l - w.top, w.per_t);
    if (!(x > -30.0)) return 0;
    // adding 2^52 rounds to a whole number, halves to even, and leaves it in the low bits
    const double y = __dadd_rn(__dmul_rn(exp_f64(x), kOne), 4503599627370496.0);
    return (uint64_t)__double_as_longlong(y) & (((uint64_t)1 << 52) - 1);
}

// its place among the bins: never smaller for a smaller logit (each step keeps the
// order); from kBins on the weight is 0
__device__ __forceinline__ float place_of(const Weigh& w, float l)
{
    if (w.inf) return l == w.topf ? 0.0f : (float)kBins;
    return __fmul_rn(fminf(__fsub_rn(w.topf, l), kMaxF), w.per_bin);
}

struct RowFilters {
    float t;
    int k;
    double p;
    uint64_t least;  // smallest weight that stays
    float u;
};

__device__ __forceinline__ RowFilters filters_at(const SampleArgs& a, int row)
{
    RowFilters f;
    f.t = a.temperature ? a.temperature[row] : 1.0f;
    f.k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, m = a.min_p ? a.min_p[row] : 0.0f;
    f.p = p < 1.0f ? (p > 0.0f ? (double)p : 0.0) : 1.0;
    // w >= min_p * 2^40 for whole w (2^40 times an f32 is exact); never more than the first token's
    f.least = m > 0.0f ? (uint64_t)__builtin_ceil((double)(m < 1.0f ? m : 1.0f) * kOne) : 1;
    if (f.least < 1) f.least = 1;
    f.u = a.u[row];
    return f;
}

// Whether the bins' weights are asked for: where top-k leaves few tokens they are all
// brought together, and only counted before.
__device__ __forceinline__ bool weighed(const RowFilters& f) { return !(f.k > 0 && f.k <= kFewK); }

// Every logit of [i0, i1) of a row to f(value, index), spread over the workgroup's
// threads, U loads ahead; four logits a load where the row is 16-byte aligned (i0 is
// a multiple of 4).
template <int NTHR, int U, typename F>
__device__ __forceinline__ void each(const float* x, int i0, int i1, int tid, F f)
{
    if (((uintptr_t)x & 15u) == 0) {
        const int n4 = i1 >> 2;
        for (int i = (i0 >> 2) + tid; i < n4; i += NTHR * U) {
            float4 v[U];
#pragma unroll
            for (int b = 0; b < U; ++b) v[b] = ((const float4*)x)[min(i + NTHR * b, n4 - 1)];
#pragma unroll
            for (int b = 0; b < U; ++b)
                if (i + NTHR * b < n4) {
                    const int at = 4 * (i + NTHR * b);
                    f(v[b].x, at);
                    f(v[b].y, at + 1);
                    f(v[b].z, at + 2);
                    f(v[b].w, at + 3);
                }
        }
        const int i = max(4 * n4, i0) + tid;
        if (i < i1) f(x[i], i);
    } else {
        for (int i = i0 + tid; i < i1; i += NTHR * U) {
            float v[U];
#pragma unroll
            for (int b = 0; b < U; ++b) v[b] = x[min(i + NTHR * b, i1 - 1)];
#pragma unroll
            for (int b = 0; b < U; ++b)
                if (i + NTHR * b < i1) f(v[b], i + NTHR * b);
        }
    }
}

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int off)
{
    const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)v, off, 64);
    const uint32_t hi = (uint32_t)__shfl_up((int)(uint32_t)(v >> 32), off, 64);
    return (uint64_t)hi << 32 | lo;
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int off)
{
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, off, 64);
    const uint32_t hi = (uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), off, 64);
    return (uint64_t)hi << 32 | lo;
}

__device__ __forceinline__ uint64_t wave_max64(uint64_t v)
{
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = max(v, shfl_xor64(v, off));
    return v;
}

}  // namespace

// grid (slices, rows), block 256
__global__ __launch_bounds__(256) void k_sample_max(SampleArgs a)
{
    __shared__ uint64_t s_best[4];
    const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    const float* x = a.logits + (int64_t)row * a.ld;
    uint64_t best = 0;
    each<256, 4>(x, slice * a.slice, min(a.n, (slice + 1) * a.slice), tid,
                 [&](float v, int i) { best = max(best, word_of(key_of(v), (uint32_t)i)); });
    best = wave_max64(best);
    if ((tid & 63) == 0) s_best[tid >> 6] = best;
    for (int b = slice * 256 + tid; b < kBins; b += a.slices * 256) {
        a.mass[(int64_t)row * kBins + b] = 0;
        a.count[(int64_t)row * kBins + b] = 0;
    }
    __syncthreads();
    if (tid == 0)
        a.best[(int64_t)row * a.slices + slice] = max(max(s_best[0], s_best[1]), max(s_best[2], s_best[3]));
}

// the row's first token, by every thread of a workgroup of NW waves
template <int NW>
__device__ __forceinline__ uint64_t row_best(const SampleArgs& a, int row, int tid, uint64_t* s_best)
{
    uint64_t best = 0;
    for (int i = tid; i < a.slices; i += 64 * NW) best = max(best, a.best[(int64_t)row * a.slices + i]);
    best = wave_max64(best);
    if ((tid & 63) == 0) s_best[tid >> 6] = best;
    __syncthreads();
    best = s_best[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) best = max(best, s_best[w]);
    return best;
}

// grid (slices, rows), block 256.  Every token up to the last bin is counted; its
// weight goes in where min-p keeps it.
__global__ __launch_bounds__(256) void k_sample_hist(SampleArgs a)
{
    __shared__ uint64_t s_best[4];
    __shared__ uint64_t s_mass[kBins];
    __shared__ uint32_t s_count[kBins];
    const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    const RowFilters f = filters_at(a, row);
    if (!(f.t > 0.0f)) return;
    for (int b = tid; b < kBins; b += 256) {
        s_mass[b] = 0;
        s_count[b] = 0;
    }
    const uint32_t top = (uint32_t)(row_best<4>(a, row, tid, s_best) >> 32);  // holds a barrier
    if (top <= kMinusInf) return;
    const Weigh w = weigh_at(top, f.t);
    const bool weigh = weighed(f);
    each<256, 1>(a.logits + (int64_t)row * a.ld, slice * a.slice, min(a.n, (slice + 1) * a.slice), tid,
                 [&](float v, int) {
                     const float p = place_of(w, v);
                     if (p >= (float)kBins || v != v) return;
                     atomicAdd(&s_count[(int)p], 1u);
                     if (!weigh) return;
                     const uint64_t m = weight(w, v);
                     if (m >= f.least) atomicAdd((unsigned long long*)&s_mass[(int)p], (unsigned long long)m);
                 });
    __syncthreads();
    for (int b = tid; b < kBins; b += 256)
        if (s_count[b]) {
            if (s_mass[b])
                __hip_atomic_fetch_add(&a.mass[(int64_t)row * kBins + b], s_mass[b], __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_fetch_add(&a.count[(int64_t)row * kBins + b], s_count[b], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
        }
}

namespace {

constexpr int kThr = 512;
constexpr int kU = 16;       // loads ahead over a whole row
constexpr int kList = 2048;  // tokens that are brought together at once
constexpr int kOrdered = 256;  // of them, that are sorted; more are narrowed down first
constexpr int kSub = kThr;   // parts that a fuller bin is split into
static_assert(kOrdered <= kThr, "a token a thread");

struct PickLds {
    uint64_t mass[kBins];    // running weight up to and with a bin
    uint32_t count[kBins];   // running count
    uint64_t list[kList];    // words
    uint64_t part[64];       // those that a search is down to
    uint64_t cum[kOrdered];  // running weights of the ordered list
    uint64_t sub_mass[kSub];
    uint32_t sub_count[kSub];
    uint64_t scan[kThr / 64];
    uint32_t scan_c[kThr / 64];
    uint64_t best[kThr / 64];
    uint32_t fill;
    int found;
};

// running sums of one (weight, count) a thread over the workgroup
__device__ __forceinline__ void scan_pairs(PickLds& s, int tid, uint64_t& m, uint32_t& c)
{
    const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint64_t om = shfl_up64(m, off);
        const uint32_t oc = (uint32_t)__shfl_up((int)c, off, 64);
        if (lane >= off) {
            m += om;
            c += oc;
        }
    }
    __syncthreads();  // the last use of the scratch is over
    if (lane == 63) {
        s.scan[wave] = m;
        s.scan_c[wave] = c;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        m += s.scan[w];
        c += s.scan_c[w];
    }
}

// the bins' weights and counts into running ones, two bins a thread
__device__ __forceinline__ void run_bins(PickLds& s, int tid)
{
    static_assert(kBins == 2 * kThr, "two bins a thread");
    __syncthreads();
    const uint64_t m1 = s.mass[2 * tid + 1];
    const uint32_t c1 = s.count[2 * tid + 1];
    uint64_t m = s.mass[2 * tid] + m1;
    uint32_t c = s.count[2 * tid] + c1;
    scan_pairs(s, tid, m, c);  // holds barriers
    s.mass[2 * tid] = m - m1;
    s.mass[2 * tid + 1] = m;
    s.count[2 * tid] = c - c1;
    s.count[2 * tid + 1] = c;
    __syncthreads();
}

// The row, and what is asked of it.
struct Row {
    const float* x;
    int n;
    Weigh w;
    uint64_t least;
};

__device__ __forceinline__ uint64_t kept(const Row& r, uint64_t word)
{
    const uint64_t m = weight(r.w, value_of((uint32_t)(word >> 32)));
    return m >= r.least ? m : 0;
}

// The smallest logit whose place is before p (place_of falls as the logit rises, so
// bins are intervals of logits): 32 halvings over the ordered keys.
__device__ __forceinline__ float first_before(const Weigh& w, float p)
{
    uint32_t lo = kMinusInf, hi = kPlusInf;  // place_of(value_of(hi)) < p <= place_of(value_of(lo)), or lo is it
    if (place_of(w, value_of(lo)) < p) return value_of(lo);
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (place_of(w, value_of(mid)) < p) hi = mid;
        else lo = mid;
    }
    return value_of(hi);
}

// Every token of bins b0 .. b1 to f(value, index).  The loads run kU ahead and leave
// a bit a token; f's code is there once, behind them (unrolled with the loads it was
// fetched slower than it ran).  Two comparisons a token: one workgroup reads the
// whole row, and three rounded operations a token were more than its loads.
template <typename F>
__device__ __forceinline__ void each_in(const Row& r, int tid, int b0, int b1, F f)
{
    const float v0 = first_before(r.w, (float)(b1 + 1));
    const float v1 = b0 > 0 ? first_before(r.w, (float)b0) : __builtin_inff();
    const bool any = b0 <= 0;  // no upper end
    auto in = [&](float v) { return v >= v0 && (any || v < v1); };
    const bool wide = ((uintptr_t)r.x & 15u) == 0;
    const int per = wide ? 4 : 1;
    const int m = wide ? r.n >> 2 : r.n;  // loads
    for (int i0 = tid; i0 < m; i0 += kThr * kU) {
        uint64_t hit = 0;
        if (wide) {
            float4 v[kU];
#pragma unroll
            for (int b = 0; b < kU; ++b) v[b] = ((const float4*)r.x)[min(i0 + kThr * b, m - 1)];
#pragma unroll
            for (int b = 0; b < kU; ++b) {
                const float most = fmaxf(fmaxf(v[b].x, v[b].y), fmaxf(v[b].z, v[b].w));
                if (!__any(most >= v0)) continue;
                const uint32_t bits = (in(v[b].x) ? 1u : 0u) | (in(v[b].y) ? 2u : 0u) | (in(v[b].z) ? 4u : 0u) |
                                      (in(v[b].w) ? 8u : 0u);
                hit |= (uint64_t)(i0 + kThr * b < m ? bits : 0u) << (4 * b);
            }
        } else {
            float v[kU];
#pragma unroll
            for (int b = 0; b < kU; ++b) v[b] = r.x[min(i0 + kThr * b, m - 1)];
#pragma unroll
            for (int b = 0; b < kU; ++b) hit |= (uint64_t)(i0 + kThr * b < m && in(v[b]) ? 1u : 0u) << b;
        }
        while (hit) {
            const int bit = __ffsll((unsigned long long)hit) - 1;
            hit &= hit - 1;
            const int i = wide ? 4 * (i0 + kThr * (bit >> 2)) + (bit & 3) : i0 + kThr * bit;
            f(r.x[i], i);
        }
    }
    const int i = per * m + tid;
    if (i < r.n && in(r.x[i])) f(r.x[i], i);
}

// The words of bins b0 .. b1 from lo to hi into the list, in any order; returns how
// many (at most kList of them are there).
__device__ __forceinline__ int gather(PickLds& s, const Row& r, int tid, int b0, int b1, uint64_t lo, uint64_t hi)
{
    __syncthreads();
    if (tid == 0) s.fill = 0;
    __syncthreads();
    each_in(r, tid, b0, b1, [&](float v, int i) {
        const uint64_t o = word_of(key_of(v), (uint32_t)i);
        if (o < lo || o > hi) return;
        const uint32_t at = atomicAdd(&s.fill, 1u);
        if (at < kList) s.list[at] = o;
    });
    __syncthreads();
    return (int)min(s.fill, (uint32_t)kList);
}

// The list's c <= kOrdered words in order, with their running weights.
__device__ __forceinline__ void order_list(PickLds& s, const Row& r, int tid, int c)
{
    __syncthreads();
    if (c <= 64) {
        // one wave, in registers
        if (tid < 64) {
            uint64_t v = tid < c ? s.list[tid] : 0;  // 0: behind every word
#pragma unroll
            for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
                for (int j = k >> 1; j > 0; j >>= 1) {
                    const uint64_t o = shfl_xor64(v, j);
                    v = ((tid & k) == 0) == ((tid & j) == 0) ? max(v, o) : min(v, o);
                }
            if (tid < c) s.list[tid] = v;
        }
        __syncthreads();
    } else {
        int size = 128;
        while (size < c) size <<= 1;
        for (int i = c + tid; i < size; i += kThr) s.list[i] = 0;
        __syncthreads();
        for (int k = 2; k <= size; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int i = tid; i < size / 2; i += kThr) {
                    const int at = 2 * i - (i & (j - 1));
                    const uint64_t x = s.list[at], y = s.list[at + j];
                    if ((x < y) == ((at & k) == 0)) {
                        s.list[at] = y;
                        s.list[at + j] = x;
                    }
                }
                __syncthreads();
            }
    }
    uint64_t m = tid < c ? kept(r, s.list[tid]) : 0;
    uint32_t one = 0;
    scan_pairs(s, tid, m, one);
    if (tid < c) s.cum[tid] = m;
    __syncthreads();
}

// The bin at which the running count reaches `goal` (by_count) or the running weight does.
__device__ __forceinline__ int bin_at(PickLds& s, int tid, bool by_count, uint64_t goal)
{
    __syncthreads();
    if (tid == 0) s.found = 0;
    __syncthreads();
    for (int b = tid; b < kBins; b += kThr) {
        const uint64_t before = by_count ? (b ? s.count[b - 1] : 0) : (b ? s.mass[b - 1] : 0);
        const uint64_t with = by_count ? s.count[b] : s.mass[b];
        if (before < goal && with >= goal) s.found = b;
    }
    __syncthreads();
    return s.found;
}

// The token of the list at which the running count, mass0 and count0 ahead of it,
// reaches `goal`, or the running weight does.
__device__ __forceinline__ int list_at(PickLds& s, int tid, int c, uint64_t mass0, uint64_t count0, bool by_count,
                                       uint64_t goal)
{
    __syncthreads();
    if (tid == 0) s.found = c - 1;
    __syncthreads();
    for (int i = tid; i < c; i += kThr) {
        const uint64_t before = by_count ? count0 + i : mass0 + (i ? s.cum[i - 1] : 0);
        const uint64_t with = by_count ? count0 + i + 1 : mass0 + s.cum[i];
        if (before < goal && with >= goal) s.found = i;
    }
    __syncthreads();
    return s.found;
}

// A place in the order: the word there, the running weight up to and with it.
struct Place {
    uint64_t word, upto;
};

// kSub parts of the words lo .. hi, larger words first: cleared, a word counted and
// weighed, and on with the part that holds the place.
__device__ __forceinline__ int clear_parts(PickLds& s, int tid, uint64_t lo, uint64_t hi)
{
    int shift = 0;
    while (((hi - lo) >> shift) >= kSub) ++shift;
    __syncthreads();
    s.sub_mass[tid] = 0;
    s.sub_count[tid] = 0;
    if (tid == 0) {
        // no part holds the place: nothing is left to look at, and the search ends
        s.best[2] = 0;
        s.found = 0;
    }
    __syncthreads();
    return shift;
}

__device__ __forceinline__ void to_part(PickLds& s, const Row& r, uint64_t o, uint64_t lo, int shift)
{
    const int part = kSub - 1 - (int)((o - lo) >> shift);
    atomicAdd((unsigned long long*)&s.sub_mass[part], (unsigned long long)kept(r, o));
    atomicAdd(&s.sub_count[part], 1u);
}

__device__ __forceinline__ uint32_t take_part(PickLds& s, int tid, bool by_count, uint64_t goal, int shift, uint64_t& lo,
                                              uint64_t& hi, uint64_t& mass0, uint64_t& count0)
{
    __syncthreads();
    uint64_t m = s.sub_mass[tid];
    uint32_t c = s.sub_count[tid];
    const uint64_t m1 = m;
    const uint32_t c1 = c;
    scan_pairs(s, tid, m, c);
    const uint64_t before = by_count ? count0 + c - c1 : mass0 + m - m1, with = by_count ? count0 + c : mass0 + m;
    if (c1 && before < goal && with >= goal) {
        s.found = tid;
        s.best[0] = mass0 + m - m1;
        s.best[1] = count0 + c - c1;
        s.best[2] = c1;
    }
    __syncthreads();
    mass0 = s.best[0];
    count0 = s.best[1];
    const uint32_t held = (uint32_t)s.best[2];
    lo += (uint64_t)(kSub - 1 - s.found) << shift;
    hi = min(hi, lo + (((uint64_t)1 << shift) - 1));
    __syncthreads();
    return held;
}

// The place among the list's c words (kept as they are): narrowed down part by part
// to one wave's.
__device__ __forceinline__ Place search_list(PickLds& s, const Row& r, int tid, int c, uint64_t mass0, uint64_t count0,
                                             bool by_count, uint64_t goal)
{
    uint64_t wl = ~(uint64_t)0, wh = 0;
    for (int i = tid; i < c; i += kThr) {
        wl = min(wl, s.list[i]);
        wh = max(wh, s.list[i]);
    }
    wl = ~wave_max64(~wl);
    wh = wave_max64(wh);
    __syncthreads();
    if ((tid & 63) == 0) {
        s.best[tid >> 6] = wh;
        s.scan[tid >> 6] = wl;
    }
    __syncthreads();
    uint64_t lo = s.scan[0], hi = s.best[0];
    for (int i = 1; i < kThr / 64; ++i) {
        lo = min(lo, s.scan[i]);
        hi = max(hi, s.best[i]);
    }
    uint32_t held = (uint32_t)c;
    while (held > 64) {
        const int shift = clear_parts(s, tid, lo, hi);
        for (int i = tid; i < c; i += kThr) {
            const uint64_t o = s.list[i];
            if (o >= lo && o <= hi) to_part(s, r, o, lo, shift);
        }
        held = take_part(s, tid, by_count, goal, shift, lo, hi, mass0, count0);
    }
    if (tid == 0) {
        s.fill = 0;
        s.best[0] = s.list[0];
        s.best[1] = mass0;
    }
    __syncthreads();
    for (int i = tid; i < c; i += kThr) {
        const uint64_t o = s.list[i];
        if (o >= lo && o <= hi) s.part[atomicAdd(&s.fill, 1u) & 63] = o;
    }
    __syncthreads();
    if (tid < 64) {
        uint64_t v = (uint32_t)tid < held ? s.part[tid] : 0;
#pragma unroll
        for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
            for (int j = k >> 1; j > 0; j >>= 1) {
                const uint64_t o = shfl_xor64(v, j);
                v = ((tid & k) == 0) == ((tid & j) == 0) ? max(v, o) : min(v, o);
            }
        const uint64_t m1 = (uint32_t)tid < held ? kept(r, v) : 0;
        uint64_t m = m1;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint64_t o = shfl_up64(m, off);
            m += tid >= off ? o : 0;
        }
        const uint64_t before = by_count ? count0 + tid : mass0 + m - m1, with = by_count ? count0 + tid + 1 : mass0 + m;
        if ((uint32_t)tid < held && before < goal && with >= goal) {
            s.best[0] = v;
            s.best[1] = mass0 + m;
        }
    }
    __syncthreads();
    const Place p = {s.best[0], s.best[1]};
    __syncthreads();
    return p;
}

// The first token at which the running count reaches `goal` (by_count) or the
// running weight does.  1 <= goal <= the row's.
__device__ __forceinline__ Place locate(PickLds& s, const Row& r, int tid, bool by_count, uint64_t goal)
{
    const int bin = bin_at(s, tid, by_count, goal);
    uint64_t mass0 = bin ? s.mass[bin - 1] : 0;  // weight ahead of what is looked at
    uint64_t count0 = bin ? s.count[bin - 1] : 0;
    uint32_t held = s.count[bin] - (uint32_t)count0;
    uint64_t lo = 0, hi = ~(uint64_t)0;  // words that are looked at
    if (held > kList) {
        // too many to order: their words' range first
        uint64_t wl = ~(uint64_t)0, wh = 0;
        each_in(r, tid, bin, bin, [&](float v, int i) {
            const uint64_t o = word_of(key_of(v), (uint32_t)i);
            wl = min(wl, o);
            wh = max(wh, o);
        });
        wl = ~wave_max64(~wl);
        wh = wave_max64(wh);
        if ((tid & 63) == 0) {
            s.best[tid >> 6] = wh;
            s.scan[tid >> 6] = wl;
        }
        __syncthreads();
        lo = s.scan[0];
        hi = s.best[0];
        for (int i = 1; i < kThr / 64; ++i) {
            lo = min(lo, s.scan[i]);
            hi = max(hi, s.best[i]);
        }
        __syncthreads();
    }
    while (held > kList) {
        // kSub parts of the range, counted and weighed, and on with the one that holds the place
        const int shift = clear_parts(s, tid, lo, hi);
        each_in(r, tid, bin, bin, [&](float v, int i) {
            const uint64_t o = word_of(key_of(v), (uint32_t)i);
            if (o >= lo && o <= hi) to_part(s, r, o, lo, shift);
        });
        held = take_part(s, tid, by_count, goal, shift, lo, hi, mass0, count0);
    }
    const int c = gather(s, r, tid, bin, bin, lo, hi);
    if (c > kOrdered) return search_list(s, r, tid, c, mass0, count0, by_count, goal);
    order_list(s, r, tid, c);
    const int at = list_at(s, tid, c, mass0, count0, by_count, goal);
    const Place p = {s.list[at], mass0 + s.cum[at]};
    __syncthreads();
    return p;
}

// top-p's running weight
__device__ __forceinline__ uint64_t goal_of(double p, uint64_t W)
{
    return min(max((uint64_t)__builtin_ceil(__dmul_rn(p, (double)W)), (uint64_t)1), W);
}

// the draw's
__device__ __forceinline__ uint64_t draw_of(float u, uint64_t W)
{
    const double r = __dmul_rn(u > 0.0f ? (double)u : 0.0, (double)W);
    return (r < (double)W ? min((uint64_t)r, W - 1) : W - 1) + 1;
}

}  // namespace

// grid rows, block kThr
__global__ __launch_bounds__(kThr) void k_sample_pick(SampleArgs a)
{
    __shared__ PickLds s;
    const int row = blockIdx.x, tid = threadIdx.x;
    const RowFilters f = filters_at(a, row);
    const uint64_t best = row_best<kThr / 64>(a, row, tid, s.best);
    const uint32_t top = (uint32_t)(best >> 32);
    if (top <= kMinusInf || !(f.t > 0.0f)) {
        if (tid == 0) {
            a.ids[row] = top <= kMinusInf ? -1 : (int32_t)~(uint32_t)best;
            if (a.probs) a.probs[row] = top <= kMinusInf ? 0.0f : 1.0f;
        }
        return;
    }
    const Row r = {a.logits + (int64_t)row * a.ld, a.n, weigh_at(top, f.t), f.least};
    for (int b = tid; b < kBins; b += kThr) {
        s.mass[b] = a.mass[(int64_t)row * kBins + b];
        s.count[b] = a.count[(int64_t)row * kBins + b];
    }
    run_bins(s, tid);
    const uint32_t c0 = s.count[kBins - 1];
    const uint64_t m0 = s.mass[kBins - 1];
    const bool by_k = f.k > 0 && (uint32_t)f.k < c0, by_p = f.p < 1.0;
    const bool few = !weighed(f);
    uint64_t W = m0;  // the weight of what stays
    Place p{};
    int last = kBins;  // the bin that the first filter cuts in
    if (by_k) last = bin_at(s, tid, true, (uint64_t)f.k);
    else if (few) last = kBins - 1;
    else if (by_p) last = bin_at(s, tid, false, goal_of(f.p, W));
    if (last < kBins && s.count[last] <= kList) {
        // the tokens up to there in one list: every place is in it
        const int c = gather(s, r, tid, 0, last, 0, ~(uint64_t)0);
        const bool ordered = c <= kOrdered;
        if (ordered) order_list(s, r, tid, c);
        auto place = [&](bool by_count, uint64_t goal) {
            if (!ordered) return search_list(s, r, tid, c, 0, 0, by_count, goal);
            const int at = list_at(s, tid, c, 0, 0, by_count, goal);
            return Place{s.list[at], s.cum[at]};
        };
        for (int step = 0; step < 3; ++step) {  // where top-k cuts (or all of them), where top-p cuts, the draw
            if ((step == 0 && !by_k && !few) || (step == 1 && !by_p)) continue;
            p = place(step == 0, step == 0 ? (uint64_t)(by_k ? f.k : c) : (step == 1 ? goal_of(f.p, W) : draw_of(f.u, W)));
            if (step < 2) W = p.upto;
        }
    } else {
        if (few) {
            // few are asked for, but the bin that top-k cuts in is full of tokens: its weights after all
            __syncthreads();
            for (int b = tid; b < kBins; b += kThr) s.mass[b] = 0;
            __syncthreads();
            each_in(r, tid, 0, kBins - 1, [&](float v, int) {
                const uint64_t m = weight(r.w, v);
                if (m >= r.least) atomicAdd((unsigned long long*)&s.mass[(int)place_of(r.w, v)], (unsigned long long)m);
            });
            __syncthreads();
            for (int b = tid; b < kBins; b += kThr) s.count[b] = a.count[(int64_t)row * kBins + b];
            run_bins(s, tid);
            W = s.mass[kBins - 1];
        }
        // in turn: where top-k cuts, where top-p cuts, the draw
        for (int step = 0; step < 3; ++step) {
            if ((step == 0 && !by_k) || (step == 1 && !by_p)) continue;
            const uint64_t goal = step == 0 ? (uint64_t)f.k : (step == 1 ? goal_of(f.p, W) : draw_of(f.u, W));
            p = locate(s, r, tid, step == 0, goal);
            if (step < 2) W = p.upto;
        }
    }
    if (tid == 0) {
        a.ids[row] = (int32_t)~(uint32_t)p.word;
        if (a.probs) a.probs[row] = (float)__ddiv_rn((double)kept(r, p.word), (double)W);
    }
}

// logits of one workgroup of the first two launches: some 512 workgroups, so that few
// rows spread over the chip and many rows add few histograms together
int sample_slice(int64_t rows, int64_t n)
{
    int slice = 2048;
    while (slice < 32768 && rows * n > (int64_t)512 * slice) slice *= 2;
    return slice;
}

hipError_t launch_sample(const SampleArgs& a, hipStream_t st)
{
    const dim3 grid((unsigned)a.slices, (unsigned)a.rows);
    hipLaunchKernelGGL(k_sample_max, grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_sample_hist, grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_sample_pick, dim3((unsigned)a.rows), dim3(kThr), 0, st, a);
    return hipGetLastError();
}

}  // namespace btl
