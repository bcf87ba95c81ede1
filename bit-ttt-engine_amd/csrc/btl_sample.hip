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
// says which bin holds the place, and only that bin's tokens are brought together.
//
// Kernels:
//   k_sample_max   per slice of a row the first token in the order; clears the
//                  row's histogram.
//   k_sample_hist  counts and weights of the row's bins: in LDS per slice, then
//                  added to the row's (whole numbers: any order, the same sums).
//   k_sample_pick  per row: the places in turn.
#include <hip/hip_runtime.h>

#include "btl_device.hpp"
#include "btl_serve.hpp"

namespace btl {

namespace {

constexpr int kBins = kSampleBins;
constexpr int kSlice = kSampleSlice;
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
    double top, t;
    float topf, per_bin;
    bool inf;  // the maximum is +inf: those tokens alone, alike
};

__device__ __forceinline__ Weigh weigh_at(uint32_t top_key, float t)
{
    Weigh w;
    w.topf = value_of(top_key);
    w.inf = top_key >= kPlusInf;
    w.top = w.inf ? 0.0 : (double)w.topf;
    w.t = (double)t;
    w.per_bin = fminf(__fdiv_rn((float)kBins / kSpan, t), kMaxF);  // finite: 0 times it is 0
    return w;
}

// the weight of a logit (2^40 for the largest); 0 for -inf and NaN
__device__ __forceinline__ uint64_t weight(const Weigh& w, float l)
{
    if (w.inf) return l == w.topf ? (uint64_t)1 << 40 : 0;
    if (!(l > -__builtin_inff())) return 0;
    const double x = ((double)l - w.top) / w.t;
    // adding 2^52 rounds to a whole number, halves to even, and leaves it in the low bits
    const double y = __dadd_rn(__dmul_rn(exp(x), kOne), 4503599627370496.0);
    return (uint64_t)__double_as_longlong(y) & (((uint64_t)1 << 52) - 1);
}

// its place among the bins: never smaller for a smaller logit (each step keeps the
// order); from kBins on the weight is 0
__device__ __forceinline__ float place_of(const Weigh& w, float l)
{
    return w.inf ? 0.0f : __fmul_rn(fminf(__fsub_rn(w.topf, l), kMaxF), w.per_bin);
}

__device__ __forceinline__ int bin_of(const Weigh& w, float l) { return (int)fminf(place_of(w, l), (float)(kBins - 1)); }

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

// Every logit of [i0, i1) of a row to f(value, index), spread over the workgroup's
// threads, four at a time where the row is 16-byte aligned.
template <int NTHR, typename F>
__device__ __forceinline__ void each(const float* x, int i0, int i1, int tid, F f)
{
    if (((uintptr_t)x & 15u) == 0) {  // i0 is a multiple of 4
        const int n4 = i1 >> 2;
        for (int i = (i0 >> 2) + tid; i < n4; i += NTHR * 4) {
            float4 v[4];
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (i + NTHR * b < n4) v[b] = ((const float4*)x)[i + NTHR * b];
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (i + NTHR * b < n4) {
                    const int at = 4 * (i + NTHR * b);
                    f(v[b].x, at);
                    f(v[b].y, at + 1);
                    f(v[b].z, at + 2);
                    f(v[b].w, at + 3);
                }
        }
        for (int i = max(4 * n4, i0) + tid; i < i1; i += NTHR) f(x[i], i);
    } else {
        for (int i = i0 + tid; i < i1; i += NTHR) f(x[i], i);
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
    each<256>(x, slice * kSlice, min(a.n, (slice + 1) * kSlice), tid,
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

// grid (slices, rows), block 256
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
    each<256>(a.logits + (int64_t)row * a.ld, slice * kSlice, min(a.n, (slice + 1) * kSlice), tid, [&](float v, int) {
        if (place_of(w, v) >= (float)kBins) return;
        const uint64_t m = weight(w, v);
        if (m < f.least) return;
        const int b = bin_of(w, v);
        atomicAdd((unsigned long long*)&s_mass[b], (unsigned long long)m);
        atomicAdd(&s_count[b], 1u);
    });
    __syncthreads();
    for (int b = tid; b < kBins; b += 256)
        if (s_count[b]) {
            __hip_atomic_fetch_add(&a.mass[(int64_t)row * kBins + b], s_mass[b], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_fetch_add(&a.count[(int64_t)row * kBins + b], s_count[b], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
        }
}

namespace {

constexpr int kThr = 512;
constexpr int kList = 2048;  // tokens that are ordered at once
constexpr int kSub = kThr;  // parts that a fuller bin is split into

struct PickLds {
    uint64_t mass[kBins];    // running weight up to and with a bin
    uint32_t count[kBins];   // running count
    uint64_t list[kList];    // words, ordered
    uint64_t cum[kList];     // running weights of the list
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

// Words of the list in order (largest first), then their running weights.
__device__ __forceinline__ void order_list(PickLds& s, int tid, int c, const Weigh& w)
{
    __syncthreads();
    int size = 2;
    while (size < c) size <<= 1;
    for (int i = c + tid; i < size; i += kThr) s.list[i] = 0;  // behind every word
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = tid; i < size / 2; i += kThr) {
                const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                const uint64_t x = s.list[lo], y = s.list[hi];
                if ((x < y) == ((lo & k) == 0)) {
                    s.list[lo] = y;
                    s.list[hi] = x;
                }
            }
            __syncthreads();
        }
    uint64_t carry = 0;
    for (int i0 = 0; i0 < c; i0 += kThr) {
        const int i = i0 + tid;
        uint64_t m = i < c ? weight(w, value_of((uint32_t)(s.list[i] >> 32))) : 0;
        uint32_t one = 0;
        scan_pairs(s, tid, m, one);
        if (i < c) s.cum[i] = carry + m;
        __syncthreads();
        carry = s.cum[min(i0 + kThr, c) - 1];
    }
}

// A place in the order: the word there, the running weight up to and with it.
struct Place {
    uint64_t word, upto;
};

// The first token at which the running count reaches `goal` (by_count) or the
// running weight does.  1 <= goal <= the row's.  `x`, `n`: the row.
__device__ __forceinline__ Place locate(PickLds& s, const SampleArgs& a, const float* x, const Weigh& w, uint64_t least, int tid,
                        bool by_count, uint64_t goal)
{
    // the bin
    if (tid == 0) s.found = 0;
    __syncthreads();
    for (int b = tid; b < kBins; b += kThr) {
        const uint64_t before = by_count ? (b ? s.count[b - 1] : 0) : (b ? s.mass[b - 1] : 0);
        const uint64_t with = by_count ? s.count[b] : s.mass[b];
        if (before < goal && with >= goal) s.found = b;
    }
    __syncthreads();
    const int bin = s.found;
    uint64_t mass0 = bin ? s.mass[bin - 1] : 0;                      // weight ahead of what is looked at
    uint64_t count0 = bin ? s.count[bin - 1] : 0;
    uint32_t held = s.count[bin] - (uint32_t)count0;
    uint64_t lo = 0, hi = ~(uint64_t)0;  // words that are looked at
    if (held > kList) {
        // too many to order: their words' range first
        uint64_t wl = ~(uint64_t)0, wh = 0;
        each<kThr>(x, 0, a.n, tid, [&](float v, int i) {
            if (bin_of(w, v) != bin || weight(w, v) < least) return;
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
        int shift = 0;
        while (((hi - lo) >> shift) >= kSub) ++shift;
        for (int i = tid; i < kSub; i += kThr) {
            s.sub_mass[i] = 0;
            s.sub_count[i] = 0;
        }
        __syncthreads();
        each<kThr>(x, 0, a.n, tid, [&](float v, int i) {
            if (bin_of(w, v) != bin) return;
            const uint64_t o = word_of(key_of(v), (uint32_t)i);
            if (o < lo || o > hi) return;
            const uint64_t m = weight(w, v);
            if (m < least) return;
            const int part = kSub - 1 - (int)((o - lo) >> shift);  // larger words first
            atomicAdd((unsigned long long*)&s.sub_mass[part], (unsigned long long)m);
            atomicAdd(&s.sub_count[part], 1u);
        });
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
        const int part = kSub - 1 - s.found;
        mass0 = s.best[0];
        count0 = s.best[1];
        held = (uint32_t)s.best[2];
        lo += (uint64_t)part << shift;
        hi = min(hi, lo + (((uint64_t)1 << shift) - 1));
        __syncthreads();
    }
    if (tid == 0) s.fill = 0;
    __syncthreads();
    each<kThr>(x, 0, a.n, tid, [&](float v, int i) {
        if (bin_of(w, v) != bin) return;
        const uint64_t o = word_of(key_of(v), (uint32_t)i);
        if (o < lo || o > hi || weight(w, v) < least) return;
        const uint32_t at = atomicAdd(&s.fill, 1u);
        if (at < kList) s.list[at] = o;
    });
    __syncthreads();
    const int c = (int)min(s.fill, (uint32_t)kList);
    order_list(s, tid, c, w);
    __syncthreads();
    for (int i = tid; i < c; i += kThr) {
        const uint64_t before = by_count ? count0 + i : mass0 + (i ? s.cum[i - 1] : 0);
        const uint64_t with = by_count ? count0 + i + 1 : mass0 + s.cum[i];
        if (before < goal && with >= goal) s.found = i;
    }
    __syncthreads();
    const int at = min(s.found, c - 1);
    const Place p = {s.list[at], mass0 + s.cum[at]};
    __syncthreads();
    return p;
}

}  // namespace

// grid rows, block kThr
__global__ __launch_bounds__(kThr) void k_sample_pick(SampleArgs a)
{
    __shared__ PickLds s;
    const int row = blockIdx.x, tid = threadIdx.x;
    const RowFilters f = filters_at(a, row);
    const uint64_t best = row_best<kThr / 64>(a, row, tid, s.best);
    __syncthreads();
    const uint32_t top = (uint32_t)(best >> 32);
    if (top <= kMinusInf || !(f.t > 0.0f)) {
        if (tid == 0) {
            a.ids[row] = top <= kMinusInf ? -1 : (int32_t)~(uint32_t)best;
            if (a.probs) a.probs[row] = top <= kMinusInf ? 0.0f : 1.0f;
        }
        return;
    }
    const Weigh w = weigh_at(top, f.t);
    const float* x = a.logits + (int64_t)row * a.ld;
    uint64_t m0 = 0;
    uint32_t c0 = 0;
    for (int b0 = 0; b0 < kBins; b0 += kThr) {
        uint64_t m = a.mass[(int64_t)row * kBins + b0 + tid];
        uint32_t c = a.count[(int64_t)row * kBins + b0 + tid];
        scan_pairs(s, tid, m, c);
        s.mass[b0 + tid] = m0 + m;
        s.count[b0 + tid] = c0 + c;
        __syncthreads();
        m0 = s.mass[b0 + kThr - 1];
        c0 = s.count[b0 + kThr - 1];
    }
    uint64_t W = m0;  // the weight of what stays
    Place p{};
    // in turn: where top-k cuts, where top-p cuts, the draw
    for (int step = 0; step < 3; ++step) {
        if (step == 0 && !(f.k > 0 && (uint32_t)f.k < c0)) continue;
        if (step == 1 && !(f.p < 1.0)) continue;
        uint64_t goal = (uint64_t)f.k;
        if (step == 1) goal = min(max((uint64_t)__builtin_ceil(__dmul_rn(f.p, (double)W)), (uint64_t)1), W);
        if (step == 2) {
            const double r = __dmul_rn(f.u > 0.0f ? (double)f.u : 0.0, (double)W);
            goal = (r < (double)W ? min((uint64_t)r, W - 1) : W - 1) + 1;
        }
        p = locate(s, a, x, w, f.least, tid, step == 0, goal);
        if (step < 2) W = p.upto;
    }
    if (tid == 0) {
        a.ids[row] = (int32_t)~(uint32_t)p.word;
        if (a.probs) a.probs[row] = (float)__ddiv_rn((double)weight(w, value_of((uint32_t)(p.word >> 32))), (double)W);
    }
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
