// btl_serve.hip -- gfx950 kernels of a batch of sequences over a paged Q8 cache:
// RoPE and append, reading back, attention.
//
// Kernels:
//   k_paged_append   RoPE of the new q and k rows, Q8 of k and v into their slots.
//   k_paged_read     rows of the cache dequantised.
//   k_paged_attn     attention of a tile of rows over a chunk of keys.
//   k_paged_merge    the chunks of a row merged.
//
// The sequences' sizes, positions and pages are read on the device, so a captured
// launch follows them; whatever they hold, every address stays inside the arrays
// (rows are clamped to `rows`, page ids checked, slots clamped to the last visible
// one).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "btl_device.hpp"
#include "btl_serve.hpp"

namespace btl {

namespace {

// One sequence of the batch: its first row, rows and first position; `ok` unless
// it breaks a bound of the call.
struct Seq {
    int a, n, p0;
    bool ok;
};

__device__ __forceinline__ Seq seq_at(const Paged& c, int s)
{
    Seq q;
    q.a = min(max(c.row_start[s], 0), c.rows);
    q.n = min(max(c.row_start[s + 1], q.a), c.rows) - q.a;
    q.p0 = c.pos[s];
    q.ok = q.p0 >= 0 && q.n <= c.max_rows && (int64_t)q.p0 + q.n <= c.cap;
    return q;
}

// The last sequence that starts at or before `row` (uniform over the wave), -1: none.
// 64 starts at a time are looked at, so up to 63 sequences cost one load and 4095 two.
__device__ __forceinline__ int find_seq(const Paged& c, int row, int lane)
{
    int lo = 0, count = c.n_seqs + 1;
    for (bool first = true;; first = false) {
        const int step = (count + 63) / 64;
        const bool in = lane * step < count;
        const int v = in ? c.row_start[lo + lane * step] : INT_MAX;
        const uint64_t le = __ballot(in && v <= row);
        if (!le) return first ? -1 : lo;
        const int top = 63 - __clzll(le);
        lo += top * step;
        count = min(step, count - top * step);
        if (step == 1) return lo;
    }
}

// The sequence that piece `at` of a launch belongs to (-1: none) and the piece's number
// in it, where sequence s has count(s) of them; 64 sequences are counted at a time.
template <typename F>
__device__ __forceinline__ int find_piece(const Paged& c, int lane, int& at, F count)
{
    if (c.n_seqs == 1) return at < count(0) ? 0 : -1;
    for (int base = 0; base < c.n_seqs; base += 64) {
        const int mine = base + lane < c.n_seqs ? count(base + lane) : 0;
        int upto = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(upto, off, 64);
            upto += lane >= off ? o : 0;
        }
        const uint64_t past = __ballot(upto > at);
        if (past) {
            const int hit = __ffsll((unsigned long long)past) - 1;
            at = __builtin_amdgcn_readfirstlane(at - __builtin_amdgcn_readlane(upto - mine, hit));
            return base + hit;
        }
        at -= __builtin_amdgcn_readlane(upto, 63);
    }
    return -1;
}

// page id of a group of 16 positions (-1: none in the pool) and the group's place in the page
__device__ __forceinline__ int page_of(const Paged& c, const int32_t* table, int grp, int* in_page)
{
    const int j = (int)__umulhi(2u * (uint32_t)grp, c.ppg_mul);  // grp / ppg
    *in_page = grp - j * c.ppg;
    const int id = table[j];
    return id >= 0 && id < c.n_pages ? id : -1;
}

template <bool BF>
__device__ __forceinline__ float load1(const void* p, int64_t i)
{
    return BF ? bf16_to_f32(((const uint16_t*)p)[i]) : ((const float*)p)[i];
}

template <bool BF>
__device__ __forceinline__ void store1(void* p, int64_t i, float v)
{
    store_y<BF ? YK_BF16 : YK_F32>(p, i, v);
}

// Rust `f32 as u8`: saturating, NaN -> 0
__device__ __forceinline__ uint8_t to_u8(float r)
{
    if (!(r > 0.0f)) return 0;
    return (uint8_t)(r >= 255.0f ? 255u : (uint32_t)r);
}

}  // namespace

// ---------------------------------------------------------------------------
// k_paged_append
// ---------------------------------------------------------------------------
// grid (rows, ceil((nh + 2 nkv) / (4 N))), block 256, N slots a wave: q heads, then k
// heads, then v heads, each as k_rope_kv_q8 does it (lane i holds the pair
// (i, i + hd / 2) that RoPE turns together).  A wave waits for four loads in a row
// (sequence, position, table and page, store), so with many rows it takes N slots
// together, their loads issued first.
template <bool BF, int N>
__global__ __launch_bounds__(256) void k_paged_append(PagedAppend a)
{
    const int t = blockIdx.x, lane = threadIdx.x & 63;
    const int first = N * (4 * blockIdx.y + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    const int nkv = a.c.nkv, slots = a.nh + 2 * nkv;
    if (first >= slots) return;
    const int hd = a.c.hd, half = hd >> 1;
    const bool act = lane < half;
    // slot -> kind (0 q, 1 k, 2 v) and head
    auto kind_of = [&](int slot) { return slot < a.nh ? 0 : (slot < a.nh + nkv ? 1 : 2); };
    auto head_of = [&](int slot) { return slot < a.nh ? slot : (slot < a.nh + nkv ? slot - a.nh : slot - a.nh - nkv); };
    float x1[N], x2[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int slot = min(first + e, slots - 1), kind = kind_of(slot);
        const void* src = kind == 0 ? a.q : (kind == 1 ? a.k : a.v);
        const int64_t row = ((int64_t)t * (kind == 0 ? a.nh : nkv) + head_of(slot)) * hd;
        x1[e] = act ? load1<BF>(src, row + lane) : 0.0f;
        x2[e] = act ? load1<BF>(src, row + lane + half) : 0.0f;
    }
    const int s = find_seq(a.c, t, lane);
    if (s < 0 || s >= a.c.n_seqs) return;
    const Seq q = seq_at(a.c, s);
    const int i = t - q.a;
    if (i < 0 || i >= q.n) return;
    const int pos = q.p0 + i;
    const bool good = q.ok && pos < a.rope_len;
    int grp = 0, page = -1;
    float c = 0.0f, w = 0.0f;
    if (good) {
        page = page_of(a.c, a.c.pages + (int64_t)s * a.c.max_pages, pos >> 4, &grp);
        if (act) {
            c = a.cos_t[(int64_t)pos * half + lane];
            w = a.sin_t[(int64_t)pos * half + lane];
        }
    }
    const int in = pos & 15;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int slot = first + e, kind = kind_of(slot), head = head_of(slot);
        if (slot >= slots) return;
        float y1 = x1[e], y2 = x2[e];
        if (kind < 2) {
            y1 = __fsub_rn(__fmul_rn(x1[e], c), __fmul_rn(x2[e], w));
            y2 = __fadd_rn(__fmul_rn(x1[e], w), __fmul_rn(x2[e], c));
        }
        if (kind == 0) {
            const int64_t row = ((int64_t)t * a.nh + head) * hd;
            if (act) {
                store1<BF>(a.q_out, row + lane, good ? y1 : __builtin_nanf(""));
                store1<BF>(a.q_out, row + lane + half, good ? y2 : __builtin_nanf(""));
            }
            continue;
        }
        if (page < 0) continue;
        const uint32_t am = wave_max_dpp(max(__float_as_uint(y1) & 0x7FFFFFFFu, __float_as_uint(y2) & 0x7FFFFFFFu));
        const float sc = __fadd_rn(__fmul_rn(__uint_as_float(am), (float)(1.0 / 127.0)), 0.0f);
        const int64_t blk = ((int64_t)page * nkv + head) * a.c.ps + 16 * grp;  // first slot of the group of 16
        if (act) {
            const uint8_t c1 = to_u8(__fadd_rn(__builtin_roundf(__fdiv_rn(y1, sc)), 128.0f));
            const uint8_t c2 = to_u8(__fadd_rn(__builtin_roundf(__fdiv_rn(y2, sc)), 128.0f));
            if (kind == 1) {
                a.c.k[(blk + in) * hd + lane] = c1;
                a.c.k[(blk + in) * hd + lane + half] = c2;
            } else {
                a.c.v[blk * hd + 16 * lane + in] = c1;
                a.c.v[blk * hd + 16 * (lane + half) + in] = c2;
            }
        }
        if (lane == 0) (kind == 1 ? a.c.ks : a.c.vs)[blk + in] = sc;
    }
}

// The same for rows that come in runs: k and v by groups of 16 positions, a wave the k
// or the v of a (group, KV head), so that a group's v, whose 16 tokens are neighbours
// in memory, is put down in 16-byte pieces instead of bytes; behind them, as the
// shorter work, the q heads by rows, N heads a wave.  2998 bf16 rows of 32 + 2 * 8
// heads of 128: 68 MB in 20 us, 3.4 TB/s, a third of it latency (by rows 36 us; N = 4
// or 16: 22 us).
// grid groups * ceil(2 nkv / 4) + rows * ceil(nh / (4 N)).
namespace {

// two neighbouring elements
template <bool BF>
__device__ __forceinline__ float2 load2(const void* p, int64_t i)
{
    if (!BF) return *(const float2*)((const float*)p + i);
    const uint32_t w = *(const uint32_t*)((const uint16_t*)p + i);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

template <bool BF>
__device__ __forceinline__ void store2(void* p, int64_t i, float x, float y)
{
    if (BF) *(uint32_t*)((uint16_t*)p + i) = (uint32_t)f32_to_bf16(x) | (uint32_t)f32_to_bf16(y) << 16;
    else *(float2*)((float*)p + i) = make_float2(x, y);
}

__device__ __forceinline__ float q8_scale(uint32_t amax)
{
    return __fadd_rn(__fmul_rn(__uint_as_float(amax), (float)(1.0 / 127.0)), 0.0f);
}

__device__ __forceinline__ uint32_t q8_code(float x, float s)
{
    return to_u8(__fadd_rn(__builtin_roundf(__fdiv_rn(x, s)), 128.0f));
}

__device__ __forceinline__ uint32_t mag(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

}  // namespace

template <bool BF, int N>
__global__ __launch_bounds__(256) void k_paged_append_runs(PagedAppend a, int groups)
{
    const Paged& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hd = c.hd, half = hd >> 1, nkv = c.nkv;
    const float nan = __builtin_nanf("");
    const unsigned kvs = (unsigned)groups * ((2 * nkv + 3) / 4);  // workgroups of k and v
    if (blockIdx.x >= kvs) {
        const unsigned b = blockIdx.x - kvs;
        const int t = b % (unsigned)c.rows, first = N * (4 * (int)(b / (unsigned)c.rows) + wave);
        if (first >= a.nh) return;
        // two heads at a time, half a wave each, two neighbouring pairs a lane
        const int m = lane & 31, up = lane >> 5;
        const bool act = 2 * m < half;
        float2 x1[N / 2], x2[N / 2];
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            x1[e] = x2[e] = make_float2(0.0f, 0.0f);
            if (act && first + 2 * e + up < a.nh) {
                const int64_t row = ((int64_t)t * a.nh + first + 2 * e + up) * hd + 2 * m;
                x1[e] = load2<BF>(a.q, row);
                x2[e] = load2<BF>(a.q, row + half);
            }
        }
        const int s = find_seq(c, t, lane);
        if (s < 0 || s >= c.n_seqs) return;
        const Seq q = seq_at(c, s);
        const int i = t - q.a;
        if (i < 0 || i >= q.n || !act) return;
        const int pos = q.p0 + i;
        float2 co = make_float2(nan, nan), si = co;
        if (q.ok && pos < a.rope_len) {
            co = *(const float2*)(a.cos_t + (int64_t)pos * half + 2 * m);
            si = *(const float2*)(a.sin_t + (int64_t)pos * half + 2 * m);
        }
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            if (first + 2 * e + up >= a.nh) return;
            const int64_t row = ((int64_t)t * a.nh + first + 2 * e + up) * hd + 2 * m;
            store2<BF>(a.q_out, row, __fsub_rn(__fmul_rn(x1[e].x, co.x), __fmul_rn(x2[e].x, si.x)),
                       __fsub_rn(__fmul_rn(x1[e].y, co.y), __fmul_rn(x2[e].y, si.y)));
            store2<BF>(a.q_out, row + half, __fadd_rn(__fmul_rn(x1[e].x, si.x), __fmul_rn(x2[e].x, co.x)),
                       __fadd_rn(__fmul_rn(x1[e].y, si.y), __fmul_rn(x2[e].y, co.y)));
        }
        return;
    }
    const int slot = 4 * (int)(blockIdx.x / (unsigned)groups) + wave, head = slot >> 1;
    if (head >= nkv) return;
    int piece = blockIdx.x % (unsigned)groups;
    const int s = __builtin_amdgcn_readfirstlane(find_piece(c, lane, piece, [&](int x) {
        const Seq q = seq_at(c, x);
        return q.n && q.ok ? ((q.p0 + q.n - 1) >> 4) - (q.p0 >> 4) + 1 : 0;
    }));
    if (s < 0) return;
    const Seq q = seq_at(c, s);
    const int grp = (q.p0 >> 4) + piece, i0 = 16 * grp - q.p0;  // the sequence's row of the group's first position
    int in;
    const int page = page_of(c, c.pages + (int64_t)s * c.max_pages, grp, &in);
    if (page < 0) return;
    // tokens r0 <= r < r1 of the group are rows of the call with a RoPE position
    const int r0 = max(0, -i0), r1 = min(min(16, q.n - i0), a.rope_len - 16 * grp);
    if (r0 >= r1) return;
    const int64_t blk = ((int64_t)page * nkv + head) * c.ps + 16 * in;
    const int64_t row0 = ((int64_t)(q.a + i0) * nkv + head) * hd, step = (int64_t)nkv * hd;

    if (slot & 1) {
        // v: two neighbouring values of every token a lane
        const bool act = 2 * lane < hd;
        float2 x[16];
#pragma unroll
        for (int r = 0; r < 16; ++r)
            x[r] = act && r >= r0 && r < r1 ? load2<BF>(a.v, row0 + r * step + 2 * lane) : make_float2(0.0f, 0.0f);
        uint32_t w0[4] = {}, w1[4] = {};
        float mine = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float sc = q8_scale(wave_max_dpp(max(mag(x[r].x), mag(x[r].y))));
            w0[r >> 2] |= q8_code(x[r].x, sc) << (8 * (r & 3));
            w1[r >> 2] |= q8_code(x[r].y, sc) << (8 * (r & 3));
            mine = lane == r ? sc : mine;
        }
        if (lane >= r0 && lane < r1) c.vs[blk + lane] = mine;
        uint8_t* p = c.v + blk * hd + 32 * lane;
        if (act && r0 == 0 && r1 == 16) {
            ((uint4*)p)[0] = make_uint4(w0[0], w0[1], w0[2], w0[3]);
            ((uint4*)p)[1] = make_uint4(w1[0], w1[1], w1[2], w1[3]);
        } else if (act) {
            // shifted out byte by byte: the other tokens' bytes stay as they are
            for (int r = 0; r < r1; ++r) {
                if (r >= r0) {
                    p[r] = (uint8_t)w0[0];
                    p[16 + r] = (uint8_t)w1[0];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w0[e] = w0[e] >> 8 | (e < 3 ? w0[e < 3 ? e + 1 : 3] << 24 : 0u);
                    w1[e] = w1[e] >> 8 | (e < 3 ? w1[e < 3 ? e + 1 : 3] << 24 : 0u);
                }
            }
        }
        return;
    }
    // k: two tokens at a time, half a wave each, two neighbouring pairs a lane
    const int m = lane & 31, up = lane >> 5;
    const bool act = 2 * m < half;
    float2 x1[8], x2[8], co[8], si[8];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const int r = 2 * b + up;
        const bool on = act && r >= r0 && r < r1;
        x1[b] = x2[b] = co[b] = si[b] = make_float2(0.0f, 0.0f);
        if (on) {
            x1[b] = load2<BF>(a.k, row0 + r * step + 2 * m);
            x2[b] = load2<BF>(a.k, row0 + r * step + half + 2 * m);
            co[b] = *(const float2*)(a.cos_t + (int64_t)(16 * grp + r) * half + 2 * m);
            si[b] = *(const float2*)(a.sin_t + (int64_t)(16 * grp + r) * half + 2 * m);
        }
    }
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const int r = 2 * b + up;
        const float y0 = __fsub_rn(__fmul_rn(x1[b].x, co[b].x), __fmul_rn(x2[b].x, si[b].x));
        const float y1 = __fsub_rn(__fmul_rn(x1[b].y, co[b].y), __fmul_rn(x2[b].y, si[b].y));
        const float z0 = __fadd_rn(__fmul_rn(x1[b].x, si[b].x), __fmul_rn(x2[b].x, co[b].x));
        const float z1 = __fadd_rn(__fmul_rn(x1[b].y, si[b].y), __fmul_rn(x2[b].y, co[b].y));
        const uint32_t am = max(max(mag(y0), mag(y1)), max(mag(z0), mag(z1)));
        const uint32_t lo = wave_max_dpp(up ? 0u : am), hi = wave_max_dpp(up ? am : 0u);
        const float sc = q8_scale(up ? hi : lo);
        if (r < r0 || r >= r1) continue;
        if (act) {
            uint8_t* p = c.k + (blk + r) * hd + 2 * m;
            *(uint16_t*)p = (uint16_t)(q8_code(y0, sc) | q8_code(y1, sc) << 8);
            *(uint16_t*)(p + half) = (uint16_t)(q8_code(z0, sc) | q8_code(z1, sc) << 8);
        }
        if (m == 0) c.ks[blk + r] = sc;
    }
}

// groups of 16 positions that the rows lie in: a sequence's rows touch at most a
// sixteenth as many and two more
static int64_t groups_at_most(const Paged& c)
{
    return std::min<int64_t>(c.rows, c.rows / 16 + 2 * (int64_t)c.n_seqs);
}

hipError_t launch_paged_append(const PagedAppend& a, hipStream_t st)
{
    const int slots = a.nh + 2 * a.c.nkv;
    auto go = [&](auto k, int n) {
        hipLaunchKernelGGL(k, dim3((unsigned)a.c.rows, (unsigned)((slots + 4 * n - 1) / (4 * n))), dim3(256), 0, st, a);
    };
    // one slot a wave while they all run at once (256 CUs of 32 waves)
    const bool many = (int64_t)a.c.rows * slots > 8192;
    if (many && a.c.rows >= 8 * a.c.n_seqs && (int64_t)a.c.rows * slots < ((int64_t)1 << 24)) {
        constexpr int N = 8;
        const int64_t groups = groups_at_most(a.c);
        const dim3 grid((unsigned)(groups * ((2 * a.c.nkv + 3) / 4) + (int64_t)a.c.rows * ((a.nh + 4 * N - 1) / (4 * N))));
        if (a.bf) hipLaunchKernelGGL((k_paged_append_runs<true, N>), grid, dim3(256), 0, st, a, (int)groups);
        else hipLaunchKernelGGL((k_paged_append_runs<false, N>), grid, dim3(256), 0, st, a, (int)groups);
        return hipGetLastError();
    }
    if (a.bf) many ? go(k_paged_append<true, 6>, 6) : go(k_paged_append<true, 1>, 1);
    else many ? go(k_paged_append<false, 6>, 6) : go(k_paged_append<false, 1>, 1);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// k_paged_read
// ---------------------------------------------------------------------------
// A wave takes a group of 16 positions of a sequence for one KV head, its k or its v:
// one run of 16 hd bytes, read once in 16-byte pieces.  Of k a lane has 16
// neighbouring values of a row; of v 16 rows of two neighbouring values, put out row by
// row.  grid (groups, ceil(2 nkv / 4)), block 256.  42.7 K positions of 8 heads of 128
// into bf16: 264 MB in 46 us, 5.7 TB/s (row by row, v byte by byte: 134 us).
namespace {

// v[0 .. 16) of a row
template <bool BF>
__device__ __forceinline__ void store16(void* p, int64_t i, const float* v)
{
    if (BF) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = (uint32_t)f32_to_bf16(v[2 * e]) | (uint32_t)f32_to_bf16(v[2 * e + 1]) << 16;
        uint4* o = (uint4*)((uint16_t*)p + i);
        o[0] = make_uint4(w[0], w[1], w[2], w[3]);
        o[1] = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
        float4* o = (float4*)((float*)p + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
    }
}

// (code - 128) * s of byte b of a word
__device__ __forceinline__ float value_at(uint32_t w, int b, float s)
{
    return __fmul_rn(__fsub_rn((float)(w >> (8 * b) & 255u), 128.0f), s);
}

}  // namespace

template <bool BF>
__global__ __launch_bounds__(256) void k_paged_read(PagedRead a)
{
    const Paged& c = a.c;
    const int lane = threadIdx.x & 63;
    const int slot = 4 * blockIdx.y + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = slot >> 1;
    const bool is_v = slot & 1;
    if (head >= c.nkv || !(is_v ? a.v_out : a.k_out)) return;
    int piece = blockIdx.x;
    const int s = __builtin_amdgcn_readfirstlane(find_piece(c, lane, piece, [&](int x) {
        const Seq q = seq_at(c, x);
        const int p0 = q.ok ? q.p0 : 0;
        return q.n ? ((p0 + q.n - 1) >> 4) - (p0 >> 4) + 1 : 0;
    }));
    if (s < 0) return;
    const Seq q = seq_at(c, s);
    const int p0 = q.ok ? q.p0 : 0, grp = (p0 >> 4) + piece;
    int in = 0, page = -1;
    if (q.ok) page = page_of(c, c.pages + (int64_t)s * c.max_pages, grp, &in);
    const int hd = c.hd;
    const int64_t blk = ((int64_t)max(page, 0) * c.nkv + head) * c.ps + 16 * in;
    const int i0 = 16 * grp - p0;  // the sequence's row of the group's first position
    const int64_t out = ((int64_t)q.a * c.nkv + head) * hd, step = (int64_t)c.nkv * hd;
    const float nan = __builtin_nanf("");
    if (!is_v) {
        const int D = hd >> 4, mul = (1024 + D - 1) / D;  // x / D = x * mul >> 10 for x < 192
        uint4 kw[2];
        float ks[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int x = min(lane + 64 * e, hd - 1);
            kw[e] = *(const uint4*)(c.k + blk * hd + 16 * x);
            ks[e] = c.ks[blk + (x * mul >> 10)];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int x = lane + 64 * e, r = x * mul >> 10, i = i0 + r;  // 16-byte piece x, of token r
            if (x >= hd || i < 0 || i >= q.n) continue;
            const float sc = page < 0 ? nan : ks[e];
            const uint32_t ws[4] = {kw[e].x, kw[e].y, kw[e].z, kw[e].w};
            float v[16];
#pragma unroll
            for (int b = 0; b < 16; ++b) v[b] = value_at(ws[b >> 2], b & 3, sc);
            store16<BF>(a.k_out, out + i * step + 16 * (x - r * D), v);
        }
        return;
    }
    if (lane >= (hd >> 1)) return;
    const uint4* p = (const uint4*)(c.v + blk * hd + 32 * lane);
    const uint4 w0 = p[0], w1 = p[1];
    float4 vs[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) vs[e] = *(const float4*)(c.vs + blk + 4 * e);
    const uint32_t a0[4] = {w0.x, w0.y, w0.z, w0.w}, a1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
        const float ss[4] = {vs[r4].x, vs[r4].y, vs[r4].z, vs[r4].w};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int i = i0 + 4 * r4 + b;
            if (i < 0 || i >= q.n) continue;
            const float f = page < 0 ? nan : ss[b];
            const float v0 = value_at(a0[r4], b, f), v1 = value_at(a1[r4], b, f);
            const int64_t at = out + i * step + 2 * lane;
            store2<BF>(a.v_out, at, v0, v1);
        }
    }
}

hipError_t launch_paged_read(const PagedRead& a, hipStream_t st)
{
    const int64_t groups = groups_at_most(a.c);
    const dim3 grid((unsigned)groups, (unsigned)((2 * a.c.nkv + 3) / 4));
    if (a.bf) hipLaunchKernelGGL(k_paged_read<true>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_paged_read<false>, grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Attention: k_paged_tok, k_paged_tile
// ---------------------------------------------------------------------------
// Per KV head the rows of a sequence times the query heads of the group are one
// list of query rows m = i * group + e; a wave takes 16 of them a column tile
// (NT tiles) against 64 keys at a time, both products on v_mfma_f32_16x16x32_f16:
//
//   S^T [16 keys][16 queries] = K [16 keys][hd] . Q^T       four key tiles t
//   O^T [16 values][16 queries] += V^T [16 values][64 keys] . P^T [64 keys][16 queries]
//
// A matrix instruction contracts over (lane group g = lane / 16, element j) in
// any order, as long as both operands agree.  So the dimension of a product is
// laid out by what one 16-byte load brings: for S, lane group g of step pair j
// holds values 16 (4 j + g) .. + 15 of its key; and key tile t puts key
// 16 (r / 4) + 4 t + r % 4 in row r, which makes the four tiles' results in one
// lane -- rows 4 g .. 4 g + 3 -- the 16 neighbours 16 g .. 16 g + 15.  Those are,
// as they stand, the second product's operand: its other side, 16 keys of one
// value, is one 16-byte load of the blocked v.  Nothing crosses lanes on the way.
//
// A code u8 becomes the f16 1024 + u8 by one byte permute, less 1152 (exact).
// Queries are scaled by a power of two per row to just under 2^15, softmax weights
// times the value's scale by one per (row, largest value scale so far), which is then
// in [2^8, 2^9): two parts keep 22 bits of a weight at the reference down to 2^-10 of
// that scale, and what they lose of any is below 2^-33 of it, whatever the weight of
// the key that has it.
//
// The softmax is taken in one pass against a reference that follows the row's
// largest score, but only when a score passes it by 2^6: then the sums so far are
// scaled down.  A few times a row, so the common step has neither a maximum across
// lanes nor a scaling of the outputs.
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

namespace {

constexpr float kAhead = 6.0f;   // a score may pass the reference by this (log2)
constexpr int kVUp = 8;          // weights times value scales stay below 2^(kAhead + 1 + kVUp) = 2^15
// The least exponent of a query row, and of a value scale, that is scaled up in full:
// a row's products are scaled as its queries are, by 2^(14 - e), so that q . k reaches
// 2^128 there from 2^(114 + e) on; e = -96 leaves 2^18.
constexpr int kLeastExp = -96;

// four codes -> four f16 (code - 128)
__device__ __forceinline__ void widen4(uint32_t w, uint32_t* o)
{
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off;
    const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off;
    o[0] = __builtin_bit_cast(uint32_t, a);
    o[1] = __builtin_bit_cast(uint32_t, b);
}

__device__ __forceinline__ h8 widen8(uint32_t w0, uint32_t w1)
{
    uint32_t o[4];
    widen4(w0, o);
    widen4(w1, o + 2);
    return __builtin_bit_cast(h8, *(uint4*)o);
}

// The largest / the sum of a value over the four lanes n, n + 16, n + 32, n + 48,
// in each of them.  Swapping rows of a register with rows of its copy leaves the
// pairs' other values in the two results.
typedef unsigned u2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float xor16_max(float v)
{
    u2 p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
    p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
}

__device__ __forceinline__ float xor16_sum(float v)
{
    u2 p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __fadd_rn(__uint_as_float(p.x), __uint_as_float(p.y));
    p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __fadd_rn(__uint_as_float(p.x), __uint_as_float(p.y));
}

// Keeps the f32 product v as it was rounded.  The compiler may turn an f16
// conversion of a product into one instruction that rounds once; where the two
// parts of a number each convert it, that made a first part of one rounding and a
// rest of the other, off by a step of f16 in some of 10^4 weights.
__device__ __forceinline__ void as_rounded(float& v) { asm("" : "+v"(v)); }

// 2^e, -126 <= e <= 127
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// exponent of |v|, at least kLeastExp (0, subnormal, not finite: that)
__device__ __forceinline__ int expo(float v)
{
    const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
    return b >= 0x7F800000u ? kLeastExp : max((int)(b >> 23) - 127, kLeastExp);
}

// v's 4 neighbouring values of a row
template <bool BF>
__device__ __forceinline__ void store4(void* p, int64_t i, f4 v)
{
    if (BF) {
        uint2 w;
        w.x = (uint32_t)f32_to_bf16(v.x) | (uint32_t)f32_to_bf16(v.y) << 16;
        w.y = (uint32_t)f32_to_bf16(v.z) | (uint32_t)f32_to_bf16(v.w) << 16;
        *(uint2*)((uint16_t*)p + i) = w;
    } else {
        *(f4*)((float*)p + i) = v;
    }
}

// row of a sequence that query row m belongs to: m / group
__device__ __forceinline__ int row_of(const PagedAttn& a, int m) { return (int)__umulhi(2u * (uint32_t)m, a.group_mul); }

// The query rows of a wave: NT tiles of 16, in PARTS f16 parts.
template <int NJ, int NT, bool BF>
struct Queries {
    static constexpr int PARTS = BF ? 1 : 2;
    float cq[NT];  // log2 units of one unit of the scaled product
    h8 v[PARTS][NT][2 * NJ];

    // rows m0 .. of a sequence, none past m_last (those repeat it); row0: the output row of m = 0
    __device__ __forceinline__ void load(const PagedAttn& a, const Seq& q, int64_t row0, int m0, int m_last, int lane)
    {
        const int g = lane >> 4, n = lane & 15, hd = a.c.hd;
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            const int m = m0 + 16 * u + n;
            const int mm = min(m, m_last);
            const int i = row_of(a, mm);
            const int64_t r = row0 + (int64_t)i * a.nh + (mm - i * a.group);
            float f[NJ][16];
            float am = 0.0f;
            bool bad = false;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int d = 16 * (4 * j + g);
                if (BF) {
                    uint4 w[2] = {};
                    if (d < hd) {
                        w[0] = *(const uint4*)((const uint16_t*)a.q + r * hd + d);
                        w[1] = *(const uint4*)((const uint16_t*)a.q + r * hd + d + 8);
                    }
                    widen16<XK_BF16>(w, f[j]);
                } else {
                    uint4 w[4] = {};
                    if (d < hd)
#pragma unroll
                        for (int x = 0; x < 4; ++x) w[x] = *(const uint4*)((const float*)a.q + r * hd + d + 4 * x);
                    widen16<XK_F32>(w, f[j]);
                }
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    am = fmaxf(am, __builtin_fabsf(f[j][x]));
                    bad |= !(__builtin_fabsf(f[j][x]) < __builtin_inff());
                }
            }
            am = xor16_max(bad ? __builtin_inff() : am);
            const bool fin = am < __builtin_inff();
            const int sh = fin ? 14 - expo(am) : 0;
            const float up = exp2i(sh);
            cq[u] = fin ? __fmul_rn(a.scale_log2, exp2i(-sh)) : __builtin_nanf("");
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float y = fin ? __fmul_rn(f[j][x], up) : 0.0f;  // exact
                    const _Float16 hi = (_Float16)y;
                    v[0][u][2 * j + (x >> 3)][x & 7] = hi;
                    if (PARTS == 2) v[PARTS - 1][u][2 * j + (x >> 3)][x & 7] = (_Float16)__fsub_rn(y, (float)hi);
                }
        }
    }
};

// One column tile's running softmax and output.
template <int DT>
struct Running {
    float ref, l;  // reference (log2; -inf before the first key), this lane's part of the sum
    int ve;        // exponent of the value scales that the weights are scaled by
    f4 o[DT];

    __device__ __forceinline__ void clear()
    {
        ref = -__builtin_inff();
        l = 0.0f;
        ve = kLeastExp;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    __device__ __forceinline__ void scale(float f)
    {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= f;
    }

    // the value scales up to exponent e are to come
    __device__ __forceinline__ void raise(int e)
    {
        scale(__builtin_ldexpf(1.0f, ve - e));
        ve = e;
    }

    // 16 scores in log2 units, less the reference: two roundings, not a fused one, so that
    // the largest score's is the reference exactly however large it is.
    __device__ __forceinline__ static void score(const f4* sc, float cq, float at, float* y)
    {
#pragma unroll
        for (int x = 0; x < 16; ++x) y[x] = __fsub_rn(__fmul_rn(sc[x >> 2][x & 3], cq), at);
    }

    // sc: the products of 16 keys with their scales (-inf: not seen); vs: value
    // scales times 2^(kVUp - ve).  Leaves the weights, in f16 parts.
    template <int PARTS>
    __device__ __forceinline__ void weigh(const f4* sc, const f4* vs, float cq, h8 (*pw)[2])
    {
        float y[16];
        float big = -__builtin_inff();
        float at = ref == -__builtin_inff() ? 0.0f : ref;
        score(sc, cq, at, y);
#pragma unroll
        for (int x = 0; x < 16; ++x) big = fmaxf(big, y[x]);
        if (__any(big > kAhead || ref == -__builtin_inff())) {
            float top = -__builtin_inff();
#pragma unroll
            for (int x = 0; x < 16; ++x) top = fmaxf(top, __fmul_rn(sc[x >> 2][x & 3], cq));
            top = xor16_max(top);
            const bool moves = ref == -__builtin_inff() ? top > ref : xor16_max(big) > kAhead;
            const float to = moves ? top : ref;
            const float down = ref == -__builtin_inff() ? 0.0f : (moves ? __builtin_amdgcn_exp2f(__fsub_rn(at, to)) : 1.0f);
            l = __fmul_rn(l, down);
            scale(down);
            ref = to;
            at = ref == -__builtin_inff() ? 0.0f : ref;
            score(sc, cq, at, y);
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const float p = __builtin_amdgcn_exp2f(y[x]);
            l = __fadd_rn(l, p);
            float w = __fmul_rn(p, vs[x >> 2][x & 3]);
            if (PARTS == 2) as_rounded(w);
            const _Float16 hi = (_Float16)w;
            pw[0][x >> 3][x & 7] = hi;
            if (PARTS == 2) pw[PARTS - 1][x >> 3][x & 7] = (_Float16)__fsub_rn(w, (float)hi);
        }
    }

    // the largest finite value scale among 16, over the four lanes of a row
    __device__ __forceinline__ static float largest(const f4* vs)
    {
        float m = 0.0f;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const float v = __builtin_fabsf(vs[x >> 2][x & 3]);
            m = v < __builtin_inff() ? fmaxf(m, v) : m;
        }
        return xor16_max(m);
    }

    // a step whose keys this lane's row sees below `vis` only (key: its first)
    template <int PARTS>
    __device__ __forceinline__ void weigh_masked(f4* sc, const f4* vs, int key, int vis, float cq, h8 (*pw)[2])
    {
        f4 vm[4];
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const bool see = key + x < vis;
            sc[x >> 2][x & 3] = see ? sc[x >> 2][x & 3] : -__builtin_inff();
            vm[x >> 2][x & 3] = see ? vs[x >> 2][x & 3] : 0.0f;
        }
        const int e = max(ve, expo(largest(vm)));
        if (__any(e != ve)) raise(e);
        const float up = exp2i(kVUp - ve);
#pragma unroll
        for (int t = 0; t < 4; ++t) vm[t] *= up;
        weigh<PARTS>(sc, vm, cq, pw);
    }

    // one unit of o
    __device__ __forceinline__ float unit() const { return exp2i(ve - kVUp); }
};

struct True {
    constexpr operator bool() const { return true; }
};
struct False {
    constexpr operator bool() const { return false; }
};

// The groups of 16 slots, counted over all pages and heads, that hold 64 neighbouring
// groups of a sequence's keys, one a lane (past its last group: that one; -1: the
// page is outside the pool).  Looked up together, so a step takes its four from
// registers instead of waiting for the page table.
struct Slots {
    int mine, base;

    __device__ __forceinline__ void find(const Paged& c, const int32_t* table, int grp, int last_grp, int h, int lane)
    {
        int in;
        const int page = page_of(c, table, min(grp + lane, last_grp), &in);
        mine = page < 0 ? -1 : (page * c.nkv + h) * c.ppg + in;  // below 2^31: the host checks it
        base = grp;
    }
    // of group `grp`, base <= grp < base + 64
    __device__ __forceinline__ int of(int grp) const { return __builtin_amdgcn_ds_bpermute(4 * (grp - base), mine); }
};

// Where a workgroup works: its KV head, chunk of keys and sequence.
struct Place {
    int h, chunk, tile, s;
};

// blockIdx.x = h + nkv (chunk + chunks * tile): the head varies fastest.  Workgroups
// go to the XCDs in turn, so with 8 KV heads the tiles and chunks of one head share
// an XCD's L2.
__device__ __forceinline__ Place place_of(const Paged& c, int chunks)
{
    Place p;
    p.h = (int)(blockIdx.x % (unsigned)c.nkv);
    const unsigned b = blockIdx.x / (unsigned)c.nkv;
    p.chunk = (int)(b % (unsigned)chunks);
    p.tile = (int)(b / (unsigned)chunks);
    p.s = p.tile;
    return p;
}

// The rows of a refused sequence.
template <bool BF>
__device__ __forceinline__ void fill_nan(const PagedAttn& a, const Seq& q, int h, int wave, int waves, int lane)
{
    for (int i = wave; i < q.n; i += waves)
        for (int x = lane; x < a.group * a.c.hd; x += 64)
            store1<BF>(a.out, ((int64_t)(q.a + i) * a.nh + h * a.group) * a.c.hd + x, __builtin_nanf(""));
}

}  // namespace

// The token form: at most 16 query rows of a sequence.  grid nkv * chunks * n_seqs,
// block 64 NW: the waves take the chunk's keys in turn, 64 at a time, straight from
// memory into the operands' registers, and are merged in LDS.  NW is 4; 8 where the
// sequences are short enough to be one chunk each, which saves the merge's launch.  DT: 16-value
// tiles of a head, hd / 16 or one more.
//
// Bound by the cache's bytes: every code is read once, 16 KB a step and wave in
// flight, two waves a SIMD (registers: with one, loads prefetched a step ahead, it was
// 92 us; with three it spills).  32 sequences of up to 8192 positions, 8 heads of 128,
// bf16: 353 MB in 75 us, 4.7 TB/s; one of 100001, f32: 211 MB in 35 us, 6.0 TB/s (a
// sum of 4 GiB reads 6.15 TB/s).
template <int DT, int NW, bool BF>
__global__ __launch_bounds__(64 * NW, 2) void k_paged_tok(PagedAttn a)
{
    constexpr int NJ = (DT + 3) / 4;
    constexpr int PARTS = BF ? 1 : 2;  // of the queries (bf16 ones are exact in one)
    // Of the weights.  One part in bf16 would save 1.7 us of the batch's 81.4, and one output in
    // twelve would round the other way; in two it is one in 3000.
    constexpr int WP = 2;
    __shared__ __align__(16) float s_o[NW][16][16 * DT + 4];
    __shared__ float s_m[NW][16], s_l[NW][16];
    const Paged& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int hd = c.hd, ndt = hd >> 4, C = a.p.tok_c;
    const Place at = place_of(c, a.p.tok_n);
    const int key0 = at.chunk * C;
    const int32_t* table = c.pages + (int64_t)at.s * c.max_pages;
    // the pages are looked up beside the sequence's size, not after it: what the table holds
    // behind its last page is checked like any id, and its keys are masked
    const int last_grp = (c.cap - 1) >> 4;
    Slots slots{};
    if (c.cap > 0) slots.find(c, table, (key0 + 64 * wave) >> 4, last_grp, at.h, lane);
    const Seq q = seq_at(c, at.s);
    const int64_t M = (int64_t)q.n * a.group;
    if (M == 0 || M > a.p.lo) return;
    const int64_t row0 = (int64_t)q.a * a.nh + at.h * a.group;  // output row of m: row0 + (m / group) * nh + m % group
    if (!q.ok) {
        if (at.chunk == 0) fill_nan<BF>(a, q, at.h, wave, NW, lane);
        return;
    }
    const int seen = q.p0 + q.n;  // keys that the last row sees
    const int key1 = min(key0 + C, seen);
    if (key0 >= key1) return;

    Queries<NJ, 1, BF> qs;
    qs.load(a, q, row0, 0, (int)M - 1, lane);
    Running<DT> r;
    r.clear();
    for (int kb = key0 + 64 * wave; kb < key1; kb += 64 * NW) {
        // a lane loads a key row of group n / 4, and takes the scales and values of group g
        const int grp = kb >> 4;
        if (grp + 4 > slots.base + 64) slots.find(c, table, grp, last_grp, at.h, lane);
        const int own = slots.of(grp + g), at_v = max(own, 0);
        const uint8_t* kp = c.k + (uint64_t)(uint32_t)max(slots.of(grp + (n >> 2)), 0) * (uint32_t)(16 * hd) + (n & 3) * hd;
        const uint8_t* vp = c.v + (uint64_t)(uint32_t)at_v * (uint32_t)(16 * hd) + 16 * n;
        const float* kscale = c.ks + 16 * (int64_t)at_v;
        const float* vscale = c.vs + 16 * (int64_t)at_v;
        uint4 kw[4][NJ];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < NJ; ++j) kw[t][j] = *(const uint4*)(kp + 4 * t * hd + 16 * (4 * j + g < ndt ? 4 * j + g : 0));
        f4 ks[4], vs[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            ks[t] = *(const f4*)(kscale + 4 * t);
            vs[t] = *(const f4*)(vscale + 4 * t);
        }
        uint4 vw[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) vw[d] = *(const uint4*)(vp + 256 * min(d, ndt - 1));
        const float lost = own < 0 ? __builtin_nanf("") : 0.0f;

        f4 sc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            sc[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const h8 k0 = widen8(kw[t][j].x, kw[t][j].y), k1 = widen8(kw[t][j].z, kw[t][j].w);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qs.v[p][0][2 * j], sc[t], 0, 0, 0);
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qs.v[p][0][2 * j + 1], sc[t], 0, 0, 0);
                }
            }
            // NaN where the page is outside the pool or a scale is not finite: an infinite one
            // times a negative product would be -inf, which is a key that no row sees
#pragma unroll
            for (int e = 0; e < 4; ++e)
                sc[t][e] = __fmaf_rn(sc[t][e], ks[t][e], __fmaf_rn(ks[t][e], 0.0f, __fmaf_rn(vs[t][e], 0.0f, lost)));
        }
        h8 pw[WP][2];
        if (kb + 64 <= q.p0 + 1) {  // every row sees every key
            const int e = max(r.ve, expo(r.largest(vs)));
            if (__any(e != r.ve)) r.raise(e);
            const float up = exp2i(kVUp - r.ve);
#pragma unroll
            for (int t = 0; t < 4; ++t) vs[t] *= up;
            r.template weigh<WP>(sc, vs, qs.cq[0], pw);
        } else {
            const int vis = q.p0 + row_of(a, min(n, (int)M - 1)) + 1;  // keys that this lane's row sees
            r.template weigh_masked<WP>(sc, vs, kb + 16 * g, vis, qs.cq[0], pw);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const h8 v0 = widen8(vw[d].x, vw[d].y), v1 = widen8(vw[d].z, vw[d].w);
#pragma unroll
            for (int p = 0; p < WP; ++p) {
                r.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pw[p][0], r.o[d], 0, 0, 0);
                r.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pw[p][1], r.o[d], 0, 0, 0);
            }
        }
    }

    const float l = xor16_sum(r.l), unit = r.unit();
    if (g == 0) {
        s_m[wave][n] = r.ref;
        s_l[wave][n] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) *(f4*)&s_o[wave][n][16 * d + 4 * g] = r.o[d] * unit;
    __syncthreads();
    const bool whole = seen <= C;  // the sequence is one chunk
    for (int x = threadIdx.x; x < (int)M * (hd >> 2); x += 64 * NW) {
        const int m = x / (hd >> 2), d = 4 * (x - m * (hd >> 2));
        float top = s_m[0][m];
#pragma unroll
        for (int w = 1; w < NW; ++w) top = fmaxf(top, s_m[w][m]);
        top = top == -__builtin_inff() ? 0.0f : top;
        float sum = 0.0f;
        f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float b = __builtin_amdgcn_exp2f(__fsub_rn(s_m[w][m], top));
            sum = __fmaf_rn(b, s_l[w][m], sum);
            const f4 ow = *(const f4*)&s_o[w][m][d];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __fmaf_rn(b, ow[e], v[e]);
        }
        const int i = row_of(a, m);
        const int64_t row = row0 + (int64_t)i * a.nh + (m - i * a.group);
        if (whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __fdiv_rn(v[e], sum);
            store4<BF>(a.out, row * hd + d, v);
        } else {
            const int64_t part = row * a.parts + at.chunk;
            store4<false>(a.part_o, part * hd + d, v);
            if (d == 0) *(float2*)(a.part_ml + 2 * part) = make_float2(top, sum);
        }
    }
}

// The tile form: 64 NT query rows of a sequence, 16 NT a wave, every key to all four
// waves.  grid nkv * chunks * tiles, block 256.  Each wave widens a quarter of the
// next 64 keys' codes while the present ones are worked on: they lie in LDS as
// operand fragments (64 lanes x 16 bytes, read and written without conflicts), so a
// code is widened once a workgroup instead of once a wave.
//
// 512 rows over 8192 positions, 32 heads over 8 of 128: 66.6 GFLOP in 114 us in bf16
// (584 TFLOP/s; a large library product reaches 1116), 192 us in f32, whose two parts
// are two products.  Per wave and 64 keys of 32 rows the matrix instructions take 1024
// cycles, the softmax and the widening some 1900 of the vector unit, on which two waves
// a SIMD take turns: that, and what is left of LDS latency between them, is the bound.
// Tried: each wave widening for itself 267 us; 48 or 64 rows a wave 280 and 223 (one
// wave a SIMD); without reading operands ahead 124 to 115; a branch-free step 117; wave
// priorities 129.
template <int DT, int NT, bool BF>
__global__ __launch_bounds__(256, 2) void k_paged_tile(PagedAttn a)
{
    constexpr int NJ = (DT + 3) / 4;
    // Of the queries and of the weights.  In bf16 a query is exact in one part, and weights are
    // rounded to one, off by 2^-11 of themselves at most, ahead of an output that is rounded by
    // 2^-8: the 512-row chunk is 1.677e-3 (two-norm) off the exact result so and 1.663e-3, which
    // is the output's rounding alone, in two parts; it takes 114 us so and 137 in two.
    constexpr int PARTS = BF ? 1 : 2;
    constexpr int MT = 64 * NT;
    __shared__ __align__(16) h8 s_k[2][4][2 * NJ][64];
    __shared__ __align__(16) h8 s_v[2][DT][2][64];
    __shared__ __align__(16) float s_ks[2][64], s_vs[2][64];
    __shared__ float s_top[2];
    const Paged& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int hd = c.hd, ndt = hd >> 4, C = a.p.tile_c;
    Place at = place_of(c, a.p.tile_n);

    // the sequence that the tile belongs to: sequences of more than `lo` query rows have
    // one for every MT of them.  A refused one has one for its NaN: the launch has tiles for
    // max_rows rows of it, and the others come behind.
    at.s = __builtin_amdgcn_readfirstlane(find_piece(c, lane, at.tile, [&](int s) {
        const Seq q = seq_at(c, s);
        const int64_t rows = (int64_t)q.n * a.group;
        return rows > a.p.lo ? (q.ok ? (int)((rows + MT - 1) / MT) : 1) : 0;
    }));
    if (at.s < 0) return;
    const Seq q = seq_at(c, at.s);
    const int64_t M = (int64_t)q.n * a.group;
    const int64_t row0 = (int64_t)q.a * a.nh + at.h * a.group;
    if (!q.ok) {
        if (at.chunk == 0 && at.tile == 0) fill_nan<BF>(a, q, at.h, wave, 4, lane);
        return;
    }
    const int m_tile = at.tile * MT;
    const int m_wave = m_tile + 16 * NT * wave;
    const int m_last = (int)min(M, (int64_t)m_tile + MT) - 1;
    const int seen = q.p0 + row_of(a, m_last) + 1;  // keys that the tile's last row sees
    const int key0 = at.chunk * C, key1 = min(key0 + C, seen);
    if (key0 >= key1) return;
    const int32_t* table = c.pages + (int64_t)at.s * c.max_pages;
    const int last_grp = (key1 - 1) >> 4;

    // this wave's share of 64 keys: key tile t = wave of k, value tiles wave, wave + 4 of v,
    // the scales (waves 0 and 1)
    uint4 kw[NJ], vw[NJ];
    float scale = 0.0f;
    bool lost = false;  // its page is outside the pool
    Slots slots;
    slots.find(c, table, key0 >> 4, last_grp, at.h, lane);
    auto fetch = [&](int kb) {
        const int grp = kb >> 4;
        if (grp + 4 > slots.base + 64) slots.find(c, table, grp, last_grp, at.h, lane);
        // offsets made anew from the lane each time: the compiler kept them across the
        // loop as 64-bit addresses, and spilled
        int ln = lane;
        asm("" : "+v"(ln));
        const int n = ln & 15, g = ln >> 4, g16 = 16 * g;
        const int koff = ((n & 3) + 4 * wave) * hd, voff = 16 * n;
        const int own = slots.of(grp + g), at_v = max(own, 0);
        const uint8_t* kp = c.k + (uint64_t)(uint32_t)max(slots.of(grp + (n >> 2)), 0) * (uint32_t)(16 * hd);
        const uint8_t* vp = c.v + (uint64_t)(uint32_t)at_v * (uint32_t)(16 * hd);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int ko = 64 * j + g16;
            kw[j] = *(const uint4*)(kp + (koff + (ko < hd ? ko : 0)));
            vw[j] = *(const uint4*)(vp + (voff + 256 * min(wave + 4 * j, ndt - 1)));
        }
        scale = (wave & 1 ? c.vs : c.ks)[16 * (int64_t)at_v + n];
        lost = own < 0;
    };
    auto put = [&](int b) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            s_k[b][wave][2 * j][lane] = widen8(kw[j].x, kw[j].y);
            s_k[b][wave][2 * j + 1][lane] = widen8(kw[j].z, kw[j].w);
            if (wave + 4 * j < DT) {
                s_v[b][wave + 4 * j][0][lane] = widen8(vw[j].x, vw[j].y);
                s_v[b][wave + 4 * j][1][lane] = widen8(vw[j].z, vw[j].w);
            }
        }
        // a scale that is not finite is NaN for whoever sees its key: an infinite one times a
        // negative product would be -inf, which is a key that no row sees
        const bool bad = !(__builtin_fabsf(scale) < __builtin_inff());
        if (wave == 0) s_ks[b][lane] = lost || bad ? __builtin_nanf("") : scale;
        if (wave == 1) {
            s_vs[b][lane] = bad ? __builtin_nanf("") : scale;
            const uint32_t m = __float_as_uint(scale) & 0x7FFFFFFFu;
            const uint32_t top = wave_max_dpp(m < 0x7F800000u ? m : 0u);  // of finite ones
            if (lane == 0) s_top[b] = __uint_as_float(top);
        }
    };

    Running<DT> r[NT];
    Queries<NJ, NT, BF> qs;
    auto step = [&](int kb, int b, auto masked) {
        if (kb + 64 < key1) fetch(kb + 64);
        f4 sc[NT][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const f4 ks = *(const f4*)&s_ks[b][16 * g + 4 * t];
#pragma unroll
            for (int u = 0; u < NT; ++u) sc[u][t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 2 * NJ; ++j) {
                const h8 k = s_k[b][t][j][lane];
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
#pragma unroll
                    for (int u = 0; u < NT; ++u)
                        sc[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qs.v[p][u][j], sc[u][t], 0, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < NT; ++u) sc[u][t] *= ks;
        }
        // operands are read some products ahead: LDS answers after some 130 cycles, two products take 32
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
        for (int x = 0; x < 4 * 2 * NJ; ++x) {
            __builtin_amdgcn_sched_group_barrier(0x008, PARTS * NT, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        f4 vs[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) vs[t] = *(const f4*)&s_vs[b][16 * g + 4 * t];
        h8 pw[NT][PARTS][2];
        if (masked) {
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                int m = m_wave + 16 * u + n;
                asm("" : "+v"(m));  // not kept across the loop
                const int vis = q.p0 + row_of(a, min(m, m_last)) + 1;  // keys that this lane's row sees
                r[u].template weigh_masked<PARTS>(sc[u], vs, kb + 16 * g, vis, qs.cq[u], pw[u]);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            // every row sees every key, and so far saw the same: their ve are one
            const int e = max(r[0].ve, expo(s_top[b]));
            if (e != r[0].ve)
#pragma unroll
                for (int u = 0; u < NT; ++u) r[u].raise(e);
            const float up = exp2i(kVUp - r[0].ve);
#pragma unroll
            for (int t = 0; t < 4; ++t) vs[t] *= up;
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                r[u].template weigh<PARTS>(sc[u], vs, qs.cq[u], pw[u]);
                __builtin_amdgcn_sched_barrier(0);  // one tile's temporaries at a time
            }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const h8 v = s_v[b][d][x][lane];
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
#pragma unroll
                    for (int u = 0; u < NT; ++u)
                        r[u].o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pw[u][p][x], r[u].o[d], 0, 0, 0);
            }
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 1);
#pragma unroll
        for (int x = 0; x < 2 * DT; ++x) {
            __builtin_amdgcn_sched_group_barrier(0x008, PARTS * NT, 1);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
        }
        if (kb + 64 < key1) put(b ^ 1);
        __syncthreads();
    };

    fetch(key0);
    qs.load(a, q, row0, m_wave, m_last, lane);
#pragma unroll
    for (int u = 0; u < NT; ++u) r[u].clear();
    put(0);
    __syncthreads();
    const int vis_least = q.p0 + row_of(a, m_tile) + 1;
    int b = 0, kb = key0;
    for (; kb + 64 <= min(key1, vis_least); kb += 64, b ^= 1) step(kb, b, False{});
    for (; kb < key1; kb += 64, b ^= 1) step(kb, b, True{});

    const bool whole = q.p0 + q.n <= C;  // the sequence is one chunk
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        const float l = xor16_sum(r[u].l), unit = r[u].unit();
        int m = m_wave + 16 * u + n;
        asm("" : "+v"(m));
        const int i = row_of(a, m);
        if (m > m_last) continue;
        const int64_t row = row0 + (int64_t)i * a.nh + (m - i * a.group), part = row * a.parts + at.chunk;
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (d < ndt) {
                f4 v = r[u].o[d] * unit;
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __fdiv_rn(v[e], l);
                    store4<BF>(a.out, row * hd + 16 * d + 4 * g, v);
                } else {
                    store4<false>(a.part_o, part * hd + 16 * d + 4 * g, v);
                }
            }
        if (!whole && g == 0)
            *(float2*)(a.part_ml + 2 * part) = make_float2(r[u].ref == -__builtin_inff() ? 0.0f : r[u].ref, l);
    }
}

// ---------------------------------------------------------------------------
// k_paged_merge
// ---------------------------------------------------------------------------
// The chunks' outputs of a (row, head) weighed by 2^(m_c - max m).  Its threads are
// sets of 32 lanes, a chunk a set and 4 values a lane: W = 1: a wave a (row, head),
// for few chunks; W = 4: a workgroup, its sets' sums added in order in LDS.
// grid (rows, ceil(nh / (4 / W))), block 256.
template <int W, bool BF>
__global__ __launch_bounds__(256) void k_paged_merge(PagedAttn a)
{
    __shared__ f4 s_v[4][32];
    __shared__ float s_sum[4];
    const Paged& c = a.c;
    const int t = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = W == 1 ? 4 * blockIdx.y + wave : blockIdx.y;
    if (head >= a.nh) return;
    const int s = find_seq(c, t, lane);
    if (s < 0 || s >= c.n_seqs) return;
    const Seq q = seq_at(c, s);
    const int i = t - q.a;
    if (i < 0 || i >= q.n || !q.ok) return;
    const int C = (int64_t)q.n * a.group > a.p.lo ? a.p.tile_c : a.p.tok_c;
    if (q.p0 + q.n <= C) return;  // written by its one chunk
    const int nc = (q.p0 + i) / C + 1;  // chunks that the row sees any key of
    const int64_t r = (int64_t)t * a.nh + head, at = r * a.parts;
    float top = -__builtin_inff();
    for (int x = lane; x < nc; x += 64) top = fmaxf(top, a.part_ml[2 * (at + x)]);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    const int hd = c.hd, d = 4 * (lane & 31), set = lane >> 5;
    float sum = 0.0f;
    f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int STEP = 2 * W, U = 4;
    for (int x0 = 2 * (W == 1 ? 0 : wave) + set; x0 < nc; x0 += STEP * U) {
        f4 o[U];
        float2 ml[U];
#pragma unroll
        for (int y = 0; y < U; ++y) {
            const int64_t x = at + min(x0 + STEP * y, nc - 1);
            ml[y] = *(const float2*)(a.part_ml + 2 * x);
            o[y] = d < hd ? *(const f4*)(a.part_o + x * hd + d) : f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int y = 0; y < U; ++y)
            if (x0 + STEP * y < nc) {
                const float b = __builtin_amdgcn_exp2f(__fsub_rn(ml[y].x, top));
                sum = __fmaf_rn(b, ml[y].y, sum);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __fmaf_rn(b, o[y][e], v[e]);
            }
    }
    sum = __fadd_rn(sum, __shfl_xor(sum, 32, 64));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __fadd_rn(v[e], __shfl_xor(v[e], 32, 64));
    if (W > 1) {
        if (lane < 32) s_v[wave][lane] = v;
        if (lane == 0) s_sum[wave] = sum;
        __syncthreads();
        if (wave) return;
        for (int w = 1; w < 4; ++w) {
            sum = __fadd_rn(sum, s_sum[w]);
            v += s_v[w][lane & 31];
        }
    }
    if (lane < 32 && d < hd) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __fdiv_rn(v[e], sum);
        store4<BF>(a.out, r * hd + d, v);
    }
}

AttnPlan plan_paged_attention(int64_t n_heads, const Paged& c, bool bf)
{
    auto up = [](int64_t v, int64_t m) { return (v + m - 1) / m * m; };
    const int64_t group = n_heads / c.nkv, longest = std::max(c.cap, 1);
    AttnPlan p{};
    // one kind of launch where the bounds leave one kind of sequence
    p.lo = c.max_rows * group <= kTokRows ? INT_MAX : (c.n_seqs == 1 ? 0 : kTokRows);
    const int64_t all = up(longest, 256), heads = (int64_t)c.n_seqs * c.nkv;
    // Workgroups aimed at: two a CU where the sequences are few (one token over 100001
    // positions: 35.8 us and 5.0 for the merge with 512, 43 + 9.3 with 2048), more
    // where they are many and, as a batch's are, of different lengths (32 of up to
    // 8192: 70.1 us with 4096, 73.2 with 512).  Between the two the rule is coarse: 8
    // sequences of 8192 over 8 heads take 29.7 us with their merge, 9 take 41.1 (their
    // chunks are the shortest, 256, and the merge the wide one), 16 take 55.8.  Chunks go
    // by the host's bound: one token at 777 takes 9.2 us bounded by 2048 or less, 9.8 by
    // 8192 and 14.4 by 131072, in one chunk a head.
    const int64_t want = heads <= 64 ? 512 : 4096;
    // 512 positions are one step of eight waves: 7.4 us, and 7.2 + 3.2 in chunks; 777 are
    // two steps: 11, and 7.2 + 3.2
    p.tok_w = longest <= 512 ? 8 : 4;
    p.tok_c = (int)(p.tok_w == 8 ? all : std::min(all, up(longest * heads / want + 1, 256)));
    p.tok_n = (int)((longest + p.tok_c - 1) / p.tok_c);
    // Query rows of a tile.  64 in f32, whose two parts leave no room for 128 beside a
    // second wave a SIMD (512 rows over 8192: 194 us and 236); in bf16 128 where there
    // are many (111 us and 144), 64 where they are few (100 rows over 1500: 20 and 26).
    auto tiles_of = [&](int64_t mt) {
        const int64_t per = ((int64_t)c.max_rows * group + mt - 1) / mt;
        return std::min<int64_t>((int64_t)c.n_seqs * per, (int64_t)c.rows * group / mt + c.n_seqs);
    };
    p.tile_rows = bf && (int64_t)c.rows * n_heads >= 96 * 128 ? 128 : 64;
    p.tiles = (int)tiles_of(p.tile_rows);
    p.tile_c = (int)std::min(all, up(longest * p.tiles * c.nkv / (p.tile_rows == 128 ? 512 : 1024) + 1, 256));
    p.tile_n = (int)((longest + p.tile_c - 1) / p.tile_c);
    if (p.lo == 0) p.tok_n = 0;
    if (p.lo == INT_MAX) p.tile_n = p.tiles = 0;
    return p;
}

bool paged_attention_fits(const Paged& c, const AttnPlan& p)
{
    const int64_t threads = ((int64_t)1 << 32) - 1;  // of a grid
    return (int64_t)c.nkv * p.tok_n * c.n_seqs * 64 * p.tok_w <= threads && (int64_t)c.nkv * p.tile_n * p.tiles * 256 <= threads;
}

template <int DT, bool BF>
static hipError_t launch_attn(const PagedAttn& a, hipStream_t st)
{
    if (a.p.tok_n) {
        const dim3 grid((unsigned)(a.c.nkv * a.p.tok_n * a.c.n_seqs));
        if (a.p.tok_w == 8) hipLaunchKernelGGL((k_paged_tok<DT, 8, BF>), grid, dim3(512), 0, st, a);
        else hipLaunchKernelGGL((k_paged_tok<DT, 4, BF>), grid, dim3(256), 0, st, a);
    }
    if (a.p.tile_n) {
        const dim3 grid((unsigned)(a.c.nkv * a.p.tile_n * a.p.tiles));
        if constexpr (BF) {
            if (a.p.tile_rows == 128) hipLaunchKernelGGL((k_paged_tile<DT, 2, BF>), grid, dim3(256), 0, st, a);
        }
        if (a.p.tile_rows == 64) hipLaunchKernelGGL((k_paged_tile<DT, 1, BF>), grid, dim3(256), 0, st, a);
    }
    if (a.parts > 8)
        hipLaunchKernelGGL((k_paged_merge<4, BF>), dim3((unsigned)a.c.rows, (unsigned)a.nh), dim3(256), 0, st, a);
    else if (a.parts > 1)
        hipLaunchKernelGGL((k_paged_merge<1, BF>), dim3((unsigned)a.c.rows, (unsigned)((a.nh + 3) / 4)), dim3(256), 0, st,
                           a);
    return hipGetLastError();
}

hipError_t launch_paged_attention(const PagedAttn& a, hipStream_t st)
{
    // tiles of 16 values, in twos
    if (a.c.hd <= 32) return a.bf ? launch_attn<2, true>(a, st) : launch_attn<2, false>(a, st);
    if (a.c.hd <= 64) return a.bf ? launch_attn<4, true>(a, st) : launch_attn<4, false>(a, st);
    if (a.c.hd <= 96) return a.bf ? launch_attn<6, true>(a, st) : launch_attn<6, false>(a, st);
    return a.bf ? launch_attn<8, true>(a, st) : launch_attn<8, false>(a, st);
}

}  // namespace btl
