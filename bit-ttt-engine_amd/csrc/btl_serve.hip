// btl_serve.hip -- gfx950 kernels of a batch of sequences over a paged Q8 cache:
// RoPE and append, reading back, attention.
//
// Kernels:
//   k_paged_append   RoPE of the new q and k rows, Q8 of k and v into their slots.
//   k_paged_read     rows of the cache dequantised.
// and those of btl_paged_attn.hpp in their form for a batch:
//   k_paged_tok, k_paged_tile   attention of rows over a chunk of keys.
//   k_paged_merge               the chunks of a row merged.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "btl_paged_attn.hpp"

namespace btl {

namespace {

// the RoPE position of a sequence's position
__device__ __forceinline__ int64_t rope_pos(const PagedAppend& a, int s, int pos)
{
    return (int64_t)pos + (a.shift ? a.shift[s] : 0);
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
    const int64_t turn = rope_pos(a, s, pos);
    const bool good = q.ok && turn >= 0 && turn < a.rope_len;
    int grp = 0, page = -1;
    float c = 0.0f, w = 0.0f;
    if (good) {
        page = page_of(a.c, a.c.pages + (int64_t)s * a.c.max_pages, pos >> 4, &grp);
        if (act) {
            c = a.cos_t[turn * half + lane];
            w = a.sin_t[turn * half + lane];
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
        const int64_t turn = rope_pos(a, s, pos);
        if (q.ok && turn >= 0 && turn < a.rope_len) {
            co = *(const float2*)(a.cos_t + turn * half + 2 * m);
            si = *(const float2*)(a.sin_t + turn * half + 2 * m);
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
    const int64_t turn = rope_pos(a, s, 16 * grp);  // of the group's first position
    const int r0 = max(max(0, -i0), (int)max(min(-turn, (int64_t)16), (int64_t)0));
    const int r1 = min(min(16, q.n - i0), (int)max(min(a.rope_len - turn, (int64_t)16), (int64_t)0));
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
            co[b] = *(const float2*)(a.cos_t + (turn + r) * half + 2 * m);
            si[b] = *(const float2*)(a.sin_t + (turn + r) * half + 2 * m);
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
// Attention (btl_paged_attn.hpp)
// ---------------------------------------------------------------------------
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
