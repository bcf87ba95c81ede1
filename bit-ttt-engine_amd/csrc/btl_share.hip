// btl_share.hip -- gfx950 kernels of attention over a paged Q8 cache beside a prefix that
// sequences share, and of the weights that its rows give the positions.
//
// Kernels: those of btl_paged_attn.hpp in their forms for a prefix, for the sequences
// beside it and for scores that are kept, and
//   k_share, k_share_tiles      these forms side by side in one launch.
//   k_share_merge               a row's parts joined.
//   k_share_ml                  their maxima and sums alone.
//   k_account_tile              the weights of 256 positions from many rows.
//   k_account_sum               the weights from the token form's scores, or from the shares of rows.
//   k_share_finish              the merge and the weights from scores in one launch.
//
// A prefix is a batch of its own: lists of rows, each of which sees every position of its
// list's pages.  Its rows' softmax parts lie beside their sequences' own, and one merge
// joins both.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "btl_paged_attn.hpp"

namespace btl {

// ---------------------------------------------------------------------------
// k_share
// ---------------------------------------------------------------------------
// The attention of a call in one launch, the forms of btl_paged_attn.hpp side by side:
// lists of rows over the prefix (token form, or tile form), then sequences over their own
// positions (tile form, token form).  The tiles are bound by the vector unit and the
// tokens by the cache's bytes, and two workgroups a CU is what either's registers allow.
// Tiles of 128 rows, which fill all of them, have a launch of their own.
//
// Times by trace, 32 heads over 8 of 128.  64 tokens behind 8192 positions, own ones up to
// 700, bf16: 34.7 us, vector unit busy 51 %, matrix units 15 %: one prefix tile a CU waits
// for its keys and for LDS, the tokens use its other half.  32 tokens over up to 8192
// positions, scores kept, bf16: 88.0 us where the form without scores takes 75.4; with 4
// heads a KV head the scores are 16 bytes a position beside the cache's 264, put out a step
// late, behind the next step's loads (without that 98).  4 tokens behind 515, f32: 8.1 us,
// latency.
namespace {

struct ShareArgs {
    PagedAttn p;   // the prefix's
    PagedShare a;  // the sequences'
};

}  // namespace

template <int DT, bool BF, bool SCORED>
__global__ __launch_bounds__(256, 2) void k_share(ShareArgs, unsigned prefix_tok, unsigned prefix_tile,
                                                      unsigned own_tile)
{
    constexpr int NW = 4, kK = 2 * 4 * (2 * ((DT + 3) / 4)) * 64, kV = 2 * DT * 2 * 64;  // fragments of k and v
    constexpr int kO = NW * 16 * (16 * DT + 4);
    constexpr int kTile = 16 * (kK + kV) + 4 * (2 * 64 + 2 * 64 + 2), kTok = 4 * (kO + 2 * NW * 16);
    __shared__ __align__(16) uint8_t s[kTile > kTok ? kTile : kTok];
    uint8_t* const sf = s + 16 * (kK + kV);
    const TileLds<DT> tile = {(h8(*)[4][2 * ((DT + 3) / 4)][64])s, (h8(*)[DT][2][64])(s + 16 * kK), (float(*)[64])sf,
                              (float(*)[64])(sf + 512), (float*)(sf + 1024)};
    const TokLds<DT, NW> tok = {(float(*)[16][16 * DT + 4])s, (float(*)[16])(s + 4 * kO), (float(*)[16])(s + 4 * kO + 64 * NW)};
    unsigned block = blockIdx.x;
    if (block < prefix_tok) return paged_tok<DT, NW, BF, kPrefix>(kernel_args<ShareArgs>().p, block, tok);
    block -= prefix_tok;
    if (block < prefix_tile) return paged_tile<DT, 1, BF, kPrefix>(kernel_args<ShareArgs>().p, block, tile);
    block -= prefix_tile;
    if (block < own_tile) return paged_tile<DT, 1, BF, kOwn>(kernel_args<ShareArgs>().a, block, tile);
    paged_tok<DT, NW, BF, SCORED ? kScored : kOwn>(kernel_args<ShareArgs>().a, block - own_tile, tok);
}

// k_share_tiles
// Tiles of 128 rows, of lists and of sequences: the sequences' short ones fill the end of
// the prefix's (12 times up to 130 rows behind 16001, 32 heads over 8 of 128: 404 us in a
// launch each, 388 so).  With the tokens beside them a register spills.
//
// Bound by the vector unit (softmax, widening), which is busy for 65 % of that time beside
// the matrix units' 33 %; no LDS bank conflicts; 270 GFLOP, some 700 TFLOP/s.
template <int DT>
__global__ __launch_bounds__(256, 2) void k_share_tiles(ShareArgs, unsigned prefix_tile)
{
    constexpr int kK = 2 * 4 * (2 * ((DT + 3) / 4)) * 64, kV = 2 * DT * 2 * 64;  // fragments of k and v
    __shared__ __align__(16) uint8_t s[16 * (kK + kV) + 4 * (2 * 64 + 2 * 64 + 2)];
    uint8_t* const sf = s + 16 * (kK + kV);
    const TileLds<DT> tile = {(h8(*)[4][2 * ((DT + 3) / 4)][64])s, (h8(*)[DT][2][64])(s + 16 * kK), (float(*)[64])sf,
                              (float(*)[64])(sf + 512), (float*)(sf + 1024)};
    if (blockIdx.x < prefix_tile) return paged_tile<DT, 2, true, kPrefix>(kernel_args<ShareArgs>().p, blockIdx.x, tile);
    paged_tile<DT, 2, true, kOwn>(kernel_args<ShareArgs>().a, blockIdx.x - prefix_tile, tile);
}

// ---------------------------------------------------------------------------
// k_share_merge
// ---------------------------------------------------------------------------
// k_paged_merge for rows of at most U parts: half a wave a (row, head), four values a
// lane, every lane holding all the parts' maxima; N heads one after the other, so that
// what is known of the row serves them all.  grid (rows, ceil(nh / (8 N))), block 256.
//
// All a row's parts are in flight at once.  Bound by that chain (sequence, sizes, parts)
// for few rows: 64 of 32 heads 5.7 us, 4 rows 4.0.  For many by the parts' bytes, some
// 4 KB a row and head: 1025 rows of 32 heads 24 us.
namespace {

// The maximum and the sum of row r from its n parts, at most U of them.
template <int U>
__device__ __forceinline__ float2 joined(const PagedShare& a, int64_t r, int n, const Behind& p)
{
    float2 part[U ? U : 1];
    float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
    for (int y = 0; y < U; ++y)
        if (y < n) {
            part[y] = *(const float2*)(a.part_ml + 2 * (r * a.parts + (y < p.parts ? y : a.own0 - p.parts + y)));
            top = fmaxf(top, part[y].x);
        }
#pragma unroll
    for (int y = 0; y < U; ++y)
        if (y < n) sum = __fmaf_rn(__builtin_amdgcn_exp2f(__fsub_rn(part[y].x, top)), part[y].y, sum);
    return make_float2(top, p.lost ? __builtin_nanf("") : sum);
}

// ML: the row's maximum and sum are put out where they are wanted
template <int N, int U, bool BF, bool ML = true>
__device__ __forceinline__ void share_merge(const PagedShare& a, int t, int block)
{
    const Paged& c = a.c;
    const int lane = threadIdx.x & 63, d = 4 * (lane & 31), hd = c.hd;
    int s, list = -1;
    if (a.g.n_seqs && c.n_seqs < 64 && a.g.n_seqs < 64) {
        // both in the time of one: 64 starts of each at once
        const int v = lane <= c.n_seqs ? c.row_start[lane] : INT_MAX, w = lane <= a.g.n_seqs ? a.g.row_start[lane] : INT_MAX;
        s = 63 - __clzll(__ballot(lane <= c.n_seqs && v <= t));
        list = 63 - __clzll(__ballot(lane <= a.g.n_seqs && w <= t));
    } else {
        s = find_seq(c, t, lane);
        if (a.g.n_seqs) list = find_seq(a.g, t, lane);
    }
    if (s < 0 || s >= c.n_seqs) return;
    const Seq q = seq_at(c, s);
    const Behind p = behind_of(a, t, list);
    const int i = t - q.a;
    if (i < 0 || i >= q.n || !q.ok) return;
    const int C = (int64_t)q.n * a.group > a.p.lo ? a.p.tile_c : a.p.tok_c;
    if (whole_of<kOwn>(a, q.p0 + q.n, C)) return;  // written by its one chunk
    const int nc = p.parts + (q.p0 + i) / C + 1;
#pragma unroll
    for (int x = 0; x < N; ++x) {
        const int head = block * 8 * N + 8 * x + (int)(threadIdx.x >> 5);
        if (head >= a.nh) return;
        const int64_t r = (int64_t)t * a.nh + head, at = r * a.parts;
        float2 ml[U];
        f4 o[U];
#pragma unroll
        for (int y = 0; y < U; ++y)
            if (y < nc) {
                const int64_t part = at + (y < p.parts ? y : a.own0 - p.parts + y);
                ml[y] = *(const float2*)(a.part_ml + 2 * part);
                o[y] = *(const f4*)(a.part_o + part * hd + (d < hd ? d : 0));
            }
        float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (int y = 0; y < U; ++y)
            if (y < nc) top = fmaxf(top, ml[y].x);
        f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int y = 0; y < U; ++y)
            if (y < nc) {
                const float b = __builtin_amdgcn_exp2f(__fsub_rn(ml[y].x, top));
                sum = __fmaf_rn(b, ml[y].y, sum);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __fmaf_rn(b, o[y][e], v[e]);
            }
        if (p.lost) sum = __builtin_nanf("");
        if (ML && a.ml && d == 0) *(float2*)(a.ml + 2 * r) = make_float2(top, sum);
        if (d < hd) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __fdiv_rn(v[e], sum);
            store4<BF>(a.out, r * hd + d, v);
        }
    }
}

}  // namespace

template <int N, int U, bool BF>
__global__ __launch_bounds__(256) void k_share_merge(PagedShare a)
{
    share_merge<N, U, BF>(a, blockIdx.x, blockIdx.y);
}

// ---------------------------------------------------------------------------
// k_share_ml
// ---------------------------------------------------------------------------
// The rows' maxima and sums alone, as k_share_merge forms them, so that k_account_tile need
// not wait for their outputs, which are joined in its launch.  A wave a row, a head a lane.
// grid ceil(rows / 4), block 256.
//
// Bound by latency: 4.7 us for 1000 rows of 32 heads, where the whole merge takes 11.4.  With
// the weights 169.0 us in all before, 166.2 so; 14 sequences of few or 201 rows 44.6 and 43.3.
template <int U>
__global__ __launch_bounds__(256) void k_share_ml(PagedShare a)
{
    const Paged& c = a.c;
    const int lane = threadIdx.x & 63, t = 4 * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= c.rows) return;
    const int s = find_seq(c, t, lane);
    if (s < 0 || s >= c.n_seqs) return;
    const Seq q = seq_at(c, s);
    const Behind p = behind(a, t, lane);
    const int i = t - q.a;
    if (i < 0 || i >= q.n || !q.ok) return;
    const int C = (int64_t)q.n * a.group > a.p.lo ? a.p.tile_c : a.p.tok_c;
    if (whole_of<kOwn>(a, q.p0 + q.n, C)) return;  // put out by its one chunk
    const int nc = p.parts + (q.p0 + i) / C + 1;
    for (int head = lane; head < a.nh; head += 64) {
        const int64_t r = (int64_t)t * a.nh + head;
        *(float2*)(a.ml + 2 * r) = joined<U>(a, r, nc, p);
    }
}

// ---------------------------------------------------------------------------
// k_account_tile
// ---------------------------------------------------------------------------
// weight[j] = sum over the rows that see j of 2^(s - m) / l, with the rows' m and l from
// the attention before it.  A wave holds 64 keys as the attention's first product takes
// them (four key tiles, widened once) and goes through a share of the sequence's rows, 16
// at a time: S^T = K . Q^T, a weight a score, and 16 sums a lane.  The rows lie in LDS as
// operand fragments, 64 at a time, one tile put there by each wave.
//
// Queries of bf16 are taken as they are, against codes in bf16 (exact) times 2^-20, so
// that no product overflows; of f32 in two f16 parts as the attention takes them.
//
// Half the attention's products, no value, and no reference to follow: a fused operation,
// an exponential and another fused one a score.  Bound by the vector unit (busy 75 %, the
// matrix units 23 %): 1000 rows over 4099 positions, 32 heads over 8 of 128, bf16, 63 us by
// trace with the rows' merges beside it, 59 and 500 TFLOP/s without.  Three workgroups a CU, and
// rows asked for a step ahead: in passes in a row some 45 us so, 61 with rows read when they are
// wanted, 78 at two workgroups.  Keys in LDS and rows in registers would need the sums across
// rows at every step, not at the end.
//
// grid nkv * ceil(cap / 256) * splits * n_seqs, block 256; behind them, where k_share_ml has
// put out the rows' maxima and sums, the merges of rows of at most 8 parts.
namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// Codes times this are what a bf16 query meets: 2^128 of a query times 128 values of
// 2^7 would pass the largest f32.
constexpr float kCodeDown = 1.0f / (1 << 20);

// eight codes -> eight bf16 (code - 128) * kCodeDown
__device__ __forceinline__ u4 widen8_bf(uint32_t w0, uint32_t w1)
{
    auto two = [](uint32_t w) {
        const float lo = ((float)(w & 255u) - 128.0f) * kCodeDown, hi = ((float)(w >> 8 & 255u) - 128.0f) * kCodeDown;
        return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
    };
    return u4{two(w0), two(w0 >> 16), two(w1), two(w1 >> 16)};
}

template <bool BF>
__device__ __forceinline__ f4 product(u4 k, u4 q, f4 c)
{
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, k), __builtin_bit_cast(b8, q), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, k), __builtin_bit_cast(h8, q), c, 0, 0, 0);
}

// a sequence's weights come from the scores that the token form kept
__device__ __forceinline__ bool has_scores(const PagedShare& a, int64_t M) { return a.scored && M <= a.p.lo; }

// The weight of a position from this call: added to what rows before this call gave it,
// or, of the rows' own positions, the first.
__device__ __forceinline__ void put_weight(const PagedShare& a, const Seq& q, int s, int h, int key, float w)
{
    float* p = a.weight + ((int64_t)s * a.c.nkv + h) * a.ld + key;
    *p = key < q.p0 ? __fadd_rn(*p, w) : w;
}

}  // namespace

template <int DT, bool BF>
__global__ __launch_bounds__(256, BF ? 3 : 2) void k_account_tile(PagedShare a, unsigned blocks_of_keys)
{
    constexpr int NJ = (DT + 3) / 4;
    constexpr int PARTS = BF ? 1 : 2;
    __shared__ __align__(16) u4 s_q[2][4][PARTS * 2 * NJ][64];
    __shared__ float2 s_r[2][4][16];           // a row's maximum and 1 / sum
    __shared__ float s_unit[2][4][BF ? 1 : 16];  // the unit of its products
    __shared__ int s_bad[2][4];       // a tile has rows that came back as NaN
    const Paged& c = a.c;
    if (blockIdx.x >= blocks_of_keys) {
        const unsigned block = blockIdx.x - blocks_of_keys;
        return share_merge<1, 8, BF, false>(a, (int)(block % (unsigned)c.rows), (int)(block / (unsigned)c.rows));
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15, hd = c.hd, ndt = hd >> 4;
    // workgroup -> head, block of 256 positions, share of the rows, sequence
    const int h = (int)(blockIdx.x % (unsigned)c.nkv);
    unsigned at = blockIdx.x / (unsigned)c.nkv;
    const unsigned blocks = (unsigned)(c.cap + 255) / 256;
    const int block = (int)(at % blocks);
    at /= blocks;
    const int share = (int)(at % (unsigned)a.splits), s = (int)(at / (unsigned)a.splits);
    const Seq q = seq_at(c, s);
    const int64_t M = (int64_t)q.n * a.group;
    const int key0 = 256 * block, seen = q.p0 + q.n;
    if (M == 0 || !q.ok || has_scores(a, M) || key0 >= seen) return;

    // this wave's keys: 64 from kb on
    const int kb = key0 + 64 * wave;
    const int32_t* table = c.pages + (int64_t)s * c.max_pages;
    Slots slots;
    slots.find(c, table, key0 >> 4, (seen - 1) >> 4, h, lane);
    const int own = slots.of((kb >> 4) + g), at_k = max(slots.of((kb >> 4) + (n >> 2)), 0);
    const uint8_t* kp = c.k + (uint64_t)(uint32_t)at_k * (uint32_t)(16 * hd) + (n & 3) * hd;
    u4 k[4][2 * NJ];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            // past the head's width the queries are zero
            const u4 w = *(const u4*)(kp + 4 * t * hd + 16 * (4 * j + g < ndt ? 4 * j + g : 0));
            if constexpr (BF) {
                k[t][2 * j] = widen8_bf(w.x, w.y);
                k[t][2 * j + 1] = widen8_bf(w.z, w.w);
            } else {
                k[t][2 * j] = __builtin_bit_cast(u4, widen8(w.x, w.y));
                k[t][2 * j + 1] = __builtin_bit_cast(u4, widen8(w.z, w.w));
            }
        }
    f4 ks[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) ks[t] = *(const f4*)(c.ks + 16 * (int64_t)max(own, 0) + 4 * t) * a.scale_log2;

    // the rows from the first that sees the block's first key on, this workgroup's share of them
    const int first = max(0, key0 - q.p0) * a.group & ~15;
    const int steps = ((int)M - first + 63) / 64;
    const int step0 = (int)((int64_t)steps * share / a.splits), step1 = (int)((int64_t)steps * (share + 1) / a.splits);
    const int64_t row0 = (int64_t)q.a * a.nh + h * a.group;
    // this wave's tile of a step: asked for ahead of the work on the step before it
    constexpr int PER = BF ? 2 : 4;  // 16-byte pieces of 16 values
    u4 raw[PER * NJ];
    float2 ml;
    auto fetch = [&](int step) {
        const int mm = min(first + 64 * step + 16 * wave + n, (int)M - 1), i = row_of(a, mm);
        const int64_t row = row0 + (int64_t)i * a.nh + (mm - i * a.group);
        ml = *(const float2*)(a.ml + 2 * row);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int d = 16 * (4 * j + g);
            const u4* p = (const u4*)((const uint8_t*)a.q + (row * hd + (d < hd ? d : 0)) * (BF ? 2 : 4));
#pragma unroll
            for (int x = 0; x < PER; ++x) raw[PER * j + x] = p[x];
        }
    };
    auto put = [&](int step, int b) {
        if constexpr (BF) {
#pragma unroll
            for (int x = 0; x < 2 * NJ; ++x) s_q[b][wave][x][lane] = 16 * (4 * (x >> 1) + g) < hd ? raw[x] : u4{0, 0, 0, 0};
        } else {
            // in two f16 parts, as the attention takes them
            float f[NJ][16];
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    f[j][x] = 16 * (4 * j + g) < hd ? __uint_as_float(raw[4 * j + (x >> 2)][x & 3]) : 0.0f;
            h8 parts[2][2 * NJ];
            const float unit = in_parts<NJ, 2>(f, 1.0f, [&](int p, int x, int e, _Float16 y) { parts[p][x][e] = y; });
            if (g == 0) s_unit[b][wave][n] = unit;
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int j = 0; j < 2 * NJ; ++j) s_q[b][wave][2 * NJ * p + j][lane] = __builtin_bit_cast(u4, parts[p][j]);
        }
        // a row that came back as NaN adds nothing (-1 says so), nor does one behind the last (0)
        const bool good = ml.y > 0.0f && ml.y < __builtin_inff(), real = first + 64 * step + 16 * wave + n < M;
        const float part = !good ? -1.0f : (real ? __fdiv_rn(1.0f, ml.y) : 0.0f);
        if (g == 0) s_r[b][wave][n] = make_float2(ml.x, part);
        const bool some = __any(!good);
        if (lane == 0) s_bad[b][wave] = some;
    };

    float sum[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) sum[x] = 0.0f;
    if (step0 < step1) {
        fetch(step0);
        put(step0, 0);
    }
    __syncthreads();
    for (int step = step0, b = 0; step < step1; ++step, b ^= 1) {
        if (step + 1 < step1) fetch(step + 1);
        // the scores of tile u, less the row's largest, in the order and the roundings of the attention
        auto scores = [&](int u, float top, f4* sc) {
            const float unit = BF ? 1.0f / kCodeDown : s_unit[b][u][BF ? 0 : n];
#pragma unroll
            for (int t = 0; t < 4; ++t) sc[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 2 * NJ; ++j)
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    const u4 x = s_q[b][u][2 * NJ * p + j][lane];
#pragma unroll
                    for (int t = 0; t < 4; ++t) sc[t] = product<BF>(k[t][j], x, sc[t]);
                }
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[t][e] = __fmaf_rn(__fmul_rn(sc[t][e], ks[t][e]), unit, -top);
        };
        const int bad = __builtin_amdgcn_readfirstlane(s_bad[b][0] | s_bad[b][1] | s_bad[b][2] | s_bad[b][3]);
        const int m0 = first + 64 * step;
        const bool all = kb + 64 <= q.p0 + row_of(a, m0) + 1;  // the step's first row sees every key
        if (all && !bad) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                f4 sc[4];
                const float2 r = s_r[b][u][n];
                scores(u, r.x, sc);
#pragma unroll
                for (int x = 0; x < 16; ++x) sum[x] = __fmaf_rn(__builtin_amdgcn_exp2f(sc[x >> 2][x & 3]), r.y, sum[x]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                f4 sc[4];
                const float2 r = s_r[b][u][n];
                scores(u, r.x, sc);
                const int vis = q.p0 + row_of(a, min(m0 + 16 * u + n, (int)M - 1)) + 1 - kb - 16 * g;
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float p = __fmul_rn(__builtin_amdgcn_exp2f(sc[x >> 2][x & 3]), r.y);
                    sum[x] = __fadd_rn(sum[x], x < vis && r.y > 0.0f ? p : 0.0f);
                }
                __builtin_amdgcn_sched_barrier(0);  // one tile's temporaries at a time
            }
        }
        if (step + 1 < step1) put(step + 1, b ^ 1);
        __syncthreads();
    }

    // over the 16 rows; lane 16 g + n puts out key 16 g + n
    float w = 0.0f;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
        float v = sum[x];
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) v = __fadd_rn(v, __shfl_xor(v, off, 64));
        w = n == x ? v : w;
    }
    if (kb + lane >= seen) return;
    // at most 1 a row, also where the products hold what the attention's scaled queries lost (bf16 ones
    // below 2^-31 of their row's largest) and a score is far above all that the row's sum is of
    w = fminf(w, (float)max(min(64 * (step1 - step0), (int)M - first - 64 * step0), 0));
    if (a.splits == 1) put_weight(a, q, s, h, kb + lane, w);
    else a.sums[(((int64_t)share * c.n_seqs + s) * c.nkv + h) * a.score_ld + kb + lane] = w;
}

// ---------------------------------------------------------------------------
// k_account_sum
// ---------------------------------------------------------------------------
// Four positions a thread: the weights from the scores of at most 16 rows, or the sum of
// the shares of k_account_tile, in order.  grid nkv * ceil(cap / 1024) * n_seqs, block 256.
// U: the rows' maxima and sums are taken from their parts, at most U of them, beside the
// merge that does the same (0: they lie in a.ml).
// Bound by latency (row sizes, maxima, scores): 777 positions 4.2 us with the merge beside
// it, 32 sequences of up to 8192 12.6 us for 21 MB of scores and 10 MB of weights.
namespace {

template <int U>
__device__ __forceinline__ void account_sum(const PagedShare& a, unsigned block)
{
    __shared__ float2 s_ml[kTokRows];
    const Paged& c = a.c;
    const int h = (int)(block % (unsigned)c.nkv);
    const unsigned at = block / (unsigned)c.nkv, blocks = (unsigned)(c.cap + 1023) / 1024;
    const int key0 = 1024 * (int)(at % blocks), key = key0 + 4 * (int)threadIdx.x, s = (int)(at / blocks);
    const Seq q = seq_at(c, s);
    const int64_t M = (int64_t)q.n * a.group, head = (int64_t)s * c.nkv + h, row0 = (int64_t)q.a * a.nh + h * a.group;
    const int seen = q.p0 + q.n;
    if (M == 0 || !q.ok || key0 >= seen) return;
    const bool scores = has_scores(a, M);
    if (!scores && a.splits == 1) return;  // put out where they were summed
    if (scores) {
        const int lane = threadIdx.x & 63;
        for (int i = threadIdx.x >> 6; i < q.n; i += 4) {
            const int64_t r = row0 + (int64_t)i * a.nh + min(lane, a.group - 1);
            const bool whole = U == 0 || whole_of<kOwn>(a, seen, a.p.tok_c);
            const Behind p = whole ? Behind{} : behind(a, q.a + i, lane);
            float2 ml;
            if (whole) {
                ml = *(const float2*)(a.ml + 2 * r);
            } else {
                ml = joined<U>(a, r, p.parts + (q.p0 + i) / a.p.tok_c + 1, p);
            }
            // a row that came back as NaN adds nothing
            const bool good = ml.y > 0.0f && ml.y < __builtin_inff();
            if (lane < a.group) s_ml[i * a.group + lane] = make_float2(ml.x, good ? __fdiv_rn(1.0f, ml.y) : 0.0f);
        }
        __syncthreads();
    }
    if (key >= seen) return;
    float* to = a.weight + head * a.ld + key;
    const bool four = key + 4 <= a.ld;
    Four old = {};  // asked for beside the scores
    if (four) old = *(const Four*)to;
    f4 w = {0.0f, 0.0f, 0.0f, 0.0f};
    if (scores) {
        const float* sc = a.scores + head * a.score_rows * a.score_ld + key;
        constexpr int V = 4;  // rows at a time
        for (int m0 = 0; m0 < (int)M; m0 += V) {
            f4 y[V];
#pragma unroll
            for (int u = 0; u < V; ++u) y[u] = *(const f4*)(sc + (int64_t)min(m0 + u, (int)M - 1) * a.score_ld);
#pragma unroll
            for (int u = 0; u < V; ++u) {
                const float2 ml = s_ml[min(m0 + u, (int)M - 1)];
                const bool good = m0 + u < (int)M && ml.y > 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __builtin_amdgcn_exp2f(__fsub_rn(y[u][e], ml.x));
                    w[e] = good ? __fmaf_rn(p, ml.y, w[e]) : w[e];
                }
            }
        }
    } else {
        constexpr int V = 8;  // shares at a time
        const float* from = a.sums + head * a.score_ld + key;
        const int64_t step = (int64_t)c.n_seqs * c.nkv * a.score_ld;
        for (int x0 = 0; x0 < a.splits; x0 += V) {
            f4 y[V];
#pragma unroll
            for (int u = 0; u < V; ++u) y[u] = *(const f4*)(from + min(x0 + u, a.splits - 1) * step);
#pragma unroll
            for (int u = 0; u < V; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = x0 + u < a.splits ? __fadd_rn(w[e], y[u][e]) : w[e];
        }
    }
    if (four && key + 4 <= seen) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            old.v[e] = key + e < q.p0 ? __float_as_uint(__fadd_rn(__uint_as_float(old.v[e]), w[e])) : __float_as_uint(w[e]);
        *(Four*)to = old;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (key + e < seen) put_weight(a, q, s, h, key + e, w[e]);
}

}  // namespace

__global__ __launch_bounds__(256) void k_account_sum(PagedShare a) { account_sum<0>(a, blockIdx.x); }

// The merge and the weights from the token form's scores in one launch, where nothing else
// is to be done between them.  grid merge + nkv * ceil(cap / 1024) * n_seqs, block 256.
template <int U, bool BF>
__global__ __launch_bounds__(256) void k_share_finish(PagedShare a, unsigned merge)
{
    if (blockIdx.x < merge) share_merge<1, U, BF>(a, (int)(blockIdx.x % (unsigned)a.c.rows), (int)(blockIdx.x / (unsigned)a.c.rows));
    else account_sum<U>(a, blockIdx.x - merge);
}

bool plan_paged_share(int64_t n_heads, PagedShare& a, bool bf, bool account)
{
    auto up = [](int64_t v, int64_t m) { return (v + m - 1) / m * m; };
    const Paged &c = a.c, &g = a.g;
    const int64_t group = n_heads / c.nkv, heads = (int64_t)c.n_seqs * c.nkv, longest = std::max(c.cap, 1);
    a.split = g.n_seqs > 0;
    AttnPlan& p = a.p;
    p = plan_paged_attention(n_heads, c, bf);
    // scores of a batch whose bounds are far above its lengths would be a large workspace:
    // above 1 GiB the keys are gone through again
    a.scored = account && p.lo > 0 &&
               heads * std::min<int64_t>(kTokRows, c.max_rows * group) * up(longest, 64) <= ((int64_t)1 << 28);
    // Sequences of at most 512 positions, their scores kept and nothing beside them, in one
    // launch of eight waves.  Else four waves.  Beside a prefix, whose tiles fill the chip as
    // well, chunks for 512 workgroups: behind 8192 positions 64 sequences of up to 700 40.2 us where
    // btl_serve.hip's 4096 take 46.8, 32 of up to 4000 60.3 and 72.9 (256: 37.8 and 61.6; 1024: 45.6
    // and 63.1).
    const bool apart = p.tok_w == 8 && p.tok_n && a.scored && !a.split && !p.tile_n;
    if (!apart) p.tok_w = 4;
    if (!apart && p.tok_n) {
        const int64_t want = a.split || heads <= 64 ? 512 : 4096;
        p.tok_c = (int)std::min(up(longest, 256), up(longest * heads / want + 1, 256));
        p.tok_n = (int)((longest + p.tok_c - 1) / p.tok_c);
    }
    a.own0 = 0;
    a.gp = AttnPlan{};
    if (a.split) {
        // One form for all lists: the token form, in tiles of 16 rows, where every list is of at most
        // two (8 rows of 4 heads behind 4000 positions: 15.8 us, 16.8 in the tile form, in f32 15.0 and
        // 17.2).  Of three it would be 16.3 and 17.4, of four 16.4 and 17.9, of five 21.4 and 19.9: the
        // rule could go up to four.  In chunks for 256 workgroups (8 sequences behind 16000: 21.9 us,
        // 24.3 with 192, 24.8 with 512).
        AttnPlan& r = a.gp;
        const int64_t far = std::max(g.cap, 1), all = up(far, 256);
        r.tok_w = 4;
        const int64_t per_list = (int64_t)g.max_rows * group;
        r.lo = per_list <= 2 * kTokRows ? INT_MAX : 0;
        r.tile_rows = p.tile_rows;
        r.tok_c = r.tile_c = (int)all;
        if (r.lo) {
            r.tiles = (int)std::max<int64_t>(1, (per_list + 15) / 16);
            r.tok_c = (int)std::min(all, up(far * g.n_seqs * g.nkv * r.tiles / 256 + 1, 256));
            r.tok_n = (int)((far + r.tok_c - 1) / r.tok_c);
        } else {
            // Chunks so that there are about 256 workgroups, one a CU beside the sequences' own (64
            // tokens behind 8192 positions: 39.9 us, 45.0 with 192, 46.4 with 512, 55.4 with 1024);
            // of many tiles 2048, as long as a chunk has 2048 positions (12 times up to 130 rows behind
            // 16001: 389 us; chunks of some 1100 430, of 4000 413, of 8000 495).
            const int64_t per = (per_list + r.tile_rows - 1) / r.tile_rows;
            r.tiles = (int)std::min<int64_t>((int64_t)g.n_seqs * per, (int64_t)g.rows * group / r.tile_rows + g.n_seqs);
            const int64_t base = (int64_t)r.tiles * g.nkv;
            const int64_t n = std::max<int64_t>({1, (256 + base / 2) / base, std::min(far / 2048, (2048 + base - 1) / base)});
            r.tile_c = (int)std::max<int64_t>(256, up((far + n - 1) / n, 64));
            r.tile_n = (int)((far + r.tile_c - 1) / r.tile_c);
        }
        a.own0 = r.parts();
    }
    a.parts = a.own0 + p.parts();
    a.splits = 1;
    const int64_t threads = ((int64_t)1 << 32) - 1;  // of a grid
    const int64_t blocks = (int64_t)c.nkv * p.tok_n * c.n_seqs + (int64_t)c.nkv * p.tile_n * p.tiles +
                           (int64_t)g.nkv * (a.gp.tok_n * (int64_t)g.n_seqs + a.gp.tile_n) * a.gp.tiles;
    if (blocks * 64 * p.tok_w > threads) return false;
    if (!account) return true;

    a.score_rows = (int)std::min<int64_t>(kTokRows, (int64_t)c.max_rows * group);
    a.score_ld = (int)up(c.cap, 64);
    // k_account_tile's rows in shares of at least 256, for some 2048 workgroups: of the sequences
    // that the bounds allow to be long, few may be (two of 14: 44.4 us, 49.0 for 768).
    const bool tiles = p.lo != INT_MAX || !a.scored;
    const int64_t seqs = !tiles ? 0 : (a.scored ? std::min<int64_t>(c.n_seqs, (int64_t)c.rows * group / 16 + 1) : c.n_seqs);
    const int64_t keys = (c.cap + 255) / 256, have = std::max<int64_t>(1, seqs * c.nkv * keys);
    a.splits = (int)std::max<int64_t>(1, std::min<int64_t>({2048 / have, 16, (int64_t)c.max_rows * group / 256}));
    return heads * keys * 256 * (tiles ? a.splits : 1) <= threads;
}

template <int DT, bool BF>
static hipError_t launch_share(const PagedShare& a, hipStream_t st)
{
    const bool prefix = a.g.n_seqs && a.g.cap;
    const unsigned prefix_tok = prefix ? (unsigned)(a.g.nkv * a.gp.tok_n * a.g.n_seqs * a.gp.tiles) : 0;
    unsigned prefix_tile = prefix ? (unsigned)(a.g.nkv * a.gp.tile_n * a.gp.tiles) : 0;
    unsigned own_tile = (unsigned)(a.c.nkv * a.p.tile_n * a.p.tiles);
    const unsigned own_tok = (unsigned)(a.c.nkv * a.p.tok_n * a.c.n_seqs);
    ShareArgs args = {a, a};
    args.p.c = a.g;
    args.p.p = a.gp;
    if constexpr (BF) {
        if (a.p.tile_rows == 128) {
            if (prefix_tile + own_tile)
                hipLaunchKernelGGL((k_share_tiles<DT>), dim3(prefix_tile + own_tile), dim3(256), 0, st, args, prefix_tile);
            prefix_tile = own_tile = 0;
        }
    }
    auto go = [&](auto k) {
        const unsigned all = prefix_tok + prefix_tile + own_tile + own_tok;
        if (all) hipLaunchKernelGGL(k, dim3(all), dim3(256), 0, st, args, prefix_tok, prefix_tile, own_tile);
    };
    if (a.p.tok_w == 8) hipLaunchKernelGGL((k_paged_tok<DT, 8, BF, kScored>), dim3(own_tok), dim3(512), 0, st, a);
    else if (a.weight && a.scored) go(k_share<DT, BF, true>);
    else go(k_share<DT, BF, false>);
    const bool account = a.weight && a.c.cap, tiles = a.p.lo != INT_MAX || !a.scored;
    const unsigned heads = (unsigned)(a.c.nkv * a.c.n_seqs), sums = heads * ((a.c.cap + 1023) / 1024);
    const dim3 one((unsigned)a.c.rows, (unsigned)((a.nh + 7) / 8)), four((unsigned)a.c.rows, (unsigned)((a.nh + 31) / 32));
    // of both kinds of blocks fewer than a grid of 2^32 threads has: 2^21 rows of 64 heads are as many
    const bool fits = (int64_t)one.x * one.y + sums < (int64_t)1 << 24;
    if (account && !tiles && fits && a.parts > 1 && a.parts <= 16) {
        const unsigned merge = one.x * one.y;
        if (a.parts > 8) hipLaunchKernelGGL((k_share_finish<16, BF>), dim3(merge + sums), dim3(256), 0, st, a, merge);
        else hipLaunchKernelGGL((k_share_finish<8, BF>), dim3(merge + sums), dim3(256), 0, st, a, merge);
        return hipGetLastError();
    }
    const int64_t keys = (int64_t)heads * ((a.c.cap + 255) / 256) * a.splits, merges = (int64_t)one.x * one.y;
    const bool beside = account && tiles && a.parts > 1 && a.parts <= 8 && keys + merges < (int64_t)1 << 24;
    if (beside)
        hipLaunchKernelGGL(k_share_ml<8>, dim3((unsigned)(a.c.rows + 3) / 4), dim3(256), 0, st, a);
    else if (a.parts > 16)
        hipLaunchKernelGGL((k_paged_merge<4, BF, kOwn>), dim3((unsigned)a.c.rows, (unsigned)a.nh), dim3(256), 0, st, a);
    else if (a.parts > 8)
        hipLaunchKernelGGL((k_share_merge<1, 16, BF>), one, dim3(256), 0, st, a);
    else if (a.parts > 1 && (int64_t)a.c.rows * a.nh > 8192)
        hipLaunchKernelGGL((k_share_merge<4, 8, BF>), four, dim3(256), 0, st, a);
    else if (a.parts > 1)
        hipLaunchKernelGGL((k_share_merge<1, 8, BF>), one, dim3(256), 0, st, a);
    if (account) {
        if (tiles)
            hipLaunchKernelGGL((k_account_tile<DT, BF>), dim3((unsigned)(keys + (beside ? merges : 0))), dim3(256), 0, st, a,
                               (unsigned)keys);
        if (a.scored || a.splits > 1) hipLaunchKernelGGL(k_account_sum, dim3(sums), dim3(256), 0, st, a);
    }
    return hipGetLastError();
}

hipError_t launch_paged_share(const PagedShare& a, hipStream_t st)
{
    if (a.c.hd <= 32) return a.bf ? launch_share<2, true>(a, st) : launch_share<2, false>(a, st);
    if (a.c.hd <= 64) return a.bf ? launch_share<4, true>(a, st) : launch_share<4, false>(a, st);
    if (a.c.hd <= 96) return a.bf ? launch_share<6, true>(a, st) : launch_share<6, false>(a, st);
    return a.bf ? launch_share<8, true>(a, st) : launch_share<8, false>(a, st);
}

}  // namespace btl
