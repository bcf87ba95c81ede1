// btl_share.hip -- gfx950 kernels of attention over a paged Q8 cache beside a prefix that
// sequences share, and of the weights that its rows give the positions.
//
// Kernels: those of btl_paged_attn.hpp in their forms for a prefix, for the sequences
// beside it and for scores that are kept, and
//   k_account_tile   the weights of 256 positions from many rows.
//   k_account_sum    the weights from the token form's scores, or from the shares of rows.
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
// grid nkv * ceil(cap / 256) * splits * n_seqs, block 256.
namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

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
__global__ __launch_bounds__(256, 2) void k_account_tile(PagedShare a)
{
    constexpr int NJ = (DT + 3) / 4;
    constexpr int PARTS = BF ? 1 : 2;
    __shared__ __align__(16) u4 s_q[2][4][PARTS * 2 * NJ][64];
    __shared__ float4 s_r[2][4][16];  // a row's unit of the product, maximum and 1 / sum
    const Paged& c = a.c;
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
    for (int t = 0; t < 4; ++t) ks[t] = *(const f4*)(c.ks + 16 * (int64_t)max(own, 0) + 4 * t);

    // the rows from the first that sees the block's first key on, this workgroup's share of them
    const int first = max(0, key0 - q.p0) * a.group & ~15;
    const int steps = ((int)M - first + 63) / 64;
    const int step0 = (int)((int64_t)steps * share / a.splits), step1 = (int)((int64_t)steps * (share + 1) / a.splits);
    const int64_t row0 = (int64_t)q.a * a.nh + h * a.group;
    auto put = [&](int step, int b) {
        const int m = first + 64 * step + 16 * wave + n, mm = min(m, (int)M - 1);
        const int i = row_of(a, mm);
        const int64_t row = row0 + (int64_t)i * a.nh + (mm - i * a.group);
        const float2 ml = *(const float2*)(a.ml + 2 * row);
        float unit;
        if constexpr (BF) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int d = 16 * (4 * j + g);
                const u4* p = (const u4*)((const uint16_t*)a.q + row * hd + (d < hd ? d : 0));
                const u4 w0 = p[0], w1 = p[1], none = {0, 0, 0, 0};
                s_q[b][wave][2 * j][lane] = d < hd ? w0 : none;
                s_q[b][wave][2 * j + 1][lane] = d < hd ? w1 : none;
            }
            unit = a.scale_log2 / kCodeDown;
        } else {
            Queries<NJ, 1, false> qs;
            qs.load(a, q, row0, first + 64 * step + 16 * wave, (int)M - 1, lane);
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int j = 0; j < 2 * NJ; ++j)
                    s_q[b][wave][2 * NJ * p + j][lane] = __builtin_bit_cast(u4, qs.v[p][0][j]);
            unit = qs.cq[0];
        }
        // a row that came back as NaN adds nothing (-1 says so), nor does one behind the last (0)
        const bool good = ml.y > 0.0f && ml.y < __builtin_inff();
        const float part = !good ? -1.0f : (m < M ? __fdiv_rn(1.0f, ml.y) : 0.0f);
        if (g == 0) s_r[b][wave][n] = make_float4(unit, ml.x, part, 0.0f);
    };

    float sum[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) sum[x] = 0.0f;
    if (step0 < step1) put(step0, 0);
    __syncthreads();
    for (int step = step0, b = 0; step < step1; ++step, b ^= 1) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            f4 sc[4];
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
            const float4 r = s_r[b][u][n];
            // the score in the roundings of the attention, whose largest is r.y
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sc[t][e] = __fsub_rn(__fmul_rn(__fmul_rn(sc[t][e], ks[t][e]), r.x), r.y);
            const int m = first + 64 * step + 16 * u;
            const bool all = kb + 64 <= q.p0 + row_of(a, m) + 1;  // the tile's first row sees every key
            if (!all || __any(r.z < 0.0f)) {
                const int vis = q.p0 + row_of(a, min(m + n, (int)M - 1)) + 1 - kb - 16 * g;
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float p = __fmul_rn(__builtin_amdgcn_exp2f(sc[x >> 2][x & 3]), r.z);
                    sum[x] = __fadd_rn(sum[x], x < vis && r.z > 0.0f ? p : 0.0f);
                }
            } else {
#pragma unroll
                for (int x = 0; x < 16; ++x) sum[x] = __fmaf_rn(__builtin_amdgcn_exp2f(sc[x >> 2][x & 3]), r.z, sum[x]);
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
    if (a.splits == 1) put_weight(a, q, s, h, kb + lane, w);
    else a.sums[(((int64_t)share * c.n_seqs + s) * c.nkv + h) * a.score_ld + kb + lane] = w;
}

// ---------------------------------------------------------------------------
// k_account_sum
// ---------------------------------------------------------------------------
// A position a thread: the weights from the scores of at most 16 rows, or the sum of the
// shares of k_account_tile, in order.  grid nkv * ceil(cap / 256) * n_seqs, block 256.
__global__ __launch_bounds__(256) void k_account_sum(PagedShare a)
{
    const Paged& c = a.c;
    const int h = (int)(blockIdx.x % (unsigned)c.nkv);
    const unsigned at = blockIdx.x / (unsigned)c.nkv, blocks = (unsigned)(c.cap + 255) / 256;
    const int key = 256 * (int)(at % blocks) + threadIdx.x, s = (int)(at / blocks);
    const Seq q = seq_at(c, s);
    const int64_t M = (int64_t)q.n * a.group;
    if (M == 0 || !q.ok || key >= q.p0 + q.n) return;
    float w = 0.0f;
    if (has_scores(a, M)) {
        const float* sc = a.scores + ((int64_t)s * c.nkv + h) * a.score_rows * a.score_ld + key;
        const int64_t row0 = (int64_t)q.a * a.nh + h * a.group;
        for (int m = 0; m < (int)M; ++m) {
            const int i = row_of(a, m);
            const float2 ml = *(const float2*)(a.ml + 2 * (row0 + (int64_t)i * a.nh + (m - i * a.group)));
            const bool good = ml.y > 0.0f && ml.y < __builtin_inff();  // else it came back as NaN and adds nothing
            const float p = __fdiv_rn(__builtin_amdgcn_exp2f(__fsub_rn(sc[(int64_t)m * a.score_ld], ml.x)), ml.y);
            w = __fadd_rn(w, good ? p : 0.0f);
        }
    } else {
        if (a.splits == 1) return;  // put out where they were summed
        for (int x = 0; x < a.splits; ++x)
            w = __fadd_rn(w, a.sums[(((int64_t)x * c.n_seqs + s) * c.nkv + h) * a.score_ld + key]);
    }
    put_weight(a, q, s, h, key, w);
}

AttnPlan plan_paged_prefix(int64_t n_heads, const Paged& g, bool bf) { return plan_paged_attention(n_heads, g, bf); }

bool plan_paged_account(int64_t n_heads, PagedShare& a)
{
    const Paged& c = a.c;
    const int64_t group = n_heads / c.nkv, blocks = (c.cap + 255) / 256;
    a.score_rows = (int)std::min<int64_t>(kTokRows, (int64_t)c.max_rows * group);
    a.score_ld = (c.cap + 63) / 64 * 64;
    // scores of a batch whose bounds are far above its lengths would be a large workspace:
    // above 1 GiB the keys are gone through again
    a.scored = a.p.lo > 0 && (int64_t)c.n_seqs * c.nkv * a.score_rows * a.score_ld <= ((int64_t)1 << 28);
    const bool tiles = a.p.lo != INT_MAX || !a.scored;
    // sequences that k_account_tile goes through, at most
    const int64_t seqs = !tiles ? 0 : (a.scored ? std::min<int64_t>(c.n_seqs, (int64_t)c.rows * group / 16 + 1) : c.n_seqs);
    const int64_t want = 768, have = std::max<int64_t>(1, seqs * c.nkv * blocks);
    a.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want / have, 16, (int64_t)c.max_rows * group / 64}));
    const int64_t threads = ((int64_t)1 << 32) - 1;
    return (int64_t)c.nkv * blocks * c.n_seqs * 256 * (tiles ? a.splits : 1) <= threads;
}

template <int DT, bool BF>
static hipError_t launch_share(const PagedShare& a, hipStream_t st)
{
    if (a.g.n_seqs && a.g.cap) {
        PagedShare b = a;
        b.c = a.g;
        b.p = a.gp;
        if (b.p.tok_n) {
            const dim3 grid((unsigned)(b.c.nkv * b.p.tok_n * b.c.n_seqs));
            if (b.p.tok_w == 8) hipLaunchKernelGGL((k_paged_tok<DT, 8, BF, kPrefix>), grid, dim3(512), 0, st, b);
            else hipLaunchKernelGGL((k_paged_tok<DT, 4, BF, kPrefix>), grid, dim3(256), 0, st, b);
        }
        if (b.p.tile_n) {
            const dim3 grid((unsigned)(b.c.nkv * b.p.tile_n * b.p.tiles));
            if constexpr (BF) {
                if (b.p.tile_rows == 128) hipLaunchKernelGGL((k_paged_tile<DT, 2, BF, kPrefix>), grid, dim3(256), 0, st, b);
            }
            if (b.p.tile_rows == 64) hipLaunchKernelGGL((k_paged_tile<DT, 1, BF, kPrefix>), grid, dim3(256), 0, st, b);
        }
    }
    if (a.p.tok_n) {
        const dim3 grid((unsigned)(a.c.nkv * a.p.tok_n * a.c.n_seqs));
        if (a.weight && a.scored) {
            if (a.p.tok_w == 8) hipLaunchKernelGGL((k_paged_tok<DT, 8, BF, kScored>), grid, dim3(512), 0, st, a);
            else hipLaunchKernelGGL((k_paged_tok<DT, 4, BF, kScored>), grid, dim3(256), 0, st, a);
        } else {
            if (a.p.tok_w == 8) hipLaunchKernelGGL((k_paged_tok<DT, 8, BF, kOwn>), grid, dim3(512), 0, st, a);
            else hipLaunchKernelGGL((k_paged_tok<DT, 4, BF, kOwn>), grid, dim3(256), 0, st, a);
        }
    }
    if (a.p.tile_n) {
        const dim3 grid((unsigned)(a.c.nkv * a.p.tile_n * a.p.tiles));
        if constexpr (BF) {
            if (a.p.tile_rows == 128) hipLaunchKernelGGL((k_paged_tile<DT, 2, BF, kOwn>), grid, dim3(256), 0, st, a);
        }
        if (a.p.tile_rows == 64) hipLaunchKernelGGL((k_paged_tile<DT, 1, BF, kOwn>), grid, dim3(256), 0, st, a);
    }
    if (a.parts > 8)
        hipLaunchKernelGGL((k_paged_merge<4, BF, kOwn>), dim3((unsigned)a.c.rows, (unsigned)a.nh), dim3(256), 0, st, a);
    else if (a.parts > 1 || a.split)
        hipLaunchKernelGGL((k_paged_merge<1, BF, kOwn>), dim3((unsigned)a.c.rows, (unsigned)((a.nh + 3) / 4)), dim3(256), 0,
                           st, a);
    if (a.weight && a.c.cap) {
        const unsigned blocks = (unsigned)a.c.nkv * ((a.c.cap + 255) / 256) * a.c.n_seqs;
        const bool tiles = a.p.lo != INT_MAX || !a.scored;
        if (tiles) hipLaunchKernelGGL((k_account_tile<DT, BF>), dim3(blocks * a.splits), dim3(256), 0, st, a);
        if (a.scored || a.splits > 1) hipLaunchKernelGGL(k_account_sum, dim3(blocks), dim3(256), 0, st, a);
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
