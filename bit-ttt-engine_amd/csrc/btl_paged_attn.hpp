// btl_paged_attn.hpp -- gfx950 kernels of attention over a paged Q8 cache, instantiated
// by btl_serve.hip (a batch) and btl_share.hip (with a shared prefix, with accounted
// weights).  Not part of the public ABI.
#pragma once

#include <type_traits>

#include "btl_paged.hpp"

namespace btl {

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

__device__ __forceinline__ uint32_t xor16_max(uint32_t v)
{
    u2 p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(p.x, p.y);
    p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(p.x, p.y);
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

// A row's values, 16 NJ a lane over the four lanes of the row, scaled by a power of two to
// just under 2^15 and put out in f16 parts: set(part, step, element, value).  Returns the
// log2 units of one unit of a product with them; NaN if one is not finite.
template <int NJ, int PARTS, typename F>
__device__ __forceinline__ float in_parts(const float (*f)[16], float scale_log2, F set)
{
    uint32_t am = 0;  // the largest magnitude's bits: what is not finite is above all that is
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int x = 0; x < 16; ++x) am = max(am, __float_as_uint(f[j][x]) & 0x7FFFFFFFu);
    am = xor16_max(am);
    const bool fin = am < 0x7F800000u;
    const int sh = fin ? 14 - expo(__uint_as_float(am)) : 0;
    const float up = exp2i(sh);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const float y = fin ? __fmul_rn(f[j][x], up) : 0.0f;  // exact
            const _Float16 hi = (_Float16)y;
            set(0, 2 * j + (x >> 3), x & 7, hi);
            if (PARTS == 2) set(1, 2 * j + (x >> 3), x & 7, (_Float16)__fsub_rn(y, (float)hi));
        }
    return fin ? __fmul_rn(scale_log2, exp2i(-sh)) : __builtin_nanf("");
}

// The query rows of a wave: NT tiles of 16, in PARTS f16 parts.
template <int NJ, int NT, bool BF>
struct Queries {
    static constexpr int PARTS = BF ? 1 : 2;
    float cq[NT];  // log2 units of one unit of the scaled product
    h8 v[PARTS][NT][2 * NJ];

    // rows m0 .. of a sequence, none past m_last (those repeat it); row0: the output row of m = 0
    __device__ __forceinline__ void load(const PagedAttn& a, const Seq& q, int64_t row0, int m0, int m_last, int lane,
                                         float scale)
    {
        const int g = lane >> 4, n = lane & 15, hd = a.c.hd;
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            const int m = m0 + 16 * u + n;
            const int mm = min(m, m_last);
            const int i = row_of(a, mm);
            const int64_t r = row0 + (int64_t)i * a.nh + (mm - i * a.group);
            float f[NJ][16];
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
            }
            cq[u] = in_parts<NJ, PARTS>(f, scale, [&](int p, int x, int e, _Float16 y) { v[p][u][x][e] = y; });
        }
    }
};

// One column tile's running softmax and output.
// EXACT: the products come with scale_log2 in them and cq is a power of two, so that one
// fused operation takes a score and the reference apart as exactly as two do.
template <int DT, bool EXACT = false>
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
        for (int x = 0; x < 16; ++x)
            y[x] = EXACT ? __fmaf_rn(sc[x >> 2][x & 3], cq, -at) : __fsub_rn(__fmul_rn(sc[x >> 2][x & 3], cq), at);
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

// block = h + nkv (chunk + chunks * tile): the head varies fastest.  Workgroups
// go to the XCDs in turn, so with 8 KV heads the tiles and chunks of one head share
// an XCD's L2.
__device__ __forceinline__ Place place_of(const Paged& c, int chunks, unsigned block)
{
    Place p;
    p.h = (int)(block % (unsigned)c.nkv);
    const unsigned b = block / (unsigned)c.nkv;
    p.chunk = (int)(b % (unsigned)chunks);
    p.tile = (int)(b / (unsigned)chunks);
    p.s = p.tile;
    return p;
}

// What a launch of the kernels below is for.
constexpr int kPlain = 0;   // the rows over their sequences' positions, causal
constexpr int kPrefix = 1;  // row lists over a prefix: every row sees the `pos` positions of its list
constexpr int kOwn = 2;     // as kPlain, beside a prefix or with the rows' maxima and sums put out
constexpr int kScored = 3;  // as kOwn, with the scores put out too (the token form)
template <int MODE>
using PagedArgs = std::conditional_t<MODE == kPlain || MODE == kPrefix, PagedAttn, PagedShare>;

template <int MODE>
__device__ __forceinline__ Seq seq_of(const Paged& c, int s)
{
    Seq q = seq_at(c, s);
    if (MODE == kPrefix) q.ok = q.p0 >= 0 && q.n <= c.max_rows && q.p0 <= c.cap;
    return q;
}

// the keys that a row of a sequence sees
template <int MODE>
__device__ __forceinline__ int sees(const Seq& q, int row)
{
    return MODE == kPrefix ? q.p0 : q.p0 + row + 1;
}

// the place of a chunk among a row's parts
template <int MODE>
__device__ __forceinline__ int part_of(const PagedArgs<MODE>& a, int chunk)
{
    if constexpr (MODE == kOwn || MODE == kScored) return a.own0 + chunk;
    else return chunk;
}

// a sequence's only chunk writes its rows out
template <int MODE>
__device__ __forceinline__ bool whole_of(const PagedArgs<MODE>& a, int seen, int C)
{
    if constexpr (MODE == kPlain) return seen <= C;
    else if constexpr (MODE == kPrefix) return false;
    else return !a.split && seen <= C;
}

// The kernel's arguments, or some that are one of its arguments' parts, to be read from here
// on.  All that a kernel asks for is read at its top otherwise: of several forms in one
// kernel, and of what only its end needs, that is more than the scalar registers hold.
template <typename T>
__device__ __forceinline__ const T& from_here(const __attribute__((address_space(4))) T* p)
{
    asm volatile("" : "+s"(p));
    return *(const T*)p;
}
template <typename T>
__device__ __forceinline__ const T& kernel_args()
{
    return from_here((const __attribute__((address_space(4))) T*)__builtin_amdgcn_kernarg_segment_ptr());
}
template <int MODE>
__device__ __forceinline__ const PagedArgs<MODE>& at_the_end(const PagedArgs<MODE>& a)
{
    if constexpr (MODE == kOwn || MODE == kScored)
        return from_here((const __attribute__((address_space(4))) PagedArgs<MODE>*)&a);
    else
        return a;
}

// What row t has in the prefix: its chunks, or that its list is refused.
struct Behind {
    int parts;
    bool lost;
};

// list: the last that starts at or before the row
__device__ __forceinline__ Behind behind_of(const PagedShare& a, int t, int list)
{
    if (list < 0 || list >= a.g.n_seqs) return {0, false};
    const Seq p = seq_of<kPrefix>(a.g, list);
    if (t < p.a || t >= p.a + p.n) return {0, false};
    const int C = (int64_t)p.n * a.group > a.gp.lo ? a.gp.tile_c : a.gp.tok_c;
    return {p.ok ? (p.p0 + C - 1) / C : 0, !p.ok};
}

__device__ __forceinline__ Behind behind(const PagedShare& a, int t, int lane)
{
    return behind_of(a, t, a.g.n_seqs ? find_seq(a.g, t, lane) : -1);
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
template <int DT, int NW>
struct TokLds {
    float (*o)[16][16 * DT + 4];  // [NW]
    float (*m)[16];               // [NW]
    float (*l)[16];               // [NW]
};

template <int DT, int NW, bool BF, int MODE>
__device__ __forceinline__ void paged_tok(const PagedArgs<MODE>& a, unsigned block, TokLds<DT, NW> lds)
{
    constexpr int NJ = (DT + 3) / 4;
    constexpr int PARTS = BF ? 1 : 2;  // of the queries (bf16 ones are exact in one)
    // Of the weights.  One part in bf16 would save 1.7 us of the batch's 81.4, and one output in
    // twelve would round the other way; in two it is one in 3000.
    constexpr int WP = 2;
    const auto s_o = lds.o;
    const auto s_m = lds.m, s_l = lds.l;
    const Paged& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int hd = c.hd, ndt = hd >> 4, C = a.p.tok_c;
    Place at = place_of(c, a.p.tok_n, block);
    // over a prefix a list may have several tiles of 16 rows
    const int m0 = MODE == kPrefix ? 16 * (at.tile % a.p.tiles) : 0;
    if (MODE == kPrefix) at.s = at.tile / a.p.tiles;
    const int key0 = at.chunk * C;
    const int32_t* table = c.pages + (int64_t)at.s * c.max_pages;
    // the pages are looked up beside the sequence's size, not after it: what the table holds
    // behind its last page is checked like any id, and its keys are masked
    const int last_grp = (c.cap - 1) >> 4;
    Slots slots{};
    if (c.cap > 0) slots.find(c, table, (key0 + 64 * wave) >> 4, last_grp, at.h, lane);
    const Seq q = seq_of<MODE>(c, at.s);
    const int64_t M = (int64_t)q.n * a.group;
    if (M <= m0 || M > a.p.lo) return;
    const int64_t row0 = (int64_t)q.a * a.nh + at.h * a.group;  // output row of m: row0 + (m / group) * nh + m % group
    if (!q.ok) {
        if (MODE != kPrefix && at.chunk == 0) fill_nan<BF>(a, q, at.h, wave, NW, lane);
        return;
    }
    const int seen = sees<MODE>(q, q.n - 1);  // keys that the last row sees
    const int key1 = min(key0 + C, seen);
    if (key0 >= key1) return;

    Queries<NJ, 1, BF> qs;
    qs.load(a, q, row0, m0, (int)M - 1, lane, MODE == kPlain ? a.scale_log2 : 1.0f);
    Running<DT, MODE != kPlain> r;
    r.clear();
    f4 kept[4];  // the last step's scores
    int kept_at = -1;
    auto keep = [&] {
        if constexpr (MODE == kScored) {
            if (kept_at < 0 || n >= M) return;
            float* to = a.scores + (((int64_t)at.s * c.nkv + at.h) * a.score_rows + n) * a.score_ld + kept_at + 16 * g;
#pragma unroll
            for (int t = 0; t < 4; ++t) *(f4*)(to + 4 * t) = kept[t];
        }
    };
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
            if (MODE != kPlain) ks[t] *= a.scale_log2;
            vs[t] = *(const f4*)(vscale + 4 * t);
        }
        uint4 vw[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) vw[d] = *(const uint4*)(vp + 256 * min(d, ndt - 1));
        const float lost = own < 0 ? __builtin_nanf("") : 0.0f;
        // behind the loads, which would be waited for with what was stored ahead of them
        if constexpr (MODE == kScored) keep();

        f4 sc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            sc[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const h8 k0 = widen8(kw[t][j].x, kw[t][j].y), k1 = widen8(kw[t][j].z, kw[t][j].w);
                // Where k_account_tile may make these scores again, they are added up in its order:
                // sums of another would be apart by roundings, which of large scores are any number.
#pragma unroll
                for (int x = 0; x < 2 * PARTS; ++x) {
                    const int p = MODE == kPlain ? x >> 1 : x % PARTS, half = MODE == kPlain ? x & 1 : x / PARTS;
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(half ? k1 : k0, qs.v[p][0][2 * j + half], sc[t], 0, 0, 0);
                }
            }
            // NaN where the page is outside the pool or a scale is not finite: an infinite one
            // times a negative product would be -inf, which is a key that no row sees
#pragma unroll
            for (int e = 0; e < 4; ++e)
                sc[t][e] = __fmaf_rn(sc[t][e], ks[t][e], __fmaf_rn(ks[t][e], 0.0f, __fmaf_rn(vs[t][e], 0.0f, lost)));
        }
        h8 pw[WP][2];
        if (kb + 64 <= sees<MODE>(q, 0)) {  // every row sees every key
            const int e = max(r.ve, expo(r.largest(vs)));
            if (__any(e != r.ve)) r.raise(e);
            const float up = exp2i(kVUp - r.ve);
#pragma unroll
            for (int t = 0; t < 4; ++t) vs[t] *= up;
            r.template weigh<WP>(sc, vs, qs.cq[0], pw);
        } else {
            const int vis = sees<MODE>(q, row_of(a, min(n, (int)M - 1)));  // keys that this lane's row sees
            r.template weigh_masked<WP>(sc, vs, kb + 16 * g, vis, qs.cq[0], pw);
        }
        if constexpr (MODE == kScored) {
#pragma unroll
            for (int t = 0; t < 4; ++t) kept[t] = sc[t] * qs.cq[0];
            kept_at = kb;
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

    keep();
    const float l = xor16_sum(r.l), unit = r.unit();
    if (g == 0) {
        s_m[wave][n] = r.ref;
        s_l[wave][n] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) *(f4*)&s_o[wave][n][16 * d + 4 * g] = r.o[d] * unit;
    __syncthreads();
    const PagedArgs<MODE>& z = at_the_end<MODE>(a);
    const bool whole = whole_of<MODE>(z, seen, C);
    for (int x = threadIdx.x; x < min((int)M - m0, 16) * (hd >> 2); x += 64 * NW) {
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
        const int i = row_of(a, m0 + m);
        const int64_t row = row0 + (int64_t)i * a.nh + (m0 + m - i * a.group);
        if (whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __fdiv_rn(v[e], sum);
            store4<BF>(z.out, row * hd + d, v);
            if constexpr (MODE == kOwn || MODE == kScored) {
                if (d == 0 && z.ml) *(float2*)(z.ml + 2 * row) = make_float2(top, sum);
            }
        } else {
            const int64_t part = row * z.parts + part_of<MODE>(z, at.chunk);
            store4<false>(z.part_o, part * hd + d, v);
            if (d == 0) *(float2*)(z.part_ml + 2 * part) = make_float2(top, sum);
        }
    }
}

template <int DT, int NW, bool BF, int MODE = kPlain>
__global__ __launch_bounds__(64 * NW, 2) void k_paged_tok(PagedArgs<MODE> a)
{
    __shared__ __align__(16) float s_o[NW][16][16 * DT + 4];
    __shared__ float s_m[NW][16], s_l[NW][16];
    if constexpr (MODE == kPlain) paged_tok<DT, NW, BF, MODE>(a, blockIdx.x, {s_o, s_m, s_l});
    else paged_tok<DT, NW, BF, MODE>(kernel_args<PagedArgs<MODE>>(), blockIdx.x, {s_o, s_m, s_l});
}

// The tile form: 64 NT query rows of a sequence, 16 NT a wave, every key to all four
// waves.  grid nkv * chunks * tiles, block 256.  Each wave widens a quarter of the
// next 64 keys' codes while the present ones are worked on: they lie in LDS as
// operand fragments (64 lanes x 16 bytes, read and written without conflicts), so a
// code is widened once a workgroup instead of once a wave.
//
// 512 rows over 8192 positions, 32 heads over 8 of 128: 66.6 GFLOP in 114 us in bf16
// (584 TFLOP/s; a large library product reaches 1116 to 1232), 192 us in f32, whose two parts
// are two products.  Per wave and 64 keys of 32 rows the matrix instructions take 1024
// cycles, the softmax and the widening some 1900 of the vector unit, on which two waves
// a SIMD take turns: that, and what is left of LDS latency between them, is the bound.
// Tried: each wave widening for itself 267 us; 48 or 64 rows a wave 280 and 223 (one
// wave a SIMD); without reading operands ahead 124 to 115; a branch-free step 117; wave
// priorities 129.
template <int DT>
struct TileLds {
    h8 (*k)[4][2 * ((DT + 3) / 4)][64];  // [2]
    h8 (*v)[DT][2][64];                  // [2]
    float (*ks)[64], (*vs)[64];          // [2]
    float* top;                          // [2]
};

template <int DT, int NT, bool BF, int MODE>
__device__ __forceinline__ void paged_tile(const PagedArgs<MODE>& a, unsigned block, TileLds<DT> lds)
{
    constexpr int NJ = (DT + 3) / 4;
    // Of the queries and of the weights.  In bf16 a query is exact in one part, and weights are
    // rounded to one, off by 2^-11 of themselves at most, ahead of an output that is rounded by
    // 2^-8: the 512-row chunk is 1.677e-3 (two-norm) off the exact result so and 1.663e-3, which
    // is the output's rounding alone, in two parts; it takes 114 us so and 137 in two.
    constexpr int PARTS = BF ? 1 : 2;
    constexpr int MT = 64 * NT;
    const auto s_k = lds.k;
    const auto s_v = lds.v;
    const auto s_ks = lds.ks, s_vs = lds.vs;
    const auto s_top = lds.top;
    const Paged& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int hd = c.hd, ndt = hd >> 4, C = a.p.tile_c;
    Place at = place_of(c, a.p.tile_n, block);

    // the sequence that the tile belongs to: sequences of more than `lo` query rows have
    // one for every MT of them.  A refused one has one for its NaN: the launch has tiles for
    // max_rows rows of it, and the others come behind.
    at.s = __builtin_amdgcn_readfirstlane(find_piece(c, lane, at.tile, [&](int s) {
        const Seq q = seq_of<MODE>(c, s);
        const int64_t rows = (int64_t)q.n * a.group;
        return rows > a.p.lo ? (q.ok ? (int)((rows + MT - 1) / MT) : 1) : 0;
    }));
    if (at.s < 0) return;
    const Seq q = seq_of<MODE>(c, at.s);
    const int64_t M = (int64_t)q.n * a.group;
    const int64_t row0 = (int64_t)q.a * a.nh + at.h * a.group;
    if (!q.ok) {
        if (MODE != kPrefix && at.chunk == 0 && at.tile == 0) fill_nan<BF>(a, q, at.h, wave, 4, lane);
        return;
    }
    const int m_tile = at.tile * MT;
    const int m_wave = m_tile + 16 * NT * wave;
    const int m_last = (int)min(M, (int64_t)m_tile + MT) - 1;
    const int seen = sees<MODE>(q, row_of(a, m_last));  // keys that the tile's last row sees
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
        scale = (wave & 1 ? +c.vs : +c.ks)[16 * (int64_t)at_v + n];
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
        if (wave == 0) s_ks[b][lane] = lost || bad ? __builtin_nanf("") : (MODE == kPlain ? scale : __fmul_rn(scale, a.scale_log2));
        if (wave == 1) {
            s_vs[b][lane] = bad ? __builtin_nanf("") : scale;
            const uint32_t m = __float_as_uint(scale) & 0x7FFFFFFFu;
            const uint32_t top = wave_max_dpp(m < 0x7F800000u ? m : 0u);  // of finite ones
            if (lane == 0) s_top[b] = __uint_as_float(top);
        }
    };

    Running<DT, MODE != kPlain> r[NT];
    Queries<NJ, NT, BF> qs;
    auto work = [&](int kb, int b, auto masked) {
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
                const int vis = sees<MODE>(q, row_of(a, min(m, m_last)));  // keys that this lane's row sees
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
    };
    // a wave behind the tile's last row widens its share and leaves the rest to the others
    const bool busy = MODE == kPlain || m_wave <= m_last;
    auto step = [&](int kb, int b, auto masked) {
        if (kb + 64 < key1) fetch(kb + 64);
        if (busy) work(kb, b, masked);
        if (kb + 64 < key1) put(b ^ 1);
        __syncthreads();
    };

    fetch(key0);
    qs.load(a, q, row0, m_wave, m_last, lane, MODE == kPlain ? a.scale_log2 : 1.0f);
#pragma unroll
    for (int u = 0; u < NT; ++u) r[u].clear();
    put(0);
    __syncthreads();
    const int vis_least = sees<MODE>(q, row_of(a, m_tile));
    int b = 0, kb = key0;
    for (; kb + 64 <= min(key1, vis_least); kb += 64, b ^= 1) step(kb, b, False{});
    for (; kb < key1; kb += 64, b ^= 1) step(kb, b, True{});

    const PagedArgs<MODE>& z = at_the_end<MODE>(a);
    const bool whole = whole_of<MODE>(z, sees<MODE>(q, q.n - 1), C);
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        float l = xor16_sum(r[u].l);
        const float unit = r[u].unit();
        // a value scale that is not finite makes all of a row's values NaN, but is in no score:
        // its sum says so too, to whoever adds up its weights
        if (MODE != kPlain && r[u].o[0].x != r[u].o[0].x) l = __builtin_nanf("");
        int m = m_wave + 16 * u + n;
        asm("" : "+v"(m));
        const int i = row_of(a, m);
        if (m > m_last) continue;
        const int64_t row = row0 + (int64_t)i * a.nh + (m - i * a.group), part = row * z.parts + part_of<MODE>(z, at.chunk);
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (d < ndt) {
                f4 v = r[u].o[d] * unit;
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __fdiv_rn(v[e], l);
                    store4<BF>(z.out, row * hd + 16 * d + 4 * g, v);
                } else {
                    store4<false>(z.part_o, part * hd + 16 * d + 4 * g, v);
                }
            }
        if (!whole && g == 0)
            *(float2*)(z.part_ml + 2 * part) = make_float2(r[u].ref == -__builtin_inff() ? 0.0f : r[u].ref, l);
        if constexpr (MODE == kOwn) {
            if (whole && g == 0 && z.ml)
                *(float2*)(z.ml + 2 * row) = make_float2(r[u].ref == -__builtin_inff() ? 0.0f : r[u].ref, l);
        }
    }
}

template <int DT, int NT, bool BF, int MODE = kPlain>
__global__ __launch_bounds__(256, 2) void k_paged_tile(PagedArgs<MODE> a)
{
    __shared__ __align__(16) h8 s_k[2][4][2 * ((DT + 3) / 4)][64];
    __shared__ __align__(16) h8 s_v[2][DT][2][64];
    __shared__ __align__(16) float s_ks[2][64], s_vs[2][64];
    __shared__ float s_top[2];
    if constexpr (MODE == kPlain) paged_tile<DT, NT, BF, MODE>(a, blockIdx.x, {s_k, s_v, s_ks, s_vs, s_top});
    else paged_tile<DT, NT, BF, MODE>(kernel_args<PagedArgs<MODE>>(), blockIdx.x, {s_k, s_v, s_ks, s_vs, s_top});
}

// ---------------------------------------------------------------------------
// k_paged_merge
// ---------------------------------------------------------------------------
// The chunks' outputs of a (row, head) weighed by 2^(m_c - max m).  Its threads are
// sets of 32 lanes, a chunk a set and 4 values a lane: W = 1: a wave a (row, head),
// for few chunks; W = 4: a workgroup, its sets' sums added in order in LDS.
// grid (rows, ceil(nh / (4 / W))), block 256.
// Beside a prefix (kOwn) a row's parts are the prefix's chunks and its sequence's, those
// from own0 on; a row whose prefix is refused is NaN.
template <int W, bool BF, int MODE = kPlain>
__global__ __launch_bounds__(256) void k_paged_merge(PagedArgs<MODE> a)
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
    if (whole_of<MODE>(a, q.p0 + q.n, C)) return;  // written by its one chunk
    int nc = (q.p0 + i) / C + 1;  // chunks that the row sees any key of
    int np = 0;                   // of them of the prefix
    bool lost = false;
    if constexpr (MODE != kPlain) {
        const Behind b = behind(a, t, lane);
        np = b.parts;
        lost = b.lost;
        nc += np;
    }
    const int64_t r = (int64_t)t * a.nh + head, at = r * a.parts;
    // the place of a row's x-th part
    auto place = [&](int x) {
        if constexpr (MODE != kPlain) return at + (x < np ? x : a.own0 - np + x);
        else return at + x;
    };
    float top = -__builtin_inff();
    for (int x = lane; x < nc; x += 64) top = fmaxf(top, a.part_ml[2 * place(x)]);
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
            const int64_t x = place(min(x0 + STEP * y, nc - 1));
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
    if constexpr (MODE != kPlain) {
        if (lost) sum = __builtin_nanf("");
        if (a.ml && lane == 0) *(float2*)(a.ml + 2 * r) = make_float2(top, sum);
    }
    if (lane < 32 && d < hd) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __fdiv_rn(v[e], sum);
        store4<BF>(a.out, r * hd + d, v);
    }
}

}  // namespace btl
