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

// page id of a group of 16 positions (-1: none in the pool) and the group's place in the page
__device__ __forceinline__ int page_of(const Paged& c, const int32_t* table, int grp, int* in_page)
{
    const int j = c.ppg_shift >= 0 ? grp >> c.ppg_shift : grp / c.ppg;
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
// grid (rows, ceil((nh + 2 nkv) / 4)), block 256, a wave per slot: q heads, then k
// heads, then v heads, each as k_rope_kv_q8 does it (lane i holds the pair
// (i, i + hd / 2) that RoPE turns together).
template <bool BF>
__global__ __launch_bounds__(256) void k_paged_append(PagedAppend a)
{
    const int t = blockIdx.x, lane = threadIdx.x & 63;
    const int slot = 4 * blockIdx.y + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nkv = a.c.nkv;
    if (slot >= a.nh + 2 * nkv) return;
    const int s = find_seq(a.c, t, lane);
    if (s < 0 || s >= a.c.n_seqs) return;
    const Seq q = seq_at(a.c, s);
    const int i = t - q.a;
    if (i < 0 || i >= q.n) return;
    const int pos = q.p0 + i;
    const bool good = q.ok && pos < a.rope_len;
    const int hd = a.c.hd, half = hd >> 1;
    const bool act = lane < half;
    const int kind = slot < a.nh ? 0 : (slot < a.nh + nkv ? 1 : 2);
    const int head = kind == 0 ? slot : (kind == 1 ? slot - a.nh : slot - a.nh - nkv);
    const void* src = kind == 0 ? a.q : (kind == 1 ? a.k : a.v);
    const int64_t row = ((int64_t)t * (kind == 0 ? a.nh : nkv) + head) * hd;
    if (!good) {
        if (kind == 0 && act) {
            store1<BF>(a.q_out, row + lane, __builtin_nanf(""));
            store1<BF>(a.q_out, row + lane + half, __builtin_nanf(""));
        }
        return;
    }
    float x1 = act ? load1<BF>(src, row + lane) : 0.0f, x2 = act ? load1<BF>(src, row + lane + half) : 0.0f;
    if (kind < 2 && act) {
        const float c = a.cos_t[(int64_t)pos * half + lane], w = a.sin_t[(int64_t)pos * half + lane];
        const float o1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, w));
        const float o2 = __fadd_rn(__fmul_rn(x1, w), __fmul_rn(x2, c));
        x1 = o1;
        x2 = o2;
    }
    if (kind == 0) {
        if (act) {
            store1<BF>(a.q_out, row + lane, x1);
            store1<BF>(a.q_out, row + lane + half, x2);
        }
        return;
    }
    int grp;
    const int page = page_of(a.c, a.c.pages + (int64_t)s * a.c.max_pages, pos >> 4, &grp);
    if (page < 0) return;
    const uint32_t am = wave_max_dpp(max(__float_as_uint(x1) & 0x7FFFFFFFu, __float_as_uint(x2) & 0x7FFFFFFFu));
    const float sc = __fadd_rn(__fmul_rn(__uint_as_float(am), (float)(1.0 / 127.0)), 0.0f);
    const int64_t blk = ((int64_t)page * nkv + head) * a.c.ps + 16 * grp;  // first slot of the group of 16
    const int in = pos & 15;
    if (act) {
        const uint8_t c1 = to_u8(__fadd_rn(__builtin_roundf(__fdiv_rn(x1, sc)), 128.0f));
        const uint8_t c2 = to_u8(__fadd_rn(__builtin_roundf(__fdiv_rn(x2, sc)), 128.0f));
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

hipError_t launch_paged_append(const PagedAppend& a, hipStream_t st)
{
    const dim3 grid((unsigned)a.c.rows, (unsigned)((a.nh + 2 * a.c.nkv + 3) / 4));
    if (a.bf) hipLaunchKernelGGL(k_paged_append<true>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_paged_append<false>, grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// k_paged_read
// ---------------------------------------------------------------------------
// grid (rows, ceil(nkv / 4)), block 256, a wave per (row, KV head).
template <bool BF>
__global__ __launch_bounds__(256) void k_paged_read(PagedRead a)
{
    const int t = blockIdx.x, lane = threadIdx.x & 63;
    const int head = 4 * blockIdx.y + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (head >= a.c.nkv) return;
    const int s = find_seq(a.c, t, lane);
    if (s < 0 || s >= a.c.n_seqs) return;
    const Seq q = seq_at(a.c, s);
    const int i = t - q.a;
    if (i < 0 || i >= q.n) return;
    const int pos = q.p0 + i, hd = a.c.hd;
    int grp = 0, page = -1;
    if (q.ok) page = page_of(a.c, a.c.pages + (int64_t)s * a.c.max_pages, pos >> 4, &grp);
    const int64_t blk = ((int64_t)max(page, 0) * a.c.nkv + head) * a.c.ps + 16 * grp;
    const int64_t out = ((int64_t)t * a.c.nkv + head) * hd;
    const int in = pos & 15;
    const float nan = __builtin_nanf("");
    const float ks = page < 0 ? nan : a.c.ks[blk + in], vs = page < 0 ? nan : a.c.vs[blk + in];
    for (int d = lane; d < hd; d += 64) {
        const float k = page < 0 ? 0.0f : __fsub_rn((float)a.c.k[(blk + in) * hd + d], 128.0f);
        const float v = page < 0 ? 0.0f : __fsub_rn((float)a.c.v[blk * hd + 16 * d + in], 128.0f);
        if (a.k_out) store1<BF>(a.k_out, out + d, __fmul_rn(k, ks));
        if (a.v_out) store1<BF>(a.v_out, out + d, __fmul_rn(v, vs));
    }
}

hipError_t launch_paged_read(const PagedRead& a, hipStream_t st)
{
    const dim3 grid((unsigned)a.c.rows, (unsigned)((a.c.nkv + 3) / 4));
    if (a.bf) hipLaunchKernelGGL(k_paged_read<true>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_paged_read<false>, grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// k_paged_attn
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
// value, is one 16-byte load of the blocked v.  Nothing crosses lanes but the
// row maxima (two shuffles), and no operand goes through LDS.
//
// A code u8 becomes the f16 1024 + u8 by one byte permute, less 1152 (exact).
// Queries are scaled by a power of two per row to just under 2^15, softmax weights
// times the value's scale by one per (row, largest value scale so far): what is
// lost is below 2^-39 of the row's largest term, not below f16's smallest number.
//
// The token form (TOK, at most 16 query rows) gives the keys of a chunk to its
// four waves in turn and merges them in LDS; the tile form gives 16 NT query rows
// to each of its four waves and every key to all of them.
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

namespace {

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

__device__ __forceinline__ float xor16_max(float v)
{
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}

__device__ __forceinline__ float xor16_sum(float v)
{
    v = __fadd_rn(v, __shfl_xor(v, 16, 64));
    return __fadd_rn(v, __shfl_xor(v, 32, 64));
}

// Keeps the f32 product v as it was rounded.  The compiler may turn an f16
// conversion of a product into one instruction that rounds once; where the two
// parts of a number each convert it, that made a first part of one rounding and a
// rest of the other, off by a step of f16 in some of 10^4 weights.
__device__ __forceinline__ void as_rounded(float& v) { asm("" : "+v"(v)); }

// 2^e, -126 <= e <= 127
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// exponent of |v|, kept in [-110, 127] (0, subnormal: -110; not finite: as 0)
__device__ __forceinline__ int expo(float v)
{
    const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
    return b >= 0x7F800000u ? -110 : max((int)(b >> 23) - 127, -110);
}

// The rows' chunk or the whole output of one query row: v of 4 neighbouring values.
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

}  // namespace

template <int NJ, int NT, bool TOK, bool BF>
__global__ __launch_bounds__(256) void k_paged_attn(PagedAttn a)
{
    constexpr int DT = 4 * NJ;         // 16-value tiles of a head, at most
    constexpr int PARTS = BF ? 1 : 2;  // f16 parts of a query and of a weight
    constexpr int MT = TOK ? kTokRows : 64 * NT;
    const Paged& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int hd = c.hd, ndt = hd >> 4;
    // the head varies fastest: neighbouring workgroups go to different XCDs, so with
    // 8 KV heads the tiles and chunks of one head share that XCD's L2
    const int h = (int)(blockIdx.x % (unsigned)c.nkv);
    const unsigned bi = blockIdx.x / (unsigned)c.nkv;
    const int chunks = TOK ? a.p.tok_n : a.p.tile_n, C = TOK ? a.p.tok_c : a.p.tile_c;
    const int chunk = (int)(bi % (unsigned)chunks);
    int tile = (int)(bi / (unsigned)chunks);

    // the sequence and its tile
    int s;
    if (TOK) {
        s = tile;
        tile = 0;
    } else {
        int base = 0;
        for (s = -1; base < c.n_seqs; base += 64) {
            int mine = 0;
            if (base + lane < c.n_seqs) {
                const int64_t rows = (int64_t)seq_at(c, base + lane).n * a.group;
                mine = rows > a.p.lo ? (int)((rows + MT - 1) / MT) : 0;
            }
            int upto = mine;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int o = __shfl_up(upto, off, 64);
                upto += lane >= off ? o : 0;
            }
            const uint64_t past = __ballot(upto > tile);
            if (past) {
                const int at = __ffsll((unsigned long long)past) - 1;
                s = base + at;
                tile -= __builtin_amdgcn_readlane(upto - mine, at);
                break;
            }
            tile -= __builtin_amdgcn_readlane(upto, 63);
        }
        if (s < 0) return;
    }
    s = __builtin_amdgcn_readfirstlane(s);
    tile = __builtin_amdgcn_readfirstlane(tile);
    const Seq q = seq_at(c, s);
    const int64_t M = (int64_t)q.n * a.group;
    if (M == 0 || (TOK && M > a.p.lo)) return;
    const int64_t row0 = (int64_t)q.a * a.nh + h * a.group;  // output row of m: row0 + (m / group) * nh + m % group
    if (!q.ok) {
        if (chunk == 0 && tile == 0)
            for (int i = wave; i < q.n; i += 4)
                for (int x = lane; x < a.group * hd; x += 64)
                    store1<BF>(a.out, (row0 + (int64_t)i * a.nh) * hd + x, __builtin_nanf(""));
        return;
    }
    const int m_tile = tile * MT;
    const int m_last = (int)min(M, (int64_t)m_tile + MT) - 1;
    const int seen = q.p0 + m_last / a.group + 1;  // keys that the tile's last row sees
    const int key0 = chunk * C, key1 = min(key0 + C, seen);
    if (key0 >= key1) return;
    const int32_t* table = c.pages + (int64_t)s * c.max_pages;

    // ---- queries
    const int m_wave = m_tile + (TOK ? 0 : 16 * NT * wave);
    int vis[NT];           // keys that this lane's query row sees
    int64_t orow[NT];      // its output row, -1: none
    float cq[NT];          // log2 units of one unit of the scaled product
    h8 qv[PARTS][NT][2 * NJ];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        const int m = m_wave + 16 * u + n;
        const bool on = m <= m_last;
        const int mm = on ? m : m_last;
        const int i = mm / a.group;
        vis[u] = q.p0 + i + 1;
        const int64_t r = row0 + (int64_t)i * a.nh + (mm - i * a.group);
        orow[u] = on ? r : -1;
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
        const int sh = fin ? min(14 - expo(am), 120) : 0;
        const float up = exp2i(sh);
        cq[u] = fin ? __fmul_rn(a.scale_log2, exp2i(-sh)) : __builtin_nanf("");
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const float y = fin ? __fmul_rn(f[j][x], up) : 0.0f;
                const _Float16 hi = (_Float16)y;
                qv[0][u][2 * j + (x >> 3)][x & 7] = hi;
                if (PARTS == 2) qv[PARTS - 1][u][2 * j + (x >> 3)][x & 7] = (_Float16)__fsub_rn(y, (float)hi);
            }
    }

    // ---- keys
    float mx[NT], l[NT];
    int ve[NT];  // exponent that the weights are scaled by
    f4 o[DT][NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        mx[u] = -__builtin_inff();
        l[u] = 0.0f;
        ve[u] = -110;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d][u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int last_grp = (key1 - 1) >> 4;
    const int vis_least = q.p0 + min(m_wave, m_last) / a.group + 1;
    for (int kb = key0 + (TOK ? 64 * wave : 0); kb < key1; kb += TOK ? 256 : 64) {
        // pages of this lane's groups: of the key row it loads, of the keys whose scales and values it takes
        int ik, iv;
        const int pk = page_of(c, table, min((kb >> 4) + (n >> 2), last_grp), &ik);
        const int pv = page_of(c, table, min((kb >> 4) + g, last_grp), &iv);
        const uint8_t* kp = c.k + (((int64_t)max(pk, 0) * c.nkv + h) * c.ps + 16 * ik + (n & 3)) * hd;
        const int64_t sv = ((int64_t)max(pv, 0) * c.nkv + h) * c.ps + 16 * iv;
        const uint8_t* vp = c.v + sv * hd + 16 * n;
        uint4 kw[4][NJ];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int d = 16 * (4 * j + g);
                kw[t][j] = *(const uint4*)(kp + 4 * t * hd + (d < hd ? d : 0));
            }
        f4 ksc[4], vsc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            ksc[t] = *(const f4*)(c.ks + sv + 4 * t);
            vsc[t] = *(const f4*)(c.vs + sv + 4 * t);
            if (pv < 0) ksc[t] = f4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
        }
        uint4 vw[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) vw[d] = d < ndt ? *(const uint4*)(vp + 256 * d) : uint4{};

        f4 sc[NT][4];
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int t = 0; t < 4; ++t) sc[u][t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const h8 k0 = widen8(kw[t][j].x, kw[t][j].y), k1 = widen8(kw[t][j].z, kw[t][j].w);
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
#pragma unroll
                    for (int u = 0; u < NT; ++u) {
                        sc[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qv[p][u][2 * j], sc[u][t], 0, 0, 0);
                        sc[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qv[p][u][2 * j + 1], sc[u][t], 0, 0, 0);
                    }
            }

        h8 pw[PARTS][NT][2];
        const int kl = kb + 16 * g;               // this lane's first key
        const bool full = kb + 64 <= vis_least;  // every row of the wave sees every key
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            f4 vm[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                vm[t] = vsc[t];
                sc[u][t] *= ksc[t];
            }
            if (!full) {
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool see = kl + 4 * t + e < vis[u];
                        sc[u][t][e] = see ? sc[u][t][e] : -__builtin_inff();
                        vm[t][e] = see ? vm[t][e] : 0.0f;
                    }
            }
            float big = -__builtin_inff(), vmax = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    big = fmaxf(big, sc[u][t][e]);
                    const float av = __builtin_fabsf(vm[t][e]);
                    vmax = av < __builtin_inff() ? fmaxf(vmax, av) : vmax;
                }
            const float mnew = fmaxf(mx[u], xor16_max(big));
            const int enew = max(ve[u], expo(xor16_max(vmax)));
            const float ref = mnew == -__builtin_inff() ? 0.0f : __fmul_rn(mnew, cq[u]);
            const float alpha = mx[u] == -__builtin_inff() ? 0.0f
                                                           : __builtin_amdgcn_exp2f(__fmaf_rn(mx[u], cq[u], -ref));
            const float oscale = __builtin_ldexpf(alpha, ve[u] - enew);
            l[u] = __fmul_rn(l[u], alpha);
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d][u] *= oscale;
            mx[u] = mnew;
            ve[u] = enew;
            const float vup = exp2i(min(14 - enew, 124));
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __builtin_amdgcn_exp2f(__fmaf_rn(sc[u][t][e], cq[u], -ref));
                    l[u] = __fadd_rn(l[u], p);
                    float w = __fmul_rn(p, __fmul_rn(vm[t][e], vup));
                    if (PARTS == 2) as_rounded(w);
                    const _Float16 hi = (_Float16)w;
                    pw[0][u][t >> 1][4 * (t & 1) + e] = hi;
                    if (PARTS == 2) pw[PARTS - 1][u][t >> 1][4 * (t & 1) + e] = (_Float16)__fsub_rn(w, (float)hi);
                }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (d < ndt) {
                const h8 v0 = widen8(vw[d].x, vw[d].y), v1 = widen8(vw[d].z, vw[d].w);
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
#pragma unroll
                    for (int u = 0; u < NT; ++u) {
                        o[d][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pw[p][u][0], o[d][u], 0, 0, 0);
                        o[d][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pw[p][u][1], o[d][u], 0, 0, 0);
                    }
            }
    }

    // ---- out, or the chunk's part of it
    const bool whole = q.p0 + q.n <= C;  // the sequence is one chunk
#pragma unroll
    for (int u = 0; u < NT; ++u) l[u] = xor16_sum(l[u]);
    if (TOK) {
        __shared__ float s_o[4][16][16 * DT + 4];
        __shared__ float s_m[4][16], s_l[4][16];
        const float down = exp2i(max(ve[0] - 14, -124));
        const float m2 = mx[0] == -__builtin_inff() ? mx[0] : __fmul_rn(mx[0], cq[0]);
        if (g == 0) {
            s_m[wave][n] = m2;
            s_l[wave][n] = l[0];
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (d < ndt) *(f4*)&s_o[wave][n][16 * d + 4 * g] = o[d][0] * down;
        __syncthreads();
        const int rows = m_last + 1;
        for (int x = threadIdx.x; x < rows * (hd >> 2); x += 256) {
            const int m = x / (hd >> 2), d = 4 * (x - m * (hd >> 2));
            float top = s_m[0][m];
#pragma unroll
            for (int w = 1; w < 4; ++w) top = fmaxf(top, s_m[w][m]);
            top = top == -__builtin_inff() ? 0.0f : top;
            float sum = 0.0f;
            f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float b = __builtin_amdgcn_exp2f(__fsub_rn(s_m[w][m], top));
                sum = __fmaf_rn(b, s_l[w][m], sum);
                const f4 ow = *(const f4*)&s_o[w][m][d];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __fmaf_rn(b, ow[e], v[e]);
            }
            const int i = m / a.group;
            const int64_t r = row0 + (int64_t)i * a.nh + (m - i * a.group);
            if (whole) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __fdiv_rn(v[e], sum);
                store4<BF>(a.out, r * hd + d, v);
            } else {
                const int64_t at = r * a.parts + chunk;
                store4<false>(a.part_o, at * hd + d, v);
                if (d == 0) *(float2*)(a.part_ml + 2 * at) = make_float2(top, sum);
            }
        }
        return;
    }
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        if (orow[u] < 0) continue;
        const float down = exp2i(max(ve[u] - 14, -124));
        const int64_t at = orow[u] * a.parts + chunk;
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (d < ndt) {
                f4 v = o[d][u] * down;
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __fdiv_rn(v[e], l[u]);
                    store4<BF>(a.out, orow[u] * hd + 16 * d + 4 * g, v);
                } else {
                    store4<false>(a.part_o, at * hd + 16 * d + 4 * g, v);
                }
            }
        if (!whole && g == 0)
            *(float2*)(a.part_ml + 2 * at) =
                make_float2(mx[u] == -__builtin_inff() ? 0.0f : __fmul_rn(mx[u], cq[u]), l[u]);
    }
}

// ---------------------------------------------------------------------------
// k_paged_merge
// ---------------------------------------------------------------------------
// grid (rows, ceil(nh / 4)), block 256, a wave per (row, head): the chunks' outputs
// weighed by 2^(m_c - max m), in chunk order.
template <bool BF>
__global__ __launch_bounds__(256) void k_paged_merge(PagedAttn a)
{
    const Paged& c = a.c;
    const int t = blockIdx.x, lane = threadIdx.x & 63;
    const int head = 4 * blockIdx.y + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
    const int hd = c.hd, d0 = lane, d1 = lane + 64;
    float sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int x = 0; x < nc; ++x) {
        const float2 ml = *(const float2*)(a.part_ml + 2 * (at + x));
        const float b = __builtin_amdgcn_exp2f(__fsub_rn(ml.x, top));
        sum = __fmaf_rn(b, ml.y, sum);
        if (d0 < hd) o0 = __fmaf_rn(b, a.part_o[(at + x) * hd + d0], o0);
        if (d1 < hd) o1 = __fmaf_rn(b, a.part_o[(at + x) * hd + d1], o1);
    }
    if (d0 < hd) store1<BF>(a.out, r * hd + d0, __fdiv_rn(o0, sum));
    if (d1 < hd) store1<BF>(a.out, r * hd + d1, __fdiv_rn(o1, sum));
}

AttnPlan plan_paged_attention(int64_t n_heads, const Paged& c)
{
    auto up = [](int64_t v, int64_t m) { return (v + m - 1) / m * m; };
    const int64_t group = n_heads / c.nkv, longest = std::max(c.cap, 1);
    AttnPlan p{};
    // one kind of launch where the bounds leave one kind of sequence
    p.lo = c.max_rows * group <= kTokRows ? INT_MAX : (c.n_seqs == 1 ? 0 : kTokRows);
    const int64_t want = 2048;
    const int64_t all = up(longest, 256);
    p.tok_c = (int)std::min(all, up(longest * c.n_seqs * c.nkv / want + 1, 256));
    p.tok_n = (int)((longest + p.tok_c - 1) / p.tok_c);
    const int64_t per = ((int64_t)c.max_rows * group + kTileRows - 1) / kTileRows;
    p.tiles = (int)std::min<int64_t>((int64_t)c.n_seqs * per, (int64_t)c.rows * group / kTileRows + c.n_seqs);
    p.tile_c = (int)std::min(all, up(longest * p.tiles * c.nkv / 512 + 1, 256));
    p.tile_n = (int)((longest + p.tile_c - 1) / p.tile_c);
    if (p.lo == 0) p.tok_n = 0;
    if (p.lo == INT_MAX) p.tile_n = p.tiles = 0;
    return p;
}

bool paged_attention_fits(const Paged& c, const AttnPlan& p)
{
    const int64_t most = ((int64_t)1 << 24) - 1;  // of 256 threads: under 2^32
    return (int64_t)c.nkv * p.tok_n * c.n_seqs <= most && (int64_t)c.nkv * p.tile_n * p.tiles <= most;
}

template <int NJ, bool BF>
static hipError_t launch_attn(const PagedAttn& a, hipStream_t st)
{
    if (a.p.tok_n)
        hipLaunchKernelGGL((k_paged_attn<NJ, 1, true, BF>), dim3((unsigned)(a.c.nkv * a.p.tok_n * a.c.n_seqs)), dim3(256),
                           0, st, a);
    if (a.p.tile_n)
        hipLaunchKernelGGL((k_paged_attn<NJ, kTileRows / 64, false, BF>),
                           dim3((unsigned)(a.c.nkv * a.p.tile_n * a.p.tiles)), dim3(256), 0, st, a);
    if (a.parts > 1)
        hipLaunchKernelGGL(k_paged_merge<BF>, dim3((unsigned)a.c.rows, (unsigned)((a.nh + 3) / 4)), dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_paged_attention(const PagedAttn& a, hipStream_t st)
{
    if (a.c.hd <= 64) return a.bf ? launch_attn<1, true>(a, st) : launch_attn<1, false>(a, st);
    return a.bf ? launch_attn<2, true>(a, st) : launch_attn<2, false>(a, st);
}

}  // namespace btl
