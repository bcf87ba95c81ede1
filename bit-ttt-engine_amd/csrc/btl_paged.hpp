// btl_paged.hpp -- device helpers of the kernels over a paged Q8 cache (btl_serve.hip,
// btl_share.hip, btl_evict.hip).  Not part of the public ABI.
//
// The sequences' sizes, positions and pages are read on the device, so a captured
// launch follows them; whatever they hold, every address stays inside the arrays
// (rows are clamped to `rows`, page ids checked, slots clamped to the last visible
// one).
#pragma once

#include <hip/hip_runtime.h>

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

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// four neighbours, 4-byte aligned
struct __attribute__((packed, aligned(4))) Four {
    uint32_t v[4];
};

// Rust `f32 as u8`: saturating, NaN -> 0
__device__ __forceinline__ uint8_t to_u8(float r)
{
    if (!(r > 0.0f)) return 0;
    return (uint8_t)(r >= 255.0f ? 255u : (uint32_t)r);
}

}  // namespace

}  // namespace btl
