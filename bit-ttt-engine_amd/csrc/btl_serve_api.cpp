// btl_serve_api.cpp -- C ABI of the batched serving ops (include/bitserve.h):
// validation and dispatch to the kernels of btl_serve.hip and btl_sample.hip.
#include "bitserve.h"

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>

#include "btl_host.hpp"
#include "btl_serve.hpp"

namespace {

using btl::host::fail_msg;
using btl::host::hip_error;

template <typename... A>
int failf(int code, const char* fmt, A... args)
{
    char buf[512];
    snprintf(buf, sizeof(buf), fmt, args...);
    return fail_msg(code, buf);
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
inline bool aligned4(const void* p) { return ((uintptr_t)p & 3u) == 0; }
inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

bool overlap(const void* a, size_t na, const void* b, size_t nb)
{
    return a && b && (const uint8_t*)a < (const uint8_t*)b + nb && (const uint8_t*)b < (const uint8_t*)a + na;
}

int check_dtype(int dt)
{
    if (dt != BTL_F32 && dt != BTL_BF16) return failf(BTL_ERR_DTYPE, "dtype %d is not BTL_F32/BTL_BF16", dt);
    return BTL_OK;
}

// Sizes of the cache and the batch, before any pointer is looked at; c: filled.
int check_sizes(const btl_kv_paged_t* k, const btl_paged_batch_t* b, btl::Paged* c)
{
    if (!k) return fail_msg(BTL_ERR_ARG, "null paged cache");
    if (!b) return fail_msg(BTL_ERR_ARG, "null batch");
    if (k->n_pages < 1 || k->n_kv_heads < 1 || k->n_pages > (1 << 28) || k->n_kv_heads > 1024)
        return failf(BTL_ERR_SHAPE, "paged cache needs 1 .. 2^28 pages and 1 .. 1024 KV heads (got %lld, %lld)",
                     (long long)k->n_pages, (long long)k->n_kv_heads);
    if (k->page_size < 16 || k->page_size % 16 || k->page_size > (1 << 16))
        return failf(BTL_ERR_SHAPE, "page_size %lld: need a multiple of 16 up to 65536", (long long)k->page_size);
    if (k->head_dim < 16 || k->head_dim % 16 || k->head_dim > 128)
        return failf(BTL_ERR_SHAPE, "head_dim %lld: need a multiple of 16 up to 128", (long long)k->head_dim);
    if (k->n_pages * k->n_kv_heads * (k->page_size / 16) >= ((int64_t)1 << 31))
        return fail_msg(BTL_ERR_SHAPE, "paged cache too large: n_pages * n_kv_heads * page_size / 16 must be below 2^31");
    if (b->n_seqs < 0 || b->n_seqs > (1 << 20) || b->rows < 0 || b->rows > (1 << 23) || b->max_pages < 0 ||
        b->max_pages > (1 << 24) || b->max_rows < 0 || b->max_len < 0)
        return fail_msg(BTL_ERR_SHAPE, "batch size out of range");
    c->n_pages = (int)k->n_pages;
    c->nkv = (int)k->n_kv_heads;
    c->ps = (int)k->page_size;
    c->hd = (int)k->head_dim;
    c->ppg = c->ps / 16;
    c->ppg_mul = (uint32_t)((((int64_t)1 << 31) + c->ppg - 1) / c->ppg);
    c->n_seqs = (int)b->n_seqs;
    c->max_pages = (int)b->max_pages;
    c->rows = (int)b->rows;
    c->max_rows = (int)std::min(b->max_rows, b->rows);
    c->cap = (int)std::min<int64_t>(std::min(b->max_len, b->max_pages * k->page_size), 1 << 23);
    return BTL_OK;
}

int check_pointers(const btl_kv_paged_t* k, const btl_paged_batch_t* b, btl::Paged* c)
{
    if (!k->k || !k->v || !k->k_scale || !k->v_scale) return fail_msg(BTL_ERR_LAYOUT, "null paged cache buffer");
    if (!aligned16(k->k) || !aligned16(k->v) || !aligned16(k->k_scale) || !aligned16(k->v_scale))
        return fail_msg(BTL_ERR_LAYOUT, "paged cache buffers must be 16-byte aligned");
    if (!b->row_start || !b->pos || (!b->pages && b->max_pages)) return fail_msg(BTL_ERR_LAYOUT, "null batch array");
    if (!aligned4(b->row_start) || !aligned4(b->pos) || !aligned4(b->pages))
        return fail_msg(BTL_ERR_LAYOUT, "batch arrays must be 4-byte aligned");
    c->k = k->k;
    c->v = k->v;
    c->ks = k->k_scale;
    c->vs = k->v_scale;
    c->row_start = b->row_start;
    c->pos = b->pos;
    c->pages = b->pages;
    return BTL_OK;
}

int check_heads(int64_t n_heads, const btl::Paged& c)
{
    if (n_heads < 1 || n_heads % c.nkv || n_heads / c.nkv > 16)
        return failf(BTL_ERR_SHAPE, "n_heads %lld must be a multiple of n_kv_heads %d, at most 16 times it",
                     (long long)n_heads, c.nkv);
    return BTL_OK;
}

size_t attention_bytes(const btl::Paged& c, int64_t n_heads, const btl::AttnPlan& p)
{
    if (p.parts() <= 1) return 0;
    const size_t n = (size_t)c.rows * n_heads * p.parts();
    return up256(n * c.hd * 4) + up256(n * 8);
}

struct SampleWs {
    size_t mass, count, total;
};
SampleWs sample_ws(int64_t rows, int64_t n)
{
    // of the smallest slice: a workspace for some rows serves fewer
    const size_t slices = (size_t)((n + 2047) / 2048);
    SampleWs w;
    w.mass = up256((size_t)rows * slices * 8);
    w.count = w.mass + up256((size_t)rows * btl::kSampleBins * 8);
    w.total = w.count + up256((size_t)rows * btl::kSampleBins * 4);
    return w;
}

}  // namespace

extern "C" {

int btl_paged_rope_append(const void* q, const void* k, const void* v, int dtype, int64_t n_heads,
                          const btl_kv_paged_t* cache, const btl_paged_batch_t* batch, const float* rope_cos,
                          const float* rope_sin, int64_t rope_len, void* q_out, void* stream)
{
    btl::PagedAppend a{};
    int rc;
    if ((rc = check_dtype(dtype)) || (rc = check_sizes(cache, batch, &a.c)) || (rc = check_heads(n_heads, a.c))) return rc;
    if (rope_len < 0 || rope_len > INT_MAX) return fail_msg(BTL_ERR_SHAPE, "rope table length out of range");
    if (a.c.rows == 0 || a.c.n_seqs == 0) return BTL_OK;
    if ((rc = check_pointers(cache, batch, &a.c))) return rc;
    if (!q || !k || !v || !q_out || (rope_len && (!rope_cos || !rope_sin))) return fail_msg(BTL_ERR_LAYOUT, "null pointer");
    const size_t size = dtype == BTL_F32 ? 4 : 2;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) || !aligned16(rope_cos) || !aligned16(rope_sin))
        return fail_msg(BTL_ERR_LAYOUT, "q, k, v, q_out and the rope tables must be 16-byte aligned");
    const size_t qn = (size_t)a.c.rows * n_heads * a.c.hd * size, kn = (size_t)a.c.rows * a.c.nkv * a.c.hd * size;
    if ((q_out != q && overlap(q_out, qn, q, qn)) || overlap(q_out, qn, k, kn) || overlap(q_out, qn, v, kn))
        return fail_msg(BTL_ERR_LAYOUT, "q_out must be q itself or not overlap q, k and v");
    int dev;
    if ((rc = btl::host::device(&dev))) return rc;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.cos_t = rope_cos;
    a.sin_t = rope_sin;
    a.rope_len = (int)rope_len;
    a.nh = (int)n_heads;
    a.bf = dtype == BTL_BF16;
    const hipError_t e = btl::launch_paged_append(a, (hipStream_t)stream);
    return e == hipSuccess ? BTL_OK : hip_error(e, "paged append kernel launch");
}

int btl_paged_read(const btl_kv_paged_t* cache, const btl_paged_batch_t* batch, void* k_out, void* v_out, int dtype,
                   void* stream)
{
    btl::PagedRead a{};
    int rc;
    if ((rc = check_dtype(dtype)) || (rc = check_sizes(cache, batch, &a.c))) return rc;
    if (a.c.rows == 0 || a.c.n_seqs == 0 || (!k_out && !v_out)) return BTL_OK;
    if ((rc = check_pointers(cache, batch, &a.c))) return rc;
    const size_t size = dtype == BTL_F32 ? 4 : 2, n = (size_t)a.c.rows * a.c.nkv * a.c.hd * size;
    if (!aligned16(k_out) || !aligned16(v_out)) return fail_msg(BTL_ERR_LAYOUT, "k_out and v_out must be 16-byte aligned");
    if (overlap(k_out, n, v_out, n)) return fail_msg(BTL_ERR_LAYOUT, "k_out and v_out overlap");
    int dev;
    if ((rc = btl::host::device(&dev))) return rc;
    a.k_out = k_out;
    a.v_out = v_out;
    a.bf = dtype == BTL_BF16;
    const hipError_t e = btl::launch_paged_read(a, (hipStream_t)stream);
    return e == hipSuccess ? BTL_OK : hip_error(e, "paged read kernel launch");
}

size_t btl_paged_attention_workspace_bytes(int64_t n_heads, const btl_kv_paged_t* cache,
                                           const btl_paged_batch_t* batch)
{
    btl::Paged c{};
    if (check_sizes(cache, batch, &c) || check_heads(n_heads, c) || c.rows == 0 || c.n_seqs == 0) return 0;
    return std::max(attention_bytes(c, n_heads, btl::plan_paged_attention(n_heads, c, false)),
                    attention_bytes(c, n_heads, btl::plan_paged_attention(n_heads, c, true)));
}

int btl_paged_attention(const void* q, int dtype, int64_t n_heads, const btl_kv_paged_t* cache,
                        const btl_paged_batch_t* batch, void* out, void* ws, size_t ws_bytes, void* stream)
{
    btl::PagedAttn a{};
    int rc;
    if ((rc = check_dtype(dtype)) || (rc = check_sizes(cache, batch, &a.c)) || (rc = check_heads(n_heads, a.c))) return rc;
    if (a.c.rows == 0 || a.c.n_seqs == 0) return BTL_OK;
    a.p = btl::plan_paged_attention(n_heads, a.c, dtype == BTL_BF16);
    if (!btl::paged_attention_fits(a.c, a.p)) return fail_msg(BTL_ERR_SHAPE, "batch too large for one launch");
    if ((rc = check_pointers(cache, batch, &a.c))) return rc;
    if (!q || !out) return fail_msg(BTL_ERR_LAYOUT, "null pointer");
    if (!aligned16(q) || !aligned16(out)) return fail_msg(BTL_ERR_LAYOUT, "q and out must be 16-byte aligned");
    const size_t qn = (size_t)a.c.rows * n_heads * a.c.hd * (dtype == BTL_F32 ? 4 : 2);
    if (overlap(out, qn, q, qn)) return fail_msg(BTL_ERR_LAYOUT, "out overlaps q");
    int dev;
    if ((rc = btl::host::device(&dev))) return rc;
    a.parts = a.p.parts();
    const size_t need = attention_bytes(a.c, n_heads, a.p);
    if (need) {
        void* w = nullptr;
        if ((rc = btl::host::workspace(dev, ws, ws_bytes, need, &w, (hipStream_t)stream))) return rc;
        a.part_o = (float*)w;
        a.part_ml = (float*)((uint8_t*)w + up256((size_t)a.c.rows * n_heads * a.parts * a.c.hd * 4));
    }
    a.q = q;
    a.out = out;
    a.nh = (int)n_heads;
    a.group = (int)n_heads / a.c.nkv;
    a.group_mul = (uint32_t)((((int64_t)1 << 31) + a.group - 1) / a.group);
    a.scale_log2 = (float)(1.4426950408889634074 / std::sqrt((double)a.c.hd));
    a.bf = dtype == BTL_BF16;
    const hipError_t e = btl::launch_paged_attention(a, (hipStream_t)stream);
    return e == hipSuccess ? BTL_OK : hip_error(e, "paged attention kernel launch");
}

size_t btl_sample_workspace_bytes(int64_t rows, int64_t n)
{
    if (rows < 1 || rows > 65535 || n < 1 || n > (1 << 22)) return 0;
    return sample_ws(rows, n).total;
}

int btl_sample(const float* logits, int64_t rows, int64_t n, int64_t ld, const float* temperature,
               const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* ids,
               float* probs, void* ws, size_t ws_bytes, void* stream)
{
    if (rows < 0 || rows > 65535) return failf(BTL_ERR_SHAPE, "%lld rows: at most 65535", (long long)rows);
    if (n < 1 || n > (1 << 22)) return failf(BTL_ERR_SHAPE, "%lld logits a row: need 1 .. 2^22", (long long)n);
    if (ld < n || ld > ((int64_t)1 << 40)) return failf(BTL_ERR_SHAPE, "row stride %lld is less than the row of %lld", (long long)ld, (long long)n);
    if (rows == 0) return BTL_OK;
    if (!logits || !u || !ids) return fail_msg(BTL_ERR_LAYOUT, "null pointer");
    if (((uintptr_t)logits | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p |
         (uintptr_t)u | (uintptr_t)ids | (uintptr_t)probs) & 3u)
        return fail_msg(BTL_ERR_LAYOUT, "arrays must be 4-byte aligned");
    int dev, rc;
    if ((rc = btl::host::device(&dev))) return rc;
    const SampleWs w = sample_ws(rows, n);
    void* p = nullptr;
    if ((rc = btl::host::workspace(dev, ws, ws_bytes, w.total, &p, (hipStream_t)stream))) return rc;
    btl::SampleArgs a{};
    a.logits = logits;
    a.ld = ld;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.u = u;
    a.ids = ids;
    a.probs = probs;
    a.best = (uint64_t*)p;
    a.mass = (uint64_t*)((uint8_t*)p + w.mass);
    a.count = (uint32_t*)((uint8_t*)p + w.count);
    a.rows = (int)rows;
    a.n = (int)n;
    a.slice = btl::sample_slice(rows, n);
    a.slices = (int)((n + a.slice - 1) / a.slice);
    const hipError_t e = btl::launch_sample(a, (hipStream_t)stream);
    return e == hipSuccess ? BTL_OK : hip_error(e, "sampling kernel launch");
}

}  // extern "C"
