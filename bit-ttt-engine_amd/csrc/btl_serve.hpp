// btl_serve.hpp -- kernel arguments and launchers of the batched serving ops
// (btl_serve.hip, btl_share.hip, btl_evict.hip, btl_sample.hip), checked and filled by btl_serve_api.cpp.
// Not part of the public ABI.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

namespace btl {

// A paged cache and the sequences of one call (btl_kv_paged_t, btl_paged_batch_t).
struct Paged {
    uint8_t* k;    // [n_pages][nkv][ps][hd]
    uint8_t* v;    // [n_pages][nkv][ps / 16][hd][16]
    float* ks;     // [n_pages][nkv][ps]
    float* vs;
    const int32_t* row_start;
    const int32_t* pos;
    const int32_t* pages;
    int n_pages, nkv, ps, hd;
    int ppg;             // groups of 16 slots a page
    uint32_t ppg_mul;    // ceil(2^31 / ppg): g / ppg = (2 g * ppg_mul) >> 32 for g < 2^19, ppg <= 2^12
    int n_seqs, max_pages, rows, max_rows;
    int cap;             // tokens a sequence may have: min(max_len, max_pages * ps, 2^23)
};

struct PagedAppend {
    Paged c;
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    const float* cos_t;
    const float* sin_t;
    int rope_len, nh;
    int bf;  // rows are bf16
    const int32_t* shift;  // RoPE positions less positions, a sequence, or NULL
};
hipError_t launch_paged_append(const PagedAppend& a, hipStream_t st);

struct PagedRead {
    Paged c;
    void* k_out;
    void* v_out;
    int bf;
};
hipError_t launch_paged_read(const PagedRead& a, hipStream_t st);

// How one attention call splits its work: sequences of at most `lo` rows times
// query heads of a group go to the token form, the others to the tile form;
// each takes its keys in chunks (multiples of 256).
constexpr int kTokRows = 16;    // rows times heads of one workgroup of the token form, at most
struct AttnPlan {
    int lo;               // 0: no token form, INT_MAX: no tile form
    int tok_w;            // waves of a workgroup of the token form
    int tok_c, tile_c;    // keys a chunk
    int tok_n, tile_n;    // chunks of max_len keys
    int tile_rows;        // rows times heads of one workgroup of the tile form: 64 or 128
    int tiles;            // workgroups along the rows of the tile form, at most; over a prefix a list's of the token form
    int parts() const { return tok_n > tile_n ? tok_n : tile_n; }
};
AttnPlan plan_paged_attention(int64_t n_heads, const Paged& c, bool bf);
// its launches stay within a grid's size
bool paged_attention_fits(const Paged& c, const AttnPlan& p);

struct PagedAttn {
    Paged c;
    const void* q;
    void* out;
    float* part_o;   // [rows * nh][parts][hd]
    float* part_ml;  // [rows * nh][parts][2]: log2-domain maximum, sum
    AttnPlan p;
    int parts;
    int nh, group;
    uint32_t group_mul;  // ceil(2^31 / group): m / group = (2 m * group_mul) >> 32 for m < 2^27, group <= 16
    float scale_log2;  // log2(e) / sqrt(hd)
    int bf;
};
hipError_t launch_paged_attention(const PagedAttn& a, hipStream_t st);

// Attention beside a prefix that row lists share, and with the rows' weights added up.
struct PagedShare : PagedAttn {
    Paged g;       // the prefix: its lists of rows and pages (n_seqs 0: none)
    AttnPlan gp;
    int own0;      // a row's parts: the prefix's chunks, and from here on its sequence's
    int split;     // a sequence of one chunk is merged as well
    float* ml;     // [rows * nh][2]: a row's maximum and sum (log2 domain), or NULL
    // the token form's scores, log2 domain, -inf where a row does not see: [n_seqs][nkv][score_rows][score_ld]
    float* scores;
    int score_rows;
    int score_ld;
    // accounted weights
    float* weight;  // [n_seqs][nkv][ld]
    int64_t ld;
    float* sums;    // [splits][n_seqs][nkv][score_ld]: a position's weight from a share of the rows
    int splits;     // shares of the rows of a sequence that is too long for the token form's scores
    int scored;     // sequences of the token form have scores
};
// fills in a's split of the work; false: too large for one launch
bool plan_paged_share(int64_t n_heads, PagedShare& a, bool bf, bool account);
hipError_t launch_paged_share(const PagedShare& a, hipStream_t st);

struct PagedEvict {
    Paged c;
    // a head's weights and tokens lie ld apart
    const float* weight;
    const int32_t* token;
    const int32_t* filled;
    const int32_t* shift;
    float* weight_out;
    int32_t* token_out;
    int32_t* filled_out;
    int32_t* shift_out;
    int64_t ld, ld_out;
    const int32_t* keep;
    const int32_t* sink;    // or NULL
    const int32_t* recent;  // or NULL
    int32_t* held;
    int max_keep;
    int spans;         // of kEvictSpan positions: ceil(cap / kEvictSpan)
    int32_t* from;     // [n_seqs][nkv][cap]
    // where there are several spans
    int32_t* movers;   // [n_seqs][nkv][cap]
    uint32_t* keys;    // [n_seqs][nkv][cap]
    uint32_t* counts;  // [n_seqs][nkv][spans][kEvictBins / 2]
    int32_t* spanned;  // [n_seqs][nkv][spans][4]
    int32_t* holes;    // [n_seqs][nkv]
    int32_t* was;      // [2][n_seqs]: filled and shift as they came in
};
constexpr int kEvictSpan = 8192;
constexpr int kEvictBins = 2048;
// workgroups along the slots that may be written to
inline int evict_blocks(const PagedEvict& a)
{
    const int most = a.max_keep < a.c.cap ? a.max_keep : a.c.cap;
    return most > 64 ? (most + 63) / 64 : 1;
}
hipError_t launch_paged_evict(const PagedEvict& a, hipStream_t st);

// sampling
constexpr int kSampleBins = 1024;
int sample_slice(int64_t rows, int64_t n);  // logits of one workgroup of the first two launches
struct SampleArgs {
    const float* logits;
    int64_t ld;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int32_t* ids;
    float* probs;
    uint64_t* best;   // [rows][slices] largest (key, index) word of a slice
    uint64_t* mass;   // [rows][kSampleBins]
    uint32_t* count;  // [rows][kSampleBins]
    int rows, n, slice, slices;
};
hipError_t launch_sample(const SampleArgs& a, hipStream_t st);

}  // namespace btl
