// kv4.h -- structures of the 4-bit key/value cache's kernels (kern_kv4.hip, kern_attn.hip)
// and of their host side (kv4.cpp).
#pragma once

#include "moe_internal.h"

namespace mvllm_hip {

enum : int { KV4_F32 = 0, KV4_BF16 = 1 };
enum : int { KV4_WEIGHTS_NONE = 0, KV4_WEIGHTS_ADD = 1, KV4_WEIGHTS_STORE = 2 };

// Quantization limits (see the header): magnitudes above kKv4Held are held as it, int4 groups
// whose largest magnitude is below kKv4Tiny as zeros.
constexpr float kKv4Held = 0x1.8p127f;  // 6 * 2^125
constexpr float kKv4Tiny = 0x1p-100f;

// The cache as the kernels see it.  Row (page, head, slot) of k / v has head_dim / 2 bytes of
// codes; of ks / vs head_dim / 64 f32 (fmt 4) or head_dim / 32 bytes (fmt 7).
struct Kv4View {
    uint8_t *k, *v;
    uint8_t *ks, *vs;
    float *score;  // may be null
    int n_kv, page, n_pages;
    uint32_t rcp;  // see kv4_page_of
};

// The tokens of a call: sequence b's new tokens are rows [q_start[b], q_start[b + 1]), the
// last of its lens[b] tokens; token t lies in page table[b][t / page].
struct Kv4Seqs {
    const int *q_start, *lens, *table;
    int n_seq, max_pages, n_tok;
};

struct RopeArgs {
    const void *q, *k;
    void *qo, *ko;
    long long q_stride, k_stride, qo_stride, ko_stride;  // elements between tokens
    const float *wq, *wk;  // may be null
    const int *pos;
    const double *freq;    // may be null
    float eps;
    int n_q, n_kv, rot, heads_per_wg;
};

struct AttnArgs {
    Kv4View c;
    Kv4Seqs s;
    const void *q;
    void *out;
    float *part;   // [splits][n_tok][n_q][D] sums relative to the split's maximum
    float2 *ml;    // [splits][n_tok][n_q] maximum (log2) and sum of a split
    float *lse;    // [n_tok][n_q] log2 of a row's sum of exponentials (-inf: sees nothing), or null
    float *logit;  // [n_tok][n_q][logits] products of queries and keys, or null
    int logits;
    unsigned long long group_rcp;  // floor(2^40 / group) + 1
    long long q_stride;
    int n_q, group, splits, chunk, tiles, waves;
    bool few;  // at most 16 rows a sequence and kv head, by max_new
    float scale2, scale2_lo;  // scale * log2(e), and what the f32 leaves of it
    int window, weights;
};

struct EvictArgs {
    Kv4View c;
    const int *lens, *table, *dst_table;
    int *kept, *new_lens;
    int n_seq, max_pages, dst_max_pages, keep, recent;
};

hipError_t launch_qk_norm_rope(int dtype, int n_tok, int head_dim, bool interleaved, RopeArgs a,
                               hipStream_t st);
hipError_t launch_kv4_append(int fmt, int head_dim, int dtype, const Kv4View &c, const Kv4Seqs &s,
                             const void *k, long long k_stride, const void *v, long long v_stride,
                             hipStream_t st);
hipError_t launch_kv4_read(int fmt, int head_dim, int dtype, const Kv4View &c, const Kv4Seqs &s,
                           void *k, void *v, hipStream_t st);
hipError_t launch_kv4_evict(int fmt, int head_dim, const EvictArgs &a, int max_len, hipStream_t st);

// How a call is cut: the parts of its workspace follow from it.
struct AttnPlan {
    int waves;  // 0: 16 rows a workgroup, else 32 a wave
    int splits, chunk, tiles;
    int logits;           // logits kept of each row (0: none)
    size_t part, ml, lse, logit, bytes;  // offsets into the workspace, and its size
};
// choice: 0 by size, 1 the 16-row kernel, 2 the other.
AttnPlan kv4_attention_plan(int choice, int fmt, int dtype, int head_dim, int n_kv, int n_q, int n_tok,
                            int n_seq, int max_new, int max_len, int window, bool weights);
// The workspace that serves every choice, format, type and window.
size_t kv4_attention_bytes(int head_dim, int n_kv, int n_q, int n_tok, int n_seq, int max_new,
                           int max_len, bool weights);
hipError_t launch_kv4_prompt(int fmt, int head_dim, int dtype, const AttnArgs &a, hipStream_t st);
hipError_t launch_kv4_attention(int fmt, int head_dim, int dtype, const AttnArgs &a, int max_len,
                                hipStream_t st);

}  // namespace mvllm_hip
