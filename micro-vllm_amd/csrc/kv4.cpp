// kv4.cpp -- C entry points of attention over 4-bit keys and values: argument checks and
// launches (the kernels are in kern_kv4.hip, kern_attn.hip and kern_prompt.hip).  The calls share no scratch
// and keep no state: every buffer is the caller's.
#include "../../include/mvllm_hip.h"

#include "kv4.h"

#include <cmath>
#include <cstring>
#include <string>

#include "kv4_common.h"

namespace mvllm_hip {
void set_error(const std::string &s);  // mvllm_hip.cpp: the text of mvllm_hip_last_error
int ready_device();                    // mvllm_hip.cpp: the device of mvllm_hip_init, or -1
int kv4_rows_option();                 // mvllm_hip.cpp: option "kv4_rows"

namespace {

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool head_dim_ok(int d) { return d == 64 || d == 128 || d == 192 || d == 256; }

int refuse(const std::string &s) {
    set_error(s);
    return 0;
}

bool ranges_meet(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

// Launches go to the device of mvllm_hip_init whatever the thread's current device is (the
// null stream is the current device's).
class OnDevice {
    int prev_ = -1, dev_;

  public:
    explicit OnDevice(int dev) : dev_(dev) {
        if (hipGetDevice(&prev_) != hipSuccess)
            prev_ = -1;
        if (prev_ != dev_)
            (void)hipSetDevice(dev_);
    }
    ~OnDevice() {
        if (prev_ >= 0 && prev_ != dev_)
            (void)hipSetDevice(prev_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
};

// Runs launch() on the library's device; 1, or 0 with the error's text.
template <typename F> int enqueue(const char *what, void *stream, F &&launch) {
    const int dev = ready_device();
    if (dev < 0)
        return refuse(std::string(what) + ": mvllm_hip_init has not succeeded");
    if (stream) {
        int sd = dev;
        if (hipStreamGetDevice(static_cast<hipStream_t>(stream), &sd) != hipSuccess || sd != dev) {
            (void)hipGetLastError();
            return refuse(std::string(what) + ": a stream of another device");
        }
    }
    const OnDevice on(dev);
    const hipError_t e = launch(static_cast<hipStream_t>(stream));
    if (e != hipSuccess)
        return refuse(std::string(what) + ": " + hipGetErrorString(e));
    return 1;
}

const char *const kCacheRule =
    ": bad cache (fmt 4 or 7, head_dim 64, 128, 192 or 256, 1 <= n_kv <= 1024, page a multiple "
    "of 16 up to 1024, n_pages >= 1, 16-byte aligned k, ks, v, vs)";

bool view_of(const mvllm_kv4 *c, Kv4View &v) {
    if (!c || !c->k || !c->ks || !c->v || !c->vs || (c->fmt != 4 && c->fmt != 7) ||
        !head_dim_ok(c->head_dim) || c->n_kv < 1 || c->n_kv > 1024 || c->page < 16 ||
        c->page > 1024 || c->page % 16 || c->n_pages < 1 || !aligned16(c->k) ||
        !aligned16(c->ks) || !aligned16(c->v) || !aligned16(c->vs) ||
        (reinterpret_cast<uintptr_t>(c->score) & 3))
        return false;
    v.k = static_cast<uint8_t *>(c->k);
    v.ks = static_cast<uint8_t *>(c->ks);
    v.v = static_cast<uint8_t *>(c->v);
    v.vs = static_cast<uint8_t *>(c->vs);
    v.score = c->score;
    v.n_kv = c->n_kv;
    v.page = c->page;
    v.n_pages = c->n_pages;
    v.rcp = kv4_page_rcp(c->page);
    return true;
}

bool table_ok(const mvllm_kv4 *c, int max_pages) {
    return max_pages >= 1 && (long long)max_pages * c->page <= (1ll << 30);
}

// (a launch has fewer than 2^32 threads along a side: a workgroup a token)
bool tokens_ok(int n_tok) { return n_tok >= 1 && n_tok <= (1 << 23); }

const char *const kSeqRule =
    ": bad sequences (q_start, lens and table, 1 <= n_seq <= 65535, 1 <= n_tok <= 2^23, max_pages "
    ">= 1, max_pages * page <= 2^30, n_tok * n_kv * head_dim <= 2^34)";

bool seqs_of(const mvllm_kv4 *c, int n_tok, const int *q_start, const int *lens, const int *table,
             int n_seq, int max_pages, Kv4Seqs &s) {
    if (!q_start || !lens || !table || !tokens_ok(n_tok) || n_seq < 1 || n_seq > 65535 ||
        !table_ok(c, max_pages) || (long long)n_tok * c->n_kv * c->head_dim > (1ll << 34))
        return false;
    s = Kv4Seqs{q_start, lens, table, n_seq, max_pages, n_tok};
    return true;
}

// A row of heads of `dtype`: 16-byte aligned, every `stride` elements.
bool rows_ok(const void *p, long long stride, int dtype) {
    return p && aligned16(p) && stride >= 0 && stride <= (1ll << 36) &&
           stride % (dtype == KV4_BF16 ? 8 : 4) == 0;
}

bool dtype_ok(int dtype) { return dtype == KV4_F32 || dtype == KV4_BF16; }

size_t rows_bytes(int dtype, int n_tok, long long stride, long long row) {
    return (size_t)((n_tok - 1) * stride + row) * (dtype == KV4_BF16 ? 2 : 4);
}

}  // namespace
}  // namespace mvllm_hip

using namespace mvllm_hip;

extern "C" {

long long mvllm_kv4_geom(int fmt, int n_kv, int head_dim, int page, long long bytes[4]) {
    if ((fmt != 4 && fmt != 7) || n_kv < 1 || n_kv > 1024 || !head_dim_ok(head_dim) || page < 16 ||
        page > 1024 || page % 16)
        return -1;
    const long long rows = (long long)n_kv * page;
    const long long codes = rows * (head_dim / 2);
    const long long scales = rows * (fmt == 4 ? head_dim / 64 * 4 : head_dim / 32);
    if (bytes) {
        bytes[0] = bytes[2] = codes;
        bytes[1] = bytes[3] = scales;
    }
    return 2 * (codes + scales);
}

int mvllm_hip_qk_norm_rope_dev(int dtype, int n_tok, int head_dim, const void *q,
                               long long q_stride, int n_q, void *qo, long long qo_stride,
                               const void *k, long long k_stride, int n_kv, void *ko,
                               long long ko_stride, const float *wq, const float *wk, float eps,
                               const int *pos, const double *freq, int rot, int interleaved,
                               void *stream) {
    set_error("");
    if (!dtype_ok(dtype) || !tokens_ok(n_tok) || !head_dim_ok(head_dim) || n_q < 0 || n_kv < 0 ||
        n_q + (long long)n_kv < 1 || n_q + (long long)n_kv > 65535 ||
        (n_q && (!rows_ok(q, q_stride, dtype) || !rows_ok(qo, qo_stride, dtype) ||
                 (n_tok > 1 && qo_stride < (long long)n_q * head_dim))) ||
        (n_kv && (!rows_ok(k, k_stride, dtype) || !rows_ok(ko, ko_stride, dtype) ||
                  (n_tok > 1 && ko_stride < (long long)n_kv * head_dim))) ||
        !aligned16(wq) || !aligned16(wk) || !(eps >= 0.f) ||
        (freq && (!pos || rot < 16 || rot > head_dim || rot % 16)))
        return refuse("qk_norm_rope_dev: bad arguments (dtype 0 or 1, 1 <= n_tok <= 2^23, head_dim "
                      "64, 128, 192 or 256, 1 <= n_q + n_kv <= 65535, 16-byte aligned rows and "
                      "weights, output rows apart, eps >= 0, with freq: pos and rot a multiple of "
                      "16 up to head_dim)");
    RopeArgs a{};
    a.q = q;
    a.k = k;
    a.qo = qo;
    a.ko = ko;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.qo_stride = qo_stride;
    a.ko_stride = ko_stride;
    a.wq = wq;
    a.wk = wk;
    a.pos = pos;
    a.freq = freq;
    a.eps = eps;
    a.n_q = n_q;
    a.n_kv = n_kv;
    a.rot = rot;
    return enqueue("qk_norm_rope_dev", stream, [&](hipStream_t st) {
        return launch_qk_norm_rope(dtype, n_tok, head_dim, interleaved != 0, a, st);
    });
}

int mvllm_hip_kv4_append_dev(const mvllm_kv4 *cache, int dtype, const void *k, long long k_stride,
                             const void *v, long long v_stride, int n_tok, const int *q_start,
                             const int *lens, const int *table, int n_seq, int max_pages,
                             void *stream) {
    set_error("");
    Kv4View c;
    Kv4Seqs s;
    if (!view_of(cache, c))
        return refuse(std::string("kv4_append_dev") + kCacheRule);
    if (!seqs_of(cache, n_tok, q_start, lens, table, n_seq, max_pages, s))
        return refuse(std::string("kv4_append_dev") + kSeqRule);
    if (!dtype_ok(dtype) || !rows_ok(k, k_stride, dtype) || !rows_ok(v, v_stride, dtype))
        return refuse("kv4_append_dev: bad arguments (dtype 0 or 1, 16-byte aligned rows)");
    return enqueue("kv4_append_dev", stream, [&](hipStream_t st) {
        return launch_kv4_append(cache->fmt, cache->head_dim, dtype, c, s, k, k_stride, v,
                                 v_stride, st);
    });
}

int mvllm_hip_kv4_read_dev(const mvllm_kv4 *cache, int dtype, void *k, void *v, int n_tok,
                           const int *q_start, const int *lens, const int *table, int n_seq,
                           int max_pages, void *stream) {
    set_error("");
    Kv4View c;
    Kv4Seqs s;
    if (!view_of(cache, c))
        return refuse(std::string("kv4_read_dev") + kCacheRule);
    if (!seqs_of(cache, n_tok, q_start, lens, table, n_seq, max_pages, s))
        return refuse(std::string("kv4_read_dev") + kSeqRule);
    const long long row = (long long)c.n_kv * cache->head_dim;
    const size_t bytes = rows_bytes(dtype, n_tok, row, row);
    if (!dtype_ok(dtype) || !k || !v || !aligned16(k) || !aligned16(v) ||
        ranges_meet(k, bytes, v, bytes))
        return refuse("kv4_read_dev: bad arguments (dtype 0 or 1, 16-byte aligned k and v that do "
                      "not overlap)");
    return enqueue("kv4_read_dev", stream, [&](hipStream_t st) {
        return launch_kv4_read(cache->fmt, cache->head_dim, dtype, c, s, k, v, st);
    });
}

static bool attention_sizes_ok(int head_dim, int n_kv, int n_q, int n_tok, int n_seq, int max_new,
                               int max_len) {
    return head_dim_ok(head_dim) && n_kv >= 1 && n_kv <= 1024 && n_q >= n_kv && n_q % n_kv == 0 &&
           n_q <= 65535 && n_q / n_kv <= 1024 && tokens_ok(n_tok) && n_seq >= 1 &&
           n_seq <= 65535 && max_new >= 1 && max_len >= 1 && max_len <= (1 << 30) &&
           (long long)n_tok * n_q <= (1ll << 30) &&
           (long long)max_new * n_q <= (1ll << 30);
}

long long mvllm_hip_kv4_attention_work(int n_kv, int head_dim, int n_q, int n_tok, int n_seq,
                                       int max_new, int max_len, int weights) {
    if (!attention_sizes_ok(head_dim, n_kv, n_q, n_tok, n_seq, max_new, max_len))
        return -1;
    return (long long)kv4_attention_bytes(head_dim, n_kv, n_q, n_tok, n_seq, max_new, max_len,
                                          weights != KV4_WEIGHTS_NONE);
}

int mvllm_hip_kv4_attention_dev(const mvllm_kv4 *cache, int dtype, const void *q,
                                long long q_stride, int n_q, int n_tok, const int *q_start,
                                const int *lens, const int *table, int n_seq, int max_pages,
                                int max_new, int max_len, float scale, int window, int weights,
                                void *out, void *work, size_t work_bytes, void *stream) {
    set_error("");
    AttnArgs a{};
    if (!view_of(cache, a.c))
        return refuse(std::string("kv4_attention_dev") + kCacheRule);
    if (!seqs_of(cache, n_tok, q_start, lens, table, n_seq, max_pages, a.s))
        return refuse(std::string("kv4_attention_dev") + kSeqRule);
    const int D = cache->head_dim;
    if (!dtype_ok(dtype) || !rows_ok(q, q_stride, dtype) || !out || !aligned16(out) ||
        !attention_sizes_ok(D, a.c.n_kv, n_q, n_tok, n_seq, max_new, max_len) ||
        !std::isfinite(scale) || window < 0 ||
        ranges_meet(q, rows_bytes(dtype, n_tok, q_stride, (long long)n_q * D), out,
                    rows_bytes(dtype, n_tok, (long long)n_q * D, (long long)n_q * D)))
        return refuse("kv4_attention_dev: bad arguments (dtype 0 or 1, n_q a multiple of n_kv up "
                      "to 1024 times it, 16-byte aligned q and out that do not overlap, max_new "
                      ">= 1, 1 <= max_len <= 2^30, n_tok * n_q and max_new * n_q up to 2^30, "
                      "finite scale, window >= 0)");
    if (weights < KV4_WEIGHTS_NONE || weights > KV4_WEIGHTS_STORE ||
        (weights != KV4_WEIGHTS_NONE && !cache->score))
        return refuse("kv4_attention_dev: weights is 0, 1 or 2, and the cache has a score array "
                      "where it is not 0");
    const AttnPlan p =
        kv4_attention_plan(kv4_rows_option(), cache->fmt, dtype, D, a.c.n_kv, n_q, n_tok, n_seq,
                           max_new, max_len, window, weights != KV4_WEIGHTS_NONE);
    const size_t need = kv4_attention_bytes(D, a.c.n_kv, n_q, n_tok, n_seq, max_new, max_len,
                                            weights != KV4_WEIGHTS_NONE);
    if (need > work_bytes || (need && (!work || !aligned16(work))))
        return refuse("kv4_attention_dev: the workspace needs " + std::to_string(need) +
                      " bytes, 16-byte aligned (mvllm_hip_kv4_attention_work)");
    char *w = static_cast<char *>(work);
    a.q = q;
    a.out = out;
    a.part = reinterpret_cast<float *>(w + p.part);
    a.ml = reinterpret_cast<float2 *>(w + p.ml);
    a.lse = weights != KV4_WEIGHTS_NONE ? reinterpret_cast<float *>(w + p.lse) : nullptr;
    a.logit = p.logits && !p.waves ? reinterpret_cast<float *>(w + p.logit) : nullptr;
    a.logits = p.logits;
    a.group_rcp = (1ull << 40) / (unsigned)(n_q / a.c.n_kv) + 1;
    a.q_stride = q_stride;
    a.n_q = n_q;
    a.group = n_q / a.c.n_kv;
    a.splits = p.splits;
    a.chunk = p.chunk;
    a.tiles = p.tiles;
    a.waves = p.waves;
    a.few = (long long)max_new * a.group <= 16;
    const double scale2 = (double)scale * 1.44269504088896340736;
    a.scale2 = (float)scale2;
    a.scale2_lo = (float)(scale2 - (double)a.scale2);
    a.window = window;
    a.weights = weights;
    return enqueue("kv4_attention_dev", stream, [&](hipStream_t st) {
        return launch_kv4_attention(cache->fmt, D, dtype, a, max_len, st);
    });
}

int mvllm_hip_kv4_evict_dev(const mvllm_kv4 *cache, const int *lens, const int *table, int n_seq,
                            int max_pages, int max_len, int keep, int recent,
                            const int *dst_table, int dst_max_pages, int *kept, int *new_lens,
                            void *stream) {
    set_error("");
    EvictArgs a{};
    if (!view_of(cache, a.c) || !cache->score)
        return refuse(std::string("kv4_evict_dev") + kCacheRule + ", and a score array");
    if (!lens || !table || n_seq < 1 || n_seq > 65535 || !table_ok(cache, max_pages) ||
        max_len < 1 || keep < 1 || keep > (1 << 29) || recent < 0 || recent > keep || !dst_table ||
        !table_ok(cache, dst_max_pages) || (long long)dst_max_pages * cache->page < keep ||
        !kept || !new_lens ||
        ranges_meet(table, (size_t)n_seq * max_pages * 4, dst_table,
                    (size_t)n_seq * dst_max_pages * 4) ||
        ranges_meet(lens, (size_t)n_seq * 4, new_lens, (size_t)n_seq * 4))
        return refuse("kv4_evict_dev: bad arguments (lens, table, 1 <= n_seq <= 65535, max_pages * "
                      "page <= 2^30, max_len >= 1, 0 <= recent <= keep, 1 <= keep <= 2^29, a "
                      "dst_table of its own whose pages hold keep tokens, kept, and new_lens "
                      "apart from lens)");
    a.lens = lens;
    a.table = table;
    a.dst_table = dst_table;
    a.kept = kept;
    a.new_lens = new_lens;
    a.n_seq = n_seq;
    a.max_pages = max_pages;
    a.dst_max_pages = dst_max_pages;
    a.keep = keep;
    a.recent = recent;
    return enqueue("kv4_evict_dev", stream, [&](hipStream_t st) {
        return launch_kv4_evict(cache->fmt, cache->head_dim, a, max_len, st);
    });
}

}  // extern "C"
