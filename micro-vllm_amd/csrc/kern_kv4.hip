// kern_kv4.hip -- what stands around the attention kernels for gfx950: the norms of query and
// key heads with the position rotation, the 4-bit key/value cache's quantizing append and its
// read-back, and the eviction of its least attended tokens.
#include "kv4_common.h"

#include <algorithm>
#include <cmath>

namespace mvllm_hip {

// ---- norms of query and key heads, and the rotation --------------------------------------

// y = x / sqrt(mean(x^2) + eps) * w over each head's D elements, then the pairs (a, b) of its
// first `rot` elements turn by pos * freq[j]: (a cos - b sin, b cos + a sin), b = a's partner
// rot / 2 further on, or the next element (INTER).
//
// One workgroup: heads_per_wg heads of one token.  A head lies in LPH lanes, 8 consecutive
// elements each (NC blocks of them for D = 192), so its sum of squares is a butterfly within
// the wave.  The token's cosines and sines are formed once per workgroup, in LDS: the angle in
// 64 bits (pos up to 2^31 turns an f32 angle by radians), reduced by quarter turns to +-1/8
// turn before it is rounded to f32, so far positions are as exact as near ones.  Bound by the
// bytes: 4096 tokens, 72 heads of 128 in bf16 read and written in 33.6 us, 4.5 TB/s (a large
// copy reaches 5.0).
template <typename T, int D, bool INTER>
__global__ __launch_bounds__(256) void k_qk_norm_rope(RopeArgs A) {
    constexpr int LPH = D == 64 || D == 192 ? 8 : D / 8, NC = D / 8 / LPH, HPW = 64 / LPH;
    __shared__ float2 turn[D / 2];
    __shared__ __attribute__((aligned(16))) float row[4][INTER ? 4 : HPW * D];
    const int tok = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int li = lane & (LPH - 1), hi = lane / LPH;
    const int total = A.n_q + A.n_kv;
    const int h0 = blockIdx.y * A.heads_per_wg, h1 = min(total, h0 + A.heads_per_wg);
    const int rot = A.freq ? A.rot : 0;
    if (tid < rot / 2) {
        const double t = (double)A.pos[tok] * A.freq[tid] * 0.63661977236758134308;  // quarters
        const double n = rint(t);
        const float r = (float)(t - n);
        float s, c;
        sincospif(0.5f * r, &s, &c);
        const int quarter = (int)(long long)n & 3;
        const float cs = quarter & 1 ? s : c, sn = quarter & 1 ? c : s;
        turn[tid] = make_float2(quarter == 1 || quarter == 2 ? -cs : cs, quarter >= 2 ? -sn : sn);
    }
    __syncthreads();
    for (int hb = h0 + wave * HPW; hb < h1; hb += 4 * HPW) {  // wave-uniform
        const int h = hb + hi;
        const bool live = h < h1, isq = h < A.n_q;
        const T *x = isq ? static_cast<const T *>(A.q) + (size_t)tok * A.q_stride + (size_t)h * D
                         : static_cast<const T *>(A.k) + (size_t)tok * A.k_stride +
                               (size_t)(h - A.n_q) * D;
        T *y = isq ? static_cast<T *>(A.qo) + (size_t)tok * A.qo_stride + (size_t)h * D
                   : static_cast<T *>(A.ko) + (size_t)tok * A.ko_stride + (size_t)(h - A.n_q) * D;
        const float *w = isq ? A.wq : A.wk;
        float v[NC][8], ss = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[c][i] = 0.f;
            if (live)
                Vec8<T>::load(x + (c * LPH + li) * 8, v[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                ss = fmaf(v[c][i], v[c][i], ss);
        }
#pragma unroll
        for (int o = LPH / 2; o >= 1; o >>= 1)
            ss += __shfl_xor(ss, o);
        const float inv = 1.f / sqrtf(ss / (float)D + A.eps);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = (c * LPH + li) * 8;
            float g[8];
            if (w)
                Vec8<float>::load(w + d, g);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[c][i] = v[c][i] * inv * (w ? g[i] : 1.f);
            if constexpr (!INTER)
                Vec8<float>::store(row[wave] + hi * D + d, v[c]);
        }
        // the wave's own rows: only its LDS writes have to come before its reads
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = (c * LPH + li) * 8;
            if (d < rot) {
                if constexpr (INTER) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const float2 t = turn[(d + i) / 2];
                        const float a = v[c][i], b = v[c][i + 1];
                        v[c][i] = a * t.x - b * t.y;
                        v[c][i + 1] = b * t.x + a * t.y;
                    }
                } else {  // rot % 16 == 0: the 8 elements have their partners 8 in a row too
                    const bool low = d < rot / 2;
                    const int j = low ? d : d - rot / 2;
                    float p[8];
                    Vec8<float>::load(row[wave] + hi * D + (low ? d + rot / 2 : j), p);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 t = turn[j + i];
                        v[c][i] = low ? v[c][i] * t.x - p[i] * t.y : v[c][i] * t.x + p[i] * t.y;
                    }
                }
            }
            if (live)
                Vec8<T>::store(y + d, v[c]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

template <typename T, bool INTER>
static hipError_t rope_dim(int n_tok, int D, const RopeArgs &a, dim3 grid, hipStream_t st) {
    if (D == 64)
        hipLaunchKernelGGL((k_qk_norm_rope<T, 64, INTER>), grid, dim3(256), 0, st, a);
    else if (D == 128)
        hipLaunchKernelGGL((k_qk_norm_rope<T, 128, INTER>), grid, dim3(256), 0, st, a);
    else if (D == 192)
        hipLaunchKernelGGL((k_qk_norm_rope<T, 192, INTER>), grid, dim3(256), 0, st, a);
    else if (D == 256)
        hipLaunchKernelGGL((k_qk_norm_rope<T, 256, INTER>), grid, dim3(256), 0, st, a);
    else
        return hipErrorInvalidValue;
    return hipGetLastError();
}

hipError_t launch_qk_norm_rope(int dtype, int n_tok, int D, bool interleaved, RopeArgs a,
                               hipStream_t st) {
    const int per = 4 * (D == 64 || D == 192 ? 8 : 512 / D);  // heads of one pass of a workgroup
    const int total = a.n_q + a.n_kv;
    // All heads of a token in one workgroup, so that its angles are formed once (4096 tokens, 72
    // heads of 128 in bf16: 33.6 us, and 36.7 with a workgroup for each pass), unless that leaves
    // fewer than 2048 workgroups (16 tokens: one pass each, 3.6 us).
    const long long parts = (total + per - 1) / per;
    a.heads_per_wg = per * (int)std::max(1ll, std::min(parts, n_tok * parts / 2048));
    const dim3 grid((unsigned)n_tok, (unsigned)((total + a.heads_per_wg - 1) / a.heads_per_wg));
    if (dtype == KV4_BF16)
        return interleaved ? rope_dim<__bf16, true>(n_tok, D, a, grid, st)
                           : rope_dim<__bf16, false>(n_tok, D, a, grid, st);
    return interleaved ? rope_dim<float, true>(n_tok, D, a, grid, st)
                       : rope_dim<float, false>(n_tok, D, a, grid, st);
}

// ---- append and read-back -----------------------------------------------------------------

// The sequence of row `tok`, and the row's token in it (may be negative: none): the first that
// ends behind the row (q_start does not fall).  A wave looks at 64 ends at a time, of more
// sequences first at every 64th, so 16 and 4096 sequences take one and two round trips.
// False for rows behind the last sequence (or ahead of the first).
__device__ __forceinline__ bool kv4_find(const Kv4Seqs &s, int tok, int &seq, int &at, int &len) {
    const int lane = threadIdx.x & 63;
    int b0 = 0, b1 = s.n_seq;
    while (b1 - b0 > 64) {
        const int step = (b1 - b0 + 63) / 64;
        const uint64_t later = __ballot(s.q_start[min(b0 + (lane + 1) * step, b1)] > tok);
        if (!later)
            return false;
        b0 += (int)__builtin_ctzll(later) * step;
        b1 = min(b1, b0 + step);
    }
    const int b = min(b0 + lane, b1 - 1);
    const int end = s.q_start[b + 1], n = s.lens[b];
    const uint64_t later = __ballot(b0 + lane < b1 && end > tok);
    if (!later)
        return false;
    const int i = __builtin_ctzll(later);
    seq = b0 + i;
    len = __builtin_amdgcn_readlane(n, i);
    at = len - __builtin_amdgcn_readlane(end, i) + tok;
    return seq > 0 || tok >= s.q_start[0];
}

// Round to nearest, ties to even, of the real quotient x / s (s >= 2^-103): the product with
// the reciprocal may land on the wrong side of a border, which the signs of x - s (n +- 1/2),
// each formed with one rounding that keeps the sign, tell.
__device__ __forceinline__ int kv4_round(float x, float s, float inv) {
    const float n = rintf(x * inv);
    const float up = fmaf(-(n + 0.5f), s, x), down = fmaf(-(n - 0.5f), s, x);
    const bool odd = (int)n & 1;
    int r = (int)n;
    if (up > 0.f || (up == 0.f && odd))
        r += 1;
    else if (down < 0.f || (down == 0.f && odd))
        r -= 1;
    return min(7, max(-7, r));
}

// e2m1 code of q in [-6, 6]: the nearest value, a tie to the smaller magnitude, no -0 (the
// rule of the MXFP4 activation quantizer).
__device__ __forceinline__ uint32_t kv4_e2m1(float q) {
    const float m = fabsf(q);
    const uint32_t c = (m > 0.25f) + (m > 0.75f) + (m > 1.25f) + (m > 1.75f) + (m > 2.5f) +
                       (m > 3.5f) + (m > 5.f);
    return (q < 0.f && c > 0u) ? (c | 8u) : c;
}

// One wave: 64 blocks of 8 elements of one token's keys (grid y 0) or values (y 1); a group's
// largest magnitude is a butterfly over its 8 (int4) or 4 (MXFP4) lanes.  The wave's first
// loads are its elements and the sequences' ends and lengths, one round trip; the table
// entry is the second, then it stores.  Few tokens are bound by those two trips and the launch
// (16 tokens, 8 heads of 128: 4.0 us), many by their stores of 4 bytes a lane (4096 tokens, 8
// heads of 128 in bf16, 22 MB: 12.9 us, 1.7 TB/s; a wave with two heads in flight took 13.9,
// one with four tokens of four heads, a page's rows side by side, 14.5).
template <int FMT, typename T, int D>
__global__ __launch_bounds__(256) void k_kv4_append(Kv4View C, Kv4Seqs S, const T *k,
                                                    long long k_stride, const T *v,
                                                    long long v_stride, int chunks) {
    constexpr int BPH = D / 8;  // blocks of 8 in a head
    const int wid = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int tok = wid / chunks, lane = threadIdx.x & 63;
    if (tok >= S.n_tok)
        return;
    const int e = (wid - tok * chunks) * 64 + lane;
    const bool live = e < C.n_kv * BPH, isv = blockIdx.y;
    const int head = e / BPH, blk = e - head * BPH;
    const T *src = isv ? v + (size_t)tok * v_stride : k + (size_t)tok * k_stride;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live)
        Vec8<T>::load(src + (size_t)e * 8, x);
    int seq, at, len;
    if (!kv4_find(S, tok, seq, at, len) || at < 0)
        return;
    const int pg = kv4_page_of(C, at);
    const int phys = kv4_phys(C, S.table + (size_t)seq * S.max_pages, S.max_pages, pg);
    if (phys < 0)
        return;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = x[i] != x[i] ? 0.f : fmaxf(-kKv4Held, fminf(kKv4Held, x[i]));
        top = fmaxf(top, fabsf(x[i]));
    }
#pragma unroll
    for (int o = FMT == 4 ? 4 : 2; o >= 1; o >>= 1)
        top = fmaxf(top, __shfl_xor(top, o));
    const size_t r = kv4_row(C, phys, head, at - pg * C.page);
    uint32_t codes = 0;
    uint8_t *sc = isv ? C.vs : C.ks;
    if constexpr (FMT == 4) {
        const bool tiny = top < kKv4Tiny;
        const float s = tiny ? 0.f : top * (1.f / 7.f), inv = tiny ? 0.f : 1.f / s;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            codes |= (uint32_t)(tiny ? 8 : kv4_round(x[i], s, inv) + 8) << (4 * i);
        if (live && (blk & 7) == 0)
            reinterpret_cast<float *>(sc)[r * (D / 64) + blk / 8] = s;
    } else {
        // the smallest ex with top <= 6 * 2^ex: the rounded quotient's exponent gives it (the
        // next f32 above 6 * 2^ex divides to one above 2^ex)
        const uint32_t b = __float_as_uint(fmaxf(top, 0x1.8p-124f) / 6.f);
        const int ex = (int)(b >> 23) - 127 + ((b & 0x7fffffu) ? 1 : 0);  // -126 .. 125
        const float inv = __uint_as_float((uint32_t)(127 - ex) << 23);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            codes |= kv4_e2m1(fmaxf(-6.f, fminf(6.f, x[i] * inv))) << (4 * i);
        if (live && (blk & 3) == 0)
            sc[r * (D / 32) + blk / 4] = (uint8_t)(ex + 127);
    }
    if (!live)
        return;
    reinterpret_cast<uint32_t *>(isv ? C.v : C.k)[r * (D / 8) + blk] = codes;
    if (C.score && !isv && blk == 0)
        C.score[r] = 0.f;
}

// One wave: 64 blocks of 8 elements of one token's keys (grid y 0) or values (y 1), as the
// cache holds them.  Bound by its stores (32768 tokens of 8 heads of 128 to f32, 304 MB: 66 us, 4.6
// TB/s).
template <int FMT, typename T, int D>
__global__ __launch_bounds__(256) void k_kv4_read(Kv4View C, Kv4Seqs S, T *k, T *v, int chunks) {
    constexpr int BPH = D / 8;
    const int wid = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int tok = wid / chunks, lane = threadIdx.x & 63;
    if (tok >= S.n_tok)
        return;
    const int e = (wid - tok * chunks) * 64 + lane;
    const bool isv = blockIdx.y;
    int seq, at, len;
    if (!kv4_find(S, tok, seq, at, len))
        return;
    if (e >= C.n_kv * BPH)
        return;
    const int head = e / BPH, blk = e - head * BPH;
    const int pg = kv4_page_of(C, max(at, 0));
    const int phys = at < 0 ? -1
                            : kv4_phys(C, S.table + (size_t)seq * S.max_pages, S.max_pages, pg);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (phys >= 0) {
        const size_t r = kv4_row(C, phys, head, at - pg * C.page);
        const uint32_t codes = reinterpret_cast<const uint32_t *>(isv ? C.v : C.k)[r * (D / 8) + blk];
        const uint8_t *sc = isv ? C.vs : C.ks;
        const float s = FMT == 4 ? reinterpret_cast<const float *>(sc)[r * (D / 64) + blk / 8]
                                 : ue8m0_ref(sc[r * (D / 32) + blk / 4]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t n = (codes >> (4 * i)) & 15u;
            x[i] = (FMT == 4 ? (float)((int)n - 8) : e2m1_val(n)) * s;
        }
    }
    Vec8<T>::store((isv ? v : k) + ((size_t)tok * C.n_kv * BPH + e) * 8, x);
}

template <int FMT, typename T, int D>
static void append_one(const Kv4View &c, const Kv4Seqs &s, const void *k, long long ks,
                       const void *v, long long vs, hipStream_t st) {
    const int chunks = (c.n_kv * (D / 8) + 63) / 64;
    const unsigned wgs = (unsigned)(((size_t)s.n_tok * chunks + 3) / 4);
    hipLaunchKernelGGL((k_kv4_append<FMT, T, D>), dim3(wgs, 2), dim3(256), 0, st, c, s,
                       static_cast<const T *>(k), ks, static_cast<const T *>(v), vs, chunks);
}
template <int FMT, typename T, int D>
static void read_one(const Kv4View &c, const Kv4Seqs &s, void *k, void *v, hipStream_t st) {
    const int chunks = (c.n_kv * (D / 8) + 63) / 64;
    const unsigned wgs = (unsigned)(((size_t)s.n_tok * chunks + 3) / 4);
    hipLaunchKernelGGL((k_kv4_read<FMT, T, D>), dim3(wgs, 2), dim3(256), 0, st, c, s,
                       static_cast<T *>(k), static_cast<T *>(v), chunks);
}

// Calls f with the format, the type and the head size as constants.
template <typename F>
static hipError_t kv4_by_shape(int fmt, int dtype, int D, F &&f) {
    auto dim = [&](auto fm, auto ty) {
        if (D == 64)
            f(fm, ty, std::integral_constant<int, 64>());
        else if (D == 128)
            f(fm, ty, std::integral_constant<int, 128>());
        else if (D == 192)
            f(fm, ty, std::integral_constant<int, 192>());
        else if (D == 256)
            f(fm, ty, std::integral_constant<int, 256>());
        else
            return hipErrorInvalidValue;
        return hipGetLastError();
    };
    const std::integral_constant<int, 4> f4;
    const std::integral_constant<int, 7> f7;
    if (dtype == KV4_BF16)
        return fmt == 4 ? dim(f4, __bf16()) : dim(f7, __bf16());
    return fmt == 4 ? dim(f4, float()) : dim(f7, float());
}

hipError_t launch_kv4_append(int fmt, int D, int dtype, const Kv4View &c, const Kv4Seqs &s,
                             const void *k, long long k_stride, const void *v, long long v_stride,
                             hipStream_t st) {
    return kv4_by_shape(fmt, dtype, D, [&](auto fm, auto ty, auto d) {
        append_one<fm.value, decltype(ty), d.value>(c, s, k, k_stride, v, v_stride, st);
    });
}

hipError_t launch_kv4_read(int fmt, int D, int dtype, const Kv4View &c, const Kv4Seqs &s, void *k,
                           void *v, hipStream_t st) {
    return kv4_by_shape(fmt, dtype, D, [&](auto fm, auto ty, auto d) {
        read_one<fm.value, decltype(ty), d.value>(c, s, k, v, st);
    });
}

// ---- eviction -----------------------------------------------------------------------------

// A weight's rank: larger is kept first; NaN is the least, -0 equals +0.
__device__ __forceinline__ uint32_t evict_key(float w) {
    if (w != w)
        return 0u;
    const uint32_t b = __float_as_uint(w + 0.f);
    return (b >> 31) ? ~b : (b | 0x80000000u);
}

// Sums over a wave's lanes up to each one.
__device__ __forceinline__ uint32_t row_scan(uint32_t x) {  // of its row of 16
#define SCAN_STEP(ctrl, rows) \
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false)
    SCAN_STEP(0x111, 0xf);  // row_shr:1, 2, 4, 8
    SCAN_STEP(0x112, 0xf);
    SCAN_STEP(0x114, 0xf);
    SCAN_STEP(0x118, 0xf);
    return x;
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    x = row_scan(x);
    SCAN_STEP(0x142, 0xa);  // a row's last lane on to the next row, then the second's to the last two
    SCAN_STEP(0x143, 0xc);
#undef SCAN_STEP
    return x;
}
// The sum of the 16 waves' numbers ahead of wave w.
__device__ __forceinline__ uint32_t ahead_of(const uint32_t *x, int w) {
    const uint32_t s = row_scan(x[threadIdx.x & 15]);
    return w ? (uint32_t)__builtin_amdgcn_readlane((int)s, w - 1) : 0u;
}

// One workgroup: the kept tokens of one head of one sequence, in order.  The last `recent`
// tokens stay; of the `old` others the `pick` of largest weight, ties to the lowest index.
// The pick-th largest key is found by its digits, 11 + 11 + 10 bits from the top: a histogram
// in LDS of the keys that share the digits found so far, then the bin where the count from the
// top passes what is still to pick.  Each wave then walks its own stretch of the tokens
// twice: to count the larger and the equal keys, and, with the counts ahead of it known, to
// write the kept indices.  Keys stay in LDS (kcap of them); of longer sequences they are formed
// again in each pass.
//
// Everything takes four tokens a lane (a page keeps a head's scores together, and has a multiple
// of 16 of them).  Bound by the round trips and barriers of its one workgroup: 4 sequences of 8
// heads, 12000 to 32768 tokens, 8192 kept, 26.7 us (46.9 with one token a lane); 4 of 4 to 1500
// tokens 7.2 us.
__global__ __launch_bounds__(1024) void k_kv4_select(EvictArgs A, int kcap) {
    extern __shared__ __attribute__((aligned(16))) uint32_t keys[];
    __shared__ uint32_t hist[2][2048];  // of the even and the odd lanes: keys crowd in few bins
    __shared__ uint32_t part[16], above[16], same[16];
    __shared__ uint32_t found[2];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = kv4_len(A.c, A.lens[b], A.max_pages);
    const int m = min(n, A.keep);
    int *kept = A.kept + ((size_t)b * A.c.n_kv + h) * A.keep;
    if (h == 0 && tid == 0)
        A.new_lens[b] = m;
    if (n <= A.keep) {
        for (int j = tid; j < A.keep; j += 1024)
            kept[j] = j < n ? j : -1;
        return;
    }
    const int recent = min(A.recent, A.keep), old = n - recent;
    const int pick = A.keep - recent;  // 0 <= pick < old
    const int *row = A.table + (size_t)b * A.max_pages;
    // the table entry of token t, and the keys of four tokens from t on (a multiple of 4)
    auto entry_of = [&](int t) { return kv4_phys(A.c, row, A.max_pages, kv4_page_of(A.c, t)); };
    auto scores_of = [&](int t, int phys) {
        const int slot = t - kv4_page_of(A.c, t) * A.c.page;
        return *reinterpret_cast<const f4v *>(A.c.score + kv4_row(A.c, max(phys, 0), h, slot));
    };
    auto keys_of = [&](f4v w, int phys) {
        u32x4 k;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            k[e] = phys < 0 ? 0u : evict_key(w[e]);
        return k;
    };
    const bool held = old <= kcap;
    if (held) {
        // 32 at a time: their table entries, then their scores, are on their way together
        for (int t = 4 * tid; t < old; t += 8 * 4096) {
            int phys[8];
            f4v w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                phys[i] = entry_of(min(t + 4096 * i, (old - 1) & ~3));
#pragma unroll
            for (int i = 0; i < 8; ++i)
                w[i] = scores_of(min(t + 4096 * i, (old - 1) & ~3), phys[i]);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (t + 4096 * i < old)
                    *reinterpret_cast<u32x4 *>(keys + t + 4096 * i) = keys_of(w[i], phys[i]);
        }
    }
    auto quad = [&](int t) {
        if (held)
            return *reinterpret_cast<const u32x4 *>(keys + t);
        const int phys = entry_of(t);
        return keys_of(scores_of(t, phys), phys);
    };
    uint32_t prefix = 0, mask = 0;
    uint32_t want = (uint32_t)pick;  // of the keys that share the prefix
    if (pick > 0) {
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            hist[0][tid] = hist[0][tid + 1024] = hist[1][tid] = hist[1][tid + 1024] = 0;
            __syncthreads();
            for (int t = 4 * tid; t < old; t += 4096) {
                const u32x4 k = quad(t);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (t + e < old && (k[e] & mask) == prefix)
                        atomicAdd(&hist[lane & 1][(k[e] >> shift) & ((1u << bits) - 1)], 1u);
            }
            __syncthreads();
            // two bins a thread, from the top
            const int bin = 2047 - 2 * tid;
            const uint32_t c0 = hist[0][bin] + hist[1][bin];
            const uint32_t c1 = hist[0][bin - 1] + hist[1][bin - 1];
            uint32_t upto = wave_scan(c0 + c1);
            if (lane == 63)
                part[wave] = upto;
            __syncthreads();
            upto += ahead_of(part, wave);
            const uint32_t before = upto - c0 - c1;
            if (before < want && want <= upto) {
                const bool first = want <= before + c0;
                found[0] = (uint32_t)(first ? bin : bin - 1);
                found[1] = want - before - (first ? 0u : c0);
            }
            __syncthreads();
            prefix |= found[0] << shift;
            mask |= ((1u << bits) - 1) << shift;
            want = found[1];
        }
    } else {
        __syncthreads();
    }
    // prefix: the pick-th largest key; `want` of the keys equal to it are kept
    const int span = ((old + 15) / 16 + 255) & ~255;
    const int t0 = min(old, wave * span), t1 = min(old, t0 + span);
    uint32_t gt = 0, eq = 0;
    for (int t = t0 + 4 * lane; t < t1; t += 256) {
        const u32x4 k = quad(t);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            gt += t + e < t1 && k[e] > prefix;
            eq += t + e < t1 && k[e] == prefix;
        }
    }
    gt = wave_scan(gt);
    eq = wave_scan(eq);
    if (lane == 63) {
        above[wave] = gt;
        same[wave] = eq;
    }
    __syncthreads();
    uint32_t g = ahead_of(above, wave), q = ahead_of(same, wave);
    for (int t = t0 + 4 * lane; t - 4 * lane < t1; t += 256) {  // wave-uniform trips
        u32x4 k = {0, 0, 0, 0};
        if (t < t1)
            k = quad(t);
        uint32_t both = 0;  // larger keys, and equal ones from bit 16 on
#pragma unroll
        for (int e = 0; e < 4; ++e)
            both += t + e < t1 ? (k[e] > prefix) + ((uint32_t)(k[e] == prefix) << 16) : 0u;
        const uint32_t upto = wave_scan(both);
        uint32_t ag = g + ((upto - both) & 0xffffu), aq = q + ((upto - both) >> 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = t + e < t1, larger = in && k[e] > prefix, equal = in && k[e] == prefix;
            if (pick > 0 && (larger || (equal && aq < want)))
                kept[ag + min(aq, want)] = t + e;
            ag += larger;
            aq += equal;
        }
        const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        g += all & 0xffffu;
        q += all >> 16;
    }
    for (int j = tid; j < recent; j += 1024)
        kept[pick + j] = old + j;
}

// One workgroup: 64 slots of one head of one sequence's fresh pages.  The kept rows' codes move
// in 16-byte pieces, scales and scores after them, each thread's loads all on their way before
// its first store.  Bound by the rows' scattered reads, 64 bytes each behind three dependent
// loads (4 sequences, 8 heads of 128 in MXFP4, 8192 rows each kept: 73 MB in 33 us, 2.2 TB/s;
// with 128 or 256 slots a workgroup, more loads on their way, 33 too).
template <int FMT, int D>
__global__ __launch_bounds__(256) void k_kv4_move(EvictArgs A) {
    constexpr int CP = D / 32;                          // 16-byte pieces of a row's codes
    constexpr int SB = FMT == 4 ? D / 16 : D / 32;      // bytes of a row's scales
    constexpr int SU = FMT == 4 ? 4 : 2, SP = SB / SU;  // their pieces
    constexpr int NC = 2 * CP / 4, NS = (2 * SP + 1 + 3) / 4;  // pieces of a thread
    __shared__ long long from[64], to[64];
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, j0 = blockIdx.x * 64;
    const int n = min(kv4_len(A.c, A.lens[b], A.max_pages), A.keep);
    if (j0 >= n)
        return;
    if (tid < 64) {
        const int j = j0 + tid;
        long long f = -1, t = -1;
        if (j < n) {
            const int src = A.kept[((size_t)b * A.c.n_kv + h) * A.keep + j];
            const int sp = kv4_page_of(A.c, src), dp = kv4_page_of(A.c, j);
            const int ps = kv4_phys(A.c, A.table + (size_t)b * A.max_pages, A.max_pages, sp);
            const int pd = kv4_phys(A.c, A.dst_table + (size_t)b * A.dst_max_pages,
                                    A.dst_max_pages, dp);
            if (ps >= 0 && pd >= 0) {
                f = (long long)kv4_row(A.c, ps, h, src - sp * A.c.page);
                t = (long long)kv4_row(A.c, pd, h, j - dp * A.c.page);
            }
        }
        from[tid] = f;
        to[tid] = t;
    }
    __syncthreads();
    u32x4 code[NC];
    uint32_t rest[NS];
    // piece i of the codes: its place in the pools' rows
    auto codes_at = [&](int i, const long long *rows, uint8_t *&pool, long long &o) {
        const int r = i / (2 * CP), p = i - r * 2 * CP;
        pool = p < CP ? A.c.k : A.c.v;
        o = rows[r] < 0 ? -1 : rows[r] * CP + (p < CP ? p : p - CP);
    };
    auto rest_at = [&](int i, const long long *rows, uint8_t *&pool, long long &o, bool &score) {
        const int r = i / (2 * SP + 1), p = i - r * (2 * SP + 1);
        const long long at = r < 64 ? rows[r & 63] : -1;
        score = p == 2 * SP;
        pool = p < SP ? A.c.ks : A.c.vs;
        o = at < 0 ? -1 : score ? at : at * SP + (p < SP ? p : p - SP);
    };
    uint8_t *pool;
    long long o;
    bool score;
#pragma unroll
    for (int u = 0; u < NC; ++u) {
        codes_at(tid + 256 * u, from, pool, o);
        code[u] = reinterpret_cast<const u32x4 *>(pool)[max(o, 0ll)];
    }
#pragma unroll
    for (int u = 0; u < NS; ++u) {
        rest_at(tid + 256 * u, from, pool, o, score);
        o = max(o, 0ll);
        if (score)
            rest[u] = __float_as_uint(A.c.score[o]);
        else if (SU == 4)
            rest[u] = reinterpret_cast<const uint32_t *>(pool)[o];
        else
            rest[u] = reinterpret_cast<const uint16_t *>(pool)[o];
    }
#pragma unroll
    for (int u = 0; u < NC; ++u) {
        codes_at(tid + 256 * u, to, pool, o);
        if (o >= 0)
            reinterpret_cast<u32x4 *>(pool)[o] = code[u];
    }
#pragma unroll
    for (int u = 0; u < NS; ++u) {
        rest_at(tid + 256 * u, to, pool, o, score);
        if (o >= 0) {
            if (score)
                A.c.score[o] = __uint_as_float(rest[u]);
            else if (SU == 4)
                reinterpret_cast<uint32_t *>(pool)[o] = rest[u];
            else
                reinterpret_cast<uint16_t *>(pool)[o] = (uint16_t)rest[u];
        }
    }
}

// Keys that a selecting workgroup holds in LDS beside its histogram.
constexpr int kEvictKeys = 34 * 1024;

hipError_t launch_kv4_evict(int fmt, int D, const EvictArgs &a, int max_len, hipStream_t st) {
    static const hipError_t lds = hipFuncSetAttribute(
        reinterpret_cast<const void *>(&k_kv4_select), hipFuncAttributeMaxDynamicSharedMemorySize,
        kEvictKeys * 4);
    if (lds != hipSuccess)
        return lds;
    const int kcap = std::min(kEvictKeys, std::max(64, (max_len + 3) & ~3));
    hipLaunchKernelGGL(k_kv4_select, dim3((unsigned)a.c.n_kv, (unsigned)a.n_seq), dim3(1024),
                       (size_t)kcap * 4, st, a, kcap);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        return e;
    return kv4_by_shape(fmt, KV4_F32, D, [&](auto fm, auto, auto d) {
        hipLaunchKernelGGL((k_kv4_move<fm.value, d.value>),
                           dim3((unsigned)((a.keep + 63) / 64), (unsigned)a.c.n_kv,
                                (unsigned)a.n_seq),
                           dim3(256), 0, st, a);
    });
}

}  // namespace mvllm_hip
