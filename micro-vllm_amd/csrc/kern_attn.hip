// kern_attn.hip -- attention over keys and values held in 4 bits, for gfx950.
//
// Row r of a sequence and kv head is query r / group of its new tokens under head
// r % group of the kv head's group.  With S_tr = scale2 * (k_t . q_r) (log2 units), row r sees
// token t if t <= pos_r (and t > pos_r - window), out_r = sum_t 2^(S_tr - m) v_t / sum_t
// 2^(S_tr - m) for any m.
#include "kv4_common.h"

#include <algorithm>
#include <cmath>

namespace mvllm_hip {

namespace {

typedef float fl2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f4v mfma(bf16x8 a, bf16x8 b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x2 as_bf2(uint32_t u) { return __builtin_bit_cast(bf16x2, u); }
__device__ __forceinline__ uint32_t as_u32(bf16x2 b) { return __builtin_bit_cast(uint32_t, b); }

// Sum over the 16 lanes of a row, in each of them.
__device__ __forceinline__ float row_sum(float x) {
#define ROW_STEP(ctrl)                                                                         \
    x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), ctrl, \
                                                               0xf, 0xf, false))
    ROW_STEP(0x128);  // row_ror:8, 4, 2, 1
    ROW_STEP(0x124);
    ROW_STEP(0x122);
    ROW_STEP(0x121);
#undef ROW_STEP
    return x;
}
// Maximum and sum over the four lanes that hold one matrix column (lane, +16, +32, +48).
__device__ __forceinline__ float col_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float col_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// s * scale * log2(e) - ref in one rounding, and its power of two; f32 inputs take the part of
// scale * log2(e) that an f32 does not hold along (it would be off by 3e-8 of each exponent).
template <typename T> __device__ __forceinline__ float exponent(const AttnArgs &A, float s, float ref) {
    if constexpr (sizeof(T) == 4)
        return fmaf(s, A.scale2, fmaf(s, A.scale2_lo, -ref));
    return fmaf(s, A.scale2, -ref);
}
template <typename T> __device__ __forceinline__ float power(const AttnArgs &A, float s, float ref) {
    return __builtin_amdgcn_exp2f(exponent<T>(A, s, ref));
}

// x[8] as T bf16 operands that add up to it (T = 3: all 24 bits).  An infinite x becomes NaN,
// as does every row that an infinite query or probability is in.
template <int T>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&t)[T]) {
    u32x4 w[T];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // two at a time: one conversion, and two words to take off
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int k = 0; k < T; ++k) {
            const uint32_t u = as_u32(__builtin_convertvector(fl2{a, b}, bf16x2));
            w[k][i] = u;
            a -= __uint_as_float(u << 16);
            b -= __uint_as_float(u & 0xffff0000u);
        }
    }
#pragma unroll
    for (int k = 0; k < T; ++k)
        t[k] = __builtin_bit_cast(bf16x8, w[k]);
}

// row / group and row % group by a multiplication: with M = floor(2^40 / g) + 1, row * M >> 40 is
// the quotient for row < 2^30 and g <= 1024 (M g exceeds 2^40 by at most g).
__device__ __forceinline__ int token_of(const AttnArgs &A, int row) {
    return (int)(((unsigned long long)(unsigned)row * A.group_rcp) >> 40);
}

// What a workgroup works on: one tile of 16 rows of one sequence and kv head.
struct Tile {
    int seq, head;
    int first;  // q row of the sequence's first new token
    int rows;   // rows of the sequence under this head
    int len, pos0;  // tokens; position of the first new token
    const int *table;
};

__device__ __forceinline__ Tile tile_of(const AttnArgs &A, int seq, int head) {
    Tile t;
    t.seq = seq;
    t.head = head;
    const int q0 = max(0, min(A.s.q_start[seq], A.s.n_tok));
    const int q1 = max(q0, min(A.s.q_start[seq + 1], A.s.n_tok));
    t.first = q0;
    t.rows = (q1 - q0) * A.group;
    t.len = A.s.lens[seq];
    t.pos0 = t.len - (q1 - q0);
    t.table = A.s.table + (size_t)seq * A.s.max_pages;
    return t;
}

// The tokens that rows [r0, r1) may see: [lo, hi).  (A row ahead of the sequence's first token
// moves neither, and its position no difference past 32 bits.)
__device__ __forceinline__ void span_of(const AttnArgs &A, const Tile &t, int r0, int r1, int &lo,
                                        int &hi) {
    const int p0 = t.pos0 + token_of(A, r0), p1 = t.pos0 + token_of(A, r1 - 1);
    hi = max(0, min(p1 + 1, kv4_len(A.c, t.len, A.s.max_pages)));
    lo = A.window > 0 ? max(0, min(max(p0, 0) - A.window + 1, hi)) : 0;
}

// B operands of 16 rows of queries: lane (column c, group of lanes kg) holds, of each 64
// elements g, the 16 from 64 g + 16 kg, as two operands (int4: in decode_b<4>'s order).  k8, of
// bf16 queries: -8 times a row's sum of queries in each group, from which the sums of products
// with int4 codes n start, so that they end as those with n - 8 (one instruction for 4 codes in
// place of five).  f32 calls take n - 8 itself: the larger sums on the way make their
// outputs' error 1.1e-6 in place of 4e-7 (16 streams to 4096 tokens; 43.8 and 44.7 us).
// Rows that are not live: zeros (GUARD), or the sequence's first one's queries (there is one).
// Loads without a branch start sooner, which f32 rows gain by (16 streams to 4096 tokens 41.7 us,
// 45.0 with it); half empty tiles of bf16 ones are better with it (32 streams to 16384 tokens,
// groups of 8: 96.3 and 98.3).
template <int FMT, int NG, int TQ, typename T, bool GUARD>
__device__ __forceinline__ void load_q(const AttnArgs &A, const Tile &t, int row, bool live,
                                       bf16x8 (&q)[NG][2][TQ], float (&k8)[NG]) {
    const int kg = (threadIdx.x & 63) >> 4;
    const int i = live ? token_of(A, row) : 0, tok = t.first + i;
    const int head = t.head * A.group + (live ? row - i * A.group : 0);
    const T *p = static_cast<const T *>(A.q) + (size_t)tok * A.q_stride +
                 (size_t)head * (64 * NG) + 16 * kg;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        float sum = 0.f;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, y[8];
            if (!GUARD || live)
                Vec8<T>::load(p + 64 * g + 8 * s, x);
            sum += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
            for (int e = 0; e < 8; ++e)
                y[a_slot<FMT>(e)] = x[e];
            split8<TQ>(y, q[g][s]);
        }
        k8[g] = FMT == 4 && TQ == 1 ? -8.f * col_sum(sum) : 0.f;
    }
}

// 16 tokens' keys as the lanes need them: lane (token m, kg) codes of the 16 elements from
// 64 g + 16 kg; int4 scales of the accumulator's tokens 4 kg + i, MXFP4 scales of its own.
template <int FMT, int NG> struct Keys {
    uint2 w[NG];
    float s[FMT == 4 ? 4 * NG : NG];

    __device__ __forceinline__ void load(const Kv4View &c, size_t row) {
        // (a base that the wave shares, and a lane's offset)
        const uint32_t lane = threadIdx.x & 63, m = lane & 15, kg = lane >> 4;
        const uint8_t *p = c.k + row * (32 * NG), *sp = c.ks + row * (FMT == 4 ? 4 * NG : 2 * NG);
#pragma unroll
        for (int g = 0; g < NG; ++g)
            w[g] = *reinterpret_cast<const uint2 *>(p + (m * (32 * NG) + 8 * kg + 32 * g));
        if constexpr (FMT == 4) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float4 v =
                    *reinterpret_cast<const float4 *>(sp + (4 * kg * (4 * NG) + 16 * g));
                s[4 * g] = v.x; s[4 * g + 1] = v.y; s[4 * g + 2] = v.z; s[4 * g + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int g = 0; g < NG; ++g)
                s[g] = ue8m0_ref(sp[m * (2 * NG) + (kg >> 1) + 2 * g]);
        }
    }
};

// Products of 16 tokens' keys with 16 rows of queries: S[i] is token 4 kg + i, row c.  An int4
// group's codes are summed exactly and its scale applied to the sum; an MXFP4 code times its
// scale is exact in bf16.
template <int FMT, int NG, int TQ>
__device__ __forceinline__ f4v dot_keys(const Keys<FMT, NG> &k, const bf16x8 (&q)[NG][2][TQ],
                                        const float (&k8)[NG]) {
    f4v sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const float s7 = FMT == 7 ? k.s[g] : 0.f;
        const bf16x8 a0 = FMT == 4 && TQ > 1 ? decode_b4_signed(k.w[g].x) : decode_b<FMT>(k.w[g].x, s7);
        const bf16x8 a1 = FMT == 4 && TQ > 1 ? decode_b4_signed(k.w[g].y) : decode_b<FMT>(k.w[g].y, s7);
        f4v acc = FMT == 4 ? f4v{k8[g], k8[g], k8[g], k8[g]} : sum;
#pragma unroll
        for (int t = TQ - 1; t >= 0; --t) {
            acc = mfma(a0, q[g][0][t], acc);
            acc = mfma(a1, q[g][1][t], acc);
        }
        if constexpr (FMT == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sum[i] = fmaf(k.s[i * NG + g], acc[i], sum[i]);
        } else {
            sum = acc;
        }
    }
    return sum;
}

// 32 tokens' values as the lanes need them: lane (m, kg), of tokens 4 kg + i and 16 + 4 kg + i
// (the tokens whose probabilities the lane holds), and what is summed of them.
//
// int4: elements 64 g + 4 m + j, so that a product's rows share one group and the group's scale
// can go to the probabilities.  UNS: the codes enter as n, without the offset of 8, and one
// more product of the probabilities with a constant takes 8 of their sum off again; the sums
// are then off by 2^-24 of sum p s n in place of sum p s |n - 8|, too much for f32 outputs.
template <int FMT, int NG, bool UNS> struct Vals;

template <int NG, bool UNS> struct Vals<4, NG, UNS> {
    uint16_t w[NG][8];
    float s[8 * NG];  // [token][group]

    __device__ __forceinline__ void load(const Kv4View &c, size_t row, int half) {
        const uint32_t lane = threadIdx.x & 63, m = lane & 15, kg = lane >> 4;
        const uint8_t *p = c.v + row * (32 * NG), *sp = c.vs + row * (4 * NG);
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[g][4 * half + i] = *reinterpret_cast<const uint16_t *>(
                    p + ((4 * kg + i) * (32 * NG) + 32 * g + 2 * m));
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const float4 v = *reinterpret_cast<const float4 *>(sp + (4 * kg * (4 * NG) + 16 * g));
            const int o = 4 * NG * half + 4 * g;
            s[o] = v.x; s[o + 1] = v.y; s[o + 2] = v.z; s[o + 3] = v.w;
        }
    }
    // A masked token's scale may be anything: the lane's row takes none.
    __device__ __forceinline__ void hide(uint32_t seen) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int g = 0; g < NG; ++g)
                s[i * NG + g] = (seen >> i) & 1 ? s[i * NG + g] : 0.f;
    }

    struct Acc {
        f4v o[NG][4], e[NG];

        __device__ __forceinline__ void clear() {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                e[g] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[g][j] = f4v{0.f, 0.f, 0.f, 0.f};
            }
        }
        __device__ __forceinline__ void scale(float f) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                e[g] *= f;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[g][j] *= f;
            }
        }
        template <int TP>
        __device__ __forceinline__ void add(const Vals &v, const float (&p)[8]) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float ps[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    ps[i] = p[i] * v.s[i * NG + g];
                __builtin_amdgcn_sched_barrier(0);  // one group's operands at a time
                bf16x8 b[TP], a[4];
                split8<TP>(ps, b);
#pragma unroll
                for (int h = 0; h < 4; ++h) {  // tokens 2 h and 2 h + 1
                    const uint32_t x = (uint32_t)v.w[g][2 * h] | ((uint32_t)v.w[g][2 * h + 1] << 16);
                    const uint32_t y = __builtin_amdgcn_perm(x, x, 0x03010200u);  // pairs of bytes
                    const int lo = (int)(UNS ? y & 0x0f0f0f0fu : int4_signed_codes(y));
                    const int hi = (int)(UNS ? (y >> 4) & 0x0f0f0f0fu : int4_signed_codes(y >> 4));
                    const bf16x2 c[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, false),
                                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, false),
                                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, true),
                                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, true)};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        a[j][2 * h] = c[j][0];
                        a[j][2 * h + 1] = c[j][1];
                    }
                }
                bf16x8 minus8;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    minus8[i] = (__bf16)-8.f;
#pragma unroll
                for (int k = TP - 1; k >= 0; --k) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        o[g][j] = mfma(a[j], b[k], o[g][j]);
                    if constexpr (UNS)
                        e[g] = mfma(minus8, b[k], e[g]);
                }
            }
        }
        // f(d, four sums from element d on) over the lane's elements
        template <typename F> __device__ __forceinline__ void pieces(int kg, F &&f) const {
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4 y = make_float4(o[g][0][i], o[g][1][i], o[g][2][i], o[g][3][i]);
                    if constexpr (UNS) {
                        y.x += e[g][i]; y.y += e[g][i]; y.z += e[g][i]; y.w += e[g][i];
                    }
                    f(64 * g + 16 * kg + 4 * i, y);
                }
        }
    };
};

// MXFP4: elements 128 c + 8 m + j, and of a last 64 (head_dim 64 or 192) 4 m + j; a code times
// its scale is exact in bf16, so the scale goes to the code.
template <int NG, bool UNS> struct Vals<7, NG, UNS> {
    static constexpr int NC = NG / 2, ODD = NG & 1;
    uint32_t w[NC + ODD][8];
    uint32_t b[2][2 * NG];  // scale bytes [token][2 NG] of 4 tokens

    __device__ __forceinline__ void load(const Kv4View &c, size_t row, int half) {
        const uint32_t lane = threadIdx.x & 63, m = lane & 15, kg = lane >> 4;
        const uint8_t *p = c.v + row * (32 * NG), *sp = c.vs + row * (2 * NG);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t at = (4 * kg + i) * (32 * NG);
#pragma unroll
            for (int n = 0; n < NC; ++n)
                w[n][4 * half + i] =
                    *reinterpret_cast<const uint32_t *>(p + (at + 64 * n + 4 * m));
            if constexpr (ODD)
                w[NC][4 * half + i] =
                    *reinterpret_cast<const uint16_t *>(p + (at + 64 * NC + 2 * m));
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const uint2 v = *reinterpret_cast<const uint2 *>(sp + (4 * kg * (2 * NG) + 8 * g));
            b[half][2 * g] = v.x;
            b[half][2 * g + 1] = v.y;
        }
    }
    // Bytes above 252, which no append writes, count as 252 in a block with masked tokens: such
    // a token's values stay finite.
    __device__ __forceinline__ void hide(uint32_t) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2 * NG; ++i) {
                const uint32_t x = b[h][i];
                b[h][i] = min(x & 0xffu, 252u) | min(x & 0xff00u, 252u << 8) |
                          min(x & 0xff0000u, 252u << 16) | min(x & 0xff000000u, 252u << 24);
            }
    }

    // Scale of token t for the lane's elements of chunk n.
    __device__ __forceinline__ float scale(int t, int n) const {
        const int m = threadIdx.x & 15;
        const int byte = (t & 3) * 2 * NG + 4 * n;  // the chunk's first, a multiple of 2
        uint32_t d = b[t >> 2][byte >> 2];
        if (byte & 2)  // (then NG is odd, and four bytes may lie in two words)
            d = n < NC ? __builtin_amdgcn_alignbyte(b[t >> 2][(byte >> 2) + 1], d, 2) : d >> 16;
        const uint32_t e = (d >> (8 * (n < NC ? m >> 2 : m >> 3))) & 0xffu;
        return __uint_as_float(e << 23);
    }

    struct Acc {
        f4v o[NC][8], x[ODD ? 4 : 1];

        __device__ __forceinline__ void clear() { each([](f4v &y) { y = f4v{0.f, 0.f, 0.f, 0.f}; }); }
        __device__ __forceinline__ void scale(float f) { each([=](f4v &y) { y *= f; }); }
        template <typename F> __device__ __forceinline__ void each(F &&f) {
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    f(o[n][j]);
            if constexpr (ODD) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    f(x[j]);
            }
        }
        template <int TP>
        __device__ __forceinline__ void add(const Vals &v, const float (&p)[8]) {
            bf16x8 b[TP];
            split8<TP>(p, b);
#pragma unroll
            for (int n = 0; n < NC + ODD; ++n) {
                float s[8];
#pragma unroll
                for (int t = 0; t < 8; ++t)
                    s[t] = v.scale(t, n);
#pragma unroll
                for (int z = 0; z < (n < NC ? 4 : 2); ++z) {  // byte z: elements 2 z and 2 z + 1
                    bf16x8 a0, a1;
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const uint32_t c = as_u32(cvt4(v.w[n][2 * h], s[2 * h], z));
                        const uint32_t d = as_u32(cvt4(v.w[n][2 * h + 1], s[2 * h + 1], z));
                        const bf16x2 lo = as_bf2(__builtin_amdgcn_perm(d, c, 0x05040100u));
                        const bf16x2 hi = as_bf2(__builtin_amdgcn_perm(d, c, 0x07060302u));
                        a0[2 * h] = lo[0]; a0[2 * h + 1] = lo[1];
                        a1[2 * h] = hi[0]; a1[2 * h + 1] = hi[1];
                    }
                    f4v &y0 = n < NC ? o[n < NC ? n : 0][2 * z] : x[ODD ? (2 * z) & 3 : 0];
                    f4v &y1 = n < NC ? o[n < NC ? n : 0][2 * z + 1] : x[ODD ? (2 * z + 1) & 3 : 0];
#pragma unroll
                    for (int k = TP - 1; k >= 0; --k) {
                        y0 = mfma(a0, b[k], y0);
                        y1 = mfma(a1, b[k], y1);
                    }
                }
            }
        }
        static __device__ __forceinline__ bf16x2 cvt4(uint32_t w, float s, int z) {
            return z == 0   ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0)
                   : z == 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1)
                   : z == 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2)
                            : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
        }
        template <typename F> __device__ __forceinline__ void pieces(int kg, F &&f) const {
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 128 * n + 32 * kg + 8 * i;
                    f(d, make_float4(o[n][0][i], o[n][1][i], o[n][2][i], o[n][3][i]));
                    f(d + 4, make_float4(o[n][4][i], o[n][5][i], o[n][6][i], o[n][7][i]));
                }
            if constexpr (ODD) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    f(128 * NC + 16 * kg + 4 * i, make_float4(x[0][i], x[1][i], x[2][i], x[3][i]));
            }
        }
    };
};

__device__ __forceinline__ void store4(float *p, float4 y) { *reinterpret_cast<float4 *>(p) = y; }
__device__ __forceinline__ void store4(__bf16 *p, float4 y) {
    const bf16x2 a = {(__bf16)y.x, (__bf16)y.y}, b = {(__bf16)y.z, (__bf16)y.w};
    *reinterpret_cast<uint2 *>(p) = make_uint2(as_u32(a), as_u32(b));
}

// Where 16 tokens from t0 on (a multiple of 16) lie: the cache's row of the first (page 0's where
// there is none), and whether they are there.
struct Place {
    size_t row;
    bool ok;
};
// A table entry on its way: loaded a block ahead and looked at only when it is needed (loads
// come back in order, so a wave that looked at once would wait for the keys before it too).
struct Entry {
    int t0, pg, raw;

    __device__ __forceinline__ void load(const AttnArgs &A, const Tile &t, int tok) {
        t0 = tok;
        pg = kv4_page_of(A.c, tok);
        raw = t.table[min(pg, A.s.max_pages - 1)];
    }
    __device__ __forceinline__ Place place(const AttnArgs &A, const Tile &t) const {
        const int phys = __builtin_amdgcn_readfirstlane(raw);
        const bool ok = pg < A.s.max_pages && (unsigned)phys < (unsigned)A.c.n_pages;
        return {kv4_row(A.c, ok ? phys : 0, t.head, t0 - pg * A.c.page), ok};
    }
};

}  // namespace

// Waves a SIMD whose registers hold an attention kernel without spilling.
constexpr int attn_waves(int fmt, int ng, bool f32) {
    if (ng <= 2)
        return !f32 && (ng == 1 || fmt == 7) ? 3 : 2;
    return fmt == 7 && (ng == 3 || !f32) ? 2 : 1;
}

// One workgroup: tiles of 16 rows of one sequence and kv head over one split of the tokens;
// its four waves take blocks of 32 tokens in turn and join at the end.  S^T = K q^T puts a row
// in a column of the accumulator (lanes c, c + 16, ...), so the probabilities are already where
// the second product O^T = V^T P^T wants its right operand: token order inside a product is
// free, and the value loads follow it.  Codes go from memory to the operands in registers.
//
// Each wave asks for the next block's keys as soon as it is done with this one's, so they are
// on their way during the exponentials and the second product, and for its values after that
// (two whole blocks in registers gained nothing and halved the waves that fit).  The pool pages
// are asked for one block earlier and looked at a block after: looking at once would wait for
// the keys before them (long decode 98 us and 96).  Pages of a multiple of 32 tokens need one
// entry a block (110 and 99).  The maximum is raised only when a block passes it by 2^8 (sums stay
// in range, and relative precision does not depend on it), so most blocks need no exchange
// between lanes and no rescaling.
//
// With the join: 32 bf16 streams over MXFP4, 64 heads on 8 of 128, 4096 to 16384 tokens, 364 MB in
// 96 us, 3.8 TB/s, bound by how many bytes are on their way; 16 f32 streams over int4, 16
// heads of 128, 100 to 4096 tokens, 85 MB in 42 us, bound by issue (three-term operands: 12
// products of queries and 24 of values a block of 32 tokens) and by the workgroups' starts
// and ends; one stream of 777 tokens 10.6 us, two launches' latency.
template <int FMT, int NG, typename T>
__global__ __launch_bounds__(256, attn_waves(FMT, NG, sizeof(T) == 4)) void k_kv4_attn(AttnArgs A) {
    constexpr int D = 64 * NG, TQ = sizeof(T) == 4 ? 3 : 1, TP = sizeof(T) == 4 ? 3 : 2;
    using V = Vals<FMT, NG, TP == 2>;
    __shared__ __attribute__((aligned(16))) float osum[3][16][D + 4];
    __shared__ float wm[4][16], wl[4][16];
    const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int split = blockIdx.z % A.splits;
    const Tile t = tile_of(A, blockIdx.y, blockIdx.x);
    for (int r0 = blockIdx.z / A.splits * 16; r0 < t.rows; r0 += A.tiles * 16) {
        const int r1 = min(t.rows, r0 + 16);
        int lo, hi;
        span_of(A, t, r0, r1, lo, hi);
        const int s0 = (int)min((long long)hi, (lo & ~31) + (long long)split * A.chunk);
        const int s1 = split + 1 == A.splits ? hi : min(hi - s0, A.chunk) + s0;
        const int row = r0 + col;
        const bool live = row < r1;
        const int pos = t.pos0 + token_of(A, live ? row : r0);
        const int from = A.window > 0 ? pos - A.window : -1;  // sees tokens above `from`
        // tokens that every row of the tile sees: [all0, all1)
        const int all1 = min(s1, t.pos0 + token_of(A, r0) + 1);
        const int all0 = A.window > 0 ? t.pos0 + token_of(A, r1 - 1) - A.window + 1 : 0;

        Place at[2];
        Entry ahead[2];
        Keys<FMT, NG> k[2];
        V v;
        auto look = [&](int t0) {
            ahead[0].load(A, t, t0);
            if (A.c.page & 16) {  // else 32 tokens lie in one page
                asm volatile("");
                ahead[1].load(A, t, t0 + 16);
            }
        };
        auto arrive = [&] {
            at[0] = ahead[0].place(A, t);
            at[1] = {at[0].row + 16, at[0].ok};
            if (A.c.page & 16) {
                asm volatile("");
                at[1] = ahead[1].place(A, t);
            }
        };
        auto fetch_keys = [&] {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                k[h].load(A.c, at[h].row);
        };
        auto fetch_vals = [&] {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                v.load(A.c, at[h].row, h);
        };
        const int ri = live ? token_of(A, row) : 0;
        const size_t logit_row =
            ((size_t)(t.first + ri) * A.n_q + t.head * A.group + (live ? row - ri * A.group : 0)) *
            (size_t)A.logits;
        const int b0 = s0 + 32 * wave;
        if (b0 < s1) {
            look(b0);
            arrive();
            look(b0 + 128);
            fetch_keys();
            fetch_vals();
        }
        bf16x8 q[NG][2][TQ];
        float k8[NG];
        load_q<FMT, NG, TQ, T, TQ == 1>(A, t, row, live, q, k8);
        typename V::Acc o;
        o.clear();
        float m = -INFINITY, l = 0.f;

        for (int t0 = b0; t0 < s1; t0 += 128) {
            // a page that is none: its tokens are not there
            const bool ok[2] = {at[0].ok, at[1].ok};
            const bool more = t0 + 128 < s1;
            float s[8], x[8], p[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f4v y = dot_keys<FMT, NG, TQ>(k[h], q, k8);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[4 * h + i] = y[i];
                    x[4 * h + i] = y[i] * A.scale2;
                }
                if (A.logit && live && t0 + 16 * h < A.logits)
                    store4(A.logit + logit_row + t0 + 16 * h + 4 * kg,
                           make_float4(y[0], y[1], y[2], y[3]));
            }
            if (more) {
                arrive();
                look(t0 + 256);
                fetch_keys();
            }
            if (!(ok[0] && ok[1] && t0 >= all0 && t0 + 32 <= all1)) {
                asm volatile("");  // a branch, not 70 selects in every block
                uint32_t seen = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int tok = t0 + 16 * (i >> 2) + 4 * kg + (i & 3);
                    const bool sees = ok[i >> 2] && live && tok < s1 && tok <= pos && tok > from;
                    seen |= (uint32_t)sees << i;
                    x[i] = sees ? x[i] : -INFINITY;
                }
                v.hide(seen);
            }
            const float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                                    fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            if (__any(top > m + 8.f)) {
                const float up = fmaxf(m, col_max(top));
                const float fix = up == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - up);
                m = up;
                l *= fix;
                o.scale(fix);
            }
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                p[i] = sizeof(T) == 2       ? __builtin_amdgcn_exp2f(x[i] - ref)
                       : x[i] == -INFINITY ? 0.f
                                            : power<T>(A, s[i], ref);
            l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            o.template add<TP>(v, p);
            if (more)
                fetch_vals();
        }
        // join the waves: each one's sums relative to the common maximum
        l = col_sum(l);
        if (kg == 0) {
            wm[wave][col] = m;
            wl[wave][col] = l;
        }
        __syncthreads();
        float M = wm[0][col], L = 0.f;
#pragma unroll
        for (int w = 1; w < 4; ++w)
            M = fmaxf(M, wm[w][col]);
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            L += wl[w][col] * __builtin_amdgcn_exp2f(wm[w][col] - ref);
        const float fix = __builtin_amdgcn_exp2f(m - ref);
        if (wave > 0) {
            o.pieces(kg, [&](int d, float4 y) {
                *reinterpret_cast<float4 *>(&osum[wave - 1][col][d]) =
                    make_float4(y.x * fix, y.y * fix, y.z * fix, y.w * fix);
            });
        }
        __syncthreads();
        if (wave == 0 && live) {
            const int i = token_of(A, row), tok = t.first + i;
            const int head = t.head * A.group + row - i * A.group;
            const size_t at = ((size_t)split * A.s.n_tok + tok) * A.n_q + head;
            if (A.splits > 1) {
                if (kg == 0)
                    A.ml[at] = make_float2(M, L);
            } else if (A.lse && kg == 0) {
                A.lse[at] = L > 0.f ? M + log2f(L) : -INFINITY;
            }
            const float scale = A.splits > 1 ? 1.f : L > 0.f || L != L ? 1.f / L : 0.f;
            if (A.splits == 1 || M != -INFINITY) {  // (the join leaves a split of nothing out)
                o.pieces(kg, [&](int d, float4 y) {
                    y = make_float4(y.x * fix, y.y * fix, y.z * fix, y.w * fix);
#pragma unroll
                    for (int w = 0; w < 3; ++w) {
                        const float4 z = *reinterpret_cast<const float4 *>(&osum[w][col][d]);
                        y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
                    }
                    y = make_float4(y.x * scale, y.y * scale, y.z * scale, y.w * scale);
                    if (A.splits > 1)
                        *reinterpret_cast<float4 *>(A.part + at * D + d) = y;
                    else
                        store4(static_cast<T *>(A.out) + ((size_t)tok * A.n_q + head) * D + d, y);
                });
            }
        }
        __syncthreads();
    }
}

// Joins the splits of the rows that belong to a sequence.  One wave a head of a token: lane s
// holds split s's maximum and sum (at most 64 splits), and groups of D / 8 lanes take every
// other split's sums.  Bound by latency: 4.7 us for 16 tokens of 16 heads in three splits, 4.9 for
// 32 of 64 in eight.
template <int NG, typename T>
__device__ __forceinline__ void join(const AttnArgs &A, int tok, int head) {
    constexpr int D = 64 * NG, LPH = D / 8, G = 64 / LPH;
    const int lane = threadIdx.x & 63;
    if (head >= A.n_q || tok < A.s.q_start[0] || tok >= A.s.q_start[A.s.n_seq])
        return;
    const size_t at = (size_t)tok * A.n_q + head, step = (size_t)A.s.n_tok * A.n_q;
    const float2 ml = lane < A.splits ? A.ml[at + lane * step] : make_float2(-INFINITY, 0.f);
    float M = ml.x;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
        M = fmaxf(M, __shfl_xor(M, o));
    const float f = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - M);
    float L = ml.y * f;  // a split of nothing: 0 (or NaN, which stays)
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
        L += __shfl_xor(L, o);
    const int g = lane / LPH, d = (lane - g * LPH) * 8;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < A.splits; s0 += 4 * G) {
        float y[4][8], w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {  // four loads on their way
            const int s = min(s0 + u * G + g, 63);
            const float has = __shfl(ml.x, s);
            w[u] = __shfl(f, s);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                y[u][i] = 0.f;
            if (g < G && has != -INFINITY)  // splits from A.splits on have none
                Vec8<float>::load(A.part + (at + s * step) * D + d, y[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = fmaf(y[u][i], w[u], x[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float sum = x[i];
#pragma unroll
        for (int n = 1; n < G; ++n)
            sum += __shfl(x[i], (lane + n * LPH) & 63);
        x[i] = sum;
    }
    const float scale = L > 0.f || L != L ? 1.f / L : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] *= scale;
    if (g == 0)
        Vec8<T>::store(static_cast<T *>(A.out) + at * D + d, x);
    if (A.lse && lane == 0)
        A.lse[at] = L > 0.f ? M + log2f(L) : -INFINITY;
}

template <int NG, typename T>
__global__ __launch_bounds__(256) void k_kv4_join(AttnArgs A) {
    join<NG, T>(A, blockIdx.x, blockIdx.y * 4 + (threadIdx.x >> 6));
}

// One row's products with four tokens' keys from cache row `place` on, a key after the other.
template <int FMT, int NG, typename T>
__device__ __forceinline__ void dot_four(const AttnArgs &A, size_t place, const T *q, float (&s)[4]) {
    constexpr int D = 64 * NG;
#pragma unroll 1
    for (int e = 0; e < 4; ++e) {
        const size_t row = place + e;
        float sum = 0.f;
#pragma unroll 1
        for (int d = 0; d < D; d += 8) {
            const float sc = FMT == 4 ? reinterpret_cast<const float *>(A.c.ks)[row * NG + d / 64]
                                      : ue8m0_ref(A.c.ks[row * (2 * NG) + d / 32]);
            const uint32_t c = reinterpret_cast<const uint32_t *>(A.c.k)[(row * D + d) / 8];
            float part = 0.f;
#pragma unroll
            for (int z = 0; z < 8; ++z) {
                const uint32_t x = (c >> (4 * z)) & 15u;
                part = fmaf((float)q[d + z], FMT == 4 ? (float)((int)x - 8) : e2m1_val(x), part);
            }
            sum = fmaf(part, sc, sum);
        }
        s[e] = sum;
    }
}

// The end of a decode call that collects weights, in one launch.  The first `joins` workgroups
// join the splits, as above.  The others take 1024 tokens each of one sequence and kv head, four
// a thread: the rows' maxima and sums from the splits', the tokens' logits as the attention
// kernel left them (it has every key in its hands; reading its 4 bytes a row again costs less
// than the key's codes and products: 8 sequences to 8192 tokens, groups of 4, 21 us with the
// keys, 5.6 so).  Four rows' logits are on their way at a time (6.7 us one by one).  Tokens past
// the logits' room (longer sequences than max_len) are multiplied out.
template <int FMT, int NG, typename T>
__global__ __launch_bounds__(256) void k_kv4_finish(AttnArgs A, int joins) {
    constexpr int D = 64 * NG;
    __shared__ float lse[16];
    const int bx = blockIdx.x;
    if (bx < joins) {
        const int per = (A.n_q + 3) / 4;
        join<NG, T>(A, bx / per, bx % per * 4 + (threadIdx.x >> 6));
        return;
    }
    const int pairs = A.c.n_kv * A.s.n_seq;
    const int pair = (bx - joins) % pairs, part = (bx - joins) / pairs;
    const int parts = ((int)gridDim.x - joins) / pairs;
    const Tile t = tile_of(A, pair / A.c.n_kv, pair % A.c.n_kv);
    const int len = kv4_len(A.c, t.len, A.s.max_pages);
    for (int r0 = 0; r0 < max(t.rows, 1); r0 += 16) {  // (more than 16 rows: max_new was less)
        const int n_rows = min(16, t.rows - r0);
        {
            const int r = r0 + (threadIdx.x >> 4), j = threadIdx.x & 15;
            const bool live = r < t.rows;
            const int i = live ? token_of(A, r) : 0;
            const size_t at = (size_t)(t.first + i) * A.n_q + t.head * A.group +
                              (live ? r - i * A.group : 0);
            if (A.splits == 1) {
                if (j == 0)
                    lse[threadIdx.x >> 4] = live ? A.lse[at] : -INFINITY;
            } else {
                const size_t step = (size_t)A.s.n_tok * A.n_q;
                float2 ml[4];
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int s = j + 16 * u;
                    ml[u] = live && s < A.splits ? A.ml[at + s * step] : make_float2(-INFINITY, 0.f);
                    M = fmaxf(M, ml[u].x);
                }
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1)
                    M = fmaxf(M, __shfl_xor(M, o));
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    L += ml[u].y * (M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml[u].x - M));
                L = row_sum(L);
                if (j == 0)
                    lse[threadIdx.x >> 4] = L > 0.f || L != L ? M + log2f(L) : -INFINITY;
            }
        }
        __syncthreads();
        for (int t0 = (part * 256 + (int)threadIdx.x) * 4; t0 < len; t0 += parts * 1024) {
            const int pg = kv4_page_of(A.c, t0);
            const int phys = kv4_phys(A.c, t.table, A.s.max_pages, pg);
            if (phys < 0)
                continue;
            const size_t place = kv4_row(A.c, phys, t.head, t0 - pg * A.c.page);
            float w[4] = {0.f, 0.f, 0.f, 0.f};
            const bool kept = t0 < A.logits;
            for (int n0 = 0; n0 < n_rows; n0 += 4) {
                float4 y[4] = {};  // four rows' logits on their way
                if (kept) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int r = r0 + min(n0 + u, n_rows - 1), i = token_of(A, r);
                        y[u] = *reinterpret_cast<const float4 *>(
                            A.logit +
                            ((size_t)(t.first + i) * A.n_q + t.head * A.group + r - i * A.group) *
                                (size_t)A.logits +
                            t0);
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int n = n0 + u, r = r0 + n, i = token_of(A, r), pos = t.pos0 + i;
                    const int from = A.window > 0 ? pos - A.window : -1;
                    if (n >= n_rows)  // (of the whole workgroup)
                        break;
                    float s[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
                    if (!kept)
                        dot_four<FMT, NG, T>(A, place,
                                             static_cast<const T *>(A.q) +
                                                 (size_t)(t.first + i) * A.q_stride +
                                                 (size_t)(t.head * A.group + r - i * A.group) * D,
                                             s);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool sees = (t0 + e <= pos) & (t0 + e > from);
                        const float x = exponent<T>(A, s[e], lse[n]);
                        w[e] += __builtin_amdgcn_exp2f(sees ? x : -INFINITY);
                    }
                }
            }
            float *p = A.c.score + place;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (t0 + e < len)
                    p[e] = A.weights == KV4_WEIGHTS_ADD || r0 > 0 ? p[e] + w[e] : w[e];
        }
        __syncthreads();
    }
}

// The weights of blocks of 16 NB tokens of one sequence and kv head, over all of its rows.  The
// keys stay in registers as operands while the rows pass by, 16 at a time, and each token's sum
// is formed in one place, in one order.
//
// FEW (decode whose logits are too many to keep): each wave takes blocks of its own, the next
// one's keys on their way, with the operands of up to 16 rows loaded once.  Otherwise the four
// waves share a block and take every fourth 16 of its rows; bound by the exponentials and the
// way to the rows (7 sequences, 24 heads on 4 of 64, up to 97 new tokens, window 1024: 14.6 us;
// 20.2 with a branch an element, 28.6 with 16 waves a block).
template <int FMT, int NG, typename T, bool FEW>
__global__ __launch_bounds__(256) void k_kv4_weights(AttnArgs A) {
    constexpr int TQ = sizeof(T) == 4 ? 3 : 1, NB = FEW ? 2 : 4, BLK = 16 * NB;
    __shared__ float part[FEW ? 1 : 4][BLK];
    const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const Tile t = tile_of(A, blockIdx.y, blockIdx.x);
    const int len = kv4_len(A.c, t.len, A.s.max_pages);
    int row = -1, pos = -1, from = -1;
    float lse = -INFINITY, k8[NG];
    bool live = false;
    bf16x8 q[NG][2][TQ];
    auto rows_at = [&](int r) {
        row = r + col;
        live = row < t.rows;
        const int i = live ? token_of(A, row) : 0;
        pos = t.pos0 + i;
        from = A.window > 0 ? pos - A.window : -1;
        lse = A.lse[(size_t)(t.first + i) * A.n_q + t.head * A.group +
                    (live ? row - i * A.group : 0)];
        load_q<FMT, NG, TQ, T, false>(A, t, row, live, q, k8);
    };
    Keys<FMT, NG> k[NB], ahead[FEW ? NB : 1];
    bool ok[NB];
    size_t at[NB];
    auto fetch = [&](int t0, Keys<FMT, NG> *to) {
        Entry e[NB];
#pragma unroll
        for (int h = 0; h < NB; ++h)
            e[h].load(A, t, t0 + 16 * h);
#pragma unroll
        for (int h = 0; h < NB; ++h) {
            const Place pl = e[h].place(A, t);
            ok[h] = pl.ok;
            at[h] = pl.row;
            to[h].load(A.c, at[h]);
        }
    };
    const int step = (int)gridDim.z * (FEW ? 4 : 1) * BLK;
    int t0 = ((int)blockIdx.z * (FEW ? 4 : 1) + (FEW ? wave : 0)) * BLK;
    if (FEW && t0 < len)
        fetch(t0, ahead);
    const bool once = FEW && t.rows <= 16;
    if (once && t0 < len && t.rows > 0)
        rows_at(0);
    for (; t0 < len; t0 += step) {
        bool there[NB];
        size_t place[NB];
        if constexpr (FEW) {
#pragma unroll
            for (int h = 0; h < NB; ++h) {
                k[h] = ahead[h];
                there[h] = ok[h];
                place[h] = at[h];
            }
            if (t0 + step < len)
                fetch(t0 + step, ahead);
        } else {
            fetch(t0, k);
#pragma unroll
            for (int h = 0; h < NB; ++h) {
                there[h] = ok[h];
                place[h] = at[h];
            }
        }
        float w[NB][4] = {};
        // whole: every row sees every token
        auto add = [&](bool whole) {
#pragma unroll
            for (int h = 0; h < NB; ++h) {
                const f4v s = dot_keys<FMT, NG, TQ>(k[h], q, k8);
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x[i] = exponent<T>(A, s[i], lse);
                if (!whole) {
                    asm volatile("");  // a branch; within it selects, no branch an element
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int tok = t0 + 16 * h + 4 * kg + i;
                        const bool sees = live & (tok <= pos) & (tok > from);
                        x[i] = sees ? x[i] : -INFINITY;
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[h][i] += __builtin_amdgcn_exp2f(x[i]);
            }
        };
        if (once) {
            if (t.rows > 0)
                add(false);
        } else {
            // from the first row that may see the first token to the last whose window holds
            // the last one
            int r = (int)min((long long)t.rows, max(0ll, (long long)t0 - t.pos0) * A.group);
            int rend = t.rows;
            if (A.window > 0)
                rend = (int)min((long long)rend,
                                max(0ll, (long long)t0 + BLK - 1 + A.window - t.pos0) * A.group);
            for (r = (r & ~15) + (FEW ? 0 : 16 * wave); r < rend; r += FEW ? 16 : 64) {
                rows_at(r);
                add(r + 16 <= t.rows && t0 + BLK - 1 <= t.pos0 + token_of(A, r) &&
                    (A.window == 0 || t0 > t.pos0 + token_of(A, r + 15) - A.window));
            }
        }
        // a lane's four tokens of each 16, over the 16 rows of its columns; lane (kg, col < 4)
        // is left with token 4 kg + col
        float mine[NB];
#pragma unroll
        for (int h = 0; h < NB; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[h][i] = row_sum(w[h][i]);
            mine[h] = col == 0 ? w[h][0] : col == 1 ? w[h][1] : col == 2 ? w[h][2] : w[h][3];
        }
        if constexpr (!FEW) {
            __syncthreads();  // the block before has been read
            if (col < 4) {
#pragma unroll
                for (int h = 0; h < NB; ++h)
                    part[wave][16 * h + 4 * kg + col] = mine[h];
            }
            __syncthreads();
            if (wave > 0)
                continue;
#pragma unroll
            for (int h = 0; h < NB; ++h) {
                const int n = 16 * h + 4 * kg + (col & 3);
                mine[h] = (part[0][n] + part[1][n]) + (part[2][n] + part[3][n]);
            }
        }
#pragma unroll
        for (int h = 0; h < NB; ++h) {
            if (col < 4 && there[h] && t0 + 16 * h + 4 * kg + col < len) {
                float *p = A.c.score + place[h] + 4 * kg + col;
                *p = A.weights == KV4_WEIGHTS_ADD ? *p + mine[h] : mine[h];
            }
        }
    }
}

// How a call is cut, for the 16-row kernel or (prompt) that of kern_prompt.hip, 8 waves of 32 rows
// a workgroup (4 for head_dim 192 and 256, whose sums fill the registers).
//
// Splits of the tokens, at most the 64 that a wave joins, in chunks of 128 tokens (one block a
// wave) at least, 384 of long sequences (2 streams of 4 kv heads to 11000 tokens: 29 splits 15.0 us,
// 43 16.8); up to 384 tokens stay whole, which saves the join (300 tokens: 9.2 us, 11.2 in three).
// The 16-row kernel: as many as make one round of the chip with every sequence full, two
// workgroups a CU, or three of bf16 over MXFP4 (8 f32 MXFP4 streams of 8 kv heads, all of 8192
// tokens: 8 splits 27 us, 7 32, 10 35; of 1000 to 8192: 26, and 30 with 12).  Where its chunks are
// long, more, since lengths differ and the rounds even out: chunks of 1408 tokens up to one and
// a half rounds (16 int4 f32 streams of 16 heads, 100 to 4096 tokens: 2 splits 50 us, 3 39, 4 47,
// 8 45; all of 4096: 55, 57, 57, 63), and of 2048 up to four (32 MXFP4 bf16 streams of 8 heads,
// 4096 to 16384: 3 splits 105 us, 8 96, 16 106).
static AttnPlan plan_for(bool prompt, int fmt, int dtype, int head_dim, int n_kv, int n_q,
                         int n_tok, int n_seq, int max_new, int max_len, int window,
                         bool weights) {
    AttnPlan p{};
    const long long rows = (long long)max_new * (n_q / n_kv), pairs = (long long)n_kv * n_seq;
    p.waves = !prompt ? 0 : head_dim <= 128 ? 8 : 4;
    const int tile = p.waves ? 32 * p.waves : 16, least = p.waves ? 256 : 128;
    const int slots = p.waves ? 256 : fmt == 7 && dtype == KV4_BF16 ? 768 : 512;
    p.tiles = (int)std::min(32768ll, (rows + tile - 1) / tile);
    // the most tokens that a tile's rows see, from a multiple of 64 on
    const long long seen =
        window > 0 ? std::min((long long)max_len, (long long)window + tile / (n_q / n_kv) + 65)
                   : max_len;
    const long long each = p.tiles * pairs;  // workgroups of a split
    long long want = slots / each;
    if (!p.waves)
        want = std::max({want, std::min(slots * 3 / 2 / each, (seen + 1407) / 1408),
                         std::min(slots * 4 / each, (seen + 2047) / 2048)});
    want = seen <= 384 ? 1 : std::max(1ll, std::min(64ll, want));
    p.chunk = (int)std::max({(long long)least, ((seen + want - 1) / want + 127) / 128 * 128,
                             p.waves ? 0 : std::min(384ll, (seen / 32 + 127) / 128 * 128)});
    p.splits = (int)((seen + p.chunk - 1) / p.chunk);
    auto add = [&](size_t bytes) {
        const size_t at = p.bytes;
        p.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    // room for the splits that any window would have
    const size_t heads = (size_t)n_tok * n_q;
    const size_t most = (size_t)std::min(want, ((long long)max_len + least - 1) / least);
    if (most > 1) {
        p.part = add(most * heads * head_dim * 4);
        p.ml = add(most * heads * 8);
    }
    if (weights)
        p.lse = add(heads * 4);
    // decode keeps its logits for the weights, up to half a gigabyte of them
    const size_t logits = ((size_t)max_len + 127) / 128 * 128;
    if (weights && rows <= 16 && heads * logits * 4 <= (size_t(1) << 29)) {
        p.logits = (int)logits;
        p.logit = add(heads * logits * 4);
    }
    return p;
}

// More than 16 rows a sequence and kv head take either kernel.  The 16-row one starts sooner and
// spreads wider; the other reads and decodes a tile of tokens once for 256 rows.  They meet at
// about 12 million (row, token) pairs of 128 elements, summed over sequences and kv heads, in
// bf16 (int4, 8 heads, groups of 4: 64 rows of 4 sequences over 4096 tokens 37 and 32 us, 256
// rows of one 41 and 41, of 8 with a window of 1024 44 and 42, 2048 rows of 4 516 and 173; 128
// rows of the 8 25 and 34), and at 20 million in f32, whose second terms cost the tiles more.
AttnPlan kv4_attention_plan(int choice, int fmt, int dtype, int head_dim, int n_kv, int n_q,
                            int n_tok, int n_seq, int max_new, int max_len, int window,
                            bool weights) {
    const double rows = (double)max_new * (n_q / n_kv) * n_kv * n_seq;
    const double seen = window > 0 ? std::min((double)max_len, (double)window + max_new) : max_len;
    const bool many = max_new * (long long)(n_q / n_kv) > 16;
    const bool prompt = choice == 2 || (choice == 0 && many &&
                                        rows * seen * head_dim >=
                                            128e6 * (dtype == KV4_BF16 ? 12 : 20));
    return plan_for(prompt, fmt, dtype, head_dim, n_kv, n_q, n_tok, n_seq, max_new, max_len, window,
                    weights);
}

size_t kv4_attention_bytes(int head_dim, int n_kv, int n_q, int n_tok, int n_seq, int max_new,
                           int max_len, bool weights) {
    size_t most = 0;
    for (bool prompt : {false, true})
        for (int fmt : {4, 7})
            for (int dtype : {KV4_F32, KV4_BF16})
                most = std::max(most, plan_for(prompt, fmt, dtype, head_dim, n_kv, n_q, n_tok,
                                               n_seq, max_new, max_len, 0, weights)
                                          .bytes);
    return most;
}

template <int FMT, int NG, typename T>
static hipError_t attention(const AttnArgs &a, int max_len, hipStream_t st) {
    hipError_t e;
    if (a.waves) {
        if ((e = launch_kv4_prompt(FMT, 64 * NG, sizeof(T) == 2 ? KV4_BF16 : KV4_F32, a, st)) !=
            hipSuccess)
            return e;
    } else {
        // Heads go round the XCDs first, splits last: sequences of unlike length leave the later
        // splits empty, and with the splits first the XCDs that got those had nothing to do.
        const dim3 grid((unsigned)a.c.n_kv, (unsigned)a.s.n_seq, (unsigned)(a.splits * a.tiles));
        hipLaunchKernelGGL((k_kv4_attn<FMT, NG, T>), grid, dim3(256), 0, st, a);
        if ((e = hipGetLastError()) != hipSuccess)
            return e;
    }
    if (a.logit && !a.waves) {
        const int pairs = a.c.n_kv * a.s.n_seq;
        const int joins = a.splits > 1 ? a.s.n_tok * ((a.n_q + 3) / 4) : 0;
        const int parts = std::max(1, std::min((max_len + 1023) / 1024, (1 << 24) / pairs));
        hipLaunchKernelGGL((k_kv4_finish<FMT, NG, T>), dim3((unsigned)(joins + parts * pairs)),
                           dim3(256), 0, st, a, joins);
        return hipGetLastError();
    }
    if (a.splits > 1) {
        hipLaunchKernelGGL((k_kv4_join<NG, T>),
                           dim3((unsigned)a.s.n_tok, (unsigned)((a.n_q + 3) / 4)), dim3(256), 0,
                           st, a);
        if ((e = hipGetLastError()) != hipSuccess)
            return e;
    }
    if (a.weights != KV4_WEIGHTS_NONE) {
        // eight blocks a wave (8 sequences to 8192 tokens: 8 blocks were 7 % better than 2 and 20 %
        // than 16), or one a workgroup
        const int per = a.few ? 1024 : 64;
        const dim3 grid((unsigned)a.c.n_kv, (unsigned)a.s.n_seq,
                        (unsigned)std::min(65535, (max_len + per - 1) / per));
        if (a.few)
            hipLaunchKernelGGL((k_kv4_weights<FMT, NG, T, true>), grid, dim3(256), 0, st, a);
        else
            hipLaunchKernelGGL((k_kv4_weights<FMT, NG, T, false>), grid, dim3(256), 0, st, a);
        e = hipGetLastError();
    }
    return e;
}

template <int FMT, typename T>
static hipError_t attention_dim(int D, const AttnArgs &a, int max_len, hipStream_t st) {
    return D == 64    ? attention<FMT, 1, T>(a, max_len, st)
           : D == 128 ? attention<FMT, 2, T>(a, max_len, st)
           : D == 192 ? attention<FMT, 3, T>(a, max_len, st)
           : D == 256 ? attention<FMT, 4, T>(a, max_len, st)
                      : hipErrorInvalidValue;
}

hipError_t launch_kv4_attention(int fmt, int D, int dtype, const AttnArgs &a, int max_len,
                                hipStream_t st) {
    if (dtype == KV4_BF16)
        return fmt == 4 ? attention_dim<4, __bf16>(D, a, max_len, st)
                        : attention_dim<7, __bf16>(D, a, max_len, st);
    return fmt == 4 ? attention_dim<4, float>(D, a, max_len, st)
                    : attention_dim<7, float>(D, a, max_len, st);
}

}  // namespace mvllm_hip
