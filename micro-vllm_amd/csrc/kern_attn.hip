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

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f4v mfma(bf16x8 a, bf16x8 b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x2 as_bf2(uint32_t u) { return __builtin_bit_cast(bf16x2, u); }
__device__ __forceinline__ uint32_t as_u32(bf16x2 b) { return __builtin_bit_cast(uint32_t, b); }

// Maximum and sum over the four lanes that hold one matrix column (lane, +16, +32, +48).
__device__ __forceinline__ float col_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float col_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// 2^(s * scale * log2(e) - ref) in one rounding of the exponent; f32 inputs take the part of
// scale * log2(e) that an f32 does not hold along (it would be off by 3e-8 of each exponent).
template <typename T> __device__ __forceinline__ float power(const AttnArgs &A, float s, float ref) {
    if constexpr (sizeof(T) == 4)
        return __builtin_amdgcn_exp2f(fmaf(s, A.scale2, fmaf(s, A.scale2_lo, -ref)));
    return __builtin_amdgcn_exp2f(fmaf(s, A.scale2, -ref));
}

// x[8] as T bf16 operands that add up to it (T = 3: all 24 bits).
template <int T>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&t)[T]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float r = x[i];
#pragma unroll
        for (int k = 0; k < T; ++k) {
            t[k][i] = (__bf16)r;
            if (k + 1 < T)
                r = nonfinite((float)t[k][i]) ? 0.f : r - (float)t[k][i];
        }
    }
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

// The tokens that rows [r0, r1) may see: [lo, hi).
__device__ __forceinline__ void span_of(const AttnArgs &A, const Tile &t, int r0, int r1, int &lo,
                                        int &hi) {
    const int p0 = t.pos0 + r0 / A.group, p1 = t.pos0 + (r1 - 1) / A.group;
    hi = max(0, min(p1 + 1, kv4_len(A.c, t.len, A.s.max_pages)));
    lo = A.window > 0 ? max(0, min(p0 - A.window + 1, hi)) : 0;
}

// B operands of 16 rows of queries: lane (column c, group of lanes kg) holds, of each 64
// elements g, the 16 from 64 g + 16 kg, as two operands (int4: in decode_b4_signed's order).
template <int FMT, int NG, int TQ, typename T>
__device__ __forceinline__ void load_q(const AttnArgs &A, const Tile &t, int row, bool live,
                                       bf16x8 (&q)[NG][2][TQ]) {
    const int kg = (threadIdx.x & 63) >> 4;
    const int tok = t.first + (live ? row / A.group : 0);
    const int head = t.head * A.group + (live ? row % A.group : 0);
    const T *p = static_cast<const T *>(A.q) + (size_t)tok * A.q_stride +
                 (size_t)head * (64 * NG) + 16 * kg;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, y[8];
            if (live)
                Vec8<T>::load(p + 64 * g + 8 * s, x);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                y[a_slot<FMT>(e)] = x[e];
            split8<TQ>(y, q[g][s]);
        }
}

// 16 tokens' keys as the lanes need them: lane (token m, kg) codes of the 16 elements from
// 64 g + 16 kg; int4 scales of the accumulator's tokens 4 kg + i, MXFP4 scales of its own.
template <int FMT, int NG> struct Keys {
    uint2 w[NG];
    float s[FMT == 4 ? 4 * NG : NG];

    __device__ __forceinline__ void load(const Kv4View &c, size_t row) {
        const int lane = threadIdx.x & 63, m = lane & 15, kg = lane >> 4;
        const uint8_t *p = c.k + (row + m) * (32 * NG) + 8 * kg;
#pragma unroll
        for (int g = 0; g < NG; ++g)
            w[g] = *reinterpret_cast<const uint2 *>(p + 32 * g);
        if constexpr (FMT == 4) {
            const float4 *sp =
                reinterpret_cast<const float4 *>(c.ks + (row + 4 * kg) * (4 * NG));
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float4 v = sp[g];
                s[4 * g] = v.x; s[4 * g + 1] = v.y; s[4 * g + 2] = v.z; s[4 * g + 3] = v.w;
            }
        } else {
            const uint8_t *sp = c.ks + (row + m) * (2 * NG) + (kg >> 1);
#pragma unroll
            for (int g = 0; g < NG; ++g)
                s[g] = ue8m0_ref(sp[2 * g]);
        }
    }
};

// Products of 16 tokens' keys with 16 rows of queries: S[i] is token 4 kg + i, row c.  An int4
// group's codes are summed exactly and its scale applied to the sum; an MXFP4 code times its
// scale is exact in bf16.
template <int FMT, int NG, int TQ>
__device__ __forceinline__ f4v dot_keys(const Keys<FMT, NG> &k, const bf16x8 (&q)[NG][2][TQ]) {
    f4v sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const bf16x8 a0 = FMT == 4 ? decode_b4_signed(k.w[g].x) : decode_b<7>(k.w[g].x, k.s[g]);
        const bf16x8 a1 = FMT == 4 ? decode_b4_signed(k.w[g].y) : decode_b<7>(k.w[g].y, k.s[g]);
        f4v acc = {0.f, 0.f, 0.f, 0.f};
        if constexpr (FMT == 7)
            acc = sum;
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
// (the tokens whose probabilities the lane holds), elements 64 g + 4 m + j.
template <int FMT, int NG> struct Vals {
    uint16_t w[NG][8];
    float s[FMT == 4 ? 8 * NG : 1];      // int4: [token][group]
    uint2 b[FMT == 4 ? 1 : 2][NG];       // MXFP4: bytes [token][2 NG] of 4 tokens

    __device__ __forceinline__ void load(const Kv4View &c, size_t row, int half) {
        const int lane = threadIdx.x & 63, m = lane & 15, kg = lane >> 4;
        row += 4 * kg;
        const uint8_t *p = c.v + row * (32 * NG) + 2 * m;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[g][4 * half + i] =
                    *reinterpret_cast<const uint16_t *>(p + i * (32 * NG) + 32 * g);
        if constexpr (FMT == 4) {
            const float4 *sp = reinterpret_cast<const float4 *>(c.vs + row * (4 * NG));
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float4 v = sp[g];
                const int o = 4 * NG * half + 4 * g;
                s[o] = v.x; s[o + 1] = v.y; s[o + 2] = v.z; s[o + 3] = v.w;
            }
        } else {
            const uint2 *sp = reinterpret_cast<const uint2 *>(c.vs + row * (2 * NG));
#pragma unroll
            for (int g = 0; g < NG; ++g)
                b[half][g] = sp[g];
        }
    }
    // MXFP4 scale of token t (0..7) for the lane's elements of group g.  Bytes above 252,
    // which no append writes, count as 252: a masked token's value stays finite.
    __device__ __forceinline__ float scale7(int t, int g) const {
        const int m = threadIdx.x & 15, h = (t & 3) * NG + g;  // 16-bit piece of the 4 tokens
        const uint2 v = b[t >> 2][h / 4];
        const uint32_t d = (h & 2) ? v.y : v.x;
        const uint32_t e = (d >> (16 * (h & 1) + 8 * (m >> 3))) & 0xffu;
        return __uint_as_float(min(e, 252u) << 23);
    }
};

// A operands of one group's values: a[j] holds element 64 g + 4 m + j of the 8 tokens.
template <int FMT, int NG>
__device__ __forceinline__ void decode_vals(const Vals<FMT, NG> &v, int g, bf16x8 (&a)[4]) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {  // tokens 2 p and 2 p + 1
        const uint32_t x = (uint32_t)v.w[g][2 * p] | ((uint32_t)v.w[g][2 * p + 1] << 16);
        uint32_t o[4];
        if constexpr (FMT == 4) {
            const uint32_t y = __builtin_amdgcn_perm(x, x, 0x03010200u);  // byte pairs of a place
            const int lo = (int)int4_signed_codes(y), hi = (int)int4_signed_codes(y >> 4);
            o[0] = as_u32(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, false));
            o[1] = as_u32(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, false));
            o[2] = as_u32(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, true));
            o[3] = as_u32(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, true));
        } else {
            const float s0 = v.scale7(2 * p, g), s1 = v.scale7(2 * p + 1, g);
            const uint32_t c0 = as_u32(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, s0, 0));
            const uint32_t c1 = as_u32(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, s0, 1));
            const uint32_t d0 = as_u32(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, s1, 2));
            const uint32_t d1 = as_u32(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, s1, 3));
            o[0] = __builtin_amdgcn_perm(d0, c0, 0x05040100u);
            o[1] = __builtin_amdgcn_perm(d0, c0, 0x07060302u);
            o[2] = __builtin_amdgcn_perm(d1, c1, 0x05040100u);
            o[3] = __builtin_amdgcn_perm(d1, c1, 0x07060302u);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bf16x2 b = as_bf2(o[j]);
            a[j][2 * p] = b[0];
            a[j][2 * p + 1] = b[1];
        }
    }
}

}  // namespace

// One workgroup: 16 rows of one sequence and kv head over one split of the tokens; its four
// waves take blocks of 32 tokens in turn and join at the end.  S^T = K q^T puts a row in a
// column of the accumulator (lanes c, c + 16, ...), so the probabilities are already where
// the second product O^T = V^T P^T wants its right operand: token order inside a product is
// free, and the value loads follow it.
template <int FMT, int NG, typename T>
__global__ __launch_bounds__(256) void k_kv4_attn(AttnArgs A) {
    constexpr int D = 64 * NG, TQ = sizeof(T) == 4 ? 3 : 1, TP = sizeof(T) == 4 ? 3 : 2;
    __shared__ __attribute__((aligned(16))) float osum[3][16][D + 4];
    __shared__ float wm[4][16], wl[4][16];
    const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int split = blockIdx.x % A.splits;
    const Tile t = tile_of(A, blockIdx.z, blockIdx.y);
    for (int r0 = blockIdx.x / A.splits * 16; r0 < t.rows; r0 += A.tiles * 16) {
    const int r1 = min(t.rows, r0 + 16);
    int lo, hi;
    span_of(A, t, r0, r1, lo, hi);
    const int s0 = max(lo & ~31, split * A.chunk);
    const int s1 = split + 1 == A.splits ? hi : min(hi, (split + 1) * A.chunk);
    const int row = r0 + col;
    const bool live = row < r1;
    const int pos = t.pos0 + (live ? row : r0) / A.group;
    const int from = A.window > 0 ? pos - A.window : -1;  // sees tokens above `from`

    bf16x8 q[NG][2][TQ];
    load_q<FMT, NG, TQ, T>(A, t, row, live, q);
    f4v o[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            o[g][j] = f4v{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    for (int t0 = s0 + 32 * wave; t0 < s1; t0 += 128) {
        Keys<FMT, NG> k[2];
        Vals<FMT, NG> v;
        bool ok[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int tt = t0 + 16 * h, pg = kv4_page_of(A.c, tt);
            const int phys = __builtin_amdgcn_readfirstlane(
                kv4_phys(A.c, t.table, A.s.max_pages, pg));
            ok[h] = phys >= 0;  // a page that is none: its tokens are not there
            const size_t r = kv4_row(A.c, max(phys, 0), t.head, tt - pg * A.c.page);
            k[h].load(A.c, r);
            v.load(A.c, r, h);
        }
        float p[8], top = m;
        uint32_t seen = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f4v s = dot_keys<FMT, NG, TQ>(k[h], q);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int tok = t0 + 16 * h + 4 * kg + i;
                const bool sees = ok[h] && live && tok < s1 && tok <= pos && tok > from;
                p[4 * h + i] = s[i];
                seen |= (uint32_t)sees << (4 * h + i);
                top = fmaxf(top, sees ? s[i] * A.scale2 : -INFINITY);
            }
        }
        top = col_max(top);
        const float ref = top == -INFINITY ? 0.f : top;
        const float fix = __builtin_amdgcn_exp2f(m - ref);
        m = top;
        l *= fix;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = (seen >> i) & 1 ? power<T>(A, p[i], ref) : 0.f;
            l += p[i];
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            bf16x8 a[4], b[TP];
            decode_vals<FMT, NG>(v, g, a);
            if constexpr (FMT == 4) {
                float ps[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)  // a masked token's scale may be anything
                    ps[i] = p[i] == 0.f ? 0.f : p[i] * v.s[i * NG + g];
                split8<TP>(ps, b);
            } else {
                split8<TP>(p, b);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[g][j] *= fix;
#pragma unroll
                for (int k = TP - 1; k >= 0; --k)
                    o[g][j] = mfma(a[j], b[k], o[g][j]);
            }
        }
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
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)  // lane: elements 64 g + 16 kg + 4 i + j
                *reinterpret_cast<float4 *>(&osum[wave - 1][col][64 * g + 16 * kg + 4 * i]) =
                    make_float4(o[g][0][i] * fix, o[g][1][i] * fix, o[g][2][i] * fix,
                                o[g][3][i] * fix);
    }
    __syncthreads();
    if (wave == 0 && live) {
    const int tok = t.first + row / A.group, head = t.head * A.group + row % A.group;
    const size_t at = ((size_t)split * A.s.n_tok + tok) * A.n_q + head;
    if (A.splits > 1) {
        if (kg == 0)
            A.ml[at] = make_float2(M, L);
    } else if (A.lse && kg == 0) {
        A.lse[at] = L > 0.f ? M + log2f(L) : -INFINITY;
    }
    // (the joining kernel leaves a part of nothing out)
    const float scale = A.splits > 1 ? 1.f : L > 0.f || L != L ? 1.f / L : 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float4 y = make_float4(o[g][0][i] * fix, o[g][1][i] * fix, o[g][2][i] * fix,
                                   o[g][3][i] * fix);
#pragma unroll
            for (int w = 0; w < 3; ++w) {
                const float4 z =
                    *reinterpret_cast<const float4 *>(&osum[w][col][64 * g + 16 * kg + 4 * i]);
                y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
            }
            x[4 * i] = y.x * scale; x[4 * i + 1] = y.y * scale;
            x[4 * i + 2] = y.z * scale; x[4 * i + 3] = y.w * scale;
        }
        const int d = 64 * g + 16 * kg;
        float x0[8], x1[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x0[i] = x[i];
            x1[i] = x[8 + i];
        }
        if (A.splits > 1) {
            Vec8<float>::store(A.part + at * D + d, x0);
            Vec8<float>::store(A.part + at * D + d + 8, x1);
        } else {
            T *out = static_cast<T *>(A.out) + ((size_t)tok * A.n_q + head) * D + d;
            Vec8<T>::store(out, x0);
            Vec8<T>::store(out + 8, x1);
        }
    }
    }
    __syncthreads();
    }
}

// Joins the splits of the rows that belong to a sequence: one workgroup of D / 8 lanes a head,
// 256 / (D / 8) heads of one token.
template <int NG, typename T>
__global__ __launch_bounds__(256) void k_kv4_join(AttnArgs A) {
    constexpr int D = 64 * NG, LPH = D / 8, HPG = 256 / LPH;
    const int tok = blockIdx.x, hi = threadIdx.x / LPH, d = (threadIdx.x % LPH) * 8;
    const int head = blockIdx.y * HPG + hi;
    if (hi >= HPG || head >= A.n_q)
        return;
    if (tok < A.s.q_start[0] || tok >= A.s.q_start[A.s.n_seq])
        return;
    const size_t at = (size_t)tok * A.n_q + head, step = (size_t)A.s.n_tok * A.n_q;
    float M = -INFINITY;
    for (int s = 0; s < A.splits; ++s)
        M = fmaxf(M, A.ml[at + s * step].x);
    float L = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < A.splits; ++s) {
        const float2 ml = A.ml[at + s * step];
        if (ml.x == -INFINITY) {
            L += ml.y;  // 0, or NaN
            continue;
        }
        const float f = __builtin_amdgcn_exp2f(ml.x - M);
        float y[8];
        Vec8<float>::load(A.part + (at + s * step) * D + d, y);
        L = fmaf(ml.y, f, L);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = fmaf(y[i], f, x[i]);
    }
    const float scale = L > 0.f || L != L ? 1.f / L : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] *= scale;
    Vec8<T>::store(static_cast<T *>(A.out) + at * D + d, x);
    if (A.lse && d == 0)
        A.lse[at] = L > 0.f ? M + log2f(L) : -INFINITY;
}

// One wave: the weights of 32 tokens of one sequence and kv head, over all of its rows: the
// keys stay in registers as operands, the rows pass by 16 at a time, and each token's sum is
// formed by this wave alone.
template <int FMT, int NG, typename T>
__global__ __launch_bounds__(256) void k_kv4_weights(AttnArgs A) {
    constexpr int TQ = sizeof(T) == 4 ? 3 : 1;
    const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const Tile t = tile_of(A, blockIdx.z, blockIdx.y);
    const int len = kv4_len(A.c, t.len, A.s.max_pages);
    for (int t0 = (blockIdx.x * 4 + wave) * 32; t0 < len; t0 += gridDim.x * 128) {
        Keys<FMT, NG> k[2];
        bool ok[2];
        size_t at[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int tt = t0 + 16 * h, pg = kv4_page_of(A.c, tt);
            const int phys = __builtin_amdgcn_readfirstlane(
                kv4_phys(A.c, t.table, A.s.max_pages, pg));
            ok[h] = phys >= 0;
            at[h] = kv4_row(A.c, max(phys, 0), t.head, tt - pg * A.c.page);
            k[h].load(A.c, at[h]);
        }
        float w[2][4] = {};
        // the first row that may see the first token, and the rows whose window it has left
        int r = (int)min((long long)t.rows, max(0ll, (long long)t0 - t.pos0) * A.group);
        int rend = t.rows;
        if (A.window > 0)
            rend = min((long long)rend,
                       max(0ll, (long long)t0 + 31 + A.window - t.pos0) * A.group);
        for (r &= ~15; r < rend; r += 16) {
            const int row = r + col;
            const bool live = row < t.rows;
            const int pos = t.pos0 + (live ? row : 0) / A.group;
            const int from = A.window > 0 ? pos - A.window : -1;
            const float lse =
                live ? A.lse[(size_t)(t.first + row / A.group) * A.n_q + t.head * A.group +
                             row % A.group]
                     : -INFINITY;
            bf16x8 q[NG][2][TQ];
            load_q<FMT, NG, TQ, T>(A, t, row, live, q);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f4v s = dot_keys<FMT, NG, TQ>(k[h], q);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = t0 + 16 * h + 4 * kg + i;
                    const bool sees = live && tok <= pos && tok > from;
                    w[h][i] += sees ? power<T>(A, s[i], lse) : 0.f;
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1)
                    w[h][i] += __shfl_xor(w[h][i], o);
            if (col < 4 && ok[h]) {
                const int tok = t0 + 16 * h + 4 * kg + col;
                const float x = col == 0 ? w[h][0] : col == 1 ? w[h][1] : col == 2 ? w[h][2]
                                                                                     : w[h][3];
                float *p = A.c.score + at[h] + 4 * kg + col;
                if (tok < len)
                    *p = A.weights == KV4_WEIGHTS_ADD ? *p + x : x;
            }
        }
    }
}

AttnPlan kv4_attention_plan(int head_dim, int n_kv, int n_q, int n_tok, int n_seq, int max_new,
                            int max_len, bool weights) {
    AttnPlan p{};
    const long long rows = (long long)max_new * (n_q / n_kv);
    p.tiles = (int)((rows + 15) / 16);
    const long long base = (long long)p.tiles * n_kv * n_seq;
    const long long want = std::max(1ll, 1024 / base);
    p.chunk = (int)std::max(256ll, ((max_len + want - 1) / want + 127) / 128 * 128);
    p.splits = (max_len + p.chunk - 1) / p.chunk;
    auto add = [&](size_t bytes) {
        const size_t at = p.bytes;
        p.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    const size_t heads = (size_t)n_tok * n_q;
    if (p.splits > 1) {
        p.part = add(p.splits * heads * head_dim * 4);
        p.ml = add(p.splits * heads * 8);
    }
    if (weights)
        p.lse = add(heads * 4);
    return p;
}

template <int FMT, int NG, typename T>
static hipError_t attention(const AttnArgs &a, int max_len, hipStream_t st) {
    const dim3 grid((unsigned)(a.splits * a.tiles), (unsigned)a.c.n_kv, (unsigned)a.s.n_seq);
    hipLaunchKernelGGL((k_kv4_attn<FMT, NG, T>), grid, dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        return e;
    if (a.splits > 1) {
        constexpr int HPG = 256 / (8 * NG);
        hipLaunchKernelGGL((k_kv4_join<NG, T>),
                           dim3((unsigned)a.s.n_tok, (unsigned)((a.n_q + HPG - 1) / HPG)),
                           dim3(256), 0, st, a);
        if ((e = hipGetLastError()) != hipSuccess)
            return e;
    }
    if (a.weights != KV4_WEIGHTS_NONE) {
        const unsigned wgs = (unsigned)std::max(1, (max_len + 127) / 128);
        hipLaunchKernelGGL((k_kv4_weights<FMT, NG, T>),
                           dim3(wgs, (unsigned)a.c.n_kv, (unsigned)a.s.n_seq), dim3(256), 0, st,
                           a);
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
