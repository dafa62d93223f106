// kern_prompt.hip -- attention of many new tokens over keys and values held in 4 bits, for
// gfx950 (the rows and formulas of kern_attn.hip).
//
// One workgroup: W waves of 32 rows each over the same tokens, in tiles of KT.  The tile's codes
// are decoded once for all waves, into LDS, as the matrix cores' left operands in the order of
// the lanes that read them: S^T = K q^T, then O^T = V^T P^T with the probabilities where the
// first product left them.
//
// Operands are f16, with powers of two taken out: a row of queries by its largest magnitude, a
// tile of keys by its largest scale, the values by the largest scale so far (the sums move
// along), so that each set's largest magnitude lies near 2^14 and what is up to 2^28 smaller
// keeps its 11 bits.  bf16 queries and MXFP4 codes times their scales are then exact; int4 codes
// times their scales, and probabilities, are rounded by up to 2^-11 of themselves, values' scales
// before as well (bf16 outputs round by 2^-8; bf16 operands would have added as much again).
// Keys' scales are not: a token's exponents would all be off by its scale's rounding, which
// 6000 tokens of narrow heads made half as much again as the output's own rounding (2-norm 2.4e-3
// of it, 1.9e-3 so; 64-element heads).  f32 calls take two f16 terms of each rounded operand and
// leave out the product of the two second ones (2^-22 each); calls that collect weights two
// of the keys.
//
// A tile's scales are prepared by one wave, in turn, two tiles ahead: it takes the powers out,
// zeroes the scales of tokens that are not there, and gives a token whose value scales are not
// finite a NaN key (so the rows that see it become NaN, and no others).
//
// 2 sequences, 32 heads on 8 of 128, 1024 new tokens over 6000 to 8192, bf16 over int4: 197 GFLOP
// in 324 us, 607 TFLOP/s, half of what a large matrix product reaches.  What bounds it is that a
// tile's decoding, products and exponentials cover each other only in part: the vector ALU is
// busy 51 % of the time and the matrix cores 36 %, two waves a SIMD.  4 waves a workgroup were
// slower (each decodes twice as much); waves half a tile apart, priorities and interleaved
// exponentials changed nothing.
#include "kv4_common.h"

#include <algorithm>
#include <cmath>

namespace mvllm_hip {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float fl2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f4v mfma16(h8 a, h8 b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ h2 as_h2(uint32_t u) { return __builtin_bit_cast(h2, u); }
__device__ __forceinline__ uint32_t as_u32(h2 h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ h2 round2(float a, float b) {
    return __builtin_convertvector(fl2{a, b}, h2);
}
__device__ __forceinline__ float col_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float col_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
// Largest of the wave's values, each not negative (ordered as their bits).
__device__ __forceinline__ float wave_top(float x) {
    uint32_t v = __float_as_uint(x);
#define TOP_STEP(ctrl) \
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, false))
    TOP_STEP(0x111);  // row_shr:1, 2, 4, 8, then the rows' last lanes on to the next rows
    TOP_STEP(0x112);
    TOP_STEP(0x114);
    TOP_STEP(0x118);
    TOP_STEP(0x142);
    TOP_STEP(0x143);
#undef TOP_STEP
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)v, 63));
}
__device__ __forceinline__ int exponent(float x) {
    return (int)((__float_as_uint(x) >> 23) & 255u) - 127;
}

// What the scale wave says of a tile.
struct TileInfo {
    int ek, ev;              // powers of two taken out of the keys and of the values
    uint32_t there[2];       // bit t: token t of the tile exists
};

// LSE: the call collects weights, so the rows' sums are held to f32: keys in two terms.
template <int FMT, int NG, typename T, bool LSE> struct PromptShape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int D = 64 * NG, KS = 2 * NG, NF = 4 * NG;  // 32-element steps, row blocks
    static constexpr int KT = (F32 || LSE) && FMT == 4 && NG >= 3 ? 32 : 64;
    // terms of queries and probabilities, of keys, of values
    static constexpr int QT = F32 ? 2 : 1;
    static constexpr int KKT = FMT == 4 && (F32 || LSE) ? 2 : 1, KVT = FMT == 4 && F32 ? 2 : 1;
    static constexpr int SB = FMT == 4 ? NG : 2 * NG;  // scales of a row
    // a scale as the decoding reads it, where its product with a code is rounded to f16: of
    // values an f16, of keys an f16 and what that leaves
    using KScale = std::conditional_t<FMT == 4 && KKT == 1, h2, float>;
    using VScale = std::conditional_t<FMT == 4 && KVT == 1, _Float16, float>;
    struct Buf {
        h8 k[KKT][KT / 16][KS][64];
        h8 v[KVT][KT / 32][NF][64];
    };
    struct Lds {
        Buf buf[2];
        KScale sk[2][SB][KT];
        VScale sv[2][SB][KT];
        TileInfo info[4];
    };
};

// (n - 8) of the nibbles of one dword's low bits, as f16 pairs: the two nibbles at bits 0 and 16
// (o[0]) and at bits 4 and 20 (o[1]).  A nibble in the mantissa of 1024 (or, 4 bits up, of 64)
// adds itself.
struct Int4Pairs {
    uint32_t m1024 = 0x64006400u, m64 = 0x54005400u;

    // The constants in vector registers: masking and inserting are one instruction then.
    __device__ __forceinline__ Int4Pairs() { asm("" : "+v"(m1024), "+v"(m64)); }
    __device__ __forceinline__ void operator()(uint32_t x, h2 &a, h2 &b) const {
        a = as_h2((x & 0x000f000fu) | m1024) - h2{(_Float16)1032.f, (_Float16)1032.f};
        b = as_h2((x & 0x00f000f0u) | m64) - h2{(_Float16)72.f, (_Float16)72.f};
    }
};

template <int FMT, int NG, typename T, int W, bool LSE> struct Prompt {
    using S = PromptShape<FMT, NG, T, LSE>;
    static constexpr int KT = S::KT, KS = S::KS, NF = S::NF, KKT = S::KKT, KVT = S::KVT;
    static constexpr int SB = S::SB, D = S::D;
    static constexpr int U = KT * KS;                     // units of keys, and of values
    static constexpr int NT = 64 * W, NU = (2 * U + NT - 1) / NT;  // a thread's units

    const AttnArgs &A;
    typename S::Lds &L;
    const int *table;
    int head, s0, s1, wave;

    // One unit of a tile on its way: 32 codes.  Keys: 16 bytes of one token (elements 32 p..);
    // values: elements 64 G + 4 m + j of the 8 tokens of one lane of the second product.
    struct Unit {
        int entry[2];  // of the table, as loaded
        uint4 k;
        uint16_t v[8];
    };
    Unit u[NU];

    // A token's table entry: loaded a tile ahead and looked at only where it is used, so that no
    // wave waits for it.
    __device__ __forceinline__ int entry_of(int t) const {
        return table[min(kv4_page_of(A.c, t), A.s.max_pages - 1)];
    }
    __device__ __forceinline__ int page_of(int t, int entry) const {  // -1: none
        return kv4_page_of(A.c, t) < A.s.max_pages && (unsigned)entry < (unsigned)A.c.n_pages ? entry
                                                                                              : -1;
    }
    __device__ __forceinline__ int slot_of(int t) const { return t - kv4_page_of(A.c, t) * A.c.page; }

    // The table entries of the units' tokens in a tile.
    __device__ __forceinline__ void look(int tile) {
        const int t0 = s0 + tile * KT;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int n = (int)threadIdx.x + i * NT, w = 64 * wave + i * NT;  // (U % 64 = 0)
            if (w < U) {
                u[i].entry[0] = entry_of(t0 + n / (16 * KS) * 16);
            } else if (w < 2 * U) {
                const int b = (n - U) / (64 * NG);
                u[i].entry[0] = entry_of(t0 + 32 * b);
                u[i].entry[1] = entry_of(t0 + 32 * b + 16);
            }
        }
    }
    // Their codes (page 0's in place of none).
    __device__ __forceinline__ void fetch(int tile) {
        const int t0 = s0 + tile * KT;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int n = (int)threadIdx.x + i * NT, w = 64 * wave + i * NT;
            if (w < U) {
                const int m = n & 15, p = (n >> 4) % KS, t = t0 + n / (16 * KS) * 16;
                const size_t r = kv4_row(A.c, max(page_of(t, u[i].entry[0]), 0), head, slot_of(t) + m);
                u[i].k = *reinterpret_cast<const uint4 *>(A.c.k + r * (D / 2) + 16 * p);
            } else if (w < 2 * U) {
                const int v = n - U, m = v & 15, kg = (v >> 4) & 3, G = (v >> 6) % NG;
                const int t = t0 + v / (64 * NG) * 32;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int th = t + 16 * h, pg = max(page_of(th, u[i].entry[h]), 0);
                    const size_t r = kv4_row(A.c, pg, head, slot_of(th) + 4 * kg);
                    const uint8_t *x = A.c.v + r * (D / 2) + 32 * G + 2 * m;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        u[i].v[4 * h + e] = *reinterpret_cast<const uint16_t *>(x + e * (D / 2));
                }
            }
        }
    }

    // (n - 8) * s, rounded to f16: keys' with one rounding, values' with the scale's own before.
    __device__ __forceinline__ static void scaled(h2 n, h2 s, h2, h2 (&o)[1]) {
        o[0] = __builtin_elementwise_fma(n, h2{s[0], s[0]}, n * h2{s[1], s[1]});
    }
    __device__ __forceinline__ static void scaled(h2 n, _Float16 s0, _Float16 s1, h2 (&o)[1]) {
        o[0] = n * h2{s0, s1};
    }
    // Two terms of the f32 product.
    __device__ __forceinline__ static void scaled(h2 n, float s0, float s1, h2 (&o)[2]) {
        const float a = (float)n[0] * s0, b = (float)n[1] * s1;
        o[0] = round2(a, b);
        o[1] = round2(a - (float)o[0][0], b - (float)o[0][1]);
    }

    // Decodes the fetched tile into its buffer.
    __device__ __forceinline__ void decode(int tile) {
        auto &B = L.buf[tile & 1];
        const Int4Pairs int4_pairs;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int n = (int)threadIdx.x + i * NT, w = 64 * wave + i * NT;
            if (w < U) {
                const uint32_t word[4] = {u[i].k.x, u[i].k.y, u[i].k.z, u[i].k.w};
                const int m = n & 15, p = (n >> 4) % KS, st = n / (16 * KS);
                const auto s = L.sk[tile & 1][FMT == 4 ? p / 2 : p][st * 16 + m];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    h8 o[KKT];
                    if constexpr (FMT == 4) {  // order 0 4 1 5 2 6 3 7
                        h2 x[4];
                        int4_pairs(word[j], x[0], x[1]);
                        int4_pairs(word[j] >> 8, x[2], x[3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            h2 y[KKT];
                            scaled(x[e], s, s, y);
#pragma unroll
                            for (int k = 0; k < KKT; ++k) {
                                o[k][2 * e] = y[k][0];
                                o[k][2 * e + 1] = y[k][1];
                            }
                        }
                    } else {
                        const h2 x[4] = {
                            __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word[j], s, 0),
                            __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word[j], s, 1),
                            __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word[j], s, 2),
                            __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word[j], s, 3)};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[0][2 * e] = x[e][0];
                            o[0][2 * e + 1] = x[e][1];
                        }
                    }
#pragma unroll
                    for (int k = 0; k < KKT; ++k)
                        B.k[k][st][p][j * 16 + m] = o[k];
                }
            } else if (w < 2 * U) {
                const int v = n - U, m = v & 15, kg = (v >> 4) & 3, G = (v >> 6) % NG;
                const int b = v / (64 * NG);
                const auto *sp = L.sv[tile & 1][FMT == 4 ? G : 2 * G + (m >> 3)] + 32 * b + 4 * kg;
                h8 o[KVT][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // tokens 2 e and 2 e + 1 of the lane's eight
                    const auto s0 = sp[16 * (e >> 1) + 2 * (e & 1)];
                    const auto s1 = sp[16 * (e >> 1) + 2 * (e & 1) + 1];
                    const uint32_t x = u[i].v[2 * e] | ((uint32_t)u[i].v[2 * e + 1] << 16);
                    h2 y[4][KVT];
                    if constexpr (FMT == 4) {
                        h2 z[4];
                        int4_pairs(x, z[0], z[1]);
                        int4_pairs(x >> 8, z[2], z[3]);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            scaled(z[j], s0, s1, y[j]);
                    } else {
                        // (the token's own pair of bytes, its own scale)
                        const uint32_t c[4] = {
                            as_u32(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, s0, 0)),
                            as_u32(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, s0, 1)),
                            as_u32(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, s1, 2)),
                            as_u32(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, s1, 3))};
                        y[0][0] = as_h2(__builtin_amdgcn_perm(c[2], c[0], 0x05040100u));
                        y[1][0] = as_h2(__builtin_amdgcn_perm(c[2], c[0], 0x07060302u));
                        y[2][0] = as_h2(__builtin_amdgcn_perm(c[3], c[1], 0x05040100u));
                        y[3][0] = as_h2(__builtin_amdgcn_perm(c[3], c[1], 0x07060302u));
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int k = 0; k < KVT; ++k) {
                            o[k][j][2 * e] = y[j][k][0];
                            o[k][j][2 * e + 1] = y[j][k][1];
                        }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int k = 0; k < KVT; ++k)
                        B.v[k][b][4 * G + j][kg * 16 + m] = o[k][j];
            }
        }
    }

    // ---- the scale wave: lane t is token t of the tile (KT = 32: the upper half repeats it)
    float sk[FMT == 4 ? NG : 2 * NG], sv[FMT == 4 ? NG : 2 * NG];
    int entry;
    bool there;

    __device__ __forceinline__ void look_scales(int tile) {
        entry = entry_of(s0 + tile * KT + ((int)threadIdx.x & (KT - 1)));
    }
    __device__ __forceinline__ void fetch_scales(int tile) {
        const int t = s0 + tile * KT + ((int)threadIdx.x & (KT - 1));
        const int phys = t < s1 ? page_of(t, entry) : -1;
        there = phys >= 0;
        const size_t r = there ? kv4_row(A.c, phys, head, slot_of(t)) : 0;
#pragma unroll
        for (int g = 0; g < SB; ++g) {
            if constexpr (FMT == 4) {
                sk[g] = reinterpret_cast<const float *>(A.c.ks)[r * SB + g];
                sv[g] = reinterpret_cast<const float *>(A.c.vs)[r * SB + g];
            } else {
                sk[g] = ue8m0_ref(A.c.ks[r * SB + g]);
                sv[g] = ue8m0_ref(A.c.vs[r * SB + g]);
            }
        }
    }
    __device__ __forceinline__ void put_scales(int tile) {
        // the largest scale goes to 2^10..2^11 (codes up to 8), or 2^12 (codes up to 6)
        constexpr int TOP = FMT == 4 ? 10 : 12;
        const int lane = (int)threadIdx.x & 63, t = lane & (KT - 1);
        bool good = true;
        float mk = 0.f, mv = 0.f;
#pragma unroll
        for (int g = 0; g < SB; ++g) {
            good = good && !nonfinite(sv[g]);
            sk[g] = there ? sk[g] : 0.f;
            sv[g] = there && !nonfinite(sv[g]) ? sv[g] : 0.f;
            mk = fmaxf(mk, nonfinite(sk[g]) ? 0.f : fabsf(sk[g]));
            mv = fmaxf(mv, fabsf(sv[g]));
        }
        mk = wave_top(mk);
        mv = wave_top(mv);
        const int ek = mk > 0.f ? exponent(mk) - TOP : 0;
        int ev = tile > 0 ? L.info[(tile - 1) & 3].ev : -1000;
        ev = mv > 0.f ? max(ev, exponent(mv) - TOP) : ev;
        const uint64_t mask = __ballot(there);
        if (lane < KT) {
#pragma unroll
            for (int g = 0; g < SB; ++g) {
                const float k = there && !good ? NAN : ldexpf(sk[g], -ek);
                if constexpr (std::is_same_v<typename S::KScale, h2>)
                    L.sk[tile & 1][g][t] = h2{(_Float16)k, (_Float16)(k - (float)(_Float16)k)};
                else
                    L.sk[tile & 1][g][t] = k;
                L.sv[tile & 1][g][t] = (typename S::VScale)ldexpf(sv[g], -max(ev, -400));
            }
        }
        if (lane == 0) {
            TileInfo &I = L.info[tile & 3];
            I.ek = ek;
            I.ev = ev;
            I.there[0] = (uint32_t)mask;
            I.there[1] = KT == 64 ? (uint32_t)(mask >> 32) : 0u;
        }
    }
};

}  // namespace

template <int FMT, int NG, typename T, int W, bool LSE>
__global__ __launch_bounds__(64 * W, NG <= 2 ? 2 : 1) void k_kv4_prompt(AttnArgs A) {
    using S = PromptShape<FMT, NG, T, LSE>;
    constexpr int D = S::D, KT = S::KT, KS = S::KS, NF = S::NF, QT = S::QT;
    constexpr int KKT = S::KKT, KVT = S::KVT;
    // The rows' sums come with the values' products, of the probabilities as rounded; where they
    // have to be f32 and one term is all there is, from the f32 ones.
    constexpr bool SUMS = LSE && QT == 1;
    // Probabilities are carried as 2^(x - ref): up to 2^15 in f16, and so that a maximum that is
    // not raised yet (it may pass by 2^SLACK) still fits.
    constexpr float SLACK = S::F32 ? 1.f : 8.f, LIFT = 15.f - SLACK;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typename S::Lds &L = *reinterpret_cast<typename S::Lds *>(smem);
    const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int split = blockIdx.z % A.splits, seq = blockIdx.y, head = blockIdx.x;
    const int q0 = max(0, min(A.s.q_start[seq], A.s.n_tok));
    const int rows = (max(q0, min(A.s.q_start[seq + 1], A.s.n_tok)) - q0) * A.group;
    const int slen = A.s.lens[seq], pos0 = slen - rows / A.group;
    const int len = kv4_len(A.c, slen, A.s.max_pages);
    for (int base = blockIdx.z / A.splits * 32 * W; base < rows; base += A.tiles * 32 * W) {
        const int last = min(rows, base + 32 * W) - 1;
        const int hi = max(0, min(pos0 + last / A.group + 1, len));
        const int lo =
            A.window > 0 ? max(0, min(max(pos0 + base / A.group, 0) - A.window + 1, hi)) : 0;
        const int s0 = (int)min((long long)hi, (lo & ~(KT - 1)) + (long long)split * A.chunk);
        const int s1 = split + 1 == A.splits ? hi : min(hi - s0, A.chunk) + s0;
        const int n_tiles = s1 > s0 ? (s1 - s0 + KT - 1) / KT : 0;
        Prompt<FMT, NG, T, W, LSE> P{A, L, A.s.table + (size_t)seq * A.s.max_pages, head, s0, s1, wave};

        // the wave's rows: columns col and 16 + col
        const int w0 = base + 32 * wave, w1 = min(rows, w0 + 32);
        int row[2], pos[2], from[2];
        float c2[2];  // log2 units of a product of the rows' operands, without the keys' power
        int eq[2];
        bool live[2];
        h8 q[2][KS][QT];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            row[c] = w0 + 16 * c + col;
            live[c] = row[c] < w1;
            const int r = live[c] ? row[c] : base;
            pos[c] = pos0 + r / A.group;
            from[c] = A.window > 0 ? pos[c] - A.window : -1;
            const T *p = static_cast<const T *>(A.q) + (size_t)(q0 + r / A.group) * A.q_stride +
                         (size_t)(head * A.group + r % A.group) * D + 8 * kg;
            float x[KS][8], top = 0.f;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                Vec8<T>::load(p + 32 * s, x[s]);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    top = fmaxf(top, fabsf(x[s][e]));
            }
            top = col_max(top);
            eq[c] = top > 0.f && !nonfinite(top) ? exponent(top) - 14 : 0;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float y = ldexpf(A.scale2 < 0.f ? -x[s][e] : x[s][e], -eq[c]);
                    const int at = FMT == 4 ? 2 * (e & 3) + (e >> 2) : e;
#pragma unroll
                    for (int k = 0; k < QT; ++k) {
                        q[c][s][k][at] = (_Float16)y;
                        y -= (float)q[c][s][k][at];
                    }
                }
            c2[c] = fabsf(A.scale2);
        }
        // tokens that all of the wave's rows see
        const int all1 = min(s1, pos0 + w0 / A.group + 1);
        const int all0 = A.window > 0 ? pos0 + (w1 - 1) / A.group - A.window + 1 : 0;
        // tokens past the last that some row of the wave sees
        const int end = w0 < w1 ? pos0 + (w1 - 1) / A.group + 1 : 0;

        f4v o[NF][2];
#pragma unroll
        for (int f = 0; f < NF; ++f)
            o[f][0] = o[f][1] = f4v{0.f, 0.f, 0.f, 0.f};
        // the rows' sums of probabilities (in every row of the accumulator); ref: see LIFT
        f4v l[2] = {f4v{0.f, 0.f, 0.f, 0.f}, f4v{0.f, 0.f, 0.f, 0.f}};
        float ref[2] = {-INFINITY, -INFINITY};
        h8 ones;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            ones[i] = (_Float16)1.f;
        int ev = -1000;

        if (n_tiles > 0) {
            P.look(0);
            // (a tile behind the last: nothing there)
            P.look_scales(wave);
            if (wave < 3) {
                P.fetch_scales(wave);
                P.look_scales(wave + W);
            }
            P.fetch(0);
            P.look(1);
            if (wave == 0)
                P.put_scales(0);
            __syncthreads();
            if (wave == 1)
                P.put_scales(1);
            P.decode(0);
            P.fetch(1);
            P.look(2);
            __syncthreads();
        }
        for (int tile = 0; tile < n_tiles; ++tile) {
            if (wave == (tile + 2) % W)
                P.put_scales(tile + 2);
            if (wave == (tile + 3) % W) {
                P.fetch_scales(tile + 3);
                P.look_scales(tile + 3 + W);
            }
            P.decode(tile + 1);  // (of a tile behind the last: zeros)
            P.fetch(tile + 2);
            P.look(tile + 3);
            const int t0 = s0 + tile * KT;
            const TileInfo I = L.info[tile & 3];
            const auto &B = L.buf[tile & 1];
            if (t0 < end) {  // (wave-uniform)
                f4v s[KT / 16][2];
#pragma unroll
                for (int b = 0; b < KT / 16; ++b) {
                    s[b][0] = s[b][1] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int p = 0; p < KS; ++p) {
#pragma unroll
                        for (int k = KKT - 1; k >= 0; --k) {
                            const h8 a = B.k[k][b][p][lane];
#pragma unroll
                            for (int t = (KKT > QT ? KKT : QT) - 1 - k; t >= 0; --t) {
                                if (t >= QT)
                                    continue;
                                s[b][0] = mfma16(a, q[0][p][t], s[b][0]);
                                s[b][1] = mfma16(a, q[1][p][t], s[b][1]);
                            }
                        }
                    }
                }
                const uint32_t full = KT == 64 ? ~0u : 0u;
                const bool whole = t0 >= all0 && t0 + KT <= all1 && I.there[0] == ~0u &&
                                   I.there[1] == full;
                if (!whole) {
                    asm volatile("");  // a branch, not selects in every tile
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int b = 0; b < KT / 16; ++b)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int n = 16 * b + 4 * kg + i, tok = t0 + n;
                                const bool sees = ((I.there[b >> 1] >> (n & 31)) & 1) &&
                                                  tok <= pos[c] && tok > from[c];
                                s[b][c][i] = sees ? s[b][c][i] : -INFINITY;
                            }
                }
                // the values' power of two has grown: so do the sums' units
                if (I.ev != ev) {
                    const float f = ldexpf(1.f, max(ev - I.ev, -400));
                    ev = I.ev;
#pragma unroll
                    for (int n = 0; n < NF; ++n) {
                        o[n][0] *= f;
                        o[n][1] *= f;
                    }
                }
                h8 pr[2][KT / 32][QT];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    // never 0: a masked -inf stays -inf
                    const float k2 = fmaxf(ldexpf(c2[c], I.ek + eq[c]), 0x1p-126f);
                    const float k2lo =
                        S::F32 ? ldexpf(A.scale2 < 0.f ? -A.scale2_lo : A.scale2_lo, I.ek + eq[c])
                               : 0.f;
                    float top = -INFINITY;
#pragma unroll
                    for (int b = 0; b < KT / 16; ++b) {
                        top = fmaxf(fmaxf(top, s[b][c][0]), s[b][c][1]);
                        top = fmaxf(fmaxf(top, s[b][c][2]), s[b][c][3]);
                    }
                    top = top * k2 - LIFT;
                    if (__any(top > ref[c] + SLACK)) {
                        const float up = fmaxf(ref[c], col_max(top));
                        const float f = up == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref[c] - up);
                        ref[c] = up;
                        l[c] *= f;
#pragma unroll
                        for (int n = 0; n < NF; ++n)
                            o[n][c] *= f;
                    }
                    const float r = ref[c] == -INFINITY ? 0.f : ref[c];
#pragma unroll
                    for (int b = 0; b < KT / 32; ++b) {
                        float p[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float x = s[2 * b + (i >> 2)][c][i & 3];
                            if constexpr (S::F32)
                                p[i] = x == -INFINITY
                                           ? 0.f
                                           : __builtin_amdgcn_exp2f(fmaf(x, k2, fmaf(x, k2lo, -r)));
                            else
                                p[i] = __builtin_amdgcn_exp2f(fmaf(x, k2, -r));
                        }
                        if constexpr (SUMS)
                            l[c][0] += ((p[0] + p[1]) + (p[2] + p[3])) +
                                       ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
                        for (int k = 0; k < QT; ++k)
#pragma unroll
                            for (int i = 0; i < 8; i += 2) {
                                const h2 y = round2(p[i], p[i + 1]);
                                pr[c][b][k][i] = y[0];
                                pr[c][b][k][i + 1] = y[1];
                                p[i] -= (float)y[0];
                                p[i + 1] -= (float)y[1];
                            }
                    }
                }
#pragma unroll
                for (int b = 0; b < KT / 32; ++b) {
#pragma unroll
                    for (int t = SUMS ? -1 : QT - 1; t >= 0; --t) {
                        l[0] = mfma16(ones, pr[0][b][t], l[0]);
                        l[1] = mfma16(ones, pr[1][b][t], l[1]);
                    }
#pragma unroll
                    for (int n = 0; n < NF; ++n)
#pragma unroll
                        for (int k = KVT - 1; k >= 0; --k) {
                            const h8 a = B.v[k][b][n][lane];
#pragma unroll
                            for (int t = QT - 1 - k; t >= 0; --t) {
                                o[n][0] = mfma16(a, pr[0][b][t], o[n][0]);
                                o[n][1] = mfma16(a, pr[1][b][t], o[n][1]);
                            }
                        }
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float sum = SUMS ? col_sum(l[c][0]) : l[c][0];
            if (live[c]) {
                const int tok = q0 + row[c] / A.group, hq = head * A.group + row[c] % A.group;
                const size_t at = ((size_t)split * A.s.n_tok + tok) * A.n_q + hq;
                if (A.splits > 1) {
                    if (kg == 0)
                        A.ml[at] = make_float2(ref[c], sum);
                } else if (A.lse && kg == 0) {
                    A.lse[at] = sum > 0.f ? ref[c] + log2f(sum) : -INFINITY;
                }
                const float f = ldexpf(A.splits > 1           ? 1.f
                                       : sum > 0.f || sum != sum ? 1.f / sum
                                                                 : 0.f,
                                       max(ev, -400));
                if (A.splits == 1 || ref[c] != -INFINITY) {  // (the join leaves nothing out)
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        float x[2][8];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                x[i >> 1][4 * (i & 1) + j] = o[4 * g + j][c][i] * f;
                        const int d = 64 * g + 16 * kg;
                        if (A.splits > 1) {
                            Vec8<float>::store(A.part + at * D + d, x[0]);
                            Vec8<float>::store(A.part + at * D + d + 8, x[1]);
                        } else {
                            T *out = static_cast<T *>(A.out) + ((size_t)tok * A.n_q + hq) * D + d;
                            Vec8<T>::store(out, x[0]);
                            Vec8<T>::store(out + 8, x[1]);
                        }
                    }
                }
            }
        }
        __syncthreads();
    }
}

template <int FMT, int NG, typename T, int W, bool LSE>
static hipError_t prompt_one(const AttnArgs &a, hipStream_t st) {
    using Lds = typename PromptShape<FMT, NG, T, LSE>::Lds;
    static_assert(sizeof(Lds) <= 160 * 1024, "LDS");
    static const hipError_t lds = hipFuncSetAttribute(
        reinterpret_cast<const void *>(&k_kv4_prompt<FMT, NG, T, W, LSE>),
        hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Lds));
    if (lds != hipSuccess)
        return lds;
    const dim3 grid((unsigned)a.c.n_kv, (unsigned)a.s.n_seq, (unsigned)(a.splits * a.tiles));
    hipLaunchKernelGGL((k_kv4_prompt<FMT, NG, T, W, LSE>), grid, dim3(64 * W), sizeof(Lds), st, a);
    return hipGetLastError();
}

template <int FMT, int NG, typename T, int W>
static hipError_t prompt(const AttnArgs &a, hipStream_t st) {
    if constexpr (sizeof(T) == 2)  // (f32 calls hold their sums to f32 anyway)
        return a.lse ? prompt_one<FMT, NG, T, W, true>(a, st)
                     : prompt_one<FMT, NG, T, W, false>(a, st);
    return prompt_one<FMT, NG, T, W, false>(a, st);
}

template <int FMT, typename T>
static hipError_t prompt_dim(int D, const AttnArgs &a, hipStream_t st) {
    return D == 64    ? prompt<FMT, 1, T, 8>(a, st)
           : D == 128 ? prompt<FMT, 2, T, 8>(a, st)
           : D == 192 ? prompt<FMT, 3, T, 4>(a, st)
           : D == 256 ? prompt<FMT, 4, T, 4>(a, st)
                      : hipErrorInvalidValue;
}

hipError_t launch_kv4_prompt(int fmt, int D, int dtype, const AttnArgs &a, hipStream_t st) {
    if (dtype == KV4_BF16)
        return fmt == 4 ? prompt_dim<4, __bf16>(D, a, st) : prompt_dim<7, __bf16>(D, a, st);
    return fmt == 4 ? prompt_dim<4, float>(D, a, st) : prompt_dim<7, float>(D, a, st);
}

}  // namespace mvllm_hip
