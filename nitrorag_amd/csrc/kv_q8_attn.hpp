// Attention over an 8-bit paged cache on gfx950 (layout: kv_q8.hpp): what decode and
// causal prefill share, a wave's pass over tiles of 64 keys for 16 query rows.
//
// Mathematics.  Keys and values are k_j = ks_j * K_j, v_j = vs_j * V_j with int8
// codes K_j, V_j.  A query row q is held as q = qa/F * Q, Q = rint(q * F/qa) a
// 24-bit integer (qa = max |q|, F = 8355000), in three signed 8-bit digits
// Q = 65536 D2 + 256 D1 + D0, so
//   q.k_j = qa/F * ks_j * (256 * (256 D2.K_j + D1.K_j) + D0.K_j)
// with every dot product an exact integer (v_mfma_i32_16x16x64_i8, the codes as
// they lie in the cache).  A tile of 64 keys has m = max_j s_j, p_j = 2^(s_j - m)
// and w_j = p_j vs_j, which becomes a 24-bit integer of its own largest value W
// in the same three digits: sum_j w_j V_j comes out of the same instructions, and
// joins the running (max, sum, output) in fp32.
//
// Error: Q is off by at most half a unit of the row's largest entry / F, w by half a
// unit of the largest weight / F of the tile (in prefill of two tiles).  The digits'
// sums are exact; joined, they are rounded to 256 units once per score and once per
// output and tile (16 bits below the largest entry times one code, beside a sum over
// all dimensions or keys).  Against 64 bits, outputs over N(0, 1) rows are off by 2e-7
// of their norm at 1 to 16 keys, 2.5e-7 at 64 and 3.4e-7 at 4096, where fp32 products
// summed one after the other leave 3e-8 at one key, 2e-7 at 16, 3e-7 at 64 and 1.4e-6
// at 4096: short contexts are held less exactly than in fp32, longer ones more so.  Two
// digits would leave 1e-5 and more; bf16 or fp16 parts of q and w need K and V
// converted, one or more vector instructions per element and wave.
//
// Operand order.  A wave's tile is four pages.  For its keys as the product's
// rows, row m of product t (t = 0..3) is page m / 4, token 4t + m % 4; the result
// then leaves lane (g = lane / 16, column) with the 16 tokens of page g in token
// order, which is what the second product wants as its operand: the weights never
// leave their lane.  V columns come as 16 bytes = 16 tokens of one page.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "device_pool.hpp"
#include "kv_q8.hpp"

namespace nitro {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // caller's rows

constexpr float FIXED = 8355000.0f;  // below 127 * 65536 + 127 * 256 + 127, the largest three digits hold
constexpr float UNIT = 0x1p-20f;  // between a score's two factors
// Least W that fixed point takes (FIXED / W stays in fp32's range).
constexpr float LEAST = 0x1p-104f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float scale_of(float m, float m_new) { return m == -INFINITY ? 0.0f : exp2_fast(m - m_new); }

// Over the four lanes that share a column (l, l ^ 16, l ^ 32, l ^ 48).
template <bool HALVES>
__device__ __forceinline__ void pair_values(float x, float& a, float& b) {
    if constexpr (HALVES) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
    } else {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
    }
}
__device__ __forceinline__ float column_max(float x) {
    float a, b;
    pair_values<false>(x, a, b);
    x = fmaxf(a, b);
    pair_values<true>(x, a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float column_sum(float x) {
    float a, b;
    pair_values<false>(x, a, b);
    x = a + b;
    pair_values<true>(x, a, b);
    return a + b;
}

// Digits of four integers v (|v| <= FIXED), v = 65536 d2 + 256 d1 + d0, given as
// words whose low three bytes are v + 0x8080, that is d2, d1 + 128 and d0 + 128.
// Digit n of each goes to the bytes of d[n].  For v >= 0 the word is the float
// v + BIAS: its mantissa is v + 0x8080, and the exponent's lowest bit is 0.
constexpr float BIAS = 8388608.0f + 32896.0f;  // 2^23 + 0x8080
__device__ __forceinline__ void digits(float x0, float x1, float x2, float x3, int& d0, int& d1, int& d2) {
    const uint32_t u0 = __float_as_uint(x0), u1 = __float_as_uint(x1), u2 = __float_as_uint(x2), u3 = __float_as_uint(x3);
    const uint32_t a = __builtin_amdgcn_perm(u1, u0, 0x05010400u), b = __builtin_amdgcn_perm(u3, u2, 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(u1, u0, 0x0c0c0602u), d = __builtin_amdgcn_perm(u3, u2, 0x0c0c0602u);
    d0 = (int)(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u);
    d1 = (int)(__builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u);
    d2 = (int)__builtin_amdgcn_perm(d, c, 0x05040100u);
}

// A lane's query operand (column lane % 16, dimensions 16 * (4j + lane / 16) ..
// + 16 of step j): three digits, and what a score's integer is multiplied by.
template <int NC>
struct Query {
    i4 d[NC][3];
    float scale;
};

// A lane's part of its column's query row as it lies in memory (zeros where row is
// nullptr: a column without one).
template <int NC>
struct QueryRow {
    f4 x[NC][4];
};
template <int NC>
__device__ __forceinline__ QueryRow<NC> load_row(const float* row, int hd, int g) {
    QueryRow<NC> q;
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int dim = 16 * (4 * j + g) + 4 * i;
            q.x[j][i] = f4{0.f, 0.f, 0.f, 0.f};
            if (row && dim < hd) q.x[j][i] = *reinterpret_cast<const f4*>(row + dim);
        }
    return q;
}

template <int NC>
__device__ __forceinline__ Query<NC> query_of(const QueryRow<NC>& from, float qscale) {
    float top = 0.0f, bad = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                top = fmaxf(top, fabsf(from.x[j][i][e]));
                bad = fmaf(from.x[j][i][e], 0.0f, bad);
            }
    top = column_max(top);
    bad = column_sum(bad);  // NaN where the row holds an infinity or a NaN
    const float inv = top >= 0x1p-100f ? FIXED / top : 0.0f;
    Query<NC> q;
    // (never 0: a hidden key's -infinity stays one)
    q.scale = (top >= 0x1p-100f ? top : 0x1p-100f) * (qscale * (256.0f / UNIT / FIXED)) + bad;
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // signed: as an integer, its bits then like a biased float's
            float v[4];
            int d0, d1, d2;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = __int_as_float((int)rintf(from.x[j][i][e] * inv) + 0x8080);
            digits(v[0], v[1], v[2], v[3], d0, d1, d2);
            q.d[j][0][i] = d0, q.d[j][1][i] = d1, q.d[j][2][i] = d2;
        }
    return q;
}

// What a wave carries from tile to tile: per lane, of its column, the maximum, its
// own pages' part of the sum, and output dimensions 16t + 4 * (lane / 16) .. + 4.
template <int CH>
struct State {
    float m = -INFINITY, l = 0.0f;
    f4 o[CH];
};

// What a wave holds of a tile: the K operands of its four products and the V
// operands, and both scales of token lane % 16 of page lane / 16.  STREAM: lines that nothing else
// reads, kept out of the caches.
// CH: hdp / 16; a K row is CH runs of 16 dimensions, of which a lane has NC = CH / 4,
// rounded up (zeros where there are fewer).
template <int CH>
struct KTile {
    i4 k[4][(CH + 3) / 4];
    float ks, vs;
};
template <int CH>
struct VTile {
    i4 v[CH];
};
template <bool STREAM, class T>
__device__ __forceinline__ T load_kv(const uint8_t* p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
    return *reinterpret_cast<const T*>(p);
}
// kr: record of page (lane % 16) / 4, vr: of page lane / 16.
template <int CH, bool STREAM>
__device__ __forceinline__ void load_k(KTile<CH>& x, const uint8_t* kr, const uint8_t* vr, int lane) {
    const int g = lane >> 4;
    const uint8_t* at = kr + (g * 4 + (lane & 3)) * 16;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int j = 0; j < (CH + 3) / 4; j++)
            if (4 * j + 3 < CH || 4 * j + g < CH) x.k[t][j] = load_kv<STREAM, i4>(at + (t * CH + 4 * j) * 64);
    x.ks = load_kv<STREAM, float>(vr + 512 * CH + (lane & 15) * 4);
    x.vs = load_kv<STREAM, float>(vr + 512 * CH + 64 + (lane & 15) * 4);
}
template <int CH, bool STREAM>
__device__ __forceinline__ void load_v(VTile<CH>& x, const uint8_t* vr, int lane) {
    const uint8_t* at = vr + 256 * CH + (lane & 15) * 16;
#pragma unroll
    for (int t = 0; t < CH; t++) x.v[t] = load_kv<STREAM, i4>(at + t * 256);
}

// Lane n of each 16 lanes' x, in all 16 (row_newbcast).
template <int N>
__device__ __forceinline__ float of_token(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 | N, 0xF, 0xF, true));
}
// f(token 0), .. f(token 15), the number a template argument.
template <int N = 0, class F>
__device__ __forceinline__ void each_token(F f) {
    f(std::integral_constant<int, N>());
    if constexpr (N < 15) each_token<N + 1>(f);
}

// The sum of products with a number's digits, in units of 256: x2 with the third
// digit's, x1 with the second's and the first's, this rounded to a whole unit (its
// sum began at 128 and was shifted down; half a unit is 2^-16 of the number's
// largest value times one code, beside a sum over 64 codes).
__device__ __forceinline__ int joined(int x2, int x1) { return (int)(((uint32_t)x2 << 8) + (uint32_t)x1); }

// Scores of a tile before the query's factor, s[t][r] of the lane's column and
// token 4t + r of page lane / 16; -infinity past the first `keys` of the page's
// tokens (whatever bits their slots hold).  The column's largest comes back.
template <int CH>
__device__ __forceinline__ float scores(f4 (&s)[4], const KTile<CH>& x, const Query<(CH + 3) / 4>& q, int keys) {
    constexpr int NC = (CH + 3) / 4;
    // (a score before the query's factor stays in fp32's range; a token with a scale
    // that is not finite gives NaN by its score)
    const float ks = fabsf(x.ks) + fabsf(x.vs) < INFINITY ? x.ks * UNIT : __uint_as_float(0x7fc00000u);
    i4 x2[4], x1[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        x2[t] = i4{0, 0, 0, 0}, x1[t] = i4{128, 128, 128, 128};
#pragma unroll
        for (int j = 0; j < NC; j++) x1[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.k[t][j], q.d[j][0], x1[t], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < 4; t++) {
#pragma unroll
        for (int j = 0; j < NC; j++) x2[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.k[t][j], q.d[j][2], x2[t], 0, 0, 0);
        x1[t] >>= 8;
#pragma unroll
        for (int j = 0; j < NC; j++) x1[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.k[t][j], q.d[j][1], x1[t], 0, 0, 0);
    }
    each_token([&](auto n) {
        constexpr int t = n / 4, r = n % 4;
        s[t][r] = (float)joined(x2[t][r], x1[t][r]) * of_token<n>(ks);
    });
    // few tiles have hidden keys: a sequence's last, those on a chunk's diagonal
    if (__builtin_amdgcn_ballot_w64(keys < 16))
        each_token([&](auto n) { s[n / 4][n % 4] = n < keys ? s[n / 4][n % 4] : -INFINITY; });
    float top = -INFINITY;
    each_token([&](auto n) { top = fmaxf(top, s[n / 4][n % 4]); });
    return column_max(top);
}

// The weights' three digits, from the scores and the V scales.  (A scale there that is
// not finite is a hidden slot's, or its token's score is NaN.)  H: tiles that
// share a maximum and a unit, so that their products are added up as integers: what
// takes an output's integers to fp32 (five operations) is then paid once for them.
template <int H>
struct Weights {
    i4 d[H][3];
    float unit;  // what the new integers are multiplied by
};
template <int CH, int H>
__device__ __forceinline__ Weights<H> weigh(State<CH>& st, f4 (&s)[H][4], float top, float scale, const float (&scales)[H]) {
    const float base = top == -INFINITY ? 0.0f : top * scale;  // no key (or only NaN ones) in the tiles
    // base is rounded and s * scale below is not: they differ by up to 2^-24 of base at the
    // maximum itself.  A small difference is the tiles' common factor (m carries it), a large
    // one would leave exp2's range: past 2^26 both are brought down to it, by a power of two.
    // (Scores that far are 2^-24 of themselves exact at best, so two that differ are then
    // still 4 apart, and those that are clearly less keep no weight.)
    const int down = min(26 - __builtin_amdgcn_frexp_expf(base), 0);
    const float near = __builtin_amdgcn_ldexpf(scale, down), shift = __builtin_amdgcn_ldexpf(base, down);
    float sum = 0.0f, big = 0.0f;
#pragma unroll
    for (int h = 0; h < H; h++) {
        const float vs = fabsf(scales[h]) < INFINITY ? scales[h] : 0.0f;
        each_token([&](auto n) {
            constexpr int t = n / 4, r = n % 4;
            const float p = exp2_fast(fmaf(s[h][t][r], near, -shift));
            sum += p;
            s[h][t][r] = p * of_token<n>(vs);
            big = fmaxf(big, s[h][t][r]);
        });
    }
    big = column_max(big);
    const float inv = big >= LEAST ? FIXED * __builtin_amdgcn_rcpf(big) : 0.0f;
    Weights<H> x;
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
        for (int t = 0; t < 4; t++) {
            int d0, d1, d2;
            digits(fmaf(s[h][t][0], inv, BIAS), fmaf(s[h][t][1], inv, BIAS), fmaf(s[h][t][2], inv, BIAS),
                   fmaf(s[h][t][3], inv, BIAS), d0, d1, d2);
            x.d[h][0][t] = d0, x.d[h][1][t] = d1, x.d[h][2][t] = d2;
        }
    const float m = top == -INFINITY ? top : base, m_new = fmaxf(st.m, m);
    const float f = scale_of(m, m_new), alpha = scale_of(st.m, m_new);
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {  // a column's maximum grew
#pragma unroll
        for (int t = 0; t < CH; t++) st.o[t] *= alpha;
        st.l *= alpha;
    }
    st.l += m == -INFINITY ? sum : sum * f;  // (a NaN stays)
    st.m = m_new;
    x.unit = (big >= LEAST ? big : 0.0f) * (256.0f / FIXED) * f;
    return x;
}

template <int CH, int H>
__device__ __forceinline__ void add_values(State<CH>& st, const VTile<CH> (&x)[H], const Weights<H>& w) {
#pragma unroll
    for (int t = 0; t < CH; t++) {
        i4 x2 = {0, 0, 0, 0}, x1 = {128, 128, 128, 128};
#pragma unroll
        for (int h = 0; h < H; h++) x1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[h].v[t], w.d[h][0], x1, 0, 0, 0);
#pragma unroll
        for (int h = 0; h < H; h++) x2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[h].v[t], w.d[h][2], x2, 0, 0, 0);
        x1 >>= 8;
#pragma unroll
        for (int h = 0; h < H; h++) x1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[h].v[t], w.d[h][1], x1, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; r++) st.o[t][r] = fmaf((float)joined(x2[r], x1[r]), w.unit, st.o[t][r]);
    }
}

template <int CH>
__device__ __forceinline__ KTile<CH> no_k() {  // (a lane without a last run of its own keeps zeros there)
    KTile<CH> k;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int j = 0; j < (CH + 3) / 4; j++) k.k[t][j] = i4{0, 0, 0, 0};
    return k;
}
// The record of a table entry's page; page 0's of one outside the pool, whose keys
// seen_on hides (and counts, once for each page and wave).
__device__ __forceinline__ const uint8_t* record(const KvQ8& c, const uint8_t* base, int id) {
    // (records are whole multiples of 128 bytes, their places below 2^39)
    return base + ((uint64_t)(((unsigned)id < (unsigned)c.num_pages ? id : 0) * (uint32_t)(c.page_stride >> 7)) << 7);
}
__device__ __forceinline__ int seen_on(const KvQ8& c, int id, int keys, int lane) {
    if ((unsigned)id < (unsigned)c.num_pages) return keys;
    if (keys > 0 && (lane & 15) == 15) atomicAdd(c.bad_pages, 1);
    return 0;
}

}  // namespace
}  // namespace nitro
