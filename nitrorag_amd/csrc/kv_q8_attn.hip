// Attention over an 8-bit paged cache on gfx950 (layout: kv_q8.hpp): decode (one
// token per sequence) and causal prefill.
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
// joins the running (max, sum, output) in fp32.  Error: Q is off by at most half
// a unit of 2^-23 of the row's largest entry, w by half a unit of 2^-23 of the
// tile's largest weight; the sums of products themselves are exact.
//
// Operand order.  A wave's tile is four pages.  For its keys as the product's
// rows, row m of product t (t = 0..3) is page m / 4, token 4t + m % 4; the result
// then leaves lane (g = lane / 16, column) with the 16 tokens of page g in token
// order, which is what the second product wants as its operand: the weights never
// leave their lane.  V columns come as 16 bytes = 16 tokens of one page.
#include <hip/hip_runtime.h>

#include "device_pool.hpp"
#include "kv_q8.hpp"

namespace nitro {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr float FIXED = 8355000.0f;  // below 127 * 65536 + 127 * 256 + 127, the largest three digits hold
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

// Digits of four 24-bit integers, digit n of each in the bytes of d[n]
// (v = 65536 d2 + 256 d1 + d0, each in [-128, 127]).
__device__ __forceinline__ void digits(int v0, int v1, int v2, int v3, int& d0, int& d1, int& d2) {
    const uint32_t x0 = (uint32_t)(v0 + 0x8080) ^ 0x8080u, x1 = (uint32_t)(v1 + 0x8080) ^ 0x8080u;
    const uint32_t x2 = (uint32_t)(v2 + 0x8080) ^ 0x8080u, x3 = (uint32_t)(v3 + 0x8080) ^ 0x8080u;
    const uint32_t a = __builtin_amdgcn_perm(x1, x0, 0x05010400u), b = __builtin_amdgcn_perm(x3, x2, 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(x1, x0, 0x0c0c0602u), d = __builtin_amdgcn_perm(x3, x2, 0x0c0c0602u);
    d0 = (int)__builtin_amdgcn_perm(b, a, 0x05040100u);
    d1 = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
    d2 = (int)__builtin_amdgcn_perm(d, c, 0x05040100u);
}

// A lane's query operand (column lane % 16, dimensions 16 * (4j + lane / 16) ..
// + 16 of step j): three digits, and what a score's integer is multiplied by.
template <int NC>
struct Query {
    i4 d[NC][3];
    float scale;
};

// row: the column's query row, nullptr for a column without one.
template <int NC>
__device__ __forceinline__ Query<NC> load_query(const float* row, int hd, float qscale, int g) {
    f4 x[NC][4];
    float top = 0.0f, bad = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int dim = 16 * (4 * j + g) + 4 * i;
            x[j][i] = f4{0.f, 0.f, 0.f, 0.f};
            if (row && dim < hd) x[j][i] = *reinterpret_cast<const f4*>(row + dim);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                top = fmaxf(top, fabsf(x[j][i][e]));
                bad = fmaf(x[j][i][e], 0.0f, bad);
            }
        }
    top = column_max(top);
    bad = column_sum(bad);  // NaN where the row holds an infinity or a NaN
    const float inv = top >= 0x1p-100f ? FIXED / top : 0.0f;
    Query<NC> q;
    q.scale = (top >= 0x1p-100f ? top : 0.0f) * (qscale / FIXED) + bad;
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            int v[4], d0, d1, d2;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = (int)rintf(x[j][i][e] * inv);
            digits(v[0], v[1], v[2], v[3], d0, d1, d2);
            q.d[j][0][i] = d0, q.d[j][1][i] = d1, q.d[j][2][i] = d2;
        }
    return q;
}

// What a wave carries from tile to tile: per lane, of its column, the maximum, its
// own sixteenth.. of the sum, and output dimensions 16t + 4 * (lane / 16) .. + 4.
template <int NC>
struct State {
    float m = -INFINITY, l = 0.0f;
    f4 o[4 * NC];
};

// One tile of 64 keys.  kr / vr: the records of this lane's K page ((lane % 16) /
// 4) and V page (lane / 16); keys: how many of the V page's tokens this column
// sees (0 where the page id is bad; less than 1: none).
template <int NC>
__device__ __forceinline__ void attend(State<NC>& st, const Query<NC>& q, const uint8_t* __restrict__ kr,
                                       const uint8_t* __restrict__ vr, int keys, int hdp, int lane) {
    const int g = lane >> 4, chunks = hdp >> 4;
    i4 k[4][NC];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int c = 4 * j + g;
            k[t][j] = i4{0, 0, 0, 0};
            if (c < chunks) k[t][j] = *reinterpret_cast<const i4*>(kr + ((t * chunks + c) * 4 + (lane & 3)) * 16);
        }
    f4 ks[4], vs[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        ks[t] = *reinterpret_cast<const f4*>(vr + 32 * hdp + 16 * t);
        vs[t] = *reinterpret_cast<const f4*>(vr + 32 * hdp + 64 + 16 * t);
    }
    i4 v[4 * NC];
#pragma unroll
    for (int t = 0; t < 4 * NC; t++)
        if (t < chunks) v[t] = *reinterpret_cast<const i4*>(vr + 16 * hdp + (t * 16 + (lane & 15)) * 16);

    f4 s[4];
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        i4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NC; j++) hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][j], q.d[j][2], hi, 0, 0, 0);
        hi <<= 8;
#pragma unroll
        for (int j = 0; j < NC; j++) hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][j], q.d[j][1], hi, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < NC; j++) lo = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][j], q.d[j][0], lo, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float x = fmaf((float)hi[r], 256.0f, (float)lo[r]) * (ks[t][r] * q.scale);
            s[t][r] = 4 * t + r < keys ? x : -INFINITY;
            top = fmaxf(top, s[t][r]);
        }
    }
    top = column_max(top);
    const float base = top == -INFINITY ? 0.0f : top;  // no key (or only NaN ones) in the tile
    float sum = 0.0f, big = 0.0f;
    f4 w[4];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float p = exp2_fast(s[t][r] - base);
            sum += p;
            // a slot past the last key may hold any bits: its weight is 0, not 0 * scale
            w[t][r] = 4 * t + r < keys ? p * vs[t][r] : 0.0f;
            big = fmaxf(big, w[t][r]);
        }
    big = column_max(big);
    const float inv = big >= LEAST ? FIXED * __builtin_amdgcn_rcpf(big) : 0.0f;
    i4 d[3];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        int x[4], d0, d1, d2;
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] = (int)fmaf(w[t][r], inv, 0.5f);
        digits(x[0], x[1], x[2], x[3], d0, d1, d2);
        d[0][t] = d0, d[1][t] = d1, d[2][t] = d2;
    }
    const float m_new = fmaxf(st.m, top);
    const float alpha = scale_of(st.m, m_new), f = scale_of(top, m_new);
    st.l = fmaf(st.l, alpha, top == -INFINITY ? sum : sum * f);  // (a NaN stays)
    st.m = m_new;
    const float fo = (big >= LEAST ? big : 0.0f) * (1.0f / FIXED) * f, fh = fo * 256.0f;
#pragma unroll
    for (int t = 0; t < 4 * NC; t++)
        if (t < chunks) {
            i4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
            hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[t], d[2], hi, 0, 0, 0);
            hi <<= 8;
            hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[t], d[1], hi, 0, 0, 0);
            lo = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[t], d[0], lo, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; r++)
                st.o[t][r] = fmaf(st.o[t][r], alpha, fmaf((float)hi[r], fh, (float)lo[r] * fo));
        }
}

// Device-coherent accesses of the partials and counters: relaxed atomics at agent
// scope, written through to and read from where the XCDs' caches agree.
__device__ __forceinline__ void store_coherent(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_coherent(const float* p) {
    return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Joins (M, L, A) with another part's.
__device__ __forceinline__ void join(float& M, float& L, float& A, float m, float l, float a) {
    const float mm = fmaxf(M, m), f = scale_of(M, mm), fs = scale_of(m, mm);
    L = L * f + (m == -INFINITY ? l : l * fs);  // a part without a finite maximum has l = 0 or NaN
    A = A * f + a * fs;
    M = mm;
}

// out = A / L; 0 where no key was seen.
__device__ __forceinline__ float divided(float A, float L) { return L == 0.0f ? 0.0f : A / L; }

template <int NC>
__global__ __launch_bounds__(256) void kv_q8_decode_kernel(KvQ8Decode a) {
    extern __shared__ float s_part[];  // [waves][columns][pstride]
    __shared__ int s_last;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int kv_mul = a.n_heads / a.c.kv_heads;
    const int groups = (kv_mul + KV_Q8_COLUMNS - 1) / KV_Q8_COLUMNS;
    int w = blockIdx.x;
    const int hg = w % groups;
    w /= groups;
    const int kv_h = w % a.c.kv_heads;
    w /= a.c.kv_heads;
    const int split = w % a.num_splits, b = w / a.num_splits;
    const int h0 = kv_h * kv_mul + hg * KV_Q8_COLUMNS;  // first query head
    const int cols = min(KV_Q8_COLUMNS, kv_mul - hg * KV_Q8_COLUMNS);
    const int hd = a.c.head_dim;

    const int ctx = max(0, min(a.positions[b] + 1, a.ctx_limit));
    const int tiles = (ctx + KV_Q8_TILE - 1) / KV_Q8_TILE;
    const int parts = max(1, (tiles + a.tiles_per_split - 1) / a.tiles_per_split);
    if (split >= parts) return;
    if (ctx == 0 && hg == 0 && kv_h == 0 && threadIdx.x == 0) atomicAdd(a.c.bad_pages, 1);  // a position below 0
    const int t0 = split * a.tiles_per_split, t1 = min(tiles, t0 + a.tiles_per_split);

    const int col = lane & 15, g = lane >> 4;
    const Query<NC> q =
        load_query<NC>(col < cols ? a.q + ((int64_t)b * a.n_heads + h0 + col) * hd : nullptr, hd, a.qscale, g);
    State<NC> st;
#pragma unroll
    for (int t = 0; t < 4 * NC; t++) st.o[t] = f4{0.f, 0.f, 0.f, 0.f};

    const int32_t* trow = a.tables + (int64_t)b * a.max_pages;
    const uint8_t* base = a.c.cache + a.c.layer_off + (int64_t)kv_h * a.c.record;
    const int last_page = max(0, (ctx - 1) >> 4);
    for (int t = t0 + wave; t < t1; t += a.waves) {
        int kp = trow[min(4 * t + (col >> 2), last_page)];
        int vp = trow[min(4 * t + g, last_page)];
        int keys = ctx - t * KV_Q8_TILE - 16 * g;
        if ((unsigned)kp >= (unsigned)a.c.num_pages) kp = 0;
        if ((unsigned)vp >= (unsigned)a.c.num_pages) {
            if (col == 0 && keys > 0) atomicAdd(a.c.bad_pages, 1);
            vp = 0;
            keys = 0;
        }
        attend<NC>(st, q, base + kp * a.c.page_stride, base + vp * a.c.page_stride, keys, a.c.hdp, lane);
    }

    // The waves' parts meet in LDS.
    st.l = column_sum(st.l);
    if (col < cols) {
        float* part = s_part + (wave * cols + col) * a.pstride;
#pragma unroll
        for (int t = 0; t < 4 * NC; t++) {
            const int dim = 16 * t + 4 * g;
            if (dim < hd) *reinterpret_cast<f4*>(part + dim) = st.o[t];
        }
        if (g == 0) {
            part[hd] = st.m;
            part[hd + 1] = st.l;
        }
    }
    __syncthreads();
    for (int o = threadIdx.x; o < cols * hd; o += blockDim.x) {
        const int c = o / hd, d = o - c * hd;
        float M = -INFINITY, L = 0.0f, A = 0.0f;
        for (int wv = 0; wv < a.waves; wv++) {
            const float* part = s_part + (wv * cols + c) * a.pstride;
            join(M, L, A, part[hd], part[hd + 1], part[d]);
        }
        if (parts == 1) {
            a.out[((int64_t)b * a.n_heads + h0 + c) * hd + d] = divided(A, L);
        } else {
            float* part = a.partials + (((int64_t)b * a.num_splits + split) * a.n_heads + h0 + c) * a.pstride;
            store_coherent(part + d, A);
            if (d == 0) {
                store_coherent(part + hd, M);
                store_coherent(part + hd + 1, L);
            }
        }
    }
    if (parts == 1) return;

    // The last workgroup of these heads to arrive joins the splits, in their order.
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's stores have arrived
    __syncthreads();
    if (threadIdx.x == 0) {
        int* counter = a.counters + ((int64_t)b * a.c.kv_heads + kv_h) * groups + hg;
        const int before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = before == parts - 1;
        if (s_last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!s_last) return;
    for (int o = threadIdx.x; o < cols * hd; o += blockDim.x) {
        const int c = o / hd, d = o - c * hd;
        float M = -INFINITY, L = 0.0f, A = 0.0f;
        for (int sp = 0; sp < parts; sp++) {
            const float* part = a.partials + (((int64_t)b * a.num_splits + sp) * a.n_heads + h0 + c) * a.pstride;
            join(M, L, A, load_coherent(part + hd), load_coherent(part + hd + 1), load_coherent(part + d));
        }
        a.out[((int64_t)b * a.n_heads + h0 + c) * hd + d] = divided(A, L);
    }
}

// A wave takes 16 query rows of one head as its columns; the workgroup's waves
// take consecutive ones and read the same K/V at about the same time.
template <int NC>
__global__ __launch_bounds__(256) void kv_q8_prefill_kernel(KvQ8Prefill a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = blockIdx.x % a.n_heads, item = blockIdx.x / a.n_heads;
    const int b = a.work[2 * item];
    const PrefillSeq seq = a.seqs[b];
    const int col = lane & 15, g = lane >> 4, hd = a.c.head_dim;
    const int first = a.work[2 * item + 1] + 16 * wave;  // of the wave's rows, in the chunk
    const int kv_h = h / (a.n_heads / a.c.kv_heads);
    const int32_t* trow = a.tables + (int64_t)b * a.max_pages;
    const uint8_t* base = a.c.cache + a.c.layer_off + (int64_t)kv_h * a.c.record;

    if (first >= seq.num_tokens) return;
    const bool in = first + col < seq.num_tokens;
    const int64_t row = (int64_t)seq.row_off + first + col;
    const int pos = seq.start_pos + first + col;
    const Query<NC> q = load_query<NC>(in ? a.q + (row * a.n_heads + h) * hd : nullptr, hd, a.qscale, g);
    State<NC> st;
#pragma unroll
    for (int t = 0; t < 4 * NC; t++) st.o[t] = f4{0.f, 0.f, 0.f, 0.f};
    const int last = seq.start_pos + min(first + 16, seq.num_tokens) - 1;  // the wave's last position
    for (int t = 0; t <= last / KV_Q8_TILE; t++) {
        int kp = trow[min(4 * t + (col >> 2), last >> 4)];
        int vp = trow[min(4 * t + g, last >> 4)];
        int keys = min(pos, last) + 1 - t * KV_Q8_TILE - 16 * g;
        if ((unsigned)kp >= (unsigned)a.c.num_pages) kp = 0;
        if ((unsigned)vp >= (unsigned)a.c.num_pages) {
            if (col == 0 && t * KV_Q8_TILE + 16 * g <= last) atomicAdd(a.c.bad_pages, 1);
            vp = 0;
            keys = 0;
        }
        attend<NC>(st, q, base + kp * a.c.page_stride, base + vp * a.c.page_stride, keys, a.c.hdp, lane);
    }
    const float l = column_sum(st.l);
    if (!in) return;
    float* out = a.out + (row * a.n_heads + h) * hd;
#pragma unroll
    for (int t = 0; t < 4 * NC; t++) {
        const int dim = 16 * t + 4 * g;
        if (dim < hd)
            *reinterpret_cast<f4*>(out + dim) = f4{divided(st.o[t][0], l), divided(st.o[t][1], l),
                                                   divided(st.o[t][2], l), divided(st.o[t][3], l)};
    }
}

}  // namespace

hipError_t launch_kv_q8_decode(const KvQ8Decode& a, hipStream_t stream) {
    const int kv_mul = a.n_heads / a.c.kv_heads;
    const int groups = (kv_mul + KV_Q8_COLUMNS - 1) / KV_Q8_COLUMNS;
    const int64_t blocks = (int64_t)a.batch * a.num_splits * a.c.kv_heads * groups;
    if (a.waves < 1 || a.waves > 4 || a.pstride < a.c.head_dim + 2 || a.pstride % 4 || a.c.hdp > 256 || blocks > INT32_MAX)
        return hipErrorInvalidValue;
    const size_t lds = sizeof(float) * a.waves * (kv_mul < KV_Q8_COLUMNS ? kv_mul : KV_Q8_COLUMNS) * a.pstride;
    const dim3 grid((unsigned)blocks), block(64 * a.waves);
    switch ((a.c.hdp + 63) / 64) {
        case 1: hipLaunchKernelGGL((kv_q8_decode_kernel<1>), grid, block, lds, stream, a); break;
        case 2: hipLaunchKernelGGL((kv_q8_decode_kernel<2>), grid, block, lds, stream, a); break;
        case 3: hipLaunchKernelGGL((kv_q8_decode_kernel<3>), grid, block, lds, stream, a); break;
        default: hipLaunchKernelGGL((kv_q8_decode_kernel<4>), grid, block, lds, stream, a); break;
    }
    return hipGetLastError();
}

hipError_t launch_kv_q8_prefill(const KvQ8Prefill& a, hipStream_t stream) {
    const int64_t blocks = (int64_t)a.work_items * a.n_heads;
    if (a.item_rows != 64 || a.c.hdp > 256 || blocks > INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid((unsigned)blocks), block(256);
    switch ((a.c.hdp + 63) / 64) {
        case 1: hipLaunchKernelGGL((kv_q8_prefill_kernel<1>), grid, block, 0, stream, a); break;
        case 2: hipLaunchKernelGGL((kv_q8_prefill_kernel<2>), grid, block, 0, stream, a); break;
        case 3: hipLaunchKernelGGL((kv_q8_prefill_kernel<3>), grid, block, 0, stream, a); break;
        default: hipLaunchKernelGGL((kv_q8_prefill_kernel<4>), grid, block, 0, stream, a); break;
    }
    return hipGetLastError();
}

}  // namespace nitro
