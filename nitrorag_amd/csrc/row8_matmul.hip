// Products of 8-bit rows with Q8_0 matrices for gfx950 (row8.hpp):
//   p[b][i] = xs[b] * sum_j ws[i][j] * (sum_t wq[i][32j + t] * xq[b][32j + t])
//   out[b][i] = act(p + bias[i]) [* (p' + bias'[i])] + residual[b][i]
// The inner sums are exact integers (at most 32 * 128 * 128: codes and weights may be -128)
// on the integer matrix cores, and exact in fp32 (24 bits); a block of 32 k has its weight
// scale, so each takes one conversion and one fma into fp32 sums.  The row's scale comes in
// once, at the end.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "nitro_paged_attn.h"
#include "q8_group.hpp"
#include "row8.hpp"

namespace nitro {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i16 __attribute__((ext_vector_type(16)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

// exp and the quotient by the hardware's 2^x and 1 / x: a few roundings of the result, and as
// many of the exponent's argument as that is large: its rounding moves 2^t by t of them, which
// expf does not let grow.  Past t = 126 the quotient may be 0 where the result is below 1e-35.
// (NaN goes through all of the activations; a quotient by an infinity is 0.)  They are a tile's
// whole time where n is small: 8192 rows of 768 x 2048 with gelu 49 us, 63 through erfcf; 4637
// rows of 32 x 5522 31 us, with gelu_tanh 34, gelu 38, and 51 and 52 through expf, erfcf and
// divisions.
__device__ __forceinline__ float logistic_of(float x, float t) {  // x / (1 + 2^t)
    return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t));
}
__device__ __forceinline__ float relu(float x) { return x < 0.0f ? 0.0f : x; }
__device__ __forceinline__ float silu(float x) { return logistic_of(x, x * -1.4426950408889634f); }
// x Phi(x), with Phi(-|x|) = exp(-x^2 / 2) t Q(t), t = 1 / (1 + 0.35 |x|): Q is a polynomial of
// degree 8, fitted in 64 bits by least squares, its weights raised where the relative error was
// largest until that stayed below 3.2e-8 for |x| <= 14.5 (where Phi(-|x|) leaves fp32); 5.4e-8,
// a rounding, with the coefficients in fp32.  The whole is off by at most 7 (1 + x^2) roundings.
__device__ __forceinline__ float gelu(float x) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, fabsf(x), 1.0f));
    float q = -0.029157886f;
    q = fmaf(q, t, 0.14403091f);
    q = fmaf(q, t, -0.25583899f);
    q = fmaf(q, t, 0.1593197f);
    q = fmaf(q, t, -0.023212353f);
    q = fmaf(q, t, 0.1055525f);
    q = fmaf(q, t, 0.11982129f);
    q = fmaf(q, t, 0.13986352f);
    q = fmaf(q, t, 0.1396213f);
    const float below = q * t * __builtin_amdgcn_exp2f(x * x * -0.72134752f);
    return x * (x < 0.0f ? below : 1.0f - below);
}
// 0.5 x (1 + tanh(u)) = x / (1 + exp(-2u)), u = sqrt(2 / pi) (x + 0.044715 x^3)
__device__ __forceinline__ float gelu_tanh(float x) {
    return logistic_of(x, x * fmaf(x * x, -0.10294324f, -2.3022082f));
}
__device__ __forceinline__ float activate(float x, int activation) {
    switch (activation) {
        case NITRO_ACT_RELU: return relu(x);
        case NITRO_ACT_SILU: return silu(x);
        case NITRO_ACT_GELU: return gelu(x);
        case NITRO_ACT_GELU_TANH: return gelu_tanh(x);
        default: return x;
    }
}

// The member that column tile ct of `cols` columns each belongs to, and ct within it.
__device__ __forceinline__ int member_of(const Row8Matmul& a, int& ct, int cols) {
    int m = 0;
    if (!a.gated)
        for (; m + 1 < a.mats; m++) {
            const int tiles = (a.d[m] + cols - 1) / cols;
            if (ct < tiles) break;
            ct -= tiles;
        }
    return m;
}

// A launch's output tiles, and which of the two orders of them the XCDs share out: each
// takes an eighth, of the rows' panels (every column tile of one after the other) or of the
// columns', whichever brings less into its L2.  (512 rows of 4096 x 4096 as panels of rows:
// every L2 reads the whole matrix, 161 MB of misses where the matrix has 19.)  A single panel
// of rows is taken as it comes: there is nothing to share, and neighbouring tiles on different
// XCDs read faster (one row of 11008 x 4096: 10.1 against 11.3 us).
struct Tiles {
    int rows, cols;
    bool by_columns;
};
struct Place {
    int row, col;
};
__device__ __forceinline__ Place place_of(const Tiles& t) {
    if (t.rows == 1) return {0, (int)blockIdx.x};
    const int wg = blockIdx.x, total = gridDim.x, per = total >> 3, rem = total & 7, xcd = wg & 7;
    const int i = xcd * per + min(xcd, rem) + (wg >> 3);
    if (t.by_columns) return {i % t.rows, i / t.rows};
    return {i / t.cols, i % t.cols};
}

// ---------------------------------------------------------- split over waves
// A workgroup owns RT x CT tiles of U batch rows x U weight rows (U = 16 or 32, the matrix
// instruction's); its W waves split the blocks, each with sums of its own, which are
// added through LDS in wave order.  No wave waits for another before that.
//  - weights: straight from memory in operand order, 512 bytes a load;
//  - x: 128 bytes of a row at a time (eight lanes to a row) into a region of LDS of the
//    wave's own, and back in operand order.  (Loaded in operand order, 16 rows to a load,
//    every eight bytes were a lookup of their own in the vector cache: 128 rows of 4096 x
//    4096 23 us, 14 us so; 16 rows of 4096 x 11008 17 us, 11 us so.)
// Bound by the weights' bytes for few rows (8 rows of a gated 4096 x 11008 pair 23 us, 4.4
// TB/s, where the loads alone take 18), by latency for small matrices (16 rows of 768 x 2048
// 3.1 us; one of 4096 x 4096 5.7, 3.3 TB/s), and from 32 rows on by its loads' latency and
// the vector unit together (64 rows of the pair 36 us, 128 of 4096 x 4096 13 us).
template <int U>
struct Tile;
template <>
struct Tile<16> {
    typedef long Operand;
    static constexpr int SUMS = 4, MASK = 15;
    typedef f4 Sums;
    // Row (x) or column (weights) lane % 16, k = 8 * (lane / 16) .. + 8.
    static __device__ __forceinline__ Operand x(const int8_t* row, int lane) {
        return *reinterpret_cast<const long*>(row + 8 * (lane >> 4));
    }
    static __device__ __forceinline__ Operand w(const uint8_t* record, int lane) {
        return *reinterpret_cast<const long*>(record + 64 + 8 * lane);
    }
    static __device__ __forceinline__ void multiply(Operand x, Operand w, int (&p)[SUMS]) {
        const i4 r = __builtin_amdgcn_mfma_i32_16x16x32_i8(x, w, i4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < SUMS; i++) p[i] = r[i];
    }
    // Where the sum of (row, column) lies: its place among a lane's, and the lane.
    static __device__ __forceinline__ int sum_at(int row) { return row % 4; }
    static __device__ __forceinline__ int lane_at(int row, int col) { return row / 4 * 16 + col; }
};
template <>
struct Tile<32> {
    typedef i4 Operand;
    static constexpr int SUMS = 16, MASK = 31;
    typedef f16v Sums;
    // Row or column lane % 32, k = 16 * (lane / 32) .. + 16.
    static __device__ __forceinline__ Operand x(const int8_t* row, int lane) {
        return *reinterpret_cast<const i4*>(row + 16 * (lane >> 5));
    }
    static __device__ __forceinline__ Operand w(const uint8_t* record, int lane) {
        const uint8_t* p = record + 64 + 256 * (lane >> 5) + 8 * (lane & 15);
        const int2 lo = *reinterpret_cast<const int2*>(p), hi = *reinterpret_cast<const int2*>(p + 128);
        return i4{lo.x, lo.y, hi.x, hi.y};
    }
    static __device__ __forceinline__ void multiply(Operand x, Operand w, int (&p)[SUMS]) {
        i16 zero;
#pragma unroll
        for (int i = 0; i < 16; i++) zero[i] = 0;
        const i16 r = __builtin_amdgcn_mfma_i32_32x32x32_i8(x, w, zero, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < SUMS; i++) p[i] = r[i];
    }
    static __device__ __forceinline__ int sum_at(int row) { return row / 8 * 4 + row % 4; }
    static __device__ __forceinline__ int lane_at(int row, int col) { return row / 4 % 2 * 32 + col; }
};

// X: rows of x that are loaded, all of the tile's or 8 (for up to 8 rows; the tile's others are
// the same again and go nowhere: one row of 4096 x 11008 10.1 us, 10.5 with all 16 loaded; 8 rows
// of 11008 x 4096 10.5, 11.1).
template <int U, int RT, int CT, int W, int OCC, int X, bool GATED>
__global__ __launch_bounds__(64 * W, OCC) void row8_split_kernel(Row8Matmul a, Tiles tiling) {
    typedef Tile<U> T;
    constexpr int ROWS = U * RT, COLS = U * CT / (GATED ? 2 : 1);  // of the output
    constexpr int ROUND = 4, PITCH = ROUND * Q8_BLOCK + 16;  // blocks a round; bytes of a row in LDS
    constexpr int LOADS = X / 8;                             // of 8 rows of x
    constexpr int PART = RT * CT * T::SUMS * 64, XBYTES = W * X * PITCH, SBYTES = W * PART * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[XBYTES > SBYTES ? XBYTES : SBYTES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Place place = place_of(tiling);
    int ct = place.col;
    const int member = member_of(a, ct, COLS);
    const int d = a.d[member], n = a.n, nb = n / Q8_BLOCK, tiles = (d + 15) / 16;
    const int b0 = place.row * ROWS;

    // Weight tiles of 16 rows, the last one for those past the end; with a gate, tile 2t is
    // the gate's and 2t + 1 the other matrix's.
    const uint8_t* w[CT];
#pragma unroll
    for (int t = 0; t < CT; t++) {
        const int tile = min((ct * COLS + U * (GATED ? t / 2 : t) + (lane & T::MASK)) / 16, tiles - 1);
        w[t] = a.w[GATED ? t % 2 : member] + (size_t)tile * nb * Q8_TILE_BYTES;
    }
    const int8_t* x[LOADS];
    const int xk = lane % 8 * 16;
#pragma unroll
    for (int r = 0; r < LOADS; r++) x[r] = a.codes + (size_t)min(b0 + 8 * r + lane / 8, a.rows - 1) * n;
    int8_t* const mine = reinterpret_cast<int8_t*>(lds) + wave * X * PITCH;

    typename T::Sums acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int t = 0; t < CT; t++)
#pragma unroll
            for (int i = 0; i < T::SUMS; i++) acc[r][t][i] = 0.0f;

    // Rounds first .. end, the next round's loads ahead of this one's use.  A block past
    // the end repeats the last one, times 0.
    const int rounds = (nb + ROUND - 1) / ROUND;
    const int first = (int)((int64_t)rounds * wave / W), end = (int)((int64_t)rounds * (wave + 1) / W);
    struct Weights {
        typename T::Operand q[ROUND][CT];
        float s[ROUND][CT];
    } wa, wb;
    i4 xn[LOADS];
    auto load = [&](Weights& R, int round) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < LOADS; r++)
            xn[r] = *reinterpret_cast<const i4*>(x[r] + min(round * (ROUND * Q8_BLOCK) + xk, n - 16));
#pragma unroll
        for (int u = 0; u < ROUND; u++) {
            const int k = min(round * ROUND + u, nb - 1);
#pragma unroll
            for (int t = 0; t < CT; t++) {
                const uint8_t* record = w[t] + (size_t)k * Q8_TILE_BYTES;
                R.q[u][t] = T::w(record, lane);
                R.s[u][t] = *reinterpret_cast<const float*>(record + 4 * (lane & 15));
            }
        }
    };
    // Lanes read what other lanes of the wave wrote, and write where others read: no
    // access may pass another between them.
    auto exchange = []() __attribute__((always_inline)) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    auto use = [&](const Weights& R, Weights& next, int round) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < LOADS; r++) *reinterpret_cast<i4*>(mine + (8 * r + lane / 8) * PITCH + xk) = xn[r];
        exchange();
        load(next, round + 1);
#pragma unroll
        for (int u = 0; u < ROUND; u++) {
            typename T::Operand xq[RT];
#pragma unroll
            for (int r = 0; r < RT; r++) xq[r] = T::x(mine + (U * r + (lane & T::MASK)) % X * PITCH + u * Q8_BLOCK, lane);
#pragma unroll
            for (int t = 0; t < CT; t++) {
                const float s = round * ROUND + u < nb ? R.s[u][t] : 0.0f;
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    int p[T::SUMS];
                    T::multiply(xq[r], R.q[u][t], p);
#pragma unroll
                    for (int i = 0; i < T::SUMS; i++) acc[r][t][i] = fmaf(s, (float)p[i], acc[r][t][i]);
                }
            }
        }
        exchange();
    };
    if (first < end) {
        load(wa, first);
#pragma unroll 1
        for (int round = first; round < end; round += 2) {
            use(wa, wb, round);
            if (round + 1 < end) use(wb, wa, round + 1);
        }
    }
    // What a thread's outputs need besides the sums, loaded while those are joined.  (Loaded for
    // each output by itself, 64 rows of 4096 x 4096 with a residual took 10.6 us, 9.3 so.)
    constexpr int OUTS = (ROWS * COLS + 64 * W - 1) / (64 * W);
    float xs[OUTS], bias[OUTS], second[OUTS], residual[OUTS];
#pragma unroll
    for (int k = 0; k < OUTS; k++) {
        const int e = threadIdx.x + k * 64 * W, b = min(b0 + e / COLS, a.rows - 1), i = min(ct * COLS + e % COLS, d - 1);
        xs[k] = a.scales[b];
        bias[k] = a.bias ? a.bias[i] : 0.0f;
        second[k] = GATED && a.bias ? a.bias[d + i] : 0.0f;
        residual[k] = a.residual ? a.residual[(size_t)b * d + i] : 0.0f;
    }
    float* const parts = reinterpret_cast<float*>(lds);  // [wave][tile][sum][lane]
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int t = 0; t < CT; t++)
#pragma unroll
            for (int i = 0; i < T::SUMS; i++) parts[wave * PART + ((r * CT + t) * T::SUMS + i) * 64 + lane] = acc[r][t][i];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < OUTS; k++) {
        const int e = threadIdx.x + k * 64 * W, row = e / COLS, col = e % COLS;
        const int tile = row / U * CT + (GATED ? col / U * 2 : col / U);
        const int at = (tile * T::SUMS + T::sum_at(row % U)) * 64 + T::lane_at(row % U, col % U);
        const int b = b0 + row, i = ct * COLS + col;
        if (row >= ROWS || b >= a.rows || i >= d) continue;
        float s = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int v = 0; v < W; v++) {
            s += parts[v * PART + at];
            if constexpr (GATED) s2 += parts[v * PART + at + T::SUMS * 64];
        }
        float y = activate(s * xs[k] + bias[k], a.activation);
        if constexpr (GATED) y *= s2 * xs[k] + second[k];
        a.out[member][(size_t)b * d + i] = y + residual[k];
    }
}

// --------------------------------------------------------------- many rows
// A workgroup of 4 waves owns 64 MT batch rows x 64 NT weight rows (wave: half of each, as
// MT x NT tiles of v_mfma_i32_32x32x32_i8: lane l holds 16 k, half l / 32 of a block, of
// row l % 32).  STEP blocks of x and of the weights lie in LDS, in two buffers with a barrier
// for each, and are loaded DEPTH steps before they are put there.  x lies as 2 STEP planes
// (the blocks' halves) of 16 bytes a row, so that lanes read consecutive rows; the weights as
// in the tile layout, runs of 8 k.
// Bound by the vector unit: a product's 16 sums a lane take 16 conversions and 16 fma, 64 + 64
// cycles of a SIMD, next to the matrix instruction's 32.  4096 rows of 11008 x 4096: 390 to 425
// us, 870 to 950 TFLOP/s, with the vector unit busy for 86 to 89% of the cycles; 1024 rows of a gated
// 4096 x 11008 pair 215 to 230 us, 800 to 860.  (The codes as halves, whose sums need no
// conversion but two matrix instructions a block, took 387 us where this took 374 in the same run,
// with the two back to back and the fma behind them: 148 cycles of a SIMD for a tile and block, of
// which either unit has work for 64.  Other orders of them were not measured.)  512 rows of
// 4096 x 4096, 32 us, 540 TFLOP/s: few workgroups a CU, and each waits for its loads.
template <int MT, int NT, int STEP, int DEPTH, int OCC, bool GATED>
__global__ __launch_bounds__(256, OCC) void row8_gemm_kernel(Row8Matmul a, Tiles tiling) {
    constexpr int BM = 64 * MT, BN = 64 * NT, COLS = GATED ? BN / 2 : BN;
    constexpr int PLANE = BM * 16 + 32;  // (the planes' banks lie 32 bytes apart: a row's four runs are written together)
    constexpr int XB = 2 * STEP * PLANE, WB = STEP * BN * 32, BUF = XB + WB + STEP * BN * 4;
    constexpr int XU = MT * STEP / 2, WU = NT * STEP / 2, SU = STEP * BN / 256;  // units a thread
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * BUF];
    __shared__ __attribute__((aligned(16))) float row_scales[BM];
    const int tid = threadIdx.x;
    auto xl = [&](int buf) __attribute__((always_inline)) { return lds + buf * BUF; };
    auto wl = [&](int buf) __attribute__((always_inline)) { return lds + buf * BUF + XB; };
    auto sl = [&](int buf) __attribute__((always_inline)) { return reinterpret_cast<float*>(lds + buf * BUF + XB + WB); };
    static_assert(!GATED || NT == 2, "a wave's two column tiles are the gate's and the other's");
    const int lane = tid & 63, wave = tid >> 6;
    const int wm = wave & 1, wn = wave >> 1, lc = lane & 31, lh = lane >> 5;

    const Place place = place_of(tiling);
    const int b0 = place.row * BM;
    int ct = place.col;
    const int member = member_of(a, ct, COLS);
    const int d = a.d[member], n = a.n, nb = n / Q8_BLOCK, tiles = (d + 15) / 16;

    // The 16-row weight tile at place j (of BN / 16) of the workgroup's.
    auto tile_at = [&](int j) __attribute__((always_inline)) {
        const int at = GATED ? ct * (COLS / 16) + j / 4 * 2 + j % 2 : ct * (COLS / 16) + j;
        return a.w[GATED ? j / 2 % 2 : member] + (size_t)min(at, tiles - 1) * nb * Q8_TILE_BYTES;
    };
    // Staging: x and weights in units of 16 bytes, scales one by one.
    static_assert(STEP * BN % 256 == 0, "every thread has its scales");
    const int8_t* xp[XU];
    int xdst[XU];
    const int xk = tid % (2 * STEP) * 16;
#pragma unroll
    for (int u = 0; u < XU; u++) {
        const int row = (tid + 256 * u) / (2 * STEP);
        xp[u] = a.codes + (size_t)min(b0 + row, a.rows - 1) * n;
        xdst[u] = tid % (2 * STEP) * PLANE + row * 16;
    }
    const uint8_t* wp[WU];
    int wblk[WU];
#pragma unroll
    for (int u = 0; u < WU; u++) {
        const int e = tid + 256 * u;
        wblk[u] = e / (2 * BN);
        wp[u] = tile_at(e / 32 % (BN / 16)) + 64 + e % 32 * 16;
    }
    const uint8_t* sp[SU];
    int sblk[SU];
#pragma unroll
    for (int u = 0; u < SU; u++) {
        const int e = tid + 256 * u;
        sblk[u] = e / BN;
        sp[u] = tile_at(e % BN / 16) + 4 * (e % 16);
    }

    struct Stage {
        i4 x[XU], w[WU];
        float s[SU];
    };
    auto load = [&](Stage& S, int blk) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < XU; u++)
            S.x[u] = *reinterpret_cast<const i4*>(xp[u] + min(blk * Q8_BLOCK + xk, n - 16));
#pragma unroll
        for (int u = 0; u < WU; u++)
            S.w[u] = *reinterpret_cast<const i4*>(wp[u] + (size_t)min(blk + wblk[u], nb - 1) * Q8_TILE_BYTES);
#pragma unroll
        for (int u = 0; u < SU; u++)
            S.s[u] = *reinterpret_cast<const float*>(sp[u] + (size_t)min(blk + sblk[u], nb - 1) * Q8_TILE_BYTES);
    };
    auto put = [&](const Stage& S, int buf, int blk) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < XU; u++) *reinterpret_cast<i4*>(xl(buf) + xdst[u]) = S.x[u];
#pragma unroll
        for (int u = 0; u < WU; u++) *reinterpret_cast<i4*>(wl(buf) + (tid + 256 * u) * 16) = S.w[u];
        // (a block past the end repeats the last one, times 0)
#pragma unroll
        for (int u = 0; u < SU; u++) sl(buf)[tid + 256 * u] = blk + sblk[u] < nb ? S.s[u] : 0.0f;
    };

    f16v acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[m][t][i] = 0.0f;

    // The products of one 32 x 32 tile and block, scaled in while the next tile's run.
    i16 late;
    float late_s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) late[i] = 0;
    auto scale_in = [&](f16v& to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 16; i++) to[i] = fmaf(late_s, (float)late[i], to[i]);
    };
    // A block's operands.  AHEAD: read while the block before is multiplied (larger tiles
    // have no registers for it, and more to do meanwhile).
    constexpr bool AHEAD = MT * NT <= 2;
    struct Operands {
        i4 x[MT], w[NT];
        float s[NT];
    };
    auto read = [&](Operands& o, int buf, int h) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int j = wn * 2 * NT + 2 * t + lc / 16;
            const uint8_t* p = wl(buf) + (h * (BN / 16) + j) * 512 + (2 * lh * 16 + lc % 16) * 8;
            const int2 lo = *reinterpret_cast<const int2*>(p), hi = *reinterpret_cast<const int2*>(p + 128);
            o.w[t] = i4{lo.x, lo.y, hi.x, hi.y};
            o.s[t] = sl(buf)[h * BN + wn * 32 * NT + 32 * t + lc];
        }
#pragma unroll
        for (int m = 0; m < MT; m++)
            o.x[m] = *reinterpret_cast<const i4*>(xl(buf) + (2 * h + lh) * PLANE + (wm * 32 * MT + 32 * m + lc) * 16);
    };
    auto compute = [&](int buf) __attribute__((always_inline)) {
        Operands o[AHEAD ? 2 : 1];
        if constexpr (AHEAD) read(o[0], buf, 0);
#pragma unroll
        for (int h = 0; h < STEP; h++) {
            Operands& now = o[AHEAD ? h % 2 : 0];
            if constexpr (!AHEAD) read(now, buf, h);
            else if (h + 1 < STEP) read(o[(h + 1) % 2], buf, h + 1);
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    i16 zero;
#pragma unroll
                    for (int i = 0; i < 16; i++) zero[i] = 0;
                    const i16 p = __builtin_amdgcn_mfma_i32_32x32x32_i8(now.x[m], now.w[t], zero, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    scale_in(m ? acc[m - 1][t] : t ? acc[MT - 1][t - 1] : acc[MT - 1][NT - 1]);
                    late = p, late_s = now.s[t];
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    };
    const int steps = (nb + STEP - 1) / STEP;
    auto step = [&](int i, Stage& S) __attribute__((always_inline)) {
        __syncthreads();  // step i is staged; the other buffer's readers are done
        put(S, (i + 1) & 1, STEP * (i + 1));
        load(S, STEP * (i + 1 + DEPTH));
        compute(i & 1);
    };
    // What the outputs need besides the sums and the residual comes ahead of the first step.
    // (4637 rows of 32 x 5522 with a bias 40 us when it came behind the last, 34.5 so.)
    const float row_scale = a.scales[min(b0 + tid % BM, a.rows - 1)];
    float bias[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int col = ct * COLS + (GATED ? wn * 32 : (wn * NT + t) * 32) + lc;
        bias[t] = a.bias ? a.bias[(GATED && t ? d : 0) + min(col, d - 1)] : 0.0f;
    }
    Stage sa, sb;
    load(sa, 0);
    if constexpr (DEPTH == 2) load(sb, STEP);
    if (tid < BM) row_scales[tid] = row_scale;
    put(sa, 0, 0);
    load(sa, STEP * DEPTH);
    if constexpr (DEPTH == 1) {
#pragma unroll 1
        for (int i = 0; i < steps; i++) step(i, sa);
    } else {
#pragma unroll 1
        for (int i = 0; i + 1 < steps; i += 2) {
            step(i, sb);
            step(i + 1, sa);
        }
        if (steps & 1) step(steps - 1, sb);
    }
    scale_in(acc[MT - 1][NT - 1]);

    // Lane l holds row 8 * (i / 4) + 4 * (l / 32) + i % 4, column l % 32 of a tile.
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int row0 = b0 + (wm * MT + m) * 32 + 4 * lh;
        float xs[16];
#pragma unroll
        for (int i = 0; i < 16; i++) xs[i] = row_scales[row0 - b0 + 8 * (i / 4) + i % 4];
#pragma unroll
        for (int t = 0; t < (GATED ? 1 : NT); t++) {
            const int col = ct * COLS + (GATED ? wn * 32 : (wn * NT + t) * 32) + lc, near = min(col, d - 1);
            float y[16], r[16];
            if (a.residual) {  // (all read before the first is written: it may be the output)
#pragma unroll
                for (int i = 0; i < 16; i++) r[i] = a.residual[(size_t)min(row0 + 8 * (i / 4) + i % 4, a.rows - 1) * d + near];
            }
#pragma unroll
            for (int i = 0; i < 16; i++) y[i] = acc[m][t][i] * xs[i] + bias[t];
            switch (a.activation) {
                case NITRO_ACT_RELU:
#pragma unroll
                    for (int i = 0; i < 16; i++) y[i] = relu(y[i]);
                    break;
                case NITRO_ACT_SILU:
#pragma unroll
                    for (int i = 0; i < 16; i++) y[i] = silu(y[i]);
                    break;
                case NITRO_ACT_GELU_TANH:
#pragma unroll
                    for (int i = 0; i < 16; i++) y[i] = gelu_tanh(y[i]);
                    break;
                case NITRO_ACT_GELU:
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        y[i] = gelu(y[i]);
                        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (four at a time: registers)
                    }
                    break;
                default: break;
            }
            if constexpr (GATED) {
#pragma unroll
                for (int i = 0; i < 16; i++) y[i] *= acc[m][1][i] * xs[i] + bias[1];
            }
            if (a.residual) {
#pragma unroll
                for (int i = 0; i < 16; i++) y[i] += r[i];
            }
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int b = row0 + 8 * (i / 4) + i % 4;
                if (b < a.rows && col < d) a.out[member][(size_t)b * d + col] = y[i];
            }
        }
    }
}

constexpr int log2_of(int x) { return x == 1 ? 0 : 1 + log2_of(x / 2); }
int tiles_over(int x, int log2) { return (int)(((int64_t)x + (1 << log2) - 1) >> log2); }

int col_tiles_of(const Row8Matmul& a, int log2) {
    int t = 0;
    for (int m = 0; m < (a.gated ? 1 : a.mats); m++) t += tiles_over(a.d[m], log2);
    return t;
}

// A kernel, its workgroup's tile, and what its time is estimated with: a wave's chain of
// steps (`blocks` blocks each, the blocks split over `split` waves), of which one takes
// `alone` us where few workgroups share a CU and `busy` us times their number where many
// do, at most `resident` at once; `fixed` us for a launch, a third of it again for every
// set of resident workgroups.
struct Form {
    int rows, cols, blocks, split;  // their logarithms to base 2 (a call looks at every form)
    int resident;
    float fixed, alone, busy;
    bool single, pairs;  // takes matrices one by one; takes gated pairs
    int threads;
    void (*launch)(const Row8Matmul&, const Tiles&, hipStream_t);
};

template <int U, int RT, int CT, int W, int OCC, bool GATED>
void launch_split(const Row8Matmul& a, const Tiles& t, hipStream_t stream) {
    const dim3 grid((unsigned)t.rows * (unsigned)t.cols), block(64 * W);
    if constexpr (U * RT == 16)
        if (a.rows <= 8) {
            hipLaunchKernelGGL((row8_split_kernel<U, RT, CT, W, OCC, 8, GATED>), grid, block, 0, stream, a, t);
            return;
        }
    hipLaunchKernelGGL((row8_split_kernel<U, RT, CT, W, OCC, U * RT, GATED>), grid, block, 0, stream, a, t);
}

// (A pair needs column tiles that are even in number.)
template <int U, int RT, int CT, int W, int OCC, bool SINGLE = true>
constexpr Form split_form(int resident, float fixed, float alone, float busy) {
    return {log2_of(U * RT), log2_of(U * CT), 2, log2_of(W), resident, fixed, alone, busy, SINGLE, CT % 2 == 0, 64 * W,
            [](const Row8Matmul& a, const Tiles& t, hipStream_t stream) {
                if constexpr (CT % 2 == 0)
                    if (a.gated) launch_split<U, RT, CT, W, OCC, true>(a, t, stream);
                if constexpr (SINGLE)
                    if (!a.gated) launch_split<U, RT, CT, W, OCC, false>(a, t, stream);
            }};
}

template <int MT, int NT, int STEP, int DEPTH, int OCC>
constexpr Form gemm_form(int resident, float fixed, float alone, float busy) {
    return {log2_of(64 * MT), log2_of(64 * NT), log2_of(STEP), 0, resident, fixed, alone, busy, true, NT == 2, 256,
            [](const Row8Matmul& a, const Tiles& t, hipStream_t stream) {
                const dim3 grid((unsigned)t.rows * (unsigned)t.cols), block(256);
                if constexpr (NT == 2)
                    if (a.gated)
                        hipLaunchKernelGGL((row8_gemm_kernel<MT, NT, STEP, DEPTH, OCC, true>), grid, block, 0, stream, a, t);
                if (!a.gated)
                    hipLaunchKernelGGL((row8_gemm_kernel<MT, NT, STEP, DEPTH, OCC, false>), grid, block, 0, stream, a, t);
            }};
}

// Each timed over 420 shapes (1 to 8192 rows, n from 32 to 16384, d from 16 to 16384, gated
// or not) as graph replays, and fitted to within 4 to 8% of its own times.  The choice by
// these estimates takes 1.2% longer in the mean than the best of the forms each time; at
// most 23%, 7.1 against 5.8 us, for 35 rows and a gated pair of 9588 x 32.  (Two of the forms are the
// least only for pairs.)
constexpr Form FORMS[] = {
    split_form<16, 1, 1, 4, 5>(8, 2.23f, 0.313f, 0.282f),
    split_form<16, 1, 1, 8, 4>(4, 2.15f, 0.138f, 0.582f),
    split_form<16, 1, 2, 4, 4>(6, 2.39f, 0.664f, 0.494f),
    split_form<16, 1, 2, 8, 4>(3, 2.19f, 0.053f, 1.009f),
    split_form<16, 2, 2, 4, 4, false>(4, 2.69f, 0.873f, 0.649f),
    split_form<16, 2, 2, 8, 4>(2, 2.35f, 0.038f, 1.308f),
    split_form<32, 1, 1, 4, 4>(4, 2.72f, 0.589f, 0.549f),
    split_form<32, 2, 2, 4, 2, false>(1, 4.57f, 1.636f, 0.043f),
    gemm_form<1, 1, 4, 2, 3>(2, 3.00f, 0.520f, 0.362f),
    gemm_form<1, 2, 2, 2, 3>(2, 3.81f, 0.454f, 0.335f),
    gemm_form<2, 2, 2, 1, 3>(2, 5.58f, 0.787f, 0.596f),
    gemm_form<4, 2, 2, 1, 2>(2, 9.49f, 1.484f, 1.071f),
};

// (A grid's threads count in 32 bits.)
bool tiles_of(const Form& f, const Row8Matmul& a, Tiles& t) {
    t.cols = col_tiles_of(a, f.cols - (a.gated ? 1 : 0));
    t.rows = tiles_over(a.rows, f.rows);
    // codes against weights, as rows of n (a weight has 1.125 bytes)
    const float x = (float)t.rows * (float)(1 << f.rows), w = 1.125f * (float)t.cols * (float)(1 << f.cols);
    t.by_columns = x + w / 8 < x / 8 + w;
    return (a.gated ? f.pairs : f.single) && (int64_t)t.rows * t.cols * f.threads < (1ll << 32);
}

float estimate(const Form& f, const Row8Matmul& a, const Tiles& t, int cus) {
    const int groups = (t.rows * t.cols + cus - 1) / cus;  // of the busiest CU
    const float chain = (float)tiles_over(tiles_over(a.n / Q8_BLOCK, f.blocks), f.split);
    const float set = 0.3f * f.fixed;
    const int full = groups / f.resident, rest = groups % f.resident;
    float us = f.fixed + full * (set + chain * std::max(f.alone, f.resident * f.busy));
    if (rest) us += set + chain * std::max(f.alone, rest * f.busy);
    return us;
}

// Rows of one launch at most.
constexpr int SLICE = 1 << 20;

// The form with the least estimate (null: none takes the launch), and its tiles.
const Form* chosen_form(const Row8Matmul& a, Tiles& tiles) {
    const int cus = device_cus();
    const Form* best = nullptr;
    float least = 0.0f;
    for (const Form& f : FORMS) {
        Tiles t;
        if (!tiles_of(f, a, t)) continue;
        const float us = estimate(f, a, t, cus);
        if (!best || us < least) best = &f, least = us, tiles = t;
    }
    return best;
}

}  // namespace

bool row8_matmul_tile(const Row8Matmul& whole, int32_t* tile) {
    Row8Matmul a = whole;
    a.rows = std::min(SLICE, whole.rows);
    Tiles tiles{};
    const Form* f = chosen_form(a, tiles);
    if (!f) return false;
    tile[0] = 1 << f->rows, tile[1] = 1 << f->cols, tile[2] = 1 << f->split;
    return true;
}

hipError_t launch_row8_matmul(const Row8Matmul& whole, hipStream_t stream) {
    for (int r0 = 0; r0 < whole.rows; r0 += std::min(SLICE, whole.rows - r0)) {
        Row8Matmul a = whole;
        a.rows = std::min(SLICE, whole.rows - r0);
        a.codes += (size_t)r0 * a.n;
        a.scales += r0;
        if (a.residual) a.residual += (size_t)r0 * a.d[0];
        for (int m = 0; m < a.mats; m++) a.out[m] += (size_t)r0 * a.d[m];
        Tiles tiles{};
        const Form* best = chosen_form(a, tiles);
        if (!best) return hipErrorInvalidConfiguration;
        best->launch(a, tiles, stream);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace nitro
