// Products of 8-bit rows with Q8_0 matrices for gfx950 (row8.hpp):
//   p[b][i] = xs[b] * sum_j ws[i][j] * (sum_t wq[i][32j + t] * xq[b][32j + t])
//   out[b][i] = act(p + bias[i]) [* (p' + bias'[i])] + residual[b][i]
// The inner sums are exact integers (at most 32 * 127 * 128) on the integer matrix cores,
// and exact in fp32 (24 bits); a block of 32 k has its weight scale, so each takes one
// conversion and one fma into fp32 sums.  The row's scale comes in once, at the end.
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

// (NaN goes through all of them.)
__device__ __forceinline__ float activate(float x, int activation) {
    switch (activation) {
        case NITRO_ACT_RELU: return x < 0.0f ? 0.0f : x;
        case NITRO_ACT_SILU: return x / (1.0f + expf(-x));
        case NITRO_ACT_GELU: return 0.5f * x * erfcf(x * -0.70710678118654752f);
        // 0.5 x (1 + tanh(u)) = x / (1 + exp(-2u)), u = sqrt(2 / pi) (x + 0.044715 x^3)
        case NITRO_ACT_GELU_TANH: return x / (1.0f + expf(-1.5957691216057308f * (x + 0.044715f * x * x * x)));
        default: return x;
    }
}

// The output at batch row b, row i of member m, from its sums (second: the gated one's).
__device__ __forceinline__ float finish(const Row8Matmul& a, int m, int b, int i, float sum, float second, float xs) {
    float p = sum * xs;
    if (a.bias) p += a.bias[i];
    p = activate(p, a.activation);
    if (a.gated) {
        float q = second * xs;
        if (a.bias) q += a.bias[a.d[0] + i];
        p *= q;
    }
    return p;
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

// ---------------------------------------------------------------- few rows
// A workgroup owns RT tiles of 16 batch rows x CT tiles of 16 weight rows; its waves
// split the blocks, each keeping sums of its own, and add them through LDS in wave order.
constexpr int FEW_WAVES = 8;

template <int RT, int CT, bool GATED>
__global__ __launch_bounds__(64 * FEW_WAVES) void row8_few_kernel(Row8Matmul a) {
    extern __shared__ float parts[];  // [wave][RT * CT][64][4]
    constexpr int COLS = 16 * CT / (GATED ? 2 : 1);  // outputs
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15, lg = lane >> 4;
    int ct = blockIdx.x;
    const int member = member_of(a, ct, COLS);
    const int d = a.d[member], n = a.n, nb = n / Q8_BLOCK, tiles = (d + 15) / 16;
    const int b0 = blockIdx.y * 16 * RT;

    const uint8_t* w[CT];
#pragma unroll
    for (int t = 0; t < CT; t++) {
        const int tile = min(ct * (COLS / 16) + (GATED ? t / 2 : t), tiles - 1);
        w[t] = a.w[GATED ? t % 2 : member] + (size_t)tile * nb * Q8_TILE_BYTES;
    }
    const int8_t* x[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) x[r] = a.codes + (size_t)min(b0 + 16 * r + lr, a.rows - 1) * n + 8 * lg;

    f4 acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int t = 0; t < CT; t++) acc[r][t] = f4{0.f, 0.f, 0.f, 0.f};

    // Blocks first .. end, U to a round, the next round's loads ahead of this one's use.
    // A block past the end repeats the last one, times 0.
    constexpr int U = CT * (1 + RT) <= 4 ? 4 : 2;
    const int first = (int)((int64_t)nb * wave / FEW_WAVES), end = (int)((int64_t)nb * (wave + 1) / FEW_WAVES);
    struct Round {
        long wq[U][CT];
        float ws[U][CT];
        long xq[U][RT];
    } ra, rb;
    auto load = [&](Round& R, int blk) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = min(blk + u, nb - 1);
#pragma unroll
            for (int t = 0; t < CT; t++) {
                const uint8_t* p = w[t] + (size_t)k * Q8_TILE_BYTES;
                R.wq[u][t] = *reinterpret_cast<const long*>(p + 64 + 8 * lane);
                R.ws[u][t] = *reinterpret_cast<const float*>(p + 4 * lr);
            }
#pragma unroll
            for (int r = 0; r < RT; r++) R.xq[u][r] = *reinterpret_cast<const long*>(x[r] + (size_t)k * Q8_BLOCK);
        }
    };
    auto use = [&](const Round& R, int blk) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int t = 0; t < CT; t++) {
                const float s = blk + u < end ? R.ws[u][t] : 0.0f;
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    const i4 p = __builtin_amdgcn_mfma_i32_16x16x32_i8(R.xq[u][r], R.wq[u][t], i4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[r][t][i] = fmaf(s, (float)p[i], acc[r][t][i]);
                }
            }
    };
    load(ra, first);
    for (int blk = first; blk < end; blk += 2 * U) {
        load(rb, blk + U);
        use(ra, blk);
        load(ra, blk + 2 * U);
        use(rb, blk + U);
    }
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int t = 0; t < CT; t++)
            *reinterpret_cast<f4*>(&parts[((wave * RT * CT + r * CT + t) * 64 + lane) * 4]) = acc[r][t];
    __syncthreads();
    // Lane l has rows 4 * (l / 16) + i, column l % 16 of a tile.
    for (int e = threadIdx.x; e < 16 * RT * COLS; e += 64 * FEW_WAVES) {
        const int row = e / COLS, col = e % COLS;
        const int at = (row / 16 * CT + (GATED ? col / 16 * 2 : col / 16)) * 256 + (row % 16 / 4 * 16 + col % 16) * 4 + row % 4;
        float s = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int v = 0; v < FEW_WAVES; v++) {
            s += parts[v * RT * CT * 256 + at];
            if constexpr (GATED) s2 += parts[v * RT * CT * 256 + at + 256];
        }
        const int b = b0 + row, i = ct * COLS + col;
        if (b < a.rows && i < d) {
            float y = finish(a, member, b, i, s, s2, a.scales[b]);
            const size_t o = (size_t)b * d + i;
            if (a.residual) y += a.residual[o];
            a.out[member][o] = y;
        }
    }
}

// --------------------------------------------------------------- many rows
// A workgroup of 4 waves owns 64 MT batch rows x 64 NT weight rows (wave: half of each, as
// MT x NT tiles of v_mfma_i32_32x32x32_i8: lane l holds 16 k, half l / 32 of a block, of
// row l % 32).  Two blocks of x and of the weights lie in LDS, two buffers, a barrier for
// each two.  x lies as four planes (a block's halves) of 16 bytes a row, so that lanes read
// consecutive rows; the weights as in the tile layout, runs of 8 k.
template <int MT, int NT, bool GATED>
__global__ __launch_bounds__(256, 2) void row8_gemm_kernel(Row8Matmul a, int col_tiles) {
    constexpr int BM = 64 * MT, BN = 64 * NT, COLS = GATED ? BN / 2 : BN;
    constexpr int PLANE = BM * 16 + 32;  // (the planes' banks lie 32 bytes apart: a row's four runs are written together)
    __shared__ __attribute__((aligned(16))) uint8_t xl[2][4 * PLANE];
    __shared__ __attribute__((aligned(16))) uint8_t wl[2][2 * BN * 32];
    __shared__ float sl[2][2 * BN];
    static_assert(!GATED || NT == 2, "a wave's two column tiles are the gate's and the other's");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave & 1, wn = wave >> 1, lc = lane & 31, lh = lane >> 5;

    // Column tiles fastest, XCD i taking the i-th eighth of the work.
    int wg = blockIdx.x;
    {
        const int total = gridDim.x, per = total >> 3, rem = total & 7, xcd = wg & 7;
        wg = xcd * per + min(xcd, rem) + (wg >> 3);
    }
    const int b0 = wg / col_tiles * BM;
    int ct = wg % col_tiles;
    const int member = member_of(a, ct, COLS);
    const int d = a.d[member], n = a.n, nb = n / Q8_BLOCK, tiles = (d + 15) / 16;

    // The 16-row weight tile at place j (of BN / 16) of the workgroup's.
    auto tile_at = [&](int j) __attribute__((always_inline)) {
        const int at = GATED ? ct * (COLS / 16) + j / 4 * 2 + j % 2 : ct * (COLS / 16) + j;
        return a.w[GATED ? j / 2 % 2 : member] + (size_t)min(at, tiles - 1) * nb * Q8_TILE_BYTES;
    };
    // Staging: x as MT units of 16 bytes a thread, weights NT, one scale (of 2 BN).
    const int8_t* xp[MT];
    int xk, xdst[MT];
    xk = threadIdx.x % 4 * 16;
#pragma unroll
    for (int u = 0; u < MT; u++) {
        const int row = threadIdx.x / 4 + 64 * u;
        xp[u] = a.codes + (size_t)min(b0 + row, a.rows - 1) * n;
        xdst[u] = threadIdx.x % 4 * PLANE + row * 16;
    }
    const uint8_t* wp[NT];
    int wblk[NT];
#pragma unroll
    for (int u = 0; u < NT; u++) {
        const int e = threadIdx.x + 256 * u;
        wblk[u] = e / (2 * BN);
        wp[u] = tile_at(e / 32 % (BN / 16)) + 64 + e % 32 * 16;
    }
    const int sblk = threadIdx.x / BN, srow = threadIdx.x % BN;
    const uint8_t* sp = tile_at(srow / 16) + 4 * (srow % 16);

    struct Stage {
        i4 x[MT], w[NT];
        float s;
    };
    auto load = [&](Stage& S, int blk) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < MT; u++)
            S.x[u] = *reinterpret_cast<const i4*>(xp[u] + min(blk * Q8_BLOCK + xk, n - 16));
#pragma unroll
        for (int u = 0; u < NT; u++)
            S.w[u] = *reinterpret_cast<const i4*>(wp[u] + (size_t)min(blk + wblk[u], nb - 1) * Q8_TILE_BYTES);
        if (2 * BN == 256 || threadIdx.x < 2 * BN)
            S.s = *reinterpret_cast<const float*>(sp + (size_t)min(blk + sblk, nb - 1) * Q8_TILE_BYTES);
    };
    auto put = [&](const Stage& S, int buf, int blk) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < MT; u++) *reinterpret_cast<i4*>(&xl[buf][xdst[u]]) = S.x[u];
#pragma unroll
        for (int u = 0; u < NT; u++) *reinterpret_cast<i4*>(&wl[buf][(threadIdx.x + 256 * u) * 16]) = S.w[u];
        // (a block past the end repeats the last one, times 0)
        if (2 * BN == 256 || threadIdx.x < 2 * BN) sl[buf][threadIdx.x] = blk + sblk < nb ? S.s : 0.0f;
    };

    f16v acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[m][t][i] = 0.0f;

    auto compute = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            i4 x[MT], w[NT];
            float s[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int j = wn * 2 * NT + 2 * t + lc / 16;
                const uint8_t* p = &wl[buf][(h * (BN / 16) + j) * 512 + (2 * lh * 16 + lc % 16) * 8];
                const int2 lo = *reinterpret_cast<const int2*>(p), hi = *reinterpret_cast<const int2*>(p + 128);
                w[t] = i4{lo.x, lo.y, hi.x, hi.y};
                s[t] = sl[buf][h * BN + wn * 32 * NT + 32 * t + lc];
            }
#pragma unroll
            for (int m = 0; m < MT; m++)
                x[m] = *reinterpret_cast<const i4*>(&xl[buf][(2 * h + lh) * PLANE + (wm * 32 * MT + 32 * m + lc) * 16]);
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    i16 zero;
#pragma unroll
                    for (int i = 0; i < 16; i++) zero[i] = 0;
                    const i16 p = __builtin_amdgcn_mfma_i32_32x32x32_i8(x[m], w[t], zero, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[m][t][i] = fmaf(s[t], (float)p[i], acc[m][t][i]);
                }
        }
    };
    const int steps = (nb + 1) / 2;
    Stage st;
    load(st, 0);
    put(st, 0, 0);
    load(st, 2);
#pragma unroll 1
    for (int i = 0; i < steps; i++) {
        __syncthreads();  // step i is staged; the other buffer's readers are done
        put(st, (i + 1) & 1, 2 * i + 2);
        load(st, 2 * i + 4);
        compute(i & 1);
    }

    // Lane l holds row 8 * (i / 4) + 4 * (l / 32) + i % 4, column l % 32 of a tile.
    __syncthreads();
    float* const mine = reinterpret_cast<float*>(&xl[0][0]) + wave * 1024 + lane;
    static_assert(sizeof(xl) >= 4 * 1024 * sizeof(float), "a tile for each wave");
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int row0 = b0 + (wm * MT + m) * 32 + 4 * lh;
        float xs[16];
#pragma unroll
        for (int i = 0; i < 16; i++) xs[i] = a.scales[min(row0 + 8 * (i / 4) + i % 4, a.rows - 1)];
#pragma unroll
        for (int t = 0; t < (GATED ? 1 : NT); t++) {
            const int col = ct * COLS + (GATED ? wn * 32 : (wn * NT + t) * 32) + lc, near = min(col, d - 1);
            float y[16], r[16];
            if (a.residual) {  // (all read before the first is written: it may be the output)
#pragma unroll
                for (int i = 0; i < 16; i++) r[i] = a.residual[(size_t)min(row0 + 8 * (i / 4) + i % 4, a.rows - 1) * d + near];
            }
            const float bias = a.bias ? a.bias[near] : 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) y[i] = acc[m][t][i] * xs[i] + bias;
            if (a.activation) {
                // (through LDS: one copy of the functions, not 16 MT NT)
#pragma unroll
                for (int i = 0; i < 16; i++) mine[64 * i] = y[i];
#pragma unroll 1
                for (int i = 0; i < 16; i++) mine[64 * i] = activate(mine[64 * i], a.activation);
#pragma unroll
                for (int i = 0; i < 16; i++) y[i] = mine[64 * i];
            }
            if constexpr (GATED) {
                const float second = a.bias ? a.bias[d + near] : 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i++) y[i] *= acc[m][1][i] * xs[i] + second;
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

int col_tiles_of(const Row8Matmul& a, int cols) {
    if (a.gated) return (a.d[0] + cols - 1) / cols;
    int t = 0;
    for (int m = 0; m < a.mats; m++) t += (a.d[m] + cols - 1) / cols;
    return t;
}

template <int RT, int CT>
void launch_few(const Row8Matmul& a, hipStream_t stream) {
    const int cols = 16 * CT / (a.gated ? 2 : 1);
    const dim3 grid((unsigned)col_tiles_of(a, cols), (unsigned)((a.rows + 16 * RT - 1) / (16 * RT)));
    constexpr size_t lds = sizeof(float) * FEW_WAVES * RT * CT * 256;
    if constexpr (CT % 2 == 0) {
        if (a.gated) {
            hipLaunchKernelGGL((row8_few_kernel<RT, CT, true>), grid, dim3(64 * FEW_WAVES), lds, stream, a);
            return;
        }
    }
    hipLaunchKernelGGL((row8_few_kernel<RT, CT, false>), grid, dim3(64 * FEW_WAVES), lds, stream, a);
}

template <int MT, int NT>
void launch_gemm(const Row8Matmul& a, hipStream_t stream) {
    const int cols = 64 * NT / (a.gated ? 2 : 1);
    const int ct = col_tiles_of(a, cols);
    const dim3 grid((unsigned)ct * (unsigned)((a.rows + 64 * MT - 1) / (64 * MT)));
    if constexpr (NT == 2) {
        if (a.gated) {
            hipLaunchKernelGGL((row8_gemm_kernel<MT, NT, true>), grid, dim3(256), 0, stream, a, ct);
            return;
        }
    }
    hipLaunchKernelGGL((row8_gemm_kernel<MT, NT, false>), grid, dim3(256), 0, stream, a, ct);
}

}  // namespace

hipError_t launch_row8_matmul(const Row8Matmul& a, hipStream_t stream) {
    if (a.rows <= 16) {
        a.gated ? launch_few<1, 2>(a, stream) : launch_few<1, 1>(a, stream);
    } else if (a.rows <= 64) {
        launch_few<2, 2>(a, stream);
    } else if ((int64_t)a.rows * col_tiles_of(a, 1) < (int64_t)4 << 20) {
        launch_gemm<2, 2>(a, stream);
    } else {
        launch_gemm<4, 2>(a, stream);
    }
    return hipGetLastError();
}

}  // namespace nitro
