// Rows into 8 bits for gfx950 (row8.hpp), with the rms_norm and the residual's
// addition that come before in a model's layer (src/model_q8.cpp:128-140).
//
// Mathematics.  h = fp32(x + residual), y = fp32(h * weight / sqrt(mean(h^2) + eps)).
// The mean, its root and the products are taken in 64 bits and y is rounded once:
// a code is a step of 1/127 of the row's largest entry, so an error of one fp32 rounding
// in y moves the codes that lie next to a border, and which they are would depend on the
// order of a sum.  In 64 bits rows come out the same whatever the split over lanes.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "q8_group.hpp"
#include "row8.hpp"

namespace nitro {
namespace {

// Four entries of a row of any width: rows start at any multiple of 4 (floats) or 1
// (codes) bytes.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32_any __attribute__((aligned(1)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Entries 4v .. 4v + 3 of a row of n (zeros past its end).
__device__ __forceinline__ f32x4 load4(const float* row, int v, int n) {
    if (4 * v + 3 < n) return *reinterpret_cast<const f32x4_any*>(row + 4 * v);
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 3; e++)
        if (4 * v + e < n) x[e] = row[4 * v + e];
    return x;
}
__device__ __forceinline__ void store4(float* row, int v, int n, f32x4 x) {
    if (4 * v + 3 < n) {
        *reinterpret_cast<f32x4_any*>(row + 4 * v) = x;
        return;
    }
#pragma unroll
    for (int e = 0; e < 3; e++)
        if (4 * v + e < n) row[4 * v + e] = x[e];
}
// c: entries 4v .. 4v + 3's codes, a byte each.
__device__ __forceinline__ void store_codes(int8_t* row, int v, int n, uint32_t c) {
    if (4 * v + 3 < n) {
        *reinterpret_cast<u32_any*>(row + 4 * v) = c;
        return;
    }
#pragma unroll
    for (int e = 0; e < 3; e++)
        if (4 * v + e < n) row[4 * v + e] = (int8_t)(c >> (8 * e));
}

__device__ __forceinline__ double joined(double a, double b) { return a + b; }
__device__ __forceinline__ uint32_t joined(uint32_t a, uint32_t b) { return a > b ? a : b; }
// Sums (double) or the largest (bits) over the T lanes of a row, in the same order every
// time; all of them get the result.
template <int T, class V>
__device__ __forceinline__ V over_row(V x, V* parts) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x = joined(x, (V)__shfl_xor(x, m));
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = x;
        __syncthreads();
        x = parts[0];
#pragma unroll
        for (int w = 1; w < T / 64; w++) x = joined(x, parts[w]);
    }
    return x;
}

__device__ __forceinline__ f32x4 normed(f32x4 h, const float* weight, int v, int n, double r) {
    const f32x4 w = load4(weight, v, n);
#pragma unroll
    for (int e = 0; e < 4; e++) h[e] = (float)((double)h[e] * r * (double)w[e]);
    return h;
}
__device__ __forceinline__ double squares(f32x4 h, double s) {
#pragma unroll
    for (int e = 0; e < 4; e++) s = fma((double)h[e], (double)h[e], s);
    return s;
}
__device__ __forceinline__ uint32_t largest(f32x4 y, uint32_t top) {
#pragma unroll
    for (int e = 0; e < 4; e++) top = joined(top, __float_as_uint(y[e]) & 0x7fffffffu);
    return top;
}

// What a row with the largest entry of these bits (without sign) is held with.
__device__ __forceinline__ float scale_of(uint32_t top) {
    if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    return __uint_as_float(top) < 0x1p-100f ? 0.0f : __uint_as_float(top) / 127.0f;
}
__device__ __forceinline__ float inverse_of(uint32_t top) {
    return top >= 0x7f800000u || __uint_as_float(top) < 0x1p-100f ? 0.0f : 127.0f / __uint_as_float(top);
}
// The codes of four entries, a byte each (inv = 0: zeros).
__device__ __forceinline__ uint32_t codes_of(f32x4 y, float inv) {
    uint32_t c = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const double p = (double)(inv == 0.0f ? 0.0f : y[e]) * (double)inv;
        c |= ((uint32_t)(int)rint(p) & 255u) << (8 * e);
    }
    return c;
}

// T lanes to a row (256 / T rows to a workgroup, or one), the row in V groups of four
// entries per lane.
template <int T, int V, bool NORM>
__global__ __launch_bounds__(T < 256 ? 256 : T) void row8_norm_kernel(Row8Norm a) {
    constexpr int ROWS = T < 256 ? 256 / T : 1;
    __shared__ double sums[T / 64];
    __shared__ uint32_t tops[T / 64];
    const int lane = threadIdx.x % T, n = a.n, groups = (n + 3) / 4;
    const int row = blockIdx.x * ROWS + threadIdx.x / T;
    if (row >= a.rows) return;  // (only where a wave has a row: no barrier there)
    const size_t at = (size_t)row * n;
    f32x4 h[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        h[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (lane + i * T < groups) h[i] = load4(a.x + at, lane + i * T, n);
    }
    if constexpr (NORM) {
        if (a.residual) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (lane + i * T < groups) h[i] += load4(a.residual + at, lane + i * T, n);
        }
        if (a.sum) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (lane + i * T < groups) store4(a.sum + at, lane + i * T, n, h[i]);
        }
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < V; i++) s = squares(h[i], s);
        s = over_row<T>(s, sums);
        const double r = 1.0 / sqrt(s / n + a.eps);
#pragma unroll
        for (int i = 0; i < V; i++)
            if (lane + i * T < groups) h[i] = normed(h[i], a.weight, lane + i * T, n, r);
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < V; i++) top = largest(h[i], top);
    top = over_row<T>(top, tops);
    if (lane == 0) a.scales[row] = scale_of(top);
    const float inv = inverse_of(top);
#pragma unroll
    for (int i = 0; i < V; i++)
        if (lane + i * T < groups) store_codes(a.codes + at, lane + i * T, n, codes_of(h[i], inv));
}

// Rows of any width, a workgroup each, read again for every use.
template <bool NORM>
__global__ __launch_bounds__(1024) void row8_long_kernel(Row8Norm a) {
    constexpr int T = 1024;
    __shared__ double sums[T / 64];
    __shared__ uint32_t tops[T / 64];
    const int lane = threadIdx.x, n = a.n, groups = (n + 3) / 4;
    const size_t at = (size_t)blockIdx.x * n;
    const float* x = a.x + at;
    const float* residual = a.residual ? a.residual + at : nullptr;
    double r = 0.0;
    if constexpr (NORM) {
        double s = 0.0;
        for (int v = lane; v < groups; v += T) {
            f32x4 h = load4(x, v, n);
            if (residual) h += load4(residual, v, n);
            if (a.sum) store4(a.sum + at, v, n, h);
            s = squares(h, s);
        }
        if (a.sum) x = a.sum + at, residual = nullptr;  // (it may lie over either; a lane reads what it wrote)
        r = 1.0 / sqrt(over_row<T>(s, sums) / n + a.eps);
    }
    uint32_t top = 0;
    for (int pass = 0; pass < 2; pass++) {
        const float inv = inverse_of(top);
        for (int v = lane; v < groups; v += T) {
            f32x4 h = load4(x, v, n);
            if (residual) h += load4(residual, v, n);
            if constexpr (NORM) h = normed(h, a.weight, v, n, r);
            if (pass == 0) top = largest(h, top);
            else store_codes(a.codes + at, v, n, codes_of(h, inv));
        }
        if (pass == 0) top = over_row<T>(top, tops);
    }
    if (lane == 0) a.scales[blockIdx.x] = scale_of(top);
}

// A wave takes READ entries of one row.
constexpr int READ = 1024;
__global__ __launch_bounds__(256) void row8_read_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales,
                                                        float* __restrict__ x, int64_t parts, int per_row, int n) {
    const int64_t part = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (part >= parts) return;
    const int row = (int)(part / per_row), first = (int)(part % per_row) * READ, lane = threadIdx.x & 63;
    const float scale = scales[row];
    const int8_t* from = codes + (size_t)row * n;
    float* to = x + (size_t)row * n;
    uint32_t c[READ / 256];
#pragma unroll
    for (int i = 0; i < READ / 256; i++) {
        const int at = first + i * 256 + lane * 4;
        c[i] = 0;
        if (at + 3 < n) {
            c[i] = *reinterpret_cast<const u32_any*>(from + at);
        } else {
            for (int e = 0; e < 3; e++)
                if (at + e < n) c[i] |= (uint32_t)(uint8_t)from[at + e] << (8 * e);
        }
    }
#pragma unroll
    for (int i = 0; i < READ / 256; i++) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = q8_value(c[i], e) * scale;
        store4(to, first / 4 + i * 64 + lane, n, v);
    }
}

template <int T, int V>
void launch_rows(const Row8Norm& a, hipStream_t stream) {
    constexpr int ROWS = T < 256 ? 256 / T : 1;
    const dim3 grid((unsigned)((a.rows + ROWS - 1) / ROWS)), block(T < 256 ? 256 : T);
    if (a.weight)
        hipLaunchKernelGGL((row8_norm_kernel<T, V, true>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((row8_norm_kernel<T, V, false>), grid, block, 0, stream, a);
}

}  // namespace

hipError_t launch_row8_norm(const Row8Norm& a, hipStream_t stream) {
    const int n = a.n;
    if (n <= 256) launch_rows<64, 1>(a, stream);
    else if (n <= 512) launch_rows<64, 2>(a, stream);
    else if (n <= 1024) launch_rows<64, 4>(a, stream);
    else if (a.rows <= 256 && n <= 4096) launch_rows<1024, 1>(a, stream);
    else if (a.rows <= 256 && n <= 8192) launch_rows<1024, 2>(a, stream);
    else if (a.rows <= 256 && n <= 16384) launch_rows<1024, 4>(a, stream);
    else if (n <= 2048) launch_rows<256, 2>(a, stream);
    else if (n <= 4096) launch_rows<256, 4>(a, stream);
    else if (n <= 8192) launch_rows<256, 8>(a, stream);
    else if (n <= 16384) launch_rows<256, 16>(a, stream);
    else if (n <= 32768) launch_rows<1024, 8>(a, stream);
    else if (n <= 65536) launch_rows<1024, 16>(a, stream);
    else if (a.weight) hipLaunchKernelGGL((row8_long_kernel<true>), dim3(a.rows), dim3(1024), 0, stream, a);
    else hipLaunchKernelGGL((row8_long_kernel<false>), dim3(a.rows), dim3(1024), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_row8_read(const int8_t* codes, const float* scales, float* x, int rows, int n, hipStream_t stream) {
    const int per_row = (n + READ - 1) / READ;
    const int64_t parts = (int64_t)rows * per_row;
    hipLaunchKernelGGL(row8_read_kernel, dim3((unsigned)((parts + 3) / 4)), dim3(256), 0, stream, codes, scales, x, parts,
                       per_row, n);
    return hipGetLastError();
}

}  // namespace nitro
