// Rows into 8 bits for gfx950 (row8.hpp), with the rms_norm and the residual's
// addition that come before in a model's layer (src/model_q8.cpp:128-140).
//
// Bound by bytes, 5 or 9 (with a residual and its sum 13) an entry: 8192 rows of 4096 with
// residual and sum 82 us (5.3 TB/s, what a copy has), held only 31 us, read back 34 us; one
// row of 4096 3.6, 2.3 and 2.4 us: latency (launch, loads, two joins over the row).
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

__device__ __forceinline__ f32x4 load4(const float* row, int at) { return *reinterpret_cast<const f32x4_any*>(row + at); }
__device__ __forceinline__ void store4(float* row, int at, f32x4 x) { *reinterpret_cast<f32x4_any*>(row + at) = x; }
__device__ __forceinline__ void store4(int8_t* row, int at, uint32_t codes) { *reinterpret_cast<u32_any*>(row + at) = codes; }

__device__ __forceinline__ double joined(double a, double b) { return a + b; }
__device__ __forceinline__ uint32_t joined(uint32_t a, uint32_t b) { return a > b ? a : b; }
// x joined with another lane's, by a data-parallel move; with the next 16 lanes', 32 lanes'.
template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ double moved(double x) {
    return __hiloint2double((int)moved<CTRL>((uint32_t)__double2hiint(x)), (int)moved<CTRL>((uint32_t)__double2loint(x)));
}
__device__ __forceinline__ uint32_t over_16(uint32_t x) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return joined((uint32_t)r[0], (uint32_t)r[1]);
}
__device__ __forceinline__ uint32_t over_32(uint32_t x) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return joined((uint32_t)r[0], (uint32_t)r[1]);
}
__device__ __forceinline__ double over_16(double x) {
    const uint32_t h = (uint32_t)__double2hiint(x), l = (uint32_t)__double2loint(x);
    const auto hi = __builtin_amdgcn_permlane16_swap(h, h, false, false), lo = __builtin_amdgcn_permlane16_swap(l, l, false, false);
    return joined(__hiloint2double((int)hi[0], (int)lo[0]), __hiloint2double((int)hi[1], (int)lo[1]));
}
__device__ __forceinline__ double over_32(double x) {
    const uint32_t h = (uint32_t)__double2hiint(x), l = (uint32_t)__double2loint(x);
    const auto hi = __builtin_amdgcn_permlane32_swap(h, h, false, false), lo = __builtin_amdgcn_permlane32_swap(l, l, false, false);
    return joined(__hiloint2double((int)hi[0], (int)lo[0]), __hiloint2double((int)hi[1], (int)lo[1]));
}
// Sums (double) or the largest (bits) over the T lanes of a row, in the same order every
// time; all of them get the result.  (Moves between lanes take a few cycles, through LDS a
// hundred each: they and the weights loaded with x took 0.5 us off one row of 4096, held only 0.15.)
template <int T, class V>
__device__ __forceinline__ V over_row(V x, V* parts) {
    x = joined(x, moved<0xB1>(x));   // quad_perm [1,0,3,2]
    x = joined(x, moved<0x4E>(x));   // quad_perm [2,3,0,1]
    x = joined(x, moved<0x141>(x));  // row_half_mirror: the other four of eight
    x = joined(x, moved<0x140>(x));  // row_mirror: the other eight of sixteen
    x = over_32(over_16(x));
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = x;
        __syncthreads();
        x = parts[0];
#pragma unroll
        for (int w = 1; w < T / 64; w++) x = joined(x, parts[w]);
    }
    return x;
}

__device__ __forceinline__ float normed(float h, float weight, double r) { return (float)((double)h * r * (double)weight); }
__device__ __forceinline__ f32x4 normed(f32x4 h, f32x4 w, double r) {
#pragma unroll
    for (int e = 0; e < 4; e++) h[e] = normed(h[e], w[e], r);
    return h;
}
__device__ __forceinline__ double squares(f32x4 h, double s) {
#pragma unroll
    for (int e = 0; e < 4; e++) s = fma((double)h[e], (double)h[e], s);
    return s;
}
__device__ __forceinline__ uint32_t largest(float y, uint32_t top) { return joined(top, __float_as_uint(y) & 0x7fffffffu); }
__device__ __forceinline__ uint32_t largest(f32x4 y, uint32_t top) {
#pragma unroll
    for (int e = 0; e < 4; e++) top = largest(y[e], top);
    return top;
}

// What a row with the largest entry of these bits (without sign) is held with.
__device__ __forceinline__ float scale_of(uint32_t top) {
    if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    return __uint_as_float(top) < 0x1p-100f ? 0.0f : __uint_as_float(top) / 127.0f;
}
// (0: zeros for codes)
__device__ __forceinline__ float inverse_of(uint32_t top) {
    return top >= 0x7f800000u || __uint_as_float(top) < 0x1p-100f ? 0.0f : 127.0f / __uint_as_float(top);
}
// The code in the lowest byte: the fma rounds the exact product to an integer, once (a sum
// with 1.5 * 2^23 has whole units).
__device__ __forceinline__ uint32_t code_of(float y, float inv) {
    return __float_as_uint(fmaf(inv == 0.0f ? 0.0f : y, inv, 12582912.0f));
}
__device__ __forceinline__ uint32_t codes_of(f32x4 y, float inv) {
    const uint32_t low = __builtin_amdgcn_perm(code_of(y[1], inv), code_of(y[0], inv), 0x0c0c0400u);
    const uint32_t high = __builtin_amdgcn_perm(code_of(y[3], inv), code_of(y[2], inv), 0x0c0c0400u);
    return low | high << 16;
}

// T lanes to a row (256 / T rows to a workgroup, or one), the row in V groups of four
// entries per lane; the last n % 4 entries are one more of the first lanes each.
template <int T, int V, bool NORM>
__global__ __launch_bounds__(T < 256 ? 256 : T) void row8_norm_kernel(Row8Norm a) {
    constexpr int ROWS = T < 256 ? 256 / T : 1;
    constexpr bool EARLY = T < 1024;  // the weights come with x (more lanes have no registers for it)
    __shared__ double sums[T / 64];
    __shared__ uint32_t tops[T / 64];
    const int lane = threadIdx.x % T, n = a.n, end = n & ~3;
    const int row = blockIdx.x * ROWS + (ROWS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / T) : 0);
    if (row >= a.rows) return;  // (only where a wave has a row: no barrier there)
    const size_t at = (size_t)row * n;
    const float* const x = a.x + at;
    int8_t* const codes = a.codes + at;
    const bool last = lane < n - end;
    f32x4 h[V];
    float tail = 0.0f;
#pragma unroll
    for (int i = 0; i < V; i++) {
        h[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (4 * (lane + i * T) < end) h[i] = load4(x, 4 * (lane + i * T));
    }
    if (last) tail = x[end + lane];
    if constexpr (NORM) {
        f32x4 w[EARLY ? V : 1];
        if constexpr (EARLY) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                w[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (4 * (lane + i * T) < end) w[i] = load4(a.weight, 4 * (lane + i * T));
            }
        }
        if (a.residual) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (4 * (lane + i * T) < end) h[i] += load4(a.residual + at, 4 * (lane + i * T));
            if (last) tail += a.residual[at + end + lane];
        }
        if (a.sum) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (4 * (lane + i * T) < end) store4(a.sum + at, 4 * (lane + i * T), h[i]);
            if (last) a.sum[at + end + lane] = tail;
        }
        const double each = 1.0 / n;  // (while x comes; a quotient behind the sum cost 0.1 us)
        double s = (double)tail * (double)tail;
#pragma unroll
        for (int i = 0; i < V; i++) {
            s = squares(h[i], s);
            if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (64-bit values of four groups at a time)
        }
        const double r = rsqrt(over_row<T>(s, sums) * each + a.eps);
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (4 * (lane + i * T) < end) h[i] = normed(h[i], EARLY ? w[EARLY ? i : 0] : load4(a.weight, 4 * (lane + i * T)), r);
            if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
        if (last) tail = normed(tail, a.weight[end + lane], r);
    }
    uint32_t top = largest(tail, 0);
#pragma unroll
    for (int i = 0; i < V; i++) top = largest(h[i], top);
    top = over_row<T>(top, tops);
    if (lane == 0) a.scales[row] = scale_of(top);
    const float inv = inverse_of(top);
#pragma unroll
    for (int i = 0; i < V; i++)
        if (4 * (lane + i * T) < end) store4(codes, 4 * (lane + i * T), codes_of(h[i], inv));
    if (last) codes[end + lane] = (int8_t)code_of(tail, inv);
}

// Rows past the registers of a workgroup, a workgroup each, read again for every use: the sum
// of squares, y and its maximum, the codes.  With V > 0 (rows up to 4096 V entries, normed) y
// stays in V groups of registers: one row of 65536 with residual and sum 14.7 us, 18.2 without;
// 2000 rows of 20000 112 us, 124.
template <bool NORM, int V>
__global__ __launch_bounds__(1024) void row8_long_kernel(Row8Norm a) {
    constexpr int T = 1024;
    __shared__ double sums[T / 64];
    __shared__ uint32_t tops[T / 64];
    const int lane = threadIdx.x, n = a.n, end = n & ~3;
    const size_t at = (size_t)blockIdx.x * n;
    const float* x = a.x + at;
    const float* residual = a.residual ? a.residual + at : nullptr;
    int8_t* const codes = a.codes + at;
    const bool last = lane < n - end;
    float tail = last ? x[end + lane] : 0.0f;
    double r = 0.0;
    if constexpr (NORM) {
        if (last && residual) tail += residual[end + lane];
        if (last && a.sum) a.sum[at + end + lane] = tail;
        const double each = 1.0 / n;
        double s = (double)tail * (double)tail;
#pragma unroll 4
        for (int v = 4 * lane; v < end; v += 4 * T) {
            f32x4 h = load4(x, v);
            if (residual) h += load4(residual, v);
            if (a.sum) store4(a.sum + at, v, h);
            s = squares(h, s);
        }
        if (a.sum) x = a.sum + at, residual = nullptr;  // (it may lie over either; a lane reads what it wrote)
        r = rsqrt(over_row<T>(s, sums) * each + a.eps);
        if (last) tail = normed(tail, a.weight[end + lane], r);
    }
    auto value = [&](int v) __attribute__((always_inline)) {
        f32x4 h = load4(x, v);
        if (residual) h += load4(residual, v);
        if constexpr (NORM) h = normed(h, load4(a.weight, v), r);
        return h;
    };
    uint32_t top = largest(tail, 0);
    if constexpr (V > 0) {
        f32x4 y[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (4 * (lane + i * T) < end) y[i] = value(4 * (lane + i * T));
            top = largest(y[i], top);
            if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (64-bit values of four groups at a time)
        }
        top = over_row<T>(top, tops);
        const float inv = inverse_of(top);
#pragma unroll
        for (int i = 0; i < V; i++)
            if (4 * (lane + i * T) < end) store4(codes, 4 * (lane + i * T), codes_of(y[i], inv));
    } else {
#pragma unroll 4
        for (int v = 4 * lane; v < end; v += 4 * T) top = largest(value(v), top);
        top = over_row<T>(top, tops);
        const float inv = inverse_of(top);
#pragma unroll 4
        for (int v = 4 * lane; v < end; v += 4 * T) store4(codes, v, codes_of(value(v), inv));
    }
    if (last) codes[end + lane] = (int8_t)code_of(tail, inverse_of(top));
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
        c[i] = at + 3 < n ? *reinterpret_cast<const u32_any*>(from + at) : 0;
    }
#pragma unroll
    for (int i = 0; i < READ / 256; i++) {
        const int at = first + i * 256 + lane * 4;
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = q8_value(c[i], e) * scale;
        if (at + 3 < n) store4(to, at, v);
    }
    const int at = (n & ~3) + lane;  // the last n % 4
    if (at < n && at >= first && at < first + READ) to[at] = (float)from[at] * scale;
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

template <bool NORM>
void launch_long(const Row8Norm& a, hipStream_t stream) {
    const dim3 grid(a.rows), block(1024);
    if (a.n > 65536)
        hipLaunchKernelGGL((row8_long_kernel<NORM, 0>), grid, block, 0, stream, a);
    else if (a.n > 32768) {
        if constexpr (NORM) hipLaunchKernelGGL((row8_long_kernel<true, 16>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((row8_norm_kernel<1024, 16, false>), grid, block, 0, stream, a);
    } else {
        if constexpr (NORM) hipLaunchKernelGGL((row8_long_kernel<true, 8>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((row8_norm_kernel<1024, 8, false>), grid, block, 0, stream, a);
    }
}

}  // namespace

// A wave to a row up to 1024 entries, then a workgroup with four groups of four to a lane
// (as many lanes as groups, 1024 of one each, gained 0.2 us at one row of 4096 and lost 15 to
// 40% past 512 rows).  Past 16384 entries a norm's row is read twice, its 64-bit values leaving
// no registers for it; past 65536 every row three times, or two where nothing is normed.
hipError_t launch_row8_norm(const Row8Norm& whole, hipStream_t stream) {
    constexpr int SLICE = 1 << 21;  // rows of a launch at most (a grid's threads count in 32 bits)
    for (int r0 = 0; r0 < whole.rows; r0 += std::min(SLICE, whole.rows - r0)) {
        Row8Norm a = whole;
        const size_t at = (size_t)r0 * whole.n;
        const int n = a.n;
        a.rows = std::min(SLICE, whole.rows - r0);
        a.x += at, a.codes += at, a.scales += r0;
        if (a.residual) a.residual += at;
        if (a.sum) a.sum += at;
        if (n <= 256) launch_rows<64, 1>(a, stream);
        else if (n <= 512) launch_rows<64, 2>(a, stream);
        else if (n <= 1024) launch_rows<64, 4>(a, stream);
        else if (n <= 2048) launch_rows<256, 2>(a, stream);
        else if (n <= 4096) launch_rows<256, 4>(a, stream);
        else if (n <= 8192) launch_rows<512, 4>(a, stream);
        else if (n <= 16384) launch_rows<1024, 4>(a, stream);
        else if (a.weight) launch_long<true>(a, stream);
        else launch_long<false>(a, stream);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_row8_read(const int8_t* codes, const float* scales, float* x, int rows, int n, hipStream_t stream) {
    const int per_row = (n + READ - 1) / READ;
    const int slice = std::max(1, (1 << 25) / per_row);  // rows of a launch
    for (int r0 = 0; r0 < rows; r0 += std::min(slice, rows - r0)) {
        const int64_t parts = (int64_t)std::min(slice, rows - r0) * per_row;
        const size_t at = (size_t)r0 * n;
        hipLaunchKernelGGL(row8_read_kernel, dim3((unsigned)((parts + 3) / 4)), dim3(256), 0, stream, codes + at, scales + r0,
                           x + at, parts, per_row, n);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace nitro
