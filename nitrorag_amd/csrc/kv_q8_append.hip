// Appending K/V rows to an 8-bit paged cache on gfx950 (layout: kv_q8.hpp), with
// the rotation to their positions on the way, and reading rows back.
//
// Mathematics, per row and K/V head (x the head's K row after rotation, or its V
// row):  a = max |x|,  scale = fl32(a / 127),  inv = fl32(127 / a),
//   code = rint(x * inv) of the exact product,  value = code * scale.
// The product is rounded to an integer once, by one fma that adds 1.5 * 2^23 (the
// integer is then the sum's low mantissa bits), so a code depends on x and a
// alone, not on how products round: |value - x| <= scale / 2 * (1 + 2^-15).
// a < 2^-100 gives scale 0 (inv would leave fp32's range).  A row that holds an
// infinity or a NaN in K or V makes both of its head's scales NaN: attention then
// gives NaN to every query that sees the token and leaves the others alone.
//
// Rotation: pair (j, j+1) by (c, s) = freq[pos][j/2 of the head], products taken
// exactly (in 64 bits) and rounded to fp32 once, so that the codes do not depend
// on fused multiply-adds either.
//
// Bound by bytes, and below a few hundred rows by the launch.
#include <hip/hip_runtime.h>

#include "device_pool.hpp"
#include "kv_q8.hpp"

namespace nitro {
namespace {

constexpr int THREADS = 256;
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

// Maximum of x over the LPH (16, 32, 64) lanes that hold a head's row.
template <int LPH>
__device__ __forceinline__ float head_max(float x) {
#pragma unroll
    for (int d = 1; d < LPH; d *= 2) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}

__device__ __forceinline__ f4 rotated(f4 x, const float* fr, const float* fi) {
    const double c0 = fr[0], s0 = fi[0], c1 = fr[1], s1 = fi[1];
    const double x0 = x.x, x1 = x.y, x2 = x.z, x3 = x.w;
    f4 r;
    r.x = (float)(x0 * c0 - x1 * s0);
    r.y = (float)(x0 * s0 + x1 * c0);
    r.z = (float)(x2 * c1 - x3 * s1);
    r.w = (float)(x2 * s1 + x3 * c1);
    return r;
}

// Four codes, one to a byte.
__device__ __forceinline__ uint32_t codes_of(f4 x, float inv) {
    constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23: sums are integers
    const uint32_t a = __float_as_uint(fmaf(x.x, inv, MAGIC)), b = __float_as_uint(fmaf(x.y, inv, MAGIC));
    const uint32_t c = __float_as_uint(fmaf(x.z, inv, MAGIC)), d = __float_as_uint(fmaf(x.w, inv, MAGIC));
    return (a & 255) | (b & 255) << 8 | (c & 255) << 16 | d << 24;
}

__device__ __forceinline__ float abs_max(f4 x) {
    return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
}
// 0, or NaN where x holds an infinity or a NaN (which a maximum would drop).
__device__ __forceinline__ float poison(f4 x) { return (x.x * 0.0f + x.y * 0.0f) + (x.z * 0.0f + x.w * 0.0f); }

// A unit is one head of one row: query heads first (rotation only), then K/V
// heads.  LPH lanes hold a unit, four dimensions each.
template <int LPH, bool ROPE>
__global__ __launch_bounds__(THREADS) void kv_q8_append_kernel(KvQ8 c, KvQ8Rows rows, float* __restrict__ q,
                                                               float* __restrict__ k, const float* __restrict__ v,
                                                               const float* __restrict__ freq_real,
                                                               const float* __restrict__ freq_imag, int n_heads) {
    const int units = (ROPE ? n_heads : 0) + c.kv_heads;
    const int64_t total = (int64_t)rows.rows * units;
    const int lane = threadIdx.x % LPH, dim = lane * 4;
    for (int64_t u = (int64_t)blockIdx.x * (THREADS / LPH) + threadIdx.x / LPH; u < total;
         u += (int64_t)gridDim.x * (THREADS / LPH)) {
        const int row = (int)(u / units);
        int h = (int)(u - (int64_t)row * units);
        const bool in = dim < c.head_dim;
        const float *fr = nullptr, *fi = nullptr;
        if (ROPE && in) {
            const int64_t at = (int64_t)rows.pos[row] * (c.head_dim / 2) + dim / 2;
            fr = freq_real + at;
            fi = freq_imag + at;
        }
        if (ROPE && h < n_heads) {
            if (in) {
                f4* at = reinterpret_cast<f4*>(q + ((int64_t)row * n_heads + h) * c.head_dim + dim);
                *at = rotated(*at, fr, fi);
            }
            continue;
        }
        if (ROPE) h -= n_heads;
        f4 kx = {0.f, 0.f, 0.f, 0.f}, vx = kx;
        if (in) {
            const int64_t at = ((int64_t)row * c.kv_heads + h) * c.head_dim + dim;
            kx = *reinterpret_cast<const f4*>(k + at);
            vx = *reinterpret_cast<const f4*>(v + at);
            if (ROPE) {
                kx = rotated(kx, fr, fi);
                *reinterpret_cast<f4*>(k + at) = kx;
            }
        }
        const float ka = head_max<LPH>(abs_max(kx)), va = head_max<LPH>(abs_max(vx));
        const bool good = head_max<LPH>(poison(kx) + poison(vx) == 0.0f ? 0.0f : 1.0f) == 0.0f;
        const int slot = rows.slots[row];
        const int page = slot >> 4, t = slot & 15;
        if (slot < 0 || page >= c.num_pages) {
            if (lane == 0 && h == 0) atomicAdd(c.bad_pages, 1);
            continue;
        }
        constexpr float LEAST = 0x1p-100f;
        const float nan = __uint_as_float(0x7fc00000u);
        const uint32_t kc = codes_of(kx, good && ka >= LEAST ? 127.0f / ka : 0.0f);
        const uint32_t vc = codes_of(vx, good && va >= LEAST ? 127.0f / va : 0.0f);
        uint8_t* rec = c.cache + (int64_t)page * c.page_stride + c.layer_off + (int64_t)h * c.record;
        if (dim < c.hdp) {
            const int at = (((t >> 2) * (c.hdp >> 4) + (dim >> 4)) * 4 + (t & 3)) * 16 + (dim & 15);
            *reinterpret_cast<uint32_t*>(rec + at) = good ? kc : 0;
            uint8_t* vb = rec + 16 * c.hdp + dim * 16 + t;
            const uint32_t w = good ? vc : 0;
            vb[0] = (uint8_t)w;
            vb[16] = (uint8_t)(w >> 8);
            vb[32] = (uint8_t)(w >> 16);
            vb[48] = (uint8_t)(w >> 24);
        }
        if (lane == 0) {
            float* s = reinterpret_cast<float*>(rec + 32 * c.hdp);
            s[t] = !good ? nan : ka >= LEAST ? ka / 127.0f : 0.0f;
            s[16 + t] = !good ? nan : va >= LEAST ? va / 127.0f : 0.0f;
        }
    }
}

template <int LPH>
__global__ __launch_bounds__(THREADS) void kv_q8_read_kernel(KvQ8 c, KvQ8Rows rows, float* __restrict__ k,
                                                             float* __restrict__ v) {
    const int64_t total = (int64_t)rows.rows * c.kv_heads;
    const int lane = threadIdx.x % LPH, dim = lane * 4;
    for (int64_t u = (int64_t)blockIdx.x * (THREADS / LPH) + threadIdx.x / LPH; u < total;
         u += (int64_t)gridDim.x * (THREADS / LPH)) {
        const int row = (int)(u / c.kv_heads), h = (int)(u - (int64_t)row * c.kv_heads);
        const int slot = rows.slots[row];
        const int page = slot >> 4, t = slot & 15;
        if (slot < 0 || page >= c.num_pages) {
            if (lane == 0 && h == 0) atomicAdd(c.bad_pages, 1);
            continue;
        }
        if (dim >= c.head_dim) continue;
        const uint8_t* rec = c.cache + (int64_t)page * c.page_stride + c.layer_off + (int64_t)h * c.record;
        const float* s = reinterpret_cast<const float*>(rec + 32 * c.hdp);
        const float ks = s[t], vs = s[16 + t];
        const int at = (((t >> 2) * (c.hdp >> 4) + (dim >> 4)) * 4 + (t & 3)) * 16 + (dim & 15);
        const int8_t* kb = reinterpret_cast<const int8_t*>(rec + at);
        const int8_t* vb = reinterpret_cast<const int8_t*>(rec + 16 * c.hdp + dim * 16 + t);
        const f4 kx = {kb[0] * ks, kb[1] * ks, kb[2] * ks, kb[3] * ks};
        const f4 vx = {vb[0] * vs, vb[16] * vs, vb[32] * vs, vb[48] * vs};
        const int64_t to = ((int64_t)row * c.kv_heads + h) * c.head_dim + dim;
        *reinterpret_cast<f4*>(k + to) = kx;
        *reinterpret_cast<f4*>(v + to) = vx;
    }
}

unsigned groups(int64_t units, int lph) {
    const int64_t per = THREADS / lph, g = (units + per - 1) / per;
    return (unsigned)(g < 1 ? 1 : g > 65536 ? 65536 : g);
}

template <int LPH>
void append(const KvQ8& c, const KvQ8Rows& r, float* q, float* k, const float* v, const float* fr, const float* fi,
            int n_heads, hipStream_t s) {
    const int64_t units = (int64_t)r.rows * ((fr ? n_heads : 0) + c.kv_heads);
    if (fr)
        hipLaunchKernelGGL((kv_q8_append_kernel<LPH, true>), dim3(groups(units, LPH)), dim3(THREADS), 0, s, c, r, q, k,
                           v, fr, fi, n_heads);
    else
        hipLaunchKernelGGL((kv_q8_append_kernel<LPH, false>), dim3(groups(units, LPH)), dim3(THREADS), 0, s, c, r, q, k,
                           v, fr, fi, n_heads);
}

template <int LPH>
void read(const KvQ8& c, const KvQ8Rows& r, float* k, float* v, hipStream_t s) {
    hipLaunchKernelGGL((kv_q8_read_kernel<LPH>), dim3(groups((int64_t)r.rows * c.kv_heads, LPH)), dim3(THREADS), 0, s, c,
                       r, k, v);
}

}  // namespace

hipError_t launch_kv_q8_append(const KvQ8& c, const KvQ8Rows& r, float* q, float* k, const float* v,
                               const float* freq_real, const float* freq_imag, int n_heads, hipStream_t stream) {
    if (c.head_dim > 256 || c.head_dim % 4) return hipErrorInvalidValue;
    (c.hdp <= 64 ? append<16> : c.hdp <= 128 ? append<32> : append<64>)(c, r, q, k, v, freq_real, freq_imag, n_heads,
                                                                       stream);
    return hipGetLastError();
}

hipError_t launch_kv_q8_read(const KvQ8& c, const KvQ8Rows& r, float* k, float* v, hipStream_t stream) {
    if (c.head_dim > 256 || c.head_dim % 4) return hipErrorInvalidValue;
    (c.hdp <= 64 ? read<16> : c.hdp <= 128 ? read<32> : read<64>)(c, r, k, v, stream);
    return hipGetLastError();
}

}  // namespace nitro
