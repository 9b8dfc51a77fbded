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
// Bound by bytes, and below a few hundred rows by the launch.  16384 rows of 32 + 32
// heads of 128 with the rotation take 290-300 us (1.48 GB, 5.0 TB/s; a large copy
// reaches 5.13), read back 131 us (0.68 GB, 5.2 TB/s); one row of 12 heads of 64 takes
// 3.1 and 2.1 us.  A decode batch's rows pay for the order of V: a byte in each of a
// page's 16-byte runs, 16 lines per head (64 rows of 32 heads of 128: 9 us, 5 without
// those stores); attention reads whole operands for it, many times.
#include <hip/hip_runtime.h>

#include "device_pool.hpp"
#include "kv_q8.hpp"

namespace nitro {
namespace {

constexpr int THREADS = 256;
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float f2 __attribute__((ext_vector_type(2), aligned(4)));

constexpr float LEAST = 0x1p-100f;

template <int CTRL>
__device__ __forceinline__ int dpp(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __int_as_float(dpp<CTRL>(__float_as_int(x)));
}
// A lane's partner l ^ M within 16 lanes.
template <int M>
__device__ __forceinline__ int from_xor(int x) {
    if constexpr (M == 1) return dpp<0xB1>(x);                // quad_perm [1,0,3,2]
    if constexpr (M == 2) return dpp<0x4E>(x);                // quad_perm [2,3,0,1]
    if constexpr (M == 4) return dpp<0x1B>(dpp<0x141>(x));    // row_half_mirror (l ^ 7), then quad_perm [3,2,1,0]
    return dpp<0x128>(x);                                     // row_ror:8
}
__device__ __forceinline__ float max_across_16(float x) {  // l, l ^ 16
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_across_32(float x) {  // l, l ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Maximum of x over the LPH (16, 32, 64) lanes that hold a head's row.
template <int LPH>
__device__ __forceinline__ float head_max(float x) {
    x = fmaxf(x, dpp<0xB1>(x));
    x = fmaxf(x, dpp<0x4E>(x));
    x = fmaxf(x, dpp<0x141>(x));  // row_half_mirror: the other four of eight
    x = fmaxf(x, dpp<0x140>(x));  // row_mirror: the other eight of sixteen
    if constexpr (LPH >= 32) x = max_across_16(x);
    if constexpr (LPH >= 64) x = max_across_32(x);
    return x;
}

__device__ __forceinline__ f2 pair(const float* p) { return *reinterpret_cast<const f2*>(p); }
__device__ __forceinline__ f4 rotated(f4 x, f2 fr, f2 fi) {
    const double c0 = fr.x, s0 = fi.x, c1 = fr.y, s1 = fi.y;
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

// What a page's or row's scale and inverse are, from the largest magnitude; a row
// that is not good is held as NaN.
__device__ __forceinline__ float inverse_of(float top, bool good) { return good && top >= LEAST ? 127.0f / top : 0.0f; }
__device__ __forceinline__ float scale_of(float top, bool good) {
    return !good ? __uint_as_float(0x7fc00000u) : top >= LEAST ? top / 127.0f : 0.0f;
}

// Rows anywhere (a decode batch).  A unit is one head of one row: query heads first
// (rotation only), then K/V heads.  LPH lanes hold a unit, four dimensions each.
template <int LPH, bool ROPE>
__global__ __launch_bounds__(THREADS) void kv_q8_append_kernel(KvQ8 c, KvQ8Rows rows, float* __restrict__ q,
                                                               float* __restrict__ k, const float* __restrict__ v,
                                                               const float* __restrict__ freq_real,
                                                               const float* __restrict__ freq_imag, int n_heads) {
    const int units = (ROPE ? n_heads : 0) + c.kv_heads;
    const int64_t total = (int64_t)rows.rows * units;
    const int lane = threadIdx.x % LPH, dim = lane * 4;
    const bool in = dim < c.head_dim;
    for (int64_t u = (int64_t)blockIdx.x * (THREADS / LPH) + threadIdx.x / LPH; u < total;
         u += (int64_t)gridDim.x * (THREADS / LPH)) {
        const int row = (int)(u / units);
        int h = (int)(u - (int64_t)row * units);
        const bool query = ROPE && h < n_heads;
        if (ROPE && !query) h -= n_heads;
        // every load that waits for nothing, then the angles, which wait for the position
        const int pos = ROPE ? rows.pos[row] : 0, slot = rows.slots[row];
        float* const x_at = query ? q + ((int64_t)row * n_heads + h) * c.head_dim + dim
                                  : k + ((int64_t)row * c.kv_heads + h) * c.head_dim + dim;
        f4 x = {0.f, 0.f, 0.f, 0.f}, vx = x;
        if (in) {
            x = *reinterpret_cast<const f4*>(x_at);
            if (!query) vx = *reinterpret_cast<const f4*>(v + ((int64_t)row * c.kv_heads + h) * c.head_dim + dim);
            if (ROPE) {
                const int64_t at = (int64_t)pos * (c.head_dim / 2) + dim / 2;
                x = rotated(x, pair(freq_real + at), pair(freq_imag + at));
                *reinterpret_cast<f4*>(x_at) = x;
            }
        }
        if (query) continue;  // (all the lanes of a unit)
        const float ka = head_max<LPH>(abs_max(x)), va = head_max<LPH>(abs_max(vx));
        const bool good = head_max<LPH>(poison(x) + poison(vx) == 0.0f ? 0.0f : 1.0f) == 0.0f;
        const int page = slot >> 4, t = slot & 15;
        if (slot < 0 || page >= c.num_pages) {
            if (lane == 0 && h == 0) atomicAdd(c.bad_pages, 1);
            continue;
        }
        const uint32_t kc = good ? codes_of(x, inverse_of(ka, good)) : 0, vc = good ? codes_of(vx, inverse_of(va, good)) : 0;
        uint8_t* rec = c.cache + (int64_t)page * c.page_stride + c.layer_off + (int64_t)h * c.record;
        if (dim < c.hdp) {
            const int at = (((t >> 2) * (c.hdp >> 4) + (dim >> 4)) * 4 + (t & 3)) * 16 + (dim & 15);
            *reinterpret_cast<uint32_t*>(rec + at) = kc;
            uint8_t* vb = rec + 16 * c.hdp + dim * 16 + t;
            vb[0] = (uint8_t)vc;
            vb[16] = (uint8_t)(vc >> 8);
            vb[32] = (uint8_t)(vc >> 16);
            vb[48] = (uint8_t)(vc >> 24);
        }
        if (lane == 0) {
            float* s = reinterpret_cast<float*>(rec + 32 * c.hdp);
            s[t] = scale_of(ka, good);
            s[16 + t] = scale_of(va, good);
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

// -------------------------------------------------------------- whole pages
//
// Rows of chunks lie together, up to 16 of one sequence to a page.  A wave takes
// one K/V head of one page: lane (tq = lane % 4, dg = lane / 4) holds four tokens
// (4 tq ..) of dimensions 64 j + 4 dg ..+ 4.  That makes both operand orders whole
// 16-byte runs after a 4 x 4 exchange: K among the lanes dg % 4 (16 dimensions of
// one token each), V among tq (the 16 tokens of one dimension each, after the
// bytes of a lane's own 4 x 4 are turned).  A byte of V at a time, as the kernel
// above writes it, took 815 us for 16384 rows of 32 heads of 128.

__device__ __forceinline__ int pick(bool c, int a, int b) { return c ? a : b; }

// x[j] of lane i of four = x[i] of lane j; the four differ in bits A and 2A (A = 1
// or 4) of the lane.
template <int A>
__device__ __forceinline__ void exchange(int (&x)[4], int lane) {
    const bool lo = lane & A, hi = lane & (2 * A);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const int got = from_xor<A>(pick(lo, x[i], x[i + 1]));
        x[i] = pick(lo, got, x[i]);
        x[i + 1] = pick(lo, x[i + 1], got);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int got = from_xor<2 * A>(pick(hi, x[i], x[i + 2]));
        x[i] = pick(hi, got, x[i]);
        x[i + 2] = pick(hi, x[i + 2], got);
    }
}
// Byte r of x[i] <-> byte i of x[r].
__device__ __forceinline__ void turn_bytes(int (&x)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
    x[0] = (int)__builtin_amdgcn_perm(b, a, 0x05040100u);
    x[1] = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
    x[2] = (int)__builtin_amdgcn_perm(d, c, 0x05040100u);
    x[3] = (int)__builtin_amdgcn_perm(d, c, 0x07060302u);
}
__device__ __forceinline__ float page_max(float x) {  // over dg
    x = fmaxf(x, dpp<0x124>(x));                      // row_ror:4
    x = fmaxf(x, dpp<0x128>(x));                      // row_ror:8
    return max_across_32(max_across_16(x));
}

// Rows of one page: first .. first + count - 1 of the packed ones, tokens t0 .. t0 +
// count - 1 of the page; pos: the first one's position.
struct PageRows {
    int first, count, t0, page, pos;
};
// The pages that begin (with the page, or with a chunk) in rows 64 block .. + 64 are
// dealt to five waves: four pages where all are whole, a fifth where chunks meet.
constexpr int PAGE_BLOCK = 64, PAGE_WAVES = 5;
// f(lane, PageRows) for each page of wave `rest` % 5 of block `rest` / 5, the same in all
// lanes.  Found from the rows' slots and positions alone, so that a captured launch
// works on any batch of as many rows.
template <class F>
__device__ __forceinline__ void each_page(const KvQ8Rows& rows, int64_t rest, F f) {
    const int64_t base = rest / PAGE_WAVES * PAGE_BLOCK;
    if (base >= rows.rows) return;
    const int lane = threadIdx.x & 63, row = (int)base + lane;
    const bool in = row < rows.rows, in_after = lane < 16 && row + PAGE_BLOCK < rows.rows;
    // (all loads at once)
    const int here = in ? row : 0, later = in_after ? row + PAGE_BLOCK : here;
    const int at[4] = {here, max(here - 1, 0), later, max(later - 1, 0)};
    int slots[4], pos[4];
#pragma unroll
    for (int i = 0; i < 4; i++) slots[i] = rows.slots[at[i]], pos[i] = rows.pos[at[i]];
    // does a row go on where the one before it ends?
    auto follows = [&](int i) {
        return (slots[i] & 15) != 0 && slots[i] == slots[i + 1] + 1 && pos[i] == pos[i + 1] + 1;
    };
    const uint64_t next = __builtin_amdgcn_ballot_w64(in && row > 0 && follows(0));
    const uint64_t after = __builtin_amdgcn_ballot_w64(in_after && follows(2));
    uint64_t starts = __builtin_amdgcn_ballot_w64(in) & ~next;
    for (int i = (int)(rest % PAGE_WAVES); i > 0; i--) starts &= starts - 1;
    while (starts) {
        int self = lane;
        asm volatile("" : "+v"(self));  // (what follows from the lane is made anew, not kept in registers)
        const int i = __builtin_ctzll(starts);
        const uint64_t run = (next >> i >> 1) | (after << (63 - i));  // (15 follow at most)
        const int slot = __builtin_amdgcn_readlane(slots[0], i);
        f(self, PageRows{(int)base + i, 1 + __builtin_ctzll(~run), slot & 15, slot >> 4,
                         __builtin_amdgcn_readlane(pos[0], i)});
        for (int n = 0; n < PAGE_WAVES; n++) starts &= starts - 1;
    }
}

typedef int i4 __attribute__((ext_vector_type(4)));

// J = hdp / 64, rounded up.
template <int J, bool ROPE>
__device__ __forceinline__ void append_page(const KvQ8& c, const PageRows& p, int h, int lane, float* __restrict__ k,
                                            const float* __restrict__ v, const float* __restrict__ freq_real,
                                            const float* __restrict__ freq_imag) {
    const int tq = lane & 3, dg = lane >> 2;
    f4 kx[J][4], vx[J][4];
    f2 fr[J][4], fi[J][4];
    bool here[4];
    // (lanes without a row of their own load the page's last one: no branches between the loads)
    int row[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        row[r] = min(max(4 * tq + r - p.t0, 0), p.count - 1);
        here[r] = row[r] == 4 * tq + r - p.t0;
    }
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int dim = 64 * j + 4 * dg;
#pragma unroll
        for (int r = 0; r < 4; r++) kx[j][r] = vx[j][r] = f4{0.f, 0.f, 0.f, 0.f}, fr[j][r] = fi[j][r] = f2{0.f, 0.f};
        if (dim < c.head_dim) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int64_t at = ((int64_t)(p.first + row[r]) * c.kv_heads + h) * c.head_dim + dim;
                kx[j][r] = *reinterpret_cast<const f4*>(k + at);
                vx[j][r] = *reinterpret_cast<const f4*>(v + at);
                if (ROPE) {
                    const int64_t f = (int64_t)(p.pos + row[r]) * (c.head_dim / 2) + dim / 2;
                    fr[j][r] = pair(freq_real + f);
                    fi[j][r] = pair(freq_imag + f);
                }
            }
        }
    }
    float ka[4] = {0.f, 0.f, 0.f, 0.f}, va[4] = {0.f, 0.f, 0.f, 0.f}, bad[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int j = 0; j < J; j++) {
            const int dim = 64 * j + 4 * dg;
            const bool in = here[r] && dim < c.head_dim;
            if (ROPE) {
                kx[j][r] = rotated(kx[j][r], fr[j][r], fi[j][r]);
                const int64_t at = ((int64_t)(p.first + 4 * tq + r - p.t0) * c.kv_heads + h) * c.head_dim + dim;
                if (in) *reinterpret_cast<f4*>(k + at) = kx[j][r];
            }
            const f4 zero = {0.f, 0.f, 0.f, 0.f};
            kx[j][r] = here[r] ? kx[j][r] : zero;
            vx[j][r] = here[r] ? vx[j][r] : zero;
        }
    float ks[4], vs[4], ki[4], vi[4];
    bool good[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
#pragma unroll
        for (int j = 0; j < J; j++) {
            ka[r] = fmaxf(ka[r], abs_max(kx[j][r]));
            va[r] = fmaxf(va[r], abs_max(vx[j][r]));
            bad[r] += poison(kx[j][r]) + poison(vx[j][r]);
        }
        ka[r] = page_max(ka[r]);
        va[r] = page_max(va[r]);
        good[r] = page_max(bad[r] == 0.0f ? 0.0f : 1.0f) == 0.0f;
        ks[r] = scale_of(ka[r], good[r]), ki[r] = inverse_of(ka[r], good[r]);
        vs[r] = scale_of(va[r], good[r]), vi[r] = inverse_of(va[r], good[r]);
    }
    if (p.page < 0 || p.page >= c.num_pages) {
        if (lane == 0 && h == 0) atomicAdd(c.bad_pages, p.count);
        return;
    }
    uint8_t* rec = c.cache + (int64_t)p.page * c.page_stride + c.layer_off + (int64_t)h * c.record;
    const int chunks = c.hdp >> 4, mine = 4 * tq + (dg & 3);  // the token this lane has of K after the exchange
    const bool whole = p.count == 16;
#pragma unroll
    for (int j = 0; j < J; j++) {
        int kc[4], vc[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            kc[r] = good[r] ? (int)codes_of(kx[j][r], ki[r]) : 0;
            vc[r] = good[r] ? (int)codes_of(vx[j][r], vi[r]) : 0;
        }
        exchange<4>(kc, lane);
        turn_bytes(vc);
        exchange<1>(vc, lane);
        const int chunk = 4 * j + (dg >> 2);
        if (chunk >= chunks) continue;
        if (whole || (unsigned)(mine - p.t0) < (unsigned)p.count)
            *reinterpret_cast<i4*>(rec + ((tq * chunks + chunk) * 4 + (dg & 3)) * 16) = i4{kc[0], kc[1], kc[2], kc[3]};
        uint8_t* vb = rec + 16 * c.hdp + (64 * j + 4 * dg + tq) * 16;
        if (whole) {
            *reinterpret_cast<i4*>(vb) = i4{vc[0], vc[1], vc[2], vc[3]};
        } else {  // the page's other tokens stay as they are
#pragma unroll
            for (int t = 0; t < 16; t++)
                if ((unsigned)(t - p.t0) < (unsigned)p.count) vb[t] = (uint8_t)(vc[t >> 2] >> (8 * (t & 3)));
        }
    }
    if (dg == 0) {
        float* s = reinterpret_cast<float*>(rec + 32 * c.hdp) + 4 * tq;
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (here[r]) s[r] = ks[r], s[16 + r] = vs[r];
    }
}

// Workgroups past page_blocks rotate q.
template <int J, bool ROPE>
__global__ __launch_bounds__(THREADS) void kv_q8_append_pages_kernel(KvQ8 c, KvQ8Rows rows, float* __restrict__ q,
                                                                     float* __restrict__ k, const float* __restrict__ v,
                                                                     const float* __restrict__ freq_real,
                                                                     const float* __restrict__ freq_imag, int n_heads,
                                                                     unsigned page_blocks) {
    if (ROPE && blockIdx.x >= page_blocks) {
        const int per_row = n_heads * c.head_dim / 4;  // float4
        const int64_t total = (int64_t)rows.rows * per_row;
        for (int64_t i = (int64_t)(blockIdx.x - page_blocks) * THREADS + threadIdx.x; i < total;
             i += (int64_t)(gridDim.x - page_blocks) * THREADS) {
            const int row = (int)(i / per_row), dim = (int)(i - (int64_t)row * per_row) * 4 % c.head_dim;
            const int64_t at = (int64_t)rows.pos[row] * (c.head_dim / 2) + dim / 2;
            f4* x = reinterpret_cast<f4*>(q + 4 * i);
            *x = rotated(*x, pair(freq_real + at), pair(freq_imag + at));
        }
        return;
    }
    const int64_t unit = (int64_t)blockIdx.x * (THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = (int)(unit % c.kv_heads);
    each_page(rows, unit / c.kv_heads, [&](int lane, const PageRows& p) {
        append_page<J, ROPE>(c, p, h, lane, k, v, freq_real, freq_imag);
    });
}

template <int J>
__device__ __forceinline__ void read_page(const KvQ8& c, const PageRows& p, int h, int lane, float* __restrict__ k,
                                          float* __restrict__ v) {
    const int tq = lane & 3, dg = lane >> 2;
    if (p.page < 0 || p.page >= c.num_pages) {
        if (lane == 0 && h == 0) atomicAdd(c.bad_pages, p.count);
        return;
    }
    const uint8_t* rec = c.cache + (int64_t)p.page * c.page_stride + c.layer_off + (int64_t)h * c.record;
    const int chunks = c.hdp >> 4;
    const f4 ks = *reinterpret_cast<const f4*>(rec + 32 * c.hdp + 16 * tq);
    const f4 vs = *reinterpret_cast<const f4*>(rec + 32 * c.hdp + 64 + 16 * tq);
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int chunk = 4 * j + (dg >> 2), dim = 64 * j + 4 * dg;
        i4 kl = {0, 0, 0, 0}, vl = kl;
        if (chunk < chunks) {
            kl = *reinterpret_cast<const i4*>(rec + ((tq * chunks + chunk) * 4 + (dg & 3)) * 16);
            vl = *reinterpret_cast<const i4*>(rec + 16 * c.hdp + (dim + tq) * 16);
        }
        int kc[4] = {kl[0], kl[1], kl[2], kl[3]}, vc[4] = {vl[0], vl[1], vl[2], vl[3]};
        exchange<4>(kc, lane);
        exchange<1>(vc, lane);
        turn_bytes(vc);
        if (dim >= c.head_dim) continue;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if ((unsigned)(4 * tq + r - p.t0) >= (unsigned)p.count) continue;
            const int64_t at = ((int64_t)(p.first + 4 * tq + r - p.t0) * c.kv_heads + h) * c.head_dim + dim;
            *reinterpret_cast<f4*>(k + at) = f4{(float)(int8_t)kc[r] * ks[r], (float)(int8_t)(kc[r] >> 8) * ks[r],
                                                (float)(int8_t)(kc[r] >> 16) * ks[r], (float)(kc[r] >> 24) * ks[r]};
            *reinterpret_cast<f4*>(v + at) = f4{(float)(int8_t)vc[r] * vs[r], (float)(int8_t)(vc[r] >> 8) * vs[r],
                                                (float)(int8_t)(vc[r] >> 16) * vs[r], (float)(vc[r] >> 24) * vs[r]};
        }
    }
}

template <int J>
__global__ __launch_bounds__(THREADS) void kv_q8_read_pages_kernel(KvQ8 c, KvQ8Rows rows, float* __restrict__ k,
                                                                   float* __restrict__ v) {
    const int64_t unit = (int64_t)blockIdx.x * (THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = (int)(unit % c.kv_heads);
    each_page(rows, unit / c.kv_heads, [&](int lane, const PageRows& p) { read_page<J>(c, p, h, lane, k, v); });
}

unsigned groups(int64_t units, int lph) {
    const int64_t per = THREADS / lph, g = (units + per - 1) / per;
    return (unsigned)(g < 1 ? 1 : g > 65536 ? 65536 : g);
}
// Workgroups that take a batch by its pages.
int64_t page_groups(const KvQ8& c, const KvQ8Rows& r) {
    const int64_t waves = ((int64_t)r.rows + PAGE_BLOCK - 1) / PAGE_BLOCK * PAGE_WAVES * c.kv_heads;
    return (waves + THREADS / 64 - 1) / (THREADS / 64);
}

template <int J>
void append(const KvQ8& c, const KvQ8Rows& r, float* q, float* k, const float* v, const float* fr,
            const float* fi, int n_heads, hipStream_t s) {
    constexpr int LPH = J == 1 ? 16 : J == 2 ? 32 : 64;
    if (r.together) {
        const unsigned pages = (unsigned)page_groups(c, r);
        const unsigned turn = fr ? groups((int64_t)r.rows * n_heads * c.head_dim / 4, 1) : 0;
        if (fr)
            hipLaunchKernelGGL((kv_q8_append_pages_kernel<J, true>), dim3(pages + turn), dim3(THREADS), 0, s, c, r, q,
                               k, v, fr, fi, n_heads, pages);
        else
            hipLaunchKernelGGL((kv_q8_append_pages_kernel<J, false>), dim3(pages), dim3(THREADS), 0, s, c, r, q, k, v,
                               fr, fi, n_heads, pages);
        return;
    }
    const int64_t units = (int64_t)r.rows * ((fr ? n_heads : 0) + c.kv_heads);
    if (fr)
        hipLaunchKernelGGL((kv_q8_append_kernel<LPH, true>), dim3(groups(units, LPH)), dim3(THREADS), 0, s, c, r, q, k,
                           v, fr, fi, n_heads);
    else
        hipLaunchKernelGGL((kv_q8_append_kernel<LPH, false>), dim3(groups(units, LPH)), dim3(THREADS), 0, s, c, r, q, k,
                           v, fr, fi, n_heads);
}

template <int J>
void read(const KvQ8& c, const KvQ8Rows& r, float* k, float* v, hipStream_t s) {
    constexpr int LPH = J == 1 ? 16 : J == 2 ? 32 : 64;
    if (r.together)
        hipLaunchKernelGGL((kv_q8_read_pages_kernel<J>), dim3((unsigned)page_groups(c, r)), dim3(THREADS), 0, s, c, r,
                           k, v);
    else
        hipLaunchKernelGGL((kv_q8_read_kernel<LPH>), dim3(groups((int64_t)r.rows * c.kv_heads, LPH)), dim3(THREADS), 0, s,
                           c, r, k, v);
}

// The pages' workgroups have a grid index each.
bool fits(const KvQ8& c, const KvQ8Rows& r) {
    return c.head_dim >= 4 && c.head_dim <= 256 && c.head_dim % 4 == 0 &&
           page_groups(c, r) <= INT32_MAX - 65536;
}

}  // namespace

hipError_t launch_kv_q8_append(const KvQ8& c, const KvQ8Rows& r, float* q, float* k,
                               const float* v, const float* freq_real, const float* freq_imag, int n_heads,
                               hipStream_t stream) {
    if (!fits(c, r)) return hipErrorInvalidValue;
    auto* const f = c.hdp <= 64 ? append<1> : c.hdp <= 128 ? append<2> : c.hdp <= 192 ? append<3> : append<4>;
    f(c, r, q, k, v, freq_real, freq_imag, n_heads, stream);
    return hipGetLastError();
}

hipError_t launch_kv_q8_read(const KvQ8& c, const KvQ8Rows& r, float* k, float* v,
                             hipStream_t stream) {
    if (!fits(c, r)) return hipErrorInvalidValue;
    auto* const f = c.hdp <= 64 ? read<1> : c.hdp <= 128 ? read<2> : c.hdp <= 192 ? read<3> : read<4>;
    f(c, r, k, v, stream);
    return hipGetLastError();
}

}  // namespace nitro
