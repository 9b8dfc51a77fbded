// Decode over an 8-bit paged cache on gfx950: one token per sequence, long contexts
// split over workgroups (the products and the softmax: kv_q8_attn.hpp).
//
// Bound by bytes: 2 * head_dim + 8 per key and K/V head.  64 x 4096 tokens at 32 x 128
// take 328 us (6.74 TB/s, what this card streams; vector instructions in a third of the
// SIMDs' cycles), one sequence of 131072 at 32/8 x 128 48 us (5.8 TB/s: start and the
// join of 32 splits are 7 us), 24 of 512 to 8192 41 us (the same, and splits that do not
// fill the CUs evenly), 32 of 16 to 1024 at 12 x 64 9 us and one of 256 5 us (latency:
// launch, table entry, K/V, products, join).
//
// A product's 16 columns are the query heads of one K/V head, so K and V are read once
// for up to 16 of them; with fewer the other columns compute nothing, which the matrix
// cores have room for.  A wave has a tile of 64 keys in registers and the next one's
// loads in flight; four waves to a workgroup (eight, joined in LDS rather than through
// memory: 11.4 against 10.9 us for the 32 sequences, 53.2 against 51.9 for the long
// one).
#include <hip/hip_runtime.h>

#include "device_pool.hpp"
#include "kv_q8.hpp"
#include "kv_q8_attn.hpp"

namespace nitro {
namespace {

// A wave's tiles first, first + step, ... below end (end > first) of the keys of one
// table row.  A tile's K loads go out as soon as the previous tile's K is in its
// products and its V loads likewise, so loads are in flight throughout; loads return
// in order, so table entries are asked for two tiles ahead, where waiting for them is
// waiting for nothing younger.  Of tile t the lane's column sees seen(t) tokens of
// page lane / 16.  kp, vp: the first tile's table entries; page(i): entry i (any i).
template <int CH, bool STREAM, class Page, class Seen>
__device__ __forceinline__ void attend(State<CH>& st, const QueryRow<(CH + 3) / 4>& row, float qscale, const KvQ8& c,
                                       const uint8_t* base, int first, int end, int step, int lane, int kp, int vp,
                                       Page page, Seen seen) {
    const int g = lane >> 4, sub = (lane & 15) >> 2;
    KTile<CH> k = no_k<CH>();
    VTile<CH> v[1];
    load_k<CH, STREAM>(k, record(c, base, kp), record(c, base, vp), lane);
    int kp_next = page(4 * (first + step) + sub), vp_next = page(4 * (first + step) + g);
    load_v<CH, STREAM>(v[0], record(c, base, vp), lane);
    __builtin_amdgcn_sched_barrier(0);  // the loads are on their way before the query is waited for
    const auto q = query_of(row, qscale);
    int t = first;
    auto tile = [&](auto more) {
        int kp_then = 0, vp_then = 0;
        if (more) kp_then = page(4 * (t + 2 * step) + sub), vp_then = page(4 * (t + 2 * step) + g);
        const int keys = seen_on(c, vp, seen(t), lane);
        f4 s[1][4];
        const float top = scores<CH>(s[0], k, q, keys);
        const float scales[1] = {k.vs};
        if (more) load_k<CH, STREAM>(k, record(c, base, kp_next), record(c, base, vp_next), lane);
        const Weights<1> w = weigh<CH, 1>(st, s, top, q.scale, scales);
        add_values<CH, 1>(st, v, w);
        if (more) {
            load_v<CH, STREAM>(v[0], record(c, base, vp_next), lane);
            vp = vp_next;
            asm volatile("" : "+v"(kp_then), "+v"(vp_then));  // here by now
            kp_next = kp_then, vp_next = vp_then;
        }
        t += step;
    };
    while (t + step < end) tile(std::true_type());
    tile(std::false_type());  // (on its own: a load that may be missing costs waits for all of them)
}

// Device-coherent accesses of the partials and counters: relaxed atomics at agent
// scope, written through to and read from where the XCDs' caches agree.  Two floats
// at a time (8-byte aligned).
__device__ __forceinline__ void store_coherent(float* p, float x, float y) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_coherent(const float* p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<uint64_t*>(const_cast<float*>(p)), __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
    return x;
}

// out = A / L; 0 where no key was seen.
__device__ __forceinline__ float divided(float A, float L) { return L == 0.0f ? 0.0f : A / L; }

constexpr int JOIN = 16;  // partials whose loads go out together

// Tokens that sequence b's row attends.
__device__ __forceinline__ int seen_by(const KvQ8Decode& a, int b) {
    return max(0, min(a.positions[b], a.ctx_limit - 1) + 1);
}
// Tiles per split of a sequence.  (More than planned in a captured launch that is
// replayed over a later batch with a longer sequence.)
__device__ __forceinline__ int split_tiles(const KvQ8Decode& a, int tiles) {
    return tiles > a.num_splits * a.tiles_per_split ? (tiles + a.num_splits - 1) / a.num_splits : a.tiles_per_split;
}
// The sequence and split of work item i, the sequences' splits one after the other; -1
// past the last.  (Workgroups go round the CUs in order of their index: with an index
// for every sequence and each split that the longest has, the CUs had more or less
// work as those that a short one lacks fell.)
__device__ __forceinline__ int item_of(const KvQ8Decode& a, int i, int lane, int& split) {
    for (int base = 0; base < a.batch; base += 64) {
        int n = 0;
        if (base + lane < a.batch) {
            const int tiles = (seen_by(a, base + lane) + KV_Q8_TILE - 1) / KV_Q8_TILE, tps = split_tiles(a, tiles);
            n = max(1, (tiles + tps - 1) / tps);
        }
        int upto = n;  // splits of the sequences up to the lane's
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int x = __shfl_up(upto, d);
            if (lane >= d) upto += x;
        }
        const int total = __builtin_amdgcn_readlane(upto, 63);
        if (i < total) {
            const int at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto <= i));
            split = i - __builtin_amdgcn_readlane(upto - n, at);
            return base + at;
        }
        i -= total;
    }
    return -1;
}

// A workgroup takes one split of one sequence's keys for up to 16 query heads of a
// K/V head; its waves take the split's tiles in turn.  Waves per SIMD are what the
// registers allow without spills (at head size 128 210; an earlier form had 183, and
// three waves with 13 of them spilled took 404 us where two took 337).  At head sizes
// 132 to 176 the build keeps a K operand in scratch, 80 bytes a lane: 16 sequences of
// 1024 at 16/8 x 160 take 18.6 us where 16/8 x 192 take 14.8.
template <int CH, bool STREAM>
__global__ __launch_bounds__(256, kv_q8_decode_occupancy(16 * CH)) void kv_q8_decode_kernel(KvQ8Decode a) {
    extern __shared__ float s_part[];  // [waves][cols][pstride], then of a join [cols][parts] factors and [cols] sums
    __shared__ int s_last;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv_mul = a.n_heads / a.c.kv_heads;
    const int groups = (kv_mul + KV_Q8_COLUMNS - 1) / KV_Q8_COLUMNS;
    int w = blockIdx.x;
    if (a.ordered) {
        const int round = w / a.ordered, in_round = min(a.ordered, (int)gridDim.x - round * a.ordered);
        if (round % 2) w = round * a.ordered + in_round - 1 - (w - round * a.ordered);
    }
    const int hg = w % groups;
    w /= groups;
    const int kv_h = w % a.c.kv_heads;
    w /= a.c.kv_heads;
    int split = w, b = 0;
    if (a.num_splits == 1) {
        split = 0, b = a.ordered ? a.order[w] : w;
    } else if (a.batch > 1) {
        b = item_of(a, w, lane, split);
        if (b < 0) return;
    }
    const int h0 = kv_h * kv_mul + hg * KV_Q8_COLUMNS;  // first query head
    const int cols = min(KV_Q8_COLUMNS, kv_mul - hg * KV_Q8_COLUMNS);
    const int hd = a.c.head_dim;
    const int col = lane & 15, g = lane >> 4;

    // Table entries past the sequence's own may be read (their ids are checked,
    // their keys hidden): the first tile's loads wait for its entries alone.
    const int32_t* trow = a.tables + (int64_t)b * a.max_pages;
    auto page = [&](int i) {  // (atomic: a load that stays where it is written)
        return __hip_atomic_load(trow + min(i, a.max_pages - 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
    };
    int tps = a.tiles_per_split, t0 = split * tps;
    int kp = page(4 * (t0 + wave) + (col >> 2)), vp = page(4 * (t0 + wave) + g);
    const float* q_at = a.q + ((int64_t)b * a.n_heads + h0 + col) * hd;
    const auto row = load_row<(CH + 3) / 4>(col < cols ? q_at : nullptr, hd, g);
    const int ctx = seen_by(a, b), tiles = (ctx + KV_Q8_TILE - 1) / KV_Q8_TILE;
    if (tiles > a.num_splits * tps) {
        tps = split_tiles(a, tiles);
        t0 = split * tps;
        kp = page(4 * (t0 + wave) + (col >> 2)), vp = page(4 * (t0 + wave) + g);
    }
    const int parts = max(1, (tiles + tps - 1) / tps);
    if (split >= parts) return;
    if (ctx == 0 && hg == 0 && kv_h == 0 && threadIdx.x == 0) atomicAdd(a.c.bad_pages, 1);  // a position below 0
    const int t1 = min(tiles, t0 + tps);

    State<CH> st;
#pragma unroll
    for (int t = 0; t < CH; t++) st.o[t] = f4{0.f, 0.f, 0.f, 0.f};
    if (t0 + wave < t1) {
        const uint8_t* base = a.c.cache + a.c.layer_off + (int64_t)kv_h * a.c.record;
        attend<CH, STREAM>(st, row, a.qscale, a.c, base, t0 + wave, t1, a.waves, lane, kp, vp, page, [&](int t) { return ctx - t * KV_Q8_TILE - 16 * g; });
    }

    // The waves' parts meet in LDS.
    st.l = column_sum(st.l);
    if (col < cols) {
        float* part = s_part + (wave * cols + col) * a.pstride;
#pragma unroll
        for (int t = 0; t < CH; t++) {
            const int dim = 16 * t + 4 * g;
            if (dim < hd) *reinterpret_cast<f4*>(part + dim) = st.o[t];
        }
        if (g == 0) {
            part[hd] = st.m;
            part[hd + 1] = st.l;
        }
    }
    __syncthreads();
    const int pairs = cols * hd / 2;
    for (int o = threadIdx.x; o < pairs; o += blockDim.x) {
        const int c = 2 * o / hd, d = 2 * o - c * hd;
        float M = -INFINITY, L = 0.0f, A0 = 0.0f, A1 = 0.0f;
        for (int wv = 0; wv < a.waves; wv++) M = fmaxf(M, s_part[(wv * cols + c) * a.pstride + hd]);
        for (int wv = 0; wv < a.waves; wv++) {
            const float* part = s_part + (wv * cols + c) * a.pstride;
            const float m = part[hd], f = scale_of(m, M);
            L += m == -INFINITY ? part[hd + 1] : part[hd + 1] * f;  // no finite maximum: 0 or NaN
            A0 = fmaf(part[d], f, A0);
            A1 = fmaf(part[d + 1], f, A1);
        }
        if (parts == 1) {
            float* out = a.out + ((int64_t)b * a.n_heads + h0 + c) * hd + d;
            out[0] = divided(A0, L);
            out[1] = divided(A1, L);
        } else {
            float* part = a.partials + (((int64_t)b * a.num_splits + split) * a.n_heads + h0 + c) * a.pstride;
            store_coherent(part + d, A0, A1);
            if (d == 0) store_coherent(part + hd, M, L);
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
    const int64_t stride = (int64_t)a.n_heads * a.pstride;  // from split to split
    const float* parts0 = a.partials + ((int64_t)b * a.num_splits * a.n_heads + h0) * a.pstride;
    // a wave per head: the splits' factors 2^(m - M) and the sum (lane i holds splits i, i + 64, ..)
    for (int c = wave; c < cols; c += a.waves) {
        auto m_and_l = [&](int sp) { return load_coherent(parts0 + sp * stride + c * a.pstride + hd); };
        const float2 first = m_and_l(min(lane, parts - 1));
        float M = first.x, L = 0.0f;
        for (int sp = lane + 64; sp < parts; sp += 64) M = fmaxf(M, m_and_l(sp).x);
        M = wave_max(M);
        for (int sp = lane; sp < parts; sp += 64) {
            const float2 ml = sp == lane ? first : m_and_l(sp);
            const float f = scale_of(ml.x, M);
            s_part[c * parts + sp] = f;
            L += ml.x == -INFINITY ? ml.y : ml.y * f;
        }
        L = wave_sum(L);
        if (lane == 0) s_part[cols * parts + c] = L;
    }
    __syncthreads();
    for (int o = threadIdx.x; o < pairs; o += blockDim.x) {
        const int c = 2 * o / hd, d = 2 * o - c * hd;
        const float* from = parts0 + c * a.pstride + d;
        const float* f = s_part + c * parts;
        float A0 = 0.0f, A1 = 0.0f;
        int sp = 0;
        for (; sp + JOIN <= parts; sp += JOIN) {
            float2 x[JOIN];
#pragma unroll
            for (int i = 0; i < JOIN; i++) x[i] = load_coherent(from + (sp + i) * stride);
#pragma unroll
            for (int i = 0; i < JOIN; i++) A0 = fmaf(x[i].x, f[sp + i], A0), A1 = fmaf(x[i].y, f[sp + i], A1);
        }
        // the rest four at a time (past the last: the last again, times 0)
        for (; sp < parts; sp += 4) {
            float2 x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = load_coherent(from + min(sp + i, parts - 1) * stride);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float w = sp + i < parts ? f[sp + i] : 0.0f;
                A0 = fmaf(x[i].x, w, A0), A1 = fmaf(x[i].y, w, A1);
            }
        }
        float* out = a.out + ((int64_t)b * a.n_heads + h0 + c) * hd + d;
        const float L = s_part[cols * parts + c];
        out[0] = divided(A0, L);
        out[1] = divided(A1, L);
    }
}

// launch(kernel) with the kernel built for `chunks` runs of 16 dimensions.
template <int CH, class F>
void pick(int chunks, bool stream, F launch) {
    if (chunks == CH)
        stream ? launch(kv_q8_decode_kernel<CH, true>) : launch(kv_q8_decode_kernel<CH, false>);
    else if constexpr (CH < 16)
        pick<CH + 1>(chunks, stream, launch);
}

}  // namespace

hipError_t launch_kv_q8_decode(const KvQ8Decode& a, hipStream_t stream) {
    const int kv_mul = a.n_heads / a.c.kv_heads;
    const int groups = (kv_mul + KV_Q8_COLUMNS - 1) / KV_Q8_COLUMNS;
    const int64_t blocks = (int64_t)a.batch * a.num_splits * a.c.kv_heads * groups;
    const int chunks = a.c.hdp / 16;
    const size_t lds = kv_q8_decode_lds(a.n_heads, a.c.kv_heads, a.pstride, a.waves, a.num_splits);
    if ((a.ordered && (a.num_splits != 1 || a.batch > KV_Q8_ORDERED)) || a.waves < 1 || a.waves > 4 ||
        a.pstride < a.c.head_dim + 2 || a.pstride % 4 || chunks < 1 || chunks > 16 ||
        blocks > INT32_MAX || lds > KV_Q8_LDS)
        return hipErrorInvalidValue;
    const dim3 grid((unsigned)blocks), block(64 * a.waves);
    pick<1>(chunks, a.stream_kv, [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, lds, stream, a); });
    return hipGetLastError();
}

}  // namespace nitro
