// Causal prefill over an 8-bit paged cache on gfx950: packed chunks of prompts, each
// row over the keys up to its own position (the products and the softmax:
// kv_q8_attn.hpp).
//
// Bound by the vector instructions around the products, 350 per tile of 64 keys and 16
// rows at head size 128 beside 48 matrix ones: 79% of the SIMDs' cycles, the matrix
// cores are busy in 38%.  8192 tokens at 32 x 128: 975-1060 us (520-560 TFLOP/s of
// fp32-grade work; cards differ), four chunks of 384 to 512 behind up to 4096 cached
// tokens at 32/8 x 128 130-140 us, 8 prompts of 128 to 1024 at 12 x 64 21-23 us.  (Four
// tiles under one maximum rather than two: 8% fewer vector instructions, V a run of 16
// dimensions at a time, 1029 us.)  Builds that hold part of their operands in scratch,
// in bytes a lane: head sizes 20-32 52, 36-48 112, 100-112 56, 132-176 432, 212-224 48,
// 228-240 140.  2048 tokens at 16/8 heads of 112, 128, 160 and 192 take 48, 47, 156 and
// 86 us.
#include <hip/hip_runtime.h>

#include "device_pool.hpp"
#include "kv_q8.hpp"
#include "kv_q8_attn.hpp"

namespace nitro {
namespace {

// Tiles 0 .. end - 1 (end > 0) of the keys of one table row, two at a time.  K and V
// come from the caches here (a prompt's rows read them again and again), and what
// bounds the pass is the vector instructions around the products: V loads go out as
// the scores are made, the next K's around the V products, so that two waves per SIMD
// have the registers they need.  Of tile t the lane's column sees seen(t) tokens of
// page lane / 16.  page(i): table entry i (any i).
template <int CH, class Page, class Seen>
__device__ __forceinline__ void attend_pairs(State<CH>& st, const Query<(CH + 3) / 4>& q, const KvQ8& c,
                                             const uint8_t* base, int end, int lane, Page page, Seen seen) {
    const int g = lane >> 4, sub = (lane & 15) >> 2;
    KTile<CH> k[2] = {no_k<CH>(), no_k<CH>()};
    VTile<CH> v[2];
    int kp[2], vp[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        kp[h] = page(4 * h + sub), vp[h] = page(4 * h + g);
        load_k<CH, false>(k[h], record(c, base, kp[h]), record(c, base, vp[h]), lane);
    }
    int t = 0;
    auto pair = [&](auto more) {
        f4 s[2][4];
        float top = -INFINITY, scales[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            load_v<CH, false>(v[h], record(c, base, vp[h]), lane);
            const int keys = seen_on(c, vp[h], t + h < end ? seen(t + h) : 0, lane);
            top = fmaxf(top, scores<CH>(s[h], k[h], q, keys));
            scales[h] = k[h].vs;
            if (more) kp[h] = page(4 * (t + 2 + h) + sub), vp[h] = page(4 * (t + 2 + h) + g);
        }
        const Weights<2> w = weigh<CH, 2>(st, s, top, q.scale, scales);
        if (more) load_k<CH, false>(k[0], record(c, base, kp[0]), record(c, base, vp[0]), lane);
        add_values<CH, 2>(st, v, w);
        if (more) load_k<CH, false>(k[1], record(c, base, kp[1]), record(c, base, vp[1]), lane);
        t += 2;
    };
    while (t + 2 < end) pair(std::true_type());
    pair(std::false_type());  // (on its own: a load that may be missing costs waits for all of them)
}

// Query rows first .. + 16 of an item, one head.
template <int CH>
__device__ __forceinline__ void attend_item(const KvQ8Prefill& a, int item, int h, int wave, int lane) {
    const int b = a.work[2 * item];
    const PrefillSeq seq = a.seqs[b];
    const int col = lane & 15, g = lane >> 4, hd = a.c.head_dim;
    const int first = a.work[2 * item + 1] + 16 * wave;  // of the wave's rows, in the chunk
    if (first >= seq.num_tokens) return;
    const int kv_h = h / (a.n_heads / a.c.kv_heads);
    const int32_t* trow = a.tables + (int64_t)b * a.max_pages;
    const uint8_t* base = a.c.cache + a.c.layer_off + (int64_t)kv_h * a.c.record;

    const bool in = first + col < seq.num_tokens;
    const int64_t row = (int64_t)seq.row_off + first + col;
    const int pos = seq.start_pos + first + col;
    const int last = seq.start_pos + min(first + 16, seq.num_tokens) - 1;  // the wave's last position
    const auto q = query_of(load_row<(CH + 3) / 4>(in ? a.q + (row * a.n_heads + h) * hd : nullptr, hd, g), a.qscale);
    State<CH> st;
#pragma unroll
    for (int t = 0; t < CH; t++) st.o[t] = f4{0.f, 0.f, 0.f, 0.f};
    auto page = [&](int i) { return trow[min(i, last >> 4)]; };
    // (the wave's last column sees most: it is the one that counts a bad page)
    attend_pairs<CH>(st, q, a.c, base, last / KV_Q8_TILE + 1, lane, page,
                     [&](int t) { return min(pos, last) + 1 - t * KV_Q8_TILE - 16 * g; });
    const float l = column_sum(st.l), inv = l == 0.0f ? 0.0f : 1.0f / l;  // 0 where no key was seen
    if (!in) return;
    float* out = a.out + (row * a.n_heads + h) * hd;
#pragma unroll
    for (int t = 0; t < CH; t++) {
        const int dim = 16 * t + 4 * g;
        if (dim < hd) *reinterpret_cast<f4*>(out + dim) = st.o[t] * inv;
    }
}

// A wave takes 16 query rows of one head as its columns; the workgroup's waves take
// consecutive ones and read the same K/V at about the same time.  (Rows of a wave
// dealt out to two or four waves by their keys, so that a launch with few rows has
// more to balance: never faster, 24.4 and 29.7 us against 24.2 for 8 prompts at 12 x
// 64, 147 and 158 against 145 for four chunks at 32/8 x 128.)
template <int CH>
__global__ __launch_bounds__(256, CH <= 4 ? 3 : CH <= 8 ? 2 : 1) void kv_q8_prefill_kernel(KvQ8Prefill a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // The items come longest first.  Workgroups go round the CUs in order of their
    // index, so every second round goes backwards: the CU that has the longest of one
    // round has the shortest of the next.  As many workgroups as items and heads, but
    // for a captured launch that is replayed over a later batch.
    const int total = a.seqs[0].work_items * a.n_heads;
    for (int block = blockIdx.x; block < total; block += gridDim.x) {
        const int round = block / a.num_cus, place = block - round * a.num_cus;
        const int in_round = min(a.num_cus, total - round * a.num_cus);
        const int w = round * a.num_cus + (round % 2 ? in_round - 1 - place : place);
        const int item = w / a.n_heads;
        int here = lane;
        asm volatile("" : "+v"(here));  // (what follows from the lane is made anew, not kept in registers)
        attend_item<CH>(a, item, w - item * a.n_heads, wave, here);
        if (total - block <= (int)gridDim.x) break;
    }
}

// launch(kernel) with the kernel built for `chunks` runs of 16 dimensions.
template <int CH, class F>
void pick(int chunks, F launch) {
    if (chunks == CH)
        launch(kv_q8_prefill_kernel<CH>);
    else if constexpr (CH < 16)
        pick<CH + 1>(chunks, launch);
}

}  // namespace

hipError_t launch_kv_q8_prefill(const KvQ8Prefill& a, hipStream_t stream) {
    const int64_t blocks = (int64_t)a.work_items * a.n_heads;
    if (a.item_rows != 64 || a.c.hdp > 256 || blocks > INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid((unsigned)blocks), block(256);
    pick<1>(a.c.hdp / 16, [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a); });
    return hipGetLastError();
}

}  // namespace nitro
