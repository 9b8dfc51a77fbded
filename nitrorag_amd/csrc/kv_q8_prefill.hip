// Causal prefill over an 8-bit paged cache on gfx950: packed chunks of prompts, each
// row over the keys up to its own position (the pass over the keys: kv_q8_attn.hpp).
#include <hip/hip_runtime.h>

#include "device_pool.hpp"
#include "kv_q8.hpp"
#include "kv_q8_attn.hpp"

namespace nitro {
namespace {

// out = A / L; 0 where no key was seen.
__device__ __forceinline__ float divided(float A, float L) { return L == 0.0f ? 0.0f : A / L; }

// A wave takes 16 query rows of one head as its columns; the workgroup's waves
// take consecutive ones and read the same K/V at about the same time.
template <int CH>
__global__ __launch_bounds__(256, CH <= 4 ? 3 : CH <= 8 ? 2 : 1) void kv_q8_prefill_kernel(KvQ8Prefill a) {
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
    const auto q = load_query<(CH + 3) / 4>(in ? a.q + (row * a.n_heads + h) * hd : nullptr, hd, a.qscale, g);
    State<CH> st;
#pragma unroll
    for (int t = 0; t < CH; t++) st.o[t] = f4{0.f, 0.f, 0.f, 0.f};
    const int last = seq.start_pos + min(first + 16, seq.num_tokens) - 1;  // the wave's last position
    auto page = [&](int i) { return trow[min(i, last >> 4)]; };
    // (the wave's last column sees most: it is the one that counts a bad page)
    attend<CH, false>(st, q, a.c, base, 0, last / KV_Q8_TILE + 1, 1, lane, page(col >> 2), page(g), page,
                      [&](int t) { return min(pos, last) + 1 - t * KV_Q8_TILE - 16 * g; });
    const float l = column_sum(st.l);
    if (!in) return;
    float* out = a.out + (row * a.n_heads + h) * hd;
#pragma unroll
    for (int t = 0; t < CH; t++) {
        const int dim = 16 * t + 4 * g;
        if (dim < hd)
            *reinterpret_cast<f4*>(out + dim) = f4{divided(st.o[t][0], l), divided(st.o[t][1], l),
                                                   divided(st.o[t][2], l), divided(st.o[t][3], l)};
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
