// C ABI of rows held in 8 bits and their products with Q8_0 matrices.  Declared in
// include/nitro_paged_attn.h.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <memory>

#include "capi_common.hpp"
#include "device_pool.hpp"
#include "nitro_paged_attn.h"
#include "row8.hpp"

using namespace nitro;

// One matrix, or a gated pair (the gate first), in the tile layout.
struct nitro_q8_weights {
    DeviceBuffer<uint8_t> tiled[2];
    int32_t n = 0, d = 0, device = 0;
    bool gated = false;
};

namespace {

hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }
bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

void check_rows(const void* codes, const float* scales, int32_t rows, int32_t n) {
    require(codes != nullptr && scales != nullptr, ERR_INVALID_ARGUMENT, "null pointer");
    require(rows > 0 && n > 0, ERR_INVALID_ARGUMENT, "rows and n must be positive");
    require(n <= 1 << 30, ERR_UNSUPPORTED, "rows of more than 2^30 entries");
}

int current_device() {
    int dev = 0;
    hip_check(hipGetDevice(&dev), "hipGetDevice");
    return dev;
}

}  // namespace

extern "C" {

int nitro_rms_norm_row8(const float* x, const float* residual, const float* weight, double eps, float* sum,
                        int8_t* codes, float* scales, int32_t rows, int32_t n, void* stream) {
    return guarded([&] {
        check_rows(codes, scales, rows, n);
        require(x != nullptr && weight != nullptr, ERR_INVALID_ARGUMENT, "null pointer");
        require(eps > 0.0 && eps <= 1e300, ERR_INVALID_ARGUMENT, "eps must be positive and finite");
        hip_check(launch_row8_norm({x, residual, weight, sum, codes, scales, rows, n, eps}, as_stream(stream)),
                  "rms_norm_row8 launch");
    });
}

int nitro_row8_quantize(const float* x, int8_t* codes, float* scales, int32_t rows, int32_t n, void* stream) {
    return guarded([&] {
        check_rows(codes, scales, rows, n);
        require(x != nullptr, ERR_INVALID_ARGUMENT, "null pointer");
        hip_check(launch_row8_norm({x, nullptr, nullptr, nullptr, codes, scales, rows, n, 0.0}, as_stream(stream)),
                  "row8_quantize launch");
    });
}

int nitro_row8_read(const int8_t* codes, const float* scales, float* x, int32_t rows, int32_t n, void* stream) {
    return guarded([&] {
        check_rows(codes, scales, rows, n);
        require(x != nullptr, ERR_INVALID_ARGUMENT, "null pointer");
        hip_check(launch_row8_read(codes, scales, x, rows, n, as_stream(stream)), "row8_read launch");
    });
}

int nitro_q8_weights_create(const void* w, const void* w_gate, int32_t n, int32_t d, nitro_q8_weights** out) {
    return guarded([&] {
        require(out != nullptr, ERR_INVALID_ARGUMENT, "null output pointer");
        *out = nullptr;
        require(w != nullptr, ERR_INVALID_ARGUMENT, "null weights");
        require(n > 0 && d > 0, ERR_INVALID_ARGUMENT, "n and d must be positive");
        require(n % 32 == 0, ERR_INVALID_ARGUMENT, "n must be a multiple of 32 (Q8 block)");
        require(n <= 1 << 30 && d <= 1 << 29, ERR_UNSUPPORTED, "more than 2^30 columns or 2^29 rows");
        require(aligned(w, 4) && aligned(w_gate, 4), ERR_INVALID_ARGUMENT, "weights must be 4-byte aligned");
        auto m = std::make_unique<nitro_q8_weights>();
        m->n = n, m->d = d, m->gated = w_gate != nullptr, m->device = current_device();
        const void* from[2] = {w_gate ? w_gate : w, w};
        const size_t bytes = q8_tiled_bytes(d, n);
        // whichever stream wrote w, and whichever will read the copy
        hip_check(hipDeviceSynchronize(), "hipDeviceSynchronize");
        for (int i = 0; i < (m->gated ? 2 : 1); i++) {
            hip_check(hipMalloc((void**)&m->tiled[i].ptr, bytes), "hipMalloc(weights)");
            m->tiled[i].count = bytes;
            hip_check(launch_q8_tile(from[i], m->tiled[i].ptr, d, n, nullptr), "q8 tile launch");
        }
        hip_check(hipDeviceSynchronize(), "q8 tile");
        *out = m.release();
    });
}

int nitro_q8_weights_destroy(nitro_q8_weights* weights) {
    if (!weights) return NITRO_OK;
    return guarded([&] {
        int now = 0;  // the launches to wait for are on the weights' device
        const bool other = hipGetDevice(&now) == hipSuccess && now != weights->device;
        if (other) (void)hipSetDevice(weights->device);
        (void)hipDeviceSynchronize();
        delete weights;
        if (other) (void)hipSetDevice(now);
    });
}

int nitro_row8_matmul(const nitro_q8_weights* weights, const int8_t* codes, const float* scales, const float* bias,
                      const float* residual, float* out, int32_t rows, int32_t activation, void* stream) {
    return guarded([&] {
        require(weights != nullptr, ERR_INVALID_ARGUMENT, "null weights");
        check_rows(codes, scales, rows, weights->n);
        require(out != nullptr, ERR_INVALID_ARGUMENT, "null pointer");
        require(aligned(codes, 16), ERR_INVALID_ARGUMENT, "codes must be 16-byte aligned");
        require(activation >= NITRO_ACT_NONE && activation <= NITRO_ACT_GELU_TANH, ERR_INVALID_ARGUMENT,
                "activation must be one of NITRO_ACT_*");
        require(current_device() == weights->device, ERR_INVALID_ARGUMENT,
                "the weights belong to another device than the current one");
        Row8Matmul a{};
        a.w[0] = weights->tiled[0].ptr, a.w[1] = weights->tiled[1].ptr;
        a.out[0] = out, a.d[0] = weights->d;
        a.mats = 1, a.gated = weights->gated;
        a.codes = codes, a.scales = scales, a.bias = bias, a.residual = residual;
        a.rows = rows, a.n = weights->n, a.activation = activation;
        hip_check(launch_row8_matmul(a, as_stream(stream)), "row8_matmul launch");
    });
}

int nitro_row8_tile(int32_t rows, int32_t n, int32_t d, int32_t d_kv, int32_t gated, int32_t* tile) {
    return guarded([&] {
        require(tile != nullptr, ERR_INVALID_ARGUMENT, "null output pointer");
        require(rows > 0 && n > 0 && d > 0 && d_kv >= 0 && n % 32 == 0, ERR_INVALID_ARGUMENT,
                "rows, n and d must be positive, d_kv not negative, n a multiple of 32");
        require(n <= 1 << 30 && d <= 1 << 29 && d_kv <= 1 << 29, ERR_UNSUPPORTED, "more than 2^30 columns or 2^29 rows");
        require(!gated || d_kv == 0, ERR_INVALID_ARGUMENT, "a pair has no d_kv");
        Row8Matmul a{};
        a.d[0] = d, a.d[1] = a.d[2] = d_kv;
        a.mats = d_kv ? 3 : 1, a.gated = gated != 0;
        a.rows = rows, a.n = n;
        require(row8_matmul_tile(a, tile), ERR_UNSUPPORTED, "no kernel takes a product of these sizes");
    });
}

}  // extern "C"
