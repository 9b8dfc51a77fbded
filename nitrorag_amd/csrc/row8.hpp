// Rows held in 8 bits and what their kernels are launched with.
//
// A row y of n fp32 numbers is held as n int8 codes and one fp32 scale: with a =
// max |y|, scale = a / 127 and code = rint(y * inv), inv = 127 / a (both quotients
// fp32, the product exact, ties to even); the value is code * scale.  Rows with
// a < 2^-100 are zeros; one with an infinity or a NaN has a NaN for its scale.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace nitro {

// codes, scales = the rows y = x, or with NORM y = (x + residual) * weight / rms.
struct Row8Norm {
    const float* x;
    const float* residual;  // or null
    const float* weight;    // null: no norm
    float* sum;             // x + residual, or null
    int8_t* codes;
    float* scales;
    int32_t rows, n;
    double eps;
};
hipError_t launch_row8_norm(const Row8Norm& a, hipStream_t stream);
// x = the values held.
hipError_t launch_row8_read(const int8_t* codes, const float* scales, float* x, int rows, int n, hipStream_t stream);

// Up to three matrices over the same rows (wq, wk, wv), each with an output of its own;
// gated: two of d[0] rows with one output, act(first) * second.
struct Row8Matmul {
    const uint8_t* w[3];  // tile layout (Q8Tiled)
    float* out[3];
    int32_t d[3];
    int32_t mats;
    bool gated;
    const int8_t* codes;
    const float* scales;
    const float* bias;      // one matrix: [d], gated: [2][d]; or null
    const float* residual;  // of the first output; or null
    int32_t rows, n, activation;
};
hipError_t launch_row8_matmul(const Row8Matmul& a, hipStream_t stream);
// nitro_row8_tile: of a's sizes (rows, n, d, mats, gated); false where no kernel takes them.
bool row8_matmul_tile(const Row8Matmul& a, int32_t* tile);

}  // namespace nitro
