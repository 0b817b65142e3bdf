// qz_ortho.h -- what the Newton-Schulz kernels (qz_ortho.hip) take from the C ABI (qz_abi.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

struct OrthoMatrix {
    int64_t rows, cols;
    const void* update;  // gradient (optimiser step) or update, `ld` elements between rows
    int64_t ld;
    void* out;           // orthogonalise: the result, `out_ld` elements between rows
    int64_t out_ld;
    float* momentum;     // optimiser step: [rows][cols]
    float* param;        // optimiser step: [rows][cols]
    float scale;         // optimiser step: factor of the learning rate
};
struct OrthoStep {
    int32_t dtype;       // of update / out: 0 float32, 1 bfloat16, 2 float16
    int32_t steps;
    int32_t muon;        // 0: out = orthogonalised update; 1: the optimiser step
    int32_t nesterov;
    float lr, momentum, weight_decay;
    const float* lr_dev; // or null: lr
};

namespace qzl {
int64_t ortho_workspace_bytes(const OrthoMatrix*, int count, const OrthoStep&);
hipError_t orthogonalize(const OrthoMatrix*, int count, const OrthoStep&, void* ws, hipStream_t);
}  // namespace qzl
