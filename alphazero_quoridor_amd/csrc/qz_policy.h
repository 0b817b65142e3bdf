// qz_policy.h -- the arguments of the policy-loss kernels (qz_policy.hip), as the C ABI (qz_abi.hip) hands them over.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

struct PolicyRows {
    const void* logits;      // [n] rows of `a` elements, `ld` elements apart
    int64_t ld;
    int64_t n;
    const int64_t* actions;  // [n]
    const void* legal;       // legal_kind 1: 32-bit words, 2: bytes; legal_ld in those units
    int64_t legal_ld;
    int32_t legal_kind;
    int32_t dtype;           // 0 float32, 1 bfloat16, 2 float16
    int32_t a;
    int64_t row0 = 0;        // first row of a launch
};
struct PolicyTerms {
    const float *advantages, *old_logp, *ref_logp, *weights;  // [n]; ref_logp, weights may be null
    const void* ref_logits;                                   // or null
    int64_t ref_ld;
    float clip_low, clip_high, kl_coef, entropy_coef, default_weight;
};
struct PolicyOut {
    float *logp, *kl, *entropy;  // [n]
    void* grad;                  // or null
    int64_t ld_grad;
    const float* scale;          // the gradient's factor, on the device; null = 1
    int32_t only_if_scaled;      // do nothing where *scale is 1
    double* parts;               // partial sums of the loss
};

namespace qzl {
int64_t policy_workspace_bytes(int64_t n, int a);
hipError_t action_logp(const PolicyRows&, float* logp, float* entropy, float* stats, void* ws, hipStream_t);
hipError_t action_logp_backward(const PolicyRows&, const float* stats, const float* entropy, const float* dlogp, const float* dentropy, void* grad,
                                int64_t ld_grad, hipStream_t);
hipError_t policy_loss(const PolicyRows&, const PolicyTerms&, PolicyOut, float* loss, void* ws, hipStream_t);
}  // namespace qzl
