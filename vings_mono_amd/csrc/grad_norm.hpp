// Pieces shared by the kernels that need the global norm of a set of gradients before they can
// write anything (grad_norm.hip, sparse_adam.hip): how partial results of workgroups are formed
// and joined in a fixed order, and the clipping coefficient.
#pragma once
#include "common.hpp"

namespace vings {

// What is accumulated: squares for the 2-norm, the largest magnitude for the max-norm.  Both are
// held in 64 bits: a square of any 32-bit float is exact there and neither overflows nor
// vanishes, and the vector units convert and multiply-add doubles faster than HBM delivers floats
// (806 MB of bfloat16: 2-norm 142 us, max-norm, whose compares and selects are more, 148).
enum NormKind { NORM_2 = 0, NORM_MAX = 1 };

template <int KIND>
__device__ __forceinline__ double norm_join(double a, double b) {
    if (KIND == NORM_2) return a + b;
    return (b > a || b != b) ? b : a;       // a NaN on either side stays
}

template <int KIND>
__device__ __forceinline__ void norm_take(double& acc, float x) {
    if (KIND == NORM_2) {
        const double d = (double)x;
        acc = __builtin_fma(d, d, acc);
    } else {
        acc = norm_join<KIND>(acc, (double)fabsf(x));
    }
}

// Joins one value per lane over a workgroup of at most 1024 lanes (whole waves); every lane
// receives the result.  `scratch` holds 16 doubles.
template <int KIND>
__device__ __forceinline__ double norm_join_block(double v, double* scratch) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = norm_join<KIND>(v, __shfl_xor(v, o, 64));
    const int waves = blockDim.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = scratch[0];
    for (int k = 1; k < waves; ++k) v = norm_join<KIND>(v, scratch[k]);
    return v;
}

// The norm from `n` partial results: the same order in every workgroup and every run.
template <int KIND>
__device__ __forceinline__ float norm_of_partials(const double* __restrict__ partial, int n,
                                                  double* scratch) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) v = norm_join<KIND>(v, partial[i]);
    v = norm_join_block<KIND>(v, scratch);
    return (float)(KIND == NORM_2 ? sqrt(v) : v);
}

// min(1, max_norm / (norm + 1e-6)); a NaN norm gives NaN, an infinite one 0.
__device__ __forceinline__ float clip_coefficient(float norm, float max_norm) {
    const double c = (double)max_norm / ((double)norm + 1e-6);
    return c >= 1.0 ? 1.0f : (float)c;
}

}  // namespace vings
