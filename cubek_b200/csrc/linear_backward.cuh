// Arguments of the activation-gradient and bias-gradient kernels (linear_backward.cu).
#pragma once

#include "linear_kernels.cuh"

namespace qk {

struct ActBackwardArgs {
    const void *grad;   // [rows, n]
    long long grad_stride;
    const void *pre;    // [rows, n]; unread with QK_ACT_IDENTITY
    long long pre_stride;
    void *dz, *dz2;     // up to two places for the products, rounded to F; nullptr: not written
    long long dz_stride, dz2_stride;
    void *grad_bias;    // [experts, n]; nullptr: no sums
    long long grad_bias_stride, grad_bias_expert;
    float *partial;     // [experts, slices, n] where slices > 1
    int slices;
    int n, rows, act, experts, vec;
    const void *offsets;
    int offsets64;
};

int bias_slices(long long rows, long long n, int experts);
cudaError_t launch_activation_backward(int fdt, const ActBackwardArgs &a, const LaunchCfg &cfg, cudaStream_t stream, int *launches);
// Whether x [rows, ..] cannot be loaded as it lies: its rows do not start on 16 bytes.
bool product_needs_aligned_rows(long long rows, const void *x, long long stride);
// Whether the tiles of a product can be numbered; of `a`: rows, feats, k, experts and offsets.
bool product_tiles_fit(bool backward, const LinearArgs &a);
cudaError_t launch_linear_product(int fdt, int kind, bool backward, const LinearArgs &a, const LaunchCfg &cfg, cudaStream_t stream);

}  // namespace qk
