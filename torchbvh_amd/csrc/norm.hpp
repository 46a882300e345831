// Group norm with an activation over channels-last rows (see norm.hip).
#pragma once

#include "tbvh_internal.hpp"

namespace tbvh {

enum Activation { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

struct NormArgs {
    const void* x = nullptr;          // (rows, channels)
    const int64_t* offsets = nullptr; // (clouds + 1), or null: equal clouds
    const void* weight = nullptr;     // (channels), of x's type or fp32
    const void* bias = nullptr;
    int64_t rows = 0;
    int clouds = 0, channels = 0, groups = 0;
    float eps = 0.0f;
    int activation = kNone;
    void* y = nullptr;
    float* mean = nullptr;            // (clouds, groups)
    float* rstd = nullptr;
    const void* grad = nullptr;       // (rows, channels)
    void* dx = nullptr;
    void* dweight = nullptr;
    void* dbias = nullptr;
    float* parts = nullptr;           // scratch: norm_scratch floats
};

// Row slices of a cloud that are reduced apart.
int norm_parts(int64_t rows, int clouds, int channels);
// Floats of scratch of one call.
int64_t norm_scratch(int64_t rows, int clouds, int channels, int groups);

hipError_t launch_norm(const NormArgs& a, bool bf16, bool wide_weights, hipStream_t stream);
hipError_t launch_norm_backward(const NormArgs& a, bool bf16, bool wide_weights, hipStream_t stream);

}  // namespace tbvh
