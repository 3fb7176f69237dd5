// Group norm of channels-last feature images with an activation and dropout behind it: what its forward and
// backward kernels share. A workgroup takes a run of pixels of one sample; its threads lie tx to a pixel, V
// consecutive channels each, and ty pixels side by side, so that its accesses are one run of memory.
#pragma once
#include "xsg_elements.h"
#include "xsg_random.h"

constexpr int kNormThreads = 512;    // most a workgroup has

struct NormArgs {
    const void* x;
    int64_t batch_stride, pixel_stride;
    int64_t batch, pixels;
    int channels, groups, cg;        // cg: channels of a group
    int tx, ty, nv;                  // threads to a pixel (as many vectors: nv), pixels side by side
    int64_t chunk;                   // pixels of a workgroup
    int chunks;                      // workgroups of a sample
    const uint8_t* mask;
    const void *weight, *bias;
    int weight_dtype, bias_dtype;
    float eps;
    DropArgs drop;

    // the last vector of a pixel ends with the last channel, so it repeats some where V does not divide the channels
    template <int V> XSG_HD int first_channel(int v) const { return v * V < channels - V ? v * V : channels - V; }
};

XSG_DEV float norm_param(const void* p, int dtype, int i, float otherwise) {
    if (!p) return otherwise;
    return dtype == XSG_DTYPE_F32 ? load_one<XSG_DTYPE_F32>(p, i)
         : dtype == XSG_DTYPE_BF16 ? load_one<XSG_DTYPE_BF16>(p, i) : load_one<XSG_DTYPE_F16>(p, i);
}

// 1 / (1 + exp(-z)). EXACT for float32 results; the others are rounded to 8 or 11 bits right after, so the
// hardware's exponential and reciprocal (1 ulp) do.
template <bool EXACT> XSG_DEV float norm_sigmoid(float z) {
    if (EXACT) return 1.0f / (1.0f + expf(-z));
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}
template <int ACT, bool EXACT> XSG_DEV float norm_act(float z) {
    if (ACT == XSG_ACT_RELU) return z < 0.0f ? 0.0f : z;
    if (ACT == XSG_ACT_SILU) return z * norm_sigmoid<EXACT>(z);
    if (ACT == XSG_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678f));
    return z;
}
template <int ACT, bool EXACT> XSG_DEV float norm_act_slope(float z) {
    if (ACT == XSG_ACT_RELU) return z > 0.0f ? 1.0f : z == z ? 0.0f : z;
    if (ACT == XSG_ACT_SILU) {
        const float s = norm_sigmoid<EXACT>(z);
        return s * (1.0f + z * (1.0f - s));
    }
    if (ACT == XSG_ACT_GELU) {
        const float e = EXACT ? expf(-0.5f * z * z) : __builtin_amdgcn_exp2f(z * z * -0.72134752f);
        return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * e * 0.39894228f;
    }
    return 1.0f;
}

// Segments of a wavefront's lanes (a power of two) share out `count` tasks of a workgroup: the largest that
// leaves a segment to each.
XSG_DEV int norm_segment(int threads, int count) {
    int l = 64;
    while (l > 1 && threads / l < count) l >>= 1;
    return l;
}
XSG_DEV float segment_sum(float x, int l) {
    for (int d = l >> 1; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}
XSG_DEV double segment_sum(double x, int l) {
    for (int d = l >> 1; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

// Host side: checks a description and lays the work out; `pixels_in_flight` of a thread, `workgroups` wanted.
int norm_args(const xsg_norm_desc* d, NormArgs& a, const char* who);
int norm_vector(const xsg_norm_desc* d);
void norm_layout(NormArgs& a, int vector, int pixels_in_flight, int64_t workgroups);

template <typename F> void with_norm_flags(const xsg_norm_desc* d, const NormArgs& a, F&& f) {
    const bool drop = a.drop.threshold != 0, mask = d->mask != nullptr;
    auto flags = [&](auto act) {
        if (drop && mask) f(act, std::true_type{}, std::true_type{});
        else if (drop) f(act, std::true_type{}, std::false_type{});
        else if (mask) f(act, std::false_type{}, std::true_type{});
        else f(act, std::false_type{}, std::false_type{});
    };
    switch (d->act) {
        case XSG_ACT_NONE: flags(std::integral_constant<int, XSG_ACT_NONE>{}); break;
        case XSG_ACT_RELU: flags(std::integral_constant<int, XSG_ACT_RELU>{}); break;
        case XSG_ACT_SILU: flags(std::integral_constant<int, XSG_ACT_SILU>{}); break;
        default: flags(std::integral_constant<int, XSG_ACT_GELU>{}); break;
    }
}
// vectors of 8, 4 or 1 elements
template <typename F> void with_vector(int vector, F&& f) {
    switch (vector) {
        case 8: f(std::integral_constant<int, 8>{}); break;
        case 4: f(std::integral_constant<int, 4>{}); break;
        default: f(std::integral_constant<int, 1>{}); break;
    }
}
