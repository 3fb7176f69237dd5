// Group norm with an activation and dropout, channels last: the backward kernels. With xh = (x - mean) rstd,
// z = xh weight + bias and dz = v_y act'(z) times the draw's factor, over a sample's pixels
//   v_bias = sum dz,  v_weight = sum dz xh,
//   v_x = rstd (weight dz - mean_group(weight dz) - xh mean_group(weight dz xh)).
// A first pass leaves each workgroup's sums of dz and dz xh for each channel, a second joins them, a third
// writes v_x; sums are added in a fixed order. No reference counterpart.
#include <algorithm>
#include <limits.h>

#include "xsg_norm.h"

namespace {

constexpr int64_t kSumsGroups = 1024;

template <int DT, int V, int ACT, bool DROP, bool MASK>
__global__ __launch_bounds__(kNormThreads) void norm_sums_kernel(NormArgs a, const float4* __restrict__ stats,
                                                                 const void* __restrict__ v_y, float2* __restrict__ part) {
    constexpr int U = 2;
    constexpr bool EXACT = DT == XSG_DTYPE_F32;
    extern __shared__ float2 s_sums[];   // [rows][tx][V]
    const int t = threadIdx.x, v = t % a.tx, r = t / a.tx;
    const int64_t b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const int64_t p0 = chunk * a.chunk, p1 = min(p0 + a.chunk, a.pixels);
    const int c0 = a.first_channel<V>(v);
    float s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0f;
    if (r < a.ty) {
        float mean[V], scale[V], bias[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float4 s = stats[b * a.groups + (c0 + j) / a.cg];
            mean[j] = s.x;
            scale[j] = s.y * norm_param(a.weight, a.weight_dtype, c0 + j, 1.0f);
            bias[j] = norm_param(a.bias, a.bias_dtype, c0 + j, 0.0f);
        }
        const Draws draws(a.drop);
        const uint8_t* const mask = MASK ? a.mask + b * a.pixels : nullptr;
        const int64_t x0 = b * a.batch_stride + c0, y0 = b * a.pixels * a.channels + c0;
        for (int64_t p = p0 + r; p < p1; p += U * a.ty) {
            Raw<V * ElementSize<DT>::value> rx[U], rg[U];
            bool kept[U];
#pragma unroll
            for (int u = 0; u < U; ++u) kept[u] = p + u * a.ty < p1;
            if (MASK) {
#pragma unroll
                for (int u = 0; u < U; ++u) kept[u] = kept[u] && mask[p + u * a.ty] != 0;
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (kept[u]) {
                    rx[u] = load_raw<DT, V>(a.x, x0 + (p + u * a.ty) * a.pixel_stride);
                    rg[u] = load_raw<DT, V>(v_y, y0 + (p + u * a.ty) * a.channels);
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (kept[u]) {
                    float x[V], g[V];
                    unpack<DT, V>(rx[u], x);
                    unpack<DT, V>(rg[u], g);
                    const uint32_t keep = DROP ? draws.keep((uint64_t)(y0 + (p + u * a.ty) * a.channels), V) : 0;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float e = x[j] - mean[j];
                        float dz = g[j] * norm_act_slope<ACT, EXACT>(e * scale[j] + bias[j]);
                        if (DROP) dz = keep >> j & 1 ? dz * a.drop.factor : 0.0f;
                        s1[j] += dz;
                        s2[j] += dz * e;
                    }
                }
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) s_sums[t * V + j] = make_float2(s1[j], s2[j]);
    __syncthreads();
    const int l = norm_segment(blockDim.x, a.channels), lane = t & (l - 1);
    for (int c = t / l; c < a.channels; c += blockDim.x / l) {
        const int vec = c / V, at = vec * V + c - a.first_channel<V>(vec);
        float2 sum = make_float2(0.0f, 0.0f);
        for (int row = lane; row < a.ty; row += l) {
            const float2 e = s_sums[row * a.tx * V + at];
            sum.x += e.x;
            sum.y += e.y;
        }
        sum.x = segment_sum(sum.x, l);
        sum.y = segment_sum(sum.y, l);
        if (lane == 0)
            part[(int64_t)blockIdx.x * a.channels + c] = make_float2(sum.x, sum.y * stats[b * a.groups + c / a.cg].y);
    }
}

// Sums over `rows` rows of [rows, channels] pairs, for the eight channels from c0 on, in 64 bits: out(channel, pair).
template <typename F>
XSG_DEV void column_sums(const float2* __restrict__ rows, int64_t n, int channels, int c0, F out) {
    __shared__ double s_x[256], s_y[256];
    const int t = threadIdx.x, c = c0 + (t & 7);
    double x = 0.0, y = 0.0;
    if (t < 256 && c < channels)
        for (int64_t i = t >> 3; i < n; i += 32) {
            const float2 e = rows[i * channels + c];
            x += e.x;
            y += e.y;
        }
    if (t < 256) { s_x[t] = x; s_y[t] = y; }
    __syncthreads();
    if (t < 8 && c < channels) {
        for (int k = t + 8; k < 256; k += 8) { x += s_x[k]; y += s_y[k]; }
        out(c, make_float2((float)x, (float)y));
    }
}

__global__ __launch_bounds__(256) void norm_columns_kernel(int64_t rows, int channels, const float2* __restrict__ part,
                                                           float2* __restrict__ total) {
    const int tiles = (channels + 7) / 8;
    const int64_t b = blockIdx.x / tiles;
    column_sums(part + b * rows * channels, rows, channels, 8 * (int)(blockIdx.x % tiles),
                [&](int c, float2 e) { total[b * channels + c] = e; });
}

// total over the samples as the parameters' gradients, eight channels a workgroup
__global__ __launch_bounds__(256) void norm_params_kernel(int64_t batch, int channels, const float2* __restrict__ total,
                                                          float* __restrict__ v_weight, float* __restrict__ v_bias) {
    column_sums(total, batch, channels, 8 * (int)blockIdx.x, [&](int c, float2 e) {
        if (v_bias) v_bias[c] = e.x;
        if (v_weight) v_weight[c] = e.y;
    });
}

template <int DT, int V, int ACT, bool DROP, bool MASK>
__global__ __launch_bounds__(kNormThreads) void norm_grad_kernel(NormArgs a, const float4* __restrict__ stats,
                                                                 const void* __restrict__ v_y,
                                                                 const float2* __restrict__ total, void* __restrict__ v_x) {
    constexpr int U = 2;
    constexpr bool EXACT = DT == XSG_DTYPE_F32;
    extern __shared__ float2 s_group[];   // each group's means of weight dz and weight dz xh
    const int t = threadIdx.x, v = t % a.tx, r = t / a.tx;
    const int64_t b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const int64_t p0 = chunk * a.chunk, p1 = min(p0 + a.chunk, a.pixels);
    {
        const int l = norm_segment(blockDim.x, a.groups), lane = t & (l - 1);
        for (int g = t / l; g < a.groups; g += blockDim.x / l) {
            float2 sum = make_float2(0.0f, 0.0f);
            for (int c = g * a.cg + lane; c < (g + 1) * a.cg; c += l) {
                const float w = norm_param(a.weight, a.weight_dtype, c, 1.0f);
                const float2 e = total[b * a.channels + c];
                sum.x += w * e.x;
                sum.y += w * e.y;
            }
            sum.x = segment_sum(sum.x, l);
            sum.y = segment_sum(sum.y, l);
            const float inv = stats[b * a.groups + g].z;
            if (lane == 0) s_group[g] = make_float2(sum.x * inv, sum.y * inv);
        }
    }
    __syncthreads();
    if (r >= a.ty) return;
    const int c0 = a.first_channel<V>(v);
    // v_x = scale dz - shift - (x - mean) slope
    float mean[V], scale[V], bias[V], shift[V], slope[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int g = (c0 + j) / a.cg;
        const float4 s = stats[b * a.groups + g];
        mean[j] = s.x;
        scale[j] = s.y * norm_param(a.weight, a.weight_dtype, c0 + j, 1.0f);
        bias[j] = norm_param(a.bias, a.bias_dtype, c0 + j, 0.0f);
        shift[j] = s.y * s_group[g].x;
        slope[j] = s.y * s.y * s_group[g].y;
    }
    const Draws draws(a.drop);
    const uint8_t* const mask = MASK ? a.mask + b * a.pixels : nullptr;
    const int64_t x0 = b * a.batch_stride + c0, y0 = b * a.pixels * a.channels + c0;
    for (int64_t p = p0 + r; p < p1; p += U * a.ty) {
        Raw<V * ElementSize<DT>::value> rx[U], rg[U];
        bool in[U], kept[U];
#pragma unroll
        for (int u = 0; u < U; ++u) in[u] = p + u * a.ty < p1;
#pragma unroll
        for (int u = 0; u < U; ++u) kept[u] = in[u] && (!MASK || mask[p + u * a.ty] != 0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (kept[u]) {
                rx[u] = load_raw<DT, V>(a.x, x0 + (p + u * a.ty) * a.pixel_stride);
                rg[u] = load_raw<DT, V>(v_y, y0 + (p + u * a.ty) * a.channels);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!in[u]) break;
            const int64_t at = y0 + (p + u * a.ty) * a.channels;
            Raw<V * ElementSize<DT>::value> out = {};
            if (kept[u]) {
                float x[V], g[V];
                unpack<DT, V>(rx[u], x);
                unpack<DT, V>(rg[u], g);
                const uint32_t keep = DROP ? draws.keep((uint64_t)at, V) : 0;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float e = x[j] - mean[j];
                    float dz = g[j] * norm_act_slope<ACT, EXACT>(e * scale[j] + bias[j]);
                    if (DROP) dz = keep >> j & 1 ? dz * a.drop.factor : 0.0f;
                    x[j] = scale[j] * dz - shift[j] - e * slope[j];
                }
                out = pack<DT, V>(x);
            }
            store_raw<DT, V>(v_x, at, out);
        }
    }
}

__global__ __launch_bounds__(256) void norm_zero_kernel(int channels, float* v_weight, float* v_bias) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= channels) return;
    if (v_weight) v_weight[c] = 0.0f;
    if (v_bias) v_bias[c] = 0.0f;
}

}  // namespace

extern "C" int xsg_group_norm_act_bwd(const xsg_norm_desc* d, const float* stats, const void* v_y, void* v_x,
                                      float* v_weight, float* v_bias, void* workspace, xsg_stream_t stream) {
    NormArgs a;
    if (const int rc = norm_args(d, a, "group_norm_act_bwd")) return rc;
    const hipStream_t s = (hipStream_t)stream;
    if (!v_x && !v_weight && !v_bias) return XSG_OK;
    if (a.batch == 0 || a.pixels == 0) {
        if (v_weight || v_bias) norm_zero_kernel<<<xsg_blocks(a.channels, 256), 256, 0, s>>>(a.channels, v_weight, v_bias);
        XSG_TRY_LAUNCH("group_norm_act_bwd");
        return XSG_OK;
    }
    if (!stats || !v_y || !workspace) return xsg_fail(XSG_ERR_INVALID, "group_norm_act_bwd: null tensor");
    if (const int rc = xsg_check_workspace(workspace, "group_norm_act_bwd")) return rc;
    if ((uintptr_t)stats % 16) return xsg_fail(XSG_ERR_INVALID, "group_norm_act_bwd: stats must be 16-byte aligned");
    const int vector = norm_vector(d);
    norm_layout(a, vector, 2, kSumsGroups);
    if (a.batch * a.chunks > INT_MAX / 2 || a.batch * ((a.channels + 7) / 8) > INT_MAX / 2)
        return xsg_fail(XSG_ERR_INVALID, "group_norm_act_bwd: too large");
    const unsigned grid = (unsigned)(a.batch * a.chunks), threads = (unsigned)((a.tx * a.ty + 63) / 64 * 64);
    float2* const part = (float2*)workspace;
    float2* const total = part + a.batch * a.chunks * a.channels;
    const float4* const st = (const float4*)stats;
    with_dtype(d->dtype, [&](auto dt) {
        with_vector(vector, [&](auto vec) {
            with_norm_flags(d, a, [&](auto act, auto drop, auto mask) {
                constexpr int DT = decltype(dt)::value, V = decltype(vec)::value, ACT = decltype(act)::value;
                constexpr bool DROP = decltype(drop)::value, MASK = decltype(mask)::value;
                norm_sums_kernel<DT, V, ACT, DROP, MASK><<<grid, threads, sizeof(float2) * V * threads, s>>>(a, st, v_y, part);
                norm_columns_kernel<<<(unsigned)(a.batch * ((a.channels + 7) / 8)), 256, 0, s>>>(a.chunks, a.channels, part, total);
                if (v_weight || v_bias)
                    norm_params_kernel<<<(unsigned)((a.channels + 7) / 8), 256, 0, s>>>(a.batch, a.channels, total, v_weight, v_bias);
                if (v_x)
                    norm_grad_kernel<DT, V, ACT, DROP, MASK><<<grid, threads, sizeof(float2) * a.groups, s>>>(a, st, v_y, total, v_x);
            });
        });
    });
    XSG_TRY_LAUNCH("group_norm_act_bwd");
    return XSG_OK;
}
