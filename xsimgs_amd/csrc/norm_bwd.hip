// Group norm with an activation and dropout, channels last: the backward kernels. With xh = (x - mean) rstd,
// z = xh weight + bias and dz = v_y act'(z) times the draw's factor, over a sample's pixels
//   v_bias = sum dz,  v_weight = sum dz xh,
//   v_x = rstd (weight dz - mean_group(weight dz) - xh mean_group(weight dz xh)).
// A first pass leaves each workgroup's sums of dz and dz xh for each channel, and of their products with the weight
// for each group; a second joins the groups' (its own workgroups do, where they are few) and writes v_x, while
// some more of its workgroups join the channels'. Sums are added in a fixed order. No reference counterpart.

#include "xsg_norm.h"

namespace {

// A batch of U pixels of x and of v_y.
template <int DT, int V, int U, bool MASK> struct GradBatch {
    typedef Raw<V * ElementSize<DT>::value> Vec;
    Vec x[U], g[U];
    uint32_t in;
    XSG_DEV void fetch(const NormArgs& a, const NormPlace<V>& at, const NormPath<DT>& x_at, const NormPath<DT>& g_at, int64_t p) {
        in = norm_pixels<U, MASK>(a, at, p);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (in >> (16 + u) & 1) {
                x[u] = load_raw<DT, V>(x_at(p + u * a.ty));
                g[u] = load_raw<DT, V>(g_at(p + u * a.ty));
            }
    }
};

template <int DT, int V, int ACT, bool DROP, bool MASK>
__global__ __launch_bounds__(kNormThreads) void norm_sums_kernel(NormArgs a, const float4* __restrict__ stats,
                                                                 const void* __restrict__ v_y, float2* __restrict__ groups,
                                                                 float2* __restrict__ channels) {
    constexpr int U = kNormGradUnroll;
    constexpr bool AHEAD = norm_ahead(V * ElementSize<DT>::value);
    constexpr bool EXACT = DT == XSG_DTYPE_F32;
    extern __shared__ float2 s_sums[];   // [threads][V], then [channels]
    float2* const s_channel = s_sums + V * blockDim.x;
    const int t = threadIdx.x;
    const NormPlace<V> at(a, blockIdx.x, U * a.ty);
    const bool mine = at.r < a.ty;
    const NormPath<DT> x_at(a.x, at.b * a.batch_stride, a.pixel_stride, at.r, at.c0);
    const NormPath<DT> g_at(v_y, at.b * a.pixels * a.channels, a.channels, at.r, at.c0);
    const int64_t first = (at.b * a.pixels + at.r) * a.channels + at.c0;   // element, for the draws
    GradBatch<DT, V, U, MASK> now, next;
    now.fetch(a, at, x_at, g_at, at.p0);
    float mean[V], scale[V], bias[V], s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = mine ? at.c0 + j : 0;
        const float4 s = stats[at.b * a.groups + a.by_cg(c)];
        mean[j] = s.x;
        scale[j] = s.y * norm_param(a.weight, a.weight_dtype, c, 1.0f);
        bias[j] = norm_param(a.bias, a.bias_dtype, c, 0.0f);
        s1[j] = s2[j] = 0.0f;
    }
    const Draws draws(a.drop);
    for (int64_t p = at.p0; p < a.pixels; p += at.jump) {
        const bool more = p + at.jump < a.pixels;
        if (AHEAD && more) next.fetch(a, at, x_at, g_at, p + at.jump);
        NormDraws<DT, V> drawn(draws, a.channels, first + p * a.channels, (int64_t)a.ty * a.channels);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (DROP) drawn.draw(u);
            if (!(now.in >> (16 + u) & 1)) continue;
            float x[V], g[V];
            unpack<DT, V>(now.x[u], x);
            if (DROP) drawn.mask(now.g[u]);
            unpack<DT, V>(now.g[u], g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float e = x[j] - mean[j];
                float dz = g[j] * norm_act_slope<ACT, EXACT>(e * scale[j] + bias[j]);
                if (DROP) dz = drawn.one(dz, j);   // the factor comes at the end
                s1[j] += dz;
                s2[j] += dz * e;
            }
            if (DROP) __builtin_amdgcn_sched_barrier(0);   // several pixels' draws at once take too many registers
        }
        if (!more) break;
        if (AHEAD) now = next;
        else now.fetch(a, at, x_at, g_at, p + at.jump);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) s_sums[t * V + j] = make_float2(s1[j], s2[j]);
    __syncthreads();
    {
        const int l = norm_segment(blockDim.x, a.channels), lane = t & (l - 1);
        for (int c = t / l; c < a.channels; c += blockDim.x / l) {
            const int vec = c / V, first = vec * V + c - a.first_channel<V>(vec);
            float2 sum = make_float2(0.0f, 0.0f);
            for (int row = lane; row < a.ty; row += l) {
                const float2 e = s_sums[row * a.tx * V + first];
                sum.x += e.x;
                sum.y += e.y;
            }
            sum.x = segment_sum(sum.x, l) * a.drop.factor;
            sum.y = segment_sum(sum.y, l) * stats[at.b * a.groups + a.by_cg(c)].y * a.drop.factor;
            if (lane == 0) {
                if (channels) channels[(int64_t)blockIdx.x * a.channels + c] = sum;
                const float w = norm_param(a.weight, a.weight_dtype, c, 1.0f);
                s_channel[c] = make_float2(w * sum.x, w * sum.y);
            }
        }
    }
    if (!groups) return;
    __syncthreads();
    const int l = norm_segment(blockDim.x, a.groups), lane = t & (l - 1);
    for (int g = t / l; g < a.groups; g += blockDim.x / l) {
        float2 sum = make_float2(0.0f, 0.0f);
        for (int c = g * a.cg + lane; c < (g + 1) * a.cg; c += l) {
            sum.x += s_channel[c].x;
            sum.y += s_channel[c].y;
        }
        sum.x = segment_sum(sum.x, l);
        sum.y = segment_sum(sum.y, l);
        if (lane == 0) groups[(int64_t)blockIdx.x * a.groups + g] = sum;
    }
}

// Adds the entries first, first + step, ... of a column, eight on their way at a time.
XSG_DEV void add_parts(const float2* __restrict__ part, int columns, int64_t parts, int first, int step, double& x, double& y) {
    for (int64_t k0 = first; k0 < parts; k0 += 8 * step) {
        float2 m[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = part[(k0 + i * step < parts ? k0 + i * step : first) * columns];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k0 + i * step < parts) {
                x += m[i].x;
                y += m[i].y;
            }
    }
}

// One workgroup to a group of a sample, or to several in turn: the means of weight dz and weight dz xh, sums in 64 bits.
__global__ __launch_bounds__(256) void norm_means_kernel(int64_t all, int groups, int chunks, const float4* __restrict__ stats,
                                                         const float2* __restrict__ part, float2* __restrict__ means) {
    __shared__ double s_x[4], s_y[4];
    for (int64_t i = blockIdx.x; i < all; i += gridDim.x) {
        const int64_t b = i / groups;
        const float2* const p = part + b * chunks * groups + (i - b * groups);
        double x = 0.0, y = 0.0;
        add_parts(p, groups, chunks, threadIdx.x, 256, x, y);
        x = segment_sum(x, 64);
        y = segment_sum(y, 64);
        if ((threadIdx.x & 63) == 0) { s_x[threadIdx.x >> 6] = x; s_y[threadIdx.x >> 6] = y; }
        __syncthreads();
        if (threadIdx.x == 0) {
            const double inv = stats[i].z;
            means[i] = make_float2((float)((s_x[0] + s_x[1] + s_x[2] + s_x[3]) * inv),
                                   (float)((s_y[0] + s_y[1] + s_y[2] + s_y[3]) * inv));
        }
        __syncthreads();
    }
}

// The parameters' gradients of eight channels: sums over the rows of [rows, channels] pairs, in 64 bits. A workgroup
// of a multiple of 64 threads.
XSG_DEV void norm_columns(int64_t rows, int channels, int c0, const float2* __restrict__ part, float* __restrict__ v_weight,
                          float* __restrict__ v_bias) {
    __shared__ double s_x[kNormThreads], s_y[kNormThreads];
    const int t = threadIdx.x, c = c0 + (t & 7);
    double x = 0.0, y = 0.0;
    if (c < channels && t >> 3 < rows) add_parts(part + c, channels, rows, t >> 3, blockDim.x >> 3, x, y);
    s_x[t] = x;
    s_y[t] = y;
    __syncthreads();
    if (t < 8 && c < channels) {
        for (int k = t + 8; k < (int)blockDim.x; k += 8) { x += s_x[k]; y += s_y[k]; }
        if (v_bias) v_bias[c] = (float)x;
        if (v_weight) v_weight[c] = (float)y;
    }
}
__global__ __launch_bounds__(256) void norm_params_kernel(int64_t rows, int channels, const float2* __restrict__ part,
                                                          float* __restrict__ v_weight, float* __restrict__ v_bias) {
    norm_columns(rows, channels, 8 * (int)blockIdx.x, part, v_weight, v_bias);
}

// The first `param_blocks` workgroups add up the parameters' gradients, the others write v_x.
template <int DT, int V, int ACT, bool DROP, bool MASK, bool STREAM>
__global__ __launch_bounds__(kNormThreads) void norm_grad_kernel(NormArgs a, int param_blocks, const float4* __restrict__ stats,
                                                                 const void* __restrict__ v_y, const float2* __restrict__ groups,
                                                                 const float2* __restrict__ means,
                                                                 const float2* __restrict__ channels, void* __restrict__ v_x,
                                                                 float* __restrict__ v_weight, float* __restrict__ v_bias) {
    constexpr int U = kNormGradUnroll;
    constexpr bool AHEAD = norm_ahead(V * ElementSize<DT>::value);
    constexpr bool EXACT = DT == XSG_DTYPE_F32;
    if ((int)blockIdx.x < param_blocks)
        return norm_columns(a.batch * a.chunks, a.channels, 8 * (int)blockIdx.x, channels, v_weight, v_bias);
    extern __shared__ float2 s_group[];   // each group's means of weight dz and weight dz xh
    const NormPlace<V> at(a, gridDim.x - 1 - blockIdx.x, U * a.ty);   // from the end, which was read last
    const bool mine = at.r < a.ty;
    const NormPath<DT> x_at(a.x, at.b * a.batch_stride, a.pixel_stride, at.r, at.c0);
    const NormPath<DT> g_at(v_y, at.b * a.pixels * a.channels, a.channels, at.r, at.c0);
    const int64_t first = (at.b * a.pixels + at.r) * a.channels + at.c0;   // element, for the draws
    const NormPath<DT> to_at(v_x, at.b * a.pixels * a.channels, a.channels, at.r, at.c0);
    GradBatch<DT, V, U, MASK> now, next;
    now.fetch(a, at, x_at, g_at, at.p0);
    float mean[V], scale[V], bias[V], shift[V], slope[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        scale[j] = norm_param(a.weight, a.weight_dtype, mine ? at.c0 + j : 0, 1.0f);
        bias[j] = norm_param(a.bias, a.bias_dtype, mine ? at.c0 + j : 0, 0.0f);
    }
    const float2* mean_of = means + at.b * a.groups;
    if (a.join) {
        const int l = norm_segment(blockDim.x, a.groups), lane = threadIdx.x & (l - 1);
        const float2* const p = groups + at.b * a.chunks * a.groups;
        for (int g = threadIdx.x / l; g < a.groups; g += blockDim.x / l) {
            double x = 0.0, y = 0.0;
            add_parts(p + g, a.groups, a.chunks, lane, l, x, y);
            x = segment_sum(x, l);
            y = segment_sum(y, l);
            const double inv = stats[at.b * a.groups + g].z;
            if (lane == 0) s_group[g] = make_float2((float)(x * inv), (float)(y * inv));
        }
        __syncthreads();
        mean_of = s_group;
    }
    // v_x = scale dz - shift - (x - mean) slope
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int g = a.by_cg(mine ? at.c0 + j : 0);
        const float4 s = stats[at.b * a.groups + g];
        const float2 m = mean_of[g];
        mean[j] = s.x;
        scale[j] *= s.y;
        shift[j] = s.y * m.x;
        slope[j] = s.y * s.y * m.y;
    }
    const Draws draws(a.drop);
    for (int64_t p = at.p0; p < a.pixels; p += at.jump) {
        const bool more = p + at.jump < a.pixels;
        if (AHEAD && more) next.fetch(a, at, x_at, g_at, p + at.jump);
        NormDraws<DT, V> drawn(draws, a.channels, first + p * a.channels, (int64_t)a.ty * a.channels);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (DROP) drawn.draw(u);
            if (!(now.in >> u & 1)) continue;
            Raw<V * ElementSize<DT>::value> out = {};
            if (!MASK || (now.in >> (16 + u) & 1)) {
                float x[V], g[V];
                unpack<DT, V>(now.x[u], x);
                if (DROP) drawn.mask(now.g[u]);
                unpack<DT, V>(now.g[u], g);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float e = x[j] - mean[j];
                    float dz = g[j] * norm_act_slope<ACT, EXACT>(e * scale[j] + bias[j]);
                    if (DROP) dz = drawn.one(dz * a.drop.factor, j);
                    x[j] = scale[j] * dz - shift[j] - e * slope[j];
                }
                out = pack<DT, V>(x);
            }
            store_raw<DT, V, STREAM>(to_at(p + u * a.ty), 0, out);
            if (DROP) __builtin_amdgcn_sched_barrier(0);
        }
        if (!more) break;
        if (AHEAD) now = next;
        else now.fetch(a, at, x_at, g_at, p + at.jump);
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
    const int vector = norm_vector(d, true), size = d->dtype == XSG_DTYPE_F32 ? 4 : 2;
    norm_layout(a, vector, kNormGradUnroll, size, 3, 256);
    const int tiles = (a.channels + 7) / 8;
    if (a.batch * a.chunks > kNormBlocks)
        return xsg_fail(XSG_ERR_INVALID, "group_norm_act_bwd: too many samples (%lld)", (long long)a.batch);
    const int64_t parts = a.batch * a.chunks;
    float2* const groups = (float2*)workspace;
    float2* const channels = groups + parts * a.groups;
    float2* const means = channels + parts * a.channels;
    const bool params = v_weight || v_bias;
    const float4* const st = (const float4*)stats;
    with_dtype(d->dtype, [&](auto dt) {
        with_vector(vector, [&](auto vec) {
            with_norm_flags(d, a, [&](auto act, auto drop, auto mask) {
                constexpr int DT = decltype(dt)::value, V = decltype(vec)::value, ACT = decltype(act)::value;
                constexpr bool DROP = decltype(drop)::value, MASK = decltype(mask)::value;
                const unsigned threads = norm_threads(a);
                norm_sums_kernel<DT, V, ACT, DROP, MASK><<<(unsigned)parts, threads, sizeof(float2) * (V * threads + a.channels), s>>>(
                    a, st, v_y, v_x ? groups : nullptr, params ? channels : nullptr);
                // in a launch of their own where that of v_x has no workgroups left for them
                const bool apart = params && (!v_x || parts + tiles > kNormBlocks);
                if (apart) norm_params_kernel<<<(unsigned)tiles, 256, 0, s>>>(parts, a.channels, channels, v_weight, v_bias);
                if (!v_x) return;
                if (!a.join)
                    norm_means_kernel<<<norm_join_blocks(a), 256, 0, s>>>(a.batch * a.groups, a.groups, a.chunks, st, groups, means);
                const int param_blocks = params && !apart ? tiles : 0;
                const unsigned grid = (unsigned)parts + param_blocks;
                const size_t lds = a.join ? sizeof(float2) * a.groups : 0;
                if (norm_may_stream<DT, V>() && a.stream)
                    norm_grad_kernel<DT, V, ACT, DROP, MASK, norm_may_stream<DT, V>()><<<grid, threads, lds, s>>>(
                        a, param_blocks, st, v_y, groups, means, channels, v_x, v_weight, v_bias);
                else
                    norm_grad_kernel<DT, V, ACT, DROP, MASK, false><<<grid, threads, lds, s>>>(
                        a, param_blocks, st, v_y, groups, means, channels, v_x, v_weight, v_bias);
            });
        });
    });
    XSG_TRY_LAUNCH("group_norm_act_bwd");
    return XSG_OK;
}
