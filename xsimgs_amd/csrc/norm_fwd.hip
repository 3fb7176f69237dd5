// Group norm with an activation and dropout, channels last: the forward kernels and the argument checks. No
// reference counterpart.
#include <algorithm>
#include <limits.h>
#include <math.h>

#include "xsg_norm.h"

namespace {

// Mean and sum of squared deviations of a run of pixels, per group. Nothing is subtracted from a sum of squares:
// each thread takes its pixels a batch at a time, whose mean and deviations come from registers, and joins
// them to what it has by the rule of Chan, Golub and LeVeque ("Algorithms for computing the sample variance", 1983);
// so an offset that is large against the spread costs no digits. ONE: a vector lies in one group.
template <int DT, int V, bool ONE, bool MASK>
__global__ __launch_bounds__(kNormThreads) void norm_stats_kernel(NormArgs a, float4* __restrict__ part) {
    constexpr int NS = ONE ? 1 : V, U = V == 8 ? 4 : 8;
    extern __shared__ float s_stats[];   // (mean, deviations) of each thread and slot, then counts of each thread
    float2* const s_pair = (float2*)s_stats;
    float* const s_count = s_stats + 2 * NS * blockDim.x;
    const int t = threadIdx.x, v = t % a.tx, r = t / a.tx;
    const int64_t b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const int64_t p0 = chunk * a.chunk, p1 = min(p0 + a.chunk, a.pixels);
    float n = 0.0f, mean[NS], dev[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) mean[s] = dev[s] = 0.0f;

    const auto join = [&](const Raw<V * ElementSize<DT>::value>* raw, uint32_t in, int count, auto most) {
        constexpr int M = decltype(most)::value;
        if (MASK && count == 0) return;
        const float nb = (float)count, inv = 1.0f / nb;
        const float total = n + nb, share = nb / total;
        float sum[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) sum[s] = 0.0f;
#pragma unroll
        for (int u = 0; u < M; ++u) {
            float x[V];
            unpack<DT, V>(raw[u], x);
#pragma unroll
            for (int j = 0; j < V; ++j) sum[ONE ? 0 : j] += x[j];   // zeros of pixels out of the mask
        }
        float mb[NS], db[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) { mb[s] = sum[s] * (ONE ? inv * (1.0f / V) : inv); db[s] = 0.0f; }
#pragma unroll
        for (int u = 0; u < M; ++u) {
            if (MASK && !(in >> u & 1)) continue;
            float x[V];
            unpack<DT, V>(raw[u], x);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float e = x[j] - mb[ONE ? 0 : j];
                db[ONE ? 0 : j] += e * e;
            }
        }
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const float e = mb[s] - mean[s];
            mean[s] += e * share;
            dev[s] += db[s] + e * e * (n * share * (ONE ? V : 1));
        }
        n = total;
    };

    if (r < a.ty) {
        const int c0 = a.first_channel<V>(v);
        const uint8_t* const mask = MASK ? a.mask + b * a.pixels : nullptr;
        const int64_t x0 = b * a.batch_stride + c0;
        int64_t p = p0 + r;
        for (; p + (U - 1) * a.ty < p1; p += U * a.ty) {
            Raw<V * ElementSize<DT>::value> raw[U];
            uint32_t in = (1u << U) - 1;
            if (MASK) {
                in = 0;
#pragma unroll
                for (int u = 0; u < U; ++u) in |= (uint32_t)(mask[p + u * a.ty] != 0) << u;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                raw[u] = {};
                if (!MASK || (in >> u & 1)) raw[u] = load_raw<DT, V>(a.x, x0 + (p + u * a.ty) * a.pixel_stride);
            }
            join(raw, in, MASK ? __popc(in) : U, std::integral_constant<int, U>{});
        }
        for (; p < p1; p += a.ty) {
            if (MASK && !mask[p]) continue;
            const auto raw = load_raw<DT, V>(a.x, x0 + p * a.pixel_stride);
            join(&raw, 1, 1, std::integral_constant<int, 1>{});
        }
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) s_pair[t * NS + s] = make_float2(mean[s], dev[s]);
    s_count[t] = ONE ? n * V : n;
    __syncthreads();

    // a segment of lanes joins a group's entries: ty rows of its vectors (ONE) or channels
    const int l = norm_segment(blockDim.x, a.groups), lane = t & (l - 1);
    const int width = ONE ? a.cg / V : a.cg, entries = width * a.ty;
    for (int g = t / l; g < a.groups; g += blockDim.x / l) {
        const auto at = [&](int e, int& thread) {
            const int row = e / width, c = g * width + e % width;
            if (ONE) {
                thread = row * a.tx + c;
                return s_pair[thread];
            }
            const int vec = c / V;
            thread = row * a.tx + vec;
            return s_pair[thread * NS + c - a.first_channel<V>(vec)];
        };
        float count = 0.0f, sum = 0.0f;
        for (int e = lane; e < entries; e += l) {
            int thread;
            const float2 m = at(e, thread);
            count += s_count[thread];
            sum += s_count[thread] * m.x;
        }
        count = segment_sum(count, l);
        sum = segment_sum(sum, l);
        const float mu = count > 0.0f ? sum / count : 0.0f;
        float d = 0.0f;
        for (int e = lane; e < entries; e += l) {
            int thread;
            const float2 m = at(e, thread);
            d += m.y + s_count[thread] * (m.x - mu) * (m.x - mu);
        }
        d = segment_sum(d, l);
        if (lane == 0) part[(int64_t)blockIdx.x * a.groups + g] = make_float4(count, mu, d, 0.0f);
    }
}

// The parts of a sample's group joined, in 64 bits: one wavefront to a group.
__global__ __launch_bounds__(256) void norm_join_kernel(int64_t n_groups, int groups, int chunks, double eps,
                                                        const float4* __restrict__ part, float4* __restrict__ stats) {
    const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (i >= n_groups) return;
    const int lane = threadIdx.x & 63;
    const float4* const p = part + i / groups * chunks * groups + i % groups;
    double n = 0.0, sum = 0.0;
    for (int k = lane; k < chunks; k += 64) {
        const float4 e = p[(int64_t)k * groups];
        n += e.x;
        sum += (double)e.x * e.y;
    }
    n = segment_sum(n, 64);
    sum = segment_sum(sum, 64);
    const double mean = n > 0.0 ? sum / n : 0.0;
    double d = 0.0;
    for (int k = lane; k < chunks; k += 64) {
        const float4 e = p[(int64_t)k * groups];
        if (e.x > 0.0f) d += e.z + e.x * (e.y - mean) * (e.y - mean);
    }
    d = segment_sum(d, 64);
    if (lane == 0) {
        const double inv = n > 0.0 ? 1.0 / n : 0.0;
        stats[i] = make_float4((float)mean, (float)(1.0 / sqrt(d * inv + eps)), (float)inv, 0.0f);
    }
}

template <int DT, int V, int ACT, bool DROP, bool MASK>
__global__ __launch_bounds__(kNormThreads) void norm_apply_kernel(NormArgs a, const float4* __restrict__ stats,
                                                                  void* __restrict__ y) {
    constexpr int U = 4;
    constexpr bool EXACT = DT == XSG_DTYPE_F32;
    const int t = threadIdx.x, v = t % a.tx, r = t / a.tx;
    if (r >= a.ty) return;
    const int64_t b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const int64_t p0 = chunk * a.chunk, p1 = min(p0 + a.chunk, a.pixels);
    const int c0 = a.first_channel<V>(v);
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
        Raw<V * ElementSize<DT>::value> raw[U];
        bool in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) in[u] = p + u * a.ty < p1;
        bool kept[U];
#pragma unroll
        for (int u = 0; u < U; ++u) kept[u] = in[u] && (!MASK || mask[p + u * a.ty] != 0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            raw[u] = {};
            if (kept[u]) raw[u] = load_raw<DT, V>(a.x, x0 + (p + u * a.ty) * a.pixel_stride);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!in[u]) break;
            const int64_t at = y0 + (p + u * a.ty) * a.channels;
            Raw<V * ElementSize<DT>::value> out = {};
            if (!MASK || kept[u]) {
                float x[V];
                unpack<DT, V>(raw[u], x);
                const uint32_t keep = DROP ? draws.keep((uint64_t)at, V) : 0;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    x[j] = norm_act<ACT, EXACT>((x[j] - mean[j]) * scale[j] + bias[j]);
                    if (DROP) x[j] = keep >> j & 1 ? x[j] * a.drop.factor : 0.0f;
                }
                out = pack<DT, V>(x);
            }
            store_raw<DT, V>(y, at, out);
        }
    }
}

constexpr int64_t kStatsGroups = 1024;   // workgroups of a pass

}  // namespace

int norm_vector(const xsg_norm_desc* d) {
    // vectors of 16 bytes; eight float32 where a vector then holds a whole block of draws, or a workgroup the channels
    if (d->dtype != XSG_DTYPE_F32) return d->channels >= 8 ? 8 : d->channels >= 4 ? 4 : 1;
    if (d->channels > 4 * kNormThreads || (d->drop.p > 0.0 && d->channels % 8 == 0)) return 8;
    return d->channels >= 4 ? 4 : 1;
}

int norm_args(const xsg_norm_desc* d, NormArgs& a, const char* who) {
    if (!d) return xsg_fail(XSG_ERR_INVALID, "%s: null description", who);
    if (d->dtype < XSG_DTYPE_F32 || d->dtype > XSG_DTYPE_F16) return xsg_fail(XSG_ERR_INVALID, "%s: unknown type %d", who, d->dtype);
    if (d->batch < 0 || d->pixels < 0) return xsg_fail(XSG_ERR_INVALID, "%s: negative size", who);
    if (d->channels < 1 || d->channels > XSG_NORM_MAX_CHANNELS)
        return xsg_fail(XSG_ERR_INVALID, "%s: 1 to %d channels, not %d", who, XSG_NORM_MAX_CHANNELS, d->channels);
    if (d->groups < 1 || d->channels % d->groups)
        return xsg_fail(XSG_ERR_INVALID, "%s: %d groups do not divide %d channels", who, d->groups, d->channels);
    if (d->act < XSG_ACT_NONE || d->act > XSG_ACT_GELU) return xsg_fail(XSG_ERR_INVALID, "%s: unknown activation %d", who, d->act);
    if (!(d->eps >= 0.0)) return xsg_fail(XSG_ERR_INVALID, "%s: eps must not be negative", who);
    for (const int w : {d->weight ? d->weight_dtype : d->dtype, d->bias ? d->bias_dtype : d->dtype})
        if (w != XSG_DTYPE_F32 && w != d->dtype)
            return xsg_fail(XSG_ERR_INVALID, "%s: weight and bias are float32 or of x's type", who);
    if (d->batch > 0 && d->pixels > 0) {
        if (!d->x) return xsg_fail(XSG_ERR_INVALID, "%s: null tensor", who);
        if (d->batch_stride < 0 || d->pixel_stride < 0) return xsg_fail(XSG_ERR_INVALID, "%s: negative stride", who);
        // sizes that 64-bit offsets in bytes and the launches hold
        if (d->batch > INT_MAX || d->pixels > ((int64_t)1 << 45) / d->channels / d->batch ||
            d->pixel_stride > ((int64_t)1 << 60) / d->pixels || d->batch_stride > ((int64_t)1 << 60) / d->batch)
            return xsg_fail(XSG_ERR_INVALID, "%s: too large", who);
    }
    a = {};
    a.x = d->x;
    a.batch_stride = d->batch_stride; a.pixel_stride = d->pixel_stride;
    a.batch = d->batch; a.pixels = d->pixels;
    a.channels = d->channels; a.groups = d->groups; a.cg = d->channels / d->groups;
    a.mask = d->mask;
    a.weight = d->weight; a.bias = d->bias;
    a.weight_dtype = d->weight_dtype; a.bias_dtype = d->bias_dtype;
    a.eps = (float)d->eps;
    return drop_args(&d->drop, a.drop, who);
}

void norm_layout(NormArgs& a, int vector, int in_flight, int64_t workgroups) {
    a.nv = (a.channels + vector - 1) / vector;
    a.tx = a.nv;
    // about 256 threads, of which as few as possible idle in the last wavefront
    double best = 0.0;
    for (int ty = std::max(1, 256 / a.tx); ty * a.tx <= kNormThreads; ++ty) {
        const double used = (double)(ty * a.tx) / ((ty * a.tx + 63) / 64 * 64);
        if (used > best) { best = used; a.ty = ty; }
    }
    const int64_t step = (int64_t)a.ty * in_flight;
    const int64_t wanted = std::max<int64_t>(1, std::min((a.pixels + step - 1) / step, (workgroups + a.batch - 1) / a.batch));
    a.chunk = ((a.pixels + wanted - 1) / wanted + step - 1) / step * step;
    a.chunks = (int)((a.pixels + a.chunk - 1) / a.chunk);
}

static unsigned norm_threads(const NormArgs& a) { return (unsigned)((a.tx * a.ty + 63) / 64 * 64); }

extern "C" size_t xsg_group_norm_act_workspace_bytes(const xsg_norm_desc* d, int backward) {
    NormArgs a;
    if (norm_args(d, a, "group_norm_act") != XSG_OK || d->batch == 0 || d->pixels == 0) return 0;
    if (backward) {
        norm_layout(a, norm_vector(d), 2, kStatsGroups);
        return sizeof(float2) * (size_t)a.channels * (size_t)(a.batch * a.chunks + a.batch);
    }
    norm_layout(a, norm_vector(d), 4, kStatsGroups);
    return sizeof(float4) * (size_t)a.groups * (size_t)(a.batch * a.chunks);
}

extern "C" int xsg_group_norm_act_fwd(const xsg_norm_desc* d, void* y, float* stats, void* workspace, xsg_stream_t stream) {
    NormArgs a;
    if (const int rc = norm_args(d, a, "group_norm_act_fwd")) return rc;
    if (a.batch == 0 || a.pixels == 0) return XSG_OK;
    if (!y || !stats || !workspace) return xsg_fail(XSG_ERR_INVALID, "group_norm_act_fwd: null tensor");
    if (const int rc = xsg_check_workspace(workspace, "group_norm_act_fwd")) return rc;
    if ((uintptr_t)stats % 16) return xsg_fail(XSG_ERR_INVALID, "group_norm_act_fwd: stats must be 16-byte aligned");
    const int vector = norm_vector(d);
    norm_layout(a, vector, 4, kStatsGroups);
    if (a.batch * a.chunks > INT_MAX / 2) return xsg_fail(XSG_ERR_INVALID, "group_norm_act_fwd: too large");
    const hipStream_t s = (hipStream_t)stream;
    const unsigned grid = (unsigned)(a.batch * a.chunks), threads = norm_threads(a);
    const bool one = a.cg % vector == 0;
    with_dtype(d->dtype, [&](auto dt) {
        with_vector(vector, [&](auto vec) {
            constexpr int DT = decltype(dt)::value, V = decltype(vec)::value;
            const size_t lds = sizeof(float) * threads * (2 * (one ? 1 : V) + 1);
            float4* const part = (float4*)workspace;
            if (one && a.mask) norm_stats_kernel<DT, V, true, true><<<grid, threads, lds, s>>>(a, part);
            else if (one) norm_stats_kernel<DT, V, true, false><<<grid, threads, lds, s>>>(a, part);
            else if (a.mask) norm_stats_kernel<DT, V, false, true><<<grid, threads, lds, s>>>(a, part);
            else norm_stats_kernel<DT, V, false, false><<<grid, threads, lds, s>>>(a, part);
            const int64_t n_groups = a.batch * a.groups;
            norm_join_kernel<<<xsg_blocks(n_groups, 4), 256, 0, s>>>(n_groups, a.groups, a.chunks, d->eps, part, (float4*)stats);
            with_norm_flags(d, a, [&](auto act, auto drop, auto mask) {
                norm_apply_kernel<DT, V, decltype(act)::value, decltype(drop)::value, decltype(mask)::value>
                    <<<grid, threads, 0, s>>>(a, (const float4*)stats, y);
            });
        });
    });
    XSG_TRY_LAUNCH("group_norm_act_fwd");
    return XSG_OK;
}
