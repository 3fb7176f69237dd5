// Group norm with an activation and dropout, channels last: the forward kernels and the argument checks. No
// reference counterpart.
#include <algorithm>
#include <limits.h>
#include <math.h>

#include "xsg_norm.h"

namespace {

constexpr int kStatsUnroll = 4;      // pixels in flight in a thread

// Mean and sum of squared deviations of a workgroup's pixels, per group. A thread takes its pixels a batch at a time:
// with m the mean and D the squared deviations of the n values so far, and s1, s2 the sums of x - m and of its square over
// a batch, the joint mean is m + s1 / (n + nb) and the joint D is D + s2 - s1^2 / (n + nb) (the earlier values' deviations
// add up to 0). s1^2 is at most nb s2, so no more than the bits of n / (n + nb) cancel, however large the mean is
// against the spread; the first batch takes its own mean for m. ONE: a vector lies in one group.
template <int DT, int V, bool ONE, bool MASK>
__global__ __launch_bounds__(kNormThreads) void norm_stats_kernel(NormArgs a, float2* __restrict__ part,
                                                                  float* __restrict__ counts) {
    constexpr int NS = ONE ? 1 : V, U = kStatsUnroll;
    typedef Raw<V * ElementSize<DT>::value> Vec;
    extern __shared__ float s_stats[];   // (mean, deviations) of each thread and slot, then counts of each thread
    float2* const s_pair = (float2*)s_stats;
    float* const s_count = s_stats + 2 * NS * blockDim.x;
    const NormPlace<V> at(a, blockIdx.x, U * a.ty);
    const int t = threadIdx.x;
    float n = 0.0f, mean[NS], dev[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) mean[s] = dev[s] = 0.0f;

    const auto add = [&](const Vec* raw, uint32_t in, int count, auto most) {
        constexpr int M = decltype(most)::value;
        if (MASK && count == 0) return;
        const float nb = (float)count;
        if (n == 0.0f) {
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
#pragma unroll
            for (int s = 0; s < NS; ++s) mean[s] = sum[s] / (nb * (ONE ? V : 1));
        }
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0f;
#pragma unroll
        for (int u = 0; u < M; ++u) {
            float x[V];
            unpack<DT, V>(raw[u], x);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float e = x[j] - mean[ONE ? 0 : j];
                if (MASK) e = in >> u & 1 ? e : 0.0f;
                s1[j] += e;
                s2[j] += e * e;
            }
        }
        n += nb;
        const float inv = 1.0f / (n * (ONE ? V : 1));
        if (ONE) {
#pragma unroll
            for (int j = 1; j < V; ++j) { s1[0] += s1[j]; s2[0] += s2[j]; }
        }
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const float e = s1[s] * inv;
            mean[s] += e;
            dev[s] += s2[s] - s1[s] * e;
        }
    };

    if (at.r < a.ty) {
        const NormPath<DT> x(a.x, at.b * a.batch_stride, a.pixel_stride, at.r, at.c0);
        const uint8_t* const mask = MASK ? a.mask + at.b * a.pixels + at.r : nullptr;
        const int step = U * a.ty;
        int64_t p = at.p0;
        for (; p + step <= a.pixels; p += at.jump) {
            Vec raw[U];
            uint32_t in = (1u << U) - 1;
            if (MASK) {
                in = 0;
#pragma unroll
                for (int u = 0; u < U; ++u) in |= (uint32_t)(mask[p + u * a.ty] != 0) << u;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                raw[u] = {};
                if (!MASK || (in >> u & 1)) raw[u] = load_raw<DT, V>(x(p + u * a.ty));
            }
            add(raw, in, MASK ? __popc(in) : U, std::integral_constant<int, U>{});
        }
        // a last batch of fewer pixels
        for (int u = 0; u < U && p + u * a.ty + at.r < a.pixels; ++u) {
            if (MASK && !mask[p + u * a.ty]) continue;
            const Vec raw = load_raw<DT, V>(x(p + u * a.ty));
            add(&raw, 1, 1, std::integral_constant<int, 1>{});
        }
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) s_pair[t * NS + s] = make_float2(mean[s], dev[s]);
    s_count[t] = ONE ? n * V : n;
    __syncthreads();

    // a segment of lanes joins a group's entries: ty rows of its vectors (ONE) or channels
    const int l = norm_segment(blockDim.x, a.groups), lane = t & (l - 1);
    const int width = ONE ? a.cg / V : a.cg, entries = width * a.ty;
    const float inv_width = ONE ? a.inv_cg * V : a.inv_cg;
    const int row0 = (int)((lane + 0.5f) * inv_width), col0 = lane - row0 * width;
    const int rows = (int)((l + 0.5f) * inv_width), cols = l - rows * width;
    for (int g = t / l; g < a.groups; g += blockDim.x / l) {
        // (row, col) of entry lane, lane + l, ...
        const auto each = [&](auto f) {
            int row = row0, col = col0;
            for (int e = lane; e < entries; e += l) {
                const int c = g * width + col, vec = ONE ? c : c / V, thread = row * a.tx + vec;
                f(s_pair[ONE ? thread : thread * NS + c - a.first_channel<V>(vec)], s_count[thread]);
                row += rows;
                col += cols;
                if (col >= width) { col -= width; ++row; }
            }
        };
        float count = 0.0f, sum = 0.0f;
        each([&](float2 m, float k) { count += k; sum += k * m.x; });
        segment_sums(count, sum, l);
        const float mu = count > 0.0f ? sum / count : 0.0f;
        // deviations about that mean, and what its own rounding left of their sum
        float d = 0.0f, left = 0.0f;
        each([&](float2 m, float k) {
            const float e = m.x - mu;
            d += m.y + k * e * e;
            left += k * e;
        });
        segment_sums(d, left, l);
        const float shift = count > 0.0f ? left / count : 0.0f;
        if (lane == 0) part[(int64_t)blockIdx.x * a.groups + g] = make_float2(mu + shift, d - left * shift);
        if (lane == 0 && g == 0) counts[blockIdx.x] = count;
    }
}

// A group's chunks joined in 64 bits, about the mean of the first chunk that has any pixels: squares of differences of
// means, in digits to spare (with that chunk of one pixel and n values behind it, they cancel to 1 / n at worst).
struct NormSums {
    double n, s1, s2, d;
    XSG_DEV NormSums() : n(0.0), s1(0.0), s2(0.0), d(0.0) {}
    XSG_DEV void add(float2 m, float count, float about) {
        const double e = (double)m.x - about;
        n += count;
        s1 += count * e;
        s2 += count * e * e;
        d += m.y;
    }
    // what cancels is divided in 64 bits too: a reciprocal of 32 leaves 6e-8 of s2
    XSG_DEV float4 stats(float about, float eps) const {
        if (!(n > 0.0)) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);   // nothing in the mask: zeros, also without eps
        const double shift = s1 / n;
        const float inv = 1.0f / (float)n;
        float var = (float)(d + s2 - s1 * shift) * inv;
        if (var < 0.0f) var = 0.0f;   // a NaN stays
        return make_float4((float)(about + shift), 1.0f / sqrtf(var + eps), inv, 0.0f);
    }
    // the mean of the first chunk that has any pixels (of an empty one it is 0, which may be far away): a segment of l lanes
    template <bool MASK> XSG_DEV static float about(const float2* __restrict__ part, const float* __restrict__ counts, int groups,
                                                    int parts, int lane, int l) {
        if (!MASK || counts[0] > 0.0f) return part[0].x;
        int k = lane;
        while (k < parts && !(counts[k] > 0.0f)) k += l;
        for (int d = l >> 1; d; d >>= 1) k = min(k, __shfl_xor(k, d));
        return k < parts ? part[(int64_t)k * groups].x : 0.0f;
    }
    // entries first, first + step, ... of a group's parts, eight on their way at a time
    XSG_DEV void add_parts(const float2* __restrict__ part, const float* __restrict__ counts, int groups, int parts,
                           int first, int step, float about) {
        for (int k0 = first; k0 < parts; k0 += 8 * step) {
            float2 m[8];
            float c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int k = k0 + i * step < parts ? k0 + i * step : first;
                m[i] = part[(int64_t)k * groups];
                c[i] = counts[k];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k0 + i * step < parts) add(m[i], c[i], about);
        }
    }
};

// One workgroup to a group of a sample (1080p x 64: 5 us, as long as a launch takes), or to several in turn where a launch
// does not have as many.
template <bool MASK>
__global__ __launch_bounds__(256) void norm_join_kernel(int64_t all, int groups, int chunks, float eps,
                                                        const float2* __restrict__ part, const float* __restrict__ counts,
                                                        float4* __restrict__ stats) {
    __shared__ double s_sum[4][4];
    for (int64_t i = blockIdx.x; i < all; i += gridDim.x) {
        const int64_t b = i / groups;
        const float2* const p = part + b * chunks * groups + (i - b * groups);
        const float* const c = counts + b * chunks;
        const float about = NormSums::about<MASK>(p, c, groups, chunks, threadIdx.x & 63, 64);   // the same in each wavefront
        NormSums sum;
        sum.add_parts(p, c, groups, chunks, threadIdx.x, 256, about);
        double* const mine = s_sum[threadIdx.x >> 6];
        const double n = segment_sum(sum.n, 64), s1 = segment_sum(sum.s1, 64), s2 = segment_sum(sum.s2, 64), d = segment_sum(sum.d, 64);
        if ((threadIdx.x & 63) == 0) { mine[0] = n; mine[1] = s1; mine[2] = s2; mine[3] = d; }
        __syncthreads();
        if (threadIdx.x == 0) {
            NormSums all_sums;
            for (int w = 0; w < 4; ++w) {
                all_sums.n += s_sum[w][0];
                all_sums.s1 += s_sum[w][1];
                all_sums.s2 += s_sum[w][2];
                all_sums.d += s_sum[w][3];
            }
            stats[i] = all_sums.stats(about, eps);
        }
        __syncthreads();
    }
}

template <int DT, int V, int ACT, bool DROP, bool MASK, bool STREAM>
__global__ __launch_bounds__(kNormThreads) void norm_apply_kernel(NormArgs a, int parts, const float2* __restrict__ part,
                                                                  const float* __restrict__ counts,
                                                                  float4* __restrict__ stats, void* __restrict__ y) {
    constexpr int U = norm_apply_unroll(V * ElementSize<DT>::value);
    constexpr bool AHEAD = norm_ahead(V * ElementSize<DT>::value);
    constexpr bool EXACT = DT == XSG_DTYPE_F32;
    typedef Raw<V * ElementSize<DT>::value> Vec;
    extern __shared__ float4 s_group[];
    const NormPlace<V> at(a, gridDim.x - 1 - blockIdx.x, U * a.ty);   // from the end, which was read last
    const bool mine = at.r < a.ty;
    const NormPath<DT> x_at(a.x, at.b * a.batch_stride, a.pixel_stride, at.r, at.c0);
    const NormPath<DT> y_at(y, at.b * a.pixels * a.channels, a.channels, at.r, at.c0);
    const int64_t first = (at.b * a.pixels + at.r) * a.channels + at.c0;   // element, for the draws
    const auto fetch = [&](int64_t p, Vec* raw) {
        const uint32_t in = norm_pixels<U, MASK>(a, at, p);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            raw[u] = {};
            if (in >> (16 + u) & 1) raw[u] = load_raw<DT, V>(x_at(p + u * a.ty));
        }
        return in;
    };
    Vec raw[U], next[U];
    uint32_t in = fetch(at.p0, raw), in_next = 0;

    float mean[V], scale[V], bias[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        scale[j] = norm_param(a.weight, a.weight_dtype, mine ? at.c0 + j : 0, 1.0f);
        bias[j] = norm_param(a.bias, a.bias_dtype, mine ? at.c0 + j : 0, 0.0f);
    }
    const float4* group = stats + at.b * a.groups;
    if (a.join) {
        const int l = norm_segment(blockDim.x, a.groups), lane = threadIdx.x & (l - 1);
        const float2* const p = part + at.b * parts * a.groups;
        for (int g = threadIdx.x / l; g < a.groups; g += blockDim.x / l) {
            NormSums sum;
            const float about = NormSums::about<MASK>(p + g, counts + at.b * parts, a.groups, parts, lane, l);
            sum.add_parts(p + g, counts + at.b * parts, a.groups, parts, lane, l, about);
            sum.n = segment_sum(sum.n, l);
            sum.s1 = segment_sum(sum.s1, l);
            sum.s2 = segment_sum(sum.s2, l);
            sum.d = segment_sum(sum.d, l);
            if (lane == 0) {
                s_group[g] = sum.stats(about, a.eps);
                if (at.chunk == 0) stats[at.b * a.groups + g] = s_group[g];
            }
        }
        __syncthreads();
        group = s_group;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float4 s = group[a.by_cg(mine ? at.c0 + j : 0)];
        mean[j] = s.x;
        scale[j] *= s.y;
    }
    const Draws draws(a.drop);
    const float kept = 1.0f / a.drop.factor;
    // every lane goes through every batch: draws are shared between them
    for (int64_t p = at.p0; p < a.pixels; p += at.jump) {
        const bool more = p + at.jump < a.pixels;
        if (AHEAD && more) in_next = fetch(p + at.jump, next);
        NormDraws<DT, V> drawn(draws, a.channels, first + p * a.channels, (int64_t)a.ty * a.channels);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (DROP) drawn.draw(u);
            if (!(in >> u & 1)) continue;
            Vec out = {};
            if (!MASK || (in >> (16 + u) & 1)) {
                float x[V];
                unpack<DT, V>(raw[u], x);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    x[j] = norm_act<ACT, EXACT, DROP>(fmaf(x[j] - mean[j], scale[j], bias[j]), a.drop.factor, kept);
                    if (DROP) x[j] = drawn.one(x[j], j);
                }
                out = pack<DT, V>(x);
                if (DROP) drawn.mask(out);
            }
            store_raw<DT, V, STREAM>(y_at(p + u * a.ty), 0, out);
            if (DROP) __builtin_amdgcn_sched_barrier(0);   // several pixels' draws at once take too many registers
        }
        if (!more) break;
        if (AHEAD) {
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = next[u];
            in = in_next;
        } else {
            in = fetch(p + at.jump, raw);
        }
    }
}

// Workgroups of a pass: as many as 64 KB of x to each 256 threads make, eight of those to a CU at most (six images of 92
// MB: 2048 863 us forward and backward, 1024 960) and two at least (31 MB: 512 77 us, 1024 87, whose results take
// longer to join).
constexpr int64_t kThreadBytes = 256, kMostThreads = 2048 * 256, kFewThreads = 512 * 256;
// Results go around the last-level cache where a call moves more than half of it: they would push out what the next pass
// or the next call reads (265 MB of x: statistics 73 -> 46 us; 132 MB: 37 -> 22, also with a kernel that reads the
// result right behind, 126 -> 121 us the two).
constexpr int64_t kCacheBytes = (int64_t)128 << 20;

}  // namespace

int norm_vector(const xsg_norm_desc* d, bool draws) {
    const int c = d->channels;
    if (d->dtype != XSG_DTYPE_F32) return c >= 8 ? 8 : c >= 4 ? 4 : 1;
    if (c > 4 * kNormThreads) return 8;   // a workgroup would not have the threads
    // With draws: a wavefront's vectors of four lie in 32 blocks of draws where the channels are a multiple of eight, or
    // where the vectors overlap by enough (65 channels, 17 M values: 120 us the three passes, 125 with vectors of eight);
    // else some lane needs a 33rd, and eight are better (513 channels, 246 M values: 1460 us, 1797 with four)
    const int vectors = (c + 3) / 4;
    if (draws && d->drop.p > 0.0 && c >= 8 && c % 8 != 0 && 64 * (4 * vectors - c) < 8 * vectors) return 8;
    return c >= 4 ? 4 : 1;
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
    a.inv_cg = 1.0f / a.cg;
    a.mask = d->mask;
    a.weight = d->weight; a.bias = d->bias;
    a.weight_dtype = d->weight_dtype; a.bias_dtype = d->bias_dtype;
    a.eps = (float)d->eps;
    return drop_args(&d->drop, a.drop, who);
}

void norm_layout(NormArgs& a, int vector, int in_flight, int element_size, int tensors, int threads) {
    a.tx = (a.channels + vector - 1) / vector;
    a.inv_tx = 1.0f / a.tx;
    // about so many threads, of which as few as possible idle in the last wavefront
    double best = 0.0;
    for (int ty = std::max(1, threads / a.tx); ty * a.tx <= kNormThreads; ++ty) {
        const double used = (double)(ty * a.tx) / ((ty * a.tx + 63) / 64 * 64);
        if (used > best) { best = used; a.ty = ty; }
    }
    const int64_t bytes = a.batch * a.pixels * a.channels * element_size, step = (int64_t)a.ty * in_flight;
    const int64_t workgroups = std::min(kMostThreads, std::max(kFewThreads, bytes / kThreadBytes)) / threads;
    a.chunks = (int)std::max<int64_t>(1, std::min((a.pixels + step - 1) / step, (workgroups + a.batch - 1) / a.batch));
    a.join = (int64_t)a.chunks * a.groups <= kNormJoin;
    a.stream = bytes * tensors > kCacheBytes;
}

extern "C" size_t xsg_group_norm_act_workspace_bytes(const xsg_norm_desc* d, int backward) {
    NormArgs a;
    if (norm_args(d, a, "group_norm_act") != XSG_OK || d->batch == 0 || d->pixels == 0) return 0;
    const int vector = norm_vector(d, backward != 0), size = d->dtype == XSG_DTYPE_F32 ? 4 : 2;
    norm_layout(a, vector, backward ? kNormGradUnroll : kStatsUnroll, size, 0, backward ? 256 : 512);
    const size_t parts = (size_t)(a.batch * a.chunks);
    if (backward) return sizeof(float2) * (parts * (size_t)(a.channels + a.groups) + (size_t)(a.batch * a.groups));
    return sizeof(float2) * parts * (size_t)a.groups + sizeof(float) * parts;
}

extern "C" int xsg_group_norm_act_fwd(const xsg_norm_desc* d, void* y, float* stats, void* workspace, xsg_stream_t stream) {
    NormArgs a;
    if (const int rc = norm_args(d, a, "group_norm_act_fwd")) return rc;
    if (a.batch == 0 || a.pixels == 0) return XSG_OK;
    if (!y || !stats || !workspace) return xsg_fail(XSG_ERR_INVALID, "group_norm_act_fwd: null tensor");
    if (const int rc = xsg_check_workspace(workspace, "group_norm_act_fwd")) return rc;
    if ((uintptr_t)stats % 16) return xsg_fail(XSG_ERR_INVALID, "group_norm_act_fwd: stats must be 16-byte aligned");
    if (norm_small(d, a, y, stats, (hipStream_t)stream)) {
        XSG_TRY_LAUNCH("group_norm_act_fwd");
        return XSG_OK;
    }
    const int size = d->dtype == XSG_DTYPE_F32 ? 4 : 2, vector = norm_vector(d, false), draw_vector = norm_vector(d, true);
    norm_layout(a, vector, kStatsUnroll, size, 2, 512);
    if (a.batch * a.chunks > kNormBlocks)
        return xsg_fail(XSG_ERR_INVALID, "group_norm_act_fwd: too many samples (%lld)", (long long)a.batch);
    const hipStream_t s = (hipStream_t)stream;
    float2* const part = (float2*)workspace;
    float* const counts = (float*)(part + a.batch * a.chunks * a.groups);
    const int chunks = a.chunks;
    with_dtype(d->dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        with_vector(vector, [&](auto vec) {
            constexpr int V = decltype(vec)::value;
            const auto stats_pass = [&](auto one_group) {
                constexpr bool ONE = decltype(one_group)::value;
                const unsigned grid = (unsigned)(a.batch * chunks), threads = norm_threads(a);
                const size_t lds = sizeof(float) * threads * (2 * (ONE ? 1 : V) + 1);
                if (a.mask) norm_stats_kernel<DT, V, ONE, true><<<grid, threads, lds, s>>>(a, part, counts);
                else norm_stats_kernel<DT, V, ONE, false><<<grid, threads, lds, s>>>(a, part, counts);
            };
            if constexpr (V == 1) stats_pass(std::true_type{});
            else if (a.cg % V == 0) stats_pass(std::true_type{});
            else stats_pass(std::false_type{});
        });
        if (!a.join)
            (a.mask ? norm_join_kernel<true> : norm_join_kernel<false>)<<<norm_join_blocks(a), 256, 0, s>>>(
                a.batch * a.groups, a.groups, chunks, a.eps, part, counts, (float4*)stats);
        const int join = a.join;
        norm_layout(a, draw_vector, norm_apply_unroll(draw_vector * size), size, 2, 256);
        a.join = join;
        with_vector(draw_vector, [&](auto vec) {
            with_norm_flags(d, a, [&](auto act, auto drop, auto mask) {
                constexpr int V = decltype(vec)::value, ACT = decltype(act)::value;
                constexpr bool DROP = decltype(drop)::value, MASK = decltype(mask)::value;
                const unsigned grid = (unsigned)(a.batch * a.chunks), threads = norm_threads(a);
                const size_t lds = join ? sizeof(float4) * a.groups : 0;
                if (norm_may_stream<DT, V>() && a.stream)
                    norm_apply_kernel<DT, V, ACT, DROP, MASK, norm_may_stream<DT, V>()>
                        <<<grid, threads, lds, s>>>(a, chunks, part, counts, (float4*)stats, y);
                else
                    norm_apply_kernel<DT, V, ACT, DROP, MASK, false>
                        <<<grid, threads, lds, s>>>(a, chunks, part, counts, (float4*)stats, y);
            });
        });
    });
    XSG_TRY_LAUNCH("group_norm_act_fwd");
    return XSG_OK;
}
