// Group norm with an activation and dropout, channels last, of small images: a sample's group (or a few of them side by
// side) stays in one workgroup's registers, so one launch reads x once: a 16 x 16 patch of 32 channels takes 6.6 us, 10.6
// in two launches. Bound by the latency of its loads and four barriers; more than 16 KB to a workgroup were slower than
// two launches (32 x 32 x 512 bfloat16: 21 us with 1024 threads, 12 in two launches). No reference counterpart.
#include <algorithm>

#include "xsg_norm.h"

namespace {

constexpr int kSmallThreads = 256, kSmallVectors = 4;   // vectors a thread holds

struct SmallArgs {
    int width, bundle;    // channels and groups of a workgroup
    int tx, ty;
    float inv_tx;
};

template <int DT, int V, int ACT, bool DROP, bool MASK>
__global__ __launch_bounds__(kSmallThreads) void norm_small_kernel(NormArgs a, SmallArgs k, float4* __restrict__ stats,
                                                                   void* __restrict__ y) {
    constexpr bool EXACT = DT == XSG_DTYPE_F32;
    constexpr int N = kSmallVectors;
    typedef Raw<V * ElementSize<DT>::value> Vec;
    extern __shared__ float s_sums[];                      // [threads][V], twice; [threads] counts; [bundle] float4
    float* const s_dev = s_sums + V * blockDim.x;
    float* const s_count = s_dev + V * blockDim.x;
    float4* const s_group = (float4*)(s_count + blockDim.x);
    const int t = threadIdx.x, r = (int)((t + 0.5f) * k.inv_tx), v = t - r * k.tx;
    const int bundles = a.groups / k.bundle;
    const int64_t b = blockIdx.x / (uint32_t)bundles;
    const int g0 = (int)(blockIdx.x - (uint32_t)b * bundles) * k.bundle;
    // the last vector ends with the last channel of the bundle, so it may repeat some
    const int in_bundle = min(v * V, k.width - V), c0 = g0 * a.cg + in_bundle, pixels = (int)a.pixels;
    const NormPath<DT> x_at(a.x, b * a.batch_stride, a.pixel_stride, r, c0);
    const uint8_t* const mask = MASK ? a.mask + b * a.pixels : nullptr;

    Vec raw[N];
    uint32_t in = 0;   // bit n: in the image, bit 16 + n: in the mask too
#pragma unroll
    for (int n = 0; n < N; ++n)
        if (r < k.ty && r + n * k.ty < pixels) in |= (!MASK || mask[r + n * k.ty] != 0 ? 0x10001u : 1u) << n;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        raw[n] = {};
        if (in >> (16 + n) & 1) raw[n] = load_raw<DT, V>(x_at(n * k.ty));
    }
    float scale[V], bias[V], s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        scale[j] = norm_param(a.weight, a.weight_dtype, c0 + j, 1.0f);
        bias[j] = norm_param(a.bias, a.bias_dtype, c0 + j, 0.0f);
        s1[j] = s2[j] = 0.0f;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        float x[V];
        unpack<DT, V>(raw[n], x);
#pragma unroll
        for (int j = 0; j < V; ++j) s1[j] += x[j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) s_sums[t * V + j] = s1[j];
    s_count[t] = (float)__popc(in >> 16);
    __syncthreads();

    // a segment of lanes adds up a group's entries: ty rows of its channels
    const int l = norm_segment(blockDim.x, k.bundle), lane = t & (l - 1), entries = a.cg * k.ty;
    const int row0 = a.by_cg(lane), col0 = lane - row0 * a.cg, rows = a.by_cg(l), cols = l - rows * a.cg;
    const auto each = [&](int g, auto f) {
        int row = row0, col = col0;
        for (int e = lane; e < entries; e += l) {
            const int c = g * a.cg + col, vec = min(c / V, k.tx - 1), thread = row * k.tx + vec;
            f(thread * V + c - min(vec * V, k.width - V), thread);
            row += rows;
            col += cols;
            if (col >= a.cg) { col -= a.cg; ++row; }
        }
    };
    for (int g = t / l; g < k.bundle; g += blockDim.x / l) {
        float count = 0.0f, sum = 0.0f;
        each(g, [&](int at, int thread) { sum += s_sums[at]; count += s_count[thread]; });
        count = segment_sum(count, l);
        sum = segment_sum(sum, l);
        if (lane == 0) s_group[g] = make_float4(count > 0.0f ? sum / count : 0.0f, 0.0f, count, 0.0f);
    }
    __syncthreads();
    // deviations about that mean, and what its own rounding left of their sum
    float mean[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        mean[j] = s_group[a.by_cg(in_bundle + j)].x;
        s1[j] = 0.0f;
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
        if (in >> (16 + n) & 1) {
            float x[V];
            unpack<DT, V>(raw[n], x);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float e = x[j] - mean[j];
                s1[j] += e;
                s2[j] += e * e;
            }
        }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        s_sums[t * V + j] = s1[j];
        s_dev[t * V + j] = s2[j];
    }
    __syncthreads();
    for (int g = t / l; g < k.bundle; g += blockDim.x / l) {
        float sum = 0.0f, dev = 0.0f;
        each(g, [&](int at, int) { sum += s_sums[at]; dev += s_dev[at]; });
        sum = segment_sum(sum, l);
        dev = segment_sum(dev, l);
        if (lane == 0) {
            const float4 m = s_group[g];
            const float inv = m.z > 0.0f ? 1.0f / m.z : 0.0f, left = sum * inv;
            float var = dev * inv - left * left;
            if (var < 0.0f) var = 0.0f;   // a NaN stays
            s_group[g] = make_float4(m.x + left, inv > 0.0f ? 1.0f / sqrtf(var + a.eps) : 0.0f, inv, 0.0f);
            stats[b * a.groups + g0 + g] = s_group[g];
        }
    }
    __syncthreads();
    if (r >= k.ty) return;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float4 s = s_group[a.by_cg(in_bundle + j)];
        mean[j] = s.x;
        scale[j] *= s.y;
    }
    const NormPath<DT> y_at(y, b * a.pixels * a.channels, a.channels, r, c0);
    const int64_t first = (b * a.pixels + r) * a.channels + c0;
    const Draws draws(a.drop);
    const float kept = 1.0f / a.drop.factor;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if (!(in >> n & 1)) break;
        Vec out = {};
        if (!MASK || (in >> (16 + n) & 1)) {
            float x[V];
            unpack<DT, V>(raw[n], x);
            const uint32_t keep = DROP ? draws.keep((uint64_t)(first + (int64_t)n * k.ty * a.channels), V) : 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x[j] = norm_act<ACT, EXACT, DROP>(fmaf(x[j] - mean[j], scale[j], bias[j]), a.drop.factor, kept);
                if (DROP) x[j] = keep_bit(x[j], keep, j);
            }
            out = pack<DT, V>(x);
        }
        store_raw<DT, V>(y_at(n * k.ty), 0, out);
    }
}

}  // namespace

bool norm_small(const xsg_norm_desc* d, const NormArgs& a, void* y, float* stats, hipStream_t s) {
    const int size = d->dtype == XSG_DTYPE_F32 ? 4 : 2;
    if (a.pixels > kSmallThreads * kSmallVectors) return false;
    // the fewest groups whose channels fill 64 bytes of a pixel, or all of them
    SmallArgs k{};
    for (k.bundle = 1; k.bundle < a.groups && (a.groups % k.bundle || k.bundle * a.cg * size < 64); ++k.bundle) {}
    int vector = 0;
    for (;; k.bundle = 1) {
        k.width = k.bundle * a.cg;
        vector = size == 2 && k.width >= 8 ? 8 : k.width >= 4 ? 4 : 1;
        k.tx = (k.width + vector - 1) / vector;
        if (k.tx <= kSmallThreads && (a.pixels + kSmallThreads / k.tx - 1) / (kSmallThreads / k.tx) <= kSmallVectors) break;
        if (k.bundle == 1) return false;
    }
    k.inv_tx = 1.0f / k.tx;
    k.ty = (int)std::min<int64_t>(a.pixels, kSmallThreads / k.tx);
    const int64_t grid = a.batch * (a.groups / k.bundle);
    if (grid > kNormBlocks) return false;
    const unsigned threads = (unsigned)((k.tx * k.ty + 63) / 64 * 64);
    with_dtype(d->dtype, [&](auto dt) {
        with_vector(vector, [&](auto vec) {
            with_norm_flags(d, a, [&](auto act, auto drop, auto mask) {
                constexpr int DT = decltype(dt)::value, V = decltype(vec)::value;
                if constexpr (DT != XSG_DTYPE_F32 || V < 8) {
                    const size_t lds = sizeof(float) * (2 * V + 1) * threads + sizeof(float4) * k.bundle;
                    norm_small_kernel<DT, V, decltype(act)::value, decltype(drop)::value, decltype(mask)::value>
                        <<<(unsigned)grid, threads, lds, s>>>(a, k, (float4*)stats, y);
                }
            });
        });
    });
    return true;
}
