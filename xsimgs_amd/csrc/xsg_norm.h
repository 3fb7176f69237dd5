// Group norm of channels-last feature images with an activation and dropout behind it: what its forward and
// backward kernels share. A workgroup takes batches of pixels of one sample in turn with the others; its threads lie tx
// to a pixel, V consecutive channels each, and ty pixels side by side, so that its accesses are one run of memory.
//
// All of it is bound by memory where images are large and nothing is drawn: x is read for its statistics and again for the
// result, x and v_y for their sums and again for v_x, at 5.3 to 6.2 TB/s (1080p x 64 bfloat16, silu: statistics 48 us,
// result 87, sums 94, v_x 140). Draws hold back the result and the sums (225 x 400 x 128 x 6 float16: 56 us, 4.9 TB/s, and
// 66, 4.2; v_x stays at the memory's rate, 76, 5.5 TB/s). A mask in front of short passes with draws does too: its bytes come
// before the loads that they decide on (128 x 2048 x 65 float32, gelu: result 38, sums 42, v_x 43 us, 2.6 to 4.1 TB/s, at
// 330 to 360 vector instructions a microsecond and SIMD of about 540 that other kernels here reach, with waves waiting 40 to
// 48 % of their time; a training pass of the whole takes 139 us, 133 without the mask, 109 without draws).
#pragma once
#include "xsg_elements.h"
#include "xsg_random.h"

constexpr int kNormThreads = 512;    // most a workgroup has
constexpr int64_t kNormBlocks = ((int64_t)1 << 32) / kNormThreads - 1;   // most of a launch, whose threads stay below 2^32

struct NormArgs {
    const void* x;
    int64_t batch_stride, pixel_stride;
    int64_t batch, pixels;
    int channels, groups, cg;        // cg: channels of a group
    int tx, ty;                      // threads to a pixel (as many as vectors), pixels side by side
    float inv_tx, inv_cg;
    int chunks;                      // workgroups of a sample
    int stream;                      // results go around the caches
    int join;                        // the chunks' results are joined by the kernel that needs them
    const uint8_t* mask;
    const void *weight, *bias;
    int weight_dtype, bias_dtype;
    float eps;
    DropArgs drop;

    // i / tx and i / cg of small i: what lies between two whole numbers is far above a rounding
    XSG_DEV int by_tx(int i) const { return (int)((i + 0.5f) * inv_tx); }
    XSG_DEV int by_cg(int i) const { return (int)((i + 0.5f) * inv_cg); }
    // the last vector of a pixel ends with the last channel, so it repeats some where V does not divide the channels
    template <int V> XSG_HD int first_channel(int v) const { return v * V < channels - V ? v * V : channels - V; }
};

XSG_DEV float norm_param(const void* p, int dtype, int i, float otherwise) {
    if (!p) return otherwise;
    return dtype == XSG_DTYPE_F32 ? load_one<XSG_DTYPE_F32>(p, i)
         : dtype == XSG_DTYPE_BF16 ? load_one<XSG_DTYPE_BF16>(p, i) : load_one<XSG_DTYPE_F16>(p, i);
}

// 1 / (1 + exp(-z)) from the hardware's exponential and reciprocal (1 ulp each). EXACT, for float32 results: the
// exponent's rounding and the reciprocal's last bit are made good, within 2^+-126 (beyond, the corrections would be differences
// of infinities; what lies above the exponent's range is 1, and what lies below is no normal number: 0, so that z times it is
// small for every z); the other types are rounded to 8 or 11 bits next.
template <bool EXACT> XSG_DEV float norm_sigmoid(float z) {
    const float p = z * -1.44269504f;
    float e = __builtin_amdgcn_exp2f(p);
    if (EXACT) {
        const float low = fmaf(z, -1.44269504f, -p) + z * -1.92596303e-8f;
        if (fabsf(p) < 126.0f) e = fmaf(e * 0.69314718f, low, e);
        const float d = 1.0f + e, r = __builtin_amdgcn_rcpf(d);
        return p < 126.0f ? fmaf(r, fmaf(-d, r, 1.0f), r) : 0.0f;
    }
    return __builtin_amdgcn_rcpf(1.0f + e);
}
// The normal distribution function and exp(-z^2 / 2). With t = 1 / (1 + 0.29 |z|), the tail is exp(-z^2 / 2) times a
// polynomial in t of degree 8 (a least-squares fit of erfc(x) exp(x^2) / 2, weighted towards the least largest error: 8e-9
// of the function, 2e-7 with its roundings); relative to the tail itself it stays within 1e-6 down to z = -3, where
// 1 + erf has lost that. Without branches, and both functions share the exponential.
XSG_DEV float norm_phi(float z, float& e) {
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.28991377f, 1.0f));
    e = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
    float q = fmaf(t, 0.035170738f, -0.17173174f);
    q = fmaf(t, q, 0.26084802f);
    q = fmaf(t, q, -0.0976587f);
    q = fmaf(t, q, 0.14824487f);
    q = fmaf(t, q, 0.092404984f);
    q = fmaf(t, q, 0.11711739f);
    q = fmaf(t, q, 0.11560444f);
    const float tail = q * t * e;
    return z < 0.0f ? tail : 1.0f - tail;
}
// the activation times the factor of what is kept, with its reciprocal at hand
template <int ACT, bool EXACT, bool DROP> XSG_DEV float norm_act(float z, float factor, float kept) {
    if (ACT == XSG_ACT_SILU && DROP && !EXACT)   // factor / (1 + e) = 1 / (kept + kept e)
        return z * __builtin_amdgcn_rcpf(fmaf(kept, __builtin_amdgcn_exp2f(z * -1.44269504f), kept));
    float y = z, e;
    if (ACT == XSG_ACT_RELU) y = z < 0.0f ? 0.0f : z;
    if (ACT == XSG_ACT_SILU) y = z * norm_sigmoid<EXACT>(z);
    if (ACT == XSG_ACT_GELU) y = z * norm_phi(z, e);
    return DROP ? y * factor : y;
}
template <int ACT, bool EXACT> XSG_DEV float norm_act_slope(float z) {
    if (ACT == XSG_ACT_RELU) return z > 0.0f ? 1.0f : z == z ? 0.0f : z;
    if (ACT == XSG_ACT_SILU) {
        const float s = norm_sigmoid<EXACT>(z);
        return s * (1.0f + z * (1.0f - s));
    }
    if (ACT == XSG_ACT_GELU) {
        float e;
        const float phi = norm_phi(z, e);
        return fmaf(z * e, 0.39894228f, phi);
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
template <typename T> XSG_DEV T segment_sum(T x, int l) {
    for (int d = l >> 1; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}
// two sums side by side, which wait for each other's lanes once
XSG_DEV void segment_sums(float& x, float& y, int l) {
    for (int d = l >> 1; d; d >>= 1) {
        const float x2 = __shfl_xor(x, d), y2 = __shfl_xor(y, d);
        x += x2;
        y += y2;
    }
}

// A thread's place: its first channel, its row of the pixels side by side, and its workgroup's batches of pixels: from
// p0 on in jumps, in turn with the sample's other workgroups, so that all of them together move through one stretch of
// memory (runs of a workgroup's own: 436 us a training pass of 265 MB images, 422 in turn).
template <int V> struct NormPlace {
    int v, r, c0;
    int64_t b, chunk, p0, jump;
    XSG_DEV NormPlace(const NormArgs& a, uint32_t block, int batch) {
        r = a.by_tx(threadIdx.x);
        v = (int)threadIdx.x - r * a.tx;
        c0 = a.first_channel<V>(v);
        const uint32_t sample = block / (uint32_t)a.chunks;
        b = sample;
        chunk = block - sample * (uint32_t)a.chunks;
        p0 = chunk * batch;
        jump = (int64_t)batch * a.chunks;
    }
};

// A thread's way through an array of pixels: its own place in the first of a sample, and uniform steps from there.
template <int DT> struct NormPath {
    const char* at;
    int64_t pixel;   // bytes
    XSG_DEV NormPath(const void* base, int64_t sample, int64_t pixel_stride, int r, int c0)
        : at((const char*)base + (sample + r * pixel_stride + c0) * ElementSize<DT>::value),
          pixel(pixel_stride * ElementSize<DT>::value) {}
    XSG_DEV char* operator()(int64_t p) const { return const_cast<char*>(at) + p * pixel; }
};

// Which of U pixels, ty apart from p on, a thread has: bit u, and bit 16 + u where the mask has it too.
template <int U, bool MASK, int V> XSG_DEV uint32_t norm_pixels(const NormArgs& a, const NormPlace<V>& at, int64_t p) {
    uint32_t in = 0;
    const int left = (int)min(a.pixels - p, (int64_t)(U * kNormThreads));   // of this batch and what follows
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (at.r < a.ty && at.r + u * a.ty < left) in |= (!MASK || a.mask[at.b * a.pixels + p + at.r + u * a.ty] != 0 ? 0x10001u : 1u) << u;
    return in;
}

// A thread's draws of pixel u of a batch, from element first + u step on. Every lane of the wavefront comes here for every
// pixel, in the order of their elements. With vectors of four, two pixels' draws come at once; with eight 16-bit values
// they are words that the packed values are masked with, two values an operation (69 M float16 values: 214 us the three
// passes, 227 with bits).
template <int DT, int V> struct NormDraws {
    static constexpr bool HALVES = DT != XSG_DTYPE_F32 && V == 8;
    const Draws& draws;
    int channels;
    int64_t first, step;   // element of the batch's first pixel, and from pixel to pixel
    uint32_t bits, next;
    Words4 halves;
    XSG_DEV NormDraws(const Draws& draws_, int channels_, int64_t first_, int64_t step_)
        : draws(draws_), channels(channels_), first(first_), step(step_), bits(0), next(0), halves{} {}
    XSG_DEV void draw(int u) {
        const int64_t e = first + u * step;
        if (HALVES) {
            halves = channels % 8 == 0 ? draws.halves8((uint64_t)e >> 3) : Draws::halves_of(draws.keep_in_order((uint64_t)e));
        } else if (V == 8) {
            bits = channels % 8 == 0 ? draws.keep8((uint64_t)e >> 3) : draws.keep_in_order((uint64_t)e);
        } else if (V == 4) {
            if (u % 2) bits = next;
            else draws.keep_in_order((uint64_t)e, (uint64_t)(e + step), bits, next);
        } else {
            bits = draws.keep((uint64_t)e, V);
        }
    }
    // zeros in packed values that are dropped, whatever they hold
    XSG_DEV void mask(Raw<V * ElementSize<DT>::value>& r) const {
        if constexpr (HALVES) {
#pragma unroll
            for (int k = 0; k < 4; ++k) r.w[k] &= halves.w[k];
        }
    }
    // the same of one value, where mask() does nothing
    XSG_DEV float one(float x, int j) const { return HALVES ? x : keep_bit(x, bits, j); }
};

// Statistics of a sample's groups lie in `part` (mean and squared deviations of each chunk) and `counts` (elements of
// a group in each); up to this many pairs the next launch's workgroups each join them themselves (8 bytes each, from
// the second-level cache), beyond a launch of its own does.
constexpr int64_t kNormJoin = 2048;

// Host side: checks a description and lays the work out; `pixels_in_flight` of a thread, `workgroups` wanted.
int norm_args(const xsg_norm_desc* d, NormArgs& a, const char* who);
int norm_vector(const xsg_norm_desc* d, bool draws);
// `tensors` of x's size move through a call, of which those written may go around the caches; workgroups of about
// `threads` (256, or 512 where they leave results for the next launch to join)
void norm_layout(NormArgs& a, int vector, int pixels_in_flight, int element_size, int tensors, int threads);
// Results around the caches, which would push out what the next pass reads: for whole vectors (small images do without)
template <int DT, int V> constexpr bool norm_may_stream() { return V * ElementSize<DT>::value >= 16; }
// Pixels in flight in a thread, with the next as many on their way where vectors are of 16 bytes (a rig's blocks of 69 M
// values with draws: 213 us the three passes, 226 without; wider ones run out of registers by it: 135 and 121 us)
constexpr int norm_apply_unroll(int bytes) { return bytes > 16 ? 2 : 4; }
constexpr int kNormGradUnroll = 2;
constexpr bool norm_ahead(int bytes) { return bytes <= 16; }
// The forward in one launch, where a sample's groups fit workgroups; false where they do not.
bool norm_small(const xsg_norm_desc* d, const NormArgs& a, void* y, float* stats, hipStream_t s);
// of the launches that join parts, one to a group of a sample
inline unsigned norm_join_blocks(const NormArgs& a) { return (unsigned)(a.batch * a.groups < kNormBlocks ? a.batch * a.groups : kNormBlocks); }
inline unsigned norm_threads(const NormArgs& a) { return (unsigned)((a.tx * a.ty + 63) / 64 * 64); }

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
