// What a training step does behind the frame's backward: the global norm of many gradient tensors, clipping
// by it, and the Adam update that takes the clip factor and the packed visibility mask. No reference
// counterpart (the reference's trainer is outside its rendering library).
//
// All three run over a list of tensors cut into chunks of one length; a workgroup takes one chunk. The list
// travels in the kernel's arguments (no copy, no allocation, and a captured graph holds it by value), as many
// tensors to a launch as 4 KB of arguments hold. Sums are held in 64 bits and added in a fixed order, so a
// call's results are the same bits each time.
#include <math.h>

#include <algorithm>

#include "xsg_common.h"

namespace {

constexpr int kBlock = 256;
constexpr int64_t kChunkUnit = 1024;      // chunks are multiples of this many elements
constexpr int64_t kTargetChunks = 2048;   // chunks of a call, when its tensors are long enough
constexpr int64_t kMaxChunk = 1 << 30;    // offsets inside a chunk are 32-bit
constexpr int64_t kMaxRow = 1 << 30;      // and so are rows under a mask
constexpr int64_t kMaxElements = (int64_t)1 << 48;
constexpr int kListMax = 112;             // gradient tensors to a launch
constexpr int kAdamMax = 52;              // tensors with their states to a launch

struct GradList {
    void* data[kListMax];
    int64_t numel[kListMax];
    const uint32_t* mask[kListMax];
    int32_t row[kListMax];        // elements to a mask bit
    int32_t first[kListMax + 1];  // first chunk of each tensor in this launch
    uint8_t dtype[kListMax];
    int32_t n;
    int64_t chunk;
};
static_assert(sizeof(GradList) <= 3900, "the list and the other arguments share 4 KB");

struct AdamList {
    void* param[kAdamMax];
    const void* grad[kAdamMax];
    float* avg[kAdamMax];
    float* sq[kAdamMax];
    int64_t numel[kAdamMax];
    const uint32_t* mask[kAdamMax];
    int32_t row[kAdamMax];
    int32_t first[kAdamMax + 1];
    float lr[kAdamMax];
    float keep[kAdamMax];         // 1 - lr * weight decay
    uint8_t pdtype[kAdamMax], gdtype[kAdamMax];
    int32_t n;
    int64_t chunk;
};
static_assert(sizeof(AdamList) <= 3900, "the list and the other arguments share 4 KB");

XSG_DEV float load_as_float(const void* p, int64_t i, int dtype) {
    if (dtype == XSG_DTYPE_F32) return ((const float*)p)[i];
    if (dtype == XSG_DTYPE_BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
    return (float)((const _Float16*)p)[i];
}

// round to nearest even; a NaN stays one
XSG_DEV uint16_t bf16_bits(float x) {
    const uint32_t u = __float_as_uint(x);
    if (x != x) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

XSG_DEV void store_from_float(void* p, int64_t i, int dtype, float x) {
    if (dtype == XSG_DTYPE_F32) ((float*)p)[i] = x;
    else if (dtype == XSG_DTYPE_BF16) ((uint16_t*)p)[i] = bf16_bits(x);
    else ((_Float16*)p)[i] = (_Float16)x;
}

XSG_DEV bool in_mask(const uint32_t* mask, int64_t i, int32_t row) {
    if (!mask) return true;
    const int64_t r = i / row;
    return (mask[r >> 5] >> (r & 31)) & 1u;
}

// the tensor whose chunks hold chunk b: the last one with first[t] <= b (empty tensors have no chunk)
XSG_DEV int find_tensor(const int32_t* first, int n, int b) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= b) lo = mid; else hi = mid;
    }
    return lo;
}

// Accumulation of one kind of norm in 64 bits: squares of any float32 stay finite and above zero there. A
// maximum keeps a NaN once it has seen one.
template <int NORM> XSG_DEV double norm_add(double acc, double x) {
    if (NORM == XSG_NORM_L2) return acc + x * x;
    if (NORM == XSG_NORM_L1) return acc + fabs(x);
    x = fabs(x);
    return (x > acc || x != x) ? x : acc;
}
template <int NORM> XSG_DEV double norm_join(double a, double b) {
    if (NORM == XSG_NORM_INF) return (b > a || b != b) ? b : a;
    return a + b;
}
template <int NORM> XSG_DEV double norm_finish(double a) { return NORM == XSG_NORM_L2 ? sqrt(a) : a; }

// The workgroup's joined value, in every thread; the order is fixed.
template <int NORM> XSG_DEV double block_join(double v) {
    __shared__ double part[kBlock / 64];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = norm_join<NORM>(v, __shfl_xor(v, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < kBlock / 64; ++w) v = norm_join<NORM>(v, part[w]);
    return v;
}

template <int NORM>
__global__ __launch_bounds__(kBlock) void norm_partial_kernel(GradList list, double* __restrict__ partial) {
    const int b = blockIdx.x, t = find_tensor(list.first, list.n, b);
    const int64_t base = (int64_t)(b - list.first[t]) * list.chunk;
    const int64_t end = min(base + list.chunk, list.numel[t]);
    double acc = 0.0;
    for (int64_t i = base + threadIdx.x; i < end; i += kBlock)
        if (in_mask(list.mask[t], i, list.row[t]))
            acc = norm_add<NORM>(acc, load_as_float(list.data[t], i, list.dtype[t]));
    acc = block_join<NORM>(acc);
    if (threadIdx.x == 0) partial[b] = acc;
}

template <int NORM> XSG_DEV double join_partials(const double* __restrict__ partial, int n) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < n; i += kBlock) acc = norm_join<NORM>(acc, partial[i]);
    return block_join<NORM>(acc);
}

// Block 0: the norm over every chunk of the call, to `total` (float32) and `sum` (64 bits).
// Blocks 1..n: the norm of each tensor of this list, whose chunks start at partial[0].
template <int NORM>
__global__ __launch_bounds__(kBlock) void norm_finish_kernel(GradList list, const double* __restrict__ all,
                                                             int n_all, const double* __restrict__ partial,
                                                             float* __restrict__ total, double* __restrict__ sum,
                                                             float* __restrict__ each) {
    if (blockIdx.x == 0) {
        const double v = norm_finish<NORM>(join_partials<NORM>(all, n_all));
        if (threadIdx.x == 0) {
            if (total) *total = (float)v;
            *sum = v;
        }
    } else {
        const int t = blockIdx.x - 1;
        const int lo = list.first[t], hi = list.first[t + 1];
        const double v = norm_finish<NORM>(join_partials<NORM>(partial + lo, hi - lo));
        if (threadIdx.x == 0) each[t] = (float)v;
    }
}

// min(1, max_norm / (norm + eps)); a NaN norm gives NaN, an infinite one 0
XSG_DEV float clip_factor(double norm, double max_norm, double eps) {
    const double c = max_norm / (norm + eps);
    return c > 1.0 ? 1.0f : (float)c;
}

__global__ __launch_bounds__(kBlock) void clip_scale_kernel(GradList list, const double* __restrict__ norm,
                                                            double max_norm, double eps) {
    const float c = clip_factor(*norm, max_norm, eps);
    if (c == 1.0f) return;   // the values stay as they are
    const int b = blockIdx.x, t = find_tensor(list.first, list.n, b);
    const int64_t base = (int64_t)(b - list.first[t]) * list.chunk;
    const int64_t end = min(base + list.chunk, list.numel[t]);
    for (int64_t i = base + threadIdx.x; i < end; i += kBlock)
        if (in_mask(list.mask[t], i, list.row[t]))
            store_from_float(list.data[t], i, list.dtype[t], load_as_float(list.data[t], i, list.dtype[t]) * c);
}

struct AdamScalars {
    double log_beta1, log_beta2;   // natural logarithms
    float beta1, beta2, one_minus_beta1, one_minus_beta2, eps;
    int clip, skip_nonfinite;
    double max_norm;
};
constexpr double kAdamClipEps = 1e-6;

// The step counter counts this step; adam_kernel takes it back where the step is not taken.
__global__ void adam_count_kernel(int64_t* step) { *step += 1; }

__global__ __launch_bounds__(kBlock) void adam_kernel(AdamList list, AdamScalars s, const double* __restrict__ norm,
                                                      int64_t* __restrict__ step, int last_launch) {
    float c = 1.0f;
    if (norm) {
        const double v = *norm;
        if (s.skip_nonfinite && !(v < (double)INFINITY)) {
            // no workgroup of any of the call's launches reads the counter in this case
            if (last_launch && blockIdx.x == 0 && threadIdx.x == 0) *step -= 1;
            return;
        }
        if (s.clip) c = clip_factor(v, s.max_norm, kAdamClipEps);
    }
    const int b = blockIdx.x;
    if (b >= list.first[list.n]) return;   // a launch without elements still takes a step back
    const int t = find_tensor(list.first, list.n, b);
    const double k = (double)*step;
    // 1 - beta^k without the cancellation
    const float fix1 = (float)-expm1(k * s.log_beta1), fix2 = (float)sqrt(-expm1(k * s.log_beta2));
    const int64_t base = (int64_t)(b - list.first[t]) * list.chunk;
    const int64_t end = min(base + list.chunk, list.numel[t]);
    const float rate = list.lr[t] / fix1;
    for (int64_t i = base + threadIdx.x; i < end; i += kBlock) {
        if (!in_mask(list.mask[t], i, list.row[t])) continue;
        const float g = load_as_float(list.grad[t], i, list.gdtype[t]) * c;
        const float m0 = list.avg[t][i], v0 = list.sq[t][i];
        const float m = m0 + s.one_minus_beta1 * (g - m0);
        const float v = s.beta2 * v0 + s.one_minus_beta2 * g * g;
        const float p = load_as_float(list.param[t], i, list.pdtype[t]) * list.keep[t]
                        - rate * m / (sqrtf(v) / fix2 + s.eps);
        list.avg[t][i] = m;
        list.sq[t][i] = v;
        store_from_float(list.param[t], i, list.pdtype[t], p);
    }
}

// ------------------------------------------------------------------------------------------------ host
int64_t chunk_for(int64_t elements) {
    int64_t c = (elements + kTargetChunks - 1) / kTargetChunks;
    c = (c + kChunkUnit - 1) / kChunkUnit * kChunkUnit;
    return std::min(std::max(c, kChunkUnit), kMaxChunk);
}
int64_t chunks_of(int64_t numel, int64_t chunk) { return (numel + chunk - 1) / chunk; }

int check_dtype(int dtype, const char* who, int i) {
    if (dtype != XSG_DTYPE_F32 && dtype != XSG_DTYPE_BF16 && dtype != XSG_DTYPE_F16)
        return xsg_fail(XSG_ERR_INVALID, "%s: tensor %d has unknown type %d", who, i, dtype);
    return XSG_OK;
}

int check_rows(int64_t numel, const void* mask, int64_t rows, const char* who, int i) {
    if (numel < 0) return xsg_fail(XSG_ERR_INVALID, "%s: tensor %d has a negative size", who, i);
    if (!mask || numel == 0) return XSG_OK;
    if (rows <= 0 || numel % rows != 0)
        return xsg_fail(XSG_ERR_INVALID, "%s: tensor %d of %lld elements cannot have %lld rows under its mask", who, i,
                        (long long)numel, (long long)rows);
    if (numel / rows > kMaxRow)
        return xsg_fail(XSG_ERR_INVALID, "%s: tensor %d has rows of %lld elements under its mask, more than %lld", who,
                        i, (long long)(numel / rows), (long long)kMaxRow);
    return XSG_OK;
}

xsg_grad_tensor grad_of(const xsg_grad_tensor& x) { return x; }
xsg_grad_tensor grad_of(const xsg_adam_tensor& x) {
    return xsg_grad_tensor{const_cast<void*>(x.grad), x.numel, x.mask, x.rows, x.grad_dtype};
}

struct Plan {
    int64_t elements = 0, chunk = 0, chunks = 0;
};

template <typename T> int make_plan(const T* ts, int n, const char* who, Plan* p) {
    if (n < 0 || (n > 0 && !ts)) return xsg_fail(XSG_ERR_INVALID, "%s: null or negative list of tensors", who);
    for (int i = 0; i < n; ++i) {
        if (ts[i].numel < 0) return xsg_fail(XSG_ERR_INVALID, "%s: tensor %d has a negative size", who, i);
        if (ts[i].numel > kMaxElements - p->elements) return xsg_fail(XSG_ERR_INVALID, "%s: too many elements", who);
        p->elements += ts[i].numel;
    }
    p->chunk = chunk_for(p->elements);
    for (int i = 0; i < n; ++i) p->chunks += chunks_of(ts[i].numel, p->chunk);
    if (p->chunks > kMaxChunk) return xsg_fail(XSG_ERR_INVALID, "%s: too many tensors", who);
    return XSG_OK;
}

size_t partial_bytes(int64_t chunks) { return 256 + (size_t)chunks * sizeof(double); }

// fills list from ts[i0...] and returns how many tensors it took
template <typename T> int fill_list(const T* ts, int n, int i0, int64_t chunk, GradList* list) {
    list->chunk = chunk;
    int k = 0;
    int32_t at = 0;
    for (; k < kListMax && i0 + k < n; ++k) {
        const xsg_grad_tensor x = grad_of(ts[i0 + k]);
        list->data[k] = x.data;
        list->numel[k] = x.numel;
        list->mask[k] = x.mask;
        list->row[k] = x.mask && x.numel ? (int32_t)(x.numel / x.rows) : 1;
        list->dtype[k] = (uint8_t)x.dtype;
        list->first[k] = at;
        at += (int32_t)chunks_of(x.numel, chunk);
    }
    list->first[k] = at;
    list->n = k;
    return k;
}

template <typename T> int check_list(const T* ts, int n, int norm, const char* who) {
    if (norm != XSG_NORM_INF && norm != XSG_NORM_L1 && norm != XSG_NORM_L2)
        return xsg_fail(XSG_ERR_INVALID, "%s: unknown norm %d", who, norm);
    for (int i = 0; i < n; ++i) {
        const xsg_grad_tensor x = grad_of(ts[i]);
        if (x.numel > 0 && !x.data) return xsg_fail(XSG_ERR_INVALID, "%s: tensor %d is null", who, i);
        int rc = check_dtype(x.dtype, who, i);
        if (rc == XSG_OK) rc = check_rows(x.numel, x.mask, x.rows, who, i);
        if (rc != XSG_OK) return rc;
    }
    return XSG_OK;
}

template <typename F> void with_norm(int norm, F&& f) {
    if (norm == XSG_NORM_L2) f(std::integral_constant<int, XSG_NORM_L2>{});
    else if (norm == XSG_NORM_L1) f(std::integral_constant<int, XSG_NORM_L1>{});
    else f(std::integral_constant<int, XSG_NORM_INF>{});
}

// workspace: the norm in 64 bits, then (256 bytes on) one partial per chunk
template <typename T>
int launch_norm(const T* ts, int n, int norm, const Plan& p, float* total, float* each, void* ws, hipStream_t s) {
    double* sum = (double*)ws;
    double* partial = (double*)((char*)ws + 256);
    GradList list;
    int64_t at = 0;
    for (int i = 0; i < n;) {
        const int k = fill_list(ts, n, i, p.chunk, &list);
        const int chunks = list.first[k];
        if (chunks > 0) {
            with_norm(norm, [&](auto kind) {
                norm_partial_kernel<kind.value><<<chunks, kBlock, 0, s>>>(list, partial + at);
            });
            XSG_TRY_LAUNCH("grad_norm");
        }
        at += chunks;
        i += k;
    }
    at = 0;
    int i = 0;
    do {
        const int k = fill_list(ts, n, i, p.chunk, &list);
        with_norm(norm, [&](auto kind) {
            norm_finish_kernel<kind.value><<<each ? 1 + k : 1, kBlock, 0, s>>>(list, partial, (int)p.chunks,
                                                                              partial + at, total, sum,
                                                                              each ? each + i : nullptr);
        });
        XSG_TRY_LAUNCH("grad_norm");
        at += list.first[k];
        i += k;
    } while (each && i < n);
    return XSG_OK;
}

}  // namespace

extern "C" size_t xsg_grad_norm_workspace_bytes(const xsg_grad_tensor* ts, int n) {
    Plan p;
    return make_plan(ts, n, "grad_norm", &p) == XSG_OK ? partial_bytes(p.chunks) : 0;
}

extern "C" int xsg_grad_norm(const xsg_grad_tensor* ts, int n, int norm, float* total, float* each, void* workspace,
                             xsg_stream_t stream) {
    Plan p;
    int rc = make_plan(ts, n, "grad_norm", &p);
    if (rc == XSG_OK) rc = check_list(ts, n, norm, "grad_norm");
    if (rc != XSG_OK) return rc;
    if (!total || !workspace) return xsg_fail(XSG_ERR_INVALID, "grad_norm: null output or workspace");
    rc = xsg_check_workspace(workspace, "grad_norm");
    if (rc != XSG_OK) return rc;
    return launch_norm(ts, n, norm, p, total, each, workspace, (hipStream_t)stream);
}

extern "C" int xsg_clip_grads(const xsg_grad_tensor* ts, int n, int norm, double max_norm, double eps, float* total,
                              void* workspace, xsg_stream_t stream) {
    Plan p;
    int rc = make_plan(ts, n, "clip_grads", &p);
    if (rc == XSG_OK) rc = check_list(ts, n, norm, "clip_grads");
    if (rc != XSG_OK) return rc;
    if (!(max_norm >= 0.0) || !(eps >= 0.0))
        return xsg_fail(XSG_ERR_INVALID, "clip_grads: max_norm %g and eps %g must not be negative", max_norm, eps);
    if (!total || !workspace) return xsg_fail(XSG_ERR_INVALID, "clip_grads: null output or workspace");
    rc = xsg_check_workspace(workspace, "clip_grads");
    if (rc != XSG_OK) return rc;
    hipStream_t s = (hipStream_t)stream;
    rc = launch_norm(ts, n, norm, p, total, nullptr, workspace, s);
    if (rc != XSG_OK) return rc;
    GradList list;
    for (int i = 0; i < n;) {
        const int k = fill_list(ts, n, i, p.chunk, &list);
        if (list.first[k] > 0) {
            clip_scale_kernel<<<list.first[k], kBlock, 0, s>>>(list, (const double*)workspace, max_norm, eps);
            XSG_TRY_LAUNCH("clip_grads");
        }
        i += k;
    }
    return XSG_OK;
}

extern "C" size_t xsg_adam_step_workspace_bytes(const xsg_adam_tensor* ts, int n, const xsg_adam_options* o) {
    Plan p;
    if (!o || make_plan(ts, n, "adam_step", &p) != XSG_OK) return 0;
    return o->clip || o->skip_nonfinite ? partial_bytes(p.chunks) : 0;
}

extern "C" int xsg_adam_step(const xsg_adam_tensor* ts, int n, const xsg_adam_options* o, int64_t* step, float* total,
                             void* workspace, xsg_stream_t stream) {
    if (!o || !step) return xsg_fail(XSG_ERR_INVALID, "adam_step: null options or step counter");
    Plan p;
    int rc = make_plan(ts, n, "adam_step", &p);
    if (rc != XSG_OK) return rc;
    if (!(o->beta1 >= 0.0 && o->beta1 < 1.0 && o->beta2 >= 0.0 && o->beta2 < 1.0))
        return xsg_fail(XSG_ERR_INVALID, "adam_step: betas %g and %g must lie in [0, 1)", o->beta1, o->beta2);
    if (!(o->eps >= 0.0)) return xsg_fail(XSG_ERR_INVALID, "adam_step: eps %g must not be negative", o->eps);
    if (o->clip && !(o->max_norm >= 0.0))
        return xsg_fail(XSG_ERR_INVALID, "adam_step: max_norm %g must not be negative", o->max_norm);
    for (int i = 0; i < n; ++i) {
        const xsg_adam_tensor& x = ts[i];
        if (x.numel > 0 && (!x.param || !x.grad || !x.exp_avg || !x.exp_avg_sq))
            return xsg_fail(XSG_ERR_INVALID, "adam_step: tensor %d has a null array", i);
        rc = check_dtype(x.param_dtype, "adam_step", i);
        if (rc != XSG_OK) return rc;
    }
    const bool needs_norm = o->clip || o->skip_nonfinite;
    rc = check_list(ts, n, needs_norm ? o->norm : XSG_NORM_L2, "adam_step");
    if (rc != XSG_OK) return rc;
    hipStream_t s = (hipStream_t)stream;
    const double* norm = nullptr;
    if (needs_norm) {
        if (!workspace) return xsg_fail(XSG_ERR_INVALID, "adam_step: null workspace");
        rc = xsg_check_workspace(workspace, "adam_step");
        if (rc != XSG_OK) return rc;
        rc = launch_norm(ts, n, o->norm, p, total, nullptr, workspace, s);
        if (rc != XSG_OK) return rc;
        norm = (const double*)workspace;
    }
    adam_count_kernel<<<1, 1, 0, s>>>(step);
    XSG_TRY_LAUNCH("adam_step");
    AdamScalars a;
    a.log_beta1 = log(o->beta1);   // beta 0: -inf, and 1 - beta^k is 1
    a.log_beta2 = log(o->beta2);
    a.beta1 = (float)o->beta1;
    a.beta2 = (float)o->beta2;
    a.one_minus_beta1 = (float)(1.0 - o->beta1);
    a.one_minus_beta2 = (float)(1.0 - o->beta2);
    a.eps = (float)o->eps;
    a.clip = o->clip;
    a.skip_nonfinite = o->skip_nonfinite;
    a.max_norm = o->max_norm;
    AdamList list;
    for (int i = 0; i < n;) {
        list.chunk = p.chunk;
        int k = 0;
        int32_t at = 0;
        for (; k < kAdamMax && i + k < n; ++k) {
            const xsg_adam_tensor& x = ts[i + k];
            list.param[k] = x.param;
            list.grad[k] = x.grad;
            list.avg[k] = x.exp_avg;
            list.sq[k] = x.exp_avg_sq;
            list.numel[k] = x.numel;
            list.mask[k] = x.mask;
            list.row[k] = x.mask && x.numel ? (int32_t)(x.numel / x.rows) : 1;
            list.pdtype[k] = (uint8_t)x.param_dtype;
            list.gdtype[k] = (uint8_t)x.grad_dtype;
            list.lr[k] = (float)x.lr;
            list.keep[k] = (float)(1.0 - x.lr * x.weight_decay);
            list.first[k] = at;
            at += (int32_t)chunks_of(x.numel, p.chunk);
        }
        list.first[k] = at;
        list.n = k;
        i += k;
        const int last = i >= n;
        if (at > 0 || last) {
            adam_kernel<<<std::max(at, 1), kBlock, 0, s>>>(list, a, norm, step, last);
            XSG_TRY_LAUNCH("adam_step");
        }
    }
    return XSG_OK;
}
