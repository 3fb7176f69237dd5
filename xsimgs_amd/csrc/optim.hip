// What a training step does behind the frame's backward: the global norm of many gradient tensors, clipping
// by it, and the Adam update that takes the clip factor and the packed visibility mask. No reference
// counterpart (the reference's trainer is outside its rendering library).
//
// All three run over a list of tensors cut into chunks of one length; a workgroup takes one chunk. The list
// travels in the kernels' arguments (no copy from the host, and a captured graph holds it by value): a short one
// in the arguments of each kernel, a long one piece by piece into the workspace, so that each pass stays one
// launch over all tensors. Sums are held in 64 bits and added in a fixed order, so a call's results are the
// same bits each time.
#include <math.h>

#include <algorithm>
#include <utility>

#include "xsg_common.h"

namespace {

constexpr int kBlock = 256;
constexpr int64_t kChunkUnit = 1024;      // chunks are multiples of this many elements
constexpr int64_t kTargetChunks = 2048;   // chunks of a call, when its tensors are long enough
constexpr int64_t kMaxChunk = 1 << 30;    // offsets inside a chunk are 32-bit
constexpr int64_t kMaxRow = 1 << 30;      // and so are rows under a mask
constexpr int64_t kMaxElements = (int64_t)1 << 48;
constexpr int kArgumentBytes = 3900;      // of a list, beside the other arguments in 4 KB
constexpr int kJoinMax = 4096;            // partial sums that every workgroup joins by itself

// Division of n < 2^31 by the row length: (mulhi(n, magic) + n) >> shift
struct RowDiv {
    uint32_t row, magic;
    uint32_t shift;
};

struct GradEntry {
    void* data;
    int64_t numel;
    const uint32_t* mask;
    uint32_t row, magic;      // elements to a mask bit, and its division
    uint8_t shift, dtype;
    XSG_HD const void* grad() const { return data; }
    XSG_HD int grad_dtype() const { return dtype; }
};

struct AdamEntry {
    void* param;
    const void* gradient;
    float *avg, *sq;
    int64_t numel;
    const uint32_t* mask;
    uint32_t row, magic;
    float lr, keep;           // keep: 1 - lr * weight decay
    uint8_t shift, pdtype, gdtype;
    XSG_HD const void* grad() const { return gradient; }
    XSG_HD int grad_dtype() const { return gdtype; }
};

template <typename E> constexpr int kInline = kArgumentBytes / (sizeof(E) + 4);

// first[t]: the first chunk of tensor t; first[n] = chunks
template <typename E> struct InlineList {
    E entry[kInline<E>];
    int32_t first[kInline<E> + 1];
    int32_t n, chunk, chunks;
};
template <typename E> struct TableList {
    const E* __restrict__ entry;
    const int32_t* __restrict__ first;
    int32_t n, chunk, chunks;
};
// a piece of a table on its way to the workspace
template <typename E> struct TablePiece {
    E entry[kInline<E>];
    int32_t first[kInline<E>];
    int32_t n;
};
static_assert(sizeof(InlineList<GradEntry>) <= 3920 && sizeof(InlineList<AdamEntry>) <= 3920 &&
                  sizeof(GradEntry) % 8 == 0 && sizeof(AdamEntry) % 8 == 0,
              "lists share 4 KB with the other arguments and are copied by words");

template <typename E>
__global__ __launch_bounds__(kBlock) void table_kernel(TablePiece<E> piece, E* __restrict__ entry,
                                                       int32_t* __restrict__ first, int last) {
    const uint64_t* const from = reinterpret_cast<const uint64_t*>(piece.entry);
    uint64_t* const to = reinterpret_cast<uint64_t*>(entry);
    for (int i = threadIdx.x; i < piece.n * (int)(sizeof(E) / 8); i += kBlock) to[i] = from[i];
    if (threadIdx.x < piece.n + last) first[threadIdx.x] = piece.first[threadIdx.x];
}

// round to nearest even; a NaN stays one
XSG_DEV uint32_t bf16_bits(float x) {
    const uint32_t u = __float_as_uint(x);
    if (x != x) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// Elements of one type, one at a time or four at a time from a place aligned for that (16 bytes of float32, 8
// of the others).
template <int DT> XSG_DEV float load1(const void* p, uint32_t i) {
    if (DT == XSG_DTYPE_F32) return ((const float*)p)[i];
    if (DT == XSG_DTYPE_BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
    return (float)((const _Float16*)p)[i];
}
template <int DT> XSG_DEV void store1(void* p, uint32_t i, float x) {
    if (DT == XSG_DTYPE_F32) ((float*)p)[i] = x;
    else if (DT == XSG_DTYPE_BF16) ((uint16_t*)p)[i] = (uint16_t)bf16_bits(x);
    else ((_Float16*)p)[i] = (_Float16)x;
}
template <int DT> XSG_DEV float4 load4(const void* p, uint32_t i) {
    if (DT == XSG_DTYPE_F32) return *reinterpret_cast<const float4*>((const float*)p + i);
    const uint2 u = *reinterpret_cast<const uint2*>((const uint16_t*)p + i);
    if (DT == XSG_DTYPE_BF16)
        return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                           __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
    union { uint2 u; _Float16 h[4]; } c{u};
    return make_float4((float)c.h[0], (float)c.h[1], (float)c.h[2], (float)c.h[3]);
}
template <int DT> XSG_DEV void store4(void* p, uint32_t i, float4 x) {
    if (DT == XSG_DTYPE_F32) {
        *reinterpret_cast<float4*>((float*)p + i) = x;
    } else if (DT == XSG_DTYPE_BF16) {
        *reinterpret_cast<uint2*>((uint16_t*)p + i) =
            make_uint2(bf16_bits(x.x) | bf16_bits(x.y) << 16, bf16_bits(x.z) | bf16_bits(x.w) << 16);
    } else {
        union { uint2 u; _Float16 h[4]; } c;
        c.h[0] = (_Float16)x.x; c.h[1] = (_Float16)x.y; c.h[2] = (_Float16)x.z; c.h[3] = (_Float16)x.w;
        *reinterpret_cast<uint2*>((uint16_t*)p + i) = c.u;
    }
}
XSG_HD uint32_t type_size(int dtype) { return dtype == XSG_DTYPE_F32 ? 4 : 2; }
XSG_DEV const void* at(const void* p, int64_t i, int dtype) { return (const char*)p + i * type_size(dtype); }
XSG_DEV void* at(void* p, int64_t i, int dtype) { return (char*)p + i * type_size(dtype); }

// Elements before p is aligned for four of its type at once (0 to 3).
XSG_DEV uint32_t phase_of(const void* p, int dtype) {
    const uint32_t e = (uint32_t)((uintptr_t)p / type_size(dtype)) & 3u;
    return (4u - e) & 3u;
}

constexpr uint32_t kRowBatch = 2048;   // rows a wavefront lists at once

// The packed mask seen from one chunk: element i of the chunk lies in row (rem + i) / row after word `words`
// and bit `bit`.
struct ChunkMask {
    const uint32_t* words;
    uint32_t bit, rem, row, magic, shift;
    uint16_t* list;   // in LDS, kRowBatch entries for each wavefront

    XSG_DEV void open(const uint32_t* mask, int64_t base, uint32_t row_, uint32_t magic_, uint32_t shift_) {
        const int64_t r = base / row_;
        words = mask + (r >> 5);
        bit = (uint32_t)(r & 31);
        rem = (uint32_t)(base - r * row_);
        row = row_;
        magic = magic_;
        shift = shift_;
    }
    XSG_DEV uint32_t quotient(uint32_t n) const { return (__umulhi(n, magic) + n) >> shift; }
    XSG_DEV bool one(uint32_t i) const {
        const uint32_t r = bit + quotient(rem + i);
        return (words[r >> 5] >> (r & 31)) & 1u;
    }
    // bit k: element i + k; all four lie in the chunk. Their rows span at most two words.
    XSG_DEV uint32_t four(uint32_t i) const {
        const uint32_t n = rem + i, q = quotient(n), r0 = bit + q;
        const uint32_t r3 = bit + quotient(n + 3);
        const uint64_t w = (uint64_t)words[r0 >> 5] | (uint64_t)words[r3 >> 5] << 32;
        uint32_t at = n - q * row, r = r0 & 31, keep = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            keep |= (uint32_t)((w >> r) & 1u) << k;
            if (++at == row) { at = 0; ++r; }
        }
        return keep;
    }
};

// The tensor whose chunks hold chunk b: the last one with first[t] <= b (empty tensors have no chunk). The
// wavefront looks at 64 places of what is left at once.
template <typename L> XSG_DEV int find_tensor(const L& list, int b) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = list.n;
    for (;;) {
        const int step = (n + 63) >> 6, i = lane * step;
        const int below = __popcll(__ballot(i < n && list.first[lo + min(i, n - 1)] <= b)) - 1;
        lo += below * step;
        n = min(step, n - below * step);
        if (step == 1) return __builtin_amdgcn_readfirstlane(lo);
    }
}

// Accumulation of one kind of norm. Sums are in 64 bits, where squares of any float32 stay finite and above
// zero. The largest magnitude is the largest of the values' bits without their sign, where a NaN is above
// infinity and so stays.
template <int NORM> struct Accum {
    double sum = 0.0;
    XSG_DEV void add(float x) {
        const double d = x;
        if (NORM == XSG_NORM_L2) sum = fma(d, d, sum);
        else sum += fabs(d);
    }
    XSG_DEV void join(const Accum& o) { sum += o.sum; }
    XSG_DEV double value() const { return sum; }
    XSG_DEV void join_value(double v) { sum += v; }
    XSG_DEV Accum shuffled(int d) const { Accum a; a.sum = __shfl_xor(sum, d); return a; }
    XSG_DEV double finish() const { return NORM == XSG_NORM_L2 ? sqrt(sum) : sum; }
};
template <> struct Accum<XSG_NORM_INF> {
    uint32_t bits = 0;
    XSG_DEV void add(float x) { bits = max(bits, __float_as_uint(x) & 0x7fffffffu); }
    XSG_DEV void join(const Accum& o) { bits = max(bits, o.bits); }
    XSG_DEV double value() const { return __uint_as_float(bits); }
    XSG_DEV void join_value(double v) { add((float)v); }
    XSG_DEV Accum shuffled(int d) const { Accum a; a.bits = __shfl_xor(bits, d); return a; }
    XSG_DEV double finish() const { return value(); }
};

// The workgroup's joined value, in every thread; the order is fixed.
template <int NORM> XSG_DEV Accum<NORM> block_join(Accum<NORM> v) {
    __shared__ double part[kBlock / 64];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v.join(v.shuffled(d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v.value();
    __syncthreads();
    Accum<NORM> all;
#pragma unroll
    for (int w = 0; w < kBlock / 64; ++w) all.join_value(part[w]);
    return all;
}

// A chunk's elements: `head` single ones up to the first aligned group of four, `groups` groups, `tail`
// single ones. Bodies take (first element, group in mask bits or 15).
struct ChunkSpan {
    uint32_t head, groups, tail;
    XSG_DEV ChunkSpan(uint32_t count, uint32_t phase) {
        head = min(phase, count);
        groups = (count - head) >> 2;
        tail = (count - head) & 3u;
    }
    XSG_DEV uint32_t tail_at() const { return head + 4 * groups; }
};

constexpr int kUnroll = 4;   // groups in flight per thread

// one(i): a single element; many(i[], keep[]): kUnroll groups, of which those with keep 0 are left out
template <bool MASK, typename One, typename Many>
XSG_DEV void for_chunk(const ChunkSpan& span, const ChunkMask& mask, One&& one, Many&& many) {
    for (uint32_t g = threadIdx.x; g < span.groups; g += kBlock * kUnroll) {
        uint32_t i[kUnroll], keep[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            i[u] = span.head + 4 * (g + u * kBlock);
            keep[u] = g + u * kBlock < span.groups ? (MASK ? mask.four(i[u]) : 15u) : 0u;
        }
        many(i, keep);
    }
    if (threadIdx.x < span.head && (!MASK || mask.one(threadIdx.x))) one(threadIdx.x);
    const uint32_t i = span.tail_at() + threadIdx.x;
    if (threadIdx.x < span.tail && (!MASK || mask.one(i))) one(i);
}

// Under a mask of short rows each wavefront lists the kept rows of its share of the chunk (a mask word a lane, so
// up to 2048 rows for one load's latency) and then walks their elements alone, VEC at a time, so that lanes are
// busy and loads in flight however few rows are kept.
// many(i[], on[]): UNROLL units of VEC elements from element i, of which those not on are left out.
constexpr uint32_t kShortRow = 128;

template <int VEC, int UNROLL, typename Many>
XSG_DEV void for_kept_rows(const ChunkMask& mask, uint32_t count, Many&& many) {
    uint16_t* const list = mask.list + (threadIdx.x >> 6) * kRowBatch;
    const uint32_t lane = threadIdx.x & 63, rows = mask.quotient(mask.rem + count - 1) + 1;
    const uint32_t share = (rows + kBlock / 64 - 1) / (kBlock / 64);
    // the wavefront's rows as bits from mask.words[0] on
    const uint32_t lo = mask.bit + min((threadIdx.x >> 6) * share, rows);
    const uint32_t hi = min(lo + share, mask.bit + rows);
    const uint32_t units = mask.row / VEC, magic = 0xffffffffu / units + 1;   // exact: units^2 kRowBatch < 2^32
    const auto word_of = [&](uint32_t first) {   // bits of rows outside lo..hi are cleared
        const uint32_t at = first + 32 * lane;
        if (at >= hi) return 0u;
        uint32_t w = mask.words[at >> 5];
        if (at < lo) w &= 0xffffffffu << (lo - at);   // lo lies in the first word
        return hi - at < 32 ? w & ~(0xffffffffu << (hi - at)) : w;
    };
    uint32_t next = word_of(lo & ~31u);
    for (uint32_t batch = lo & ~31u; batch < hi; batch += kRowBatch) {
        uint32_t word = next, upto = (uint32_t)__popc(word);
        next = word_of(batch + kRowBatch);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t below = __shfl_up(upto, d);
            if (lane >= d) upto += below;
        }
        const uint32_t n = __shfl(upto, 63);
        for (uint32_t k = upto - (uint32_t)__popc(word); word; word &= word - 1)
            list[k++] = (uint16_t)(32 * lane + __ffs(word) - 1);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const uint32_t total = n * units;
        for (uint32_t w0 = lane; w0 < total; w0 += 64 * UNROLL) {
            uint32_t i[UNROLL];
            bool on[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const uint32_t w = w0 + 64 * u;
                on[u] = w < total;
                const uint32_t q = units == 1 ? w : __umulhi(w, magic);
                const uint32_t r = batch + (on[u] ? list[q] : 0u) - mask.bit;
                // the chunk's first and last row may lie in it in part; before it the difference wraps
                i[u] = r * mask.row + (w - q * units) * VEC - mask.rem;
                on[u] = on[u] && i[u] < count;
            }
            many(i, on);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

template <int NORM, int DT>
XSG_DEV Accum<NORM> rows_norm(const void* p, uint32_t count, bool whole, const ChunkMask& mask) {
    Accum<NORM> acc[4];
    if (whole) {
        for_kept_rows<4, 4>(mask, count, [&](const uint32_t* i, const bool* on) {
            float4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = on[u] ? load4<DT>(p, i[u]) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                acc[u].add(x[u].x);
                acc[u].add(x[u].y);
                acc[u].add(x[u].z);
                acc[u].add(x[u].w);
            }
        });
    } else {
        for_kept_rows<1, 4>(mask, count, [&](const uint32_t* i, const bool* on) {
            float x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = on[u] ? load1<DT>(p, i[u]) : 0.f;
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[u].add(x[u]);
        });
    }
#pragma unroll
    for (int u = 1; u < 4; ++u) acc[0].join(acc[u]);
    return acc[0];
}

template <int DT> XSG_DEV void rows_scale(void* p, float c, uint32_t count, bool whole, const ChunkMask& mask) {
    if (whole) {
        for_kept_rows<4, 4>(mask, count, [&](const uint32_t* i, const bool* on) {
            float4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (on[u]) x[u] = load4<DT>(p, i[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (on[u]) store4<DT>(p, i[u], make_float4(x[u].x * c, x[u].y * c, x[u].z * c, x[u].w * c));
        });
    } else {
        for_kept_rows<1, 4>(mask, count, [&](const uint32_t* i, const bool* on) {
            float x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (on[u]) x[u] = load1<DT>(p, i[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (on[u]) store1<DT>(p, i[u], x[u] * c);
        });
    }
}

template <int NORM, int DT, bool MASK>
XSG_DEV Accum<NORM> chunk_norm(const void* p, const ChunkSpan& span, const ChunkMask& mask) {
    Accum<NORM> acc[kUnroll];
    for_chunk<MASK>(span, mask, [&](uint32_t i) { acc[0].add(load1<DT>(p, i)); },
                    [&](const uint32_t* i, const uint32_t* keep) {
        float4 x[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) x[u] = keep[u] ? load4<DT>(p, i[u]) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            acc[u].add(!MASK || (keep[u] & 1) ? x[u].x : 0.f);
            acc[u].add(!MASK || (keep[u] & 2) ? x[u].y : 0.f);
            acc[u].add(!MASK || (keep[u] & 4) ? x[u].z : 0.f);
            acc[u].add(!MASK || (keep[u] & 8) ? x[u].w : 0.f);
        }
    });
#pragma unroll
    for (int u = 1; u < kUnroll; ++u) acc[0].join(acc[u]);
    return acc[0];
}

// calls f with the type as a constant
template <typename F> XSG_DEV void with_type(int dtype, F&& f) {
    if (dtype == XSG_DTYPE_F32) f(std::integral_constant<int, XSG_DTYPE_F32>{});
    else if (dtype == XSG_DTYPE_BF16) f(std::integral_constant<int, XSG_DTYPE_BF16>{});
    else f(std::integral_constant<int, XSG_DTYPE_F16>{});
}

// What a workgroup does first: its chunk of its tensor.
struct Chunk {
    int64_t base;
    uint32_t count;
    template <typename L, typename E> XSG_DEV Chunk(const L& list, const E& e, int b, int t) {
        base = (int64_t)(b - list.first[t]) * list.chunk;
        count = (uint32_t)min((int64_t)list.chunk, e.numel - base);
    }
};

// `step`, unless null, counts one step more; the launches behind this one read it.
template <int NORM, typename L>
__global__ __launch_bounds__(kBlock) void norm_partial_kernel(L list, double* __restrict__ partial, int64_t* step) {
    const int b = blockIdx.x;
    if (step && b == 0 && threadIdx.x == 0) *step += 1;
    if (b >= list.chunks) return;   // no elements at all
    const int t = find_tensor(list, b);
    const auto& e = list.entry[t];
    const Chunk chunk(list, e, b, t);
    const int dtype = e.grad_dtype();
    const void* p = at(e.grad(), chunk.base, dtype);
    const ChunkSpan span(chunk.count, phase_of(p, dtype));
    ChunkMask mask;
    __shared__ uint16_t listed[kBlock / 64 * kRowBatch];
    mask.list = listed;
    if (e.mask) mask.open(e.mask, chunk.base, e.row, e.magic, e.shift);
    Accum<NORM> acc;
    with_type(dtype, [&](auto dt) {
        if (!e.mask) acc = chunk_norm<NORM, dt.value, false>(p, span, mask);
        else if (mask.row > kShortRow) acc = chunk_norm<NORM, dt.value, true>(p, span, mask);
        else acc = rows_norm<NORM, dt.value>(p, chunk.count, span.head == 0 && mask.row % 4 == 0, mask);
    });
    acc = block_join<NORM>(acc);
    if (threadIdx.x == 0) partial[b] = acc.value();
}

template <int NORM> XSG_DEV Accum<NORM> join_partials(const double* __restrict__ partial, int n) {
    Accum<NORM> acc;
    for (int i = threadIdx.x; i < n; i += kBlock) acc.join_value(partial[i]);
    return block_join<NORM>(acc);
}

// The norm from the partial sums of its chunks, in every thread of the workgroup.
XSG_DEV double norm_of(const double* __restrict__ partial, int n, int norm) {
    if (norm == XSG_NORM_L2) return join_partials<XSG_NORM_L2>(partial, n).finish();
    if (norm == XSG_NORM_L1) return join_partials<XSG_NORM_L1>(partial, n).finish();
    return join_partials<XSG_NORM_INF>(partial, n).finish();
}

// Many partial sums become one, where each workgroup of the next launch would join them all again.
__global__ __launch_bounds__(kBlock) void norm_reduce_kernel(const double* __restrict__ partial, int n, int norm,
                                                             double* __restrict__ one) {
    double v;
    if (norm == XSG_NORM_L2) v = join_partials<XSG_NORM_L2>(partial, n).value();
    else if (norm == XSG_NORM_L1) v = join_partials<XSG_NORM_L1>(partial, n).value();
    else v = join_partials<XSG_NORM_INF>(partial, n).value();
    if (threadIdx.x == 0) *one = v;
}

__global__ __launch_bounds__(kBlock) void norm_total_kernel(const double* __restrict__ partial, int n, int norm,
                                                            float* __restrict__ total) {
    const double v = norm_of(partial, n, norm);
    if (threadIdx.x == 0) *total = (float)v;
}

// Block t < n: the norm of tensor t. Block n: the norm over all of them.
template <typename L>
__global__ __launch_bounds__(kBlock) void norm_each_kernel(L list, const double* __restrict__ partial, int norm,
                                                           float* __restrict__ total, float* __restrict__ each) {
    const int t = blockIdx.x;
    const int lo = t < list.n ? list.first[t] : 0, hi = t < list.n ? list.first[t + 1] : list.chunks;
    const double v = norm_of(partial + lo, hi - lo, norm);
    if (threadIdx.x == 0) *(t < list.n ? each + t : total) = (float)v;
}

// min(1, max_norm / (norm + eps)); a NaN norm gives NaN, an infinite one 0
XSG_DEV float clip_factor(double norm, double max_norm, double eps) {
    const double c = max_norm / (norm + eps);
    return c > 1.0 ? 1.0f : (float)c;
}

template <int DT, bool MASK>
XSG_DEV void chunk_scale(void* p, float c, const ChunkSpan& span, const ChunkMask& mask) {
    for_chunk<MASK>(span, mask, [&](uint32_t i) { store1<DT>(p, i, load1<DT>(p, i) * c); },
                    [&](const uint32_t* i, const uint32_t* keep) {
        float4 x[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (keep[u]) x[u] = load4<DT>(p, i[u]);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const float4 y = make_float4(x[u].x * c, x[u].y * c, x[u].z * c, x[u].w * c);
            if (keep[u] == 15u) {
                store4<DT>(p, i[u], y);
            } else if (keep[u]) {
                if (keep[u] & 1) store1<DT>(p, i[u], y.x);
                if (keep[u] & 2) store1<DT>(p, i[u] + 1, y.y);
                if (keep[u] & 4) store1<DT>(p, i[u] + 2, y.z);
                if (keep[u] & 8) store1<DT>(p, i[u] + 3, y.w);
            }
        }
    });
}

// The norm that a launch clips by: partial sums, how many, and what kind.
struct NormParts {
    const double* __restrict__ partial;
    int n, norm;
};

template <typename L>
__global__ __launch_bounds__(kBlock) void clip_scale_kernel(L list, NormParts parts, double max_norm, double eps,
                                                            float* __restrict__ total) {
    const double norm = norm_of(parts.partial, parts.n, parts.norm);
    const int b = blockIdx.x;
    if (b == 0 && threadIdx.x == 0) *total = (float)norm;
    const float c = clip_factor(norm, max_norm, eps);
    if (c == 1.0f || b >= list.chunks) return;   // the values stay as they are
    const int t = find_tensor(list, b);
    const auto& e = list.entry[t];
    const Chunk chunk(list, e, b, t);
    const int dtype = e.dtype;
    void* p = at(e.data, chunk.base, dtype);
    const ChunkSpan span(chunk.count, phase_of(p, dtype));
    ChunkMask mask;
    __shared__ uint16_t listed[kBlock / 64 * kRowBatch];
    mask.list = listed;
    if (e.mask) mask.open(e.mask, chunk.base, e.row, e.magic, e.shift);
    with_type(dtype, [&](auto dt) {
        if (!e.mask) chunk_scale<dt.value, false>(p, c, span, mask);
        else if (mask.row > kShortRow) chunk_scale<dt.value, true>(p, c, span, mask);
        else rows_scale<dt.value>(p, c, chunk.count, span.head == 0 && mask.row % 4 == 0, mask);
    });
}

struct AdamScalars {
    double log_beta1, log_beta2;   // natural logarithms
    float beta2, one_minus_beta1, one_minus_beta2, eps;
    int clip, skip_nonfinite;
    double max_norm;
};
constexpr double kAdamClipEps = 1e-6;

// Without a norm to compute, the step is counted by a launch of its own.
__global__ void adam_count_kernel(int64_t* step) { *step += 1; }

// One value of the update; rate: lr / (1 - beta1^t), root: 1 / sqrt(1 - beta2^t)
struct AdamTerms {
    float beta2, one_minus_beta1, one_minus_beta2, eps, c, rate, root, keep;
    XSG_DEV void update(float& p, float g, float& m, float& v) const {
        g *= c;
        m += one_minus_beta1 * (g - m);
        v = beta2 * v + one_minus_beta2 * g * g;
        p = p * keep - rate * m / (sqrtf(v) * root + eps);
    }
};

struct AdamArrays {
    void* p;
    const void* g;
    float *m, *v;
};

template <int PT, int GT> XSG_DEV void adam_one(const AdamArrays& a, const AdamTerms& s, uint32_t i) {
    float p = load1<PT>(a.p, i), m = a.m[i], v = a.v[i];
    s.update(p, load1<GT>(a.g, i), m, v);
    store1<PT>(a.p, i, p);
    a.m[i] = m;
    a.v[i] = v;
}

constexpr int kAdamUnroll = 2;

template <int PT, int GT, bool MASK>
XSG_DEV void chunk_adam(const AdamArrays& a, const AdamTerms& s, const ChunkSpan& span, const ChunkMask& mask) {
    for (uint32_t g0 = threadIdx.x; g0 < span.groups; g0 += kBlock * kAdamUnroll) {
        uint32_t i[kAdamUnroll], keep[kAdamUnroll];
        float4 p[kAdamUnroll], g[kAdamUnroll], m[kAdamUnroll], v[kAdamUnroll];
#pragma unroll
        for (int u = 0; u < kAdamUnroll; ++u) {
            i[u] = span.head + 4 * (g0 + u * kBlock);
            keep[u] = g0 + u * kBlock < span.groups ? (MASK ? mask.four(i[u]) : 15u) : 0u;
        }
#pragma unroll
        for (int u = 0; u < kAdamUnroll; ++u) {
            if (keep[u]) {
                p[u] = load4<PT>(a.p, i[u]);
                g[u] = load4<GT>(a.g, i[u]);
                m[u] = load4<XSG_DTYPE_F32>(a.m, i[u]);
                v[u] = load4<XSG_DTYPE_F32>(a.v, i[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < kAdamUnroll; ++u) {
            if (!keep[u]) continue;
            s.update(p[u].x, g[u].x, m[u].x, v[u].x);
            s.update(p[u].y, g[u].y, m[u].y, v[u].y);
            s.update(p[u].z, g[u].z, m[u].z, v[u].z);
            s.update(p[u].w, g[u].w, m[u].w, v[u].w);
            if (keep[u] == 15u) {
                store4<PT>(a.p, i[u], p[u]);
                store4<XSG_DTYPE_F32>(a.m, i[u], m[u]);
                store4<XSG_DTYPE_F32>(a.v, i[u], v[u]);
            } else {
                const float pe[4] = {p[u].x, p[u].y, p[u].z, p[u].w}, me[4] = {m[u].x, m[u].y, m[u].z, m[u].w},
                            ve[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (!((keep[u] >> k) & 1)) continue;
                    store1<PT>(a.p, i[u] + k, pe[k]);
                    a.m[i[u] + k] = me[k];
                    a.v[i[u] + k] = ve[k];
                }
            }
        }
    }
    if (threadIdx.x < span.head && (!MASK || mask.one(threadIdx.x))) adam_one<PT, GT>(a, s, threadIdx.x);
    for (uint32_t i = span.tail_at() + threadIdx.x, end = span.tail_at() + span.tail; i < end; i += kBlock)
        if (!MASK || mask.one(i)) adam_one<PT, GT>(a, s, i);
}

template <int PT, int GT>
XSG_DEV void rows_adam(const AdamArrays& a, const AdamTerms& s, uint32_t count, bool whole, const ChunkMask& mask) {
    if (whole) {
        for_kept_rows<4, kAdamUnroll>(mask, count, [&](const uint32_t* i, const bool* on) {
            float4 p[kAdamUnroll], g[kAdamUnroll], m[kAdamUnroll], v[kAdamUnroll];
#pragma unroll
            for (int u = 0; u < kAdamUnroll; ++u) {
                if (!on[u]) continue;
                p[u] = load4<PT>(a.p, i[u]);
                g[u] = load4<GT>(a.g, i[u]);
                m[u] = load4<XSG_DTYPE_F32>(a.m, i[u]);
                v[u] = load4<XSG_DTYPE_F32>(a.v, i[u]);
            }
#pragma unroll
            for (int u = 0; u < kAdamUnroll; ++u) {
                if (!on[u]) continue;
                s.update(p[u].x, g[u].x, m[u].x, v[u].x);
                s.update(p[u].y, g[u].y, m[u].y, v[u].y);
                s.update(p[u].z, g[u].z, m[u].z, v[u].z);
                s.update(p[u].w, g[u].w, m[u].w, v[u].w);
                store4<PT>(a.p, i[u], p[u]);
                store4<XSG_DTYPE_F32>(a.m, i[u], m[u]);
                store4<XSG_DTYPE_F32>(a.v, i[u], v[u]);
            }
        });
    } else {
        for_kept_rows<1, 4>(mask, count, [&](const uint32_t* i, const bool* on) {
            float p[4], g[4], m[4], v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (!on[u]) continue;
                p[u] = load1<PT>(a.p, i[u]);
                g[u] = load1<GT>(a.g, i[u]);
                m[u] = a.m[i[u]];
                v[u] = a.v[i[u]];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (!on[u]) continue;
                s.update(p[u], g[u], m[u], v[u]);
                store1<PT>(a.p, i[u], p[u]);
                a.m[i[u]] = m[u];
                a.v[i[u]] = v[u];
            }
        });
    }
}

// parts.n < 0: no norm. The counter already counts this step; it is taken back where the step is not taken.
template <typename L>
__global__ __launch_bounds__(kBlock) void adam_kernel(L list, AdamScalars s, NormParts parts, int64_t* step,
                                                      float* __restrict__ total) {
    const int b = blockIdx.x;
    AdamTerms terms;
    terms.c = 1.0f;
    if (parts.n >= 0) {
        const double norm = norm_of(parts.partial, parts.n, parts.norm);
        if (total && b == 0 && threadIdx.x == 0) *total = (float)norm;
        if (s.skip_nonfinite && !(norm < (double)INFINITY)) {
            if (b == 0 && threadIdx.x == 0) *step -= 1;   // no other workgroup reads the counter in this case
            return;
        }
        if (s.clip) terms.c = clip_factor(norm, s.max_norm, kAdamClipEps);
    }
    if (b >= list.chunks) return;
    const int t = find_tensor(list, b);
    const auto& e = list.entry[t];
    const Chunk chunk(list, e, b, t);
    const double k = (double)*step;
    // 1 - beta^k without the cancellation
    terms.rate = (float)(e.lr / -expm1(k * s.log_beta1));
    terms.root = (float)(1.0 / sqrt(-expm1(k * s.log_beta2)));
    terms.beta2 = s.beta2;
    terms.one_minus_beta1 = s.one_minus_beta1;
    terms.one_minus_beta2 = s.one_minus_beta2;
    terms.eps = s.eps;
    terms.keep = e.keep;
    const int pt = e.pdtype, gt = e.gdtype;
    const AdamArrays a{at(e.param, chunk.base, pt), at(e.gradient, chunk.base, gt), e.avg + chunk.base,
                       e.sq + chunk.base};
    const uint32_t phase = phase_of(a.p, pt);
    ChunkSpan span(chunk.count, phase);
    if (phase != phase_of(a.g, gt) || phase != phase_of(a.m, XSG_DTYPE_F32) || phase != phase_of(a.v, XSG_DTYPE_F32)) {
        span.head = span.groups = 0;   // the arrays are not aligned alike: one element at a time
        span.tail = chunk.count;
    }
    const bool whole = span.groups > 0 && span.head == 0 && e.row % 4 == 0;   // rows of whole groups
    ChunkMask mask;
    __shared__ uint16_t listed[kBlock / 64 * kRowBatch];
    mask.list = listed;
    if (e.mask) mask.open(e.mask, chunk.base, e.row, e.magic, e.shift);
    with_type(pt, [&](auto p) {
        with_type(gt, [&](auto g) {
            if (!e.mask) chunk_adam<p.value, g.value, false>(a, terms, span, mask);
            else if (mask.row > kShortRow) chunk_adam<p.value, g.value, true>(a, terms, span, mask);
            else rows_adam<p.value, g.value>(a, terms, chunk.count, whole, mask);
        });
    });
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

// rows of a mask: d = 2^shift needs no magic; else magic = floor(2^32 (2^shift - d) / d) + 1, 2^(shift-1) < d < 2^shift
RowDiv row_div(int64_t numel, const void* mask, int64_t rows) {
    const uint32_t d = mask && numel ? (uint32_t)(numel / rows) : 1u;
    uint32_t shift = 0;
    while (((uint64_t)1 << shift) < d) ++shift;
    return RowDiv{d, (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1), shift};
}

xsg_grad_tensor grad_of(const xsg_grad_tensor& x) { return x; }
xsg_grad_tensor grad_of(const xsg_adam_tensor& x) {
    return xsg_grad_tensor{const_cast<void*>(x.grad), x.numel, x.mask, x.rows, x.grad_dtype};
}

GradEntry entry_of(const xsg_grad_tensor& x) {
    const RowDiv div = row_div(x.numel, x.mask, x.rows);
    return GradEntry{x.data, x.numel, x.numel ? x.mask : nullptr, div.row, div.magic, (uint8_t)div.shift, (uint8_t)x.dtype};
}
AdamEntry entry_of(const xsg_adam_tensor& x) {
    const RowDiv div = row_div(x.numel, x.mask, x.rows);
    return AdamEntry{x.param, x.grad, x.exp_avg, x.exp_avg_sq, x.numel, x.numel ? x.mask : nullptr, div.row, div.magic,
                     (float)x.lr, (float)(1.0 - x.lr * x.weight_decay), (uint8_t)div.shift, (uint8_t)x.param_dtype,
                     (uint8_t)x.grad_dtype};
}
template <typename T> using EntryOf = decltype(entry_of(std::declval<const T&>()));

// How a call is cut, and where things lie in its workspace: one double for a reduced norm, then (256 bytes on)
// a partial sum per chunk, then a long list's table.
struct Plan {
    int64_t elements = 0, chunk = 0, chunks = 0;
    bool table = false;
    size_t first_at = 0, entry_at = 0, bytes = 0;
};

size_t aligned(size_t x) { return (x + 255) / 256 * 256; }

template <typename T> int make_plan(const T* ts, int n, const char* who, bool norm, Plan* p) {
    if (n < 0 || (n > 0 && !ts)) return xsg_fail(XSG_ERR_INVALID, "%s: null or negative list of tensors", who);
    for (int i = 0; i < n; ++i) {
        if (ts[i].numel < 0) return xsg_fail(XSG_ERR_INVALID, "%s: tensor %d has a negative size", who, i);
        if (ts[i].numel > kMaxElements - p->elements) return xsg_fail(XSG_ERR_INVALID, "%s: too many elements", who);
        p->elements += ts[i].numel;
    }
    p->chunk = chunk_for(p->elements);
    for (int i = 0; i < n; ++i) p->chunks += chunks_of(ts[i].numel, p->chunk);
    if (p->chunks > kMaxChunk) return xsg_fail(XSG_ERR_INVALID, "%s: too many tensors", who);
    p->table = n > kInline<EntryOf<T>>;
    p->bytes = norm ? 256 + aligned((size_t)p->chunks * sizeof(double)) : 0;
    if (p->table) {
        p->first_at = p->bytes;
        p->entry_at = p->first_at + aligned(((size_t)n + 1) * sizeof(int32_t));
        p->bytes = p->entry_at + aligned((size_t)n * sizeof(EntryOf<T>));
    }
    return XSG_OK;
}

template <typename T> void fill_inline(const T* ts, int n, const Plan& p, InlineList<EntryOf<T>>* list) {
    int32_t at = 0;
    for (int i = 0; i < n; ++i) {
        list->entry[i] = entry_of(ts[i]);
        list->first[i] = at;
        at += (int32_t)chunks_of(ts[i].numel, p.chunk);
    }
    list->first[n] = at;
    list->n = n;
    list->chunk = (int32_t)p.chunk;
    list->chunks = at;
}

template <typename T>
int send_table(const T* ts, int n, const Plan& p, void* ws, hipStream_t s, TableList<EntryOf<T>>* list) {
    using E = EntryOf<T>;
    int32_t* const first = (int32_t*)((char*)ws + p.first_at);
    E* const entry = (E*)((char*)ws + p.entry_at);
    TablePiece<E> piece;
    int32_t at = 0;
    // first[n], the end, goes as one more tensor's first chunk
    for (int i = 0; i <= n;) {
        const int i0 = i;
        for (piece.n = 0; piece.n < kInline<E> && i < n; ++i, ++piece.n) {
            piece.entry[piece.n] = entry_of(ts[i]);
            piece.first[piece.n] = at;
            at += (int32_t)chunks_of(ts[i].numel, p.chunk);
        }
        const bool last = i == n && piece.n < kInline<E>;
        if (last) piece.first[piece.n] = at;
        table_kernel<E><<<1, kBlock, 0, s>>>(piece, entry + i0, first + i0, last);
        XSG_TRY_LAUNCH("table");
        if (last) break;
    }
    *list = TableList<E>{entry, first, n, (int32_t)p.chunk, at};
    return XSG_OK;
}

// calls f with the list as the kernels take it
template <typename T, typename F> int with_list(const T* ts, int n, const Plan& p, void* ws, hipStream_t s, F&& f) {
    if (p.table) {
        TableList<EntryOf<T>> list;
        const int rc = send_table(ts, n, p, ws, s, &list);
        return rc == XSG_OK ? f(list) : rc;
    }
    InlineList<EntryOf<T>> list;
    fill_inline(ts, n, p, &list);
    return f(list);
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

double* partials(void* ws) { return (double*)((char*)ws + 256); }

template <typename L>
int launch_partials(const L& list, int norm, void* ws, int64_t* step, hipStream_t s) {
    with_norm(norm, [&](auto kind) {
        norm_partial_kernel<kind.value><<<std::max(list.chunks, 1), kBlock, 0, s>>>(list, partials(ws), step);
    });
    return xsg_launch_status("grad_norm");
}

// the partial sums as the next launch's workgroups join them
int join_parts(int chunks, int norm, void* ws, hipStream_t s, NormParts* parts) {
    *parts = NormParts{partials(ws), chunks, norm};
    if (chunks <= kJoinMax) return XSG_OK;
    norm_reduce_kernel<<<1, kBlock, 0, s>>>(partials(ws), chunks, norm, (double*)ws);
    *parts = NormParts{(const double*)ws, 1, norm};
    return xsg_launch_status("grad_norm");
}

}  // namespace

extern "C" size_t xsg_grad_norm_workspace_bytes(const xsg_grad_tensor* ts, int n) {
    Plan p;
    return make_plan(ts, n, "grad_norm", true, &p) == XSG_OK ? p.bytes : 0;
}

extern "C" int xsg_grad_norm(const xsg_grad_tensor* ts, int n, int norm, float* total, float* each, void* workspace,
                             xsg_stream_t stream) {
    Plan p;
    int rc = make_plan(ts, n, "grad_norm", true, &p);
    if (rc == XSG_OK) rc = check_list(ts, n, norm, "grad_norm");
    if (rc != XSG_OK) return rc;
    if (!total || !workspace) return xsg_fail(XSG_ERR_INVALID, "grad_norm: null output or workspace");
    rc = xsg_check_workspace(workspace, "grad_norm");
    if (rc != XSG_OK) return rc;
    const hipStream_t s = (hipStream_t)stream;
    return with_list(ts, n, p, workspace, s, [&](const auto& list) {
        const int status = launch_partials(list, norm, workspace, nullptr, s);
        if (status != XSG_OK) return status;
        const double* const partial = partials(workspace);
        if (each) norm_each_kernel<<<n + 1, kBlock, 0, s>>>(list, partial, norm, total, each);
        else norm_total_kernel<<<1, kBlock, 0, s>>>(partial, (int)p.chunks, norm, total);
        return xsg_launch_status("grad_norm");
    });
}

extern "C" int xsg_clip_grads(const xsg_grad_tensor* ts, int n, int norm, double max_norm, double eps, float* total,
                              void* workspace, xsg_stream_t stream) {
    Plan p;
    int rc = make_plan(ts, n, "clip_grads", true, &p);
    if (rc == XSG_OK) rc = check_list(ts, n, norm, "clip_grads");
    if (rc != XSG_OK) return rc;
    if (!(max_norm >= 0.0) || !(eps >= 0.0))
        return xsg_fail(XSG_ERR_INVALID, "clip_grads: max_norm %g and eps %g must not be negative", max_norm, eps);
    if (!total || !workspace) return xsg_fail(XSG_ERR_INVALID, "clip_grads: null output or workspace");
    rc = xsg_check_workspace(workspace, "clip_grads");
    if (rc != XSG_OK) return rc;
    const hipStream_t s = (hipStream_t)stream;
    return with_list(ts, n, p, workspace, s, [&](const auto& list) {
        int status = launch_partials(list, norm, workspace, nullptr, s);
        if (status != XSG_OK) return status;
        NormParts parts;
        status = join_parts(list.chunks, norm, workspace, s, &parts);
        if (status != XSG_OK) return status;
        clip_scale_kernel<<<std::max(list.chunks, 1), kBlock, 0, s>>>(list, parts, max_norm, eps, total);
        return xsg_launch_status("clip_grads");
    });
}

extern "C" size_t xsg_adam_step_workspace_bytes(const xsg_adam_tensor* ts, int n, const xsg_adam_options* o) {
    Plan p;
    return o && make_plan(ts, n, "adam_step", o->clip || o->skip_nonfinite, &p) == XSG_OK ? p.bytes : 0;
}

extern "C" int xsg_adam_step(const xsg_adam_tensor* ts, int n, const xsg_adam_options* o, int64_t* step, float* total,
                             void* workspace, xsg_stream_t stream) {
    if (!o || !step) return xsg_fail(XSG_ERR_INVALID, "adam_step: null options or step counter");
    const bool needs_norm = o->clip || o->skip_nonfinite;
    Plan p;
    int rc = make_plan(ts, n, "adam_step", needs_norm, &p);
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
    rc = check_list(ts, n, needs_norm ? o->norm : XSG_NORM_L2, "adam_step");
    if (rc != XSG_OK) return rc;
    if (p.bytes > 0) {
        if (!workspace) return xsg_fail(XSG_ERR_INVALID, "adam_step: null workspace");
        rc = xsg_check_workspace(workspace, "adam_step");
        if (rc != XSG_OK) return rc;
    }
    AdamScalars a;
    a.log_beta1 = log(o->beta1);   // beta 0: -inf, and 1 - beta^k is 1
    a.log_beta2 = log(o->beta2);
    a.beta2 = (float)o->beta2;
    a.one_minus_beta1 = (float)(1.0 - o->beta1);
    a.one_minus_beta2 = (float)(1.0 - o->beta2);
    a.eps = (float)o->eps;
    a.clip = o->clip;
    a.skip_nonfinite = o->skip_nonfinite;
    a.max_norm = o->max_norm;
    const hipStream_t s = (hipStream_t)stream;
    return with_list(ts, n, p, workspace, s, [&](const auto& list) {
        NormParts parts{nullptr, -1, o->norm};
        int status;
        if (needs_norm) {
            status = launch_partials(list, o->norm, workspace, step, s);
            if (status == XSG_OK) status = join_parts(list.chunks, o->norm, workspace, s, &parts);
        } else {
            adam_count_kernel<<<1, 1, 0, s>>>(step);
            status = xsg_launch_status("adam_step");
        }
        if (status != XSG_OK) return status;
        adam_kernel<<<std::max(list.chunks, 1), kBlock, 0, s>>>(list, a, parts, step, total);
        return xsg_launch_status("adam_step");
    });
}
