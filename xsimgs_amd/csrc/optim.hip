// What a training step does behind the frame's backward: the global norm of many gradient tensors, clipping
// by it, and the Adam update that takes the clip factor and the packed visibility mask. No reference
// counterpart (the reference's trainer is outside its rendering library).
//
// All three run over a list of tensors cut into chunks of one length; a workgroup takes one chunk. The list
// travels in the kernels' arguments (no copy from the host, and a captured graph holds it by value): a short one
// in the arguments of each kernel, a long one piece by piece into the workspace, so that each pass stays one
// launch over all tensors. Sums are held in 64 bits and added in a fixed order, so a call's results are the
// same bits each time. Scaling and update are computed in 32 bits and rounded once, to the type the tensor has;
// moments stay in 32 bits, since squares of half-precision gradients would fall out of 16 (1e-4 squared).
#include <math.h>

#include <algorithm>
#include <utility>

#include "xsg_common.h"

namespace {

constexpr int kBlock = 256;
constexpr int64_t kChunkUnit = 1024;      // chunks are multiples of this many elements
// Workgroups that share out the elements of a call whose tensors are long enough. Dense tensors stream best from
// four long runs to a CU (4 M Gaussians: clip 442 us, 456 with eight), under masks the lists of rows are latency that
// eight hide (1 M with 14 % kept: norm 19 us, 27 with four).
constexpr int64_t kDenseChunks = 1024, kMaskedChunks = 2048;
// Longest chunk of a call that writes more than the caches hold: many short workgroups follow each other through
// memory, where few long ones write in as many places at once (an update of 236 M elements: 2048 chunks 1310 us,
// 57618 chunks 1230, around the caches 1145).
constexpr int64_t kWriteChunk = 4096;
// Such chunks to one of a masked tensor, of which little is kept (1 M Gaussians with 14 % kept: one 148 us, two 119,
// four and eight 114; 101 nodes with 40 %: one and two 148, four 151, eight 166).
constexpr int64_t kMaskedFactor = 4;
constexpr int64_t kMaxChunk = 1 << 26;    // offsets inside a chunk are 32-bit, in bytes
constexpr int64_t kCacheBytes = (int64_t)256 << 20;   // of the last-level cache
constexpr int64_t kMaxRow = 1 << 30;      // and so are rows under a mask
constexpr int64_t kMaxElements = (int64_t)1 << 41;
constexpr int64_t kMaxChunks = (1 << 24) - 1;   // a launch of one workgroup each holds fewer than 2^32 threads
constexpr int64_t kFarChunks = 1 << 22;         // of long writing calls, beside a last short one of every tensor
constexpr int kArgumentBytes = 3900;      // of a list, beside the other arguments in 4 KB

// Division of n < 2^31 by the row length: (mulhi(n, magic) + n) >> shift, by the method of Granlund and Montgomery
// ("Division by Invariant Integers using Multiplication", 1994)
struct RowDiv {
    uint32_t row, magic;
    uint32_t shift;
};

// round to nearest even; a NaN stays one
XSG_DEV uint32_t bf16_bits(float x) {
    const uint32_t u = __float_as_uint(x);
    if (x != x) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// Elements of one type, one at a time or four at a time from a place aligned for that (16 bytes of float32, 8
// of the others). A chunk's bytes fit 32 bits, so an access is a base held by the wavefront and a lane's offset.
// STREAM: around the caches, for arrays that would only push each other out of them.
#define XSG_GLOBAL __attribute__((address_space(1)))
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <typename V, bool STREAM = false> XSG_DEV V get(const void* p, uint32_t byte) {
    const XSG_GLOBAL V* const q = (const XSG_GLOBAL V*)((const XSG_GLOBAL char*)p + byte);
    return STREAM ? __builtin_nontemporal_load(q) : *q;
}
template <bool STREAM = false, typename V> XSG_DEV void put(void* p, uint32_t byte, V x) {
    XSG_GLOBAL V* const q = (XSG_GLOBAL V*)((XSG_GLOBAL char*)p + byte);
    if (STREAM) __builtin_nontemporal_store(x, q);
    else *q = x;
}

template <int DT> XSG_DEV float load1(const void* p, uint32_t i) {
    if (DT == XSG_DTYPE_F32) return get<float>(p, 4 * i);
    if (DT == XSG_DTYPE_BF16) return __uint_as_float((uint32_t)get<uint16_t>(p, 2 * i) << 16);
    return (float)get<_Float16>(p, 2 * i);
}
template <int DT> XSG_DEV void store1(void* p, uint32_t i, float x) {
    if (DT == XSG_DTYPE_F32) put(p, 4 * i, x);
    else if (DT == XSG_DTYPE_BF16) put(p, 2 * i, (uint16_t)bf16_bits(x));
    else put(p, 2 * i, (_Float16)x);
}
template <int DT, bool STREAM = false> XSG_DEV f32x4 load4(const void* p, uint32_t i) {
    if (DT == XSG_DTYPE_F32) return get<f32x4, STREAM>(p, 4 * i);
    if (DT == XSG_DTYPE_BF16) {
        const u32x2 u = get<u32x2, STREAM>(p, 2 * i);
        return f32x4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u)};
    }
    return __builtin_convertvector(get<f16x4, STREAM>(p, 2 * i), f32x4);
}
template <int DT, bool STREAM = false> XSG_DEV void store4(void* p, uint32_t i, f32x4 x) {
    if (DT == XSG_DTYPE_F32)
        put<STREAM>(p, 4 * i, x);
    else if (DT == XSG_DTYPE_BF16)
        put<STREAM>(p, 2 * i, u32x2{bf16_bits(x.x) | bf16_bits(x.y) << 16, bf16_bits(x.z) | bf16_bits(x.w) << 16});
    else
        put<STREAM>(p, 2 * i, __builtin_convertvector(x, f16x4));
}
// those of x whose bit in keep is set
template <int DT, bool STREAM> XSG_DEV void store4(void* p, uint32_t i, f32x4 x, uint32_t keep) {
    if (keep == 15u) return store4<DT, STREAM>(p, i, x);
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if ((keep >> k) & 1) store1<DT>(p, i + k, x[k]);
}
// What tensors of a long list have in common: most of it has few kinds.
struct EntryKind {
    double lr;
    uint32_t row, magic;
    float keep;
    uint8_t shift, dtype, gdtype;
    bool operator==(const EntryKind& o) const {
        return row == o.row && lr == o.lr && keep == o.keep && dtype == o.dtype && gdtype == o.gdtype;
    }
};

struct GradEntry {
    static constexpr int kPointers = 1;
    void* data;
    int64_t numel;
    const uint32_t* mask;
    uint32_t row, magic;      // elements to a mask bit, and its division
    uint8_t shift, dtype;
    XSG_HD const void* grad() const { return data; }
    XSG_HD int grad_dtype() const { return dtype; }
    EntryKind kind() const { return EntryKind{0.0, row, magic, 0.0f, shift, dtype, 0}; }
    void pointers(uint64_t* to) const { to[0] = (uint64_t)data; }
    XSG_DEV void set(const uint64_t* ptr, int64_t numel_, const uint32_t* mask_, const EntryKind& k) {
        data = (void*)ptr[0];
        numel = numel_;
        mask = mask_;
        row = k.row;
        magic = k.magic;
        shift = k.shift;
        dtype = k.dtype;
    }
};

struct AdamEntry {
    static constexpr int kPointers = 4;
    void* param;
    const void* gradient;
    float *avg, *sq;
    int64_t numel;
    const uint32_t* mask;
    double lr;
    uint32_t row, magic;
    float keep;               // 1 - lr * weight decay
    uint8_t shift, pdtype, gdtype;
    XSG_HD const void* grad() const { return gradient; }
    XSG_HD int grad_dtype() const { return gdtype; }
    EntryKind kind() const { return EntryKind{lr, row, magic, keep, shift, pdtype, gdtype}; }
    void pointers(uint64_t* to) const {
        to[0] = (uint64_t)param;
        to[1] = (uint64_t)gradient;
        to[2] = (uint64_t)avg;
        to[3] = (uint64_t)sq;
    }
    XSG_DEV void set(const uint64_t* ptr, int64_t numel_, const uint32_t* mask_, const EntryKind& k) {
        param = (void*)ptr[0];
        gradient = (const void*)ptr[1];
        avg = (float*)ptr[2];
        sq = (float*)ptr[3];
        numel = numel_;
        mask = mask_;
        row = k.row;
        magic = k.magic;
        lr = k.lr;
        keep = k.keep;
        shift = k.shift;
        pdtype = k.dtype;
        gdtype = k.gdtype;
    }
};

template <typename E> constexpr int kInline = kArgumentBytes / (sizeof(E) + 4);

// first[t]: the first chunk of tensor t; first[n] = chunks
// masked_chunk: the chunk of a masked tensor
template <typename E> struct InlineList {
    typedef E Entry;
    E entry[kInline<E>];
    int32_t first[kInline<E> + 1];
    int32_t n, chunk, masked_chunk, chunks;
    XSG_DEV const E& at(int t) const { return entry[t]; }
    XSG_DEV int32_t first_of(int t) const { return first[t]; }
};
template <typename E> struct TableList {
    typedef E Entry;
    const E* entry;
    const int32_t* first;
    int32_t n, chunk, masked_chunk, chunks;
    // t is the wavefront's: the entry comes by scalar loads, as an inline one does
    XSG_DEV E at(int t) const {
        typedef const uint64_t __attribute__((address_space(4)))* Words;
        const Words w = (Words)(entry + t);
        union { uint64_t words[sizeof(E) / 8]; E e; } u;
#pragma unroll
        for (int k = 0; k < (int)(sizeof(E) / 8); ++k) u.words[k] = w[k];
        return u.e;
    }
    XSG_DEV int32_t first_of(int t) const { return get<int32_t>(first, 4 * t); }
};
// A piece of a long list on its way to the workspace: pointers, first chunk, and a word of a tensor's size (48
// bits), kind and mask (8 bits each; 0: no mask).
template <typename E> struct TablePiece {
    static constexpr int kKinds = 16, kMasks = E::kPointers == 1 ? 48 : 24;
    static constexpr int kSpace = kArgumentBytes - kKinds * sizeof(EntryKind) - kMasks * 8 - 24;
    static constexpr int kMax = kSpace / (8 * E::kPointers + 12);
    static_assert(kMax <= kBlock, "a thread to a tensor");
    uint64_t pointer[kMax][E::kPointers];
    uint64_t word[kMax];
    const uint32_t* mask[kMasks];
    EntryKind kind[kKinds];
    int32_t first[kMax];
    int32_t n, kinds, masks, end;   // end: the list's number of chunks with its last piece, else -1
};
static_assert(sizeof(InlineList<GradEntry>) <= 3920 && sizeof(InlineList<AdamEntry>) <= 3920 &&
                  sizeof(TablePiece<GradEntry>) <= 3920 && sizeof(TablePiece<AdamEntry>) <= 3920 &&
                  sizeof(GradEntry) % 8 == 0 && sizeof(AdamEntry) % 8 == 0,
              "lists share 4 KB with the other arguments; entries are loaded by words");

// 2.1 us a piece, a launch's and an argument's latency: 505 tensors take four pieces (gradients) or seven (updates).
template <typename E>
__global__ __launch_bounds__(kBlock) void table_kernel(TablePiece<E> piece, E* __restrict__ entry,
                                                       int32_t* __restrict__ first) {
    __shared__ EntryKind kind[TablePiece<E>::kKinds];
    __shared__ const uint32_t* mask[TablePiece<E>::kMasks];
    const int i = threadIdx.x;
    if (i < piece.kinds) kind[i] = piece.kind[i];
    if (i < piece.masks) mask[i] = piece.mask[i];
    const int mine = min(i, piece.n - 1);
    const uint64_t word = piece.word[mine];
    uint64_t pointer[E::kPointers];
#pragma unroll
    for (int k = 0; k < E::kPointers; ++k) pointer[k] = piece.pointer[mine][k];
    const int32_t chunk = piece.first[mine];
    __syncthreads();
    if (i < piece.n) {
        const int m = (int)(word >> 56);
        E e;
        e.set(pointer, (int64_t)(word & (((uint64_t)1 << 48) - 1)), m ? mask[m - 1] : nullptr, kind[(word >> 48) & 255]);
        entry[i] = e;
        first[i] = chunk;
    }
    if (piece.end >= 0 && i == 0) first[piece.n] = piece.end;
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
        return (word(r >> 5) >> (r & 31)) & 1u;
    }
    XSG_DEV uint32_t word(uint32_t k) const { return get<uint32_t>(words, 4 * k); }
    // bit k: element i + k; all four lie in the chunk. Their rows span at most two words.
    XSG_DEV uint32_t four(uint32_t i) const {
        const uint32_t n = rem + i, q = quotient(n), r0 = bit + q;
        const uint32_t r3 = bit + quotient(n + 3);
        const uint64_t w = (uint64_t)word(r0 >> 5) | (uint64_t)word(r3 >> 5) << 32;
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
    if (n == 0) return 0;
    for (;;) {
        const int step = (n + 63) >> 6, i = lane * step;
        const int below = max((int)__popcll(__ballot(i < n && list.first_of(lo + min(i, n - 1)) <= b)) - 1, 0);
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

// many(i[], keep[], all): UNROLL groups, of which those with keep 0 are left out; `all` is a constant that says
// that every group is there and kept. one(i): a single element.
template <bool MASK, int UNROLL, typename One, typename Many>
XSG_DEV void for_chunk(const ChunkSpan& span, const ChunkMask& mask, One&& one, Many&& many) {
    constexpr uint32_t tile = kBlock * UNROLL;
    const uint32_t whole = span.groups / tile * tile;
    uint32_t g = threadIdx.x, i[UNROLL], keep[UNROLL];
#pragma unroll 1
    for (; g < whole; g += tile) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            i[u] = span.head + 4 * (g + u * kBlock);
            keep[u] = MASK ? mask.four(i[u]) : 15u;
        }
        many(i, keep, std::integral_constant<bool, !MASK>{});
    }
    if (whole < span.groups) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            i[u] = span.head + 4 * (g + u * kBlock);
            keep[u] = g + u * kBlock < span.groups ? (MASK ? mask.four(i[u]) : 15u) : 0u;
        }
        many(i, keep, std::false_type{});
    }
    if (threadIdx.x < span.head && (!MASK || mask.one(threadIdx.x))) one(threadIdx.x);
#pragma unroll 1
    for (uint32_t k = span.tail_at() + threadIdx.x; k < span.tail_at() + span.tail; k += kBlock)
        if (!MASK || mask.one(k)) one(k);
}

constexpr int kUnroll = 4;   // groups in flight per thread and array
// An update of four arrays has as many where it streams (4 M Gaussians 1251 us, with two 1267), two where the
// caches answer and more wavefronts do better.
template <bool STREAM> constexpr int kAdamUnroll = STREAM ? 4 : 2;

// Under a mask of short rows each wavefront lists the kept rows of its share of the chunk (a mask word a lane, so
// up to 2048 rows for one load's latency) and then walks their elements alone, VEC at a time, so that lanes are
// busy and loads in flight however few rows are kept (1 M Gaussians with 14 % kept: norm 41 -> 24 us against a look
// at every group of four, the update's kernel 119 -> 86).
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
        uint32_t w = mask.word(at >> 5);
        if (at < lo) w &= 0xffffffffu << (lo - at);   // lo lies in the first word
        return hi - at < 32 ? w & ~(0xffffffffu << (hi - at)) : w;
    };
    uint32_t next = word_of(lo & ~31u);
#pragma unroll 1
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
#pragma unroll 1
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

template <int NORM> struct AccumSet {   // one for each group in flight
    Accum<NORM> acc[kUnroll];
    XSG_DEV void add(int u, f32x4 x) {
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[u].add(x[k]);
    }
    XSG_DEV Accum<NORM> joined() {
#pragma unroll
        for (int u = 1; u < kUnroll; ++u) acc[0].join(acc[u]);
        return acc[0];
    }
};

template <int NORM, int DT, bool MASK, bool STREAM>
XSG_DEV Accum<NORM> chunk_norm(const void* p, const ChunkSpan& span, const ChunkMask& mask) {
    AccumSet<NORM> acc;
    for_chunk<MASK, kUnroll>(span, mask, [&](uint32_t i) { acc.acc[0].add(load1<DT>(p, i)); },
                             [&](const uint32_t* i, const uint32_t* keep, auto all) {
        f32x4 x[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (all.value || keep[u]) x[u] = load4<DT, STREAM>(p, i[u]);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (MASK) {
#pragma unroll
                for (int k = 0; k < 4; ++k) x[u][k] = (keep[u] >> k) & 1 ? x[u][k] : 0.f;
            }
            acc.add(u, x[u]);
        }
    });
    return acc.joined();
}

template <int NORM, int DT>
XSG_DEV Accum<NORM> rows_norm(const void* p, uint32_t count, bool whole, const ChunkMask& mask) {
    AccumSet<NORM> acc;
    if (whole) {
        for_kept_rows<4, kUnroll>(mask, count, [&](const uint32_t* i, const bool* on) {
            f32x4 x[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (on[u]) x[u] = load4<DT>(p, i[u]);
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) acc.add(u, x[u]);
        });
    } else {
        for_kept_rows<1, kUnroll>(mask, count, [&](const uint32_t* i, const bool* on) {
            float x[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                x[u] = 0.f;
                if (on[u]) x[u] = load1<DT>(p, i[u]);
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) acc.acc[u].add(x[u]);
        });
    }
    return acc.joined();
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
        const int64_t size = e.mask ? list.masked_chunk : list.chunk;
        base = (b - list.first_of(t)) * size;
        count = (uint32_t)min(size, e.numel - base);
    }
};

// Bound by its reads: 236 M float32 166 us (5.7 TB/s), 59 M 35 us (in part from the last-level cache); 1 M
// Gaussians with 14 % kept 17 us, of which the list of rows is most.
// A workgroup sums `each` chunks in a row. `step`, unless null, counts one step more; the launches behind this
// one read it.
template <int NORM, bool STREAM, typename L>
__global__ __launch_bounds__(kBlock) void norm_partial_kernel(L list, int each, double* __restrict__ partial,
                                                              int64_t* step) {
    __shared__ uint16_t listed[kBlock / 64 * kRowBatch];
    if (step && blockIdx.x == 0 && threadIdx.x == 0) *step += 1;
    Accum<NORM> acc;
    const int end = min(((int)blockIdx.x + 1) * each, list.chunks);
#pragma unroll 1
    for (int b = blockIdx.x * each; b < end; ++b) {
        const int t = find_tensor(list, b);
        const auto& e = list.at(t);
        const Chunk chunk(list, e, b, t);
        const int dtype = e.grad_dtype();
        const void* p = at(e.grad(), chunk.base, dtype);
        const ChunkSpan span(chunk.count, phase_of(p, dtype));
        ChunkMask mask;
        mask.list = listed;
        if (e.mask) mask.open(e.mask, chunk.base, e.row, e.magic, e.shift);
        with_type(dtype, [&](auto dt) {
            if (!e.mask) acc.join(chunk_norm<NORM, dt.value, false, STREAM>(p, span, mask));
            else if (mask.row > kShortRow) acc.join(chunk_norm<NORM, dt.value, true, STREAM>(p, span, mask));
            else acc.join(rows_norm<NORM, dt.value>(p, chunk.count, span.head == 0 && mask.row % 4 == 0, mask));
        });
    }
    acc = block_join<NORM>(acc);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc.value();
}

template <int NORM> XSG_DEV Accum<NORM> join_partials(const double* __restrict__ partial, int n) {
    Accum<NORM> acc;
    for (int i0 = threadIdx.x; i0 < n; i0 += 8 * kBlock) {   // other XCDs wrote them: one far latency for eight
        double v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = i0 + u * kBlock < n ? partial[i0 + u * kBlock] : 0.0;
#pragma unroll
        for (int u = 0; u < 8; ++u) acc.join_value(v[u]);
    }
    return block_join<NORM>(acc);
}

// The norm from the partial sums of its chunks, in every thread of the workgroup.
XSG_DEV double norm_of(const double* __restrict__ partial, int n, int norm) {
    if (norm == XSG_NORM_L2) return join_partials<XSG_NORM_L2>(partial, n).finish();
    if (norm == XSG_NORM_L1) return join_partials<XSG_NORM_L1>(partial, n).finish();
    return join_partials<XSG_NORM_INF>(partial, n).finish();
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
    const int lo = t < list.n ? list.first_of(t) : 0, hi = t < list.n ? list.first_of(t + 1) : list.chunks;
    const double v = norm_of(partial + lo, hi - lo, norm);
    if (threadIdx.x == 0) *(t < list.n ? each + t : total) = (float)v;
}

// min(1, max_norm / (norm + eps)); a NaN norm gives NaN, an infinite one 0
XSG_DEV float clip_factor(double norm, double max_norm, double eps) {
    const double c = max_norm / (norm + eps);
    return c > 1.0 ? 1.0f : (float)c;
}

// What a call that writes takes from the norm and the step counter.
struct StepTerms {
    double over1;   // 1 / (1 - beta1^t); its product with a rate is rounded, not itself
    float c;        // the clip factor
    float root;     // 1 / sqrt(1 - beta2^t)
    int taken;      // 0: the step is left out
};

struct StepRule {
    double max_norm, clip_eps;
    double log_beta1, log_beta2;   // natural logarithms
    int norm;                      // the kind; -1: none is computed
    int clip, skip_nonfinite;
};

// In every thread of the workgroup; the first workgroup also gives the norm out and takes the counter back where
// the step is not taken (what another one then made of it goes unused). The counter already counts this step.
XSG_DEV StepTerms step_terms(const StepRule& rule, const double* __restrict__ partial, int n, int64_t* step,
                             float* __restrict__ total) {
    StepTerms terms{1.0, 1.0f, 1.0f, 1};
    __shared__ double over1;
    __shared__ float root;
    // 1 - beta^t without the cancellation, in 64 bits not cheap: by the wavefront with the fewest partial sums
    if (step && threadIdx.x >= kBlock - 64) {
        const double t = (double)*step;
        over1 = -1.0 / expm1(t * rule.log_beta1);
        root = (float)(1.0 / sqrt(-expm1(t * rule.log_beta2)));
    }
    if (rule.norm >= 0) {
        const double norm = norm_of(partial, n, rule.norm);
        const bool first = blockIdx.x == 0 && threadIdx.x == 0;
        if (first && total) *total = (float)norm;
        if (rule.clip) terms.c = clip_factor(norm, rule.max_norm, rule.clip_eps);
        if (rule.skip_nonfinite && !((float)norm < INFINITY)) {   // by the norm as the caller has it
            if (first) *step -= 1;
            terms.taken = 0;
        }
    } else {
        __syncthreads();
    }
    if (step) {
        terms.over1 = over1;
        terms.root = root;
    }
    return terms;
}

// Of many partial sums the terms are made once, in a launch of their own.
__global__ __launch_bounds__(kBlock) void step_terms_kernel(StepRule rule, const double* __restrict__ partial, int n,
                                                            int64_t* step, float* __restrict__ total,
                                                            StepTerms* __restrict__ ready) {
    const StepTerms terms = step_terms(rule, partial, n, step, total);
    if (threadIdx.x == 0) *ready = terms;
}

// Where a launch that writes has its terms from: made before, or its own to make from the partial sums.
struct StepSource {
    StepRule rule;
    const double* __restrict__ partial;
    int n;
    int64_t* step;
    float* __restrict__ total;
    const StepTerms* __restrict__ ready;
    XSG_DEV StepTerms terms() const { return ready ? *ready : step_terms(rule, partial, n, step, total); }
};

template <int DT, bool MASK, bool STREAM>
XSG_DEV void chunk_scale(void* p, float c, const ChunkSpan& span, const ChunkMask& mask) {
    for_chunk<MASK, kUnroll>(span, mask, [&](uint32_t i) { store1<DT>(p, i, load1<DT>(p, i) * c); },
                             [&](const uint32_t* i, const uint32_t* keep, auto all) {
        f32x4 x[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (all.value || keep[u]) x[u] = load4<DT, STREAM>(p, i[u]);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (all.value || keep[u]) store4<DT, STREAM>(p, i[u], x[u] * c, all.value ? 15u : keep[u]);
    });
}

template <int DT, bool STREAM>
XSG_DEV void rows_scale(void* p, float c, uint32_t count, bool whole, const ChunkMask& mask) {
    if (whole) {
        for_kept_rows<4, kUnroll>(mask, count, [&](const uint32_t* i, const bool* on) {
            f32x4 x[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (on[u]) x[u] = load4<DT>(p, i[u]);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (on[u]) store4<DT, STREAM>(p, i[u], x[u] * c);
        });
    } else {
        for_kept_rows<1, kUnroll>(mask, count, [&](const uint32_t* i, const bool* on) {
            float x[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (on[u]) x[u] = load1<DT>(p, i[u]);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (on[u]) store1<DT>(p, i[u], x[u] * c);
        });
    }
}

// x <- c x, bound by reads and writes: 236 M float32 268 us (7.0 TB/s of both). One chunk a workgroup.
template <bool STREAM, typename L>
__global__ __launch_bounds__(kBlock) void clip_scale_kernel(L list, StepSource source) {
    const int b = blockIdx.x, t = find_tensor(list, b);   // while the partial sums are on their way
    const auto& e = list.at(t);
    const float c = source.terms().c;
    if (c == 1.0f || b >= list.chunks) return;   // the values stay as they are
    const Chunk chunk(list, e, b, t);
    const int dtype = e.dtype;
    void* p = at(e.data, chunk.base, dtype);
    const ChunkSpan span(chunk.count, phase_of(p, dtype));
    ChunkMask mask;
    __shared__ uint16_t listed[kBlock / 64 * kRowBatch];
    mask.list = listed;
    if (e.mask) mask.open(e.mask, chunk.base, e.row, e.magic, e.shift);
    with_type(dtype, [&](auto dt) {
        if (!e.mask) chunk_scale<dt.value, false, STREAM>(p, c, span, mask);
        else if (mask.row > kShortRow) chunk_scale<dt.value, true, STREAM>(p, c, span, mask);
        else rows_scale<dt.value, STREAM>(p, c, chunk.count, span.head == 0 && mask.row % 4 == 0, mask);
    });
}

// Elements of a strided tensor that took their turn in a dense copy. Rows out of the mask are not touched (they may be
// another stream's to write meanwhile), and what did not change is not written. An element a lane and turn, its place
// by a division for each dimension left.
constexpr int kMaxDims = 16;
struct Strides {
    int64_t size[kMaxDims], stride[kMaxDims];
    int dims;
};

template <typename T, typename I>
__global__ __launch_bounds__(kBlock) void write_back_kernel(T* __restrict__ dst, const T* __restrict__ src, I numel,
                                                            Strides at, const uint32_t* __restrict__ mask, I row) {
    for (I i = (I)blockIdx.x * kBlock + threadIdx.x; i < numel; i += (I)gridDim.x * kBlock) {
        if (mask) {
            const I r = i / row;
            if (!((mask[r >> 5] >> (r & 31)) & 1u)) continue;
        }
        I rest = i;
        int64_t place = 0;
        for (int d = at.dims - 1; d >= 0; --d) {
            const I q = rest / (I)at.size[d];
            place += (int64_t)(rest - q * (I)at.size[d]) * at.stride[d];
            rest = q;
        }
        const T x = src[i];
        if (dst[place] != x) dst[place] = x;
    }
}

struct AdamScalars {
    float beta2, one_minus_beta1, one_minus_beta2, eps;
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

XSG_DEV AdamTerms adam_terms(const StepTerms& now, const AdamScalars& s, double lr, float keep) {
    return AdamTerms{s.beta2, s.one_minus_beta1, s.one_minus_beta2, s.eps, now.c, (float)(lr * now.over1), now.root, keep};
}
XSG_DEV AdamArrays adam_arrays(const AdamEntry& e, int64_t base) {
    return AdamArrays{at(e.param, base, e.pdtype), at(e.gradient, base, e.gdtype), e.avg + base, e.sq + base};
}

// One element, or four, of the four arrays.
template <int PT, int GT> struct Adam1 {
    float p, g, m, v;
    XSG_DEV void load(const AdamArrays& a, uint32_t i) {
        p = load1<PT>(a.p, i);
        g = load1<GT>(a.g, i);
        m = load1<XSG_DTYPE_F32>(a.m, i);
        v = load1<XSG_DTYPE_F32>(a.v, i);
    }
    XSG_DEV void update(const AdamTerms& s) { s.update(p, g, m, v); }
    XSG_DEV void store(const AdamArrays& a, uint32_t i) const {
        store1<PT>(a.p, i, p);
        store1<XSG_DTYPE_F32>(a.m, i, m);
        store1<XSG_DTYPE_F32>(a.v, i, v);
    }
};
template <int PT, int GT, bool STREAM> struct Adam4 {
    f32x4 p, g, m, v;
    XSG_DEV void load(const AdamArrays& a, uint32_t i) {
        p = load4<PT, STREAM>(a.p, i);
        g = load4<GT, STREAM>(a.g, i);
        m = load4<XSG_DTYPE_F32, STREAM>(a.m, i);
        v = load4<XSG_DTYPE_F32, STREAM>(a.v, i);
    }
    XSG_DEV void update(const AdamTerms& s) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float pk = p[k], mk = m[k], vk = v[k];
            s.update(pk, g[k], mk, vk);
            p[k] = pk;
            m[k] = mk;
            v[k] = vk;
        }
    }
    XSG_DEV void store(const AdamArrays& a, uint32_t i, uint32_t keep) const {
        store4<PT, STREAM>(a.p, i, p, keep);
        store4<XSG_DTYPE_F32, STREAM>(a.m, i, m, keep);
        store4<XSG_DTYPE_F32, STREAM>(a.v, i, v, keep);
    }
};

template <int PT, int GT, bool MASK, bool STREAM>
XSG_DEV void chunk_adam(const AdamArrays& a, const AdamTerms& s, const ChunkSpan& span, const ChunkMask& mask) {
    for_chunk<MASK, kAdamUnroll<STREAM>>(span, mask, [&](uint32_t i) {
        Adam1<PT, GT> x;
        x.load(a, i);
        x.update(s);
        x.store(a, i);
    }, [&](const uint32_t* i, const uint32_t* keep, auto all) {
        Adam4<PT, GT, STREAM> x[kAdamUnroll<STREAM>];
#pragma unroll
        for (int u = 0; u < kAdamUnroll<STREAM>; ++u)
            if (all.value || keep[u]) x[u].load(a, i[u]);
#pragma unroll
        for (int u = 0; u < kAdamUnroll<STREAM>; ++u) {
            if (!(all.value || keep[u])) continue;
            x[u].update(s);
            x[u].store(a, i[u], all.value ? 15u : keep[u]);
        }
    });
}

template <int PT, int GT, bool STREAM>
XSG_DEV void rows_adam(const AdamArrays& a, const AdamTerms& s, uint32_t count, bool whole, const ChunkMask& mask) {
    if (whole) {
        for_kept_rows<4, kAdamUnroll<STREAM>>(mask, count, [&](const uint32_t* i, const bool* on) {
            Adam4<PT, GT, STREAM> x[kAdamUnroll<STREAM>];
#pragma unroll
            for (int u = 0; u < kAdamUnroll<STREAM>; ++u)
                if (on[u]) x[u].load(a, i[u]);
#pragma unroll
            for (int u = 0; u < kAdamUnroll<STREAM>; ++u) {
                if (!on[u]) continue;
                x[u].update(s);
                x[u].store(a, i[u], 15u);
            }
        });
    } else {
        for_kept_rows<1, kUnroll>(mask, count, [&](const uint32_t* i, const bool* on) {
            Adam1<PT, GT> x[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (on[u]) x[u].load(a, i[u]);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (!on[u]) continue;
                x[u].update(s);
                x[u].store(a, i[u]);
            }
        });
    }
}

// The update, bound by four reads and three writes of an element: 236 M float32 1000 to 1080 us from card to card (6.6
// to 6.1 TB/s), 1 M Gaussians with 14 % kept 77 to 80 us (412 MB moved in sectors of 64 bytes, 5.1 TB/s). Dense arrays
// that are not aligned alike go one element at a time: 59 M with the parameters one element further 371 us, 288 aligned.
// F32: every parameter and gradient is float32
template <bool F32, bool STREAM, typename L>
__global__ __launch_bounds__(kBlock) void adam_kernel(L list, AdamScalars s, StepSource source) {
    const int b = blockIdx.x, t = find_tensor(list, b);   // while the partial sums are on their way
    const auto& e = list.at(t);
    const StepTerms now = source.terms();
    if (!now.taken || b >= list.chunks) return;
    const Chunk chunk(list, e, b, t);
    const AdamTerms terms = adam_terms(now, s, e.lr, e.keep);
    const int pt = F32 ? XSG_DTYPE_F32 : e.pdtype, gt = F32 ? XSG_DTYPE_F32 : e.gdtype;
    const AdamArrays a = adam_arrays(e, chunk.base);
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
    const auto run = [&](auto p, auto g) {
        if (!e.mask) chunk_adam<p.value, g.value, false, STREAM>(a, terms, span, mask);
        else if (mask.row > kShortRow) chunk_adam<p.value, g.value, true, STREAM>(a, terms, span, mask);
        else rows_adam<p.value, g.value, STREAM>(a, terms, chunk.count, whole, mask);
    };
    if constexpr (F32) {
        const std::integral_constant<int, XSG_DTYPE_F32> f32;
        run(f32, f32);
    } else {
        with_type(pt, [&](auto p) { with_type(gt, [&](auto g) { run(p, g); }); });
    }
}

// A short list of few chunks (poses, biases, a head's weights): one workgroup does the whole call, a chunk to a
// wavefront, so that there is one launch, which is most of such a call's time.
// 16 chunks of 1024 elements: norm 5.8 us against 8.4 in two launches, clip 6.0 against 8.8; 24: 8.2 either way; 24
// tensors of 4: 5.9. The update does more to an element: 24 tensors of 4 take 8.4 us against 9.7, 8 of 1024 take
// 12.1 against 9.5.
constexpr int kSmallBlock = 1024;
constexpr int kSmallChunks = 64;                  // of tensors of up to kSmallTensor elements
constexpr int kOneRound = kSmallBlock / 64;       // of longer ones, not for an update
constexpr int64_t kSmallTensor = 256;

enum SmallOp { kSmallNorm, kSmallClip, kSmallAdam };

template <int UNROLL, typename F> XSG_DEV void for_lanes(const Chunk& chunk, const ChunkMask& mask, bool masked, F&& f) {
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t i0 = lane; i0 < chunk.count; i0 += 64 * UNROLL) {
        uint32_t i[UNROLL];
        bool on[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            i[u] = i0 + 64 * u;
            on[u] = i[u] < chunk.count && (!masked || mask.one(i[u]));
        }
        f(i, on);
    }
}

template <int NORM, int OP, typename E>
__global__ __launch_bounds__(kSmallBlock) void small_kernel(InlineList<E> list, StepRule rule, AdamScalars s,
                                                            int64_t* step, float* __restrict__ total,
                                                            float* __restrict__ each) {
    __shared__ double part[kSmallChunks];
    __shared__ StepTerms shared;
    __shared__ double over1;
    __shared__ float root;
    const int wave = threadIdx.x >> 6;
    const double count = OP == kSmallAdam ? (double)(*step + 1) : 0.0;   // before it may change
    if (OP == kSmallAdam && wave == kSmallBlock / 64 - 1) {
        over1 = -1.0 / expm1(count * rule.log_beta1);
        root = (float)(1.0 / sqrt(-expm1(count * rule.log_beta2)));
    }
    if (OP != kSmallAdam || rule.norm >= 0) {
        for (int b = wave; b < list.chunks; b += kSmallBlock / 64) {
            const int t = find_tensor(list, b);
            const E& e = list.at(t);
            const Chunk chunk(list, e, b, t);
            const void* p = at(e.grad(), chunk.base, e.grad_dtype());
            ChunkMask mask;
            if (e.mask) mask.open(e.mask, chunk.base, e.row, e.magic, e.shift);
            Accum<NORM> acc[kUnroll];
            with_type(e.grad_dtype(), [&](auto dt) {
                for_lanes<kUnroll>(chunk, mask, e.mask != nullptr, [&](const uint32_t* i, const bool* on) {
#pragma unroll
                    for (int u = 0; u < kUnroll; ++u)
                        if (on[u]) acc[u].add(load1<dt.value>(p, i[u]));
                });
            });
#pragma unroll
            for (int u = 1; u < kUnroll; ++u) acc[0].join(acc[u]);
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) acc[0].join(acc[0].shuffled(d));
            if ((threadIdx.x & 63) == 0) part[b] = acc[0].value();
        }
    }
    __syncthreads();
    if (OP == kSmallNorm && each && threadIdx.x >= 64 && threadIdx.x - 64 < list.n) {
        const int t = threadIdx.x - 64;
        Accum<NORM> acc;
        for (int b = list.first_of(t); b < list.first_of(t + 1); ++b) acc.join_value(part[b]);
        each[t] = (float)acc.finish();
    }
    if (threadIdx.x < 64) {
        StepTerms terms{1.0, 1.0f, 1.0f, 1};
        if (OP != kSmallAdam || rule.norm >= 0) {
            Accum<NORM> acc;
            if (threadIdx.x < list.chunks) acc.join_value(part[threadIdx.x]);
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) acc.join(acc.shuffled(d));
            const double norm = acc.finish();
            if (threadIdx.x == 0 && total) *total = (float)norm;
            if (rule.clip) terms.c = clip_factor(norm, rule.max_norm, rule.clip_eps);
            terms.taken = !rule.skip_nonfinite || (float)norm < INFINITY;   // by the norm as the caller has it
        }
        if (threadIdx.x == 0) {
            if (OP == kSmallAdam && terms.taken) *step += 1;
            shared = terms;
        }
    }
    if (OP == kSmallNorm) return;
    __syncthreads();
    StepTerms now = shared;
    if (OP == kSmallAdam) {
        now.over1 = over1;
        now.root = root;
    }
    if (OP == kSmallClip ? now.c == 1.0f : !now.taken) return;
    for (int b = wave; b < list.chunks; b += kSmallBlock / 64) {
        const int t = find_tensor(list, b);
        const E& e = list.at(t);
        const Chunk chunk(list, e, b, t);
        ChunkMask mask;
        if (e.mask) mask.open(e.mask, chunk.base, e.row, e.magic, e.shift);
        if constexpr (OP == kSmallClip) {
            void* p = at(e.data, chunk.base, e.dtype);
            with_type(e.dtype, [&](auto dt) {
                for_lanes<kUnroll>(chunk, mask, e.mask != nullptr, [&](const uint32_t* i, const bool* on) {
                    float x[kUnroll];
#pragma unroll
                    for (int u = 0; u < kUnroll; ++u)
                        if (on[u]) x[u] = load1<dt.value>(p, i[u]);
#pragma unroll
                    for (int u = 0; u < kUnroll; ++u)
                        if (on[u]) store1<dt.value>(p, i[u], x[u] * now.c);
                });
            });
        } else if constexpr (OP == kSmallAdam) {
            const AdamTerms terms = adam_terms(now, s, e.lr, e.keep);
            const AdamArrays a = adam_arrays(e, chunk.base);
            with_type(e.pdtype, [&](auto pt) {
                with_type(e.gdtype, [&](auto gt) {
                    for_lanes<kUnroll>(chunk, mask, e.mask != nullptr, [&](const uint32_t* i, const bool* on) {
                        Adam1<pt.value, gt.value> x[kUnroll];
#pragma unroll
                        for (int u = 0; u < kUnroll; ++u)
                            if (on[u]) x[u].load(a, i[u]);
#pragma unroll
                        for (int u = 0; u < kUnroll; ++u) {
                            if (!on[u]) continue;
                            x[u].update(terms);
                            x[u].store(a, i[u]);
                        }
                    });
                });
            });
        }
    }
}

// ------------------------------------------------------------------------------------------------ host
int64_t chunks_of(int64_t numel, int64_t size) {
    return numel <= size ? (numel > 0 ? 1 : 0) : (numel + size - 1) / size;
}
int64_t chunk_for(int64_t elements, int64_t target, bool writes_far) {
    const auto share = [&](int64_t of) { return ((elements + of - 1) / of + kChunkUnit - 1) / kChunkUnit * kChunkUnit; };
    return std::min(std::max(share(target), kChunkUnit), writes_far ? std::max(kWriteChunk, share(kFarChunks)) : kMaxChunk);
}

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
    if (!mask || numel == 0) return RowDiv{1, 1, 0};
    const uint32_t d = (uint32_t)(numel / rows);
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
    return AdamEntry{x.param, x.grad, x.exp_avg, x.exp_avg_sq, x.numel, x.numel ? x.mask : nullptr, x.lr, div.row, div.magic,
                     (float)(1.0 - x.lr * x.weight_decay), (uint8_t)div.shift, (uint8_t)x.param_dtype,
                     (uint8_t)x.grad_dtype};
}
template <typename T> using EntryOf = decltype(entry_of(std::declval<const T&>()));

int64_t touched(const xsg_grad_tensor& x) { return x.numel * type_size(x.dtype); }
int64_t touched(const xsg_adam_tensor& x) { return x.numel * (type_size(x.param_dtype) + type_size(x.grad_dtype) + 8); }
bool all_f32(const xsg_grad_tensor& x) { return x.dtype == XSG_DTYPE_F32; }
bool all_f32(const xsg_adam_tensor& x) { return x.param_dtype == XSG_DTYPE_F32 && x.grad_dtype == XSG_DTYPE_F32; }

// calls f with the flag as a constant
template <typename F> void with_flag(bool flag, F&& f) {
    if (flag) f(std::true_type{});
    else f(std::false_type{});
}

// How a call is cut, and where things lie in its workspace: the step's terms, then (256 bytes on) the partial
// sums, of `each` chunks in a row, then a long list's table.
struct Plan {
    int64_t elements = 0, bytes_touched = 0, chunk = 0, masked_chunk = 0, chunks = 0, each = 1, parts = 0;
    bool table = false, f32 = true, stream = false, stream_norm = false;
    size_t first_at = 0, entry_at = 0, bytes = 0;
};

size_t aligned(size_t x) { return (x + 255) / 256 * 256; }

template <typename T> int make_plan(const T* ts, int n, const char* who, bool norm, bool writes, Plan* p) {
    if (n < 0 || (n > 0 && !ts)) return xsg_fail(XSG_ERR_INVALID, "%s: null or negative list of tensors", who);
    int64_t grad_bytes = 0;
    bool masked = false;
    for (int i = 0; i < n; ++i) {
        if (ts[i].numel < 0) return xsg_fail(XSG_ERR_INVALID, "%s: tensor %d has a negative size", who, i);
        if (ts[i].numel > kMaxElements - p->elements) return xsg_fail(XSG_ERR_INVALID, "%s: too many elements", who);
        p->elements += ts[i].numel;
        p->bytes_touched += touched(ts[i]);
        grad_bytes += ts[i].numel * type_size(grad_of(ts[i]).dtype);
        p->f32 = p->f32 && all_f32(ts[i]);
        masked = masked || ts[i].mask;
    }
    p->stream = p->bytes_touched > kCacheBytes;
    // a call that writes loses by it (4 M Gaussians: clip 440 us, around the caches 446; update 1239 and 1271)
    p->stream_norm = !writes && grad_bytes > kCacheBytes;
    const int64_t target = masked ? kMaskedChunks : kDenseChunks;
    p->chunk = chunk_for(p->elements, target, writes && p->stream);
    p->masked_chunk = writes && p->stream ? kMaskedFactor * p->chunk : p->chunk;
    for (int i = 0; i < n; ++i) p->chunks += chunks_of(ts[i].numel, ts[i].mask ? p->masked_chunk : p->chunk);
    if (p->chunks > kMaxChunks) return xsg_fail(XSG_ERR_INVALID, "%s: too many tensors", who);
    if (writes) p->each = std::max<int64_t>((p->chunks + target - 1) / target, 1);
    p->parts = (p->chunks + p->each - 1) / p->each;
    p->table = n > kInline<EntryOf<T>>;
    p->bytes = norm ? 256 + aligned((size_t)p->parts * sizeof(double)) : 0;
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
        at += (int32_t)chunks_of(ts[i].numel, ts[i].mask ? p.masked_chunk : p.chunk);
    }
    list->first[n] = at;
    list->n = n;
    list->chunk = (int32_t)p.chunk;
    list->masked_chunk = (int32_t)p.masked_chunk;
    list->chunks = at;
}

template <typename T>
int send_table(const T* ts, int n, const Plan& p, void* ws, hipStream_t s, TableList<EntryOf<T>>* list) {
    using E = EntryOf<T>;
    using Piece = TablePiece<E>;
    int32_t* const first = (int32_t*)((char*)ws + p.first_at);
    E* const entry = (E*)((char*)ws + p.entry_at);
    Piece piece;
    int64_t chunks = 0;
    for (int i = 0; i < n;) {
        const int i0 = i;
        int kinds = 0, masks = 0;
        for (piece.n = 0; piece.n < Piece::kMax && i < n; ++i, ++piece.n) {
            const E e = entry_of(ts[i]);
            const EntryKind kind = e.kind();
            int k = 0, m = masks;   // a mask is mostly the last tensor's
            while (k < kinds && !(piece.kind[k] == kind)) ++k;
            while (e.mask && m > 0 && piece.mask[m - 1] != e.mask) --m;
            if (k == Piece::kKinds || (e.mask && m == 0 && masks == Piece::kMasks)) break;
            if (k == kinds) piece.kind[kinds++] = kind;
            if (!e.mask) m = 0;
            else if (m == 0) piece.mask[(m = ++masks) - 1] = e.mask;
            e.pointers(piece.pointer[piece.n]);
            piece.word[piece.n] = (uint64_t)e.numel | (uint64_t)k << 48 | (uint64_t)m << 56;
            piece.first[piece.n] = (int32_t)chunks;
            chunks += chunks_of(e.numel, e.mask ? p.masked_chunk : p.chunk);
        }
        piece.kinds = kinds;
        piece.masks = masks;
        piece.end = i == n ? (int32_t)chunks : -1;
        table_kernel<E><<<1, kBlock, 0, s>>>(piece, entry + i0, first + i0);
        XSG_TRY_LAUNCH("table");
    }
    *list = TableList<E>{entry, first, n, (int32_t)p.chunk, (int32_t)p.masked_chunk, (int32_t)chunks};
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

template <typename L> int launch_partials(const L& list, int norm, const Plan& p, void* ws, int64_t* step, hipStream_t s) {
    const int blocks = std::max<int>((int)p.parts, 1);
    with_norm(norm, [&](auto kind) {
        with_flag(p.stream_norm, [&](auto stream) {
            norm_partial_kernel<kind.value, stream.value><<<blocks, kBlock, 0, s>>>(list, (int)p.each, partials(ws), step);
        });
    });
    return xsg_launch_status("grad_norm");
}

template <int OP, typename T> bool is_small(const T* ts, int n, const Plan& p) {
    if (p.table || p.chunks > kSmallChunks) return false;
    return (OP != kSmallAdam && p.chunks <= kOneRound) ||
           std::all_of(ts, ts + n, [](const T& x) { return x.numel <= kSmallTensor; });
}

template <int OP, typename T>
int launch_small(const T* ts, int n, const Plan& p, const StepRule& rule, const AdamScalars& a, int64_t* step,
                 float* total, float* each, hipStream_t s) {
    InlineList<EntryOf<T>> list;
    fill_inline(ts, n, p, &list);
    with_norm(rule.norm, [&](auto kind) {
        small_kernel<kind.value, OP><<<1, kSmallBlock, 0, s>>>(list, rule, a, step, total, each);
    });
    return xsg_launch_status("small list");
}

// the norm (where the rule has one) and the step's terms, for the launch behind
template <typename L>
int make_terms(const L& list, const StepRule& rule, const Plan& p, void* ws, int64_t* step, float* total, hipStream_t s,
               StepSource* source) {
    *source = StepSource{rule, nullptr, 0, step, total, nullptr};
    if (rule.norm < 0) {
        adam_count_kernel<<<1, 1, 0, s>>>(step);
        return xsg_launch_status("adam_step");
    }
    const int rc = launch_partials(list, rule.norm, p, ws, step, s);
    if (rc != XSG_OK) return rc;
    source->partial = partials(ws);
    source->n = (int)p.parts;
    if (p.each == 1) return XSG_OK;
    step_terms_kernel<<<1, kBlock, 0, s>>>(rule, partials(ws), (int)p.parts, step, total, (StepTerms*)ws);
    source->ready = (const StepTerms*)ws;
    return xsg_launch_status("grad_norm");
}

}  // namespace

extern "C" size_t xsg_grad_norm_workspace_bytes(const xsg_grad_tensor* ts, int n) {
    Plan p;
    return make_plan(ts, n, "grad_norm", true, false, &p) == XSG_OK ? p.bytes : 0;
}

extern "C" int xsg_grad_norm(const xsg_grad_tensor* ts, int n, int norm, float* total, float* each, void* workspace,
                             xsg_stream_t stream) {
    Plan p;
    int rc = make_plan(ts, n, "grad_norm", true, false, &p);
    if (rc == XSG_OK) rc = check_list(ts, n, norm, "grad_norm");
    if (rc != XSG_OK) return rc;
    if (!total || !workspace) return xsg_fail(XSG_ERR_INVALID, "grad_norm: null output or workspace");
    rc = xsg_check_workspace(workspace, "grad_norm");
    if (rc != XSG_OK) return rc;
    const hipStream_t s = (hipStream_t)stream;
    if (is_small<kSmallNorm>(ts, n, p))
        return launch_small<kSmallNorm>(ts, n, p, StepRule{0.0, 0.0, 0.0, 0.0, norm, 0, 0}, AdamScalars{}, nullptr, total,
                                        each, s);
    return with_list(ts, n, p, workspace, s, [&](const auto& list) {
        const int status = launch_partials(list, norm, p, workspace, nullptr, s);
        if (status != XSG_OK) return status;
        const double* const partial = partials(workspace);
        if (each) norm_each_kernel<<<n + 1, kBlock, 0, s>>>(list, partial, norm, total, each);
        else norm_total_kernel<<<1, kBlock, 0, s>>>(partial, (int)p.chunks, norm, total);
        return xsg_launch_status("grad_norm");
    });
}

extern "C" size_t xsg_clip_grads_workspace_bytes(const xsg_grad_tensor* ts, int n) {
    Plan p;
    return make_plan(ts, n, "clip_grads", true, true, &p) == XSG_OK ? p.bytes : 0;
}

extern "C" int xsg_clip_grads(const xsg_grad_tensor* ts, int n, int norm, double max_norm, double eps, float* total,
                              void* workspace, xsg_stream_t stream) {
    Plan p;
    int rc = make_plan(ts, n, "clip_grads", true, true, &p);
    if (rc == XSG_OK) rc = check_list(ts, n, norm, "clip_grads");
    if (rc != XSG_OK) return rc;
    if (!(max_norm >= 0.0) || !(eps >= 0.0))
        return xsg_fail(XSG_ERR_INVALID, "clip_grads: max_norm %g and eps %g must not be negative", max_norm, eps);
    if (!total || !workspace) return xsg_fail(XSG_ERR_INVALID, "clip_grads: null output or workspace");
    rc = xsg_check_workspace(workspace, "clip_grads");
    if (rc != XSG_OK) return rc;
    const hipStream_t s = (hipStream_t)stream;
    const StepRule rule{max_norm, eps, 0.0, 0.0, norm, 1, 0};
    if (is_small<kSmallClip>(ts, n, p))
        return launch_small<kSmallClip>(ts, n, p, rule, AdamScalars{}, nullptr, total, nullptr, s);
    return with_list(ts, n, p, workspace, s, [&](const auto& list) {
        StepSource source;
        const int status = make_terms(list, rule, p, workspace, nullptr, total, s, &source);
        if (status != XSG_OK) return status;
        with_flag(p.stream, [&](auto stream) {
            clip_scale_kernel<stream.value><<<std::max(list.chunks, 1), kBlock, 0, s>>>(list, source);
        });
        return xsg_launch_status("clip_grads");
    });
}

extern "C" int xsg_write_back(void* dst, const void* src, int64_t numel, int element_bytes, int dims, const int64_t* sizes,
                              const int64_t* strides, const uint32_t* mask, int64_t rows, xsg_stream_t stream) {
    if (numel < 0 || numel > kMaxElements) return xsg_fail(XSG_ERR_INVALID, "write_back: %lld elements", (long long)numel);
    if (dims < 0 || dims > kMaxDims || (dims > 0 && (!sizes || !strides)))
        return xsg_fail(XSG_ERR_INVALID, "write_back: %d dimensions, more than %d or without sizes", dims, kMaxDims);
    if (element_bytes != 2 && element_bytes != 4)
        return xsg_fail(XSG_ERR_INVALID, "write_back: elements of %d bytes", element_bytes);
    Strides at{};
    at.dims = dims;
    int64_t count = 1;
    for (int d = 0; d < dims; ++d) {
        at.size[d] = sizes[d];
        at.stride[d] = strides[d];
        if (sizes[d] < 0) count = -1;
        if (count < 0) break;
        count = sizes[d] > 0 && count > kMaxElements / sizes[d] ? kMaxElements + 1 : count * sizes[d];
    }
    if (count != numel)
        return xsg_fail(XSG_ERR_INVALID, "write_back: sizes do not make %lld elements", (long long)numel);
    const int rc = check_rows(numel, mask, rows, "write_back", 0);
    if (rc != XSG_OK || numel == 0) return rc;
    if (!dst || !src) return xsg_fail(XSG_ERR_INVALID, "write_back: null array");
    const int blocks = (int)std::min<int64_t>((numel + kBlock - 1) / kBlock, 1 << 14);
    const int64_t row = mask ? numel / rows : 1;
    // indices of 32 bits where a turn past the last element stays within them
    const bool narrow = numel <= ((int64_t)1 << 31);
    const hipStream_t s = (hipStream_t)stream;
    const auto launch = [&](auto element, auto index) {
        using T = decltype(element);
        using I = decltype(index);
        write_back_kernel<T, I><<<blocks, kBlock, 0, s>>>((T*)dst, (const T*)src, (I)numel, at, mask, (I)row);
    };
    if (element_bytes == 4) narrow ? launch(uint32_t{}, uint32_t{}) : launch(uint32_t{}, uint64_t{});
    else narrow ? launch(uint16_t{}, uint32_t{}) : launch(uint16_t{}, uint64_t{});
    return xsg_launch_status("write_back");
}

extern "C" size_t xsg_adam_step_workspace_bytes(const xsg_adam_tensor* ts, int n, const xsg_adam_options* o) {
    Plan p;
    return o && make_plan(ts, n, "adam_step", o->clip || o->skip_nonfinite, true, &p) == XSG_OK ? p.bytes : 0;
}

extern "C" int xsg_adam_step(const xsg_adam_tensor* ts, int n, const xsg_adam_options* o, int64_t* step, float* total,
                             void* workspace, xsg_stream_t stream) {
    if (!o || !step) return xsg_fail(XSG_ERR_INVALID, "adam_step: null options or step counter");
    const bool needs_norm = o->clip || o->skip_nonfinite;
    Plan p;
    int rc = make_plan(ts, n, "adam_step", needs_norm, true, &p);
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
    const AdamScalars a{(float)o->beta2, (float)(1.0 - o->beta1), (float)(1.0 - o->beta2), (float)o->eps};
    // beta 0: the logarithm is -inf, and 1 - beta^t is 1
    const StepRule rule{o->max_norm, kAdamClipEps, log(o->beta1), log(o->beta2), needs_norm ? o->norm : -1, o->clip,
                        o->skip_nonfinite};
    const hipStream_t s = (hipStream_t)stream;
    if (is_small<kSmallAdam>(ts, n, p)) return launch_small<kSmallAdam>(ts, n, p, rule, a, step, total, nullptr, s);
    return with_list(ts, n, p, workspace, s, [&](const auto& list) {
        StepSource source;
        const int status = make_terms(list, rule, p, workspace, step, total, s, &source);
        if (status != XSG_OK) return status;
        with_flag(p.f32, [&](auto f32) {
            with_flag(p.stream, [&](auto stream) {
                adam_kernel<f32.value, stream.value><<<std::max(list.chunks, 1), kBlock, 0, s>>>(list, a, source);
            });
        });
        return xsg_launch_status("adam_step");
    });
}
