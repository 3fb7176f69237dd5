// Dropout with draws made anew from (number, seed, stream) in the forward and in the backward, so that no mask is
// stored; and the draws as a packed mask, for the tiling. No reference counterpart.
#include <algorithm>

#include "xsg_elements.h"
#include "xsg_random.h"

namespace {

constexpr int kBlock = 256;
constexpr int kUnroll = 2;                          // blocks of eight elements in flight in a thread
constexpr int kSpan = kBlock * kUnroll * 8;         // elements a workgroup takes at a time
constexpr int64_t kMaxGrid = 1 << 23;               // below 2^32 threads a launch; longer tensors loop

// the elements from i0 on (up to eight) times factor where keep's bit is set
template <int DT> XSG_DEV void drop_tail(const void* x, void* out, int64_t i0, int64_t n, uint32_t keep, float factor) {
    for (int j = 0; j < 8 && i0 + j < n; ++j)
        store_one<DT>(out, i0 + j, keep >> j & 1 ? load_one<DT>(x, i0 + j) * factor : 0.0f);
}

template <int DT, bool STREAM> XSG_DEV void drop_store(void* out, int64_t i0, const Raw<8 * ElementSize<DT>::value>& raw,
                                          uint32_t keep, float factor) {
    float v[8];
    unpack<DT, 8>(raw, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = keep_bit(v[j] * factor, keep, j);
    store_raw<DT, 8, STREAM>(out, i0, pack<DT, 8>(v));
}

// One draw an element. Bound by memory: 133 M bfloat16 values take 85 us, 6.2 TB/s read and written; the draws issue
// about 17 operations a value beside it.
template <int DT, bool STREAM>
__global__ __launch_bounds__(kBlock) void dropout_kernel(int64_t n, DropArgs drop, const void* x, void* out) {
    const Draws draws(drop);
    for (int64_t base = (int64_t)blockIdx.x * kSpan; base < n; base += (int64_t)gridDim.x * kSpan) {
        const int64_t first = base + 8 * threadIdx.x;
        if (base + kSpan <= n) {
            Raw<8 * ElementSize<DT>::value> raw[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) raw[u] = load_raw<DT, 8, STREAM>(x, first + u * 8 * kBlock);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int64_t i0 = first + u * 8 * kBlock;
                drop_store<DT, STREAM>(out, i0, raw[u], draws.keep8((uint64_t)i0 >> 3), drop.factor);
            }
        } else {
            for (int u = 0; u < kUnroll; ++u) {
                const int64_t i0 = first + u * 8 * kBlock;
                if (i0 >= n) break;
                const uint32_t keep = draws.keep8((uint64_t)i0 >> 3);
                if (i0 + 8 <= n) drop_store<DT, STREAM>(out, i0, load_raw<DT, 8, STREAM>(x, i0), keep, drop.factor);
                else drop_tail<DT>(x, out, i0, n, keep, drop.factor);
            }
        }
    }
}

// One draw to `row` consecutive elements. A workgroup's elements start in row `base / row`; within its span a row's
// number comes from a multiply (exact: offsets and rows below 2^15), or, in rows as long as the span, a comparison.
// Bound by memory: 1 M rows of 48 float32, a quarter dropped, take 69 us (336 MB, 4.8 TB/s).
template <int DT, bool STREAM>
__global__ __launch_bounds__(kBlock) void dropout_rows_kernel(int64_t n, int64_t row, uint32_t magic, DropArgs drop,
                                                              const void* x, void* out) {
    const Draws draws(drop);
    for (int64_t base = (int64_t)blockIdx.x * kSpan; base < n; base += (int64_t)gridDim.x * kSpan) {
        const int64_t base_row = base / row, base_at = base - base_row * row;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int local = u * 8 * kBlock + 8 * (int)threadIdx.x;
            const int64_t i0 = base + local;
            if (i0 >= n) break;
            int64_t first, at;
            if (row < kSpan) {
                const uint32_t o = (uint32_t)base_at + local, q = __umulhi(o, magic);
                first = base_row + q;
                at = o - q * (uint32_t)row;
            } else {
                const bool next = base_at + local >= row;
                first = base_row + next;
                at = base_at + local - (next ? row : 0);
            }
            // rows that these eight elements touch, then each element's bit
            const int touched = row >= 8 ? 1 + (at + 8 > row) : 8;
            const uint32_t bits = draws.keep((uint64_t)first, touched);
            uint32_t keep = 0;
#pragma unroll
            for (int j = 0, r = 0; j < 8; ++j) {
                keep |= (bits >> r & 1) << j;
                if (++at == row) { at = 0; ++r; }
            }
            if (i0 + 8 <= n) {
                Raw<8 * ElementSize<DT>::value> raw = {};
                if (keep) raw = load_raw<DT, 8, STREAM>(x, i0);
                drop_store<DT, STREAM>(out, i0, raw, keep, drop.factor);
            } else {
                drop_tail<DT>(x, out, i0, n, keep, drop.factor);
            }
        }
    }
}

// One byte of the packed mask a thread, zeros behind the last value.
__global__ __launch_bounds__(kBlock) void drop_mask_kernel(int64_t n, int64_t bytes, DropArgs drop, uint8_t* out) {
    const Draws draws(drop);
    for (int64_t q = (int64_t)blockIdx.x * kBlock + threadIdx.x; q < bytes; q += (int64_t)gridDim.x * kBlock) {
        const int64_t left = n - 8 * q;
        const uint32_t valid = left >= 8 ? 0xffu : left > 0 ? (1u << left) - 1u : 0u;
        out[q] = (uint8_t)(draws.keep8((uint64_t)q) & valid);
    }
}

// Values of 16 bits go around the last-level cache where a call moves more than half of it (133 M: 85 us, 90 through it).
// Those of 32 do not: a thread's eight are two accesses of half a line (48 M in rows of 48: 73 us around, 69 through).
constexpr int64_t kCacheBytes = (int64_t)128 << 20;

unsigned spans(int64_t n, int64_t span) { return (unsigned)std::min<int64_t>((n + span - 1) / span, kMaxGrid); }

}  // namespace

extern "C" int xsg_dropout(const xsg_drop_desc* drop, int dtype, int64_t numel, int64_t shared, const void* x, void* out,
                           xsg_stream_t stream) {
    DropArgs d;
    if (const int rc = drop_args(drop, d, "dropout")) return rc;
    if (!drop) return xsg_fail(XSG_ERR_INVALID, "dropout: null description");
    if (numel < 0 || shared < 1 || numel % shared)
        return xsg_fail(XSG_ERR_INVALID, "dropout: bad sizes (%lld elements, %lld to a draw)", (long long)numel, (long long)shared);
    if (numel > 0 && (!x || !out)) return xsg_fail(XSG_ERR_INVALID, "dropout: null tensor");
    if (dtype < XSG_DTYPE_F32 || dtype > XSG_DTYPE_F16) return xsg_fail(XSG_ERR_INVALID, "dropout: unknown type %d", dtype);
    if (numel == 0) return XSG_OK;
    const hipStream_t s = (hipStream_t)stream;
    with_dtype(dtype, [&](auto t) {
        constexpr int DT = decltype(t)::value;
        const auto launch = [&](auto stream_by) {
            constexpr bool STREAM = decltype(stream_by)::value;
            if (shared == 1)
                dropout_kernel<DT, STREAM><<<spans(numel, kSpan), kBlock, 0, s>>>(numel, d, x, out);
            else
                dropout_rows_kernel<DT, STREAM><<<spans(numel, kSpan), kBlock, 0, s>>>(
                    numel, shared, (uint32_t)(((uint64_t)1 << 32) / (uint64_t)shared + 1), d, x, out);
        };
        if constexpr (DT != XSG_DTYPE_F32) {
            if (2 * numel * ElementSize<DT>::value > kCacheBytes) return launch(std::true_type{});
        }
        launch(std::false_type{});
    });
    XSG_TRY_LAUNCH("dropout");
    return XSG_OK;
}

extern "C" int xsg_drop_mask(const xsg_drop_desc* drop, int64_t n, uint32_t* out, xsg_stream_t stream) {
    DropArgs d;
    if (const int rc = drop_args(drop, d, "drop_mask")) return rc;
    if (!drop) return xsg_fail(XSG_ERR_INVALID, "drop_mask: null description");
    if (n < 0) return xsg_fail(XSG_ERR_INVALID, "drop_mask: negative size");
    if (n == 0) return XSG_OK;
    if (!out) return xsg_fail(XSG_ERR_INVALID, "drop_mask: null tensor");
    const int64_t bytes = (n + 31) / 32 * 4;
    drop_mask_kernel<<<spans(bytes, kBlock), kBlock, 0, (hipStream_t)stream>>>(n, bytes, d, (uint8_t*)out);
    XSG_TRY_LAUNCH("drop_mask");
    return XSG_OK;
}
