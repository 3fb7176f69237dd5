// Runs of consecutive elements of float32, bfloat16 or float16 as float32 in registers, from places of any
// alignment that the type allows (the hardware takes unaligned vector accesses).
#pragma once
#include "xsg_common.h"

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int DT> struct ElementSize { static constexpr int value = DT == XSG_DTYPE_F32 ? 4 : 2; };

// BYTES consecutive bytes (2, 4, 8, 16 or 32) aligned to ALIGN
template <int BYTES> struct Raw { uint32_t w[BYTES >= 4 ? BYTES / 4 : 1]; };

template <int ALIGN, bool STREAM, typename T> XSG_DEV T raw_get(const void* p) {
    typedef T U __attribute__((aligned(ALIGN)));
    const U* q = (const U*)p;
    return STREAM ? __builtin_nontemporal_load(q) : *q;
}
template <int ALIGN, bool STREAM, typename T> XSG_DEV void raw_put(void* p, T x) {
    typedef T U __attribute__((aligned(ALIGN)));
    U* q = (U*)p;
    if (STREAM) __builtin_nontemporal_store(x, q);
    else *q = x;
}

template <int DT, int V, bool STREAM = false>
XSG_DEV Raw<V * ElementSize<DT>::value> load_raw(const void* base, int64_t at = 0) {
    constexpr int E = ElementSize<DT>::value, BYTES = V * E;
    const char* p = (const char*)base + at * E;
    Raw<BYTES> r;
    if constexpr (BYTES == 2) {
        r.w[0] = raw_get<E, STREAM, uint16_t>(p);
    } else if constexpr (BYTES == 4) {
        r.w[0] = raw_get<E, STREAM, uint32_t>(p);
    } else if constexpr (BYTES == 8) {
        const u32x2 a = raw_get<E, STREAM, u32x2>(p);
        r.w[0] = a.x; r.w[1] = a.y;
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const u32x4 a = raw_get<E, STREAM, u32x4>(p + 16 * i);
#pragma unroll
            for (int k = 0; k < 4; ++k) r.w[4 * i + k] = a[k];
        }
    }
    return r;
}

template <int DT, int V, bool STREAM = false>
XSG_DEV void store_raw(void* base, int64_t at, const Raw<V * ElementSize<DT>::value>& r) {
    constexpr int E = ElementSize<DT>::value, BYTES = V * E;
    char* p = (char*)base + at * E;
    if constexpr (BYTES == 2) {
        raw_put<E, STREAM, uint16_t>(p, (uint16_t)r.w[0]);
    } else if constexpr (BYTES == 4) {
        raw_put<E, STREAM, uint32_t>(p, r.w[0]);
    } else if constexpr (BYTES == 8) {
        raw_put<E, STREAM, u32x2>(p, u32x2{r.w[0], r.w[1]});
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i)
            raw_put<E, STREAM, u32x4>(p + 16 * i, u32x4{r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]});
    }
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int DT, int V> XSG_DEV void unpack(const Raw<V * ElementSize<DT>::value>& r, float (&x)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if constexpr (DT == XSG_DTYPE_F32) x[j] = __uint_as_float(r.w[j]);
        else if constexpr (DT == XSG_DTYPE_BF16) x[j] = __uint_as_float(j & 1 ? r.w[j >> 1] & 0xffff0000u : r.w[j >> 1] << 16);
        else x[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(j & 1 ? r.w[j >> 1] >> 16 : r.w[j >> 1]));
    }
}

// rounded once, to nearest even; NaNs stay NaNs
template <int DT, int V> XSG_DEV Raw<V * ElementSize<DT>::value> pack(const float (&x)[V]) {
    Raw<V * ElementSize<DT>::value> r;
    if constexpr (DT == XSG_DTYPE_F32) {
#pragma unroll
        for (int j = 0; j < V; ++j) r.w[j] = __float_as_uint(x[j]);
    } else {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const float a = x[j], b = j + 1 < V ? x[j + 1] : 0.0f;
            if constexpr (DT == XSG_DTYPE_BF16) r.w[j >> 1] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
            else r.w[j >> 1] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
        }
    }
    return r;
}

template <int DT> XSG_DEV float load_one(const void* base, int64_t at) {
    float x[1];
    unpack<DT, 1>(load_raw<DT, 1>(base, at), x);
    return x[0];
}
template <int DT> XSG_DEV void store_one(void* base, int64_t at, float x) {
    const float y[1] = {x};
    store_raw<DT, 1>(base, at, pack<DT, 1>(y));
}

// calls f(std::integral_constant<int, XSG_DTYPE_*>{}) for a checked type
template <typename F> void with_dtype(int dtype, F&& f) {
    if (dtype == XSG_DTYPE_F32) f(std::integral_constant<int, XSG_DTYPE_F32>{});
    else if (dtype == XSG_DTYPE_BF16) f(std::integral_constant<int, XSG_DTYPE_BF16>{});
    else f(std::integral_constant<int, XSG_DTYPE_F16>{});
}
