// Dropout's random numbers: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", 2011), a bijection of a 128-bit counter under a 64-bit key. Draw e is a function of its number, the
// seed and a stream alone, so a backward pass draws the same bits again and no mask is stored.
#pragma once
#include <math.h>

#include "xsg_common.h"

struct Words4 { uint32_t w[4]; };

XSG_HD Words4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        const uint32_t n0 = (uint32_t)(b >> 32) ^ c1 ^ k0, n2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c0 = n0; c1 = (uint32_t)b; c2 = n2; c3 = (uint32_t)a;
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
    return Words4{{c0, c1, c2, c3}};
}

// What a kernel needs of a drop: value e is dropped where its 32 bits are below threshold = round(p 2^32), and kept
// ones are multiplied by factor = 1 / (1 - threshold / 2^32), so that expectations stay as they are exactly.
struct DropArgs {
    uint64_t threshold;     // 0 .. 2^32
    uint64_t seed;
    const uint64_t* seed_at;   // on the device, in place of seed where not NULL (a replayed graph reads it anew)
    uint32_t stream;
    float factor;
};

// The arguments of a checked xsg_drop_desc (NULL: nothing is dropped).
inline int drop_args(const xsg_drop_desc* d, DropArgs& out, const char* who) {
    out = DropArgs{0, 0, nullptr, 0, 1.0f};
    if (!d) return XSG_OK;
    if (!(d->p >= 0.0 && d->p <= 1.0)) return xsg_fail(XSG_ERR_INVALID, "%s: a drop probability lies in [0, 1]", who);
    out.threshold = (uint64_t)nearbyint(d->p * 4294967296.0);
    out.seed = d->seed;
    out.seed_at = d->seed_at;
    out.stream = d->stream;
    out.factor = out.threshold >> 32 ? 0.0f : (float)(4294967296.0 / (4294967296.0 - (double)out.threshold));
    return XSG_OK;
}

// The draws of one call in the kernel.
struct Draws {
    uint32_t k0, k1, stream, upper, lower;   // upper: the threshold's upper 16 bits (up to 2^16)

    XSG_DEV explicit Draws(const DropArgs& d) {
        const uint64_t seed = d.seed_at ? *d.seed_at : d.seed;
        k0 = (uint32_t)seed; k1 = (uint32_t)(seed >> 32);
        stream = d.stream;
        upper = (uint32_t)(d.threshold >> 16); lower = (uint32_t)d.threshold & 0xffffu;
    }
    XSG_DEV Words4 words(uint64_t block, uint32_t last) const {
        return philox((uint32_t)block, (uint32_t)(block >> 32), stream, last, k0, k1);
    }
    // Bit j: value 8 block + j is kept. Sixteen bits a value, so one call serves eight; only a value whose sixteen
    // equal the threshold's (1 in 65536) needs the lower sixteen, from a second call. So the comparison is of 32
    // bits at the price of 16: the generator's integer products issue at a quarter of the rate, and with 32 bits
    // a value they would take as long as moving it.
    XSG_DEV uint32_t keep8(uint64_t block) const {
        const Words4 r = words(block, 0);
        uint32_t keep = 0, tie = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t h = j & 1 ? r.w[j >> 1] >> 16 : r.w[j >> 1] & 0xffffu;
            keep |= (uint32_t)(h >= upper) << j;
            tie |= (uint32_t)(h == upper) << j;
        }
        if (lower != 0 && tie != 0) {
            const Words4 s = words(block, 1);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t h = j & 1 ? s.w[j >> 1] >> 16 : s.w[j >> 1] & 0xffffu;
                if ((tie >> j & 1) && h < lower) keep &= ~(1u << j);
            }
        }
        return keep;
    }
    // Bit j < n: value first + j is kept, n up to 8; two calls where they lie in two blocks.
    XSG_DEV uint32_t keep(uint64_t first, int n) const {
        const uint32_t at = (uint32_t)first & 7u;
        uint32_t bits = keep8(first >> 3);
        if (at + n > 8) bits |= keep8((first >> 3) + 1) << 8;
        return bits >> at;
    }
};
