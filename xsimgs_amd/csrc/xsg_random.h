// Dropout's random numbers: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", 2011), a bijection of a 128-bit counter under a 64-bit key. Draw e is a function of its number, the
// seed and a stream alone, so a backward pass draws the same bits again and no mask is stored.
#pragma once
#include <math.h>

#include "xsg_common.h"

struct Words4 { uint32_t w[4]; };

XSG_DEV uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }

XSG_DEV Words4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        const uint32_t n0 = xor3((uint32_t)(b >> 32), c1, k0), n2 = xor3((uint32_t)(a >> 32), c3, k1);
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
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
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
    // a value they would take as long as moving it. The halves are compared two at a time.
    XSG_DEV uint32_t keep8(uint64_t block) const {
        const Words4 r = words(block, 0);
        const uint32_t below = (upper ? upper - 1 : 0) * 0x10001u;
        uint32_t m = upper ? 0 : 0x550055u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            // 1 in each half that is above `below`: the saturated difference, or 1 (by name: the compiler takes this
            // apart into comparisons and selections of single halves)
            uint32_t over;
            asm("v_pk_sub_u16 %0, %1, %2 clamp\n\tv_pk_min_u16 %0, %0, %3" : "=&v"(over) : "v"(r.w[k]), "v"(below), "v"(0x10001u));
            m |= over << (2 * k);
        }
        uint32_t keep = (m | m >> 15) & 0xffu;
        ties(r, block, [&](int j) { keep &= ~(1u << j); });
        return keep;
    }
    // The same as words of ones and zeros: half j % 2 of word j / 2 for value 8 block + j.
    XSG_DEV Words4 halves8(uint64_t block) const {
        const Words4 r = words(block, 0);
        const uint32_t below = (upper ? upper - 1 : 0) * 0x10001u;
        Words4 m;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            asm("v_pk_sub_u16 %0, %1, %2 clamp\n\tv_pk_min_u16 %0, %0, %3\n\tv_pk_sub_u16 %0, 0, %0"
                : "=&v"(m.w[k]) : "v"(r.w[k]), "v"(below), "v"(0x10001u));
            if (upper == 0) m.w[k] = ~0u;
        }
        ties(r, block, [&](int j) { m.w[j >> 1] &= j & 1 ? 0xffffu : 0xffff0000u; });
        return m;
    }
    // drop(j) for each value whose upper bits are the threshold's and whose lower ones are below it
    template <typename F> XSG_DEV void ties(const Words4& r, uint64_t block, F drop) const {
        const uint32_t at = upper * 0x10001u;
        uint32_t apart = ~0u;   // a half of 0 where one equals the threshold's
#pragma unroll
        for (int k = 0; k < 4; ++k)
            apart = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, apart),
                                                                           __builtin_bit_cast(u16x2, r.w[k] ^ at)));
        if (lower != 0 && ((apart & 0xffffu) == 0 || apart < 0x10000u)) {
            const Words4 s = words(block, 1);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t h = r.w[j >> 1] >> 16 * (j & 1) & 0xffffu, l = s.w[j >> 1] >> 16 * (j & 1) & 0xffffu;
                if (h == upper && l < lower) drop(j);
            }
        }
    }
    XSG_DEV static Words4 halves_of(uint32_t keep) {
        Words4 m;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            m.w[k] = ((uint32_t)__builtin_amdgcn_sbfe((int)keep, 2 * k, 1) & 0xffffu) |
                     ((uint32_t)__builtin_amdgcn_sbfe((int)keep, 2 * k + 1, 1) & 0xffff0000u);
        return m;
    }
    // Bit j < n: value first + j is kept, n up to 8; two calls where they lie in two blocks.
    XSG_DEV uint32_t keep(uint64_t first, int n) const {
        const uint32_t at = (uint32_t)first & 7u;
        uint32_t bits = keep8(first >> 3);
        if (at + n > 8) bits |= keep8((first >> 3) + 1) << 8;
        return bits >> at;
    }
    // Bits from value first on (eight, or four where they need not reach further) for two sets of runs, in each of which the
    // lanes of a wavefront, all of them here, hold runs of eight (four) in order, next to each other or overlapping: they
    // lie in about 64 (32) blocks, so a lane draws one block of the set (half the lanes for each of two sets) and takes its
    // own two from the lanes that have them.
    XSG_DEV uint32_t shared_keep(uint64_t first, uint64_t base, uint32_t drawn, int lane0, int lanes, int values) const {
        const uint64_t mine = first >> 3, from = mine - base;
        uint32_t bits = __shfl(drawn, lane0 + (int)(from & (lanes - 1))) | __shfl(drawn, lane0 + (int)((from + 1) & (lanes - 1))) << 8;
        // lanes at the end of a wavefront may reach past what it drew
        if (from + 2 > (uint64_t)lanes) {
            if (from >= (uint64_t)lanes) bits = keep8(mine) | (bits & 0xff00u);
            if ((first & 7u) + values > 8) bits = (bits & 0xffu) | keep8(mine + 1) << 8;
        }
        return bits >> ((uint32_t)first & 7u);
    }
    XSG_DEV static uint64_t of_first_lane(uint64_t x) {
        return (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)x) | (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32;
    }
    XSG_DEV uint32_t keep_in_order(uint64_t first) const {
        const uint64_t base = of_first_lane(first >> 3);
        return shared_keep(first, base, keep8(base + __lane_id()), 0, 64, 8);
    }
    XSG_DEV void keep_in_order(uint64_t first, uint64_t second, uint32_t& a, uint32_t& b) const {
        const uint64_t base = of_first_lane(first >> 3), base2 = of_first_lane(second >> 3);
        const uint32_t lane = __lane_id();
        const uint32_t drawn = keep8((lane < 32 ? base : base2) + (lane & 31));
        a = shared_keep(first, base, drawn, 0, 32, 4);
        b = shared_keep(second, base2, drawn, 32, 32, 4);
    }
};

// x where bit j of keep is set, else 0, whatever x holds
XSG_DEV float keep_bit(float x, uint32_t keep, int j) {
    uint32_t all = (uint32_t)__builtin_amdgcn_sbfe((int)keep, j, 1);
    asm("" : "+v"(all));   // one AND: the compiler would make a comparison and a selection of it
    return __uint_as_float(__float_as_uint(x) & all);
}
