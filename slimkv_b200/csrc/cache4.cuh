// Rows of the 4-bit cache: geometry, and codes to 16-bit values.
//
// A row of D dims (a multiple of 32) holds
//   [D / 2 bytes of codes | D / 32 pairs (scale, low) of 16 bits | up to a multiple of 16 bytes]
// and a code c of a group of 32 dims stands for T(c * scale + low), one
// rounding to the rows' type T (bf16 or fp16).  Word w of the codes holds the
// dims 8w .. 8w + 7: dim 8w + 2j + h at bits 16h + 4j, so that one mask (and a
// shift) takes the pair (2j, 2j + 1) out as the two halves of a register.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace slimkv {

constexpr int kGroupDims = 32;
constexpr int kMaxDims4 = 320;

__host__ __device__ __forceinline__ constexpr int codes_bytes(int dim) { return dim / 2; }
__host__ __device__ __forceinline__ constexpr int row4_bytes(int dim) { return (dim / 2 + dim / 8 + 15) & ~15; }

// n / d for any 32-bit n by a multiplication (Granlund and Montgomery, 1994).
struct FastDiv {
    uint32_t mul, shift, d;
    FastDiv() = default;
    explicit FastDiv(uint32_t divisor) : d(divisor) {
        shift = 0;
        while ((uint64_t(1) << shift) < divisor) ++shift;
        mul = uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - divisor)) / divisor + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const {         // n < 2^31
        return (__umulhi(mul, n) + n) >> shift;
    }
};

// a & b | c in one instruction, b and c in registers: given as constants they cost two.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
// A constant that the compiler keeps in a register.
__device__ __forceinline__ uint32_t in_register(uint32_t x) {
    uint32_t y;
    asm volatile("mov.b32 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// The arithmetic of a type on pairs of values in a register.
template <bool kHalf>
struct Pair {
    using T2 = typename std::conditional<kHalf, __half2, __nv_bfloat162>::type;
    static __device__ __forceinline__ T2 as(uint32_t x) { return *reinterpret_cast<T2*>(&x); }
    static __device__ __forceinline__ uint32_t bits(T2 x) { return *reinterpret_cast<uint32_t*>(&x); }
    // Masks and powers of two of codes() (once for a thread).
    struct Constants {
        uint32_t even = in_register(0x000f000fu), odd = kHalf ? in_register(0x00f000f0u) : 0u;
        uint32_t power = in_register(kHalf ? 0x64006400u : 0x43004300u);
    };
    // The codes at bits 4j of both halves of x, exactly, as values of the type: put into the last
    // bits of a power of two (128 has bf16's last bit at 1, 1024 fp16's), which is then taken off.
    // fp16's ten bits hold a code at bits 4 to 7 too (1024 + 16 c), which saves every other shift.
    template <int j>
    static __device__ __forceinline__ T2 codes(const Constants& c, uint32_t x) {
        if constexpr (kHalf) {
            const uint32_t s = j >= 2 ? x >> 8 : x;
            if constexpr (j % 2 == 0) return __hsub2(as(and_or(s, c.even, c.power)), as(c.power));
            else return __hfma2(as(and_or(s, c.odd, c.power)), as(0x2c002c00u), as(0xd400d400u));   // / 16 - 64
        } else {
            return __hsub2(as(and_or(x >> (4 * j), c.even, c.power)), as(c.power));
        }
    }
    // T(c * scale + low) of the pair at bits 4j.
    template <int j>
    static __device__ __forceinline__ uint32_t values(const Constants& c, uint32_t x, T2 scale, T2 low) {
        return bits(__hfma2(codes<j>(c, x), scale, low));
    }
    static __device__ __forceinline__ bool finite(uint32_t param) {     // of (scale, low)
        constexpr uint32_t kExp = kHalf ? 0x7c00u : 0x7f80u;
        return (param & kExp) != kExp && (param >> 16 & kExp) != kExp;
    }
};
// Both halves the low (high) half of x; the low (high) halves of a and b.
__device__ __forceinline__ uint32_t low_twice(uint32_t x) { return __byte_perm(x, x, 0x1010); }
__device__ __forceinline__ uint32_t high_twice(uint32_t x) { return __byte_perm(x, x, 0x3232); }
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

// -------------------------------------------------------------- products --
// D += A . B of 16-bit pairs in the rows' type.
template <bool kHalf>
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (kHalf) mma_f16(d, a, b0, b1);
    else mma_bf16(d, a, b0, b1);
}
// W words of shared memory (4 W-byte aligned): plain loads, which the compiler may move.
template <int W>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
    if constexpr (W == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    } else if constexpr (W == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[0] = x.x; w[1] = x.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}
__device__ __forceinline__ uint32_t load_word(const uint8_t* p) { return *reinterpret_cast<const uint32_t*>(p); }
// The words (8 dims each) of a K row that lane column t of the MMA takes, G of
// them: of every four groups one (four words in one load), then half of one of
// two groups, then a quarter of the last.
template <int G>
struct KeyWords {
    static constexpr int kQuads = G / 4, kPair = G / 2 % 2, kOne = G % 2;
    // First dim of lane t's word i.
    __device__ __forceinline__ static constexpr int dim(int i, int t) {
        return i < 4 * kQuads            ? 128 * (i / 4) + 32 * t + 8 * (i % 4)
               : i < 4 * kQuads + 2 * kPair ? 128 * kQuads + 16 * t + 8 * (i - 4 * kQuads)
                                         : 128 * kQuads + 64 * kPair + 8 * t;
    }
};

// Lengths of a kernel's rows: those that it is made for, or shorter ones.
template <int G, bool kExact>
struct RowShape {
    int given;                                  // groups
    __device__ __forceinline__ int groups() const { return kExact ? G : given; }
    __device__ __forceinline__ int pitch() const { return row4_bytes(kGroupDims * groups()); }
    // Byte of the pair of the group of dim d; for a dim behind the row (which stands for a zero) of the last one.
    __device__ __forceinline__ int pair_at(int d) const {
        return 16 * groups() + 4 * (kExact ? d / kGroupDims : min(d / kGroupDims, given - 1));
    }
    __device__ __forceinline__ bool has(int d) const { return kExact || d < kGroupDims * given; }
};

// S [16 keys x 8 rows] of NT row tiles += K . Q^T: k0 (shared memory) the row of
// the key g of this lane (g = lane / 4), query(n, i) the dims of word i and row g
// of tile n.  Called with constant n and i.
template <int G, int NT, bool kHalf, class Shape, class Query>
__device__ __forceinline__ void key_products(float (&s)[NT][4], const uint8_t* k0, Shape shape, int t, const typename Pair<kHalf>::Constants& c, Query query) {
    using P = Pair<kHalf>;
    using KW = KeyWords<G>;
    const uint8_t* k1 = k0 + 8 * shape.pitch();
    auto words = [&](auto width, auto first) {
        constexpr int W = decltype(width)::value, i0 = decltype(first)::value;
        uint32_t a0[W], a1[W];
        const int d0 = KW::dim(i0, t);
        load_words<W>(k0 + d0 / 2, a0);
        load_words<W>(k1 + d0 / 2, a1);
        uint32_t p0 = load_word(k0 + shape.pair_at(d0)), p1 = load_word(k1 + shape.pair_at(d0));
        if (!shape.has(d0)) p0 = p1 = 0;
        const auto sc0 = P::as(low_twice(p0)), lo0 = P::as(high_twice(p0)), sc1 = P::as(low_twice(p1)), lo1 = P::as(high_twice(p1));
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const uint32_t x[4] = {P::template values<0>(c, a0[k], sc0, lo0), P::template values<0>(c, a1[k], sc1, lo1),
                                   P::template values<1>(c, a0[k], sc0, lo0), P::template values<1>(c, a1[k], sc1, lo1)};
            const uint32_t y[4] = {P::template values<2>(c, a0[k], sc0, lo0), P::template values<2>(c, a1[k], sc1, lo1),
                                   P::template values<3>(c, a0[k], sc0, lo0), P::template values<3>(c, a1[k], sc1, lo1)};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint4 q = query(n, i0 + k);
                mma<kHalf>(s[n], x, q.x, q.y);
                mma<kHalf>(s[n], y, q.z, q.w);
            }
        }
    };
    using std::integral_constant;
    if constexpr (KW::kQuads > 0) words(integral_constant<int, 4>(), integral_constant<int, 0>());
    if constexpr (KW::kQuads > 1) words(integral_constant<int, 4>(), integral_constant<int, 4>());
    if constexpr (KW::kPair != 0) words(integral_constant<int, 2>(), integral_constant<int, 4 * KW::kQuads>());
    if constexpr (KW::kOne != 0) words(integral_constant<int, 1>(), integral_constant<int, 4 * KW::kQuads + 2 * KW::kPair>());
}

}  // namespace slimkv
