// mem_delta_math.h -- products of the gated delta rule at float32 precision, as
// the matrix instructions give them for each input type, and the LDS tiles
// their operands come from.
//
// Every product sums over 32 inner elements (the tokens of a chunk, or 32 of a
// head's dimensions).  A result tile C[x][y] of 16x16 has C[4g + i][r] in lane
// (r = lane % 16, g = lane / 16); two of them below each other, 32 values of x,
// are the operand of a product over x as they lie: lane (r, g) holds the inner
// elements 4g + i and 16 + 4g + i.  Operands from LDS follow that order.
#pragma once

#include "mem_delta.h"

namespace nesle::mem {

// Place of an inner element within 32 so that a lane's eight lie together.
__device__ constexpr int place_of(int c) { return (c & ~31) | ((c >> 2) & 3) << 3 | ((c >> 4) & 1) << 2 | (c & 3); }

// ---- float32 inputs: v_mfma_f32_16x16x4_f32 -----------------------------------
struct F32Math {
    using In = float;
    struct Op {
        f4 a, b;
    };
    static __device__ Op full(f4 a, f4 b) { return {a, b}; }
    static __device__ Op exact(f4 a, f4 b) { return {a, b}; }
    static __device__ f4 mul(const Op& x, const Op& y, f4 c) { return mma(x.b, y.b, mma(x.a, y.a, c)); }

    // [ROWS][COLS] of float.  A row is 4 words more than a multiple of 32, so
    // that 16 rows start at 16 different groups of four banks.
    template <int ROWS, int COLS, bool FULL>
    struct Tile {
        static constexpr int kRow = COLS + 4;
        alignas(16) float d[ROWS * kRow];
        __device__ void put(int row, int col, float v) { d[row * kRow + col] = v; }
        __device__ void put4(int row, int col, f4 v) { *reinterpret_cast<f4*>(&d[row * kRow + col]) = v; }
        // Eight columns as they lie in memory.
        __device__ void put8(int row, int col, const std::uint32_t (&w)[8]) {
            *reinterpret_cast<u4*>(&d[row * kRow + col]) = u4{w[0], w[1], w[2], w[3]};
            *reinterpret_cast<u4*>(&d[row * kRow + col + 4]) = u4{w[4], w[5], w[6], w[7]};
        }
        // Operand of the 16 rows from row0 over the inner columns 32 p ...
        __device__ Op rows(int row0, int p, int r, int g) const {
            const float* x = &d[(row0 + r) * kRow + 32 * p + 4 * g];
            return {*reinterpret_cast<const f4*>(x), *reinterpret_cast<const f4*>(x + 16)};
        }
        // Operand of the 16 columns from col0 over the inner rows row0 ...
        __device__ Op cols(int row0, int col0, int r, int g) const {
            const float* x = &d[(row0 + 4 * g) * kRow + col0 + r];
            return {f4{x[0], x[kRow], x[2 * kRow], x[3 * kRow]},
                    f4{x[16 * kRow], x[17 * kRow], x[18 * kRow], x[19 * kRow]}};
        }
    };
};

// ---- bfloat16 inputs: v_mfma_f32_16x16x32_bf16 ----------------------------------
// A float32 value is the sum of three bfloat16 values, its 24 significant bits
// cut in three (by truncation, so nothing is lost).  A product of two such
// operands takes the six instructions of the pairs that weigh 2^-16 or more
// against the first; the rest is below 2^-24, where float32 rounds.  Against an
// input, which is one bfloat16 value, three instructions give the product
// whole.  At 16 cycles for 32 inner elements that is 48 or 96 cycles where
// float32's instructions take 256.
struct SplitMath {
    using In = bf16;
    using b8 = bf16 __attribute__((ext_vector_type(8)));
    struct Op {                // float32
        u4 h, m, l;
    };
    struct Exact {             // bfloat16
        u4 h;
    };
    static __device__ std::uint32_t tops(std::uint32_t low, std::uint32_t high) {      // the upper halves of two words
        return __builtin_amdgcn_perm(high, low, 0x07060302u);
    }
    static __device__ void split(f4 x, u2& h, u2& m, u2& l) {
        std::uint32_t w[4], wm[4], wl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = x[i];              // bit casts of a vector's element itself take its first
            w[i] = __builtin_bit_cast(std::uint32_t, v);
            const float rest = v - __builtin_bit_cast(float, w[i] & 0xffff0000u);
            wm[i] = __builtin_bit_cast(std::uint32_t, rest);
            wl[i] = __builtin_bit_cast(std::uint32_t, rest - __builtin_bit_cast(float, wm[i] & 0xffff0000u));
        }
        h = u2{tops(w[0], w[1]), tops(w[2], w[3])};
        m = u2{tops(wm[0], wm[1]), tops(wm[2], wm[3])};
        l = u2{tops(wl[0], wl[1]), tops(wl[2], wl[3])};
    }
    static __device__ u4 both(u2 a, u2 b) { return u4{a.x, a.y, b.x, b.y}; }
    static __device__ Op full(f4 a, f4 b) {
        u2 h0, m0, l0, h1, m1, l1;
        split(a, h0, m0, l0);
        split(b, h1, m1, l1);
        return {both(h0, h1), both(m0, m1), both(l0, l1)};
    }
    static __device__ Exact exact(f4 a, f4 b) {            // values that are bfloat16
        const auto w = [](float x) { return __builtin_bit_cast(std::uint32_t, x); };
        return {u4{tops(w(a.x), w(a.y)), tops(w(a.z), w(a.w)), tops(w(b.x), w(b.y)), tops(w(b.z), w(b.w))}};
    }
    static __device__ f4 one(u4 x, u4 y, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
    }
    static __device__ f4 mul(const Exact& x, const Exact& y, f4 c) { return one(x.h, y.h, c); }
    static __device__ f4 mul(const Exact& x, const Op& y, f4 c) { return one(x.h, y.h, one(x.h, y.m, one(x.h, y.l, c))); }
    static __device__ f4 mul(const Op& x, const Exact& y, f4 c) { return one(x.h, y.h, one(x.m, y.h, one(x.l, y.h, c))); }
    static __device__ f4 mul(const Op& x, const Op& y, f4 c) {
        c = one(x.m, y.m, one(x.h, y.l, one(x.l, y.h, c)));
        return one(x.h, y.h, one(x.h, y.m, one(x.m, y.h, c)));
    }

    // [ROWS][COLS] of bfloat16 (FULL: of float32, in three planes), columns in
    // place_of order.  A row is 16 bytes more than a multiple of 64, so that
    // 16-byte reads of 16 rows spread over the banks.
    template <int ROWS, int COLS, bool FULL>
    struct Tile {
        static constexpr int kRow = COLS + 8, kPlane = ROWS * kRow;
        alignas(16) std::uint16_t d[(FULL ? 3 : 1) * kPlane];
        __device__ void put(int row, int col, float v) {
            const std::uint32_t w = __builtin_bit_cast(std::uint32_t, v);
            std::uint16_t* to = &d[row * kRow + place_of(col)];
            to[0] = static_cast<std::uint16_t>(w >> 16);
            if constexpr (FULL) {
                const float rest = v - __builtin_bit_cast(float, w & 0xffff0000u);
                const std::uint32_t wm = __builtin_bit_cast(std::uint32_t, rest);
                const float low = rest - __builtin_bit_cast(float, wm & 0xffff0000u);
                to[kPlane] = static_cast<std::uint16_t>(wm >> 16);
                to[2 * kPlane] = static_cast<std::uint16_t>(__builtin_bit_cast(std::uint32_t, low) >> 16);
            }
        }
        __device__ void put4(int row, int col, f4 v) {
            u2 h, m, l;
            split(v, h, m, l);
            std::uint16_t* to = &d[row * kRow + place_of(col)];
            *reinterpret_cast<u2*>(to) = h;
            if constexpr (FULL) {
                *reinterpret_cast<u2*>(to + kPlane) = m;
                *reinterpret_cast<u2*>(to + 2 * kPlane) = l;
            }
        }
        __device__ void put8(int row, int col, const std::uint32_t (&w)[4]) {
            static_assert(!FULL);
            *reinterpret_cast<u2*>(&d[row * kRow + place_of(col)]) = u2{w[0], w[1]};
            *reinterpret_cast<u2*>(&d[row * kRow + place_of(col + 4)]) = u2{w[2], w[3]};
        }
        __device__ auto rows(int row0, int p, int r, int g) const {
            const auto at = [&](int plane) { return *reinterpret_cast<const u4*>(&d[plane * kPlane + (row0 + r) * kRow + 32 * p + 8 * g]); };
            if constexpr (FULL) return Op{at(0), at(1), at(2)};
            else return Exact{at(0)};
        }
        // The transposing read hands 16 lanes a block of 4 rows and 16 columns:
        // lane 4 j + q fetches columns 4 q .. of row j, lane r gets column r.
        __device__ auto cols(int row0, int col0, int r, int g) const {
            using s4 = short __attribute__((ext_vector_type(4)));
            using lds = __attribute__((address_space(3))) s4;
            const std::uint16_t* from = &d[(row0 + 4 * g + r / 4) * kRow + place_of(col0 + 4 * (r % 4))];
            const auto at = [&](int plane) {
                const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(from + plane * kPlane));
                const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(from + plane * kPlane + 16 * kRow));
                return both(__builtin_bit_cast(u2, a), __builtin_bit_cast(u2, b));
            };
            if constexpr (FULL) return Op{at(0), at(1), at(2)};
            else return Exact{at(0)};
        }
    };
};

template <typename T>
struct MathOf;
template <>
struct MathOf<float> {
    using type = F32Math;
};
template <>
struct MathOf<bf16> {
    using type = SplitMath;
};

// v as lane r - N (ROW_SHR: zero where there is none) or r + N around (ROW_ROR)
// of the same 16 lanes holds it.
constexpr int kRowShr = 0x110, kRowRor = 0x120;
template <int CTRL>
__device__ float moved(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// Sum over the 16 lanes of a row, in all of them.
__device__ inline float sum16(float v) {
    v += moved<kRowRor + 8>(v);
    v += moved<kRowRor + 4>(v);
    v += moved<kRowRor + 2>(v);
    return v + moved<kRowRor + 1>(v);
}
// Sum over the lanes below in a row of 16.
__device__ inline float sum_below(float v) {
    v += moved<kRowShr + 1>(v);
    v += moved<kRowShr + 2>(v);
    v += moved<kRowShr + 4>(v);
    v += moved<kRowShr + 8>(v);
    return moved<kRowShr + 1>(v);
}
// Sum over the wave's four rows of 16 lanes.
__device__ inline float over_groups(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

}  // namespace nesle::mem
