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

#include <type_traits>

#include "mem_delta.h"

namespace nesle::mem {

// Place of an inner element within 32 so that a lane's eight lie together.
__device__ constexpr int place_of(int c) { return (c & ~31) | ((c >> 2) & 3) << 3 | ((c >> 4) & 1) << 2 | (c & 3); }

// Planes of an operand or a tile that hold float32.  Each kind of products has
// planes of its own for the inputs, kIn.
constexpr int kFull = 3;

// ---- v_mfma_f32_16x16x4_f32 ------------------------------------------------------
struct F32Math {
    static constexpr int kIn = 1;
    struct Op {
        f4 a, b;
    };
    static __device__ Op full(f4 a, f4 b) { return {a, b}; }
    static __device__ f4 mul(const Op& x, const Op& y, f4 c) { return mma(x.b, y.b, mma(x.a, y.a, c)); }
    // The same, summed by itself, 16 inner elements at a time, and then added: for
    // sums that cancel later, where the roundings of one long chain would show.
    static __device__ f4 mul_apart(const Op& x, const Op& y, f4 c) {
        const f4 zero = {0, 0, 0, 0};
        return c + (mma(x.a, y.a, zero) + mma(x.b, y.b, zero));
    }
    // The two result tiles that an operand of inputs holds.
    static __device__ void values(const Op& x, f4 (&to)[2]) {
        to[0] = x.a;
        to[1] = x.b;
    }

    // [ROWS][COLS] of float.  A row is 4 words more than a multiple of 32, so
    // that 16 rows start at 16 different groups of four banks.
    template <int ROWS, int COLS, int PLANES, int PAD = 0>
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

// ---- v_mfma_f32_16x16x32_bf16 ----------------------------------------------------
// A float32 value is the sum of three bfloat16 values: itself rounded to nearest,
// at most 2^-8 of it away, what that leaves rounded again, 2^-17, and the rest,
// which fits (the 24 significant bits are 8 and 8 and 8).  A product of two such
// operands takes the six instructions of the pairs that weigh 2^-17 or more
// against the first; the three left out are at most 2^-24 of the product, where
// float32 rounds, and of either sign (planes cut off instead of rounded would leave
// out up to 2^-21, always toward zero).  Against a bfloat16 input, which is one such
// value (IN = 1, else 3), three instructions give the product whole.  At 16 cycles
// for 32 inner elements that is 48 or 96 cycles where float32's instructions take
// 256.  Values above bfloat16's largest, within 2^-9 of float32's, come out not
// finite.
template <int IN>
struct SplitMath {
    static constexpr int kIn = IN;
    using b8 = bf16 __attribute__((ext_vector_type(8)));
    template <int PLANES>
    struct Op {
        u4 x[PLANES];          // from the most significant on
    };
    template <int PLANES>
    static __device__ void split(f4 x, u2 (&to)[PLANES]) {
#pragma unroll
        for (int p = 0; p < PLANES; ++p) {
            to[p] = u2{pack_bf16(x.x, x.y), pack_bf16(x.z, x.w)};
            // As packed words from here on: the compiler would round the lower half of
            // each a second time rather than shift it out.
            asm("" : "+v"(to[p].x), "+v"(to[p].y));
            if (p + 1 < PLANES) x -= f4{lo_half(to[p].x), hi_half(to[p].x), lo_half(to[p].y), hi_half(to[p].y)};
        }
    }
    static __device__ Op<kFull> full(f4 a, f4 b) {
        u2 x[kFull], y[kFull];
        split(a, x);
        split(b, y);
        Op<kFull> o;
#pragma unroll
        for (int p = 0; p < kFull; ++p) o.x[p] = u4{x[p].x, x[p].y, y[p].x, y[p].y};
        return o;
    }
    // The two result tiles that an operand of inputs holds.
    static __device__ void values(const Op<kIn>& o, f4 (&to)[2]) {
        to[0] = to[1] = f4{0, 0, 0, 0};
#pragma unroll
        for (int p = kIn - 1; p >= 0; --p) {
            const u4 w = o.x[p];
            to[0] += f4{lo_half(w.x), hi_half(w.x), lo_half(w.y), hi_half(w.y)};
            to[1] += f4{lo_half(w.z), hi_half(w.z), lo_half(w.w), hi_half(w.w)};
        }
    }
    // The pairs of planes that together weigh no less than the wider operand's last.
    template <int P, int Q>
    static __device__ f4 mul(const Op<P>& x, const Op<Q>& y, f4 c) {
        constexpr int most = (P > Q ? P : Q) - 1;
#pragma unroll
        for (int sum = most; sum >= 0; --sum)
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (sum - p >= 0 && sum - p < Q)
                    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x.x[p]),
                                                                __builtin_bit_cast(b8, y.x[sum - p]), c, 0, 0, 0);
        return c;
    }

    template <int P, int Q>
    static __device__ f4 mul_apart(const Op<P>& x, const Op<Q>& y, f4 c) { return c + mul(x, y, f4{0, 0, 0, 0}); }

    // [ROWS][COLS] of values in planes of bfloat16, columns in place_of order.
    // A row is PAD elements longer: 8 (16 bytes) for a tile that is read by rows,
    // whose 16-byte reads of 16 rows then spread over the banks.
    template <int ROWS, int COLS, int PLANES, int PAD = 8>
    struct Tile {
        static constexpr int kRow = COLS + PAD, kPlane = ROWS * kRow;
        alignas(16) std::uint16_t d[PLANES * kPlane];
        __device__ void put(int row, int col, float v) {
            std::uint16_t* to = &d[row * kRow + place_of(col)];
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
                const bf16 top = static_cast<bf16>(v);
                to[p * kPlane] = __builtin_bit_cast(std::uint16_t, top);
                v -= static_cast<float>(top);
            }
        }
        __device__ void put4(int row, int col, f4 v) {
            u2 x[PLANES];
            split(v, x);
#pragma unroll
            for (int p = 0; p < PLANES; ++p) *reinterpret_cast<u2*>(&d[p * kPlane + row * kRow + place_of(col)]) = x[p];
        }
        // Eight columns as they lie in memory.
        __device__ void put8(int row, int col, const std::uint32_t (&w)[4]) {
            static_assert(PLANES == 1);
            *reinterpret_cast<u2*>(&d[row * kRow + place_of(col)]) = u2{w[0], w[1]};
            *reinterpret_cast<u2*>(&d[row * kRow + place_of(col + 4)]) = u2{w[2], w[3]};
        }
        __device__ void put8(int row, int col, const std::uint32_t (&w)[8]) {
            put4(row, col, __builtin_bit_cast(f4, u4{w[0], w[1], w[2], w[3]}));
            put4(row, col + 4, __builtin_bit_cast(f4, u4{w[4], w[5], w[6], w[7]}));
        }
        // Operand of the 16 rows from row0 over the inner columns 32 p ...
        __device__ Op<PLANES> rows(int row0, int p, int r, int g) const {
            static_assert(PAD % 8 == 0);
            Op<PLANES> o;
#pragma unroll
            for (int i = 0; i < PLANES; ++i)
                o.x[i] = *reinterpret_cast<const u4*>(&d[i * kPlane + (row0 + r) * kRow + 32 * p + 8 * g]);
            return o;
        }
        // Operand of the 16 columns from col0 over the inner rows row0 ...  The
        // transposing read hands 16 lanes a block of 4 rows and 16 columns: lane
        // 4 j + q fetches columns 4 q .. of row j, lane r gets column r.
        __device__ Op<PLANES> cols(int row0, int col0, int r, int g) const {
            using s4 = short __attribute__((ext_vector_type(4)));
            using lds = __attribute__((address_space(3))) s4;
            const std::uint16_t* from = &d[(row0 + 4 * g + r / 4) * kRow + place_of(col0 + 4 * (r % 4))];
            Op<PLANES> o;
#pragma unroll
            for (int i = 0; i < PLANES; ++i) {
                const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(from + i * kPlane)));
                const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(from + i * kPlane + 16 * kRow)));
                o.x[i] = u4{a.x, a.y, b.x, b.y};
            }
            return o;
        }
    };
};

// Float32 inputs in three planes take up to twice the LDS of a tile of float32:
// quicker in the forward of 64 dimensions (128 steps of 128 consoles of 4 heads, by
// float32 instructions 38, by planes 34 us; of 256 consoles 64 and 60) and of 128 (64
// consoles 52 and 44, 256 207 and 178), not of 32 (256 consoles 32 and 51, 512 69 and
// 83); in the gradient they would leave one workgroup a compute unit, or none.
template <typename T, int DP>
struct MathOf {
    using forward = SplitMath<1>;
    using gradient = SplitMath<1>;
};
template <int DP>
struct MathOf<float, DP> {
    using forward = std::conditional_t<DP == 32, F32Math, SplitMath<3>>;
    using gradient = F32Math;
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
// Four such sums at once, that of v[i] in the i-th four of the 16 lanes: as soon
// as half the lanes hold a sum they take another's.
template <int BANKS>
__device__ float taken(float v, float from) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, v), __builtin_bit_cast(int, from), 0xe4, 0xf, BANKS, false));
}
__device__ inline float sum16_of(f4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = v[i];
        v[i] = x + moved<kRowRor + 8>(x);
    }
    float x = taken<0xc>(v[0], v[2]), y = taken<0xc>(v[1], v[3]);
    x += moved<kRowRor + 12>(x);
    y += moved<kRowRor + 4>(y);
    x = taken<0xa>(x, y);
    x += moved<0xb1>(x);           // the other of two, then of two pairs
    return x + moved<0x4e>(x);
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
