// mem_delta_tile.h -- one chunk of the gated delta rule: its inputs on their
// way through registers, and the tiles in LDS that the forward and the
// gradient kernels both make of it.
#pragma once

#include "mem_delta_math.h"

namespace nesle::mem {

// ---- strided rows of a chunk ------------------------------------------------------
// Rows start .. start + 31 of a tensor whose row 0 is at `base`.  Loads go
// through a buffer descriptor: one scalar base, 32-bit offsets, and an offset
// past its range, which a row or column outside the tensor is given, reads as
// zero and is not written.  WIDE: rows may lie 2^31 bytes apart, 64-bit
// addresses.
constexpr std::uint32_t kOutside = 0x80000000u, kRange = 0x7fffffffu;

template <typename T, bool WIDE>
struct Rows {
    T* base;
    std::int64_t step;          // elements from row to row
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ Rows(const T* b, std::int64_t s) : base(const_cast<T*>(b)), step(s) {
        if constexpr (!WIDE) rsrc = __builtin_amdgcn_make_buffer_rsrc(base, 0, static_cast<int>(kRange), 0x00027000);
    }
    __device__ std::uint32_t offset(bool in, int row, int col) const {
        return in ? static_cast<std::uint32_t>(row * static_cast<int>(step) + col) * sizeof(T) : kOutside;
    }
    // An element's bits, upper half of the word for two-byte types once
    // value_of() has it: nothing here waits for the load.
    __device__ std::uint32_t get(bool in, int row, int col) const {
        if constexpr (WIDE) {
            if (!in) return 0u;
            if constexpr (sizeof(T) == 4) return __builtin_bit_cast(std::uint32_t, base[row * step + col]);
            else if constexpr (sizeof(T) == 2) return __builtin_bit_cast(std::uint16_t, base[row * step + col]);
            else return base[row * step + col];
        }
        const int at = static_cast<int>(offset(in, row, col));
        if constexpr (sizeof(T) == 4) return __builtin_amdgcn_raw_buffer_load_b32(rsrc, at, 0, 0);
        else if constexpr (sizeof(T) == 1) return static_cast<std::uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(rsrc, at, 0, 0));
        else return static_cast<std::uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(rsrc, at, 0, 0));
    }
    // At a byte offset already made, plus a scalar one (from 0 to kRange, so
    // that an offset outside stays outside).
    __device__ void put_at(std::uint32_t at, std::uint32_t plus, float x) const {
        const int v = static_cast<int>(at), s = static_cast<int>(plus);
        if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, static_cast<T>(x)), rsrc, v, s, 0);
        else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, static_cast<T>(x)), rsrc, v, s, 0);
    }
    static __device__ float value_of(std::uint32_t bits) {
        return __builtin_bit_cast(float, sizeof(T) == 4 ? bits : bits << 16);
    }
    __device__ void put(bool in, int row, int col, float v) const {
        const T x = static_cast<T>(v);
        if constexpr (WIDE) {
            if (in) base[row * step + col] = x;
        } else {
            const int at = static_cast<int>(offset(in, row, col));
            if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, x), rsrc, at, 0, 0);
            else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, x), rsrc, at, 0, 0);
        }
    }
    // Four consecutive float32 elements on a 16-byte boundary.
    __device__ f4 get4(bool in, int row, int col) const {
        static_assert(sizeof(T) == 4 && !WIDE);
        const auto x = __builtin_amdgcn_raw_buffer_load_b128(rsrc, static_cast<int>(offset(in, row, col)), 0, 0);
        return __builtin_bit_cast(f4, x);
    }
    __device__ void put4(bool in, int row, int col, f4 v) const {
        static_assert(sizeof(T) == 4 && !WIDE);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), rsrc, static_cast<int>(offset(in, row, col)), 0, 0);
    }
    // Eight consecutive bfloat16 on a 16-byte boundary.
    __device__ void put8(bool in, int row, int col, u4 v) const {
        static_assert(sizeof(T) == 2);
        if constexpr (WIDE) {
            if (in) *reinterpret_cast<u4*>(base + row * step + col) = v;
        } else {
            __builtin_amdgcn_raw_buffer_store_b128(v, rsrc, static_cast<int>(offset(in, row, col)), 0, 0);
        }
    }
    // Eight consecutive elements, as they lie in memory.
    static constexpr int kWords = sizeof(T) * 8 / 4;
    __device__ void get8(bool in, int row, int col, bool vec, std::uint32_t (&w)[kWords]) const {
        if (!vec || WIDE) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const std::uint32_t x = get(in, row, col + i);
                if constexpr (sizeof(T) == 4) w[i] = x;
                else if (i % 2 == 0) w[i / 2] = x;
                else w[i / 2] |= x << 16;
            }
            return;
        }
        const int at = static_cast<int>(offset(in, row, col));
#pragma unroll
        for (int i = 0; i < 2; ++i) {          // four elements at a time: their alignment is what `vec` says
            if constexpr (sizeof(T) == 4) {
                const auto x = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at + 16 * i, 0, 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[4 * i + j] = x[j];
            } else {
                const auto x = __builtin_amdgcn_raw_buffer_load_b64(rsrc, at + 8 * i, 0, 0);
                w[2 * i] = x[0];
                w[2 * i + 1] = x[1];
            }
        }
    }
};

// Where a workgroup's lanes stand.
template <int DP>
struct Lane {
    int tid, lane, r, g, wave, col, key_row, key_col;
    __device__ explicit Lane(int id)
        : tid(id), lane(tid % 64), r(lane % 16), g(lane / 16), wave(__builtin_amdgcn_readfirstlane(threadIdx.x / 64)),
          col(16 * wave + r), key_row(tid / (DP / 8)), key_col(8 * (tid % (DP / 8))) {}
    __device__ Lane() : Lane(static_cast<int>(threadIdx.x)) {}
    // The same, made anew: addresses that follow from it are worked out where
    // they are used, rather than all held in registers through a loop.
    static __device__ Lane anew() {
        int id = static_cast<int>(threadIdx.x);
        asm volatile("" : "+v"(id));
        return Lane(id);
    }
    // Token row e = 0..7 of a wave's columns.
    __device__ int row(int e) const { return 16 * (e / 4) + 4 * g + e % 4; }
};

// The inputs of the tokens [start, start + width) of a chunk, loaded into
// registers ahead of their use: a thread has eight elements of one token's key,
// query and value, every wave the gates, one token a lane.
template <typename T, int DP, bool WIDE>
struct Ahead {
    using In = Rows<T, WIDE>;
    std::uint32_t k[In::kWords], q[In::kWords], v[In::kWords], g, beta, reset;

    static __device__ void part(const Heads<T>& from, std::uint32_t dim, std::uint32_t start, int width, std::uint32_t env,
                                std::uint32_t h, const Lane<DP>& at, std::uint32_t (&to)[In::kWords]) {
        const bool in = at.key_row < width && at.key_col < static_cast<int>(dim);
        In(from.row(start, env, h), from.t).get8(in, at.key_row, at.key_col, from.vec, to);
    }
    template <bool QUERIES = true>
    __device__ void fetch(const DeltaArgs<T>& x, std::uint32_t start, int width, std::uint32_t env, std::uint32_t h,
                          const Lane<DP>& at) {
        part(x.k, x.dk_dim, start, width, env, h / x.group, at, k);
        if constexpr (QUERIES) part(x.q, x.dk_dim, start, width, env, h / x.group, at, q);
        part(x.v, x.dv_dim, start, width, env, h, at, v);
        const std::size_t token = static_cast<std::size_t>(start) * x.batch + env;
        const bool mine = at.lane < width;
        const Rows<float, WIDE> gates(x.g + token * x.hv + h, static_cast<std::int64_t>(x.batch) * x.hv);
        const Rows<float, WIDE> betas(x.beta + token * x.hv + h, static_cast<std::int64_t>(x.batch) * x.hv);
        g = gates.get(mine, at.lane, 0);
        beta = betas.get(mine, at.lane, 0);
        reset = 0;
        if (x.resets != nullptr) reset = Rows<std::uint8_t, WIDE>(x.resets + token, x.batch).get(mine, at.lane, 0);
    }
    // Zeros in the rows from n on.
    __device__ void cut(int n) {
        const bool mine = Lane<DP>::anew().key_row < n;
#pragma unroll
        for (int i = 0; i < In::kWords; ++i) {
            k[i] = mine ? k[i] : 0;
            q[i] = mine ? q[i] : 0;
            v[i] = mine ? v[i] : 0;
        }
    }
    // Tokens whose key or value holds something that is not finite.
    __device__ std::uint32_t odd() const {
        using s2 = unsigned short __attribute__((ext_vector_type(2)));
        std::uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < In::kWords; ++i)
#pragma unroll
            for (const std::uint32_t w : {k[i], v[i]})
                if constexpr (sizeof(T) == 4) most = max(most, w & 0x7fffffffu);
                else most = __builtin_bit_cast(std::uint32_t, __builtin_elementwise_max(
                                __builtin_bit_cast(s2, most), __builtin_bit_cast(s2, w & 0x7fff7fffu)));
        if constexpr (sizeof(T) == 2) most = max(most >> 16, most & 0xffffu);
        const bool bad = most >= (sizeof(T) == 4 ? 0x7f800000u : 0x7f80u);
        if (!__any(bad)) return 0;
        return bad ? 1u << Lane<DP>::anew().key_row : 0;
    }
    static __device__ float value(std::uint32_t bits) { return __builtin_bit_cast(float, bits); }
    __device__ bool drop() const { return reset != 0 || value(g) < kDropBelow; }
    // Bit t: the state is dropped before token start + t.
    __device__ std::uint32_t drops() const { return static_cast<std::uint32_t>(__ballot(drop())); }
};

// ---- results [tokens][dim] of the inputs' type, a wave's 16 columns at a time ----
// Float32: from the registers, 64 bytes of a row together.
template <typename T, int DP>
struct Results {
    template <bool WIDE>
    __device__ void put(const Rows<T, WIDE>& to, int dim, int n, const Lane<DP>& at, const f4 (&x)[2]) {
        const bool in = at.col < dim;
        if (!WIDE && n == kChunk) {
            const std::uint32_t base = to.offset(in, 4 * at.g, at.col);
#pragma unroll
            for (int e = 0; e < 8; ++e) to.put_at(base, (16 * (e / 4) + e % 4) * static_cast<std::uint32_t>(to.step) * sizeof(T), x[e / 4][e % 4]);
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) to.put(in && at.row(e) < n, at.row(e), at.col, x[e / 4][e % 4]);
    }
    template <bool WIDE>
    __device__ void flush(const Rows<T, WIDE>&, int, int, const Lane<DP>&) const {}
};
// bfloat16: two bytes a lane would be 32 of a row, so through LDS ([column]
// [token], rows of 18 words: no bank twice) and, after a barrier, eight elements
// of a token a lane by transposing reads: a wave's block is 16 tokens of 32
// columns.
template <int DP>
struct Results<bf16, DP> {
    static constexpr int kRow = kChunk + 4;
    alignas(16) std::uint16_t d[DP * kRow];
    template <bool WIDE>
    __device__ void put(const Rows<bf16, WIDE>&, int, int, const Lane<DP>& at, const f4 (&x)[2]) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
            *reinterpret_cast<u2*>(&d[at.col * kRow + 16 * m + 4 * at.g]) = u2{pack_bf16(x[m].x, x[m].y), pack_bf16(x[m].z, x[m].w)};
    }
    template <bool WIDE>
    __device__ void flush(const Rows<bf16, WIDE>& to, int dim, int n, const Lane<DP>& at) const {
        using s4 = short __attribute__((ext_vector_type(4)));
        using lds = __attribute__((address_space(3))) s4;
        const int token = 16 * (at.wave % 2), col = 32 * (at.wave / 2) + 8 * at.g;
        const std::uint16_t* from = &d[(col + at.r / 4) * kRow + token + 4 * (at.r % 4)];
        const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)from));
        const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(from + 4 * kRow)));
        to.put8(token + at.r < n && col < dim, token + at.r, col, u4{a.x, a.y, b.x, b.y});
    }
};

// What a chunk's gates come to: two of these, one staged while the other is used.
struct Gates {
    alignas(16) double G[kChunk];              // running sum of g: differences of it are taken
    alignas(16) float gamma[kChunk], decay[kChunk], beta[kChunk];

    // Of the tokens below n (one wave); other rows neither decay nor write.
    // Returns the bits of tokens whose gate or write strength is not finite.
    template <typename T, int DP, bool WIDE>
    __device__ std::uint32_t stage(const Ahead<T, DP, WIDE>& in, int n, int lane) {
        const bool use = lane < n;
        const float g = !use ? 0.0f : in.drop() ? kGone : in.value(in.g), b = use ? in.value(in.beta) : 0.0f;
        double sum = g;
#pragma unroll
        for (int d = 1; d < kChunk; d *= 2) {
            const double below = __shfl_up(sum, d);
            if (lane >= d) sum += below;
        }
        const double end = __shfl(sum, kChunk - 1);
        if (lane < kChunk) {
            G[lane] = sum;
            gamma[lane] = expf(static_cast<float>(sum));
            decay[lane] = expf(static_cast<float>(end - sum));
            beta[lane] = b;
        }
        return fabsf(b) < INFINITY && g < INFINITY ? 0u : 1u << lane;
    }
    // Of a wave's token rows.
    static __device__ f4 of_rows(const float* x, int m, int g) { return *reinterpret_cast<const f4*>(x + 16 * m + 4 * g); }
    // L_ij.  exp2 of the rounded product is off by |x| 2^-24 of itself, which
    // is 2^-25 of 1 at most where L <= 1.
    __device__ float ratio(int i, int j) const {
        return __builtin_amdgcn_exp2f(static_cast<float>(G[i] - G[j]) * 1.44269504f);
    }
};

// Math: the kind of products.  DP: head dimensions padded to 32, 64 or 128; DP / 16 waves.
// Later: what takes the place of the values, A and the results afterwards.
template <typename T, typename Math, int DP, typename Later = char>
struct ChunkTile {
    using M = Math;
    static constexpr int KT = DP / 16, KP = DP / 32, kWaves = DP / 16, kSmall = kChunk + 4;

    typename M::template Tile<kChunk, DP, M::kIn, 8> k, q;
    typename M::template Tile<kChunk, kChunk, kFull, 8> p;     // P: scale L_ij (q_i . k_j), j <= i; else 0
    typename M::template Tile<kChunk, kChunk, kFull, 8> t;     // (I + A)^-1
    union {
        struct {
            typename M::template Tile<kChunk, DP, M::kIn, 8> v;
            union {
                alignas(16) float a[kChunk * kSmall];  // A without beta: L_ij (k_i . k_j), j < i; else 0
                Results<T, DP> results;                // of the values, once A is inverted
            };
        };
        Later later;
    };
    Gates gates[2];
    unsigned bad;                              // tokens with a value that is not finite

    // ---- matrices [k_dim][cols] beside a head's keys (its state and its
    // transition): lane (r, g) of a wave holds rows 16 i + 4 g + j of one column ----
    static __device__ void load_columns(const float* from, int rows, int cols, int col, int g, f4 (&S)[KT]) {
        if (from == nullptr) {
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] = f4{0, 0, 0, 0};
            return;
        }
        const Rows<float, false> x(from, cols);
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = 16 * i + 4 * g + j;
                S[i][j] = x.value_of(x.get(col < cols && row < rows, row, col));
            }
    }
    static __device__ void store_columns(float* to, int rows, int cols, int col, int g, const f4 (&S)[KT]) {
        const Rows<float, false> x(to, cols);
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = 16 * i + 4 * g + j;
                x.put(col < cols && row < rows, row, col, S[i][j]);
            }
    }
    static __device__ void load_state(const DeltaArgs<T>& a, const float* from, std::size_t head, const Lane<DP>& at,
                                      f4 (&S)[KT]) {
        if (from != nullptr) from += head * a.dk_dim * a.dv_dim;
        load_columns(from, static_cast<int>(a.dk_dim), static_cast<int>(a.dv_dim), at.col, at.g, S);
    }
    static __device__ void store_state(const DeltaArgs<T>& a, float* to, std::size_t head, const Lane<DP>& at,
                                       const f4 (&S)[KT]) {
        store_columns(to + head * a.dk_dim * a.dv_dim, static_cast<int>(a.dk_dim), static_cast<int>(a.dv_dim), at.col, at.g, S);
    }

    // A state before a chunk, kept for the gradient as [v_dim][k_dim]: the four
    // rows a lane holds lie together.
    static __device__ void keep(const DeltaArgs<T>& a, float* to, std::size_t head, const Lane<DP>& at, const f4 (&S)[KT]) {
        const Rows<float, false> x(to + head * a.dk_dim * a.dv_dim, a.dk_dim);
#pragma unroll
        for (int i = 0; i < KT; ++i)
            x.put4(at.col < static_cast<int>(a.dv_dim) && 16 * i + 4 * at.g < static_cast<int>(a.dk_dim), at.col, 16 * i + 4 * at.g, S[i]);
    }
    static __device__ void kept(const DeltaArgs<T>& a, const float* from, std::size_t head, const Lane<DP>& at, f4 (&S)[KT]) {
        const Rows<float, false> x(from + head * a.dk_dim * a.dv_dim, a.dk_dim);
#pragma unroll
        for (int i = 0; i < KT; ++i)
            S[i] = x.get4(at.col < static_cast<int>(a.dv_dim) && 16 * i + 4 * at.g < static_cast<int>(a.dk_dim), at.col, 16 * i + 4 * at.g);
    }

    static __device__ bool finite(const f4 (&S)[KT]) {
        f4 none = {0, 0, 0, 0};
        asm volatile("" : "+v"(none));         // here, not ahead of the condition around the call
#pragma unroll
        for (int i = 0; i < KT; ++i) none += S[i] - S[i];      // 0, or NaN
        return none.x + none.y + none.z + none.w == 0.0f;
    }

    // The tiles' blocks above the diagonal, once.
    __device__ void start(const Lane<DP>& at) {
        if (at.tid == 0) bad = 0;
        if (at.tid < 64)
            for (int i = 0; i < 4; ++i) {
                p.put(at.r, 16 + 4 * at.g + i, 0.0f);
                t.put(at.r, 16 + 4 * at.g + i, 0.0f);
            }
    }

    template <bool QUERIES = true, bool WIDE>
    __device__ void stage(const Ahead<T, DP, WIDE>& in, const Lane<DP>& at) {
        if (!QUERIES && at.key_row >= kChunk) return;          // more waves than the tiles need
        k.put8(at.key_row, at.key_col, in.k);
        if constexpr (QUERIES) q.put8(at.key_row, at.key_col, in.q);
        v.put8(at.key_row, at.key_col, in.v);
    }

    // Tokens with something that is not finite, from all waves.
    __device__ void report(std::uint32_t bits) {
        if (__any(bits != 0)) atomicOr(&bad, bits);
    }

    // A tile of 16x16 token pairs on or below the diagonal: place 0, 1, 2 starts
    // at (0, 0), (16, 0), (16, 16).  `each(row, col, i, L_ij)` for the lane's four.
    static __device__ int first_row(int place) { return place != 0 ? 16 : 0; }
    static __device__ int first_col(int place) { return place == 2 ? 16 : 0; }

    // k_i . k_j and q_i . k_j of a tile, times L_ij and zero where j is not
    // before (not after) i; into A and P.
    template <bool QUERIES = true>
    __device__ void products(int place, float scale, const Gates& now, const Lane<DP>& at, f4& kk, f4& qk) {
        const int mi = first_row(place), nj = first_col(place);
        kk = qk = f4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const auto right = k.rows(nj, i, at.r, at.g);
            kk = M::mul(k.rows(mi, i, at.r, at.g), right, kk);
            if constexpr (QUERIES) qk = M::mul(q.rows(mi, i, at.r, at.g), right, qk);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = mi + 4 * at.g + i, col = nj + at.r;
            const float L = now.ratio(row, col);
            kk[i] = col < row ? kk[i] * L : 0.0f;
            qk[i] = col <= row ? qk[i] * L * scale : 0.0f;
            a[row * kSmall + col] = kk[i];
            if constexpr (QUERIES) p.put(row, col, qk[i]);
        }
    }

    // (I + A)^-1 into t (one wave).  The two diagonal tiles by substitution,
    // tile b in the lanes of rows b and b + 2 of 16, a column a lane: once an
    // entry is known it is taken out of all below, and the lane of row m hands
    // its A[m][i] to the others.  The block below the diagonal is
    // -T1 (A10 T0), its factors read from where A's diagonal tiles were.
    __device__ void invert(const Gates& now, const Lane<DP>& at) {
        const int b = at.g % 2, r = at.r, g = at.g;
        float x[16], row[16];
        const float* from = &a[(16 * b + r) * kSmall + 16 * b];
        const float less = -now.beta[16 * b + r];
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const f4 w = *reinterpret_cast<const f4*>(from + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                row[i + j] = w[j] * less;
                x[i + j] = i + j == r ? 1.0f : 0.0f;
            }
        }
        // Two wait states between a register's write and its read by another
        // lane, which the compiler does not see in the lines it reads below.
#pragma unroll
        for (int i = 0; i < 16; i += 4) asm volatile("s_nop 1" : "+v"(row[i]), "+v"(row[i + 1]), "+v"(row[i + 2]), "+v"(row[i + 3]));
        substitute(std::make_integer_sequence<int, 15>{}, row, x);
        if (g < 2)
#pragma unroll
            for (int i = 0; i < 16; ++i) a[(16 * b + i) * kSmall + 16 * b + r] = x[i];
        __builtin_amdgcn_wave_barrier();       // in order within the wave
        const f4 zero = {0, 0, 0, 0};
        const f4 t0 = down<kSmall>(a, 0, 0, r, g), t1 = down<kSmall>(a, 16, 16, r, g);
        const f4 w = mma(along<kSmall>(a, 16, 0, r, g) * now.beta[16 + r], t0, zero);
        const f4 below = mma(along<kSmall>(a, 16, 16, r, g), w, zero);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            t.put(4 * g + i, r, t0[i]);
            t.put(16 + 4 * g + i, 16 + r, t1[i]);
            t.put(16 + 4 * g + i, r, -below[i]);
        }
    }
    // x += (row, in lane M of each 16) y.
    template <int M1>
    static __device__ void take_out_one(float& x, float row, float y) {
        asm("v_fmac_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf" : "+v"(x) : "v"(row), "v"(y), "n"(M1));
    }
    template <int I, int... D>
    static __device__ void take_out(std::integer_sequence<int, D...>, const float (&row)[16], float (&x)[16]) {
        (take_out_one<I + 1 + D>(x[I + 1 + D], row[I], x[I]), ...);
    }
    template <int... I>
    static __device__ void substitute(std::integer_sequence<int, I...>, const float (&row)[16], float (&x)[16]) {
        (take_out<I>(std::make_integer_sequence<int, 15 - I>{}, row, x), ...);
    }
};

}  // namespace nesle::mem
