// mem_decay.h -- what the kernels of linear attention with a decay for each head
// share: their arguments, a chunk's inputs on their way through registers, the
// powers of the decay, and which tokens of a chunk see each other.
#pragma once

#include "mem_delta_tile.h"

namespace nesle::mem {

template <typename T>
struct DecayArgs {
    Heads<T> q, k, v, dout;
    const float* g;
    const std::uint8_t* resets;
    const float* state;
    T* out;
    float *state_out, *saved;
    const float* dstate_out;
    T *dq, *dk, *dv;
    float *dg, *dstate, *scratch;
    std::uint32_t steps, batch, hk, hv, group, dk_dim, dv_dim;     // group: value heads of a key head
    float scale;
};

template <typename T>
DecayArgs<T> decay_args(const nesle_decay_args& a) {
    DecayArgs<T> d{};
    d.q = heads<T>(a.q);
    d.k = heads<T>(a.k);
    d.v = heads<T>(a.v);
    d.dout = heads<T>(a.dout);
    d.g = a.g;
    d.resets = a.resets;
    d.state = a.state;
    d.out = static_cast<T*>(a.out);
    d.state_out = a.state_out;
    d.saved = a.saved;
    d.dstate_out = a.dstate_out;
    d.dq = static_cast<T*>(a.dq);
    d.dk = static_cast<T*>(a.dk);
    d.dv = static_cast<T*>(a.dv);
    d.dg = a.dg;
    d.dstate = a.dstate;
    d.scratch = a.scratch;
    d.steps = a.steps;
    d.batch = a.batch;
    d.hk = a.k_heads;
    d.hv = a.v_heads;
    d.group = a.v_heads / a.k_heads;
    d.dk_dim = a.k_dim;
    d.dv_dim = a.v_dim;
    d.scale = a.scale;
    return d;
}

inline std::uint32_t padded_dim(const nesle_decay_args& a) {
    const std::uint32_t d = a.k_dim > a.v_dim ? a.k_dim : a.v_dim;
    return d <= 32 ? 32 : d <= 64 ? 64 : 128;
}

// Tokens of a chunk of the forward.  What a token costs beside its pairs does not depend
// on it; 64 halves the barriers.  In float32 the pairs' products, made again by every
// wave, weigh more than that: 32.
template <typename T>
constexpr int kDecayChunk = sizeof(T) == 2 ? 64 : 32;
// Tokens between the states that the forward keeps and the gradient takes up: a chunk of
// the gradient, as many as leave room in LDS.  A matter of type and dimension alone:
// strides, which may differ between the two calls (the outputs' gradient has its own),
// have no part in it.
template <typename T, int DP>
constexpr int kDecaySpan = sizeof(T) == 4 && DP == 128 ? 32 : 64;

// f of the dimension that the kernels for these arguments are made for.
template <typename F>
auto at_dim(const nesle_decay_args& a, F&& f) {
    switch (padded_dim(a)) {
        case 32: return f(std::integral_constant<int, 32>());
        case 64: return f(std::integral_constant<int, 64>());
        default: return f(std::integral_constant<int, 128>());
    }
}
inline std::uint32_t decay_span(const nesle_decay_args& a) {
    return at_dim(a, [&](auto dim) -> std::uint32_t {
        return a.dtype == NESLE_MEM_F32 ? kDecaySpan<float, dim()> : kDecaySpan<bf16, dim()>;
    });
}

// Whether 64 rows of any tensor span 2^31 bytes or more, past what a
// 32-bit offset reaches.
inline bool wide_rows(const nesle_decay_args& a) {
    const std::int64_t item = a.dtype == NESLE_MEM_F32 ? 4 : 2, limit = ((1ll << 31) - 4096) / 63;
    for (const nesle_heads* x : {&a.q, &a.k, &a.v, &a.dout})
        if (x->stride_t < 0 || x->stride_t * item >= limit) return true;
    // What the kernels write: of the inputs' type, and shares of key heads' gradients in float32.
    const std::int64_t heads = static_cast<std::int64_t>(a.batch) * a.v_heads;
    return heads * (a.k_dim > a.v_dim ? a.k_dim : a.v_dim) * (a.v_heads > a.k_heads ? 4 : item) >= limit;
}

// Arguments that no call may have.
inline int check_decay(const char* who, const nesle_decay_args* a) {
    if (a == nullptr) return refuse(who, "null arguments");
    if (a->dtype != NESLE_MEM_F32 && a->dtype != NESLE_MEM_BF16) return refuse(who, "dtype must be NESLE_MEM_F32 or NESLE_MEM_BF16");
    for (const std::uint32_t d : {a->k_dim, a->v_dim})
        if (d == 0 || d % 8 != 0 || d > NESLE_DECAY_MAX_DIM)
            return refuse(who, "k_dim and v_dim must be multiples of 8 up to " + std::to_string(NESLE_DECAY_MAX_DIM));
    if (a->k_heads == 0 || a->v_heads == 0 || a->v_heads % a->k_heads != 0)
        return refuse(who, "v_heads must be a multiple of k_heads");
    if (static_cast<std::uint64_t>(a->batch) * a->v_heads > (1u << 22))
        return refuse(who, "batch * v_heads must be at most 4,194,304");
    if (a->steps > (1u << 30)) return refuse(who, "steps must be at most 2^30");
    return NESLE_OK;
}

inline int check_decay_alignment(const char* who, const nesle_decay_args* a) {
    if (!aligned16(a->state) || !aligned16(a->state_out) || !aligned16(a->saved) || !aligned16(a->dstate_out) ||
        !aligned16(a->dstate) || !aligned16(a->scratch) || !aligned16(a->out) || !aligned16(a->dq) || !aligned16(a->dk) ||
        !aligned16(a->dv))
        return refuse(who, "states, outputs and workspaces must lie on 16-byte boundaries");
    return NESLE_OK;
}

// Pointers that a call over at least one token and console needs.
inline int check_decay_inputs(const char* who, const nesle_decay_args* a) {
    if (!a->q.data || !a->k.data || !a->v.data || !a->g) return refuse(who, "null device pointer");
    return NESLE_OK;
}

// ---- a chunk ------------------------------------------------------------------------

// Where a workgroup's lanes stand: DP / 16 waves, one for 16 columns, in each of ROLES
// roles.
template <int DP, int ROLES = 1>
struct Place {
    static constexpr int kRows = 32 * ROLES;       // tokens that the workgroup loads at once
    int tid, lane, r, g, wave, role, col, key_row, key_col;
    // (Unsigned: a signed quotient by a power of two takes four instructions.)
    __device__ explicit Place(unsigned id)
        : tid(static_cast<int>(id & 1023u)), lane(static_cast<int>(id & 63u)), r(static_cast<int>(id & 15u)), g(static_cast<int>(id >> 4 & 3u)) {
        const unsigned of_all = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
        wave = static_cast<int>(of_all % (DP / 16u));
        role = static_cast<int>(of_all / (DP / 16u));
        col = 16 * wave + r;
        key_row = static_cast<int>((id & 1023u) / (DP / 8u));
        key_col = static_cast<int>(8 * (id % (DP / 8u)));
    }
    __device__ Place() : Place(threadIdx.x) {}
    // The same, made anew: what follows from it is worked out, and read from LDS, where it
    // is used, rather than held in registers from an earlier use.
    static __device__ Place anew() {
        unsigned id = threadIdx.x;
        asm volatile("" : "+v"(id));
        return Place(id);
    }
};

// Eight elements of each of a chunk's tokens that a thread loads of one tensor.  A row
// from n on, and a column outside the head, reads as zero.
template <typename T, int DP, int CH, bool WIDE, int ROLES = 1>
struct Piece {
    using In = Rows<T, WIDE>;
    using At = Place<DP, ROLES>;
    static constexpr int kPieces = CH / At::kRows;
    std::uint32_t w[kPieces][In::kWords];
    __device__ void fetch(const Heads<T>& from, std::uint32_t dim, std::uint32_t start, int n, std::uint32_t env,
                          std::uint32_t h, const At& at) {
        const In rows(from.row(start, env, h), from.t);
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            const int row = at.key_row + At::kRows * p;
            rows.get8(row < n && at.key_col < static_cast<int>(dim), row, at.key_col, from.vec, w[p]);
        }
    }
    template <typename Tile>
    __device__ void stage(Tile& to, const At& at) const {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) to.put8(at.key_row + At::kRows * p, at.key_col, w[p]);
    }
    // Zeros in the rows from n on.
    __device__ void cut(int n, const At& at) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p)
#pragma unroll
            for (int i = 0; i < In::kWords; ++i) w[p][i] = at.key_row + At::kRows * p < n ? w[p][i] : 0;
    }
    // And in the rows before n.
    __device__ void cut_before(int n, const At& at) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p)
#pragma unroll
            for (int i = 0; i < In::kWords; ++i) w[p][i] = at.key_row + At::kRows * p >= n ? w[p][i] : 0;
    }
    // Tokens with something that is not finite.
    __device__ std::uint64_t odd(const At& at) const {
        using s2 = unsigned short __attribute__((ext_vector_type(2)));
        std::uint64_t bits = 0;
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            std::uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < In::kWords; ++i)
                if constexpr (sizeof(T) == 4) most = max(most, w[p][i] & 0x7fffffffu);
                else most = __builtin_bit_cast(std::uint32_t, __builtin_elementwise_max(
                                __builtin_bit_cast(s2, most), __builtin_bit_cast(s2, w[p][i] & 0x7fff7fffu)));
            if constexpr (sizeof(T) == 2) most = max(most >> 16, most & 0xffffu);
            if (most >= (sizeof(T) == 4 ? 0x7f800000u : 0x7f80u)) bits |= 1ull << (at.key_row + At::kRows * p);
        }
        return bits;
    }
};

// Ends of episodes among a chunk's tokens, one a lane, fetched ahead: nothing here waits
// for the load before drops().
template <typename T>
struct Resets {
    std::uint32_t mine = 0;
    __device__ void fetch(const DecayArgs<T>& a, std::uint32_t start, int n, std::uint32_t env, int lane) {
        if (a.resets != nullptr) mine = a.resets[(start + static_cast<std::size_t>(min(lane, n - 1))) * a.batch + env];
    }
    // Bit t: the state is dropped before token t of the n.
    __device__ std::uint64_t drops(int n, int lane, bool always) const { return __ballot(lane < n && (always || mine != 0)); }
};

// exp(n g) of a head, n = 0 .. CH: made once by a workgroup.  exp of the rounded
// product is off by |n g| 2^-24 of itself, which is 2^-25 of 1 at most where g <= 0.
template <int CH>
struct Powers {
    // up[i] = a^(i + 1), read[i] = scale a^(i + 1), down[i] = a^(CH - 1 - i), with room
    // past its end.
    alignas(16) float up[CH], read[CH], down[CH + 4];
    __device__ void make(float g, float scale, bool always, int tid) {
        if (tid < CH) {
            up[tid] = always ? 0.0f : expf(static_cast<float>(tid + 1) * g);
            read[tid] = up[tid] * scale;
            down[tid] = tid == CH - 1 ? 1.0f : always ? 0.0f : expf(static_cast<float>(CH - 1 - tid) * g);
        }
        if (tid < 4) down[CH + tid] = 1.0f;
    }
    __device__ float at(int n) const { return down[CH - 1 - n]; }       // a^n, n < CH
};

// Which tokens of a chunk of n see what: `drops` as above, zero nearly always.  Rows from
// n on weigh nothing, by selection: their inputs are zeros, but a decay that grows may
// have infinite powers there, and zero times one is NaN in sums over rows.
struct Seen {
    std::uint64_t drops;
    int n, first, last;        // tokens; the first and the last that drop the state (n, 0: none)
    __device__ Seen(std::uint64_t d, int count) : drops(d), n(count), first(count), last(0) {
        if (d != 0) {
            first = __ffsll(static_cast<long long>(d)) - 1;
            last = 63 - __clzll(static_cast<long long>(d));
        }
    }
    // Episodes that ended up to token i: two tokens see each other where these agree.
    __device__ int episode(int i) const { return __popcll(drops & (~0ull >> (63 - i))); }
    // Of the four rows from `row` on: the decay from before the chunk times the scale, and
    // the decay to its end.
    template <int CH>
    __device__ f4 in(const Powers<CH>& p, int row) const {
        f4 v = *reinterpret_cast<const f4*>(p.read + row);
        if (first < CH)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = row + e < first ? v[e] : 0.0f;
        return v;
    }
    template <int CH>
    __device__ f4 out(const Powers<CH>& p, int row) const {
        f4 v;
        if (n == CH) v = *reinterpret_cast<const f4*>(p.down + row);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = p.down[min(row + e + CH - n, CH)];
        if (drops != 0)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = row + e >= last ? v[e] : 0.0f;
        return v;
    }
    template <int CH>
    __device__ float whole(const Powers<CH>& p) const { return drops != 0 ? 0.0f : p.up[n - 1]; }
};

// a^(i - j) for tiles of 16x16 pairs of tokens, of the lane's four elements.
// LATER_ROWS: a tile's rows are the later tokens i = 16 it + 4 g + e and its columns
// the earlier j = 16 jt + r; else rows are j and columns i.  With s = 4 g + e - r, or
// r - 4 g - e, the power is a^(16 (it - jt) + s), which is a^(15 + s) times
// a^(16 (it - jt) - 15): both exponents are zero or more below the diagonal, where
// s may be negative.
template <int CH, bool LATER_ROWS>
struct PairPowers {
    static constexpr int kFar = CH / 16 - 1;
    f4 same, base;
    float far[kFar];
    __device__ void make(const Powers<CH>& p, float scale, int r, int g) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int s = LATER_ROWS ? 4 * g + e - r : r - 4 * g - e;
            same[e] = s < 0 ? 0.0f : p.at(s) * scale;
            base[e] = p.at(15 + s) * scale;
        }
#pragma unroll
        for (int d = 0; d < kFar; ++d) far[d] = p.at(16 * d + 1);
    }
    // Of a tile d = it - jt below the diagonal.
    __device__ f4 of(int d) const { return d == 0 ? same : base * far[d - 1]; }
    // x times its weights; zero, by selection, where the pair does not see each other.
    // `episodes`: Seen::episode of the chunk's tokens, in LDS.
    __device__ f4 weigh(f4 x, int it, int jt, const Seen& seen, const int* episodes, int r, int g) const {
        x *= of(it - jt);
        if (it == jt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (LATER_ROWS ? 4 * g + e < r : r < 4 * g + e) x[e] = 0.0f;
        if (LATER_ROWS && seen.n < CH)     // (else such a row is a column, which is not written)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = 16 * it + 4 * g + e < seen.n ? x[e] : 0.0f;
        if (seen.drops != 0) {
            using i4 = int __attribute__((ext_vector_type(4)));
            const i4 rows = *reinterpret_cast<const i4*>(episodes + 16 * (LATER_ROWS ? it : jt) + 4 * g);
            const int col = episodes[16 * (LATER_ROWS ? jt : it) + r];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = rows[e] == col ? x[e] : 0.0f;
        }
        return x;
    }
};

// Results [tokens][dim] of the inputs' type, a wave's 16 columns at a time: float32
// from the registers, 64 bytes of a row together.
template <typename T, int DP, int CH, int ROLES = 1>
struct DecayResults {
    using At = Place<DP, ROLES>;
    // A finished tile, as it waits for its place.
    using Tile = f4;
    static __device__ Tile tile(f4 x) { return x; }
    template <bool WIDE>
    static __device__ void put_tile(const Rows<T, WIDE>& to, int dim, int n, const At& at, int m, f4 x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = 16 * m + 4 * at.g + e;
            to.put(at.col < dim && row < n, row, at.col, x[e]);
        }
    }
    template <bool WIDE>
    __device__ void put(const Rows<T, WIDE>& to, int dim, int n, const At& at, const Tile (&x)[CH / 16]) {
#pragma unroll
        for (int m = 0; m < CH / 16; ++m) put_tile(to, dim, n, at, m, x[m]);
    }
    template <bool WIDE>
    __device__ void flush(const Rows<T, WIDE>&, int, int, const At&) const {}
};
// bfloat16: two bytes a lane would be 32 of a row, so through LDS ([column][token])
// and, after a barrier, eight elements of a token a lane by transposing reads: a
// wave's block is 16 tokens of 32 columns.
template <int DP, int CH, int ROLES>
struct DecayResults<bf16, DP, CH, ROLES> {
    using At = Place<DP, ROLES>;
    static constexpr int kRow = CH + 8;
    alignas(16) std::uint16_t d[DP * kRow];
    using Tile = u2;
    static __device__ Tile tile(f4 x) { return u2{pack_bf16(x.x, x.y), pack_bf16(x.z, x.w)}; }
    template <bool WIDE>
    __device__ void put(const Rows<bf16, WIDE>&, int, int, const At& at, const Tile (&x)[CH / 16]) {
#pragma unroll
        for (int m = 0; m < CH / 16; ++m) *reinterpret_cast<u2*>(&d[at.col * kRow + 16 * m + 4 * at.g]) = x[m];
    }
    template <bool WIDE>
    __device__ void flush(const Rows<bf16, WIDE>& to, int dim, int n, const At& at) const {
        using s4 = short __attribute__((ext_vector_type(4)));
        using lds = __attribute__((address_space(3))) s4;
#pragma unroll
        for (int p = at.role; p < CH / 32; p += ROLES) {
            const int token = 32 * p + 16 * (at.wave % 2), col = 32 * (at.wave / 2) + 8 * at.g;
            const std::uint16_t* from = &d[(col + at.r / 4) * kRow + token + 4 * (at.r % 4)];
            const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)from));
            const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(from + 4 * kRow)));
            to.put8(token + at.r < n && col < dim, token + at.r, col, u4{a.x, a.y, b.x, b.y});
        }
    }
};

// ---- a wave's slab of a state -----------------------------------------------------
// Four consecutive float32 along a row of [k_dim][v_dim] a lane: tile i holds
// C[x = value 16 i + 4 g + e][y = key 16 wave + r].
template <int DP, typename At>
__device__ void load_key_slab(const float* from, int dk, int dv, const At& at, f4 (&S)[DP / 16]) {
    const Rows<float, false> x(from, dv);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
        S[i] = from == nullptr ? f4{0, 0, 0, 0} : x.get4(at.col < dk && 16 * i + 4 * at.g < dv, at.col, 16 * i + 4 * at.g);
}
template <int DP, typename At>
__device__ void store_key_slab(float* to, int dk, int dv, const At& at, const f4 (&S)[DP / 16]) {
    const Rows<float, false> x(to, dv);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) x.put4(at.col < dk && 16 * i + 4 * at.g < dv, at.col, 16 * i + 4 * at.g, S[i]);
}
// Tile i holds C[x = key 16 i + 4 g + e][y = value 16 wave + r].
template <int DP, typename At>
__device__ void load_value_slab(const float* from, int dk, int dv, const At& at, f4 (&S)[DP / 16]) {
    const Rows<float, false> x(from, dv);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = 16 * i + 4 * at.g + e;
            S[i][e] = from == nullptr ? 0.0f : x.value_of(x.get(at.col < dv && row < dk, row, at.col));
        }
}
template <int DP, typename At>
__device__ void store_value_slab(float* to, int dk, int dv, const At& at, const f4 (&S)[DP / 16]) {
    const Rows<float, false> x(to, dv);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = 16 * i + 4 * at.g + e;
            x.put(at.col < dv && row < dk, row, at.col, S[i][e]);
        }
}

// Kinds of products (mem_delta_math.h).  Float32 inputs in three planes take a third of the
// matrix instructions' time, and half as much LDS again and the cutting.  By float32
// instructions / by planes, us of 128 steps of 64 (512) consoles of 4 heads: forward of 32
// dimensions 15 / 16 (37 / 43), of 64 23 / 25 (108 / 116), of 128 52 / 42 (256 consoles 178 /
// 172); gradient of 32 23 / 23 (105 / 110), of 64 38 / 34 (299 / 274), of 128 96 / 88 (399 / 385).
template <typename T, int DP>
struct DecayMathOf {
    using forward = SplitMath<1>;
    using gradient = SplitMath<1>;
};
template <int DP>
struct DecayMathOf<float, DP> {
    using forward = std::conditional_t<DP == 128, SplitMath<3>, F32Math>;
    using gradient = std::conditional_t<DP == 32, F32Math, SplitMath<3>>;
};

}  // namespace nesle::mem
