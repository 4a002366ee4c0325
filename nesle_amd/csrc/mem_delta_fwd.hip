// The gated delta rule over a rollout, in chunks of 32 tokens.
//
// Inside a chunk, with G the running sum of the gates' logarithms from its
// first token, gamma_i = exp(G_i) and L_ij = exp(G_i - G_j), the tokens'
// writes u are the solution of a unit lower triangular system, and everything
// else is matrix products (S is the state before the chunk):
//   (I + A) U = R,   A_ij = beta_i L_ij (k_i . k_j) for j < i,
//   R = beta (V - gamma K S)
//   O = scale gamma Q S + P U,   P_ij = scale L_ij (q_i . k_j) for j <= i
//   S <- gamma_last S + K^T (gamma_last / gamma) U
//
// One workgroup walks one head of one console; a wave holds 16 columns of the
// state, in registers for the whole rollout, and its 16 columns of R, U and O.
// A result tile is the operand of the next product as it lies in the
// registers (mem_delta_math.h), so only what all columns share goes through
// LDS: K, Q, P and (I + A)^-1.  That inverse is found by substitution:
// neighbouring frames have nearly equal keys, where the powers of A grow to
// thousands and a product form of the inverse cancels.
//
// All products keep float32 precision: the state and the gates' gradients are
// float32 results whatever the inputs' type.
//
// A token that drops the state counts as a gate that lets nothing through: L and
// gamma across it are zero.  A product with a masked zero would still carry NaN,
// so where a key, a value, a gate or (with a drop in the chunk) the state is
// not finite, the chunk is cut before that token and at the drops: nothing of it
// reaches a token it must not.
//
// A chunk takes its state to M S + B, with M [k_dim][k_dim] and B [k_dim][v_dim]
// from its inputs alone.  Few heads over many tokens are cut into segments: one
// launch finds each segment's M and B (the same walk over 2 DP columns, from
// [0 | I], with values for the first half only), one takes the state through
// the segments, one walks all segments from their states at once.
#include <algorithm>

#include "mem_delta_tile.h"

namespace nesle::mem {
namespace {

// Segments of `steps` tokens (a multiple of the chunk length).
struct Segments {
    std::uint32_t steps, count;
    float* maps;           // [segment][head]: M, then B
    float* states;         // [segment][head][k_dim][v_dim]: the state before it
    std::uint32_t* dropped;    // [segment][head]: whether the state is dropped inside
    // Of `per` segments each; one group: all.  The same of the groups.
    std::uint32_t per, groups;
    float *group_maps, *group_states;
    std::uint32_t* group_dropped;
};

// What LDS leaves room for.
template <typename T, int DP>
constexpr int kWavesPerSimd = DP == 32 ? 3 : DP == 64 && sizeof(T) == 2 ? 4 : 2;

// MAP: the segment's M and B; else outputs and states.
//
// Bound by memory where there are many heads: 128 steps of 512 consoles of 4 heads
// of 64 in bfloat16 move 0.30 GB (inputs, outputs, the states in and out and the
// ones kept for the gradient) in 88 us, 3.4 TB/s against a large copy's 4.9.  With
// the parts left out one at a time: kept states -19 us, first and last states -19,
// loads of the inputs -16, outputs -13, the inverse -3.  With one workgroup a compute
// unit a chunk takes 3.6 us, a chain of short parts of which the inverse is 0.4 (64
// consoles 22 us, in float32 28).  A chunk of 32 tokens is one inner step of the bfloat16 instruction
// and the largest whose inverse one wave finds in registers; its tile leaves room
// for four workgroups a compute unit.
template <typename T, int DP, bool WIDE, bool MAP>
__global__ void __launch_bounds__(DP * (MAP ? 8 : 4), (kWavesPerSimd<T, DP>)) delta_forward_kernel(DeltaArgs<T> a, Segments seg) {
    using Tile = ChunkTile<T, typename MathOf<T, DP>::forward, DP>;
    using M = typename Tile::M;
    constexpr int KT = Tile::KT, KP = Tile::KP, kWaves = Tile::kWaves * (MAP ? 2 : 1);
    __shared__ Tile sh;
    const Lane<DP> first;
    const std::uint32_t env = blockIdx.x / a.hv, h = blockIdx.x % a.hv;
    const std::size_t head = blockIdx.x, state_size = static_cast<std::size_t>(a.dk_dim) * a.dv_dim;
    const std::int64_t out_step = static_cast<std::int64_t>(a.batch) * a.hv * a.dv_dim;
    const f4 zero = {0, 0, 0, 0};

    const std::size_t slot = static_cast<std::size_t>(blockIdx.y) * gridDim.x + head;
    const std::uint32_t begin = blockIdx.y * seg.steps;
    const std::uint32_t end = a.steps - begin < seg.steps ? a.steps : begin + seg.steps;

    f4 S[KT];
    if constexpr (MAP) {
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i][j] = first.col - DP == 16 * i + 4 * first.g + j ? 1.0f : 0.0f;
    } else if (seg.count > 1) {
        Tile::load_state(a, seg.states, slot, first, S);
    } else {
        Tile::load_state(a, a.state, head, first, S);
    }
    sh.start(first);
    __syncthreads();

    // Tokens from t0 to the next multiple of the chunk length or the end.
    const auto width = [&](std::uint32_t t0) {
        const std::uint32_t whole = kChunk - t0 % kChunk, left = end - t0;
        return static_cast<int>(whole < left ? whole : left);
    };
    // The inverse takes one wave as long as the rest of its part takes the
    // others: that wave (turn 0) has no tile of A and P, and reads the state
    // first.  The last one stages the next chunk's gates meanwhile.  Other waves
    // each workgroup, as the waves of a compute unit's workgroups share its four
    // SIMDs by their number.
    const int turn = (first.wave + static_cast<int>(blockIdx.x)) % kWaves;
    Ahead<T, DP, WIDE> in;
    bool any_drop = false;
    std::uint32_t odd_gates = 0;
    if (begin < end) {
        in.template fetch<!MAP>(a, begin, width(begin), env, h, first);
        if (turn == kWaves - 1) odd_gates = sh.gates[0].stage(in, width(begin), first.lane);
    }
    int which = 0;
    for (std::uint32_t t0 = begin; t0 < end;) {
        const Lane<DP> at = Lane<DP>::anew();
        const int r = at.r, g = at.g;
        Gates& now = sh.gates[which];
        if (!MAP && t0 != 0 && t0 % kChunk == 0 && a.saved != nullptr)
            Tile::keep(a, a.saved + (t0 / kChunk - 1) * state_size * a.batch * a.hv, head, at, S);
        const std::uint32_t drops = in.drops();
        if (drops & 1u)
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] = zero;
        int n = width(t0);
        const std::uint32_t inside = drops & ~1u;
        any_drop |= drops != 0;
        for (;;) {
            sh.template stage<!MAP>(in, at);
            std::uint32_t odd = in.odd();
            odd |= odd_gates;
            if (inside != 0 && !Tile::finite(S)) odd |= inside;
            sh.report(odd);
            __syncthreads();
            const std::uint32_t bad = __builtin_amdgcn_readfirstlane(sh.bad) & ((n < 32 ? 1u << n : 0u) - 1u);
            if (bad == 0 || n == 1) break;
            // Rare: stage again, up to the first such token or drop, or a first
            // such token alone; what is left is the next turn's.
            n = (bad & 1u) ? 1 : min(n, __ffs(static_cast<int>(bad | inside)) - 1);
            in.cut(n);
            __syncthreads();
            if (at.tid == 0) sh.bad = 0;
            if (turn == kWaves - 1) odd_gates = now.stage(in, n, at.lane);
            __syncthreads();
        }
        const std::uint32_t next = t0 + n;
        if (next < end) in.template fetch<!MAP>(a, next, width(next), env, h, at);
        // K S and Q S for this wave's columns.
        f4 ks[2] = {}, qs[2] = {};
        const auto read_state = [&] {
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                const auto s = M::full(S[2 * i], S[2 * i + 1]);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    ks[m] = M::mul(sh.k.rows(16 * m, i, r, g), s, ks[m]);
                    if constexpr (!MAP) qs[m] = M::mul(sh.q.rows(16 * m, i, r, g), s, qs[m]);
                }
            }
        };
        if (turn == 0 || turn > 3) {
            read_state();
        } else {
            for (int place = turn - 1; place < 3; place += kWaves - 1) {
                f4 kk, qk;
                sh.template products<!MAP>(place, a.scale, now, at, kk, qk);
            }
        }
        __syncthreads();
        if (at.tid == 0) sh.bad = 0;
        if (turn == 0) sh.invert(now, at);
        else if (turn <= 3) read_state();
        which ^= 1;
        if (turn == kWaves - 1 && next < end) odd_gates = sh.gates[which].stage(in, width(next), at.lane);
        f4 R[2], V[2] = {};
        if (!MAP || at.wave < KT) M::values(sh.v.cols(0, 16 * at.wave, r, g), V);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const f4 gam = now.of_rows(now.gamma, m, g);
            R[m] = now.of_rows(now.beta, m, g) * (V[m] - gam * ks[m]);
            qs[m] *= gam * a.scale;
        }
        const auto right = M::full(R[0], R[1]);
        __syncthreads();
        const Rows<T, WIDE> out(a.out + static_cast<std::int64_t>(t0) * out_step + head * a.dv_dim, out_step);
        f4 U[2], O[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) U[m] = M::mul(sh.t.rows(16 * m, 0, r, g), right, zero);
        if constexpr (!MAP) {
            const auto u = M::full(U[0], U[1]);
#pragma unroll
            for (int m = 0; m < 2; ++m) O[m] = M::mul(sh.p.rows(16 * m, 0, r, g), u, qs[m]);
            sh.results.put(out, static_cast<int>(a.dv_dim), n, at, O);
        }
        const float last = now.gamma[kChunk - 1];
        const auto w = M::full(U[0] * now.of_rows(now.decay, 0, g), U[1] * now.of_rows(now.decay, 1, g));
#pragma unroll
        for (int i = 0; i < KT; ++i) S[i] = S[i] * last + M::mul(sh.k.cols(0, 16 * i, r, g), w, zero);
        t0 = next;
        __syncthreads();
        if constexpr (!MAP) sh.results.flush(out, static_cast<int>(a.dv_dim), n, at);
    }
    const Lane<DP> at = Lane<DP>::anew();
    const int rows = static_cast<int>(a.dk_dim), cols = static_cast<int>(a.dv_dim);
    if constexpr (MAP) {
        float* map = seg.maps + slot * a.dk_dim * (a.dk_dim + a.dv_dim);
        if (at.wave < KT) Tile::store_columns(map + a.dk_dim * a.dk_dim, rows, cols, at.col, at.g, S);
        else Tile::store_columns(map, rows, rows, at.col - DP, at.g, S);
        if (at.tid == 0) seg.dropped[slot] = any_drop;
    } else if (end == a.steps) {
        Tile::store_state(a, a.state_out, head, at, S);
    }
}

// From segment to segment, S <- M S + B; a segment that drops the state inside
// leaves B alone, whatever S held.  The steps are a chain, so where there are
// many, the segments go in groups: COMPOSE takes [I | 0] through a group's
// segments to the group's own M and B, a second launch takes the state through
// the groups, a third takes it through the segments of every group at once.
struct Chain {
    const float* maps;             // [segment][head]: M, then B
    const std::uint32_t* dropped;
    const float* first;            // [group][head]: the state before it; null: zeros
    float* to;                     // COMPOSE: the groups' maps; else [segment][head]: the state before it
    std::uint32_t* to_dropped;     // COMPOSE: the groups'
    std::uint32_t count, per;      // segments; of a group
};

// One workgroup for 16 columns, a wave for 16 rows of them: a step is kept short
// (one tile a wave by float32 matrix instructions, the tiles exchanged through
// LDS) and M and B are loaded two to four steps ahead.
template <int DP, bool COMPOSE>
__global__ void __launch_bounds__(DP * 4) delta_join_kernel(Chain x, int dk, int dv) {
    constexpr int KT = DP / 16, kAhead = DP == 128 ? 2 : 4;
    __shared__ f4 tiles[2][KT][64];
    const int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const bool of_m = COMPOSE && blockIdx.y < KT;          // these columns are M's, else the state's
    const int col = 16 * (of_m || !COMPOSE ? blockIdx.y : blockIdx.y - KT) + r, cols = of_m ? dk : dv;
    const std::size_t heads = gridDim.x, head = blockIdx.x, map_size = static_cast<std::size_t>(dk) * (dk + dv);
    const std::uint32_t begin = blockIdx.z * x.per;
    const auto tile = [&](const float* from) {             // rows 16 wave .., of this workgroup's columns
        const Rows<float, false> rows(from, cols);
        f4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = 16 * wave + 4 * g + j;
            v[j] = rows.value_of(rows.get(col < cols && row < dk, row, col));
        }
        return v;
    };
    f4 M[kAhead][KT], B[kAhead];
    std::uint32_t dropped[kAhead];
    const auto load = [&](int slot, std::uint32_t s) {
        const std::size_t at = (begin + s) * heads + head;
        const float* map = x.maps + at * map_size;
        const Rows<float, false> m(map, dk);
#pragma unroll
        for (int c = 0; c < KT; ++c)
            M[slot][c] = m.get4(16 * wave + r < dk && 16 * c + 4 * g < dk, 16 * wave + r, 16 * c + 4 * g);
        B[slot] = of_m ? f4{0, 0, 0, 0} : tile(map + static_cast<std::size_t>(dk) * dk);
        // A vector load, counted in order with the others.
        dropped[slot] = __builtin_amdgcn_raw_buffer_load_b32(
            __builtin_amdgcn_make_buffer_rsrc(const_cast<std::uint32_t*>(x.dropped) + at, 0, 4, 0x00027000), 0, 0, 0);
    };
    f4 S = {0, 0, 0, 0};
    if constexpr (COMPOSE) {
#pragma unroll
        for (int j = 0; j < 4; ++j) S[j] = of_m && col == 16 * wave + 4 * g + j ? 1.0f : 0.0f;
    } else if (x.first != nullptr) {
        S = tile(x.first + (blockIdx.z * heads + head) * dk * dv);
    }
    const auto store = [&](float* to) {
        const Rows<float, false> rows(to, cols);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = 16 * wave + 4 * g + j;
            rows.put(col < cols && row < dk, row, col, S[j]);
        }
    };
    const auto keep = [&](std::uint32_t s) {
        if constexpr (!COMPOSE) store(x.to + ((begin + s) * heads + head) * dk * dv);
    };
    bool any_dropped = false;
    const auto step = [&](int slot) {
        tiles[slot % 2][wave][lane] = S;
        __syncthreads();                                   // two buffers: the next write is a barrier later
        f4 sum = {0, 0, 0, 0};
        if (__builtin_amdgcn_readfirstlane(dropped[slot]) == 0) {
#pragma unroll
            for (int c = 0; c < KT; ++c) sum = mma(M[slot][c], tiles[slot % 2][c][lane], sum);
        } else {
            any_dropped = true;
        }
        S = sum + B[slot];
    };
    // Past the last map its loads are made again: without a condition around
    // them they stay in flight through the steps before they are needed.
    const std::uint32_t left = min(x.per, x.count - begin), steps = COMPOSE ? left : left - 1;
    const std::uint32_t last = steps == 0 ? 0 : steps - 1;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(i, min(static_cast<std::uint32_t>(i), last));
    std::uint32_t s = 0;
    for (; s + kAhead <= steps; s += kAhead)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            keep(s + i);
            step(i);
            load(i, min(s + i + kAhead, last));
        }
#pragma unroll
    for (int i = 0; i < kAhead - 1; ++i)
        if (s + i < steps) {
            keep(s + i);
            step(i);
        }
    if constexpr (COMPOSE) {
        const std::size_t at = blockIdx.z * heads + head;
        store(x.to + at * map_size + (of_m ? 0 : static_cast<std::size_t>(dk) * dk));
        if (threadIdx.x == 0 && blockIdx.y == 0) x.to_dropped[at] = any_dropped;
    } else {
        keep(steps);
    }
}

// Segments for few heads over many tokens.  The walk of one head of 64 through a
// chunk takes 3.6 us by itself and 6 us beside another on its compute unit, a step of
// a chain 0.6 us, a launch of one 5 us and more, and the launches walk every chunk
// twice.  So: as many segments as the card holds workgroups of the maps at once (DP / 8
// waves each, 16 waves a compute unit: 1,024, 512 or 256 of them), four at least to
// make up for the second walk, two chunks or more in each, or four chunks where there
// are only four to seven segments, and no more than balance the chain's steps against
// the walks; in groups, of as many segments as there are groups, once the chain would
// be longer than 40.
// Whole walk against segments, us, bfloat16 / float32 (* where the rule walks whole):
//   32 dimensions, 256 tokens of 128 heads 37 / 39, 27 / 30; 1,024 of 256 heads 137 /
//   143, 89 / 102; 64 dimensions, 256 of 64 heads 32 / 41, 27 / 31; 256 of 128 heads*
//   32 / 41, 38 / 44; 512 of 128 heads 61 / 78, 57 / 69; 1,024 of 256 heads* 127, 157 in
//   bfloat16; 128 dimensions, 256 of 32 heads 46 / 70, 47 / 57; 256 of 64 heads* 48 / 71,
//   58 / 71; 512 of 64 heads 90 / 137, 81 / 105; 1,024 of 128 heads* 174 / 279, 215 / 309.
// One chain against groups, heads of 64 in bfloat16: 4,096 tokens of 8 heads 60 / 63
// us, 8,192 of 8 heads 94 / 79, 32,768 of 4 heads 175 / 121; of 32 and 128 dimensions,
// 16,384 of 4 heads 84 / 55 and 236 / 191.
Segments segments(const nesle_delta_args& a) {
    const std::uint64_t heads = static_cast<std::uint64_t>(a.batch) * a.v_heads;
    const std::uint32_t chunks = (a.steps + kChunk - 1) / kChunk;
    const auto root = [](std::uint64_t x) {
        std::uint32_t n = 1;
        while (static_cast<std::uint64_t>(n + 1) * (n + 1) <= x) ++n;
        return n;
    };
    std::uint32_t count = 1;
    const std::uint64_t at_once = (1u << 15) / padded_dim(a);
    if (4 * heads <= at_once && chunks >= (8 * heads <= at_once ? 8 : 16)) {
        const std::uint32_t most = std::min(static_cast<std::uint32_t>(at_once / heads), chunks / 2);
        count = std::min(root(8ull * chunks), most);
        if (count > 40) count = std::min(root(64ull * chunks), most);
    }
    const std::uint32_t each = count < 2 ? chunks : (chunks + count - 1) / count;
    Segments s{};
    s.steps = each * kChunk;
    s.count = chunks == 0 ? 1 : (chunks + each - 1) / each;
    if (s.steps == 0) s.steps = kChunk;
    s.per = s.count > 40 ? root(s.count) : s.count;
    s.groups = (s.count + s.per - 1) / s.per;
    return s;
}

std::uint64_t segment_floats(const nesle_delta_args& a, const Segments& s) {
    if (s.count < 2) return 0;
    const std::uint64_t slots = (s.count + (s.groups > 1 ? s.groups : 0ull)) * a.batch * a.v_heads;
    return slots * (static_cast<std::uint64_t>(a.k_dim) * (a.k_dim + 2 * a.v_dim) + 1);
}

template <typename T, int DP, bool WIDE>
void launch_dim(const DeltaArgs<T>& a, const Segments& seg, hipStream_t s) {
    const std::uint32_t heads = a.batch * a.hv;
    if (seg.count > 1) {
        // The last segment's M and B are not needed.
        hipLaunchKernelGGL((delta_forward_kernel<T, DP, WIDE, true>), dim3(heads, seg.count - 1), dim3(DP * 8), 0, s, a, seg);
        const int dk = static_cast<int>(a.dk_dim), dv = static_cast<int>(a.dv_dim);
        const std::uint32_t slices = (a.dv_dim + 15) / 16;
        const float* first = a.state;
        if (seg.groups > 1) {                              // of the last group neither
            const Chain in_groups{seg.maps, seg.dropped, nullptr, seg.group_maps, seg.group_dropped, seg.count, seg.per};
            hipLaunchKernelGGL((delta_join_kernel<DP, true>), dim3(heads, DP / 16 + slices, seg.groups - 1), dim3(DP * 4), 0, s,
                               in_groups, dk, dv);
            const Chain of_groups{seg.group_maps, seg.group_dropped, first, seg.group_states, nullptr, seg.groups, seg.groups};
            hipLaunchKernelGGL((delta_join_kernel<DP, false>), dim3(heads, slices), dim3(DP * 4), 0, s, of_groups, dk, dv);
            first = seg.group_states;
        }
        const Chain of_segments{seg.maps, seg.dropped, first, seg.states, nullptr, seg.count, seg.per};
        hipLaunchKernelGGL((delta_join_kernel<DP, false>), dim3(heads, slices, seg.groups), dim3(DP * 4), 0, s, of_segments, dk,
                           dv);
    }
    hipLaunchKernelGGL((delta_forward_kernel<T, DP, WIDE, false>), dim3(heads, seg.count), dim3(DP * 4), 0, s, a, seg);
}

template <typename T>
int forward(const char* who, const nesle_delta_args& x, hipStream_t s) {
    const DeltaArgs<T> a = delta_args<T>(x);
    Segments seg = segments(x);
    if (seg.count > 1) {
        const std::size_t heads = static_cast<std::size_t>(a.batch) * a.hv, slots = seg.count * heads;
        const std::size_t groups = seg.groups > 1 ? seg.groups * heads : 0;
        const std::size_t map_size = static_cast<std::size_t>(a.dk_dim) * (a.dk_dim + a.dv_dim), size = static_cast<std::size_t>(a.dk_dim) * a.dv_dim;
        seg.maps = a.scratch;
        seg.states = seg.maps + slots * map_size;
        seg.group_maps = seg.states + slots * size;
        seg.group_states = seg.group_maps + groups * map_size;
        seg.dropped = reinterpret_cast<std::uint32_t*>(seg.group_states + groups * size);
        seg.group_dropped = seg.dropped + slots;
    }
    const std::uint32_t dim = wide_rows(x) ? 0 : padded_dim(x);
    switch (dim) {
        case 0: launch_dim<T, 128, true>(a, seg, s); break;
        case 32: launch_dim<T, 32, false>(a, seg, s); break;
        case 64: launch_dim<T, 64, false>(a, seg, s); break;
        default: launch_dim<T, 128, false>(a, seg, s); break;
    }
    return launched(who);
}

}  // namespace
}  // namespace nesle::mem

using namespace nesle::mem;

extern "C" {

std::uint64_t nesle_delta_saved_floats(const nesle_delta_args* a) {
    if (a == nullptr || a->steps <= static_cast<std::uint32_t>(kChunk)) return 0;
    const std::uint64_t chunks = (static_cast<std::uint64_t>(a->steps) + kChunk - 1) / kChunk - 1;
    return chunks * a->batch * a->v_heads * a->k_dim * a->v_dim;
}

std::uint64_t nesle_delta_forward_scratch_floats(const nesle_delta_args* a) {
    if (a == nullptr || a->batch == 0 || a->v_heads == 0) return 0;
    return segment_floats(*a, segments(*a));
}

int nesle_delta_forward(const nesle_delta_args* a, void* stream) {
    const char* who = "nesle_delta_forward";
    int rc = check_delta(who, a);
    if (rc != NESLE_OK || a->batch == 0) return rc;
    if (!a->state_out) return refuse(who, "null device pointer");
    if (a->steps != 0) {
        rc = check_delta_inputs(who, a);
        if (rc != NESLE_OK) return rc;
        if (!a->out || (!a->scratch && nesle_delta_forward_scratch_floats(a) != 0)) return refuse(who, "null device pointer");
    }
    const auto s = static_cast<hipStream_t>(stream);
    return a->dtype == NESLE_MEM_F32 ? forward<float>(who, *a, s) : forward<bf16>(who, *a, s);
}

}  // extern "C"
