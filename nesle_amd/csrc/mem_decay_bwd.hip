// Gradient of linear attention with a decay for each head over a rollout
// (mem_decay_fwd.hip has the forward's formulas).  Chunks are taken last to first
// from the states before them, which the forward kept.  With dO the outputs'
// gradient, dS the gradient of the state after a chunk of n tokens, and i, j
// counted from its first one:
//   P_ij = scale a^(i - j) (q_i . k_j),  R_ij = scale a^(i - j) (do_i . v_j),  j <= i
//   dQ = scale a^(i + 1) dO S^T + R K
//   dK = a^(n - 1 - j) V dS^T + R^T Q
//   dV = a^(n - 1 - j) K dS + P^T dO
//   dS before = a^n dS + scale Q^T a^(i + 1) dO
// A head's decay counts once for every token that a value crosses on its way from
// the token that wrote it to the one that read it, so its gradient is the sum of
// the ways times their lengths within the chunk:
//   dg += sum (i - j) P_ij (do_i . v_j) + sum (i + 1) q_i . (scale a^(i + 1) dO S^T)_i
//       + sum (n - 1 - j) k_j . (a^(n - 1 - j) V dS^T)_j + n a^n <dS, S>
// (nothing here is a difference of sums: row sums less column sums weighed by the
// tokens' places would be equal, but cancel).
//
// One workgroup walks one head of one console, a wave for 16 columns of each of dQ,
// dK and dV, or two waves: one has dQ and the pairs, the other dK, dV and dS.  dS is
// needed by key columns (dK) and by value columns (dV): a wave holds both slabs of it in
// registers and updates both, which costs a product more and saves passing it through
// LDS.
//
// Inputs come and results go a chunk at a time, and the forward kept one state a
// chunk; inside, the work goes in parts of 32 tokens, last to first, as pairs of
// tokens of different parts would cost more than the state between them, which is
// made from the chunk's.  A part's P and R are made by tiles of 16 x 16 pairs, a wave
// each, and shared through LDS, turned round: [j][i].
//
// No atomics: the decays' gradient is added up per workgroup, then over workgroups
// in a fixed order; in float64 from a part's sum on, as a head's consoles and tokens may
// nearly cancel.
//
// What does not fit goes to scratch memory.  Of 64 bfloat16 dimensions, in 128 registers
// for four waves a SIMD: 5 vector and 62 scalar ones, 80 bytes a lane; of 128 dimensions, in
// 256: 104 (float32) and 146 vector ones, 176 and 192 bytes; of 32, and of 64 in float32,
// scalar ones alone, 64 bytes.  What that costs has not been measured by itself.
//
// What bounds it: 128 tokens of 512 consoles' 4 heads of 64 in bfloat16 take 140 us, where
// the 370 MB they move take 76 at a large copy's rate, the matrix instructions 19 and all
// vector instructions 63: issue and barriers, at four waves a SIMD (69 KB of LDS, two
// workgroups a compute unit).  With the parts left out one at a time: results' stores -25
// us, loads ahead -15, pairs -13, the decays' gradient -14, dS's loads -4.  On the way
// here: operands held in registers through a chunk 249 us; LDS read again where they are
// used 185; parts of 32 tokens instead of pairs of all 64 169; two waves for 16 columns
// 150; their inputs' waits put off to where they are used 140.  64 consoles take 26 us, in
// float32 34 (one workgroup a compute unit: 143 KB), in float32 with heads of 128 88, where
// two waves for 16 columns would not have registers enough.
#include "mem_decay_segments.h"

namespace nesle::mem {
namespace {

constexpr int kPart = 32;

__device__ double lanes_sum(double v) {
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

// Two waves for 16 columns where their registers leave room for it.
template <int DP>
constexpr int kGradRoles = DP == 128 ? 1 : 2;

// Waves of a SIMD that registers are to leave room for: what LDS does.
template <typename T, int DP>
constexpr int kGradWaves = sizeof(T) == 2 && DP <= 64 ? 4 : 2;

template <typename T, int DP>
struct GradTile {
    static constexpr int CH = kDecaySpan<T, DP>, ROLES = kGradRoles<DP>;
    using M = typename DecayMathOf<T, DP>::gradient;
    using In = typename M::template Tile<CH, DP, M::kIn, 8>;
    union Out {
        In in;
        DecayResults<T, DP, CH, ROLES> results;
    };
    Out q, k, v;               // then dQ, dK, dV
    In dout;
    typename M::template Tile<kPart, kPart, kFull, 8> p, r;        // [j][i]; zero where i is in an earlier tile
    f4 before[ROLES == 1 ? 1 : DP / 16][DP / 16][64];              // the state before a part, from role to role
    Powers<kPart> powers;
    alignas(16) int episodes[kPart];
    double sums[ROLES * DP / 16];
};

// The walk of a wave that has dQ and the pairs, dK, dV and dS, or both.  The waves of
// either kind meet at the same barriers.
template <typename T, int DP, bool WIDE, bool HAS_Q, bool HAS_KV>
__device__ __forceinline__ void grad_walk(const DecayArgs<T>& a, const DecaySegments& seg, double* partials, GradTile<T, DP>& sh) {
    using Tile = GradTile<T, DP>;
    constexpr int CH = Tile::CH, ROLES = Tile::ROLES, PARTS = CH / kPart, KT = DP / 16, KP = DP / 32, CT = kPart / 16, kWaves = DP / 16;
    using M = typename Tile::M;
    using In = Rows<T, WIDE>;
    using At = Place<DP, ROLES>;
    using Done = DecayResults<T, DP, CH, ROLES>;
    const At first;
    const std::uint32_t env = blockIdx.x / a.hv, h = blockIdx.x % a.hv, hk = h / a.group;
    const std::size_t head = blockIdx.x, state_size = static_cast<std::size_t>(a.dk_dim) * a.dv_dim;
    const std::size_t slot = static_cast<std::size_t>(blockIdx.y) * gridDim.x + head;
    const int dk_dim = static_cast<int>(a.dk_dim), dv_dim = static_cast<int>(a.dv_dim);
    const std::int64_t v_step = static_cast<std::int64_t>(a.batch) * a.hv * a.dv_dim;
    const f4 zero = {0, 0, 0, 0};
    const std::uint32_t begin = blockIdx.y * seg.steps;
    const std::uint32_t end = a.steps - begin < seg.steps ? a.steps : begin + seg.steps;

    Piece<T, DP, CH, WIDE, ROLES> q, k, v, dout;
    Resets<T> resets;
    f4 next[KT];                           // the state before the chunk
    const auto fetch = [&](std::uint32_t t1, const At& at) {
        const std::uint32_t start = (t1 - 1) / CH * CH;
        const int n = static_cast<int>(t1 - start);
        q.fetch(a.q, a.dk_dim, start, n, env, hk, at);
        k.fetch(a.k, a.dk_dim, start, n, env, hk, at);
        v.fetch(a.v, a.dv_dim, start, n, env, h, at);
        dout.fetch(a.dout, a.dv_dim, start, n, env, h, at);
        resets.fetch(a, start, n, env, at.lane);
        const float* from = start == 0 ? (a.state == nullptr ? nullptr : a.state + head * state_size)
                                       : a.saved + ((start / CH - 1) * static_cast<std::size_t>(a.batch) * a.hv + head) * state_size;
        if constexpr (HAS_Q) load_key_slab<DP>(from, dk_dim, dv_dim, at, next);
    };
    if (begin < end) fetch(end, first);
    f4 by_key[KT], by_value[KT];           // dS
    if constexpr (HAS_KV) {
        const float* from = seg.count > 1 ? seg.states + slot * state_size
                                          : a.dstate_out == nullptr ? nullptr : a.dstate_out + head * state_size;
        load_key_slab<DP>(from, dk_dim, dv_dim, first, by_key);
        load_value_slab<DP>(from, dk_dim, dv_dim, first, by_value);
    }
    const float gate = a.steps != 0 ? a.g[h] : 0.0f;
    const bool always = gate < kDropBelow;
    sh.powers.make(gate, a.scale, always, first.tid);
    if (first.tid < 64)
        for (int i = 0; i < 4; ++i) {
            sh.p.put(16 + 4 * first.g + i, first.r, 0.0f);
            sh.r.put(16 + 4 * first.g + i, first.r, 0.0f);
        }

    double decay = 0.0;                    // this lane's share of the decay's gradient
    for (std::uint32_t t1 = end; t1 > begin;) {
        At at = At::anew();
        const std::uint32_t start = (t1 - 1) / CH * CH;
        const int n = static_cast<int>(t1 - start);
        const std::uint64_t drops = resets.drops(n, at.lane, always);
        f4 S[KT];
#pragma unroll
        for (int i = 0; i < KT; ++i)
            if constexpr (HAS_Q) S[i] = (drops & 1u) ? zero : next[i];
        q.stage(sh.q.in, at);
        k.stage(sh.k.in, at);
        v.stage(sh.v.in, at);
        dout.stage(sh.dout, at);
        t1 = start;
        __syncthreads();
        if (t1 > begin) fetch(t1, at);
        typename Done::Tile done_q[CH / 16], done_k[CH / 16], done_v[CH / 16];
        const std::int64_t token = static_cast<std::int64_t>(start) * a.batch + env;
        // Of several value heads of a key head: one share each, added up afterwards.
        const std::int64_t share_step = static_cast<std::int64_t>(a.batch) * a.hv * a.dk_dim;
        const auto share = [&](bool of_k, int m, f4 x) {
            if (a.group == 1) return;
            const Rows<float, WIDE> to(a.scratch + (of_k ? a.steps * share_step : 0) + (token * a.hv + h) * a.dk_dim, share_step);
            DecayResults<float, DP, CH, ROLES>::put_tile(to, dk_dim, n, at, m, x);
        };

#pragma unroll
        for (int part = PARTS - 1; part >= 0; --part) {
            const int row0 = kPart * part, tile0 = row0 / 16;
            const std::uint32_t mine = static_cast<std::uint32_t>(drops >> row0);
            const bool dropped = mine & 1u;        // the state before the part is
            const Seen seen(mine & ~1u, min(n - row0, kPart));
            if (PARTS > 1 && n <= row0) {
#pragma unroll
                for (int m = 0; m < CT; ++m) done_q[tile0 + m] = done_k[tile0 + m] = done_v[tile0 + m] = Done::tile(zero);
                continue;
            }
            at = At::anew();
            const int r = at.r, g = at.g;
            if (seen.drops != 0) {
                if (at.tid < kPart) sh.episodes[at.tid] = seen.episode(at.tid);
                __syncthreads();
            }
            float here = 0.0f;             // of it, this part's
            const float whole = seen.whole(sh.powers), row4 = static_cast<float>(4 * g);
            f4 before[KT], dK[CT] = {}, dV[CT] = {};
            if constexpr (HAS_Q) {
                // P and R, a tile a wave; the workgroups of a compute unit leave out
                // different waves.
                for (int place = (at.wave + static_cast<int>(blockIdx.x)) % kWaves; place < 3; place += kWaves) {
                    const int it = place == 0 ? 0 : 1, jt = place == 2 ? 1 : 0;
                    f4 x = zero, y = zero;
#pragma unroll
                    for (int i = 0; i < KP; ++i) {
                        x = M::mul(sh.q.in.rows(row0 + 16 * it, i, r, g), sh.k.in.rows(row0 + 16 * jt, i, r, g), x);
                        y = M::mul(sh.dout.rows(row0 + 16 * it, i, r, g), sh.v.in.rows(row0 + 16 * jt, i, r, g), y);
                    }
                    PairPowers<kPart, true> pair;
                    pair.make(sh.powers, a.scale, r, g);
                    x = pair.weigh(x, it, jt, seen, sh.episodes, r, g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) here += (row4 + static_cast<float>(16 * (it - jt) + e - r)) * x[e] * y[e];
                    y = pair.weigh(y, it, jt, seen, sh.episodes, r, g);
                    sh.p.put4(16 * jt + r, 16 * it + 4 * g, x);
                    sh.r.put4(16 * jt + r, 16 * it + 4 * g, y);
                }
                // The state before the part.
                if (part == 0) {
#pragma unroll
                    for (int i = 0; i < KT; ++i) before[i] = S[i];
                } else {
                    const Seen ahead(drops & 0xffffffffu, kPart);
                    const float through = ahead.whole(sh.powers);
                    f4 K[2];
                    M::values(sh.k.in.cols(0, 16 * at.wave, r, g), K);
                    const auto held = M::full(K[0] * ahead.out(sh.powers, 4 * g), K[1] * ahead.out(sh.powers, 16 + 4 * g));
#pragma unroll
                    for (int i = 0; i < KT; ++i) before[i] = dropped ? zero : M::mul(sh.v.in.cols(0, 16 * i, r, g), held, S[i] * through);
                }
                if (ROLES > 1 && partials != nullptr)
#pragma unroll
                    for (int i = 0; i < KT; ++i) sh.before[at.wave][i][at.lane] = before[i];
            }
            if constexpr (HAS_KV) {
                // dK and dV from the tokens after the part.
#pragma unroll
                for (int i = 0; i < KP; ++i) {
                    const auto s = M::full(by_key[2 * i], by_key[2 * i + 1]);
#pragma unroll
                    for (int m = 0; m < CT; ++m) dK[m] = M::mul(sh.v.in.rows(row0 + 16 * m, i, r, g), s, dK[m]);
                }
#pragma unroll
                for (int i = 0; i < KP; ++i) {
                    __builtin_amdgcn_sched_barrier(0);
                    const auto s = M::full(by_value[2 * i], by_value[2 * i + 1]);
#pragma unroll
                    for (int m = 0; m < CT; ++m) dV[m] = M::mul(sh.k.in.rows(row0 + 16 * m, i, r, g), s, dV[m]);
                }
                __builtin_amdgcn_sched_barrier(0);
                f4 K[CT];
                M::values(sh.k.in.cols(row0, 16 * at.wave, r, g), K);
#pragma unroll
                for (int m = 0; m < CT; ++m) {
                    const f4 out = seen.out(sh.powers, 16 * m + 4 * g);
                    dK[m] *= out;
                    dV[m] *= out;
#pragma unroll
                    for (int e = 0; e < 4; ++e) here += (static_cast<float>(seen.n - 1 - 16 * m - e) - row4) * K[m][e] * dK[m][e];
                }
            }
            __syncthreads();
            if constexpr (HAS_Q) {
                // dQ: from the tokens before the part, then within.
                f4 x[CT] = {}, Q[CT];
#pragma unroll
                for (int i = 0; i < KP; ++i) {
                    const auto s = M::full(before[2 * i], before[2 * i + 1]);
#pragma unroll
                    for (int m = 0; m < CT; ++m) x[m] = M::mul(sh.dout.rows(row0 + 16 * m, i, r, g), s, x[m]);
                }
                M::values(sh.q.in.cols(row0, 16 * at.wave, r, g), Q);
                const auto key = sh.k.in.cols(row0, 16 * at.wave, r, g);
#pragma unroll
                for (int m = 0; m < CT; ++m) {
                    x[m] *= seen.in(sh.powers, 16 * m + 4 * g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) here += (row4 + static_cast<float>(16 * m + e + 1)) * Q[m][e] * x[m][e];
                    x[m] = M::mul(sh.r.cols(0, 16 * m, r, g), key, x[m]);
                    share(false, tile0 + m, x[m]);
                    done_q[tile0 + m] = Done::tile(x[m]);
                }
            }
            if constexpr (HAS_KV) {
                if (partials != nullptr) {
                    float held = 0.0f;
#pragma unroll
                    for (int i = 0; i < KT; ++i) {
                        const f4 s = ROLES > 1 ? sh.before[at.wave][i][at.lane] : before[i];
#pragma unroll
                        for (int e = 0; e < 4; ++e) held += by_key[i][e] * s[e];
                    }
                    here += static_cast<float>(seen.n) * whole * held;
                }
                // dK and dV within the part, and the two slabs of dS before it.
                f4 x[CT];
                const auto query = sh.q.in.cols(row0, 16 * at.wave, r, g);
                M::values(query, x);
#pragma unroll
                for (int m = 0; m < CT; ++m) {
                    dK[m] = M::mul(sh.r.rows(16 * m, 0, r, g), query, dK[m]);
                    share(true, tile0 + m, dK[m]);
                    done_k[tile0 + m] = Done::tile(dK[m]);
                    x[m] *= seen.in(sh.powers, 16 * m + 4 * g);
                }
                {
                    const auto read = M::full(x[0], x[1]);
#pragma unroll
                    for (int i = 0; i < KT; ++i)
                        by_key[i] = dropped ? zero : M::mul(sh.dout.cols(row0, 16 * i, r, g), read, by_key[i] * whole);
                }
                __builtin_amdgcn_sched_barrier(0);
                const auto grad = sh.dout.cols(row0, 16 * at.wave, r, g);
                M::values(grad, x);
#pragma unroll
                for (int m = 0; m < CT; ++m) {
                    dV[m] = M::mul(sh.p.rows(16 * m, 0, r, g), grad, dV[m]);
                    done_v[tile0 + m] = Done::tile(dV[m]);
                    x[m] *= seen.in(sh.powers, 16 * m + 4 * g);
                }
                __builtin_amdgcn_sched_barrier(0);
                const auto read = M::full(x[0], x[1]);
#pragma unroll
                for (int i = 0; i < KT; ++i)
                    by_value[i] = dropped ? zero : M::mul(sh.q.in.cols(row0, 16 * i, r, g), read, by_value[i] * whole);
            }
            decay += here;
            __syncthreads();               // P, R and, in the end, the inputs have been read
        }
        const std::int64_t key_step = static_cast<std::int64_t>(a.batch) * a.hk * a.dk_dim;
        const In dq(a.dq + (token * a.hk + hk) * a.dk_dim, key_step), dk(a.dk + (token * a.hk + hk) * a.dk_dim, key_step),
            dv(a.dv + static_cast<std::int64_t>(start) * v_step + head * a.dv_dim, v_step);
        at = At::anew();
        if (HAS_Q && a.group == 1) sh.q.results.put(dq, dk_dim, n, at, done_q);
        if constexpr (HAS_KV) {
            if (a.group == 1) sh.k.results.put(dk, dk_dim, n, at, done_k);
            sh.v.results.put(dv, dv_dim, n, at, done_v);
        }
        __syncthreads();
        if (a.group == 1) {
            sh.q.results.flush(dq, dk_dim, n, at);
            sh.k.results.flush(dk, dk_dim, n, at);
        }
        sh.v.results.flush(dv, dv_dim, n, at);
        __syncthreads();                   // before the next chunk takes their place
    }
    if (HAS_KV && a.dstate != nullptr && begin == 0) store_key_slab<DP>(a.dstate + head * state_size, dk_dim, dv_dim, At::anew(), by_key);
    if (partials != nullptr) {
        decay = lanes_sum(decay);
        if (first.lane == 0) sh.sums[first.role * kWaves + first.wave] = decay;
        __syncthreads();
        if (first.tid == 0) {
            double sum = 0.0;
            for (int w = 0; w < ROLES * kWaves; ++w) sum += sh.sums[w];
            partials[slot] = sum;
        }
    }
}

template <typename T, int DP, bool WIDE>
__global__ void __launch_bounds__(DP * 4 * kGradRoles<DP>, (kGradWaves<T, DP>)) decay_backward_kernel(DecayArgs<T> a, DecaySegments seg, double* partials) {
    __shared__ GradTile<T, DP> sh;
    if constexpr (kGradRoles<DP> == 1) grad_walk<T, DP, WIDE, true, true>(a, seg, partials, sh);
    else if (Place<DP, kGradRoles<DP>>().role == 0) grad_walk<T, DP, WIDE, true, false>(a, seg, partials, sh);
    else grad_walk<T, DP, WIDE, false, true>(a, seg, partials, sh);
}

// dg of a head: the sum of its workgroups' shares, by a workgroup.
__device__ __forceinline__ void gate_sum(const double* partials, float* dg, std::uint32_t h, std::uint32_t heads, std::uint64_t all) {
    __shared__ double sums[4];
    double sum = 0.0;
    for (std::uint64_t i = h + static_cast<std::uint64_t>(threadIdx.x) * heads; i < all; i += 256ull * heads) sum += partials[i];
    sum = lanes_sum(sum);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x == 0) dg[h] = static_cast<float>(sums[0] + sums[1] + sums[2] + sums[3]);
}
__global__ void __launch_bounds__(256) decay_gate_sum(const double* partials, float* dg, std::uint32_t heads, std::uint64_t all) {
    gate_sum(partials, dg, blockIdx.x, heads, all);
}

// dq and dk of a key head: the sum of its value heads' shares; and, by the workgroups from
// `blocks` on, the decays' sums (a launch of their own took 4 us more).
template <typename T>
__global__ void __launch_bounds__(256) decay_share_sum(DecayArgs<T> a, std::uint64_t quads, std::uint32_t blocks, const double* partials,
                                                       std::uint64_t all_partials) {
    if (blockIdx.x >= blocks) {
        gate_sum(partials, a.dg, blockIdx.x - blocks, a.hv, all_partials);
        return;
    }
    const std::uint64_t all = static_cast<std::uint64_t>(a.steps) * a.batch * a.hv * a.dk_dim;
    const std::uint32_t per_head = a.dk_dim / 4;
    for (std::uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < 2 * quads; i += blocks * 256ull) {
        const bool of_k = i >= quads;
        const std::uint64_t e = of_k ? i - quads : i, head = e / per_head;
        const float* from = a.scratch + (of_k ? all : 0) + head * a.group * a.dk_dim + 4 * (e % per_head);
        f4 v = load4(from, true);
        for (std::uint32_t s = 1; s < a.group; ++s) v += load4(from + static_cast<std::size_t>(s) * a.dk_dim, true);
        store4((of_k ? a.dk : a.dq) + 4 * e, v);
    }
}

// Floats of the shares, ahead of the segments' states and the decays' partial sums.
std::uint64_t share_floats(const nesle_decay_args& a) {
    const std::uint64_t floats = a.v_heads > a.k_heads ? 2ull * a.steps * a.batch * a.v_heads * a.k_dim : 0;
    return (floats + 3) / 4 * 4;
}

// A float64 sum a workgroup follows.
std::uint64_t ahead_of_partials(const nesle_decay_args& a, const DecaySegments& seg) { return (share_floats(a) + seg.floats(a) + 1) / 2 * 2; }

template <typename T, int DP, bool WIDE>
void launch_dim(const DecayArgs<T>& a, const DecaySegments& seg, double* partials, hipStream_t s) {
    if (seg.count > 1) launch_states<T, DP, WIDE, true>(a, seg, s);
    hipLaunchKernelGGL((decay_backward_kernel<T, DP, WIDE>), dim3(a.batch * a.hv, seg.count), dim3(DP * 4 * kGradRoles<DP>), 0, s, a, seg,
                       partials);
}

template <typename T>
int backward(const char* who, const nesle_decay_args& x, hipStream_t s) {
    const DecayArgs<T> a = decay_args<T>(x);
    DecaySegments seg = decay_segments(x, true);
    seg.place(x, a.scratch + share_floats(x));
    double* partials = a.dg == nullptr ? nullptr : reinterpret_cast<double*>(a.scratch + ahead_of_partials(x, seg));
    at_dim(x, [&](auto dim) {
        if (wide_rows(x)) launch_dim<T, dim(), true>(a, seg, partials, s);
        else launch_dim<T, dim(), false>(a, seg, partials, s);
    });
    const std::uint64_t all_partials = static_cast<std::uint64_t>(seg.count) * a.batch * a.hv;
    if (a.group > 1 && a.steps != 0) {
        const std::uint64_t quads = static_cast<std::uint64_t>(a.steps) * a.batch * a.hk * a.dk_dim / 4;
        const auto blocks = static_cast<std::uint32_t>(std::min<std::uint64_t>((2 * quads + 255) / 256, 4096));
        hipLaunchKernelGGL(decay_share_sum<T>, dim3(blocks + (partials != nullptr ? a.hv : 0)), dim3(256), 0, s, a, quads, blocks, partials,
                           all_partials);
    } else if (partials != nullptr) {
        hipLaunchKernelGGL(decay_gate_sum, dim3(a.hv), dim3(256), 0, s, partials, a.dg, a.hv, all_partials);
    }
    return launched(who);
}

// dg without a console: zeros.
__global__ void decay_gate_zero(float* dg, std::uint32_t heads) {
    const std::uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i < heads) dg[i] = 0.0f;
}

}  // namespace
}  // namespace nesle::mem

using namespace nesle::mem;

extern "C" {

std::uint64_t nesle_decay_scratch_floats(const nesle_decay_args* a) {
    if (a == nullptr || a->k_heads == 0 || a->batch == 0 || a->v_heads == 0) return 0;
    const DecaySegments seg = decay_segments(*a, true);
    return ahead_of_partials(*a, seg) + 2ull * seg.count * a->batch * a->v_heads;
}

int nesle_decay_backward(const nesle_decay_args* a, void* stream) {
    const char* who = "nesle_decay_backward";
    int rc = check_decay(who, a);
    if (rc != NESLE_OK) return rc;
    const auto s = static_cast<hipStream_t>(stream);
    if (a->batch == 0) {
        if (a->dg == nullptr) return NESLE_OK;
        hipLaunchKernelGGL(decay_gate_zero, dim3((a->v_heads + 255) / 256), dim3(256), 0, s, a->dg, a->v_heads);
        return launched(who);
    }
    rc = check_decay_alignment(who, a);
    if (rc != NESLE_OK) return rc;
    if (a->steps != 0) {
        rc = check_decay_inputs(who, a);
        if (rc != NESLE_OK) return rc;
        if (!a->dout.data || !a->dq || !a->dk || !a->dv || (!a->saved && nesle_decay_saved_floats(a) != 0))
            return refuse(who, "null device pointer");
    }
    if (!a->scratch && ((a->steps != 0 && a->v_heads > a->k_heads) || decay_segments(*a, true).count > 1 || a->dg)) return refuse(who, "null device pointer");
    return a->dtype == NESLE_MEM_F32 ? backward<float>(who, *a, s) : backward<bf16>(who, *a, s);
}

}  // extern "C"
