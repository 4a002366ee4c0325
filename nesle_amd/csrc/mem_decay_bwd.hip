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
// dK and dV.  dS is needed by key columns (dK) and by value columns (dV): a wave
// holds both slabs of it in registers and updates both, which costs a product more
// and saves passing it through LDS.
//
// Inputs come and results go a chunk at a time, and the forward kept one state a
// chunk; inside, the work goes in parts of 32 tokens, last to first, as pairs of
// tokens of different parts would cost more than the state between them, which is
// made from the chunk's.  A part's P and R are made by tiles of 16 x 16 pairs, a wave
// each, and shared through LDS, turned round: [j][i].
//
// No atomics: the decays' gradient is added up per workgroup, then over workgroups
// in a fixed order.
#include "mem_decay_segments.h"

namespace nesle::mem {
namespace {

constexpr int kPart = 32;

template <typename T, int DP, int CH>
struct GradTile {
    using M = DecayMath<T>;
    using In = typename M::template Tile<CH, DP, M::kIn, 8>;
    union Out {
        In in;
        DecayResults<T, DP, CH> results;
    };
    Out q, k, v;               // then dQ, dK, dV
    In dout;
    typename M::template Tile<kPart, kPart, kFull, 8> p, r;        // [j][i]; zero where i is in an earlier tile
    Powers<kPart> powers;
    alignas(16) int episodes[kPart];
    float sums[DP / 16];
};

// Waves of a SIMD that registers are to leave room for: what LDS does.
template <typename T, int DP>
constexpr int kGradWaves = sizeof(T) == 2 && DP <= 64 ? 3 : 2;

template <typename T, int DP, bool WIDE>
__global__ void __launch_bounds__(DP * 4, (kGradWaves<T, DP>)) decay_backward_kernel(DecayArgs<T> a, DecaySegments seg, float* partials) {
    constexpr int CH = kDecayChunk<T>, PARTS = CH / kPart, KT = DP / 16, KP = DP / 32, kWaves = DP / 16;
    using Tile = GradTile<T, DP, CH>;
    using M = typename Tile::M;
    using In = Rows<T, WIDE>;
    using Done = DecayResults<T, DP, CH>;
    __shared__ Tile sh;
    const Lane<DP> first;
    const std::uint32_t env = blockIdx.x / a.hv, h = blockIdx.x % a.hv, hk = h / a.group;
    const std::size_t head = blockIdx.x, state_size = static_cast<std::size_t>(a.dk_dim) * a.dv_dim;
    const std::size_t slot = static_cast<std::size_t>(blockIdx.y) * gridDim.x + head;
    const int dk_dim = static_cast<int>(a.dk_dim), dv_dim = static_cast<int>(a.dv_dim);
    const std::int64_t v_step = static_cast<std::int64_t>(a.batch) * a.hv * a.dv_dim;
    const f4 zero = {0, 0, 0, 0};
    const std::uint32_t begin = blockIdx.y * seg.steps;
    const std::uint32_t end = a.steps - begin < seg.steps ? a.steps : begin + seg.steps;

    const float gate = a.steps != 0 ? a.g[h] : 0.0f;
    const bool always = gate < kDropBelow;
    sh.powers.make(gate, always, first.tid);
    if (first.tid < 64)
        for (int i = 0; i < 4; ++i) {
            sh.p.put(16 + 4 * first.g + i, first.r, 0.0f);
            sh.r.put(16 + 4 * first.g + i, first.r, 0.0f);
        }
    f4 by_key[KT], by_value[KT];           // dS
    {
        const float* from = seg.count > 1 ? seg.states + slot * state_size
                                          : a.dstate_out == nullptr ? nullptr : a.dstate_out + head * state_size;
        load_key_slab<DP>(from, dk_dim, dv_dim, first, by_key);
        load_value_slab<DP>(from, dk_dim, dv_dim, first, by_value);
    }

    Piece<T, DP, CH, WIDE> q, k, v, dout;
    std::uint64_t next_drops = 0;
    const auto fetch = [&](std::uint32_t t1, const Lane<DP>& at) {
        const std::uint32_t start = (t1 - 1) / CH * CH;
        const int n = static_cast<int>(t1 - start);
        q.fetch(a.q, a.dk_dim, start, n, env, hk, at);
        k.fetch(a.k, a.dk_dim, start, n, env, hk, at);
        v.fetch(a.v, a.dv_dim, start, n, env, h, at);
        dout.fetch(a.dout, a.dv_dim, start, n, env, h, at);
        next_drops = drops_of<CH>(a, start, n, env, at.lane, always);
    };
    if (begin < end) fetch(end, first);
    float decay = 0.0f;                    // this lane's share of the decay's gradient
    for (std::uint32_t t1 = end; t1 > begin;) {
        // Made anew for each step of the work: what one has read from LDS is read again
        // by the next, rather than held in registers through both.
        Lane<DP> at = Lane<DP>::anew();
        int r = at.r, g = at.g;
        const auto anew = [&] {
            at = Lane<DP>::anew();
            r = at.r;
            g = at.g;
        };
        const std::uint32_t start = (t1 - 1) / CH * CH;
        const int n = static_cast<int>(t1 - start);
        const std::uint64_t drops = next_drops;
        const float* from = (drops & 1u) ? nullptr : start == 0 ? (a.state == nullptr ? nullptr : a.state + head * state_size)
                                         : a.saved + ((start / CH - 1) * static_cast<std::size_t>(a.batch) * a.hv + head) * state_size;
        f4 S[KT];
        load_key_slab<DP>(from, dk_dim, dv_dim, at, S);
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
            DecayResults<float, DP, CH>::put_tile(to, dk_dim, n, at, m, x);
        };

#pragma unroll
        for (int part = PARTS - 1; part >= 0; --part) {
            constexpr int CT = kPart / 16;
            const int row0 = kPart * part;
            const std::uint32_t mine = static_cast<std::uint32_t>(drops >> row0);
            const bool dropped = mine & 1u;        // the state before the part is
            const Seen seen(mine & ~1u, min(n - row0, kPart));
            if (PARTS > 1 && n <= row0) {
#pragma unroll
                for (int m = 0; m < CT; ++m) done_q[row0 / 16 + m] = done_k[row0 / 16 + m] = done_v[row0 / 16 + m] = Done::tile(zero);
                continue;
            }
            anew();
            if (seen.drops != 0 && at.tid < kPart) sh.episodes[at.tid] = seen.episode(at.tid);
            if (seen.drops != 0) __syncthreads();
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
                for (int e = 0; e < 4; ++e) decay += static_cast<float>(16 * (it - jt) + 4 * g + e - r) * x[e] * y[e];
                y = pair.weigh(y, it, jt, seen, sh.episodes, r, g);
                sh.p.put4(16 * jt + r, 16 * it + 4 * g, x);
                sh.r.put4(16 * jt + r, 16 * it + 4 * g, y);
            }
            // The state before the part.
            f4 before[KT];
            if (part == 0) {
#pragma unroll
                for (int i = 0; i < KT; ++i) before[i] = S[i];
            } else {
                const Seen ahead(drops & 0xffffffffu, kPart);
                const float whole = ahead.whole(sh.powers);
                f4 K[2];
                M::values(sh.k.in.cols(0, 16 * at.wave, r, g), K);
                const auto held = M::full(K[0] * ahead.out(sh.powers, 4 * g), K[1] * ahead.out(sh.powers, 16 + 4 * g));
#pragma unroll
                for (int i = 0; i < KT; ++i) before[i] = dropped ? zero : M::mul(sh.v.in.cols(0, 16 * i, r, g), held, S[i] * whole);
            }
            const float whole = seen.whole(sh.powers);
            {
                float held = 0.0f;
#pragma unroll
                for (int i = 0; i < KT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) held += by_key[i][e] * before[i][e];
                decay += static_cast<float>(seen.n) * whole * held;
            }
            __syncthreads();

            // dQ: from the tokens before the part, then within.
            {
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
                    x[m] *= seen.in(sh.powers, 16 * m + 4 * g) * a.scale;
#pragma unroll
                    for (int e = 0; e < 4; ++e) decay += static_cast<float>(16 * m + 4 * g + e + 1) * Q[m][e] * x[m][e];
                    x[m] = M::mul(sh.r.cols(0, 16 * m, r, g), key, x[m]);
                    share(false, row0 / 16 + m, x[m]);
                    done_q[row0 / 16 + m] = Done::tile(x[m]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            anew();
            // dK: from the tokens after the part, then within; the slab of dS that it reads.
            {
                f4 x[CT] = {}, K[CT], Q[CT];
#pragma unroll
                for (int i = 0; i < KP; ++i) {
                    const auto s = M::full(by_key[2 * i], by_key[2 * i + 1]);
#pragma unroll
                    for (int m = 0; m < CT; ++m) x[m] = M::mul(sh.v.in.rows(row0 + 16 * m, i, r, g), s, x[m]);
                }
                M::values(sh.k.in.cols(row0, 16 * at.wave, r, g), K);
                const auto query = sh.q.in.cols(row0, 16 * at.wave, r, g);
                M::values(query, Q);
#pragma unroll
                for (int m = 0; m < CT; ++m) {
                    x[m] *= seen.out(sh.powers, 16 * m + 4 * g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) decay += static_cast<float>(seen.n - 1 - (16 * m + 4 * g + e)) * K[m][e] * x[m][e];
                    x[m] = M::mul(sh.r.rows(16 * m, 0, r, g), query, x[m]);
                    share(true, row0 / 16 + m, x[m]);
                    done_k[row0 / 16 + m] = Done::tile(x[m]);
                    Q[m] *= seen.in(sh.powers, 16 * m + 4 * g) * a.scale;
                }
                const auto read = M::full(Q[0], Q[1]);
#pragma unroll
                for (int i = 0; i < KT; ++i)
                    by_key[i] = dropped ? zero : M::mul(sh.dout.cols(row0, 16 * i, r, g), read, by_key[i] * whole);
            }
            __builtin_amdgcn_sched_barrier(0);
            anew();
            // dV, the same.
            {
                f4 x[CT] = {}, dO[CT];
#pragma unroll
                for (int i = 0; i < KP; ++i) {
                    const auto s = M::full(by_value[2 * i], by_value[2 * i + 1]);
#pragma unroll
                    for (int m = 0; m < CT; ++m) x[m] = M::mul(sh.k.in.rows(row0 + 16 * m, i, r, g), s, x[m]);
                }
                const auto grad = sh.dout.cols(row0, 16 * at.wave, r, g);
                M::values(grad, dO);
#pragma unroll
                for (int m = 0; m < CT; ++m) {
                    x[m] *= seen.out(sh.powers, 16 * m + 4 * g);
                    x[m] = M::mul(sh.p.rows(16 * m, 0, r, g), grad, x[m]);
                    done_v[row0 / 16 + m] = Done::tile(x[m]);
                    dO[m] *= seen.in(sh.powers, 16 * m + 4 * g) * a.scale;
                }
                const auto read = M::full(dO[0], dO[1]);
#pragma unroll
                for (int i = 0; i < KT; ++i)
                    by_value[i] = dropped ? zero : M::mul(sh.q.in.cols(row0, 16 * i, r, g), read, by_value[i] * whole);
            }
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();               // P, R and, in the end, the inputs have been read
        }
        const std::int64_t key_step = static_cast<std::int64_t>(a.batch) * a.hk * a.dk_dim;
        const In dq(a.dq + (token * a.hk + hk) * a.dk_dim, key_step), dk(a.dk + (token * a.hk + hk) * a.dk_dim, key_step),
            dv(a.dv + static_cast<std::int64_t>(start) * v_step + head * a.dv_dim, v_step);
        anew();
        if (a.group == 1) {
            sh.q.results.put(dq, dk_dim, n, at, done_q);
            sh.k.results.put(dk, dk_dim, n, at, done_k);
        }
        sh.v.results.put(dv, dv_dim, n, at, done_v);
        __syncthreads();
        if (a.group == 1) {
            sh.q.results.flush(dq, dk_dim, n, at);
            sh.k.results.flush(dk, dk_dim, n, at);
        }
        sh.v.results.flush(dv, dv_dim, n, at);
        __syncthreads();                   // before the next chunk takes their place
    }
    if (a.dstate != nullptr && begin == 0) store_key_slab<DP>(a.dstate + head * state_size, dk_dim, dv_dim, Lane<DP>::anew(), by_key);
    if (partials != nullptr) {
        decay = over_groups(sum16(decay));
        if (first.lane == 0) sh.sums[first.wave] = decay;
        __syncthreads();
        if (first.tid == 0) {
            float sum = 0.0f;
            for (int w = 0; w < kWaves; ++w) sum += sh.sums[w];
            partials[slot] = sum;
        }
    }
}

// dg of a head: the sum of its workgroups' shares, a workgroup a head.
__global__ void __launch_bounds__(256) decay_gate_sum(const float* partials, float* dg, std::uint32_t heads, std::uint64_t all) {
    __shared__ float sums[4];
    float sum = 0.0f;
    for (std::uint64_t i = blockIdx.x + static_cast<std::uint64_t>(threadIdx.x) * heads; i < all; i += 256ull * heads) sum += partials[i];
    sum = over_groups(sum16(sum));
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x == 0) dg[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

// dq and dk of a key head: the sum of its value heads' shares.
template <typename T>
__global__ void __launch_bounds__(256) decay_share_sum(DecayArgs<T> a, std::uint64_t quads) {
    const std::uint64_t all = static_cast<std::uint64_t>(a.steps) * a.batch * a.hv * a.dk_dim;
    const std::uint32_t per_head = a.dk_dim / 4;
    for (std::uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < 2 * quads; i += gridDim.x * 256ull) {
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

template <typename T, int DP, bool WIDE>
void launch_dim(const DecayArgs<T>& a, const DecaySegments& seg, float* partials, hipStream_t s) {
    if (seg.count > 1) launch_states<T, DP, WIDE, true>(a, seg, s);
    hipLaunchKernelGGL((decay_backward_kernel<T, DP, WIDE>), dim3(a.batch * a.hv, seg.count), dim3(DP * 4), 0, s, a, seg, partials);
}

template <typename T>
int backward(const char* who, const nesle_decay_args& x, hipStream_t s) {
    const DecayArgs<T> a = decay_args<T>(x);
    DecaySegments seg = decay_segments(x);
    seg.place(x, a.scratch + share_floats(x));
    float* partials = a.dg == nullptr ? nullptr : a.scratch + share_floats(x) + seg.floats(x);
    const std::uint32_t dim = wide_rows(x) ? 0 : padded_dim(x);
    switch (dim) {
        case 0: launch_dim<T, 128, true>(a, seg, partials, s); break;
        case 32: launch_dim<T, 32, false>(a, seg, partials, s); break;
        case 64: launch_dim<T, 64, false>(a, seg, partials, s); break;
        default: launch_dim<T, 128, false>(a, seg, partials, s); break;
    }
    if (a.group > 1 && a.steps != 0) {
        const std::uint64_t quads = static_cast<std::uint64_t>(a.steps) * a.batch * a.hk * a.dk_dim / 4;
        const std::uint64_t want = (2 * quads + 255) / 256;
        hipLaunchKernelGGL(decay_share_sum<T>, dim3(static_cast<std::uint32_t>(want < 4096 ? want : 4096)), dim3(256), 0, s, a, quads);
    }
    if (partials != nullptr)
        hipLaunchKernelGGL(decay_gate_sum, dim3(a.hv), dim3(256), 0, s, partials, a.dg, a.hv, static_cast<std::uint64_t>(seg.count) * a.batch * a.hv);
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
    const DecaySegments seg = decay_segments(*a);
    return share_floats(*a) + seg.floats(*a) + static_cast<std::uint64_t>(seg.count) * a->batch * a->v_heads;
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
    if (a->steps != 0) {
        rc = check_decay_inputs(who, a);
        if (rc != NESLE_OK) return rc;
        if (!a->dout.data || !a->dq || !a->dk || !a->dv || (!a->saved && nesle_decay_saved_floats(a) != 0))
            return refuse(who, "null device pointer");
    }
    if (!a->scratch && ((a->steps != 0 && a->v_heads > a->k_heads) || decay_segments(*a).count > 1 || a->dg)) return refuse(who, "null device pointer");
    return a->dtype == NESLE_MEM_F32 ? backward<float>(who, *a, s) : backward<bf16>(who, *a, s);
}

}  // extern "C"
