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
// and saves passing it through LDS.  P, R and R turned round are made by every wave
// for itself and stay in registers, as in the forward; LDS holds Q, K, V and dO of
// the chunk and, once they have been read, the results on their way out.
//
// No atomics: the decays' gradient is added up per workgroup, then over workgroups
// in a fixed order.
#include "mem_decay.h"

namespace nesle::mem {
namespace {

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
    Powers<CH> powers;
    alignas(16) int episodes[CH];
    float sums[DP / 16];
};

// With 128 dimensions eight waves make a workgroup and two of them a SIMD.
template <typename T, int DP, bool WIDE>
__global__ void __launch_bounds__(DP * 4, 2) decay_backward_kernel(DecayArgs<T> a, float* partials) {
    constexpr int CH = kDecayChunk<T>, CT = CH / 16, KT = DP / 16, KP = DP / 32, kWaves = DP / 16;
    using Tile = GradTile<T, DP, CH>;
    using M = typename Tile::M;
    using In = Rows<T, WIDE>;
    __shared__ Tile sh;
    const Lane<DP> first;
    const std::uint32_t env = blockIdx.x / a.hv, h = blockIdx.x % a.hv, hk = h / a.group;
    const std::size_t head = blockIdx.x, state_size = static_cast<std::size_t>(a.dk_dim) * a.dv_dim;
    const int dk_dim = static_cast<int>(a.dk_dim), dv_dim = static_cast<int>(a.dv_dim);
    const std::int64_t v_step = static_cast<std::int64_t>(a.batch) * a.hv * a.dv_dim;
    const f4 zero = {0, 0, 0, 0};

    const float gate = a.steps != 0 ? a.g[h] : 0.0f;
    const bool always = gate < kDropBelow;
    sh.powers.make(gate, always, first.tid);
    f4 by_key[KT], by_value[KT];           // dS
    {
        const float* from = a.dstate_out == nullptr ? nullptr : a.dstate_out + head * state_size;
        load_key_slab<DP>(from, dk_dim, dv_dim, first, by_key);
        load_value_slab<DP>(from, dk_dim, dv_dim, first, by_value);
    }
    __syncthreads();
    PairPowers<CH, true> later;
    PairPowers<CH, false> earlier;
    later.make(sh.powers, a.scale, first.r, first.g);
    earlier.make(sh.powers, a.scale, first.r, first.g);

    Piece<T, DP, CH, WIDE> q, k, v, dout;
    std::uint64_t next_drops = 0;
    const auto fetch = [&](std::uint32_t end, const Lane<DP>& at) {
        const std::uint32_t start = (end - 1) / CH * CH;
        const int n = static_cast<int>(end - start);
        q.fetch(a.q, a.dk_dim, start, n, env, hk, at);
        k.fetch(a.k, a.dk_dim, start, n, env, hk, at);
        v.fetch(a.v, a.dv_dim, start, n, env, h, at);
        dout.fetch(a.dout, a.dv_dim, start, n, env, h, at);
        next_drops = drops_of<CH>(a, start, n, env, at.lane, always);
    };
    if (a.steps != 0) fetch(a.steps, first);
    float decay = 0.0f;                    // this lane's share of the decay's gradient
    for (std::uint32_t t1 = a.steps; t1 > 0;) {
        // Made anew for each part of the chunk: what one part has read from LDS is read
        // again by the next, rather than held in registers through both.
        Lane<DP> at = Lane<DP>::anew();
        int r = at.r, g = at.g;
        const auto next_part = [&] {
            at = Lane<DP>::anew();
            r = at.r;
            g = at.g;
        };
        const std::uint32_t start = (t1 - 1) / CH * CH;
        const int n = static_cast<int>(t1 - start);
        const bool dropped = next_drops & 1u;      // the state before the chunk is
        const Seen seen(next_drops & ~1ull, n);
        const float* from = dropped ? nullptr : start == 0 ? (a.state == nullptr ? nullptr : a.state + head * state_size)
                                              : a.saved + ((start / CH - 1) * static_cast<std::size_t>(a.batch) * a.hv + head) * state_size;
        f4 S[KT];
        load_key_slab<DP>(from, dk_dim, dv_dim, at, S);
        q.stage(sh.q.in, at);
        k.stage(sh.k.in, at);
        v.stage(sh.v.in, at);
        dout.stage(sh.dout, at);
        if (seen.drops != 0 && at.tid < CH) sh.episodes[at.tid] = seen.episode(at.tid);
        t1 = start;
        const float whole = seen.whole(sh.powers);
        {
            float held = 0.0f;
#pragma unroll
            for (int i = 0; i < KT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) held += by_key[i][e] * S[i][e];
            decay += static_cast<float>(n) * whole * held;
        }
        __syncthreads();
        using Done = DecayResults<T, DP, CH>;
        typename Done::Tile done_q[CT], done_k[CT], done_v[CT];
        const std::int64_t token = static_cast<std::int64_t>(start) * a.batch + env;
        // Of several value heads of a key head: one share each, added up afterwards.
        const std::int64_t share_step = static_cast<std::int64_t>(a.batch) * a.hv * a.dk_dim;
        const auto share = [&](bool of_k, int m, f4 x) {
            if (a.group == 1) return;
            const Rows<float, WIDE> to(a.scratch + (of_k ? a.steps * share_step : 0) + (token * a.hv + h) * a.dk_dim, share_step);
            DecayResults<float, DP, CH>::put_tile(to, dk_dim, n, at, m, x);
        };

        // dQ: from the chunks before, then R turned round.
        {
            f4 dQ[CT];
#pragma unroll
            for (int m = 0; m < CT; ++m) dQ[m] = zero;
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                const auto s = M::full(S[2 * i], S[2 * i + 1]);
#pragma unroll
                for (int m = 0; m < CT; ++m) dQ[m] = M::mul(sh.dout.rows(16 * m, i, r, g), s, dQ[m]);
            }
#pragma unroll
            for (int p = 0; p < CT / 2; ++p) {
                f4 Q[2];
                M::values(sh.q.in.cols(32 * p, 16 * at.wave, r, g), Q);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int m = 2 * p + t;
                    dQ[m] *= seen.in(sh.powers, 16 * m + 4 * g) * a.scale;
#pragma unroll
                    for (int e = 0; e < 4; ++e) decay += static_cast<float>(16 * m + 4 * g + e + 1) * Q[t][e] * dQ[m][e];
                }
            }
#pragma unroll
            for (int m = 0; m < CT; ++m) {
#pragma unroll
                for (int p = 0; p <= m / 2; ++p) {
                    f4 x[2] = {zero, zero};
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (2 * p + t > m) break;
#pragma unroll
                        for (int i = 0; i < KP; ++i)
                            x[t] = M::mul(sh.v.in.rows(16 * (2 * p + t), i, r, g), sh.dout.rows(16 * m, i, r, g), x[t]);
                        x[t] = earlier.weigh(x[t], m, 2 * p + t, seen, sh.episodes, r, g);
                    }
                    dQ[m] = M::mul(M::full(x[0], x[1]), sh.k.in.cols(32 * p, 16 * at.wave, r, g), dQ[m]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                share(false, m, dQ[m]);
                done_q[m] = Done::tile(dQ[m]);
            }
        }
        next_part();
        if (t1 > 0) fetch(t1, at);
        // dK and dV: from the chunks after, then R and P.
        {
            f4 dK[CT], dV[CT];
#pragma unroll
            for (int m = 0; m < CT; ++m) dK[m] = dV[m] = zero;
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                const auto dk = M::full(by_key[2 * i], by_key[2 * i + 1]), dv = M::full(by_value[2 * i], by_value[2 * i + 1]);
#pragma unroll
                for (int m = 0; m < CT; ++m) {
                    dK[m] = M::mul(sh.v.in.rows(16 * m, i, r, g), dk, dK[m]);
                    dV[m] = M::mul(sh.k.in.rows(16 * m, i, r, g), dv, dV[m]);
                }
            }
#pragma unroll
            for (int p = 0; p < CT / 2; ++p) {
                f4 K[2];
                M::values(sh.k.in.cols(32 * p, 16 * at.wave, r, g), K);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int m = 2 * p + t;
                    const f4 out = seen.out(sh.powers, 16 * m + 4 * g);
                    dK[m] *= out;
                    dV[m] *= out;
#pragma unroll
                    for (int e = 0; e < 4; ++e) decay += static_cast<float>(n - 1 - (16 * m + 4 * g + e)) * K[t][e] * dK[m][e];
                }
            }
#pragma unroll
            for (int m = 0; m < CT; ++m) {
#pragma unroll
                for (int p = m / 2; p < CT / 2; ++p) {
                    f4 x[2] = {zero, zero}, y[2] = {zero, zero};
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int it = 2 * p + t;
                        if (it < m) continue;
#pragma unroll
                        for (int i = 0; i < KP; ++i) {
                            x[t] = M::mul(sh.q.in.rows(16 * it, i, r, g), sh.k.in.rows(16 * m, i, r, g), x[t]);
                            y[t] = M::mul(sh.dout.rows(16 * it, i, r, g), sh.v.in.rows(16 * m, i, r, g), y[t]);
                        }
                        x[t] = later.weigh(x[t], it, m, seen, sh.episodes, r, g);
                        if ((it * CT + m) % kWaves == at.wave)         // a tile is one wave's
#pragma unroll
                            for (int e = 0; e < 4; ++e) decay += static_cast<float>(16 * (it - m) + 4 * g + e - r) * x[t][e] * y[t][e];
                        y[t] = later.weigh(y[t], it, m, seen, sh.episodes, r, g);
                    }
                    dV[m] = M::mul(M::full(x[0], x[1]), sh.dout.cols(32 * p, 16 * at.wave, r, g), dV[m]);
                    dK[m] = M::mul(M::full(y[0], y[1]), sh.q.in.cols(32 * p, 16 * at.wave, r, g), dK[m]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                share(true, m, dK[m]);
                done_k[m] = Done::tile(dK[m]);
                done_v[m] = Done::tile(dV[m]);
                next_part();
            }
        }
        next_part();
        // The state's gradient before the chunk.
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            by_key[i] *= whole;
            by_value[i] *= whole;
        }
#pragma unroll
        for (int p = 0; p < CT / 2; ++p) {
            f4 x[2];
            M::values(sh.q.in.cols(32 * p, 16 * at.wave, r, g), x);
            const f4 in[2] = {seen.in(sh.powers, 32 * p + 4 * g) * a.scale, seen.in(sh.powers, 32 * p + 16 + 4 * g) * a.scale};
            const auto of_q = M::full(x[0] * in[0], x[1] * in[1]);
            M::values(sh.dout.cols(32 * p, 16 * at.wave, r, g), x);
            const auto of_do = M::full(x[0] * in[0], x[1] * in[1]);
#pragma unroll
            for (int i = 0; i < KT; ++i) {
                by_key[i] = M::mul(sh.dout.cols(32 * p, 16 * i, r, g), of_q, by_key[i]);
                by_value[i] = M::mul(sh.q.in.cols(32 * p, 16 * i, r, g), of_do, by_value[i]);
            }
            }
        if (dropped)
#pragma unroll
            for (int i = 0; i < KT; ++i) by_key[i] = by_value[i] = zero;

        const std::int64_t key_step = static_cast<std::int64_t>(a.batch) * a.hk * a.dk_dim;
        const In dq(a.dq + (token * a.hk + hk) * a.dk_dim, key_step), dk(a.dk + (token * a.hk + hk) * a.dk_dim, key_step),
            dv(a.dv + static_cast<std::int64_t>(start) * v_step + head * a.dv_dim, v_step);
        __syncthreads();                   // the inputs have been read
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
    if (a.dstate != nullptr) store_key_slab<DP>(a.dstate + head * state_size, dk_dim, dv_dim, Lane<DP>::anew(), by_key);
    if (partials != nullptr) {
        decay = over_groups(sum16(decay));
        if (first.lane == 0) sh.sums[first.wave] = decay;
        __syncthreads();
        if (first.tid == 0) {
            float sum = 0.0f;
            for (int w = 0; w < kWaves; ++w) sum += sh.sums[w];
            partials[head] = sum;
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

// Floats of the shares, ahead of the decays' partial sums.
std::uint64_t share_floats(const nesle_decay_args& a) {
    return a.v_heads > a.k_heads ? 2ull * a.steps * a.batch * a.v_heads * a.k_dim : 0;
}

template <typename T>
int backward(const char* who, const nesle_decay_args& x, hipStream_t s) {
    const DecayArgs<T> a = decay_args<T>(x);
    const dim3 grid(a.batch * a.hv);
    float* partials = a.dg == nullptr ? nullptr : a.scratch + share_floats(x);
    const std::uint32_t dim = wide_rows(x) ? 0 : padded_dim(x);
    switch (dim) {
        case 0: hipLaunchKernelGGL((decay_backward_kernel<T, 128, true>), grid, dim3(512), 0, s, a, partials); break;
        case 32: hipLaunchKernelGGL((decay_backward_kernel<T, 32, false>), grid, dim3(128), 0, s, a, partials); break;
        case 64: hipLaunchKernelGGL((decay_backward_kernel<T, 64, false>), grid, dim3(256), 0, s, a, partials); break;
        default: hipLaunchKernelGGL((decay_backward_kernel<T, 128, false>), grid, dim3(512), 0, s, a, partials); break;
    }
    if (a.group > 1 && a.steps != 0) {
        const std::uint64_t quads = static_cast<std::uint64_t>(a.steps) * a.batch * a.hk * a.dk_dim / 4;
        const std::uint64_t want = (2 * quads + 255) / 256;
        hipLaunchKernelGGL(decay_share_sum<T>, dim3(static_cast<std::uint32_t>(want < 4096 ? want : 4096)), dim3(256), 0, s, a, quads);
    }
    if (partials != nullptr)
        hipLaunchKernelGGL(decay_gate_sum, dim3(a.hv), dim3(256), 0, s, partials, a.dg, a.hv, static_cast<std::uint64_t>(a.batch) * a.hv);
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
    if (a == nullptr || a->k_heads == 0) return 0;
    return share_floats(*a) + static_cast<std::uint64_t>(a->batch) * a->v_heads;
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
    if (!a->scratch && ((a->steps != 0 && a->v_heads > a->k_heads) || a->dg)) return refuse(who, "null device pointer");
    return a->dtype == NESLE_MEM_F32 ? backward<float>(who, *a, s) : backward<bf16>(who, *a, s);
}

}  // extern "C"
