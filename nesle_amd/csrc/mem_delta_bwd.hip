// Gradient of the gated delta rule over a rollout (mem_delta_fwd.hip has the
// forward's formulas and layout).  Chunks are taken last to first; each makes
// A, P, U again from its inputs and the state before it, which the forward
// kept.  With dO the outputs' gradient, dS the gradient of the state after the
// chunk, E = gamma_last / gamma and all products within the chunk:
//   dU = P^T dO + E K dS,   (I + A)^T dR = dU,   dV = beta dR,   X = beta gamma dR
//   dS before = gamma_last dS + scale Q^T (gamma dO) - K^T X
//   dP = dO U^T (j <= i),   dA = -dR U^T (j < i)
//   dQ = scale gamma (dO S^T) + M1 K,                M1 = scale L dP
//   dK = M1^T Q + E (U dS^T) - beta gamma (dR S^T) + M2 K + M2^T K,   M2 = beta L dA
//   dbeta = dR . (V - gamma K S) + rowsum(dA L kk)
// The gate of token t scales what crosses from before t to t or later: dg_t is
// the sum of E_ij = dP_ij P_ij + dA_ij A_ij over j < t <= i, of
// gamma_i (scale dO.QS - beta dR.KS) over i >= t, of e_j = E_j (K dS)_j.U_j over
// j < t, and of gamma_last <dS, S>.  (As sums of what crosses: the row sums less
// the column sums over i >= t would be equal, but cancel where neighbouring
// keys are alike.  There e_j and dA_ij A_ij still nearly cancel: dP and dA are summed
// in short pieces; one chain of 128 products left 4.5e-6 of the gates' gradient where
// all keys are equal.)  It is zero where the state is dropped.
//
// The part over value columns runs a wave per 16 columns, as in the forward;
// the part that sums over the value dimension runs a wave per 16 key columns,
// on U, dR and dO left in LDS, S and dS passed through LDS 32 columns at a time.
// No atomics: sums over waves are added in a fixed order.
//
// Bound by neither memory nor the matrix units: 128 steps of 512 consoles of 4 heads
// of 64 in bfloat16 take 250 us, where the 0.30 GB they move take 61 us at a large
// copy's rate and the products' instructions 41 us.  78 KB of LDS and 229 registers
// leave two waves a SIMD, whose vector units are busy half the time (with cutting
// float32 values in three, masks, and addresses), in a chain of eight parts between
// barriers.  With the parts left out one at a time: tiles of dP and dA -19 us, the
// inverse -16, results -12, loads ahead -10, the gates' end -5.  64 consoles in
// float32: 64 us, of which the float32 matrix instructions are 21.
#include "mem_delta_tile.h"

namespace nesle::mem {
namespace {

// 32 columns of a state or its gradient, transposed: [value column][key].  In
// float32, which takes less room than three planes; a reader cuts its own.
template <int DP>
using Slab = F32Math::Tile<32, DP, 1>;

template <typename T, int DP>
struct GradTile : ChunkTile<T, typename MathOf<T, DP>::gradient, DP, Slab<DP>> {
    using Base = ChunkTile<T, typename MathOf<T, DP>::gradient, DP, Slab<DP>>;
    using M = typename Base::M;
    typename M::template Tile<kChunk, DP, M::kIn, 8> dout;
    // Transposed: [value column][token].  With rows of 18 and 42 words (mod 64)
    // the transposing reads meet no bank twice.
    typename M::template Tile<DP, kChunk, kFull, 4> u;
    union {
        typename M::template Tile<DP, kChunk, kFull, 4> dr;
        Results<T, DP> keys[2];                            // dQ and dK, once dR has been read
    };
    Slab<DP> slab;
    float row_beta[Base::kWaves][kChunk], row_gate[Base::kWaves][kChunk], row_after[Base::kWaves][kChunk];
    float place_beta[3][16], cross[4][16];     // of a tile: sums over columns; pairs that cross a token
    float whole[Base::kWaves];
};

template <typename T, int DP, bool WIDE>
__global__ void __launch_bounds__(DP * 4, 2) delta_backward_kernel(DeltaArgs<T> a) {
    using Tile = GradTile<T, DP>;
    using M = typename Tile::M;
    using In = Rows<T, WIDE>;
    constexpr int KT = Tile::KT, KP = Tile::KP, kWaves = Tile::kWaves, kPlaces = (3 + kWaves - 2) / (kWaves - 1);     // tiles of a wave
    __shared__ Tile sh;
    const Lane<DP> first;
    const std::uint32_t env = blockIdx.x / a.hv, h = blockIdx.x % a.hv, hk = h / a.group;
    const std::size_t head = blockIdx.x, state_size = static_cast<std::size_t>(a.dk_dim) * a.dv_dim;
    const std::int64_t v_step = static_cast<std::int64_t>(a.batch) * a.hv * a.dv_dim;
    const f4 zero = {0, 0, 0, 0};

    f4 dS[KT];
    Tile::load_state(a, a.dstate_out, head, first, dS);
    sh.start(first);

    Ahead<T, DP, WIDE> in;
    std::uint32_t dout[In::kWords];
    const auto fetch = [&](std::uint32_t end, const Lane<DP>& at) {
        const std::uint32_t start = (end - 1) / kChunk * kChunk;
        in.fetch(a, start, static_cast<int>(end - start), env, h, at);
        in.part(a.dout, a.dv_dim, start, static_cast<int>(end - start), env, h, at, dout);
    };
    // As in the forward, the wave that inverts (turn 0) reads the states first
    // and has no tile; the last one stages the next chunk's gates meanwhile.
    const int turn = (first.wave + static_cast<int>(blockIdx.x)) % kWaves;
    if (a.steps != 0) {
        fetch(a.steps, first);
        if (turn == kWaves - 1) sh.gates[0].stage(in, static_cast<int>((a.steps - 1) % kChunk) + 1, first.lane);
    }
    int which = 0;
    for (std::uint32_t t1 = a.steps; t1 > 0;) {
        const Lane<DP> at = Lane<DP>::anew();
        const int r = at.r, g = at.g;
        Gates& now = sh.gates[which];
        // A chunk from its start to t1.  Where it drops the state, gammas and
        // decays are zero across that token, as in the forward.
        const std::uint32_t start = (t1 - 1) / kChunk * kChunk;
        const int n = static_cast<int>(t1 - start);
        const std::uint32_t drops = in.drops();
        const float* from = (drops & 1u) ? nullptr : start == 0 ? a.state
                                                   : a.saved + (start / kChunk - 1) * state_size * a.batch * a.hv;
        const bool of_chunk = start != 0;          // kept by the forward as [v_dim][k_dim]; else the initial state
        f4 S[KT];
        if (of_chunk && from != nullptr) Tile::kept(a, from, head, at, S);
        else Tile::load_state(a, from, head, at, S);

        sh.stage(in, at);
        sh.dout.put8(at.key_row, at.key_col, dout);
        t1 = start;
        if (t1 > 0) fetch(t1, at);
        __syncthreads();
        f4 kk[kPlaces], qk[kPlaces], ks[2] = {}, qs[2] = {}, kds[2] = {};
        const auto read_states = [&] {
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                const auto s = M::full(S[2 * i], S[2 * i + 1]), ds = M::full(dS[2 * i], dS[2 * i + 1]);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const auto key = sh.k.rows(16 * m, i, r, g);
                    ks[m] = M::mul(key, s, ks[m]);
                    kds[m] = M::mul(key, ds, kds[m]);
                    qs[m] = M::mul(sh.q.rows(16 * m, i, r, g), s, qs[m]);
                }
            }
        };
        if (turn == 0 || turn > 3) {
            read_states();
        } else {
#pragma unroll
            for (int j = 0; j < kPlaces; ++j)
                if (turn - 1 + j * (kWaves - 1) < 3) sh.products(turn - 1 + j * (kWaves - 1), a.scale, now, at, kk[j], qk[j]);
        }
        __syncthreads();
        if (turn == 0) sh.invert(now, at);
        else if (turn <= 3) read_states();
        which ^= 1;
        if (turn == kWaves - 1 && t1 > 0) sh.gates[which].stage(in, kChunk, at.lane);
        f4 V[2], dO[2], Y[2], gam[2], dec[2], beta[2];
        M::values(sh.v.cols(0, 16 * at.wave, r, g), V);
        const auto grad = sh.dout.cols(0, 16 * at.wave, r, g);
        M::values(grad, dO);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            gam[m] = now.of_rows(now.gamma, m, g);
            dec[m] = now.of_rows(now.decay, m, g);
            beta[m] = now.of_rows(now.beta, m, g);
            Y[m] = V[m] - gam[m] * ks[m];
        }
        const auto right = M::full(beta[0] * Y[0], beta[1] * Y[1]);
        __syncthreads();
        f4 U[2], dU[2], dR[2], X[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            U[m] = M::mul(sh.t.rows(16 * m, 0, r, g), right, zero);
            dU[m] = M::mul(sh.p.cols(0, 16 * m, r, g), grad, dec[m] * kds[m]);
        }
        const auto du = M::full(dU[0], dU[1]);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            dR[m] = M::mul(sh.t.cols(0, 16 * m, r, g), du, zero);
            X[m] = beta[m] * gam[m] * dR[m];
            sh.u.put4(at.col, 16 * m + 4 * g, U[m]);
            sh.dr.put4(at.col, 16 * m + 4 * g, dR[m]);
        }
        const In dv(a.dv + static_cast<std::int64_t>(start) * v_step + head * a.dv_dim, v_step);
        const f4 dV[2] = {beta[0] * dR[0], beta[1] * dR[1]};
        sh.results.put(dv, static_cast<int>(a.dv_dim), n, at, dV);

        // Sums over the value dimension of dbeta and the gates, this wave's share.
        const float last = now.gamma[kChunk - 1];
        float whole = 0.0f;
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) whole += dS[i][j] * S[i][j];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const f4 by_beta = dR[m] * Y[m];
            const f4 e = dec[m] * kds[m] * U[m];
            const f4 by_gate = gam[m] * a.scale * dO[m] * qs[m] - X[m] * ks[m];
            const float sb = sum16_of(by_beta), sg = sum16_of(by_gate), se = sum16_of(e);
            if (r % 4 == 0) {
                sh.row_beta[at.wave][16 * m + 4 * g + r / 4] = sb;
                sh.row_gate[at.wave][16 * m + 4 * g + r / 4] = sg;
                sh.row_after[at.wave][16 * m + 4 * g + r / 4] = se;
            }
        }
        whole = over_groups(sum16(whole)) * last;
        if (at.lane == 0) sh.whole[at.wave] = whole;

        // The state's gradient before the chunk (dS itself is still needed).
        f4 before[KT];
        {
            const auto read = M::full(gam[0] * a.scale * dO[0], gam[1] * a.scale * dO[1]);
            const auto held = M::full(-X[0], -X[1]);
#pragma unroll
            for (int i = 0; i < KT; ++i) {
                before[i] = M::mul(sh.q.cols(0, 16 * i, r, g), read, drops != 0 ? zero : dS[i] * last);
                before[i] = M::mul(sh.k.cols(0, 16 * i, r, g), held, before[i]);
            }
        }
        __syncthreads();
        sh.results.flush(dv, static_cast<int>(a.dv_dim), n, at);

        // dP and dA by tiles; P's space becomes M1 and the inverse's M2.
#pragma unroll
        for (int j = 0; j < kPlaces; ++j) {
            const int place = turn - 1 + j * (kWaves - 1);
            if (place < 0 || place >= 3) break;
            const int mi = Tile::first_row(place), nj = Tile::first_col(place);
            f4 dP = zero, dA = zero;
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                const auto uu = sh.u.cols(32 * i, nj, r, g);
                dP = M::mul_apart(sh.dout.rows(mi, i, r, g), uu, dP);
                dA = M::mul_apart(sh.dr.cols(32 * i, mi, r, g), uu, dA);
            }
            // With token t = 16 x + r in lane r: pairs of this tile with
            // j < t <= i.  Tile (16, 0) has them for both halves of t.
            float cross = 0.0f, cross_below = 0.0f;
            f4 by_a, pairs;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = mi + 4 * g + i, c = nj + r;
                const float L = now.ratio(row, c), b = now.beta[row];
                sh.p.put(row, c, c <= row ? a.scale * L * dP[i] : 0.0f);
                sh.t.put(row, c, c < row ? -b * L * dA[i] : 0.0f);
                by_a[i] = -dA[i] * kk[j][i];
                pairs[i] = c < row ? dP[i] * qk[j][i] + b * by_a[i] : 0.0f;
                const float before_t = sum_below(pairs[i]);
                cross += place == 1 || row >= c ? before_t : 0.0f;
            }
            const float sb = sum16_of(by_a);
            if (r % 4 == 0) sh.place_beta[place][4 * g + r / 4] = sb;
            cross = over_groups(cross);
            if (g == 0) sh.cross[place][r] = cross;
            if (place == 1) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float all = sum16(pairs[i]);
                    if (4 * g + i >= r) cross_below += all;
                }
                cross_below = over_groups(cross_below);
                if (g == 0) sh.cross[3][r] = cross_below;
            }
        }
        // dO S^T and dR S^T, then U dS^T: this wave's 16 key columns.  The waves
        // that hold 32 columns put them in one of two places in turn; the second
        // is free once all have passed a barrier.
        f4 dQ[2] = {}, dK[2] = {}, drs[2] = {};
        const auto pass = [&](const f4 (&x)[KT], int i, int turns, const auto& use) {
            const auto put = [&](auto& to) {
                if (at.wave / 2 == i)
#pragma unroll
                    for (int j = 0; j < KT; ++j) to.put4(16 * (at.wave % 2) + r, 16 * j + 4 * g, x[j]);
                __syncthreads();
                const auto held = to.cols(0, 16 * at.wave, r, g);
                use(i, M::full(held.a, held.b));
            };
            if (turns % 2 == 0) put(sh.slab);
            else put(sh.later);
        };
        if (KP == 1 || from != nullptr) {
#pragma unroll
            for (int i = 0; i < KP; ++i)
                pass(S, i, i, [&](int i, const auto& s) {
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        dQ[m] = M::mul(sh.dout.rows(16 * m, i, r, g), s, dQ[m]);
                        drs[m] = M::mul(sh.dr.cols(32 * i, 16 * m, r, g), s, drs[m]);
                    }
                });
        }
#pragma unroll
        for (int i = 0; i < KP; ++i)
            pass(dS, i, KP + i, [&](int i, const auto& ds) {
#pragma unroll
                for (int m = 0; m < 2; ++m) dK[m] = M::mul(sh.u.cols(32 * i, 16 * m, r, g), ds, dK[m]);
            });
        const auto key = sh.k.cols(0, 16 * at.wave, r, g), query = sh.q.cols(0, 16 * at.wave, r, g);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            dQ[m] = M::mul(sh.p.rows(16 * m, 0, r, g), key, gam[m] * a.scale * dQ[m]);
            dK[m] = M::mul(sh.p.cols(0, 16 * m, r, g), query, dec[m] * dK[m] - beta[m] * gam[m] * drs[m]);
            dK[m] = M::mul(sh.t.rows(16 * m, 0, r, g), key, dK[m]);
            dK[m] = M::mul(sh.t.cols(0, 16 * m, r, g), key, dK[m]);
        }
        const std::int64_t token = static_cast<std::int64_t>(start) * a.batch + env;
        const std::int64_t key_step = static_cast<std::int64_t>(a.batch) * a.hk * a.dk_dim;
        const In dq(a.dq + (token * a.hk + hk) * a.dk_dim, key_step), dk(a.dk + (token * a.hk + hk) * a.dk_dim, key_step);
        if (a.group == 1) {
            sh.keys[0].put(dq, static_cast<int>(a.dk_dim), n, at, dQ);
            sh.keys[1].put(dk, static_cast<int>(a.dk_dim), n, at, dK);
        } else {            // one share a value head, added up afterwards
            const std::int64_t step = static_cast<std::int64_t>(a.batch) * a.hv * a.dk_dim;
            float* share = a.scratch + (token * a.hv + h) * a.dk_dim;
            Results<float, DP>{}.put(Rows<float, WIDE>(share, step), static_cast<int>(a.dk_dim), n, at, dQ);
            Results<float, DP>{}.put(Rows<float, WIDE>(share + a.steps * step, step), static_cast<int>(a.dk_dim), n, at, dK);
        }
        if (at.wave == 0) {            // one token a lane
            const int t = at.lane % kChunk, i = t % 16;
            float db = t < 16 ? sh.place_beta[0][i] : sh.place_beta[1][i] + sh.place_beta[2][i];
            float dg = t < 16 ? sh.cross[0][i] + sh.cross[1][i] : sh.cross[2][i] + sh.cross[3][i];
            float from_t = 0.0f, to_t = 0.0f;
            for (int w = 0; w < kWaves; ++w) {
                db += sh.row_beta[w][t];
                from_t += sh.row_gate[w][t];
                to_t += sh.row_after[w][t];
                dg += sh.whole[w];
            }
#pragma unroll
            for (int d = 1; d < kChunk; d *= 2) {
                const float above = __shfl_down(from_t, d), below = __shfl_up(to_t, d);
                if (t + d < kChunk) from_t += above;
                if (t >= d) to_t += below;
            }
            to_t = __shfl_up(to_t, 1);
            dg += from_t + (t > 0 ? to_t : 0.0f);
            if (at.lane < n) {
                const std::size_t to = ((static_cast<std::size_t>(start) + t) * a.batch + env) * a.hv + h;
                a.dbeta[to] = db;
                a.dg[to] = drops >> t & 1u ? 0.0f : dg;
            }
        }
#pragma unroll
        for (int i = 0; i < KT; ++i) dS[i] = (drops & 1u) ? zero : before[i];
        __syncthreads();
        if (a.group == 1) {
            sh.keys[0].flush(dq, static_cast<int>(a.dk_dim), n, at);
            sh.keys[1].flush(dk, static_cast<int>(a.dk_dim), n, at);
        }
    }
    if (a.dstate != nullptr) Tile::store_state(a, a.dstate, head, Lane<DP>::anew(), dS);
}

// dq and dk of a key head: the sum of its value heads' shares.
template <typename T>
__global__ void __launch_bounds__(256) delta_share_sum(DeltaArgs<T> a, std::uint64_t quads) {
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

template <typename T>
int backward(const char* who, const nesle_delta_args& x, hipStream_t s) {
    const DeltaArgs<T> a = delta_args<T>(x);
    const dim3 grid(a.batch * a.hv);
    const std::uint32_t dim = wide_rows(x) ? 0 : padded_dim(x);
    switch (dim) {
        case 0: hipLaunchKernelGGL((delta_backward_kernel<T, 128, true>), grid, dim3(512), 0, s, a); break;
        case 32: hipLaunchKernelGGL((delta_backward_kernel<T, 32, false>), grid, dim3(128), 0, s, a); break;
        case 64: hipLaunchKernelGGL((delta_backward_kernel<T, 64, false>), grid, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL((delta_backward_kernel<T, 128, false>), grid, dim3(512), 0, s, a); break;
    }
    if (a.group > 1 && a.steps != 0) {
        const std::uint64_t quads = static_cast<std::uint64_t>(a.steps) * a.batch * a.hk * a.dk_dim / 4;
        const std::uint64_t want = (2 * quads + 255) / 256;
        hipLaunchKernelGGL(delta_share_sum<T>, dim3(static_cast<std::uint32_t>(want < 4096 ? want : 4096)), dim3(256), 0, s,
                           a, quads);
    }
    return launched(who);
}

}  // namespace
}  // namespace nesle::mem

using namespace nesle::mem;

extern "C" {

std::uint64_t nesle_delta_scratch_floats(const nesle_delta_args* a) {
    if (a == nullptr || a->k_heads == 0 || a->v_heads <= a->k_heads) return 0;
    return 2ull * a->steps * a->batch * a->v_heads * a->k_dim;
}

int nesle_delta_backward(const nesle_delta_args* a, void* stream) {
    const char* who = "nesle_delta_backward";
    int rc = check_delta(who, a);
    if (rc != NESLE_OK || a->batch == 0) return rc;
    if (a->steps != 0) {
        rc = check_delta_inputs(who, a);
        if (rc != NESLE_OK) return rc;
        if (!a->dout.data || !a->dq || !a->dk || !a->dv || !a->dg || !a->dbeta ||
            (!a->saved && nesle_delta_saved_floats(a) != 0) || (!a->scratch && nesle_delta_scratch_floats(a) != 0))
            return refuse(who, "null device pointer");
    }
    const auto s = static_cast<hipStream_t>(stream);
    return a->dtype == NESLE_MEM_F32 ? backward<float>(who, *a, s) : backward<bf16>(who, *a, s);
}

}  // extern "C"
