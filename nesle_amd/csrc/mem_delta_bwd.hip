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
// A gate enters through the G_i that include it.  dG_i is the row sum less the
// column sum of dP P + dA A, plus gamma_i (scale dO.QS - beta dR.KS), less
// e_i = E_i (K dS).U; the last G also has gamma_last <dS, S> + sum of e.
// dg_t is the sum of dG_i over i >= t, and zero where the state is dropped.
//
// The part over value columns runs a wave per 16 columns, as in the forward;
// the part that sums over the value dimension runs a wave per 16 key columns,
// on U, dR, dO, S and dS written to LDS (the states in slabs of 64 columns).
// No atomics: the sums over waves are added in a fixed order.
#include "mem_delta.h"
#include "mem_delta_tile.h"

namespace nesle::mem {
namespace {

template <typename T, int DP>
struct GradTile : ChunkTile<T, DP> {
    using Base = ChunkTile<T, DP>;
    static constexpr int kSlab = DP < 64 ? DP : 64;        // columns of a state slab
    static constexpr int kSlabStride = kSlab + 4;
    alignas(16) float dout[kChunk * Base::kStride];
    alignas(16) float u[kChunk * Base::kStride];
    alignas(16) float dr[kChunk * Base::kStride];
    alignas(16) float slab[DP * kSlabStride];              // [key][value column]
    alignas(16) float m1[kChunk * Base::kSmall];
    alignas(16) float m2[kChunk * Base::kSmall];
    float row_beta[Base::kWaves][kChunk], row_gate[Base::kWaves][kChunk];
    float last_gate[Base::kWaves];
};

__device__ inline float sum16(float v) {
    for (int d = 1; d < 16; d *= 2) v += __shfl_xor(v, d);
    return v;
}

template <typename T, int DP>
__global__ void __launch_bounds__(DP * 4, 2) delta_backward_kernel(DeltaArgs<T> a) {
    using Tile = GradTile<T, DP>;
    constexpr int KT = DP / 16, ST = Tile::kStride, SM = Tile::kSmall, SL = Tile::kSlabStride;
    constexpr int kPerSlab = Tile::kSlab / 16;              // waves whose columns make a slab
    __shared__ Tile sh;
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, r = lane % 16, g4 = lane / 16;
    const std::uint32_t env = blockIdx.x / a.hv, h = blockIdx.x % a.hv, hk = h / a.group;
    const std::size_t head = blockIdx.x;
    const unsigned col = 16 * wave + r;
    const bool in_v = col < a.dv_dim, in_k = col < a.dk_dim;
    const f4 zero = {0, 0, 0, 0};

    f4 dS[KT];
    Tile::load_state(a, a.dstate_out, head, col, g4, dS);

    for (std::uint32_t t1 = a.steps; t1 > 0;) {
        // The chunk ends at t1; it starts at the last multiple of the chunk
        // length, or at the last token after that which drops the state.
        const std::uint32_t start = (t1 - 1) / kChunk * kChunk;
        const bool cut = lane < static_cast<int>(t1 - start) && drops(a, start + lane, env, h);
        const unsigned long long cuts = __ballot(cut);
        const bool dropped = cuts != 0;
        const std::uint32_t t0 = dropped ? start + 63 - __clzll(static_cast<long long>(cuts)) : start;
        const int n = static_cast<int>(t1 - t0);

        f4 S[KT];
        if (dropped)
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] = zero;
        else if (t0 == 0)
            Tile::load_state(a, a.state, head, col, g4, S);
        else
            Tile::get_saved(a, t0 / kChunk - 1, head, wave, lane, S);

        sh.stage_keys(a, t0, n, env, hk, tid);
        if (wave == 0) sh.stage_gates(a, t0, n, env, h, lane);
        f4 V[2], dO[2];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 16 * m + 4 * g4 + i;
                const bool in = row < n && in_v;
                V[m][i] = in ? static_cast<float>(a.v.row(t0 + row, env, h)[col]) : 0.0f;
                dO[m][i] = in ? static_cast<float>(a.dout.row(t0 + row, env, h)[col]) : 0.0f;
                sh.dout[row * ST + col] = dO[m][i];
            }
        __syncthreads();
        sh.products(a.scale, wave, r, g4);
        __syncthreads();
        if (wave < 2) sh.invert(wave, r, g4);

        f4 ks[2] = {}, qs[2] = {}, kds[2] = {};
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const f4 kk = along<ST>(sh.k, 16 * m, 16 * i, r, g4);
                ks[m] = mma(kk, S[i], ks[m]);
                kds[m] = mma(kk, dS[i], kds[m]);
                qs[m] = mma(along<ST>(sh.q, 16 * m, 16 * i, r, g4), S[i], qs[m]);
            }
        f4 Y[2], R[2], U[2], dU[2], dR[2], gam[2], dec[2], beta[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            gam[m] = *reinterpret_cast<const f4*>(&sh.gamma[16 * m + 4 * g4]);
            dec[m] = *reinterpret_cast<const f4*>(&sh.decay[16 * m + 4 * g4]);
            beta[m] = *reinterpret_cast<const f4*>(&sh.beta[16 * m + 4 * g4]);
            Y[m] = V[m] - gam[m] * ks[m];
            R[m] = beta[m] * Y[m];
        }
        __syncthreads();
        sh.solve(R, U, r, g4);
        dU[0] = mma(down<SM>(sh.p, 0, 0, r, g4), dO[0], dec[0] * kds[0]);
        dU[0] = mma(down<SM>(sh.p, 16, 0, r, g4), dO[1], dU[0]);
        dU[1] = mma(down<SM>(sh.p, 16, 16, r, g4), dO[1], dec[1] * kds[1]);
        // (I + A)^T dR = dU, last tile first; the rows of A carry beta.
        dR[1] = mma(down<20>(sh.t[1], 0, 0, r, g4), dU[1], zero);
        const f4 above = mma(down<SM>(sh.a, 16, 0, r, g4) * beta[1], dR[1], zero);
        dR[0] = mma(down<20>(sh.t[0], 0, 0, r, g4), dU[0] - above, zero);

        // Sums over the value dimension of dbeta and the gates, this wave's share.
        const float last = sh.gamma[kChunk - 1];
        float last_gate = 0.0f;
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) last_gate += dS[i][j] * S[i][j];
        last_gate *= last;
        f4 X[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            X[m] = beta[m] * gam[m] * dR[m];
            const f4 by_beta = dR[m] * Y[m];
            const f4 e = dec[m] * kds[m] * U[m];
            const f4 by_gate = gam[m] * a.scale * dO[m] * qs[m] - X[m] * ks[m] - e;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                last_gate += e[i];
                const int row = 16 * m + 4 * g4 + i;
                const float sb = sum16(by_beta[i]), sg = sum16(by_gate[i]);
                if (r == 0) {
                    sh.row_beta[wave][row] = sb;
                    sh.row_gate[wave][row] = sg;
                }
                if (row < n && in_v)
                    a.dv[((static_cast<std::size_t>(t0) + row) * a.batch + env) * a.hv * a.dv_dim + h * a.dv_dim + col] =
                        static_cast<T>(beta[m][i] * dR[m][i]);
                sh.u[row * ST + col] = U[m][i];
                sh.dr[row * ST + col] = dR[m][i];
            }
        }
        last_gate = sum16(last_gate);
        last_gate += __shfl_xor(last_gate, 16);
        last_gate += __shfl_xor(last_gate, 32);
        if (lane == 0) sh.last_gate[wave] = last_gate;

        // The state's gradient before the chunk (dS itself is still needed).
        f4 before[KT];
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            f4 add = mma(down<ST>(sh.q, 0, 16 * i, r, g4), gam[0] * a.scale * dO[0], dS[i] * last);
            add = mma(down<ST>(sh.q, 16, 16 * i, r, g4), gam[1] * a.scale * dO[1], add);
            add = mma(down<ST>(sh.k, 0, 16 * i, r, g4), -X[0], add);
            before[i] = mma(down<ST>(sh.k, 16, 16 * i, r, g4), -X[1], add);
        }
        __syncthreads();

        // dP and dA by tiles; a and p become the gates' terms, m1 and m2 what
        // multiplies K and Q.
        for (int place = wave; place < 3; place += Tile::kWaves) {
            const int mi = place != 0 ? 16 : 0, nj = place == 2 ? 16 : 0;
            f4 dP = zero, dA = zero;
#pragma unroll
            for (int i = 0; i < KT; ++i) {
                const f4 uu = along<ST>(sh.u, nj, 16 * i, r, g4);
                dP = mma(along<ST>(sh.dout, mi, 16 * i, r, g4), uu, dP);
                dA = mma(along<ST>(sh.dr, mi, 16 * i, r, g4), uu, dA);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = mi + 4 * g4 + i, c = nj + r, at = row * SM + c;
                const float L = c <= row ? sh.ratio(row, c) : 0.0f;
                sh.m1[at] = c <= row ? a.scale * L * dP[i] : 0.0f;
                sh.m2[at] = c < row ? -sh.beta[row] * L * dA[i] : 0.0f;
                sh.p[at] = c <= row ? dP[i] * sh.p[at] : 0.0f;
                sh.a[at] = c < row ? -dA[i] * sh.a[at] : 0.0f;
            }
        }
        // dO S^T, dR S^T, U dS^T: this wave's 16 key columns.
        f4 dos[2] = {}, drs[2] = {}, uds[2] = {};
#pragma unroll
        for (int s = 0; s < 2 * KT / kPerSlab; ++s) {
            const bool of_grad = s >= KT / kPerSlab;
            const int first = (s % (KT / kPerSlab)) * kPerSlab;     // first wave of the slab's columns
            if (wave >= first && wave < first + kPerSlab)
#pragma unroll
                for (int i = 0; i < KT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        sh.slab[(16 * i + 4 * g4 + j) * SL + 16 * (wave - first) + r] = of_grad ? dS[i][j] : S[i][j];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kPerSlab; ++i) {
                const f4 b = along<SL>(sh.slab, 16 * wave, 16 * i, r, g4);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const int c = 16 * (first + i);
                    if (of_grad) {
                        uds[m] = mma(along<ST>(sh.u, 16 * m, c, r, g4), b, uds[m]);
                    } else {
                        dos[m] = mma(along<ST>(sh.dout, 16 * m, c, r, g4), b, dos[m]);
                        drs[m] = mma(along<ST>(sh.dr, 16 * m, c, r, g4), b, drs[m]);
                    }
                }
            }
            __syncthreads();
        }
        f4 dQ[2], dK[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            dQ[m] = gam[m] * a.scale * dos[m];
            dK[m] = dec[m] * uds[m] - beta[m] * gam[m] * drs[m];
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {                               // the tile of tokens summed over
            const f4 kx = down<ST>(sh.k, 16 * x, 16 * wave, r, g4), qx = down<ST>(sh.q, 16 * x, 16 * wave, r, g4);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if (x <= m) {
                    dQ[m] = mma(along<SM>(sh.m1, 16 * m, 16 * x, r, g4), kx, dQ[m]);
                    dK[m] = mma(along<SM>(sh.m2, 16 * m, 16 * x, r, g4), kx, dK[m]);
                }
                if (x >= m) {
                    dK[m] = mma(down<SM>(sh.m1, 16 * x, 16 * m, r, g4), qx, dK[m]);
                    dK[m] = mma(down<SM>(sh.m2, 16 * x, 16 * m, r, g4), kx, dK[m]);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 16 * m + 4 * g4 + i;
                if (row >= n || !in_k) continue;
                const std::size_t at = (static_cast<std::size_t>(t0) + row) * a.batch + env;
                if (a.group == 1) {
                    a.dq[(at * a.hk + hk) * a.dk_dim + col] = static_cast<T>(dQ[m][i]);
                    a.dk[(at * a.hk + hk) * a.dk_dim + col] = static_cast<T>(dK[m][i]);
                } else {            // one share a value head, added up afterwards
                    const std::size_t all = static_cast<std::size_t>(a.steps) * a.batch * a.hv * a.dk_dim;
                    a.scratch[(at * a.hv + h) * a.dk_dim + col] = dQ[m][i];
                    a.scratch[all + (at * a.hv + h) * a.dk_dim + col] = dK[m][i];
                }
            }
        if (wave == 0) {            // one token a lane
            const int t = lane % kChunk;
            float db = 0.0f, gate = 0.0f;
            for (int c = 0; c <= t; ++c) {
                db += sh.a[t * SM + c];
                gate += sh.p[t * SM + c];
            }
            gate += sh.beta[t] * db;
            for (int c = t; c < kChunk; ++c) gate -= sh.p[c * SM + t] + sh.beta[c] * sh.a[c * SM + t];
            for (int w = 0; w < Tile::kWaves; ++w) {
                db += sh.row_beta[w][t];
                gate += sh.row_gate[w][t];
            }
            if (t == kChunk - 1)
                for (int w = 0; w < Tile::kWaves; ++w) gate += sh.last_gate[w];
            double sum = gate;                                      // of the tokens from t on
#pragma unroll
            for (int d = 1; d < kChunk; d *= 2) {
                const double above = __shfl_down(sum, d);
                if (t + d < kChunk) sum += above;
            }
            if (lane < n) {
                const std::size_t at = ((static_cast<std::size_t>(t0) + t) * a.batch + env) * a.hv + h;
                a.dbeta[at] = db;
                a.dg[at] = dropped && t == 0 ? 0.0f : static_cast<float>(sum);
            }
        }
#pragma unroll
        for (int i = 0; i < KT; ++i) dS[i] = dropped ? zero : before[i];
        t1 = t0;
        __syncthreads();
    }
    if (a.dstate != nullptr) Tile::store_state(a, a.dstate, head, col, g4, dS);
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
    switch (padded_dim(x)) {
        case 32: hipLaunchKernelGGL((delta_backward_kernel<T, 32>), grid, dim3(128), 0, s, a); break;
        case 64: hipLaunchKernelGGL((delta_backward_kernel<T, 64>), grid, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL((delta_backward_kernel<T, 128>), grid, dim3(512), 0, s, a); break;
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
