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
// registers (mem_common.h), so only what all columns share goes through LDS:
// K, Q, A, P and the inverses of (I + A)'s two diagonal tiles.  Those are
// found by substitution: neighbouring frames have nearly equal keys, where the
// powers of A grow to thousands and a product form of the inverse cancels.
//
// Float32 throughout, products by v_mfma_f32_16x16x4_f32: the state and the
// gates' gradients are float32 results whatever the inputs' type.
//
// A chunk ends early at a token that drops the state (its episode ended) and
// before one that holds a value that is not finite, so that neither reaches a
// token it must not (a product with a masked zero would carry NaN).
#include "mem_delta.h"
#include "mem_delta_tile.h"

namespace nesle::mem {
namespace {

template <typename T, int DP>
__global__ void __launch_bounds__(DP * 4) delta_forward_kernel(DeltaArgs<T> a) {
    using Tile = ChunkTile<T, DP>;
    constexpr int KT = DP / 16;                 // tiles of the key dimension
    __shared__ Tile sh;
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, r = lane % 16, g4 = lane / 16;
    const std::uint32_t env = blockIdx.x / a.hv, h = blockIdx.x % a.hv, hk = h / a.group;
    const std::size_t head = blockIdx.x;
    const unsigned col = 16 * wave + r;
    const bool in_col = col < a.dv_dim;

    f4 S[KT];
    Tile::load_state(a, a.state, head, col, g4, S);
    if (tid == 0) sh.bad = 0;
    __syncthreads();

    for (std::uint32_t t0 = 0; t0 < a.steps;) {
        if (t0 != 0 && t0 % kChunk == 0 && a.saved != nullptr)
            Tile::put_saved(a, t0 / kChunk - 1, head, wave, lane, S);
        if (drops(a, t0, env, h))
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] = f4{0, 0, 0, 0};
        int n = Tile::extent(a, t0, env, h, lane);
        f4 V[2];
        for (;;) {
            sh.stage_keys(a, t0, n, env, hk, tid);
            if (wave == 0) sh.stage_gates(a, t0, n, env, h, lane);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 16 * m + 4 * g4 + i;
                    float x = 0.0f;
                    if (row < n && in_col) x = static_cast<float>(a.v.row(t0 + row, env, h)[col]);
                    if (!(fabsf(x) < INFINITY)) atomicOr(&sh.bad, 1u << row);
                    V[m][i] = x;
                }
            __syncthreads();
            const unsigned bad = sh.bad;
            if (bad == 0 || n == 1) break;
            // Rare: stage again, up to the first such token, or it alone.
            n = (bad & 1u) ? 1 : __ffs(bad) - 1;
            __syncthreads();
            if (tid == 0) sh.bad = 0;
            __syncthreads();
        }
        sh.products(a.scale, wave, r, g4);
        __syncthreads();
        if (tid == 0) sh.bad = 0;
        if (wave < 2) sh.invert(wave, r, g4);

        // K S and Q S for this wave's columns.
        f4 ks[2] = {}, qs[2] = {};
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                ks[m] = mma(along<Tile::kStride>(sh.k, 16 * m, 16 * i, r, g4), S[i], ks[m]);
                qs[m] = mma(along<Tile::kStride>(sh.q, 16 * m, 16 * i, r, g4), S[i], qs[m]);
            }
        f4 R[2], gam[2], dec[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            gam[m] = *reinterpret_cast<const f4*>(&sh.gamma[16 * m + 4 * g4]);
            dec[m] = *reinterpret_cast<const f4*>(&sh.decay[16 * m + 4 * g4]);
            const f4 b = *reinterpret_cast<const f4*>(&sh.beta[16 * m + 4 * g4]);
            R[m] = b * (V[m] - gam[m] * ks[m]);
        }
        __syncthreads();
        f4 U[2];
        sh.solve(R, U, r, g4);
        const f4 zero = {0, 0, 0, 0};
        f4 O[2];
        O[0] = mma(along<Tile::kSmall>(sh.p, 0, 0, r, g4), U[0], qs[0] * gam[0] * a.scale);
        O[1] = mma(along<Tile::kSmall>(sh.p, 16, 0, r, g4), U[0], qs[1] * gam[1] * a.scale);
        O[1] = mma(along<Tile::kSmall>(sh.p, 16, 16, r, g4), U[1], O[1]);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 16 * m + 4 * g4 + i;
                if (row < n && in_col)
                    a.out[((static_cast<std::size_t>(t0) + row) * a.batch + env) * a.hv * a.dv_dim + h * a.dv_dim + col] =
                        static_cast<T>(O[m][i]);
            }
        const float last = sh.gamma[kChunk - 1];
        const f4 W[2] = {U[0] * dec[0], U[1] * dec[1]};
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            f4 add = mma(down<Tile::kStride>(sh.k, 0, 16 * i, r, g4), W[0], zero);
            add = mma(down<Tile::kStride>(sh.k, 16, 16 * i, r, g4), W[1], add);
            S[i] = S[i] * last + add;
        }
        t0 += n;
        __syncthreads();
    }
    Tile::store_state(a, a.state_out, head, col, g4, S);
}

template <typename T>
int forward(const char* who, const nesle_delta_args& x, hipStream_t s) {
    const DeltaArgs<T> a = delta_args<T>(x);
    const dim3 grid(a.batch * a.hv);
    switch (padded_dim(x)) {
        case 32: hipLaunchKernelGGL((delta_forward_kernel<T, 32>), grid, dim3(128), 0, s, a); break;
        case 64: hipLaunchKernelGGL((delta_forward_kernel<T, 64>), grid, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL((delta_forward_kernel<T, 128>), grid, dim3(512), 0, s, a); break;
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
    const std::uint64_t d = padded_dim(*a);
    return chunks * a->batch * a->v_heads * d * d;
}

int nesle_delta_forward(const nesle_delta_args* a, void* stream) {
    const char* who = "nesle_delta_forward";
    int rc = check_delta(who, a);
    if (rc != NESLE_OK || a->batch == 0) return rc;
    if (!a->state_out) return refuse(who, "null device pointer");
    if (a->steps != 0) {
        rc = check_delta_inputs(who, a);
        if (rc != NESLE_OK) return rc;
        if (!a->out) return refuse(who, "null device pointer");
    }
    const auto s = static_cast<hipStream_t>(stream);
    return a->dtype == NESLE_MEM_F32 ? forward<float>(who, *a, s) : forward<bf16>(who, *a, s);
}

}  // extern "C"
