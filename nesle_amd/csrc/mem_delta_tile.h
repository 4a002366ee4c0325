// mem_delta_tile.h -- one chunk of the gated delta rule in LDS: what the
// forward and the gradient kernels both make of it.
#pragma once

#include "mem_delta.h"

namespace nesle::mem {

template <typename T, int DP>          // DP: head dimensions padded to 32, 64 or 128; DP / 16 waves
struct ChunkTile {
    static constexpr int kStride = DP + 4, kSmall = kChunk + 4;
    static constexpr int KT = DP / 16, kWaves = DP / 16;

    alignas(16) float k[kChunk * kStride];
    alignas(16) float q[kChunk * kStride];
    alignas(16) float a[kChunk * kSmall];      // A without beta: L_ij (k_i . k_j), j < i; else 0
    alignas(16) float p[kChunk * kSmall];      // P: scale L_ij (q_i . k_j), j <= i; else 0
    alignas(16) float t[2][16 * 20];           // inverses of (I + A)'s diagonal tiles
    alignas(16) double G[kChunk];              // running sum of g: differences of it are taken
    alignas(16) float gamma[kChunk], decay[kChunk], beta[kChunk];
    unsigned bad;                              // tokens with a value that is not finite

    // ---- states: lane (r, g4) of a wave holds S[16 i + 4 g4 + j][16 wave + r] ----
    static __device__ void load_state(const DeltaArgs<T>& a, const float* from, std::size_t head, unsigned col, int g4,
                                      f4 (&S)[KT]) {
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned row = 16 * i + 4 * g4 + j;
                S[i][j] = from != nullptr && row < a.dk_dim && col < a.dv_dim
                              ? from[(head * a.dk_dim + row) * a.dv_dim + col] : 0.0f;
            }
    }
    static __device__ void store_state(const DeltaArgs<T>& a, float* to, std::size_t head, unsigned col, int g4,
                                       const f4 (&S)[KT]) {
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned row = 16 * i + 4 * g4 + j;
                if (row < a.dk_dim && col < a.dv_dim) to[(head * a.dk_dim + row) * a.dv_dim + col] = S[i][j];
            }
    }
    // The state before a chunk, kept for the gradient as the registers hold it.
    static __device__ f4* saved_at(const DeltaArgs<T>& a, std::uint32_t slot, std::size_t head, int wave, int lane) {
        const std::size_t state = static_cast<std::size_t>(slot) * a.batch * a.hv + head;
        return reinterpret_cast<f4*>(a.saved + state * DP * DP) + static_cast<std::size_t>(wave) * KT * 64 + lane;
    }
    static __device__ void put_saved(const DeltaArgs<T>& a, std::uint32_t slot, std::size_t head, int wave, int lane,
                                     const f4 (&S)[KT]) {
        f4* to = saved_at(a, slot, head, wave, lane);
#pragma unroll
        for (int i = 0; i < KT; ++i) to[64 * i] = S[i];
    }
    static __device__ void get_saved(const DeltaArgs<T>& a, std::uint32_t slot, std::size_t head, int wave, int lane,
                                     f4 (&S)[KT]) {
        const f4* from = saved_at(a, slot, head, wave, lane);
#pragma unroll
        for (int i = 0; i < KT; ++i) S[i] = from[64 * i];
    }

    // Tokens of the chunk that starts at t0: up to the next multiple of the
    // chunk length, the end, or the next token that drops the state.
    static __device__ int extent(const DeltaArgs<T>& a, std::uint32_t t0, std::uint32_t env, std::uint32_t h, int lane) {
        const std::uint32_t whole = kChunk - t0 % kChunk, left = a.steps - t0;
        const int n = static_cast<int>(whole < left ? whole : left);
        const bool drop = lane > 0 && lane < n && drops(a, t0 + lane, env, h);
        const unsigned long long at = __ballot(drop);
        return at == 0 ? n : __ffsll(static_cast<long long>(at)) - 1;
    }

    // Rows t0 .. t0 + n - 1 of K and Q, zeros below; marks keys that are not
    // finite in `bad`.
    __device__ void stage_keys(const DeltaArgs<T>& x, std::uint32_t t0, int n, std::uint32_t env, std::uint32_t hk,
                               int tid) {
        const int row = tid / (DP / 8), c = 8 * (tid % (DP / 8));
        f4 k0 = {0, 0, 0, 0}, k1 = k0, q0 = k0, q1 = k0;
        if (row < n && c < static_cast<int>(x.dk_dim)) {
            const T* kp = x.k.row(t0 + row, env, hk) + c;
            const T* qp = x.q.row(t0 + row, env, hk) + c;
            k0 = load4(kp, x.k.vec);
            k1 = load4(kp + 4, x.k.vec);
            q0 = load4(qp, x.q.vec);
            q1 = load4(qp + 4, x.q.vec);
        }
        f4* kt = reinterpret_cast<f4*>(&k[row * kStride + c]);
        f4* qt = reinterpret_cast<f4*>(&q[row * kStride + c]);
        kt[0] = k0;
        kt[1] = k1;
        qt[0] = q0;
        qt[1] = q1;
        const f4 z = (k0 - k0) + (k1 - k1);                // 0, or NaN
        if (!(z.x + z.y + z.z + z.w == 0.0f)) atomicOr(&bad, 1u << row);
    }

    // Gates and write strengths of the chunk's tokens (one wave); rows past
    // the last token neither decay nor write.
    __device__ void stage_gates(const DeltaArgs<T>& x, std::uint32_t t0, int n, std::uint32_t env, std::uint32_t h,
                                int lane) {
        float g = 0.0f, b = 0.0f;
        if (lane < n) {
            const std::size_t at = ((static_cast<std::size_t>(t0) + lane) * x.batch + env) * x.hv + h;
            g = x.g[at];
            b = x.beta[at];
            if (!(fabsf(b) < INFINITY) || g != g || g == INFINITY) atomicOr(&bad, 1u << lane);
            if (g < kDropBelow) g = 0.0f;                  // the chunk's first token: the state is dropped
        }
        double sum = g;
#pragma unroll
        for (int d = 1; d < kChunk; d *= 2) {
            const double below = __shfl_up(sum, d);
            if (lane % kChunk >= d) sum += below;
        }
        const double end = __shfl(sum, kChunk - 1);
        if (lane < kChunk) {
            G[lane] = sum;
            gamma[lane] = expf(static_cast<float>(sum));
            decay[lane] = expf(static_cast<float>(end - sum));
            beta[lane] = b;
        }
    }

    // L_ij.
    __device__ float ratio(int i, int j) const { return expf(static_cast<float>(G[i] - G[j])); }

    // A and P: six tiles of products over the key dimension, spread over the
    // waves; the tiles above the diagonal are not read.
    __device__ void products(float scale, int wave, int r, int g4) {
        for (int job = wave; job < 6; job += kWaves) {
            const bool is_p = job >= 3;
            const int place = job % 3, mi = place != 0 ? 16 : 0, nj = place == 2 ? 16 : 0;
            const float* left = is_p ? q : k;
            f4 c = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KT; ++i)
                c = mma(along<kStride>(left, mi, 16 * i, r, g4), along<kStride>(k, nj, 16 * i, r, g4), c);
            float* to = is_p ? p : a;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = mi + 4 * g4 + i, col = nj + r;
                float v = 0.0f;
                if (is_p ? col <= row : col < row) v = c[i] * ratio(row, col) * (is_p ? scale : 1.0f);
                to[row * kSmall + col] = v;
            }
        }
    }

    // Inverse of diagonal tile b of I + A, one column a lane, by substitution.
    __device__ void invert(int b, int r, int g4) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float* row = &a[(16 * b + i) * kSmall + 16 * b];
            float sum = 0.0f;
#pragma unroll
            for (int m = 0; m < i; ++m) sum += row[m] * x[m];
            x[i] = (i == r ? 1.0f : 0.0f) - beta[16 * b + i] * sum;
            if (g4 == 0) t[b][i * 20 + r] = x[i];
        }
    }

    // U = (I + A)^-1 R for a wave's columns.
    __device__ void solve(const f4 (&R)[2], f4 (&U)[2], int r, int g4) const {
        const f4 zero = {0, 0, 0, 0};
        U[0] = mma(along<20>(t[0], 0, 0, r, g4), R[0], zero);
        const f4 below = mma(along<kSmall>(a, 16, 0, r, g4) * beta[16 + r], U[0], zero);
        U[1] = mma(along<20>(t[1], 0, 0, r, g4), R[1] - below, zero);
    }
};

}  // namespace nesle::mem
