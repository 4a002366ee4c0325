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
// A chunk ends early at a token that drops the state (its episode ended) and
// before one that holds a value that is not finite, so that neither reaches a
// token it must not (a product with a masked zero would carry NaN).
#include "mem_delta_tile.h"

namespace nesle::mem {
namespace {

template <typename T, int DP, bool WIDE>
__global__ void __launch_bounds__(DP * 4, DP == 128 ? 2 : 4) delta_forward_kernel(DeltaArgs<T> a) {
    using Tile = ChunkTile<T, DP>;
    using M = typename Tile::M;
    constexpr int KT = Tile::KT, KP = Tile::KP;
    __shared__ Tile sh;
    const Lane<DP> first;
    const std::uint32_t env = blockIdx.x / a.hv, h = blockIdx.x % a.hv;
    const std::size_t head = blockIdx.x, state_size = static_cast<std::size_t>(a.dk_dim) * a.dv_dim;
    const std::int64_t out_step = static_cast<std::int64_t>(a.batch) * a.hv * a.dv_dim;
    const f4 zero = {0, 0, 0, 0};

    f4 S[KT];
    Tile::load_state(a, a.state, head, first, S);
    sh.start(first);
    __syncthreads();

    // Tokens from t0 to the next multiple of the chunk length or the end.
    const auto width = [&](std::uint32_t t0) {
        const std::uint32_t whole = kChunk - t0 % kChunk, left = a.steps - t0;
        return static_cast<int>(whole < left ? whole : left);
    };
    Ahead<T, DP, WIDE> in;
    if (a.steps != 0) in.fetch(a, 0, width(0), env, h, first);
    for (std::uint32_t t0 = 0; t0 < a.steps;) {
        const Lane<DP> at = Lane<DP>::anew();
        const int r = at.r, g = at.g;
        const bool in_col = at.col < static_cast<int>(a.dv_dim);
        if (t0 != 0 && t0 % kChunk == 0 && a.saved != nullptr)
            Tile::store_state(a, a.saved + (t0 / kChunk - 1) * state_size * a.batch * a.hv, head, at, S);
        const std::uint32_t drops = in.drops();
        if (drops & 1u)
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] = zero;
        int n = drops & ~1u ? __ffs(static_cast<int>(drops & ~1u)) - 1 : width(t0);
        f4 V[2];
        for (;;) {
            std::uint32_t odd = sh.stage_keys(in, 0, n, at);
            if (at.wave == 0) odd |= sh.stage_gates(in, 0, n, at.lane);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = at.row(e) < n ? Rows<T, WIDE>::value_of(in.v[e]) : 0.0f;
                if (!(fabsf(x) < INFINITY)) odd |= 1u << at.row(e);
                V[e / 4][e % 4] = x;
            }
            sh.report(odd);
            __syncthreads();
            const unsigned bad = __builtin_amdgcn_readfirstlane(sh.bad);
            if (bad == 0 || n == 1) break;
            // Rare: stage again, up to the first such token, or it alone.
            n = (bad & 1u) ? 1 : __ffs(static_cast<int>(bad)) - 1;
            __syncthreads();
            if (at.tid == 0) sh.bad = 0;
            __syncthreads();
        }
        const std::uint32_t next = t0 + n;
        if (next < a.steps) in.fetch(a, next, width(next), env, h, at);
        for (int place = at.wave; place < 3; place += Tile::kWaves) {
            f4 kk, qk;
            sh.products(place, a.scale, at, kk, qk);
        }
        __syncthreads();
        if (at.tid == 0) sh.bad = 0;
        // A different wave each workgroup, as the waves of a compute unit's
        // workgroups share its four SIMDs by their number.
        if (at.wave == static_cast<int>(blockIdx.x % Tile::kWaves)) sh.invert(at);

        // K S and Q S for this wave's columns.
        f4 ks[2] = {}, qs[2] = {};
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const auto s = M::full(S[2 * i], S[2 * i + 1]);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                ks[m] = M::mul(sh.k.rows(16 * m, i, r, g), s, ks[m]);
                qs[m] = M::mul(sh.q.rows(16 * m, i, r, g), s, qs[m]);
            }
        }
        f4 R[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const f4 gam = sh.of_rows(sh.gamma, m, g);
            R[m] = sh.of_rows(sh.beta, m, g) * (V[m] - gam * ks[m]);
            qs[m] *= gam * a.scale;
        }
        const auto right = M::full(R[0], R[1]);
        __syncthreads();
        f4 U[2], O[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) U[m] = M::mul(sh.t.rows(16 * m, 0, r, g), right, zero);
        const auto u = M::full(U[0], U[1]);
#pragma unroll
        for (int m = 0; m < 2; ++m) O[m] = M::mul(sh.p.rows(16 * m, 0, r, g), u, qs[m]);
        const Rows<T, WIDE> out(a.out + static_cast<std::int64_t>(t0) * out_step + head * a.dv_dim, out_step);
#pragma unroll
        for (int e = 0; e < 8; ++e) out.put(in_col && at.row(e) < n, at.row(e), at.col, O[e / 4][e % 4]);
        const float last = sh.gamma[kChunk - 1];
        const auto w = M::full(U[0] * sh.of_rows(sh.decay, 0, g), U[1] * sh.of_rows(sh.decay, 1, g));
#pragma unroll
        for (int i = 0; i < KT; ++i) S[i] = S[i] * last + M::mul(sh.k.cols(0, 16 * i, r, g), w, zero);
        t0 = next;
        __syncthreads();
    }
    Tile::store_state(a, a.state_out, head, Lane<DP>::anew(), S);
}

template <typename T>
int forward(const char* who, const nesle_delta_args& x, hipStream_t s) {
    const DeltaArgs<T> a = delta_args<T>(x);
    const dim3 grid(a.batch * a.hv);
    const std::uint32_t dim = wide_rows(x) ? 0 : padded_dim(x);
    switch (dim) {
        case 0: hipLaunchKernelGGL((delta_forward_kernel<T, 128, true>), grid, dim3(512), 0, s, a); break;
        case 32: hipLaunchKernelGGL((delta_forward_kernel<T, 32, false>), grid, dim3(128), 0, s, a); break;
        case 64: hipLaunchKernelGGL((delta_forward_kernel<T, 64, false>), grid, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL((delta_forward_kernel<T, 128, false>), grid, dim3(512), 0, s, a); break;
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
