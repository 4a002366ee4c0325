// Linear attention with a decay for each head over a rollout, in chunks of tokens.
//
// With a = exp(g) of the head, S the state before a chunk of n tokens and i, j
// counted from its first one:
//   O = scale a^(i + 1) Q S + P V,   P_ij = scale a^(i - j) (q_i . k_j) for j <= i
//   S <- a^n S + K^T a^(n - 1 - j) V
// where a power is zero, by selection, if an episode ends between its two tokens.
//
// One workgroup walks one head of one console; a wave holds 16 columns of the
// state, in registers for the whole rollout, and makes its 16 columns of O.  P is
// made by every wave for itself: its tiles are the operand of P V as the products
// leave them in the registers (mem_delta_math.h), so they need neither LDS nor a
// barrier.  LDS holds K, Q and V of the chunk; two barriers a chunk.
//
// All products keep float32 precision: the state is a float32 result whatever the
// inputs' type.
//
// A product with a masked zero would still carry NaN, so where a key, a value or
// (with an episode's end in the chunk) the state is not finite, the chunk is cut
// before that token and at the ends: nothing of it reaches a token it must not.
//
// What bounds it.  Many heads: memory.  128 tokens of 512 consoles' 4 heads of 64 in
// bfloat16 move 235 MB (inputs, results, states in, out and kept) in 62 us, 3.8 TB/s
// against a large copy's 4.9; two chunks are too short a walk to hide their first loads
// and last stores.  64 consoles take 17 us, in float32 23, in float32 with heads of 128
// 42.  Few heads: the chain of chunks, 2 us each alone on a compute unit, which is why
// long walks are cut (mem_decay_segments.h).  P made by every wave for itself costs
// matrix time that is idle (18 us of 62 here) and saves a barrier.  The state is kept
// every 64 tokens, where the gradient's chunks begin.
#include "mem_decay_segments.h"

namespace nesle::mem {
namespace {

template <typename T, int DP, int CH>
struct ForwardTile {
    using M = typename DecayMathOf<T, DP>::forward;
    typename M::template Tile<CH, DP, M::kIn, 8> k, q, v;
    DecayResults<T, DP, CH> results;
    Powers<CH> powers;
    alignas(16) int episodes[CH];
    std::uint32_t bad[2][2];       // tokens with a value that is not finite, of every other chunk
};

// Waves of a SIMD that registers are to leave room for.
template <int DP>
constexpr int kForwardWaves = DP == 128 ? 2 : 4;

template <int KT>
__device__ bool finite(const f4 (&S)[KT]) {
    f4 none = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KT; ++i) none += S[i] - S[i];      // 0, or NaN
    return none.x + none.y + none.z + none.w == 0.0f;
}

template <typename T, int DP, bool WIDE>
__global__ void __launch_bounds__(DP * 4, kForwardWaves<DP>) decay_forward_kernel(DecayArgs<T> a, DecaySegments seg) {
    constexpr int CH = kDecayChunk<T>, SPAN = kDecaySpan<T, DP>, CT = CH / 16, KT = DP / 16, KP = DP / 32;
    using Tile = ForwardTile<T, DP, CH>;
    using M = typename Tile::M;
    __shared__ Tile sh;
    const Place<DP> first;
    const std::uint32_t env = blockIdx.x / a.hv, h = blockIdx.x % a.hv;
    const std::size_t head = blockIdx.x, state_size = static_cast<std::size_t>(a.dk_dim) * a.dv_dim;
    const std::int64_t out_step = static_cast<std::int64_t>(a.batch) * a.hv * a.dv_dim;
    const int dk = static_cast<int>(a.dk_dim), dv = static_cast<int>(a.dv_dim);
    const f4 zero = {0, 0, 0, 0};
    const std::uint32_t begin = blockIdx.y * seg.steps;
    const std::uint32_t end = a.steps - begin < seg.steps ? a.steps : begin + seg.steps;

    const float gate = a.steps != 0 ? a.g[h] : 0.0f;
    const bool always = gate < kDropBelow;
    sh.powers.make(gate, a.scale, always, first.tid);
    if (first.tid < 4) sh.bad[first.tid / 2][first.tid % 2] = 0;
    f4 S[KT];
    if (seg.count <= kAlone) gather_state<DP>(seg, a.state, gate, blockIdx.y, gridDim.x, head, dk, dv, first, S);
    else load_value_slab<DP>(seg.states + (static_cast<std::size_t>(blockIdx.y) * gridDim.x + head) * state_size, dk, dv, first, S);
    __syncthreads();
    PairPowers<CH, false> pair;
    pair.make(sh.powers, a.scale, first.r, first.g);

    // Tokens from t0 to the next multiple of the chunk length or the end.
    const auto width = [&](std::uint32_t t0) {
        const std::uint32_t whole = CH - t0 % CH, left = end - t0;
        return static_cast<int>(whole < left ? whole : left);
    };
    Piece<T, DP, CH, WIDE> k, q, v;
    Resets<T> resets;
    const auto fetch = [&](std::uint32_t t0, const Place<DP>& at) {
        const int n = width(t0);
        k.fetch(a.k, a.dk_dim, t0, n, env, h / a.group, at);
        q.fetch(a.q, a.dk_dim, t0, n, env, h / a.group, at);
        v.fetch(a.v, a.dv_dim, t0, n, env, h, at);
        resets.fetch(a, t0, n, env, at.lane);
    };
    if (begin < end) fetch(begin, first);
    int which = 0;
    for (std::uint32_t t0 = begin; t0 < end; which ^= 1) {
        const Place<DP> at = Place<DP>::anew();
        const int r = at.r, g = at.g;
        if (t0 != 0 && t0 % SPAN == 0 && a.saved != nullptr)
            store_value_slab<DP>(a.saved + ((t0 / SPAN - 1) * static_cast<std::size_t>(a.batch) * a.hv + head) * state_size, dk, dv, at, S);
        int n = width(t0);
        const std::uint64_t drops = resets.drops(n, at.lane, always);
        if (drops & 1u)
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] = zero;
        const std::uint64_t inside = drops & ~1ull;
        for (;;) {
            k.stage(sh.k, at);
            q.stage(sh.q, at);
            v.stage(sh.v, at);
            if (inside != 0 && at.tid < CH) sh.episodes[at.tid] = Seen(inside, CH).episode(at.tid);
            std::uint64_t odd = k.odd(at) | v.odd(at);
            if (inside != 0 && !finite(S)) odd |= inside;
            if (odd != 0) {
                if (static_cast<std::uint32_t>(odd) != 0) atomicOr(&sh.bad[which][0], static_cast<std::uint32_t>(odd));
                if (static_cast<std::uint32_t>(odd >> 32) != 0) atomicOr(&sh.bad[which][1], static_cast<std::uint32_t>(odd >> 32));
            }
            __syncthreads();
            const std::uint64_t said = sh.bad[which][0] | static_cast<std::uint64_t>(sh.bad[which][1]) << 32;
            const std::uint64_t bad = (static_cast<std::uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<std::uint32_t>(said >> 32))) << 32 |
                                       __builtin_amdgcn_readfirstlane(static_cast<std::uint32_t>(said))) & (~0ull >> (64 - n));
            if (bad == 0 || n == 1) break;
            // Rare: stage again, up to the first such token or end, or a first such
            // token alone; what is left is the next turn's.
            n = (bad & 1u) ? 1 : min(n, __ffsll(static_cast<long long>(bad | inside)) - 1);
            k.cut(n, at);
            q.cut(n, at);
            v.cut(n, at);
            __syncthreads();
            if (at.tid < 2) sh.bad[which][at.tid] = 0;
            __syncthreads();
        }
        if (at.tid < 2) sh.bad[which ^ 1][at.tid] = 0;     // read before the last barrier but one
        const Seen seen(inside & (~0ull >> (64 - n)), n);
        const std::uint32_t next = t0 + n;
        if (next < end) fetch(next, at);

        f4 O[CT];
#pragma unroll
        for (int m = 0; m < CT; ++m) O[m] = zero;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const auto s = M::full(S[2 * i], S[2 * i + 1]);
#pragma unroll
            for (int m = 0; m < CT; ++m) O[m] = M::mul(sh.q.rows(16 * m, i, r, g), s, O[m]);
        }
#pragma unroll
        for (int m = 0; m < CT; ++m) {
            O[m] *= seen.in(sh.powers, 16 * m + 4 * g);
            if (seen.drops != 0)       // by selection: the state may be large
#pragma unroll
                for (int e = 0; e < 4; ++e) O[m][e] = 16 * m + 4 * g + e < seen.first ? O[m][e] : 0.0f;
        }
#pragma unroll
        for (int m = 0; m < CT; ++m)
#pragma unroll
            for (int p = 0; p <= m / 2; ++p) {
                f4 x[2] = {zero, zero};
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (2 * p + t > m) break;
#pragma unroll
                    for (int i = 0; i < KP; ++i)
                        x[t] = M::mul(sh.k.rows(16 * (2 * p + t), i, r, g), sh.q.rows(16 * m, i, r, g), x[t]);
                    x[t] = pair.weigh(x[t], m, 2 * p + t, seen, sh.episodes, r, g);
                }
                O[m] = M::mul(M::full(x[0], x[1]), sh.v.cols(32 * p, 16 * at.wave, r, g), O[m]);
            }
        const float whole = seen.whole(sh.powers);
#pragma unroll
        for (int i = 0; i < KT; ++i) S[i] = seen.drops != 0 ? zero : S[i] * whole;
#pragma unroll
        for (int p = 0; p < CH / 32; ++p) {
            f4 V[2];
            M::values(sh.v.cols(32 * p, 16 * at.wave, r, g), V);
            const auto held = M::full(V[0] * seen.out(sh.powers, 32 * p + 4 * g), V[1] * seen.out(sh.powers, 32 * p + 16 + 4 * g));
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] = M::mul(sh.k.cols(32 * p, 16 * i, r, g), held, S[i]);
        }
        const Rows<T, WIDE> out(a.out + static_cast<std::int64_t>(t0) * out_step + head * a.dv_dim, out_step);
        typename DecayResults<T, DP, CH>::Tile done[CT];
#pragma unroll
        for (int m = 0; m < CT; ++m) done[m] = sh.results.tile(O[m]);
        sh.results.put(out, dv, n, at, done);
        t0 = next;
        __syncthreads();
        sh.results.flush(out, dv, n, at);
    }
    if (end == a.steps) store_value_slab<DP>(a.state_out + head * state_size, dk, dv, Place<DP>::anew(), S);
}

template <typename T, int DP, bool WIDE>
void launch_dim(const DecayArgs<T>& a, const DecaySegments& seg, hipStream_t s) {
    if (seg.count > 1) launch_states<T, DP, WIDE, false>(a, seg, s);
    hipLaunchKernelGGL((decay_forward_kernel<T, DP, WIDE>), dim3(a.batch * a.hv, seg.count), dim3(DP * 4), 0, s, a, seg);
}

template <typename T>
int forward(const char* who, const nesle_decay_args& x, hipStream_t s) {
    const DecayArgs<T> a = decay_args<T>(x);
    DecaySegments seg = decay_segments(x, false);
    seg.place(x, a.scratch);
    at_dim(x, [&](auto dim) {
        if (wide_rows(x)) launch_dim<T, dim(), true>(a, seg, s);
        else launch_dim<T, dim(), false>(a, seg, s);
    });
    return launched(who);
}

}  // namespace
}  // namespace nesle::mem

using namespace nesle::mem;

extern "C" {

std::uint64_t nesle_decay_saved_floats(const nesle_decay_args* a) {
    if (a == nullptr || a->steps <= decay_span(*a)) return 0;
    const std::uint64_t chunks = (static_cast<std::uint64_t>(a->steps) + decay_span(*a) - 1) / decay_span(*a) - 1;
    return chunks * a->batch * a->v_heads * a->k_dim * a->v_dim;
}

std::uint64_t nesle_decay_forward_scratch_floats(const nesle_decay_args* a) {
    if (a == nullptr || a->batch == 0 || a->v_heads == 0) return 0;
    return decay_segments(*a, false).floats(*a);
}

int nesle_decay_forward(const nesle_decay_args* a, void* stream) {
    const char* who = "nesle_decay_forward";
    int rc = check_decay(who, a);
    if (rc != NESLE_OK || a->batch == 0) return rc;
    if (!a->state_out) return refuse(who, "null device pointer");
    rc = check_decay_alignment(who, a);
    if (rc != NESLE_OK) return rc;
    if (a->steps != 0) {
        rc = check_decay_inputs(who, a);
        if (rc != NESLE_OK) return rc;
        if (!a->out || (!a->scratch && nesle_decay_forward_scratch_floats(a) != 0)) return refuse(who, "null device pointer");
    }
    const auto s = static_cast<hipStream_t>(stream);
    return a->dtype == NESLE_MEM_F32 ? forward<float>(who, *a, s) : forward<bf16>(who, *a, s);
}

}  // extern "C"
