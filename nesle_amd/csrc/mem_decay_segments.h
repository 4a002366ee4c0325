// mem_decay_segments.h -- few heads over many tokens, cut into segments that are walked
// at once.
//
// A segment of L tokens takes the state before it to a^L S + B, with B from its keys
// and values alone.  One launch finds every segment's B, one, or the walk where there
// are few, takes the state through the segments, and then the walk runs from each
// segment's own state.  The gradient of
// the state goes the same way backwards, with queries and the outputs' gradients.
#pragma once

#include <algorithm>

#include "mem_decay.h"

namespace nesle::mem {

struct DecaySegments {
    std::uint32_t steps, count;        // tokens of one, a multiple of the chunk length
    float* states;                     // [segment][head][k_dim][v_dim]: B, then the state before (after) it
    std::uint32_t* dropped;            // [segment][head]: whether the state is dropped inside
    std::uint64_t floats(const nesle_decay_args& a) const {
        return count < 2 ? 0 : static_cast<std::uint64_t>(count) * a.batch * a.v_heads * (static_cast<std::uint64_t>(a.k_dim) * a.v_dim + 1);
    }
    void place(const nesle_decay_args& a, float* scratch) {
        states = scratch;
        dropped = reinterpret_cast<std::uint32_t*>(scratch + static_cast<std::uint64_t>(count) * a.batch * a.v_heads * a.k_dim * a.v_dim);
    }
};

constexpr std::uint32_t kMostSegments = 128;      // what one workgroup takes a state through

// As many segments as the card holds their workgroups at once with room to spare: 1,024,
// 512 and 256 heads' of 32, 64 and 128 dimensions.  The launch more, or two, and the second
// reading of the inputs are worth it from 3 times 64 tokens on forward and from 8 in the
// gradient, from 8 in both where that makes only two or three segments.  One walk /
// segments, us a call, bfloat16, float32, and bfloat16 with gradient (from the host, whose
// part is 85 and 95; * where the rule walks whole):
//   64 dimensions, 64 heads, 128 tokens* 14 / 14, 19 / 18, 88 / 100; 192 18 / 14, 27 / 18; 256
//   22 / 15, 34 / 19, 87 / 98*; 512 40 / 18, 63 / 27, 114 / 98; 1,024 74 / 27, 122 / 42, 215 / 77;
//   256 heads, 256 tokens* 24 / 25, 35 / 38; 512 42 / 38, 65 / 66, 121 / 112; 1,024 77 / 66, 125 / 121,
//   237 / 203; 128 dimensions, 64 heads, 256 tokens 36 / 24, 62 / 34, 130 / 98*; 512 66 / 35, 118 /
//   55, 246 / 112; 32 dimensions, 256 heads, 256 tokens 20 / 15, 25 / 19, 54 / 99*; 1,024 65 / 40,
//   86 / 50, 179 / 112.
// Segments of 64 dimensions for 1,024 heads at once: 1,024 tokens of 64 heads 33 -> 37, 8,191
// of 8 32 -> 34; for 256: 38 and 37.
inline DecaySegments decay_segments(const nesle_decay_args& a, bool back) {
    constexpr std::uint32_t kSpan = 64;            // tokens: a multiple of any chunk length
    const std::uint64_t heads = static_cast<std::uint64_t>(a.batch) * a.v_heads, at_once = (1u << 15) / padded_dim(a);
    const std::uint32_t spans = (a.steps + kSpan - 1) / kSpan;
    std::uint32_t count = 1;
    if (2 * heads <= at_once && spans >= (!back && 4 * heads <= at_once ? 3u : 8u))
        count = static_cast<std::uint32_t>(std::min<std::uint64_t>({spans, kMostSegments, at_once / heads}));
    const std::uint32_t each = count < 2 ? spans : (spans + count - 1) / count;
    DecaySegments s{};
    s.steps = std::max(each, 1u) * kSpan;
    s.count = spans == 0 ? 1 : (spans + each - 1) / each;
    return s;
}

// ---- B of every segment -----------------------------------------------------------

template <typename T, int DP, int CH, bool BACK>
struct LocalTile {
    using M = std::conditional_t<BACK, typename DecayMathOf<T, DP>::gradient, typename DecayMathOf<T, DP>::forward>;
    typename M::template Tile<CH, DP, M::kIn, 8> x, y;
    Powers<CH> powers;
};

// A workgroup walks one segment of one head, 16 value columns a wave.  BACK: queries
// and the outputs' gradients, last to first, decayed to the segment's beginning.
template <typename T, int DP, bool WIDE, bool BACK>
__global__ void __launch_bounds__(DP * 4, DP == 128 ? 2 : 4) decay_local_kernel(DecayArgs<T> a, DecaySegments seg) {
    constexpr int CH = kDecayChunk<T>, KT = DP / 16;
    using Tile = LocalTile<T, DP, CH, BACK>;
    using M = typename Tile::M;
    __shared__ Tile sh;
    const Place<DP> first;
    const std::uint32_t env = blockIdx.x / a.hv, h = blockIdx.x % a.hv;
    const std::uint32_t segment = blockIdx.y + (BACK ? 1 : 0);      // the first one's, or the last one's, is not needed
    const std::uint32_t begin = segment * seg.steps;
    const std::uint32_t end = a.steps - begin < seg.steps ? a.steps : begin + seg.steps;
    const std::uint32_t chunks = (end - begin + CH - 1) / CH;
    const float gate = a.g[h];
    const bool always = gate < kDropBelow;
    sh.powers.make(gate, a.scale, always, first.tid);
    f4 S[KT];
#pragma unroll
    for (int i = 0; i < KT; ++i) S[i] = f4{0, 0, 0, 0};

    Piece<T, DP, CH, WIDE> x, y;
    Resets<T> resets;
    const auto start_of = [&](std::uint32_t c) { return begin + (BACK ? chunks - 1 - c : c) * CH; };
    const auto width = [&](std::uint32_t t0) { return static_cast<int>(end - t0 < CH ? end - t0 : CH); };
    const auto fetch = [&](std::uint32_t c, const Place<DP>& at) {
        const std::uint32_t t0 = start_of(c);
        x.fetch(BACK ? a.q : a.k, a.dk_dim, t0, width(t0), env, h / a.group, at);
        y.fetch(BACK ? a.dout : a.v, a.dv_dim, t0, width(t0), env, h, at);
        resets.fetch(a, t0, width(t0), env, at.lane);
    };
    fetch(0, first);
    bool any_drop = false;
    for (std::uint32_t c = 0; c < chunks; ++c) {
        const Place<DP> at = Place<DP>::anew();
        const int n = width(start_of(c));
        const Seen seen(resets.drops(n, at.lane, always), n);
        // Tokens before the last end of an episode leave nothing in the state, and what
        // is not finite in them must not either.  (The gradient of such inputs is
        // unspecified.)
        if (!BACK && seen.drops != 0) {
            x.cut_before(seen.last, at);
            y.cut_before(seen.last, at);
        }
        any_drop |= seen.drops != 0;
        x.stage(sh.x, at);
        y.stage(sh.y, at);
        __syncthreads();
        if (c + 1 < chunks) fetch(c + 1, at);
        const float whole = seen.whole(sh.powers);
#pragma unroll
        for (int i = 0; i < KT; ++i) S[i] = seen.drops != 0 ? f4{0, 0, 0, 0} : S[i] * whole;
#pragma unroll
        for (int p = 0; p < CH / 32; ++p) {
            f4 V[2], w[2];
            M::values(sh.y.cols(32 * p, 16 * at.wave, at.r, at.g), V);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int row = 32 * p + 16 * t + 4 * at.g;
                w[t] = BACK ? seen.in(sh.powers, row) : seen.out(sh.powers, row);
            }
            const auto held = M::full(V[0] * w[0], V[1] * w[1]);
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] = M::mul(sh.x.cols(32 * p, 16 * i, at.r, at.g), held, S[i]);
        }
        __syncthreads();
    }
    const std::size_t slot = static_cast<std::size_t>(segment) * gridDim.x + blockIdx.x;
    store_value_slab<DP>(seg.states + slot * a.dk_dim * a.dv_dim, static_cast<int>(a.dk_dim), static_cast<int>(a.dv_dim),
                         Place<DP>::anew(), S);
    if (first.tid == 0) seg.dropped[slot] = any_drop;
}

// ---- the state through the segments -------------------------------------------------

// S <- a^L S + B from segment to segment; a segment that drops the state inside leaves
// B alone, whatever S held.
//
// Forward, up to 16 segments: each workgroup of the walk takes the state through the ones
// before its own by itself, and a launch less pays for that.  The forward's launches, 1,024
// tokens of 64, 128 and 32 heads of 64 in bfloat16 (8, 4 and 16 segments): 32 -> 29, 48 ->
// 44 and 26 -> 24 us.  Not the gradient, which needs dS twice, by key and by value: even
// with 8 segments, 38 -> 44 us with 16, and 5 % slower where there is but one.
constexpr std::uint32_t kAlone = 16;
template <int DP>
__device__ __forceinline__ void gather_state(const DecaySegments& seg, const float* start, float gate, std::uint32_t segment, std::size_t heads,
                                             std::size_t head, int dk, int dv, const Place<DP>& at, f4 (&S)[DP / 16]) {
    const std::size_t size = static_cast<std::size_t>(dk) * dv;
    load_value_slab<DP>(start == nullptr ? nullptr : start + head * size, dk, dv, at, S);
    const float factor = expf(static_cast<float>(seg.steps) * gate);
#pragma unroll 2
    for (std::uint32_t i = 0; i < segment; ++i) {
        const std::size_t slot = i * heads + head;
        f4 B[DP / 16];
        load_value_slab<DP>(seg.states + slot * size, dk, dv, at, B);
        const bool dropped = seg.dropped[slot] != 0;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) S[k] = dropped ? B[k] : S[k] * factor + B[k];
    }
}

// Else a launch of their own, after which B has given way to the state before the segment
// (BACK: the gradient after it).  A lane has four elements of a state and reads its share
// of the segments at once: all of them (GROUPS 1, up to 8 segments), or an equal share of 16
// groups', joined through LDS, after which every group walks its own from where the ones
// before it end.  16 groups / one: 4 segments of 128 heads of 64 18 / 6 us, 8 of 64 11 / 7, 16
// of 32 8 / 10.
constexpr std::uint32_t kFew = 8;
template <bool BACK, int GROUPS>
__global__ void __launch_bounds__(256) decay_join_kernel(DecaySegments seg, const float* start, const float* g, std::uint32_t hv,
                                                         std::uint32_t size, std::uint32_t last_steps) {
    constexpr int kShare = GROUPS == 1 ? kFew : kMostSegments / GROUPS, kLanes = 256 / GROUPS;
    __shared__ f4 sums[GROUPS][kLanes];
    __shared__ float factors[GROUPS];                      // negative: dropped
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const std::uint32_t at = (blockIdx.y * kLanes + lane) * 4;
    const bool in = at < size;
    const std::size_t heads = gridDim.x, head = blockIdx.x;
    const int count = static_cast<int>(seg.count), share = (count + GROUPS - 1) / GROUPS, begin = group * share;
    const auto slot = [&](int i) { return static_cast<std::size_t>(BACK ? count - 1 - i : i) * heads + head; };
    const float gate = g[head % hv];
    const float all = expf(static_cast<float>(seg.steps) * gate), tail = expf(static_cast<float>(last_steps) * gate);
    const auto factor = [&](int i) { return BACK && i == 0 ? tail : all; };
    const f4 zero = {0, 0, 0, 0};

    f4 B[kShare];
    bool dropped[kShare];
#pragma unroll
    for (int k = 0; k < kShare; ++k) {
        const int i = begin + k;
        const bool use = k < share && i < count - 1;       // the last one's is not needed
        B[k] = use && in ? *reinterpret_cast<const f4*>(seg.states + slot(i) * size + at) : zero;
        dropped[k] = use && seg.dropped[slot(i)] != 0;
    }
    f4 S = start != nullptr && in ? *reinterpret_cast<const f4*>(start + head * size + at) : zero;
    if constexpr (GROUPS > 1) {
        f4 sum = zero;
        bool any = false;
        float f = 1.0f;
#pragma unroll
        for (int k = 0; k < kShare; ++k)
            if (k < share && begin + k < count - 1) {
                sum = dropped[k] ? B[k] : sum * factor(begin + k) + B[k];
                f *= factor(begin + k);
                any |= dropped[k];
            }
        sums[group][lane] = sum;
        if (lane == 0) factors[group] = any ? -1.0f : f;
        __syncthreads();
        for (int before = 0; before < group; ++before) S = factors[before] < 0.0f ? sums[before][lane] : S * factors[before] + sums[before][lane];
    }
#pragma unroll
    for (int k = 0; k < kShare; ++k) {
        const int i = begin + k;
        if (k >= share || i >= count) break;
        if (in) *reinterpret_cast<f4*>(seg.states + slot(i) * size + at) = S;
        S = dropped[k] ? B[k] : S * factor(i) + B[k];
    }
}

template <typename T, int DP, bool WIDE, bool BACK>
void launch_states(const DecayArgs<T>& a, const DecaySegments& seg, hipStream_t s) {
    const std::uint32_t heads = a.batch * a.hv, size = a.dk_dim * a.dv_dim;
    hipLaunchKernelGGL((decay_local_kernel<T, DP, WIDE, BACK>), dim3(heads, seg.count - 1), dim3(DP * 4), 0, s, a, seg);
    const float* start = BACK ? a.dstate_out : a.state;
    const std::uint32_t last = a.steps - (seg.count - 1) * seg.steps;
    if constexpr (BACK) {
        if (seg.count <= kFew) {
            hipLaunchKernelGGL((decay_join_kernel<BACK, 1>), dim3(heads, (size + 1023) / 1024), dim3(256), 0, s, seg, start, a.g, a.hv, size, last);
            return;
        }
    } else if (seg.count <= kAlone) {
        return;
    }
    hipLaunchKernelGGL((decay_join_kernel<BACK, 16>), dim3(heads, (size + 63) / 64), dim3(256), 0, s, seg, start, a.g, a.hv, size, last);
}

}  // namespace nesle::mem
