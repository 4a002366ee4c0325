// Sampling of actions from given random numbers (include/nesle_memory.h has the
// rules).
//
// Which actions are left and which one a uniform number falls on turn on comparisons
// of sums, so weights and sums are float64: in float32 a border would be off by up to
// 2^-24 of the whole, and one row in 10^5 or so would get another action than the
// rules say.
//
// Up to 16 actions, a row is 16 lanes, an action a lane: what is ahead of an action in
// the order of falling scores is found by comparing it with the other 15, which pass
// by in turn.  Up to 64, a row is a wave, an action a lane, and the lanes sort
// themselves.  With more, lane l has the actions E l .. E l + E - 1, and the border that
// top_k or top_p draws is found without sorting.  For top_k by halving the scores' range,
// each time with a count, a vote of the lanes; what it leaves, if that is 64 or fewer,
// moves to one action a lane and sorts itself.  For top_p the 64 largest are tried that
// way.  If they do not reach its share, scores become whole numbers of the same order, and
// the bits of one at the border are found from the top, each with a sum in float32: the
// border that it ends at is then tested in float64, and the search done again in float64
// if the sums' roundings led it astray.
//
// Bound by instructions, and by a launch where there are few rows.  8,192 rows of 12: 3.9
// us.  65,536 rows, unfiltered / with top_k 40, top_p 0.9 and min_p: of 12 in all 15 with
// limits, of 60 23 / 40, of 256 41 / 101 (661 vector instructions a row, 70 us if none
// waited; their 69 MB would take 14), with top_p alone 154; 16,384 rows of 1,000 38 / 99.
// The search of top_k and top_p halves the scores' range, so a finite mask far below them
// costs rounds, where -infinity costs none: of 65,536 rows of 256, a quarter of the actions
// masked, with limits 82 us by -infinity, 95 by -1e4, 124 by -1e9, 309 by float32's lowest
// value; top_k alone 65, 81, 112, 301; top_p alone 119, 132, 158, 333.  With more than 64
// actions a lane spills up to 12 vector registers (24 to 52 bytes of scratch).
// On the way here, of 256 with limits: borders searched with sums in float64 449 us; by
// votes, what top_k leaves on one lane each 112; settings and logarithms of several rows
// at once, scores sorted, 101.
#include <algorithm>

#include "mem_delta_math.h"

namespace nesle::mem {
namespace {

template <typename T>
struct SampleArgs {
    Heads<T> logits;
    const float* uniform;
    double temperature, top_p, min_p;
    std::uint32_t top_k;             // at most the actions
    const float *temperatures, *top_ps, *min_ps;
    const std::int32_t* top_ks;
    std::int64_t* action;
    float* logprob;
    std::uint32_t rows, batch, actions;
};

// A launch takes fewer than 2^32 threads in a row of its grid, which 2^28 rows of 16 lanes
// would pass: workgroups go in several rows of 2^20 there.
dim3 grid_of(std::uint32_t blocks) {
    constexpr std::uint32_t kRow = 1u << 20;
    return blocks <= kRow ? dim3(blocks) : dim3(kRow, (blocks + kRow - 1) / kRow);
}
__device__ std::uint64_t block_of() { return static_cast<std::uint64_t>(blockIdx.y) * gridDim.x + blockIdx.x; }

// ---- across lanes: data-parallel moves, no LDS -------------------------------------
template <int CTRL, int ROWS = 0xf>
__device__ std::uint32_t moved_bits(std::uint32_t v) {
    return static_cast<std::uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, true));
}
// v as the lane that CTRL names holds it, zero where there is none.
template <int CTRL, int ROWS = 0xf, typename X>
__device__ X from_lane(X v) {
    if constexpr (sizeof(X) == 8) {
        const auto b = __builtin_bit_cast(std::uint64_t, v);
        return __builtin_bit_cast(X, static_cast<std::uint64_t>(moved_bits<CTRL, ROWS>(static_cast<std::uint32_t>(b >> 32))) << 32 |
                                         moved_bits<CTRL, ROWS>(static_cast<std::uint32_t>(b)));
    } else {
        return __builtin_bit_cast(X, moved_bits<CTRL, ROWS>(__builtin_bit_cast(std::uint32_t, v)));
    }
}
// Sums over the lanes below, and the lane itself: of 16 lanes, and of a wave.
template <typename X>
__device__ X scan16(X v) {
    v += from_lane<kRowShr + 1>(v);
    v += from_lane<kRowShr + 2>(v);
    v += from_lane<kRowShr + 4>(v);
    return v + from_lane<kRowShr + 8>(v);
}
constexpr int kRowBcast15 = 0x142, kRowBcast31 = 0x143, kRowLast = 0x15f;     // the 16th lane's of the row, to all
template <typename X>
__device__ X scan64(X v) {
    v = scan16(v);
    v += from_lane<kRowBcast15, 0xa>(v);       // row 0's sum to row 1, row 2's to row 3
    return v + from_lane<kRowBcast31, 0xc>(v); // rows 0 and 1's to rows 2 and 3
}
template <typename X>
__device__ X of_lane(X v, int lane) {
    if constexpr (sizeof(X) == 8) {
        const auto b = __builtin_bit_cast(std::uint64_t, v);
        const std::uint32_t hi = __builtin_amdgcn_readlane(static_cast<std::uint32_t>(b >> 32), lane),
                            lo = __builtin_amdgcn_readlane(static_cast<std::uint32_t>(b), lane);
        return __builtin_bit_cast(X, static_cast<std::uint64_t>(hi) << 32 | lo);
    } else {
        return __builtin_bit_cast(X, __builtin_amdgcn_readlane(__builtin_bit_cast(std::uint32_t, v), lane));
    }
}
template <typename X>
__device__ X sum64(X v) { return of_lane(scan64(v), 63); }

__device__ int lanes_in(std::uint64_t mask) { return __popcll(mask); }
__device__ int lanes_below(std::uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<std::uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<std::uint32_t>(mask), 0));
}
__device__ int first_lane(std::uint64_t mask) { return __ffsll(static_cast<long long>(mask)) - 1; }
__device__ int last_lane(std::uint64_t mask) { return 63 - __clzll(static_cast<long long>(mask)); }

// Whole numbers in the order of the floats, -0 as 0; 0 for -infinity.
__device__ std::uint32_t key_of(float x) {
    if (x == -INFINITY) return 0u;
    const std::uint32_t b = __builtin_bit_cast(std::uint32_t, x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// A row's settings.
struct Settings {
    double temperature, inverse, top_p, min_p, u;
    int top_k;
    template <typename T>
    __device__ Settings(const SampleArgs<T>& a, std::uint32_t r)
        : temperature(a.temperatures != nullptr ? a.temperatures[r] : a.temperature), inverse(1.0 / temperature),
          top_p(a.top_ps != nullptr ? a.top_ps[r] : a.top_p), min_p(a.min_ps != nullptr ? a.min_ps[r] : a.min_p), u(a.uniform[r]),
          top_k(a.top_ks != nullptr ? a.top_ks[r] : static_cast<int>(a.top_k)) {}
    __device__ bool fine() const {
        return temperature >= 0.0 && temperature < INFINITY && top_p > 0.0 && top_p <= 1.0 && min_p >= 0.0 && min_p <= 1.0 &&
               top_k >= 0 && u == u;
    }
    // The difference first: a quotient may pass the largest number.  (1 / temperature may
    // too; 0 times that would be NaN.)
    __device__ double weight(float x, float most) const {
        const double w = exp((static_cast<double>(x) - most) * inverse);
        return x == most ? 1.0 : x > -INFINITY ? w : 0.0;
    }
};

// ---- up to 16 actions: 16 lanes a row -----------------------------------------------
__device__ float most16(float v) {
    v = fmaxf(v, moved<kRowRor + 8>(v));
    v = fmaxf(v, moved<kRowRor + 4>(v));
    v = fmaxf(v, moved<kRowRor + 2>(v));
    return fmaxf(v, moved<kRowRor + 1>(v));
}
// Bit s: the action that is s lanes round is ahead; their number, and of those that
// `ahead` has, the sum of their weights.
template <int... S>
__device__ std::uint32_t ahead16(std::integer_sequence<int, S...>, std::uint32_t key, std::uint32_t lane) {
    std::uint32_t ahead = 0;
    const auto meet = [&](std::uint32_t other, std::uint32_t from, int s) {
        if (other > key || (other == key && from < lane)) ahead |= 1u << s;
    };
    (meet(from_lane<kRowRor + S + 1>(key), from_lane<kRowRor + S + 1>(lane), S), ...);
    return ahead;
}
template <int... S>
__device__ double before16(std::integer_sequence<int, S...>, std::uint32_t ahead, double w) {
    double sum = 0.0;
    const auto meet = [&](double other, int s) { sum += ahead >> s & 1u ? other : 0.0; };
    (meet(from_lane<kRowRor + S + 1>(w), S), ...);
    return sum;
}

template <typename T>
__global__ void __launch_bounds__(256) sample16_kernel(SampleArgs<T> a) {
    const std::uint32_t lane = threadIdx.x % 16;
    const std::uint64_t row = (block_of() * 256 + threadIdx.x) / 16;
    const auto r = static_cast<std::uint32_t>(row < a.rows ? row : a.rows - 1);        // past the end: the last one's again, not written
    const Settings set(a, r);
    const float x = lane < a.actions ? static_cast<float>(a.logits.row(r / a.batch, r % a.batch, 0)[lane]) : -INFINITY;
    const auto of_row = [&](bool v) { return static_cast<std::uint32_t>(__ballot(v) >> (threadIdx.x % 64 / 16 * 16)) & 0xffffu; };
    const bool odd = of_row(!(x < INFINITY)) != 0;             // NaN or +infinity
    const float most = most16(x);
    const bool fine = !odd && most > -INFINITY && set.fine(), greedy = set.temperature == 0.0;
    const std::uint32_t best = of_row(x == most);
    double w = fine && !greedy ? set.weight(x, most) : 0.0;
    const bool narrow = set.top_p < 1.0 || (set.top_k > 0 && set.top_k < a.actions);
    if (__any(narrow)) {
        constexpr std::make_integer_sequence<int, 15> others{};
        const std::uint32_t ahead = ahead16(others, key_of(x), lane);
        if (set.top_k > 0 && __popc(ahead) >= set.top_k) w = 0.0;
        const double share = set.top_p * from_lane<kRowLast>(scan16(w));
        const double before = before16(others, ahead, w);
        if (set.top_p < 1.0 && !(before < share)) w = 0.0;
    }
    if (w < set.min_p) w = 0.0;
    const double run = scan16(w), all = from_lane<kRowLast>(run), target = (set.u > 0.0 ? set.u : 0.0) * all;
    const std::uint32_t left = of_row(w > 0.0), past = of_row(w > 0.0 && run > target);
    const int found = greedy ? __ffs(static_cast<int>(best)) - 1 : past != 0 ? __ffs(static_cast<int>(past)) - 1 : 31 - __clz(static_cast<int>(left));
    if (row >= a.rows) return;
    if (!fine) {
        if (lane == 0) {
            a.action[r] = -1;
            a.logprob[r] = NAN;
        }
    } else if (static_cast<int>(lane) == found) {
        a.action[r] = found;
        a.logprob[r] = greedy ? 0.0f : static_cast<float>(log(w / all));
    }
}

// ---- more: a wave a row ---------------------------------------------------------------

// The value of the lane whose number differs in the bits of MASK.
template <int MASK>
__device__ std::uint32_t of_other(std::uint32_t v) {
    if constexpr (MASK == 1) return from_lane<0xb1>(v);
    else if constexpr (MASK == 2) return from_lane<0x4e>(v);
    else if constexpr (MASK == 3) return from_lane<0x1b>(v);
    else if constexpr (MASK == 4) return from_lane<0x1b>(from_lane<0x141>(v));     // 7, then 3
    else if constexpr (MASK == 7) return from_lane<0x141>(v);
    else if constexpr (MASK == 8) return from_lane<kRowRor + 8>(v);
    else if constexpr (MASK == 15) return from_lane<0x140>(v);
    else return static_cast<std::uint32_t>(__shfl_xor(static_cast<int>(v), MASK));
}
// Larger of two lanes' values to the lower one.
template <int MASK>
__device__ void order(std::uint64_t& v, int lane) {
    constexpr int top = MASK >= 32 ? 32 : MASK >= 16 ? 16 : MASK >= 8 ? 8 : MASK >= 4 ? 4 : MASK >= 2 ? 2 : 1;
    const std::uint64_t other = static_cast<std::uint64_t>(of_other<MASK>(static_cast<std::uint32_t>(v >> 32))) << 32 |
                                of_other<MASK>(static_cast<std::uint32_t>(v));
    v = (other > v) == ((lane & top) == 0) ? other : v;
}
// The lanes' values in falling order: runs of 2, 4, .. lanes are merged, the first step
// of each with the other run turned round.
__device__ __forceinline__ void sort64(std::uint64_t& v, int lane) {
    order<1>(v, lane);
    order<3>(v, lane), order<1>(v, lane);
    order<7>(v, lane), order<2>(v, lane), order<1>(v, lane);
    order<15>(v, lane), order<4>(v, lane), order<2>(v, lane), order<1>(v, lane);
    order<31>(v, lane), order<8>(v, lane), order<4>(v, lane), order<2>(v, lane), order<1>(v, lane);
    order<63>(v, lane), order<16>(v, lane), order<8>(v, lane), order<4>(v, lane), order<2>(v, lane), order<1>(v, lane);
}

// One action a lane: what top_k (0: all) and top_p leave; weights of the rest become
// zero.  share: of all, where the lanes do not hold all; else 0.
__device__ __forceinline__ void keep64(float x, double& w, double top_p, int top_k, double share) {
    const int lane = threadIdx.x % 64;
    const std::uint32_t key = key_of(x);
    std::uint64_t v = static_cast<std::uint64_t>(key) << 32 | static_cast<std::uint32_t>(63 - lane);
    sort64(v, lane);
    const int place = 63 - static_cast<int>(v & 63u);
    const auto bits = __builtin_bit_cast(std::uint64_t, w);
    const std::uint32_t lo = __shfl(static_cast<int>(bits), place), hi = __shfl(static_cast<int>(bits >> 32), place);
    double sorted = __builtin_bit_cast(double, static_cast<std::uint64_t>(hi) << 32 | lo);
    if (top_k > 0 && lane >= top_k) sorted = 0.0;
    const double upto = scan64(sorted);
    if (share == 0.0) share = top_p * of_lane(upto, 63);
    // In this order what stays is a beginning of it.
    const int kept = lanes_in(__ballot(sorted > 0.0 && (top_p >= 1.0 || lane == 0 || upto - sorted < share)));
    const std::uint32_t border = of_lane(static_cast<std::uint32_t>(v >> 32), kept - 1);
    // Read here, with all lanes: under the condition the others' places need not be there.
    const int last = of_lane(place, kept - 1);
    if (key < border || (key == border && lane > last)) w = 0.0;
}

// What top_p leaves: weights of the rest become zero.  low and high: no score that has a
// weight is outside.
template <int E>
__device__ __forceinline__ void nucleus(const float (&x)[E], double (&w)[E], double top_p, std::uint32_t low, std::uint32_t high) {
    std::uint32_t key[E];
    float light[E];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        key[i] = key_of(x[i]);
        light[i] = static_cast<float>(w[i]);
        sum += w[i];
    }
    const double share = top_p * sum64(sum);
    const float about = static_cast<float>(share);
    // The border is the largest score at or above which the weights reach the share.
    // border: they do; beyond: they do not (0: none such is known).
    // Bits that low and high share are the border's too.
    std::uint32_t bit = low == high ? 0u : 0x80000000u >> __clz(static_cast<int>(low ^ high));
    std::uint32_t border = bit == 0 ? low : high & ~(2 * bit - 1), beyond = 0;
    for (; bit != 0; bit >>= 1) {
        const std::uint32_t at = border | bit;
        float reached = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) reached += key[i] >= at ? light[i] : 0.0f;
        if (sum64(reached) >= about) border = at;
        else beyond = at;
        if (beyond == 0) continue;
        int left = 0;
        std::uint32_t only = border;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const std::uint64_t between = __ballot(key[i] >= border && key[i] < beyond);
            left += lanes_in(between);
            if (between != 0) only = of_lane(key[i], first_lane(between));
        }
        if (left == 1) {
            border = only;
            break;
        }
    }
    const auto above = [&](std::uint32_t at, bool or_at) {
        double v = 0.0;
#pragma unroll
        for (int i = 0; i < E; ++i) v += key[i] > at || (or_at && key[i] == at) ? w[i] : 0.0;
        return sum64(v);
    };
    double before = above(border, false);
    if (!(before < share && above(border, true) >= share)) {
        border = 0;
        for (bit = 0x80000000u; bit != 0; bit >>= 1)
            if (above((border | bit) - 1, false) >= share) border |= bit;
        before = above(border, false);
    }
    // Of equal scores at the border the first few by index stay.
    int ahead = 0;
    double each = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const std::uint64_t here = __ballot(key[i] == border);
        if (here != 0) each = of_lane(w[i], first_lane(here));
        ahead += lanes_below(here);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const bool stays = key[i] > border || (key[i] == border && before + ahead * each < share);
        ahead += key[i] == border;
        if (!stays) w[i] = 0.0;
    }
}

// A row's answer, and what its log probability is the logarithm of the quotient of.
struct Answer {
    int action;
    double chosen, all;
};

// The action that the uniform number falls on, as its place E lane + i.
template <int E>
__device__ __forceinline__ Answer pick(const float (&x)[E], float most, const Settings& set, std::uint32_t low, int top_k, double share = 0.0) {
    double w[E], sum = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = set.weight(x[i], most);
    if constexpr (E == 1) {
        if (set.top_p < 1.0 || top_k > 0) keep64(x[0], w[0], set.top_p, top_k, share);
    } else if (set.top_p < 1.0) {
        nucleus(x, w, set.top_p, low, key_of(most));
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (w[i] < set.min_p) w[i] = 0.0;
        sum += w[i];
    }
    const double upto = scan64(sum), all = of_lane(upto, 63), target = (set.u > 0.0 ? set.u : 0.0) * all;
    // The first place at which the running sum exceeds the target; if rounding or u
    // leaves none, the last one of any weight.
    double run = upto - sum;
    int past = E, last = -1;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        run += w[i];
        if (w[i] > 0.0) {
            last = i;
            if (past == E && run > target) past = i;
        }
    }
    const std::uint64_t have = __ballot(past < E);
    const int of = have != 0 ? first_lane(have) : last_lane(__ballot(last >= 0));
    const int mine = have != 0 ? past : last;
    double chosen = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) chosen = mine == i ? w[i] : chosen;
    return {E * of + of_lane(mine, of), of_lane(chosen, of), all};
}

constexpr int kWaves = 4;      // of a workgroup: they do not meet

// A row's scores, E a lane.
template <typename T, int E>
__device__ __forceinline__ void load_row(const SampleArgs<T>& a, std::uint32_t r, int lane, float (&x)[E]) {
    const T* from = a.logits.row(r / a.batch, r % a.batch, 0);
    if (E > 1 && a.logits.vec && a.actions % 4 == 0) {
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
            const std::uint32_t at = E * lane + 4 * i;
            const f4 v = at < a.actions ? load4(from + at, true) : f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = v[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = E * lane + i < a.actions ? static_cast<float>(from[E * lane + i]) : -INFINITY;
    }
}

// What top_k leaves of the scores, of which the largest is `most`: the others become
// -infinity.  Returns a number that none of them is above and none that is left below;
// with `move` what is left lies, in order, in scores and places.
template <int E>
__device__ __forceinline__ float largest(float (&x)[E], float most, int count, bool move, int lane, float* scores, int* places, int& kept) {
    // One that just `count` scores are not below, if there is, by halving the range.
    float least = INFINITY;
    int all = 0, at_most = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        least = x[i] > -INFINITY ? fminf(least, x[i]) : least;
        all += lanes_in(__ballot(x[i] > -INFINITY));
        at_most += lanes_in(__ballot(x[i] == most));
    }
    least = -most16(-least);
    least = fminf(fminf(of_lane(least, 0), of_lane(least, 16)), fminf(of_lane(least, 32), of_lane(least, 48)));
    float border = at_most >= count ? most : least;
    int reached = at_most >= count ? at_most : all;        // not below it
    if (at_most < count && all > count) {
        float beyond = most;           // fewer are not below it; more are not below the border
        for (;;) {
            const float half = 0.5f * border + 0.5f * beyond;
            if (!(half > border && half < beyond)) break;      // next to each other: equal scores at the border
            int now = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) now += lanes_in(__ballot(x[i] >= half));
            if (now < count) {
                beyond = half;
                continue;
            }
            border = half;
            reached = now;
            if (now == count) break;
        }
    }
    // Of equal scores at the border the first few by index stay.
    bool stays[E];
    kept = 0;
    if (reached <= count) {
#pragma unroll
        for (int i = 0; i < E; ++i) stays[i] = x[i] >= border;
    } else {
        int left = count;
#pragma unroll
        for (int i = 0; i < E; ++i) left -= lanes_in(__ballot(x[i] > border)) + lanes_below(__ballot(x[i] == border));
#pragma unroll
        for (int i = 0; i < E; ++i) {
            stays[i] = x[i] > border || (x[i] == border && left > 0);
            left -= x[i] == border;
        }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        kept += lanes_below(__ballot(stays[i]));
        if (!stays[i]) x[i] = -INFINITY;
    }
    if (move) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (stays[i]) {
                scores[kept] = x[i];
                places[kept] = E * lane + i;
                ++kept;
            }
        kept = of_lane(kept, 63);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();       // in order within the wave
    }
    return border;
}

// A wave takes `each` rows one after the other; settings and log probabilities are
// worked out for all of them at once, a row a lane.
template <typename T, int E>
__global__ void __launch_bounds__(64 * kWaves, E == 16 ? 3 : E == 4 ? 6 : 8) sample64_kernel(SampleArgs<T> a, int each) {
    __shared__ float scores[kWaves][64];
    __shared__ int places[kWaves][64];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const std::uint64_t begin = (block_of() * kWaves + wave) * each;
    if (begin >= a.rows) return;
    const int count = static_cast<int>(a.rows - begin < static_cast<std::uint64_t>(each) ? a.rows - begin : each);
    const auto first = static_cast<std::uint32_t>(begin);
    const Settings mine(a, first + min(lane, count - 1));
    const bool mine_fine = mine.fine();
    Answer answer{-1, NAN, 1.0};
    float next[E];
    load_row<T, E>(a, first, lane, next);
    for (int j = 0; j < count; ++j) {
        float x[E], most = -INFINITY;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x[i] = next[i];
            odd |= !(x[i] < INFINITY);                 // NaN or +infinity
            most = fmaxf(most, x[i]);
        }
        if (j + 1 < count) load_row<T, E>(a, first + j + 1, lane, next);
        most = most16(most);
        most = fmaxf(fmaxf(of_lane(most, 0), of_lane(most, 16)), fmaxf(of_lane(most, 32), of_lane(most, 48)));
        if (__any(odd) || !(most > -INFINITY) || of_lane(static_cast<int>(mine_fine), j) == 0) continue;
        Settings set = mine;
        set.temperature = of_lane(mine.temperature, j);
        set.inverse = of_lane(mine.inverse, j);
        set.top_p = of_lane(mine.top_p, j);
        set.min_p = of_lane(mine.min_p, j);
        set.u = of_lane(mine.u, j);
        set.top_k = of_lane(mine.top_k, j);
        Answer found;
        if (set.temperature == 0.0) {                  // the largest, the first of equal ones
            int best = E;
#pragma unroll
            for (int i = E - 1; i >= 0; --i) best = x[i] == most ? i : best;
            const int of = first_lane(__ballot(best < E));
            found = {E * of + of_lane(best, of), 1.0, 1.0};
        } else if constexpr (E == 1) {
            found = pick<1>(x, most, set, 0, set.top_k);
        } else {
            const auto of_moved = [&](int kept, double share) {
                const float one[1] = {lane < kept ? scores[wave][lane] : -INFINITY};
                Answer got = pick<1>(one, most, set, 0, 0, share);
                got.action = places[wave][got.action];
                return got;
            };
            const bool narrow = set.top_k > 0 && set.top_k < static_cast<int>(a.actions);
            float border = -INFINITY;
            int kept;
            if (narrow) border = largest<E>(x, most, set.top_k, set.top_k <= 64, lane, scores[wave], places[wave], kept);
            if (narrow && set.top_k <= 64) {
                found = of_moved(kept, 0.0);
            } else if (set.top_p < 1.0) {
                // Where the 64 largest reach the share, no other stays.
                double sum = 0.0;
                float y[E];
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    sum += set.weight(x[i], most);
                    y[i] = x[i];
                }
                const double share = set.top_p * sum64(sum);
                largest<E>(y, most, 64, true, lane, scores[wave], places[wave], kept);
                const double held = set.weight(lane < kept ? scores[wave][lane] : -INFINITY, most);
                if (sum64(held) >= share) found = of_moved(kept, share);
                else found = pick<E>(x, most, set, key_of(border), 0);
            } else {
                found = pick<E>(x, most, set, 0, 0);
            }
        }
        if (lane == j) answer = found;
    }
    if (lane < count) {
        a.action[first + lane] = answer.action;
        a.logprob[first + lane] = static_cast<float>(log(answer.chosen / answer.all));
    }
}

template <typename T>
int sample(const char* who, const nesle_sample_args& x, hipStream_t s) {
    const SampleArgs<T> a{heads<T>(x.logits), x.uniform, x.temperature, x.top_p, x.min_p, std::min(x.top_k, x.actions), x.temperatures, x.top_ps,
                          x.min_ps, x.top_ks, x.action, x.logprob, x.steps * x.batch, x.batch, x.actions};
    const dim3 block(256);
    if (x.actions <= 16) {
        hipLaunchKernelGGL((sample16_kernel<T>), grid_of((a.rows + 15) / 16), block, 0, s, a);
        return launched(who);
    }
    // As many rows a wave as leave the card twice the waves that it holds.  65,536 rows of
    // 256 with 1, 2, 4 and 8 a wave, us: 60, 48, 41, 39 unfiltered, 130, 118, 117, 123 with limits.
    const int each = static_cast<int>(std::min(std::max(a.rows / 16384, 1u), 16u));
    const std::uint32_t rows = kWaves * static_cast<std::uint32_t>(each);
    const dim3 grid = grid_of((a.rows + rows - 1) / rows);
    if (x.actions <= 64) hipLaunchKernelGGL((sample64_kernel<T, 1>), grid, block, 0, s, a, each);
    else if (x.actions <= 256) hipLaunchKernelGGL((sample64_kernel<T, 4>), grid, block, 0, s, a, each);
    else hipLaunchKernelGGL((sample64_kernel<T, 16>), grid, block, 0, s, a, each);
    return launched(who);
}

}  // namespace
}  // namespace nesle::mem

using namespace nesle::mem;

extern "C" int nesle_sample(const nesle_sample_args* a, void* stream) {
    const char* who = "nesle_sample";
    if (a == nullptr) return refuse(who, "null arguments");
    if (a->dtype != NESLE_MEM_F32 && a->dtype != NESLE_MEM_BF16) return refuse(who, "dtype must be NESLE_MEM_F32 or NESLE_MEM_BF16");
    if (a->actions == 0 || a->actions > NESLE_SAMPLE_MAX_ACTIONS)
        return refuse(who, "actions must be 1 to " + std::to_string(NESLE_SAMPLE_MAX_ACTIONS));
    if (static_cast<std::uint64_t>(a->steps) * a->batch > (1ull << 30)) return refuse(who, "rows must be at most 2^30");
    if (a->temperatures == nullptr && (!(a->temperature >= 0.0) || !(a->temperature < INFINITY)))
        return refuse(who, "temperature must be finite and not below 0");
    if (a->top_ps == nullptr && (!(a->top_p > 0.0) || !(a->top_p <= 1.0))) return refuse(who, "top_p must be above 0 and at most 1");
    if (a->min_ps == nullptr && (!(a->min_p >= 0.0) || !(a->min_p <= 1.0))) return refuse(who, "min_p must be 0 to 1");
    if (a->steps == 0 || a->batch == 0) return NESLE_OK;
    if (!a->logits.data || !a->uniform || !a->action || !a->logprob) return refuse(who, "null device pointer");
    const auto s = static_cast<hipStream_t>(stream);
    return a->dtype == NESLE_MEM_F32 ? sample<float>(who, *a, s) : sample<bf16>(who, *a, s);
}
