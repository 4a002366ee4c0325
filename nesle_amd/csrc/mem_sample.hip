// Sampling of actions from given random numbers (include/nesle_memory.h has the
// rules).
//
// A row's scores are held in the registers of a group of lanes, lane l those of the
// actions l E .. l E + E - 1, so that the order of actions is the order of lanes.
// Which actions are left and which one a uniform number falls on turn on comparisons
// of sums, so weights and sums are float64: in float32 a border would be off by up to
// 2^-24 of the whole, and one row in 10^5 or so would get another action than the
// rules say.
//
// top_k and top_p need the actions in order of falling weight only up to a border.
// The border is found without sorting: scores become whole numbers of the same order,
// and the bits of the one at the border are found from the top, each by one sum over
// the group of what lies above a candidate.  Of equal scores at the border the first
// few by index stay.
#include "mem_delta_math.h"

namespace nesle::mem {
namespace {

template <typename T>
struct SampleArgs {
    Heads<T> logits;
    const float* uniform;
    double temperature, top_p, min_p;
    std::uint32_t top_k;
    const float *temperatures, *top_ps, *min_ps;
    const std::int32_t* top_ks;
    std::int64_t* action;
    float* logprob;
    std::uint32_t rows, batch, actions;
};

// Sums over the L lanes of a group, in all of them.
template <int L, typename X>
__device__ X group_sum(X v) {
#pragma unroll
    for (int d = 1; d < L; d *= 2) v += __shfl_xor(v, d);
    return v;
}
// Over the lanes below, of the group.
template <int L, typename X>
__device__ X group_below(X v, unsigned lane) {
    X sum = v;
#pragma unroll
    for (int d = 1; d < L; d *= 2) {
        const X below = __shfl_up(sum, d, L);
        if (lane >= d) sum += below;
    }
    return sum - v;
}

// Whole numbers in the order of the floats; -0 as 0.
__device__ std::uint32_t key_of(float x) {
    const std::uint32_t b = __builtin_bit_cast(std::uint32_t, x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T, int L, int E>
__global__ void __launch_bounds__(256) sample_kernel(SampleArgs<T> a) {
    const unsigned lane = threadIdx.x % L;
    const std::uint64_t row = (blockIdx.x * 256ull + threadIdx.x) / L;
    if (row >= a.rows) return;                         // whole groups, and nobody waits for them
    const std::uint32_t r = static_cast<std::uint32_t>(row), first = lane * E;
    const T* from = a.logits.row(r / a.batch, r % a.batch, 0);
    float x[E];
    float most = -INFINITY;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        x[i] = first + i < a.actions ? static_cast<float>(from[first + i]) : -INFINITY;
        odd |= !(x[i] < INFINITY);                     // NaN or +infinity
        most = fmaxf(most, x[i]);
    }
    const double temperature = a.temperatures != nullptr ? a.temperatures[r] : a.temperature;
    const double top_p = a.top_ps != nullptr ? a.top_ps[r] : a.top_p;
    const double min_p = a.min_ps != nullptr ? a.min_ps[r] : a.min_p;
    const auto top_k = a.top_ks != nullptr ? std::int64_t{a.top_ks[r]} : std::int64_t{a.top_k};
    const double u = a.uniform[r];
#pragma unroll
    for (int d = 1; d < L; d *= 2) {
        most = fmaxf(most, __shfl_xor(most, d));
        odd |= __shfl_xor(static_cast<int>(odd), d) != 0;
    }
    const bool fine = !odd && most > -INFINITY && temperature >= 0.0 && temperature < INFINITY && top_p > 0.0 &&
                      top_p <= 1.0 && min_p >= 0.0 && min_p <= 1.0 && top_k >= 0 && u == u;
    if (!fine) {
        if (lane == 0) {
            a.action[r] = -1;
            a.logprob[r] = NAN;
        }
        return;
    }
    double w[E];
    std::uint32_t key[E];
    if (temperature == 0.0) {                          // the largest, the first of equal ones
        std::uint32_t best = 0xffffffffu;
#pragma unroll
        for (int i = E - 1; i >= 0; --i) best = x[i] == most ? first + i : best;
#pragma unroll
        for (int d = 1; d < L; d *= 2) best = min(best, static_cast<std::uint32_t>(__shfl_xor(static_cast<int>(best), d)));
        if (lane == 0) {
            a.action[r] = best;
            a.logprob[r] = 0.0f;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        // The difference first: a quotient may pass the largest number.
        w[i] = x[i] > -INFINITY ? exp((static_cast<double>(x[i]) - most) / temperature) : 0.0;
        key[i] = x[i] > -INFINITY ? key_of(x[i]) : 0u;
    }
    if (top_k > 0 && top_k < a.actions) {
        // The k-th largest: the largest number that k or more are not below.
        std::uint32_t border = 0;
        for (std::uint32_t bit = 0x80000000u; bit != 0; bit >>= 1) {
            int count = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) count += key[i] >= (border | bit);
            if (group_sum<L>(count) >= top_k) border |= bit;
        }
        int above = 0, equal = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            above += key[i] > border;
            equal += key[i] == border;
        }
        int left = static_cast<int>(top_k) - group_sum<L>(above) - group_below<L>(equal, lane);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const bool stays = key[i] > border || (key[i] == border && left > 0);
            left -= key[i] == border;
            if (!stays) {
                w[i] = 0.0;
                key[i] = 0u;
            }
        }
    }
    if (top_p < 1.0) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < E; ++i) sum += w[i];
        const double most_before = top_p * group_sum<L>(sum);
        // The smallest score that some action may have and stay: the largest number
        // at or above which the weights reach the share.
        std::uint32_t border = 0;
        for (std::uint32_t bit = 0x80000000u; bit != 0; bit >>= 1) {
            double reached = 0.0;
#pragma unroll
            for (int i = 0; i < E; ++i) reached += key[i] >= (border | bit) ? w[i] : 0.0;
            if (group_sum<L>(reached) >= most_before) border |= bit;
        }
        double above = 0.0, at_border = 0.0;
        int equal = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            above += key[i] > border ? w[i] : 0.0;
            at_border = key[i] == border ? w[i] : at_border;
            equal += key[i] == border;
        }
        above = group_sum<L>(above);
#pragma unroll
        for (int d = 1; d < L; d *= 2) at_border = fmax(at_border, __shfl_xor(at_border, d));
        int ahead = group_below<L>(equal, lane);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const bool stays = key[i] > border || (key[i] == border && above + ahead * at_border < most_before);
            ahead += key[i] == border;
            if (!stays) w[i] = 0.0;
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (w[i] < min_p) w[i] = 0.0;
        sum += w[i];
    }
    const double below = group_below<L>(sum, lane), all = group_sum<L>(sum), target = (u > 0.0 ? u : 0.0) * all;
    // The first action at which the running sum exceeds the target; if rounding or u
    // leaves none, the last one of any weight.
    double run = below;
    std::uint32_t found = 0xffffffffu, last = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        run += w[i];
        if (w[i] > 0.0) {
            last = first + i + 1;
            if (run > target && found == 0xffffffffu) found = first + i;
        }
    }
#pragma unroll
    for (int d = 1; d < L; d *= 2) {
        found = min(found, static_cast<std::uint32_t>(__shfl_xor(static_cast<int>(found), d)));
        last = max(last, static_cast<std::uint32_t>(__shfl_xor(static_cast<int>(last), d)));
    }
    if (found == 0xffffffffu) found = last - 1;
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (first + i == found) {
            a.action[r] = found;
            a.logprob[r] = static_cast<float>(log(w[i] / all));
        }
}

template <typename T>
int sample(const char* who, const nesle_sample_args& x, hipStream_t s) {
    const SampleArgs<T> a{heads<T>(x.logits), x.uniform, x.temperature, x.top_p, x.min_p, x.top_k, x.temperatures, x.top_ps,
                          x.min_ps, x.top_ks, x.action, x.logprob, x.steps * x.batch, x.batch, x.actions};
    const int lanes = x.actions <= 16 ? 16 : 64;
    const std::uint32_t rows = 256 / lanes;
    const dim3 grid((a.rows + rows - 1) / rows), block(256);
    if (x.actions <= 16) hipLaunchKernelGGL((sample_kernel<T, 16, 1>), grid, block, 0, s, a);
    else if (x.actions <= 64) hipLaunchKernelGGL((sample_kernel<T, 64, 1>), grid, block, 0, s, a);
    else if (x.actions <= 256) hipLaunchKernelGGL((sample_kernel<T, 64, 4>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((sample_kernel<T, 64, 16>), grid, block, 0, s, a);
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
