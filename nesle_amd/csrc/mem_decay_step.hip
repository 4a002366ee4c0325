// One token of linear attention with a decay for each head, for every console
// (acting): each state is read once and written once, which is all the work there
// is (8 bytes an element against 5 operations), so the kernel is bound by memory,
// and by latency for a few consoles: 8,192 consoles of 4 heads of 64 x 64, 1.09 GB in 207
// us (5.3 TB/s); one console 4 us, a launch.
//
// A wave holds all k_dim rows of 16 columns of one state in registers, four columns a
// lane: 16 lanes share the rows of a column group.  A row's loads are then 64 bytes
// together, and one console's 4 heads of 64 are 16 waves.  Columns do not interact,
// so nothing crosses a wave and the state may be updated in place:
//   S <- a S + k v^T,  out = scale S^T q
#include "mem_decay.h"

namespace nesle::mem {
namespace {

constexpr unsigned kWaves = 4;      // waves of a workgroup; they do not meet
constexpr unsigned kCols = 16;

template <typename T, int ROWS>      // ROWS: rows a lane holds
__global__ void __launch_bounds__(64 * kWaves) decay_step_kernel(DecayArgs<T> a, std::uint32_t slices, std::uint32_t waves) {
    constexpr unsigned V = kCols / 4, R = 64 / V;      // lanes along columns, along rows
    const std::uint32_t w = blockIdx.x * kWaves + threadIdx.x / 64;
    if (w >= waves) return;                            // whole waves: nobody waits for them
    const unsigned lane = threadIdx.x % 64, r0 = lane / V;
    const std::uint32_t head_of_all = w / slices;
    const unsigned col = (w % slices) * kCols + 4 * (lane % V);
    const std::uint32_t env = head_of_all / a.hv, h = head_of_all % a.hv;
    const bool in_cols = col < a.dv_dim;
    const std::size_t at = static_cast<std::size_t>(head_of_all);
    const float* S = a.state + at * a.dk_dim * a.dv_dim + col;
    const float g = a.g[h];
    const bool keep = a.state != nullptr && !(a.resets != nullptr && a.resets[env] != 0) && !(g < kDropBelow);
    const float decay = expf(g);

    const T* q = a.q.row(0, env, h / a.group);
    const T* k = a.k.row(0, env, h / a.group);
    f4 D[ROWS];
    float kr[ROWS], qr[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const unsigned row = r0 + R * i;
        const bool in = row < a.dk_dim;
        D[i] = in && in_cols && keep ? *reinterpret_cast<const f4*>(S + static_cast<std::size_t>(row) * a.dv_dim) : f4{0, 0, 0, 0};
        kr[i] = in ? static_cast<float>(k[row]) : 0.0f;
        qr[i] = in ? static_cast<float>(q[row]) : 0.0f;
    }
    const f4 v = in_cols ? load4(a.v.row(0, env, h) + col, a.v.vec) : f4{0, 0, 0, 0};
    f4 sq = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (keep) D[i] *= decay;
        if (r0 + R * i < a.dk_dim) {
            D[i] += v * kr[i];
            sq += D[i] * qr[i];
        }
    }
    for (unsigned d = V; d < 64; d *= 2) sq += f4{__shfl_xor(sq.x, d), __shfl_xor(sq.y, d), __shfl_xor(sq.z, d), __shfl_xor(sq.w, d)};
    if (!in_cols) return;
    float* to = a.state_out + at * a.dk_dim * a.dv_dim + col;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const unsigned row = r0 + R * i;
        if (row < a.dk_dim) *reinterpret_cast<f4*>(to + static_cast<std::size_t>(row) * a.dv_dim) = D[i];
    }
    if (r0 == 0) store4(a.out + at * a.dv_dim + col, sq * a.scale);
}

template <typename T>
int step(const char* who, const nesle_decay_args& x, hipStream_t s) {
    const DecayArgs<T> a = decay_args<T>(x);
    const std::uint32_t slices = (a.dv_dim + kCols - 1) / kCols;
    const std::uint32_t waves = a.batch * a.hv * slices;
    const dim3 grid((waves + kWaves - 1) / kWaves), block(64 * kWaves);
    if (a.dk_dim <= 32)
        hipLaunchKernelGGL((decay_step_kernel<T, 2>), grid, block, 0, s, a, slices, waves);
    else if (a.dk_dim <= 64)
        hipLaunchKernelGGL((decay_step_kernel<T, 4>), grid, block, 0, s, a, slices, waves);
    else
        hipLaunchKernelGGL((decay_step_kernel<T, 8>), grid, block, 0, s, a, slices, waves);
    return launched(who);
}

}  // namespace
}  // namespace nesle::mem

using namespace nesle::mem;

extern "C" int nesle_decay_step(const nesle_decay_args* a, void* stream) {
    const char* who = "nesle_decay_step";
    int rc = check_decay(who, a);
    if (rc != NESLE_OK) return rc;
    if (a->steps != 1) return refuse(who, "steps must be 1");
    if (a->batch == 0) return NESLE_OK;
    rc = check_decay_alignment(who, a);
    if (rc == NESLE_OK) rc = check_decay_inputs(who, a);
    if (rc != NESLE_OK) return rc;
    if (!a->out || !a->state_out) return refuse(who, "null device pointer");
    const auto s = static_cast<hipStream_t>(stream);
    return a->dtype == NESLE_MEM_F32 ? step<float>(who, *a, s) : step<bf16>(who, *a, s);
}
