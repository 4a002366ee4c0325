// One token of the gated delta rule for every console (acting): each state is
// read once and written once, which is all the work there is (8 bytes an
// element against 7 operations), so the kernel is bound by memory, and by
// latency for a few consoles.  Measured against a large copy's 4.9 TB/s: 8,192
// consoles of 4 heads of 64 x 64, 1.09 GB in 207 us (5.3 TB/s); 1,000 of 6 heads
// of 48 x 40 in float32, 95 MB in 22.6 us (4.2 TB/s); one console 3.9 us, a launch.
//
// A wave holds all k_dim rows of COLS columns of one state in registers, four
// columns a lane: 64 / (COLS / 4) lanes share the rows of a column group.  With 16
// columns a row's loads are 64 bytes together, and one console's 4 heads of 64 are
// 16 waves.  Columns do not interact, so nothing crosses a wave and the state may be
// updated in place.  With D = a S (S^T k and S^T q read in one pass):
//   u = beta (v - D^T k),  out = scale (D^T q + (k . q) u),  S <- D + k u^T
#include "mem_delta.h"

namespace nesle::mem {
namespace {

constexpr unsigned kWaves = 4;      // waves of a workgroup; they do not meet

template <typename T, int COLS, int ROWS>      // ROWS: rows a lane holds
__global__ void __launch_bounds__(64 * kWaves) delta_step_kernel(DeltaArgs<T> a, std::uint32_t slices, std::uint32_t waves) {
    constexpr unsigned V = COLS / 4, R = 64 / V;       // lanes along columns, along rows
    const std::uint32_t w = blockIdx.x * kWaves + threadIdx.x / 64;
    if (w >= waves) return;                            // whole waves: nobody waits for them
    const unsigned lane = threadIdx.x % 64, r0 = lane / V;
    const std::uint32_t head_of_all = w / slices;
    const unsigned col = (w % slices) * COLS + 4 * (lane % V);
    const std::uint32_t env = head_of_all / a.hv, h = head_of_all % a.hv;
    const bool in_cols = col < a.dv_dim;
    const std::size_t at = static_cast<std::size_t>(head_of_all);
    const float* S = a.state + at * a.dk_dim * a.dv_dim + col;
    const bool keep = a.state != nullptr && !(a.resets != nullptr && a.resets[env] != 0) && !(a.g[at] < kDropBelow);
    const float decay = expf(a.g[at]), beta = a.beta[at];

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
    f4 sk = {0, 0, 0, 0}, sq = sk;
    float kq = 0.0f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (keep) D[i] *= decay;
        sk += D[i] * kr[i];
        sq += D[i] * qr[i];
        kq += kr[i] * qr[i];
    }
    for (unsigned d = V; d < 64; d *= 2) {
        sk += f4{__shfl_xor(sk.x, d), __shfl_xor(sk.y, d), __shfl_xor(sk.z, d), __shfl_xor(sk.w, d)};
        sq += f4{__shfl_xor(sq.x, d), __shfl_xor(sq.y, d), __shfl_xor(sq.z, d), __shfl_xor(sq.w, d)};
        kq += __shfl_xor(kq, d);
    }
    const f4 u = (v - sk) * beta;
    if (!in_cols) return;
    float* to = a.state_out + at * a.dk_dim * a.dv_dim + col;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const unsigned row = r0 + R * i;
        if (row < a.dk_dim) *reinterpret_cast<f4*>(to + static_cast<std::size_t>(row) * a.dv_dim) = D[i] + u * kr[i];
    }
    if (r0 == 0) store4(a.out + at * a.dv_dim + col, (sq + u * kq) * a.scale);
}

template <typename T, int COLS>
void launch_cols(const DeltaArgs<T>& a, hipStream_t s) {
    constexpr int R = 64 / (COLS / 4);
    const std::uint32_t slices = (a.dv_dim + COLS - 1) / COLS;
    const std::uint32_t waves = a.batch * a.hv * slices;
    const dim3 grid((waves + kWaves - 1) / kWaves), block(64 * kWaves);
    if (a.dk_dim <= 32)
        hipLaunchKernelGGL((delta_step_kernel<T, COLS, 32 / R>), grid, block, 0, s, a, slices, waves);
    else if (a.dk_dim <= 64)
        hipLaunchKernelGGL((delta_step_kernel<T, COLS, 64 / R>), grid, block, 0, s, a, slices, waves);
    else
        hipLaunchKernelGGL((delta_step_kernel<T, COLS, 128 / R>), grid, block, 0, s, a, slices, waves);
}

template <typename T>
int step(const char* who, const nesle_delta_args& x, hipStream_t s) {
    launch_cols<T, 16>(delta_args<T>(x), s);
    return launched(who);
}

}  // namespace
}  // namespace nesle::mem

using namespace nesle::mem;

extern "C" int nesle_delta_step(const nesle_delta_args* a, void* stream) {
    const char* who = "nesle_delta_step";
    int rc = check_delta(who, a);
    if (rc != NESLE_OK) return rc;
    if (a->steps != 1) return refuse(who, "steps must be 1");
    if (a->batch == 0) return NESLE_OK;
    rc = check_delta_inputs(who, a);
    if (rc != NESLE_OK) return rc;
    if (!a->out || !a->state_out) return refuse(who, "null device pointer");
    const auto s = static_cast<hipStream_t>(stream);
    return a->dtype == NESLE_MEM_F32 ? step<float>(who, *a, s) : step<bf16>(who, *a, s);
}
