// Norms of queries and keys for each head with the position rotation, and the
// gradient (include/nesle_memory.h has the formulas).
//
// One pass: a group of lanes holds one head in registers, eight elements a
// lane, so the sum of squares is a few lane exchanges and every element is
// read and written once.  A lane's eight elements are four from the first
// half of the rotated part and the four they are paired with in the second
// half (two loads), so that a pair never crosses lanes in either layout;
// lanes past the rotated part hold eight consecutive ones.
//
// Bound by memory: about 10 operations an element.
#include "mem_common.h"

namespace nesle::mem {
namespace {

constexpr unsigned kThreads = 256;
// Workgroups of the gradient with weights: each adds up its rows' share of
// the weights' gradient, and one more launch adds the workgroups' in order.
constexpr unsigned kGradBlocks = 1024;

template <typename T>
struct QkArgs {
    Heads<T> q, k, dq_out, dk_out;
    const float *wq, *wk;
    const std::int32_t* positions;
    const float* table;
    T *q_out, *k_out;        // forward: outputs; gradient: dq, dk
    float* partials;         // [blocks][2][dim]
    std::uint32_t batch, hq, hk, dim, rotated, table_rows, lanes;   // lanes of one head: a power of two
    std::uint64_t groups;    // heads of all rows
    float inv_count, eps;
    bool interleaved;
};

// The two element offsets of lane j's groups of four.
template <typename T>
__device__ void places(const QkArgs<T>& a, unsigned j, unsigned& first, unsigned& second) {
    if (8 * j >= a.rotated || a.interleaved) {
        first = 8 * j;
        second = first + 4;
    } else {
        first = 4 * j;
        second = a.rotated / 2 + first;
    }
}

// Cosines and sines of a lane's four pairs.
template <typename T>
__device__ void turns(const QkArgs<T>& a, std::uint64_t row, unsigned j, f4& c, f4& s) {
    const std::int32_t p = a.positions[row];
    if (p < 0 || static_cast<std::uint32_t>(p) >= a.table_rows) {
        c = s = f4{NAN, NAN, NAN, NAN};
        return;
    }
    const float* t = a.table + static_cast<std::size_t>(p) * a.rotated + 4 * j;
    c = *reinterpret_cast<const f4*>(t);
    s = *reinterpret_cast<const f4*>(t + a.rotated / 2);
}

// Turn (x, y), the lane's two groups, by the angles (c, s); sign -1 turns back.
__device__ inline void turn(f4& x, f4& y, f4 c, f4 s, bool interleaved) {
    if (interleaved) {
        const f4 u = {x.x * c.x - x.y * s.x, x.x * s.x + x.y * c.x, x.z * c.y - x.w * s.y, x.z * s.y + x.w * c.y};
        const f4 w = {y.x * c.z - y.y * s.z, y.x * s.z + y.y * c.z, y.z * c.w - y.w * s.w, y.z * s.w + y.w * c.w};
        x = u;
        y = w;
    } else {
        const f4 u = x * c - y * s;
        y = x * s + y * c;
        x = u;
    }
}

__device__ inline float across(float v, unsigned lanes) {
    for (unsigned d = 1; d < lanes; d *= 2) v += __shfl_xor(v, d);
    return v;
}

__device__ inline float dot(f4 a, f4 b) { return a.x * b.x + a.y * b.y + a.z * b.z + a.w * b.w; }

template <typename T>
__global__ void __launch_bounds__(kThreads) qk_forward(QkArgs<T> a) {
    const unsigned j = threadIdx.x % a.lanes;
    const std::uint64_t group = (static_cast<std::uint64_t>(blockIdx.x) * kThreads + threadIdx.x) / a.lanes;
    const bool mine = group < a.groups && 8 * j < a.dim;
    const std::uint32_t per_row = a.hq + a.hk;
    const std::uint64_t row = mine ? group / per_row : 0;
    const std::uint32_t head = mine ? static_cast<std::uint32_t>(group % per_row) : 0;
    const bool is_q = head < a.hq;
    const std::uint32_t h = is_q ? head : head - a.hq;
    const Heads<T> in = is_q ? a.q : a.k;
    unsigned first, second;
    places(a, j, first, second);
    f4 x = {0, 0, 0, 0}, y = x;
    if (mine) {
        const T* p = in.row(row / a.batch, row % a.batch, h);
        x = load4(p + first, in.vec);
        y = load4(p + second, in.vec);
    }
    const float inv = 1.0f / sqrtf(across(dot(x, x) + dot(y, y), a.lanes) * a.inv_count + a.eps);
    if (!mine) return;
    x *= inv;
    y *= inv;
    const float* w = is_q ? a.wq : a.wk;
    if (w != nullptr) {
        x *= load4(w + first, true);
        y *= load4(w + second, true);
    }
    if (8 * j < a.rotated) {
        f4 c, s;
        turns(a, row, j, c, s);
        turn(x, y, c, s, a.interleaved);
    }
    T* out = (is_q ? a.q_out : a.k_out) + (row * (is_q ? a.hq : a.hk) + h) * a.dim;
    store4(out + first, x);
    store4(out + second, y);
}

// dy = the output's gradient turned back; dx = inv w dy - x inv^3 <x, w dy> / count;
// dw = sum over rows of x inv dy.
template <typename T>
__global__ void __launch_bounds__(kThreads) qk_gradient(QkArgs<T> a) {
    __shared__ f4 sums[kThreads / 64][2][2][32];       // [wave][q, k][first, second][lane of the head]
    const unsigned j = threadIdx.x % a.lanes;
    const std::uint32_t per_row = a.hq + a.hk;
    unsigned first, second;
    places(a, j, first, second);
    const bool has = 8 * j < a.dim;
    f4 dw[2][2] = {};
    const std::uint64_t at_once = static_cast<std::uint64_t>(gridDim.x) * (kThreads / a.lanes);
    // Every lane of a workgroup takes every turn, as the lane exchanges need.
    for (std::uint64_t base = static_cast<std::uint64_t>(blockIdx.x) * (kThreads / a.lanes); base < a.groups; base += at_once) {
        const std::uint64_t group = base + threadIdx.x / a.lanes;
        const bool mine = group < a.groups && has;
        const std::uint64_t row = mine ? group / per_row : 0;
        const std::uint32_t head = mine ? static_cast<std::uint32_t>(group % per_row) : 0;
        const bool is_q = head < a.hq;
        const std::uint32_t h = is_q ? head : head - a.hq;
        const Heads<T> in = is_q ? a.q : a.k;
        const Heads<T> grad = is_q ? a.dq_out : a.dk_out;
        f4 x = {0, 0, 0, 0}, y = x, dx = x, dy = x;
        if (mine) {
            const std::uint64_t t = row / a.batch, n = row % a.batch;
            const T* p = in.row(t, n, h);
            const T* d = grad.row(t, n, h);
            x = load4(p + first, in.vec);
            y = load4(p + second, in.vec);
            dx = load4(d + first, grad.vec);
            dy = load4(d + second, grad.vec);
            if (8 * j < a.rotated) {
                f4 c, s;
                turns(a, row, j, c, s);
                turn(dx, dy, c, -s, a.interleaved);
            }
        }
        const float inv = 1.0f / sqrtf(across(dot(x, x) + dot(y, y), a.lanes) * a.inv_count + a.eps);
        const float* w = is_q ? a.wq : a.wk;
        if (w != nullptr && mine) {
            dw[is_q ? 0 : 1][0] += x * inv * dx;
            dw[is_q ? 0 : 1][1] += y * inv * dy;
            dx *= load4(w + first, true);
            dy *= load4(w + second, true);
        }
        const float along = across(dot(x, dx) + dot(y, dy), a.lanes) * inv * inv * inv * a.inv_count;
        if (mine) {
            T* out = (is_q ? a.q_out : a.k_out) + (row * (is_q ? a.hq : a.hk) + h) * a.dim;
            store4(out + first, dx * inv - x * along);
            store4(out + second, dy * inv - y * along);
        }
    }
    if (a.partials == nullptr) return;
    // Lanes that hold the same elements, first within the wave, then over the
    // waves, in a fixed order.
    const unsigned lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    for (int kind = 0; kind < 2; ++kind)
        for (int half = 0; half < 2; ++half) {
            f4 v = dw[kind][half];
            for (unsigned d = a.lanes; d < 64; d *= 2)
                v += f4{__shfl_xor(v.x, d), __shfl_xor(v.y, d), __shfl_xor(v.z, d), __shfl_xor(v.w, d)};
            if (lane < a.lanes) sums[wave][kind][half][lane] = v;
        }
    __syncthreads();
    if (threadIdx.x < a.lanes && has)
        for (int kind = 0; kind < 2; ++kind)
            for (int half = 0; half < 2; ++half) {
                f4 v = sums[0][kind][half][j];
                for (unsigned u = 1; u < kThreads / 64; ++u) v += sums[u][kind][half][j];
                float* p = a.partials + (static_cast<std::size_t>(blockIdx.x) * 2 + kind) * a.dim;
                store4(p + (half ? second : first), v);
            }
}

// One element of one weight's gradient a workgroup: the partials of all
// workgroups, added in a fixed order.
__global__ void __launch_bounds__(kThreads) qk_weight_sum(const float* partials, std::uint32_t blocks,
                                                          std::uint32_t dim, float* dwq, float* dwk) {
    __shared__ float sh[kThreads];
    const std::uint32_t e = blockIdx.x;                // 0 .. 2 dim - 1
    float v = 0.0f;
    for (std::uint32_t b = threadIdx.x; b < blocks; b += kThreads) v += partials[static_cast<std::size_t>(b) * 2 * dim + e];
    sh[threadIdx.x] = v;
    __syncthreads();
    for (unsigned s = kThreads / 2; s > 0; s /= 2) {
        if (threadIdx.x < s) sh[threadIdx.x] += sh[threadIdx.x + s];
        __syncthreads();
    }
    float* out = e < dim ? dwq : dwk;
    if (threadIdx.x == 0 && out != nullptr) out[e < dim ? e : e - dim] = sh[0];
}

std::uint32_t lanes_of(std::uint32_t dim) {
    std::uint32_t n = 1;
    while (8 * n < dim) n *= 2;
    return n;
}

std::uint64_t blocks_for(const nesle_qk_args& a) {
    const std::uint64_t per = kThreads / lanes_of(a.dim);
    return (static_cast<std::uint64_t>(a.steps) * a.batch * (a.q_heads + a.k_heads) + per - 1) / per;
}

std::uint32_t grad_blocks(const nesle_qk_args& a) {
    const std::uint64_t all = blocks_for(a);
    return static_cast<std::uint32_t>(all < kGradBlocks ? all : kGradBlocks);
}

bool empty(const nesle_qk_args* a) { return a->steps == 0 || a->batch == 0; }

int check(const char* who, const nesle_qk_args* a) {
    if (a == nullptr) return refuse(who, "null arguments");
    if (a->dtype != NESLE_MEM_F32 && a->dtype != NESLE_MEM_BF16) return refuse(who, "dtype must be NESLE_MEM_F32 or NESLE_MEM_BF16");
    if (a->dim == 0 || a->dim % 8 != 0 || a->dim > NESLE_QK_MAX_DIM)
        return refuse(who, "dim must be a multiple of 8 up to " + std::to_string(NESLE_QK_MAX_DIM));
    if (a->rotated % 8 != 0 || a->rotated > a->dim) return refuse(who, "rotated must be a multiple of 8 up to dim");
    if (a->q_heads + static_cast<std::uint64_t>(a->k_heads) == 0 || a->q_heads > 65535u || a->k_heads > 65535u)
        return refuse(who, "heads must be in 1..65535");
    // One launch takes fewer than 2^32 threads of eight elements; the first
    // test keeps the second one's product below 2^64.
    if (static_cast<std::uint64_t>(a->steps) * a->batch > (1ull << 32) || blocks_for(*a) * kThreads > 0xffffffffull)
        return refuse(who, "more than 2^35 elements");
    if (!(a->eps >= 0.0f)) return refuse(who, "eps must not be negative");
    if (a->rotated != 0 && !empty(a) && (a->positions == nullptr || a->table == nullptr || a->table_rows == 0))
        return refuse(who, "the rotation needs positions and a table");
    return NESLE_OK;
}

template <typename T>
QkArgs<T> pack(const nesle_qk_args& a) {
    QkArgs<T> k{};
    k.q = heads<T>(a.q);
    k.k = heads<T>(a.k);
    k.wq = a.q_weight;
    k.wk = a.k_weight;
    k.positions = a.positions;
    k.table = a.table;
    k.batch = a.batch;
    k.hq = a.q_heads;
    k.hk = a.k_heads;
    k.dim = a.dim;
    k.rotated = a.rotated;
    k.table_rows = a.table_rows;
    k.lanes = lanes_of(a.dim);
    k.groups = static_cast<std::uint64_t>(a.steps) * a.batch * (a.q_heads + a.k_heads);
    k.inv_count = a.unit ? 1.0f : 1.0f / static_cast<float>(a.dim);
    k.eps = a.eps;
    k.interleaved = a.interleaved != 0;
    return k;
}

template <typename T>
int forward(const char* who, const nesle_qk_args& a, hipStream_t s) {
    QkArgs<T> k = pack<T>(a);
    k.q_out = static_cast<T*>(a.q_out);
    k.k_out = static_cast<T*>(a.k_out);
    hipLaunchKernelGGL(qk_forward<T>, dim3(static_cast<std::uint32_t>(blocks_for(a))), dim3(kThreads), 0, s, k);
    return launched(who);
}

template <typename T>
int gradient(const char* who, const nesle_qk_args& a, hipStream_t s) {
    QkArgs<T> k = pack<T>(a);
    k.dq_out = heads<T>(a.dq_out);
    k.dk_out = heads<T>(a.dk_out);
    k.q_out = static_cast<T*>(a.dq);
    k.k_out = static_cast<T*>(a.dk);
    const bool weights = a.q_weight != nullptr || a.k_weight != nullptr;
    k.partials = weights ? a.scratch : nullptr;
    const std::uint32_t blocks = grad_blocks(a);
    hipLaunchKernelGGL(qk_gradient<T>, dim3(blocks), dim3(kThreads), 0, s, k);
    if (weights)
        hipLaunchKernelGGL(qk_weight_sum, dim3(2 * a.dim), dim3(kThreads), 0, s, a.scratch, blocks, a.dim, a.dq_weight,
                           a.dk_weight);
    return launched(who);
}

}  // namespace
}  // namespace nesle::mem

using namespace nesle::mem;

extern "C" {

std::uint64_t nesle_qk_scratch_floats(const nesle_qk_args* a) {
    if (a == nullptr || (a->q_weight == nullptr && a->k_weight == nullptr)) return 0;
    return static_cast<std::uint64_t>(grad_blocks(*a)) * 2 * a->dim;
}

int nesle_qk_norm_rotate(const nesle_qk_args* a, void* stream) {
    const char* who = "nesle_qk_norm_rotate";
    const int rc = check(who, a);
    if (rc != NESLE_OK || empty(a)) return rc;
    if ((a->q_heads != 0 && (a->q.data == nullptr || a->q_out == nullptr)) ||
        (a->k_heads != 0 && (a->k.data == nullptr || a->k_out == nullptr)))
        return refuse(who, "null device pointer");
    const auto s = static_cast<hipStream_t>(stream);
    return a->dtype == NESLE_MEM_F32 ? forward<float>(who, *a, s) : forward<bf16>(who, *a, s);
}

int nesle_qk_norm_rotate_grad(const nesle_qk_args* a, void* stream) {
    const char* who = "nesle_qk_norm_rotate_grad";
    const int rc = check(who, a);
    if (rc != NESLE_OK) return rc;
    const bool weights = a->q_weight != nullptr || a->k_weight != nullptr;
    if ((a->q_weight == nullptr) != (a->dq_weight == nullptr) || (a->k_weight == nullptr) != (a->dk_weight == nullptr))
        return refuse(who, "a weight and its gradient go together");
    if (!empty(a)) {
        if ((a->q_heads != 0 && (a->q.data == nullptr || a->dq_out.data == nullptr || a->dq == nullptr)) ||
            (a->k_heads != 0 && (a->k.data == nullptr || a->dk_out.data == nullptr || a->dk == nullptr)) ||
            (weights && a->scratch == nullptr))
            return refuse(who, "null device pointer");
    }
    const auto s = static_cast<hipStream_t>(stream);
    if (empty(a)) {       // no rows: the weights' gradient is zero
        if (!weights) return NESLE_OK;
        hipLaunchKernelGGL(qk_weight_sum, dim3(2 * a->dim), dim3(kThreads), 0, s, nullptr, 0u, a->dim, a->dq_weight,
                           a->dk_weight);
        return launched(who);
    }
    return a->dtype == NESLE_MEM_F32 ? gradient<float>(who, *a, s) : gradient<bf16>(who, *a, s);
}

}  // extern "C"
