// Norms of queries and keys for each head with the position rotation, and the
// gradient (include/nesle_memory.h has the formulas).
//
// One pass: a group of lanes holds one head in registers, so the sum of squares
// is a few lane exchanges and every element is read and written once.  A lane's
// elements are PAIRS from the first half of the rotated part and the PAIRS they
// are paired with in the second half, so that a pair never crosses lanes in
// either layout; lanes past the rotated part hold 2 PAIRS consecutive ones.
// PAIRS is what a 16-byte load holds, or four where the sizes or addresses do
// not allow eight bfloat16.
//
// Bound by memory: about 10 operations an element.  Measured against a large
// copy's 4.9 TB/s, bfloat16: 1.08 GB of 128 steps of 4,096 rows and 8 heads of 64
// in 222 us (4.9 TB/s); 128 steps of 512 rows, forward 134 MB in 29 us (4.6 TB/s),
// gradient 202 MB in 41 us (4.9 TB/s) and the weights' sum 4 us.  A head has a power of
// two lanes: of 40 float32 elements 5 of 8 work (23,177 rows of 8 such heads: forward
// 59 MB in 16 us, 3.7 TB/s).  Loads of 8 bytes a
// lane in place of 16 took 309 us for the first; heads of one row side by side in a
// thread, which share a row of the table, 338 us.  Below about 100 rows a call is a
// launch: 3.6 us.
#include <algorithm>
#include <initializer_list>

#include "mem_common.h"

namespace nesle::mem {
namespace {

constexpr unsigned kThreads = 256;
// Heads a thread works on at once, rows apart: their loads are in flight together.
// One where the rows do not fill the card, fewer than 1,024 workgroups: latency
// counts there.  In float32, 4 + 4 heads of 64, together / one: 1,024 rows 6.1 / 3.4
// us, 8,192 rows 9.0 / 7.5, 16,384 rows (the first together) 13.9 / 13.9, 65,536 rows
// 45.4 / 46.5.
constexpr unsigned kTogether = 4, kGradTogether = 2;
// Workgroups of the gradient, four a compute unit, which their registers leave
// room for (twice as many: 47 us for 43): each adds up its rows' share of a
// weight's gradient, and one more launch adds the workgroups' in order.
constexpr unsigned kGradBlocks = 1024;

// x / d for x < 2^16 (d as it is) or x < 2 d (d of 2^15 or more).
struct Divide {
    std::uint32_t d, magic;
    Divide(std::uint32_t by = 1) : d(by), magic(by > 1 ? static_cast<std::uint32_t>((0x100000000ull + by - 1) / by) : 0) {}
    __device__ std::uint32_t operator()(std::uint32_t x) const {
        if (d >= (1u << 15)) return x >= d ? 1u : 0u;
        return d == 1 ? x : __umulhi(x, magic);
    }
};

template <typename T>
struct QkArgs {
    Heads<T> q, k, dq_out, dk_out;
    const float *wq, *wk;
    const std::int32_t* positions;
    const float* table;
    T *q_out, *k_out;        // forward: outputs; gradient: dq, dk
    float* partials;         // [blocks][dim]
    Divide batch, per_row, per_q, per_k;   // rows of a step, heads of a row, of either kind
    std::uint32_t hq, hk, dim, rotated, table_rows, lanes;   // lanes of one head: a power of two
    std::uint32_t q_blocks;  // gradient: the workgroups that take queries
    std::uint64_t groups;    // heads of all rows
    float inv_count, eps;
    bool interleaved;
};

// The two element offsets of lane j's groups.
template <int PAIRS, typename T>
__device__ void places(const QkArgs<T>& a, unsigned j, unsigned& first, unsigned& second) {
    if (2 * PAIRS * j >= a.rotated || a.interleaved) {
        first = 2 * PAIRS * j;
        second = first + PAIRS;
    } else {
        first = PAIRS * j;
        second = a.rotated / 2 + first;
    }
}

// A lane's elements of a head, or the angles of its pairs.
template <int PAIRS>
struct Part {
    static constexpr int N = PAIRS / 4;
    f4 a[N], b[N];
    __device__ void fill(float v) {
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] = b[i] = f4{v, v, v, v};
    }
    template <typename T>
    __device__ void load(const T* p, unsigned first, unsigned second, bool vec) {
        if constexpr (PAIRS == 8) {
            load8(p + first, a[0], a[1]);
            load8(p + second, b[0], b[1]);
        } else {
            a[0] = load4(p + first, vec);
            b[0] = load4(p + second, vec);
        }
    }
    __device__ void load_floats(const float* p, unsigned first, unsigned second) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            a[i] = load4(p + first + 4 * i, true);
            b[i] = load4(p + second + 4 * i, true);
        }
    }
    template <typename T>
    __device__ void store(T* p, unsigned first, unsigned second) const {
        if constexpr (PAIRS == 8) {
            store8(p + first, a[0], a[1]);
            store8(p + second, b[0], b[1]);
        } else {
            store4(p + first, a[0]);
            store4(p + second, b[0]);
        }
    }
    __device__ float dot(const Part& o) const {
        f4 v = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < N; ++i) v += a[i] * o.a[i] + b[i] * o.b[i];
        return v.x + v.y + v.z + v.w;
    }
    __device__ void scale(float v) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            a[i] *= v;
            b[i] *= v;
        }
    }
    __device__ void scale(const Part& o) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            a[i] *= o.a[i];
            b[i] *= o.b[i];
        }
    }
    // Turn by the angles whose cosines are in t.a and sines in t.b, or back.
    __device__ void turn(const Part& t, bool back, bool interleaved) {
        if (interleaved) {
            const auto pair = [&](float& x, float& y, int k) {
                const float c = t.a[k / 4][k % 4], s = back ? -t.b[k / 4][k % 4] : t.b[k / 4][k % 4];
                const float u = x * c - y * s;
                y = x * s + y * c;
                x = u;
            };
#pragma unroll
            for (int k = 0; k < PAIRS / 2; ++k) {
                float x = a[k / 2][2 * (k % 2)], y = a[k / 2][2 * (k % 2) + 1];
                pair(x, y, k);
                a[k / 2][2 * (k % 2)] = x;
                a[k / 2][2 * (k % 2) + 1] = y;
                x = b[k / 2][2 * (k % 2)], y = b[k / 2][2 * (k % 2) + 1];
                pair(x, y, PAIRS / 2 + k);
                b[k / 2][2 * (k % 2)] = x;
                b[k / 2][2 * (k % 2) + 1] = y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const f4 s = back ? -t.b[i] : t.b[i], u = a[i] * t.a[i] - b[i] * s;
                b[i] = a[i] * s + b[i] * t.a[i];
                a[i] = u;
            }
        }
    }
};

// Where a run of heads starts: divisions of 64-bit numbers once a workgroup,
// small ones for each of its heads.
struct Start {
    std::uint64_t row, step;
    std::uint32_t head, env;
    __device__ Start(const Divide& batch, const Divide& per_row, std::uint64_t group)
        : row(group / per_row.d), step(row / batch.d), head(static_cast<std::uint32_t>(group % per_row.d)),
          env(static_cast<std::uint32_t>(row % batch.d)) {}
};

// One head of those of a row.
struct Spot {
    std::uint32_t h, env;
    std::uint64_t row, step;
    __device__ Spot(const Divide& batch, const Divide& per_row, const Start& at, std::uint32_t plus) {
        const std::uint32_t x = at.head + plus, down = per_row(x), y = at.env + down, over = batch(y);
        h = x - down * per_row.d;
        row = at.row + down;
        step = at.step + over;
        env = y - over * batch.d;
    }
    template <typename T>
    __device__ const T* in(const Heads<T>& x) const { return x.row(step, env, h); }
};
// One of all: its kind too.
template <typename T>
struct AnySpot : Spot {
    bool is_q;
    __device__ AnySpot(const QkArgs<T>& a, const Start& at, std::uint32_t plus) : Spot(a.batch, a.per_row, at, plus) {
        is_q = h < a.hq;
        h = is_q ? h : h - a.hq;
    }
    __device__ T* out(const QkArgs<T>& a) const {
        return is_q ? a.q_out + (row * a.hq + h) * a.dim : a.k_out + (row * a.hk + h) * a.dim;
    }
};

// Lane j's part of a head, turned (back) by its row of the table; where the table
// has no such row all of the head is NaN, its elements past the rotated ones too.
template <int PAIRS, typename T>
__device__ void rotate(const QkArgs<T>& a, std::int32_t p, unsigned j, bool rotates, bool back, Part<PAIRS>& x) {
    if (a.rotated == 0) return;
    if (static_cast<std::uint32_t>(p) >= a.table_rows || p < 0) {
        x.fill(NAN);
    } else if (rotates) {
        Part<PAIRS> t;
        t.load_floats(a.table + static_cast<std::size_t>(p) * a.rotated, PAIRS * j, PAIRS * j + a.rotated / 2);
        x.turn(t, back, a.interleaved);
    }
}

__device__ inline float across(float v, unsigned lanes) {
    for (unsigned d = 1; d < lanes; d *= 2) v += __shfl_xor(v, d);
    return v;
}

template <typename T, int PAIRS, unsigned TOGETHER>
__global__ void __launch_bounds__(kThreads) qk_forward(QkArgs<T> a) {
    const unsigned j = threadIdx.x % a.lanes, per = kThreads / a.lanes;
    const std::uint64_t base = static_cast<std::uint64_t>(blockIdx.x) * per * TOGETHER;
    const Start start(a.batch, a.per_row, base);
    const bool has = 2 * PAIRS * j < a.dim, rotates = 2 * PAIRS * j < a.rotated;
    unsigned first, second;
    places<PAIRS>(a, j, first, second);
    Part<PAIRS> x[TOGETHER];
    std::int32_t position[TOGETHER];
#pragma unroll
    for (unsigned i = 0; i < TOGETHER; ++i) {
        const std::uint32_t plus = i * per + threadIdx.x / a.lanes;
        x[i].fill(0.0f);
        position[i] = 0;
        if (base + plus < a.groups && has) {
            const AnySpot<T> at(a, start, plus);
            x[i].load(at.is_q ? at.in(a.q) : at.in(a.k), first, second, at.is_q ? a.q.vec : a.k.vec);
            if (a.rotated != 0) position[i] = a.positions[at.row];
        }
    }
#pragma unroll
    for (unsigned i = 0; i < TOGETHER; ++i) {
        const std::uint32_t plus = i * per + threadIdx.x / a.lanes;
        const float inv = 1.0f / sqrtf(across(x[i].dot(x[i]), a.lanes) * a.inv_count + a.eps);
        if (base + plus >= a.groups || !has) continue;
        const AnySpot<T> at(a, start, plus);
        x[i].scale(inv);
        const float* w = at.is_q ? a.wq : a.wk;
        if (w != nullptr) {
            Part<PAIRS> weight;
            weight.load_floats(w, first, second);
            x[i].scale(weight);
        }
        rotate(a, position[i], j, rotates, false, x[i]);
        x[i].store(at.out(a), first, second);
    }
}

// dy = the output's gradient turned back; dx = inv w dy - x inv^3 <x, w dy> / count;
// dw = sum over rows of x inv dy.  A workgroup takes heads of one kind, so that a
// lane adds up one weight's gradient and reads neighbouring heads: both kinds' took
// 130 registers for 116, three waves a SIMD for four, and 55 us for 40 in the case
// above.
template <typename T, int PAIRS>
__global__ void __launch_bounds__(kThreads) qk_gradient(QkArgs<T> a) {
    constexpr int N = PAIRS / 4;
    constexpr unsigned kTogether = kGradTogether / N;
    __shared__ f4 sums[kThreads / 64][2 * N][32 / N];       // [wave][four of them][lane of the head]
    const bool is_q = blockIdx.x < a.q_blocks;
    const std::uint32_t block = is_q ? blockIdx.x : blockIdx.x - a.q_blocks;
    const std::uint32_t blocks = is_q ? a.q_blocks : gridDim.x - a.q_blocks;
    const Heads<T> in = is_q ? a.q : a.k, dy = is_q ? a.dq_out : a.dk_out;
    const Divide per_row = is_q ? a.per_q : a.per_k;
    const std::uint64_t groups = a.groups / a.per_row.d * per_row.d;
    const float* w = is_q ? a.wq : a.wk;
    T* out = is_q ? a.q_out : a.k_out;
    const unsigned j = threadIdx.x % a.lanes, per = kThreads / a.lanes;
    unsigned first, second;
    places<PAIRS>(a, j, first, second);
    const bool has = 2 * PAIRS * j < a.dim, rotates = 2 * PAIRS * j < a.rotated;
    Part<PAIRS> dw;
    dw.fill(0.0f);
    const std::uint64_t at_once = static_cast<std::uint64_t>(blocks) * per * kTogether;
    // Every lane of a workgroup takes every turn, as the lane exchanges need.
    for (std::uint64_t base = static_cast<std::uint64_t>(block) * per * kTogether; base < groups; base += at_once) {
        const Start start(a.batch, per_row, base);
        Part<PAIRS> x[kTogether], d[kTogether];
        std::int32_t position[kTogether];
#pragma unroll
        for (unsigned i = 0; i < kTogether; ++i) {
            const std::uint32_t plus = i * per + threadIdx.x / a.lanes;
            x[i].fill(0.0f);
            d[i].fill(0.0f);
            position[i] = 0;
            if (base + plus < groups && has) {
                const Spot at(a.batch, per_row, start, plus);
                x[i].load(at.in(in), first, second, in.vec);
                d[i].load(at.in(dy), first, second, dy.vec);
                if (a.rotated != 0) position[i] = a.positions[at.row];
            }
        }
#pragma unroll
        for (unsigned i = 0; i < kTogether; ++i) {
            const std::uint32_t plus = i * per + threadIdx.x / a.lanes;
            const bool mine = base + plus < groups && has;
            const float inv = 1.0f / sqrtf(across(x[i].dot(x[i]), a.lanes) * a.inv_count + a.eps);
            if (mine) rotate(a, position[i], j, rotates, true, d[i]);
            if (w != nullptr && mine) {
                Part<PAIRS> weight;
                weight.load_floats(w, first, second);
#pragma unroll
                for (int u = 0; u < N; ++u) {
                    dw.a[u] += x[i].a[u] * inv * d[i].a[u];
                    dw.b[u] += x[i].b[u] * inv * d[i].b[u];
                }
                d[i].scale(weight);
            }
            const float along = across(x[i].dot(d[i]), a.lanes) * inv * inv * inv * a.inv_count;
            if (mine) {
#pragma unroll
                for (int u = 0; u < N; ++u) {
                    d[i].a[u] = d[i].a[u] * inv - x[i].a[u] * along;
                    d[i].b[u] = d[i].b[u] * inv - x[i].b[u] * along;
                }
                d[i].store(out + (base + plus) * a.dim, first, second);
            }
        }
    }
    if (a.partials == nullptr) return;
    // Lanes that hold the same elements, first within the wave, then over the
    // waves, in a fixed order.
    const unsigned lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
    for (int u = 0; u < 2 * N; ++u) {
        f4 v = u < N ? dw.a[u] : dw.b[u - N];
        for (unsigned d = a.lanes; d < 64; d *= 2)
            v += f4{__shfl_xor(v.x, d), __shfl_xor(v.y, d), __shfl_xor(v.z, d), __shfl_xor(v.w, d)};
        if (lane < a.lanes) sums[wave][u][lane] = v;
    }
    __syncthreads();
    if (threadIdx.x < a.lanes && has)
        for (int u = 0; u < 2 * N; ++u) {
            f4 v = sums[0][u][j];
            for (unsigned o = 1; o < kThreads / 64; ++o) v += sums[o][u][j];
            float* p = a.partials + static_cast<std::size_t>(blockIdx.x) * a.dim;
            store4(p + (u < N ? first + 4 * u : second + 4 * (u - N)), v);
        }
}

// One element of one weight's gradient a workgroup: the partials of the kind's
// workgroups, added in a fixed order.
__global__ void __launch_bounds__(kThreads) qk_weight_sum(const float* partials, std::uint32_t q_blocks, std::uint32_t blocks,
                                                          std::uint32_t dim, float* dwq, float* dwk) {
    __shared__ float sh[kThreads];
    const bool is_q = blockIdx.x < dim;
    const std::uint32_t e = is_q ? blockIdx.x : blockIdx.x - dim, end = is_q ? q_blocks : blocks;
    float v = 0.0f;
    for (std::uint32_t b = (is_q ? 0 : q_blocks) + threadIdx.x; b < end; b += kThreads) v += partials[static_cast<std::size_t>(b) * dim + e];
    sh[threadIdx.x] = v;
    __syncthreads();
    for (unsigned s = kThreads / 2; s > 0; s /= 2) {
        if (threadIdx.x < s) sh[threadIdx.x] += sh[threadIdx.x + s];
        __syncthreads();
    }
    float* out = is_q ? dwq : dwk;
    if (threadIdx.x == 0 && out != nullptr) out[e] = sh[0];
}

std::uint32_t lanes_of(std::uint32_t dim, unsigned pairs) {
    std::uint32_t n = 1;
    while (2 * pairs * n < dim) n *= 2;
    return n;
}

std::uint64_t blocks_for(const nesle_qk_args& a, unsigned pairs, unsigned together) {
    const std::uint64_t per = kThreads / lanes_of(a.dim, pairs) * together;
    return (static_cast<std::uint64_t>(a.steps) * a.batch * (a.q_heads + a.k_heads) + per - 1) / per;
}

// Workgroups of the gradient for heads of one kind.
std::uint32_t grad_blocks(const nesle_qk_args& a, std::uint32_t kind_heads) {
    if (kind_heads == 0) return 0;
    const std::uint64_t per = kThreads / lanes_of(a.dim, 4) * kGradTogether;      // of eight pairs: as many
    const std::uint64_t all = (static_cast<std::uint64_t>(a.steps) * a.batch * kind_heads + per - 1) / per;
    const std::uint64_t most = std::max(1u, kGradBlocks * kind_heads / (a.q_heads + a.k_heads));
    return static_cast<std::uint32_t>(std::min(all, most));
}

bool aligned(std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if (reinterpret_cast<std::uintptr_t>(p) % 16 != 0) return false;
    return true;
}

bool empty(const nesle_qk_args* a) { return a->steps == 0 || a->batch == 0; }

int check(const char* who, const nesle_qk_args* a) {
    if (a == nullptr) return refuse(who, "null arguments");
    if (a->dtype != NESLE_MEM_F32 && a->dtype != NESLE_MEM_BF16) return refuse(who, "dtype must be NESLE_MEM_F32 or NESLE_MEM_BF16");
    if (a->dim == 0 || a->dim % 8 != 0 || a->dim > NESLE_QK_MAX_DIM)
        return refuse(who, "dim must be a multiple of 8 up to " + std::to_string(NESLE_QK_MAX_DIM));
    if (a->rotated % 8 != 0 || a->rotated > a->dim) return refuse(who, "rotated must be a multiple of 8 up to dim");
    if (a->q_heads + static_cast<std::uint64_t>(a->k_heads) == 0 || a->q_heads > 4096u || a->k_heads > 4096u)
        return refuse(who, "heads must be in 1..4096");
    // One launch takes fewer than 2^32 threads of 32 elements; the first
    // test keeps the second one's product below 2^64.
    if (static_cast<std::uint64_t>(a->steps) * a->batch > (1ull << 32) || blocks_for(*a, 4, kTogether) * kThreads > 0xffffffffull)
        return refuse(who, "more than 2^37 elements");
    if (!(a->eps >= 0.0f)) return refuse(who, "eps must not be negative");
    if (a->rotated != 0 && !empty(a) && (a->positions == nullptr || a->table == nullptr || a->table_rows == 0))
        return refuse(who, "the rotation needs positions and a table");
    if (!aligned({a->q_weight, a->k_weight, a->table, a->q_out, a->k_out, a->dq, a->dk, a->scratch}))
        return refuse(who, "weights, table, outputs and workspace must lie on 16-byte boundaries");
    return NESLE_OK;
}

template <typename T>
QkArgs<T> pack(const nesle_qk_args& a, unsigned pairs) {
    QkArgs<T> k{};
    k.q = heads<T>(a.q);
    k.k = heads<T>(a.k);
    k.wq = a.q_weight;
    k.wk = a.k_weight;
    k.positions = a.positions;
    k.table = a.table;
    k.batch = Divide(a.batch);
    k.per_row = Divide(a.q_heads + a.k_heads);
    k.per_q = Divide(a.q_heads);
    k.per_k = Divide(a.k_heads);
    k.hq = a.q_heads;
    k.hk = a.k_heads;
    k.dim = a.dim;
    k.rotated = a.rotated;
    k.table_rows = a.table_rows;
    k.lanes = lanes_of(a.dim, pairs);
    k.groups = static_cast<std::uint64_t>(a.steps) * a.batch * (a.q_heads + a.k_heads);
    k.inv_count = a.unit ? 1.0f : 1.0f / static_cast<float>(a.dim);
    k.eps = a.eps;
    k.interleaved = a.interleaved != 0;
    return k;
}

// Eight bfloat16 a load where heads, halves and addresses allow it.
bool by_eight(const nesle_qk_args& a, bool gradient) {
    if (a.dtype != NESLE_MEM_BF16 || a.dim % 16 != 0 || a.rotated % 16 != 0) return false;
    const auto wide = [](const nesle_heads& x, std::uint32_t n) { return n == 0 || heads<bf16>(x).wide; };
    return wide(a.q, a.q_heads) && wide(a.k, a.k_heads) &&
           (!gradient || (wide(a.dq_out, a.q_heads) && wide(a.dk_out, a.k_heads)));
}

template <typename T, int PAIRS>
void launch_forward(const nesle_qk_args& a, hipStream_t s) {
    QkArgs<T> k = pack<T>(a, PAIRS);
    k.q_out = static_cast<T*>(a.q_out);
    k.k_out = static_cast<T*>(a.k_out);
    constexpr unsigned together = kTogether * 4 / PAIRS;
    const auto blocks = static_cast<std::uint32_t>(blocks_for(a, PAIRS, together));
    if (blocks < 1024)
        hipLaunchKernelGGL((qk_forward<T, PAIRS, 1>), dim3(static_cast<std::uint32_t>(blocks_for(a, PAIRS, 1))), dim3(kThreads), 0, s, k);
    else
        hipLaunchKernelGGL((qk_forward<T, PAIRS, together>), dim3(blocks), dim3(kThreads), 0, s, k);
}

int forward(const char* who, const nesle_qk_args& a, hipStream_t s) {
    if (a.dtype == NESLE_MEM_F32) launch_forward<float, 4>(a, s);
    else if (by_eight(a, false)) launch_forward<bf16, 8>(a, s);
    else launch_forward<bf16, 4>(a, s);
    return launched(who);
}

template <typename T, int PAIRS>
void launch_gradient(const nesle_qk_args& a, hipStream_t s) {
    QkArgs<T> k = pack<T>(a, PAIRS);
    k.dq_out = heads<T>(a.dq_out);
    k.dk_out = heads<T>(a.dk_out);
    k.q_out = static_cast<T*>(a.dq);
    k.k_out = static_cast<T*>(a.dk);
    const bool weights = a.q_weight != nullptr || a.k_weight != nullptr;
    k.partials = weights ? a.scratch : nullptr;
    k.q_blocks = grad_blocks(a, a.q_heads);
    const std::uint32_t blocks = k.q_blocks + grad_blocks(a, a.k_heads);
    hipLaunchKernelGGL((qk_gradient<T, PAIRS>), dim3(blocks), dim3(kThreads), 0, s, k);
    if (weights)
        hipLaunchKernelGGL(qk_weight_sum, dim3(2 * a.dim), dim3(kThreads), 0, s, a.scratch, k.q_blocks, blocks, a.dim,
                           a.dq_weight, a.dk_weight);
}

int gradient(const char* who, const nesle_qk_args& a, hipStream_t s) {
    if (a.dtype == NESLE_MEM_F32) launch_gradient<float, 4>(a, s);
    else if (by_eight(a, true)) launch_gradient<bf16, 8>(a, s);
    else launch_gradient<bf16, 4>(a, s);
    return launched(who);
}

}  // namespace
}  // namespace nesle::mem

using namespace nesle::mem;

extern "C" {

std::uint64_t nesle_qk_scratch_floats(const nesle_qk_args* a) {
    if (a == nullptr || (a->q_weight == nullptr && a->k_weight == nullptr)) return 0;
    if (a->dim == 0 || a->dim > NESLE_QK_MAX_DIM) return 0;        // no call takes it, and no workgroup a head of it
    return (static_cast<std::uint64_t>(grad_blocks(*a, a->q_heads)) + grad_blocks(*a, a->k_heads)) * a->dim;
}

int nesle_qk_norm_rotate(const nesle_qk_args* a, void* stream) {
    const char* who = "nesle_qk_norm_rotate";
    const int rc = check(who, a);
    if (rc != NESLE_OK || empty(a)) return rc;
    if ((a->q_heads != 0 && (a->q.data == nullptr || a->q_out == nullptr)) ||
        (a->k_heads != 0 && (a->k.data == nullptr || a->k_out == nullptr)))
        return refuse(who, "null device pointer");
    const auto s = static_cast<hipStream_t>(stream);
    return forward(who, *a, s);
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
        hipLaunchKernelGGL(qk_weight_sum, dim3(2 * a->dim), dim3(kThreads), 0, s, nullptr, 0u, 0u, a->dim,
                           a->dq_weight, a->dk_weight);
        return launched(who);
    }
    return gradient(who, *a, s);
}

}  // extern "C"
