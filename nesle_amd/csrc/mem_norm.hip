// Layer norm of rows and its gradient (include/nesle_memory.h has the formula).
//
// A row is held in the registers of a group of lanes, so it is read once, its mean
// and then the mean of squares about it are sums over the group (two steps: a sum of
// squares less the squared mean would cancel where a row's level is large; the second
// step also sums the differences, which corrects the mean's rounding, and costs nothing to
// 3 % of a call, 7 % with rows of 64), and the result is written once.  With
// xh = (x - mean) rstd and d = dy weight, the gradient is
//   dx = rstd (d - mean(d) - xh mean(d xh)),  dweight = sum dy xh,  dbias = sum dy
// over rows; mean and rstd are found again from x, which is read anyway.  A group
// takes rows a grid apart and keeps the weights, and the sums of their gradients, of
// its columns in registers; workgroups' sums are added by a second launch in a fixed
// order.
//
// Bound by memory: 65,536 rows of 256 in bfloat16 take 14.3 us forward (67 MB, 4.7 TB/s)
// and 22.6 + 4 for the gradient (100 MB, 4.5 TB/s); eight times the rows 98 (5.4) and 142 +
// 4 (5.7); 23,177 rows of 201 in float32, an element at a time, 9.4 and 13 + 4; 262,144 rows
// of 64 in bfloat16, which leave half of 16 lanes empty, 17.7 (3.8) and 29 + 4 (3.5).  A
// weight or a bias read an element at a time took 36 us forward where 14 are; the second
// launch with one lane a column 21.
#include <algorithm>
#include <initializer_list>

#include "mem_delta_math.h"

namespace nesle::mem {
namespace {

template <typename T>
struct NormArgs {
    Heads<T> x, dy;
    const float *weight, *bias;
    T *y, *dx;
    float* partials;               // [blocks][2][dim]
    std::uint32_t rows, batch, heads, dim;
    bool plain, plain_dy;          // rows lie one stride_h after the other
    float inv_dim, eps;
};

template <typename T>
__device__ const T* row_of(const Heads<T>& x, bool plain, std::uint32_t row, std::uint32_t batch, std::uint32_t heads) {
    if (plain) return x.data + static_cast<std::int64_t>(row) * x.h;
    const std::uint32_t all = row / heads;
    return x.row(all / batch, all % batch, row % heads);
}

// V elements of a row that lie together, as float32: eight bfloat16 or four float32
// of aligned rows, or one.
template <typename T, int V>
struct Vec {
    float v[V];
    __device__ void load(const T* p) {
        if constexpr (V == 8) {
            f4 a, b;
            load8(p, a, b);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = a[i];
                v[4 + i] = b[i];
            }
        } else if constexpr (V == 4) {
            const f4 a = load4(p, true);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = a[i];
        } else {
            v[0] = static_cast<float>(*p);
        }
    }
    __device__ void store(T* p) const {
        if constexpr (V == 8) store8(p, f4{v[0], v[1], v[2], v[3]}, f4{v[4], v[5], v[6], v[7]});
        else if constexpr (V == 4) store4(p, f4{v[0], v[1], v[2], v[3]});
        else *p = static_cast<T>(v[0]);
    }
};

// Sums over a group of L lanes, in all of them.  A group of more than a wave is a
// workgroup: `slot` names one of three places, so that one barrier a sum is enough.
template <int L, int COUNT>
struct GroupSum {
    float (*place)[COUNT][L > 64 ? L / 64 : 1];
    template <int N>
    __device__ void operator()(float (&v)[N], int slot) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = sum16(v[i]);
            if constexpr (L > 16) v[i] = over_groups(v[i]);
        }
        if constexpr (L > 64) {
            if (threadIdx.x % 64 == 0)
#pragma unroll
                for (int i = 0; i < N; ++i) place[slot][i][threadIdx.x / 64] = v[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float sum = 0.0f;
                for (int w = 0; w < L / 64; ++w) sum += place[slot][i][w];
                v[i] = sum;
            }
        }
    }
};

// N vectors of a lane, L lanes' apart.
template <typename T, int V, int N, int L>
struct Row {
    Vec<T, V> e[N];
    static __device__ std::uint32_t col(int c, unsigned lane) { return (c * L + lane) * V; }
    __device__ void load(const T* p, std::uint32_t dim, unsigned lane) {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            if (col(c, lane) < dim) {
                e[c].load(p + col(c, lane));
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) e[c].v[j] = 0.0f;
            }
        }
    }
    // Elements less the mean as it rounds, zero past the row's end; x scale + shift is what
    // the norm makes of one.  The mean is off by up to a few 2^-24 of the row's level.  The
    // differences' own mean is that error, to their precision, so the shift takes it out of
    // them, and the variance is the mean of their squares less its square.
    struct Normal {
        float scale, shift;
        __device__ float operator()(float x) const { return fmaf(x, scale, shift); }
    };
    template <typename Sum>
    __device__ Normal center(const Sum& group, std::uint32_t dim, float inv_dim, float eps, unsigned lane) {
        float level[1] = {0.0f}, s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) level[0] += e[c].v[j];
        group(level, 0);
        const float mean = level[0] * inv_dim;
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                e[c].v[j] = col(c, lane) < dim ? e[c].v[j] - mean : 0.0f;
                s[0] += e[c].v[j];
                s[1] += e[c].v[j] * e[c].v[j];
            }
        group(s, 1);
        const float more = s[0] * inv_dim, variance = s[1] * inv_dim - more * more;
        const float rstd = 1.0f / sqrtf((variance < 0.0f ? 0.0f : variance) + eps);        // NaN stays NaN
        return {rstd, -more * rstd};
    }
};

// V floats of a weight that lie together; `or_else` where there is none.
template <int V>
__device__ void load_weight(const float* p, std::uint32_t col, std::uint32_t dim, float or_else, float (&v)[V]) {
    const bool has = p != nullptr && col < dim;
    if constexpr (V == 1) {
        v[0] = has ? p[col] : or_else;
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const f4 x = has ? *reinterpret_cast<const f4*>(p + col + i) : f4{or_else, or_else, or_else, or_else};
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i + j] = x[j];
        }
    }
}

template <int L>
constexpr int kBlock = L > 256 ? L : 256;

template <typename T, int V, int N, int L>
__global__ void __launch_bounds__(kBlock<L>) layer_norm_kernel(NormArgs<T> a) {
    __shared__ float place[3][2][L > 64 ? L / 64 : 1];
    const GroupSum<L, 2> group{place};
    const unsigned lane = threadIdx.x % L;
    constexpr unsigned kGroups = kBlock<L> / L;
    const std::uint32_t stride = gridDim.x * kGroups;
    Vec<float, V> w[N], b[N];
#pragma unroll
    for (int c = 0; c < N; ++c) {
        load_weight<V>(a.weight, Row<T, V, N, L>::col(c, lane), a.dim, 1.0f, w[c].v);
        load_weight<V>(a.bias, Row<T, V, N, L>::col(c, lane), a.dim, 0.0f, b[c].v);
    }
    for (std::uint64_t row = blockIdx.x * kGroups + threadIdx.x / L; row < a.rows; row += stride) {
        Row<T, V, N, L> x;
        x.load(row_of(a.x, a.plain, static_cast<std::uint32_t>(row), a.batch, a.heads), a.dim, lane);
        const auto normal = x.center(group, a.dim, a.inv_dim, a.eps, lane);
        T* y = a.y + row * a.dim;
#pragma unroll
        for (int c = 0; c < N; ++c) {
            Vec<T, V> out;
#pragma unroll
            for (int j = 0; j < V; ++j) out.v[j] = normal(x.e[c].v[j]) * w[c].v[j] + b[c].v[j];
            if (x.col(c, lane) < a.dim) out.store(y + x.col(c, lane));
        }
    }
}

template <typename T, int V, int N, int L>
__global__ void __launch_bounds__(kBlock<L>) layer_norm_grad_kernel(NormArgs<T> a) {
    constexpr int kWaves = kBlock<L> / 64;
    constexpr unsigned kGroups = kBlock<L> / L;
    __shared__ float place[3][2][L > 64 ? L / 64 : 1];
    __shared__ float columns[L > 64 ? 1 : kWaves * N * V * L];
    const GroupSum<L, 2> group{place};
    const unsigned lane = threadIdx.x % L;
    const std::uint32_t stride = gridDim.x * kGroups;
    float w[N][V], dw[N][V], db[N][V];
#pragma unroll
    for (int c = 0; c < N; ++c) {
        load_weight<V>(a.weight, Row<T, V, N, L>::col(c, lane), a.dim, 1.0f, w[c]);
#pragma unroll
        for (int j = 0; j < V; ++j) dw[c][j] = db[c][j] = 0.0f;
    }
    for (std::uint64_t row = blockIdx.x * kGroups + threadIdx.x / L; row < a.rows; row += stride) {
        Row<T, V, N, L> x, dy;
        const auto r = static_cast<std::uint32_t>(row);
        x.load(row_of(a.x, a.plain, r, a.batch, a.heads), a.dim, lane);
        dy.load(row_of(a.dy, a.plain_dy, r, a.batch, a.heads), a.dim, lane);
        const auto normal = x.center(group, a.dim, a.inv_dim, a.eps, lane);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = normal(x.e[c].v[j]), d = dy.e[c].v[j];
                dw[c][j] += d * xh;
                db[c][j] += d;
                x.e[c].v[j] = xh;
                dy.e[c].v[j] = d * w[c][j];
                s[0] += dy.e[c].v[j];
                s[1] += dy.e[c].v[j] * xh;
            }
        group(s, 2);
        const float mean = s[0] * a.inv_dim, along = s[1] * a.inv_dim;
        T* dx = a.dx + row * a.dim;
#pragma unroll
        for (int c = 0; c < N; ++c) {
            Vec<T, V> out;
#pragma unroll
            for (int j = 0; j < V; ++j) out.v[j] = normal.scale * (dy.e[c].v[j] - mean - x.e[c].v[j] * along);
            if (x.col(c, lane) < a.dim) out.store(dx + x.col(c, lane));
        }
    }
    if (a.partials == nullptr) return;
    // The workgroup's sums, dweight and then dbias: over the groups of a wave by
    // lane exchanges, over waves through LDS.
    for (int which = 0; which < 2; ++which) {
        float* to = a.partials + (2ull * blockIdx.x + which) * a.dim;
        if constexpr (L <= 64) {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < N; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float v = which == 0 ? dw[c][j] : db[c][j];
                    if constexpr (L == 16) v = over_groups(v);
                    if (L == 64 || threadIdx.x % 64 < 16) columns[threadIdx.x / 64 * N * V * L + Row<T, V, N, L>::col(c, lane) + j] = v;
                }
            __syncthreads();
            for (std::uint32_t i = threadIdx.x; i < a.dim; i += kBlock<L>) {
                float sum = 0.0f;
                for (int v = 0; v < kWaves; ++v) sum += columns[v * N * V * L + i];
                to[i] = sum;
            }
        } else {
#pragma unroll
            for (int c = 0; c < N; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (Row<T, V, N, L>::col(c, lane) < a.dim) to[Row<T, V, N, L>::col(c, lane) + j] = which == 0 ? dw[c][j] : db[c][j];
        }
    }
}

// The workgroups' sums added up: 16 columns a workgroup, 64 lanes a column, each of which
// has at most kMostPartials / 64 sums in flight at once.
constexpr std::uint32_t kMostPartials = 1024;
__global__ void __launch_bounds__(1024) norm_weight_sum(const float* partials, float* dweight, float* dbias, std::uint32_t dim,
                                                        std::uint32_t blocks) {
    __shared__ float part[64][17];
    const std::uint32_t i = blockIdx.x * 16 + threadIdx.x % 16, all = 2 * dim, first = threadIdx.x / 16;
    float v[kMostPartials / 64], sum = 0.0f;
#pragma unroll
    for (std::uint32_t k = 0; k < kMostPartials / 64; ++k)
        v[k] = i < all && first + 64 * k < blocks ? partials[static_cast<std::size_t>(first + 64 * k) * all + i] : 0.0f;
#pragma unroll
    for (std::uint32_t k = 0; k < kMostPartials / 64; ++k) sum += v[k];
    part[first][threadIdx.x % 16] = sum;
    __syncthreads();
    // A wave for each column: the sum over its 64 lanes.
    const unsigned column = threadIdx.x / 64;
    sum = over_groups(sum16(part[threadIdx.x % 64][column]));
    const std::uint32_t at = blockIdx.x * 16 + column;
    if (threadIdx.x % 64 != 0 || at >= all) return;
    float* to = at < dim ? dweight : dbias;
    if (to != nullptr) to[at < dim ? at : at - dim] = sum;
}

// How a row is laid over lanes.
struct Shape {
    int lanes, vectors;
    std::uint32_t groups;      // rows of a workgroup at once
};

// Fewest lanes whose registers hold the row: sums over 16 lanes need no exchange
// between rows of lanes, over a wave no barrier.  More than 32 elements a lane, five
// arrays of them in the gradient, would not stay in registers.
constexpr int kMostElements = 32;
constexpr Shape shape_of(std::uint32_t dim, int v) {
    const std::uint32_t need = (dim + v - 1) / v;
    constexpr int kShapes[][2] = {{16, 1}, {16, 2}, {64, 1}, {64, 2}, {64, 4}, {64, 8}, {256, 4}, {256, 8}, {1024, 2}, {1024, 4}, {1024, 16}};
    for (const auto& s : kShapes)
        if (need <= static_cast<std::uint32_t>(s[0] * s[1]) && s[1] * v <= kMostElements) return {s[0], s[1], s[0] < 256 ? 256u / s[0] : 1u};
    return {0, 0, 0};
}

bool rows_in_line(const nesle_heads& x, const nesle_norm_args& a) {
    return (a.batch == 1 || x.stride_n == a.heads * x.stride_h) &&
           (a.steps == 1 || x.stride_t == static_cast<std::int64_t>(a.batch) * a.heads * x.stride_h);
}

std::uint64_t rows_of(const nesle_norm_args& a) { return static_cast<std::uint64_t>(a.steps) * a.batch * a.heads; }

// Elements a load: both directions take as many.
template <typename T>
int vector_of(const nesle_norm_args& x, bool grad) {
    constexpr int v = 16 / sizeof(T);
    const auto aligned = [](const nesle_heads& t) {
        const Heads<T> h = heads<T>(t);
        return sizeof(T) == 4 ? h.vec : h.wide;
    };
    return x.dim % v == 0 && aligned(x.x) && (!grad || aligned(x.dy)) ? v : 1;
}

// Workgroups: as many as fill the card a few times over.  65,536 rows of 256 in bfloat16 and
// eight times the rows, us, with at most 1,024, 2,048 and 4,096: 12.7, 13.0, 13.6 and 95,
// 105, 89; the gradient with 512, 768 and 1,024: 25, 22, 21.7 and 216, 172, 152.
constexpr std::uint32_t kMostBlocks = 4096, kGradBlocks = 1024;
static_assert(kGradBlocks <= kMostPartials);

std::uint32_t blocks_of(const nesle_norm_args& a, const Shape& s, std::uint32_t most) {
    const std::uint64_t want = (rows_of(a) + s.groups - 1) / s.groups;
    return static_cast<std::uint32_t>(std::min<std::uint64_t>(std::max<std::uint64_t>(want, 1), most));
}

template <typename T>
NormArgs<T> norm_args(const nesle_norm_args& x) {
    NormArgs<T> a{};
    a.x = heads<T>(x.x);
    a.dy = heads<T>(x.dy);
    a.weight = x.weight;
    a.bias = x.bias;
    a.y = static_cast<T*>(x.y);
    a.dx = static_cast<T*>(x.dx);
    a.partials = x.scratch;
    a.rows = static_cast<std::uint32_t>(rows_of(x));
    a.batch = x.batch;
    a.heads = x.heads;
    a.dim = x.dim;
    a.plain = rows_in_line(x.x, x);
    a.plain_dy = rows_in_line(x.dy, x);
    a.inv_dim = 1.0f / static_cast<float>(x.dim);
    a.eps = x.eps;
    return a;
}

template <typename T, int V, bool GRAD, int L, int N>
void launch_shape(const NormArgs<T>& a, std::uint32_t blocks, hipStream_t s) {
    constexpr std::uint32_t kDim = L * N * V < NESLE_NORM_MAX_DIM ? L * N * V : NESLE_NORM_MAX_DIM;
    constexpr Shape kShape = shape_of(kDim, V);        // of the largest row that this shape holds
    if constexpr (kShape.lanes != L || kShape.vectors != N) return;      // another one does
    else if constexpr (GRAD) hipLaunchKernelGGL((layer_norm_grad_kernel<T, V, N, L>), dim3(blocks), dim3(kBlock<L>), 0, s, a);
    else hipLaunchKernelGGL((layer_norm_kernel<T, V, N, L>), dim3(blocks), dim3(kBlock<L>), 0, s, a);
}

template <typename T, int V, bool GRAD>
void launch(const NormArgs<T>& a, const Shape& shape, std::uint32_t blocks, hipStream_t s) {
    switch (shape.lanes * 100 + shape.vectors) {
        case 1601: launch_shape<T, V, GRAD, 16, 1>(a, blocks, s); break;
        case 1602: launch_shape<T, V, GRAD, 16, 2>(a, blocks, s); break;
        case 6401: launch_shape<T, V, GRAD, 64, 1>(a, blocks, s); break;
        case 6402: launch_shape<T, V, GRAD, 64, 2>(a, blocks, s); break;
        case 6404: launch_shape<T, V, GRAD, 64, 4>(a, blocks, s); break;
        case 6408: launch_shape<T, V, GRAD, 64, 8>(a, blocks, s); break;
        case 25604: launch_shape<T, V, GRAD, 256, 4>(a, blocks, s); break;
        case 25608: launch_shape<T, V, GRAD, 256, 8>(a, blocks, s); break;
        case 102402: launch_shape<T, V, GRAD, 1024, 2>(a, blocks, s); break;
        case 102404: launch_shape<T, V, GRAD, 1024, 4>(a, blocks, s); break;
        default: launch_shape<T, V, GRAD, 1024, 16>(a, blocks, s); break;
    }
}

template <typename T, bool GRAD>
int norm(const char* who, const nesle_norm_args& x, hipStream_t s) {
    NormArgs<T> a = norm_args<T>(x);
    const int v = vector_of<T>(x, GRAD);
    const Shape shape = shape_of(x.dim, v);
    const std::uint32_t blocks = blocks_of(x, shape, GRAD ? kGradBlocks : kMostBlocks);
    const bool sums = GRAD && (x.dweight != nullptr || x.dbias != nullptr);
    if (!sums) a.partials = nullptr;
    if (v == 1) launch<T, 1, GRAD>(a, shape, blocks, s);
    else launch<T, 16 / sizeof(T), GRAD>(a, shape, blocks, s);
    if (sums)
        hipLaunchKernelGGL(norm_weight_sum, dim3((2 * x.dim + 15) / 16), dim3(1024), 0, s, x.scratch, x.dweight, x.dbias, x.dim, blocks);
    return launched(who);
}

int check(const char* who, const nesle_norm_args* a) {
    if (a == nullptr) return refuse(who, "null arguments");
    if (a->dtype != NESLE_MEM_F32 && a->dtype != NESLE_MEM_BF16) return refuse(who, "dtype must be NESLE_MEM_F32 or NESLE_MEM_BF16");
    if (a->dim == 0 || a->dim > NESLE_NORM_MAX_DIM) return refuse(who, "dim must be 1 to " + std::to_string(NESLE_NORM_MAX_DIM));
    if (!(a->eps >= 0.0f) || !(a->eps < INFINITY)) return refuse(who, "eps must be finite and not below 0");
    // Two factors at a time: the product of three may pass 64 bits.
    const std::uint64_t of_step = static_cast<std::uint64_t>(a->batch) * a->heads;
    if (a->steps != 0 && of_step > 0xffffffffull / a->steps) return refuse(who, "rows must be below 2^32");
    return NESLE_OK;
}

int check_pointers(const char* who, std::initializer_list<const void*> needed, std::initializer_list<const void*> aligned) {
    for (const void* p : needed)
        if (p == nullptr) return refuse(who, "null device pointer");
    for (const void* p : aligned)
        if (reinterpret_cast<std::uintptr_t>(p) % 16 != 0) return refuse(who, "outputs, weights and workspaces must lie on 16-byte boundaries");
    return NESLE_OK;
}

}  // namespace
}  // namespace nesle::mem

using namespace nesle::mem;

extern "C" {

std::uint64_t nesle_norm_scratch_floats(const nesle_norm_args* a) {
    if (a == nullptr || a->dim == 0 || a->dim > NESLE_NORM_MAX_DIM) return 0;
    return 2ull * kGradBlocks * a->dim;
}

int nesle_layer_norm(const nesle_norm_args* a, void* stream) {
    const char* who = "nesle_layer_norm";
    int rc = check(who, a);
    if (rc != NESLE_OK || rows_of(*a) == 0) return rc;
    rc = check_pointers(who, {a->x.data, a->y}, {a->y, a->weight, a->bias});
    if (rc != NESLE_OK) return rc;
    const auto s = static_cast<hipStream_t>(stream);
    return a->dtype == NESLE_MEM_F32 ? norm<float, false>(who, *a, s) : norm<bf16, false>(who, *a, s);
}

int nesle_layer_norm_grad(const nesle_norm_args* a, void* stream) {
    const char* who = "nesle_layer_norm_grad";
    int rc = check(who, a);
    if (rc != NESLE_OK) return rc;
    const bool sums = a->dweight != nullptr || a->dbias != nullptr;
    if (rows_of(*a) != 0) {
        rc = check_pointers(who, {a->x.data, a->dy.data, a->dx}, {a->dx, a->weight, a->scratch, a->dweight, a->dbias});
        if (rc != NESLE_OK) return rc;
    } else if (!sums) {
        return NESLE_OK;
    }
    if (sums && a->scratch == nullptr) return refuse(who, "null device pointer");
    const auto s = static_cast<hipStream_t>(stream);
    return a->dtype == NESLE_MEM_F32 ? norm<float, true>(who, *a, s) : norm<bf16, true>(who, *a, s);
}

}  // extern "C"
