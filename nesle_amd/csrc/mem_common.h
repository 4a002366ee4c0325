// mem_common.h -- element types, strided loads and 16x16 float32 matrix tiles
// shared by the kernels of the memory operators (include/nesle_memory.h).
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "nes_launch.h"
#include "../../include/nesle_memory.h"

namespace nesle::mem {

using bf16 = __bf16;
using f4 = float __attribute__((ext_vector_type(4)));
using u4 = std::uint32_t __attribute__((ext_vector_type(4)));
using u2 = std::uint32_t __attribute__((ext_vector_type(2)));

__device__ inline float lo_half(std::uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ inline float hi_half(std::uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ inline std::uint32_t pack_bf16(float a, float b) {
    using b2 = bf16 __attribute__((ext_vector_type(2)));
    const b2 p = {static_cast<bf16>(a), static_cast<bf16>(b)};      // rounds to nearest even
    return __builtin_bit_cast(std::uint32_t, p);
}

// Four consecutive elements; `vec` says that their address is a multiple of
// their size (uniform over the launch).
__device__ inline f4 load4(const float* p, bool vec) {
    if (vec) return *reinterpret_cast<const f4*>(p);
    return f4{p[0], p[1], p[2], p[3]};
}
__device__ inline f4 load4(const bf16* p, bool vec) {
    if (vec) {
        const u2 w = *reinterpret_cast<const u2*>(p);
        return f4{lo_half(w.x), hi_half(w.x), lo_half(w.y), hi_half(w.y)};
    }
    return f4{static_cast<float>(p[0]), static_cast<float>(p[1]), static_cast<float>(p[2]), static_cast<float>(p[3])};
}
// Eight consecutive elements of aligned ones.
__device__ inline void load8(const bf16* p, f4& a, f4& b) {
    const u4 w = *reinterpret_cast<const u4*>(p);
    a = f4{lo_half(w.x), hi_half(w.x), lo_half(w.y), hi_half(w.y)};
    b = f4{lo_half(w.z), hi_half(w.z), lo_half(w.w), hi_half(w.w)};
}
__device__ inline void store8(bf16* p, f4 a, f4 b) {
    *reinterpret_cast<u4*>(p) = u4{pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w)};
}
__device__ inline void store4(float* p, f4 v) { *reinterpret_cast<f4*>(p) = v; }
__device__ inline void store4(bf16* p, f4 v) {
    *reinterpret_cast<u2*>(p) = u2{pack_bf16(v.x, v.y), pack_bf16(v.z, v.w)};
}

// A strided [steps][batch][heads][dim] tensor on the device, as the kernels
// take it: `vec` is set where every group of four elements is aligned.
template <typename T>
struct Heads {
    const T* data;
    std::int64_t t, n, h;
    bool vec, wide;      // wide: of eight
    __device__ const T* row(std::int64_t step, std::int64_t env, std::int64_t head) const {
        return data + step * t + env * n + head * h;
    }
};

template <typename T>
Heads<T> heads(const nesle_heads& x) {
    const auto aligned = [&](std::int64_t elements) {
        const std::int64_t bytes = elements * static_cast<std::int64_t>(sizeof(T));
        const auto whole = [&](std::int64_t stride) { return stride * static_cast<std::int64_t>(sizeof(T)) % bytes == 0; };
        return reinterpret_cast<std::uintptr_t>(x.data) % static_cast<std::uintptr_t>(bytes) == 0 && whole(x.stride_t) &&
               whole(x.stride_n) && whole(x.stride_h);
    };
    return {static_cast<const T*>(x.data), x.stride_t, x.stride_n, x.stride_h, aligned(4), aligned(8)};
}

inline int refuse(const char* who, const std::string& why) {
    set_last_error(std::string(who) + ": " + why);
    return NESLE_EINVAL;
}

inline int launched(const char* who) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return NESLE_OK;
    set_last_error(std::string(who) + ": launch failed: " + hipGetErrorString(e));
    return NESLE_EDEVICE;
}

// ---- 16x16 tiles --------------------------------------------------------------
// C[16][16] += A[16][16] B[16][16] in float32 by four v_mfma_f32_16x16x4_f32.
// With r = lane % 16 and g = lane / 16, the instruction reads A[r][g] and
// B[g][r] and holds C[4g + i][r], i = 0..3.  The sum over the inner index may
// be taken in any order, so instruction i takes inner indices 4g + i: an
// operand is four consecutive inner elements of one row, and a result tile
// C[x][y] is, as it lies in the registers, the operand of a product over x.
__device__ inline f4 mma(f4 a, f4 b, f4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b.z, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b.w, c, 0, 0, 0);
}

// Operand whose inner index runs along the rows of an LDS tile (row0, col0):
// lane r takes row r.  Row strides are 4 more than a multiple of 32 words, so
// 16 rows start at 16 different groups of four banks.
template <int STRIDE>
__device__ inline f4 along(const float* tile, int row0, int col0, int r, int g) {
    return *reinterpret_cast<const f4*>(tile + (row0 + r) * STRIDE + col0 + 4 * g);
}
// Operand whose inner index runs down the columns: lane r takes column r.
template <int STRIDE>
__device__ inline f4 down(const float* tile, int row0, int col0, int r, int g) {
    const float* p = tile + (row0 + 4 * g) * STRIDE + col0 + r;
    return f4{p[0], p[STRIDE], p[2 * STRIDE], p[3 * STRIDE]};
}

}  // namespace nesle::mem
