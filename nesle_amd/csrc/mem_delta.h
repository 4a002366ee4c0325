// mem_delta.h -- what the kernels of the gated delta rule share: their
// arguments and the rule that ends an episode.
#pragma once

#include <initializer_list>
#include <type_traits>
#include <utility>

#include "mem_common.h"

namespace nesle::mem {

constexpr int kChunk = NESLE_DELTA_CHUNK;

// exp(g) is zero in float32 below this: its smallest value is 2^-149, and half of
// that, which rounds to zero, is exp(-103.9720771), between this number and the next
// lower one.  The state is dropped there, not multiplied by zero, and every gate that
// is multiplied keeps a finite logarithm.
constexpr float kDropBelow = -103.972076f;
// What a dropping token's gate counts for in the running sums: exp of any
// difference across it is zero, and 32 of them leave a double 9 digits after the
// point for the others.
constexpr float kGone = -100000.0f;

template <typename T>
struct DeltaArgs {
    Heads<T> q, k, v, dout;
    const float *g, *beta;
    const std::uint8_t* resets;
    const float* state;
    T* out;
    float *state_out, *saved;
    const float* dstate_out;
    T *dq, *dk, *dv;
    float *dg, *dbeta, *dstate, *scratch;
    std::uint32_t steps, batch, hk, hv, group, dk_dim, dv_dim;     // group: value heads of a key head
    float scale;
};

template <typename T>
DeltaArgs<T> delta_args(const nesle_delta_args& a) {
    DeltaArgs<T> d{};
    d.q = heads<T>(a.q);
    d.k = heads<T>(a.k);
    d.v = heads<T>(a.v);
    d.dout = heads<T>(a.dout);
    d.g = a.g;
    d.beta = a.beta;
    d.resets = a.resets;
    d.state = a.state;
    d.out = static_cast<T*>(a.out);
    d.state_out = a.state_out;
    d.saved = a.saved;
    d.dstate_out = a.dstate_out;
    d.dq = static_cast<T*>(a.dq);
    d.dk = static_cast<T*>(a.dk);
    d.dv = static_cast<T*>(a.dv);
    d.dg = a.dg;
    d.dbeta = a.dbeta;
    d.dstate = a.dstate;
    d.scratch = a.scratch;
    d.steps = a.steps;
    d.batch = a.batch;
    d.hk = a.k_heads;
    d.hv = a.v_heads;
    d.group = a.v_heads / a.k_heads;
    d.dk_dim = a.k_dim;
    d.dv_dim = a.v_dim;
    d.scale = a.scale;
    return d;
}

inline std::uint32_t padded_dim(const nesle_delta_args& a) {
    const std::uint32_t d = a.k_dim > a.v_dim ? a.k_dim : a.v_dim;
    return d <= 32 ? 32 : d <= 64 ? 64 : 128;
}

// Whether a chunk's rows of any tensor span 2^31 bytes or more, past what a
// 32-bit offset reaches.
inline bool wide_rows(const nesle_delta_args& a) {
    const std::int64_t item = a.dtype == NESLE_MEM_F32 ? 4 : 2, limit = ((1ll << 31) - 4096) / (kChunk - 1);
    for (const nesle_heads* x : {&a.q, &a.k, &a.v, &a.dout})
        if (x->stride_t < 0 || x->stride_t * item >= limit) return true;
    // What the kernels write: of the inputs' type, and shares of key heads' gradients in float32.
    const std::int64_t heads = static_cast<std::int64_t>(a.batch) * a.v_heads;
    return heads * (a.k_dim > a.v_dim ? a.k_dim : a.v_dim) * (a.v_heads > a.k_heads ? 4 : item) >= limit;
}

// Arguments that no call may have.
inline int check_delta(const char* who, const nesle_delta_args* a) {
    if (a == nullptr) return refuse(who, "null arguments");
    if (a->dtype != NESLE_MEM_F32 && a->dtype != NESLE_MEM_BF16) return refuse(who, "dtype must be NESLE_MEM_F32 or NESLE_MEM_BF16");
    for (const std::uint32_t d : {a->k_dim, a->v_dim})
        if (d == 0 || d % 8 != 0 || d > NESLE_DELTA_MAX_DIM)
            return refuse(who, "k_dim and v_dim must be multiples of 8 up to " + std::to_string(NESLE_DELTA_MAX_DIM));
    if (a->k_heads == 0 || a->v_heads == 0 || a->v_heads % a->k_heads != 0)
        return refuse(who, "v_heads must be a multiple of k_heads");
    if (static_cast<std::uint64_t>(a->batch) * a->v_heads > (1u << 22))
        return refuse(who, "batch * v_heads must be at most 4,194,304");
    if (a->steps > (1u << 30)) return refuse(who, "steps must be at most 2^30");
    return NESLE_OK;
}

// The state tensors are read and written as 16-byte words.
inline bool aligned16(const void* p) { return reinterpret_cast<std::uintptr_t>(p) % 16 == 0; }

// Pointers that a call over at least one token and console needs.
inline int check_delta_inputs(const char* who, const nesle_delta_args* a) {
    if (!a->q.data || !a->k.data || !a->v.data || !a->g || !a->beta) return refuse(who, "null device pointer");
    if (!aligned16(a->state) || !aligned16(a->state_out) || !aligned16(a->saved) || !aligned16(a->dstate_out) ||
        !aligned16(a->dstate) || !aligned16(a->scratch) || !aligned16(a->out) || !aligned16(a->dq) || !aligned16(a->dk) ||
        !aligned16(a->dv))
        return refuse(who, "states, outputs and workspaces must lie on 16-byte boundaries");
    return NESLE_OK;
}

}  // namespace nesle::mem
