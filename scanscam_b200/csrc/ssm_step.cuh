// Single-token forms: one step of the selective scan or of the short convolution for each entry of
// a batch, on states that live in a pool and are updated in place.
//
// Entry m works on state slots[m] (or m).  A slot outside the pool marks an idle entry: its output
// is zero and no state is touched.  Entries that name the same slot are consecutive tokens of that
// sequence, in the order of the batch: the first of them computes them all, so that no two CTAs
// ever work on one state and the result does not depend on their timing.
//
// Bound by the state pool's rows, read and written once (4-byte states: 8 S bytes per channel), and
// for few entries by the launch.
#pragma once

#include "ssm_common.cuh"

namespace ssb {

struct View2 {  // [M, C] or, for projections, [M, G, S]
    void *data;
    int64_t s0, s1, s2, extent;
};

struct Slots {
    const int32_t *slots;  // nullptr: entry m has state m
    int64_t entries, pool;
};

// Which state entry m works on (-1: idle), and whether this CTA computes it; `more`: later entries
// name the same slot.  Called by all threads of the CTA.
struct Turn {
    int64_t slot;
    bool mine, more;
};
__device__ __forceinline__ Turn turn_of(const Slots &s, int64_t m) {
    if (s.slots == nullptr) return {m < s.pool ? m : -1, true, false};
    const int64_t slot = s.slots[m];
    if (slot < 0 || slot >= s.pool) return {-1, true, false};
    bool before = false, after = false;
    for (int64_t i = threadIdx.x; i < s.entries; i += blockDim.x) {
        if (s.slots[i] == slot) {
            before |= i < m;
            after |= i > m;
        }
    }
    const bool mine = __syncthreads_or(before) == 0, more = __syncthreads_or(after) != 0;
    return {slot, mine, more};
}

struct SelectiveStepArgs {
    int64_t channels, per_group, states;
    int softplus, vec;  // vec: S is a multiple of 4 and the states and decays are 16-byte aligned
    Slots slots;
    View2 x, dt, z, out, B, C;
    const float *A, *D, *dt_bias;
    float *state;
};

// LANES lanes share a channel, each with 4 adjacent states at a time (one 16-byte access where S is
// a multiple of 4); the read-out is summed over them by shuffles.
template <typename io_t, int LANES>
__global__ void __launch_bounds__(128) selective_step_kernel(const __grid_constant__ SelectiveStepArgs p) {
    constexpr int CB = 128 / LANES;
    const int64_t m0 = blockIdx.x;
    const int part = threadIdx.x % LANES;
    const int64_t c = (int64_t)blockIdx.y * CB + threadIdx.x / LANES;
    const bool live = c < p.channels;
    const int S = (int)p.states;
    const Turn turn = turn_of(p.slots, m0);
    if (!turn.mine) return;
    if (turn.slot < 0) {
        if (live && part == 0) store_one(static_cast<io_t *>(p.out.data), m0 * p.out.s0 + c * p.out.s1, p.out.extent, 300, 0.0f);
        return;
    }
    const int64_t cc = live ? c : p.channels - 1;  // lanes behind the last channel stay for the shuffles
    const int64_t g = cc / p.per_group;
    const float D = p.D != nullptr ? load_one(p.D, cc, p.channels, 301) : 0.0f;
    const float bias = p.dt_bias != nullptr ? load_one(p.dt_bias, cc, p.channels, 302) : 0.0f;
    const bool vec = p.vec != 0;
    const int64_t state_extent = p.slots.pool * p.channels * S;
    for (int64_t m = m0; m < p.slots.entries; ++m) {
        if (m > m0) {
            if (!turn.more) break;
            if (p.slots.slots[m] != turn.slot) continue;
        }
        const float x = load_one(static_cast<const io_t *>(p.x.data), m * p.x.s0 + cc * p.x.s1, p.x.extent, 303);
        float dt = load_one(static_cast<const io_t *>(p.dt.data), m * p.dt.s0 + cc * p.dt.s1, p.dt.extent, 304) + bias;
        if (p.softplus) dt = softplus(dt);
        const float u = dt * x;
        float y = 0.0f;
        for (int n = part * 4; n < S; n += LANES * 4) {
            const int64_t at = (turn.slot * p.channels + cc) * S + n;
            const int have = S - n < 4 ? S - n : 4;
            float h[4] = {0, 0, 0, 0}, a[4] = {0, 0, 0, 0};
            if (vec && SSB_VECTOR_OK(p.state + at, 16, at + 3, state_extent, 305) && SSB_VECTOR_OK(p.A + cc * S + n, 16, cc * S + n + 3, p.channels * S, 306)) {
                const float4 hv = *reinterpret_cast<const float4 *>(p.state + at);
                const float4 av = *reinterpret_cast<const float4 *>(p.A + cc * S + n);
                h[0] = hv.x; h[1] = hv.y; h[2] = hv.z; h[3] = hv.w;
                a[0] = av.x; a[1] = av.y; a[2] = av.z; a[3] = av.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < have) {
                        h[i] = load_one(p.state, at + i, state_extent, 305);
                        a[i] = load_one(p.A, cc * S + n + i, p.channels * S, 306);
                    }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < have) {
                    const float b = load_one(static_cast<const io_t *>(p.B.data), m * p.B.s0 + g * p.B.s1 + (n + i) * p.B.s2, p.B.extent, 307);
                    const float r = load_one(static_cast<const io_t *>(p.C.data), m * p.C.s0 + g * p.C.s1 + (n + i) * p.C.s2, p.C.extent, 308);
                    h[i] = fmaf(exp2_approx(dt * (a[i] * kLog2e)), h[i], u * b);
                    y = fmaf(r, h[i], y);
                }
            if (live) {
                if (vec && SSB_VECTOR_OK(p.state + at, 16, at + 3, state_extent, 309)) {
                    *reinterpret_cast<float4 *>(p.state + at) = make_float4(h[0], h[1], h[2], h[3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i < have) store_one(p.state, at + i, state_extent, 309, h[i]);
                }
            }
        }
#pragma unroll
        for (int d = LANES / 2; d >= 1; d >>= 1) y += __shfl_xor_sync(kFullMask, y, d);
        if (live && part == 0) {
            y = fmaf(D, x, y);
            if (p.z.data != nullptr) {
                const float z = load_one(static_cast<const io_t *>(p.z.data), m * p.z.s0 + cc * p.z.s1, p.z.extent, 310);
                y *= z * logistic(z);
            }
            store_one(static_cast<io_t *>(p.out.data), m * p.out.s0 + c * p.out.s1, p.out.extent, 300, y);
        }
    }
}

struct ConvStepArgs {
    int64_t channels;
    int width, silu, weight_f32;
    Slots slots;
    View2 x, out;
    const void *weight, *bias;  // [C, W], [C]; in the inputs' type, or float32
    void *state;                // [pool, C, W-1]
};

template <typename io_t>
__device__ __forceinline__ float load_weight(const void *w, int f32, int64_t at, int64_t extent, int site) {
    return f32 ? load_one(static_cast<const float *>(w), at, extent, site) : load_one(static_cast<const io_t *>(w), at, extent, site);
}

template <typename io_t, int W>
__global__ void __launch_bounds__(128) conv_step_kernel(const __grid_constant__ ConvStepArgs p) {
    const int64_t m0 = blockIdx.x, c = (int64_t)blockIdx.y * 128 + threadIdx.x;
    const Turn turn = turn_of(p.slots, m0);
    if (!turn.mine || c >= p.channels) return;
    io_t *out = static_cast<io_t *>(p.out.data);
    if (turn.slot < 0) {
        store_one(out, m0 * p.out.s0 + c * p.out.s1, p.out.extent, 320, 0.0f);
        return;
    }
    io_t *state = static_cast<io_t *>(p.state);
    const int64_t at = (turn.slot * p.channels + c) * (W - 1), extent = p.slots.pool * p.channels * (W - 1);
    float w[W], seen[W - 1];
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = load_weight<io_t>(p.weight, p.weight_f32, c * W + i, p.channels * W, 321);
    const float bias = p.bias != nullptr ? load_weight<io_t>(p.bias, p.weight_f32, c, p.channels, 322) : 0.0f;
#pragma unroll
    for (int i = 0; i < W - 1; ++i) seen[i] = load_one(state, at + i, extent, 323);
    for (int64_t m = m0; m < p.slots.entries; ++m) {
        if (m > m0) {
            if (!turn.more) break;
            if (p.slots.slots[m] != turn.slot) continue;
        }
        const float x = load_one(static_cast<const io_t *>(p.x.data), m * p.x.s0 + c * p.x.s1, p.x.extent, 324);
        float v = bias;
#pragma unroll
        for (int i = 0; i < W - 1; ++i) v = fmaf(w[i], seen[i], v);
        v = fmaf(w[W - 1], x, v);
        if (p.silu) v *= logistic(v);
        store_one(out, m * p.out.s0 + c * p.out.s1, p.out.extent, 320, v);
#pragma unroll
        for (int i = 0; i + 1 < W - 1; ++i) seen[i] = seen[i + 1];
        seen[W - 2] = x;
    }
#pragma unroll
    for (int i = 0; i < W - 1; ++i) store_one(state, at + i, extent, 323, seen[i]);
}

}  // namespace ssb
