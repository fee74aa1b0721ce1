// Single-token forms: one step of the selective scan or of the short convolution for each entry of
// a batch, on states that live in a pool and are updated in place.
//
// Entry m works on state slots[m] (or m).  A slot outside the pool marks an idle entry: its output
// is zero and no state is touched.  Entries that name the same slot are consecutive tokens of that
// sequence, in the order of the batch: the first of them computes them all, so that no two CTAs
// ever work on one state and the result does not depend on their timing.
//
// The floor: the state pool's rows, read and written once (4-byte states: 8 S bytes per channel); for few entries the
// launch.  256 entries, bf16: scan of 4096 channels with 16 states 48 us (22 for the bytes), convolution of 8192 channels 9.3
// (5.1).  What is between: the slot, the list of slots and the state are asked for one after the other, and every CTA
// reads the whole list: 8192 entries of 1024 channels take 379 us without slots and 678 with them, the convolution 25 and 126.
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
    int softplus, vec, vec_proj;  // vec: S is a multiple of 4 and the states and decays are 16-byte aligned; vec_proj: 4 states of B and C likewise
    Slots slots;
    View2 x, dt, z, out, B, C;
    const float *A, *D, *dt_bias;
    float *state;
};

// N (a multiple of 4) adjacent elements, 8 (16-bit types) or 16 bytes at a time.
template <typename T, int N>
__device__ __forceinline__ void load_array(const T *p, int64_t at, int64_t extent, int site, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        f[i] = f[i + 1] = f[i + 2] = f[i + 3] = 0.0f;
        if (!SSB_VECTOR_OK(p + at + i, 4 * (int)sizeof(T), at + i + 3, extent, site)) continue;
        if constexpr (sizeof(T) == 4) {
            const float4 w = *reinterpret_cast<const float4 *>(p + at + i);
            f[i] = w.x; f[i + 1] = w.y; f[i + 2] = w.z; f[i + 3] = w.w;
        } else {
            const uint2 w = *reinterpret_cast<const uint2 *>(p + at + i);
            unpack2<T>(w.x, f[i], f[i + 1]);
            unpack2<T>(w.y, f[i + 2], f[i + 3]);
        }
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_array(T *p, int64_t at, int64_t extent, int site, const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        if (!SSB_VECTOR_OK(p + at + i, 4 * (int)sizeof(T), at + i + 3, extent, site)) continue;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(p + at + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
        else *reinterpret_cast<uint2 *>(p + at + i) = make_uint2(pack2<T>(f[i], f[i + 1]), pack2<T>(f[i + 2], f[i + 3]));
    }
}

// LANES lanes share a channel, each with 4 adjacent states at a time (one 16-byte access where S is
// a multiple of 4).  EACH adjacent channels a thread, 4 or 1: with 4, each lane of a quad prepares one of the
// four channels (its step size, input, gate) and hands it to the others, and the sums over the states are
// exchanged so that each is left with one.  Instructions bound the large calls, not the states' bytes: with every
// lane preparing every channel, 256 entries of 4096 channels took 59 us whatever the loads in flight.
template <typename io_t, int LANES, int EACH>
__global__ void __launch_bounds__(128) selective_step_kernel(const __grid_constant__ SelectiveStepArgs p) {
    static_assert(EACH == 1 || (EACH == 4 && LANES >= 4), "a lane of a quad for each channel");
    constexpr int CB = 128 / LANES * EACH;
    const int64_t m0 = blockIdx.x;
    const int part = threadIdx.x % LANES;
    const int64_t first = (int64_t)blockIdx.y * CB + threadIdx.x / LANES * EACH;
    const int S = (int)p.states;
    const Turn turn = turn_of(p.slots, m0);
    if (!turn.mine) return;
    // the channel this lane prepares and stores; lanes behind the last one stay for the shuffles, on the last one's values
    const int64_t own = first + part % EACH;
    const bool stores = part < EACH && own < p.channels;
    if (turn.slot < 0) {
        if (stores) store_one(static_cast<io_t *>(p.out.data), m0 * p.out.s0 + own * p.out.s1, p.out.extent, 300, 0.0f);
        return;
    }
    const int64_t co = own < p.channels ? own : p.channels - 1;
    const int64_t state_extent = p.slots.pool * p.channels * S;
    const float D = p.D != nullptr ? load_one(p.D, co, p.channels, 301) : 0.0f;
    const float bias = p.dt_bias != nullptr ? load_one(p.dt_bias, co, p.channels, 302) : 0.0f;
    const auto projection = [&](const View2 &v, int64_t at, int have, int site, float (&f)[4]) {
        if (p.vec_proj) {
            load_array(static_cast<const io_t *>(v.data), at, v.extent, site, f);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = i < have ? load_one(static_cast<const io_t *>(v.data), at + i * v.s2, v.extent, site) : 0.0f;
        }
    };
    const auto quad = [&](const float *v, int64_t at, int have, int64_t extent, int site, float (&f)[4]) {
        if (p.vec) {
            load_array(v, at, extent, site, f);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = i < have ? load_one(v, at + i, extent, site) : 0.0f;
        }
    };
    for (int64_t m = m0; m < p.slots.entries; ++m) {
        if (m > m0) {
            if (!turn.more) break;
            if (p.slots.slots[m] != turn.slot) continue;
        }
        const float x = load_one(static_cast<const io_t *>(p.x.data), m * p.x.s0 + co * p.x.s1, p.x.extent, 303);
        float dt = load_one(static_cast<const io_t *>(p.dt.data), m * p.dt.s0 + co * p.dt.s1, p.dt.extent, 304);
        const float z = p.z.data != nullptr ? load_one(static_cast<const io_t *>(p.z.data), m * p.z.s0 + co * p.z.s1, p.z.extent, 310) : 0.0f;
        float y[EACH];
#pragma unroll
        for (int k = 0; k < EACH; ++k) y[k] = 0.0f;
        bool prepared = false;
        for (int n = part * 4; n - part * 4 < S; n += LANES * 4) {  // as often in all lanes
            const int have = S - n < 4 ? S - n : 4;                // none: below 1
            float h[EACH][4], a[EACH][4], b[4] = {}, r[4] = {};
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                const int64_t c = first + k < p.channels ? first + k : p.channels - 1;
#pragma unroll
                for (int i = 0; i < 4; ++i) h[k][i] = a[k][i] = 0.0f;
                if (have > 0) {
                    quad(p.state, (turn.slot * p.channels + c) * S + n, have, state_extent, 305, h[k]);
                    quad(p.A, c * S + n, have, p.channels * S, 306, a[k]);
                }
            }
            if (!prepared) {
                dt += bias;
                if (p.softplus) dt = softplus(dt);
                prepared = true;
            }
            int64_t group = -1;
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                const int64_t c = first + k < p.channels ? first + k : p.channels - 1;
                const int64_t g = p.per_group == p.channels ? 0 : c / p.per_group;
                if (g != group && have > 0) {
                    projection(p.B, m * p.B.s0 + g * p.B.s1 + n * p.B.s2, have, 307, b);
                    projection(p.C, m * p.C.s0 + g * p.C.s1 + n * p.C.s2, have, 308, r);
                    group = g;
                }
                float d = dt, v = x;
                if constexpr (EACH > 1) {
                    d = __shfl_sync(kFullMask, dt, k, 4);
                    v = __shfl_sync(kFullMask, x, k, 4);
                }
                const float u = d * v, d2 = d * kLog2e;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    h[k][i] = fmaf(exp2_approx(fmaf(d2, a[k][i], kExponentShift)), h[k][i], u * b[i]);
                    if (i < have) y[k] = fmaf(r[i], h[k][i], y[k]);
                }
                if (first + k < p.channels && have > 0) {
                    const int64_t at = (turn.slot * p.channels + c) * S + n;
                    if (p.vec) {
                        store_array(p.state, at, state_extent, 309, h[k]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (i < have) store_one(p.state, at + i, state_extent, 309, h[k][i]);
                    }
                }
            }
        }
        float sum = sum_and_spread<LANES>(y, part);
        if (stores) {
            sum = fmaf(D, x, sum);
            if (p.z.data != nullptr) sum *= z * logistic(z);
            store_one(static_cast<io_t *>(p.out.data), m * p.out.s0 + own * p.out.s1, p.out.extent, 300, sum);
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

// V adjacent channels a thread: 4 where their pieces are whole and aligned, else 1.
template <typename io_t, int W, int V>
__global__ void __launch_bounds__(128) conv_step_kernel(const __grid_constant__ ConvStepArgs p) {
    const int64_t m0 = blockIdx.x, c = ((int64_t)blockIdx.y * 128 + threadIdx.x) * V;
    const Turn turn = turn_of(p.slots, m0);
    if (!turn.mine || c >= p.channels) return;
    io_t *out = static_cast<io_t *>(p.out.data);
    const auto put = [&](int64_t m, const float (&v)[V]) {
        const int64_t at = m * p.out.s0 + c * p.out.s1;
        if constexpr (V == 4) store_array(out, at, p.out.extent, 320, v);
        else store_one(out, at, p.out.extent, 320, v[0]);
    };
    if (turn.slot < 0) {
        const float zero[V] = {};
        put(m0, zero);
        return;
    }
    io_t *state = static_cast<io_t *>(p.state);
    const int64_t at = (turn.slot * p.channels + c) * (W - 1), extent = p.slots.pool * p.channels * (W - 1);
    float w[V * W], bias[V] = {}, seen[V * (W - 1)];  // [channel][tap], [channel][input]
    if constexpr (V == 4) {
        load_array(state, at, extent, 323, seen);
        if (p.weight_f32) {
            load_array(static_cast<const float *>(p.weight), c * W, p.channels * W, 321, w);
            if (p.bias != nullptr) load_array(static_cast<const float *>(p.bias), c, p.channels, 322, bias);
        } else {
            load_array(static_cast<const io_t *>(p.weight), c * W, p.channels * W, 321, w);
            if (p.bias != nullptr) load_array(static_cast<const io_t *>(p.bias), c, p.channels, 322, bias);
        }
    } else {
#pragma unroll
        for (int i = 0; i < W - 1; ++i) seen[i] = load_one(state, at + i, extent, 323);
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = load_weight<io_t>(p.weight, p.weight_f32, c * W + i, p.channels * W, 321);
        if (p.bias != nullptr) bias[0] = load_weight<io_t>(p.bias, p.weight_f32, c, p.channels, 322);
    }
    for (int64_t m = m0; m < p.slots.entries; ++m) {
        if (m > m0) {
            if (!turn.more) break;
            if (p.slots.slots[m] != turn.slot) continue;
        }
        float x[V], v[V];
        const int64_t from = m * p.x.s0 + c * p.x.s1;
        if constexpr (V == 4) load_array(static_cast<const io_t *>(p.x.data), from, p.x.extent, 324, x);
        else x[0] = load_one(static_cast<const io_t *>(p.x.data), from, p.x.extent, 324);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            v[k] = bias[k];
#pragma unroll
            for (int i = 0; i < W - 1; ++i) v[k] = fmaf(w[k * W + i], seen[k * (W - 1) + i], v[k]);
            v[k] = fmaf(w[k * W + W - 1], x[k], v[k]);
            if (p.silu) v[k] *= logistic(v[k]);
#pragma unroll
            for (int i = 0; i + 1 < W - 1; ++i) seen[k * (W - 1) + i] = seen[k * (W - 1) + i + 1];
            seen[k * (W - 1) + W - 2] = x[k];
        }
        put(m, v);
    }
    if constexpr (V == 4) {
        store_array(state, at, extent, 323, seen);
    } else {
#pragma unroll
        for (int i = 0; i < W - 1; ++i) store_one(state, at + i, extent, 323, seen[i]);
    }
}

}  // namespace ssb
