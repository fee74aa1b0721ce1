// Selective scan over whole sequences, forward: per channel c and state n
//     h_t = exp(dt_t A[c,n]) h_{t-1} + dt_t x_t B_t[n],     y_t = sum_n C_t[n] h_t + D x_t,     out = y silu(z).
//
// What bounds it: one exponential per (step, channel, state).  At 16 a clock and SM they take three
// times as long as the tensors' bytes in 16-bit storage, so the states never leave the registers and
// everything else is kept below 8 issue slots an exponential.
//
// LN lanes share a channel, each with SPL of its states (4; 8 beyond 128 states); a warp holds
// 32 / LN channels and walks the steps in order.  Per step and 4 states a lane issues 4 exponentials,
// 8 packed operations (exponent, input, recurrence, read-out, two states each) and 3 shared loads.
// The read-out is summed over the LN lanes once per LN steps, in LN - 1 shuffles that leave each lane
// with the sum of one step.  A tile of 32 steps is put into shared memory by the whole CTA: (dt, x)
// after the softplus, B and C as fp32; the next tile's bytes are fetched meanwhile.  The sums take the
// place of the steps in shared memory and leave, gated, with 16-byte stores.
#pragma once

#include "ssm_scan.cuh"

namespace ssb {

constexpr int kTile = 32;  // steps of a tile

// 16-byte pieces of a tile of a [N, C, T] view: 8 (4) adjacent channels of a step, or adjacent steps of a channel.
enum TileAccess : int { kTileAny = 0, kTileChannels = 1, kTileSteps = 2 };

template <typename io_t, int CB, int THREADS>
struct TilePieces {
    static constexpr int kPer = 16 / (int)sizeof(io_t);
    static constexpr int kPieces = (kTile * CB / kPer + THREADS - 1) / THREADS;
    static_assert(CB % kPer == 0, "whole pieces of channels");
    uint4 piece[kPieces];

    // where piece j of this thread lies in the tile: first step and channel
    __device__ __forceinline__ static bool place(int access, int j, int &t, int &c) {
        const int i = threadIdx.x + j * THREADS;
        if (access == kTileSteps) {
            c = i % CB;
            t = i / CB * kPer;
        } else {
            c = i % (CB / kPer) * kPer;
            t = i / (CB / kPer);
        }
        return i < kTile * CB / kPer;
    }
    __device__ __forceinline__ void fetch(const View3 &v, int64_t row, int64_t c0, int channels, int64_t t0, int64_t steps, int site) {
        const io_t *base = static_cast<const io_t *>(v.data);
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            int t, c;
            piece[j] = make_uint4(0, 0, 0, 0);
            if (!place(v.access, j, t, c) || t >= steps || c >= channels) continue;
            const int64_t at = row * v.sn + (c0 + c) * v.sc + (t0 + t) * v.st;
            const bool whole = v.access == kTileChannels ? c + kPer <= channels : v.access == kTileSteps;
            if (whole) {
                if (SSB_VECTOR_OK(base + at, 16, at + kPer - 1, v.extent, site)) piece[j] = *reinterpret_cast<const uint4 *>(base + at);
            } else {
                io_t e[kPer];
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    const int64_t i = at + k * v.sc;
                    e[k] = io_t(0.0f);
                    if (c + k < channels && SSB_INDEX_OK(i, v.extent, site)) e[k] = base[i];
                }
                memcpy(&piece[j], e, 16);
            }
        }
    }
    // element k of piece j as fp32; elements behind the last step are zero
    __device__ __forceinline__ void open(int j, float (&f)[kPer]) const {
        if constexpr (sizeof(io_t) == 2) {
            unpack2<io_t>(piece[j].x, f[0], f[1]);
            unpack2<io_t>(piece[j].y, f[2], f[3]);
            unpack2<io_t>(piece[j].z, f[4], f[5]);
            unpack2<io_t>(piece[j].w, f[6], f[7]);
        } else {
            f[0] = __uint_as_float(piece[j].x); f[1] = __uint_as_float(piece[j].y);
            f[2] = __uint_as_float(piece[j].z); f[3] = __uint_as_float(piece[j].w);
        }
    }
    __device__ __forceinline__ static void store(const View3 &v, int64_t row, int64_t c0, int channels, int64_t t0, int64_t steps, int site,
                                                 int t, int c, const float (&f)[kPer]) {
        io_t *base = static_cast<io_t *>(v.data);
        if (t >= steps || c >= channels) return;
        const int64_t at = row * v.sn + (c0 + c) * v.sc + (t0 + t) * v.st;
        const bool whole = v.access == kTileChannels ? c + kPer <= channels : v.access == kTileSteps && t + kPer <= steps;
        if (whole) {
            if (!SSB_VECTOR_OK(base + at, 16, at + kPer - 1, v.extent, site)) return;
            if constexpr (sizeof(io_t) == 2)
                *reinterpret_cast<uint4 *>(base + at) = make_uint4(pack2<io_t>(f[0], f[1]), pack2<io_t>(f[2], f[3]),
                                                                   pack2<io_t>(f[4], f[5]), pack2<io_t>(f[6], f[7]));
            else
                *reinterpret_cast<float4 *>(base + at) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int dc = v.access == kTileSteps ? 0 : k, dt = v.access == kTileSteps ? k : 0;
                if (c + dc < channels && t + dt < steps) store_one(base, at + dc * v.sc + dt * v.st, v.extent, site, f[k]);
            }
        }
    }
};

// B and C of a tile, as 16-byte pieces: states of a step, or steps of a state.
template <typename io_t, int SP, int THREADS>
struct ProjectionPieces {
    static constexpr int kPer = 16 / (int)sizeof(io_t);
    static constexpr int kEach = kTile * SP / kPer;  // pieces of one of the two
    static constexpr int kPieces = (2 * kEach + THREADS - 1) / THREADS;
    uint4 piece[kPieces];

    __device__ __forceinline__ static bool place(int access, int j, int &which, int &t, int &n) {
        const int i = threadIdx.x + j * THREADS, r = i % kEach;
        which = i / kEach;
        if (access == kProjSteps) {
            n = r % SP;
            t = r / SP * kPer;
        } else {
            n = r % (SP / kPer) * kPer;
            t = r / (SP / kPer);
        }
        return i < 2 * kEach;
    }
    __device__ __forceinline__ void fetch(const ProjView &B, const ProjView &C, int64_t row, int64_t g, int states, int64_t t0, int64_t steps) {
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            int which, t, n;
            piece[j] = make_uint4(0, 0, 0, 0);
            if (!place(B.access, j, which, t, n) || t >= steps || n >= states) continue;
            const ProjView &v = which ? C : B;
            const io_t *base = static_cast<const io_t *>(v.data);
            const int64_t at = row * v.sn + g * v.sg + n * v.ss + (t0 + t) * v.st;
            if (B.access != kProjAny) {
                if (SSB_VECTOR_OK(base + at, 16, at + kPer - 1, v.extent, 260)) piece[j] = *reinterpret_cast<const uint4 *>(base + at);
            } else {
                io_t e[kPer];
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    e[k] = io_t(0.0f);
                    if (n + k < states && SSB_INDEX_OK(at + k * v.ss, v.extent, 260)) e[k] = base[at + k * v.ss];
                }
                memcpy(&piece[j], e, 16);
            }
        }
    }
    // into [2][step][SP] floats
    __device__ __forceinline__ void put(int access, int64_t steps, float *smem) const {
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            int which, t, n;
            if (!place(access, j, which, t, n)) continue;
            float f[kPer];
            if constexpr (sizeof(io_t) == 2) {
                unpack2<io_t>(piece[j].x, f[0], f[1]);
                unpack2<io_t>(piece[j].y, f[2], f[3]);
                unpack2<io_t>(piece[j].z, f[4], f[5]);
                unpack2<io_t>(piece[j].w, f[6], f[7]);
            } else {
                f[0] = __uint_as_float(piece[j].x); f[1] = __uint_as_float(piece[j].y);
                f[2] = __uint_as_float(piece[j].z); f[3] = __uint_as_float(piece[j].w);
            }
            float *to = smem + (which * kTile + t) * SP + n;
            if (access == kProjSteps) {
#pragma unroll
                for (int k = 0; k < kPer; ++k) to[k * SP] = t + k < steps ? f[k] : 0.0f;
            } else {
#pragma unroll
                for (int k = 0; k < kPer; k += 4) *reinterpret_cast<float4 *>(to + k) = make_float4(f[k], f[k + 1], f[k + 2], f[k + 3]);
            }
        }
    }
};

// Sums v[i] of step i over the LN lanes of a channel; lane q of them is left with step q's sum.
template <int LN>
__device__ __forceinline__ float sum_and_spread(float (&v)[LN], int q) {
#pragma unroll
    for (int half = LN / 2; half >= 1; half >>= 1) {
        const bool upper = (q & half) != 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float give = upper ? v[i] : v[i + half], keep = upper ? v[i + half] : v[i];
            v[i] = keep + __shfl_xor_sync(kFullMask, give, half);
        }
    }
    return v[0];
}

template <int LN, int SPL>
struct LaneShape {
    static constexpr int SP = LN * SPL;                  // states, padded
    static constexpr int DL = 32 / LN;                   // channels of a warp
    static constexpr int W = LN >= 16 ? 8 : 4;           // warps
    static constexpr int CB = W * DL;                    // channels of a CTA
    static constexpr int THREADS = W * 32;
};

// Where the pair of step t and channel c lies in a tile of pairs [step][channel].  A thread writes 4 adjacent
// 16-byte units (8 channels) of a step; exchanging units with the step's parity and the thread's number in
// the row lets the 8 lanes of a shared-memory phase meet 8 different banks groups.
template <int CB>
__device__ __forceinline__ int pair_slot(int t, int c) {
    return t * CB + 2 * ((c >> 1) ^ ((c >> 3) & 3) ^ (t & 1)) + (c & 1);
}

template <int LN, int SPL>
__host__ __device__ constexpr size_t selective_lane_smem() {
    using H = LaneShape<LN, SPL>;
    return sizeof(float) * 2 * (size_t)(2 * kTile * H::CB + 2 * kTile * H::SP);  // two tiles of (dt, x) and of B and C
}

// SPL states of the lane's channel at [..., S] floats, zero behind the last.
template <int SPL>
__device__ __forceinline__ void load_lane_states(const float *src, int64_t at, int have, bool vec, int64_t extent, int site, pair_t (&h)[SPL / 2]) {
#pragma unroll
    for (int i = 0; i < SPL; i += 4) {
        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (vec && i < have) {
            if (SSB_VECTOR_OK(src + at + i, 16, at + i + 3, extent, site)) f = *reinterpret_cast<const float4 *>(src + at + i);
        } else {
            if (i + 0 < have) f.x = load_one(src, at + i + 0, extent, site);
            if (i + 1 < have) f.y = load_one(src, at + i + 1, extent, site);
            if (i + 2 < have) f.z = load_one(src, at + i + 2, extent, site);
            if (i + 3 < have) f.w = load_one(src, at + i + 3, extent, site);
        }
        h[i / 2] = make_pair(f.x, f.y);
        h[i / 2 + 1] = make_pair(f.z, f.w);
    }
}
template <int SPL>
__device__ __forceinline__ void store_lane_states(float *dst, int64_t at, int have, bool vec, int64_t extent, int site, const pair_t (&h)[SPL / 2]) {
#pragma unroll
    for (int i = 0; i < SPL; i += 4) {
        const float2 lo = halves(h[i / 2]), hi = halves(h[i / 2 + 1]);
        if (vec && i < have) {
            if (SSB_VECTOR_OK(dst + at + i, 16, at + i + 3, extent, site)) *reinterpret_cast<float4 *>(dst + at + i) = make_float4(lo.x, lo.y, hi.x, hi.y);
        } else {
            if (i + 0 < have) store_one(dst, at + i + 0, extent, site, lo.x);
            if (i + 1 < have) store_one(dst, at + i + 1, extent, site, lo.y);
            if (i + 2 < have) store_one(dst, at + i + 2, extent, site, hi.x);
            if (i + 3 < have) store_one(dst, at + i + 3, extent, site, hi.y);
        }
    }
}

// A[c, n] * log2(e) of the lane's states; an infinite entry becomes the largest finite one: with a step of
// zero it then decays by 2^0 = 1, as padding has to.
template <int SPL>
__device__ __forceinline__ void load_lane_decays(const float *A, int64_t at, int have, bool vec, int64_t extent, int site, pair_t (&d)[SPL / 2]) {
    load_lane_states<SPL>(A, at, have, vec, extent, site, d);
#pragma unroll
    for (int i = 0; i < SPL / 2; ++i) {
        float2 f = halves(d[i]);
        f.x *= kLog2e;
        f.y *= kLog2e;
        if (isinf(f.x)) f.x = copysignf(3.402823466e38f, f.x);
        if (isinf(f.y)) f.y = copysignf(3.402823466e38f, f.y);
        d[i] = make_pair(f.x, f.y);
    }
}

// SPL states of B or C from shared memory.
template <int SPL>
__device__ __forceinline__ void load_lane_projection(const float *smem, pair_t (&v)[SPL / 2]) {
#pragma unroll
    for (int i = 0; i < SPL / 4; ++i) {
        const ulonglong2 f = *reinterpret_cast<const ulonglong2 *>(smem + 4 * i);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

template <typename io_t, int LN, int SPL>
__global__ void __launch_bounds__(LaneShape<LN, SPL>::THREADS) selective_lane_fwd_kernel(const __grid_constant__ SelectiveArgs p) {
    using H = LaneShape<LN, SPL>;
    using Tile = TilePieces<io_t, H::CB, H::THREADS>;
    using Proj = ProjectionPieces<io_t, H::SP, H::THREADS>;
    constexpr int kGroup = LN > 4 ? LN : 4;  // steps worked on together
    extern __shared__ __align__(16) float smem[];
    float2 *const all_steps = reinterpret_cast<float2 *>(smem);  // [2 tiles][step][channel]: (dt, x), then (y, x)
    float *const all_proj = smem + 4 * kTile * H::CB;            // [2 tiles][B, C][step][SP]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int q = lane % LN, cl = warp * H::DL + lane / LN;  // lanes of a channel are neighbours
    const int64_t g = blockIdx.x / p.blocks_per_group, j = blockIdx.x % p.blocks_per_group;
    const int64_t c0 = g * p.per_group + j * H::CB, left_channels = (g + 1) * p.per_group - c0;
    const int channels = left_channels < H::CB ? (int)left_channels : H::CB;
    const bool live = cl < channels;
    const int64_t c = c0 + (live ? cl : 0);
    const int S = (int)p.states, have = live ? (S - q * SPL < SPL ? S - q * SPL : SPL) : 0;  // states of this lane (none: < 1)
    pair_t A[SPL / 2];
    load_lane_decays<SPL>(p.A, c * S + q * SPL, have, p.vec, p.channels * S, 261, A);
    const float D = q == 0 && p.D != nullptr ? load_one(p.D, c, p.channels, 212) : 0.0f;

    for (int64_t s = blockIdx.y; s < p.seq.count; s += gridDim.y) {
        const Span sp = span_of(p.seq, s);
        const int64_t state_at = (s * p.channels + c) * S + q * SPL, state_extent = p.seq.count * p.channels * S;
        pair_t h[SPL / 2] = {};
        if (p.state != nullptr) load_lane_states<SPL>(p.state, state_at, have, p.vec, state_extent, 214, h);
        const int64_t slot0 = p.checkpoints != nullptr ? checkpoint_base(p, s, sp.start) : 0;
        Tile next_x, next_dt, next_z;
        Proj next_proj;
        const auto fetch = [&](int64_t t0) {
            next_x.fetch(p.x, sp.row, c0, channels, sp.start + t0, sp.length - t0, 215);
            next_dt.fetch(p.dt, sp.row, c0, channels, sp.start + t0, sp.length - t0, 216);
            next_proj.fetch(p.B, p.C, sp.row, g, S, sp.start + t0, sp.length - t0);
        };
        if (sp.length > 0) fetch(0);
        int buffer = 0;
        for (int64_t t0 = 0; t0 < sp.length; t0 += kTile, buffer ^= 1) {
            const int64_t left = sp.length - t0;
            float2 *steps = all_steps + buffer * kTile * H::CB;
            float *proj = all_proj + buffer * 2 * kTile * H::SP;
#pragma unroll
            for (int i = 0; i < Tile::kPieces; ++i) {
                int t, cc;
                if (!Tile::place(p.x.access, i, t, cc)) continue;
                float x[Tile::kPer], d[Tile::kPer];
                next_x.open(i, x);
                next_dt.open(i, d);
                if (p.x.access == kTileSteps) {
                    const float ba = p.dt_bias != nullptr && cc < channels ? load_one(p.dt_bias, c0 + cc, p.channels, 213) : 0.0f;
#pragma unroll
                    for (int k = 0; k < Tile::kPer; k += 2) {
                        pair_t w = make_pair(d[k] + ba, d[k + 1] + ba);
                        if (p.softplus) w = softplus2(w);
                        const float2 f = halves(w);
                        // behind the last step: decay 1, no input
                        steps[pair_slot<H::CB>(t + k, cc)] = t + k < left ? make_float2(f.x, x[k]) : make_float2(0.0f, 0.0f);
                        steps[pair_slot<H::CB>(t + k + 1, cc)] = t + k + 1 < left ? make_float2(f.y, x[k + 1]) : make_float2(0.0f, 0.0f);
                    }
                } else {
                    float bias[Tile::kPer];
#pragma unroll
                    for (int k = 0; k < Tile::kPer; ++k)
                        bias[k] = p.dt_bias != nullptr && cc + k < channels ? load_one(p.dt_bias, c0 + cc + k, p.channels, 213) : 0.0f;
#pragma unroll
                    for (int k = 0; k < Tile::kPer; k += 2) {
                        pair_t w = make_pair(d[k] + bias[k], d[k + 1] + bias[k + 1]);
                        if (p.softplus) w = softplus2(w);
                        const float2 f = halves(w);
                        *reinterpret_cast<float4 *>(steps + pair_slot<H::CB>(t, cc + k)) =
                            t < left ? make_float4(f.x, x[k], f.y, x[k + 1]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
                }
            }
            next_proj.put(p.B.access, left, proj);
            __syncthreads();
            if (p.z.data != nullptr) next_z.fetch(p.z, sp.row, c0, channels, sp.start + t0, left, 218);
            if (t0 + kTile < sp.length) fetch(t0 + kTile);
            const int here = left < kTile ? ((int)left + kGroup - 1) / kGroup * kGroup : kTile;
#pragma unroll 1
            for (int t = 0; t < here; t += kGroup) {
                if (p.checkpoints != nullptr && ((t0 + t) & ((1ll << p.tile_log2) - 1)) == 0)
                    store_lane_states<SPL>(p.checkpoints, ((slot0 + ((t0 + t) >> p.tile_log2)) * p.channels + c) * S + q * SPL, have, p.vec,
                                           p.checkpoint_slots * S * p.channels, 217, h);
                float y[kGroup];
#pragma unroll
                for (int i = 0; i < kGroup; ++i) {
                    const float2 dx = steps[pair_slot<H::CB>(t + i, cl)];
                    pair_t b[SPL / 2], r[SPL / 2], sum = 0;
                    load_lane_projection<SPL>(proj + (t + i) * H::SP + q * SPL, b);
                    load_lane_projection<SPL>(proj + (kTile + t + i) * H::SP + q * SPL, r);
                    const pair_t dt2 = both(dx.x), u2 = both(dx.x * dx.y);
#pragma unroll
                    for (int k = 0; k < SPL / 2; ++k) {
                        h[k] = fma2(exp2_pair(mul2(dt2, A[k])), h[k], mul2(u2, b[k]));
                        sum = fma2(h[k], r[k], sum);
                    }
                    const float2 f = halves(sum);
                    y[i] = fmaf(D, dx.y, f.x + f.y);
                }
                __syncwarp();  // the lanes of a channel have read the steps that are replaced
                if constexpr (LN <= 4) {
#pragma unroll
                    for (int i = 0; i < kGroup; i += LN) {
                        float v[LN];
#pragma unroll
                        for (int k = 0; k < LN; ++k) v[k] = y[i + k];
                        steps[pair_slot<H::CB>(t + i + q, cl)].x = sum_and_spread<LN>(v, q);
                    }
                } else {
                    steps[pair_slot<H::CB>(t + q, cl)].x = sum_and_spread<LN>(y, q);
                }
            }
            __syncthreads();
            // gate and store
#pragma unroll
            for (int i = 0; i < Tile::kPieces; ++i) {
                int t, cc;
                if (!Tile::place(p.out.access, i, t, cc)) continue;
                float f[Tile::kPer], z[Tile::kPer];
#pragma unroll
                for (int k = 0; k < Tile::kPer; k += 2) {
                    if (p.out.access == kTileSteps) {
                        f[k] = steps[pair_slot<H::CB>(t + k, cc)].x;
                        f[k + 1] = steps[pair_slot<H::CB>(t + k + 1, cc)].x;
                    } else {
                        const float4 w = *reinterpret_cast<const float4 *>(steps + pair_slot<H::CB>(t, cc + k));
                        f[k] = w.x;
                        f[k + 1] = w.z;
                    }
                }
                if (p.z.data != nullptr) {
                    next_z.open(i, z);
#pragma unroll
                    for (int k = 0; k < Tile::kPer; ++k) f[k] *= z[k] * logistic(z[k]);
                }
                Tile::store(p.out, sp.row, c0, channels, sp.start + t0, left, 219, t, cc, f);
            }
        }
        if (p.state_out != nullptr) store_lane_states<SPL>(p.state_out, state_at, have, p.vec, state_extent, 220, h);
        zero_uncovered<io_t>(p.seq, s, sp, p.out, c0, c0 + channels, 219);
        __syncthreads();  // the last tile is no longer read
    }
}

}  // namespace ssb
