// Selective scan over whole sequences, forward: per channel c and state n
//     h_t = exp(dt_t A[c,n]) h_{t-1} + dt_t x_t B_t[n],     y_t = sum_n C_t[n] h_t + D x_t,     out = y silu(z).
//
// The floor: one exponential per (step, channel, state).  At 16 a clock and SM they take three times as long as the
// tensors' bytes in 16-bit storage, so the states stay in registers (but for the checkpoints of a training call).
// What bounds it: everything else takes 9.9 instructions an exponential with 8 states a lane, 12.6 with 4 and 13.5
// where checkpoints are written, in all warps together; and with few channels a warp waits out each step alone.
//
// LN lanes share a channel, each with SPL of its states (4; 8 where warps abound, and beyond 128 states); a warp
// holds 32 / LN channels and walks the steps in order.  Per step and 4 states a lane issues 4 exponentials,
// 8 packed operations (exponent, input, recurrence, read-out, two states each) and 3 shared loads.
// The read-out is summed over the LN lanes for groups of steps, so that each lane is left with the sum
// of one step (LN = 4: 3 shuffles for 4 steps).  Half of the CTA's warps scan; the other half put tiles of 32
// steps into shared memory, (dt, x) after the softplus, B and C as fp32, and fetch the next tile's bytes meanwhile.  The
// sums take the place of the steps in shared memory, from where those warps send them, gated: 16 bytes at a time where
// all operands allow it.
//
// Measured, bf16, 16 states: 13 packed prompts in [1, 4096, 4096] 136 us with 8 states a lane (169 with 4); [4, 2048, 2048]
// 183 us; [1, 2048, 8192] 505 us, where a scheduler has one scanning warp and a step's latency (121 cycles at 1.965 GHz) counts.
// The exponentials alone are 58 us in each.
#pragma once

#include "ssm_scan.cuh"

namespace ssb {

constexpr int kTile = 32;  // steps of a tile

// 16-byte pieces of a tile of a [N, C, T] view: 8 (4) adjacent channels of a step, or adjacent steps of a channel.
enum TileAccess : int { kTileAny = 0, kTileChannels = 1, kTileSteps = 2 };

// Which pieces of a tile a thread handles: always the same channels, steps `next` apart.
template <typename io_t, int CB, int THREADS>
struct TileShare {
    static constexpr int kPer = 16 / (int)sizeof(io_t);
    static constexpr int kPieces = (kTile * CB / kPer + THREADS - 1) / THREADS;
    static_assert(CB % kPer == 0 && THREADS % CB == 0, "whole pieces of channels");
    bool by_step, whole, works;  // whole: one 16-byte access; works: not a thread too many
    int t, c, next, channels;    // first step, first channel, steps between pieces, channels of the CTA

    __device__ __forceinline__ TileShare(int access, int tid, int channels_) : channels(channels_) {
        by_step = access == kTileSteps;
        c = by_step ? tid % CB : tid % (CB / kPer) * kPer;
        t = by_step ? tid / CB * kPer : tid / (CB / kPer);
        next = by_step ? THREADS / CB * kPer : THREADS / (CB / kPer);
        works = t < kTile && c < channels;
        whole = access == kTileChannels ? c + kPer <= channels : by_step;
    }
    // the address of the thread's first piece in the tile that starts at step t0
    __device__ __forceinline__ int64_t offset(const View3 &v, int64_t row, int64_t c0, int64_t t0) const {
        return row * v.sn + (c0 + c) * v.sc + (t0 + t) * v.st;
    }
    // pieces of the tile at `at`, zero behind `left` steps; the elements of a piece along the steps that lie behind
    // are whatever memory holds
    __device__ __forceinline__ void fetch(const View3 &v, int64_t at, int left, int site, uint4 (&piece)[kPieces]) const {
        const io_t *base = static_cast<const io_t *>(v.data);
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            piece[j] = make_uint4(0, 0, 0, 0);
            if (works && t + j * next < left) {
                const int64_t i = at + j * next * v.st;
                if (whole) {
                    if (SSB_VECTOR_OK(base + i, 16, i + kPer - 1, v.extent, site)) piece[j] = *reinterpret_cast<const uint4 *>(base + i);
                } else {
                    io_t e[kPer];
#pragma unroll
                    for (int k = 0; k < kPer; ++k) {
                        e[k] = io_t(0.0f);
                        if (c + k < channels && SSB_INDEX_OK(i + k * v.sc, v.extent, site)) e[k] = base[i + k * v.sc];
                    }
                    memcpy(&piece[j], e, 16);
                }
            }
        }
    }
    __device__ __forceinline__ static void open(const uint4 &piece, float (&f)[kPer]) {
        if constexpr (sizeof(io_t) == 2) {
            unpack2<io_t>(piece.x, f[0], f[1]);
            unpack2<io_t>(piece.y, f[2], f[3]);
            unpack2<io_t>(piece.z, f[4], f[5]);
            unpack2<io_t>(piece.w, f[6], f[7]);
        } else {
            f[0] = __uint_as_float(piece.x); f[1] = __uint_as_float(piece.y);
            f[2] = __uint_as_float(piece.z); f[3] = __uint_as_float(piece.w);
        }
    }
    __device__ __forceinline__ void store(const View3 &v, int64_t at, int j, int left, int site, const float (&f)[kPer]) const {
        io_t *base = static_cast<io_t *>(v.data);
        const int64_t i = at + j * next * v.st;
        const int here = t + j * next;
        if (!works || here >= left) return;
        if (whole && (!by_step || here + kPer <= left)) {
            if (!SSB_VECTOR_OK(base + i, 16, i + kPer - 1, v.extent, site)) return;
            if constexpr (sizeof(io_t) == 2)
                *reinterpret_cast<uint4 *>(base + i) = make_uint4(pack2<io_t>(f[0], f[1]), pack2<io_t>(f[2], f[3]),
                                                                  pack2<io_t>(f[4], f[5]), pack2<io_t>(f[6], f[7]));
            else
                *reinterpret_cast<float4 *>(base + i) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                if (by_step ? here + k < left : c + k < channels) store_one(base, i + k * (by_step ? v.st : v.sc), v.extent, site, f[k]);
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

    __device__ __forceinline__ static bool place(int access, int tid, int j, int &which, int &t, int &n) {
        const int i = tid + j * THREADS, r = i % kEach;
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
    __device__ __forceinline__ void fetch(int tid, const ProjView &B, const ProjView &C, int64_t row, int64_t g, int states, int64_t t0, int64_t steps) {
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            int which, t, n;
            piece[j] = make_uint4(0, 0, 0, 0);
            if (!place(B.access, tid, j, which, t, n) || t >= steps || n >= states) continue;
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
    __device__ __forceinline__ void put(int tid, int access, int64_t steps, float *smem) const {
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            int which, t, n;
            if (!place(access, tid, j, which, t, n)) continue;
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

template <int LN, int SPL, int WARPS>
struct LaneShape {
    static constexpr int SP = LN * SPL;                  // states, padded
    static constexpr int DL = 32 / LN;                   // channels of a warp
    static constexpr int W = WARPS;                      // warps that scan, and as many that move tiles
    static constexpr int CB = W * DL;                    // channels of a CTA
    static constexpr int THREADS = W * 32;               // of either kind
};

// Where the pair of step t and channel c lies in a tile of pairs [step][channel].  A thread writes 4 adjacent
// 16-byte units (8 channels) of a step; exchanging units with the step's parity and the thread's number in
// the row lets the 8 lanes of a shared-memory phase meet 8 different banks groups.
template <int CB>
__device__ __forceinline__ int pair_slot(int t, int c) {
    return t * CB + 2 * ((c >> 1) ^ ((c >> 3) & 3) ^ (t & 1)) + (c & 1);
}

template <int LN, int SPL, int WARPS>
__host__ __device__ constexpr size_t selective_lane_smem() {
    using H = LaneShape<LN, SPL, WARPS>;
    return sizeof(float) * (size_t)(3 * 2 * kTile * H::CB + 2 * 2 * kTile * H::SP);  // three tiles of (dt, x), two of B and C
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

// One group of steps in registers: what a lane needs of them.
template <int STEPS, int SPL>
struct StepGroup {
    float2 dx[STEPS];
    pair_t b[STEPS][SPL / 2], r[STEPS][SPL / 2];
};

template <typename io_t, int LN, int SPL, int WARPS>
__global__ void __launch_bounds__(2 * WARPS * 32, 8 / WARPS) selective_lane_fwd_kernel(const __grid_constant__ SelectiveArgs p) {
    using H = LaneShape<LN, SPL, WARPS>;
    using Share = TileShare<io_t, H::CB, H::THREADS>;
    using Proj = ProjectionPieces<io_t, H::SP, H::THREADS>;
    constexpr int kGroup = 8;                      // steps whose sums are exchanged together
    constexpr int kAhead = SPL > 4 ? 2 : 4;        // steps loaded together, one such part ahead of their use
    extern __shared__ __align__(16) float smem[];
    float2 *const all_steps = reinterpret_cast<float2 *>(smem);  // [3 tiles][step][channel]: (dt, x), then (y, x)
    float *const all_proj = smem + 3 * 2 * kTile * H::CB;        // [2 tiles][B, C][step][SP]
    const bool scans = threadIdx.x < H::THREADS;
    const int tid = scans ? threadIdx.x : threadIdx.x - H::THREADS;
    const int64_t g = blockIdx.x / p.blocks_per_group, j = blockIdx.x % p.blocks_per_group;
    const int64_t c0 = g * p.per_group + j * H::CB, left_channels = (g + 1) * p.per_group - c0;
    const int channels = left_channels < H::CB ? (int)left_channels : H::CB;
    const int S = (int)p.states;

    if (!scans) {
        // ---- moves tiles: at phase k it puts down tile k + 1, fetches tile k + 2, and sends off tile k - 1
        const Share share(p.x.access, tid, channels);
        const int slot0 = pair_slot<H::CB>(0, share.c);  // of an even step
        float bias[Share::kPer];
#pragma unroll
        for (int e = 0; e < Share::kPer; ++e) {
            const int ch = share.by_step ? share.c : share.c + e;
            bias[e] = p.dt_bias != nullptr && ch < channels ? load_one(p.dt_bias, c0 + ch, p.channels, 213) : 0.0f;
        }
        for (int64_t s = blockIdx.y; s < p.seq.count; s += gridDim.y) {
            const Span sp = span_of(p.seq, s);
            const int64_t tiles = (sp.length + kTile - 1) / kTile;
            const auto left_at = [&](int64_t k) { return (int)(sp.length - k * kTile < kTile ? sp.length - k * kTile : kTile); };
            int64_t at_x = share.offset(p.x, sp.row, c0, sp.start), at_dt = share.offset(p.dt, sp.row, c0, sp.start);
            int64_t at_z = share.offset(p.z, sp.row, c0, sp.start), at_out = share.offset(p.out, sp.row, c0, sp.start);
            uint4 next_x[Share::kPieces], next_dt[Share::kPieces], next_z[Share::kPieces];
            Proj next_proj;
            const auto fetch = [&](int64_t k) {
                if (k >= tiles) return;
                share.fetch(p.x, at_x, left_at(k), 215, next_x);
                share.fetch(p.dt, at_dt, left_at(k), 216, next_dt);
                next_proj.fetch(tid, p.B, p.C, sp.row, g, S, sp.start + k * kTile, left_at(k));
                at_x += kTile * p.x.st;
                at_dt += kTile * p.dt.st;
            };
            fetch(0);
            int put_at = 0, send_at = 1;  // tiles k + 1 and k - 1 modulo 3
            for (int64_t k = -1; k <= tiles; ++k) {
                if (k + 1 < tiles) {
                    const int left = left_at(k + 1);
                    float2 *steps = all_steps + put_at * kTile * H::CB;
#pragma unroll
                    for (int i = 0; i < Share::kPieces; ++i) {
                        const int t = share.t + i * share.next;
                        float x[Share::kPer], d[Share::kPer];
                        Share::open(next_x[i], x);
                        Share::open(next_dt[i], d);
#pragma unroll
                        for (int e = 0; e < Share::kPer; ++e) {
                            d[e] += bias[e];
                            if (p.softplus) d[e] = softplus(d[e]);
                            if ((share.by_step ? t + e : t) >= left) d[e] = x[e] = 0.0f;  // behind the last step: decay 1, no input
                        }
                        if (share.t >= kTile) continue;
                        if (share.by_step) {
#pragma unroll
                            for (int e = 0; e < Share::kPer; ++e) steps[pair_slot<H::CB>(t + e, share.c)] = make_float2(d[e], x[e]);
                        } else {
                            // 8 adjacent channels are 4 units of 16 bytes whose order the step's parity turns
                            float2 *to = steps + t * H::CB;
#pragma unroll
                            for (int e = 0; e < Share::kPer; e += 2)
                                *reinterpret_cast<float4 *>(to + ((slot0 ^ e) ^ (2 * (t & 1)))) = make_float4(d[e], x[e], d[e + 1], x[e + 1]);
                        }
                    }
                    next_proj.put(tid, p.B.access, left, all_proj + ((k + 1) & 1) * 2 * kTile * H::SP);
                    fetch(k + 2);
                }
                if (k >= 1) {
                    const float2 *steps = all_steps + send_at * kTile * H::CB;
#pragma unroll
                    for (int i = 0; i < Share::kPieces; ++i) {
                        const int t = share.t + i * share.next;
                        if (share.t >= kTile) continue;
                        float f[Share::kPer], z[Share::kPer];
                        if (share.by_step) {
#pragma unroll
                            for (int e = 0; e < Share::kPer; ++e) f[e] = steps[pair_slot<H::CB>(t + e, share.c)].x;
                        } else {
                            const float2 *from = steps + t * H::CB;
#pragma unroll
                            for (int e = 0; e < Share::kPer; e += 2) {
                                const float4 w = *reinterpret_cast<const float4 *>(from + ((slot0 ^ e) ^ (2 * (t & 1))));
                                f[e] = w.x;
                                f[e + 1] = w.z;
                            }
                        }
                        if (p.z.data != nullptr) {
                            Share::open(next_z[i], z);
#pragma unroll
                            for (int e = 0; e < Share::kPer; ++e) f[e] *= z[e] * logistic(z[e]);
                        }
                        share.store(p.out, at_out, i, left_at(k - 1), 219, f);
                    }
                    at_out += kTile * p.out.st;
                }
                if (p.z.data != nullptr && k >= 0 && k < tiles) {
                    share.fetch(p.z, at_z, left_at(k), 218, next_z);
                    at_z += kTile * p.z.st;
                }
                put_at = put_at == 2 ? 0 : put_at + 1;
                send_at = send_at == 2 ? 0 : send_at + 1;
                __syncthreads();
            }
        }
    } else {
        // ---- scans: at phase k tile k
        const int lane = tid & 31, warp = tid >> 5;
        const int q = lane % LN, cl = warp * H::DL + lane / LN;  // lanes of a channel are neighbours
        const bool live = cl < channels;
        const int64_t c = c0 + (live ? cl : 0);
        const int have = live ? (S - q * SPL < SPL ? S - q * SPL : SPL) : 0;  // states of this lane (none: < 1)
        pair_t A[SPL / 2];
        load_lane_decays<SPL>(p.A, c * S + q * SPL, have, p.vec, p.channels * S, 261, A);
        const float D = q == 0 && p.D != nullptr ? load_one(p.D, c, p.channels, 212) : 0.0f;
        for (int64_t s = blockIdx.y; s < p.seq.count; s += gridDim.y) {
            const Span sp = span_of(p.seq, s);
            const int64_t tiles = (sp.length + kTile - 1) / kTile;
            const int64_t state_at = (s * p.channels + c) * S + q * SPL, state_extent = p.seq.count * p.channels * S;
            pair_t h[SPL / 2] = {};
            if (p.state != nullptr) load_lane_states<SPL>(p.state, state_at, have, p.vec, state_extent, 214, h);
            const int64_t slot0 = p.checkpoints != nullptr ? checkpoint_base(p, s, sp.start) : 0;
            int at = 0;  // tile k modulo 3
            __syncthreads();  // phase -1
            for (int64_t k = 0; k <= tiles; ++k) {
                if (k < tiles) {
                    float2 *steps = all_steps + at * kTile * H::CB;
                    const float *proj = all_proj + (k & 1) * 2 * kTile * H::SP + q * SPL;
                    const auto load = [&](int t, StepGroup<kAhead, SPL> &w) {
#pragma unroll
                        for (int i = 0; i < kAhead; ++i) {
                            w.dx[i] = steps[pair_slot<H::CB>(t + i, cl)];
                            load_lane_projection<SPL>(proj + (t + i) * H::SP, w.b[i]);
                            load_lane_projection<SPL>(proj + (kTile + t + i) * H::SP, w.r[i]);
                        }
                    };
                    // Sums of the group before are exchanged while the next group is worked on; their place is that of
                    // steps which all lanes of the channel have loaded.
                    const auto exchange = [&](int t, float (&y)[kGroup]) {
                        constexpr int kSpread = LN < kGroup ? LN : kGroup;
#pragma unroll
                        for (int i = 0; i < kGroup; i += kSpread) {
                            float v[kSpread];
#pragma unroll
                            for (int e = 0; e < kSpread; ++e) v[e] = y[i + e];
                            const float sum = sum_and_spread<LN>(v, q);
                            if (q < kSpread) steps[pair_slot<H::CB>(t + i + q, cl)].x = sum;
                        }
                    };
                    const int64_t left = sp.length - k * kTile;
                    const int here = left < kTile ? ((int)left + kGroup - 1) / kGroup * kGroup : kTile;
                    StepGroup<kAhead, SPL> part[2];
                    float y[kGroup], y_before[kGroup];
                    load(0, part[0]);
#pragma unroll 1
                    for (int t = 0; t < here; t += kGroup) {
                        if (p.checkpoints != nullptr && ((k * kTile + t) & ((1ll << p.tile_log2) - 1)) == 0)
                            store_lane_states<SPL>(p.checkpoints, ((slot0 + ((k * kTile + t) >> p.tile_log2)) * p.channels + c) * S + q * SPL, have,
                                                   p.vec, p.checkpoint_slots * S * p.channels, 217, h);
#pragma unroll
                        for (int i0 = 0; i0 < kGroup; i0 += kAhead) {
                            const StepGroup<kAhead, SPL> &now = part[i0 / kAhead & 1];
                            // the last part of a tile loads the first steps of no tile: any, and does not use them
                            load((t + i0 + kAhead) & (kTile - 1), part[(i0 / kAhead + 1) & 1]);
#pragma unroll
                            for (int i = 0; i < kAhead; ++i) {
                                pair_t sum;
                                const pair_t dt2 = both(now.dx[i].x), u2 = both(now.dx[i].x * now.dx[i].y);
#pragma unroll
                                for (int e = 0; e < SPL / 2; ++e) {
                                    h[e] = fma2(exp2_pair(fma2(dt2, A[e], both(kExponentShift))), h[e], mul2(u2, now.b[i][e]));
                                    sum = e == 0 ? mul2(h[e], now.r[i][e]) : fma2(h[e], now.r[i][e], sum);
                                }
                                const float2 f = halves(sum);
                                y[i0 + i] = fmaf(D, now.dx[i].y, f.x + f.y);
                            }
                        }
                        if (t > 0) exchange(t - kGroup, y_before);
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < kGroup; ++i) y_before[i] = y[i];
                    }
                    exchange(here - kGroup, y_before);
                }
                at = at == 2 ? 0 : at + 1;
                __syncthreads();
            }
            if (p.state_out != nullptr) store_lane_states<SPL>(p.state_out, state_at, have, p.vec, state_extent, 220, h);
        }
    }
    for (int64_t s = blockIdx.y; s < p.seq.count; s += gridDim.y)
        zero_uncovered<io_t>(p.seq, s, span_of(p.seq, s), p.out, c0, c0 + channels, 219);
}

}  // namespace ssb
