// Backward of the selective scan for up to 32 states, laid out as the forward is (ssm_forward.cuh): LN lanes
// share a channel, each with 4 of its states; half of a CTA's warps scan, half move tiles.
//
// Tiles of 32 steps run from the last to the first.  With the adjoint r_t = a_t (gy_t C_t + r_{t+1}) the lane
// needs the states in the opposite order.  The forward has written the state every 16 steps; from there a first
// pass finds the states at steps 4, 8 and 12 (three quarters of an exponential per state and step), and each
// run of 4 steps is then done forwards, which leaves a_t and a_t h_{t-1} in registers, and backwards.
//
// Per (step, channel, state): 1.75 exponentials, 13 fp32 operations, and the sums.  The gradients of x, dt and
// the gate sum over a channel's states: over the LN lanes, as the forward's read-out.  Those of B and C sum over
// channels: over the warp's in an exchange that halves the values at each step (8 values over 8 channels: 7
// shuffles), then over the warps in shared memory, where each has rows of its own, and over CTAs by
// selective_reduce_kernel.  All in a fixed order.  Shuffles and shared loads bound it:
// [4, 2048, 2048], 16 states, bf16, 468 us: 33 instructions a (step, channel, state) in 56 % of the issue slots, the shared-memory
// pipe taken 48 % of the time by loads and stores alone, with the shuffles on top.
#pragma once

#include "ssm_forward.cuh"

namespace ssb {

constexpr int kCheckpointSteps = 16;

// Registers of a thread at launch, and after the two kinds of warps have parted (one warpgroup of 4 warps each):
// what the ones give up the others take, so the sum never exceeds the launch's.
constexpr int kLaunchRegisters = 128, kScanRegisters = 152, kMoveRegisters = 104;
static_assert(kScanRegisters + kMoveRegisters <= 2 * kLaunchRegisters, "a block's registers are what it was launched with");
template <int N>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <typename io_t, int LN, int WARPS>
__host__ __device__ constexpr size_t selective_lane_bwd_smem() {
    using H = LaneShape<LN, 4, WARPS>;
    using Share = TileShare<io_t, H::CB, H::THREADS>;
    // two tiles of (dt, x) and gy, of B and C, of every warp's sums for the gradients of B and C, and of what the
    // threads that move tiles keep for themselves: x, gout and z as they came, dt and its slope; dt_bias and D
    return sizeof(float) * (size_t)(2 * 3 * kTile * H::CB + 2 * 2 * kTile * H::SP + 2 * WARPS * kTile * 2 * H::SP) +
           2 * (size_t)(3 + 8 / (int)sizeof(io_t)) * Share::kPieces * H::THREADS * 16 + 2 * H::CB * sizeof(float);
}

// Sums v over the DL channels of a warp (r: the lane's channel among them); the lane is left with the
// 8 / DL values (1 for DL >= 8) that start at the returned index.
template <int DL, int LN>
__device__ __forceinline__ int sum_over_channels(float (&v)[8], int r) {
    constexpr int kStages = DL < 8 ? DL : 8;
    int at = 0;
    int held = 8;
#pragma unroll
    for (int bit = kStages / 2; bit >= 1; bit >>= 1) {
        held >>= 1;
        const bool upper = (r & bit) != 0;
        if (upper) at += held;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i < held) {
                const float give = upper ? v[i] : v[i + held], keep = upper ? v[i + held] : v[i];
                v[i] = keep + __shfl_xor_sync(kFullMask, give, bit * LN);
            }
        }
    }
#pragma unroll
    for (int d = 8; d < DL; d <<= 1) v[0] += __shfl_xor_sync(kFullMask, v[0], d * LN);
    return at;
}

template <typename io_t, int LN, int WARPS>
__global__ void __launch_bounds__(2 * WARPS * 32, 8 / WARPS) selective_lane_bwd_kernel(const __grid_constant__ SelectiveArgs p,
                                                                                      const __grid_constant__ SelectiveGradArgs q) {
    constexpr int SPL = 4;
    using H = LaneShape<LN, SPL, WARPS>;
    using Share = TileShare<io_t, H::CB, H::THREADS>;
    using Proj = ProjectionPieces<io_t, H::SP, H::THREADS>;
    constexpr int kPer = Share::kPer;
    extern __shared__ __align__(16) float smem[];
    float2 *const all_steps = reinterpret_cast<float2 *>(smem);   // [2 tiles][step][channel]: (dt, x), then (sum dh B, sum dh a h A)
    float *const all_gy = smem + 2 * 2 * kTile * H::CB;           // [2 tiles][step][channel]: gy, then y
    float *const all_proj = all_gy + 2 * kTile * H::CB;           // [2 tiles][B, C][step][SP]
    float *const all_sums = all_proj + 2 * 2 * kTile * H::SP;     // [2 tiles][warp][step][B, C][SP]
    uint4 *const all_kept = reinterpret_cast<uint4 *>(all_sums + 2 * WARPS * kTile * 2 * H::SP);  // [2 tiles][what][thread's pieces]
    constexpr int kKept = 3 + 8 / (int)sizeof(io_t);  // 16-byte words a piece: x, gout, z, then dt and its slope as fp32
    float *const biases = reinterpret_cast<float *>(all_kept + 2 * kKept * Share::kPieces * H::THREADS), *const Ds = biases + H::CB;  // [channel]
    const bool scans = threadIdx.x < H::THREADS;
    const int tid = scans ? threadIdx.x : threadIdx.x - H::THREADS;
    const int64_t g = blockIdx.x / p.blocks_per_group, j = blockIdx.x % p.blocks_per_group;
    const int64_t c0 = g * p.per_group + j * H::CB, left_channels = (g + 1) * p.per_group - c0;
    const int channels = left_channels < H::CB ? (int)left_channels : H::CB;
    const int S = (int)p.states;
    if (threadIdx.x < H::CB) {
        const int ch = threadIdx.x;
        biases[ch] = p.dt_bias != nullptr && ch < channels ? load_one(p.dt_bias, c0 + ch, p.channels, 231) : 0.0f;
        Ds[ch] = p.D != nullptr && ch < channels ? load_one(p.D, c0 + ch, p.channels, 230) : 0.0f;
    }
    __syncthreads();

    if (!scans) {
        registers_down<kMoveRegisters>();
        const Share share(p.x.access, tid, channels);
        const int slot0 = pair_slot<H::CB>(0, share.c);
        float gD[kPer], gbias[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) gD[e] = gbias[e] = 0.0f;
        // a channel's value for every element of a piece
        const auto of_channels = [&](const float *from, float (&f)[kPer]) {
            if (share.by_step) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) f[e] = from[share.c];
            } else {
#pragma unroll
                for (int e = 0; e < kPer; e += 4) {
                    const float4 w = *reinterpret_cast<const float4 *>(from + share.c + e);
                    f[e] = w.x; f[e + 1] = w.y; f[e + 2] = w.z; f[e + 3] = w.w;
                }
            }
        };
        const bool gated = p.z.data != nullptr;
        for (int64_t s = blockIdx.y; s < p.seq.count; s += gridDim.y) {
            const Span sp = span_of(p.seq, s);
            const int64_t tiles = (sp.length + kTile - 1) / kTile;
            const auto left_at = [&](int64_t k) { return (int)(sp.length - k * kTile < kTile ? sp.length - k * kTile : kTile); };
            const int64_t at_x = share.offset(p.x, sp.row, c0, sp.start), at_dt = share.offset(p.dt, sp.row, c0, sp.start);
            const int64_t at_z = share.offset(p.z, sp.row, c0, sp.start), at_g = share.offset(q.gout, sp.row, c0, sp.start);
            const int64_t to_x = share.offset(q.gx, sp.row, c0, sp.start), to_dt = share.offset(q.gdt, sp.row, c0, sp.start);
            const int64_t to_z = share.offset(q.gz, sp.row, c0, sp.start);
            uint4 raw_x[Share::kPieces], raw_dt[Share::kPieces], raw_z[Share::kPieces], raw_g[Share::kPieces];
            Proj next_proj;
            const auto fetch = [&](int64_t k) {  // tile k
                if (k < 0) return;
                share.fetch(p.x, at_x + k * kTile * p.x.st, left_at(k), 235, raw_x);
                share.fetch(p.dt, at_dt + k * kTile * p.dt.st, left_at(k), 236, raw_dt);
                share.fetch(q.gout, at_g + k * kTile * q.gout.st, left_at(k), 233, raw_g);
                if (gated) share.fetch(p.z, at_z + k * kTile * p.z.st, left_at(k), 234, raw_z);
                next_proj.fetch(tid, p.B, p.C, sp.row, g, S, sp.start + k * kTile, left_at(k));
            };
            fetch(tiles - 1);
            // A phase first sends off tile ph - 1 and then puts tile ph + 1 into the same buffers: a thread's pieces of
            // both lie at the same places, which no other of these threads touches.
            for (int64_t phase = -1; phase <= tiles; ++phase) {
                const int64_t put = tiles - 2 - phase, send = tiles - phase;  // the tiles put down and sent off now
                const int buffer = (int)((phase + 1) & 1);
                float2 *steps = all_steps + buffer * kTile * H::CB;
                float *gys = all_gy + buffer * kTile * H::CB;
                uint4 *kept = all_kept + buffer * kKept * Share::kPieces * H::THREADS + tid;
                if (send >= 0 && send < tiles) {
                    const int left = left_at(send);
                    // the warps' sums for B and C
                    const float *sums = all_sums + buffer * WARPS * kTile * 2 * H::SP;
                    const int64_t extent = (int64_t)p.blocks_per_group * q.rows * p.seq.steps * p.groups * S;
                    const int64_t base = (((j * q.rows + sp.row) * p.seq.steps + sp.start + send * kTile) * p.groups + g) * S;
                    for (int i = 4 * tid; i < left * 2 * H::SP; i += 4 * H::THREADS) {
                        const int n = i % H::SP, which = i / H::SP & 1, t = i / (2 * H::SP);
                        float4 v = *reinterpret_cast<const float4 *>(sums + i);
#pragma unroll
                        for (int w = 1; w < WARPS; ++w) {
                            const float4 f = *reinterpret_cast<const float4 *>(sums + w * kTile * 2 * H::SP + i);
                            v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
                        }
                        float *to = which ? q.part_C : q.part_B;
                        const int64_t at = base + (int64_t)t * p.groups * S + n;
                        if (p.vec && n < S) {
                            if (SSB_VECTOR_OK(to + at, 16, at + 3, extent, 238 + which)) *reinterpret_cast<float4 *>(to + at) = v;
                        } else {
                            if (n + 0 < S) store_one(to, at + 0, extent, 238 + which, v.x);
                            if (n + 1 < S) store_one(to, at + 1, extent, 238 + which, v.y);
                            if (n + 2 < S) store_one(to, at + 2, extent, 238 + which, v.z);
                            if (n + 3 < S) store_one(to, at + 3, extent, 238 + which, v.w);
                        }
                    }
                    // the gradients of x, dt and z
#pragma unroll
                    for (int i = 0; i < Share::kPieces; ++i) {
                        const int t = share.t + i * share.next;
                        if (share.t >= kTile) continue;
                        float x[kPer], gy[kPer], z[kPer], through[kPer], bydecay[kPer], y[kPer];
                        if (share.by_step) {
#pragma unroll
                            for (int e = 0; e < kPer; ++e) {
                                const float2 w = steps[pair_slot<H::CB>(t + e, share.c)];
                                through[e] = w.x;
                                bydecay[e] = w.y;
                                y[e] = gys[(t + e) * H::CB + share.c];
                            }
                        } else {
                            const float2 *from = steps + t * H::CB;
#pragma unroll
                            for (int e = 0; e < kPer; e += 2) {
                                const float4 w = *reinterpret_cast<const float4 *>(from + ((slot0 ^ e) ^ (2 * (t & 1))));
                                through[e] = w.x; bydecay[e] = w.y;
                                through[e + 1] = w.z; bydecay[e + 1] = w.w;
                            }
#pragma unroll
                            for (int e = 0; e < kPer; e += 4) {
                                const float4 w = *reinterpret_cast<const float4 *>(gys + t * H::CB + share.c + e);
                                y[e] = w.x; y[e + 1] = w.y; y[e + 2] = w.z; y[e + 3] = w.w;
                            }
                        }
                        const uint4 *mine = kept + i * kKept * H::THREADS;
                        float D[kPer];
                        of_channels(Ds, D);
                        Share::open(mine[0], x);
                        Share::open(mine[H::THREADS], gy);
                        if (gated) {
                            Share::open(mine[2 * H::THREADS], z);
#pragma unroll
                            for (int e = 0; e < kPer; ++e) {
                                const float sg = logistic(z[e]), out = gy[e];
                                gy[e] = out * z[e] * sg;
                                z[e] = out * fmaf(D[e], x[e], y[e]) * sg * fmaf(z[e], 1.0f - sg, 1.0f);
                            }
                            share.store(q.gz, to_z + send * kTile * q.gz.st, i, left, 242, z);
                        }
                        float gdt[kPer];
#pragma unroll
                        for (int e = 0; e < kPer; e += 2) {  // (dt, slope) of two elements
                            const uint4 w = mine[(3 + e / 2) * H::THREADS];
                            const float dt[2] = {__uint_as_float(w.x), __uint_as_float(w.z)}, slope[2] = {__uint_as_float(w.y), __uint_as_float(w.w)};
#pragma unroll
                            for (int f = 0; f < 2; ++f) {
                                const bool inside = (share.by_step ? t + e + f : t) < left;
                                gdt[e + f] = fmaf(through[e + f], x[e + f], bydecay[e + f] * kLn2) * slope[f];
                                if (inside) {
                                    gD[e + f] = fmaf(gy[e + f], x[e + f], gD[e + f]);
                                    gbias[e + f] += gdt[e + f];
                                }
                                x[e + f] = fmaf(through[e + f], dt[f], D[e + f] * gy[e + f]);
                            }
                        }
                        share.store(q.gx, to_x + send * kTile * q.gx.st, i, left, 240, x);
                        share.store(q.gdt, to_dt + send * kTile * q.gdt.st, i, left, 241, gdt);
                    }
                }
                if (put >= 0) {
                    const int left = left_at(put);
#pragma unroll
                    for (int i = 0; i < Share::kPieces; ++i) {
                        const int t = share.t + i * share.next;
                        float x[kPer], d[kPer], gy[kPer], z[kPer], bias[kPer];
                        of_channels(biases, bias);
                        uint4 *mine = kept + i * kKept * H::THREADS;
                        mine[0] = raw_x[i];
                        mine[H::THREADS] = raw_g[i];
                        Share::open(raw_x[i], x);
                        Share::open(raw_dt[i], d);
                        Share::open(raw_g[i], gy);
                        if (gated) {
                            mine[2 * H::THREADS] = raw_z[i];
                            Share::open(raw_z[i], z);
#pragma unroll
                            for (int e = 0; e < kPer; ++e) gy[e] *= z[e] * logistic(z[e]);
                        }
#pragma unroll
                        for (int e = 0; e < kPer; e += 2) {
                            float slope[2] = {1.0f, 1.0f};
#pragma unroll
                            for (int f = 0; f < 2; ++f) {
                                d[e + f] += bias[e + f];
                                if (p.softplus) d[e + f] = softplus_and_slope(d[e + f], slope[f]);
                                if ((share.by_step ? t + e + f : t) >= left) d[e + f] = x[e + f] = gy[e + f] = 0.0f;  // behind the last step: decay 1, no input
                            }
                            mine[(3 + e / 2) * H::THREADS] =
                                make_uint4(__float_as_uint(d[e]), __float_as_uint(slope[0]), __float_as_uint(d[e + 1]), __float_as_uint(slope[1]));
                        }
                        if (share.t >= kTile) continue;
                        if (share.by_step) {
#pragma unroll
                            for (int e = 0; e < kPer; ++e) {
                                steps[pair_slot<H::CB>(t + e, share.c)] = make_float2(d[e], x[e]);
                                gys[(t + e) * H::CB + share.c] = gy[e];
                            }
                        } else {
                            float2 *to = steps + t * H::CB;
#pragma unroll
                            for (int e = 0; e < kPer; e += 2)
                                *reinterpret_cast<float4 *>(to + ((slot0 ^ e) ^ (2 * (t & 1)))) = make_float4(d[e], x[e], d[e + 1], x[e + 1]);
#pragma unroll
                            for (int e = 0; e < kPer; e += 4)
                                *reinterpret_cast<float4 *>(gys + t * H::CB + share.c + e) = make_float4(gy[e], gy[e + 1], gy[e + 2], gy[e + 3]);
                        }
                    }
                    next_proj.put(tid, p.B.access, left, all_proj + buffer * 2 * kTile * H::SP);
                }
                fetch(put - 1);
                __syncthreads();
            }
        }
        // this CTA's sums for D and dt_bias: the threads of a channel one after the other
        float *mine = smem + tid * kPer, *mine_b = smem + (H::THREADS + tid) * kPer;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            mine[e] = share.works ? gD[e] : 0.0f;
            mine_b[e] = share.works ? gbias[e] : 0.0f;
        }
    } else {
        registers_up<kScanRegisters>();
        const int lane = tid & 31, warp = tid >> 5;
        const int ql = lane % LN, r = lane / LN, cl = warp * H::DL + r;
        const bool live = cl < channels;
        const int64_t c = c0 + (live ? cl : 0);
        const int have = live ? (S - ql * SPL < SPL ? S - ql * SPL : SPL) : 0;
        pair_t A[2];
        // the gradient of A: a tile's sum, and the sum over tiles.  One running sum would round thousands of terms against the whole.
        pair_t dA[2] = {0, 0}, dA_tiles[2] = {0, 0};
        load_lane_decays<SPL>(p.A, c * S + ql * SPL, have, p.vec, p.channels * S, 261, A);
        for (int64_t s = blockIdx.y; s < p.seq.count; s += gridDim.y) {
            const Span sp = span_of(p.seq, s);
            const int64_t tiles = (sp.length + kTile - 1) / kTile;
            const int64_t state_at = (s * p.channels + c) * S + ql * SPL, state_extent = p.seq.count * p.channels * S;
            const int64_t slot0 = checkpoint_base(p, s, sp.start);
            pair_t adjoint[2] = {0, 0}, first[2] = {0, 0};
            if (q.gstate_out != nullptr) load_lane_states<SPL>(q.gstate_out, state_at, have, p.vec, state_extent, 232, adjoint);
            const auto checkpoint = [&](int64_t slot, pair_t (&h)[2]) {
                load_lane_states<SPL>(p.checkpoints, ((slot0 + slot) * p.channels + c) * S + ql * SPL, have, p.vec,
                                      p.checkpoint_slots * S * p.channels, 237, h);
            };
            int64_t slot = (sp.length + kCheckpointSteps - 1) / kCheckpointSteps - 1;  // of the run of 16 steps to come
            if (slot >= 0) checkpoint(slot, first);
            __syncthreads();  // phase -1
            for (int64_t phase = 0; phase <= tiles; ++phase) {
                if (phase < tiles) {
                    const int64_t k = tiles - 1 - phase;
                    const int here = sp.length - k * kTile < kTile ? (int)(sp.length - k * kTile) : kTile;
                    float2 *steps = all_steps + (phase & 1) * kTile * H::CB;
                    float *gys = all_gy + (phase & 1) * kTile * H::CB + cl;
                    const float *Bs = all_proj + (phase & 1) * 2 * kTile * H::SP + ql * SPL, *Cs = Bs + kTile * H::SP;
                    float *sums = all_sums + ((phase & 1) * WARPS + warp) * kTile * 2 * H::SP + ql * SPL;
                    // two steps' 8 sums over the warp's channels, into the rows of B (0) or C (1)
                    const auto send_sums = [&](float (&v)[8], int i, int t, int which) {
                        float *to = sums + ((t + (i >> 2)) * 2 + which) * H::SP + (i & 3);
                        if constexpr (H::DL >= 8) {
                            if (r < 8) *to = v[0];
                        } else {
                            static_assert(H::DL == 4, "two sums a lane");
                            *reinterpret_cast<float2 *>(to) = make_float2(v[0], v[1]);
                        }
                    };
#pragma unroll 1
                    for (int t16 = here > kCheckpointSteps ? kCheckpointSteps : 0; t16 >= 0; t16 -= kCheckpointSteps) {
                        pair_t start[4][2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) start[0][e] = first[e];
                        if (--slot >= 0) checkpoint(slot, first);  // for the 16 steps before these
#pragma unroll
                        for (int sub = 0; sub < 3; ++sub) {
                            pair_t h[2] = {start[sub][0], start[sub][1]};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int t = t16 + sub * 4 + i;
                                const float2 dx = steps[pair_slot<H::CB>(t, cl)];
                                const pair_t dt2 = both(dx.x), u2 = both(dx.x * dx.y);
                                pair_t b[2];
                                load_lane_projection<SPL>(Bs + t * H::SP, b);
#pragma unroll
                                for (int e = 0; e < 2; ++e) h[e] = fma2(exp2_pair(fma2(dt2, A[e], both(kExponentShift))), h[e], mul2(u2, b[e]));
                            }
                            start[sub + 1][0] = h[0];
                            start[sub + 1][1] = h[1];
                        }
#pragma unroll
                        for (int sub = 3; sub >= 0; --sub) {
                            const int t4 = t16 + sub * 4;
                            pair_t h[2] = {start[sub][0], start[sub][1]}, a[4][2], m[4][2], b[4][2], cc[4][2];
                            float2 dx[4];
                            float gy[4], y[4], vB[2][8], vC[2][8];
                            // everything these steps need is loaded before anything is stored
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                dx[i] = steps[pair_slot<H::CB>(t4 + i, cl)];
                                gy[i] = gys[(t4 + i) * H::CB];
                                load_lane_projection<SPL>(Bs + (t4 + i) * H::SP, b[i]);
                                load_lane_projection<SPL>(Cs + (t4 + i) * H::SP, cc[i]);
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const pair_t dt2 = both(dx[i].x), u2 = both(dx[i].x * dx[i].y), gy2 = both(gy[i]);
                                pair_t sum;
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    a[i][e] = exp2_pair(fma2(dt2, A[e], both(kExponentShift)));
                                    m[i][e] = mul2(a[i][e], h[e]);  // a_t h_{t-1}
                                    h[e] = fma2(u2, b[i][e], m[i][e]);
                                    sum = e == 0 ? mul2(h[e], cc[i][e]) : fma2(h[e], cc[i][e], sum);
                                    const float2 f = halves(mul2(gy2, h[e]));
                                    vC[i >> 1][(i & 1) * 4 + 2 * e] = f.x;
                                    vC[i >> 1][(i & 1) * 4 + 2 * e + 1] = f.y;
                                }
                                const float2 f = halves(sum);
                                y[i] = f.x + f.y;
                            }
                            float through[4], bydecay[4];
#pragma unroll
                            for (int i = 3; i >= 0; --i) {
                                const pair_t dt2 = both(dx[i].x), u2 = both(dx[i].x * dx[i].y), gy2 = both(gy[i]);
                                pair_t sum_b, sum_a;
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const pair_t dh = fma2(gy2, cc[i][e], adjoint[e]);
                                    adjoint[e] = mul2(a[i][e], dh);
                                    const pair_t w = mul2(dh, m[i][e]);
                                    sum_b = e == 0 ? mul2(dh, b[i][e]) : fma2(dh, b[i][e], sum_b);
                                    sum_a = e == 0 ? mul2(w, A[e]) : fma2(w, A[e], sum_a);
                                    dA[e] = fma2(w, dt2, dA[e]);
                                    const float2 f = halves(mul2(dh, u2));
                                    vB[i >> 1][(i & 1) * 4 + 2 * e] = f.x;
                                    vB[i >> 1][(i & 1) * 4 + 2 * e + 1] = f.y;
                                }
                                const float2 f = halves(sum_b), o = halves(sum_a);
                                through[i] = f.x + f.y;
                                bydecay[i] = o.x + o.y;
                            }
                            // independent exchanges, then the stores
                            const int i0 = sum_over_channels<H::DL, LN>(vC[0], r), i1 = sum_over_channels<H::DL, LN>(vC[1], r);
                            sum_over_channels<H::DL, LN>(vB[0], r);
                            sum_over_channels<H::DL, LN>(vB[1], r);
                            send_sums(vC[0], i0, t4, 1);
                            send_sums(vC[1], i1, t4 + 2, 1);
                            send_sums(vB[0], i0, t4, 0);
                            send_sums(vB[1], i1, t4 + 2, 0);
                            // the channel's sums take the place of the steps, which all its lanes have read
                            __syncwarp();
                            constexpr int kSpread = LN < 4 ? LN : 4;
#pragma unroll
                            for (int i = 0; i < 4; i += kSpread) {
                                float v0[kSpread], v1[kSpread], v2[kSpread];
#pragma unroll
                                for (int e = 0; e < kSpread; ++e) {
                                    v0[e] = through[i + e];
                                    v1[e] = bydecay[i + e];
                                    v2[e] = y[i + e];
                                }
                                const float f0 = sum_and_spread<LN>(v0, ql), f1 = sum_and_spread<LN>(v1, ql), f2 = sum_and_spread<LN>(v2, ql);
                                if (ql < kSpread) {
                                    steps[pair_slot<H::CB>(t4 + i + ql, cl)] = make_float2(f0, f1);
                                    gys[(t4 + i + ql) * H::CB] = f2;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        dA_tiles[e] = add2(dA_tiles[e], dA[e]);
                        dA[e] = 0;
                    }
                }
                __syncthreads();
            }
            if (q.gstate != nullptr) store_lane_states<SPL>(q.gstate, state_at, have, p.vec, state_extent, 243, adjoint);
        }
        store_lane_states<SPL>(q.part_A, ((int64_t)blockIdx.y * p.channels + c) * S + ql * SPL, have, p.vec,
                               (int64_t)gridDim.y * p.channels * S, 244, dA_tiles);
    }
    __syncthreads();
    if (threadIdx.x < channels) {
        const int ch = threadIdx.x;
        const bool by_step = p.x.access == kTileSteps;
        float d = 0.0f, b = 0.0f;
        const int first = by_step ? ch : ch / kPer, apart = by_step ? H::CB : H::CB / kPer;
        for (int i = first; i < H::THREADS; i += apart)
            for (int e = by_step ? 0 : ch % kPer; e < (by_step ? kPer : ch % kPer + 1); ++e) {
                d += smem[i * kPer + e];
                b += smem[(H::THREADS + i) * kPer + e];
            }
        const int64_t to = (int64_t)blockIdx.y * p.channels + c0 + ch, extent = (int64_t)gridDim.y * p.channels;
        store_one(q.part_D, to, extent, 245, d);
        store_one(q.part_bias, to, extent, 246, b);
    }
    for (int64_t s = blockIdx.y; s < p.seq.count; s += gridDim.y) {
        const Span sp = span_of(p.seq, s);
        zero_uncovered<io_t>(p.seq, s, sp, q.gx, c0, c0 + channels, 240);
        zero_uncovered<io_t>(p.seq, s, sp, q.gdt, c0, c0 + channels, 241);
        if (p.z.data != nullptr) zero_uncovered<io_t>(p.seq, s, sp, q.gz, c0, c0 + channels, 242);
    }
}

}  // namespace ssb
