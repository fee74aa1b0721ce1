// Backward of the selective scan where channels are few or states more than 32 (else ssm_backward.cuh), with lanes
// across time, and the sums over CTAs that both forms leave to it.  Per channel c and state n
//     h_t = exp(dt_t A[c,n]) h_{t-1} + dt_t x_t B_t[n],     y_t = sum_n C_t[n] h_t + D x_t,     out = y silu(z),
// whose backward runs the adjoint r_t = exp(dt_t A) (gy_t C_t + r_{t+1}) from the right.
//
// The forward writes one state in a tile of steps; the others are rebuilt here.  The recurrence is cut along time inside
// the warp so that an exponential is computed once and used in both directions (fold and replay), with one more for the
// decay over a thread's 8 steps: 9/8 a (step, channel, state).
//
// What bounds it: latency.  254 registers leave 8 warps an SM, and a turn over a state composes two maps by dependent
// shuffles and ends in a barrier.  [2, 1024, 1024], 64 states in 4 groups, fp16: 422 us, 40 instructions an exponential in
// 37 % of the issue slots, against 29 us for the exponentials alone.
//
// A thread holds 8 consecutive steps of 2 adjacent channels (pairs in 64-bit registers) and goes
// through the states one by one.  For a state it folds its 8 steps to an affine map, the TL lanes
// that hold the same channels compose their maps with log2(TL) shuffle steps, and each thread then
// replays its steps from the state that enters them, adding C_t h_t to its 16 sums: the sum over
// states needs no communication.  A warp covers TL * 8 steps of 2 * 32 / TL channels; a CTA of W
// warps W times the channels of the same steps, whose B and C it stages in shared memory as fp32.
// TL is the split of the 32 lanes between time and channels: larger where there are few channels.
#pragma once

#include "ssm_common.cuh"

namespace ssb {

struct ProjView {  // B or C: [N, G, S, T]
    void *data;
    int64_t sn, sg, ss, st, extent;
    int access;  // ProjAccess
};

struct SelectiveArgs {
    int64_t channels, per_group, groups, states;
    int blocks_per_group, softplus, tile_log2, vec;  // tile_log2: steps between checkpoints; vec: 4 states at a time are whole and aligned
    Sequences seq;
    View3 x, dt, z, out;
    ProjView B, C;
    const float *A, *D, *dt_bias, *state;
    float *state_out, *checkpoints;
    int64_t checkpoint_slots;
};

struct SelectiveGradArgs {
    View3 gout, gx, gdt, gz;
    const float *gstate_out;
    float *gstate;
    float *part_B, *part_C;  // [blocks per group][N, T, G, S]
    float *part_A, *part_D, *part_bias;  // [gridDim.y][C, S], [gridDim.y][C] twice
    int64_t rows;
};

constexpr int kSlab = 32;  // most states staged at a time

__host__ __device__ constexpr int scan_pad(int tile) { return tile + 4; }  // floats per staged state: keeps 16-byte alignment

// First checkpoint slot of a sequence: ceil(length / tile) slots from here never reach the next one's.
__device__ __forceinline__ int64_t checkpoint_base(const SelectiveArgs &p, int64_t s, int64_t start) {
    const int64_t per_row = (p.seq.steps + (1ll << p.tile_log2) - 1) >> p.tile_log2;
    return p.seq.offsets != nullptr ? (start >> p.tile_log2) + s : s * per_row;
}

// How B and C are fetched: 16 bytes along the states of a step or along the steps of a state where
// the strides allow it, else element by element.
enum ProjAccess : int { kProjAny = 0, kProjStates = 1, kProjSteps = 2 };

// States staged at a time: so many that a thread fetches at most two 16-byte pieces of each of B and C.
template <typename io_t, int TILE, int THREADS>
__host__ __device__ constexpr int slab_states() {
    const int n = 2 * THREADS * (16 / (int)sizeof(io_t)) / TILE;
    return n > kSlab ? kSlab : n;
}

// One slab's pieces, fetched ahead and put down as fp32 [state][step] when the tile before is done.
template <typename io_t, int TILE, int THREADS>
struct ProjPieces {
    static constexpr int kPer = 16 / (int)sizeof(io_t);  // elements of a piece
    static constexpr int kSlabStates = slab_states<io_t, TILE, THREADS>();
    static constexpr int kPieces = (kSlabStates * TILE / kPer + THREADS - 1) / THREADS;
    uint4 piece[kPieces];

    // Steps [t, t + TILE) of states [n0, n0 + count); zero behind `steps` steps.
    __device__ __forceinline__ void fetch(const ProjView &v, int64_t row, int64_t g, int n0, int count, int64_t t, int64_t steps) {
        if (v.access == kProjAny) return;
        const io_t *base = static_cast<const io_t *>(v.data);
        const int64_t at = row * v.sn + g * v.sg + n0 * v.ss + t * v.st;
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int i = threadIdx.x + j * THREADS;
            // along the states: lanes hold neighbouring steps, so that the fp32 stores below meet no bank twice
            const int n = v.access == kProjStates ? i / TILE * kPer : i / (TILE / kPer);
            const int k = v.access == kProjStates ? i % TILE : i % (TILE / kPer) * kPer;
            piece[j] = make_uint4(0, 0, 0, 0);
            const int64_t e = at + n * v.ss + k * v.st;
            if (n < count && k < steps && SSB_VECTOR_OK(base + e, 16, e + kPer - 1, v.extent, 210))
                piece[j] = *reinterpret_cast<const uint4 *>(base + e);
        }
    }
    __device__ __forceinline__ void put(const ProjView &v, int64_t row, int64_t g, int n0, int count, int64_t t, int64_t steps,
                                        float *smem) const {
        if (v.access == kProjAny) {
            const io_t *base = static_cast<const io_t *>(v.data);
            const int64_t at = row * v.sn + g * v.sg + n0 * v.ss + t * v.st;
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            // the lanes run along whichever index is adjacent in memory
            const bool by_state = v.ss <= v.st;
            const int outer = by_state ? TILE : count, inner = by_state ? count : TILE;
            for (int o = warp; o < outer; o += THREADS / 32)
                for (int i = lane; i < inner; i += 32) {
                    const int n = by_state ? i : o, k = by_state ? o : i;
                    smem[n * scan_pad(TILE) + k] = k < steps ? load_one<io_t>(base, at + n * v.ss + k * v.st, v.extent, 210) : 0.0f;
                }
            return;
        }
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int i = threadIdx.x + j * THREADS;
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
            if (v.access == kProjStates) {
                const int n = i / TILE * kPer, k = i % TILE;
                if (n < count) {
#pragma unroll
                    for (int e = 0; e < kPer; ++e) smem[(n + e) * scan_pad(TILE) + k] = f[e];
                }
            } else {
                const int n = i / (TILE / kPer), k = i % (TILE / kPer) * kPer;
                if (n < count) {
#pragma unroll
                    for (int e = 0; e < kPer; e += 4) {
                        // a fetched piece may reach behind the last step: those elements are not the sequence's
                        float4 q = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
                        if (k + e + 0 >= steps) q.x = 0.0f;
                        if (k + e + 1 >= steps) q.y = 0.0f;
                        if (k + e + 2 >= steps) q.z = 0.0f;
                        if (k + e + 3 >= steps) q.w = 0.0f;
                        *reinterpret_cast<float4 *>(smem + n * scan_pad(TILE) + k + e) = q;
                    }
                }
            }
        }
    }
};

// A[c, n] * log2(e) of the CTA's channels, [state][channel]; zero behind the last channel.  An
// infinite entry becomes the largest finite one: with a step of zero it then decays by 2^0 = 1, as
// padding has to.
template <int CB>
__device__ __forceinline__ void stage_decays(const SelectiveArgs &p, int64_t c0, int64_t c_end, int n0, int count, float *smem) {
    for (int i = threadIdx.x; i < count * CB; i += blockDim.x) {
        const int c = i / count, n = i - c * count;
        float v = 0.0f;
        if (c0 + c < c_end) {
            const int64_t at = (c0 + c) * p.states + n0 + n;
            if (SSB_INDEX_OK(at, p.channels * p.states, 211)) v = p.A[at] * kLog2e;
            if (isinf(v)) v = copysignf(3.402823466e38f, v);
        }
        smem[n * CB + c] = v;
    }
}

// Zeros into steps [from, to) of a row of the CTA's channels.
template <typename io_t>
__device__ __forceinline__ void zero_steps(const View3 &v, int64_t row, int64_t c0, int64_t c_end, int64_t from, int64_t to, int site) {
    io_t *base = static_cast<io_t *>(v.data);
    const int64_t nc = c_end - c0, nt = to - from;
    if (nc <= 0 || nt <= 0) return;
    for (int64_t i = threadIdx.x; i < nc * nt; i += blockDim.x) {
        int64_t c, t;
        if (v.sc == 1) {
            t = i / nc;
            c = i - t * nc;
        } else {
            c = i / nt;
            t = i - c * nt;
        }
        store_one<io_t>(base, row * v.sn + (c0 + c) * v.sc + (from + t) * v.st, v.extent, site, 0.0f);
    }
}

// The steps of an output that belong to no sequence are zero: behind a row's length, before the
// first packed sequence and behind the last.
template <typename io_t>
__device__ __forceinline__ void zero_uncovered(const Sequences &q, int64_t s, const Span &sp, const View3 &v, int64_t c0,
                                               int64_t c_end, int site) {
    if (q.offsets == nullptr) {
        zero_steps<io_t>(v, sp.row, c0, c_end, sp.length, q.steps, site);
    } else {
        if (s == 0) zero_steps<io_t>(v, 0, c0, c_end, 0, sp.start, site);
        if (s == q.count - 1) zero_steps<io_t>(v, 0, c0, c_end, sp.start + sp.length, q.steps, site);
    }
}

// Per-channel [C, S] values of a warp's own channels between global memory and [state][channel] in shared memory.
template <int CB, int CW>
__device__ __forceinline__ void load_states(const float *src, int64_t seq, const SelectiveArgs &p, int64_t c0, int64_t c_end,
                                            int warp, int lane, int site, float *smem) {
    for (int i = lane; i < CW * (int)p.states; i += 32) {
        const int c = i / (int)p.states, n = i - c * (int)p.states, cl = warp * CW + c;
        float v = 0.0f;
        if (src != nullptr && c0 + cl < c_end) {
            const int64_t at = (seq * p.channels + c0 + cl) * p.states + n;
            if (SSB_INDEX_OK(at, p.seq.count * p.channels * p.states, site)) v = src[at];
        }
        smem[n * CB + cl] = v;
    }
    __syncwarp();
}
template <int CB, int CW>
__device__ __forceinline__ void store_states(float *dst, int64_t seq, const SelectiveArgs &p, int64_t c0, int64_t c_end,
                                             int warp, int lane, int site, const float *smem) {
    __syncwarp();
    for (int i = lane; i < CW * (int)p.states; i += 32) {
        const int c = i / (int)p.states, n = i - c * (int)p.states, cl = warp * CW + c;
        if (c0 + cl < c_end) {
            const int64_t at = (seq * p.channels + c0 + cl) * p.states + n;
            if (SSB_INDEX_OK(at, p.seq.count * p.channels * p.states, site)) dst[at] = smem[n * CB + cl];
        }
    }
    __syncwarp();
}

// The step sizes of a run: softplus(raw + bias) or raw + bias; zero (decay 1, no input) behind the last step.
__device__ __forceinline__ void make_steps(pair_t (&dt)[kRun], float2 bias, int softplus_on, int steps) {
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
        dt[k] = add2(dt[k], make_pair(bias.x, bias.y));
        if (softplus_on) dt[k] = softplus2(dt[k]);
        if (k >= steps) dt[k] = 0;
    }
}

// Composes the maps (P, S) of a channel's TL lanes from the left: inclusive prefix.
template <int TL>
__device__ __forceinline__ void compose_left(pair_t &P, pair_t &S, int tl) {
    constexpr int DL = 32 / TL;
#pragma unroll
    for (int d = 1; d < TL; d <<= 1) {
        const pair_t P0 = shfl_up2(P, d * DL), S0 = shfl_up2(S, d * DL);
        if (tl >= d) {
            S = fma2(P, S0, S);
            P = mul2(P, P0);
        }
    }
}
template <int TL>
__device__ __forceinline__ void compose_right(pair_t &P, pair_t &S, int tl) {
    constexpr int DL = 32 / TL;
#pragma unroll
    for (int d = 1; d < TL; d <<= 1) {
        const pair_t P0 = shfl_down2(P, d * DL), S0 = shfl_down2(S, d * DL);
        if (tl + d < TL) {
            S = fma2(P, S0, S);
            P = mul2(P, P0);
        }
    }
}

__device__ __forceinline__ void load8(const float *smem, float (&v)[kRun]) {
    const float4 a = *reinterpret_cast<const float4 *>(smem), b = *reinterpret_cast<const float4 *>(smem + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// N adjacent floats in shared memory, 16 (8) bytes at a time.
template <int N>
__device__ __forceinline__ void add_to(float *to, const float *v) {
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            float4 f = *reinterpret_cast<float4 *>(to + i);
            f.x += v[i]; f.y += v[i + 1]; f.z += v[i + 2]; f.w += v[i + 3];
            *reinterpret_cast<float4 *>(to + i) = f;
        }
    } else if constexpr (N == 2) {
        float2 f = *reinterpret_cast<float2 *>(to);
        f.x += v[0]; f.y += v[1];
        *reinterpret_cast<float2 *>(to) = f;
    } else {
        *to += *v;
    }
}

template <int TL, int W>
struct ScanShape {
    static constexpr int DL = 32 / TL;       // lanes across channels
    static constexpr int CW = 2 * DL;        // channels of a warp
    static constexpr int CB = W * CW;        // channels of a CTA
    static constexpr int TILE = TL * kRun;   // steps of a tile
    static constexpr int PAD = scan_pad(TILE);
};

// ---- backward -----------------------------------------------------------------------------------
// Tiles run from the last to the first.  Each starts from its checkpoint (the state the forward
// wrote at the tile's first step), rebuilds the states as the forward does, and carries the adjoint
// r to the tile on its left.  Per (step, channel, state) there are 9/8 exponentials and 17 fp32 operations.
//
// The gradients of B and C sum over channels: over the pair in the thread, over the DL lanes by an
// exchange that halves the number of values at each step (16 values: 8 + 4 shuffles for DL = 4),
// over the warps of the CTA in shared memory, over CTAs by selective_reduce_kernel in a fixed order.  The warps of
// a CTA work on different states at a time (warp w on state (i + w) mod count), with a barrier per
// state, so that none adds to a row of sums that another is adding to, and the order of the additions is always the same.
template <typename io_t, int TL, int W>
__host__ __device__ constexpr size_t selective_bwd_smem(int64_t states) {
    using H = ScanShape<TL, W>;
    constexpr int most = slab_states<io_t, H::TILE, W * 32>();
    const int64_t slab = states < most ? states : most;
    return sizeof(float) * (size_t)(states * H::CB * 2 + slab * (2 * H::CB + 4 * H::PAD));
}

template <typename io_t, int TL, int W>
__global__ void __launch_bounds__(W * 32) selective_bwd_kernel(const __grid_constant__ SelectiveArgs p,
                                                              const __grid_constant__ SelectiveGradArgs q) {
    using H = ScanShape<TL, W>;
    using Pieces = ProjPieces<io_t, H::TILE, W * 32>;
    extern __shared__ __align__(16) float smem[];
    const int S = (int)p.states, slab = S < Pieces::kSlabStates ? S : Pieces::kSlabStates;
    float *adjoint = smem;                              // [states][CB]: r entering the tile from the right
    float *gA = adjoint + S * H::CB;                    // [states][CB]: sums over this CTA's steps
    float *decay = gA + S * H::CB;                      // [slab][CB]
    float *first = decay + slab * H::CB;                // [slab][CB]: the state entering the tile
    float *Bs = first + slab * H::CB, *Cs = Bs + slab * H::PAD;
    float *sumB = Cs + slab * H::PAD, *sumC = sumB + slab * H::PAD;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tl = lane / H::DL, dl = lane % H::DL, cl = warp * H::CW + 2 * dl;
    const int64_t g = blockIdx.x / p.blocks_per_group, j = blockIdx.x % p.blocks_per_group;
    const int64_t c0 = g * p.per_group + j * H::CB;
    const int64_t c_end = c0 + H::CB < (g + 1) * p.per_group ? c0 + H::CB : (g + 1) * p.per_group;
    const int64_t c = c0 + cl;
    const int nc = c_end - c >= 2 ? 2 : (c_end > c ? 1 : 0);
    float2 D = make_float2(0.0f, 0.0f), bias = D;
    if (p.D != nullptr) {
        if (nc > 0) D.x = load_one(p.D, c, p.channels, 230);
        if (nc > 1) D.y = load_one(p.D, c + 1, p.channels, 230);
    }
    if (p.dt_bias != nullptr) {
        if (nc > 0) bias.x = load_one(p.dt_bias, c, p.channels, 231);
        if (nc > 1) bias.y = load_one(p.dt_bias, c + 1, p.channels, 231);
    }
    const pair_t Dp = make_pair(D.x, D.y);
    for (int i = threadIdx.x; i < S * H::CB; i += blockDim.x) gA[i] = 0.0f;
    if (S <= slab) stage_decays<H::CB>(p, c0, c_end, 0, S, decay);
    pair_t gD = 0, gbias = 0;

    for (int64_t s = blockIdx.y; s < p.seq.count; s += gridDim.y) {
        const Span sp = span_of(p.seq, s);
        load_states<H::CB, H::CW>(q.gstate_out, s, p, c0, c_end, warp, lane, 232, adjoint);
        const int64_t slot0 = checkpoint_base(p, s, sp.start);
        const int64_t tiles = (sp.length + H::TILE - 1) / H::TILE;
        for (int64_t i_tile = tiles - 1; i_tile >= 0; --i_tile) {
            const int64_t t0 = i_tile * H::TILE;
            const int64_t left = sp.length - t0 - tl * kRun;
            const int steps = left >= kRun ? kRun : (left > 0 ? (int)left : 0);
            const int64_t t = sp.start + t0 + tl * kRun;
            pair_t dt[kRun], u[kRun], gy[kRun], y[kRun];
            pair_t through[kRun], bydecay[kRun];  // sum_n dh B  and  sum_n dh (a h_{t-1}) A log2(e)
            RawRun<io_t> raw_x, raw_dt, raw_z, raw_g;  // all under way before the first is used
            fetch_run(q.gout, sp.row, c, t, steps, nc, 233, raw_g);
            if (p.z.data != nullptr) fetch_run(p.z, sp.row, c, t, steps, nc, 234, raw_z);
            fetch_run(p.x, sp.row, c, t, steps, nc, 235, raw_x);
            fetch_run(p.dt, sp.row, c, t, steps, nc, 236, raw_dt);
            open_run(raw_g, gy);
            if (p.z.data != nullptr) {
                open_run(raw_z, y);
#pragma unroll
                for (int k = 0; k < kRun; ++k) {
                    const float2 z = halves(y[k]), f = halves(gy[k]);
                    gy[k] = make_pair(f.x * (z.x * logistic(z.x)), f.y * (z.y * logistic(z.y)));
                }
            }
            open_run(raw_x, u);
            open_run(raw_dt, dt);
            make_steps(dt, bias, p.softplus, steps);
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                y[k] = mul2(Dp, u[k]);
                gD = fma2(gy[k], u[k], gD);
                u[k] = mul2(dt[k], u[k]);
                through[k] = 0;
                bydecay[k] = 0;
            }
            const pair_t span = add2(add2(add2(dt[0], dt[1]), add2(dt[2], dt[3])), add2(add2(dt[4], dt[5]), add2(dt[6], dt[7])));
            for (int n0 = 0; n0 < S; n0 += slab) {
                const int count = S - n0 < slab ? S - n0 : slab;
                Pieces next_B, next_C;
                next_B.fetch(p.B, sp.row, g, n0, count, sp.start + t0, sp.length - t0);
                next_C.fetch(p.C, sp.row, g, n0, count, sp.start + t0, sp.length - t0);
                __syncthreads();
                if (S > slab) stage_decays<H::CB>(p, c0, c_end, n0, count, decay);
                next_B.put(p.B, sp.row, g, n0, count, sp.start + t0, sp.length - t0, Bs);
                next_C.put(p.C, sp.row, g, n0, count, sp.start + t0, sp.length - t0, Cs);
                for (int i = threadIdx.x; i < count * H::CB; i += blockDim.x) {
                    const int cc = i / count, n = i - cc * count;
                    const int64_t at = ((slot0 + i_tile) * p.channels + c0 + cc) * S + n0 + n;
                    first[n * H::CB + cc] = c0 + cc < c_end ? load_one(p.checkpoints, at, p.checkpoint_slots * S * p.channels, 237) : 0.0f;
                }
                for (int i = threadIdx.x; i < count * H::PAD; i += blockDim.x) {
                    sumB[i] = 0.0f;
                    sumC[i] = 0.0f;
                }
                __syncthreads();
                const int turns = count > W ? count : W;
                for (int turn = 0; turn < turns; ++turn) {
                    int n = turn + warp;
                    if (n >= turns) n -= turns;
                    if (n < count) {
                        const pair_t A = *reinterpret_cast<const pair_t *>(decay + n * H::CB + cl);
                        pair_t *held = reinterpret_cast<pair_t *>(adjoint + (n0 + n) * H::CB + cl);
                        const pair_t r_in = *held;
                        const pair_t h_in = *reinterpret_cast<const pair_t *>(first + n * H::CB + cl);
                        pair_t a[kRun], m[kRun];
                        float bv[kRun], cv[kRun], v[2 * kRun];
                        load8(Bs + n * H::PAD + tl * kRun, bv);
                        load8(Cs + n * H::PAD + tl * kRun, cv);
#pragma unroll
                        for (int k = 0; k < kRun; ++k) a[k] = exp2_pair(fma2(dt[k], A, both(kExponentShift)));
                        pair_t P = exp2_pair(fma2(span, A, both(kExponentShift))), F = mul2(u[0], both(bv[0]));  // P: the decay over all 8 steps
#pragma unroll
                        for (int k = 1; k < kRun; ++k) F = fma2(u[k], both(bv[k]), mul2(a[k], F));
                        const pair_t P0 = P;
                        compose_left<TL>(P, F, tl);
                        pair_t h = shfl_up2(fma2(P, h_in, F), H::DL);
                        if (tl == 0) h = h_in;
#pragma unroll
                        for (int k = 0; k < kRun; ++k) {
                            m[k] = mul2(a[k], h);                    // a_t h_{t-1}
                            h = fma2(u[k], both(bv[k]), m[k]);
                            y[k] = fma2(h, both(cv[k]), y[k]);
                            const float2 f = halves(mul2(gy[k], h));
                            v[kRun + k] = f.x + f.y;                 // this pair's part of the gradient of C
                        }
                        pair_t Q = 0;
#pragma unroll
                        for (int k = kRun - 1; k >= 0; --k) Q = mul2(a[k], fma2(gy[k], both(cv[k]), Q));
                        P = P0;
                        compose_right<TL>(P, Q, tl);
                        const pair_t r_out = fma2(P, r_in, Q);       // r of this lane's first step
                        pair_t r = shfl_down2(r_out, H::DL);
                        if (tl == TL - 1) r = r_in;
                        __syncwarp();
                        if (tl == 0) *held = r_out;
                        pair_t dA = 0;
#pragma unroll
                        for (int k = kRun - 1; k >= 0; --k) {
                            const pair_t dh = fma2(gy[k], both(cv[k]), r);
                            r = mul2(a[k], dh);
                            const float2 f = halves(mul2(dh, u[k]));
                            v[k] = f.x + f.y;                        // this pair's part of the gradient of B
                            through[k] = fma2(dh, both(bv[k]), through[k]);
                            const pair_t w = mul2(dh, m[k]);
                            bydecay[k] = fma2(w, A, bydecay[k]);
                            dA = fma2(w, dt[k], dA);
                        }
#pragma unroll
                        for (int d = H::DL; d < 32; d <<= 1) {       // over the lanes of the channel
                            const float2 f = halves(dA);
                            dA = add2(dA, make_pair(__shfl_xor_sync(kFullMask, f.x, d), __shfl_xor_sync(kFullMask, f.y, d)));
                        }
                        if (tl == 0) {
                            pair_t *to = reinterpret_cast<pair_t *>(gA + (n0 + n) * H::CB + cl);
                            *to = add2(*to, dA);
                        }
                        // over the DL lanes: each ends with 16 / DL of the 16 sums
                        int at = 0, held_values = 2 * kRun;
#pragma unroll
                        for (int bit = H::DL / 2; bit >= 1; bit >>= 1) {
                            held_values >>= 1;
                            const bool upper = (dl & bit) != 0;
                            if (upper) at += held_values;
#pragma unroll
                            for (int i = 0; i < kRun; ++i) {
                                if (i < held_values) {
                                    const float give = upper ? v[i] : v[i + held_values];
                                    const float keep = upper ? v[i + held_values] : v[i];
                                    v[i] = keep + __shfl_xor_sync(kFullMask, give, bit);
                                }
                            }
                        }
                        constexpr int kHeld = 2 * kRun / H::DL;  // sums that this lane is left with: adjacent steps of B or of C
                        if constexpr (kHeld == 2 * kRun) {
                            add_to<kRun>(sumB + n * H::PAD + tl * kRun, v);
                            add_to<kRun>(sumC + n * H::PAD + tl * kRun, v + kRun);
                        } else {
                            add_to<kHeld>((at < kRun ? sumB : sumC) + n * H::PAD + tl * kRun + (at & (kRun - 1)), v);
                        }
                    }
                    __syncthreads();
                }
                // the CTA's sums: [block][row, step, group, state]
                const int64_t extent = (int64_t)p.blocks_per_group * q.rows * p.seq.steps * p.groups * S;
                const int valid = sp.length - t0 < H::TILE ? (int)(sp.length - t0) : H::TILE;
                for (int i = threadIdx.x; i < count * valid; i += blockDim.x) {
                    const int k = i / count, n = i - k * count;
                    const int64_t at = (((j * q.rows + sp.row) * p.seq.steps + sp.start + t0 + k) * p.groups + g) * S + n0 + n;
                    store_one(q.part_B, at, extent, 238, sumB[n * H::PAD + k]);
                    store_one(q.part_C, at, extent, 239, sumC[n * H::PAD + k]);
                }
            }
            // per step and channel: the gradients of x, dt, z
            pair_t raw[kRun], xv[kRun], t2[kRun];
            load_run<io_t>(p.x, sp.row, c, t, steps, nc, 235, xv);
            load_run<io_t>(p.dt, sp.row, c, t, steps, nc, 236, raw);
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                t2[k] = fma2(through[k], dt[k], mul2(Dp, gy[k]));
                float2 f = halves(fma2(through[k], xv[k], mul2(bydecay[k], both(kLn2))));
                if (p.softplus) {
                    const float2 w = halves(raw[k]);
                    f.x *= logistic_accurate(w.x + bias.x);
                    f.y *= logistic_accurate(w.y + bias.y);
                }
                raw[k] = make_pair(f.x, f.y);
                if (k < steps) gbias = add2(gbias, raw[k]);
            }
            store_run<io_t>(q.gx, sp.row, c, t, steps, nc, 240, t2);
            store_run<io_t>(q.gdt, sp.row, c, t, steps, nc, 241, raw);
            if (p.z.data != nullptr) {
                load_run<io_t>(p.z, sp.row, c, t, steps, nc, 234, xv);
                load_run<io_t>(q.gout, sp.row, c, t, steps, nc, 233, raw);
#pragma unroll
                for (int k = 0; k < kRun; ++k) {
                    const float2 z = halves(xv[k]), f = halves(mul2(raw[k], y[k]));
                    const float sx = logistic(z.x), sy = logistic(z.y);
                    t2[k] = make_pair(f.x * sx * fmaf(z.x, 1.0f - sx, 1.0f), f.y * sy * fmaf(z.y, 1.0f - sy, 1.0f));
                }
                store_run<io_t>(q.gz, sp.row, c, t, steps, nc, 242, t2);
            }
        }
        if (q.gstate != nullptr) store_states<H::CB, H::CW>(q.gstate, s, p, c0, c_end, warp, lane, 243, adjoint);
        zero_uncovered<io_t>(p.seq, s, sp, q.gx, c0, c_end, 240);
        zero_uncovered<io_t>(p.seq, s, sp, q.gdt, c0, c_end, 241);
        if (p.z.data != nullptr) zero_uncovered<io_t>(p.seq, s, sp, q.gz, c0, c_end, 242);
        __syncthreads();
    }
    // this CTA's sums over its steps
    __syncthreads();
    for (int i = threadIdx.x; i < S * H::CB; i += blockDim.x) {
        const int cc = i / S, n = i - cc * S;
        if (c0 + cc < c_end)
            store_one(q.part_A, ((int64_t)blockIdx.y * p.channels + c0 + cc) * S + n, (int64_t)gridDim.y * p.channels * S, 244,
                      gA[n * H::CB + cc]);
    }
#pragma unroll
    for (int d = H::DL; d < 32; d <<= 1) {
        const float2 f = halves(gD), b = halves(gbias);
        gD = add2(gD, make_pair(__shfl_xor_sync(kFullMask, f.x, d), __shfl_xor_sync(kFullMask, f.y, d)));
        gbias = add2(gbias, make_pair(__shfl_xor_sync(kFullMask, b.x, d), __shfl_xor_sync(kFullMask, b.y, d)));
    }
    if (tl == 0) {
        const float2 f = halves(gD), b = halves(gbias);
        const int64_t at = (int64_t)blockIdx.y * p.channels + c, extent = (int64_t)gridDim.y * p.channels;
        if (nc > 0) {
            store_one(q.part_D, at, extent, 245, f.x);
            store_one(q.part_bias, at, extent, 246, b.x);
        }
        if (nc > 1) {
            store_one(q.part_D, at + 1, extent, 245, f.y);
            store_one(q.part_bias, at + 1, extent, 246, b.y);
        }
    }
}

// Sums the CTAs' parts, in the order of their numbers: B and C over the channel blocks of a group
// (blocks [0, proj_blocks) of the grid), A, D and dt_bias over the CTAs that shared the sequences.
// Steps that no sequence covers were not written and give zero.
struct SelectiveReduceArgs {
    Sequences seq;
    int64_t rows, groups, states, channels;
    int parts_proj, parts_seq, proj_blocks;
    const float *part_B, *part_C, *part_A, *part_D, *part_bias;
    ProjView gB, gC;
    float *gA, *gD, *gbias;
};

__device__ __forceinline__ bool step_covered(const Sequences &q, int64_t row, int64_t t) {
    if (q.offsets != nullptr) {  // sequences follow one another
        const int64_t a = clamp_step(q.offsets[0], 0, q.steps), b = clamp_step(q.offsets[q.count], a, q.steps);
        return t >= a && t < b;
    }
    return q.lengths == nullptr || t < clamp_step(q.lengths[row], 0, q.steps);
}

template <typename io_t>
__global__ void __launch_bounds__(256) selective_reduce_kernel(const __grid_constant__ SelectiveReduceArgs p) {
    const int64_t each = p.rows * p.seq.steps * p.groups * p.states;
    if ((int)blockIdx.x < p.proj_blocks) {
        for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < each; i += (int64_t)p.proj_blocks * blockDim.x) {
            const int64_t n = i % p.states, g = i / p.states % p.groups, rt = i / (p.states * p.groups);
            const int64_t t = rt % p.seq.steps, row = rt / p.seq.steps;
            float b = 0.0f, c = 0.0f;
            if (step_covered(p.seq, row, t)) {
#pragma unroll 4
                for (int j = 0; j < p.parts_proj; ++j) {
                    b += load_one(p.part_B, j * each + i, p.parts_proj * each, 250);
                    c += load_one(p.part_C, j * each + i, p.parts_proj * each, 251);
                }
            }
            store_one(static_cast<io_t *>(p.gB.data), row * p.gB.sn + g * p.gB.sg + n * p.gB.ss + t * p.gB.st, p.gB.extent, 252, b);
            store_one(static_cast<io_t *>(p.gC.data), row * p.gC.sn + g * p.gC.sg + n * p.gC.ss + t * p.gC.st, p.gC.extent, 253, c);
        }
    } else {
        const int64_t cs = p.channels * p.states, total = cs + 2 * p.channels;
        const int64_t stride = (int64_t)(gridDim.x - p.proj_blocks) * blockDim.x;
        for (int64_t i = (int64_t)(blockIdx.x - p.proj_blocks) * blockDim.x + threadIdx.x; i < total; i += stride) {
            const float *part = i < cs ? p.part_A : (i < cs + p.channels ? p.part_D : p.part_bias);
            float *to = i < cs ? p.gA : (i < cs + p.channels ? p.gD : p.gbias);
            const int64_t size = i < cs ? cs : p.channels, at = i < cs ? i : (i - cs) % p.channels;
            if (to == nullptr) continue;
            float v = 0.0f;
#pragma unroll 4
            for (int j = 0; j < p.parts_seq; ++j) v += load_one(part, j * size + at, p.parts_seq * size, 254);
            store_one(to, at, size, 255, v);
        }
    }
}

}  // namespace ssb
