// Short causal convolution per channel: v_t = bias + sum_j w[j] x_{t-W+1+j}, out = v or silu(v), for
// widths 2, 3 and 4, and its backward.  What lies before a sequence's first step is the window
// carried in (the last W-1 inputs of the piece before, oldest first), or zero.
//
// Memory-bound: 2 tensors forward, 3 more backward.  Two forms:
//   channels last   a thread owns V adjacent channels (one 8- or 16-byte access per step) and walks
//                   a chunk of steps with its window in registers; the steps before its chunk are read again;
//   rows            a warp owns a row; a lane takes 8 adjacent steps and reads its neighbours' few from cache.
#pragma once

#include "ssm_common.cuh"
#include "ssm_step.cuh"

namespace ssb {

struct ConvArgs {
    int64_t channels, rows, channel_blocks, chunk_blocks;
    int silu, weight_f32;
    Sequences seq;
    View3 x, out;
    const void *weight, *bias, *state;  // [C, W], [C]; [sequences, C, W-1] in the inputs' type
    void *state_out;
};
struct ConvGradArgs {
    View3 gout, gx;
    const void *gstate_out;
    void *gstate;
    float *part;  // [parts][C][W + 1]: gradients of the taps and the bias
};

constexpr int kConvWarps = 8;
constexpr int kConvChunk = 32;  // steps a warp walks

// The sequence that step t of a packed row lies in: the last one that starts at or before t (of
// several that start there, the last is the one with steps).  The lanes look at 32 offsets at a time.
__device__ __forceinline__ int64_t find_sequence(const Sequences &q, int64_t t, int lane) {
    int64_t lo = 0, n = q.count;  // the answer is in [lo, lo + n)
    while (n > 1) {
        const int64_t step = (n + 31) / 32, at = lo + lane * step;
        const bool at_or_before = lane * step < n && (lane == 0 || (int64_t)q.offsets[at] <= t);
        const unsigned votes = __ballot_sync(kFullMask, at_or_before);
        const int last = 31 - __clz(votes);
        const int64_t end = lo + n;
        lo += last * step;
        n = end - lo < step ? end - lo : step;
    }
    return lo;
}

template <typename io_t, int V>
struct Lump {
    float v[V];
};
template <typename io_t, int V>
__device__ __forceinline__ Lump<io_t, V> load_lump(const View3 &w, int64_t at, int site) {
    Lump<io_t, V> r;
    const io_t *p = static_cast<const io_t *>(w.data) + at;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = 0.0f;
    if (!SSB_VECTOR_OK(p, V * (int)sizeof(io_t), at + V - 1, w.extent, site)) return r;
    if constexpr (V == 1) {
        r.v[0] = static_cast<float>(*p);
    } else if constexpr (sizeof(io_t) == 4) {
        static_assert(V == 4, "16-byte accesses");
        const float4 f = *reinterpret_cast<const float4 *>(p);
        r.v[0] = f.x; r.v[1] = f.y; r.v[2] = f.z; r.v[3] = f.w;
    } else {
        static_assert(V == 4, "8-byte accesses");
        const uint2 f = *reinterpret_cast<const uint2 *>(p);
        unpack2<io_t>(f.x, r.v[0], r.v[1]);
        unpack2<io_t>(f.y, r.v[2], r.v[3]);
    }
    return r;
}
template <typename io_t, int V>
__device__ __forceinline__ void store_lump(const View3 &w, int64_t at, int site, const float (&v)[V]) {
    io_t *p = static_cast<io_t *>(w.data) + at;
    if (!SSB_VECTOR_OK(p, V * (int)sizeof(io_t), at + V - 1, w.extent, site)) return;
    if constexpr (V == 1) *p = static_cast<io_t>(v[0]);
    else if constexpr (sizeof(io_t) == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<io_t>(v[0], v[1]), pack2<io_t>(v[2], v[3]));
}

// Step `pos` (relative to the sequence's start; below zero: in the carried window) of V channels.
template <typename io_t, int V, int W>
__device__ __forceinline__ void input_at(const ConvArgs &p, const Span &sp, int64_t s, int64_t pos, int64_t c, float (&r)[V]) {
    if (pos >= 0) {
        const auto l = load_lump<io_t, V>(p.x, sp.row * p.x.sn + c * p.x.sc + (sp.start + pos) * p.x.st, 400);
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = l.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            r[i] = p.state != nullptr ? load_one(static_cast<const io_t *>(p.state), (s * p.channels + c + i) * (W - 1) + W - 1 + pos,
                                                 p.seq.count * p.channels * (W - 1), 401)
                                      : 0.0f;
    }
}

// The window behind a sequence's last step.
template <typename io_t, int V, int W>
__device__ __forceinline__ void store_window(const ConvArgs &p, int64_t s, int64_t c) {
    const Span sp = span_of(p.seq, s);
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        float r[V];
        input_at<io_t, V, W>(p, sp, s, sp.length - (W - 1) + i, c, r);
#pragma unroll
        for (int k = 0; k < V; ++k)
            store_one(static_cast<io_t *>(p.state_out), (s * p.channels + c + k) * (W - 1) + i, p.seq.count * p.channels * (W - 1), 402, r[k]);
    }
}

template <typename io_t, int V, int W>
__device__ __forceinline__ void load_taps(const ConvArgs &p, int64_t c, float (&w)[W][V], float (&bias)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i][k] = load_weight<io_t>(p.weight, p.weight_f32, (c + k) * W + i, p.channels * W, 403);
        bias[k] = p.bias != nullptr ? load_weight<io_t>(p.bias, p.weight_f32, c + k, p.channels, 404) : 0.0f;
    }
}

// The flat grid's coordinates: channel blocks fastest, then blocks of chunks, then rows; the channels-last
// kernels have one slice more, which does what is done once per sequence (the windows carried out).
struct ConvBlock {
    int64_t channels, chunks, row;
};
__device__ __forceinline__ ConvBlock conv_block(const ConvArgs &p) {
    const int64_t i = blockIdx.x, rest = i / p.channel_blocks;
    return {i - rest * p.channel_blocks, rest % p.chunk_blocks, rest / p.chunk_blocks};
}

template <typename io_t, int V, int W>
__global__ void __launch_bounds__(kConvWarps * 32) conv_cl_fwd_kernel(const __grid_constant__ ConvArgs p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const ConvBlock at = conv_block(p);
    const int64_t c = (at.channels * 32 + lane) * V;
    const bool live = c < p.channels;
    if (at.row == p.rows) {
        if (live && p.state_out != nullptr)
            for (int64_t s = at.chunks * kConvWarps + warp; s < p.seq.count; s += p.chunk_blocks * kConvWarps)
                store_window<io_t, V, W>(p, s, c);
        return;
    }
    const int64_t row = at.row;
    int64_t t = (at.chunks * kConvWarps + warp) * kConvChunk;
    const int64_t t_end = t + kConvChunk < p.seq.steps ? t + kConvChunk : p.seq.steps;
    if (t >= t_end) return;
    int64_t s = p.seq.offsets != nullptr ? find_sequence(p.seq, t, lane) : row;
    if (!live) return;
    float w[W][V], bias[V];
    load_taps<io_t, V, W>(p, c, w, bias);
    Span sp = span_of(p.seq, s);
    while (t < t_end) {
        const int64_t pos = t - sp.start;
        if (pos < 0 || pos >= sp.length) {
            // no step of this sequence: go to the next one that has steps, or fill with zeros
            int64_t upto = t_end;
            if (pos < 0) {
                upto = sp.start < t_end ? sp.start : t_end;
            } else if (p.seq.offsets != nullptr && s + 1 < p.seq.count) {
                sp = span_of(p.seq, ++s);
                continue;
            }
            const float zero[V] = {};
            for (; t < upto; ++t) store_lump<io_t, V>(p.out, row * p.out.sn + c * p.out.sc + t * p.out.st, 405, zero);
            continue;
        }
        const int64_t end = sp.start + sp.length < t_end ? sp.start + sp.length : t_end;
        float win[W - 1][V];
#pragma unroll
        for (int i = 0; i < W - 1; ++i) input_at<io_t, V, W>(p, sp, s, pos - (W - 1) + i, c, win[i]);
        constexpr int kAhead = 8;  // loads in flight
        for (; t < end; t += kAhead) {
            Lump<io_t, V> in[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (t + k < end) in[k] = load_lump<io_t, V>(p.x, row * p.x.sn + c * p.x.sc + (t + k) * p.x.st, 400);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (t + k < end) {
                    float v[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        v[i] = bias[i];
#pragma unroll
                        for (int j = 0; j < W - 1; ++j) v[i] = fmaf(w[j][i], win[j][i], v[i]);
                        v[i] = fmaf(w[W - 1][i], in[k].v[i], v[i]);
                        if (p.silu) v[i] *= logistic(v[i]);
#pragma unroll
                        for (int j = 0; j + 1 < W - 1; ++j) win[j][i] = win[j + 1][i];
                        win[W - 2][i] = in[k].v[i];
                    }
                    store_lump<io_t, V>(p.out, row * p.out.sn + c * p.out.sc + (t + k) * p.out.st, 405, v);
                }
            }
        }
        t = end;
    }
}

// d/dv of v or silu(v)
__device__ __forceinline__ float activation_slope(float v, int silu) {
    if (!silu) return 1.0f;
    const float g = logistic(v);
    return g * fmaf(v, 1.0f - g, 1.0f);
}

template <typename io_t, int W>
__device__ __forceinline__ float carried_gradient(const ConvArgs &p, const ConvGradArgs &q, const Span &sp, int64_t s, int64_t pos, int64_t c) {
    // the input at `pos` is also entry pos - (length - (W-1)) of the window carried out
    const int64_t i = pos - (sp.length - (W - 1));
    if (q.gstate_out == nullptr || i < 0) return 0.0f;
    return load_one(static_cast<const io_t *>(q.gstate_out), (s * p.channels + c) * (W - 1) + i, p.seq.count * p.channels * (W - 1), 410);
}

// A warp walks its chunk [t, b) and W-1 steps more: the gradient of step u's input is complete once
// gv of step u + W-1 is known.  The sums over steps stay in registers, are added over the warps of
// the CTA in shared memory and written as one part per CTA.
template <typename io_t, int V, int W>
__global__ void __launch_bounds__(kConvWarps * 32) conv_cl_bwd_kernel(const __grid_constant__ ConvArgs p,
                                                                      const __grid_constant__ ConvGradArgs q) {
    __shared__ float sums[kConvWarps][(W + 1) * V][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const ConvBlock at = conv_block(p);
    const int64_t c = (at.channels * 32 + lane) * V;
    const bool live = c < p.channels;
    if (at.row == p.rows) {  // sequences without steps hand the window's gradient through
        if (live && q.gstate != nullptr)
            for (int64_t s = at.chunks * kConvWarps + warp; s < p.seq.count; s += p.chunk_blocks * kConvWarps) {
                const Span sp = span_of(p.seq, s);
                if (sp.length == 0)
                    for (int k = 0; k < V; ++k)
                        for (int i = 0; i < W - 1; ++i)
                            store_one(static_cast<io_t *>(q.gstate), (s * p.channels + c + k) * (W - 1) + i,
                                      p.seq.count * p.channels * (W - 1), 411, carried_gradient<io_t, W>(p, q, sp, s, i - (W - 1), c + k));
            }
        return;
    }
    const int64_t row = at.row;
    int64_t t = (at.chunks * kConvWarps + warp) * kConvChunk;
    const int64_t t_end = t + kConvChunk < p.seq.steps ? t + kConvChunk : p.seq.steps;
    float gw[W + 1][V];
#pragma unroll
    for (int i = 0; i <= W; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) gw[i][k] = 0.0f;
    if (t < t_end) {
        int64_t s = p.seq.offsets != nullptr ? find_sequence(p.seq, t, lane) : row;
        if (live) {
            float w[W][V], bias[V];
            load_taps<io_t, V, W>(p, c, w, bias);
            Span sp = span_of(p.seq, s);
            while (t < t_end) {
                const int64_t pos = t - sp.start;
                if (pos < 0 || pos >= sp.length) {
                    int64_t upto = t_end;
                    if (pos < 0) {
                        upto = sp.start < t_end ? sp.start : t_end;
                    } else if (p.seq.offsets != nullptr && s + 1 < p.seq.count) {
                        sp = span_of(p.seq, ++s);
                        continue;
                    }
                    const float zero[V] = {};
                    for (; t < upto; ++t) store_lump<io_t, V>(q.gx, row * q.gx.sn + c * q.gx.sc + t * q.gx.st, 412, zero);
                    continue;
                }
                const int64_t a = t, seq_end = sp.start + sp.length, b = seq_end < t_end ? seq_end : t_end;
                float win[W - 1][V], part[W - 1][V];  // part[i]: gradient so far of the input W-1-i steps back
#pragma unroll
                for (int i = 0; i < W - 1; ++i) {
                    input_at<io_t, V, W>(p, sp, s, pos - (W - 1) + i, c, win[i]);
#pragma unroll
                    for (int k = 0; k < V; ++k) part[i][k] = 0.0f;
                }
                constexpr int kAhead = 4;
                const int64_t last = b + W - 1;
                for (; t < last; t += kAhead) {
                    Lump<io_t, V> in[kAhead], up[kAhead];
#pragma unroll
                    for (int k = 0; k < kAhead; ++k) {
                        if (t + k < last && t + k < seq_end) {
                            in[k] = load_lump<io_t, V>(p.x, row * p.x.sn + c * p.x.sc + (t + k) * p.x.st, 400);
                            up[k] = load_lump<io_t, V>(q.gout, row * q.gout.sn + c * q.gout.sc + (t + k) * q.gout.st, 413);
                        } else {
#pragma unroll
                            for (int i = 0; i < V; ++i) in[k].v[i] = up[k].v[i] = 0.0f;
                        }
                    }
#pragma unroll
                    for (int k = 0; k < kAhead; ++k) {
                        const int64_t now = t + k;
                        if (now < last) {
                            float done[V];
#pragma unroll
                            for (int i = 0; i < V; ++i) {
                                float v = bias[i];
#pragma unroll
                                for (int j = 0; j < W - 1; ++j) v = fmaf(w[j][i], win[j][i], v);
                                v = fmaf(w[W - 1][i], in[k].v[i], v);
                                const float gv = now < seq_end ? up[k].v[i] * activation_slope(v, p.silu) : 0.0f;
                                if (now < b) {
#pragma unroll
                                    for (int j = 0; j < W - 1; ++j) gw[j][i] = fmaf(gv, win[j][i], gw[j][i]);
                                    gw[W - 1][i] = fmaf(gv, in[k].v[i], gw[W - 1][i]);
                                    gw[W][i] += gv;
                                }
                                done[i] = fmaf(w[0][i], gv, part[0][i]);
#pragma unroll
                                for (int j = 0; j + 1 < W - 1; ++j) part[j][i] = fmaf(w[j + 1][i], gv, part[j + 1][i]);
                                part[W - 2][i] = w[W - 1][i] * gv;
#pragma unroll
                                for (int j = 0; j + 1 < W - 1; ++j) win[j][i] = win[j + 1][i];
                                win[W - 2][i] = in[k].v[i];
                            }
                            const int64_t u = now - (W - 1);  // the input whose gradient is complete
                            if (u >= a || (a == sp.start && q.gstate != nullptr)) {
                                const int64_t at_pos = u - sp.start;
                                if (at_pos >= sp.length - (W - 1)) {
#pragma unroll
                                    for (int i = 0; i < V; ++i) done[i] += carried_gradient<io_t, W>(p, q, sp, s, at_pos, c + i);
                                }
                                if (u >= a) {
                                    store_lump<io_t, V>(q.gx, row * q.gx.sn + c * q.gx.sc + u * q.gx.st, 412, done);
                                } else {
#pragma unroll
                                    for (int i = 0; i < V; ++i)
                                        store_one(static_cast<io_t *>(q.gstate), (s * p.channels + c + i) * (W - 1) + W - 1 + at_pos,
                                                  p.seq.count * p.channels * (W - 1), 411, done[i]);
                                }
                            }
                        }
                    }
                }
                t = b;
            }
        }
    }
#pragma unroll
    for (int i = 0; i <= W; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) sums[warp][i * V + k][lane] = gw[i][k];
    __syncthreads();
    const int64_t part = at.row * p.chunk_blocks + at.chunks, parts = p.rows * p.chunk_blocks;
    for (int i = threadIdx.x; i < (W + 1) * V * 32; i += blockDim.x) {
        const int tap = i % (W + 1), cc = i / (W + 1);  // cc: channel within the block
        const int64_t ch = at.channels * 32 * V + cc;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < kConvWarps; ++k) v += sums[k][tap * V + cc % V][cc / V];
        if (ch < p.channels) store_one(q.part, (part * p.channels + ch) * (W + 1) + tap, parts * p.channels * (W + 1), 414, v);
    }
}

// ---- rows: time adjacent ---------------------------------------------------------------------------
// Warp = one row; lane = 8 adjacent steps of a 256-step tile.  Any strides; one sequence a row.
template <typename io_t, int N>
__device__ __forceinline__ void load_steps(const View3 &v, int64_t base, int64_t t, int64_t from, int64_t to, int site, float (&r)[N]) {
    // r[i] = step t + i where it lies in [from, to), else 0
    const io_t *p = static_cast<const io_t *>(v.data);
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = t + i >= from && t + i < to ? load_one(p, base + (t + i) * v.st, v.extent, site) : 0.0f;
}

template <typename io_t, int W>
__global__ void __launch_bounds__(kConvWarps * 32) conv_rows_fwd_kernel(const __grid_constant__ ConvArgs p) {
    const int lane = threadIdx.x & 31;
    const ConvBlock at = conv_block(p);
    const int64_t c = at.channels * kConvWarps + (threadIdx.x >> 5), row = at.row;
    if (c >= p.channels) return;
    float w[W][1], bias[1];
    load_taps<io_t, 1, W>(p, c, w, bias);
    const Span sp = span_of(p.seq, row);
    const int64_t x0 = row * p.x.sn + c * p.x.sc, o0 = row * p.out.sn + c * p.out.sc;
    for (int64_t t = (at.chunks * 32 + lane) * kRun; t < p.seq.steps; t += p.chunk_blocks * 32 * kRun) {
        float in[kRun + W - 1], edge[1];
        load_steps<io_t>(p.x, x0, t - (W - 1), 0, sp.length, 420, in);
#pragma unroll
        for (int i = 0; i < W - 1; ++i)
            if (t - (W - 1) + i < 0) {
                input_at<io_t, 1, W>(p, sp, row, t - (W - 1) + i, c, edge);
                in[i] = edge[0];
            }
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            float v = bias[0];
#pragma unroll
            for (int j = 0; j < W; ++j) v = fmaf(w[j][0], in[k + j], v);
            if (p.silu) v *= logistic(v);
            if (t + k < p.seq.steps)
                store_one(static_cast<io_t *>(p.out.data), o0 + (t + k) * p.out.st, p.out.extent, 421, t + k < sp.length ? v : 0.0f);
        }
    }
    if (at.chunks == 0 && lane == 0 && p.state_out != nullptr) store_window<io_t, 1, W>(p, row, c);
}

template <typename io_t, int W>
__global__ void __launch_bounds__(kConvWarps * 32) conv_rows_bwd_kernel(const __grid_constant__ ConvArgs p,
                                                                        const __grid_constant__ ConvGradArgs q) {
    const int lane = threadIdx.x & 31;
    const ConvBlock at = conv_block(p);
    const int64_t c = at.channels * kConvWarps + (threadIdx.x >> 5), row = at.row;
    if (c >= p.channels) return;
    float w[W][1], bias[1], gw[W + 1];
    load_taps<io_t, 1, W>(p, c, w, bias);
#pragma unroll
    for (int i = 0; i <= W; ++i) gw[i] = 0.0f;
    const Span sp = span_of(p.seq, row);
    const int64_t x0 = row * p.x.sn + c * p.x.sc, g0 = row * q.gout.sn + c * q.gout.sc, o0 = row * q.gx.sn + c * q.gx.sc;
    for (int64_t t = (at.chunks * 32 + lane) * kRun; t < p.seq.steps; t += p.chunk_blocks * 32 * kRun) {
        float in[kRun + 2 * (W - 1)], gv[kRun + W - 1], edge[1];
        load_steps<io_t>(p.x, x0, t - (W - 1), 0, sp.length, 420, in);
        load_steps<io_t>(q.gout, g0, t, 0, sp.length, 422, gv);
#pragma unroll
        for (int i = 0; i < W - 1; ++i)
            if (t - (W - 1) + i < 0) {
                input_at<io_t, 1, W>(p, sp, row, t - (W - 1) + i, c, edge);
                in[i] = edge[0];
            }
#pragma unroll
        for (int k = 0; k < kRun + W - 1; ++k) {
            float v = bias[0];
#pragma unroll
            for (int j = 0; j < W; ++j) v = fmaf(w[j][0], in[k + j], v);
            gv[k] = t + k < sp.length ? gv[k] * activation_slope(v, p.silu) : 0.0f;
            if (k < kRun) {
#pragma unroll
                for (int j = 0; j < W; ++j) gw[j] = fmaf(gv[k], in[k + j], gw[j]);
                gw[W] += gv[k];
            }
        }
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            float v = 0.0f;
#pragma unroll
            for (int j = 0; j < W; ++j) v = fmaf(w[j][0], gv[k + W - 1 - j], v);
            if (t + k < sp.length) {
                if (t + k >= sp.length - (W - 1)) v += carried_gradient<io_t, W>(p, q, sp, row, t + k, c);
            } else {
                v = 0.0f;
            }
            if (t + k < p.seq.steps) store_one(static_cast<io_t *>(q.gx.data), o0 + (t + k) * q.gx.st, q.gx.extent, 423, v);
        }
        if (t == 0 && q.gstate != nullptr) {  // the carried window's inputs: step u = -(W-1) + i meets gv of steps 0 .. u + W-1
#pragma unroll
            for (int i = 0; i < W - 1; ++i) {
                float v = carried_gradient<io_t, W>(p, q, sp, row, i - (W - 1), c);
#pragma unroll
                for (int j = 0; j <= i; ++j) v = fmaf(w[j][0], gv[i - j], v);
                store_one(static_cast<io_t *>(q.gstate), (row * p.channels + c) * (W - 1) + i, p.seq.count * p.channels * (W - 1), 411, v);
            }
        }
    }
    if (p.seq.steps == 0 && q.gstate != nullptr && at.chunks == 0 && lane == 0) {
#pragma unroll
        for (int i = 0; i < W - 1; ++i)
            store_one(static_cast<io_t *>(q.gstate), (row * p.channels + c) * (W - 1) + i, p.seq.count * p.channels * (W - 1), 411,
                      carried_gradient<io_t, W>(p, q, sp, row, i - (W - 1), c));
    }
    const int64_t part = row * p.chunk_blocks + at.chunks, parts = p.rows * p.chunk_blocks;
#pragma unroll
    for (int i = 0; i <= W; ++i) {
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) gw[i] += __shfl_xor_sync(kFullMask, gw[i], d);
        if (lane == 0) store_one(q.part, (part * p.channels + c) * (W + 1) + i, parts * p.channels * (W + 1), 414, gw[i]);
    }
}

// Adds the parts in the order of their numbers; weight and bias gradients in the weight's type.
template <typename io_t>
__global__ void __launch_bounds__(256) conv_reduce_kernel(const float *part, int64_t parts, int64_t channels, int width, int weight_f32,
                                                          void *gweight, void *gbias) {
    const int64_t total = channels * (width + 1);
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t c = i / (width + 1);
        const int tap = (int)(i - c * (width + 1));
        float v = 0.0f;
#pragma unroll 8
        for (int64_t j = 0; j < parts; ++j) v += load_one(part, j * total + i, parts * total, 415);
        void *to = tap < width ? gweight : gbias;
        const int64_t at = tap < width ? c * width + tap : c, extent = tap < width ? channels * width : channels;
        if (to == nullptr) continue;
        if (weight_f32) store_one(static_cast<float *>(to), at, extent, 416, v);
        else store_one(static_cast<io_t *>(to), at, extent, 416, v);
    }
}

}  // namespace ssb
