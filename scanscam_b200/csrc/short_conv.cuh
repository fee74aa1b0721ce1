// Short causal convolution per channel: v_t = bias + sum_j w[j] x_{t-W+1+j}, out = v or silu(v), for
// widths 2, 3 and 4, and its backward.  What lies before a sequence's first step is the window
// carried in (the last W-1 inputs of the piece before, oldest first), or zero.
//
// The floor: 2 tensors forward, 3 more backward.  Channels last, [8, 4096, 2048] in bf16 with 4 taps: 73 us forward (41 for the bytes), where
// 14 warps an SM wait for their loads, and 141 backward (61), where instructions count (160 a warp for 4 channels and a step).
// Two forms:
//   channels last   a thread owns V adjacent channels (one 8- or 16-byte access per step) and walks
//                   a chunk of steps with its window in registers; the steps before its chunk are read again;
//   rows            a warp owns a row; a lane takes 8 adjacent steps, element by element, and reads its neighbours' few from cache
//                   ([3, 515, 1001] fp32, 3 taps: 14 + 20 us, 1.9 + 2.8 for the bytes).
#pragma once

#include "ssm_common.cuh"
#include "ssm_step.cuh"

namespace ssb {

struct ConvArgs {
    int64_t channels, rows, channel_blocks, chunk_blocks;
    int silu, weight_f32, chunk;  // chunk: steps that a warp of the channels-last kernels walks
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

struct True { static constexpr bool value = true; };
struct False { static constexpr bool value = false; };

constexpr int kConvWarps = 8;

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

// V adjacent channels of one step (4 or 1), as fetched and as pairs.
template <typename io_t, int V>
struct Lump {
    static constexpr int kPairs = (V + 1) / 2, kWords = V == 1 ? 1 : V * (int)sizeof(io_t) / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void open(pair_t (&f)[kPairs]) const {
        if constexpr (V == 1) {
            float v;
            if constexpr (sizeof(io_t) == 4) {
                v = __uint_as_float(w[0]);
            } else {
                float unused;
                unpack2<io_t>(w[0], v, unused);
            }
            f[0] = make_pair(v, 0.0f);
        } else {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                if constexpr (sizeof(io_t) == 4) {
                    f[i] = make_pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
                } else {
                    float lo, hi;
                    unpack2<io_t>(w[i], lo, hi);
                    f[i] = make_pair(lo, hi);
                }
            }
        }
    }
};
template <typename io_t, int V>
__device__ __forceinline__ Lump<io_t, V> load_lump(const View3 &v, int64_t at, int site) {
    Lump<io_t, V> r;
    const io_t *p = static_cast<const io_t *>(v.data) + at;
#pragma unroll
    for (int i = 0; i < Lump<io_t, V>::kWords; ++i) r.w[i] = 0;
    if (!SSB_VECTOR_OK(p, V * (int)sizeof(io_t), at + V - 1, v.extent, site)) return r;
    if constexpr (V == 1) {
        if constexpr (sizeof(io_t) == 4) r.w[0] = *reinterpret_cast<const uint32_t *>(p);
        else r.w[0] = *reinterpret_cast<const uint16_t *>(p);
    } else if constexpr (sizeof(io_t) == 4) {
        const uint4 f = *reinterpret_cast<const uint4 *>(p);
        r.w[0] = f.x; r.w[1] = f.y; r.w[2] = f.z; r.w[3] = f.w;
    } else {
        const uint2 f = *reinterpret_cast<const uint2 *>(p);
        r.w[0] = f.x; r.w[1] = f.y;
    }
    return r;
}
template <typename io_t, int V>
__device__ __forceinline__ void store_lump(const View3 &v, int64_t at, int site, const pair_t (&f)[(V + 1) / 2]) {
    io_t *p = static_cast<io_t *>(v.data) + at;
    if (!SSB_VECTOR_OK(p, V * (int)sizeof(io_t), at + V - 1, v.extent, site)) return;
    const float2 a = halves(f[0]);
    if constexpr (V == 1) {
        *p = static_cast<io_t>(a.x);
    } else {
        const float2 b = halves(f[1]);
        if constexpr (sizeof(io_t) == 4) *reinterpret_cast<float4 *>(p) = make_float4(a.x, a.y, b.x, b.y);
        else *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<io_t>(a.x, a.y), pack2<io_t>(b.x, b.y));
    }
}
// channel i of V
template <int N>
__device__ __forceinline__ float channel_of(const pair_t (&f)[N], int i) {
    const float2 h = halves(f[i / 2]);
    return i & 1 ? h.y : h.x;
}

// Step `pos` (relative to the sequence's start; below zero: in the carried window) of V channels.
template <typename io_t, int V, int W>
__device__ __forceinline__ void input_at(const ConvArgs &p, const Span &sp, int64_t s, int64_t pos, int64_t c, pair_t (&r)[(V + 1) / 2]) {
    if (pos >= 0) {
        load_lump<io_t, V>(p.x, sp.row * p.x.sn + c * p.x.sc + (sp.start + pos) * p.x.st, 400).open(r);
    } else {
        float f[V + 1] = {};
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (p.state != nullptr)
                f[i] = load_one(static_cast<const io_t *>(p.state), (s * p.channels + c + i) * (W - 1) + W - 1 + pos,
                                p.seq.count * p.channels * (W - 1), 401);
#pragma unroll
        for (int i = 0; i < (V + 1) / 2; ++i) r[i] = make_pair(f[2 * i], f[2 * i + 1]);
    }
}

// The window behind a sequence's last step.
template <typename io_t, int V, int W>
__device__ __forceinline__ void store_window(const ConvArgs &p, int64_t s, int64_t c) {
    const Span sp = span_of(p.seq, s);
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        pair_t r[(V + 1) / 2];
        input_at<io_t, V, W>(p, sp, s, sp.length - (W - 1) + i, c, r);
#pragma unroll
        for (int k = 0; k < V; ++k)
            store_one(static_cast<io_t *>(p.state_out), (s * p.channels + c + k) * (W - 1) + i, p.seq.count * p.channels * (W - 1), 402,
                      channel_of(r, k));
    }
}

template <typename io_t, int V, int W>
__device__ __forceinline__ void load_taps(const ConvArgs &p, int64_t c, pair_t (&w)[W][(V + 1) / 2], pair_t (&bias)[(V + 1) / 2]) {
    float f[W + 1][V + 1] = {};
#pragma unroll
    for (int k = 0; k < V; ++k) {
#pragma unroll
        for (int i = 0; i < W; ++i) f[i][k] = load_weight<io_t>(p.weight, p.weight_f32, (c + k) * W + i, p.channels * W, 403);
        if (p.bias != nullptr) f[W][k] = load_weight<io_t>(p.bias, p.weight_f32, c + k, p.channels, 404);
    }
#pragma unroll
    for (int k = 0; k < (V + 1) / 2; ++k) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i][k] = make_pair(f[i][2 * k], f[i][2 * k + 1]);
        bias[k] = make_pair(f[W][2 * k], f[W][2 * k + 1]);
    }
}

__device__ __forceinline__ pair_t logistic2(pair_t v) {
    const float2 x = halves(mul2(v, both(-kLog2e)));
    const float2 d = halves(add2(make_pair(exp2_approx(x.x), exp2_approx(x.y)), both(1.0f)));
    return make_pair(reciprocal_approx(d.x), reciprocal_approx(d.y));
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
__global__ void __launch_bounds__(kConvWarps * 32, 2) conv_cl_fwd_kernel(const __grid_constant__ ConvArgs p) {
    constexpr int N = (V + 1) / 2;
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
    int64_t t = (at.chunks * kConvWarps + warp) * p.chunk;
    const int64_t t_end = t + p.chunk < p.seq.steps ? t + p.chunk : p.seq.steps;
    if (t >= t_end) return;
    int64_t s = p.seq.offsets != nullptr ? find_sequence(p.seq, t, lane) : row;
    if (!live) return;
    const int64_t x0 = row * p.x.sn + c * p.x.sc, o0 = row * p.out.sn + c * p.out.sc;
    pair_t w[W][N], bias[N];
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
            const pair_t zero[N] = {};
            for (; t < upto; ++t) store_lump<io_t, V>(p.out, o0 + t * p.out.st, 405, zero);
            continue;
        }
        constexpr int kAhead = 8;  // steps whose loads are in flight while the 8 before are worked on
        const int64_t end = sp.start + sp.length < t_end ? sp.start + sp.length : t_end;
        Lump<io_t, V> in[kAhead], next[kAhead];
        const auto fetch = [&](int64_t from, Lump<io_t, V> (&to)[kAhead]) {
            const int n = (int)(end - from);
            int64_t at = x0 + from * p.x.st;
#pragma unroll
            for (int k = 0; k < kAhead; ++k, at += p.x.st)
                if (k < n) to[k] = load_lump<io_t, V>(p.x, at, 400);
        };
        fetch(t, in);
        pair_t win[W - 1][N];
#pragma unroll
        for (int i = 0; i < W - 1; ++i) input_at<io_t, V, W>(p, sp, s, pos - (W - 1) + i, c, win[i]);
        for (; t < end; t += kAhead) {
            fetch(t + kAhead, next);
            const int n = (int)(end - t);
            const auto group = [&](auto whole) {  // whole: all 8 steps exist, and nothing is asked per step
                int64_t to = o0 + t * p.out.st;
#pragma unroll
                for (int k = 0; k < kAhead; ++k, to += p.out.st) {
                    if (decltype(whole)::value || k < n) {
                        pair_t x[N], v[N];
                        in[k].open(x);
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            v[i] = bias[i];
#pragma unroll
                            for (int j = 0; j < W - 1; ++j) v[i] = fma2(w[j][i], win[j][i], v[i]);
                            v[i] = fma2(w[W - 1][i], x[i], v[i]);
                            if (p.silu) v[i] = mul2(v[i], logistic2(v[i]));
#pragma unroll
                            for (int j = 0; j + 1 < W - 1; ++j) win[j][i] = win[j + 1][i];
                            win[W - 2][i] = x[i];
                        }
                        store_lump<io_t, V>(p.out, to, 405, v);
                    }
                }
            };
            if (n >= kAhead) group(True{});
            else group(False{});
#pragma unroll
            for (int k = 0; k < kAhead; ++k) in[k] = next[k];
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
__global__ void __launch_bounds__(kConvWarps * 32, 2) conv_cl_bwd_kernel(const __grid_constant__ ConvArgs p,
                                                                         const __grid_constant__ ConvGradArgs q) {
    constexpr int N = (V + 1) / 2;
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
    int64_t t = (at.chunks * kConvWarps + warp) * p.chunk;
    const int64_t t_end = t + p.chunk < p.seq.steps ? t + p.chunk : p.seq.steps;
    pair_t gw[W + 1][N];
#pragma unroll
    for (int i = 0; i <= W; ++i)
#pragma unroll
        for (int k = 0; k < N; ++k) gw[i][k] = 0;
    if (t < t_end) {
        int64_t s = p.seq.offsets != nullptr ? find_sequence(p.seq, t, lane) : row;
        if (live) {
            const int64_t x0 = row * p.x.sn + c * p.x.sc, g0 = row * q.gout.sn + c * q.gout.sc, o0 = row * q.gx.sn + c * q.gx.sc;
            pair_t w[W][N], bias[N];
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
                    const pair_t zero[N] = {};
                    for (; t < upto; ++t) store_lump<io_t, V>(q.gx, o0 + t * q.gx.st, 412, zero);
                    continue;
                }
                constexpr int kAhead = 4;
                const int64_t a = t, seq_end = sp.start + sp.length, b = seq_end < t_end ? seq_end : t_end;
                Lump<io_t, V> in[kAhead], up[kAhead], next_in[kAhead], next_up[kAhead];
                const auto fetch = [&](int64_t from, Lump<io_t, V> (&x)[kAhead], Lump<io_t, V> (&g)[kAhead]) {
                    const int n = (int)((b + W - 1 < seq_end ? b + W - 1 : seq_end) - from);
                    int64_t at_x = x0 + from * p.x.st, at_g = g0 + from * q.gout.st;
#pragma unroll
                    for (int k = 0; k < kAhead; ++k, at_x += p.x.st, at_g += q.gout.st) {
                        if (k < n) {
                            x[k] = load_lump<io_t, V>(p.x, at_x, 400);
                            g[k] = load_lump<io_t, V>(q.gout, at_g, 413);
                        } else {
#pragma unroll
                            for (int i = 0; i < Lump<io_t, V>::kWords; ++i) x[k].w[i] = g[k].w[i] = 0;
                        }
                    }
                };
                fetch(t, in, up);
                pair_t win[W - 1][N], part[W - 1][N];  // part[i]: gradient so far of the input W-1-i steps back
#pragma unroll
                for (int i = 0; i < W - 1; ++i) {
                    input_at<io_t, V, W>(p, sp, s, pos - (W - 1) + i, c, win[i]);
#pragma unroll
                    for (int k = 0; k < N; ++k) part[i][k] = 0;
                }
                const int64_t last = b + W - 1;
                for (; t < last; t += kAhead) {
                    fetch(t + kAhead, next_in, next_up);
                    const int n_last = (int)(last - t), n_b = (int)(b - t), n_seq = (int)(seq_end - t < kAhead ? seq_end - t : kAhead);
                    const bool inner = t - (W - 1) >= a && n_b >= kAhead && n_seq >= kAhead && q.gstate_out == nullptr;
                    const auto group = [&](auto whole) {  // whole: the group lies inside the chunk, and nothing is asked per step
                        constexpr bool kWhole = decltype(whole)::value;
                        int64_t to = o0 + (t - (W - 1)) * q.gx.st;
#pragma unroll
                        for (int k = 0; k < kAhead; ++k, to += q.gx.st) {
                            if (kWhole || k < n_last) {
                                pair_t x[N], g[N], done[N];
                                in[k].open(x);
                                up[k].open(g);
#pragma unroll
                                for (int i = 0; i < N; ++i) {
                                    pair_t gv = g[i];
                                    if (p.silu) {
                                        pair_t v = bias[i];
#pragma unroll
                                        for (int j = 0; j < W - 1; ++j) v = fma2(w[j][i], win[j][i], v);
                                        v = fma2(w[W - 1][i], x[i], v);
                                        const pair_t l = logistic2(v);
                                        // silu'(v) = l (1 + v (1 - l))
                                        gv = mul2(gv, mul2(l, fma2(v, fma2(l, both(-1.0f), both(1.0f)), both(1.0f))));
                                    }
                                    if (!kWhole && k >= n_seq) gv = 0;
                                    if (kWhole || k < n_b) {
#pragma unroll
                                        for (int j = 0; j < W - 1; ++j) gw[j][i] = fma2(gv, win[j][i], gw[j][i]);
                                        gw[W - 1][i] = fma2(gv, x[i], gw[W - 1][i]);
                                        gw[W][i] = add2(gw[W][i], gv);
                                    }
                                    done[i] = fma2(w[0][i], gv, part[0][i]);
#pragma unroll
                                    for (int j = 0; j + 1 < W - 1; ++j) part[j][i] = fma2(w[j + 1][i], gv, part[j + 1][i]);
                                    part[W - 2][i] = mul2(w[W - 1][i], gv);
#pragma unroll
                                    for (int j = 0; j + 1 < W - 1; ++j) win[j][i] = win[j + 1][i];
                                    win[W - 2][i] = x[i];
                                }
                                const int64_t u = t + k - (W - 1);  // the input whose gradient is complete
                                if (kWhole) {
                                    store_lump<io_t, V>(q.gx, to, 412, done);
                                } else if (u >= a || (a == sp.start && q.gstate != nullptr)) {
                                    const int64_t at_pos = u - sp.start;
                                    if (q.gstate_out != nullptr && at_pos >= sp.length - (W - 1)) {
                                        float f[V + 1] = {};
#pragma unroll
                                        for (int i = 0; i < V; ++i) f[i] = carried_gradient<io_t, W>(p, q, sp, s, at_pos, c + i);
#pragma unroll
                                        for (int i = 0; i < N; ++i) done[i] = add2(done[i], make_pair(f[2 * i], f[2 * i + 1]));
                                    }
                                    if (u >= a) {
                                        store_lump<io_t, V>(q.gx, to, 412, done);
                                    } else {
#pragma unroll
                                        for (int i = 0; i < V; ++i)
                                            store_one(static_cast<io_t *>(q.gstate), (s * p.channels + c + i) * (W - 1) + W - 1 + at_pos,
                                                      p.seq.count * p.channels * (W - 1), 411, channel_of(done, i));
                                    }
                                }
                            }
                        }
                    };
                    if (inner) group(True{});
                    else group(False{});
#pragma unroll
                    for (int k = 0; k < kAhead; ++k) {
                        in[k] = next_in[k];
                        up[k] = next_up[k];
                    }
                }
                t = b;
            }
        }
    }
#pragma unroll
    for (int i = 0; i <= W; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) sums[warp][i * V + k][lane] = channel_of(gw[i], k);
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
    pair_t taps[W][1], bias[1];
    load_taps<io_t, 1, W>(p, c, taps, bias);
    const float b0 = halves(bias[0]).x;
    float w[W];
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = halves(taps[i][0]).x;
    const Span sp = span_of(p.seq, row);
    const int64_t x0 = row * p.x.sn + c * p.x.sc, o0 = row * p.out.sn + c * p.out.sc;
    for (int64_t t = (at.chunks * 32 + lane) * kRun; t < p.seq.steps; t += p.chunk_blocks * 32 * kRun) {
        float in[kRun + W - 1];
        pair_t edge[1];
        load_steps<io_t>(p.x, x0, t - (W - 1), 0, sp.length, 420, in);
#pragma unroll
        for (int i = 0; i < W - 1; ++i)
            if (t - (W - 1) + i < 0) {
                input_at<io_t, 1, W>(p, sp, row, t - (W - 1) + i, c, edge);
                in[i] = halves(edge[0]).x;
            }
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            float v = b0;
#pragma unroll
            for (int j = 0; j < W; ++j) v = fmaf(w[j], in[k + j], v);
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
    pair_t taps[W][1], bias[1];
    load_taps<io_t, 1, W>(p, c, taps, bias);
    const float b0 = halves(bias[0]).x;
    float w[W], gw[W + 1];
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = halves(taps[i][0]).x;
#pragma unroll
    for (int i = 0; i <= W; ++i) gw[i] = 0.0f;
    const Span sp = span_of(p.seq, row);
    const int64_t x0 = row * p.x.sn + c * p.x.sc, g0 = row * q.gout.sn + c * q.gout.sc, o0 = row * q.gx.sn + c * q.gx.sc;
    for (int64_t t = (at.chunks * 32 + lane) * kRun; t < p.seq.steps; t += p.chunk_blocks * 32 * kRun) {
        float in[kRun + 2 * (W - 1)], gv[kRun + W - 1];
        pair_t edge[1];
        load_steps<io_t>(p.x, x0, t - (W - 1), 0, sp.length, 420, in);
        load_steps<io_t>(q.gout, g0, t, 0, sp.length, 422, gv);
#pragma unroll
        for (int i = 0; i < W - 1; ++i)
            if (t - (W - 1) + i < 0) {
                input_at<io_t, 1, W>(p, sp, row, t - (W - 1) + i, c, edge);
                in[i] = halves(edge[0]).x;
            }
#pragma unroll
        for (int k = 0; k < kRun + W - 1; ++k) {
            float v = b0;
#pragma unroll
            for (int j = 0; j < W; ++j) v = fmaf(w[j], in[k + j], v);
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
            for (int j = 0; j < W; ++j) v = fmaf(w[j], gv[k + W - 1 - j], v);
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
                for (int j = 0; j <= i; ++j) v = fmaf(w[j], gv[i - j], v);
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
