// Device helpers of the state-space kernels: strided views, runs of steps in registers, pairs of
// channels in one 64-bit register, and the three functions (2^x, softplus, logistic) they use.
#pragma once

#include "scan_common.cuh"

namespace ssb {

// The checked build's test of an access of several elements: the last of them lies inside, and the
// address is a multiple of the access's size.
#ifdef SSB_CHECKED
__device__ __forceinline__ bool vector_in_range(const void *p, int bytes, int64_t last, int64_t extent, int site) {
    if (reinterpret_cast<uintptr_t>(p) % bytes == 0) return index_in_range(last, extent, site);
    report_device_check(site);
    return false;
}
#define SSB_VECTOR_OK(p, bytes, last, extent, site) ::ssb::vector_in_range((p), (bytes), (int64_t)(last), (int64_t)(extent), (site))
#else
#define SSB_VECTOR_OK(p, bytes, last, extent, site) true
#endif

typedef unsigned long long pair_t;  // two floats: the even channel in the low half

__device__ __forceinline__ pair_t make_pair(float lo, float hi) {
    pair_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ pair_t both(float v) { return make_pair(v, v); }
__device__ __forceinline__ float2 halves(pair_t p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
// Packed arithmetic: one issue slot for two results (the rate per result is that of the scalar
// forms: 2.2 cycles a warp instruction against 1.04, measured).
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) {
    pair_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b) {
    pair_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) {
    pair_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ pair_t shfl_up2(pair_t p, int delta) {
    const float2 f = halves(p);
    return make_pair(__shfl_up_sync(kFullMask, f.x, delta), __shfl_up_sync(kFullMask, f.y, delta));
}
__device__ __forceinline__ pair_t shfl_down2(pair_t p, int delta) {
    const float2 f = halves(p);
    return make_pair(__shfl_down_sync(kFullMask, f.x, delta), __shfl_down_sync(kFullMask, f.y, delta));
}

// Sums v[i] over LN neighbouring lanes; lane q of them is left with the sum of v[q mod STEPS].
template <int LN, int STEPS>
__device__ __forceinline__ float sum_and_spread(float (&v)[STEPS], int q) {
    static_assert(STEPS <= LN, "a lane is left with one sum");
#pragma unroll
    for (int half = STEPS / 2; half >= 1; half >>= 1) {
        const bool upper = (q & half) != 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float give = upper ? v[i] : v[i + half], keep = upper ? v[i + half] : v[i];
            v[i] = keep + __shfl_xor_sync(kFullMask, give, half);
        }
    }
#pragma unroll
    for (int d = STEPS; d < LN; d <<= 1) v[0] += __shfl_xor_sync(kFullMask, v[0], d);
    return v[0];
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Added to the exponents of decays.  The unit's results lie 2e-8 of the value too low on average where decays are
// slow (measured over [-0.1, -0.001]), which a state that remembers hundreds of steps adds up; a shift of the
// exponent takes most of it back for the price of a multiply that becomes a multiply-add, and is lost in the
// rounding of larger exponents, where nothing is remembered.  An exponent of zero still gives exactly 1.
// [4, 2048, 2048], 16 states: error of the states 2.6e-7 of the norm with it, 5.0e-7 without.
constexpr float kExponentShift = 2e-8f;

// 2^x on the special function unit: 8 cycles a warp instruction and sub-partition, error below
// 1.5e-7 of the value (measured over [-100, 0]; a bias of at most 5e-8).
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ pair_t exp2_pair(pair_t x) {
    const float2 f = halves(x);
    return make_pair(exp2_approx(f.x), exp2_approx(f.y));
}
// e^x without the error that rounding x * log2(e) would bring: the product's rounding error and log2(e)'s own
// tail are put back as a factor 1 + lo * ln 2.  Infinite from 88.7 up, where the factor, which may lie below 1, is left out.
__device__ __forceinline__ float exp_accurate(float x) {
    const float hi = x * kLog2e;
    const float lo = fmaf(x, 1.925963033500945e-8f, fmaf(x, kLog2e, -hi));
    const float e = exp2_approx(hi);
    return isfinite(e) ? fmaf(e, lo * kLn2, e) : e;
}
__device__ __forceinline__ float reciprocal_approx(float x) {  // 0 for infinity; one unit in the last place
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 1 / (1 + e^-x).  The plain form is off by up to |x| 2^-24 of the value where x is far below zero,
// which a gate x * logistic(x) does not feel; the derivative of softplus does (its arguments are
// around -5), and takes the other.
__device__ __forceinline__ float logistic(float x) { return reciprocal_approx(1.0f + exp2_approx(-x * kLog2e)); }
__device__ __forceinline__ float logistic_accurate(float x) { return __fdividef(1.0f, 1.0f + exp_accurate(-x)); }

__device__ __forceinline__ float relu_or_nan(float v) {
    float y;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(v));
    return y;
}
// log(1 + e^v) = max(v, 0) + log1p(e^-|v|).  log1p(e) = 2 atanh(s) with s = e / (2 + e) of at most 1/3;
// atanh(s) = s + s q P(q), q = s^2, where P is a cubic fitted (Chebyshev, weighted with q) to
// (atanh(s) / s - 1) / q on [0, 1/9]: 4.6e-9 of the value.  Below -87 the result stays at e^-87 = 1.6e-38,
// where the type's normal range ends.  The exponential as in exp_accurate.
__device__ __forceinline__ float softplus_and_slope(float v, float &slope) {  // the slope is 1 / (1 + e^-v)
    const float x = fmaxf(-fabsf(v), -87.0f);
    const float hi = x * kLog2e;
    const float lo = fmaf(x, 1.925963033500945e-8f, fmaf(x, kLog2e, -hi));
    float e = exp2_approx(hi);
    e = fmaf(e, lo * kLn2, e);
    slope = (v < 0.0f ? e : 1.0f) * reciprocal_approx(1.0f + e);
    const float s = e * reciprocal_approx(e + 2.0f), q = s * s;
    float p = fmaf(q, 0.13988047f, 0.14004979f);
    p = fmaf(p, q, 0.20010476f);
    p = fmaf(p, q, 0.33333215f);
    return fmaf(fmaf(p * q, s, s), 2.0f, relu_or_nan(v));
}
__device__ __forceinline__ float softplus(float v) {
    float slope;
    return softplus_and_slope(v, slope);
}
__device__ __forceinline__ pair_t softplus2(pair_t v) {
    const float2 f = halves(v);
    return make_pair(softplus(f.x), softplus(f.y));
}

// ---- views ------------------------------------------------------------------------------------
// How runs of 8 steps x 2 channels of a [N, C, T] view may be fetched:
//   kAnyStride   element by element;
//   kPairs       channels adjacent and pairs of them aligned: one access per step and pair;
//   kRuns        steps adjacent and runs of 8 aligned to 16 bytes: 16-byte accesses per channel.
enum Access : int { kAnyStride = 0, kPairs = 1, kRuns = 2 };

struct View3 {
    void *data;
    int64_t sn, sc, st;  // strides in elements
    int64_t extent;      // one past the largest element offset (the checked build's bound)
    int access;
};

template <typename io_t>
__device__ __forceinline__ float load_one(const io_t *base, int64_t at, int64_t extent, int site) {
    if (!SSB_INDEX_OK(at, extent, site)) return 0.0f;
    return static_cast<float>(base[at]);
}
template <typename io_t>
__device__ __forceinline__ void store_one(io_t *base, int64_t at, int64_t extent, int site, float v) {
    if (SSB_INDEX_OK(at, extent, site)) base[at] = static_cast<io_t>(v);
}

constexpr int kRun = 8;  // steps a thread holds of each of its two channels

// Steps t .. t+7 of channels c, c+1 of row n, as they lie in memory: fetched ahead of their use, opened
// into pairs when they are needed.  What lies behind `steps` steps or `channels` channels is zero and
// is not read.
template <typename io_t>
struct RawRun {
    static constexpr int kWords = kRun * 2 * (int)sizeof(io_t) / 4;
    uint32_t w[kWords];
    bool by_channel;  // words hold 8 steps of one channel, then of the other; else the pair of one step after the other
};

template <typename io_t>
__device__ __forceinline__ void fetch_run(const View3 &v, int64_t n, int64_t c, int64_t t, int steps, int channels, int site,
                                          RawRun<io_t> &r) {
    const io_t *base = static_cast<const io_t *>(v.data);
    const int64_t at = n * v.sn + c * v.sc + t * v.st;
#pragma unroll
    for (int k = 0; k < RawRun<io_t>::kWords; ++k) r.w[k] = 0;
    r.by_channel = false;
    if (v.access == kPairs && channels == 2) {
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const int64_t i = at + k * v.st;
            if (k < steps && SSB_VECTOR_OK(base + i, 2 * (int)sizeof(io_t), i + 1, v.extent, site)) {
                if constexpr (sizeof(io_t) == 2) {
                    r.w[k] = *reinterpret_cast<const uint32_t *>(base + i);
                } else {
                    const uint2 q = *reinterpret_cast<const uint2 *>(base + i);
                    r.w[2 * k] = q.x;
                    r.w[2 * k + 1] = q.y;
                }
            }
        }
    } else if (v.access == kRuns && channels == 2 && steps == kRun) {
        r.by_channel = true;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int64_t i = at + q * v.sc;
            if (!SSB_VECTOR_OK(base + i, 16, i + kRun - 1, v.extent, site)) continue;
#pragma unroll
            for (int k = 0; k < RawRun<io_t>::kWords / 8; ++k) {
                const uint4 f = reinterpret_cast<const uint4 *>(base + i)[k];
                uint32_t *w = r.w + q * (RawRun<io_t>::kWords / 2) + 4 * k;
                w[0] = f.x; w[1] = f.y; w[2] = f.z; w[3] = f.w;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int64_t i = at + k * v.st + q * v.sc;
                if (k < steps && q < channels && SSB_INDEX_OK(i, v.extent, site)) {
                    if constexpr (sizeof(io_t) == 2) r.w[k] |= (uint32_t)reinterpret_cast<const uint16_t *>(base)[i] << (16 * q);
                    else r.w[2 * k + q] = reinterpret_cast<const uint32_t *>(base)[i];
                }
            }
        }
    }
}

template <typename io_t>
__device__ __forceinline__ void open_run(const RawRun<io_t> &raw, pair_t (&r)[kRun]) {
    if constexpr (sizeof(io_t) == 2) {
        if (raw.by_channel) {
#pragma unroll
            for (int k = 0; k < kRun / 2; ++k) {
                float a, b, c, d;
                unpack2<io_t>(raw.w[k], a, b);
                unpack2<io_t>(raw.w[kRun / 2 + k], c, d);
                r[2 * k] = make_pair(a, c);
                r[2 * k + 1] = make_pair(b, d);
            }
        } else {
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                float a, b;
                unpack2<io_t>(raw.w[k], a, b);
                r[k] = make_pair(a, b);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < kRun; ++k)
            r[k] = raw.by_channel ? make_pair(__uint_as_float(raw.w[k]), __uint_as_float(raw.w[kRun + k]))
                                  : make_pair(__uint_as_float(raw.w[2 * k]), __uint_as_float(raw.w[2 * k + 1]));
    }
}

template <typename io_t>
__device__ __forceinline__ void load_run(const View3 &v, int64_t n, int64_t c, int64_t t, int steps, int channels,
                                         int site, pair_t (&r)[kRun]) {
    RawRun<io_t> raw;
    fetch_run(v, n, c, t, steps, channels, site, raw);
    open_run(raw, r);
}

template <typename io_t>
__device__ __forceinline__ void store_run(const View3 &v, int64_t n, int64_t c, int64_t t, int steps, int channels,
                                          int site, const pair_t (&r)[kRun]) {
    io_t *base = static_cast<io_t *>(v.data);
    const int64_t at = n * v.sn + c * v.sc + t * v.st;
    if (v.access == kPairs && channels == 2) {
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const int64_t i = at + k * v.st;
            if (k < steps && SSB_VECTOR_OK(base + i, 2 * (int)sizeof(io_t), i + 1, v.extent, site)) {
                if constexpr (sizeof(io_t) == 2) {
                    const float2 f = halves(r[k]);
                    *reinterpret_cast<uint32_t *>(base + i) = pack2<io_t>(f.x, f.y);
                } else {
                    *reinterpret_cast<pair_t *>(base + i) = r[k];
                }
            }
        }
    } else if (v.access == kRuns && channels == 2 && steps == kRun) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int64_t i = at + q * v.sc;
            float f[kRun];
#pragma unroll
            for (int k = 0; k < kRun; ++k) f[k] = q ? halves(r[k]).y : halves(r[k]).x;
            if (SSB_VECTOR_OK(base + i, 16, i + kRun - 1, v.extent, site)) {
                if constexpr (sizeof(io_t) == 2) {
                    *reinterpret_cast<uint4 *>(base + i) = make_uint4(pack2<io_t>(f[0], f[1]), pack2<io_t>(f[2], f[3]),
                                                                      pack2<io_t>(f[4], f[5]), pack2<io_t>(f[6], f[7]));
                } else {
                    *reinterpret_cast<float4 *>(base + i) = make_float4(f[0], f[1], f[2], f[3]);
                    *reinterpret_cast<float4 *>(base + i + 4) = make_float4(f[4], f[5], f[6], f[7]);
                }
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const float2 f = halves(r[k]);
            if (k < steps && channels > 0) store_one<io_t>(base, at + k * v.st, v.extent, site, f.x);
            if (k < steps && channels > 1) store_one<io_t>(base, at + k * v.st + v.sc, v.extent, site, f.y);
        }
    }
}

// ---- sequences ----------------------------------------------------------------------------------
// Packed: sequence s is steps offsets[s] .. offsets[s+1] of row 0.  Else sequence s is row s, all of
// it or its first lengths[s] steps.  What the device reads is cut to [0, T], so that offsets or
// lengths that are not what the caller promised give wrong numbers but no access outside.
struct Sequences {
    const int32_t *offsets, *lengths;
    int64_t count, steps;
};
struct Span {
    int64_t row, start, length;
};
__device__ __forceinline__ int64_t clamp_step(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }
__device__ __forceinline__ Span span_of(const Sequences &q, int64_t s) {
    if (q.offsets != nullptr) {
        const int64_t a = clamp_step(q.offsets[s], 0, q.steps), b = clamp_step(q.offsets[s + 1], a, q.steps);
        return {0, a, b - a};
    }
    return {s, 0, q.lengths != nullptr ? clamp_step(q.lengths[s], 0, q.steps) : q.steps};
}

}  // namespace ssb
