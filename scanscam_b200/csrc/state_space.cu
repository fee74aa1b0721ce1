// C-ABI entry points of the state-space operators: argument checks, choice of the kernel's shape,
// launches.  Kernels: ssm_forward.cuh, ssm_backward.cuh, ssm_scan.cuh, ssm_step.cuh, short_conv.cuh.
#include "../../include/scanscam_b200.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <limits>

#include "host_common.h"
#include "short_conv.cuh"
#include "ssm_backward.cuh"
#include "ssm_forward.cuh"
#include "ssm_scan.cuh"
#include "ssm_step.cuh"

using ssb_host::check_launch;
using ssb_host::fail;
using ssb_host::sm_count;

namespace {

constexpr int64_t kMaxStates = 256, kLaneBackwardStates = 32;
constexpr size_t kSmemLimit = 227 * 1024;

size_t size_of(int dtype) { return dtype == SSB_F32 ? 4 : 2; }
bool aligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Calls f with a null pointer of the storage type.
template <typename F>
int with_type(int dtype, F &&f) {
    if (dtype == SSB_F32) return f(static_cast<float *>(nullptr));
    if (dtype == SSB_BF16) return f(static_cast<__nv_bfloat16 *>(nullptr));
    return f(static_cast<__half *>(nullptr));
}

int check_sizes(int dtype, std::initializer_list<int64_t> sizes) {
    if (dtype != SSB_F32 && dtype != SSB_BF16 && dtype != SSB_F16) return fail(SSB_ERR_BAD_ARG, "unknown element type %d", dtype);
    int64_t all = 1;
    for (int64_t s : sizes) {
        if (s < 0) return fail(SSB_ERR_BAD_ARG, "negative size: %lld", (long long)s);
        if (s > 0 && all > std::numeric_limits<int64_t>::max() / 64 / s) return fail(SSB_ERR_BAD_ARG, "sizes overflow");
        if (s > 0) all *= s;
    }
    return SSB_OK;
}

int check_sequences(int64_t batch, int64_t sequences, const int32_t *offsets, const int32_t *lengths) {
    if (offsets == nullptr) return SSB_OK;
    if (lengths != nullptr) return fail(SSB_ERR_BAD_ARG, "offsets and lengths exclude each other");
    if (batch != 1) return fail(SSB_ERR_BAD_ARG, "packed sequences need a batch of 1, got %lld", (long long)batch);
    if (sequences < 1) return fail(SSB_ERR_BAD_ARG, "offsets must bound at least one sequence, got %lld", (long long)sequences);
    return SSB_OK;
}

ssb::Sequences sequences_of(int64_t batch, int64_t steps, int64_t sequences, const int32_t *offsets, const int32_t *lengths) {
    return {offsets, lengths, offsets != nullptr ? sequences : batch, steps};
}

int check_data(const void *p, int dtype, const char *name) {
    if (p == nullptr) return fail(SSB_ERR_BAD_ARG, "%s is NULL", name);
    if (!aligned(p, size_of(dtype))) return fail(SSB_ERR_ALIGNMENT, "%s is not aligned to its element size", name);
    return SSB_OK;
}

int64_t extent_of(const ssb_view_t &v, std::initializer_list<int64_t> sizes) {
    int64_t last = 0;
    int i = 0;
    for (int64_t s : sizes) last += (s - 1) * v.stride[i++];
    return last + 1;
}

// A [N, C, T] view and how runs of it may be fetched.  `from_zero`: every run starts at a multiple of
// 8 steps; `even`: every pair of channels starts at an even one (not so in groups of an odd size).
ssb::View3 view3(const ssb_view_t &v, int dtype, int64_t n, int64_t c, int64_t t, bool from_zero, bool even) {
    const size_t e = size_of(dtype);
    ssb::View3 r{v.data, v.stride[0], v.stride[1], v.stride[2], v.data != nullptr ? extent_of(v, {n, c, t}) : 0, ssb::kAnyStride};
    if (even && v.stride[1] == 1 && v.stride[2] % 2 == 0 && v.stride[0] % 2 == 0 && aligned(v.data, 2 * e)) r.access = ssb::kPairs;
    else if (v.stride[2] == 1 && from_zero && v.stride[1] % 8 == 0 && v.stride[0] % 8 == 0 && aligned(v.data, 16)) r.access = ssb::kRuns;
    return r;
}
// B or C, and whether 16-byte pieces of it lie whole and aligned: along the states, or along the steps
// (tiles start at multiples of 32 steps only where sequences start at step 0).
ssb::ProjView proj_view(const ssb_view_t &v, int dtype, int64_t n, int64_t g, int64_t s, int64_t t, bool from_zero) {
    const int64_t per = 16 / (int64_t)size_of(dtype);
    ssb::ProjView r{v.data, v.stride[0], v.stride[1], v.stride[2], v.stride[3], v.data != nullptr ? extent_of(v, {n, g, s, t}) : 0,
                    ssb::kProjAny};
    const bool outer = aligned(v.data, 16) && v.stride[0] % per == 0 && v.stride[1] % per == 0;
    if (outer && v.stride[2] == 1 && v.stride[3] % per == 0 && s % per == 0) r.access = ssb::kProjStates;
    else if (outer && from_zero && v.stride[3] == 1 && v.stride[2] % per == 0 && t % per == 0) r.access = ssb::kProjSteps;
    return r;
}
ssb::View2 view2(const ssb_view_t &v, int64_t a, int64_t b, int64_t c = 1) {
    return {v.data, v.stride[0], v.stride[1], v.stride[2], v.data != nullptr ? extent_of(v, {a, b, c}) : 0};
}

template <typename K>
int allow_smem(K kernel, size_t bytes) {
    if (bytes <= 48 * 1024) return SSB_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e == cudaSuccess ? SSB_OK : fail(SSB_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
}

// Registers of a thread of a kernel, as built; -1 where no device answers.
template <auto kKernel>
int registers_of() {
    static std::atomic<int> known{-1};
    if (known < 0) {
        cudaFuncAttributes a;
        if (cudaFuncGetAttributes(&a, kKernel) == cudaSuccess) known = a.numRegs;
        else (void)cudaGetLastError();
    }
    return known;
}

// ---- selective scan -----------------------------------------------------------------------------
constexpr int kBwdWarps = 4, kLaneWarps = 4;

// Calls f with the lanes that share a channel, the states each of them holds, and the warps of a CTA
// that scan.  `eight`: 8 states a lane instead of 4, which leaves half the warps.
template <typename F>
auto with_lanes(int64_t states, bool eight, F &&f) {
    using std::integral_constant;
    const integral_constant<int, 2> two;
    const integral_constant<int, 4> four;
    const integral_constant<int, 8> each8;
    const integral_constant<int, 16> sixteen;
    const integral_constant<int, 32> all;
    if (states <= 8) return f(two, four, four);
    if (states <= 16) return eight ? f(two, each8, four) : f(four, four, four);
    if (states <= 32) return eight ? f(four, each8, four) : f(each8, four, four);
    if (states <= 64) return eight ? f(each8, each8, four) : f(sixteen, four, four);
    if (states <= 128) return eight ? f(sixteen, each8, four) : f(all, four, each8);
    return f(all, each8, each8);
}

// Calls f with the split of a warp between time and channels as a compile-time constant.
template <typename F>
auto with_split(int tl, F &&f) {
    switch (tl) {
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: return f(std::integral_constant<int, 8>{});
        case 16: return f(std::integral_constant<int, 16>{});
        default: return f(std::integral_constant<int, 32>{});
    }
}

int64_t channel_blocks(int64_t per_group, int tl, int warps) {
    const int64_t cb = (int64_t)warps * 2 * (32 / tl);
    return (per_group + cb - 1) / cb;
}

size_t smem_of(int tl, int64_t states) {  // the largest of any type
    return with_split(tl, [&](auto k) {
        constexpr int TL = decltype(k)::value;
        return std::max(ssb::selective_bwd_smem<float, TL, kBwdWarps>(states), ssb::selective_bwd_smem<__half, TL, kBwdWarps>(states));
    });
}

// Lanes across time: the fewest (they cost shuffles) that give the SMs three CTAs for two.
int split_of(int64_t per_group, int64_t groups, int64_t sequences, int64_t states) {
    for (int tl = 4; tl < 32; tl *= 2)
        if (groups * channel_blocks(per_group, tl, kBwdWarps) * std::max<int64_t>(sequences, 1) * 2 >= 3 * sm_count() &&
            smem_of(tl, states) <= kSmemLimit)
            return tl;
    return 32;
}

int check_selective(const ssb_selective_t *p, bool data) {
    if (p == nullptr) return fail(SSB_ERR_BAD_ARG, "NULL argument");
    if (int rc = check_sizes(p->dtype, {p->batch, p->channels, p->steps, p->states})) return rc;
    if (p->states < 1 || p->states > kMaxStates)
        return fail(SSB_ERR_UNSUPPORTED, "states=%lld: 1 to %lld are supported", (long long)p->states, (long long)kMaxStates);
    if (p->groups < 1 || p->channels % p->groups != 0)
        return fail(SSB_ERR_BAD_ARG, "%lld channels do not divide into %lld groups", (long long)p->channels, (long long)p->groups);
    if (int rc = check_sequences(p->batch, p->sequences, p->offsets, p->lengths)) return rc;
    if (!data || p->channels == 0) return SSB_OK;
    if (p->batch > 0 && p->steps > 0) {
        for (const auto &[v, name] : {std::pair<const ssb_view_t &, const char *>{p->x, "x"}, {p->dt, "dt"}, {p->B, "B"}, {p->C, "C"}})
            if (int rc = check_data(v.data, p->dtype, name)) return rc;
        if (!aligned(p->z.data, size_of(p->dtype))) return fail(SSB_ERR_ALIGNMENT, "z is not aligned to its element size");
    }
    if (int rc = check_data(p->A, SSB_F32, "A")) return rc;
    for (const void *f : {(const void *)p->D, (const void *)p->dt_bias, (const void *)p->state, (const void *)p->state_out,
                          (const void *)p->checkpoints})
        if (!aligned(f, 4)) return fail(SSB_ERR_ALIGNMENT, "a float32 operand is not aligned to its element size");
    return SSB_OK;
}

int64_t count_of(const ssb_selective_t *p) { return p->offsets != nullptr ? p->sequences : p->batch; }

// Calls f with the lanes that share a channel in the backward with lanes across states.
template <typename F>
int with_backward_lanes(int64_t states, F &&f) {
    if (states <= 8) return f(std::integral_constant<int, 2>{});
    if (states <= 16) return f(std::integral_constant<int, 4>{});
    return f(std::integral_constant<int, 8>{});
}

// That form's warps pass registers to one another: its kernel has to be launched with as many as they will hold in
// all, or those that ask for more wait for good.  How many it was built with is the compiler's doing.
template <auto kKernel>
bool registers_fit() {
    const int registers = registers_of<kKernel>();
    return registers < 0 || registers == ssb::kLaunchRegisters;
}
bool lane_backward_fits(const ssb_selective_t *p) {
    return with_type(p->dtype, [&](auto *type) {
        using io_t = std::remove_pointer_t<decltype(type)>;
        return with_backward_lanes(p->states, [](auto lanes) {
            return (int)registers_fit<ssb::selective_lane_bwd_kernel<io_t, decltype(lanes)::value, kLaneWarps>>();
        });
    });
}

// The backward's shape.  Up to 32 states and with a warp for most schedulers: lanes across states
// (ssm_backward.cuh; [4, 2048, 2048], 16 states: 469 us against 699).  The sums of B and C that its warps keep in
// shared memory grow with the states, and a warp walks all steps of its sequence, so else lanes across time
// (ssm_scan.cuh; [2, 1024, 1024], 64 states: 423 us against 703; [2, 387, 1001], 10 states: 106 us against 166).
// The forward asks as well: the steps between its checkpoints depend on the answer.
struct BackwardForm {
    bool lanes;
    int split;             // lanes across time of the other form
    int64_t tile, blocks;  // steps between checkpoints; channel blocks of a group
};
BackwardForm backward_form(const ssb_selective_t *p) {
    const int64_t per_group = p->channels / p->groups;
    if (p->states <= kLaneBackwardStates && p->channels * count_of(p) * ((p->states + 3) / 4) >= 4 * 32 * (int64_t)sm_count() &&
        lane_backward_fits(p)) {
        const int64_t cb = kLaneWarps * 32 / (p->states <= 8 ? 2 : p->states <= 16 ? 4 : 8);
        return {true, 0, ssb::kCheckpointSteps, (per_group + cb - 1) / cb};
    }
    const int tl = split_of(per_group, p->groups, count_of(p), p->states);
    return {false, tl, tl * ssb::kRun, channel_blocks(per_group, tl, kBwdWarps)};
}
int64_t checkpoint_slots(const ssb_selective_t *p) {
    const int64_t tile = backward_form(p).tile;
    return p->offsets != nullptr ? p->steps / tile + p->sequences + 1 : p->batch * ((p->steps + tile - 1) / tile);
}

// How pieces of all [N, C, T] operands of a kernel may be fetched: the same way for each of them.
int tile_access(const ssb_selective_t *p, std::initializer_list<const ssb_view_t *> views) {
    const int64_t per = 16 / (int64_t)size_of(p->dtype);
    bool channels = p->groups == 1 || p->channels / p->groups % per == 0;  // blocks of channels start at whole pieces
    bool steps = p->offsets == nullptr && p->steps % per == 0;
    for (const ssb_view_t *v : views) {
        if (v->data == nullptr) continue;
        const bool base = aligned(v->data, 16) && v->stride[0] % per == 0;
        channels = channels && base && v->stride[1] == 1 && v->stride[2] % per == 0;
        steps = steps && base && v->stride[2] == 1 && v->stride[1] % per == 0;
    }
    return channels ? ssb::kTileChannels : (steps ? ssb::kTileSteps : ssb::kTileAny);
}

ssb::SelectiveArgs selective_args(const ssb_selective_t *p, int64_t blocks_per_group) {
    ssb::SelectiveArgs a{};
    const bool from_zero = p->offsets == nullptr, even = p->groups == 1 || p->channels / p->groups % 2 == 0;
    a.channels = p->channels;
    a.groups = p->groups;
    a.per_group = p->channels / p->groups;
    a.states = p->states;
    a.blocks_per_group = (int)blocks_per_group;
    a.vec = p->states % 4 == 0;
    for (const void *f : {(const void *)p->A, (const void *)p->state, (const void *)p->state_out, (const void *)p->checkpoints}) a.vec = a.vec && aligned(f, 16);
    a.softplus = p->softplus;
    a.seq = sequences_of(p->batch, p->steps, p->sequences, p->offsets, p->lengths);
    a.x = view3(p->x, p->dtype, p->batch, p->channels, p->steps, from_zero, even);
    a.dt = view3(p->dt, p->dtype, p->batch, p->channels, p->steps, from_zero, even);
    a.z = view3(p->z, p->dtype, p->batch, p->channels, p->steps, from_zero, even);
    a.out = view3(p->out, p->dtype, p->batch, p->channels, p->steps, from_zero, even);
    a.B = proj_view(p->B, p->dtype, p->batch, p->groups, p->states, p->steps, from_zero);
    a.C = proj_view(p->C, p->dtype, p->batch, p->groups, p->states, p->steps, from_zero);
    a.A = p->A;
    a.D = p->D;
    a.dt_bias = p->dt_bias;
    a.state = p->state;
    a.state_out = p->state_out;
    a.checkpoints = p->checkpoints;
    if (p->checkpoints != nullptr) {
        a.checkpoint_slots = checkpoint_slots(p);
        for (a.tile_log2 = 3; (1 << a.tile_log2) < backward_form(p).tile;) ++a.tile_log2;
    }
    return a;
}

// CTAs that share the sequences of one channel block in the backward: each keeps one set of sums for A, D and dt_bias.
int64_t backward_rows(const ssb_selective_t *p) {
    const int64_t blocks = p->groups * backward_form(p).blocks;
    const int64_t want = std::max<int64_t>(1, (4 * (int64_t)sm_count() + blocks - 1) / std::max<int64_t>(blocks, 1));
    return std::max<int64_t>(1, std::min(count_of(p), want));
}

struct BackwardParts {
    int64_t proj, A, channel;  // floats of one part
    int64_t parts_proj, parts_seq;
    size_t bytes() const { return sizeof(float) * (2 * parts_proj * proj + parts_seq * (A + 2 * channel)); }
};
BackwardParts backward_parts(const ssb_selective_t *p) {
    return {p->batch * p->steps * p->groups * p->states, p->channels * p->states, p->channels,
            backward_form(p).blocks, backward_rows(p)};
}

// ---- short convolution ----------------------------------------------------------------------------
template <typename F>
int with_width(int64_t width, F &&f) {
    if (width == 2) return f(std::integral_constant<int, 2>{});
    if (width == 3) return f(std::integral_constant<int, 3>{});
    return f(std::integral_constant<int, 4>{});
}
int check_width(int64_t width) {
    return width >= 2 && width <= 4 ? SSB_OK : fail(SSB_ERR_UNSUPPORTED, "width=%lld: 2, 3 and 4 are supported", (long long)width);
}

// Whether neighbouring channels are adjacent: always so of a single one, whose stride says nothing.
bool adjacent_channels(const ssb_view_t &v, int64_t channels) { return channels == 1 || v.stride[1] == 1; }

int check_conv(const ssb_short_conv_t *p, bool data) {
    if (p == nullptr) return fail(SSB_ERR_BAD_ARG, "NULL argument");
    if (int rc = check_sizes(p->dtype, {p->batch, p->channels, p->steps})) return rc;
    if (int rc = check_width(p->width)) return rc;
    if (int rc = check_sequences(p->batch, p->sequences, p->offsets, p->lengths)) return rc;
    if (!data || p->channels == 0) return SSB_OK;
    if (p->batch > 0 && p->steps > 0) {
        if (int rc = check_data(p->x.data, p->dtype, "x")) return rc;
        if (p->offsets != nullptr && !adjacent_channels(p->x, p->channels))
            return fail(SSB_ERR_UNSUPPORTED, "packed sequences need a channels-last view of x");
    }
    if (int rc = check_data(p->weight, p->weight_f32 ? SSB_F32 : p->dtype, "weight")) return rc;
    if (!aligned(p->bias, p->weight_f32 ? 4 : size_of(p->dtype))) return fail(SSB_ERR_ALIGNMENT, "bias is not aligned to its element size");
    if (!aligned(p->state, size_of(p->dtype)) || !aligned(p->state_out, size_of(p->dtype)))
        return fail(SSB_ERR_ALIGNMENT, "a state is not aligned to its element size");
    return SSB_OK;
}

// Channels-last kernels take any view whose channels are adjacent; with 4 channels per access where all of them allow it.
struct ConvForm {
    bool channels_last;
    int lump;
    int64_t channel_blocks, chunk_blocks;
};
bool lumps(const ssb_view_t &v, int dtype) {
    return v.stride[1] == 1 && v.stride[0] % 4 == 0 && v.stride[2] % 4 == 0 && aligned(v.data, 4 * size_of(dtype));
}
// Steps a warp walks: the more, the fewer steps are read twice (W - 1 a chunk) and the shorter the chunk's ends weigh
// ([8, 4096, 2048], bf16: 73 and 141 us forward and backward with 64 steps, 80 and 167 with 32), but the SMs want
// three CTAs each.
int conv_chunk(const ssb_short_conv_t *p) {
    for (int chunk = 64; chunk > 16; chunk /= 2)
        if ((p->channels + 127) / 128 * p->batch * ((p->steps + ssb::kConvWarps * chunk - 1) / (ssb::kConvWarps * chunk)) >= 3 * sm_count()) return chunk;
    return 16;
}
ConvForm conv_form(const ssb_short_conv_t *p, std::initializer_list<const ssb_view_t *> views) {
    bool cl = true, vec = p->channels % 4 == 0;
    for (const ssb_view_t *v : views) {
        // one channel of which time is adjacent is a row, but packed sequences need the channels-last kernels
        cl = cl && (p->offsets != nullptr ? adjacent_channels(*v, p->channels) : v->stride[1] == 1);
        vec = vec && lumps(*v, p->dtype);
    }
    ConvForm f{cl, vec ? 4 : 1, 0, 0};
    const int64_t chunk = cl ? conv_chunk(p) * ssb::kConvWarps : 4 * 32 * ssb::kRun;
    f.channel_blocks = cl ? (p->channels + 32 * f.lump - 1) / (32 * f.lump) : (p->channels + ssb::kConvWarps - 1) / ssb::kConvWarps;
    f.chunk_blocks = std::max<int64_t>(1, (p->steps + chunk - 1) / chunk);
    return f;
}
// Parts of the taps' gradient: the same for either form and lump, so that the query needs no views.
int64_t conv_parts(const ssb_short_conv_t *p) {
    const int64_t chunk = conv_chunk(p) * ssb::kConvWarps;  // 512 at most; the rows form has chunks of 1024
    return std::max<int64_t>(1, p->batch) * std::max<int64_t>(1, (p->steps + chunk - 1) / chunk);
}

ssb::ConvArgs conv_args(const ssb_short_conv_t *p, const ConvForm &f) {
    ssb::ConvArgs a{};
    a.channels = p->channels;
    a.rows = p->batch;
    a.channel_blocks = f.channel_blocks;
    a.chunk_blocks = f.chunk_blocks;
    a.silu = p->silu;
    a.weight_f32 = p->weight_f32;
    a.chunk = conv_chunk(p);
    a.seq = sequences_of(p->batch, p->steps, p->sequences, p->offsets, p->lengths);
    a.x = view3(p->x, p->dtype, p->batch, p->channels, p->steps, false, false);
    a.out = view3(p->out, p->dtype, p->batch, p->channels, p->steps, false, false);
    a.weight = p->weight;
    a.bias = p->bias;
    a.state = p->state;
    a.state_out = p->state_out;
    return a;
}

int conv_grid(const ConvForm &f, int64_t rows, unsigned *grid) {
    const int64_t blocks = f.channel_blocks * f.chunk_blocks * (rows + (f.channels_last ? 1 : 0));
    if (blocks > 2147483647) return fail(SSB_ERR_UNSUPPORTED, "more than 2^31 blocks");
    *grid = (unsigned)blocks;
    return SSB_OK;
}

int check_step(int dtype, int64_t entries, int64_t channels, int64_t pool, const int32_t *slots) {
    if (int rc = check_sizes(dtype, {entries, channels, pool})) return rc;
    if (entries > 2147483647) return fail(SSB_ERR_UNSUPPORTED, "more than 2^31 entries");
    if (slots == nullptr && pool < entries)
        return fail(SSB_ERR_BAD_ARG, "%lld entries without slots need as many states, got %lld", (long long)entries, (long long)pool);
    return SSB_OK;
}

}  // namespace

namespace ssb_host {
int take_state_space_status(int word[2]) {
    cudaError_t e = cudaMemcpyFromSymbol(word, ssb::g_status_word, 2 * sizeof(int));
    if (e == cudaSuccess && word[0] != 0) {
        const int zero[2] = {0, 0};
        e = cudaMemcpyToSymbol(ssb::g_status_word, zero, sizeof(zero));
    }
    return (int)e;
}
}  // namespace ssb_host

extern "C" {

size_t ssb_selective_checkpoint_bytes(const ssb_selective_t *p) {
    if (check_selective(p, false) != SSB_OK) return 0;
    return sizeof(float) * (size_t)(checkpoint_slots(p) * p->states * p->channels);
}

int ssb_selective_fwd(const ssb_selective_t *p, void *stream) {
    if (int rc = check_selective(p, true)) return rc;
    const int64_t count = count_of(p);
    if (p->channels == 0 || count == 0) return SSB_OK;
    if (p->steps > 0 && p->batch > 0)
        if (int rc = check_data(p->out.data, p->dtype, "out")) return rc;
    return with_type(p->dtype, [&](auto *type) {
        using io_t = std::remove_pointer_t<decltype(type)>;
        const int64_t per_group = p->channels / p->groups;
        // 8 states a lane need 9.9 instructions an exponential where 4 need 12.6, but a warp alone on its scheduler takes
        // as long for either: from two warps a scheduler up (13 prompts of 4096 channels, 16 states: 136 us against
        // 169; [4, 2048, 2048], half a warp a scheduler: 179 against 177; [1, 2048, 8192]: 636 against 505).
        const bool eight = p->channels * count * ((p->states + 7) / 8) >= 2 * 4 * 32 * (int64_t)sm_count();
        return with_lanes(p->states, eight, [&](auto lanes, auto each, auto warps) {
            constexpr int LN = decltype(lanes)::value, SPL = decltype(each)::value, W = decltype(warps)::value;
            using H = ssb::LaneShape<LN, SPL, W>;
            ssb::SelectiveArgs a = selective_args(p, (per_group + H::CB - 1) / H::CB);
            a.x.access = a.dt.access = a.z.access = a.out.access = tile_access(p, {&p->x, &p->dt, &p->z, &p->out});
            if (a.B.access != a.C.access) a.B.access = a.C.access = ssb::kProjAny;
            auto kernel = ssb::selective_lane_fwd_kernel<io_t, LN, SPL, W>;
            constexpr size_t smem = ssb::selective_lane_smem<LN, SPL, W>();
            if (int rc = allow_smem(kernel, smem)) return rc;
            const dim3 grid((unsigned)(a.blocks_per_group * p->groups), (unsigned)std::min<int64_t>(count, 65535));
            kernel<<<grid, 2 * H::THREADS, smem, (cudaStream_t)stream>>>(a);
            return check_launch("selective_lane_fwd_kernel");
        });
    });
}

size_t ssb_selective_bwd_workspace_bytes(const ssb_selective_t *p) {
    if (check_selective(p, false) != SSB_OK) return 0;
    return backward_parts(p).bytes();
}

int ssb_selective_bwd(const ssb_selective_t *p, const ssb_selective_grads_t *g, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_selective(p, true)) return rc;
    if (g == nullptr) return fail(SSB_ERR_BAD_ARG, "NULL argument");
    if (p->channels == 0) return SSB_OK;
    const int64_t count = count_of(p);
    if (p->steps > 0 && p->batch > 0) {
        for (const auto &[v, name] : {std::pair<const ssb_view_t &, const char *>{g->gout, "gout"}, {g->gx, "gx"}, {g->gdt, "gdt"},
                                      {g->gB, "gB"}, {g->gC, "gC"}})
            if (int rc = check_data(v.data, p->dtype, name)) return rc;
        if (p->z.data != nullptr)
            if (int rc = check_data(g->gz.data, p->dtype, "gz")) return rc;
        if (p->checkpoints == nullptr) return fail(SSB_ERR_BAD_ARG, "the backward needs the forward's checkpoints");
    }
    if (int rc = check_data(g->gA, SSB_F32, "gA")) return rc;
    const BackwardParts parts = backward_parts(p);
    if (workspace == nullptr || workspace_bytes < parts.bytes() || !aligned(workspace, 4))
        return fail(SSB_ERR_WORKSPACE, "the backward needs %zu bytes of workspace, got %zu", parts.bytes(), workspace_bytes);
    float *part = static_cast<float *>(workspace);
    ssb::SelectiveGradArgs q{};
    const bool from_zero = p->offsets == nullptr, even = p->groups == 1 || p->channels / p->groups % 2 == 0;
    q.gout = view3(g->gout, p->dtype, p->batch, p->channels, p->steps, from_zero, even);
    q.gx = view3(g->gx, p->dtype, p->batch, p->channels, p->steps, from_zero, even);
    q.gdt = view3(g->gdt, p->dtype, p->batch, p->channels, p->steps, from_zero, even);
    q.gz = view3(g->gz, p->dtype, p->batch, p->channels, p->steps, from_zero, even);
    q.gstate_out = g->gstate_out;
    q.gstate = g->gstate;
    q.part_A = part;
    q.part_D = q.part_A + parts.parts_seq * parts.A;
    q.part_bias = q.part_D + parts.parts_seq * parts.channel;
    q.part_B = q.part_bias + parts.parts_seq * parts.channel;
    q.part_C = q.part_B + parts.parts_proj * parts.proj;
    q.rows = p->batch;
    const BackwardForm form = backward_form(p);
    const int rc = with_type(p->dtype, [&](auto *type) {
        using io_t = std::remove_pointer_t<decltype(type)>;
        if (form.lanes) {
            return with_backward_lanes(p->states, [&](auto lanes) {
                constexpr int LN = decltype(lanes)::value;
                using H = ssb::LaneShape<LN, 4, kLaneWarps>;
                ssb::SelectiveArgs a = selective_args(p, form.blocks);
                ssb::SelectiveGradArgs b = q;
                a.vec = a.vec && aligned(q.gstate_out, 16) && aligned(q.gstate, 16) && aligned(q.part_A, 16) && aligned(q.part_B, 16) && aligned(q.part_C, 16);
                a.x.access = a.dt.access = a.z.access = b.gout.access = b.gx.access = b.gdt.access = b.gz.access =
                    tile_access(p, {&p->x, &p->dt, &p->z, &g->gout, &g->gx, &g->gdt, p->z.data != nullptr ? &g->gz : &p->z});
                if (a.B.access != a.C.access) a.B.access = a.C.access = ssb::kProjAny;
                auto kernel = ssb::selective_lane_bwd_kernel<io_t, LN, kLaneWarps>;
                constexpr size_t smem = ssb::selective_lane_bwd_smem<io_t, LN, kLaneWarps>();
                if (int bad = allow_smem(kernel, smem)) return bad;
                if (registers_of<ssb::selective_lane_bwd_kernel<io_t, LN, kLaneWarps>>() != ssb::kLaunchRegisters)
                    return fail(SSB_ERR_LAUNCH, "the registers of selective_lane_bwd_kernel are not known");
                const dim3 grid((unsigned)(form.blocks * p->groups), (unsigned)parts.parts_seq);
                kernel<<<grid, 2 * H::THREADS, smem, (cudaStream_t)stream>>>(a, b);
                return check_launch("selective_lane_bwd_kernel");
            });
        }
        return with_split(form.split, [&](auto k) {
            constexpr int TL = decltype(k)::value;
            const ssb::SelectiveArgs a = selective_args(p, form.blocks);
            auto kernel = ssb::selective_bwd_kernel<io_t, TL, kBwdWarps>;
            const size_t smem = ssb::selective_bwd_smem<io_t, TL, kBwdWarps>(p->states);
            if (int bad = allow_smem(kernel, smem)) return bad;
            const dim3 grid((unsigned)(a.blocks_per_group * p->groups), (unsigned)parts.parts_seq);
            kernel<<<grid, kBwdWarps * 32, smem, (cudaStream_t)stream>>>(a, q);
            return check_launch("selective_bwd_kernel");
        });
    });
    if (rc != SSB_OK) return rc;
    ssb::SelectiveReduceArgs r{};
    r.seq = sequences_of(p->batch, p->steps, p->sequences, p->offsets, p->lengths);
    r.rows = p->batch;
    r.groups = p->groups;
    r.states = p->states;
    r.channels = p->channels;
    r.parts_proj = (int)parts.parts_proj;
    r.parts_seq = (int)parts.parts_seq;
    r.part_B = q.part_B;
    r.part_C = q.part_C;
    r.part_A = q.part_A;
    r.part_D = q.part_D;
    r.part_bias = q.part_bias;
    r.gB = proj_view(g->gB, p->dtype, p->batch, p->groups, p->states, p->steps, false);
    r.gC = proj_view(g->gC, p->dtype, p->batch, p->groups, p->states, p->steps, false);
    r.gA = g->gA;
    r.gD = g->gD;
    r.gbias = g->gdt_bias;
    const auto blocks = [](int64_t n, int64_t cap) { return std::min<int64_t>((n + 255) / 256, cap); };
    r.proj_blocks = count > 0 ? (int)blocks(parts.proj, 16ll * sm_count()) : 0;
    const int64_t others = blocks(parts.A + 2 * parts.channel, 4ll * sm_count());
    return with_type(p->dtype, [&](auto *type) {
        using io_t = std::remove_pointer_t<decltype(type)>;
        ssb::selective_reduce_kernel<io_t><<<(unsigned)(r.proj_blocks + others), 256, 0, (cudaStream_t)stream>>>(r);
        return check_launch("selective_reduce_kernel");
    });
}

int ssb_selective_step(const ssb_selective_step_t *p, void *stream) {
    if (p == nullptr) return fail(SSB_ERR_BAD_ARG, "NULL argument");
    if (int rc = check_step(p->dtype, p->entries, p->channels, p->pool, p->slots)) return rc;
    if (int rc = check_sizes(p->dtype, {std::max(p->entries, p->pool), p->channels, p->states})) return rc;
    if (p->states < 1 || p->states > kMaxStates)
        return fail(SSB_ERR_UNSUPPORTED, "states=%lld: 1 to %lld are supported", (long long)p->states, (long long)kMaxStates);
    if (p->groups < 1 || p->channels % p->groups != 0)
        return fail(SSB_ERR_BAD_ARG, "%lld channels do not divide into %lld groups", (long long)p->channels, (long long)p->groups);
    if (p->entries == 0 || p->channels == 0) return SSB_OK;
    for (const auto &[v, name] : {std::pair<const ssb_view_t &, const char *>{p->x, "x"}, {p->dt, "dt"}, {p->B, "B"}, {p->C, "C"}, {p->out, "out"}})
        if (int rc = check_data(v.data, p->dtype, name)) return rc;
    if (!aligned(p->z.data, size_of(p->dtype))) return fail(SSB_ERR_ALIGNMENT, "z is not aligned to its element size");
    if (int rc = check_data(p->A, SSB_F32, "A")) return rc;
    if (p->pool > 0)
        if (int rc = check_data(p->state, SSB_F32, "state")) return rc;
    if (!aligned(p->D, 4) || !aligned(p->dt_bias, 4)) return fail(SSB_ERR_ALIGNMENT, "a float32 operand is not aligned to its element size");
    ssb::SelectiveStepArgs a{};
    a.channels = p->channels;
    a.per_group = p->channels / p->groups;
    a.states = p->states;
    a.softplus = p->softplus;
    a.vec = p->states % 4 == 0 && aligned(p->state, 16) && aligned(p->A, 16);
    a.vec_proj = p->states % 4 == 0;
    for (const ssb_view_t *v : {&p->B, &p->C})
        a.vec_proj = a.vec_proj && aligned(v->data, 4 * size_of(p->dtype)) && v->stride[2] == 1 && v->stride[0] % 4 == 0 &&
                     (p->groups == 1 || v->stride[1] % 4 == 0);  // of one group the stride says nothing
    a.slots = {p->slots, p->entries, p->pool};
    a.x = view2(p->x, p->entries, p->channels);
    a.dt = view2(p->dt, p->entries, p->channels);
    a.z = view2(p->z, p->entries, p->channels);
    a.out = view2(p->out, p->entries, p->channels);
    a.B = view2(p->B, p->entries, p->groups, p->states);
    a.C = view2(p->C, p->entries, p->groups, p->states);
    a.A = p->A;
    a.D = p->D;
    a.dt_bias = p->dt_bias;
    a.state = p->state;
    return with_type(p->dtype, [&](auto *type) {
        using io_t = std::remove_pointer_t<decltype(type)>;
        // 4 channels a thread where that leaves the SMs two CTAs each
        const auto launch = [&](auto lanes) {
            constexpr int L = decltype(lanes)::value, CB = 128 / L, kEach = L >= 4 ? 4 : 1;
            const bool many = p->entries * ((p->channels + kEach * CB - 1) / (kEach * CB)) >= 2 * sm_count();
            const int64_t blocks = (p->channels + CB * (many ? kEach : 1) - 1) / (CB * (many ? kEach : 1));
            if (blocks > 65535) return fail(SSB_ERR_UNSUPPORTED, "too many channels");
            const dim3 grid((unsigned)p->entries, (unsigned)blocks);
            if (many) ssb::selective_step_kernel<io_t, L, kEach><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
            else ssb::selective_step_kernel<io_t, L, 1><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
            return check_launch("selective_step_kernel");
        };
        using std::integral_constant;
        if (p->states <= 4) return launch(integral_constant<int, 1>{});
        if (p->states <= 8) return launch(integral_constant<int, 2>{});
        if (p->states <= 16) return launch(integral_constant<int, 4>{});
        if (p->states <= 32) return launch(integral_constant<int, 8>{});
        return launch(integral_constant<int, 16>{});
    });
}

int ssb_short_conv_fwd(const ssb_short_conv_t *p, void *stream) {
    if (int rc = check_conv(p, true)) return rc;
    const int64_t count = p->offsets != nullptr ? p->sequences : p->batch;
    if (p->channels == 0 || count == 0) return SSB_OK;
    if (p->steps > 0)
        if (int rc = check_data(p->out.data, p->dtype, "out")) return rc;
    if (p->offsets != nullptr && p->steps > 0 && !adjacent_channels(p->out, p->channels))
        return fail(SSB_ERR_UNSUPPORTED, "packed sequences need a channels-last view of out");
    ConvForm f = conv_form(p, {&p->x, &p->out});
    if (p->steps == 0) f = {true, 1, (p->channels + 31) / 32, 1};
    const ssb::ConvArgs a = conv_args(p, f);
    unsigned grid = 0;
    if (int rc = conv_grid(f, p->batch, &grid)) return rc;
    return with_type(p->dtype, [&](auto *type) {
        using io_t = std::remove_pointer_t<decltype(type)>;
        return with_width(p->width, [&](auto k) {
            constexpr int W = decltype(k)::value;
            const int threads = ssb::kConvWarps * 32;
            if (!f.channels_last) ssb::conv_rows_fwd_kernel<io_t, W><<<grid, threads, 0, (cudaStream_t)stream>>>(a);
            else if (f.lump == 4) ssb::conv_cl_fwd_kernel<io_t, 4, W><<<grid, threads, 0, (cudaStream_t)stream>>>(a);
            else ssb::conv_cl_fwd_kernel<io_t, 1, W><<<grid, threads, 0, (cudaStream_t)stream>>>(a);
            return check_launch("short convolution");
        });
    });
}

size_t ssb_short_conv_bwd_workspace_bytes(const ssb_short_conv_t *p) {
    if (check_conv(p, false) != SSB_OK) return 0;
    return sizeof(float) * (size_t)(conv_parts(p) * p->channels * (p->width + 1));
}

int ssb_short_conv_bwd(const ssb_short_conv_t *p, const ssb_short_conv_grads_t *g, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_conv(p, true)) return rc;
    if (g == nullptr) return fail(SSB_ERR_BAD_ARG, "NULL argument");
    if (p->channels == 0) return SSB_OK;
    if (p->steps > 0 && p->batch > 0) {
        if (int rc = check_data(g->gout.data, p->dtype, "gout")) return rc;
        if (int rc = check_data(g->gx.data, p->dtype, "gx")) return rc;
        if (p->offsets != nullptr && (!adjacent_channels(g->gout, p->channels) || !adjacent_channels(g->gx, p->channels)))
            return fail(SSB_ERR_UNSUPPORTED, "packed sequences need channels-last views");
    }
    const int weight_type = p->weight_f32 ? SSB_F32 : p->dtype;
    if (int rc = check_data(g->gweight, weight_type, "gweight")) return rc;
    if (!aligned(g->gbias, size_of(weight_type)) || !aligned(g->gstate, size_of(p->dtype)) || !aligned(g->gstate_out, size_of(p->dtype)))
        return fail(SSB_ERR_ALIGNMENT, "a gradient is not aligned to its element size");
    const size_t need = ssb_short_conv_bwd_workspace_bytes(p);
    if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 4))
        return fail(SSB_ERR_WORKSPACE, "the backward needs %zu bytes of workspace, got %zu", need, workspace_bytes);
    ConvForm f = conv_form(p, {&p->x, &g->gout, &g->gx});
    if (p->steps == 0) f = {true, 1, (p->channels + 31) / 32, 1};
    const ssb::ConvArgs a = conv_args(p, f);
    ssb::ConvGradArgs q{};
    q.gout = view3(g->gout, p->dtype, p->batch, p->channels, p->steps, false, false);
    q.gx = view3(g->gx, p->dtype, p->batch, p->channels, p->steps, false, false);
    q.gstate_out = g->gstate_out;
    q.gstate = g->gstate;
    q.part = static_cast<float *>(workspace);
    unsigned grid = 0;
    if (int rc = conv_grid(f, p->batch, &grid)) return rc;
    const int64_t parts = p->batch * f.chunk_blocks;
    return with_type(p->dtype, [&](auto *type) {
        using io_t = std::remove_pointer_t<decltype(type)>;
        const int rc = with_width(p->width, [&](auto k) {
            constexpr int W = decltype(k)::value;
            const int threads = ssb::kConvWarps * 32;
            if (grid == 0) return (int)SSB_OK;
            if (!f.channels_last) ssb::conv_rows_bwd_kernel<io_t, W><<<grid, threads, 0, (cudaStream_t)stream>>>(a, q);
            else if (f.lump == 4) ssb::conv_cl_bwd_kernel<io_t, 4, W><<<grid, threads, 0, (cudaStream_t)stream>>>(a, q);
            else ssb::conv_cl_bwd_kernel<io_t, 1, W><<<grid, threads, 0, (cudaStream_t)stream>>>(a, q);
            return check_launch("short convolution backward");
        });
        if (rc != SSB_OK) return rc;
        const int64_t blocks = std::min<int64_t>((p->channels * (p->width + 1) + 255) / 256, 8ll * sm_count());
        ssb::conv_reduce_kernel<io_t><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(q.part, parts, p->channels, (int)p->width,
                                                                                          p->weight_f32, g->gweight, g->gbias);
        return check_launch("conv_reduce_kernel");
    });
}

int ssb_short_conv_step(const ssb_short_conv_step_t *p, void *stream) {
    if (p == nullptr) return fail(SSB_ERR_BAD_ARG, "NULL argument");
    if (int rc = check_step(p->dtype, p->entries, p->channels, p->pool, p->slots)) return rc;
    if (int rc = check_width(p->width)) return rc;
    if (p->entries == 0 || p->channels == 0) return SSB_OK;
    if (int rc = check_data(p->x.data, p->dtype, "x")) return rc;
    if (int rc = check_data(p->out.data, p->dtype, "out")) return rc;
    if (int rc = check_data(p->weight, p->weight_f32 ? SSB_F32 : p->dtype, "weight")) return rc;
    if (!aligned(p->bias, p->weight_f32 ? 4 : size_of(p->dtype))) return fail(SSB_ERR_ALIGNMENT, "bias is not aligned to its element size");
    if (p->pool > 0)
        if (int rc = check_data(p->state, p->dtype, "state")) return rc;
    ssb::ConvStepArgs a{};
    a.channels = p->channels;
    a.width = (int)p->width;
    a.silu = p->silu;
    a.weight_f32 = p->weight_f32;
    a.slots = {p->slots, p->entries, p->pool};
    a.x = view2(p->x, p->entries, p->channels);
    a.out = view2(p->out, p->entries, p->channels);
    a.weight = p->weight;
    a.bias = p->bias;
    a.state = p->state;
    return with_type(p->dtype, [&](auto *type) {
        using io_t = std::remove_pointer_t<decltype(type)>;
        return with_width(p->width, [&](auto k) {
            constexpr int W = decltype(k)::value;
            // 4 channels a thread where all their pieces are whole and aligned
            const size_t piece = 4 * size_of(p->dtype), wide = 4 * (p->weight_f32 ? 4 : size_of(p->dtype));
            const bool lumps = p->channels % 4 == 0 && aligned(p->state, piece) && aligned(p->weight, wide) && aligned(p->bias, wide) &&
                               aligned(p->x.data, piece) && p->x.stride[1] == 1 && p->x.stride[0] % 4 == 0 &&
                               aligned(p->out.data, piece) && p->out.stride[1] == 1 && p->out.stride[0] % 4 == 0;
            const int64_t blocks = (p->channels + 128 * (lumps ? 4 : 1) - 1) / (128 * (lumps ? 4 : 1));
            if (blocks > 65535) return fail(SSB_ERR_UNSUPPORTED, "too many channels");
            const dim3 grid((unsigned)p->entries, (unsigned)blocks);
            if (lumps) ssb::conv_step_kernel<io_t, W, 4><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
            else ssb::conv_step_kernel<io_t, W, 1><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
            return check_launch("conv_step_kernel");
        });
    });
}

}  // extern "C"
