// The state-space operators of the extension module: argument checks, output allocation and thin
// calls into the C-ABI.  Shapes and types are checked before devices, so that a wrong call is
// refused in the same words with or without a GPU.  Included by torch_ext.cpp.
#pragma once

using OptTensor = c10::optional<torch::Tensor>;

// Numbers and shapes as text for messages, without streams.
std::string text(int64_t v) { return std::to_string(v); }
std::string text(at::IntArrayRef v) {
    std::string s = "[";
    for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
    return s + "]";
}

bool present(const OptTensor &t) { return t.has_value() && t->defined(); }

int element_type(const torch::Tensor &x, const char *op) {
    switch (x.scalar_type()) {
        case torch::kFloat32: return SSB_F32;
        case torch::kBFloat16: return SSB_BF16;
        case torch::kHalf: return SSB_F16;
        default: TORCH_CHECK_NOT_IMPLEMENTED(false, "\"", op, "\" not implemented for '", toString(x.scalar_type()), "'");
    }
}

void check_like(const torch::Tensor &ref, const torch::Tensor &x, const char *name, const char *like) {
    TORCH_CHECK(x.scalar_type() == ref.scalar_type(), name, " must have the same dtype as ", like);
    TORCH_CHECK(x.device() == ref.device(), name, " must be on the same device as ", like);
}

void check_shape_is(const torch::Tensor &x, at::IntArrayRef want, const char *name) {
    TORCH_CHECK(x.sizes() == want, name, " must have the shape ", text(want), ", got ", text(x.sizes()));
}

// A dense float32 operand.
const float *f32_operand(const OptTensor &t, const torch::Tensor &ref, at::IntArrayRef want, const char *name) {
    if (!present(t)) return nullptr;
    check_shape_is(*t, want, name);
    TORCH_CHECK(t->scalar_type() == torch::kFloat32, name, " must be float32");
    TORCH_CHECK(t->device() == ref.device(), name, " must be on the same device as x");
    TORCH_CHECK(t->is_contiguous(), name, " must be contiguous");
    return t->data_ptr<float>();
}

const int32_t *int_operand(const OptTensor &t, const torch::Tensor &ref, const char *name) {
    if (!present(t)) return nullptr;
    TORCH_CHECK(t->dim() == 1, name, " must be 1-D");
    TORCH_CHECK(t->scalar_type() == torch::kInt32, name, " must be int32");
    TORCH_CHECK(t->device() == ref.device(), name, " must be on the same device as x");
    TORCH_CHECK(t->is_contiguous(), name, " must be contiguous");
    return t->data_ptr<int32_t>();
}

void need_cuda(const torch::Tensor &x, const char *op) {
    TORCH_CHECK(x.device().is_cuda(), "scanscam_b200.", op, " needs CUDA tensors (got a tensor on '", x.device().str(),
                "'); this build has no CPU path");
}

// The kernel wrote into `t` behind autograd's back: a saved copy of it is stale.
void mark_written(const torch::Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

ssb_view_t view_of(const torch::Tensor &t) {
    ssb_view_t v{};
    v.data = t.data_ptr();
    for (int64_t i = 0; i < t.dim() && i < 4; ++i) v.stride[i] = t.stride(i);
    return v;
}

// [N, C, T] dense with channels adjacent, or with steps adjacent.
torch::Tensor empty_like_layout(const torch::Tensor &x) {
    const auto n = x.size(0), c = x.size(1), t = x.size(2);
    return x.stride(1) == 1 ? torch::empty({n, t, c}, x.options()).transpose(1, 2) : torch::empty({n, c, t}, x.options());
}
// A projection [N, G, S, T], dense, with whichever of states and steps is adjacent in `like` adjacent.
torch::Tensor empty_projection(const torch::Tensor &like) {
    const auto n = like.size(0), g = like.size(1), s = like.size(2), t = like.size(3);
    return like.stride(3) == 1 && like.stride(2) != 1 ? torch::empty({n, g, s, t}, like.options())
                                                      : torch::empty({n, t, g, s}, like.options()).permute({0, 2, 3, 1});
}

// Which sequences a batch holds; fills the struct's fields and returns their number.
template <typename P>
int64_t set_sequences(P &p, const torch::Tensor &x, const OptTensor &lengths, const OptTensor &offsets) {
    TORCH_CHECK(!(present(lengths) && present(offsets)), "lengths and offsets exclude each other");
    p.lengths = int_operand(lengths, x, "lengths");
    p.offsets = int_operand(offsets, x, "offsets");
    if (present(lengths)) TORCH_CHECK(lengths->size(0) == x.size(0), "lengths must have one entry per row of x");
    if (present(offsets)) {
        TORCH_CHECK(x.size(0) == 1, "packed sequences (offsets) need x of shape [1, C, T]");
        TORCH_CHECK(offsets->size(0) >= 2, "offsets must bound at least one sequence");
        p.sequences = offsets->size(0) - 1;
        return p.sequences;
    }
    p.sequences = x.size(0);
    return x.size(0);
}

// ---- selective scan -----------------------------------------------------------------------------
struct SelectiveInputs {
    const torch::Tensor &x, &dt, &A, &B, &C;
    const OptTensor &D, &z, &dt_bias, &state, &lengths, &offsets;
};

ssb_selective_t selective_problem(const SelectiveInputs &in, bool softplus, int64_t *sequences, const char *op) {
    const torch::Tensor &x = in.x;
    ssb_selective_t p{};
    TORCH_CHECK(x.dim() == 3, "x must be 3-D [N, C, T]");
    p.dtype = element_type(x, op);
    p.softplus = softplus;
    p.batch = x.size(0);
    p.channels = x.size(1);
    p.steps = x.size(2);
    check_shape_is(in.dt, x.sizes(), "dt");
    check_like(x, in.dt, "dt", "x");
    TORCH_CHECK(in.A.dim() == 2 && in.A.size(0) == p.channels, "A must be [C, S] with C = ", text(p.channels));
    p.states = in.A.size(1);
    TORCH_CHECK(p.states >= 1 && p.states <= 256, "A must have 1 to 256 states, got ", text(p.states));
    TORCH_CHECK(in.B.dim() == 4 && in.B.size(0) == p.batch && in.B.size(2) == p.states && in.B.size(3) == p.steps,
                "B must be [N, S, T] or [N, G, S, T] with S as in A and N, T as in x");
    p.groups = in.B.size(1);
    TORCH_CHECK(p.groups >= 1 && p.channels % p.groups == 0, text(p.channels), " channels do not divide into ", text(p.groups), " groups");
    check_shape_is(in.C, in.B.sizes(), "C");
    check_like(x, in.B, "B", "x");
    check_like(x, in.C, "C", "x");
    p.A = f32_operand(in.A, x, in.A.sizes(), "A");
    p.D = f32_operand(in.D, x, {p.channels}, "D");
    p.dt_bias = f32_operand(in.dt_bias, x, {p.channels}, "dt_bias");
    if (present(in.z)) {
        check_shape_is(*in.z, x.sizes(), "z");
        check_like(x, *in.z, "z", "x");
        p.z = view_of(*in.z);
    }
    *sequences = set_sequences(p, x, in.lengths, in.offsets);
    p.state = f32_operand(in.state, x, {*sequences, p.channels, p.states}, "state");
    p.x = view_of(x);
    p.dt = view_of(in.dt);
    p.B = view_of(in.B);
    p.C = view_of(in.C);
    return p;
}

// -> (out, state behind the last step, checkpoints or an empty tensor)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> selective_forward(
    const torch::Tensor &x, const torch::Tensor &dt, const torch::Tensor &A, const torch::Tensor &B, const torch::Tensor &C,
    const OptTensor &D, const OptTensor &z, const OptTensor &dt_bias, bool softplus, const OptTensor &state,
    const OptTensor &lengths, const OptTensor &offsets, bool for_backward) {
    int64_t sequences = 0;
    ssb_selective_t p = selective_problem({x, dt, A, B, C, D, z, dt_bias, state, lengths, offsets}, softplus, &sequences, "scan_selective");
    need_cuda(x, "scan_selective");
    c10::cuda::CUDAGuard guard(x.device());
    torch::Tensor out = empty_like_layout(x);
    const auto f32 = x.options().dtype(torch::kFloat32);
    torch::Tensor state_out = torch::empty({sequences, p.channels, p.states}, f32), checkpoints = torch::empty({0}, f32);
    p.out = view_of(out);
    p.state_out = state_out.data_ptr<float>();
    if (for_backward) {
        checkpoints = torch::empty({(int64_t)(ssb_selective_checkpoint_bytes(&p) / sizeof(float))}, f32);
        p.checkpoints = checkpoints.numel() ? checkpoints.data_ptr<float>() : nullptr;
    }
    raise_on(ssb_selective_fwd(&p, current_stream()), "scan_selective");
    return {out, state_out, checkpoints};
}

// -> gradients of x, dt, A, B, C, D, z, dt_bias, state (undefined where the operand is absent)
std::vector<OptTensor> selective_backward(
    const torch::Tensor &x, const torch::Tensor &dt, const torch::Tensor &A, const torch::Tensor &B, const torch::Tensor &C,
    const OptTensor &D, const OptTensor &z, const OptTensor &dt_bias, bool softplus, const OptTensor &state,
    const OptTensor &lengths, const OptTensor &offsets, const torch::Tensor &checkpoints, const torch::Tensor &grad_out,
    const OptTensor &grad_state) {
    int64_t sequences = 0;
    ssb_selective_t p = selective_problem({x, dt, A, B, C, D, z, dt_bias, state, lengths, offsets}, softplus, &sequences, "scan_selective");
    need_cuda(x, "scan_selective");
    check_shape_is(grad_out, x.sizes(), "grad_out");
    check_like(x, grad_out, "grad_out", "x");
    c10::cuda::CUDAGuard guard(x.device());
    TORCH_CHECK((size_t)checkpoints.numel() * sizeof(float) >= ssb_selective_checkpoint_bytes(&p), "checkpoints of another problem");
    p.checkpoints = checkpoints.numel() ? checkpoints.data_ptr<float>() : nullptr;
    ssb_selective_grads_t g{};
    g.gout = view_of(grad_out);
    g.gstate_out = f32_operand(grad_state, x, {sequences, p.channels, p.states}, "grad_state");
    torch::Tensor gx = empty_like_layout(x), gdt = empty_like_layout(dt), gB = empty_projection(B), gC = empty_projection(C);
    torch::Tensor gA = torch::empty_like(A);
    OptTensor gD, gz, gbias, gstate;
    g.gx = view_of(gx);
    g.gdt = view_of(gdt);
    g.gB = view_of(gB);
    g.gC = view_of(gC);
    g.gA = gA.data_ptr<float>();
    if (present(D)) g.gD = (gD = torch::empty_like(*D))->data_ptr<float>();
    if (present(z)) g.gz = view_of(*(gz = empty_like_layout(*z)));
    if (present(dt_bias)) g.gdt_bias = (gbias = torch::empty_like(*dt_bias))->data_ptr<float>();
    if (present(state)) g.gstate = (gstate = torch::empty_like(*state))->data_ptr<float>();
    const size_t bytes = ssb_selective_bwd_workspace_bytes(&p);
    torch::Tensor ws = scratch(std::max<size_t>(bytes, 4), x);
    raise_on(ssb_selective_bwd(&p, &g, ws.data_ptr(), bytes, current_stream()), "scan_selective backward");
    return {gx, gdt, gA, gB, gC, gD, gz, gbias, gstate};
}

torch::Tensor selective_step(const torch::Tensor &x, const torch::Tensor &dt, const torch::Tensor &A, const torch::Tensor &B,
                             const torch::Tensor &C, torch::Tensor state, const OptTensor &D, const OptTensor &z,
                             const OptTensor &dt_bias, bool softplus, const OptTensor &slots) {
    ssb_selective_step_t p{};
    TORCH_CHECK(x.dim() == 2, "x must be 2-D [M, C]");
    p.dtype = element_type(x, "scan_selective_step");
    p.softplus = softplus;
    p.entries = x.size(0);
    p.channels = x.size(1);
    check_shape_is(dt, x.sizes(), "dt");
    check_like(x, dt, "dt", "x");
    TORCH_CHECK(A.dim() == 2 && A.size(0) == p.channels, "A must be [C, S] with C = ", text(p.channels));
    p.states = A.size(1);
    TORCH_CHECK(p.states >= 1 && p.states <= 256, "A must have 1 to 256 states, got ", text(p.states));
    TORCH_CHECK((B.dim() == 2 || B.dim() == 3) && B.size(0) == p.entries && B.size(-1) == p.states,
                "B must be [M, S] or [M, G, S] with S as in A and M as in x");
    p.groups = B.dim() == 3 ? B.size(1) : 1;
    TORCH_CHECK(p.groups >= 1 && p.channels % p.groups == 0, text(p.channels), " channels do not divide into ", text(p.groups), " groups");
    check_shape_is(C, B.sizes(), "C");
    check_like(x, B, "B", "x");
    check_like(x, C, "C", "x");
    p.A = f32_operand(A, x, A.sizes(), "A");
    p.D = f32_operand(D, x, {p.channels}, "D");
    p.dt_bias = f32_operand(dt_bias, x, {p.channels}, "dt_bias");
    p.slots = int_operand(slots, x, "slots");
    if (present(slots)) TORCH_CHECK(slots->size(0) == p.entries, "slots must have one entry per row of x");
    TORCH_CHECK(state.dim() == 3, "state must be 3-D [pool, C, S]");
    p.pool = state.size(0);
    p.state = const_cast<float *>(f32_operand(state, x, {p.pool, p.channels, p.states}, "state"));
    TORCH_CHECK(present(slots) || p.pool == p.entries, "without slots, state must have one row per row of x");
    if (present(z)) {
        check_shape_is(*z, x.sizes(), "z");
        check_like(x, *z, "z", "x");
        p.z = view_of(*z);
    }
    need_cuda(x, "scan_selective_step");
    c10::cuda::CUDAGuard guard(x.device());
    torch::Tensor out = torch::empty({p.entries, p.channels}, x.options());
    p.x = view_of(x);
    p.dt = view_of(dt);
    p.out = view_of(out);
    const auto projection = [](const torch::Tensor &t) {
        ssb_view_t v = view_of(t);
        if (t.dim() == 2) v.stride[2] = v.stride[1];
        return v;
    };
    p.B = projection(B);
    p.C = projection(C);
    raise_on(ssb_selective_step(&p, current_stream()), "scan_selective_step");
    mark_written(state);
    return out;
}

// ---- short convolution ----------------------------------------------------------------------------
const void *tap_operand(const OptTensor &t, const torch::Tensor &x, const torch::Tensor &weight, at::IntArrayRef want, const char *name) {
    if (!present(t)) return nullptr;
    check_shape_is(*t, want, name);
    TORCH_CHECK(t->scalar_type() == x.scalar_type() || t->scalar_type() == torch::kFloat32, name, " must be float32 or have the dtype of x");
    TORCH_CHECK(t->scalar_type() == weight.scalar_type(), name, " must have the same dtype as weight");
    TORCH_CHECK(t->device() == x.device(), name, " must be on the same device as x");
    TORCH_CHECK(t->is_contiguous(), name, " must be contiguous");
    return t->data_ptr();
}
const void *window_operand(const OptTensor &t, const torch::Tensor &x, at::IntArrayRef want, const char *name) {
    if (!present(t)) return nullptr;
    check_shape_is(*t, want, name);
    check_like(x, *t, name, "x");
    TORCH_CHECK(t->is_contiguous(), name, " must be contiguous");
    return t->data_ptr();
}

void check_width(const torch::Tensor &weight, int64_t channels) {
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) == channels, "weight must be [C, W] with C = ", text(channels));
    TORCH_CHECK(weight.size(1) >= 2 && weight.size(1) <= 4, "weight must have 2, 3 or 4 taps, got ", text(weight.size(1)));
}

ssb_short_conv_t conv_problem(const torch::Tensor &x, const torch::Tensor &weight, const OptTensor &bias, bool silu,
                              const OptTensor &state, const OptTensor &lengths, const OptTensor &offsets, int64_t *sequences) {
    ssb_short_conv_t p{};
    TORCH_CHECK(x.dim() == 3, "x must be 3-D [N, C, T]");
    p.dtype = element_type(x, "short_conv");
    p.silu = silu;
    p.batch = x.size(0);
    p.channels = x.size(1);
    p.steps = x.size(2);
    check_width(weight, p.channels);
    p.width = weight.size(1);
    p.weight = tap_operand(weight, x, weight, weight.sizes(), "weight");
    p.bias = tap_operand(bias, x, weight, {p.channels}, "bias");
    p.weight_f32 = weight.scalar_type() == torch::kFloat32;
    *sequences = set_sequences(p, x, lengths, offsets);
    p.state = window_operand(state, x, {*sequences, p.channels, p.width - 1}, "state");
    p.x = view_of(x);
    return p;
}

// -> (out, window behind the last step)
std::tuple<torch::Tensor, torch::Tensor> short_conv_forward(const torch::Tensor &x, const torch::Tensor &weight, const OptTensor &bias,
                                                            bool silu, const OptTensor &state, const OptTensor &lengths,
                                                            const OptTensor &offsets) {
    int64_t sequences = 0;
    ssb_short_conv_t p = conv_problem(x, weight, bias, silu, state, lengths, offsets, &sequences);
    need_cuda(x, "short_conv");
    c10::cuda::CUDAGuard guard(x.device());
    torch::Tensor out = empty_like_layout(x), state_out = torch::empty({sequences, p.channels, p.width - 1}, x.options());
    p.out = view_of(out);
    p.state_out = state_out.data_ptr();
    raise_on(ssb_short_conv_fwd(&p, current_stream()), "short_conv");
    return {out, state_out};
}

// -> gradients of x, weight, bias, state
std::vector<OptTensor> short_conv_backward(const torch::Tensor &x, const torch::Tensor &weight, const OptTensor &bias, bool silu,
                                           const OptTensor &state, const OptTensor &lengths, const OptTensor &offsets,
                                           const torch::Tensor &grad_out, const OptTensor &grad_state) {
    int64_t sequences = 0;
    ssb_short_conv_t p = conv_problem(x, weight, bias, silu, state, lengths, offsets, &sequences);
    need_cuda(x, "short_conv");
    check_shape_is(grad_out, x.sizes(), "grad_out");
    check_like(x, grad_out, "grad_out", "x");
    c10::cuda::CUDAGuard guard(x.device());
    ssb_short_conv_grads_t g{};
    g.gout = view_of(grad_out);
    g.gstate_out = window_operand(grad_state, x, {sequences, p.channels, p.width - 1}, "grad_state");
    torch::Tensor gx = empty_like_layout(x), gweight = torch::empty_like(weight);
    OptTensor gbias, gstate;
    g.gx = view_of(gx);
    g.gweight = gweight.data_ptr();
    if (present(bias)) g.gbias = (gbias = torch::empty_like(*bias))->data_ptr();
    if (present(state)) g.gstate = (gstate = torch::empty_like(*state))->data_ptr();
    const size_t bytes = ssb_short_conv_bwd_workspace_bytes(&p);
    torch::Tensor ws = scratch(std::max<size_t>(bytes, 4), x);
    raise_on(ssb_short_conv_bwd(&p, &g, ws.data_ptr(), bytes, current_stream()), "short_conv backward");
    return {gx, gweight, gbias, gstate};
}

torch::Tensor short_conv_step(const torch::Tensor &x, torch::Tensor state, const torch::Tensor &weight, const OptTensor &bias, bool silu,
                              const OptTensor &slots) {
    ssb_short_conv_step_t p{};
    TORCH_CHECK(x.dim() == 2, "x must be 2-D [M, C]");
    p.dtype = element_type(x, "short_conv_step");
    p.silu = silu;
    p.entries = x.size(0);
    p.channels = x.size(1);
    check_width(weight, p.channels);
    p.width = weight.size(1);
    p.weight = tap_operand(weight, x, weight, weight.sizes(), "weight");
    p.bias = tap_operand(bias, x, weight, {p.channels}, "bias");
    p.weight_f32 = weight.scalar_type() == torch::kFloat32;
    p.slots = int_operand(slots, x, "slots");
    if (present(slots)) TORCH_CHECK(slots->size(0) == p.entries, "slots must have one entry per row of x");
    TORCH_CHECK(state.dim() == 3, "state must be 3-D [pool, C, W-1]");
    p.pool = state.size(0);
    p.state = const_cast<void *>(window_operand(state, x, {p.pool, p.channels, p.width - 1}, "state"));
    TORCH_CHECK(present(slots) || p.pool == p.entries, "without slots, state must have one row per row of x");
    need_cuda(x, "short_conv_step");
    c10::cuda::CUDAGuard guard(x.device());
    torch::Tensor out = torch::empty({p.entries, p.channels}, x.options());
    p.x = view_of(x);
    p.out = view_of(out);
    raise_on(ssb_short_conv_step(&p, current_stream()), "short_conv_step");
    mark_written(state);
    return out;
}
