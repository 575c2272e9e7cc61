// The host side of what stands between the projections of a state-space layer, part of host.cpp (inside its anonymous namespace, behind
// host_attention.hpp): argument checks, the outputs' allocation and the launch in one native step, as for the calls there.

decltype(&uniql_causal_conv) p_conv = nullptr;
decltype(&uniql_state_space_scan) p_scan = nullptr;
decltype(&uniql_state_space_scan_workspace) p_scan_workspace = nullptr;
decltype(&uniql_gated_group_norm) p_norm = nullptr;

void bind_state_space(uintptr_t conv, uintptr_t scan, uintptr_t workspace, uintptr_t norm) {
    p_conv = reinterpret_cast<decltype(p_conv)>(conv);
    p_scan = reinterpret_cast<decltype(p_scan)>(scan);
    p_scan_workspace = reinterpret_cast<decltype(p_scan_workspace)>(workspace);
    p_norm = reinterpret_cast<decltype(p_norm)>(norm);
}

// fp16 [rows, channels] with unit inner stride
void require_rows(const Tensor& t, const char* name) {
    if (t.scalar_type() != at::kHalf || t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1))
        fail(std::string(name) + " must be float16 [rows, channels] with unit stride along the channels");
    if (t.size(0) > 0x7fffffff || t.size(1) > 0x7fffffff) fail(std::string(name) + " is larger than a call can take");
    if (t.size(1) == 0) fail(std::string(name) + " has no channels");
}
// [rows, channels] or [rows, heads, width] as the latter
Tensor as_heads(const Tensor& t) { return t.dim() == 2 ? t.unsqueeze(1) : t; }
// Whether the memory between the first and the last element of two tensors has a byte in common.
bool ranges_meet(const Tensor& x, const Tensor& y) {
    if (x.numel() == 0 || y.numel() == 0) return false;
    const auto bytes = [](const Tensor& t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        return (last + 1) * (int64_t)t.element_size();
    };
    const char *a = static_cast<const char*>(x.data_ptr()), *b = static_cast<const char*>(y.data_ptr());
    return a < b + bytes(y) && b < a + bytes(x);
}
// One float a head, or nothing.
const float* per_head(const std::optional<Tensor>& t, const char* name, int64_t heads, const Tensor& like) {
    if (!t) return nullptr;
    require_plain(*t, name, at::kFloat, 1, like);
    if (t->size(0) != heads) fail(std::string(name) + " must have one entry per head");
    return t->data_ptr<float>();
}
Tensor rows_output(const std::optional<Tensor>& out, const Tensor& like) {
    if (!out) return new_output({like.size(0), like.size(1)}, at::kHalf, like);
    require_device(*out, "out", like);
    require_rows(*out, "out");
    if (out->size(0) != like.size(0) || out->size(1) != like.size(1))
        fail("out must be [" + std::to_string(like.size(0)) + ", " + std::to_string(like.size(1)) + "]");
    if (overlaps_itself(as_heads(*out))) fail("out overlaps itself");
    return *out;
}

// Outputs and new states are written while others read; neither may lie in what is read.
void require_apart(const Tensor& out, const char* name, const std::optional<Tensor>& other, const char* other_name) {
    if (other && ranges_meet(out, *other)) fail(std::string(name) + " must not be " + other_name + " or share memory with it");
}

// The sequences of a call and the states that they read and replace: `state` and `state_out` are [places, ...] with `shape` behind.
struct States {
    uniql_sequences sequences;
    void *from, *to;
};
States states_of(const std::optional<Tensor>& state, const std::optional<Tensor>& state_out, const std::optional<Tensor>& cu,
                 const std::optional<Tensor>& places, const std::optional<Tensor>& starts, at::ScalarType type, at::IntArrayRef shape,
                 int64_t rows, const Tensor& like) {
    States s = {};
    const auto check = [&](const Tensor& t, const char* name) {
        require_plain(t, name, type, 1 + (int64_t)shape.size(), like);
        bool fits = t.size(0) <= 0x7fffffff;
        for (size_t i = 0; i < shape.size(); ++i) fits = fits && t.size(1 + (int64_t)i) == shape[i];
        if (!fits) {
            std::string want = "[places";
            for (const int64_t n : shape) want += ", " + std::to_string(n);
            fail(std::string(name) + " must be " + want + "]");
        }
    };
    int64_t pool = 0x7fffffff;
    if (state) {
        check(*state, "state");
        pool = state->size(0);
        s.from = s.to = state->data_ptr();
    }
    if (state_out) {
        check(*state_out, "state_out");
        if (state && state_out->size(0) != pool) fail("state and state_out must have the same places");
        pool = state_out->size(0);
        s.to = state_out->data_ptr();
        if (state && s.to != s.from && ranges_meet(*state, *state_out)) fail("state_out must be state itself or share no memory with it");
    }
    int64_t count = rows;
    if (cu) {
        require_plain(*cu, "cu", at::kInt, 1, like);
        if (cu->size(0) < 1) fail("cu must have at least one entry");
        count = cu->size(0) - 1;
        s.sequences.cu = cu->data_ptr<int>();
    } else if (!state) {
        fail("without cu every row is the next token of a request of its own, which needs a state");
    }
    if (count > (1 << 24)) fail("there must be 2^24 sequences at most");
    if (places) {
        require_plain(*places, "places", at::kInt, 1, like);
        if (places->size(0) != count) fail("places must have one entry per sequence");
        s.sequences.places = places->data_ptr<int>();
    } else if (count > pool) {
        fail("without places there must be one place per sequence");
    }
    if (starts) {
        if (!state) fail("starts without a state");
        require_plain(*starts, "starts", at::kInt, 1, like);
        if (starts->size(0) != count) fail("starts must have one entry per sequence");
        s.sequences.starts = starts->data_ptr<int>();
    }
    if (s.to)
        for (const auto* t : {&cu, &places, &starts}) require_apart(state_out ? *state_out : *state, "state_out", *t, "cu, places or starts");
    s.sequences.count = (int)count;
    s.sequences.pool = (int)pool;
    return s;
}
Tensor causal_conv(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, const std::optional<Tensor>& state,
                   const std::optional<Tensor>& cu, const std::optional<Tensor>& places, const std::optional<Tensor>& starts,
                   const std::optional<Tensor>& state_out, bool activation, const std::optional<Tensor>& out_in, uintptr_t stream) {
    const py::gil_scoped_release release;
    const at::NoGradGuard no_grad;
    require_gpu(x, "x");
    require_rows(x, "x");
    const int64_t rows = x.size(0), channels = x.size(1);
    require_plain(weight, "weight", at::kHalf, 2, x);
    const int64_t width = weight.size(1);
    if (weight.size(0) != channels || width < 2 || width > 4) fail("weight must be [" + std::to_string(channels) + ", 2 to 4]");
    if (bias) {
        require_plain(*bias, "bias", at::kHalf, 1, x);
        if (bias->size(0) != channels) fail("bias must have one entry per channel");
    }
    const c10::DeviceGuard guard(x.device());
    const States s = states_of(state, state_out, cu, places, starts, at::kHalf, {width - 1, channels}, rows, x);
    Tensor out = rows_output(out_in, x);
    if (out_in) {
        if (share_memory(as_heads(out), as_heads(x))) fail("out must not be x or share memory with it");
        for (const auto* t : {&state, &state_out}) require_apart(out, "out", *t, "a state");
        require_apart(out, "out", weight, "weight");
        for (const auto* t : {&bias, &cu, &places, &starts}) require_apart(out, "out", *t, "an input");
    }
    if (s.to) {
        const Tensor& to = state_out ? *state_out : *state;
        for (const Tensor* t : {&x, &weight}) require_apart(to, "state_out", *t, "an input");
        require_apart(to, "state_out", bias, "bias");
    }
    check(p_conv(x.data_ptr(), x.stride(0), weight.data_ptr(), bias ? bias->data_ptr() : nullptr, s.from, s.to, &s.sequences, out.data_ptr(),
                 out.stride(0), (int)rows, (int)channels, (int)width, activation, reinterpret_cast<void*>(stream)),
          "uniql_causal_conv");
    return out;
}

void require_limits(double dt_min, double dt_max) {
    if (!(dt_min >= 0.0 && dt_min <= dt_max)) fail("dt_limit must be two numbers from 0 on, the smaller one first");
}
// The weight of the norm and its groups.
void require_norm(const Tensor& weight, int64_t channels, int64_t groups, double eps, const Tensor& like) {
    require_plain(weight, "weight", at::kHalf, 1, like);
    if (weight.size(0) != channels) fail("weight must have one entry per channel");
    if (groups < 1 || channels % groups) fail("groups must divide the channels");
    if (!(eps >= 0.0)) fail("eps must not be negative");
}

Tensor state_space_scan(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const std::optional<Tensor>& d,
                        const std::optional<Tensor>& dt_bias, bool softplus, double dt_min, double dt_max, const std::optional<Tensor>& state,
                        const std::optional<Tensor>& cu, const std::optional<Tensor>& places, const std::optional<Tensor>& starts,
                        const std::optional<Tensor>& state_out, const std::optional<Tensor>& out_in, uintptr_t stream) {
    const py::gil_scoped_release release;
    const at::NoGradGuard no_grad;
    require_gpu(x, "x");
    require_device(dt, "dt", x);
    require_device(b, "b", x);
    require_device(c, "c", x);
    require_heads(x, "x");
    require_heads(b, "b");
    require_heads(c, "c");
    require_rows(dt, "dt");
    const int64_t rows = x.size(0), heads = x.size(1), head_dim = x.size(2), groups = b.size(1), states = b.size(2);
    if (dt.size(0) != rows || dt.size(1) != heads) fail("dt must have one entry per row and head of x");
    if (b.size(0) != rows || c.sizes() != b.sizes()) fail("b and c must have x's rows, and the same groups and states");
    if (heads % groups) fail("x's heads must be a multiple of b's groups");
    if (head_dim > 128 || states > 256) fail("heads must be 1 to 128 wide, with 1 to 256 states");
    require_limits(dt_min, dt_max);
    const float* const rate = per_head(a, "a", heads, x);
    const float *const skip = per_head(d, "d", heads, x), *const bias = per_head(dt_bias, "dt_bias", heads, x);
    const c10::DeviceGuard guard(x.device());
    const States s = states_of(state, state_out, cu, places, starts, at::kFloat, {heads, head_dim, states}, rows, x);
    Tensor out = heads_output(out_in, "out", rows, heads, head_dim, x);
    if (out_in) {
        if (share_memory(out, x) || share_memory(out, b) || share_memory(out, c) || share_memory(out, as_heads(dt)))
            fail("out must not be x, dt, b or c or share memory with them");
        for (const auto* t : {&state, &state_out}) require_apart(out, "out", *t, "a state");
        require_apart(out, "out", a, "a");
        for (const auto* t : {&d, &dt_bias, &cu, &places, &starts}) require_apart(out, "out", *t, "an input");
    }
    if (s.to) {
        const Tensor& to = state_out ? *state_out : *state;
        for (const Tensor* t : {&x, &dt, &b, &c, &a}) require_apart(to, "state_out", *t, "an input");
        for (const auto* t : {&d, &dt_bias}) require_apart(to, "state_out", *t, "an input");
    }
    size_t need = 0;
    if (cu)
        check(p_scan_workspace((int)rows, s.sequences.count, (int)heads, (int)groups, (int)head_dim, (int)states, &need),
              "uniql_state_space_scan_workspace");
    Tensor temp;
    if (need) temp = new_output({(int64_t)need}, at::kByte, x);
    check(p_scan(x.data_ptr(), x.stride(0), x.stride(1), dt.data_ptr(), dt.stride(0), rate, b.data_ptr(), b.stride(0), b.stride(1),
                 c.data_ptr(), c.stride(0), c.stride(1), skip, bias, softplus, (float)dt_min, (float)dt_max, static_cast<float*>(s.from),
                 static_cast<float*>(s.to), &s.sequences, out.data_ptr(), out.stride(0), out.stride(1), need ? temp.data_ptr() : nullptr,
                 need, (int)rows, (int)heads, (int)groups, (int)head_dim, (int)states, reinterpret_cast<void*>(stream)),
          "uniql_state_space_scan");
    return out;
}

Tensor gated_group_norm(const Tensor& x, const Tensor& z, const Tensor& weight, int64_t groups, double eps, const std::optional<Tensor>& out_in,
                        uintptr_t stream) {
    const py::gil_scoped_release release;
    const at::NoGradGuard no_grad;
    require_gpu(x, "x");
    require_device(z, "z", x);
    require_rows(x, "x");
    require_rows(z, "z");
    const int64_t rows = x.size(0), channels = x.size(1);
    if (z.sizes() != x.sizes()) fail("z must have x's shape");
    require_norm(weight, channels, groups, eps, x);
    const c10::DeviceGuard guard(x.device());
    Tensor out = rows_output(out_in, x);
    if (out_in) {
        const auto same = [&](const Tensor& t) { return out.data_ptr() == t.data_ptr() && (rows < 2 || out.stride(0) == t.stride(0)); };
        for (const Tensor* t : {&x, &z})
            if (!same(*t) && share_memory(as_heads(out), as_heads(*t))) fail("out must be x or z itself or share no memory with them");
        require_apart(out, "out", weight, "weight");
    }
    check(p_norm(x.data_ptr(), x.stride(0), z.data_ptr(), z.stride(0), weight.data_ptr(), out.data_ptr(), out.stride(0), (int)rows,
                 (int)channels, (int)groups, (float)eps, reinterpret_cast<void*>(stream)),
          "uniql_gated_group_norm");
    return out;
}

// What the scan and the norm of a layer would refuse of its parameters and states, asked before the convolution replaces its own states: all three
// are one step of the requests, or none is.
void check_state_space_layer(const Tensor& rows, const Tensor& a, const std::optional<Tensor>& d, const std::optional<Tensor>& dt_bias, double dt_min,
                             double dt_max, const Tensor& state, const std::optional<Tensor>& cu, const std::optional<Tensor>& places,
                             const std::optional<Tensor>& starts, const Tensor& norm_weight, int64_t norm_groups, double eps, int64_t heads,
                             int64_t head_dim, int64_t groups, int64_t states) {
    require_gpu(rows, "projected");
    require_rows(rows, "projected");
    per_head(a, "a", heads, rows);
    per_head(d, "d", heads, rows);
    per_head(dt_bias, "dt_bias", heads, rows);
    require_limits(dt_min, dt_max);
    const States s = states_of(state, std::nullopt, cu, places, starts, at::kFloat, {heads, head_dim, states}, rows.size(0), rows);
    if (reinterpret_cast<uintptr_t>(s.to) & 15u) fail("state must be 16-byte aligned");
    for (const Tensor* t : {&rows, &a}) require_apart(state, "state", *t, "an input");
    for (const auto* t : {&d, &dt_bias}) require_apart(state, "state", *t, "an input");
    size_t need = 0;
    check(p_scan_workspace((int)rows.size(0), s.sequences.count, (int)heads, (int)groups, (int)head_dim, (int)states, &need),
          "uniql_state_space_scan_workspace");
    require_norm(norm_weight, heads * head_dim, norm_groups, eps, rows);
}
