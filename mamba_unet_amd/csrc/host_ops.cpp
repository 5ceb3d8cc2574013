// The host's side of linear attention, of the norms around a block and of gradient clipping: argument checks, outputs and workspaces, autograd and the
// launches, in one native call each.  Their smallest calls (one new token, a prompt of 17, a network's gradients) take the GPU 5 to 25 us; written
// in Python on the ctypes binding the host took 10 to 55.  The kernels are reached through the addresses that _lib hands over (so that an
// A/B build of the library serves both), on torch's current stream of the tensors' device.
#include <algorithm>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/ss2d.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

#define SS2D_CALLS(X) X(ss2d_last_error) X(ss2d_linattn_chunk) X(ss2d_linattn_state_floats) X(ss2d_linattn_segments) X(ss2d_linattn_fwd) X(ss2d_linattn_bwd) \
    X(ss2d_linattn_step) X(ss2d_block_norm_fwd) X(ss2d_block_norm_bwd) X(ss2d_block_norm_bwd_workspace_floats) X(ss2d_colsum) X(ss2d_colsum_workspace_floats) \
    X(ss2d_grad_clip) X(ss2d_grad_clip_workspace_bytes)
struct Api {
#define X(f) decltype(&::f) f = nullptr;
    SS2D_CALLS(X)
#undef X
} api;

std::vector<std::string> names() {
#define X(f) #f,
    return {SS2D_CALLS(X)};
#undef X
}
void bind(const std::map<std::string, uintptr_t> &at) {
#define X(f) api.f = reinterpret_cast<decltype(&::f)>(at.at(#f));
    SS2D_CALLS(X)
#undef X
}

void check_rc(int rc, const char *what) {
    if (!rc) return;
    const std::string msg = api.ss2d_last_error();
    TORCH_CHECK_VALUE(rc > 0, what, ": ", msg, " (rc=", rc, ")");
    TORCH_CHECK(false, what, ": ", msg, " (hipError ", rc, ")");
}

struct Here {                     // the tensors' device is the current one; its current stream
    c10::DeviceGuard guard;
    void *stream;
    explicit Here(at::Device d) : guard(d), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(d.index()).stream()) {}
};

template <typename T = void>
T *ptr(const Tensor &t) { return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr; }
Tensor get(const Maybe &t) { return t ? *t : Tensor(); }
Tensor cast(const Tensor &t, at::ScalarType d) { return !t.defined() || t.scalar_type() == d ? t : t.to(d); }
int code_of(at::ScalarType io) { return io == at::kBFloat16 ? SS2D_DTYPE_BF16 : SS2D_DTYPE_F32; }
std::string shape(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + (s.size() == 1 ? ",)" : ")");
}
Tensor empty(at::IntArrayRef s, at::Device d, at::ScalarType t = at::kFloat) { return at::empty(s, at::TensorOptions().device(d).dtype(t)); }

struct Named {
    const char *name;
    const Tensor *t;
};
// Forward-mode derivatives: the kernels carry no tangents, and leaving them out would make a function's derivative wrong without a word.
void check_no_tangent(const char *op, const Tensor &t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), op, ": forward-mode derivatives are not implemented (a tensor with a tangent was given)");
}
constexpr c10::DispatchKeySet WITHOUT_MEMORY({c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
// most tensors need neither check (reading the tangent itself takes a lock: 15 ns a tensor)
inline bool plain(const Tensor &t) {
    const auto *meta = static_cast<const torch::autograd::AutogradMeta *>(t.unsafeGetTensorImpl()->autograd_meta());
    return (!meta || !meta->fw_grad_) && !t.key_set().has_any(WITHOUT_MEMORY);
}
// Views that stand for other values than their memory holds (the imaginary part of a conjugate: the sign is left to whoever reads it) or for none
void check_memory(const char *op, const Tensor &t) {
    TORCH_CHECK_VALUE(!t.defined() || !t.key_set().has_any(WITHOUT_MEMORY), op, ": a negated view or a tensor without memory was given: call resolve_neg() or clone() on it first");
}
// a tensor with a tangent or without memory of its values raises, and the first one that is not on the GPU, or on another one than the first
void check_tensors(const char *op, std::initializer_list<Named> all) {
    for (const Named &n : all)
        if (n.t->defined() && !plain(*n.t)) {
            check_no_tangent(op, *n.t);
            check_memory(op, *n.t);
        }
    const Named *first = nullptr;
    for (const Named &n : all) {
        if (!n.t->defined()) continue;
        TORCH_CHECK(n.t->is_cuda(), op, ": `", n.name, "` must be a GPU tensor (no CPU path in mamba_unet_amd)");
        if (!first) first = &n;
        TORCH_CHECK_VALUE(n.t->device() == first->t->device(), op, ": `", n.name, "` is on ", n.t->device(), ", `", first->name, "` on ", first->t->device());
    }
}
bool any_requires_grad(std::initializer_list<Named> all) {
    for (const Named &n : all)
        if (n.t->defined() && n.t->requires_grad()) return true;
    return false;
}

// Gradients that come from kernels have no graph of their own: asked for with create_graph they raise when they are differentiated again.
variable_list once(variable_list out) {
    if (!at::GradMode::is_enabled()) return out;
    for (Tensor &t : out)
        if (t.defined()) t = t.detach().set_requires_grad(true);
    return torch::autograd::DelayedError("trying to differentiate twice an operator whose backward is a kernel", (int)out.size())(std::move(out));
}
// dense, in the storage type, on a 16-byte boundary
Tensor dense16(const Tensor &g0, at::ScalarType io) {
    const Tensor g = !g0.defined() ? g0 : g0._is_zerotensor() ? at::zeros(g0.sizes(), g0.options()) : g0.resolve_neg();
    if (!g.defined() || (g.scalar_type() == io && g.is_contiguous() && (uintptr_t)g.data_ptr() % 16 == 0)) return g;
    return g.to(io).clone(at::MemoryFormat::Contiguous);
}

// what hooks on saved tensors gave back in the place of a dense fp32 tensor of this shape
Tensor as_saved(const char *op, const Tensor &t, at::IntArrayRef want) {
    TORCH_CHECK_VALUE(t.sizes() == want, op, ": a saved tensor came back as ", shape(t.sizes()), ", not ", shape(want));
    return cast(t, at::kFloat).contiguous();
}

// ------------------------------------------------------------------------------------------------ linear attention

constexpr int64_t MAX_DIM = 128;

struct Dims {
    int64_t B, L, G, dk, H, dv, N;
};

at::ScalarType storage(const Tensor &q, const Tensor &k, const Tensor &v) {
    return q.scalar_type() == at::kBFloat16 && k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
}

// In the storage type, the last axis dense and the tokens apart by less than 2^22 elements and not overlapping (an expanded or far-flung view is copied; a
// slice of a fused projection is used in place).  bf16 heads made of 16-byte pieces that begin inside a 32-bit word are copied, too.
Tensor operand(const Tensor &t0, at::ScalarType io) {
    const Tensor t = cast(t0, io);
    const int64_t n = t.size(3), s0 = t.stride(0), s1 = t.stride(1), s2 = t.stride(2);
    const bool move = (n > 1 && t.stride(3) != 1) || s1 < n || s1 >= (1 << 22)
        || (n % 8 == 0 && io == at::kBFloat16 && ((uintptr_t)t.data_ptr() % 4 || ((s0 | s1 | s2) & 1)));
    return move ? t.clone(at::MemoryFormat::Contiguous) : t;
}

Dims attention_dims(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, const Tensor &s0, const Tensor &cu) {
    check_tensors("linear_attention_fn", {{"q", &q}, {"k", &k}, {"v", &v}, {"log_decay", &g}, {"initial_state", &s0}, {"cu_seqlens", &cu}});
    TORCH_CHECK_VALUE(q.is_floating_point() && k.is_floating_point() && v.is_floating_point() && g.is_floating_point() && (!s0.defined() || s0.is_floating_point()),
                      "linear_attention_fn: q, k, v, log_decay and initial_state must be floating-point tensors");
    TORCH_CHECK_VALUE(q.dim() == 4 && k.sizes() == q.sizes() && v.dim() == 4 && v.size(0) == q.size(0) && v.size(1) == q.size(1),
                      "q/k must be (batch, L, groups, dk) and equal, v (batch, L, heads, dv): ", shape(q.sizes()), " / ", shape(k.sizes()), " / ", shape(v.sizes()));
    Dims d{q.size(0), q.size(1), q.size(2), q.size(3), v.size(2), v.size(3), q.size(0)};
    TORCH_CHECK_VALUE(d.G > 0 && d.H > 0 && d.H % d.G == 0, d.H, " heads are not a multiple of ", d.G, " key heads");
    TORCH_CHECK_VALUE(d.dk >= 1 && d.dk <= MAX_DIM && d.dv >= 1 && d.dv <= MAX_DIM, "dk ", d.dk, " and dv ", d.dv, " must lie in 1 ... ", MAX_DIM);
    TORCH_CHECK_VALUE(g.sizes() == at::IntArrayRef({d.H}) || g.sizes() == at::IntArrayRef({d.B, d.L, d.H}), "log_decay must be ", shape({d.H}), " or ",
                      shape({d.B, d.L, d.H}), ", got ", shape(g.sizes()));
    if (cu.defined()) {
        TORCH_CHECK_VALUE(cu.dim() == 1 && cu.numel() >= 2 && cu.scalar_type() == at::kInt && cu.is_contiguous(),
                          "cu_seqlens must be a contiguous int32 tensor of at least two offsets");
        TORCH_CHECK_VALUE(d.B == 1, "packed sequences lie in one row: batch must be 1 with cu_seqlens, got ", d.B);
        d.N = cu.numel() - 1;
    }
    TORCH_CHECK_VALUE(!s0.defined() || s0.sizes() == at::IntArrayRef({d.N, d.H, d.dk, d.dv}), "initial_state must be ", shape({d.N, d.H, d.dk, d.dv}), ", got ",
                      s0.defined() ? shape(s0.sizes()) : "");
    TORCH_CHECK_VALUE(d.N > 0, "linear_attention_fn: empty batch");
    return d;
}

struct Strides {                  // batch, token, head of q, k, v, g; a decay for each head only has stride 0 over tokens
    long long s[12];
    Strides(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g) {
        int n = 0;
        for (const Tensor *t : {&q, &k, &v})
            for (int i = 0; i < 3; ++i) s[n++] = t->stride(i);
        for (int i = 0; i < 3; ++i) s[n++] = g.dim() == 3 ? g.stride(i) : i < 2 ? 0 : g.stride(0);
    }
};

struct Segments {
    int nseg, segc;
    Tensor states, decay;
    Segments(int code, const Dims &d, at::Device dev, int64_t longest, bool packed, bool backward) {
        const long long plan = api.ss2d_linattn_segments(code, d.B * d.L, longest, (int)d.H, (int)d.dk, (int)d.dv, backward);
        nseg = (int)(plan >> 32);
        segc = (int)(plan & 0xffffffff);
        if (nseg == 1) return;
        const int64_t slots = packed ? d.L / ((int64_t)segc * api.ss2d_linattn_chunk(code, (int)d.dk, (int)d.dv)) + d.N : d.N * nseg;
        states = empty({slots, d.H, d.dk, d.dv}, dev);
        decay = empty({slots, d.H}, dev, at::kDouble);
    }
};

struct Attention {
    Tensor out, last, chunks;
};
int64_t chunk_slots(int code, const Dims &d, bool packed) {
    const int64_t C = api.ss2d_linattn_chunk(code, (int)d.dk, (int)d.dv);
    return packed ? d.L / C + d.N : d.N * ((d.L + C - 1) / C);
}
// operands as `operand` leaves them; s0 fp32 and dense
Attention attention_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, const Tensor &s0, const Tensor &cu, double scale, const Dims &d,
                            int64_t longest, bool want_last, bool want_chunks) {
    const at::ScalarType io = q.scalar_type();
    const at::Device dev = q.device();
    Attention r;
    r.out = empty({d.B, d.L, d.H, d.dv}, dev, io);
    if (want_last) r.last = empty({d.N, d.H, d.dk, d.dv}, dev);
    if (d.L == 0) {
        if (want_last) s0.defined() ? r.last.copy_(s0) : r.last.zero_();
        return r;
    }
    const int code = code_of(io), dk = (int)d.dk, dv = (int)d.dv;
    if (want_chunks) {
        r.chunks = empty({chunk_slots(code, d, cu.defined()), d.H, (int64_t)api.ss2d_linattn_state_floats(code, dk, dv)}, dev);
    }
    const Segments seg(code, d, dev, longest, cu.defined(), false);
    const Strides st(q, k, v, g);
    const Here here(dev);
    check_rc(api.ss2d_linattn_fwd(code, ptr(q), ptr(k), ptr(v), ptr<float>(g), st.s, ptr<int>(cu), ptr<float>(s0), ptr(r.out), ptr<float>(r.last), ptr<float>(r.chunks),
                                  ptr<float>(seg.states), ptr<double>(seg.decay), (int)d.N, d.L, (int)d.H, (int)d.G, dk, dv, (float)scale, seg.nseg, seg.segc, here.stream),
             "ss2d_linattn_fwd");
    return r;
}

// a decay for every token has a token stride (0 says: one for each head)
Tensor decays(const Tensor &g) {
    const Tensor t = cast(g, at::kFloat);
    return t.dim() == 3 && t.stride(1) == 0 && t.size(1) > 1 ? t.contiguous() : t;
}
Tensor fp32_dense(const Tensor &t) { return t.defined() ? cast(t, at::kFloat).contiguous() : t; }

struct LinearAttention : torch::autograd::Function<LinearAttention> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, const Maybe &s0, const Maybe &cu,
                                 double scale, int64_t longest, bool want_last) {
        const Dims d = attention_dims(q, k, v, g, get(s0), get(cu));
        const at::ScalarType io = storage(q, k, v);
        const Tensor q_ = operand(q, io), k_ = operand(k, io), v_ = operand(v, io), g_ = decays(g);
        const Attention r = attention_forward(q_, k_, v_, g_, fp32_dense(get(s0)), get(cu), scale, d, longest, want_last, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({q_, k_, v_, g_, get(cu), r.chunks});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["meta"] = std::vector<int64_t>{d.B, d.L, d.G, d.dk, d.H, d.dv, d.N, longest, (int64_t)q.scalar_type(), (int64_t)k.scalar_type(),
                                                       (int64_t)v.scalar_type(), (int64_t)g.scalar_type(), s0 ? (int64_t)s0->scalar_type() : -1};
        variable_list out{cast(r.out, v.scalar_type())};
        if (want_last) out.push_back(r.last);
        return out;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const Tensor dout = grads[0], dlast = grads.size() > 1 ? grads[1] : Tensor();
        for (const Tensor &t : grads) check_no_tangent("linear_attention_fn", t);
        variable_list res(9);
        if (!dout.defined() && !dlast.defined()) return res;
        {
            const at::NoGradGuard no_grad;
            run(ctx, dout, dlast, res);
        }
        return once(std::move(res));
    }
    static void run(AutogradContext *ctx, const Tensor &dout, const Tensor &dlast, variable_list &res) {
        const variable_list saved = ctx->get_saved_variables();
        const std::vector<int64_t> m = ctx->saved_data["meta"].toIntVector();
        const Dims d{m[0], m[1], m[2], m[3], m[4], m[5], m[6]};
        const auto type = [&](int i) { return (at::ScalarType)m[8 + i]; };
        const float scale = (float)ctx->saved_data["scale"].toDouble();
        const at::ScalarType io = type(0) == at::kBFloat16 && type(1) == at::kBFloat16 && type(2) == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
        // hooks on saved tensors (offloaded or packed activations) may hand them back in another layout: they are checked and laid out as in the forward
        const Tensor cu = saved[4].defined() ? saved[4].contiguous() : saved[4];
        const Dims now = attention_dims(saved[0], saved[1], saved[2], saved[3], Tensor(), cu);
        TORCH_CHECK_VALUE(now.B == d.B && now.L == d.L && now.G == d.G && now.dk == d.dk && now.H == d.H && now.dv == d.dv && now.N == d.N,
                          "linear_attention_fn: a saved tensor came back with another shape");
        const Tensor q = operand(saved[0], io), k = operand(saved[1], io), v = operand(saved[2], io), g = decays(saved[3]);
        const at::Device dev = q.device();
        Tensor chunks;
        if (d.L > 0) {
            const int code = code_of(io), dk = (int)d.dk, dv = (int)d.dv;
            chunks = as_saved("linear_attention_fn", saved[5], {chunk_slots(code, d, cu.defined()), d.H, (int64_t)api.ss2d_linattn_state_floats(code, dk, dv)});
            check_tensors("linear_attention_fn", {{"q", &q}, {"states", &chunks}});
        }
        const bool want_g = ctx->needs_input_grad(3), want_s0 = m[12] >= 0 && ctx->needs_input_grad(4);
        Tensor dq = empty({d.B, d.L, d.G, d.dk}, dev, io), dk = empty({d.B, d.L, d.G, d.dk}, dev, io), dv = empty({d.B, d.L, d.H, d.dv}, dev, io);
        Tensor dg = empty({d.B, d.L, d.H}, dev), ds0;
        if (want_s0) ds0 = empty({d.N, d.H, d.dk, d.dv}, dev);
        const Tensor gl = dense16(dlast, at::kFloat);
        if (d.L == 0) {
            if (want_s0) gl.defined() ? ds0.copy_(gl) : ds0.zero_();
        } else {
            const Tensor go = dout.defined() ? dense16(dout, io) : at::zeros({d.B, d.L, d.H, d.dv}, v.options());
            Tensor hq, hk;
            if (d.H > d.G) {
                hq = empty({d.B, d.L, d.H, d.dk}, dev);
                hk = empty({d.B, d.L, d.H, d.dk}, dev);
            }
            const int code = code_of(io);
            const Segments seg(code, d, dev, m[7], cu.defined(), true);
            const Strides st(q, k, v, g);
            const Here here(dev);
            check_rc(api.ss2d_linattn_bwd(code, ptr(q), ptr(k), ptr(v), ptr<float>(g), st.s, ptr<int>(cu), ptr(go), ptr<float>(gl), ptr<float>(chunks), ptr(dq), ptr(dk),
                                          ptr(dv), ptr<float>(dg), ptr<float>(ds0), ptr<float>(hq), ptr<float>(hk), ptr<float>(seg.states), ptr<double>(seg.decay),
                                          (int)d.N, d.L, (int)d.H, (int)d.G, (int)d.dk, (int)d.dv, scale, seg.nseg, seg.segc, here.stream),
                     "ss2d_linattn_bwd");
        }
        if (g.dim() == 1 && want_g) {                  // a decay for each head: the sum over all tokens (in a fixed order, and right in a replayed graph)
            const Tensor all = dg;
            dg = d.L > 0 ? empty({d.H}, dev) : at::zeros({d.H}, all.options());
            if (d.L > 0) {
                const Tensor ws = empty({(int64_t)api.ss2d_colsum_workspace_floats((int)d.H)}, dev);
                const Here here(dev);
                check_rc(api.ss2d_colsum(SS2D_DTYPE_F32, ptr(all), ptr<float>(dg), ptr<float>(ws), d.B * d.L, (int)d.H, d.H, here.stream), "ss2d_colsum");
            }
        }
        res[0] = cast(dq, type(0));
        res[1] = cast(dk, type(1));
        res[2] = cast(dv, type(2));
        if (want_g) res[3] = cast(dg, type(3));
        if (want_s0) res[4] = cast(ds0, type(4));
    }
};

py::object attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, std::optional<double> scale0, const Maybe &s0, const Maybe &cu,
                     std::optional<int64_t> max_seqlen, bool want_last) {
    const Tensor s = get(s0), c = get(cu);
    const Dims d = attention_dims(q, k, v, g, s, c);
    const double scale = scale0 ? *scale0 : 1.0 / std::sqrt((double)d.dk);
    const int64_t longest = c.defined() && max_seqlen ? std::min(d.L, std::max<int64_t>(1, *max_seqlen)) : d.L;
    if (at::GradMode::is_enabled() && any_requires_grad({{"", &q}, {"", &k}, {"", &v}, {"", &g}, {"", &s}})) {
        const variable_list r = LinearAttention::apply(q, k, v, g, s0, cu, scale, longest, want_last);
        return want_last ? py::cast(std::make_tuple(r[0], r[1])) : py::cast(r[0]);
    }
    const at::ScalarType io = storage(q, k, v);
    const Attention r = attention_forward(operand(q, io), operand(k, io), operand(v, io), cast(g, at::kFloat), fp32_dense(s), c, scale, d, longest, want_last, false);
    const Tensor out = cast(r.out, v.scalar_type());
    return want_last ? py::cast(std::make_tuple(out, r.last)) : py::cast(out);
}

Tensor token(const Tensor &t0, at::ScalarType io) {
    const Tensor t = cast(t0, io);
    return t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous();
}

Tensor attention_step(const Tensor &state, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, std::optional<double> scale, const Maybe &indices) {
    const Tensor idx = get(indices);
    check_tensors("linear_attention_step", {{"state", &state}, {"q", &q}, {"k", &k}, {"v", &v}, {"log_decay", &g}, {"state_indices", &idx}});
    TORCH_CHECK(!at::GradMode::is_enabled() || !any_requires_grad({{"", &state}, {"", &q}, {"", &k}, {"", &v}, {"", &g}}),
                "linear_attention_step updates its state in place and has no gradient: call it under torch.no_grad(), or linear_attention_fn");
    TORCH_CHECK_VALUE(q.is_floating_point() && k.is_floating_point() && v.is_floating_point() && g.is_floating_point(),
                      "linear_attention_step: q, k, v and log_decay must be floating-point tensors");
    TORCH_CHECK_VALUE(q.dim() == 3 && k.sizes() == q.sizes() && v.dim() == 3 && v.size(0) == q.size(0),
                      "q/k must be (b, groups, dk) and equal, v (b, heads, dv): ", shape(q.sizes()), " / ", shape(k.sizes()), " / ", shape(v.sizes()));
    const int64_t B = q.size(0), G = q.size(1), dk = q.size(2), H = v.size(1), dv = v.size(2);
    TORCH_CHECK_VALUE(G > 0 && H > 0 && H % G == 0, H, " heads are not a multiple of ", G, " key heads");
    TORCH_CHECK_VALUE(dk >= 1 && dk <= MAX_DIM && dv >= 1 && dv <= MAX_DIM, "dk ", dk, " and dv ", dv, " must lie in 1 ... ", MAX_DIM);
    TORCH_CHECK_VALUE(state.scalar_type() == at::kFloat && state.dim() == 4 && state.size(1) == H && state.size(2) == dk && state.size(3) == dv, "state must be fp32 (slots, ",
                      H, ", ", dk, ", ", dv, "), got ", state.scalar_type(), " ", shape(state.sizes()));
    const int64_t pool = state.size(0), n = H * dk * dv, pitch = state.stride(0);
    TORCH_CHECK_VALUE(pool == 0 || (state.select(0, 0).is_contiguous() && (pool == 1 || pitch >= n)),
                      "the slots of state must be dense and must not overlap: it is updated in place");
    TORCH_CHECK_VALUE(g.sizes() == at::IntArrayRef({H}) || g.sizes() == at::IntArrayRef({B, H}), "log_decay must be ", shape({H}), " or ", shape({B, H}), ", got ",
                      shape(g.sizes()));
    Tensor slots;
    if (idx.defined()) {
        TORCH_CHECK_VALUE(idx.dim() == 1 && idx.size(0) == B && (idx.scalar_type() == at::kInt || idx.scalar_type() == at::kLong), "state_indices must be ", shape({B}),
                          " int32 or int64, got ", idx.scalar_type(), " ", shape(idx.sizes()));
        slots = idx.contiguous();
    } else {
        TORCH_CHECK_VALUE(pool == B, B, " requests and ", pool, " states: give state_indices");
    }
    const at::ScalarType io = storage(q, k, v);
    const Tensor q_ = token(q, io), k_ = token(k, io), v_ = token(v, io), g_ = cast(g, at::kFloat);
    Tensor out = empty({B, H, dv}, state.device(), io);
    if (B == 0 || pool == 0) return cast(out.zero_(), v.scalar_type());
    const bool rows = g_.dim() == 2;
    const long long st[8] = {q_.stride(0), q_.stride(1), k_.stride(0), k_.stride(1), v_.stride(0), v_.stride(1), rows ? g_.stride(0) : 0, rows ? g_.stride(1) : g_.stride(0)};
    {
        const Here here(state.device());
        check_rc(api.ss2d_linattn_step(code_of(io), ptr<float>(state), ptr(q_), ptr(k_), ptr(v_), ptr<float>(g_), st, ptr(slots), slots.defined() && slots.scalar_type() == at::kLong,
                                       ptr(out), pool, std::max(n, pitch), (int)B, (int)H, (int)G, (int)dk, (int)dv, (float)(scale ? *scale : 1.0 / std::sqrt((double)dk)),
                                       here.stream),
                 "ss2d_linattn_step");
    }
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();     // (tensors made under inference_mode have no version)
    return cast(out, v.scalar_type());
}

// ------------------------------------------------------------------------------------------------ norms around a block

// (rows, D) rows in the storage type with a dense last axis and one distance between rows: in place where the tensor has that layout (a channel slice of a
// wider tensor), else a copy
struct Rows {
    Tensor t;
    int64_t ld = 0;
    Rows(const Tensor &t0, at::ScalarType io, int64_t D) : t(cast(t0, io)), ld(D) {
        if (!t.defined() || t.is_contiguous()) return;
        const int64_t n = t.dim();
        bool ok = n > 1 && t.stride(n - 1) == 1 && t.stride(n - 2) >= D;
        for (int64_t i = 0; ok && i < n - 2; ++i) ok = t.stride(i) == t.stride(i + 1) * t.size(i + 1);
        if (ok) ld = t.stride(n - 2);
        else t = t.contiguous();
    }
};
at::ScalarType store_type(at::ScalarType t) { return t == at::kBFloat16 ? at::kBFloat16 : at::kFloat; }
Tensor fp32_param(const Tensor &t) { return t.defined() && (t.scalar_type() != at::kFloat || !t.is_contiguous()) ? t.detach().to(at::kFloat).contiguous() : t; }

struct Norms {
    Tensor x_out, h, stats, x, y, z, w1, b1, a, w2, b2, drop;
    int64_t D, rows, ldx, ldy, ldz, rps;
};
Norms norms_forward(const Tensor &x, const Tensor &y, const Tensor &z, const Tensor &w1, const Tensor &b1, const Tensor &a, const Tensor &w2, const Tensor &b2,
                    const Tensor &drop, double eps, bool rms, bool want_stats) {
    Norms r;
    r.D = x.size(-1);
    r.rows = x.numel() / r.D;
    const at::ScalarType rt = store_type(x.scalar_type()), io = store_type(y.scalar_type());
    const Rows rx(x, rt, r.D), ry(y, io, r.D), rz(z, io, r.D);
    r.x = rx.t; r.y = ry.t; r.z = rz.t; r.ldx = rx.ld; r.ldy = ry.ld; r.ldz = rz.ld;
    r.w1 = fp32_param(w1); r.b1 = fp32_param(b1); r.a = fp32_param(a); r.w2 = fp32_param(w2); r.b2 = fp32_param(b2); r.drop = fp32_param(drop);
    const at::Device dev = x.device();
    r.x_out = empty(x.sizes(), dev, rt);
    r.h = empty(x.sizes(), dev, io);
    if (want_stats) r.stats = empty({r.rows, 4}, dev);
    r.rps = drop.defined() && drop.numel() ? r.rows / drop.numel() : 0;
    if (!r.rows) return r;
    const Here here(dev);
    check_rc(api.ss2d_block_norm_fwd(code_of(rt), code_of(io), ptr(r.x), ptr(r.y), ptr(r.z), ptr<float>(r.w1), ptr<float>(r.b1), ptr<float>(r.w2), ptr<float>(r.b2),
                                     ptr<float>(r.a), ptr<float>(r.drop), r.rps, ptr(r.x_out), ptr(r.h), ptr<float>(r.stats), r.rows, (int)r.D, r.ldx, r.ldy, r.ldz,
                                     (float)eps, rms, here.stream),
             "ss2d_block_norm_fwd");
    return r;
}

struct NormGateResidual : torch::autograd::Function<NormGateResidual> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &y, const Maybe &z, const Tensor &w1, const Maybe &b1, const Maybe &a, const Tensor &w2,
                                 const Maybe &b2, const Maybe &drop, double eps, bool rms) {
        const Norms r = norms_forward(x, y, get(z), w1, get(b1), get(a), w2, get(b2), get(drop), eps, rms, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({r.x, r.y, r.z, r.w1, r.b1, r.a, r.w2, r.drop, r.stats});
        std::vector<int64_t> m{r.D, r.rows, r.rps, rms};
        for (const Maybe &t : {Maybe(x), Maybe(y), z, Maybe(w1), b1, a, Maybe(w2), b2}) m.push_back(t ? (int64_t)t->scalar_type() : -1);
        for (const int64_t n : x.sizes()) m.push_back(n);
        ctx->saved_data["meta"] = std::move(m);
        return {cast(r.x_out, x.scalar_type()), cast(r.h, y.scalar_type())};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        variable_list res(11);
        for (const Tensor &t : grads) check_no_tangent("norm_gate_residual", t);
        if (!grads[0].defined() && !grads[1].defined()) return res;
        {
            const at::NoGradGuard no_grad;
            run(ctx, grads[0], grads[1], res);
        }
        return once(std::move(res));
    }
    static void run(AutogradContext *ctx, const Tensor &dxo, const Tensor &dh, variable_list &res) {
        const variable_list saved = ctx->get_saved_variables();
        const std::vector<int64_t> m = ctx->saved_data["meta"].toIntVector();
        const int64_t D = m[0], rows = m[1];
        const at::IntArrayRef sizes(m.data() + 12, m.size() - 12);
        const auto type = [&](int i) { return (at::ScalarType)m[4 + i]; };
        // hooks on saved tensors (offloaded or packed activations) may hand them back in another layout: rows are found anew
        const char *op = "norm_gate_residual";
        check_tensors(op, {{"x", &saved[0]}, {"y", &saved[1]}, {"z", &saved[2]}, {"post_weight", &saved[3]}, {"post_bias", &saved[4]}, {"res_scale", &saved[5]},
                           {"pre_weight", &saved[6]}, {"drop_scale", &saved[7]}, {"statistics", &saved[8]}});
        const auto rows_of = [&](int i) {
            const Tensor &t = saved[i];
            TORCH_CHECK_VALUE(!t.defined() || t.sizes() == sizes, op, ": a saved tensor came back with another shape");
            return Rows(t, store_type(type(i)), D);
        };
        const auto dense = [&](int i, at::IntArrayRef want) { return saved[i].defined() ? as_saved(op, saved[i], want) : saved[i]; };
        const Rows rx = rows_of(0), ry = rows_of(1), rz = rows_of(2);
        const Tensor &x = rx.t, &y = ry.t, &z = rz.t;
        const Tensor w1 = dense(3, {D}), b1 = dense(4, {D}), a = dense(5, {D}), w2 = dense(6, {D}), stats = dense(8, {rows, 4});
        const Tensor drop = saved[7].defined() ? as_saved(op, saved[7], saved[7].sizes()) : saved[7];
        TORCH_CHECK_VALUE(!drop.defined() || drop.numel() * m[2] == rows, op, ": a saved tensor came back with another shape");
        const at::Device dev = x.device();
        const Tensor gx = dense16(dxo, x.scalar_type()), gh = dense16(dh, y.scalar_type());
        Tensor dx = empty(sizes, dev, x.scalar_type()), dy = empty(sizes, dev, y.scalar_type()), dz, dp;
        if (z.defined()) dz = empty(sizes, dev, y.scalar_type());
        if (rows) {
            dp = empty({5, D}, dev);
            const Tensor ws = empty({(int64_t)api.ss2d_block_norm_bwd_workspace_floats(rows, (int)D)}, dev);
            const Here here(dev);
            check_rc(api.ss2d_block_norm_bwd(code_of(x.scalar_type()), code_of(y.scalar_type()), ptr(gx), ptr(gh), ptr(x), ptr(y), ptr(z), ptr<float>(w1), ptr<float>(b1),
                                             ptr<float>(w2), ptr<float>(a), ptr<float>(drop), m[2], ptr<float>(stats), ptr(dx), ptr(dy), ptr(dz), ptr<float>(dp),
                                             ptr<float>(ws), rows, (int)D, rx.ld, ry.ld, rz.ld, (int)m[3], here.stream),
                     "ss2d_block_norm_bwd");
        } else {
            dp = at::zeros({5, D}, w1.options());
        }
        size_t edge = 0;                               // counts the tensors that are there
        for (int i = 0; i < 8; ++i) {
            if (m[4 + i] < 0) continue;
            if (!ctx->needs_input_grad(edge++)) continue;
            const Tensor t = i == 0 ? dx : i == 1 ? dy : i == 2 ? dz : dp.select(0, i - 3);
            res[i] = cast(t, type(i));
        }
    }
};

std::tuple<Tensor, Tensor> norm_gate_residual(const Tensor &x, const Tensor &y, const Tensor &w1, const Tensor &w2, const Maybe &b1, const Maybe &b2, const Maybe &z,
                                              const Maybe &a, const Maybe &drop, double eps, bool rms) {
    const Tensor tb1 = get(b1), tb2 = get(b2), tz = get(z), ta = get(a), td = get(drop);
    check_tensors("norm_gate_residual", {{"x", &x}, {"y", &y}, {"post_weight", &w1}, {"pre_weight", &w2}, {"z", &tz}, {"post_bias", &tb1}, {"pre_bias", &tb2},
                                         {"res_scale", &ta}, {"drop_scale", &td}});
    TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) >= 1 && x.size(-1) <= 8192, "norm_gate_residual: the last axis must hold 1 ... 8192 channels, got ", shape(x.sizes()));
    const auto same = [&](const char *name, const Tensor &t, at::IntArrayRef want) {
        TORCH_CHECK_VALUE(!t.defined() || t.sizes() == want, "norm_gate_residual: `", name, "` must be ", shape(want), ", got ", shape(t.sizes()));
    };
    const at::IntArrayRef vec = x.sizes().slice(x.dim() - 1);
    same("y", y, x.sizes()); same("z", tz, x.sizes());
    same("post_weight", w1, vec); same("pre_weight", w2, vec); same("post_bias", tb1, vec); same("pre_bias", tb2, vec); same("res_scale", ta, vec);
    TORCH_CHECK_VALUE(!td.defined() || (x.dim() > 1 && td.numel() == x.size(0)), "norm_gate_residual: `drop_scale` must hold one factor per sample");
    if (at::GradMode::is_enabled() && any_requires_grad({{"", &x}, {"", &y}, {"", &w1}, {"", &w2}, {"", &tb1}, {"", &tb2}, {"", &tz}, {"", &ta}})) {
        const variable_list r = NormGateResidual::apply(x, y, z, w1, b1, a, w2, b2, drop, eps, rms);
        return {r[0], r[1]};
    }
    const Norms r = norms_forward(x, y, tz, w1, tb1, ta, w2, tb2, td, eps, rms, false);
    return {cast(r.x_out, x.scalar_type()), cast(r.h, y.scalar_type())};
}

// ------------------------------------------------------------------------------------------------ gradient clipping

// whether the first element of `inner` is an element of `t` too (strides in falling order: each index is as large as what is left allows)
bool holds_start_of(const Tensor &t, const Tensor &inner) {
    if (!t.numel() || !inner.numel()) return false;
    int64_t left = (const char *)inner.data_ptr() - (const char *)t.data_ptr();
    const int64_t size = (int64_t)t.element_size();
    if (left < 0 || left % size) return false;
    left /= size;
    std::vector<std::pair<int64_t, int64_t>> axes;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) axes.emplace_back(t.stride(i), t.size(i));
    std::sort(axes.rbegin(), axes.rend());
    for (const auto &[stride, n] : axes)
        if (stride > 0) left -= std::min(left / stride, n - 1) * stride;
    return left == 0;
}

Tensor clip_grad_norm(const py::object &given, double max_norm, double norm_type) {
    std::vector<Tensor> grads;
    const auto take = [&](PyObject *o) {
        if (o == Py_None) return;
        TORCH_CHECK_TYPE(THPVariable_Check(o), "clip_grad_norm: tensors required, got ", Py_TYPE(o)->tp_name);
        const Tensor &t = THPVariable_Unpack(o);
        if (!t.requires_grad() && !PyType_IsSubtype(Py_TYPE(o), reinterpret_cast<PyTypeObject *>(ParameterClass))) {      // (isinstance would run Python code)
            grads.push_back(t);
            return;
        }
        TORCH_CHECK_VALUE(t.is_leaf(), "clip_grad_norm: a tensor with a gradient of its own that is no leaf: give gradients (detached), or the leaves they belong to");
        if (t.grad().defined()) grads.push_back(t.grad());
    };
    if (THPVariable_Check(given.ptr())) take(given.ptr());
    else for (const py::handle &o : given) take(o.ptr());
    TORCH_CHECK_VALUE(max_norm >= 0.0, "clip_grad_norm: max_norm must be >= 0, got ", max_norm);
    const bool inf_norm = std::isinf(norm_type) && norm_type > 0, scale = !std::isinf(max_norm);
    TORCH_CHECK_VALUE(inf_norm || norm_type == 2.0, "clip_grad_norm: norm_type must be 2 or inf, got ", norm_type);
    if (grads.empty()) return at::zeros({});
    const at::NoGradGuard no_grad;
    const at::Device dev = grads[0].device();
    const size_t n = grads.size();
    std::vector<unsigned long long> ptrs(n);
    std::vector<long long> sizes(n);
    std::vector<unsigned char> is_bf16(n);
    std::vector<std::pair<size_t, Tensor>> copies;     // of what is not dense in any order of its axes
    for (size_t i = 0; i < n; ++i) {
        const Tensor &g = grads[i];
        if (!plain(g)) {
            check_no_tangent("clip_grad_norm", g);
            check_memory("clip_grad_norm", g);
        }
        TORCH_CHECK(g.is_cuda(), "clip_grad_norm: GPU tensors required (no CPU path in mamba_unet_amd)");
        TORCH_CHECK_VALUE(g.device() == dev, "clip_grad_norm: gradients on several devices: ", dev, ", ", g.device());
        TORCH_CHECK_VALUE(g.layout() == at::kStrided && (g.scalar_type() == at::kFloat || g.scalar_type() == at::kBFloat16),
                          "clip_grad_norm: dense fp32 or bf16 gradients required, got ", g.scalar_type());
        Tensor w = g;
        if (!g.is_non_overlapping_and_dense()) {
            w = g.contiguous();
            copies.emplace_back(i, w);
        }
        ptrs[i] = (unsigned long long)(uintptr_t)w.data_ptr();
        sizes[i] = w.numel();
        is_bf16[i] = g.scalar_type() == at::kBFloat16;
    }
    // the library looks at the dense ones; a tensor with gaps is clipped in a copy, which shares nothing
    for (const auto &c : copies)
        for (size_t i = 0; i < n; ++i)
            TORCH_CHECK_VALUE(i == c.first || !(holds_start_of(grads[i], grads[c.first]) || holds_start_of(grads[c.first], grads[i])), "clip_grad_norm: tensor ",
                              c.first, " shares memory with another one");
    const size_t bytes = api.ss2d_grad_clip_workspace_bytes((int)n);
    const Tensor norm = empty({}, dev), ws = empty({(int64_t)(bytes / 8)}, dev, at::kDouble);
    {
        const Here here(dev);
        check_rc(api.ss2d_grad_clip(is_bf16.data(), ptrs.data(), sizes.data(), (int)n, inf_norm, (float)max_norm, scale, ptr<float>(norm), ptr<double>(ws), bytes, here.stream),
                 "ss2d_grad_clip");
    }
    if (scale) {
        for (const auto &c : copies) grads[c.first].copy_(c.second);
        for (const Tensor &g : grads)
            if (!g.is_inference()) g.unsafeGetTensorImpl()->bump_version();
    }
    return norm;
}

}  // namespace

PYBIND11_MODULE(_host, m) {
    m.def("names", &names);
    m.def("bind", &bind);
    m.def("attention", torch::wrap_pybind_function(attention));
    m.def("attention_step", torch::wrap_pybind_function(attention_step));
    m.def("norm_gate_residual", torch::wrap_pybind_function(norm_gate_residual));
    m.def("clip_grad_norm", torch::wrap_pybind_function(clip_grad_norm));
}
