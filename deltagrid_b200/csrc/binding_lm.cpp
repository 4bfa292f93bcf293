// binding_lm.cpp -- the language-model operators of the compiled module: the gated linear
// recurrence, the gated feed-forward block and token sampling, with their autograd
// functions.  Each call checks its tensors, allocates its outputs with torch's caching
// allocator and calls the C ABI on torch's current stream of the input's device.
#include "binding_util.h"

#include <ATen/autocast_mode.h>
#include <torch/csrc/autograd/custom_function.h>

using namespace dgb;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

typedef c10::optional<Tensor> OptTensor;

inline Tensor value(const OptTensor& t) { return t.has_value() && t->defined() ? *t : Tensor(); }

inline void same_device(const Tensor& ref, const char* op, const char* name, const Tensor& t) {
    check_cuda(t, name);
    TORCH_CHECK(t.device() == ref.device(), op, ": ", name, " is on ", t.device().str(), ", expected ",
                ref.device().str());
}

inline void no_second_order(const char* op) {
    TORCH_CHECK(!at::GradMode::is_enabled(), op, ": the backward pass is not differentiable (create_graph=True)");
}

// tangents would be dropped without a word
inline void no_forward_mode(const char* op, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), op, ": forward-mode differentiation is not supported");
}

inline int to_int(int64_t n, const char* op) {
    TORCH_CHECK(n <= 0x7fffffff, op, ": a size of ", n, " is too large");
    return (int)n;
}

// ---------------------------------------------------------------------------
// gated linear recurrence
// ---------------------------------------------------------------------------

// x, gate, out_gate as the kernels take them: last dimension contiguous, any other strides
inline Tensor rows(const Tensor& t) { return t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

struct ScanArgs {
    Tensor x, gate, out_gate, h0, lengths, resets;
    int code = 0, B = 0, T = 0, D = 0;
};

void check_seq(const ScanArgs& a, const char* op, const char* name, const Tensor& t) {
    same_device(a.x, op, name, t);
    same_dtype(a.x, op, name, t);
    TORCH_CHECK(t.sizes() == a.x.sizes(), op, ": expected ", name, " to have x's shape ", a.x.sizes(), ", got ",
                t.sizes());
}

ScanArgs scan_args(const Tensor& x, const Tensor& gate, const Tensor& out_gate, const Tensor& h0, const Tensor& lengths,
                   const Tensor& resets) {
    const char* op = "gated_scan";
    ScanArgs a;
    check_cuda(x, "x");
    TORCH_CHECK(x.dim() == 3, op, ": expected x [B,T,D], got ", x.sizes());
    a.x = rows(x);
    a.code = dtype_code(x, op);
    TORCH_CHECK(a.code != DG_DTYPE_F64, "\"", op, "\" not implemented for 'Double'");
    check_seq(a, op, "gate", gate);
    a.gate = rows(gate);
    if (out_gate.defined()) {
        check_seq(a, op, "out_gate", out_gate);
        a.out_gate = rows(out_gate);
    }
    a.B = to_int(x.size(0), op), a.T = to_int(x.size(1), op), a.D = to_int(x.size(2), op);
    if (h0.defined()) {
        same_device(x, op, "h0", h0);
        TORCH_CHECK(h0.scalar_type() == at::kFloat && h0.dim() == 2 && h0.size(0) == a.B && h0.size(1) == a.D, op,
                    ": expected h0 to be float32 [B,D]");
        a.h0 = contig(h0);
    }
    if (lengths.defined()) {
        same_device(x, op, "lengths", lengths);
        TORCH_CHECK((lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong) && lengths.dim() == 1 &&
                        lengths.size(0) == a.B, op, ": expected lengths to be int32 or int64 [B]");
        a.lengths = contig(lengths.scalar_type() == at::kInt ? lengths : lengths.clamp(0, a.T).to(at::kInt));
    }
    if (resets.defined()) {
        same_device(x, op, "resets", resets);
        TORCH_CHECK((resets.scalar_type() == at::kBool || resets.scalar_type() == at::kByte) && resets.dim() == 2 &&
                        resets.size(0) == a.B && resets.size(1) == a.T, op, ": expected resets to be bool or uint8 [B,T]");
        a.resets = contig(resets);
    }
    return a;
}

inline int64_t st(const Tensor& t, int d) { return t.defined() ? t.stride(d) : 0; }

struct ScanOut {
    Tensor y, h_last, marks;
};

ScanOut scan_forward(const ScanArgs& a, bool save) {
    ScanOut r;
    const auto f32 = a.x.options().dtype(at::kFloat);
    r.y = at::empty({a.B, a.T, a.D}, a.x.options());
    r.h_last = at::empty({a.B, a.D}, f32);
    if (save) r.marks = at::empty({a.B, (a.T + DG_SCAN_MARK_STEPS - 1) / DG_SCAN_MARK_STEPS, a.D}, f32);
    const c10::cuda::CUDAGuard guard(a.x.device());
    check(dg_gated_scan_forward(a.code, a.B, a.T, a.D, a.x.data_ptr(), st(a.x, 0), st(a.x, 1), a.gate.data_ptr(),
                                st(a.gate, 0), st(a.gate, 1), ptr_or_null(a.out_gate), st(a.out_gate, 0),
                                st(a.out_gate, 1), (const float*)ptr_or_null(a.h0),
                                (const int32_t*)ptr_or_null(a.lengths), (const uint8_t*)ptr_or_null(a.resets),
                                r.y.data_ptr(), r.h_last.data_ptr<float>(), (float*)ptr_or_null(r.marks),
                                status_word(a.x.device()).data_ptr<int32_t>(), stream_of(a.x)),
          "dg_gated_scan_forward");
    return r;
}

// gradients into dx, dgate, dout_gate (views of one tensor or tensors of their own); returns dh0
Tensor scan_backward(const ScanArgs& a, const Tensor& marks, const Tensor& g_y, const Tensor& g_h, const Tensor& dx,
                     const Tensor& dgate, const Tensor& dout, bool want_h0) {
    const auto f32 = a.x.options().dtype(at::kFloat);
    const Tensor dy = g_y.defined() ? rows(g_y) : at::zeros({a.B, a.T, a.D}, a.x.options());
    const Tensor dh = g_h.defined() ? contig(g_h) : Tensor();
    Tensor dh0;
    if (want_h0) dh0 = at::empty({a.B, a.D}, f32);
    const c10::cuda::CUDAGuard guard(a.x.device());
    check(dg_gated_scan_backward(
              a.code, a.B, a.T, a.D, a.x.data_ptr(), st(a.x, 0), st(a.x, 1), a.gate.data_ptr(), st(a.gate, 0),
              st(a.gate, 1), ptr_or_null(a.out_gate), st(a.out_gate, 0), st(a.out_gate, 1),
              (const int32_t*)ptr_or_null(a.lengths), (const uint8_t*)ptr_or_null(a.resets), marks.data_ptr<float>(),
              dy.data_ptr(), st(dy, 0), st(dy, 1), (const float*)ptr_or_null(dh), dx.data_ptr(), st(dx, 0), st(dx, 1),
              dgate.data_ptr(), st(dgate, 0), st(dgate, 1), ptr_or_null(dout), st(dout, 0), st(dout, 1),
              (float*)ptr_or_null(dh0), status_word(a.x.device()).data_ptr<int32_t>(), stream_of(a.x)),
          "dg_gated_scan_backward");
    return dh0;
}

// the parts of a packed [B,T,2D or 3D] tensor: x, gate and, with out_gate, the output gate
std::vector<Tensor> parts_of(const Tensor& p, bool out_gate) {
    const int64_t n = out_gate ? 3 : 2, D = p.size(2) / n;
    std::vector<Tensor> r;
    for (int64_t i = 0; i < 3; ++i) r.push_back(i < n ? p.narrow(2, i * D, D) : Tensor());
    return r;
}

struct GatedScan : public torch::autograd::Function<GatedScan> {
    // packed: x is the packed tensor (gate and out_gate undefined), and so is its gradient
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& gate_,
                                 const OptTensor& out_gate_, const OptTensor& h0_, const OptTensor& lengths_,
                                 const OptTensor& resets_, bool packed, bool packed_out) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor gate = value(gate_), out_gate = value(out_gate_), h0 = value(h0_), lengths = value(lengths_),
                     resets = value(resets_);
        ScanArgs a;
        if (packed) {
            const auto p = parts_of(x, packed_out);
            a = scan_args(p[0], p[1], p[2], h0, lengths, resets);
        } else {
            a = scan_args(x, gate, out_gate, h0, lengths, resets);
        }
        const ScanOut r = scan_forward(a, true);
        ctx->set_materialize_grads(false);
        ctx->saved_data["packed"] = packed;
        ctx->saved_data["packed_out"] = packed_out;
        ctx->saved_data["want_h0"] = h0.defined() && h0.requires_grad();
        if (packed) ctx->save_for_backward({x, Tensor(), Tensor(), a.lengths, a.resets, r.marks});
        else ctx->save_for_backward({a.x, a.gate, a.out_gate, a.lengths, a.resets, r.marks});
        return {r.y, r.h_last};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_second_order("gated_scan");
        const auto s = ctx->get_saved_variables();
        const bool packed = ctx->saved_data["packed"].toBool(), packed_out = ctx->saved_data["packed_out"].toBool();
        const bool want_h0 = ctx->saved_data["want_h0"].toBool();
        if (packed) {
            const auto p = parts_of(s[0], packed_out);
            const ScanArgs a = scan_args(p[0], p[1], p[2], Tensor(), s[3], s[4]);
            const Tensor dp = at::empty({a.B, a.T, s[0].size(2)}, a.x.options());
            const auto d = parts_of(dp, packed_out);
            const Tensor dh0 = scan_backward(a, s[5], grads[0], grads[1], d[0], d[1], d[2], want_h0);
            return {dp, Tensor(), Tensor(), dh0, Tensor(), Tensor(), Tensor(), Tensor()};
        }
        const ScanArgs a = scan_args(s[0], s[1], s[2], Tensor(), s[3], s[4]);
        const Tensor dx = at::empty({a.B, a.T, a.D}, a.x.options()), dg = at::empty_like(dx);
        const Tensor dout = a.out_gate.defined() ? at::empty_like(dx) : Tensor();
        const Tensor dh0 = scan_backward(a, s[5], grads[0], grads[1], dx, dg, dout, want_h0);
        return {dx, dg, dout, dh0, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

inline bool needs_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

std::vector<Tensor> gated_scan(const Tensor& x, const Tensor& gate, const OptTensor& out_gate, const OptTensor& h0,
                               const OptTensor& lengths, const OptTensor& resets) {
    const Tensor o = value(out_gate), h = value(h0), n = value(lengths), r = value(resets);
    no_forward_mode("gated_scan", {&x, &gate, &o, &h});
    if (needs_grad({&x, &gate, &o, &h})) return GatedScan::apply(x, OptTensor(gate), out_gate, h0, lengths, resets, false, false);
    const ScanOut out = scan_forward(scan_args(x, gate, o, h, n, r), false);
    return {out.y, out.h_last};
}

std::vector<Tensor> gated_scan_packed(const Tensor& packed, const OptTensor& h0, const OptTensor& lengths,
                                      const OptTensor& resets, bool out_gate) {
    check_cuda(packed, "packed");
    TORCH_CHECK(packed.dim() == 3 && packed.size(2) % (out_gate ? 3 : 2) == 0, "gated_scan_packed: expected packed [B,T,",
                out_gate ? 3 : 2, "D], got ", packed.sizes());
    const Tensor h = value(h0), n = value(lengths), r = value(resets);
    no_forward_mode("gated_scan_packed", {&packed, &h});
    if (needs_grad({&packed, &h})) return GatedScan::apply(packed, OptTensor(), OptTensor(), h0, lengths, resets, true, out_gate);
    const auto p = parts_of(packed, out_gate);
    const ScanOut out = scan_forward(scan_args(p[0], p[1], p[2], h, n, r), false);
    return {out.y, out.h_last};
}

Tensor gated_scan_step(const Tensor& x, const Tensor& gate, const Tensor& h, const OptTensor& out_gate) {
    const char* op = "gated_scan_step";
    check_cuda(x, "x");
    TORCH_CHECK(x.dim() == 2, op, ": expected x [B,D], got ", x.sizes());
    const int code = dtype_code(x, op);
    TORCH_CHECK(code != DG_DTYPE_F64, "\"", op, "\" not implemented for 'Double'");
    const Tensor o = value(out_gate);
    ScanArgs a;
    a.x = rows(x);
    check_seq(a, op, "gate", gate);
    if (o.defined()) check_seq(a, op, "out_gate", o);
    same_device(x, op, "h", h);
    TORCH_CHECK(h.scalar_type() == at::kFloat && h.sizes() == x.sizes() && h.is_contiguous(), op,
                ": expected h to be contiguous float32 with x's shape (it is updated in place)");
    no_forward_mode(op, {&x, &gate, &o, &h});
    TORCH_CHECK(!needs_grad({&x, &gate, &o, &h}), op, ": has no backward pass (use gated_scan, or torch.no_grad())");
    const Tensor g_c = rows(gate), o_c = o.defined() ? rows(o) : o;
    Tensor y = at::empty(x.sizes(), x.options());
    const c10::cuda::CUDAGuard guard(x.device());
    check(dg_gated_scan_step(code, to_int(x.size(0), op), to_int(x.size(1), op), a.x.data_ptr(), st(a.x, 0),
                             g_c.data_ptr(), st(g_c, 0), ptr_or_null(o_c), st(o_c, 0), h.data_ptr<float>(),
                             y.data_ptr(), stream_of(x)),
          "dg_gated_scan_step");
    // as any in-place operation: a backward pass that has saved h finds that it has changed
    if (!h.is_inference()) h.unsafeGetTensorImpl()->bump_version();
    return y;
}

// ---------------------------------------------------------------------------
// gated feed-forward
// ---------------------------------------------------------------------------

// a matrix as TMA can read it: rows of 16-bit values start on 16-byte boundaries.  One that is laid
// out otherwise is copied, where its row length allows: the copy costs less than the kernel for
// any alignment.
Tensor matrix(const Tensor& t) {
    Tensor r = rows(t);
    if (r.size(0) > 1 && r.stride(0) < r.size(1)) r = r.contiguous();
    const bool off = (reinterpret_cast<uintptr_t>(r.data_ptr()) & 15) || (r.size(0) > 1 && r.stride(0) % 8);
    return off && r.element_size() == 2 && r.size(1) % 8 == 0 ? r.clone(at::MemoryFormat::Contiguous) : r;
}

struct FfnArgs {
    Tensor x, w, b;             // x [M,D] rows
    int code = 0, D = 0, F = 0, act = 0;
    int64_t M = 0;
};

FfnArgs ffn_args(const Tensor& x, const Tensor& w, const Tensor& b, int64_t act) {
    const char* op = "gated_ffn";
    FfnArgs a;
    check_cuda(x, "x");
    a.code = dtype_code(x, op);
    TORCH_CHECK(a.code != DG_DTYPE_F64, "\"", op, "\" not implemented for 'Double'");
    TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && w.size(0) % 2 == 0 && w.size(1) == x.size(-1) && w.size(0) > 0 &&
                    w.size(1) > 0, op, ": expected x [...,D] and weight [2F,D], got ", x.sizes(), " and ", w.sizes());
    same_device(x, op, "weight", w);
    same_dtype(x, op, "weight", w);
    a.D = to_int(w.size(1), op), a.F = to_int(w.size(0) / 2, op), a.act = (int)act;
    a.w = matrix(contig(w));
    if (b.defined()) {
        same_device(x, op, "bias", b);
        same_dtype(x, op, "bias", b);
        TORCH_CHECK(b.dim() == 1 && b.size(0) == w.size(0), op, ": expected bias [2F], got ", b.sizes());
        a.b = matrix(contig(b).view({1, -1}));
    }
    a.x = matrix(x.dim() == 2 ? x : x.contiguous().view({-1, a.D}));
    a.M = a.x.size(0);
    return a;
}

inline int64_t ld(const Tensor& t, int cols) { return t.size(0) > 1 ? t.stride(0) : cols; }

std::vector<int64_t> out_sizes(const Tensor& x, int64_t last) {
    auto s = x.sizes().vec();
    s.back() = last;
    return s;
}

Tensor ffn_forward(const FfnArgs& a, const Tensor& x) {
    Tensor h = at::empty(out_sizes(x, a.F), x.options());
    const c10::cuda::CUDAGuard guard(x.device());
    check(dg_gated_ffn_forward(a.code, a.M, a.D, a.F, a.act, a.x.data_ptr(), ld(a.x, a.D), a.w.data_ptr(),
                               ptr_or_null(a.b), h.data_ptr(), status_word(x.device()).data_ptr<int32_t>(),
                               stream_of(x)),
          "dg_gated_ffn_forward");
    return h;
}

struct GatedFfn : public torch::autograd::Function<GatedFfn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias, int64_t act) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor b = value(bias);
        const FfnArgs a = ffn_args(x, w, b, act);
        ctx->save_for_backward({x, w, b});
        ctx->saved_data["act"] = act;
        ctx->saved_data["want"] = (int64_t)(x.requires_grad() | (w.requires_grad() << 1) |
                                            ((b.defined() && b.requires_grad()) << 2));
        return ffn_forward(a, x);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_second_order("gated_ffn");
        const auto s = ctx->get_saved_variables();
        const FfnArgs a = ffn_args(s[0], s[1], s[2], ctx->saved_data["act"].toInt());
        const int64_t want = ctx->saved_data["want"].toInt();
        const Tensor dh = matrix(grads[0].dim() == 2 ? grads[0] : grads[0].contiguous().view({-1, a.F}));
        Tensor dx, dw, db;
        if (want & 1) dx = at::empty(s[0].sizes(), s[0].options());
        if (want & 2) dw = at::empty(s[1].sizes(), s[1].options());
        if (want & 4) db = at::empty(s[2].sizes(), s[2].options());
        const c10::cuda::CUDAGuard guard(a.x.device());
        const size_t n = dg_gated_ffn_backward_workspace_size(a.code, a.M, a.D, a.F);
        const Tensor ws = at::empty({(int64_t)n}, a.x.options().dtype(at::kByte));
        check(dg_gated_ffn_backward(a.code, a.M, a.D, a.F, a.act, a.x.data_ptr(), ld(a.x, a.D), a.w.data_ptr(),
                                    ptr_or_null(a.b), dh.data_ptr(), ld(dh, a.F), ptr_or_null(dx), ptr_or_null(dw),
                                    ptr_or_null(db), ws.data_ptr(), n,
                                    status_word(a.x.device()).data_ptr<int32_t>(), stream_of(a.x)),
              "dg_gated_ffn_backward");
        return {dx, dw, db, Tensor()};
    }
};

Tensor gated_ffn(const Tensor& x_, const Tensor& weight_, const OptTensor& bias, int64_t activation) {
    Tensor x = x_, weight = weight_, b = value(bias);
    if (at::autocast::is_autocast_enabled(at::kCUDA))
        for (Tensor* t : {&x, &weight, &b})    // as a product of torch's own; f64 is left alone there too
            if (t->defined() && t->is_cuda() && t->is_floating_point() && t->scalar_type() != at::kDouble)
                *t = t->to(at::autocast::get_autocast_dtype(at::kCUDA));
    no_forward_mode("gated_ffn", {&x, &weight, &b});
    if (needs_grad({&x, &weight, &b})) return GatedFfn::apply(x, weight, OptTensor(b), activation);
    return ffn_forward(ffn_args(x, weight, b, activation), x);
}

// ---------------------------------------------------------------------------
// sampling
// ---------------------------------------------------------------------------

// a per-row parameter: a [B] tensor of `type`, or None with the scalar beside it
Tensor per_row(const Tensor& logits, const char* name, const OptTensor& t, at::ScalarType type) {
    const Tensor v = value(t);
    if (!v.defined()) return v;
    same_device(logits, "sample", name, v);
    TORCH_CHECK(v.dim() == 1 && v.size(0) == logits.size(0), "sample: expected ", name, " to be a number or [B], got ",
                v.sizes());
    if (v.scalar_type() == type) return contig(v);
    // a number beyond 32 bits must not wrap around (top_k: any above V keeps all)
    return contig(type == at::kInt ? v.clamp(-1, 1 << 30).to(type) : v.to(type));
}

std::vector<Tensor> sample(const Tensor& logits, const Tensor& u, const OptTensor& temperature, double temperature_v,
                           const OptTensor& top_k, int64_t top_k_v, const OptTensor& top_p, double top_p_v,
                           const OptTensor& min_p, double min_p_v) {
    const char* op = "sample";
    check_cuda(logits, "logits");
    TORCH_CHECK(logits.dim() == 2 && logits.size(1) > 0, op, ": expected logits [B,V], got ", logits.sizes());
    const int code = dtype_code(logits, op);
    TORCH_CHECK(code != DG_DTYPE_F64, "\"", op, "\" not implemented for 'Double'");
    const Tensor l = rows(logits);
    same_device(l, op, "u", u);
    TORCH_CHECK(u.scalar_type() == at::kFloat && u.dim() == 1 && u.size(0) == l.size(0), op,
                ": expected u to be float32 [B]");
    const Tensor u_c = contig(u), t = per_row(l, "temperature", temperature, at::kFloat),
                 k = per_row(l, "top_k", top_k, at::kInt), p = per_row(l, "top_p", top_p, at::kFloat),
                 m = per_row(l, "min_p", min_p, at::kFloat);
    Tensor token = at::empty({l.size(0)}, l.options().dtype(at::kLong));
    Tensor logprob = at::empty({l.size(0)}, l.options().dtype(at::kFloat));
    const int64_t k_v = top_k_v < 0 ? 0 : top_k_v > 0x7fffffff ? 0 : top_k_v;
    const c10::cuda::CUDAGuard guard(l.device());
    check(dg_sample(code, to_int(l.size(0), op), to_int(l.size(1), op), l.data_ptr(), l.stride(0),
                    u_c.data_ptr<float>(), (const float*)ptr_or_null(t), (float)temperature_v,
                    (const int32_t*)ptr_or_null(k), (int32_t)k_v, (const float*)ptr_or_null(p), (float)top_p_v,
                    (const float*)ptr_or_null(m), (float)min_p_v, token.data_ptr<int64_t>(),
                    logprob.data_ptr<float>(), stream_of(l)),
          "dg_sample");
    return {token, logprob};
}

}  // namespace

void dgb::bind_lm(py::module_& m) {
    m.def("gated_scan", &gated_scan, "Gated linear recurrence", py::arg("x"), py::arg("gate"),
          py::arg("out_gate") = py::none(), py::arg("h0") = py::none(), py::arg("lengths") = py::none(),
          py::arg("resets") = py::none());
    m.def("gated_scan_packed", &gated_scan_packed, "Gated linear recurrence of one packed projection",
          py::arg("packed"), py::arg("h0") = py::none(), py::arg("lengths") = py::none(),
          py::arg("resets") = py::none(), py::arg("out_gate") = true);
    m.def("gated_scan_step", &gated_scan_step, "One step of the gated linear recurrence (state in place)",
          py::arg("x"), py::arg("gate"), py::arg("h"), py::arg("out_gate") = py::none());
    m.def("gated_ffn", &gated_ffn, "Gated feed-forward block", py::arg("x"), py::arg("weight"),
          py::arg("bias") = py::none(), py::arg("activation") = 0);
    m.def("sample", &sample, "Token sampling", py::arg("logits"), py::arg("u"), py::arg("temperature"),
          py::arg("temperature_value"), py::arg("top_k"), py::arg("top_k_value"), py::arg("top_p"),
          py::arg("top_p_value"), py::arg("min_p"), py::arg("min_p_value"));
}
