// Host side of the operators around a decode step: the RMS norm (with its autograd node), paged caches, 4-bit projections.
#include "dsqg_torch.h"

namespace {

constexpr at::ScalarType kE4M3 = at::kFloat8_e4m3fn, kE8M0 = at::kFloat8_e8m0fnu;

void need_cuda(const char* who, const Tensor& t) {
    if (!t.is_cuda()) throw std::runtime_error(std::string(who) + ": tensors must live on a CUDA device (there is no CPU path)");
}
int float_code(const char* who, const char* name, at::ScalarType t) {
    if (t == at::kBFloat16) return DSQG_DTYPE_BF16;
    if (t == at::kFloat) return DSQG_DTYPE_F32;
    throw py::type_error(std::string(who) + ": " + name + " must be bfloat16 or float32, got " + toString(t));
}
void no_grad_path(const char* who, std::initializer_list<const Tensor*> ts) {
    if (wants_grad(ts)) throw std::runtime_error(std::string(who) + ": has no backward pass; call it under torch.no_grad()");
}
Tensor rows_in(const Tensor& t) { return t.defined() ? aligned(t.contiguous()) : t; }
std::string dims(std::initializer_list<int64_t> s) {
    std::string r = "[";
    for (int64_t v : s) r += (r.size() > 1 ? "," : "") + std::to_string(v);
    return r + "]";
}

// ------------------------------------------------------------------------------------ RMS norm
struct Normed { Tensor x, w, y, h, scale, rstd; };

Normed norm_forward(const char* who, const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, at::ScalarType y_type, bool with_rstd) {
    need_cuda(who, x);
    if (x.dim() < 1 || x.size(-1) < 1) throw py::value_error(std::string(who) + ": x must be [..., D]");
    const int64_t D = x.size(-1), rows = x.numel() / D;
    if (D > 0x7fffffff || rows > 0x7fffffff) throw py::value_error(std::string(who) + ": too many rows or columns");
    if (!shape_is(weight, {D})) throw py::value_error(std::string(who) + ": weight must be " + dims({D}) + ", got " + shape_of(weight));
    if (residual.defined() && residual.sizes() != x.sizes()) throw py::value_error(std::string(who) + ": residual must have the shape of x, got " + shape_of(residual));
    check_device(who, x, {&weight, &residual});
    dsqg_rms_norm p = {};
    p.x_dtype = float_code(who, "x", x.scalar_type());
    if (residual.defined()) p.stream_dtype = float_code(who, "residual", residual.scalar_type());
    if (!weight.is_floating_point()) throw py::type_error(std::string(who) + ": weight must be a floating-point tensor");
    p.y_dtype = y_type == kE4M3 ? DSQG_DTYPE_E4M3 : float_code(who, "out_dtype", y_type);
    const c10::cuda::CUDAGuard guard(x.device());
    Normed r;
    r.x = rows_in(x);
    r.w = aligned(f32c(weight));
    const Tensor res = rows_in(residual);
    r.y = new_tensor(x.sizes(), y_type, x);
    if (residual.defined()) r.h = new_tensor(x.sizes(), residual.scalar_type(), x);
    if (y_type == kE4M3) r.scale = new_tensor(x.sizes().slice(0, x.dim() - 1), kE8M0, x);
    if (with_rstd) r.rstd = new_tensor({rows}, at::kFloat, x);
    if (!rows) return r;
    p.x = ptr(r.x); p.residual = ptr(res); p.weight = fptr(r.w); p.h = ptr(r.h); p.y = ptr(r.y); p.y_scale = ptr(r.scale); p.rstd = fptr(r.rstd);
    p.rows = rows; p.D = (int)D; p.eps = (float)eps;
    check(dsqg_rms_norm_fwd(&p, stream_of(x)), "dsqg_rms_norm_fwd");
    return r;
}

struct NormNode : torch::autograd::Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& residual, double eps, int64_t y_type) {
        Normed n = norm_forward("rms_norm", x, weight, opt(residual), eps, (at::ScalarType)y_type, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({residual.has_value() ? n.h : n.x, n.rstd, n.w});
        ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)x.scalar_type(), (int64_t)weight.scalar_type(), y_type, residual.has_value()};
        return residual.has_value() ? variable_list{n.y, n.h} : variable_list{n.y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return backward_body(grads[0].defined() || grads.size() < 2 ? grads[0] : grads[1], [&] { return run(ctx, grads); });
    }
    static variable_list run(AutogradContext* ctx, const variable_list& grads) {
        if (at::GradMode::is_enabled()) throw std::runtime_error("rms_norm: has no second derivative (create_graph=True)");
        const variable_list s = ctx->get_saved_variables();
        const Tensor &h = s[0], &rstd = s[1], &w = s[2];
        const auto types = ctx->saved_data["types"].toIntVector();
        const auto x_type = (at::ScalarType)types[0], w_type = (at::ScalarType)types[1], y_type = (at::ScalarType)types[2];
        const bool res = types[3];
        const c10::cuda::CUDAGuard guard(h.device());
        const bool n_x = ctx->needs_input_grad(0), n_w = ctx->needs_input_grad(1), n_r = res && ctx->needs_input_grad(2);
        const Tensor dy = grads[0].defined() ? rows_in(grads[0].to(y_type)) : Tensor();
        const Tensor dh = res && grads[1].defined() ? rows_in(grads[1].to(h.scalar_type())) : Tensor();
        const int64_t D = h.size(-1), rows = h.numel() / D;
        Tensor dx, dr, dw;
        if (!dy.defined()) {                                   // y was not used: only the addition is left
            if (dh.defined() && n_x) dx = dh.to(x_type, /*non_blocking=*/false, /*copy=*/true);
            if (dh.defined() && n_r) dr = dh.clone();
        } else if (!rows) {
            if (n_x) dx = at::zeros(h.sizes(), h.options().dtype(x_type));
            if (n_r) dr = at::zeros_like(h);
            if (n_w) dw = at::zeros({D}, w.options());
        } else if (n_x || n_w || n_r) {
            if (n_x) dx = new_tensor(h.sizes(), x_type, h);
            if (n_r) dr = new_like(h);
            if (n_w) dw = new_like(w);
            dsqg_rms_norm p = {};
            p.x = ptr(h); p.h = ptr(h); p.residual = res ? ptr(h) : nullptr; p.weight = fptr(w); p.rstd = fptr(rstd);
            p.rows = rows; p.D = (int)D;
            p.x_dtype = dtype_code_of(x_type); p.stream_dtype = dtype_code_of(h.scalar_type()); p.y_dtype = dtype_code_of(y_type);
            const size_t bytes = n_w ? dsqg_rms_norm_bwd_scratch_bytes(rows, (int)D) : 0;
            const at::DataPtr scratch = bytes ? scratch_for(bytes) : at::DataPtr();
            check(dsqg_rms_norm_bwd(&p, ptr(dy), ptr(dh), ptr(dx), ptr(dr), fptr(dw), scratch.get(), bytes, stream_of(h)), "dsqg_rms_norm_bwd");
        }
        return {dx, like_param(dw, w_type), dr, Tensor(), Tensor()};
    }
    static int dtype_code_of(at::ScalarType t) { return t == at::kFloat ? DSQG_DTYPE_F32 : DSQG_DTYPE_BF16; }
};

// (y, h); h undefined without a residual
std::tuple<Tensor, std::optional<Tensor>> rms_norm(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& residual, double eps,
                                                   std::optional<at::ScalarType> out_dtype) {
    py::gil_scoped_release no_gil;
    const Tensor res = opt(residual);
    const at::ScalarType y_type = out_dtype.has_value() ? *out_dtype : res.defined() ? res.scalar_type() : x.scalar_type();
    float_code("rms_norm", "out_dtype", y_type);
    if (wants_grad({&x, &weight, &res})) {
        const variable_list r = NormNode::apply(x, weight, residual, eps, (int64_t)y_type);
        return {r[0], res.defined() ? std::optional<Tensor>(r[1]) : std::nullopt};
    }
    Normed n = norm_forward("rms_norm", x, weight, res, eps, y_type, false);
    return {n.y, res.defined() ? std::optional<Tensor>(n.h) : std::nullopt};
}

std::tuple<Tensor, Tensor, std::optional<Tensor>> rms_norm_e4m3(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& residual, double eps) {
    py::gil_scoped_release no_gil;
    const Tensor res = opt(residual);
    no_grad_path("rms_norm_e4m3", {&x, &weight, &res});
    Normed n = norm_forward("rms_norm_e4m3", x, weight, res, eps, kE4M3, false);
    return {n.y, n.scale, res.defined() ? std::optional<Tensor>(n.h) : std::nullopt};
}

// ------------------------------------------------------------------------------------ paged caches
dsqg_pages pages_of(const char* who, const Tensor& kv, const Tensor& table, const Tensor& scale) {
    const std::string w = who;
    need_cuda(who, kv);
    if (kv.dim() != 5 || kv.size(3) != 2 || !kv.is_contiguous()) throw py::value_error(w + ": kv_pages must be contiguous [pages,heads,page_size,2,D], got " + shape_of(kv));
    dsqg_pages p = {};
    p.dtype = kv.scalar_type() == kE4M3 ? DSQG_DTYPE_E4M3 : kv.scalar_type() == at::kBFloat16 ? DSQG_DTYPE_BF16 : DSQG_DTYPE_F32;
    if (p.dtype == DSQG_DTYPE_F32 && kv.scalar_type() != at::kFloat)
        throw py::type_error(w + ": kv_pages must be bfloat16, float32 or float8_e4m3fn, got " + toString(kv.scalar_type()));
    if ((p.dtype == DSQG_DTYPE_E4M3) != scale.defined()) throw py::value_error(w + ": kv_scale belongs to kv_pages in float8_e4m3fn");
    if (scale.defined() && ((scale.scalar_type() != kE8M0 && scale.scalar_type() != at::kByte) || !scale.is_contiguous() ||
                            scale.sizes() != kv.sizes().slice(0, 4)))
        throw py::value_error(w + ": kv_scale must be contiguous [pages,heads,page_size,2] float8_e8m0fnu, got " + shape_of(scale));
    if (table.dim() != 2 || table.scalar_type() != at::kInt || !table.is_contiguous()) throw py::value_error(w + ": block_table must be contiguous int32 [sequences,columns]");
    check_device(who, kv, {&table, &scale});
    for (int i = 0; i < 5; ++i)
        if (kv.size(i) > 0x7fffffff) throw py::value_error(w + ": kv_pages too large");
    if (table.size(0) > 0x7fffffff || table.size(1) > 0x7fffffff) throw py::value_error(w + ": block_table too large");
    p.kv = ptr(kv); p.scale = ptr(scale); p.table = static_cast<const int32_t*>(ptr(table));
    p.sequences = (int)table.size(0); p.columns = (int)table.size(1);
    p.pages = (int)kv.size(0); p.heads = (int)kv.size(1); p.page_size = (int)kv.size(2); p.D = (int)kv.size(4);
    return p;
}
const int32_t* ints(const char* who, const char* name, const Tensor& t, int64_t n, const Tensor& on) {
    if (!t.defined()) return nullptr;
    if (t.scalar_type() != at::kInt || !shape_is(t, {n}) || !t.is_contiguous()) throw py::value_error(std::string(who) + ": " + name + " must be contiguous int32 " + dims({n}));
    check_device(who, on, {&t});
    return static_cast<const int32_t*>(ptr(t));
}
// Rows of D contiguous elements whose token and head strides the kernels take; copied otherwise.
Tensor token_rows(const Tensor& t) {
    return t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && on_16(t.data_ptr()) ? t : aligned(t.contiguous());
}

void paged_kv_write(const Tensor& k0, const Tensor& v0, const Tensor& kv, const Tensor& table, const Tensor& cu, const std::optional<Tensor>& start0,
                    const std::optional<Tensor>& scale0) {
    py::gil_scoped_release no_gil;
    const char* who = "paged_kv_write";
    const Tensor scale = opt(scale0), start = opt(start0);
    const dsqg_pages p = pages_of(who, kv, table, scale);
    no_grad_path(who, {&k0, &v0, &kv});
    if (k0.dim() != 3 || k0.size(1) != p.heads || k0.size(2) != p.D || v0.sizes() != k0.sizes() || v0.scalar_type() != k0.scalar_type())
        throw py::value_error(std::string(who) + ": k and v must be [tokens," + std::to_string(p.heads) + "," + std::to_string(p.D) + "] of one type, got " + shape_of(k0) + " and " + shape_of(v0));
    check_device(who, kv, {&k0, &v0});
    const int dt = float_code(who, "k", k0.scalar_type());
    const int32_t *c = ints(who, "cu_seqlens", cu, p.sequences + 1, kv), *st = ints(who, "start", start, p.sequences, kv);
    if (!k0.size(0) || !p.sequences) return;
    const c10::cuda::CUDAGuard guard(kv.device());
    const Tensor k = token_rows(k0), v = token_rows(v0);
    check(dsqg_paged_write(&p, ptr(k), ptr(v), k.stride(0), k.stride(1), v.stride(0), v.stride(1), c, st, k.size(0), dt, stream_of(kv)), "dsqg_paged_write");
}

std::tuple<Tensor, Tensor> paged_kv_read(const Tensor& kv, const Tensor& table, const Tensor& cu, int64_t tokens, const std::optional<Tensor>& start0,
                                         const std::optional<Tensor>& scale0, at::ScalarType dtype) {
    py::gil_scoped_release no_gil;
    const char* who = "paged_kv_read";
    const Tensor scale = opt(scale0), start = opt(start0);
    const dsqg_pages p = pages_of(who, kv, table, scale);
    const int dt = float_code(who, "dtype", dtype);
    if (tokens < 0) throw py::value_error(std::string(who) + ": tokens must not be negative");
    const int32_t *c = ints(who, "cu_seqlens", cu, p.sequences + 1, kv), *st = ints(who, "start", start, p.sequences, kv);
    const c10::cuda::CUDAGuard guard(kv.device());
    Tensor k = new_tensor({tokens, p.heads, p.D}, dtype, kv), v = new_like(k);
    if (tokens && !p.sequences) { k.zero_(); v.zero_(); }
    if (tokens && p.sequences) check(dsqg_paged_read(&p, ptr(k), ptr(v), c, st, tokens, dt, stream_of(kv)), "dsqg_paged_read");
    return {k, v};
}

Tensor paged_attention_step(const Tensor& q0, const std::optional<Tensor>& k0, const std::optional<Tensor>& v0, const Tensor& kv, const Tensor& table, const Tensor& lengths,
                            const std::optional<Tensor>& scale0, std::optional<double> softmax_scale, std::optional<int64_t> max_length, const std::optional<Tensor>& out0) {
    py::gil_scoped_release no_gil;
    const char* who = "paged_attention_step";
    const std::string w = who;
    const Tensor scale = opt(scale0), kn = opt(k0), vn = opt(v0);
    const dsqg_pages p = pages_of(who, kv, table, scale);
    no_grad_path(who, {&q0, &kn, &vn, &kv});
    const int64_t S = p.sequences;
    if (q0.dim() != 3 || q0.size(0) != S || q0.size(2) != p.D || q0.size(1) < 1 || q0.size(1) % p.heads)
        throw py::value_error(w + ": q must be [" + std::to_string(S) + ",a multiple of " + std::to_string(p.heads) + "," + std::to_string(p.D) + "], got " + shape_of(q0));
    const int dt = float_code(who, "q", q0.scalar_type());
    if (kn.defined() != vn.defined()) throw py::value_error(w + ": k_new and v_new come together");
    for (const Tensor* t : {&kn, &vn})
        if (t->defined() && (!shape_is(*t, {S, p.heads, p.D}) || t->scalar_type() != q0.scalar_type()))
            throw py::value_error(w + ": k_new and v_new must be " + dims({S, p.heads, p.D}) + " of the type of q, got " + shape_of(*t));
    check_device(who, kv, {&q0, &kn, &vn});
    const int32_t* n = ints(who, "lengths", lengths, S, kv);
    const int64_t room = (int64_t)p.columns * p.page_size;
    const int64_t limit = std::min(max_length.has_value() ? *max_length : room, room);
    if (limit < 0) throw py::value_error(w + ": max_length must not be negative");
    if (limit > 0x7fffff00) throw py::value_error(w + ": block_table covers too many positions");
    // in fp32, as the kernels take it: 0 there would stand for the default
    if (softmax_scale.has_value() && !((float)*softmax_scale > 0.f && *softmax_scale < 3e38)) throw py::value_error(w + ": scale must be positive and finite in float32");
    const c10::cuda::CUDAGuard guard(kv.device());
    const Tensor q = rows_in(q0), k = rows_in(kn), v = rows_in(vn);
    Tensor out;
    if (out0.has_value()) {
        out = *out0;
        if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || !out.is_contiguous() || out.device() != kv.device())
            throw py::value_error(w + ": out must be contiguous and like q");
    } else out = new_like(q);
    if (!S) return out;
    const size_t bytes = dsqg_paged_step_scratch_bytes((int)S, p.heads, (int)q.size(1), p.D, (int)limit);
    const at::DataPtr scratch = bytes ? scratch_for(bytes) : at::DataPtr();
    check(dsqg_paged_step(&p, ptr(q), ptr(k), ptr(v), n, (int)q.size(1), (int)limit, softmax_scale.has_value() ? (float)*softmax_scale : 0.f, ptr(out), scratch.get(), bytes, dt,
                          stream_of(kv)), "dsqg_paged_step");
    return out;
}

// ------------------------------------------------------------------------------------ 4-bit projections
Tensor int4_linear(const Tensor& x0, const Tensor& weight, const Tensor& scales, const std::optional<Tensor>& bias0, const std::optional<Tensor>& x_scale0) {
    py::gil_scoped_release no_gil;
    const char* who = "int4_linear";
    const std::string w = who;
    const Tensor bias = opt(bias0), xs0 = opt(x_scale0);
    need_cuda(who, x0);
    no_grad_path(who, {&x0, &scales, &bias});
    if (weight.dim() != 2 || weight.scalar_type() != at::kByte || !weight.is_contiguous()) throw py::value_error(w + ": weight must be contiguous uint8 [N,K/2]");
    const int64_t N = weight.size(0), K = weight.size(1) * 2;
    if (N < 1 || K < 1 || N > 0x7fffffff || K > 0x7fffffff) throw py::value_error(w + ": weight must be [N,K/2], got " + shape_of(weight));
    if (scales.dim() != 2 || scales.scalar_type() != at::kBFloat16 || !scales.is_contiguous() || scales.size(0) != N || scales.size(1) < 1 || K % scales.size(1))
        throw py::value_error(w + ": scales must be contiguous bfloat16 [" + std::to_string(N) + ",K/group], got " + shape_of(scales));
    const int64_t group = K / scales.size(1);
    if (group != 32 && group != 64 && group != 128) throw py::value_error(w + ": a group must be of 32, 64 or 128 columns, got " + std::to_string(group));
    if (x0.dim() < 1 || x0.size(-1) != K) throw py::value_error(w + ": x must be [...," + std::to_string(K) + "], got " + shape_of(x0));
    if (x0.scalar_type() != at::kBFloat16 && x0.scalar_type() != kE4M3) throw py::type_error(w + ": x must be bfloat16 or float8_e4m3fn, got " + toString(x0.scalar_type()));
    const bool f8 = x0.scalar_type() == kE4M3;
    if (f8 != xs0.defined()) throw py::value_error(w + ": x_scale belongs to x in float8_e4m3fn");
    if (f8 && ((xs0.scalar_type() != kE8M0 && xs0.scalar_type() != at::kByte) || xs0.sizes() != x0.sizes().slice(0, x0.dim() - 1)))
        throw py::value_error(w + ": x_scale must be float8_e8m0fnu, one a row of x, got " + shape_of(xs0));
    if (bias.defined() && (!shape_is(bias, {N}) || !bias.is_floating_point())) throw py::value_error(w + ": bias must be " + dims({N}) + ", got " + shape_of(bias));
    check_device(who, x0, {&weight, &scales, &bias, &xs0});
    const c10::cuda::CUDAGuard guard(x0.device());
    std::vector<int64_t> sizes = x0.sizes().vec();
    sizes.back() = N;
    Tensor y = new_tensor(sizes, at::kBFloat16, x0);
    const int64_t M = x0.numel() / K;
    if (!M) return y;
    if (M > 0x7fffffff) throw py::value_error(w + ": too many rows");
    const Tensor x = rows_in(x0), xs = f8 ? xs0.contiguous() : xs0, b = f32c(bias), wt = aligned(weight);
    check(dsqg_int4_linear(ptr(x), ptr(xs), ptr(wt), ptr(scales), fptr(b), ptr(y), (int)M, (int)N, (int)K, (int)group, f8 ? DSQG_DTYPE_E4M3 : DSQG_DTYPE_BF16, stream_of(x)),
          "dsqg_int4_linear");
    return y;
}

}  // namespace

void bind_serving(py::module_& m) {
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_e4m3", &rms_norm_e4m3);
    m.def("paged_kv_write", &paged_kv_write);
    m.def("paged_kv_read", &paged_kv_read);
    m.def("paged_attention_step", &paged_attention_step);
    m.def("int4_linear", &int4_linear);
}
