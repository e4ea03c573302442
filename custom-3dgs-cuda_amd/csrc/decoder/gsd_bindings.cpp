// gsd_bindings.cpp — the decoder's operators in the custom_rasterizer_cuda
// module, over the C ABI of libgsrdecoder.so.  Outputs and workspaces come from
// torch's caching allocator on the inputs' device; every launch goes on torch's
// current HIP stream.
#include <torch/extension.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <algorithm>
#include <tuple>
#include <vector>

#include "../../../include/gsrdecoder.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

void check_rc(int rc, const char* what) {
    TORCH_CHECK(rc == GSR_OK, "custom_rasterizer_cuda.", what, ": ", gsd_last_error());
}

void* current_stream() {
    return static_cast<void*>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream());
}

int dtype_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case torch::kFloat32: return GSD_F32;
        case torch::kBFloat16: return GSD_BF16;
        case torch::kFloat16: return GSD_F16;
        default: break;
    }
    TORCH_CHECK(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
}

void check_like(const Tensor& t, const char* name, const Tensor& x) {
    TORCH_CHECK(t.is_cuda() && t.device() == x.device(), name,
                " must be a CUDA tensor on the inputs' device");
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must have the inputs' type ",
                x.scalar_type(), ", got ", t.scalar_type());
}

// The kernels read any strides but the last dimension's.
Tensor dense_last(const Tensor& t) {
    return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// The stride of a dimension as the kernels step over it: over one element, never.
int64_t step(const Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// The attention kernels reach a tile's rows by offsets from its first: keys at
// strides in [0, GSD_MAX_ATTENTION_STRIDE] or less, queries (in the backward) so that 65
// of them and a group's heads span at most 2^30 elements.
Tensor near_keys(const Tensor& t, bool mask) {
    if (t.dim() != 4) return t;
    // with a mask, keys are reached by offsets from the first
    const int64_t span = (INT64_C(1) << 30) - 1024;
    const auto fits = [&](int64_t stride) {
        return stride >= 0 && stride <= GSD_MAX_ATTENTION_STRIDE &&
               !(mask && t.size(1) > 0 && stride >= span / t.size(1));
    };
    if (fits(step(t, 1))) return dense_last(t);
    if (fits(t.size(2) * t.size(3))) return t.contiguous();
    return t.transpose(1, 2).contiguous().transpose(1, 2);  // head by head
}
Tensor near_queries(const Tensor& t, int64_t group) {
    const int64_t most = INT64_C(1) << 30;
    const int64_t l = step(t, 1), h = step(t, 2);
    const bool ok = l >= 0 && h >= 0 && l < most / 65 && h < most / group &&
                    65 * l + group * h + t.size(3) <= most;
    return ok ? dense_last(t) : t.contiguous();
}

Tensor workspace(size_t bytes, const Tensor& like) {
    return torch::empty({(int64_t)bytes}, like.options().dtype(torch::kUInt8));
}
void* ptr(const Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; }

// ---- rotary positions ----
Tensor rotary_axes(const Tensor& x_in, const Tensor& positions, const Tensor& inv_freq,
                   const std::vector<int64_t>& sections, bool interleaved, bool inverse) {
    TORCH_CHECK(x_in.is_cuda(), "x must be a CUDA tensor");
    TORCH_CHECK(x_in.dim() == 4, "x must have shape (batch, length, heads, dim)");
    gsd_rotary a{};
    a.dtype = dtype_of(x_in, "x");
    TORCH_CHECK(!sections.empty() && sections.size() <= GSD_MAX_AXES,
                "sections must name between 1 and ", GSD_MAX_AXES, " axes");
    const int64_t axes = (int64_t)sections.size();
    int64_t pairs = 0;
    for (int64_t i = 0; i < axes; ++i) {
        a.sections[i] = sections[i];
        TORCH_CHECK(sections[i] >= 0 && sections[i] <= x_in.size(3), "sections[", i,
                    "] is out of range");
        pairs += sections[i];
    }
    TORCH_CHECK(2 * pairs <= x_in.size(3), "the sections turn ", 2 * pairs, " channels of ",
                x_in.size(3));
    TORCH_CHECK(positions.is_cuda() && positions.device() == x_in.device() &&
                    inv_freq.is_cuda() && inv_freq.device() == x_in.device(),
                "positions and inv_freq must be CUDA tensors on x's device");
    TORCH_CHECK((positions.dim() == 2 && positions.size(0) == x_in.size(1)) ||
                    (positions.dim() == 3 && positions.size(0) == x_in.size(0) &&
                     positions.size(1) == x_in.size(1)),
                "positions must have shape (length, axes) or (batch, length, axes)");
    TORCH_CHECK(positions.size(-1) == axes, "positions must hold one value per section, ", axes,
                ", got ", positions.size(-1));
    switch (positions.scalar_type()) {
        case torch::kFloat32: a.positions_type = GSD_POS_F32; break;
        case torch::kInt32: a.positions_type = GSD_POS_I32; break;
        case torch::kInt64: a.positions_type = GSD_POS_I64; break;
        default:
            TORCH_CHECK(false, "positions must be float32, int32 or int64, got ",
                        positions.scalar_type());
    }
    TORCH_CHECK(inv_freq.scalar_type() == torch::kFloat32 && inv_freq.dim() == 1 &&
                    inv_freq.size(0) == pairs && inv_freq.is_contiguous(),
                "inv_freq must be a contiguous float32 tensor of ", pairs, " values");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x_in.device());
    const Tensor x = dense_last(x_in);
    Tensor y = torch::empty(x.sizes(), x.options());
    a.batch = x.size(0);
    a.length = x.size(1);
    a.heads = x.size(2);
    a.dim = x.size(3);
    if (x.numel() == 0) return y;
    a.x = x.data_ptr();
    a.x_stride_b = x.stride(0);
    a.x_stride_l = x.stride(1);
    a.x_stride_h = x.stride(2);
    a.positions = ptr(positions);
    const bool batched = positions.dim() == 3;
    a.pos_stride_b = batched ? positions.stride(0) : 0;
    a.pos_stride_l = positions.stride(batched ? 1 : 0);
    a.pos_stride_a = positions.stride(batched ? 2 : 1);
    a.axes = (int)axes;
    a.inv_freq = static_cast<const float*>(ptr(inv_freq));
    a.interleaved = interleaved;
    a.inverse = inverse;
    a.y = y.data_ptr();
    check_rc(gsd_rotary_axes(&a, current_stream()), "rotary_axes");
    return y;
}

// ---- the norm with the residual's addition ----
// x as rows: any leading dimensions that one row stride describes, else a copy
struct Rows {
    Tensor t;
    int64_t rows, stride;
};
Rows rows_of(const Tensor& x) {
    const int64_t width = x.size(-1);
    const int64_t rows = width ? x.numel() / width : 0;
    if (x.is_contiguous()) return {x, rows, width};
    if (x.stride(-1) == 1 || width == 1) {
        // leading dimensions that fold into one
        int64_t stride = 0;
        bool fold = true, first = true;
        int64_t expect = 0;
        for (int64_t d = x.dim() - 2; d >= 0; --d) {
            if (x.size(d) == 1) continue;
            if (first) {
                stride = x.stride(d);
                first = false;
            } else if (x.stride(d) != expect) {
                fold = false;
            }
            expect = x.stride(d) * x.size(d);
        }
        if (fold) return {x, rows, first ? width : stride};
    }
    const Tensor c = x.contiguous();
    return {c, rows, width};
}

void check_norm_inputs(const Tensor& x, const OptTensor& residual, const Tensor& weight) {
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    dtype_of(x, "x");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= GSD_MAX_NORM_WIDTH,
                "x's last dimension must lie in [1, ", GSD_MAX_NORM_WIDTH, "]");
    check_like(weight, "weight", x);
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == x.size(-1) && weight.is_contiguous(),
                "weight must be contiguous with shape (", x.size(-1), ",)");
    if (residual.has_value()) {
        check_like(*residual, "residual", x);
        TORCH_CHECK(residual->sizes() == x.sizes(), "Shape mismatch: residual ",
                    residual->sizes(), " vs x ", x.sizes());
    }
}

// (y, h, rstd); h is x itself where there is no residual
std::tuple<Tensor, Tensor, Tensor> rms_norm_residual(const Tensor& x, const OptTensor& residual,
                                                     const Tensor& weight, double eps,
                                                     bool want_rstd) {
    check_norm_inputs(x, residual, weight);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const Rows xr = rows_of(x);
    Rows rr{};
    if (residual.has_value()) rr = rows_of(*residual);
    Tensor y = torch::empty(x.sizes(), x.options());
    Tensor h = residual.has_value() ? torch::empty(x.sizes(), x.options()) : x;
    Tensor rstd = torch::empty({want_rstd ? xr.rows : 0}, x.options().dtype(torch::kFloat32));
    gsd_norm a{};
    a.dtype = dtype_of(x, "x");
    a.rows = xr.rows;
    a.width = x.size(-1);
    a.x = ptr(xr.t);
    a.x_stride = xr.stride;
    a.residual = residual.has_value() ? ptr(rr.t) : nullptr;
    a.residual_stride = rr.stride;
    a.weight = weight.data_ptr();
    a.eps = eps;
    a.h = residual.has_value() ? ptr(h) : nullptr;
    a.rstd = want_rstd ? static_cast<float*>(ptr(rstd)) : nullptr;
    check_rc(gsd_rms_norm(&a, ptr(y), current_stream()), "rms_norm_residual");
    return {y, h, rstd};
}

// (y8, scale, h)
std::tuple<Tensor, Tensor, Tensor> rms_norm_residual_fp8(const Tensor& x,
                                                         const OptTensor& residual,
                                                         const Tensor& weight, double eps) {
    check_norm_inputs(x, residual, weight);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const Rows xr = rows_of(x);
    Rows rr{};
    if (residual.has_value()) rr = rows_of(*residual);
    Tensor y = torch::empty(x.sizes(), x.options().dtype(torch::kFloat8_e4m3fn));
    Tensor h = residual.has_value() ? torch::empty(x.sizes(), x.options()) : x;
    Tensor scale = torch::empty(x.sizes().slice(0, x.dim() - 1),
                                x.options().dtype(torch::kFloat32));
    gsd_norm a{};
    a.dtype = dtype_of(x, "x");
    a.rows = xr.rows;
    a.width = x.size(-1);
    a.x = ptr(xr.t);
    a.x_stride = xr.stride;
    a.residual = residual.has_value() ? ptr(rr.t) : nullptr;
    a.residual_stride = rr.stride;
    a.weight = weight.data_ptr();
    a.eps = eps;
    a.h = residual.has_value() ? ptr(h) : nullptr;
    check_rc(gsd_rms_norm_fp8(&a, static_cast<uint8_t*>(ptr(y)), static_cast<float*>(ptr(scale)),
                              current_stream()),
             "rms_norm_residual_fp8");
    return {y, scale, h};
}

// (dx, dweight): dx is the gradient of x and of the residual
std::tuple<Tensor, Tensor> rms_norm_residual_backward(const Tensor& h_in, const Tensor& rstd,
                                                      const Tensor& weight, const Tensor& dy,
                                                      const OptTensor& dh) {
    check_norm_inputs(h_in, dh, weight);
    check_like(dy, "dy", h_in);
    TORCH_CHECK(dy.sizes() == h_in.sizes(), "Shape mismatch: dy ", dy.sizes(), " vs h ",
                h_in.sizes());
    c10::hip::HIPGuardMasqueradingAsCUDA guard(h_in.device());
    const Tensor h = h_in.contiguous();
    const int64_t width = h.size(-1), rows = h.numel() / width;
    TORCH_CHECK(rstd.is_cuda() && rstd.device() == h.device() &&
                    rstd.scalar_type() == torch::kFloat32 && rstd.is_contiguous() &&
                    rstd.numel() == rows,
                "rstd must be the forward's");
    const Rows yr = rows_of(dy);
    Rows hr{};
    if (dh.has_value()) hr = rows_of(*dh);
    Tensor dx = torch::empty(h.sizes(), h.options());
    Tensor dw = torch::empty(weight.sizes(), weight.options());
    Tensor ws = workspace(gsd_rms_norm_backward_workspace_bytes(rows, width), h);
    check_rc(gsd_rms_norm_backward(dtype_of(h, "h"), rows, width, ptr(h),
                                   static_cast<const float*>(ptr(rstd)), weight.data_ptr(),
                                   ptr(yr.t), yr.stride, dh.has_value() ? ptr(hr.t) : nullptr,
                                   hr.stride, ptr(dx), dw.data_ptr(), ptr(ws),
                                   (size_t)ws.numel(), current_stream()),
             "rms_norm_residual_backward");
    return {dx, dw};
}

// ---- cross attention ----
gsd_attention attention_args(const Tensor& q, const Tensor& k, const Tensor& v,
                             const OptTensor& lengths, const OptTensor& mask, double scale) {
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    TORCH_CHECK(q.scalar_type() == torch::kBFloat16 || q.scalar_type() == torch::kFloat16,
                "q must be bfloat16 or float16, got ", q.scalar_type());
    check_like(k, "k", q);
    check_like(v, "v", q);
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
                "q, k and v must have shape (batch, length, heads, dim)");
    TORCH_CHECK(k.sizes() == v.sizes(), "Shape mismatch: k ", k.sizes(), " vs v ", v.sizes());
    TORCH_CHECK(k.size(0) == q.size(0) && k.size(3) == q.size(3),
                "k and v must have q's batch and dim: q ", q.sizes(), ", k ", k.sizes());
    TORCH_CHECK(q.size(2) >= 1 && k.size(2) >= 1 && q.size(2) % k.size(2) == 0, "q's ",
                q.size(2), " heads must be a multiple of k's ", k.size(2));
    TORCH_CHECK(q.size(3) >= 8 && q.size(3) <= GSD_MAX_HEAD_DIM && q.size(3) % 8 == 0,
                "dim must be a multiple of 8 in [8, ", GSD_MAX_HEAD_DIM, "], got ", q.size(3));
    gsd_attention a{};
    a.dtype = dtype_of(q, "q");
    a.batch = q.size(0);
    a.queries = q.size(1);
    a.keys = k.size(1);
    a.heads = q.size(2);
    a.kv_heads = k.size(2);
    a.dim = q.size(3);
    a.q = ptr(q);
    a.q_stride_b = step(q, 0);
    a.q_stride_l = step(q, 1);
    a.q_stride_h = step(q, 2);
    a.k = ptr(k);
    a.k_stride_b = step(k, 0);
    a.k_stride_l = step(k, 1);
    a.k_stride_h = step(k, 2);
    a.v = ptr(v);
    a.v_stride_b = step(v, 0);
    a.v_stride_l = step(v, 1);
    a.v_stride_h = step(v, 2);
    if (lengths.has_value()) {
        TORCH_CHECK(lengths->is_cuda() && lengths->device() == q.device() &&
                        lengths->scalar_type() == torch::kInt32 && lengths->dim() == 1 &&
                        lengths->size(0) == q.size(0) && lengths->is_contiguous(),
                    "key_lengths must be a contiguous int32 CUDA tensor of shape (batch,)");
        a.key_lengths = static_cast<const int32_t*>(ptr(*lengths));
    }
    if (mask.has_value()) {
        TORCH_CHECK(mask->is_cuda() && mask->device() == q.device() &&
                        mask->scalar_type() == torch::kBool && mask->dim() == 2 &&
                        mask->size(0) == q.size(0) && mask->size(1) == k.size(1),
                    "key_mask must be a bool CUDA tensor of shape (batch, keys)");
        a.key_mask = static_cast<const uint8_t*>(ptr(*mask));
        a.mask_stride_b = mask->stride(0);
        a.mask_stride_s = mask->stride(1);
    }
    a.scale = (float)scale;
    return a;
}

// (o, lse, o_low); the last two, which the backward takes, are empty unless wanted
std::tuple<Tensor, Tensor, Tensor> cross_attention(const Tensor& q_in, const Tensor& k_in,
                                           const Tensor& v_in, const OptTensor& key_lengths,
                                           const OptTensor& key_mask, double scale,
                                           bool for_backward) {
    TORCH_CHECK(q_in.dim() == 4 && k_in.dim() == 4 && v_in.dim() == 4,
                "q, k and v must have shape (batch, length, heads, dim)");
    c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard;
    if (q_in.is_cuda()) guard.set_device(q_in.device());
    const Tensor q = dense_last(q_in), k = near_keys(k_in, key_mask.has_value()),
                 v = near_keys(v_in, key_mask.has_value());
    gsd_attention a = attention_args(q, k, v, key_lengths, key_mask, scale);
    Tensor o = torch::empty(q.sizes(), q.options());
    Tensor lse, o_low;
    a.o = ptr(o);
    if (for_backward) {
        lse = torch::empty({a.batch * a.heads * a.queries}, q.options().dtype(torch::kFloat32));
        o_low = torch::empty(q.sizes(), q.options());
        a.lse = static_cast<float*>(ptr(lse));
        a.o_low = ptr(o_low);
    }
    const size_t bytes = gsd_attention_workspace_bytes(&a);
    Tensor ws;
    if (bytes) ws = workspace(bytes, q);
    check_rc(gsd_cross_attention(&a, bytes ? ws.data_ptr() : nullptr, bytes, current_stream()),
             "cross_attention");
    if (!for_backward) return {o, torch::empty({0}, o.options()), torch::empty({0}, o.options())};
    return {o, lse, o_low};
}

// want_dq, want_dkv: the gradients that are formed; the others come back empty
std::tuple<Tensor, Tensor, Tensor> cross_attention_backward(
    const Tensor& grad_in, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
    const Tensor& o, const Tensor& lse, const Tensor& o_low, const OptTensor& key_lengths,
    const OptTensor& key_mask, double scale, bool want_dq, bool want_dkv) {
    TORCH_CHECK(q_in.dim() == 4 && k_in.dim() == 4 && v_in.dim() == 4,
                "q, k and v must have shape (batch, length, heads, dim)");
    c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard;
    if (q_in.is_cuda()) guard.set_device(q_in.device());
    const int64_t group = std::max<int64_t>(1, q_in.size(2) / std::max<int64_t>(1, k_in.size(2)));
    const Tensor q = near_queries(q_in, group), k = near_keys(k_in, key_mask.has_value()),
                 v = near_keys(v_in, key_mask.has_value());
    gsd_attention a = attention_args(q, k, v, key_lengths, key_mask, scale);
    check_like(grad_in, "grad_output", q);
    check_like(o, "o", q);
    check_like(o_low, "o_low", q);
    TORCH_CHECK(grad_in.sizes() == q.sizes(), "Shape mismatch: grad_output ", grad_in.sizes(),
                " vs q ", q.sizes());
    TORCH_CHECK(o.sizes() == q.sizes() && o.is_contiguous() && o_low.sizes() == q.sizes() &&
                    o_low.is_contiguous() && lse.is_cuda() &&
                    lse.device() == q.device() && lse.scalar_type() == torch::kFloat32 &&
                    lse.is_contiguous() && lse.numel() == a.batch * a.heads * a.queries,
                "o, lse and o_low must be the forward's");
    const Tensor grad = near_queries(grad_in, group);
    a.o = ptr(o);
    a.o_low = ptr(o_low);
    a.lse = static_cast<float*>(ptr(lse));
    Tensor dq, dk, dv;
    dq = want_dq ? torch::empty(q.sizes(), q.options()) : torch::empty({0}, q.options());
    dk = want_dkv ? torch::empty(k.sizes(), k.options()) : torch::empty({0}, q.options());
    dv = want_dkv ? torch::empty(v.sizes(), v.options()) : torch::empty({0}, q.options());
    gsd_attention_grad g{};
    g.d_o = ptr(grad);
    g.do_stride_b = step(grad, 0);
    g.do_stride_l = step(grad, 1);
    g.do_stride_h = step(grad, 2);
    g.dq = ptr(dq);
    g.dk = ptr(dk);
    g.dv = ptr(dv);
    const size_t bytes = gsd_attention_backward_workspace_bytes(&a);
    Tensor ws = workspace(bytes, q);
    check_rc(gsd_cross_attention_backward(&a, &g, ptr(ws), bytes, current_stream()),
             "cross_attention_backward");
    return {dq, dk, dv};
}

// ---- the same as differentiable calls ----
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }
Tensor or_undefined(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

bool wants_grad(std::initializer_list<Tensor> inputs) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : inputs)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

// The gradients are formed by kernels that record nothing: a gradient that depends on
// something that requires one, the incoming gradients or an input (where a constant
// comes in, as sum()'s, that input alone), raises when it is differentiated again.
Tensor once(const Tensor& t, bool depends, const char* what) {
    if (!t.defined() || !depends || !at::GradMode::is_enabled()) return t;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string(what) + " is differentiable once", 1);
    return (*error)({t.detach().set_requires_grad(true)})[0];
}
bool any_requires_grad(const tensor_list& list) {
    for (const Tensor& t : list)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions,
                          const Tensor& inv_freq, const std::vector<int64_t>& sections,
                          bool interleaved) {
        ctx->save_for_backward({positions, inv_freq});
        ctx->saved_data["sections"] = sections;
        ctx->saved_data["interleaved"] = interleaved;
        return rotary_axes(x, positions, inv_freq, sections, interleaved, false);
    }
    static tensor_list backward(AutogradContext* ctx, const tensor_list& grads) {
        const tensor_list saved = ctx->get_saved_variables();
        tensor_list out(5);
        {
            at::AutoGradMode off(false);
            out[0] = rotary_axes(grads[0], saved[0], saved[1],
                                 ctx->saved_data["sections"].toIntVector(),
                                 ctx->saved_data["interleaved"].toBool(), true);
        }
        out[0] = once(out[0], any_requires_grad(grads), "rotary_axes");  // linear in x
        return out;
    }
};

Tensor decoder_rotary(const Tensor& x, const Tensor& positions, const Tensor& inv_freq,
                      const std::vector<int64_t>& sections, bool interleaved) {
    if (wants_grad({x}))
        return RotaryFunction::apply(x, positions, inv_freq, sections, interleaved);
    return rotary_axes(x, positions, inv_freq, sections, interleaved, false);
}

struct NormFunction : torch::autograd::Function<NormFunction> {
    // Without a residual h is x itself: the gradient that reaches x through it is
    // added by the backward kernel all the same.
    static tensor_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual,
                               const Tensor& weight, double eps) {
        auto [y, h, rstd] = rms_norm_residual(x, residual, weight, eps, true);
        ctx->save_for_backward({h, rstd, weight});
        ctx->saved_data["residual"] = residual.has_value();
        ctx->saved_data["of_h"] = any_requires_grad({x, or_undefined(residual)});
        ctx->set_materialize_grads(false);
        return {y, h};
    }
    static tensor_list backward(AutogradContext* ctx, const tensor_list& grads) {
        const tensor_list saved = ctx->get_saved_variables();
        const bool residual = ctx->saved_data["residual"].toBool();
        tensor_list out(4);
        if (!grads[0].defined()) {
            out[0] = grads[1];
        } else {
            {
                at::AutoGradMode off(false);
                std::tie(out[0], out[2]) = rms_norm_residual_backward(saved[0], saved[1], saved[2],
                                                                      grads[0], opt(grads[1]));
            }
            const bool of_h = ctx->saved_data["of_h"].toBool() || any_requires_grad(grads);
            out[0] = once(out[0], of_h || saved[2].requires_grad(), "rms_norm_residual");
            out[2] = once(out[2], of_h, "rms_norm_residual");
        }
        if (residual) out[1] = out[0];
        return out;
    }
};

std::tuple<Tensor, Tensor> decoder_norm(const Tensor& x, const OptTensor& residual,
                                        const Tensor& weight, double eps) {
    const Tensor r = or_undefined(residual);
    if (wants_grad({x, r, weight})) {
        const tensor_list out = NormFunction::apply(x, residual, weight, eps);
        return {out[0], out[1]};
    }
    auto [y, h, rstd] = rms_norm_residual(x, residual, weight, eps, false);
    return {y, h};
}

struct AttentionFunction : torch::autograd::Function<AttentionFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                          const OptTensor& lengths, const OptTensor& mask, double scale) {
        auto [o, lse, o_low] = cross_attention(q, k, v, lengths, mask, scale, true);
        ctx->save_for_backward({q, k, v, o, lse, o_low, or_undefined(lengths), or_undefined(mask)});
        ctx->saved_data["scale"] = scale;
        return o;
    }
    static tensor_list backward(AutogradContext* ctx, const tensor_list& grads) {
        const tensor_list s = ctx->get_saved_variables();
        const bool want_q = ctx->needs_input_grad(0);
        const bool want_k = ctx->needs_input_grad(1), want_v = ctx->needs_input_grad(2);
        tensor_list out(6);
        {
            at::AutoGradMode off(false);
            auto [dq, dk, dv] = cross_attention_backward(
                grads[0], s[0], s[1], s[2], s[3], s[4], s[5], opt(s[6]), opt(s[7]),
                ctx->saved_data["scale"].toDouble(), want_q, want_k || want_v);
            if (want_q) out[0] = dq;
            if (want_k) out[1] = dk;
            if (want_v) out[2] = dv;
        }
        const bool of_p = any_requires_grad({grads[0], s[0], s[1]});
        for (int i = 0; i < 2; ++i)
            out[i] = once(out[i], of_p || s[2].requires_grad(), "cross_attention");
        out[2] = once(out[2], of_p, "cross_attention");
        return out;
    }
};

Tensor decoder_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                         const OptTensor& lengths, const OptTensor& mask, double scale) {
    if (wants_grad({q, k, v}))
        return AttentionFunction::apply(q, k, v, lengths, mask, scale);
    return std::get<0>(cross_attention(q, k, v, lengths, mask, scale, false));
}

}  // namespace

void bind_decoder(pybind11::module& m) {
    m.def("rotary_axes", &rotary_axes, "decoder: rotary positions with several axes");
    m.def("rms_norm_residual", &rms_norm_residual,
          "decoder: (y, h, rstd) of the root-mean-square norm of x + residual");
    m.def("rms_norm_residual_fp8", &rms_norm_residual_fp8,
          "decoder: (y, scale, h), y in 8-bit floats with a scale per row");
    m.def("rms_norm_residual_backward", &rms_norm_residual_backward, "decoder: (dx, dweight)");
    m.def("cross_attention", &cross_attention, "decoder: (o, lse, o_low) of cross attention");
    m.def("cross_attention_backward", &cross_attention_backward, "decoder: (dq, dk, dv)");
    m.def("decoder_rotary", &decoder_rotary, "decoder: rotary_axes, differentiable in x");
    m.def("decoder_norm", &decoder_norm,
          "decoder: (y, h) of rms_norm_residual, differentiable in x, residual and weight");
    m.def("decoder_attention", &decoder_attention,
          "decoder: cross_attention, differentiable in q, k and v");
}
