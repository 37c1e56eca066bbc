// Torch front end of the low-precision operators: checks of arguments, outputs and workspaces from torch's caching
// allocator, autograd nodes, and the calls of libgnnagg's C ABI (include/gnnagg.h) on the tensors' current stream.
//
// These operators run in few microseconds at small sizes, where the same steps in Python cost five to ten times the
// kernel (a node's backward in Python 60 us next to 40 us for the engine's own hand-over).
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <optional>
#include <unordered_set>
#include <vector>

#include "gnnagg.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxRmsWidth = 16384;

void check(int rc, const char *what) {
    TORCH_CHECK(rc == GNNAGG_OK, "libgnnagg ", what, " failed (status ", rc, "): ", gnnagg_error_string(rc));
}

// Element type of the C ABI, -1 for another.
int type_of(at::ScalarType t) {
    return t == at::kFloat ? GNNAGG_F32 : t == at::kBFloat16 ? GNNAGG_BF16 : t == at::kHalf ? GNNAGG_F16 : -1;
}
int type_of(const Tensor &t) { return type_of(t.scalar_type()); }

void require_cuda(const Tensor &t) {
    TORCH_CHECK(t.is_cuda(), "libgnnagg kernels take CUDA tensors only (this package has no CPU fallback)");
}

void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor &like) {
    return at::empty(sizes, like.options().dtype(type).memory_format(std::nullopt));
}
Tensor bytes(size_t n, const Tensor &like) { return empty({(int64_t)n}, at::kByte, like); }

// `t` itself when its rows are contiguous and do not overlap, else a copy; and its row stride, for which torch may keep
// anything when there is a single row or column.
Tensor rows_of(const Tensor &t) {
    return t.stride(1) == 1 && t.stride(0) >= t.size(1) ? t : t.contiguous();
}
int64_t ld(const Tensor &t) { return std::max(t.stride(0), t.size(1)); }

// Uninitialised e4m3 codes whose rows start on 16 bytes, and scales, one per row and 128 columns, that lie column by
// column, each column on 16 bytes.
Tensor empty_codes(int64_t rows, int64_t cols, const Tensor &like) {
    const int64_t wide = (cols + 15) / 16 * 16;
    Tensor t = empty({rows, wide}, at::kFloat8_e4m3fn, like);
    return wide == cols ? t : t.narrow(1, 0, cols);
}
Tensor empty_scales(int64_t rows, int64_t cols, const Tensor &like) {
    return at::empty_strided({rows, (cols + 127) / 128}, {1, (rows + 3) / 4 * 4}, like.options().dtype(at::kFloat));
}

bool wants_grad(const Tensor &t) { return t.requires_grad(); }
bool wants_grad(const std::optional<Tensor> &t) { return t.has_value() && t->requires_grad(); }

// The results would be without the tangents that torch.autograd.forward_ad gave the inputs.
bool has_tangent(const Tensor &t) { return t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const std::optional<Tensor> &t) { return t.has_value() && has_tangent(*t); }
template <typename... Ts>
void check_tangents(const char *what, const Ts &...ts) {
    TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !(has_tangent(ts) || ...), what,
                " has no forward-mode derivative: take the tangents off its inputs (torch.autograd.forward_ad.unpack_dual)");
}

// A captured backward may not reach the default stream: a forward's node goes on where the forward ran, and the gradients
// of a leaf are added up there when a graph that was made there still holds that leaf.  The process would end inside the
// capture, so the node refuses before.
void check_capture(const char *what, const Tensor &t) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(static_cast<cudaStream_t>(stream_of(t)), &status) != cudaSuccess ||
        status == cudaStreamCaptureStatusNone)
        return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    const c10::Stream other = c10::cuda::getDefaultCUDAStream(t.get_device()).unwrap();
    // all nodes that this pass goes on to: those behind a view of the leaf, and only those whose gradient it computes
    std::vector<torch::autograd::Node *> todo{node.get()};
    std::unordered_set<torch::autograd::Node *> seen;
    while (!todo.empty()) {
        torch::autograd::Node *at = todo.back();
        todo.pop_back();
        for (uint32_t i = 0; i < at->num_outputs(); ++i) {
            torch::autograd::Node *next = at->next_edge(i).function.get();
            if (next == nullptr || !at->task_should_compute_output(i) || !seen.insert(next).second) continue;
            const auto stream = next->stream();
            const bool leaf = next->num_outputs() == 0;  // a leaf's node leads nowhere
            TORCH_CHECK(!stream.has_value() || *stream != other || !leaf, what,
                        ": captured backward of a leaf that a graph made on the default stream still holds (delete what that "
                        "graph computed, its loss for example, before the capture, or compute it on a side stream)");
            TORCH_CHECK(!stream.has_value() || *stream != other, what, ": captured backward reaches ", next->name(),
                        ", whose forward ran on the default stream (capture that too, or run it on a side stream)");
            todo.push_back(next);
        }
    }
}

// What torch's own in-place operators leave behind: a graph that kept the old values then raises in its backward.
void written(const Tensor &t) {
    if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

// ------------------------------------------------------------------------------------------ root-mean-square norm

void check_rms(const char *what, const Tensor &x, const Tensor &w, const std::optional<Tensor> &res) {
    require_cuda(x);
    TORCH_CHECK(x.dim() == 2 && type_of(x) >= 0 && x.size(1) > 0 && x.size(1) <= kMaxRmsWidth, what,
                ": x must be (rows, F) float32, bfloat16 or float16 with 1 <= F <= ", kMaxRmsWidth, ", not ", x.sizes(), " ",
                x.scalar_type());
    TORCH_CHECK(w.dim() == 1 && w.size(0) == x.size(1) && (w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat) &&
                    w.device() == x.device(),
                what, ": weight must be a vector of ", x.size(1), " elements of x's type or float32 on x's device");
    TORCH_CHECK(!res.has_value() || (res->sizes() == x.sizes() && res->scalar_type() == x.scalar_type() &&
                                     res->device() == x.device()),
                what, ": residual must match x in shape, type and device");
}

struct Normed {
    Tensor y, h, rstd, w;
};

Normed rms_forward(const Tensor &x_, const Tensor &w_, const std::optional<Tensor> &res_, double eps, bool need_rstd) {
    const Tensor x = rows_of(x_), w = w_.contiguous();
    const c10::cuda::CUDAGuard guard(x.device());
    Normed n;
    n.y = empty(x.sizes(), x.scalar_type(), x);
    n.h = x;
    n.w = w;
    if (need_rstd) n.rstd = empty({x.size(0)}, at::kFloat, x);
    Tensor res;
    if (res_.has_value()) {
        res = rows_of(*res_);
        n.h = empty(x.sizes(), x.scalar_type(), x);
    }
    const bool add = res.defined();
    check(gnnagg_rms_norm_fwd(x.data_ptr(), ld(x), add ? res.data_ptr() : nullptr, add ? ld(res) : 0, w.data_ptr(), type_of(w),
                              x.size(0), (int32_t)x.size(1), type_of(x), (float)eps, add ? n.h.data_ptr() : nullptr, x.size(1),
                              n.y.data_ptr(), x.size(1), need_rstd ? n.rstd.data_ptr<float>() : nullptr, stream_of(x)),
          "rms_norm_fwd");
    return n;
}

// (y, h) = norm of h = x + residual; without a residual h is x itself and only y is an output.
struct RMSNorm : torch::autograd::Function<RMSNorm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const std::optional<Tensor> &res,
                                 double eps) {
        Normed n = rms_forward(x, w, res, eps, true);
        ctx->save_for_backward({n.h, n.w, n.rstd});
        ctx->saved_data["residual"] = res.has_value();
        ctx->set_materialize_grads(false);
        return res.has_value() ? variable_list{n.y, n.h} : variable_list{n.y};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "rms_norm has no second derivative");
        for (const Tensor &g : grads)
            if (g.defined()) check_capture("rms_norm", g);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &h = saved[0], &w = saved[1], &rstd = saved[2];
        const bool residual = ctx->saved_data["residual"].toBool();
        Tensor gh = residual ? grads[1] : Tensor();
        if (!grads[0].defined())  // only the sum was used
            return {gh, Tensor(), residual ? gh : Tensor(), Tensor()};
        const c10::cuda::CUDAGuard guard(h.device());
        const Tensor gy = rows_of(grads[0]);
        if (gh.defined()) gh = rows_of(gh);
        const int64_t rows = h.size(0), f = h.size(1);
        Tensor gx = empty(h.sizes(), h.scalar_type(), h), dw = empty({f}, w.scalar_type(), h);
        const size_t need = gnnagg_rms_norm_partial_bytes(rows, (int32_t)f, type_of(h));
        const Tensor partial = bytes(need, h);
        check(gnnagg_rms_norm_bwd(gy.data_ptr(), ld(gy), gh.defined() ? gh.data_ptr() : nullptr, gh.defined() ? ld(gh) : 0,
                                  h.data_ptr(), ld(h), rstd.data_ptr<float>(), w.data_ptr(), type_of(w), rows, (int32_t)f,
                                  type_of(h), gx.data_ptr(), f, dw.data_ptr(), static_cast<float *>(partial.data_ptr()), need,
                                  stream_of(h)),
              "rms_norm_bwd");
        return {gx, dw, residual ? gx : Tensor(), Tensor()};
    }
};

std::vector<Tensor> rms_norm(const Tensor &x, const Tensor &w, const std::optional<Tensor> &res, double eps) {
    check_rms("rms_norm", x, w, res);
    check_tangents("rms_norm", x, w, res);
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(res))) return RMSNorm::apply(x, w, res, eps);
    Normed n = rms_forward(x, w, res, eps, false);
    return res.has_value() ? std::vector<Tensor>{n.y, n.h} : std::vector<Tensor>{n.y};
}

std::vector<Tensor> rms_norm_fp8(const Tensor &x_, const Tensor &w_, const std::optional<Tensor> &res_, double eps) {
    check_rms("rms_norm_fp8", x_, w_, res_);
    check_tangents("rms_norm_fp8", x_, w_, res_);
    TORCH_CHECK(!at::GradMode::is_enabled() || !(wants_grad(x_) || wants_grad(w_) || wants_grad(res_)),
                "rms_norm_fp8 has no gradient: call it under torch.no_grad(), or use rms_norm");
    const Tensor x = rows_of(x_), w = w_.contiguous();
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor codes = empty_codes(x.size(0), x.size(1), x), scales = empty_scales(x.size(0), x.size(1), x), res, h;
    if (res_.has_value()) {
        res = rows_of(*res_);
        h = empty(x.sizes(), x.scalar_type(), x);
    }
    const bool add = res.defined();
    check(gnnagg_rms_norm_fp8(x.data_ptr(), ld(x), add ? res.data_ptr() : nullptr, add ? ld(res) : 0, w.data_ptr(), type_of(w),
                              x.size(0), (int32_t)x.size(1), type_of(x), (float)eps, add ? h.data_ptr() : nullptr, x.size(1),
                              static_cast<uint8_t *>(codes.data_ptr()), codes.stride(0), scales.data_ptr<float>(),
                              scales.stride(1), stream_of(x)),
          "rms_norm_fp8");
    return add ? std::vector<Tensor>{codes, scales, h} : std::vector<Tensor>{codes, scales};
}

// ------------------------------------------------------------------------------------------ 8-bit products

// Codes and scales of x, of its transpose, or of both from one read (in that order).
std::vector<Tensor> quantize_fp8(const Tensor &x_, int64_t block_rows, bool rows, bool cols) {
    TORCH_CHECK(x_.dim() == 2 && type_of(x_) >= 0, "quantize_fp8: x must be a float32, bfloat16 or float16 matrix, not ",
                x_.sizes(), " ", x_.scalar_type());
    require_cuda(x_);
    const Tensor x = rows_of(x_);
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t m = x.size(0), k = x.size(1);
    const bool block = block_rows == 128;
    Tensor c, s, ct, st;
    std::vector<Tensor> out;
    if (rows) {
        c = empty_codes(m, k, x);
        s = empty_scales(block ? (m + 127) / 128 : m, k, x);
        out = {c, s};
    }
    if (cols) {
        ct = empty_codes(k, m, x);
        st = empty_scales(block ? (k + 127) / 128 : k, m, x);
        out.push_back(ct);
        out.push_back(st);
    }
    check(gnnagg_fp8_quantize(x.data_ptr(), ld(x), m, k, type_of(x), (int32_t)block_rows,
                              rows ? static_cast<uint8_t *>(c.data_ptr()) : nullptr, rows ? c.stride(0) : 0,
                              rows ? s.data_ptr<float>() : nullptr, rows ? s.stride(1) : 0,
                              cols ? static_cast<uint8_t *>(ct.data_ptr()) : nullptr, cols ? ct.stride(0) : 0,
                              cols ? st.data_ptr<float>() : nullptr, cols ? st.stride(1) : 0, nullptr, stream_of(x)),
          "fp8_quantize");
    return out;
}

struct Operand {
    int32_t block;  // rows that a scale covers
    int64_t ld;
};
Operand operand(const char *name, const Tensor &codes, const Tensor &scales, const Tensor &like) {
    TORCH_CHECK(codes.dim() == 2 && codes.scalar_type() == at::kFloat8_e4m3fn && codes.device() == like.device(), "matmul_fp8: ",
                name, " must be a float8_e4m3fn matrix on the operands' device");
    const int64_t rows = codes.size(0), k = codes.size(1), high = (rows + 127) / 128, kb = (k + 127) / 128;
    int64_t ld = codes.stride(0);
    if (rows <= 1 || k == 0) ld = kb * 128;  // torch may keep any stride
    TORCH_CHECK(rows == 0 || k == 0 ||
                    ((codes.stride(1) == 1 || k == 1) && ld >= k && ld % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0),
                "matmul_fp8: ", name, "'s rows must be contiguous and start on 16 bytes (as quantize_fp8 lays them)");
    TORCH_CHECK(scales.dim() == 2 && scales.scalar_type() == at::kFloat && scales.device() == like.device() &&
                    (scales.size(0) == rows || scales.size(0) == high) && scales.size(1) == kb,
                "matmul_fp8: ", name, "'s scales must be float32 (", rows, " or ", high, ", ", kb, ") on the operands' device, not ",
                scales.sizes(), " ", scales.scalar_type());
    return {scales.size(0) == rows ? 1 : 128, ld};
}

Tensor matmul_fp8(const Tensor &a, const Tensor &sa, const Tensor &b, const Tensor &sb, const std::optional<Tensor> &bias,
                  const std::optional<Tensor> &out_, at::ScalarType out_type, bool accumulate) {
    require_cuda(a);
    const Operand oa = operand("a", a, sa, a), ob = operand("b", b, sb, a);
    const int64_t m = a.size(0), k = a.size(1), n = b.size(0);
    TORCH_CHECK(b.size(1) == k, "matmul_fp8: shape mismatch a=", a.sizes(), " b=", b.sizes());
    TORCH_CHECK(!at::GradMode::is_enabled() || !(wants_grad(a) || wants_grad(sa) || wants_grad(b) || wants_grad(sb) ||
                                                 wants_grad(bias) || wants_grad(out_)),
                "matmul_fp8 has no gradient: call it under torch.no_grad(), or use linear_fp8");
    check_tangents("matmul_fp8", a, sa, b, sb, bias, out_);
    TORCH_CHECK(!bias.has_value() || (type_of(*bias) >= 0 && bias->dim() == 1 && bias->size(0) == n && bias->is_contiguous() &&
                                      bias->device() == a.device()),
                "matmul_fp8: bias must be a contiguous float32, bfloat16 or float16 vector of N elements on the operands' device");
    const c10::cuda::CUDAGuard guard(a.device());
    Tensor out;
    int64_t ldc = n;
    if (out_.has_value()) {
        out = *out_;
        if (out.dim() == 2 && m > 1) ldc = out.stride(0);
        TORCH_CHECK(out.dim() == 2 && out.size(0) == m && out.size(1) == n && type_of(out) >= 0 && out.device() == a.device() &&
                        (out.numel() == 0 || ((out.stride(1) == 1 || n == 1) && ldc >= n)),
                    "matmul_fp8: out must be (M, N) float32, bfloat16 or float16 with contiguous rows on the operands' device");
    } else {
        TORCH_CHECK(!accumulate, "matmul_fp8: accumulate needs an output to accumulate into");
        TORCH_CHECK(type_of(out_type) >= 0, "matmul_fp8: out_dtype must be float32, bfloat16 or float16");
        out = empty({m, n}, out_type, a);
    }
    TORCH_CHECK(!accumulate || out.scalar_type() == at::kFloat, "matmul_fp8: accumulate needs a float32 output");
    // from the caching allocator at every call: ordered with the stream, and a captured graph has its own
    const size_t need = gnnagg_fp8_matmul_workspace_bytes(m, n, k);
    const Tensor ws = need > 0 ? bytes(need, a) : Tensor();
    check(gnnagg_fp8_matmul(static_cast<const uint8_t *>(a.data_ptr()), oa.ld, sa.data_ptr<float>(), sa.stride(0), sa.stride(1),
                            oa.block, static_cast<const uint8_t *>(b.data_ptr()), ob.ld, sb.data_ptr<float>(), sb.stride(0),
                            sb.stride(1), ob.block, m, n, k, bias.has_value() ? bias->data_ptr() : nullptr,
                            bias.has_value() ? type_of(*bias) : 0, accumulate ? 1 : 0, out.data_ptr(), ldc, type_of(out),
                            need > 0 ? ws.data_ptr() : nullptr, need, stream_of(a)),
          "fp8_matmul");
    if (out_.has_value()) written(out);
    return out;
}

// y = x W^T (+ b) with e4m3 operands in all three products.  x and the output's gradient are rounded in blocks of 1 x 128
// along the sum they enter (columns for y and the input gradient, rows for the weight gradient), the weight in blocks of
// 128 x 128.  What is kept for the backward is 8-bit: x's transposed codes and the weight's.
struct LinearFP8 : torch::autograd::Function<LinearFP8> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x_, const Tensor &w_, const std::optional<Tensor> &bias_,
                          bool need_x, bool need_w) {
        const Tensor x = rows_of(x_), w = rows_of(w_);
        const Tensor bias = bias_.has_value() ? bias_->contiguous() : Tensor();
        const c10::cuda::CUDAGuard guard(x.device());
        const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
        const size_t kept_bytes = gnnagg_fp8_linear_kept_bytes(m, n, k, need_x, need_w);
        const size_t scratch_bytes = gnnagg_fp8_linear_scratch_bytes(m, n, k, 0);
        const Tensor kept = bytes(kept_bytes, x), scratch = bytes(scratch_bytes, x);
        Tensor y = empty({m, n}, x.scalar_type(), x);
        check(gnnagg_fp8_linear_fwd(x.data_ptr(), ld(x), type_of(x), w.data_ptr(), ld(w), type_of(w),
                                    bias.defined() ? bias.data_ptr() : nullptr, bias.defined() ? type_of(bias) : 0, m, n, k,
                                    y.data_ptr(), type_of(x), need_x, need_w, kept.data_ptr(), kept_bytes, scratch.data_ptr(),
                                    scratch_bytes, stream_of(x)),
              "fp8_linear_fwd");
        ctx->save_for_backward({kept});
        ctx->saved_data["k"] = k;
        ctx->saved_data["need_x"] = need_x;
        ctx->saved_data["need_w"] = need_w;
        ctx->saved_data["w_type"] = (int64_t)w.scalar_type();
        ctx->saved_data["has_bias"] = bias.defined();
        ctx->saved_data["b_type"] = (int64_t)(bias.defined() ? bias.scalar_type() : at::kFloat);
        return y;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "linear_fp8 has no second derivative");
        check_capture("linear_fp8", grads[0]);
        const Tensor kept = ctx->get_saved_variables()[0], g = rows_of(grads[0]);
        const c10::cuda::CUDAGuard guard(g.device());
        const int64_t m = g.size(0), n = g.size(1), k = ctx->saved_data["k"].toInt();
        const bool need_x = ctx->saved_data["need_x"].toBool(), need_w = ctx->saved_data["need_w"].toBool();
        const auto w_type = (at::ScalarType)ctx->saved_data["w_type"].toInt();
        const auto b_type = (at::ScalarType)ctx->saved_data["b_type"].toInt();
        Tensor gx, gw, gb;
        if (need_x && ctx->needs_input_grad(0)) gx = empty({m, k}, g.scalar_type(), g);
        if (need_w && ctx->needs_input_grad(1)) gw = empty({n, k}, w_type, g);
        if (ctx->saved_data["has_bias"].toBool() && ctx->needs_input_grad(2)) gb = empty({n}, b_type, g);
        const size_t scratch_bytes = gnnagg_fp8_linear_scratch_bytes(m, n, k, 1);
        const Tensor scratch = bytes(scratch_bytes, g);
        check(gnnagg_fp8_linear_bwd(g.data_ptr(), ld(g), type_of(g), m, n, k, need_x, need_w, kept.data_ptr(), kept.numel(),
                                    gx.defined() ? gx.data_ptr() : nullptr, type_of(g), gw.defined() ? gw.data_ptr() : nullptr,
                                    type_of(w_type), gb.defined() ? gb.data_ptr() : nullptr, type_of(b_type), scratch.data_ptr(),
                                    scratch_bytes, stream_of(g)),
              "fp8_linear_bwd");
        return {gx, gw, gb, Tensor(), Tensor()};
    }
};

Tensor linear_fp8(const Tensor &x, const Tensor &w, const std::optional<Tensor> &bias) {
    require_cuda(x);
    TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1), "linear_fp8: shape mismatch x=", x.sizes(), " weight=",
                w.sizes());
    TORCH_CHECK(type_of(x) >= 0 && type_of(w) >= 0 && w.device() == x.device(),
                "linear_fp8: x and weight must be float32, bfloat16 or float16 on one device");
    TORCH_CHECK(!bias.has_value() || (bias->dim() == 1 && bias->size(0) == w.size(0) && type_of(*bias) >= 0 &&
                                      bias->device() == x.device()),
                "linear_fp8: bias must be a float32, bfloat16 or float16 vector of N elements on x's device");
    check_tangents("linear_fp8", x, w, bias);
    const bool grad = at::GradMode::is_enabled();
    return LinearFP8::apply(x, w, bias, grad && wants_grad(x), grad && wants_grad(w));
}

// ------------------------------------------------------------------------------------------ AdamW

void check_list(const char *what, const std::vector<Tensor> &ts, const std::vector<Tensor> &params, at::ScalarType type,
                int64_t per_block, int64_t each) {
    for (size_t i = 0; i < ts.size(); ++i) {
        const Tensor &t = ts[i];
        const int64_t n = (params[i].numel() + per_block - 1) / per_block * each;
        TORCH_CHECK(t.numel() == n && t.scalar_type() == type && t.device() == params[0].device() && t.is_contiguous(),
                    "adamw_step: ", what, " ", i, " must be a contiguous ", type, " tensor of ", n,
                    " elements on the parameters' device, not ", t.sizes(), " ", t.scalar_type(), " on ", t.device());
    }
}

void adamw_step(const std::vector<Tensor> &params, const std::vector<Tensor> &grads, const std::vector<Tensor> &exp_avgs,
                const std::vector<Tensor> &exp_avg_sqs, const std::optional<std::vector<Tensor>> &scales,
                const std::optional<std::vector<std::optional<Tensor>>> &masters, const std::optional<Tensor> &device_scalars,
                int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay) {
    const size_t count = params.size();
    TORCH_CHECK(grads.size() == count && exp_avgs.size() == count && exp_avg_sqs.size() == count &&
                    (!scales.has_value() || scales->size() == count) && (!masters.has_value() || masters->size() == count),
                "adamw_step: the lists must have one entry per parameter");
    TORCH_CHECK(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adamw_step: betas must be in [0, 1), not (", beta1,
                ", ", beta2, ")");
    TORCH_CHECK(device_scalars.has_value() || step >= 1, "adamw_step: the first step is 1");
    if (count == 0) return;
    require_cuda(params[0]);
    TORCH_CHECK(!device_scalars.has_value() ||
                    (device_scalars->scalar_type() == at::kByte && device_scalars->is_contiguous() &&
                     (size_t)device_scalars->numel() == gnnagg_adamw_scalars_bytes() &&
                     reinterpret_cast<uintptr_t>(device_scalars->data_ptr()) % 4 == 0 &&
                     device_scalars->device() == params[0].device()),
                "adamw_step: device_scalars must be the ", gnnagg_adamw_scalars_bytes(),
                " bytes that AdamW keeps, on the parameters' device");
    const at::ScalarType type = params[0].scalar_type(), state = scales.has_value() ? at::kFloat8_e4m3fn : at::kFloat;
    TORCH_CHECK(type_of(type) >= 0, "adamw_step: parameters must be float32, bfloat16 or float16, not ", type);
    check_list("parameter", params, params, type, 1, 1);
    check_list("gradient", grads, params, type, 1, 1);
    for (size_t i = 0; i < count; ++i)
        TORCH_CHECK(grads[i].sizes() == params[i].sizes(), "adamw_step: gradient ", i, " has the shape ", grads[i].sizes(),
                    ", its parameter ", params[i].sizes());
    check_list("exp_avg", exp_avgs, params, state, 1, 1);
    check_list("exp_avg_sq", exp_avg_sqs, params, state, 1, 1);
    if (scales.has_value()) check_list("scales", *scales, params, at::kFloat, 256, 2);
    std::vector<gnnagg_adamw_tensor> table(count);
    for (size_t i = 0; i < count; ++i) {
        gnnagg_adamw_tensor &t = table[i];
        t.param = params[i].data_ptr();
        t.grad = grads[i].data_ptr();
        t.exp_avg = exp_avgs[i].data_ptr();
        t.exp_avg_sq = exp_avg_sqs[i].data_ptr();
        t.scales = scales.has_value() ? (*scales)[i].data_ptr<float>() : nullptr;
        t.master = nullptr;
        t.n = params[i].numel();
        if (masters.has_value() && (*masters)[i].has_value()) {
            const Tensor &m = *(*masters)[i];
            TORCH_CHECK(m.numel() == t.n && m.scalar_type() == at::kFloat && m.device() == params[0].device() && m.is_contiguous(),
                        "adamw_step: master ", i, " must be a contiguous float32 tensor of ", t.n,
                        " elements on the parameters' device");
            t.master = m.data_ptr<float>();
        }
    }
    const c10::cuda::CUDAGuard guard(params[0].device());
    check(gnnagg_adamw_step(table.data(), (int64_t)count, type_of(type), scales.has_value() ? 8 : 32, lr, beta1, beta2, eps,
                            weight_decay, step, device_scalars.has_value() ? device_scalars->data_ptr() : nullptr,
                            stream_of(params[0])),
          "adamw_step");
    for (size_t i = 0; i < count; ++i) {
        written(params[i]);
        written(exp_avgs[i]);
        written(exp_avg_sqs[i]);
        if (scales.has_value()) written((*scales)[i]);
        if (masters.has_value() && (*masters)[i].has_value()) written(*(*masters)[i]);
    }
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_fp8", &rms_norm_fp8);
    m.def("quantize_fp8", &quantize_fp8);
    m.def("matmul_fp8", &matmul_fp8);
    m.def("linear_fp8", &linear_fp8);
    m.def("adamw_step", &adamw_step);
}
