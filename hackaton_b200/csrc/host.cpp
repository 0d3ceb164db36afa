// The host side of the calls that training and decoding make most: views, output tensors, device
// and stream look-ups and the call into the C ABI, in one step out of Python. The same work through
// ctypes costs several times the kernels of a small call (q/k/v with LoRA at 810 tokens: 16 launches
// of 86 us GPU time in all took 668 us from Python). Argument checks that need the quant state, and most
// autograd functions, stay in Python; nothing is kept here between calls. The newer operators have their autograd
// functions here too: a node of Python costs a backward pass about 40 us of interpreter and thread hand-over (a SwiGLU of
// 333 x 1000 both ways took 96 us that way). What one of those calls refuses comes back as None, and Python says why.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <initializer_list>
#include <optional>
#include <utility>
#include <vector>

#include "../../include/nf4b200.h"

namespace py = pybind11;
using at::Tensor;
using Opt = std::optional<Tensor>;
using Opts = std::vector<Opt>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

constexpr int64_t RANK = 16;
constexpr int MAX_GROUP = 4, MAX_BATCH = 8;

// A non-zero status becomes the package's own exception. (The calls run without the interpreter lock.)
void check(int rc) {
    if (rc == 0) return;
    const py::gil_scoped_acquire lock;
    py::module_::import("hackaton_b200._lib").attr("check")(rc);
}

void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

const void* ptr(const Opt& t) { return t.has_value() ? t->const_data_ptr() : nullptr; }

const nf4b200_weight* weight(int64_t address) { return reinterpret_cast<const nf4b200_weight*>(address); }

// Where the tensors of a weight lie and how often each has been written (inference tensors do not count
// that), in a form that compares as a whole.
py::bytes stamps(const Tensor& packed, const Tensor& absmax, const Tensor& code, const Opt& absmax2, const Opt& code2,
                 const Opt& offset) {
    const Tensor none;
    const Tensor* all[] = {&packed, &absmax, &code, absmax2 ? &*absmax2 : &none, code2 ? &*code2 : &none,
                           offset ? &*offset : &none};
    int64_t r[12];
    int n = 0;
    for (const Tensor* t : all) {
        r[n++] = t->defined() ? reinterpret_cast<int64_t>(t->const_data_ptr()) : 0;
        r[n++] = t->defined() && !t->is_inference() ? t->_version() : -1;
    }
    return py::bytes(reinterpret_cast<const char*>(r), sizeof r);
}

// [..., cols] -> 2-D view with contiguous rows, 16-byte aligned and 8 elements apart (copied only if the
// layout forces it; columns that are no eights stay where they are).
Tensor rows_view(const Tensor& t, int64_t cols) {
    const auto aligned = [](const Tensor& v) { return (reinterpret_cast<uintptr_t>(v.const_data_ptr()) & 15) == 0; };
    Tensor v = t.dim() == 2 && t.size(1) == cols ? t : t.reshape({-1, cols});
    if (v.stride(1) == 1 && v.stride(0) % 8 == 0 && aligned(v) && v.stride(0) >= cols) return v;
    v = v.contiguous();
    // (a tensor that counts as contiguous keeps its address, and a single row its stride)
    if (cols % 8 == 0 && (!aligned(v) || v.stride(0) != cols)) v = v.clone(at::MemoryFormat::Contiguous);
    return v;
}

// Output with the leading dimensions of `like` and `cols` columns.
Tensor output(const Tensor& like, int64_t cols, at::ScalarType type = at::kHalf) {
    at::DimVector shape(like.sizes().begin(), like.sizes().end());
    shape.back() = cols;
    return at::empty(shape, like.options().dtype(type).memory_format(c10::nullopt));
}

// Scratch of one call on the current stream (see hackaton_b200.nf4.scratch_bytes): the allocator hands it
// out again only behind the work of that stream.
struct Scratch {
    Tensor buffer;
    Scratch(int64_t bytes, const Tensor& like) {
        if (bytes > 0) buffer = at::empty({bytes}, like.options().dtype(at::kByte).memory_format(c10::nullopt));
    }
    void* get() const { return buffer.defined() ? buffer.data_ptr() : nullptr; }
};

// What a kernel reads besides its input has to be there: a rank-16 pair of `rows` and `cols`, a bias.
void check_pair(const Opt& a, int64_t rows, const Opt& b, int64_t cols) {
    TORCH_CHECK(a.has_value() == b.has_value() &&
                    (!a.has_value() || (a->numel() >= rows * RANK && b->numel() >= cols * RANK)),
                "rank-16 pair does not reach over ", rows, " rows and ", cols, " columns");
}

void check_bias(const Opt& bias, int64_t cols) {
    TORCH_CHECK(!bias.has_value() || bias->numel() >= cols, "bias of ", bias->numel(), " values for ", cols, " outputs");
}

Opt half(const Opt& t) {
    if (!t.has_value()) return t;
    return t->to(at::kHalf).contiguous();
}

Tensor linear_fwd(int64_t w, const Tensor& x, const Opt& bias, const Opt& xa, const Opt& lora_b, int64_t ws_bytes) {
    const nf4b200_weight* q = weight(w);
    if (x.numel() == 0) return output(x, q->n_rows);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor x2 = rows_view(x, q->n_cols);
    check_pair(xa, x2.size(0), lora_b, q->n_rows);
    check_bias(bias, q->n_rows);
    Tensor y = output(x, q->n_rows);
    const Opt b = half(bias);
    const Scratch ws(ws_bytes, x);
    check(nf4b200_linear_fwd(q, x2.const_data_ptr(), x2.size(0), x2.stride(0), ptr(b), ptr(xa), ptr(lora_b),
                             y.data_ptr(), q->n_rows, ws.get(), (size_t)ws_bytes, stream_of(x)));
    return y;
}

Tensor linear_bwd_dx(int64_t w, const Tensor& dy, const Opt& u, const Opt& lora_a, int64_t ws_bytes) {
    const nf4b200_weight* q = weight(w);
    if (dy.numel() == 0) return output(dy, q->n_cols);
    const c10::cuda::CUDAGuard guard(dy.device());
    const Tensor g2 = rows_view(dy, q->n_rows);
    check_pair(u, g2.size(0), lora_a, q->n_cols);
    Tensor dx = output(dy, q->n_cols);
    const Scratch ws(ws_bytes, dy);
    check(nf4b200_linear_bwd_dx(q, g2.const_data_ptr(), g2.size(0), g2.stride(0), ptr(u), ptr(lora_a), dx.data_ptr(),
                                q->n_cols, ws.get(), (size_t)ws_bytes, stream_of(dy)));
    return dx;
}

std::vector<Tensor> linear_fwd_group(const std::vector<int64_t>& ws_addr, const Tensor& x, const Opts& biases,
                                     const Opts& xas, const Opts& lora_bs, int64_t ws_bytes) {
    const int n = (int)ws_addr.size();
    TORCH_CHECK(n >= 1 && n <= MAX_GROUP, "a group holds 1..", MAX_GROUP, " projections, got ", n);
    std::vector<Tensor> ys;
    for (const int64_t address : ws_addr) ys.push_back(output(x, weight(address)->n_rows));
    if (x.numel() == 0) return ys;
    const c10::cuda::CUDAGuard guard(x.device());
    const nf4b200_weight* q[MAX_GROUP];
    const void *b[MAX_GROUP], *a[MAX_GROUP], *l[MAX_GROUP];
    void* y[MAX_GROUP];
    int64_t ld[MAX_GROUP];
    Opts keep;
    const Tensor x2 = rows_view(x, weight(ws_addr[0])->n_cols);
    for (int i = 0; i < n; ++i) {
        q[i] = weight(ws_addr[i]);
        check_pair(xas[i], x2.size(0), lora_bs[i], q[i]->n_rows);
        check_bias(biases[i], q[i]->n_rows);
        keep.push_back(half(biases[i]));
        b[i] = ptr(keep.back());
        a[i] = ptr(xas[i]);
        l[i] = ptr(lora_bs[i]);
        y[i] = ys[i].data_ptr();
        ld[i] = q[i]->n_rows;
    }
    const Scratch ws(ws_bytes, x);
    check(nf4b200_linear_fwd_group(n, q, x2.const_data_ptr(), x2.size(0), x2.stride(0), b, a, l, y, ld,
                                   ws.get(), (size_t)ws_bytes, stream_of(x)));
    return ys;
}

Tensor linear_bwd_dx_group(const std::vector<int64_t>& ws_addr, const std::vector<Tensor>& grads, const Opts& us,
                           const Opts& lora_as, int64_t ws_bytes) {
    const int n = (int)ws_addr.size();
    TORCH_CHECK(n >= 1 && n <= MAX_GROUP && (int)grads.size() == n, "a group holds 1..", MAX_GROUP, " projections");
    if (grads[0].numel() == 0) return output(grads[0], weight(ws_addr[0])->n_cols);
    const c10::cuda::CUDAGuard guard(grads[0].device());
    const nf4b200_weight* q[MAX_GROUP];
    const void *g[MAX_GROUP], *u[MAX_GROUP], *a[MAX_GROUP];
    int64_t ld[MAX_GROUP];
    std::vector<Tensor> keep;
    for (int i = 0; i < n; ++i) {
        q[i] = weight(ws_addr[i]);
        keep.push_back(rows_view(grads[i], q[i]->n_rows));
        g[i] = keep.back().const_data_ptr();
        ld[i] = keep.back().stride(0);
        TORCH_CHECK(keep.back().size(0) == keep[0].size(0), "gradients differ in their number of rows");
        check_pair(us[i], keep[0].size(0), lora_as[i], q[i]->n_cols);
        u[i] = ptr(us[i]);
        a[i] = ptr(lora_as[i]);
    }
    const int64_t m = keep[0].size(0), cols = q[0]->n_cols;
    Tensor dx = output(grads[0], cols);
    const Scratch ws(ws_bytes, dx);
    check(nf4b200_linear_bwd_dx_group(n, q, g, m, ld, u, a, dx.data_ptr(), cols, ws.get(), (size_t)ws_bytes, stream_of(dx)));
    return dx;
}

// A LoRA factor as the side kernel reads it: contiguous, 16-byte aligned fp32 or fp16.
Tensor factor(const Tensor& t) {
    Tensor p = t.detach();
    if (p.scalar_type() != at::kFloat && p.scalar_type() != at::kHalf) p = p.to(at::kHalf);
    p = p.contiguous();
    return (reinterpret_cast<uintptr_t>(p.const_data_ptr()) & 15) == 0 ? p : p.clone();
}

// (products, p16s, b16s, b16ts): see hackaton_b200.lora.lora_side.
std::tuple<std::vector<Tensor>, std::vector<Tensor>, std::vector<Tensor>, Opts>
lora_side(const std::vector<Tensor>& inputs, const std::vector<Tensor>& ps, const std::vector<double>& scalings,
          const std::vector<Tensor>& bs, bool transpose, const Opt& zero) {
    const int n = (int)inputs.size();
    TORCH_CHECK(n >= 1 && n <= MAX_BATCH && (int)ps.size() == n && (int)scalings.size() == n &&
                (bs.empty() || (int)bs.size() == n), "lora_side: 1..", MAX_BATCH, " adapters, one factor each");
    const c10::cuda::CUDAGuard guard(inputs[0].device());
    const auto options = inputs[0].options().dtype(at::kHalf);
    nf4b200_lora_item items[MAX_BATCH] = {};
    std::vector<Tensor> keep, products, p16s, b16s;
    Opts b16ts;
    int64_t m = -1;
    bool whole = true;   // every input in whole 16-byte pieces, as the side kernel reads it
    for (int i = 0; i < n; ++i) {
        const int64_t c = inputs[i].size(-1);
        const Tensor i2 = rows_view(inputs[i], c), p = factor(ps[i]);
        TORCH_CHECK(p.dim() == 2 && p.size(0) == RANK && p.size(1) == c, "lora_side: factor ", p.sizes(), " for ", c,
                    " columns");
        if (m < 0) m = i2.size(0);
        TORCH_CHECK(i2.size(0) == m, "lora_side: inputs differ in their number of rows");
        nf4b200_lora_item& it = items[i];
        it.in = i2.const_data_ptr(); it.c = c; it.ld_in = i2.stride(0);
        whole = whole && c % 8 == 0 && it.ld_in % 8 == 0 && (reinterpret_cast<uintptr_t>(it.in) & 15) == 0;
        it.p = p.const_data_ptr(); it.p_f32 = p.scalar_type() == at::kFloat;
        it.scaling = (float)scalings[i];
        products.push_back(at::empty({m, RANK}, options));
        it.out = products.back().data_ptr();
        p16s.push_back(it.p_f32 ? at::empty({RANK, c}, options) : p);
        it.p16 = it.p_f32 ? p16s.back().data_ptr() : nullptr;
        keep.push_back(i2);
        keep.push_back(p);
        if (bs.empty()) continue;
        const Tensor b = factor(bs[i]);
        TORCH_CHECK(b.dim() == 2 && b.size(1) == RANK, "lora_side: second factor ", b.sizes());
        const int64_t rows = b.size(0);
        it.b = b.const_data_ptr(); it.n = rows; it.b_f32 = b.scalar_type() == at::kFloat;
        b16s.push_back(it.b_f32 ? at::empty({rows, RANK}, options) : b);
        it.b16 = it.b_f32 ? b16s.back().data_ptr() : nullptr;
        b16ts.push_back(transpose ? Opt(at::empty({RANK, rows}, options)) : Opt());
        it.b16t = transpose ? b16ts.back()->data_ptr() : nullptr;
        keep.push_back(b);
    }
    if (m == 0 || !whole) {   // nothing to multiply, or columns that are not eights: copies and zeros by torch
        for (int i = 0; i < n; ++i) {
            if (items[i].p_f32) p16s[i].copy_(ps[i].detach());
            if (m > 0)
                check(nf4b200_lora_down(items[i].in, m, items[i].c, items[i].ld_in, p16s[i].const_data_ptr(),
                                        items[i].c, 1, items[i].scaling, items[i].out, stream_of(inputs[0])));
            if (bs.empty()) continue;
            if (items[i].b_f32) b16s[i].copy_(bs[i].detach());
            if (transpose) b16ts[i]->copy_(bs[i].detach().t());
        }
        if (zero.has_value()) zero->zero_();
    } else {
        check(nf4b200_lora_side(n, items, m, zero.has_value() ? zero->data_ptr() : nullptr,
                                zero.has_value() ? (size_t)zero->numel() * 4 : 0, stream_of(inputs[0])));
    }
    return {products, p16s, b16s, b16ts};
}

int64_t grad_piece(int64_t c) { return (c * RANK + 63) / 64 * 64; }   // 256-byte aligned pieces

// Adds the gradients zᵀ . s to pieces of the zeroed buffer `flat`, [16, C] or [C, 16] each.
std::vector<Tensor> lora_grad_batch(const std::vector<Tensor>& zs, const std::vector<Tensor>& ss,
                                    const std::vector<bool>& rank_major, const Tensor& flat) {
    const int n = (int)zs.size();
    TORCH_CHECK(n >= 1 && n <= MAX_BATCH && (int)ss.size() == n && (int)rank_major.size() == n,
                "lora_grad_batch: 1..", MAX_BATCH, " problems");
    const c10::cuda::CUDAGuard guard(zs[0].device());
    const void *z[MAX_BATCH], *s[MAX_BATCH];
    float* out[MAX_BATCH];
    int64_t m[MAX_BATCH], c[MAX_BATCH], ld[MAX_BATCH], sr[MAX_BATCH], sc[MAX_BATCH];
    std::vector<Tensor> keep, outs;
    int64_t at = 0;
    for (int i = 0; i < n; ++i) {
        c[i] = zs[i].size(-1);
        keep.push_back(rows_view(zs[i], c[i]));
        z[i] = keep.back().const_data_ptr();
        m[i] = keep.back().size(0);
        ld[i] = keep.back().stride(0);
        s[i] = ss[i].const_data_ptr();
        const bool rm = rank_major[i];
        TORCH_CHECK(at + c[i] * RANK <= flat.numel(), "lora_grad_batch: buffer too small");
        outs.push_back(rm ? flat.as_strided({RANK, c[i]}, {c[i], 1}, flat.storage_offset() + at)
                          : flat.as_strided({c[i], RANK}, {RANK, 1}, flat.storage_offset() + at));
        out[i] = static_cast<float*>(outs.back().data_ptr());
        sr[i] = rm ? c[i] : 1;
        sc[i] = rm ? 1 : RANK;
        at += grad_piece(c[i]);
    }
    if (m[0] > 0)
        check(nf4b200_lora_grad_batch(n, z, m, c, ld, s, out, sr, sc, stream_of(zs[0])));
    return outs;
}

int dtype_code(at::ScalarType t) { return t == at::kHalf ? NF4B200_F16 : NF4B200_F32; }

// (normalised rows, 1/rms, sum or None)
std::tuple<Tensor, Tensor, Opt> rmsnorm_fwd(const Tensor& x2, const Opt& delta2, const Tensor& weight, double eps,
                                            bool to_half) {
    const c10::cuda::CUDAGuard guard(x2.device());
    const int64_t rows = x2.size(0), hidden = x2.size(1);
    Tensor out = at::empty({rows, hidden}, x2.options().dtype(to_half ? at::kHalf : at::kFloat));
    Tensor rstd = at::empty({rows}, x2.options().dtype(at::kFloat));
    Opt total;
    if (delta2.has_value()) total = at::empty_like(x2);
    check(nf4b200_rmsnorm_fwd(x2.const_data_ptr(), ptr(delta2), weight.const_data_ptr(),
                              total.has_value() ? total->data_ptr() : nullptr, out.data_ptr(),
                              dtype_code(out.scalar_type()), rstd.data_ptr(), rows, hidden, (float)eps, stream_of(x2)));
    return {out, rstd, total};
}

Tensor rmsnorm_bwd(const Tensor& x2, const Tensor& weight, const Tensor& rstd, const Tensor& dy2, const Opt& d_total,
                   const Opt& dx16) {
    const c10::cuda::CUDAGuard guard(x2.device());
    Tensor dx = at::empty_like(x2);
    check(nf4b200_add_rmsnorm_bwd(x2.const_data_ptr(), weight.const_data_ptr(), rstd.const_data_ptr(),
                                  dy2.const_data_ptr(), dtype_code(dy2.scalar_type()), ptr(d_total), dx.data_ptr(),
                                  dx16.has_value() ? dx16->data_ptr() : nullptr, x2.size(0), x2.size(1),
                                  stream_of(x2)));
    return dx;
}

// Forward-mode differentiation is refused: nothing here would carry a tangent along.
void no_tangent(const char* what, std::initializer_list<const Tensor*> operands) {
    for (const Tensor* t : operands)
        TORCH_CHECK_NOT_IMPLEMENTED(t == nullptr || !t->_fw_grad(0).defined(), "hackaton_b200: ", what,
                                    " has no forward-mode derivative (an operand carries a tangent)");
}

int type_code(at::ScalarType t) { return t == at::kHalf ? NF4B200_F16 : t == at::kBFloat16 ? NF4B200_BF16 : NF4B200_F32; }

// (codes, steps) of a contiguous [rows, cols] tensor; see hackaton_b200.act8.
std::tuple<Tensor, Tensor> act8_room(const Tensor& like, int64_t rows, int64_t cols) {
    const int64_t blocks = (cols + 31) / 32;
    const auto options = like.options().memory_format(c10::nullopt);
    return {at::empty({rows, blocks * 32}, options.dtype(at::kChar)), at::empty({rows, blocks}, options.dtype(at::kByte))};
}

// [..., cols] as contiguous [rows, cols].
Tensor flat_rows(const Tensor& t) {
    const int64_t cols = t.dim() == 0 ? 1 : t.size(-1);
    if (t.dim() == 2 && t.is_contiguous()) return t;
    return t.reshape({cols > 0 ? t.numel() / cols : 0, cols}).contiguous();
}

std::optional<std::tuple<Tensor, Tensor>> act8_quantize(const Tensor& x) {
    const auto type = x.scalar_type();
    if (!x.is_cuda() || x.dim() == 0 || (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat)) return {};
    no_tangent("act8_quantize", {&x});
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor x2 = flat_rows(x.requires_grad() ? x.detach() : x);
    auto [codes, steps] = act8_room(x2, x2.size(0), x2.size(1));
    check(nf4b200_act8_quantize(x2.const_data_ptr(), type_code(type), codes.data_ptr(), steps.data_ptr(), x2.size(0),
                                x2.size(1), stream_of(x2)));
    return std::make_tuple(codes, steps);
}

// Whether codes and steps lie as the kernels read them, for rows of `cols` values.
bool act8_fits(const Tensor& codes, const Tensor& steps, int64_t cols) {
    const int64_t blocks = (cols + 31) / 32;
    return codes.is_cuda() && steps.device() == codes.device() && codes.scalar_type() == at::kChar &&
           steps.scalar_type() == at::kByte && codes.dim() == 2 && steps.dim() == 2 && codes.is_contiguous() &&
           steps.is_contiguous() && codes.size(1) == 32 * blocks && steps.size(1) == blocks && steps.size(0) == codes.size(0) &&
           (reinterpret_cast<uintptr_t>(codes.const_data_ptr()) & 15) == 0;
}

// None for parts that do not make a tensor of that shape.
Opt act8_dequantize(const Tensor& codes, const Tensor& steps, const std::vector<int64_t>& shape, const Tensor& like) {
    if (shape.empty() || !act8_fits(codes, steps, shape.back())) return {};
    int64_t rows = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
    if (shape.back() > 0 && rows != codes.size(0)) return {};
    const c10::cuda::CUDAGuard guard(codes.device());
    Tensor out = at::empty(shape, codes.options().dtype(like.scalar_type()));
    check(nf4b200_act8_dequantize(codes.const_data_ptr(), steps.const_data_ptr(), out.data_ptr(),
                                  type_code(out.scalar_type()), codes.size(0), shape.back(), stream_of(codes)));
    return out;
}

// (Outputs of an autograd function get their shapes when they are made: a view of one could not be changed in place.)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> act8_swiglu_fwd(const Tensor& gate2, const Tensor& up2, at::IntArrayRef shape) {
    const c10::cuda::CUDAGuard guard(gate2.device());
    const int64_t rows = gate2.size(0), cols = gate2.size(1);
    Tensor hidden = at::empty(shape, gate2.options().memory_format(c10::nullopt));
    auto [gc, gs] = act8_room(gate2, rows, cols);
    auto [uc, us] = act8_room(up2, rows, cols);
    check(nf4b200_act8_swiglu_fwd(gate2.const_data_ptr(), up2.const_data_ptr(), hidden.data_ptr(), gc.data_ptr(),
                                  gs.data_ptr(), uc.data_ptr(), us.data_ptr(), rows, cols, stream_of(gate2)));
    return {hidden, gc, gs, uc, us};
}

std::tuple<Tensor, Tensor> act8_swiglu_bwd(const Tensor& d2, const Tensor& gc, const Tensor& gs, const Tensor& uc,
                                           const Tensor& us) {
    const c10::cuda::CUDAGuard guard(d2.device());
    Tensor dg = at::empty_like(d2), du = at::empty_like(d2);
    check(nf4b200_act8_swiglu_bwd(d2.const_data_ptr(), gc.const_data_ptr(), gs.const_data_ptr(), uc.const_data_ptr(),
                                  us.const_data_ptr(), dg.data_ptr(), du.data_ptr(), d2.size(0), d2.size(1),
                                  stream_of(d2)));
    return {dg, du};
}

// Gradients of gradients are refused: the kernels' results would enter them as constants.
void differentiate_once(const char* what) {
    TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), "hackaton_b200: ", what, " has no second derivative (create_graph)");
}

struct SiluMulAct8 : torch::autograd::Function<SiluMulAct8> {
    static Tensor forward(AutogradContext* ctx, const Tensor& gate, const Tensor& up) {
        auto [hidden, gc, gs, uc, us] = act8_swiglu_fwd(flat_rows(gate), flat_rows(up), gate.sizes());
        ctx->save_for_backward({gc, gs, uc, us});
        return hidden;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        differentiate_once("silu_mul with keep8");
        const auto kept = ctx->get_saved_variables();
        auto [dg, du] = act8_swiglu_bwd(flat_rows(grads[0]), kept[0], kept[1], kept[2], kept[3]);
        return {dg.view(grads[0].sizes()), du.view(grads[0].sizes())};
    }
};

Opt silu_mul_act8(const Tensor& gate, const Tensor& up) {
    if (!gate.is_cuda() || gate.device() != up.device() || gate.scalar_type() != at::kHalf || up.scalar_type() != at::kHalf ||
        gate.sizes() != up.sizes())
        return {};
    no_tangent("silu_mul with keep8", {&gate, &up});
    return SiluMulAct8::apply(gate, up);
}

// None for an s that does not fit the kept input.
Opt act8_lora_grad(const Tensor& codes, const Tensor& steps, const Tensor& s, int64_t cols) {
    if (!act8_fits(codes, steps, cols)) return {};
    const int64_t rows = codes.size(0);
    if (s.scalar_type() != at::kHalf || s.device() != codes.device() || s.dim() == 0 || s.size(-1) != RANK || s.numel() != rows * RANK)
        return {};
    no_tangent("lora_grad_act8", {&s});
    const c10::cuda::CUDAGuard guard(codes.device());
    Tensor s2 = flat_rows(s.requires_grad() ? s.detach() : s);
    if ((reinterpret_cast<uintptr_t>(s2.const_data_ptr()) & 15) != 0) s2 = s2.clone();
    const auto options = s2.options().dtype(at::kFloat).memory_format(c10::nullopt);
    if (rows == 0 || cols == 0) return at::zeros({RANK, cols}, options);
    Tensor out = at::empty({RANK, cols}, options);
    const int64_t need = nf4b200_act8_lora_grad_workspace_bytes(rows, cols);
    if (need < 0) check((int)need);
    const Scratch ws(need, s2);
    check(nf4b200_act8_lora_grad(codes.const_data_ptr(), steps.const_data_ptr(), s2.const_data_ptr(), out.data_ptr(),
                                 rows, cols, ws.get(), (size_t)need, stream_of(codes)));
    return out;
}

struct SandwichRows {   // the operands as the kernels read them
    Tensor residual, delta, post, pre;
    Opt gate;
    int64_t rows, hidden;
};

SandwichRows sandwich_rows(const Tensor& residual, const Tensor& delta, const Tensor& post, const Tensor& pre, const Opt& gate) {
    SandwichRows r{residual.contiguous(), delta.contiguous(), post.contiguous(), pre.contiguous(), {}, 0, residual.size(-1)};
    r.rows = residual.numel() / r.hidden;
    if (gate.has_value() && r.rows > 0) r.gate = gate->contiguous();
    return r;
}

// (stream, normed, what the gradient needs or None)
std::tuple<Tensor, Tensor, Opt> sandwich_fwd(const SandwichRows& r, double scale, double eps, bool f32_out, bool train) {
    const c10::cuda::CUDAGuard guard(r.residual.device());
    Tensor out = at::empty_like(r.residual);
    Tensor normed = at::empty(r.residual.sizes(), r.delta.options().dtype(f32_out ? at::kFloat : r.delta.scalar_type()));
    Opt rstd;
    if (train) rstd = at::empty({r.rows, 4}, r.residual.options());
    check(nf4b200_sandwich_norm_fwd(r.residual.const_data_ptr(), r.delta.const_data_ptr(), type_code(r.delta.scalar_type()),
                                    r.post.const_data_ptr(), r.pre.const_data_ptr(), ptr(r.gate),
                                    r.gate.has_value() ? r.gate->numel() / r.hidden : 0, out.data_ptr(), normed.data_ptr(),
                                    type_code(normed.scalar_type()), train ? rstd->data_ptr() : nullptr, r.rows, r.hidden,
                                    (float)scale, (float)eps, stream_of(r.residual)));
    return {out, normed, rstd};
}

struct SandwichNorm : torch::autograd::Function<SandwichNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& residual, const Tensor& delta, const Tensor& post,
                                 const Tensor& pre, const Opt& gate, double scale, double eps, bool f32_out) {
        const SandwichRows r = sandwich_rows(residual, delta, post, pre, gate);
        auto [stream, normed, rstd] = sandwich_fwd(r, scale, eps, f32_out, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({stream, r.delta, r.post, r.pre, r.gate.has_value() ? *r.gate : Tensor(), *rstd});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["normed"] = (int64_t)normed.scalar_type();
        ctx->saved_data["no rows"] = gate.has_value() && r.rows == 0;
        if (gate.has_value()) ctx->saved_data["gate"] = gate->sizes().vec();
        return {stream, normed};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        differentiate_once("sandwich_norm");
        const auto kept = ctx->get_saved_variables();
        const Tensor &s = kept[0], &d = kept[1], &post = kept[2], &pre = kept[3], &gate = kept[4], &rstd = kept[5];
        variable_list g(8);
        if (!grads[0].defined() && !grads[1].defined()) return g;
        const c10::cuda::CUDAGuard guard(s.device());
        const int64_t hidden = s.size(-1), rows = s.numel() / hidden, gates = gate.defined() ? gate.numel() / hidden : 0;
        const Tensor* like[] = {&s, &d, &post, &pre, &gate};
        void* at_[5] = {};
        for (int i = 0; i < 5; ++i) {
            if (!like[i]->defined() || !ctx->needs_input_grad(i)) continue;
            g[i] = rows == 0 ? at::zeros_like(*like[i]) : at::empty_like(*like[i]);
            at_[i] = g[i].data_ptr();
        }
        if (rows == 0) {
            if (ctx->saved_data["no rows"].toBool() && ctx->needs_input_grad(4))
                g[4] = at::zeros(ctx->saved_data["gate"].toIntVector(), s.options());
            return g;
        }
        const Tensor d_stream = grads[0].defined() ? grads[0].to(at::kFloat).contiguous() : Tensor();
        const auto normed = (at::ScalarType)ctx->saved_data["normed"].toInt();
        const Tensor d_normed = grads[1].defined() ? grads[1].to(normed).contiguous() : at::zeros(s.sizes(), s.options().dtype(normed));
        const int64_t need = nf4b200_sandwich_norm_workspace_bytes(rows, hidden, gates);
        if (need < 0) check((int)need);
        const Scratch ws(need, s);
        check(nf4b200_sandwich_norm_bwd(s.const_data_ptr(), d.const_data_ptr(), type_code(d.scalar_type()),
                                        post.const_data_ptr(), pre.const_data_ptr(),
                                        gate.defined() ? gate.const_data_ptr() : nullptr, gates, rstd.const_data_ptr(),
                                        d_stream.defined() ? d_stream.const_data_ptr() : nullptr, d_normed.const_data_ptr(),
                                        type_code(d_normed.scalar_type()), at_[0], at_[1], at_[2], at_[3], at_[4], rows, hidden,
                                        (float)ctx->saved_data["scale"].toDouble(), ws.get(), (size_t)need, stream_of(s)));
        return g;
    }
};

// (stream, normed); gate: [hidden] or [gates, hidden] over the stream's rows. None for what it does not take.
std::optional<std::tuple<Tensor, Tensor>> sandwich_norm(const Tensor& residual, const Tensor& delta, const Tensor& post,
                                                        const Tensor& pre, const Opt& gate, double scale, double eps, bool f32_out) {
    if (!residual.is_cuda() || residual.scalar_type() != at::kFloat || residual.dim() == 0 || delta.sizes() != residual.sizes() ||
        delta.device() != residual.device())
        return {};
    const auto type = delta.scalar_type();
    if (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) return {};
    const int64_t hidden = residual.size(-1);
    if (hidden < 1 || hidden > 16384) return {};
    const int64_t rows = residual.numel() / hidden;
    const auto weight = [&](const Tensor& w) { return w.scalar_type() == at::kFloat && w.device() == residual.device(); };
    const auto row = [&](const Tensor& w) { return weight(w) && w.dim() == 1 && w.size(0) == hidden; };
    if (!row(post) || !row(pre)) return {};
    if (gate.has_value() && (!weight(*gate) || gate->dim() == 0 || gate->dim() > 2 || gate->size(-1) != hidden ||
                             (rows > 0 && (gate->numel() == 0 || rows % (gate->numel() / hidden) != 0))))
        return {};
    no_tangent("sandwich_norm", {&residual, &delta, &post, &pre, gate.has_value() ? &*gate : nullptr});
    if (at::GradMode::is_enabled() && (residual.requires_grad() || delta.requires_grad() || post.requires_grad() ||
                                       pre.requires_grad() || (gate.has_value() && gate->requires_grad()))) {
        const variable_list out = SandwichNorm::apply(residual, delta, post, pre, gate, scale, eps, f32_out);
        return std::make_tuple(out[0], out[1]);
    }
    auto [stream, normed, rstd] = sandwich_fwd(sandwich_rows(residual, delta, post, pre, gate), scale, eps, f32_out, false);
    return std::make_tuple(stream, normed);
}

// Weight of the vocabulary loss as the kernels read it.
Tensor head_view(const Tensor& w) {
    if (w.stride(1) == 1 && w.stride(0) % 8 == 0 && w.stride(0) >= w.size(1) &&
        (reinterpret_cast<uintptr_t>(w.const_data_ptr()) & 15) == 0)
        return w;
    return w.clone(at::MemoryFormat::Contiguous);
}

int64_t sized(int64_t bytes) {
    if (bytes < 0) check((int)bytes);
    return bytes;
}

// (losses, logsumexps, both in the targets' shape, what the gradient needs)
std::tuple<Tensor, Tensor, Tensor> vocab_loss_fwd(const Tensor& x, const Tensor& weight, const Tensor& targets, int64_t grads) {
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t hidden = weight.size(1), vocab = weight.size(0);
    const Tensor x2 = rows_view(x, hidden), w = head_view(weight), t = targets.reshape({-1}).contiguous();
    const int64_t rows = x2.size(0);
    const auto options = x.options().dtype(at::kFloat).memory_format(c10::nullopt);
    Tensor losses = at::empty(targets.sizes(), options), lse = at::empty(targets.sizes(), options);
    Tensor kept = at::empty({sized(nf4b200_vocab_loss_kept_bytes(rows, hidden, (int)grads))}, options.dtype(at::kByte));
    const int64_t need = sized(nf4b200_vocab_loss_workspace_bytes(rows, vocab, hidden, (int)grads, 0));
    const Scratch ws(need, x2);
    check(nf4b200_vocab_loss_fwd(x2.const_data_ptr(), x2.stride(0), w.const_data_ptr(), w.stride(0), type_code(x.scalar_type()),
                                 t.const_data_ptr(), losses.data_ptr(), lse.data_ptr(), rows, vocab, hidden, (int)grads, kept.data_ptr(),
                                 ws.get(), (size_t)need, stream_of(x)));
    return {losses, lse, kept};
}

// (gradient of the hidden states [rows, hidden], of the weight), as far as they are wanted
std::tuple<Opt, Opt> vocab_loss_bwd(const Tensor& weight, const Tensor& kept, const Opt& d_losses, const Opt& d_lse,
                                    int64_t rows, int64_t grads, bool want_x, bool want_weight) {
    const c10::cuda::CUDAGuard guard(weight.device());
    const int64_t hidden = weight.size(1), vocab = weight.size(0);
    const Tensor w = head_view(weight);
    const auto options = weight.options().memory_format(c10::nullopt);
    const auto flat = [](const Opt& g) { return g.has_value() ? Opt(g->reshape({-1}).to(at::kFloat)) : Opt(); };
    const Opt dl = flat(d_losses), dz = flat(d_lse);
    const bool none = rows == 0 || (!dl.has_value() && !dz.has_value());
    Opt dx, dw;
    if (want_x) dx = none ? at::zeros({rows, hidden}, options) : at::empty({rows, hidden}, options);
    if (want_weight) dw = none ? at::zeros({vocab, hidden}, options) : at::empty({vocab, hidden}, options);
    if (none || (!want_x && !want_weight)) return {dx, dw};
    const int64_t need = want_weight ? sized(nf4b200_vocab_loss_workspace_bytes(rows, vocab, hidden, (int)grads, 1)) : 0;
    const Scratch ws(need, w);
    const auto step = [](const Opt& g) { return g.has_value() && g->size(0) > 1 ? g->stride(0) : (int64_t)0; };
    check(nf4b200_vocab_loss_bwd(w.const_data_ptr(), w.stride(0), type_code(w.scalar_type()), ptr(dl), step(dl), ptr(dz), step(dz),
                                 dx.has_value() ? dx->data_ptr() : nullptr, dw.has_value() ? dw->data_ptr() : nullptr, rows,
                                 vocab, hidden, (int)grads, const_cast<void*>(kept.const_data_ptr()), ws.get(), (size_t)need, stream_of(w)));
    return {dx, dw};
}

struct VocabLoss : torch::autograd::Function<VocabLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& targets,
                                 int64_t grads) {
        auto [losses, lse, kept] = vocab_loss_fwd(hidden, weight, targets, grads);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({weight, kept});
        ctx->saved_data["grads"] = grads;
        ctx->saved_data["rows"] = targets.numel();
        ctx->saved_data["shape"] = hidden.sizes().vec();
        return {losses, lse};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        differentiate_once("vocab_cross_entropy");
        variable_list g(4);
        if (!grads[0].defined() && !grads[1].defined()) return g;
        const auto kept = ctx->get_saved_variables();
        const auto opt = [](const Tensor& t) { return t.defined() ? Opt(t) : Opt(); };
        auto [dx, dw] = vocab_loss_bwd(kept[0], kept[1], opt(grads[0]), opt(grads[1]), ctx->saved_data["rows"].toInt(),
                                       ctx->saved_data["grads"].toInt(), ctx->needs_input_grad(0), ctx->needs_input_grad(1));
        if (dx.has_value()) g[0] = dx->view(ctx->saved_data["shape"].toIntVector());
        if (dw.has_value()) g[1] = *dw;
        return g;
    }
};

// (losses, logsumexps), or None for what it does not take.
std::optional<std::tuple<Tensor, Tensor>> vocab_loss(const Tensor& hidden, const Tensor& weight, const Tensor& targets) {
    const auto type = hidden.scalar_type();
    if (!hidden.is_cuda() || weight.device() != hidden.device() || targets.device() != hidden.device() ||
        (type != at::kHalf && type != at::kBFloat16) || weight.scalar_type() != type || targets.scalar_type() != at::kLong ||
        weight.dim() != 2 || hidden.dim() != targets.dim() + 1 || weight.size(0) == 0 || weight.size(1) == 0 ||
        weight.size(1) % 8 != 0 || hidden.size(-1) != weight.size(1) || hidden.sizes().slice(0, targets.dim()) != targets.sizes())
        return {};
    no_tangent("vocab_cross_entropy", {&hidden, &weight});
    int64_t grads = 0;
    if (at::GradMode::is_enabled()) grads = (hidden.requires_grad() ? 1 : 0) | (weight.requires_grad() ? 2 : 0);
    if (grads != 0) {
        const variable_list out = VocabLoss::apply(hidden, weight, targets, grads);
        return std::make_tuple(out[0], out[1]);
    }
    auto [losses, lse, kept] = vocab_loss_fwd(hidden, weight, targets, 0);
    return std::make_tuple(losses, lse);
}

struct Rotation {   // everything about one rotation that is not a tensor
    int64_t tokens, seq, heads, kv_heads, dim, batch_stride;
    bool padded, f32;
};

void rotate(const Rotation& r, const Tensor (&src)[3], Tensor (&dst)[3], const Tensor& cos, const Tensor& sin,
            const Tensor& b_idx, const Tensor& t_idx, bool backward) {
    check(nf4b200_qkv_rotate(src[0].const_data_ptr(), src[1].const_data_ptr(), src[2].const_data_ptr(),
                             dst[0].data_ptr(), dst[1].data_ptr(), dst[2].data_ptr(), cos.const_data_ptr(),
                             sin.const_data_ptr(), r.batch_stride, cos.stride(1), b_idx.const_data_ptr(),
                             t_idx.const_data_ptr(), r.tokens, r.seq, (int)r.heads, (int)r.kv_heads, (int)r.dim,
                             r.padded ? 1 : 0, backward ? 1 : 0, r.f32 ? NF4B200_F32 : NF4B200_F16,
                             stream_of(dst[0])));
}

// (q, k, v heads, and what the gradient needs: cos, sin, b_idx, t_idx as the kernel read them, geometry)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Rotation>
rotate_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos_in, const Tensor& sin_in,
           const Tensor& b_in, const Tensor& t_in, int64_t batch, int64_t seq, int64_t heads, int64_t kv_heads,
           int64_t dim, bool padded) {
    const c10::cuda::CUDAGuard guard(q.device());
    const Tensor cos = cos_in.contiguous(), sin = sin_in.contiguous();
    const Tensor b_idx = b_in.to(at::kInt).contiguous(), t_idx = t_in.to(at::kInt).contiguous();
    Rotation r = {q.size(0), seq, heads, kv_heads, dim, cos.size(0) == 1 ? 0 : cos.stride(0), padded,
                  q.scalar_type() == at::kFloat};
    const Tensor src[3] = {q.contiguous(), k.contiguous(), v.contiguous()};
    const auto options = q.options().dtype(at::kHalf);
    Tensor dst[3];
    for (auto& d : dst)   // padded: positions no token maps to stay zero
        d = padded ? at::zeros({batch, heads, seq, r.dim}, options) : at::empty({r.tokens, heads, r.dim}, options);
    rotate(r, src, dst, cos, sin, b_idx, t_idx, false);
    return {dst[0], dst[1], dst[2], cos, sin, b_idx, t_idx, r};
}

std::tuple<Tensor, Tensor, Tensor> rotate_bwd(const Tensor& gq, const Tensor& gk, const Tensor& gv, const Tensor& cos,
                                              const Tensor& sin, const Tensor& b_idx, const Tensor& t_idx,
                                              const Rotation& r) {
    const c10::cuda::CUDAGuard guard(gq.device());
    const Tensor src[3] = {gq.to(at::kHalf).contiguous(), gk.to(at::kHalf).contiguous(),
                           gv.to(at::kHalf).contiguous()};
    const auto options = gq.options().dtype(r.f32 ? at::kFloat : at::kHalf);
    Tensor dst[3];
    for (int i = 0; i < 3; ++i) dst[i] = at::empty({r.tokens, (i == 0 ? r.heads : r.kv_heads) * r.dim}, options);
    rotate(r, src, dst, cos, sin, b_idx, t_idx, true);
    return {dst[0], dst[1], dst[2]};
}

}  // namespace

// What the module was compiled against; the build looks for the text in the file.
#ifndef NF4B200_HOST_TARGET
#define NF4B200_HOST_TARGET "unknown"
#endif
const char BUILT_FOR[] = "built for " NF4B200_HOST_TARGET ";";

PYBIND11_MODULE(_host, m) {
    m.attr("built_for") = py::str(BUILT_FOR + sizeof "built for " - 1, sizeof NF4B200_HOST_TARGET - 1);
    py::class_<Rotation>(m, "Rotation");
    m.def("stamps", &stamps);
    // An allocation or a launch can block (cudaMalloc, a full launch queue): other Python threads go on.
    using unlocked = py::call_guard<py::gil_scoped_release>;
    m.def("linear_fwd", &linear_fwd, unlocked());
    m.def("linear_bwd_dx", &linear_bwd_dx, unlocked());
    m.def("linear_fwd_group", &linear_fwd_group, unlocked());
    m.def("linear_bwd_dx_group", &linear_bwd_dx_group, unlocked());
    m.def("lora_side", &lora_side, unlocked());
    m.def("lora_grad_batch", &lora_grad_batch, unlocked());
    m.def("rmsnorm_fwd", &rmsnorm_fwd, unlocked());
    m.def("rmsnorm_bwd", &rmsnorm_bwd, unlocked());
    m.def("act8_quantize", &act8_quantize, unlocked());
    m.def("act8_dequantize", &act8_dequantize, unlocked());
    m.def("silu_mul_act8", &silu_mul_act8, unlocked());
    m.def("act8_swiglu_bwd", &act8_swiglu_bwd, unlocked());
    m.def("act8_lora_grad", &act8_lora_grad, unlocked());
    m.def("sandwich_norm", &sandwich_norm, unlocked());
    m.def("vocab_loss", &vocab_loss, unlocked());
    m.def("rotate_fwd", &rotate_fwd, unlocked());
    m.def("rotate_bwd", &rotate_bwd, unlocked());
}
