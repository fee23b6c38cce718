// The _training PyTorch extension: what tcc_amd/training.py calls.  It checks
// tensors, allocates outputs and workspaces and calls the C-ABI of
// include/tcc_training.h on torch's current stream.  The same checks and calls
// from Python through ctypes took 11 to 26 us a call, more than the kernels of
// small batches run.
//
// TypeError: a tensor of the wrong type or place; ValueError: sizes, strides
// and values that no call takes; tcc_amd._lib.TccError: an error of the
// library.
#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/variable.h>

#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cstdint>
#include <memory>
#include <numeric>
#include <optional>
#include <string>
#include <unordered_set>
#include <utility>
#include <vector>

#include "tcc_swtcf.h"
#include "tcc_training.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using MaybeTensor = std::optional<Tensor>;

[[noreturn]] void type_error(const std::string& what) { throw py::type_error(what); }
[[noreturn]] void value_error(const std::string& what) { throw py::value_error(what); }

void check(int rc) {
    if (rc == TCC_OK) return;
    const std::string what = tcc_last_error();
    const py::object cls = py::module_::import("tcc_amd._lib").attr("TccError");
    const py::object err = cls(rc, what);
    PyErr_SetObject(cls.ptr(), err.ptr());
    throw py::error_already_set();
}

std::string shape_of(const Tensor& t) {
    std::string s = "(";
    for (std::int64_t d = 0; d < t.dim(); ++d) s += (d ? ", " : "") + std::to_string(t.size(d));
    return s + ")";
}

std::string place_of(const Tensor& t) { return std::string(t.dtype().name()) + " on " + t.device().str(); }

std::uint32_t dtype_of(const Tensor& t, const char* name) {
    if (t.is_cuda()) {
        switch (t.scalar_type()) {
            case at::kFloat: return TCC_F32;
            case at::kBFloat16: return TCC_BF16;
            case at::kHalf: return TCC_F16;
            default: break;
        }
    }
    type_error(std::string(name) + " must be an fp32, bf16 or fp16 device tensor (got " + place_of(t) + ")");
}

std::uint32_t index_bytes(const Tensor& t, const char* name) {
    if (t.is_cuda() && t.scalar_type() == at::kLong) return 8;
    if (t.is_cuda() && t.scalar_type() == at::kInt) return 4;
    type_error(std::string(name) + " must be an int32 or int64 device tensor (got " + place_of(t) + ")");
}

void on_current_device(const Tensor& t) {
    const auto d = c10::hip::current_device();
    if (t.get_device() != d)
        value_error("a tensor is on " + t.device().str() + ", the current device is cuda:" + std::to_string(d));
}
void on_current_device(const MaybeTensor& t) {
    if (t) on_current_device(*t);
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// torch.empty; where memory is short, what the builders keep is given back
// first.
Tensor empty(at::IntArrayRef shape, const at::TensorOptions& options) {
    try {
        return at::empty(shape, options);
    } catch (const c10::OutOfMemoryError&) {
        tcc_release_kept_memory();
    }
    return at::empty(shape, options);
}

Tensor workspace(std::size_t bytes, const Tensor& like) {
    return empty({static_cast<std::int64_t>(bytes)}, like.options().dtype(at::kByte));
}

// Autograd has to know of what a call wrote in place: a graph that saved the
// tensor refuses its backward pass then, instead of taking the new values.
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(const std::vector<Tensor>& list) {
    for (const Tensor& t : list) written(t);
}

void* ptr(const MaybeTensor& t) { return t ? t->data_ptr() : nullptr; }

// A matrix whose rows are contiguous, and its row stride (a copy where the
// rows are not contiguous or overlap).
struct Rows {
    Tensor t;
    std::int64_t ld;
    Rows(const Tensor& x, const char* name) : t(x) {
        if (x.dim() != 2 || x.size(1) == 0) value_error(std::string(name) + " must be a matrix with columns (got " + shape_of(x) + ")");
        ld = x.size(1);
        if (x.is_contiguous()) return;
        if (x.stride(1) == 1 && x.stride(0) >= ld) ld = x.stride(0);
        else t = x.contiguous();
    }
};

// The row stride of a matrix that is written in place.
std::int64_t own_rows(const Tensor& t, const char* name) {
    if (t.is_contiguous()) return t.size(-1);
    if (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= t.size(1)) return t.stride(0);
    value_error(std::string(name) + " must have contiguous rows");
}

std::int64_t padding_of(std::optional<std::int64_t> padding, std::int64_t rows) {
    if (!padding) return -1;
    if (*padding < 0 || *padding >= rows)
        value_error("padding_idx " + std::to_string(*padding) + " is no row of a table of " + std::to_string(rows));
    return *padding;
}

// The columns of a table; the C-ABI counts them in 32 bits.
std::uint32_t columns_of(std::int64_t D) {
    if (D > 0xFFFFFFFFll) value_error("a table of " + std::to_string(D) + " columns is too wide");
    return static_cast<std::uint32_t>(D);
}

std::uint32_t* error_word(const MaybeTensor& t) {
    if (!t) return nullptr;
    if (!t->is_cuda() || t->scalar_type() != at::kInt || t->numel() < 1) type_error("device_error must be an int32 device tensor");
    on_current_device(*t);
    return static_cast<std::uint32_t*>(t->data_ptr());
}

// ---------------------------------------------------------------- embedding

Tensor embedding_lookup(const Tensor& table, const Tensor& ids, double scale, std::optional<std::int64_t> padding,
                        const MaybeTensor& out, const MaybeTensor& deviceError) {
    const std::uint32_t code = dtype_of(table, "table");
    const std::uint32_t width = index_bytes(ids, "ids");
    const std::uint32_t cols = table.dim() == 2 ? columns_of(table.size(1)) : 0;
    const Rows rows(table, "table");
    const Tensor flat = ids.contiguous();
    const std::int64_t V = table.size(0), D = table.size(1), pad = padding_of(padding, V);
    std::uint32_t* err = error_word(deviceError);
    on_current_device(table);
    on_current_device(ids);
    on_current_device(out);
    std::vector<std::int64_t> shape(ids.sizes().begin(), ids.sizes().end());
    shape.push_back(D);
    Tensor to;
    std::int64_t ldo = D;
    if (out) {
        to = *out;
        if (to.scalar_type() != table.scalar_type() || to.sizes() != at::IntArrayRef(shape))
            value_error("out must be of the table's type and of the shape of ids and a row");
        ldo = own_rows(to, "out");
    } else {
        to = empty(shape, table.options());
    }
    check(tcc_embedding_lookup(rows.t.data_ptr(), rows.ld, code, flat.data_ptr(), width, flat.numel(), V, cols,
                               static_cast<float>(scale), pad, to.data_ptr(), ldo, err, stream_of(table)));
    if (out) written(to);
    return to;
}

Tensor embedding_grad(const Tensor& dOut, const Tensor& ids, std::int64_t V, double scale,
                      std::optional<std::int64_t> padding, const MaybeTensor& grad, bool accumulate,
                      const MaybeTensor& deviceError) {
    const std::uint32_t code = dtype_of(dOut, "d_out");
    const std::uint32_t width = index_bytes(ids, "ids");
    if (dOut.dim() < 1 || dOut.sizes().slice(0, dOut.dim() - 1) != ids.sizes())
        value_error("d_out " + shape_of(dOut) + " does not have a row for each of the ids " + shape_of(ids));
    if (V < 0) value_error("num_rows is not negative");
    const std::int64_t n = ids.numel(), D = dOut.size(-1);
    const std::uint32_t cols = columns_of(D);
    const Rows rows(dOut.dim() == 2 ? dOut : dOut.reshape({n, D}), "d_out");
    const Tensor flat = ids.contiguous();
    const std::int64_t pad = padding_of(padding, V);
    std::uint32_t* err = error_word(deviceError);
    on_current_device(dOut);
    on_current_device(ids);
    on_current_device(grad);
    Tensor to;
    std::int64_t ldg = D;
    if (grad) {
        to = *grad;
        if (to.scalar_type() != dOut.scalar_type() || to.dim() != 2 || to.size(0) != V || to.size(1) != D)
            value_error("grad must be of d_out's type and of shape (" + std::to_string(V) + ", " + std::to_string(D) + ")");
        ldg = own_rows(to, "grad");
    } else {
        if (accumulate) value_error("accumulate=True needs a gradient to add to");
        to = empty({V, D}, dOut.options());
    }
    const std::size_t need = tcc_embedding_grad_workspace_bytes(n, V, cols);
    const Tensor ws = workspace(need, dOut);
    check(tcc_embedding_grad(rows.t.data_ptr(), rows.ld, code, flat.data_ptr(), width, n, V, cols,
                             static_cast<float>(scale), pad, to.data_ptr(), ldg, accumulate, err, ws.data_ptr(), need,
                             stream_of(dOut)));
    if (grad) written(to);
    return to;
}

// ---------------------------------------------------------------- group norm

// A group norm's tensors as the C-ABI takes them.
struct Norm {
    tcc_group_norm_shape s{};
    Rows rows;
    MaybeTensor weight, bias, offsets;  // kept until the launch

    static Tensor as_rows(const Tensor& x) {
        if (x.dim() < 2) value_error("x must be [rows x channels] or [segments x ... x channels]");
        return x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    }

    Norm(const Tensor& x, std::int64_t groups, const MaybeTensor& w, const MaybeTensor& b, const MaybeTensor& off, double eps,
         std::uint32_t activation, std::optional<std::int64_t> maxRows)
        : rows(((void)dtype_of(x, "x"), as_rows(x)), "x") {
        s.dtype = dtype_of(x, "x");
        const std::int64_t C = x.size(-1);
        if (groups < 1 || C % groups != 0)
            value_error(std::to_string(groups) + " groups do not divide " + std::to_string(C) + " channels");
        if (C > 4096) value_error("at most 4096 channels (got " + std::to_string(C) + ")");
        std::int64_t segments = x.dim() == 2 ? 1 : x.size(0);
        if (off) {
            if (x.dim() != 2) value_error("offsets go with x of [rows x channels]");
            s.offsetBytes = index_bytes(*off, "offsets");
            if (off->dim() != 1 || off->numel() < 2) value_error("offsets are one more than the segments");
            offsets = off->contiguous();
            segments = off->numel() - 1;
            s.offsets = offsets->data_ptr();
        }
        if (maxRows && *maxRows < 0) value_error("max_rows is not negative");
        const std::int64_t N = rows.t.size(0);
        s.N = N;
        s.B = segments;
        s.maxRows = off ? maxRows.value_or(0) : segments > 0 ? N / segments : 0;
        s.C = static_cast<std::uint32_t>(C);
        s.G = static_cast<std::uint32_t>(groups);
        s.paramDtype = TCC_F32;
        for (const auto& [p, name, to] : {std::tuple{&w, "weight", &weight}, std::tuple{&b, "bias", &bias}}) {
            if (!*p) continue;
            s.paramDtype = dtype_of(**p, name);
            if ((*p)->dim() != 1 || (*p)->size(0) != C)
                value_error(std::string(name) + " must hold a value for each of the " + std::to_string(C) + " channels (got " +
                            shape_of(**p) + ")");
            on_current_device(**p);
            *to = (*p)->contiguous();
        }
        if (w && b && w->scalar_type() != b->scalar_type()) value_error("weight and bias must be of one type");
        on_current_device(x);
        on_current_device(off);
        s.activation = activation;
        s.eps = static_cast<float>(eps);
    }
};

std::tuple<Tensor, Tensor, Tensor> group_norm(const Tensor& x, std::int64_t groups, const MaybeTensor& weight,
                                              const MaybeTensor& bias, const MaybeTensor& offsets, double eps,
                                              std::uint32_t activation, std::optional<std::int64_t> maxRows) {
    const Norm k(x, groups, weight, bias, offsets, eps, activation, maxRows);
    const std::size_t need = tcc_group_norm_workspace_bytes(&k.s, 0);
    const Tensor y = empty(x.sizes(), x.options());
    const auto f32 = x.options().dtype(at::kFloat);
    const std::int64_t B = static_cast<std::int64_t>(k.s.B);
    const Tensor mean = empty({B, groups}, f32), rstd = empty({B, groups}, f32);
    const Tensor ws = workspace(need, x);
    check(tcc_group_norm(&k.s, k.rows.t.data_ptr(), k.rows.ld, ptr(k.weight), ptr(k.bias), y.data_ptr(), k.s.C,
                         mean.data_ptr<float>(), rstd.data_ptr<float>(), ws.data_ptr(), need, stream_of(x)));
    return {y, mean, rstd};
}

std::tuple<Tensor, MaybeTensor, MaybeTensor> group_norm_grad(const Tensor& dy, const Tensor& x, const Tensor& mean,
                                                             const Tensor& rstd, std::int64_t groups,
                                                             const MaybeTensor& weight, const MaybeTensor& bias,
                                                             const MaybeTensor& offsets, std::uint32_t activation,
                                                             std::optional<std::int64_t> maxRows) {
    (void)dtype_of(x, "x");
    if (dy.scalar_type() != x.scalar_type() || dy.sizes() != x.sizes() || !dy.is_cuda())
        value_error("d_y must be of x's type, shape " + shape_of(x) + " and device");
    const Norm k(x, groups, weight, bias, offsets, 0.0, activation, maxRows);
    const std::int64_t B = static_cast<std::int64_t>(k.s.B);
    for (const auto& [t, name] : {std::pair{&mean, "mean"}, std::pair{&rstd, "rstd"}}) {
        if (!t->is_cuda() || t->scalar_type() != at::kFloat || !t->is_contiguous() || t->dim() != 2 || t->size(0) != B ||
            t->size(1) != groups)
            value_error(std::string(name) + " must be contiguous float32 of shape (" + std::to_string(B) + ", " +
                        std::to_string(groups) + ")");
        on_current_device(*t);
    }
    on_current_device(dy);
    const Rows rows(Norm::as_rows(dy), "d_y");
    const std::size_t need = tcc_group_norm_workspace_bytes(&k.s, 1);
    const Tensor dx = empty(x.sizes(), x.options());
    const auto f32 = x.options().dtype(at::kFloat);
    MaybeTensor dw, db;
    if (weight) dw = empty({x.size(-1)}, f32);
    if (bias) db = empty({x.size(-1)}, f32);
    const Tensor ws = workspace(need, x);
    check(tcc_group_norm_grad(&k.s, rows.t.data_ptr(), rows.ld, k.rows.t.data_ptr(), k.rows.ld, mean.data_ptr<float>(),
                              rstd.data_ptr<float>(), ptr(k.weight), ptr(k.bias), dx.data_ptr(), k.s.C,
                              static_cast<float*>(ptr(dw)), static_cast<float*>(ptr(db)), ws.data_ptr(), need,
                              stream_of(x)));
    return {dx, dw, db};
}

// ---------------------------------------------------------------- capture

// Whether a gradient of one of these would run through a node of a living graph
// that was made on the default stream, or be accumulated in a leaf that such a graph
// holds, however far behind the tensor: a captured backward pass would have to wait
// for that stream, which a capture does not allow.
bool held_by_default_stream(const std::vector<MaybeTensor>& tensors) {
    using torch::autograd::Node;
    std::vector<std::shared_ptr<Node>> next;
    std::unordered_set<const Node*> seen;
    const auto take = [&](std::shared_ptr<Node> node) {
        if (node != nullptr && seen.insert(node.get()).second) next.push_back(std::move(node));
    };
    for (const MaybeTensor& t : tensors)
        if (t && t->requires_grad()) take(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    while (!next.empty()) {
        const std::shared_ptr<Node> node = std::move(next.back());
        next.pop_back();
        const std::optional<c10::Stream> stream = node->stream();
        if (stream && stream->id() == 0) return true;
        for (const torch::autograd::Edge& e : node->next_edges()) take(e.function);
    }
    return false;
}

// ---------------------------------------------------------------- layer norm

// Rows of x's last dimension (a view or a copy).
Tensor rows_of(const Tensor& x, const char* name) {
    if (x.dim() < 1 || x.size(-1) == 0) value_error(std::string(name) + " must have channels (got " + shape_of(x) + ")");
    return x.dim() == 2 ? x : x.reshape({x.numel() / x.size(-1), x.size(-1)});
}

// A tensor of x's type, shape and device, as rows.
Rows rows_like(const Tensor& t, const Tensor& x, const char* name) {
    if (t.scalar_type() != x.scalar_type() || t.sizes() != x.sizes() || !t.is_cuda())
        value_error(std::string(name) + " must be of x's type, shape " + shape_of(x) + " and device");
    on_current_device(t);
    return Rows(rows_of(t, name), name);
}

// A layer norm's tensors as the C-ABI takes them.
struct LayerNorm {
    tcc_layer_norm_shape s{};
    Rows rows;
    MaybeTensor weight, bias;  // kept until the launch

    LayerNorm(const Tensor& x, const MaybeTensor& w, const MaybeTensor& b, double eps, std::uint32_t activation)
        : rows(((void)dtype_of(x, "x"), rows_of(x, "x")), "x") {
        s.dtype = dtype_of(x, "x");
        const std::int64_t C = x.size(-1);
        if (C > 16384) value_error("at most 16384 channels (got " + std::to_string(C) + ")");
        if (!(eps >= 0)) value_error("eps is not negative (got " + std::to_string(eps) + ")");
        s.N = rows.t.size(0);
        s.C = static_cast<std::uint32_t>(C);
        s.paramDtype = TCC_F32;
        for (const auto& [p, name, to] : {std::tuple{&w, "weight", &weight}, std::tuple{&b, "bias", &bias}}) {
            if (!*p) continue;
            s.paramDtype = dtype_of(**p, name);
            if ((*p)->dim() != 1 || (*p)->size(0) != C)
                value_error(std::string(name) + " must hold a value for each of the " + std::to_string(C) + " channels (got " +
                            shape_of(**p) + ")");
            on_current_device(**p);
            *to = (*p)->contiguous();
        }
        if (w && b && w->scalar_type() != b->scalar_type()) value_error("weight and bias must be of one type");
        on_current_device(x);
        s.activation = activation;
        s.eps = static_cast<float>(eps);
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias,
                                                      const MaybeTensor& residual, double eps, std::uint32_t activation) {
    const LayerNorm k(x, weight, bias, eps, activation);
    std::optional<Rows> res;
    if (residual) res.emplace(rows_like(*residual, x, "residual"));
    const Tensor y = empty(x.sizes(), x.options());
    const Tensor h = residual ? empty(x.sizes(), x.options()) : x;
    const auto stats = x.sizes().slice(0, x.dim() - 1);
    const auto f32 = x.options().dtype(at::kFloat);
    const Tensor mean = empty(stats, f32), rstd = empty(stats, f32);
    check(tcc_layer_norm(&k.s, k.rows.t.data_ptr(), k.rows.ld, res ? res->t.data_ptr() : nullptr, res ? res->ld : 0,
                         ptr(k.weight), ptr(k.bias), y.data_ptr(), k.s.C, residual ? h.data_ptr() : nullptr, k.s.C,
                         mean.data_ptr<float>(), rstd.data_ptr<float>(), stream_of(x)));
    return {y, h, mean, rstd};
}

std::tuple<Tensor, MaybeTensor, MaybeTensor> layer_norm_grad(const Tensor& dy, const Tensor& h, const Tensor& mean,
                                                             const Tensor& rstd, const MaybeTensor& weight,
                                                             const MaybeTensor& bias, const MaybeTensor& dSum,
                                                             std::uint32_t activation, bool parameters) {
    const LayerNorm k(h, weight, bias, 0.0, activation);
    const Rows rows = rows_like(dy, h, "d_y");
    std::optional<Rows> add;
    if (dSum) add.emplace(rows_like(*dSum, h, "d_sum"));
    const auto stats = h.sizes().slice(0, h.dim() - 1);
    for (const auto& [t, name] : {std::pair{&mean, "mean"}, std::pair{&rstd, "rstd"}}) {
        if (!t->is_cuda() || t->scalar_type() != at::kFloat || !t->is_contiguous() || t->sizes() != stats)
            value_error(std::string(name) + " must be contiguous float32, a value for each row of x");
        on_current_device(*t);
    }
    const Tensor dx = empty(h.sizes(), h.options());
    const auto f32 = h.options().dtype(at::kFloat);
    MaybeTensor dw, db, ws;
    if (weight && parameters) dw = empty({h.size(-1)}, f32);
    if (bias && parameters) db = empty({h.size(-1)}, f32);
    const std::size_t need = dw || db ? tcc_layer_norm_grad_workspace_bytes(&k.s) : 0;
    if (need > 0) ws = workspace(need, h);
    check(tcc_layer_norm_grad(&k.s, rows.t.data_ptr(), rows.ld, k.rows.t.data_ptr(), k.rows.ld, mean.data_ptr<float>(),
                              rstd.data_ptr<float>(), ptr(k.weight), ptr(k.bias), add ? add->t.data_ptr() : nullptr,
                              add ? add->ld : 0, dx.data_ptr(), k.s.C, static_cast<float*>(ptr(dw)),
                              static_cast<float*>(ptr(db)), ptr(ws), need, stream_of(h)));
    return {dx, dw, db};
}

// ---------------------------------------------------------------- distillation

void check_temperature(double t) {  // as the kernels have it: its inverse and its square are finite
    const float f = static_cast<float>(t);
    if (!(f >= 1e-18f && f <= 1e18f)) value_error("the temperature lies between 1e-18 and 1e18 (got " + std::to_string(t) + ")");
}

std::tuple<Tensor, Tensor, Tensor> top_logits(const Tensor& logits, std::int64_t k, double temperature) {
    const std::uint32_t code = dtype_of(logits, "logits");
    const Rows rows(logits, "logits");
    const std::int64_t n = logits.size(0), C = logits.size(1);
    if (C > 0x7FFFFFFFll) value_error("rows of " + std::to_string(C) + " logits are too long");
    if (k < 1 || k > std::min<std::int64_t>(C, 64))
        value_error("k must be between 1 and the " + std::to_string(C) + " classes, and at most 64 (got " + std::to_string(k) + ")");
    check_temperature(temperature);
    on_current_device(logits);
    const Tensor values = empty({n, k}, logits.options()), ids = empty({n, k}, logits.options().dtype(at::kInt));
    const Tensor rest = empty({n}, logits.options().dtype(at::kFloat));
    check(tcc_top_logits(rows.t.data_ptr(), rows.ld, code, n, static_cast<std::uint32_t>(C), static_cast<std::uint32_t>(k),
                         static_cast<float>(temperature), values.data_ptr(), k, ids.data_ptr<std::int32_t>(), k,
                         rest.data_ptr<float>(), stream_of(logits)));
    return {values, ids, rest};
}

// A distillation's tensors as the C-ABI takes them.
struct Distill {
    tcc_distill_shape s{};
    Rows z;
    std::optional<Rows> values, ids;
    MaybeTensor rest, weight;  // kept until the launch

    Distill(const Tensor& logits, const Tensor& v, const Tensor& i, const MaybeTensor& r, const MaybeTensor& w,
            double temperature, std::uint32_t reduction)
        : z(((void)dtype_of(logits, "logits"), logits), "logits") {
        s.dtype = dtype_of(logits, "logits");
        s.valueDtype = dtype_of(v, "values");
        s.idBytes = index_bytes(i, "ids");
        s.reduction = reduction;
        const std::int64_t n = logits.size(0), C = logits.size(1);
        if (v.dim() != 2 || v.size(0) != n || v.size(1) < 1 || v.size(1) > 64 || i.sizes() != v.sizes())
            value_error("values " + shape_of(v) + " and ids " + shape_of(i) + " must be 1 to 64 entries for each of the " +
                        std::to_string(n) + " rows");
        if (C > 0x7FFFFFFFll) value_error("rows of " + std::to_string(C) + " logits are too long");
        check_temperature(temperature);
        values.emplace(v, "values");
        ids.emplace(i, "ids");
        for (const auto& [t, name, to] : {std::tuple{&r, "rest", &rest}, std::tuple{&w, "weight", &weight}}) {
            if (!*t) continue;
            if (!(*t)->is_cuda() || (*t)->scalar_type() != at::kFloat)
                type_error(std::string(name) + " must be a float32 device tensor (got " + place_of(**t) + ")");
            if ((*t)->dim() != 1 || (*t)->size(0) != n)
                value_error(std::string(name) + " must hold a value for each of the " + std::to_string(n) + " rows (got " +
                            shape_of(**t) + ")");
            on_current_device(**t);
            *to = (*t)->contiguous();
        }
        on_current_device(logits);
        on_current_device(v);
        on_current_device(i);
        s.n = static_cast<std::uint64_t>(n);
        s.C = static_cast<std::uint32_t>(C);
        s.K = static_cast<std::uint32_t>(v.size(1));
        s.temperature = static_cast<float>(temperature);
    }
};

std::tuple<Tensor, Tensor, MaybeTensor> distill_loss(const Tensor& logits, const Tensor& values, const Tensor& ids,
                                                     const MaybeTensor& rest, double temperature, const MaybeTensor& weight,
                                                     std::uint32_t reduction, const MaybeTensor& deviceError) {
    const Distill k(logits, values, ids, rest, weight, temperature, reduction);
    std::uint32_t* err = error_word(deviceError);
    const auto f32 = logits.options().dtype(at::kFloat);
    const std::int64_t n = logits.size(0);
    const Tensor loss = reduction == TCC_REDUCE_NONE ? empty({n}, f32) : empty({}, f32);
    const Tensor stats = empty({n, 4}, f32);
    MaybeTensor total, ws;
    if (weight && reduction == TCC_REDUCE_MEAN) total = empty({}, f32);
    const std::size_t need = tcc_distill_loss_workspace_bytes(&k.s);
    if (need > 0) ws = workspace(need, logits);
    check(tcc_distill_loss(&k.s, k.z.t.data_ptr(), k.z.ld, k.values->t.data_ptr(), k.values->ld, k.ids->t.data_ptr(),
                           k.ids->ld, static_cast<const float*>(ptr(k.rest)), static_cast<const float*>(ptr(k.weight)),
                           loss.data_ptr<float>(), static_cast<float*>(ptr(total)), stats.data_ptr<float>(), err, ptr(ws),
                           need, stream_of(logits)));
    if (deviceError) written(*deviceError);
    return {loss, stats, total};
}

Tensor distill_grad(const Tensor& dLoss, const Tensor& logits, const Tensor& values, const Tensor& ids, const Tensor& stats,
                    const MaybeTensor& rest, double temperature, const MaybeTensor& weight, const MaybeTensor& total,
                    std::uint32_t reduction) {
    const Distill k(logits, values, ids, rest, weight, temperature, reduction);
    const std::int64_t n = logits.size(0);
    const bool each = reduction == TCC_REDUCE_NONE;
    const auto is_float = [](const Tensor& t, const char* name) {
        if (!t.is_cuda() || t.scalar_type() != at::kFloat)
            type_error(std::string(name) + " must be a float32 device tensor (got " + place_of(t) + ")");
        on_current_device(t);
    };
    is_float(dLoss, "d_loss");
    is_float(stats, "stats");
    if (each ? dLoss.dim() != 1 || dLoss.size(0) != n : dLoss.numel() != 1)
        value_error("d_loss " + shape_of(dLoss) + " must be of the loss's shape");
    if (stats.dim() != 2 || stats.size(0) != n || stats.size(1) != 4) value_error("stats must be those of the loss");
    if (weight && reduction == TCC_REDUCE_MEAN) {
        if (!total) value_error("a mean with weights needs their total");
        is_float(*total, "total");
        if (total->numel() != 1) value_error("total must be that of the loss");
    }
    const Tensor d = dLoss.contiguous();
    Tensor st = stats.contiguous();
    if ((reinterpret_cast<std::uintptr_t>(st.data_ptr()) & 15) != 0) st = st.clone();
    const Tensor dz = empty(logits.sizes(), logits.options());
    const float* sum = weight && reduction == TCC_REDUCE_MEAN ? total->data_ptr<float>() : nullptr;
    check(tcc_distill_grad(&k.s, d.data_ptr<float>(), k.z.t.data_ptr(), k.z.ld, k.values->t.data_ptr(), k.values->ld,
                           k.ids->t.data_ptr(), k.ids->ld, static_cast<const float*>(ptr(k.rest)),
                           static_cast<const float*>(ptr(k.weight)), sum, st.data_ptr<float>(), dz.data_ptr(), k.s.C,
                           stream_of(logits)));
    return dz;
}

// ---------------------------------------------------------------- lists

using TensorList = std::vector<Tensor>;
using Described = std::vector<tcc_tensor>;

// The elements of t in the order of its dimensions `order`, as rows.
bool collapse(const Tensor& t, const std::vector<std::int64_t>& order, tcc_tensor& to) {
    std::uint64_t cols = 1, rows = 1, ld = 0;
    std::size_t d = order.size();
    for (; d > 0; --d) {
        const std::int64_t n = t.size(order[d - 1]);
        if (n == 1) continue;
        if (static_cast<std::uint64_t>(t.stride(order[d - 1])) != cols) break;
        cols *= static_cast<std::uint64_t>(n);
    }
    for (; d > 0; --d) {
        const std::int64_t n = t.size(order[d - 1]);
        if (n == 1) continue;
        const std::uint64_t stride = static_cast<std::uint64_t>(t.stride(order[d - 1]));
        if (ld == 0) {
            ld = stride;
            if (ld < cols) return false;
        } else if (stride != rows * ld) {
            return false;
        }
        rows *= static_cast<std::uint64_t>(n);
    }
    to.rows = rows;
    to.cols = cols;
    to.ld = ld == 0 ? cols : ld;
    return true;
}

// The i-th tensors of all lists: the same elements in the same order, the
// first one's order in memory.
void describe_strided(const std::vector<const TensorList*>& lists, const std::vector<const char*>& names, std::size_t i,
                      std::vector<Described>& to) {
    const Tensor& first = (*lists[0])[i];
    std::vector<std::int64_t> order(static_cast<std::size_t>(first.dim()));
    std::iota(order.begin(), order.end(), 0);
    std::stable_sort(order.begin(), order.end(),
                     [&](std::int64_t a, std::int64_t b) { return first.stride(a) > first.stride(b); });
    std::uint64_t rows = 1, cols = 0;
    for (std::size_t l = 0; l < lists.size(); ++l) {
        const Tensor& t = (*lists[l])[i];
        tcc_tensor& x = to[l][i];
        if (!collapse(t, order, x))
            value_error(std::string(names[l]) + " of shape " + shape_of(t) +
                        " is not rows at one distance in the order of " + names[0]);
        if (x.rows > 1) {
            if (rows > 1 && (rows != x.rows || cols != x.cols))
                value_error(std::string(names[l]) + " is split into rows in another way than the other tensors");
            rows = x.rows;
            cols = x.cols;
        }
    }
    if (rows == 1) return;
    for (std::size_t l = 0; l < lists.size(); ++l) {
        tcc_tensor& x = to[l][i];
        if (x.rows == 1) {
            x.rows = rows;
            x.cols = x.ld = cols;
        }
    }
}

std::vector<Described> describe(const std::vector<const TensorList*>& lists, const std::vector<const char*>& names) {
    const std::size_t count = lists[0]->size();
    for (std::size_t l = 1; l < lists.size(); ++l)
        if (lists[l]->size() != count)
            value_error(std::to_string(lists[l]->size()) + " " + names[l] + " for " + std::to_string(count) + " " + names[0]);
    std::vector<Described> to(lists.size(), Described(count));
    for (std::size_t i = 0; i < count; ++i) {
        bool plain = true;
        for (std::size_t l = 0; l < lists.size(); ++l) {
            const Tensor& t = (*lists[l])[i];
            tcc_tensor& x = to[l][i];
            x.dtype = dtype_of(t, names[l]);
            on_current_device(t);
            if (l > 0 && t.sizes() != (*lists[0])[i].sizes())
                value_error(std::string(names[l]) + " of shape " + shape_of(t) + " for " + names[0] + " of shape " +
                            shape_of((*lists[0])[i]));
            plain = plain && t.is_contiguous();
            x.data = t.data_ptr();
            x.rows = 1;
            x.cols = x.ld = static_cast<std::uint64_t>(t.numel());
        }
        if (!plain && to[0][i].cols > 0) describe_strided(lists, names, i, to);
    }
    return to;
}

// A place for a norm and the workspace, on the current device.
struct NormPlace {
    Tensor norm, ws;
    std::size_t bytes = tcc_grad_norm_workspace_bytes();
    explicit NormPlace(bool wantNorm) {
        const auto options = at::TensorOptions().device(at::kCUDA, c10::hip::current_device());
        if (wantNorm) norm = empty({}, options.dtype(at::kFloat));
        ws = empty({static_cast<std::int64_t>(bytes)}, options.dtype(at::kByte));
    }
    float* at() const { return norm.defined() ? norm.data_ptr<float>() : nullptr; }
};

Tensor grad_norm(const TensorList& grads) {
    const auto lists = describe({&grads}, {"grads"});
    const NormPlace p(true);
    check(tcc_grad_norm(lists[0].data(), static_cast<std::uint32_t>(grads.size()), p.at(), p.ws.data_ptr(), p.bytes,
                        stream_of(p.ws)));
    return p.norm;
}

Tensor clip_grad_norm(const TensorList& grads, double maxNorm, const std::optional<TensorList>& out) {
    if (!(maxNorm >= 0)) value_error("max_norm is not negative (got " + std::to_string(maxNorm) + ")");
    const TensorList& to = out ? *out : grads;
    if (to.size() == grads.size())
        for (std::size_t i = 0; i < to.size(); ++i)
            if (to[i].scalar_type() != grads[i].scalar_type()) value_error("out must be of the gradients' types");
    const auto lists = describe({&grads, &to}, {"grads", "out"});
    const NormPlace p(true);
    check(tcc_clip_grad_norm(lists[0].data(), lists[1].data(), static_cast<std::uint32_t>(grads.size()),
                             static_cast<float>(maxNorm), p.at(), p.ws.data_ptr(), p.bytes, stream_of(p.ws)));
    written(to);
    return p.norm;
}

MaybeTensor adam_step(const TensorList& params, const TensorList& grads, const TensorList& expAvg,
                      const TensorList& expAvgSq, const Tensor& step, double lr, double beta1, double beta2, double eps,
                      double weightDecay, bool decoupled, std::optional<double> maxNorm) {
    if (!step.is_cuda() || step.scalar_type() != at::kLong || step.numel() != 1)
        type_error("step must be an int64 device scalar");
    if (maxNorm && !(*maxNorm >= 0)) value_error("max_norm is not negative (got " + std::to_string(*maxNorm) + ")");
    if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0))
        value_error("betas must be in [0, 1) and eps not negative");
    for (const TensorList* l : {&expAvg, &expAvgSq})
        for (const Tensor& t : *l)
            if (t.scalar_type() != at::kFloat) type_error("moments must be float32 (got " + place_of(t) + ")");
    on_current_device(step);
    const auto lists = describe({&params, &grads, &expAvg, &expAvgSq}, {"params", "grads", "exp_avg", "exp_avg_sq"});
    const NormPlace p(maxNorm.has_value());
    const tcc_adam a{lr, beta1, beta2, eps, weightDecay, maxNorm.value_or(-1.0), decoupled};
    check(tcc_adam_step(lists[0].data(), lists[1].data(), lists[2].data(), lists[3].data(),
                        static_cast<std::uint32_t>(params.size()), &a, step.data_ptr<std::int64_t>(), p.at(),
                        p.ws.data_ptr(), p.bytes, stream_of(p.ws)));
    for (const TensorList* l : {&params, &expAvg, &expAvgSq}) written(*l);
    written(step);
    return maxNorm ? MaybeTensor(p.norm) : std::nullopt;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "The operators of tcc_amd.training over libtcc_swtcf.so.";
    m.def("embedding_lookup", &embedding_lookup);
    m.def("embedding_grad", &embedding_grad);
    m.def("group_norm", &group_norm);
    m.def("group_norm_grad", &group_norm_grad);
    m.def("held_by_default_stream", &held_by_default_stream);
    m.def("layer_norm", &layer_norm);
    m.def("layer_norm_grad", &layer_norm_grad);
    m.def("top_logits", &top_logits);
    m.def("distill_loss", &distill_loss);
    m.def("distill_grad", &distill_grad);
    m.def("grad_norm", &grad_norm);
    m.def("clip_grad_norm", &clip_grad_norm);
    m.def("adam_step", &adam_step);
}
