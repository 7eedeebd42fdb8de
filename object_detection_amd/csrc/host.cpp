// The torch side of layers.py and grads.py: checks of tensors, outputs, workspaces, streams and the autograd nodes, over the C
// ABI of libdethead.  These entries are called per layer and per step with few or very many small tensors, where what the Python
// interpreter needs for the same work is longer than the kernels (a linear call 11 us, a backward 70 us, a list of 111 gradients
// 85 us); everything that computes is in libdethead.
#include <torch/extension.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/autocast_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/utils.h>

#include "../../include/dethead.h"

#include <algorithm>
#include <array>
#include <memory>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

namespace py = pybind11;

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

[[noreturn]] void fail(const std::string& what) { throw std::runtime_error(what); }

std::string shape(const Tensor& t)
{
    std::string s = "(";
    for (int64_t k = 0; k < t.dim(); ++k) s += (k ? ", " : "") + std::to_string(t.size(k));
    return s + ")";
}

void checked(int rc, const char* entry)
{
    static const char* const text[] = {"", "invalid argument (shape / null pointer / unsupported size)", "HIP kernel launch failed",
                                       "pointer not aligned to its type", "workspace too small"};
    if (rc == 0) return;
    fail(std::string(entry) + " failed: " + (rc >= -4 && rc < 0 ? text[-rc] : std::to_string(rc)));
}

int code_of(at::ScalarType t)
{
    switch (t) {
    case at::kFloat: return DH_F32;
    case at::kHalf: return DH_F16;
    case at::kBFloat16: return DH_BF16;
    default: return -1;
    }
}

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* at_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor scratch(size_t bytes, const Tensor& like)
{
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// ------------------------------------------------------------------------------------------------ products

struct Item {
    Tensor x, w, bias, res;
    std::array<Tensor*, 4> all() { return {&x, &w, &bias, &res}; }
};

// The kernels read memory: a view whose sign is kept beside it (the imaginary part of a conjugate) is written out first.
Tensor in_memory(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// Kernels carry no tangents: a dual tensor is refused, its derivative not taken for zero.  Asked of the tensors only where a level of
// forward mode is open (a view's answer costs 15 ns).
bool dual_level()
{
    return c10::AutogradState::get_tls_state().get_fw_grad_mode() && torch::autograd::ForwardADLevel::try_get_by_idx(0);
}
void refuse_dual(const char* where, const Tensor& t)
{
    if (t._fw_grad(0).defined()) fail(std::string(where) + ": forward-mode derivatives are not offered");
}

// One supported type on one ROCm device; under autocast its type.
void check_tensors(const char* where, Item& it)
{
    if (!it.x.is_cuda())
        fail(std::string(where) + ": x is on " + it.x.device().str() + ": object_detection_amd only runs on ROCm devices (no CPU fallback)");
    for (Tensor* t : it.all())
        if (t->defined() && t->is_neg()) *t = t->resolve_neg();
    if (dual_level())
        for (Tensor* t : it.all())
            if (t->defined()) refuse_dual(where, *t);
    for (Tensor* t : it.all())
        if (t->defined() && t->device() != it.x.device())
            fail(std::string(where) + ": tensors on " + t->device().str() + " and " + it.x.device().str());
    if (at::autocast::is_autocast_enabled(at::kCUDA)) {
        const at::ScalarType to = at::autocast::get_autocast_dtype(at::kCUDA);
        for (Tensor* t : it.all())
            if (t->defined() && t->is_floating_point() && t->scalar_type() != at::kDouble && t->scalar_type() != to) *t = t->to(to);
    }
    const at::ScalarType type = it.x.scalar_type();
    for (Tensor* t : it.all())
        if (t->defined() && (t->scalar_type() != type || t->layout() != at::kStrided || code_of(type) < 0))
            fail(std::string(where) + ": x, weight, bias and residual must be dense tensors of one type, fp32, fp16 or bf16; got " +
                 c10::toString(t->scalar_type()) + " and " + c10::toString(type));
}

void check_weight(const char* where, const Item& it, int64_t inputs, bool may_be_4d)
{
    const Tensor& w = it.w;
    const bool four = may_be_4d && w.dim() == 4 && w.size(2) == 1 && w.size(3) == 1;
    if (!(w.dim() == 2 || four) || w.size(1) != inputs)
        fail(std::string(where) + ": weight must be (outputs, " + std::to_string(inputs) + ")" + (may_be_4d ? " or (outputs, inputs, 1, 1)" : "") +
             ", got " + shape(w));
    if (it.bias.defined() && (it.bias.dim() != 1 || it.bias.size(0) != w.size(0)))
        fail(std::string(where) + ": bias must be (" + std::to_string(w.size(0)) + ",), got " + shape(it.bias));
}

// (M, C) with the last axis dense and one stride between rows; a copy only where the strides do not allow it, or rows overlap.
Tensor as_rows(const Tensor& t)
{
    if (t.is_contiguous() || ((t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)))) return t;
    return t.contiguous();
}

// (B, C, ny, nx) with dense planes; images may be apart (a slice of a wider tensor's channels is read where it is).
Tensor as_planes(const Tensor& t)
{
    if (t.is_contiguous()) return t;
    const int64_t c = t.size(1), h = t.size(2), v = t.size(3);
    if (t.stride(3) == 1 && t.stride(2) == v && t.stride(1) == h * v && t.stride(0) >= c * h * v) return t;
    return t.contiguous();
}

int as_int(int64_t v)
{
    if (v < 0 || v > DH_MAX_EXTENT) fail("a dimension of a product exceeds " + std::to_string(DH_MAX_EXTENT));
    return (int)v;
}

dh_product forward_product(bool rows, const Item& it, const Tensor& out, const Tensor& z)
{
    dh_product p{};
    const int64_t n = it.w.size(0), k = it.w.size(1);
    p.bias = at_or_null(it.bias);
    p.residual = at_or_null(it.res);
    p.out = out.data_ptr();
    p.z = at_or_null(z);
    p.a_by_reduction = 1;
    p.R = as_int(k);
    if (rows) {
        const int64_t m = it.x.size(0);
        p.a = it.x.data_ptr();
        p.b = it.w.data_ptr();
        p.lda = m > 1 ? it.x.stride(0) : k;
        p.ldb = k;
        p.ldo = n;
        p.ldr = it.res.defined() && m > 1 ? it.res.stride(0) : n;
        p.I = as_int(m);
        p.J = as_int(n);
        p.batch = 1;
        p.b_by_reduction = 1;
    } else {
        const int64_t cells = it.x.size(2) * it.x.size(3);
        p.a = it.w.data_ptr();
        p.b = it.x.data_ptr();
        p.lda = k;
        p.ldb = p.ldo = p.ldr = cells;
        p.b_batch = it.x.stride(0);
        p.o_batch = n * cells;
        p.res_batch = it.res.defined() ? it.res.stride(0) : 0;
        p.I = as_int(n);
        p.J = as_int(cells);
        p.batch = as_int(it.x.size(0));
        p.bias_on_i = 1;
    }
    return p;
}

dh_product input_gradient(bool rows, const Tensor& dz, const Tensor& w, const Tensor& out)
{
    dh_product p{};
    const int64_t n = w.size(0), k = w.size(1);
    p.out = out.data_ptr();
    p.R = as_int(n);
    if (rows) {
        p.a = dz.data_ptr();
        p.b = w.data_ptr();
        p.lda = n;
        p.ldb = p.ldo = k;
        p.I = as_int(dz.size(0));
        p.J = as_int(k);
        p.batch = 1;
        p.a_by_reduction = 1;
    } else {
        const int64_t cells = dz.size(2) * dz.size(3);
        p.a = w.data_ptr();
        p.b = dz.data_ptr();
        p.lda = k;
        p.ldb = p.ldo = cells;
        p.b_batch = n * cells;
        p.o_batch = k * cells;
        p.I = as_int(k);
        p.J = as_int(cells);
        p.batch = as_int(dz.size(0));
    }
    return p;
}

// dbias: the bias gradient beside the weight's, from the same read of dz.
dh_product weight_gradient(bool rows, const Tensor& dz, const Tensor& x, const Tensor& out, const Tensor& dbias)
{
    dh_product p{};
    const int64_t n = dz.size(1), k = x.size(1);
    p.a = dz.data_ptr();
    p.b = x.data_ptr();
    p.out = out.data_ptr();
    p.a_sum = at_or_null(dbias);
    p.ldo = k;
    p.I = as_int(n);
    p.J = as_int(k);
    if (rows) {
        p.lda = n;
        p.ldb = x.size(0) > 1 ? x.stride(0) : k;
        p.R = as_int(x.size(0));
        p.batch = 1;
    } else {
        const int64_t cells = x.size(2) * x.size(3);
        p.lda = p.ldb = cells;
        p.a_batch = n * cells;
        p.b_batch = x.stride(0);
        p.R = as_int(cells);
        p.batch = as_int(x.size(0));
        p.a_by_reduction = p.b_by_reduction = p.reduce_batch = 1;
    }
    return p;
}

void run(const std::vector<dh_product>& products, int act, const Tensor& like)
{
    if (products.empty()) return;
    const c10::DeviceGuard guard(like.device());
    const int code = code_of(like.scalar_type()), n = (int)products.size();
    const size_t need = dh_products_workspace(products.data(), n, code);
    const Tensor ws = scratch(need, like);
    checked(dh_products(products.data(), n, code, act, at_or_null(ws), need, stream_of(like)), "dh_products");
}

// The outputs of all items from one launch; `kept` receives what a backward needs of each: x as it was read, the weight, z.
variable_list forward_all(bool rows, int act, std::vector<Item>& items, variable_list* kept)
{
    variable_list outs;
    std::vector<dh_product> products;
    for (Item& it : items) {
        it.w = it.w.contiguous();
        if (it.bias.defined()) it.bias = it.bias.contiguous();
        it.x = rows ? as_rows(it.x) : as_planes(it.x);
        if (it.res.defined()) it.res = rows ? as_rows(it.res) : as_planes(it.res);
        const int64_t n = it.w.size(0);
        const Tensor out = rows ? at::empty({it.x.size(0), n}, it.x.options())
                                : at::empty({it.x.size(0), n, it.x.size(2), it.x.size(3)}, it.x.options());
        const Tensor z = kept && act ? at::empty_like(out) : Tensor();
        products.push_back(forward_product(rows, it, out, z));
        outs.push_back(out);
        if (kept) kept->insert(kept->end(), {it.x, it.w, z});
    }
    run(products, act, items[0].x);
    return outs;
}

// dy times the activation's derivative, and its sum for the bias (undefined where not wanted).
std::tuple<Tensor, Tensor> slope(bool rows, const Tensor& dy, const Tensor& z, int act, bool want_bias)
{
    const Tensor dz = z.defined() ? at::empty_like(dy) : dy;
    if (!z.defined() && !want_bias) return {dz, Tensor()};
    const c10::DeviceGuard guard(dy.device());
    const int64_t outer = dy.size(0), n = dy.size(1), inner = rows ? 1 : dy.size(2) * dy.size(3);
    const Tensor dbias = want_bias ? at::empty({n}, dy.options()) : Tensor();
    const size_t need = want_bias ? dh_product_slope_workspace(n) : 0;
    const Tensor ws = scratch(need, dy);
    checked(dh_product_slope(dy.data_ptr(), at_or_null(z), dz.data_ptr(), at_or_null(dbias), outer, n, inner, act, code_of(dy.scalar_type()),
                             at_or_null(ws), need, stream_of(dy)),
            "dh_product_slope");
    return {dz, dbias};
}

// Under create_graph the gradients leave through this node, whose edges lead to all that they depend on: a second derivative is
// refused, not taken for zero.
struct Last : torch::autograd::Node {
    variable_list apply(variable_list&&) override
    {
        fail("object_detection_amd.layers: a second derivative of a product is not offered");
    }
};

struct Products : torch::autograd::Function<Products> {
    // ts: x, weight, bias, residual of each product; what is absent has no edge in the graph
    template <typename... Ts>
    static variable_list forward(AutogradContext* ctx, bool rows, int64_t act, const Ts&... ts)
    {
        const std::array<Tensor, sizeof...(Ts)> t{ts.value_or(Tensor())...};
        int64_t present = 0;
        for (size_t k = 0; k < t.size(); ++k) present |= (int64_t)t[k].defined() << k;
        ctx->saved_data["present"] = present;
        std::vector<Item> items;
        for (size_t k = 0; k + 3 < t.size() && t[k].defined(); k += 4) items.push_back({t[k], t[k + 1], t[k + 2], t[k + 3]});
        variable_list kept;
        variable_list outs = forward_all(rows, (int)act, items, &kept);
        ctx->save_for_backward(std::move(kept));
        ctx->saved_data["how"] = (int64_t)(act * 2 + rows) * 32 + (int64_t)t.size();
        ctx->set_materialize_grads(false);
        return outs;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const int64_t how = ctx->saved_data["how"].toInt();
        const int arguments = (int)(how % 32), act = (int)(how / 64);
        const bool rows = how / 32 % 2, create_graph = at::GradMode::is_enabled();
        const int64_t present = ctx->saved_data["present"].toInt();
        const auto place_of = [&](size_t k) { return (size_t)__builtin_popcountll(present & ((1ll << k) - 1)); };     // among this node's edges
        const auto wanted = [&](size_t k) { return (present >> k & 1) && ctx->needs_input_grad(place_of(k)); };
        const at::AutoGradMode off(false);
        const variable_list saved = ctx->get_saved_variables();
        variable_list result(2 + arguments);
        std::vector<dh_product> inputs, weights;
        variable_list alive;
        for (size_t k = 0; k < grads.size(); ++k) {
            if (!grads[k].defined()) continue;
            const Tensor &x = saved[3 * k], &w = saved[3 * k + 1], &z = saved[3 * k + 2];
            const bool want_x = wanted(4 * k), want_w = wanted(4 * k + 1), want_b = wanted(4 * k + 2), want_r = wanted(4 * k + 3);
            const Tensor dy = in_memory(grads[k]).contiguous();
            Tensor* to = &result[2 + 4 * k];
            if (want_r) to[3] = dy;
            if (!want_x && !want_w && !want_b) continue;
            // without an activation dy is dz: the weight's gradient reads it anyway and sums it for the bias
            const bool beside = !z.defined() && want_w && x.size(1) > 0;
            Tensor dz = dy;
            if (beside) {
                if (want_b) to[2] = at::empty({dy.size(1)}, dy.options());
            } else {
                std::tie(dz, to[2]) = slope(rows, dy, z, act, want_b);
            }
            if (want_x) {
                to[0] = at::empty(x.sizes(), x.options());
                inputs.push_back(input_gradient(rows, dz, w, to[0]));
            }
            if (want_w) {
                to[1] = at::empty_like(w);
                weights.push_back(weight_gradient(rows, dz, x, to[1], beside ? to[2] : Tensor()));
            }
            alive.push_back(dz);
        }
        run(inputs, 0, saved[0]);
        run(weights, 0, saved[0]);
        if (create_graph) {
            // the inputs' edges are this node's own: what was saved may be a copy that was made without a graph
            const auto node = torch::autograd::get_current_node();
            for (size_t k = 0; k < grads.size(); ++k) {
                if (!grads[k].defined()) continue;
                torch::autograd::edge_list edges{torch::autograd::impl::gradient_edge(grads[k])};
                for (size_t e = 4 * k; e < 4 * k + 3; ++e)
                    if (present >> e & 1) edges.push_back(node->next_edge(place_of(e)));
                if (std::none_of(edges.begin(), edges.end(), [](const torch::autograd::Edge& e) { return e.is_valid(); })) continue;
                const std::shared_ptr<Last> last(new Last, torch::autograd::deleteNode);
                last->set_next_edges(std::move(edges));
                for (int e = 0; e < 3; ++e)
                    if (result[2 + 4 * k + e].defined()) torch::autograd::set_history(result[2 + 4 * k + e], last);
                if (result[2 + 4 * k + 3].defined()) result[2 + 4 * k + 3] = grads[k];      // the residual's: dy, with its own graph
            }
        }
        return result;
    }
};

variable_list products(bool rows, int act, std::vector<Item> items)
{
    bool wants = false;
    if (at::GradMode::is_enabled())
        for (Item& it : items)
            for (const Tensor* t : it.all()) wants |= t->defined() && t->requires_grad();
    if (!wants) return forward_all(rows, act, items, nullptr);
    const auto apply = [&](auto t) {
        for (size_t k = 0; k < items.size(); ++k)
            for (int e = 0; e < 4; ++e)
                if (items[k].all()[e]->defined()) t[4 * k + e] = *items[k].all()[e];
        return std::apply([&](const auto&... ts) { return Products::apply(rows, (int64_t)act, ts...); }, t);
    };
    if (items.size() == 1) return apply(std::array<std::optional<Tensor>, 4>());
    return apply(std::array<std::optional<Tensor>, 4 * DH_MAX_PRODUCTS>());
}

Item item(const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias, const std::optional<Tensor>& res)
{
    return {x, w, bias.value_or(Tensor()), res.value_or(Tensor())};
}

Tensor linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, int act, const std::optional<Tensor>& residual)
{
    Item it = item(x, weight, bias, residual);
    check_tensors("linear", it);
    if (it.x.dim() < 1) fail("linear: x must be (..., C), got a scalar");
    check_weight("linear", it, it.x.size(-1), false);
    std::vector<int64_t> to(it.x.sizes().begin(), it.x.sizes().end());
    to.back() = it.w.size(0);
    if (it.res.defined() && it.res.sizes() != at::IntArrayRef(to)) fail("linear: residual must have the output's shape, got " + shape(it.res));
    if (it.x.dim() == 2) return products(true, act, {it})[0];
    int64_t rows = 1;
    for (size_t k = 0; k + 1 < to.size(); ++k) rows *= to[k];
    it.x = it.x.reshape({rows, it.x.size(-1)});
    if (it.res.defined()) it.res = it.res.reshape({rows, to.back()});
    return products(true, act, {it})[0].view(to);
}

Tensor pointwise_conv(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, int act, const std::optional<Tensor>& residual)
{
    Item it = item(x, weight, bias, residual);
    check_tensors("pointwise_conv", it);
    if (it.x.dim() != 4) fail("pointwise_conv: x must be (B, C, ny, nx), got " + shape(it.x));
    check_weight("pointwise_conv", it, it.x.size(1), true);
    const int64_t b = it.x.size(0), c = it.x.size(1), h = it.x.size(2), v = it.x.size(3), n = it.w.size(0);
    if (it.res.defined() && it.res.sizes() != at::IntArrayRef({b, n, h, v}))
        fail("pointwise_conv: residual must have the output's shape, got " + shape(it.res));
    if (it.x.is_contiguous() || !it.x.is_contiguous(at::MemoryFormat::ChannelsLast)) return products(false, act, {it})[0];
    it.x = it.x.permute({0, 2, 3, 1}).reshape({b * h * v, c});
    if (it.res.defined()) it.res = it.res.permute({0, 2, 3, 1}).reshape({b * h * v, n});
    return products(true, act, {it})[0].view({b, h, v, n}).permute({0, 3, 1, 2});
}

variable_list head_convs(const std::vector<Tensor>& xs, const std::vector<Tensor>& weights, const std::vector<std::optional<Tensor>>& biases)
{
    if (xs.empty() || xs.size() > DH_MAX_PRODUCTS || weights.size() != xs.size() || biases.size() != xs.size())
        fail("head_convs: 1 to " + std::to_string(DH_MAX_PRODUCTS) + " levels with a weight and a bias each, got " + std::to_string(xs.size()) + ", " +
             std::to_string(weights.size()) + ", " + std::to_string(biases.size()));
    std::vector<Item> items;
    for (size_t l = 0; l < xs.size(); ++l) {
        Item it = item(xs[l], weights[l], biases[l], std::nullopt);
        check_tensors("head_convs", it);
        if (it.x.dim() != 4) fail("head_convs: level " + std::to_string(l) + " must be (B, C, ny, nx), got " + shape(it.x));
        check_weight("head_convs", it, it.x.size(1), true);
        if (l && (it.x.scalar_type() != items[0].x.scalar_type() || it.x.device() != items[0].x.device()))
            fail("head_convs: all levels must have one type and device");
        items.push_back(std::move(it));
    }
    return products(false, 0, std::move(items));
}

// ------------------------------------------------------------------------------------------------ gradients

// Gradients of one type as the C entries take them.
struct List {
    at::ScalarType type;
    std::vector<const void*> at;
    std::vector<int64_t> n;
    std::vector<size_t> index;              // in the caller's list
    int64_t parts = 0;
};

// A tensor as the kernels read it: its elements in one piece, in any order of the axes.
bool dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

std::vector<List> listed(const char* where, const variable_list& grads, variable_list* read)
{
    std::vector<List> lists;
    const bool dual = dual_level();
    for (size_t k = 0; k < grads.size(); ++k) {
        const Tensor& g = grads[k];
        if (!g.is_cuda())
            fail(std::string(where) + ": a gradient is on " + g.device().str() + ": object_detection_amd only runs on ROCm devices (no CPU fallback)");
        if (g.layout() != at::kStrided) fail(std::string(where) + ": gradients must be dense tensors");
        if (dual) refuse_dual(where, g);
        if (g.device() != grads[0].device()) fail(std::string(where) + ": gradients on " + grads[0].device().str() + " and " + g.device().str());
        const at::ScalarType type = g.scalar_type();
        if (code_of(type) < 0) fail(std::string(where) + ": gradients must be fp32, fp16 or bf16, got " + c10::toString(type));
        auto it = std::find_if(lists.begin(), lists.end(), [&](const List& l) { return l.type == type; });
        if (it == lists.end()) {
            lists.push_back({type, {}, {}, {}, 0});
            it = lists.end() - 1;
        }
        const Tensor r = in_memory(dense(g) ? g : g.contiguous());
        it->at.push_back(r.data_ptr());
        it->n.push_back(r.numel());
        it->index.push_back(k);
        read->push_back(r);
    }
    for (List& l : lists) l.parts = dh_grad_parts(l.n.data(), (int)l.n.size());
    return lists;
}

// The partial sums of every list, one after the other; `reduce` (a Python callable on the one joined power) over several processes.
Tensor powers(const std::vector<List>& lists, const Tensor& like, int norm, const py::object& reduce)
{
    int64_t parts = 0;
    for (const List& l : lists) parts += l.parts;
    Tensor partial = at::empty({parts}, like.options().dtype(at::kDouble));
    double* to = parts ? partial.data_ptr<double>() : nullptr;
    for (const List& l : lists) {
        checked(dh_grad_power(l.at.data(), l.n.data(), (int)l.n.size(), code_of(l.type), norm, to, l.parts, stream_of(like)), "dh_grad_power");
        to += l.parts;
    }
    if (reduce.is_none()) return partial;
    Tensor power = at::empty({1}, partial.options());
    checked(dh_grad_norm((const double*)at_or_null(partial), parts, norm, nullptr, power.data_ptr<double>(), nullptr, stream_of(like)), "dh_grad_norm");
    return reduce(power).cast<Tensor>();
}

// The loss scale as one device float; undefined for 1.
Tensor scale_on(const char* where, const py::object& scale, const Tensor& like)
{
    if (scale.is_none()) return {};
    if (THPVariable_Check(scale.ptr())) {
        const Tensor t = scale.cast<Tensor>();
        if (t.numel() != 1) fail(std::string(where) + ": scale must be one number, got shape " + shape(t));
        if (t.is_cpu()) return at::full({}, t.detach().item<double>(), like.options().dtype(at::kFloat));      // no copy to wait for
        return t.detach().to(like.device(), at::kFloat);
    }
    const double v = scale.cast<double>();
    return v == 1.0 ? Tensor() : at::full({}, v, like.options().dtype(at::kFloat));
}

Tensor total_norm(const variable_list& grads, int norm, const py::object& scale, const py::object& reduce)
{
    const at::NoGradGuard off;
    variable_list read;
    const std::vector<List> lists = listed("total_grad_norm", grads, &read);
    const c10::DeviceGuard guard(grads[0].device());
    const Tensor factor = scale_on("total_grad_norm", scale, grads[0]);
    const Tensor partial = powers(lists, grads[0], norm, reduce);
    const Tensor out = at::empty({}, grads[0].options().dtype(at::kFloat));
    checked(dh_grad_norm((const double*)at_or_null(partial), partial.numel(), norm, (const float*)at_or_null(factor), nullptr, out.data_ptr<float>(),
                         stream_of(grads[0])),
            "dh_grad_norm");
    return out;
}

// Two workgroups must not scale one piece of memory, nor read what another writes: nothing is written twice, and what is written
// is read by its own gradient only, at the same places.
void apart(const char* where, const variable_list& read, const variable_list& written, bool in_place)
{
    struct At {
        const char *begin, *end;
        size_t k;
        bool operator<(const At& o) const { return begin < o.begin; }
    };
    const auto sorted = [](const variable_list& tensors) {
        std::vector<At> v;
        v.reserve(tensors.size());
        for (size_t k = 0; k < tensors.size(); ++k)
            if (tensors[k].numel()) {
                const char* at = (const char*)tensors[k].data_ptr();
                v.push_back({at, at + tensors[k].nbytes(), k});
            }
        std::sort(v.begin(), v.end());
        return v;
    };
    const std::vector<At> to = sorted(written);
    for (size_t k = 1; k < to.size(); ++k)
        if (to[k].begin < to[k - 1].end) fail(std::string(where) + ": a gradient is in the list twice, or two outputs overlap");
    if (in_place) return;                   // read where it is written
    // what is read is in the order of its beginnings, what is written is apart: the outputs behind every gradient that begins
    // later than they end are left behind, and each gradient is held against those it reaches
    const std::vector<At> from = sorted(read);
    size_t w = 0;
    for (const At& r : from) {
        while (w < to.size() && to[w].end <= r.begin) ++w;
        for (size_t o = w; o < to.size() && to[o].begin < r.end; ++o)
            if (to[o].k != r.k || to[o].begin != r.begin || to[o].end != r.end)
                fail(std::string(where) + ": an output overlaps a gradient of the list that is not its own");
    }
}

// The same for outputs that are written through a copy, `strided` among `into`: no element of their own twice (an expanded tensor), none
// begins where another begins, and neither their first nor their last element lies in an output that is written directly.
void strided_apart(const char* where, const variable_list& into, const std::vector<size_t>& strided)
{
    std::vector<std::pair<const char*, const char*>> whole;
    std::vector<bool> copied(into.size());
    std::vector<const char*> ends, begins;
    for (const size_t k : strided) {
        const Tensor& o = into[k];
        copied[k] = true;
        if (at::has_internal_overlap(o) == at::MemOverlap::Yes)
            fail(std::string(where) + ": a gradient or output whose elements share memory (an expanded tensor) cannot be written");
        if (!o.numel()) continue;
        int64_t last = 0;
        for (int64_t d = 0; d < o.dim(); ++d) last += (o.size(d) - 1) * o.stride(d);
        begins.push_back((const char*)o.data_ptr());
        ends.push_back(begins.back());
        ends.push_back(begins.back() + last * (int64_t)o.element_size());
    }
    for (size_t k = 0; k < into.size(); ++k)
        if (!copied[k] && into[k].numel()) whole.push_back({(const char*)into[k].data_ptr(), (const char*)into[k].data_ptr() + into[k].nbytes()});
    std::sort(begins.begin(), begins.end());
    std::sort(whole.begin(), whole.end());
    bool bad = std::adjacent_find(begins.begin(), begins.end()) != begins.end();
    for (const char* e : ends) {
        const auto after = std::upper_bound(whole.begin(), whole.end(), e, [](const char* v, const auto& w) { return v < w.first; });
        bad |= after != whole.begin() && e < (after - 1)->second;
    }
    if (bad) fail(std::string(where) + ": a gradient is in the list twice, or two outputs overlap");
}

// Norm, and outs[k] = grads[k] / scale * factor; without outs in place.
Tensor clip(const char* where, const variable_list& grads, const std::optional<variable_list>& outs, double limit, int norm,
            const py::object& scale, const py::object& reduce)
{
    const at::NoGradGuard off;
    variable_list read, written;
    read.reserve(grads.size());
    written.reserve(grads.size());
    const std::vector<List> lists = listed(where, grads, &read);
    const variable_list& into = outs ? *outs : grads;
    if (into.size() != grads.size())
        fail(std::string(where) + ": " + std::to_string(grads.size()) + " gradients and " + std::to_string(into.size()) + " outputs");
    const c10::DeviceGuard guard(grads[0].device());
    std::vector<size_t> copies;             // outputs that are written through a copy
    for (size_t k = 0; k < into.size(); ++k) {
        const Tensor &o = into[k], &g = grads[k];
        if (outs && (o.device() != g.device() || o.numel() != g.numel() || o.layout() != at::kStrided ||
                     (o.scalar_type() != g.scalar_type() && o.scalar_type() != at::kFloat)))
            fail(std::string(where) + ": an output must have its gradient's number of elements and device, and its type or fp32");
        // elements in one piece and in the order they are read in, or through a copy
        const bool direct = read[k].is_same(o) ||
                            (!o.is_neg() && ((read[k].is_contiguous() && o.is_contiguous()) ||
                                             (dense(o) && o.sizes() == read[k].sizes() && o.strides() == read[k].strides())));
        written.push_back(direct ? o : at::empty_like(read[k], read[k].options().dtype(o.scalar_type())));
        if (!direct) copies.push_back(k);
    }
    // the lists again, by the outputs' type: both kinds may occur for one kind of gradient
    struct Out {
        at::ScalarType type;
        List list;
        std::vector<void*> to;
    };
    std::vector<Out> launches;
    apart(where, read, written, !outs);
    if (!copies.empty()) strided_apart(where, into, copies);
    for (const List& l : lists)
        for (const at::ScalarType type : {l.type, at::kFloat}) {
            if (type == l.type && !launches.empty() && launches.back().list.type == l.type && launches.back().type == type) continue;
            Out o{type, {l.type, {}, {}, {}, 0}, {}};
            for (size_t e = 0; e < l.index.size(); ++e) {
                const size_t k = l.index[e];
                if (written[k].scalar_type() != type) continue;
                o.list.at.push_back(l.at[e]);
                o.list.n.push_back(l.n[e]);
                o.to.push_back(written[k].data_ptr());
            }
            if (!o.to.empty()) launches.push_back(std::move(o));
        }
    const Tensor factor = scale_on(where, scale, grads[0]);
    const Tensor partial = powers(lists, grads[0], norm, reduce);
    const Tensor out = at::empty({}, grads[0].options().dtype(at::kFloat));
    for (const Out& o : launches)
        checked(dh_grad_clip(o.list.at.data(), o.to.data(), o.list.n.data(), (int)o.to.size(), code_of(o.list.type), code_of(o.type), norm,
                             (const double*)at_or_null(partial), partial.numel(), (const float*)at_or_null(factor), limit, out.data_ptr<float>(),
                             stream_of(grads[0])),
                "dh_grad_clip");
    for (const size_t k : copies)
        into[k].copy_(written[k].sizes() == into[k].sizes() ? written[k] : written[k].reshape(into[k].sizes()));
    for (const Tensor& o : into)            // written through raw pointers: keep the version counters honest
        if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
    return out;
}

// clip() in place on what the parameters' .grad hold; nothing where none has one.
std::optional<Tensor> clip_parameters(const char* where, const variable_list& parameters, double limit, int norm, const py::object& scale,
                                      const py::object& reduce)
{
    variable_list grads;
    grads.reserve(parameters.size());
    for (const Tensor& p : parameters)
        if (p.grad().defined()) grads.push_back(p.grad());
    if (grads.empty()) return std::nullopt;
    return clip(where, grads, std::nullopt, limit, norm, scale, reduce);
}

}  // namespace

PYBIND11_MODULE(_host, m)
{
    m.def("linear", &linear);
    m.def("pointwise_conv", &pointwise_conv);
    m.def("head_convs", &head_convs);
    m.def("total_norm", &total_norm);
    m.def("clip", &clip);
    m.def("clip_parameters", &clip_parameters);
}
