// The host side of the calls whose device time is a few microseconds: walking a list of several hundred gradients, and the 4-bit products with their autograd node,
// as an extension module over torch's C++ API.  It adds no arithmetic: checks, allocations, current stream, and the C ABI of libvhap_hip.so, whose entry points
// it is handed as addresses (bind) by vhap_amd/_lib.py -- the library that the process already uses.
// Why not in Python like the rest: reading five attributes each of 504 gradients and 504 results took 1.2 ms, forty times the two launches they were read for; a Python
// autograd node's backward took about 100 us of host time around 40 us of kernels.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <unordered_set>

#include "vhap_hip.h"

namespace py = pybind11;
using at::Tensor;

namespace {

struct Api {
    decltype(&vhap_strerror) strerror = nullptr;
    decltype(&vhap_grad_norm_workspace_bytes) norm_bytes = nullptr;
    decltype(&vhap_grad_norm) norm = nullptr;
    decltype(&vhap_grad_clip) clip = nullptr;
    decltype(&vhap_adam_step_clipped) adam = nullptr;
    decltype(&vhap_mx4_quantize) quantize = nullptr;
    decltype(&vhap_mx4_dequantize) dequantize = nullptr;
    decltype(&vhap_mx4_linear) linear = nullptr;
    decltype(&vhap_mx4_linear_input_grad_workspace_bytes) grad_bytes = nullptr;
    decltype(&vhap_mx4_linear_input_grad) input_grad = nullptr;
    decltype(&vhap_mx4_column_sums) column_sums = nullptr;
    decltype(&vhap_mx4_matmul) matmul = nullptr;
} api;
PyObject* hip_error = nullptr;      // vhap_amd._lib.VhapHipError

struct HipError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

void check(int rc, const char* what) {
    if (rc != VHAP_OK) throw HipError(std::string(what) + ": " + api.strerror(rc) + " (" + std::to_string(rc) + ")");
}

template <typename... A>
std::string text(const A&... a) {
    std::ostringstream o;
    (void)std::initializer_list<int>{(o << a, 0)...};
    return o.str();
}

int dtype_code(at::ScalarType t) {
    return t == at::kFloat ? VHAP_DTYPE_F32 : t == at::kBFloat16 ? VHAP_DTYPE_BF16 : t == at::kHalf ? VHAP_DTYPE_F16 : -1;
}

vhap_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void plain(const Tensor& t, const char* what) {
    if (t.is_neg()) throw py::type_error(text(what, ": a view whose elements are negated when they are read (resolve_neg() it first)"));
}

void on_hip(const Tensor& t, const char* what) {
    if (!t.is_cuda()) throw std::runtime_error(text(what, ": tensors on a HIP device (no CPU fallback)"));
}

// ---- the global norm ----
// The tensors of a Python sequence, borrowed: `keep` holds the sequence, which holds them.
struct List {
    py::object keep;
    std::vector<const Tensor*> t;
    size_t size() const { return t.size(); }
    const Tensor& operator[](size_t i) const { return *t[i]; }
};

List gradients(py::handle given, const char* what) {
    List l;
    l.keep = py::reinterpret_steal<py::object>(PySequence_Fast(given.ptr(), "expected a sequence of tensors"));
    if (!l.keep) throw py::error_already_set();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(l.keep.ptr());
    PyObject** items = PySequence_Fast_ITEMS(l.keep.ptr());
    l.t.reserve(n);
    for (Py_ssize_t i = 0; i < n; i++) {
        if (!THPVariable_Check(items[i])) throw py::type_error(text(what, ": expected tensors, got ", Py_TYPE(items[i])->tp_name));
        const Tensor& t = THPVariable_Unpack(items[i]);
        if (t.layout() != at::kStrided || dtype_code(t.scalar_type()) < 0)
            throw py::type_error(text(what, ": dense float32, bfloat16 or float16 tensors, got ", t.scalar_type(), " (", t.layout(), ")"));
        plain(t, what);
        on_hip(t, what);
        if (i > 0 && t.device() != l[0].device()) throw py::value_error(text(what, ": tensors on one device, got ", l[0].device(), " and ", t.device()));
        l.t.push_back(&t);
    }
    return l;
}

struct Table {
    std::vector<const void*> src;
    std::vector<void*> dst;
    std::vector<int64_t> numel;
    std::vector<int32_t> dtype;
    explicit Table(size_t n) {
        src.reserve(n);
        dst.reserve(n);
        numel.reserve(n);
        dtype.reserve(n);
    }
    void add(const Tensor& s, const Tensor* d) {
        src.push_back(s.data_ptr());
        if (d) dst.push_back(d->data_ptr());
        numel.push_back(s.numel());
        dtype.push_back(dtype_code(s.scalar_type()));
    }
};

Tensor workspace(size_t bytes, const Tensor& like) { return at::empty({(int64_t)((bytes + 7) / 8)}, like.options().dtype(at::kDouble)); }

Tensor grad_norm(py::handle given, int kind) {
    at::NoGradGuard no_grad;
    const List ts = gradients(given, "grad_norm");
    if (ts.size() == 0) return at::zeros({});
    c10::DeviceGuard guard(ts[0].device());
    Table t(ts.size());
    std::vector<Tensor> copies;
    for (size_t i = 0; i < ts.size(); i++) {
        if (ts[i].is_non_overlapping_and_dense()) {
            t.add(ts[i], nullptr);
        } else {
            copies.push_back(ts[i].contiguous());
            t.add(copies.back(), nullptr);
        }
    }
    const size_t bytes = api.norm_bytes((int)ts.size());
    Tensor ws = workspace(bytes, ts[0]), norm = at::empty({}, ts[0].options().dtype(at::kFloat));
    check(api.norm((int)ts.size(), t.src.data(), t.numel.data(), t.dtype.data(), kind, ws.data_ptr(), bytes, norm.data_ptr<float>(), stream_of(norm)), "vhap_grad_norm");
    return norm;
}

// The bytes of a tensor: lo + sum c z over its axes (c: stride, 0 <= z <= most) and over the bytes of an element; all in [lo, hi).
struct Place {
    struct Axis {
        int64_t c, most;
    };
    int64_t lo, hi, step = 0, run;            // the largest stride (0: none), and what lies within one
    std::vector<Axis> axes;
    explicit Place(const Tensor& t) {
        const int64_t size = (int64_t)t.element_size();
        lo = (int64_t)(uintptr_t)t.data_ptr();
        hi = lo + size;
        axes.push_back({1, size - 1});
        for (int64_t d = 0; d < t.dim(); d++) {
            if (t.size(d) < 2 || t.stride(d) == 0) continue;
            axes.push_back({t.stride(d) * size, t.size(d) - 1});
            hi += axes.back().c * axes.back().most;
        }
        run = hi - lo;
        for (const Axis& a : axes)
            if (a.c > step && a.most > 0) {
                step = a.c;
                run = hi - lo - a.c * a.most;
            }
    }
    // Nothing in common.  Columns of one matrix are told apart by where their runs lie in a row.  Otherwise: lo + sum c z = b.lo + sum c' z', with z' counted from its other
    // end, is sum c z + sum c' (most' - z') = b.hi - 1 - lo: one sum of positive steps that reaches a given place, or does not.
    bool apart(const Place& b) const {
        if (hi <= b.lo || b.hi <= lo) return true;
        if (step == b.step && step > 0) {
            const int64_t to = ((b.lo - lo) % step + step) % step;
            if (to >= run && to + b.run <= step) return true;
        }
        std::vector<Axis> all(axes);
        all.insert(all.end(), b.axes.begin(), b.axes.end());
        int steps = 20000;
        return !reaches(all, b.hi - 1 - lo, steps);
    }
    // Two of its own elements in one place: a difference of indices d, not zero, with sum c d = 0.  For each axis as the first with d_k > 0, c_k + c_k (d_k - 1) plus the later
    // axes' c (d + most), 0 <= d + most <= 2 most, is the later axes' sum c most.
    bool folded() const {
        int steps = 20000;
        for (size_t k = 1; k < axes.size(); k++) {
            std::vector<Axis> rest{{axes[k].c, axes[k].most - 1}};
            int64_t place = -axes[k].c;
            for (size_t j = k + 1; j < axes.size(); j++) {
                rest.push_back({axes[j].c, 2 * axes[j].most});
                place += axes[j].c * axes[j].most;
            }
            if (reaches(rest, place, steps)) return true;
        }
        return false;
    }
    // is there a z, 0 <= z_k <= most_k, with sum c_k z_k = place?  Largest c first, and only what the smaller ones can make up for: for axes that nest, two or three values
    // each.  Yes where `steps` run out.
    static bool reaches(std::vector<Axis>& axes, int64_t place, int& steps) {
        std::sort(axes.begin(), axes.end(), [](const Axis& a, const Axis& b) { return a.c > b.c; });
        size_t n = 0;
        int64_t all = 0;
        for (const Axis& a : axes) {          // (equal steps are one)
            if (n > 0 && axes[n - 1].c == a.c) axes[n - 1].most += a.most;
            else axes[n++] = a;
            all += a.c * a.most;
        }
        axes.resize(n);
        return search(axes, 0, place, all, steps);
    }
    static bool search(const std::vector<Axis>& axes, size_t k, int64_t place, int64_t all, int& steps) {       // all: the most that axes k, k + 1, ... add up to
        if (place < 0 || place > all) return false;
        if (place == 0 || place == all) return true;
        if (--steps < 0) return true;
        const int64_t c = axes[k].c, rest = all - c * axes[k].most;
        for (int64_t z = std::min(axes[k].most, place / c); z >= 0 && place - c * z <= rest; z--)
            if (search(axes, k + 1, place - c * z, rest, steps)) return true;
        return false;
    }
};

// -> (results, norm); `out` None: new tensors
py::tuple clip(py::handle given, py::object out, int kind, double max_norm) {
    at::NoGradGuard no_grad;
    static const char* what = "clip_by_global_norm";
    const List gs = gradients(given, what);
    const bool made = out.is_none(), in_place = !made && out.ptr() == given.ptr();
    std::vector<Tensor> fresh;
    List outs;
    if (made) {
        fresh.reserve(gs.size());
        for (size_t i = 0; i < gs.size(); i++) {
            fresh.push_back(at::empty(gs[i].sizes(), gs[i].options()));
            outs.t.push_back(&fresh.back());
        }
    } else if (in_place) {
        outs.t = gs.t;
    } else {
        outs = gradients(out, "clip_by_global_norm(out=)");
        if (outs.size() != gs.size()) throw py::value_error(text(what, ": ", gs.size(), " gradients, ", outs.size(), " results"));
        for (size_t i = 0; i < gs.size(); i++)
            if (outs[i].sizes() != gs[i].sizes() || outs[i].scalar_type() != gs[i].scalar_type() || outs[i].device() != gs[i].device())
                throw py::value_error(text(what, ": a result is like its gradient: ", gs[i].sizes(), " ", gs[i].scalar_type(), " ", gs[i].device(), ", got ", outs[i].sizes(), " ",
                                           outs[i].scalar_type(), " ", outs[i].device()));
    }
    py::object results = made ? py::cast(fresh) : in_place ? py::reinterpret_borrow<py::object>(given) : out;
    if (gs.size() == 0) return py::make_tuple(results, at::zeros({}));
    c10::DeviceGuard guard(gs[0].device());
    // the kernels walk memory in order: a pair that is dense with the same strides is taken as it stands, anything else goes through contiguous copies
    Table t(gs.size());
    struct Back {
        Tensor to, from;
        size_t place;                         // in the list
    };
    std::vector<Back> back;
    std::vector<Tensor> keep;
    for (size_t i = 0; i < gs.size(); i++) {
        const Tensor &g = gs[i], &o = outs[i];
        if ((g.is_contiguous() && o.is_contiguous()) || (g.strides() == o.strides() && g.is_non_overlapping_and_dense())) {
            t.add(g, &o);
            continue;
        }
        bool shared = false;
        for (int64_t d = 0; d < o.dim(); d++) shared |= o.stride(d) == 0 && o.size(d) > 1;
        if (shared || (o.numel() > 1 && !o.is_non_overlapping_and_dense() && Place(o).folded()))
            throw py::value_error(text(what, ": a result whose elements share memory (an expanded tensor, windows of one)"));
        const Tensor c = g.contiguous(), r = at::empty(c.sizes(), c.options());
        t.add(c, &r);
        keep.push_back(c);
        back.push_back({o, r, i});
    }
    if (!back.empty()) {                      // (dense ones among themselves: vhap_grad_clip sees to it)
        std::vector<std::pair<Place, size_t>> at;
        for (size_t i = 0; i < outs.size(); i++)
            if (outs[i].numel() > 0) at.emplace_back(Place(outs[i]), i);
        for (auto& b : back) {
            if (b.to.numel() == 0) continue;
            const Place mine(b.to);
            for (auto& x : at)
                if (x.second != b.place && !mine.apart(x.first))
                    throw py::value_error("clipping: a strided result overlaps another result in memory (the same tensor twice in the list?)");
        }
    }
    const size_t bytes = api.norm_bytes((int)gs.size());
    const Tensor ws = workspace(bytes, gs[0]), norm = at::empty({}, gs[0].options().dtype(at::kFloat));
    const int rc = api.clip((int)gs.size(), t.src.data(), t.dst.data(), t.numel.data(), t.dtype.data(), kind, max_norm, ws.data_ptr(), bytes, norm.data_ptr<float>(),
                            stream_of(norm));
    if (rc == VHAP_E_UNSUPPORTED) throw py::value_error("clipping: a result overlaps another result, or another gradient, in memory (the same tensor twice in the list?)");
    check(rc, "vhap_grad_clip");
    for (auto& b : back) b.to.copy_(b.from);
    if (!made)
        for (const Tensor* o : outs.t)
            if (!o->is_inference()) o->unsafeGetTensorImpl()->bump_version();       // (written behind autograd's back)
    return py::make_tuple(results, norm);
}

// What vhap_adam_step_clipped reads of an optimiser, per set of parameters that have a gradient; the gradients come with every step.
struct AdamTable {
    std::vector<float*> p, m, v;
    std::vector<int64_t> numel;
    std::vector<int32_t> lr_index;
    AdamTable(const std::vector<uintptr_t>& ps, const std::vector<uintptr_t>& ms, const std::vector<uintptr_t>& vs, std::vector<int64_t> n, std::vector<int32_t> lr)
        : numel(std::move(n)), lr_index(std::move(lr)) {
        for (uintptr_t x : ps) p.push_back(reinterpret_cast<float*>(x));
        for (uintptr_t x : ms) m.push_back(reinterpret_cast<float*>(x));
        for (uintptr_t x : vs) v.push_back(reinterpret_cast<float*>(x));
    }
    void step(py::handle grads, const Tensor& lr, const Tensor& step, double beta1, double beta2, double eps, double max_norm, const Tensor& ws, const Tensor& norm, int flags) const {
        const List g = gradients(grads, "HipAdam");
        if (g.size() != p.size()) throw py::value_error("HipAdam: a gradient for every parameter of the table");
        std::vector<const float*> gp(g.size());
        for (size_t i = 0; i < g.size(); i++) {
            if (g[i].scalar_type() != at::kFloat || !g[i].is_contiguous() || g[i].numel() != numel[i] || g[i].device() != norm.device())
                throw std::runtime_error("HipAdam needs contiguous float32 gradients like its parameters");
            gp[i] = static_cast<const float*>(g[i].data_ptr());
        }
        c10::DeviceGuard guard(norm.device());
        check(api.adam((int)g.size(), p.data(), gp.data(), m.data(), v.data(), numel.data(), lr_index.data(), lr.data_ptr<float>(), step.data_ptr<int32_t>(), beta1, beta2, eps,
                       max_norm, ws.data_ptr(), (size_t)ws.nbytes(), norm.data_ptr<float>(), flags, stream_of(norm)), "vhap_adam_step_clipped");
    }
};

// ---- 4-bit products ----
// [..., K] -> (rows, row stride): a matrix with consecutive elements along K; anything else is copied
struct Rows {
    Tensor t;
    int64_t rows, ld;
};
Rows rows_of(const Tensor& t, int64_t K) {
    Tensor m = t.dim() == 2 ? t : t.reshape({t.numel() / K, K});
    if (K > 1 && m.stride(1) != 1) m = m.contiguous();
    const int64_t rows = m.size(0), ld = rows > 1 ? m.stride(0) : K;
    return {std::move(m), rows, ld};
}

std::vector<int64_t> with_last(const Tensor& t, int64_t last) {
    std::vector<int64_t> s = t.sizes().vec();
    s.back() = last;
    return s;
}

void floats(const Tensor& t, const char* what) {
    if (t.layout() != at::kStrided || dtype_code(t.scalar_type()) < 0)
        throw py::type_error(text(what, ": a float32, bfloat16 or float16 tensor, got ", t.scalar_type(), " (", t.layout(), ")"));
    plain(t, what);
}

// what a forward-mode tangent would be is the same product, but nothing here computes it: left out it would count as zero
void no_tangent(const Tensor& t, const char* what) {
    if (t._fw_grad(/*level=*/0).defined()) throw std::runtime_error(text(what, ": no forward-mode derivative (an input carries a tangent)"));
}

void pair_ok(const Tensor& x, const Tensor& codes, int64_t n, int64_t N, int64_t K, const char* what) {
    floats(x, what);
    no_tangent(x, what);
    if (x.dim() < 1 || x.size(-1) != n) throw py::value_error(text(what, ": ", n, " elements along the last axis for a matrix of [", N, ", ", K, "], got ", x.sizes()));
    if (x.device() != codes.device()) throw py::value_error(text(what, ": tensors on one device, got ", x.device(), " and ", codes.device()));
    on_hip(x, what);
}

void bias_ok(const std::optional<Tensor>& bias, int64_t N, c10::Device device, const char* what) {
    if (!bias) return;
    if (bias->scalar_type() != at::kFloat || bias->dim() != 1 || bias->size(0) != N) throw py::value_error(text(what, ": a float32 bias of ", N, " elements"));
    plain(*bias, what);
    no_tangent(*bias, what);
    if (bias->device() != device) throw py::value_error(text(what, ": the bias on ", device, ", got ", bias->device()));
}

std::pair<Tensor, Tensor> quantize(const Tensor& x) {
    at::NoGradGuard no_grad;
    floats(x, "quantize");
    on_hip(x, "quantize");
    if (x.dim() < 1 || x.size(-1) < 1) throw py::value_error(text("quantize: at least one element along the last axis, got ", x.sizes()));
    const int64_t K = x.size(-1), kb = (K + 31) / 32;
    c10::DeviceGuard guard(x.device());
    const auto bytes = x.options().dtype(at::kByte);
    Tensor codes = at::empty(with_last(x, 16 * kb), bytes), scales = at::empty(with_last(x, kb), bytes);
    const Rows r = rows_of(x, K);
    check(api.quantize(r.t.data_ptr(), dtype_code(x.scalar_type()), r.ld, r.rows, (int)K, codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), stream_of(x)), "vhap_mx4_quantize");
    return {codes, scales};
}

Tensor dequantize(const Tensor& codes, const Tensor& scales, int64_t K, at::ScalarType dtype) {
    at::NoGradGuard no_grad;
    c10::DeviceGuard guard(codes.device());
    Tensor out = at::empty(with_last(scales, K), codes.options().dtype(dtype));
    check(api.dequantize(codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), scales.numel() / scales.size(-1), (int)K, out.data_ptr(), dtype_code(dtype), stream_of(out)),
          "vhap_mx4_dequantize");
    return out;
}

Tensor run_linear(const Tensor& x, const Tensor& codes, const Tensor& scales, int64_t N, int64_t K, const Tensor& bias) {
    c10::DeviceGuard guard(x.device());
    Tensor y = at::empty(with_last(x, N), x.options());
    const Rows r = rows_of(x, K);
    const Tensor b = bias.defined() ? bias.contiguous() : bias;
    check(api.linear(r.t.data_ptr(), dtype_code(x.scalar_type()), r.ld, r.rows, codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), N, (int)K,
                     b.defined() ? b.data_ptr<float>() : nullptr, y.data_ptr(), stream_of(y)), "vhap_mx4_linear");
    return y;
}

Tensor run_input_grad(const Tensor& g, const Tensor& codes, const Tensor& scales, int64_t N, int64_t K) {
    c10::DeviceGuard guard(g.device());
    if (N == 0) return at::zeros(with_last(g, K), g.options());
    Tensor dx = at::empty(with_last(g, K), g.options());
    const Rows r = rows_of(g, N);
    const size_t bytes = api.grad_bytes(r.rows, N, (int)K);
    Tensor ws = workspace(bytes, g);
    check(api.input_grad(r.t.data_ptr(), dtype_code(g.scalar_type()), r.ld, r.rows, codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), N, (int)K, ws.data_ptr(), bytes,
                         dx.data_ptr(), 0, stream_of(dx)), "vhap_mx4_linear_input_grad");
    return dx;
}

Tensor run_column_sums(const Tensor& g, int64_t N) {
    c10::DeviceGuard guard(g.device());
    Tensor out = at::empty({N}, g.options().dtype(at::kFloat));
    if (N == 0) return out;
    const Rows r = rows_of(g, N);
    check(api.column_sums(r.t.data_ptr(), dtype_code(g.scalar_type()), r.ld, r.rows, N, out.data_ptr<float>(), stream_of(out)), "vhap_mx4_column_sums");
    return out;
}

struct MxLinear : torch::autograd::Function<MxLinear> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& codes, const Tensor& scales, int64_t N, int64_t K,
                          const std::optional<Tensor>& bias) {
        ctx->save_for_backward({codes, scales});
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["N"] = N;
        ctx->saved_data["K"] = K;
        return run_linear(x, codes, scales, N, K, bias ? *bias : Tensor());
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        TORCH_CHECK(!(at::GradMode::is_enabled() && grads[0].requires_grad()), "mx.linear is not twice differentiable");
        no_tangent(grads[0], "mx.linear's gradient");
        const Tensor g = grads[0].resolve_neg();      // (autograd makes such views by itself: the imaginary part of a conjugate; what a user passes is refused)
        const auto saved = ctx->get_saved_variables();
        const int64_t N = ctx->saved_data["N"].toInt(), K = ctx->saved_data["K"].toInt();
        Tensor dx, db;
        if (ctx->needs_input_grad(0)) dx = run_input_grad(g, saved[0], saved[1], N, K);
        if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3)) db = run_column_sums(g, N);      // (edges: x, codes, scales, bias if there is one)
        return {dx, Tensor(), Tensor(), Tensor(), Tensor(), db};
    }
};

// A node keeps the stream it was made on, a leaf's gradient node for as long as any graph holds it.  One made outside a capture makes the captured backward wait for that
// stream; where it is the default stream, that is nothing a capture survives (the runtime ends the process), wherever behind the input it lies.  Said here, while it can
// be.  (Other streams join the capture and leave it again; for the input's own node they are refused too.)
void capture_ok(const Tensor& t, const char* what) {
    if (!t.requires_grad()) return;
    const auto index = t.device().index();
    const auto here = c10::hip::getCurrentHIPStream(index).id(), standard = c10::hip::getDefaultHIPStream(index).id();
    const std::shared_ptr<torch::autograd::Node> first = t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn();
    std::vector<torch::autograd::Node*> todo;
    std::unordered_set<torch::autograd::Node*> seen;
    auto meet = [&](torch::autograd::Node* n) {
        if (n && seen.insert(n).second) todo.push_back(n);
    };
    meet(first.get());
    while (!todo.empty()) {
        torch::autograd::Node* const n = todo.back();
        todo.pop_back();
        const auto made_on = n->stream();
        if (made_on && made_on->device() == t.device() && made_on->id() != here && (n == first.get() || made_on->id() == standard))
            throw std::runtime_error(text(what, ": in a stream capture, while a graph behind its input made on another stream is alive (delete its results, or detach the input)"));
        for (const auto& e : n->next_edges()) meet(e.function.get());
    }
}

Tensor linear(const Tensor& x, const Tensor& codes, const Tensor& scales, int64_t N, int64_t K, const std::optional<Tensor>& bias) {
    bias_ok(bias, N, x.device(), "linear");
    pair_ok(x, codes, K, N, K, "linear");
    if (!at::GradMode::is_enabled() || !(x.requires_grad() || (bias && bias->requires_grad()))) {
        at::NoGradGuard no_grad;
        return run_linear(x, codes, scales, N, K, bias ? *bias : Tensor());
    }
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) {
        capture_ok(x, "linear");
        if (bias) capture_ok(*bias, "linear");
    }
    return MxLinear::apply(x, codes, scales, N, K, bias);
}

Tensor input_grad(const Tensor& g, const Tensor& codes, const Tensor& scales, int64_t N, int64_t K) {
    at::NoGradGuard no_grad;
    pair_ok(g, codes, N, N, K, "linear_input_grad");
    return run_input_grad(g, codes, scales, N, K);
}

Tensor matmul(const Tensor& ac, const Tensor& as, const Tensor& bc, const Tensor& bs, int64_t M, int64_t N, int64_t K, const std::optional<Tensor>& bias, bool relu,
              at::ScalarType dtype) {
    at::NoGradGuard no_grad;
    bias_ok(bias, N, ac.device(), "matmul");
    on_hip(ac, "matmul");
    c10::DeviceGuard guard(ac.device());
    Tensor y = at::empty({M, N}, ac.options().dtype(dtype));
    const Tensor b = bias ? bias->contiguous() : Tensor();
    check(api.matmul(ac.data_ptr<uint8_t>(), as.data_ptr<uint8_t>(), M, bc.data_ptr<uint8_t>(), bs.data_ptr<uint8_t>(), N, (int)K, b.defined() ? b.data_ptr<float>() : nullptr,
                     y.data_ptr(), dtype_code(dtype), relu ? VHAP_CONV_OUT_RELU : 0, stream_of(y)), "vhap_mx4_matmul");
    return y;
}

void bind(const py::dict& at, py::object error) {
    auto take = [&](auto& f, const char* name) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(at[name].cast<uintptr_t>()); };
    take(api.strerror, "vhap_strerror");
    take(api.norm_bytes, "vhap_grad_norm_workspace_bytes");
    take(api.norm, "vhap_grad_norm");
    take(api.clip, "vhap_grad_clip");
    take(api.adam, "vhap_adam_step_clipped");
    take(api.quantize, "vhap_mx4_quantize");
    take(api.dequantize, "vhap_mx4_dequantize");
    take(api.linear, "vhap_mx4_linear");
    take(api.grad_bytes, "vhap_mx4_linear_input_grad_workspace_bytes");
    take(api.input_grad, "vhap_mx4_linear_input_grad");
    take(api.column_sums, "vhap_mx4_column_sums");
    take(api.matmul, "vhap_mx4_matmul");
    hip_error = error.release().ptr();       // (for the life of the process)
}

}  // namespace

PYBIND11_MODULE(vhap_host, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const HipError& e) {
            PyErr_SetString(hip_error ? hip_error : PyExc_RuntimeError, e.what());
        }
    });
    m.def("bind", &bind);
    m.def("grad_norm", &grad_norm);
    m.def("clip", &clip);
    py::class_<AdamTable>(m, "AdamTable")
        .def(py::init<std::vector<uintptr_t>, std::vector<uintptr_t>, std::vector<uintptr_t>, std::vector<int64_t>, std::vector<int32_t>>())
        .def("step", &AdamTable::step);
    m.def("quantize", &quantize);
    m.def("dequantize", &dequantize);
    m.def("linear", &linear);
    m.def("input_grad", &input_grad);
    m.def("matmul", &matmul);
}
