// rows_torch.cpp -- the row operators' calls (rows.py) in the torch extension
// _plattice_torch: one combined test of the arguments, the outputs' and the
// workspace's allocation and the library call without the Python interpreter
// in between (a call of a small image costs 4 to 6 us of host time instead of
// 10 to 15).  Arguments that fail the test give None: rows.py then checks them
// one by one and raises the message, or makes the call itself.  A failed
// library call gives its status as an int.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include "plattice.h"

namespace {

struct Entry {
    decltype(&plattice_rows_pack8) pack8 = nullptr;
    decltype(&plattice_rows_unpack8) unpack8 = nullptr;
    decltype(&plattice_rms_norm) norm = nullptr;
    decltype(&plattice_rms_norm_backward_workspace_size) norm_ws = nullptr;
    decltype(&plattice_rms_norm_backward) norm_backward = nullptr;
    decltype(&plattice_linear_workspace_size) linear_ws = nullptr;
    decltype(&plattice_linear) linear = nullptr;
    decltype(&plattice_linear_backward_workspace_size) linear_backward_ws = nullptr;
    decltype(&plattice_linear_backward) linear_backward = nullptr;
} g_rows;

template <typename F> void set_one(F& f, int64_t address) { f = reinterpret_cast<F>(address); }

void set_rows_entry_points(const std::vector<int64_t>& a) {
    TORCH_CHECK(a.size() == 9, "nine entry points");
    set_one(g_rows.pack8, a[0]);
    set_one(g_rows.unpack8, a[1]);
    set_one(g_rows.norm, a[2]);
    set_one(g_rows.norm_ws, a[3]);
    set_one(g_rows.norm_backward, a[4]);
    set_one(g_rows.linear_ws, a[5]);
    set_one(g_rows.linear, a[6]);
    set_one(g_rows.linear_backward_ws, a[7]);
    set_one(g_rows.linear_backward, a[8]);
}

int dtype_code(at::ScalarType t) {
    return t == at::kFloat ? PLATTICE_F32 : t == at::kBFloat16 ? PLATTICE_BF16 : t == at::kHalf ? PLATTICE_F16 : -1;
}

// A contiguous CUDA tensor of one of the three types.
const at::Tensor* floating(const py::handle& o) {
    if (!THPVariable_Check(o.ptr())) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o.ptr());
    return t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() && dtype_code(t.scalar_type()) >= 0 ? &t
                                                                                                              : nullptr;
}

const at::Tensor* bytes(const py::handle& o) {
    if (!THPVariable_Check(o.ptr())) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o.ptr());
    return t.is_cuda() && t.is_contiguous() && t.scalar_type() == at::kByte && t.dim() == 2 ? &t : nullptr;
}

bool rows_tensor(const at::Tensor* t) { return t && t->dim() >= 1 && t->size(-1) >= 1; }
bool like(const at::Tensor& t, const at::Tensor& o) {
    return t.sizes() == o.sizes() && t.scalar_type() == o.scalar_type() && t.device() == o.device();
}
bool param(const at::Tensor* t, int64_t n, const at::Device& d) {
    return t && t->dim() == 1 && t->size(0) == n && t->device() == d;
}
int64_t width8(int64_t c) { return (c + 31) / 32 * 32; }

void* stream_of(const at::Device& d) { return at::cuda::getCurrentCUDAStream(d.index()).stream(); }

struct Rows8 {
    at::Tensor q, scale;
};

// Whether q and scale are the 8-bit rows of a tensor of `rows` x c (a Rows8's
// fields can be changed after it was checked).
bool holds(const at::Tensor& q, const at::Tensor& scale, int64_t rows, int64_t c) {
    return c >= 1 && c <= (1 << 30) && q.size(0) == rows && q.size(1) == width8(c) && scale.size(0) == rows &&
           scale.size(1) == width8(c) / 32 && q.device() == scale.device() && (uintptr_t)q.data_ptr() % 16 == 0;
}

int64_t rows_of(const std::vector<int64_t>& shape) {
    int64_t n = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) n *= shape[i];
    return n;
}

// at::empty without the dispatcher's way there (0.3 us of a call's host time
// per tensor; a call makes up to five).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType t, const at::Device& d) {
    return at::detail::empty_cuda(sizes, t, d, std::nullopt);
}
at::Tensor fresh_like(const at::Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t.device()); }

at::ScalarType type_of(int dtype) {
    return dtype == PLATTICE_F32 ? at::kFloat : dtype == PLATTICE_BF16 ? at::kBFloat16 : at::kHalf;
}

Rows8 empty8(int64_t rows, int64_t c, const at::Device& d) {
    return {fresh({rows, width8(c)}, at::kByte, d), fresh({rows, width8(c) / 32}, at::kByte, d)};
}

py::object wrap(const at::Tensor& t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(t)); }
py::object pair(const Rows8& r) { return py::make_tuple(wrap(r.q), wrap(r.scale)); }

py::object rows_pack8(const py::object& x_) {
    const at::Tensor* x = floating(x_);
    if (!rows_tensor(x)) return py::none();
    const int64_t c = x->size(-1), rows = x->numel() / c;
    if (c > (1 << 30)) return py::none();
    const c10::cuda::CUDAGuard guard(x->device());
    const Rows8 r = empty8(rows, c, x->device());
    const int rc = g_rows.pack8(r.q.data_ptr<uint8_t>(), r.scale.data_ptr<uint8_t>(), x->data_ptr(),
                                dtype_code(x->scalar_type()), rows, (int)c, stream_of(x->device()));
    if (rc) return py::int_(rc);
    return pair(r);
}

py::object rows_unpack8(const py::object& q_, const py::object& scale_, const std::vector<int64_t>& shape, int dtype) {
    const at::Tensor *q = bytes(q_), *scale = bytes(scale_);
    if (!q || !scale || shape.empty() || dtype < 0 || dtype > 2 || !holds(*q, *scale, rows_of(shape), shape.back()))
        return py::none();
    const c10::cuda::CUDAGuard guard(q->device());
    const at::Tensor y = fresh(shape, type_of(dtype), q->device());
    const int rc = g_rows.unpack8(y.data_ptr(), dtype, q->data_ptr<uint8_t>(), scale->data_ptr<uint8_t>(), q->size(0),
                                  (int)shape.back(), stream_of(q->device()));
    if (rc) return py::int_(rc);
    return wrap(y);
}

py::object rows_rms_norm(const py::object& x_, const py::object& gain_, const py::object& residual_, double eps,
                         bool pack) {
    const at::Tensor *x = floating(x_), *gain = floating(gain_);
    const at::Tensor* residual = residual_.is_none() ? nullptr : floating(residual_);
    if (!rows_tensor(x)) return py::none();
    const int64_t c = x->size(-1), rows = x->numel() / c;
    if (c > PLATTICE_NORM_MAX_CHANNELS || !param(gain, c, x->device()) ||
        (!residual_.is_none() && (!residual || !like(*residual, *x))))
        return py::none();
    const c10::cuda::CUDAGuard guard(x->device());
    const at::Tensor rstd = fresh(x->sizes().slice(0, x->dim() - 1), at::kFloat, x->device());
    const at::Tensor h = residual ? fresh_like(*x) : at::Tensor();
    Rows8 y8;
    at::Tensor y;
    if (pack) y8 = empty8(rows, c, x->device());
    else y = fresh_like(*x);
    const int rc = g_rows.norm(pack ? y8.q.data_ptr() : y.data_ptr(), pack ? y8.scale.data_ptr<uint8_t>() : nullptr,
                               residual ? h.data_ptr() : nullptr, rstd.data_ptr<float>(), x->data_ptr(),
                               residual ? residual->data_ptr() : nullptr, gain->data_ptr(), dtype_code(x->scalar_type()),
                               dtype_code(gain->scalar_type()), (float)eps, rows, (int)c, stream_of(x->device()));
    if (rc) return py::int_(rc);
    return py::make_tuple(pack ? pair(y8) : wrap(y), residual ? wrap(h) : x_, wrap(rstd));
}

py::object rows_rms_norm_backward(const py::object& gy_, const py::object& h_, const py::object& rstd_,
                                  const py::object& gain_, const py::object& gh_) {
    const at::Tensor *gy = floating(gy_), *h = floating(h_), *rstd = floating(rstd_), *gain = floating(gain_);
    const at::Tensor* gh = gh_.is_none() ? nullptr : floating(gh_);
    if (!rows_tensor(h) || !gy || !rstd) return py::none();
    const int64_t c = h->size(-1), rows = h->numel() / c;
    if (c > PLATTICE_NORM_MAX_CHANNELS || !like(*gy, *h) || !param(gain, c, h->device()) ||
        rstd->sizes() != h->sizes().slice(0, h->dim() - 1) || rstd->scalar_type() != at::kFloat ||
        rstd->device() != h->device() || (!gh_.is_none() && (!gh || !like(*gh, *h))))
        return py::none();
    const c10::cuda::CUDAGuard guard(h->device());
    size_t need = 0;
    int rc = g_rows.norm_ws(rows, (int)c, &need);
    if (rc) return py::int_(rc);
    const at::Tensor gx = fresh_like(*h), gg = fresh_like(*gain);
    const at::Tensor ws = fresh({(int64_t)need}, at::kByte, h->device());
    rc = g_rows.norm_backward(gx.data_ptr(), gg.data_ptr(), gy->data_ptr(), h->data_ptr(), rstd->data_ptr<float>(),
                              gain->data_ptr(), gh ? gh->data_ptr() : nullptr, ws.data_ptr(), need,
                              dtype_code(h->scalar_type()), dtype_code(gain->scalar_type()), rows, (int)c,
                              stream_of(h->device()));
    if (rc) return py::int_(rc);
    return py::make_tuple(wrap(gx), wrap(gg));
}

// The x of a linear call: a tensor, or a Rows8's q, scale and shape.
struct Input {
    const at::Tensor* x = nullptr;
    const at::Tensor* scale = nullptr;
    std::vector<int64_t> lead;
    int64_t rows = 1, k = 0;
    bool ok = false;
};

Input input_of(const py::object& x_, const py::object& scale_, const py::object& shape_, const at::Tensor& w) {
    Input in;
    if (scale_.is_none()) {
        in.x = floating(x_);
        if (!rows_tensor(in.x) || in.x->scalar_type() != w.scalar_type()) return in;
        in.lead.assign(in.x->sizes().begin(), in.x->sizes().end());
    } else {
        in.x = bytes(x_);
        in.scale = bytes(scale_);
        if (!in.x || !in.scale || w.scalar_type() == at::kHalf) return in;
        in.lead = shape_.cast<std::vector<int64_t>>();
        if (in.lead.empty() || !holds(*in.x, *in.scale, rows_of(in.lead), in.lead.back())) return in;
    }
    in.k = in.lead.back();
    in.lead.pop_back();
    for (int64_t s : in.lead) in.rows *= s;
    in.ok = in.x->device() == w.device() && in.k == w.size(1);
    return in;
}

bool weight_ok(const at::Tensor* w) {
    return w && w->dim() == 2 && w->size(0) >= 1 && w->size(1) >= 1 && w->size(0) <= (1 << 30) && w->size(1) <= (1 << 30);
}

// keep: 0 nothing, 1 as 8-bit rows, 2 in the output's type.  Gives
// (y0, y1 or None, z, z_scale), the latter two None as they apply.
py::object rows_linear(const py::object& x_, const py::object& scale_, const py::object& shape_, const py::object& w_,
                       const py::object& bias_, int act, const py::object& residual_, int64_t split, bool out32,
                       int keep) {
    const at::Tensor* w = floating(w_);
    if (!weight_ok(w)) return py::none();
    const Input in = input_of(x_, scale_, shape_, *w);
    if (!in.ok) return py::none();
    const int64_t n = w->size(0);
    const at::Tensor* bias = bias_.is_none() ? nullptr : floating(bias_);
    const at::Tensor* residual = residual_.is_none() ? nullptr : floating(residual_);
    const at::ScalarType out = out32 ? at::kFloat : w->scalar_type();
    if ((!bias_.is_none() && !param(bias, n, w->device())) || split < 0 || split >= n || (split && (act || residual)))
        return py::none();
    std::vector<int64_t> shape(in.lead);
    shape.push_back(n);
    if (!residual_.is_none() && (!residual || residual->sizes() != at::IntArrayRef(shape) ||
                                 residual->scalar_type() != out || residual->device() != w->device()))
        return py::none();
    const c10::cuda::CUDAGuard guard(w->device());
    plattice_linear_args a = {};
    at::Tensor y0, y1, z, z_scale;
    if (split) {
        shape.back() = split;
        y0 = fresh(shape, out, w->device());
        shape.back() = n - split;
        y1 = fresh(shape, out, w->device());
        a.y1 = y1.data_ptr();
    } else {
        y0 = fresh(shape, out, w->device());
    }
    if (keep == 1) {
        const Rows8 r = empty8(in.rows, n, w->device());
        z = r.q;
        z_scale = r.scale;
        a.z_scale = z_scale.data_ptr<uint8_t>();
    } else if (keep == 2) {
        shape.back() = n;
        z = fresh(shape, out, w->device());
    }
    a.x = in.x->data_ptr();
    a.x_scale = in.scale ? in.scale->data_ptr<uint8_t>() : nullptr;
    a.w = w->data_ptr();
    a.bias = bias ? bias->data_ptr() : nullptr;
    a.residual = residual ? residual->data_ptr() : nullptr;
    a.y0 = y0.data_ptr();
    a.z = keep ? z.data_ptr() : nullptr;
    a.rows = in.rows;
    a.k = (int)in.k;
    a.n = (int)n;
    a.split = (int)split;
    a.dtype = dtype_code(w->scalar_type());
    a.out_dtype = out32 ? PLATTICE_F32 : a.dtype;
    a.bias_dtype = bias ? dtype_code(bias->scalar_type()) : a.dtype;
    a.act = act;
    int rc = g_rows.linear_ws(&a, &a.workspace_bytes);
    if (rc) return py::int_(rc);
    at::Tensor ws;
    if (a.workspace_bytes) {
        ws = fresh({(int64_t)a.workspace_bytes}, at::kByte, w->device());
        a.workspace = ws.data_ptr();
    }
    rc = g_rows.linear(&a, stream_of(w->device()));
    if (rc) return py::int_(rc);
    const py::object none = py::none();
    return py::make_tuple(wrap(y0), split ? wrap(y1) : none, keep ? wrap(z) : none, keep == 1 ? wrap(z_scale) : none);
}

// g1 None: no split.  Gives (grad_x, grad_w, grad_b), None where not wanted.
py::object rows_linear_backward(const py::object& g0_, const py::object& g1_, const py::object& x_,
                                const py::object& scale_, const py::object& shape_, const py::object& w_,
                                const py::object& z_, const py::object& z_scale_, const py::object& z_shape_, int act,
                                int bias_dtype, bool need_x, bool need_w, bool need_b) {
    const at::Tensor *w = floating(w_), *g0 = floating(g0_), *g1 = g1_.is_none() ? nullptr : floating(g1_);
    if (!weight_ok(w) || !rows_tensor(g0) || x_.is_none() || bias_dtype < 0 || bias_dtype > 2) return py::none();
    const Input in = input_of(x_, scale_, shape_, *w);
    if (!in.ok) return py::none();
    const int64_t n = w->size(0);
    std::vector<int64_t> shape(in.lead);
    shape.push_back(n);
    plattice_linear_args a = {};
    if (!g1_.is_none()) {
        const int64_t split = g0->size(-1);
        if (act || split >= n || !g1) return py::none();
        a.split = (int)split;
        shape.back() = n - split;
        if (g1->sizes() != at::IntArrayRef(shape) || g1->scalar_type() != g0->scalar_type() || g1->device() != w->device())
            return py::none();
        shape.back() = split;
    }
    const at::ScalarType t = g0->scalar_type();
    if (g0->sizes() != at::IntArrayRef(shape) || g0->device() != w->device() || (t != at::kFloat && t != w->scalar_type()))
        return py::none();
    if (act) {
        if (z_scale_.is_none()) {
            const at::Tensor* z = z_.is_none() ? nullptr : floating(z_);
            if (!z || !like(*z, *g0)) return py::none();
            a.z = z->data_ptr();
        } else {
            const at::Tensor *z = bytes(z_), *zs = bytes(z_scale_);
            if (!z || !zs || z_shape_.cast<std::vector<int64_t>>() != shape || z->device() != w->device() ||
                !holds(*z, *zs, in.rows, n))
                return py::none();
            a.z = z->data_ptr();
            a.z_scale = zs->data_ptr<uint8_t>();
        }
    }
    const c10::cuda::CUDAGuard guard(w->device());
    at::Tensor gx, gw, gb;
    if (need_x) {
        shape.back() = in.k;
        gx = fresh(shape, w->scalar_type(), w->device());
        a.grad_x = gx.data_ptr();
    }
    if (need_w) {
        gw = fresh_like(*w);
        a.grad_w = gw.data_ptr();
    }
    if (need_b) {
        gb = fresh({n}, type_of(bias_dtype), w->device());
        a.grad_bias = gb.data_ptr();
    }
    a.x = in.x->data_ptr();
    a.x_scale = in.scale ? in.scale->data_ptr<uint8_t>() : nullptr;
    a.w = w->data_ptr();
    a.grad0 = g0->data_ptr();
    a.grad1 = g1 ? g1->data_ptr() : nullptr;
    a.rows = in.rows;
    a.k = (int)in.k;
    a.n = (int)n;
    a.dtype = dtype_code(w->scalar_type());
    a.out_dtype = dtype_code(t);
    a.bias_dtype = bias_dtype;
    a.act = act;
    int rc = g_rows.linear_backward_ws(&a, &a.workspace_bytes);
    if (rc) return py::int_(rc);
    const at::Tensor ws = fresh({(int64_t)a.workspace_bytes}, at::kByte, w->device());
    a.workspace = ws.data_ptr();
    rc = g_rows.linear_backward(&a, stream_of(w->device()));
    if (rc) return py::int_(rc);
    const py::object none = py::none();
    return py::make_tuple(need_x ? wrap(gx) : none, need_w ? wrap(gw) : none, need_b ? wrap(gb) : none);
}

}  // namespace

void register_rows(py::module_& m) {
    m.def("set_rows_entry_points", &set_rows_entry_points, "addresses of the library's row operators");
    m.def("rows_pack8", &rows_pack8);
    m.def("rows_unpack8", &rows_unpack8);
    m.def("rows_rms_norm", &rows_rms_norm);
    m.def("rows_rms_norm_backward", &rows_rms_norm_backward);
    m.def("rows_linear", &rows_linear);
    m.def("rows_linear_backward", &rows_linear_backward);
}
