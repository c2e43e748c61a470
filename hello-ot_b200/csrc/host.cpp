// Host path of the routing, lookup and clipping calls: argument checks, output allocation and the call of
// the C ABI, as a Python extension module (hello_ot_b200._host).
//
// The kernels of a small call take 2 to 8 us, so what a user waits for is the host: through ctypes and
// Python-level checks a call took 10 to 13 us, 3 of them the launch itself.  The functions here take the
// tensors themselves and do the same in compiled code.  They hold no state; tensors and workspaces come
// from torch's allocator on the current stream.  Shapes and types are refused with ValueError; errors of
// the C ABI are raised by hello_ot_b200._lib.check.
#include <algorithm>
#include <cstring>
#include <initializer_list>
#include <vector>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include "../../include/hello_b200.h"

namespace {

using at::Tensor;

// ---------------------------------------------------------------- arguments
// Whether a tensor carries a forward-mode tangent; inside an autograd function, whose tangents go their own way, none does.
bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }
const Tensor& tensor(PyObject* o, const char* name) {
    TORCH_CHECK_VALUE(THPVariable_Check(o), name, " must be a tensor");
    const Tensor& t = THPVariable_Unpack(o);
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(t), name, " carries a forward-mode tangent, and this call has no derivative");
    return t;
}
int64_t integer(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
// A tensor may stand for a number where no derivative is taken through it: none would come back.
double number(PyObject* o) {
    if (THPVariable_Check(o)) {
        const Tensor& t = THPVariable_Unpack(o);
        TORCH_CHECK_VALUE(!has_tangent(t) && !(t.requires_grad() && c10::GradMode::is_enabled()),
                          "a scale or limit is a number, not a tensor that takes a derivative");
        const Tensor plain = t.detach();
        return plain.item().toDouble();
    }
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
void expect(Py_ssize_t got, Py_ssize_t want, const char* what) {
    TORCH_CHECK_TYPE(got == want, what, " takes ", want, " arguments, got ", got);
}
PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }

// The interpreter let go, as torch's own calls do: an allocation or a launch can wait for the device, and a full launch
// queue for work that another Python thread has to do.
struct Unlocked {
    PyThreadState* const state = PyEval_SaveThread();
    Unlocked() = default;
    Unlocked(const Unlocked&) = delete;
    ~Unlocked() { PyEval_RestoreThread(state); }
};
template <typename F>
auto unlocked(F&& work) {
    const Unlocked now;
    return work();
}

// A function of hello_ot_b200._lib, for the error paths alone; called while the interpreter is let go.
void call_lib(const char* name, int arg, bool with_arg) {
    pybind11::gil_scoped_acquire held;
    THPObjectPtr module(PyImport_ImportModule("hello_ot_b200._lib"));
    if (!module) throw python_error();
    THPObjectPtr result(with_arg ? PyObject_CallMethod(module, name, "i", arg) : PyObject_CallMethod(module, name, nullptr));
    if (!result) throw python_error();
}
void check(int rc) {
    if (rc != HB_OK) call_lib("check", rc, true);
}

int type_or(at::ScalarType t, int otherwise) {
    return t == at::kFloat ? HB_F32 : t == at::kHalf ? HB_F16 : t == at::kBFloat16 ? HB_BF16 : otherwise;
}
int type_of(const Tensor& t, const char* name) {
    const int type = type_or(t.scalar_type(), -1);
    TORCH_CHECK_VALUE(type >= 0, name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
    return type;
}
int index_bytes(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, name, " must be int32 or int64, got ",
                      t.scalar_type());
    return t.scalar_type() == at::kLong ? 8 : 4;
}
// The one CUDA device of all tensors.
c10::Device device_of(const char* what, std::initializer_list<const Tensor*> tensors) {
    const c10::Device device = (*tensors.begin())->device();
    for (const Tensor* t : tensors)
        if (!t->is_cuda() || t->device() != device) {
            call_lib("lib", 0, false);  // without CUDA: the library's own error
            TORCH_CHECK_VALUE(false, what, ": expected CUDA tensors on one device, got ", device, " and ", t->device());
        }
    return device;
}

// A tensor whose memory holds its values: a lazily negated view's has the other sign, zeros of a tangent have none.
Tensor resolved(const Tensor& t) {
    if (t._is_zerotensor()) return at::zeros(t.sizes(), at::TensorOptions().dtype(t.scalar_type()).device(t.device()));
    return t.is_neg() ? t.resolve_neg() : t;
}

// Features whose rows are contiguous (a copy where they are not) and the rows' distance in elements.
struct Rows {
    Tensor t;
    int64_t stride;
    int type;
};
Rows feature_rows(const Tensor& given, const char* name) {
    TORCH_CHECK_VALUE(given.dim() == 2, name, " must be 2-D (rows x features), got ", given.sizes());
    const int type = type_of(given, name);
    const Tensor t = resolved(given);
    const int64_t width = t.size(1);
    if (t.is_contiguous()) return {t, width, type};
    if (width > 1 && t.stride(1) != 1) return {t.contiguous(), width, type};
    return {t, t.size(0) > 1 ? t.stride(0) : width, type};
}

// Whether rows share memory with a contiguous tensor.
bool meet(const Rows& r, const Tensor& t) {
    if (r.t.numel() == 0 || t.numel() == 0) return false;
    const int64_t size = r.t.element_size(), step = r.stride * size, row = r.t.size(1) * size;
    const int64_t begin = reinterpret_cast<const char*>(t.const_data_ptr()) - reinterpret_cast<const char*>(r.t.const_data_ptr());
    const int64_t end = begin + (int64_t)t.nbytes();  // both counted from the first row
    if (begin < row || step == 0) return begin < row && end > 0;  // a row at step 0 is the first one again
    const int64_t i = (begin - row) / step + 1;  // the first row that ends behind the tensor's begin
    return i < r.t.size(0) && i * step < end;
}

// Tells autograd that a tensor of the caller's was written.
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The device made current, its current stream, and a workspace on it.
struct Launch {
    c10::cuda::CUDAGuard guard;
    void* stream;
    explicit Launch(c10::Device d) : guard(d), stream(c10::cuda::getCurrentCUDAStream(d.index()).stream()) {}
};
Tensor workspace(size_t bytes, c10::Device device) {
    return at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(device));
}

// A trace records torch's operations and autograd functions: of a call that is neither it would keep the empty output.
void untraced(const char* what) {
    TORCH_CHECK_NOT_IMPLEMENTED(!at::tracer::impl::is_dispatch_enabled(), what, " cannot be recorded in a trace");
}

// number(value) -> the value as a float
PyObject* number_of(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 1, "number");
    return PyFloat_FromDouble(number(args[0]));
    END_HANDLE_TH_ERRORS
}

// recorded(tensor or None, ...) -> whether a call on them has to go through its autograd function: a derivative is
// taken through one of them, or a trace is made
PyObject* recorded(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (at::tracer::impl::is_dispatch_enabled()) Py_RETURN_TRUE;
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (!THPVariable_Check(args[i])) continue;
        const Tensor& t = THPVariable_Unpack(args[i]);
        if (has_tangent(t) || (t.requires_grad() && c10::GradMode::is_enabled())) Py_RETURN_TRUE;
    }
    Py_RETURN_FALSE;
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- routing
struct Places {
    const Tensor &position, &offsets;
    int64_t tokens, slots;
    const int32_t* at() const { return position.const_data_ptr<int32_t>(); }
    const int32_t* kept() const { return offsets.const_data_ptr<int32_t>() + offsets.numel() - 1; }
};
Places places(const Tensor& p, const Tensor& o, const char* what) {
    TORCH_CHECK_VALUE(p.scalar_type() == at::kInt && o.scalar_type() == at::kInt && p.dim() == 2 && o.dim() == 1, what,
                      ": a plan holds int32 position [tokens, slots] and offsets [num_experts + 1]");
    TORCH_CHECK_VALUE(p.is_contiguous() && o.is_contiguous() && o.numel() >= 2 && p.size(1) >= 1, what,
                      ": a plan's tensors are contiguous, with at least one slot and one expert");
    return {p, o, p.size(0), p.size(1)};
}
Tensor weights_of(const Tensor& given, const Places& p, const char* what) {
    const Tensor t = resolved(given);
    type_of(t, "weights");
    TORCH_CHECK_VALUE(t.sizes() == p.position.sizes() || (t.dim() == 1 && p.slots == 1 && t.size(0) == p.tokens), what,
                      ": weights ", t.sizes(), " do not fit an assignment ", p.position.sizes());
    return t.contiguous();
}

// A tensor, or an undefined one for None.
Tensor tensor_or_none(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor(o, name); }

// route_plan(index, num_experts) -> (order, position, offsets)
PyObject* route_plan(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 2, "route_plan");
    untraced("route_plan");
    const Tensor& given = tensor(args[0], "index");
    const int64_t experts = integer(args[1]);
    Tensor order, position, offsets;
    unlocked([&] {
        TORCH_CHECK_VALUE(given.dim() == 1 || (given.dim() == 2 && given.size(1) >= 1),
                          "index must be [tokens] or [tokens, slots], got ", given.sizes());
        const int bytes = index_bytes(given, "index");
        const int64_t entries = given.numel();
        TORCH_CHECK_VALUE(experts >= 1 && experts < INT32_MAX, "num_experts must be positive and below 2^31 - 1");
        TORCH_CHECK_VALUE(entries <= INT32_MAX, "an assignment holds at most 2^31 - 1 entries");
        const c10::Device device = device_of("route_plan", {&given});
        const Tensor index = given.contiguous();
        const auto options = at::TensorOptions().dtype(at::kInt).device(device);
        order = at::empty({entries}, options), offsets = at::empty({experts + 1}, options);
        position = at::empty({index.size(0), index.dim() == 2 ? index.size(1) : 1}, options);
        const size_t size = hb_index_sort_workspace(entries, experts);
        Tensor ws;
        if (size) ws = workspace(size, device);
        const Launch on(device);
        check(hb_index_sort(index.const_data_ptr(), bytes, entries, experts, order.data_ptr<int32_t>(),
                            position.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(), size ? ws.data_ptr() : nullptr, size,
                            on.stream));
    });
    THPObjectPtr result(PyTuple_New(3));
    if (!result) throw python_error();
    PyTuple_SET_ITEM(result.get(), 0, wrap(order));
    PyTuple_SET_ITEM(result.get(), 1, wrap(position));
    PyTuple_SET_ITEM(result.get(), 2, wrap(offsets));
    return result.release();
    END_HANDLE_TH_ERRORS
}

// route_dispatch(x, position, offsets) -> sorted
PyObject* route_dispatch(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 3, "route_dispatch");
    const Tensor &given = tensor(args[0], "x"), &position = tensor(args[1], "position"), &offsets = tensor(args[2], "offsets");
    return wrap(unlocked([&] {
        const Rows x = feature_rows(given, "x");
        const Places p = places(position, offsets, "route_dispatch");
        TORCH_CHECK_VALUE(x.t.size(0) == p.tokens, "route_dispatch: x has ", x.t.size(0), " rows for ", p.tokens, " tokens");
        const c10::Device device = device_of("route_dispatch", {&x.t, &p.position, &p.offsets});
        Tensor out = at::empty({p.tokens * p.slots, x.t.size(1)}, x.t.options());
        const Launch on(device);
        check(hb_route_dispatch(x.type, x.t.const_data_ptr(), x.stride, p.tokens, p.slots, x.t.size(1), p.at(), p.kept(),
                                out.data_ptr(), on.stream));
        return out;
    }));
    END_HANDLE_TH_ERRORS
}

// route_combine(z, position, offsets, weights or None, name) -> combined
PyObject* route_combine(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 5, "route_combine");
    const char* what = PyUnicode_AsUTF8(args[4]);
    if (!what) throw python_error();
    if (std::strcmp(what, "route_combine") != 0) untraced(what);  // by the name of another call it has no function of its own
    const Tensor &given = tensor(args[0], "z"), &position = tensor(args[1], "position"), &offsets = tensor(args[2], "offsets");
    const Tensor given_weights = tensor_or_none(args[3], "weights");
    return wrap(unlocked([&] {
        const Rows z = feature_rows(given, "z");
        const Places p = places(position, offsets, what);
        TORCH_CHECK_VALUE(z.t.size(0) == p.tokens * p.slots, what, ": ", z.t.size(0), " sorted rows for ", p.tokens, " x ",
                          p.slots, " entries");
        const bool weighted = given_weights.defined();
        Tensor weights;
        if (weighted) weights = weights_of(given_weights, p, what);
        const c10::Device device = device_of(what, {&z.t, &p.position, &p.offsets, weighted ? &weights : &z.t});
        Tensor out = at::empty({p.tokens, z.t.size(1)}, z.t.options());
        const Launch on(device);
        check(hb_route_combine(z.type, z.t.const_data_ptr(), z.stride, p.tokens, p.slots, z.t.size(1), p.at(), p.kept(),
                               weighted ? weights.const_data_ptr() : nullptr, weighted ? type_of(weights, "weights") : 0,
                               out.data_ptr(), on.stream));
        return out;
    }));
    END_HANDLE_TH_ERRORS
}

// route_combine_grad(dy, z, position, offsets, weights or None, need_weights) -> (dz, dweights or None)
PyObject* route_combine_grad(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* what = "route_combine_grad";
    expect(n, 6, what);
    untraced(what);
    const Tensor &given_dy = tensor(args[0], "dy"), &given_z = tensor(args[1], "z");
    const Tensor &position = tensor(args[2], "position"), &offsets = tensor(args[3], "offsets");
    const Tensor given_weights = tensor_or_none(args[4], "weights");
    const bool need_weights = args[5] == Py_True;
    Tensor dz, dw;
    unlocked([&] {
        const Rows dy = feature_rows(given_dy, "dy"), z = feature_rows(given_z, "z");
        const Places p = places(position, offsets, what);
        const int64_t width = z.t.size(1);
        TORCH_CHECK_VALUE(dy.t.size(0) == p.tokens && dy.t.size(1) == width && z.t.size(0) == p.tokens * p.slots &&
                              dy.type == z.type,
                          what, ": dy ", dy.t.sizes(), " ", dy.t.scalar_type(), " and z ", z.t.sizes(), " ",
                          z.t.scalar_type(), " do not fit an assignment ", p.position.sizes());
        const bool weighted = given_weights.defined();
        Tensor weights;
        if (weighted) weights = weights_of(given_weights, p, what);
        const c10::Device device = device_of(what, {&z.t, &dy.t, &p.position, &p.offsets, weighted ? &weights : &z.t});
        if (weighted && need_weights) dw = at::empty_like(weights);
        dz = at::empty({p.tokens * p.slots, width}, z.t.options());
        const Launch on(device);
        check(hb_route_combine_grad(z.type, dy.t.const_data_ptr(), dy.stride, z.t.const_data_ptr(), z.stride, p.tokens,
                                    p.slots, width, p.at(), p.kept(), weighted ? weights.const_data_ptr() : nullptr,
                                    weighted ? type_of(weights, "weights") : 0, dz.data_ptr(),
                                    dw.defined() ? dw.data_ptr() : nullptr, on.stream));
    });
    THPObjectPtr result(PyTuple_New(2));
    if (!result) throw python_error();
    PyTuple_SET_ITEM(result.get(), 0, wrap(dz));
    PyTuple_SET_ITEM(result.get(), 1, wrap(dw));  // None when undefined
    return result.release();
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- embedding
// embedding_lookup(table, ids, scale) -> rows
PyObject* embedding_lookup(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 3, "embedding_lookup");
    const Tensor &given = tensor(args[1], "ids"), &given_table = tensor(args[0], "table");
    const double scale = number(args[2]);
    return wrap(unlocked([&] {
        const int bytes = index_bytes(given, "ids");
        const Rows table = feature_rows(given_table, "table");
        const c10::Device device = device_of("embedding_lookup", {&table.t, &given});
        TORCH_CHECK_VALUE(given.numel() <= INT32_MAX, "embedding_lookup: at most 2^31 - 1 ids");
        const Tensor ids = given.contiguous();
        c10::SmallVector<int64_t, 8> shape(ids.sizes().begin(), ids.sizes().end());
        shape.push_back(table.t.size(1));
        Tensor out = at::empty(shape, table.t.options());
        const Launch on(device);
        check(hb_embedding_lookup(table.type, table.t.const_data_ptr(), table.stride, table.t.size(0), table.t.size(1),
                                  ids.const_data_ptr(), bytes, ids.numel(), scale, out.data_ptr(), on.stream));
        return out;
    }));
    END_HANDLE_TH_ERRORS
}

// embedding_grad(dy, ids, rows, scale, dtype or None, out or None, accumulate) -> gradient
PyObject* embedding_grad(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* what = "embedding_grad";
    expect(n, 7, what);
    untraced(what);
    const Tensor &dy_given = tensor(args[0], "dy"), &given = tensor(args[1], "ids");
    const int64_t rows = integer(args[2]);
    const double scale = number(args[3]);
    TORCH_CHECK_VALUE(args[4] == Py_None || THPDtype_Check(args[4]), what, ": dtype must be a torch.dtype");
    const Tensor given_out = tensor_or_none(args[5], "out");
    at::ScalarType type = given_out.defined() ? given_out.scalar_type() : dy_given.scalar_type();
    if (args[4] != Py_None) type = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    const bool accumulate = args[6] == Py_True;
    return wrap(unlocked([&] {
        const int bytes = index_bytes(given, "ids");
        const int64_t count = given.numel();
        TORCH_CHECK_VALUE(dy_given.dim() >= 1 && dy_given.sizes().slice(0, dy_given.dim() - 1) == given.sizes(), what,
                          ": dy ", dy_given.sizes(), " does not fit ids ", given.sizes());
        const int64_t width = dy_given.size(-1);
        TORCH_CHECK_VALUE(rows >= 1 && rows < INT32_MAX, what, ": rows must be positive and below 2^31 - 1");
        TORCH_CHECK_VALUE(count <= INT32_MAX, what, ": at most 2^31 - 1 ids");
        Rows dy = feature_rows(dy_given.dim() == 2 ? dy_given : dy_given.reshape({count, width}), "dy");
        if (dy.stride * dy.t.element_size() > (int64_t)UINT32_MAX) dy = {dy.t.contiguous(), width, dy.type};
        TORCH_CHECK_VALUE(type == dy.t.scalar_type() || type == at::kFloat, what, ": the gradient of ", dy.t.scalar_type(),
                          " rows is ", dy.t.scalar_type(), " or float32, not ", type);
        Tensor out = given_out;
        const bool given_one = out.defined();
        TORCH_CHECK_VALUE(given_one || !accumulate, what, ": accumulate needs out");
        const c10::Device device = device_of(what, {&dy.t, &given, given_one ? &out : &dy.t});
        if (!given_one)
            out = at::empty({rows, width}, dy.t.options().dtype(type));
        else
            TORCH_CHECK_VALUE(out.scalar_type() == type && out.dim() == 2 && out.size(0) == rows && out.size(1) == width &&
                                  out.is_contiguous() && !out.is_neg(),
                              what, ": out must be a contiguous ", type, " tensor of shape [", rows, ", ", width, "]");
        TORCH_CHECK_VALUE(!given_one || !meet(dy, out), what, ": out overlaps dy in memory");
        const Tensor ids = given.contiguous();
        const size_t size = hb_embedding_grad_workspace(count, rows, width);
        Tensor ws = workspace(size, device);
        if (given_one) written(out);
        const Launch on(device);
        check(hb_embedding_grad(dy.type, dy.t.const_data_ptr(), dy.stride, ids.const_data_ptr(), bytes, count, rows, width,
                                scale, type_or(type, HB_F32), out.data_ptr(), accumulate, ws.data_ptr(), size, on.stream));
        return out;
    }));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- clipping
struct Extent {  // the memory of a list's tensor
    const char *begin, *end;
    int64_t index;
};
struct List {
    std::vector<Tensor> tensors;
    std::vector<Extent> extents;  // by address, of the tensors that hold elements
    std::vector<void*> address;
    std::vector<int64_t> size;
    std::vector<int32_t> type;
};
// A list of float tensors on one device, each dense in memory and listed once.
List list_of(PyObject* o, const char* what, c10::Device* device) {
    THPObjectPtr items(PySequence_Fast(o, "gradients must be a list of tensors"));
    if (!items) throw python_error();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(items.get());
    List l;
    l.tensors.reserve(n), l.extents.reserve(n), l.address.reserve(n), l.size.reserve(n), l.type.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const Tensor& t = tensor(PySequence_Fast_GET_ITEM(items.get(), i), "a gradient");
        if (i == 0 && !device->is_cuda()) *device = device_of(what, {&t});
        if (t.device() != *device) device_of(what, {&t, i > 0 ? &l.tensors[0] : &t});
        TORCH_CHECK_VALUE(t.device() == *device, what, ": outputs on another device than their gradients");
        l.type.push_back(type_of(t, "gradients"));
        TORCH_CHECK_VALUE(!t.is_neg(), what, ": gradients must not be lazily negated views");
        TORCH_CHECK_VALUE(t.is_contiguous() || t.is_non_overlapping_and_dense(), what,
                          ": gradients must be dense in memory, got strides ", t.strides(), " for ", t.sizes());
        l.tensors.push_back(t);
        l.size.push_back(t.numel());
        l.address.push_back(t.numel() ? t.data_ptr() : nullptr);
        if (t.numel()) {
            const char* begin = static_cast<const char*>(l.address.back());
            l.extents.push_back({begin, begin + t.nbytes(), i});
        }
    }
    std::sort(l.extents.begin(), l.extents.end(), [](const Extent& a, const Extent& b) { return a.begin < b.begin; });
    for (size_t i = 1; i < l.extents.size(); ++i)
        TORCH_CHECK_VALUE(l.extents[i].begin != l.extents[i - 1].begin, what, ": a tensor is listed twice");
    return l;
}
// Blocks write the outputs while others still read the gradients: outputs share no memory with one another, nor with a
// gradient unless it is their own and they are in place.
void check_shared(const List& grads, const List& outs, const char* what) {
    const std::vector<Extent>& to = outs.extents;
    for (size_t i = 1; i < to.size(); ++i)
        TORCH_CHECK_VALUE(to[i].begin >= to[i - 1].end, what, ": tensors that are written overlap in memory");
    if (&grads == &outs) return;
    for (const Extent& g : grads.extents) {
        auto o = std::upper_bound(to.begin(), to.end(), g.begin, [](const char* p, const Extent& e) { return p < e.end; });
        for (; o != to.end() && o->begin < g.end; ++o)
            TORCH_CHECK_VALUE(o->index == g.index && o->begin == g.begin && o->end == g.end, what,
                              ": an output overlaps a gradient in memory and is not in its place");
    }
}

// clip(gradients, limit or None, outputs or None, name) -> norm
PyObject* clip(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 4, "clip");
    const char* what = PyUnicode_AsUTF8(args[3]);
    if (!what) throw python_error();
    untraced(what);
    c10::Device device(c10::kCPU);
    const List grads = list_of(args[0], what, &device);
    const int64_t count = (int64_t)grads.tensors.size();
    TORCH_CHECK_VALUE(count > 0, what, ": no gradients");
    const bool scale = args[1] != Py_None;
    const double limit = scale ? number(args[1]) : 0.0;
    TORCH_CHECK_VALUE(limit >= 0.0, what, ": max_norm must be a number >= 0, got ", limit);
    List outs;
    const List* to = &grads;
    if (args[2] != Py_None) {
        outs = list_of(args[2], what, &device);
        to = &outs;
        TORCH_CHECK_VALUE(outs.tensors.size() == grads.tensors.size(), what, ": ", outs.tensors.size(), " outputs for ",
                          count, " gradients");
        for (int64_t i = 0; i < count; ++i) {
            const Tensor &g = grads.tensors[i], &o = outs.tensors[i];
            TORCH_CHECK_VALUE(o.sizes() == g.sizes(), what, ": outputs have their gradients' shapes, got ", o.sizes(), " for ",
                              g.sizes());
            TORCH_CHECK_VALUE((o.is_contiguous() && g.is_contiguous()) || o.strides() == g.strides(), what,
                              ": outputs have their gradients' strides");
            TORCH_CHECK_VALUE(outs.type[i] == grads.type[i] ||
                                  (outs.type[i] == HB_F32 && (!outs.address[i] || outs.address[i] != grads.address[i])),
                              what, ": an output has its gradient's type, or is float32 and not in place; got ",
                              o.scalar_type(), " for ", g.scalar_type());
        }
    }
    if (scale) check_shared(grads, *to, what);
    return wrap(unlocked([&] {
        Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(device));
        const size_t size = hb_clip_workspace(count);
        Tensor ws = workspace(size, device);
        const Launch on(device);
        if (scale) {
            for (const Tensor& t : to->tensors) written(t);
            check(hb_clip_grad_norm(count, grads.address.data(), grads.size.data(), grads.type.data(), to->address.data(),
                                    to->type.data(), limit, norm.data_ptr<float>(), ws.data_ptr(), size, on.stream));
        } else {
            check(hb_grad_norm(count, grads.address.data(), grads.size.data(), grads.type.data(), norm.data_ptr<float>(),
                               ws.data_ptr(), size, on.stream));
        }
        return norm;
    }));
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"number", reinterpret_cast<PyCFunction>(number_of), METH_FASTCALL, nullptr},
    {"recorded", reinterpret_cast<PyCFunction>(recorded), METH_FASTCALL, nullptr},
    {"route_plan", reinterpret_cast<PyCFunction>(route_plan), METH_FASTCALL, nullptr},
    {"route_dispatch", reinterpret_cast<PyCFunction>(route_dispatch), METH_FASTCALL, nullptr},
    {"route_combine", reinterpret_cast<PyCFunction>(route_combine), METH_FASTCALL, nullptr},
    {"route_combine_grad", reinterpret_cast<PyCFunction>(route_combine_grad), METH_FASTCALL, nullptr},
    {"embedding_lookup", reinterpret_cast<PyCFunction>(embedding_lookup), METH_FASTCALL, nullptr},
    {"embedding_grad", reinterpret_cast<PyCFunction>(embedding_grad), METH_FASTCALL, nullptr},
    {"clip", reinterpret_cast<PyCFunction>(clip), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef definition = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&definition); }
