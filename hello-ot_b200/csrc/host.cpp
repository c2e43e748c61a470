// Host path of the calls around and in a routed layer (routing, lookup, clipping, experts, norm, optimizer step): argument checks, output allocation and the call of
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

// ---------------------------------------------------------------- experts
int64_t on_eight(int64_t width) { return (width + 7) / 8 * 8; }
bool off(const void* p, size_t unit) { return reinterpret_cast<uintptr_t>(p) % unit != 0; }

// 16-bit operands off the 16-byte grid are copied to rows that lie on it, all of a call's in one launch into one buffer.
struct Grid {
    static constexpr int MOST = 3;
    int count = 0;
    Tensor buffer, source[MOST];
    const void** pointer[MOST];  // where the copies' addresses and distances go
    int64_t *row_out[MOST], *group_out[MOST];
    int64_t groups[MOST], rows[MOST], width[MOST], group[MOST], row[MOST];
    void add(const Tensor& t, const void** at, int64_t* row_at, int64_t* group_at) {
        const int i = count++;
        const bool weight = t.dim() == 3;
        source[i] = t, pointer[i] = at, row_out[i] = row_at, group_out[i] = group_at;
        groups[i] = weight ? t.size(0) : 1, rows[i] = t.size(-2), width[i] = t.size(-1);
        group[i] = weight ? t.stride(0) : 0, row[i] = t.stride(-2);
    }
    void copy(const Launch& on) {
        if (count == 0) return;
        int64_t at[MOST], stride[MOST], size = 0;
        for (int i = 0; i < count; ++i) {
            stride[i] = on_eight(width[i]);
            at[i] = size;
            size += (groups[i] * rows[i] * stride[i] * 2 + 255) / 256 * 256;
        }
        buffer = workspace(size, source[0].device());
        const void* from[MOST];
        void* to[MOST];
        for (int i = 0; i < count; ++i) {
            from[i] = source[i].const_data_ptr();
            to[i] = static_cast<char*>(buffer.data_ptr()) + at[i];
            *pointer[i] = to[i];
            *row_out[i] = stride[i];
            if (group_out[i]) *group_out[i] = rows[i] * stride[i];
        }
        check(hb_expert_copy(count, from, groups, rows, width, group, row, to, stride, on.stream));
    }
};

// Sorted rows as the products take them.
struct Sorted {
    Tensor t;
    int type;
    const void* data;
    int64_t stride;
};
Sorted expert_rows(const Tensor& given, const char* name) {
    Rows r = feature_rows(given, name);
    if (r.stride > INT32_MAX) r.t = r.t.contiguous(), r.stride = r.t.size(1);  // farther apart than the kernels step
    return {r.t, r.type, r.t.const_data_ptr(), r.stride};
}
void to_grid(Sorted& r, Grid& grid) {
    if (r.type == HB_F32 || r.t.numel() == 0) return;
    if (off(r.data, 16) || (r.t.size(0) > 1 && (r.stride % 8 != 0 || r.stride < r.t.size(1))))
        grid.add(r.t, &r.data, &r.stride, nullptr);
}
struct Weight {
    Tensor t;
    hb_expert_weight w;
};
// [experts, hidden, width], or [hidden, width] of one expert, without a copy where its rows are contiguous.
Weight expert_weight(const Tensor& given, const char* name) {
    TORCH_CHECK_VALUE(given.dim() == 3 || given.dim() == 2, name, " must be [experts, hidden, width], or [hidden, width] of one expert, got ",
                      given.sizes());
    type_of(given, name);
    Tensor t = resolved(given.dim() == 3 ? given : given.unsqueeze(0));
    const int64_t experts = t.size(0), hidden = t.size(1), width = t.size(2);
    TORCH_CHECK_VALUE(hidden >= 1 && width >= 1 && experts >= 1, name, " must have elements, got ", given.sizes());
    const bool plain = (width == 1 || t.stride(2) == 1) && (hidden == 1 || (t.stride(1) >= width && t.stride(1) <= INT32_MAX)) &&
                       (experts == 1 || t.stride(0) < (int64_t(1) << 38));
    if (!plain) t = t.contiguous();
    return {t, {t.const_data_ptr(), hidden > 1 ? t.stride(1) : on_eight(width), experts > 1 ? t.stride(0) : 0}};
}
void to_grid(Weight& w, Grid& grid) {
    if (w.t.scalar_type() == at::kFloat) return;
    if (off(w.w.data, 16) || (w.t.size(1) > 1 && w.t.stride(1) % 8 != 0) || (w.t.size(0) > 1 && w.t.stride(0) % 8 != 0))
        grid.add(w.t, &w.w.data, &w.w.row_stride, &w.w.expert_stride);
}
int activation_of(PyObject* o) {
    const char* name = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : "";
    if (!name) throw python_error();
    if (std::strcmp(name, "silu") == 0) return HB_SILU;
    TORCH_CHECK_VALUE(std::strcmp(name, "gelu") == 0, "activation must be 'silu' or 'gelu'");
    return HB_GELU;
}
// The first rows of the experts, null without them.
const int32_t* first_rows(const Tensor& offsets, int64_t experts, const char* what) {
    if (!offsets.defined()) {
        TORCH_CHECK_VALUE(experts == 1, what, ": offsets are needed for ", experts, " experts");
        return nullptr;
    }
    TORCH_CHECK_VALUE(offsets.scalar_type() == at::kInt && offsets.dim() == 1 && offsets.is_contiguous() && offsets.numel() == experts + 1, what,
                      ": offsets must be int32 [experts + 1], contiguous; got ", offsets.scalar_type(), " ", offsets.sizes(), " for ",
                      experts, " experts");
    return offsets.const_data_ptr<int32_t>();
}
// Shapes that belong together: x [rows, width], weights [experts, hidden, width], dy [rows, hidden].
hb_expert_shape shape_of(const Sorted& x, std::initializer_list<const Weight*> weights, const Sorted* dy, int activation, const char* what) {
    const Weight& w = **weights.begin();
    const int64_t experts = w.t.size(0), hidden = w.t.size(1), width = w.t.size(2), rows = x.t.size(0);
    for (const Weight* v : weights)
        TORCH_CHECK_VALUE(v->t.sizes() == w.t.sizes() && v->t.scalar_type() == x.t.scalar_type() && width == x.t.size(1), what, ": x ",
                          x.t.sizes(), " ", x.t.scalar_type(), " and weights ", w.t.sizes(), ", ", v->t.sizes(), " ", v->t.scalar_type(),
                          " do not fit");
    TORCH_CHECK_VALUE(!dy || (dy->t.size(0) == rows && dy->t.size(1) == hidden && dy->type == x.type), what,
                      ": the gradient's rows do not fit x and the weights");
    TORCH_CHECK_VALUE(experts <= 2048, what, ": at most 2048 experts, got ", experts);
    TORCH_CHECK_VALUE(rows <= INT32_MAX - 1024, what, ": too many rows");
    return {rows, width, hidden, experts, x.type, activation};
}

// expert_product(x, weight, offsets or None) -> y
PyObject* expert_product(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* what = "expert_product";
    expect(n, 3, what);
    const Tensor &given = tensor(args[0], "x"), &given_weight = tensor(args[1], "weight");
    const Tensor offsets = tensor_or_none(args[2], "offsets");
    return wrap(unlocked([&] {
        const c10::Device device = device_of(what, {&given, &given_weight, offsets.defined() ? &offsets : &given});
        const Launch on(device);
        Sorted x = expert_rows(given, "x");
        Weight w = expert_weight(given_weight, "weight");
        const hb_expert_shape shape = shape_of(x, {&w}, nullptr, HB_SILU, what);
        const int32_t* first = first_rows(offsets, shape.experts, what);
        Grid grid;
        if (!hb_expert_any_grid(&shape, 1)) to_grid(x, grid), to_grid(w, grid), grid.copy(on);
        Tensor out = at::empty({shape.rows, shape.hidden}, x.t.options());
        check(hb_expert_product(&shape, x.data, x.stride, first, &w.w, out.data_ptr(), on.stream));
        return out;
    }));
    END_HANDLE_TH_ERRORS
}

// expert_gated(x, gate, up, offsets or None, activation) -> h
PyObject* expert_gated(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* what = "expert_gated";
    expect(n, 5, what);
    const Tensor &given = tensor(args[0], "x"), &given_gate = tensor(args[1], "w_gate"), &given_up = tensor(args[2], "w_up");
    const Tensor offsets = tensor_or_none(args[3], "offsets");
    const int activation = activation_of(args[4]);
    return wrap(unlocked([&] {
        const c10::Device device = device_of(what, {&given, &given_gate, &given_up, offsets.defined() ? &offsets : &given});
        const Launch on(device);
        Sorted x = expert_rows(given, "x");
        Weight g = expert_weight(given_gate, "w_gate"), u = expert_weight(given_up, "w_up");
        const hb_expert_shape shape = shape_of(x, {&g, &u}, nullptr, activation, what);
        const int32_t* first = first_rows(offsets, shape.experts, what);
        Grid grid;
        if (!hb_expert_any_grid(&shape, 2)) to_grid(x, grid), to_grid(g, grid), to_grid(u, grid), grid.copy(on);
        Tensor out = at::empty({shape.rows, shape.hidden}, x.t.options());
        check(hb_expert_gated(&shape, x.data, x.stride, first, &g.w, &u.w, out.data_ptr(), on.stream));
        return out;
    }));
    END_HANDLE_TH_ERRORS
}

PyObject* tuple_of(std::initializer_list<const Tensor*> tensors) {  // undefined ones are None
    THPObjectPtr result(PyTuple_New((Py_ssize_t)tensors.size()));
    if (!result) throw python_error();
    Py_ssize_t i = 0;
    for (const Tensor* t : tensors) PyTuple_SET_ITEM(result.get(), i++, wrap(*t));
    return result.release();
}

// expert_product_grad(dy, x, weight, offsets or None, need_x, need_weight) -> (dx or None, dweight or None)
PyObject* expert_product_grad(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* what = "expert_product_grad";
    expect(n, 6, what);
    untraced(what);
    const Tensor &given_dy = tensor(args[0], "dy"), &given = tensor(args[1], "x"), &given_weight = tensor(args[2], "weight");
    const Tensor offsets = tensor_or_none(args[3], "offsets");
    const bool need_x = args[4] == Py_True, need_w = args[5] == Py_True;
    Tensor dx, dw;
    unlocked([&] {
        const c10::Device device = device_of(what, {&given, &given_dy, &given_weight, offsets.defined() ? &offsets : &given});
        const Launch on(device);
        Sorted dy = expert_rows(given_dy, "dy"), x = expert_rows(given, "x");
        Weight w = expert_weight(given_weight, "weight");
        const hb_expert_shape shape = shape_of(x, {&w}, &dy, HB_SILU, what);
        const int32_t* first = first_rows(offsets, shape.experts, what);
        if (need_x) dx = at::empty({shape.rows, shape.width}, x.t.options());
        if (need_w) dw = at::empty(given_weight.sizes(), x.t.options());
        Grid grid;
        if (!need_x && !need_w) return;
        to_grid(dy, grid);
        if (need_w) to_grid(x, grid);
        if (need_x) to_grid(w, grid);
        grid.copy(on);
        const size_t size = need_w ? hb_expert_product_grad_workspace(&shape) : 0;
        Tensor ws;
        if (size) ws = workspace(size, device);
        check(hb_expert_product_grad(&shape, dy.data, dy.stride, x.data, x.stride, first, &w.w,
                                     need_x ? dx.data_ptr() : nullptr, need_w ? dw.data_ptr() : nullptr, size ? ws.data_ptr() : nullptr, size,
                                     on.stream));
    });
    return tuple_of({&dx, &dw});
    END_HANDLE_TH_ERRORS
}

// expert_gated_grad(dh, x, gate, up, offsets or None, activation, need_x, need_gate, need_up) -> (dx, dgate, dup), None for those not needed
PyObject* expert_gated_grad(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* what = "expert_gated_grad";
    expect(n, 9, what);
    untraced(what);
    const Tensor &given_dh = tensor(args[0], "dh"), &given = tensor(args[1], "x"), &given_gate = tensor(args[2], "w_gate"),
                 &given_up = tensor(args[3], "w_up");
    const Tensor offsets = tensor_or_none(args[4], "offsets");
    const int activation = activation_of(args[5]);
    const bool need_x = args[6] == Py_True, need_g = args[7] == Py_True, need_u = args[8] == Py_True;
    Tensor dx, dg, du;
    unlocked([&] {
        const c10::Device device = device_of(what, {&given, &given_dh, &given_gate, &given_up, offsets.defined() ? &offsets : &given});
        const Launch on(device);
        const Sorted dh = expert_rows(given_dh, "dh");
        Sorted x = expert_rows(given, "x");
        Weight g = expert_weight(given_gate, "w_gate"), u = expert_weight(given_up, "w_up");
        const hb_expert_shape shape = shape_of(x, {&g, &u}, &dh, activation, what);
        const int32_t* first = first_rows(offsets, shape.experts, what);
        if (need_x) dx = at::empty({shape.rows, shape.width}, x.t.options());
        if (need_g) dg = at::empty(given_gate.sizes(), x.t.options());
        if (need_u) du = at::empty(given_up.sizes(), x.t.options());
        if (!need_x && !need_g && !need_u) return;
        Grid grid;
        to_grid(x, grid), to_grid(g, grid), to_grid(u, grid), grid.copy(on);
        const size_t size = hb_expert_gated_grad_workspace(&shape);
        Tensor ws = workspace(size, device);
        check(hb_expert_gated_grad(&shape, dh.data, dh.stride, x.data, x.stride, first, &g.w, &u.w,
                                   need_x ? dx.data_ptr() : nullptr, need_g ? dg.data_ptr() : nullptr, need_u ? du.data_ptr() : nullptr,
                                   ws.data_ptr(), size, on.stream));
    });
    return tuple_of({&dx, &dg, &du});
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- norm
// A tensor [..., width] as rows.
Rows rows_2d(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, name, " must be [..., width] with at least one column, got ", t.sizes());
    return feature_rows(t.dim() == 2 ? t : t.reshape({t.numel() / t.size(-1), t.size(-1)}), name);
}
Tensor norm_weight(const Tensor& given, int64_t width) {
    type_of(given, "weight");
    TORCH_CHECK_VALUE(given.dim() == 1 && given.size(0) == width, "weight must be [", width, "], got ", given.sizes());
    return resolved(given).contiguous();
}

// rms_norm(x, weight, residual or None, eps, bits8) -> (y or codes, None or scales, total or None)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* what = "rms_norm";
    expect(n, 5, what);
    const bool bits8 = args[4] == Py_True;
    if (bits8) untraced("rms_norm_8bit");
    const Tensor &given = tensor(args[0], "x"), &given_weight = tensor(args[1], "weight");
    const Tensor given_residual = tensor_or_none(args[2], "residual");
    const double eps = number(args[3]);
    Tensor y, scales, total;
    unlocked([&] {
        const bool add = given_residual.defined();
        const c10::Device device = device_of(what, {&given, &given_weight, add ? &given_residual : &given});
        const Launch on(device);
        const Rows x = rows_2d(given, "x");
        const int64_t count = x.t.size(0), width = x.t.size(1);
        TORCH_CHECK_VALUE(!add || (given_residual.sizes() == given.sizes() && given_residual.scalar_type() == given.scalar_type()), what,
                          ": the residual has x's shape and type, got ", given_residual.sizes(), " ", given_residual.scalar_type());
        const Rows residual = add ? rows_2d(given_residual, "residual") : x;
        const Tensor weight = norm_weight(given_weight, width);
        if (bits8) {
            y = at::empty(given.sizes(), x.t.options().dtype(at::kFloat8_e4m3fn));
            c10::SmallVector<int64_t, 8> shape(given.sizes().begin(), given.sizes().end());
            shape.back() = (width + 31) / 32;
            scales = at::empty(shape, x.t.options().dtype(at::kFloat8_e8m0fnu));
        } else {
            y = at::empty(given.sizes(), x.t.options());
        }
        if (add) total = at::empty(given.sizes(), x.t.options());
        check(hb_rms_norm(x.type, x.t.const_data_ptr(), x.stride, add ? residual.t.const_data_ptr() : nullptr, residual.stride, count, width,
                          weight.const_data_ptr(), type_of(weight, "weight"), eps, bits8 ? nullptr : y.data_ptr(),
                          bits8 ? y.data_ptr() : nullptr, bits8 ? scales.data_ptr() : nullptr, add ? total.data_ptr() : nullptr, on.stream));
    });
    return tuple_of({&y, &scales, &total});
    END_HANDLE_TH_ERRORS
}

// rows_of_8bit(codes, scales, dtype) -> values
PyObject* rows_of_8bit(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* what = "rows_of_8bit";
    expect(n, 3, what);
    untraced(what);
    const Tensor &given = tensor(args[0], "values"), &given_scales = tensor(args[1], "scales");
    TORCH_CHECK_VALUE(THPDtype_Check(args[2]), what, ": dtype must be a torch.dtype");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(args[2])->scalar_type;
    return wrap(unlocked([&] {
        const c10::Device device = device_of(what, {&given, &given_scales});
        const Launch on(device);
        TORCH_CHECK_VALUE(type_or(type, -1) >= 0, what, ": dtype must be float32, float16 or bfloat16, got ", type);
        TORCH_CHECK_VALUE(given.scalar_type() == at::kFloat8_e4m3fn && given_scales.scalar_type() == at::kFloat8_e8m0fnu && given.dim() >= 1 &&
                              given.size(-1) >= 1 && given_scales.dim() == given.dim() && given_scales.size(-1) == (given.size(-1) + 31) / 32 &&
                              given_scales.sizes().slice(0, given.dim() - 1) == given.sizes().slice(0, given.dim() - 1),
                          what, ": values e4m3 [..., width] with scales e8m0 [..., ceil(width / 32)], got ", given.sizes(), " and ",
                          given_scales.sizes());
        const Tensor codes = given.contiguous(), scales = given_scales.contiguous();
        Tensor out = at::empty(given.sizes(), given.options().dtype(type));
        check(hb_rows_of_8bit(codes.const_data_ptr(), scales.const_data_ptr(), codes.numel() / codes.size(-1), codes.size(-1),
                              type_or(type, HB_F32), out.data_ptr(), on.stream));
        return out;
    }));
    END_HANDLE_TH_ERRORS
}

// rms_norm_grad(dy, x, weight, dsum or None, eps, need_x, need_weight) -> (dx or None, dweight or None)
PyObject* rms_norm_grad(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* what = "rms_norm_grad";
    expect(n, 7, what);
    untraced(what);
    const Tensor &given_dy = tensor(args[0], "dy"), &given = tensor(args[1], "x"), &given_weight = tensor(args[2], "weight");
    const Tensor given_dsum = tensor_or_none(args[3], "dsum");
    const double eps = number(args[4]);
    const bool need_x = args[5] == Py_True, need_w = args[6] == Py_True;
    Tensor dx, dw;
    unlocked([&] {
        const bool add = given_dsum.defined();
        const c10::Device device = device_of(what, {&given, &given_dy, &given_weight, add ? &given_dsum : &given});
        const Launch on(device);
        TORCH_CHECK_VALUE(given_dy.sizes() == given.sizes() && given_dy.scalar_type() == given.scalar_type() &&
                              (!add || (given_dsum.sizes() == given.sizes() && given_dsum.scalar_type() == given.scalar_type())),
                          what, ": gradients have x's shape and type, got ", given_dy.sizes(), " ", given_dy.scalar_type(), " for ",
                          given.sizes(), " ", given.scalar_type());
        const Rows x = rows_2d(given, "x"), dy = rows_2d(given_dy, "dy"), dsum = add ? rows_2d(given_dsum, "dsum") : x;
        const int64_t count = x.t.size(0), width = x.t.size(1);
        const Tensor weight = norm_weight(given_weight, width);
        if (need_x) dx = at::empty(given.sizes(), x.t.options());
        if (need_w) dw = at::empty({width}, weight.options());
        const size_t size = hb_rms_norm_grad_workspace(count, width);
        Tensor ws = workspace(size, device);
        check(hb_rms_norm_grad(x.type, dy.t.const_data_ptr(), dy.stride, x.t.const_data_ptr(), x.stride,
                               add ? dsum.t.const_data_ptr() : nullptr, dsum.stride, count, width, weight.const_data_ptr(),
                               type_of(weight, "weight"), eps, need_x ? dx.data_ptr() : nullptr, need_w ? dw.data_ptr() : nullptr,
                               ws.data_ptr(), size, on.stream));
    });
    return tuple_of({&dx, &dw});
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- optimizer step
// Lists of a step: tensor i of each belongs to parameter i.
struct Step {
    const char* what;
    c10::Device device{c10::kCPU};
    std::vector<Tensor> params, changed;
    std::vector<int64_t> size;
    std::vector<Extent> written, read;
    Step(const char* name) : what(name) {}
    void span(const Tensor& t, std::vector<Extent>& to) {
        if (t.numel() == 0) return;
        const char* begin = static_cast<const char*>(t.const_data_ptr());
        to.push_back({begin, begin + t.nbytes(), 0});
    }
    const Tensor& on_device(PyObject* o, const char* name) {
        const Tensor& t = tensor(o, name);
        if (!device.is_cuda()) device = device_of(what, {&t});
        if (t.device() != device) device_of(what, {&t, params.empty() ? &t : &params[0]});
        TORCH_CHECK_VALUE(t.device() == device, what, ": ", name, " on another device than the parameters");
        TORCH_CHECK_VALUE(!t.is_neg() && !t._is_zerotensor(), what, ": ", name, " must hold its values in memory");
        return t;
    }
};
struct Items {  // a list of tensors, or of None
    THPObjectPtr items;
    Items(PyObject* o, const char* name, Py_ssize_t want, const char* what) : items(PySequence_Fast(o, "a list of tensors is needed")) {
        if (!items) throw python_error();
        TORCH_CHECK_VALUE(want < 0 || size() == want, what, ": ", size(), " ", name, " for ", want, " parameters");
    }
    Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(items.get()); }
    PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(items.get(), i); }
};
// The addresses of a list whose tensors lie in memory as the parameters do.
std::vector<void*> like_params(Step& s, PyObject* o, const char* name, at::ScalarType type, bool gaps, bool writes) {
    const Py_ssize_t n = (Py_ssize_t)s.params.size();
    const Items items(o, name, n, s.what);
    std::vector<void*> at(n, nullptr);
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (gaps && items[i] == Py_None) continue;
        const Tensor &t = s.on_device(items[i], name), &p = s.params[i];
        TORCH_CHECK_VALUE(t.scalar_type() == type, s.what, ": ", name, " must be ", type, ", got ", t.scalar_type());
        TORCH_CHECK_VALUE(t.sizes() == p.sizes() && ((t.is_contiguous() && p.is_contiguous()) || t.strides() == p.strides()), s.what, ": ", name,
                          " have their parameters' shapes and strides, got ", t.sizes(), " for ", p.sizes());
        if (t.numel()) at[i] = t.data_ptr();
        if (writes) s.span(t, s.written), s.changed.push_back(t);
    }
    return at;
}
std::vector<float*> scales_of(Step& s, PyObject* o, const char* name, bool writes) {
    const Py_ssize_t n = (Py_ssize_t)s.size.size();
    const Items items(o, name, n, s.what);
    std::vector<float*> at(n, nullptr);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const Tensor& t = s.on_device(items[i], name);
        TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == (s.size[i] + 255) / 256, s.what, ": ", name,
                          " must be float32, one for each 256 elements");
        if (t.numel()) at[i] = static_cast<float*>(t.data_ptr());
        if (writes) s.span(t, s.written), s.changed.push_back(t);
    }
    return at;
}
// A float32 number on the device.
const float* device_number(Step& s, PyObject* o, const char* name) {
    const Tensor& t = s.on_device(o, name);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.numel() == 1, s.what, ": ", name, " on the device must be one float32 value");
    TORCH_CHECK_VALUE(!(t.requires_grad() && c10::GradMode::is_enabled()), s.what, ": ", name, " is a number, not a tensor that takes a derivative");
    s.span(t, s.read);
    return static_cast<const float*>(t.const_data_ptr());
}
void check_apart(Step& s) {
    auto before = [](const Extent& a, const Extent& b) { return a.begin < b.begin; };
    std::sort(s.written.begin(), s.written.end(), before);
    for (size_t i = 1; i < s.written.size(); ++i)
        TORCH_CHECK_VALUE(s.written[i].begin >= s.written[i - 1].end, s.what, ": tensors that are written overlap in memory");
    for (const Extent& r : s.read) {
        auto w = std::upper_bound(s.written.begin(), s.written.end(), r.begin, [](const char* p, const Extent& e) { return p < e.end; });
        TORCH_CHECK_VALUE(w == s.written.end() || w->begin >= r.end, s.what, ": a tensor that is written overlaps a gradient or number in memory");
    }
}

// adamw_step(params, grads, first, second, first_scale or None, second_scale or None, master or None, step, lr, beta1, beta2, eps,
//            decay, norm or None, max_norm)
PyObject* adamw_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Step s("adamw_step");
    expect(n, 15, s.what);
    untraced(s.what);
    const Items params(args[0], "parameters", -1, s.what);
    const Py_ssize_t count = params.size();
    TORCH_CHECK_VALUE(count > 0, s.what, ": no parameters");
    s.params.reserve(count), s.size.reserve(count), s.written.reserve(6 * count + 1), s.read.reserve(count + 2), s.changed.reserve(6 * count + 1);
    std::vector<void*> param(count);
    std::vector<int32_t> type(count), grad_type(count);
    for (Py_ssize_t i = 0; i < count; ++i) {
        const Tensor& t = s.on_device(params[i], "a parameter");
        type[i] = type_of(t, "parameters");
        TORCH_CHECK_VALUE(t.is_contiguous() || t.is_non_overlapping_and_dense(), s.what, ": parameters must be dense in memory, got strides ",
                          t.strides(), " for ", t.sizes());
        param[i] = t.numel() ? t.data_ptr() : nullptr;
        s.params.push_back(t);
        s.size.push_back(t.numel());
        s.span(t, s.written);
        s.changed.push_back(t);
    }
    const Items grads(args[1], "gradients", count, s.what);
    std::vector<const void*> grad(count);
    for (Py_ssize_t i = 0; i < count; ++i) {
        const Tensor &t = s.on_device(grads[i], "a gradient"), &p = s.params[i];
        grad_type[i] = type_of(t, "gradients");
        TORCH_CHECK_VALUE(grad_type[i] == type[i] || grad_type[i] == HB_F32, s.what, ": a gradient has its parameter's type or is float32, got ",
                          t.scalar_type(), " for ", p.scalar_type());
        TORCH_CHECK_VALUE(t.sizes() == p.sizes() && ((t.is_contiguous() && p.is_contiguous()) || t.strides() == p.strides()), s.what,
                          ": gradients have their parameters' shapes and strides, got ", t.sizes(), " for ", p.sizes());
        grad[i] = t.numel() ? t.const_data_ptr() : nullptr;
        s.span(t, s.read);
    }
    const bool bits8 = args[4] != Py_None || args[5] != Py_None;
    const at::ScalarType held = bits8 ? at::kFloat8_e4m3fn : at::kFloat;
    const std::vector<void*> first = like_params(s, args[2], "first moments", held, false, true);
    const std::vector<void*> second = like_params(s, args[3], "second moments", held, false, true);
    std::vector<float*> first_scale, second_scale;
    if (bits8) first_scale = scales_of(s, args[4], "scales", true), second_scale = scales_of(s, args[5], "scales", true);
    std::vector<void*> master;
    if (args[6] != Py_None) master = like_params(s, args[6], "masters", at::kFloat, true, true);
    const Tensor& step = s.on_device(args[7], "step");
    TORCH_CHECK_VALUE(step.scalar_type() == at::kInt && step.numel() == 1, s.what, ": step must be one int32 value on the device");
    s.span(step, s.written);
    s.changed.push_back(step);
    hb_adamw_rule rule{};
    if (THPVariable_Check(args[8]) && THPVariable_Unpack(args[8]).is_cuda()) rule.rate = device_number(s, args[8], "lr");
    else rule.lr = number(args[8]);
    rule.beta1 = number(args[9]), rule.beta2 = number(args[10]), rule.eps = number(args[11]), rule.decay = number(args[12]);
    if (args[13] != Py_None) {
        TORCH_CHECK_VALUE(args[14] != Py_None, s.what, ": max_norm is needed with norm");
        rule.norm = device_number(s, args[13], "norm");
        rule.max_norm = number(args[14]);
    }
    TORCH_CHECK_VALUE(args[13] != Py_None || args[14] == Py_None, s.what, ": norm is needed with max_norm");
    check_apart(s);
    unlocked([&] {
        const Launch on(s.device);
        const size_t size = hb_adamw_workspace();
        Tensor ws = workspace(size, s.device);
        check(hb_adamw_step(count, param.data(), grad.data(), first.data(), second.data(), bits8 ? first_scale.data() : nullptr,
                            bits8 ? second_scale.data() : nullptr, master.empty() ? nullptr : reinterpret_cast<float* const*>(master.data()),
                            s.size.data(), type.data(), grad_type.data(), bits8 ? 8 : 32, &rule, static_cast<int32_t*>(step.data_ptr()),
                            ws.data_ptr(), size, on.stream));
        for (const Tensor& t : s.changed) written(t);
    });
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// adamw_moments(first, second, first_scale, second_scale) -> ([m], [v])
PyObject* adamw_moments(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Step s("adamw_moments");
    expect(n, 4, s.what);
    untraced(s.what);
    const Items codes(args[0], "first moments", -1, s.what);
    const Py_ssize_t count = codes.size();
    TORCH_CHECK_VALUE(count > 0, s.what, ": no moments");
    for (Py_ssize_t i = 0; i < count; ++i) {
        const Tensor& t = s.on_device(codes[i], "first moments");
        TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat8_e4m3fn && (t.is_contiguous() || t.is_non_overlapping_and_dense()), s.what,
                          ": 8-bit moments must be e4m3 and dense in memory");
        s.params.push_back(t);
        s.size.push_back(t.numel());
    }
    const std::vector<void*> first = like_params(s, args[0], "first moments", at::kFloat8_e4m3fn, false, false);
    const std::vector<void*> second = like_params(s, args[1], "second moments", at::kFloat8_e4m3fn, false, false);
    const std::vector<float*> first_scale = scales_of(s, args[2], "scales", false), second_scale = scales_of(s, args[3], "scales", false);
    std::vector<Tensor> out[2];
    unlocked([&] {
        std::vector<float*> at[2];
        for (int k = 0; k < 2; ++k)
            for (const Tensor& t : s.params) {
                out[k].push_back(at::empty_strided(t.sizes(), t.strides(), t.options().dtype(at::kFloat)));
                at[k].push_back(t.numel() ? out[k].back().data_ptr<float>() : nullptr);
            }
        const Launch on(s.device);
        check(hb_adamw_moments(count, const_cast<const void* const*>(first.data()), const_cast<const void* const*>(second.data()),
                               first_scale.data(), second_scale.data(), s.size.data(), at[0].data(), at[1].data(), on.stream));
    });
    THPObjectPtr result(PyTuple_New(2));
    if (!result) throw python_error();
    for (int k = 0; k < 2; ++k) {
        PyObject* list = PyList_New(count);
        if (!list) throw python_error();
        PyTuple_SET_ITEM(result.get(), k, list);
        for (Py_ssize_t i = 0; i < count; ++i) PyList_SET_ITEM(list, i, wrap(out[k][i]));
    }
    return result.release();
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
    {"expert_product", reinterpret_cast<PyCFunction>(expert_product), METH_FASTCALL, nullptr},
    {"expert_gated", reinterpret_cast<PyCFunction>(expert_gated), METH_FASTCALL, nullptr},
    {"expert_product_grad", reinterpret_cast<PyCFunction>(expert_product_grad), METH_FASTCALL, nullptr},
    {"expert_gated_grad", reinterpret_cast<PyCFunction>(expert_gated_grad), METH_FASTCALL, nullptr},
    {"rms_norm", reinterpret_cast<PyCFunction>(rms_norm), METH_FASTCALL, nullptr},
    {"rows_of_8bit", reinterpret_cast<PyCFunction>(rows_of_8bit), METH_FASTCALL, nullptr},
    {"rms_norm_grad", reinterpret_cast<PyCFunction>(rms_norm_grad), METH_FASTCALL, nullptr},
    {"adamw_step", reinterpret_cast<PyCFunction>(adamw_step), METH_FASTCALL, nullptr},
    {"adamw_moments", reinterpret_cast<PyCFunction>(adamw_moments), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef definition = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&definition); }
