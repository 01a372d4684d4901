// The operators of tiramisu_hip_wrappers.h on torch tensors: what their arguments have to be, where results are allocated, and the call on torch's
// current stream.  tiramisu_amd/operators.py is the interface; this is its inner part, in C++ because a call of few tokens takes as long as its
// Python does (a norm of one token to 8 bits: 9.5 us a call with these steps in Python, 6.2 - 7.1 here, of which the launch is 2.9 and the kernel 4.8).
// Functions take positional arguments and return a tuple; ValueError says what does not fit.
#include <ATen/ATen.h>
#include <c10/core/Allocator.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <initializer_list>
#include <string>
#include <utility>
#include <vector>

#include "../../include/tiramisu_hip_wrappers.h"

namespace {

using at::ScalarType;
using at::Tensor;

int element_of(ScalarType t) {
    return t == at::kFloat ? TIRAMISU_HIP_FLOAT32 : t == at::kHalf ? TIRAMISU_HIP_FLOAT16 : t == at::kBFloat16 ? TIRAMISU_HIP_BFLOAT16 : TIRAMISU_HIP_FLOAT8_E4M3;
}
constexpr ScalarType EIGHT = ScalarType::Float8_e4m3fn;
const std::initializer_list<ScalarType> NORM_TYPES = {at::kBFloat16, at::kHalf, at::kFloat}, PRODUCT_TYPES = {at::kBFloat16, at::kHalf, EIGHT}, HALVES = {at::kBFloat16, at::kHalf};

// A type as Python calls it
std::string name_of(ScalarType t) {
    switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case EIGHT: return "torch.float8_e4m3fn";
    case at::kDouble: return "torch.float64";
    case at::kByte: return "torch.uint8";
    case at::kChar: return "torch.int8";
    case at::kShort: return "torch.int16";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return std::string("torch ") + c10::toString(t);
    }
}
std::string names_of(std::initializer_list<ScalarType> types) {
    std::string s;
    for (ScalarType t : types) s += (s.empty() ? "" : ", ") + name_of(t);
    return s;
}

// ---- arguments
Tensor tensor_of(PyObject *o, const char *name) {
    TORCH_CHECK_VALUE(THPVariable_Check(o), name, " is a tensor, not ", Py_TYPE(o)->tp_name);
    const Tensor &t = THPVariable_Unpack(o);
    // (a result without a graph would say nothing of the gradient that it loses)
    TORCH_CHECK_VALUE(!t.requires_grad() || !c10::GradMode::is_enabled(), name, " requires a gradient, which operators do not record: call them under torch.no_grad(), and their "
                      "backward functions");
    return t;
}
bool given(PyObject *o) { return o != Py_None; }

struct device_rows {
    int64_t rows, width, step;              // step: elements from row to row
    void *p;
};
// A tensor on the GPU whose rows are dense and one stride apart; `like`: whose GPU
device_rows rows_of(const Tensor &t, const char *name, std::initializer_list<ScalarType> types, const Tensor *like = nullptr) {
    bool known = false;
    for (ScalarType type : types) known = known || t.scalar_type() == type;
    TORCH_CHECK_VALUE(known, name, " holds ", name_of(t.scalar_type()), ": ", names_of(types), " are taken here");
    const int64_t dims = t.dim();
    TORCH_CHECK_VALUE(dims >= 1, name, " has no rows");
    TORCH_CHECK_VALUE(t.is_cuda(), name, " lives on ", t.device(), ": operators run on the GPU");
    TORCH_CHECK_VALUE(!like || t.device() == like->device(), name, " lives on another GPU");
    const int64_t width = t.size(dims - 1);
    int64_t rows = 1;
    for (int64_t d = 0; d + 1 < dims; d++) rows *= t.size(d);
    device_rows r = {rows, width, width, t.data_ptr()};
    if (t.is_contiguous()) return r;
    TORCH_CHECK_VALUE(t.stride(dims - 1) == 1 || width <= 1, name, ": the elements of a row are not next to each other");
    // dimensions of one row do not count, the others follow each other
    int64_t step = -1, expected = 0;
    for (int64_t d = dims - 2; d >= 0; d--) {
        if (t.size(d) == 1) continue;
        if (step < 0) step = t.stride(d);
        else TORCH_CHECK_VALUE(t.stride(d) == expected, name, ": rows are not one stride apart");
        expected = t.stride(d) * t.size(d);
    }
    r.step = step < 0 ? width : step;
    TORCH_CHECK_VALUE(r.step >= width, name, ": rows overlap");
    return r;
}
// ... of the shape of `x`'s leading dimensions and `columns` more
device_rows rows_like(PyObject *o, const char *name, const Tensor &x, int64_t columns, ScalarType type) {
    const Tensor t = tensor_of(o, name);
    bool same = t.dim() == x.dim() && t.size(t.dim() - 1) == columns;
    for (int64_t d = 0; same && d + 1 < x.dim(); d++) same = t.size(d) == x.size(d);
    if (!same) {
        std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = columns;
        TORCH_CHECK_VALUE(false, name, " has shape ", t.sizes(), ", not ", at::IntArrayRef(shape));
    }
    return rows_of(t, name, {type}, &x);
}
// rows < 0: any number
device_rows matrix_of(PyObject *o, const char *name, int64_t rows, int64_t columns, const Tensor &x, int64_t *outputs = nullptr) {
    const Tensor t = tensor_of(o, name);
    TORCH_CHECK_VALUE(t.dim() == 2 && (rows < 0 || t.size(0) == rows) && t.size(1) == columns, name, " is a matrix of [", rows < 0 ? std::string("outputs") : std::to_string(rows), ", ",
                      columns, "], not ", t.sizes());
    if (outputs) *outputs = t.size(0);
    return rows_of(t, name, {x.scalar_type()}, &x);
}
void *vector_of(PyObject *o, const char *name, int64_t size, ScalarType type, const Tensor &x) {
    const Tensor t = tensor_of(o, name);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == size && t.scalar_type() == type && t.is_cuda() && (size <= 1 || t.stride(0) == 1), name, " is a dense vector of ", size, " ",
                      name_of(type), " on the GPU, not ", name_of(t.scalar_type()), " of ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == x.device(), name, " lives on another GPU");
    return t.data_ptr();
}
// a number for each row of x, in the shape of its leading dimensions or flat
const float *row_numbers(PyObject *o, const char *name, const Tensor &x, int64_t rows) {
    const Tensor t = tensor_of(o, name);
    bool leading = t.dim() == x.dim() - 1 && t.is_contiguous();
    for (int64_t d = 0; leading && d < t.dim(); d++) leading = t.size(d) == x.size(d);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.is_cuda() && (leading || (t.dim() == 1 && t.size(0) == rows && (rows <= 1 || t.stride(0) == 1))), name, " is a dense vector of ", rows,
                      " ", name_of(at::kFloat), " on the GPU, not ", name_of(t.scalar_type()), " of ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == x.device(), name, " lives on another GPU");
    return (const float *)t.data_ptr();
}
int activation_of(PyObject *o) { return (int)PyLong_AsLong(o); }            // (its number: the names are the interface's)
void with_scales(const Tensor &x, std::initializer_list<std::pair<PyObject *, const char *>> scales) {
    for (const auto &s : scales) TORCH_CHECK_VALUE(given(s.first) == (x.scalar_type() == EIGHT), s.second, ": 8-bit operands and their scales belong together");
}
// the type of a product's results: 1 float16, 2 bfloat16, 0 not said
ScalarType result_type(const Tensor &x, PyObject *o) {
    const long said = PyLong_AsLong(o);
    const ScalarType type = said == TIRAMISU_HIP_FLOAT16 ? at::kHalf : at::kBFloat16;
    if (x.scalar_type() == EIGHT) return type;
    TORCH_CHECK_VALUE(said == 0 || type == x.scalar_type(), "results of 16-bit operands are of their type, ", name_of(x.scalar_type()));
    return x.scalar_type();
}
int64_t tokens_of(const Tensor &x) {
    int64_t n = 1;
    for (int64_t d = 0; d + 1 < x.dim(); d++) n *= x.size(d);
    return n;
}

// ---- results
Tensor new_like(const Tensor &x, int64_t columns, ScalarType type) {
    c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = columns;
    return at::empty(shape, x.options().dtype(type).requires_grad(false));
}
Tensor new_of_rows(const Tensor &x) { return at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat).requires_grad(false)); }
Tensor new_of(const Tensor &x, at::IntArrayRef shape) { return at::empty(shape, x.options().requires_grad(false)); }
// Several results in one piece of memory, each at a multiple of 256 bytes: one allocation, and no dispatch for each of them (a route's five: 8.4 us a call as
// tensors of their own, 5.4 so).
class results {
public:
    int add(at::IntArrayRef shape, ScalarType type) {
        int64_t n = 1;
        for (int64_t d : shape) n *= d;
        const int64_t bytes = n * (int64_t)c10::elementSize(type);
        wanted.push_back({c10::SmallVector<int64_t, 6>(shape.begin(), shape.end()), type, total});
        total += (bytes + 255) / 256 * 256;
        return (int)wanted.size() - 1;
    }
    void allocate(const Tensor &like) {
        c10::Allocator *const allocator = c10::GetAllocator(c10::DeviceType::CUDA);
        c10::DataPtr memory = allocator->allocate(total);
        memory.unsafe_set_device(like.device());           // (the allocator names the device as HIP's, tensors as torch's)
        storage = c10::Storage(c10::Storage::use_byte_size_t(), total, std::move(memory), allocator, false);
    }
    Tensor at(int i) const {
        const result &r = wanted[i];
        Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(r.type));
        t.unsafeGetTensorImpl()->set_sizes_contiguous(r.shape);
        t.unsafeGetTensorImpl()->set_storage_offset(r.first / (int64_t)c10::elementSize(r.type));
        return t;
    }

private:
    struct result { c10::SmallVector<int64_t, 6> shape; ScalarType type; int64_t first; };
    c10::SmallVector<result, 5> wanted;
    int64_t total = 0;
    c10::Storage storage;
};
PyObject *tuple_of(std::initializer_list<Tensor> tensors) {                 // undefined ones become None
    PyObject *t = PyTuple_New((Py_ssize_t)tensors.size());
    Py_ssize_t i = 0;
    for (const Tensor &r : tensors) {
        if (!r.defined()) Py_INCREF(Py_None);
        PyTuple_SET_ITEM(t, i++, r.defined() ? THPVariable_Wrap(r) : Py_None);
    }
    return t;
}
void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// The thread's stream of the runtime while a call lasts, torch's current one of the tensors' GPU, which is the current device meanwhile; and its scratch,
// torch's memory: in the stream's order like any tensor's, a recording's own in a graph, and an exception of torch's where there is none left.
class on_stream_of {
public:
    explicit on_stream_of(const Tensor &x) : guard(x.device()), before(tiramisu_hip_get_stream()) {
        void *const handle = (void *)c10::hip::getCurrentHIPStream(x.get_device()).stream();
        // torch's default stream is HIP's null stream; its handle, null, means the thread's own stream to the runtime
        tiramisu_hip_set_stream(handle ? handle : tiramisu_hip_null_stream());
        tiramisu_hip_exchange_scratch_source(&source);
    }
    ~on_stream_of() {
        tiramisu_hip_exchange_scratch_source(&source);
        tiramisu_hip_set_stream(before);
    }
    on_stream_of(const on_stream_of &) = delete;
    void accepted(int status) const {
        if (failure) std::rethrow_exception(failure);
        TORCH_CHECK(status == 0, "the runtime refused the call (its reason is on stderr)");
    }

private:
    static void *take(uint64_t bytes, void *self) {
        on_stream_of &call = *(on_stream_of *)self;
        try {
            // (the allocator itself: as a tensor, half a microsecond more; a norm's backward pass of few rows takes 9.5)
            call.scratch = c10::GetAllocator(c10::DeviceType::CUDA)->allocate(bytes);
            return call.scratch.get();
        } catch (...) {
            call.failure = std::current_exception();
            return nullptr;
        }
    }
    c10::DeviceGuard guard;
    void *before;
    c10::DataPtr scratch;
    std::exception_ptr failure;
    tiramisu_hip_scratch_source source = {take, this};
};
void count(Py_ssize_t n, Py_ssize_t expected) { TORCH_CHECK_TYPE(n == expected, expected, " arguments, not ", n); }

// ---- the operators
// x, weight, residual, eps, eight_bit, keep_rstd -> y, sum (None: x), scale, rstd
PyObject *rms_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 6);
    const Tensor x = tensor_of(a[0], "x");
    const device_rows r = rows_of(x, "x", NORM_TYPES);
    const ScalarType type = x.scalar_type();
    const void *const weight = vector_of(a[1], "weight", r.width, type, x);
    device_rows residual = {0, 0, 0, nullptr};
    if (given(a[2])) residual = rows_like(a[2], "residual", x, r.width, type);
    const double eps = PyFloat_AsDouble(a[3]);
    if (eps == -1.0 && PyErr_Occurred()) throw python_error();
    const bool eight = PyObject_IsTrue(a[4]) == 1, keep = PyObject_IsTrue(a[5]) == 1;
    const Tensor y = new_like(x, r.width, eight ? EIGHT : type), sum = given(a[2]) ? new_like(x, r.width, type) : Tensor();
    const Tensor scale = eight ? new_of_rows(x) : Tensor(), rstd = keep ? new_of_rows(x) : Tensor();
    {
        on_stream_of stream(x);
        // (a residual of no rows may have no address)
        stream.accepted(tiramisu_hip_rms_norm(r.p, residual.p, weight, address(y), residual.p ? address(sum) : nullptr, (float *)address(scale), (float *)address(rstd), r.rows, r.width, r.step,
                                              residual.step, (float)eps, element_of(type), element_of(y.scalar_type())));
    }
    return tuple_of({y, sum, scale, rstd});
    END_HANDLE_TH_ERRORS
}

// dy, sum, weight, rstd, dsum -> dx, dweight
PyObject *rms_norm_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 5);
    const Tensor sum = tensor_of(a[1], "sum");
    const device_rows s = rows_of(sum, "sum", NORM_TYPES);
    const ScalarType type = sum.scalar_type();
    const device_rows dy = rows_like(a[0], "dy", sum, s.width, type);
    const void *const weight = vector_of(a[2], "weight", s.width, type, sum);
    const float *const rstd = row_numbers(a[3], "rstd", sum, s.rows);
    device_rows dsum = {0, 0, 0, nullptr};
    if (given(a[4])) dsum = rows_like(a[4], "dsum", sum, s.width, type);
    const Tensor dx = new_like(sum, s.width, type), dweight = new_of(sum, {s.width});
    {
        on_stream_of stream(sum);
        stream.accepted(tiramisu_hip_rms_norm_backward(dy.p, s.p, weight, rstd, dsum.p, address(dx), address(dweight), s.rows, s.width, dy.step, s.step, dsum.step, element_of(type)));
    }
    return tuple_of({dx, dweight});
    END_HANDLE_TH_ERRORS
}

// x -> q, scale
PyObject *quantize_rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 1);
    const Tensor x = tensor_of(a[0], "x");
    const device_rows r = rows_of(x, "x", NORM_TYPES);
    const Tensor q = new_like(x, r.width, EIGHT), scale = new_of_rows(x);
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_quantize_rows(r.p, address(q), (float *)address(scale), r.rows, r.width, r.step, element_of(x.scalar_type())));
    }
    return tuple_of({q, scale});
    END_HANDLE_TH_ERRORS
}

// x, weight, bias, residual, activation, x_scale, weight_scale, type, keep_pre -> y, pre
PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 9);
    const Tensor x = tensor_of(a[0], "x");
    const device_rows r = rows_of(x, "x", PRODUCT_TYPES);
    int64_t outputs;
    const device_rows weight = matrix_of(a[1], "weight", -1, r.width, x, &outputs);
    const ScalarType type = result_type(x, a[7]);
    with_scales(x, {{a[5], "x_scale"}, {a[6], "weight_scale"}});
    const int64_t tokens = tokens_of(x);
    const float *const x_scale = given(a[5]) ? row_numbers(a[5], "x_scale", x, tokens) : nullptr;
    const float *const weight_scale = given(a[6]) ? (const float *)vector_of(a[6], "weight_scale", outputs, at::kFloat, x) : nullptr;
    const void *const bias = given(a[2]) ? vector_of(a[2], "bias", outputs, type, x) : nullptr;
    device_rows residual = {0, 0, 0, nullptr};
    if (given(a[3])) residual = rows_like(a[3], "residual", x, outputs, type);
    const Tensor y = new_like(x, outputs, type), pre = PyObject_IsTrue(a[8]) == 1 ? new_like(x, outputs, type) : Tensor();
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_linear(r.p, weight.p, bias, residual.p, x_scale, weight_scale, address(y), address(pre), tokens, outputs, r.width, r.step, weight.step, residual.step,
                                            activation_of(a[4]), element_of(x.scalar_type()), element_of(type)));
    }
    return tuple_of({y, pre});
    END_HANDLE_TH_ERRORS
}

// dy, x, weight, pre, activation, bias -> dx, dweight, dbias
PyObject *linear_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 6);
    const Tensor x = tensor_of(a[1], "x");
    const device_rows r = rows_of(x, "x", HALVES);
    const ScalarType type = x.scalar_type();
    int64_t outputs;
    const device_rows weight = matrix_of(a[2], "weight", -1, r.width, x, &outputs);
    const device_rows dy = rows_like(a[0], "dy", x, outputs, type);
    const int activation = activation_of(a[4]);
    TORCH_CHECK_VALUE(given(a[3]) == (activation != 0), "pre: an activation and the sums ahead of it belong together");
    device_rows pre = {0, 0, 0, nullptr};
    if (given(a[3])) pre = rows_like(a[3], "pre", x, outputs, type);
    const int64_t tokens = tokens_of(x);
    const Tensor dx = new_like(x, r.width, type), dweight = new_of(x, {outputs, r.width}), dbias = PyObject_IsTrue(a[5]) == 1 ? new_of(x, {outputs}) : Tensor();
    {
        on_stream_of stream(x);
        // (pre of no tokens has no address, and there is nothing to do with it)
        stream.accepted(tiramisu_hip_linear_backward(dy.p, r.p, weight.p, pre.p, address(dx), address(dweight), address(dbias), tokens, outputs, r.width, dy.step, r.step, weight.step, pre.step,
                                                     pre.p ? activation : 0, element_of(type)));
    }
    return tuple_of({dx, dweight, dbias});
    END_HANDLE_TH_ERRORS
}

// x, gate_weight, up_weight, activation, x_scale, gate_scale, up_scale, type, keep_pre -> h, gate, up
PyObject *gated_linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 9);
    const Tensor x = tensor_of(a[0], "x");
    const device_rows r = rows_of(x, "x", PRODUCT_TYPES);
    int64_t outputs;
    const device_rows gate_weight = matrix_of(a[1], "gate_weight", -1, r.width, x, &outputs), up_weight = matrix_of(a[2], "up_weight", outputs, r.width, x);
    const ScalarType type = result_type(x, a[7]);
    with_scales(x, {{a[4], "x_scale"}, {a[5], "gate_scale"}, {a[6], "up_scale"}});
    const int64_t tokens = tokens_of(x);
    const float *const x_scale = given(a[4]) ? row_numbers(a[4], "x_scale", x, tokens) : nullptr;
    const float *const gate_scale = given(a[5]) ? (const float *)vector_of(a[5], "gate_scale", outputs, at::kFloat, x) : nullptr;
    const float *const up_scale = given(a[6]) ? (const float *)vector_of(a[6], "up_scale", outputs, at::kFloat, x) : nullptr;
    const bool keep = PyObject_IsTrue(a[8]) == 1;
    const Tensor h = new_like(x, outputs, type), gate = keep ? new_like(x, outputs, type) : Tensor(), up = keep ? new_like(x, outputs, type) : Tensor();
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_gated_linear(r.p, gate_weight.p, up_weight.p, x_scale, gate_scale, up_scale, address(h), address(gate), address(up), tokens, outputs, r.width, r.step,
                                                  gate_weight.step, up_weight.step, activation_of(a[3]), element_of(x.scalar_type()), element_of(type)));
    }
    return tuple_of({h, gate, up});
    END_HANDLE_TH_ERRORS
}

// dh, x, gate_weight, up_weight, gate, up, activation -> dx, dgate_weight, dup_weight
PyObject *gated_linear_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 7);
    const Tensor x = tensor_of(a[1], "x");
    const device_rows r = rows_of(x, "x", HALVES);
    const ScalarType type = x.scalar_type();
    int64_t outputs;
    const device_rows gate_weight = matrix_of(a[2], "gate_weight", -1, r.width, x, &outputs), up_weight = matrix_of(a[3], "up_weight", outputs, r.width, x);
    const device_rows dh = rows_like(a[0], "dh", x, outputs, type), gate = rows_like(a[4], "gate", x, outputs, type), up = rows_like(a[5], "up", x, outputs, type);
    const Tensor dx = new_like(x, r.width, type), dgate = new_of(x, {outputs, r.width}), dup = new_of(x, {outputs, r.width});
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_gated_linear_backward(dh.p, r.p, gate_weight.p, up_weight.p, gate.p, up.p, address(dx), address(dgate), address(dup), tokens_of(x), outputs, r.width, dh.step,
                                                           r.step, gate_weight.step, up_weight.step, gate.step, up.step, activation_of(a[6]), element_of(type)));
    }
    return tuple_of({dx, dgate, dup});
    END_HANDLE_TH_ERRORS
}

// ---- rows grouped by expert
// 32-bit numbers, dense
Tensor ints_of(PyObject *o, const char *name, const Tensor &x) {
    const Tensor t = tensor_of(o, name);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.is_cuda() && t.is_contiguous(), name, " holds dense ", name_of(at::kInt), " on the GPU, not ", name_of(t.scalar_type()), " of ", t.sizes(),
                      " on ", t.device());
    TORCH_CHECK_VALUE(t.device() == x.device(), name, " lives on another GPU");
    return t;
}
const int32_t *ints(const Tensor &t) { return t.defined() ? (const int32_t *)t.data_ptr() : nullptr; }
std::string shape_of(at::IntArrayRef leading, const std::string &last) {
    std::string s = "[";
    for (int64_t n : leading) s += std::to_string(n) + ", ";
    return s + last + "]";
}
// [groups, outputs, columns], groups one below the other; outputs < 0: any number
device_rows weights_of(PyObject *o, const char *name, int64_t groups, int64_t outputs, int64_t columns, const Tensor &x, ScalarType type, int64_t *found = nullptr) {
    const Tensor t = tensor_of(o, name);
    TORCH_CHECK_VALUE(t.dim() == 3 && t.size(0) == groups && (outputs < 0 || t.size(1) == outputs) && t.size(2) == columns, name, " holds matrices, [", groups, ", ",
                      outputs < 0 ? std::string("outputs") : std::to_string(outputs), ", ", columns, "], not ", t.sizes());
    if (found) *found = t.size(1);
    return rows_of(t, name, {type}, &x);
}
const float *group_scales_of(PyObject *o, const char *name, int64_t groups, int64_t outputs, const Tensor &x) {
    const Tensor t = tensor_of(o, name);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) == groups && t.size(1) == outputs && t.is_cuda() && t.is_contiguous(), name, " is dense, [", groups, ", ", outputs, "] of ",
                      name_of(at::kFloat), " on the GPU, not ", name_of(t.scalar_type()), " of ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == x.device(), name, " lives on another GPU");
    return (const float *)t.data_ptr();
}
// What places there are, of how many groups, and which rows of x they take
struct grouping {
    Tensor offsets, rows;
    int64_t groups, places;
};
grouping grouping_of(PyObject *offsets, PyObject *rows, const Tensor &x, int64_t x_rows) {
    grouping g = {ints_of(offsets, "offsets", x), Tensor(), 0, x_rows};
    TORCH_CHECK_VALUE(g.offsets.dim() == 1 && g.offsets.size(0) >= 2, "offsets are those of the groups and the end, [groups + 1], not ", g.offsets.sizes());
    g.groups = g.offsets.size(0) - 1;
    if (given(rows)) {
        g.rows = ints_of(rows, "rows", x);
        TORCH_CHECK_VALUE(g.rows.dim() == 1, "rows are one number for each place, not ", g.rows.sizes());
        g.places = g.rows.size(0);
    }
    return g;
}
device_rows places_of(PyObject *o, const char *name, int64_t places, int64_t columns, const Tensor &x) {
    const Tensor t = tensor_of(o, name);
    TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == places && (columns < 0 || t.size(1) == columns), name, " holds a row for each place, [", places, ", ",
                      columns < 0 ? std::string("columns") : std::to_string(columns), "], not ", t.sizes());
    return rows_of(t, name, {x.scalar_type()}, &x);
}
Tensor new_of(const Tensor &x, at::IntArrayRef shape, ScalarType type) { return at::empty(shape, x.options().dtype(type).requires_grad(false)); }

// logits, k, normalise -> experts, weights, offsets, rows, places
PyObject *route(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 3);
    const Tensor logits = tensor_of(a[0], "logits");
    const device_rows r = rows_of(logits, "logits", NORM_TYPES);
    const int64_t k = PyLong_AsLongLong(a[1]);
    if (k == -1 && PyErr_Occurred()) throw python_error();
    TORCH_CHECK_VALUE(r.width >= 1 && r.width <= 1024, "logits of ", r.width, " experts: 1 to 1024");
    TORCH_CHECK_VALUE(k >= 1 && k <= r.width && k <= 16, "k of ", k, ": 1 to 16, of ", r.width, " experts");
    TORCH_CHECK_VALUE(r.rows <= 1 << 24, r.rows, " tokens: at most 2^24");
    c10::SmallVector<int64_t, 6> shape(logits.sizes().begin(), logits.sizes().end());
    shape.back() = k;
    results all;
    const int of[] = {all.add(shape, at::kInt), all.add(shape, at::kFloat), all.add({r.width + 1}, at::kInt), all.add({r.rows * k}, at::kInt), all.add(shape, at::kInt)};
    Tensor experts, weights, offsets, rows, places;
    {
        on_stream_of stream(logits);
        all.allocate(logits);
        experts = all.at(of[0]), weights = all.at(of[1]), offsets = all.at(of[2]), rows = all.at(of[3]), places = all.at(of[4]);
        stream.accepted(tiramisu_hip_route(r.p, (int32_t *)address(experts), (float *)address(weights), (int32_t *)address(offsets), (int32_t *)address(rows), (int32_t *)address(places), r.rows, r.width,
                                           k, r.step, PyObject_IsTrue(a[2]) == 1, element_of(logits.scalar_type())));
    }
    return tuple_of({experts, weights, offsets, rows, places});
    END_HANDLE_TH_ERRORS
}

// the choices of x's rows: [..., k] of ints or floats
Tensor choices_of(PyObject *o, const char *name, const Tensor &x, int64_t k, ScalarType type) {
    const Tensor t = tensor_of(o, name);
    bool same = t.dim() == x.dim() && t.scalar_type() == type && t.is_cuda() && t.is_contiguous() && (k < 0 || t.size(t.dim() - 1) == k);
    for (int64_t d = 0; same && d + 1 < x.dim(); d++) same = t.size(d) == x.size(d);
    TORCH_CHECK_VALUE(same, name, " is dense, ", shape_of(x.sizes().slice(0, x.dim() - 1), k < 0 ? "k" : std::to_string(k)), " of ", name_of(type), " on the GPU, not ", name_of(t.scalar_type()), " of ",
                      t.sizes());
    TORCH_CHECK_VALUE(t.device() == x.device(), name, " lives on another GPU");
    return t;
}

// dweights, logits, experts, normalise -> dlogits
PyObject *route_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 4);
    const Tensor logits = tensor_of(a[1], "logits");
    const device_rows r = rows_of(logits, "logits", NORM_TYPES);
    const Tensor experts = choices_of(a[2], "experts", logits, -1, at::kInt);
    const int64_t k = experts.size(experts.dim() - 1);
    const Tensor dweights = choices_of(a[0], "dweights", logits, k, at::kFloat), dlogits = new_like(logits, r.width, logits.scalar_type());
    TORCH_CHECK_VALUE(r.width >= 1 && r.width <= 1024, "logits of ", r.width, " experts: 1 to 1024");
    TORCH_CHECK_VALUE(k >= 1 && k <= r.width && k <= 16, "k of ", k, ": 1 to 16, of ", r.width, " experts");
    {
        on_stream_of stream(logits);
        stream.accepted(tiramisu_hip_route_backward((const float *)address(dweights), r.p, ints(experts), address(dlogits), r.rows, r.width, k, r.step, PyObject_IsTrue(a[3]) == 1,
                                                    element_of(logits.scalar_type())));
    }
    return tuple_of({dlogits});
    END_HANDLE_TH_ERRORS
}

// x, weight, offsets, rows, x_scale, weight_scale, type -> y
PyObject *grouped_linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 7);
    const Tensor x = tensor_of(a[0], "x");
    const device_rows r = rows_of(x, "x", PRODUCT_TYPES);
    const grouping g = grouping_of(a[2], a[3], x, r.rows);
    int64_t outputs;
    const device_rows weight = weights_of(a[1], "weight", g.groups, -1, r.width, x, x.scalar_type(), &outputs);
    const ScalarType type = result_type(x, a[6]);
    with_scales(x, {{a[4], "x_scale"}, {a[5], "weight_scale"}});
    const float *const x_scale = given(a[4]) ? row_numbers(a[4], "x_scale", x, r.rows) : nullptr;
    const float *const weight_scale = given(a[5]) ? group_scales_of(a[5], "weight_scale", g.groups, outputs, x) : nullptr;
    const Tensor y = new_of(x, {g.places, outputs}, type);
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_grouped_linear(r.p, weight.p, ints(g.offsets), ints(g.rows), x_scale, weight_scale, address(y), g.places, r.rows, g.groups, outputs, r.width, r.step, weight.step,
                                                    element_of(x.scalar_type()), element_of(type)));
    }
    return tuple_of({y});
    END_HANDLE_TH_ERRORS
}

// dy, x, weight, offsets, rows -> dx, dweight
PyObject *grouped_linear_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 5);
    const Tensor x = tensor_of(a[1], "x");
    const device_rows r = rows_of(x, "x", HALVES);
    const ScalarType type = x.scalar_type();
    const grouping g = grouping_of(a[3], a[4], x, r.rows);
    int64_t outputs;
    const device_rows weight = weights_of(a[2], "weight", g.groups, -1, r.width, x, type, &outputs), dy = places_of(a[0], "dy", g.places, outputs, x);
    const Tensor dx = new_of(x, {g.places, r.width}, type), dweight = new_of(x, {g.groups, outputs, r.width}, type);
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_grouped_linear_backward(dy.p, r.p, weight.p, ints(g.offsets), ints(g.rows), address(dx), address(dweight), g.places, r.rows, g.groups, outputs, r.width, dy.step,
                                                             r.step, weight.step, element_of(type)));
    }
    return tuple_of({dx, dweight});
    END_HANDLE_TH_ERRORS
}

// x, gate_weight, up_weight, offsets, rows, activation, x_scale, gate_scale, up_scale, type, keep_pre -> h, gate, up
PyObject *grouped_gated_linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 11);
    const Tensor x = tensor_of(a[0], "x");
    const device_rows r = rows_of(x, "x", PRODUCT_TYPES);
    const grouping g = grouping_of(a[3], a[4], x, r.rows);
    int64_t outputs;
    const device_rows gate_weight = weights_of(a[1], "gate_weight", g.groups, -1, r.width, x, x.scalar_type(), &outputs),
                      up_weight = weights_of(a[2], "up_weight", g.groups, outputs, r.width, x, x.scalar_type());
    const ScalarType type = result_type(x, a[9]);
    with_scales(x, {{a[6], "x_scale"}, {a[7], "gate_scale"}, {a[8], "up_scale"}});
    const float *const x_scale = given(a[6]) ? row_numbers(a[6], "x_scale", x, r.rows) : nullptr;
    const float *const gate_scale = given(a[7]) ? group_scales_of(a[7], "gate_scale", g.groups, outputs, x) : nullptr;
    const float *const up_scale = given(a[8]) ? group_scales_of(a[8], "up_scale", g.groups, outputs, x) : nullptr;
    const bool keep = PyObject_IsTrue(a[10]) == 1;
    const Tensor h = new_of(x, {g.places, outputs}, type), gate = keep ? new_of(x, {g.places, outputs}, type) : Tensor(), up = keep ? new_of(x, {g.places, outputs}, type) : Tensor();
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_grouped_gated_linear(r.p, gate_weight.p, up_weight.p, ints(g.offsets), ints(g.rows), x_scale, gate_scale, up_scale, address(h), address(gate), address(up), g.places,
                                                          r.rows, g.groups, outputs, r.width, r.step, gate_weight.step, up_weight.step, activation_of(a[5]), element_of(x.scalar_type()),
                                                          element_of(type)));
    }
    return tuple_of({h, gate, up});
    END_HANDLE_TH_ERRORS
}

// dh, x, gate_weight, up_weight, gate, up, offsets, rows, activation -> dx, dgate_weight, dup_weight
PyObject *grouped_gated_linear_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 9);
    const Tensor x = tensor_of(a[1], "x");
    const device_rows r = rows_of(x, "x", HALVES);
    const ScalarType type = x.scalar_type();
    const grouping g = grouping_of(a[6], a[7], x, r.rows);
    int64_t outputs;
    const device_rows gate_weight = weights_of(a[2], "gate_weight", g.groups, -1, r.width, x, type, &outputs), up_weight = weights_of(a[3], "up_weight", g.groups, outputs, r.width, x, type);
    const device_rows dh = places_of(a[0], "dh", g.places, outputs, x), gate = places_of(a[4], "gate", g.places, outputs, x), up = places_of(a[5], "up", g.places, outputs, x);
    const Tensor dx = new_of(x, {g.places, r.width}, type), dgate = new_of(x, {g.groups, outputs, r.width}, type), dup = new_of(x, {g.groups, outputs, r.width}, type);
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_grouped_gated_linear_backward(dh.p, r.p, gate_weight.p, up_weight.p, gate.p, up.p, ints(g.offsets), ints(g.rows), address(dx), address(dgate), address(dup), g.places,
                                                                   r.rows, g.groups, outputs, r.width, dh.step, r.step, gate_weight.step, up_weight.step, gate.step, up.step, activation_of(a[8]),
                                                                   element_of(type)));
    }
    return tuple_of({dx, dgate, dup});
    END_HANDLE_TH_ERRORS
}

// x, places, weights, residual -> y
PyObject *combine(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 4);
    const Tensor x = tensor_of(a[0], "x");
    const device_rows r = rows_of(x, "x", HALVES);
    TORCH_CHECK_VALUE(x.dim() == 2, "x holds a row for each place, [places, columns], not ", x.sizes());
    const Tensor places = ints_of(a[1], "places", x);
    TORCH_CHECK_VALUE(places.dim() >= 1, "places are a token's, [..., k], not ", places.sizes());
    const int64_t k = places.size(places.dim() - 1);
    TORCH_CHECK_VALUE(k <= 1024, "places of ", k, " rows a token: at most 1024");
    const Tensor weights = given(a[2]) ? choices_of(a[2], "weights", places, k, at::kFloat) : Tensor();
    c10::SmallVector<int64_t, 6> shape(places.sizes().begin(), places.sizes().end());
    shape.back() = r.width;
    const Tensor y = new_of(x, shape, x.scalar_type());
    device_rows residual = {0, 0, 0, nullptr};
    if (given(a[3])) residual = rows_like(a[3], "residual", y, r.width, x.scalar_type());
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_combine_rows(r.p, ints(places), (const float *)address(weights), residual.p, address(y), tokens_of(places), k, r.rows, r.width, r.step, residual.step,
                                                  element_of(x.scalar_type())));
    }
    return tuple_of({y});
    END_HANDLE_TH_ERRORS
}

// dy, x, places, weights, rows -> dx, dweights
PyObject *combine_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 5);
    const Tensor x = tensor_of(a[1], "x");
    const device_rows r = rows_of(x, "x", HALVES);
    TORCH_CHECK_VALUE(x.dim() == 2, "x holds a row for each place, [places, columns], not ", x.sizes());
    const Tensor places = ints_of(a[2], "places", x), owners = ints_of(a[4], "rows", x);
    TORCH_CHECK_VALUE(places.dim() >= 1, "places are a token's, [..., k], not ", places.sizes());
    TORCH_CHECK_VALUE(owners.dim() == 1 && owners.size(0) == r.rows, "rows are the token of each place, [", r.rows, "], not ", owners.sizes());
    const int64_t k = places.size(places.dim() - 1);
    TORCH_CHECK_VALUE(k <= 1024, "places of ", k, " rows a token: at most 1024");
    const Tensor weights = given(a[3]) ? choices_of(a[3], "weights", places, k, at::kFloat) : Tensor();
    const device_rows dy = rows_like(a[0], "dy", places, r.width, x.scalar_type());
    const Tensor dx = new_of(x, {r.rows, r.width}, x.scalar_type()), dweights = weights.defined() ? at::empty_like(weights) : Tensor();
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_combine_rows_backward(dy.p, r.p, ints(places), ints(owners), (const float *)address(weights), address(dx), (float *)address(dweights), tokens_of(places), k, r.rows,
                                                           r.width, dy.step, r.step, element_of(x.scalar_type())));
    }
    return tuple_of({dx, dweights});
    END_HANDLE_TH_ERRORS
}

// ---- 4-bit weights
constexpr int64_t FOUR_BIT_GROUP = 32;
// x -> q, scale
PyObject *quantize_groups(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 1);
    const Tensor x = tensor_of(a[0], "x");
    const device_rows r = rows_of(x, "x", NORM_TYPES);
    const Tensor q = new_like(x, (r.width + 1) / 2, at::kByte), scale = new_like(x, (r.width + FOUR_BIT_GROUP - 1) / FOUR_BIT_GROUP, at::kByte);
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_quantize_groups(r.p, address(q), (uint8_t *)address(scale), r.rows, r.width, r.step, element_of(x.scalar_type())));
    }
    return tuple_of({q, scale});
    END_HANDLE_TH_ERRORS
}
// [outputs, columns] of bytes
device_rows bytes_of(PyObject *o, const char *name, int64_t outputs, int64_t columns, const Tensor &x, int64_t *found = nullptr) {
    const Tensor t = tensor_of(o, name);
    TORCH_CHECK_VALUE(t.dim() == 2 && (outputs < 0 || t.size(0) == outputs) && t.size(1) == columns, name, " holds bytes, [", outputs < 0 ? std::string("outputs") : std::to_string(outputs), ", ", columns,
                      "], not ", t.sizes());
    if (found) *found = t.size(0);
    return rows_of(t, name, {at::kByte}, &x);
}

// x, weight, weight_scale, bias, residual, activation -> y
PyObject *four_bit_linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 6);
    const Tensor x = tensor_of(a[0], "x");
    const device_rows r = rows_of(x, "x", HALVES);
    const ScalarType type = x.scalar_type();
    int64_t outputs;
    const device_rows weight = bytes_of(a[1], "weight", -1, (r.width + 1) / 2, x, &outputs);
    const device_rows scale = bytes_of(a[2], "weight_scale", outputs, (r.width + FOUR_BIT_GROUP - 1) / FOUR_BIT_GROUP, x);
    const void *const bias = given(a[3]) ? vector_of(a[3], "bias", outputs, type, x) : nullptr;
    device_rows residual = {0, 0, 0, nullptr};
    if (given(a[4])) residual = rows_like(a[4], "residual", x, outputs, type);
    const Tensor y = new_like(x, outputs, type);
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_four_bit_linear(r.p, weight.p, (const uint8_t *)scale.p, bias, residual.p, address(y), r.rows, outputs, r.width, r.step, weight.step, scale.step, residual.step,
                                                     activation_of(a[5]), element_of(type)));
    }
    return tuple_of({y});
    END_HANDLE_TH_ERRORS
}

// x, gate_weight, up_weight, gate_scale, up_scale, activation -> h
PyObject *four_bit_gated_linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 6);
    const Tensor x = tensor_of(a[0], "x");
    const device_rows r = rows_of(x, "x", HALVES);
    const ScalarType type = x.scalar_type();
    const int64_t groups = (r.width + FOUR_BIT_GROUP - 1) / FOUR_BIT_GROUP;
    int64_t outputs;
    const device_rows gate = bytes_of(a[1], "gate_weight", -1, (r.width + 1) / 2, x, &outputs), up = bytes_of(a[2], "up_weight", outputs, (r.width + 1) / 2, x);
    const device_rows gate_scale = bytes_of(a[3], "gate_scale", outputs, groups, x), up_scale = bytes_of(a[4], "up_scale", outputs, groups, x);
    const Tensor h = new_like(x, outputs, type);
    {
        on_stream_of stream(x);
        stream.accepted(tiramisu_hip_four_bit_gated_linear(r.p, gate.p, up.p, (const uint8_t *)gate_scale.p, (const uint8_t *)up_scale.p, address(h), r.rows, outputs, r.width, r.step, gate.step, up.step,
                                                           gate_scale.step, up_scale.step, activation_of(a[5]), element_of(type)));
    }
    return tuple_of({h});
    END_HANDLE_TH_ERRORS
}

#define OPERATOR(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {OPERATOR(rms_norm), OPERATOR(rms_norm_backward), OPERATOR(quantize_rows), OPERATOR(linear), OPERATOR(linear_backward),
                         OPERATOR(gated_linear), OPERATOR(gated_linear_backward), OPERATOR(route), OPERATOR(route_backward), OPERATOR(grouped_linear),
                         OPERATOR(grouped_linear_backward), OPERATOR(grouped_gated_linear), OPERATOR(grouped_gated_linear_backward), OPERATOR(combine), OPERATOR(combine_backward),
                         OPERATOR(quantize_groups), OPERATOR(four_bit_linear), OPERATOR(four_bit_gated_linear), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_operators", "The inner part of tiramisu_amd.operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_operators(void) { return PyModule_Create(&module); }
