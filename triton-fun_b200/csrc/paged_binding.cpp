// Native host path of the paged cache's and the rotary positions' launchers, part of the splat_host module.
//
// Unlike the functions of host_binding.cpp, which hand everything unusual to Python code, these are the whole host side: they check
// the operands, word the errors (ValueError, TypeError, RuntimeError for a status of the library) and call the C ABI.  Shapes, types and
// layouts are looked at before the device, so that a refusal does not need one.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/_make_dual.h>
#include <ATen/ops/_unpack_dual.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <optional>
#include <string>
#include <vector>

#include "splat_b200.h"
#include "paged_binding.h"

namespace {

decltype(&splat_paged_tables) g_tables;
decltype(&splat_rotary) g_rotary;
decltype(&splat_paged_attention_workspace) g_workspace;
decltype(&splat_paged_attention) g_attention;
decltype(&splat_status_string) g_status_string;
PyObject* g_prepare;          // splat_native: sets up a device's status word, or raises what an earlier kernel reported

struct Refused {              // a Python exception to be
    PyObject* type;
    std::string what;
};
struct PythonError {};        // a Python exception that is set
[[noreturn]] void refuse(std::string what) { throw Refused{PyExc_ValueError, std::move(what)}; }

struct Operand {
    const at::Tensor* t;
    const char* name;
    const at::Tensor* operator->() const { return t; }
};
Operand tensor(PyObject* o, const char* name, int64_t dims = -1) {
    if (o == nullptr || !THPVariable_Check(o)) throw Refused{PyExc_TypeError, std::string(name) + " must be a tensor"};
    const at::Tensor* t = &THPVariable_Unpack(o);
    if (t->layout() != at::kStrided) throw Refused{PyExc_TypeError, std::string(name) + " must be a strided tensor"};
    if (t->is_neg() || t->is_conj() || t->_is_zerotensor())        // (not what its memory holds)
        throw Refused{PyExc_TypeError, std::string(name) + " must hold its values in memory: see torch.resolve_neg and torch.clone"};
    if (dims >= 0 && t->dim() != dims) refuse(std::string(name) + " must be " + std::to_string(dims) + "-dimensional");
    return {t, name};
}
bool given(PyObject* o) { return o != nullptr && o != Py_None; }
int64_t integer(PyObject* o, const char* name, int64_t least, int64_t most = INT64_MAX) {
    const long long v = PyLong_Check(o) ? PyLong_AsLongLong(o) : [&] {
        PyObject* i = PyNumber_Index(o);
        if (i == nullptr) return -1LL;
        const long long x = PyLong_AsLongLong(i);
        Py_DECREF(i);
        return x;
    }();
    if (PyErr_Occurred()) throw PythonError{};
    if (v < least || v > most)
        refuse(std::string(name) + (v < least ? " must be at least " + std::to_string(least) : " must be at most " + std::to_string(most)));
    return v;
}
float number(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (PyErr_Occurred()) throw PythonError{};
    if (!std::isfinite(v) || !std::isfinite(static_cast<float>(v))) refuse(std::string(name) + " must be finite");
    return static_cast<float>(v);
}
int64_t same_size(int64_t a, int64_t b, const char* what) {
    if (a != b) refuse(std::string(what) + ": " + std::to_string(a) + " and " + std::to_string(b));
    return a;
}
int32_t element_type(const Operand& x) {
    switch (x->scalar_type()) {
        case at::kFloat: return SPLAT_F32;
        case at::kHalf: return SPLAT_F16;
        case at::kBFloat16: return SPLAT_BF16;
        default: throw Refused{PyExc_TypeError, std::string(x.name) + ": unsupported dtype; expected float32, float16 or bfloat16"};
    }
}
void like(const Operand& x, const Operand& y) {
    if (x->scalar_type() != y->scalar_type()) throw Refused{PyExc_TypeError, std::string(x.name) + " must have the dtype of " + y.name};
}
void of_type(const Operand& x, at::ScalarType type, const char* word) {
    if (x->scalar_type() != type) throw Refused{PyExc_TypeError, std::string(x.name) + " must be " + word};
}
void rows_contiguous(const Operand& x) {
    if (x->size(-1) > 1 && x->stride(-1) != 1) refuse(std::string(x.name) + ": the last dimension must be contiguous");
}
void contiguous(const Operand& x) {
    if (!x->is_contiguous()) refuse(std::string(x.name) + " must be contiguous");
}
// ---- memory that operands share.  Outputs may interleave with other operands (heads of a fused projection, K and V as halves of one array), so
// what counts is elements, not ranges.
struct Steps { int64_t stride, lo, hi; };     // d strides, for any lo <= d <= hi
// Whether a sum of d_k stride_k lies in [from, to]: steps in descending order of their strides (all above 0).  The steps of tensors, whose rows lie within
// one another, leave two d_k to try at most; where that does not hold and `tries` run out, the answer is yes.
bool reaches(const Steps* s, int n, int64_t from, int64_t to, int& tries) {
    if (--tries < 0) return true;
    int64_t lo = 0, hi = 0;                    // what the steps can add up to
    for (int i = 0; i < n; ++i) {
        lo += s[i].lo * s[i].stride;
        hi += s[i].hi * s[i].stride;
    }
    if (lo > to || hi < from) return false;
    if (n == 0) return true;
    lo -= s[0].lo * s[0].stride;
    hi -= s[0].hi * s[0].stride;
    auto floor_div = [](int64_t a, int64_t b) { return a >= 0 ? a / b : -((b - 1 - a) / b); };
    const int64_t first = std::max(s[0].lo, -floor_div(hi - from, s[0].stride)), last = std::min(s[0].hi, floor_div(to - lo, s[0].stride));
    for (int64_t d = first; d <= last; ++d)
        if (reaches(s + 1, n - 1, from - d * s[0].stride, to - d * s[0].stride, tries)) return true;
    return false;
}
constexpr int kMaxSteps = 8, kTries = 4096;
int add_steps(Steps* s, int n, const at::Tensor& t, int64_t sign) {
    const auto size = t.sizes(), steps = t.strides();
    const int64_t e = t.element_size();
    for (size_t i = 0; i < size.size(); ++i) {
        if (size[i] < 2 || steps[i] == 0) continue;
        const int64_t stride = steps[i] * e, far = size[i] - 1;
        int k = 0;
        while (k < n && s[k].stride != stride) ++k;
        if (k == n) s[n++] = {stride, 0, 0};
        (sign > 0 ? s[k].hi : s[k].lo) += sign * far;
    }
    return n;
}
void descending(Steps* s, int n) {
    std::sort(s, s + n, [](const Steps& a, const Steps& b) { return a.stride > b.stride; });
}
// no element twice in what is written
void no_overlap(const Operand& x) {
    const auto size = x->sizes(), steps = x->strides();
    const int64_t e = x->element_size();
    Steps s[kMaxSteps];
    int n = 0;
    for (size_t i = 0; i < size.size(); ++i) {
        if (size[i] < 2) continue;
        if (steps[i] == 0) refuse(std::string(x.name) + " must not be an expanded tensor");
        int k = n++;                           // (descending)
        for (; k > 0 && s[k - 1].stride < steps[i] * e; --k) s[k] = s[k - 1];
        s[k] = {steps[i] * e, 0, size[i] - 1};
    }
    int64_t inner = e;                         // bytes of the steps behind
    for (int k = n - 1; k >= 0; --k) {
        if (s[k].stride < inner) {             // two elements whose first difference is in step k
            Steps t[kMaxSteps] = {{s[k].stride, 1, s[k].hi}};
            for (int i = k + 1; i < n; ++i) t[i - k] = {s[i].stride, -s[i].hi, s[i].hi};
            int tries = kTries;
            if (reaches(t, n - k, -(e - 1), e - 1, tries)) refuse(std::string(x.name) + " must not overlap itself");
        }
        inner += s[k].hi * s[k].stride;
    }
}
struct Range { const char *begin, *end; };
Range range_of(const Operand& x) {
    if (x.t == nullptr || x->numel() == 0) return {nullptr, nullptr};
    const char* begin = static_cast<const char*>(x->const_data_ptr());
    if (begin == nullptr) return {nullptr, nullptr};
    const auto size = x->sizes(), steps = x->strides();
    int64_t far = 0;
    for (size_t i = 0; i < size.size(); ++i) far += (size[i] - 1) * steps[i];
    return {begin, begin + (far + 1) * static_cast<int64_t>(x->element_size())};
}
bool share_elements(const Operand& x, const Operand& y) {
    Steps s[kMaxSteps];
    const int n = add_steps(s, add_steps(s, 0, *x.t, 1), *y.t, -1);
    descending(s, n);
    const int64_t apart = static_cast<const char*>(x->const_data_ptr()) - static_cast<const char*>(y->const_data_ptr());
    int tries = kTries;
    return reaches(s, n, -(static_cast<int64_t>(x->element_size()) - 1) - apart, static_cast<int64_t>(y->element_size()) - 1 - apart, tries);
}
bool share(const Operand& x, const Range& rx, const Operand& y, const Range& ry) {
    return rx.begin < ry.end && ry.begin < rx.end && share_elements(x, y);
}
bool is_itself(const Operand& x, const Operand& y) {
    if (x->const_data_ptr() != y->const_data_ptr() || x->sizes() != y->sizes()) return false;
    for (int64_t i = 0; i < x->dim(); ++i)
        if (x->size(i) > 1 && x->stride(i) != y->stride(i)) return false;
    return true;
}
// Outputs (the first `outputs` of all; operands that are not there have no tensor) share memory with nobody, but where inputs[i] is given output i may be it.
template <int N> void apart(const Operand (&all)[N], int outputs, std::initializer_list<const Operand*> inputs = {}) {
    Range r[N];
    for (int i = 0; i < N; ++i) r[i] = range_of(all[i]);
    for (int i = 0; i < outputs; ++i) {
        const Operand* own = i < static_cast<int>(inputs.size()) ? inputs.begin()[i] : nullptr;
        for (int j = i + 1; j < N; ++j) {
            if (!share(all[i], r[i], all[j], r[j])) continue;
            if (own == nullptr || own->t != all[j].t) refuse(std::string(all[i].name) + " and " + all[j].name + " must not share memory");
            if (!is_itself(all[i], all[j])) refuse(std::string(all[i].name) + " must be " + all[j].name + " itself or not share memory with it");
        }
    }
}
int device_of(std::initializer_list<Operand> all) {
    const Operand* first = nullptr;
    for (const Operand& x : all) {
        if (x.t == nullptr) continue;
        if (!x->is_cuda())
            refuse(std::string(x.name) + " is on " + x->device().str() + ": this implementation runs on CUDA devices only (there is no CPU path)");
        if (first == nullptr) first = &x;
        else if (x->get_device() != (*first)->get_device()) refuse(std::string(x.name) + " and " + first->name + " are on different devices");
    }
    return (*first)->get_device();
}
void check(int32_t rc, const char* what) {
    if (rc != 0)
        throw Refused{PyExc_RuntimeError, std::string(what) + ": splat status " + std::to_string(rc) + " (" + g_status_string(rc) + ")"};
}
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }
template <class T> T* data(const Operand& x) { return static_cast<T*>(x->data_ptr()); }
void arguments(Py_ssize_t n, Py_ssize_t wanted) {
    if (g_tables == nullptr) throw Refused{PyExc_RuntimeError, "splat_host is not bound to the library"};
    if (n != wanted) throw Refused{PyExc_TypeError, "wrong number of arguments"};
}

// paged_tables(ctx_lens, q_lens, block_table, ring, span, page, kv_lens, q_start, slots, positions, requests, taken)
PyObject* paged_tables(PyObject* const* a, Py_ssize_t n) {
    arguments(n, 12);
    const Operand ctx = tensor(a[0], "ctx_lens", 1), fresh = tensor(a[1], "q_lens", 1), table = tensor(a[2], "block_table", 2),
                  ring = tensor(a[3], "free_pages", 1), span = tensor(a[4], "free_span", 1);
    const int64_t page = integer(a[5], "page_size", 1, 1 << 30);
    const Operand kv = tensor(a[6], "kv_lens", 1), start = tensor(a[7], "q_start", 1), slots = tensor(a[8], "slots", 1),
                  positions = tensor(a[9], "positions", 1), requests = tensor(a[10], "requests", 1), taken = tensor(a[11], "free_span_out", 1);
    for (const Operand* x : {&ctx, &fresh, &table, &ring, &kv, &start, &positions, &requests}) of_type(*x, at::kInt, "int32");
    for (const Operand* x : {&span, &slots, &taken}) of_type(*x, at::kLong, "int64");
    const int64_t B = ctx->size(0), T = slots->size(0);
    same_size(fresh->size(0), B, "q_lens and ctx_lens differ in length");
    same_size(kv->size(0), B, "kv_lens and ctx_lens differ in length");
    same_size(table->size(0), B, "block_table must have a row for each request");
    same_size(start->size(0), B + 1, "q_start must have one entry more than there are requests");
    same_size(positions->size(0), T, "positions and slots differ in length");
    same_size(requests->size(0), T, "requests and slots differ in length");
    same_size(span->size(0), 2, "free_span must have 2 entries");
    same_size(taken->size(0), 3, "free_span_out must have 3 entries");
    if (ring->size(0) < 1) refuse("free_pages must not be empty");
    if (B > SPLAT_PAGED_MAX_REQUESTS) refuse("at most " + std::to_string(SPLAT_PAGED_MAX_REQUESTS) + " requests");
    for (const Operand* x : {&ctx, &fresh, &ring, &span, &kv, &start, &slots, &positions, &requests, &taken}) contiguous(*x);
    rows_contiguous(table);
    if (B > 1 && table->stride(0) < table->size(1)) refuse("block_table: its rows must not overlap");
    apart<11>({table, kv, start, slots, positions, requests, taken, ctx, fresh, ring, span}, 7);
    const int dev = device_of({ctx, fresh, table, ring, span, kv, start, slots, positions, requests, taken});
    c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    check(g_tables(data<int32_t>(ctx), data<int32_t>(fresh), data<int32_t>(table), B > 1 ? table->stride(0) : table->size(1),
                   data<int32_t>(ring), ring->size(0), data<int64_t>(span), page, B, table->size(1), T, data<int32_t>(kv),
                   data<int32_t>(start), data<int64_t>(slots), data<int32_t>(positions), data<int32_t>(requests), data<int64_t>(taken),
                   stream_of(dev)),
          "splat_paged_tables");
    Py_RETURN_NONE;
}

// positions, inv_freq and sections, as the callers below take them
struct Turn {
    Operand positions{nullptr, nullptr}, inv_freq{nullptr, nullptr};
    int64_t half = 0, sections[SPLAT_ROTARY_MAX_AXES] = {}, axis = 0, b = 0, l = 0;
    int32_t axes = 0, wide = 0;
};
// a sequence of integers; none without one
std::vector<int64_t> sections_of(PyObject* sections) {
    std::vector<int64_t> out;
    if (!given(sections)) return out;
    PyObject* list = PySequence_Fast(sections, "sections must be a sequence of integers");
    if (list == nullptr) throw PythonError{};
    try {
        if (PySequence_Fast_GET_SIZE(list) < 1) refuse("sections must have an entry for each axis of positions");
        for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(list); ++i)
            out.push_back(integer(PySequence_Fast_GET_ITEM(list, i), "sections", 0, 1 << 30));
    } catch (...) {
        Py_DECREF(list);
        throw;
    }
    Py_DECREF(list);
    return out;
}
Turn turn_of(const Operand& positions, const Operand& inv_freq, const std::vector<int64_t>& sections, int64_t d, int64_t B, int64_t L, bool batched) {
    Turn t;
    t.positions = positions;
    t.inv_freq = inv_freq;
    if (t.positions->scalar_type() != at::kInt && t.positions->scalar_type() != at::kLong)
        throw Refused{PyExc_TypeError, "positions must be int32 or int64"};
    t.wide = t.positions->scalar_type() == at::kLong;
    of_type(t.inv_freq, at::kFloat, "float32");
    contiguous(t.inv_freq);
    const at::Tensor& p = *t.positions.t;
    const int64_t dims = p.dim();
    if (dims < 1 || dims > (batched ? 3 : 2))
        refuse(batched ? "positions must be (axes, B, L), (axes, L) or (L)" : "positions must be (axes, tokens) or (tokens)");
    same_size(p.size(dims - 1), L, "positions and tokens differ in length");
    if (dims == 3) same_size(p.size(1), B, "positions and operands differ in batch");
    const int64_t axes = dims > 1 ? p.size(0) : 1;
    if (axes < 1 || axes > SPLAT_ROTARY_MAX_AXES) refuse("positions must have 1 to " + std::to_string(SPLAT_ROTARY_MAX_AXES) + " axes");
    t.axes = static_cast<int32_t>(axes);
    t.axis = dims > 1 ? p.stride(0) : 0;
    t.b = dims == 3 ? p.stride(1) : 0;
    t.l = p.stride(dims - 1);
    t.half = t.inv_freq->size(0);
    if (2 * t.half > d) refuse("inv_freq has " + std::to_string(t.half) + " frequencies, but a row only " + std::to_string(d) + " elements");
    if (sections.empty()) {
        if (axes != 1) refuse("sections must be given for positions of several axes");
        t.sections[0] = t.half;
        return t;
    }
    same_size(static_cast<int64_t>(sections.size()), axes, "sections must have an entry for each axis of positions");
    int64_t sum = 0;
    for (int64_t i = 0; i < axes; ++i) sum += t.sections[i] = sections[i];
    same_size(sum, t.half, "sections must add up to the number of frequencies");
    return t;
}
int flag(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PythonError{};
    return v;
}

// q, k (or an operand without a tensor) turned into out, or into new tensors where out has none
void rotate(Operand (&in)[2], Operand (&out)[2], at::Tensor (&made)[2], const Operand& positions, const Operand& inv_freq,
            const std::vector<int64_t>& sections, int interleaved, int inverse) {
    static const char* const names[2] = {"q_out", "k_out"};
    const int count = in[1].t != nullptr ? 2 : 1;
    const int64_t B = in[0]->size(0), L = in[0]->size(2), d = in[0]->size(3);
    const int32_t type = element_type(in[0]);
    if (d < 1) refuse("q must have rows of at least one element");
    const Turn t = turn_of(positions, inv_freq, sections, d, B, L, true);
    for (int i = 0; i < count; ++i) {
        like(in[i], in[0]);
        if (in[i]->size(0) != B || in[i]->size(2) != L || in[i]->size(3) != d) refuse("k must agree with q in batch, length and head size");
        rows_contiguous(in[i]);
        if (out[i].t == nullptr) continue;
        like(out[i], in[0]);
        if (out[i]->sizes() != in[i]->sizes()) refuse(std::string(names[i]) + " must have the shape of its operand");
        rows_contiguous(out[i]);
        no_overlap(out[i]);
    }
    if (out[0].t != nullptr || out[1].t != nullptr) apart<6>({out[0], out[1], in[0], in[1], t.positions, t.inv_freq}, 2, {&in[0], &in[1]});
    const int dev = device_of({in[0], in[1], t.positions, t.inv_freq, out[0], out[1]});
    c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    splat_rows rows[2] = {};
    for (int i = 0; i < count; ++i) {
        if (out[i].t == nullptr) {
            made[i] = at::empty(in[i]->sizes(), in[i]->options());
            out[i] = {&made[i], names[i]};
        }
        const at::Tensor &x = *in[i].t, &y = *out[i].t;
        rows[i] = {x.const_data_ptr(), y.data_ptr(), x.size(1), x.stride(0), x.stride(1), x.stride(2), y.stride(0), y.stride(1), y.stride(2), 1, 0};
    }
    if (in[0]->numel() > 0 || (count == 2 && in[1]->numel() > 0))
        check(g_rotary(rows, count, t.positions->const_data_ptr(), t.wide, t.axis, t.b, t.l, data<float>(t.inv_freq), t.half, t.sections, t.axes,
                       interleaved, inverse, B, L, d, type, nullptr, 1, 0, stream_of(dev)),
              "splat_rotary");
}

PyObject* pair_of(PyObject* first, PyObject* second) {         // takes both
    PyObject* result = PyTuple_New(2);
    if (result == nullptr) throw PythonError{};
    PyTuple_SET_ITEM(result, 0, first);
    PyTuple_SET_ITEM(result, 1, second);
    return result;
}
PyObject* wrapped(const at::Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

// rotary(x, y or None, positions, inv_freq, sections, interleaved, inverse, out x or None, out y or None) -> (out x, out y or None)
// x, y: (B, H, L, d); without an output, a new contiguous tensor
PyObject* rotary(PyObject* const* a, Py_ssize_t n) {
    arguments(n, 9);
    Operand in[2] = {tensor(a[0], "q", 4), {nullptr, nullptr}}, out[2] = {{nullptr, nullptr}, {nullptr, nullptr}};
    at::Tensor made[2];
    if (given(a[1])) in[1] = tensor(a[1], "k", 4);
    if (given(a[7])) out[0] = tensor(a[7], "q_out", 4);
    if (given(a[8])) {
        if (in[1].t == nullptr) refuse("k_out without k");
        out[1] = tensor(a[8], "k_out", 4);
    }
    rotate(in, out, made, tensor(a[2], "positions"), tensor(a[3], "inv_freq", 1), sections_of(a[4]), flag(a[5]), flag(a[6]));
    PyObject* y[2];
    for (int i = 0; i < 2; ++i) {
        y[i] = given(a[7 + i]) ? a[7 + i] : nullptr;
        if (y[i] != nullptr) Py_INCREF(y[i]);
        else y[i] = wrapped(made[i]);
    }
    return pair_of(y[0], y[1]);
}

// A gradient or tangent that may be a view with its sign to be turned, or zeros without memory
at::Tensor in_memory(const at::Tensor& t) { return t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t.resolve_neg(); }

// The same with gradients: that of a rotation is the rotation by the opposite angle.  In native code, since the Python form of such a
// function takes as long as the kernels of ordinary calls do (fp32 B3 H12+4 L1369 d64, forward and backward: 97 us).
struct Rotary : torch::autograd::Function<Rotary> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const std::optional<at::Tensor>& k,
                                                  const at::Tensor& positions, const at::Tensor& inv_freq, std::vector<int64_t> sections,
                                                  bool interleaved, bool inverse) {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({positions, inv_freq});
        Operand in[2] = {{&q, "q"}, {nullptr, nullptr}}, out[2] = {{nullptr, nullptr}, {nullptr, nullptr}};
        if (k.has_value()) in[1] = {&*k, "k"};
        at::Tensor made[2];
        rotate(in, out, made, {&positions, "positions"}, {&inv_freq, "inv_freq"}, sections, interleaved, inverse);
        ctx->saved_data["sections"] = std::move(sections);
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        if (!k.has_value()) return {made[0]};
        return {made[0], made[1]};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        at::Tensor g[2], d[2];
        for (size_t i = 0; i < grads.size(); ++i) {
            g[i] = grads[i];                               // (may come expanded, as that of a sum, and with its sign to be turned)
            if (g[i].defined()) g[i] = in_memory(g[i]);
            if (g[i].defined() && g[i].size(-1) > 1 && g[i].stride(-1) != 1) g[i] = g[i].contiguous();
        }
        const int first = g[0].defined() ? 0 : 1;
        if (g[first].defined()) {
            try {
                const auto y = apply(g[first], first == 0 && g[1].defined() ? std::optional<at::Tensor>(g[1]) : std::nullopt, saved[0], saved[1],
                                     ctx->saved_data["sections"].toIntVector(), ctx->saved_data["interleaved"].toBool(),
                                     !ctx->saved_data["inverse"].toBool());
                for (size_t i = 0; i < y.size(); ++i) d[first + i] = y[i];
            } catch (const Refused& r) {                   // (in a thread of the engine, which knows torch's errors)
                TORCH_CHECK(false, r.what);
            }
        }
        return {d[0], d[1], at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

// q and k (if defined) turned into y, differentiable in both; the tangents of dual tensors (forward mode) are turned as they are
void turned(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions, const at::Tensor& inv_freq, const std::vector<int64_t>& sections,
            bool interleaved, at::Tensor (&y)[2]) {
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && (q._fw_grad(0).defined() || (k.defined() && k._fw_grad(0).defined()))) {
        at::Tensor x[2], t[2], dt[2];
        for (int i = 0; i < 2; ++i) {
            const at::Tensor& in = i == 0 ? q : k;
            if (!in.defined()) continue;
            std::tie(x[i], t[i]) = at::_unpack_dual(in, 0);
            if (t[i].defined()) t[i] = in_memory(t[i]);
        }
        turned(x[0], x[1], positions, inv_freq, sections, interleaved, y);
        if (t[0].defined()) turned(t[0], t[1], positions, inv_freq, sections, interleaved, dt);
        else turned(t[1], at::Tensor(), positions, inv_freq, sections, interleaved, dt);
        if (!t[0].defined()) std::swap(dt[0], dt[1]);
        for (int i = 0; i < 2; ++i)
            if (dt[i].defined()) y[i] = at::_make_dual(y[i], dt[i], 0);
        return;
    }
    if (at::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()))) {
        auto out = Rotary::apply(q, k.defined() ? std::optional<at::Tensor>(k) : std::nullopt, positions, inv_freq, sections, interleaved, false);
        for (size_t i = 0; i < out.size(); ++i) y[i] = std::move(out[i]);
        return;
    }
    Operand in[2] = {{&q, "q"}, {nullptr, nullptr}}, out[2] = {{nullptr, nullptr}, {nullptr, nullptr}};
    if (k.defined()) in[1] = {&k, "k"};
    rotate(in, out, y, {&positions, "positions"}, {&inv_freq, "inv_freq"}, sections, interleaved, 0);
}

// rotary_grad(q, k or None, positions, inv_freq, sections, interleaved) -> (q', k' or None), differentiable in q and k
PyObject* rotary_grad(PyObject* const* a, Py_ssize_t n) {
    arguments(n, 6);
    const Operand q = tensor(a[0], "q", 4);
    const at::Tensor none;
    Operand k{&none, "k"};
    if (given(a[1])) k = tensor(a[1], "k", 4);
    const Operand positions = tensor(a[2], "positions"), inv_freq = tensor(a[3], "inv_freq", 1);
    const std::vector<int64_t> sections = sections_of(a[4]);
    const int interleaved = flag(a[5]);
    if ((at::GradMode::is_enabled() && inv_freq->requires_grad()) ||
        (c10::AutogradState::get_tls_state().get_fw_grad_mode() && inv_freq->_fw_grad(0).defined()))
        refuse("inv_freq must not require a gradient: there is none for the frequencies");
    at::Tensor y[2];
    turned(*q.t, *k.t, *positions.t, *inv_freq.t, sections, interleaved != 0, y);
    return pair_of(wrapped(y[0]), wrapped(y[1]));
}

struct Cache { int64_t pages, heads, page; };
Cache cache_of(const Operand& k, const Operand& v, int64_t d) {
    if (k->sizes() != v->sizes()) refuse("k_cache and v_cache must have the same shape");
    same_size(k->size(3), d, "rows of the cache and of the operands differ in length");
    rows_contiguous(k);
    rows_contiguous(v);
    if (k->size(2) < 1) refuse("pages of the cache must have at least one row");
    return {k->size(0), k->size(1), k->size(2)};
}

// paged_append(q or None, k, v, k_cache, v_cache, slots, q_out or None, positions or None, inv_freq, sections, interleaved)
PyObject* paged_append(PyObject* const* a, Py_ssize_t n) {
    arguments(n, 11);
    const Operand k = tensor(a[1], "k", 3), v = tensor(a[2], "v", 3), kc = tensor(a[3], "k_cache", 4), vc = tensor(a[4], "v_cache", 4),
                  slots = tensor(a[5], "slots", 1);
    Operand q{nullptr, nullptr}, q_out{nullptr, nullptr};
    if (given(a[0])) {
        q = tensor(a[0], "q", 3);
        q_out = tensor(a[6], "q_out", 3);
    } else if (given(a[6])) {
        refuse("q_out without q");
    }
    const int64_t T = k->size(0), d = k->size(2);
    const int32_t type = element_type(k);
    if (d < 1) refuse("k must have rows of at least one element");
    if (k->sizes() != v->sizes()) refuse("k and v must have the same shape");
    const Cache c = cache_of(kc, vc, d);
    same_size(k->size(1), c.heads, "k and the cache differ in heads");
    same_size(slots->size(0), T, "slots and tokens differ in length");
    of_type(slots, at::kLong, "int64");
    contiguous(slots);
    for (const Operand* x : {&v, &kc, &vc}) like(*x, k);
    for (const Operand* x : {&k, &v}) rows_contiguous(*x);
    for (const Operand* x : {&kc, &vc}) no_overlap(*x);
    if (q.t != nullptr) {
        like(q, k);
        like(q_out, k);
        if (q->size(0) != T || q->size(2) != d) refuse("q and k differ in tokens or head size");
        if (q_out->sizes() != q->sizes()) refuse("q_out must have the shape of q");
        rows_contiguous(q);
        rows_contiguous(q_out);
        no_overlap(q_out);
    }
    Turn t;
    const bool turned = given(a[7]);
    if (turned) {
        if (!given(a[8])) refuse("positions without inv_freq");
        t = turn_of(tensor(a[7], "positions"), tensor(a[8], "inv_freq", 1), sections_of(a[9]), d, 1, T, false);
    } else if (given(a[8])) {
        refuse("inv_freq without positions");
    }
    const int interleaved = flag(a[10]);
    apart<9>({q_out, kc, vc, q, k, v, slots, t.positions, t.inv_freq}, 3, {&q});
    const int dev = device_of({k, v, kc, vc, slots, q, q_out, t.positions, t.inv_freq});
    c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    splat_rows rows[3] = {};
    int count = 0;
    if (q.t != nullptr)
        rows[count++] = {q->const_data_ptr(), q_out->data_ptr(), q->size(1), 0, q->stride(1), q->stride(0), 0, q_out->stride(1), q_out->stride(0), 1, 0};
    rows[count++] = {k->const_data_ptr(), kc->data_ptr(), c.heads, 0, k->stride(1), k->stride(0), kc->stride(0), kc->stride(1), kc->stride(2), 1, 1};
    rows[count++] = {v->const_data_ptr(), vc->data_ptr(), c.heads, 0, v->stride(1), v->stride(0), vc->stride(0), vc->stride(1), vc->stride(2), 0, 1};
    if (T > 0)
        check(g_rotary(rows, count, turned ? t.positions->const_data_ptr() : nullptr, t.wide, t.axis, 0, t.l,
                       turned ? data<float>(t.inv_freq) : nullptr, t.half, t.sections, t.axes, interleaved, 0, 1, T, d, type,
                       data<int64_t>(slots), c.page, c.pages, stream_of(dev)),
              "splat_rotary");
    Py_RETURN_NONE;
}

// paged_attention(q, k_cache, v_cache, block_table, kv_lens, out, q_start or None, max_q_len or None, scale, taps, stride, softcap,
//                 slopes or None, lse or None)
PyObject* paged_attention(PyObject* const* a, Py_ssize_t n) {
    arguments(n, 14);
    const Operand q = tensor(a[0], "q", 3), kc = tensor(a[1], "k_cache", 4), vc = tensor(a[2], "v_cache", 4), table = tensor(a[3], "block_table", 2),
                  kv = tensor(a[4], "kv_lens", 1), out = tensor(a[5], "output", 3);
    Operand start{nullptr, nullptr}, slopes{nullptr, nullptr}, lse{nullptr, nullptr};
    const int64_t T = q->size(0), H = q->size(1), d = q->size(2), B = kv->size(0);
    splat_paged_args x = {};
    x.dtype = element_type(q);
    if (d < 1 || d > 256) refuse("the head size must be 1 to 256");
    if (H < 1) refuse("q must have at least one head");
    const Cache c = cache_of(kc, vc, d);
    for (const Operand* y : {&kc, &vc, &out}) like(*y, q);
    if (c.heads < 1 || H % c.heads != 0) refuse("the number of heads must be a multiple of the cache's");
    if (out->sizes() != q->sizes()) refuse("output must have the shape of q");
    rows_contiguous(q);
    contiguous(out);
    of_type(table, at::kInt, "int32");
    of_type(kv, at::kInt, "int32");
    contiguous(kv);
    rows_contiguous(table);
    same_size(table->size(0), B, "block_table must have a row for each request");
    if (B > SPLAT_PAGED_MAX_REQUESTS) refuse("at most " + std::to_string(SPLAT_PAGED_MAX_REQUESTS) + " requests");
    if (given(a[6])) {
        start = tensor(a[6], "q_start", 1);
        of_type(start, at::kInt, "int32");
        contiguous(start);
        same_size(start->size(0), B + 1, "q_start must have one entry more than there are requests");
    } else {
        same_size(T, B, "without q_start there must be one token for each request");
    }
    x.max_q_len = given(a[7]) ? integer(a[7], "max_q_len", 0) : start.t != nullptr ? T : 1;
    x.scale = number(a[8], "scale");
    x.taps = integer(a[9], "taps", 0);
    x.stride = integer(a[10], "stride", 1);
    x.softcap = number(a[11], "softcap");
    if (x.softcap < 0.f) refuse("softcap must not be negative");
    if (x.softcap > 0.f && !std::isfinite(x.scale / x.softcap)) refuse("softcap is too small for the scale");
    // (scores are held in powers of two: log2 e and twice of it are in front of them)
    if (std::abs(x.scale) > 2e38f) refuse("scale must be at most 2e38");
    if (x.softcap > 1e38f || (x.softcap > 0.f && x.scale != 0.f && std::abs(x.scale / x.softcap) < 1.2e-38f))
        refuse("softcap is too large for the scale: it caps nothing, leave it out");
    if (given(a[12])) {
        slopes = tensor(a[12], "slopes", 1);
        of_type(slopes, at::kFloat, "float32");
        contiguous(slopes);
        same_size(slopes->size(0), H, "slopes must have an entry for each head");
    }
    if (given(a[13])) {
        lse = tensor(a[13], "lse", 2);
        of_type(lse, at::kFloat, "float32");
        contiguous(lse);
        if (lse->size(0) != T || lse->size(1) != H) refuse("lse must have shape (tokens, heads)");
    }
    if (c.pages > INT32_MAX || table->size(1) > (1 << 30) / c.page || T >= (1 << 30) / H)
        refuse("pages, tokens of a request or tokens times heads beyond what the kernels count (2^31, 2^30)");
    apart<9>({out, lse, q, kc, vc, table, kv, start, slopes}, 2);
    const int dev = device_of({q, kc, vc, table, kv, out, start, slopes, lse});
    if (T == 0 || B == 0) Py_RETURN_NONE;
    c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    if (x.dtype != SPLAT_F32) {
        if (!splat_host::status_ready(dev)) {      // first call on the device, or a report of an earlier kernel
            PyObject* r = PyObject_CallFunction(g_prepare, "i", dev);
            if (r == nullptr) throw PythonError{};
            Py_DECREF(r);
        }
        x.status_word = splat_host::status_word(dev);
    }
    x.q = q->const_data_ptr(); x.k_cache = kc->const_data_ptr(); x.v_cache = vc->const_data_ptr();
    x.o = out->data_ptr();
    x.lse = lse.t != nullptr ? data<float>(lse) : nullptr;
    x.q_row = q->stride(0); x.q_head = q->stride(1); x.o_row = out->stride(0); x.o_head = out->stride(1);
    x.k_page = kc->stride(0); x.k_head = kc->stride(1); x.k_row = kc->stride(2);
    x.v_page = vc->stride(0); x.v_head = vc->stride(1); x.v_row = vc->stride(2);
    x.block_table = data<int32_t>(table);
    x.table_stride = B > 1 ? table->stride(0) : table->size(1);
    x.table_width = table->size(1);
    x.kv_lens = data<int32_t>(kv);
    x.q_start = start.t != nullptr ? data<int32_t>(start) : nullptr;
    x.slopes = slopes.t != nullptr ? data<float>(slopes) : nullptr;
    x.tokens = T; x.requests = B; x.pages = c.pages; x.page = c.page; x.heads = H; x.kv_heads = c.heads; x.d = d;
    if (B > 1 && x.table_stride < x.table_width) {           // (an expanded table: every request has the same row)
        refuse("block_table: its rows must not overlap");
    }
    // Scratch of this call alone, from torch's allocator: calls on other streams and captured graphs have their own
    x.workspace_bytes = g_workspace(&x);
    const at::Tensor workspace = at::empty({x.workspace_bytes}, q->options().dtype(at::kByte));
    x.workspace = workspace.data_ptr();
    check(g_attention(&x, stream_of(dev)), "splat_paged_attention");
    Py_RETURN_NONE;
}

// Errors of the functions above as Python exceptions
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)> PyObject* worded(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        return F(a, n);
    } catch (const Refused& r) {
        PyErr_SetString(r.type, r.what.c_str());
        return nullptr;
    } catch (const PythonError&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// bind_paged(tables, rotary, workspace, attention, status_string, prepare)
PyObject* bind_paged(PyObject*, PyObject* args) {
    unsigned long long f[5];
    PyObject* prepare;
    if (!PyArg_ParseTuple(args, "KKKKKO", f, f + 1, f + 2, f + 3, f + 4, &prepare)) return nullptr;
    g_tables = reinterpret_cast<decltype(g_tables)>(f[0]);
    g_rotary = reinterpret_cast<decltype(g_rotary)>(f[1]);
    g_workspace = reinterpret_cast<decltype(g_workspace)>(f[2]);
    g_attention = reinterpret_cast<decltype(g_attention)>(f[3]);
    g_status_string = reinterpret_cast<decltype(g_status_string)>(f[4]);
    Py_INCREF(prepare);
    Py_XDECREF(g_prepare);
    g_prepare = prepare;
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)> PyCFunction method() {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(worded<F>));
}
PyMethodDef methods[] = {{"bind_paged", bind_paged, METH_VARARGS, nullptr},
                         {"paged_tables", method<paged_tables>(), METH_FASTCALL, nullptr},
                         {"rotary", method<rotary>(), METH_FASTCALL, nullptr},
                         {"rotary_grad", method<rotary_grad>(), METH_FASTCALL, nullptr},
                         {"paged_append", method<paged_append>(), METH_FASTCALL, nullptr},
                         {"paged_attention", method<paged_attention>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

}  // namespace

namespace splat_host {
PyMethodDef* paged_methods() { return methods; }
}  // namespace splat_host
