// Host side of the many-tensor operators and of the embedding lookup (Python module _fgs_host): reads tensors, checks
// them and calls the C entry points of libfgs_b200.so, whose addresses `bind` receives. A step over 300 tensors reads
// and checks some 2000 tensor properties, at about 75 ns each through Python attributes; the lookup's backward runs on
// autograd's thread without the interpreter. Everything is read anew at every call.
#include <Python.h>
#include <algorithm>
#include <exception>
#include <stdexcept>
#include <string>
#include <vector>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include "../../include/fgs_b200.h"

namespace {

constexpr int64_t kBlock = FGS_ADAMW_BLOCK;

struct Entries {
    decltype(&fgs_last_error) last_error;
    decltype(&fgs_adamw_step) adamw_step;
    decltype(&fgs_grad_squares_capacity) grad_squares_capacity;
    decltype(&fgs_grad_squares) grad_squares;
    decltype(&fgs_adamw_read_moments) read_moments;
    decltype(&fgs_embedding_lookup) lookup;
    decltype(&fgs_embedding_workspace_bytes) workspace_bytes;
    decltype(&fgs_embedding_grad) lookup_grad;
} lib;

[[noreturn]] void refuse(const std::string& why) { throw std::runtime_error(why); }

void check(int rc) {
    if (rc != FGS_OK) refuse(lib.last_error());
}

// Python objects that belong to this scope
struct Ref {
    PyObject* p;
    explicit Ref(PyObject* o = nullptr) : p(o) {}
    Ref(const Ref&) = delete;
    ~Ref() { Py_XDECREF(p); }
};

struct PythonError {};  // the interpreter's error is set

// Looks parameters up in the optimizer's state dict. It is in the parameters' order as a rule, so the entry behind the
// last one is tried first, by identity: a lookup hashes the tensor, which calls into the interpreter.
struct StateCursor {
    PyObject* dict;
    Py_ssize_t at = 0;
    PyObject* find(PyObject* param) {
        PyObject *key, *value;
        Py_ssize_t next = at;
        if (PyDict_Next(dict, &next, &key, &value) && key == param) {
            at = next;
            return value;
        }
        value = PyDict_GetItemWithError(dict, param);
        if (!value && PyErr_Occurred()) throw PythonError();
        return value;
    }
};

PyObject* must(PyObject* o) {
    if (!o) throw PythonError();
    return o;
}

// Runs f() for Python: every C++ exception becomes a Python one, as torch translates its own (out of memory, and what a
// Python hook raised below, which torch.utils.checkpoint needs back as it was).
template <typename F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const PythonError&) {
        return nullptr;
    } catch (const std::length_error& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

enum { kU8 = 3 };
const char* kTypeNames[] = {"float32", "bfloat16", "float16", "uint8"};

int type_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return FGS_DTYPE_F32;
        case at::kBFloat16: return FGS_DTYPE_BF16;
        case at::kHalf: return FGS_DTYPE_F16;
        case at::kByte: return kU8;
        default: return -1;
    }
}

// The kernels work on memory, past torch's dispatcher: whatever records calls there would see an allocation and none of the
// writes to it, and give uninitialised memory when it is run again.
void refuse_recorded(const char* what) {
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Key = c10::impl::TorchDispatchModeKey;
    if (torch::jit::tracer::isTracing()) refuse(std::string(what) + " cannot be traced by torch.jit.trace");
    if (!Modes::any_modes_set()) return;
    for (const Key k : {Key::FAKE, Key::PROXY, Key::FUNCTIONAL})
        if (Modes::get_mode(k).has_value()) refuse(std::string(what) + " cannot be traced by torch.fx or run on fake tensors");
}

// refuses tensors that do not own their value's memory: fake ones, wrappers of function transforms, other subclasses that
// dispatch to Python
constexpr c10::DispatchKeySet kWrapped({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                        c10::DispatchKey::Functionalize, c10::DispatchKey::ZeroTensor});
void refuse_wrapped(const at::Tensor& t, const char* name) {
    if (t.key_set().has_any(kWrapped)) refuse(std::string(name) + " must be a plain tensor: fake tensors and tensors of function transforms have no memory");
}

// Refuses tensors whose storage has been freed or shrunk beneath them (resize_, as sharded training does between its uses):
// their address would be no null pointer, but their place within nothing.
void refuse_unbacked(const at::Tensor& t, const char* name) {
    int64_t last = t.storage_offset() + t.numel() - 1;
    if (!t.is_contiguous()) {
        last = t.storage_offset();
        for (int64_t d = 0; d < t.dim(); d++) last += (t.size(d) - 1) * t.stride(d);
    }
    if (t.numel() > 0 && t.storage().nbytes() < static_cast<size_t>(last + 1) * t.element_size())
        refuse(std::string(name) + " has less memory than elements: its storage was resized");
}

// says what keeps `address` from taking a tensor
[[noreturn]] __attribute__((noinline)) void refuse_tensor(const at::Tensor& t, const char* name, int code, int64_t count, int device) {
    refuse_wrapped(t, name);
    if (t.is_neg()) refuse(std::string(name) + " must not be a lazily negated view: its memory holds the negative");
    if (t.layout() != at::kStrided || type_code(t) != code || !t.is_contiguous())
        refuse(std::string(name) + " must be a contiguous " + kTypeNames[code] + " tensor");
    refuse_unbacked(t, name);
    if (!t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
    if (t.get_device() != device) refuse(std::string(name) + " must be on device cuda:" + std::to_string(device) + " like the others");
    refuse(std::string(name) + " has " + std::to_string(t.numel()) + " elements, expected " + std::to_string(count));
}

// Data address of a contiguous CUDA tensor of the given type and element count on `device` (-1: any, and sets it). Some 2700
// calls per step over 300 tensors with its moments read, so one test of everything: the host's work of step and reading on one
// core takes 92 and 84 us (113 and 108 with one test after the other).
void* address(const at::Tensor& t, const char* name, int code, int64_t count, int& device) {
    constexpr at::ScalarType types[] = {at::kFloat, at::kBFloat16, at::kHalf, at::kByte};
    constexpr uint64_t bytes[] = {4, 2, 2, 1};
    constexpr c10::DispatchKeySet odd = kWrapped | c10::DispatchKeySet({c10::DispatchKey::Negative});
    const c10::TensorImpl& i = *t.unsafeGetTensorImpl();
    if (i.key_set().has_any(odd) || i.layout() != at::kStrided || i.dtype() != types[code] || !i.is_contiguous() || !i.is_cuda() ||
        (i.get_device() != device && device >= 0) || i.numel() != count ||
        (count > 0 && i.unsafe_storage().nbytes() < static_cast<uint64_t>(i.storage_offset() + count) * bytes[code]))
        refuse_tensor(t, name, code, count, device < 0 ? 0 : device);
    device = i.get_device();
    return t.data_ptr();
}

const at::Tensor& tensor_of(PyObject* o, const char* name) {
    if (!o || !(THPVariable_CheckExact(o) || THPVariable_Check(o))) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

// Tells autograd of a change in place: a graph that saved the tensor before raises an error in its backward.
void changed(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// names of the state and of the group options, made once
struct Names {
    PyObject *params, *lr, *betas, *eps, *weight_decay, *state_bits, *master_weights, *step, *exp_avg, *exp_avg_sq, *exp_avg_exponent,
        *exp_avg_sq_exponent, *master, *maximize, *amsgrad, *differentiable, *decoupled_weight_decay, *grad_norm;
} names;

const at::Tensor& state_tensor(PyObject* state, PyObject* key) {
    PyObject* o = PyDict_GetItemWithError(state, key);
    if (!o) refuse(std::string("the optimizer state has no ") + PyUnicode_AsUTF8(key) + ": it was made with other state_bits or master_weights");
    if (!THPVariable_CheckExact(o)) tensor_of(o, PyUnicode_AsUTF8(key));
    return THPVariable_Unpack(o);
}

double number(PyObject* o) {
    const double x = PyFloat_AsDouble(must(o));
    if (x == -1.0 && PyErr_Occurred()) throw PythonError();
    return x;
}

PyObject* option(PyObject* group, PyObject* key) {
    PyObject* o = PyDict_GetItemWithError(group, key);
    if (!o) refuse(std::string("a parameter group has no ") + PyUnicode_AsUTF8(key));
    return o;
}

// truth of a group's option, `otherwise` where it has none
bool is_set(PyObject* group, PyObject* key, bool otherwise) {
    PyObject* o = PyDict_GetItemWithError(group, key);
    const int set = o ? PyObject_IsTrue(o) : otherwise;
    if (set < 0 || (!o && PyErr_Occurred())) throw PythonError();
    return set;
}

// options of torch's Adams that a step cannot follow (adamw.py refuses them where groups are made and loaded)
void refuse_options(PyObject* group) {
    for (PyObject* name : {names.maximize, names.amsgrad, names.differentiable})
        if (is_set(group, name, false)) refuse(std::string(PyUnicode_AsUTF8(name)) + " is not supported");
    if (!is_set(group, names.decoupled_weight_decay, true) && number(option(group, names.weight_decay)) != 0.0)
        refuse("weight decay is always decoupled: that of Adam (decoupled_weight_decay=False) is not supported");
}

fgs_adamw_hyper hyper_of(PyObject* group, int64_t step) {
    fgs_adamw_hyper h{};
    PyObject* lr = option(group, names.lr);
    if (PyList_Check(lr) || PyTuple_Check(lr)) {
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(lr);
        if (n < 1 || n > 7) refuse("between 1 and 7 learning rates are supported");
        for (Py_ssize_t i = 0; i < n; i++) h.learning_rates[i] = number(PySequence_Fast_GET_ITEM(lr, i));
        h.n_learning_rates = static_cast<int32_t>(n);
    } else {
        h.learning_rates[0] = number(lr);
        h.n_learning_rates = 1;
    }
    Ref b1(must(PySequence_GetItem(option(group, names.betas), 0))), b2(must(PySequence_GetItem(option(group, names.betas), 1)));
    h.beta1 = number(b1.p);
    h.beta2 = number(b2.p);
    h.eps = number(option(group, names.eps));
    h.weight_decay = number(option(group, names.weight_decay));
    // as fgs_adamw_step, which would come to it behind the launches of the norm and of other types
    if (!(h.beta1 >= 0.0 && h.beta1 < 1.0 && h.beta2 >= 0.0 && h.beta2 < 1.0)) refuse("betas must be in [0, 1)");
    if (!(h.eps >= 0.0) || (h.eps > 0.0 && h.eps < 1.2e-38)) refuse("eps must be zero or a normal float (at least 1.2e-38)");
    h.step = step;
    return h;
}

// tensors of one call of the kernel: one type, one kind of state
struct Job {
    std::vector<void*> param, exp_avg, exp_avg_sq;
    std::vector<const void*> grad;
    std::vector<uint8_t*> exp_avg_exponent, exp_avg_sq_exponent;
    std::vector<float*> master;
    std::vector<int64_t> count;
    std::vector<int32_t> hyper;
    void expect(size_t n) {  // room for the rest of a group (300 tensors: 9 us of the step's host work)
        for (auto* v : {&param, &exp_avg, &exp_avg_sq}) v->reserve(n);
        grad.reserve(n);
        count.reserve(n);
        hyper.reserve(n);
    }
};

// a parameter without state, which is made once nothing can be refused any more
struct Fresh {
    Job* job;
    size_t at;
    PyObject* param;  // borrowed
    int bits;
    bool master;
};

// places the addresses of a parameter's state as tensor `at` of a job
void place_state(Job& job, size_t at, PyObject* state, int bits, bool master, int& device) {
    const int64_t n = job.count[at], blocks = (n + kBlock - 1) / kBlock;
    const int kind = bits == 8 ? kU8 : FGS_DTYPE_F32;
    job.exp_avg[at] = address(state_tensor(state, names.exp_avg), "exp_avg", kind, n, device);
    job.exp_avg_sq[at] = address(state_tensor(state, names.exp_avg_sq), "exp_avg_sq", kind, n, device);
    if (bits == 8) {
        job.exp_avg_exponent[at] = static_cast<uint8_t*>(address(state_tensor(state, names.exp_avg_exponent), "exp_avg_exponent", kU8, blocks, device));
        job.exp_avg_sq_exponent[at] =
            static_cast<uint8_t*>(address(state_tensor(state, names.exp_avg_sq_exponent), "exp_avg_sq_exponent", kU8, blocks, device));
    }
    if (master) job.master[at] = static_cast<float*>(address(state_tensor(state, names.master), "master", FGS_DTYPE_F32, n, device));
}

// Address ranges that a kernel writes by different threads: refused if two overlap. 300 of them are sorted in some 5 us, of
// a step whose kernels take 100 and more.
struct Written {
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    void add(const void* a, int64_t count, int code) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(a);
        if (count > 0) spans.emplace_back(at, at + static_cast<uintptr_t>(count) * (code == FGS_DTYPE_F32 ? 4 : 2));
    }
    void refuse_shared(const char* why) {
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); i++)
            if (spans[i].first < spans[i - 1].second) refuse(why);
    }
};

// adamw_step(state dict, parameter groups, new_state(parameter, bits, master), max_grad_norm or None[, optimizer]) -> the norm
// or None; it also becomes the optimizer's grad_norm. (Set from here: torch.compile, which leaves this call out of its graphs,
// fails on an attribute of an optimizer that is set between them.)
PyObject* adamw_step(PyObject*, PyObject* args) {
    PyObject *all_state, *groups, *new_state, *limit, *optimizer = nullptr;
    if (!PyArg_ParseTuple(args, "O!O!OO|O", &PyDict_Type, &all_state, &PyList_Type, &groups, &new_state, &limit, &optimizer)) return nullptr;
    const auto done = [&](PyObject* norm) {
        Ref n(must(norm));
        if (optimizer && PyObject_SetAttr(optimizer, names.grad_norm, n.p)) throw PythonError();
        Py_INCREF(n.p);
        return n.p;
    };
    return guarded([&]() -> PyObject* {
        refuse_recorded("FusedAdamW.step");
        const double max_norm = limit == Py_None ? 0.0 : number(limit);
        if (limit != Py_None && !(max_norm > 0.0)) refuse("max_grad_norm must be positive (or None for no clipping)");
        Job jobs[3][2][2];
        StateCursor states{all_state};
        std::vector<fgs_adamw_hyper> hypers;
        std::vector<Py_ssize_t> hyper_group;
        std::vector<std::pair<PyObject*, int64_t>> counted;  // states and their new step counts (borrowed)
        std::vector<PyObject*> updated;                      // borrowed
        Written params_written;
        std::vector<Fresh> fresh;
        int device = -1;
        bool any = false;
        for (Py_ssize_t gi = 0; gi < PyList_GET_SIZE(groups); gi++) {
            PyObject* group = PyList_GET_ITEM(groups, gi);
            if (!PyDict_Check(group)) refuse("parameter groups must be dicts");
            PyObject* params = option(group, names.params);
            if (!PyList_Check(params)) refuse("a group's parameters must be a list");
            const long bits = PyLong_AsLong(option(group, names.state_bits));
            if (bits != 8 && bits != 32) {
                PyErr_Clear();
                refuse("state_bits must be 8 or 32");
            }
            refuse_options(group);
            const int wants_master = PyObject_IsTrue(option(group, names.master_weights));
            for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); i++) {
                PyObject* o = PyList_GET_ITEM(params, i);
                const at::Tensor& p = tensor_of(o, "a parameter");
                const at::Tensor& g = p.grad();
                if (!g.defined()) continue;
                any = true;
                const int code = type_code(p);
                if (code < 0 || code > FGS_DTYPE_F16) refuse("parameters must be float32, bfloat16 or float16 tensors");
                const bool eight = bits == 8, master = wants_master && code != FGS_DTYPE_F32;
                Job& job = jobs[code][eight][master];
                const int64_t n = p.numel();
                if (job.count.empty()) job.expect(static_cast<size_t>(PyList_GET_SIZE(params) - i));
                job.param.push_back(address(p, "a parameter", code, n, device));
                job.grad.push_back(address(g, "a gradient", code, n, device));
                job.count.push_back(n);
                const size_t at = job.count.size() - 1;
                job.exp_avg.push_back(nullptr);
                job.exp_avg_sq.push_back(nullptr);
                if (eight) {
                    job.exp_avg_exponent.push_back(nullptr);
                    job.exp_avg_sq_exponent.push_back(nullptr);
                }
                if (master) job.master.push_back(nullptr);
                PyObject* state = states.find(o);
                int64_t t = 1;
                if (!state || (PyDict_Check(state) && PyDict_GET_SIZE(state) == 0)) {
                    fresh.push_back({&job, at, o, static_cast<int>(bits), master});
                } else {
                    if (!PyDict_Check(state)) refuse("the optimizer state of a parameter must be a dict");
                    PyObject* was = PyDict_GetItemWithError(state, names.step);
                    if (!was) refuse("the optimizer state has no step");
                    Ref whole(must(PyNumber_Long(was)));
                    t = PyLong_AsLongLong(whole.p) + 1;
                    if (t < 1) {
                        PyErr_Clear();
                        refuse("step must not be negative");
                    }
                    place_state(job, at, state, static_cast<int>(bits), master, device);
                    counted.emplace_back(state, t);
                }
                updated.push_back(o);
                params_written.add(job.param.back(), n, code);
                size_t h = hypers.size();
                while (h > 0 && hyper_group[h - 1] == gi && hypers[h - 1].step != t) h--;
                if (h == 0 || hyper_group[h - 1] != gi) {
                    hypers.push_back(hyper_of(group, t));
                    hyper_group.push_back(gi);
                    h = hypers.size();
                }
                job.hyper.push_back(static_cast<int32_t>(h - 1));
            }
        }
        if (!any) return done(Py_NewRef(Py_None));
        params_written.refuse_shared("two parameters share memory (or one is in the groups twice)");
        const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
        if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
            refuse("FusedAdamW.step cannot be captured into a CUDA graph: its step count is a host value");
        Ref made(must(PyList_New(0)));  // the states of `fresh`
        for (const Fresh& f : fresh) {
            Ref state(must(PyObject_CallFunction(new_state, "Oii", f.param, f.bits, static_cast<int>(f.master))));
            if (PyList_Append(made.p, state.p)) throw PythonError();  // the list keeps it
            if (!PyDict_Check(state.p)) refuse("the optimizer state of a parameter must be a dict");
            place_state(*f.job, f.at, state.p, f.bits, f.master, device);
            counted.emplace_back(state.p, 1);
        }
        const cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
        at::Tensor norm, partials;
        int n_partials = 0;
        if (max_norm > 0.0) {
            const auto on = at::TensorOptions().device(at::kCUDA, static_cast<c10::DeviceIndex>(device));
            int room = 0;
            for (auto& by_type : jobs)
                for (auto& by_bits : by_type)
                    for (Job& j : by_bits) {
                        int need = 0;
                        check(lib.grad_squares_capacity(static_cast<int64_t>(j.count.size()), &need));
                        room += need;
                    }
            partials = at::empty({room}, on.dtype(at::kDouble));
            norm = at::empty({}, on.dtype(at::kFloat));
            double* to = partials.data_ptr<double>();
            for (int code = 0; code < 3; code++)
                for (auto& by_bits : jobs[code])
                    for (Job& j : by_bits) {
                        if (j.count.empty()) continue;
                        int used = 0;
                        const std::vector<uint8_t> types(j.count.size(), static_cast<uint8_t>(code));
                        check(lib.grad_squares(j.grad.data(), j.count.data(), types.data(), static_cast<int64_t>(j.count.size()), to + n_partials,
                                               room - n_partials, &used, stream));
                        n_partials += used;
                    }
            if (n_partials == 0) norm.zero_();  // empty gradients only: no kernel writes the norm
        }
        for (int code = 0; code < 3; code++)
            for (int eight = 0; eight < 2; eight++)
                for (int master = 0; master < 2; master++) {
                    Job& j = jobs[code][eight][master];
                    if (j.count.empty()) continue;
                    const fgs_adamw_tensors t{static_cast<int64_t>(j.count.size()), j.param.data(), j.grad.data(), j.exp_avg.data(), j.exp_avg_sq.data(),
                                              eight ? j.exp_avg_exponent.data() : nullptr, eight ? j.exp_avg_sq_exponent.data() : nullptr,
                                              master ? j.master.data() : nullptr, j.count.data(), j.hyper.data()};
                    check(lib.adamw_step(&t, hypers.data(), static_cast<int>(hypers.size()), code, eight ? 8 : 32,
                                         n_partials ? partials.data_ptr<double>() : nullptr, n_partials, max_norm,
                                         n_partials ? norm.data_ptr<float>() : nullptr, stream));
                }
        for (PyObject* o : updated) changed(THPVariable_Unpack(o));
        for (size_t i = 0; i < fresh.size(); i++)
            if (PyDict_SetItem(all_state, fresh[i].param, PyList_GET_ITEM(made.p, static_cast<Py_ssize_t>(i)))) throw PythonError();
        Ref count;  // most parameters have the same step count
        int64_t counts = -1;
        for (const auto& c : counted) {
            if (c.second != counts) {
                Py_XDECREF(count.p);
                count.p = nullptr;
                count.p = must(PyLong_FromLongLong(counts = c.second));
            }
            if (PyDict_SetItem(c.first, names.step, count.p)) throw PythonError();
        }
        return done(norm.defined() ? THPVariable_Wrap(norm) : Py_NewRef(Py_None));
    });
}

// read_moments(state dict, parameters, outputs of exp_avg, outputs of exp_avg_sq)
PyObject* read_moments(PyObject*, PyObject* args) {
    PyObject *all_state, *params, *outs[2];
    if (!PyArg_ParseTuple(args, "O!O!O!O!", &PyDict_Type, &all_state, &PyList_Type, &params, &PyList_Type, &outs[0], &PyList_Type, &outs[1]))
        return nullptr;
    return guarded([&]() -> PyObject* {
        refuse_recorded("FusedAdamW.read_moments");
        const Py_ssize_t n = PyList_GET_SIZE(params);
        if (PyList_GET_SIZE(outs[0]) != n || PyList_GET_SIZE(outs[1]) != n) refuse("one tensor per parameter is needed");
        const at::NoGradGuard no_graph;
        std::vector<const uint8_t*> codes, exponents;
        std::vector<void*> to;
        std::vector<uint8_t> is_signed;
        std::vector<int64_t> counts;
        int device = -1, out_code = -1;
        StateCursor states{all_state};
        Written written;
        written.spans.reserve(2 * n);
        std::vector<std::pair<at::Tensor, at::Tensor>> copies;  // moments in 32 bits; an undefined source: zeros
        for (Py_ssize_t i = 0; i < n; i++) {
            PyObject* o = PyList_GET_ITEM(params, i);
            const int64_t count = tensor_of(o, "a parameter").numel();
            PyObject* state = states.find(o);
            const bool none = !state || !PyDict_Check(state) || PyDict_GET_SIZE(state) == 0;
            for (int k = 0; k < 2; k++) {
                const at::Tensor& out = tensor_of(PyList_GET_ITEM(outs[k], i), "an output");
                if (out_code < 0) out_code = type_code(out);
                if (out_code != FGS_DTYPE_F32 && out_code != FGS_DTYPE_BF16) refuse("moments are read as float32 or bfloat16");
                if (out.numel() != count) throw std::length_error("moments must be read into tensors of the size of their parameter");
                void* at_out = address(out, "an output", out_code, count, device);
                written.add(at_out, count, out_code);
                if (none) {
                    copies.emplace_back(out, at::Tensor());
                    continue;
                }
                const at::Tensor& m = state_tensor(state, k ? names.exp_avg_sq : names.exp_avg);
                if (m.scalar_type() != at::kByte) {
                    address(m, "a moment", FGS_DTYPE_F32, count, device);
                    copies.emplace_back(out, m);
                    continue;
                }
                codes.push_back(static_cast<const uint8_t*>(address(m, "a moment", kU8, count, device)));
                exponents.push_back(static_cast<const uint8_t*>(address(state_tensor(state, k ? names.exp_avg_sq_exponent : names.exp_avg_exponent),
                                                                        "an exponent", kU8, (count + kBlock - 1) / kBlock, device)));
                to.push_back(at_out);
                is_signed.push_back(k == 0);
                counts.push_back(count);
            }
        }
        if (device < 0) Py_RETURN_NONE;
        written.refuse_shared("two tensors to read moments into share memory");
        const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
        for (auto& c : copies) {
            if (c.second.defined()) c.first.copy_(c.second.view(c.first.sizes()));
            else c.first.zero_();
        }
        check(lib.read_moments(codes.data(), exponents.data(), is_signed.data(), counts.data(), static_cast<int64_t>(codes.size()), to.data(), out_code,
                               c10::cuda::getCurrentCUDAStream().stream()));
        for (PyObject* list : outs)
            for (Py_ssize_t i = 0; i < n; i++) changed(THPVariable_Unpack(PyList_GET_ITEM(list, i)));
        Py_RETURN_NONE;
    });
}

// ---------------------------------------------------------------------------------------------------
// embedding lookup

// a contiguous tensor whose memory holds its values (each of torch's calls costs some 0.1 us even where it has nothing to do)
at::Tensor settled(const at::Tensor& t) {
    const at::Tensor c = t.is_contiguous() ? t : t.contiguous();
    return c.is_neg() ? c.resolve_neg() : c;
}

at::Tensor lookup(const at::Tensor& table, const at::Tensor& indices, double scale, int64_t padding) {
    const c10::cuda::CUDAGuard guard(table.device());
    const at::Tensor negated = table.is_neg() ? table.detach().resolve_neg() : at::Tensor();
    const at::Tensor& values = negated.defined() ? negated : table;
    std::vector<int64_t> shape = indices.sizes().vec();
    int64_t width = 1;
    for (int64_t d = 1; d < table.dim(); d++) {
        shape.push_back(table.size(d));
        width *= table.size(d);
    }
    at::Tensor out = at::empty(shape, table.options().requires_grad(false));
    refuse_wrapped(out, "the output");
    check(lib.lookup(values.data_ptr(), table.size(0), width, type_code(table), indices.data_ptr(), indices.numel(),
                     static_cast<int>(indices.element_size()), scale, padding, out.data_ptr(), c10::cuda::getCurrentCUDAStream().stream()));
    return out;
}

// autograd node of a lookup: the table's gradient from its output's
struct LookupBackward : torch::autograd::Node {
    torch::autograd::SavedVariable indices;
    std::vector<int64_t> shape;
    at::ScalarType type;
    at::Device device{at::kCUDA};
    int64_t tokens;
    double scale;
    int64_t padding;

    std::string name() const override { return "EmbeddingLookupBackward"; }
    void release_variables() override { indices.reset_data(); }

    // A leaf's accumulation runs on the stream on which its first living graph was made. If that is the default stream
    // and this backward is being captured, the engine would have the default stream wait for a captured event.
    void refuse_uncapturable() const {
        const auto& leaf = next_edge(0).function;
        if (!leaf || leaf->num_outputs() != 0) return;
        const auto at = leaf->stream();
        if (at && at->id() == 0 && c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
            refuse("the backward of embedding_lookup cannot be captured while a graph of the table made on the default stream lives: release it first");
    }

    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        if (!grads[0].defined()) return {at::Tensor()};
        refuse_recorded("the backward of embedding_lookup");
        refuse_uncapturable();
        const at::Tensor idx = indices.unpack();
        // direct calls of the node and hooks on saved tensors may hand over anything
        int64_t width = 1;
        for (size_t d = 1; d < shape.size(); d++) width *= shape[d];
        refuse_wrapped(idx, "saved indices");
        if (idx.layout() != at::kStrided || idx.is_neg() || (idx.scalar_type() != at::kLong && idx.scalar_type() != at::kInt) || !idx.is_contiguous() ||
            idx.device() != device || idx.numel() != tokens)
            refuse("the saved indices of embedding_lookup came back with another type, size, order or device");
        refuse_unbacked(idx, "saved indices");
        if (grads[0].layout() != at::kStrided || grads[0].device() != device || grads[0].numel() != tokens * width)
            refuse("embedding_lookup was given a gradient of another size or device than its output");
        refuse_wrapped(grads[0], "the gradient of a lookup");
        refuse_unbacked(grads[0], "the gradient of a lookup");
        at::Tensor grad;
        {
            const at::AutoGradMode no_graph(false);
            const at::Tensor g = settled(grads[0].scalar_type() == type ? grads[0] : grads[0].to(type));
            const c10::cuda::CUDAGuard guard(g.device());
            grad = at::empty(shape, g.options());
            refuse_wrapped(grad, "the table's gradient");
            size_t bytes = 0;
            check(lib.workspace_bytes(idx.numel(), shape[0], width, &bytes));
            const at::Tensor space = at::empty({static_cast<int64_t>(bytes)}, g.options().dtype(at::kByte));
            check(lib.lookup_grad(idx.data_ptr(), idx.numel(), static_cast<int>(idx.element_size()), g.data_ptr(), type_code(g), shape[0], width, scale,
                                  padding, grad.data_ptr(), space.data_ptr(), bytes, c10::cuda::getCurrentCUDAStream().stream()));
        }
        if (at::GradMode::is_enabled() && grads[0].requires_grad()) {  // asked for a graph of the gradient: an error if it is used
            grad.set_requires_grad(true);
            auto error = std::make_shared<torch::autograd::DelayedError>("embedding_lookup is differentiable once", 1);
            return (*error)({grad});
        }
        return {grad};
    }
};

at::Tensor lookup_with_grad(const at::Tensor& table, const at::Tensor& indices, double scale, int64_t padding) {
    std::shared_ptr<LookupBackward> node(new LookupBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(table));
    node->indices = torch::autograd::SavedVariable(indices, false);
    node->shape = table.sizes().vec();
    node->type = table.scalar_type();
    node->device = table.device();
    node->tokens = indices.numel();
    node->scale = scale;
    node->padding = padding;
    at::Tensor out = lookup(table, indices, scale, padding);
    torch::autograd::set_history(out, node);
    return out;
}

// embedding_lookup(table, indices, scale, padding index or None)
PyObject* embedding_lookup(PyObject*, PyObject* args) {
    PyObject *table_o, *indices_o, *padding_o;
    double scale;
    if (!PyArg_ParseTuple(args, "OOdO", &table_o, &indices_o, &scale, &padding_o)) return nullptr;
    return guarded([&]() -> PyObject* {
        refuse_recorded("embedding_lookup");
        const at::Tensor& table = tensor_of(table_o, "table");
        refuse_wrapped(table, "table");
        const int code = type_code(table);
        if (table.layout() != at::kStrided || !table.is_cuda() || code < 0 || code > FGS_DTYPE_F16 || table.dim() < 1 || !table.is_contiguous())
            refuse("table must be a contiguous CUDA float32, bfloat16 or float16 tensor [rows, ...]");
        if (table._fw_grad(0).defined()) refuse("embedding_lookup has no forward-mode derivative");
        const at::Tensor& given = tensor_of(indices_o, "indices");
        refuse_wrapped(given, "indices");
        if (given.layout() != at::kStrided || (given.scalar_type() != at::kLong && given.scalar_type() != at::kInt) || given.device() != table.device())
            refuse("indices must be an int64 or int32 tensor on the device of the table");
        int64_t padding = -1;
        if (padding_o != Py_None) {
            padding = PyLong_AsLongLong(padding_o);
            if (padding == -1 && PyErr_Occurred()) throw PythonError();
            if (padding < 0 || padding >= table.size(0)) {
                PyErr_SetString(PyExc_ValueError, "padding_index must be a row of the table (negative indices are padding anyway)");
                throw PythonError();
            }
        }
        refuse_unbacked(table, "table");
        refuse_unbacked(given, "indices");
        const at::Tensor indices = settled(given);
        return THPVariable_Wrap(table.requires_grad() && at::GradMode::is_enabled() ? lookup_with_grad(table, indices, scale, padding)
                                                                                   : lookup(table, indices, scale, padding));
    });
}

// bind(addresses of the C entry points, in the order of Entries)
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long a[8];
    if (!PyArg_ParseTuple(args, "KKKKKKKK", a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6, a + 7)) return nullptr;
    lib = {reinterpret_cast<decltype(lib.last_error)>(a[0]),   reinterpret_cast<decltype(lib.adamw_step)>(a[1]),
           reinterpret_cast<decltype(lib.grad_squares_capacity)>(a[2]), reinterpret_cast<decltype(lib.grad_squares)>(a[3]),
           reinterpret_cast<decltype(lib.read_moments)>(a[4]), reinterpret_cast<decltype(lib.lookup)>(a[5]),
           reinterpret_cast<decltype(lib.workspace_bytes)>(a[6]), reinterpret_cast<decltype(lib.lookup_grad)>(a[7])};
    Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {{"bind", bind, METH_VARARGS, "addresses of the C entry points"},
                          {"adamw_step", adamw_step, METH_VARARGS, "one AdamW step over parameter groups"},
                          {"read_moments", read_moments, METH_VARARGS, "values of the moments"},
                          {"embedding_lookup", embedding_lookup, METH_VARARGS, "scaled rows of a table"},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fgs_host", "host side of the many-tensor operators", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fgs_host() {
    const auto name = [](const char* s) { return PyUnicode_InternFromString(s); };
    names = {name("params"),  name("lr"),         name("betas"),            name("eps"),                 name("weight_decay"), name("state_bits"), name("master_weights"),
             name("step"),    name("exp_avg"),    name("exp_avg_sq"),       name("exp_avg_exponent"),    name("exp_avg_sq_exponent"), name("master"),
             name("maximize"), name("amsgrad"), name("differentiable"), name("decoupled_weight_decay"), name("grad_norm")};
    return PyModule_Create(&kModule);
}
