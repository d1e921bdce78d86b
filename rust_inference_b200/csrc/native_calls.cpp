// The host side of calls whose device time is a few microseconds: a Python extension that looks at the tensors and calls the kernel
// libraries' C entry points.  Through ctypes a call cost the host 8 to 11 us (token_logprobs, with its four results, 14), most of it
// for twenty to thirty arguments that are looked at and converted one by one in Python; from here it is 3.1 to 3.8 us (6.4), of
// which the launch is 2.7.
//
// The functions take their arguments by position (kernels/quantized_cache.py, kernels/microscaled.py and kernels/ops.py have the interfaces and their
// documentation).  `bind` names the entry points, by address, and the exception class that refusals and failed launches raise.
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>

#include <stdint.h>
#include <string>

namespace {

PyObject* error_class = nullptr;
long long launches = 0;

struct Bound {
    void* fn = nullptr;
    const char* (*last_error)() = nullptr;
};
enum { WRITE = 0, READ = 1, ATTEND = 2, LOGPROBS = 3, MX_HOLD = 4, MX_VALUES = 5, MX_NORM = 6, MX_PRODUCT = 7, ENTRIES = 8 };
Bound bound[ENTRIES];

struct Refused {                                 // thrown with a message for `error_class`
    std::string what;
};
struct Raised {};                                // a Python exception is set

[[noreturn]] void refuse(const std::string& what) { throw Refused{what}; }
void need(bool good, const char* what) {
    if (!good) refuse(what);
}

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse(std::string(what) + ": a tensor is missing");
    return THPVariable_Unpack(o);
}
long long number(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}
int small(long long v) {
    if (v < INT32_MIN || v > INT32_MAX) refuse("a size of more than 31 bits");
    return static_cast<int>(v);
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
}
// the i-th number of a tuple
long long item(PyObject* tuple, Py_ssize_t i) {
    if (!PyTuple_Check(tuple) || i >= PyTuple_GET_SIZE(tuple)) refuse("a tuple of numbers is missing");
    return number(PyTuple_GET_ITEM(tuple, i));
}
template <typename T> T* address(long long v) { return reinterpret_cast<T*>(static_cast<intptr_t>(v)); }

int code_of(const at::Tensor& t, const char* what) {
    if (t.scalar_type() == at::kFloat) return 0;
    if (t.scalar_type() == at::kBFloat16) return 1;
    refuse(std::string(what) + ": float32 or bfloat16 is wanted");
}
const int* index(PyObject* o, long long least, const char* what) {
    const at::Tensor& t = tensor(o, what);
    if (t.scalar_type() != at::kInt || !t.is_cuda() || t.numel() < least || !t.is_contiguous())
        refuse(std::string(what) + ": index arrays are contiguous int32 on the device, " + std::to_string(least) + " entries or more here");
    return t.const_data_ptr<int>();
}
const float* floats(PyObject* o, long long least, const char* what) {
    const at::Tensor& t = tensor(o, what);
    if (t.scalar_type() != at::kFloat || !t.is_cuda() || t.numel() < least || !t.is_contiguous())
        refuse(std::string(what) + ": contiguous float32 numbers on the device are wanted, " + std::to_string(least) + " or more here");
    return t.const_data_ptr<float>();
}
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

void finish(int rc, int which, const char* what) {
    if (rc != 0) refuse(std::string(what) + ": " + bound[which].last_error());
    ++launches;
}
template <typename F> F* entry(int which) {
    if (bound[which].fn == nullptr) refuse("native calls: an entry point that nobody has named");
    return reinterpret_cast<F*>(bound[which].fn);
}

template <typename F> PyObject* guarded(F f) {
    try {
        return f();
    } catch (const Refused& r) {
        PyErr_SetString(error_class != nullptr ? error_class : PyExc_RuntimeError, r.what.c_str());
    } catch (const Raised&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "native calls: an unknown exception");
    }
    return nullptr;
}

// ---- quantized_cache.write -----------------------------------------------------------------------------------------------
// (src, q_out or None, cos or None, sin or None, layer, page_table, seq_slot, seq_start, cu_seqlens, n_heads, n_kv_heads, head_dim,
//  v_head_dim, max_new, style, rot_dims, bias or None, clear); layer: (k, v, k scales, v scales, kv heads, head size, value head size)
typedef int WriteFn(void*, int, int, const float*, int, void*, int, const float*, const float*, const int*, int, const int*, const int*, const int*,
                    int8_t*, int8_t*, float*, float*, int, int, int, int, int, int, int, int, int, void*);
PyObject* py_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* what = "quantized_cache.write";
        need(n == 18, "quantized_cache.write: 18 arguments");
        const long long heads = number(a[9]), kv = number(a[10]), hd = number(a[11]), v_hd = number(a[12]), rot = number(a[15]);
        PyObject* layer = a[4];
        if (item(layer, 4) != kv || item(layer, 5) != hd || item(layer, 6) != v_hd) refuse("quantized_cache.write: the layer has other heads");
        need(heads >= 0, "quantized_cache.write: a negative number of heads");
        const long long cols = (heads + kv) * hd + kv * v_hd;
        const at::Tensor& src = tensor(a[0], what);
        need(src.is_cuda() && src.dim() == 2 && src.is_contiguous() && src.size(1) >= cols,
             "quantized_cache.write: a contiguous [tokens, q | k | v columns] on the device is wanted");
        const int code = code_of(src, what);
        void* q_at = nullptr;
        int q_code = code;
        if (a[1] != Py_None) {
            const at::Tensor& q = tensor(a[1], what);
            q_code = code_of(q, what);
            need(q.is_cuda() && q.dim() == 2 && q.is_contiguous() && q.size(0) == src.size(0) && q.size(1) == heads * hd && (q_code == code || code == 0),
                 "quantized_cache.write: q_out must be [tokens, heads * head size]");
            q_at = q.data_ptr();
        }
        const float *cos_at = nullptr, *sin_at = nullptr;
        if (rot != 0) {
            const at::Tensor &c = tensor(a[2], what), &s = tensor(a[3], what);
            need(c.dim() == 2 && c.size(1) * 2 == rot && s.sizes() == c.sizes(), "quantized_cache.write: tables must be float32 [positions, rotated channels / 2]");
            cos_at = floats(a[2], 0, what);
            sin_at = floats(a[3], 0, what);
        }
        const float* bias = a[16] == Py_None ? nullptr : floats(a[16], cols, what);
        const at::Tensor& table = tensor(a[5], what);
        need(table.dim() == 2, "quantized_cache.write: the page table must be int32 [slots, pages]");
        const long long seqs = tensor(a[6], what).numel();
        const int* slot = index(a[6], seqs, what);
        const int clear = PyObject_IsTrue(a[17]);
        if (clear < 0) throw Raised{};
        finish(entry<WriteFn>(WRITE)(src.data_ptr(), code, small(src.size(1)), bias, clear, q_at, q_code, cos_at, sin_at,
                                     index(a[5], 1, what), small(table.size(1)), slot, index(a[7], seqs, what), index(a[8], seqs + 1, what),
                                     address<int8_t>(item(layer, 0)), address<int8_t>(item(layer, 1)), address<float>(item(layer, 2)),
                                     address<float>(item(layer, 3)), small(src.size(0)), small(seqs), small(number(a[13])), small(heads), small(kv), small(hd),
                                     small(v_hd), small(rot), small(number(a[14])), stream()),
               WRITE, what);
        Py_RETURN_NONE;
    });
}

// ---- quantized_cache.read ------------------------------------------------------------------------------------------------
// (layer, k_out, v_out, page_table, seq_slot, seq_first, seq_len, max_len, cu_rows or None, pages, seen, span, out_pages); pages: the layer's
typedef int ReadFn(const int8_t*, const int8_t*, const float*, const float*, void*, void*, int, const int*, int, const int*, const int*, const int*,
                   const int*, int, int, int, int, int, int, int, int, void*);
PyObject* py_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* what = "quantized_cache.read";
        need(n == 13, "quantized_cache.read: 13 arguments");
        PyObject* layer = a[0];
        const long long kv = item(layer, 4), hd = item(layer, 5), v_hd = item(layer, 6), pages = number(a[9]);
        const at::Tensor &k = tensor(a[1], what), &v = tensor(a[2], what), &table = tensor(a[3], what);
        const int code = code_of(k, what);
        need(k.is_cuda() && v.is_cuda() && v.scalar_type() == k.scalar_type() && k.is_contiguous() && v.is_contiguous(),
             "quantized_cache.read: outputs of one dtype, contiguous, on the device");
        need(table.dim() == 2, "quantized_cache.read: the page table must be int32 [slots, pages]");
        const long long seqs = tensor(a[4], what).numel();
        const int* rows = nullptr;
        if (a[8] == Py_None) {
            const long long own = number(a[12]), out_pages = own > 0 ? seqs * own : pages;
            const int64_t ks[4] = {out_pages, kv, 64, hd}, vs[4] = {out_pages, kv, 64, v_hd};
            need(k.sizes() == at::IntArrayRef(ks, 4) && v.sizes() == at::IntArrayRef(vs, 4),
                 "quantized_cache.read: without cu_rows the outputs have the cache's shape, or so many pages for each sequence");
        } else {
            need(k.dim() == 3 && v.dim() == 3 && k.size(1) == kv && k.size(2) == hd && v.size(0) == k.size(0) && v.size(1) == kv && v.size(2) == v_hd,
                 "quantized_cache.read: with cu_rows the outputs are [rows, kv heads, head size]");
            rows = index(a[8], seqs, what);
        }
        finish(entry<ReadFn>(READ)(address<int8_t>(item(layer, 0)), address<int8_t>(item(layer, 1)), address<float>(item(layer, 2)),
                                   address<float>(item(layer, 3)), k.data_ptr(), v.data_ptr(), code, index(a[3], 1, what), small(table.size(1)),
                                   index(a[4], seqs, what), index(a[5], seqs, what), index(a[6], seqs, what), rows, small(seqs), small(number(a[7])),
                                   small(kv), small(hd), small(v_hd), small(number(a[10])), small(number(a[11])), small(number(a[12])), stream()),
               READ, what);
        Py_RETURN_NONE;
    });
}

// ---- quantized_cache.attend_step -----------------------------------------------------------------------------------------
// (q, layer, out, step, scale, span, out_scale); step: (page table, pages per slot, slots, starts, offsets, sequences, max_new, heads,
//  kv heads, head size, scratch, its floats, counters, the longest sequence)
typedef int AttendFn(const void*, int, int, const int8_t*, const int8_t*, const float*, const float*, const int*, int, const int*, const int*,
                     const int*, void*, int, int, int, int, int, int, int, float, int, float, float*, long long, int*, void*);
PyObject* py_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* what = "quantized_cache.attend_step";
        need(n == 7, "quantized_cache.attend_step: 7 arguments");
        PyObject *layer = a[1], *step = a[3];
        const long long heads = item(step, 7), kv = item(step, 8), hd = item(step, 9), width = heads * hd;
        const at::Tensor &q = tensor(a[0], what), &out = tensor(a[2], what);
        const int code = code_of(q, what);
        need(item(layer, 4) == kv && item(layer, 5) == hd && item(layer, 6) == hd && (item(layer, 0) | item(layer, 1)) % 16 == 0,
             "quantized_cache.attend_step: the layer has other heads, or lies off a 16-byte boundary");
        need(q.is_cuda() && out.is_cuda() && out.scalar_type() == q.scalar_type() && q.dim() == 2 && out.dim() == 2 && q.stride(1) == 1 &&
                 out.stride(1) == 1 && q.size(0) == out.size(0) && q.size(1) >= width && out.size(1) >= width,
             "quantized_cache.attend_step: rows of queries and result hold all heads side by side, in one dtype, on the device");
        finish(entry<AttendFn>(ATTEND)(q.data_ptr(), code, small(q.stride(0)), address<int8_t>(item(layer, 0)), address<int8_t>(item(layer, 1)),
                                       address<float>(item(layer, 2)), address<float>(item(layer, 3)), address<int>(item(step, 0)),
                                       small(item(step, 1)), address<int>(item(step, 2)), address<int>(item(step, 3)), address<int>(item(step, 4)),
                                       out.data_ptr(), small(out.stride(0)), small(item(step, 5)), small(item(step, 6)), small(item(step, 13)), small(heads), small(kv), small(hd),
                                       (float)real(a[4]), small(number(a[5])), (float)real(a[6]), address<float>(item(step, 10)), item(step, 11),
                                       address<int>(item(step, 12)), stream()),
               ATTEND, what);
        Py_INCREF(a[2]);
        return a[2];
    });
}

// ---- token_logprobs ------------------------------------------------------------------------------------------------------
// (logits, targets, top, most) -> (logprob, entropy, ids or None, log probabilities or None)
typedef int LogprobsFn(const void*, int, long long, int, int, const int*, int, float*, float*, int*, float*, void*);
PyObject* py_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* what = "token_logprobs";
        need(n == 4, "token_logprobs: 4 arguments");
        const at::Tensor &x = tensor(a[0], what), &targets = tensor(a[1], what);
        const long long top = number(a[2]), most = number(a[3]);
        const int code = code_of(x, what);
        need(x.is_cuda() && x.dim() == 2 && x.size(1) > 0 && (x.stride(1) == 1 || x.size(1) == 1),
             "token_logprobs: logits must be [rows, vocabulary] on the device, neighbours side by side");
        const long long rows = x.size(0), vocab = x.size(1);
        const int* ids = index(a[1], rows, what);
        need(targets.numel() == rows, "token_logprobs: a target per row");
        need(top >= 0 && top <= vocab && top <= most, "token_logprobs: too many alternatives, or fewer than none");
        // the results lie one behind the other in one allocation (a microsecond and a half for each)
        const at::Tensor room = at::empty({rows * (2 + 2 * top)}, x.options().dtype(at::kFloat).layout(at::kStrided));
        auto piece = [&](long long at, bool whole_numbers, at::IntArrayRef sizes) {
            at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(room.storage()), room.key_set(),
                                                                    whole_numbers ? caffe2::TypeMeta::Make<int>() : caffe2::TypeMeta::Make<float>());
            t.unsafeGetTensorImpl()->set_storage_offset(at);
            t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
            return t;
        };
        const int64_t one[1] = {rows}, two[2] = {rows, top};
        at::Tensor logprob = piece(0, false, one), entropy = piece(rows, false, one), best, best_ids;
        if (top) {
            best = piece(2 * rows, false, two);
            best_ids = piece((2 + top) * rows, true, two);
        }
        finish(entry<LogprobsFn>(LOGPROBS)(x.data_ptr(), code, x.stride(0), small(rows), small(vocab), ids, small(top), logprob.data_ptr<float>(),
                                           entropy.data_ptr<float>(), top ? best_ids.data_ptr<int>() : nullptr,
                                           top ? best.data_ptr<float>() : nullptr, stream()),
               LOGPROBS, what);
        PyObject* out = PyTuple_New(4);
        if (out == nullptr) throw Raised{};
        const at::Tensor* all[4] = {&logprob, &entropy, &best_ids, &best};
        for (int i = 0; i < 4; ++i) {
            PyObject* o = Py_None;
            if (all[i]->defined()) {
                o = THPVariable_Wrap(*all[i]);
                if (o == nullptr) {
                    Py_DECREF(out);
                    throw Raised{};
                }
            } else {
                Py_INCREF(Py_None);
            }
            PyTuple_SET_ITEM(out, i, o);
        }
        return out;
    });
}

// ---- microscaled ---------------------------------------------------------------------------------------------------------
// What is held comes as the address of its description in host memory (`Held`, microscaled.cuh); its library looks at that.
bool here(const at::Tensor& t) { return t.is_cuda() && t.get_device() == c10::cuda::current_device(); }
const at::Tensor& rows(PyObject* o, const char* what) {                 // numbers of a row lie side by side
    const at::Tensor& t = tensor(o, what);
    if (!here(t) || t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1)))
        refuse(std::string(what) + ": rows [n, k] on the current device, their numbers side by side, are wanted");
    return t;
}
const at::Tensor& dense(PyObject* o, const char* what) {
    const at::Tensor& t = tensor(o, what);
    if (!here(t) || t.dim() != 2 || !t.is_contiguous()) refuse(std::string(what) + ": a contiguous [n, k] on the current device is wanted");
    return t;
}
// Whether two tensors' numbers lie in the same memory, in part at least.
bool overlap(const at::Tensor& a, const at::Tensor& b) {
    auto ends = [](const at::Tensor& t, uintptr_t& from, uintptr_t& to) {
        long long last = 0;
        for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
        from = reinterpret_cast<uintptr_t>(t.data_ptr());
        to = from + static_cast<uintptr_t>(last + 1) * t.element_size();
    };
    if (a.numel() == 0 || b.numel() == 0) return false;
    uintptr_t a0, a1, b0, b1;
    ends(a, a0, a1);
    ends(b, b0, b1);
    return a0 < b1 && b0 < a1;
}
typedef int Mx_holdFn(const void*, int, long long, long long, long long, void*, void*);
void mx_hold(const at::Tensor& x, void* held, const char* what) {
    finish(entry<Mx_holdFn>(MX_HOLD)(x.data_ptr(), code_of(x, what), x.size(0), x.size(1), x.size(0) > 1 ? x.stride(0) : x.size(1), held, stream()), MX_HOLD, what);
}
// (matrix) -> (codes, exponents, description): 4 bits.  `make` and `held_bytes`: addresses of ri_mx_make and the bytes of a description.
typedef int MxMakeFn(void*, void*, void*, long long, long long, int, int);
PyObject* py_mx_matrix(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* what = "microscaled.Matrix";
        need(n == 3, "microscaled.Matrix: 3 arguments");
        const at::Tensor& x = rows(a[0], what);
        const int64_t N = x.size(0), spans = (x.size(1) + 127) / 128;
        need(N > 0 && spans > 0, "microscaled.Matrix: a matrix of at least one number is wanted");
        code_of(x, what);
        const auto bytes = x.options().dtype(at::kByte).layout(at::kStrided).requires_grad(false);
        const at::Tensor made[3] = {at::empty({(N + 127) / 128, spans, 128, 64}, bytes), at::empty({(N + 127) / 128, spans, 512}, bytes),
                                    at::empty({number(a[2])}, bytes.device(at::kCPU))};
        if (address<MxMakeFn>(number(a[1]))(made[2].data_ptr(), made[0].data_ptr(), made[1].data_ptr(), N, x.size(1), 4, x.get_device()) != 0)
            refuse(std::string(what) + ": " + bound[MX_HOLD].last_error());
        mx_hold(x, made[2].data_ptr(), what);
        PyObject* out = PyTuple_New(3);
        if (out == nullptr) throw Raised{};
        for (int i = 0; i < 3; ++i) {
            PyObject* o = THPVariable_Wrap(made[i]);
            if (o == nullptr) {
                Py_DECREF(out);
                throw Raised{};
            }
            PyTuple_SET_ITEM(out, i, o);
        }
        return out;
    });
}
// (x, held)
PyObject* py_mx_hold(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        need(n == 2, "microscaled: 2 arguments");
        mx_hold(rows(a[0], "microscaled"), address<void>(number(a[1])), "microscaled");
        Py_RETURN_NONE;
    });
}
// (held, out), or (held, None, bfloat16 or float32, n, k) for a new tensor
typedef int Mx_valuesFn(const void*, int, long long, long long, void*, void*);
PyObject* py_mx_values(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* what = "microscaled.values";
        need(n == 2 || n == 5, "microscaled.values: 2 or 5 arguments");
        const bool made = n == 5 && a[1] == Py_None;
        const at::Tensor out = made ? at::empty({number(a[3]), number(a[4])}, at::TensorOptions().device(at::kCUDA, c10::cuda::current_device())
                                                                                  .dtype(number(a[2]) ? at::kBFloat16 : at::kFloat))
                                    : dense(a[1], what);
        finish(entry<Mx_valuesFn>(MX_VALUES)(address<void>(number(a[0])), code_of(out, what), out.size(0), out.size(1), out.data_ptr(), stream()), MX_VALUES, what);
        return THPVariable_Wrap(out);
    });
}
// (x, branch or None, weight, total or None, eps, held)
typedef int Mx_rmsnormFn(const float*, const void*, int, const float*, float*, long long, long long, double, void*, void*);
PyObject* py_mx_rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* what = "microscaled.rmsnorm";
        need(n == 6, "microscaled.rmsnorm: 6 arguments");
        const at::Tensor &x = dense(a[0], what), &weight = tensor(a[2], what);
        need(x.scalar_type() == at::kFloat, "microscaled.rmsnorm: x must be float32");
        need(here(weight) && weight.scalar_type() == at::kFloat && weight.is_contiguous() && weight.numel() == x.size(1), "microscaled.rmsnorm: weight must be float32 [k]");
        const void* branch = nullptr;
        int branch_code = 0;
        if (a[1] != Py_None) {
            const at::Tensor& b = dense(a[1], what);
            need(b.sizes() == x.sizes(), "microscaled.rmsnorm: a branch as x is wanted");
            branch = b.data_ptr();
            branch_code = code_of(b, what);
        }
        float* total = nullptr;
        if (a[3] != Py_None) {
            const at::Tensor& t = dense(a[3], what);
            need(t.scalar_type() == at::kFloat && t.sizes() == x.sizes(), "microscaled.rmsnorm: total must be float32, as x");
            for (PyObject* o : {a[0], a[1]}) {
                if (o == Py_None) continue;
                const at::Tensor& other = tensor(o, what);
                need(!overlap(t, other) || (t.data_ptr() == other.data_ptr() && t.scalar_type() == other.scalar_type()),
                     "microscaled.rmsnorm: total is x or the branch itself, or lies apart from them");
            }
            need(!overlap(t, weight), "microscaled.rmsnorm: total lies apart from the weight");
            total = t.data_ptr<float>();
        }
        finish(entry<Mx_rmsnormFn>(MX_NORM)(x.data_ptr<float>(), branch, branch_code, weight.data_ptr<float>(), total, x.size(0), x.size(1), real(a[4]),
                                        address<void>(number(a[5])), stream()), MX_NORM, what);
        Py_RETURN_NONE;
    });
}
// (plain rows or None, held rows (scratch, where there are plain ones), matrix, second matrix or 0, constants or None, act, add, out or None,
//  held result or 0, status word).  A few plain rows go to the product as they are, others by way of the scratch: 2 is its answer to those.
typedef int Mx_productFn(void*, const void*, int, long long, long long, long long, void*, void*, const float*, long long, int, int, void*, int, long long,
                         long long, void*, int*, void*);
PyObject* py_mx_product(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* what = "microscaled.product";
        need(n == 10, "microscaled.product: 10 arguments");
        void* held = address<void>(number(a[1]));
        const float* constants = nullptr;
        long long n_constants = 0;
        if (a[4] != Py_None) {
            const at::Tensor& t = tensor(a[4], what);
            need(here(t) && t.scalar_type() == at::kFloat && t.is_contiguous(), "microscaled.product: a bias or an activation's constants are contiguous float32 on the current device");
            constants = t.data_ptr<float>();
            n_constants = t.numel();
        }
        void* out = nullptr;
        int out_code = 0;
        long long out_rows = 0, out_cols = 0;
        if (a[7] != Py_None) {
            const at::Tensor& o = dense(a[7], what);
            out = o.data_ptr();
            out_code = code_of(o, what);
            out_rows = o.size(0);
            out_cols = o.size(1);
        }
        const at::Tensor* x = a[0] == Py_None ? nullptr : &rows(a[0], what);
        const int x_code = x ? code_of(*x, what) : 0;
        if (x && out) need(!overlap(*x, tensor(a[7], what)), "microscaled.product: the result lies apart from the rows");
        auto call = [&](bool plain) {
            return entry<Mx_productFn>(MX_PRODUCT)(held, plain ? x->data_ptr() : nullptr, x_code, plain ? x->size(0) : 0, plain ? x->size(1) : 0,
                                                   plain ? (x->size(0) > 1 ? x->stride(0) : x->size(1)) : 0, address<void>(number(a[2])),
                                                   address<void>(number(a[3])), constants, n_constants, (int)number(a[5]), (int)number(a[6]), out, out_code,
                                                   out_rows, out_cols, address<void>(number(a[8])), address<int>(number(a[9])), stream());
        };
        int rc = call(x != nullptr);
        if (rc == 2) {
            mx_hold(*x, held, what);
            rc = call(false);
        }
        finish(rc, MX_PRODUCT, what);
        Py_RETURN_NONE;
    });
}

// (which, address of the entry point, address of its library's ri_last_error, exception class)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        need(n == 4, "bind: 4 arguments");
        const long long which = number(a[0]);
        need(which >= 0 && which < ENTRIES, "bind: no such entry point");
        bound[which].fn = address<void>(number(a[1]));
        bound[which].last_error = reinterpret_cast<const char* (*)()>(static_cast<intptr_t>(number(a[2])));
        Py_INCREF(a[3]);
        Py_XDECREF(error_class);
        error_class = a[3];
        Py_RETURN_NONE;
    });
}
PyObject* py_launches(PyObject*, PyObject* const*, Py_ssize_t) { return PyLong_FromLongLong(launches); }

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)> PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<py_write>("write"), method<py_read>("read"), method<py_attend>("attend"), method<py_logprobs>("logprobs"),
                         method<py_mx_hold>("mx_hold"), method<py_mx_matrix>("mx_matrix"), method<py_mx_values>("mx_values"), method<py_mx_rmsnorm>("mx_rmsnorm"),
                         method<py_mx_product>("mx_product"),
                         method<py_bind>("bind"), method<py_launches>("launches"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "ri_native_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_ri_native_calls() { return PyModule_Create(&module_def); }
