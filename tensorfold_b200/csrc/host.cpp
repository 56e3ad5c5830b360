// Python binding of the C ABI (include/tensorfold_b200.h) and the native host path of the single-operator calls.
//
// A single projection at 1..8 rows keeps the GPU busy for 5 to 15 us; the Python and ctypes work around it (argument
// conversion, torch.cuda.device contexts, Stream objects, views, allocations) took 42 us a call, so the host
// bound every small call. Here an entry point is a METH_FASTCALL function generated from its C signature (about 0.3 us
// of conversion for 17 arguments; tensors are passed as tensors), and the matmul calls do their checks,
// allocations and launches in one native call.
//
// The functions take the arguments of the C entry point, in order: a pointer is a CUDA tensor, an address or None. While the
// C call runs the interpreter is released, as under ctypes: a launch that waits for a place in a full queue stops no other thread.

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <atomic>
#include <cmath>
#include <cstring>
#include <map>
#include <mutex>
#include <tuple>
#include <utility>

#include "../../include/tensorfold_b200.h"

namespace {

std::atomic<long long> g_launches{0};      // kernels queued by successful calls

struct PyErr {};                           // thrown with a Python error set

struct Released {                          // the interpreter lock given up for a scope; no Python object is touched in it
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
};
[[noreturn]] void fail(PyObject* type, const char* text) {
    PyErr_SetString(type, text);
    throw PyErr{};
}

// ---- one Python object -> one C argument --------------------------------------------------------------
template <class T>
T convert(PyObject* o) {
    if constexpr (std::is_pointer_v<T>) {
        if (o == Py_None) return nullptr;
        if (THPVariable_Check(o)) return reinterpret_cast<T>(THPVariable_Unpack(o).unsafeGetTensorImpl()->mutable_data());
        const unsigned long long v = PyLong_AsUnsignedLongLong(o);
        if (v == ~0ull && PyErr_Occurred()) throw PyErr{};
        return reinterpret_cast<T>(v);
    } else if constexpr (std::is_floating_point_v<T>) {
        const double v = PyFloat_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred()) throw PyErr{};
        return static_cast<T>(v);
    } else if constexpr (sizeof(T) == 8 && std::is_unsigned_v<T>) {
        const unsigned long long v = PyLong_AsUnsignedLongLong(o);
        if (v == ~0ull && PyErr_Occurred()) throw PyErr{};
        return static_cast<T>(v);
    } else {
        const long long v = PyLong_AsLongLong(o);
        if (v == -1 && PyErr_Occurred()) throw PyErr{};
        return static_cast<T>(v);
    }
}

template <class R>
PyObject* to_python(R v) {
    if constexpr (std::is_unsigned_v<R>) return PyLong_FromUnsignedLongLong(v);
    else return PyLong_FromLongLong(v);
}

// LAUNCHES: kernels that a successful call queues (0: a host-only function)
template <auto Fn, int LAUNCHES>
struct Entry;
template <class R, class... A, R (*Fn)(A...), int LAUNCHES>
struct Entry<Fn, LAUNCHES> {
    template <size_t... I>
    static PyObject* apply(PyObject* const* args, std::index_sequence<I...>) {
        std::tuple<A...> v{convert<A>(args[I])...};
        if constexpr (std::is_void_v<R>) {
            {
                const Released unlocked;
                Fn(std::get<I>(v)...);
            }
            Py_RETURN_NONE;
        } else {
            const R rc = [&] {
                const Released unlocked;
                return Fn(std::get<I>(v)...);
            }();
            if (LAUNCHES > 0 && rc == 0) g_launches.fetch_add(LAUNCHES, std::memory_order_relaxed);
            return to_python(rc);
        }
    }
    // `self` is the entry point through ctypes where bound() made the function: it takes what the conversions here do not
    // (ctypes objects, byref, arrays, sizes to be wrapped), or says why not.
    static PyObject* call(PyObject* self, PyObject* const* args, Py_ssize_t n) {
        const bool bound = self != nullptr && PyCallable_Check(self);
        try {
            if (n == (Py_ssize_t)sizeof...(A)) return apply(args, std::index_sequence_for<A...>{});
            PyErr_Format(PyExc_TypeError, "this entry point takes %d arguments, got %zd", (int)sizeof...(A), n);
            throw PyErr{};
        } catch (const PyErr&) {
            if (!bound || !(PyErr_ExceptionMatches(PyExc_TypeError) || PyErr_ExceptionMatches(PyExc_OverflowError))) return nullptr;
            PyErr_Clear();
            PyObject* result = PyObject_Vectorcall(self, args, (size_t)n, nullptr);
            if (LAUNCHES > 0 && result != nullptr && PyLong_Check(result) && PyLong_AsLong(result) == 0)
                g_launches.fetch_add(LAUNCHES, std::memory_order_relaxed);
            return result;
        } catch (const std::exception& e) {
            PyErr_SetString(PyExc_RuntimeError, e.what());
            return nullptr;
        }
    }
};

// ---- matmul scratch: one buffer a (device, stream), zeroed once, kept while the process runs -----------------
// A stream's launches share it in order; other streams have their own, so calls on different streams may overlap.
std::mutex g_scratch_lock;
std::map<std::pair<int, cudaStream_t>, at::Tensor> g_scratch;

at::Tensor scratch_on(int device, cudaStream_t stream) {
    std::lock_guard<std::mutex> hold(g_scratch_lock);
    at::Tensor& t = g_scratch[{device, stream}];
    if (!t.defined())
        t = at::zeros({(int64_t)tf_qmm_scratch_bytes()}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
    return t;
}

void check_rc(int rc, const char* what) {
    if (rc == TF_OK) return;
    const char* name = rc == TF_EINVAL ? "TF_EINVAL (unsupported shape, size or flag)" : rc == TF_EALIGN ? "TF_EALIGN (misaligned pointer)"
                     : rc == TF_ESCRATCH ? "TF_ESCRATCH (scratch missing or too small)" : "TF_ECUDA (launch refused)";
    PyErr_Format(rc == TF_ECUDA ? PyExc_RuntimeError : PyExc_ValueError, "%s: %s", what, name);
    throw PyErr{};
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        return F(args, n);
    } catch (const PyErr&) {
        return nullptr;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// scratch(device index) -> the current stream's matmul scratch
PyObject* scratch_py(PyObject* const* args, Py_ssize_t) {
    const int dev = convert<int>(args[0]);
    return THPVariable_Wrap(scratch_on(dev, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream()));
}

const at::Tensor& tensor(PyObject* o) {
    if (!THPVariable_Check(o)) fail(PyExc_TypeError, "expected a tensor");
    return THPVariable_Unpack(o);
}

// rows of a projection's input: (x as [m, k] contiguous rows, m)
at::Tensor rows_of(const at::Tensor& x, int64_t k, const char* who, int64_t n) {
    if (!x.is_cuda()) fail(PyExc_ValueError, "lane kernels take CUDA tensors only (there is no CPU path)");
    if (x.scalar_type() != at::kBFloat16) {
        PyErr_Format(PyExc_ValueError, "%s: x must be bf16", who);
        throw PyErr{};
    }
    if (x.dim() < 1 || x.size(-1) != k) {
        PyErr_Format(PyExc_ValueError, "%s: weight (N=%lld, K=%lld) does not match K=%lld", who, (long long)n, (long long)k,
                     (long long)(x.dim() ? x.size(-1) : 0));
        throw PyErr{};
    }
    at::Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, k});
    if (x2.size(0) < 1) {
        PyErr_Format(PyExc_ValueError, "%s: needs at least one row", who);
        throw PyErr{};
    }
    return x2.is_contiguous() ? x2 : x2.contiguous();
}

at::Tensor output_for(PyObject* given, const at::Tensor& x, int64_t m, int64_t n, bool f32, const char* who) {
    const auto type = f32 ? at::kFloat : at::kBFloat16;
    if (given == Py_None) return at::empty({m, n}, x.options().dtype(type));
    at::Tensor out = tensor(given);
    if (out.dim() != 2 || out.size(0) != m || out.size(1) != n || out.scalar_type() != type || !out.is_contiguous()) {
        PyErr_Format(PyExc_ValueError, "%s: out has the wrong shape or dtype", who);
        throw PyErr{};
    }
    return out;
}

PyObject* shaped(const at::Tensor& out, const at::Tensor& x, int64_t n) {
    if (x.dim() == 2) return THPVariable_Wrap(out);
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    return THPVariable_Wrap(out.reshape(shape));
}

// lane_matmul(x, tiled, n, k, group, f32, out, next_tiled, next_n, next_k, next_group, status): row-major rows in any
// number, packed and multiplied in launches of up to TF_QMM_MAX_ROWS rows
PyObject* lane_matmul_py(PyObject* const* args, Py_ssize_t) {
    at::AutoDispatchBelowADInplaceOrView no_grad;
    const at::Tensor x = tensor(args[0]), w = tensor(args[1]);       // held: the interpreter lock is given up below
    const int n = convert<int>(args[2]), k = convert<int>(args[3]), group = convert<int>(args[4]);
    const bool f32 = convert<int>(args[5]) != 0;
    const at::Tensor x2 = rows_of(x, k, "lane_matmul", n);
    const int64_t m = x2.size(0);
    const c10::cuda::CUDAGuard on(x.device());
    const auto stream = c10::cuda::getCurrentCUDAStream(x.device().index());
    const at::Tensor out = output_for(args[6], x, m, n, f32, "lane_matmul");
    const at::Tensor scratch = scratch_on(x.device().index(), stream.stream());
    const void* next_w = convert<const void*>(args[7]);
    const int next_n = convert<int>(args[8]), next_k = convert<int>(args[9]), next_group = convert<int>(args[10]);
    int* status = convert<int*>(args[11]);
    const int64_t most = m < TF_QMM_MAX_ROWS ? m : TF_QMM_MAX_ROWS;
    const at::Tensor packed = at::empty({(int64_t)tf_packed_bytes((int)most, k, group)}, x.options().dtype(at::kByte));
    const size_t out_row = (size_t)n * (f32 ? 4 : 2);
    const char* what = "pack_rows";
    const int rc = [&] {
        const Released unlocked;
        for (int64_t r0 = 0; r0 < m; r0 += TF_QMM_MAX_ROWS) {
            const int rows = (int)std::min<int64_t>(m - r0, TF_QMM_MAX_ROWS);
            const bool last = r0 + rows >= m;
            what = "pack_rows";
            if (const int bad = tf_pack_rows(static_cast<const uint8_t*>(x2.const_data_ptr()) + (size_t)r0 * k * 2, packed.mutable_data_ptr(),
                                             nullptr, rows, k, group, stream.stream())) return bad;
            what = "lane_matmul";
            if (const int bad = tf_qmm_next(packed.const_data_ptr(), w.const_data_ptr(), static_cast<uint8_t*>(out.mutable_data_ptr()) + r0 * out_row,
                                            scratch.mutable_data_ptr(), (size_t)scratch.numel(), rows, n, k, group, f32 ? TF_QMM_F32_OUT : 0,
                                            last ? next_w : w.const_data_ptr(), last ? next_n : n, last ? next_k : k,
                                            last ? next_group : group, status, stream.stream())) return bad;
            g_launches.fetch_add(2, std::memory_order_relaxed);
        }
        return (int)TF_OK;
    }();
    check_rc(rc, what);
    return shaped(out, x, n);
}

// prefill_matmul(x, tiled, n, k, group, f32, out, staging, status): the same on the wide-row kernel
PyObject* prefill_matmul_py(PyObject* const* args, Py_ssize_t) {
    at::AutoDispatchBelowADInplaceOrView no_grad;
    const at::Tensor x = tensor(args[0]), w = tensor(args[1]);       // held: the interpreter lock is given up below
    const int n = convert<int>(args[2]), k = convert<int>(args[3]), group = convert<int>(args[4]);
    const bool f32 = convert<int>(args[5]) != 0;
    const at::Tensor x2 = rows_of(x, k, "prefill_matmul", n);
    const int64_t m = x2.size(0);
    const c10::cuda::CUDAGuard on(x.device());
    const auto stream = c10::cuda::getCurrentCUDAStream(x.device().index());
    const at::Tensor out = output_for(args[6], x, m, n, f32, "prefill_matmul");
    const at::Tensor scratch = scratch_on(x.device().index(), stream.stream());
    const int64_t most = m < TF_QMM_MAX_ROWS ? m : TF_QMM_MAX_ROWS;
    const size_t need = tf_packed_tc_bytes((int)most, k, group);
    const at::Tensor packed = args[7] == Py_None ? at::empty({(int64_t)need}, x.options().dtype(at::kByte)) : tensor(args[7]);
    if ((size_t)packed.numel() < need) fail(PyExc_ValueError, "prefill_matmul: staging buffer too small");
    int* status = convert<int*>(args[8]);
    const size_t out_row = (size_t)n * (f32 ? 4 : 2);
    const char* what = "prefill pack_rows";
    const int rc = [&] {
        const Released unlocked;
        for (int64_t r0 = 0; r0 < m; r0 += TF_QMM_MAX_ROWS) {
            const int rows = (int)std::min<int64_t>(m - r0, TF_QMM_MAX_ROWS);
            what = "prefill pack_rows";
            if (const int bad = tf_pack_rows_tc(static_cast<const uint8_t*>(x2.const_data_ptr()) + (size_t)r0 * k * 2, packed.mutable_data_ptr(),
                                                nullptr, rows, k, group, stream.stream())) return bad;
            what = "prefill_matmul";
            if (const int bad = tf_qmm_tc(packed.const_data_ptr(), w.const_data_ptr(), static_cast<uint8_t*>(out.mutable_data_ptr()) + r0 * out_row,
                                          scratch.mutable_data_ptr(), (size_t)scratch.numel(), rows, n, k, group, f32 ? TF_QMM_F32_OUT : 0,
                                          status, stream.stream())) return bad;
            g_launches.fetch_add(2, std::memory_order_relaxed);
        }
        return (int)TF_OK;
    }();
    check_rc(rc, what);
    return shaped(out, x, n);
}

// ---- the calls of a bounded cache and of draft verification: checks, allocations and launches in one native call -----------------
// Their device work is 5 to 20 us on small calls; the same steps from Python took 15 to 20.

// Arguments that must hold, with the text of the ValueError where one does not.
void need(bool ok, const char* text) {
    if (!ok) fail(PyExc_ValueError, text);
}
at::Tensor optional_tensor(PyObject* o) { return o == Py_None ? at::Tensor() : tensor(o); }
bool plain(const at::Tensor& t, at::ScalarType type) { return t.scalar_type() == type && t.is_contiguous(); }
template <class... T>
void on_device(const at::Tensor& first, const T&... others) {
    const auto is_cuda = [](const at::Tensor& t) { return !t.defined() || t.is_cuda(); };
    need(first.is_cuda() && (is_cuda(others) && ...), "lane kernels take CUDA tensors only (there is no CPU path)");
    need(((!others.defined() || others.device() == first.device()) && ...), "the tensors must be on one device");
}
template <class T>
T* data_of(const at::Tensor& t) { return t.defined() ? static_cast<T*>(t.mutable_data_ptr()) : nullptr; }
// The caller's buffer or one of `bytes` from the allocator. (A buffer that is too small is refused by the entry point.)
at::Tensor buffer(PyObject* given, size_t bytes, const at::Tensor& like) {
    if (given != Py_None) {
        at::Tensor t = tensor(given);
        need(t.is_contiguous(), "scratch must be contiguous");
        return t;
    }
    return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}
size_t bytes_of(const at::Tensor& t) { return (size_t)t.numel() * t.element_size(); }
int32_t checked_int(PyObject* o, const char* text) {
    const long long v = convert<long long>(o);
    need(v >= INT32_MIN && v <= INT32_MAX, text);
    return (int32_t)v;
}

// window_attention(q, k_new, v_new, k_pages, v_pages, page_table, seq_lens, seq_start, scale, max_window, max_context, window (0: none), sinks,
//                  chunk_keys (0: tf_window_chunk_keys), scratch, out, lse, gate, packed data, packed group, status) -> out or None
PyObject* window_attention_py(PyObject* const* args, Py_ssize_t n) {
    if (n != 21) fail(PyExc_TypeError, "window_attention takes 21 arguments");
    at::AutoDispatchBelowADInplaceOrView no_grad;
    const at::Tensor q = tensor(args[0]), k_new = tensor(args[1]), v_new = tensor(args[2]), k_pages = tensor(args[3]), v_pages = tensor(args[4]),
                     table = tensor(args[5]), lens = tensor(args[6]), start = tensor(args[7]), lse = optional_tensor(args[16]),
                     gate = optional_tensor(args[17]), packed = optional_tensor(args[18]);
    at::Tensor out = optional_tensor(args[15]);
    const double scale = convert<double>(args[8]);
    const char* sizes = "window >= 1 (or None), sinks >= 0, chunk_keys a positive multiple of 64 and max_context >= max_window >= 1 required";
    const int max_window = checked_int(args[9], sizes), max_context = checked_int(args[10], sizes), window = checked_int(args[11], sizes),
              sinks = checked_int(args[12], sizes), given_chunk = checked_int(args[13], sizes), group = convert<int>(args[19]);
    on_device(q, k_new, v_new, k_pages, v_pages, table, lens, start, lse, gate, packed, out, args[14] == Py_None ? at::Tensor() : tensor(args[14]));
    need(q.dim() == 3 && k_new.dim() == 3 && k_pages.dim() == 4 && table.dim() == 2 && lens.dim() == 1 && start.dim() == 1, "unsupported attention shape");
    const int64_t r = q.size(0), h = q.size(1), d = q.size(2), hk = k_new.size(1), s = lens.size(0);
    need(r >= 1 && s >= 1 && h >= 1 && hk >= 1 && k_new.size(0) == r && k_new.size(2) == d && v_new.sizes() == k_new.sizes() && (d == 128 || d == 256) && h % hk == 0 &&
             h / hk <= 16 && k_pages.size(0) >= 1 && k_pages.size(1) == hk && k_pages.size(2) == 16 && k_pages.size(3) == d && v_pages.sizes() == k_pages.sizes() &&
             table.size(0) == s && table.size(1) >= 1 && start.size(0) == s + 1 && r <= 65535 && s <= 65535 && h <= 65535 && r * h <= INT32_MAX && k_pages.size(0) <= INT32_MAX &&
             table.size(1) <= INT32_MAX,
         "unsupported attention shape");
    need(plain(q, at::kBFloat16) && plain(k_new, at::kBFloat16) && plain(v_new, at::kBFloat16) && plain(k_pages, at::kBFloat16) && plain(v_pages, at::kBFloat16),
         "attention tensors must be contiguous bf16");
    need(plain(table, at::kInt) && plain(lens, at::kInt) && plain(start, at::kInt), "page_table, seq_lens and seq_start must be contiguous int32");
    need(scale > 0 && scale < INFINITY, "scale must be positive and finite");
    const int chunk = given_chunk != 0 ? given_chunk : tf_window_chunk_keys((int)s, (int)h, (int)hk, max_window, max_context, window, sinks);
    const int slots = tf_window_slots(window, sinks, max_window, max_context, chunk);
    need(slots > 0, sizes);
    need(!lse.defined() || (plain(lse, at::kFloat) && lse.dim() == 2 && lse.size(0) == r && lse.size(1) == h), "lse must be contiguous float32 (R, H)");
    need(!out.defined() || (plain(out, at::kBFloat16) && out.sizes() == q.sizes()), "out must be contiguous bf16 (R, H, D)");
    need(!gate.defined() || (gate.scalar_type() == at::kBFloat16 && gate.dim() == 2 && gate.size(0) == r && gate.size(1) == h * 2 * d && gate.stride(1) == 1),
         "gate must be the (R, H * 2 * D) bf16 rows of the q projection");
    const c10::cuda::CUDAGuard on(q.device());
    const auto stream = c10::cuda::getCurrentCUDAStream(q.device().index());
    const at::Tensor scratch = buffer(args[14], tf_window_scratch_bytes((int)r, (int)h, (int)d, slots), q);
    if (!out.defined() && !packed.defined()) out = at::empty_like(q);
    int* status = convert<int*>(args[20]);
    const int rc = [&] {
        const Released unlocked;
        return tf_window_attention(q.const_data_ptr(), k_new.const_data_ptr(), v_new.const_data_ptr(), k_pages.const_data_ptr(), v_pages.const_data_ptr(),
                                   (int)k_pages.size(0), data_of<int>(table), (int)table.size(1), data_of<int>(lens), data_of<int>(start), data_of<void>(out),
                                   data_of<float>(lse), data_of<void>(gate), gate.defined() ? (size_t)gate.stride(0) : 0, data_of<void>(packed), group,
                                   scratch.mutable_data_ptr(), bytes_of(scratch), (int)r, (int)s, max_window, max_context, window, sinks, chunk, (int)h, (int)hk,
                                   (int)d, (float)scale, status, stream.stream());
    }();
    check_rc(rc, "window_attention");
    g_launches.fetch_add(tf_window_launches((int)r, (int)s, max_window, slots, (int)h, (int)hk, (int)d, !gate.defined() && !packed.defined()), std::memory_order_relaxed);
    if (!out.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
}

// pages [layers, pages, HK, 16, D] with the planes mass and pos, and the sequences' table and lengths
void check_cache(const at::Tensor& k_pages, const at::Tensor& mass, const at::Tensor& pos, const at::Tensor& table, const at::Tensor& lens) {
    need(k_pages.dim() == 5 && k_pages.size(0) >= 1 && k_pages.size(1) >= 1 && k_pages.size(2) >= 1 && k_pages.size(3) == 16 &&
             (k_pages.size(4) == 128 || k_pages.size(4) == 256) && plain(k_pages, at::kBFloat16) && k_pages.size(0) <= 65535 && k_pages.size(1) <= INT32_MAX &&
             k_pages.size(2) <= 65535,
         "the pages must be contiguous bf16 (layers, pages, HK, 16, D), D 128 or 256");
    const auto cells = k_pages.sizes().slice(0, 4);
    need(mass.sizes() == cells && pos.sizes() == cells && plain(mass, at::kFloat) && plain(pos, at::kInt),
         "mass must be contiguous float32 and pos int32, (layers, pages, HK, 16)");
    need(table.dim() == 2 && lens.dim() == 1 && table.size(0) == lens.size(0) && lens.size(0) >= 1 && lens.size(0) <= 65535 && table.size(1) >= 1 &&
             table.size(1) <= INT32_MAX,
         "page_table must be (S, max_pages) and seq_lens (S,)");
    need(plain(table, at::kInt) && plain(lens, at::kInt), "page_table, lengths, positions and counts must be contiguous int32");
}

// attention_mass(q, lse, k_pages, page_table, seq_lens, seq_start, keep, row_pos, mass, pos, scale, max_window, max_context, status)
PyObject* attention_mass_py(PyObject* const* args, Py_ssize_t n) {
    if (n != 14) fail(PyExc_TypeError, "attention_mass takes 14 arguments");
    at::AutoDispatchBelowADInplaceOrView no_grad;
    const at::Tensor q = tensor(args[0]), lse = tensor(args[1]), k_pages = tensor(args[2]), table = tensor(args[3]), lens = tensor(args[4]), start = tensor(args[5]),
                     keep = tensor(args[6]), row_pos = tensor(args[7]), mass = tensor(args[8]), pos = tensor(args[9]);
    const double scale = convert<double>(args[10]);
    const char* sizes = "scale must be positive and finite, max_context >= max_window >= 1";
    const int max_window = checked_int(args[11], sizes), max_context = checked_int(args[12], sizes);
    on_device(q, lse, k_pages, table, lens, start, keep, row_pos, mass, pos);
    check_cache(k_pages, mass, pos, table, lens);
    const int64_t layers = k_pages.size(0), hk = k_pages.size(2), d = k_pages.size(4), s = lens.size(0);
    need(q.dim() == 4 && q.size(0) == layers && q.size(1) >= 1 && q.size(1) <= INT32_MAX && q.size(3) == d && plain(q, at::kBFloat16),
         "q must be contiguous bf16 (layers, R, H, D)");
    const int64_t r = q.size(1), h = q.size(2);
    need(h >= 1 && h % hk == 0 && h / hk <= 16, "H must be a multiple of HK, at most 16 heads a KV head");
    need(lse.dim() == 3 && lse.size(0) == layers && lse.size(1) == r && lse.size(2) == h && plain(lse, at::kFloat), "lse must be contiguous float32 (layers, R, H)");
    need(start.dim() == 1 && start.size(0) == s + 1 && keep.dim() == 1 && keep.size(0) == s && row_pos.dim() == 1 && row_pos.size(0) == r && plain(start, at::kInt) &&
             plain(keep, at::kInt) && plain(row_pos, at::kInt),
         "seq_start (S+1,), keep (S,) and row_pos (R,), contiguous int32, required");
    need(scale > 0 && scale < INFINITY && max_window >= 1 && max_context >= max_window, sizes);
    const c10::cuda::CUDAGuard on(q.device());
    const auto stream = c10::cuda::getCurrentCUDAStream(q.device().index());
    int* status = convert<int*>(args[13]);
    const int rc = [&] {
        const Released unlocked;
        return tf_attention_mass(q.const_data_ptr(), data_of<float>(lse), k_pages.const_data_ptr(), (int)k_pages.size(1), data_of<int>(table), (int)table.size(1),
                                 data_of<int>(lens), data_of<int>(start), data_of<int>(keep), data_of<int>(row_pos), data_of<float>(mass), data_of<int>(pos),
                                 (int)layers, (int)r, (int)s, max_window, max_context, (int)h, (int)hk, (int)d, (float)scale, status, stream.stream());
    }();
    check_rc(rc, "attention_mass");
    g_launches.fetch_add(1, std::memory_order_relaxed);
    Py_RETURN_NONE;
}

// evict(k_pages, v_pages, page_table, seq_lens, next_pos, mass, pos, budget, recent, sinks, max_context, scratch, status) -> moved
PyObject* evict_py(PyObject* const* args, Py_ssize_t n) {
    if (n != 13) fail(PyExc_TypeError, "evict takes 13 arguments");
    at::AutoDispatchBelowADInplaceOrView no_grad;
    const at::Tensor k_pages = tensor(args[0]), v_pages = tensor(args[1]), table = tensor(args[2]), lens = tensor(args[3]), next_pos = tensor(args[4]),
                     mass = tensor(args[5]), pos = tensor(args[6]);
    const char* sizes = "budget >= recent + sinks, all non-negative, budget and max_context at least 1";
    const int budget = checked_int(args[7], sizes), recent = checked_int(args[8], sizes), sinks = checked_int(args[9], sizes), max_context = checked_int(args[10], sizes);
    on_device(k_pages, v_pages, table, lens, next_pos, mass, pos, args[11] == Py_None ? at::Tensor() : tensor(args[11]));
    check_cache(k_pages, mass, pos, table, lens);
    const int64_t layers = k_pages.size(0), hk = k_pages.size(2), d = k_pages.size(4), s = lens.size(0);
    need(v_pages.sizes() == k_pages.sizes() && plain(v_pages, at::kBFloat16) && next_pos.dim() == 1 && next_pos.size(0) == s && plain(next_pos, at::kInt),
         "v_pages must match k_pages and next_pos be (S,) int32");
    need(budget >= 1 && recent >= 0 && sinks >= 0 && (int64_t)recent + sinks <= budget && max_context >= 1, sizes);
    const c10::cuda::CUDAGuard on(k_pages.device());
    const auto stream = c10::cuda::getCurrentCUDAStream(k_pages.device().index());
    const at::Tensor scratch = buffer(args[11], tf_evict_scratch_bytes((int)layers, (int)s, (int)hk, budget, max_context), k_pages);
    const at::Tensor moved = at::empty({layers, s, hk}, k_pages.options().dtype(at::kInt));
    int* status = convert<int*>(args[12]);
    const int rc = [&] {
        const Released unlocked;
        return tf_kv_evict(data_of<void>(k_pages), data_of<void>(v_pages), (int)k_pages.size(1), data_of<int>(table), (int)table.size(1), data_of<int>(lens),
                           data_of<int>(next_pos), data_of<float>(mass), data_of<int>(pos), data_of<int>(moved), scratch.mutable_data_ptr(), bytes_of(scratch), (int)layers,
                           (int)s, budget, recent, sinks, max_context, (int)hk, (int)d, status, stream.stream());
    }();
    check_rc(rc, "evict");
    g_launches.fetch_add(2, std::memory_order_relaxed);
    return THPVariable_Wrap(moved);
}

// verify_drafts(logits, tokens, seq_start, uniforms, temperature, draft_logits, draft_temperature, scratch) -> (keep, next)
PyObject* verify_drafts_py(PyObject* const* args, Py_ssize_t n) {
    if (n != 8) fail(PyExc_TypeError, "verify_drafts takes 8 arguments");
    at::AutoDispatchBelowADInplaceOrView no_grad;
    at::Tensor x = tensor(args[0]), near = optional_tensor(args[5]);
    const at::Tensor tokens = tensor(args[1]), start = tensor(args[2]), uniforms = tensor(args[3]);
    const double temperature = convert<double>(args[4]), near_temperature = args[6] == Py_None ? temperature : convert<double>(args[6]);
    on_device(x, tokens, start, uniforms, near, args[7] == Py_None ? at::Tensor() : tensor(args[7]));
    const auto rows = [](at::Tensor& t, const char* text) {
        need(t.dim() == 2 && t.scalar_type() == at::kBFloat16 && t.size(0) >= 1 && t.size(0) <= 32767 && t.size(1) >= 1 && t.size(1) <= (1 << 20), text);
        if (t.stride(1) != 1 || t.stride(0) < t.size(1)) t = t.contiguous();
    };
    rows(x, "verify_drafts: logits must be 1..32767 bf16 rows of 1..1048576 logits");
    if (near.defined()) {
        need(near.sizes() == x.sizes(), "verify_drafts: draft_logits must have the shape of logits");
        rows(near, "verify_drafts: draft_logits must be bf16 rows");
    }
    const int64_t r = x.size(0), v = x.size(1);
    need(tokens.dim() == 1 && tokens.size(0) == r && plain(tokens, at::kInt), "verify_drafts: tokens must be contiguous int32, one per row");
    need(start.dim() == 1 && start.size(0) >= 2 && start.size(0) <= (1 << 24) && plain(start, at::kInt), "verify_drafts: seq_start must be contiguous int32 (S+1,)");
    need(uniforms.dim() == 2 && uniforms.size(0) == r && uniforms.size(1) == 2 && (plain(uniforms, at::kFloat) || plain(uniforms, at::kDouble)),
         "verify_drafts: uniforms must be contiguous float32 or float64 (R, 2)");
    need(temperature >= 1e-6 && temperature <= 1e6 && near_temperature >= 1e-6 && near_temperature <= 1e6,
         "verify_drafts: temperatures must be in 1e-6..1e6 (greedy: sample_rows and accept_path)");
    const int64_t s = start.size(0) - 1;
    const c10::cuda::CUDAGuard on(x.device());
    const auto stream = c10::cuda::getCurrentCUDAStream(x.device().index());
    const at::Tensor scratch = buffer(args[7], tf_verify_scratch_bytes((int)r, (int)v), x);
    const at::Tensor keep = at::empty({s}, tokens.options()), next = at::empty({s}, tokens.options());
    const int rc = [&] {
        const Released unlocked;
        return tf_verify_rows(x.const_data_ptr(), (size_t)x.stride(0), data_of<void>(near), near.defined() ? (size_t)near.stride(0) : 0, data_of<int>(tokens),
                              data_of<int>(start), uniforms.const_data_ptr(), uniforms.scalar_type() == at::kDouble, data_of<int>(keep), data_of<int>(next),
                              scratch.mutable_data_ptr(), bytes_of(scratch), (int)r, (int)v, (int)s, temperature, near_temperature, stream.stream());
    }();
    check_rc(rc, "verify_drafts");
    g_launches.fetch_add(2, std::memory_order_relaxed);
    PyObject* pair = PyTuple_New(2);
    if (pair == nullptr) throw PyErr{};
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(keep));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(next));
    return pair;
}

// current_stream(device index) -> cudaStream_t as an int; -1: the current device's
PyObject* stream_py(PyObject* const* args, Py_ssize_t n) {
    const int dev = n > 0 ? convert<int>(args[0]) : -1;
    return PyLong_FromVoidPtr(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
}
PyObject* device_py(PyObject* const*, Py_ssize_t) { return PyLong_FromLong(c10::cuda::current_device()); }
PyObject* count_py(PyObject* const*, Py_ssize_t) { return PyLong_FromLongLong(g_launches.load(std::memory_order_relaxed)); }

PyObject* bound_py(PyObject* const* args, Py_ssize_t n);

#define TF_FN(name, launches) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&Entry<&name, launches>::call)), METH_FASTCALL, nullptr}
#define TF_OWN(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&guarded<&fn>)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {
    TF_FN(tf_version, 0), TF_FN(tf_qmm_workers, 0), TF_FN(tf_qmm_scratch_bytes, 0), TF_FN(tf_packed_bytes, 0), TF_FN(tf_qmm, 1),
    TF_FN(tf_qmm_set_trace, 0), TF_FN(tf_qmm_next, 1), TF_FN(tf_qmm_grouped, 1), TF_FN(tf_pack_rows, 1), TF_FN(tf_qmm_tiled_bytes, 0),
    TF_FN(tf_qmm_tile, 1), TF_FN(tf_qmm_untile, 1), TF_FN(tf_packed_tc_bytes, 0), TF_FN(tf_qmm_tc_tiled_bytes, 0), TF_FN(tf_qmm_tc, 1),
    TF_FN(tf_pack_rows_tc, 1), TF_FN(tf_qmm_tc_set_trace, 0), TF_FN(tf_repack_tc, 1), TF_FN(tf_qmm_tc_tile, 1), TF_FN(tf_qmm_tc_untile, 1),
    TF_FN(tf_norm_xs, 1), TF_FN(tf_swiglu, 1), TF_FN(tf_gated_norm, 1), TF_FN(tf_gate_mul, 1), TF_FN(tf_attn_prep, 1), TF_FN(tf_gdn_pre, 1),
    TF_FN(tf_embed, 1), TF_FN(tf_gdn_chain, 1), TF_FN(tf_gdn_fused, 1), TF_FN(tf_gdn_replay, 1), TF_FN(tf_conv_commit, 1),
    TF_FN(tf_attention_scratch_bytes, 0), TF_FN(tf_attention_chunks, 0), TF_FN(tf_lane_attention_paged_gated, 2),
    TF_FN(tf_lane_attention_paged, 2), TF_FN(tf_lane_attention_paged_static, 2), TF_FN(tf_kv_commit, 1), TF_FN(tf_moe_max_problems, 0),
    TF_FN(tf_moe_router, 1), TF_FN(tf_moe_select, 1), TF_FN(tf_moe_group, 1), TF_FN(tf_moe_slot_bytes, 0), TF_FN(tf_moe_push, 1),
    TF_FN(tf_moe_combine_peer, 1), TF_FN(tf_moe_pack, 1), TF_FN(tf_moe_act, 1), TF_FN(tf_moe_combine, 1), TF_FN(tf_peer_slot_bytes, 0),
    TF_FN(tf_peer_exchange, 1), TF_FN(tf_qmm_act, 1), TF_FN(tf_swiglu_tiled, 1), TF_FN(tf_qmm_peer, 1), TF_FN(tf_norm_xs_peer, 1),
    TF_FN(tf_set_poll_limit, 0), TF_FN(tf_topk_scratch_bytes, 0), TF_FN(tf_topk_rows, 2), TF_FN(tf_topk_sample_rows, 2), TF_FN(tf_sample_rows, 1),
    TF_FN(tf_window_chunk_keys, 0), TF_FN(tf_window_slots, 0), TF_FN(tf_window_scratch_bytes, 0), TF_FN(tf_window_launches, 0),
    TF_FN(tf_window_attention, 2), TF_FN(tf_attention_mass, 1),        // (without a plan; window_attention() counts it)
    TF_FN(tf_evict_scratch_bytes, 0), TF_FN(tf_kv_evict, 2), TF_FN(tf_verify_scratch_bytes, 0), TF_FN(tf_verify_rows, 2),
    TF_OWN("bound", bound_py), TF_OWN("scratch", scratch_py), TF_OWN("lane_matmul", lane_matmul_py), TF_OWN("prefill_matmul", prefill_matmul_py),
    TF_OWN("window_attention", window_attention_py), TF_OWN("attention_mass", attention_mass_py), TF_OWN("evict", evict_py),
    TF_OWN("verify_drafts", verify_drafts_py),
    TF_OWN("current_stream", stream_py), TF_OWN("current_device", device_py), TF_OWN("launch_count", count_py),
    {nullptr, nullptr, 0, nullptr}};

// bound(name, fn): the entry point `name`, with `fn` (the same one through ctypes) for the arguments it does not convert itself
PyObject* bound_py(PyObject* const* args, Py_ssize_t n) {
    const char* name = n == 2 ? PyUnicode_AsUTF8(args[0]) : nullptr;
    if (name == nullptr) fail(PyExc_TypeError, "bound(name, function)");
    for (PyMethodDef* def = methods; def->ml_name != nullptr; ++def)
        if (std::strcmp(def->ml_name, name) == 0) return PyCFunction_NewEx(def, args[1], nullptr);
    fail(PyExc_AttributeError, name);
}

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Native binding of libtensorfold_b200.so", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
