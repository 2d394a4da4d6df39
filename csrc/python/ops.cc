// ops.cc - operators on torch tensors as Python functions (module _ops): arguments checked, results made, launched on the current stream.
//
// An op on small tensors is bound by its host path, not by its kernel. Of the 9 us of a norm with five results, 2.7 were the checks in Python and 3.8 its
// tensors made through torch's Python interface, beside a launch of 2.6; of the rotation's 6, 3.3 the checks. Here a check costs nothing to speak of, an allocation
// 0.5 us and a tensor made of one less than 0.1, so that results that are kept and dropped together share one: the norm 5.9 -> 4.2 us, windowed
// attention forward 4.3 -> 3.5, backward of 333 tokens, 8 heads 9.6 -> 8.5. What an op refuses raises KernelError, which bind() is given; the documentation stands in
// cai_b200/ops.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "../kernels/cai_kernels.h"

namespace {

PyObject* g_error = nullptr;     // KernelError

struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct Raised {};    // the Python exception is set

void need(bool ok, const char* op, const char* what) {
    if (__builtin_expect(!ok, 0)) throw Refused(std::string(op) + ": " + what);
}
void launched(int rc, const char* op) {
    if (__builtin_expect(rc != 0, 0)) throw Refused(std::string(op) + " failed (rc=" + std::to_string(rc) + "): " + cai_last_error());
}
// A launch waits when the stream's queue is full: others may run meanwhile. What is thrown meanwhile finds the thread's state restored; tensors are asked for their
// addresses before, since that is what throws (under torch.vmap they have none).
struct WithoutGil {
    PyThreadState* const state = PyEval_SaveThread();
    WithoutGil() = default;
    WithoutGil(const WithoutGil&) = delete;
    ~WithoutGil() { PyEval_RestoreThread(state); }
};
template <typename F> int without_gil(F&& f) {
    const WithoutGil released;
    return f();
}

// ---------------------------------------------------------------- arguments
const at::Tensor& tensor(PyObject* o, const char* op) {
    need(THPVariable_Check(o), op, "a tensor is wanted");
    return THPVariable_Unpack(o);
}
const at::Tensor* tensor_or_none(PyObject* o, const char* op) { return o == Py_None ? nullptr : &tensor(o, op); }
long long integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return v;
}
// As the launchers take it: a number that does not fit is no number of rows, heads or columns.
int small(PyObject* o, const char* op) {
    const long long v = integer(o);
    need(v >= -0x7fffffffll && v <= 0x7fffffffll, op, "a number is out of range");
    return static_cast<int>(v);
}
// A window or a number of sinks: any number of keys, of which no sequence has more than 2^31 - 1.
int keys(PyObject* o) {
    const long long v = integer(o);
    return v > 0x7fffffffll ? 0x7fffffff : v < -1 ? -1 : static_cast<int>(v);
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised();
    return v != 0;
}
bool shaped(const at::Tensor& t, int64_t a, int64_t b) { return t.dim() == 2 && t.size(0) == a && t.size(1) == b; }

// The stream of a call on these tensors, which have to be the current device's: a launch goes to that device's current stream.
struct Place {
    at::Device device;
    void* stream;
};
Place place(const char* op, std::initializer_list<const at::Tensor*> tensors) {
    for (const at::Tensor* t : tensors)
        if (t) {
            need(t->is_cuda() && t->layout() == at::kStrided, op, "a tensor is not on the current device");
            // Of a wrapper, a fake tensor or one whose storage was given back an address is nothing, or nothing and an offset.
            need(t->numel() == 0 || (t->has_storage() && t->storage().data()), op, "a tensor has no memory");
        }
    const c10::DeviceIndex device = c10::cuda::current_device();
    for (const at::Tensor* t : tensors)
        if (t) need(t->get_device() == device, op, "a tensor is not on the current device");
    return {at::Device(at::kCUDA, device), c10::cuda::getCurrentCUDAStream(device).stream()};
}

at::Tensor make(const Place& at, at::ScalarType type, std::initializer_list<int64_t> sizes) {
    return at::Tensor(at::detail::empty_cuda(at::IntArrayRef(sizes), type, at.device, std::nullopt));
}
// Results that live and die together in one piece of memory, one behind the other, each a whole number of 16 bytes behind the start: an allocation costs more than
// the tensor made of it.
struct Piece {
    c10::Storage memory;
    int64_t at = 0;
    explicit Piece(int64_t bytes)
        : memory(c10::make_intrusive<c10::StorageImpl>(c10::StorageImpl::use_byte_size_t(), bytes, c10::cuda::CUDACachingAllocator::get(), true)) {}
    at::Tensor make(at::ScalarType type, std::initializer_list<int64_t> sizes) {
        const auto meta = c10::scalarTypeToTypeMeta(type);
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(memory), c10::DispatchKeySet(c10::DispatchKey::CUDA), meta);
        c10::TensorImpl* impl = t.unsafeGetTensorImpl();
        impl->set_storage_offset(at / static_cast<int64_t>(meta.itemsize()));
        impl->set_sizes_contiguous(at::IntArrayRef(sizes));
        at += impl->numel() * static_cast<int64_t>(meta.itemsize());
        return t;
    }
};
void* p(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T> T* p(const at::Tensor& t) { return static_cast<T*>(p(t)); }

// Calls an op's body; what it throws becomes a Python exception.
template <PyObject* (*kBody)(PyObject* const*)> PyObject* guarded(PyObject* const* args, Py_ssize_t n, Py_ssize_t wanted) {
    if (n != wanted) {
        PyErr_Format(PyExc_TypeError, "%zd arguments are wanted, %zd given", wanted, n);
        return nullptr;
    }
    HANDLE_TH_ERRORS
    try {
        return kBody(args);
    } catch (const Refused& e) {
        PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
        return nullptr;
    } catch (const Raised&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- the operators
// (x, residual, g, eps, keep_y) -> (h, q, s, rstd, y)
PyObject* add_rmsnorm_quant(PyObject* const* a) {
    constexpr const char* op = "add_rmsnorm_quant";
    const at::Tensor &x = tensor(a[0], op), &g = tensor(a[2], op);
    const at::Tensor* residual = tensor_or_none(a[1], op);
    need(x.scalar_type() == at::kBFloat16 && g.scalar_type() == at::kBFloat16 && x.dim() == 2, op, "x is bf16 [rows, H], g bf16 [H]");
    const int64_t rows = x.size(0), H = x.size(1);
    need(rows <= 0x7fffffff && H <= 0x7fffffff, op, "too many rows or columns");
    need(g.dim() == 1 && g.size(0) == H && g.is_contiguous(), op, "g has one element a column");
    need(H < 2 || x.stride(1) == 1, op, "rows of x have to be contiguous");
    if (residual)
        need(residual->scalar_type() == at::kBFloat16 && shaped(*residual, rows, H) && (H < 2 || residual->stride(1) == 1), op, "the residual is like x");
    const bool keep_y = truth(a[4]);
    const float eps = static_cast<float>(real(a[3]));
    const Place at = place(op, {&x, residual, &g});
    // what the backward pass keeps, and what the product reads
    need(H > 0 && H % 128 == 0, op, "needs a multiple of 128 columns");
    Piece kept(rows * H * 2 * ((residual != nullptr) + keep_y) + rows * 4), read(rows * H + rows * (H / 128) * 4);
    const at::Tensor h = residual ? kept.make(at::kBFloat16, {rows, H}) : at::Tensor(), y = keep_y ? kept.make(at::kBFloat16, {rows, H}) : at::Tensor();
    const at::Tensor rstd = kept.make(at::kFloat, {rows}), q = read.make(at::kFloat8_e4m3fn, {rows, H}), s = read.make(at::kFloat, {rows, H / 128});
    const int64_t ldx = rows > 1 ? x.stride(0) : 0, ldr = residual && rows > 1 ? residual->stride(0) : 0;
    const void *xp = p(x), *rp = residual ? p(*residual) : nullptr, *gp = p(g);
    void *hp = p(h), *yp = p(y), *qp = p(q);
    float *sp = p<float>(s), *rstdp = p<float>(rstd);
    launched(without_gil([&] {
        return cai_add_rmsnorm_quant(xp, ldx, rp, ldr, gp, hp, yp, qp, sp, rstdp, static_cast<int>(rows), static_cast<int>(H), eps, at.stream);
    }), op);
    THPObjectPtr out(PyTuple_New(5));
    if (!out) throw Raised();
    PyTuple_SET_ITEM(out.get(), 0, residual ? THPVariable_Wrap(h) : Py_NewRef(a[0]));
    PyTuple_SET_ITEM(out.get(), 1, THPVariable_Wrap(q));
    PyTuple_SET_ITEM(out.get(), 2, THPVariable_Wrap(s));
    PyTuple_SET_ITEM(out.get(), 3, THPVariable_Wrap(rstd));
    PyTuple_SET_ITEM(out.get(), 4, keep_y ? THPVariable_Wrap(y) : Py_NewRef(Py_None));
    return out.release();
}

// (qkv, freqs, pos, nh, nkv, hd, sections, interleaved, inverse) -> qkv
PyObject* rope_apply_axes(PyObject* const* a) {
    constexpr const char* op = "rope_apply_axes_";
    const at::Tensor &qkv = tensor(a[0], op), &freqs = tensor(a[1], op), &pos = tensor(a[2], op);
    const int nh = small(a[3], op), nkv = small(a[4], op), hd = small(a[5], op);
    THPObjectPtr sections(PySequence_Fast(a[6], "the sections are a sequence of numbers"));
    if (!sections) throw Raised();
    const Py_ssize_t axes = PySequence_Fast_GET_SIZE(sections.get());
    need(axes >= 1 && axes <= 4, op, "there are one to four axes");
    int n[4] = {0, 0, 0, 0};
    for (Py_ssize_t i = 0; i < axes; ++i) n[i] = small(PySequence_Fast_GET_ITEM(sections.get(), i), op);
    const bool interleaved = truth(a[7]), inverse = truth(a[8]);
    need(qkv.scalar_type() == at::kBFloat16 && qkv.dim() == 2, op, "qkv is bf16 [T, columns]");
    const int64_t T = qkv.size(0), cols = qkv.size(1);
    need(T <= 0x7fffffff, op, "too many rows");
    need(nh >= 0 && nkv >= 0 && hd > 0 && cols >= (static_cast<int64_t>(nh) + nkv) * hd, op, "qkv holds fewer columns than its q and k heads");
    need((cols < 2 || qkv.stride(1) == 1) && (T < 2 || qkv.stride(0) >= cols), op, "rows of qkv have to be contiguous and apart");
    need(pos.scalar_type() == at::kInt && shaped(pos, axes, T) && (T < 2 || pos.stride(1) == 1), op, "pos is int32 [axes, T], an axis' positions contiguous");
    need(freqs.scalar_type() == at::kDouble && freqs.dim() == 1 && freqs.size(0) == hd / 2 && freqs.is_contiguous(), op, "freqs is f64 [hd / 2]");
    const Place at = place(op, {&qkv, &freqs, &pos});
    const int64_t ldp = axes > 1 ? pos.stride(0) : 0, ld = T > 1 ? qkv.stride(0) : (cols + 7) / 8 * 8;
    void* qkvp = p(qkv);
    const double* freqsp = p<double>(freqs);
    const int* posp = p<int>(pos);
    launched(without_gil([&] {
        return cai_rope_apply_axes(qkvp, freqsp, posp, ldp, static_cast<int>(T), nh, nkv, hd, ld, static_cast<int>(axes), n[0], n[1], n[2], n[3], interleaved, inverse,
                                   at.stream);
    }), op);
    return Py_NewRef(a[0]);
}

// Row pitch of a packed [B * S, cols] bf16 tensor.
int64_t packed_pitch(const char* op, const at::Tensor& t, int64_t rows, int64_t cols) {
    need(t.scalar_type() == at::kBFloat16 && shaped(t, rows, cols), op, "needs bf16 [B * S, (heads + 2 kv_heads) * head_dim]");
    need((cols < 2 || t.stride(1) == 1) && (rows < 2 || t.stride(0) >= cols), op, "rows have to be contiguous and apart");
    return rows > 1 ? t.stride(0) : cols;
}
// Do two packed tensors share memory? (Columns of one buffer beside each other do not.)
bool overlap(const at::Tensor& a, int64_t lda, const at::Tensor& b, int64_t ldb) {
    if (a.numel() == 0 || b.numel() == 0) return false;
    const auto at = reinterpret_cast<uintptr_t>(a.data_ptr()) / 2, bt = reinterpret_cast<uintptr_t>(b.data_ptr()) / 2;     // in elements
    if (at + (a.size(0) - 1) * lda + a.size(1) <= bt || bt + (b.size(0) - 1) * ldb + b.size(1) <= at) return false;
    if (lda != ldb) return true;
    const int64_t off = ((static_cast<int64_t>(bt) - static_cast<int64_t>(at)) % lda + lda) % lda;     // b's first column, from a's
    return off < a.size(1) || off + b.size(1) > lda;
}
// Workspaces are written while everything else is in use.
bool overlap(const at::Tensor& a, const at::Tensor& b) {
    const auto end = [](const at::Tensor& t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        return reinterpret_cast<uintptr_t>(t.data_ptr()) + (last + 1) * t.element_size();
    };
    if (a.numel() == 0 || b.numel() == 0) return false;
    return reinterpret_cast<uintptr_t>(a.data_ptr()) < end(b) && reinterpret_cast<uintptr_t>(b.data_ptr()) < end(a);
}
struct WindowCall {
    int B, S, nh, nkv, hd, window, sinks;
    float scale;
    int64_t rows, cols;
    // args: B, S, nh, nkv, hd, window, sinks, scale (None: hd ** -0.5)
    WindowCall(PyObject* const* a, const char* op)
        : B(small(a[0], op)), S(small(a[1], op)), nh(small(a[2], op)), nkv(small(a[3], op)), hd(small(a[4], op)), window(keys(a[5])), sinks(keys(a[6])) {
        need(B >= 0 && S >= 0 && nh > 0 && nkv > 0 && hd > 0, op, "needs sequences, heads and a head dimension");
        scale = static_cast<float>(a[7] == Py_None ? 1.0 / std::sqrt(static_cast<double>(hd)) : real(a[7]));
        rows = static_cast<int64_t>(B) * S;
        cols = (static_cast<int64_t>(nh) + 2 * static_cast<int64_t>(nkv)) * hd;
    }
};

// (qkv, B, S, nh, nkv, hd, window, sinks, scale) -> (out, lse)
PyObject* window_fwd(PyObject* const* a) {
    constexpr const char* op = "flash_attn_window_fwd";
    const at::Tensor& qkv = tensor(a[0], op);
    const WindowCall c(a + 1, op);
    const int64_t ld = packed_pitch(op, qkv, c.rows, c.cols);
    const Place at = place(op, {&qkv});
    const int64_t width = static_cast<int64_t>(c.nh) * c.hd;
    need(c.hd % 8 == 0, op, "needs a head dimension of a multiple of 8");
    Piece both_of(c.rows * width * 2 + c.rows * c.nh * 4);
    const at::Tensor out = both_of.make(at::kBFloat16, {c.rows, width}), lse = both_of.make(at::kFloat, {c.B, c.nh, c.S});
    const void* qkvp = p(qkv);
    void* outp = p(out);
    float* lsep = p<float>(lse);
    launched(without_gil([&] {
        return cai_flash_attn_window_fwd(qkvp, ld, outp, lsep, c.B, c.S, c.nh, c.nkv, c.hd, c.scale, c.window, c.sinks, at.stream);
    }), op);
    THPObjectPtr both(PyTuple_New(2));
    if (!both) throw Raised();
    PyTuple_SET_ITEM(both.get(), 0, THPVariable_Wrap(out));
    PyTuple_SET_ITEM(both.get(), 1, THPVariable_Wrap(lse));
    return both.release();
}

// (qkv, out, dout, lse, B, S, nh, nkv, hd, window, sinks, scale, dqkv, delta, scratch) -> dqkv
PyObject* window_bwd(PyObject* const* a) {
    constexpr const char* op = "flash_attn_window_bwd";
    const at::Tensor &qkv = tensor(a[0], op), &out = tensor(a[1], op), &dout = tensor(a[2], op), &lse = tensor(a[3], op);
    const WindowCall c(a + 4, op);
    const at::Tensor *dqkv = tensor_or_none(a[12], op), *delta = tensor_or_none(a[13], op), *scratch = tensor_or_none(a[14], op);
    const int64_t ld = packed_pitch(op, qkv, c.rows, c.cols), ldq = dqkv ? packed_pitch(op, *dqkv, c.rows, c.cols) : c.cols;
    const int64_t width = static_cast<int64_t>(c.nh) * c.hd, stats = c.rows * c.nh;
    for (const at::Tensor* t : {&out, &dout}) {
        need(t->scalar_type() == at::kBFloat16 && shaped(*t, c.rows, width) && t->is_contiguous(), op, "out and dout are bf16 [B * S, heads * head_dim]");
        need(!dqkv || !overlap(*t, width, *dqkv, ldq), op, "dqkv shares memory with what is read");
    }
    need(!dqkv || !overlap(qkv, ld, *dqkv, ldq), op, "dqkv shares memory with what is read");
    need(lse.scalar_type() == at::kFloat && lse.dim() == 3 && lse.size(0) == c.B && lse.size(1) == c.nh && lse.size(2) == c.S && lse.is_contiguous(), op,
         "lse is f32 [B, heads, S]");
    need(!dqkv || !overlap(lse, *dqkv), op, "dqkv shares memory with what is read");
    if (delta) need(delta->scalar_type() == at::kFloat && delta->numel() >= stats && delta->is_contiguous(), op, "delta is f32 [B, heads, S]");
    for (const at::Tensor* w : {delta, scratch})
        for (const at::Tensor* t : {&qkv, &out, &dout, &lse, dqkv, w == scratch ? delta : nullptr})
            need(!w || !t || !overlap(*w, *t), op, "a workspace shares memory with another argument");
    const Place at = place(op, {&qkv, &out, &dout, &lse, dqkv, delta, scratch});
    const int64_t bytes = cai_flash_attn_window_bwd_scratch(c.B, c.S, c.nh, c.nkv, c.window, c.sinks);
    if (scratch) need(static_cast<int64_t>(scratch->nbytes()) >= bytes && scratch->is_contiguous(), op, "the scratch is too small, see flash_attn_window_bwd_scratch");
    const at::Tensor made = dqkv ? at::Tensor() : make(at, at::kBFloat16, {c.rows, c.cols});
    Piece work((scratch ? 0 : bytes) + (delta ? 0 : stats * 4));
    const at::Tensor parts = scratch ? *scratch : bytes ? work.make(at::kByte, {bytes}) : at::Tensor(), sums = delta ? *delta : work.make(at::kFloat, {stats});
    const void *qkvp = p(qkv), *outp = p(out), *doutp = p(dout);
    const float* lsep = p<float>(lse);
    float* sumsp = p<float>(sums);
    void *dqkvp = dqkv ? p(*dqkv) : p(made), *partsp = p(parts);
    launched(without_gil([&] {
        return cai_flash_attn_window_bwd(qkvp, ld, outp, doutp, lsep, sumsp, dqkvp, ldq, partsp, c.B, c.S, c.nh, c.nkv, c.hd, c.scale, c.window, c.sinks, at.stream);
    }), op);
    return dqkv ? Py_NewRef(a[12]) : THPVariable_Wrap(made);
}

// bind(KernelError): what the operators raise.
PyObject* bind(PyObject*, PyObject* error) {
    Py_INCREF(error);
    Py_XSETREF(g_error, error);
    Py_RETURN_NONE;
}

template <PyObject* (*kBody)(PyObject* const*), Py_ssize_t kArgs> PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded<kBody>(args, n, kArgs);
}
#define OP(name, body, args) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<&body, args>)), METH_FASTCALL, nullptr}
PyMethodDef functions[] = {
    {"bind", &bind, METH_O, nullptr},
    OP("add_rmsnorm_quant", add_rmsnorm_quant, 5),
    OP("rope_apply_axes_", rope_apply_axes, 9),
    OP("flash_attn_window_fwd", window_fwd, 9),
    OP("flash_attn_window_bwd", window_bwd, 15),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, functions, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&module); }
