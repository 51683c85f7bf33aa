// sx8_py.cpp -- the per-call host path of the Python wrappers, as a CPython module.
//
// A linear layer's kernel on one token takes 4-9 us; argument conversion for a 14-argument
// ctypes call, the stream query and the output allocation in Python took 11-12 (6.0 now for
// 1024 x 2560 and one token, launch included, and 7.4 for 2560 x 9728, where the kernel bounds
// it; 512 embedding rows 13.0 -> 6.4, a whole 9728 x 2560 weight back to fp16 22.5 -> 16.9).
// Each function here does what the wrapper of the same name does for the calls a runtime makes
// all the time -- plain device tensors of the right type -- and returns None for every other
// call, which the wrapper then takes through its general path (conversions, copies, padding,
// error messages); without the module every call goes there.  The library's entry points are bound by address from the copy that ctypes
// loaded, so both paths run the same library, and as in a ctypes call the interpreter lock is
// given up while a launch or an allocation may wait.  Nothing is kept between calls.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <string>

#include "sx8_draft.h"
#include "sx8_hip.h"
#include "sx8_paged.h"

namespace {

typedef const void* CP;
struct Lib {
    int32_t (*abi_version)();
    const char* (*last_error)();
    int32_t (*linear)(CP, int64_t, int64_t, int64_t, CP, CP, int32_t, CP, CP, CP, int64_t, int64_t, void*, void*);
    int32_t (*gemv)(CP, CP, CP, int32_t, CP, CP, CP, void*, int64_t, int64_t, void*, void*, int64_t, void*);
    int64_t (*gemm_ws)(int64_t, int32_t, const int64_t*, int64_t);
    int32_t (*gemm)(CP, int64_t, int64_t, int64_t, CP, CP, int32_t, CP, CP, int64_t, int64_t, void*, void*, int64_t,
                    void*);
    int32_t (*gemm_split)(CP, int64_t, int64_t, int64_t, CP, CP, CP, CP, CP, CP, CP, CP, int64_t, int64_t, void*, void*,
                          int64_t, void*);
    int32_t (*dequant)(CP, CP, CP, CP, CP, CP, CP, CP, int64_t, int64_t, int64_t, void*, void*);
    int32_t (*embed)(CP, int64_t, CP, CP, int32_t, CP, CP, int64_t, int64_t, int64_t, void*, void*);
    decltype(&sx8_attn_varlen) varlen;
    decltype(&sx8_attn_varlen_workspace_bytes) varlen_ws;
    decltype(&sx8_kv4_append) kv4_append;
    decltype(&sx8_kv4_read) kv4_read;
    decltype(&sx8_kv4_attend) kv4_attend;
    decltype(&sx8_kv4_reserve_marked) kv4_reserve;
    decltype(&sx8_kv4_fork) kv4_fork;
    decltype(&sx8_kv4_free) kv4_free;
    decltype(&sx8_kv4_compact) kv4_compact;
    decltype(&sx8_kv4_append_rope_marked) kv4_append_rope;
    decltype(&sx8_kv4_attend_tree) kv4_attend_tree;
    decltype(&sx8_kv4_keep_marked) kv4_keep;
    decltype(&sx8_kv4_keep_workspace_bytes) kv4_keep_ws;
    decltype(&sx8_draft_tree) draft_tree;
    decltype(&sx8_draft_verify_within) draft_verify;
    decltype(&sx8_draft_verify_workspace_bytes) draft_verify_ws;
} lib;

constexpr int32_t kUnsupported = SX8_ERR_UNSUPPORTED;
constexpr int64_t kLinearRows = 32, kLdsMaxKb = 640;

// A plain tensor (or Parameter) whose memory holds its values, else null: subclasses, the wrappers of
// function transforms (vmap, jvp) and views that negate on reading go through the general path.
const at::Tensor* plain(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    using K = c10::DispatchKey;
    const at::Tensor& x = THPVariable_Unpack(o);
    static const c10::DispatchKeySet other({K::FuncTorchBatched, K::FuncTorchGradWrapper, K::Batched, K::Functionalize, K::Python,
                                     K::Conjugate, K::Negative, K::ZeroTensor});
    return x.key_set().has_any(other) ? nullptr : &x;
}

const at::Tensor* dev(PyObject* o, at::ScalarType t) {
    const at::Tensor* x = plain(o);
    return x && x->is_cuda() && x->layout() == at::kStrided && x->scalar_type() == t ? x : nullptr;
}

const at::Tensor* dense(PyObject* o, at::ScalarType t) {
    const at::Tensor* x = dev(o, t);
    return x && x->is_contiguous() ? x : nullptr;
}

typedef pybind11::gil_scoped_release Unlocked;

int64_t num(PyObject* o) { return PyLong_AsLongLong(o); }

// A size that is no integer (a float, say) is the general path's to convert or refuse.
#define SX8_SIZES_OK()      \
    if (PyErr_Occurred()) { \
        PyErr_Clear();      \
        Py_RETURN_NONE;     \
    }

void* stream_of(const at::Tensor& x) { return c10::hip::getCurrentHIPStream(x.device().index()).stream(); }

PyObject* failed(const char* name, int32_t rc) {
    PyErr_Format(PyExc_RuntimeError, "%s failed (code %d): %s", name, (int)rc, lib.last_error());
    return nullptr;
}

at::Tensor empty_like_device(at::IntArrayRef sizes, at::ScalarType t, const at::Tensor& x) {
    return at::empty(sizes, at::TensorOptions().dtype(t).device(x.device()));
}

#define SX8_ARGS(n)                                                                \
    if (na != (n)) {                                                               \
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %d", n, (int)na); \
        return nullptr;                                                            \
    }

// bind({name: address}): RuntimeError for a library of another ABI version.
PyObject* py_bind(PyObject*, PyObject* d) {
    auto get = [&](const char* name) -> void* {
        PyObject* v = PyDict_GetItemString(d, name);
        if (!v) PyErr_Format(PyExc_KeyError, "%s", name);
        return v ? PyLong_AsVoidPtr(v) : nullptr;
    };
#define SX8_BIND(field, name) \
    if (!(lib.field = reinterpret_cast<decltype(lib.field)>(get(name)))) return nullptr;
    SX8_BIND(abi_version, "sx8_abi_version")
    if (lib.abi_version() != SX8_ABI_VERSION) {
        PyErr_Format(PyExc_RuntimeError, "built for ABI version %d, the library has %d", SX8_ABI_VERSION,
                     (int)lib.abi_version());
        return nullptr;
    }
    SX8_BIND(last_error, "sx8_last_error")
    SX8_BIND(linear, "sx8_linear_f16")
    SX8_BIND(gemv, "sx8_gemv")
    SX8_BIND(gemm_ws, "sx8_gemm_prefill_workspace_bytes")
    SX8_BIND(gemm, "sx8_gemm_prefill")
    SX8_BIND(gemm_split, "sx8_gemm_prefill_split")
    SX8_BIND(dequant, "sx8_dequant_f16")
    SX8_BIND(embed, "sx8_embed_gather")
    SX8_BIND(varlen, "sx8_attn_varlen")
    SX8_BIND(varlen_ws, "sx8_attn_varlen_workspace_bytes")
    SX8_BIND(kv4_append, "sx8_kv4_append")
    SX8_BIND(kv4_read, "sx8_kv4_read")
    SX8_BIND(kv4_attend, "sx8_kv4_attend")
    SX8_BIND(kv4_reserve, "sx8_kv4_reserve_marked")
    SX8_BIND(kv4_fork, "sx8_kv4_fork")
    SX8_BIND(kv4_free, "sx8_kv4_free")
    SX8_BIND(kv4_compact, "sx8_kv4_compact")
    SX8_BIND(kv4_append_rope, "sx8_kv4_append_rope_marked")
    SX8_BIND(kv4_attend_tree, "sx8_kv4_attend_tree")
    SX8_BIND(kv4_keep, "sx8_kv4_keep_marked")
    SX8_BIND(kv4_keep_ws, "sx8_kv4_keep_workspace_bytes")
    SX8_BIND(draft_tree, "sx8_draft_tree")
    SX8_BIND(draft_verify, "sx8_draft_verify_within")
    SX8_BIND(draft_verify_ws, "sx8_draft_verify_workspace_bytes")
#undef SX8_BIND
    Py_RETURN_NONE;
}

// linear(x, (hdr, levels, bases, scales), hdr_bytes, bias, out_f, N, in_f, n_cb): fp16(x W^T) (+ bias) of
// up to 32 rows, shape (*x.shape[:-1], out_f).
PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(8)
    const at::Tensor* x = dev(a[0], at::kHalf);
    if (!x || x->dim() < 1 || !PyTuple_Check(a[1]) || PyTuple_GET_SIZE(a[1]) != 4) Py_RETURN_NONE;
    const int64_t out_f = num(a[4]), N = num(a[5]), K = num(a[6]), n_cb = num(a[7]), hb = num(a[2]);
    SX8_SIZES_OK()
    const int64_t M = K > 0 && x->size(-1) == K ? x->numel() / K : 0;
    // (K blocks that are not the row's: decode1_v44 cuts or pads the row, the GEMM refuses)
    if (M < 1 || M > kLinearRows || out_f != N || n_cb != (K + 31) / 32) Py_RETURN_NONE;
    if (M > 1) {
        const char* wmma = std::getenv("SX8_USE_WMMA");
        if (N < 64 || (wmma && std::strcmp(wmma, "1") == 0)) Py_RETURN_NONE;
    }
    const at::Tensor* t[4];
    for (int i = 0; i < 4; ++i)
        if (!(t[i] = plain(PyTuple_GET_ITEM(a[1], i))) || t[i]->device() != x->device()) Py_RETURN_NONE;
    const at::Tensor* b = nullptr;
    if (a[3] != Py_None) {
        b = dense(a[3], at::kHalf);
        // (a bias that either mode of autograd follows is added by torch)
        if (!b || b->device() != x->device() || b->dim() != 1 || b->size(0) != N ||
            (b->requires_grad() && c10::GradMode::is_enabled()) || b->_fw_grad(0).defined())
            Py_RETURN_NONE;
    }
    c10::SmallVector<int64_t, 5> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = N;
    at::Tensor y;
    int32_t rc;
    {
        Unlocked u;
        const at::Tensor xc = x->is_contiguous() ? *x : x->contiguous();
        y = empty_like_device(shape, at::kHalf, *x);
        rc = lib.linear(xc.data_ptr(), M, K, K, t[0]->data_ptr(), t[1]->data_ptr(), (int32_t)hb, t[2]->data_ptr(),
                        t[3]->data_ptr(), b ? b->data_ptr() : nullptr, N, n_cb, y.data_ptr(), stream_of(*x));
    }
    if (rc == kUnsupported) Py_RETURN_NONE;
    if (rc) return failed("sx8_linear_f16", rc);
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// gemv(x, hdr, levels, bases, scales, hdr_bytes, N, n_cb, Y): True, or None.
PyObject* py_gemv(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(9)
    const at::Tensor* x = dense(a[0], at::kHalf);
    const at::Tensor* y = dense(a[8], at::kFloat);
    const int64_t N = num(a[6]), n_cb = num(a[7]), hb = num(a[5]);
    SX8_SIZES_OK()
    if (!x || !y || n_cb > kLdsMaxKb || x->numel() != n_cb * 32 || y->numel() != N || x->device() != y->device())
        Py_RETURN_NONE;
    if (reinterpret_cast<uintptr_t>(x->data_ptr()) & 15) Py_RETURN_NONE;
    const at::Tensor* t[4];
    for (int i = 0; i < 4; ++i)
        if (!(t[i] = plain(a[1 + i]))) Py_RETURN_NONE;
    int32_t rc;
    {
        Unlocked u;
        rc = lib.gemv(x->data_ptr(), t[0]->data_ptr(), t[1]->data_ptr(), (int32_t)hb, t[2]->data_ptr(), t[3]->data_ptr(), nullptr,
                      nullptr, N, n_cb, y->data_ptr(), nullptr, 0, stream_of(*x));
    }
    if (rc) return failed("sx8_gemv", rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// X (M, K) fp16 dense with the output and workspace of its product.
struct GemmCall {
    const at::Tensor* x;
    int64_t M, K, N, n_cb, ws_bytes;
    at::Tensor ws, y;
    bool make(PyObject* X, int64_t N_, int64_t n_cb_) {          // false: the general path
        x = dense(X, at::kHalf);
        if (!x || x->dim() != 2 || x->size(0) < 1) return false;
        M = x->size(0);
        K = x->size(1);
        N = N_;
        n_cb = n_cb_;
        ws_bytes = lib.gemm_ws(M, 1, &N, n_cb);
        return ws_bytes >= 0;
    }
    void allocate() {
        y = empty_like_device({M, N}, at::kFloat, *x);
        ws = empty_like_device({std::max<int64_t>(ws_bytes, 256)}, at::kByte, *x);
    }
};

// gemm(X, hdr, levels, bases, scales, hdr_bytes, N, in_f, n_cb): Y (M, N) float32, or None.
PyObject* py_gemm(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(9)
    const at::Tensor* t[4];
    for (int i = 0; i < 4; ++i)
        if (!(t[i] = plain(a[1 + i]))) Py_RETURN_NONE;
    GemmCall c;
    const int64_t N = num(a[6]), in_f = num(a[7]), n_cb = num(a[8]), hb = num(a[5]);
    SX8_SIZES_OK()
    if (!c.make(a[0], N, n_cb) || c.K < in_f) Py_RETURN_NONE;
    int32_t rc;
    {
        Unlocked u;
        c.allocate();
        rc = lib.gemm(c.x->data_ptr(), c.M, c.K, in_f, t[0]->data_ptr(), t[1]->data_ptr(), (int32_t)hb, t[2]->data_ptr(),
                      t[3]->data_ptr(), c.N, c.n_cb, c.y.data_ptr(), c.ws.data_ptr(), c.ws_bytes, stream_of(*c.x));
    }
    if (rc) return failed("sx8_gemm_prefill", rc);
    return THPVariable_Wrap(std::move(c.y));
    END_HANDLE_TH_ERRORS
}

// gemm_split(X, dmin, dmax, config, coeff, hi, lo, basis, scales, n_cb): Y (M, N) float32, or None.
PyObject* py_gemm_split(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(10)
    const at::Tensor* t[8];
    for (int i = 0; i < 8; ++i)
        if (!(t[i] = plain(a[1 + i]))) Py_RETURN_NONE;
    const int64_t n_cb = num(a[9]);
    SX8_SIZES_OK()
    GemmCall c;
    if (n_cb < 1 || !c.make(a[0], t[0]->numel() / n_cb, n_cb)) Py_RETURN_NONE;
    int32_t rc;
    {
        Unlocked u;
        c.allocate();
        rc = lib.gemm_split(c.x->data_ptr(), c.M, c.K, std::min(c.K, n_cb * 32), t[0]->data_ptr(), t[1]->data_ptr(),
                            t[2]->data_ptr(), t[3]->data_ptr(), t[4]->data_ptr(), t[5]->data_ptr(), t[6]->data_ptr(),
                            t[7]->data_ptr(), c.N, n_cb, c.y.data_ptr(), c.ws.data_ptr(), c.ws_bytes, stream_of(*c.x));
    }
    if (rc) return failed("sx8_gemm_prefill_split", rc);
    return THPVariable_Wrap(std::move(c.y));
    END_HANDLE_TH_ERRORS
}

// dequant(dmin, dmax, config, coeff, hi, lo, basis, scales, out_f, in_f, n_cb): W (out_f, in_f) fp16 on the
// current device, or None unless every field is already there in its stored type.
PyObject* py_dequant(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(11)
    const at::Tensor* t[8];
    for (int i = 0; i < 8; ++i) {
        const at::ScalarType want = i < 2 ? at::kHalf : i < 6 ? at::kByte : at::kFloat;
        t[i] = dense(a[i], want);
        if (!t[i] && i < 2) t[i] = dense(a[i], at::kShort);
        if (!t[i] || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
    }
    if (t[0]->device().index() != c10::hip::current_device()) Py_RETURN_NONE;
    const int64_t out_f = num(a[8]), in_f = num(a[9]), n_cb = num(a[10]);
    SX8_SIZES_OK()
    if (t[6]->numel() != n_cb * 64 || t[7]->numel() != n_cb * 2) Py_RETURN_NONE;
    at::Tensor w;
    int32_t rc;
    {
        Unlocked u;
        w = empty_like_device({out_f, in_f}, at::kHalf, *t[0]);
        rc = lib.dequant(t[0]->data_ptr(), t[1]->data_ptr(), t[2]->data_ptr(), t[3]->data_ptr(), t[4]->data_ptr(),
                         t[5]->data_ptr(), t[6]->data_ptr(), t[7]->data_ptr(), out_f, in_f, n_cb, w.data_ptr(),
                         stream_of(w));
    }
    if (rc) return failed("sx8_dequant_f16", rc);
    return THPVariable_Wrap(std::move(w));
    END_HANDLE_TH_ERRORS
}

// embed(ids, hdr, levels, basis, scales, K, N, n_cb, out): rows of ids into out's first rows, returned as
// a view (*ids.shape, K); or None.
PyObject* py_embed(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(9)
    const at::Tensor* ids = dense(a[0], at::kLong);
    const at::Tensor* out = dense(a[8], at::kHalf);
    const at::Tensor* h = plain(a[1]);
    const at::Tensor* l = plain(a[2]);
    const at::Tensor* b = dense(a[3], at::kFloat);
    const at::Tensor* s = dense(a[4], at::kFloat);
    const int64_t K = num(a[5]), N = num(a[6]), n_cb = num(a[7]);
    SX8_SIZES_OK()
    if (!ids || !out || !h || !l || !b || !s || out->dim() != 2 || out->size(1) != K || ids->device() != out->device() ||
        ids->numel() < 1 || out->size(0) < ids->numel())
        Py_RETURN_NONE;
    const int64_t T = ids->numel();
    c10::SmallVector<int64_t, 5> shape(ids->sizes().begin(), ids->sizes().end());
    shape.push_back(K);
    at::Tensor rows;
    int32_t rc;
    {
        Unlocked u;
        rc = lib.embed(ids->data_ptr(), T, h->data_ptr(), l->data_ptr(), h->dim() == 2 ? (int32_t)h->size(1) : 6,
                       b->data_ptr(), s->data_ptr(), K, N, n_cb, out->data_ptr(), stream_of(*out));
        if (!rc) rows = out->narrow(0, 0, T).view(shape);
    }
    if (rc) return failed("sx8_embed_gather", rc);
    return THPVariable_Wrap(std::move(rows));
    END_HANDLE_TH_ERRORS
}

struct Event {
    hipEvent_t e = nullptr;
    ~Event() {
        if (e) (void)hipEventDestroy(e);
    }
};

void hip_ok(hipError_t e) { TORCH_CHECK(e == hipSuccess, "copy to the host: ", hipGetErrorString(e)); }

// to_host(x): a host copy of a dense device tensor of bytes; to_host(x, ((offset, bytes), ...)): host
// copies of those parts, each in memory of its own (a part kept alive keeps no other).  Through two
// pinned pieces of 1 MB (torch's caching host allocator): the GPU fills one while the host empties the
// other.  10 MB take 0.39 ms, 3 MB 0.14; the runtime's own copy to pageable memory 0.55 and 0.17 (up to
// 0.9).  Pieces of 2 and 4 MB measured no faster: the link takes 20 us a MB, one host thread about 39 to
// empty a piece.
PyObject* py_to_host(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    constexpr int64_t kPiece = 1 << 20;
    if (na != 2) SX8_ARGS(1)
    const at::Tensor* x = dense(a[0], at::kByte);
    if (!x || x->numel() < 1 || (na == 1 && x->numel() <= kPiece)) Py_RETURN_NONE;
    const int64_t n = x->numel(), pieces = (n + kPiece - 1) / kPiece;
    struct Part {
        int64_t off, n;
        at::Tensor y;
    };
    c10::SmallVector<Part, 8> parts;
    if (na == 1) {
        parts.push_back(Part{0, n, at::Tensor()});
    } else {
        if (!PyTuple_Check(a[1])) Py_RETURN_NONE;
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[1]); ++i) {
            PyObject* p = PyTuple_GET_ITEM(a[1], i);
            if (!PyTuple_Check(p) || PyTuple_GET_SIZE(p) != 2) Py_RETURN_NONE;
            const int64_t off = num(PyTuple_GET_ITEM(p, 0)), len = num(PyTuple_GET_ITEM(p, 1));
            SX8_SIZES_OK()
            if (off < 0 || len < 0 || off > n || len > n - off) {
                PyErr_SetString(PyExc_ValueError, "to_host: a part outside the tensor");
                return nullptr;
            }
            parts.push_back(Part{off, len, at::Tensor()});
        }
    }
    {
        Unlocked u;
        c10::DeviceGuard on(x->device());
        for (Part& p : parts) p.y = at::empty({p.n}, at::TensorOptions().dtype(at::kByte));
        const at::Tensor pin = at::empty({std::min(n, 2 * kPiece)}, at::TensorOptions().dtype(at::kByte).pinned_memory(true));
        const hipStream_t st = c10::hip::getCurrentHIPStream(x->device().index()).stream();
        Event ev[2];                      // (one piece: a copy that waits, 10-15 us less than event or stream waits)
        if (pieces > 1)
            for (Event& v : ev) hip_ok(hipEventCreateWithFlags(&v.e, hipEventDisableTiming));
        uint8_t* const stage = static_cast<uint8_t*>(pin.data_ptr());
        auto send = [&](int64_t k) {
            const int64_t off = k * kPiece;
            const auto copy = pieces > 1 ? hipMemcpyAsync : hipMemcpyWithStream;
            hip_ok(copy(stage + (k & 1) * kPiece, static_cast<const uint8_t*>(x->data_ptr()) + off,
                        std::min(kPiece, n - off), hipMemcpyDeviceToHost, st));
            if (pieces > 1) hip_ok(hipEventRecord(ev[k & 1].e, st));
        };
        send(0);
        for (int64_t k = 0; k < pieces; ++k) {
            if (k + 1 < pieces) send(k + 1);
            if (pieces > 1) hip_ok(hipEventSynchronize(ev[k & 1].e));
            const int64_t lo = k * kPiece, hi = std::min(lo + kPiece, n);
            const uint8_t* src = stage + (k & 1) * kPiece;
            for (Part& p : parts) {
                const int64_t from = std::max(lo, p.off), to = std::min(hi, p.off + p.n);
                if (from < to) std::memcpy(static_cast<uint8_t*>(p.y.data_ptr()) + (from - p.off), src + (from - lo), to - from);
            }
        }
    }
    if (na == 1) return THPVariable_Wrap(std::move(parts[0].y));
    PyObject* list = PyList_New((Py_ssize_t)parts.size());
    for (size_t i = 0; list && i < parts.size(); ++i) PyList_SET_ITEM(list, (Py_ssize_t)i, THPVariable_Wrap(std::move(parts[i].y)));
    return list;
    END_HANDLE_TH_ERRORS
}

// ---- packed sequences and the paged cache (sx8_paged_kv.py) ------------------------------------
// A (rows, heads, hd) tensor of fp16 or bf16 (wide: or float32) that the kernels read in place (sx8_paged_kv._in_place), else
// null.
const at::Tensor* head_rows(PyObject* o, int64_t min_ts, bool wide = false) {
    const at::Tensor* x = plain(o);
    if (!x || !x->is_cuda() || x->layout() != at::kStrided || x->dim() != 3 || x->size(0) < 1 ||
        (x->scalar_type() != at::kHalf && x->scalar_type() != at::kBFloat16 && !(wide && x->scalar_type() == at::kFloat)))
        return nullptr;
    const int64_t ts = x->stride(0), hs = x->stride(1);
    const bool ok = x->stride(2) == 1 && ts % 8 == 0 && hs % 8 == 0 && hs >= 0 && ts >= min_ts && ts <= 1 << 23 &&
                    reinterpret_cast<uintptr_t>(x->data_ptr()) % 16 == 0;
    return ok ? x : nullptr;
}

// A contiguous int32 vector of n values (any number: n < 0) on the device of `like`, else null.
const at::Tensor* int_vector(PyObject* o, int64_t n, const at::Tensor& like) {
    const at::Tensor* x = dense(o, at::kInt);
    return x && x->dim() == 1 && x->numel() > 0 && (n < 0 || x->numel() == n) && x->device() == like.device() ? x : nullptr;
}

int32_t dtype_of(const at::Tensor& x) { return x.scalar_type() == at::kBFloat16; }

// varlen(q, k, v, cu_q, cu_k or None, scale, causal): attn_varlen into a new tensor.
PyObject* py_varlen(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(7)
    const at::Tensor* q = head_rows(a[0], 0);
    if (!q) Py_RETURN_NONE;
    const int64_t hd = q->size(2);
    const at::Tensor* k = head_rows(a[1], hd);
    const at::Tensor* v = head_rows(a[2], hd);
    const at::Tensor* cq = int_vector(a[3], -1, *q);
    const at::Tensor* ck = a[4] == Py_None ? cq : int_vector(a[4], cq ? cq->numel() : 0, *q);
    if (!k || !v || !cq || !ck || k->sizes() != v->sizes() || k->size(2) != hd || k->scalar_type() != q->scalar_type() ||
        v->scalar_type() != q->scalar_type() || k->device() != q->device() || v->device() != q->device() ||
        !PyFloat_Check(a[5]) || !PyBool_Check(a[6]))
        Py_RETURN_NONE;
    const float scale = (float)PyFloat_AS_DOUBLE(a[5]);
    int32_t rc;
    at::Tensor o;
    {
        Unlocked u;
        c10::DeviceGuard on(q->device());
        o = empty_like_device(q->sizes(), q->scalar_type(), *q);
        const int64_t nb = lib.varlen_ws(cq->numel() - 1, q->size(0), k->size(0), (int32_t)q->size(1), (int32_t)hd);
        at::Tensor ws;
        if (nb > 0) ws = empty_like_device({nb}, at::kByte, *q);
        rc = lib.varlen(q->data_ptr(), k->data_ptr(), v->data_ptr(), o.data_ptr(), cq->data_ptr<int32_t>(),
                        ck->data_ptr<int32_t>(), cq->numel() - 1, q->size(0), k->size(0), (int32_t)q->size(1),
                        (int32_t)k->size(1), (int32_t)hd, q->stride(0), q->stride(1), k->stride(0), k->stride(1), v->stride(0),
                        v->stride(1), o.stride(0), o.stride(1), scale, a[6] == Py_True, dtype_of(*q),
                        nb > 0 ? ws.data_ptr() : nullptr, nb > 0 ? nb : 0, stream_of(*q));
    }
    if (rc) return failed("sx8_attn_varlen", rc);
    return THPVariable_Wrap(std::move(o));
    END_HANDLE_TH_ERRORS
}

// What PagedKV4 keeps for these calls: (pages, table, lens, refs, status, page_bytes, n_kv, head_dim, page_tokens,
// bytes of attend's workspace, of the page operations', of attend_tree's, marks); the wrapper checked it.
struct Cache {
    const at::Tensor *pages, *table, *lens, *refs, *status, *marks;
    int64_t layers, n_pages, slots, width, page_bytes, ws_attend, ws_pages, ws_tree;
    int32_t nk, hd, pt;
    void* stream;
    int32_t* ints(const at::Tensor* t) const { return t->data_ptr<int32_t>(); }
    uint8_t* layer(int64_t i) const { return pages->data_ptr<uint8_t>() + i * n_pages * page_bytes; }
};
bool cache(PyObject* o, Cache* c) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 13) return false;
    const at::Tensor** t[6] = {&c->pages, &c->table, &c->lens, &c->refs, &c->status, &c->marks};
    for (int i = 0; i < 6; ++i)
        if (!(*t[i] = plain(PyTuple_GET_ITEM(o, i < 5 ? i : 12)))) return false;
    int64_t n[7];
    for (int i = 0; i < 7; ++i) n[i] = num(PyTuple_GET_ITEM(o, 5 + i));
    c->page_bytes = n[0];
    c->nk = (int32_t)n[1];
    c->hd = (int32_t)n[2];
    c->pt = (int32_t)n[3];
    c->ws_attend = n[4];
    c->ws_pages = n[5];
    c->ws_tree = n[6];
    c->layers = c->pages->size(0);
    c->n_pages = c->pages->size(1);
    c->slots = c->table->size(0);
    c->width = c->table->size(1);
    c->stream = stream_of(*c->pages);
    return true;
}
// cu (None or a vector of slots + 1) and layer of a call with rows
bool cache_call(PyObject* desc, PyObject* layer, PyObject* cu, Cache* c, int64_t* li, const int32_t** cup) {
    if (!cache(desc, c)) return false;
    *li = num(layer);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    if (*li < 0 || *li >= c->layers) return false;
    *cup = nullptr;
    if (cu == Py_None) return true;
    const at::Tensor* t = int_vector(cu, c->slots + 1, *c->pages);
    if (!t) return false;
    *cup = t->data_ptr<int32_t>();
    return true;
}

// kv4_append(cache, layer, k, v, cu or None) -> True
PyObject* py_kv4_append(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(5)
    Cache c;
    int64_t layer;
    const int32_t* cu;
    const at::Tensor* k = head_rows(a[2], 0);
    const at::Tensor* v = head_rows(a[3], 0);
    if (!k || !v || !cache_call(a[0], a[1], a[4], &c, &layer, &cu) || k->sizes() != v->sizes() || k->size(1) != c.nk ||
        k->size(2) != c.hd || k->scalar_type() != v->scalar_type() || k->device() != c.pages->device() ||
        v->device() != c.pages->device())
        Py_RETURN_NONE;
    int32_t rc;
    {
        Unlocked u;
        c10::DeviceGuard on(c.pages->device());
        rc = lib.kv4_append(c.layer(layer), c.ints(c.table), c.ints(c.lens), cu, c.slots, c.width, c.n_pages, k->data_ptr(),
                            v->data_ptr(), k->size(0), k->stride(0), k->stride(1), v->stride(0), v->stride(1), c.nk, c.hd, c.pt,
                            dtype_of(*k), c.stream);
    }
    if (rc) return failed("sx8_kv4_append", rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// kv4_read(cache, layer, rows, cu or None, bf16) -> (k, v)
PyObject* py_kv4_read(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(5)
    Cache c;
    int64_t layer;
    const int32_t* cu;
    const int64_t rows = num(a[2]);
    SX8_SIZES_OK()
    if (rows < 1 || !cache_call(a[0], a[1], a[3], &c, &layer, &cu)) Py_RETURN_NONE;
    const bool bf = a[4] == Py_True;
    int32_t rc;
    at::Tensor k, v;
    {
        Unlocked u;
        c10::DeviceGuard on(c.pages->device());
        k = empty_like_device({rows, c.nk, c.hd}, bf ? at::kBFloat16 : at::kHalf, *c.pages);
        v = empty_like_device({rows, c.nk, c.hd}, bf ? at::kBFloat16 : at::kHalf, *c.pages);
        rc = lib.kv4_read(c.layer(layer), c.ints(c.table), c.ints(c.lens), cu, c.slots, c.width, c.n_pages, k.data_ptr(),
                          v.data_ptr(), rows, k.stride(0), k.stride(1), v.stride(0), v.stride(1), c.nk, c.hd, c.pt, bf, c.stream);
    }
    if (rc) return failed("sx8_kv4_read", rc);
    PyObject* pk = THPVariable_Wrap(std::move(k));
    PyObject* pv = THPVariable_Wrap(std::move(v));
    PyObject* both = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
    Py_XDECREF(pk);
    Py_XDECREF(pv);
    return both;
    END_HANDLE_TH_ERRORS
}

// kv4_attend(cache, layer, q, cu or None, scale) -> out
PyObject* py_kv4_attend(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(5)
    Cache c;
    int64_t layer;
    const int32_t* cu;
    const at::Tensor* q = head_rows(a[2], 0);
    if (!q || !PyFloat_Check(a[4]) || !cache_call(a[0], a[1], a[3], &c, &layer, &cu) || q->size(2) != c.hd ||
        q->device() != c.pages->device())
        Py_RETURN_NONE;
    const float scale = (float)PyFloat_AS_DOUBLE(a[4]);
    int32_t rc;
    at::Tensor o;
    {
        Unlocked u;
        c10::DeviceGuard on(c.pages->device());
        o = empty_like_device(q->sizes(), q->scalar_type(), *q);
        const at::Tensor ws = empty_like_device({c.ws_attend}, at::kByte, *q);
        rc = lib.kv4_attend(c.layer(layer), c.ints(c.table), c.ints(c.lens), cu, c.slots, c.width, c.n_pages, q->data_ptr(),
                            o.data_ptr(), q->size(0), q->stride(0), q->stride(1), o.stride(0), o.stride(1), (int32_t)q->size(1),
                            c.nk, c.hd, c.pt, scale, dtype_of(*q), ws.data_ptr(), c.ws_attend, c.stream);
    }
    if (rc) return failed("sx8_kv4_attend", rc);
    return THPVariable_Wrap(std::move(o));
    END_HANDLE_TH_ERRORS
}

// kv4_pages(cache, "reserve", add) / ("fork", src, dst) / ("free", slots) / ("compact") -> True
PyObject* py_kv4_pages(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    Cache c;
    if (na < 2 || na > 4 || !PyUnicode_Check(a[1]) || !cache(a[0], &c)) Py_RETURN_NONE;
    const char* what = PyUnicode_AsUTF8(a[1]);
    if (!what) return nullptr;
    const at::Tensor* x = na > 2 ? int_vector(a[2], what[0] == 'r' ? c.slots : -1, *c.pages) : nullptr;
    const at::Tensor* y = na > 3 && x ? int_vector(a[3], x->numel(), *c.pages) : nullptr;
    if ((na > 2 && !x) || (na > 3 && !y)) Py_RETURN_NONE;
    int32_t rc;
    {
        Unlocked u;
        c10::DeviceGuard on(c.pages->device());
        at::Tensor ws;
        if (std::strcmp(what, "free") != 0) ws = empty_like_device({c.ws_pages}, at::kByte, *c.pages);
        void* const w = ws.defined() ? ws.data_ptr() : nullptr;
        int32_t *const table = c.ints(c.table), *const lens = c.ints(c.lens), *const refs = c.ints(c.refs),
                       *const status = c.ints(c.status);
        if (!std::strcmp(what, "reserve") && na == 3)
            rc = lib.kv4_reserve(table, lens, refs, c.ints(x), c.slots, c.width, c.n_pages, c.pt, status, c.ints(c.marks), w,
                                 c.ws_pages, c.stream);
        else if (!std::strcmp(what, "fork") && na == 4)
            rc = lib.kv4_fork(c.layer(0), c.layers, c.page_bytes, table, lens, refs, c.ints(x), c.ints(y), x->numel(), c.slots,
                              c.width, c.n_pages, c.pt, status, w, c.ws_pages, c.stream);
        else if (!std::strcmp(what, "free") && na == 3)
            rc = lib.kv4_free(table, lens, refs, c.ints(x), x->numel(), c.slots, c.width, c.n_pages, status, c.stream);
        else if (!std::strcmp(what, "compact") && na == 2)
            rc = lib.kv4_compact(c.layer(0), c.layers, c.page_bytes, table, refs, c.slots, c.width, c.n_pages, w, c.ws_pages,
                                 c.stream);
        else
            rc = -1;
    }
    if (rc == -1) Py_RETURN_NONE;
    if (rc) return failed(("sx8_kv4_" + std::string(what)).c_str(), rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// None, or a dense vector of n values of type t on the device of `like`; ok false: something else.
const at::Tensor* vector_or_none(PyObject* o, at::ScalarType t, int64_t n, const at::Tensor& like, bool* ok) {
    if (o == Py_None) return nullptr;
    const at::Tensor* x = dense(o, t);
    if (x && x->dim() == 1 && x->numel() == n && x->device() == like.device()) return x;
    *ok = false;
    return nullptr;
}
bool aligned16(const at::Tensor* x) { return !x || reinterpret_cast<uintptr_t>(x->data_ptr()) % 16 == 0; }
PyObject* tuple_of(std::initializer_list<at::Tensor*> ts) {
    PyObject* t = PyTuple_New((Py_ssize_t)ts.size());
    Py_ssize_t i = 0;
    for (at::Tensor* x : ts) {
        PyObject* o = t ? THPVariable_Wrap(std::move(*x)) : nullptr;
        if (!o) {
            Py_XDECREF(t);
            return nullptr;
        }
        PyTuple_SET_ITEM(t, i++, o);
    }
    return t;
}

// kv4_append_rope(cache, layer, q, k, v, cos, sin, cu, depth, q_norm, k_norm, eps, interleaved, bf16) -> the query rows; cu,
// depth and the norms may be None
PyObject* py_kv4_append_rope(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(14)
    Cache c;
    int64_t layer;
    const int32_t* cu;
    const at::Tensor* q = head_rows(a[2], 0, true);
    const at::Tensor* k = head_rows(a[3], 0, true);
    const at::Tensor* v = head_rows(a[4], 0, true);
    const at::Tensor* cs = dense(a[5], at::kFloat);
    const at::Tensor* sn = dense(a[6], at::kFloat);
    if (!q || !k || !v || !cs || !sn || !cache_call(a[0], a[1], a[7], &c, &layer, &cu) || !PyFloat_Check(a[11]) ||
        !PyBool_Check(a[12]) || !PyBool_Check(a[13]))
        Py_RETURN_NONE;
    const at::Device on = c.pages->device();
    const bool bf = a[13] == Py_True, wide = q->scalar_type() == at::kFloat;
    const at::ScalarType to = bf ? at::kBFloat16 : at::kHalf;
    bool fits = true;
    const at::Tensor* depth = vector_or_none(a[8], at::kInt, q->size(0), *c.pages, &fits);
    const at::Tensor* qw = vector_or_none(a[9], to, c.hd, *c.pages, &fits);
    const at::Tensor* kw = vector_or_none(a[10], to, c.hd, *c.pages, &fits);
    if (!fits || !aligned16(qw) || !aligned16(kw) || !aligned16(cs) || !aligned16(sn) || q->size(2) != c.hd ||
        k->sizes() != v->sizes() || k->size(0) != q->size(0) || k->size(1) != c.nk || k->size(2) != c.hd ||
        k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || (!wide && q->scalar_type() != to) ||
        cs->dim() != 2 || cs->sizes() != sn->sizes() || q->device() != on || k->device() != on || v->device() != on ||
        cs->device() != on || sn->device() != on)
        Py_RETURN_NONE;
    const double eps = PyFloat_AS_DOUBLE(a[11]);
    int32_t rc;
    at::Tensor o;
    {
        Unlocked u;
        c10::DeviceGuard guard(on);
        o = empty_like_device(q->sizes(), to, *q);
        rc = lib.kv4_append_rope(c.layer(layer), c.ints(c.table), c.ints(c.lens), cu, c.slots, c.width, c.n_pages, q->data_ptr(),
                                 k->data_ptr(), v->data_ptr(), o.data_ptr(), q->size(0), q->stride(0), q->stride(1), k->stride(0),
                                 k->stride(1), v->stride(0), v->stride(1), o.stride(0), o.stride(1), (int32_t)q->size(1), c.nk,
                                 c.hd, c.pt, cs->data_ptr<float>(), sn->data_ptr<float>(), cs->size(0),
                                 (int32_t)(2 * cs->size(1)), a[12] == Py_True, depth ? depth->data_ptr<int32_t>() : nullptr, c.ints(c.marks),
                                 qw ? qw->data_ptr() : nullptr, kw ? kw->data_ptr() : nullptr, eps, wide ? 2 : bf, bf, c.stream);
    }
    if (rc) return failed("sx8_kv4_append_rope", rc);
    return THPVariable_Wrap(std::move(o));
    END_HANDLE_TH_ERRORS
}

// kv4_attend_tree(cache, layer, q, mask, cu or None, scale) -> out
PyObject* py_kv4_attend_tree(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(6)
    Cache c;
    int64_t layer;
    const int32_t* cu;
    const at::Tensor* q = head_rows(a[2], 0);
    const at::Tensor* m = dense(a[3], at::kLong);
    if (!q || !m || !PyFloat_Check(a[5]) || !cache_call(a[0], a[1], a[4], &c, &layer, &cu) || q->size(2) != c.hd ||
        m->dim() != 2 || m->size(0) != q->size(0) || m->size(1) < 1 || m->size(1) > 4 || q->device() != c.pages->device() ||
        m->device() != c.pages->device())
        Py_RETURN_NONE;
    const float scale = (float)PyFloat_AS_DOUBLE(a[5]);
    int32_t rc;
    at::Tensor o;
    {
        Unlocked u;
        c10::DeviceGuard on(c.pages->device());
        o = empty_like_device(q->sizes(), q->scalar_type(), *q);
        const at::Tensor ws = empty_like_device({c.ws_tree}, at::kByte, *q);
        rc = lib.kv4_attend_tree(c.layer(layer), c.ints(c.table), c.ints(c.lens), cu, c.slots, c.width, c.n_pages, q->data_ptr(),
                                 o.data_ptr(), q->size(0), q->stride(0), q->stride(1), o.stride(0), o.stride(1),
                                 reinterpret_cast<const uint64_t*>(m->data_ptr()), (int32_t)m->size(1), (int32_t)q->size(1), c.nk,
                                 c.hd, c.pt, scale, dtype_of(*q), ws.data_ptr(), c.ws_tree, c.stream);
    }
    if (rc) return failed("sx8_kv4_attend_tree", rc);
    return THPVariable_Wrap(std::move(o));
    END_HANDLE_TH_ERRORS
}

// kv4_keep(cache, path, counts, cu or None) -> True
PyObject* py_kv4_keep(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(4)
    Cache c;
    if (!cache(a[0], &c)) Py_RETURN_NONE;
    const at::Tensor* path = int_vector(a[1], -1, *c.pages);
    const at::Tensor* counts = int_vector(a[2], c.slots, *c.pages);
    const at::Tensor* cu = a[3] == Py_None ? nullptr : int_vector(a[3], c.slots + 1, *c.pages);
    if (!path || !counts || (a[3] != Py_None && !cu)) Py_RETURN_NONE;
    int32_t rc;
    {
        Unlocked u;
        c10::DeviceGuard on(c.pages->device());
        const int64_t nb = lib.kv4_keep_ws(c.slots, path->numel());
        const at::Tensor ws = empty_like_device({nb > 0 ? nb : 0}, at::kByte, *c.pages);
        rc = lib.kv4_keep(c.layer(0), c.layers, c.ints(c.table), c.ints(c.lens), c.ints(c.refs), cu ? c.ints(cu) : nullptr,
                          c.ints(path), c.ints(counts), path->numel(), c.slots, c.width, c.n_pages, c.nk, c.hd, c.pt,
                          c.ints(c.status), c.ints(c.marks), ws.data_ptr(), nb, c.stream);
    }
    if (rc) return failed("sx8_kv4_keep", rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// ---- drafted tokens (sx8_draft.py) -------------------------------------------------------------
// draft_tree(parents, cu, words) -> (mask, depth)
PyObject* py_draft_tree(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(3)
    const at::Tensor* p = dense(a[0], at::kInt);
    const int64_t words = num(a[2]);
    SX8_SIZES_OK()
    if (!p || p->dim() != 1 || p->numel() < 1 || words < 1 || words > 4) Py_RETURN_NONE;
    const at::Tensor* cu = int_vector(a[1], -1, *p);
    if (!cu) Py_RETURN_NONE;
    int32_t rc;
    at::Tensor mask, depth;
    {
        Unlocked u;
        c10::DeviceGuard on(p->device());
        mask = empty_like_device({p->numel(), words}, at::kLong, *p);
        depth = empty_like_device({p->numel()}, at::kInt, *p);
        rc = lib.draft_tree(p->data_ptr<int32_t>(), cu->data_ptr<int32_t>(), cu->numel() - 1, p->numel(), (int32_t)words,
                            reinterpret_cast<uint64_t*>(mask.data_ptr()), depth.data_ptr<int32_t>(), stream_of(*p));
    }
    if (rc) return failed("sx8_draft_tree", rc);
    return tuple_of({&mask, &depth});
    END_HANDLE_TH_ERRORS
}

// (rows, vocabulary) values of a type that sx8_draft_verify takes, rows one after another or apart; null: something else
const at::Tensor* matrix(PyObject* o, int32_t* type) {
    const at::Tensor* x = plain(o);
    if (!x || !x->is_cuda() || x->layout() != at::kStrided || x->dim() != 2 || x->size(0) < 1 || x->size(1) < 1 || x->stride(1) != 1 ||
        x->stride(0) < x->size(1))
        return nullptr;
    *type = x->scalar_type() == at::kHalf ? 0 : x->scalar_type() == at::kBFloat16 ? 1 : x->scalar_type() == at::kFloat ? 2 : -1;
    return *type < 0 ? nullptr : x;
}

// draft_verify(logits, tokens, parents, cu, uniforms or None, temperature (a float or a vector), probs or None, depth or None)
//   -> (path, counts, next)
PyObject* py_draft_verify(PyObject*, PyObject* const* a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    SX8_ARGS(8)
    int32_t type = 0, ptype = 0;
    const at::Tensor* x = matrix(a[0], &type);
    if (!x) Py_RETURN_NONE;
    const int64_t rows = x->size(0), V = x->size(1);
    const at::Tensor* tok = dense(a[1], at::kLong);
    const at::Tensor* par = int_vector(a[2], rows, *x);
    const at::Tensor* cu = int_vector(a[3], -1, *x);
    if (!tok || tok->dim() != 1 || tok->numel() != rows || tok->device() != x->device() || !par || !cu || cu->numel() < 2)
        Py_RETURN_NONE;
    const int64_t slots = cu->numel() - 1;
    bool fits = true;
    const at::Tensor* un = vector_or_none(a[4], at::kFloat, rows, *x, &fits);
    const at::Tensor* depth = vector_or_none(a[7], at::kInt, rows, *x, &fits);
    const at::Tensor* temp = nullptr;
    float t = 0.f;
    if (PyFloat_Check(a[5])) t = (float)PyFloat_AS_DOUBLE(a[5]);
    else temp = vector_or_none(a[5], at::kFloat, slots, *x, &fits);
    const at::Tensor* pr = a[6] == Py_None ? nullptr : matrix(a[6], &ptype);
    if (!fits || (!temp && !PyFloat_Check(a[5])) || (a[6] != Py_None && (!pr || pr->sizes() != x->sizes() || pr->device() != x->device())))
        Py_RETURN_NONE;
    int32_t rc;
    at::Tensor path, counts, next;
    {
        Unlocked u;
        c10::DeviceGuard on(x->device());
        path = empty_like_device({rows}, at::kInt, *x);
        counts = empty_like_device({slots}, at::kInt, *x);
        next = empty_like_device({slots}, at::kLong, *x);
        const int64_t nb = lib.draft_verify_ws(slots, rows, V);
        const at::Tensor ws = empty_like_device({nb > 0 ? nb : 0}, at::kByte, *x);
        rc = lib.draft_verify(x->data_ptr(), x->stride(0), type, tok->data_ptr<int64_t>(), par->data_ptr<int32_t>(),
                              depth ? depth->data_ptr<int32_t>() : nullptr, cu->data_ptr<int32_t>(), slots, rows, V, un ? un->data_ptr<float>() : nullptr,
                              temp ? temp->data_ptr<float>() : nullptr, t, pr ? pr->data_ptr() : nullptr, pr ? pr->stride(0) : 0,
                              ptype, path.data_ptr<int32_t>(), counts.data_ptr<int32_t>(), next.data_ptr<int64_t>(), ws.data_ptr(),
                              nb, stream_of(*x));
    }
    if (rc) return failed("sx8_draft_verify", rc);
    return tuple_of({&path, &counts, &next});
    END_HANDLE_TH_ERRORS
}

#define SX8_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {{"bind", py_bind, METH_O, nullptr},
                         {"linear", SX8_FAST(py_linear), nullptr},
                         {"gemv", SX8_FAST(py_gemv), nullptr},
                         {"gemm", SX8_FAST(py_gemm), nullptr},
                         {"gemm_split", SX8_FAST(py_gemm_split), nullptr},
                         {"dequant", SX8_FAST(py_dequant), nullptr},
                         {"embed", SX8_FAST(py_embed), nullptr},
                         {"to_host", SX8_FAST(py_to_host), nullptr},
                         {"varlen", SX8_FAST(py_varlen), nullptr},
                         {"kv4_append", SX8_FAST(py_kv4_append), nullptr},
                         {"kv4_read", SX8_FAST(py_kv4_read), nullptr},
                         {"kv4_attend", SX8_FAST(py_kv4_attend), nullptr},
                         {"kv4_pages", SX8_FAST(py_kv4_pages), nullptr},
                         {"kv4_append_rope", SX8_FAST(py_kv4_append_rope), nullptr},
                         {"kv4_attend_tree", SX8_FAST(py_kv4_attend_tree), nullptr},
                         {"kv4_keep", SX8_FAST(py_kv4_keep), nullptr},
                         {"draft_tree", SX8_FAST(py_draft_tree), nullptr},
                         {"draft_verify", SX8_FAST(py_draft_verify), nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_sx8py", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__sx8py() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", SX8_TORCH) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
