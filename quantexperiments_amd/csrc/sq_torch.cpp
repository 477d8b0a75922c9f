// The native call path between Python and libsqhip.so: argument checks, workspace lookup, output allocation and the call
// itself, on torch tensors, in one C function per entry point.
//
// A decode-time product takes the GPU 5 to 20 us.  The same steps in Python (a ctypes struct per piece, a device context, the
// stream, the workspace, a ctypes call) took 18 us for one piece and 24 for three, 6 more through a Python custom op, so a
// program without a graph waited for its host on every call; here they take 4 to 6 us, of which the launch is 3.5.
//
// Every function answers 0 (done), a negative SQ_E* code (sq_last_error has the text), or 1: not a call this path covers (an
// unusual dtype or stride, a workspace that has to grow, a stream under capture), and the caller goes on in Python, which
// also words the errors.  Nothing is kept between calls but what a matrix is (its tensors and sizes, dropped by PackedLinear
// whenever one of its attributes is set).
#include <Python.h>
#include <algorithm>
#include <cmath>
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>
#include "../../include/sqhip.h"

namespace {

constexpr int MAX_PIECES = 8;
constexpr int NOT_COVERED = 1;

struct Native {                      // one packed matrix: its tensors and what the library wants to know about them
    PyObject_HEAD
    sq_matrix m;
    at::Tensor* t;                   // words, table, row_scale, row_book, row_mask, perms, row_order, stream
};

PyObject *s_native, *s_make_native, *s_rls, *s_cross, *s_large, *s_dequant_from, *s_enabled, *s_forward, *s_trace, *s_fused;
PyObject *g_bufs;                    // kernels._Workspace.bufs
PyObject *g_registry, *g_core;       // vllm_ext.core._REGISTRY and the module itself (its _trace is looked up per call)
PyTypeObject* g_shards_type;         // vllm_ext.core.PackedShards
PyObject* g_keys[64];                // (str(device), "kernels") per device

void native_dealloc(PyObject* self) {
    delete[] reinterpret_cast<Native*>(self)->t;
    Py_TYPE(self)->tp_free(self);
}

PyTypeObject NativeType = {PyVarObject_HEAD_INIT(nullptr, 0)};

// native(words, table, row_scale, row_book, row_mask, perms, row_order, stream, R, C, d, bits, G, M, W, stream_runs, stream_groups)
PyObject* make_native(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 17) { PyErr_SetString(PyExc_TypeError, "native: 17 arguments"); return nullptr; }
    Native* o = reinterpret_cast<Native*>(NativeType.tp_alloc(&NativeType, 0));
    if (!o) return nullptr;
    o->t = new at::Tensor[8];
    for (int i = 0; i < 8; ++i)
        if (THPVariable_Check(a[i])) o->t[i] = THPVariable_Unpack(a[i]);
    int32_t v[9];
    for (int i = 0; i < 9; ++i) v[i] = (int32_t)PyLong_AsLong(a[8 + i]);
    if (PyErr_Occurred()) { Py_DECREF(o); return nullptr; }
    sq_matrix& m = o->m;
    m.R = v[0]; m.C = v[1]; m.d = v[2]; m.bits = v[3]; m.G = v[4]; m.M = v[5]; m.W = v[6]; m.y_off = 0;
    m.stream_runs = v[7]; m.stream_groups = v[8];
    return reinterpret_cast<PyObject*>(o);
}

// The pieces of a call as the library takes them, and what owns their tensors: the library runs without the GIL, so another
// thread may set an attribute of a piece (which drops its Native) before the kernels are launched.
// 0, NOT_COVERED, or -1 with a Python error set.
struct Pieces { sq_matrix m[MAX_PIECES]; int n = 0, dev = -1; int64_t rows = 0; pybind11::object held[MAX_PIECES]; };
int unpack_pieces(PyObject* seq, Pieces& p) {
    if (!PyList_CheckExact(seq) && !PyTuple_CheckExact(seq)) return NOT_COVERED;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    if (n < 1 || n > MAX_PIECES) return NOT_COVERED;
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* piece = PySequence_Fast_GET_ITEM(seq, i);
        PyObject* o = PyObject_GetAttr(piece, s_native);
        if (!o) { PyErr_Clear(); return NOT_COVERED; }
        if (o == Py_None) {
            Py_DECREF(o);
            o = PyObject_CallMethodObjArgs(piece, s_make_native, nullptr);
            if (!o) return -1;
        }
        p.held[i] = pybind11::reinterpret_steal<pybind11::object>(o);
        if (Py_TYPE(o) != &NativeType) return NOT_COVERED;
        const Native* nat = reinterpret_cast<Native*>(o);
        sq_matrix& m = p.m[i];
        m = nat->m;
        const at::Tensor* t = nat->t;
        auto ptr = [](const at::Tensor& x) { return x.defined() ? x.data_ptr() : nullptr; };
        m.tags = (const int32_t*)ptr(t[0]); m.table = (const uint16_t*)ptr(t[1]); m.row_scale = (const uint16_t*)ptr(t[2]);
        m.row_book = (const uint8_t*)ptr(t[3]); m.row_mask = (const uint8_t*)ptr(t[4]); m.perms = (const int32_t*)ptr(t[5]);
        m.row_order = (const int32_t*)ptr(t[6]); m.stream = ptr(t[7]);
        m.y_off = (int32_t)p.rows;
        p.rows += m.R;
        const int dev = t[1].is_cuda() ? t[1].get_device() : -1;
        if (dev < 0 || dev >= 64 || (i > 0 && dev != p.dev) || m.C != p.m[0].C) return NOT_COVERED;
        p.dev = dev;
    }
    p.n = (int)n;
    return 0;
}

int dtype_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return SQ_F32;
        case at::kHalf: return SQ_F16;
        case at::kBFloat16: return SQ_BF16;
        default: return -1;
    }
}
bool is16(int dt) { return dt == SQ_F16 || dt == SQ_BF16; }

// a [rows, cols] matrix on device `dev` with unit column stride; a subclass or a tensor that needs Python dispatch is left alone
bool matrix_on(const at::Tensor& t, int dev) {
    return t.dim() == 2 && t.is_cuda() && t.get_device() == dev && t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() &&
           (t.stride(1) == 1 || t.size(1) == 1);
}
int64_t row_ld(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)); }
bool vec16(const at::Tensor& t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }

// The device as it was, and the current stream of `dev`.
struct OnDevice {
    int prev = -1;
    hipStream_t stream;
    explicit OnDevice(int dev) {
        const int cur = c10::hip::current_device();
        if (cur != dev) { prev = cur; c10::hip::set_device((c10::DeviceIndex)dev); }
        stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream();
    }
    ~OnDevice() { if (prev >= 0) c10::hip::set_device((c10::DeviceIndex)prev); }
};

// The shared workspace of a device (kernels._Workspace), held for as long as the call uses it: the library runs without the
// GIL, and a call of another thread may meanwhile replace the buffer by a larger one.  (Its kernels are enqueued when the call
// returns; what is freed after that is given out again behind them on this stream.)
struct Workspace { at::Tensor held; void* p = nullptr; size_t bytes = 0; };
// It if it holds `need` bytes and the stream is not being captured (who was captured with which buffer is recorded in Python).
bool workspace(int dev, size_t need, hipStream_t s, Workspace& ws) {
    if (need == 0) return true;
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &st) != hipSuccess || st != hipStreamCaptureStatusNone) { (void)hipGetLastError(); return false; }
    if (!g_keys[dev]) g_keys[dev] = Py_BuildValue("(Ns)", PyUnicode_FromFormat("cuda:%d", dev), "kernels");
    PyObject* b = g_bufs && g_keys[dev] ? PyDict_GetItem(g_bufs, g_keys[dev]) : nullptr;
    if (!b || !THPVariable_Check(b)) return false;
    const at::Tensor& t = THPVariable_Unpack(b);
    if ((size_t)t.numel() < need) return false;
    ws.held = t;
    ws.p = t.data_ptr();
    ws.bytes = (size_t)t.numel();
    return true;
}

// The workspace of a product: the shared one; a buffer of the call's own where the pieces could run without any (their partial sums
// only make them faster), so that streams may run them side by side.
bool product_workspace(const Pieces& p, int rows, int which, const at::Tensor& like, hipStream_t s, Workspace& ws) {
    const size_t need = sq_workspace_bytes(p.m, p.n, rows, which);
    if (need == 0 || rows > SQ_SMALL_BMAX || sq_workspace_bytes(p.m, p.n, rows, which | 4) != 0) return workspace(p.dev, need, s, ws);
    ws.bytes = sq_workspace_bytes(p.m, p.n, rows, which | 2);
    ws.held = at::empty({(int64_t)ws.bytes}, like.options().dtype(at::kByte));
    ws.p = ws.held.data_ptr();
    return true;
}

int linear_into(const Pieces& p, const at::Tensor& x, const at::Tensor& y, bool gemm) {
    const int xd = dtype_of(x), yd = dtype_of(y);
    if (!is16(xd) || yd < 0 || !matrix_on(x, p.dev) || !matrix_on(y, p.dev) || x.size(0) != y.size(0) || y.size(1) != p.rows || x.size(1) != p.m[0].C ||
        x.size(0) < 1)
        return NOT_COVERED;
    const int B = (int)x.size(0);
    OnDevice on(p.dev);
    Workspace ws;
    if (!product_workspace(p, B, gemm, x, on.stream, ws)) return NOT_COVERED;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = (gemm ? sq_linear_gemm : sq_linear_small)(p.m, p.n, x.data_ptr(), xd, row_ld(x), y.data_ptr(), yd, row_ld(y), B, ws.p, ws.bytes, on.stream);
    Py_END_ALLOW_THREADS
    return rc;
}

PyObject* answer(int rc) { return rc == -1 && PyErr_Occurred() ? nullptr : PyLong_FromLong(rc); }
bool tensors(PyObject* const* a, int n) {
    for (int i = 0; i < n; ++i) if (!THPVariable_Check(a[i])) return false;
    return true;
}

// (torch's own translation: an allocation that fails is a torch.OutOfMemoryError here too)
#define SQ_GUARD(...) try { __VA_ARGS__ } catch (...) { if (!PyErr_Occurred()) torch::translate_exception_to_python(std::current_exception()); return nullptr; }

// linear(pieces, x, y, gemm)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 4 || !tensors(a + 1, 2)) return answer(NOT_COVERED);
    SQ_GUARD(
        Pieces p;
        if (int rc = unpack_pieces(a[0], p)) return answer(rc);
        return answer(linear_into(p, THPVariable_Unpack(a[1]), THPVariable_Unpack(a[2]), a[3] == Py_True));
    )
}

// The forward of a PackedShards: a tensor, an undefined tensor (not covered), or a Python error.
bool shards_forward(PyObject* ps, const at::Tensor& x, at::Tensor& out, int* rc) {
    *rc = NOT_COVERED;
    if (x.dim() < 1 || !x.is_cuda() || !is16(dtype_of(x)) || !x.is_contiguous() || x.unsafeGetTensorImpl()->is_python_dispatch()) return true;
    auto get = [&](PyObject* name) { return pybind11::reinterpret_steal<pybind11::object>(PyObject_GetAttr(ps, name)); };
    pybind11::object rls = get(s_rls), cross = get(s_cross);
    if (!rls || !cross) return false;
    Pieces p;
    if (int r = unpack_pieces(rls.ptr(), p)) { *rc = r; return r >= 0 || !PyErr_Occurred(); }
    const int64_t C = p.m[0].C;
    if (x.size(-1) != C || x.numel() == 0 || x.get_device() != p.dev || C % 8 || !vec16(x)) return true;
    const int64_t M = x.numel() / C;
    const long cr = PyLong_AsLong(cross.ptr());
    if (cr == -1 && PyErr_Occurred()) { PyErr_Clear(); return true; }
    bool gemm = false;
    if (M > cr) {
        pybind11::object large = get(s_large), from = get(s_dequant_from);
        if (!large || !from) return false;
        if (PyUnicode_Compare(large.ptr(), s_fused) != 0) return true;
        const long f = PyLong_AsLong(from.ptr());
        if ((f == -1 && PyErr_Occurred()) || M >= f || M > INT32_MAX) { PyErr_Clear(); return true; }
        gemm = true;
    }
    const at::Tensor x2 = x.dim() == 2 ? x : x.view({M, C});
    at::Tensor y = at::empty({M, p.rows}, x.options());
    *rc = linear_into(p, x2, y, gemm);
    if (*rc) return true;
    if (x.dim() == 2) { out = std::move(y); return true; }
    auto sizes = x.sizes().vec();
    sizes.back() = p.rows;
    out = y.view(sizes);
    return true;
}

// forward(shards, x) -> tensor or a code
PyObject* forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 2 || !THPVariable_Check(a[1])) return answer(NOT_COVERED);
    SQ_GUARD(
        at::Tensor out;
        int rc;
        if (!shards_forward(a[0], THPVariable_Unpack(a[1]), out, &rc)) return nullptr;
        return rc ? answer(rc) : THPVariable_Wrap(std::move(out));
    )
}

// addnorm operands as the library takes them; `C` columns, `B` rows, the 16-bit operands of type `dt` (dt < 0: their own)
struct Norm { const float* h_in; float* h_out; const void* add; const void* w; int add_dt = 0, w_dt = 0; int64_t ld_h = 0, ld_add = 0; };
bool norm_operands(PyObject* h_in, PyObject* add, PyObject* w, PyObject* h_out, int dev, int64_t B, int64_t C, int dt, Norm& o) {
    if (!THPVariable_Check(h_in) || !THPVariable_Check(w)) return false;
    const at::Tensor& h = THPVariable_Unpack(h_in);
    const at::Tensor& wt = THPVariable_Unpack(w);
    if (h.scalar_type() != at::kFloat || !matrix_on(h, dev) || h.size(0) != B || h.size(1) != C) return false;
    o.w_dt = dtype_of(wt);
    if (!wt.is_cuda() || wt.get_device() != dev || wt.numel() != C || !wt.is_contiguous() || !is16(o.w_dt) || (dt >= 0 && o.w_dt != dt)) return false;
    o.h_in = (const float*)h.data_ptr(); o.ld_h = row_ld(h); o.w = wt.data_ptr();
    o.add = nullptr; o.h_out = nullptr;
    if (add != Py_None) {
        if (!THPVariable_Check(add)) return false;
        const at::Tensor& t = THPVariable_Unpack(add);
        o.add_dt = dtype_of(t);
        if (!is16(o.add_dt) || (dt >= 0 && o.add_dt != dt) || !matrix_on(t, dev) || t.size(0) != B || t.size(1) != C) return false;
        o.add = t.data_ptr(); o.ld_add = row_ld(t);
    }
    if (h_out != Py_None) {
        if (!THPVariable_Check(h_out)) return false;
        const at::Tensor& t = THPVariable_Unpack(h_out);
        if (t.scalar_type() != at::kFloat || !matrix_on(t, dev) || t.sizes() != h.sizes() || t.strides() != h.strides()) return false;
        o.h_out = (float*)t.data_ptr();
    }
    return true;
}
bool perm_operand(PyObject* perms, int dev, int64_t C, const int32_t** pp, int* M) {
    *pp = nullptr; *M = 1;
    if (perms == Py_None) return true;
    if (!THPVariable_Check(perms)) return false;
    const at::Tensor& t = THPVariable_Unpack(perms);
    if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(1) != C || !t.is_contiguous() || !t.is_cuda() || t.get_device() != dev) return false;
    *pp = (const int32_t*)t.data_ptr(); *M = (int)t.size(0);
    return true;
}

// addnorm(h_in, add, w, eps, out, h_out, perms)
PyObject* addnorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 7 || !THPVariable_Check(a[0]) || !THPVariable_Check(a[4])) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& h = THPVariable_Unpack(a[0]);
        const at::Tensor& out = THPVariable_Unpack(a[4]);
        if (h.dim() != 2 || !h.is_cuda()) return answer(NOT_COVERED);
        const int dev = h.get_device();
        const int64_t B = h.size(0); const int64_t C = h.size(1);
        Norm o; const int32_t* pp; int M;
        const double eps = PyFloat_AsDouble(a[3]);
        if (PyErr_Occurred()) return nullptr;
        if (B < 1 || !norm_operands(a[0], a[1], a[2], a[5], dev, B, C, -1, o) || !perm_operand(a[6], dev, C, &pp, &M) || !is16(dtype_of(out)) ||
            !out.is_cuda() || out.get_device() != dev || !out.is_contiguous() || out.numel() != B * M * C)
            return answer(NOT_COVERED);
        OnDevice on(dev);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_addnorm(o.h_in, o.h_out, h.stride(0), o.add, o.add_dt, o.ld_add, o.w, o.w_dt, pp, M, (int)B, (int)C, (float)eps, out.data_ptr(), dtype_of(out), on.stream);
        Py_END_ALLOW_THREADS
        return answer(rc);
    )
}

// silu_mul(gate, up, out, perms)
PyObject* silu_mul(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 4 || !tensors(a, 3)) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& g = THPVariable_Unpack(a[0]);
        const at::Tensor& u = THPVariable_Unpack(a[1]);
        const at::Tensor& out = THPVariable_Unpack(a[2]);
        if (g.dim() != 2 || !g.is_cuda()) return answer(NOT_COVERED);
        const int dev = g.get_device(); const int dt = dtype_of(g);
        const int64_t B = g.size(0); const int64_t C = g.size(1);
        const int32_t* pp; int M;
        if (B < 1 || !is16(dt) || !matrix_on(g, dev) || !matrix_on(u, dev) || dtype_of(u) != dt || u.sizes() != g.sizes() || u.strides() != g.strides() ||
            !perm_operand(a[3], dev, C, &pp, &M) || dtype_of(out) != dt || !out.is_cuda() || out.get_device() != dev || !out.is_contiguous() || out.numel() != B * M * C)
            return answer(NOT_COVERED);
        OnDevice on(dev);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_silu_mul(g.data_ptr(), u.data_ptr(), dt, g.stride(0), pp, M, (int)B, (int)C, out.data_ptr(), on.stream);
        Py_END_ALLOW_THREADS
        return answer(rc);
    )
}

// linear_from(pieces, y, x_out, h_in, add, w, eps, h_out, gate, up)
PyObject* linear_from(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 10 || !tensors(a + 1, 2) || (a[3] == Py_None) == (a[8] == Py_None)) return answer(NOT_COVERED);
    SQ_GUARD(
        Pieces p;
        if (int rc = unpack_pieces(a[0], p)) return answer(rc);
        const at::Tensor& y = THPVariable_Unpack(a[1]);
        const at::Tensor& x = THPVariable_Unpack(a[2]);
        const int dt = dtype_of(x); const int yd = dtype_of(y);
        if (!is16(dt) || yd < 0 || !matrix_on(x, p.dev) || !x.is_contiguous() || !matrix_on(y, p.dev) || x.size(0) != y.size(0) || x.size(0) < 1 ||
            y.size(1) != p.rows || x.size(1) != p.m[0].C)
            return answer(NOT_COVERED);
        const int64_t B = x.size(0); const int64_t C = x.size(1);
        sq_producer pr{};
        pr.x_out = x.data_ptr();
        pr.eps = (float)PyFloat_AsDouble(a[6]);
        if (PyErr_Occurred()) return nullptr;
        if (a[3] != Py_None) {
            Norm o;
            if (!norm_operands(a[3], a[4], a[5], a[7], p.dev, B, C, dt, o)) return answer(NOT_COVERED);
            pr.mode = SQ_FROM_ADDNORM; pr.h_in = o.h_in; pr.h_out = o.h_out; pr.add = o.add; pr.w = o.w; pr.ld_h = o.ld_h; pr.ld_in = o.ld_add;
        } else {
            if (!tensors(a + 8, 2)) return answer(NOT_COVERED);
            const at::Tensor& g = THPVariable_Unpack(a[8]);
            const at::Tensor& u = THPVariable_Unpack(a[9]);
            if (dtype_of(g) != dt || dtype_of(u) != dt || !matrix_on(g, p.dev) || !matrix_on(u, p.dev) || g.sizes() != x.sizes() || u.sizes() != g.sizes() ||
                u.strides() != g.strides())
                return answer(NOT_COVERED);
            pr.mode = SQ_FROM_SILU_MUL; pr.add = g.data_ptr(); pr.up = u.data_ptr(); pr.ld_in = row_ld(g);
        }
        OnDevice on(p.dev);
        Workspace ws;
        if (!product_workspace(p, (int)B, 0, y, on.stream, ws)) return answer(NOT_COVERED);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_linear_small_from(p.m, p.n, &pr, dt, y.data_ptr(), yd, row_ld(y), (int)B, ws.p, ws.bytes, on.stream);
        Py_END_ALLOW_THREADS
        return answer(rc);
    )
}

// linear_silu(pieces, x, out, x_out, h_in, add, w, eps, h_out)
PyObject* linear_silu(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const bool norm = n == 9 && a[4] != Py_None;
    if (n != 9 || !THPVariable_Check(a[norm ? 3 : 1]) || !THPVariable_Check(a[2])) return answer(NOT_COVERED);
    SQ_GUARD(
        Pieces p;
        if (int rc = unpack_pieces(a[0], p)) return answer(rc);
        const at::Tensor& x = THPVariable_Unpack(a[norm ? 3 : 1]);
        const at::Tensor& out = THPVariable_Unpack(a[2]);
        const int dt = dtype_of(x);
        if (p.n != 2 || p.m[0].R != p.m[1].R || !is16(dt) || dtype_of(out) != dt || !matrix_on(x, p.dev) || !matrix_on(out, p.dev) || x.size(0) < 1 ||
            out.size(0) != x.size(0) || out.size(1) != p.m[0].R || x.size(1) != p.m[0].C)
            return answer(NOT_COVERED);
        const int64_t B = x.size(0);
        sq_producer pr{};
        if (norm) {
            Norm o;
            pr.eps = (float)PyFloat_AsDouble(a[7]);
            if (PyErr_Occurred()) return nullptr;
            if (B != 1 || !x.is_contiguous() || !norm_operands(a[4], a[5], a[6], a[8], p.dev, B, x.size(1), dt, o)) return answer(NOT_COVERED);
            pr.mode = SQ_FROM_ADDNORM; pr.x_out = x.data_ptr();
            pr.h_in = o.h_in; pr.h_out = o.h_out; pr.add = o.add; pr.w = o.w; pr.ld_h = o.ld_h; pr.ld_in = o.ld_add;
        }
        OnDevice on(p.dev);
        Workspace ws;
        if (!product_workspace(p, (int)B, 0, out, on.stream, ws)) return answer(NOT_COVERED);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_linear_small_silu(p.m, 2, norm ? &pr : nullptr, norm ? nullptr : x.data_ptr(), dt, norm ? 0 : row_ld(x), out.data_ptr(), row_ld(out), (int)B,
                                  ws.p, ws.bytes, on.stream);
        Py_END_ALLOW_THREADS
        if (rc != SQ_EUNSUPPORTED) return answer(rc);
        // no fused kernel for this stack: the product into a temporary, then SiLU * up (which writes whole rows)
        if (!out.is_contiguous()) return answer(NOT_COVERED);
        const at::Tensor y = at::empty({B, p.rows}, x.options());
        uint16_t* yp = (uint16_t*)y.data_ptr();
        Py_BEGIN_ALLOW_THREADS
        rc = norm ? sq_linear_small_from(p.m, 2, &pr, dt, yp, dt, p.rows, (int)B, ws.p, ws.bytes, on.stream)
                  : sq_linear_small(p.m, 2, x.data_ptr(), dt, row_ld(x), yp, dt, p.rows, (int)B, ws.p, ws.bytes, on.stream);
        if (rc == SQ_OK) rc = sq_silu_mul(yp, yp + p.m[0].R, dt, p.rows, nullptr, 1, (int)B, p.m[0].R, out.data_ptr(), on.stream);
        Py_END_ALLOW_THREADS
        return answer(rc);
    )
}

// q8_linear(q, scale, x, y)
PyObject* q8_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 4 || !tensors(a, 4)) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& q = THPVariable_Unpack(a[0]);
        const at::Tensor& sc = THPVariable_Unpack(a[1]);
        const at::Tensor& x = THPVariable_Unpack(a[2]);
        const at::Tensor& y = THPVariable_Unpack(a[3]);
        if (!q.is_cuda() || q.dim() != 2 || q.scalar_type() != at::kChar || !q.is_contiguous()) return answer(NOT_COVERED);
        const int dev = q.get_device(); const int xd = dtype_of(x); const int yd = dtype_of(y);
        const int64_t V = q.size(0); const int64_t C = q.size(1);
        if (C % 32 || !sc.is_cuda() || sc.get_device() != dev || sc.scalar_type() != at::kHalf || !sc.is_contiguous() || sc.dim() != 2 || sc.size(0) != V ||
            sc.size(1) != C / 32 || !is16(xd) || yd < 0 || !matrix_on(x, dev) || !matrix_on(y, dev) || x.size(1) != C || x.size(0) < 1 || y.size(0) != x.size(0) ||
            y.size(1) < V)
            return answer(NOT_COVERED);
        OnDevice on(dev);
        Workspace ws;
        const size_t need = sq_q8_workspace_bytes((int)V, (int)C, (int)x.size(0));
        if (need && C % 256 && x.size(0) <= SQ_SMALL_BMAX) {     // (a buffer of its own: see kernels.q8_linear)
            ws.held = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
            ws.p = ws.held.data_ptr();
            ws.bytes = need;
        } else if (!workspace(dev, need, on.stream, ws)) {
            return answer(NOT_COVERED);
        }
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_q8_linear((const int8_t*)q.data_ptr(), (const uint16_t*)sc.data_ptr(), (int)V, (int)C, x.data_ptr(), xd, x.stride(0), y.data_ptr(), yd, y.stride(0),
                          (int)x.size(0), ws.p, ws.bytes, on.stream);
        Py_END_ALLOW_THREADS
        return answer(rc);
    )
}

// q4_rows(q, scale, ids, dtype code) -> [len(ids), C], or a code; tables on the GPU (pinned host tables: Python)
PyObject* q4_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 4 || !tensors(a, 3)) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& q = THPVariable_Unpack(a[0]);
        const at::Tensor& sc = THPVariable_Unpack(a[1]);
        const at::Tensor& ids = THPVariable_Unpack(a[2]);
        const long dt = PyLong_AsLong(a[3]);
        if (PyErr_Occurred()) return nullptr;
        if (!q.is_cuda() || q.dim() != 2 || q.scalar_type() != at::kByte || !q.is_contiguous() || !ids.is_cuda() || ids.get_device() != q.get_device() ||
            ids.dim() != 1 || ids.scalar_type() != at::kLong || !ids.is_contiguous() || ids.unsafeGetTensorImpl()->is_python_dispatch() || dt < SQ_F32 || dt > SQ_BF16)
            return answer(NOT_COVERED);
        const int dev = q.get_device();
        const int64_t V = q.size(0); const int64_t C = q.size(1) * 2;
        if (C % 32 || !sc.is_cuda() || sc.get_device() != dev || sc.scalar_type() != at::kHalf || !sc.is_contiguous() || sc.dim() != 2 || sc.size(0) != V ||
            sc.size(1) != C / 32)
            return answer(NOT_COVERED);
        OnDevice on(dev);
        at::Tensor out = at::empty({ids.numel(), C}, q.options().dtype(dt == SQ_F32 ? at::kFloat : dt == SQ_F16 ? at::kHalf : at::kBFloat16));
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_q4_embed((const uint8_t*)q.data_ptr(), (const uint16_t*)sc.data_ptr(), (int)V, (int)C, (const int64_t*)ids.data_ptr(), ids.numel(), out.data_ptr(),
                         (int)dt, C, on.stream);
        Py_END_ALLOW_THREADS
        return rc ? answer(rc) : THPVariable_Wrap(std::move(out));
    )
}

// ------------------------------------------------------------------------------------------ heads of q|k|v, attention

// A tensor these calls take as it is: on `dev`, strided, nothing that Python dispatches, that a gradient would be recorded for or that has a tangent
bool plain_on(const at::Tensor& t, int dev) {
    return t.is_cuda() && t.get_device() == dev && t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() &&
           !(t.requires_grad() && at::GradMode::is_enabled()) && !t._fw_grad(0).defined();
}
// An argument that may be None: NULL, or the tensor; false where it is neither
bool maybe(PyObject* o, const at::Tensor*& t) {
    t = nullptr;
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) return false;
    t = &THPVariable_Unpack(o);
    return true;
}
bool heads_on(const at::Tensor& t, int dev) { return t.dim() == 3 && plain_on(t, dev) && dtype_of(t) >= 0 && (t.stride(2) == 1 || t.size(2) == 1); }
bool vector_on(const at::Tensor& t, int dev, int64_t n, at::ScalarType a, at::ScalarType b) {
    return t.dim() == 1 && t.size(0) == n && (t.scalar_type() == a || t.scalar_type() == b) && plain_on(t, dev) && t.is_contiguous();
}
bool rows_on(const at::Tensor& t, int dev, int64_t n, at::ScalarType type) {
    return t.dim() == 2 && t.size(0) == n && t.scalar_type() == type && plain_on(t, dev) && (t.stride(1) == 1 || t.size(1) <= 1) &&
           (n <= 1 || t.stride(0) >= t.size(1));
}
bool apart(const at::Tensor& a, const at::Tensor& b) {       // no byte between the first and the last of both
    auto ends = [](const at::Tensor& t, uintptr_t& lo, uintptr_t& hi) {
        lo = hi = (uintptr_t)t.data_ptr();
        for (int i = 0; i < t.dim(); ++i) (t.stride(i) > 0 ? hi : lo) += (t.size(i) - 1) * t.stride(i) * (int64_t)t.element_size();
        hi += t.element_size();
    };
    uintptr_t al, ah, bl, bh;
    ends(a, al, ah);
    ends(b, bl, bh);
    return ah <= bl || bh <= al;
}
// No element of heads a in heads b: apart, or in different columns of one stacked product's rows
bool columns_apart(const at::Tensor& a, const at::Tensor& b) {
    if (apart(a, b)) return true;
    const int64_t row = a.stride(0); const int64_t size = a.element_size(); const int64_t bytes = (const char*)b.data_ptr() - (const char*)a.data_ptr();
    if (b.element_size() != size || b.stride(0) != row || row <= 0 || a.stride(1) < 0 || b.stride(1) < 0 || bytes % size) return false;
    const int64_t at = ((bytes / size) % row + row) % row;
    return at >= (a.size(1) - 1) * a.stride(1) + a.size(2) && at + (b.size(1) - 1) * b.stride(1) + b.size(2) <= row;
}
// out is x, or apart from it, with x's shape and type
bool out_ok(const at::Tensor& out, const at::Tensor& x, int dev) {
    return heads_on(out, dev) && out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() &&
           ((out.data_ptr() == x.data_ptr() && out.strides() == x.strides()) || apart(out, x));
}
sq_heads part_of(const at::Tensor& x, const at::Tensor* out, const at::Tensor* w) {
    const at::Tensor& o = out ? *out : x;
    return {x.data_ptr(), out ? out->data_ptr() : nullptr, w ? w->data_ptr() : nullptr, x.stride(0), x.stride(1), o.stride(0), o.stride(1), (int32_t)x.size(1)};
}
bool rotation_of(const at::Tensor& pos, const at::Tensor& freqs, int64_t n, int64_t dim, bool interleaved, double scale, bool inverse, int dev, sq_rotation& r) {
    if (!vector_on(pos, dev, n, at::kLong, at::kInt) || !vector_on(freqs, dev, freqs.numel(), at::kDouble, at::kDouble) || 2 * freqs.numel() > dim) return false;
    r = {(const double*)freqs.data_ptr(), pos.data_ptr(), (int32_t)freqs.numel(), pos.scalar_type() == at::kLong, interleaved, inverse, (float)scale};
    return true;
}
// the last four dimensions of a pair of caches; not where they are written and expanded
bool cache_of(const at::Tensor& k, const at::Tensor& v, int dev, bool written, sq_cache& c) {
    const int d = (int)k.dim();
    if ((d != 4 && d != 5) || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || dtype_of(k) < 0 || !plain_on(k, dev) || !plain_on(v, dev) || k.numel() == 0 ||
        k.numel() / k.size(d - 4) > INT32_MAX || k.size(d - 4) > INT32_MAX)
        return false;
    for (const at::Tensor* t : {&k, &v}) {
        if (t->stride(d - 1) != 1 && t->size(d - 1) > 1) return false;
        for (int i = 0; written && i < d; ++i) if (t->stride(i) == 0 && t->size(i) > 1) return false;
    }
    if (written && k.data_ptr() == v.data_ptr()) return false;
    c = {k.data_ptr(), v.data_ptr(), k.stride(d - 4), k.stride(d - 3), k.stride(d - 2), v.stride(d - 4), v.stride(d - 3), v.stride(d - 2), (int32_t)k.size(d - 4),
         (int32_t)k.size(d - 3), (int32_t)k.size(d - 2), (int32_t)k.size(d - 1), dtype_of(k)};
    return true;
}

// rotary(x, positions, freqs, out, interleaved, scale, inverse) -> out, or a code
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const at::Tensor* given;
    if (n != 7 || !tensors(a, 3) || !maybe(a[3], given)) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& x = THPVariable_Unpack(a[0]);
        const double scale = PyFloat_AsDouble(a[5]);
        const int inter = PyObject_IsTrue(a[4]); const int inverse = PyObject_IsTrue(a[6]);
        if (PyErr_Occurred()) return nullptr;
        if (x.dim() != 3 || !x.is_cuda() || x.numel() == 0 || x.size(0) > INT32_MAX || x.size(1) > INT32_MAX || x.size(2) > INT32_MAX) return answer(NOT_COVERED);
        const int dev = x.get_device();
        sq_rotation r;
        if (!heads_on(x, dev) || !rotation_of(THPVariable_Unpack(a[1]), THPVariable_Unpack(a[2]), x.size(0), x.size(2), inter, scale, inverse, dev, r) ||
            (given && !out_ok(*given, x, dev)))
            return answer(NOT_COVERED);
        OnDevice on(dev);
        at::Tensor out = given ? *given : at::empty(x.sizes(), x.options());
        const sq_heads h = part_of(x, &out, nullptr);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_rotary(&h, (int)x.size(0), (int)x.size(2), dtype_of(x), &r, on.stream);
        Py_END_ALLOW_THREADS
        return rc ? answer(rc) : THPVariable_Wrap(std::move(out));
    )
}

// qk_norm_rotary(q, k, positions, freqs, q_w, k_w, eps, q_out, k_out, v, k_cache, v_cache, slots, interleaved, scale, offset) -> (q_out, k_out), or a code
PyObject* qk_norm_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const at::Tensor *qw, *kw, *qg, *kg, *v, *kc, *vc, *slots;
    if (n != 16 || !tensors(a, 4) || !maybe(a[4], qw) || !maybe(a[5], kw) || !maybe(a[7], qg) || !maybe(a[8], kg) || !maybe(a[9], v) || !maybe(a[10], kc) ||
        !maybe(a[11], vc) || !maybe(a[12], slots))
        return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& q = THPVariable_Unpack(a[0]);
        const at::Tensor& k = THPVariable_Unpack(a[1]);
        const double eps = PyFloat_AsDouble(a[6]); const double scale = PyFloat_AsDouble(a[14]); const double offset = PyFloat_AsDouble(a[15]);
        const int inter = PyObject_IsTrue(a[13]);
        if (PyErr_Occurred()) return nullptr;
        if (q.dim() != 3 || !q.is_cuda() || q.numel() == 0 || k.dim() != 3 || k.numel() == 0 || q.numel() > INT32_MAX || k.numel() > INT32_MAX) return answer(NOT_COVERED);
        const int dev = q.get_device(); const int dt = dtype_of(q);
        const int64_t rows = q.size(0); const int64_t d = q.size(2);
        const bool cached = kc != nullptr;
        sq_rotation r; sq_cache c;
        if (!heads_on(q, dev) || !heads_on(k, dev) || k.scalar_type() != q.scalar_type() || k.size(0) != rows || k.size(2) != d || (vc != nullptr) != cached ||
            (v != nullptr) != cached || (slots != nullptr) != cached ||
            !rotation_of(THPVariable_Unpack(a[2]), THPVariable_Unpack(a[3]), rows, d, inter, scale, false, dev, r))
            return answer(NOT_COVERED);
        int wd = dt;
        for (const at::Tensor* w : {qw, kw})
            if (w && (dtype_of(*w) < 0 || !vector_on(*w, dev, d, w->scalar_type(), w->scalar_type()))) return answer(NOT_COVERED);
        if (qw && kw && qw->scalar_type() != kw->scalar_type()) return answer(NOT_COVERED);
        if (qw || kw) wd = dtype_of(qw ? *qw : *kw);
        if (v && (v->dim() != 3 || v->numel() == 0)) return answer(NOT_COVERED);
        for (int i = 0; i < 2; ++i) {
            const at::Tensor* g = i ? kg : qg;
            if (g && (!out_ok(*g, i ? k : q, dev) || !columns_apart(*g, i ? q : k) || (v && !columns_apart(*g, *v)) || (i && qg && !columns_apart(*g, *qg))))
                return answer(NOT_COVERED);                  // (Python says what is wrong)
        }
        if (cached) {
            if (!heads_on(*v, dev) || v->sizes() != k.sizes() || v->scalar_type() != q.scalar_type() || !vector_on(*slots, dev, rows, at::kLong, at::kInt) || kc->dim() != 4 ||
                !cache_of(*kc, *vc, dev, true, c) || c.dtype != dt || c.heads != k.size(1) || c.dim != d)
                return answer(NOT_COVERED);
            for (const at::Tensor* t : {&q, &k, v, qg, kg})
                if (t && (!apart(*kc, *t) || !apart(*vc, *t))) return answer(NOT_COVERED);
        }
        OnDevice on(dev);
        at::Tensor qo = qg ? *qg : at::empty(q.sizes(), q.options());
        at::Tensor ko;
        if (kg) ko = *kg; else if (!cached) ko = at::empty(k.sizes(), k.options());
        const sq_heads hq = part_of(q, &qo, qw); const sq_heads hk = part_of(k, ko.defined() ? &ko : nullptr, kw);
        sq_heads hv{};
        if (cached) hv = part_of(*v, nullptr, nullptr);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_qk_norm_rotary(&hq, &hk, cached ? &hv : nullptr, (int)rows, (int)d, dt, &r, wd, (float)eps, (float)offset, cached ? &c : nullptr,
                               cached ? slots->data_ptr() : nullptr, cached && slots->scalar_type() == at::kLong, on.stream);
        Py_END_ALLOW_THREADS
        if (rc) return answer(rc);
        PyObject* both = PyTuple_New(2);
        if (!both) return nullptr;
        PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(qo)));
        if (ko.defined()) PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(ko)));
        else { Py_INCREF(Py_None); PyTuple_SET_ITEM(both, 1, Py_None); }
        return both;
    )
}

// tree_attention(q, k_cache, v_cache, table, lens, starts, most_new, mask, scale, out, lse) -> out, or a code
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const at::Tensor *starts, *mask, *given, *lse;
    if (n != 11 || !tensors(a, 5) || !maybe(a[5], starts) || !maybe(a[7], mask) || !maybe(a[9], given) || !maybe(a[10], lse)) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& q = THPVariable_Unpack(a[0]);
        const at::Tensor& kc = THPVariable_Unpack(a[1]);
        const at::Tensor& vc = THPVariable_Unpack(a[2]);
        const at::Tensor& table = THPVariable_Unpack(a[3]);
        const at::Tensor& lens = THPVariable_Unpack(a[4]);
        if (q.dim() != 3 || !q.is_cuda() || q.numel() == 0 || q.numel() > INT32_MAX || lens.dim() != 1 || lens.size(0) < 1 || lens.size(0) > INT32_MAX) return answer(NOT_COVERED);
        const int dev = q.get_device();
        const int64_t rows = q.size(0); const int64_t b = lens.size(0);
        sq_cache c; sq_attention t{};
        if (!heads_on(q, dev) || kc.dim() != 4 || !cache_of(kc, vc, dev, false, c) || c.dtype == SQ_F32 || c.dtype != dtype_of(q) || c.dim != q.size(2) ||
            q.size(1) % c.heads || !vector_on(lens, dev, b, at::kInt, at::kInt) || !rows_on(table, dev, b, at::kInt) || table.size(1) > INT32_MAX ||
            (starts && !vector_on(*starts, dev, b + 1, at::kInt, at::kInt)) || (!starts && rows % b) || (mask && (!rows_on(*mask, dev, rows, at::kLong) || mask->size(1) > INT32_MAX)) ||
            (lse && (lse->scalar_type() != at::kFloat || lse->dim() != 2 || lse->size(0) != rows || lse->size(1) != q.size(1) || !plain_on(*lse, dev) || !lse->is_contiguous())))
            return answer(NOT_COVERED);
        int64_t most = starts ? rows : rows / b;
        if (a[6] != Py_None) most = starts ? std::min<int64_t>(PyLong_AsLongLong(a[6]), rows) : PyLong_AsLongLong(a[6]);
        const double scale = a[8] == Py_None ? std::pow((double)c.dim, -0.5) : PyFloat_AsDouble(a[8]);
        if (PyErr_Occurred()) return nullptr;
        if (most < 0 || most > INT32_MAX || (!starts && most * b != rows) || !(scale > 0 && scale < 2.3e38)) return answer(NOT_COVERED);
        if (given && (!heads_on(*given, dev) || given->sizes() != q.sizes() || given->scalar_type() != q.scalar_type() || !apart(*given, q) || !apart(*given, kc) || !apart(*given, vc) ||
                      (given->stride(0) == 0 && rows > 1) || (given->stride(1) == 0 && q.size(1) > 1)))
            return answer(NOT_COVERED);
        OnDevice on(dev);
        at::Tensor out = given ? *given : at::empty(q.sizes(), q.options());
        t.q = q.data_ptr(); t.out = out.data_ptr(); t.lse = lse ? (float*)lse->data_ptr() : nullptr; t.table = (const int32_t*)table.data_ptr();
        t.lens = (const int32_t*)lens.data_ptr(); t.starts = starts ? (const int32_t*)starts->data_ptr() : nullptr; t.mask = mask ? (const int64_t*)mask->data_ptr() : nullptr;
        if (mask && !t.mask) t.mask = (const int64_t*)lens.data_ptr();       // (a mask without words has no address, and none would mean no mask; nothing is read there)
        t.q_token = q.stride(0); t.q_head = q.stride(1); t.out_token = out.stride(0); t.out_head = out.stride(1);
        t.ld_table = b > 1 ? table.stride(0) : table.size(1); t.ld_mask = mask ? rows > 1 ? mask->stride(0) : mask->size(1) : 0;
        t.tokens = (int32_t)rows; t.seqs = (int32_t)b; t.most_new = (int32_t)most; t.q_heads = (int32_t)q.size(1); t.max_pages = (int32_t)table.size(1);
        t.mask_words = mask ? (int32_t)mask->size(1) : 0; t.scale = (float)scale;
        // (a buffer of the call's own: streams and captured graphs run side by side)
        const size_t need = sq_tree_attention_workspace_bytes(&t, &c);
        at::Tensor ws;
        if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_tree_attention(&t, &c, need ? ws.data_ptr() : nullptr, need, on.stream);
        Py_END_ALLOW_THREADS
        return rc ? answer(rc) : THPVariable_Wrap(std::move(out));
    )
}

// keep_drafted(k_cache, v_cache, table, lens, path, counts)
PyObject* keep_drafted(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 6 || !tensors(a, 6)) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& kc = THPVariable_Unpack(a[0]);
        const at::Tensor& vc = THPVariable_Unpack(a[1]);
        const at::Tensor& table = THPVariable_Unpack(a[2]);
        const at::Tensor& lens = THPVariable_Unpack(a[3]);
        const at::Tensor& path = THPVariable_Unpack(a[4]);
        if (!kc.is_cuda() || lens.dim() != 1 || lens.size(0) < 1 || lens.size(0) > INT32_MAX) return answer(NOT_COVERED);
        const int dev = kc.get_device();
        const int64_t b = lens.size(0);
        sq_cache c;
        if (!cache_of(kc, vc, dev, true, c) || !vector_on(lens, dev, b, at::kInt, at::kInt) || !vector_on(THPVariable_Unpack(a[5]), dev, b, at::kInt, at::kInt) ||
            !rows_on(table, dev, b, at::kInt) || !rows_on(path, dev, b, at::kInt) || table.size(1) > INT32_MAX || path.size(1) > INT32_MAX)
            return answer(NOT_COVERED);
        const bool stacked = kc.dim() == 5;
        if (stacked && kc.size(0) > INT32_MAX) return answer(NOT_COVERED);
        OnDevice on(dev);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_keep_drafted(&c, stacked ? (int)kc.size(0) : 1, stacked ? kc.stride(0) : 0, stacked ? vc.stride(0) : 0, (const int32_t*)table.data_ptr(),
                             b > 1 ? table.stride(0) : table.size(1), (int)table.size(1), (const int32_t*)lens.data_ptr(), (const int32_t*)path.data_ptr(),
                             b > 1 ? path.stride(0) : path.size(1), (int)path.size(1), (const int32_t*)THPVariable_Unpack(a[5]).data_ptr(), (int)b, on.stream);
        Py_END_ALLOW_THREADS
        return answer(rc);
    )
}

// ------------------------------------------------------------------------------------------ 8-bit caches, pages

// the last dimensions of an 8-bit cache's four tensors, for a call that takes these numbers of dimensions; not where they are written and expanded
bool cache8_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs, int dev, bool stacked, bool written, sq_cache8& c) {
    const int d = (int)k.dim(); const int e = d - 1;
    if ((d != 4 && !(stacked && d == 5)) || k.sizes() != v.sizes() || ks.dim() != e || ks.sizes() != vs.sizes() || k.numel() == 0 || ks.numel() == 0) return false;
    const at::Tensor* every[4] = {&k, &v, &ks, &vs};         // (one tensor given twice is one address twice)
    for (int j = 0; j < 4; ++j) {
        const at::Tensor& t = *every[j];
        if (t.scalar_type() != (j < 2 ? at::kFloat8_e4m3fn : at::kFloat8_e8m0fnu) || !plain_on(t, dev)) return false;
        for (int i = 0; written && i < t.dim(); ++i) if (t.stride(i) == 0 && t.size(i) > 1) return false;
        for (int i = 0; written && i < j; ++i) if (every[i]->data_ptr() == t.data_ptr()) return false;
    }
    if ((k.stride(d - 1) != 1 && k.size(d - 1) > 1) || (v.stride(d - 1) != 1 && v.size(d - 1) > 1)) return false;
    for (int i = 0; i < d - 3; ++i) if (ks.size(i) != k.size(i)) return false;
    for (int i = 0; i < d; ++i) if (k.size(i) > INT32_MAX) return false;
    if (ks.size(e - 1) != k.size(d - 2) || k.size(d - 3) % ks.size(e - 2)) return false;
    c = {k.data_ptr(), v.data_ptr(), (uint8_t*)ks.data_ptr(), (uint8_t*)vs.data_ptr(), k.stride(d - 4), k.stride(d - 3), k.stride(d - 2), v.stride(d - 4), v.stride(d - 3), v.stride(d - 2),
         ks.stride(e - 3), ks.stride(e - 2), ks.stride(e - 1), vs.stride(e - 3), vs.stride(e - 2), vs.stride(e - 1),
         (int32_t)k.size(d - 4), (int32_t)k.size(d - 3), (int32_t)ks.size(e - 2), (int32_t)k.size(d - 2), (int32_t)k.size(d - 1)};
    return true;
}
// a batch of sequences: lens, table and, or NULL, starts
bool batch_on(const at::Tensor& table, const at::Tensor& lens, const at::Tensor* starts, int dev) {
    if (lens.dim() != 1 || lens.size(0) < 1 || lens.size(0) > INT32_MAX) return false;
    const int64_t b = lens.size(0);
    return vector_on(lens, dev, b, at::kInt, at::kInt) && rows_on(table, dev, b, at::kInt) && table.size(1) <= INT32_MAX && (!starts || vector_on(*starts, dev, b + 1, at::kInt, at::kInt));
}
int64_t table_ld(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
// the most new tokens of a sequence, of `rows` in all; -1: not covered
int64_t most_of(PyObject* o, const at::Tensor* starts, int64_t rows, int64_t b) {
    if (!starts && rows % b) return -1;
    int64_t most = starts ? rows : rows / b;
    if (o != Py_None) most = starts ? std::min<int64_t>(PyLong_AsLongLong(o), rows) : PyLong_AsLongLong(o);
    return most < 0 || most > INT32_MAX || (!starts && most * b != rows) ? -1 : most;
}

// put_tokens8(k, v, k_cache, v_cache, k_scale, v_scale, table, lens, starts, most_new)
PyObject* put_tokens8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const at::Tensor* starts;
    if (n != 10 || !tensors(a, 8) || !maybe(a[8], starts)) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& k = THPVariable_Unpack(a[0]);
        const at::Tensor& v = THPVariable_Unpack(a[1]);
        const at::Tensor& table = THPVariable_Unpack(a[6]);
        const at::Tensor& lens = THPVariable_Unpack(a[7]);
        if (k.dim() != 3 || !k.is_cuda() || k.numel() == 0 || k.numel() > INT32_MAX || v.dim() != 3) return answer(NOT_COVERED);
        const int dev = k.get_device(); const int dt = dtype_of(k);
        sq_cache8 c;
        if (!heads_on(k, dev) || !heads_on(v, dev) || !is16(dt) || v.scalar_type() != k.scalar_type() || v.sizes() != k.sizes() || !batch_on(table, lens, starts, dev) ||
            !cache8_of(THPVariable_Unpack(a[2]), THPVariable_Unpack(a[3]), THPVariable_Unpack(a[4]), THPVariable_Unpack(a[5]), dev, false, true, c) ||
            c.heads != k.size(1) || c.dim != k.size(2))
            return answer(NOT_COVERED);
        for (int i = 2; i < 6; ++i)
            if (!apart(THPVariable_Unpack(a[i]), k) || !apart(THPVariable_Unpack(a[i]), v)) return answer(NOT_COVERED);
        const int64_t most = most_of(a[9], starts, k.size(0), lens.size(0));
        if (PyErr_Occurred()) return nullptr;
        if (most < 0) return answer(NOT_COVERED);
        OnDevice on(dev);
        const sq_heads hk = part_of(k, nullptr, nullptr); const sq_heads hv = part_of(v, nullptr, nullptr);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_put_tokens8(&hk, &hv, (int)k.size(0), dt, &c, (const int32_t*)table.data_ptr(), table_ld(table), (int)table.size(1), (const int32_t*)lens.data_ptr(),
                            starts ? (const int32_t*)starts->data_ptr() : nullptr, (int)lens.size(0), (int)most, on.stream);
        Py_END_ALLOW_THREADS
        return answer(rc);
    )
}

// tree_attention8(q, k_cache, v_cache, k_scale, v_scale, table, lens, starts, most_new, mask, scale, out, lse) -> out, or a code
PyObject* tree_attention8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const at::Tensor *starts, *mask, *given, *lse;
    if (n != 13 || !tensors(a, 7) || !maybe(a[7], starts) || !maybe(a[9], mask) || !maybe(a[11], given) || !maybe(a[12], lse)) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& q = THPVariable_Unpack(a[0]);
        const at::Tensor& table = THPVariable_Unpack(a[5]);
        const at::Tensor& lens = THPVariable_Unpack(a[6]);
        if (q.dim() != 3 || !q.is_cuda() || q.numel() == 0 || q.numel() > INT32_MAX) return answer(NOT_COVERED);
        const int dev = q.get_device(); const int dt = dtype_of(q);
        const int64_t rows = q.size(0);
        sq_cache8 c; sq_attention t{};
        if (!heads_on(q, dev) || !is16(dt) || !batch_on(table, lens, starts, dev) ||
            !cache8_of(THPVariable_Unpack(a[1]), THPVariable_Unpack(a[2]), THPVariable_Unpack(a[3]), THPVariable_Unpack(a[4]), dev, false, false, c) || c.dim != q.size(2) ||
            q.size(1) % c.heads || (mask && (!rows_on(*mask, dev, rows, at::kLong) || mask->size(1) > INT32_MAX)) ||
            (lse && (lse->scalar_type() != at::kFloat || lse->dim() != 2 || lse->size(0) != rows || lse->size(1) != q.size(1) || !plain_on(*lse, dev) || !lse->is_contiguous())))
            return answer(NOT_COVERED);
        const int64_t b = lens.size(0); const int64_t most = most_of(a[8], starts, rows, b);
        const double scale = a[10] == Py_None ? std::pow((double)c.dim, -0.5) : PyFloat_AsDouble(a[10]);
        if (PyErr_Occurred()) return nullptr;
        if (most < 0 || !(scale > 0 && scale < 2.3e38)) return answer(NOT_COVERED);
        if (given) {
            if (!heads_on(*given, dev) || given->sizes() != q.sizes() || given->scalar_type() != q.scalar_type() || !apart(*given, q) || (given->stride(0) == 0 && rows > 1) ||
                (given->stride(1) == 0 && q.size(1) > 1))
                return answer(NOT_COVERED);
            for (int i = 1; i < 5; ++i) if (!apart(*given, THPVariable_Unpack(a[i]))) return answer(NOT_COVERED);
        }
        OnDevice on(dev);
        at::Tensor out = given ? *given : at::empty(q.sizes(), q.options());
        t.q = q.data_ptr(); t.out = out.data_ptr(); t.lse = lse ? (float*)lse->data_ptr() : nullptr; t.table = (const int32_t*)table.data_ptr();
        t.lens = (const int32_t*)lens.data_ptr(); t.starts = starts ? (const int32_t*)starts->data_ptr() : nullptr; t.mask = mask ? (const int64_t*)mask->data_ptr() : nullptr;
        if (mask && !t.mask) t.mask = (const int64_t*)lens.data_ptr();       // (a mask without words has no address, and none would mean no mask; nothing is read there)
        t.q_token = q.stride(0); t.q_head = q.stride(1); t.out_token = out.stride(0); t.out_head = out.stride(1);
        t.ld_table = table_ld(table); t.ld_mask = mask ? table_ld(*mask) : 0;
        t.tokens = (int32_t)rows; t.seqs = (int32_t)b; t.most_new = (int32_t)most; t.q_heads = (int32_t)q.size(1); t.max_pages = (int32_t)table.size(1);
        t.mask_words = mask ? (int32_t)mask->size(1) : 0; t.scale = (float)scale;
        // (a buffer of the call's own: streams and captured graphs run side by side)
        const size_t need = sq_tree_attention8_workspace_bytes(&t, &c, dt);
        at::Tensor ws;
        if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_tree_attention8(&t, &c, dt, need ? ws.data_ptr() : nullptr, need, on.stream);
        Py_END_ALLOW_THREADS
        return rc ? answer(rc) : THPVariable_Wrap(std::move(out));
    )
}

// keep_drafted8(k_cache, v_cache, k_scale, v_scale, table, lens, path, counts)
PyObject* keep_drafted8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 8 || !tensors(a, 8)) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& kc = THPVariable_Unpack(a[0]);
        const at::Tensor& table = THPVariable_Unpack(a[4]);
        const at::Tensor& lens = THPVariable_Unpack(a[5]);
        const at::Tensor& path = THPVariable_Unpack(a[6]);
        const at::Tensor& counts = THPVariable_Unpack(a[7]);
        if (!kc.is_cuda()) return answer(NOT_COVERED);
        const int dev = kc.get_device();
        sq_cache8 c;
        if (!batch_on(table, lens, nullptr, dev) || !vector_on(counts, dev, lens.size(0), at::kInt, at::kInt) || !rows_on(path, dev, lens.size(0), at::kInt) || path.size(1) > INT32_MAX ||
            !cache8_of(kc, THPVariable_Unpack(a[1]), THPVariable_Unpack(a[2]), THPVariable_Unpack(a[3]), dev, true, true, c))
            return answer(NOT_COVERED);
        const bool stacked = kc.dim() == 5;
        auto step = [&](int i) { return stacked ? THPVariable_Unpack(a[i]).stride(0) : 0; };
        OnDevice on(dev);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_keep_drafted8(&c, stacked ? (int)kc.size(0) : 1, step(0), step(1), step(2), step(3), (const int32_t*)table.data_ptr(), table_ld(table), (int)table.size(1),
                              (const int32_t*)lens.data_ptr(), (const int32_t*)path.data_ptr(), table_ld(path), (int)path.size(1), (const int32_t*)counts.data_ptr(), (int)lens.size(0),
                              on.stream);
        Py_END_ALLOW_THREADS
        return answer(rc);
    )
}

// caches and, or NULL, scales as planes
struct Planes { sq_plane p[4]; int n = 0, layers, pages, page; };
bool planes_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor* ks, const at::Tensor* vs, int dev, Planes& o) {
    const int d = (int)k.dim();
    if ((d != 4 && d != 5) || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || k.numel() == 0 || (ks != nullptr) != (vs != nullptr)) return false;
    if (ks && (ks->dim() != d - 1 || ks->sizes() != vs->sizes() || ks->scalar_type() != vs->scalar_type() || ks->numel() == 0)) return false;
    for (int i = 0; i < d; ++i) if (k.size(i) > INT32_MAX) return false;
    for (int i = 0; ks && i < d - 3; ++i) if (ks->size(i) != k.size(i)) return false;
    o.layers = d == 5 ? (int)k.size(0) : 1; o.pages = (int)k.size(d - 4); o.page = (int)k.size(d - 3);
    const at::Tensor* every[4] = {&k, &v, ks, vs};
    for (int j = 0; j < 4 && every[j]; ++j) {
        const at::Tensor* t = every[j];
        const bool code = j < 2; const int64_t size = t->element_size(); const int e = (int)t->dim() - (code ? 4 : 3);
        if (!plain_on(*t, dev) || (code && t->stride(e + 3) != 1 && t->size(e + 3) > 1) || t->size(e + 2) > INT32_MAX) return false;
        for (int i = 0; i < t->dim(); ++i) if (t->stride(i) == 0 && t->size(i) > 1) return false;
        for (int i = 0; i < o.n; ++i) if (o.p[i].at == t->data_ptr()) return false;
        if (o.page % t->size(e + 1)) return false;
        o.p[o.n++] = {t->data_ptr(), e ? t->stride(0) * size : 0, t->stride(e) * size, t->stride(e + 1) * size, t->stride(e + 2) * size, (int32_t)t->size(e + 1),
                      (int32_t)t->size(e + 2), (int32_t)((code ? t->size(e + 3) : 1) * size)};
    }
    return true;
}

// fork_pages(k_cache, v_cache, table, lens, parent, pages, k_scale, v_scale, out_table, out_lens) -> (table, lens), or a code
PyObject* fork_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const at::Tensor *ks, *vs, *given, *given_lens;
    if (n != 10 || !tensors(a, 6) || !maybe(a[6], ks) || !maybe(a[7], vs) || !maybe(a[8], given) || !maybe(a[9], given_lens)) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& kc = THPVariable_Unpack(a[0]);
        const at::Tensor& table = THPVariable_Unpack(a[2]);
        const at::Tensor& lens = THPVariable_Unpack(a[3]);
        const at::Tensor& parent = THPVariable_Unpack(a[4]);
        const at::Tensor& pages = THPVariable_Unpack(a[5]);
        if (!kc.is_cuda() || parent.dim() != 1 || parent.size(0) < 1 || parent.size(0) > INT32_MAX || given || given_lens) return answer(NOT_COVERED);
        const int dev = kc.get_device(); const int64_t r = parent.size(0);
        Planes p;
        if (!batch_on(table, lens, nullptr, dev) || !vector_on(parent, dev, r, at::kInt, at::kInt) || !vector_on(pages, dev, r, at::kInt, at::kInt) ||
            !planes_of(kc, THPVariable_Unpack(a[1]), ks, vs, dev, p))
            return answer(NOT_COVERED);
        OnDevice on(dev);
        at::Tensor out = at::empty({r, table.size(1)}, lens.options()); at::Tensor out_lens = at::empty({r}, lens.options());
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_fork_pages(p.p, p.n, p.layers, p.pages, p.page, (const int32_t*)table.data_ptr(), table_ld(table), (int)table.size(1), (const int32_t*)lens.data_ptr(), (int)lens.size(0),
                           (const int32_t*)parent.data_ptr(), (const int32_t*)pages.data_ptr(), (int)r, (int32_t*)out.data_ptr(), table.size(1), (int32_t*)out_lens.data_ptr(), on.stream);
        Py_END_ALLOW_THREADS
        if (rc) return answer(rc);
        return pybind11::make_tuple(pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(out))),
                                    pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(out_lens)))).release().ptr();
    )
}

// compact_pages(k_cache, v_cache, table, lens, k_scale, v_scale, out_table) -> (table, used), or a code
PyObject* compact_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const at::Tensor *ks, *vs, *given;
    if (n != 7 || !tensors(a, 4) || !maybe(a[4], ks) || !maybe(a[5], vs) || !maybe(a[6], given)) return answer(NOT_COVERED);
    SQ_GUARD(
        const at::Tensor& kc = THPVariable_Unpack(a[0]);
        const at::Tensor& table = THPVariable_Unpack(a[2]);
        const at::Tensor& lens = THPVariable_Unpack(a[3]);
        if (!kc.is_cuda() || given) return answer(NOT_COVERED);
        const int dev = kc.get_device();
        Planes p;
        if (!batch_on(table, lens, nullptr, dev) || !planes_of(kc, THPVariable_Unpack(a[1]), ks, vs, dev, p)) return answer(NOT_COVERED);
        OnDevice on(dev);
        // (a workspace of the call's own: streams and captured graphs run side by side)
        const size_t need = sq_compact_pages_workspace_bytes(p.pages);
        at::Tensor out = at::empty({lens.size(0), table.size(1)}, lens.options()); at::Tensor used = at::empty({1}, lens.options());
        at::Tensor ws = at::empty({(int64_t)need}, lens.options().dtype(at::kByte));
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = sq_compact_pages(p.p, p.n, p.layers, p.pages, p.page, (const int32_t*)table.data_ptr(), table_ld(table), (int)table.size(1), (const int32_t*)lens.data_ptr(),
                              (int)lens.size(0), (int32_t*)out.data_ptr(), table.size(1), (int32_t*)used.data_ptr(), ws.data_ptr(), need, on.stream);
        Py_END_ALLOW_THREADS
        if (rc) return answer(rc);
        return pybind11::make_tuple(pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(out))),
                                    pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(used)))).release().ptr();
    )
}

// ------------------------------------------------------------------------------------------ torch.ops.shapequant.linear

at::Tensor linear_op(const at::Tensor& x, int64_t handle) {
    pybind11::gil_scoped_acquire gil;
    if (!g_core) throw std::runtime_error("shapequant::linear: quantexperiments_amd.vllm_ext.core is not loaded");
    auto own = [](PyObject* o) { if (!o) throw pybind11::error_already_set(); return pybind11::reinterpret_steal<pybind11::object>(o); };
    pybind11::object obj = own(PySequence_GetItem(g_registry, (Py_ssize_t)handle));
    pybind11::object trace = own(PyObject_GetAttr(g_core, s_trace)), on = own(PyObject_GetAttr(trace.ptr(), s_enabled));
    if (on.ptr() == Py_False && Py_TYPE(obj.ptr()) == g_shards_type) {
        at::Tensor out;
        int rc;
        if (!shards_forward(obj.ptr(), x, out, &rc)) throw pybind11::error_already_set();
        if (rc == 0) return out;
    }
    pybind11::object fn = own(PyObject_GetAttr(g_core, s_forward)), h = own(PyLong_FromLongLong(handle)), xo = own(THPVariable_Wrap(x));
    pybind11::object y = own(PyObject_CallFunctionObjArgs(fn.ptr(), xo.ptr(), h.ptr(), nullptr));
    if (!THPVariable_Check(y.ptr())) throw std::runtime_error("shapequant::linear: forward did not return a tensor");
    return THPVariable_Unpack(y.ptr());
}

const c10::TypedOperatorHandle<at::Tensor(const at::Tensor&, int64_t)>& linear_handle() {
    static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow("shapequant::linear", "").typed<at::Tensor(const at::Tensor&, int64_t)>();
    return h;
}

// inference only: the forward runs on inputs that require a gradient, its backward raises
struct NoBackward : torch::autograd::Function<NoBackward> {
    static at::Tensor forward(torch::autograd::AutogradContext*, const at::Tensor& x, int64_t handle) {
        at::AutoDispatchBelowADInplaceOrView below;
        return linear_handle().call(x, handle);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
        C10_THROW_ERROR(NotImplementedError, "shapequant::linear has no autograd formula");
    }
};

at::Tensor linear_autograd(const at::Tensor& x, int64_t handle) {
    if (at::GradMode::is_enabled() && x.requires_grad()) return NoBackward::apply(x, handle);
    at::AutoDispatchBelowADInplaceOrView below;
    return linear_handle().call(x, handle);
}

// install(bufs): where the workspaces are;  install_op(core module, registry, PackedShards)
PyObject* install(PyObject*, PyObject* bufs) {
    Py_INCREF(bufs);
    Py_XDECREF(g_bufs);
    g_bufs = bufs;
    Py_RETURN_NONE;
}
PyObject* install_op(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 3 || !PyType_Check(a[2])) { PyErr_SetString(PyExc_TypeError, "install_op(core, registry, shards type)"); return nullptr; }
    for (int i = 0; i < 3; ++i) Py_INCREF(a[i]);
    g_core = a[0];
    g_registry = a[1];
    g_shards_type = reinterpret_cast<PyTypeObject*>(a[2]);
    Py_RETURN_NONE;
}

#define SQ_FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"native", (PyCFunction)(void (*)(void))make_native, METH_FASTCALL, nullptr}, {"install", install, METH_O, nullptr}, SQ_FAST(install_op),
                         SQ_FAST(linear), SQ_FAST(forward), SQ_FAST(linear_from), SQ_FAST(linear_silu), SQ_FAST(addnorm), SQ_FAST(silu_mul), SQ_FAST(q8_linear), SQ_FAST(q4_rows),
                         SQ_FAST(rotary), SQ_FAST(qk_norm_rotary), SQ_FAST(tree_attention), SQ_FAST(keep_drafted),
                         SQ_FAST(put_tokens8), SQ_FAST(tree_attention8), SQ_FAST(keep_drafted8), SQ_FAST(fork_pages), SQ_FAST(compact_pages),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods};

}  // namespace

TORCH_LIBRARY_IMPL(shapequant, CUDA, m) { m.impl("linear", linear_op); }
TORCH_LIBRARY_IMPL(shapequant, AutogradCUDA, m) { m.impl("linear", linear_autograd); }

PyMODINIT_FUNC PyInit__native() {
    NativeType.tp_name = "quantexperiments_amd._native.Native";
    NativeType.tp_basicsize = sizeof(Native);
    NativeType.tp_flags = Py_TPFLAGS_DEFAULT;
    NativeType.tp_dealloc = native_dealloc;
    if (PyType_Ready(&NativeType) < 0) return nullptr;
    struct { PyObject** at; const char* s; } names[] = {{&s_native, "_native"}, {&s_make_native, "_make_native"}, {&s_rls, "rls"}, {&s_cross, "cross"},
        {&s_large, "large"}, {&s_dequant_from, "dequant_from"}, {&s_enabled, "enabled"}, {&s_forward, "_linear_in_python"}, {&s_trace, "_trace"},
        {&s_fused, "fused"}};
    for (auto& nm : names) if (!(*nm.at = PyUnicode_InternFromString(nm.s))) return nullptr;
    return PyModule_Create(&module_def);
}
