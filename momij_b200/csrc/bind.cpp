// bind.cpp -- Python entry of the operators in attn.py and head.py: argument
// checks, output allocation and the call into libmomij_moe.so's C ABI, in one
// native step.  (Through ctypes a call of these thirty-argument functions, its
// checks and its output cost 10 to 13 us of host time, several times what the
// kernels take for a single token; this way about 4.)
//
// The library's functions are handed over as addresses (bind), so that this
// module uses the copy of the library that the process has loaded.  C++
// exceptions end at each function's edge as Python errors.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <stdexcept>
#include <string>

#include "momij_moe.h"

namespace {

using at::Tensor;

struct Functions {
    decltype(&momij_qk_norm_rope_append) append;
    decltype(&momij_cache_read) read;
    decltype(&momij_attention) attention;
    decltype(&momij_qmm4) qmm4;
    decltype(&momij_process_logits) logits;
} F;
PyObject* g_fail = nullptr;  // Python callable (status, where) that raises

struct TypeErr : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct ValueErr : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void value(bool ok, const char* what) {
    if (!ok) throw ValueErr(what);
}
void type(bool ok, const char* what) {
    if (!ok) throw TypeErr(what);
}

// ---- arguments -------------------------------------------------------------------
const Tensor* opt(PyObject* o, const char* name) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) throw TypeErr(std::string(name) + " is a tensor");
    return &THPVariable_Unpack(o);
}
// A workspace's bytes lie together: a strided or expanded tensor has others between, or fewer.
const Tensor* workspace(PyObject* o) {
    const Tensor* t = opt(o, "workspace");
    value(!t || t->is_contiguous(), "a workspace is a contiguous tensor");
    return t;
}
const Tensor& need(PyObject* o, const char* name) {
    const Tensor* t = opt(o, name);
    if (!t) throw TypeErr(std::string(name) + " is a tensor");
    return *t;
}
long long integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
int int32(PyObject* o, const char* name) {
    const long long v = integer(o);
    if (v < -2147483647LL || v > 2147483647LL) throw ValueErr(std::string(name) + " is out of range");
    return (int)v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
int dim32(int64_t n) {
    value(n <= 2147483647LL, "a size does not fit 32 bits");
    return (int)n;
}
void* ptr(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

int half_code(const Tensor& t) {
    if (t.scalar_type() == at::kBFloat16) return MOMIJ_DTYPE_BF16;
    if (t.scalar_type() == at::kHalf) return MOMIJ_DTYPE_F16;
    throw TypeErr("activations must be bf16 or fp16");
}
// All tensors on the current device.
int on_current(std::initializer_list<const Tensor*> ts) {
    const int cur = c10::cuda::current_device();
    for (const Tensor* t : ts)
        if (t && !(t->is_cuda() && t->get_device() == cur))
            throw ValueErr("tensors must lie on the current CUDA device");
    return cur;
}
// Calls go to the current stream, as their outputs' memory does.
momij_stream_t stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }
const int32_t* ints(const Tensor* t, const char* name, int64_t n) {
    if (!t) return nullptr;
    if (t->scalar_type() != at::kInt) throw TypeErr(std::string(name) + " is int32");
    if (t->dim() != 1 || t->size(0) != n || !t->is_contiguous())
        throw ValueErr(std::string(name) + " is a contiguous vector of " + std::to_string(n));
    return t->const_data_ptr<int32_t>();
}
const float* floats(const Tensor* t, const char* name, int64_t n) {
    if (!t) return nullptr;
    if (t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != n || !t->is_contiguous())
        throw ValueErr(std::string(name) + " is a contiguous float32 vector of " + std::to_string(n));
    return t->const_data_ptr<float>();
}
Tensor empty(at::IntArrayRef sizes, at::ScalarType dt, int dev) {
    return at::detail::empty_cuda(sizes, dt, at::Device(at::kCUDA, (c10::DeviceIndex)dev), std::nullopt);
}

struct Cache {
    const Tensor *k, *v, *ks, *vs;
    int pages, Hkv, D;
};
Cache cache_of(PyObject* const* o) {
    Cache c{&need(o[0], "k"), &need(o[1], "v"), &need(o[2], "k_scale"), &need(o[3], "v_scale"), 0, 0, 0};
    type(c.k->scalar_type() == at::kByte && c.v->scalar_type() == at::kByte, "codes are uint8");
    type(c.ks->scalar_type() == at::kFloat && c.vs->scalar_type() == at::kFloat, "scales are float32");
    value(c.k->dim() == 4 && c.v->dim() == 4 && c.ks->dim() == 2 && c.vs->dim() == 2, "k is [pages, Hkv, 64, D], scales [pages, Hkv]");
    const int64_t P = c.k->size(0), H = c.k->size(1), D = c.k->size(3);
    value(c.k->size(2) == MOMIJ_KV_PAGE && c.v->size(0) == P && c.v->size(1) == H && c.v->size(2) == D && c.v->size(3) == MOMIJ_KV_PAGE,
          "k is [pages, Hkv, 64, D] and v [pages, Hkv, D, 64]");
    value(c.ks->size(0) == P && c.ks->size(1) == H && c.vs->size(0) == P && c.vs->size(1) == H, "scales are [pages, Hkv]");
    value(c.k->is_contiguous() && c.v->is_contiguous() && c.ks->is_contiguous() && c.vs->is_contiguous(),
          "cache tensors must be contiguous");
    c.pages = dim32(P);
    c.Hkv = dim32(H);
    c.D = dim32(D);
    return c;
}
const int32_t* table_of(const Tensor& t, int64_t B) {
    type(t.scalar_type() == at::kInt, "block_table is int32");
    value(t.dim() == 2 && t.size(0) == B && t.is_contiguous(), "block_table is a contiguous [B, columns] tensor");
    return t.const_data_ptr<int32_t>();
}

// Runs one entry: `body` returns a new reference or throws.
template <typename Fn>
PyObject* guarded(Fn&& body) {
    try {
        return body();
    } catch (const TypeErr& e) {
        PyErr_SetString(PyExc_TypeError, e.what());
    } catch (const ValueErr& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (python_error& e) {
        e.restore();
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}
void check(int rc, const char* where) {
    if (rc == MOMIJ_OK) return;
    PyObject* r = PyObject_CallFunction(g_fail, "is", rc, where);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) throw std::runtime_error(std::string(where) + " failed");
    throw python_error();
}
void count(Py_ssize_t n, Py_ssize_t want) { type(n == want, "wrong number of arguments"); }

// ---- entries ---------------------------------------------------------------------
// (qkv, k, v, ks, vs, block_table, lens, n_heads, q_weight, k_weight, eps, rope, interleaved, cu_q, max_q, q_out, workspace)
PyObject* append(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 17);
        const Tensor& qkv = need(o[0], "qkv");
        const Cache c = cache_of(o + 1);
        const Tensor &table = need(o[5], "block_table"), &lens = need(o[6], "lens");
        const int Hq = int32(o[7], "n_heads");
        const Tensor *qw = opt(o[8], "q_weight"), *kw = opt(o[9], "k_weight"), *rope = opt(o[11], "rope"), *cu = opt(o[13], "cu_q"),
                     *given = opt(o[15], "q_out"), *ws = workspace(o[16]);
        const int dev = on_current({&qkv, c.k, c.v, c.ks, c.vs, &table, &lens, qw, kw, rope, cu, given, ws});
        const int dt = half_code(qkv);
        value(qkv.dim() == 2 && lens.dim() == 1, "qkv is [T, (Hq + 2 Hkv) D] and lens [B]");
        const int64_t T = qkv.size(0), width = qkv.size(1), B = lens.size(0);
        value(Hq >= 1 && width == ((int64_t)Hq + 2 * c.Hkv) * c.D && qkv.stride(1) == 1 && (T <= 1 || qkv.stride(0) >= width),
              "qkv is [T, (Hq + 2 Hkv) D] with contiguous rows");
        for (const Tensor* w : {qw, kw})
            value(!w || (w->scalar_type() == qkv.scalar_type() && w->dim() == 1 && w->size(0) == c.D && w->is_contiguous()),
                  "norm weights are contiguous [D] of the activations' dtype");
        value(!rope || (rope->scalar_type() == at::kFloat && rope->dim() == 2 && rope->is_contiguous()),
              "rope is a contiguous float32 [positions, rot] table");
        Tensor q;
        if (given) {
            q = *given;
            value(q.dim() == 3 && q.size(0) == T && q.size(1) == Hq && q.size(2) == c.D && q.scalar_type() == qkv.scalar_type() &&
                      q.is_contiguous(),
                  "q_out is a contiguous [T, Hq, D] tensor of the activations' dtype");
        } else {
            q = empty({T, Hq, c.D}, qkv.scalar_type(), dev);
        }
        check(F.append(qkv.data_ptr(), T > 1 ? qkv.stride(0) : width, q.data_ptr(), ptr(qw), ptr(kw), (float)real(o[10]),
                       rope ? rope->const_data_ptr<float>() : nullptr, rope ? dim32(rope->size(0)) : 0, rope ? dim32(rope->size(1)) : 0,
                       truth(o[12]), c.k->data_ptr<uint8_t>(), c.v->data_ptr<uint8_t>(), c.ks->data_ptr<float>(),
                       c.vs->data_ptr<float>(), c.pages, table_of(table, B), dim32(table.size(1)), ints(&lens, "lens", B),
                       ints(cu, "cu_q", B + 1), dim32(T), dim32(B), int32(o[14], "max_q"), Hq, c.Hkv, c.D, dt, ptr(ws),
                       ws ? ws->nbytes() : 0, stream_of(dev)),
              "qkNormRopeAppend");
        return THPVariable_Wrap(std::move(q));
    });
}

// (k, v, ks, vs, block_table, lens, first, count, f16, workspace)
PyObject* read(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 10);
        const Cache c = cache_of(o);
        const Tensor &table = need(o[4], "block_table"), &lens = need(o[5], "lens");
        const Tensor *first = opt(o[6], "first"), *ws = workspace(o[9]);
        const int dev = on_current({c.k, c.v, c.ks, c.vs, &table, &lens, first, ws});
        const int cnt = int32(o[7], "count"), f16 = truth(o[8]);
        value(lens.dim() == 1 && cnt >= 0, "lens is [B], count not negative");
        const int64_t B = lens.size(0);
        const at::ScalarType dt = f16 ? at::kHalf : at::kBFloat16;
        Tensor k = empty({B, cnt, c.Hkv, c.D}, dt, dev), v = empty({B, cnt, c.Hkv, c.D}, dt, dev);
        check(F.read(c.k->data_ptr<uint8_t>(), c.v->data_ptr<uint8_t>(), c.ks->data_ptr<float>(), c.vs->data_ptr<float>(), c.pages,
                     table_of(table, B), dim32(table.size(1)), ints(&lens, "lens", B), ints(first, "first", B), cnt, k.data_ptr(),
                     v.data_ptr(), dim32(B), c.Hkv, c.D, f16 ? MOMIJ_DTYPE_F16 : MOMIJ_DTYPE_BF16, ptr(ws), ws ? ws->nbytes() : 0,
                     stream_of(dev)),
              "cacheRead");
        PyObject* kp = THPVariable_Wrap(std::move(k));
        PyObject* vp = THPVariable_Wrap(std::move(v));
        if (!kp || !vp) {
            Py_XDECREF(kp);
            Py_XDECREF(vp);
            throw python_error();
        }
        return Py_BuildValue("(NN)", kp, vp);
    });
}

// (q, k, v, ks, vs, block_table, lens, scale or None, window, cu_q, max_q, out, workspace)
PyObject* attention(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 13);
        const Tensor& q = need(o[0], "q");
        const Cache c = cache_of(o + 1);
        const Tensor &table = need(o[5], "block_table"), &lens = need(o[6], "lens");
        const Tensor *cu = opt(o[9], "cu_q"), *given = opt(o[11], "out"), *wsp = workspace(o[12]);
        type(wsp != nullptr, "workspace is a tensor");
        const Tensor& ws = *wsp;
        const int dev = on_current({&q, c.k, c.v, c.ks, c.vs, &table, &lens, cu, given, &ws});
        const int dt = half_code(q);
        value(q.dim() == 3 && lens.dim() == 1, "q is [T, Hq, D] and lens [B]");
        const int64_t T = q.size(0), Hq = q.size(1), B = lens.size(0);
        auto rows = [&](const Tensor& t) {
            return t.dim() == 3 && t.size(0) == T && t.size(1) == Hq && t.size(2) == c.D && t.stride(2) == 1 && (Hq <= 1 || t.stride(1) == c.D);
        };
        value(rows(q), "q is [T, Hq, D] with contiguous rows");
        Tensor out;
        if (given) {
            out = *given;
            value(rows(out) && out.scalar_type() == q.scalar_type(), "out is [T, Hq, D] of q's dtype with contiguous rows");
        } else {
            out = empty({T, Hq, c.D}, q.scalar_type(), dev);
        }
        const double scale = o[7] == Py_None ? (c.D == 64 ? 0.125 : 0.08838834764831845) : real(o[7]);
        check(F.attention(q.data_ptr(), T > 1 ? q.stride(0) : Hq * c.D, out.data_ptr(), T > 1 ? out.stride(0) : Hq * c.D,
                          c.k->data_ptr<uint8_t>(), c.v->data_ptr<uint8_t>(), c.ks->data_ptr<float>(), c.vs->data_ptr<float>(), c.pages,
                          table_of(table, B), dim32(table.size(1)), ints(&lens, "lens", B), ints(cu, "cu_q", B + 1), dim32(T), dim32(B),
                          int32(o[10], "max_q"), dim32(Hq), c.Hkv, c.D, (float)scale, int32(o[8], "window"), dt, ws.data_ptr(), ws.nbytes(),
                          stream_of(dev)),
              "attention");
        return THPVariable_Wrap(std::move(out));
    });
}

// (x, w, scales, biases, gs, out)
PyObject* qmm4(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 6);
        const Tensor &x = need(o[0], "x"), &w = need(o[1], "w"), &s = need(o[2], "scales"), &b = need(o[3], "biases");
        const Tensor* given = opt(o[5], "out");
        const int dev = on_current({&x, &w, &s, &b, given});
        const int gs = int32(o[4], "gs"), dt = half_code(x);
        type(s.scalar_type() == x.scalar_type() && b.scalar_type() == x.scalar_type(), "scales and biases have the activations' dtype");
        type(w.scalar_type() == at::kInt || w.scalar_type() == at::kUInt32, "codes are packed in 32-bit words");
        value(x.dim() == 2 && w.dim() == 2 && s.dim() == 2 && b.dim() == 2 && gs > 0, "x, w, scales and biases are matrices");
        const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
        value(K <= 1 || x.stride(1) == 1, "rows of x must be contiguous");
        value(w.size(1) == K / 8 && s.size(0) == N && s.size(1) == K / gs && b.sizes() == s.sizes() && w.is_contiguous() &&
                  s.is_contiguous() && b.is_contiguous(),
              "w is [N, K/8], scales and biases [N, K/gs], contiguous");
        Tensor y;
        if (given) {
            y = *given;
            value(y.dim() == 2 && y.size(0) == M && y.size(1) == N && y.scalar_type() == x.scalar_type() && (N <= 1 || y.stride(1) == 1),
                  "out is [M, N] of the activations' dtype with contiguous rows");
        } else {
            y = empty({M, N}, x.scalar_type(), dev);
        }
        check(F.qmm4(x.data_ptr(), M > 1 ? x.stride(0) : K, static_cast<const uint32_t*>(w.data_ptr()), s.data_ptr(), b.data_ptr(),
                     y.data_ptr(), M > 1 ? y.stride(0) : N, dim32(M), dim32(K), dim32(N), gs, dt, stream_of(dev)),
              "qmm4");
        return THPVariable_Wrap(std::move(y));
    });
}

// (logits, history, cu_history, repetition, presence, frequency, bias_ids, bias, cu_bias, allowed, out)
PyObject* logits(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 11);
        const Tensor& l = need(o[0], "logits");
        const Tensor *h = opt(o[1], "history"), *ch = opt(o[2], "cu_history"), *rep = opt(o[3], "repetition"), *pres = opt(o[4], "presence"),
                     *freq = opt(o[5], "frequency"), *bi = opt(o[6], "bias_ids"), *bv = opt(o[7], "bias"), *cb = opt(o[8], "cu_bias"),
                     *al = opt(o[9], "allowed"), *given = opt(o[10], "out");
        const int dev = on_current({&l, h, ch, rep, pres, freq, bi, bv, cb, al, given});
        int dt;
        if (l.scalar_type() == at::kFloat) dt = MOMIJ_DTYPE_F32;
        else if (l.scalar_type() == at::kBFloat16) dt = MOMIJ_DTYPE_BF16;
        else if (l.scalar_type() == at::kHalf) dt = MOMIJ_DTYPE_F16;
        else throw TypeErr("logits are bf16, fp16 or fp32");
        value(l.dim() == 2, "logits are [B, V]");
        const int64_t B = l.size(0), V = l.size(1);
        value(V <= 1 || l.stride(1) == 1, "rows of the logits must be contiguous");
        value(!h == !ch, "history and cu_history go together");
        value(!bi == !cb && !bi == !bv, "bias_ids, bias and cu_bias go together");
        value(!al || (al->scalar_type() == at::kInt && al->dim() == 2 && al->size(0) == B && al->size(1) == (V + 31) / 32 &&
                      (al->size(1) <= 1 || al->stride(1) == 1)),
              "allowed is int32 [B, ceil(V/32)] with contiguous rows");
        const int64_t nh = h ? h->numel() : 0, nb = bi ? bi->numel() : 0;
        Tensor out;
        if (given) {
            out = *given;
            value(out.dim() == 2 && out.size(0) == B && out.size(1) == V && out.scalar_type() == at::kFloat && out.is_contiguous(),
                  "out is a contiguous float32 [B, V] tensor");
        } else {
            out = empty({B, V}, at::kFloat, dev);
        }
        check(F.logits(l.data_ptr(), B > 1 ? l.stride(0) : V, dt, out.data_ptr<float>(), dim32(B), dim32(V), ints(h, "history", nh),
                       ints(ch, "cu_history", B + 1), dim32(nh), floats(rep, "repetition", B), floats(pres, "presence", B),
                       floats(freq, "frequency", B), ints(bi, "bias_ids", nb), floats(bv, "bias", nb), ints(cb, "cu_bias", B + 1), dim32(nb),
                       al ? reinterpret_cast<const uint32_t*>(al->const_data_ptr<int32_t>()) : nullptr,
                       al ? (B > 1 ? al->stride(0) : al->size(1)) : 0, stream_of(dev)),
              "processLogits");
        return THPVariable_Wrap(std::move(out));
    });
}

// bind(fail, append, read, attention, qmm4, process_logits): a callable and function addresses
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 6);
        auto at = [&](int i) { return static_cast<uintptr_t>(integer(o[i])); };
        F.append = reinterpret_cast<decltype(F.append)>(at(1));
        F.read = reinterpret_cast<decltype(F.read)>(at(2));
        F.attention = reinterpret_cast<decltype(F.attention)>(at(3));
        F.qmm4 = reinterpret_cast<decltype(F.qmm4)>(at(4));
        F.logits = reinterpret_cast<decltype(F.logits)>(at(5));
        Py_INCREF(o[0]);
        Py_XDECREF(g_fail);
        g_fail = o[0];
        Py_RETURN_NONE;
    });
}

PyMethodDef methods[] = {{"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
                         {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
                         {"read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(read)), METH_FASTCALL, nullptr},
                         {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL, nullptr},
                         {"qmm4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(qmm4)), METH_FASTCALL, nullptr},
                         {"logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(logits)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_momij_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__momij_ops() { return PyModule_Create(&module); }
