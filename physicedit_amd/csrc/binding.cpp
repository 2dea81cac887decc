// Python binding of the low-bit decode step's operators: what physicedit_amd/ops.py's functions of the same names do between the caller's tensors and the
// C entry points (include/physicedit_amd.h).  These operators take 2 to 20 us on the device and are called once per token and layer; reading a
// dozen tensor attributes and filling a struct costs 4 to 8 us in Python and less than one here.  Checks, allocation of results and
// workspaces, the launch on the current stream: nothing is computed and nothing is kept between calls.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <stdarg.h>

#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/physicedit_amd.h"

namespace {

struct Api {
    decltype(&pe_last_error) last_error;
    decltype(&pe_gemv_w4) gemv_w4;
    decltype(&pe_kv_append_e4m3) kv_append_e4m3;
    decltype(&pe_kv_attention_workspace_bytes) kv_attention_workspace_bytes;
    decltype(&pe_kv_attention_e4m3) kv_attention_e4m3;
    decltype(&pe_process_logits) process_logits;
    decltype(&pe_select_token_workspace_bytes) select_token_workspace_bytes;
    decltype(&pe_select_token) select_token;
    decltype(&pe_token_counts_add) token_counts_add;
} api;
PyObject *get_device, *raw_stream, *pe_error, *oom_error;      // torch's two functions and two exception types, held for good

// an error to raise: ValueError for arguments that do not fit, PeError for what the library refuses, Python's own where one is set
struct Raise { PyObject* type; std::string text; };
[[noreturn]] void bad(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
[[noreturn]] void bad(const char* fmt, ...) {
    char text[640];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    throw Raise{PyExc_ValueError, text};
}

std::string show(at::IntArrayRef s) {
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + ")";
}
std::string show(const at::Tensor& t) { return std::string(c10::toString(t.scalar_type())) + " " + show(t.sizes()) + " on " + t.device().str(); }

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) bad("%s: expected a tensor, got %s", name, Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
bool on(const at::Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }

long call_long(PyObject* f, PyObject* arg) {
    PyObject* r = arg ? PyObject_CallOneArg(f, arg) : PyObject_CallNoArgs(f);
    if (!r) throw Raise{nullptr, ""};
    const long long v = PyLong_AsLongLong(r);
    Py_DECREF(r);
    if (v == -1 && PyErr_Occurred()) throw Raise{nullptr, ""};
    return (long)v;
}
// the current stream of device `dev`, which has to be the current device
void* stream_of(long dev, const char* name) {
    if (dev < 0) bad("%s: expected a CUDA/HIP tensor (physicedit_amd has no CPU path)", name);
    const long cur = call_long(get_device, nullptr);
    if (dev != cur) bad("%s: on cuda:%ld, but the current device is cuda:%ld (torch.cuda.device(...))", name, dev, cur);
    PyObject* d = PyLong_FromLong(dev);
    if (!d) throw Raise{nullptr, ""};
    struct Free { PyObject* o; ~Free() { Py_DECREF(o); } } f{d};
    return (void*)(intptr_t)call_long(raw_stream, d);
}
long cuda_index(const at::Tensor& t) { return t.is_cuda() ? (long)t.get_device() : -1; }

// address of a contiguous tensor of exactly this type and shape on device `dev`; null for None
void* at_(PyObject* o, const char* name, at::ScalarType type, at::IntArrayRef shape, long dev) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != type || t.sizes() != shape || !t.is_contiguous() || !on(t, (int)dev))
        bad("%s: expected a contiguous %s tensor of shape %s on cuda:%ld, got %s", name, c10::toString(type), show(shape).c_str(), dev, show(t).c_str());
    return t.data_ptr();
}

// address and strides (batch, token, head) of a bf16 [batch, T, heads, D] tensor with contiguous channels and rows of whole 16 bytes; a dimension of one
// entry has any stride
void* heads_(const at::Tensor& t, const char* name, at::IntArrayRef shape, long dev, long long (&st)[3]) {
    if (t.scalar_type() != at::kBFloat16 || t.sizes() != shape || t.stride(3) != 1 || !on(t, (int)dev))
        bad("%s: expected bf16 %s with contiguous channels on cuda:%ld, got %s", name, show(shape).c_str(), dev, show(t).c_str());
    long long all = 0;
    for (int i = 0; i < 3; ++i) { st[i] = shape[i] == 1 ? 0 : t.stride(i); all |= st[i]; }
    void* p = t.data_ptr();
    if (((uintptr_t)p & 15) || (all & 7)) bad("%s: rows must be 16-byte aligned (strides %s)", name, show(t.strides()).c_str());
    return p;
}

// What a call writes for the caller (`result`: out, a workspace, counts) lies apart from input `in` -- or, where `over` says that each of its elements is read before it is written, exactly over it.
// A dimension of strides counts with all that lies between its ends.
void apart(PyObject* result, PyObject* in, const char* name, bool over = false, const char* what = "out") {
    if (result == Py_None || in == Py_None) return;
    const at::Tensor &r = tensor(result, what), &t = tensor(in, name);
    int64_t span = 1;
    for (int64_t i = 0; i < t.dim(); ++i) span += (t.size(i) - 1) * t.stride(i);
    const char *r0 = (const char*)r.data_ptr(), *t0 = (const char*)t.data_ptr(), *r1 = r0 + r.nbytes(), *t1 = t0 + span * (int64_t)t.element_size();
    if (r1 <= t0 || t1 <= r0 || (over && r0 == t0 && t.is_contiguous() && t.nbytes() == r.nbytes())) return;
    bad("%s: overlaps %s%s", what, name, over ? " (it may only lie exactly over it)" : "");
}

const at::Tensor& four_dims(PyObject* o, const char* name, const char* what) {
    const at::Tensor& t = tensor(o, name);
    if (t.dim() != 4) bad("%s: expected %s, got %s", name, what, show(t).c_str());
    return t;
}
at::Tensor empty_like_type(const at::Tensor& t, at::IntArrayRef shape, at::ScalarType type) { return at::empty(shape, t.options().dtype(type).requires_grad(false)); }
PyObject* wrap_or(PyObject* given, at::Tensor& made) {
    if (given == Py_None) return THPVariable_Wrap(std::move(made));
    Py_INCREF(given);
    return given;
}
template <typename F>
void launch(const char* what, F&& f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    if (rc) throw Raise{pe_error, std::string(what) + " failed (rc=" + std::to_string(rc) + "): " + api.last_error()};
}
template <typename F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const Raise& e) {
        if (e.type) PyErr_SetString(e.type, e.text.c_str());
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(oom_error, e.what_without_backtrace());
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
bool count_ok(Py_ssize_t n, Py_ssize_t want, const char* name) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%s: %zd arguments, %zd given", name, want, n);
    return false;
}
template <typename T>
const T* record(PyObject* address) { return (const T*)PyLong_AsVoidPtr(address); }
long integer(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raise{nullptr, ""};
    return v;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raise{nullptr, ""};
    return v;
}

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raise{nullptr, ""};
    return v == 1;
}

// gemv_w4(x, address of the pe_w4_weight, its device, bias, res, swiglu, norm_eps, out)
PyObject* gemv_w4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count_ok(n, 8, "gemv_w4")) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& x = tensor(a[0], "x");
        const pe_w4_weight* w = record<pe_w4_weight>(a[1]);
        const long dev = integer(a[2]);
        void* stream = stream_of(dev, "w");
        const bool swiglu = truth(a[5]);
        const int64_t dims = x.dim(), K = w->K, cols = swiglu ? w->N / 2 : w->N;
        if (x.scalar_type() != at::kBFloat16 || (dims != 1 && dims != 2) || x.size(-1) != K || x.stride(-1) != 1 || !on(x, (int)dev))
            bad("gemv_w4: expected bf16 rows of %lld contiguous values on cuda:%ld, got %s", (long long)K, dev, show(x).c_str());
        const int64_t M = dims == 1 ? 1 : x.size(0), two[2] = {M, cols};
        const at::IntArrayRef shape = dims == 1 ? at::IntArrayRef(&two[1], 1) : at::IntArrayRef(two, 2);
        const void *bias = at_(a[3], "bias", at::kBFloat16, {(int64_t)w->N}, dev), *res = at_(a[4], "res", at::kBFloat16, shape, dev);
        void* to = at_(a[7], "out", at::kBFloat16, shape, dev);
        if (M < 1 || M > 1 << 20) bad("gemv_w4: %lld rows", (long long)M);
        apart(a[7], a[3], "bias");
        apart(a[7], a[4], "res", true);
        if (to != x.data_ptr()) apart(a[7], a[0], "x");        // at x itself: the library's own refusal
        at::Tensor out;
        if (a[7] == Py_None) { out = empty_like_type(x, shape, at::kBFloat16); to = out.data_ptr(); }
        const float eps = (float)number(a[6]);
        launch("pe_gemv_w4", [&] { return api.gemv_w4(x.data_ptr(), M > 1 ? x.stride(0) : K, (int)M, w, bias, res, cols, to, cols, swiglu, eps, stream); });
        return wrap_or(a[7], out);
    });
}

// kv_append_e4m3(address of the pe_kv_cache, its device, k, v, start, q, cos, sin, positions, out)
PyObject* kv_append_e4m3(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count_ok(n, 10, "kv_append_e4m3")) return nullptr;
    return guarded([&]() -> PyObject* {
        const pe_kv_cache* c = record<pe_kv_cache>(a[0]);
        const long dev = integer(a[1]);
        void* stream = stream_of(dev, "cache");
        const at::Tensor &k = four_dims(a[2], "k", "[batch, T, n_kv, D]"), &v = four_dims(a[3], "v", "[batch, T, n_kv, D]");
        const int64_t B = c->batch, D = c->head_dim, T = k.size(1);
        if (T < 1 || T > INT32_MAX) bad("k: %lld tokens", (long long)T);
        pe_kv_append_args s = {};
        s.T = (int)T;
        s.k = heads_(k, "k", {B, T, c->n_kv, D}, dev, s.k_strides);
        s.v = heads_(v, "v", {B, T, c->n_kv, D}, dev, s.v_strides);
        s.start = (const int*)at_(a[4], "start", at::kInt, {B}, dev);
        if (!s.start) bad("start: expected a tensor");
        const bool has_q = a[5] != Py_None, tables = a[6] != Py_None;
        if (tables != (a[7] != Py_None) || (!tables && (has_q || a[8] != Py_None))) bad("kv_append_e4m3: q and positions need cos and sin, which come together");
        if (tables) {
            const at::Tensor& cos = tensor(a[6], "cos");
            if ((cos.scalar_type() != at::kBFloat16 && cos.scalar_type() != at::kFloat) || cos.dim() != 2 || cos.size(0) < 1 || cos.size(0) > INT32_MAX)
                bad("cos: expected bf16 or fp32 [rows, %lld], got %s", (long long)D, show(cos).c_str());
            s.table_rows = (int)cos.size(0);
            s.table_f32 = cos.scalar_type() == at::kFloat;
            s.cos = at_(a[6], "cos", cos.scalar_type(), {s.table_rows, D}, dev);
            s.sin = at_(a[7], "sin", cos.scalar_type(), {s.table_rows, D}, dev);
            s.positions = (const int*)at_(a[8], "positions", at::kInt, {B, T}, dev);
        }
        at::Tensor out;
        if (has_q) {
            const at::Tensor& q = four_dims(a[5], "q", "[batch, T, n_q, D]");
            const int64_t nq = q.size(2);
            s.n_q = (int)nq;
            s.q = heads_(q, "q", {B, T, nq, D}, dev, s.q_strides);
            s.q_out = at_(a[9], "out", at::kBFloat16, {B, T, nq, D}, dev);
            if (a[9] == Py_None) { out = empty_like_type(q, {B, T, nq, D}, at::kBFloat16); s.q_out = out.data_ptr(); }
            apart(a[9], a[5], "q", true);
            apart(a[9], a[2], "k");
            apart(a[9], a[3], "v");
            apart(a[9], a[6], "cos");
            apart(a[9], a[7], "sin");
            apart(a[9], a[4], "start");
            apart(a[9], a[8], "positions");
        }
        launch("pe_kv_append_e4m3", [&] { return api.kv_append_e4m3(c, &s, stream); });
        if (!has_q) Py_RETURN_NONE;
        return wrap_or(a[9], out);
    });
}

// kv_attention_e4m3(q, address of the pe_kv_cache, its device, start, tree, scale or None, out, workspace)
PyObject* kv_attention_e4m3(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count_ok(n, 8, "kv_attention_e4m3")) return nullptr;
    return guarded([&]() -> PyObject* {
        const pe_kv_cache* c = record<pe_kv_cache>(a[1]);
        const long dev = integer(a[2]);
        void* stream = stream_of(dev, "cache");
        const at::Tensor& q = four_dims(a[0], "q", "[batch, T, n_q, D]");
        const int64_t B = c->batch, D = c->head_dim, T = q.size(1), nq = q.size(2);
        long long st[3];
        void* qa = heads_(q, "q", {B, T, nq, D}, dev, st);
        if (T < 1 || T > 64 || nq < 1 || nq % c->n_kv) bad("kv_attention_e4m3: %lld new tokens (1 ... 64), %lld query heads over %d kv heads", (long long)T, (long long)nq, c->n_kv);
        const int* start = (const int*)at_(a[3], "start", at::kInt, {B}, dev);
        if (!start) bad("start: expected a tensor");
        const void* tree = at_(a[4], "tree", at::kLong, {B, T}, dev);
        const float scale = a[5] == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)number(a[5]);
        void* to = at_(a[6], "out", at::kBFloat16, {B, T, nq * D}, dev);
        apart(a[6], a[0], "q", true);
        apart(a[6], a[3], "start");
        apart(a[6], a[4], "tree");
        apart(a[7], a[6], "out", false, "workspace");
        apart(a[7], a[0], "q", false, "workspace");
        apart(a[7], a[3], "start", false, "workspace");
        apart(a[7], a[4], "tree", false, "workspace");
        at::Tensor out, ws;
        if (a[6] == Py_None) { out = empty_like_type(q, {B, T, nq * D}, at::kBFloat16); to = out.data_ptr(); }
        void* wp = nullptr;
        size_t wn = 0;
        if (a[7] == Py_None) {
            wn = api.kv_attention_workspace_bytes((int)B, c->n_kv, (int)T, (int)nq, (int)D, c->capacity);
            if (wn) { ws = empty_like_type(q, {(int64_t)wn}, at::kByte); wp = ws.data_ptr(); }
        } else {
            const at::Tensor& t = tensor(a[7], "workspace");
            if (!on(t, (int)dev) || !t.is_contiguous()) bad("workspace: expected a contiguous tensor on cuda:%ld", dev);
            wp = t.data_ptr();
            wn = t.nbytes();
        }
        launch("pe_kv_attention_e4m3", [&] { return api.kv_attention_e4m3(c, qa, st, start, tree, (int)T, (int)nq, scale, to, wp, wn, stream); });
        return wrap_or(a[6], out);
    });
}

// a table that is there once ([n], row stride 0) or for every row ([R, n])
void* table(PyObject* o, const char* name, at::ScalarType type, int64_t R, int64_t n, long dev, long long& ld) {
    ld = 0;
    if (o == Py_None) return nullptr;
    if (tensor(o, name).dim() == 1) return at_(o, name, type, {n}, dev);
    ld = n;
    return at_(o, name, type, {R, n}, dev);
}
pe_logits_args logits_args(PyObject* const* a, long& dev, void*& stream) {
    const at::Tensor& x = tensor(a[0], "logits");
    dev = cuda_index(x);
    stream = stream_of(dev, "logits");
    const bool f32 = x.scalar_type() == at::kFloat;
    if ((!f32 && x.scalar_type() != at::kBFloat16) || x.dim() != 2 || x.numel() == 0 || (x.size(1) > 1 && x.stride(1) != 1) || x.size(0) > INT32_MAX || x.size(1) > INT32_MAX)
        bad("logits: expected bf16 or fp32 [rows, vocab] with contiguous rows, got %s", show(x).c_str());
    if (a[2] != Py_None && a[1] == Py_None) bad("penalties: they need the counts");
    const int64_t R = x.size(0), V = x.size(1);
    pe_logits_args s = {};
    s.logits = x.data_ptr(); s.ld = R > 1 ? x.stride(0) : V; s.f32 = f32; s.rows = (int)R; s.vocab = (int)V;
    s.counts = at_(a[1], "counts", at::kShort, {R, V}, dev);
    s.ld_counts = V;
    s.penalties = (const float*)table(a[2], "penalties", at::kFloat, R, 3, dev, s.ld_penalties);
    s.bias = (const float*)table(a[3], "bias", at::kFloat, R, V, dev, s.ld_bias);
    s.allowed = table(a[4], "allowed", at::kInt, R, (V + 31) / 32, dev, s.ld_allowed);
    return s;
}

// process_logits(logits, counts, penalties, bias, allowed, out)
PyObject* process_logits(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count_ok(n, 6, "process_logits")) return nullptr;
    return guarded([&]() -> PyObject* {
        long dev;
        void* stream;
        const pe_logits_args s = logits_args(a, dev, stream);
        void* to = at_(a[5], "out", at::kFloat, {s.rows, s.vocab}, dev);
        at::Tensor out;
        if (a[5] == Py_None) { out = empty_like_type(tensor(a[0], "logits"), {s.rows, s.vocab}, at::kFloat); to = out.data_ptr(); }
        apart(a[5], a[0], "logits", true);
        apart(a[5], a[1], "counts");
        apart(a[5], a[2], "penalties");
        apart(a[5], a[3], "bias", true);
        apart(a[5], a[4], "allowed");
        launch("pe_process_logits", [&] { return api.process_logits(&s, (float*)to, stream); });
        return wrap_or(a[5], out);
    });
}

// select_token(logits, counts, penalties, bias, allowed, update_counts, out, out_ids, step, workspace)
PyObject* select_token(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count_ok(n, 10, "select_token")) return nullptr;
    return guarded([&]() -> PyObject* {
        long dev;
        void* stream;
        const pe_logits_args s = logits_args(a, dev, stream);
        const at::Tensor& x = tensor(a[0], "logits");
        const bool update = truth(a[5]);
        if (update && !s.counts) bad("select_token: update_counts without counts");
        int* to = (int*)at_(a[6], "out", at::kInt, {s.rows}, dev);
        int *ids = nullptr, *step = nullptr;
        int64_t room = 0;
        if (a[7] != Py_None || a[8] != Py_None) {
            if (a[7] == Py_None || a[8] == Py_None || s.rows != 1 || tensor(a[8], "step").numel() != 1 || tensor(a[7], "out_ids").dim() != 1 || tensor(a[7], "out_ids").numel() < 1)
                bad("select_token: step and out_ids come together, for one row");
            room = tensor(a[7], "out_ids").numel();
            ids = (int*)at_(a[7], "out_ids", at::kInt, {room}, dev);
            step = (int*)at_(a[8], "step", at::kInt, tensor(a[8], "step").sizes(), dev);
        }
        for (int i = 0; i < 5; ++i) {
            static const char* const names[5] = {"logits", "counts", "penalties", "bias", "allowed"};
            apart(a[6], a[i], names[i]);
            apart(a[7], a[i], names[i]);
            apart(a[8], a[i], names[i]);
            apart(a[9], a[i], names[i], false, "workspace");
        }
        for (int i = 6; i < 9; ++i) apart(a[9], a[i], i == 6 ? "out" : i == 7 ? "out_ids" : "step", false, "workspace");
        apart(a[6], a[7], "out_ids");
        apart(a[6], a[8], "step");
        apart(a[7], a[8], "step");
        at::Tensor out, ws;
        if (!to) { out = empty_like_type(x, {s.rows}, at::kInt); to = (int*)out.data_ptr(); }
        void* wp = nullptr;
        size_t wn = 0;
        if (a[9] == Py_None) {
            wn = api.select_token_workspace_bytes(s.rows, s.vocab);
            if (wn) { ws = empty_like_type(x, {(int64_t)wn}, at::kByte); wp = ws.data_ptr(); }
        } else {
            const at::Tensor& t = tensor(a[9], "workspace");
            if (!on(t, (int)dev) || !t.is_contiguous()) bad("workspace: expected a contiguous tensor on cuda:%ld", dev);
            wp = t.data_ptr();
            wn = t.nbytes();
        }
        launch("pe_select_token", [&] { return api.select_token(&s, to, update, ids, step, (int)std::min<int64_t>(room, INT32_MAX), wp, wn, stream); });
        return wrap_or(a[6], out);
    });
}

// token_counts_add(counts, tokens, prompt)
PyObject* token_counts_add(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count_ok(n, 3, "token_counts_add")) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &c = tensor(a[0], "counts"), &t = tensor(a[1], "tokens");
        const long dev = cuda_index(c);
        void* stream = stream_of(dev, "counts");
        if (c.dim() != 2 || c.numel() == 0 || t.dim() != 2 || t.size(1) < 1 || c.size(0) > INT32_MAX || c.size(1) > INT32_MAX || t.size(1) > INT32_MAX)
            bad("token_counts_add: counts [rows, vocab] and tokens [rows, n], got %s and %s", show(c).c_str(), show(t).c_str());
        const int64_t R = c.size(0), V = c.size(1), m = t.size(1);
        void* cp = at_(a[0], "counts", at::kShort, {R, V}, dev);
        const int* tp = (const int*)at_(a[1], "tokens", at::kInt, {R, m}, dev);
        apart(a[0], a[1], "tokens", false, "counts");
        const bool prompt = truth(a[2]);
        launch("pe_token_counts_add", [&] { return api.token_counts_add(cp, V, (int)R, (int)V, tp, (int)m, prompt, stream); });
        Py_INCREF(a[0]);
        return a[0];
    });
}

// bind(addresses of the Api's functions, torch's device and raw-stream functions, PeError, OutOfMemoryError)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count_ok(n, 5, "bind")) return nullptr;
    void** to = (void**)&api;
    constexpr Py_ssize_t count = sizeof(Api) / sizeof(void*);
    if (!PyTuple_Check(a[0]) || PyTuple_GET_SIZE(a[0]) != count) {
        PyErr_Format(PyExc_TypeError, "bind: %zd addresses", count);
        return nullptr;
    }
    for (Py_ssize_t i = 0; i < count; ++i) {
        to[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(a[0], i));
        if (!to[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null address");
            return nullptr;
        }
    }
    PyObject** keep[4] = {&get_device, &raw_stream, &pe_error, &oom_error};
    for (int i = 0; i < 4; ++i) { Py_INCREF(a[i + 1]); Py_XSETREF(*keep[i], a[i + 1]); }
    Py_RETURN_NONE;
}

#define PE_METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {PE_METHOD(bind), PE_METHOD(gemv_w4), PE_METHOD(kv_append_e4m3), PE_METHOD(kv_attention_e4m3), PE_METHOD(process_logits),
                         PE_METHOD(select_token), PE_METHOD(token_counts_add), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "physicedit_amd._binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "build_id", PE_BINDING_ID) != 0) { Py_DECREF(m); return nullptr; }
    return m;
}
