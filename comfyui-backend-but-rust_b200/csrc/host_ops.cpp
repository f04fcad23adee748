// The hot entry points of linear.py as a CPython extension: arguments in, one call of the C ABI, results out. A block is
// fifteen calls, and through ctypes each of them cost 10 to 12 us of host time beside the launch itself (two tensor
// allocations and a stream lookup through the Python bindings, seventeen converted arguments), more than most of the kernels
// of a small block run for: two prompts' cross-attention K and V took 40 us for 25 us of kernels. Here the same steps take
// about 3 us. linear.py keeps the signatures; what is not on a block's path stays on ctypes there.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "gpu_kernels.h"

namespace {

struct Error {};               // a Python exception is set

[[noreturn]] void raise(PyObject* type, const char* text) {
    PyErr_SetString(type, text);
    throw Error();
}
// The module's attribute `ok` (ffi.ok, put there by linear.py) raises the error a return code stands for.
[[noreturn]] void failed(PyObject* self, int rc, const char* what) {
    PyObject* r = PyObject_CallMethod(self, "ok", "is", rc, what);
    Py_XDECREF(r);
    if (r) PyErr_SetString(PyExc_RuntimeError, what);
    throw Error();
}
// One call of the C ABI without the interpreter lock (a launch can block on a full queue), as ctypes makes it.
template <typename... P, typename... A> void call(PyObject* self, const char* name, int (*f)(P...), A... args) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(static_cast<P>(args)...);
    Py_END_ALLOW_THREADS
    if (rc != 0) failed(self, rc, name);
}
#define CALL(f, ...) call(self, #f, f, __VA_ARGS__)
const at::Tensor* opt(PyObject* o) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "expected a torch tensor");
    return &THPVariable_Unpack(o);
}
const at::Tensor& ten(PyObject* o) {
    const at::Tensor* t = opt(o);
    if (!t) raise(PyExc_TypeError, "expected a torch tensor");
    return *t;
}
const at::Tensor& on_gpu(PyObject* o) {
    const at::Tensor& t = ten(o);
    if (!t.is_cuda()) raise(PyExc_ValueError, "this path runs on CUDA tensors only");
    return t;
}
template <typename T = void> T* ptr(const at::Tensor* t) { return t ? reinterpret_cast<T*>(t->data_ptr()) : nullptr; }
template <typename T = void> T* ptr(const at::Tensor& t) { return reinterpret_cast<T*>(t.data_ptr()); }
int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Error();
    return v;
}
int integer32(PyObject* o) { return (int)integer(o); }
float real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Error();
    return (float)v;
}
int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kHalf: return 1;
        case at::kBFloat16: return 2;
        default: raise(PyExc_KeyError, c10::toString(t.scalar_type()));
    }
}
at::ScalarType out_dtype(PyObject* o) {
    if (!THPDtype_Check(o)) raise(PyExc_TypeError, "out_dtype is not a torch dtype");
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
void rows_cols(const at::Tensor& t, int64_t& M, int64_t& K) {
    if (t.dim() != 2) raise(PyExc_ValueError, "expected a matrix");
    M = t.size(0), K = t.size(1);
}
at::Tensor matrix(const at::Tensor& like, int64_t M, int64_t K, at::ScalarType dt) {
    return at::empty({M, K}, at::TensorOptions().dtype(dt).device(like.device()));
}
at::Tensor vec(const at::Tensor& like, int64_t M, at::ScalarType dt = at::kFloat) {
    return at::empty({M}, at::TensorOptions().dtype(dt).device(like.device()));
}
at::Tensor given_or(PyObject* o, at::Tensor (*make)(const at::Tensor&, int64_t, int64_t, at::ScalarType), const at::Tensor& like, int64_t M,
                    int64_t K, at::ScalarType dt) {
    const at::Tensor* t = opt(o);
    return t ? *t : make(like, M, K, dt);
}
void* stream() { return (void*)c10::cuda::getCurrentCUDAStream().stream(); }
PyObject* wrap(PyObject* given, const at::Tensor& t) {
    if (given && given != Py_None) return Py_NewRef(given);
    return THPVariable_Wrap(t);
}
PyObject* pair(PyObject* ga, const at::Tensor& a, PyObject* gb, const at::Tensor& b) {
    PyObject* pa = wrap(ga, a);
    PyObject* pb = pa ? wrap(gb, b) : nullptr;
    PyObject* r = pb ? PyTuple_Pack(2, pa, pb) : nullptr;
    Py_XDECREF(pa), Py_XDECREF(pb);
    return r;
}
template <typename F> PyObject* guarded(Py_ssize_t have, Py_ssize_t want, F&& f) {
    HANDLE_TH_ERRORS                       // torch's own errors (out of memory among them) as its bindings raise them
    if (have != want) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, have);
        return nullptr;
    }
    try {
        return f();
    } catch (const Error&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}
#define FAST(name, n) PyObject* name(PyObject* self, PyObject* const* a, Py_ssize_t nargs) { return guarded(nargs, n, [&]() -> PyObject* {
#define END }); }

// x, prologue, rotate, K, g, up_offset, q, scales, norm_w, norm_b, eps, mod_scale, mod_shift
FAST(quant_rows, 13)
    const at::Tensor& x = on_gpu(a[0]);
    const int64_t M = x.size(0), K = a[3] == Py_None ? x.size(1) : integer(a[3]);
    at::Tensor q = given_or(a[6], matrix, x, M, K, at::kChar);
    const at::Tensor* given_s = opt(a[7]);
    at::Tensor s = given_s ? *given_s : vec(x, M);
    const at::Tensor *g = opt(a[4]), *nb = opt(a[9]);
    const int dt = dtype_code(x);
    if (nb)
        CALL(gpu_quant_rows_b, dt, integer32(a[1]), ptr(x), x.stride(0), ptr<float>(opt(a[8])), ptr<float>(nb), real(a[10]), ptr(opt(a[11])),
                               ptr(opt(a[12])), ptr<int8_t>(q), ptr<float>(s), (int)M, (int)K, integer32(a[2]), stream());
    else
        CALL(gpu_quant_rows, dt, integer32(a[1]), ptr(x), x.stride(0), ptr(g), g ? g->stride(0) : 0, integer(a[5]), ptr<float>(opt(a[8])), real(a[10]),
                             ptr(opt(a[11])), ptr(opt(a[12])), ptr<int8_t>(q), ptr<float>(s), (int)M, (int)K, integer32(a[2]), stream());
    return pair(a[6], q, a[7], s);
END
// x, rotate
FAST(sd_quant_rows, 2)
    const at::Tensor& x = on_gpu(a[0]);
    int64_t M, K;
    rows_cols(x, M, K);
    at::Tensor q = matrix(x, M, K, at::kChar), s = vec(x, M);
    CALL(gpu_sd_quant_rows, ptr(x), x.stride(0), ptr<int8_t>(q), ptr<float>(s), (int)M, (int)K, integer32(a[1]), stream());
    return pair(nullptr, q, nullptr, s);
END
// x, w, b, eps, rotate
FAST(sd_ln_quant_rows, 5)
    const at::Tensor& x = on_gpu(a[0]);
    int64_t M, K;
    rows_cols(x, M, K);
    at::Tensor q = matrix(x, M, K, at::kChar), s = vec(x, M);
    CALL(gpu_sd_ln_quant_rows, ptr(x), x.stride(0), ptr<float>(opt(a[1])), ptr<float>(opt(a[2])), real(a[3]), ptr<int8_t>(q), ptr<float>(s), (int)M, (int)K,
                               integer32(a[4]), stream());
    return pair(nullptr, q, nullptr, s);
END
// x, rotate
FAST(sd_geglu_quant_rows, 2)
    const at::Tensor& x = on_gpu(a[0]);
    const int64_t M = x.size(0), I = x.size(1) / 2;
    at::Tensor q = matrix(x, M, I, at::kChar), s = vec(x, M);
    CALL(gpu_sd_geglu_quant_rows, ptr(x), ptr<int8_t>(q), ptr<float>(s), (int)M, (int)I, integer32(a[1]), stream());
    return pair(nullptr, q, nullptr, s);
END
// x, w, b, groups, eps, rotate
FAST(sd_group_norm_quant_rows, 6)
    const at::Tensor& x = on_gpu(a[0]);
    if (x.dim() != 3) raise(PyExc_ValueError, "expected [N, P, C]");
    const int64_t N = x.size(0), P = x.size(1), C = x.size(2), G = integer(a[3]);
    at::Tensor q = matrix(x, N * P, C, at::kChar), s = vec(x, N * P), sums = vec(x, N * G * 2 + 2, at::kDouble);
    CALL(gpu_sd_group_norm_quant_rows, ptr(x), ptr<float>(opt(a[1])), ptr<float>(opt(a[2])), ptr(sums), (int)N, P, (int)C, (int)G, real(a[4]),
                                       ptr<int8_t>(q), ptr<float>(s), integer32(a[5]), stream());
    return pair(nullptr, q, nullptr, s);
END
// x, d, rotate
FAST(sd_unpad_quant_rows, 3)
    const at::Tensor& x = on_gpu(a[0]);
    if (x.dim() != 3) raise(PyExc_ValueError, "expected [M, H, dp]");
    const int64_t M = x.size(0), H = x.size(1), dp = x.size(2), d = integer(a[1]);
    at::Tensor q = matrix(x, M, H * d, at::kChar), s = vec(x, M);
    CALL(gpu_sd_unpad_quant_rows, ptr(x), ptr<int8_t>(q), ptr<float>(s), (int)M, (int)H, (int)d, (int)dp, integer32(a[2]), stream());
    return pair(nullptr, q, nullptr, s);
END
// A, W, xs, ws, bias, out_dtype, act, rscale, resid, out
FAST(int8_gemm, 10)
    const at::Tensor &A = on_gpu(a[0]), &W = ten(a[1]);
    int64_t M, K;
    rows_cols(A, M, K);
    const int64_t N = W.size(0);
    at::Tensor D = given_or(a[9], matrix, A, M, N, a[9] == Py_None ? out_dtype(a[5]) : at::kFloat);
    const int dt = dtype_code(D), act = integer32(a[6]);
    const at::Tensor *bias = opt(a[4]), *resid = opt(a[8]);
    const int8_t *pa = ptr<int8_t>(A), *pw = ptr<int8_t>(W);
    const float *xs = ptr<float>(opt(a[2])), *ws = ptr<float>(opt(a[3]));
    if (resid)
        CALL(gpu_int8_gemm_residual, pa, pw, xs, ws, ptr(bias), ptr(opt(a[7])), ptr(resid), ptr(D), M, N, K, dt, stream());
    else if (act) CALL(gpu_int8_gemm_act, pa, pw, xs, ws, ptr(bias), ptr(D), M, N, K, dt, act, stream());
    else CALL(gpu_int8_gemm, pa, pw, xs, ws, ptr(bias), ptr(D), M, N, K, dt, stream());
    return wrap(a[9], D);
END
// A, W, xs, ws, bias, act, out, amax_part
FAST(int8_gemm_act_rot, 8)
    const at::Tensor &A = on_gpu(a[0]), &W = ten(a[1]);
    int64_t M, K;
    rows_cols(A, M, K);
    const int64_t N = W.size(0);
    at::Tensor D = given_or(a[6], matrix, A, M, N, at::kBFloat16), parts = given_or(a[7], matrix, A, N / 64, M, at::kFloat);
    CALL(gpu_int8_gemm_act_rot, ptr<int8_t>(A), ptr<int8_t>(W), ptr<float>(opt(a[2])), ptr<float>(opt(a[3])), ptr(opt(a[4])), ptr(D), ptr<float>(parts),
                                M, N, K, integer32(a[5]), stream());
    return pair(a[6], D, a[7], parts);
END
// xr, amax_part, q, scales
FAST(quant_rows_rotated, 4)
    const at::Tensor& x = on_gpu(a[0]);
    int64_t M, K;
    rows_cols(x, M, K);
    at::Tensor q = given_or(a[2], matrix, x, M, K, at::kChar);
    const at::Tensor* given_s = opt(a[3]);
    at::Tensor s = given_s ? *given_s : vec(x, M);
    CALL(gpu_quant_rows_rotated, ptr(x), ptr<float>(ten(a[1])), ptr<int8_t>(q), ptr<float>(s), (int)M, (int)K, stream());
    return pair(a[2], q, a[3], s);
END
// A, packed, s_rel, xs, s_channel, bias, out_dtype, act, rscale, resid, out, G
FAST(w6a8_gemm, 12)
    const at::Tensor &A = on_gpu(a[0]), &W = ten(a[1]);
    int64_t M, K;
    rows_cols(A, M, K);
    const int64_t N = W.size(0);
    at::Tensor D = given_or(a[10], matrix, A, M, N, a[10] == Py_None ? out_dtype(a[6]) : at::kFloat);
    const int dt = dtype_code(D), act = integer32(a[7]), G = integer32(a[11]);
    const at::Tensor *bias = opt(a[5]), *resid = opt(a[9]);
    const int8_t* pa = ptr<int8_t>(A);
    const uint8_t *pw = ptr<uint8_t>(W), *rel = ptr<uint8_t>(opt(a[2]));
    const float *xs = ptr<float>(opt(a[3])), *ch = ptr<float>(opt(a[4]));
    if (resid)
        CALL(gpu_w6a8_gemm_residual, pa, pw, rel, xs, ch, ptr(bias), ptr(opt(a[8])), ptr(resid), ptr(D), M, N, K, G, dt, stream());
    else if (act) CALL(gpu_w6a8_gemm_act, pa, pw, rel, xs, ch, ptr(bias), ptr(D), M, N, K, G, dt, act, stream());
    else CALL(gpu_w6a8_gemm, pa, pw, rel, xs, ch, ptr(bias), ptr(D), M, N, K, G, dt, stream());
    return wrap(a[10], D);
END

// ---- operators that check their tensors: shapes, types and devices before anything is launched ---------------------------------

void check(bool ok, const char* text) {
    if (!ok) raise(PyExc_ValueError, text);
}
// On the device of x whichever is current, on that device's current stream.
struct On {
    c10::cuda::CUDAGuard guard;
    c10::Device device;
    explicit On(const at::Tensor& x) : guard(x.device()), device(x.device()) {}
    void same(std::initializer_list<const at::Tensor*> all) const {
        for (const at::Tensor* t : all)
            if (t) check(t->device() == device, "the tensors of a call lie on one device");
    }
};
bool shaped(const at::Tensor& t, std::initializer_list<int64_t> sizes) { return t.sizes() == at::IntArrayRef(sizes); }
bool plain(const at::Tensor& t, at::ScalarType dt, std::initializer_list<int64_t> sizes) { return t.scalar_type() == dt && t.is_contiguous() && shaped(t, sizes); }
int attention_dtype(const at::Tensor& t) {
    check(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, "attention takes fp16 or bf16 rows");
    return dtype_code(t);
}
// Strides of batch, row and head; a dimension of one has none.
void put_strides(const at::Tensor& t, int64_t* s) {
    check(t.dim() == 4 && (t.size(3) <= 1 || t.stride(3) == 1), "expected [B, L, heads, D] with the values of a head side by side");
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
}
int small(int64_t v) {
    check(v <= INT32_MAX, "a dimension does not fit 32 bits");
    return (int)v;
}

// x, packed, scales, zeros, bias, out, beta, out_dtype
FAST(w4_linear, 8)
    const at::Tensor &x = on_gpu(a[0]), &W = ten(a[1]), &sc = ten(a[2]);
    const at::Tensor *z = opt(a[3]), *bias = opt(a[4]), *given = opt(a[5]);
    const On on(x);
    on.same({&W, &sc, z, bias, given});
    int64_t M, K;
    rows_cols(x, M, K);
    check(W.dim() == 2 && sc.dim() == 2 && sc.size(1) > 0 && K > 0 && K % sc.size(1) == 0, "expected packed [N, K / 2] and scales [N, K / G]");
    const int64_t N = W.size(0), groups = sc.size(1);
    check(plain(W, at::kByte, {N, K / 2}) && K % 2 == 0 && shaped(sc, {N, groups}) && sc.is_contiguous(), "packed is uint8 [N, K / 2], scales [N, K / G], both contiguous");
    check(sc.scalar_type() == at::kHalf || sc.scalar_type() == at::kBFloat16, "scales are fp16 or bf16");
    check(!z || plain(*z, at::kByte, {N, groups}), "zero points are uint8 [N, K / G]");
    check(x.stride(1) == 1 || K == 1, "the values of a row of x lie side by side");
    const float beta = real(a[6]);
    check(beta == 0.f || given, "beta needs the out that it scales");
    at::Tensor D = given ? *given : matrix(x, M, N, a[7] == Py_None ? x.scalar_type() : out_dtype(a[7]));
    check(shaped(D, {M, N}) && (D.stride(1) == 1 || N == 1), "out is [M, N], the values of a row side by side");
    check(!bias || plain(*bias, D.scalar_type(), {N}), "bias is [N] in the type of out");
    CALL(gpu_w4_linear, dtype_code(x), ptr(x), M > 1 ? x.stride(0) : K, ptr(W), dtype_code(sc), ptr(sc), ptr(z), ptr(bias), dtype_code(D), ptr(D),
                        M > 1 ? D.stride(0) : N, beta, small(M), small(N), small(K), small(K / groups), stream());
    return wrap(a[5], D);
END
// q, k, v, kv_len, key_mask, scale, out
FAST(cross_attention, 7)
    const at::Tensor &q = on_gpu(a[0]), &k = ten(a[1]), &v = ten(a[2]);
    const at::Tensor *kv_len = opt(a[3]), *mask = opt(a[4]), *given = opt(a[6]);
    const On on(q);
    on.same({&k, &v, kv_len, mask, given});
    const int dt = attention_dtype(q);
    int64_t st[12];
    put_strides(q, st), put_strides(k, st + 3), put_strides(v, st + 6);
    const int64_t B = q.size(0), Lq = q.size(1), H = q.size(2), D = q.size(3), Lkv = k.size(1), Hkv = k.size(2);
    check(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v have one type");
    check(shaped(k, {B, Lkv, Hkv, D}) && shaped(v, {B, Lkv, Hkv, D}) && Hkv > 0 && H % Hkv == 0, "expected k and v [B, Lkv, Hkv, D], H a multiple of Hkv");
    check(!kv_len || plain(*kv_len, at::kInt, {B}), "kv_len is int32 [B]");
    check(!mask || ((mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte) && shaped(*mask, {B, Lkv}) && (mask->stride(1) == 1 || Lkv <= 1)),
          "key_mask is bool [B, Lkv]");
    at::Tensor out = given ? *given : at::empty(q.sizes(), q.options());
    check(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type(), "out has the shape and type of q");
    put_strides(out, st + 9);
    CALL(gpu_cross_attention, dt, ptr(q), ptr(k), ptr(v), ptr(out), st, ptr<int32_t>(kv_len), ptr<uint8_t>(mask), mask && B > 1 ? mask->stride(0) : 0, small(B),
                              small(Lq), small(Lkv), small(H), small(Hkv), small(D), real(a[5]), stream());
    return wrap(a[6], out);
END

// k, v, k_scale, v_scale of a cache
struct Cache {
    const at::Tensor &k, &v, &ks, &vs;
    int64_t pages, Hkv, T, D;
    explicit Cache(PyObject* const* a) : k(on_gpu(a[0])), v(ten(a[1])), ks(ten(a[2])), vs(ten(a[3])) {
        check(k.dim() == 4, "a cache's keys and values are int8 [pages, Hkv, T, D]");
        pages = k.size(0), Hkv = k.size(1), T = k.size(2), D = k.size(3);
        check(plain(k, at::kChar, {pages, Hkv, T, D}) && plain(v, at::kChar, {pages, Hkv, T, D}), "a cache's keys and values are int8 [pages, Hkv, T, D]");
        check(plain(ks, at::kFloat, {pages, Hkv}) && plain(vs, at::kFloat, {pages, Hkv}), "a cache's scales are f32 [pages, Hkv]");
    }
};
void check_table(const at::Tensor& t, int64_t B) {
    check(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == B && (t.stride(1) == 1 || t.size(1) <= 1), "table is int32 [B, pages to a sequence]");
}
int64_t table_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : 0; }

// cache (4), k, v, table, start, count
FAST(kv8_append, 9)
    const Cache c(a);
    const at::Tensor &k = ten(a[4]), &v = ten(a[5]), &table = ten(a[6]), &start = ten(a[7]);
    const at::Tensor* count = opt(a[8]);
    const On on(c.k);
    on.same({&c.v, &c.ks, &c.vs, &k, &v, &table, &start, count});
    int64_t st[6];
    put_strides(k, st), put_strides(v, st + 3);
    const int64_t B = k.size(0), L = k.size(1);
    check(shaped(k, {B, L, c.Hkv, c.D}) && shaped(v, {B, L, c.Hkv, c.D}) && k.scalar_type() == v.scalar_type(), "expected k and v [B, L, Hkv, D] of one type");
    check_table(table, B);
    check(plain(start, at::kInt, {B}) && (!count || plain(*count, at::kInt, {B})), "start and count are int32 [B]");
    CALL(gpu_kv8_append, dtype_code(k), ptr(k), ptr(v), st, ptr<int8_t>(c.k), ptr<int8_t>(c.v), ptr<float>(c.ks), ptr<float>(c.vs), ptr<int32_t>(table),
                         table_stride(table), ptr<int32_t>(start), ptr<int32_t>(count), small(B), small(L), small(c.Hkv), small(c.D), small(c.T), c.pages,
                         small(table.size(1)), stream());
    Py_RETURN_NONE;
END
// cache (4), table, lengths, rows, dtype
FAST(kv8_dequant, 8)
    const Cache c(a);
    const at::Tensor &table = ten(a[4]), &len = ten(a[5]);
    const On on(c.k);
    on.same({&c.v, &c.ks, &c.vs, &table, &len});
    const int64_t B = table.size(0), rows = integer(a[6]);
    check_table(table, B);
    check(plain(len, at::kInt, {B}) && rows >= 0, "lengths is int32 [B], rows at least 0");
    const auto opts = at::TensorOptions().dtype(out_dtype(a[7])).device(c.k.device());
    at::Tensor k = at::empty({B, rows, c.Hkv, c.D}, opts), v = at::empty({B, rows, c.Hkv, c.D}, opts);
    CALL(gpu_kv8_dequant, dtype_code(k), ptr<int8_t>(c.k), ptr<int8_t>(c.v), ptr<float>(c.ks), ptr<float>(c.vs), ptr<int32_t>(table), table_stride(table),
                          ptr<int32_t>(len), ptr(k), ptr(v), small(B), rows, small(c.Hkv), small(c.D), small(c.T), c.pages, small(table.size(1)), stream());
    return pair(nullptr, k, nullptr, v);
END
// cache (4), q, table, lengths, q_len, causal, scale, out
FAST(kv8_attention, 11)
    const Cache c(a);
    const at::Tensor &q = on_gpu(a[4]), &table = ten(a[5]), &len = ten(a[6]);
    const at::Tensor *q_len = opt(a[7]), *given = opt(a[10]);
    const On on(q);
    on.same({&c.k, &c.v, &c.ks, &c.vs, &table, &len, q_len, given});
    const int dt = attention_dtype(q);
    int64_t st[6];
    put_strides(q, st);
    const int64_t B = q.size(0), L = q.size(1), H = q.size(2), D = q.size(3);
    check(D == c.D && c.Hkv > 0 && H % c.Hkv == 0, "expected q [B, L, H, D] with the cache's D, H a multiple of its heads");
    check_table(table, B);
    check(plain(len, at::kInt, {B}) && (!q_len || plain(*q_len, at::kInt, {B})), "lengths and q_len are int32 [B]");
    at::Tensor out = given ? *given : q_len ? at::zeros(q.sizes(), q.options()) : at::empty(q.sizes(), q.options());
    check(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type(), "out has the shape and type of q");
    put_strides(out, st + 3);
    CALL(gpu_kv8_attention, dt, ptr(q), ptr(out), st, ptr<int8_t>(c.k), ptr<int8_t>(c.v), ptr<float>(c.ks), ptr<float>(c.vs), ptr<int32_t>(table),
                            table_stride(table), ptr<int32_t>(len), ptr<int32_t>(q_len), integer32(a[8]), small(B), small(L), small(H), small(c.Hkv), small(D),
                            small(c.T), c.pages, small(table.size(1)), real(a[9]), stream());
    return wrap(a[10], out);
END
// Strides of rows and heads of [rows, heads, D]
void put_row_strides(const at::Tensor& t, int64_t* s) {
    check(t.dim() == 3 && (t.size(2) <= 1 || t.stride(2) == 1), "expected [rows, heads, D] with the values of a head side by side");
    for (int i = 0; i < 2; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
}
// q, k, v, offsets, causal, scale, out
FAST(packed_attention, 7)
    const at::Tensor &q = on_gpu(a[0]), &k = ten(a[1]), &v = ten(a[2]), &offsets = ten(a[3]);
    const at::Tensor* given = opt(a[6]);
    const On on(q);
    on.same({&k, &v, &offsets, given});
    const int dt = attention_dtype(q);
    int64_t st[8];
    put_row_strides(q, st), put_row_strides(k, st + 2), put_row_strides(v, st + 4);
    const int64_t rows = q.size(0), H = q.size(1), D = q.size(2), Hkv = k.size(1);
    check(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v have one type");
    check(shaped(k, {rows, Hkv, D}) && shaped(v, {rows, Hkv, D}) && Hkv > 0 && H % Hkv == 0, "expected k and v [rows, Hkv, D], H a multiple of Hkv");
    check(offsets.dim() == 1 && offsets.size(0) >= 1 && plain(offsets, at::kInt, {offsets.size(0)}), "offsets is int32 [sequences + 1]");
    at::Tensor out = given ? *given : at::zeros(q.sizes(), q.options());
    check(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type(), "out has the shape and type of q");
    put_row_strides(out, st + 6);
    CALL(gpu_packed_attention, dt, ptr(q), ptr(k), ptr(v), ptr(out), st, ptr<int32_t>(offsets), integer32(a[4]), small(offsets.size(0) - 1), small(rows),
                               small(H), small(Hkv), small(D), real(a[5]), stream());
    return wrap(a[6], out);
END
// q, k, pos, freq, interleaved, axis, q_norm, k_norm, eps, scale, q_out, k_out
FAST(rotary, 12)
    const at::Tensor &q = on_gpu(a[0]), &pos = ten(a[2]), &freq = ten(a[3]);
    const at::Tensor *k = opt(a[1]), *axis = opt(a[5]), *qn = opt(a[6]), *kn = opt(a[7]), *gq = opt(a[10]), *gk = opt(a[11]);
    const On on(q);
    on.same({k, &pos, &freq, axis, qn, kn, gq, gk});
    const int dt = dtype_code(q);
    int64_t st[12] = {};
    put_strides(q, st);
    const int64_t B = q.size(0), L = q.size(1), D = q.size(3), half = freq.numel();
    if (k) {
        put_strides(*k, st + 3);
        check(k->scalar_type() == q.scalar_type() && k->size(0) == B && k->size(1) == L && k->size(3) == D, "expected q [B, L, H, D] and k [B, L, Hkv, D] of one type");
    }
    check(plain(freq, at::kDouble, {half}) && 2 * half <= D, "freq is f64 [rot / 2], rot at most D");
    const bool many = pos.dim() == 3;
    check(pos.scalar_type() == at::kInt && (many || pos.dim() == 2) && pos.size(-1) == L && pos.size(-2) == B && (L <= 1 || pos.stride(-1) == 1),
          "positions are int32 [B, L] or [axes, B, L]");
    const int64_t axes = many ? pos.size(0) : 1;
    check(axes >= 1 && (axes == 1 || axis), "positions of several axes need the axis of each frequency");
    check(!axis || plain(*axis, at::kByte, {half}), "axis is uint8 [rot / 2]");
    check((!qn || plain(*qn, at::kFloat, {D})) && (!kn || plain(*kn, at::kFloat, {D})), "q_norm and k_norm are f32 [D]");
    at::Tensor qo = gq ? *gq : at::empty(q.sizes(), q.options()), ko;
    check(qo.sizes() == q.sizes() && qo.scalar_type() == q.scalar_type(), "q_out has the shape and type of q");
    put_strides(qo, st + 6);
    check(k || !gk, "k_out needs k");
    if (k) {
        ko = gk ? *gk : at::empty(k->sizes(), k->options());
        check(ko.sizes() == k->sizes() && ko.scalar_type() == k->scalar_type(), "k_out has the shape and type of k");
        put_strides(ko, st + 9);
    }
    CALL(gpu_rotary, dt, ptr(q), ptr(k), ptr(qo), k ? ptr(ko) : nullptr, st, ptr<int32_t>(pos), many ? pos.stride(0) : 0, B > 1 ? pos.stride(-2) : 0, small(axes),
                     ptr<uint8_t>(axis), ptr<double>(freq), small(2 * half), integer32(a[4]), real(a[9]), ptr<float>(qn), ptr<float>(kn), real(a[8]), small(B),
                     small(L), small(q.size(2)), k ? small(k->size(2)) : 0, small(D), stream());
    if (!k) {
        PyObject* r = wrap(a[10], qo);
        PyObject* both = r ? PyTuple_Pack(2, r, Py_None) : nullptr;
        Py_XDECREF(r);
        return both;
    }
    return pair(a[10], qo, a[11], ko);
END

bool side_by_side(const at::Tensor& t) { return t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1); }
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
int64_t blocks_of(int64_t K) { return (K + 127) / 128; }

// x, prologue, K, up_offset, norm_w, eps, resid, resid_out, out, scales, out_dtype
FAST(norm_rows, 11)
    const at::Tensor& x = on_gpu(a[0]);
    const at::Tensor *w = opt(a[4]), *resid = opt(a[6]), *resid_out = opt(a[7]), *given = opt(a[8]), *given_s = opt(a[9]);
    const On on(x);
    on.same({w, resid, resid_out, given, given_s});
    check(side_by_side(x), "x is a matrix, the values of a row side by side");
    const int64_t M = x.size(0), K = a[2] == Py_None ? x.size(1) : integer(a[2]), up = integer(a[3]);
    const int prologue = integer32(a[1]);
    check(K >= 0 && K <= x.size(1) && (prologue != 3 || (up >= 0 && up + K <= x.size(1))), "x has fewer columns than the call reads");
    check(!w || plain(*w, at::kFloat, {K}), "norm_w is f32 [K]");
    check(resid || !resid_out, "resid_out needs resid");
    if (resid && !resid_out) resid_out = resid;
    for (const at::Tensor* t : {resid, resid_out})
        check(!t || (shaped(*t, {M, K}) && side_by_side(*t) && t->scalar_type() == x.scalar_type()), "resid and resid_out are [M, K] in x's type");
    const at::ScalarType dt = given ? given->scalar_type() : a[10] == Py_None ? x.scalar_type() : out_dtype(a[10]);
    const bool f8 = dt == at::kFloat8_e4m3fn;
    at::Tensor out = given ? *given : matrix(x, M, K, dt), s;
    check(shaped(out, {M, K}) && side_by_side(out), "out is [M, K], the values of a row side by side");
    check(f8 || !given_s, "scales are for e4m3");
    if (f8) {
        s = given_s ? *given_s : matrix(x, M, blocks_of(K), at::kFloat);
        check(plain(s, at::kFloat, {M, blocks_of(K)}), "scales are f32 [M, ceil(K / 128)]");
    }
    CALL(gpu_norm_rows, dtype_code(x), prologue, ptr(x), row_stride(x), up, ptr(resid), resid ? row_stride(*resid) : 0, ptr(resid_out),
                        resid_out ? row_stride(*resid_out) : 0, ptr<float>(w), real(a[5]), f8 ? 3 : dtype_code(out), ptr(out), row_stride(out),
                        f8 ? ptr<float>(s) : nullptr, small(M), small(K), stream());
    if (!f8) return wrap(a[8], out);
    return pair(a[8], out, a[9], s);
END
// x, xs, W, ws, bias, out, beta, out_dtype
FAST(f8_linear, 8)
    const at::Tensor &x = on_gpu(a[0]), &xs = ten(a[1]), &W = ten(a[2]), &ws = ten(a[3]);
    const at::Tensor *bias = opt(a[4]), *given = opt(a[5]);
    const On on(x);
    on.same({&xs, &W, &ws, bias, given});
    int64_t M, K;
    rows_cols(x, M, K);
    check(x.scalar_type() == at::kFloat8_e4m3fn && side_by_side(x), "x is e4m3, the values of a row side by side");
    check(W.dim() == 2, "the weight is e4m3 [N, K], contiguous");
    const int64_t N = W.size(0);
    check(plain(W, at::kFloat8_e4m3fn, {N, K}), "the weight is e4m3 [N, K], contiguous");
    check(plain(xs, at::kFloat, {M, blocks_of(K)}) && plain(ws, at::kFloat, {blocks_of(N), blocks_of(K)}),
          "scales are f32, contiguous: [M, ceil(K / 128)] of x, [ceil(N / 128), ceil(K / 128)] of the weight");
    const float beta = real(a[6]);
    check(beta == 0.f || given, "beta needs the out that it scales");
    at::Tensor D = given ? *given : matrix(x, M, N, out_dtype(a[7]));
    check(shaped(D, {M, N}) && side_by_side(D), "out is [M, N], the values of a row side by side");
    check(!bias || plain(*bias, D.scalar_type(), {N}), "bias is [N] in the type of out");
    CALL(gpu_f8_linear, ptr(x), row_stride(x), ptr<float>(xs), ptr(W), ptr<float>(ws), ptr(bias), dtype_code(D), ptr(D), row_stride(D), beta, small(M), small(N),
                        small(K), stream());
    return wrap(a[5], D);
END

#define M(name) {#name, (PyCFunction)(void (*)())name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {M(quant_rows), M(sd_quant_rows), M(sd_ln_quant_rows), M(sd_geglu_quant_rows), M(sd_group_norm_quant_rows),
                         M(sd_unpad_quant_rows), M(int8_gemm), M(int8_gemm_act_rot), M(quant_rows_rotated), M(w6a8_gemm),
                         M(w4_linear), M(cross_attention), M(kv8_append), M(kv8_dequant), M(kv8_attention),
                         M(packed_attention), M(rotary), M(norm_rows), M(f8_linear),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host_ops() { return PyModule_Create(&module); }
