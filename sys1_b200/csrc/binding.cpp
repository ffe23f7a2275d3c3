// The Python side of the decode-step calls (module sys1_b200._binding): arguments checked, outputs allocated, the C ABI called. From
// Python itself the checks of up to 14 tensors, at 0.1 us an attribute, and the conversion of up to 27 arguments took longer than
// the kernels of a small step. Measured, calls one after the other: block tables 14.1 -> 6.8 us, cache write 11.2 -> 4.0, attention
// 16.0 -> 7.0, delta step 15.0 -> 5.5 (a tenth more where the host is busy); what is left is the launches (3.3 us one, 5.6 the
// attention's two) and the outputs.
// Every function takes a context's handle, then the arguments of the Python function of the same name in its order (None where one is
// left out), and returns its result, or the error code of the C call as an int. Bad arguments raise ValueError.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/ops/as_strided.h>
#include <ATen/ops/empty.h>

#include <cmath>
#include <initializer_list>
#include <limits>
#include <string>

#include "../../include/sys1_b200.h"

namespace {

using at::Tensor;

struct Refused {
    std::string why;
};

std::string shape_of(at::IntArrayRef s) {
    std::string r = "[";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}

// ------------------------------------------------------------------------------------------------ arguments
struct Args {
    PyObject* const* at;
    Py_ssize_t n;

    bool given(int i) const { return at[i] != Py_None; }
    const Tensor& tensor(int i, const char* name) const {
        if (!THPVariable_Check(at[i])) throw Refused{std::string(name) + " must be a tensor"};
        return THPVariable_Unpack(at[i]);
    }
    int small(int i, const char* name) const {  // what the C ABI takes as an int
        const int64_t v = PyLong_Check(at[i]) ? PyLong_AsLongLong(at[i]) : index(at[i]);
        if (v == -1 && PyErr_Occurred()) throw python_error();
        if (v < std::numeric_limits<int>::min() || v > std::numeric_limits<int>::max()) throw Refused{std::string(name) + " is beyond 32 bits"};
        return static_cast<int>(v);
    }
    float real(int i) const {
        const double v = PyFloat_AsDouble(at[i]);
        if (v == -1.0 && PyErr_Occurred()) throw python_error();
        return static_cast<float>(v);
    }
    s1_ctx* context() const {
        if (!given(0)) return nullptr;
        void* p = PyLong_AsVoidPtr(at[0]);
        if (!p && PyErr_Occurred()) throw python_error();
        return static_cast<s1_ctx*>(p);
    }

  private:
    static int64_t index(PyObject* o) {
        PyObject* whole = PyNumber_Index(o);
        if (!whole) return -1;
        const int64_t v = PyLong_AsLongLong(whole);
        Py_DECREF(whole);
        return v;
    }
};

int gpu_of(const Tensor& t) { return t.is_cuda() ? static_cast<int>(t.get_device()) : -1; }
bool on(const Tensor& t, int dev, at::ScalarType type) { return dev >= 0 && t.is_cuda() && t.get_device() == dev && t.scalar_type() == type; }
bool has_shape(const Tensor& t, std::initializer_list<int64_t> s) { return t.sizes().equals(at::IntArrayRef(s)); }
int64_t extent(int64_t n, const char* name) {
    if (n > std::numeric_limits<int>::max()) throw Refused{std::string(name) + " has an extent beyond 32 bits"};
    return n;
}

// A dimension of size 1 has no stride: what a transposed or expanded tensor says there is of no account, and `otherwise` is used.
bool next_to(const Tensor& t, int dim) { return t.stride(dim) == 1 || t.size(dim) == 1; }
int64_t stride(const Tensor& t, int dim, int64_t otherwise) { return t.size(dim) == 1 ? otherwise : t.stride(dim); }

template <typename T>
T* address(const Tensor& t) {
    return static_cast<T*>(t.data_ptr());
}

int32_t* ints(const Tensor& t, int dev, int64_t n, const char* name) {
    if (!on(t, dev, at::kInt) || !t.is_contiguous()) throw Refused{std::string(name) + " must be a contiguous int32 CUDA tensor on the call's GPU (no CPU fallback)"};
    if (!has_shape(t, {n})) throw Refused{std::string(name) + " must have shape " + shape_of({n}) + ", not " + shape_of(t.sizes())};
    return address<int32_t>(t);
}

struct Table {
    int32_t* at;
    int64_t ld;
    int width;
};
Table table(const Tensor& t, int dev, int64_t rows) {
    if (!on(t, dev, at::kInt) || t.dim() != 2 || t.size(0) != rows || !next_to(t, 1))
        throw Refused{"block tables must be an int32 CUDA tensor [" + std::to_string(rows) + ", pages] with contiguous rows"};
    return {address<int32_t>(t), stride(t, 0, t.size(1)), static_cast<int>(extent(t.size(1), "the block table"))};
}

struct Heads {  // a tensor of head rows
    void* at = nullptr;
    int64_t token = 0, head = 0;
};
Heads heads(const Tensor& t, int dev, std::initializer_list<int64_t> shape, const char* name) {
    if (!on(t, dev, at::kBFloat16) || t.dim() != 3)
        throw Refused{std::string(name) + " must be a bf16 CUDA tensor [tokens, heads, head_dim] with contiguous head rows (no CPU fallback)"};
    if (!has_shape(t, shape)) throw Refused{std::string(name) + " must have shape " + shape_of(shape) + ", not " + shape_of(t.sizes())};
    if (t.stride(2) != 1) throw Refused{std::string(name) + " must have contiguous head rows"};
    const int64_t head = stride(t, 1, t.size(2));
    return {t.data_ptr(), stride(t, 0, (t.size(1) - 1) * head + t.size(2)), head};
}

struct Cache {
    int64_t page, token, head;
};
Cache caches(const Tensor& k, const Tensor& v, int dev) {
    if (!on(k, dev, at::kBFloat16) || k.dim() != 4 || !on(v, dev, at::kBFloat16) || v.dim() != 4)
        throw Refused{"k_cache and v_cache must be bf16 CUDA tensors [pages, page_size, kv_heads, head_dim] with contiguous head rows (no CPU fallback)"};
    bool alike = k.sizes() == v.sizes() && k.stride(3) == 1 && v.stride(3) == 1;
    for (int i = 0; i < 3 && alike; ++i) alike = k.size(i) == 1 || k.stride(i) == v.stride(i);
    if (!alike)
        throw Refused{"k_cache and v_cache must have the same shape and strides, and contiguous head rows"};
    for (int i = 0; i < 4; ++i) extent(k.size(i), "the cache");
    return {stride(k, 0, k.size(3)), stride(k, 1, k.size(3)), stride(k, 2, k.size(3))};
}

PyObject* wrapped(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* code(int rc) { return PyLong_FromLong(rc); }
// an output that was given (the same object goes back) or the one allocated here
PyObject* result(const Args& a, int i, const Tensor& made) {
    if (!a.given(i)) return wrapped(made);
    Py_INCREF(a.at[i]);
    return a.at[i];
}

template <typename Call>
int run(const Call& call) {  // the launch itself needs no interpreter
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = call();
    Py_END_ALLOW_THREADS
    return rc;
}

// ------------------------------------------------------------------------------------------------ calls
// (handle, cached, tables, free_pages, free_count, page_size, added, max_tokens, lengths, free_count_out)
PyObject* block_tables(const Args& a) {
    s1_ctx* const ctx = a.context();
    const Tensor &cached = a.tensor(1, "cached"), &tables = a.tensor(2, "block tables"), &free_pages = a.tensor(3, "free_pages"), &free_count = a.tensor(4, "free_count");
    const int dev = gpu_of(cached);
    const int rows = static_cast<int>(extent(cached.numel(), "cached")), pool = static_cast<int>(extent(free_pages.numel(), "free_pages"));
    if (!a.given(7) && a.given(6)) throw Refused{"max_tokens is needed with `added`: the host knows how many tokens the batch has"};
    const int page = a.small(5, "page_size"), tokens = a.given(7) ? a.small(7, "max_tokens") : rows;
    if (tokens < 0) throw Refused{"max_tokens must not be negative"};
    const int32_t *cp = ints(cached, dev, rows, "cached"), *fp = ints(free_pages, dev, pool, "free_pages"), *np = ints(free_count, dev, 1, "free_count");
    const int32_t* ap = a.given(6) ? ints(a.tensor(6, "added"), dev, rows, "added") : nullptr;
    const Table t = table(tables, dev, rows);
    int32_t* lengths = a.given(8) ? ints(a.tensor(8, "lengths"), dev, rows, "lengths") : nullptr;
    int32_t* left = a.given(9) ? ints(a.tensor(9, "free_count_out"), dev, 1, "free_count_out") : nullptr;
    // one buffer for what is new: positions, slots, first tokens, lengths, pages left
    const Tensor out = at::empty({2LL * tokens + 2LL * rows + 2}, cached.options());
    int32_t* at = address<int32_t>(out);
    const int64_t cu = 2LL * tokens, len = cu + rows + 1, cnt = len + rows;
    const int rc = run([&] {
        return s1_block_tables(ctx, cp, ap, rows, page, fp, pool, np, left ? left : at + cnt, t.at, t.ld, t.width, lengths ? lengths : at + len, at + cu, at,
                               at + tokens, tokens);
    });
    if (rc) return code(rc);
    PyObject* r = PyTuple_New(5);
    if (!r) throw python_error();
    at::AutoDispatchBelowADInplaceOrView plain;  // integers: no gradients, and no bookkeeping of views (5 us a call)
    auto part = [&](int64_t from, int64_t n) { return at::as_strided(out, {n}, {1}, from); };
    PyTuple_SET_ITEM(r, 0, lengths ? result(a, 8, out) : wrapped(part(len, rows)));
    PyTuple_SET_ITEM(r, 1, wrapped(part(cu, rows + 1)));
    PyTuple_SET_ITEM(r, 2, wrapped(part(0, tokens)));
    PyTuple_SET_ITEM(r, 3, wrapped(part(tokens, tokens)));
    PyTuple_SET_ITEM(r, 4, left ? result(a, 9, out) : wrapped(part(cnt, 1)));
    return r;
}

// (handle, k, v, k_cache, v_cache, slots, norm_weight, eps, cos, sin, positions, rotary_dim, bf16_ops)
PyObject* cache_write(const Args& a) {
    s1_ctx* const ctx = a.context();
    const Tensor &k = a.tensor(1, "k"), &v = a.tensor(2, "v"), &kc = a.tensor(3, "k_cache"), &vc = a.tensor(4, "v_cache"), &slots = a.tensor(5, "slots");
    const int dev = gpu_of(k);
    const Cache cache = caches(kc, vc, dev);
    const int64_t kv = kc.size(2), dim = kc.size(3), T = k.dim() ? extent(k.size(0), "k") : 0;
    const Heads kh = heads(k, dev, {T, kv, dim}, "k"), vh = heads(v, dev, {T, kv, dim}, "v");
    const int32_t* sp = ints(slots, dev, T, "slots");
    const void* weight = nullptr;
    const float *cos = nullptr, *sin = nullptr;
    const int32_t* positions = nullptr;
    int rows = 0;
    const int rotary = a.small(11, "rotary_dim");
    if (a.given(6)) {
        if (!a.given(8) || !a.given(9) || !a.given(10)) throw Refused{"keys that are normed are rotated too: cos, sin and positions are needed"};
        const Tensor& w = a.tensor(6, "norm_weight");
        if (!on(w, dev, at::kBFloat16) || !has_shape(w, {dim}) || !w.is_contiguous())
            throw Refused{"norm_weight must be a contiguous bf16 CUDA tensor " + shape_of({dim})};
        const Tensor &c = a.tensor(8, "cos"), &s = a.tensor(9, "sin");
        rows = static_cast<int>(c.dim() ? extent(c.size(0), "cos") : 0);
        for (const Tensor* t : {&c, &s})
            if (!on(*t, dev, at::kFloat) || !has_shape(*t, {rows, rotary / 2}) || !t->is_contiguous())
                throw Refused{"cos and sin must be contiguous f32 CUDA tensors [positions, rotary_dim / 2]"};
        weight = w.data_ptr(), cos = address<float>(c), sin = address<float>(s), positions = ints(a.tensor(10, "positions"), dev, T, "positions");
    }
    if (T == 0) return code(0);
    const float eps = a.real(7);
    const int bf16_ops = PyObject_IsTrue(a.at[12]);
    if (bf16_ops < 0) throw python_error();
    return code(run([&] {
        return s1_cache_write(ctx, kh.at, kh.token, kh.head, vh.at, vh.token, vh.head, sp, static_cast<int>(T), static_cast<int>(kv), static_cast<int>(dim), weight,
                              eps, cos, sin, positions, rows, rotary, bf16_ops, kc.data_ptr(), vc.data_ptr(), static_cast<int>(kc.size(0)),
                              static_cast<int>(kc.size(1)), cache.page, cache.token, cache.head);
    }));
}

// (handle, q, k_cache, v_cache, tables, lengths, gate, scale, out, workspace)
PyObject* attention_paged(const Args& a) {
    s1_ctx* const ctx = a.context();
    const Tensor &q = a.tensor(1, "q"), &kc = a.tensor(2, "k_cache"), &vc = a.tensor(3, "v_cache"), &tables = a.tensor(4, "block tables"), &lengths = a.tensor(5, "lengths");
    const int dev = gpu_of(q);
    const Cache cache = caches(kc, vc, dev);
    const int64_t kv = kc.size(2), dim = kc.size(3), B = q.dim() == 3 ? extent(q.size(0), "q") : 0, H = q.dim() == 3 ? extent(q.size(1), "q") : 0;
    const Heads qh = heads(q, dev, {B, H, dim}, "q");
    const Table t = table(tables, dev, B);
    const int32_t* lp = ints(lengths, dev, B, "lengths");
    Heads gh;
    if (a.given(6)) gh = heads(a.tensor(6, "gate"), dev, {B, H, dim}, "gate");
    const float scale = a.given(7) ? a.real(7) : static_cast<float>(std::pow(static_cast<double>(dim), -0.5));
    Tensor out;
    if (!a.given(8)) {
        out = at::empty({B, H * dim}, q.options());
    } else {
        out = a.tensor(8, "out");
        if (!on(out, dev, at::kBFloat16) || !has_shape(out, {B, H * dim}) || out.stride(1) != 1)
            throw Refused{"out must be a bf16 CUDA tensor " + shape_of({B, H * dim}) + " with contiguous rows"};
    }
    if (B == 0) return result(a, 8, out);
    const Tensor& ws = a.tensor(9, "the workspace");
    if (!on(ws, dev, at::kByte) || !ws.is_contiguous()) throw Refused{"the workspace must be a contiguous uint8 CUDA tensor"};
    const int rc = run([&] {
        return s1_attention_paged(ctx, qh.at, qh.token, qh.head, kc.data_ptr(), vc.data_ptr(), static_cast<int>(kc.size(0)), static_cast<int>(kc.size(1)),
                                  cache.page, cache.token, cache.head, t.at, t.ld, t.width, lp, static_cast<int>(B), static_cast<int>(H), static_cast<int>(kv),
                                  static_cast<int>(dim), scale, gh.at, gh.token, gh.head, out.data_ptr(), stride(out, 0, H * dim), ws.data_ptr(),
                                  static_cast<size_t>(ws.numel()));
    });
    return rc ? code(rc) : result(a, 8, out);
}

// (handle, mixed, conv_weight, positions, b, a, dt_bias, neg_exp_a, z, norm_weight, eps, conv_state, state, key_heads, state_index, out)
PyObject* gated_delta_rule_step(const Args& args) {
    s1_ctx* const ctx = args.context();
    const Tensor &mixed = args.tensor(1, "mixed"), &state = args.tensor(12, "state");
    const int dev = gpu_of(mixed);
    if (mixed.dim() != 2 || state.dim() != 4) throw Refused{"mixed must be [rows, channels] and state [states, value_heads, 128, 128]"};
    const int64_t rows = extent(mixed.size(0), "mixed"), C = mixed.size(1), states = extent(state.size(0), "state"), Hv = extent(state.size(1), "state"), inner = Hv * 128;
    const int key_heads = args.small(13, "key_heads");
    if (C != (2LL * key_heads + Hv) * 128)
        throw Refused{"mixed must have " + std::to_string((2LL * key_heads + Hv) * 128) + " columns for " + std::to_string(key_heads) + " key and " + std::to_string(Hv) +
                      " value heads, not " + std::to_string(C)};
    auto check = [&](const Tensor& t, const char* name, at::ScalarType type, std::initializer_list<int64_t> shape, bool by_rows) {
        if (!on(t, dev, type) || !has_shape(t, shape) || !(by_rows ? next_to(t, 1) : t.is_contiguous()))
            throw Refused{std::string(name) + " must be a " + (by_rows ? "" : "contiguous ") +
                          (type == at::kBFloat16 ? "bfloat16" : type == at::kFloat ? "float32" : "int32") + " CUDA tensor " + shape_of(shape) +
                          (by_rows ? " with contiguous rows" : "") + " on the call's GPU (no CPU fallback)"};
        return t.data_ptr();
    };
    const Tensor &conv_weight = args.tensor(2, "conv_weight"), &b = args.tensor(4, "b"), &a = args.tensor(5, "a"), &z = args.tensor(8, "z");
    const void* x = check(mixed, "mixed", at::kBFloat16, {rows, C}, true);
    const void *bp = check(b, "b", at::kBFloat16, {rows, Hv}, true), *ap = check(a, "a", at::kBFloat16, {rows, Hv}, true);
    if (a.stride(0) != b.stride(0) && rows > 1) throw Refused{"b and a must have the same row stride (column ranges of one projection, or contiguous)"};
    const void* zp = check(z, "z", at::kBFloat16, {rows, inner}, true);
    const auto* positions = static_cast<const int32_t*>(check(args.tensor(3, "positions"), "positions", at::kInt, {rows}, false));
    const int32_t* index = args.given(14) ? static_cast<const int32_t*>(check(args.tensor(14, "state_index"), "state_index", at::kInt, {rows}, false)) : nullptr;
    const void* taps = conv_weight.dim() == 3 ? check(conv_weight, "conv_weight", at::kBFloat16, {C, 1, 4}, false)
                                              : check(conv_weight, "conv_weight", at::kBFloat16, {C, 4}, false);
    const auto* dt_bias = static_cast<const float*>(check(args.tensor(6, "dt_bias"), "dt_bias", at::kFloat, {Hv}, false));
    const auto* decay = static_cast<const float*>(check(args.tensor(7, "neg_exp_a"), "neg_exp_a", at::kFloat, {Hv}, false));
    const void* weight = check(args.tensor(9, "norm_weight"), "norm_weight", at::kBFloat16, {128}, false);
    auto* sp = static_cast<float*>(check(state, "state", at::kFloat, {states, Hv, 128, 128}, false));
    void* cs = check(args.tensor(11, "conv_state"), "conv_state", at::kBFloat16, {states, 4, C}, false);
    const float eps = args.real(10);
    Tensor out;
    if (!args.given(15)) {
        out = at::empty({rows, inner}, mixed.options());
    } else {
        out = args.tensor(15, "out");
        if (!on(out, dev, at::kBFloat16) || !has_shape(out, {rows, inner}) || out.stride(1) != 1)
            throw Refused{"out must be a bf16 CUDA tensor " + shape_of({rows, inner}) + " with contiguous rows"};
    }
    if (rows == 0) return result(args, 15, out);
    const int rc = run([&] {
        return s1_gated_delta_rule_step(ctx, x, stride(mixed, 0, C), taps, positions, bp, ap, stride(b, 0, Hv), dt_bias, decay, zp, stride(z, 0, inner), weight, eps,
                                        index, static_cast<int>(states), cs, sp, static_cast<int>(rows), key_heads, static_cast<int>(Hv), out.data_ptr(),
                                        stride(out, 0, inner));
    });
    return rc ? code(rc) : result(args, 15, out);
}

template <PyObject* (*F)(const Args&), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%d arguments, not %zd", N, n);
        return nullptr;
    }
    try {
        return F(Args{args, n});
    } catch (const Refused& r) {
        PyErr_SetString(PyExc_ValueError, r.why.c_str());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(const Args&), int N>
PyCFunction fast() {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>));
}

PyMethodDef methods[] = {{"block_tables", fast<block_tables, 10>(), METH_FASTCALL, nullptr},
                         {"cache_write", fast<cache_write, 13>(), METH_FASTCALL, nullptr},
                         {"attention_paged", fast<attention_paged, 10>(), METH_FASTCALL, nullptr},
                         {"gated_delta_rule_step", fast<gated_delta_rule_step, 16>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__binding() { return PyModule_Create(&module); }
