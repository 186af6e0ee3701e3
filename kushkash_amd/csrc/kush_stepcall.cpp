// The host side of the calls around a windowed serving step (Ops.decode and append_decode under a window,
// window_attention, block_table, step_maps, sample): the argument checks of their Python wrappers, the outputs and the
// library call in one native function each, as kush_fastcall.cpp has it for the step's other calls. In Python they
// cost 13-35 us, more than the launches of a small step.
//
// Each function returns its result, or None for anything that is not the plain, valid case: the caller then takes its
// Python path, which makes the same checks and raises the errors. Every pointer is read before the GIL is released.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include <cstdint>

#include "kushkash_amd_step.h"
#include "kushkash_amd_window.h"

namespace {

constexpr int64_t PAGE = 32, MOST = 1 << 30;

decltype(&kush_window_decode) g_decode = nullptr;
decltype(&kush_window_attend) g_attend = nullptr;
decltype(&kush_block_table) g_table = nullptr;
decltype(&kush_step_maps) g_maps = nullptr;
decltype(&kush_sample) g_sample = nullptr;
decltype(&kush_sample_scratch) g_scratch = nullptr;
PyObject* g_check = nullptr;             // raises the error of a library code

struct NotTaken {};
struct Failed {                          // a library code other than 0
    const char* name;
    int rc;
};

void need(bool ok) {
    if (!ok) throw NotTaken{};
}

const at::Tensor& tensor(PyObject* o) {
    need(THPVariable_CheckExact(o));
    const at::Tensor& t = THPVariable_Unpack(o);
    need(t.defined() && t.is_cuda() && t.layout() == c10::kStrided);
    return t;
}

// the device that every tensor of a call is on: the current one (others take the Python path, which switches to it)
c10::DeviceIndex checked_device(const at::Tensor& t) {
    static const c10::impl::DeviceGuardImplInterface* const impl = c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA);
    need(t.get_device() == impl->getDevice().index());
    return t.get_device();
}

const at::Tensor& on(PyObject* o, c10::DeviceIndex d) {
    const at::Tensor& t = tensor(o);
    need(t.get_device() == d);
    return t;
}

const at::Tensor& vec(PyObject* o, c10::DeviceIndex d, int64_t n, at::ScalarType type) {
    const at::Tensor& t = on(o, d);
    need(t.dim() == 1 && t.numel() == n && t.scalar_type() == type && t.is_contiguous());
    return t;
}

const at::Tensor& map2(PyObject* o, c10::DeviceIndex d) {
    const at::Tensor& t = on(o, d);
    need(t.dim() == 2 && t.scalar_type() == at::kInt && (t.size(1) <= 1 || t.stride(1) == 1));
    return t;
}

int64_t integer(PyObject* o, int64_t low, int64_t high) {
    need(PyLong_CheckExact(o));
    int over = 0;
    const int64_t x = PyLong_AsLongLongAndOverflow(o, &over);
    need(over == 0 && x >= low && x <= high);
    return x;
}

double number(PyObject* o, double low, double high) {
    double x = 0;
    if (PyFloat_CheckExact(o))
        x = PyFloat_AS_DOUBLE(o);
    else
        x = (double)integer(o, -MOST, MOST);
    need(x >= low && x <= high);
    return x;
}

template <typename T>
T* ptr(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) {
    return at::empty(size, like.options().dtype(type).requires_grad(false));
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }

// A contiguous tensor over part of buf's storage, without the dispatcher (a step's maps are eleven of them)
at::Tensor part_of(const at::Tensor& buf, at::IntArrayRef size, int64_t offset, at::ScalarType type = at::kInt) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(buf.storage()), buf.key_set(),
                                                            c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(size);
    return t;
}

#define CALL(NAME, EXPR)                  \
    do {                                  \
        int rc_;                          \
        Py_BEGIN_ALLOW_THREADS;           \
        rc_ = EXPR;                       \
        Py_END_ALLOW_THREADS;             \
        if (rc_ != 0) throw Failed{NAME, rc_}; \
    } while (0)

at::ScalarType type_of(int64_t dtype) { return dtype == 0 ? at::kFloat : (dtype == 1 ? at::kHalf : at::kBFloat16); }

const at::Tensor& rows(PyObject* o, c10::DeviceIndex d, int64_t H, int64_t D, at::ScalarType type, int64_t least) {
    const at::Tensor& t = on(o, d);
    need(t.dim() == 3 && t.size(0) >= least && t.size(1) == H && t.size(2) == D && t.stride(2) == 1 && t.stride(1) == D &&
         t.scalar_type() == type);
    return t;
}

// head_dim, bits, group, dtype code, device, sync address, sync slots, k, v (both None: decode alone), q, out, cache,
// block_table, seq_lens, tail_idx, tail_k, scale, n_splits, work, waves, order, rot, window, sinks, stream: True
PyObject* decode(PyObject* const* a) {
    const int64_t D = integer(a[0], 1, 256), bits = integer(a[1], 4, 8), G = integer(a[2], 1, MOST), dtype = integer(a[3], 0, 2);
    const at::Tensor &q = tensor(a[9]), &out = tensor(a[10]), &cache = tensor(a[11]), &tail = tensor(a[15]);
    const c10::DeviceIndex dev = checked_device(q);
    need(dev == integer(a[4], 0, 127) && out.get_device() == dev && cache.get_device() == dev && tail.get_device() == dev);
    const at::ScalarType type = type_of(dtype);
    need(tail.dim() == 4 && tail.size(2) == PAGE && tail.size(3) == D && tail.is_contiguous() && tail.scalar_type() == type);
    const int64_t S = q.dim() == 3 ? q.size(0) : -1, H = tail.size(1), e = cache.element_size();
    need(S >= 0 && q.size(1) == H * G && q.size(2) == D && q.is_contiguous() && q.scalar_type() == type &&
         out.sizes() == q.sizes() && out.is_contiguous() && out.scalar_type() == type && cache.dim() >= 2 && cache.size(1) >= H);
    const int64_t bs = cache.stride(0) * e, hs = cache.stride(1) * e;
    const at::Tensor &table = on(a[12], dev), &lens = on(a[13], dev), &tidx = on(a[14], dev);
    need(table.dim() == 2 && table.scalar_type() == at::kInt && table.stride(1) == 1 && table.size(0) >= S);
    for (const at::Tensor* t : {&lens, &tidx}) need(t->scalar_type() == at::kInt && t->is_contiguous() && t->numel() >= S);
    need(PyFloat_CheckExact(a[16]) && PyBool_Check(a[21]));
    const int64_t ns = integer(a[17], 1, 1 << 20), waves = integer(a[19], 0, 8), need_rows = S * H * ns * G;
    float *ml = nullptr, *po = nullptr;
    if (ns > 1) {                                            // merged in the launch, or left to the caller
        const at::Tensor& w = on(a[18], dev);
        need(w.scalar_type() == at::kFloat && w.is_contiguous() && w.numel() >= need_rows * (D + 2) &&
             S * H * ((G + 15) / 16) <= integer(a[6], 0, MOST));
        ml = ptr<float>(w);
        po = ml + 2 * need_rows;
    }
    const int32_t* order = nullptr;
    if (a[20] != Py_None) {
        const at::Tensor& o = on(a[20], dev);
        need(o.scalar_type() == at::kInt && o.is_contiguous() && o.numel() >= S);
        order = ptr<int32_t>(o);
    }
    const void *pk = nullptr, *pv = nullptr;
    int64_t ks = 0, vs = 0;
    if (a[7] != Py_None) {
        const at::Tensor &k = rows(a[7], dev, H, D, type, S), &v = rows(a[8], dev, H, D, type, S);
        pk = k.data_ptr();
        pv = v.data_ptr();
        ks = k.stride(0);
        vs = v.stride(0);
        const uint64_t b = k.element_size();
        need(G <= 16 && (((uint64_t)(uintptr_t)pk | (uint64_t)(uintptr_t)pv | ks * b | vs * b) & 15) == 0);
    }
    void *const pc = cache.data_ptr(), *const pt = tail.data_ptr(), *const pout = out.data_ptr();
    const void* const pq = q.data_ptr();
    need((((uint64_t)(uintptr_t)pc | (uint64_t)bs | (uint64_t)hs) & 15) == 0);
    const int32_t *const ptab = ptr<int32_t>(table), *const plen = ptr<int32_t>(lens), *const ptix = ptr<int32_t>(tidx);
    const int64_t row = table.stride(0), window = integer(a[22], 1, MOST), sinks = integer(a[23], 0, MOST);
    int32_t* const sync = ns > 1 ? (int32_t*)integer(a[5], 0, INT64_MAX) : nullptr;
    const float scale = (float)PyFloat_AS_DOUBLE(a[16]);
    const int rot = a[21] == Py_True;
    void* const stream = (void*)integer(a[24], 0, INT64_MAX);
    CALL("kush_window_decode",
         g_decode(D, bits, G, dtype, pq, pout, pc, bs, hs, pt, ptix, ptab, plen, row, H, scale, ns, ml, po, S, stream, pk, pv,
                  ks, vs, (int32_t)std::min<int64_t>(table.size(1), 1 << 30), sync, waves, order, rot, window, sinks));
    Py_RETURN_TRUE;
}

// (batch, row, head) strides of [.., rows, heads, dim]; a dim of one entry counts as packed
void strides_of(const at::Tensor& t, int64_t* st) {
    const int64_t n = t.dim(), D = t.size(n - 1);
    st[0] = n == 3 || t.size(0) == 1 ? 0 : t.stride(0);
    st[1] = t.size(n - 3) == 1 ? D : t.stride(n - 3);
    st[2] = t.size(n - 2) == 1 ? D : t.stride(n - 2);
}

void aligned(const at::Tensor& t, const int64_t* st) {
    need(t.stride(-1) == 1 && (uintptr_t)t.data_ptr() % 16 == 0);
    for (int i = 0; i < 3; ++i) need(st[i] >= 0 && st[i] % 8 == 0);
}

// q, k, v (of shapes that the plan is for), out or None, cu_q, cu_k (or None), scale, window, sinks, then the plan -- n_q,
// n_k, waves, chunk, partial rows, row tiles of ragged rows, sequences -- and the stream: the output
PyObject* attend(PyObject* const* a) {
    const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]);
    const c10::DeviceIndex dev = checked_device(q);
    const int64_t n = q.dim(), D = q.size(n - 1), Hq = q.size(n - 2), Hk = k.size(n - 2);
    need(k.get_device() == dev && v.get_device() == dev && (n == 3 || n == 4) && k.dim() == n && k.sizes() == v.sizes() &&
         (q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16) && k.scalar_type() == q.scalar_type() &&
         v.scalar_type() == q.scalar_type());
    int64_t st[15] = {};
    strides_of(q, st);
    strides_of(k, st + 3);
    strides_of(v, st + 6);
    aligned(q, st);
    aligned(k, st + 3);
    aligned(v, st + 6);
    for (int i : {4, 7}) need(st[i] >= D && st[i] <= (1 << 23));
    const int32_t *cq = nullptr, *ck = nullptr;
    const int64_t seqs = integer(a[15], 1, INT32_MAX), total = n == 4 ? seqs * q.size(1) : q.size(0);
    need(n == 3 || q.size(0) == seqs);
    if (n == 3) {
        const at::Tensor &x = on(a[4], dev), &y = on(a[5], dev);
        need(x.scalar_type() == at::kInt && y.scalar_type() == at::kInt && x.is_contiguous() && y.is_contiguous() &&
             x.numel() == seqs + 1 && y.numel() == seqs + 1);
        cq = ptr<int32_t>(x);
        ck = ptr<int32_t>(y);
    }
    at::Tensor out;
    if (a[3] == Py_None) {
        out = empty(q.sizes(), q.scalar_type(), q);
    } else {
        out = tensor(a[3]);
        need(!out.requires_grad());
        need(out.get_device() == dev && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type());
    }
    strides_of(out, st + 9);
    aligned(out, st + 9);
    const int64_t part_rows = integer(a[13], 0, INT64_MAX / 1024);
    at::Tensor part;
    if (part_rows) part = empty({part_rows * (D + 2)}, at::kFloat, q);
    float *const po = part_rows ? ptr<float>(part) : nullptr, *const ml = part_rows ? po + part_rows * D : nullptr;
    const int dtype = q.scalar_type() == at::kHalf ? 1 : 2;
    const int64_t window = integer(a[7], 1, MOST), sinks = integer(a[8], 0, MOST), n_q = integer(a[9], 1, MOST),
                  n_k = integer(a[10], 1, MOST), waves = integer(a[11], 4, 8), chunk = integer(a[12], 0, MOST),
                  row_tiles = integer(a[14], 0, INT32_MAX);
    const float scale = (float)number(a[6], 0.0, 1e30);
    need(scale > 0.0f);
    void* const stream = (void*)integer(a[16], 0, INT64_MAX);
    const void *const pq = q.data_ptr(), *const pk = k.data_ptr(), *const pv = v.data_ptr();
    void* const pout = out.data_ptr();
    CALL("kush_window_attend",
         g_attend(D, dtype, pq, pk, pv, pout, nullptr, st, cq, ck, n_q, n_k, total, seqs, Hk, Hq / Hk, scale, 0, waves, chunk, po,
                  ml, stream, window, sinks, row_tiles));
    return wrap(out);
}

// req_to_token, req, seq_lens, pages, out or None, stream: (table, lens, slots)
PyObject* block_table(PyObject* const* a) {
    const at::Tensor& map = tensor(a[0]);
    const c10::DeviceIndex dev = checked_device(map);
    map2(a[0], dev);
    const at::Tensor &req = on(a[1], dev), &lens = on(a[2], dev);
    const int64_t R = req.numel(), pages = integer(a[3], 0, 65535 * 256);
    for (const at::Tensor* t : {&req, &lens})
        need((t->scalar_type() == at::kInt || t->scalar_type() == at::kLong) && t->dim() == 1 && t->is_contiguous() && t->numel() == R);
    need(R > 0);
    at::Tensor table, l, s;
    if (a[4] == Py_None) {
        const at::Tensor buf = empty({R * (pages + 2)}, at::kInt, map);
        table = part_of(buf, {R, pages}, 2 * R);
        l = part_of(buf, {R}, 0);
        s = part_of(buf, {R}, R);
    } else {
        need(PyTuple_CheckExact(a[4]) && PyTuple_GET_SIZE(a[4]) == 3);
        table = map2(PyTuple_GET_ITEM(a[4], 0), dev);
        need(table.size(0) == R && table.size(1) == pages && (R == 1 || table.stride(0) >= pages));
        l = vec(PyTuple_GET_ITEM(a[4], 1), dev, R, at::kInt);
        s = vec(PyTuple_GET_ITEM(a[4], 2), dev, R, at::kInt);
    }
    const int32_t* const pm = ptr<int32_t>(map);
    const void *const pr = req.data_ptr(), *const pl = lens.data_ptr();
    int32_t *const pt = ptr<int32_t>(table), *const po = ptr<int32_t>(l), *const ps = ptr<int32_t>(s);
    const int wr = req.scalar_type() == at::kLong, wl = lens.scalar_type() == at::kLong;
    const int64_t ms = map.stride(0), m0 = map.size(0), m1 = map.size(1), ts = std::max(table.stride(0), pages);
    void* const stream = (void*)integer(a[5], 0, INT64_MAX);
    CALL("kush_block_table", g_table(pm, ms, m0, m1, pr, wr, pl, wl, R, pages, pt, ts, po, ps, stream));
    if (a[4] != Py_None) return Py_NewRef(a[4]);
    return Py_BuildValue("(NNN)", wrap(table), wrap(l), wrap(s));
}

// new_tokens, history, slots, block_table, (requests, tokens, keys, jobs, pages, tails, window, sinks), stream: the maps
PyObject* step_maps(PyObject* const* a) {
    const at::Tensor& nt = tensor(a[0]);
    const c10::DeviceIndex dev = checked_device(nt);
    int64_t z[8];
    need(PyTuple_CheckExact(a[4]) && PyTuple_GET_SIZE(a[4]) == 8);
    for (int i = 0; i < 8; ++i) z[i] = integer(PyTuple_GET_ITEM(a[4], i), 0, INT32_MAX);
    const int64_t R = z[0], tokens = z[1], jobs = z[3], pages = z[4], tails = z[5];
    need(R > 0);
    vec(a[0], dev, R, at::kInt);
    const at::Tensor &h = vec(a[1], dev, R, at::kInt), &sl = vec(a[2], dev, R, at::kInt), &bt = map2(a[3], dev);
    need(bt.size(0) >= R);
    // one buffer: the int32 arrays, then the int64 one 8-byte aligned
    const int64_t count[10] = {R + 1, R + 1, R, jobs, jobs, pages, pages, tails, 3 * tails, tokens};
    int64_t at[11] = {};
    for (int i = 0; i < 10; ++i) at[i + 1] = at[i] + count[i];
    const int64_t wide = at[10] + (at[10] & 1);
    const at::Tensor buf = empty({wide + 2 * tokens}, at::kInt, nt);
    int32_t* const p = ptr<int32_t>(buf);
    const int32_t *const pn = ptr<int32_t>(nt), *const ph = ptr<int32_t>(h), *const ps = ptr<int32_t>(sl), *const pb = ptr<int32_t>(bt);
    const int64_t row = bt.stride(0), cols = bt.size(1);
    void* const stream = (void*)integer(a[5], 0, INT64_MAX);
    CALL("kush_step_maps",
         g_maps(pn, ph, ps, pb, row, cols, R, z[6], z[7], jobs, pages, tails, tokens, p + at[0], p + at[1], p + at[2], p + at[3],
                p + at[4], p + at[5], p + at[6], p + at[7], p + at[8], p + at[9], (int64_t*)(p + wide), stream));
    PyObject* const got = PyTuple_New(11);
    if (!got) return nullptr;
    for (int i = 0; i < 10; ++i)
        PyTuple_SET_ITEM(got, i, wrap(i == 8 ? part_of(buf, {tails, 3}, at[8]) : part_of(buf, {count[i]}, at[i])));
    PyTuple_SET_ITEM(got, 10, wrap(part_of(buf, {tokens}, wide / 2, at::kLong)));
    return got;
}

// logits, uniforms, temperature, top_k, top_p, min_p, out or None, stream: the tokens
PyObject* sample(PyObject* const* a) {
    const at::Tensor& x = tensor(a[0]);
    const c10::DeviceIndex dev = checked_device(x);
    const at::ScalarType type = x.scalar_type();
    const int dtype = type == at::kFloat ? 0 : (type == at::kHalf ? 1 : 2);
    need((type == at::kFloat || type == at::kHalf || type == at::kBFloat16) && x.dim() == 2 && !x.requires_grad());
    const int64_t B = x.size(0), V = x.size(1), row = B > 1 ? x.stride(0) : V;
    need(B > 0 && V >= 1 && V <= (1 << 24) && (V == 1 || x.stride(1) == 1) && row >= 0);
    const at::Tensor& u = vec(a[1], dev, B, at::kFloat);
    double value[4] = {};
    const void* each[4] = {};
    const double high[4] = {1e30, (double)INT32_MAX, 1e300, 1e300};
    for (int i = 0; i < 4; ++i) {
        if (THPVariable_CheckExact(a[2 + i]))
            each[i] = vec(a[2 + i], dev, B, i == 1 ? at::kInt : at::kFloat).data_ptr();
        else
            value[i] = i == 1 ? (double)integer(a[3], 0, INT32_MAX) : number(a[2 + i], 0.0, high[i]);
    }
    const at::Tensor out = a[6] == Py_None ? empty({B}, at::kLong, x) : vec(a[6], dev, B, at::kLong);
    const int64_t bytes = g_scratch(B, V);
    const at::Tensor scratch = empty({bytes}, at::kByte, x);
    const void* const px = x.data_ptr();
    const float* const pu = ptr<float>(u);
    int64_t* const po = ptr<int64_t>(out);
    void *const pw = scratch.data_ptr(), *const stream = (void*)integer(a[7], 0, INT64_MAX);
    CALL("kush_sample", g_sample(dtype, px, row, B, V, pu, value[0], (const float*)each[0], (int32_t)value[1], (const int32_t*)each[1],
                                 value[2], (const float*)each[2], value[3], (const float*)each[3], po, pw, bytes, stream));
    return a[6] == Py_None ? wrap(out) : Py_NewRef(a[6]);
}

// A tensor without storage throws on its pointer, with the GIL held: not taken either
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N || g_check == nullptr) {
        PyErr_SetString(PyExc_TypeError, "kushkash_amd._stepcall: bad arguments, or not bound");
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Failed& f) {
        return PyObject_CallFunction(g_check, "si", f.name, f.rc);
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_Clear();                                       // the Python path meets it too, and raises torch's own
    } catch (...) {
        PyErr_Clear();
    }
    Py_RETURN_NONE;
}

// bind(check, addresses of kush_window_decode, kush_window_attend, kush_block_table, kush_step_maps, kush_sample,
// kush_sample_scratch)
PyObject* bind(PyObject*, PyObject* args) {
    long long f[6];
    PyObject* check;
    if (!PyArg_ParseTuple(args, "OLLLLLL", &check, &f[0], &f[1], &f[2], &f[3], &f[4], &f[5])) return nullptr;
    g_decode = (decltype(g_decode))f[0];
    g_attend = (decltype(g_attend))f[1];
    g_table = (decltype(g_table))f[2];
    g_maps = (decltype(g_maps))f[3];
    g_sample = (decltype(g_sample))f[4];
    g_scratch = (decltype(g_scratch))f[5];
    Py_INCREF(check);
    Py_XSETREF(g_check, check);
    Py_RETURN_NONE;
}

#define FAST(F, N) {#F, (PyCFunction)(void (*)(void))entry<F, N>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr}, FAST(decode, 25), FAST(attend, 17), FAST(block_table, 6),
                         FAST(step_maps, 6), FAST(sample, 8), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_stepcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__stepcall(void) {
    PyObject* m = PyModule_Create(&module);
    if (m) PyModule_AddIntConstant(m, "ABI", KUSH_FASTCALL_ABI);      // the library's revision it was built for
    return m;
}
