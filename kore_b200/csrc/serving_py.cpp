// The calls of kore_b200/serving.py on plain arguments: checks, results, workspace and launch without the interpreter.
//
// A function returns what its Python counterpart returns where every argument is as the operator takes it, and None where one
// is not (another type, shape, device or order, a refusal by the library): the caller then goes its own way, which copies what
// may be copied and says what is wrong with the rest.  A call of the append over 16 tokens takes the host 4.7 us, 13.4 us by way of
// the interpreter and ctypes (attention 4.0 and 9.5, a draw 5.4 and 13); 2.6 us of all of them are the launch.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/kore_b200.h"

namespace {

struct Library {
    decltype(&kb_qknorm_rope_kv) append32;
    decltype(&kb_qknorm_rope_kv4) append4;
    decltype(&kb_kv4_read) read;
    decltype(&kb_attn_kv4) attn;
    decltype(&kb_attn_kv4_workspace_bytes) attn_bytes;
    decltype(&kb_sample) sample;
} lib;

struct Unusual {};  // thrown where the caller has to look

void need(bool ok) {
    if (!ok) throw Unusual();
}
const at::Tensor &tensor(PyObject *o) {
    need(THPVariable_CheckExact(o));
    return THPVariable_Unpack(o);
}
// a tensor of this type and shape, in its natural order, on this GPU
const at::Tensor &tensor(PyObject *o, at::ScalarType type, at::IntArrayRef shape, int dev) {
    const at::Tensor &t = tensor(o);
    need(t.is_cuda() && t.get_device() == dev && t.scalar_type() == type && t.sizes() == shape && t.is_contiguous());
    return t;
}
template <typename T>
T *pointer(PyObject *o, at::ScalarType type, at::IntArrayRef shape, int dev) {
    return static_cast<T *>(tensor(o, type, shape, dev).data_ptr());
}
template <typename T>
T *pointer_or_null(PyObject *o, at::ScalarType type, at::IntArrayRef shape, int dev) {
    return o == Py_None ? nullptr : pointer<T>(o, type, shape, dev);
}
int whole(PyObject *o) {
    need(PyLong_CheckExact(o));
    const long long v = PyLong_AsLongLong(o);  // -1 and an error where it does not fit
    if (v == -1 && PyErr_Occurred()) PyErr_Clear();
    need(v >= 0 && v <= INT_MAX);
    return (int)v;
}
float real(PyObject *o) {
    need(PyFloat_CheckExact(o));
    return (float)PyFloat_AS_DOUBLE(o);
}
// the device of a matrix of floats whose rows are in order, and the distance of its rows
int rows(const at::Tensor &t, size_t &ld) {
    need(t.is_cuda() && t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) > 0 && t.size(1) > 0);
    need(t.stride(1) == 1 || t.size(1) == 1);
    need(t.size(0) == 1 || t.stride(0) >= t.size(1));
    ld = (size_t)(t.size(0) == 1 ? t.size(1) : t.stride(0));
    const int dev = t.get_device();
    need(dev == c10::cuda::current_device());
    return dev;
}
template <typename T>
T *data(const at::Tensor &t) {
    return static_cast<T *>(t.data_ptr());
}
at::Tensor fresh(at::IntArrayRef shape, const at::Tensor &like, at::ScalarType type = at::kFloat) {
    return at::empty(shape, at::TensorOptions().device(like.device()).dtype(type));
}
// the library's call on the device's current stream; the interpreter may go on meanwhile
template <typename F>
void call(int dev, F f) {
    const kb_stream stream = static_cast<kb_stream>(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(stream);
    Py_END_ALLOW_THREADS
    need(rc == KB_OK);
}

// the planes of a KV4Cache, which checked them
struct Planes {
    uint32_t *k_codes, *k_steps, *v_codes, *v_steps;
    int64_t seqs, kv, lmax;
    int dev;
    Planes() = default;
    explicit Planes(PyObject *held) {
        need(PyTuple_CheckExact(held) && PyTuple_GET_SIZE(held) == 4);
        uint32_t *at[4];
        for (int i = 0; i < 4; ++i) at[i] = data<uint32_t>(tensor(PyTuple_GET_ITEM(held, i)));
        k_codes = at[0]; k_steps = at[1]; v_codes = at[2]; v_steps = at[3];
        const at::Tensor &steps = tensor(PyTuple_GET_ITEM(held, 1));
        need(steps.dim() == 3);
        seqs = steps.size(0); kv = steps.size(1); lmax = steps.size(2);
        need(kv <= INT_MAX && lmax <= INT_MAX);
        dev = steps.get_device();
    }
};

// append(qkv, positions, cache_rows, cos, sin, caches, head_dim, n_heads, q_gamma, k_gamma, eps, q_out); caches: the planes, or a pair
PyObject *append(PyObject *const *a) {
    const at::Tensor &qkv = tensor(a[0]);
    size_t ld;
    const int dev = rows(qkv, ld);
    PyObject *caches = a[5];
    need(PyTuple_CheckExact(caches));
    const int heads = whole(a[7]);
    const int64_t n = qkv.size(0);
    int64_t seqs, kv, lmax, hd;
    const bool four = PyTuple_GET_SIZE(caches) == 4;
    Planes planes = four ? Planes(caches) : Planes();
    float *k = nullptr, *v = nullptr;
    if (four) {
        need(planes.dev == dev);
        seqs = planes.seqs; kv = planes.kv; lmax = planes.lmax; hd = whole(a[6]);
    } else {
        need(PyTuple_GET_SIZE(caches) == 2);
        const at::Tensor &kc = tensor(PyTuple_GET_ITEM(caches, 0));
        need(kc.dim() == 4 && kc.numel() > 0);
        seqs = kc.size(0); kv = kc.size(1); lmax = kc.size(2); hd = kc.size(3);
        k = pointer<float>(PyTuple_GET_ITEM(caches, 0), at::kFloat, kc.sizes(), dev);
        v = pointer<float>(PyTuple_GET_ITEM(caches, 1), at::kFloat, kc.sizes(), dev);
    }
    need(lmax <= INT_MAX && kv <= INT_MAX && hd <= 128 && qkv.size(1) == (heads + 2 * kv) * hd);
    const int *positions = pointer<int>(a[1], at::kInt, {n}, dev);
    const long long *cache_rows = pointer<long long>(a[2], at::kLong, {n}, dev);
    const at::Tensor &cos_t = tensor(a[3]);
    need(cos_t.dim() == 2 && cos_t.size(0) > 0);
    const int64_t max_pos = cos_t.size(0);
    const float *cos = pointer<float>(a[3], at::kFloat, {max_pos, hd / 2}, dev), *sin = pointer<float>(a[4], at::kFloat, {max_pos, hd / 2}, dev);
    const float *gq = pointer_or_null<float>(a[8], at::kFloat, {hd}, dev), *gk = pointer_or_null<float>(a[9], at::kFloat, {hd}, dev);
    const float eps = real(a[10]);
    const at::Tensor out = a[11] == Py_None ? fresh({n, heads, hd}, qkv) : tensor(a[11], at::kFloat, {n, heads, hd}, dev);
    call(dev, [&](kb_stream stream) {
        return four ? lib.append4(data<float>(qkv), ld, positions, cache_rows, cos, sin, max_pos, gq, gk, eps, n, heads, kv, hd, seqs, lmax,
                                  data<float>(out), planes.k_codes, planes.k_steps, planes.v_codes, planes.v_steps, stream)
                    : lib.append32(data<float>(qkv), ld, positions, cache_rows, cos, sin, max_pos, gq, gk, eps, n, heads, kv, hd, seqs, lmax,
                                   data<float>(out), k, v, stream);
    });
    return THPVariable_Wrap(out);
}

// read(planes, head_dim, cache_rows, k_out, v_out)
PyObject *read(PyObject *const *a) {
    const Planes p(a[0]);
    need(p.dev == c10::cuda::current_device());
    const int64_t hd = whole(a[1]);
    const at::Tensor &idx = tensor(a[2]);
    need(idx.dim() == 1 && idx.size(0) > 0);
    const int64_t n = idx.size(0);
    const long long *cache_rows = pointer<long long>(a[2], at::kLong, {n}, p.dev);
    const at::Tensor k = a[3] == Py_None ? fresh({n, p.kv, hd}, idx) : tensor(a[3], at::kFloat, {n, p.kv, hd}, p.dev);
    const at::Tensor v = a[4] == Py_None ? fresh({n, p.kv, hd}, idx) : tensor(a[4], at::kFloat, {n, p.kv, hd}, p.dev);
    call(p.dev, [&](kb_stream stream) {
        return lib.read(p.k_codes, p.k_steps, p.v_codes, p.v_steps, cache_rows, n, (int)p.kv, (int)hd, p.seqs, (int)p.lmax, data<float>(k),
                        data<float>(v), stream);
    });
    return Py_BuildValue("NN", THPVariable_Wrap(k), THPVariable_Wrap(v));
}

// attend(planes, head_dim, q, lens, scale, out)
PyObject *attend(PyObject *const *a) {
    const Planes p(a[0]);
    need(p.dev == c10::cuda::current_device());
    const int64_t hd = whole(a[1]);
    const at::Tensor &q = tensor(a[2]);
    need(q.dim() == 3 || q.dim() == 4);
    need(q.size(0) == p.seqs && q.size(-1) == hd && q.numel() > 0 && q.numel() <= (int64_t)INT_MAX * hd);
    const float *query = pointer<float>(a[2], at::kFloat, q.sizes(), p.dev);
    const int *lens = pointer<int>(a[3], at::kInt, {p.seqs}, p.dev);
    const float scale = real(a[4]);
    const int t = q.dim() == 3 ? 1 : (int)q.size(1), heads = (int)q.size(-2);
    const at::Tensor out = a[5] == Py_None ? fresh(q.sizes(), q) : tensor(a[5], at::kFloat, q.sizes(), p.dev);
    // the allocator orders its reuse by stream and keeps a captured graph's blocks to that graph
    const size_t bytes = lib.attn_bytes(p.seqs, t, heads, (int)p.kv, (int)hd, (int)p.lmax);
    const at::Tensor space = bytes ? fresh({(int64_t)bytes}, q, at::kByte) : at::Tensor();
    call(p.dev, [&](kb_stream stream) {
        return lib.attn(query, p.k_codes, p.k_steps, p.v_codes, p.v_steps, lens, p.seqs, t, heads, (int)p.kv, (int)hd, (int)p.lmax, scale,
                        data<float>(out), bytes ? space.data_ptr() : nullptr, bytes, stream);
    });
    return THPVariable_Wrap(out);
}

// sample(logits, u, temperature, top_k, top_p, min_p, return_logprobs, tokens)
PyObject *sample(PyObject *const *a) {
    const at::Tensor &logits = tensor(a[0]);
    size_t ld;
    const int dev = rows(logits, ld);
    const int64_t n = logits.size(0);
    const float *u = pointer<float>(a[1], at::kFloat, {n}, dev);
    const float *temperature = pointer_or_null<float>(a[2], at::kFloat, {n}, dev);
    const int *top_k = pointer_or_null<int>(a[3], at::kInt, {n}, dev);
    const float *top_p = pointer_or_null<float>(a[4], at::kFloat, {n}, dev), *min_p = pointer_or_null<float>(a[5], at::kFloat, {n}, dev);
    need(PyBool_Check(a[6]));
    const bool logs = a[6] == Py_True;
    const at::Tensor tokens = a[7] == Py_None ? fresh({n}, logits, at::kLong) : tensor(a[7], at::kLong, {n}, dev);
    const at::Tensor logprobs = logs ? fresh({n}, logits) : at::Tensor();
    call(dev, [&](kb_stream stream) {
        return lib.sample(data<float>(logits), n, logits.size(1), ld, temperature, top_k, top_p, min_p, u, data<long long>(tokens),
                          logs ? data<float>(logprobs) : nullptr, stream);
    });
    if (!logs) return THPVariable_Wrap(tokens);
    return Py_BuildValue("NN", THPVariable_Wrap(tokens), THPVariable_Wrap(logprobs));
}

template <PyObject *(*F)(PyObject *const *), int ARGS>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t count) {
    try {
        if (count == ARGS) return F(args);
    } catch (...) {  // torch's exceptions, too (no memory): the caller meets them again
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

// addresses of the library's functions, in the order of Library
PyObject *setup(PyObject *, PyObject *const *args, Py_ssize_t count) {
    void *at[6] = {};
    if (count != 6) return PyErr_Format(PyExc_TypeError, "setup: six addresses");
    for (int i = 0; i < 6; ++i) at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
    lib = {reinterpret_cast<decltype(lib.append32)>(at[0]), reinterpret_cast<decltype(lib.append4)>(at[1]), reinterpret_cast<decltype(lib.read)>(at[2]),
           reinterpret_cast<decltype(lib.attn)>(at[3]), reinterpret_cast<decltype(lib.attn_bytes)>(at[4]), reinterpret_cast<decltype(lib.sample)>(at[5])};
    Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef methods[] = {{"setup", fast(setup), METH_FASTCALL, nullptr},
                         {"append", fast(entry<append, 12>), METH_FASTCALL, nullptr},
                         {"read", fast(entry<read, 5>), METH_FASTCALL, nullptr},
                         {"attend", fast(entry<attend, 6>), METH_FASTCALL, nullptr},
                         {"sample", fast(entry<sample, 8>), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "kore_b200_serving", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_kore_b200_serving() { return PyModule_Create(&module); }
