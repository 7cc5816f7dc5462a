// Python binding of the products and of the operators between them: checks the tensors, allocates results and scratch
// from torch's allocator and calls the C ABI, without building Python or ctypes objects on the way.  A product took 14 us
// of host time through ctypes; the smallest ones take the GPU 5.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "mask_b200.h"

namespace {

PyObject* raise(const char* what) {
    PyErr_SetString(PyExc_RuntimeError, what);
    return nullptr;
}

// NULL for None, else the tensor's address
bool pointer_of(PyObject* o, const void** out) {
    *out = nullptr;
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) return false;
    *out = THPVariable_Unpack(o).data_ptr();
    return true;
}

// The tensor must be a contiguous float32 CUDA tensor; messages as the package's own checks word them.
const at::Tensor* float_tensor(PyObject* o, const char* name) {
    const char* rule = "a CUDA tensor";
    if (THPVariable_Check(o)) {
        const at::Tensor& t = THPVariable_Unpack(o);
        rule = !t.is_cuda() ? "a CUDA tensor" : (!t.is_contiguous() ? "contiguous" : (t.scalar_type() != at::kFloat ? "float32" : nullptr));
        if (!rule) return &t;
    }
    PyErr_Format(PyExc_RuntimeError, "%s must be %s", name, rule);
    return nullptr;
}

// spmm(format, M, K, val_sidx, offsets, index, values, plan, dense, out or None, epilogue, whole_vectors) -> out, or an
// int: the status of a C-ABI call that failed.  whole_vectors: only N % 4 == 0 (else -1) and 16-byte aligned dense and
// out (else -2) are taken.
PyObject* product(PyObject* const* args, Py_ssize_t n_args) {
    if (n_args != 12) return raise("spmm takes 12 arguments");
    mask_matrix m{};
    m.format = (int32_t)PyLong_AsLong(args[0]);
    m.M = (int32_t)PyLong_AsLong(args[1]);
    m.K = (int32_t)PyLong_AsLong(args[2]);
    const void *sidx, *offsets;
    if (!pointer_of(args[3], &sidx) || !pointer_of(args[4], &offsets) || !pointer_of(args[5], &m.index) || !pointer_of(args[6], &m.values))
        return raise("the packed arrays must be tensors");
    m.val_sidx = static_cast<const int32_t*>(sidx);
    m.offsets = static_cast<const int32_t*>(offsets);
    const auto* plan = static_cast<const mask_plan*>(PyLong_AsVoidPtr(args[7]));
    const int epilogue = (int)PyLong_AsLong(args[10]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor* dense = float_tensor(args[8], "dense");
    if (!dense) return nullptr;
    if (dense->dim() != 2) return raise("dense must be 2-D");
    const int64_t K = dense->size(0), N = dense->size(1);
    if (K != m.K) {
        PyErr_Format(PyExc_RuntimeError, "dense has %lld rows, the matrix has %d columns", (long long)K, (int)m.K);
        return nullptr;
    }
    if (N > 0x7ffffffc) return raise("dense has too many columns");
    at::Tensor out;
    if (args[9] == Py_None) {
        out = at::empty({m.M, N}, dense->options());
    } else {
        const at::Tensor* given = float_tensor(args[9], "out");
        if (!given) return nullptr;
        if (given->dim() != 2 || given->size(0) != m.M || given->size(1) != N) return raise("out has the wrong shape");
        out = *given;
    }
    if (N > 0) {
        if (args[11] == Py_True) {
            if (N % 4) return PyLong_FromLong(-1);
            if ((reinterpret_cast<uintptr_t>(dense->data_ptr()) | reinterpret_cast<uintptr_t>(out.data_ptr())) & 15) return PyLong_FromLong(-2);
        }
        const int32_t n4 = (int32_t)((N + 3) & ~(int64_t)3);
        const float* B = static_cast<const float*>(dense->data_ptr());
        // freed to torch's allocator on return: it is reused in stream order
        at::Tensor pad, scratch;
        if (n4 != N || (reinterpret_cast<uintptr_t>(B) & 15)) pad = at::empty({K * n4}, dense->options());
        const size_t need = mask_plan_scratch_bytes(plan, n4);
        if (need) scratch = at::empty({(int64_t)need}, dense->options().dtype(at::kByte));
        float* C = static_cast<float*>(out.data_ptr());
        cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = mask_spmm(plan, &m, (int32_t)N, B, N, C, N, pad.defined() ? static_cast<float*>(pad.data_ptr()) : nullptr,
                       need ? scratch.data_ptr() : nullptr, need, epilogue, stream);
        Py_END_ALLOW_THREADS
        if (rc != MASK_OK) return PyLong_FromLong(rc);
    }
    if (args[9] != Py_None) {
        Py_INCREF(args[9]);
        return args[9];
    }
    return THPVariable_Wrap(std::move(out));
}

// A dense CUDA tensor of the current device (asked for once, -1 before), or nullptr with the exception set.
const at::Tensor* device_tensor(PyObject* o, const char* name, int dims, int* device) {
    if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda()) {
        PyErr_Format(PyExc_RuntimeError, "%s must be a CUDA tensor", name);
        return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.layout() != at::kStrided || t.dim() != dims) {
        PyErr_Format(PyExc_RuntimeError, "%s must be a dense %d-D tensor", name, dims);
        return nullptr;
    }
    if (t.is_neg()) {       // a view whose values have another sign than its memory
        PyErr_Format(PyExc_RuntimeError, "%s is a negative view: pass resolve_neg() of it", name);
        return nullptr;
    }
    if (*device < 0) *device = at::cuda::current_device();
    if (t.get_device() != *device) {
        PyErr_Format(PyExc_RuntimeError, "%s is on cuda:%d, the current device is cuda:%d", name, (int)t.get_device(), *device);
        return nullptr;
    }
    return &t;
}

// mask_dtype of a tensor, or -1 with the exception set
int dtype_of(const at::Tensor& t, const char* name) {
    if (t.scalar_type() == at::kFloat) return MASK_F32;
    if (t.scalar_type() == at::kBFloat16) return MASK_BF16;
    if (t.scalar_type() == at::kHalf) return MASK_F16;
    PyErr_Format(PyExc_RuntimeError, "%s must be float32, bfloat16 or float16", name);
    return -1;
}

// linear_xent(hidden, weight, labels, reduction, grad_scale, grads) -> loss or (loss, dhidden, dweight), or the status of
// a C-ABI call that failed.
PyObject* linear_xent_checked(PyObject* const* args, Py_ssize_t n_args) {
    if (n_args != 6) return raise("linear_xent takes 6 arguments");
    int device = -1;
    const at::Tensor* hidden = device_tensor(args[0], "hidden", 2, &device);
    if (!hidden) return nullptr;
    const at::Tensor* weight = device_tensor(args[1], "weight", 2, &device);
    if (!weight) return nullptr;
    const at::Tensor* labels = device_tensor(args[2], "labels", 1, &device);
    if (!labels) return nullptr;
    mask_head h{};
    h.dtype = dtype_of(*hidden, "hidden");
    if (h.dtype < 0) return nullptr;
    if (weight->scalar_type() != hidden->scalar_type()) return raise("weight must have hidden's dtype");
    if (labels->scalar_type() != at::kLong) return raise("labels must be int64");
    const int64_t rows = hidden->size(0), dim = hidden->size(1), classes = weight->size(1);
    if (weight->size(0) != dim) {
        PyErr_Format(PyExc_RuntimeError, "weight has %lld rows, hidden has %lld columns", (long long)weight->size(0), (long long)dim);
        return nullptr;
    }
    if (labels->size(0) != rows) {
        PyErr_Format(PyExc_RuntimeError, "there are %lld labels for %lld rows", (long long)labels->size(0), (long long)rows);
        return nullptr;
    }
    if (rows > 1 && labels->stride(0) != 1) return raise("labels must be contiguous");
    if (dim > 1 && hidden->stride(1) != 1) return raise("rows of hidden must be contiguous");
    constexpr int64_t most = ((int64_t)1 << 31) - 256;
    if (dim < 1 || classes < 1 || dim > (1 << 20) || rows >= most || classes >= most)
        return raise("hidden must have 1 to 2^20 columns, weight at least one, both fewer than 2^31 - 256 rows and columns");
    h.reduction = (int32_t)PyLong_AsLong(args[3]);
    h.grad_scale = (float)PyFloat_AsDouble(args[4]);
    const bool grads = PyObject_IsTrue(args[5]) == 1;
    if (PyErr_Occurred()) return nullptr;
    h.rows = rows;
    h.dim = (int32_t)dim;
    h.classes = (int32_t)classes;
    h.d_hidden = hidden->const_data_ptr();
    h.hidden_stride = hidden->stride(0);
    h.d_weight = weight->const_data_ptr();
    h.weight_dim_stride = weight->stride(0);
    h.weight_class_stride = weight->stride(1);
    h.d_labels = labels->const_data_ptr<int64_t>();
    const auto float_options = hidden->options().dtype(at::kFloat);
    at::Tensor loss = h.reduction == MASK_REDUCE_NONE ? at::empty({rows}, float_options) : at::empty({}, float_options), dhidden, dweight;
    h.d_loss = loss.mutable_data_ptr<float>();
    if (grads) {
        dhidden = at::empty({rows, dim}, hidden->options());
        // like the weight: the axis that is contiguous there
        dweight = h.weight_dim_stride == 1 && h.weight_class_stride != 1 ? at::empty({classes, dim}, weight->options()).t() : at::empty({dim, classes}, weight->options());
        h.d_dhidden = dhidden.mutable_data_ptr();
        h.dhidden_stride = dim;
        h.d_dweight = dweight.mutable_data_ptr();
        h.dweight_dim_stride = dweight.stride(0);
        h.dweight_class_stride = dweight.stride(1);
    }
    const size_t need = mask_linear_xent_scratch_bytes(&h);
    // freed to torch's allocator on return: it is reused in stream order
    at::Tensor scratch = at::empty({(int64_t)need}, float_options.dtype(at::kByte));
    cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = mask_linear_xent(&h, scratch.mutable_data_ptr(), need, stream);
    Py_END_ALLOW_THREADS
    if (rc != MASK_OK) return PyLong_FromLong(rc);
    if (!grads) return THPVariable_Wrap(std::move(loss));
    return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(loss)), THPVariable_Wrap(std::move(dhidden)), THPVariable_Wrap(std::move(dweight)));
}

// What both directions of group norm take: x, its result, the affine parameters and the batch's offsets.
bool norm_operands(mask_norm& n, PyObject* px, PyObject* groups, PyObject* weight, PyObject* bias, PyObject* offsets, PyObject* activation, PyObject* out,
                   int* device, const at::Tensor** x, at::Tensor& y) {
    *x = device_tensor(px, "x", 2, device);
    if (!*x) return false;
    n.dtype = dtype_of(**x, "x");
    if (n.dtype < 0) return false;
    const int64_t rows = (*x)->size(0), channels = (*x)->size(1), g = PyLong_AsLong(groups);
    n.activation = (int32_t)PyLong_AsLong(activation);
    if (PyErr_Occurred()) return false;
    if (channels < 1 || channels > (1 << 20) || rows >= ((int64_t)1 << 31)) return raise("x must have 1 to 2^20 columns and fewer than 2^31 rows"), false;
    if (g < 1 || channels % g) {
        PyErr_Format(PyExc_RuntimeError, "%lld channels are not a multiple of %lld groups", (long long)channels, (long long)g);
        return false;
    }
    if (channels > 1 && (*x)->stride(1) != 1) return raise("rows of x must be contiguous"), false;
    n.rows = rows;
    n.channels = (int32_t)channels;
    n.groups = (int32_t)g;
    n.d_x = (*x)->const_data_ptr();
    n.x_stride = (*x)->stride(0);
    const char* names[2] = {"weight", "bias"};
    PyObject* objects[2] = {weight, bias};
    const float** to[2] = {&n.d_weight, &n.d_bias};
    for (int i = 0; i < 2; i++) {
        if (objects[i] == Py_None) continue;
        const at::Tensor* t = device_tensor(objects[i], names[i], 1, device);
        if (!t) return false;
        if (t->scalar_type() != at::kFloat || t->size(0) != channels || !t->is_contiguous()) {
            PyErr_Format(PyExc_RuntimeError, "%s must be contiguous float32 with one value per channel", names[i]);
            return false;
        }
        *to[i] = t->const_data_ptr<float>();
    }
    n.graphs = 1;
    if (offsets != Py_None) {
        const at::Tensor* t = device_tensor(offsets, "offsets", 1, device);
        if (!t) return false;
        if (t->scalar_type() != at::kInt || !t->is_contiguous() || t->size(0) < 2 || t->size(0) > (1 << 24))
            return raise("offsets must be contiguous int32 with one entry more than there are graphs"), false;
        n.graphs = (int32_t)(t->size(0) - 1);
        n.d_offsets = t->const_data_ptr<int32_t>();
    }
    if (out == Py_None) {
        y = at::empty({rows, channels}, (*x)->options());
    } else {
        const at::Tensor* t = device_tensor(out, "out", 2, device);
        if (!t) return false;
        if (t->scalar_type() != (*x)->scalar_type() || t->size(0) != rows || t->size(1) != channels) return raise("out must have x's shape and dtype"), false;
        if ((channels > 1 && t->stride(1) != 1) || (rows > 1 && t->stride(0) < channels)) return raise("rows of out must be contiguous and apart"), false;
        y = *t;
    }
    n.d_y = y.mutable_data_ptr();
    n.y_stride = y.stride(0);
    return true;
}

int run_norm(const mask_norm& n, bool backward, const at::Tensor& x) {
    const size_t need = mask_group_norm_scratch_bytes(&n, backward);
    at::Tensor scratch = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
    cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = backward ? mask_group_norm_backward(&n, scratch.mutable_data_ptr(), need, stream) : mask_group_norm(&n, scratch.mutable_data_ptr(), need, stream);
    Py_END_ALLOW_THREADS
    return rc;
}

PyObject* result_of(PyObject* out, at::Tensor&& y) {
    if (out == Py_None) return THPVariable_Wrap(std::move(y));
    Py_INCREF(out);
    return out;
}

// group_norm(x, groups, weight, bias, offsets, eps, activation, out) -> (y, mean, rstd), or the status of a call that failed
PyObject* group_norm_checked(PyObject* const* args, Py_ssize_t n_args) {
    if (n_args != 8) return raise("group_norm takes 8 arguments");
    mask_norm n{};
    int device = -1;
    const at::Tensor* x;
    at::Tensor y;
    n.eps = (float)PyFloat_AsDouble(args[5]);
    if (PyErr_Occurred()) return nullptr;
    if (!(n.eps >= 0.f)) return raise("eps must not be negative");
    if (!norm_operands(n, args[0], args[1], args[2], args[3], args[4], args[6], args[7], &device, &x, y)) return nullptr;
    at::Tensor mean = at::empty({n.graphs, n.groups}, x->options().dtype(at::kFloat)), rstd = at::empty_like(mean);
    n.d_mean = mean.mutable_data_ptr<float>();
    n.d_rstd = rstd.mutable_data_ptr<float>();
    const int rc = run_norm(n, false, *x);
    if (rc != MASK_OK) return PyLong_FromLong(rc);
    return Py_BuildValue("(NNN)", result_of(args[7], std::move(y)), THPVariable_Wrap(std::move(mean)), THPVariable_Wrap(std::move(rstd)));
}

// group_norm_backward(grad, x, mean, rstd, groups, weight, bias, offsets, activation, out) -> (dx, dweight, dbias), or a status
PyObject* group_norm_backward_checked(PyObject* const* args, Py_ssize_t n_args) {
    if (n_args != 10) return raise("group_norm_backward takes 10 arguments");
    mask_norm n{};
    int device = -1;
    const at::Tensor* x;
    at::Tensor dx;
    if (!norm_operands(n, args[1], args[4], args[5], args[6], args[7], args[8], args[9], &device, &x, dx)) return nullptr;
    const at::Tensor* grad = device_tensor(args[0], "grad", 2, &device);
    if (!grad) return nullptr;
    if (grad->scalar_type() != x->scalar_type() || grad->size(0) != n.rows || grad->size(1) != n.channels) return raise("grad must have x's shape and dtype");
    if (n.channels > 1 && grad->stride(1) != 1) return raise("rows of grad must be contiguous");
    n.d_grad = grad->const_data_ptr();
    n.grad_stride = grad->stride(0);
    const char* names[2] = {"mean", "rstd"};
    float** to[2] = {&n.d_mean, &n.d_rstd};
    for (int i = 0; i < 2; i++) {
        const at::Tensor* t = device_tensor(args[2 + i], names[i], 2, &device);
        if (!t) return nullptr;
        if (t->scalar_type() != at::kFloat || t->size(0) != n.graphs || t->size(1) != n.groups || !t->is_contiguous()) {
            PyErr_Format(PyExc_RuntimeError, "%s must be contiguous float32 [graphs, groups]", names[i]);
            return nullptr;
        }
        *to[i] = const_cast<float*>(t->const_data_ptr<float>());   // read only
    }
    at::Tensor dweight = at::empty({n.channels}, x->options().dtype(at::kFloat)), dbias = at::empty_like(dweight);
    n.d_dweight = dweight.mutable_data_ptr<float>();
    n.d_dbias = dbias.mutable_data_ptr<float>();
    const int rc = run_norm(n, true, *x);
    if (rc != MASK_OK) return PyLong_FromLong(rc);
    return Py_BuildValue("(NNN)", result_of(args[9], std::move(dx)), THPVariable_Wrap(std::move(dweight)), THPVariable_Wrap(std::move(dbias)));
}

// Tensors without storage or strides (sparse ones, those of torch.func's transforms) throw already when they are asked
// for an address or whether they are contiguous.
template <PyObject* (*Body)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    try {
        return Body(args, n_args);
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

template <PyObject* (*Body)(PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name, const char* doc) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(guarded<Body>)), METH_FASTCALL, doc};
}

PyMethodDef methods[] = {
    method<product>("spmm", "out = A @ dense, or a status"),
    method<linear_xent_checked>("linear_xent", "loss, or (loss, dhidden, dweight), or a status"),
    method<group_norm_checked>("group_norm", "(y, mean, rstd), or a status"),
    method<group_norm_backward_checked>("group_norm_backward", "(dx, dweight, dbias), or a status"),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
