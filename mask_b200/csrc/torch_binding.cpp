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
    if (dim < 1 || classes < 1 || rows >= most || dim >= most || classes >= most)
        return raise("hidden and weight must have at least one column and fewer than 2^31 - 256 rows and columns");
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
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
