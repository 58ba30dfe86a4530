// The Python mirror's call path in native code: ruy_amd.api.mul hands its
// objects over here, where their fields are gathered into the plain structs of
// c_api.h and ruyamd_mul is called. Filling four ctypes structures field by
// field and calling through ctypes took 2.4 us of a call whose launch takes
// 2.4 and whose kernel, for the smallest products, takes no more than both.
//
// Fields are read from the instances' dictionaries, where the classes of
// api.py keep them; an instance that does not have them there (a subclass with
// properties, say) is left to the Python code (kNotHandled).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <cstring>
#include <initializer_list>

#include "ruy_amd/c_api.h"

namespace {

using MulFunction = int (*)(ruyamd_ctx*, const ruyamd_mat*, const ruyamd_mat*, const ruyamd_mul_params*,
                            const ruyamd_mat*);
MulFunction mul_function = nullptr;
PyTypeObject* matrix_type = nullptr;
PyTypeObject* layout_type = nullptr;
PyTypeObject* params_type = nullptr;

template <typename Lhs>
using GroupedFunction = int (*)(ruyamd_ctx*, const Lhs*, const ruyamd_mat*, const ruyamd_groups*,
                                const ruyamd_mul_params*, const ruyamd_mat*);
uintptr_t grouped_functions[3] = {};  // ruyamd_mul_grouped, ruyamd_mul_grouped_depth, ruyamd_mul_int4
PyTypeObject* groups_type = nullptr;
PyTypeObject* int4_type = nullptr;

#define RUYAMD_NAMES(X)                                                                                        \
  X(dtype) X(data) X(layout) X(zero_point) X(cache_policy) X(rows) X(cols) X(stride) X(order) X(data_ptr)      \
  X(ctypes) X(bias) X(_perchannel) X(_mf) X(_me) X(_mf_pc) X(_me_pc) X(clamp_min) X(clamp_max) X(accum_dtype) \
  X(dst_dtype) X(channel_dimension) X(_rounding_log2) X(offsets) X(count) X(matrix_stride) X(bias_stride)      \
  X(group_size) X(scales) X(scale_dtype) X(zero_points) X(row_bytes) X(scale_stride) X(matrix_bytes)          \
  X(scales_matrix_stride)
#define RUYAMD_DECLARE(name) PyObject* name_##name;
RUYAMD_NAMES(RUYAMD_DECLARE)

// What a step of the conversion came to.
enum Outcome { kDone, kNotHandled, kError };

// A reference of our own. Asking a buffer for its address or a value for its
// float may run any code, also code that takes that object out of the instance
// it was found in, or the instance's dictionary away.
class Ref {
 public:
  explicit Ref(PyObject* borrowed) : p_(borrowed) { Py_XINCREF(p_); }
  ~Ref() { Py_XDECREF(p_); }
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
  operator PyObject*() const { return p_; }

 private:
  PyObject* p_;
};

// A field of an instance; null if it is not in the dictionary (or there is none).
Ref Field(PyObject* dict, PyObject* name) { return Ref(dict ? PyDict_GetItemWithError(dict, name) : nullptr); }

Ref DictOf(PyObject* object) {
  PyObject** p = _PyObject_GetDictPtr(object);
  return Ref(p ? *p : nullptr);
}

// Only Python integers are taken here (as ctypes does, bits beyond the field's
// are dropped); anything else is left to the Python code.
bool Integer(PyObject* dict, PyObject* name, uint64_t* out) {
  const Ref v = Field(dict, name);
  if (!v || !PyLong_Check(v)) return false;
  *out = PyLong_AsUnsignedLongLongMask(v);
  return true;
}

// api._address: None, an integer, a tensor or an array.
Outcome Address(PyObject* buffer, void** out) {
  if (buffer == Py_None) {
    *out = nullptr;
    return kDone;
  }
  if (PyLong_Check(buffer)) {
    *out = reinterpret_cast<void*>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLongMask(buffer)));
    return kDone;
  }
  PyObject* value = PyObject_CallMethodNoArgs(buffer, name_data_ptr);
  if (!value) {
    if (!PyErr_ExceptionMatches(PyExc_AttributeError)) return kError;
    PyErr_Clear();
    PyObject* ctypes = PyObject_GetAttr(buffer, name_ctypes);
    if (!ctypes) {
      PyErr_Clear();
      return kNotHandled;  // (the Python code raises)
    }
    value = PyObject_GetAttr(ctypes, name_data);
    Py_DECREF(ctypes);
    if (!value) return kError;
  }
  if (!PyLong_Check(value)) {
    Py_DECREF(value);
    return kNotHandled;
  }
  *out = reinterpret_cast<void*>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLongMask(value)));
  Py_DECREF(value);
  return kDone;
}

Outcome Matrix(PyObject* object, ruyamd_mat* m) {
  if (Py_TYPE(object) != matrix_type) return kNotHandled;
  const Ref dict = DictOf(object);
  const Ref layout = Field(dict, name_layout);
  const Ref data = Field(dict, name_data);
  if (!layout || !data || Py_TYPE(layout) != layout_type) return kNotHandled;
  const Ref shape = DictOf(layout);
  uint64_t rows, cols, stride, order, zero_point, dtype, policy;
  if (!Integer(shape, name_rows, &rows) || !Integer(shape, name_cols, &cols) ||
      !Integer(shape, name_stride, &stride) || !Integer(shape, name_order, &order) ||
      !Integer(dict, name_zero_point, &zero_point) || !Integer(dict, name_dtype, &dtype) ||
      !Integer(dict, name_cache_policy, &policy))
    return kNotHandled;
  m->rows = static_cast<int32_t>(rows);
  m->cols = static_cast<int32_t>(cols);
  m->stride = static_cast<int32_t>(stride);
  m->zero_point = static_cast<int32_t>(zero_point);
  m->order = static_cast<uint8_t>(order);
  m->dtype = static_cast<uint8_t>(dtype);
  m->cache_policy = static_cast<uint8_t>(policy);
  m->reserved = 0;
  return Address(data, &m->data);
}

Outcome Params(PyObject* object, ruyamd_mul_params* p, uint64_t* dst_dtype) {
  if (Py_TYPE(object) != params_type) return kNotHandled;
  const Ref dict = DictOf(object);
  const Ref perchannel = Field(dict, name__perchannel);
  uint64_t accum, channel, rounding;
  if (!perchannel || !PyBool_Check(perchannel) || !Integer(dict, name_accum_dtype, &accum) ||
      !Integer(dict, name_dst_dtype, dst_dtype) || !Integer(dict, name_channel_dimension, &channel) ||
      !Integer(dict, name__rounding_log2, &rounding))
    return kNotHandled;
  std::memset(p, 0, sizeof(*p));
  p->accum_dtype = static_cast<uint8_t>(accum);
  p->channel_dimension = static_cast<uint8_t>(channel);
  p->perchannel_buffers_capacity_rounding_log2 = static_cast<uint8_t>(rounding);
  const Ref clamp_min = Field(dict, name_clamp_min);
  const Ref clamp_max = Field(dict, name_clamp_max);
  if (!clamp_min || !clamp_max) return kNotHandled;
  p->clamp_min = PyFloat_AsDouble(clamp_min);
  p->clamp_max = PyFloat_AsDouble(clamp_max);
  if (PyErr_Occurred()) return kError;
  const Ref bias = Field(dict, name_bias);
  if (!bias) return kNotHandled;
  void* address = nullptr;
  if (Outcome o = Address(bias, &address)) return o;
  p->bias = address;
  if (perchannel == Py_True) {
    const Ref mf = Field(dict, name__mf_pc);
    const Ref me = Field(dict, name__me_pc);
    if (!mf || !me) return kNotHandled;
    if (Outcome o = Address(mf, &address)) return o;
    p->multiplier_fixedpoint_perchannel = static_cast<const int32_t*>(address);
    if (Outcome o = Address(me, &address)) return o;
    p->multiplier_exponent_perchannel = static_cast<const int32_t*>(address);
  } else {
    uint64_t mf, me;
    if (!Integer(dict, name__mf, &mf) || !Integer(dict, name__me, &me)) return kNotHandled;
    p->multiplier_fixedpoint = static_cast<int32_t>(mf);
    p->multiplier_exponent = static_cast<int32_t>(me);
  }
  return kDone;
}

// mul(lhs, rhs, mul_params, context address, dst): the return code, or None if
// the objects are not handled here.
PyObject* Mul(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 5 || !mul_function) {
    PyErr_SetString(PyExc_TypeError, "mul(lhs, rhs, mul_params, context address, dst)");
    return nullptr;
  }
  ruyamd_mat lhs, rhs, dst;
  ruyamd_mul_params params;
  uint64_t dst_dtype = 0;
  Outcome o = Params(args[2], &params, &dst_dtype);
  if (o == kDone) o = Matrix(args[0], &lhs);
  if (o == kDone) o = Matrix(args[1], &rhs);
  if (o == kDone) o = Matrix(args[4], &dst);
  if (o == kError) return nullptr;
  if (o == kNotHandled || dst_dtype != dst.dtype || !PyLong_Check(args[3])) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  ruyamd_ctx* ctx = reinterpret_cast<ruyamd_ctx*>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLongMask(args[3])));
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = mul_function(ctx, &lhs, &rhs, &params, &dst);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

Outcome Groups(PyObject* object, ruyamd_groups* g) {
  if (Py_TYPE(object) != groups_type) return kNotHandled;
  const Ref dict = DictOf(object);
  const Ref offsets = Field(dict, name_offsets);
  uint64_t count, matrix_stride, bias_stride;
  if (!offsets || !Integer(dict, name_count, &count) || !Integer(dict, name_matrix_stride, &matrix_stride) ||
      !Integer(dict, name_bias_stride, &bias_stride))
    return kNotHandled;
  g->count = static_cast<int32_t>(count);
  g->reserved = 0;
  g->matrix_stride = static_cast<int64_t>(matrix_stride);
  g->bias_stride = static_cast<int64_t>(bias_stride);
  void* address = nullptr;
  if (Outcome o = Address(offsets, &address)) return o;
  g->offsets = static_cast<const int32_t*>(address);
  return kDone;
}

Outcome Int4(PyObject* object, ruyamd_int4_mat* m) {
  if (Py_TYPE(object) != int4_type) return kNotHandled;
  const Ref dict = DictOf(object);
  const Ref data = Field(dict, name_data);
  const Ref scales = Field(dict, name_scales);
  const Ref zero_points = Field(dict, name_zero_points);
  uint64_t rows, cols, group_size, row_bytes, scale_stride, scale_dtype, matrix_bytes, scales_matrix_stride;
  if (!data || !scales || !zero_points || !Integer(dict, name_rows, &rows) || !Integer(dict, name_cols, &cols) ||
      !Integer(dict, name_group_size, &group_size) || !Integer(dict, name_row_bytes, &row_bytes) ||
      !Integer(dict, name_scale_stride, &scale_stride) || !Integer(dict, name_scale_dtype, &scale_dtype) ||
      !Integer(dict, name_matrix_bytes, &matrix_bytes) ||
      !Integer(dict, name_scales_matrix_stride, &scales_matrix_stride))
    return kNotHandled;
  std::memset(m, 0, sizeof(*m));
  m->rows = static_cast<int32_t>(rows);
  m->cols = static_cast<int32_t>(cols);
  m->group_size = static_cast<int32_t>(group_size);
  m->row_bytes = static_cast<int32_t>(row_bytes);
  m->scale_stride = static_cast<int32_t>(scale_stride);
  m->scale_dtype = static_cast<uint8_t>(scale_dtype);
  m->matrix_bytes = static_cast<int64_t>(matrix_bytes);
  m->scales_matrix_stride = static_cast<int64_t>(scales_matrix_stride);
  void* address = nullptr;
  if (Outcome o = Address(data, &address)) return o;
  m->data = address;
  if (Outcome o = Address(scales, &address)) return o;
  m->scales = address;
  if (Outcome o = Address(zero_points, &address)) return o;
  m->zero_points = static_cast<const uint8_t*>(address);
  return kDone;
}

// mul_with_groups(which, lhs, rhs, groups, mul_params, context address, dst): as
// Mul, of the function number `which`.
PyObject* MulWithGroups(PyObject*, PyObject* const* args, Py_ssize_t count) {
  const long which = count == 7 && PyLong_Check(args[0]) ? PyLong_AsLong(args[0]) : -1;
  if (which < 0 || which > 2 || !grouped_functions[which]) {
    PyErr_SetString(PyExc_TypeError,
                    "mul_with_groups(which, lhs, rhs, groups, mul_params, context address, dst)");
    return nullptr;
  }
  ruyamd_mat lhs, rhs, dst;
  ruyamd_int4_mat int4;
  ruyamd_groups groups;
  ruyamd_mul_params params;
  uint64_t dst_dtype = 0;
  const bool has_groups = args[3] != Py_None;
  Outcome o = Params(args[4], &params, &dst_dtype);
  if (o == kDone) o = which == 2 ? Int4(args[1], &int4) : Matrix(args[1], &lhs);
  if (o == kDone) o = Matrix(args[2], &rhs);
  if (o == kDone && has_groups) o = Groups(args[3], &groups);
  if (o == kDone) o = Matrix(args[6], &dst);
  if (o == kError) return nullptr;
  if (o == kNotHandled || dst_dtype != dst.dtype || !PyLong_Check(args[5])) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  ruyamd_ctx* ctx = reinterpret_cast<ruyamd_ctx*>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLongMask(args[5])));
  const ruyamd_groups* g = has_groups ? &groups : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (which == 2)
    rc = reinterpret_cast<GroupedFunction<ruyamd_int4_mat>>(grouped_functions[2])(ctx, &int4, &rhs, g, &params, &dst);
  else
    rc = reinterpret_cast<GroupedFunction<ruyamd_mat>>(grouped_functions[which])(ctx, &lhs, &rhs, g, &params, &dst);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// bind_with_groups([addresses of the three functions], Groups, Int4Matrix)
PyObject* BindWithGroups(PyObject*, PyObject* args) {
  PyObject *addresses, *groups, *int4;
  if (!PyArg_ParseTuple(args, "O!O!O!", &PyList_Type, &addresses, &PyType_Type, &groups, &PyType_Type, &int4))
    return nullptr;
  if (PyList_GET_SIZE(addresses) != 3) {
    PyErr_SetString(PyExc_ValueError, "three addresses");
    return nullptr;
  }
  for (int i = 0; i < 3; ++i) {
    const unsigned long long address = PyLong_AsUnsignedLongLong(PyList_GET_ITEM(addresses, i));
    if (PyErr_Occurred()) return nullptr;
    grouped_functions[i] = static_cast<uintptr_t>(address);
  }
  for (PyObject* t : {groups, int4}) Py_INCREF(t);
  groups_type = reinterpret_cast<PyTypeObject*>(groups);
  int4_type = reinterpret_cast<PyTypeObject*>(int4);
  Py_RETURN_NONE;
}

// bind(address of ruyamd_mul, Matrix, Layout, MulParams)
PyObject* Bind(PyObject*, PyObject* args) {
  unsigned long long address = 0;
  PyObject *matrix, *layout, *params;
  if (!PyArg_ParseTuple(args, "KO!O!O!", &address, &PyType_Type, &matrix, &PyType_Type, &layout, &PyType_Type, &params))
    return nullptr;
  mul_function = reinterpret_cast<MulFunction>(static_cast<uintptr_t>(address));
  for (PyObject* t : {matrix, layout, params}) Py_INCREF(t);
  matrix_type = reinterpret_cast<PyTypeObject*>(matrix);
  layout_type = reinterpret_cast<PyTypeObject*>(layout);
  params_type = reinterpret_cast<PyTypeObject*>(params);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"mul", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(Mul)), METH_FASTCALL, nullptr},
    {"bind", Bind, METH_VARARGS, nullptr},
    {"mul_with_groups", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(MulWithGroups)), METH_FASTCALL,
     nullptr},
    {"bind_with_groups", BindWithGroups, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() {
#define RUYAMD_INTERN(name) \
  if (!(name_##name = PyUnicode_InternFromString(#name))) return nullptr;
  RUYAMD_NAMES(RUYAMD_INTERN)
  return PyModule_Create(&module);
}
