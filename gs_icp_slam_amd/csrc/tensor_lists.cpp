// Python module _tensor_lists: lists of torch tensors -> the host arrays that the many-tensor entry points of the C ABI take (addresses, element counts, dtype codes), checked.
// Host code only.  Why native: a step over a hundred small tensors is bound by the host, and five Python calls per tensor and list (device, dtype, contiguity, size, address;
// ~0.2 us together) cost more than the kernel; here they are a few loads.
//
//   pack(what, names, rules, list, ...) -> (device index, whether it is the current one, its current stream, n, address, keep)
//   wrote(keep, which)                  after a launch: raises the version counters of the tensors that it writes
//
// One rule (a character) and one name (for the errors) per list; the first list has rule 'p' or 'c' and says device, length and element counts:
//   p  float32 / bfloat16 / float16 (their codes are recorded)      g  the first list's dtype, read only      f  float32         h  int16
//   b  int16, one element per 128 of the first list's               m  float32 or None                        c  int16 (as p, codes 0)
// At `address` (kept alive by `keep`, which holds the lists too): for each list n 8-byte addresses (0 for None and for empty tensors), then n int64 element counts, then n int32 codes.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <cstring>
#include <exception>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {

constexpr int64_t BLOCK = 128;

struct Refs {      // fast-sequence views of the lists, released on every way out
    PyObject* seq[16];
    int n = 0;
    ~Refs() { for (int i = 0; i < n; ++i) Py_DECREF(seq[i]); }
};

PyObject* refuse(const char* what, const char* name, const char* why) {
    PyErr_Format(PyExc_RuntimeError, "%s: %s %s", what, name, why);
    return nullptr;
}

PyObject* pack(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    const int lists = (int)nargs - 3;
    if (lists < 1 || lists > 16) { PyErr_SetString(PyExc_TypeError, "pack(what, names, rules, list, ...): 1 to 16 lists"); return nullptr; }
    const char* what = PyUnicode_AsUTF8(args[0]);
    Py_ssize_t n_rules = 0;
    const char* rules = PyUnicode_AsUTF8AndSize(args[2], &n_rules);
    if (!what || !rules) return nullptr;
    if (!PyTuple_Check(args[1]) || PyTuple_GET_SIZE(args[1]) != lists || n_rules != lists || (rules[0] != 'p' && rules[0] != 'c')) {
        PyErr_SetString(PyExc_TypeError, "pack: one name and one rule per list, the first 'p' or 'c'");
        return nullptr;
    }
    Refs refs;
    PyObject* keep = nullptr;
    try {
        for (int l = 0; l < lists; ++l) {
            PyObject* s = PySequence_Fast(args[3 + l], "pack: not a list of tensors");
            if (!s) return nullptr;
            refs.seq[refs.n++] = s;
        }
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(refs.seq[0]);
        if (n < 1 || n > (1 << 24)) return refuse(what, PyUnicode_AsUTF8(PyTuple_GET_ITEM(args[1], 0)), "must be a list of 1 to 2^24 tensors");
        keep = PyBytes_FromStringAndSize(nullptr, n * (8 * lists + 8 + 4));
        if (!keep) return nullptr;
        char* base = PyBytes_AS_STRING(keep);
        uint64_t* address = (uint64_t*)base;
        int64_t* numel = (int64_t*)(base + 8 * n * lists);
        int32_t* code = (int32_t*)(base + 8 * n * (lists + 1));
        int device = -1;
        for (int l = 0; l < lists; ++l) {
            const char* name = PyUnicode_AsUTF8(PyTuple_GET_ITEM(args[1], l));
            const char rule = rules[l];
            const char* why = nullptr;
            if (!name) { Py_DECREF(keep); return nullptr; }
            if (PySequence_Fast_GET_SIZE(refs.seq[l]) != n) {
                PyErr_Format(PyExc_RuntimeError, "%s: %zd %s for a list of %zd", what, PySequence_Fast_GET_SIZE(refs.seq[l]), name, n);
                Py_DECREF(keep);
                return nullptr;
            }
            PyObject** item = PySequence_Fast_ITEMS(refs.seq[l]);
            for (Py_ssize_t i = 0; i < n && !why; ++i) {
                uint64_t& out = address[l * n + i];
                if (rule == 'm' && item[i] == Py_None) { out = 0; continue; }
                if (!THPVariable_Check(item[i])) { why = "must be tensors"; break; }
                const at::Tensor& t = THPVariable_Unpack(item[i]);
                const at::ScalarType dt = t.scalar_type();
                if (!t.is_cuda()) { why = "must live on the HIP device (gfx950): there is no CPU path"; break; }
                if (t.layout() != at::kStrided || !t.is_contiguous()) { why = "must be contiguous"; break; }
                if (t.is_neg()) { why = "must not be negated lazily (resolve_neg())"; break; }      // the memory holds the other sign
                if (device < 0) device = t.get_device();
                if (t.get_device() != device) { why = "must live on one device"; break; }
                if (l == 0) {
                    numel[i] = t.numel();
                    if (rule == 'c') code[i] = 0;
                    else if (dt == at::kFloat) code[i] = 0;
                    else if (dt == at::kBFloat16) code[i] = 1;
                    else if (dt == at::kHalf) code[i] = 2;
                    else { why = "must be float32, bfloat16 or float16"; break; }
                }
                const int64_t want = rule == 'b' ? (numel[i] + BLOCK - 1) / BLOCK : numel[i];
                if (t.numel() != want) { why = rule == 'b' ? "have one element per 128 of the moments" : "have the wrong number of elements"; break; }
                const bool ok = rule == 'p' ? true
                                : rule == 'g' ? dt == (code[i] == 0 ? at::kFloat : code[i] == 1 ? at::kBFloat16 : at::kHalf)
                                : (rule == 'f' || rule == 'm') ? dt == at::kFloat
                                                               : dt == at::kShort;
                if (!ok) { why = "have the wrong dtype"; break; }
                out = t.numel() == 0 ? 0 : (uint64_t)(rule == 'g' ? t.const_data_ptr() : t.data_ptr());
            }
            if (why) { Py_DECREF(keep); return refuse(what, name, why); }
        }
        const unsigned long long stream = (unsigned long long)(uintptr_t)c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream();
        PyObject* current = c10::hip::current_device() == device ? Py_True : Py_False;
        PyObject* alive = PyTuple_New(1 + lists);      // also the tensors that an iterator has made: nothing else may hold them
        if (!alive) { Py_DECREF(keep); return nullptr; }
        PyTuple_SET_ITEM(alive, 0, keep);
        for (int l = 0; l < lists; ++l) { Py_INCREF(refs.seq[l]); PyTuple_SET_ITEM(alive, 1 + l, refs.seq[l]); }
        return Py_BuildValue("(iOKnKN)", device, current, stream, n, (unsigned long long)(uintptr_t)base, alive);
    } catch (const std::exception& e) {
        Py_XDECREF(keep);
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// The tensors of the lists whose bit is set in `which` were written: autograd must notice when a backward meets one that it saved before.
PyObject* wrote(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    const long which = nargs == 2 && PyTuple_Check(args[0]) ? PyLong_AsLong(args[1]) : -1;
    if (which < 0) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "wrote(keep, which)");
        return nullptr;
    }
    try {
        for (Py_ssize_t l = 0; l + 1 < PyTuple_GET_SIZE(args[0]); ++l) {
            PyObject* seq = PyTuple_GET_ITEM(args[0], l + 1);
            if (!(which >> l & 1) || !(PyList_Check(seq) || PyTuple_Check(seq))) continue;
            for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq); ++i) {
                PyObject* item = PySequence_Fast_GET_ITEM(seq, i);
                if (!THPVariable_Check(item)) continue;
                const at::Tensor& t = THPVariable_Unpack(item);
                if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
            }
        }
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"pack", (PyCFunction)(void (*)(void))pack, METH_FASTCALL, "pack(what, names, rules, list, ...) -> (device index, current, stream, n, address, keep)"},
                         {"wrote", (PyCFunction)(void (*)(void))wrote, METH_FASTCALL, "wrote(keep, which): raises the version counters of the lists whose bit is set in which"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_lists", "lists of torch tensors as host arrays of the C ABI", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_lists(void) { return PyModule_Create(&module); }
