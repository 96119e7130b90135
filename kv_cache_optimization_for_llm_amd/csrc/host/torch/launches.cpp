// Launches whose kernels take less time than a look at their arguments in Python: their tensors are checked here and the kernel library's C
// entry is called from here, one native call from the caller's arguments to the launch.  us a call, checked in Python / here: adjusted
// logits of one row, 13 tensors, 10.4 / 4.1 (its kernel takes 4.0); rows of 64 requests, 10 tensors, 9.4 / 5.0 (5.0); pages of 64 requests 7.2 / 4.1 (3.1).
//
// What the calls mean stands in ops/kernels.py, where the same checks stand in Python: they run where a function here returns None - something
// is not as it should be, and the checks there say what - and where this module could not be built.  A number that is returned is the C entry's.
// Every function is called with the interpreter's lock held, with the device's number and its current stream as the last arguments.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>

namespace {

typedef long long ll;
struct {
    int (*adjust)(const ll *, float *, ll, const void *, int, ll, int, int, int, int, int, void *);
    int (*count)(unsigned char *, int *, int, int, const int *, const int *, int, void *);
    int (*sample)(const ll *, const float *, ll, int, int, unsigned, int *, void *, void *);
    ll (*sample_bytes)(int, int);
    int (*grow)(const ll *, int, int, int, int, int, void *);
    int (*rows)(const ll *, const ll *, int, int, int, int, void *);
} entry;

const at::Tensor *tensor(PyObject *o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// A contiguous tensor of this type and shape on the device, or None: its address.
bool take(PyObject *o, at::ScalarType type, at::IntArrayRef shape, int64_t device, ll &address) {
    address = 0;
    if (o == Py_None) return true;
    const at::Tensor *x = tensor(o);
    if (x == nullptr || !x->is_cuda() || x->layout() != at::kStrided || x->get_device() != device || x->scalar_type() != type ||
        x->sizes() != shape || !x->is_contiguous())
        return false;
    address = (ll)(uintptr_t)x->data_ptr();
    return true;
}

// A matrix whose rows' elements lie next to each other and whose rows do not overlap.
struct Matrix {
    char *address;
    int64_t rows, cols, stride;
    at::ScalarType type;
    int bytes;
};
bool take_matrix(PyObject *o, int64_t device, Matrix &m) {
    const at::Tensor *x = tensor(o);
    if (x == nullptr || !x->is_cuda() || x->layout() != at::kStrided || x->dim() != 2 || x->get_device() != device) return false;
    m.type = x->scalar_type();
    if (m.type != at::kFloat && m.type != at::kBFloat16) return false;
    m.rows = x->size(0), m.cols = x->size(1), m.bytes = m.type == at::kFloat ? 4 : 2;
    if ((m.cols > 1 && x->stride(1) != 1) || (m.rows > 1 && x->stride(0) < m.cols) || m.rows > INT_MAX || m.cols > INT_MAX) return false;
    m.stride = m.rows > 1 ? x->stride(0) : m.cols;
    m.address = (char *)x->data_ptr();
    return true;
}

// Elements of a vector; below 0: it is none.
int64_t length(PyObject *o) {
    const at::Tensor *x = tensor(o);
    return x != nullptr && x->dim() == 1 && x->size(0) <= INT_MAX ? x->size(0) : -1;
}
// Rows of a matrix; below 0: it is none.
int64_t height(PyObject *o) {
    const at::Tensor *x = tensor(o);
    return x != nullptr && x->dim() == 2 && x->size(0) <= INT_MAX && x->size(1) <= INT_MAX ? x->size(0) : -1;
}

bool whole(PyObject *o, ll &v) {
    if (!PyLong_Check(o)) return false;
    v = PyLong_AsLongLong(o);
    if (v != -1 || !PyErr_Occurred()) return true;
    PyErr_Clear();
    return false;
}
bool whole_int(PyObject *o, int &v) {
    ll wide;
    if (!whole(o, wide) || wide < INT_MIN || wide > INT_MAX) return false;
    v = (int)wide;
    return true;
}

struct Place {                          // the last two arguments
    ll device, stream;
    bool ok;
    Place(PyObject *const *args, Py_ssize_t n) { ok = whole(args[n - 2], device) && whole(args[n - 1], stream) && device >= 0; }
    void *on() const { return (void *)(uintptr_t)stream; }
};

template <typename F>
PyObject *guarded(F f) {
    try {
        int code;
        if (f(code)) return PyLong_FromLong(code);
    } catch (...) {
    }
    Py_RETURN_NONE;
}

// logits, out, row_seat, marks, counts, repetition, presence, frequency, (bias start, token, value) or None, allowed_row, allowed
PyObject *adjust_logits(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&](int &code) {
        if (n != 13) return false;
        const Place at(args, n);
        Matrix in, out;
        if (!at.ok || !take_matrix(args[0], at.device, in) || !take_matrix(args[1], at.device, out)) return false;
        if (out.type != at::kFloat || out.rows != in.rows || out.cols != in.cols) return false;
        PyObject *row_seat = args[2], *marks = args[3], *counts = args[4], *bias = args[8], *allowed_row = args[9], *allowed = args[10];
        const bool seated = marks != Py_None, counted = counts != Py_None, masked = allowed != Py_None;
        if (seated != (row_seat != Py_None) || (!seated && (counted || args[5] != Py_None)) ||
            (!counted && (args[6] != Py_None || args[7] != Py_None)) || masked != (allowed_row != Py_None))
            return false;
        const int64_t rows = in.rows, vocab = in.cols, words = (vocab + 31) / 32;
        const int64_t seats = seated ? height(marks) : 0, grammars = masked ? height(allowed) : 0;
        if ((seated && seats < 1) || (masked && grammars < 1)) return false;
        ll address[11];
        int64_t biases = 0;
        address[6] = address[7] = address[8] = 0;
        if (bias != Py_None) {
            if (!PyTuple_Check(bias) || PyTuple_GET_SIZE(bias) != 3) return false;
            PyObject *start = PyTuple_GET_ITEM(bias, 0), *token = PyTuple_GET_ITEM(bias, 1), *value = PyTuple_GET_ITEM(bias, 2);
            biases = length(token);
            if (biases < 0 || start == Py_None || value == Py_None || !take(start, at::kInt, {rows + 1}, at.device, address[6]) ||
                !take(token, at::kInt, {biases}, at.device, address[7]) || !take(value, at::kFloat, {biases}, at.device, address[8]))
                return false;
        }
        if (!take(row_seat, at::kInt, {rows}, at.device, address[0]) || !take(marks, at::kByte, {seats, vocab}, at.device, address[1]) ||
            !take(counts, at::kInt, {seats, vocab}, at.device, address[2]) || !take(args[5], at::kFloat, {rows}, at.device, address[3]) ||
            !take(args[6], at::kFloat, {rows}, at.device, address[4]) || !take(args[7], at::kFloat, {rows}, at.device, address[5]) ||
            !take(allowed_row, at::kInt, {rows}, at.device, address[9]) || !take(allowed, at::kInt, {grammars, words}, at.device, address[10]))
            return false;
        const bool itself = in.address == out.address && in.type == at::kFloat && in.stride == out.stride;
        if (rows > 0 && vocab > 0 && !itself && in.address < out.address + 4 * ((rows - 1) * out.stride + vocab) &&
            out.address < in.address + in.bytes * ((rows - 1) * in.stride + vocab))
            return false;
        code = entry.adjust(address, (float *)out.address, out.stride, in.address, in.type == at::kFloat ? 0 : 1, in.stride, (int)rows, (int)vocab,
                            (int)seats, (int)biases, (int)grammars, at.on());
        return true;
    });
}

// marks, counts or None, seats, tokens
PyObject *count_tokens(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&](int &code) {
        if (n != 6) return false;
        const Place at(args, n);
        const int64_t seats = height(args[0]), tokens = length(args[3]);
        if (!at.ok || seats < 0 || tokens < 0 || args[2] == Py_None) return false;
        const at::IntArrayRef table = tensor(args[0])->sizes();
        ll marks, counts, of, ids;
        if (!take(args[0], at::kByte, table, at.device, marks) || !take(args[1], at::kInt, table, at.device, counts) ||
            !take(args[2], at::kInt, {tokens}, at.device, of) || !take(args[3], at::kInt, {tokens}, at.device, ids))
            return false;
        code = entry.count((unsigned char *)marks, (int *)counts, (int)seats, (int)table[1], (const int *)of, (const int *)ids, (int)tokens, at.on());
        return true;
    });
}

// logits, out_tokens, inv_temperature, top_k, top_p, min_p, uniform, rng_key, rng_step, kept, logprob, host_tokens, seed
PyObject *sample_truncated(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&](int &code) {
        if (n != 15) return false;
        const Place at(args, n);
        Matrix in;
        ll seed;
        if (!at.ok || !take_matrix(args[0], at.device, in) || in.type != at::kFloat || !whole(args[12], seed)) return false;
        const bool given = args[6] != Py_None, key = args[7] != Py_None, step = args[8] != Py_None;
        if (args[1] == Py_None || args[2] == Py_None || (given ? key || step : !key || !step)) return false;
        ll address[10];
        static const at::ScalarType types[10] = {at::kInt, at::kFloat, at::kInt, at::kFloat, at::kFloat, at::kFloat, at::kInt, at::kInt, at::kInt, at::kFloat};
        for (int i = 0; i < 10; ++i)
            if (!take(args[1 + i], types[i], {in.rows}, at.device, address[i])) return false;
        int *host = nullptr;
        if (args[11] != Py_None) {
            const at::Tensor *x = tensor(args[11]);
            if (x == nullptr || x->is_cuda() || x->layout() != at::kStrided || x->scalar_type() != at::kInt || x->dim() != 1 || x->size(0) < in.rows ||
                !x->is_contiguous() || !x->is_pinned())
                return false;
            host = (int *)x->data_ptr();
        }
        const ll bytes = entry.sample_bytes((int)in.rows, (int)in.cols);
        at::Tensor space;               // (given back behind the launch: what takes it next runs behind it, on its stream)
        if (bytes > 0) space = at::empty({(int64_t)(bytes / 4)}, tensor(args[0])->options().dtype(at::kInt));
        code = entry.sample(address, (const float *)in.address, in.stride, (int)in.rows, (int)in.cols, (unsigned)seed, host,
                            bytes > 0 ? space.data_ptr() : nullptr, at.on());
        return true;
    });
}

// table, seats, held, lengths, pages, offsets, page_size
PyObject *grow_tables(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&](int &code) {
        if (n != 9) return false;
        const Place at(args, n);
        const int64_t rows = height(args[0]), entries = length(args[1]), pages = length(args[4]);
        int page_size;
        if (!at.ok || rows < 0 || entries < 1 || pages < 0 || !whole_int(args[6], page_size)) return false;
        const at::IntArrayRef table = tensor(args[0])->sizes();
        ll address[6];
        if (!take(args[0], at::kInt, table, at.device, address[0]) || !take(args[1], at::kInt, {entries}, at.device, address[1]) ||
            !take(args[2], at::kInt, {entries}, at.device, address[2]) || !take(args[3], at::kInt, {entries}, at.device, address[3]) ||
            !take(args[4], at::kInt, {pages}, at.device, address[4]) || !take(args[5], at::kInt, {entries + 1}, at.device, address[5]))
            return false;
        code = entry.grow(address, (int)rows, (int)table[1], (int)entries, page_size, (int)pages, at.on());
        return true;
    });
}

// lengths, starts, seats, tables, page_size, q_start, positions, tok_seat, slots
PyObject *step_rows(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&](int &code) {
        constexpr Py_ssize_t MOST = 8;
        if (n != 11) return false;
        const Place at(args, n);
        PyObject *tables = args[3], *slots = args[8];
        const int64_t entries = length(args[0]), tokens = length(args[6]);
        int page_size;
        if (!at.ok || entries < 0 || tokens < 0 || !whole_int(args[4], page_size) || !(PyList_Check(tables) || PyTuple_Check(tables)) ||
            !(PyList_Check(slots) || PyTuple_Check(slots)))
            return false;
        const Py_ssize_t groups = PySequence_Fast_GET_SIZE(tables);
        if (groups > MOST || PySequence_Fast_GET_SIZE(slots) != groups) return false;
        ll address[6 + 2 * MOST], size[2 * MOST + 1];
        if (!take(args[0], at::kInt, {entries}, at.device, address[0]) || !take(args[1], at::kInt, {entries}, at.device, address[1]) ||
            !take(args[2], at::kInt, {entries}, at.device, address[2]) || !take(args[5], at::kInt, {entries + 1}, at.device, address[3]) ||
            !take(args[6], at::kInt, {tokens}, at.device, address[4]) || !take(args[7], at::kInt, {tokens}, at.device, address[5]))
            return false;
        for (Py_ssize_t g = 0; g < groups; ++g) {
            PyObject *table = PySequence_Fast_GET_ITEM(tables, g);
            if (height(table) < 0) return false;
            const at::IntArrayRef shape = tensor(table)->sizes();
            size[2 * g] = shape[0], size[2 * g + 1] = shape[1];
            if (!take(table, at::kInt, shape, at.device, address[6 + 2 * g]) ||
                !take(PySequence_Fast_GET_ITEM(slots, g), at::kInt, {tokens}, at.device, address[7 + 2 * g]))
                return false;
        }
        code = entry.rows(address, size, (int)entries, (int)groups, page_size, (int)tokens, at.on());
        return true;
    });
}

// the addresses of the C entries: kva_adjust_logits, kva_count_tokens, kva_sample_truncated, its workspace's bytes, kva_grow_tables, kva_step_rows
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
    ll at[6];
    if (n != 6) {
        PyErr_SetString(PyExc_TypeError, "six addresses are needed");
        return nullptr;
    }
    for (int i = 0; i < 6; ++i)
        if (!whole(args[i], at[i]) || at[i] == 0) {
            PyErr_SetString(PyExc_TypeError, "an address is missing");
            return nullptr;
        }
    entry = {reinterpret_cast<decltype(entry.adjust)>(at[0]), reinterpret_cast<decltype(entry.count)>(at[1]),
             reinterpret_cast<decltype(entry.sample)>(at[2]), reinterpret_cast<decltype(entry.sample_bytes)>(at[3]),
             reinterpret_cast<decltype(entry.grow)>(at[4]), reinterpret_cast<decltype(entry.rows)>(at[5])};
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(adjust_logits), METHOD(count_tokens), METHOD(sample_truncated), METHOD(grow_tables), METHOD(step_rows),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "kva_launches", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_kva_launches() { return PyModule_Create(&module); }
