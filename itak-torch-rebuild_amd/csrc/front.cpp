// The calls a serving program makes per layer and per round, from Python to the C ABI without ctypes: arguments are
// read where Python holds them and the library is entered with the interpreter released, as ctypes does.
//
// Bound: host instructions. A step of one launch takes 2.8 us of host time from C and of two 5.1; through ctypes, which
// converts every argument by its declared type, and the packing of the items in Python they took 4.3 and 7.5, and with
// two launches of 7.2 us of device time a decode forward was the host's to finish. Host time a layer, ctypes -> this: 8
// layers of one row at 4,096 7.65 -> 6.3 us, of preparing steps 8.65 -> 6.9, f32 8.2 -> 6.6.
//
// Only plain arguments are taken here: exact ints, floats and bools, items in lists or tuples, C-contiguous float32
// arrays, views and page tables as paged.py makes them. Whatever else a caller passes (numpy scalars, pointer objects, other sequences) is answered with kNotPlain before
// anything is called, and hip_compute.py or paged.py then makes the same call through ctypes with that module's conversions.
//
// The library's functions are bound by address (bind), so that this module serves whichever build is loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#define NPY_NO_DEPRECATED_API NPY_2_0_API_VERSION
#include <numpy/arrayobject.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "../../include/itak_hip_kv.h"

namespace {

constexpr long kNotPlain = -1;
constexpr Py_ssize_t kMostItems = 64;

decltype(&itak_attention_step_device) step_fn;
decltype(&itak_attention_prep_step_device) prep_step_fn;
decltype(&itak_kv_truncate) truncate_fn;
decltype(&itak_compute_attention) compute_fn;
decltype(&itak_gqa_attention) gqa_fn;
decltype(&itak_rotate_device) rotate_fn;
decltype(&itak_paged_set_batch) set_batch_fn;
decltype(&itak_paged_append_device) append_fn;
decltype(&itak_paged_attention_device) paged_attention_fn;
decltype(&itak_paged_step_device) paged_step_fn;
decltype(&itak_paged_set_batch_tree) set_batch_tree_fn;
decltype(&itak_paged_fit_tables_device) fit_fn;
decltype(&itak_paged_set_batch_device) set_batch_device_fn;
decltype(&itak_paged_batch_rows_device) batch_rows_fn;
decltype(&itak_paged_accept_device) accept_fn;
decltype(&itak_paged_keep_device) keep_fn;
PyTypeObject *cache_type;  // hip_compute.KvCache
PyTypeObject *rows_type;   // paged.Rows
PyObject *slot_name, *address_name, *rows_name, *channels_name;

// An exact int as ctypes takes it for an unsigned 64-bit argument or a pointer: modulo 2^64.
bool plain_u64(PyObject *o, uint64_t &v) {
    if (!PyLong_CheckExact(o)) return false;
    v = PyLong_AsUnsignedLongLongMask(o);
    return true;
}
template <typename T>
bool plain_ptr(PyObject *o, T *&p) {
    uint64_t v;
    if (!plain_u64(o, v)) return false;
    p = reinterpret_cast<T *>(uintptr_t(v));
    return true;
}
// An exact int that is an unsigned value of `bits` bits.
bool plain_within(PyObject *o, int bits, uint64_t &v) {
    if (!PyLong_CheckExact(o)) return false;
    v = PyLong_AsUnsignedLongLong(o);
    if (v == ~0ull && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return bits == 64 || v >> bits == 0;
}
bool plain_float(PyObject *o, float &f) {
    if (PyFloat_CheckExact(o)) {
        f = float(PyFloat_AS_DOUBLE(o));
        return true;
    }
    if (!PyLong_CheckExact(o)) return false;
    const double d = PyLong_AsDouble(o);
    if (d == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    f = float(d);
    return true;
}
// None is the default scale.
bool plain_scale(PyObject *o, float &f) {
    if (o != Py_None) return plain_float(o, f);
    f = NAN;
    return true;
}
bool plain_slot(PyObject *o, uint32_t &slot) {
    uint64_t v;
    if (Py_TYPE(o) == cache_type) {
        PyObject *s = PyObject_GetAttr(o, slot_name);
        if (!s) {
            PyErr_Clear();
            return false;
        }
        const bool ok = plain_within(s, 32, v);
        Py_DECREF(s);
        if (!ok) return false;
    } else if (!plain_within(o, 32, v)) {
        return false;
    }
    slot = uint32_t(v);
    return true;
}
bool plain_sequence(PyObject *o, PyObject **&at, Py_ssize_t &n) {
    if (!PyList_CheckExact(o) && !PyTuple_CheckExact(o)) return false;
    at = PySequence_Fast_ITEMS(o);
    n = PySequence_Fast_GET_SIZE(o);
    return true;
}
bool plain_items(PyObject *o, itak_batch_item *items, uint32_t &count) {
    PyObject **at;
    Py_ssize_t n;
    if (!plain_sequence(o, at, n) || n > kMostItems) return false;
    for (Py_ssize_t i = 0; i < n; ++i) {
        uint64_t rows;
        if (!PyTuple_CheckExact(at[i]) || PyTuple_GET_SIZE(at[i]) != 2 ||
            !plain_slot(PyTuple_GET_ITEM(at[i], 0), items[i].slot) || !plain_within(PyTuple_GET_ITEM(at[i], 1), 32, rows))
            return false;
        items[i].rows = uint32_t(rows);
    }
    count = uint32_t(n);
    return true;
}
// A C-contiguous array of native floats; its address is null where it is empty.
bool plain_array(PyObject *o, const float *&data, uint64_t &size) {
    if (!PyArray_CheckExact(o)) return false;
    PyArrayObject *a = reinterpret_cast<PyArrayObject *>(o);
    if (PyArray_TYPE(a) != NPY_FLOAT32 || !PyArray_ISCARRAY_RO(a)) return false;
    size = uint64_t(PyArray_SIZE(a));
    data = size ? static_cast<const float *>(PyArray_DATA(a)) : nullptr;
    return true;
}
bool int_of(PyObject *o, PyObject *name, int64_t &v) {
    PyObject *x = PyObject_GetAttr(o, name);
    if (!x) {
        PyErr_Clear();
        return false;
    }
    const bool ok = PyLong_CheckExact(x);
    if (ok) v = int64_t(PyLong_AsUnsignedLongLongMask(x));
    Py_DECREF(x);
    return ok;
}
// A paged.Rows of at least `need` rows of `head_dim` channels (or of a bare pointer, which says nothing of either): where its itak_rows lies.
bool plain_rows(PyObject *o, uint64_t need, uint64_t head_dim, const itak_rows *&rows) {
    int64_t at, have, channels;
    if (Py_TYPE(o) != rows_type || !int_of(o, address_name, at) || !int_of(o, rows_name, have) || !int_of(o, channels_name, channels))
        return false;
    rows = reinterpret_cast<const itak_rows *>(uintptr_t(at));
    return rows && (have < 0 || (uint64_t(have) >= need && uint64_t(channels) == head_dim));
}
// A C-contiguous run of 32-bit words.
bool plain_words(PyObject *o, const void *&data, Py_ssize_t &n) {
    if (!PyArray_CheckExact(o)) return false;
    PyArrayObject *a = reinterpret_cast<PyArrayObject *>(o);
    const int type = PyArray_TYPE(a);
    if ((type != NPY_UINT32 && type != NPY_INT32) || PyArray_NDIM(a) != 1 || !PyArray_ISCARRAY_RO(a)) return false;
    n = PyArray_SIZE(a);
    data = PyArray_DATA(a);
    return true;
}
PyObject *not_plain() { return PyLong_FromLong(kNotPlain); }
bool arity(Py_ssize_t got, Py_ssize_t want) {
    if (got != want) PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, got);
    return got == want;
}

// step(pool, layer, items, q, k, v, out, q_heads, scale, softcap) -> status
PyObject *step(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 10)) return nullptr;
    itak_pool *pool;
    const float *q, *k, *v;
    float *out, scale, softcap;
    uint64_t layer, heads;
    uint32_t count;
    itak_batch_item items[kMostItems];
    if (!plain_ptr(a[0], pool) || !plain_u64(a[1], layer) || !plain_items(a[2], items, count) || !plain_ptr(a[3], q) ||
        !plain_ptr(a[4], k) || !plain_ptr(a[5], v) || !plain_ptr(a[6], out) || !plain_u64(a[7], heads) ||
        !plain_scale(a[8], scale) || !plain_float(a[9], softcap))
        return not_plain();
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = step_fn(pool, layer, items, count, q, k, v, out, heads, scale, softcap);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

// prep_step(pool, layer, items, q, k, v, gate, out, q_heads, scale, softcap, q_norm, k_norm, eps, rope_base, interleaved,
// rotary_dim) -> status
PyObject *prep_step(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 17)) return nullptr;
    itak_pool *pool;
    const float *q, *k, *v, *gate;
    float *out, scale, softcap;
    uint64_t layer, heads, rotary;
    uint32_t count;
    itak_batch_item items[kMostItems];
    itak_prep_params prep{};
    if (!plain_ptr(a[0], pool) || !plain_u64(a[1], layer) || !plain_items(a[2], items, count) || !plain_ptr(a[3], q) ||
        !plain_ptr(a[4], k) || !plain_ptr(a[5], v) || !plain_ptr(a[6], gate) || !plain_ptr(a[7], out) ||
        !plain_u64(a[8], heads) || !plain_float(a[9], scale) || !plain_float(a[10], softcap) ||
        !plain_ptr(a[11], prep.q_norm_weight) || !plain_ptr(a[12], prep.k_norm_weight) || !plain_float(a[13], prep.eps) ||
        !plain_float(a[14], prep.rope_base) || !PyBool_Check(a[15]) || !plain_u64(a[16], rotary))
        return not_plain();
    prep.rope_interleaved = a[15] == Py_True ? 1 : 0;
    prep.rotary_dim = uint32_t(rotary);
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = prep_step_fn(pool, layer, items, count, q, k, v, gate, out, heads, scale, softcap, &prep);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

// truncate(pool, slots, lengths) -> status
PyObject *truncate(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 3)) return nullptr;
    itak_pool *pool;
    PyObject **slot_at, **length_at;
    Py_ssize_t slots, lengths;
    uint32_t slot[kMostItems];
    uint64_t length[kMostItems];
    if (!plain_ptr(a[0], pool) || !plain_sequence(a[1], slot_at, slots) || !plain_sequence(a[2], length_at, lengths) ||
        slots > kMostItems || lengths != slots)
        return not_plain();
    for (Py_ssize_t i = 0; i < slots; ++i)
        if (!plain_slot(slot_at[i], slot[i]) || !plain_within(length_at[i], 64, length[i])) return not_plain();
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = truncate_fn(pool, slot, length, uint32_t(slots));
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

// compute(pool, slot, layer, q, k, v, q_heads, position, softcap, rope_base) -> outputs, or a status
PyObject *compute(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 10)) return nullptr;
    itak_pool *pool;
    const float *q, *k, *v;
    uint64_t slot, layer, q_size, k_size, v_size, heads, position;
    float softcap, base;
    if (!plain_ptr(a[0], pool) || !plain_u64(a[1], slot) || !plain_u64(a[2], layer) || !plain_array(a[3], q, q_size) ||
        !plain_array(a[4], k, k_size) || !plain_array(a[5], v, v_size) || !plain_u64(a[6], heads) ||
        !plain_u64(a[7], position) || !plain_float(a[8], softcap) || !plain_float(a[9], base))
        return not_plain();
    npy_intp dims[] = {npy_intp(q_size)};
    PyObject *out = PyArray_SimpleNew(1, dims, NPY_FLOAT32);  // every element is written, or a status comes back
    if (!out) return nullptr;
    float *to = q_size ? static_cast<float *>(PyArray_DATA(reinterpret_cast<PyArrayObject *>(out))) : nullptr;
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = compute_fn(pool, uint32_t(slot), layer, q, q_size, k, k_size, v, v_size, heads, position, softcap, base, to);
    Py_END_ALLOW_THREADS
    if (st == ITAK_OK) return out;
    Py_DECREF(out);
    return PyLong_FromLong(st);
}

// gqa(pool, slot, layer, q, queries, q_heads, positions, scale, softcap) -> outputs, or a status
PyObject *gqa(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 9)) return nullptr;
    itak_pool *pool;
    const float *q;
    uint64_t slot, layer, q_size, queries, heads, position[kMostItems];
    float scale, softcap;
    PyObject **position_at;
    Py_ssize_t positions;
    if (!plain_ptr(a[0], pool) || !plain_u64(a[1], slot) || !plain_u64(a[2], layer) || !plain_array(a[3], q, q_size) ||
        !plain_u64(a[4], queries) || !plain_u64(a[5], heads) || !plain_sequence(a[6], position_at, positions) ||
        positions > kMostItems || !plain_scale(a[7], scale) || !plain_float(a[8], softcap))
        return not_plain();
    for (Py_ssize_t i = 0; i < positions; ++i)
        if (!plain_within(position_at[i], 64, position[i])) return not_plain();
    npy_intp dims[] = {npy_intp(q_size)};
    PyObject *out = PyArray_SimpleNew(1, dims, NPY_FLOAT32);
    if (!out) return nullptr;
    float *to = q_size ? static_cast<float *>(PyArray_DATA(reinterpret_cast<PyArrayObject *>(out))) : nullptr;
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = gqa_fn(pool, uint32_t(slot), layer, q, q_size, queries, heads, positions ? position : nullptr, uint64_t(positions),
                scale, softcap, to);
    Py_END_ALLOW_THREADS
    if (st == ITAK_OK) return out;
    Py_DECREF(out);
    return PyLong_FromLong(st);
}

bool bound_type(PyObject *o) {
    if (!PyType_Check(o)) PyErr_SetString(PyExc_TypeError, "a type comes first");
    return PyType_Check(o);
}
template <int N>
bool bound_addresses(PyObject *const *a, uint64_t (&at)[N]) {
    for (int i = 0; i < N; ++i)
        if (!plain_within(a[i], 64, at[i]) || at[i] == 0) {
            PyErr_SetString(PyExc_TypeError, "an address is an int that is not zero");
            return false;
        }
    return true;
}

// rotate(rotation, stream, head_dim, rows, positions, inputs, outputs, inverse) -> status
PyObject *rotate(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 8)) return nullptr;
    constexpr Py_ssize_t kMostTensors = 4;
    itak_rotation *rotation;
    void *stream;
    uint64_t head_dim, rows;
    const int64_t *positions;
    PyObject **in_at, **out_at;
    Py_ssize_t ins, outs;
    itak_rows in[kMostTensors], out[kMostTensors];
    if (!plain_ptr(a[0], rotation) || !plain_ptr(a[1], stream) || !plain_u64(a[2], head_dim) || !plain_u64(a[3], rows) ||
        !plain_ptr(a[4], positions) || !plain_sequence(a[5], in_at, ins) || !plain_sequence(a[6], out_at, outs) || ins != outs ||
        ins > kMostTensors || !PyBool_Check(a[7]))
        return not_plain();
    for (Py_ssize_t i = 0; i < ins; ++i) {
        const itak_rows *x, *y;
        if (!plain_rows(in_at[i], rows, head_dim, x) || !plain_rows(out_at[i], rows, head_dim, y)) return not_plain();
        in[i] = *x, out[i] = *y;
    }
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = rotate_fn(rotation, stream, head_dim, rows, positions, in, out, uint32_t(ins), a[7] == Py_True ? 1 : 0);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

// set_batch(paged, items, tables) -> status, and set_batch_tree(paged, items, tables, parents) -> status
PyObject *set_batch_with(PyObject *const *a, const int32_t *parents, Py_ssize_t parent_count) {
    itak_paged *paged;
    PyObject **item_at, **table_at;
    Py_ssize_t items, tables;
    itak_paged_item item[kMostItems];
    const void *run[kMostItems];
    if (!plain_ptr(a[0], paged) || !plain_sequence(a[1], item_at, items) || !plain_sequence(a[2], table_at, tables) ||
        items != tables || items > kMostItems)
        return not_plain();
    uint64_t all = 0, new_rows = 0;
    for (Py_ssize_t i = 0; i < items; ++i) {
        uint64_t rows;
        Py_ssize_t pages;
        if (!PyTuple_CheckExact(item_at[i]) || PyTuple_GET_SIZE(item_at[i]) != 2 ||
            !plain_within(PyTuple_GET_ITEM(item_at[i], 0), 64, item[i].position) ||
            !plain_within(PyTuple_GET_ITEM(item_at[i], 1), 32, rows) || !plain_words(table_at[i], run[i], pages) ||
            pages > Py_ssize_t(0xffffffffu))
            return not_plain();
        item[i].rows = uint32_t(rows), item[i].pages = uint32_t(pages);
        all += uint64_t(pages);
        new_rows += rows;
    }
    if (parents && uint64_t(parent_count) != new_rows) return not_plain();
    // (A batch of one sequence is read where it lies.)
    uint32_t *joined = nullptr;
    const uint32_t *ids = items && all ? static_cast<const uint32_t *>(run[0]) : nullptr;
    if (items > 1 && all) {
        joined = static_cast<uint32_t *>(PyMem_Malloc(all * sizeof(uint32_t)));
        if (!joined) return PyErr_NoMemory();
        uint64_t at = 0;
        for (Py_ssize_t i = 0; i < items; at += item[i].pages, ++i)
            if (item[i].pages) std::memcpy(joined + at, run[i], item[i].pages * sizeof(uint32_t));
        ids = joined;
    }
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = parents ? set_batch_tree_fn(paged, item, uint32_t(items), ids, all, parents) : set_batch_fn(paged, item, uint32_t(items), ids, all);
    Py_END_ALLOW_THREADS
    PyMem_Free(joined);
    return PyLong_FromLong(st);
}
PyObject *set_batch(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 3)) return nullptr;
    return set_batch_with(a, nullptr, 0);
}
PyObject *set_batch_tree(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 4)) return nullptr;
    const void *parents;
    Py_ssize_t count;
    if (!plain_words(a[3], parents, count) || count == 0 || PyArray_TYPE(reinterpret_cast<PyArrayObject *>(a[3])) != NPY_INT32) return not_plain();
    return set_batch_with(a, static_cast<const int32_t *>(parents), count);
}

// Every sequence's rows: a list or tuple of exact ints of 32 bits, as many as the tables have sequences.
constexpr Py_ssize_t kMostSequences = 1024;
bool plain_counts(PyObject *o, Py_ssize_t want, uint32_t *counts, uint64_t &sum) {
    PyObject **at;
    Py_ssize_t n;
    if (!plain_sequence(o, at, n) || n != want || n > kMostSequences) return false;
    sum = 0;
    for (Py_ssize_t i = 0; i < n; ++i) {
        uint64_t v;
        if (!plain_within(at[i], 32, v)) return false;
        counts[i] = uint32_t(v);
        sum += v;
    }
    return true;
}

// fit_tables(paged, tables, sequences, lengths, rows or None, status) -> status
PyObject *fit_tables(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 6)) return nullptr;
    itak_paged *paged;
    const itak_page_tables *tables;
    const int32_t *lengths;
    int32_t *status;
    uint64_t sequences, sum;
    uint32_t counts[kMostSequences];
    const bool rows = a[4] != Py_None;
    if (!plain_ptr(a[0], paged) || !plain_ptr(a[1], tables) || !plain_within(a[2], 32, sequences) || !plain_ptr(a[3], lengths) ||
        !plain_ptr(a[5], status) || (rows && !plain_counts(a[4], Py_ssize_t(sequences), counts, sum)))
        return not_plain();
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = fit_fn(paged, tables, lengths, rows ? counts : nullptr, status);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

// set_batch_device(paged, tables, sequences, positions, rows, most_positions, parents, status) -> status << 32 | the batch's rows
PyObject *set_batch_device(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 8)) return nullptr;
    itak_paged *paged;
    const itak_page_tables *tables;
    const int32_t *positions, *parents;
    int32_t *status;
    uint64_t sequences, most, sum = 0;
    uint32_t counts[kMostSequences];
    if (!plain_ptr(a[0], paged) || !plain_ptr(a[1], tables) || !plain_within(a[2], 32, sequences) || !plain_ptr(a[3], positions) ||
        !plain_counts(a[4], Py_ssize_t(sequences), counts, sum) || sum >> 32 || !plain_within(a[5], 64, most) || !plain_ptr(a[6], parents) ||
        !plain_ptr(a[7], status))
        return not_plain();
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = set_batch_device_fn(paged, tables, positions, counts, most, parents, status);
    Py_END_ALLOW_THREADS
    return PyLong_FromLongLong((long long)(uint32_t(st)) << 32 | (long long)sum);
}

// batch_rows(paged, positions, slots) -> status
PyObject *batch_rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 3)) return nullptr;
    itak_paged *paged;
    int64_t *positions, *slots;
    if (!plain_ptr(a[0], paged) || !plain_ptr(a[1], positions) || !plain_ptr(a[2], slots)) return not_plain();
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = batch_rows_fn(paged, positions, slots);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

// accept(paged, tokens, chosen, path, next) -> status
PyObject *accept(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 5)) return nullptr;
    itak_paged *paged;
    const int32_t *tokens, *chosen;
    int32_t *path, *next;
    if (!plain_ptr(a[0], paged) || !plain_ptr(a[1], tokens) || !plain_ptr(a[2], chosen) || !plain_ptr(a[3], path) || !plain_ptr(a[4], next))
        return not_plain();
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = accept_fn(paged, tokens, chosen, path, next);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

// keep(paged, path, lengths) -> status
PyObject *keep(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 3)) return nullptr;
    itak_paged *paged;
    const int32_t *path;
    int32_t *lengths;
    if (!plain_ptr(a[0], paged) || !plain_ptr(a[1], path) || !plain_ptr(a[2], lengths)) return not_plain();
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = keep_fn(paged, path, lengths);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

// append(paged, rows, head_dim, layer, k, v, rotation) -> status
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 7)) return nullptr;
    itak_paged *paged;
    uint64_t layer, rows, d;
    const itak_rows *k, *v;
    itak_rotation *rotation;
    if (!plain_ptr(a[0], paged) || !plain_u64(a[1], rows) || !plain_u64(a[2], d) || !plain_u64(a[3], layer) ||
        !plain_rows(a[4], rows, d, k) || !plain_rows(a[5], rows, d, v) || !plain_ptr(a[6], rotation))
        return not_plain();
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = append_fn(paged, layer, k, v, rotation);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

// paged_attention(paged, rows, head_dim, layer, q, out, scale, softcap, window, rotation) -> status
PyObject *paged_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 10)) return nullptr;
    itak_paged *paged;
    uint64_t layer, window, rows, d;
    const itak_rows *q, *out;
    float scale, softcap;
    itak_rotation *rotation;
    if (!plain_ptr(a[0], paged) || !plain_u64(a[1], rows) || !plain_u64(a[2], d) || !plain_u64(a[3], layer) ||
        !plain_rows(a[4], rows, d, q) || !plain_rows(a[5], rows, d, out) || !plain_scale(a[6], scale) ||
        !plain_float(a[7], softcap) || !plain_u64(a[8], window) || !plain_ptr(a[9], rotation))
        return not_plain();
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = paged_attention_fn(paged, layer, q, out, scale, softcap, window, rotation);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

// paged_step(paged, rows, head_dim, layer, q, k, v, out, scale, softcap, window, rotation) -> status
PyObject *paged_step(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 12)) return nullptr;
    itak_paged *paged;
    uint64_t layer, window, rows, d;
    const itak_rows *q, *k, *v, *out;
    float scale, softcap;
    itak_rotation *rotation;
    if (!plain_ptr(a[0], paged) || !plain_u64(a[1], rows) || !plain_u64(a[2], d) || !plain_u64(a[3], layer) ||
        !plain_rows(a[4], rows, d, q) || !plain_rows(a[5], rows, d, k) || !plain_rows(a[6], rows, d, v) ||
        !plain_rows(a[7], rows, d, out) || !plain_scale(a[8], scale) || !plain_float(a[9], softcap) || !plain_u64(a[10], window) ||
        !plain_ptr(a[11], rotation))
        return not_plain();
    itak_status st;
    Py_BEGIN_ALLOW_THREADS
    st = paged_step_fn(paged, layer, q, k, v, out, scale, softcap, window, rotation);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

// bind_paged(Rows, address of each of the five functions above, in their order)
PyObject *bind_paged(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 6)) return nullptr;
    uint64_t at[5];
    if (!bound_type(a[0]) || !bound_addresses(a + 1, at)) return nullptr;
    Py_INCREF(a[0]);
    Py_XDECREF(reinterpret_cast<PyObject *>(rows_type));
    rows_type = reinterpret_cast<PyTypeObject *>(a[0]);
    rotate_fn = reinterpret_cast<decltype(rotate_fn)>(uintptr_t(at[0]));
    set_batch_fn = reinterpret_cast<decltype(set_batch_fn)>(uintptr_t(at[1]));
    append_fn = reinterpret_cast<decltype(append_fn)>(uintptr_t(at[2]));
    paged_attention_fn = reinterpret_cast<decltype(paged_attention_fn)>(uintptr_t(at[3]));
    paged_step_fn = reinterpret_cast<decltype(paged_step_fn)>(uintptr_t(at[4]));
    Py_RETURN_NONE;
}

// bind_trees(address of the six functions from set_batch_tree's to keep's, in their order)
PyObject *bind_trees(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 6)) return nullptr;
    uint64_t at[6];
    if (!bound_addresses(a, at)) return nullptr;
    set_batch_tree_fn = reinterpret_cast<decltype(set_batch_tree_fn)>(uintptr_t(at[0]));
    fit_fn = reinterpret_cast<decltype(fit_fn)>(uintptr_t(at[1]));
    set_batch_device_fn = reinterpret_cast<decltype(set_batch_device_fn)>(uintptr_t(at[2]));
    batch_rows_fn = reinterpret_cast<decltype(batch_rows_fn)>(uintptr_t(at[3]));
    accept_fn = reinterpret_cast<decltype(accept_fn)>(uintptr_t(at[4]));
    keep_fn = reinterpret_cast<decltype(keep_fn)>(uintptr_t(at[5]));
    Py_RETURN_NONE;
}

// bind(KvCache, address of step's, prep_step's, truncate's, compute's and gqa's function)
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 6)) return nullptr;
    uint64_t at[5];
    if (!bound_type(a[0]) || !bound_addresses(a + 1, at)) return nullptr;
    Py_INCREF(a[0]);
    Py_XDECREF(reinterpret_cast<PyObject *>(cache_type));
    cache_type = reinterpret_cast<PyTypeObject *>(a[0]);
    step_fn = reinterpret_cast<decltype(step_fn)>(uintptr_t(at[0]));
    prep_step_fn = reinterpret_cast<decltype(prep_step_fn)>(uintptr_t(at[1]));
    truncate_fn = reinterpret_cast<decltype(truncate_fn)>(uintptr_t(at[2]));
    compute_fn = reinterpret_cast<decltype(compute_fn)>(uintptr_t(at[3]));
    gqa_fn = reinterpret_cast<decltype(gqa_fn)>(uintptr_t(at[4]));
    Py_RETURN_NONE;
}

template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyMethodDef method(const char *name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<bind>("bind"), method<step>("step"),       method<prep_step>("prep_step"),
                         method<truncate>("truncate"), method<compute>("compute"), method<gqa>("gqa"),
                         method<bind_paged>("bind_paged"), method<rotate>("rotate"), method<set_batch>("set_batch"),
                         method<append>("append"), method<paged_attention>("paged_attention"),
                         method<paged_step>("paged_step"),
                         method<bind_trees>("bind_trees"), method<set_batch_tree>("set_batch_tree"),
                         method<fit_tables>("fit_tables"), method<set_batch_device>("set_batch_device"),
                         method<batch_rows>("batch_rows"), method<accept>("accept"), method<keep>("keep"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_itak_front", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__itak_front(void) {
    import_array();
    slot_name = PyUnicode_InternFromString("slot");
    address_name = PyUnicode_InternFromString("at");
    rows_name = PyUnicode_InternFromString("rows");
    channels_name = PyUnicode_InternFromString("channels");
    return slot_name && address_name && rows_name && channels_name ? PyModule_Create(&module) : nullptr;
}
