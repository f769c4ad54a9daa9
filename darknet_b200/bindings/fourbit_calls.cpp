// The host side of a four-bit call: what darknet_b200/fourbit.py asks of its tensors, and the call into libxnor_b200.so.
//
// A decoding step is a dozen kernels of 4 to 8 us, so the host that issues them is what it waits for.  Asked through ctypes, a call took 8 us
// (a product) to 11 us (attention), 3 of them the launch; most of the others went into looking up shapes, types, strides and addresses one by
// one.  Here they are read from the tensors themselves.  Every function returns None where an argument is not what it has to be (fourbit.py
// then looks for what is wrong and says so), the library's code as a number where the library refused, and its result otherwise; outputs that
// share memory with inputs are refused here, where the addresses are.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <optional>
#include <vector>

#include "xnor_b200.h"

namespace
{

using at::Tensor;

// A tensor argument; null for None.  False: neither.
bool take(PyObject * o, const Tensor *& t)
{
	t = nullptr;
	if (o == Py_None) { return true; }
	if (!THPVariable_Check(o)) { return false; }
	t = &THPVariable_Unpack(o);
	return true;
}

int type_of(const Tensor & t)
{
	switch (t.scalar_type())
	{
		case at::kFloat: return XNOR_B200_F32;
		case at::kHalf: return XNOR_B200_F16;
		case at::kBFloat16: return XNOR_B200_BF16;
		default: return -1;
	}
}

bool on(const Tensor & t, const c10::Device & d) { return t.is_cuda() && t.device() == d && t.layout() == at::kStrided; }

bool int32s(const Tensor * t, const c10::Device & d, int64_t n)
{
	return t != nullptr && on(*t, d) && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->is_contiguous();
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const c10::Device & d)
{
	return at::detail::empty_cuda(sizes, type, at::kStrided, d, false, std::nullopt);
}

struct Failed {};                 // a Python error is set

[[noreturn]] void refuse(const char * what)
{
	PyErr_SetString(PyExc_ValueError, what);
	throw Failed();
}

// A handle's buffers may have been resized or given other memory since it was made: the kernels go by the sizes.
void as_made(bool still)
{
	if (!still) { refuse("a buffer of the handle is not the one it was made with: it has been resized or set to other memory"); }
}

void out_of_memory(const char * what)
{
	PyObject * torch = PyImport_ImportModule("torch");
	PyObject * type = torch != nullptr ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
	if (type != nullptr) { PyErr_SetString(type, what); }
	Py_XDECREF(type);
	Py_XDECREF(torch);
}

// The entry points: C++ exceptions (out of memory) become Python's, and nothing else runs meanwhile than has to.
template <class F>
PyObject * guarded(F && f)
{
	try { return f(); }
	catch (const Failed &) { return nullptr; }
	catch (const c10::OutOfMemoryError & e) { out_of_memory(e.what_without_backtrace()); }
	catch (const std::exception & e) { PyErr_SetString(PyExc_RuntimeError, e.what()); }
	catch (...) { PyErr_SetString(PyExc_RuntimeError, "four-bit call failed"); }
	return nullptr;
}

struct WithoutGil
{
	PyThreadState * state = PyEval_SaveThread();
	~WithoutGil() { PyEval_RestoreThread(state); }
};
template <class F>
int without_gil(F && f)
{
	const WithoutGil released;
	return f();
}

long long whole(PyObject * o)
{
	const long long v = PyLong_AsLongLong(o);
	if (v == -1 && PyErr_Occurred()) { throw Failed(); }
	return v;
}

// ---- memory in common.  What a call writes to is looked at where it was given: a comparison of two ranges, and only where those meet (views of
// one buffer, side by side) the elements themselves.
struct Dim { int64_t size, stride; };

// A tensor's dimensions of more than one entry, the widest stride first; false where more of them would be than in any call.
bool layout(const Tensor & t, Dim (&d)[4], int & n)
{
	n = 0;
	for (int64_t i = 0; i < t.dim(); ++i)
	{
		if (t.size(i) == 1) { continue; }
		if (n == 4) { return false; }
		d[n++] = {t.size(i), t.stride(i)};
	}
	std::sort(d, d + n, [](const Dim & a, const Dim & b) { return a.stride > b.stride; });
	return true;
}

// Entries from the first to behind the last.
int64_t extent(const Dim * d, int n)
{
	int64_t e = 1;
	for (int i = 0; i < n; ++i) { e += (d[i].size - 1) * d[i].stride; }
	return e;
}

// Every dimension's steps pass over all that the narrower ones cover: no entry is there twice.
bool nested(const Dim * d, int n)
{
	for (int i = 0; i < n; ++i)
	{
		if (d[i].stride < extent(d + i + 1, n - i - 1)) { return false; }
	}
	return true;
}

// Two tensors of these nested dimensions, the second `apart` entries behind the first, have an entry in common: two steps of a dimension at
// most come near enough for the narrower ones.
bool within(const Dim * d, int n, int64_t apart)
{
	if (n == 0) { return apart == 0; }
	const int64_t inner = extent(d + 1, n - 1), first = apart >= 0 ? apart / d->stride : -((-apart + d->stride - 1) / d->stride);
	for (int64_t steps = first; steps <= first + 1; ++steps)
	{
		const int64_t rest = apart - steps * d->stride;
		if (steps > -d->size && steps < d->size && rest > -inner && rest < inner && within(d + 1, n - 1, rest)) { return true; }
	}
	return false;
}

// Where a tensor's rows start, in order, and their bytes.  One row where all of it is contiguous.
std::vector<uintptr_t> rows_of(const Tensor & t, size_t & bytes)
{
	const uintptr_t first = (uintptr_t)t.data_ptr();
	const int64_t size = t.element_size(), dims = t.dim();
	std::vector<uintptr_t> rows = {first};
	if (t.is_contiguous())
	{
		bytes = (size_t)(t.numel() * size);
		return rows;
	}
	const bool whole_rows = t.stride(dims - 1) == 1 || t.size(dims - 1) == 1;
	bytes = (size_t)(whole_rows ? t.size(dims - 1) * size : size);
	for (int64_t i = 0; i < dims - (whole_rows ? 1 : 0); ++i)
	{
		const size_t before = rows.size();
		for (int64_t j = 1; j < t.size(i); ++j)
		{
			for (size_t r = 0; r < before; ++r) { rows.push_back(rows[r] + j * t.stride(i) * size); }
		}
	}
	std::sort(rows.begin(), rows.end());
	return rows;
}

bool meet(const Tensor & a, const Tensor & b)
{
	if (a.numel() == 0 || b.numel() == 0) { return false; }
	Dim da[4], db[4];
	int na, nb;
	const bool known = layout(a, da, na) && layout(b, db, nb);
	const uintptr_t a0 = (uintptr_t)a.data_ptr(), b0 = (uintptr_t)b.data_ptr();
	const int64_t size = a.element_size();
	if (known)
	{
		if (a0 + extent(da, na) * size <= b0 || b0 + extent(db, nb) * b.element_size() <= a0) { return false; }
		const int64_t bytes = (int64_t)(b0 - a0);
		if (na == nb && b.element_size() == size && bytes % size == 0 && nested(da, na)
				&& std::equal(da, da + na, db, [](const Dim & x, const Dim & y) { return x.size == y.size && x.stride == y.stride; }))
		{
			return within(da, na, bytes / size);
		}
	}
	size_t a_bytes, b_bytes;
	const std::vector<uintptr_t> ra = rows_of(a, a_bytes), rb = rows_of(b, b_bytes);
	for (size_t i = 0, j = 0; i < ra.size() && j < rb.size(); )
	{
		if (ra[i] + a_bytes <= rb[j]) { ++i; }
		else if (rb[j] + b_bytes <= ra[i]) { ++j; }
		else { return true; }
	}
	return false;
}

bool meets_itself(const Tensor & t)
{
	Dim d[4];
	int n;
	if (t.numel() == 0 || (layout(t, d, n) && nested(d, n))) { return false; }
	size_t bytes;
	const std::vector<uintptr_t> rows = rows_of(t, bytes);
	for (size_t i = 1; i < rows.size(); ++i)
	{
		if (rows[i - 1] + bytes > rows[i]) { return true; }
	}
	return false;
}

// The same entries in the same order.
bool same(const Tensor & a, const Tensor & b)
{
	if (a.data_ptr() != b.data_ptr() || a.sizes() != b.sizes()) { return false; }
	for (int64_t i = 0; i < a.dim(); ++i)
	{
		if (a.size(i) > 1 && a.stride(i) != b.stride(i)) { return false; }
	}
	return true;
}

// ---- products: ((codes, scales, k, group), x, biases, activation, out)
PyObject * product(PyObject *, PyObject * const * args, Py_ssize_t n_args)
{
	return guarded([&]() -> PyObject *
	{
		const Tensor * codes, * scales, * x, * biases, * given;
		if (n_args != 5 || !PyTuple_Check(args[0]) || PyTuple_GET_SIZE(args[0]) != 4) { Py_RETURN_NONE; }
		if (!take(PyTuple_GET_ITEM(args[0], 0), codes) || !take(PyTuple_GET_ITEM(args[0], 1), scales) || !take(args[1], x) || !take(args[2], biases)
				|| !take(args[4], given) || codes == nullptr || scales == nullptr || x == nullptr || !PyLong_Check(args[3])) { Py_RETURN_NONE; }
		if (codes->dim() != 2) { Py_RETURN_NONE; }
		const int64_t n = codes->size(0), k = whole(PyTuple_GET_ITEM(args[0], 2));
		if (n > INT_MAX || k > INT_MAX) { Py_RETURN_NONE; }
		const int64_t group = whole(PyTuple_GET_ITEM(args[0], 3));
		as_made(k > 0 && group > 0 && codes->scalar_type() == at::kByte && codes->size(1) == (k + 31) / 32 * 16 && codes->is_contiguous()
				&& scales->scalar_type() == at::kHalf && scales->dim() == 3 && scales->size(0) == n && scales->size(1) == (k + group - 1) / group && scales->size(2) == 2
				&& scales->is_contiguous());
		const c10::Device d = codes->device();
		const int type = type_of(*x);
		if (!on(*codes, d) || !on(*scales, d) || !on(*x, d) || type < 0 || x->dim() != 2 || x->size(1) != k || (k != 1 && x->stride(1) != 1)) { Py_RETURN_NONE; }
		if (biases != nullptr && (!on(*biases, d) || biases->scalar_type() != at::kFloat || biases->dim() != 1 || biases->size(0) != n || !biases->is_contiguous()))
		{
			Py_RETURN_NONE;
		}
		const int64_t rows = x->size(0);
		if (given != nullptr && (!on(*given, d) || given->scalar_type() != x->scalar_type() || given->dim() != 2 || given->size(0) != rows || given->size(1) != n
				|| (n != 1 && given->stride(1) != 1))) { Py_RETURN_NONE; }
		if (given != nullptr)
		{
			for (const Tensor * input : {x, biases, codes, scales})
			{
				if (input != nullptr && meet(*given, *input)) { refuse("out has memory in common with what the product reads"); }
			}
			if (meets_itself(*given)) { refuse("out has entries that are the same memory"); }
		}
		const c10::cuda::CUDAGuard guard(d);
		const Tensor out = given != nullptr ? *given : empty({rows, n}, x->scalar_type(), d);
		if (rows == 0) { return THPVariable_Wrap(out); }
		const long long activation = whole(args[3]);
		if (rows > INT_MAX || activation < 0 || activation > 1) { Py_RETURN_NONE; }
		const xnor_b200_w4_desc desc = {(int)n, (int)k, (int)group, (int)activation};
		const size_t bytes = xnor_b200_w4_scratch_bytes(&desc, type, (int)rows);
		const Tensor scratch = bytes != 0 ? empty({(int64_t)bytes}, at::kByte, d) : Tensor();
		void * const stream = (void *)c10::cuda::getCurrentCUDAStream(d.index()).stream();
		const int rc = without_gil([&]
		{
			return xnor_b200_w4_forward(&desc, x->data_ptr(), type, (int)rows, rows > 1 ? x->stride(0) : k, (const uint8_t *)codes->data_ptr(), scales->data_ptr(),
					biases != nullptr ? (const float *)biases->data_ptr() : nullptr, out.data_ptr(), rows > 1 ? out.stride(0) : n,
					bytes != 0 ? scratch.data_ptr() : nullptr, bytes, stream);
		});
		return rc != XNOR_B200_OK ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
	});
}

// ---- the cache: (k_codes, k_scales, v_codes, v_scales, group), as Cache4 has checked them
bool take_cache(PyObject * o, xnor_b200_kv4_cache & c, std::optional<c10::Device> & d)
{
	const Tensor * t[4];
	if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 5) { return false; }
	for (int i = 0; i < 4; ++i)
	{
		if (!take(PyTuple_GET_ITEM(o, i), t[i]) || t[i] == nullptr) { return false; }
	}
	const at::IntArrayRef s = t[0]->sizes();
	if (s.size() != 4 || s[0] > INT_MAX || s[1] > INT_MAX || s[2] > INT_MAX || s[3] > INT_MAX / 2) { return false; }
	const int64_t group = whole(PyTuple_GET_ITEM(o, 4));
	for (int i = 0; i < 4; i += 2)
	{
		const Tensor & codes = *t[i], & scales = *t[i + 1];
		as_made(group > 0 && codes.scalar_type() == at::kByte && codes.sizes() == s && codes.is_contiguous() && scales.scalar_type() == at::kHalf && scales.dim() == 5
				&& scales.sizes().slice(0, 3) == s.slice(0, 3) && scales.size(3) == 2 * s[3] / group && scales.size(4) == 2 && scales.is_contiguous());
	}
	d = t[0]->device();
	for (const Tensor * v : t)
	{
		if (!on(*v, *d)) { return false; }
	}
	c = {(uint8_t *)t[0]->data_ptr(), t[1]->data_ptr(), (uint8_t *)t[2]->data_ptr(), t[3]->data_ptr(), (int)s[0], (int)s[1], (int)s[2], (int)(2 * s[3]),
			(int)group};
	return true;
}

bool take_rows(PyObject * table_o, PyObject * lengths_o, PyObject * counts_o, const c10::Device & d, int64_t batch, int64_t tokens, xnor_b200_kv4_rows & r)
{
	const Tensor * table, * lengths, * counts;
	if (!take(table_o, table) || !take(lengths_o, lengths) || !take(counts_o, counts) || table == nullptr) { return false; }
	if (!on(*table, d) || table->scalar_type() != at::kInt || table->dim() != 2 || table->size(0) != batch || table->size(1) == 0 || !table->is_contiguous()
			|| !int32s(lengths, d, batch) || (counts != nullptr && !int32s(counts, d, batch)) || batch > INT_MAX || tokens > INT_MAX || table->size(1) > INT_MAX)
	{
		return false;
	}
	r = {(int)batch, (int)tokens, (int)table->size(1), (const int32_t *)table->data_ptr(), (const int32_t *)lengths->data_ptr(),
			counts != nullptr ? (const int32_t *)counts->data_ptr() : nullptr};
	return true;
}

bool take_tensor(const Tensor & t, const c10::Device & d, xnor_b200_kv4_tensor & k)
{
	const int type = type_of(t);
	if (!on(t, d) || type < 0 || t.dim() != 4 || (t.size(3) != 1 && t.stride(3) != 1)) { return false; }
	k = {t.data_ptr(), type, t.stride(0), t.stride(1), t.stride(2)};
	return true;
}

// (cache, k, v, table, lengths, counts)
PyObject * append(PyObject *, PyObject * const * args, Py_ssize_t n_args)
{
	return guarded([&]() -> PyObject *
	{
		xnor_b200_kv4_cache c;
		xnor_b200_kv4_rows r;
		xnor_b200_kv4_tensor kt, vt;
		std::optional<c10::Device> d;
		const Tensor * k, * v;
		if (n_args != 6 || !take_cache(args[0], c, d) || !take(args[1], k) || !take(args[2], v) || k == nullptr || v == nullptr) { Py_RETURN_NONE; }
		if (!take_tensor(*k, *d, kt) || !take_tensor(*v, *d, vt) || kt.dtype != vt.dtype || k->sizes() != v->sizes() || k->size(2) != c.kv_heads || k->size(3) != c.dim
				|| !take_rows(args[3], args[4], args[5], *d, k->size(0), k->size(1), r)) { Py_RETURN_NONE; }
		if (k->numel() == 0) { Py_RETURN_TRUE; }
		const c10::cuda::CUDAGuard guard(*d);
		void * const stream = (void *)c10::cuda::getCurrentCUDAStream(d->index()).stream();
		const int rc = without_gil([&] { return xnor_b200_kv4_append(&c, &r, &kt, &vt, stream); });
		if (rc != XNOR_B200_OK) { return PyLong_FromLong(rc); }
		Py_RETURN_TRUE;
	});
}

// (cache, table, lengths, tokens, counts, type)
PyObject * read(PyObject *, PyObject * const * args, Py_ssize_t n_args)
{
	return guarded([&]() -> PyObject *
	{
		static const at::ScalarType types[3] = {at::kFloat, at::kHalf, at::kBFloat16};
		xnor_b200_kv4_cache c;
		xnor_b200_kv4_rows r;
		std::optional<c10::Device> d;
		const Tensor * table;
		if (n_args != 6 || !take_cache(args[0], c, d) || !take(args[1], table) || table == nullptr || table->dim() != 2 || !PyLong_Check(args[3])) { Py_RETURN_NONE; }
		const long long tokens = whole(args[3]), type = whole(args[5]);
		if (tokens < 0 || type < 0 || type > 2 || !take_rows(args[1], args[2], args[4], *d, table->size(0), tokens, r)) { Py_RETURN_NONE; }
		const c10::cuda::CUDAGuard guard(*d);
		const Tensor k = empty({r.batch, r.tokens, c.kv_heads, c.dim}, types[type], *d), v = empty(k.sizes(), types[type], *d);
		if (k.numel() != 0)
		{
			const long long token = (long long)c.kv_heads * c.dim;
			const xnor_b200_kv4_tensor kt = {k.data_ptr(), (int)type, token * r.tokens, token, c.dim}, vt = {v.data_ptr(), (int)type, token * r.tokens, token, c.dim};
			void * const stream = (void *)c10::cuda::getCurrentCUDAStream(d->index()).stream();
			const int rc = without_gil([&] { return xnor_b200_kv4_read(&c, &r, &kt, &vt, stream); });
			if (rc != XNOR_B200_OK) { return PyLong_FromLong(rc); }
		}
		return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(v));
	});
}

// (cache, q, table, lengths, counts, scale, window, out, lse)
PyObject * attend(PyObject *, PyObject * const * args, Py_ssize_t n_args)
{
	return guarded([&]() -> PyObject *
	{
		xnor_b200_kv4_cache c;
		xnor_b200_kv4_rows r;
		xnor_b200_kv4_tensor qt, ot;
		std::optional<c10::Device> d;
		const Tensor * q, * given, * lse;
		if (n_args != 9 || !take_cache(args[0], c, d) || !take(args[1], q) || !take(args[7], given) || !take(args[8], lse) || q == nullptr || !PyLong_Check(args[6]))
		{
			Py_RETURN_NONE;
		}
		if (!take_tensor(*q, *d, qt) || q->size(3) != c.dim || q->size(2) == 0 || q->size(2) % c.kv_heads != 0 || q->size(2) > INT_MAX
				|| !take_rows(args[2], args[3], args[4], *d, q->size(0), q->size(1), r)) { Py_RETURN_NONE; }
		const long long window = whole(args[6]);
		const double scale = args[5] == Py_None ? 1.0 / std::sqrt((double)c.dim) : PyFloat_AsDouble(args[5]);
		if (scale == -1.0 && PyErr_Occurred()) { throw Failed(); }
		if (window < 0) { Py_RETURN_NONE; }
		if (lse != nullptr && (!on(*lse, *d) || lse->scalar_type() != at::kFloat || lse->dim() != 3 || lse->sizes() != q->sizes().slice(0, 3) || !lse->is_contiguous()))
		{
			Py_RETURN_NONE;
		}
		if (given != nullptr)
		{
			if (given->sizes() != q->sizes() || !take_tensor(*given, *d, ot) || ot.dtype != qt.dtype) { Py_RETURN_NONE; }
			if (meets_itself(*given)) { refuse("out has entries that are the same memory"); }
			// (every CTA has read its queries before any writes the same ones' results)
			if (!same(*given, *q) && meet(*given, *q)) { refuse("out has memory in common with q, and is not q itself"); }
		}
		if (lse != nullptr && (meet(*lse, *q) || (given != nullptr && meet(*lse, *given)))) { refuse("lse has memory in common with q or out"); }
		const c10::cuda::CUDAGuard guard(*d);
		const Tensor out = given != nullptr ? *given : empty(q->sizes(), q->scalar_type(), *d);
		if (q->numel() == 0) { return THPVariable_Wrap(out); }
		take_tensor(out, *d, ot);
		const int heads = (int)q->size(2), reach = (int)std::min(window, (long long)INT_MAX);
		const size_t bytes = xnor_b200_kv4_attend_scratch_bytes(&c, &r, heads, reach);
		const Tensor scratch = bytes != 0 ? empty({(int64_t)bytes}, at::kByte, *d) : Tensor();
		void * const stream = (void *)c10::cuda::getCurrentCUDAStream(d->index()).stream();
		const int rc = without_gil([&]
		{
			return xnor_b200_kv4_attend(&c, &r, &qt, heads, (float)scale, reach, &ot, lse != nullptr ? (float *)lse->data_ptr() : nullptr,
					bytes != 0 ? scratch.data_ptr() : nullptr, bytes, stream);
		});
		return rc != XNOR_B200_OK ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
	});
}

// (a, b): whether two tensors have memory in common; (a): whether entries of one are the same memory.
PyObject * shares(PyObject *, PyObject * const * args, Py_ssize_t n_args)
{
	return guarded([&]() -> PyObject *
	{
		const Tensor * a, * b = nullptr;
		if (n_args < 1 || n_args > 2 || !take(args[0], a) || a == nullptr || (n_args == 2 && (!take(args[1], b) || b == nullptr))) { Py_RETURN_NONE; }
		return PyBool_FromLong(b != nullptr ? meet(*a, *b) : meets_itself(*a));
	});
}

PyMethodDef methods[] = {
	{"product", (PyCFunction)(void *)product, METH_FASTCALL, "xnor_b200_w4_forward"},
	{"append", (PyCFunction)(void *)append, METH_FASTCALL, "xnor_b200_kv4_append"},
	{"read", (PyCFunction)(void *)read, METH_FASTCALL, "xnor_b200_kv4_read"},
	{"attend", (PyCFunction)(void *)attend, METH_FASTCALL, "xnor_b200_kv4_attend"},
	{"shares", (PyCFunction)(void *)shares, METH_FASTCALL, "whether two tensors, or entries of one, are the same memory"},
	{nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fourbit", "Calls of darknet_b200.fourbit into libxnor_b200.so", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// (build.py looks for these words in the file)
extern "C" __attribute__((used)) const char fourbit_built_for[] = "built for torch " BUILT_FOR_TORCH ";";

PyMODINIT_FUNC PyInit__fourbit()
{
	PyObject * m = PyModule_Create(&module);
	if (m != nullptr && PyModule_AddStringConstant(m, "built_for", BUILT_FOR_TORCH) < 0)
	{
		Py_DECREF(m);
		return nullptr;
	}
	return m;
}
