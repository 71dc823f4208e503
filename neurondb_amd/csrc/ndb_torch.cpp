/*
 * ndb_torch.cpp — calls on torch tensors that are asked for so little that the way to the kernel is what they cost: checks of
 * the arguments, the result and the launch in one crossing from Python.  neurondb_amd/int8.py loads it and hands it the
 * library's functions, so that a process has one libndbhip.so whichever it is.
 *
 * One row of 1000 scores and a bias (us a call, back to back): checks in Python and three foreign calls 10.0, this 4.1, of which
 * the launch is 2.6; torch adds the two in 4.7.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <cstdarg>
#include <cstdio>
#include "ndbhip.h"

static PyObject *g_error;			/* NdbHipError(code, message) */
static at::Device g_device(at::kCPU);
static decltype(&ndbhip_swap_thread_stream) g_swap;
static decltype(&ndbhip_last_error) g_last_error;
static decltype(&ndbhip_scores_adjust_device) g_adjust;

/* a Python exception is set */
struct Refused
{
};

static void
raise(int code, const char *msg)
{
	PyObject   *e = PyObject_CallFunction(g_error, "is", code, msg);

	if (e)
	{
		PyErr_SetObject(g_error, e);
		Py_DECREF(e);
	}
	throw Refused();
}

__attribute__((format(printf, 1, 2))) static void
refuse(const char *fmt, ...)
{
	char		buf[256];
	va_list		ap;

	va_start(ap, fmt);
	vsnprintf(buf, sizeof(buf), fmt, ap);
	va_end(ap);
	raise(NDBHIP_ERR_INVALID, buf);
}

/* what every tensor argument has to be; t: bits of the types it may have */
enum Types
{
	F32 = 1, F16 = 2, BF16 = 4, FLOATS = 7, I32 = 8, I64 = 16, U32 = 32
};

static int
type_bit(at::ScalarType t)
{
	switch (t)
	{
		case at::kFloat:
			return F32;
		case at::kHalf:
			return F16;
		case at::kBFloat16:
			return BF16;
		case at::kInt:
			return I32;
		case at::kLong:
			return I64;
		case at::ScalarType::UInt32:
			return U32;
		default:
			return 0;
	}
}

static const at::Tensor &
tensor(PyObject *o, const char *name, int types, int ndim, int ndim2 = -1)
{
	if (!THPVariable_Check(o))
		refuse("%s must be a torch tensor", name);
	const at::Tensor &t = THPVariable_Unpack(o);

	if (t.device() != g_device)
		refuse("%s is on %s, the library on %s", name, t.device().str().c_str(), g_device.str().c_str());
	if (!(type_bit(t.scalar_type()) & types))
		refuse("%s must not be of %s", name, c10::toString(t.scalar_type()));
	if (t.layout() != at::kStrided)
		refuse("%s must be a dense tensor", name);
	if (t.dim() != ndim && t.dim() != ndim2)
		refuse("%s has %d dimensions", name, (int) t.dim());
	if (t.requires_grad() && at::GradMode::is_enabled())
		refuse("%s requires a gradient, which this call has none of: detach() it, or call under no_grad()", name);
	return t;
}

/* rows of a matrix (a vector: its one row): neighbouring elements side by side, rows that do not overlap */
static bool
rows_apart(const at::Tensor &t, int64_t n, int64_t dim, int64_t rstride, int64_t estride)
{
	return !((dim > 1 && estride != 1) || (n > 1 && rstride < dim));
}

static at::Tensor
as_rows(const at::Tensor &t, int64_t *stride)
{
	const int	d = (int) t.dim();
	const int64_t n = d == 2 ? t.size(0) : 1, dim = t.size(d - 1);
	const int64_t rs = d == 2 ? t.stride(0) : dim;

	if (!rows_apart(t, n, dim, rs, t.stride(d - 1)))
	{
		*stride = dim;
		return t.contiguous();
	}
	*stride = n > 1 ? rs : dim;
	return t;
}

/* adjust(stream, scores, seen, penalties, bias, mask, out) */
static PyObject *
adjust(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
	HANDLE_TH_ERRORS
	try
	{
		if (nargs != 7)
			refuse("adjust takes 7 arguments, not %d", (int) nargs);
		void	   *const stream = PyLong_AsVoidPtr(args[0]);

		if (!stream && PyErr_Occurred())
			return nullptr;
		PyObject   *const seen = args[2], *const pen = args[3], *const obias = args[4], *const omask = args[5], *const oout = args[6];
		const at::Tensor &scores = tensor(args[1], "scores", FLOATS, 2);
		const int64_t nq = scores.size(0), n = scores.size(1), words = (n + 31) / 32;
		int64_t		stride, ostride = n, bstride = 0, mstride = 0, nids = 0;
		at::Tensor	src = as_rows(scores, &stride), off, ids, penalties, bias, mask, made;

		if (nq > INT32_MAX)
			refuse("scores has %lld rows", (long long) nq);
		if (oout != Py_None)
		{
			const at::Tensor &out = tensor(oout, "out", type_bit(scores.scalar_type()), 2);

			if (out.size(0) != nq || out.size(1) != n)
				refuse("out must have the scores' shape");
			if (!rows_apart(out, nq, n, out.stride(0), out.stride(1)))
				refuse("out must have neighbouring elements in a row and rows that do not overlap");
			ostride = nq > 1 ? out.stride(0) : n;
			made = out;
		}
		if ((seen == Py_None) != (pen == Py_None))
			refuse("seen and penalties go together");
		if (seen != Py_None)
		{
			THPObjectPtr pair(PySequence_Fast(seen, "seen must be (offsets, ids)"));

			if (!pair)
				return nullptr;
			if (PySequence_Fast_GET_SIZE(pair.get()) != 2)
				refuse("seen must be (offsets, ids)");
			off = tensor(PySequence_Fast_GET_ITEM(pair.get(), 0), "offsets", I64, 1).contiguous();
			ids = tensor(PySequence_Fast_GET_ITEM(pair.get(), 1), "ids", I32, 1).contiguous();
			penalties = tensor(pen, "penalties", F32, 2).contiguous();
			if (off.size(0) != nq + 1 || penalties.size(0) != nq || penalties.size(1) != 3)
				refuse("offsets must be [nq + 1] and penalties [nq, 3]");
			nids = ids.size(0);
		}
		if (obias != Py_None)
		{
			const at::Tensor &b = tensor(obias, "bias", F32, 1, 2);

			if (b.size(b.dim() - 1) != n || (b.dim() == 2 && b.size(0) != 1 && b.size(0) != nq))
				refuse("bias must be [%lld] or [1 or %lld, %lld]", (long long) n, (long long) nq, (long long) n);
			bias = as_rows(b, &bstride);
			if (b.dim() == 1 || b.size(0) == 1)
				bstride = 0;
		}
		if (omask != Py_None)
		{
			const at::Tensor &m = tensor(omask, "mask", I32 | U32, 1, 2);

			if (m.size(m.dim() - 1) < words || (m.dim() == 2 && m.size(0) != 1 && m.size(0) != nq))
				refuse("mask must be [words] or [1 or %lld, words] with at least %lld words of 32 rows", (long long) nq, (long long) words);
			mask = as_rows(m, &mstride);
			if (m.dim() == 1 || m.size(0) == 1)
				mstride = 0;
		}
		if (oout == Py_None)
			made = at::empty({nq, n}, at::TensorOptions().dtype(scores.scalar_type()).device(scores.device()));

		const int	type = scores.scalar_type() == at::kFloat ? NDBHIP_F32 : scores.scalar_type() == at::kHalf ? NDBHIP_F16 : NDBHIP_BF16;
		const void *const p = src.const_data_ptr(), *const pb = bias.defined() ? bias.const_data_ptr() : nullptr,
				   *const pm = mask.defined() ? mask.const_data_ptr() : nullptr;
		void	   *const po = made.mutable_data_ptr(), *prev = nullptr;
		const int64_t *const poff = nids ? off.const_data_ptr<int64_t>() : nullptr;
		const int32_t *const pids = nids ? ids.const_data_ptr<int32_t>() : nullptr;
		const float *const ppen = nids ? penalties.const_data_ptr<float>() : nullptr;
		int			rc;

		/* (a launch can wait for the device) */
		Py_BEGIN_ALLOW_THREADS
		rc = g_swap(stream, &prev);
		if (!rc)
		{
			void	   *mine;

			rc = g_adjust(p, type, (int) nq, n, stride, poff, pids, nids, ppen, (const float *) pb, bstride, (const uint32_t *) pm, mstride, po,
						  ostride);
			(void) g_swap(prev, &mine);
		}
		Py_END_ALLOW_THREADS
		if (rc)
			raise(rc, g_last_error());
		if (oout == Py_None)
			return THPVariable_Wrap(std::move(made));
		/* (what autograd has saved of the caller's tensor is another version now) */
		if (!made.is_inference())
			made.unsafeGetTensorImpl()->bump_version();
		Py_INCREF(oout);
		return oout;
	}
	catch (const Refused &)
	{
		return nullptr;
	}
	END_HANDLE_TH_ERRORS
}

/* setup(error class, name of the library's device, addresses of swap_thread_stream, last_error, scores_adjust_device) */
static PyObject *
setup(PyObject *, PyObject *args)
{
	HANDLE_TH_ERRORS
	PyObject   *error;
	const char *device;
	unsigned long long swap, last, adj;

	if (!PyArg_ParseTuple(args, "OsKKK", &error, &device, &swap, &last, &adj))
		return nullptr;
	g_device = at::Device(device);
	Py_INCREF(error);
	Py_XSETREF(g_error, error);
	g_swap = (decltype(g_swap)) swap;
	g_last_error = (decltype(g_last_error)) last;
	g_adjust = (decltype(g_adjust)) adj;
	Py_RETURN_NONE;
	END_HANDLE_TH_ERRORS
}

static PyMethodDef methods[] = {
	{"setup", setup, METH_VARARGS, nullptr},
	{"adjust", (PyCFunction) (void (*)(void)) adjust, METH_FASTCALL, nullptr},
	{nullptr, nullptr, 0, nullptr}
};

static PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ndb_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

PyMODINIT_FUNC
PyInit__ndb_torch(void)
{
	return PyModule_Create(&module);
}
