// Calls of the paged-cache entry points on torch tensors, without the interpreter in
// between: a decode step makes several, each with a dozen tensors, and its kernels take
// microseconds.
//
// Every function takes what its namesake in nntile_b200/sdpa.py takes (missing arguments as
// None), and answers None when anything about a call is not as it should be, or tensors are
// not on the current device: the Python function then goes through the call step by step
// and says what is wrong.  An int is the status of an entry point that refused.
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <Python.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>

#include "../../include/nntile_b200.h"

namespace {

struct Refused {};                               // leave it to the Python function

// Interned attribute names of KVPages.
PyObject *name_k, *name_v, *name_k_scales, *name_v_scales, *name_bounds;

const at::Tensor *tensor(PyObject *o)
{
    if(o == Py_None)
    {
        return nullptr;
    }
    if(!THPVariable_Check(o))
    {
        throw Refused();
    }
    return &THPVariable_Unpack(o);
}

const at::Tensor &need(PyObject *o)
{
    const at::Tensor *t = tensor(o);
    if(!t)
    {
        throw Refused();
    }
    return *t;
}

void check(bool ok)
{
    if(!ok)
    {
        throw Refused();
    }
}

int64_t number(PyObject *o)
{
    check(PyLong_Check(o));
    const long long v = PyLong_AsLongLong(o);
    if(v == -1 && PyErr_Occurred())
    {
        PyErr_Clear();
        throw Refused();
    }
    return v;
}

bool is_row(at::ScalarType t)
{
    return t == at::kBFloat16 || t == at::kHalf;
}

// What a tensor holds, if there is one: all tensors of a call are contiguous on one device.
template<typename P>
P *address(const at::Tensor *t, int device)
{
    if(!t)
    {
        return nullptr;
    }
    check(t->is_cuda() && t->get_device() == device && t->is_contiguous());
    return static_cast<P *>(t->data_ptr());
}

// The attributes are held until the call is on its way, whatever kind of object they are of.
struct Pages
{
    const at::Tensor *k, *v, *k_scales, *v_scales, *bounds;
    int64_t num_pages, kv_heads, page_size, head;
    bool e4m3;

    Pages(const Pages &) = delete;

    explicit Pages(PyObject *o)
    {
        k = attribute(o, name_k);
        v = attribute(o, name_v);
        k_scales = attribute(o, name_k_scales);
        v_scales = attribute(o, name_v_scales);
        bounds = attribute(o, name_bounds);
        check(k && v && k->dim() == 4 && k->sizes() == v->sizes()
                && k->scalar_type() == v->scalar_type());
        num_pages = k->size(0);
        kv_heads = k->size(1);
        page_size = k->size(2);
        head = k->size(3);
        e4m3 = !is_row(k->scalar_type());
        if(e4m3)
        {
            check(k->scalar_type() == at::kByte || k->scalar_type() == at::kFloat8_e4m3fn);
        }
        for(const at::Tensor *s : {k_scales, v_scales})
        {
            check(e4m3 == (s != nullptr));
            check(!s || (s->scalar_type() == at::kByte && s->dim() == 3
                    && s->numel() == num_pages*kv_heads*page_size));
        }
        check(!bounds || (bounds->dim() == 4 && bounds->numel() == num_pages*kv_heads*2*head
                && is_row(bounds->scalar_type())));
    }

    void rows(const at::Tensor &t) const
    {
        check(is_row(t.scalar_type()) && (e4m3 || t.scalar_type() == k->scalar_type()));
    }

private:
    struct Held
    {
        PyObject *objects[5];
        int count = 0;

        ~Held()                                  // also when a check ends the constructor
        {
            while(count > 0)
            {
                Py_DECREF(objects[--count]);
            }
        }
    };
    Held held;

    const at::Tensor *attribute(PyObject *o, PyObject *name)
    {
        PyObject *found = PyObject_GetAttr(o, name);
        if(!found)
        {
            PyErr_Clear();
            throw Refused();
        }
        held.objects[held.count++] = found;
        return tensor(found);
    }
};

struct Place
{
    int device;
    nntile_b200_stream_t stream;

    explicit Place(const at::Tensor &t)
    {
        check(t.is_cuda());
        device = t.get_device();
        check(c10::cuda::current_device() == device);
        stream = c10::cuda::getCurrentCUDAStream(device).stream();
    }
};

int64_t table_blocks(const at::Tensor &lengths, const at::Tensor &table, int64_t batch)
{
    check(lengths.scalar_type() == at::kInt && table.scalar_type() == at::kInt);
    check(lengths.dim() == 1 && lengths.size(0) == batch && table.dim() == 2
            && table.size(0) == batch);
    return table.size(1);
}

uint32_t *status_word(const at::Tensor *t, int device)
{
    check(!t || ((t->scalar_type() == at::kInt || t->scalar_type() == at::kUInt32)
            && t->numel() == 1));
    return address<uint32_t>(t, device);
}

PyObject *answer(int status)
{
    if(status != 0)
    {
        return PyLong_FromLong(status);
    }
    Py_RETURN_TRUE;
}

// Memory of the current device and stream, as at::empty takes it, but without the dispatcher's
// share of its time (1.2 us a tensor, of 3 for the rest of a call).
at::Tensor result(at::IntArrayRef sizes, at::ScalarType type)
{
    return at::detail::empty_generic(sizes, c10::cuda::CUDACachingAllocator::get(),
            c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}

// The caller's, or one for this call: kernels that are in the stream when it goes back to the
// allocator are done before the next use of it there.
struct Workspace
{
    c10::DataPtr made;
    void *at;
    size_t bytes;

    Workspace(const at::Tensor *given, size_t wanted, int device)
    {
        if(given)
        {
            at = address<void>(given, device);
            bytes = given->nbytes();
        }
        else
        {
            bytes = wanted < 16 ? 16 : wanted;
            made = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
            at = made.get();
        }
    }
};

template<typename F>
PyObject *guarded(Py_ssize_t got, Py_ssize_t wanted, F &&f)
{
    try
    {
        check(got == wanted);
        return f();
    }
    catch(const Refused &)
    {
        Py_RETURN_NONE;
    }
    catch(const std::exception &)
    {
        Py_RETURN_NONE;                          // such as no memory: raised again, in Python
    }
}

// (pages, lengths, block_table, k, v, new_lens, status)
PyObject *append(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded(n, 7, [&]() -> PyObject *
    {
        const Pages p(args[0]);
        const at::Tensor &lengths = need(args[1]), &table = need(args[2]);
        const at::Tensor &k = need(args[3]), &v = need(args[4]), *lens = tensor(args[5]);
        check(k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == p.kv_heads
                && k.size(3) == p.head && v.scalar_type() == k.scalar_type());
        p.rows(k);
        check(!p.bounds || p.bounds->scalar_type() == k.scalar_type());
        const int64_t batch = k.size(1), blocks = table_blocks(lengths, table, batch);
        check(!lens || (lens->scalar_type() == at::kInt && lens->dim() == 1
                && lens->size(0) == batch));
        const Place at(k);
        const int d = at.device;
        auto entry = k.scalar_type() == at::kHalf ? nntile_b200_paged_kv_append_fp16
                : nntile_b200_paged_kv_append_bf16;
        return answer(entry(at.stream, p.head, p.page_size, p.num_pages, blocks, batch,
                p.kv_heads, k.size(2), p.e4m3, address<int32_t>(&lengths, d),
                address<int32_t>(lens, d), address<int32_t>(&table, d), address<void>(&k, d),
                address<void>(&v, d), address<void>(p.k, d), address<void>(p.v, d),
                address<uint8_t>(p.k_scales, d), address<uint8_t>(p.v_scales, d),
                address<void>(p.bounds, d), status_word(tensor(args[6]), d)));
    });
}

// (pages, lengths, block_table, k, v, status)
PyObject *gather(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded(n, 6, [&]() -> PyObject *
    {
        const Pages p(args[0]);
        const at::Tensor &lengths = need(args[1]), &table = need(args[2]);
        const at::Tensor &k = need(args[3]), &v = need(args[4]);
        check(k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == p.kv_heads
                && k.size(3) == p.head && v.scalar_type() == k.scalar_type());
        p.rows(k);
        const int64_t batch = k.size(1), blocks = table_blocks(lengths, table, batch);
        const Place at(k);
        const int d = at.device;
        auto entry = k.scalar_type() == at::kHalf ? nntile_b200_paged_kv_gather_fp16
                : nntile_b200_paged_kv_gather_bf16;
        return answer(entry(at.stream, p.head, p.page_size, p.num_pages, blocks, batch,
                p.kv_heads, k.size(2), p.e4m3, address<int32_t>(&lengths, d),
                address<int32_t>(&table, d), address<void>(p.k, d), address<void>(p.v, d),
                address<uint8_t>(p.k_scales, d), address<uint8_t>(p.v_scales, d),
                address<void>(&k, d), address<void>(&v, d), status_word(tensor(args[5]), d)));
    });
}

void check_query(const at::Tensor &q, const Pages &p)
{
    check(q.dim() == 5 && q.size(0) == p.kv_heads && q.size(3) == 1 && q.size(4) == p.head);
    p.rows(q);
}

// (q, pages, lengths, block_table, num_selected, first_blocks, last_blocks, out, workspace,
// status); answers the selection
PyObject *select(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded(n, 10, [&]() -> PyObject *
    {
        const at::Tensor &q = need(args[0]);
        const Pages p(args[1]);
        const at::Tensor &lengths = need(args[2]), &table = need(args[3]);
        const int64_t count = number(args[4]), first = number(args[5]), last = number(args[6]);
        const at::Tensor *given = tensor(args[7]), *ws = tensor(args[8]);
        check_query(q, p);
        check(p.bounds && p.bounds->scalar_type() == q.scalar_type() && count >= 0);
        const int64_t group = q.size(1), batch = q.size(2);
        check(group > 0 || given);               // otherwise there is a result to fill in
        const int64_t blocks = table_blocks(lengths, table, batch);
        check(!given || (given->scalar_type() == at::kInt && given->dim() == 3
                && given->size(0) == p.kv_heads && given->size(1) == batch
                && given->size(2) == count));
        const Place at(q);
        const int d = at.device;
        at::Tensor made;
        if(!given)
        {
            made = result({p.kv_heads, batch, count}, at::kInt);
        }
        const at::Tensor &out = given ? *given : made;
        const Workspace space(ws, nntile_b200_paged_select_workspace_bytes(blocks, batch,
                p.kv_heads), d);
        auto entry = q.scalar_type() == at::kHalf ? nntile_b200_paged_select_fp16
                : nntile_b200_paged_select_bf16;
        const int status = entry(at.stream, p.head, p.page_size, p.num_pages, blocks, batch,
                group, p.kv_heads, count, first, last, address<int32_t>(&lengths, d),
                address<int32_t>(&table, d), address<void>(&q, d), address<void>(p.bounds, d),
                address<int32_t>(&out, d), space.at, space.bytes,
                status_word(tensor(args[9]), d));
        if(status != 0)
        {
            return answer(status);
        }
        if(given)
        {
            Py_INCREF(args[7]);
            return args[7];
        }
        return THPVariable_Wrap(out);
    });
}

// (q, pages, lengths, block_table, selected, out, lse_out, workspace, status); answers out
PyObject *decode(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded(n, 9, [&]() -> PyObject *
    {
        const at::Tensor &q = need(args[0]);
        const Pages p(args[1]);
        const at::Tensor &lengths = need(args[2]), &table = need(args[3]);
        const at::Tensor *selected = tensor(args[4]), *given = tensor(args[5]);
        const at::Tensor *lse = tensor(args[6]), *ws = tensor(args[7]);
        check_query(q, p);
        const int64_t group = q.size(1), batch = q.size(2);
        const int64_t blocks = table_blocks(lengths, table, batch);
        check(!selected || (selected->scalar_type() == at::kInt && selected->dim() == 3
                && selected->size(0) == p.kv_heads && selected->size(1) == batch
                && selected->size(2) > 0));
        check(!given || (given->sizes() == q.sizes() && given->scalar_type() == q.scalar_type()));
        check(!lse || (lse->scalar_type() == at::kFloat && lse->numel() == p.kv_heads*group*batch));
        const Place at(q);
        const int d = at.device;
        check(q.is_contiguous());
        const int64_t count = selected ? selected->size(2) : 0;
        at::Tensor made;
        if(!given)
        {
            made = result(q.sizes(), q.scalar_type());
        }
        const at::Tensor &out = given ? *given : made;
        const Workspace space(ws, nntile_b200_paged_decode_sdpa_workspace_bytes(p.head,
                p.page_size, blocks, batch, group, p.kv_heads, count), d);
        auto entry = q.scalar_type() == at::kHalf ? nntile_b200_paged_decode_sdpa_fp16
                : nntile_b200_paged_decode_sdpa_bf16;
        const int status = entry(at.stream, p.head, p.page_size, p.num_pages, blocks, batch,
                group, p.kv_heads, count, p.e4m3, address<int32_t>(&lengths, d),
                address<int32_t>(&table, d), address<int32_t>(selected, d),
                address<void>(&q, d), address<void>(p.k, d), address<void>(p.v, d),
                address<uint8_t>(p.k_scales, d), address<uint8_t>(p.v_scales, d),
                address<void>(&out, d), address<float>(lse, d), space.at, space.bytes,
                status_word(tensor(args[8]), d));
        if(status != 0)
        {
            return answer(status);
        }
        if(given)
        {
            Py_INCREF(args[5]);
            return args[5];
        }
        return THPVariable_Wrap(out);
    });
}

PyMethodDef methods[] = {
    {"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL, nullptr},
    {"gather", (PyCFunction)(void (*)(void))gather, METH_FASTCALL, nullptr},
    {"select", (PyCFunction)(void (*)(void))select, METH_FASTCALL, nullptr},
    {"decode", (PyCFunction)(void (*)(void))decode, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_torch", nullptr, -1, methods, nullptr,
        nullptr, nullptr, nullptr};

} // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__paged_torch(void)
{
    name_k = PyUnicode_InternFromString("k");
    name_v = PyUnicode_InternFromString("v");
    name_k_scales = PyUnicode_InternFromString("k_scales");
    name_v_scales = PyUnicode_InternFromString("v_scales");
    name_bounds = PyUnicode_InternFromString("bounds");
    return PyModule_Create(&module);
}
