// Fast path of the operators around attention (cudalab_amd/attention.py): one
// call from Python checks the tensors on their metadata, fills the C call's
// arguments and makes it on the current HIP stream of the tensors' device.
// As in cq_pyfast.cpp, this decides no error: whatever it does not accept is
// "not taken" (None / false), nothing launched, and the Python layer's checked
// path raises its message.  Only a launch that HIP refuses raises here.
//
// A call costs 3 to 5 us of host time this way, against 15 to 20 us through
// the Python checks and ctypes (MI355X host).
#pragma once

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "cdnaqgemv.h"

namespace cqattn {
namespace {

namespace py = pybind11;

int dtype_code(at::ScalarType t) {
    return t == at::kHalf ? CQ_DTYPE_F16 : t == at::kBFloat16 ? CQ_DTYPE_BF16
           : t == at::kFloat ? CQ_DTYPE_F32 : -1;
}

// A tensor argument, or null for None; `ok` turns false for anything else.
const at::Tensor* tensor(py::handle o, bool optional, bool& ok) {
    if (THPVariable_Check(o.ptr())) {
        const at::Tensor& t = THPVariable_Unpack(o.ptr());
        if (t.defined() && t.layout() == at::kStrided) return &t;
    } else if (optional && o.is_none()) {
        return nullptr;
    }
    ok = false;
    return nullptr;
}

bool on_current(const at::Tensor& t) {
    const c10::Device d = t.device();
    return d.is_cuda() && d.index() == c10::hip::current_device();
}

void* stream_of(const at::Tensor& t) {
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

bool last_contiguous(const at::Tensor& t) {
    const int64_t n = t.dim();
    return t.size(n - 1) <= 1 || t.stride(n - 1) == 1;
}

bool ints(const at::Tensor& t, int64_t n, const c10::Device& d) {
    return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous() &&
           t.device() == d;
}

bool table_ok(const at::Tensor& t, int64_t batch, const c10::Device& d) {
    return t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == batch && t.size(1) >= 1 &&
           t.size(1) <= INT32_MAX && (t.size(1) == 1 || t.stride(1) == 1) && t.device() == d;
}

// A checked cache (KVCache checks the tensors and keeps them alive).
struct Cache {
    cq_kv_cache_t c;
    c10::Device device;
    Cache(py::handle k, int64_t v, int64_t scales, int64_t pages, int64_t heads, int64_t dim,
          int64_t page, int64_t bits)
        : c{}, device(THPVariable_Unpack(k.ptr()).device()) {
        c.k = THPVariable_Unpack(k.ptr()).data_ptr();
        c.v = reinterpret_cast<void*>(v);
        c.scales = reinterpret_cast<float*>(scales);
        c.pages = pages;
        c.heads = static_cast<int32_t>(heads);
        c.head_dim = static_cast<int32_t>(dim);
        c.page_size = static_cast<int32_t>(page);
        c.bits = static_cast<int32_t>(bits);
    }
};

class Calls {
public:
    Calls(uintptr_t norm_rope, uintptr_t append, uintptr_t read, uintptr_t attention,
          uintptr_t workspace, uintptr_t tree, uintptr_t tree_workspace, uintptr_t last_error)
        : norm_rope_(reinterpret_cast<decltype(norm_rope_)>(norm_rope)),
          append_(reinterpret_cast<decltype(append_)>(append)),
          read_(reinterpret_cast<decltype(read_)>(read)),
          attention_(reinterpret_cast<decltype(attention_)>(attention)),
          workspace_(reinterpret_cast<decltype(workspace_)>(workspace)),
          tree_(reinterpret_cast<decltype(tree_)>(tree)),
          tree_workspace_(reinterpret_cast<decltype(tree_workspace_)>(tree_workspace)),
          last_error_(reinterpret_cast<decltype(last_error_)>(last_error)) {}

    // (q_out, k_out), or None; outputs None: new ones.
    py::object norm_rope(py::handle q_, py::handle k_, py::handle qo_, py::handle ko_,
                         py::handle qw_, py::handle kw_, py::handle cos_, py::handle sin_,
                         py::handle pos_, double eps, bool interleaved) const {
        bool ok = true;
        const at::Tensor *q = tensor(q_, false, ok), *k = tensor(k_, false, ok);
        const at::Tensor *qo = tensor(qo_, true, ok), *ko = tensor(ko_, true, ok);
        const at::Tensor *qw = tensor(qw_, true, ok), *kw = tensor(kw_, true, ok);
        const at::Tensor *cos = tensor(cos_, true, ok), *sin = tensor(sin_, true, ok);
        const at::Tensor* pos = tensor(pos_, true, ok);
        if (!ok || q->dim() != 3 || !on_current(*q)) return py::none();
        const c10::Device dev = q->device();
        const int64_t tokens = q->size(0), D = q->size(2);
        const int dt = dtype_code(q->scalar_type());
        if (dt < 0 || tokens < 1 || !row(*q, *q) || !row(*k, *q) || k->size(0) != tokens ||
            k->size(2) != D || q->size(1) > INT32_MAX || k->size(1) > INT32_MAX || D > INT32_MAX)
            return py::none();
        cq_norm_rope_t a{};
        const at::Tensor* w = qw != nullptr ? qw : kw;
        for (const at::Tensor* x : {qw, kw})
            if (x != nullptr && (x->dim() != 1 || x->size(0) != D || !x->is_contiguous() ||
                                 x->device() != dev || x->scalar_type() != w->scalar_type()))
                return py::none();
        a.weight_dtype = w != nullptr ? dtype_code(w->scalar_type()) : CQ_DTYPE_F32;
        if (a.weight_dtype < 0) return py::none();
        if (cos != nullptr || sin != nullptr || pos != nullptr) {
            if (cos == nullptr || sin == nullptr || pos == nullptr) return py::none();
            for (const at::Tensor* x : {cos, sin})
                if (x->scalar_type() != at::kFloat || x->dim() != 2 || !x->is_contiguous() ||
                    x->device() != dev)
                    return py::none();
            const at::ScalarType pt = pos->scalar_type();
            if (cos->sizes() != sin->sizes() || cos->size(0) < 1 || cos->size(1) < 1 ||
                2 * cos->size(1) > D || (pt != at::kInt && pt != at::kLong) || pos->dim() != 1 ||
                pos->size(0) != tokens || !pos->is_contiguous() || pos->device() != dev)
                return py::none();
            a.cos_table = static_cast<const float*>(cos->data_ptr());
            a.sin_table = static_cast<const float*>(sin->data_ptr());
            a.positions = pos->data_ptr();
            a.positions_64 = pt == at::kLong;
            a.table_rows = cos->size(0);
            a.rot_dim = static_cast<int32_t>(2 * cos->size(1));
        }
        at::Tensor nq, nk;
        if (qo == nullptr) {
            nq = at::empty(q->sizes(), q->options());
            qo = &nq;
        }
        if (ko == nullptr) {
            nk = at::empty(k->sizes(), k->options());
            ko = &nk;
        }
        if (!row(*qo, *q) || !row(*ko, *q) || qo->sizes() != q->sizes() ||
            ko->sizes() != k->sizes())
            return py::none();
        a.q = q->data_ptr(), a.k = k->data_ptr();
        a.q_out = qo->data_ptr(), a.k_out = ko->data_ptr();
        a.q_token_stride = q->stride(0), a.q_head_stride = q->stride(1);
        a.k_token_stride = k->stride(0), a.k_head_stride = k->stride(1);
        a.q_out_token_stride = qo->stride(0), a.q_out_head_stride = qo->stride(1);
        a.k_out_token_stride = ko->stride(0), a.k_out_head_stride = ko->stride(1);
        a.q_weight = qw != nullptr ? qw->data_ptr() : nullptr;
        a.k_weight = kw != nullptr ? kw->data_ptr() : nullptr;
        a.tokens = tokens;
        a.q_heads = static_cast<int32_t>(q->size(1));
        a.k_heads = static_cast<int32_t>(k->size(1));
        a.head_dim = static_cast<int32_t>(D);
        a.dtype = dt;
        a.interleaved = interleaved;
        a.eps = static_cast<float>(eps);
        if (!done(norm_rope_(&a, stream_of(*q)), "qk_norm_rope")) return py::none();
        return py::make_tuple(*qo, *ko);
    }

    bool append(const Cache& c, py::handle k_, py::handle v_, py::handle table, py::handle starts,
                py::handle counts) const {
        bool ok = true;
        const at::Tensor *k = tensor(k_, false, ok), *v = tensor(v_, false, ok);
        if (!ok || k->dim() != 4 || k->sizes() != v->sizes() ||
            k->scalar_type() != v->scalar_type() || k->device() != c.device ||
            v->device() != c.device || !on_current(*k) || !last_contiguous(*k) ||
            !last_contiguous(*v) || k->size(2) != c.c.heads || k->size(3) != c.c.head_dim)
            return false;
        const int dt = dtype_code(k->scalar_type());
        cq_kv_slots_t s{};
        if (dt < 0 || !slots(c, table, starts, counts, k->size(0), k->size(1), s)) return false;
        return done(append_(&c.c, &s, dt, k->data_ptr(), k->stride(0), k->stride(1), k->stride(2),
                            v->data_ptr(), v->stride(0), v->stride(1), v->stride(2),
                            stream_of(*k)),
                    "append");
    }

    // (k, v), or None.
    py::object read(const Cache& c, py::handle table, py::handle starts, py::handle counts,
                    py::handle tokens_, py::handle dtype) const {
        bool ok = true;
        const at::Tensor* st = tensor(starts, false, ok);
        if (!ok || st->dim() != 1 || !PyLong_CheckExact(tokens_.ptr()) ||
            !THPDtype_Check(dtype.ptr()) || !on_current(*st))
            return py::none();
        const int64_t tokens = PyLong_AsLongLong(tokens_.ptr());
        if (tokens < 0) {
            PyErr_Clear();
            return py::none();
        }
        const at::ScalarType type = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
        cq_kv_slots_t s{};
        if (dtype_code(type) < 0 || !slots(c, table, starts, counts, st->size(0), tokens, s))
            return py::none();
        const auto options = st->options().dtype(type);
        at::Tensor k = at::empty({st->size(0), tokens, c.c.heads, c.c.head_dim}, options);
        at::Tensor v = at::empty(k.sizes(), options);
        if (!done(read_(&c.c, &s, dtype_code(type), k.data_ptr(), v.data_ptr(), stream_of(*st)),
                  "read"))
            return py::none();
        return py::make_tuple(k, v);
    }

    // out (a new one for None), or None.
    py::object forward(const Cache& c, py::handle q_, py::handle table_, py::handle lengths_,
                       py::handle counts_, py::handle out_, py::handle pages_,
                       int64_t prefix_len, double scale, py::handle seen_) const {
        bool ok = true;
        const at::Tensor *q = tensor(q_, false, ok), *out = tensor(out_, true, ok);
        const at::Tensor *table = tensor(table_, false, ok), *len = tensor(lengths_, false, ok);
        const at::Tensor *counts = tensor(counts_, true, ok), *pages = tensor(pages_, true, ok);
        const at::Tensor* seen = tensor(seen_, true, ok);
        if (!ok || q->dim() != 4 || q->device() != c.device || !on_current(*q) ||
            !last_contiguous(*q))
            return py::none();
        const at::ScalarType type = q->scalar_type();
        const int64_t batch = q->size(0), tokens = q->size(1), heads = q->size(2);
        if ((type != at::kHalf && type != at::kBFloat16) || batch < 1 || tokens < 1 ||
            heads < 1 || batch > INT32_MAX || tokens > INT32_MAX || heads > 65535 ||
            heads % c.c.heads != 0 || q->size(3) != c.c.head_dim)
            return py::none();
        if (!table_ok(*table, batch, c.device) || !ints(*len, batch, c.device) ||
            (counts != nullptr && !ints(*counts, batch, c.device)))
            return py::none();
        if (seen != nullptr &&
            (seen->scalar_type() != at::kLong || seen->dim() != 3 || seen->size(0) != batch ||
             seen->size(1) != tokens || seen->size(2) != (tokens + 63) / 64 ||
             !seen->is_contiguous() || seen->device() != c.device))
            return py::none();
        cq_attention_t a{};
        if (pages != nullptr) {
            if (!ints(*pages, pages->numel(), c.device) || prefix_len < 0 ||
                prefix_len > INT32_MAX || pages->numel() > INT32_MAX ||
                prefix_len > pages->numel() * c.c.page_size)
                return py::none();
            a.prefix_table = prefix_len > 0 ? static_cast<const int32_t*>(pages->data_ptr()) : nullptr;
            a.prefix_cols = static_cast<int32_t>(pages->numel());
            a.prefix_len = static_cast<int32_t>(prefix_len);
        }
        if (q->stride(0) % 8 != 0 || q->stride(1) % 8 != 0 || q->stride(2) % 8 != 0 ||
            reinterpret_cast<uintptr_t>(q->data_ptr()) % 16 != 0)
            return py::none();
        at::Tensor made;
        if (out == nullptr) {
            made = at::empty(q->sizes(), q->options());
            out = &made;
        }
        if (out->scalar_type() != type || out->device() != c.device ||
            out->sizes() != q->sizes() || !out->is_contiguous())
            return py::none();
        a.q = q->data_ptr(), a.out = out->data_ptr();
        a.q_batch_stride = q->stride(0);
        a.q_token_stride = q->stride(1);
        a.q_head_stride = q->stride(2);
        a.table = static_cast<const int32_t*>(table->data_ptr());
        a.lengths = static_cast<const int32_t*>(len->data_ptr());
        a.counts = counts != nullptr ? static_cast<const int32_t*>(counts->data_ptr()) : nullptr;
        a.table_stride = table->stride(0);
        a.table_cols = static_cast<int32_t>(table->size(1));
        a.batch = static_cast<int32_t>(batch);
        a.tokens = static_cast<int32_t>(tokens);
        a.q_heads = static_cast<int32_t>(heads);
        a.dtype = dtype_code(type);
        a.softmax_scale = static_cast<float>(scale);
        const int64_t need = (seen == nullptr ? workspace_ : tree_workspace_)(&c.c, &a);
        if (need < 0) return py::none();
        at::Tensor ws;      // given back at the end: work queued behind on this stream follows
        if (need > 0) {
            ws = at::empty({need}, q->options().dtype(at::kByte));
            a.workspace = ws.data_ptr();
            a.workspace_bytes = need;
        }
        void* const stream = stream_of(*q);
        const int status = seen == nullptr
                               ? attention_(&c.c, &a, stream)
                               : tree_(&c.c, &a, static_cast<const int64_t*>(seen->data_ptr()), stream);
        if (!done(status, "forward")) return py::none();
        return py::cast(*out);
    }

private:
    // [tokens, heads, D] of q's type and device, heads side by side inside.
    static bool row(const at::Tensor& t, const at::Tensor& q) {
        return t.dim() == 3 && t.scalar_type() == q.scalar_type() && t.device() == q.device() &&
               last_contiguous(t);
    }

    static bool slots(const Cache& c, py::handle table_, py::handle starts_, py::handle counts_,
                      int64_t batch, int64_t tokens, cq_kv_slots_t& s) {
        bool ok = true;
        const at::Tensor *table = tensor(table_, false, ok), *starts = tensor(starts_, false, ok);
        const at::Tensor* counts = tensor(counts_, true, ok);
        if (!ok || batch < 1 || tokens < 1 || batch > INT32_MAX || tokens > INT32_MAX ||
            !table_ok(*table, batch, c.device) || !ints(*starts, batch, c.device) ||
            (counts != nullptr && !ints(*counts, batch, c.device)))
            return false;
        s.table = static_cast<const int32_t*>(table->data_ptr());
        s.starts = static_cast<const int32_t*>(starts->data_ptr());
        s.counts = counts != nullptr ? static_cast<const int32_t*>(counts->data_ptr()) : nullptr;
        s.table_stride = table->stride(0);
        s.table_cols = static_cast<int32_t>(table->size(1));
        s.batch = static_cast<int32_t>(batch);
        s.tokens = static_cast<int32_t>(tokens);
        return true;
    }

    bool done(int status, const char* what) const {
        if (status == CQ_ERR_HIP)
            throw std::runtime_error(std::string(what) + " failed (status " +
                                     std::to_string(status) + "): " + last_error_());
        return status == CQ_OK;
    }

    int (*norm_rope_)(const cq_norm_rope_t*, void*);
    int (*append_)(const cq_kv_cache_t*, const cq_kv_slots_t*, int, const void*, int64_t, int64_t,
                   int64_t, const void*, int64_t, int64_t, int64_t, void*);
    int (*read_)(const cq_kv_cache_t*, const cq_kv_slots_t*, int, void*, void*, void*);
    int (*attention_)(const cq_kv_cache_t*, const cq_attention_t*, void*);
    int64_t (*workspace_)(const cq_kv_cache_t*, const cq_attention_t*);
    int (*tree_)(const cq_kv_cache_t*, const cq_attention_t*, const int64_t*, void*);
    int64_t (*tree_workspace_)(const cq_kv_cache_t*, const cq_attention_t*);
    const char* (*last_error_)();
};

void bind(py::module_& m) {
    py::class_<Cache>(m, "Cache")
        .def(py::init<py::handle, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t>());
    py::class_<Calls>(m, "AttentionCalls")
        .def(py::init<uintptr_t, uintptr_t, uintptr_t, uintptr_t, uintptr_t, uintptr_t,
                      uintptr_t, uintptr_t>())
        .def("norm_rope", &Calls::norm_rope)
        .def("append", &Calls::append)
        .def("read", &Calls::read)
        .def("forward", &Calls::forward);
}

}  // namespace
}  // namespace cqattn
