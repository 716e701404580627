// Fast path of the operators of a step of many tokens (cudalab_amd/attention.py,
// cudalab_amd/qgemm.py), as in cq_pyattn.h: whatever it does not accept is "not
// taken", nothing launched, and the Python layer's checked path raises.
#pragma once

#include "cq_pyattn.h"

namespace cqstep {
namespace {

namespace py = pybind11;
using cqattn::Cache;
using cqattn::dtype_code;
using cqattn::ints;
using cqattn::last_contiguous;
using cqattn::on_current;
using cqattn::stream_of;
using cqattn::table_ok;
using cqattn::tensor;

// An int that Python holds as one, not below zero; else -1.
int64_t count(py::handle o) {
    if (!PyLong_CheckExact(o.ptr())) return -1;
    const int64_t n = PyLong_AsLongLong(o.ptr());
    if (n < 0) PyErr_Clear();
    return n < 0 ? -1 : n;
}

// `n` elements of a contiguous 1-D tensor from element `from` on, as a tensor of the same
// storage (a view without the dispatcher's work: about 0.1 us instead of an allocation's
// 0.7).
at::Tensor part_of(const at::Tensor& t, int64_t from, int64_t n) {
    at::Tensor part = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()),
                                                               t.key_set(), t.dtype());
    part.unsafeGetTensorImpl()->set_storage_offset(t.storage_offset() + from);
    part.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return part;
}

class Calls {
public:
    Calls(uintptr_t place, uintptr_t place_held, uintptr_t append_rows, uintptr_t prompt, uintptr_t last_error)
        : place_(reinterpret_cast<decltype(place_)>(place)),
          place_held_(reinterpret_cast<decltype(place_held_)>(place_held)),
          append_rows_(reinterpret_cast<decltype(append_rows_)>(append_rows)),
          prompt_(reinterpret_cast<decltype(prompt_)>(prompt)),
          last_error_(reinterpret_cast<decltype(last_error_)>(last_error)) {}

    // (slots, positions, offsets, lengths, taken), with `held` also the next held, or None.
    py::object place(py::handle table_, py::handle starts_, py::handle counts_,
                     py::handle tokens_, py::handle page_, py::handle free_,
                     py::handle taken_, py::handle held_) const {
        bool ok = true;
        const at::Tensor *table = tensor(table_, false, ok), *starts = tensor(starts_, false, ok);
        const at::Tensor *counts = tensor(counts_, false, ok), *free = tensor(free_, false, ok);
        const at::Tensor *taken = tensor(taken_, true, ok), *held = tensor(held_, true, ok);
        const int64_t tokens = count(tokens_), page = count(page_);
        if (!ok || table->dim() != 2 || !on_current(*table) || tokens < 0 || tokens > INT32_MAX ||
            page < 16 || page > 256)
            return py::none();
        const c10::Device dev = table->device();
        const int64_t batch = table->size(0);
        if (batch < 1 || batch >= INT32_MAX || !table_ok(*table, batch, dev) ||
            !ints(*starts, batch, dev) || !ints(*counts, batch, dev) ||
            !ints(*free, free->numel(), dev) || (taken != nullptr && !ints(*taken, 1, dev)) ||
            (held != nullptr && !ints(*held, batch, dev)))
            return py::none();
        const auto options = starts->options();
        at::Tensor slots = at::empty({tokens}, options.dtype(at::kLong));
        // the others side by side
        const at::Tensor all =
            at::empty({tokens + (held != nullptr ? 3 : 2) * batch + 2}, options);
        at::Tensor positions = part_of(all, 0, tokens), offsets = part_of(all, tokens, batch + 1);
        at::Tensor lengths = part_of(all, tokens + batch + 1, batch);
        at::Tensor gone = part_of(all, tokens + 2 * batch + 1, 1);
        auto data = [](const at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
        cq_place_t a{};
        a.starts = data(*starts), a.counts = data(*counts), a.free_pages = data(*free);
        a.taken_in = taken != nullptr ? data(*taken) : nullptr;
        a.table = data(*table);
        a.slots = static_cast<int64_t*>(slots.data_ptr());
        a.positions = data(positions), a.offsets = data(offsets), a.lengths = data(lengths);
        a.taken_out = data(gone);
        a.table_stride = table->stride(0);
        a.tokens = tokens;
        a.free_count = free->numel();
        a.table_cols = static_cast<int32_t>(table->size(1));
        a.batch = static_cast<int32_t>(batch);
        a.page_size = static_cast<int32_t>(page);
        if (held != nullptr) {
            at::Tensor owned = part_of(all, tokens + 2 * batch + 2, batch);
            if (!done(place_held_(&a, data(*held), data(owned), stream_of(*table)), "place"))
                return py::none();
            return py::make_tuple(slots, positions, offsets, lengths, gone, owned);
        }
        if (!done(place_(&a, stream_of(*table)), "place")) return py::none();
        return py::make_tuple(slots, positions, offsets, lengths, gone);
    }

    bool append_rows(const Cache& c, py::handle k_, py::handle v_, py::handle slots_) const {
        bool ok = true;
        const at::Tensor *k = tensor(k_, false, ok), *v = tensor(v_, false, ok);
        const at::Tensor* slots = tensor(slots_, false, ok);
        if (!ok || k->dim() != 3 || k->sizes() != v->sizes() ||
            k->scalar_type() != v->scalar_type() || k->device() != c.device ||
            v->device() != c.device || !on_current(*k) || !last_contiguous(*k) ||
            !last_contiguous(*v) || k->size(1) != c.c.heads || k->size(2) != c.c.head_dim)
            return false;
        const int dt = dtype_code(k->scalar_type());
        const int64_t tokens = k->size(0);
        if (dt < 0 || tokens < 1 || slots->scalar_type() != at::kLong || slots->dim() != 1 ||
            slots->size(0) != tokens || !slots->is_contiguous() || slots->device() != c.device)
            return false;
        return done(append_rows_(&c.c, dt, tokens, static_cast<const int64_t*>(slots->data_ptr()),
                                 k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(),
                                 v->stride(0), v->stride(1), stream_of(*k)),
                    "append_rows");
    }

    // out (a new one for None), or None.
    py::object prompt(py::handle q_, py::handle k_, py::handle v_, py::handle offsets_,
                      py::handle out_, py::handle k_offsets_, bool causal, py::handle scale) const {
        bool ok = true;
        const at::Tensor *q = tensor(q_, false, ok), *k = tensor(k_, false, ok);
        const at::Tensor *v = tensor(v_, false, ok), *offsets = tensor(offsets_, false, ok);
        const at::Tensor *out = tensor(out_, true, ok), *koff = tensor(k_offsets_, true, ok);
        if (!ok || q->dim() != 3 || k->dim() != 3 || v->sizes() != k->sizes() || !on_current(*q) ||
            offsets->dim() != 1)
            return py::none();
        const c10::Device dev = q->device();
        const at::ScalarType type = q->scalar_type();
        const int64_t tokens = q->size(0), heads = q->size(1), D = q->size(2);
        const int64_t keys = k->size(0), batch = offsets->size(0) - 1;
        if ((type != at::kHalf && type != at::kBFloat16) || tokens < 1 || batch < 1 ||
            batch >= INT32_MAX || heads < 1 || heads > 65535 || k->size(1) < 1 ||
            heads % k->size(1) != 0 || k->size(2) != D || D > 256 || (koff == nullptr && keys != tokens))
            return py::none();
        for (const at::Tensor* t : {q, k, v})
            if (t->scalar_type() != type || t->device() != dev || !last_contiguous(*t) ||
                t->stride(0) % 8 != 0 || t->stride(1) % 8 != 0 ||
                reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 != 0)
                return py::none();
        if (!ints(*offsets, batch + 1, dev) || (koff != nullptr && !ints(*koff, batch + 1, dev)))
            return py::none();
        at::Tensor made;
        if (out == nullptr) {
            made = at::empty(q->sizes(), q->options());
            out = &made;
        }
        if (out->scalar_type() != type || out->device() != dev || out->sizes() != q->sizes() ||
            !out->is_contiguous())
            return py::none();
        cq_prompt_t a{};
        a.q = q->data_ptr(), a.k = k->data_ptr(), a.v = v->data_ptr(), a.out = out->data_ptr();
        a.q_token_stride = q->stride(0), a.q_head_stride = q->stride(1);
        a.k_token_stride = k->stride(0), a.k_head_stride = k->stride(1);
        a.v_token_stride = v->stride(0), a.v_head_stride = v->stride(1);
        a.q_offsets = static_cast<const int32_t*>(offsets->data_ptr());
        a.k_offsets = koff != nullptr ? static_cast<const int32_t*>(koff->data_ptr()) : nullptr;
        a.q_tokens = tokens;
        a.k_tokens = keys;
        a.batch = static_cast<int32_t>(batch);
        a.q_heads = static_cast<int32_t>(heads);
        a.k_heads = static_cast<int32_t>(k->size(1));
        a.head_dim = static_cast<int32_t>(D);
        a.dtype = dtype_code(type);
        a.causal = causal;
        a.softmax_scale = scale.is_none() ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(D)))
                                          : static_cast<float>(PyFloat_AsDouble(scale.ptr()));
        if (!done(prompt_(&a, stream_of(*q)), "prompt")) return py::none();
        return py::cast(*out);
    }

private:
    bool done(int status, const char* what) const {
        if (status == CQ_ERR_HIP)
            throw std::runtime_error(std::string(what) + " failed (status " +
                                     std::to_string(status) + "): " + last_error_());
        return status == CQ_OK;
    }

    int (*place_)(const cq_place_t*, void*);
    int (*place_held_)(const cq_place_t*, const int32_t*, int32_t*, void*);
    int (*append_rows_)(const cq_kv_cache_t*, int, int64_t, const int64_t*, const void*, int64_t,
                        int64_t, const void*, int64_t, int64_t, void*);
    int (*prompt_)(const cq_prompt_t*, void*);
    const char* (*last_error_)();
};

class Qgemm {
public:
    Qgemm(uintptr_t quantize, uintptr_t gemm, uintptr_t workspace, uintptr_t last_error)
        : quantize_(reinterpret_cast<decltype(quantize_)>(quantize)),
          gemm_(reinterpret_cast<decltype(gemm_)>(gemm)),
          workspace_(reinterpret_cast<decltype(workspace_)>(workspace)),
          last_error_(reinterpret_cast<decltype(last_error_)>(last_error)) {}

    // (codes, scales), or None.
    py::object quantize(py::handle x_) const {
        bool ok = true;
        const at::Tensor* x = tensor(x_, false, ok);
        if (!ok || x->dim() != 2 || !on_current(*x) || !last_contiguous(*x)) return py::none();
        const int dt = dtype_code(x->scalar_type());
        const int64_t tokens = x->size(0), k = x->size(1);
        if (dt < 0 || tokens < 1 || k < 1) return py::none();
        at::Tensor codes = at::empty({tokens, k}, x->options().dtype(at::kChar));
        at::Tensor scales = at::empty({tokens}, x->options().dtype(at::kFloat));
        if (!done(quantize_(dt, x->data_ptr(), x->stride(0), tokens, k,
                            static_cast<int8_t*>(codes.data_ptr()),
                            static_cast<float*>(scales.data_ptr()), stream_of(*x)),
                  "quantize_tokens"))
            return py::none();
        return py::make_tuple(codes, scales);
    }

    // out (a new one of `dtype` for None), or None.
    py::object forward(py::handle codes_, py::handle scales_, py::handle w_, py::handle scale_,
                       py::handle out_, py::handle dtype) const {
        bool ok = true;
        const at::Tensor *x = tensor(codes_, false, ok), *xs = tensor(scales_, false, ok);
        const at::Tensor *w = tensor(w_, false, ok), *ws = tensor(scale_, false, ok);
        const at::Tensor* out = tensor(out_, true, ok);
        if (!ok || x->dim() != 2 || w->dim() != 2 || x->scalar_type() != at::kChar ||
            w->scalar_type() != at::kChar || !on_current(*w) || x->device() != w->device())
            return py::none();
        const c10::Device dev = w->device();
        const int64_t tokens = x->size(0), n = w->size(0), k = w->size(1);
        if (tokens < 1 || n < 1 || k < 1 || x->size(1) != k || !w->is_contiguous() ||
            !last_contiguous(*x) || (tokens > 1 && x->stride(0) < k) || !scales_ok(*ws, n, dev) ||
            !scales_ok(*xs, tokens, dev))
            return py::none();
        at::Tensor made;
        if (out == nullptr) {
            if (!THPDtype_Check(dtype.ptr())) return py::none();
            const at::ScalarType type = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
            if (dtype_code(type) < 0) return py::none();
            made = at::empty({tokens, n}, w->options().dtype(type));
            out = &made;
        }
        cq_qgemm_t a{};
        a.dtype = dtype_code(out->scalar_type());
        if (a.dtype < 0 || out->dim() != 2 || out->size(0) != tokens || out->size(1) != n ||
            !out->is_contiguous() || out->device() != dev)
            return py::none();
        a.x = static_cast<const int8_t*>(x->data_ptr());
        a.x_scale = static_cast<const float*>(xs->data_ptr());
        a.w = static_cast<const int8_t*>(w->data_ptr());
        a.w_scale = static_cast<const float*>(ws->data_ptr());
        a.out = out->data_ptr();
        a.x_stride = x->stride(0) < k ? k : x->stride(0);
        a.tokens = tokens, a.n = n, a.k = k;
        const int64_t need = workspace_(&a);
        if (need < 0) return py::none();
        at::Tensor space;      // given back at the end: work queued behind on this stream follows
        if (need > 0) {
            space = at::empty({need}, w->options().dtype(at::kByte));
            a.workspace = space.data_ptr();
            a.workspace_bytes = need;
        }
        if (!done(gemm_(&a, stream_of(*w)), "forward")) return py::none();
        return py::cast(*out);
    }

private:
    static bool scales_ok(const at::Tensor& t, int64_t n, const c10::Device& d) {
        return t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == n &&
               t.is_contiguous() && t.device() == d;
    }

    bool done(int status, const char* what) const {
        if (status == CQ_ERR_HIP)
            throw std::runtime_error(std::string(what) + " failed (status " +
                                     std::to_string(status) + "): " + last_error_());
        return status == CQ_OK;
    }

    int (*quantize_)(int, const void*, int64_t, int64_t, int64_t, int8_t*, float*, void*);
    int (*gemm_)(const cq_qgemm_t*, void*);
    int64_t (*workspace_)(const cq_qgemm_t*);
    const char* (*last_error_)();
};

void bind(py::module_& m) {
    py::class_<Qgemm>(m, "QgemmCalls")
        .def(py::init<uintptr_t, uintptr_t, uintptr_t, uintptr_t>())
        .def("quantize", &Qgemm::quantize)
        .def("forward", &Qgemm::forward);
    py::class_<Calls>(m, "StepCalls")
        .def(py::init<uintptr_t, uintptr_t, uintptr_t, uintptr_t, uintptr_t>())
        .def("prompt", &Calls::prompt)
        .def("place", &Calls::place)
        .def("append_rows", &Calls::append_rows);
}

}  // namespace
}  // namespace cqstep
