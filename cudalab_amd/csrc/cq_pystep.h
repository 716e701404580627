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

class Calls {
public:
    Calls(uintptr_t place, uintptr_t append_rows, uintptr_t last_error)
        : place_(reinterpret_cast<decltype(place_)>(place)),
          append_rows_(reinterpret_cast<decltype(append_rows_)>(append_rows)),
          last_error_(reinterpret_cast<decltype(last_error_)>(last_error)) {}

    // (slots, positions, offsets, lengths, taken), or None.
    py::object place(py::handle table_, py::handle starts_, py::handle counts_,
                     py::handle tokens_, py::handle page_, py::handle free_,
                     py::handle taken_) const {
        bool ok = true;
        const at::Tensor *table = tensor(table_, false, ok), *starts = tensor(starts_, false, ok);
        const at::Tensor *counts = tensor(counts_, false, ok), *free = tensor(free_, false, ok);
        const at::Tensor* taken = tensor(taken_, true, ok);
        const int64_t tokens = count(tokens_), page = count(page_);
        if (!ok || table->dim() != 2 || !on_current(*table) || tokens < 0 || tokens > INT32_MAX ||
            page < 16 || page > 256)
            return py::none();
        const c10::Device dev = table->device();
        const int64_t batch = table->size(0);
        if (batch < 1 || batch >= INT32_MAX || !table_ok(*table, batch, dev) ||
            !ints(*starts, batch, dev) || !ints(*counts, batch, dev) ||
            !ints(*free, free->numel(), dev) || (taken != nullptr && !ints(*taken, 1, dev)))
            return py::none();
        const auto options = starts->options();
        at::Tensor slots = at::empty({tokens}, options.dtype(at::kLong));
        at::Tensor positions = at::empty({tokens}, options);
        at::Tensor offsets = at::empty({batch + 1}, options);
        at::Tensor lengths = at::empty({batch}, options), gone = at::empty({1}, options);
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

private:
    bool done(int status, const char* what) const {
        if (status == CQ_ERR_HIP)
            throw std::runtime_error(std::string(what) + " failed (status " +
                                     std::to_string(status) + "): " + last_error_());
        return status == CQ_OK;
    }

    int (*place_)(const cq_place_t*, void*);
    int (*append_rows_)(const cq_kv_cache_t*, int, int64_t, const int64_t*, const void*, int64_t,
                        int64_t, const void*, int64_t, int64_t, void*);
    const char* (*last_error_)();
};

void bind(py::module_& m) {
    py::class_<Calls>(m, "StepCalls")
        .def(py::init<uintptr_t, uintptr_t, uintptr_t>())
        .def("place", &Calls::place)
        .def("append_rows", &Calls::append_rows);
}

}  // namespace
}  // namespace cqstep
