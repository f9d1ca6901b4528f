// Python calls of the rotary and paged-cache entry points: the checks of
// arguments, the outputs and the descriptors in C++, since a decode step calls
// them for every layer and the same in Python took longer than the kernels
// (us a call, Python and ctypes / this file: rotary step of 64 sequences 13.2 /
// 5.0, append step 17.5 / 5.3, short read 12.7 / 5.6, attention over 1K tokens
// 16.0 / 7.4).  The kernels stay behind the C ABI: bind() gets the addresses of
// libfkv's functions from _native.py.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <string>

#include "../../include/fkv.h"

namespace {

using at::Tensor;

decltype(&fkv_last_error) p_error = nullptr;
decltype(&fkv_rotary) p_rotary = nullptr;
decltype(&fkv_paged_append) p_append = nullptr;
decltype(&fkv_paged_read) p_read = nullptr;
decltype(&fkv_paged_attend) p_attend = nullptr;
decltype(&fkv_paged_attend_workspace_bytes) p_attend_ws = nullptr;
PyObject* native_error = nullptr;

struct Refused {           // -> ValueError
    std::string what;
};
struct Failed {            // a negative return code -> FkvNativeError
    std::string what;
};

template <class... A>
void require(bool ok, const char* who, const A&... msg) {
    if (!ok) throw Refused{c10::str(who, ": ", msg...)};
}

void check(int rc, const char* what) {
    if (rc >= 0) return;
    const char* kind = rc == FKV_ERR_INVALID ? "invalid argument" : rc == FKV_ERR_UNSUPPORTED ? "unsupported"
                     : rc == FKV_ERR_CUDA ? "CUDA error" : "error";
    throw Failed{c10::str(what, " failed (", kind, "): ", p_error())};
}

const Tensor* maybe(PyObject* o, const char* who, const char* name) {
    if (o == Py_None) return nullptr;
    require(THPVariable_Check(o), who, name, " must be a tensor");
    return &THPVariable_Unpack(o);
}
const Tensor& tensor(PyObject* o, const char* who, const char* name) {
    const Tensor* t = maybe(o, who, name);
    require(t != nullptr, who, name, " must be a tensor");
    return *t;
}
bool truth(PyObject* o) {
    const int r = PyObject_IsTrue(o);
    if (r < 0) throw python_error();
    return r != 0;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
// a count of 32 bits
int32_t count(PyObject* o, const char* who, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    require(v >= 0 && v <= std::numeric_limits<int32_t>::max(), who, name, " ", v);
    return (int32_t)v;
}
int32_t size32(int64_t v, const char* who) {
    require(v <= std::numeric_limits<int32_t>::max(), who, "a size of ", v, " passes 32 bits");
    return (int32_t)v;
}

bool is16(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
int index_of(const Tensor& t) { return t.is_cuda() ? (int)t.get_device() : -1; }

// these operators serve; they carry no gradient, neither back nor forward (the
// tangent of a dual tensor)
void refuse_grad(const char* who, std::initializer_list<const Tensor*> ts) {
    const bool back = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const Tensor* t : ts) {
        if (t == nullptr || t->unsafeGetTensorImpl()->autograd_meta() == nullptr) continue;
        require(!back || !t->requires_grad(), who,
                "inputs that require a gradient are not supported (call it under torch.no_grad())");
        require(!forward || !t->_fw_grad(0).defined(), who,
                "inputs with a tangent (forward gradient) are not supported");
    }
}

// ---- shared memory --------------------------------------------------------------------------
// What a call writes must not be what it reads elsewhere, or another of its
// outputs: the kernels' blocks run in no order.  A tensor is a set of runs of
// `run` bytes at start + sum of index * step over its dimensions; two tensors
// share memory if some difference of their runs' addresses is smaller than a run.
struct Memory {
    struct Dim {
        int64_t n, step;                  // step > 0, in bytes; n > 1
    };
    int64_t start = 0, end = 0, run = 0;  // [start, end) holds every run
    Dim dim[8];
    int dims = 0;
    bool repeats = false;                 // a step of 0: several indices at one address
    explicit Memory(const Tensor& t) {
        const int64_t item = (int64_t)t.element_size();
        start = end = reinterpret_cast<int64_t>(t.data_ptr());
        if (t.numel() == 0) return;
        run = item;
        if (t.is_contiguous()) {
            run *= t.numel();
        } else {
            for (int64_t i = t.dim() - 1; i >= 0; --i) {
                const int64_t n = t.size(i), step = t.stride(i) * item;
                if (n == 1) continue;
                if (step == run) run *= n;                // a longer run
                else if (step == 0 || dims == 8) repeats = true;
                else dim[dims++] = {n, step};
            }
        }
        end += run;
        for (int i = 0; i < dims; ++i) end += (dim[i].n - 1) * dim[i].step;
    }
};
// Can base + sum x_i step_i, lo_i <= x_i <= hi_i, lie in (-below, above)?  Steps
// descend, so of ordinary layouts few x_i are left at each.  `tries` bounds the
// search; what is not found out counts as yes.
struct Step {
    int64_t step, lo, hi;
};
bool lands(int64_t base, const Step* d, int n, int64_t below, int64_t above, int& tries) {
    if (--tries < 0) return true;
    if (n == 0) return base > -below && base < above;
    int64_t least = 0, most = 0;          // of the smaller steps
    for (int i = 1; i < n; ++i) least += d[i].lo * d[i].step, most += d[i].hi * d[i].step;
    const auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
    const int64_t x0 = std::max(d->lo, floor_div(-below - base - most, d->step) + 1);
    const int64_t x1 = std::min(d->hi, floor_div(above - base - least - 1, d->step));
    for (int64_t x = x0; x <= x1; ++x)
        if (lands(base + x * d->step, d + 1, n - 1, below, above, tries)) return true;
    return false;
}
constexpr int kTries = 20000;
void by_step(Step* d, int n) {
    std::sort(d, d + n, [](const Step& a, const Step& b) { return a.step > b.step; });
}
bool share(const Memory& a, const Memory& b) {
    if (a.end <= b.start || b.end <= a.start || a.run == 0 || b.run == 0) return false;
    Step d[16];
    int n = 0;
    for (int i = 0; i < a.dims; ++i) d[n++] = {a.dim[i].step, 0, a.dim[i].n - 1};
    for (int i = 0; i < b.dims; ++i) {
        int j = 0;
        while (j < n && d[j].step != b.dim[i].step) ++j;
        if (j == n) d[n++] = {b.dim[i].step, 0, 0};
        d[j].lo -= b.dim[i].n - 1;
    }
    by_step(d, n);
    int tries = kTries;
    return lands(a.start - b.start, d, n, a.run, b.run, tries);
}
// two indices of one tensor at the same memory
bool folds(const Memory& a) {
    if (a.repeats) return true;
    Step d[8];
    for (int i = 0; i < a.dims; ++i) d[i] = {a.dim[i].step, 0, a.dim[i].n - 1};
    by_step(d, a.dims);
    int tries = kTries;
    for (int i = 0; i < a.dims; ++i) {    // the first step in which they differ
        d[i].lo = 1;
        for (int j = i + 1; j < a.dims; ++j) d[j].lo = -d[j].hi;
        if (lands(0, d + i, a.dims - i, a.run, a.run, tries)) return true;
    }
    return false;
}
// An output that is `in` itself is written in place; any other overlap is a race.
bool apart(const Tensor& out, const Tensor& in, bool same_is_fine) {
    if (same_is_fine && out.data_ptr() == in.data_ptr()) {
        bool same = true;
        for (int64_t i = 0; same && i < out.dim(); ++i) same = out.size(i) == 1 || out.stride(i) == in.stride(i);
        if (same) return true;
    }
    return !share(Memory(out), Memory(in));
}
bool apart_of(const Tensor& out, std::initializer_list<const Tensor*> ins) {
    const Memory o(out);
    for (const Tensor* t : ins)
        if (t != nullptr && share(o, Memory(*t))) return false;
    return true;
}

// 16-bit rows that the kernels can address: contiguous heads, 8-byte aligned,
// strides of a multiple of 4 elements.  (B, H, S, D) or (tokens, H, D).
struct Rows {
    Tensor t;
    int64_t st[3];         // strides of sequence, token, head
    uint16_t* ptr() const { return static_cast<uint16_t*>(t.data_ptr()); }
};
bool addressable(const Tensor& t, int64_t (&st)[3]) {
    const auto s = t.strides();
    if (s.size() == 3) {
        st[0] = 0, st[1] = s[0], st[2] = s[1];
    } else {
        st[0] = s[0], st[1] = s[2], st[2] = s[1];
    }
    return s.back() == 1 && ((st[0] | st[1] | st[2]) & 3) == 0 &&
           (reinterpret_cast<uintptr_t>(t.data_ptr()) & 7) == 0;
}
Rows rows16(const char* who, const char* name, const Tensor& t, at::ScalarType dt, int index) {
    require(t.scalar_type() == dt && index_of(t) == index, who, name, " is ", t.scalar_type(), " on ", t.device(),
            ", expected ", dt, " on cuda:", index);
    Rows r{t, {}};
    if (!addressable(r.t, r.st)) {               // copied where it is not so
        r.t = t.clone(at::MemoryFormat::Contiguous);
        addressable(r.t, r.st);
    }
    return r;
}
// A graph of autograd that saved a tensor written here must notice.
void written(const Tensor* t) {
    if (t != nullptr && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
// the same of a tensor that is written: it must be so already
Rows out16(const char* who, const char* name, const Tensor& t, const Tensor& like, int index) {
    require(t.sizes() == like.sizes() && t.scalar_type() == like.scalar_type() && index_of(t) == index, who, name,
            " is ", t.scalar_type(), " ", t.sizes(), " on ", t.device(), ", expected ", like.scalar_type(), " ",
            like.sizes(), " on cuda:", index);
    Rows r{t, {}};
    require(addressable(r.t, r.st) && !folds(Memory(t)), who, name, " must be 8-byte aligned rows that do not overlap, with strides of a multiple of 4 elements");
    return r;
}
// an output, straight from the CUDA allocator (through the dispatcher a call
// with two outputs took a microsecond longer)
Tensor make(at::IntArrayRef sizes, at::ScalarType dt, const at::Device& dev) {
    return at::detail::empty_cuda(sizes, dt, dev, std::nullopt);
}
// an output of t's shape: in t's order of memory if that is dense
Rows new16(const Tensor& like) {
    Rows r{like.is_non_overlapping_and_dense()
               ? at::detail::empty_strided_cuda(like.sizes(), like.strides(), like.scalar_type(), like.device())
               : make(like.sizes(), like.scalar_type(), like.device()),
           {}};
    addressable(r.t, r.st);
    return r;
}
const double* frequencies(const char* who, const Tensor& f, int index) {
    require(f.scalar_type() == at::kDouble && f.dim() == 1 && index_of(f) == index && f.is_contiguous(), who,
            "inv_freq must be a contiguous float64 vector on cuda:", index);
    return static_cast<const double*>(f.data_ptr());
}
void copy3(int64_t (&to)[3], const int64_t (&from)[3]) {
    for (int i = 0; i < 3; ++i) to[i] = from[i];
}

// ---- rotary(q, k, positions, inv_freq, interleaved, amplitude, inverse, q_out, k_out) ---------
PyObject* rotary(PyObject* const* args) {
    const char* who = "apply_rotary";
    const Tensor& q = tensor(args[0], who, "q");
    const Tensor* k = maybe(args[1], who, "k");
    const Tensor& pos = tensor(args[2], who, "positions");
    const Tensor& f = tensor(args[3], who, "inv_freq");
    const Tensor *q_out = maybe(args[7], who, "out"), *k_out = maybe(args[8], who, "out");
    const int index = index_of(q);
    const auto dt = q.scalar_type();
    require(index >= 0, who, "q must be a CUDA tensor");
    require(is16(dt), who, "q is ", dt, ", expected float16 or bfloat16");
    refuse_grad(who, {&q, k, &f, q_out, k_out});
    const int64_t nd = q.dim();
    require(nd == 3 || nd == 4, who, "q must be (B, H, S, D) or (T, H, D), got ", q.sizes());
    FkvRotaryShape sh = {};
    sh.B = nd == 4 ? size32(q.size(0), who) : 1;
    sh.S = size32(nd == 4 ? q.size(2) : q.size(0), who);
    sh.Hq = size32(q.size(1), who);
    sh.D = size32(q.size(-1), who);
    const auto ps = pos.sizes();
    const bool row = ps.size() == 1 && ps[0] == sh.S;
    const bool full = nd == 4 && ps.size() == 2 && ps[0] == sh.B && ps[1] == sh.S;
    require((row || full) && (pos.scalar_type() == at::kLong || pos.scalar_type() == at::kInt) && index_of(pos) == index,
            who, "positions ", ps, " ", pos.scalar_type(), " do not go with q ", q.sizes(),
            ": int32 or int64 (B, S), (S,) or, packed, (T,), on q's device");
    sh.pos_stride[0] = full ? pos.stride(0) : 0;
    sh.pos_stride[1] = full ? pos.stride(1) : pos.stride(0);
    sh.pos64 = pos.scalar_type() == at::kLong;
    const double* freq = frequencies(who, f, index);
    sh.rot = size32(2 * f.numel(), who);
    sh.bf16 = dt == at::kBFloat16;
    sh.interleaved = truth(args[4]);
    sh.amplitude = (float)number(args[5]);
    sh.inverse = truth(args[6]);
    if (k != nullptr) {
        require(k->dim() == nd && k->size(-1) == sh.D && k->size(0) == q.size(0) && (nd == 3 || k->size(2) == sh.S), who,
                "k ", k->sizes(), " does not go with q ", q.sizes());
        sh.Hk = size32(k->size(1), who);
    }
    require((q_out == nullptr) == (k_out == nullptr) || k == nullptr, who, "out must match (q, k)");
    require(k != nullptr || k_out == nullptr, who, "out must match (q, k)");
    const c10::cuda::OptionalCUDAGuard guard(q.device());
    const Rows qi = rows16(who, "q", q, dt, index);
    const Rows qo = q_out ? out16(who, "out", *q_out, q, index) : new16(qi.t);
    Rows ki{{}, {}}, ko{{}, {}};
    if (k != nullptr) {
        ki = rows16(who, "k", *k, dt, index);
        ko = k_out ? out16(who, "out", *k_out, *k, index) : new16(ki.t);
    }
    if (q_out || k_out)
        require((!q_out || (apart(qo.t, qi.t, true) && (!k || apart(qo.t, ki.t, false)))) &&
                    (!k_out || (apart(ko.t, ki.t, true) && apart(ko.t, qi.t, false))) &&
                    (!k || apart(qo.t, ko.t, false)) && (!q_out || apart_of(qo.t, {&pos, &f})) &&
                    (!k_out || apart_of(ko.t, {&pos, &f})),
                who, "out overlaps an input that it is not");
    copy3(sh.q_stride, qi.st);
    copy3(sh.q_out_stride, qo.st);
    copy3(sh.k_stride, ki.st);
    copy3(sh.k_out_stride, ko.st);
    check(p_rotary(&sh, qi.ptr(), k ? ki.ptr() : nullptr, pos.data_ptr(), freq, qo.ptr(), k ? ko.ptr() : nullptr,
                   c10::cuda::getCurrentCUDAStream(index).stream()),
          "fkv_rotary");
    written(q_out);
    written(k_out);
    if (k == nullptr) return THPVariable_Wrap(qo.t);
    PyObject* r = PyTuple_New(2);
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(qo.t));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(ko.t));
    return r;
}

// ---- the pages: k_pages, v_pages, table, lens, k_scale, v_scale, status -------------------------
struct Pages {
    FkvPagedCache c = {};
    const Tensor *k, *v, *k_scale, *v_scale, *table, *lens, *status;
    int index;
};
Pages pages(const char* who, PyObject* const* args, at::ScalarType dt) {
    Pages p;
    const Tensor &k = tensor(args[0], who, "k_pages"), &v = tensor(args[1], who, "v_pages");
    const Tensor &table = tensor(args[2], who, "table"), &lens = tensor(args[3], who, "lens");
    const Tensor *ks = maybe(args[4], who, "k_scale"), *vs = maybe(args[5], who, "v_scale");
    const Tensor* status = maybe(args[6], who, "status");
    refuse_grad(who, {&k, &v, ks, vs});
    p.k = &k;
    p.v = &v;
    p.k_scale = ks;
    p.v_scale = vs;
    p.table = &table;
    p.lens = &lens;
    p.status = status;
    const int index = p.index = index_of(k);
    const auto kind = k.scalar_type();
    require(index >= 0, who, "pages must be CUDA tensors");
    require(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == kind && index_of(v) == index &&
                k.is_contiguous() && v.is_contiguous(),
            who, "k_pages and v_pages must be contiguous (P, Hk, page, D) of one type and device");
    require(is16(dt), who, dt, " beside the pages, expected float16 or bfloat16");
    const auto sz = k.sizes();
    FkvPagedCache& c = p.c;
    c.k_pages = k.data_ptr();
    c.v_pages = v.data_ptr();
    c.fp8 = kind == at::kFloat8_e4m3fn;
    if (c.fp8) {
        for (const Tensor* s : {ks, vs})
            require(s != nullptr && s->scalar_type() == at::kFloat && index_of(*s) == index &&
                        s->sizes() == sz.slice(0, 3) && s->is_contiguous(),
                    who, "float8 pages need contiguous float32 k_scale and v_scale (P, Hk, page)");
        c.k_scale = static_cast<float*>(ks->data_ptr());
        c.v_scale = static_cast<float*>(vs->data_ptr());
    } else {
        require(kind == dt, who, "pages of ", kind, " beside ", dt, ", expected the same type or float8_e4m3fn pages");
        require(ks == nullptr && vs == nullptr, who, "scales go with float8 pages only");
    }
    require(table.dim() == 2 && table.scalar_type() == at::kInt && index_of(table) == index &&
                lens.scalar_type() == at::kInt && index_of(lens) == index && lens.dim() == 1 &&
                lens.size(0) == table.size(0) && lens.is_contiguous(),
            who, "table must be int32 (B, W) and lens contiguous int32 (B,) on cuda:", index);
    c.B = size32(table.size(0), who);
    c.width = size32(table.size(1), who);
    const int64_t stride = c.B > 1 ? table.stride(0) : c.width;
    require((c.width <= 1 || table.stride(1) == 1) && stride >= c.width, who,
            "a row of table must be contiguous, and rows must not overlap");
    c.table_stride = size32(stride, who);
    c.table = static_cast<const int32_t*>(table.data_ptr());
    c.lens = static_cast<const int32_t*>(lens.data_ptr());
    if (status != nullptr) {
        require(status->scalar_type() == at::kInt && index_of(*status) == index && status->numel() == 1, who,
                "status must be one int32 on cuda:", index);
        c.status = static_cast<int32_t*>(status->data_ptr());
    }
    c.n_pages = size32(sz[0], who);
    c.Hk = size32(sz[1], who);
    c.page = size32(sz[2], who);
    c.D = size32(sz[3], who);
    c.bf16 = dt == at::kBFloat16;
    return p;
}

// ---- paged_append(pages..., k, v, cu_new, q, inv_freq, interleaved, amplitude, q_out) ----------
PyObject* append(PyObject* const* args) {
    const char* who = "paged_append";
    const Tensor &k = tensor(args[7], who, "k"), &v = tensor(args[8], who, "v");
    const Tensor *cu = maybe(args[9], who, "cu_new"), *q = maybe(args[10], who, "q");
    const Tensor *f = maybe(args[11], who, "inv_freq"), *q_out = maybe(args[14], who, "q_out");
    refuse_grad(who, {&k, &v, q, f, q_out});
    const auto dt = k.scalar_type();
    const Pages p = pages(who, args, dt);
    const int64_t nd = k.dim();
    require(v.sizes() == k.sizes() && (nd == 3 || (nd == 4 && cu == nullptr)) && k.size(1) == p.c.Hk &&
                k.size(-1) == p.c.D,
            who, "k ", k.sizes(), " and v ", v.sizes(), " must be (tokens, ", p.c.Hk, ", ", p.c.D, "), or (B, ", p.c.Hk,
            ", n, ", p.c.D, ") without cu_new");
    FkvPagedNew n = {};
    int64_t T = k.size(0);
    if (cu != nullptr) {
        require(cu->scalar_type() == at::kInt && index_of(*cu) == p.index && cu->dim() == 1 &&
                    cu->size(0) == (int64_t)p.c.B + 1 && cu->is_contiguous(),
                who, "cu_new must be contiguous int32 (B + 1,) on cuda:", p.index);
        n.cu_new = static_cast<const int32_t*>(cu->data_ptr());
    } else {
        require(T == p.c.B, who, "k holds ", T, " sequences, the table ", p.c.B);
        n.n_uniform = nd == 4 ? size32(k.size(2), who) : 1;
        T *= n.n_uniform;
    }
    n.T = size32(T, who);
    if (f != nullptr) {
        n.inv_freq = frequencies(who, *f, p.index);
        n.rot = size32(2 * f->numel(), who);
        n.interleaved = truth(args[12]);
        n.amplitude = (float)number(args[13]);
    }
    const Memory into[4] = {Memory(*p.k), Memory(*p.v), Memory(p.c.fp8 ? *p.k_scale : *p.k),
                            Memory(p.c.fp8 ? *p.v_scale : *p.v)};
    const int parts = p.c.fp8 ? 4 : 2;
    for (int i = 1; i < parts; ++i)
        for (int j = 0; j < i; ++j)
            require(!share(into[i], into[j]), who,
                    "k_pages and v_pages (and their scales) must be different tensors that share no memory");
    require(q == nullptr || f != nullptr, who, "q is only rotated; pass inv_freq with it");
    require(q != nullptr || q_out == nullptr, who, "q_out without q");
    const c10::cuda::OptionalCUDAGuard guard(p.k->device());
    const Rows kr = rows16(who, "k", k, dt, p.index), vr = rows16(who, "v", v, dt, p.index);
    Rows qi{{}, {}}, qo{{}, {}};
    if (q != nullptr) {
        bool fits = q->dim() == nd && q->size(0) == k.size(0);
        for (int64_t i = 2; fits && i < nd; ++i) fits = q->size(i) == k.size(i);
        require(fits, who, "q ", q->sizes(), " does not go with k ", k.sizes());
        n.Hq = size32(q->size(1), who);
        qi = rows16(who, "q", *q, dt, p.index);
        qo = q_out ? out16(who, "q_out", *q_out, *q, p.index) : new16(qi.t);
        if (q_out)
            require(apart(qo.t, qi.t, true) && apart(qo.t, kr.t, false) && apart(qo.t, vr.t, false) &&
                        apart_of(qo.t, {p.k, p.v, p.k_scale, p.v_scale, p.table, p.lens, p.status, cu, f}),
                    who, "q_out overlaps an input that it is not");
        n.q = qi.ptr();
        n.q_out = qo.ptr();
    }
    for (const Rows* r : std::initializer_list<const Rows*>{&kr, &vr, &qi}) {
        if (!r->t.defined()) continue;
        const Memory m(r->t);
        for (int i = 0; i < parts; ++i) require(!share(m, into[i]), who, "k, v or q overlaps the pages or their scales");
    }
    n.k = kr.ptr();
    n.v = vr.ptr();
    copy3(n.k_stride, kr.st);
    copy3(n.v_stride, vr.st);
    copy3(n.q_stride, qi.st);
    copy3(n.q_out_stride, qo.st);
    if (cu == nullptr && nd == 3)                // one token per sequence: its row is the sequence's
        for (int64_t* s : {n.k_stride, n.v_stride, n.q_stride, n.q_out_stride}) {
            s[0] = s[1];
            s[1] = 0;
        }
    check(p_append(&p.c, &n, c10::cuda::getCurrentCUDAStream(p.index).stream()), "fkv_paged_append");
    for (const Tensor* t : {p.k, p.v, p.k_scale, p.v_scale, q_out}) written(t);
    if (q == nullptr) Py_RETURN_NONE;
    return THPVariable_Wrap(qo.t);
}

// ---- paged_read(pages..., max_len, dtype) ----------------------------------------------------------
PyObject* read(PyObject* const* args) {
    const char* who = "paged_read";
    const Tensor& kp = tensor(args[0], who, "k_pages");
    const int32_t max_len = count(args[7], who, "max_len");
    at::ScalarType dt = kp.scalar_type() == at::kFloat8_e4m3fn ? at::kHalf : kp.scalar_type();
    if (args[8] != Py_None) {
        require(THPDtype_Check(args[8]), who, "dtype must be a torch.dtype");
        dt = reinterpret_cast<THPDtype*>(args[8])->scalar_type;
    }
    const Pages p = pages(who, args, dt);
    const c10::cuda::OptionalCUDAGuard guard(kp.device());
    const int64_t shape[4] = {p.c.B, p.c.Hk, max_len, p.c.D};
    const Tensor k = make(shape, dt, kp.device()), v = make(shape, dt, kp.device());
    check(p_read(&p.c, max_len, static_cast<uint16_t*>(k.data_ptr()), static_cast<uint16_t*>(v.data_ptr()),
                 c10::cuda::getCurrentCUDAStream(p.index).stream()),
          "fkv_paged_read");
    PyObject* r = PyTuple_New(2);
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(k));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(v));
    return r;
}

// ---- paged_attend(pages..., q, scale, window, return_lse, out) -----------------------------------
PyObject* attend(PyObject* const* args) {
    const char* who = "paged_attend";
    const Tensor& q0 = tensor(args[7], who, "q");
    const Tensor* out0 = maybe(args[11], who, "out");
    refuse_grad(who, {&q0, out0});
    const auto dt = q0.scalar_type();
    const Pages p = pages(who, args, dt);
    const int64_t nd = q0.dim();
    require((nd == 3 || (nd == 4 && q0.size(2) == 1)) && q0.size(0) == p.c.B && q0.size(-1) == p.c.D &&
                q0.size(1) >= 1 && p.c.Hk > 0 && q0.size(1) % p.c.Hk == 0 && index_of(q0) == p.index,
            who, "q ", q0.sizes(), " must be (B, Hq, D) or (B, Hq, 1, D) on cuda:", p.index, " with B ", p.c.B, ", D ",
            p.c.D, " and Hq a multiple of ", p.c.Hk);
    const int32_t Hq = size32(q0.size(1), who);
    const double scale = args[8] == Py_None ? 1.0 / std::sqrt((double)p.c.D) : number(args[8]);
    const int32_t window = count(args[9], who, "window");
    const bool want_lse = truth(args[10]);
    const c10::cuda::OptionalCUDAGuard guard(p.k->device());
    Tensor q = q0.is_contiguous() ? q0 : q0.contiguous();
    if (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) q = q.clone();
    Tensor out;
    if (out0 == nullptr) {
        out = make(q.sizes(), dt, q.device());
    } else {
        out = *out0;
        require(out.sizes() == q.sizes() && out.scalar_type() == dt && index_of(out) == p.index && out.is_contiguous() &&
                    (reinterpret_cast<uintptr_t>(out.data_ptr()) & 15) == 0,
                who, "out must be a contiguous, 16-byte aligned tensor like q");
        require(apart_of(out, {&q, p.k, p.v, p.k_scale, p.v_scale, p.table, p.lens, p.status}), who,
                "out overlaps an input");
    }
    Tensor lse, ws;
    if (want_lse) lse = make({p.c.B, Hq}, at::kFloat, q.device());
    const size_t bytes = p_attend_ws(&p.c, Hq);
    if (bytes) ws = make({(int64_t)bytes}, at::kByte, q.device());
    check(p_attend(&p.c, Hq, (float)scale, window, static_cast<const uint16_t*>(q.data_ptr()),
                   static_cast<uint16_t*>(out.data_ptr()), want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr,
                   bytes ? ws.data_ptr() : nullptr, bytes, c10::cuda::getCurrentCUDAStream(p.index).stream()),
          "fkv_paged_attend");
    written(out0);
    if (!want_lse) return THPVariable_Wrap(out);
    PyObject* r = PyTuple_New(2);
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(out));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(lse));
    return r;
}

// share_memory(a, b): what the calls above refuse; b None: two indices of a
PyObject* share_memory(PyObject* const* args) {
    const char* who = "share_memory";
    const Tensor &a = tensor(args[0], who, "a"), *b = maybe(args[1], who, "b");
    return PyBool_FromLong(b ? share(Memory(a), Memory(*b)) : folds(Memory(a)));
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != N || p_error == nullptr) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, %d expected (or bind() not called)", n, N);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what.c_str());
    } catch (const Failed& e) {
        PyErr_SetString(native_error, e.what.c_str());
    }
    return nullptr;
    END_HANDLE_TH_ERRORS
}

// bind(error class, addresses of the six functions in the order below)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7) {
        PyErr_SetString(PyExc_TypeError, "bind: 7 arguments expected");
        return nullptr;
    }
    void* a[6];
    for (int i = 0; i < 6; ++i) {
        a[i] = PyLong_AsVoidPtr(args[i + 1]);
        if (a[i] == nullptr) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: NULL address");
            return nullptr;
        }
    }
    Py_INCREF(args[0]);
    Py_XDECREF(native_error);
    native_error = args[0];
    p_error = reinterpret_cast<decltype(p_error)>(a[0]);
    p_rotary = reinterpret_cast<decltype(p_rotary)>(a[1]);
    p_append = reinterpret_cast<decltype(p_append)>(a[2]);
    p_read = reinterpret_cast<decltype(p_read)>(a[3]);
    p_attend = reinterpret_cast<decltype(p_attend)>(a[4]);
    p_attend_ws = reinterpret_cast<decltype(p_attend_ws)>(a[5]);
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {
    {"bind", FAST(bind)},
    {"rotary", FAST((&entry<rotary, 9>))},
    {"paged_append", FAST((&entry<append, 15>))},
    {"paged_read", FAST((&entry<read, 9>))},
    {"paged_attend", FAST((&entry<attend, 12>))},
    {"share_memory", FAST((&entry<share_memory, 2>))},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "fkv_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// with what it was built against, which the loader compares
PyMODINIT_FUNC PyInit_fkv_ops() {
    PyObject* m = PyModule_Create(&module);
    const std::string made = c10::str("torch ", TORCH_VERSION_MAJOR, ".", TORCH_VERSION_MINOR, ".", TORCH_VERSION_PATCH,
                                      ", Python ", PY_MAJOR_VERSION, ".", PY_MINOR_VERSION);
    if (m != nullptr && PyModule_AddStringConstant(m, "built_for", made.c_str()) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
