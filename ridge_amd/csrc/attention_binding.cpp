// attention_binding.cpp -- the tensors' way to the C ABI in include/ridge_attention.h: the checks
// of arguments, the allocation of results and the current stream behind ridge_amd.attention.

#include "binding.hpp"

#include <torch/csrc/Dtype.h>

#include <cfloat>
#include <cmath>
#include <vector>

#include "ridge_attention.h"

namespace {

// A 3-D device tensor of tokens' heads, whose columns are contiguous. Strides in elements.
struct Heads {
    const at::Tensor* t = nullptr;
    int64_t tokens = 0, heads = 0, dim = 0, token = 0, head = 0;
    ridge_attention_heads_t ref() const { return {t ? t->data_ptr() : nullptr, token, head, (int32_t)heads}; }
};

// Whether rows of `bytes`, n1 of them s1 apart, n2 times s2 apart, share no byte with each other.
bool separate(int64_t bytes, int64_t n1, int64_t s1, int64_t n2, int64_t s2) {
    if (n1 <= 0 || n2 <= 0 || bytes <= 0) return true;
    if (n1 == 1) return n2 == 1 || s2 >= bytes;
    if (n2 == 1) return s1 >= bytes;
    if (s1 > s2) std::swap(n1, n2), std::swap(s1, s2);
    return s1 >= bytes && s2 >= (n1 - 1) * s1 + bytes;
}

Heads headsOf(const at::Tensor& t, const char* what, const at::Device* device = nullptr) {
    if (!t.is_cuda() || t.dim() != 3 || t.layout() != at::kStrided)
        refuse("%s must be a device tensor [tokens, heads, columns]", what);
    if (device && t.device() != *device)
        refuse("%s is on device %d, not on %d", what, (int)t.device().index(), (int)device->index());
    Heads h = {&t, t.size(0), t.size(1), t.size(2), t.stride(0), t.stride(1)};
    if (h.dim > 1 && t.stride(2) != 1) refuse("%s must have contiguous columns", what);
    if (h.heads > 65535) refuse("%s has %lld heads: 65535 at the most", what, (long long)h.heads);
    if (!separate(h.dim, h.tokens, h.token, h.heads, h.head)) refuse("the heads of %s overlap", what);
    if (h.tokens <= 1) h.token = h.heads * h.dim;
    if (h.heads <= 1) h.head = h.dim;
    return h;
}

// The heads as spans of bytes: one where they follow each other, else one for each of the fewer.
std::vector<Span> spansOf(const Heads& h, const char* what) {
    const int64_t E = h.t->element_size(), at = (int64_t)h.t->data_ptr(), dim = h.dim * E;
    if (h.tokens < 1 || h.heads < 1 || h.dim < 1) return {};
    if (h.head == h.dim) return {{what, at, h.tokens, h.heads * dim, h.token * E}};
    if (h.token == h.dim) return {{what, at, h.heads, h.tokens * dim, h.head * E}};
    std::vector<Span> spans;
    if (h.heads <= h.tokens) {
        for (int64_t i = 0; i < h.heads; ++i) spans.push_back({what, at + i * h.head * E, h.tokens, dim, h.token * E});
    } else {
        for (int64_t i = 0; i < h.tokens; ++i) spans.push_back({what, at + i * h.token * E, h.heads, dim, h.head * E});
    }
    return spans;
}

// The bytes from the first of the heads to their last.
Span hullOf(const Heads& h, const char* what) {
    const int64_t E = h.t->element_size();
    const bool none = h.tokens < 1 || h.heads < 1 || h.dim < 1;
    const int64_t bytes = none ? 0 : ((h.tokens - 1) * h.token + (h.heads - 1) * h.head + h.dim) * E;
    return {what, (int64_t)h.t->data_ptr(), 1, bytes, bytes};
}

void apart(const Heads& written, const char* what, const Heads& other, const char* otherWhat) {
    if (!meet(hullOf(written, what), hullOf(other, otherWhat))) return;
    const std::vector<Span> others = spansOf(other, otherWhat);
    for (const Span& w : spansOf(written, what))
        for (const Span& o : others) apart(w, o);
}

void apart(const Heads& written, const char* what, const Span& other) {
    for (const Span& w : spansOf(written, what)) apart(w, other);
}

bool same(const Heads& a, const Heads& b) {
    return a.t->data_ptr() == b.t->data_ptr() && a.token == b.token && a.head == b.head;
}

// Heads to write: the caller's, or new ones.
struct HeadsOut {
    at::Tensor made;
    Heads h;
    const char* what;
    PyObject* given;
    HeadsOut(PyObject* out, const char* what, int64_t tokens, int64_t heads, int64_t dim, at::ScalarType type,
             const at::Device& device)
        : what(what), given(out) {
        made = out == Py_None ? at::empty({tokens, heads, dim}, at::TensorOptions(device).dtype(type)) : tensor(out, what);
        h = headsOf(made, what, &device);
        noGradient(&made);
        if (h.tokens != tokens || h.heads != heads || h.dim != dim || made.scalar_type() != type)
            refuse("%s must be %lld x %lld x %lld of %s", what, (long long)tokens, (long long)heads, (long long)dim,
                   c10::toString(type));
    }
    HeadsOut(const HeadsOut&) = delete;
    void apartFrom(const Heads& other, const char* otherWhat) const {
        if (given != Py_None) apart(h, what, other, otherWhat);
    }
    void apartFrom(const Span& other) const {
        if (given != Py_None) apart(h, what, other);
    }
    void wrote() const {
        if (given != Py_None) written(made);
    }
    PyObject* result() const { return given != Py_None ? Py_NewRef(given) : THPVariable_Wrap(made); }
};

// Whether two nests of rows of `bytes`, alike but for where they begin, share a byte. `by`
// bytes lie between their beginnings; each level's stride passes all that is below it, so only
// the two multiples next to the distance can meet.
struct Level {
    int64_t count, stride;
};
bool nestsMeet(int64_t by, int64_t bytes, const Level* levels, int n) {
    if (n == 0) return by < bytes && -by < bytes;
    const auto [count, stride] = levels[0];
    if (count <= 1 || stride == 0) return nestsMeet(by, bytes, levels + 1, n - 1);
    const int64_t near = floorDivide(by, stride);
    for (int64_t i : {near, near + 1})
        if (i > -count && i < count && nestsMeet(by - i * stride, bytes, levels + 1, n - 1)) return true;
    return false;
}

// The cache's four tensors, checked.
struct Cache {
    at::Tensor k, kScale, v, vScale;
    ridge_attention_cache_t ref = {};
    int64_t bytes = 0, scaleBytes = 0;   // from the first to the last
    at::Device device() const { return k.device(); }
    Cache(PyObject* o, const at::Device* on) {
        if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) refuse("the cache must be (k, k_scale, v, v_scale)");
        k = tensor(PyTuple_GET_ITEM(o, 0), "the cache's k");
        kScale = tensor(PyTuple_GET_ITEM(o, 1), "the cache's k_scale");
        v = tensor(PyTuple_GET_ITEM(o, 2), "the cache's v");
        vScale = tensor(PyTuple_GET_ITEM(o, 3), "the cache's v_scale");
        if (!k.is_cuda() || k.dim() != 4 || k.layout() != at::kStrided || k.scalar_type() != at::kChar)
            refuse("the cache's k must be an int8 device tensor [pages, heads, page_size, columns]");
        if (on && device() != *on)
            refuse("the cache is on device %d, not on %d", (int)device().index(), (int)on->index());
        if (v.scalar_type() != at::kChar || v.device() != device() || v.layout() != at::kStrided || v.sizes() != k.sizes() ||
            v.strides() != k.strides())
            refuse("the cache's v must be like its k");
        const int64_t pages = k.size(0), heads = k.size(1), size = k.size(2), dim = k.size(3);
        if (dim < 1 || dim > RIDGE_ATTENTION_MAX_DIM || heads < 1 || heads > 65535 || pages < 1)
            refuse("a cache of %lld pages, %lld heads and %lld columns: 1 to 65535 heads and %d columns are wanted",
                   (long long)pages, (long long)heads, (long long)dim, (int)RIDGE_ATTENTION_MAX_DIM);
        if (size < 16 || size % 16) refuse("page_size must be a multiple of 16, not %lld", (long long)size);
        if (pages > RIDGE_ATTENTION_MAX_SLOTS / size) refuse("the cache holds 2^31 tokens or more");
        if (dim > 1 && k.stride(3) != 1) refuse("the cache must have contiguous columns");
        Level levels[3], scales[2];
        const int64_t row = to16(dim);
        for (int i = 0; i < 3; ++i) {
            levels[i].count = k.size(i);
            levels[i].stride = k.size(i) > 1 ? k.stride(i) : 0;
            if (levels[i].stride % 16) refuse("the cache's rows must start at multiples of 16 bytes (as those of empty_cache() do)");
            bytes += (levels[i].count - 1) * levels[i].stride;
        }
        if (levels[2].stride >= (int64_t)1 << 27) refuse("the rows of a page lie 2^27 bytes apart or more");
        ref.pageStride = levels[0].stride, ref.headStride = levels[1].stride, ref.tokenStride = levels[2].stride;
        for (const at::Tensor* s : {&kScale, &vScale}) {
            if (s->scalar_type() != at::kFloat || s->device() != device() || s->layout() != at::kStrided || s->dim() != 3 ||
                s->size(0) != pages || s->size(1) != heads || s->size(2) != size || s->stride(2) != 1 ||
                s->strides() != kScale.strides())
                refuse("the cache's scales must be float32 [pages, heads, page_size] with contiguous pages, alike, on its device");
            noGradient(s);
        }
        for (int i = 0; i < 2; ++i) {
            scales[i].count = kScale.size(i);
            scales[i].stride = kScale.size(i) > 1 ? kScale.stride(i) : 0;
            if (scales[i].stride % 4) refuse("the cache's scales must start at multiples of 16 bytes");
            scaleBytes += (scales[i].count - 1) * scales[i].stride * 4;
        }
        ref.scalePage = scales[0].stride, ref.scaleHead = scales[1].stride;
        bytes += row, scaleBytes += size * 4;
        for (const at::Tensor* t : {&k, &v, &kScale, &vScale})
            if ((uintptr_t)t->data_ptr() % 16) refuse("the cache must start at multiples of 16 bytes");
        for (const at::Tensor* t : {&k, &v})
            if (t->storage_offset() + bytes > (int64_t)t->storage().nbytes())
                refuse("the cache's last row ends its memory inside 16 bytes (make it with empty_cache())");
        const auto outer = [](const Level& a, const Level& b) { return a.stride > b.stride; };
        std::sort(levels, levels + 3, outer);
        std::sort(scales, scales + 2, outer);
        nested(levels, 3, dim);
        for (Level& level : scales) level.stride *= 4;
        nested(scales, 2, size * 4);
        if (nestsMeet((int64_t)v.data_ptr() - (int64_t)k.data_ptr(), dim, levels, 3) ||
            nestsMeet((int64_t)vScale.data_ptr() - (int64_t)kScale.data_ptr(), size * 4, scales, 2))
            refuse("the cache's k and v overlap");
        ref.k = (int8_t*)k.data_ptr(), ref.v = (int8_t*)v.data_ptr();
        ref.kScale = (float*)kScale.data_ptr(), ref.vScale = (float*)vScale.data_ptr();
        ref.pages = pages, ref.pageSize = (int32_t)size, ref.heads = (int32_t)heads, ref.dim = (int32_t)dim;
    }
    static int64_t to16(int64_t cols) { return (cols + 15) / 16 * 16; }
    // Whether each level of rows, from the outermost, passes the ones below it.
    static void nested(const Level* levels, int n, int64_t bytes) {
        for (int i = n - 1; i >= 0; --i) {
            if (levels[i].count <= 1) continue;
            if (levels[i].stride < bytes) refuse("the cache's rows overlap");
            bytes += (levels[i].count - 1) * levels[i].stride;
        }
    }
    // A cache lies between its first and its last byte; nothing else of a call is put there.
    void apartFrom(const Span& other) const {
        const std::pair<const at::Tensor*, int64_t> parts[] = {{&k, bytes}, {&v, bytes}, {&kScale, scaleBytes}, {&vScale, scaleBytes}};
        for (const auto& [t, size] : parts) apart({"the cache", (int64_t)t->data_ptr(), 1, size, size}, other);
    }
    void wrote() const {
        for (const at::Tensor* t : {&k, &kScale, &v, &vScale}) written(*t);
    }
};

// Whole numbers of 32 bits on the operands' device.
void integers(const at::Tensor& t, int64_t dims, const at::Device& device, const char* what) {
    if (t.scalar_type() != at::kInt || t.layout() != at::kStrided || t.dim() != dims || t.device() != device)
        refuse("%s must be %lld-D int32 on the operands' device", what, (long long)dims);
}

void slotsOf(const at::Tensor& t, int64_t n, const at::Device& device) {
    integers(t, 1, device, "slots");
    if (t.size(0) != n || (n > 1 && t.stride(0) != 1)) refuse("slots must be %lld contiguous numbers", (long long)n);
}

// A matrix of whole numbers with contiguous rows: their stride.
int64_t strideOf(const at::Tensor& t, const char* what) {
    if (t.size(1) > 1 && t.stride(1) != 1) refuse("%s must have contiguous rows", what);
    return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

Span hullOf(const at::Tensor& t, const char* what) {
    int64_t elements = 1;
    for (int64_t i = 0; i < t.dim(); ++i) {
        if (t.size(i) == 0) return {what, (int64_t)t.data_ptr(), 0, 0, 0};
        elements += (t.size(i) - 1) * t.stride(i);
    }
    const int64_t bytes = elements * t.element_size();
    return {what, (int64_t)t.data_ptr(), 1, bytes, bytes};
}

double number(PyObject* o) {
    const double value = PyFloat_AsDouble(o);
    if (value == -1.0 && PyErr_Occurred()) throw python_error();
    return value;
}

int64_t whole(PyObject* o) {
    const long long value = PyLong_AsLongLong(o);
    if (value == -1 && PyErr_Occurred()) throw python_error();
    return value;
}

bool truth(PyObject* o) {
    const int value = PyObject_IsTrue(o);
    if (value < 0) throw python_error();
    return value;
}

// (q, k, table, positions, q_weight, k_weight, eps, sections, interleaved, q_out, k_out, stream)
PyObject* normRopeImpl(PyObject* const* args, Py_ssize_t n) {
    if (n != 12) refuse("12 arguments are wanted");
    const Heads q = headsOf(tensor(args[0], "q"), "q");
    const at::Device device = q.t->device();
    const Heads k = headsOf(tensor(args[1], "k"), "k", &device);
    const at::Tensor &table = tensor(args[2], "table"), &positions = tensor(args[3], "positions");
    const at::Tensor *qWeight = optionalTensor(args[4], "q_weight"), *kWeight = optionalTensor(args[5], "k_weight");
    const double eps = number(args[6]);
    const int code = typeOf(*q.t, "q");
    if (k.t->scalar_type() != q.t->scalar_type()) refuse("k must be %s, as q is", c10::toString(q.t->scalar_type()));
    if (k.tokens != q.tokens || k.dim != q.dim) refuse("q and k must be heads of the same tokens, of one width");
    if (q.dim < 1 || q.dim > RIDGE_ATTENTION_MAX_DIM)
        refuse("heads must have 1 to %d columns, not %lld", (int)RIDGE_ATTENTION_MAX_DIM, (long long)q.dim);
    if (table.scalar_type() != at::kFloat || table.layout() != at::kStrided || table.dim() != 2 || table.device() != device ||
        (table.size(1) > 1 && table.stride(1) != 1))
        refuse("table must be a float32 matrix with contiguous rows on the operands' device (rope_table() makes it)");
    ridge_attention_rotation_t r = {};
    r.pairs = (int32_t)std::min<int64_t>(table.size(1) / 2, INT32_MAX);
    if (table.size(1) % 2 || r.pairs < 1 || 2 * (int64_t)r.pairs > q.dim || table.size(0) < 1 || table.size(0) > INT32_MAX)
        refuse("a table of %lld x %lld does not turn heads of %lld columns", (long long)table.size(0),
               (long long)table.size(1), (long long)q.dim);
    r.table = (const float*)table.data_ptr(), r.tableRows = table.size(0);
    r.tableStride = table.size(0) > 1 ? table.stride(0) : table.size(1);
    if (r.tableStride < table.size(1)) refuse("the rows of table overlap");
    if (r.tableStride >= ((int64_t)1 << 30) / r.tableRows) refuse("table spans 4 GiB or more");
    integers(positions, positions.dim() == 1 ? 1 : 2, device, "positions");
    const int64_t axes = positions.dim() == 1 ? 1 : positions.size(1);
    if (positions.size(0) != q.tokens || axes < 1 || axes > RIDGE_ATTENTION_MAX_AXES)
        refuse("positions must be [tokens] or [tokens, axes] of at most %d axes", (int)RIDGE_ATTENTION_MAX_AXES);
    r.positions = (const int32_t*)positions.data_ptr(), r.axes = (int32_t)axes, r.interleaved = truth(args[8]);
    r.positionStride = positions.dim() == 2 ? strideOf(positions, "positions") : q.tokens > 1 ? positions.stride(0) : 1;
    if (args[7] == Py_None) {
        if (axes > 1) refuse("positions on %lld axes want sections", (long long)axes);
        r.sections[0] = r.pairs;
    } else {
        PyObject* const list = PySequence_Fast(args[7], "sections must be whole numbers");
        if (!list) throw python_error();
        const Py_ssize_t count = PySequence_Fast_GET_SIZE(list);
        int64_t parts[RIDGE_ATTENTION_MAX_AXES] = {}, sum = 0;
        bool fits = count == axes;
        for (Py_ssize_t i = 0; fits && i < count; ++i) {
            parts[i] = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(list, i));
            if (parts[i] == -1 && PyErr_Occurred()) {
                Py_DECREF(list);
                throw python_error();
            }
            fits = parts[i] >= 0 && parts[i] <= r.pairs;
            sum += parts[i];
        }
        Py_DECREF(list);
        if (!fits || sum != r.pairs)
            refuse("sections must be %lld numbers of pairs that add up to %d", (long long)axes, (int)r.pairs);
        for (int i = 0; i < (int)axes; ++i) r.sections[i] = (int32_t)parts[i];
    }
    if (!(eps > 0 && (float)eps > 0 && std::isfinite((float)eps))) refuse("eps must be positive, not %g", eps);
    const at::Tensor* const weights[] = {qWeight, kWeight};
    int weightCode = code;
    for (const at::Tensor* w : weights) {
        if (!w) continue;
        weightCode = typeOf(*w, "a weight");
        if (weightCode != code && weightCode != kF32) refuse("weights must be of q's type or float32");
        if (qWeight && qWeight->scalar_type() != w->scalar_type()) refuse("both weights must be of one type");
        vector(*w, q.dim, w->scalar_type(), device, w == qWeight ? "q_weight" : "k_weight");
        noGradient(w);
    }
    noGradient(q.t);
    noGradient(k.t);
    noGradient(&table);
    const On on(device, args[11]);
    const HeadsOut qOut(args[9], "q_out", q.tokens, q.heads, q.dim, q.t->scalar_type(), device);
    const HeadsOut kOut(args[10], "k_out", k.tokens, k.heads, k.dim, k.t->scalar_type(), device);
    for (const HeadsOut* out : {&qOut, &kOut}) {
        if (out->given == Py_None) continue;
        const Heads &from = out == &qOut ? q : k, &other = out == &qOut ? k : q;
        if (!same(out->h, from)) out->apartFrom(from, out == &qOut ? "q" : "k");
        out->apartFrom(other, out == &qOut ? "k" : "q");
        out->apartFrom(hullOf(table, "table"));
        out->apartFrom(hullOf(positions, "positions"));
        for (const at::Tensor* w : weights)
            if (w) out->apartFrom(span(*w, "a weight"));
    }
    if (qOut.given != Py_None && kOut.given != Py_None) qOut.apartFrom(kOut.h, "k_out");
    const ridge_attention_heads_t refs[] = {q.ref(), k.ref(), qOut.h.ref(), kOut.h.ref()};
    enqueued("ridge_attention_norm_rope",
             ridge_attention_norm_rope(&refs[0], &refs[1], code, qWeight ? qWeight->data_ptr() : nullptr,
                                       kWeight ? kWeight->data_ptr() : nullptr, weightCode, (float)eps, &r, &refs[2], &refs[3],
                                       q.tokens, (int32_t)q.dim, on.stream()));
    qOut.wrote();
    kOut.wrote();
    return Py_BuildValue("(NN)", qOut.result(), kOut.result());
}

// (cache, slots, k, v, stream)
PyObject* writeImpl(PyObject* const* args, Py_ssize_t n) {
    if (n != 5) refuse("5 arguments are wanted");
    const Cache cache(args[0], nullptr);
    const at::Device device = cache.device();
    const Heads k = headsOf(tensor(args[2], "k"), "k", &device), v = headsOf(tensor(args[3], "v"), "v", &device);
    const int code = typeOf(*k.t, "k");
    if (v.t->scalar_type() != k.t->scalar_type()) refuse("v must be %s, as k is", c10::toString(k.t->scalar_type()));
    for (const Heads* h : {&k, &v}) {
        if (h->tokens != k.tokens || h->heads != cache.ref.heads || h->dim != cache.ref.dim)
            refuse("k and v must be heads of the same tokens, %d of %d columns", (int)cache.ref.heads, (int)cache.ref.dim);
        noGradient(h->t);
        cache.apartFrom(hullOf(*h, h == &k ? "k" : "v"));
    }
    const at::Tensor& slots = tensor(args[1], "slots");
    slotsOf(slots, k.tokens, device);
    cache.apartFrom(hullOf(slots, "slots"));
    const On on(device, args[4]);
    const ridge_attention_heads_t refs[] = {k.ref(), v.ref()};
    enqueued("ridge_attention_write", ridge_attention_write(&cache.ref, (const int32_t*)slots.data_ptr(), &refs[0], &refs[1],
                                                            code, k.tokens, on.stream()));
    if (k.tokens) cache.wrote();
    return Py_NewRef(args[0]);
}

// (cache, slots, dtype, out, stream)
PyObject* readImpl(PyObject* const* args, Py_ssize_t n) {
    if (n != 5) refuse("5 arguments are wanted");
    const Cache cache(args[0], nullptr);
    const at::Device device = cache.device();
    const at::Tensor& slots = tensor(args[1], "slots");
    integers(slots, 1, device, "slots");
    const int64_t tokens = slots.size(0);
    slotsOf(slots, tokens, device);
    if (args[2] != Py_None && !THPDtype_Check(args[2])) refuse("dtype must be a torch.dtype");
    PyObject* outs[] = {Py_None, Py_None};
    if (args[3] != Py_None) {
        if (!PyTuple_Check(args[3]) || PyTuple_GET_SIZE(args[3]) != 2) refuse("out must be (k, v)");
        outs[0] = PyTuple_GET_ITEM(args[3], 0), outs[1] = PyTuple_GET_ITEM(args[3], 1);
    }
    at::ScalarType type = at::kHalf;
    if (args[2] != Py_None) {
        type = ((THPDtype*)args[2])->scalar_type;
    } else if (outs[0] != Py_None) {
        type = tensor(outs[0], "out's k").scalar_type();
    }
    const int code = typeCode(type);
    if (code < 0) refuse("the result must be float16, bfloat16 or float32, not %s", c10::toString(type));
    const On on(device, args[4]);
    const HeadsOut k(outs[0], "out's k", tokens, cache.ref.heads, cache.ref.dim, type, device);
    const HeadsOut v(outs[1], "out's v", tokens, cache.ref.heads, cache.ref.dim, type, device);
    for (const HeadsOut* out : {&k, &v}) {
        if (out->given == Py_None) continue;
        cache.apartFrom(hullOf(out->h, out->what));
        out->apartFrom(hullOf(slots, "slots"));
    }
    if (k.given != Py_None) k.apartFrom(v.h, "out's v");
    const ridge_attention_heads_t refs[] = {k.h.ref(), v.h.ref()};
    enqueued("ridge_attention_read", ridge_attention_read(&cache.ref, (const int32_t*)slots.data_ptr(), &refs[0], &refs[1],
                                                          code, tokens, on.stream()));
    k.wrote();
    v.wrote();
    return Py_BuildValue("(NN)", k.result(), v.result());
}

// (q, cache, pages, lengths, scale, window, lse_out, out, stream)
PyObject* attendImpl(PyObject* const* args, Py_ssize_t n) {
    if (n != 9) refuse("9 arguments are wanted");
    const Heads q = headsOf(tensor(args[0], "q"), "q");
    const at::Device device = q.t->device();
    const Cache cache(args[1], &device);
    const int code = typeOf(*q.t, "q");
    const at::Tensor &pages = tensor(args[2], "pages"), &lengths = tensor(args[3], "lengths");
    noGradient(q.t);
    if (q.dim != cache.ref.dim || q.heads % cache.ref.heads)
        refuse("%lld heads of %lld columns do not share a cache of %d of %d", (long long)q.heads, (long long)q.dim,
               (int)cache.ref.heads, (int)cache.ref.dim);
    integers(pages, 2, device, "pages");
    integers(lengths, 1, device, "lengths");
    const int64_t pagesStride = strideOf(pages, "pages");
    if (pages.size(0) != q.tokens || lengths.size(0) != q.tokens || (q.tokens > 1 && lengths.stride(0) != 1))
        refuse("pages and lengths must have a row and a contiguous number for each of q's %lld", (long long)q.tokens);
    const double scale = args[4] == Py_None ? 1.0 / std::sqrt((double)q.dim) : number(args[4]);
    if (!(std::fabs((float)scale) <= FLT_MAX / 2)) refuse("scale must be finite, not %g", scale);
    if (code == kF16 && std::fabs((float)scale) > 0x1p118f) refuse("scale must be 2^118 at the most for float16, not %g", scale);
    const int64_t window = args[5] == Py_None ? 0 : whole(args[5]);
    if (window < 0 || (window == 0 && args[5] != Py_None)) refuse("window must be positive, not %lld", (long long)window);
    const On on(device, args[8]);
    const HeadsOut out(args[7], "out", q.tokens, q.heads, q.dim, q.t->scalar_type(), device);
    const at::Tensor* lse = optionalTensor(args[6], "lse_out");
    if (lse) {
        if (lse->scalar_type() != at::kFloat || lse->layout() != at::kStrided || lse->dim() != 2 || lse->device() != device ||
            lse->size(0) != q.tokens || lse->size(1) != q.heads || !lse->is_contiguous())
            refuse("lse_out must be %lld x %lld contiguous float32 on the operands' device", (long long)q.tokens,
                   (long long)q.heads);
        noGradient(lse);
        apart(q, "lse_out", hullOf(*lse, "q"));
    }
    std::vector<Span> others = {hullOf(pages, "pages"), hullOf(lengths, "lengths")};
    if (out.given != Py_None) {
        out.apartFrom(q, "q");
        cache.apartFrom(hullOf(out.h, "out"));
        for (const Span& other : others) out.apartFrom(other);
        if (lse) out.apartFrom(hullOf(*lse, "lse_out"));
    }
    if (lse) {
        cache.apartFrom(hullOf(*lse, "lse_out"));
        for (const Span& other : others) apart(hullOf(*lse, "lse_out"), other);
    }
    const int64_t bytes = ridge_attention_workspace(q.tokens, (int32_t)q.heads, cache.ref.heads, cache.ref.dim, pages.size(1),
                                                    cache.ref.pageSize);
    if (bytes < 0) refuse("%lld pages of %d tokens for each sequence are too many", (long long)pages.size(1),
                          (int)cache.ref.pageSize);
    // A new one for each call: no two calls share it, and a graph's calls have it in the graph's memory.
    at::Tensor workspace;
    if (bytes) workspace = at::empty({bytes}, at::TensorOptions(device).dtype(at::kByte));
    const ridge_attention_heads_t refs[] = {q.ref(), out.h.ref()};
    enqueued("ridge_attention_attend",
             ridge_attention_attend(&refs[0], &cache.ref, (const int32_t*)pages.data_ptr(), pagesStride, pages.size(1),
                                    (const int32_t*)lengths.data_ptr(), (float)scale, window, &refs[1],
                                    lse ? (float*)lse->data_ptr() : nullptr, code, q.tokens,
                                    bytes ? workspace.data_ptr() : nullptr, bytes, on.stream()));
    out.wrote();
    if (lse) written(*lse);
    return out.result();
}

PyMethodDef gMethods[] = {
    {"norm_rope", (PyCFunction)(void (*)(void))entry<normRopeImpl>, METH_FASTCALL,
     "(q, k, table, positions, q_weight, k_weight, eps, sections, interleaved, q_out, k_out, stream)"},
    {"write_cache", (PyCFunction)(void (*)(void))entry<writeImpl>, METH_FASTCALL, "(cache, slots, k, v, stream)"},
    {"read_cache", (PyCFunction)(void (*)(void))entry<readImpl>, METH_FASTCALL, "(cache, slots, dtype, out, stream)"},
    {"attend", (PyCFunction)(void (*)(void))entry<attendImpl>, METH_FASTCALL,
     "(q, cache, pages, lengths, scale, window, lse_out, out, stream)"},
    {"set_error", setError, METH_O, "the class that refusals are raised as"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef gModule = {PyModuleDef_HEAD_INIT, "_ridge_attention", "The calls behind ridge_amd.attention.", -1, gMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ridge_attention(void) { return PyModule_Create(&gModule); }
