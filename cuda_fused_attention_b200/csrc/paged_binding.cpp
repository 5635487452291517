// CPython binding of the paged-cache operators (include/fa_sm100_paged.h) for torch tensors.
//
// A decode step makes a few calls of some microseconds each per layer, so what the host does per
// call counts: the argument checks, allocations and the packing of structs and strides are here and
// not in Python (which took 8 to 12 us a call). cuda_fused_attention_b200/paged.py documents the
// functions and is what users import; it hands every argument on as it is. The kernels are reached
// through the C ABI of the library that paged.py names to load().
//
// Every function returns its result, or an int: the status of a call that the C ABI refused.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "fa_sm100_paged.h"

namespace {

struct Library {
    decltype(&fa_sm100_paged_plan) plan = nullptr;
    decltype(&fa_sm100_paged_schedule_bytes) schedule_bytes = nullptr;
    decltype(&fa_sm100_paged_workspace_bytes) workspace_bytes = nullptr;
    decltype(&fa_sm100_paged_fwd) fwd = nullptr;
    decltype(&fa_sm100_rotary) rotary = nullptr;
    decltype(&fa_sm100_rotary_append) append = nullptr;
} lib;

// A refused argument: the Python exception of type `kind` is set where this is caught.
struct Refused {
    PyObject* kind;
    std::string text;
};

[[noreturn]] void bad_value(const std::string& text) { throw Refused{PyExc_ValueError, text}; }
[[noreturn]] void bad_type(const std::string& text) { throw Refused{PyExc_TypeError, text}; }

std::string shown(at::IntArrayRef values)
{
    std::string text = "[";
    for (size_t i = 0; i < values.size(); ++i) text += (i ? ", " : "") + std::to_string(values[i]);
    return text + "]";
}

const at::Tensor& tensor(PyObject* object, const char* name)
{
    if (!THPVariable_Check(object)) bad_type(std::string(name) + " must be a torch.Tensor");
    return THPVariable_Unpack(object);
}

long long integer(PyObject* object, const char* name)
{
    PyObject* index = PyNumber_Index(object);
    if (index == nullptr) {
        PyErr_Clear();
        bad_type(std::string(name) + " must be an integer");
    }
    int overflow = 0;
    const long long value = PyLong_AsLongLongAndOverflow(index, &overflow);
    Py_DECREF(index);
    if (overflow) bad_value(std::string(name) + " is out of range");
    return value;
}

bool truth(PyObject* object, const char* name)
{
    const int value = PyObject_IsTrue(object);
    if (value < 0) {
        PyErr_Clear();
        bad_type(std::string(name) + " must be a truth value");
    }
    return value != 0;
}

void need_int32(const at::Tensor& t, const char* name, int64_t dims)
{
    if (t.scalar_type() != at::kInt) bad_type(std::string(name) + " must be int32, got " + std::string(t.dtype().name()));
    if (t.dim() != dims)
        bad_value(std::string(name) + " must have " + std::to_string(dims) + " dimension(s), got " + std::to_string(t.dim()));
}

void need_vector(const at::Tensor& t, const char* name, int64_t size = -1)
{
    need_int32(t, name, 1);
    if (!t.is_contiguous()) bad_value(std::string(name) + " must be contiguous");
    if (size >= 0 && t.numel() != size)
        bad_value(std::string(name) + " must have " + std::to_string(size) + " elements, got " + std::to_string(t.numel()));
}

// A bf16 tensor of this shape whose last dimension is contiguous and whose rows begin on 16-byte boundaries;
// writes the strides of the other dimensions. The stride of a dimension of one element is never used.
void need_rows(const at::Tensor& t, const char* name, at::IntArrayRef shape, long long* strides)
{
    if (t.scalar_type() != at::kBFloat16) bad_type(std::string(name) + " must be bfloat16, got " + std::string(t.dtype().name()));
    if (t.sizes() != shape) bad_value(std::string(name) + " must be " + shown(shape) + ", got " + shown(t.sizes()));
    const size_t last = shape.size() - 1;
    if (t.stride(static_cast<int64_t>(last)) != 1) bad_value(std::string(name) + " must be contiguous in its last dimension");
    for (size_t i = 0; i < last; ++i) {
        strides[i] = shape[i] > 1 ? t.stride(static_cast<int64_t>(i)) : shape[last];
        if (strides[i] % 8) bad_value(std::string(name) + " has rows off 16-byte boundaries (strides " + shown(t.strides()) + ")");
    }
    if (reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16) bad_value(std::string(name) + " must start on a 16-byte boundary");
}

// An output (or cache): no two of its elements may share memory.
void need_distinct(const at::Tensor& t, const char* name)
{
    if (t.is_contiguous() || t.numel() == 0) return;
    std::vector<std::pair<int64_t, int64_t>> spans;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) spans.emplace_back(t.stride(i), t.size(i));
    std::sort(spans.begin(), spans.end());
    int64_t reach = 1;
    for (const auto& [stride, size] : spans) {
        if (stride < reach) bad_value(std::string(name) + " has elements that share memory (strides " + shown(t.strides()) + ")");
        reach = stride * (size - 1) + reach;
    }
}

// Whether two tensors of one shape and strides, each without shared elements, have an element in common: whether
// `apart`, the distance of their first elements, is a sum of differences of indexes times strides. Taken from
// the widest stride down, only the two multiples around what is left can be part of one.
bool meet(const std::vector<std::pair<int64_t, int64_t>>& widest_first, size_t at, int64_t apart)
{
    if (at == widest_first.size()) return apart == 0;
    const auto [stride, size] = widest_first[at];
    const int64_t low = apart >= 0 ? apart / stride : -((-apart + stride - 1) / stride);
    for (int64_t index : {low, low + 1})
        if (index > -size && index < size && meet(widest_first, at + 1, apart - index * stride)) return true;
    return false;
}

// Two caches that are written in one call.
void need_apart(const at::Tensor& a, const at::Tensor& b, const char* names)
{
    if (a.numel() == 0 || a.strides() != b.strides()) return;
    const auto *pa = static_cast<const char*>(a.const_data_ptr()), *pb = static_cast<const char*>(b.const_data_ptr());
    const int64_t distance = (pb - pa) / static_cast<int64_t>(a.element_size());
    int64_t reach = 0;
    for (int64_t i = 0; i < a.dim(); ++i) reach += (a.size(i) - 1) * a.stride(i);
    if (distance > reach || distance < -reach) return;
    std::vector<std::pair<int64_t, int64_t>> spans;
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) > 1) spans.emplace_back(a.stride(i), a.size(i));
    std::sort(spans.rbegin(), spans.rend());
    if (meet(spans, 0, distance)) bad_value(std::string(names) + " must not share memory");
}

// All tensors on one CUDA device; its index.
class OneDevice {
public:
    void add(const at::Tensor& t, const char* name)
    {
        if (!t.is_cuda()) bad_type(std::string(name) + " must be a CUDA tensor");
        const int index = t.get_device();
        if (index_ < 0) index_ = index;
        else if (index != index_)
            bad_value(std::string(name) + " is on cuda:" + std::to_string(index) + ", other arguments on cuda:" + std::to_string(index_));
    }
    int index() const { return index_; }

private:
    int index_ = -1;
};

// Makes the tensors' device current for a call and finds its stream (None: the device's current one). What is
// allocated meanwhile belongs to that stream, so that its memory is not handed to another one while the call
// still uses it.
class Launching {
public:
    Launching(int index, PyObject* stream) : device_(static_cast<c10::DeviceIndex>(index))
    {
        const auto current = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index));
        handle_ = current.stream();
        if (stream == Py_None) return;
        long long value = 0;
        if (PyLong_Check(stream)) {
            value = integer(stream, "stream");
        } else {
            PyObject* attribute = PyObject_GetAttrString(stream, "cuda_stream");
            if (attribute == nullptr) {
                PyErr_Clear();
                bad_type("stream must be None, an integer or a torch.cuda.Stream");
            }
            try {
                value = integer(attribute, "stream");
            } catch (...) {
                Py_DECREF(attribute);
                throw;
            }
            Py_DECREF(attribute);
        }
        handle_ = reinterpret_cast<cudaStream_t>(value);
        if (handle_ == current.stream()) return;
        other_.emplace(handle_ == nullptr
                           ? c10::cuda::getDefaultCUDAStream(static_cast<c10::DeviceIndex>(index))
                           : c10::cuda::getStreamFromExternal(handle_, static_cast<c10::DeviceIndex>(index)));
    }
    void* handle() const { return handle_; }

private:
    c10::cuda::CUDAGuard device_;
    std::optional<c10::cuda::CUDAStreamGuard> other_;
    cudaStream_t handle_ = nullptr;
};

at::Tensor allocate(at::IntArrayRef shape, at::ScalarType type, int index)
{
    return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(index)), std::nullopt);
}

// Frequencies and sections: (rotary_dim, axes), the sections written to `counts`.
constexpr int kMaxAxes = 4;
int need_frequencies(const at::Tensor& inv_freq, int64_t dim, PyObject* sections, int (&counts)[kMaxAxes], int& axes)
{
    if (inv_freq.scalar_type() != at::kFloat) bad_type("inv_freq must be float32, got " + std::string(inv_freq.dtype().name()));
    if (inv_freq.dim() != 1 || !inv_freq.is_contiguous()) bad_value("inv_freq must be a contiguous vector");
    const int64_t pairs = inv_freq.numel();
    if (pairs == 0 || pairs % 8 || 2 * pairs > dim)
        bad_value("inv_freq must have a multiple of 8 and at most " + std::to_string(dim / 2) + " elements, got " + std::to_string(pairs));
    axes = 1;
    counts[0] = static_cast<int>(pairs);
    if (sections != Py_None) {
        PyObject* list = PySequence_Fast(sections, "");
        if (list == nullptr) {
            PyErr_Clear();
            bad_type("sections must be a sequence of counts");
        }
        const Py_ssize_t size = PySequence_Fast_GET_SIZE(list);
        long long sum = 0;
        bool good = size >= 1 && size <= kMaxAxes;
        for (Py_ssize_t i = 0; good && i < size; ++i) {
            long long count = -1;
            try {
                count = integer(PySequence_Fast_GET_ITEM(list, i), "sections");
            } catch (...) {
                Py_DECREF(list);
                throw;
            }
            good = count >= 0 && count <= pairs;
            counts[i] = static_cast<int>(count);
            sum += count;
        }
        Py_DECREF(list);
        if (!good || sum != pairs) bad_value("sections must be 1 to 4 counts that add up to " + std::to_string(pairs));
        axes = static_cast<int>(size);
    }
    return static_cast<int>(2 * pairs);
}

void need_head_dim(int64_t dim)
{
    if (dim != 64 && dim != 128) bad_value("head_dim must be 64 or 128, got " + std::to_string(dim));
}

void need_arguments(Py_ssize_t given, Py_ssize_t expected)
{
    if (given != expected) bad_type("expected " + std::to_string(expected) + " arguments, got " + std::to_string(given));
}

constexpr long long kIntMax = 2147483647LL;

// No element of a vector may be one of the table's, whose rows of `width` begin `stride` apart.
void need_outside_table(const at::Tensor& vector, const char* name, const at::Tensor& table, int64_t width, int64_t stride)
{
    const int64_t rows = table.size(0), size = vector.numel();
    if (rows == 0 || width == 0 || size == 0) return;
    const auto bytes = static_cast<const char*>(vector.const_data_ptr()) - static_cast<const char*>(table.const_data_ptr());
    const int64_t from = bytes >= 0 ? bytes / 4 : -((3 - bytes) / 4);       // element of the table at which it begins
    if (from + size <= 0) return;
    const int64_t row = from < width ? 0 : (from - width) / stride + 1;     // the first row that ends behind it
    if (row < rows && row * stride < from + size) bad_value(std::string(name) + " must not share memory with block_table");
}

// plan(cached_lens, new_lens, block_table, free_pages, total_tokens, (heads, kv_heads, head_dim, page_size),
//      num_pages, free_cursor, causal, max_new, buffer or None, stream)
//   -> (buffer, FaPagedPlan as bytes, workspace bytes, device index)
// buffer: [schedule][query_start][kv_lens][positions][slots][free_cursor], int32; an earlier plan's is written again.
PyObject* plan(PyObject* const* args, Py_ssize_t count)
{
    need_arguments(count, 12);
    const at::Tensor &cached = tensor(args[0], "cached_lens"), &fresh = tensor(args[1], "new_lens"),
                     &table = tensor(args[2], "block_table"), &free_pages = tensor(args[3], "free_pages");
    need_vector(cached, "cached_lens");
    const int64_t seqs = cached.numel();
    need_vector(fresh, "new_lens", seqs);
    need_vector(free_pages, "free_pages");
    need_int32(table, "block_table", 2);
    if (table.size(0) != seqs) bad_value("block_table must have " + std::to_string(seqs) + " rows, got " + std::to_string(table.size(0)));
    const int64_t width = table.size(1);
    if (width > 1 && table.stride(1) != 1) bad_value("block_table must be contiguous in its last dimension");
    const int64_t stride = seqs > 1 ? table.stride(0) : width;
    if (stride < width) bad_value("block_table has rows that share memory");
    const bool has_cursor = args[7] != Py_None;
    if (has_cursor) need_vector(tensor(args[7], "free_cursor"), "free_cursor", 1);
    const long long total = integer(args[4], "total_tokens"), num_pages = integer(args[6], "num_pages");
    const long long max_new = args[9] == Py_None ? total : integer(args[9], "max_new");
    if (total < 0 || num_pages < 0 || max_new < 0) bad_value("total_tokens, num_pages and max_new must not be negative");
    if (total > kIntMax / 2 || max_new > kIntMax) bad_value("total_tokens must be below 2^30");
    if (!PyTuple_Check(args[5]) || PyTuple_GET_SIZE(args[5]) != 4) bad_type("shape must be a PagedShape");
    long long shape[4];
    for (int i = 0; i < 4; ++i) shape[i] = integer(PyTuple_GET_ITEM(args[5], i), "shape");
    if (num_pages > kIntMax || num_pages * shape[3] > kIntMax || stride > kIntMax || seqs > kIntMax / 4)
        bad_value("a cache must hold fewer than 2^31 tokens");
    if (width * shape[3] > (1LL << 30)) bad_value("a table row must hold at most 2^30 tokens");
    // The kernel's blocks extend the table while others still read the inputs.
    need_outside_table(cached, "cached_lens", table, width, stride);
    need_outside_table(fresh, "new_lens", table, width, stride);
    need_outside_table(free_pages, "free_pages", table, width, stride);
    if (has_cursor) need_outside_table(tensor(args[7], "free_cursor"), "free_cursor", table, width, stride);
    OneDevice device;
    device.add(cached, "cached_lens");
    device.add(fresh, "new_lens");
    device.add(table, "block_table");
    device.add(free_pages, "free_pages");
    if (has_cursor) device.add(tensor(args[7], "free_cursor"), "free_cursor");

    const bool causal = truth(args[8], "causal");
    const int64_t schedule_words = static_cast<int64_t>(lib.schedule_bytes(static_cast<int>(seqs)) / 4);
    const int64_t words = schedule_words + 2 * seqs + 2 + 2 * total;
    const Launching launching(device.index(), args[11]);
    at::Tensor buffer;
    if (args[10] == Py_None) {
        buffer = allocate({words}, at::kInt, device.index());
    } else {
        buffer = tensor(args[10], "plan");
        if (buffer.numel() != words || buffer.scalar_type() != at::kInt || !buffer.is_cuda() || buffer.get_device() != device.index())
            bad_value("plan was made for other sizes or another device");
        // The kernel's blocks write the plan while others still read the inputs.
        auto apart = [&](const at::Tensor& t, const char* name) {
            const auto* from = static_cast<const char*>(buffer.const_data_ptr());
            const auto* at = static_cast<const char*>(t.const_data_ptr());
            if (t.numel() > 0 && at < from + 4 * words && at + t.nbytes() > from)
                bad_value(std::string(name) + " must not be a part of the plan that is written");
        };
        apart(cached, "cached_lens");
        apart(fresh, "new_lens");
        apart(free_pages, "free_pages");
        apart(table, "block_table");
        if (has_cursor) apart(tensor(args[7], "free_cursor"), "free_cursor");
    }
    FaPagedPlan c{};
    c.num_seqs = static_cast<int>(seqs);
    c.total_tokens = static_cast<int>(total);
    c.max_new = static_cast<int>(max_new);
    c.num_pages = static_cast<int>(num_pages);
    c.table_width = static_cast<int>(width);
    c.table_stride = static_cast<int>(stride);
    c.heads = static_cast<int>(shape[0]);
    c.kv_heads = static_cast<int>(shape[1]);
    c.head_dim = static_cast<int>(shape[2]);
    c.page_size = static_cast<int>(shape[3]);
    c.causal = causal ? 1 : 0;
    int* at = buffer.data_ptr<int>();
    c.schedule = reinterpret_cast<long long*>(at);
    c.query_start = at += schedule_words;
    c.kv_lens = at += seqs + 1;
    c.positions = at += seqs;
    c.slots = at += total;
    c.free_cursor = at += total;
    c.block_table = table.data_ptr<int>();
    const int status = lib.plan(&c, cached.data_ptr<int>(), fresh.data_ptr<int>(), free_pages.data_ptr<int>(),
                                static_cast<int>(free_pages.numel()), has_cursor ? tensor(args[7], "free_cursor").data_ptr<int>() : nullptr,
                                launching.handle());
    if (status != FA_STATUS_OK) return PyLong_FromLong(status);
    return Py_BuildValue("(Ny#ni)", THPVariable_Wrap(buffer), reinterpret_cast<const char*>(&c), static_cast<Py_ssize_t>(sizeof(c)),
                         static_cast<Py_ssize_t>(lib.workspace_bytes(&c)), device.index());
}

// split(buffer, num_seqs, total_tokens) -> the plan's views (query_start, kv_lens, positions, slots, free_cursor)
PyObject* split(PyObject* const* args, Py_ssize_t count)
{
    need_arguments(count, 3);
    const at::Tensor& buffer = tensor(args[0], "buffer");
    const int64_t seqs = integer(args[1], "num_seqs"), total = integer(args[2], "total_tokens");
    const int64_t sizes[5] = {seqs + 1, seqs, total, total, 1};
    int64_t from = buffer.numel() - (2 * seqs + 2 + 2 * total);
    PyObject* views = PyTuple_New(5);
    if (views == nullptr) return nullptr;
    for (int i = 0; i < 5; ++i) {
        // A tensor on the same storage (int32 views need no autograd record, which is most of narrow's cost).
        at::Tensor view = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), buffer.dtype());
        view.unsafeGetTensorImpl()->set_storage_offset(buffer.storage_offset() + from);
        view.unsafeGetTensorImpl()->set_sizes_contiguous({sizes[i]});
        PyTuple_SET_ITEM(views, i, THPVariable_Wrap(view));
        from += sizes[i];
    }
    return views;
}

// embed(x, positions, inv_freq, sections, interleaved, inverse, out or None, stream) -> out
PyObject* embed(PyObject* const* args, Py_ssize_t count)
{
    need_arguments(count, 8);
    const at::Tensor &x = tensor(args[0], "x"), &positions = tensor(args[1], "positions"), &inv_freq = tensor(args[2], "inv_freq");
    if (x.dim() != 4) bad_value("x must be [batch, heads, seq_len, head_dim]");
    const at::IntArrayRef shape = x.sizes();
    need_head_dim(shape[3]);
    long long x_strides[3], out_strides[3];
    need_rows(x, "x", shape, x_strides);
    int sections[kMaxAxes], axes;
    const int rotary_dim = need_frequencies(inv_freq, shape[3], args[3], sections, axes);
    const int64_t dims = positions.dim();
    need_int32(positions, "positions", dims >= 1 && dims <= 3 ? dims : 2);
    const bool batched = dims == 3;
    if (positions.size(dims - 1) != shape[2] || (dims == 1 ? axes != 1 : positions.size(0) != axes) ||
        (batched && positions.size(1) != shape[0]))
        bad_value("positions must be " + shown({axes, shape[2]}) + " or " + shown({axes, shape[0], shape[2]}) + ", got " +
                  shown(positions.sizes()));
    if (shape[2] > 1 && positions.stride(dims - 1) != 1) bad_value("positions must be contiguous in their last dimension");
    const long long position_strides[2] = {dims > 1 ? positions.stride(0) : 0, batched ? positions.stride(1) : 0};
    for (int64_t n : shape)
        if (n > kIntMax) bad_value("x is too large");
    OneDevice device;
    device.add(x, "x");
    device.add(positions, "positions");
    device.add(inv_freq, "inv_freq");
    const bool interleaved = truth(args[4], "interleaved"), inverse = truth(args[5], "inverse");
    if (args[6] != Py_None) {
        const at::Tensor& out = tensor(args[6], "out");
        need_rows(out, "out", shape, out_strides);
        need_distinct(out, "out");
        device.add(out, "out");
    }
    const Launching launching(device.index(), args[7]);
    at::Tensor out = args[6] != Py_None ? tensor(args[6], "out") : allocate(shape, at::kBFloat16, device.index());
    if (args[6] == Py_None)
        for (int i = 0; i < 3; ++i) out_strides[i] = out.stride(i);
    const int status = lib.rotary(x.const_data_ptr(), x_strides, out.mutable_data_ptr(), out_strides, static_cast<int>(shape[0]),
                                  static_cast<int>(shape[1]), static_cast<int>(shape[2]), static_cast<int>(shape[3]),
                                  positions.data_ptr<int>(), position_strides, inv_freq.data_ptr<float>(), rotary_dim, sections,
                                  axes, interleaved ? 1 : 0, inverse ? 1 : 0, launching.handle());
    return status != FA_STATUS_OK ? PyLong_FromLong(status) : THPVariable_Wrap(out);
}

// append(q, k, v, k_cache, v_cache, positions, slots, inv_freq, sections, interleaved, out or None, stream) -> out
PyObject* append(PyObject* const* args, Py_ssize_t count)
{
    need_arguments(count, 12);
    const at::Tensor &q = tensor(args[0], "q"), &k = tensor(args[1], "k"), &v = tensor(args[2], "v"),
                     &k_cache = tensor(args[3], "k_cache"), &v_cache = tensor(args[4], "v_cache"),
                     &positions = tensor(args[5], "positions"), &slots = tensor(args[6], "slots"), &inv_freq = tensor(args[7], "inv_freq");
    if (k_cache.dim() != 4) bad_value("k_cache must be [num_pages, kv_heads, page_size, head_dim]");
    const at::IntArrayRef cache = k_cache.sizes();
    if (q.dim() != 3) bad_value("q must be [tokens, heads, head_dim]");
    const int64_t pages = cache[0], kv_heads = cache[1], page_size = cache[2], dim = cache[3], tokens = q.size(0), heads = q.size(1);
    need_head_dim(dim);
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
        bad_value("page_size must be 16, 32, 64, 128 or 256, got " + std::to_string(page_size));
    if (pages > kIntMax || pages * page_size > kIntMax) bad_value("a cache must hold fewer than 2^31 tokens");
    if (tokens > kIntMax || heads > kIntMax || kv_heads > kIntMax) bad_value("q is too large");
    long long s[14];        // q, out, k, v (token, head); k_cache, v_cache (page, head, row)
    need_rows(q, "q", {tokens, heads, dim}, s);
    need_rows(k, "k", {tokens, kv_heads, dim}, s + 4);
    need_rows(v, "v", {tokens, kv_heads, dim}, s + 6);
    need_rows(k_cache, "k_cache", cache, s + 8);
    need_rows(v_cache, "v_cache", cache, s + 11);
    need_distinct(k_cache, "k_cache");
    need_distinct(v_cache, "v_cache");
    need_apart(k_cache, v_cache, "k_cache and v_cache");
    int sections[kMaxAxes], axes;
    const int rotary_dim = need_frequencies(inv_freq, dim, args[8], sections, axes);
    const int64_t dims = positions.dim();
    need_int32(positions, "positions", dims == 1 ? 1 : 2);
    if (positions.size(dims - 1) != tokens || (dims == 1 ? axes != 1 : positions.size(0) != axes))
        bad_value("positions must be " + shown({axes, tokens}) + ", got " + shown(positions.sizes()));
    if (tokens > 1 && positions.stride(dims - 1) != 1) bad_value("positions must be contiguous in their last dimension");
    need_vector(slots, "slots", tokens);
    OneDevice device;
    device.add(q, "q");
    device.add(k, "k");
    device.add(v, "v");
    device.add(k_cache, "k_cache");
    device.add(v_cache, "v_cache");
    device.add(positions, "positions");
    device.add(slots, "slots");
    device.add(inv_freq, "inv_freq");
    const bool interleaved = truth(args[9], "interleaved");
    if (args[10] != Py_None) {
        const at::Tensor& out = tensor(args[10], "out");
        need_rows(out, "out", {tokens, heads, dim}, s + 2);
        need_distinct(out, "out");
        device.add(out, "out");
    }
    const Launching launching(device.index(), args[11]);
    at::Tensor out = args[10] != Py_None ? tensor(args[10], "out") : allocate({tokens, heads, dim}, at::kBFloat16, device.index());
    if (args[10] == Py_None) {
        s[2] = out.stride(0);
        s[3] = out.stride(1);
    }
    const int status = lib.append(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), out.mutable_data_ptr(),
                                  k_cache.mutable_data_ptr(), v_cache.mutable_data_ptr(), s, static_cast<int>(tokens),
                                  static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(dim), static_cast<int>(page_size),
                                  static_cast<int>(pages), positions.data_ptr<int>(), dims == 2 ? positions.stride(0) : 0,
                                  slots.data_ptr<int>(), inv_freq.data_ptr<float>(), rotary_dim, sections, axes,
                                  interleaved ? 1 : 0, launching.handle());
    return status != FA_STATUS_OK ? PyLong_FromLong(status) : THPVariable_Wrap(out);
}

// attention(q, k_cache, v_cache, FaPagedPlan as bytes, workspace bytes, device index, out or None, stream) -> out
PyObject* attention(PyObject* const* args, Py_ssize_t count)
{
    need_arguments(count, 8);
    const at::Tensor &q = tensor(args[0], "q"), &k_cache = tensor(args[1], "k_cache"), &v_cache = tensor(args[2], "v_cache");
    if (!PyBytes_Check(args[3]) || PyBytes_GET_SIZE(args[3]) != static_cast<Py_ssize_t>(sizeof(FaPagedPlan)))
        bad_type("plan must be a PagedPlan");
    const auto* c = reinterpret_cast<const FaPagedPlan*>(PyBytes_AS_STRING(args[3]));
    const long long workspace_bytes = integer(args[4], "workspace");
    const int64_t rows[3] = {c->total_tokens, c->heads, c->head_dim};
    const int64_t cache[4] = {c->num_pages, c->kv_heads, c->page_size, c->head_dim};
    long long s[10];        // q, out (token, head); k_cache, v_cache (page, head, row)
    need_rows(q, "q", rows, s);
    need_rows(k_cache, "k_cache", cache, s + 4);
    need_rows(v_cache, "v_cache", cache, s + 7);
    OneDevice device;
    device.add(q, "q");
    device.add(k_cache, "k_cache");
    device.add(v_cache, "v_cache");
    const int plan_device = static_cast<int>(integer(args[5], "plan"));
    if (device.index() != plan_device)
        bad_value("plan is on cuda:" + std::to_string(plan_device) + ", other arguments on cuda:" + std::to_string(device.index()));
    if (args[6] != Py_None) {
        const at::Tensor& out = tensor(args[6], "out");
        need_rows(out, "out", rows, s + 2);
        need_distinct(out, "out");
        device.add(out, "out");
    }
    const Launching launching(device.index(), args[7]);
    at::Tensor out = args[6] != Py_None ? tensor(args[6], "out") : allocate(rows, at::kBFloat16, device.index());
    if (args[6] == Py_None) {
        s[2] = out.stride(0);
        s[3] = out.stride(1);
    }
    at::Tensor workspace;
    if (workspace_bytes > 0) workspace = allocate({workspace_bytes}, at::kByte, device.index());
    const int status = lib.fwd(c, q.const_data_ptr(), k_cache.const_data_ptr(), v_cache.const_data_ptr(), out.mutable_data_ptr(), s,
                               workspace_bytes > 0 ? workspace.mutable_data_ptr() : nullptr, static_cast<size_t>(workspace_bytes),
                               launching.handle());
    return status != FA_STATUS_OK ? PyLong_FromLong(status) : THPVariable_Wrap(out);
}

// load(path): the library whose C ABI the calls go to.
PyObject* load(PyObject* const* args, Py_ssize_t count)
{
    need_arguments(count, 1);
    const char* path = PyUnicode_AsUTF8(args[0]);
    if (path == nullptr) return nullptr;
    void* handle = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    if (handle == nullptr) throw Refused{PyExc_RuntimeError, std::string("cannot load ") + path + ": " + dlerror()};
    Library found;
    auto find = [&](auto& function, const char* name) {
        function = reinterpret_cast<std::remove_reference_t<decltype(function)>>(dlsym(handle, name));
        if (function == nullptr) throw Refused{PyExc_RuntimeError, std::string(path) + " has no " + name};
    };
    find(found.plan, "fa_sm100_paged_plan");
    find(found.schedule_bytes, "fa_sm100_paged_schedule_bytes");
    find(found.workspace_bytes, "fa_sm100_paged_workspace_bytes");
    find(found.fwd, "fa_sm100_paged_fwd");
    find(found.rotary, "fa_sm100_rotary");
    find(found.append, "fa_sm100_rotary_append");
    lib = found;
    Py_RETURN_NONE;
}

template <PyObject* (*Function)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    try {
        return Function(args, count);
    } catch (const Refused& refused) {
        PyErr_SetString(refused.kind, refused.text.c_str());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

template <PyObject* (*Function)(PyObject* const*, Py_ssize_t)>
PyCFunction entry()
{
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<Function>));
}

PyMethodDef methods[] = {
    {"load", entry<load>(), METH_FASTCALL, nullptr},
    {"plan", entry<plan>(), METH_FASTCALL, nullptr},
    {"split", entry<split>(), METH_FASTCALL, nullptr},
    {"embed", entry<embed>(), METH_FASTCALL, nullptr},
    {"append", entry<append>(), METH_FASTCALL, nullptr},
    {"attention", entry<attention>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", "Binding of the paged-cache operators; see paged.py.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged(void) { return PyModule_Create(&module); }
