// bfft_torch.cpp -- torch tensors to the C ABI for the position and cache calls.
//
// A decoding step makes these calls one token at a time, and a call's device work
// is a few microseconds: the checks of a dozen tensors' types, shapes and strides
// in Python cost more than that (rotate_positions 12.5 us a call, append_rotated
// and read_cache 38 us together).  This module makes the same checks on the
// tensors themselves, allocates the outputs and the workspace from torch's caching
// allocator, and calls the entry points of libbfft.so on the current stream.  It
// holds no CUDA code and is not linked against libbfft.so: bfft/cache.py hands it
// the entry points' addresses.
//
// Checks come before any launch; they raise TypeError for a non-tensor or a wrong
// dtype and ValueError for shapes, strides and devices.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <string>

#include "../../include/bfft.h"

namespace {

using at::Tensor;

struct Entries {
    decltype(&bfft_rotate_positions) rotate;
    decltype(&bfft_cache_append) append;
    decltype(&bfft_cache_read) read;
    decltype(&bfft_cache_attention_workspace) workspace;
    decltype(&bfft_cache_attention) attention;
    decltype(&bfft_last_error) last_error;
    decltype(&bfft_rotate_axes) rotate_axes;
    decltype(&bfft_cache_append_axes) append_axes;
    decltype(&bfft_cache_attention_span_workspace) span_workspace;
    decltype(&bfft_cache_attention_span) span_attention;
} g_entry{};

std::string text(const char* s) { return s; }
std::string text(const std::string& s) { return s; }
std::string text(int64_t v) { return std::to_string(v); }

std::string shape_of(const Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

template <typename... A>
[[noreturn]] void value_error(const A&... parts) {
    PyErr_SetString(PyExc_ValueError, (text(parts) + ...).c_str());
    throw python_error();
}
template <typename... A>
[[noreturn]] void type_error(const A&... parts) {
    PyErr_SetString(PyExc_TypeError, (text(parts) + ...).c_str());
    throw python_error();
}

// The library's status as the exception types of bfft/_lib.py.  Also reached from
// autograd's threads, which do not hold the interpreter's lock.
void check(bfft_status st, const char* what) {
    if (st == BFFT_OK) return;
    const std::string msg = std::string(what) + ": " + g_entry.last_error();
    TORCH_CHECK_VALUE(st != BFFT_ERR_VALUE && st != BFFT_ERR_SHAPE && st != BFFT_ERR_UNSUPPORTED && st != BFFT_ERR_WORKSPACE,
                      msg);
    throw std::runtime_error(msg);
}

const Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) type_error(name, " must be a torch.Tensor, got ", Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
void on_device(const Tensor& t, const char* name, int64_t device) {
    if (!t.is_cuda()) value_error(name, " must be on a CUDA device, got ", t.device().str());
    if (device >= 0 && t.get_device() != device)
        value_error(name, " is on ", t.device().str(), ", not on device ", device, " with the other tensors");
}
void of_type(const Tensor& t, const char* name, at::ScalarType want) {
    if (t.scalar_type() != want)
        type_error(name, " must be ", at::toString(want), ", got ", at::toString(t.scalar_type()));
}

int64_t type_id(const Tensor& t, const char* name, bool halves = false) {
    switch (t.scalar_type()) {
        case at::kFloat:
            if (!halves) return BFFT_F32;
            break;
        case at::kHalf:
            return BFFT_F16;
        case at::kBFloat16:
            return BFFT_BF16;
        default:
            break;
    }
    type_error(name, " must be ", halves ? "" : "float32, ", "float16 or bfloat16, got ", at::toString(t.scalar_type()));
}

// The entry points write through pointers: an operator that saved the tensor for its
// gradient learns of that by the version (tensors of inference mode have none).
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// No call has a forward-mode gradient.
void no_tangent(const Tensor& t, const char* name) {
    if (t._fw_grad(0).defined()) value_error("this call has no forward-mode gradient for ", name);
}

// Only x of a rotation has a gradient: a result that silently lacks one is refused.
void constant(const Tensor& t, const char* name) {
    no_tangent(t, name);
    if (t.requires_grad() && at::GradMode::is_enabled())
        value_error("this call has no gradient for ", name, ": detach it or call under torch.no_grad()");
}

// The dimensions of more than one element, widest stride first, and the elements
// from the first to the last one.
struct Extent {
    int64_t size[4], stride[4], span = 1;
    int dims = 0;
    bool apart = true;  // each stride passes what lies under it: no element twice
};
Extent extent_of(const Tensor& t) {
    Extent e;
    for (int64_t i = 0; i < t.dim(); ++i) {
        if (t.size(i) == 1) continue;
        int at = e.dims++;
        for (; at > 0 && e.stride[at - 1] < t.stride(i); --at) {
            e.size[at] = e.size[at - 1];
            e.stride[at] = e.stride[at - 1];
        }
        e.size[at] = t.size(i);
        e.stride[at] = t.stride(i);
    }
    for (int i = e.dims - 1; i >= 0; --i) {
        e.apart = e.apart && e.stride[i] >= e.span;
        e.span += (e.size[i] - 1) * e.stride[i];
    }
    return e;
}
// Whether an element of e lies `d` elements behind one of the same tensor: with strides
// apart, a dimension's share of d is one of two multiples of its stride.
bool meets(const Extent& e, int dim, int64_t d) {
    if (d == 0) return true;
    if (dim == e.dims) return false;
    const int64_t s = e.stride[dim], low = d / s - (d % s < 0);
    for (int64_t k = low; k <= low + 1; ++k)
        if (k < e.size[dim] && -k < e.size[dim] && meets(e, dim + 1, d - k * s)) return true;
    return false;
}
// An output whose rows overlap, or overlap those of its input (of the same shape and
// type) other than as the same tensor, is a race.
void apart(const Tensor& out, const Tensor& x, const char* name) {
    if (!out.numel()) return;
    const Extent o = extent_of(out), e = extent_of(x);
    if (!o.apart) value_error("out has elements that overlap");
    const auto bytes = static_cast<int64_t>(out.element_size());
    const int64_t d = reinterpret_cast<intptr_t>(out.data_ptr()) - reinterpret_cast<intptr_t>(x.data_ptr());
    if (d >= e.span * bytes || -d >= o.span * bytes) return;
    bool same = true;
    for (int64_t i = 0; i < out.dim(); ++i) same = same && (out.size(i) == 1 || out.stride(i) == x.stride(i));
    if (same && d % bytes == 0 && (d == 0 || !meets(o, 0, d / bytes))) return;
    value_error("out overlaps ", name, ": it has to be ", name, " itself or lie apart from it");
}
// Two contiguous tensors of a size.
void apart_whole(const Tensor& a, const Tensor& b, const char* names) {
    const intptr_t d = reinterpret_cast<intptr_t>(a.data_ptr()) - reinterpret_cast<intptr_t>(b.data_ptr());
    if (d < (intptr_t)b.nbytes() && -d < (intptr_t)a.nbytes()) value_error(names, " overlap");
}

// As torch's own out arguments, an output cannot be a part of the graph.
void writable(const Tensor& out) {
    no_tangent(out, "out");
    if (out.requires_grad() && at::GradMode::is_enabled())
        value_error("out requires a gradient: detach it or call under torch.no_grad()");
}

// (tokens, heads, dim) rows with adjacent elements
void rows(const Tensor& t, const char* name, int64_t tokens, int64_t dim, int64_t device) {
    on_device(t, name, device);
    if (t.dim() != 3 || (tokens >= 0 && t.size(0) != tokens) || t.size(2) != dim)
        value_error(name, " must be (", tokens >= 0 ? std::to_string(tokens) : "tokens", ", heads, ", dim, "), got ",
                    shape_of(t));
    if (t.stride(2) != 1) value_error(name, " must have adjacent elements in its last dimension");
}

int64_t table_rotated(const Tensor& t, int64_t most, int64_t device) {
    of_type(t, "table", at::kFloat);
    on_device(t, "table", device);
    if (t.dim() != 3 || t.size(2) != 2 || !t.is_contiguous())
        value_error("table must be a contiguous (positions, rotated / 2, 2) tensor, got ", shape_of(t));
    const int64_t rotated = 2 * t.size(1);
    if (rotated < 2 || rotated > most) value_error("table rotates ", rotated, " elements of heads of ", most);
    return rotated;
}

// The axes of a rotation's pairs as bfft/cache.py hands them over: their number, then the
// axis of each pair; empty for positions of one axis.
std::string axes_of(PyObject* o, int64_t rotated) {
    if (o == Py_None) return {};
    if (!PyBytes_Check(o) || PyBytes_GET_SIZE(o) < 2) value_error("bad axes");
    std::string axes(PyBytes_AS_STRING(o), (size_t)PyBytes_GET_SIZE(o));
    if (2 * ((int64_t)axes.size() - 1) != rotated)
        value_error("axes have ", (int64_t)axes.size() - 1, " pairs, the table has ", rotated / 2);
    return axes;
}
bfft_axes_desc axes_desc(const std::string& axes, const Tensor& positions) {
    return {axes.data() + 1, axes[0], positions.stride(0)};
}

int64_t positions_64(const Tensor& t, int64_t device) {
    if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong)
        type_error("positions must be int32 or int64, got ", at::toString(t.scalar_type()));
    on_device(t, "positions", device);
    return t.scalar_type() == at::kLong;
}

struct Cache {
    bfft_cache_desc desc;
    int64_t device;
    const Tensor* parts[4];  // k, v, k_scale, v_scale
};
Cache cache_of(PyObject* o) {
    if ((!PyTuple_Check(o) && !PyList_Check(o)) || PySequence_Fast_GET_SIZE(o) != 4)
        type_error("cache must be a PagedCache: (k, v, k_scale, v_scale)");
    PyObject** items = PySequence_Fast_ITEMS(o);
    const Tensor &k = tensor(items[0], "cache k"), &v = tensor(items[1], "cache v"),
                 &ks = tensor(items[2], "cache k_scale"), &vs = tensor(items[3], "cache v_scale");
    Cache c{{}, 0, {&k, &v, &ks, &vs}};
    if (k.scalar_type() == at::kChar)
        c.desc.code = BFFT_CODE_INT8;
    else if (k.scalar_type() == at::kFloat8_e4m3fn)
        c.desc.code = BFFT_CODE_E4M3;
    else
        type_error("cache k must be int8 or float8_e4m3fn, got ", at::toString(k.scalar_type()));
    of_type(v, "cache v", k.scalar_type());
    of_type(ks, "cache k_scale", at::kFloat);
    of_type(vs, "cache v_scale", at::kFloat);
    on_device(k, "cache k", -1);
    c.device = k.get_device();
    on_device(v, "cache v", c.device);
    on_device(ks, "cache k_scale", c.device);
    on_device(vs, "cache v_scale", c.device);
    if (k.dim() != 4 || v.sizes() != k.sizes())
        value_error("cache codes must both be (pages, kv_heads, page, dim), got ", shape_of(k), " and ", shape_of(v));
    if (ks.sizes() != k.sizes().slice(0, 2) || vs.sizes() != ks.sizes())
        value_error("cache scales must be (pages, kv_heads), got ", shape_of(ks), " and ", shape_of(vs));
    if (!k.is_contiguous() || !v.is_contiguous() || !ks.is_contiguous() || !vs.is_contiguous())
        value_error("cache tensors must be contiguous");
    constant(ks, "cache k_scale");
    constant(vs, "cache v_scale");
    c.desc.k = k.data_ptr();
    c.desc.v = v.data_ptr();
    c.desc.k_scale = ks.data_ptr();
    c.desc.v_scale = vs.data_ptr();
    c.desc.pages = k.size(0);
    c.desc.kv_heads = k.size(1);
    c.desc.page = k.size(2);
    c.desc.dim = k.size(3);
    return c;
}

bfft_sequence_desc sequences(PyObject* table_o, PyObject* lens_o, PyObject* starts_o, const char* lens_name,
                             int64_t tokens, int64_t device) {
    const Tensor &table = tensor(table_o, "block_table"), &lens = tensor(lens_o, lens_name),
                 &starts = tensor(starts_o, "starts");
    of_type(table, "block_table", at::kInt);
    of_type(lens, lens_name, at::kInt);
    of_type(starts, "starts", at::kInt);
    on_device(table, "block_table", device);
    on_device(lens, lens_name, device);
    on_device(starts, "starts", device);
    if (table.dim() != 2 || table.size(0) < 1 || table.size(1) < 1 || (table.size(1) > 1 && table.stride(1) != 1))
        value_error("block_table must be (sequences, pages) with adjacent pages, got ", shape_of(table));
    const int64_t n = table.size(0);
    if (lens.dim() != 1 || lens.size(0) != n || !lens.is_contiguous())
        value_error(lens_name, " must be contiguous (", n, ",), got ", shape_of(lens));
    if (starts.dim() != 1 || starts.size(0) != n + 1 || !starts.is_contiguous())
        value_error("starts must be contiguous (", n + 1, ",), got ", shape_of(starts));
    bfft_sequence_desc q;
    q.block_table = table.data_ptr();
    q.table_stride = table.stride(0);
    q.lens = lens.data_ptr();
    q.starts = starts.data_ptr();
    q.seqs = n;
    q.max_pages = table.size(1);
    q.tokens = tokens;
    return q;
}

void* stream_of(int64_t device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

int64_t integer(PyObject* o, const char* name, int64_t least) {
    if (!PyLong_Check(o) || PyBool_Check(o)) value_error(name, " must be an integer");
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    if (v < least) value_error(name, " must be at least ", least, ", got ", v);
    return v;
}

// ------------------------------------------------------------------ rotation

Tensor launch_rotate(const Tensor& x, const Tensor& positions, const Tensor& table, int64_t layout, int64_t direction,
                     const std::string& axes, const Tensor* out) {
    bfft_rotate_desc d;
    const bool batched = x.dim() == 4;
    const int64_t at = batched ? 1 : 0;
    Tensor y = out ? *out : at::empty(x.sizes(), x.options().requires_grad(false));
    if (!y.numel()) return y;
    d.batch = batched ? x.size(0) : 1;
    d.tokens = x.size(at);
    d.heads = x.size(at + 1);
    d.dim = x.size(at + 2);
    d.rotated = 2 * table.size(1);
    d.x_batch = batched ? x.stride(0) : 0;
    d.x_token = x.stride(at);
    d.x_head = x.stride(at + 1);
    d.y_batch = batched ? y.stride(0) : 0;
    d.y_token = y.stride(at);
    d.y_head = y.stride(at + 1);
    const int64_t lead = axes.empty() ? 0 : 1;  // positions: (axes,) before the tokens
    d.pos_batch = positions.dim() == lead + 2 ? positions.stride(lead) : 0;
    d.pos_token = positions.stride(positions.dim() - 1);
    d.table_rows = table.size(0);
    d.type = x.scalar_type() == at::kFloat ? BFFT_F32 : x.scalar_type() == at::kHalf ? BFFT_F16 : BFFT_BF16;
    d.layout = layout;
    d.transform_direction = direction;
    d.pos64 = positions.scalar_type() == at::kLong;
    d.device = x.get_device();
    if (out) written(y);
    if (axes.empty()) {
        check(g_entry.rotate(&d, x.data_ptr(), positions.data_ptr(), table.data_ptr(), y.data_ptr(), stream_of(d.device)),
              "rotate_positions");
    } else {
        const bfft_axes_desc a = axes_desc(axes, positions);
        check(g_entry.rotate_axes(&d, &a, x.data_ptr(), positions.data_ptr(), table.data_ptr(), y.data_ptr(),
                                  stream_of(d.device)),
              "rotate_positions");
    }
    return y;
}

// y is linear in x with orthogonal blocks times the table's amplitude: the gradient
// is the opposite direction's rotation, itself differentiable.
struct Rotate : public torch::autograd::Function<Rotate> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& positions,
                          const Tensor& table, int64_t layout, int64_t direction, const std::string& axes) {
        ctx->save_for_backward({positions, table});
        // (an entry less for one axis: each is some 0.2 us of a training step's host time)
        if (!axes.empty()) ctx->saved_data["axes"] = axes;
        ctx->saved_data["layout"] = layout;
        ctx->saved_data["direction"] = direction;
        return launch_rotate(x, positions, table, layout, direction, axes, nullptr);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const int64_t layout = ctx->saved_data["layout"].toInt(), direction = ctx->saved_data["direction"].toInt();
        const auto by_axis = ctx->saved_data.find("axes");
        const std::string axes = by_axis == ctx->saved_data.end() ? std::string() : by_axis->second.toStringRef();
        Tensor dy = grads[0];
        if (dy.stride(-1) != 1) dy = dy.contiguous();
        Tensor dx;
        if (at::GradMode::is_enabled() && dy.requires_grad())
            dx = Rotate::apply(dy, saved[0], saved[1], layout, 1 - direction, axes);
        else
            dx = launch_rotate(dy, saved[0], saved[1], layout, 1 - direction, axes, nullptr);
        return {dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// rotate(x, positions, table, layout, direction, out, axes)
PyObject* rotate(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 7, "rotate takes 7 arguments");
    const Tensor &x = tensor(args[0], "x"), &positions = tensor(args[1], "positions"), &table = tensor(args[2], "table");
    const int64_t layout = integer(args[3], "layout", 0), direction = integer(args[4], "direction", 0);
    type_id(x, "x");
    no_tangent(x, "x");
    on_device(x, "x", -1);
    const int64_t device = x.get_device();
    if (x.dim() != 3 && x.dim() != 4)
        value_error("x must be (tokens, heads, dim) or (batch, tokens, heads, dim), got ", shape_of(x));
    const std::string axes = axes_of(args[6], table_rotated(table, x.size(-1), device));
    constant(table, "table");
    if (x.stride(-1) != 1) value_error("x must have adjacent elements in its last dimension");
    positions_64(positions, device);
    const int64_t tokens = x.size(-3);
    const int64_t lead = axes.empty() ? 0 : 1;
    const bool all = !lead || (positions.dim() > 1 && positions.size(0) == axes[0]);
    const bool flat = positions.dim() == lead + 1 && positions.size(lead) == tokens;
    if (!all || (!flat && !(x.dim() == 4 && positions.dim() == lead + 2 && positions.size(lead) == x.size(0) &&
                            positions.size(lead + 1) == tokens))) {
        const std::string first = lead ? "(" + std::to_string((int)axes[0]) + " axes, " : "(";
        value_error("positions must be ", first, "tokens) or ", first, "batch, tokens) of x ", shape_of(x), ", got ",
                    shape_of(positions));
    }
    const Tensor* out = nullptr;
    if (args[5] != Py_None) {
        out = &tensor(args[5], "out");
        of_type(*out, "out", x.scalar_type());
        on_device(*out, "out", device);
        if (out->sizes() != x.sizes() || out->stride(-1) != 1)
            value_error("out must be ", shape_of(x), " with adjacent elements, got ", shape_of(*out));
        writable(*out);
        apart(*out, x, "x");
    }
    if (x.requires_grad() && at::GradMode::is_enabled()) {
        if (out) value_error("out cannot be given where x requires a gradient");
        return THPVariable_Wrap(Rotate::apply(x, positions, table, layout, direction, axes));
    }
    return THPVariable_Wrap(launch_rotate(x, positions, table, layout, direction, axes, out));
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ cache

// append(cache, k, v, block_table, held, starts, table, layout, positions, q, axes)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 11, "append takes 11 arguments");
    const Cache c = cache_of(args[0]);
    apart_whole(*c.parts[0], *c.parts[1], "cache k and v");
    apart_whole(*c.parts[2], *c.parts[3], "cache k_scale and v_scale");
    const Tensor &k = tensor(args[1], "k"), &v = tensor(args[2], "v");
    const int64_t heads = c.desc.kv_heads, dim = c.desc.dim;
    bfft_append_desc d{};
    d.type = type_id(k, "k");
    of_type(v, "v", k.scalar_type());
    rows(k, "k", -1, dim, c.device);
    const int64_t tokens = k.size(0);
    rows(v, "v", tokens, dim, c.device);
    if (k.size(1) != heads || v.size(1) != heads)
        value_error("k and v must have the cache's ", heads, " heads, got ", k.size(1), " and ", v.size(1));
    constant(k, "k");
    constant(v, "v");
    const bfft_sequence_desc q = sequences(args[3], args[4], args[5], "held", tokens, c.device);
    if (args[6] != Py_None) {
        const Tensor& table = tensor(args[6], "table");
        d.rotated = table_rotated(table, dim, c.device);
        constant(table, "table");
        d.table = table.data_ptr();
        d.table_rows = table.size(0);
    }
    d.layout = integer(args[7], "layout", 0);
    std::string axes;
    bfft_axes_desc by_axis{};
    if (args[10] != Py_None) {
        if (!d.table || args[8] == Py_None) value_error("axes need a table and positions");
        axes = axes_of(args[10], d.rotated);
    }
    if (args[8] != Py_None) {
        const Tensor& positions = tensor(args[8], "positions");
        d.pos64 = positions_64(positions, c.device);
        if (!axes.empty()) {
            if (positions.dim() != 2 || positions.size(0) != axes[0] || positions.size(1) != tokens ||
                (tokens > 1 && positions.stride(1) != 1))
                value_error("positions must be (", (int64_t)axes[0], " axes, ", tokens, "), adjacent within an axis, got ",
                            shape_of(positions));
            by_axis = axes_desc(axes, positions);
        } else if (positions.dim() != 1 || positions.size(0) != tokens || !positions.is_contiguous())
            value_error("positions must be contiguous (", tokens, ",), got ", shape_of(positions));
        d.positions = positions.data_ptr();
    }
    d.k = k.data_ptr();
    d.v = v.data_ptr();
    d.k_token = k.stride(0);
    d.k_head = k.stride(1);
    d.v_token = v.stride(0);
    d.v_head = v.stride(1);
    d.device = c.device;
    Tensor out;
    if (args[9] != Py_None) {
        const Tensor& query = tensor(args[9], "q");
        of_type(query, "q", k.scalar_type());
        rows(query, "q", tokens, dim, c.device);
        constant(query, "q");
        out = at::empty(query.sizes(), query.options().requires_grad(false));
        d.q = query.data_ptr();
        d.q_out = out.data_ptr();
        d.q_heads = query.size(1);
        d.q_token = query.stride(0);
        d.q_head = query.stride(1);
        d.o_token = out.stride(0);
        d.o_head = out.stride(1);
        if (!d.q_heads) d.q = d.q_out = nullptr;
    }
    if (tokens) {
        for (const Tensor* t : c.parts) written(*t);
        check(axes.empty() ? g_entry.append(&c.desc, &q, &d, stream_of(c.device))
                           : g_entry.append_axes(&c.desc, &q, &d, &by_axis, stream_of(c.device)),
              "append_rotated");
    }
    if (!out.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

PyObject* pair(const Tensor& a, const Tensor& b) {
    PyObject* x = THPVariable_Wrap(a);
    PyObject* y = x ? THPVariable_Wrap(b) : nullptr;
    PyObject* t = y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return t;
}

// read(cache, block_table, first, starts, tokens, type)
PyObject* read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 6, "read takes 6 arguments");
    const Cache c = cache_of(args[0]);
    const int64_t tokens = integer(args[4], "tokens", 0), type = integer(args[5], "type", 0);
    const bfft_sequence_desc q = sequences(args[1], args[2], args[3], "first", tokens, c.device);
    const auto options = at::TensorOptions()
                             .dtype(type == BFFT_F32 ? at::kFloat : type == BFFT_F16 ? at::kHalf : at::kBFloat16)
                             .device(at::kCUDA, (c10::DeviceIndex)c.device);
    const Tensor k = at::empty({tokens, c.desc.kv_heads, c.desc.dim}, options);
    const Tensor v = at::empty({tokens, c.desc.kv_heads, c.desc.dim}, options);
    if (tokens) check(g_entry.read(&c.desc, &q, type, k.data_ptr(), v.data_ptr(), c.device, stream_of(c.device)), "read_cache");
    return pair(k, v);
    END_HANDLE_TH_ERRORS
}

// attention(q, cache, block_table, lens, starts, softmax_scale, causal, window, return_lse, out, sinks, shared, groups)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 13, "attention takes 13 arguments");
    const Tensor& q = tensor(args[0], "q");
    const Cache c = cache_of(args[1]);
    bfft_attention_desc d{};
    d.type = type_id(q, "q", true);
    rows(q, "q", -1, c.desc.dim, c.device);
    constant(q, "q");
    const int64_t tokens = q.size(0);
    d.q_heads = q.size(1);
    if (d.q_heads < 1 || d.q_heads % c.desc.kv_heads)
        value_error(d.q_heads, " query heads are no multiple of the cache's ", c.desc.kv_heads);
    const bfft_sequence_desc s = sequences(args[2], args[3], args[4], "lens", tokens, c.device);
    d.softmax_scale = 1.0 / std::sqrt((double)c.desc.dim);
    if (args[5] != Py_None) {
        d.softmax_scale = PyFloat_AsDouble(args[5]);
        if (PyErr_Occurred()) throw python_error();
    }
    const int causal = PyObject_IsTrue(args[6]), want_lse = PyObject_IsTrue(args[8]);
    if (causal < 0 || want_lse < 0) throw python_error();
    d.causal = causal;
    d.window = integer(args[7], "window", 0);
    bfft_span_desc span{};
    span.sinks = integer(args[10], "sinks", 0);
    if (args[11] != Py_None) {
        const Tensor& shared = tensor(args[11], "shared");
        of_type(shared, "shared", at::kInt);
        on_device(shared, "shared", c.device);
        if (shared.dim() != 1 || !shared.is_contiguous())
            value_error("shared must be contiguous (groups,), got ", shape_of(shared));
        span.n_groups = shared.size(0);
        span.shared = shared.data_ptr();
        if (args[12] != Py_None) {
            const Tensor& groups = tensor(args[12], "groups");
            of_type(groups, "groups", at::kInt);
            on_device(groups, "groups", c.device);
            if (groups.dim() != 1 || groups.size(0) != span.n_groups + 1 || !groups.is_contiguous())
                value_error("groups must be contiguous (", span.n_groups + 1, ",), got ", shape_of(groups));
            span.groups = groups.data_ptr();
        } else if (span.n_groups != 1) {
            value_error("shared must be (1,) where no groups are given, got ", shape_of(shared));
        }
    } else if (args[12] != Py_None) {
        value_error("groups without shared");
    }
    const bool spans = span.sinks || span.n_groups;
    Tensor out, lse, scratch;
    if (args[9] != Py_None) {
        out = tensor(args[9], "out");
        of_type(out, "out", q.scalar_type());
        rows(out, "out", tokens, c.desc.dim, c.device);
        if (out.size(1) != d.q_heads) value_error("out must be ", shape_of(q), ", got ", shape_of(out));
        writable(out);
        apart(out, q, "q");
    } else {
        out = at::empty(q.sizes(), q.options().requires_grad(false));
    }
    if (want_lse) lse = at::empty({tokens, d.q_heads}, q.options().dtype(at::kFloat).requires_grad(false));
    if (tokens) {
        d.q = q.data_ptr();
        d.out = out.data_ptr();
        d.lse = want_lse ? lse.data_ptr() : nullptr;
        d.q_token = q.stride(0);
        d.q_head = q.stride(1);
        d.o_token = out.stride(0);
        d.o_head = out.stride(1);
        d.device = c.device;
        size_t bytes = 0;
        check(spans ? g_entry.span_workspace(&c.desc, &s, &d, &span, &bytes) : g_entry.workspace(&c.desc, &s, &d, &bytes),
              "cache_attention");
        if (bytes) {
            scratch = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte).requires_grad(false));
            d.workspace = scratch.data_ptr();
            d.workspace_bytes = (int64_t)bytes;
        }
        if (args[9] != Py_None) written(out);
        check(spans ? g_entry.span_attention(&c.desc, &s, &d, &span, stream_of(c.device))
                    : g_entry.attention(&c.desc, &s, &d, stream_of(c.device)),
              "cache_attention");
    }
    if (want_lse) return pair(out, lse);
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// bind(addresses of rotate, append, read, workspace, attention, last_error, rotate_axes, append_axes, span_workspace,
// span_attention)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 10, "bind takes 10 addresses");
    void* p[10];
    for (int i = 0; i < 10; ++i) {
        p[i] = PyLong_AsVoidPtr(args[i]);
        if (!p[i]) value_error("null entry point");
    }
    g_entry.rotate = reinterpret_cast<decltype(g_entry.rotate)>(p[0]);
    g_entry.append = reinterpret_cast<decltype(g_entry.append)>(p[1]);
    g_entry.read = reinterpret_cast<decltype(g_entry.read)>(p[2]);
    g_entry.workspace = reinterpret_cast<decltype(g_entry.workspace)>(p[3]);
    g_entry.attention = reinterpret_cast<decltype(g_entry.attention)>(p[4]);
    g_entry.last_error = reinterpret_cast<decltype(g_entry.last_error)>(p[5]);
    g_entry.rotate_axes = reinterpret_cast<decltype(g_entry.rotate_axes)>(p[6]);
    g_entry.append_axes = reinterpret_cast<decltype(g_entry.append_axes)>(p[7]);
    g_entry.span_workspace = reinterpret_cast<decltype(g_entry.span_workspace)>(p[8]);
    g_entry.span_attention = reinterpret_cast<decltype(g_entry.span_attention)>(p[9]);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

PyMethodDef g_methods[] = {{"bind", fast<bind>(), METH_FASTCALL, nullptr},
                           {"rotate", fast<rotate>(), METH_FASTCALL, nullptr},
                           {"append", fast<append>(), METH_FASTCALL, nullptr},
                           {"read", fast<read>(), METH_FASTCALL, nullptr},
                           {"attention", fast<attention>(), METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "bfft_torch", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit_bfft_torch(void) { return PyModule_Create(&g_module); }
