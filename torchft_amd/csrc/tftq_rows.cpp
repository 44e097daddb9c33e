// _rows: the calls of the row operators (rows.py), with their gradients.
//
// Every call checks its arguments, allocates what it returns, and launches with the functions of libtftq.so (tftq.h), whose
// addresses it has been given (bind), on the stream that is current on the tensors' device.  The gradients are
// autograd nodes in C++: a norm's forward and backward pass through nodes written in Python takes about 100 us
// of host time, here less than half of it.
//
// A call that the operator does not take raises AssertionError, a failure of the library RuntimeError.  The interpreter
// is left to other threads while a call works.
//
// Host code only; built with the host compiler against the Python and libtorch headers (torchft_amd/_build.py).
// Not part of libtftq.so, whose C ABI has no Python or torch types.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <atomic>
#include <string>
#include <unordered_set>
#include <vector>

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/DynamicTypes.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

// An argument that the operator does not take.
struct Refused : std::exception {
    std::string why;
    explicit Refused(std::string w) : why(std::move(w)) {}
    const char *what() const noexcept override { return why.c_str(); }
};
void require(bool ok, const char *why)
{
    if (!ok) throw Refused(why);
}

// tftq.h
struct {
    const char *(*strerror)(int) = nullptr;
    int (*check_device)(int) = nullptr;
    int (*rms_norm)(int, int, const void *, int64_t, int64_t, int64_t, const void *, int64_t, const void *, int64_t, int64_t, float, void *, void *, void *,
                    float *, int, void *) = nullptr;
    int64_t (*rms_norm_backward_workspace)(int, int64_t, int64_t) = nullptr;
    int (*rms_norm_backward)(int, int, const void *, const void *, const void *, int64_t, int64_t, int64_t, const void *, int64_t, int64_t, float, void *,
                             void *, void *, int64_t, int, void *) = nullptr;
    int (*dropout)(int, const void *, const void *, int64_t, double, int64_t, const int64_t *, int64_t, void *, int, void *) = nullptr;
    int (*embedding)(int, int, const void *, int64_t, const void *, int64_t, int64_t, int64_t, float, void *, int, void *) = nullptr;
    int64_t (*embedding_backward_workspace)(int, int64_t, int64_t, int64_t) = nullptr;
    int (*embedding_backward)(int, int, const void *, int64_t, int64_t, const void *, int64_t, int64_t, float, void *, void *, int64_t, int,
                              void *) = nullptr;
    int64_t (*expert_sort_workspace)(int64_t, int64_t) = nullptr;
    int (*expert_sort)(int, const void *, int64_t, int64_t, int32_t *, int32_t *, int32_t *, void *, int64_t, int, void *) = nullptr;
    int (*dispatch)(int, const void *, int64_t, int64_t, int64_t, int64_t, const int32_t *, const int32_t *, void *, int, void *) = nullptr;
    int (*combine)(int, int, const void *, int64_t, const void *, int64_t, int64_t, int64_t, const int32_t *, const int32_t *, void *, int,
                   void *) = nullptr;
    int (*combine_backward)(int, int, const void *, int64_t, const void *, int64_t, const void *, int64_t, int64_t, int64_t, const int32_t *,
                            const int32_t *, void *, void *, int, void *) = nullptr;
    int (*fp8_rows_dequantize)(int, const void *, const float *, int64_t, int64_t, void *, int, void *) = nullptr;
} lib;

[[noreturn]] void failed(int code, const char *what)
{
    throw std::runtime_error(std::string(what) + " failed: " + (code > 0 ? "hipError_t " + std::to_string(code) : lib.strerror(code)));
}
void checked(int code, const char *what)
{
    if (code) failed(code, what);
}
int64_t bytes_needed(int64_t size, const char *what)
{
    if (size < 0) failed(static_cast<int>(size), what);
    return size;
}

// Tensors that stand for others.
constexpr c10::DispatchKeySet WRAPPERS({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                        c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::BatchedNestedTensor,
                                        c10::DispatchKey::Functionalize});

// Whether this thread's operations are recorded, or made up, and not only done: a trace would have the allocation of a result and not the
// kernel that writes it.  Modes that look on are no matter.
bool traced()
{
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Key = c10::impl::TorchDispatchModeKey;
    if (torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch)) return true;
    return Modes::any_modes_set() && (Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::FUNCTIONAL));
}
const char *const TRACED = "Only plain tensors are supported: a trace of the call would not have its kernels";

int code_of(const Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    default: throw Refused("Only fp32, fp16 and bf16 are supported");
    }
}

// A device that runs the kernels; the last of a call's checks.
void ready(const Tensor &t)
{
    static std::atomic<uint64_t> known{0};
    require(t.device().is_cuda(), "A GPU tensor is required");
    const int i = t.device().index();
    if (i < 64 && (known.load() >> i & 1)) return;
    checked(lib.check_device(i), "tftq_check_device");
    if (i < 64) known |= 1ull << i;
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

Tensor fresh(c10::IntArrayRef sizes, at::ScalarType type, const Tensor &beside)
{
    return at::empty(sizes, at::TensorOptions(type).device(beside.device()));
}
Tensor bytes_of(int64_t n, const Tensor &beside) { return n ? fresh({n}, at::kByte, beside) : Tensor(); }
void *data_of(const Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

// A tensor as rows: the last dimension in a piece, the others one stride apart, or with `grouped` two (heads inside a wider
// row, say: groups of rows one stride apart, the groups another); `held` is what the addresses are of.
struct Rows {
    Tensor held;
    int64_t rows = 1, cols = 0, stride = 0, group = 1, group_stride = 0;

    explicit Rows(const Tensor &t, bool grouped = false) : held(t.resolve_neg())
    {
        cols = t.size(-1);
        for (int64_t d = 0; d + 1 < t.dim(); d++) rows *= t.size(d);
        if (rows != 0 && cols != 0 && !describe(grouped)) {
            held = held.contiguous();
            group = 0;
        }
        if (rows == 0 || cols == 0 || group == 0) {
            stride = cols;
            group = rows;
        }
    }
    bool describe(bool grouped)
    {
        const c10::IntArrayRef size = held.sizes(), step = held.strides();
        const int64_t last = held.dim() - 1;
        if (cols > 1 && step[last] != 1) return false;
        int levels = 0;  // 1: rows, 2: groups of them
        int64_t expect = 0;
        for (int64_t d = last - 1; d >= 0; d--) {
            if (size[d] == 1) continue;
            if (levels == 0 || step[d] != expect) {
                if (step[d] < cols || ++levels > (grouped ? 2 : 1)) return false;
                (levels == 1 ? stride : group_stride) = step[d];
            }
            if (levels == 1) group *= size[d];
            expect = step[d] * size[d];
        }
        if (levels == 0) stride = cols;
        return true;
    }
    void *data() const { return data_of(held); }
};

bool same_sizes(const Tensor &a, const Tensor &b) { return a.sizes() == b.sizes(); }
bool wants_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const Maybe &t) { return t && wants_grad(*t); }
Tensor or_none(const Maybe &t) { return t ? *t : Tensor(); }

// Begins a backward pass, which is not traced either.  Under a stream capture no gradient may go to a node of the default stream (a
// leaf's, made with an eager graph of the leaf that still lives), neither from here nor from a node behind: that stream would have to wait for
// the capture, which it cannot, and the capture breaks off in ways that the process may not survive.  Refused here, where nothing has crossed
// yet.
void begin_backward(const Tensor &beside)
{
    using torch::autograd::Node;
    require(!traced(), TRACED);
    const c10::hip::HIPStream here = c10::hip::getCurrentHIPStream(beside.device().index());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (here.id() == 0 || hipStreamIsCapturing(here.stream(), &status) != hipSuccess || status != hipStreamCaptureStatusActive) return;
    const std::shared_ptr<Node> node = torch::autograd::get_current_node();
    if (!node) return;
    const auto *runs = torch::autograd::get_current_graph_task_exec_info();  // empty: all nodes
    std::vector<const Node *> to_see = {node.get()};
    std::unordered_set<const Node *> seen = {node.get()};
    while (!to_see.empty()) {
        const Node *from = to_see.back();
        to_see.pop_back();
        for (const torch::autograd::Edge &edge : from->next_edges()) {
            Node *next = edge.function.get();
            if (!next || !seen.insert(next).second) continue;
            bool follow = true;  // a node whose gradient is only wanted gets one too, but hands none on
            if (runs && !runs->empty()) {
                const auto it = runs->find(next);
                if (it == runs->end() || !it->second.should_execute()) continue;
                follow = it->second.needed_;
            }
            const auto there = next->stream();
            require(!there || there->id() != 0, "A backward pass cannot be captured while a graph of the same tensors lives that was made on the default stream");
            if (follow) to_see.push_back(next);
        }
    }
}

// What a backward pass returns where second derivatives may be asked for: an error once they are.
variable_list once(variable_list grads, const variable_list &from, const char *name)
{
    if (!at::GradMode::is_enabled()) return grads;
    bool follow = false;
    for (const Tensor &t : from) follow = follow || wants_grad(t);
    if (!follow) return grads;
    variable_list some;
    for (const Tensor &t : grads)
        if (t.defined()) some.push_back(t.detach().set_requires_grad(true));
    if (some.empty()) return grads;
    const int64_t n = static_cast<int64_t>(some.size());
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " can be differentiated once", n);
    some = (*error)(std::move(some));
    size_t i = 0;
    for (Tensor &t : grads)
        if (t.defined()) t = some[i++];
    return grads;
}

// ---------------------------------------------------------------------------
// norm
// ---------------------------------------------------------------------------
// (y, h), or (codes, h, scales)
variable_list norm_forward(const Tensor &x_, const Tensor &weight_, const Tensor &residual_, double eps, bool fp8)
{
    const Rows x(x_, true);
    const Tensor weight = weight_.defined() ? weight_.resolve_neg().contiguous() : weight_;
    Tensor y = fresh(x_.sizes(), fp8 ? at::kFloat8_e4m3fn : x_.scalar_type(), x_), h, scales;
    if (fp8) {
        c10::SmallVector<int64_t, 6> sizes(x_.sizes().begin(), x_.sizes().end());
        sizes.back() = 1;
        scales = fresh(sizes, at::kFloat, x_);
        if (x.cols == 0) scales.fill_(1.0);
    }
    std::optional<Rows> residual;
    if (residual_.defined()) {
        residual.emplace(residual_);
        h = fresh(x_.sizes(), x_.scalar_type(), x_);
    }
    checked(lib.rms_norm(code_of(x_), weight.defined() ? code_of(weight) : 0, x.data(), x.stride, x.group, x.group_stride,
                         residual ? residual->data() : nullptr, residual ? residual->stride : 0, data_of(weight), x.rows, x.cols,
                         static_cast<float>(eps), data_of(h), fp8 ? nullptr : data_of(y), fp8 ? data_of(y) : nullptr,
                         static_cast<float *>(data_of(scales)), x_.device().index(), stream_of(x_)), "tftq_rms_norm");
    return {y, h, scales};
}

struct Norm : torch::autograd::Function<Norm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Maybe &weight, const Maybe &residual, double eps)
    {
        variable_list got = norm_forward(x, or_none(weight), or_none(residual), eps, false);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({residual ? got[1] : x, or_none(weight)});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["residual"] = residual.has_value();
        if (residual) return {got[0], got[1]};
        return {got[0]};
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &h_ = saved[0], &weight_ = saved[1];
        const bool with_residual = ctx->saved_data["residual"].toBool();
        size_t edge = 0;
        const bool for_x = ctx->needs_input_grad(edge++), for_w = weight_.defined() && ctx->needs_input_grad(edge++),
                   for_r = with_residual && ctx->needs_input_grad(edge++);
        const Tensor &dy_ = grads[0];
        const Tensor dh_ = with_residual ? grads[1] : Tensor();
        Tensor dx, dw;
        if (dy_.defined() || dh_.defined()) begin_backward(h_);
        if (!dy_.defined()) dx = dh_;
        else {
            at::NoGradGuard guard;
            const Rows h(h_, true);
            const Tensor dy = dy_.resolve_neg().contiguous(), dh = dh_.defined() ? dh_.resolve_neg().contiguous() : dh_,
                         weight = weight_.defined() ? weight_.resolve_neg().contiguous() : weight_;
            if (for_x || for_r) dx = fresh(h_.sizes(), h_.scalar_type(), h_);
            if (for_w) dw = fresh(weight.sizes(), weight.scalar_type(), h_);
            const int64_t size = bytes_needed(lib.rms_norm_backward_workspace(code_of(h_), h.rows, h.cols), "tftq_rms_norm_backward_workspace");
            const Tensor workspace = bytes_of(size, h_);
            if (dx.defined() || dw.defined())
                checked(lib.rms_norm_backward(code_of(h_), weight.defined() ? code_of(weight) : 0, data_of(dy), data_of(dh), h.data(), h.stride, h.group, h.group_stride,
                                              data_of(weight), h.rows, h.cols, static_cast<float>(ctx->saved_data["eps"].toDouble()), data_of(dx),
                                              data_of(dw), data_of(workspace), size, h_.device().index(), stream_of(h_)),
                        "tftq_rms_norm_backward");
        }
        variable_list out = {for_x ? dx : Tensor(), dw, for_r ? dx : Tensor(), Tensor()};
        return once(out, {dy_, dh_, h_, weight_}, "rms_norm");
    }
};

// ---------------------------------------------------------------------------
// dropout
// ---------------------------------------------------------------------------
Tensor dropout_run(const Tensor &x_, const Tensor &residual_, double p, int64_t seed, const Tensor &seed_at, int64_t offset)
{
    const Tensor x = x_.resolve_neg().contiguous(), residual = residual_.defined() ? residual_.resolve_neg().contiguous() : residual_;
    const Tensor out = fresh(x_.sizes(), x_.scalar_type(), x_);
    checked(lib.dropout(code_of(x_), data_of(x), data_of(residual), x.numel(), p, seed, static_cast<const int64_t *>(data_of(seed_at)), offset,
                        data_of(out), x_.device().index(), stream_of(x_)), "tftq_dropout");
    return out;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Maybe &residual, const Maybe &seed_at, double p, int64_t seed, int64_t offset)
    {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({or_none(seed_at)});
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["residual"] = residual.has_value();
        return dropout_run(x, or_none(residual), p, seed, or_none(seed_at), offset);
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const Tensor &dy = grads[0], seed_at = ctx->get_saved_variables()[0];
        Tensor dx;
        if (dy.defined()) begin_backward(dy);
        if (dy.defined() && ctx->needs_input_grad(0)) {
            at::NoGradGuard guard;
            dx = dropout_run(dy, Tensor(), ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(), seed_at, ctx->saved_data["offset"].toInt());
        }
        const bool for_r = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1);
        variable_list d = once({dx}, {dy}, "dropout");
        return {d[0], for_r ? dy : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// ---------------------------------------------------------------------------
// embedding
// ---------------------------------------------------------------------------
Tensor embedding_run(const Tensor &ids_, const Tensor &table_, double scale)
{
    const Tensor ids = ids_.contiguous();
    const Rows table(table_);
    c10::SmallVector<int64_t, 6> sizes(ids.sizes().begin(), ids.sizes().end());
    sizes.push_back(table.cols);
    const Tensor out = fresh(sizes, table_.scalar_type(), table_);
    checked(lib.embedding(code_of(table_), static_cast<int>(ids.element_size()), data_of(ids), ids.numel(), table.data(), table.rows, table.cols,
                          table.stride, static_cast<float>(scale), data_of(out), table_.device().index(), stream_of(table_)), "tftq_embedding");
    return out;
}

struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext *ctx, const Tensor &table, const Tensor &ids, double scale, int64_t skip)
    {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({ids});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["skip"] = skip;
        ctx->saved_data["vocab"] = table.size(0);
        ctx->saved_data["cols"] = table.size(1);
        return embedding_run(ids, table, scale);
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const Tensor &dy_ = grads[0];
        Tensor dtable;
        if (dy_.defined()) {
            begin_backward(dy_);
            at::NoGradGuard guard;
            const Tensor ids = ctx->get_saved_variables()[0].contiguous(), dy = dy_.resolve_neg().contiguous();
            const int64_t vocab = ctx->saved_data["vocab"].toInt(), cols = ctx->saved_data["cols"].toInt(), n = ids.numel();
            dtable = fresh({vocab, cols}, dy.scalar_type(), dy);
            const int64_t size = bytes_needed(lib.embedding_backward_workspace(code_of(dy), n, vocab, cols), "tftq_embedding_backward_workspace");
            const Tensor workspace = bytes_of(size, dy);
            checked(lib.embedding_backward(code_of(dy), static_cast<int>(ids.element_size()), data_of(ids), n, ctx->saved_data["skip"].toInt(),
                                           data_of(dy), vocab, cols, static_cast<float>(ctx->saved_data["scale"].toDouble()), data_of(dtable),
                                           data_of(workspace), size, dy.device().index(), stream_of(dy)), "tftq_embedding_backward");
        }
        variable_list d = once({dtable}, {dy_}, "embedding");
        return {d[0], Tensor(), Tensor(), Tensor()};
    }
};

// ---------------------------------------------------------------------------
// experts
// ---------------------------------------------------------------------------
// Where the tokens' choices go: position [tokens, k] and offsets [experts + 1], both int32.
struct Places {
    Tensor position, offsets;
    int64_t tokens, k;

    Places(const Tensor &p, const Tensor &o) : position(p), offsets(o), tokens(p.size(0)), k(p.size(1)) {}
    const int32_t *at() const { return static_cast<const int32_t *>(data_of(position)); }
    const int32_t *used() const { return static_cast<const int32_t *>(offsets.data_ptr()) + offsets.numel() - 1; }
};

Tensor dispatch_run(const Tensor &x_, const Places &places)
{
    const Rows x(x_);
    const Tensor out = fresh({places.tokens * places.k, x.cols}, x_.scalar_type(), x_);
    checked(lib.dispatch(static_cast<int>(x_.element_size()), x.data(), x.stride, places.tokens, places.k, x.cols, places.at(), places.used(),
                         data_of(out), x_.device().index(), stream_of(x_)), "tftq_dispatch");
    return out;
}

Tensor combine_run(const Tensor &rows_, const Places &places, const Tensor &weights_)
{
    const Rows rows(rows_);
    const Tensor weights = weights_.defined() ? weights_.resolve_neg().contiguous() : weights_;
    const Tensor out = fresh({places.tokens, rows.cols}, rows_.scalar_type(), rows_);
    checked(lib.combine(code_of(rows_), weights.defined() ? code_of(weights) : 0, rows.data(), rows.stride, data_of(weights), places.tokens, places.k,
                        rows.cols, places.at(), places.used(), data_of(out), rows_.device().index(), stream_of(rows_)), "tftq_combine");
    return out;
}

struct Dispatch : torch::autograd::Function<Dispatch> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &position, const Tensor &offsets)
    {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({position, offsets});
        return dispatch_run(x, Places(position, offsets));
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const variable_list saved = ctx->get_saved_variables();
        Tensor dx;
        if (grads[0].defined()) {
            begin_backward(grads[0]);
            at::NoGradGuard guard;
            dx = combine_run(grads[0], Places(saved[0], saved[1]), Tensor());
        }
        variable_list d = once({dx}, {grads[0]}, "dispatch");
        return {d[0], Tensor(), Tensor()};
    }
};

struct Combine : torch::autograd::Function<Combine> {
    static Tensor forward(AutogradContext *ctx, const Tensor &rows, const Maybe &weights, const Tensor &position, const Tensor &offsets)
    {
        ctx->set_materialize_grads(false);
        // the rows are needed for the weights' gradient alone
        ctx->save_for_backward({wants_grad(weights) ? rows : Tensor(), or_none(weights), position, offsets});
        return combine_run(rows, Places(position, offsets), or_none(weights));
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &rows_ = saved[0], &weights_ = saved[1], &dy_ = grads[0];
        const bool for_rows = ctx->needs_input_grad(0), for_weights = rows_.defined() && ctx->needs_input_grad(1);
        Tensor drows, dweights;
        if (dy_.defined() && (for_rows || for_weights)) {
            begin_backward(dy_);
            at::NoGradGuard guard;
            const Places places(saved[2], saved[3]);
            const Rows dy(dy_);
            const Tensor weights = weights_.defined() ? weights_.resolve_neg().contiguous() : weights_;
            if (for_rows) drows = fresh({places.tokens * places.k, dy.cols}, dy_.scalar_type(), dy_);
            if (for_weights) dweights = fresh(weights.sizes(), weights.scalar_type(), dy_);
            const Rows rows(rows_.defined() ? rows_ : dy_);
            checked(lib.combine_backward(code_of(dy_), weights.defined() ? code_of(weights) : 0, dy.data(), dy.stride,
                                         for_weights ? rows.data() : nullptr, rows.stride, data_of(weights), places.tokens, places.k, dy.cols,
                                         places.at(), places.used(), data_of(drows), data_of(dweights), dy_.device().index(), stream_of(dy_)),
                    "tftq_combine_backward");
        }
        variable_list d = once({drows, dweights}, {dy_, rows_, weights_}, "combine");
        return {d[0], d[1], Tensor(), Tensor()};
    }
};

// ---------------------------------------------------------------------------
// what Python calls
// ---------------------------------------------------------------------------
// Leaves the interpreter to other threads for the lifetime of the object, exceptions included.
struct WithoutInterpreter {
    PyThreadState *state = PyEval_SaveThread();
    ~WithoutInterpreter() { PyEval_RestoreThread(state); }
};

struct PythonError {};  // one that is set already

Tensor tensor_arg(PyObject *o, const char *why)
{
    require(THPVariable_Check(o), why);
    const Tensor t = THPVariable_Unpack(o);
    require(t.defined() && !t.key_set().has_any(WRAPPERS) && t.layout() == at::kStrided, "Only plain tensors are supported");
    require(!t._fw_grad(0).defined(), "Forward-mode differentiation is not supported");
    return t;
}
Maybe maybe_tensor(PyObject *o, const char *why) { return o == Py_None ? Maybe() : Maybe(tensor_arg(o, why)); }
double number_arg(PyObject *o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
    return v;
}
int64_t whole_arg(PyObject *o)
{
    PyObject *i = PyNumber_Index(o);
    if (!i) throw PythonError{};
    const int64_t v = PyLong_AsLongLong(i);
    Py_DECREF(i);
    if (v == -1 && PyErr_Occurred()) throw PythonError{};
    return v;
}
PyObject *wrap(const Tensor &t)
{
    PyObject *o = THPVariable_Wrap(t);
    if (!o) throw PythonError{};
    return o;
}
PyObject *tuple_of(const variable_list &list)
{
    PyObject *out = PyTuple_New(static_cast<Py_ssize_t>(list.size()));
    if (!out) throw PythonError{};
    for (size_t i = 0; i < list.size(); i++) {
        PyObject *o = THPVariable_Wrap(list[i]);
        if (!o) {
            Py_DECREF(out);
            throw PythonError{};
        }
        PyTuple_SET_ITEM(out, static_cast<Py_ssize_t>(i), o);
    }
    return out;
}

template <class F>
PyObject *call(const char *name, Py_ssize_t got, Py_ssize_t want, F body)
{
    if (got != want) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", name, want);
        return nullptr;
    }
    HANDLE_TH_ERRORS
    try {
        require(!traced(), TRACED);
        return body();
    } catch (const Refused &e) {
        PyErr_SetString(PyExc_AssertionError, e.why.c_str());
    } catch (const PythonError &) {
    }
    return nullptr;
    END_HANDLE_TH_ERRORS
}

const char *const NO_TENSOR = "A tensor is required";

void check_weight(const Tensor &w, const Tensor &x, int64_t n)
{
    require(w.dim() == 1 && w.size(0) == n, "The weight is one number for every column");
    require(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, "The weight has the type of the rows or is fp32");
    require(w.device() == x.device(), "All inputs must be on the same device");
}

// rms_norm(x, weight, residual, eps, fp8) -> y or (y, h); with fp8 (codes, scales) or (codes, scales, h)
PyObject *rms_norm(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return call("rms_norm", n, 5, [&]() -> PyObject * {
        const Tensor x = tensor_arg(args[0], NO_TENSOR);
        const Maybe weight = maybe_tensor(args[1], NO_TENSOR), residual = maybe_tensor(args[2], NO_TENSOR);
        const double eps = number_arg(args[3]);
        const bool fp8 = args[4] == Py_True;
        require(x.dim() >= 1, "x has at least one dimension");
        code_of(x);
        if (weight) check_weight(*weight, x, x.size(-1));
        if (residual) {
            require(same_sizes(*residual, x), "The residual has another shape than x");
            require(residual->scalar_type() == x.scalar_type(), "The residual has another type than x");
            require(residual->device() == x.device(), "All inputs must be on the same device");
        }
        require(eps >= 0, "eps is negative");
        const bool follow = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(residual));
        require(!fp8 || !follow, "A norm in 8 bits has no gradient");
        ready(x);
        variable_list out;
        {
            WithoutInterpreter others_run;
            if (follow) out = Norm::apply(x, weight, residual, eps);
            else {
                at::NoGradGuard guard;
                const variable_list got = norm_forward(x, or_none(weight), or_none(residual), eps, fp8);
                out = {got[0]};
                if (fp8) out.push_back(got[2]);
                if (residual) out.push_back(got[1]);
            }
        }
        return out.size() == 1 ? wrap(out[0]) : tuple_of(out);
    });
}

// fp8_rows(codes, scales, type) -> the values
PyObject *fp8_rows(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return call("fp8_rows", n, 3, [&]() -> PyObject * {
        const Tensor codes = tensor_arg(args[0], NO_TENSOR), scales = tensor_arg(args[1], NO_TENSOR);
        const int64_t type = whole_arg(args[2]);
        static const at::ScalarType types[3] = {at::kFloat, at::kHalf, at::kBFloat16};
        require(type >= 0 && type < 3, "Only fp32, fp16 and bf16 are supported");
        require(codes.scalar_type() == at::kFloat8_e4m3fn && codes.dim() >= 1, "Codes are float8_e4m3fn");
        require(scales.scalar_type() == at::kFloat && scales.dim() == codes.dim() && scales.size(-1) == 1 &&
                    scales.sizes().slice(0, codes.dim() - 1) == codes.sizes().slice(0, codes.dim() - 1),
                "Scales are one fp32 number for every row");
        require(scales.device() == codes.device(), "All inputs must be on the same device");
        ready(codes);
        Tensor out;
        {
            WithoutInterpreter others_run;
            at::NoGradGuard guard;
            const Tensor c = codes.contiguous(), s = scales.contiguous();
            out = fresh(codes.sizes(), types[type], codes);
            const int64_t cols = codes.size(-1), rows = cols ? codes.numel() / cols : 0;
            checked(lib.fp8_rows_dequantize(static_cast<int>(type), data_of(c), static_cast<const float *>(data_of(s)), rows, cols, data_of(out),
                                            codes.device().index(), stream_of(codes)), "tftq_fp8_rows_dequantize");
        }
        return wrap(out);
    });
}

// dropout(x, p, seed, offset, residual) -> residual + dropout of x
PyObject *dropout(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return call("dropout", n, 5, [&]() -> PyObject * {
        const Tensor x = tensor_arg(args[0], NO_TENSOR);
        const double p = number_arg(args[1]);
        Maybe seed_at;
        int64_t seed = 0;
        if (THPVariable_Check(args[2])) {
            seed_at = tensor_arg(args[2], NO_TENSOR);
            require(seed_at->scalar_type() == at::kLong && seed_at->numel() == 1, "The seed is a number, or a tensor of one int64");
            require(seed_at->device() == x.device(), "All inputs must be on the same device");
        } else seed = whole_arg(args[2]);
        const int64_t offset = whole_arg(args[3]);
        const Maybe residual = maybe_tensor(args[4], NO_TENSOR);
        code_of(x);
        require(p >= 0 && p <= 1, "p is between 0 and 1");
        if (residual) {
            require(same_sizes(*residual, x), "The residual has another shape than x");
            require(residual->scalar_type() == x.scalar_type(), "The residual has another type than x");
            require(residual->device() == x.device(), "All inputs must be on the same device");
        }
        const bool follow = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(residual));
        ready(x);
        Tensor out;
        {
            WithoutInterpreter others_run;
            if (follow) out = Dropout::apply(x, residual, seed_at, p, seed, offset);
            else {
                at::NoGradGuard guard;
                out = dropout_run(x, or_none(residual), p, seed, or_none(seed_at), offset);
            }
        }
        return wrap(out);
    });
}

// embedding(ids, table, scale, skip) -> rows
PyObject *embedding(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return call("embedding", n, 4, [&]() -> PyObject * {
        const Tensor ids = tensor_arg(args[0], NO_TENSOR), table = tensor_arg(args[1], NO_TENSOR);
        const double scale = number_arg(args[2]);
        const int64_t skip = args[3] == Py_None ? -1 : whole_arg(args[3]);
        require(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "Token numbers are int64 or int32");
        require(table.dim() == 2, "Only 2D tensors are supported");
        code_of(table);
        require(args[3] == Py_None || (skip >= 0 && skip < table.size(0)), "padding_idx is outside the table");
        require(ids.device() == table.device(), "All inputs must be on the same device");
        ready(table);
        Tensor out;
        {
            WithoutInterpreter others_run;
            if (at::GradMode::is_enabled() && wants_grad(table)) out = Embedding::apply(table, ids, scale, skip);
            else {
                at::NoGradGuard guard;
                out = embedding_run(ids, table, scale);
            }
        }
        return wrap(out);
    });
}

// sort_by_expert(chosen, experts) -> (order, position, offsets)
PyObject *sort_by_expert(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return call("sort_by_expert", n, 2, [&]() -> PyObject * {
        const Tensor chosen_ = tensor_arg(args[0], NO_TENSOR);
        const int64_t experts = whole_arg(args[1]);
        require(chosen_.scalar_type() == at::kLong || chosen_.scalar_type() == at::kInt, "Numbers of experts are int64 or int32");
        require(chosen_.dim() == 1 || chosen_.dim() == 2, "The experts of tokens are [tokens] or [tokens, k]");
        require(experts >= 1, "At least one expert is required");
        ready(chosen_);
        variable_list out;
        {
            WithoutInterpreter others_run;
            at::NoGradGuard guard;
            const Tensor chosen = chosen_.contiguous();
            const int64_t choices = chosen.numel();
            const int64_t size = bytes_needed(lib.expert_sort_workspace(choices, experts), "tftq_expert_sort_workspace");
            const Tensor workspace = bytes_of(size, chosen), order = fresh({choices}, at::kInt, chosen),
                         position = fresh({chosen.size(0), chosen.dim() == 2 ? chosen.size(1) : 1}, at::kInt, chosen),
                         offsets = fresh({experts + 1}, at::kInt, chosen);
            checked(lib.expert_sort(static_cast<int>(chosen.element_size()), data_of(chosen), choices, experts, static_cast<int32_t *>(data_of(order)),
                                    static_cast<int32_t *>(data_of(position)), static_cast<int32_t *>(data_of(offsets)), data_of(workspace), size,
                                    chosen.device().index(), stream_of(chosen)), "tftq_expert_sort");
            out = {order, position, offsets};
        }
        return tuple_of(out);
    });
}

// What position and offsets have to be beside x, whose kernels trust the places in them.
void check_places(const Tensor &position, const Tensor &offsets, const Tensor &x)
{
    require(position.scalar_type() == at::kInt && offsets.scalar_type() == at::kInt && position.dim() == 2 && offsets.dim() == 1 &&
                position.is_contiguous() && offsets.is_contiguous() && offsets.numel() >= 1, "The order is one of sort_by_expert");
    require(position.device() == x.device() && offsets.device() == x.device(), "All inputs must be on the same device");
}

// dispatch(x, position, offsets) -> the rows by expert
PyObject *dispatch(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return call("dispatch", n, 3, [&]() -> PyObject * {
        const Tensor x = tensor_arg(args[0], NO_TENSOR), position = tensor_arg(args[1], NO_TENSOR), offsets = tensor_arg(args[2], NO_TENSOR);
        require(x.dim() == 2, "Only 2D tensors are supported");
        check_places(position, offsets, x);
        require(x.size(0) == position.size(0), "x has another number of tokens than the order");
        const bool follow = at::GradMode::is_enabled() && wants_grad(x);
        if (follow) code_of(x);
        else
            require(!x.is_complex() && (x.element_size() == 1 || x.element_size() == 2 || x.element_size() == 4),
                    "Only elements of 1, 2 and 4 bytes are supported");
        ready(x);
        Tensor out;
        {
            WithoutInterpreter others_run;
            if (follow) out = Dispatch::apply(x, position, offsets);
            else {
                at::NoGradGuard guard;
                out = dispatch_run(x, Places(position, offsets));
            }
        }
        return wrap(out);
    });
}

// combine(rows, position, offsets, weights) -> the tokens' sums
PyObject *combine(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return call("combine", n, 4, [&]() -> PyObject * {
        const Tensor rows = tensor_arg(args[0], NO_TENSOR), position = tensor_arg(args[1], NO_TENSOR), offsets = tensor_arg(args[2], NO_TENSOR);
        const Maybe weights = maybe_tensor(args[3], NO_TENSOR);
        require(rows.dim() == 2, "Only 2D tensors are supported");
        code_of(rows);
        check_places(position, offsets, rows);
        require(rows.size(0) == position.numel(), "There are not as many rows as choices");
        if (weights) {
            require(weights->numel() == position.numel() && weights->dim() <= 2 && weights->dim() >= 1 && weights->size(0) == position.size(0),
                    "The weights are one number for every choice");
            require(weights->scalar_type() == rows.scalar_type() || weights->scalar_type() == at::kFloat, "The weights have the type of the rows or are fp32");
            require(weights->device() == rows.device(), "All inputs must be on the same device");
        }
        const bool follow = at::GradMode::is_enabled() && (wants_grad(rows) || wants_grad(weights));
        ready(rows);
        Tensor out;
        {
            WithoutInterpreter others_run;
            if (follow) out = Combine::apply(rows, weights, position, offsets);
            else {
                at::NoGradGuard guard;
                out = combine_run(rows, Places(position, offsets), or_none(weights));
            }
        }
        return wrap(out);
    });
}

// bind(name, address): a function of libtftq.so; its name without tftq_
PyObject *bind(PyObject *, PyObject *args)
{
    const char *name = nullptr;
    unsigned long long at = 0;
    if (!PyArg_ParseTuple(args, "sK", &name, &at)) return nullptr;
    bool found = false;
    auto to = [&](const char *which, auto &function) {
        if (strcmp(name, which) != 0) return;
        function = reinterpret_cast<typename std::remove_reference<decltype(function)>::type>(static_cast<uintptr_t>(at));
        found = true;
    };
#define TO(f) to(#f, lib.f)
    TO(strerror);
    TO(check_device);
    TO(rms_norm);
    TO(rms_norm_backward_workspace);
    TO(rms_norm_backward);
    TO(dropout);
    TO(embedding);
    TO(embedding_backward_workspace);
    TO(embedding_backward);
    TO(expert_sort_workspace);
    TO(expert_sort);
    TO(dispatch);
    TO(combine);
    TO(combine_backward);
    TO(fp8_rows_dequantize);
#undef TO
    if (!found) {
        PyErr_Format(PyExc_ValueError, "no function %s", name);
        return nullptr;
    }
    Py_RETURN_NONE;
}

PyCFunction fast(PyObject *(*f)(PyObject *, PyObject *const *, Py_ssize_t)) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, "bind(name, address): a function of libtftq.so"},
    {"rms_norm", fast(rms_norm), METH_FASTCALL, "rms_norm(x, weight, residual, eps, fp8)"},
    {"fp8_rows", fast(fp8_rows), METH_FASTCALL, "fp8_rows(codes, scales, type)"},
    {"dropout", fast(dropout), METH_FASTCALL, "dropout(x, p, seed, offset, residual)"},
    {"embedding", fast(embedding), METH_FASTCALL, "embedding(ids, table, scale, skip)"},
    {"sort_by_expert", fast(sort_by_expert), METH_FASTCALL, "sort_by_expert(chosen, experts)"},
    {"dispatch", fast(dispatch), METH_FASTCALL, "dispatch(x, position, offsets)"},
    {"combine", fast(combine), METH_FASTCALL, "combine(rows, position, offsets, weights)"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rows", "Calls of the row operators", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

#ifndef TFTQ_ROWS_ID
#define TFTQ_ROWS_ID "unknown"
#endif

PyMODINIT_FUNC PyInit__rows(void)
{
    PyObject *m = PyModule_Create(&module);
    // identifies the source the module was built from (a hash that the build passes in)
    if (m && PyModule_AddStringConstant(m, "BUILD_ID", TFTQ_ROWS_ID) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
