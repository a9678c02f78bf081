// The host side of the training-loss terms: argument checks, outputs, the records of include/lpmm_hip.h, and the nodes of torch's autograd
// graph, whose backward passes run on the engine's own thread.
//
// In Python the same work bounded every call on less than some ten million logits: a node written in Python takes the interpreter's lock
// on the engine's thread while the calling thread waits in the engine, and the loss and gradient of 16 rows of 8192
// logits took 120 us of host time for 25 us of kernels (forward 26, of it checks and records 10; the engine itself 30).  From here it takes 57-68,
// where torch.autograd.grad of a sum of as many values takes 42-47.
//
// Errors are Python's: RuntimeError for tensors that do not fit, ValueError for values.  What needs no GPU is checked first.
#include <ATen/SavedTensorHooks.h>
#include <ATen/TracerMode.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <limits>
#include <memory>
#include <mutex>
#include <optional>
#include <sstream>
#include <string>
#include <utility>
#include <vector>

#include "lpmm_hip.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

template <typename... Parts>
std::string said(const Parts &...parts)
{
    std::ostringstream text;
    (text << ... << parts);
    return text.str();
}

#define REQUIRE(condition, ...)                           \
    do {                                                  \
        if (!(condition))                                 \
            throw std::runtime_error(said(__VA_ARGS__));  \
    } while (0)

#define REQUIRE_VALUE(condition, ...)                     \
    do {                                                  \
        if (!(condition))                                 \
            throw py::value_error(said(__VA_ARGS__));     \
    } while (0)

int type_of(const Tensor &t, const char *name)
{
    switch (t.scalar_type()) {
    case at::kFloat: return LPMM_TYPE_F32;
    case at::kHalf: return LPMM_TYPE_F16;
    case at::kBFloat16: return LPMM_TYPE_BF16;
    default: throw std::runtime_error(said("The type of ", name, " is not float32, float16 or bfloat16: ", t.scalar_type()));
    }
}

int id_bits(const Tensor &t, const char *name)
{
    REQUIRE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64, got ", t.scalar_type());
    return t.scalar_type() == at::kInt ? 32 : 64;
}

float finite(double value, const char *name)
{
    REQUIRE_VALUE(std::isfinite((float)value), name, " must be finite, got ", value);
    return (float)value;
}

// Whether two tensors have the same sizes but for `but` dimensions at the end of each.
bool same_lead(const Tensor &a, const Tensor &b, int64_t but_a, int64_t but_b)
{
    return a.sizes().slice(0, a.dim() - but_a) == b.sizes().slice(0, b.dim() - but_b);
}

// The kernels get addresses, and what the graph sees of a call is the node for its backward pass.  Who records operators (torch.jit.trace, make_fx,
// fake tensors) would record the allocation of the outputs alone and give back memory that nothing wrote, and a forward-mode derivative would
// come out as zero: both are refused, for the loss and for its backward pass.  Modes that only look on are let through.
void require_seen(const Tensor &t, const char *name, const char *what)
{
    using c10::impl::TorchDispatchModeKey;
    bool recorded = at::tracer::impl::is_dispatch_enabled() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
    for (const TorchDispatchModeKey key : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
        recorded = recorded || c10::impl::TorchDispatchModeTLS::get_mode(key).has_value();
    REQUIRE(!recorded, what, " cannot be traced: a tracer or fake tensors are active, which do not see its kernels");
    REQUIRE(!t._fw_grad(0).defined(), name, " has a forward-mode gradient, and ", what, " has no forward-mode derivative");
}

// Whether there is an address to hand to the kernels.  Tensors that wrap others have NULL, which for labels and masks would read as none.
bool has_memory(const Tensor &t) { return t.numel() == 0 || t.const_data_ptr(); }

struct Named {
    const Tensor *tensor;
    const char *name;
};

c10::Device device_of(std::initializer_list<Named> tensors)
{
    std::optional<c10::Device> device;
    for (const Named &t : tensors) {
        if (!t.tensor)
            continue;
        REQUIRE(t.tensor->is_cuda(), t.name, " must be a CUDA tensor!");
        if (!device)
            device = t.tensor->device();
        REQUIRE(t.tensor->device() == *device, "all tensors must be on the same device, got ", *device, " and ", t.tensor->device());
        REQUIRE(has_memory(*t.tensor), t.name, " has no memory of its own: a tensor that wraps others is not taken");
    }
    return *device;
}

const Tensor *some(const MaybeTensor &t) { return t ? &*t : nullptr; }
Tensor or_none(const MaybeTensor &t) { return t ? *t : Tensor(); }

// Constants of the loss: contiguous, without a graph of their own, and with the signs they stand for (torch negates some views, such as
// the imaginary part of a conjugate, only where they are read).
Tensor constant(const Tensor &t)
{
    if (!t.defined())
        return t;
    const Tensor plain = (t.requires_grad() ? t.detach() : t).resolve_neg();
    return plain.is_contiguous() ? plain : plain.contiguous();
}

template <typename V>
V *data(const Tensor &t)
{
    return t.defined() ? static_cast<V *>(t.data_ptr()) : nullptr;
}

void check(int status, const char *what)
{
    REQUIRE(status == LPMM_OK, "lpmm: ", what, " failed: ", lpmm_status_string(status), " (status ", status, ")");
}

void *stream_of(c10::Device device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

// Which recording into a graph a stream is in; 0: none.  The default stream is never in one, and is not asked, which is an error during another's.
unsigned long long recording(void *stream)
{
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (!stream || hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &id) != hipSuccess || status == hipStreamCaptureStatusNone)
        return 0;
    return id;
}

// Row n of the flattened leading dimensions starts at (n / inner) * outer_stride + (n % inner) * inner_stride.
struct Rows {
    int64_t inner, outer_stride, inner_stride;
};

// Two levels of rows fit views such as logits[:, :-1]; nothing for what has to be copied first.
std::optional<Rows> row_strides(const Tensor &t)
{
    const int64_t dims = t.dim();
    if (t.numel() == 0)
        return Rows{1, 0, 0};
    if (t.stride(dims - 1) != 1 && t.size(dims - 1) != 1)
        return std::nullopt;
    int64_t length[2] = {1, 1}, stride[2] = {0, 0};
    int levels = 0;
    for (int64_t d = 0; d + 1 < dims; ++d) {
        const int64_t n = t.size(d), s = t.stride(d);
        if (n == 1)
            continue;
        if (levels > 0 && stride[levels - 1] == n * s) {  // adjacent dimensions that are one
            length[levels - 1] *= n;
            stride[levels - 1] = s;
        } else if (levels == 2) {
            return std::nullopt;
        } else {
            length[levels] = n;
            stride[levels++] = s;
        }
    }
    return levels == 2 ? Rows{length[1], stride[0], stride[1]} : Rows{length[0], 0, stride[0]};
}

// The gradient of a gradient is not computed: whoever asks for it meets an error on the way back to `input`, not a constant.
Tensor once(Tensor grad, const torch::autograd::Edge &input, const char *name)
{
    if (c10::GradMode::is_enabled()) {
        auto error = std::shared_ptr<torch::autograd::Error>(
            new torch::autograd::Error(said("trying to differentiate twice a function that can be differentiated once: ", name), {input}),
            torch::autograd::deleteNode);
        torch::autograd::set_history(grad, error);
    }
    return grad;
}

// What a backward pass reads again.  Hooks on saved tensors (checkpointing, offloading) may give back another tensor of the same values, so its
// address is taken where it comes back; what does not fit the call's records is refused.
struct Kept {
    SavedVariable variable;
    std::vector<int64_t> shape;
    at::ScalarType type = at::kFloat;
    bool some = false;

    void keep(const Tensor &t)
    {
        if (!t.defined())
            return;
        some = true;
        shape = t.sizes().vec();
        type = t.scalar_type();
        variable = SavedVariable(t, false);
    }
    // also checks that nothing was written over since the loss was computed
    Tensor back(c10::Device device) const
    {
        Tensor t = variable.unpack();
        if (t.defined())
            t = t.resolve_neg();
        REQUIRE(!some || (t.defined() && t.device() == device && t.scalar_type() == type && t.sizes() == shape && has_memory(t)), "a saved tensor of ", type, ", shape ",
                at::IntArrayRef(shape), " on ", device, " came back from its hooks as another");
        return t;
    }
    Tensor back_contiguous(c10::Device device) const
    {
        const Tensor t = back(device);
        return t.defined() ? t.contiguous() : t;
    }
};

bool saved_tensors_have_hooks() { return at::SavedTensorDefaultHooks::get_hooks().has_value(); }

// ---------------------------------------------------------------------------------------
// distillation
// ---------------------------------------------------------------------------------------

// The gradient of a reduced loss is written by the pass that computes the loss, while the row's logits are at hand, for the gradient 1
// that loss.backward() starts from; a backward pass that arrives with another value writes it again from the logits.
// float16 training scales its loss as a rule, so there, and for the losses of single rows, only the backward pass writes it; nor is it made
// where hooks keep saved tensors elsewhere, to have the memory.
struct DistillLossBackward : public Node {
    lpmm_distill_call call;  // its addresses are set by `apply`
    c10::Device device = c10::kCPU;
    std::vector<int64_t> shape;
    at::TensorOptions options;
    Kept rows, teacher, ids, labels, scale, map, work;
    Tensor grad;  // made along with the loss
    unsigned long long recorded = 0;  // the recording that made it

    variable_list apply(variable_list &&grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined())
            return {Tensor()};
        require_seen(grads[0], "the gradient of the loss", "distill_loss");
        Tensor grad_loss = grads[0].resolve_neg();
        const c10::DeviceGuard guard(device);
        Tensor x = rows.back(device);
        std::optional<Rows> strides = row_strides(x);
        if (!strides) {
            x = x.contiguous();
            strides = row_strides(x);
        }
        const Tensor held[] = {teacher.back_contiguous(device), ids.back_contiguous(device), labels.back_contiguous(device),
                               scale.back_contiguous(device), map.back_contiguous(device), work.back_contiguous(device)};
        Tensor out = std::move(grad);  // handed out once: a second pass over the graph gets a gradient of its own
        grad.reset();
        if (out.defined() && recording(stream_of(device)) != recorded)
            out.reset();  // every replay has to write it, to memory that is the recording's own
        const bool made = out.defined();
        if (!made)
            out = at::empty(shape, options);
        int64_t stride = 0;
        if (call.reduction == LPMM_REDUCE_NONE) {
            for (const int64_t s : grad_loss.strides())
                stride |= s;
            if (stride) {
                grad_loss = grad_loss.contiguous();
                stride = 1;
            }
        }
        lpmm_distill_call c = call;
        c.logits = x.data_ptr();
        c.inner = strides->inner;
        c.outer_stride = strides->outer_stride;
        c.inner_stride = strides->inner_stride;
        c.teacher = data<void>(held[0]);
        c.ids = data<void>(held[1]);
        c.labels = data<int64_t>(held[2]);
        c.teacher_scale = data<float>(held[3]);
        c.teacher_map = data<float>(held[4]);
        c.row_stats = data<float>(held[5]);
        c.share = c.row_stats + 4 * c.rows;
        c.row_loss = c.loss = nullptr;
        c.grad = out.data_ptr();
        check(lpmm_distill_loss_grad(&c, static_cast<const float *>(grad_loss.data_ptr()), stride, made, stream_of(device)), "distill_loss_grad");
        return {once(std::move(out), next_edge(0), "distill_loss")};
    }

    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Kept *v : {&rows, &teacher, &ids, &labels, &scale, &map, &work})
            v->variable.reset_data();
        grad.reset();
    }

    std::string name() const override { return "DistillLossBackward"; }
};

Tensor distill_loss(const Tensor &logits, const Tensor &teacher_logits, const Tensor &teacher_ids, double temperature, const MaybeTensor &labels,
                    double teacher_weight, double label_weight, int64_t ignore_index, int reduction, const MaybeTensor &scale,
                    const MaybeTensor &qmap, int64_t group, int64_t bits)
{
    require_seen(logits, "logits", "distill_loss");
    lpmm_distill_call c = {};
    REQUIRE_VALUE(temperature >= 1.0 / 1024 && temperature <= 1024.0, "temperature must lie within 1/1024 and 1024, got ", temperature);
    c.temperature = (float)temperature;
    c.teacher_weight = finite(teacher_weight, "teacher_weight");
    c.label_weight = finite(label_weight, "label_weight");
    REQUIRE_VALUE(labels || label_weight == 0.0, "label_weight needs labels");
    c.type = type_of(logits, "logits");
    REQUIRE(logits.dim() >= 1 && teacher_ids.dim() >= 1, "logits and teacher_ids must have at least one dimension");
    REQUIRE(same_lead(teacher_ids, logits, 1, 1), "teacher_ids of shape ", teacher_ids.sizes(), " do not belong to logits of shape ", logits.sizes());
    c.vocab = logits.size(-1);
    c.topk = teacher_ids.size(-1);
    c.rows = 1;
    for (const int64_t n : logits.sizes().slice(0, logits.dim() - 1))
        c.rows *= n;
    REQUIRE(c.vocab >= 1 && c.vocab < (int64_t)1 << 31, "logits must have 1 to 2^31 - 1 values in their last dimension, got ", c.vocab);
    REQUIRE(c.rows < (int64_t)1 << 31, "logits must have fewer than 2^31 rows, got ", c.rows);
    REQUIRE(c.topk <= LPMM_DISTILL_MOST, "at most ", LPMM_DISTILL_MOST, " teacher entries per row are supported, got ", c.topk);
    c.id_bits = id_bits(teacher_ids, "teacher_ids");
    c.teacher_group = group;
    c.teacher_bits = (int32_t)bits;
    REQUIRE(scale.has_value() == qmap.has_value(), "a stored teacher needs both max1 and qmap");
    if (scale) {
        const int64_t entries = teacher_ids.numel(), bytes = bits == 4 ? (entries + 1) / 2 : entries;
        REQUIRE(teacher_logits.scalar_type() == at::kChar && teacher_logits.dim() == 1 && teacher_logits.is_contiguous(),
                "stored teacher_logits must be the contiguous 1-D int8 tensor of vectorwise_quant");
        REQUIRE(scale->scalar_type() == at::kFloat && scale->is_contiguous() && qmap->scalar_type() == at::kFloat && qmap->is_contiguous(),
                "max1 and qmap of a stored teacher must be contiguous float32 tensors");
        REQUIRE(qmap->numel() >= (int64_t)1 << bits, bits, "-bit quantisation maps must have ", 1 << bits, " entries, got ", qmap->numel());
        REQUIRE(teacher_logits.numel() >= bytes && scale->numel() >= (entries + group - 1) / group, "stored teacher_logits hold fewer than the ", entries,
                " values that teacher_ids asks for");
        c.teacher_type = LPMM_TYPE_CODES;
    } else {
        REQUIRE(teacher_logits.sizes() == teacher_ids.sizes(), "teacher_logits of shape ", teacher_logits.sizes(),
                " do not belong to teacher_ids of shape ", teacher_ids.sizes());
        c.teacher_type = type_of(teacher_logits, "teacher_logits");
    }
    if (labels) {
        REQUIRE(labels->scalar_type() == at::kLong, "labels must be int64, got ", labels->scalar_type());
        REQUIRE(same_lead(*labels, logits, 0, 1), "labels of shape ", labels->sizes(), " do not belong to logits of shape ", logits.sizes());
    }
    const c10::Device device = device_of({{&logits, "logits"}, {&teacher_logits, "teacher_logits"}, {&teacher_ids, "teacher_ids"},
                                          {some(labels), "labels"}, {some(scale), "max1"}, {some(qmap), "qmap"}});
    const c10::DeviceGuard guard(device);
    const bool wants_grad = logits.requires_grad() && c10::GradMode::is_enabled();

    std::optional<Rows> strides = row_strides(logits);
    Tensor rows = logits;
    if (!strides || logits.is_neg()) {
        rows = logits.detach().resolve_neg().contiguous();
        strides = row_strides(rows);
    }
    c.inner = strides->inner;
    c.outer_stride = strides->outer_stride;
    c.inner_stride = strides->inner_stride;
    c.ignore_index = ignore_index;
    c.reduction = reduction;
    const Tensor teacher = constant(teacher_logits), ids = constant(teacher_ids), y = constant(or_none(labels));
    const Tensor scales = constant(or_none(scale)), map = constant(or_none(qmap));
    c.logits = rows.data_ptr();
    c.teacher = teacher.data_ptr();
    c.ids = ids.data_ptr();
    c.labels = data<int64_t>(y);
    c.teacher_scale = data<float>(scales);
    c.teacher_map = data<float>(map);

    const bool none = reduction == LPMM_REDUCE_NONE;
    const at::TensorOptions floats = at::TensorOptions().dtype(at::kFloat).device(device);
    Tensor loss = none ? at::empty(logits.sizes().slice(0, logits.dim() - 1), floats) : at::empty({}, floats);
    // rows' statistics (where a gradient may be asked for), share, rows' losses
    const int64_t stats = wants_grad ? 4 * c.rows : 0;
    const Tensor work = at::empty({stats + 1 + (none ? 0 : c.rows)}, floats);
    float *at = data<float>(work);
    c.row_stats = wants_grad ? at : nullptr;
    c.share = at + stats;
    c.row_loss = none ? data<float>(loss) : at + stats + 1;
    c.loss = none ? nullptr : data<float>(loss);
    Tensor grad;
    if (wants_grad && !none && c.type != LPMM_TYPE_F16 && !saved_tensors_have_hooks())
        grad = at::empty(logits.sizes(), logits.options());
    c.grad = data<void>(grad);
    check(lpmm_distill_loss(&c, stream_of(device)), "distill_loss");
    if (!wants_grad)
        return loss;

    auto node = std::shared_ptr<DistillLossBackward>(new DistillLossBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->call = c;
    node->device = device;
    node->shape = logits.sizes().vec();
    node->options = logits.options();
    node->rows.keep(rows);
    node->teacher.keep(teacher);
    node->ids.keep(ids);
    node->labels.keep(y);
    node->scale.keep(scales);
    node->map.keep(map);
    node->work.keep(work);
    node->recorded = grad.defined() ? recording(stream_of(device)) : 0;
    node->grad = std::move(grad);
    torch::autograd::set_history(loss, node);
    return loss;
}

// ---------------------------------------------------------------------------------------
// balance of experts
// ---------------------------------------------------------------------------------------
struct BalanceLossBackward : public Node {
    lpmm_balance_call call;  // its addresses are set by `apply`
    c10::Device device = c10::kCPU;
    std::vector<int64_t> shape;
    at::TensorOptions options;
    Kept rows, mask, factors;

    variable_list apply(variable_list &&grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined())
            return {Tensor()};
        require_seen(grads[0], "the gradient of the loss", "balance_loss");
        const c10::DeviceGuard guard(device);
        Tensor x = rows.back(device);
        if (x.stride(-1) != 1)
            x = x.contiguous();
        const Tensor seen = mask.back_contiguous(device), f = factors.back_contiguous(device);
        const Tensor grad_loss = grads[0].resolve_neg();
        Tensor out = at::empty(shape, options);
        lpmm_balance_call c = call;
        c.logits = x.data_ptr();
        c.outer_stride = x.dim() == 3 ? x.stride(0) : 0;
        c.inner_stride = x.stride(-2);
        c.mask = data<uint8_t>(seen);
        c.factors = data<float>(f);
        c.ids = c.work = nullptr;
        c.counts = nullptr;
        c.loss = nullptr;
        c.grad = out.data_ptr();
        check(lpmm_balance_loss_grad(&c, static_cast<const float *>(grad_loss.data_ptr()), stream_of(device)), "balance_loss_grad");
        return {once(std::move(out), next_edge(0), "balance_loss")};
    }

    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Kept *v : {&rows, &mask, &factors})
            v->variable.reset_data();
    }

    std::string name() const override { return "BalanceLossBackward"; }
};

std::pair<Tensor, Tensor> balance_loss(const Tensor &router_logits, const Tensor &expert_ids, const MaybeTensor &mask, double weight, double z_weight)
{
    require_seen(router_logits, "router_logits", "balance_loss");
    lpmm_balance_call c = {};
    c.weight = finite(weight, "weight");
    c.z_weight = finite(z_weight, "z_weight");
    c.type = type_of(router_logits, "router_logits");
    const int64_t dims = router_logits.dim();
    REQUIRE(dims == 2 || dims == 3, "router_logits must be (tokens, experts) or (groups, tokens, experts), got ", router_logits.sizes());
    REQUIRE(expert_ids.dim() == dims && same_lead(expert_ids, router_logits, 1, 1), "expert_ids of shape ", expert_ids.sizes(),
            " do not belong to router_logits of shape ", router_logits.sizes());
    c.id_bits = id_bits(expert_ids, "expert_ids");
    c.groups = dims == 3 ? router_logits.size(0) : 1;
    c.tokens = router_logits.size(-2);
    c.experts = router_logits.size(-1);
    c.picks = expert_ids.size(-1);
    REQUIRE(c.experts >= 1 && c.experts <= LPMM_BALANCE_MOST, "1 to ", LPMM_BALANCE_MOST, " experts are supported, got ", c.experts);
    REQUIRE(c.picks <= c.experts, c.picks, " picks of ", c.experts, " experts");
    REQUIRE(c.groups <= LPMM_BALANCE_GROUPS && c.tokens <= LPMM_BALANCE_TOKENS && c.groups * c.tokens <= LPMM_BALANCE_TOKENS, "at most ",
            LPMM_BALANCE_GROUPS, " groups and ", LPMM_BALANCE_TOKENS, " tokens in all are supported, got ", c.groups, " groups of ", c.tokens);
    REQUIRE(c.tokens * c.picks < (int64_t)1 << 31, "fewer than 2^31 picks in a group are supported, got ", c.tokens, " tokens of ", c.picks);
    if (mask)
        REQUIRE(mask->scalar_type() == at::kBool && same_lead(*mask, router_logits, 0, 1), "mask must be a bool tensor of shape ",
                router_logits.sizes().slice(0, dims - 1), ", got ", mask->scalar_type(), " of shape ", mask->sizes());
    const c10::Device device = device_of({{&router_logits, "router_logits"}, {&expert_ids, "expert_ids"}, {some(mask), "mask"}});
    const c10::DeviceGuard guard(device);
    const bool wants_grad = router_logits.requires_grad() && c10::GradMode::is_enabled();

    Tensor rows = router_logits;
    if ((rows.stride(-1) != 1 && c.experts > 1) || rows.is_neg())
        rows = rows.detach().resolve_neg().contiguous();
    c.outer_stride = dims == 3 ? rows.stride(0) : 0;
    c.inner_stride = rows.stride(-2);
    const Tensor ids = constant(expert_ids), seen = constant(or_none(mask));
    const at::TensorOptions on = at::TensorOptions().device(device);
    Tensor loss = at::empty({}, on.dtype(at::kFloat));
    const Tensor counts = dims == 3 ? at::empty({c.groups, c.experts}, on.dtype(at::kLong)) : at::empty({c.experts}, on.dtype(at::kLong));
    const Tensor factors = at::empty({c.groups * (c.experts + 2)}, on.dtype(at::kFloat));
    const Tensor work = at::empty({lpmm_balance_work_bytes(c.groups, c.tokens, c.experts)}, on.dtype(at::kByte));
    c.logits = rows.data_ptr();
    c.ids = ids.data_ptr();
    c.mask = data<uint8_t>(seen);
    c.loss = data<float>(loss);
    c.counts = data<int64_t>(counts);
    c.factors = data<float>(factors);
    c.work = work.data_ptr();
    check(lpmm_balance_loss(&c, stream_of(device)), "balance_loss");
    if (wants_grad) {
        auto node = std::shared_ptr<BalanceLossBackward>(new BalanceLossBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(router_logits));
        node->call = c;
        node->device = device;
        node->shape = router_logits.sizes().vec();
        node->options = router_logits.options();
        node->rows.keep(rows);
        node->mask.keep(seen);
        node->factors.keep(factors);
        torch::autograd::set_history(loss, node);
    }
    return {loss, counts};
}

}  // namespace

PYBIND11_MODULE(_losses, m)
{
    // wrapped: an exception raised by a hook on a saved tensor stays the Python exception that it is
    m.def("distill_loss", torch::wrap_pybind_function(&distill_loss));
    m.def("balance_loss", torch::wrap_pybind_function(&balance_loss));
    m.def("row_strides", [](const Tensor &t) -> std::optional<std::tuple<int64_t, int64_t, int64_t>> {
        const std::optional<Rows> r = row_strides(t);
        if (!r)
            return std::nullopt;
        return std::make_tuple(r->inner, r->outer_stride, r->inner_stride);
    });
    // what this module was compiled with: a library of another version would read its records wrongly
    m.attr("abi_version") = LPMM_HIP_ABI_VERSION;
    m.attr("record_bytes") = std::make_pair(sizeof(lpmm_distill_call), sizeof(lpmm_balance_call));
}
