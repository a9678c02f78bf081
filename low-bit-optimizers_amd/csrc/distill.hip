// Distillation from a teacher's top logits with the label's cross entropy: loss and gradient of each row of logits.
//
// With T the temperature, z = (x - max x) / T, s = sum exp z, and p the teacher's softmax over the K entries (t_k, i_k) of the row:
//     kd = T^2 sum_k p_k (log p_k - z[i_k] + log s)                 d kd / dx_v = T (exp(z_v) / s - sum_{k: i_k = v} p_k)
//     ce = log s1 - (x[y] - max x), s1 = sum exp(x - max x)         d ce / dx_v = exp(x_v - max x) / s1 - [v = y]
// so a row needs its largest value and one or two sums (one where T = 1), and each value of the gradient is exponentials times
// constants of the row, less what the few listed entries and the label take off.
//
// One workgroup takes a row.  Differences to the row's largest value are formed before they are scaled: a row of the type's lowest
// values only, at any temperature, has a uniform softmax and no overflow.
#include "losses.hpp"

namespace lpmm {
namespace {

constexpr int kDistillThreads = 512;
constexpr int64_t kDistillGrid = 2048;  // workgroups of a launch at most: eight for each CU

struct Distill {
    lpmm_distill_call c;
    const float *grad_loss;
    int64_t grad_loss_stride;
    int made;        // the gradient call: grad holds what belongs to grad_loss == 1
    int with_label;  // labels that have a weight
    float each;      // weight of a row in the reduced loss where no `share` says it
};

enum Mode { kLoss, kLossAndGrad, kGrad };

struct Row {
    float max, sum, sum1;
};

template <typename T>
__device__ __forceinline__ const typename T::Raw *row_of(const lpmm_distill_call &c, int64_t row)
{
    return static_cast<const typename T::Raw *>(c.logits) + (row / c.inner) * c.outer_stride + (row % c.inner) * c.inner_stride;
}

__device__ __forceinline__ int64_t id_of(const lpmm_distill_call &c, int64_t at)
{
    return c.id_bits == 64 ? static_cast<const int64_t *>(c.ids)[at] : static_cast<const int32_t *>(c.ids)[at];
}

__device__ __forceinline__ float teacher_of(const lpmm_distill_call &c, int64_t at)
{
    switch (c.teacher_type) {
    case LPMM_TYPE_F32: return static_cast<const float *>(c.teacher)[at];
    case LPMM_TYPE_F16: return F16::get(static_cast<const F16::Raw *>(c.teacher)[at]);
    case LPMM_TYPE_BF16: return BF16::get(static_cast<const BF16::Raw *>(c.teacher)[at]);
    default: break;
    }
    const uint8_t *codes = static_cast<const uint8_t *>(c.teacher);
    const uint32_t byte = c.teacher_bits == 4 ? codes[at >> 1] >> (4 * (at & 1)) : codes[at];
    return c.teacher_map[byte & ((1u << c.teacher_bits) - 1u)] * c.teacher_scale[at / c.teacher_group];
}

// exp((x - max) / T) as 2^((x - max) c); max = -infinity stands for "nothing yet"
__device__ __forceinline__ float scaled_exp(float x, float max, float c) { return exp2_fast((x - max) * c); }

// The row's largest value and sums.  Each thread keeps a running maximum of its own and rescales its sums when it grows.
template <typename T, bool TWO>
__device__ __forceinline__ Row row_sums(const typename T::Raw *x, uint32_t vocab, float c, float c1, float *room)
{
    float m = -INFINITY, s = 0.0f, s1 = 0.0f;
    const uint32_t whole = vocab - vocab % T::kRun;
    auto take = [&](const float(&v)[T::kRun], int n) {
        float top = m;
        for (int j = 0; j < n; ++j)
            top = fmaxf(top, v[j]);
        const float base = top == -INFINITY ? 0.0f : top;  // nothing but -infinity so far: every term is 0
        s *= scaled_exp(m, base, c);
        if (TWO)
            s1 *= scaled_exp(m, base, c1);
        for (int j = 0; j < n; ++j) {
            s += scaled_exp(v[j], base, c);
            if (TWO)
                s1 += scaled_exp(v[j], base, c1);
        }
        m = top;
    };
    for (uint32_t at = threadIdx.x * T::kRun; at < whole; at += kDistillThreads * T::kRun) {
        const Run<T> r = load_run<T>(x + at);
        float v[T::kRun];
#pragma unroll
        for (int j = 0; j < T::kRun; ++j)
            v[j] = T::get(r.v[j]);
        take(v, T::kRun);
    }
    if (threadIdx.x < vocab - whole) {
        float v[T::kRun] = {T::get(x[whole + threadIdx.x])};
        take(v, 1);
    }
    const float top = block_reduce<Max, kDistillThreads>(m, room);
    // a row of -infinity has no softmax: the sums become NaN, as 0 / 0 does
    const float base = top == -INFINITY ? NAN : top;
    Row r;
    r.max = base;
    r.sum = block_reduce<Sum, kDistillThreads>(s * scaled_exp(m, base, c), room);
    r.sum1 = TWO ? block_reduce<Sum, kDistillThreads>(s1 * scaled_exp(m, base, c1), room) : r.sum;
    return r;
}

template <typename T, bool TWO, int MODE>
__global__ __launch_bounds__(kDistillThreads) void distill_kernel(Distill a)
{
    using Raw = typename T::Raw;
    __shared__ float room[kDistillThreads / kWave];
    __shared__ int ids[LPMM_DISTILL_MOST + 1];
    __shared__ float part[LPMM_DISTILL_MOST + 1];  // what each entry takes off the gradient at its id
    const lpmm_distill_call &c = a.c;
    const int tid = threadIdx.x, topk = (int)c.topk;
    const uint32_t vocab = (uint32_t)c.vocab;  // below 2^31: a position and a workgroup's stride past it fit 32 bits
    if (MODE == kGrad && a.made && a.grad_loss[0] == 1.0f)
        return;
    const float inv_t = 1.0f / c.temperature, ce2 = inv_t * kLog2e, ce1 = kLog2e;
    const float each = c.reduction == LPMM_REDUCE_MEAN && c.labels ? c.share[0] : a.each;
    for (int64_t row = blockIdx.x; row < c.rows; row += gridDim.x) {
        Raw *grad = MODE == kLoss ? nullptr : static_cast<Raw *>(c.grad) + row * (int64_t)vocab;
        const int64_t label = c.labels ? c.labels[row] : -1;
        const Raw *x = row_of<T>(c, row);
        auto no_part = [&] {
            if (MODE != kGrad && tid == 0)
                c.row_loss[row] = 0.0f;
            if (MODE != kLoss)
                for (uint32_t v = tid; v < vocab; v += kDistillThreads)
                    grad[v] = T::put(0.0f);
        };
        if (c.labels && label == c.ignore_index) {
            no_part();
            continue;
        }
        // the teacher's entries: largest value, sum, probabilities
        bool wrong = c.labels && (label < 0 || label >= vocab);
        float top = -INFINITY;
        for (int k = tid; k < topk; k += kDistillThreads) {
            const int64_t at = row * topk + k, id = id_of(c, at);
            const float t = id < 0 ? -INFINITY : teacher_of(c, at);
            wrong |= id >= vocab || !(t < INFINITY);
            top = fmaxf(top, t);
            ids[k] = id < 0 || id >= vocab ? -1 : (int)id;
            part[k] = t;
        }
        top = block_reduce<Max, kDistillThreads>(top, room);
        const bool some = top > -INFINITY, bad = __syncthreads_or(wrong);
        if (!some && !a.with_label && !bad) {  // neither term has anything to say of the row
            no_part();
            continue;
        }
        Row r;
        if (MODE == kGrad) {
            const float4 kept = reinterpret_cast<const float4 *>(c.row_stats)[row];
            r = {kept.x, kept.y, kept.z};
        } else {
            r = row_sums<T, TWO>(x, vocab, ce2, ce1, room);
            if (c.row_stats && tid == 0)
                reinterpret_cast<float4 *>(c.row_stats)[row] = make_float4(r.max, r.sum, r.sum1, 0.0f);
        }
        float total = 0.0f;
        for (int k = tid; k < topk; k += kDistillThreads) {
            const float p = some && ids[k] >= 0 ? expf((part[k] - top) * inv_t) : 0.0f;
            total += p;
        }
        total = block_reduce<Sum, kDistillThreads>(total, room);
        const float log_total = logf(total), log_s = logf(r.sum);
        float kd = 0.0f;
        for (int k = tid; k < topk; k += kDistillThreads) {
            float p = 0.0f;
            if (some && ids[k] >= 0) {
                const float t = (part[k] - top) * inv_t;
                p = expf(t) / total;
                if (p > 0.0f && MODE != kGrad)
                    kd += p * ((t - log_total) - ((T::get(x[ids[k]]) - r.max) * inv_t - log_s));
            }
            part[k] = p;
        }
        if (MODE != kGrad) {
            kd = block_reduce<Sum, kDistillThreads>(kd, room);
            if (tid == 0) {
                float loss = c.teacher_weight * (c.temperature * c.temperature) * kd;
                if (a.with_label && !bad)
                    loss += c.label_weight * (logf(r.sum1) - (T::get(x[label]) - r.max));
                c.row_loss[row] = bad ? NAN : loss;
            }
        }
        if (MODE == kLoss) {
            __syncthreads();
            continue;
        }
        const float scale = each * (MODE == kGrad ? a.grad_loss[row * a.grad_loss_stride] : 1.0f);
        const float kt = bad ? NAN : some ? scale * c.teacher_weight * c.temperature : 0.0f, kl = a.with_label ? scale * c.label_weight : 0.0f;
        const float kq = (TWO ? kt : kt + kl) / r.sum, kq1 = kl / r.sum1;
        auto smooth = [&](float v) {
            float g = kq * scaled_exp(v, r.max, ce2);
            if (TWO)
                g += kq1 * scaled_exp(v, r.max, ce1);
            return g;
        };
        const uint32_t whole = vocab - vocab % T::kRun;
        for (uint32_t at = tid * T::kRun; at < whole; at += kDistillThreads * T::kRun) {
            const Run<T> in = load_run<T>(x + at);
            Run<T> out;
#pragma unroll
            for (int j = 0; j < T::kRun; ++j)
                out.v[j] = T::put(smooth(T::get(in.v[j])));
            store_run<T>(grad + at, out);
        }
        if ((uint32_t)tid < vocab - whole)
            grad[whole + tid] = T::put(smooth(T::get(x[whole + tid])));
        // The listed entries and the label are written again, with what they take off: one thread for each id, which sums the parts of
        // the entries with that id in their order.  The wait lets the stores above reach memory first.
        if (tid == 0) {
            ids[topk] = a.with_label && !bad ? (int)label : -1;
            part[topk] = kl;
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        for (int k = tid; k <= topk; k += kDistillThreads) {
            const int id = ids[k];
            bool first = id >= 0;
            for (int j = 0; j < k && first; ++j)
                first = ids[j] != id;
            if (!first)
                continue;
            float off = 0.0f;
            for (int j = k; j <= topk; ++j)
                if (ids[j] == id)
                    off += j < topk ? kt * part[j] : part[j];
            grad[id] = T::put(smooth(T::get(x[id])) - off);
        }
        __syncthreads();
    }
}

constexpr int kSumThreads = 1024;

// 1 / rows that count
__global__ __launch_bounds__(kSumThreads) void distill_share_kernel(const int64_t *labels, int64_t rows, int64_t ignore, float *share)
{
    __shared__ double room[kSumThreads / kWave];
    int64_t n = 0;
    for (int64_t i = threadIdx.x; i < rows; i += kSumThreads)
        n += labels[i] != ignore;
    const double all = block_sum_f64<kSumThreads>((double)n, room);
    if (threadIdx.x == 0)
        share[0] = all > 0.0 ? (float)(1.0 / all) : 0.0f;
}

// Sum of the rows' losses in double, in a fixed order, times `each` or *share.
__global__ __launch_bounds__(kSumThreads) void distill_sum_kernel(const float *row_loss, int64_t rows, const float *share, double each, float *loss)
{
    __shared__ double room[kSumThreads / kWave];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += kSumThreads)
        s += (double)row_loss[i];
    s = block_sum_f64<kSumThreads>(s, room);
    if (threadIdx.x == 0)
        loss[0] = (float)(s * (share ? (double)share[0] : each));
}

int check_call(const lpmm_distill_call &c)
{
    if (c.type < LPMM_TYPE_F32 || c.type > LPMM_TYPE_BF16 || c.teacher_type < LPMM_TYPE_F32 || c.teacher_type > LPMM_TYPE_CODES ||
        (c.id_bits != 32 && c.id_bits != 64) || c.reduction < LPMM_REDUCE_NONE || c.reduction > LPMM_REDUCE_MEAN)
        return LPMM_ERR_ARG;
    if (!(c.temperature >= 1.0f / 1024) || !(c.temperature <= 1024.0f) || !isfinite(c.teacher_weight) || !isfinite(c.label_weight))
        return LPMM_ERR_ARG;
    if (c.rows < 0 || c.vocab < 1 || c.vocab > INT32_MAX || c.topk < 0 || c.topk > LPMM_DISTILL_MOST || c.inner < 1 || c.outer_stride < 0 ||
        c.inner_stride < 0 || c.rows > (int64_t)1 << 40 || c.rows > INT64_MAX / c.vocab / 8)
        return LPMM_ERR_SIZE;
    if (c.reduction != LPMM_REDUCE_NONE && c.labels && c.reduction == LPMM_REDUCE_MEAN)
        LPMM_REQUIRE_PTR(c.share);
    if (c.rows == 0)
        return LPMM_OK;
    LPMM_REQUIRE_PTR(c.logits);
    LPMM_REQUIRE_ALIGN(c.logits, c.type == LPMM_TYPE_F32 ? 4 : 2);
    LPMM_REQUIRE_ALIGN(c.labels, 8);
    if (c.topk > 0) {
        LPMM_REQUIRE_PTR(c.teacher);
        LPMM_REQUIRE_PTR(c.ids);
        LPMM_REQUIRE_ALIGN(c.ids, c.id_bits / 8);
        LPMM_REQUIRE_ALIGN(c.teacher, c.teacher_type == LPMM_TYPE_F32 ? 4 : c.teacher_type <= LPMM_TYPE_BF16 ? 2 : 1);
        if (c.teacher_type == LPMM_TYPE_CODES) {
            LPMM_REQUIRE_PTR(c.teacher_scale);
            LPMM_REQUIRE_PTR(c.teacher_map);
            LPMM_REQUIRE_ALIGN(c.teacher_scale, 4);
            LPMM_REQUIRE_ALIGN(c.teacher_map, 4);
            if (c.teacher_group < 1 || c.teacher_bits < 4 || c.teacher_bits > 8)
                return LPMM_ERR_SIZE;
        }
    }
    return LPMM_OK;
}

Distill arguments(const lpmm_distill_call &c)
{
    Distill a = {};
    a.c = c;
    if (c.teacher_weight == 0.0f)
        a.c.topk = 0;  // a term without weight is not looked at
    a.with_label = c.labels && c.label_weight != 0.0f;
    a.each = c.reduction == LPMM_REDUCE_MEAN && c.rows > 0 ? (float)(1.0 / (double)c.rows) : 1.0f;
    return a;
}

template <typename T, int MODE>
void launch_type(const Distill &a, hipStream_t stream)
{
    const dim3 grid((unsigned)(a.c.rows < kDistillGrid ? a.c.rows : kDistillGrid));
    if (a.with_label && a.c.temperature != 1.0f)
        distill_kernel<T, true, MODE><<<grid, kDistillThreads, 0, stream>>>(a);
    else
        distill_kernel<T, false, MODE><<<grid, kDistillThreads, 0, stream>>>(a);
}

template <int MODE>
void launch_rows(const Distill &a, hipStream_t stream)
{
    switch (a.c.type) {
    case LPMM_TYPE_F32: return launch_type<F32, MODE>(a, stream);
    case LPMM_TYPE_F16: return launch_type<F16, MODE>(a, stream);
    default: return launch_type<BF16, MODE>(a, stream);
    }
}

}  // namespace
}  // namespace lpmm

extern "C" int lpmm_distill_loss(const lpmm_distill_call *call, void *stream)
{
    using namespace lpmm;
    LPMM_REQUIRE_PTR(call);
    const lpmm_distill_call &c = *call;
    if (const int status = check_call(c))
        return status;
    if (c.reduction == LPMM_REDUCE_NONE && c.grad)
        return LPMM_ERR_ARG;
    if (c.reduction != LPMM_REDUCE_NONE)
        LPMM_REQUIRE_PTR(c.loss);
    if (c.rows > 0)
        LPMM_REQUIRE_PTR(c.row_loss);
    LPMM_REQUIRE_ALIGN(c.row_loss, 4);
    LPMM_REQUIRE_ALIGN(c.row_stats, 16);
    LPMM_REQUIRE_ALIGN(c.grad, c.type == LPMM_TYPE_F32 ? 4 : 2);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const Distill a = arguments(c);
    const bool shared = c.reduction == LPMM_REDUCE_MEAN && c.labels;
    if (shared)
        distill_share_kernel<<<1, kSumThreads, 0, s>>>(c.labels, c.rows, c.ignore_index, c.share);
    if (c.rows > 0) {
        if (c.grad)
            launch_rows<kLossAndGrad>(a, s);
        else
            launch_rows<kLoss>(a, s);
    }
    if (c.reduction != LPMM_REDUCE_NONE)
        distill_sum_kernel<<<1, kSumThreads, 0, s>>>(c.row_loss, c.rows, shared ? c.share : nullptr,
                                                     c.reduction == LPMM_REDUCE_MEAN && c.rows > 0 ? 1.0 / (double)c.rows : 1.0, c.loss);
    return launch_status();
}

extern "C" int lpmm_distill_loss_grad(const lpmm_distill_call *call, const float *grad_loss, int64_t grad_loss_stride, int made, void *stream)
{
    using namespace lpmm;
    LPMM_REQUIRE_PTR(call);
    const lpmm_distill_call &c = *call;
    if (const int status = check_call(c))
        return status;
    if (grad_loss_stride < 0)
        return LPMM_ERR_SIZE;
    if (made && c.reduction == LPMM_REDUCE_NONE)
        return LPMM_ERR_ARG;
    if (c.rows == 0)
        return LPMM_OK;
    LPMM_REQUIRE_PTR(grad_loss);
    LPMM_REQUIRE_PTR(c.grad);
    LPMM_REQUIRE_PTR(c.row_stats);
    LPMM_REQUIRE_ALIGN(grad_loss, 4);
    LPMM_REQUIRE_ALIGN(c.row_stats, 16);
    LPMM_REQUIRE_ALIGN(c.grad, c.type == LPMM_TYPE_F32 ? 4 : 2);
    Distill a = arguments(c);
    a.grad_loss = grad_loss;
    a.grad_loss_stride = c.reduction == LPMM_REDUCE_NONE ? grad_loss_stride : 0;
    a.made = made;
    launch_rows<kGrad>(a, static_cast<hipStream_t>(stream));
    return launch_status();
}
