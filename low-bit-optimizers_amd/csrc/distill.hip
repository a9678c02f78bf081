// Distillation from a teacher's top logits with the label's cross entropy: loss and gradient of each row of logits.
//
// With T the temperature, z = (x - max x) / T, s = sum exp z, and p the teacher's softmax over the K entries (t_k, i_k) of the row:
//     kd = T^2 sum_k p_k (log p_k - z[i_k] + log s)                 d kd / dx_v = T (exp(z_v) / s - sum_{k: i_k = v} p_k)
//     ce = log s1 - (x[y] - max x), s1 = sum exp(x - max x)         d ce / dx_v = exp(x_v - max x) / s1 - [v = y]
// so a row needs its largest value and one or two sums (one where T = 1), and each value of the gradient is exponentials times
// constants of the row, less what the few listed entries and the label take off.
//
// One workgroup takes a row and holds it in registers, as it came, 16 bytes a run: a row of logits is read once and a row of the gradient written
// once, with the maximum, the sums and the gradient made from what is held.  The first wave takes the teacher's entries meanwhile.  Rows too long to
// hold are read twice.
#include "losses.hpp"

namespace lpmm {
namespace {

struct Distill {
    lpmm_distill_call c;
    const float *grad_loss;  // the gradient call: not NULL
    int64_t grad_loss_stride;
    int made;        // the gradient call: grad holds what belongs to grad_loss == 1
    int with_label;  // labels that have a weight
    float each;      // weight of a row in the reduced loss where no `share` says it
};

// Exponentials of a row: exp((x - max) / T), and exp(x - max) for the label's term.
enum Kind {
    kOne,     // one of them, or T = 1: the same
    kSquare,  // T = 2: the second is the square of the first
    kTwo,
};

// How exponents of 2 are formed.  16-bit types: fma(x, c, -M) with M = max c, one instruction; what rounding M leaves is the same factor
// in every exponential of the row and in its sum, so long as it is small, which |M| below 2^20 ensures (2^-4 at most in the exponent).
// Rows beyond and float32 logits subtract first: a row of the type's lowest values only has a uniform softmax and no overflow.
constexpr float kLargeShift = 1048576.0f;

struct Shift {
    float max, c, m;  // m: max c, or NaN where the difference comes first
    template <typename T>
    static __device__ __forceinline__ Shift of(float max, float c)
    {
        const float m = max * c;
        return {max, c, T::kRun == 8 && fabsf(m) < kLargeShift ? m : NAN};
    }
    __device__ __forceinline__ bool one_step() const { return m == m; }
    // the exponent, for a few values of a row
    __device__ __forceinline__ float of_value(float x) const { return one_step() ? fmaf(x, c, -m) : (x - max) * c; }
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

// The largest of three; without the two instructions that the library's maximum spends on quieting NaN, which are ignored here too.
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

template <typename T>
__device__ __forceinline__ float run_max(u32x4 r, float m)
{
    float v[T::kRun];
    T::unpack(r, v);
#pragma unroll
    for (int j = 0; j < T::kRun; j += 2)
        m = max3(m, v[j], v[j + 1]);
    return m;
}

// Adds the run's exponentials.
template <typename T, int KIND, bool ONE_STEP>
__device__ __forceinline__ void run_sums(u32x4 r, const Shift &t, const Shift &one, float &s, float &s1)
{
    float v[T::kRun];
    T::unpack(r, v);
#pragma unroll
    for (int j = 0; j < T::kRun; ++j) {
        const float e = exp2_fast(ONE_STEP ? fmaf(v[j], t.c, -t.m) : (v[j] - t.max) * t.c);
        s += e;
        if (KIND == kSquare)
            s1 = fmaf(e, e, s1);
        if (KIND == kTwo)
            s1 += exp2_fast(ONE_STEP ? fmaf(v[j], one.c, -one.m) : (v[j] - one.max) * one.c);
    }
}

struct Factors {
    float q, q1;  // of the exponentials in the gradient
};

template <int KIND>
__device__ __forceinline__ float smooth(float e, float e1, const Factors &f)
{
    if (KIND == kOne)
        return e * f.q;
    if (KIND == kSquare)
        return e * fmaf(e, f.q1, f.q);
    return fmaf(e1, f.q1, e * f.q);
}

template <typename T, int KIND, bool ONE_STEP>
__device__ __forceinline__ u32x4 run_grad(u32x4 r, const Shift &t, const Shift &one, const Factors &f)
{
    float v[T::kRun];
    T::unpack(r, v);
#pragma unroll
    for (int j = 0; j < T::kRun; ++j) {
        const float e = exp2_fast(ONE_STEP ? fmaf(v[j], t.c, -t.m) : (v[j] - t.max) * t.c);
        const float e1 = KIND == kTwo ? exp2_fast(ONE_STEP ? fmaf(v[j], one.c, -one.m) : (v[j] - one.max) * one.c) : 0.0f;
        v[j] = smooth<KIND>(e, e1, f);
    }
    return T::pack(v);
}

// What the first wave finds out about a row's entries, in shared memory.
struct Teacher {
    float log_total, top;
    int some, bad;
};

// The entries' ids (-1: empty) and probabilities; `value` keeps t.  One wave, which alone uses `value` again.
__device__ __forceinline__ void read_teacher(const Distill &a, int64_t row, int64_t label, int *ids, float *part, float *value, Teacher *out)
{
    const lpmm_distill_call &c = a.c;
    const int lane = threadIdx.x, topk = (int)c.topk;
    bool wrong = c.labels && (label < 0 || label >= c.vocab);
    float top = -INFINITY;
    for (int k = lane; k < topk; k += kWave) {
        const int64_t at = row * topk + k, id = id_of(c, at);
        const float t = id < 0 ? -INFINITY : teacher_of(c, at);
        wrong |= id >= c.vocab || !(t < INFINITY);
        top = fmaxf(top, t);
        ids[k] = id < 0 || id >= c.vocab ? -1 : (int)id;
        value[k] = t;
    }
    top = wave_max(top);
    const bool some = top > -INFINITY;
    const float inv_t = 1.0f / c.temperature;
    float total = 0.0f;
    for (int k = lane; k < topk; k += kWave) {
        const float p = some && ids[k] >= 0 ? expf((value[k] - top) * inv_t) : 0.0f;
        part[k] = p;
        total += p;
    }
    total = wave_sum(total);
    const float inv = some ? 1.0f / total : 0.0f;
    for (int k = lane; k < topk; k += kWave)
        part[k] *= inv;
    const int round = (topk + 1 + 3) & ~3;  // the label's place, and what fills the last four
    if (lane < round - topk) {
        ids[topk + lane] = lane == 0 && a.with_label && label >= 0 && label < c.vocab ? (int)label : -1;
        part[topk + lane] = 0.0f;
    }
    const bool bad = __any(wrong);
    if (lane == 0)
        *out = {some ? logf(total) : 0.0f, top, some, bad};
}

// The row's loss; one wave, once the sums are known.
template <typename T>
__device__ __forceinline__ float row_loss(const Distill &a, const typename T::Raw *x, const int *ids, const float *part, const float *value,
                                          const Teacher &teacher, const Shift &t, const Shift &one, float sum, float sum1, int64_t label)
{
    const lpmm_distill_call &c = a.c;
    const float inv_t = 1.0f / c.temperature, log_s = logf(sum);
    float kd = 0.0f;
    for (int k = threadIdx.x; k < (int)c.topk; k += kWave) {
        const float p = part[k];
        if (p > 0.0f)
            kd += p * (((value[k] - teacher.top) * inv_t - teacher.log_total) - (t.of_value(T::get(x[ids[k]])) * kLn2 - log_s));
    }
    kd = wave_sum(kd);
    float loss = c.teacher_weight * (c.temperature * c.temperature) * kd;
    if (a.with_label && !teacher.bad)
        loss += c.label_weight * (logf(sum1) - one.of_value(T::get(x[label])) * kLn2);
    return teacher.bad ? NAN : loss;
}

// The listed entries and the label, with what they take off: one thread for each id, which sums the parts of the entries with that id in
// their order.  The rest of the row has been written, by other threads of the workgroup.
template <typename T, int KIND>
__device__ __forceinline__ void write_entries(const Distill &a, const typename T::Raw *x, typename T::Raw *grad, const int *ids, const float *part,
                                              const Shift &t, const Shift &one, const Factors &f, float kt, float kl, int threads)
{
    const int topk = (int)a.c.topk;
    for (int k = threadIdx.x; k <= topk; k += threads) {
        const int id = ids[k];
        if (id < 0)
            continue;
        int same = 0;
        for (int j = 0; j <= topk; j += 4) {
            const int4 four = *reinterpret_cast<const int4 *>(ids + j);
            same += (four.x == id) + (four.y == id) + (four.z == id) + (four.w == id);
        }
        float off = k < topk ? kt * part[k] : kl;
        if (same > 1) {
            bool first = true;
            for (int j = 0; j < k && first; ++j)
                first = ids[j] != id;
            if (!first)
                continue;
            for (int j = k + 1; j <= topk; ++j)
                if (ids[j] == id)
                    off += j < topk ? kt * part[j] : kl;
        }
        const float v = T::get(x[id]), e = exp2_fast(t.of_value(v));
        const float e1 = KIND == kTwo ? exp2_fast(one.of_value(v)) : 0.0f;
        grad[id] = T::put(smooth<KIND>(e, e1, f) - off);
    }
}

template <typename T>
__device__ __forceinline__ void write_zeros(typename T::Raw *grad, uint32_t vocab, int threads)
{
    const uint32_t whole = vocab - vocab % T::kRun;
    for (uint32_t at = threadIdx.x * T::kRun; at < whole; at += threads * T::kRun)
        store_run<T>(grad + at, u32x4{});
    if (threadIdx.x < vocab - whole)
        grad[whole + threadIdx.x] = T::put(0.0f);
}

// RUNS runs of 16 bytes in each thread; RUNS = 0: rows of any length, read twice.
template <typename T, int KIND, int THREADS, int RUNS>
__global__ __launch_bounds__(THREADS) void distill_kernel(Distill a)
{
    using Raw = typename T::Raw;
    constexpr uint32_t kStride = THREADS * T::kRun;
    constexpr int kWaves = THREADS / kWave;
    __shared__ float room[3][kWaves];
    __shared__ Teacher teacher;
    extern __shared__ __attribute__((aligned(16))) int entries[];
    const lpmm_distill_call &c = a.c;
    const bool again = a.grad_loss != nullptr;  // the gradient call: the sums are known
    if (again && a.made && a.grad_loss[0] == 1.0f)
        return;
    const int places = ((int)c.topk + 1 + 3) & ~3, wave = threadIdx.x / kWave;
    int *ids = entries;
    float *part = reinterpret_cast<float *>(entries + places), *value = part + places;
    const uint32_t tid = threadIdx.x, vocab = (uint32_t)c.vocab;  // below 2^31: a position and a stride past it fit 32 bits
    const uint32_t whole = vocab - vocab % T::kRun;
    const int64_t row = blockIdx.x;
    Raw *grad = c.grad ? static_cast<Raw *>(c.grad) + row * (int64_t)vocab : nullptr;
    const int64_t label = c.labels ? c.labels[row] : -1;
    const Raw *x = row_of<T>(c, row);
    auto no_part = [&] {
        if (!again && tid == 0)
            c.row_loss[row] = 0.0f;
        if (grad)
            write_zeros<T>(grad, vocab, THREADS);
    };
    if (c.labels && label == c.ignore_index)
        return no_part();

    u32x4 held[RUNS > 0 ? RUNS : 1];
    float last = -INFINITY;  // of the values past the last whole run, one to a thread
    if (tid < vocab - whole)
        last = T::get(x[whole + tid]);
    if constexpr (RUNS > 0) {
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const uint32_t at = i * kStride + tid * T::kRun;
            held[i] = u32x4{T::kNoValue, T::kNoValue, T::kNoValue, T::kNoValue};
            if (at < whole)
                held[i] = load_run<T>(x + at);
        }
    }
    // each held run that a thread of the workgroup has
    auto runs = [&](auto &&body) {
        if constexpr (RUNS > 0) {
#pragma unroll
            for (int i = 0; i < RUNS; ++i)
                if (i * kStride < whole)
                    body(i, i * kStride + tid * T::kRun, held[i]);
        } else {
            for (uint32_t at = tid * T::kRun; at < whole; at += kStride)
                body(0, at, load_run<T>(x + at));
        }
    };
    if (wave == 0)
        read_teacher(a, row, label, ids, part, value, &teacher);

    float max, sum, sum1;
    if (again) {
        const float4 kept = reinterpret_cast<const float4 *>(c.row_stats)[row];
        max = kept.x, sum = kept.y, sum1 = kept.z;
        __syncthreads();
    } else {
        float m = last;
        runs([&](int, uint32_t, u32x4 r) { m = run_max<T>(r, m); });
        m = wave_max(m);
        if (tid % kWave == 0)
            room[0][wave] = m;
        __syncthreads();
        max = room[0][0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w)
            max = fmaxf(max, room[0][w]);
    }
    if (!teacher.some && !a.with_label && !teacher.bad)  // neither term has anything to say of the row
        return no_part();
    if (max == -INFINITY)
        max = NAN;  // no softmax: everything becomes NaN, as 0 / 0 does
    Shift one = Shift::of<T>(max, kLog2e), t = KIND == kOne && c.temperature == 1.0f ? one : Shift::of<T>(max, kLog2e / c.temperature);
    const bool one_step = t.one_step() && one.one_step();
    if (!one_step)
        t.m = one.m = NAN;
    if (!again) {
        float s = exp2_fast(t.of_value(last)), s1 = KIND == kSquare ? s * s : KIND == kTwo ? exp2_fast(one.of_value(last)) : 0.0f;
        if (one_step)
            runs([&](int, uint32_t, u32x4 r) { run_sums<T, KIND, true>(r, t, one, s, s1); });
        else
            runs([&](int, uint32_t, u32x4 r) { run_sums<T, KIND, false>(r, t, one, s, s1); });
        s = wave_sum(s);
        if (KIND != kOne)
            s1 = wave_sum(s1);
        if (tid % kWave == 0)
            room[1][wave] = s, room[2][wave] = s1;
        __syncthreads();
        sum = room[1][0], sum1 = room[2][0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w)
            sum += room[1][w], sum1 += room[2][w];
        if (KIND == kOne)
            sum1 = sum;
        if (wave == 0) {
            const float loss = row_loss<T>(a, x, ids, part, value, teacher, t, one, sum, sum1, label);
            if (tid == 0) {
                c.row_loss[row] = loss;
                if (c.row_stats)
                    reinterpret_cast<float4 *>(c.row_stats)[row] = make_float4(max, sum, sum1, 0.0f);
            }
        }
    }
    if (!grad)
        return;
    const float each = c.reduction == LPMM_REDUCE_MEAN && c.labels ? c.share[0] : a.each;
    const float scale = each * (again ? a.grad_loss[row * a.grad_loss_stride] : 1.0f);
    const float kt = teacher.bad ? NAN : teacher.some ? scale * c.teacher_weight * c.temperature : 0.0f;
    const float kl = a.with_label ? scale * c.label_weight : 0.0f;
    const Factors f = {(KIND == kOne ? kt + kl : kt) / sum, KIND == kOne ? 0.0f : kl / sum1};
    auto write = [&](auto steps) {
        runs([&](int, uint32_t at, u32x4 r) {
            const u32x4 g = run_grad<T, KIND, decltype(steps)::value>(r, t, one, f);
            if (at < whole)
                store_run<T>(grad + at, g);
        });
    };
    if (one_step)
        write(std::true_type());
    else
        write(std::false_type());
    if (tid < vocab - whole) {
        const float e = exp2_fast(t.of_value(last)), e1 = KIND == kTwo ? exp2_fast(one.of_value(last)) : 0.0f;
        grad[whole + tid] = T::put(smooth<KIND>(e, e1, f));
    }
    // The entries' places are written again: the wait lets the stores above be done first.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    write_entries<T, KIND>(a, x, grad, ids, part, t, one, f, kt, kl, THREADS);
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
        c.inner_stride < 0 || c.rows > INT32_MAX || c.rows > INT64_MAX / c.vocab / 8)
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

template <typename T, int KIND, int THREADS, int RUNS>
void launch(const Distill &a, hipStream_t stream)
{
    const int places = ((int)a.c.topk + 1 + 3) & ~3;
    distill_kernel<T, KIND, THREADS, RUNS><<<(unsigned)a.c.rows, THREADS, places * 12, stream>>>(a);
}

template <typename T, int KIND>
void launch_kind(const Distill &a, hipStream_t stream)
{
    const int64_t runs = a.c.vocab / T::kRun;  // whole ones
    if (a.c.rows < 256) {
        if (runs <= 1024 * 4)
            return launch<T, KIND, 1024, 4>(a, stream);
    } else {
        if (runs <= 256 * 4)
            return launch<T, KIND, 256, 4>(a, stream);
        if (runs <= 256 * 16)
            return launch<T, KIND, 256, 16>(a, stream);
        if (runs <= 512 * 16)
            return launch<T, KIND, 512, 16>(a, stream);
    }
    if (runs <= 1024 * 16)
        return launch<T, KIND, 1024, 16>(a, stream);
    launch<T, KIND, 1024, 0>(a, stream);
}

template <typename T>
void launch_type(const Distill &a, hipStream_t stream)
{
    if (!a.with_label || a.c.temperature == 1.0f)
        return launch_kind<T, kOne>(a, stream);
    if constexpr (T::kRun == 8)
        if (a.c.temperature == 2.0f)
            return launch_kind<T, kSquare>(a, stream);
    launch_kind<T, kTwo>(a, stream);
}

void launch_rows(const Distill &a, hipStream_t stream)
{
    switch (a.c.type) {
    case LPMM_TYPE_F32: return launch_type<F32>(a, stream);
    case LPMM_TYPE_F16: return launch_type<F16>(a, stream);
    default: return launch_type<BF16>(a, stream);
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
    if (c.rows > 0)
        launch_rows(a, s);
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
    launch_rows(a, static_cast<hipStream_t>(stream));
    return launch_status();
}
