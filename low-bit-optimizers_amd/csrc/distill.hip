// Distillation from a teacher's top logits with the label's cross entropy: loss and gradient of each row of logits.
//
// With T the temperature, z = (x - max x) / T, s = sum exp z, and p the teacher's softmax over the K entries (t_k, i_k) of the row:
//     kd = T^2 sum_k p_k (log p_k - z[i_k] + log s)                 d kd / dx_v = T (exp(z_v) / s - sum_{k: i_k = v} p_k)
//     ce = log s1 - (x[y] - max x), s1 = sum exp(x - max x)         d ce / dx_v = exp(x_v - max x) / s1 - [v = y]
// so a row needs its largest value and one or two sums (one where T = 1), and each value of the gradient is exponentials times
// constants of the row, less what the few listed entries and the label take off.
//
// One workgroup takes a row and holds it in registers, as it came, 16 bytes a run: a row of logits is read once and a row of the gradient written
// once, with the sums and the gradient made from what is held.  Entries are asked for before the row and looked at when it has come.  Rows too
// long to hold are read twice.
//
// Bound by memory: without any exponential the kernel takes as long (8188 x 32000 bf16: 203 us with them, 206 without).  Loss and gradient of that
// batch, a tenth of its rows left out by their labels, move 1.00 GB in 181-188 us, 5.3-5.5 TB/s, where a copy of 4 GB by the library reaches 4.9;
// evaluation alone reads 6.0 TB/s.  What a row costs beside its bytes is a chain of some 7 us (label, entries, logits at the entries, two barriers,
// the last stores), hidden by the other workgroups of a compute unit; rows over 65536 16-bit values leave room for one, and move 4.7 TB/s.
//
// The gradient belongs to the loss's own pass because the row is at hand there: 4 bytes a bf16 value where a second pass moves 6.
#include "losses.hpp"

namespace lpmm {
namespace {

constexpr int64_t kLastLevel = (int64_t)256 << 20;  // bytes of the memory-side cache

// Where the weight 1 / (rows that count) of the mean with labels comes from.
enum Shared {
    kNoShare,    // not that mean
    kCounted,    // a kernel before: c.share
    kCountHere,  // few rows: every workgroup counts them, a microsecond each at once, for a launch less
};
constexpr int64_t kFewRows = 256;  // at most a workgroup's threads
constexpr int kChain = 128;  // values whose exponentials a thread adds in 32 bits
constexpr int64_t kMostRows = (int64_t)1 << 21;  // of a launch, whose threads are counted in 32 bits

struct Distill {
    lpmm_distill_call c;
    const float *grad_loss;  // the gradient call: not NULL
    int64_t grad_loss_stride;
    int64_t first;    // row of the launch's first workgroup
    int made;         // the gradient call: grad holds what belongs to grad_loss == 1
    int shared;       // enum Shared
    int with_label;   // labels that have a weight
    int group_shift;  // teacher_group = 2^group_shift, or -1
    int far;          // the logits are more than the last-level cache holds
    float each;       // weight of a row in the reduced loss where `shared` does not say it
};

// Exponentials of a row: exp((x - max) / T), and exp(x - max) for the label's term.
enum Kind {
    kOne,     // one of them, or T = 1: the same
    kSquare,  // T = 2: the second is the square of the first
    kTwo,
};

// How exponents of 2 are formed.  16-bit types: fma(x, c, -M) with M = max c, one instruction; what rounding M leaves is the same factor
// in every exponential of the row and in its sum, so long as it is small, which |M| below 2^20 ensures (2^-4 at most in the exponent).
// Rows beyond subtract first: a row of the type's lowest values only has a uniform softmax and no overflow.  So do float32 logits, whose
// kernels wait for twice the bytes and need the registers (2048 x 32000 at T = 1.5 and a label's term: 185 us, 193 in one step; bf16 rows
// of 50257 at T = 1 lose 5 % if they subtract).
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

// Of the teacher's exponentials and of the label's: both in one step or neither, and the square's exponent twice the other's.
template <typename T, int KIND>
__device__ __forceinline__ void shifts(float max, float c, Shift &t, Shift &one)
{
    t = Shift::of<T>(max, c);
    one = KIND == kTwo ? Shift::of<T>(max, kLog2e) : KIND == kSquare ? Shift{max, kLog2e, 2.0f * t.m} : t;
    if (KIND == kTwo && !(t.one_step() && one.one_step()))
        t.m = one.m = NAN;
}

// 1 / rows that count, of at most as many rows as the workgroup has threads.
__device__ __forceinline__ double share_of_few(const int64_t *labels, int64_t rows, int64_t ignore)
{
    const int n = __syncthreads_count((int64_t)threadIdx.x < rows && labels[threadIdx.x] != ignore);
    return n > 0 ? 1.0 / n : 0.0;
}

template <typename T>
__device__ __forceinline__ const typename T::Raw *row_of(const lpmm_distill_call &c, int64_t row)
{
    return static_cast<const typename T::Raw *>(c.logits) + (row / c.inner) * c.outer_stride + (row % c.inner) * c.inner_stride;
}

// One entry of the teacher, as the thread that has it keeps it.  What is loaded stays as it is stored until it is used: whoever converts
// waits, and the row's loads have to be on their way by then.
struct Entry {
    uint32_t id_low, id_high;
    uint32_t value, x;  // the teacher's value and the student's logit, as stored
    float scale;        // of a value in codes
    float t;

    __device__ __forceinline__ void load(const Distill &a, int64_t at)
    {
        const lpmm_distill_call &c = a.c;
        if (c.id_bits == 64) {
            const uint2 id = static_cast<const uint2 *>(c.ids)[at];
            id_low = id.x, id_high = id.y;
        } else {
            id_low = static_cast<const uint32_t *>(c.ids)[at];
        }
        if (c.teacher_type == LPMM_TYPE_F32) {
            value = static_cast<const uint32_t *>(c.teacher)[at];
        } else if (c.teacher_type != LPMM_TYPE_CODES) {
            value = static_cast<const uint16_t *>(c.teacher)[at];
        } else {
            value = static_cast<const uint8_t *>(c.teacher)[c.teacher_bits == 4 ? at >> 1 : at];
            scale = c.teacher_scale[a.group_shift >= 0 ? at >> a.group_shift : at / c.teacher_group];
        }
    }
    __device__ __forceinline__ int64_t id(const lpmm_distill_call &c) const
    {
        return c.id_bits == 64 ? (int64_t)((uint64_t)id_high << 32 | id_low) : (int64_t)(int32_t)id_low;
    }
    __device__ __forceinline__ float value_of(const lpmm_distill_call &c, int64_t at) const
    {
        switch (c.teacher_type) {
        case LPMM_TYPE_F32: return __uint_as_float(value);
        case LPMM_TYPE_BF16: return __uint_as_float(value << 16);
        case LPMM_TYPE_F16: return (float)__builtin_bit_cast(_Float16, (uint16_t)value);
        default: return c.teacher_map[(c.teacher_bits == 4 ? value >> (4 * (at & 1)) : value) & ((1u << c.teacher_bits) - 1u)] * scale;
        }
    }
};

// A logit as it is stored.
template <typename T>
__device__ __forceinline__ uint32_t load_bits(const typename T::Raw *p)
{
    if constexpr (T::kRun == 8)
        return *reinterpret_cast<const uint16_t *>(p);
    else
        return *reinterpret_cast<const uint32_t *>(p);
}

template <typename T>
__device__ __forceinline__ float from_bits(uint32_t bits)
{
    if constexpr (T::kRun == 8)
        return T::get(__builtin_bit_cast(typename T::Raw, (uint16_t)bits));
    else
        return __uint_as_float(bits);
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

// What an entry takes off at its id, where others may have the same id: the first of them takes off the parts of all, in their order.  ids and
// part: of the row's entries, the label last; whole fours, the rest -1.  False: another entry is the first.
__device__ __forceinline__ bool takes_off(const int *ids, const float *part, int entries, int k, float &off)
{
    const int id = ids[k];
    int same = 0;
    for (int j = 0; j < entries; j += 4) {
        const int4 four = *reinterpret_cast<const int4 *>(ids + j);
        same += (four.x == id) + (four.y == id) + (four.z == id) + (four.w == id);
    }
    off = part[k];
    if (same > 1) {
        for (int j = 0; j < k; ++j)
            if (ids[j] == id)
                return false;
        double all = off;  // up to 1025 parts, each of which may be as small as what their sum leaves of the smooth term
        for (int j = k + 1; j < entries; ++j)
            if (ids[j] == id)
                all += part[j];
        off = (float)all;
    }
    return true;
}

// A row's values in runs of 16 bytes that start at aligned addresses of the array that matters, and up to 2 (kRun - 1) single ones at its
// ends, one to a thread: thread i < head takes value i, thread kRun + i value end + i.
struct Cut {
    uint32_t head, end, vocab;  // runs: [head, end)
    template <typename T>
    static __device__ __forceinline__ Cut of(const void *aligned, uint32_t vocab)
    {
        uint32_t head = (uint32_t)(-reinterpret_cast<uintptr_t>(aligned) & 15u) / sizeof(typename T::Raw);
        head = head < vocab ? head : vocab;
        return {head, head + (vocab - head) / T::kRun * T::kRun, vocab};
    }
    // the single value of a thread, or vocab
    template <typename T>
    __device__ __forceinline__ uint32_t single() const
    {
        const uint32_t tid = threadIdx.x;
        if (tid < head)
            return tid;
        return tid >= T::kRun && tid - T::kRun < vocab - end ? end + tid - T::kRun : vocab;
    }
};

// The sums of a row as one thread, one wave or the workgroup has them: relative to `max`.
struct Sums {
    float max, sum, sum1;
};

// What exponentials relative to one maximum are worth relative to another; in one step: of the two shifts as they were rounded.
template <bool ONE_STEP>
__device__ __forceinline__ float from_to(float from, float to, float c)
{
    return ONE_STEP ? exp2_fast(from * c - to * c) : exp2_fast((from - to) * c);
}

// Sums relative to another maximum.
template <int KIND, bool ONE_STEP>
__device__ __forceinline__ void rebase(Sums &s, float max, float c)
{
    if (s.sum == 0.0f)  // nothing yet, whatever its maximum
        return;
    const float f = from_to<ONE_STEP>(s.max, max, c);
    s.sum *= f;
    if (KIND == kSquare)
        s.sum1 *= f * f;
    if (KIND == kTwo)
        s.sum1 *= from_to<ONE_STEP>(s.max, max, kLog2e);
}

// RUNS runs of 16 bytes in each thread; RUNS = 0: rows of any length, read twice.
// AGAIN: the gradient call, which knows the sums.
template <typename T, int KIND, bool AGAIN, int THREADS, int RUNS, int WAVES>
__global__ __launch_bounds__(THREADS, WAVES) void distill_kernel(Distill a)
{
    using Raw = typename T::Raw;
    constexpr uint32_t kStride = THREADS * T::kRun;
    constexpr int kWaves = THREADS / kWave;
    constexpr bool kOneStep = T::kRun == 8;
    static_assert(kWaves >= 4 && kWaves <= 16, "lanes_sum");
    struct OfWave {
        float max, sum, sum1, top, total, kd;
        int fits, wrong;
    };
    __shared__ OfWave room[kWaves];
    extern __shared__ __attribute__((aligned(16))) int entries[];
    const lpmm_distill_call &c = a.c;
    const int64_t row = a.first + blockIdx.x;
    float scale = a.each;
    if constexpr (AGAIN) {
        const float g = a.grad_loss[row * a.grad_loss_stride];
        if (a.made && g == 1.0f)
            return;
        scale *= g;
    }
    if (a.shared == kCounted)
        scale *= c.share[0];
    else if (a.shared == kCountHere)
        scale *= (float)share_of_few(c.labels, c.rows, c.ignore_index);
    const int topk = (int)c.topk, listed = topk + 1, places = (listed + 3) & ~3;
    int *ids = entries;
    float *part = reinterpret_cast<float *>(entries + places);
    const uint32_t tid = threadIdx.x, wave = tid / kWave, vocab = (uint32_t)c.vocab;  // below 2^31: a position and a stride past it fit 32 bits
    Raw *grad = c.grad ? static_cast<Raw *>(c.grad) + row * (int64_t)vocab : nullptr;
    const int64_t label = c.labels ? c.labels[row] : -1;
    const Raw *x = row_of<T>(c, row);
    const Cut cut = Cut::of<T>(grad ? grad : x, vocab);
    const uint32_t single = cut.single<T>(), first = cut.head + tid * T::kRun;
    auto no_part = [&] {
        if (!AGAIN && tid == 0)
            c.row_loss[row] = 0.0f;
        if (!grad)
            return;
        for (uint32_t at = first; at < cut.end; at += kStride)
            store_run_once<T>(grad + at, u32x4{});
        if (single < vocab)
            grad[single] = T::put(0.0f);
    };
    if (c.labels && label == c.ignore_index)
        return no_part();

    // everything that the row needs is asked for before anything is looked at
    Entry entry;  // one to a thread: topk is at most THREADS
    const bool has_entry = (int)tid < topk;
    if (has_entry)
        entry.load(a, row * topk + tid);
    const bool label_wrong = c.labels && (label < 0 || label >= c.vocab), has_label = a.with_label && !label_wrong;
    const uint32_t label_bits = load_bits<T>(x + (has_label ? label : 0)), alone_bits = load_bits<T>(x + (single < vocab ? single : 0));
    u32x4 held[RUNS > 0 ? RUNS : 1];
    if constexpr (RUNS > 0) {
        auto hold = [&](auto &&load) {
#pragma unroll
            for (int i = 0; i < RUNS; ++i) {  // past the row's end its last run, so that no load is a branch
                const uint32_t at = min(first + i * kStride, cut.end - T::kRun);
                held[i] = load(reinterpret_cast<const Raw *>(reinterpret_cast<const char *>(x) + at * (uint32_t)sizeof(Raw)));
            }
        };
        if (cut.end > cut.head) {
            // the assembler comments keep the compiler from making one set of loads of the two, without the hint
            if (a.far) {
                asm volatile("; once");
                hold([](const Raw *p) { return load_run_once<T>(p); });
                asm volatile("; once");
            } else {
                asm volatile("; again");
                hold([](const Raw *p) { return load_run<T>(p); });
                asm volatile("; again");
            }
        }
    }
    bool wrong = label_wrong;
    const bool has_entries = (int)(wave * kWave) < topk;
    int64_t id = -1;  // none
    if (has_entries) {
        if (has_entry)
            id = entry.id(c);
        wrong |= id >= c.vocab;
        if (id < 0 || id >= c.vocab)  // and so 32 bits hold it
            id = -1;
        entry.x = load_bits<T>(x + (id >= 0 ? id : 0));
    }
    // each run of the thread, from where it is held; or read again, for what is seldom done (and for rows that are not held)
    auto read_runs = [&](auto &&body) {
#pragma unroll 1
        for (uint32_t at = first; at < cut.end; at += kStride)
            body(at, load_run<T>(x + at));
    };
    auto runs = [&](auto &&body) {
        if constexpr (RUNS > 0) {
#pragma unroll
            for (int i = 0; i < RUNS; ++i)
                if (cut.head + i * kStride < cut.end) {
                    const uint32_t at = first + i * kStride;
                    asm volatile("" : "+v"(held[i]));  // unpacked anew each time: the floats of a row do not fit
                    if (cut.head + (i + 1) * kStride > cut.end && at >= cut.end)  // no branch that most runs need to look at
                        held[i] = u32x4{T::kNoValue, T::kNoValue, T::kNoValue, T::kNoValue};
                    body(at, held[i]);
                }
        } else {
            read_runs(body);
        }
    };
    // adds the exponentials of all runs.  Rows that are held are 128 additions to a thread; longer ones are read, and their chains of 32-bit
    // additions end after as many (2^14, of a row of 2^24 values that are alike, are off by 1e-4)
    auto read_sums = [&](auto one_step, const Shift &t, const Shift &one, Sums &s) {
        constexpr bool kInOne = decltype(one_step)::value;
        if constexpr (RUNS > 0) {
            read_runs([&](uint32_t, u32x4 r) { run_sums<T, KIND, kInOne>(r, t, one, s.sum, s.sum1); });
        } else {
            double sum = s.sum, sum1 = s.sum1;
            for (uint32_t at = first; at < cut.end;) {
                float near = 0.0f, near1 = 0.0f;
#pragma unroll 1
                for (int n = 0; n < kChain / T::kRun && at < cut.end; ++n, at += kStride)
                    run_sums<T, KIND, kInOne>(load_run<T>(x + at), t, one, near, near1);
                sum += (double)near;
                sum1 += (double)near1;
            }
            s.sum = (float)sum;
            s.sum1 = (float)sum1;
        }
    };
    const float alone = single < vocab ? from_bits<T>(alone_bits) : -INFINITY;
    const float ct = KIND == kOne && c.temperature == 1.0f ? kLog2e : kLog2e / c.temperature;
    const float inv_t = 1.0f / c.temperature;
    float top = -INFINITY, total = 0.0f;
    auto look = [&] {  // the wave's part of the teacher's softmax
        if (!has_entries)
            return;
        entry.t = id >= 0 ? entry.value_of(c, row * topk + tid) : -INFINITY;
        wrong |= !(entry.t < INFINITY);
        if (has_entry)
            ids[tid] = (int)id;
        top = wave_max(entry.t);
        total = wave_sum(top > -INFINITY ? expf((entry.t - top) * inv_t) : 0.0f);
    };
    if ((int)tid < places - topk)
        ids[topk + tid] = tid == 0 && has_label ? (int)label : -1;
    Sums all;
    if constexpr (AGAIN) {
        look();
        const float4 kept = reinterpret_cast<const float4 *>(c.row_stats)[row];
        all = {kept.x, kept.y, kept.z};
        const bool any_wrong = __any(wrong);
        if (tid % kWave == 0)
            room[wave] = {0.0f, 0.0f, 0.0f, top, total, 0.0f, 0, any_wrong};
        __syncthreads();
    } else {
        // Each thread's exponentials are relative to the largest of its first run and its single value, so that sums grow as
        // the runs arrive, with no pass for the row's largest value before.  That fits unless a later value is so much larger that a
        // sum leaves its range, or the first run says nothing.
        float m = alone;
        if (first < cut.end)
            m = run_max<T>(RUNS > 0 ? held[0] : load_run<T>(x + first), m);
        const bool none = m == -INFINITY;
        Sums s = {none ? 0.0f : m, 0.0f, 0.0f};
        Shift t, one;
        shifts<T, KIND>(s.max, ct, t, one);
        s.sum = exp2_fast(kOneStep ? fmaf(alone, t.c, -t.m) : (alone - t.max) * t.c);
        s.sum1 = KIND == kSquare ? s.sum * s.sum : KIND == kTwo ? exp2_fast(kOneStep ? fmaf(alone, one.c, -one.m) : (alone - one.max) * one.c) : 0.0f;
        if constexpr (RUNS > 0)
            runs([&](uint32_t, u32x4 r) { run_sums<T, KIND, kOneStep>(r, t, one, s.sum, s.sum1); });
        else
            read_sums(std::bool_constant<kOneStep>(), t, one, s);
        // s.sum is NaN where t.m is: values too large for one step
        const bool fit = !(none && first < cut.end) && s.sum < 0x1p30f && (KIND != kTwo || s.sum1 < 0x1p30f);
        const float most = wave_max(s.sum == 0.0f ? -INFINITY : s.max);
        rebase<KIND, kOneStep>(s, most, ct);
        s.sum = wave_sum(s.sum);
        if (KIND != kOne)
            s.sum1 = wave_sum(s.sum1);
        look();
        const bool all_fit = __all(fit), any_wrong = __any(wrong);
        if (tid % kWave == 0)
            room[wave] = {most, s.sum, s.sum1, top, total, 0.0f, all_fit, any_wrong};
        __syncthreads();
        const OfWave of = room[tid % kWaves];
        const bool fine = __all(of.fits);
        all.max = lanes_max<kWaves>(of.max);
        s = {of.max, of.sum, of.sum1};
        rebase<KIND, kOneStep>(s, all.max, ct);
        all.sum = lanes_sum<kWaves>(s.sum);
        all.sum1 = lanes_sum<kWaves>(s.sum1);
        if (!fine || !(all.sum < 0x1p30f)) {  // the largest value first, then differences to it
            __syncthreads();
            float largest = alone;
            read_runs([&](uint32_t, u32x4 r) { largest = run_max<T>(r, largest); });
            largest = wave_max(largest);
            if (tid % kWave == 0)
                room[wave].max = largest;
            __syncthreads();
            largest = lanes_max<kWaves>(room[tid % kWaves].max);
            if (largest == -INFINITY)
                largest = NAN;  // no softmax: everything becomes NaN, as 0 / 0 does
            shifts<T, KIND>(largest, ct, t, one);
            s.sum = exp2_fast(t.of_value(alone));
            s.sum1 = KIND == kSquare ? s.sum * s.sum : KIND == kTwo ? exp2_fast(one.of_value(alone)) : 0.0f;
            if (kOneStep && t.one_step())
                read_sums(std::bool_constant<kOneStep>(), t, one, s);
            else
                read_sums(std::false_type(), t, one, s);
            s.sum = wave_sum(s.sum);
            if (KIND != kOne)
                s.sum1 = wave_sum(s.sum1);
            if (tid % kWave == 0)
                room[wave].sum = s.sum, room[wave].sum1 = s.sum1;
            __syncthreads();
            all = {largest, lanes_sum<kWaves>(room[tid % kWaves].sum), lanes_sum<kWaves>(room[tid % kWaves].sum1)};
        }
        if (KIND == kOne)
            all.sum1 = all.sum;
    }
    // the teacher's softmax from the waves' parts of it
    const OfWave of = room[tid % kWaves];
    const bool bad = __any(of.wrong);
    top = lanes_max<kWaves>(of.top);
    const bool some = top > -INFINITY;
    total = lanes_sum<kWaves>(of.total > 0.0f ? of.total * expf((of.top - top) * inv_t) : 0.0f);
    if (!some && !a.with_label && !bad)  // neither term has anything to say of the row
        return no_part();
    Shift t, one;
    shifts<T, KIND>(all.max, ct, t, one);
    const float kt = bad ? NAN : some ? scale * c.teacher_weight * c.temperature : 0.0f;
    const float kl = a.with_label ? scale * c.label_weight : 0.0f;
    if ((int)(wave * kWave) < topk) {
        const float inv_total = some ? 1.0f / total : 0.0f, log_total = some ? logf(total) : 0.0f, log_s = logf(all.sum);
        const float z = (entry.t - top) * inv_t, p = some ? expf(z) * inv_total : 0.0f;
        if (has_entry)
            part[tid] = kt * p;
        if (!AGAIN) {
            float kd = 0.0f;
            if (p > 0.0f) {
                const float value = from_bits<T>(entry.x), e = t.of_value(value), weight = c.teacher_weight * c.temperature;
                if (e != -INFINITY || value == -INFINITY)
                    kd = p * ((z - log_total) - (e * kLn2 - log_s)) * (weight * c.temperature);
                else  // a logit that far below the others has no exponent of 2 in float32, but a loss: T^2 (x - max) / T
                    kd = p * ((z - log_total) + log_s) * (weight * c.temperature) - (p * weight * value - p * weight * all.max);
            }
            kd = wave_sum(kd);
            if (tid % kWave == 0)
                room[wave].kd = kd;
        }
    }
    if (tid == 0) {
        part[topk] = kl;
        if (!AGAIN && c.row_stats)
            reinterpret_cast<float4 *>(c.row_stats)[row] = make_float4(all.max, all.sum, all.sum1, 0.0f);
    }
    const Factors f = {(KIND == kOne ? kt + kl : kt) / all.sum, KIND == kOne ? 0.0f : kl / all.sum1};
    auto value_of = [&](float v) {
        return smooth<KIND>(exp2_fast(t.of_value(v)), KIND == kTwo ? exp2_fast(one.of_value(v)) : 0.0f, f);
    };
    if (grad) {
        if (!kOneStep || t.one_step())
            runs([&](uint32_t at, u32x4 r) {
                const u32x4 g = run_grad<T, KIND, kOneStep>(r, t, one, f);
                if (at < cut.end)
                    store_run_once<T>(grad + at, g);
            });
        else
            read_runs([&](uint32_t at, u32x4 r) { store_run_once<T>(grad + at, run_grad<T, KIND, false>(r, t, one, f)); });
        if (single < vocab)
            grad[single] = T::put(value_of(alone));
    }
    __syncthreads();  // entries in shared memory; what the workgroup wrote of the row comes before what follows
    if (!AGAIN && tid == 0) {
        float loss = 0.0f;
        for (int w = 0; w < kWaves && w * kWave < topk; ++w)
            loss += room[w].kd;
        if (a.with_label) {
            const float value = from_bits<T>(label_bits), e = one.of_value(value), log_s1 = logf(all.sum1);
            if (e != -INFINITY || value == -INFINITY)
                loss += c.label_weight * (log_s1 - e * kLn2);
            else
                loss += c.label_weight * log_s1 - (c.label_weight * value - c.label_weight * all.max);
        }
        c.row_loss[row] = bad ? NAN : loss;
    }
    if (!grad)
        return;
    // the listed entries and the label again, with what they take off: one thread for each id
    float off;
    if (id >= 0 && takes_off(ids, part, listed, tid, off))
        grad[id] = T::put(value_of(from_bits<T>(entry.x)) - off);
    if (tid == 0 && ids[topk] >= 0 && takes_off(ids, part, listed, topk, off))
        grad[label] = T::put(value_of(from_bits<T>(label_bits)) - off);
}

constexpr int kSumThreads = 1024;

// 1 / rows that count
__global__ __launch_bounds__(kSumThreads) void distill_share_kernel(const int64_t *labels, int64_t rows, int64_t ignore, float *share)
{
    __shared__ double room[kSumThreads / kWave];
    int64_t n = 0;
    for (int64_t i = threadIdx.x; i < rows; i += 8 * kSumThreads)
#pragma unroll
        for (int j = 0; j < 8; ++j)  // loads that do not wait for each other
            n += i + j * kSumThreads < rows && labels[i + j * kSumThreads] != ignore;
    const double all = block_sum_f64<kSumThreads>((double)n, room);
    if (threadIdx.x == 0)
        share[0] = all > 0.0 ? (float)(1.0 / all) : 0.0f;
}

// Sum of the rows' losses in double, in a fixed order, times their weight.
__global__ __launch_bounds__(kSumThreads) void distill_sum_kernel(Distill a, double each)
{
    __shared__ double room[kSumThreads / kWave];
    const lpmm_distill_call &c = a.c;
    if (a.shared == kCountHere)
        each = share_of_few(c.labels, c.rows, c.ignore_index);
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < c.rows; i += 8 * kSumThreads)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            s += i + j * kSumThreads < c.rows ? (double)c.row_loss[i + j * kSumThreads] : 0.0;
    s = block_sum_f64<kSumThreads>(s, room);
    if (threadIdx.x == 0)
        c.loss[0] = (float)(s * (a.shared == kCounted ? (double)c.share[0] : each));
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
    if (c.reduction == LPMM_REDUCE_MEAN && c.labels)
        a.shared = c.rows <= kFewRows ? kCountHere : kCounted;
    a.group_shift = -1;
    if (c.teacher_group > 0 && (c.teacher_group & (c.teacher_group - 1)) == 0)
        a.group_shift = __builtin_ctzll((unsigned long long)c.teacher_group);
    a.far = c.rows * c.vocab * (c.type == LPMM_TYPE_F32 ? 4 : 2) > kLastLevel;
    a.each = c.reduction == LPMM_REDUCE_MEAN && !c.labels ? (float)(1.0 / (double)c.rows) : 1.0f;
    return a;
}

template <typename T, int KIND, int THREADS, int RUNS, int WAVES>
void launch(Distill a, hipStream_t stream)
{
    const int places = ((int)a.c.topk + 1 + 3) & ~3;
    for (; a.first < a.c.rows; a.first += kMostRows) {
        const unsigned rows = (unsigned)(a.c.rows - a.first < kMostRows ? a.c.rows - a.first : kMostRows);
        if (a.grad_loss)
            distill_kernel<T, KIND, true, THREADS, RUNS, WAVES><<<rows, THREADS, places * 8, stream>>>(a);
        else
            distill_kernel<T, KIND, false, THREADS, RUNS, WAVES><<<rows, THREADS, places * 8, stream>>>(a);
    }
}

template <typename T, int KIND>
void launch_kind(const Distill &a, hipStream_t stream)
{
    const int64_t runs = a.c.vocab / T::kRun;  // whole ones
    const auto fits = [&](int threads, int each) { return runs <= threads * each && a.c.topk <= threads; };
    // Small workgroups that fill a compute unit several times over, down to two with 64 registers a thread, then one with twice as many.  bf16 rows,
    // loss and gradient of 1 GB (16 KB rows: 268 MB), us with the neighbouring choices: 8192 values 60 (256 x 8 59, 512 x 8 76), 16384: 107 (512 x 8
    // 111), 32000: 196 (256 x 16 200, 1024 x 7 204), 50257: 204 (1024 x 8 210, 512 x 16 215), 65536: 196 (512 x 16 194, 1024 x 16 234).
    // Fewer rows than compute units: the most threads a row can have.
    if (a.c.rows < kFewRows) {
        if (fits(1024, 4))
            return launch<T, KIND, 1024, 4, 4>(a, stream);
    } else {
        if (fits(256, 4))
            return launch<T, KIND, 256, 4, 8>(a, stream);
        if (fits(256, 8))
            return launch<T, KIND, 256, 8, 6>(a, stream);
        if (fits(512, 8))
            return launch<T, KIND, 512, 8, 6>(a, stream);
    }
    if (fits(1024, 7))
        return launch<T, KIND, 1024, 7, 8>(a, stream);
    if (fits(1024, 8))
        return launch<T, KIND, 1024, 8, 8>(a, stream);
    if (fits(1024, 16))
        return launch<T, KIND, 1024, 16, 4>(a, stream);
    launch<T, KIND, 1024, 0, 4>(a, stream);
}

template <typename T>
void launch_type(const Distill &a, hipStream_t stream)
{
    if (!a.with_label || a.c.temperature == 1.0f)
        return launch_kind<T, kOne>(a, stream);
    if constexpr (T::kRun == 8)  // float32 rows move twice the bytes for as many exponentials
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
    if (a.shared == kCounted)
        distill_share_kernel<<<1, kSumThreads, 0, s>>>(c.labels, c.rows, c.ignore_index, c.share);
    if (c.rows > 0)
        launch_rows(a, s);
    if (c.reduction != LPMM_REDUCE_NONE)
        distill_sum_kernel<<<1, kSumThreads, 0, s>>>(a, c.reduction == LPMM_REDUCE_MEAN && c.rows > 0 ? 1.0 / (double)c.rows : 1.0);
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
