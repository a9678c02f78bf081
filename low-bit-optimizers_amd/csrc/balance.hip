// Balance of a router's experts: the loss over a batch's (or each sequence's) router logits, the experts' counts, and the gradient.
//
// With p = softmax(r) of a token, c_e the picks of expert e, T tokens and k picks a token in a group of tokens:
//     loss_g = w E sum_e c_e / (T k) * (1/T) sum_n p_ne + z / T sum_n lse_n^2        loss = 1/G sum_g loss_g
//     d loss / d r_ne = p_ne (f_e - sum_j f_j p_nj + h lse_n),  f_e = w E c_e / (T^2 k G),  h = 2 z / (T G)
// The gradient needs the counts of the whole group, so the logits are read twice: by the call that sums the probabilities and counts the
// picks, and by the one that writes the gradient, which makes the probabilities again rather than read them back (4 bytes a value).
//
// A token's logits lie across 2^l lanes of a wave, 4 or 16 side by side in each, and its maximum and sums are exchanges between those lanes.  A
// thread keeps the sums of its experts' probabilities over all the tokens that pass through it; waves and workgroups are joined in a
// fixed order.  Counts are integers: the order of their atomics, in shared memory only, does not change them.
#include "losses.hpp"

namespace lpmm {
namespace {

constexpr int kBalThreads = 256;
constexpr int kBalWaves = kBalThreads / kWave;
constexpr int64_t kBalParts = 256;  // workgroups a group's tokens are divided among at most

struct Balance {
    lpmm_balance_call c;
    const float *grad_loss;
    int64_t parts, per;  // workgroups to a group, tokens to a workgroup
    int lanes;           // lanes to a token
    // parts of the sums, [groups][parts]: of probabilities and picks [experts], of lse^2, of tokens that count (-1 - n for n with a wrong id among theirs); the groups' losses
    float *prob;
    int32_t *picked;
    double *square;
    int32_t *seen;
    double *group_loss;
};

struct Split {
    int64_t parts, per;
};

// Tokens to a workgroup: 64 at least, so that what it joins at its end is little beside what it reads.
Split split(int64_t groups, int64_t tokens)
{
    int64_t parts = (tokens + 63) / 64;
    const int64_t most = groups >= kBalParts ? 1 : kBalParts / groups;
    if (parts > most)
        parts = most;
    if (parts < 1)
        parts = 1;
    return {parts, (tokens + parts - 1) / parts};
}

__device__ __forceinline__ float spread_max(float v, int lanes)
{
    for (int o = lanes >> 1; o > 0; o >>= 1)
        v = fmaxf(v, __shfl_xor(v, o, kWave));
    return v;
}

__device__ __forceinline__ float spread_sum(float v, int lanes)
{
    for (int o = lanes >> 1; o > 0; o >>= 1)
        v += __shfl_xor(v, o, kWave);
    return v;
}

// The run of logits that a lane holds of a token; past the last expert -infinity, whose probability is 0.
template <typename T, int RUN>
__device__ __forceinline__ void load_logits(const typename T::Raw *x, int held, float (&v)[RUN])
{
    if (held >= RUN) {
        typename T::Raw raw[RUN];
        __builtin_memcpy(raw, x, sizeof raw);
#pragma unroll
        for (int j = 0; j < RUN; ++j)
            v[j] = T::get(raw[j]);
    } else {
#pragma unroll
        for (int j = 0; j < RUN; ++j)
            v[j] = j < held ? T::get(x[j]) : -INFINITY;
    }
}

// Logits become probabilities; returns logsumexp.  A token of -infinity has none: NaN.
template <int RUN>
__device__ __forceinline__ float softmax(float (&v)[RUN], int lanes)
{
    float m = v[0];
#pragma unroll
    for (int j = 1; j < RUN; ++j)
        m = fmaxf(m, v[j]);
    m = spread_max(m, lanes);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
        v[j] = exp2_fast((v[j] - m) * kLog2e);
        s += v[j];
    }
    s = spread_sum(s, lanes);
    const float inv = 1.0f / s;
#pragma unroll
    for (int j = 0; j < RUN; ++j)
        v[j] *= inv;
    return m + logf(s);
}

template <typename T, int RUN>
__global__ __launch_bounds__(kBalThreads) void balance_sums_kernel(Balance a)
{
    __shared__ float probs[kBalWaves][LPMM_BALANCE_MOST];
    __shared__ int counts[LPMM_BALANCE_MOST];
    __shared__ double room[kBalWaves];
    const lpmm_balance_call &c = a.c;
    const int tid = threadIdx.x, experts = (int)c.experts, lane = tid & (kWave - 1);
    const int64_t group = blockIdx.x / a.parts, begin = blockIdx.x % a.parts * a.per;
    const int64_t end = begin + a.per < c.tokens ? begin + a.per : c.tokens;
    const uint8_t *mask = c.mask ? c.mask + group * c.tokens : nullptr;
    for (int e = tid; e < experts; e += kBalThreads)
        counts[e] = 0;
    __syncthreads();
    bool wrong = false;
    for (int64_t i = begin * c.picks + tid; i < end * c.picks; i += kBalThreads) {
        if (mask && !mask[i / c.picks])
            continue;
        const int64_t at = group * c.tokens * c.picks + i;
        const int64_t id = c.id_bits == 64 ? static_cast<const int64_t *>(c.ids)[at] : static_cast<const int32_t *>(c.ids)[at];
        if (id >= experts)
            wrong = true;
        else if (id >= 0)
            atomicAdd(&counts[id], 1);
    }
    // the lane's first expert, and how many experts its run holds
    const int first = (lane & (a.lanes - 1)) * RUN, held = experts - first;
    float sum[RUN] = {};
    double square = 0.0;
    int seen = 0;
    const int step = kBalThreads / a.lanes;
    for (int64_t n0 = begin; n0 < end; n0 += step) {  // the waves leave together: lanes exchange values
        const int64_t n = n0 + tid / a.lanes;
        const bool takes = n < end && (!mask || mask[n]);
        float v[RUN];
        load_logits<T, RUN>(static_cast<const typename T::Raw *>(c.logits) + group * c.outer_stride + n * c.inner_stride + first, takes ? held : 0, v);
        const float lse = softmax<RUN>(v, a.lanes);
        if (!takes)
            continue;
#pragma unroll
        for (int j = 0; j < RUN; ++j)
            sum[j] += v[j];
        if (first == 0) {
            square += (double)lse * (double)lse;
            ++seen;
        }
    }
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
        for (int o = a.lanes; o < kWave; o <<= 1)
            sum[j] += __shfl_xor(sum[j], o, kWave);
        if (lane < a.lanes && j < held)
            probs[tid / kWave][first + j] = sum[j];
    }
    __syncthreads();
    for (int e = tid; e < experts; e += kBalThreads) {
        float s = probs[0][e];
        for (int w = 1; w < kBalWaves; ++w)
            s += probs[w][e];
        a.prob[(int64_t)blockIdx.x * experts + e] = s;
        a.picked[(int64_t)blockIdx.x * experts + e] = counts[e];
    }
    square = block_sum_f64<kBalThreads>(square, room);
    const int all = (int)block_sum_f64<kBalThreads>((double)seen, room);
    const bool any_wrong = __syncthreads_or(wrong);
    if (tid == 0) {
        a.square[blockIdx.x] = square;
        a.seen[blockIdx.x] = any_wrong ? -1 - all : all;
    }
}

// One workgroup a group: joins the parts, writes counts, the gradient's factors and the group's loss.
__global__ __launch_bounds__(kBalThreads) void balance_join_kernel(Balance a)
{
    __shared__ double room[kBalWaves];
    const lpmm_balance_call &c = a.c;
    const int64_t group = blockIdx.x, base = group * a.parts;
    const int experts = (int)c.experts;
    double square = 0.0, tokens = 0.0;
    bool wrong = false;
    for (int64_t p = threadIdx.x; p < a.parts; p += kBalThreads) {
        square += a.square[base + p];
        const int seen = a.seen[base + p];
        wrong |= seen < 0;
        tokens += (double)(seen < 0 ? -1 - seen : seen);
    }
    wrong = __syncthreads_or(wrong);
    square = block_sum_f64<kBalThreads>(square, room);
    tokens = block_sum_f64<kBalThreads>(tokens, room);
    const double per = tokens > 0.0 ? 1.0 / tokens : 0.0;
    const double share = c.picks > 0 ? (double)c.weight * experts * per * per / (double)c.picks : 0.0;
    float *factors = c.factors + group * (experts + 2);
    double loss = 0.0;
    for (int e = threadIdx.x; e < experts; e += kBalThreads) {
        double prob = 0.0;
        int64_t picked = 0;
        for (int64_t p = 0; p < a.parts; ++p) {
            prob += (double)a.prob[(base + p) * experts + e];
            picked += a.picked[(base + p) * experts + e];
        }
        c.counts[group * experts + e] = picked;
        factors[e] = wrong ? NAN : (float)(share * (double)picked / (double)c.groups);
        loss += share * (double)picked * prob;
    }
    loss = block_sum_f64<kBalThreads>(loss, room);
    if (threadIdx.x == 0) {
        factors[experts] = (float)(2.0 * (double)c.z_weight * per / (double)c.groups);
        factors[experts + 1] = 0.0f;
        loss = wrong ? NAN : loss + (double)c.z_weight * square * per;
        if (c.groups == 1)
            c.loss[0] = (float)loss;
        else
            a.group_loss[group] = loss;
    }
}

__global__ __launch_bounds__(kBalThreads) void balance_loss_kernel(const double *group_loss, int64_t groups, float *loss)
{
    __shared__ double room[kBalWaves];
    double s = 0.0;
    for (int64_t g = threadIdx.x; g < groups; g += kBalThreads)
        s += group_loss[g];
    s = block_sum_f64<kBalThreads>(s, room);
    if (threadIdx.x == 0)
        loss[0] = groups > 0 ? (float)(s / (double)groups) : 0.0f;
}

template <typename T, int RUN>
__global__ __launch_bounds__(kBalThreads) void balance_grad_kernel(Balance a)
{
    const lpmm_balance_call &c = a.c;
    const int tid = threadIdx.x, experts = (int)c.experts, lane = tid & (kWave - 1);
    const int64_t group = blockIdx.x / a.parts, begin = blockIdx.x % a.parts * a.per;
    const int64_t end = begin + a.per < c.tokens ? begin + a.per : c.tokens;
    const uint8_t *mask = c.mask ? c.mask + group * c.tokens : nullptr;
    const int first = (lane & (a.lanes - 1)) * RUN, held = experts - first;
    const float *factors = c.factors + group * (experts + 2);
    const float scale = a.grad_loss[0], h = factors[experts];
    float f[RUN];
#pragma unroll
    for (int j = 0; j < RUN; ++j)
        f[j] = j < held ? factors[first + j] : 0.0f;
    const int step = kBalThreads / a.lanes;
    for (int64_t n0 = begin; n0 < end; n0 += step) {
        const int64_t n = n0 + tid / a.lanes;
        const bool takes = n < end && (!mask || mask[n]);
        float v[RUN];
        load_logits<T, RUN>(static_cast<const typename T::Raw *>(c.logits) + group * c.outer_stride + n * c.inner_stride + first, takes ? held : 0, v);
        const float lse = softmax<RUN>(v, a.lanes);
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < RUN; ++j)
            dot += f[j] * v[j];
        dot = spread_sum(dot, a.lanes);
        if (n >= end)
            continue;
        typename T::Raw out[RUN];
#pragma unroll
        for (int j = 0; j < RUN; ++j)
            out[j] = T::put(takes ? scale * (v[j] * ((f[j] - dot) + (h != 0.0f ? h * lse : 0.0f))) : 0.0f);
        typename T::Raw *to = static_cast<typename T::Raw *>(c.grad) + (group * c.tokens + n) * experts + first;
        if (held >= RUN)
            __builtin_memcpy(to, out, sizeof out);
        else
            for (int j = 0; j < RUN; ++j)
                if (j < held)
                    to[j] = out[j];
    }
}

int check_call(const lpmm_balance_call &c)
{
    if (c.type < LPMM_TYPE_F32 || c.type > LPMM_TYPE_BF16 || (c.id_bits != 32 && c.id_bits != 64) || !isfinite(c.weight) || !isfinite(c.z_weight))
        return LPMM_ERR_ARG;
    if (c.experts < 1 || c.experts > LPMM_BALANCE_MOST || c.picks < 0 || c.picks > c.experts || c.groups < 0 || c.groups > (int64_t)1 << 24 ||
        c.tokens < 0 || c.tokens > INT32_MAX || c.tokens * (c.picks > 0 ? c.picks : 1) > INT32_MAX || c.outer_stride < 0 || c.inner_stride < 0)
        return LPMM_ERR_SIZE;
    LPMM_REQUIRE_ALIGN(c.factors, 4);
    if (c.groups == 0)
        return LPMM_OK;
    LPMM_REQUIRE_PTR(c.factors);
    if (c.tokens == 0)
        return LPMM_OK;
    LPMM_REQUIRE_PTR(c.logits);
    LPMM_REQUIRE_ALIGN(c.logits, c.type == LPMM_TYPE_F32 ? 4 : 2);
    return LPMM_OK;
}

Balance arguments(const lpmm_balance_call &c)
{
    Balance a = {};
    a.c = c;
    const Split s = split(c.groups < 1 ? 1 : c.groups, c.tokens);
    a.parts = s.parts;
    a.per = s.per;
    return a;
}

template <typename T, int RUN>
void launch(Balance a, bool grad, hipStream_t stream)
{
    a.lanes = 1;
    while (a.lanes * RUN < a.c.experts)
        a.lanes *= 2;
    const dim3 grid((unsigned)(a.c.groups * a.parts));
    if (grad)
        balance_grad_kernel<T, RUN><<<grid, kBalThreads, 0, stream>>>(a);
    else
        balance_sums_kernel<T, RUN><<<grid, kBalThreads, 0, stream>>>(a);
}

template <int RUN>
void launch_type(const Balance &a, bool grad, hipStream_t stream)
{
    switch (a.c.type) {
    case LPMM_TYPE_F32: return launch<F32, RUN>(a, grad, stream);
    case LPMM_TYPE_F16: return launch<F16, RUN>(a, grad, stream);
    default: return launch<BF16, RUN>(a, grad, stream);
    }
}

void launch_tokens(const Balance &a, bool grad, hipStream_t stream)
{
    if (a.c.experts <= 4 * kWave)
        launch_type<4>(a, grad, stream);
    else
        launch_type<16>(a, grad, stream);
}

}  // namespace
}  // namespace lpmm

extern "C" int64_t lpmm_balance_work_bytes(int64_t groups, int64_t tokens, int64_t experts)
{
    if (groups < 1 || tokens < 0 || experts < 1)
        return 0;
    const int64_t rows = groups * lpmm::split(groups, tokens).parts;
    return rows * 8 + groups * 8 + (rows * experts * 2 + rows) * 4;
}

extern "C" int lpmm_balance_loss(const lpmm_balance_call *call, void *stream)
{
    using namespace lpmm;
    LPMM_REQUIRE_PTR(call);
    const lpmm_balance_call &c = *call;
    if (const int status = check_call(c))
        return status;
    LPMM_REQUIRE_PTR(c.loss);
    LPMM_REQUIRE_ALIGN(c.loss, 4);
    if (c.groups > 0) {
        LPMM_REQUIRE_PTR(c.counts);
        LPMM_REQUIRE_PTR(c.work);
        if (c.tokens * c.picks > 0)
            LPMM_REQUIRE_PTR(c.ids);
    }
    LPMM_REQUIRE_ALIGN(c.ids, c.id_bits / 8);
    LPMM_REQUIRE_ALIGN(c.counts, 8);
    LPMM_REQUIRE_ALIGN(c.work, 8);
    hipStream_t s = static_cast<hipStream_t>(stream);
    Balance a = arguments(c);
    if (c.groups > 0) {
        const int64_t rows = c.groups * a.parts;
        a.square = static_cast<double *>(c.work);
        a.group_loss = a.square + rows;
        a.prob = reinterpret_cast<float *>(a.group_loss + c.groups);
        a.picked = reinterpret_cast<int32_t *>(a.prob + rows * c.experts);
        a.seen = a.picked + rows * c.experts;
        launch_tokens(a, false, s);
        balance_join_kernel<<<(unsigned)c.groups, kBalThreads, 0, s>>>(a);
    }
    if (c.groups != 1)
        balance_loss_kernel<<<1, kBalThreads, 0, s>>>(a.group_loss, c.groups, c.loss);
    return launch_status();
}

extern "C" int lpmm_balance_loss_grad(const lpmm_balance_call *call, const float *grad_loss, void *stream)
{
    using namespace lpmm;
    LPMM_REQUIRE_PTR(call);
    const lpmm_balance_call &c = *call;
    if (const int status = check_call(c))
        return status;
    if (c.groups * c.tokens == 0)
        return LPMM_OK;
    LPMM_REQUIRE_PTR(grad_loss);
    LPMM_REQUIRE_PTR(c.grad);
    LPMM_REQUIRE_ALIGN(grad_loss, 4);
    LPMM_REQUIRE_ALIGN(c.grad, c.type == LPMM_TYPE_F32 ? 4 : 2);
    Balance a = arguments(c);
    a.grad_loss = grad_loss;
    launch_tokens(a, true, static_cast<hipStream_t>(stream));
    return launch_status();
}
