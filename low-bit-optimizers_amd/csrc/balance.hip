// Balance of a router's experts: the loss over a batch's (or each sequence's) router logits, the experts' counts, and the gradient.
//
// With p = softmax(r) of a token, c_e the picks of expert e, T tokens and k picks a token in a group of tokens:
//     loss_g = w E sum_e c_e / (T k) * (1/T) sum_n p_ne + z / T sum_n lse_n^2        loss = 1/G sum_g loss_g
//     d loss / d r_ne = p_ne (f_e - sum_j f_j p_nj + h lse_n),  f_e = w E c_e / (T^2 k G),  h = 2 z / (T G)
// The logits are read twice: by the call that sums the probabilities and counts the picks, and by the one that writes the gradient, which makes the
// probabilities again rather than read them back (4 bytes a value).  The gradient needs the counts of the whole group.  These depend on ids and
// masks alone, so that counting first would let one pass over the logits give loss and gradient; that form is not built.
//
// A token's logits lie across up to 16 neighbouring lanes, in chunks of 16 bytes a lane, so that its maximum and its sums are exchanges
// within a row of lanes (no shared memory) and every load of a wave covers whole stretches of several tokens.  A thread keeps the sums of
// its experts' probabilities over all the tokens that pass through it; lanes, waves and workgroups are joined in a fixed order.  Counts are
// integers: the order of their atomics, in shared memory only, does not change them.
//
// 65536 x 256 fp32, 8 picks, masked (67 MB of logits): sums 18 us, join 9, gradient 22 (134 MB, 6.2 TB/s).  Where a lane had 16
// values side by side, so that the lanes of a load lay 64 bytes apart, and each turn waited for its own loads, sums and gradient took 92 and 120.  The join is
// a chain of reads of what 512 workgroups left, one workgroup to 16 experts and one barrier before its results; with one to all experts of a group it
// took 71.  At 16 x 8 a single workgroup does sums and join in 6 us.  Up to some 16384 x 64 the calls are bound by the host (54-68 us of loss and gradient, of them
// torch's own engine 42-47).
#include "losses.hpp"

namespace lpmm {
namespace {

constexpr int kBalThreads = 256, kBalWaves = kBalThreads / kWave, kLanes = 16;
constexpr int kJoinThreads = 1024, kJoinColumns = 16;
// Most probabilities that a thread adds in 32 bits, before doubles: one chain over all tokens of a long group drifts (identical tokens: after 2^14
// additions by 1e-4 of the sum; after 128 by 8e-6 at most).  Doubles within the workgroup instead took registers: 19 -> 23 us at 65536 x 256 fp32,
// 64 -> 94 at 1024 experts; 64 turns leave more to join (2^22 x 64 bf16: 33 us, with 128 turns 19, with chains of any length 11,
// beside 225 of sums).
constexpr int kBalTurns = 128;
// The gradient's factors are kept divided by this, and grad_loss is multiplied by it: the same bits in the end, but h lse alone would leave float32 where
// logits are of its largest or lowest values and h is 1 or 2 (a group of few tokens), and infinity times a probability of 0 is NaN.
constexpr float kLift = 16.0f;

struct Balance {
    lpmm_balance_call c;
    const float *grad_loss;
    int64_t parts, per;  // workgroups to a group, tokens to a workgroup
    int lanes;           // lanes to a token
    int tiles;           // workgroups that join a group
    // parts of the sums, [groups][parts]: of probabilities and picks [experts], of lse^2, of tokens that count (-1 - n for n with a wrong
    // id among theirs); parts of the loss [groups][tiles]; how many of these are there
    float *prob;
    int32_t *picked;
    double *square;
    int32_t *seen;
    double *loss_part;
    uint32_t *done;
};

struct Split {
    int64_t parts, per, tiles;
};

// Tokens to a workgroup of the sums: 128 at least, so that what it joins at its end is little beside what it reads; 1024 workgroups, four for
// each compute unit, unless a thread would then add more than kBalTurns tokens' probabilities in 32 bits.  One workgroup alone joins its own
// sums, without a second launch.
Split split(int64_t groups, int64_t tokens, int64_t experts)
{
    int64_t lanes = 1;  // to a token of float32; 16-bit types may have half as many, and half as many turns
    while (lanes < kLanes && lanes * F32::kRun < experts)
        lanes *= 2;
    const int64_t longest = kBalTurns * (kBalThreads / lanes), least = (tokens + longest - 1) / longest;
    const int64_t most = groups >= 1024 ? 1 : 1024 / groups;
    int64_t parts = (tokens + 127) / 128;
    parts = parts > most ? most : parts;
    parts = parts < least ? least : parts < 1 ? 1 : parts;
    return {parts, (tokens + parts - 1) / parts, (experts + kJoinColumns - 1) / kJoinColumns};
}

// Over the lanes of a token, 2^l of them at most 16, in all of them.
__device__ __forceinline__ float token_max(float v, int lanes)
{
    if (lanes > 1)
        v = fmaxf(v, dpp_f32<0xB1>(v));
    if (lanes > 2)
        v = fmaxf(v, dpp_f32<0x4E>(v));
    if (lanes > 4)
        v = fmaxf(v, dpp_f32<0x141>(v));
    if (lanes > 8)
        v = fmaxf(v, dpp_f32<0x140>(v));
    return v;
}

__device__ __forceinline__ float token_sum(float v, int lanes)
{
    if (lanes > 1)
        v += dpp_f32<0xB1>(v);
    if (lanes > 2)
        v += dpp_f32<0x4E>(v);
    if (lanes > 4)
        v += dpp_f32<0x141>(v);
    if (lanes > 8)
        v += dpp_f32<0x140>(v);
    return v;
}

// Chunk i of a lane: experts [first + i * step, ...), RUN of them where the token has so many.
struct Place {
    int first, step, experts;
    template <typename T>
    static __device__ __forceinline__ Place of(const Balance &a)
    {
        return {(int)(threadIdx.x & (a.lanes - 1)) * T::kRun, a.lanes * T::kRun, (int)a.c.experts};
    }
    __device__ __forceinline__ int held(int chunk) const { return experts - first - chunk * step; }
};

// A lane's chunks of a token's logits; past the last expert -infinity, whose probability is 0.
template <typename T, int CHUNKS>
__device__ __forceinline__ void load_logits(const typename T::Raw *x, const Place &place, bool takes, u32x4 (&raw)[CHUNKS])
{
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const int held = place.held(i);
        const typename T::Raw *p = x + place.first + i * place.step;
        raw[i] = u32x4{T::kNoValue, T::kNoValue, T::kNoValue, T::kNoValue};
        if (takes && held >= T::kRun) {
            raw[i] = load_run<T>(p);
        } else if (takes && held > 0) {
            float v[T::kRun];
#pragma unroll
            for (int j = 0; j < T::kRun; ++j)
                v[j] = j < held ? T::get(p[j]) : -INFINITY;
            raw[i] = T::pack(v);
        }
    }
}

// Probabilities of a token; returns logsumexp.  A token of -infinity has none: NaN.
template <typename T, int CHUNKS>
__device__ __forceinline__ float softmax(const u32x4 (&raw)[CHUNKS], int lanes, float (&p)[CHUNKS][T::kRun])
{
    float m = -INFINITY, s = 0.0f;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        T::unpack(raw[i], p[i]);
#pragma unroll
        for (int j = 0; j < T::kRun; ++j)
            m = fmaxf(m, p[i][j]);
    }
    m = token_max(m, lanes);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
        for (int j = 0; j < T::kRun; ++j) {
            p[i][j] = exp2_fast((p[i][j] - m) * kLog2e);
            s += p[i][j];
        }
    s = token_sum(s, lanes);
    const float inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
        for (int j = 0; j < T::kRun; ++j)
            p[i][j] *= inv;
    return m + logf(s);
}

// What the waves of a workgroup hand to its first one.
template <int THREADS>
struct Joined {
    static constexpr int kWaves = THREADS / kWave;
    double prob[kWaves][kJoinColumns], count[kWaves][kJoinColumns], square[kWaves], tokens[kWaves];
    int wrong[kWaves];
    bool last;
};

// Joins the parts of kJoinColumns experts of a group: counts, the gradient's factors, this tile's part of the loss.  The tile that comes
// last adds up the parts of the loss, in their order.  Sixteen lanes that lie side by side take a part's experts, a wave four parts at a time.
template <int THREADS>
__device__ __forceinline__ void join(const Balance &a, int64_t group, int tile, Joined<THREADS> &room)
{
    const lpmm_balance_call &c = a.c;
    constexpr int kSlices = THREADS / kJoinColumns, kWaves = THREADS / kWave;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, experts = (int)c.experts;
    const int column = tid % kJoinColumns, slice = tid / kJoinColumns, e = tile * kJoinColumns + column;
    const int64_t base = group * a.parts;
    double square = 0.0, prob = 0.0;
    int seen = 0;
    if (tid < a.parts) {  // asked for before the parts of the experts; long groups have more
        square = a.square[base + tid];
        seen = a.seen[base + tid];
    }
    int64_t picked = 0;
    if (e < experts) {
        for (int64_t p = slice; p < a.parts; p += 8 * kSlices)
#pragma unroll
            for (int j = 0; j < 8; ++j)  // loads that do not wait for each other
                if (p + j * kSlices < a.parts) {
                    const int64_t at = (base + p + j * kSlices) * experts + e;
                    prob += (double)a.prob[at];
                    picked += a.picked[at];
                }
    }
    bool wrong_ids = seen < 0;
    seen = seen < 0 ? -1 - seen : seen;
    for (int64_t p = tid + THREADS; p < a.parts; p += THREADS) {
        const int n = a.seen[base + p];
        square += a.square[base + p];
        seen += n < 0 ? -1 - n : n;  // all together at most 2^28
        wrong_ids |= n < 0;
    }
    double count = (double)picked;  // exact
#pragma unroll
    for (int o = kJoinColumns; o < kWave; o <<= 1) {
        prob += __shfl_xor(prob, o, kWave);
        count += __shfl_xor(count, o, kWave);
    }
    square = wave_sum_f64(square);
    double tokens = wave_sum_f64((double)seen);
    const bool any_wrong = __any(wrong_ids);
    if (lane < kJoinColumns)
        room.prob[wave][lane] = prob, room.count[wave][lane] = count;
    if (lane == 0)
        room.square[wave] = square, room.tokens[wave] = tokens, room.wrong[wave] = any_wrong;
    __syncthreads();
    const int64_t all = c.groups * a.tiles;
    if (wave == 0) {
        prob = count = square = tokens = 0.0;
        int wrong = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            prob += room.prob[w][column];
            count += room.count[w][column];
            square += room.square[w];
            tokens += room.tokens[w];
            wrong |= room.wrong[w];
        }
        const double per = tokens > 0.0 ? 1.0 / tokens : 0.0;
        double loss = 0.0;
        if (lane < kJoinColumns && e < experts) {
            const double share = c.picks > 0 ? (double)c.weight * experts * per * per / (double)c.picks : 0.0;
            c.counts[group * experts + e] = (int64_t)count;
            c.factors[group * (experts + 2) + e] = wrong ? NAN : (float)(share * count / (double)c.groups / kLift);
            loss = share * count * prob;
        }
        loss = wave_sum_f64(loss);
        if (lane == 0) {
            if (tile == 0) {
                c.factors[group * (experts + 2) + experts] = (float)(2.0 * (double)c.z_weight * per / (double)c.groups / kLift);
                c.factors[group * (experts + 2) + experts + 1] = 0.0f;
                loss = wrong ? NAN : loss + (double)c.z_weight * square * per;
            }
            bool last = false;
            if (all == 1) {
                c.loss[0] = (float)loss;
            } else {
                a.loss_part[group * a.tiles + tile] = loss;
                __threadfence();
                last = atomicAdd(a.done, 1u) == (uint32_t)all - 1u;
                __threadfence();
            }
            room.last = last;
        }
    }
    __syncthreads();
    if (!room.last)
        return;
    double s = 0.0;
    for (int64_t i = tid; i < all; i += THREADS)
        s += __hip_atomic_load(a.loss_part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s = block_sum_f64<THREADS>(s, room.square);
    if (tid == 0)
        c.loss[0] = (float)(s / (double)c.groups);
}

__global__ __launch_bounds__(kJoinThreads) void balance_join_kernel(Balance a)
{
    __shared__ Joined<kJoinThreads> room;
    join(a, blockIdx.x / a.tiles, blockIdx.x % a.tiles, room);
}

template <typename T, int CHUNKS>
__global__ __launch_bounds__(kBalThreads) void balance_sums_kernel(Balance a)
{
    constexpr int kRun = T::kRun;
    __shared__ float probs[kBalWaves][CHUNKS * kLanes * kRun];
    __shared__ int counts[CHUNKS * kLanes * kRun];
    __shared__ double room[kBalWaves];
    const lpmm_balance_call &c = a.c;
    const int tid = threadIdx.x, experts = (int)c.experts, lane = tid & (kWave - 1);
    const int64_t group = blockIdx.x / a.parts, begin = blockIdx.x % a.parts * a.per;
    const int64_t end = begin + a.per < c.tokens ? begin + a.per : c.tokens;
    const uint8_t *mask = c.mask ? c.mask + group * c.tokens : nullptr;
    if (blockIdx.x == 0 && tid == 0)
        *a.done = 0;
    const Place place = Place::of<T>(a);
    const int step = kBalThreads / a.lanes;
    const typename T::Raw *logits = static_cast<const typename T::Raw *>(c.logits) + group * c.outer_stride;
    auto takes = [&](int64_t n) { return n < end && (!mask || mask[n]); };
    u32x4 raw[CHUNKS];
    bool now = takes(begin + tid / a.lanes);
    load_logits<T, CHUNKS>(logits + (begin + tid / a.lanes) * c.inner_stride, place, now, raw);

    for (int e = tid; e < experts; e += kBalThreads)
        counts[e] = 0;
    __syncthreads();
    bool wrong = false;
    const uint32_t picks = (uint32_t)c.picks;  // tokens * picks fit 31 bits
    for (uint32_t i = (uint32_t)begin * picks + tid; begin < end && i < (uint32_t)end * picks; i += kBalThreads) {
        if (mask && !mask[i / picks])
            continue;
        const int64_t at = group * c.tokens * picks + i;
        const int64_t id = c.id_bits == 64 ? static_cast<const int64_t *>(c.ids)[at] : static_cast<const int32_t *>(c.ids)[at];
        if (id >= experts)
            wrong = true;
        else if (id >= 0)
            atomicAdd(&counts[id], 1);
    }
    float sum[CHUNKS][kRun] = {};
    double square = 0.0;
    int seen = 0;
    for (int64_t n0 = begin; n0 < end; n0 += step) {  // the waves leave together: lanes exchange values
        float p[CHUNKS][kRun];
        const float lse = softmax<T, CHUNKS>(raw, a.lanes, p);
        const bool taken = now;
        const int64_t next = n0 + step + tid / a.lanes;
        now = takes(next);
        load_logits<T, CHUNKS>(logits + next * c.inner_stride, place, now, raw);
        if (!taken)
            continue;
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
            for (int j = 0; j < kRun; ++j)
                sum[i][j] += p[i][j];
        if (place.first == 0) {
            square += (double)lse * (double)lse;
            ++seen;
        }
    }
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
            for (int o = a.lanes; o < kWave; o <<= 1)
                sum[i][j] += __shfl_xor(sum[i][j], o, kWave);
            if (lane < a.lanes && j < place.held(i))
                probs[tid / kWave][place.first + i * place.step + j] = sum[i][j];
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
    if (gridDim.x == 1) {
        __shared__ Joined<kBalThreads> joined;
        __syncthreads();
        for (int tile = 0; tile < a.tiles; ++tile) {
            join(a, 0, tile, joined);
            __syncthreads();
        }
    }
}

// No groups: the loss is 0.
__global__ void balance_none_kernel(float *loss) { loss[0] = 0.0f; }

template <typename T, int CHUNKS>
__global__ __launch_bounds__(kBalThreads) void balance_grad_kernel(Balance a)
{
    constexpr int kRun = T::kRun;
    const lpmm_balance_call &c = a.c;
    const int tid = threadIdx.x, experts = (int)c.experts;
    const int64_t group = blockIdx.x / a.parts, begin = blockIdx.x % a.parts * a.per;
    const int64_t end = begin + a.per < c.tokens ? begin + a.per : c.tokens;
    const uint8_t *mask = c.mask ? c.mask + group * c.tokens : nullptr;
    const Place place = Place::of<T>(a);
    const int step = kBalThreads / a.lanes;
    const typename T::Raw *logits = static_cast<const typename T::Raw *>(c.logits) + group * c.outer_stride;
    typename T::Raw *grad = static_cast<typename T::Raw *>(c.grad) + group * c.tokens * experts;
    auto takes = [&](int64_t n) { return n < end && (!mask || mask[n]); };
    u32x4 raw[CHUNKS];
    bool now = takes(begin + tid / a.lanes);
    load_logits<T, CHUNKS>(logits + (begin + tid / a.lanes) * c.inner_stride, place, now, raw);
    const float *factors = c.factors + group * (experts + 2);
    const float scale = a.grad_loss[0] * kLift, h = factors[experts];
    float f[CHUNKS][kRun];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
        for (int j = 0; j < kRun; ++j)
            f[i][j] = j < place.held(i) ? factors[place.first + i * place.step + j] : 0.0f;
    for (int64_t n0 = begin; n0 < end; n0 += step) {
        float p[CHUNKS][kRun];
        const float lse = softmax<T, CHUNKS>(raw, a.lanes, p);
        const bool taken = now;
        const int64_t n = n0 + tid / a.lanes, next = n + step;
        now = takes(next);
        load_logits<T, CHUNKS>(logits + next * c.inner_stride, place, now, raw);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
            for (int j = 0; j < kRun; ++j)
                dot += f[i][j] * p[i][j];
        dot = token_sum(dot, a.lanes);
        if (n >= end)
            continue;
        const float more = h != 0.0f ? h * lse : 0.0f;
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const int held = place.held(i);
            typename T::Raw *to = grad + n * experts + place.first + i * place.step;
#pragma unroll
            for (int j = 0; j < kRun; ++j)
                p[i][j] = taken ? scale * (p[i][j] * ((f[i][j] - dot) + more)) : 0.0f;
            if (held >= kRun)
                store_run<T>(to, T::pack(p[i]));
            else
#pragma unroll
                for (int j = 0; j < kRun; ++j)
                    if (j < held)
                        to[j] = T::put(p[i][j]);
        }
    }
}

int check_call(const lpmm_balance_call &c)
{
    if (c.type < LPMM_TYPE_F32 || c.type > LPMM_TYPE_BF16 || (c.id_bits != 32 && c.id_bits != 64) || !isfinite(c.weight) || !isfinite(c.z_weight))
        return LPMM_ERR_ARG;
    // groups and tokens: a launch's threads are counted in 32 bits, 1024 to 16 experts of a group, 256 to 32 tokens
    if (c.experts < 1 || c.experts > LPMM_BALANCE_MOST || c.picks < 0 || c.picks > c.experts || c.groups < 0 || c.groups > LPMM_BALANCE_GROUPS ||
        c.tokens < 0 || c.tokens > LPMM_BALANCE_TOKENS || c.tokens * (c.picks > 0 ? c.picks : 1) > INT32_MAX ||
        c.groups * c.tokens > LPMM_BALANCE_TOKENS || c.outer_stride < 0 || c.inner_stride < 0)
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

template <typename T, int CHUNKS>
void launch(Balance a, bool grad, hipStream_t stream)
{
    a.lanes = 1;
    while (a.lanes < kLanes && a.lanes * T::kRun < a.c.experts)
        a.lanes *= 2;
    if (grad) {  // two turns to a workgroup: the second's logits are on their way while the first is computed
        a.per = 2 * (kBalThreads / a.lanes);
        a.parts = (a.c.tokens + a.per - 1) / a.per;
        balance_grad_kernel<T, CHUNKS><<<(unsigned)(a.c.groups * a.parts), kBalThreads, 0, stream>>>(a);
    } else {
        balance_sums_kernel<T, CHUNKS><<<(unsigned)(a.c.groups * a.parts), kBalThreads, 0, stream>>>(a);
    }
}

template <typename T>
void launch_type(const Balance &a, bool grad, hipStream_t stream)
{
    const int64_t chunks = (a.c.experts + kLanes * T::kRun - 1) / (kLanes * T::kRun);
    if (chunks <= 1)
        return launch<T, 1>(a, grad, stream);
    if (chunks <= 2)
        return launch<T, 2>(a, grad, stream);
    if (chunks <= 4)
        return launch<T, 4>(a, grad, stream);
    if (T::kRun == 8 || chunks <= 8)
        return launch<T, 8>(a, grad, stream);
    if constexpr (T::kRun == 4)
        launch<T, 16>(a, grad, stream);
}

void launch_tokens(const Balance &a, bool grad, hipStream_t stream)
{
    switch (a.c.type) {
    case LPMM_TYPE_F32: return launch_type<F32>(a, grad, stream);
    case LPMM_TYPE_F16: return launch_type<F16>(a, grad, stream);
    default: return launch_type<BF16>(a, grad, stream);
    }
}

}  // namespace
}  // namespace lpmm

extern "C" int64_t lpmm_balance_work_bytes(int64_t groups, int64_t tokens, int64_t experts)
{
    if (groups < 1 || tokens < 0 || experts < 1)
        return 0;
    const lpmm::Split s = lpmm::split(groups, tokens, experts);
    const int64_t rows = groups * s.parts;
    return rows * 8 + groups * s.tiles * 8 + (rows * experts * 2 + rows + 1) * 4;
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
    if (c.groups == 0) {
        balance_none_kernel<<<1, 1, 0, s>>>(c.loss);
        return launch_status();
    }
    const Split cut = split(c.groups, c.tokens, c.experts);
    const int64_t rows = c.groups * cut.parts;
    Balance a = {};
    a.c = c;
    a.parts = cut.parts;
    a.per = cut.per;
    a.tiles = (int)cut.tiles;
    a.square = static_cast<double *>(c.work);
    a.loss_part = a.square + rows;
    a.prob = reinterpret_cast<float *>(a.loss_part + c.groups * cut.tiles);
    a.picked = reinterpret_cast<int32_t *>(a.prob + rows * c.experts);
    a.seen = a.picked + rows * c.experts;
    a.done = reinterpret_cast<uint32_t *>(a.seen + rows);
    launch_tokens(a, false, s);
    if (rows > 1)
        balance_join_kernel<<<(unsigned)(c.groups * cut.tiles), kJoinThreads, 0, s>>>(a);
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
    Balance a = {};
    a.c = c;
    a.grad_loss = grad_loss;
    launch_tokens(a, true, static_cast<hipStream_t>(stream));
    return launch_status();
}
