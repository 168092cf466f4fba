// Choosing the next token of each row of logits from a given random number, gfx950; the rules are in lutgemm_gfx950.h.
//
// Mathematics.  The order is larger logits first, equal ones by index, and every filter keeps a first part of it: the row's
// tokens are never sorted, only the element is looked for at which a running count or a running sum of weights reaches a target.  The
// weights, exp((l - m) / temperature) in 64 bits, are held as whole numbers of 2^-bits, so that sums do not depend on the order in
// which threads add; as many bits as leave room for the sum of a vocabulary, 43 (2^20 tokens) to 52.  A histogram of counts and sums over 4096 equal steps of the logit
// below the largest, as far as weights reach, says in which step a target is reached; the few tokens of that step are then looked
// at one by one.  Where they are many (equal logits, an endless temperature) digits of the logit's bits are followed instead.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lutgemm_gfx950.h"
#include "lutgemm_common.h"
#include "lutgemm_internal.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kSteps = 4096;          // of the histogram
constexpr int kPerThread = kSteps / kThreads;
constexpr int kList = 1024;           // tokens of a step that are looked at one by one, at most

typedef unsigned long long u64;

struct Args {
    const void *logits;
    int64_t row_stride;
    int rows, vocab;
    int bits;           // a weight of 1 is 2^bits
    float reach;        // (m - l) / temperature beyond which a weight is less than half of 2^-bits
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p, *uniform;
    int64_t *ids;
    float *logprob;
};

// A logit as fp32, NaN as -inf and -0 as +0 (equal logits have equal bits).
template <typename T>
__device__ __forceinline__ float logit_of(T raw);
template <>
__device__ __forceinline__ float logit_of<float>(float raw) { return raw != raw ? -INFINITY : raw + 0.0f; }
template <>
__device__ __forceinline__ float logit_of<_Float16>(_Float16 raw) { return logit_of((float)raw); }
template <>
__device__ __forceinline__ float logit_of<uint16_t>(uint16_t raw) { return logit_of(__builtin_bit_cast(float, (uint32_t)raw << 16)); }   // bf16

// Larger logits have larger keys.
__device__ __forceinline__ uint32_t key_of(float l)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, l);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of_key(uint32_t k)
{
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// exp of x in [-37, 0], by powers of two and the exponential series of what is left (|r| <= ln(2) / 2): terms to r^13, off by 2^-53.
__device__ __forceinline__ double exponential(double x)
{
    const double k = __builtin_rint(x * 1.4426950408889634);
    const double r = __builtin_fma(k, -0.6931471805599453, x);   // (|k| <= 53: what ln(2) is rounded by comes to 2^-49)
    double p = 1.0 / 6227020800.0;
    p = __builtin_fma(p, r, 1.0 / 479001600.0);
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)k);
}

// What a row's weights are formed with.
struct Scale {
    float most;        // the largest logit
    double t, inverse; // the temperature (0 where it is endless) and 1 / temperature
    float steps;       // steps of the histogram per unit of the logit
    double reach;
    int bits;
    // the weight, 0 where it is less than half of 2^-bits
    __device__ __forceinline__ double weight(float l) const
    {
        if (l == most) return 1.0;
        const double d = (double)l - (double)most, q = d * inverse;
        const double x = __builtin_fma(__builtin_fma(-q, t, d), inverse, q);   // d / t
        return l > -INFINITY && x >= -reach ? exponential(x) : 0.0;            // (an infinite `most`: x is -inf or NaN)
    }
    __device__ __forceinline__ u64 fixed(double w) const { return (u64)__builtin_rint(__builtin_amdgcn_ldexp(w, bits)); }
    __device__ __forceinline__ int step(float l) const
    {
        return l == most ? 0 : (int)fminf((most - l) * steps, (float)(kSteps - 1));
    }
};

// The element at which a target is reached: its key and index, and the count and sum of the order up to it, itself among them.
struct Found {
    uint32_t key, index, count;
    u64 sum;
};

struct Shared {
    u64 sum[kSteps];
    uint32_t count[kSteps];
    u64 list[kList], list_weight[kList];   // (key, ~index): in the order where larger comes first
    u64 wave_sum[kWaves];
    uint32_t wave_count[kWaves];
    float wave_most[kWaves];
    u64 digit_sum[256];
    uint32_t digit_count[256];
    int step;
    uint32_t listed;
    Found found;
    u64 before_sum, min_sum;
    uint32_t before_count, min_count, digit;
};

template <typename T, typename F>
__device__ __forceinline__ void for_each(const T *row, int vocab, F f)
{
    for (int i = threadIdx.x; i < vocab; i += kThreads) f(logit_of(row[i]), (uint32_t)i);
}

// Sums of (count, sum) over the threads before this one; the last thread's own added give the totals.
__device__ void exclusive_scan(Shared &s, uint32_t &count, u64 &sum)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t own_count = count;
    const u64 own_sum = sum;
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t c = __shfl_up(count, d);
        const u64 w = __shfl_up(sum, d);
        if (lane >= d) {
            count += c;
            sum += w;
        }
    }
    __syncthreads();
    if (lane == 63) {
        s.wave_count[wave] = count;
        s.wave_sum[wave] = sum;
    }
    __syncthreads();
    count -= own_count;
    sum -= own_sum;
    for (int w = 0; w < wave; ++w) {
        count += s.wave_count[w];
        sum += s.wave_sum[w];
    }
}

// The first element of the order at which the running count is at least `count` (by_sum false) or the running sum at least `sum`;
// the row holds one.
template <typename T>
__device__ Found reach(Shared &s, const T *row, int vocab, const Scale &scale, bool by_sum, uint32_t count, u64 sum)
{
    const int tid = threadIdx.x;
    __syncthreads();
    // the step (the arrays hold running totals)
    for (int i = 0; i < kPerThread; ++i) {
        const int b = tid * kPerThread + i;
        const uint32_t c0 = b > 0 ? s.count[b - 1] : 0;
        const u64 w0 = b > 0 ? s.sum[b - 1] : 0;
        if (by_sum ? w0 < sum && s.sum[b] >= sum : c0 < count && s.count[b] >= count) {
            s.step = b;
            s.before_count = c0;
            s.before_sum = w0;
        }
    }
    if (tid == 0) s.listed = 0;
    __syncthreads();
    const int step = s.step;
    uint32_t before_count = s.before_count;
    u64 before_sum = s.before_sum;
    if (s.count[step] - before_count <= (uint32_t)kList) {
        for_each(row, vocab, [&](float l, uint32_t i) {
            if (scale.step(l) != step) return;
            const u64 w = scale.fixed(scale.weight(l));
            if (w == 0) return;
            const uint32_t at = atomicAdd(&s.listed, 1u);
            s.list[at] = (u64)key_of(l) << 32 | (uint32_t)~i;
            s.list_weight[at] = w;
        });
        __syncthreads();
        if (tid < (int)s.listed) {
            const u64 mine = s.list[tid];
            uint32_t c = before_count + 1;
            u64 w = before_sum + s.list_weight[tid];
            for (uint32_t j = 0; j < s.listed; ++j) {
                const bool ahead = s.list[j] > mine;
                c += ahead;
                w += ahead ? s.list_weight[j] : 0;
            }
            if (by_sum ? w >= sum && w - s.list_weight[tid] < sum : c == count) s.found = {(uint32_t)(mine >> 32), (uint32_t)~mine, c, w};
        }
        __syncthreads();
        return s.found;
    }
    // many: the key's digits of eight bits, from the top
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (tid < 256) {
            s.digit_count[tid] = 0;
            s.digit_sum[tid] = 0;
        }
        __syncthreads();
        for_each(row, vocab, [&](float l, uint32_t) {
            const uint32_t key = key_of(l);
            if (scale.step(l) != step || (shift < 24 && key >> (shift + 8) != prefix)) return;
            const u64 w = scale.fixed(scale.weight(l));
            if (w == 0) return;
            atomicAdd(&s.digit_count[(key >> shift) & 255u], 1u);
            atomicAdd(&s.digit_sum[(key >> shift) & 255u], w);
        });
        __syncthreads();
        if (tid == 0) {
            int d = 255;
            for (; d > 0; --d) {
                if (by_sum ? before_sum + s.digit_sum[d] >= sum : before_count + s.digit_count[d] >= count) break;
                before_sum += s.digit_sum[d];
                before_count += s.digit_count[d];
            }
            s.digit = d;
            s.before_sum = before_sum;
            s.before_count = before_count;
        }
        __syncthreads();
        prefix = prefix << 8 | s.digit;
        before_sum = s.before_sum;
        before_count = s.before_count;
    }
    // equal logits: the one so many places further on
    const u64 w = scale.fixed(scale.weight(logit_of_key(prefix)));
    const uint32_t place = by_sum ? (uint32_t)((sum - before_sum + w - 1) / w) : count - before_count;   // 1 for the first
    const int own = (vocab + kThreads - 1) / kThreads, first = min(tid * own, vocab), past = min(first + own, vocab);
    uint32_t c = 0;
    for (int i = first; i < past; ++i) c += key_of(logit_of(row[i])) == prefix;
    uint32_t ahead = c;
    u64 unused = 0;
    exclusive_scan(s, ahead, unused);
    if (ahead < place && ahead + c >= place) {
        uint32_t at = ahead;
        for (int i = first; i < past; ++i)
            if (key_of(logit_of(row[i])) == prefix && ++at == place) s.found = {prefix, (uint32_t)i, before_count + place, before_sum + place * w};
    }
    __syncthreads();
    return s.found;
}

// One workgroup per row.
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Args a)
{
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x;
    const T *row = (const T *)a.logits + r * a.row_stride;

    float most = -INFINITY;
    for_each(row, a.vocab, [&](float l, uint32_t) { most = fmaxf(most, l); });
    for (int m = 1; m < 64; m *= 2) most = fmaxf(most, __shfl_xor(most, m));
    if (lane == 0) s.wave_most[wave] = most;
    for (int b = tid; b < kSteps; b += kThreads) {
        s.count[b] = 0;
        s.sum[b] = 0;
    }
    if (tid == 0) {
        s.min_count = 0;
        s.min_sum = 0;
    }
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) most = fmaxf(most, s.wave_most[w]);
    if (most == -INFINITY) {
        if (tid == 0) {
            a.ids[r] = -1;
            if (a.logprob) a.logprob[r] = -INFINITY;
        }
        return;
    }
    const float t = a.temperature ? a.temperature[r] : 1.0f;
    const bool greedy = !(t > 0.0f);
    const float p = a.top_p ? a.top_p[r] : 1.0f, asked = a.min_p ? a.min_p[r] : 0.0f;
    const float least = asked > 0.0f ? fminf(asked, 1.0f) : 0.0f;
    const int k = greedy ? 1 : a.top_k ? a.top_k[r] : 0;
    // (a greedy row: its weights are of no account, the first of its largest logits is)
    const Scale scale = {most, greedy ? 1e-30 : t == INFINITY ? 0.0 : (double)t, greedy ? 1e30 : 1.0 / (double)t,
                         greedy ? 1e30f : fminf((float)kSteps / a.reach / t, 1e30f), (double)a.reach, a.bits};

    uint32_t min_count = 0;
    u64 min_sum = 0;
    for_each(row, a.vocab, [&](float l, uint32_t) {
        const double w = scale.weight(l);
        const u64 f = scale.fixed(w);
        if (f == 0) return;
        const int b = scale.step(l);
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.sum[b], f);
        if (w >= (double)least) {
            ++min_count;
            min_sum += f;
        }
    });
    if (least > 0.0f) {
        atomicAdd(&s.min_count, min_count);
        atomicAdd(&s.min_sum, min_sum);
    }
    __syncthreads();
    {   // running totals
        uint32_t c = 0;
        u64 w = 0;
        for (int i = 0; i < kPerThread; ++i) {
            c += s.count[tid * kPerThread + i];
            w += s.sum[tid * kPerThread + i];
        }
        exclusive_scan(s, c, w);
        for (int i = 0; i < kPerThread; ++i) {
            c += s.count[tid * kPerThread + i];
            w += s.sum[tid * kPerThread + i];
            s.count[tid * kPerThread + i] = c;
            s.sum[tid * kPerThread + i] = w;
        }
    }
    __syncthreads();
    uint32_t kept = s.count[kSteps - 1];
    u64 total = s.sum[kSteps - 1];
    if (k > 0 && (uint32_t)k < kept) {
        const Found f = reach(s, row, a.vocab, scale, false, (uint32_t)k, 0);
        kept = f.count;
        total = f.sum;
    }
    if (p < 1.0f && kept > 1) {
        const double target = __builtin_ceil((double)fmaxf(p, 0.0f) * (double)total);
        const Found f = reach(s, row, a.vocab, scale, true, 0, target < 1.0 ? 1 : (u64)target);
        if (f.count < kept) {
            kept = f.count;
            total = f.sum;
        }
    }
    if (least > 0.0f && s.min_count < kept) {
        kept = s.min_count;
        total = s.min_sum;
    }
    float u = a.uniform[r];
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    u64 target = (u64)__builtin_floor((double)u * (double)total);
    if (target >= total) target = total - 1;
    const Found f = reach(s, row, a.vocab, scale, true, 0, target + 1);
    if (tid == 0) {
        a.ids[r] = f.index;
        if (a.logprob) a.logprob[r] = kept == 1 ? 0.0f : (float)log(scale.weight(logit_of_key(f.key)) * (double)(1ull << a.bits) / (double)total);
    }
}

int launch_status()
{
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? LUTGEMM_OK : lutgemm_internal_hip_fail((int)e);
}

bool sizes_fit(int rows, int vocab) { return rows >= 1 && rows <= 65535 && vocab >= 1 && vocab <= 1 << 20; }

}  // namespace

extern "C" {

size_t lutgemm_sampling_workspace(int rows, int vocab)
{
    return sizes_fit(rows, vocab) ? 16 : 0;
}

int lutgemm_sample_tokens(const lutgemm_sampling *c, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!c || !c->logits || !c->uniform || !c->ids || !sizes_fit(c->rows, c->vocab)) return LUTGEMM_EINVAL;
    if (c->logits_type < LUTGEMM_TYPE_F16 || c->logits_type > LUTGEMM_TYPE_F32) return LUTGEMM_EINVAL;
    if (c->rows > 1 && c->row_stride < 0) return LUTGEMM_EINVAL;
    if (!workspace || workspace_bytes < lutgemm_sampling_workspace(c->rows, c->vocab)) return LUTGEMM_EINVAL;
    if (((uintptr_t)workspace & 15u) || ((uintptr_t)c->logits & (c->logits_type == LUTGEMM_TYPE_F32 ? 3u : 1u)) || ((uintptr_t)c->temperature & 3u) ||
        ((uintptr_t)c->top_k & 3u) || ((uintptr_t)c->top_p & 3u) || ((uintptr_t)c->min_p & 3u) || ((uintptr_t)c->uniform & 3u) ||
        ((uintptr_t)c->ids & 7u) || ((uintptr_t)c->logprob & 3u))
        return LUTGEMM_EALIGN;
    int doublings = 0;
    while (1 << doublings < c->vocab) ++doublings;
    const int bits = 63 - doublings < 52 ? 63 - doublings : 52;
    const Args a = {c->logits, c->row_stride, c->rows, c->vocab, bits, (bits + 1) * 0.6931472f, c->temperature, c->top_k, c->top_p, c->min_p, c->uniform, c->ids, c->logprob};
    const hipStream_t hs = (hipStream_t)stream;
    const dim3 grid((unsigned)c->rows), threads(kThreads);
    if (c->logits_type == LUTGEMM_TYPE_F16) hipLaunchKernelGGL(sample_kernel<_Float16>, grid, threads, 0, hs, a);
    else if (c->logits_type == LUTGEMM_TYPE_BF16) hipLaunchKernelGGL(sample_kernel<uint16_t>, grid, threads, 0, hs, a);
    else hipLaunchKernelGGL(sample_kernel<float>, grid, threads, 0, hs, a);
    return launch_status();
}

}  // extern "C"
