// Choosing the next token of each row of logits from a given random number, gfx950; the rules are in lutgemm_gfx950.h.
//
// Mathematics.  The order is larger logits first, equal ones by index, and every filter keeps a first part of it: the row's
// tokens are never sorted, only the element is looked for at which a running count or a running sum of weights reaches a target.  The
// weights, exp((l - m) / temperature) in 64 bits, are held as whole numbers of 2^-bits, so that sums do not depend on the order in
// which threads add; as many bits as leave room for the sum of a vocabulary, 43 (2^20 tokens) to 51.  A histogram of sums over steps of
// a 64th of a power of two says in which step a target is reached; the few tokens of that step are then looked at one by one.  Where they are
// many (equal logits, an endless temperature) digits of the logit's bits are followed instead.
// Bound: 256 rows of 131072 fp32 logits, a CU each, 94 us, of which (taken apart when it was 96) 23 us to read them for the largest (134 MB, 5.8 TB/s), 50 us for the weights (some
// 25 instructions a logit 20 us, additions to the histogram in LDS 17 us, the list of the tokens near the largest 13 us), 22 us for the
// choice, which reads a row again where the target is not among the listed tokens.  Few rows: three launches that wait for one another,
// one row of 32000 with all filters 24.2 us (4, 7 and 14).
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "lutgemm_gfx950.h"
#include "lutgemm_common.h"
#include "lutgemm_internal.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kSteps = 4096;          // of the histogram, 64 to a power of two (52 powers at most)
constexpr int kCounted = 256;         // top_k from which tokens are counted in the first pass
constexpr int kPerThread = kSteps / kThreads;
constexpr int kNear = 4096;           // tokens near the largest that are kept by themselves, at most
constexpr int kMembers = 1024;        // tokens of a step that are looked at one by one, at most
constexpr int kParts = 8;            // workgroups that share a row, at most

typedef unsigned long long u64;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// What the workgroups of a row hand on, per row.
struct RowWork {
    u64 sum[kSteps];
    u64 near_[kNear];
    uint32_t count[kSteps];
    uint32_t near_count;
    int near_steps, unused[2];
    float most[kParts], total[kParts], square[kParts], number[kParts];   // of the parts
};

struct Args {
    const void *logits;
    int64_t row_stride;
    int rows, vocab;
    int bits;           // a weight of 1 is 2^bits
    int parts;          // workgroups that share a row
    float near_share, near_spread;   // which tokens are kept by themselves, see scale_of
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p, *uniform;
    int64_t *ids;
    float *logprob;
    RowWork *work;
};

// A logit as fp32.
__device__ __forceinline__ float logit_of(float raw) { return raw; }
__device__ __forceinline__ float logit_of(_Float16 raw) { return (float)raw; }
__device__ __forceinline__ float logit_of(uint16_t raw) { return __builtin_bit_cast(float, (uint32_t)raw << 16); }   // bf16

// Larger logits have larger keys, equal ones equal ones (-0 is +0).
__device__ __forceinline__ uint32_t key_of(float l)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, l + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of_key(uint32_t k)
{
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

constexpr int kFractions = 256;   // of a power of two, in the table of the exponential

struct Table {
    double power[kFractions];   // 2^(i / 256), by the exponential series
    constexpr Table() : power()
    {
        for (int i = 0; i < kFractions; ++i) {
            const double x = 0.6931471805599453094 * i / kFractions;
            double sum = 1.0;
            for (int n = 24; n > 0; --n) sum = 1.0 + sum * x / n;
            power[i] = sum;
        }
    }
};
__device__ const Table kTable;

// What a row's weights are formed with.
struct Scale {
    float most;        // the largest logit
    double origin;     // the same; 2^128 where it is infinite (then it alone has weight: `fractions` is very large)
    double inverse;    // 1 / temperature
    double fractions;  // 256 log2(e) / temperature
    double least;      // the place of a weight of 2^-bits / 4
    int bits;
    int near_steps;    // tokens of earlier steps are kept by themselves

    // 256 log2(e) (l - most) / t, not less than `least`, and that for NaN
    __device__ __forceinline__ double place(float l) const { return fmin(fmax(((double)l - origin) * fractions, least), 0.0); }
    // The weight as a whole number of 2^-bits, and the step; false where it is less than half of 2^-bits: 0, and a step behind all others.
    // The place is n + f with |f| <= 1/2; 2^(n / 256) by powers of two and a table, 2^(f / 256) by its series: terms to f^4, off by
    // 2^-54.  Conversions, roundings and scalings of 64-bit numbers take four times as long as sums and products here, so whole numbers are
    // made by adding 1.5 * 2^52 (2^52), whose last place is one, and powers of two by adding to the exponent (with such instructions and a
    // series of twelve terms 256 rows of 131072 logits took 187 us).  No branches: several weights are formed side by side.
    __device__ __forceinline__ bool weight(float l, const double *table, u64 &w, int &step) const
    {
        const double y = place(l);
        const double shifted = y + 0x1.8p52;
        const int n = (int)(uint32_t)__builtin_bit_cast(u64, shifted);
        const double f = y - (shifted - 0x1.8p52);
        constexpr double c = 0.6931471805599453 / kFractions;
        double p = __builtin_fma(f, c * c * c * c / 24.0, c * c * c / 6.0);
        p = __builtin_fma(p, f, c * c / 2.0);
        p = __builtin_fma(p, f, c);
        const double power = table[n & (kFractions - 1)];
        const double v = __builtin_fma(p * f, power, power);
        const u64 scaled = __builtin_bit_cast(u64, v) + ((u64)(uint32_t)((n >> 8) + bits) << 52);
        w = __builtin_bit_cast(u64, __builtin_bit_cast(double, scaled) + 0x1p52) & ((1ull << 52) - 1);
        step = -n >> 2;   // (larger logits in earlier ones)
        return w != 0;
    }
    // Whether a logit is of a step, but for its last hundredth on either side (a difference's place in fp32 is off by 2^-22 of itself; half
    // differences, since those of finite logits can lie beyond fp32's range).
    __device__ __forceinline__ bool near_step(float l, int step) const
    {
        const float p = (0.5f * most - 0.5f * l) * (float)(fractions * 0.5);
        return !(p < (float)step - 0.135f) && (!(p > (float)step + 0.885f) || fractions >= 1e30);
    }
    __device__ __forceinline__ double exponent(float l) const { return l == most ? 0.0 : ((double)l - (double)most) * inverse; }
};

// The element at which a target is reached: its key and index, and the sum of the order up to it, itself among them.
struct Found {
    uint32_t key, index;
    u64 sum;
};

// A thread's four steps of the histogram: the sum of all steps before them, and the sums up to each.
struct Running {
    u64 before, upto[kPerThread];
};

struct Shared {
    u64 sum[kSteps];
    u64 near_[kNear];                              // (key, ~index): in the order where larger comes first
    u64 member[kMembers], member_weight[kMembers];
    uint32_t count[kSteps];
    double table[kFractions];                      // 2^(i / 256)
    u64 wave_sum[kWaves];
    uint32_t wave_count[kWaves];
    float wave_most[kWaves], wave_total[kWaves], wave_square[kWaves], wave_number[kWaves];
    u64 digit_sum[256];
    uint32_t digit_count[256];
    int step;
    uint32_t members, near_count;
    Found found;
    u64 before_sum, total, least_sum;
    uint32_t before_count, digit;
};

// A row of logits, or a part of it, read by its 16-byte pieces (the first and the last may be part of it only: read by elements).
template <typename T>
struct Row {
    static constexpr int kPiece = 16 / sizeof(T), kAtOnce = 16 / kPiece;
    const T *first;           // where the piece lies that the row begins in
    int skip, vocab;
    int begin, past;          // the pieces of this part

    __device__ __forceinline__ Row(const T *row, int vocab_, int part, int parts) : vocab(vocab_)
    {
        skip = (int)(((uintptr_t)row & 15u) / sizeof(T));
        first = row - skip;
        const int pieces = (skip + vocab + kPiece - 1) / kPiece, own = (pieces + parts - 1) / parts;
        begin = min(part * own, pieces);
        past = min(begin + own, pieces);
    }
    __device__ __forceinline__ bool whole(int piece) const { return piece * kPiece >= skip && (piece + 1) * kPiece <= skip + vocab; }
    // f(piece, its 16 bytes, whether all of them are the row's): whole pieces, several at a time, then what the row's ends have of theirs.
    // AHEAD: the next ones are asked for while some are looked at, which pays where that is much work (the histogram's pass; a survey of 128
    // rows of 131072 takes 15 us so, and 13 without).
    template <bool AHEAD, typename F>
    __device__ __forceinline__ void raw_pieces(F f) const
    {
        if (begin == past) return;
        const int from = begin + (whole(begin) ? 0 : 1), to = past - (whole(past - 1) ? 0 : 1);
        const u32x4 *pieces = (const u32x4 *)first;
        int p0 = from + threadIdx.x, end = threadIdx.x == 0 && from > begin ? begin : threadIdx.x == 1 && to < past && past - 1 > begin ? past - 1 : -1;
        // (a row of one piece that is not whole: the first thread's)
        if (past - 1 == begin && threadIdx.x == 1) end = -1;
        u32x4 ahead[kAtOnce];
        auto ask = [&](u32x4 (&into)[kAtOnce]) {
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (p0 + u * kThreads < to) into[u] = pieces[p0 + u * kThreads];
        };
        if constexpr (AHEAD) ask(ahead);
        while (true) {
            u32x4 raw[kAtOnce];
            int number = 0, base = p0;
            const bool inside = p0 < to;
            if (inside) {
                number = min((to - p0 + kThreads - 1) / kThreads, kAtOnce);
                if constexpr (AHEAD) {
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u) raw[u] = ahead[u];
                } else {
                    ask(raw);
                }
                p0 += kAtOnce * kThreads;
                if constexpr (AHEAD) ask(ahead);
            } else if (end >= 0) {
                T part[kPiece];
#pragma unroll
                for (int e = 0; e < kPiece; ++e) {
                    const int i = end * kPiece + e;
                    part[e] = i >= skip && i < skip + vocab ? first[i] : (T)0;
                }
                raw[0] = __builtin_bit_cast(u32x4, part);
                number = 1;
                base = end;
                end = -1;
            } else {
                break;
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (u < number) f(base + u * kThreads, raw[u], inside);
        }
    }
    // f(logits of a piece, index of the first): elements outside of the row as -inf
    template <typename F>
    __device__ __forceinline__ void visit(int piece, const u32x4 &raw, bool inside, F f) const
    {
        struct Part { T v[kPiece]; };
        const Part part = __builtin_bit_cast(Part, raw);
        const int i = piece * kPiece - skip;
        float l[kPiece];
#pragma unroll
        for (int e = 0; e < kPiece; ++e) l[e] = logit_of(part.v[e]);
        if (!inside) {
#pragma unroll
            for (int e = 0; e < kPiece; ++e) l[e] = i + e >= 0 && i + e < vocab ? l[e] : -INFINITY;
        }
        f(l, i);
    }
    template <bool AHEAD, typename F>
    __device__ __forceinline__ void by_pieces(F f) const
    {
        raw_pieces<AHEAD>([&](int piece, const u32x4 &raw, bool inside) { visit(piece, raw, inside, f); });
    }
    template <typename F>
    __device__ __forceinline__ void for_each(F f) const
    {
        by_pieces<false>([&](const float (&l)[kPiece], int i) {
#pragma unroll
                for (int e = 0; e < kPiece; ++e) f(l[e], (uint32_t)(i + e));
        });
    }
    __device__ __forceinline__ float at(int i) const { return logit_of(first[skip + i]); }
};

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t from_lane(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}

// The sum over a wave's lanes up to this one.
template <typename N>
__device__ __forceinline__ N wave_scan(N v)
{
    auto add = [&](auto ctrl, auto rows) {
        constexpr int C = decltype(ctrl)::value, R = decltype(rows)::value;
        if constexpr (sizeof(N) == 8) v += (u64)from_lane<C, R>((uint32_t)(v >> 32)) << 32 | from_lane<C, R>((uint32_t)v);
        else v += from_lane<C, R>(v);
    };
    using std::integral_constant;
    constexpr integral_constant<int, 0xf> all{};
    add(integral_constant<int, 0x111>(), all);   // row_shr:1, 2, 4, 8
    add(integral_constant<int, 0x112>(), all);
    add(integral_constant<int, 0x114>(), all);
    add(integral_constant<int, 0x118>(), all);
    add(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());   // row_bcast:15 to rows 1 and 3
    add(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());   // row_bcast:31 to rows 2 and 3
    return v;
}

// Sums over the threads before this one; returns the sum of all.
template <typename N>
__device__ N exclusive_scan(Shared &s, N &value)
{
    N *waves = sizeof(N) == 8 ? (N *)s.wave_sum : (N *)s.wave_count;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const N v = wave_scan(value);
    __syncthreads();
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    value = v - value;
    N all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const N its = waves[i];
        value += i < wave ? its : 0;
        all += its;
    }
    return all;
}

// What is rarely called for stands in functions of its own: the kernel's instructions are all fetched anew for every row.

// Counts by steps (where they are not there yet) and the sum of weights of at least `least`, over all of a row.
template <typename T>
__device__ __noinline__ void count_row(Shared *s, const Row<T> row, const Scale scale, bool count, u64 least)
{
    u64 sum = 0;
    row.for_each([&](float l, uint32_t) {
        u64 w;
        int step;
        if (!scale.weight(l, s->table, w, step)) return;
        if (count) atomicAdd(&s->count[step], 1u);
        sum += w >= least ? w : 0;
    });
    sum = wave_scan(sum);
    if ((threadIdx.x & 63) == 63 && sum) atomicAdd(&s->least_sum, sum);
}

// The element of a step at which a target is reached where the step has too many to be held against each other: by the digits, of eight bits,
// of the key, then by index.
template <typename T>
__device__ __noinline__ void reach_by_digits(Shared *sp, const Row<T> row, const Scale scale, int step, uint32_t before_count, u64 before_sum, bool by_sum,
                                             uint32_t count, u64 sum)
{
    Shared &s = *sp;
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (tid < 256) {
            s.digit_count[tid] = 0;
            s.digit_sum[tid] = 0;
        }
        __syncthreads();
        row.for_each([&](float l, uint32_t) {
            const uint32_t key = key_of(l);
            u64 w;
            int its;
            if (!scale.weight(l, s.table, w, its) || its != step || (shift < 24 && key >> (shift + 8) != prefix)) return;
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
    u64 w;
    int unused;
    scale.weight(logit_of_key(prefix), s.table, w, unused);
    const uint32_t place = by_sum ? (uint32_t)((sum - before_sum + w - 1) / w) : count - before_count;   // 1 for the first
    const int own = (row.vocab + kThreads - 1) / kThreads, first = min(tid * own, row.vocab), past = min(first + own, row.vocab);
    uint32_t c = 0;
    for (int i = first; i < past; ++i) c += key_of(row.at(i)) == prefix;
    uint32_t ahead = c;
    exclusive_scan(s, ahead);
    if (ahead < place && ahead + c >= place) {
        uint32_t at = ahead;
        for (int i = first; i < past; ++i)
            if (key_of(row.at(i)) == prefix && ++at == place) s.found = {prefix, (uint32_t)i, before_sum + place * w};
    }
    __syncthreads();
}

// The first element of the order at which the running count is at least `count` (by_sum false; s.count holds the steps' counts) or the
// running sum at least `sum`; the row holds one.
template <typename T>
__device__ __forceinline__ Found reach(Shared &s, const Row<T> &row, const Scale &scale, const Running &run, bool by_sum, uint32_t count, u64 sum)
{
    const int tid = threadIdx.x;
    if (by_sum) {
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const u64 w0 = i > 0 ? run.upto[i - 1] : run.before;
            if (w0 < sum && run.upto[i] >= sum) {
                s.step = tid * kPerThread + i;
                s.before_count = 0;
                s.before_sum = w0;
            }
        }
    } else {
        uint32_t c[kPerThread], all = 0;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) all += c[i] = s.count[tid * kPerThread + i];
        uint32_t c0 = all;
        exclusive_scan(s, c0);
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            if (c0 < count && c0 + c[i] >= count) {
                s.step = tid * kPerThread + i;
                s.before_count = c0;
                s.before_sum = i > 0 ? run.upto[i - 1] : run.before;
            }
            c0 += c[i];
        }
    }
    if (tid == 0) s.members = 0;
    __syncthreads();
    const int step = s.step;
    uint32_t before_count = s.before_count;
    u64 before_sum = s.before_sum;
    auto candidate = [&](u64 entry) {
        const uint32_t at = atomicAdd(&s.members, 1u);
        if (at < (uint32_t)kMembers) s.member[at] = entry;
    };
    if (step < scale.near_steps && s.near_count <= (uint32_t)kNear)
        for (uint32_t i = tid; i < s.near_count; i += kThreads) {
            const u64 entry = s.near_[i];
            if (scale.near_step(logit_of_key((uint32_t)(entry >> 32)), step)) candidate(entry);
        }
    else row.template by_pieces<false>([&](const float (&l)[Row<T>::kPiece], int i) {
#pragma unroll
        for (int e = 0; e < Row<T>::kPiece; ++e)
            if (scale.near_step(l[e], step)) candidate((u64)key_of(l[e]) << 32 | (uint32_t)~(uint32_t)(i + e));
    });
    __syncthreads();
    const uint32_t candidates = s.members;
    if (candidates > (uint32_t)kMembers) {
        reach_by_digits(&s, row, scale, step, before_count, before_sum, by_sum, count, sum);
        return s.found;
    }
    // A candidate a thread: its weight, and the 256th of the step that it is in (-1: it is of another step).
    u64 mine = 0, own = 0;
    int part = -1;
    if (tid < (int)candidates) {
        mine = s.member[tid];
        const float l = logit_of_key((uint32_t)(mine >> 32));
        int its;
        // (the step's places lie between 4 * step - 2 and 4 * step + 6 below 0; an infinite logit's is none)
        if (scale.weight(l, s.table, own, its) && its == step)
            part = min(max((int)((-scale.place(l) - (4 * step - 2)) * 32.0), 0), 255);
    }
    const bool many = candidates > 64;   // a 256th of the step first: each of its members is held against the others
    if (many && tid < 256) {
        s.digit_count[tid] = 0;
        s.digit_sum[tid] = 0;
    }
    __syncthreads();
    if (many) {
        if (part >= 0) {
            atomicAdd(&s.digit_count[part], 1u);
            atomicAdd(&s.digit_sum[part], own);
        }
        __syncthreads();
        if (tid < 64) {
            uint32_t c[4], all_c = 0;
            u64 w[4], all_w = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                all_c += c[i] = s.digit_count[4 * tid + i];
                all_w += w[i] = s.digit_sum[4 * tid + i];
            }
            uint32_t at_c = before_count + wave_scan(all_c) - all_c;
            u64 at_w = before_sum + wave_scan(all_w) - all_w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (by_sum ? at_w < sum && at_w + w[i] >= sum : at_c < count && at_c + c[i] >= count) {
                    s.digit = 4 * tid + i;
                    s.before_count = at_c;
                    s.before_sum = at_w;
                }
                at_c += c[i];
                at_w += w[i];
            }
        }
        __syncthreads();
        before_count = s.before_count;
        before_sum = s.before_sum;
        if (part != (int)s.digit) part = -1;
    }
    if (tid == 0) s.members = 0;
    __syncthreads();
    if (part >= 0) {
        const uint32_t at = atomicAdd(&s.members, 1u);
        s.member[at] = mine;
        s.member_weight[at] = own;
    }
    __syncthreads();
    const uint32_t rivals = s.members;
    if (part >= 0) {
        uint32_t c = before_count + 1;
        u64 w = before_sum + own;
        for (uint32_t j = 0; j < rivals; ++j) {
            const bool ahead = s.member[j] > mine;
            c += ahead;
            w += ahead ? s.member_weight[j] : 0;
        }
        if (by_sum ? w >= sum && w - own < sum : c == count) s.found = {(uint32_t)(mine >> 32), (uint32_t)~mine, w};
    }
    __syncthreads();
    return s.found;
}

// What is asked of a row.
struct Asked {
    float t, p, least;
    bool greedy;
    int k;
    __device__ __forceinline__ Asked(const Args &a, int r)
    {
        t = a.temperature ? a.temperature[r] : 1.0f;
        p = a.top_p ? a.top_p[r] : 1.0f;
        const float m = a.min_p ? a.min_p[r] : 0.0f;
        greedy = !(t > 0.0f);
        k = greedy ? 1 : a.top_k ? a.top_k[r] : 0;
        least = m > 0.0f ? fminf(m, 1.0f) : 0.0f;
    }
};

// Some of a row's logits: the largest of all, and sums, of them and of their squares, and number of those looked at.
struct Survey {
    float most, total, square, number;
};

// Tokens near the largest logit are kept by themselves, so that a target that is reached among them needs no further look at the row.  They are
// those within a share of the distance from the mean to the largest, or so many standard deviations above the mean, whichever takes in
// more: some 1500 of normally distributed logits, whether or not others stand far above them.  (Rows with more of them than there is
// room for are looked at again instead, which costs time only.)  A greedy row: its weights are of no account, the first of its largest
// logits is.  An endless temperature: all that is not -inf weighs the same.
__device__ __forceinline__ Scale scale_of(const Args &a, const Asked &ask, const Survey &v)
{
    Scale s;
    s.most = v.most;
    s.origin = fmin((double)v.most, 0x1p128);
    s.inverse = ask.greedy ? 1e30 : ask.t == INFINITY ? 1e-300 : 1.0 / (double)ask.t;
    s.fractions = v.most == INFINITY ? 1e300 : s.inverse * (kFractions * 1.4426950408889634);
    s.bits = a.bits;
    s.least = -(double)(kFractions * (a.bits + 2));
    const float mean = v.total / v.number, spread = sqrtf(fmaxf(v.square / v.number - mean * mean, 0.0f));
    const float reach = fmaxf((v.most - mean) * a.near_share, v.most - mean - a.near_spread * spread);
    const float near_ = reach * (float)fmin(s.fractions * 0.25, 1e30);
    s.near_steps = min(near_ < (float)kSteps ? (int)fmaxf(near_, 0.0f) + 1 : kSteps, 64 * (a.bits + 1) + 1);   // (none without a weight)
    return s;
}

// Over the lanes of a wave: xor 1 and 2 inside quads, the mirrored quad and half of each row of 16, then the four rows.
template <typename F>
__device__ __forceinline__ float over_wave(float v, F op)
{
    auto other = [](float x, auto ctrl) {
        const int i = __builtin_bit_cast(int, x);
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, decltype(ctrl)::value, 0xf, 0xf, false));
    };
    v = op(v, other(v, std::integral_constant<int, 0xb1>()));    // quad_perm [1,0,3,2]
    v = op(v, other(v, std::integral_constant<int, 0x4e>()));    // quad_perm [2,3,0,1]
    v = op(v, other(v, std::integral_constant<int, 0x141>()));   // row_half_mirror
    v = op(v, other(v, std::integral_constant<int, 0x140>()));   // row_mirror
    const int i = __builtin_bit_cast(int, v);
    auto row = [&](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, lane)); };
    return op(op(row(0), row(16)), op(row(32), row(48)));
}

// The largest of a piece's logits (a maximum passes over NaN).
template <typename T>
__device__ __forceinline__ float largest_of(const u32x4 &raw)
{
    if constexpr (sizeof(T) == 4) {
        const f32x4 l = __builtin_bit_cast(f32x4, raw);
        return fmaxf(fmaxf(l.x, l.y), fmaxf(l.z, l.w));
    } else if constexpr (std::is_same_v<T, _Float16>) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        auto pair = [](uint32_t w) { return __builtin_bit_cast(f16x2, w); };
        const f16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(pair(raw.x), pair(raw.y)), __builtin_elementwise_max(pair(raw.z), pair(raw.w)));
        return fmaxf((float)m.x, (float)m.y);
    } else {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(__builtin_bit_cast(float, raw[i] << 16), __builtin_bit_cast(float, raw[i] & 0xffff0000u)));
        return m;
    }
}

// The largest logit of (a part of) a row, and sums and number of the finite ones among the first of every piece.
template <typename T>
__device__ Survey survey(Shared &s, const Row<T> &row)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float most = -INFINITY, total = 0.0f, square = 0.0f, number = 0.0f;
    row.template raw_pieces<false>([&](int piece, const u32x4 &raw, bool inside) {
        if (inside) {
            const float first = logit_of(*(const T *)&raw);
            most = fmaxf(most, largest_of<T>(raw));
            total += fabsf(first) < INFINITY ? first : 0.0f;
            square += fabsf(first) < INFINITY ? first * first : 0.0f;
            number += fabsf(first) < INFINITY ? 1.0f : 0.0f;
        } else {
            row.visit(piece, raw, false, [&](const float (&l)[Row<T>::kPiece], int) {
#pragma unroll
                for (int e = 0; e < Row<T>::kPiece; ++e) most = fmaxf(most, l[e]);
            });
        }
    });
    most = over_wave(most, [](float x, float y) { return fmaxf(x, y); });
    total = over_wave(total, [](float x, float y) { return x + y; });
    square = over_wave(square, [](float x, float y) { return x + y; });
    number = over_wave(number, [](float x, float y) { return x + y; });
    if (lane == 0) {
        s.wave_most[wave] = most;
        s.wave_total[wave] = total;
        s.wave_square[wave] = square;
        s.wave_number[wave] = number;
    }
    __syncthreads();
    Survey v = {most, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        v.most = fmaxf(v.most, s.wave_most[w]);
        v.total += s.wave_total[w];
        v.square += s.wave_square[w];
        v.number += s.wave_number[w];
    }
    return v;
}

__device__ void clear(Shared &s)
{
    for (int b = threadIdx.x; b < kSteps; b += kThreads) {
        s.count[b] = 0;
        s.sum[b] = 0;
    }
    if (threadIdx.x < kFractions) s.table[threadIdx.x] = kTable.power[threadIdx.x];
    if (threadIdx.x == 0) {
        s.least_sum = 0;
        s.near_count = 0;
    }
}

// Sums by steps and the tokens near the largest, of (a part of) a row; counts too where many are asked for.
template <typename T>
__device__ void histogram(Shared &s, const Row<T> &row, const Scale &scale, const Asked &ask)
{
    row.template by_pieces<true>([&](const float (&l)[Row<T>::kPiece], int i) {
        constexpr int P = Row<T>::kPiece;
        u64 w[P];
        int step[P];
#pragma unroll
        for (int e = 0; e < P; ++e) {
            scale.weight(l[e], s.table, w[e], step[e]);
            asm volatile("" : "+v"(w[e]));   // (all formed before the first is put to use)
        }
#pragma unroll
        for (int e = 0; e < P; ++e)
            if (w[e]) atomicAdd(&s.sum[step[e]], w[e]);
        if (ask.k >= kCounted) {
#pragma unroll
            for (int e = 0; e < P; ++e)
                if (w[e]) atomicAdd(&s.count[step[e]], 1u);
        }
#pragma unroll
        for (int e = 0; e < P; ++e)
            if (step[e] < scale.near_steps) {
                const uint32_t at = atomicAdd(&s.near_count, 1u);
                if (at < (uint32_t)kNear) s.near_[at] = (u64)key_of(l[e]) << 32 | (uint32_t)~(uint32_t)(i + e);
            }
    });
}

// The token, from the histogram of the whole row.
template <typename T>
__device__ void choose(const Args &a, Shared &s, const Row<T> &row, const Scale &scale, const Asked &ask, int r)
{
    const int tid = threadIdx.x;
    __syncthreads();
    Running run;
    u64 total;
    {   // running totals
        u64 w[kPerThread], all = 0;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) all += w[i] = s.sum[tid * kPerThread + i];
        run.before = all;
        total = exclusive_scan(s, run.before);
        u64 upto = run.before;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) run.upto[i] = upto += w[i];
    }
    const bool by_count = ask.k > 0 && ask.k < row.vocab, by_least = ask.least > 0.0f;
    uint32_t counted = 0;
    if (by_count || by_least) {
        // Counts and the sum of what min_p leaves, from the tokens near the largest unless very many are asked for.
        const u64 least = by_least ? min((u64)__builtin_ceil((double)ask.least * (double)(1ull << scale.bits)), 1ull << scale.bits) : ~0ull;
        const bool kept = s.near_count <= (uint32_t)kNear, count = by_count && ask.k < kCounted;
        if (kept && (!count || s.near_count >= (uint32_t)ask.k) && (!by_least || -64.0f * log2f(ask.least) + 2.0f < (float)scale.near_steps)) {
            u64 sum = 0;
            for (uint32_t i = tid; i < s.near_count; i += kThreads) {
                u64 w;
                int step;
                if (!scale.weight(logit_of_key((uint32_t)(s.near_[i] >> 32)), s.table, w, step)) continue;
                if (count) atomicAdd(&s.count[step], 1u);
                sum += w >= least ? w : 0;
            }
            sum = wave_scan(sum);
            if ((tid & 63) == 63 && sum) atomicAdd(&s.least_sum, sum);
        } else {
            count_row(&s, row, scale, count, least);
        }
        __syncthreads();
        if (by_count) {
            uint32_t some = 0;
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) some += s.count[tid * kPerThread + i];
            counted = exclusive_scan(s, some);
        }
    }
    float u = a.uniform[r];
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    Found f;
    // The ends of what top_k and top_p leave, then the token.
#pragma nounroll
    for (int turn = by_count && (uint32_t)ask.k <= counted ? 0 : 1; turn < 3; ++turn) {
        u64 target = 0;
        if (turn == 1) {
            if (!(ask.p < 1.0f)) continue;
            const double part = __builtin_ceil((double)fmaxf(ask.p, 0.0f) * (double)total);
            target = part < 1.0 ? 1 : (u64)part;
        } else if (turn == 2) {
            if (by_least) total = min(total, s.least_sum);
            target = min((u64)__builtin_floor((double)u * (double)total), total - 1) + 1;
        }
        f = reach(s, row, scale, run, turn > 0, (uint32_t)ask.k, target);
        if (turn < 2) total = min(total, f.sum);
    }
    if (tid == 0) {
        a.ids[r] = f.index;
        if (a.logprob) a.logprob[r] = ask.greedy ? 0.0f : (float)(scale.exponent(logit_of_key(f.key)) - log((double)total / (double)(1ull << a.bits)));
    }
}

__device__ __forceinline__ void nothing(const Args &a, int r)
{
    if (threadIdx.x != 0) return;
    a.ids[r] = -1;
    if (a.logprob) a.logprob[r] = -INFINITY;
}

// One workgroup per row.
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Args a)
{
    __shared__ Shared s;
    const int r = blockIdx.x;
    const Row<T> row((const T *)a.logits + r * a.row_stride, a.vocab, 0, 1);
    const Asked ask(a, r);
    clear(s);
    const Survey v = survey(s, row);
    if (v.most == -INFINITY) return nothing(a, r);
    const Scale scale = scale_of(a, ask, v);
    histogram(s, row, scale, ask);
    choose(a, s, row, scale, ask, r);
}

// The same by several workgroups a row, where rows are few: a launch that looks for the largest logit (and clears what the next one
// adds to), one that adds up histograms, one that chooses.
template <typename T>
__global__ void __launch_bounds__(kThreads) survey_kernel(const Args a)
{
    __shared__ Shared s;
    const int r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    RowWork &work = a.work[r];
    const Row<T> row((const T *)a.logits + r * a.row_stride, a.vocab, part, a.parts);
    for (int b = part * kThreads + threadIdx.x; b < kSteps; b += a.parts * kThreads) {
        work.sum[b] = 0;
        work.count[b] = 0;
    }
    const Survey v = survey(s, row);
    if (threadIdx.x != 0) return;
    work.most[part] = v.most;
    work.total[part] = v.total;
    work.square[part] = v.square;
    work.number[part] = v.number;
    if (part == 0) work.near_count = 0;
}

__device__ __forceinline__ bool scale_of_row(const Args &a, const Asked &ask, const RowWork &work, Scale &scale)
{
    Survey v = {-INFINITY, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < a.parts; ++i) {
        v.most = fmaxf(v.most, work.most[i]);
        v.total += work.total[i];
        v.square += work.square[i];
        v.number += work.number[i];
    }
    scale = scale_of(a, ask, v);
    return v.most > -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) histogram_kernel(const Args a)
{
    __shared__ Shared s;
    const int tid = threadIdx.x, r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    RowWork &work = a.work[r];
    const Row<T> row((const T *)a.logits + r * a.row_stride, a.vocab, part, a.parts);
    const Asked ask(a, r);
    Scale scale;
    if (!scale_of_row(a, ask, work, scale)) return;
    clear(s);
    __syncthreads();
    histogram(s, row, scale, ask);
    __syncthreads();
    for (int b = tid; b < kSteps; b += kThreads) {
        const u64 w = s.sum[b];
        if (w) atomicAdd(&work.sum[b], w);
        const uint32_t c = s.count[b];
        if (c) atomicAdd(&work.count[b], c);
    }
    const uint32_t own = s.near_count;
    if (tid == 0) {
        s.members = own ? atomicAdd(&work.near_count, own) : 0;
        if (part == 0) work.near_steps = scale.near_steps;   // (handed on, not formed again: the list holds these steps and no others)
    }
    __syncthreads();
    for (uint32_t i = tid; i < own && s.members + i < (uint32_t)kNear && i < (uint32_t)kNear; i += kThreads) work.near_[s.members + i] = s.near_[i];
}

template <typename T>
__global__ void __launch_bounds__(kThreads) choose_kernel(const Args a)
{
    __shared__ Shared s;
    const int tid = threadIdx.x, r = blockIdx.x;
    const RowWork &work = a.work[r];
    const Row<T> row((const T *)a.logits + r * a.row_stride, a.vocab, 0, 1);
    const Asked ask(a, r);
    // (all that may be wanted is asked for at once, before anything is known of the row: entries of the list that are not there have no meaning)
    constexpr int kSome = 2;
    u64 sums[kPerThread], some[kSome];
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) sums[i] = work.sum[tid + i * kThreads];
#pragma unroll
    for (int i = 0; i < kSome; ++i) some[i] = work.near_[tid + i * kThreads];
    const uint32_t listed = work.near_count;
    const int listed_steps = work.near_steps;
    const double power = tid < kFractions ? kTable.power[tid] : 0.0;
    Scale scale;
    if (!scale_of_row(a, ask, work, scale)) return nothing(a, r);
    scale.near_steps = listed_steps;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        s.sum[tid + i * kThreads] = sums[i];
        s.count[tid + i * kThreads] = ask.k >= kCounted ? work.count[tid + i * kThreads] : 0;
    }
#pragma unroll
    for (int i = 0; i < kSome; ++i) s.near_[tid + i * kThreads] = some[i];
    if (listed <= (uint32_t)kNear)
        for (uint32_t i = tid + kSome * kThreads; i < listed; i += kThreads) s.near_[i] = work.near_[i];
    if (tid < kFractions) s.table[tid] = power;
    if (tid == 0) {
        s.near_count = listed;
        s.least_sum = 0;
    }
    choose(a, s, row, scale, ask, r);
}

int launch_status()
{
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? LUTGEMM_OK : lutgemm_internal_hip_fail((int)e);
}

// The share of the distance from the mean to the largest of normally distributed logits above which 1500 of them lie, and the standard
// deviations above the mean (the normal distribution's quantile, Abramowitz and Stegun 26.2.22).
float near_spread(int vocab)
{
    if (vocab <= kNear) return -1e30f;   // (all of them)
    const float share = 1500.0f / vocab;
    const float t = sqrtf(-2.0f * logf(share < 0.5f ? share : 0.5f));
    return t - (2.30753f + 0.27061f * t) / (1.0f + 0.99229f * t + 0.04481f * t * t);
}

float near_share(int vocab)
{
    return vocab <= kNear ? 1.0f : 1.0f - near_spread(vocab) / sqrtf(2.0f * logf((float)vocab));
}

// Workgroups that share a row, in three launches instead of one: where rows leave CUs idle and are long enough to pay for the two more
// launches and for the addition of histograms, which takes longer the more of them there are.  With all filters, one workgroup against as many as
// here: one row of 16384 22.2 and 25.8 us, of 32000 28.2 and 26.2; 8 rows of 50272 34.7 and 27.3, 64 35.4 and 32.4; 64 rows of 131072 63.3
// and 40.3, 128 66.2 and 54.3.
int parts_of(int rows, int vocab)
{
    if (vocab < 28000) return 1;
    return rows <= 16 ? 8 : rows <= 64 ? 4 : rows <= 128 ? 2 : 1;
}

bool sizes_fit(int rows, int vocab) { return rows >= 1 && rows <= 65535 && vocab >= 1 && vocab <= 1 << 20; }

}  // namespace

extern "C" {

size_t lutgemm_sampling_workspace(int rows, int vocab)
{
    if (!sizes_fit(rows, vocab)) return 0;
    return parts_of(rows, vocab) > 1 ? rows * sizeof(RowWork) : 16;
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
    const int bits = 63 - doublings < 51 ? 63 - doublings : 51;
    Args a{};
    a.logits = c->logits;
    a.row_stride = c->row_stride;
    a.rows = c->rows;
    a.vocab = c->vocab;
    a.bits = bits;
    a.parts = parts_of(c->rows, c->vocab);
    a.near_share = near_share(c->vocab);
    a.near_spread = near_spread(c->vocab);
    a.temperature = c->temperature;
    a.top_k = c->top_k;
    a.top_p = c->top_p;
    a.min_p = c->min_p;
    a.uniform = c->uniform;
    a.ids = c->ids;
    a.logprob = c->logprob;
    a.work = (RowWork *)workspace;
    const hipStream_t hs = (hipStream_t)stream;
    auto launch = [&](auto type) {
        typedef decltype(type) T;
        const dim3 rows((unsigned)c->rows), parts((unsigned)(c->rows * a.parts)), threads(kThreads);
        if (a.parts == 1) {
            hipLaunchKernelGGL(sample_kernel<T>, rows, threads, 0, hs, a);
            return launch_status();
        }
        hipLaunchKernelGGL(survey_kernel<T>, parts, threads, 0, hs, a);
        int status = launch_status();
        if (status != LUTGEMM_OK) return status;
        hipLaunchKernelGGL(histogram_kernel<T>, parts, threads, 0, hs, a);
        status = launch_status();
        if (status != LUTGEMM_OK) return status;
        hipLaunchKernelGGL(choose_kernel<T>, rows, threads, 0, hs, a);
        return launch_status();
    };
    if (c->logits_type == LUTGEMM_TYPE_F16) return launch(_Float16());
    if (c->logits_type == LUTGEMM_TYPE_BF16) return launch(uint16_t());
    return launch(float());
}

}  // extern "C"
