// Attention over a cache of keys and values held in 4 bits, gfx950: appending of new tokens, attention of one or many query
// rows, joining of what workgroups found over different positions.  The layout and the rules of rounding are in lutgemm_gfx950.h.
//
// Mathematics.  For a (sequence, kv head) pair the query rows are (token, query head) pairs, row = token * rep + member.
// Scores are formed transposed, S^T = K Q^T: the matrix instruction's A operand is 16 positions of keys, B 16 query rows, so
// that a lane ends up with one query row (lane % 16) and four positions of either half of a block of 32.  Those eight weights
// are, as they are, the B operand of O^T = V^T P^T when the values of a block are stored with the positions in that order,
// eight to a word: no value crosses lanes between the two products, and what a row is rescaled by is a lane's own scalar.
// A held value is one fp16 number, fp16(minimum + scale * code); it is formed in registers (a shift, and-or, an exact
// subtraction and an fma for two values) and multiplied exactly, sums in fp32.
// Softmax keeps a reference per row, not the exact maximum: it is raised only when a score exceeds it by 2^8, so that most
// blocks need no exchange between lanes.  Weights are held 2^7 times as large (which cancels in every quotient), so that they take up fp16's range
// where they are rounded for the matrix product: 2^15 at most, half a step (2^-11 relative) down to 2^-21 of the reference's weight, 2^-32 of
// that below: 2^20 such positions come to 2^-12 of the largest weight.  (With the reference's weight at one, the tail of a row with a
// dominant position was lost: 8192 positions at 2^-26 each came out as nothing.)  The error of a sum over many positions averages out.  Their sum is
// formed in fp32 from the unrounded ones.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "lutgemm_gfx950.h"
#include "lutgemm_common.h"
#include "lutgemm_internal.h"

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kBlock = 32;              // positions of a block of the cache
constexpr float kLargest = 60000.0f;    // of a held number
constexpr float kSlack = 8.0f;          // by which (in powers of two) a score may exceed its row's reference
constexpr float kLift = 7.0f;           // by which weights are held larger

struct Args {
    uint8_t *cache;
    const _Float16 *q, *k, *v, *cos_t, *sin_t;
    const int64_t *start;
    const int32_t *counts;
    _Float16 *out, *k_held, *v_held;
    int64_t q_stride[2], k_stride[2], v_stride[2];
    int tokens, heads, kv_heads, rep, max_positions, blocks;   // blocks: of a (sequence, kv head) pair in the cache
    int pairs, units, tiles, splits;                           // units: tiles of a wave's rows; tiles: of a workgroup's
    int fused;                                                 // the attention launch appends
    float *partial;                                            // [split][pair][unit][rows][head_dim], then ...
    float2 *stats;                                             // ... (reference, sum) [split][pair][unit][rows]
};

// A sequence's new tokens: the first one's position and how many there are (0: all are passed over).
__device__ __forceinline__ int live_tokens(const Args &a, int b, int &start)
{
    const int64_t s = a.start[b];
    int n = a.counts ? a.counts[b] : a.tokens;
    n = min(max(n, 0), a.tokens);
    start = 0;
    if (s < 0 || s >= a.max_positions) return 0;
    start = (int)s;
    return min(n, a.max_positions - start);
}

// Eight numbers at dimensions d .. d + 7 of a head, rotated by the angles of a position and rounded to fp16.
__device__ __forceinline__ f16x8 rotated(const _Float16 *head, const _Float16 *cos_row, const _Float16 *sin_row, int d, int hd)
{
    const int half = hd / 2;
    const f16x8 x = *(const f16x8 *)(head + d), y = *(const f16x8 *)(head + (d < half ? d + half : d - half));
    const f16x8 c = *(const f16x8 *)(cos_row + d), s = *(const f16x8 *)(sin_row + d);
    const float sign = d < half ? -1.0f : 1.0f;
    f16x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // (products of fp16 numbers are exact in fp32; the sum is rounded to fp32 and then to fp16, as framework operations round it:
        // without the empty statement one instruction would round once)
        float sum = (float)x[i] * (float)c[i] + sign * (float)y[i] * (float)s[i];
        asm volatile("" : "+v"(sum));
        r[i] = (_Float16)sum;
    }
    return r;
}

// What a group of 32 numbers is held as, by the four neighbouring lanes that have eight each.
struct Held {
    _Float16 scale, low;
    uint32_t codes;   // of this lane's numbers, 4 bits each, number i at bit 4 i
    f16x8 value;
};

__device__ __forceinline__ Held quantise(f16x8 x)
{
    Held h;
    float f[8], low = kLargest, high = -kLargest;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = (float)x[i];
        f[i] = v != v ? 0.0f : fminf(fmaxf(v, -kLargest), kLargest);
        low = fminf(low, f[i]);
        high = fmaxf(high, f[i]);
    }
#pragma unroll
    for (int m = 1; m < 4; m *= 2) {
        low = fminf(low, __shfl_xor(low, m));
        high = fmaxf(high, __shfl_xor(high, m));
    }
    h.low = (_Float16)low;   // (exact: one of the numbers, or +-60000)
    h.scale = (_Float16)(float)(((double)high - (double)low) / 15.0);
    const float inverse = (float)h.scale > 0.0f ? 1.0f / (float)h.scale : 0.0f;
    h.codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // The nearest code, exactly: the quotient in fp32 is off by less than 2^-17 (two roundings and the inverse's, of at most 15.01);
        // where that might decide, what is left over is compared in 64 bits, where it is exact.
        const float quotient = (f[i] - low) * inverse;
        int c = (int)fminf(rintf(quotient), 15.0f);
        if (fabsf(fabsf(quotient - (float)c) - 0.5f) < 0x1p-16f && h.scale > (_Float16)0.0f) {
            const double s = (double)(float)h.scale, rest = ((double)f[i] - (double)low) - c * s;
            if (2.0 * rest > s || (2.0 * rest == s && (c & 1))) ++c;
            else if (-2.0 * rest > s || (-2.0 * rest == s && (c & 1))) --c;
            c = min(max(c, 0), 15);
        }
        h.codes |= (uint32_t)c << (4 * i);
        h.value[i] = __builtin_fmaf16((_Float16)(float)c, h.scale, h.low);
    }
    return h;
}

// The word in which eight codes are kept, from them in order: even ones in the low half.
__device__ __forceinline__ uint32_t word_of(uint32_t codes)
{
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= ((codes >> (4 * e)) & 15u) << (4 * (e / 2) + 16 * (e & 1));
    return w;
}

// Four codes of 4 bits each as bytes.
__device__ __forceinline__ uint32_t bytes_of(uint32_t codes)
{
    const uint32_t pairs = (codes & 0xffu) | (codes & 0xff00u) << 8;
    return (pairs & 0x000f000fu) | (pairs & 0x00f000f0u) << 4;
}

// Rows of the held values of tokens first .. past - 1 that are passed over: zeros.
template <int HD, int THREADS>
__device__ __forceinline__ void clear_held(const Args &a, int b, int kvh, int n, int first, int past)
{
    if (!a.k_held && !a.v_held) return;
    for (int u = threadIdx.x; u < (past - first) * (HD / 8); u += THREADS) {
        const int token = first + u / (HD / 8);
        if (token < n) continue;
        const size_t at = (((size_t)b * a.tokens + token) * a.kv_heads + kvh) * HD + u % (HD / 8) * 8;
        if (a.k_held) *(u32x4 *)(a.k_held + at) = (u32x4){0, 0, 0, 0};
        if (a.v_held) *(u32x4 *)(a.v_held + at) = (u32x4){0, 0, 0, 0};
    }
}

// The new tokens of a (sequence, kv head) pair whose positions lie in a block of the cache, by a workgroup of THREADS that alone writes the
// block, so that words that hold other positions too can be read, changed and written.  Lanes 4 i .. 4 i + 3 take a group of 32 numbers; the
// values' codes meet by positions in LDS (`code`: kBlock rows of HD + 4 bytes).
template <int G, int THREADS>
__device__ void append_block(const Args &a, int b, int kvh, int pair, int start, int n, int block, uint8_t *code)
{
    constexpr int HD = 32 * G, kStride = HD + 4, kWords = (128 * G + THREADS - 1) / THREADS;
    const int tid = threadIdx.x;
    const int first = block * kBlock - start;   // token of the block's first position
    const int from = max(0, -first), past = min(kBlock, n - first);
    uint8_t *base = a.cache + ((size_t)pair * a.blocks + block) * (size_t)(1280 * G);
    uint32_t *k_codes = (uint32_t *)base;
    uint32_t *k_scales = (uint32_t *)(base + 512 * G);
    uint32_t *v_codes = (uint32_t *)(base + 640 * G);
    _Float16 *v_scales = (_Float16 *)(base + 1152 * G);
    const bool whole = past - from == kBlock;
    uint32_t before[kWords];   // (asked for ahead)
#pragma unroll
    for (int i = 0; i < kWords; ++i) before[i] = !whole && tid + i * THREADS < 128 * G ? v_codes[tid + i * THREADS] : 0;

    for (int u = tid; u < (past - from) * G * 4; u += THREADS) {
        const int quad = u % 4, t = u / 4 % G, p = from + u / (4 * G), token = first + p, d = 32 * t + 8 * quad;
        const _Float16 *kh = a.k + b * a.k_stride[0] + token * a.k_stride[1] + (size_t)kvh * HD;
        const _Float16 *vh = a.v + b * a.v_stride[0] + token * a.v_stride[1] + (size_t)kvh * HD;
        const size_t angle = (size_t)(start + token) * HD;
        const f16x8 v = *(const f16x8 *)(vh + d);
        const Held hk = quantise(rotated(kh, a.cos_t + angle, a.sin_t + angle, d, HD)), hv = quantise(v);
        k_codes[(p * 4 + quad) * G + t] = word_of(hk.codes);
        *(uint32_t *)(code + p * kStride + d) = bytes_of(hv.codes);
        *(uint32_t *)(code + p * kStride + d + 4) = bytes_of(hv.codes >> 16);
        if (quad == 0) {
            const f16x2 pair_of = {hk.scale, hk.low};
            k_scales[p * G + t] = __builtin_bit_cast(uint32_t, pair_of);
            const int slot = p % 16 / 4 * 8 + p / 16 * 4 + p % 4;
            v_scales[(2 * t) * kBlock + slot] = hv.scale;
            v_scales[(2 * t + 1) * kBlock + slot] = hv.low;
        }
        const size_t at = (((size_t)b * a.tokens + token) * a.kv_heads + kvh) * HD + d;
        if (a.k_held) *(f16x8 *)(a.k_held + at) = hk.value;
        if (a.v_held) *(f16x8 *)(a.v_held + at) = hv.value;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
        const int u = tid + i * THREADS;
        if (u >= 128 * G) break;
        const int t = u % (2 * G), column = u / (2 * G) % 16, quad = u / (32 * G);
        uint32_t fresh = 0, mask = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int p = 4 * quad + e % 4 + 16 * (e / 4), shift = 4 * (e / 2) + 16 * (e & 1);
            if (p < from || p >= past) continue;
            fresh |= (uint32_t)code[p * kStride + 16 * t + column] << shift;
            mask |= 15u << shift;
        }
        if (mask) v_codes[u] = (before[i] & ~mask) | fresh;
    }
}

// The new tokens of prompts: one workgroup per block of the cache that they fall into, a thread for eight numbers of a token's key and value
// (two prompts of 2048 on 8 kv heads: 39 MB in 14 us; 256 threads, which take two turns, 15.5).
constexpr int append_threads(int groups) { return groups >= 4 ? 512 : 256; }

template <int G>
constexpr int kAppendThreads = append_threads(G);

template <int G>
__global__ void __launch_bounds__(kAppendThreads<G>) append_kernel(const Args a)
{
    __shared__ __attribute__((aligned(4))) uint8_t code[kBlock * (32 * G + 4)];
    const int pair = blockIdx.x % a.pairs, part = blockIdx.x / a.pairs;
    const int b = pair / a.kv_heads, kvh = pair % a.kv_heads;
    int start;
    const int n = live_tokens(a, b, start);
    clear_held<32 * G, kAppendThreads<G>>(a, b, kvh, n, min(part * kBlock, a.tokens), min((part + 1) * kBlock, a.tokens));
    const int block = start / kBlock + part;
    if (n > 0 && block * kBlock < start + n) append_block<G, kAppendThreads<G>>(a, b, kvh, pair, start, n, block, code);
}

// Two held values from bits 4 I .. of either half of a word (I = 0, 1): the code, put into the low bits of the significand of 1024 (64), is
// 1024 + code (64 + code) as it stands.
template <int I>
__device__ __forceinline__ f16x2 code_pair(uint32_t w)
{
    const uint32_t bits = I == 0 ? (w & 0x000f000fu) | 0x64006400u : (w & 0x00f000f0u) | 0x54005400u;
    const _Float16 off = I == 0 ? (_Float16)1024.0f : (_Float16)64.0f;
    return __builtin_bit_cast(f16x2, bits) - (f16x2){off, off};
}

__device__ __forceinline__ f16x8 codes_of(uint32_t w)
{
    const uint32_t u = w >> 8;
    const f16x2 p0 = code_pair<0>(w), p1 = code_pair<1>(w), p2 = code_pair<0>(u), p3 = code_pair<1>(u);
    return (f16x8){p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&to)[N], const void *from)
{
    __builtin_memcpy(to, from, 4 * N);
}

// Blocks of a tile that new rows up to position `last` attend to, and how they are shared by the workgroups of its positions.
__device__ __forceinline__ int blocks_per_split(const Args &a, int blocks, int least)
{
    return max((blocks + a.splits - 1) / a.splits, least);
}

// The queries of 16 RT rows from row0 on, as the matrix instruction's B operand, and the last position that each row attends to.  Rows
// behind the last live one repeat it.
template <int G, int RT>
__device__ __forceinline__ void load_queries(const Args &a, int b, int kvh, int start, int row0, int live_rows, f16x8 (&q)[RT][G], int (&limit)[RT])
{
    const int lane = threadIdx.x & 63, column = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = min(row0 + 16 * rt + column, max(live_rows, 1) - 1), token = row / a.rep;
        limit[rt] = start + token;
        const _Float16 *head = a.q + b * a.q_stride[0] + token * a.q_stride[1] + (size_t)(kvh * a.rep + row % a.rep) * (32 * G);
        const size_t angle = (size_t)(start + token) * (32 * G);
#pragma unroll
        for (int t = 0; t < G; ++t) q[rt][t] = rotated(head, a.cos_t + angle, a.sin_t + angle, 32 * t + 8 * quad, 32 * G);
    }
}

// Of one row a lane: the reference (a score), the sum of weights 2^(factor * (score - reference) + kLift), and the weighted values.
template <int G>
struct RowState {
    float reference, sum, off;   // off: kLift - reference * factor, or kLift where scores are brought to the reference ahead (`far`)
    bool far;                    // of the wave: factor * reference is so large in a row that its rounding in `off` would count
    f32x4 acc[2 * G];
    __device__ __forceinline__ void clear(float factor)
    {
        reference = -1e30f;
        sum = 0.0f;
        off = kLift - reference * factor;
        far = false;
#pragma unroll
        for (int t = 0; t < 2 * G; ++t) acc[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    // The reference raised for a block's scores where they call for it (half h of the block: positions j0 + 16 h + 4 quad + i); `edge`:
    // some may lie behind `limit`, and become -inf.
    __device__ __forceinline__ void raise(f32x4 (&score)[2], float factor, bool edge, int j0, int limit)
    {
        const int quad = (threadIdx.x & 63) >> 4;
        if (edge) {
#pragma unroll
            for (int e = 0; e < 8; ++e) score[e / 4][e % 4] = j0 + 16 * (e / 4) + 4 * quad + e % 4 <= limit ? score[e / 4][e % 4] : -INFINITY;
        }
        const f32x4 s = score[0], u = score[1];
        float most = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3])));
        if (__any((most - reference) * factor > kSlack)) {
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            const float raised = fmaxf(reference, most), keep = __builtin_amdgcn_exp2f((reference - raised) * factor);
            reference = raised;
            // A weight is one fused sum, factor * score + off, where off is rounded: by 2^-4 at most up to 2^20, so that weights stay below 2^15.1.
            // Beyond that it could make the row's largest weight any power of two: differences are formed first there, which are exact near the
            // reference.  (Rows without a score yet, beyond 2^60, do not count, nor do infinite ones: those are spoilt anyway.)
            const float size = fabsf(reference * factor);
            far = __any(size > 0x1p20f && size < 0x1p60f);
            off = far ? kLift : kLift - reference * factor;
            sum *= keep;
#pragma unroll
            for (int t = 0; t < 2 * G; ++t) acc[t] *= keep;
        }
        if (far) {
#pragma unroll
            for (int e = 0; e < 8; ++e) score[e / 4][e % 4] -= reference;
        }
    }
    __device__ __forceinline__ f16x8 weights(const f32x4 (&score)[2], float factor)
    {
        f16x8 w;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float p = __builtin_amdgcn_exp2f(fmaf(score[e / 4][e % 4], factor, off));
            sum += p;
            w[e] = (_Float16)p;
        }
        return w;
    }
    __device__ __forceinline__ void finish()
    {
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
    }
};

// Scales and minima of values at positions behind `last` become zero: whatever is there has no influence.
__device__ __forceinline__ uint32_t live_mask(int i, int j0, int last)
{
    const int quad = (threadIdx.x & 63) >> 4, p = j0 + 16 * (i / 2) + 4 * quad + 2 * (i % 2);
    return (p <= last ? 0xffffu : 0u) | (p + 1 <= last ? 0xffff0000u : 0u);
}

// Four numbers of a row at dimension d: value / total into out, or, where workgroups share positions, value with the row's reference
// (in powers of two) and total beside it.
template <int HD>
__device__ __forceinline__ void store_row(const Args &a, int b, int kvh, int pair, int split, int unit, int unit_rows, int row, int live_rows, int d,
                                          f32x4 value, float reference, float total)
{
    if (row >= a.tokens * a.rep) return;
    if (a.splits > 1) {
        const size_t at = (((size_t)split * a.pairs + pair) * a.units + unit) * unit_rows + (row - unit * unit_rows);
        *(f32x4 *)(a.partial + at * HD + d) = value;
        if (d == 0) a.stats[at] = make_float2(reference, total);
        return;
    }
    const int token = row / a.rep;
    const float inverse = row < live_rows ? 1.0f / total : 0.0f;
    if (row >= live_rows) value = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    const f16x4 o = {(_Float16)(value[0] * inverse), (_Float16)(value[1] * inverse), (_Float16)(value[2] * inverse), (_Float16)(value[3] * inverse)};
    *(f16x4 *)(a.out + (((size_t)b * a.tokens + token) * a.heads + kvh * a.rep + row % a.rep) * HD + d) = o;
}

__device__ __forceinline__ f16x8 vector_of(const uint32_t (&w)[4]) { return __builtin_bit_cast(f16x8, (u32x4){w[0], w[1], w[2], w[3]}); }

// Few query rows: the waves of a workgroup take the same 16 RT rows, and the blocks in turn, each block from memory to registers.
// Bound by the stream of the cache: a wave holds a block at a time, the next one's keys are asked for when its scores are formed, its
// values once they are folded in.  Two sequences of 131072 positions, 32 heads on 8 kv heads of 128: 336 MB in 67 us and 5 for the joining, 5.0 TB/s, as a large
// copy on this card; vector instructions (365 a block, half of them the forming of held values) issue in 88 % of the cycles then.  64 sequences of 2048 positions 40 us, 4.2 TB/s.  One sequence at position 255 takes 8.9 us, of which an empty
// launch is 2, the rest one block's way from memory through both products and the joining of four waves.
template <int G, int RT>
__global__ void __launch_bounds__(kThreads, G > 4 ? 1 : RT == 1 ? 3 : 2) attention_kernel(const Args a)
{
    constexpr int HD = 32 * G, ROWS = 16 * RT;
    constexpr int kTilesAtOnce = RT == 1 ? 8 : 4;   // of 16 dimensions, joined at a time
    constexpr int kPadded = 16 * kTilesAtOnce + 4;
    static_assert(sizeof(float) * kWaves * ROWS * kPadded >= kBlock * (HD + 4), "room for an appended block");
    __shared__ float joined[kWaves][ROWS][kPadded];
    __shared__ float2 wave_stats[kWaves][ROWS];

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int column = lane & 15, quad = lane >> 4;
    const int pair = blockIdx.x % a.pairs, rest = blockIdx.x / a.pairs;
    const int split = rest % a.splits, tile = a.tiles - 1 - rest / a.splits;
    const int b = pair / a.kv_heads, kvh = pair % a.kv_heads;
    int start;
    const int n = live_tokens(a, b, start);
    const int row0 = tile * ROWS, live_rows = n * a.rep;
    const int last = min(row0 + ROWS, live_rows) - 1;                          // its last row that is no padding
    const int limit_high = last >= row0 ? start + last / a.rep : -1, limit_low = start + row0 / a.rep;
    const int blocks = (limit_high + kBlock) / kBlock;
    const int per = blocks_per_split(a, blocks, kWaves);
    const int begin = split * per, end = min(begin + per, blocks);
    if (a.fused && split == 0) clear_held<HD, kThreads>(a, b, kvh, n, 0, a.tokens);
    if (a.splits > 1 && begin >= end) return;                                  // (nobody reads its part)

    // Fused: the one tile of a pair's rows; the workgroup whose blocks new tokens fall into appends them before anything is read.
    if (a.fused && n > 0 && start / kBlock < end) {
        for (int fresh = max(start / kBlock, begin); fresh < end; ++fresh) {
            append_block<G, kThreads>(a, b, kvh, pair, start, n, fresh, (uint8_t *)joined);
            __syncthreads();
        }
    }

    f16x8 q[RT][G];
    int limit[RT];
    load_queries<G, RT>(a, b, kvh, start, row0, live_rows, q, limit);
    const float factor = 1.4426950408889634f / sqrtf((float)HD);
    RowState<G> state[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) state[rt].clear(factor);
    const uint8_t *cache = a.cache + (size_t)pair * a.blocks * (size_t)(1280 * G);

    uint32_t k_codes[2][G], k_scales[2][G], v_codes[2 * G], v_scales[2 * G][4];
    auto fetch_keys = [&](int block) {
        const uint8_t *base = cache + (size_t)block * (1280 * G);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            load_words(k_codes[h], base + ((16 * h + column) * 4 + quad) * (4 * G));
            load_words(k_scales[h], base + 512 * G + (16 * h + column) * (4 * G));
        }
    };
    auto fetch_values = [&](int block) {
        const uint8_t *base = cache + (size_t)block * (1280 * G) + 640 * G;
        load_words(v_codes, base + (quad * 16 + column) * (8 * G));
#pragma unroll
        for (int t = 0; t < 2 * G; ++t) load_words(v_scales[t], base + 512 * G + t * 64 + quad * 16);
    };
    int block = begin + wave;
    if (block < end) {
        fetch_keys(block);
        fetch_values(block);
    }
    for (; block < end; block += kWaves) {
        const int next = block + kWaves < end ? block + kWaves : block;
        f32x4 score[RT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) score[rt][h] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < G; ++t) {
                const f16x2 sm = __builtin_bit_cast(f16x2, k_scales[h][t]);
                const f16x8 key = __builtin_elementwise_fma(codes_of(k_codes[h][t]), (f16x8)(sm.x), (f16x8)(sm.y));
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) score[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, q[rt][t], score[rt][h], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        fetch_keys(next);
        __builtin_amdgcn_sched_barrier(0);
        const int j0 = block * kBlock;
        const bool edge = j0 + kBlock - 1 > limit_low;
        f16x8 weight[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            state[rt].raise(score[rt], factor, edge, j0, limit[rt]);
            weight[rt] = state[rt].weights(score[rt], factor);
        }
        if (j0 + kBlock - 1 > limit_high) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t mask = live_mask(i, j0, limit_high);
#pragma unroll
                for (int t = 0; t < 2 * G; ++t) v_scales[t][i] &= mask;
            }
        }
#pragma unroll
        for (int t = 0; t < 2 * G; ++t) {
            const f16x8 value = __builtin_elementwise_fma(codes_of(v_codes[t]), vector_of(v_scales[t & ~1]), vector_of(v_scales[t | 1]));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) state[rt].acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value, weight[rt], state[rt].acc[t], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        fetch_values(next);
        __builtin_amdgcn_sched_barrier(0);
    }

    // ---- the waves' results joined ------------------------------------------------------------------------------------------
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        state[rt].finish();
        state[rt].reference *= factor;   // (in powers of two from here on)
        if (quad == 0) wave_stats[wave][16 * rt + column] = make_float2(state[rt].reference, state[rt].sum);
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float most = wave_stats[0][16 * rt + column].x;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) most = fmaxf(most, wave_stats[w][16 * rt + column].x);
        const float keep = __builtin_amdgcn_exp2f(state[rt].reference - most);
#pragma unroll
        for (int t = 0; t < 2 * G; ++t) state[rt].acc[t] *= keep;
    }
#pragma unroll
    for (int t0 = 0; t0 < 2 * G; t0 += kTilesAtOnce) {
        if (t0 > 0) __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = t0; t < t0 + kTilesAtOnce && t < 2 * G; ++t)
                *(f32x4 *)&joined[wave][16 * rt + column][16 * (t - t0) + 4 * quad] = state[rt].acc[t];
        __syncthreads();
        const int fours = 4 * min(kTilesAtOnce, 2 * G - t0);
        for (int u = tid; u < ROWS * fours; u += kThreads) {
            const int row = u / fours, d = u % fours * 4;
            f32x4 value = *(const f32x4 *)&joined[0][row][d];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) value += *(const f32x4 *)&joined[w][row][d];
            float most = wave_stats[0][row].x, total = 0.0f;
#pragma unroll
            for (int w = 1; w < kWaves; ++w) most = fmaxf(most, wave_stats[w][row].x);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) total += wave_stats[w][row].y * __builtin_amdgcn_exp2f(wave_stats[w][row].x - most);
            store_row<HD>(a, b, kvh, pair, split, tile, ROWS, row0 + row, live_rows, 16 * t0 + d, value, most, total);
        }
    }
}

// Many query rows (prompts): the waves of a workgroup take 16 RT rows each, side by side, and all of its blocks together.  A block's keys and
// values are formed once for all waves, by pieces, and handed over through LDS as the matrix instructions' operands: a wave that forms them for
// itself does nothing else for most of its time (two prompts of 2048 tokens, 32 heads on 8: 197 us, vector unit 62 % busy, matrix unit 15 %).
// Two buffers each, one barrier a block.  In the time of a block its weights are formed while the next block's scores are multiplied, from keys
// that stand ready, and its values multiplied while the pieces of later blocks are formed; operands are read from LDS all at once, ahead of
// their use (read one at a time, each wave waited for each: 107 us for those prompts without appending).  Now 114 us, 14 of them appending: 567 TFLOP/s
// of the 1310 that a large fp16 product reaches.  Vector instructions (forming operands, weights, masks) issue in 55 % of the cycles, matrix
// instructions run in 29 %; two waves per SIMD, which the registers of 32 rows of 128 dimensions allow, do not hide the rest.  Four waves instead of
// eight form twice as much each: 140 us.  A third buffer of keys, read ahead of the barrier: 122 us.  A chunk of 256 tokens onto 30000
// positions: 172 us, 737 TFLOP/s.
template <int G>
constexpr int kPromptTiles = G > 4 ? 1 : 2;   // tiles of 16 rows a wave takes, as registers allow

template <int G, int W>
__global__ void __launch_bounds__(64 * W, 2) prompt_kernel(const Args a)
{
    constexpr int HD = 32 * G, RT = kPromptTiles<G>, ROWS = 16 * RT;
    constexpr int kPieces = (2 * G + W - 1) / W;   // of 2 G operands of keys and as many of values, a wave's
    __shared__ f16x8 keys[2][2 * G][64], values[2][2 * G][64];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, column = lane & 15, quad = lane >> 4;
    const int pair = blockIdx.x % a.pairs, rest = blockIdx.x / a.pairs;
    const int split = rest % a.splits, tile = a.tiles - 1 - rest / a.splits;   // (the longest rows first)
    const int b = pair / a.kv_heads, kvh = pair % a.kv_heads;
    int start;
    const int n = live_tokens(a, b, start);
    const int unit = tile * W + wave, row0 = unit * ROWS, live_rows = n * a.rep;

    const int tile_last = min((tile + 1) * W * ROWS, live_rows) - 1;
    const int tile_high = tile_last >= tile * W * ROWS ? start + tile_last / a.rep : -1, blocks = (tile_high + kBlock) / kBlock;
    const int per = blocks_per_split(a, blocks, 4);
    const int begin = split * per, end = min(begin + per, blocks);
    if (a.splits > 1 && begin >= end) return;
    const int last = min(row0 + ROWS, live_rows) - 1;
    const int limit_high = last >= row0 ? start + last / a.rep : -1, limit_low = start + row0 / a.rep;
    const int own_end = min(end, (limit_high + kBlock) / kBlock);              // (the rest lies behind this wave's rows)

    const uint8_t *cache = a.cache + (size_t)pair * a.blocks * (size_t)(1280 * G);
    uint32_t k_code[kPieces], k_scale[kPieces], v_code[kPieces], v_scale[kPieces][2][4];
    auto mine = [&](int i) { return 2 * G % W == 0 || wave + i * W < 2 * G; };
    auto fetch_keys = [&](int block) {
        const uint8_t *base = cache + (size_t)block * (1280 * G);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int f = wave + i * W, position = 16 * (f / G) + column;
            if (!mine(i)) continue;
            k_code[i] = *(const uint32_t *)(base + ((position * 4 + quad) * G + f % G) * 4);
            k_scale[i] = *(const uint32_t *)(base + 512 * G + (position * G + f % G) * 4);
        }
    };
    auto fetch_values = [&](int block) {
        const uint8_t *base = cache + (size_t)block * (1280 * G);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int f = wave + i * W;
            if (!mine(i)) continue;
            v_code[i] = *(const uint32_t *)(base + 640 * G + ((quad * 16 + column) * 2 * G + f) * 4);
            load_words(v_scale[i][0], base + 1152 * G + (f & ~1) * 64 + quad * 16);
            load_words(v_scale[i][1], base + 1152 * G + (f | 1) * 64 + quad * 16);
        }
    };
    auto form_keys = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (!mine(i)) continue;
            const f16x2 sm = __builtin_bit_cast(f16x2, k_scale[i]);
            keys[buffer][wave + i * W][lane] = __builtin_elementwise_fma(codes_of(k_code[i]), (f16x8)(sm.x), (f16x8)(sm.y));
        }
    };
    auto form_values = [&](int block, int buffer) {
        const bool beyond = (block + 1) * kBlock - 1 > tile_high;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (!mine(i)) continue;
            if (beyond) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t mask = live_mask(j, block * kBlock, tile_high);
                    v_scale[i][0][j] &= mask;
                    v_scale[i][1][j] &= mask;
                }
            }
            values[buffer][wave + i * W][lane] = __builtin_elementwise_fma(codes_of(v_code[i]), vector_of(v_scale[i][0]), vector_of(v_scale[i][1]));
        }
    };
    // (blocks behind the last are asked for and formed like it, and not used: no branch in the loop)
    auto inside = [&](int block) { return min(block, end - 1); };
    if (begin < end) {
        fetch_keys(begin);
        fetch_values(begin);
    }
    f16x8 q[RT][G];
    int limit[RT];
    load_queries<G, RT>(a, b, kvh, start, row0, live_rows, q, limit);
    const float factor = 1.4426950408889634f / sqrtf((float)HD);
    RowState<G> state[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) state[rt].clear(factor);
    f32x4 score[RT][2];
    f16x8 operand[2 * G];
    auto multiply_keys = [&](f32x4 (&to)[RT][2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) to[rt][h] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < G; ++t)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) to[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand[h * G + t], q[rt][t], to[rt][h], 0, 0, 0);
        }
    };
    if (begin < end) {
        form_keys(0);
        form_values(begin, 0);
        fetch_keys(inside(begin + 1));
        fetch_values(inside(begin + 1));
        __syncthreads();
#pragma unroll
        for (int f = 0; f < 2 * G; ++f) operand[f] = keys[0][f][lane];
        multiply_keys(score);
        form_keys(1);
        fetch_keys(inside(begin + 2));
    }
    for (int block = begin; block < end; ++block) {
        const int buffer = (block - begin) & 1;
        // Here: this block's scores in registers, its values formed, the next one's keys formed; its values' codes and the keys' of the one
        // after it in registers.
        __syncthreads();
        if (block < own_end) {
#pragma unroll
            for (int f = 0; f < 2 * G; ++f) operand[f] = keys[buffer ^ 1][f][lane];
            __builtin_amdgcn_sched_barrier(0);
            const int j0 = block * kBlock;
            const bool edge = j0 + kBlock - 1 > limit_low;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) state[rt].raise(score[rt], factor, edge, j0, limit[rt]);
            f32x4 next[RT][2];
            f16x8 weight[RT];
            multiply_keys(next);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) weight[rt] = state[rt].weights(score[rt], factor);
#pragma unroll
            for (int i = 0; i < 2 * G * RT; ++i) {   // a matrix instruction, then vector ones in its time
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x402, 3, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int f = 0; f < 2 * G; ++f) operand[f] = values[buffer][f][lane];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < 2 * G; ++t)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) state[rt].acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand[t], weight[rt], state[rt].acc[t], 0, 0, 0);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                score[rt][0] = next[rt][0];
                score[rt][1] = next[rt][1];
            }
        }
        form_keys(buffer);
        form_values(inside(block + 1), buffer ^ 1);
        fetch_keys(inside(block + 3));
        fetch_values(inside(block + 2));
    }
    if (unit >= a.units) return;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        state[rt].finish();
#pragma unroll
        for (int t = 0; t < 2 * G; ++t)
            store_row<HD>(a, b, kvh, pair, split, unit, ROWS, row0 + 16 * rt + column, live_rows, 16 * t + 4 * quad, state[rt].acc[t], state[rt].reference * factor, state[rt].sum);
    }
}

// Joins the parts of a row: the sum over splits of 2^(reference - largest reference) * part.  One workgroup per row; the splits' weights are formed
// by a lane each, and groups of HD / 4 threads take the splits in turn (one thread for all of a row's splits: 64 splits of 128 rows 43 us).
constexpr int kMostSplits = 64;

template <int G>
__global__ void __launch_bounds__(kThreads) join_kernel(const Args a, int unit_rows, int tile_rows, int least)
{
    constexpr int HD = 32 * G, kGroups = kThreads / (HD / 4);
    __shared__ float weight[kMostSplits];
    __shared__ f32x4 part[kGroups][HD / 4];
    const int tid = threadIdx.x, pair = blockIdx.x % a.pairs, row = blockIdx.x / a.pairs;
    const int b = pair / a.kv_heads, kvh = pair % a.kv_heads;
    int start;
    const int n = live_tokens(a, b, start), live_rows = n * a.rep;
    f16x4 *out = (f16x4 *)(a.out + (((size_t)b * a.tokens + row / a.rep) * a.heads + kvh * a.rep + row % a.rep) * HD);
    if (row >= live_rows) {
        if (tid < HD / 4) out[tid] = (f16x4)((_Float16)0.0f);
        return;
    }
    const int unit = row / unit_rows, tile = row / tile_rows, tile_last = min((tile + 1) * tile_rows, live_rows) - 1;
    const int blocks = (start + tile_last / a.rep) / kBlock + 1, per = blocks_per_split(a, blocks, least), parts = (blocks + per - 1) / per;
    const size_t stride = (size_t)a.pairs * a.units * unit_rows, at = ((size_t)pair * a.units + unit) * unit_rows + row % unit_rows;
    const int lane = tid & 63;
    float2 st = make_float2(-INFINITY, 0.0f);
    if (lane < parts) st = a.stats[lane * stride + at];
    float most = st.x;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) most = fmaxf(most, __shfl_xor(most, m));
    const float keep = lane < parts ? __builtin_amdgcn_exp2f(st.x - most) : 0.0f;
    float total = st.y * keep;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) total += __shfl_xor(total, m);
    if (tid < kMostSplits) weight[tid] = keep;
    __syncthreads();
    const int group = tid / (HD / 4), d = tid % (HD / 4);
    if (group < kGroups) {
        f32x4 value = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int s = group; s < parts; s += kGroups) value += *(const f32x4 *)(a.partial + (s * stride + at) * HD + 4 * d) * weight[s];
        part[group][d] = value;
    }
    __syncthreads();
    if (tid >= HD / 4) return;
    f32x4 value = part[0][tid];
#pragma unroll
    for (int g = 1; g < kGroups; ++g) value += part[g][tid];
    const float inverse = 1.0f / total;
    out[tid] = (f16x4){(_Float16)(value[0] * inverse), (_Float16)(value[1] * inverse), (_Float16)(value[2] * inverse), (_Float16)(value[3] * inverse)};
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

int launch_status()
{
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? LUTGEMM_OK : lutgemm_internal_hip_fail((int)e);
}

bool cache_sizes_fit(int batch, int kv_heads, int max_positions, int head_dim)
{
    return batch >= 1 && batch <= 65535 && kv_heads >= 1 && kv_heads <= 4096 && max_positions >= 1 && max_positions <= 1 << 20 &&
           head_dim >= 32 && head_dim <= 256 && head_dim % 32 == 0;
}

struct Sizes {
    int units, tiles;
    size_t partial_floats;   // of the whole call
    size_t workspace;
};

int plan_call(int batch, int tokens, int heads, int kv_heads, int head_dim, int max_positions, lutgemm_q4_attention_plan *p, Sizes *s)
{
    if (!cache_sizes_fit(batch, kv_heads, max_positions, head_dim) || tokens < 1 || tokens > 65536) return LUTGEMM_EINVAL;
    if (heads < kv_heads || heads > 4096 || heads % kv_heads != 0) return LUTGEMM_EINVAL;
    const long rows = (long)tokens * (heads / kv_heads), pairs = (long)batch * kv_heads;
    const int blocks = (max_positions + kBlock - 1) / kBlock;
    // (one tile of rows per pair: its workgroups append themselves, a launch and 8 us less for single tokens)
    p->fused = rows <= 32;
    p->rows_apart = rows >= 4 * 32;
    p->rows_per_wave = rows > 16 && !(p->rows_apart && head_dim > 128) ? 32 : 16;
    // (eight waves share the forming of a block, where that leaves a workgroup for every CU: a prompt of 512 on 32 kv heads by fours 37.8 us, by
    // eights 44; a chunk of 256 of 32 heads on 8 kv heads onto 30000 positions, whose positions are shared, 210 and 187)
    const long eights = pairs * ((rows + 8 * p->rows_per_wave - 1) / (8 * p->rows_per_wave)) * (blocks > 32 ? blocks / 16 : 1);
    const int waves = p->rows_apart && eights >= 256 ? 8 : 4;
    p->threads = 64 * waves;
    s->units = (int)((rows + p->rows_per_wave - 1) / p->rows_per_wave);
    s->tiles = p->rows_apart ? (s->units + waves - 1) / waves : s->units;
    const long alone = pairs * s->tiles;
    // Positions are shared by workgroups where the CUs hold more of them at once than there are tiles, and a wave would have more than ten
    // blocks to itself: the joining launch takes 4 to 5 us, a block about half of one (8 sequences of 32 heads at position 1023: one 16.3 us, two
    // 20 us; one of 8 at 8191: one 33 us, 32 12.4 us; 24 of 8, up to 4096: one 27.7 us, four 18.9 us).
    long splits = 1;
    const long room = (p->rows_apart ? 512 : 768) * 4 / (alone * waves);
    if (blocks > (p->rows_apart ? 32 : 10 * waves)) splits = room;
    const long most = blocks / (p->rows_apart ? 16 : 2 * waves);   // each has some blocks to itself
    if (splits > most) splits = most;
    if (splits > kMostSplits) splits = kMostSplits;
    if (splits < 1) splits = 1;
    p->splits = (int)splits;
    p->row_tiles = s->tiles;
    p->launches = 1 + !p->fused + (splits > 1);
    // (a launch takes fewer than 2^32 work items: refused here, before the first of a call's launches)
    const long most_items = 0xffffffffl, append_parts = (tokens + kBlock - 1) / kBlock + 1;
    if (alone * splits * p->threads > most_items || (!p->fused && pairs * append_parts * append_threads(head_dim / 32) > most_items) ||
        (splits > 1 && pairs * rows * kThreads > most_items))
        return LUTGEMM_EINVAL;
    p->workgroups = (int)(alone * splits);
    const size_t part_rows = (size_t)splits * pairs * s->units * p->rows_per_wave;
    s->partial_floats = splits > 1 ? part_rows * head_dim : 0;
    s->workspace = splits > 1 ? part_rows * (head_dim * 4 + 8) : 0;
    return LUTGEMM_OK;
}

struct Span {
    uintptr_t from, past;
};

bool overlap(const Span &a, const Span &b) { return a.from < b.past && b.from < a.past; }

// Whether what a call writes lies apart from all else that it is given.
bool written_apart(const lutgemm_q4_attention *c)
{
    auto span = [](const void *p, size_t bytes) { return Span{(uintptr_t)p, (uintptr_t)p + (p ? bytes : 0)}; };
    auto rows = [&](const void *p, const int64_t (&stride)[2], int heads) {
        return span(p, 2 * ((size_t)(c->batch - 1) * stride[0] + (size_t)(c->tokens - 1) * stride[1] + (size_t)heads * c->head_dim));
    };
    const size_t tokens = (size_t)c->batch * c->tokens, table = (size_t)c->max_positions * c->head_dim * 2;
    const size_t held = tokens * c->kv_heads * c->head_dim * 2;
    const Span all[] = {span(c->cache, lutgemm_q4_cache_bytes(c->batch, c->kv_heads, c->max_positions, c->head_dim)),
                        span(c->out, tokens * c->heads * c->head_dim * 2), span(c->k_held, held), span(c->v_held, held),
                        rows(c->q, c->q_stride, c->heads), rows(c->k, c->k_stride, c->kv_heads), rows(c->v, c->v_stride, c->kv_heads),
                        span(c->cos_table, table), span(c->sin_table, table), span(c->start, (size_t)c->batch * 8), span(c->counts, (size_t)c->batch * 4)};
    for (int i = 0; i < 4; ++i)
        for (int j = i + 1; j < (int)(sizeof(all) / sizeof(all[0])); ++j)
            if (overlap(all[i], all[j])) return false;
    return true;
}

bool strides_fit(const int64_t (&s)[2], const void *p)
{
    return aligned16(p) && s[0] % 8 == 0 && s[1] % 8 == 0;
}

}  // namespace

extern "C" {

size_t lutgemm_q4_cache_bytes(int batch, int kv_heads, int max_positions, int head_dim)
{
    if (!cache_sizes_fit(batch, kv_heads, max_positions, head_dim)) return 0;
    return (size_t)batch * kv_heads * ((max_positions + kBlock - 1) / kBlock) * (size_t)(40 * head_dim);
}

size_t lutgemm_q4_attention_workspace(int batch, int tokens, int heads, int kv_heads, int head_dim, int max_positions)
{
    lutgemm_q4_attention_plan plan;
    Sizes sizes;
    if (plan_call(batch, tokens, heads, kv_heads, head_dim, max_positions, &plan, &sizes) != LUTGEMM_OK) return 0;
    return sizes.workspace;
}

int lutgemm_describe_q4_attention_plan(int batch, int tokens, int heads, int kv_heads, int head_dim, int max_positions,
                                       lutgemm_q4_attention_plan *plan)
{
    if (!plan) return LUTGEMM_EINVAL;
    Sizes sizes;
    return plan_call(batch, tokens, heads, kv_heads, head_dim, max_positions, plan, &sizes);
}

int lutgemm_q4_attention_f16(const lutgemm_q4_attention *c, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!c || !c->cache || !c->q || !c->k || !c->v || !c->cos_table || !c->sin_table || !c->start || !c->out) return LUTGEMM_EINVAL;
    lutgemm_q4_attention_plan plan;
    Sizes sizes;
    const int rc = plan_call(c->batch, c->tokens, c->heads, c->kv_heads, c->head_dim, c->max_positions, &plan, &sizes);
    if (rc != LUTGEMM_OK) return rc;
    for (int i = 0; i < 2; ++i)
        if (c->q_stride[i] < 0 || c->k_stride[i] < 0 || c->v_stride[i] < 0) return LUTGEMM_EINVAL;
    if (sizes.workspace > 0 && (!workspace || workspace_bytes < sizes.workspace)) return LUTGEMM_EINVAL;
    if (!aligned16(c->cache) || !aligned16(c->cos_table) || !aligned16(c->sin_table) || !aligned16(c->out) || !aligned16(c->k_held) ||
        !aligned16(c->v_held) || ((uintptr_t)c->start & 7u) || ((uintptr_t)c->counts & 3u) || (sizes.workspace > 0 && !aligned16(workspace)) ||
        !strides_fit(c->q_stride, c->q) || !strides_fit(c->k_stride, c->k) || !strides_fit(c->v_stride, c->v))
        return LUTGEMM_EALIGN;
    if (!written_apart(c)) return LUTGEMM_EINVAL;
    Args a{};
    a.cache = (uint8_t *)c->cache;
    a.q = (const _Float16 *)c->q;
    a.k = (const _Float16 *)c->k;
    a.v = (const _Float16 *)c->v;
    a.cos_t = (const _Float16 *)c->cos_table;
    a.sin_t = (const _Float16 *)c->sin_table;
    a.start = c->start;
    a.counts = c->counts;
    a.out = (_Float16 *)c->out;
    a.k_held = (_Float16 *)c->k_held;
    a.v_held = (_Float16 *)c->v_held;
    for (int i = 0; i < 2; ++i) {
        a.q_stride[i] = c->q_stride[i];
        a.k_stride[i] = c->k_stride[i];
        a.v_stride[i] = c->v_stride[i];
    }
    a.tokens = c->tokens;
    a.heads = c->heads;
    a.kv_heads = c->kv_heads;
    a.rep = c->heads / c->kv_heads;
    a.max_positions = c->max_positions;
    a.blocks = (c->max_positions + kBlock - 1) / kBlock;
    a.pairs = c->batch * c->kv_heads;
    a.units = sizes.units;
    a.tiles = sizes.tiles;
    a.splits = plan.splits;
    a.fused = plan.fused;
    a.partial = (float *)workspace;
    a.stats = (float2 *)((float *)workspace + sizes.partial_floats);
    const hipStream_t hs = (hipStream_t)stream;

    auto run = [&](auto g_c) -> int {
        constexpr int G = decltype(g_c)::value;
        int status = LUTGEMM_OK;
        if (!plan.fused) {
            const long parts = (a.tokens + kBlock - 1) / kBlock + 1;
            hipLaunchKernelGGL(append_kernel<G>, dim3((unsigned)(parts * a.pairs)), dim3(kAppendThreads<G>), 0, hs, a);
            status = launch_status();
            if (status != LUTGEMM_OK) return status;
        }
        const dim3 grid((unsigned)plan.workgroups), threads((unsigned)plan.threads);
        if (plan.rows_apart && plan.threads == 512) hipLaunchKernelGGL((prompt_kernel<G, 8>), grid, threads, 0, hs, a);
        else if (plan.rows_apart) hipLaunchKernelGGL((prompt_kernel<G, 4>), grid, threads, 0, hs, a);
        else if (plan.rows_per_wave == 32) hipLaunchKernelGGL((attention_kernel<G, 2>), grid, threads, 0, hs, a);
        else hipLaunchKernelGGL((attention_kernel<G, 1>), grid, threads, 0, hs, a);
        status = launch_status();
        if (status != LUTGEMM_OK || a.splits == 1) return status;
        const int tile_rows = plan.rows_apart ? plan.rows_per_wave * (plan.threads / 64) : plan.rows_per_wave;
        hipLaunchKernelGGL(join_kernel<G>, dim3((unsigned)((size_t)a.pairs * a.tokens * a.rep)), dim3(kThreads), 0, hs, a, plan.rows_per_wave, tile_rows,
                           plan.rows_apart ? 4 : kWaves);
        return launch_status();
    };
    switch (c->head_dim / 32) {
    case 1: return run(std::integral_constant<int, 1>());
    case 2: return run(std::integral_constant<int, 2>());
    case 3: return run(std::integral_constant<int, 3>());
    case 4: return run(std::integral_constant<int, 4>());
    case 5: return run(std::integral_constant<int, 5>());
    case 6: return run(std::integral_constant<int, 6>());
    case 7: return run(std::integral_constant<int, 7>());
    default: return run(std::integral_constant<int, 8>());
    }
}

}  // extern "C"
