// Low-rank adapters of many requests beside a shared linear layer, gfx950: out = base + scale * up (down x), every row through the
// adapter that its id names.  Two launches: down, which leaves h = down x in fp32, and up.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lutgemm_gfx950.h"
#include "lutgemm_common.h"
#include "lutgemm_internal.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

struct Problem {
    const _Float16 *x, *base;
    _Float16 *out;
    const int32_t *ids;
    const _Float16 *down, *up;
    const float *scale;
    int64_t x_stride, base_stride, out_stride;
    int M, N, K, rank, adapters;
    float *h;   // [M][rank]
};

struct Args {
    int count;
    Problem p[LUTGEMM_MAX_GROUP];
};

// One workgroup per row: the waves take the ranks in turn.
__global__ void __launch_bounds__(kThreads) down_kernel(const Args args)
{
    const Problem &p = args.p[blockIdx.y];
    const int m = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (m >= p.M) return;
    const int id = p.ids[m];
    if (id < 0 || id >= p.adapters) return;
    const _Float16 *x = p.x + m * p.x_stride;
    for (int r = wave; r < p.rank; r += kWaves) {
        const _Float16 *row = p.down + ((size_t)id * p.rank + r) * p.K;
        float sum = 0.0f;
        for (int k = lane * 8; k < p.K; k += 512) {
            const f16x8 xv = *(const f16x8 *)(x + k), wv = *(const f16x8 *)(row + k);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf((float)xv[i], (float)wv[i], sum);
        }
        for (int s = 1; s < 64; s *= 2) sum += __shfl_xor(sum, s);
        if (lane == 0) p.h[(size_t)m * p.rank + r] = sum;
    }
}

// One thread per four outputs of a row.
__global__ void __launch_bounds__(kThreads) up_kernel(const Args args)
{
    const Problem &p = args.p[blockIdx.z];
    const int m = blockIdx.y, n = (blockIdx.x * kThreads + threadIdx.x) * 4;
    if (m >= p.M || n >= p.N) return;
    const f16x4 base = *(const f16x4 *)(p.base + m * p.base_stride + n);
    f16x4 *out = (f16x4 *)(p.out + m * p.out_stride + n);
    const int id = p.ids[m];
    if (id < 0 || id >= p.adapters) {
        *out = base;
        return;
    }
    const float *h = p.h + (size_t)m * p.rank;
    const _Float16 *up = p.up + ((size_t)id * p.N + n) * p.rank;
    const float scale = p.scale ? p.scale[id] : 1.0f;
    f16x4 result;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float sum = 0.0f;
        for (int r = 0; r < p.rank; r += 8) {
            const f16x8 u = *(const f16x8 *)(up + (size_t)i * p.rank + r);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf((float)u[j], h[r + j], sum);
        }
        result[i] = (_Float16)((float)base[i] + scale * sum);
    }
    *out = result;
}

int launch_status()
{
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? LUTGEMM_OK : lutgemm_internal_hip_fail((int)e);
}

bool aligned(const void *p, unsigned bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

struct Span {
    uintptr_t from, past;
};

Span span_of(const void *p, int rows, int64_t stride, size_t row_values, int value_bytes)
{
    return {(uintptr_t)p, (uintptr_t)p + ((size_t)(rows - 1) * (size_t)stride + row_values) * value_bytes};
}

bool overlap(const Span &a, const Span &b) { return a.from < b.past && b.from < a.past; }

// What a call returns before anything is launched.
int check(int count, const lutgemm_adapters *ps)
{
    if (count < 1 || count > LUTGEMM_MAX_GROUP || !ps) return LUTGEMM_EINVAL;
    for (int i = 0; i < count; ++i) {
        const lutgemm_adapters &p = ps[i];
        if (!p.x_f16 || !p.base_f16 || !p.out_f16 || !p.ids || !p.down_f16 || !p.up_f16) return LUTGEMM_EINVAL;
        if (p.M < 1 || p.M > 65535 || p.K < 32 || p.K % 32 != 0 || p.K > 1 << 20 || p.N < 4 || p.N % 4 != 0 || p.N > 1 << 20) return LUTGEMM_EINVAL;
        if (p.rank < 8 || p.rank > 256 || p.rank % 8 != 0 || p.adapters < 1 || p.adapters > 65535) return LUTGEMM_EINVAL;
        if (p.M > 1 && (p.x_stride < 0 || p.base_stride < 0 || p.out_stride < p.N)) return LUTGEMM_EINVAL;
        if (p.out_f16 == p.base_f16 && p.M > 1 && p.out_stride != p.base_stride) return LUTGEMM_EINVAL;
    }
    for (int i = 0; i < count; ++i) {
        const lutgemm_adapters &p = ps[i];
        if (p.M > 1 && (p.x_stride % 8 != 0 || p.base_stride % 4 != 0 || p.out_stride % 4 != 0)) return LUTGEMM_EALIGN;
        if (!aligned(p.x_f16, 16) || !aligned(p.base_f16, 8) || !aligned(p.out_f16, 8) || !aligned(p.down_f16, 16) || !aligned(p.up_f16, 16) ||
            !aligned(p.ids, 4) || !aligned(p.scale, 4))
            return LUTGEMM_EALIGN;
    }
    for (int i = 0; i < count; ++i) {
        const Span out = span_of(ps[i].out_f16, ps[i].M, ps[i].out_stride, ps[i].N, 2);
        for (int j = 0; j < count; ++j) {
            const lutgemm_adapters &q = ps[j];
            if (i != j && overlap(out, span_of(q.out_f16, q.M, q.out_stride, q.N, 2))) return LUTGEMM_EINVAL;
            if (!(i == j && q.base_f16 == q.out_f16) && overlap(out, span_of(q.base_f16, q.M, q.base_stride, q.N, 2))) return LUTGEMM_EINVAL;
            if (overlap(out, span_of(q.x_f16, q.M, q.x_stride, q.K, 2)) || overlap(out, span_of(q.ids, 1, 0, q.M, 4)) ||
                overlap(out, span_of(q.down_f16, 1, 0, (size_t)q.adapters * q.rank * q.K, 2)) ||
                overlap(out, span_of(q.up_f16, 1, 0, (size_t)q.adapters * q.rank * q.N, 2)) ||
                (q.scale && overlap(out, span_of(q.scale, 1, 0, q.adapters, 4))))
                return LUTGEMM_EINVAL;
        }
    }
    return LUTGEMM_OK;
}

size_t h_bytes(const lutgemm_adapters &p) { return ((size_t)p.M * p.rank * 4 + 15) / 16 * 16; }

}  // namespace

extern "C" {

size_t lutgemm_adapters_workspace(int count, const lutgemm_adapters *problems)
{
    if (check(count, problems) != LUTGEMM_OK) return 0;
    size_t bytes = 0;
    for (int i = 0; i < count; ++i) bytes += h_bytes(problems[i]);
    return bytes;
}

int lutgemm_adapters_f16(int count, const lutgemm_adapters *problems, void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = check(count, problems);
    if (rc != LUTGEMM_OK) return rc;
    if (!workspace || workspace_bytes < lutgemm_adapters_workspace(count, problems)) return LUTGEMM_EINVAL;
    if (!aligned(workspace, 16)) return LUTGEMM_EALIGN;
    Args a{};
    a.count = count;
    char *h = (char *)workspace;
    int rows = 0, columns = 0;
    for (int i = 0; i < count; ++i) {
        const lutgemm_adapters &p = problems[i];
        a.p[i] = {(const _Float16 *)p.x_f16, (const _Float16 *)p.base_f16, (_Float16 *)p.out_f16, p.ids, (const _Float16 *)p.down_f16,
                  (const _Float16 *)p.up_f16, p.scale, p.x_stride, p.base_stride, p.out_stride, p.M, p.N, p.K, p.rank, p.adapters, (float *)h};
        h += h_bytes(p);
        rows = p.M > rows ? p.M : rows;
        columns = p.N > columns ? p.N : columns;
    }
    const hipStream_t hs = (hipStream_t)stream;
    hipLaunchKernelGGL(down_kernel, dim3(rows, count), dim3(kThreads), 0, hs, a);
    const int status = launch_status();
    if (status != LUTGEMM_OK) return status;
    hipLaunchKernelGGL(up_kernel, dim3((columns + 4 * kThreads - 1) / (4 * kThreads), rows, count), dim3(kThreads), 0, hs, a);
    return launch_status();
}

}  // extern "C"
