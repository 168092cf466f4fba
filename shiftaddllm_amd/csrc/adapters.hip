// Low-rank adapters of many requests beside a shared linear layer, gfx950: out = base + scale * up (down x), every row through the
// adapter that its id names.
//
// Rows of one adapter are taken together, up to 16 of them, which are the columns of the matrix instruction in both products:
//   h^T = down x^T      A: 16 ranks of down, B: 16 rows of x.  The waves of a workgroup, and workgroups, share K; parts of h are
//                       left side by side in fp32 and added up, in their order, by the next launch.
//   out^T = up h^T      A: 16 outputs of up, B: the rows' h.  h keeps its 32 bits: a row is scaled by a power of two to at most 1 and
//                       held as the sum of two fp16 numbers, 2^-25 of its largest apart from it, which the instruction multiplies one
//                       after the other.
// A column of the instruction depends on nothing but its own row, so what rows stand beside it makes no difference to a result.
// Bound by reading the adapters that are used (few rows), or x, base and out (many): 48 rows of 48 adapters of rank 64, 4096 to 11008, 95 MB
// in 26.0 us (3.7 TB/s; a large copy 4.9); 4096 rows of 6 adapters of rank 32, 4096 to 4096, 49.4 us (43.2 where x, base and out are the same ones
// pass after pass), of which sorting 6.3 to 7.5, each product 18.5 to 19.6; one row 8.9 us, two launches in a row.  Up to 256 rows every workgroup finds by
// itself which rows share its row's adapter; more rows are sorted by a launch ahead.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "lutgemm_gfx950.h"
#include "lutgemm_common.h"
#include "lutgemm_internal.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kTile = 16;              // rows taken together
constexpr int kUnsorted = 256;         // rows up to which workgroups look for their own
constexpr int kMaxAdapters = LUTGEMM_MAX_ADAPTERS;
constexpr int kDepth = 128;            // inputs a wave takes at a time
constexpr int kColumns = 64;           // outputs a wave takes at a time

// Rows of one adapter: `count` entries of the order from `first` on.
struct Tile {
    int id, first, count;
};

struct Problem {
    const _Float16 *x, *base;
    _Float16 *out;
    const int32_t *ids;
    const _Float16 *down, *up;
    const float *scale;
    int64_t x_stride, base_stride, out_stride;
    int M, N, K, rank, adapters;
    int slots;                 // tiles there can be: workgroups that look for rows
    int k_splits, k_own;       // workgroups that share K, and the inputs each takes (a multiple of kDepth)
    int n_own;                 // outputs a workgroup takes
    float *h;                  // [k_splits][M][rank]
    Tile *tiles;               // sorted rows: the tiles (a count of 0 behind the last), and
    int32_t *order, *places;   // the rows, and each one's place among its adapter's
};

struct Args {
    int count;
    Problem p[LUTGEMM_MAX_GROUP];
};

// The adapter of a row, or -1.
__device__ __forceinline__ int adapter_of(const Problem &p, int m)
{
    const int id = p.ids[m];
    return id >= 0 && id < p.adapters ? id : -1;
}

// The rows of this slot's tile: their number (0: none) and, in `rows`, which; `id` their adapter, -1 for rows without one.
__device__ int rows_of(const Problem &p, int slot, int (&rows)[kTile], unsigned long long (&alike)[kWaves], int &id)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (p.order) {
        const Tile tile = p.tiles[slot];
        id = tile.id;
        if (tid < tile.count) rows[tid] = p.order[tile.first + tid];
        __syncthreads();
        return tile.count;
    }
    // the first, 17th, ... row of an adapter's takes its next 16
    id = adapter_of(p, slot);
    const bool mine = tid < p.M && adapter_of(p, tid) == id;
    const unsigned long long ballot = __ballot(mine);
    if (lane == 0) alike[wave] = ballot;
    __syncthreads();
    int ahead = 0, before_slot = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const unsigned long long b = alike[w];
        all += __popcll(b);
        ahead += w < wave ? __popcll(b) : w == wave ? __popcll(b & ((1ull << lane) - 1)) : 0;
        before_slot += w < slot >> 6 ? __popcll(b) : w == slot >> 6 ? __popcll(b & ((1ull << (slot & 63)) - 1)) : 0;
    }
    if (before_slot % kTile != 0) return 0;
    const int place = ahead - before_slot;
    if (mine && place >= 0 && place < kTile) rows[place] = tid;
    __syncthreads();
    return min(all - before_slot, kTile);
}

// Sorts the rows of a problem by adapter (rows without one in a tile of their own) and cuts them into tiles.  One workgroup; the order of
// adapters and of an adapter's rows is any, which makes no difference to results.  Bound by its chain of round trips: a row's place among
// its adapter's is found once and kept.
__global__ void __launch_bounds__(1024) sort_kernel(const Args args)
{
    constexpr int kOwn = (kMaxAdapters + 1 + 1023) / 1024, kRows = 4;
    __shared__ int rows[kMaxAdapters + 1];
    __shared__ int wave_rows[16], wave_tiles[16];
    const Problem &p = args.p[blockIdx.x];
    if (!p.order) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kinds = p.adapters + 1;
    for (int a = tid; a < kinds; a += 1024) rows[a] = 0;
    auto kind_of = [&](int m) {
        const int id = m < p.M ? adapter_of(p, m) : 0;
        return id < 0 ? p.adapters : id;
    };
    // (a row's kind and place stay in registers where a thread has no more rows than it looks at at a time)
    const bool once = p.M <= kRows * 1024;
    int kind[kRows], places[kRows];
    __syncthreads();
    for (int m0 = tid; m0 - tid < p.M; m0 += kRows * 1024) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) kind[i] = kind_of(m0 + 1024 * i);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            // Additions to one address are made one after the other, and the rows of a prompt are beside each other: those of a wave's
            // first row's kind are added at once.
            const int m = m0 + 1024 * i, its = __builtin_amdgcn_readfirstlane(kind[i]);
            const unsigned long long same = __ballot(m < p.M && kind[i] == its);
            int place = 0;
            if (lane == 0 && same) place = atomicAdd(&rows[its], __popcll(same));
            place = __builtin_amdgcn_readfirstlane(place) + __popcll(same & ((1ull << lane) - 1));
            places[i] = 0;
            if (m >= p.M) continue;
            if (kind[i] != its) place = atomicAdd(&rows[kind[i]], 1);
            places[i] = place;
            if (!once) p.places[m] = place;
        }
    }
    __syncthreads();
    int own[kOwn], own_rows = 0, own_tiles = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        const int a = tid + 1024 * i;
        own[i] = a < kinds ? rows[a] : 0;
        own_rows += own[i];
        own_tiles += (own[i] + kTile - 1) / kTile;
    }
    int to_rows = own_rows, to_tiles = own_tiles;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int r = __shfl_up(to_rows, d), t = __shfl_up(to_tiles, d);
        to_rows += lane >= d ? r : 0;
        to_tiles += lane >= d ? t : 0;
    }
    if (lane == 63) {
        wave_rows[wave] = to_rows;
        wave_tiles[wave] = to_tiles;
    }
    __syncthreads();
    int first = to_rows - own_rows, tile = to_tiles - own_tiles, tiles = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        first += w < wave ? wave_rows[w] : 0;
        tile += w < wave ? wave_tiles[w] : 0;
        tiles += wave_tiles[w];
    }
    for (int i = 0; i < kOwn; ++i) {
        const int a = tid + 1024 * i;
        if (a - tid >= kinds) break;
        const int mine = a < kinds ? rows[a] : 0;   // (own[i]; still a count)
        // a kind of many tiles is written by the whole wave, one of few by its thread
        unsigned long long large = __ballot(mine > 4 * kTile);
        while (large) {
            const int l = __ffsll((long long)large) - 1, its_rows = __shfl(mine, l), its_first = __shfl(first, l), its_tile = __shfl(tile, l), its = __shfl(a, l);
            for (int t = lane; t * kTile < its_rows; t += 64)
                p.tiles[its_tile + t] = {its < p.adapters ? its : -1, its_first + t * kTile, min(its_rows - t * kTile, kTile)};
            large &= large - 1;
        }
        if (mine <= 4 * kTile)
            for (int t = 0; t * kTile < mine; ++t) p.tiles[tile + t] = {a < p.adapters ? a : -1, first + t * kTile, min(mine - t * kTile, kTile)};
        if (a < kinds) rows[a] = first;   // (from here on: where the kind's rows begin)
        first += mine;
        tile += (mine + kTile - 1) / kTile;
    }
    for (int t = tiles + tid; t < p.slots; t += 1024) p.tiles[t] = {-1, 0, 0};
    __syncthreads();
    for (int m0 = tid; m0 < p.M; m0 += kRows * 1024) {
        if (!once) {
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                kind[i] = kind_of(m0 + 1024 * i);
                places[i] = p.places[min(m0 + 1024 * i, p.M - 1)];
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            if (m0 + 1024 * i < p.M) p.order[rows[kind[i]] + places[i]] = m0 + 1024 * i;
    }
}

// A part of h for the rows of a tile.  A wave takes 128 inputs at a time, 32 to an instruction, so that its loads cover 64 bytes of a row
// side by side.
template <int NT>   // tiles of 16 ranks, at least as many as there are
__global__ void __launch_bounds__(kThreads) down_kernel(const Args args)
{
    __shared__ float parts[kWaves][NT * 16][kTile + 1];
    __shared__ int rows[kTile];
    __shared__ unsigned long long alike[kWaves];
    const Problem &p = args.p[blockIdx.z];
    const int slot = blockIdx.x, split = blockIdx.y;
    if (slot >= p.slots || split >= p.k_splits) return;
    int id;
    const int count = rows_of(p, slot, rows, alike, id);
    if (count == 0 || id < 0) return;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, column = lane & 15, quad = lane >> 4;
    const _Float16 *x = p.x + rows[min(column, count - 1)] * p.x_stride;
    const _Float16 *down = p.down + (size_t)id * p.rank * p.K;
    const int from = split * p.k_own, to = min(from + p.k_own, p.K), rank_tiles = (p.rank + 15) / 16;
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    // (operands of the next inputs are asked for before these are multiplied; of more than 64 ranks those of x only)
    constexpr int kAhead = NT <= 4 ? NT : 0;
    const f16x8 zero = (f16x8)((_Float16)0.0f);
    f16x8 xv[4], dv[kAhead > 0 ? kAhead : 1][4];
    auto row_of = [&](int t, int k) { return down + (size_t)min(16 * t + column, p.rank - 1) * p.K + k; };
    auto fetch = [&](int k0) {
        const int k = k0 + quad * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[i] = k0 + 32 * i < p.K ? *(const f16x8 *)(x + k + 32 * i) : zero;
#pragma unroll
        for (int t = 0; t < kAhead; ++t)
            if (t < rank_tiles) {
#pragma unroll
                for (int i = 0; i < 4; ++i) dv[t][i] = k0 + 32 * i < p.K ? *(const f16x8 *)(row_of(t, k) + 32 * i) : zero;
            }
    };
    int k0 = from + wave * kDepth;
    if (k0 < to) fetch(k0);
    for (; k0 < to; k0 += kWaves * kDepth) {
        const int k = k0 + quad * 8;
        f16x8 xc[4], dc[kAhead > 0 ? kAhead : 1][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            xc[i] = xv[i];
#pragma unroll
            for (int t = 0; t < kAhead; ++t) dc[t][i] = dv[t][i];
        }
        if (k0 + kWaves * kDepth < to) fetch(k0 + kWaves * kDepth);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (t < rank_tiles) {
                f16x8 d[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i] = t < kAhead ? dc[t < kAhead ? t : 0][i] : k0 + 32 * i < p.K ? *(const f16x8 *)(row_of(t, k) + 32 * i) : zero;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(d[i], xc[i], acc[t], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) parts[wave][16 * t + 4 * quad + i][column] = acc[t][i];
    __syncthreads();
    float *h = p.h + (size_t)split * p.M * p.rank;
    for (int u = tid; u < count * p.rank; u += kThreads) {
        const int row = u / p.rank, r = u % p.rank;
        float sum = parts[0][r][row];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += parts[w][r][row];
        h[(size_t)rows[row] * p.rank + r] = sum;
    }
}

// out for the rows of a tile and some outputs.  A wave takes 64 outputs at a time in four instructions, whose 16 outputs are dealt out so
// that a lane ends up with 16 neighbouring ones of its row.
template <int RT>   // steps of 32 ranks, at least as many as there are
__global__ void __launch_bounds__(kThreads) up_kernel(const Args args)
{
    constexpr int kPadded = RT * 32 + 8;
    __shared__ _Float16 high[kTile][kPadded], low[kTile][kPadded];
    __shared__ float back[kTile];   // what a row's sums are multiplied by
    __shared__ int rows[kTile];
    __shared__ unsigned long long alike[kWaves];
    const Problem &p = args.p[blockIdx.z];
    const int slot = blockIdx.x, from = blockIdx.y * p.n_own;
    if (slot >= p.slots || from >= p.N) return;
    const int to = min(from + p.n_own, p.N);
    int id;
    const int count = rows_of(p, slot, rows, alike, id);
    if (count == 0) return;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, column = lane & 15, quad = lane >> 4;
    if (id < 0) {
        if (p.out == p.base) return;
        const int fours = (to - from) / 4;
        for (int u = tid; u < count * fours; u += kThreads) {
            const int m = rows[u / fours], n = from + u % fours * 4;
            *(f16x4 *)(p.out + m * p.out_stride + n) = *(const f16x4 *)(p.base + m * p.base_stride + n);
        }
        return;
    }
    // What a wave multiplies and adds to is asked for ahead: before h is there, and for the next outputs before these are done.
    const int m = rows[min(column, count - 1)];
    const _Float16 *base = p.base + m * p.base_stride;
    _Float16 *out = p.out + m * p.out_stride;
    const _Float16 *up = p.up + (size_t)id * p.N * p.rank;
    typedef _Float16 f16x8_by4 __attribute__((ext_vector_type(8), aligned(8)));   // (base and out are 8-byte aligned)
    f16x8 ahead[4][RT], added[2];
    auto fetch = [&](int n0) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            // instruction t's row `column` is output (column / 4) * 16 + 4 t + column % 4
            const _Float16 *row = up + (size_t)min(n0 + column / 4 * 16 + 4 * t + column % 4, p.N - 1) * p.rank;
#pragma unroll
            for (int s = 0; s < RT; ++s) {
                const int r = 32 * s + 8 * quad;
                ahead[t][s] = r < p.rank ? *(const f16x8 *)(row + r) : (f16x8)((_Float16)0.0f);
            }
        }
        // a lane's 16 outputs, by eights; eight that are not there whole are looked for when they are needed
        const int n = n0 + 16 * quad;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (n + 8 * h + 8 <= to) added[h] = *(const f16x8_by4 *)(base + n + 8 * h);
    };
    int n0 = from + wave * kColumns;
    if (n0 < to) fetch(n0);
    {   // h of the rows: 16 threads each
        const int row = tid / 16, part = tid % 16;
        const bool live = row < count;
        const float *h = p.h + (size_t)rows[live ? row : 0] * p.rank;
        float v[RT * 2], most = 0.0f;
#pragma unroll
        for (int i = 0; i < RT * 2; ++i) v[i] = 0.0f;
#pragma unroll 4
        for (int s = 0; s < p.k_splits; ++s) {
#pragma unroll
            for (int i = 0; i < RT * 2; ++i) {
                const int r = part + 16 * i;
                v[i] += r < p.rank && live ? h[(size_t)s * p.M * p.rank + r] : 0.0f;
            }
        }
        // (infinite ones are left out: they stay infinite whatever they are scaled by)
#pragma unroll
        for (int i = 0; i < RT * 2; ++i) most = fabsf(v[i]) < INFINITY ? fmaxf(most, fabsf(v[i])) : most;
#pragma unroll
        for (int d = 1; d < 16; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
        // (a power of two not below the largest, inside what can be inverted)
        const int exponent = most > 0.0f ? min(max(__builtin_amdgcn_frexp_expf(most), -100), 100) : 0;
#pragma unroll
        for (int i = 0; i < RT * 2; ++i) {
            const float scaled = __builtin_amdgcn_ldexpf(v[i], -exponent);
            const _Float16 hi = (_Float16)scaled;
            high[row][part + 16 * i] = hi;
            low[row][part + 16 * i] = fabsf(scaled) < INFINITY ? (_Float16)(scaled - (float)hi) : (_Float16)0.0f;
        }
        if (part == 0) back[row] = __builtin_amdgcn_ldexpf(p.scale ? p.scale[id] : 1.0f, exponent);
    }
    __syncthreads();
    f16x8 hi[RT], lo[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        hi[t] = *(const f16x8 *)&high[column][32 * t + 8 * quad];
        lo[t] = *(const f16x8 *)&low[column][32 * t + 8 * quad];
    }
    const float scale = back[column];
    for (; n0 < to; n0 += kWaves * kColumns) {
        f32x4 acc[4];
        f16x8 b[2];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            acc[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < RT; ++s) {
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ahead[t][s], hi[s], acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ahead[t][s], lo[s], acc[t], 0, 0, 0);
            }
        }
        b[0] = added[0];
        b[1] = added[1];
        if (n0 + kWaves * kColumns < to) fetch(n0 + kWaves * kColumns);
        if (column < count) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = n0 + 16 * quad + 8 * h;
                auto result = [&](int i, _Float16 was) { return (_Float16)fmaf(acc[2 * h + i / 4][i % 4], scale, (float)was); };
                if (n + 8 <= to) {
                    f16x8 o;
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = result(i, b[h][i]);
                    *(f16x8_by4 *)(out + n) = o;
                } else if (n < to) {
                    const f16x4 was = *(const f16x4 *)(base + n);
                    f16x4 o;
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = result(i, was[i]);
                    *(f16x4 *)(out + n) = o;
                }
            }
        }
    }
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
        if (p.rank < 8 || p.rank > 256 || p.rank % 8 != 0 || p.adapters < 1 || p.adapters > kMaxAdapters) return LUTGEMM_EINVAL;
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

// How a problem is cut, and the bytes of workspace that it takes.
struct Cut {
    int slots, k_splits, k_own, n_own;
    size_t h_bytes, tile_bytes, order_bytes;
    size_t bytes() const { return h_bytes + tile_bytes + order_bytes; }
};

size_t round16(size_t bytes) { return (bytes + 15) / 16 * 16; }

Cut cut_of(const lutgemm_adapters &p)
{
    Cut c;
    const bool sorted = p.M > kUnsorted;
    // tiles: full ones, and one for each kind of rows that is left
    const int kinds = p.adapters + 1 < p.M ? p.adapters + 1 : p.M;
    c.slots = sorted ? p.M / kTile + kinds : p.M;
    const int expected = sorted ? (p.M + kTile - 1) / kTile : p.M;
    // workgroups enough for the CUs, as long as each wave has a step of its own
    const int most = (p.K + kWaves * kDepth - 1) / (kWaves * kDepth);
    int splits = (1024 + expected - 1) / expected;
    if (splits > most) splits = most;
    if (splits > 32) splits = 32;
    const int steps = (p.K + kDepth - 1) / kDepth;
    c.k_own = (steps + splits - 1) / splits * kDepth;
    c.k_splits = (p.K + c.k_own - 1) / c.k_own;
    // (as many workgroups as the CUs hold at once; each finds its rows and their h first.  48 rows 4096 to 11008 of rank 64: 1024 workgroups
    // 26.0 us, 2048 29.1, 512 26.9)
    const int chunks = (p.N + kWaves * kColumns - 1) / (kWaves * kColumns), wanted = (1024 + expected - 1) / expected;
    c.n_own = (chunks + wanted - 1) / wanted * kWaves * kColumns;
    c.h_bytes = round16((size_t)c.k_splits * p.M * p.rank * 4);
    c.tile_bytes = sorted ? round16((size_t)c.slots * sizeof(Tile)) : 0;
    c.order_bytes = sorted ? round16((size_t)p.M * 8) : 0;
    return c;
}

}  // namespace

extern "C" {

size_t lutgemm_adapters_workspace(int count, const lutgemm_adapters *problems)
{
    if (check(count, problems) != LUTGEMM_OK) return 0;
    size_t bytes = 0;
    for (int i = 0; i < count; ++i) bytes += cut_of(problems[i]).bytes();
    return bytes;
}

int lutgemm_adapters_f16(int count, const lutgemm_adapters *problems, void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = check(count, problems);
    if (rc != LUTGEMM_OK) return rc;
    if (!workspace) return LUTGEMM_EINVAL;
    Args a{};
    a.count = count;
    char *at = (char *)workspace;
    size_t bytes = 0;
    int slots = 0, splits = 0, chunks = 0, rank = 0;
    bool sorted = false;
    for (int i = 0; i < count; ++i) {
        const lutgemm_adapters &p = problems[i];
        const Cut c = cut_of(p);
        const bool own_order = c.order_bytes > 0;
        a.p[i] = {(const _Float16 *)p.x_f16, (const _Float16 *)p.base_f16, (_Float16 *)p.out_f16, p.ids, (const _Float16 *)p.down_f16,
                  (const _Float16 *)p.up_f16, p.scale, p.x_stride, p.base_stride, p.out_stride, p.M, p.N, p.K, p.rank, p.adapters,
                  c.slots, c.k_splits, c.k_own, c.n_own, (float *)at, own_order ? (Tile *)(at + c.h_bytes) : nullptr,
                  own_order ? (int32_t *)(at + c.h_bytes + c.tile_bytes) : nullptr,
                  own_order ? (int32_t *)(at + c.h_bytes + c.tile_bytes) + p.M : nullptr};
        at += c.bytes();
        bytes += c.bytes();
        slots = c.slots > slots ? c.slots : slots;
        splits = c.k_splits > splits ? c.k_splits : splits;
        const int own_chunks = (p.N + c.n_own - 1) / c.n_own;
        chunks = own_chunks > chunks ? own_chunks : chunks;
        rank = p.rank > rank ? p.rank : rank;
        sorted |= own_order;
    }
    if (workspace_bytes < bytes) return LUTGEMM_EINVAL;
    if (!aligned(workspace, 16)) return LUTGEMM_EALIGN;
    const hipStream_t hs = (hipStream_t)stream;
    const dim3 threads(kThreads), down_grid(slots, splits, count), up_grid(slots, chunks, count);
    if (sorted) {
        hipLaunchKernelGGL(sort_kernel, dim3(count), dim3(1024), 0, hs, a);
        const int status = launch_status();
        if (status != LUTGEMM_OK) return status;
    }
    auto launch = [&](auto down, auto up) {
        hipLaunchKernelGGL(down, down_grid, threads, 0, hs, a);
        const int status = launch_status();
        if (status != LUTGEMM_OK) return status;
        hipLaunchKernelGGL(up, up_grid, threads, 0, hs, a);
        return launch_status();
    };
    if (rank <= 16) return launch(down_kernel<1>, up_kernel<1>);
    if (rank <= 32) return launch(down_kernel<2>, up_kernel<1>);
    if (rank <= 64) return launch(down_kernel<4>, up_kernel<2>);
    if (rank <= 128) return launch(down_kernel<8>, up_kernel<4>);
    return launch(down_kernel<16>, up_kernel<8>);
}

}  // extern "C"
