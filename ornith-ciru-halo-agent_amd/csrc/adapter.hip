// Low-rank adapters of many requests beside a shared projection (definition:
// include/ornith_adapter.h).
//
// Rows are sorted by slot into tiles of one adapter.  Two products on the
// matrix cores, each row's sums its own:
//   shrink  v[t, r] = sum_k x[t, k] A[r, k]: a block per tile and chunk of r,
//           its waves share k and meet in LDS in wave order;
//   expand  out[t, n] = base[t, n] + scale sum_r B[n, r] v[t, r]: v, fp32, as the
//           sum of two 16-bit numbers hi + lo side by side along r, so the
//           second product loses no more than 2^-17 of it.  The product is
//           formed transposed (columns as rows of the instruction), with the
//           columns dealt so that a lane ends with 16 neighbouring ones of one
//           row: base and out move in 16-byte accesses, 128 bytes a row and wave.
#include <algorithm>
#include <type_traits>
#include "kernels.hpp"
#include "timing.hpp"
#include "validate.hpp"
#include "../../include/ornith_adapter.h"

namespace ornith {
namespace {

constexpr int kAdMaxN = 1 << 20, kAdMaxK = 65536, kAdMaxSlices = ORNITH_ADAPTER_MAX_SLICES,
              kAdMaxSlots = ORNITH_ADAPTER_MAX_SLOTS, kAdMaxR = ORNITH_ADAPTER_MAX_RANK;
constexpr int kAdRows = 1 << 20;                       // rows of one pass
enum : uint32_t { kAdNonfinite = 4, kAdNonfinite16 = 8, kAdBadId = 16 };

typedef __bf16 ad_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 ad_f16x8 __attribute__((ext_vector_type(8)));

template <int TYPE> __device__ __forceinline__ f32x4 ad_mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (TYPE == ORNITH_ADAPTER_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ad_bf16x8, a),
                                                       __builtin_bit_cast(ad_bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ad_f16x8, a),
                                                      __builtin_bit_cast(ad_f16x8, b), c, 0, 0, 0);
}

struct AdTile { int slot, first, rows; };              // rows order[first ..]; slot -1: no adapter

struct AdArgs {
    const uint16_t* x; int64_t ldx;
    const uint16_t* a; int64_t a_slot;
    const uint16_t* b; int64_t b_slot;
    const float* scales;
    const int32_t* ids;
    const void* base; int64_t ldb;
    void* out; int64_t ldo;
    uint32_t* flags;
    float* v;                                          // [M, SR]
    int32_t* order;                                    // [M]
    AdTile* tiles;
    int32_t* ntiles;
    int M, N, K, R, SR, slots, S;
    bool in_place;
    int ends[kAdMaxSlices];                            // of the slices, in columns
    int blocks[kAdMaxSlices];                          // of the expand's column blocks, running
};

// ---- rows by slot ---------------------------------------------------------------
// One block: counts per slot in LDS, their running sums, then each row to a place of its slot.  Which
// place it gets is open (atomics), and no result depends on it: rows of a tile do not meet.
constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int ad_key(const AdArgs& a, int t) {     // 0: no adapter
    const int id = a.ids[t];
    return id >= 0 && id < a.slots ? id + 1 : 0;
}
__device__ __forceinline__ int block_prefix(int v, int* s_wave, int& total) {      // inclusive, over kPlanThreads
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int in = wave_prefix_sum(v);
    if (lane == 63) s_wave[wv] = in;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        if (w < wv) before += s_wave[w];
        total += s_wave[w];
    }
    __syncthreads();
    return in + before;
}

__global__ __launch_bounds__(kPlanThreads) void adapter_plan_kernel(AdArgs a, int tile_rows) {
    __shared__ int s_count[kAdMaxSlots + 1], s_at[kAdMaxSlots + 1], s_wave[kPlanThreads / 64];
    const int tid = threadIdx.x, keys = a.slots + 1;
    for (int i = tid; i < keys; i += kPlanThreads) s_count[i] = 0;
    __syncthreads();
    uint32_t flags = 0;
    for (int t = tid; t < a.M; t += kPlanThreads) {
        flags |= a.ids[t] >= a.slots ? kAdBadId : 0u;
        atomicAdd(&s_count[ad_key(a, t)], 1);
    }
    flag_or(a.flags, flags);
    __syncthreads();
    int rows = 0, tiles = 0;
    for (int i0 = 0; i0 < keys; i0 += kPlanThreads) {
        const int i = i0 + tid, n = i < keys ? s_count[i] : 0;
        const int nt = i == 0 && a.in_place ? 0 : (n + tile_rows - 1) / tile_rows;
        int all, all_tiles;
        const int first = rows + block_prefix(n, s_wave, all) - n;
        const int tile0 = tiles + block_prefix(nt, s_wave, all_tiles) - nt;
        if (i < keys) s_at[i] = first;
        for (int j = 0; j < nt; ++j)
            a.tiles[tile0 + j] = AdTile{i - 1, first + j * tile_rows, min(n - j * tile_rows, tile_rows)};
        rows += all;
        tiles += all_tiles;
    }
    if (tid == 0) *a.ntiles = tiles;
    __syncthreads();
    for (int t = tid; t < a.M; t += kPlanThreads) a.order[atomicAdd(&s_at[ad_key(a, t)], 1)] = t;
}

// ---- shrink ---------------------------------------------------------------------
constexpr int kShrinkWaves = 8;

template <int TYPE, int MT, int RT>
__global__ __launch_bounds__(64 * kShrinkWaves) void adapter_shrink_kernel(AdArgs a) {
    constexpr int W = kShrinkWaves;
    __shared__ f32x4 s_acc[W][MT * RT][64];
    if (int(blockIdx.x) >= *a.ntiles) return;
    const AdTile tile = a.tiles[blockIdx.x];
    if (tile.slot < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, q = lane >> 4;
    const int r0 = int(blockIdx.y) * 16 * RT;
    const uint16_t *x[MT], *w[RT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {                     // (past the last row: that one again)
        const int t = a.order[tile.first + min(16 * m + li, tile.rows - 1)];
        x[m] = a.x + size_t(t) * size_t(a.ldx) + 8 * q;
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
        w[r] = a.a + size_t(tile.slot) * size_t(a.a_slot) + size_t(min(r0 + 16 * r + li, a.SR - 1)) * size_t(a.K) + 8 * q;
    f32x4 acc[MT][RT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[m][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 64 * wv; k0 < a.K; k0 += 64 * W) {
        u32x4 xv[2][MT], wf[2][RT];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = k0 + 32 * h;
            const bool in = k + 8 * q < a.K;
#pragma unroll
            for (int m = 0; m < MT; ++m) xv[h][m] = in ? *reinterpret_cast<const u32x4*>(x[m] + k) : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < RT; ++r) wf[h][r] = in ? *reinterpret_cast<const u32x4*>(w[r] + k) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[m][r] = ad_mfma<TYPE>(xv[h][m], wf[h][r], acc[m][r]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < RT; ++r) s_acc[wv][m * RT + r][lane] = acc[m][r];
    __syncthreads();
    for (int f = wv; f < MT * RT; f += W) {
        f32x4 v = s_acc[0][f][lane];
#pragma unroll
        for (int u = 1; u < W; ++u) {
            const f32x4 p = s_acc[u][f][lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += p[i];
        }
        const int m = f / RT, r = r0 + 16 * (f % RT) + li;
        if (r < a.SR) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 16 * m + 4 * q + i;
                if (row < tile.rows) a.v[size_t(tile.first + row) * a.SR + r] = v[i];
            }
        }
    }
}

// ---- expand ---------------------------------------------------------------------
template <int OUT> __device__ __forceinline__ float ad_get(const void* p, size_t at) {
    if constexpr (OUT == ORNITH_ADAPTER_F32) return static_cast<const float*>(p)[at];
    else if constexpr (OUT == ORNITH_ADAPTER_BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[at]);
    else return f16_bits_to_f32(static_cast<const uint16_t*>(p)[at]);
}
template <int OUT> __device__ __forceinline__ void ad_put(void* p, size_t at, float v) {
    if constexpr (OUT == ORNITH_ADAPTER_F32) static_cast<float*>(p)[at] = v;
    else if constexpr (OUT == ORNITH_ADAPTER_BF16) static_cast<__bf16*>(p)[at] = static_cast<__bf16>(v);
    else static_cast<_Float16*>(p)[at] = static_cast<_Float16>(v);
}
template <int TYPE> __device__ __forceinline__ float ad_round(float v) {
    return TYPE == ORNITH_ADAPTER_BF16 ? float(static_cast<__bf16>(v)) : float(static_cast<_Float16>(v));
}
template <int TYPE> __device__ __forceinline__ uint16_t ad_bits(float v) {
    if constexpr (TYPE == ORNITH_ADAPTER_BF16) return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
    else return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}
// Power of two that brings a row's largest |v| to [2^14, 2^15) of fp16, as fp32 (1 for 0 and non-finite rows).
__device__ __forceinline__ float ad_scale16(uint32_t most) {
    const int e = int(most >> 23);
    if (e == 0 || e == 255) return 1.f;
    return __uint_as_float(uint32_t(min(max(127 + 127 + 14 - e, 1), 254)) << 23);
}

constexpr int kExpandWaves = 4, kExpandGroups = 4;      // of 64 columns, a block

template <int TYPE, int OUT, int MT>
__global__ __launch_bounds__(64 * kExpandWaves) void adapter_expand_kernel(AdArgs a) {
    extern __shared__ __attribute__((aligned(16))) u32x4 s_v[];        // [MT][steps][64]
    __shared__ uint32_t s_most[16 * MT];
    if (int(blockIdx.x) >= *a.ntiles) return;
    const AdTile tile = a.tiles[blockIdx.x];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, q = lane >> 4;
    int p = 0;
    while (int(blockIdx.y) >= a.blocks[p]) ++p;
    const int begin = p ? a.ends[p - 1] : 0, end = a.ends[p];
    const int group0 = (int(blockIdx.y) - (p ? a.blocks[p - 1] : 0)) * kExpandGroups;
    const int chunks = a.R / 8, steps = (2 * chunks + 3) / 4;
    if (tile.slot >= 0) {
        // v of the tile's rows and this slice: hi then lo along r, in pieces of 8, as the instruction's operands
        const int rows = 16 * MT, pieces = rows * chunks;
        if constexpr (TYPE == ORNITH_ADAPTER_F16) {
            if (tid < rows) s_most[tid] = 0;
            __syncthreads();
            for (int i = tid; i < pieces; i += 64 * kExpandWaves) {
                const int row = i / chunks;
                if (row >= tile.rows) continue;
                const float* v = a.v + size_t(tile.first + row) * a.SR + p * a.R + (i % chunks) * 8;
                uint32_t most = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
                atomicMax(&s_most[row], most);
            }
            __syncthreads();
        }
        for (int i = tid; i < 16 * MT * steps * 4; i += 64 * kExpandWaves) {
            const int row = i / (steps * 4), c = i % (steps * 4);
            u32x4 piece = {0, 0, 0, 0};
            if (row < tile.rows && c < 2 * chunks) {
                const float* v = a.v + size_t(tile.first + row) * a.SR + p * a.R + (c % chunks) * 8;
                const float by = TYPE == ORNITH_ADAPTER_F16 ? ad_scale16(s_most[row]) : 1.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float f = v[e] * by, hi = ad_round<TYPE>(f);
                    const float lo = f - hi;           // (inf: no NaN beside it)
                    const uint32_t bits = c < chunks ? ad_bits<TYPE>(f) : __builtin_isinf(hi) ? 0u : ad_bits<TYPE>(lo);
                    piece[e >> 1] |= bits << (16 * (e & 1));
                }
            }
            s_v[((row >> 4) * steps + (c >> 2)) * 64 + (c & 3) * 16 + (row & 15)] = piece;
        }
        __syncthreads();
    }
    constexpr int size = OUT == ORNITH_ADAPTER_F32 ? 4 : 2;
    int t[MT];
    float by[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        t[m] = a.order[tile.first + min(16 * m + li, tile.rows - 1)];
        by[m] = 0.f;
        if (tile.slot >= 0) {
            by[m] = a.scales[tile.slot];
            if constexpr (TYPE == ORNITH_ADAPTER_F16) by[m] = by[m] / ad_scale16(s_most[16 * m + li]);
        }
    }
    float most = 0.f, zero = 0.f;
    for (int gi = wv; gi < kExpandGroups; gi += kExpandWaves) {
        const int n0 = begin + (group0 + gi) * 64;
        if (n0 >= end) break;
        const int n = n0 + 16 * q;                     // this lane's columns n .. n + 15
        if (tile.slot < 0) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
                if (16 * m + li < tile.rows)
                    for (int i = 0; i < 16; ++i)
                        if (n + i < end) {
                            const size_t to = size_t(t[m]) * size_t(a.ldo) + n + i, from = size_t(t[m]) * size_t(a.ldb) + n + i;
                            if constexpr (size == 4) static_cast<uint32_t*>(a.out)[to] = static_cast<const uint32_t*>(a.base)[from];
                            else static_cast<uint16_t*>(a.out)[to] = static_cast<const uint16_t*>(a.base)[from];
                        }
            continue;
        }
        f32x4 acc[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) acc[m][jj] = f32x4{0.f, 0.f, 0.f, 0.f};
        const uint16_t* b = a.b + size_t(tile.slot) * size_t(a.b_slot);
        for (int s = 0; s < steps; ++s) {
            const int c = 4 * s + q;
            u32x4 bv[4];
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                const int col = min(n0 + 16 * (li >> 2) + 4 * jj + (li & 3), end - 1);
                bv[jj] = c < 2 * chunks ? *reinterpret_cast<const u32x4*>(b + size_t(col) * a.R + (c % chunks) * 8) : u32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const u32x4 vv = s_v[(m * steps + s) * 64 + lane];
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) acc[m][jj] = ad_mfma<TYPE>(bv[jj], vv, acc[m][jj]);
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (16 * m + li >= tile.rows) continue;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (n + i >= end) continue;
                const float r = ad_get<OUT>(a.base, size_t(t[m]) * size_t(a.ldb) + n + i) + by[m] * acc[m][i >> 2][i & 3];
                most = fmaxf(most, __builtin_fabsf(r));
                zero = __builtin_fmaf(r, 0.f, zero);
                ad_put<OUT>(a.out, size_t(t[m]) * size_t(a.ldo) + n + i, r);
            }
        }
    }
    // 16-bit results round to infinity from half a step above the type's largest value
    const bool bad = zero != zero;
    constexpr float limit = OUT == ORNITH_ADAPTER_BF16 ? 0x1.ffp127f : 65520.f;
    flag_or(a.flags, (bad ? kAdNonfinite : 0u) | (OUT != ORNITH_ADAPTER_F32 && (bad || most >= limit) ? kAdNonfinite16 : 0u));
}

struct AdLayout { size_t v, order, tiles, count, bytes; };

bool ad_layout(int64_t M, int S, int R, AdLayout& l) {
    if (M < 0 || S < 1 || S > kAdMaxSlices || R < 8 || R > kAdMaxR || R % 8) return false;
    const size_t rows = size_t(std::min<int64_t>(M, kAdRows));
    l.v = 0;
    l.order = align256(rows * size_t(S) * size_t(R) * 4);
    l.tiles = l.order + align256(rows * 4);
    l.count = l.tiles + align256(rows * sizeof(AdTile));
    l.bytes = l.count + 256;
    return true;
}

template <int TYPE, int MT> hipError_t ad_run(const AdArgs& a, int out_type, int tiles, hipStream_t s) {
    const int rt = (a.SR + 15) / 16;
    auto shrink = [&](auto kernel, int RT) {
        timed_launch("adapter_shrink", kernel, dim3(tiles, (rt + RT - 1) / RT), dim3(64 * kShrinkWaves), 0, s, a);
    };
    shrink(adapter_shrink_kernel<TYPE, MT, 1>, 1);
    hipError_t st = hipGetLastError();
    if (st != hipSuccess) return st;
    const int steps = (a.R / 4 + 3) / 4;
    auto expand = [&](auto kernel) {
        timed_launch("adapter_expand", kernel, dim3(tiles, a.blocks[a.S - 1]), dim3(64 * kExpandWaves), uint32_t(MT * steps * 1024), s, a);
    };
    if (out_type == ORNITH_ADAPTER_F32) expand(adapter_expand_kernel<TYPE, ORNITH_ADAPTER_F32, MT>);
    else if (out_type == ORNITH_ADAPTER_BF16) expand(adapter_expand_kernel<TYPE, ORNITH_ADAPTER_BF16, MT>);
    else expand(adapter_expand_kernel<TYPE, ORNITH_ADAPTER_F16, MT>);
    return hipGetLastError();
}

}  // namespace
}  // namespace ornith

using namespace ornith;

extern "C" hipError_t ornith_adapter_get_layout(int M, int S, int R, size_t* bytes) {
    AdLayout l;
    if (!bytes || !ad_layout(M, S, R, l)) return hipErrorInvalidValue;
    *bytes = l.bytes;
    return hipSuccess;
}

extern "C" hipError_t ornith_adapter_launch(const void* x, int x_type, int64_t ldx, const void* a, int64_t a_slot,
                                            const void* b, int64_t b_slot, const void* scales, const void* ids,
                                            const void* base, int64_t ldb, void* out, int out_type, int64_t ldo,
                                            void* workspace, size_t workspace_bytes, void* flags, int M, int N, int K,
                                            int R, int S, const int* slice_ends, int slots, hipStream_t stream) {
    AdLayout l;
    if (!ad_layout(M, S, R, l) || N < 0 || N > kAdMaxN || K < 0 || K > kAdMaxK || K % 8 || slots < 0 || slots > kAdMaxSlots ||
        (x_type != ORNITH_ADAPTER_BF16 && x_type != ORNITH_ADAPTER_F16) || out_type < ORNITH_ADAPTER_BF16 ||
        out_type > ORNITH_ADAPTER_F32 || !slice_ends || ldx < K || ldx % 8 || ldb < N || ldo < N || a_slot % 8 || b_slot % 8 ||
        a_slot < int64_t(S) * R * K || b_slot < int64_t(N) * R)
        return hipErrorInvalidValue;
    for (int p = 0; p < S; ++p)
        if (slice_ends[p] < (p ? slice_ends[p - 1] : 0) || slice_ends[p] > N || (p == S - 1 && slice_ends[p] != N))
            return hipErrorInvalidValue;
    if (!M || !N) return hipSuccess;
    constexpr int64_t kFar = int64_t(1) << 62;
    for (int64_t ld : {ldx, ldb, ldo})
        if (ld > kFar / 4 / M) return hipErrorInvalidValue;
    for (int64_t ld : {a_slot, b_slot})
        if (slots && ld > kFar / 2 / slots) return hipErrorInvalidValue;
    const size_t size = out_type == ORNITH_ADAPTER_F32 ? 4 : 2;
    const bool in_place = base == out;
    if (in_place && ldb != ldo) return hipErrorInvalidValue;
    const size_t out_bytes = (size_t(M - 1) * size_t(ldo) + size_t(N)) * size;
    const bool none = !slots;                          // no bank: base alone
    const Buffer buffers[] = {{x, K ? (size_t(M - 1) * size_t(ldx) + size_t(K)) * 2 : 0, 16, false, none || !K},
                              {a, none ? 0 : (size_t(slots - 1) * size_t(a_slot) + size_t(S) * R * K) * 2, 16, false, none || !K},
                              {b, none ? 0 : (size_t(slots - 1) * size_t(b_slot) + size_t(N) * R) * 2, 16, false, none},
                              {scales, size_t(slots) * 4, 4, false, none},
                              {ids, size_t(M) * 4, 4, false, false},
                              {in_place ? nullptr : base, (size_t(M - 1) * size_t(ldb) + size_t(N)) * size, size, false, in_place},
                              {out, out_bytes, size, true, false},
                              {workspace, l.bytes, 256, true, false},
                              {flags, 4, 4, true, false}};
    if (workspace_bytes < l.bytes || !base || !check_buffers(buffers)) return hipErrorInvalidValue;
    AdArgs args{};
    args.a = static_cast<const uint16_t*>(a);
    args.a_slot = a_slot;
    args.b = static_cast<const uint16_t*>(b);
    args.b_slot = b_slot;
    args.scales = static_cast<const float*>(scales);
    args.ldx = ldx;
    args.ldb = ldb;
    args.ldo = ldo;
    args.flags = static_cast<uint32_t*>(flags);
    args.v = at<float>(workspace, l.v);
    args.order = at<int32_t>(workspace, l.order);
    args.tiles = at<AdTile>(workspace, l.tiles);
    args.ntiles = at<int32_t>(workspace, l.count);
    args.N = N;
    args.K = K;
    args.R = R;
    args.SR = S * R;
    args.S = S;
    args.slots = slots;
    args.in_place = in_place;
    int blocks = 0;
    for (int p = 0; p < S; ++p) {
        args.ends[p] = slice_ends[p];
        const int width = slice_ends[p] - (p ? slice_ends[p - 1] : 0);
        blocks += (width + 64 * kExpandGroups - 1) / (64 * kExpandGroups);
        args.blocks[p] = blocks;
    }
    for (int64_t r = 0; r < M; r += kAdRows) {
        args.M = int(std::min<int64_t>(M - r, kAdRows));
        args.x = static_cast<const uint16_t*>(x) + size_t(r) * size_t(ldx);
        args.ids = static_cast<const int32_t*>(ids) + r;
        args.base = static_cast<const uint8_t*>(base) + size_t(r) * size_t(ldb) * size;
        args.out = static_cast<uint8_t*>(out) + size_t(r) * size_t(ldo) * size;
        const int tile_rows = 16, tiles = std::min(args.M, (args.M + tile_rows - 1) / tile_rows + slots + 1);
        timed_launch("adapter_plan", adapter_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, args, tile_rows);
        hipError_t st = hipGetLastError();
        if (st != hipSuccess) return st;
        st = x_type == ORNITH_ADAPTER_BF16 ? ad_run<ORNITH_ADAPTER_BF16, 1>(args, out_type, tiles, stream)
                                           : ad_run<ORNITH_ADAPTER_F16, 1>(args, out_type, tiles, stream);
        if (st != hipSuccess) return st;
    }
    return hipSuccess;
}
