// Low-rank adapters of many requests beside a shared projection (definition:
// include/ornith_adapter.h).
//
// Rows are sorted by slot into tiles of one adapter.  Two products on the
// matrix cores, each row's sums its own:
//   shrink  v[t, r] = sum_k x[t, k] A[r, k]: a block per tile and chunk of r,
//           its waves share k and meet in LDS in wave order;
//   expand  out[t, n] = base[t, n] + scale sum_r B[n, r] v[t, r]: scale v, fp32, as
//           the sum of two or three 16-bit numbers side by side along r.  The product is
//           formed transposed (columns as rows of the instruction) and goes
//           through LDS to lanes that move whole rows' pieces of base and out.
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
constexpr int kBothRank = 64;                          // ranks that both products of one launch take
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

// A planned tile: its slot (-1: no adapter, -2: no tile), its number of rows, and them; 2 + tile_rows words.
constexpr int kTileHead = 2;

struct AdArgs {
    const uint16_t* x; int64_t ldx;
    const uint16_t* a; int64_t a_slot;
    const uint16_t* b; int64_t b_slot;
    const float* scales;
    const int32_t* ids;
    const void* base; int64_t ldb;
    void* out; int64_t ldo;
    uint32_t* flags;
    float* v;                                          // [splits, M, SR]
    int32_t* tiles;                                    // [units, 2 + tile_rows]
    int tile_rows;
    int M, N, K, R, SR, slots, S;
    int splits;                                        // shrink: parts of K
    int units, groups;                                 // tiles at most; both: groups of 64 columns a wave
    bool in_place;
    int ends[kAdMaxSlices];                            // of the slices, in columns
    int blocks[kAdMaxSlices];                          // of the expand's column blocks, running
};

// ---- rows by slot ---------------------------------------------------------------
// Few rows (ad_few): no plan.  Block t of a launch looks at all ids, and if row t is the first, 17th, .. of its
// slot it takes that row and the next 15 of the slot; other blocks end.  (Up to 64 rows one id a lane, 64 rows of 6144
// columns, rank 16, 7.5 us; with four a lane 8.2.)
// More: one block counts rows per slot in LDS, sums, and sends each row to a place of its slot.  Which place
// it gets is open (atomics), and no result depends on it: rows of a tile do not meet.  (A launch, the ids'
// round trip and two passes over LDS: 4.2 us at 1120 rows, 7.8 at 8192.)
constexpr int kWaveRows = 64, kFewRows = 256, kPlanThreads = 1024, kPlanBatch = 8;

__device__ __forceinline__ int ad_key(int id, int slots) { return id >= 0 && id < slots ? id + 1 : 0; }      // 0: no adapter

// Lane li's row of tile `unit` (past the last row: that one again), its slot and how many rows; false where there is
// nothing to do.  FEW: ids a lane looks at (0: a plan; -1: a plan, and results off the 16-byte grid).  first: the launch's
// block that raises flags.
template <int MT, int FEW>
__device__ __forceinline__ bool ad_tile(const AdArgs& a, int unit, bool first, int& slot, int& rows, int (&t)[MT]) {
    const int lane = threadIdx.x & 63, li = lane & 15;
    if constexpr (FEW > 0) {
        static_assert(MT == 1);
        int key[FEW], mine = 0, before = 0, all = 0;
        uint64_t same[FEW];
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < FEW; ++j) key[j] = 64 * j + lane < a.M ? a.ids[64 * j + lane] : -1;
#pragma unroll
        for (int j = 0; j < FEW; ++j) {
            bad |= key[j] >= a.slots ? kAdBadId : 0u;
            key[j] = ad_key(key[j], a.slots);
            if (unit >> 6 == j) mine = __builtin_amdgcn_readlane(key[j], unit & 63);
        }
        if (first) flag_or(a.flags, bad);
#pragma unroll
        for (int j = 0; j < FEW; ++j) {
            same[j] = __ballot(key[j] == mine && 64 * j + lane < a.M);
            const int below = min(max(unit - 64 * j, 0), 64);                  // lanes of rows before this one
            before += __popcll(below < 64 ? same[j] & ((uint64_t(1) << below) - 1) : same[j]);
            all += __popcll(same[j]);
        }
        slot = mine - 1;
        rows = min(all - before, 16);
        if (before & 15) return false;
        int sent = 0, rank = -before;
#pragma unroll
        for (int j = 0; j < FEW; ++j) {
            const int r = rank + int(__builtin_amdgcn_mbcnt_hi(uint32_t(same[j] >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(same[j]), 0u)));
            const bool in = (same[j] >> lane & 1) && r >= 0 && r < 16;
            sent |= __builtin_amdgcn_ds_permute(4 * (in ? r : 63), in ? 64 * j + lane + 1 : 0);
            rank += __popcll(same[j]);
        }
        t[0] = __builtin_amdgcn_ds_bpermute(4 * min(li, rows - 1), sent) - 1;
    } else {
        const int32_t* tile = a.tiles + size_t(unit) * size_t(kTileHead + a.tile_rows);
        slot = tile[0];
        rows = tile[1];
#pragma unroll
        for (int m = 0; m < MT; ++m) t[m] = tile[kTileHead + 16 * m + li];    // (past its rows: of no use)
        if (slot < -1) return false;
#pragma unroll
        for (int m = MT - 1; m >= 0; --m) {            // (from the last: its source is not yet replaced)
            const int last = min(rows - 1, 16 * MT - 1), from = 16 * m + li <= last ? 16 * m + li : last;
            int row = t[0];
#pragma unroll
            for (int mm = 0; mm < MT; ++mm) {
                const int other = __builtin_amdgcn_ds_bpermute(4 * (from & 15), t[mm]);
                row = from >> 4 == mm ? other : row;
            }
            t[m] = row;
        }
    }
    return true;
}

__device__ __forceinline__ int block_prefix(int v, int* s_wave, int& total) {      // inclusive, over kPlanThreads
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int in = wave_prefix_sum(v);
    if (lane == 63) s_wave[wv] = in;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        const int x = s_wave[w];
        before += w < wv ? x : 0;
        total += x;
    }
    __syncthreads();
    return in + before;
}
// A place of counter[key] for each lane with a key >= 0.  Rows of a request are neighbours: the first two keys
// that a wave holds take one addition each.
__device__ __forceinline__ int ad_take(int* counter, int key) {
    int place = 0;
    bool left = key >= 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint64_t todo = __ballot(left);
        if (!todo) return place;
        const int first = __ffsll((long long)todo) - 1, lead = __builtin_amdgcn_readlane(key, first);
        const uint64_t same = __ballot(left && key == lead);
        int at = 0;
        if (int(threadIdx.x & 63) == first) at = atomicAdd(&counter[lead], __popcll(same));
        at = __builtin_amdgcn_readlane(at, first);
        if (left && key == lead) {
            place = at + int(__builtin_amdgcn_mbcnt_hi(uint32_t(same >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(same), 0u)));
            left = false;
        }
    }
    if (left) place = atomicAdd(&counter[key], 1);
    return place;
}

__global__ __launch_bounds__(kPlanThreads) void adapter_plan_kernel(AdArgs a) {
    __shared__ int s_count[kAdMaxSlots + 1], s_tile[kAdMaxSlots + 2], s_wave[kPlanThreads / 64];
    const int tid = threadIdx.x, keys = a.slots + 1, span = kTileHead + a.tile_rows;
    for (int i = tid; i < keys; i += kPlanThreads) s_count[i] = 0;
    __syncthreads();
    uint32_t flags = 0;
    int id[kPlanBatch], place[kPlanBatch];
    auto take = [&](int t0) {                          // ids of a batch of rows, loaded at once, and their places
#pragma unroll
        for (int j = 0; j < kPlanBatch; ++j) id[j] = a.ids[min(t0 + j * kPlanThreads + tid, a.M - 1)];
#pragma unroll
        for (int j = 0; j < kPlanBatch; ++j) {
            if (t0 + j * kPlanThreads >= a.M) break;
            flags |= id[j] >= a.slots ? kAdBadId : 0u;
            id[j] = t0 + j * kPlanThreads + tid < a.M ? ad_key(id[j], a.slots) : -1;
            place[j] = ad_take(s_count, id[j]);
        }
    };
    constexpr int kBatchRows = kPlanThreads * kPlanBatch;
    for (int t0 = 0; t0 < a.M; t0 += kBatchRows) take(t0);
    flag_or(a.flags, flags);
    __syncthreads();
    int tiles = 0;
    for (int i0 = 0; i0 < keys; i0 += kPlanThreads) {
        const int i = i0 + tid, n = i < keys ? s_count[i] : 0;
        const int nt = i == 0 && a.in_place ? 0 : (n + a.tile_rows - 1) / a.tile_rows;
        int all;
        const int first = tiles + block_prefix(nt, s_wave, all) - nt;
        if (i < keys) s_tile[i] = first;
        tiles += all;
    }
    __syncthreads();
    for (int j = tid; j < a.units; j += kPlanThreads) {
        int32_t* tile = a.tiles + size_t(j) * span;
        if (j >= tiles) {
            tile[0] = -2;
            continue;
        }
        int lo = 0, hi = keys;                         // the last slot that begins at or before tile j
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            (s_tile[mid] <= j ? lo : hi) = mid;
        }
        tile[0] = lo - 1;
        tile[1] = min(s_count[lo] - (j - s_tile[lo]) * a.tile_rows, a.tile_rows);
    }
    auto put = [&](int t0) {
#pragma unroll
        for (int j = 0; j < kPlanBatch; ++j) {
            if (t0 + j * kPlanThreads >= a.M) break;
            if (id[j] < 0 || (id[j] == 0 && a.in_place)) continue;
            const int tile = s_tile[id[j]] + place[j] / a.tile_rows;
            a.tiles[size_t(tile) * span + kTileHead + place[j] % a.tile_rows] = t0 + j * kPlanThreads + tid;
        }
    };
    if (a.M <= kBatchRows) {
        put(0);
        return;
    }
    __syncthreads();                                   // (more rows than a batch: places again)
    for (int i = tid; i < keys; i += kPlanThreads) s_count[i] = 0;
    __syncthreads();
    for (int t0 = 0; t0 < a.M; t0 += kBatchRows) {
        take(t0);
        put(t0);
    }
}

// ---- shrink ---------------------------------------------------------------------
// acc[m][r] += x A over k in [kbegin, kend), a wave's share of it: 64 k of every 64 W, D such pieces loaded
// before the first product.  The instruction wants neighbouring lanes in different rows, and such loads (64
// lines' halves at a time) were what few rows waited for: one block's 16 x 2048 of A added 2.4 us to the 3.3 of a
// call without it, against 0.9 with eight lanes on the 128 bytes of a row.  So those, and through LDS to the
// operands' order: piece c (16 bytes) of row r at 8 r + (c ^ r % 8), free of bank conflicts both ways; a wave's
// own LDS, which needs no barrier.
template <int TYPE, int MT, int RT, int W, int D>
__device__ __forceinline__ void ad_accumulate(const AdArgs& a, const int (&t)[MT], int rows, const uint16_t* w, int wrows,
                                              u32x4* stage, int kbegin, int kend, f32x4 (&acc)[MT][RT]) {
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), li = lane & 15, q = lane >> 4;
    const int lrow = lane >> 3, piece = lane & 7;
    const uint16_t* x[MT][2];
    uint32_t of[RT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
            x[m][h] = a.x + size_t(__builtin_amdgcn_ds_bpermute(4 * (8 * h + lrow), t[m])) * size_t(a.ldx);
#pragma unroll
        for (int r = 0; r < RT; ++r) of[r][h] = uint32_t(min(16 * r + 8 * h + lrow, wrows - 1)) * uint32_t(a.K);
    }
    u32x4* const put = stage + 8 * lrow + (piece ^ lrow);              // (row 8 h + lrow: 64 h further)
    const u32x4* const get[2] = {stage + 8 * li + (q ^ (li & 7)), stage + 8 * li + ((4 + q) ^ (li & 7))};
    for (int k0 = kbegin + 64 * wv; k0 < kend; k0 += 64 * W * D) {
        u32x4 xv[D][2][MT], wf[D][2][RT];
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (d && k0 + 64 * W * d >= kend) break;
            const int k = min(k0 + 64 * W * d + 8 * piece, a.K - 8);   // (past K: its last piece, cleared below)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int r = 0; r < RT; ++r) wf[d][h][r] = *reinterpret_cast<const u32x4*>(w + (of[r][h] + uint32_t(k)));
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    if (16 * m + 8 * h < rows) xv[d][h][m] = *reinterpret_cast<const u32x4*>(x[m][h] + k);
            }
        }
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int kd = k0 + 64 * W * d;
            if (d && kd >= kend) break;
            if (kd + 64 > a.K && kd + 8 * piece >= a.K) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int r = 0; r < RT; ++r) wf[d][h][r] = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int m = 0; m < MT; ++m) xv[d][h][m] = u32x4{0, 0, 0, 0};
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int r = 0; r < RT; ++r) put[128 * r + 64 * h] = wf[d][h][r];
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    if (16 * m + 8 * h < rows) put[128 * (RT + m) + 64 * h] = xv[d][h][m];
            }
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 av[MT], bv[RT];
#pragma unroll
                for (int m = 0; m < MT; ++m) av[m] = get[h][128 * (RT + m)];
#pragma unroll
                for (int r = 0; r < RT; ++r) bv[r] = get[h][128 * r];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int r = 0; r < RT; ++r) acc[m][r] = ad_mfma<TYPE>(av[m], bv[r], acc[m][r]);
            }
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
}

constexpr int kShrinkWaves = 8;

template <int TYPE, int RT, int D, int FEW>
__global__ __launch_bounds__(64 * kShrinkWaves) void adapter_shrink_kernel(AdArgs a) {
    constexpr int W = kShrinkWaves;
    __shared__ u32x4 s_stage[W][(1 + RT) * 128];       // (then the waves' sums)
    int slot, rows, t[1];
    if (!ad_tile<1, FEW>(a, blockIdx.x, blockIdx.x + blockIdx.y + blockIdx.z == 0, slot, rows, t) || slot < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, q = lane >> 4;
    const int part = ((a.K + 63) / 64 + a.splits - 1) / a.splits * 64, kbegin = int(blockIdx.z) * part, kend = min(kbegin + part, a.K);
    const int r0 = int(blockIdx.y) * 16 * RT;
    f32x4 acc[1][RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) acc[0][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    ad_accumulate<TYPE, 1, RT, W, D>(a, t, rows, a.a + size_t(slot) * size_t(a.a_slot) + size_t(r0) * size_t(a.K), a.SR - r0,
                                      s_stage[wv], kbegin, kend, acc);
    f32x4* mine = reinterpret_cast<f32x4*>(s_stage[wv]) + lane;
#pragma unroll
    for (int r = 0; r < RT; ++r) mine[64 * r] = acc[0][r];
    __syncthreads();
    for (int f = wv; f < RT; f += W) {
        f32x4 v = reinterpret_cast<const f32x4*>(s_stage[0])[64 * f + lane];
#pragma unroll
        for (int u = 1; u < W; ++u) {
            const f32x4 p = reinterpret_cast<const f32x4*>(s_stage[u])[64 * f + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += p[i];
        }
        const int r = r0 + 16 * f + li;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int of = __builtin_amdgcn_ds_bpermute(4 * (4 * q + i), t[0]);
            if (r < a.SR && 4 * q + i < rows) a.v[(size_t(blockIdx.z) * a.M + of) * a.SR + r] = v[i];
        }
    }
}

// ---- expand ---------------------------------------------------------------------
template <int OUT> __device__ __forceinline__ float ad_float(uint32_t bits) {
    if constexpr (OUT == ORNITH_ADAPTER_F32) return __uint_as_float(bits);
    else if constexpr (OUT == ORNITH_ADAPTER_BF16) return bf16_bits_to_f32(bits);
    else return f16_bits_to_f32(bits);
}
template <int OUT> __device__ __forceinline__ uint32_t ad_bits(float v) {
    if constexpr (OUT == ORNITH_ADAPTER_F32) return __float_as_uint(v);
    else if constexpr (OUT == ORNITH_ADAPTER_BF16) return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
    else return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}
// Two rounded values in a word.
template <int OUT> __device__ __forceinline__ uint32_t ad_pair(float a, float b) {
    typedef float pair __attribute__((ext_vector_type(2)));
    if constexpr (OUT == ORNITH_ADAPTER_BF16) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(pair{a, b}, bf16x2));
    } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(pair{a, b}, f16x2));
    }
}
// Power of two that brings a row's largest |v| to [2^14, 2^15) of fp16, as fp32 (1 for 0 and non-finite rows).
__device__ __forceinline__ float ad_scale16(uint32_t most) {
    const int e = int(most >> 23);
    if (e == 0 || e == 255) return 1.f;
    return __uint_as_float(uint32_t(min(max(127 + 127 + 14 - e, 1), 254)) << 23);
}
// 16-bit numbers whose sum v is: two (off by 2^-17 of v at most in bf16, 2^-23 in fp16), and three of bf16, which
// hold its 24 bits, for fp32 results.
template <int TYPE, int OUT> constexpr int kAdParts = TYPE == ORNITH_ADAPTER_BF16 && OUT == ORNITH_ADAPTER_F32 ? 3 : 2;
template <int TYPE, int PARTS> __device__ __forceinline__ void ad_split(float v, uint32_t (&bits)[PARTS]) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        bits[p] = ad_bits<TYPE>(v);
        const float part = ad_float<TYPE>(bits[p]);
        v = __builtin_isinf(part) ? 0.f : v - part;    // (inf: no NaN beside it)
    }
}
// 16 bytes on their values' grid: global accesses need no more, so rows of any stride move in these.
typedef u32x4 ad_piece2 __attribute__((aligned(2)));
typedef u32x4 ad_piece4 __attribute__((aligned(4)));
// A wave's 16 MT rows x 64 columns of base and out, as they move: eight lanes (fp32: 16) on a row's 16-byte
// pieces, H accesses for 16 rows.  (Neighbouring lanes in different rows, as the products leave them, halve
// the rate.)  ONCE: stores that leave the caches alone,
// of many rows on the 16-byte grid (us without / with: 8192 rows 69.3 / 66.5, 4096 rows 42.4 / 31.9, off it 79.4 / 96.6;
// in two launches, rank 128, 8192 rows 146.8 / 144.9, 1120 rows 31.3 / 29.8, off it 150.4 / 155.7 and 33.1 / 32.4).
template <int OUT, int MT, bool ONCE> struct AdCells {
    typedef std::conditional_t<OUT == ORNITH_ADAPTER_F32, uint32_t, uint16_t> word;
    typedef std::conditional_t<OUT == ORNITH_ADAPTER_F32, ad_piece4, ad_piece2> piece_t;
    static constexpr int size = sizeof(word), per = 16 / size, lanes = 64 / per, rows_at_once = 64 / lanes, H = 16 / rows_at_once;
    const word* base[MT][H];                           // of this wave's next columns
    word* out[MT][H];
    u32x4 have[MT][H];
    float most = 0.f, zero = 0.f;                      // largest magnitude; 0, NaN once a result was not finite
    uint32_t mine = 0;                                 // rows of the tile that this lane moves, a bit each

    // rows as lane li of each 16 holds them
    __device__ __forceinline__ AdCells(const AdArgs& a, const int (&t)[MT], int rows, int n0) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const size_t row = size_t(__builtin_amdgcn_ds_bpermute(4 * (rows_at_once * h + lane / lanes), t[m]));
                base[m][h] = static_cast<const word*>(a.base) + row * size_t(a.ldb) + n0 + per * (lane % lanes);
                out[m][h] = static_cast<word*>(a.out) + row * size_t(a.ldo) + n0 + per * (lane % lanes);
                mine |= 16 * m + rows_at_once * h + lane / lanes < rows ? 1u << (m * H + h) : 0u;
            }
    }
    __device__ __forceinline__ void step(int columns) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < H; ++h) {
                base[m][h] += columns;
                out[m][h] += columns;
            }
    }
    // base of the wave's 64 columns: whole pieces, or (left: of the 64, inside the slice) value by value, past
    // the end the last one
    __device__ __forceinline__ void load(bool whole, int left) {
        const int last = left - 1 - per * int((threadIdx.x & 63) % lanes);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (whole) have[m][h] = *reinterpret_cast<const piece_t*>(base[m][h]);
                else {
                    u32x4 v = {0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < per; ++i) v[i * size / 4] |= uint32_t(base[m][h][min(i, last)]) << (size == 4 ? 0 : 16 * (i & 1));
                    have[m][h] = v;
                }
            }
    }
    __device__ __forceinline__ bool has(int m, int h) const { return mine >> (m * H + h) & 1; }
    __device__ __forceinline__ void put(int m, int h, u32x4 r, bool whole, int left) {
        if (whole) {
            piece_t* const to = reinterpret_cast<piece_t*>(out[m][h]);
            if constexpr (ONCE) __builtin_nontemporal_store(r, to);
            else *to = r;
            return;
        }
        const int mine_left = left - per * int((threadIdx.x & 63) % lanes);
#pragma unroll
        for (int i = 0; i < per; ++i)
            if (i < mine_left) out[m][h][i] = word(r[i * size / 4] >> (size == 4 ? 0 : 16 * (i & 1)));
    }
    // base to out, as it is
    __device__ __forceinline__ void copy(bool whole, int left) {
        load(whole, left);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < H; ++h)
                if (has(m, h)) put(m, h, have[m][h], whole, left);
    }
    // base + by * acc, rounded; acc[m][j] of lane 16 q + li: row li's columns 16 j + 4 q .. + 3.  Through LDS to
    // the lanes that move them: 16 bytes c of row r at 16 r + (c ^ r), no bank conflicts; stage: the wave's own,
    // 256 pieces.  A piece with a result that is not finite stays unwritten, and then is base + sum(m, row, column)
    // (the parts of v make NaN of inf in B, where a part is 0 or of the other sign, and inf of a v above their
    // type's largest value).
    template <bool SCALED, class F> __device__ __forceinline__ void add(const f32x4 (&acc)[MT][4], const float (&by)[MT], f32x4* stage,
                                                                        bool whole, int left, F&& sum) {
        const int lane = threadIdx.x & 63, li = lane & 15, q = lane >> 4;
        uint32_t todo = 0;                             // such pieces, as in mine
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4 v = acc[m][j];
                if constexpr (SCALED) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] *= by[m];
                }
                stage[16 * li + ((4 * j + q) ^ li)] = v;
            }
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (!has(m, h)) continue;              // (such rows' sums are of anything)
                const int row = rows_at_once * h + lane / lanes;
                float r[per];
#pragma unroll
                for (int c = 0; c < per / 4; ++c) {
                    const f32x4 v = stage[16 * row + ((per / 4 * (lane % lanes) + c) ^ row)];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int e = 4 * c + i;
                        const uint32_t w = have[m][h][e * size / 4];
                        r[e] = v[i] + ad_float<OUT>(size == 4 ? w : e & 1 ? w >> 16 : w & 0xffffu);
                    }
                }
                u32x4 bits;
                float largest = most, none = 0.f;      // none: NaN beside a result that is not finite
#pragma unroll
                for (int e = 0; e < per; e += 2) {
                    if (whole) {
                        largest = fmaxf(fmaxf(largest, __builtin_fabsf(r[e])), __builtin_fabsf(r[e + 1]));
                        none = __builtin_fmaf(r[e], 0.f, none);
                        none = __builtin_fmaf(r[e + 1], 0.f, none);
                    } else {
#pragma unroll
                        for (int i = e; i < e + 2; ++i) {
                            const float in = per * (lane % lanes) + i < left ? r[i] : 0.f;
                            largest = fmaxf(largest, __builtin_fabsf(in));
                            none = __builtin_fmaf(in, 0.f, none);
                        }
                    }
                    if constexpr (size == 4) {
                        bits[e] = __float_as_uint(r[e]);
                        bits[e + 1] = __float_as_uint(r[e + 1]);
                    } else bits[e / 2] = ad_pair<OUT>(r[e], r[e + 1]);
                }
                if (none == none) {
                    most = largest;
                    put(m, h, bits, whole, left);
                } else todo |= 1u << (m * H + h);
            }
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        for (; __builtin_expect(todo != 0, 0); todo &= todo - 1) {
            const int at = __ffs(int(todo)) - 1;
            const word* from = base[0][0];
            word* to = out[0][0];
#pragma unroll
            for (int i = 1; i < MT * H; ++i) {
                from = at == i ? base[i / H][i % H] : from;
                to = at == i ? out[i / H][i % H] : to;
            }
#pragma unroll 1
            for (int e = 0; e < per; ++e) {
                const int column = per * (lane % lanes) + e;
                if (column >= left) break;
                const float r = sum(at / H, rows_at_once * (at % H) + lane / lanes, column) + ad_float<OUT>(from[e]);
                most = fmaxf(most, __builtin_fabsf(r));
                zero = __builtin_fmaf(r, 0.f, zero);
                to[e] = word(ad_bits<OUT>(r));
            }
        }
    }
    // 16-bit results round to infinity from half a step above the type's largest value
    __device__ __forceinline__ uint32_t flags() const {
        const bool bad = zero != zero;
        constexpr float limit = OUT == ORNITH_ADAPTER_BF16 ? 0x1.ffp127f : 65520.f;
        return (bad ? kAdNonfinite : 0u) | (OUT != ORNITH_ADAPTER_F32 && (bad || most >= limit) ? kAdNonfinite16 : 0u);
    }
};

// scale sum_r B[r] v(r) of one row and column, in fp64: for results that the parts of v may have driven out of range.
// A sum that is NaN stays one, so a row of NaN costs its batch little (8192 x 6144, rank 16 59 -> 68 us, 32 rows of rank 512
// 40 -> 54; to the end of every sum 144 and 2084).
template <int TYPE, class F> __device__ __forceinline__ float ad_sum(const uint16_t* b, int R, float scale, F&& v) {
    double sum = 0.0;
#pragma unroll 1
    for (int r = 0; r < R && sum == sum; ++r) sum += double(ad_float<TYPE>(b[r])) * double(v(r));
    return float(sum * double(scale));
}

constexpr int kExpandWaves = 4;                        // a block: 64 columns a wave

template <int TYPE, int OUT, int FEW>
__global__ __launch_bounds__(64 * kExpandWaves) void adapter_expand_kernel(AdArgs a) {
    extern __shared__ __attribute__((aligned(16))) u32x4 s_v[];        // [parts][steps][64]
    constexpr int PARTS = kAdParts<TYPE, OUT>;
    __shared__ uint32_t s_most[16];
    __shared__ int s_t[16];
    __shared__ u32x4 s_stage[kExpandWaves][512];       // a wave's B of 64 columns and 64 r, then its results
    int slot, rows, t[1];
    if (!ad_tile<1, FEW>(a, blockIdx.x, false, slot, rows, t) || (slot < 0 && a.in_place)) return;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, q = lane >> 4;
    int p = 0;
    while (int(blockIdx.y) >= a.blocks[p]) ++p;
    const int end = a.ends[p];
    const int n0 = (p ? a.ends[p - 1] : 0) + ((int(blockIdx.y) - (p ? a.blocks[p - 1] : 0)) * kExpandWaves + wv) * 64;
    typedef AdCells<OUT, 1, FEW == 0> Cells;
    const bool whole = n0 + 64 <= end;
    Cells cells(a, t, rows, n0);
    if (slot < 0) {
        if (n0 < end) cells.copy(whole, end - n0);
        return;
    }
    if (n0 < end) cells.load(whole, end - n0);
    const int chunks = a.R / 8, steps = (chunks + 3) / 4;
    {
        // scale v of the tile's rows and this slice in its parts, in pieces of 8 along r, as the instruction's operands
        if (tid < 16) s_t[tid] = t[0];
        if (TYPE == ORNITH_ADAPTER_F16 && tid < 16) s_most[tid] = 0;
        __syncthreads();
        struct Piece { f32x4 v[2]; };
        const float scale = a.scales[slot];
        auto piece_of = [&](int row, int c) {          // the parts of K in order
            const float* from = a.v + size_t(s_t[row]) * a.SR + p * a.R + 8 * c;
            Piece sum{{*reinterpret_cast<const f32x4*>(from), *reinterpret_cast<const f32x4*>(from + 4)}};
            for (int z = 1; z < a.splits; ++z) {
                from += size_t(a.M) * a.SR;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4 part = *reinterpret_cast<const f32x4*>(from + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum.v[h][e] += part[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum.v[e >> 2][e & 3] *= scale;
            return sum;
        };
        if constexpr (TYPE == ORNITH_ADAPTER_F16) {
            for (int i = tid; i < 16 * chunks; i += 64 * kExpandWaves) {
                const Piece v = piece_of(i / chunks, i % chunks);
                uint32_t most = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(v.v[e >> 2][e & 3]) & 0x7fffffffu);
                atomicMax(&s_most[i / chunks], most);
            }
            __syncthreads();
        }
        for (int i = tid; i < 16 * steps * 4; i += 64 * kExpandWaves) {
            const int row = i / (steps * 4), c = i % (steps * 4);
            u32x4 part[PARTS] = {};
            if (c < chunks) {
                const Piece v = piece_of(row, c);
                const float by = TYPE == ORNITH_ADAPTER_F16 ? ad_scale16(s_most[row]) : 1.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    uint32_t bits[PARTS];
                    ad_split<TYPE, PARTS>(v.v[e >> 2][e & 3] * by, bits);
#pragma unroll
                    for (int u = 0; u < PARTS; ++u) part[u][e >> 1] |= bits[u] << (16 * (e & 1));
                }
            }
#pragma unroll
            for (int u = 0; u < PARTS; ++u)
                s_v[(u * steps + (c >> 2)) * 64 + (c & 3) * 16 + row] = part[u];
        }
        __syncthreads();
    }
    if (n0 >= end) return;
    float by[1] = {1.f};
    if constexpr (TYPE == ORNITH_ADAPTER_F16) by[0] = 1.f / ad_scale16(s_most[li]);
    f32x4 acc[1][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // 64 r at a time: eight lanes on a column's 128 bytes, through LDS to the operands' order (piece c of column
    // n at 8 n + (c ^ n % 8)); the next ones on their way meanwhile
    const uint16_t* const bank = a.b + size_t(slot) * size_t(a.b_slot);
    uint32_t of[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) of[i] = uint32_t(min(n0 + 8 * i + (lane >> 3), end - 1)) * uint32_t(a.R);  // (past the slice: its last column)
    u32x4 bv[8];
    auto load_b = [&](int s) {
        const int c = min(4 * s + (lane & 7), chunks - 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) bv[i] = *reinterpret_cast<const u32x4*>(bank + (of[i] + uint32_t(8 * c)));
    };
    u32x4* const put = s_stage[wv] + 8 * (lane >> 3) + ((lane & 7) ^ (lane >> 3));
    load_b(0);
    for (int s = 0; s < steps; s += 2) {
        const bool none = 4 * s + (lane & 7) >= chunks;          // (no 0 times inf)
#pragma unroll
        for (int i = 0; i < 8; ++i) put[64 * i] = none ? u32x4{0, 0, 0, 0} : bv[i];
        if (s + 2 < steps) load_b(s + 2);
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (s + h >= steps) break;
            u32x4 bw[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) bw[j] = s_stage[wv][8 * (16 * j + li) + ((4 * h + q) ^ (li & 7))];
#pragma unroll
            for (int u = 0; u < PARTS; ++u) {
                const u32x4 vv = s_v[(u * steps + s + h) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[0][j] = ad_mfma<TYPE>(bw[j], vv, acc[0][j]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    auto form = [&](int, int row, int column) {
        const float* from = a.v + size_t(s_t[row]) * a.SR + p * a.R;
        return ad_sum<TYPE>(bank + size_t(n0 + column) * size_t(a.R), a.R, a.scales[slot], [&](int r) {
            float v = from[r];                         // (the parts of K in order)
            for (int z = 1; z < a.splits; ++z) v += from[size_t(z) * size_t(a.M) * a.SR + r];
            return v;
        });
    };
    cells.template add<TYPE == ORNITH_ADAPTER_F16>(acc, by, reinterpret_cast<f32x4*>(s_stage[wv]), whole, end - n0, form);
    flag_or(a.flags, cells.flags());
}

// ---- both in one ----------------------------------------------------------------
// A small rank: a block forms v of its tile for itself (its waves share k) and then its columns, 64 a wave at
// a time.  Every block of columns reads x and A again, from its XCD's L2, and spares the second launch (us, one / two,
// 2048 to 6144: rank 16, 1 row 5.5 / 7.6, 32 rows 7.1 / 8.7, 1120 rows 16.3 / 30.9; rank 32, 1 row 6.6 / 7.9, 32 rows
// 11.0 / 9.1, 1120 rows 20.7 / 32.2; rank 64, 8192 rows 90 / 142, 1120 rows 30.4 / 36.7, 1 row 9.0 / 8.0, 32 rows 15.5 /
// 11.1, of 2048 columns 9.3 / 8.0, 64 rows of two times 512 columns 9.9 / 10.7.  In a graph two are faster for up to 64
// rows of rank 33 and up, but for few columns; an eager call waits for the host, which a second launch costs 3).  Few rows wait
// for one chain: id, x and A, the waves' exchange, B, the store.  Many stream base and out: 8192 rows 57 us for 239
// MB, 4.2 TB/s of the 5.1 that a copy reaches; the rest goes into the exchange of results through LDS and the
// time before a block's first columns.
template <int TYPE, int OUT, int MT, int RT, int W, int FEW>
__global__ __launch_bounds__(64 * W) void adapter_both_kernel(AdArgs a) {
    constexpr int D = FEW > 0 && MT + RT <= 3 ? 4 : 2, PARTS = kAdParts<TYPE, OUT>, STEPS = (PARTS * RT + 1) / 2;
    typedef AdCells<OUT, MT, FEW == 0> Cells;
    static_assert((MT + RT) * 128 >= std::max(MT * RT * 64, std::max(256, 128 * RT)));
    __shared__ u32x4 s_stage[W][(MT + RT) * 128];      // (then the waves' sums, B, and results)
    __shared__ u32x4 s_v[MT][STEPS][64];
    __shared__ uint32_t s_most[16 * MT];
    __shared__ f32x4 s_sum[MT * RT][64];               // v: row 4 q + i of piece m RT + r / 16 in [16 q + r % 16][i]
    int slot, rows, t[MT];
    // blocks go to the 8 XCDs in turn: a row's column blocks on one of them, whose L2 keeps its A
    const int nblocks = a.blocks[a.S - 1], unit = int(blockIdx.x / 8) / nblocks * 8 + int(blockIdx.x % 8);
    const int cb = int(blockIdx.x / 8) % nblocks;
    if (unit >= a.units || !ad_tile<MT, FEW>(a, unit, blockIdx.x == 0, slot, rows, t) || (slot < 0 && a.in_place)) return;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, q = lane >> 4;
    int p = 0;
    while (cb >= a.blocks[p]) ++p;
    const int begin = (p ? a.ends[p - 1] : 0) + (cb - (p ? a.blocks[p - 1] : 0)) * (64 * W * a.groups);
    const int end = min(a.ends[p], begin + 64 * W * a.groups);
    const int whole_end = end - 63;                    // 64 columns from before it are inside
    int n0 = begin + 64 * wv;
    Cells cells(a, t, rows, n0);
    if (slot < 0) {
        for (; n0 < end; n0 += 64 * W) {
            cells.copy(n0 < whole_end, end - n0);
            cells.step(64 * W);
        }
        return;
    }
    slot = __builtin_amdgcn_readfirstlane(slot);
    const int chunks = a.R / 8;
    const float scale = a.scales[slot];
    {
        f32x4 acc[MT][RT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[m][r] = f32x4{0.f, 0.f, 0.f, 0.f};
        ad_accumulate<TYPE, MT, RT, W, D>(a, t, rows, a.a + size_t(slot) * size_t(a.a_slot) + size_t(p * a.R) * size_t(a.K), a.R,
                                          s_stage[wv], 0, a.K, acc);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < RT; ++r) reinterpret_cast<f32x4*>(s_stage[wv])[64 * (m * RT + r) + lane] = acc[m][r];
    }
    for (int f = wv; f < MT * STEPS; f += W) s_v[f / STEPS][f % STEPS][lane] = u32x4{0, 0, 0, 0};
    if (TYPE == ORNITH_ADAPTER_F16 && tid < 16 * MT) s_most[tid] = 0;
    // B of 64 columns: 128 R neighbouring bytes, loaded as they lie (the first on their way while the waves meet)
    // and through LDS to the operands' order: piece c of column n at chunks n + (c ^ swap(n)), few bank conflicts.
    const char* const bank = reinterpret_cast<const char*>(a.b + size_t(slot) * size_t(a.b_slot));
    const int swap_bits = chunks & (chunks - 1) ? 0 : chunks - 1, swap_shift = chunks == 2 ? 2 : chunks == 4 ? 1 : 0;
    u32x4 bv[2 * RT];
    int to_b[2 * RT], from_b[STEPS];                   // places in LDS: of the pieces loaded, of the steps' operands
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) {
        const int col = (64 * i + lane) / chunks, c = (64 * i + lane) % chunks;
        to_b[i] = chunks * col + (c ^ (col >> swap_shift & swap_bits));
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int c = (4 * s + q) % chunks;
        from_b[s] = chunks * li + (c ^ (li >> swap_shift & swap_bits));    // (column 16 j + li: 16 j chunks further)
    }
    auto load_b = [&](int last) {                      // (past the last piece: that one again)
        const char* const from = bank + uint32_t(n0) * uint32_t(2 * a.R);
#pragma unroll
        for (int i = 0; i < 2 * RT; ++i)
            if (i < chunks) bv[i] = *reinterpret_cast<const u32x4*>(from + 16u * uint32_t(min(64 * i + lane, last)));
    };
    const int all_b = 64 * chunks - 1;
    if (n0 < whole_end) {
        cells.load(true, 64);
        load_b(all_b);
    }
    __syncthreads();
    constexpr int F = (MT * RT + W - 1) / W;           // pieces of 16 rows and 16 of the rank, a wave
    f32x4 v[F];
#pragma unroll
    for (int i0 = 0; i0 < F; ++i0) {
        const int f = wv + W * i0;
        if (f >= MT * RT) break;
        v[i0] = reinterpret_cast<const f32x4*>(s_stage[0])[64 * f + lane];
#pragma unroll
        for (int u = 1; u < W; ++u) {
            const f32x4 part = reinterpret_cast<const f32x4*>(s_stage[u])[64 * f + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i0][i] += part[i];
        }
        s_sum[f][lane] = v[i0];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i0][i] *= scale;
        if (TYPE == ORNITH_ADAPTER_F16 && 16 * (f % RT) + li < a.R) {
#pragma unroll
            for (int i = 0; i < 4; ++i) atomicMax(&s_most[16 * (f / RT) + 4 * q + i], __float_as_uint(v[i0][i]) & 0x7fffffffu);
        }
    }
    if (TYPE == ORNITH_ADAPTER_F16) __syncthreads();
#pragma unroll
    for (int i0 = 0; i0 < F; ++i0) {
        const int f = wv + W * i0, m = f / RT, r = 16 * (f % RT) + li;
        if (f >= MT * RT || r >= a.R) break;
        uint16_t* s16 = reinterpret_cast<uint16_t*>(&s_v[m][0][0]);
        auto put = [&](int c, int row, uint32_t bits) { s16[((c >> 2) * 64 + (c & 3) * 16 + row) * 8 + (r & 7)] = uint16_t(bits); };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 4 * q + i;
            uint32_t bits[PARTS];
            ad_split<TYPE, PARTS>(v[i0][i] * (TYPE == ORNITH_ADAPTER_F16 ? ad_scale16(s_most[16 * m + row]) : 1.f), bits);
#pragma unroll
            for (int u = 0; u < PARTS; ++u) put((r >> 3) + u * chunks, row, bits[u]);
        }
    }
    __syncthreads();
    float by[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) by[m] = TYPE == ORNITH_ADAPTER_F16 ? 1.f / ad_scale16(s_most[16 * m + li]) : 1.f;
    f32x4 sum[MT][4];
    f32x4* const stage = reinterpret_cast<f32x4*>(s_stage[wv]);
    auto product = [&] {
        u32x4* const stage_b = s_stage[wv];
#pragma unroll
        for (int i = 0; i < 2 * RT; ++i)
            if (i < chunks) stage_b[to_b[i]] = bv[i];
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (4 * s >= PARTS * chunks) break;
            u32x4 step[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                step[j] = stage_b[from_b[s] + 16 * j * chunks];
                if (4 * s + 4 > PARTS * chunks && 4 * s + q >= PARTS * chunks) step[j] = u32x4{0, 0, 0, 0};      // (no 0 times inf)
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const u32x4 vv = s_v[m][s][lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[m][j] = ad_mfma<TYPE>(step[j], vv, sum[m][j]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    constexpr bool SCALED = TYPE == ORNITH_ADAPTER_F16;
    int at = n0;                                       // the columns of the present sums
    auto form = [&](int m, int row, int column) {
        return ad_sum<TYPE>(reinterpret_cast<const uint16_t*>(bank) + size_t(at + column) * size_t(a.R), a.R, a.scales[slot],
                            [&](int r) { return s_sum[m * RT + r / 16][16 * (row >> 2) + r % 16][row & 3]; });
    };
    while (n0 < whole_end) {
        product();
        at = n0;
        n0 += 64 * W;
        if (n0 < whole_end) load_b(all_b);
        cells.template add<SCALED>(sum, by, stage, true, 64, form);
        cells.step(64 * W);
        if (n0 < whole_end) cells.load(true, 64);
    }
    for (; n0 < end; n0 += 64 * W) {
        cells.load(false, end - n0);
        load_b(min(all_b, (end - n0) * chunks - 1));
        product();
        at = n0;
        cells.template add<SCALED>(sum, by, stage, false, end - n0, form);
        cells.step(64 * W);
    }
    flag_or(a.flags, cells.flags());
}

struct AdLayout { size_t v, tiles, bytes; };

// Parts of K that a shrink of M rows may have (each has a v of its own).
int ad_splits(int64_t M) { return M <= kFewRows ? 4 : 1; }

// Whether a call goes without a plan.  It then takes one launch less (3 us of the host's time too, which a call of 8.5
// waits for), but the tiles of a long run of one request lie 16 rows apart, on one XCD, and each 512 columns form v again.
// Up to 256 rows while full tiles and 512s of columns make up to 160 blocks, above rank 16 80; in two launches up to 64
// rows.  (us of eager calls, without / with a plan, rows of as many requests and of three, K = 2048, 16 slots: rank 16, 6144
// columns, 128 rows 8.6 / 11.6 and 12.1 / 11.4, 192 rows 10.3 / 11.6 and 16.1 / 11.4, 256 rows 13.5 / 12.1 and 21.4 / 11.5;
// 12288 columns, 128 rows 14.1 / 11.9 and 19.5 / 11.7; rank 32, 4096 columns, 160 rows 11.5 / 11.6 and 18.0 / 11.6, 6144
// columns, 128 rows 13.5 / 11.9 and 18.3 / 11.6; rank 64, 4096 columns, 160 rows 12.4 / 13.9 and 20.1 / 13.9, 6144 columns,
// 128 rows 18.1 / 14.3 and 24.7 / 13.8; rank 128, 1024 columns, 72 rows 16.2 / 15.1 and 15.8 / 14.5, 6144 columns, 128 rows
// 32.3 / 18.6 and 40.3 / 15.9.)
bool ad_few(int64_t M, int N, int R) {
    if (M <= kWaveRows) return true;
    return R <= kBothRank && M <= kFewRows && (M + 15) / 16 * ((N + 511) / 512) <= (R <= 16 ? 160 : 80);
}

// Rows of a planned tile, and tiles at most.
// (us: both products of one launch in tiles of 16 / 32 rows, 6144 columns of K = 2048: rank 16, 8192 rows 66.4 /
// 69.6; rank 32, 76.3 / 75.5, 1120 rows 18.0 / 18.2; rank 64, 8192 rows 119 / 93.6, 1120 rows of 2048 columns 18.8 / 21.4.
// In two launches 64 rows, which read B less often, took 10 to 80 % longer than 16 from 512 to 8192 rows, ranks 72 to 256, 1024
// to 12288 columns and 2 to 300 requests: 8192 x 6144 of rank 128 182 / 144, 1024 rows 43 / 27.)
int ad_tile_rows(int M, int R) { return R > 32 && R <= kBothRank && M >= 4096 ? 32 : 16; }
int ad_tiles(int M, int slots, int tile_rows) { return std::min(M, (M + tile_rows - 1) / tile_rows + slots + 1); }

bool ad_layout(int64_t M, int S, int R, AdLayout& l) {
    if (M < 0 || S < 1 || S > kAdMaxSlices || R < 8 || R > kAdMaxR || R % 8) return false;
    const size_t rows = size_t(std::min<int64_t>(M, kAdRows));
    l.v = 0;
    // (no less than fewer rows need, whose K may be in parts)
    l.tiles = align256(std::max(rows * size_t(ad_splits(M)), std::min(rows, size_t(kFewRows)) * size_t(ad_splits(kFewRows))) *
                       size_t(S) * size_t(R) * 4);
    size_t words = 0;                                  // of a plan's tiles, whichever rows and slots
    for (int tile_rows : {16, 32})
        words = std::max(words, size_t(ad_tiles(int(rows), kAdMaxSlots, tile_rows)) * size_t(kTileHead + tile_rows));
    l.bytes = l.tiles + align256((M <= kWaveRows ? 0 : words) * 4) + 256;
    return true;
}

// Blocks of columns, slice by slice.
int ad_blocks(AdArgs& a, int columns) {
    int blocks = 0;
    for (int p = 0; p < a.S; ++p) {
        blocks += (a.ends[p] - (p ? a.ends[p - 1] : 0) + columns - 1) / columns;
        a.blocks[p] = blocks;
    }
    return blocks;
}
// f with the output's type as a constant.
template <class F> void ad_by_type(int out_type, F&& f) {
    if (out_type == ORNITH_ADAPTER_F32) f(std::integral_constant<int, ORNITH_ADAPTER_F32>{});
    else if (out_type == ORNITH_ADAPTER_BF16) f(std::integral_constant<int, ORNITH_ADAPTER_BF16>{});
    else f(std::integral_constant<int, ORNITH_ADAPTER_F16>{});
}

// Columns of a block, in 64 a wave: all that a tile has in as many even parts as make about 1024 blocks of 16 rows
// (two rounds of the chip's CUs with two each) of many tiles, and three groups a block, or two, of fewer, since each
// block forms v again (us, 1 / 2 / 3 / 6 groups, rank 16: 8192 x 6144 101 / 77 / 68 / 66; 4096 x 6144 57 / 35 / 32 / 34;
// 512 x 6144 14.3 / 13.6 / 13.4 / 16.8; 1120 x 2048 13.9 / 13.5 / 14.9 / 14.6; 300 x 2048 10.5 / 11.6).
int ad_groups(const AdArgs& a, int FEW, int W) {
    if (FEW > 0) return 1;
    const int all = (a.N + 64 * W - 1) / (64 * W);
    const int64_t cells = int64_t(all) * ((a.M + 15) / 16);
    const int64_t groups = std::max<int64_t>((cells + 1023) / 1024, std::min<int64_t>(3, (cells + 159) / 160));
    const int parts = int((all + groups - 1) / groups);
    return (all + parts - 1) / parts;
}

template <int TYPE, int MT, int FEW> hipError_t ad_both(AdArgs& a, int out_type, hipStream_t s) {
    constexpr int W = 8;
    a.groups = ad_groups(a, FEW, W);
    const dim3 grid((a.units + 7) / 8 * 8 * ad_blocks(a, 64 * W * a.groups));
    auto go = [&](auto kernel) { timed_launch("adapter_both", kernel, grid, dim3(64 * W), 0, s, a); };
    ad_by_type(out_type, [&](auto out) {
        constexpr int OUT = decltype(out)::value;
        if constexpr (MT == 2) go(adapter_both_kernel<TYPE, OUT, 2, 4, W, FEW>);
        else if (a.R <= 16) go(adapter_both_kernel<TYPE, OUT, 1, 1, W, FEW>);
        else if (a.R <= 32) go(adapter_both_kernel<TYPE, OUT, 1, 2, W, FEW>);
        else go(adapter_both_kernel<TYPE, OUT, 1, 4, W, FEW>);
    });
    return hipGetLastError();
}

template <int TYPE, int FEW> hipError_t ad_two(AdArgs& a, int out_type, hipStream_t s) {
    const int rt = (a.SR + 15) / 16;
    a.splits = std::max(1, std::min(ad_splits(a.M), (a.K + 511) / 512));
    auto shrink = [&](auto kernel, int RT) {
        timed_launch("adapter_shrink", kernel, dim3(a.units, (rt + RT - 1) / RT, a.splits), dim3(64 * kShrinkWaves), 0, s, a);
    };
    // Rows of A a block: 64 reads x less often, 16 makes more blocks, for up to 160 rows of x times 16s of A (us, both
    // launches, 16 / 64, as many requests as rows, K = 2048, 6144 columns: rank 128, 16 rows 12.2 / 12.6, 32 rows 15.3 / 14.0;
    // rank 256, 8 rows 13.7 / 13.9, 16 rows 16.8 / 15.8; rank 512, 4 rows 17.4 / 17.6, 8 rows 19.4 / 18.6; one row 8.7 / 9.3).
    bool narrow = false;
    if constexpr (FEW > 0) {
        narrow = a.M * rt <= 160;
        if (narrow) shrink(adapter_shrink_kernel<TYPE, 1, 4, FEW>, 1);
    }
    if (!narrow) shrink(adapter_shrink_kernel<TYPE, 4, 2, std::max(FEW, 0)>, 4);
    const hipError_t st = hipGetLastError();
    if (st != hipSuccess) return st;
    const dim3 grid(a.units, ad_blocks(a, 64 * kExpandWaves));
    const int steps = (a.R / 8 + 3) / 4;
    ad_by_type(out_type, [&](auto out) {
        constexpr int OUT = decltype(out)::value;
        timed_launch("adapter_expand", adapter_expand_kernel<TYPE, OUT, FEW>, grid, dim3(64 * kExpandWaves),
                     uint32_t(steps * kAdParts<TYPE, OUT> * 1024), s, a);
    });
    return hipGetLastError();
}

template <int TYPE> hipError_t ad_rows(AdArgs& a, int out_type, hipStream_t s) {
    const bool both = a.R <= kBothRank;
    if (ad_few(a.M, a.N, a.R)) {
        a.units = a.M;
        if (!both) return ad_two<TYPE, 1>(a, out_type, s);
        return a.M <= kWaveRows ? ad_both<TYPE, 1, 1>(a, out_type, s) : ad_both<TYPE, 1, 4>(a, out_type, s);
    }
    a.tile_rows = ad_tile_rows(a.M, a.R);
    a.units = ad_tiles(a.M, a.slots, a.tile_rows);
    timed_launch("adapter_plan", adapter_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
    const hipError_t st = hipGetLastError();
    if (st != hipSuccess) return st;
    const bool grid = ((reinterpret_cast<uintptr_t>(a.out) | size_t(a.ldo) * (out_type == ORNITH_ADAPTER_F32 ? 4 : 2)) & 15) == 0;
    if (both) {
        if (a.tile_rows == 32) return grid ? ad_both<TYPE, 2, 0>(a, out_type, s) : ad_both<TYPE, 2, -1>(a, out_type, s);
        return grid ? ad_both<TYPE, 1, 0>(a, out_type, s) : ad_both<TYPE, 1, -1>(a, out_type, s);
    }
    return grid ? ad_two<TYPE, 0>(a, out_type, s) : ad_two<TYPE, -1>(a, out_type, s);
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
    args.tiles = at<int32_t>(workspace, l.tiles);
    args.N = N;
    args.K = K;
    args.R = R;
    args.SR = S * R;
    args.S = S;
    args.slots = slots;
    args.in_place = in_place;
    for (int p = 0; p < S; ++p) args.ends[p] = slice_ends[p];
    for (int64_t r = 0; r < M; r += kAdRows) {
        args.M = int(std::min<int64_t>(M - r, kAdRows));
        args.x = static_cast<const uint16_t*>(x) + size_t(r) * size_t(ldx);
        args.ids = static_cast<const int32_t*>(ids) + r;
        args.base = static_cast<const uint8_t*>(base) + size_t(r) * size_t(ldb) * size;
        args.out = static_cast<uint8_t*>(out) + size_t(r) * size_t(ldo) * size;
        const hipError_t st = x_type == ORNITH_ADAPTER_BF16 ? ad_rows<ORNITH_ADAPTER_BF16>(args, out_type, stream)
                                                            : ad_rows<ORNITH_ADAPTER_F16>(args, out_type, stream);
        if (st != hipSuccess) return st;
    }
    return hipSuccess;
}
