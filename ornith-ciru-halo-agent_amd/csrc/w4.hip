// Plain 4-bit linears (definition and bank layout: include/ornith_w4.h).
//
// On the matrix cores, with the codes as exact small floats: 16 + c has c in
// the top four mantissa bits of a bf16 or fp16 number of [16, 32), so two codes
// become a packed pair by a shift, a mask and an or.  Over one group
//   sum x (c - z) = sum x (16 + c) - (16 + z) sum x,
// both sums in fp32 on the matrix cores (sum x against a fragment of ones);
// each product is exact.  The roundings are those of sums of at most 31 |x| a
// term where 15 |x| are wanted, and absolute: where c == z throughout, s times
// what the two sums differ by stays (off by up to 0.48 of 2^-24 * 32 sum |s x| in
// random rows with and without a mean, K = 136 to 8192).  acc += s * (that), groups in ascending order within a wave,
// waves in ascending order.
//
// Bound by the codes' stream where it is long (151936 x 2048, 32 rows, fp32
// results: 41.7 us, 181 MB, 4.3 TB/s of the 5.3 that a large copy reaches; of
// the rest x to LDS takes 5 us, and the last wave's end), and by launch and the
// round trips of one wave where it is short (6144 x 2048, 1 row: 4.5 us against
// 1.2 at that rate).  Codes lie so that a lane's 16 bytes are its column's share of four
// matrix steps: 1 KB contiguous a wave and load.
#include <algorithm>
#include <type_traits>
#include "kernels.hpp"
#include "timing.hpp"
#include "validate.hpp"
#include "../../include/ornith_w4.h"

namespace ornith {
namespace {

constexpr int kW4MaxN = 1 << 20, kW4MaxK = 65536, kW4Block = 128;

typedef __bf16 w4_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 w4_f16x8 __attribute__((ext_vector_type(8)));

template <int TYPE> __device__ __forceinline__ f32x4 w4_mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (TYPE == ORNITH_W4_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(w4_bf16x8, a),
                                                       __builtin_bit_cast(w4_bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(w4_f16x8, a),
                                                      __builtin_bit_cast(w4_f16x8, b), c, 0, 0, 0);
}
// 16 + code, k ascending, of a packed word
template <int TYPE> __device__ __forceinline__ u32x4 w4_unpack(uint32_t w) {
    if constexpr (TYPE == ORNITH_W4_BF16) {
        constexpr uint32_t m = 0x00780078u, b = 0x41804180u;
        return u32x4{((w << 3) & m) | b, ((w >> 1) & m) | b, ((w >> 5) & m) | b, ((w >> 9) & m) | b};
    } else {
        constexpr uint32_t m = 0x03c003c0u, b = 0x4c004c00u;
        return u32x4{((w << 6) & m) | b, ((w << 2) & m) | b, ((w >> 2) & m) | b, ((w >> 6) & m) | b};
    }
}

// ---- packing --------------------------------------------------------------------
__global__ __launch_bounds__(256) void w4_pack_codes_kernel(const uint32_t* __restrict__ in, uint32_t* __restrict__ out,
                                                            int N, int K, size_t first, size_t words) {
    const size_t i = first + size_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= words) return;
    const int j = int(i & 3), lane = int(i >> 2) & 63, blocks = (K + kW4Block - 1) / kW4Block;
    const size_t tb = i >> 8;
    const int n = int(tb / size_t(blocks)) * 16 + (lane & 15);
    const int k = int(tb % size_t(blocks)) * kW4Block + 32 * j + 8 * (lane >> 4);
    uint32_t w = 0x88888888u;
    if (n < N && k < K) {
        const uint32_t v = in[size_t(n) * (K / 8) + k / 8];
        w = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= ((v >> (4 * e)) & 15u) << (4 * (e >> 1) + 16 * (e & 1));
    }
    out[i] = w;
}

__global__ __launch_bounds__(256) void w4_pack_meta_kernel(const uint16_t* __restrict__ scales, int scale_type,
                                                           const uint8_t* __restrict__ zeros, uint32_t* __restrict__ out,
                                                           int N, int groups, int chunks, int per, size_t words,
                                                           uint32_t* flags) {
    const size_t i = size_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= words) return;
    const size_t tc = i / size_t(16 * per);
    const int in = int(i % size_t(16 * per)), n = int(tc / size_t(chunks)) * 16 + in / per;
    const int g = int(tc % size_t(chunks)) * per + in % per;
    uint32_t w = 8;
    if (n < N && g < groups) {
        const size_t at = size_t(n) * groups + g;
        const float s = scale_type == ORNITH_W4_BF16 ? bf16_bits_to_f32(scales[at]) : f16_bits_to_f32(scales[at]);
        const uint32_t z = zeros ? zeros[at] : 8u;
        flag_or(flags, (isfinite(s) ? 0u : 1u) | (z > 15u ? 2u : 0u));
        w = (__float_as_uint(s) & ~15u) | (z & 15u);
    }
    out[i] = w;
}

// ---- product --------------------------------------------------------------------
struct W4Args {
    const uint16_t* x; int64_t ldx;
    const uint32_t *codes, *meta;
    void* out; int out_type; int64_t ldo;
    uint32_t* flags;
    int M, N, K, log2g;
};
// Results in the output's type, and what they raise: a lane keeps the largest magnitude it stored and
// a sum of zero times each (NaN once one was not finite).
template <int OUT> __device__ __forceinline__ void w4_put(void* out, size_t at, float v) {
    if constexpr (OUT == ORNITH_W4_F32) static_cast<float*>(out)[at] = v;
    else if constexpr (OUT == ORNITH_W4_BF16) static_cast<__bf16*>(out)[at] = static_cast<__bf16>(v);
    else static_cast<_Float16*>(out)[at] = static_cast<_Float16>(v);
}
struct W4Seen {
    float most = 0.f, zero = 0.f;
    __device__ __forceinline__ void see(float v) {
        most = fmaxf(most, __builtin_fabsf(v));
        zero = __builtin_fmaf(v, 0.f, zero);
    }
    // 16-bit results round to infinity from half a step above the type's largest value
    __device__ __forceinline__ uint32_t flags(int out_type) const {
        const bool bad = zero != zero;
        const float end = out_type == ORNITH_W4_BF16 ? 0x1.ffp127f : 65520.f;
        return (bad ? kDenseNonfiniteProjection : 0u) |
               (out_type != ORNITH_W4_F32 && (bad || most >= end) ? kDenseNonfiniteBf16 : 0u);
    }
};
// f with the output's type as a constant.
template <class F> __device__ __forceinline__ void w4_by_type(int out_type, F&& f) {
    if (out_type == ORNITH_W4_F32) f(std::integral_constant<int, ORNITH_W4_F32>{});
    else if (out_type == ORNITH_W4_BF16) f(std::integral_constant<int, ORNITH_W4_BF16>{});
    else f(std::integral_constant<int, ORNITH_W4_F16>{});
}
__host__ __device__ inline int w4_blocks(int K) { return (K + kW4Block - 1) / kW4Block; }

// More than 16 rows of many tiles.  A block takes a run of pairs of 16-column tiles and all its rows' x
// (16 MT of them) into LDS once.  Its waves share the run's units (pair, 128 k) evenly, in order: a wave
// ends the pair that an earlier one began, takes whole pairs, and begins one that later waves end; the
// parts of a pair meet in LDS, in wave order.  PER: groups in 128 k (1 for groups of 128 and 256).
// x lies in pieces of 8 k: piece (k / 8) * 16 MT + row; behind it its sums over groups (of 256: over their
// halves, as the products are added per 128 k), [group, 16 MT].
// W waves of a block, D units' codes of a wave in flight: 12 and 3 for two tiles of rows (151936 x 2048, 32
// rows, fp32 results, us: 43.2; 16 waves and 2 units 45.1, 8 and 3 44.3, 8 and 4 45.3, 8 and 6 45.1); 8
// and 4 for more, whose sums and parked parts take 64 registers a tile pair.  One unit less for groups of 32,
// whose scales take four times the registers (32 rows: 151936 x 2048 51.6, spilling 4 registers with 3 units
// 53.1; 24576 x 2048 16.4 / 18.0; 64 rows of 32768 x 1024 18.3 / 19.5).
constexpr size_t kW4XBytes = 128 * 1024;               // x of a block, at most
constexpr size_t w4_x_bytes(int MT, int K) { return size_t(16 * MT) * ((K + kW4Block - 1) / kW4Block) * (2 * kW4Block); }

template <int TYPE, int MT, int PER, int W, int D>
__global__ __launch_bounds__(64 * W) void w4_run_kernel(W4Args a) {
    extern __shared__ __attribute__((aligned(16))) u32x4 s_x[];
    __shared__ int s_pair[W];                   // the pair whose end or middle a wave holds
    typedef uint32_t meta_t __attribute__((ext_vector_type(PER)));
    constexpr int RP = 16 * MT;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, q = lane >> 4;
    const int row0 = int(blockIdx.y) * RP, R = min(a.M - row0, RP);
    const int blocks = w4_blocks(a.K), last_tile = (a.N - 1) >> 4, pairs = (last_tile >> 1) + 1;
    const int half = a.log2g == 8, chunks = half ? (blocks + 1) >> 1 : blocks;
    // this block's pairs, this wave's units
    const int base = pairs / int(gridDim.x), extra = pairs % int(gridDim.x), bx = blockIdx.x;
    const int p0 = bx * base + min(bx, extra), np = base + (bx < extra);
    const int units = np * blocks, ubase = units / W, uextra = units % W;
    const int u0 = wv * ubase + min(wv, uextra), u1 = u0 + ubase + (wv < uextra);

    u32x4 cw[D][2];
    meta_t mw[D][2];
    int np_ = u0 / blocks, nk = u0 % blocks;           // pair and block to load next
    auto load = [&](int slot) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {                  // (past the last tile: that one again)
            const size_t tile = size_t(min(2 * (p0 + np_) + t, last_tile));
            cw[slot][t] = __builtin_nontemporal_load(
                reinterpret_cast<const u32x4*>(a.codes + (tile * blocks + nk) * 256 + 4 * lane));
            mw[slot][t] = *reinterpret_cast<const meta_t*>(a.meta + (tile * chunks + (nk >> half)) * (16 * PER) + PER * li);
        }
        if (++nk == blocks) {
            nk = 0;
            ++np_;
        }
    };
    float* s_sum = reinterpret_cast<float*>(s_x + size_t(RP) * blocks * 16);
    {
        // all of a thread's pieces of x, then its first codes, in flight at once; four lanes read 64 bytes
        // of a row (rows past R: the last again)
        const uint16_t* x = a.x + size_t(row0) * size_t(a.ldx);
        constexpr int kBatch = (int(kW4XBytes / 16) + 64 * W - 1) / (64 * W);
        u32x4 v[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int i = tid + 64 * W * b, r = min((i >> 2) % RP, R - 1), piece = ((i >> 2) / RP) * 4 + (i & 3);
            v[b] = u32x4{0, 0, 0, 0};
            if (8 * piece < a.K) v[b] = *reinterpret_cast<const u32x4*>(x + size_t(r) * size_t(a.ldx) + 8 * piece);
        }
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (u0 + d < u1) load(d);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int i = tid + 64 * W * b;
            if (i < RP * blocks * 16) s_x[(((i >> 2) / RP) * 4 + (i & 3)) * RP + (i >> 2) % RP] = v[b];
        }
    }
    __syncthreads();
    const u32x4* mine = s_x + q * RP + li;             // this lane's pieces: step * 4 RP + 16 mt
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    {
        const uint32_t one = TYPE == ORNITH_W4_BF16 ? 0x3f803f80u : 0x3c003c00u;
        const u32x4 ones = {one, one, one, one};
        constexpr int steps = 4 / PER;
        for (int g = wv; g < blocks * PER; g += W) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                f32x4 sum = zero;
#pragma unroll
                for (int j = 0; j < steps; ++j) sum = w4_mfma<TYPE>(mine[(g * steps + j) * (4 * RP) + 16 * mt], ones, sum);
                if (li == 0) *reinterpret_cast<f32x4*>(&s_sum[g * RP + 16 * mt + 4 * q]) = sum;
            }
        }
    }
    __syncthreads();

    f32x4 acc[2][MT], head[2][MT];                     // head: the end of a pair that an earlier wave began
    auto clear = [&] {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[t][mt] = zero;
    };
    clear();
    W4Seen seen;
    auto store = [&](int pair) {
        w4_by_type(a.out_type, [&](auto out) {
            constexpr int OUT = decltype(out)::value;
            const int n0 = (p0 + pair) * 32;
            const size_t at = size_t(row0 + 4 * q) * size_t(a.ldo) + size_t(n0 + li);
            const bool whole = R == RP && n0 + 32 <= a.N;       // (wave-uniform)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (!whole && (16 * mt + 4 * q + i >= R || n0 + 16 * t + li >= a.N)) continue;
                        seen.see(acc[t][mt][i]);
                        w4_put<OUT>(a.out, at + size_t(16 * mt + i) * size_t(a.ldo) + 16 * t, acc[t][mt][i]);
                    }
        });
    };
    int head_pair = -1, pair = u0 / blocks, kb = u0 % blocks;
    bool began = kb == 0;
    for (int u = u0; u < u1; u += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (u + d >= u1) break;
            u32x4 w4[2];
            meta_t mm[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                w4[t] = cw[d][t];
                mm[t] = mw[d][t];
            }
            if (u + d + D < u1) load(d);
            const u32x4* xk = mine + kb * (16 * RP);
            const float* sk = s_sum + kb * (PER * RP) + 4 * q;
            f32x4 c[2][MT];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool first = j % (4 / PER) == 0, last = j % (4 / PER) == 4 / PER - 1;
                u32x4 av[MT];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) av[mt] = xk[j * (4 * RP) + 16 * mt];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const u32x4 b = w4_unpack<TYPE>(w4[t][j]);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) c[t][mt] = w4_mfma<TYPE>(av[mt], b, first ? zero : c[t][mt]);
                }
                if (!last) continue;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const f32x4 sx = *reinterpret_cast<const f32x4*>(sk + (j / (4 / PER)) * RP + 16 * mt);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const uint32_t m = mm[t][j / (4 / PER)];
                        const float sc = __uint_as_float(m & ~15u), z = -16.f - float(m & 15u);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[t][mt][i] = __builtin_fmaf(sc, __builtin_fmaf(z, sx[i], c[t][mt][i]), acc[t][mt][i]);
                    }
                }
            }
            if (++kb == blocks) {
                if (began) store(pair);
                else {
                    head_pair = pair;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) head[t][mt] = acc[t][mt];
                }
                clear();
                kb = 0;
                ++pair;
                began = true;
            }
        }
    }
    // pairs that several waves share
    __syncthreads();
    float* s_part = reinterpret_cast<float*>(s_x);
    const bool middle = kb != 0 && !began;             // began by an earlier wave, ended by a later one
    if (middle) head_pair = pair;
    if (lane == 0) s_pair[wv] = head_pair;
    if (head_pair >= 0) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s_part[((wv * 2 + t) * MT * 4 + 4 * mt + i) * 64 + lane] = middle ? acc[t][mt][i] : head[t][mt][i];
    }
    __syncthreads();
    if (began && kb != 0) {
        for (int w = wv + 1; w < W && s_pair[w] == pair; ++w)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[t][mt][i] += s_part[((w * 2 + t) * MT * 4 + 4 * mt + i) * 64 + lane];
        store(pair);
    }
    flag_or(a.flags, seen.flags(a.out_type));
}

// A block per NT tiles and 16 rows, whose waves take 128-k blocks in turn, x straight from memory, and
// meet in LDS in wave order.  The waves split K because few columns leave few blocks: at 6144 x 2048 a
// wave's whole work is two 128-k blocks, and a call (4.5 us, 6.7 MB) is the launch, one round trip for
// codes and x, eight matrix steps and one exchange.
template <int TYPE, int PER, int NT, int W>
__global__ __launch_bounds__(64 * W) void w4_tile_kernel(W4Args a) {
    typedef uint32_t meta_t __attribute__((ext_vector_type(PER)));
    __shared__ float s_acc[W][NT * 4][64];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, q = lane >> 4;
    const int tile0 = int(blockIdx.x) * NT, last_tile = (a.N - 1) >> 4, row0 = int(blockIdx.y) * 16, R = min(a.M - row0, 16);
    const int blocks = w4_blocks(a.K), half = a.log2g == 8, chunks = half ? (blocks + 1) >> 1 : blocks;
    const uint16_t* x = a.x + size_t(row0 + min(li, R - 1)) * size_t(a.ldx) + 8 * q;
    const uint32_t one = TYPE == ORNITH_W4_BF16 ? 0x3f803f80u : 0x3c003c00u;
    const u32x4 ones = {one, one, one, one};
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = zero;
    u32x4 next_cw[NT], next_xa[4];
    meta_t next_mw[NT];
    auto load = [&](int kb) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {                 // (past the last tile: that one again)
            const size_t tile = size_t(min(tile0 + t, last_tile));
            next_cw[t] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.codes + (tile * blocks + kb) * 256 + 4 * lane));
            next_mw[t] = *reinterpret_cast<const meta_t*>(a.meta + (tile * chunks + (kb >> half)) * (16 * PER) + PER * li);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = kb * kW4Block + 32 * j;
            next_xa[j] = u32x4{0, 0, 0, 0};
            if (k + 8 * q < a.K) next_xa[j] = *reinterpret_cast<const u32x4*>(x + k);
        }
    };
    // one block ahead (151936 x 2048, 1 row: 2.4 us less; short ones as before; 2 to 4 ahead 16 more)
    if (wv < blocks) load(wv);
    for (int kb = wv; kb < blocks; kb += W) {
        u32x4 cw[NT], xa[4];
        meta_t mw[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            cw[t] = next_cw[t];
            mw[t] = next_mw[t];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) xa[j] = next_xa[j];
        if (kb + W < blocks) load(kb + W);
        f32x4 c[NT], sx;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool first = j % (4 / PER) == 0, last = j % (4 / PER) == 4 / PER - 1;
            sx = w4_mfma<TYPE>(xa[j], ones, first ? zero : sx);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                c[t] = w4_mfma<TYPE>(xa[j], w4_unpack<TYPE>(cw[t][j]), first ? zero : c[t]);
                if (!last) continue;
                const uint32_t m = mw[t][j / (4 / PER)];
                const float sc = __uint_as_float(m & ~15u), z = -16.f - float(m & 15u);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] = __builtin_fmaf(sc, __builtin_fmaf(z, sx[i], c[t][i]), acc[t][i]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_acc[wv][4 * t + i][lane] = acc[t][i];
    __syncthreads();
    W4Seen seen;
    for (int e = wv; e < NT * 4; e += W) {             // a wave per register of a fragment
        const int row = 4 * q + (e & 3), n = (tile0 + (e >> 2)) * 16 + li;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += s_acc[w][e][lane];
        if (row >= R || n >= a.N) continue;
        seen.see(v);
        const size_t at = size_t(row0 + row) * size_t(a.ldo) + n;
        w4_by_type(a.out_type, [&](auto out) { w4_put<decltype(out)::value>(a.out, at, v); });
    }
    flag_or(a.flags, seen.flags(a.out_type));
}

// K == 0: zeros
__global__ __launch_bounds__(256) void w4_zero_kernel(W4Args a) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= a.N) return;
    for (int row = blockIdx.y; row < a.M; row += gridDim.y) {
        const size_t at = size_t(row) * size_t(a.ldo) + n;
        if (a.out_type == ORNITH_W4_F32) static_cast<float*>(a.out)[at] = 0.f;
        else static_cast<uint16_t*>(a.out)[at] = 0;
    }
}

int w4_log2g(int G) { return G == 32 ? 5 : G == 64 ? 6 : G == 128 ? 7 : G == 256 ? 8 : -1; }

bool w4_words(int N, int K, int G, size_t& codes, size_t& meta) {
    if (N < 0 || N > kW4MaxN || K < 0 || K > kW4MaxK || K % 8 || w4_log2g(G) < 0) return false;
    const size_t tiles = (size_t(N) + 15) / 16;
    codes = tiles * ((size_t(K) + kW4Block - 1) / kW4Block) * 256;
    const size_t blocks = (size_t(K) + kW4Block - 1) / kW4Block;
    meta = tiles * (G == 256 ? (blocks + 1) / 2 : blocks * (kW4Block / G)) * 16;
    return true;
}

template <int TYPE, int MT, int W, int D> hipError_t w4_run(const W4Args& a, hipStream_t s) {
    constexpr size_t part = size_t(W) * 2 * MT * 1024;
    const int groups = a.log2g < 7 ? w4_blocks(a.K) * (kW4Block >> a.log2g) : w4_blocks(a.K);
    const size_t lds = std::max(w4_x_bytes(MT, a.K), part) + size_t(groups) * 16 * MT * 4;
    const int pairs = (a.N + 31) / 32, rows = (a.M + 16 * MT - 1) / (16 * MT);
    const dim3 grid(std::min(pairs, std::max(device_cu_count() / rows, 1)), rows);
    auto go = [&](auto kernel) { timed_launch("w4_run", kernel, grid, dim3(64 * W), uint32_t(lds), s, a); };
    if (a.log2g == 5) go(w4_run_kernel<TYPE, MT, 4, W, D - 1>);
    else if (a.log2g == 6) go(w4_run_kernel<TYPE, MT, 2, W, D>);
    else go(w4_run_kernel<TYPE, MT, 1, W, D>);
    return hipGetLastError();
}
template <int TYPE, int NT, int W> hipError_t w4_tiles(const W4Args& a, hipStream_t s) {
    const dim3 grid(((a.N + 15) / 16 + NT - 1) / NT, (a.M + 15) / 16);
    auto go = [&](auto kernel) { timed_launch("w4_tile", kernel, grid, dim3(64 * W), 0, s, a); };
    if (a.log2g == 5) go(w4_tile_kernel<TYPE, 4, NT, W>);
    else if (a.log2g == 6) go(w4_tile_kernel<TYPE, 2, NT, W>);
    else go(w4_tile_kernel<TYPE, 1, NT, W>);
    return hipGetLastError();
}
// Which kernel, by the tiles of 16 x 16 results (us a call, bf16 results, calls in a graph over banks of
// 600 MB in turn or 24; K = 2048 and groups of 128 where nothing else is said):
//  - Tiles of a block.  One keeps more blocks than CUs where tiles are few; more read x, which comes from
//    L2 for every block, less often.  1 / 2 / 4 tiles: 6144 columns, 1 row 4.6 / 4.6 / 5.9, 8 rows 5.4 / 4.9 /
//    6.2, 16 rows 7.1 / 5.3 / 6.4, 64 rows 14.9 / 10.3 / 9.6; 12288 columns, 16 rows 8.8 / 7.8 / 6.7; 24576
//    columns, 1 row 10.1 / 8.6 / 9.6, 8 rows 11.2 / 9.3 / 9.9; 151936 columns, 1 row 48.2 / 40.0 / 33.4, 8 rows
//    59.2 / 43.5 / 35.8.  Two from 384 on where a wave's blocks are many, for few rows too: 6144 columns, 1 row,
//    K = 2944 5.8 / 5.6 / -, K = 4096 7.0 / 6.4 / 8.7, K = 8192 11.2 / 10.0 / -.
//  - Four tiles of groups of 32 and 64 (with their scales 134 to 138 registers: one block a CU) only while each
//    block has a CU: 2 / 4 tiles, groups of 32, 16 rows of 16384 columns 8.7 / 8.5, 18432 10.9 / 13.8, 32 rows of 8192
//    8.5 / 7.8, 12288 11.3 / 13.6; 151936 columns, 1 row 44.2 / 58.7; of 64 41.8 / 51.9.
//  - 16 waves where a wave of 8 would take two 128-k blocks or more in turn and each block has a CU: 8 / 16
//    waves, 1 row, 1024 columns 3.5 / 3.2, 4096 3.9 / 3.7, K = 4096 5.6 / 4.7, 4608 of K = 4096 6.6 / 7.4; 2048
//    columns of K = 8192 8.5 / 6.6, 8 rows 8.9 / 7.8, 16 rows 10.5 / 10.9; K = 512 2.6 / 2.7.
//  - x in LDS, which holds that of 32 rows up to K = 2048 (beyond, the tiles read all codes once per 16 rows:
//    24576 columns of K = 4096, 32 rows 24.6, 64 rows 46.8), for more than 16 rows of many columns.  4 tiles / in LDS: 32 rows, 22528 columns 14.2 / 14.4, 24000
//    14.8 / 14.6, 24576 14.8 / 14.8, 28672 17.6 / 15.8, of groups of 32 27.0 / 18.3, 24576 of K = 1024 9.9 / 10.0;
//    151936 73.5 / 42.2, 64 rows 144 / 73.5 (two passes over the weights: 32 rows are what LDS holds).  With three
//    or four tiles of rows (K up to 1280 and 1024) later: K = 1024, 64 rows, 12288 columns 9.2 / 12.1, 16384 11.8 /
//    12.5, 18432 13.7 / 13.6, 32768 20.7 / 15.6; 48 rows of 16384 9.5 / 10.7, 24576 14.1 / 12.2; but not of groups
//    of 32 and 64 (2 tiles / in LDS: groups of 32, 64 rows, 12288 columns 13.9 / 14.2, 16384 17.2 / 14.5, 48 rows
//    of 16384 13.8 / 12.1).
template <int TYPE> hipError_t w4_rows(const W4Args& a, hipStream_t s) {
    const int64_t cells = int64_t((a.N + 15) / 16) * ((a.M + 15) / 16);      // tiles of 16 x 16 results
    const int blocks = w4_blocks(a.K);
    const bool small_groups = a.log2g < 7;
    auto fits = [&](int MT) { return a.M > 16 * (MT - 1) && w4_x_bytes(MT, a.K) <= kW4XBytes; };
    const int MT = fits(4) ? 4 : fits(3) ? 3 : fits(2) ? 2 : 0;
    if (MT && cells > (MT == 2 || small_groups ? 3000 : 4096)) {
        if (MT == 4) return w4_run<TYPE, 4, 8, 4>(a, s);
        if (MT == 3) return w4_run<TYPE, 3, 8, 4>(a, s);
        return w4_run<TYPE, 2, 12, 3>(a, s);
    }
    if (cells >= (a.M <= 8 ? 4096 : 768) && (!small_groups || cells <= 1024)) return w4_tiles<TYPE, 4, 8>(a, s);
    if (cells >= (a.M <= 4 && blocks <= 16 ? 1536 : 384)) return w4_tiles<TYPE, 2, 8>(a, s);
    if (a.M <= 8 && blocks > 8 && cells <= 256) return w4_tiles<TYPE, 1, 16>(a, s);
    return w4_tiles<TYPE, 1, 8>(a, s);
}

}  // namespace
}  // namespace ornith

using namespace ornith;

extern "C" hipError_t ornith_w4_get_layout(int N, int K, int G, size_t* code_words, size_t* meta_words) {
    size_t c = 0, m = 0;
    if (!code_words || !meta_words || !w4_words(N, K, G, c, m)) return hipErrorInvalidValue;
    *code_words = c;
    *meta_words = m;
    return hipSuccess;
}

extern "C" hipError_t ornith_w4_pack(const void* codes, const void* scales, int scale_type, const void* zeros,
                                     void* packed_codes, void* packed_meta, void* flags, int N, int K, int G,
                                     hipStream_t stream) {
    size_t c = 0, m = 0;
    if (!w4_words(N, K, G, c, m) || (scale_type != ORNITH_W4_BF16 && scale_type != ORNITH_W4_F16))
        return hipErrorInvalidValue;
    if (!N || !K) return hipSuccess;
    const int groups = (K + G - 1) / G;
    const size_t pairs = size_t(N) * groups;
    const Buffer buffers[] = {{codes, size_t(N) * (K / 2), 4, false, false},
                              {scales, pairs * 2, 2, false, false},
                              {zeros, pairs, 1, false, true},
                              {packed_codes, c * 4, 16, true, false},
                              {packed_meta, m * 4, 4, true, false},
                              {flags, 4, 4, true, false}};
    if (!check_buffers(buffers)) return hipErrorInvalidValue;
    constexpr size_t kAtOnce = size_t(1) << 31;        // (a grid has less than 2^32 threads)
    for (size_t first = 0; first < c; first += kAtOnce) {
        timed_launch("w4_pack_codes", w4_pack_codes_kernel, dim3(unsigned((std::min(c - first, kAtOnce) + 255) / 256)), dim3(256),
                     0, stream, static_cast<const uint32_t*>(codes), static_cast<uint32_t*>(packed_codes), N, K, first, c);
        const hipError_t st = hipGetLastError();
        if (st != hipSuccess) return st;
    }
    timed_launch("w4_pack_meta", w4_pack_meta_kernel, dim3(unsigned((m + 255) / 256)), dim3(256), 0, stream,
                 static_cast<const uint16_t*>(scales), scale_type, static_cast<const uint8_t*>(zeros),
                 static_cast<uint32_t*>(packed_meta), N, groups,
                 G == 256 ? (w4_blocks(K) + 1) / 2 : w4_blocks(K), G == 256 ? 1 : kW4Block / G, m, static_cast<uint32_t*>(flags));
    return hipGetLastError();
}

extern "C" hipError_t ornith_w4_launch(const void* x, int x_type, int64_t ldx, const void* codes, const void* meta,
                                       void* out, int out_type, int64_t ldo, void* flags, int M, int N, int K, int G,
                                       hipStream_t stream) {
    size_t c = 0, m = 0;
    if (!w4_words(N, K, G, c, m) || M < 0 || ldx < K || ldo < N || ldx % 8 ||
        (x_type != ORNITH_W4_BF16 && x_type != ORNITH_W4_F16) || out_type < ORNITH_W4_BF16 || out_type > ORNITH_W4_F32)
        return hipErrorInvalidValue;
    if (!M || !N) return hipSuccess;
    const size_t size = out_type == ORNITH_W4_F32 ? 4 : 2;
    const Buffer buffers[] = {{x, K ? (size_t(M - 1) * size_t(ldx) + size_t(K)) * 2 : 0, 16, false, K == 0},
                              {codes, c * 4, 16, false, K == 0},
                              {meta, m * 4, 4, false, K == 0},
                              {out, (size_t(M - 1) * size_t(ldo) + size_t(N)) * size, size, true, false},
                              {flags, 4, 4, true, false}};
    if (!check_buffers(buffers)) return hipErrorInvalidValue;
    // rows ride on the grid's y axis (65535 blocks of 16 rows at least)
    constexpr int kMost = 65535 * 16;
    for (int64_t r = 0; r < M; r += kMost) {
        const W4Args a{static_cast<const uint16_t*>(x) + size_t(r) * size_t(ldx), ldx,
                       static_cast<const uint32_t*>(codes), static_cast<const uint32_t*>(meta),
                       static_cast<uint8_t*>(out) + size_t(r) * size_t(ldo) * size, out_type, ldo,
                       static_cast<uint32_t*>(flags), int(std::min<int64_t>(M - r, kMost)), N, K, w4_log2g(G)};
        hipError_t st;
        if (!K) {
            timed_launch("w4_zero", w4_zero_kernel, dim3((N + 255) / 256, std::min(a.M, 1024)), dim3(256), 0, stream, a);
            st = hipGetLastError();
        } else st = x_type == ORNITH_W4_BF16 ? w4_rows<ORNITH_W4_BF16>(a, stream) : w4_rows<ORNITH_W4_F16>(a, stream);
        if (st != hipSuccess) return st;
    }
    return hipSuccess;
}
