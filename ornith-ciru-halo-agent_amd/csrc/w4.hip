// Plain 4-bit linears (definition and bank layout: include/ornith_w4.h).
//
// On the matrix cores, with the codes as exact small floats: 16 + c has c in
// the top four mantissa bits of a bf16 or fp16 number of [16, 32), so two codes
// become a packed pair by a shift, a mask and an or.  Over one group
//   sum x (c - z) = sum x (16 + c) - (16 + z) sum x,
// both sums in fp32 on the matrix cores (sum x against a fragment of ones);
// each product is exact, and the first sum is at most 31 / |c - z| times the
// wanted one, so its roundings cost two to three bits of fp32, not of the
// result's type.  acc += s * (that), groups in ascending order within a wave.
#include "kernels.hpp"
#include "timing.hpp"
#include "validate.hpp"
#include "../../include/ornith_w4.h"

namespace ornith {
namespace {

constexpr int kW4MaxN = 1 << 20, kW4MaxK = 65536, kW4Rows = 64, kW4Block = 128;

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
                                                            int N, int K, size_t words) {
    const size_t i = size_t(blockIdx.x) * 256 + threadIdx.x;
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
                                                           int N, int groups, size_t words) {
    const size_t i = size_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= words) return;
    const size_t tg = i >> 4;
    const int n = int(tg / size_t(groups)) * 16 + int(i & 15), g = int(tg % size_t(groups));
    uint32_t w = 8;
    if (n < N) {
        const size_t at = size_t(n) * groups + g;
        const float s = scale_type == ORNITH_W4_BF16 ? bf16_bits_to_f32(scales[at]) : f16_bits_to_f32(scales[at]);
        w = (__float_as_uint(s) & ~15u) | (zeros ? zeros[at] & 15u : 8u);
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

// One block per 16 columns and 64 rows: its waves take the 128-k blocks in
// turn and add their sums in LDS, in wave order.
template <int TYPE, int MT, int W>
__global__ __launch_bounds__(64 * W) void w4_kernel(W4Args a) {
    __shared__ float s_acc[W][MT * 4][64];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, li = lane & 15, q = lane >> 4;
    const int tile = blockIdx.x, row0 = int(blockIdx.y) * kW4Rows, rows = min(a.M - row0, MT * 16);
    const int blocks = (a.K + kW4Block - 1) / kW4Block, groups = (a.K + (1 << a.log2g) - 1) >> a.log2g;
    const uint32_t* codes = a.codes + size_t(tile) * blocks * 256 + 4 * lane;
    const uint32_t* meta = a.meta + size_t(tile) * groups * 16 + li;
    const uint16_t* x = a.x + size_t(row0) * size_t(a.ldx);
    const int per = min(a.log2g, 7) - 5;                       // 32-k steps of a group in a block: 1, 2, 4
    const uint32_t one = TYPE == ORNITH_W4_BF16 ? 0x3f803f80u : 0x3c003c00u;
    const u32x4 ones = {one, one, one, one};
    f32x4 acc[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int kb = wv; kb < blocks; kb += W) {
        const u32x4 w4 = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(codes + size_t(kb) * 256));
        f32x4 c[MT], sx[MT];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = kb * kW4Block + 32 * j + 8 * q;
            if ((j & ((1 << per) - 1)) == 0)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) c[mt] = sx[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
            const u32x4 b = w4_unpack<TYPE>(w4[j]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const int r = min(16 * mt + li, rows - 1);
                u32x4 av = {0, 0, 0, 0};
                if (k < a.K) av = *reinterpret_cast<const u32x4*>(x + size_t(r) * size_t(a.ldx) + k);
                c[mt] = w4_mfma<TYPE>(av, b, c[mt]);
                sx[mt] = w4_mfma<TYPE>(av, ones, sx[mt]);
            }
            if (((j + 1) & ((1 << per) - 1)) == 0) {
                const int g = min((kb * kW4Block + 32 * j) >> a.log2g, groups - 1);
                const uint32_t m = meta[size_t(g) * 16];
                const float s = __uint_as_float(m & ~15u), z = -16.f - float(m & 15u);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[mt][i] = __builtin_fmaf(s, __builtin_fmaf(z, sx[mt][i], c[mt][i]), acc[mt][i]);
            }
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_acc[wv][4 * mt + i][lane] = acc[mt][i];
    __syncthreads();
    uint32_t flags = 0;
    for (int o = tid; o < MT * 4 * 64; o += 64 * W) {
        const int e = o >> 6, l = o & 63, row = 16 * (e >> 2) + 4 * (l >> 4) + (e & 3), n = tile * 16 + (l & 15);
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += s_acc[w][e][l];
        if (row >= rows || n >= a.N) continue;
        if (!isfinite(v)) flags |= kDenseNonfiniteProjection;
        const size_t at = size_t(row0 + row) * size_t(a.ldo) + n;
        if (a.out_type == ORNITH_W4_F32) static_cast<float*>(a.out)[at] = v;
        else {
            const uint16_t b = a.out_type == ORNITH_W4_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
            const uint32_t top = a.out_type == ORNITH_W4_BF16 ? 0x7f80u : 0x7c00u;
            if ((b & top) == top) flags |= kDenseNonfiniteBf16;
            static_cast<uint16_t*>(a.out)[at] = b;
        }
    }
    flag_or(a.flags, flags);
}

int w4_log2g(int G) { return G == 32 ? 5 : G == 64 ? 6 : G == 128 ? 7 : G == 256 ? 8 : -1; }

bool w4_words(int N, int K, int G, size_t& codes, size_t& meta) {
    if (N < 0 || N > kW4MaxN || K < 0 || K > kW4MaxK || K % 8 || w4_log2g(G) < 0) return false;
    const size_t tiles = (size_t(N) + 15) / 16;
    codes = tiles * ((size_t(K) + kW4Block - 1) / kW4Block) * 256;
    meta = tiles * ((size_t(K) + G - 1) / G) * 16;
    return true;
}

template <int TYPE> void w4_rows(const W4Args& a, hipStream_t s) {
    constexpr int W = 8;
    const dim3 grid((a.N + 15) / 16, (a.M + kW4Rows - 1) / kW4Rows);
    const int mt = a.M > 48 ? 4 : (a.M + 15) / 16;
    auto go = [&](auto kernel) { timed_launch("w4", kernel, grid, dim3(64 * W), 0, s, a); };
    if (mt == 1) go(w4_kernel<TYPE, 1, W>);
    else if (mt == 2) go(w4_kernel<TYPE, 2, W>);
    else if (mt == 3) go(w4_kernel<TYPE, 3, W>);
    else go(w4_kernel<TYPE, 4, W>);
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
                                     void* packed_codes, void* packed_meta, int N, int K, int G, hipStream_t stream) {
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
                              {packed_meta, m * 4, 4, true, false}};
    if (!check_buffers(buffers)) return hipErrorInvalidValue;
    timed_launch("w4_pack_codes", w4_pack_codes_kernel, dim3(unsigned((c + 255) / 256)), dim3(256), 0, stream,
                 static_cast<const uint32_t*>(codes), static_cast<uint32_t*>(packed_codes), N, K, c);
    const hipError_t st = hipGetLastError();
    if (st != hipSuccess) return st;
    timed_launch("w4_pack_meta", w4_pack_meta_kernel, dim3(unsigned((m + 255) / 256)), dim3(256), 0, stream,
                 static_cast<const uint16_t*>(scales), scale_type, static_cast<const uint8_t*>(zeros),
                 static_cast<uint32_t*>(packed_meta), N, groups, m);
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
    // rows ride on the grid's y axis (65535 blocks of 64 rows at most)
    constexpr int kMost = 65535 * kW4Rows;
    for (int r = 0; r < M; r += kMost) {
        const W4Args a{static_cast<const uint16_t*>(x) + size_t(r) * size_t(ldx), ldx,
                       static_cast<const uint32_t*>(codes), static_cast<const uint32_t*>(meta),
                       static_cast<uint8_t*>(out) + size_t(r) * size_t(ldo) * size, out_type, ldo,
                       static_cast<uint32_t*>(flags), M - r < kMost ? M - r : kMost, N, K, w4_log2g(G)};
        if (x_type == ORNITH_W4_BF16) w4_rows<ORNITH_W4_BF16>(a, stream);
        else w4_rows<ORNITH_W4_F16>(a, stream);
        const hipError_t st = hipGetLastError();
        if (st != hipSuccess) return st;
    }
    return hipSuccess;
}
