// Sampling: one token per row of logits by temperature, top-k, top-p and min-p
// (definitions: include/ornith_sample.h).
//
// Every cut keeps a prefix of the order (value descending, column ascending),
// so a row's kept set is { i : comp(i) >= threshold } with
// comp = (ordered value bits << 32) | ~column.  The threshold is found through
// a histogram and a short list, without a sort:
//   parts   one block per 8192 columns: counts and masses of the part in bins
//           an eighth of a power of two of mass wide, 37 powers of two deep;
//   select  one block per row: the parts' histograms added up, the bins that
//           hold the borders; rows with no cut, and greedy ones, end here;
//   gather  one block per part: (value, column) of the logits in those bins;
//   finish  one block per row: the threshold inside its bin, the kept mass per
//           part, and the walk through the one part that holds the token.
//
// Masses.  With c = log2(e) / T and t = l c in fp64, e = 2^(t - j) for the
// whole number j = ceil(max t) of its part: a degree-8 polynomial in the
// fraction of t (relative error 2^-39.7), rounded to a whole number of units
// 2^-36.  One 64-bit LDS add carries count (14 bits) and mass (50 bits: 8192
// entries of at most 2^36).  Whole numbers make the sums independent of the
// order of the atomics.  A row adds parts in units of 2^-42 of 2^J, J the
// largest j: (mass << 6) >> (J - j), below 2^63 for 2^20 columns.  Row units
// truncate per (part, bin) where J - j > 6, a relative 2^-42 each.
// The bin, floor(8 t), comes from t alone, so equal values share a bin in every
// part and bins are ordered as values are.
#include "kernels.hpp"
#include "timing.hpp"
#include "validate.hpp"
#include "../../include/ornith_sample.h"

namespace ornith {
namespace {

constexpr int kPart = 8192, kPartsMax = 128;         // columns of a part; parts of 2^20 columns
constexpr int kOctaves = 37, kSub = 8;
constexpr int kTopBin = kOctaves * kSub;             // bin of t == j; bins 0 .. kTopBin
constexpr int kBins = 304;                           // padded
constexpr int kMaskWords = 10;
constexpr int kMassBits = 50;
constexpr uint64_t kMassMask = (uint64_t(1) << kMassBits) - 1;
constexpr int kRowShift = 6;                         // part units -> row units at j == J
constexpr int kListMax = 32768, kListLds = 4096;     // border entries kept per row, and in LDS
constexpr int kChunkRows = 64;                       // rows that share the workspace at once
constexpr int kPartThreads = 256, kRowThreads = 512;

enum : uint32_t { kSampleNan = 1, kSampleSetting = 2, kSampleEmpty = 4 };

struct PartMeta { double j; uint32_t key; int32_t arg; };     // key 0: nothing takes part

struct RowState {
    double J;
    uint64_t threshold_q;                            // min-p's threshold (0: none)
    int32_t done, walk;                              // ended in select; border bins too full for the list
    int32_t bin_k, use_k, use_p;
    uint32_t count;                                  // list entries
    uint32_t mask[kMaskWords];                       // border bins
    uint64_t cum_mass[kBins];                        // of bins >= i
    uint32_t cum_count[kBins];
};

struct SampleArgs {
    const void* logits; int64_t ld; int N, parts;
    const float *uniform, *temperature; const int32_t* top_k; const float *top_p, *min_p;
    uint64_t* hist;                                  // [rows, parts, kBins] count << 50 | mass
    PartMeta* meta;                                  // [rows, parts]
    RowState* state;                                 // [rows]
    uint2* list;                                     // [rows, kListMax] value bits (ordered), column
    int64_t* token; float* logprob; uint32_t* flags;
};

// ---- values -------------------------------------------------------------------
template <int TYPE> constexpr int kBytes = TYPE == ORNITH_LOGITS_F32 ? 4 : 2;

template <int TYPE> __device__ __forceinline__ float load1(const void* row, int col) {
    if constexpr (TYPE == ORNITH_LOGITS_F32) return static_cast<const float*>(row)[col];
    const uint32_t b = static_cast<const uint16_t*>(row)[col];
    return TYPE == ORNITH_LOGITS_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}
// Rows start at any element: 16-byte loads of element-aligned memory.
struct __attribute__((packed, aligned(2))) Raw16 { uint32_t w[4]; };
// Eight columns from col; columns at or past N read as -inf.
template <int TYPE> __device__ __forceinline__ void load8(const void* row, int col, int N, float (&v)[8]) {
    if (col + 8 <= N) {
        const auto* p = reinterpret_cast<const Raw16*>(static_cast<const uint8_t*>(row) + size_t(col) * kBytes<TYPE>);
        if constexpr (TYPE == ORNITH_LOGITS_F32) {
            const Raw16 a = p[0], b = p[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = __uint_as_float(a.w[e]);
                v[4 + e] = __uint_as_float(b.w[e]);
            }
        } else {
            const Raw16 a = p[0];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t b = (a.w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
                v[e] = TYPE == ORNITH_LOGITS_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = col + e < N ? load1<TYPE>(row, col + e) : -__builtin_huge_valf();
    }
}

// Bits ordered as the values are (-0 as +0; never 0 for a value above -inf).
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kMinusInf = 0x007fffffu;          // ordered(-inf)
__device__ __forceinline__ uint64_t comp_of(uint32_t key, int col) { return (uint64_t(key) << 32) | uint32_t(~col); }

// 2^(x + 1/2) for |x| <= 1/2, degree 8 (Chebyshev interpolation; relative error 2^-39.7)
__device__ __forceinline__ double exp2_half(double x) {
    double p = 0x1.f7318d7c8c8f4p-20;
    p = __builtin_fma(p, x, 0x1.6b416dbad124ep-16);
    p = __builtin_fma(p, x, 0x1.c8d6c3ed5deadp-13);
    p = __builtin_fma(p, x, 0x1.ee4eccd91f352p-10);
    p = __builtin_fma(p, x, 0x1.bdb6970fc2c99p-7);
    p = __builtin_fma(p, x, 0x1.41839f011e158p-4);
    p = __builtin_fma(p, x, 0x1.5be298adea926p-2);
    p = __builtin_fma(p, x, 0x1.f5e465377fff3p-1);
    return __builtin_fma(p, x, 0x1.6a09e667f3bccp+0);
}

// Bin and mass of a value in a part with the given j; bin < 0: below the bins
// (NaN and -inf too).  The high word of `packed` lacks the count.
__device__ __forceinline__ int bin_mass(float v, double c, double j, uint64_t& mass) {
    const double t = double(v) * c;
    if (j == __builtin_huge_val()) {                  // uniform: +inf in the part, its mass all there is
        mass = uint64_t(1) << (kMassBits - 14);
        return v == __builtin_huge_valf() ? kTopBin : -1;
    }
    const double n = __builtin_floor(t), r = t - n;
    const int up = int(fmax(n - j, -64.0));           // <= 0 (fmax takes the number of a NaN difference)
    const int bin = up * kSub + int(r * double(kSub)) + kTopBin;
    double e = exp2_half(r - 0.5);
    e = __longlong_as_double(__double_as_longlong(e) + (int64_t(up + 36) << 52));
    mass = uint64_t(__double_as_longlong(e + 0x1p52)) & ((uint64_t(1) << 52) - 1);
    return v > -__builtin_huge_valf() ? bin : -1;
}

__device__ __forceinline__ int part_shift(double J, double j) {
    return J == j ? 0 : int(fmin(J - j, 64.0));
}
__device__ __forceinline__ uint64_t row_mass(uint64_t m, int shift) {
    return shift < 64 ? (m << kRowShift) >> shift : 0;
}
// u in [0, 1) as a 64-bit fraction (below 2^-40 its last bits are cut)
__device__ __forceinline__ uint64_t fraction(float u) { return uint64_t(double(u) * 0x1p64); }

struct Setting { float T, p, q, u; int k; bool valid; double c; };
__device__ __forceinline__ Setting setting(const SampleArgs& a, int row) {
    Setting s;
    s.T = a.temperature ? a.temperature[row] : 1.f;
    s.k = a.top_k ? a.top_k[row] : 0;
    s.p = a.top_p ? a.top_p[row] : 1.f;
    s.q = a.min_p ? a.min_p[row] : 0.f;
    s.u = a.uniform[row];
    s.valid = s.T >= 0.f && s.T < __builtin_huge_valf() && s.p > 0.f && s.p <= 1.f && s.q >= 0.f && s.q <= 1.f &&
              s.u >= 0.f && s.u < 1.f;
    s.c = s.T > 0.f ? 0x1.71547652b82fep+0 / double(s.T) : 0.0;
    return s;
}

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
    return v;
}

// ---- parts ----------------------------------------------------------------------
template <int TYPE>
__global__ __launch_bounds__(kPartThreads) void sample_parts_kernel(SampleArgs a, int row0) {
    const int part = blockIdx.x, slot = blockIdx.y, row = row0 + slot, tid = threadIdx.x;
    __shared__ uint64_t s_hist[kBins];
    __shared__ uint32_t s_key[kPartThreads / 64];
    __shared__ int s_arg[kPartThreads / 64];
    const auto* src = static_cast<const uint8_t*>(a.logits) + size_t(row) * size_t(a.ld) * kBytes<TYPE>;
    const Setting s = setting(a, row);
    constexpr int kPieces = kPart / 8 / kPartThreads;
    float v[kPieces][8];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) load8<TYPE>(src, part * kPart + (u * kPartThreads + tid) * 8, a.N, v[u]);
    for (int i = tid; i < kBins; i += kPartThreads) s_hist[i] = 0;
    float mx = -__builtin_huge_valf();
    bool nan = false;
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            nan |= v[u][e] != v[u][e];
            mx = fmaxf(mx, v[u][e]);
        }
    if (__builtin_amdgcn_ballot_w64(nan) && (tid & 63) == 0) flag_or(a.flags, kSampleNan);
    const uint32_t wkey = wave_max_u(ordered(mx));
    if ((tid & 63) == 0) s_key[tid >> 6] = wkey;
    __syncthreads();
    uint32_t key = s_key[0];
#pragma unroll
    for (int w = 1; w < kPartThreads / 64; ++w) key = max(key, s_key[w]);
    PartMeta* meta = a.meta + size_t(slot) * a.parts + part;
    uint64_t* hist = a.hist + (size_t(slot) * a.parts + part) * kBins;
    if (key <= kMinusInf) {
        if (tid == 0) *meta = PartMeta{-__builtin_huge_val(), 0, 0};
        return;
    }
    if (s.T == 0.f) {                                 // greedy: the first column of the largest value
        int arg = 0x7fffffff;
#pragma unroll
        for (int u = kPieces - 1; u >= 0; --u)
#pragma unroll
            for (int e = 7; e >= 0; --e)
                if (ordered(v[u][e]) == key && v[u][e] == v[u][e]) arg = part * kPart + (u * kPartThreads + tid) * 8 + e;
        arg = wave_min_i(arg);
        if ((tid & 63) == 0) s_arg[tid >> 6] = arg;
        __syncthreads();
        if (tid == 0) {
#pragma unroll
            for (int w = 1; w < kPartThreads / 64; ++w) arg = min(arg, s_arg[w]);
            *meta = PartMeta{0.0, key, arg};
        }
        return;
    }
    const double j = __builtin_ceil(double(unordered(key)) * s.c);
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            uint64_t mass;
            const int bin = bin_mass(v[u][e], s.c, j, mass);
            if (bin >= 0) atomicAdd(reinterpret_cast<unsigned long long*>(&s_hist[bin]),
                                    (unsigned long long)(mass + (uint64_t(1) << kMassBits)));
        }
    __syncthreads();
    for (int i = tid; i < kBins; i += kPartThreads) hist[i] = s_hist[i];
    if (tid == 0) *meta = PartMeta{j, key, 0};
}

// ---- the end of a row --------------------------------------------------------------
struct RowShared {
    double j[kPartsMax];
    int shift[kPartsMax];
    uint64_t part_mass[kPartsMax];
    uint64_t wave[kRowThreads / 64];
    uint64_t rest, total;
    int part;
};

// Loads the parts' j and the shifts to the row's J.
__device__ __forceinline__ void load_parts(const SampleArgs& a, int slot, double J, RowShared& sh) {
    const PartMeta* meta = a.meta + size_t(slot) * a.parts;
    for (int p = threadIdx.x; p < a.parts; p += kRowThreads) {
        const double j = meta[p].key ? meta[p].j : -__builtin_huge_val();
        sh.j[p] = j;
        sh.shift[p] = meta[p].key ? part_shift(J, j) : 64;
    }
}

// part_mass[p] = the row mass of the part's bins above `bin`.
__device__ __forceinline__ void sum_parts(const SampleArgs& a, int slot, int bin, RowShared& sh) {
    const int lane = threadIdx.x & 63;
    for (int p = threadIdx.x >> 6; p < a.parts; p += kRowThreads / 64) {
        uint64_t m = 0;
        if (sh.shift[p] < 64) {
            const uint64_t* hist = a.hist + (size_t(slot) * a.parts + p) * kBins;
            for (int i = bin + 1 + lane + kSub * sh.shift[p]; i <= kTopBin; i += 64)
                m += row_mass(hist[i] & kMassMask, sh.shift[p]);
        }
        m = wave_sum_u64(m);
        if (lane == 0) sh.part_mass[p] = m;
    }
}

// part_mass holds the kept mass of every part: the part that holds the token,
// then the token inside it.  Kept: comp >= threshold.
template <int TYPE>
__device__ void draw(const SampleArgs& a, int row, const Setting& s, double J, uint64_t threshold, RowShared& sh) {
    const int tid = threadIdx.x, lane = tid & 63;
    if (tid < 64) {
        uint64_t m[kPartsMax / 64], before = 0;
#pragma unroll
        for (int h = 0; h < kPartsMax / 64; ++h) {
            const int p = h * 64 + lane;
            m[h] = p < a.parts ? sh.part_mass[p] : 0;
        }
        uint64_t total = 0;
#pragma unroll
        for (int h = 0; h < kPartsMax / 64; ++h) total += wave_sum_u64(m[h]);
        const uint64_t target = __umul64hi(fraction(s.u), total);      // token: the first column past it
#pragma unroll
        for (int h = 0; h < kPartsMax / 64; ++h) {
            uint64_t run = m[h];
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint64_t o = __shfl_up(run, d, 64);
                if (lane >= d) run += o;
            }
            if (before + run > target && before + run - m[h] <= target) {
                sh.part = h * 64 + lane;
                sh.rest = target - (before + run - m[h]);
            }
            before += __shfl(run, 63, 64);
        }
        if (lane == 0) sh.total = total;
    }
    __syncthreads();
    const int part = sh.part, shift = sh.shift[part];
    const uint64_t rest = sh.rest;
    const double j = sh.j[part];
    const auto* src = static_cast<const uint8_t*>(a.logits) + size_t(row) * size_t(a.ld) * kBytes<TYPE>;
    constexpr int kPer = kPart / kRowThreads;           // consecutive columns of a thread
    const int col0 = part * kPart + tid * kPer;
    float v[kPer / 8][8];
    uint64_t sum = 0;
    auto mass_at = [&](float x, int col) -> uint64_t {
        uint64_t m;
        const int bin = bin_mass(x, s.c, j, m);
        return bin >= 0 && comp_of(ordered(x), col) >= threshold ? m : 0;
    };
#pragma unroll
    for (int u = 0; u < kPer / 8; ++u) load8<TYPE>(src, col0 + 8 * u, a.N, v[u]);
#pragma unroll
    for (int u = 0; u < kPer / 8; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += mass_at(v[u][e], col0 + 8 * u + e);
    uint64_t run = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up(run, d, 64);
        if (lane >= d) run += o;
    }
    if (lane == 63) sh.wave[tid >> 6] = run;
    __syncthreads();
    for (int w = 0; w < (tid >> 6); ++w) run += sh.wave[w];
    if (row_mass(run, shift) > rest && row_mass(run - sum, shift) <= rest) {
        uint64_t at = run - sum;
        bool found = false;
#pragma unroll
        for (int u = 0; u < kPer / 8; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint64_t m = mass_at(v[u][e], col0 + 8 * u + e);
                at += m;
                if (!found && row_mass(at, shift) > rest) {
                    found = true;
                    a.token[row] = col0 + 8 * u + e;
                    if (a.logprob) {
                        const double t = double(v[u][e]) * s.c;
                        const double up = J == __builtin_huge_val() ? 0.0 : t - J;
                        const double ln = up * 0x1.62e42fefa39efp-1 - log(double(sh.total) * 0x1p-42);
                        a.logprob[row] = row_mass(m, shift) == sh.total ? 0.f : float(ln);   // alone
                    }
                }
            }
    }
}

// ---- select -----------------------------------------------------------------------
template <int TYPE>
__global__ __launch_bounds__(kRowThreads) void sample_select_kernel(SampleArgs a, int row0) {
    const int slot = blockIdx.x, row = row0 + slot, tid = threadIdx.x;
    __shared__ RowShared sh;
    __shared__ uint64_t s_mass[2][kRowThreads];
    __shared__ uint32_t s_count[2][kRowThreads];
    __shared__ uint32_t s_mask[kMaskWords];
    __shared__ uint64_t s_lo, s_hi;
    __shared__ int s_bin[3];
    __shared__ unsigned long long s_best;
    __shared__ uint32_t s_qkey, s_entries;
    RowState* st = a.state + slot;
    const Setting s = setting(a, row);
    const PartMeta* meta = a.meta + size_t(slot) * a.parts;

    if (tid == 0) s_best = 0;
    if (tid < kMaskWords) s_mask[tid] = 0;
    if (tid < 3) s_bin[tid] = -1;
    __syncthreads();
    // the row's largest value, and (greedy) its first column: parts ascend, so the first part wins
    for (int p = tid; p < a.parts; p += kRowThreads)
        if (meta[p].key) atomicMax(&s_best, (unsigned long long)((uint64_t(meta[p].key) << 32) | uint32_t(~p)));
    __syncthreads();
    const uint32_t top = uint32_t(s_best >> 32);
    if (!s.valid || top == 0 || s.T == 0.f) {
        if (tid == 0) {
            st->done = 1;
            const bool fine = s.valid && top != 0;
            a.token[row] = fine ? meta[~uint32_t(s_best)].arg : -1;
            if (a.logprob) a.logprob[row] = fine ? 0.f : __builtin_nanf("");
            flag_or(a.flags, !s.valid ? kSampleSetting : top == 0 ? kSampleEmpty : 0u);
        }
        return;
    }
    const float mx = unordered(top);
    const double J = __builtin_ceil(double(mx) * s.c);
    load_parts(a, slot, J, sh);
    __syncthreads();
    uint64_t mass = 0;
    uint32_t count = 0;
    if (tid <= kTopBin) {
        const uint64_t* hist = a.hist + size_t(slot) * a.parts * kBins;
        for (int p = 0; p < a.parts; ++p) {
            const int i = tid + kSub * sh.shift[p];
            if (i > kTopBin) continue;
            const uint64_t w = hist[size_t(p) * kBins + i];
            count += uint32_t(w >> kMassBits);
            mass += row_mass(w & kMassMask, sh.shift[p]);
        }
    }
    // sums over bins >= tid
    s_mass[0][tid] = mass;
    s_count[0][tid] = count;
    int from = 0;
    for (int d = 1; d < kRowThreads; d <<= 1, from ^= 1) {
        __syncthreads();
        if (tid + d < kRowThreads) {
            mass += s_mass[from][tid + d];
            count += s_count[from][tid + d];
        }
        s_mass[from ^ 1][tid] = mass;
        s_count[from ^ 1][tid] = count;
    }
    __syncthreads();
    const uint64_t* cm = s_mass[from];
    const uint32_t* cc = s_count[from];
    const bool use_k = s.k > 0 && uint32_t(s.k) < cc[0], use_p = s.p < 1.f, use_q = s.q > 0.f;
    if (!use_k && !use_p && !use_q) {
        sum_parts(a, slot, -1, sh);
        if (tid == 0) st->done = 1;
        __syncthreads();
        draw<TYPE>(a, row, s, J, 0, sh);
        return;
    }
    // the bin that holds the k-th value, and the range of the mass of the first k
    if (tid == 0) { s_lo = cm[0]; s_hi = cm[0]; s_qkey = kMinusInf + 1; }
    __syncthreads();
    if (use_k && tid <= kTopBin && cc[tid] >= uint32_t(s.k) && (tid == kTopBin || cc[tid + 1] < uint32_t(s.k))) {
        s_bin[0] = tid;
        s_hi = cm[tid];
        s_lo = cc[tid] == uint32_t(s.k) ? cm[tid] : tid == kTopBin ? 0 : cm[tid + 1];
    }
    __syncthreads();
    // the bins that top-p's border can lie in
    if (use_p && tid <= kTopBin) {
        const uint64_t f = fraction(s.p);
        const uint64_t lo = max(__umul64hi(f, s_lo), uint64_t(1)), hi = __umul64hi(f, s_hi) + 1;
        const uint64_t next = tid == kTopBin ? 0 : cm[tid + 1];
        if (cm[tid] >= lo && next < lo) s_bin[1] = tid;                      // upper end
        if ((cm[tid] >= hi || tid == 0) && next < hi) s_bin[2] = tid;        // lower end
    }
    // min-p's least value: the estimate mx + T ln q is off by less than a step of fp32 there, so
    // the 64 values around it hold the border
    if (use_q && tid < 64) {
        const float at = float(double(mx) + double(s.T) * log(double(s.q)));
        const uint32_t mid = at == at ? ordered(at) : kMinusInf + 1;
        const uint32_t k0 = max(min(mid, top), kMinusInf + 33) - 32 + tid;
        const float v = unordered(k0);
        const bool in = k0 <= top && (v == mx || (double(v) - double(mx)) * s.c >= log2(double(s.q)));
        const uint64_t b = __builtin_amdgcn_ballot_w64(in);
        if (tid == 0) s_qkey = b ? k0 + uint32_t(__builtin_ctzll(b)) : top;
    }
    __syncthreads();
    if (tid == 0) {
        uint64_t tq = 0;
        auto mark = [&](int lo, int hi) {
            for (int i = max(lo, 0); i <= hi; ++i) s_mask[i >> 5] |= 1u << (i & 31);
        };
        // the strictest bin the other cuts can end in, and the least strict
        const int kp_hi = max(use_k ? s_bin[0] : -1, use_p ? s_bin[1] : -1);
        const int kp_lo = max(use_k ? s_bin[0] : -1, use_p ? s_bin[2] : -1);
        int bq = -1;
        if (use_q) {
            tq = uint64_t(s_qkey) << 32;
            uint64_t unused;
            bq = bin_mass(unordered(s_qkey), s.c, J, unused);
        }
        int32_t k = use_k, p = use_p;
        if (bq > kp_hi) {                                  // min-p alone decides
            k = 0;
            p = 0;
            mark(bq, bq);
        } else {
            if (use_k) mark(s_bin[0], s_bin[0]);
            if (use_p) mark(s_bin[2], s_bin[1]);
            if (bq >= 0 && bq >= kp_lo) mark(bq, bq);
        }
        st->J = J;
        st->threshold_q = tq;
        st->done = 0;
        st->use_k = k;
        st->use_p = p;
        st->bin_k = s_bin[0];
        st->count = 0;
        s_entries = 0;
    }
    __syncthreads();
    if (tid <= kTopBin && (s_mask[tid >> 5] >> (tid & 31) & 1))
        atomicAdd(&s_entries, cc[tid] - (tid == kTopBin ? 0 : cc[tid + 1]));
    __syncthreads();
    if (tid == 0) st->walk = s_entries > kListMax;
    if (tid < kMaskWords) st->mask[tid] = s_mask[tid];
    if (tid < kBins) {
        st->cum_mass[tid] = cm[tid];
        st->cum_count[tid] = cc[tid];
    }
}

// ---- gather -----------------------------------------------------------------------
template <int TYPE>
__global__ __launch_bounds__(kPartThreads) void sample_gather_kernel(SampleArgs a, int row0) {
    const int part = blockIdx.x, slot = blockIdx.y, row = row0 + slot, tid = threadIdx.x;
    RowState* st = a.state + slot;
    if (st->done || st->walk) return;
    const PartMeta meta = a.meta[size_t(slot) * a.parts + part];
    if (!meta.key) return;
    const double J = st->J;
    const int shift = part_shift(J, meta.j);
    if (shift >= 64) return;
    __shared__ uint32_t s_mask[kMaskWords];
    __shared__ int s_any;
    if (tid < kMaskWords) s_mask[tid] = st->mask[tid];
    if (tid == 0) s_any = 0;
    __syncthreads();
    const uint64_t* hist = a.hist + (size_t(slot) * a.parts + part) * kBins;
    bool any = false;
    for (int i = tid + kSub * shift; i <= kTopBin; i += kPartThreads) {
        const int b = i - kSub * shift;
        any |= (s_mask[b >> 5] >> (b & 31) & 1) && (hist[i] >> kMassBits);
    }
    if (any) s_any = 1;
    __syncthreads();
    if (!s_any) return;
    const Setting s = setting(a, row);
    const auto* src = static_cast<const uint8_t*>(a.logits) + size_t(row) * size_t(a.ld) * kBytes<TYPE>;
    uint2* list = a.list + size_t(slot) * kListMax;
    constexpr int kPieces = kPart / 8 / kPartThreads;
    float v[kPieces][8];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) load8<TYPE>(src, part * kPart + (u * kPartThreads + tid) * 8, a.N, v[u]);
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            uint64_t mass;
            const int b = bin_mass(v[u][e], s.c, meta.j, mass) - kSub * shift;
            if (b >= 0 && (s_mask[b >> 5] >> (b & 31) & 1)) {
                const uint32_t at = atomicAdd(&st->count, 1u);
                if (at < kListMax)
                    list[at] = make_uint2(ordered(v[u][e]), uint32_t(part * kPart + (u * kPartThreads + tid) * 8 + e));
            }
        }
}

// ---- finish -----------------------------------------------------------------------
struct Entries {
    uint64_t comp[kListLds], mass[kListLds];
    uint16_t bin[kListLds];
};

template <int TYPE>
__global__ __launch_bounds__(kRowThreads) void sample_finish_kernel(SampleArgs a, int row0) {
    const int slot = blockIdx.x, row = row0 + slot, tid = threadIdx.x;
    RowState* st = a.state + slot;
    if (st->done) return;
    __shared__ RowShared sh;
    __shared__ Entries en;
    __shared__ uint32_t s_cnt[256];
    __shared__ unsigned long long s_mass[256], s_found;
    __shared__ uint32_t s_digit, s_group;
    __shared__ uint64_t s_need;
    __shared__ unsigned long long s_sum;
    __shared__ int s_bin;
    const Setting s = setting(a, row);
    const double J = st->J;
    load_parts(a, slot, J, sh);
    __syncthreads();
    const bool walk = st->walk;
    const int n = walk ? 0 : int(min(st->count, uint32_t(kListMax)));
    const uint2* list = a.list + size_t(slot) * kListMax;
    const auto* src = static_cast<const uint8_t*>(a.logits) + size_t(row) * size_t(a.ld) * kBytes<TYPE>;

    // f(comp, row mass, row bin, part) of a border entry
    auto entry = [&](float v, int col, auto&& f) {
        const int part = col / kPart, shift = sh.shift[part];
        if (shift >= 64) return;
        uint64_t m;
        const int b = bin_mass(v, s.c, sh.j[part], m) - kSub * shift;
        if (b >= 0) f(comp_of(ordered(v), col), row_mass(m, shift), b, part);
    };
    const bool lds = !walk && n <= kListLds;
    if (lds) {
        for (int i = tid; i < n; i += kRowThreads)
            entry(unordered(list[i].x), int(list[i].y), [&](uint64_t comp, uint64_t m, int b, int) {
                en.comp[i] = comp;
                en.mass[i] = m;
                en.bin[i] = uint16_t(b);
            });
        __syncthreads();
    }
    // every border entry (and, walking the row, every other one) once over the block
    auto each = [&](auto&& f) {
        if (lds) {
            for (int i = tid; i < n; i += kRowThreads)
                f(en.comp[i], en.mass[i], int(en.bin[i]), int(~uint32_t(en.comp[i])) / kPart);
        } else if (!walk) {
            for (int i = tid; i < n; i += kRowThreads) entry(unordered(list[i].x), int(list[i].y), f);
        } else {
            for (int i = tid; i < a.N; i += kRowThreads) entry(load1<TYPE>(src, i), i, f);
        }
    };
    // The entry of bin `bin` at which, from the largest down, `need` is reached: a count, or a mass.  Byte by byte, the entries that share the prefix counted per next byte
    // (columns stay below 2^20, so byte 3 of comp is 0xff).  Ends with s_found the comp and s_sum
    // the mass from the bin's largest entry down to it.
    auto descend = [&](int bin, bool by_mass, uint64_t need) {
        uint64_t prefix = 0, known = 0, above = 0;
        const int shifts[7] = {56, 48, 40, 32, 16, 8, 0};
        for (int d = 0; d < 7; ++d) {
            const int sft = shifts[d];
            if (sft == 16) {
                prefix |= uint64_t(0xff) << 24;
                known |= uint64_t(0xff) << 24;
            }
            __syncthreads();
            if (tid < 256) {
                s_cnt[tid] = 0;
                s_mass[tid] = 0;
            }
            __syncthreads();
            each([&](uint64_t comp, uint64_t m, int b, int) {
                if (b != bin || (comp & known) != prefix) return;
                const int i = int(comp >> sft) & 255;
                atomicAdd(&s_cnt[i], 1u);
                atomicAdd(&s_mass[i], (unsigned long long)m);
            });
            __syncthreads();
            if (tid < 64) {
                // lane l: the digits 255 - 4 l .. 252 - 4 l
                uint32_t c[4];
                uint64_t m[4], cs = 0, ms = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 255 - (4 * tid + e);
                    c[e] = s_cnt[i];
                    m[e] = s_mass[i];
                    cs += c[e];
                    ms += m[e];
                }
                uint64_t cr = cs, mr = ms;
#pragma unroll
                for (int k = 1; k < 64; k <<= 1) {
                    const uint64_t oc = __shfl_up(cr, k, 64), om = __shfl_up(mr, k, 64);
                    if (tid >= k) { cr += oc; mr += om; }
                }
                uint64_t cb = cr - cs, mb = mr - ms;
                // the bin's entries can sum to a few units less than its parts' sums (which are cut
                // once per part): then the last entry is the border
                const uint64_t of = by_mass ? mr : cr;
                const bool short_of = uint64_t(__shfl(of, 63, 64)) < need;
                const int last = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(cs != 0) | 1);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint64_t b0 = by_mass ? mb : cb, b1 = by_mass ? mb + m[e] : cb + c[e];
                    if (short_of ? tid == last && c[e] : b0 < need && b1 >= need) {
                        s_digit = 255 - (4 * tid + e);
                        s_group = c[e];
                        s_need = short_of ? ~uint64_t(0) : need - b0;
                        s_sum = above + mb;
                    }
                    cb += c[e];
                    mb += m[e];
                }
            }
            __syncthreads();
            prefix |= uint64_t(s_digit) << sft;
            known |= uint64_t(0xff) << sft;
            need = s_need;
            above = s_sum;
            if (s_group == 1) break;
        }
        __syncthreads();
        each([&](uint64_t comp, uint64_t m, int b, int) {      // one entry is left
            if (b == bin && (comp & known) == prefix) {
                s_found = comp;
                s_sum = above + m;
            }
        });
        __syncthreads();
    };

    uint64_t threshold = st->threshold_q;
    uint64_t kept_k = 0;                                  // mass of the first k
    if (st->use_k) {
        const int b = st->bin_k;
        const uint32_t count_above = b == kTopBin ? 0 : st->cum_count[b + 1];
        const uint64_t mass_above = b == kTopBin ? 0 : st->cum_mass[b + 1];
        descend(b, false, uint64_t(s.k) - count_above);
        threshold = max(threshold, uint64_t(s_found));
        kept_k = mass_above + s_sum;
    }
    if (st->use_p) {
        const uint64_t of = st->use_k ? kept_k : st->cum_mass[0];
        const uint64_t f = fraction(s.p);
        const uint64_t target = max(__umul64hi(f, of) + (f * of != 0), uint64_t(1));
        if (tid <= kTopBin) {
            const uint64_t next = tid == kTopBin ? 0 : st->cum_mass[tid + 1];
            if (st->cum_mass[tid] >= target && next < target) s_bin = tid;
        }
        __syncthreads();
        const int b = s_bin;
        descend(b, true, target - (b == kTopBin ? 0 : st->cum_mass[b + 1]));
        threshold = max(threshold, uint64_t(s_found));
    }
    __syncthreads();
    if (tid == 0) {
        uint64_t unused;
        s_bin = bin_mass(unordered(uint32_t(threshold >> 32)), s.c, J, unused);
    }
    __syncthreads();
    const int bf = s_bin;
    sum_parts(a, slot, bf < 0 ? -1 : bf, sh);
    __syncthreads();
    if (bf >= 0)
        each([&](uint64_t comp, uint64_t m, int b, int part) {
            if (b == bf && comp >= threshold)
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.part_mass[part]), (unsigned long long)m);
        });
    __syncthreads();
    draw<TYPE>(a, row, s, J, threshold, sh);
}

// rows of an empty vocabulary
__global__ __launch_bounds__(64) void sample_empty_kernel(int M, int64_t* token, float* logprob, uint32_t* flags) {
    const int row = blockIdx.x * 64 + threadIdx.x;
    if (row >= M) return;
    token[row] = -1;
    if (logprob) logprob[row] = __builtin_nanf("");
    if (threadIdx.x == 0) flag_or(flags, kSampleEmpty);
}

struct SampleLayout { size_t hist, meta, state, list, bytes; };
SampleLayout sample_layout(int Mcap, int N) {
    SampleLayout l{};
    const size_t rows = size_t(Mcap < kChunkRows ? Mcap : kChunkRows), parts = (size_t(N) + kPart - 1) / kPart;
    size_t cursor = 0;
    auto add = [&](size_t& field, size_t bytes) { field = cursor; cursor = align256(cursor + bytes); };
    add(l.hist, rows * parts * kBins * 8);
    add(l.meta, rows * parts * sizeof(PartMeta));
    add(l.state, rows * sizeof(RowState));
    add(l.list, rows * size_t(kListMax) * 8);
    l.bytes = cursor;
    return l;
}

template <int TYPE> hipError_t sample_rows(const SampleArgs& a, int row0, int rows, hipStream_t s) {
    const dim3 parts(a.parts, rows);
    timed_launch("sample_parts", sample_parts_kernel<TYPE>, parts, dim3(kPartThreads), 0, s, a, row0);
    timed_launch("sample_select", sample_select_kernel<TYPE>, dim3(rows), dim3(kRowThreads), 0, s, a, row0);
    hipError_t st = hipGetLastError();
    // with no cut at all, select has drawn every row
    if (st != hipSuccess || (!a.top_k && !a.top_p && !a.min_p)) return st;
    timed_launch("sample_gather", sample_gather_kernel<TYPE>, parts, dim3(kPartThreads), 0, s, a, row0);
    timed_launch("sample_finish", sample_finish_kernel<TYPE>, dim3(rows), dim3(kRowThreads), 0, s, a, row0);
    return hipGetLastError();
}

}  // namespace
}  // namespace ornith

using namespace ornith;

extern "C" hipError_t ornith_logits_sample_get_layout(int Mcap, int N, size_t* workspace_bytes) {
    if (!workspace_bytes || Mcap < 0 || N < 0 || N > kPart * kPartsMax) return hipErrorInvalidValue;
    *workspace_bytes = sample_layout(Mcap, N).bytes;
    return hipSuccess;
}

extern "C" hipError_t ornith_logits_sample_launch(const void* logits, int logits_type, int M, int N, int64_t ld,
                                                  const void* uniform, const void* temperature, const void* top_k,
                                                  const void* top_p, const void* min_p, void* workspace,
                                                  size_t workspace_bytes, void* token, void* logprob, void* flags,
                                                  hipStream_t stream) {
    if (logits_type < ORNITH_LOGITS_BF16 || logits_type > ORNITH_LOGITS_F32 || M < 0 || N < 0 ||
        N > kPart * kPartsMax || ld < N)
        return hipErrorInvalidValue;
    if (!M) return hipSuccess;
    const SampleLayout l = sample_layout(M, N);
    if (workspace_bytes < l.bytes) return hipErrorInvalidValue;
    const size_t size = logits_type == ORNITH_LOGITS_F32 ? 4 : 2, m = size_t(M);
    const Buffer buffers[] = {{logits, N ? ((m - 1) * size_t(ld) + size_t(N)) * size : 0, size, false, N == 0},
                              {uniform, m * 4, 4, false, false},
                              {temperature, m * 4, 4, false, true},
                              {top_k, m * 4, 4, false, true},
                              {top_p, m * 4, 4, false, true},
                              {min_p, m * 4, 4, false, true},
                              {workspace, workspace_bytes, 256, true, l.bytes == 0},
                              {token, m * 8, 8, true, false},
                              {logprob, m * 4, 4, true, true},
                              {flags, 4, 4, true, false}};
    if (!check_buffers(buffers)) return hipErrorInvalidValue;
    if (!N) {
        timed_launch("sample_empty", sample_empty_kernel, dim3((M + 63) / 64), dim3(64), 0, stream, M,
                     static_cast<int64_t*>(token), static_cast<float*>(logprob), static_cast<uint32_t*>(flags));
        return hipGetLastError();
    }
    const SampleArgs a{logits, ld, N, (N + kPart - 1) / kPart, static_cast<const float*>(uniform),
                       static_cast<const float*>(temperature), static_cast<const int32_t*>(top_k),
                       static_cast<const float*>(top_p), static_cast<const float*>(min_p),
                       at<uint64_t>(workspace, l.hist), at<PartMeta>(workspace, l.meta),
                       at<RowState>(workspace, l.state), at<uint2>(workspace, l.list),
                       static_cast<int64_t*>(token), static_cast<float*>(logprob), static_cast<uint32_t*>(flags)};
    for (int r = 0; r < M; r += kChunkRows) {
        const int rows = M - r < kChunkRows ? M - r : kChunkRows;
        const hipError_t st = logits_type == ORNITH_LOGITS_BF16  ? sample_rows<ORNITH_LOGITS_BF16>(a, r, rows, stream)
                              : logits_type == ORNITH_LOGITS_F16 ? sample_rows<ORNITH_LOGITS_F16>(a, r, rows, stream)
                                                                 : sample_rows<ORNITH_LOGITS_F32>(a, r, rows, stream);
        if (st != hipSuccess) return st;
    }
    return hipSuccess;
}
