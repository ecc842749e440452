// Sampling: one token per row of logits by temperature, top-k, top-p and min-p
// (definitions: include/ornith_sample.h).
//
// Every cut keeps a prefix of the order (value descending, column ascending),
// so a row's kept set is { i : comp(i) >= threshold } with comp = (ordered value
// bits << 20) | complement of the column.  The threshold is found through a
// histogram and a short list, without a sort:
//   parts   one block per 8192 columns: counts and masses of the part in bins
//           an eighth of a power of two of mass wide, 37 powers of two deep;
//   select  one block per row: the parts' histograms added up, the bins that
//           hold the borders; rows with no cut, and greedy ones, end here;
//   gather  one block per part: (value, column) of the logits in those bins, or,
//           where no more than 256 logits lie in or above them, of all those;
//   finish  one block per row: the threshold inside its bin, the kept mass per
//           part, and the walk through the one part that holds the token (of the
//           256: threshold and token from the list alone).
// Rows of one part do all of it in one block and one launch (sample_row).  Calls of few parts do the
// last three steps in one launch (sample_rest), whose last block to list its entries ends the row.
//
// What bounds it.  The floor is one pass over the logits (64 rows of 248320 bf16: 31.8 MB, 6.0 us at the
// 5.3 TB/s of a large copy).  `parts` takes 16.7 us there: 10.9 to load and find the maxima, the rest fp64
// for the masses (a dozen instructions a value, 7 to 8 clocks each a wave); top-p's histogram costs 9 us
// of LDS additions and bins more.  Everything behind it works on bins and lists and is a chain of launches and
// round trips: a whole row is drawn in 7.0 us, borders take 6 to 7, the list 8 to 9, its end 5 (few
// candidates) to 19 (2800 entries a row).  Calls in a graph over six inputs in turn: 1 row of top-k and
// top-p 15.7 us, 8 rows of 151936 fp32 with top-p 25.3, 64 rows of mixed settings 46, 64 uncut 22 to 23.5,
// 256 rows of 4096 columns 17.2.
//
// Masses.  With c = log2(e) / T and t = l c in fp64, e = 2^(t - j) for the
// whole number j = ceil(max t) of its part: a degree-7 polynomial in t - rint(t)
// (relative error 2^-33), rounded to a whole number of units 2^-36.  One
// 64-bit LDS add carries count (14 bits) and mass (50 bits: 8192 entries of at
// most 2^36).  Whole numbers make the sums independent of the order of the
// atomics.  A row adds parts in units of 2^-42 of 2^J, J the largest j:
// (mass << 6) >> (J - j), below 2^63 for 2^20 columns.  Row units truncate per
// (part, bin) where J - j > 6, a relative 2^-42 each.  The bin, rint(8 t), comes
// from t alone, so equal values share a bin in every part and bins are ordered
// as values are.
#include <algorithm>
#include "kernels.hpp"
#include "timing.hpp"
#include "validate.hpp"
#include "../../include/ornith_sample.h"

namespace ornith {
namespace {

constexpr int kPart = 8192, kPartsMax = 128;         // columns of a part; parts of 2^20 columns
constexpr int kColBits = 20;
constexpr int kOctaves = 37, kSub = 8;
constexpr int kTopBin = kOctaves * kSub;             // bin of t == j; bins 0 .. kTopBin
constexpr int kBins = 304;                           // padded
constexpr int kMassBits = 50;
constexpr uint64_t kMassMask = (uint64_t(1) << kMassBits) - 1;
constexpr uint64_t kPartOne = uint64_t(1) << 36;     // mass 1 in part units
constexpr int kRowShift = 6;                         // part units -> row units at j == J
// Sizes that choose a way, with both ways measured (us; 64 rows of 248320 bf16 where nothing else is said):
constexpr int kListMax = 16384;                      // border entries kept per row (more: the row is read again)
constexpr int kListLds = 8192;                       // and in LDS (top-p, 2800 a row: finish 18.9, from memory 24.6)
constexpr int kSmall = 256;                          // rows decided by a list of all their candidates (top-k 20 to 50:
                                                     // finish 4.8, by borders 13.2; 256 rows of 4096: 11.6 / 20.2)
constexpr int kMaximaK = 256;                        // top_k up to which a part drops what cannot be among it (top-k
                                                     // 20 to 50: parts 13.3, without 25.0)
constexpr int kQueue = 512;                          // a wave's surviving values, compacted up to here (the same:
                                                     // parts 13.3, without 16.7)
// Parts of a call up to which two launches do it: a block per part and CU, each with the row's plan (two /
// four launches: top-k of 1 row 16.9 / 21.1, 8 rows 18.0 / 22.7, 16 rows 30.5 / 24.0; fp32 of 151936,
// top-p, 8 rows 26.0 / 33.8, 16 rows 34.3 / 37.7, 32 rows 48.2 / 43.1).
constexpr int kFewParts = 256;
constexpr int kRowThreads = 1024, kRowWaves = kRowThreads / 64, kPer = kPart / kRowThreads;
constexpr uint32_t kMinusInf = 0x007fffffu;          // ordered(-inf)
constexpr uint32_t kKeyEnd = 0xffffffffu;            // above every key

enum : uint32_t { kSampleNan = 1, kSampleSetting = 2, kSampleEmpty = 4 };
enum : int { kDone = 0, kModeSmall = 1, kModeList = 2, kModeWalk = 3 };

// key: the largest value (0: nothing takes part); arg: its first column (greedy rows); mass: of rows
// without a cut; least: values below it are not in the histogram
struct PartMeta { double j; uint64_t mass; uint32_t key; int32_t arg; float least; };

// What select leaves for gather and finish.
struct Plan {
    double J;
    float mx;                                        // the row's largest value
    uint64_t threshold_q;                            // min-p's threshold (0: none)
    uint64_t total, above_mass;                      // row mass; mass of the bins above bin_k
    int32_t mode, use_k, use_p, bin_k, bin_q, above_count;
    int32_t bin_lo[3], bin_hi[3];                    // the ranges' bins
    uint32_t lo[3], hi[3];                           // key ranges [lo, hi) to gather (the first: bin_k's; unused: empty)
};
struct RowState {
    Plan plan;
    uint32_t count, arrived;                         // list entries; blocks that have listed theirs (few rows)
    uint64_t cum_mass[kBins];                        // of bins >= i
};

struct SampleArgs {
    const void* logits; int64_t ld; int N, parts, list_max;
    const float *uniform, *temperature; const int32_t* top_k; const float *top_p, *min_p;
    uint64_t* hist;                                  // [rows, parts, kBins] count << 50 | mass
    PartMeta* meta;                                  // [rows, parts]
    RowState* state;                                 // [rows]
    uint2* list;                                     // [rows, list_max] ordered value bits, column
    int64_t* token; float* logprob; uint32_t* flags;
};

// ---- values -------------------------------------------------------------------
template <int TYPE> constexpr int kBytes = TYPE == ORNITH_LOGITS_F32 ? 4 : 2;
// low bits of the ordered value that no logit of the type has
template <int TYPE> constexpr int kDrop = TYPE == ORNITH_LOGITS_F32 ? 0 : TYPE == ORNITH_LOGITS_BF16 ? 16 : 13;

template <int TYPE> __device__ __forceinline__ const void* row_of(const SampleArgs& a, int row) {
    return static_cast<const uint8_t*>(a.logits) + size_t(row) * size_t(a.ld) * kBytes<TYPE>;
}
// Eight consecutive columns in the type's own bits (half the registers for the 16-bit types).
// Rows start at any element: 16-byte loads of element-aligned memory.
struct __attribute__((packed, aligned(2))) Raw16 { uint32_t w[4]; };
template <int TYPE> struct Piece {
    static constexpr int kWords = TYPE == ORNITH_LOGITS_F32 ? 8 : 4;
    uint32_t w[kWords];
    __device__ __forceinline__ float operator[](int e) const {
        if constexpr (TYPE == ORNITH_LOGITS_F32) return __uint_as_float(w[e]);
        if constexpr (TYPE == ORNITH_LOGITS_BF16)
            return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
        return f16_bits_to_f32((w[e >> 1] >> (16 * (e & 1))) & 0xffffu);
    }
    // columns at or past N read as -inf
    __device__ __forceinline__ void load(const void* row, int col, int N) {
        if (col + 8 <= N) {
            const auto* p = reinterpret_cast<const Raw16*>(static_cast<const uint8_t*>(row) + size_t(col) * kBytes<TYPE>);
#pragma unroll
            for (int h = 0; h < kWords / 4; ++h) {
                const Raw16 r = p[h];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[4 * h + i] = r.w[i];
            }
        } else {
            constexpr uint32_t none = TYPE == ORNITH_LOGITS_F32 ? 0xff800000u : TYPE == ORNITH_LOGITS_BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                if constexpr (TYPE == ORNITH_LOGITS_F32) w[i] = col + i < N ? static_cast<const uint32_t*>(row)[col + i] : none;
                else {
                    const auto* h = static_cast<const uint16_t*>(row);
                    const uint32_t lo = col + 2 * i < N ? h[col + 2 * i] : none, hi = col + 2 * i + 1 < N ? h[col + 2 * i + 1] : none;
                    w[i] = lo | (hi << 16);
                }
            }
        }
    }
};

// Bits ordered as the values are (-0 as +0; never 0 for a value above -inf).
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kColMask = (1u << kColBits) - 1;
template <int TYPE> __device__ __forceinline__ uint64_t comp_of(uint32_t key, int col) {
    return (uint64_t(key >> kDrop<TYPE>) << kColBits) | (kColMask - uint32_t(col));
}
// (a negative value's dropped bits are ones)
template <int TYPE> __device__ __forceinline__ uint32_t comp_key(uint64_t comp) {
    const uint32_t k = uint32_t(comp >> kColBits) << kDrop<TYPE>;
    return k & 0x80000000u ? k : k | ((1u << kDrop<TYPE>) - 1);
}
__device__ __forceinline__ int comp_col(uint64_t comp) { return int(kColMask - (uint32_t(comp) & kColMask)); }
// comp >= threshold on values and columns
struct Cut {
    float value;
    int col;
    __device__ __forceinline__ bool keeps(float v, int c) const { return v > value || (v == value && c <= col); }
};
template <int TYPE> __device__ __forceinline__ Cut cut_of(uint64_t threshold) {
    return threshold ? Cut{unordered(comp_key<TYPE>(threshold)), comp_col(threshold)} : Cut{-__builtin_huge_valf(), 0};
}

// 2^(36 + x) for |x| <= 1/2, degree 7 (interpolation of (2^x - 1) / x at Chebyshev points; relative error
// 2^-33, 2^36 at 0; degree 8, 2^-39.7, costs 0.6 us at 64 rows of 248320; degree 6, 2^-27.6, would save 0.5).
// The coefficients are kept in scalar registers: as literals, each fma is preceded by two moves.
__device__ __forceinline__ double in_sgpr(double v) {
    asm("" : "+s"(v));
    return v;
}
__device__ __forceinline__ double exp2_units(double x) {
    double p = __builtin_fma(x, in_sgpr(0x1.00a5814f2a63cp+20), in_sgpr(0x1.443fffcaa2337p+23));
    p = __builtin_fma(p, x, in_sgpr(0x1.5d879ead1c114p+26));
    p = __builtin_fma(p, x, in_sgpr(0x1.3b2a1b7150c21p+29));
    p = __builtin_fma(p, x, in_sgpr(0x1.c6b08d883db58p+31));
    p = __builtin_fma(p, x, in_sgpr(0x1.ebfbe045f4d5cp+33));
    p = __builtin_fma(p, x, in_sgpr(0x1.62e42fefa39f0p+35));
    return __builtin_fma(p, x, in_sgpr(0x1p36));
}

// From |j| = 2^40 on, the neighbours of the largest value lie 2^16 powers of two below it: it has
// all the mass (+inf among such).  The scale (0, 0) gives it one.
constexpr double kFar = 0x1p40, kWhole = 0x1.8p52;
__device__ __forceinline__ bool is_far(double j) { return !(__builtin_fabs(j) < kFar); }
struct Scale { double c, j; };
__device__ __forceinline__ Scale scale_of(double c, double j) { return is_far(j) ? Scale{0.0, 0.0} : Scale{c, j}; }

// With the part's scale, 2^52 + the mass of a value l at or above its part's `least` and no more than
// 1000 powers of two below j (of others, anything), o = rint(l c) - j and x = l c - rint(l c).  Whole numbers come from the low word of a sum
// with 1.5 * 2^52, with one rounding of the exact product, so o + j and its eighths are the same in
// every part.
__device__ __forceinline__ double mass_sum(float v, const Scale& k, int& o, double& x) {
    const double l = double(v), m = kWhole - k.j;
    const double q = __builtin_fma(l, k.c, m);
    x = __builtin_fma(l, k.c, m - q);
    o = int(uint32_t(__double_as_longlong(q)));        // <= 0
    const uint64_t e = uint64_t(__double_as_longlong(exp2_units(x)));
    const uint32_t hi = uint32_t(e >> 32) + (uint32_t(o) << 20);
    return __longlong_as_double((int64_t(hi) << 32) | uint32_t(e)) + 0x1p52;
}
// Bin and mass of the same (bin < 0: no mass, whatever `mass` holds).
__device__ __forceinline__ int bin_mass(float v, const Scale& k, uint64_t& mass) {
    int o;
    double x;
    const uint64_t w = uint64_t(__double_as_longlong(mass_sum(fminf(v, 0x1.fffffep127f), k, o, x)));
    const int f = int(uint32_t(__double_as_longlong(__builtin_fma(x, double(kSub), in_sgpr(kWhole)))));
    uint32_t lo = uint32_t(w), hi = uint32_t(w >> 32) & 0xfffffu;
    asm volatile("" : "+v"(lo), "+v"(hi));             // (computed for every lane: no branch per value)
    mass = (uint64_t(hi) << 32) | lo;
    return o * kSub + f + kTopBin;
}
__device__ __forceinline__ int bin_alone(float v, const Scale& k) {
    const double l = double(fminf(v, 0x1.fffffep127f)), m = kWhole - k.j;
    const double q = __builtin_fma(l, k.c, m);
    const double x = __builtin_fma(l, k.c, m - q);
    const int f = int(uint32_t(__double_as_longlong(__builtin_fma(x, double(kSub), kWhole))));
    return int(uint32_t(__double_as_longlong(q))) * kSub + f + kTopBin;
}
// The bin, for the row or part with the largest value mx, of any value up to a little above it (NaN
// and -inf among them); -1: below the bins.
__device__ __forceinline__ int bin_of(float v, float mx, double c, double j) {
    if (is_far(j)) return v >= mx ? kTopBin : -1;
    const int bin = bin_alone(v, Scale{c, j});
    return double(v) * c > j - 64.0 ? max(bin, -1) : -1;
}
// A value a little below the lower edge of `bin`; never -inf.
__device__ __forceinline__ float below_bin(int bin, float mx, double inv, double j) {
    if (is_far(j)) return mx;
    const float at = float((j + (double(bin - kTopBin) - 0.5) * (1.0 / kSub)) * inv);
    return fmaxf(at - __builtin_fabsf(at) * 0x1p-20f - 0x1p-126f, -0x1.fffffep127f);
}

__device__ __forceinline__ int part_shift(double J, double j) { return J == j ? 0 : int(fmin(J - j, 64.0)); }
__device__ __forceinline__ uint64_t row_mass(uint64_t m, int shift) {
    return shift < 64 ? (m << kRowShift) >> shift : 0;
}
// u in [0, 1) as a 64-bit fraction (below 2^-40 its last bits are cut)
__device__ __forceinline__ uint64_t fraction(float u) { return uint64_t(double(u) * 0x1p64); }
// the least whole number at or above p of `mass` (p < 1), at least 1
__device__ __forceinline__ uint64_t share(float p, uint64_t mass) {
    const uint64_t f = fraction(p);
    return max(__umul64hi(f, mass) + (f * mass != 0), uint64_t(1));
}

struct Setting { float T, p, q, u; int k; bool valid, cut; double c, inv; };      // c = log2(e) / T, inv = 1 / c
__device__ __forceinline__ Setting setting(const SampleArgs& a, int row) {
    Setting s;
    s.T = a.temperature ? a.temperature[row] : 1.f;
    s.k = a.top_k ? a.top_k[row] : 0;
    s.p = a.top_p ? a.top_p[row] : 1.f;
    s.q = a.min_p ? a.min_p[row] : 0.f;
    s.u = a.uniform[row];
    // (no branch: one before the settings' loads cost 0.3 to 0.5 us a call)
    s.valid = (s.T == 0.f) | ((s.T > 0.f) & (s.T < __builtin_huge_valf()) & (s.p > 0.f) & (s.p <= 1.f) & (s.q >= 0.f) &
                              (s.q <= 1.f) & (s.u >= 0.f) & (s.u < 1.f));
    s.cut = (s.k > 0 && s.k < a.N) || s.p < 1.f || s.q > 0.f;
    s.c = s.T > 0.f ? 0x1.71547652b82fep+0 / double(s.T) : 0.0;
    s.inv = double(s.T) * 0x1.62e42fefa39efp-1;
    return s;
}

// ---- waves ----------------------------------------------------------------------
template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
    const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(v)), CTRL, ROWS, 0xF, false));
    const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(v >> 32)), CTRL, ROWS, 0xF, false));
    return (uint64_t(hi) << 32) | lo;
}
// inclusive prefix sum over the 64 lanes (wave_prefix_sum in 64 bits)
__device__ __forceinline__ uint64_t wave_prefix_u64(uint64_t v) {
    v += dpp_u64<0x111, 0xF>(v);
    v += dpp_u64<0x112, 0xF>(v);
    v += dpp_u64<0x114, 0xF>(v);
    v += dpp_u64<0x118, 0xF>(v);
    v += dpp_u64<0x142, 0xA>(v);
    v += dpp_u64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint64_t readlane_u64(uint64_t v, int lane) {
    return (uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v >> 32)), lane))) << 32) |
           uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v)), lane));
}
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) { return readlane_u64(wave_prefix_u64(v), 63); }

// The least key whose bin is at least `bin`, by the whole wave: the estimate of the bin's lower edge
// is off by less than a step of fp32, so the 64 keys around it hold it.
__device__ __forceinline__ uint32_t bin_edge(int bin, float mx, double c, double inv, double j) {
    if (is_far(j)) return ordered(mx);
    const double at = (j + (double(bin - kTopBin) - 0.5) * (1.0 / kSub)) * inv;
    const uint32_t first = max(ordered(float(at)), kMinusInf + 33) - 32, k0 = first + (threadIdx.x & 63);
    const uint64_t in = __builtin_amdgcn_ballot_w64(k0 >= ordered(__builtin_huge_valf()) ||
                                                    bin_of(unordered(k0), mx, c, j) >= bin);
    return first + (in ? uint32_t(__builtin_ctzll(in)) : 64u);
}

// ---- one part --------------------------------------------------------------------
template <int THREADS> struct PartShared {
    uint64_t hist[kBins];
    uint32_t count[kBins];                            // of thread maxima
    uint32_t key[THREADS / 64];
    int arg[THREADS / 64];
    uint64_t mass[THREADS / 64];
    float queue[THREADS / 64][kQueue];
};

// Histogram (cut rows), whole mass (others) or first maximum (greedy) of the values that the
// block's threads hold, eight consecutive columns a piece.  The histogram is complete after the
// caller's next barrier; of a cut row, it lacks values that no cut can keep.
template <int TYPE, int THREADS, int PIECES>
__device__ __forceinline__ PartMeta part_pass(const SampleArgs& a, const Setting& s, const Piece<TYPE> (&v)[PIECES],
                                              int col0, PartShared<THREADS>& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    constexpr int W = THREADS / 64;
    for (int i = tid; i < kBins; i += THREADS) {
        sh.hist[i] = 0;
        sh.count[i] = 0;
    }
    float mx = -__builtin_huge_valf();
    bool nan = false;
#pragma unroll
    for (int u = 0; u < PIECES; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            nan |= v[u][e] != v[u][e];
            mx = fmaxf(mx, v[u][e]);
        }
    if (__builtin_amdgcn_ballot_w64(nan) && lane == 0) flag_or(a.flags, kSampleNan);
    const uint32_t wkey = wave_max_u(ordered(mx));
    if (lane == 0) sh.key[wv] = wkey;
    __syncthreads();
    uint32_t key = sh.key[0];
#pragma unroll
    for (int w = 1; w < W; ++w) key = max(key, sh.key[w]);
    if (key <= kMinusInf || !s.valid) return PartMeta{-__builtin_huge_val(), 0, 0, 0, 0.f};
    if (s.T == 0.f) {                                 // greedy: the first column of the largest value
        int arg = 0x7fffffff;
#pragma unroll
        for (int u = PIECES - 1; u >= 0; --u)
#pragma unroll
            for (int e = 7; e >= 0; --e)
                if (v[u][e] == v[u][e] && ordered(v[u][e]) == key) arg = col0 + 8 * THREADS * u + e;
        arg = wave_min_i(arg);
        if (lane == 0) sh.arg[wv] = arg;
        __syncthreads();
        arg = sh.arg[0];
#pragma unroll
        for (int w = 1; w < W; ++w) arg = min(arg, sh.arg[w]);
        return PartMeta{0.0, 0, key, arg, 0.f};
    }
    const float part_mx = unordered(key);
    const double j = __builtin_ceil(double(part_mx) * s.c);
    const Scale k = scale_of(s.c, j);
    float least = below_bin(0, part_mx, s.inv, j);
    if (!s.cut) {
        uint64_t sum;
        if (is_far(j)) {
            int count = 0;
#pragma unroll
            for (int u = 0; u < PIECES; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) count += v[u][e] >= least;
            sum = uint64_t(count) * kPartOne;
        } else {
            // The bits of 2^52 + mass are those of 2^52, plus the mass.  From `least` down masses are 0, so
            // values (NaN too) are clamped to it; but not where it was cut off at the lowest fp32 (values
            // below must not count), nor where it lies so far down (it keeps 2^-20 of |j| from the bins)
            // that its octave leaves the exponent field: there the bins decide, as for cut rows.
            constexpr float kMost = 0x1.fffffep127f;
            if (least > -kMost && double(least) * s.c > j - 1000.0) {
                sum = -uint64_t(__double_as_longlong(0x1p52)) * uint64_t(8 * PIECES);
#pragma unroll
                for (int u = 0; u < PIECES; ++u)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        int o;
                        double x;
                        sum += uint64_t(__double_as_longlong(mass_sum(__builtin_amdgcn_fmed3f(v[u][e], least, kMost), k, o, x)));
                    }
            } else {
                sum = 0;
#pragma unroll
                for (int u = 0; u < PIECES; ++u)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        uint64_t m;
                        const int bin = bin_mass(v[u][e], k, m);
                        sum += bin >= 0 && v[u][e] >= least ? m : 0;
                    }
            }
        }
        sum = wave_sum_u64(sum);
        if (lane == 0) sh.mass[wv] = sum;
        __syncthreads();
        sum = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) sum += sh.mass[w];
        return PartMeta{j, sum, key, 0, least};
    }
    // Values that take part in no cut are left out: those below the bins, and with a small top_k
    // those below the bin that holds the k-th largest of the threads' maxima (k values of this
    // part alone lie in or above it).
    if (s.k > 0 && s.k <= kMaximaK && THREADS >= kMaximaK) {
        const int b = bin_alone(mx, k);
        if (b >= 0 && mx >= least) atomicAdd(&sh.count[b], 1u);
        __syncthreads();
        constexpr int per = (kTopBin + 64) / 64;
        uint32_t c[per], sum = 0;
#pragma unroll
        for (int e = 0; e < per; ++e) {
            const int i = kTopBin - (per * lane + e);
            c[e] = i >= 0 ? sh.count[i] : 0;
            sum += c[e];
        }
        uint32_t run = uint32_t(wave_prefix_sum(int(sum))) - sum;
        int found = 0;
#pragma unroll
        for (int e = 0; e < per; ++e) {
            if (run < uint32_t(s.k) && run + c[e] >= uint32_t(s.k)) found = kTopBin - (per * lane + e);
            run += c[e];
        }
        least = below_bin(int(wave_max_u(uint32_t(found))), part_mx, s.inv, j);
    }
    auto add = [&](float x) {
        uint64_t m;
        const int bin = bin_mass(x, k, m);
        if (bin >= 0) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[bin]),
                                (unsigned long long)(m + (uint64_t(1) << kMassBits)));
    };
    int left = 0;
#pragma unroll
    for (int u = 0; u < PIECES; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) left += __popcll(__builtin_amdgcn_ballot_w64(v[u][e] >= least));
    if (left <= min(kQueue, PIECES * 8 * 64 / 2)) {   // few: side by side first
        float* queue = sh.queue[wv];
        int at = 0;
#pragma unroll
        for (int u = 0; u < PIECES; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint64_t b = __builtin_amdgcn_ballot_w64(v[u][e] >= least);
                if (v[u][e] >= least) queue[at + __builtin_amdgcn_mbcnt_hi(uint32_t(b >> 32),
                                                 __builtin_amdgcn_mbcnt_lo(uint32_t(b), 0))] = v[u][e];
                at += __popcll(b);
            }
        for (int i = lane; i < left; i += 64) add(queue[i]);
    } else {
#pragma unroll
        for (int u = 0; u < PIECES; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (v[u][e] >= least) add(v[u][e]);
    }
    return PartMeta{j, 0, key, 0, least};
}

// A block per part, the values in registers, loaded once.  256 threads (four pieces each) where parts are
// many: 64 rows of 248320 bf16 16.7 us, where 512 and 1024 threads were slower (in an earlier form of the
// masses 22 / 24 / 30 us: more waves meet at each barrier).  1024 where every part has a CU of its own and the
// chain of one thread counts: 8 rows of 151936 fp32 5.6 us, with 256 threads 8.0.  Tried and slower: blocks
// that stay and load a part ahead (27 us against 22), 64 VGPRs a thread forced by launch bounds (spills).
template <int TYPE, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_parts_kernel(SampleArgs a, int row0) {
    const int part = blockIdx.x, slot = blockIdx.y, row = row0 + slot, tid = threadIdx.x;
    __shared__ PartShared<THREADS> sh;
    constexpr int kPieces = kPart / 8 / THREADS;
    const void* src = row_of<TYPE>(a, row);
    const int col0 = part * kPart + tid * 8;
    Piece<TYPE> v[kPieces];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) v[u].load(src, col0 + 8 * THREADS * u, a.N);
    const Setting s = setting(a, row);
    const PartMeta m = part_pass<TYPE, THREADS, kPieces>(a, s, v, col0, sh);
    __syncthreads();
    const size_t at = size_t(slot) * a.parts + part;
    if (tid == 0) {
        a.meta[at] = m;
        if (part == 0) a.state[slot].count = a.state[slot].arrived = 0;
    }
    if (m.key && s.cut && s.T != 0.f)
        for (int i = tid; i < kBins; i += THREADS) a.hist[at * kBins + i] = sh.hist[i];
}

// ---- the row ------------------------------------------------------------------------
struct RowShared {
    uint64_t cm[kBins];                               // mass and
    uint32_t cc[kBins];                               // count of bins >= i
    uint64_t part_mass[kPartsMax];
    Scale scale[kPartsMax];
    int shift[kPartsMax];
    float least[kPartsMax];
    uint64_t wave_mass[kRowWaves];
    uint32_t wave_count[kRowWaves];
    uint64_t lo, hi, rest, total;
    int bin[3], part;                                 // bin_k; top-p's highest and lowest
    uint32_t qkey, edge[6];
    Plan plan;
};

// What the parts of a row with the given J add to it: scale, shift, least.  (Where J is far, every
// part that adds anything has that j.)
__device__ __forceinline__ void set_part(int p, const PartMeta& m, double c, int shift, RowShared& sh) {
    sh.scale[p] = scale_of(c, m.j);
    sh.shift[p] = shift;
    sh.least[p] = m.least;
}
// Sums of the waves before this one, and of all, from every wave's own (in LDS, after a barrier).
__device__ __forceinline__ uint64_t waves_before(const uint64_t (&w)[kRowWaves], uint64_t& all) {
    const int lane = threadIdx.x & 63;
    const uint64_t own = lane < kRowWaves ? w[lane] : 0, run = wave_prefix_u64(own);
    all = readlane_u64(run, kRowWaves - 1);
    return readlane_u64(run - own, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}
__device__ __forceinline__ uint32_t waves_before(const uint32_t (&w)[kRowWaves], uint32_t& all) {
    const int lane = threadIdx.x & 63;
    const int own = lane < kRowWaves ? int(w[lane]) : 0, run = wave_prefix_sum(own);
    all = uint32_t(__builtin_amdgcn_readlane(run, kRowWaves - 1));
    return uint32_t(__builtin_amdgcn_readlane(run - own, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)));
}
// Thread i <= kTopBin holds bin kTopBin - i's mass and count: cm and cc (after the barriers in it).
__device__ __forceinline__ void cumulate(uint64_t mass, uint32_t count, RowShared& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    constexpr int W = (kTopBin + 64) / 64;
    if (wv < W) {
        mass = wave_prefix_u64(mass);
        count = uint32_t(wave_prefix_sum(int(count)));
        if (lane == 63) {
            sh.wave_mass[wv] = mass;
            sh.wave_count[wv] = count;
        }
    }
    if (tid == 0) {
        sh.bin[0] = sh.bin[1] = sh.bin[2] = -1;
        sh.qkey = kMinusInf + 1;
        sh.part = -1;
    }
    __syncthreads();
    if (wv < W) {
        uint64_t mass_all;
        uint32_t count_all;
        mass += waves_before(sh.wave_mass, mass_all);
        count += waves_before(sh.wave_count, count_all);
        if (tid <= kTopBin) {
            sh.cm[kTopBin - tid] = mass;
            sh.cc[kTopBin - tid] = count;
        }
    }
    __syncthreads();
}

// The borders of a cut row from cm and cc: sh.plan (after its last barrier).
__device__ __forceinline__ void borders(const SampleArgs& a, const Setting& s, float mx, double J, int list_max,
                                        RowShared& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const uint64_t* cm = sh.cm;
    const uint32_t* cc = sh.cc;
    const bool use_k = s.k > 0 && s.k < a.N && cc[0] >= uint32_t(s.k), use_p = s.p < 1.f, use_q = s.q > 0.f;
    // the bin that holds the k-th value, and the range of the mass of the first k
    if (tid <= kTopBin) {
        const uint64_t next = tid == kTopBin ? 0 : cm[tid + 1];
        const uint32_t before = tid == kTopBin ? 0 : cc[tid + 1];
        if (use_k) {
            if (cc[tid] >= uint32_t(s.k) && before < uint32_t(s.k)) {
                sh.bin[0] = tid;
                sh.hi = cm[tid];
                sh.lo = cc[tid] == uint32_t(s.k) ? cm[tid] : next;
            }
        } else if (tid == 0) sh.hi = sh.lo = cm[0];
    }
    // min-p's least value: mostly among the 64 keys around the estimate mx + T ln q.  Where those two nearly
    // cancel, the estimate is off by many steps of the small fp32 numbers there: then all 64 keys pass, or
    // none, and the rest on that side is searched, 64 keys a round (the largest value passes).
    if (use_q && wv == kRowWaves - 1) {
        const uint32_t top = ordered(mx);
        const double least_t = log2(double(s.q));
        const float at = float(double(mx) + double(s.T) * log(double(s.q)));
        const uint32_t mid = at == at ? ordered(at) : kMinusInf + 1;
        auto passing = [&](uint32_t key) {
            const float v = unordered(key);
            return __builtin_amdgcn_ballot_w64(key >= top || v == mx || (double(v) - double(mx)) * s.c >= least_t);
        };
        uint32_t lo = kMinusInf + 1, hi = top;         // the least that passes lies in [lo, hi]
        const uint32_t first = max(min(mid, top), kMinusInf + 33) - 32;
        const uint64_t near = passing(first + lane);
        const uint32_t from = first + (near ? uint32_t(__builtin_ctzll(near)) : 64u);
        if (near) hi = min(from, top);
        if (from > first) lo = min(from, top);
        while (lo < hi) {
            const uint32_t step = (hi - lo + 63) / 64;
            const uint64_t b = passing(min(lo + step * lane, hi));
            const uint32_t i = b ? uint32_t(__builtin_ctzll(b)) : 64u;
            if (b) hi = min(lo + step * i, hi);
            if (i) lo = min(lo + step * (i - 1) + 1, hi);
        }
        if (lane == 0) sh.qkey = hi;
    }
    __syncthreads();
    // the bins that top-p's border can lie in
    if (use_p && tid <= kTopBin) {
        const uint64_t f = fraction(s.p);
        const uint64_t lo = max(__umul64hi(f, sh.lo), uint64_t(1)), hi = __umul64hi(f, sh.hi) + 1;
        const uint64_t next = tid == kTopBin ? 0 : cm[tid + 1];
        if (cm[tid] >= lo && next < lo) sh.bin[1] = tid;
        if ((cm[tid] >= hi || tid == 0) && next < hi) sh.bin[2] = tid;
    }
    __syncthreads();
    const int bk = sh.bin[0], p_hi = use_p ? sh.bin[1] : -1, p_lo = use_p ? sh.bin[2] : -1;
    const int bq = use_q ? bin_of(unordered(sh.qkey), mx, s.c, J) : -1;
    const bool q_alone = bq > max(bk, p_hi);          // min-p's border lies above the others' bins
    const bool q_in = bq >= 0 && bq >= max(bk, p_lo);
    int lo[3] = {q_alone ? -1 : bk, q_alone ? -1 : p_lo, q_in ? bq : -1}, hi[3] = {lo[0], q_alone ? -1 : p_hi, lo[2]};
    int least = kTopBin + 1;
    uint32_t entries = 0;
#pragma unroll
    for (int r = 0; r < 3; ++r)
        if (lo[r] >= 0) {
            least = min(least, lo[r]);
            entries += cc[lo[r]] - (hi[r] == kTopBin ? 0 : cc[hi[r] + 1]);
        }
    const bool none = least > kTopBin;                // every border lies below the bins
    const bool small = !none && cc[least] <= uint32_t(kSmall);
    if (small) {
        lo[0] = least;
        hi[0] = kTopBin;
        lo[1] = lo[2] = -1;
    }
    if (wv < 6) {
        const int r = wv >> 1, b = wv & 1 ? hi[r] + 1 : lo[r];
        const uint32_t edge = lo[r] < 0 || b > kTopBin ? kKeyEnd : bin_edge(b, mx, s.c, s.inv, J);
        if (lane == 0) sh.edge[wv] = edge;
    }
    __syncthreads();
    if (tid == 0) {
        Plan& p = sh.plan;
        p.J = J;
        p.mx = mx;
        p.threshold_q = 0;
        p.total = cm[0];
        p.mode = small ? kModeSmall : entries <= uint32_t(list_max) ? kModeList : kModeWalk;
        p.use_k = use_k && !q_alone;
        p.use_p = use_p && !q_alone;
        p.bin_k = bk;
        p.bin_q = bq;
        p.above_count = bk < 0 || bk == kTopBin ? 0 : int(cc[bk + 1]);
        p.above_mass = bk < 0 || bk == kTopBin ? 0 : cm[bk + 1];
#pragma unroll
        for (int r = 0; r < 3; ++r) {
            p.bin_lo[r] = lo[r];
            p.bin_hi[r] = hi[r];
            p.lo[r] = sh.edge[2 * r];
            p.hi[r] = sh.edge[2 * r + 1];
        }
    }
    __syncthreads();
}
// The key range of one bin into sh.edge[0 .. 1] (after the barrier in it); mostly a range of the plan.
__device__ __forceinline__ void bin_range(int bin, const Setting& s, const Plan& plan, RowShared& sh) {
    const int tid = threadIdx.x, wv = tid >> 6;
    int at = -1;
#pragma unroll
    for (int r = 0; r < 3; ++r)
        if (plan.bin_lo[r] == bin && plan.bin_hi[r] == bin) at = r;
    if (at >= 0) {
        if (tid == 0) {
            sh.edge[0] = plan.lo[at];
            sh.edge[1] = plan.hi[at];
        }
    } else if (wv < 2) {
        const uint32_t edge = bin < 0 || bin + wv > kTopBin ? kKeyEnd : bin_edge(bin + wv, plan.mx, s.c, s.inv, plan.J);
        if ((tid & 63) == 0) sh.edge[wv] = edge;
    }
    __syncthreads();
}
template <int TYPE> __device__ __forceinline__ uint64_t q_threshold(uint32_t qkey) {
    const uint32_t up = qkey & 0x80000000u ? (1u << kDrop<TYPE>) - 1 : 0;     // to a value of the type
    return uint64_t((qkey + up) >> kDrop<TYPE>) << kColBits;
}
__device__ __forceinline__ bool in_ranges(const Plan& p, uint32_t key) {
    return key - p.lo[0] < p.hi[0] - p.lo[0] || key - p.lo[1] < p.hi[1] - p.lo[1] || key - p.lo[2] < p.hi[2] - p.lo[2];
}

__device__ __forceinline__ void give(const SampleArgs& a, int row, int token, float logprob) {
    a.token[row] = token;
    if (a.logprob) a.logprob[row] = logprob;
}
// ln of mass(v) / total; 0 where the token is all there is
__device__ __forceinline__ float log_share(float v, const Setting& s, double J, uint64_t mass, uint64_t total) {
    if (mass == total) return 0.f;
    const double up = is_far(J) ? 0.0 : __builtin_fma(double(v), s.c, -J);
    return float(up * 0x1.62e42fefa39efp-1 - log(double(total) * 0x1p-42));
}

// part_mass holds the kept mass of every part (after a barrier): sh.part, sh.rest (what is left of
// u S there) and sh.total.
__device__ __forceinline__ void draw_part(int parts, const Setting& s, RowShared& sh) {
    const int tid = threadIdx.x;
    if (tid < 64) {
        uint64_t m[kPartsMax / 64], run[kPartsMax / 64], total = 0;
#pragma unroll
        for (int h = 0; h < kPartsMax / 64; ++h) {
            const int p = h * 64 + tid;
            m[h] = p < parts ? sh.part_mass[p] : 0;
            run[h] = wave_prefix_u64(m[h]) + total;
            total = readlane_u64(run[h], 63);
        }
        const uint64_t target = __umul64hi(fraction(s.u), total);      // token: the first column past it
        if (tid == 0) {
            sh.total = total;
            sh.part = -1;
        }
#pragma unroll
        for (int h = 0; h < kPartsMax / 64; ++h)
            if (run[h] > target && run[h] - m[h] <= target) {
                sh.part = h * 64 + tid;
                sh.rest = target - (run[h] - m[h]);
            }
    }
    __syncthreads();
}
// The token inside the part: thread i holds its columns col0 .. col0 + 7, ascending over the block.
// Unless most of the part is kept, the kept values are set side by side in LDS first: fewer masses a thread.
struct DrawShared { float val[kPart]; uint16_t col[kPart]; };
template <int TYPE, bool CUT>
__device__ __forceinline__ void draw_column(const SampleArgs& a, int row, const Setting& s, double J, const Scale& k,
                                            float least, int shift, uint64_t threshold, const Piece<TYPE>& v, int col0,
                                            RowShared& sh, DrawShared& ds) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const uint64_t rest = sh.rest, total = sh.total;
    const Cut cut = cut_of<TYPE>(threshold);
    uint32_t keep = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) keep |= uint32_t(v[e] >= least && (!CUT || cut.keeps(v[e], col0 + e))) << e;
    const uint32_t own = uint32_t(__popc(keep));
    uint32_t at = uint32_t(wave_prefix_sum(int(own))), kept;
    if (lane == 63) sh.wave_count[wv] = at;
    __syncthreads();
    at += waves_before(sh.wave_count, kept) - own;
    auto mass_of = [&](float x) -> uint64_t {
        uint64_t m;
        return bin_mass(x, k, m) >= 0 ? m : 0;
    };
    // sums up to and including a thread's
    auto upto = [&](uint64_t sum) -> uint64_t {
        const uint64_t run = wave_prefix_u64(sum);
        if (lane == 63) sh.wave_mass[wv] = run;
        __syncthreads();
        uint64_t all;
        const uint64_t before = waves_before(sh.wave_mass, all);
        // (logits that changed under the call: no column is past u S)
        if (tid == 0 && row_mass(all, shift) <= rest) give(a, row, -1, __builtin_nanf(""));
        return run + before;
    };
    const int per = int(kept + kRowThreads - 1) / kRowThreads;
    if (per <= kPer / 2) {
#pragma unroll
        for (int e = 0; e < kPer; ++e)
            if (keep >> e & 1) {
                ds.val[at] = v[e];
                ds.col[at] = uint16_t(tid * kPer + e);
                ++at;
            }
        __syncthreads();
        const int i0 = tid * per, i1 = min(i0 + per, int(kept));
        uint64_t sum = 0;
        for (int i = i0; i < i1; ++i) sum += mass_of(ds.val[i]);
        const uint64_t run = upto(sum);
        if (row_mass(run, shift) > rest && row_mass(run - sum, shift) <= rest) {
            uint64_t before = run - sum;
            for (int i = i0; i < i1; ++i) {
                const uint64_t m = mass_of(ds.val[i]);
                before += m;
                if (row_mass(before, shift) > rest) {
                    give(a, row, col0 - tid * kPer + ds.col[i], log_share(ds.val[i], s, J, row_mass(m, shift), total));
                    break;
                }
            }
        }
        return;
    }
    uint64_t m[kPer], sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        m[e] = keep >> e & 1 ? mass_of(v[e]) : 0;
        sum += m[e];
    }
    const uint64_t run = upto(sum);
    if (row_mass(run, shift) > rest && row_mass(run - sum, shift) <= rest) {
        uint64_t before = run - sum, mass = 0;
        int col = -1;
        float val = 0.f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            before += m[e];
            if (col < 0 && row_mass(before, shift) > rest) {
                col = col0 + e;
                val = v[e];
                mass = m[e];
            }
        }
        give(a, row, col, log_share(val, s, J, row_mass(mass, shift), total));
    }
}

// A list of every candidate (n <= kSmall, zeros past n): each entry's rank by value and by column
// (four threads an entry), then one wave walks both orders, four entries a lane.
struct SmallList {
    uint64_t comp[kSmall], mass[kSmall], by_value[kSmall], by_column[kSmall];
    float val[kSmall];
    uint32_t at[kSmall];                              // of a column rank: value rank << 8 | entry
};
__device__ __forceinline__ void finish_small(const SampleArgs& a, int row, const Setting& s, const Plan& plan, int n,
                                             uint64_t threshold, SmallList& sl) {
    const int tid = threadIdx.x, e = tid >> 2;
    __syncthreads();
    const int end = (n + 31) & ~31;
    if ((tid & ~63) < 4 * end) {                      // (whole waves)
        const uint64_t comp = sl.comp[e];
        const uint32_t col = uint32_t(comp) & kColMask;
        uint32_t by_value = 0, by_column = 0;
#pragma unroll 8
        for (int i = tid & 3; i < end; i += 4) {
            const uint64_t c = sl.comp[i];
            by_value += c > comp;
            by_column += (uint32_t(c) & kColMask) > col;      // (complements: lower columns)
        }
        by_value += uint32_t(dpp_i<kDppXor1>(int(by_value)));
        by_value += uint32_t(dpp_i<kDppXor2>(int(by_value)));
        by_column += uint32_t(dpp_i<kDppXor1>(int(by_column)));
        by_column += uint32_t(dpp_i<kDppXor2>(int(by_column)));
        if (e < n && (tid & 3) == 0) {
            const uint64_t mass = sl.mass[e];
            sl.by_value[by_value] = mass;
            sl.by_column[by_column] = mass;
            sl.at[by_column] = by_value << 8 | uint32_t(e);
        }
    }
    __syncthreads();
    if (tid >= 64) return;
    constexpr int per = kSmall / 64;
    static_assert(kSmall == 256, "four entries a lane, eight bits an entry");
    uint64_t m[per], sum = 0;
    auto walk = [&](auto&& mass_of) {                 // m[i]: sums up to entry per * tid + i
        sum = 0;
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int r = per * tid + i;
            sum += r < n ? mass_of(r, i) : 0;
            m[i] = sum;
        }
        const uint64_t before = wave_prefix_u64(sum) - sum;
#pragma unroll
        for (int i = 0; i < per; ++i) m[i] += before;
    };
    walk([&](int r, int) { return sl.by_value[r]; });
    // how many the cuts keep
    int keep = n;
    uint64_t of = plan.total;
    if (plan.use_k) {
        keep = min(keep, s.k);
        const int lane = (keep - 1) / per, i = (keep - 1) % per;
        const uint64_t at = i == 0 ? m[0] : i == 1 ? m[1] : i == 2 ? m[2] : m[3];
        of = readlane_u64(at, __builtin_amdgcn_readfirstlane(lane));
    }
    if (plan.use_p) {
        // (the entries can sum to a few units less than their bins, which are cut once per part: then all stay)
        const uint64_t target = share(s.p, of);
        int below = 0;
#pragma unroll
        for (int i = 0; i < per; ++i) below += __popcll(__builtin_amdgcn_ballot_w64(per * tid + i < n && m[i] < target));
        keep = min(keep, below + 1);
    }
    if (threshold) {
        int above = 0;
#pragma unroll
        for (int i = 0; i < per; ++i)
            above += __popcll(__builtin_amdgcn_ballot_w64(per * tid + i < n && sl.comp[per * tid + i] >= threshold));
        keep = min(keep, above);
    }
    uint64_t col_mass[per];
    uint32_t col_at[per];
#pragma unroll
    for (int i = 0; i < per; ++i) {
        col_at[i] = sl.at[per * tid + i];
        col_mass[i] = per * tid + i < n && col_at[i] >> 8 < uint32_t(keep) ? sl.by_column[per * tid + i] : 0;
    }
    walk([&](int, int i) { return col_mass[i]; });
    const uint64_t total = readlane_u64(m[per - 1], 63), target = __umul64hi(fraction(s.u), total);
    if (tid == 0 && !total) give(a, row, -1, __builtin_nanf(""));      // (logits that changed under the call)
#pragma unroll
    for (int i = 0; i < per; ++i) {
        if (per * tid + i < n && m[i] > target && m[i] - col_mass[i] <= target) {
            const int x = int(col_at[i] & 255u);
            give(a, row, comp_col(sl.comp[x]), log_share(sl.val[x], s, plan.J, col_mass[i], total));
        }
    }
}

// Descent to a border inside one bin's key range: the entry at which, from the largest down, `need`
// is reached - a count, or a mass.  each(f) runs f(comp, row mass) over the entries of the range
// [lo, hi) of keys, spread over the block.  A round counts the entries by the next eight bits of
// comp - base; 64 or fewer are ranked, four threads an entry.
struct Descent {
    uint32_t count[256];
    unsigned long long mass[256];
    uint64_t comp[64], m[64];
    uint64_t wave_mass[kRowWaves];
    uint32_t wave_count[kRowWaves];
    uint64_t need, above, found;
    uint32_t digit, group, n;
};
template <int TYPE, class Each>
__device__ __forceinline__ void descend(uint32_t lo, uint32_t hi, bool by_mass, uint64_t need, uint32_t group, Each&& each, Descent& d) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    uint64_t base = uint64_t(lo >> kDrop<TYPE>) << kColBits;
    uint64_t span = (uint64_t(((hi - 1) >> kDrop<TYPE>) + 1) << kColBits) - base;   // comps lie in [base, base + span)
    uint64_t above = 0;
    while (true) {                                    // group: entries left, or more
        const int bits = 64 - __builtin_clzll(span - 1 | 1);
        const int sft = bits > 8 ? bits - 8 : 0;
        __syncthreads();
        if (tid < 256) {
            d.count[tid] = 0;
            d.mass[tid] = 0;
            if (tid < 64) {
                d.comp[tid] = 0;
                d.m[tid] = 0;
            }
        }
        if (tid == 0) {
            d.n = 0;
            d.group = 0;
            d.found = 0;
        }
        __syncthreads();
        if (group <= 64) break;
        each([&](uint64_t comp, uint64_t m) {
            if (comp - base >= span) return;
            const uint32_t i = uint32_t((comp - base) >> sft);
            atomicAdd(&d.count[i], 1u);
            atomicAdd(&d.mass[i], (unsigned long long)m);
        });
        __syncthreads();
        // thread i < 256: digit 255 - i
        uint32_t c = 0, cr = 0;
        uint64_t m = 0, mr = 0;
        if (wv < 4) {
            c = d.count[255 - tid];
            m = d.mass[255 - tid];
            cr = uint32_t(wave_prefix_sum(int(c)));
            mr = wave_prefix_u64(m);
            if (lane == 63) {
                d.wave_count[wv] = cr;
                d.wave_mass[wv] = mr;
            }
        }
        __syncthreads();
        if (wv < 4) {
            uint32_t call = 0;
            uint64_t mall = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t cw = d.wave_count[w];
                const uint64_t mw = d.wave_mass[w];
                cr += w < wv ? cw : 0;
                mr += w < wv ? mw : 0;
                call += cw;
                mall += mw;
            }
            // the entries can sum to a few units less than their bin (cut once per part): then the last is the border
            const bool short_of = by_mass ? mall < need : call < need;
            const uint64_t b0 = by_mass ? mr - m : cr - c, b1 = by_mass ? mr : cr;
            if (c && (short_of ? cr == call : b0 < need && b1 >= need)) {
                d.digit = uint32_t(255 - tid);
                d.group = c;
                d.need = short_of ? ~uint64_t(0) : need - b0;
                d.above = above + (mr - m);
            }
        }
        __syncthreads();
        group = d.group;
        if (group == 0) break;                        // nothing in the range
        need = d.need;
        above = d.above;
        base += uint64_t(d.digit) << sft;
        span = uint64_t(1) << sft;
    }
    if (group == 0) {
        if (tid == 0) d.above = 0;
        __syncthreads();
        return;
    }
    each([&](uint64_t comp, uint64_t m) {
        if (comp - base >= span) return;
        const uint32_t i = atomicAdd(&d.n, 1u);
        if (i < 64) {
            d.comp[i] = comp;
            d.m[i] = m;
        }
    });
    __syncthreads();
    const int n = min(int(d.n), 64);
    if (tid < 256) {                                  // (zeros past n)
        const int e = tid >> 2;
        const uint64_t comp = d.comp[e], m = d.m[e];
        uint32_t count = 0;
        uint64_t before = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint64_t ci = d.comp[4 * i + (tid & 3)], mi = d.m[4 * i + (tid & 3)];
            count += ci > comp;
            before += ci > comp ? mi : 0;
        }
        count += uint32_t(dpp_i<kDppXor1>(int(count)));
        count += uint32_t(dpp_i<kDppXor2>(int(count)));
        before += dpp_u64<kDppXor1, 0xF>(before);
        before += dpp_u64<kDppXor2, 0xF>(before);
        // (short of `need` again: the last)
        const bool at = by_mass ? before < need && (before + m >= need || count + 1 == uint32_t(n)) : count + 1 == min(need, uint64_t(n));
        if (e < n && at) {
            d.found = comp;
            d.above = above + before + m;
        }
    }
    __syncthreads();
}

// Threshold of a row in list (or walk) mode.  group: the entries of all ranges, or more; bf: the bin it
// lies in (-1: below the bins).
template <int TYPE, class Each>
__device__ __forceinline__ uint64_t threshold_of(const Setting& s, const Plan& plan, const uint64_t* cm, uint64_t threshold,
                                                 uint32_t group, Each&& each, Descent& d, RowShared& sh, int& bf) {
    const int tid = threadIdx.x;
    bf = threshold ? plan.bin_q : -1;
    uint64_t of = plan.total;
    if (plan.use_k) {
        descend<TYPE>(plan.lo[0], plan.hi[0], false, uint64_t(s.k) - uint64_t(plan.above_count), group,
                      [&](auto&& f) { each(plan.lo[0], plan.hi[0], f); }, d);
        if (d.found > threshold) {
            threshold = d.found;
            bf = plan.bin_k;
        }
        of = plan.above_mass + d.above;
    }
    if (plan.use_p) {
        const uint64_t target = share(s.p, of);
        int b = plan.bin_hi[1];
        uint32_t lo = plan.lo[1], hi = plan.hi[1];
        const uint64_t above = b == kTopBin ? 0 : cm[b + 1];
        uint64_t need = target > above ? target - above : 1;      // (the first k can sum to a few units less than their bins)
        if (plan.bin_lo[1] != b) {                    // one of several bins
            __syncthreads();
            if (tid == 0) sh.bin[0] = 0;
            __syncthreads();
            if (tid <= kTopBin) {
                const uint64_t next = tid == kTopBin ? 0 : cm[tid + 1];
                if (cm[tid] >= target && next < target) {
                    sh.bin[0] = tid;
                    sh.lo = target - next;
                }
            }
            __syncthreads();
            b = sh.bin[0];
            need = sh.lo;
            bin_range(b, s, plan, sh);
            lo = sh.edge[0];
            hi = sh.edge[1];
        }
        descend<TYPE>(lo, hi, true, need, group, [&](auto&& f) { each(lo, hi, f); }, d);
        if (d.found > threshold) {
            threshold = d.found;
            bf = b;
        }
    }
    __syncthreads();
    return threshold;
}

// The row's plan in sh.plan, with sh.cm, scale, shift and least; or, of a row that needs none (greedy,
// empty, refused, without a cut), its token (given by the block with `lead`) and false.
struct PlanShared { uint64_t mass[2][kTopBin + 24]; uint32_t count[2][kTopBin + 24]; };
template <int TYPE>
__device__ __forceinline__ bool plan_row(const SampleArgs& a, int slot, int row, const Setting& s, bool lead, RowShared& sh,
                                         PlanShared& ps, DrawShared& ds) {
    const int tid = threadIdx.x, lane = tid & 63;
    const PartMeta* meta = a.meta + size_t(slot) * a.parts;
    // the parts, a lane each (every wave for itself), and the row's largest value
    PartMeta part[kPartsMax / 64];
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < kPartsMax / 64; ++h) {
        const int p = h * 64 + lane;
        part[h] = meta[min(p, a.parts - 1)];
    }
#pragma unroll
    for (int h = 0; h < kPartsMax / 64; ++h) {        // (all of it loaded here, not where it is used)
        asm volatile("" : "+v"(part[h].j), "+v"(part[h].mass), "+v"(part[h].key), "+v"(part[h].arg), "+v"(part[h].least));
        if (h * 64 + lane >= a.parts) part[h].key = 0;
        top = max(top, wave_max_u(part[h].key));
    }
    if (!s.valid || top == 0 || s.T == 0.f) {
        int first = 0;
#pragma unroll
        for (int h = kPartsMax / 64 - 1; h >= 0; --h) {
            const uint64_t at = __builtin_amdgcn_ballot_w64(part[h].key == top);
            if (at) first = h * 64 + __builtin_ctzll(at);
        }
        if (lead && tid == 0) {
            const bool fine = s.valid && top != 0;
            give(a, row, fine ? meta[first].arg : -1, fine ? 0.f : __builtin_nanf(""));
            flag_or(a.flags, !s.valid ? kSampleSetting : top == 0 ? kSampleEmpty : 0u);
        }
        return false;
    }
    if (!s.cut && !lead) return false;
    const float mx = unordered(top);
    const double J = __builtin_ceil(double(mx) * s.c);
    int shift[kPartsMax / 64];
#pragma unroll
    for (int h = 0; h < kPartsMax / 64; ++h) {
        const int p = h * 64 + lane;
        shift[h] = part[h].key ? part_shift(J, part[h].j) : 64;
        if (tid < 64 && p < a.parts) {
            set_part(p, part[h], s.c, shift[h], sh);
            sh.part_mass[p] = row_mass(part[h].mass, shift[h]);
        }
    }
    if (!s.cut) {
        __syncthreads();
        draw_part(a.parts, s, sh);
        const int in = sh.part;
        if (in < 0) {                                 // (logits that changed under the call)
            if (tid == 0) give(a, row, -1, __builtin_nanf(""));
            return false;
        }
        Piece<TYPE> v;
        const int col0 = in * kPart + tid * kPer;
        v.load(row_of<TYPE>(a, row), col0, a.N);
        draw_column<TYPE, false>(a, row, s, J, sh.scale[in], sh.least[in], sh.shift[in], 0, v, col0, sh, ds);
        return false;
    }
    // the parts' bins: three groups of threads, a third of the parts each
    constexpr int kGroup = kTopBin + 24;
    static_assert(kGroup % 64 == 0, "a wave lies in one group");
    const int g = __builtin_amdgcn_readfirstlane(tid / kGroup), i = tid - g * kGroup, bin = kTopBin - i;
    uint64_t mass = 0;
    uint32_t count = 0;
    if (g < 3) {
        const uint64_t* hist = a.hist + size_t(slot) * a.parts * kBins;
        constexpr int U = 11;                         // (33 parts' loads in flight at once)
        for (int p0 = g; p0 < a.parts; p0 += 3 * U) {
            uint64_t w[U];
            int sf[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                // (no branch may part the loads; bins past kTopBin are zeros, parts past the last add nothing)
                const int p = min(p0 + 3 * u, a.parts - 1);
                sf[u] = p0 + 3 * u < a.parts ? __builtin_amdgcn_readlane(p < 64 ? shift[0] : shift[1], p & 63) : 64;
                w[u] = hist[p * kBins + min(max(bin, 0) + kSub * sf[u], kBins - 1)];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {             // (row_mass of the mass, whose bits the first shift leaves)
                const uint64_t x = sf[u] < 64 ? w[u] : 0;
                count += uint32_t(x >> kMassBits);
                mass += (x << (64 - kMassBits)) >> min(64 - kMassBits - kRowShift + sf[u], 63);
            }
        }
        if (g && bin >= 0) {
            ps.mass[g - 1][i] = mass;
            ps.count[g - 1][i] = count;
        }
    }
    __syncthreads();
    if (tid <= kTopBin) {
        mass += ps.mass[0][tid] + ps.mass[1][tid];
        count += ps.count[0][tid] + ps.count[1][tid];
    }
    cumulate(mass, count, sh);
    borders(a, s, mx, J, a.list_max, sh);
    if (tid == 0) sh.plan.threshold_q = s.q > 0.f ? q_threshold<TYPE>(sh.qkey) : 0;
    return true;
}

template <int TYPE>
__global__ __launch_bounds__(kRowThreads) void sample_select_kernel(SampleArgs a, int row0) {
    const int slot = blockIdx.x, row = row0 + slot, tid = threadIdx.x;
    __shared__ RowShared sh;
    __shared__ PlanShared s_plan;
    __shared__ DrawShared s_draw;
    RowState* st = a.state + slot;
    const Setting s = setting(a, row);
    if (!plan_row<TYPE>(a, slot, row, s, true, sh, s_plan, s_draw)) {
        if (tid == 0) st->plan.mode = kDone;
        return;
    }
    if (tid == 0) {
        st->plan = sh.plan;
        st->count = 0;
    }
    if (tid < kBins) st->cum_mass[tid] = sh.cm[tid];
}

// Lists the entries of the plan's ranges among the values that the block's threads hold.  The block takes
// its place in the list with one addition.
// Inside one launch (HERE) the entries pass between blocks: relaxed accesses of device scope, past the
// caches that are not coherent between the chip's parts.
template <bool HERE> __device__ __forceinline__ void put_entry(uint2* list, uint32_t at, uint32_t key, uint32_t col) {
    if constexpr (HERE)
        __hip_atomic_store(reinterpret_cast<uint64_t*>(list) + at, (uint64_t(col) << 32) | key, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    else list[at] = make_uint2(key, col);
}
template <bool HERE> __device__ __forceinline__ uint2 get_entry(const uint2* list, int at) {
    if constexpr (!HERE) return list[at];
    const uint64_t w = __hip_atomic_load(reinterpret_cast<const uint64_t*>(list) + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_uint2(uint32_t(w), uint32_t(w >> 32));
}
template <int THREADS> struct GatherShared { int n[THREADS / 64]; uint32_t at; };
template <int TYPE, int THREADS, int PIECES, bool HERE>
__device__ __forceinline__ void gather_part(const SampleArgs& a, int slot, const Plan& plan, float least,
                                            const Piece<TYPE> (&v)[PIECES], int col0, GatherShared<THREADS>& gs) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    uint2* list = a.list + size_t(slot) * a.list_max;
    uint32_t in = 0;
    if (HERE && plan.mode == kModeSmall) {            // the first range alone, which has no upper end
        const float from = fmaxf(least, unordered(plan.lo[0]));
#pragma unroll
        for (int u = 0; u < PIECES; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) in |= uint32_t(v[u][e] >= from) << (8 * u + e);
    } else {
#pragma unroll
        for (int u = 0; u < PIECES; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e)               // (v >= least is false for NaN)
                in |= uint32_t(v[u][e] >= least && in_ranges(plan, ordered(v[u][e]))) << (8 * u + e);
    }
    const int own = __popc(in), run = wave_prefix_sum(own);
    if (lane == 63) gs.n[wv] = run;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        before += w < wv ? gs.n[w] : 0;
        total += gs.n[w];
    }
    if (!total) return;
    if (tid == 0) gs.at = atomicAdd(&a.state[slot].count, uint32_t(total));
    __syncthreads();
    uint32_t at = gs.at + uint32_t(before + run - own);
#pragma unroll
    for (int u = 0; u < PIECES; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (in >> (8 * u + e) & 1) {
                if (at < uint32_t(a.list_max)) put_entry<HERE>(list, at, ordered(v[u][e]), uint32_t(col0 + 8 * THREADS * u + e));
                ++at;
            }
}

// Reads the logits of the parts that reach a range a second time (mostly from L2 and the memory-side
// cache: 5.4 MB of 31.8 missed), 8 to 9 us; one addition to the row's count a block.
template <int TYPE, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_gather_kernel(SampleArgs a, int row0) {
    const int part = blockIdx.x, slot = blockIdx.y, row = row0 + slot;
    const Plan& plan = a.state[slot].plan;
    __shared__ GatherShared<THREADS> gs;
    if (plan.mode != kModeSmall && plan.mode != kModeList) return;
    const PartMeta meta = a.meta[size_t(slot) * a.parts + part];
    if (meta.key < plan.lo[0] && meta.key < plan.lo[1] && meta.key < plan.lo[2]) return;
    const void* src = row_of<TYPE>(a, row);
    constexpr int kPieces = kPart / 8 / THREADS;
    const int col0 = part * kPart + int(threadIdx.x) * 8;
    Piece<TYPE> v[kPieces];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) v[u].load(src, col0 + 8 * THREADS * u, a.N);
    gather_part<TYPE, THREADS, kPieces, false>(a, slot, plan, meta.least, v, col0, gs);
}

// The parts' histograms, in registers ahead of the border they are cut at: lane l of a wave holds
// bins l, l + 64, .. of parts wave, wave + 16 (rows of more parts load the others when they sum).
constexpr int kAhead = 2, kBinSteps = (kTopBin + 64) / 64;
__device__ __forceinline__ void load_bins(const SampleArgs& a, int slot, int p, uint64_t (&w)[kBinSteps]) {
    const uint64_t* hist = a.hist + (size_t(slot) * a.parts + p) * kBins;
#pragma unroll
    for (int i = 0; i < kBinSteps; ++i) {
        const int b = 64 * i + int(threadIdx.x & 63);
        w[i] = p < a.parts && b <= kTopBin ? hist[b] : 0;
    }
}
// part_mass[p] = the row mass of the part's bins above `bin` of the row
__device__ __forceinline__ void sum_parts(const SampleArgs& a, int slot, int bin, uint64_t (&ahead)[kAhead][kBinSteps],
                                          RowShared& sh) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    auto sum = [&](int p, const uint64_t (&w)[kBinSteps]) {
        const int shift = sh.shift[p];
        uint64_t m = 0;
#pragma unroll
        for (int i = 0; i < kBinSteps; ++i)            // (row_mass, as in plan_row; a part without bins has shift 64)
            m += 64 * i + lane > bin + kSub * shift ? (w[i] << (64 - kMassBits)) >> min(64 - kMassBits - kRowShift + shift, 63) : 0;
        m = wave_sum_u64(m);
        if (lane == 0) sh.part_mass[p] = m;
    };
#pragma unroll
    for (int h = 0; h < kAhead; ++h)
        if (wv + h * kRowWaves < a.parts) sum(wv + h * kRowWaves, ahead[h]);
    for (int p = wv + kAhead * kRowWaves; p < a.parts; p += kRowWaves) {
        uint64_t w[kBinSteps];
        load_bins(a, slot, p, w);
        sum(p, w);
    }
}

struct EntryList { uint64_t comp[kListLds], mass[kListLds]; };

union FinishShared { PlanShared plan; SmallList small; struct { EntryList list; Descent descent; } border; DrawShared draw; };

// The token of a row with a plan and its entries listed (n of them; ahead0: entry `tid`, of which
// there is room for 1024 at least).
template <int TYPE, bool HERE>
__device__ __forceinline__ void finish_row(const SampleArgs& a, int slot, int row, const Setting& s, int n, uint2 ahead0,
                                           RowShared& sh, FinishShared& un) {
    const int tid = threadIdx.x, mode = sh.plan.mode;
    const double J = sh.plan.J;
    const uint2* list = a.list + size_t(slot) * a.list_max;
    const void* src = row_of<TYPE>(a, row);
    const Plan& plan = sh.plan;
    const uint64_t tq = plan.threshold_q;
    auto entry_mass = [&](uint32_t key, int col) -> uint64_t {
        const int part = (col / kPart) & (kPartsMax - 1);
        uint64_t m;
        return bin_mass(unordered(key), sh.scale[part], m) >= 0 ? row_mass(m, sh.shift[part]) : 0;
    };
    if (mode == kModeSmall) {
        const int e = min(n, kSmall);
        if (tid < kSmall) {
            un.small.comp[tid] = tid < e ? comp_of<TYPE>(ahead0.x, int(ahead0.y)) : 0;
            un.small.mass[tid] = tid < e ? entry_mass(ahead0.x, int(ahead0.y)) : 0;
            un.small.val[tid] = unordered(ahead0.x);
        }
        finish_small(a, row, s, plan, e, tq, un.small);
        return;
    }
    uint64_t ahead[kAhead][kBinSteps];
#pragma unroll
    for (int h = 0; h < kAhead; ++h) load_bins(a, slot, (tid >> 6) + h * kRowWaves, ahead[h]);
    const bool lds = mode == kModeList && n <= kListLds;
    EntryList& en = un.border.list;
    if (lds) {
        constexpr int kBatch = 4;                     // loads of a thread in flight
        uint2 w[kBatch] = {ahead0};
        for (int i0 = tid; i0 < n; i0 += kBatch * kRowThreads) {
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int i = i0 + b * kRowThreads;
                if (i != tid && i < n) w[b] = get_entry<HERE>(list, i);
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int i = i0 + b * kRowThreads;
                if (i >= n) break;
                en.comp[i] = comp_of<TYPE>(w[b].x, int(w[b].y));
                en.mass[i] = entry_mass(w[b].x, int(w[b].y));
            }
        }
        __syncthreads();
    }
    // f(comp, row mass) of the entries with a key in [lo, hi).  The list holds a part's entries side by
    // side: a wave's lanes take entries n / 64 apart, or its LDS additions would mostly meet at one address
    // (2800 entries of a few bf16 values: 7200 clocks a round, 64 columns of one part a wave).
    const int apart = ((n + 63) >> 6) | 1;            // (odd: no bank conflicts)
    auto each = [&](uint32_t lo, uint32_t hi, auto&& f) {
        if (lds) {
            for (int t = tid >> 6; t < apart; t += kRowWaves) {
                const int i = (tid & 63) * apart + t;
                if (i >= n) continue;
                const uint32_t k = comp_key<TYPE>(en.comp[i]);
                if (k >= lo && k < hi) f(en.comp[i], en.mass[i]);
            }
        } else if (mode == kModeList) {
            for (int i = tid; i < n; i += kRowThreads) {
                const uint2 w = get_entry<HERE>(list, i);
                if (w.x >= lo && w.x < hi) f(comp_of<TYPE>(w.x, int(w.y)), entry_mass(w.x, int(w.y)));
            }
        } else {
            for (int c0 = tid * 8; c0 < a.N; c0 += kRowThreads * 8) {
                Piece<TYPE> v;
                v.load(src, c0, a.N);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t k = ordered(v[e]);
                    if (k >= lo && k < hi && v[e] >= sh.least[(c0 + e) / kPart]) f(comp_of<TYPE>(k, c0 + e), entry_mass(k, c0 + e));
                }
            }
        }
    };
    int bf;
    const uint64_t threshold = threshold_of<TYPE>(s, plan, sh.cm, tq, mode == kModeWalk ? ~0u : uint32_t(n), each, un.border.descent, sh, bf);
    sum_parts(a, slot, bf, ahead, sh);
    bin_range(bf, s, plan, sh);
    if (bf >= 0)
        each(sh.edge[0], sh.edge[1], [&](uint64_t comp, uint64_t m) {
            if (comp >= threshold)
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.part_mass[comp_col(comp) / kPart]), (unsigned long long)m);
        });
    __syncthreads();
    draw_part(a.parts, s, sh);
    const int part = sh.part;
    if (part < 0) {                                   // (logits that changed under the call)
        if (tid == 0) give(a, row, -1, __builtin_nanf(""));
        return;
    }
    Piece<TYPE> v;
    const int col0 = part * kPart + tid * kPer;
    v.load(src, col0, a.N);
    draw_column<TYPE, true>(a, row, s, J, sh.scale[part], sh.least[part], sh.shift[part], threshold, v, col0, sh, un.draw);
}

// Bound by its chain of LDS passes and barriers: 5 us where 256 candidates decide, 14 to 19 where borders
// are found in lists.
template <int TYPE>
__global__ __launch_bounds__(kRowThreads) void sample_finish_kernel(SampleArgs a, int row0) {
    const int slot = blockIdx.x, row = row0 + slot, tid = threadIdx.x;
    const RowState* st = a.state + slot;
    __shared__ RowShared sh;
    __shared__ FinishShared un;
    // all that the row needs is loaded at once
    const uint2 ahead0 = a.list[size_t(slot) * a.list_max + tid];
    const uint64_t cum = tid < kBins ? st->cum_mass[tid] : 0;
    const int mode = st->plan.mode;
    const double J = st->plan.J;
    const uint32_t listed = st->count;
    const Setting s = setting(a, row);
    if (mode == kDone) return;
    if (tid < a.parts) {
        const PartMeta m = a.meta[size_t(slot) * a.parts + tid];
        set_part(tid, m, s.c, m.key ? part_shift(J, m.j) : 64, sh);
    }
    if (tid == 0) sh.plan = st->plan;
    if (tid < kBins) sh.cm[tid] = cum;
    __syncthreads();
    finish_row<TYPE, false>(a, slot, row, s, mode == kModeWalk ? 0 : int(min(listed, uint32_t(a.list_max))), ahead0, sh, un);
}

// Select, gather and finish of few rows in one launch: every block of a row makes its plan, lists its
// part's entries, and the last one to have done so ends the row.  Entries, their count and the arrivals
// pass through relaxed accesses of device scope, ordered by a wait for the wave's own stores: a fence of
// every thread wrote back and dropped the caches, 20 to 90 us.  11.5 us for a row of top-k (6 of them
// plan and list), 16 to 21 with top-p's list of some thousand entries.
template <int TYPE>
__global__ __launch_bounds__(kRowThreads) void sample_rest_kernel(SampleArgs a, int row0) {
    const int part = blockIdx.x, slot = blockIdx.y, row = row0 + slot, tid = threadIdx.x;
    RowState* st = a.state + slot;
    __shared__ RowShared sh;
    __shared__ FinishShared un;
    __shared__ GatherShared<kRowThreads> gs;
    __shared__ uint32_t s_arrived;
    Piece<TYPE> v[1];
    const int col0 = part * kPart + tid * kPer;
    v[0].load(row_of<TYPE>(a, row), col0, a.N);
    const Setting s = setting(a, row);
    // (a draw's scratch lies over the plan's: rows without a cut do not use that)
    if (!plan_row<TYPE>(a, slot, row, s, part == 0, sh, un.plan, un.draw)) return;
    __syncthreads();
    if (sh.plan.mode != kModeWalk && sh.shift[part] < 64)
        gather_part<TYPE, kRowThreads, 1, true>(a, slot, sh.plan, sh.least[part], v, col0, gs);
    // every wave's entries have reached the device's memory before the block counts as done
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) s_arrived = __hip_atomic_fetch_add(&st->arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (s_arrived != uint32_t(a.parts) - 1) return;
    const uint32_t listed = __hip_atomic_load(&st->count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint2 ahead0 = get_entry<true>(a.list + size_t(slot) * a.list_max, tid);
    finish_row<TYPE, true>(a, slot, row, s, sh.plan.mode == kModeWalk ? 0 : int(min(listed, uint32_t(a.list_max))), ahead0, sh, un);
}

// Rows of one part: all of it by one block, the logits in LDS after the histogram.  One block a CU (its
// registers, 76 to 80 where two blocks of 1024 threads would need 64; LDS, 78 KB, would hold two), so bound
// by the chain of its steps: 256 rows of 4096 bf16 17.2 us with mixed settings, 11.4 with top-k of 20 to 50.
template <int TYPE>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(SampleArgs a, int row0) {
    const int row = row0 + int(blockIdx.x), tid = threadIdx.x;
    __shared__ RowShared sh;
    __shared__ union {
        struct { union { PartShared<kRowThreads> part; SmallList small; Descent descent; }; float v[kPart]; };
        DrawShared draw;
    } un;
    float* s_v = un.v;
    __shared__ uint32_t s_count;
    const int col0 = tid * kPer;
    Piece<TYPE> v[1];
    v[0].load(row_of<TYPE>(a, row), col0, a.N);
    const Setting s = setting(a, row);
    const PartMeta m = part_pass<TYPE, kRowThreads, 1>(a, s, v, col0, un.part);
    if (!s.valid || !m.key || s.T == 0.f) {
        if (tid == 0) {
            const bool fine = s.valid && m.key;
            give(a, row, fine ? m.arg : -1, fine ? 0.f : __builtin_nanf(""));
            flag_or(a.flags, !s.valid ? kSampleSetting : !m.key ? kSampleEmpty : 0u);
        }
        return;
    }
    const double J = m.j;
    const Scale k = scale_of(s.c, J);
    uint64_t threshold = 0;
    if (s.cut) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) s_v[col0 + e] = v[0][e];
        if (tid == 0) s_count = 0;
        __syncthreads();
        const uint64_t w = tid <= kTopBin ? un.part.hist[kTopBin - tid] : 0;
        cumulate(row_mass(w & kMassMask, 0), uint32_t(w >> kMassBits), sh);
        borders(a, s, unordered(m.key), J, kPart, sh);
        const Plan& plan = sh.plan;
        threshold = s.q > 0.f ? q_threshold<TYPE>(sh.qkey) : 0;
        auto mass_of = [&](float x) -> uint64_t {
            uint64_t e;
            return bin_mass(x, k, e) >= 0 ? row_mass(e, 0) : 0;
        };
        if (plan.mode == kModeSmall) {
            if (tid < kSmall) {
                un.small.comp[tid] = 0;
                un.small.mass[tid] = 0;
            }
            __syncthreads();
            for (int c = tid; c < a.N; c += kRowThreads) {
                const float x = s_v[c];
                const uint32_t key = ordered(x);
                if (x >= m.least && in_ranges(plan, key)) {
                    const uint32_t at = atomicAdd(&s_count, 1u);
                    if (at < uint32_t(kSmall)) {
                        un.small.comp[at] = comp_of<TYPE>(key, c);
                        un.small.mass[at] = mass_of(x);
                        un.small.val[at] = x;
                    }
                }
            }
            __syncthreads();
            finish_small(a, row, s, plan, min(int(s_count), kSmall), threshold, un.small);
            return;
        }
        auto each = [&](uint32_t lo, uint32_t hi, auto&& f) {
            for (int c = tid; c < a.N; c += kRowThreads) {
                const float x = s_v[c];
                const uint32_t key = ordered(x);
                if (key >= lo && key < hi && x >= m.least) f(comp_of<TYPE>(key, c), mass_of(x));
            }
        };
        int bf;
        threshold = threshold_of<TYPE>(s, plan, sh.cm, threshold, ~0u, each, un.descent, sh, bf);
    }
    // the kept mass, and the token
    const Cut cut = cut_of<TYPE>(threshold);
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        uint64_t x;
        const int bin = bin_mass(v[0][e], k, x);
        if (bin >= 0 && v[0][e] >= m.least && cut.keeps(v[0][e], col0 + e)) sum += x;
    }
    sum = wave_sum_u64(sum);
    __syncthreads();
    if ((tid & 63) == 0) sh.wave_mass[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
        uint64_t total = 0;
#pragma unroll
        for (int w = 0; w < kRowWaves; ++w) total += sh.wave_mass[w];
        sh.total = row_mass(total, 0);
        sh.rest = __umul64hi(fraction(s.u), sh.total);
    }
    __syncthreads();
    draw_column<TYPE, true>(a, row, s, J, k, m.least, 0, threshold, v[0], col0, sh, un.draw);
}

// rows of an empty vocabulary
__global__ __launch_bounds__(64) void sample_empty_kernel(int M, int64_t* token, float* logprob, uint32_t* flags) {
    const int row = blockIdx.x * 64 + threadIdx.x;
    if (row >= M) return;
    token[row] = -1;
    if (logprob) logprob[row] = __builtin_nanf("");
    if (threadIdx.x == 0) flag_or(flags, kSampleEmpty);
}

int sample_parts_of(int N) { return (N + kPart - 1) / kPart; }
// rows that share the workspace at once: at least 64, and 1024 parts
int sample_chunk(int N) { return std::max(64, 1024 / std::max(sample_parts_of(N), 1)); }

struct SampleLayout { size_t hist, meta, state, list, bytes; int list_max; };
SampleLayout sample_layout(int Mcap, int N) {
    SampleLayout l{};
    const int parts = sample_parts_of(N);
    if (parts <= 1) return l;                        // one launch, nothing between blocks
    const size_t rows = size_t(std::min(Mcap, sample_chunk(N)));
    size_t cursor = 0;
    auto add = [&](size_t& field, size_t bytes) { field = cursor; cursor = align256(cursor + bytes); };
    l.list_max = std::min(N, kListMax);
    add(l.hist, rows * parts * kBins * 8);
    add(l.meta, rows * parts * sizeof(PartMeta));
    add(l.state, rows * sizeof(RowState));
    add(l.list, rows * size_t(l.list_max) * 8);
    l.bytes = cursor;
    return l;
}

template <int TYPE> hipError_t sample_rows(const SampleArgs& a, int row0, int rows, hipStream_t s) {
    const dim3 parts(a.parts, rows);
    if (a.parts * rows <= kFewParts) {
        timed_launch("sample_parts", sample_parts_kernel<TYPE, 1024>, parts, dim3(1024), 0, s, a, row0);
        timed_launch("sample_rest", sample_rest_kernel<TYPE>, parts, dim3(kRowThreads), 0, s, a, row0);
        return hipGetLastError();
    }
    timed_launch("sample_parts", sample_parts_kernel<TYPE, 256>, parts, dim3(256), 0, s, a, row0);
    timed_launch("sample_select", sample_select_kernel<TYPE>, dim3(rows), dim3(kRowThreads), 0, s, a, row0);
    const hipError_t st = hipGetLastError();
    // with no cut at all, select has drawn every row
    if (st != hipSuccess || (!a.top_k && !a.top_p && !a.min_p)) return st;
    timed_launch("sample_gather", sample_gather_kernel<TYPE, 256>, parts, dim3(256), 0, s, a, row0);
    timed_launch("sample_finish", sample_finish_kernel<TYPE>, dim3(rows), dim3(kRowThreads), 0, s, a, row0);
    return hipGetLastError();
}

template <int TYPE> hipError_t sample_all(const SampleArgs& a, int M, hipStream_t s) {
    const int chunk = a.parts == 1 ? 1 << 20 : sample_chunk(a.N);      // (a grid has less than 2^32 threads)
    for (int64_t r = 0; r < M; r += chunk) {
        const int row0 = int(r), rows = int(std::min<int64_t>(M - r, chunk));
        hipError_t st;
        if (a.parts == 1) {
            timed_launch("sample_row", sample_row_kernel<TYPE>, dim3(rows), dim3(kRowThreads), 0, s, a, row0);
            st = hipGetLastError();
        } else st = sample_rows<TYPE>(a, row0, rows, s);
        if (st != hipSuccess) return st;
    }
    return hipSuccess;
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
        timed_launch("sample_empty", sample_empty_kernel, dim3((unsigned(M) + 63) / 64), dim3(64), 0, stream, M,
                     static_cast<int64_t*>(token), static_cast<float*>(logprob), static_cast<uint32_t*>(flags));
        return hipGetLastError();
    }
    const SampleArgs a{logits, ld, N, sample_parts_of(N), l.list_max, static_cast<const float*>(uniform),
                       static_cast<const float*>(temperature), static_cast<const int32_t*>(top_k),
                       static_cast<const float*>(top_p), static_cast<const float*>(min_p),
                       at<uint64_t>(workspace, l.hist), at<PartMeta>(workspace, l.meta),
                       at<RowState>(workspace, l.state), at<uint2>(workspace, l.list),
                       static_cast<int64_t*>(token), static_cast<float*>(logprob), static_cast<uint32_t*>(flags)};
    if (logits_type == ORNITH_LOGITS_BF16) return sample_all<ORNITH_LOGITS_BF16>(a, M, stream);
    if (logits_type == ORNITH_LOGITS_F16) return sample_all<ORNITH_LOGITS_F16>(a, M, stream);
    return sample_all<ORNITH_LOGITS_F32>(a, M, stream);
}
