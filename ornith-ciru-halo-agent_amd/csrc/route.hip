// Routing to experts from given logits (definition: include/ornith_route.h).
//
// A row on L lanes of a wave, a group's experts on S of them, NPL neighbouring
// experts a lane.  Values to pick by are fp64 numbers with the expert's id in
// their lowest ten bits, so no two are equal and a maximum over lanes is a
// pick; what those bits displace is below 2^-42 of the value.  An fp32 logit
// leaves 29 bits clear, so picks without a bias are exact.  On a whole wave the
// picks come from a threshold and a count (route_pick); on fewer lanes each sorts
// its own once, and a pick is the largest of the lanes' first, which its lane drops.  Scores in fp64 (which the vector unit multiplies at the rate of
// fp32): without a bias only those of the picks.
//
// Bound by vector issue where rows are many (8192 rows of 256 in 8 groups, sigmoid
// and bias: 12.4 us in a graph, 770 instructions a row, 8.4 MB that a copy's rate
// would read in 1.7; without bias and groups 7.9), by launch and one chain where they
// are few (1 row 3.3 us: logits, threshold, count, the picks' logits again).
#include <algorithm>
#include <cmath>
#include <type_traits>
#include "kernels.hpp"
#include "timing.hpp"
#include "topk.hpp"
#include "validate.hpp"
#include "../../include/ornith_route.h"

namespace ornith {
namespace {

constexpr int kRouteMaxE = 1024, kRouteMaxK = 32, kRouteMaxG = 64;
enum : uint32_t { kRouteNan = 1, kRouteFew = 4 };

struct RouteArgs {
    const void* logits;
    int64_t ld;
    const float* bias;
    float* weights;
    int32_t* ids;
    uint32_t* flags;
    int M, E, G, Gk, k;
    int gs, S;                      // experts and lanes of a group
    bool wide;                      // rows and lanes' experts on the 16-byte grid
    int score, two, renormalize;
    double scale;
};

constexpr double kNone = -__builtin_huge_val();

// (asm: the builtins quieten both operands first; keys and scores are never NaN)
__device__ __forceinline__ double max_d(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double min_d(double a, double b) {
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
template <int CTRL> __device__ __forceinline__ double dpp_d(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = uint32_t(__builtin_amdgcn_mov_dpp(int(uint32_t(b)), CTRL, 0xF, 0xF, true));
    const uint32_t hi = uint32_t(__builtin_amdgcn_mov_dpp(int(uint32_t(b >> 32)), CTRL, 0xF, 0xF, true));
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
template <int M> __device__ __forceinline__ double xor_perm_d(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = uint32_t(xor_perm_i<M>(int(uint32_t(b)))), hi = uint32_t(xor_perm_i<M>(int(uint32_t(b >> 32))));
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
// f over N neighbouring lanes (a power of two), the result in each of them: after each step 2, 4, .. lanes
// agree, so a mirror pairs whole halves.
template <class T, class F, class X> __device__ __forceinline__ T lanes_fold(T v, int N, F&& f, X&& across) {
    if (N > 1) v = f(v, across(v, std::integral_constant<int, 1>{}));
    if (N > 2) v = f(v, across(v, std::integral_constant<int, 2>{}));
    if (N > 4) v = f(v, across(v, std::integral_constant<int, 4>{}));
    if (N > 8) v = f(v, across(v, std::integral_constant<int, 8>{}));
    if (N > 16) v = f(v, across(v, std::integral_constant<int, 16>{}));
    if (N > 32) v = f(v, across(v, std::integral_constant<int, 32>{}));
    return v;
}
template <int M> __device__ __forceinline__ double across_d(double v) {
    if constexpr (M == 1) return dpp_d<kDppXor1>(v);
    else if constexpr (M == 2) return dpp_d<kDppXor2>(v);
    else if constexpr (M == 4) return dpp_d<kDppHalfMirror>(v);
    else if constexpr (M == 8) return dpp_d<kDppMirror>(v);
    else return xor_perm_d<M>(v);
}
__device__ __forceinline__ double lanes_max(double v, int N) {
    return lanes_fold(v, N, [](double a, double b) { return max_d(a, b); },
                      [](double x, auto m) { return across_d<decltype(m)::value>(x); });
}
template <int M> __device__ __forceinline__ float across_f(float v) {
    if constexpr (M == 1) return dpp_f<kDppXor1>(v);
    else if constexpr (M == 2) return dpp_f<kDppXor2>(v);
    else if constexpr (M == 4) return dpp_f<kDppHalfMirror>(v);
    else if constexpr (M == 8) return dpp_f<kDppMirror>(v);
    else return xor_perm_f<M>(v);
}
__device__ __forceinline__ float lanes_maxf(float v, int N) {
    return lanes_fold(v, N, [](float a, float b) { return fmaxf(a, b); },
                      [](float x, auto m) { return across_f<decltype(m)::value>(x); });
}
__device__ __forceinline__ double lanes_sum(double v, int N) {
    return lanes_fold(v, N, [](double a, double b) { return a + b; },
                      [](double x, auto m) { return across_d<decltype(m)::value>(x); });
}

template <int TYPE> __device__ __forceinline__ float route_logit(const void* row, int e) {
    if constexpr (TYPE == 2) return static_cast<const float*>(row)[e];
    else if constexpr (TYPE == 1) return f16_bits_to_f32(static_cast<const uint16_t*>(row)[e]);
    else return bf16_bits_to_f32(static_cast<const uint16_t*>(row)[e]);
}
// exp(x) of x <= 700 (below -800: 0): x = n ln 2 + r, |r| <= ln 2 / 2, the exponential series to r^11 (2^-46 off at
// most), 2^n.
__device__ __forceinline__ double exp_d(double x) {
    x = max_d(x, -800.0);
    const double n = __builtin_rint(x * 0x1.71547652b82fep+0);
    double r = __builtin_fma(n, -0x1.62e42fefa39efp-1, x);
    r = __builtin_fma(n, -0x1.abc9e3b39803fp-56, r);
    double p = 1.0 / 39916800.0;
    constexpr double c[] = {1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0, 1.0 / 120.0, 1.0 / 24.0,
                            1.0 / 6.0, 0.5, 1.0, 1.0};
#pragma unroll
    for (int i = 0; i < 11; ++i) p = __builtin_fma(p, r, c[i]);
    return __builtin_ldexp(p, int(n));
}
// 1 / x of x in [2^-1000, 2^1011]: the instruction's estimate and two of Newton's steps
__device__ __forceinline__ double rcp_d(double x) {
    double y = __builtin_amdgcn_rcp(x);
    y = __builtin_fma(y, __builtin_fma(-x, y, 1.0), y);
    return __builtin_fma(y, __builtin_fma(-x, y, 1.0), y);
}
// exp(l - mx) with mx the row's largest, and 1 / (1 + exp(-l))
__device__ __forceinline__ double soft_mass(float l, float mx) { return l == mx ? 1.0 : exp_d(double(l) - double(mx)); }
__device__ __forceinline__ double sigmoid_d(float l) { return rcp_d(1.0 + exp_d(-max_d(double(l), -700.0))); }

// c with the id behind it: of two equal c the lower id is the larger.
__device__ __forceinline__ double route_key(double c, int id) {
    c = min_d(max_d(c, -0x1p1000), 0x1p1000) + 0.0;
    const uint64_t b = __builtin_bit_cast(uint64_t, c);
    const uint64_t low = (b >> 63) ? uint64_t(id) : uint64_t(1023 - id);
    return __builtin_bit_cast(double, (b & ~uint64_t(1023)) | low);
}
__device__ __forceinline__ int route_id(double key) {
    const uint64_t b = __builtin_bit_cast(uint64_t, key);
    return (b >> 63) ? int(b & 1023) : 1023 - int(b & 1023);
}

// Descending, by the comparisons of Batcher's odd-even merge sort (N a power of two).
template <int N> __device__ __forceinline__ void sort_d(double* v) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const double a = v[i + j], b = v[i + j + k];
                        v[i + j] = max_d(a, b);
                        v[i + j + k] = min_d(a, b);
                    }
}
// Picks of one row on a wave, by a threshold and a count (fp64 maxima take several times an fp32 one's time):
//  1. t, the k-th largest of the maxima of 2 lanes (K = 8; of one for 32), of fp32 roundings: at least k
//     experts reach it, so the picks are among those that do, about half as many more;
//  2. those compacted, lane i counts who is ahead of the i-th, and the first k are handed out by that.
// More than 64 that reach t (many equal values): k maxima over the lanes instead.
template <int NPL, int K> __device__ __forceinline__ double route_pick(double (&c)[NPL], int e0, int k) {
    __shared__ double s_keys[4][64 + 2], s_picks[4][kRouteMaxK];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    double *keys = s_keys[wv], *picks = s_picks[wv];
    uint32_t h[NPL], most = 0;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        h[i] = c[i] > kNone ? f32_order_key(float(c[i]) + 0.f) : 0u;
        most = max(most, h[i]);
    }
    constexpr int T = K <= 8 ? 2 : 1;                  // lanes of a maximum
    if constexpr (T >= 2) most = max(most, uint32_t(dpp_i<kDppXor1>(int(most))));
    int ahead = 0;                                     // maxima that reach this one
#pragma unroll
    for (int j = 0; j < 64 / T; ++j) ahead += uint32_t(__builtin_amdgcn_readlane(int(most), T * j)) >= most ? 1 : 0;
    const uint32_t t = max(wave_max_u(ahead >= k ? most : 0u), 1u);
    int n = 0, place[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        const uint64_t in = __ballot(h[i] >= t);
        place[i] = h[i] >= t ? n + int(__builtin_amdgcn_mbcnt_hi(uint32_t(in >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(in), 0u))) : 64;
        n += __popcll(in);
    }
    if (n > 64) {
#pragma unroll
        for (int i = 0; i < NPL; ++i) c[i] = c[i] > kNone ? route_key(c[i], e0 + i) : kNone;
        double mine = kNone;
        for (int r = 0; r < k; ++r) {
            double m = kNone;
#pragma unroll
            for (int i = 0; i < NPL; ++i) m = max_d(m, c[i]);
            m = lanes_max(m, 64);
#pragma unroll
            for (int i = 0; i < NPL; ++i) c[i] = c[i] == m ? kNone : c[i];
            mine = lane == r ? m : mine;
        }
        return mine;
    }
    if (lane < kRouteMaxK) picks[lane] = kNone;
    keys[lane] = kNone;                                // (reads go by two)
#pragma unroll
    for (int i = 0; i < NPL; ++i)
        if (__ballot(place[i] < 64)) keys[place[i]] = route_key(c[i], e0 + i);        // (others: the 65th)
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const double mine = keys[lane];
    int rank = 0;
    for (int j = 0; j < n; j += 4) {
        double v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = keys[j + u];
#pragma unroll
        for (int u = 0; u < 4; ++u) rank += v[u] > mine ? 1 : 0;
    }
    if (lane < n && rank < k) picks[rank] = mine;
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return lane < kRouteMaxK ? picks[lane] : kNone;
}

// Lane j of group g's S lanes holds the group's experts NPL j, NPL j + 1, ..  K: picks at most.
template <int TYPE, int L, int NPL, int K>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, ll = lane & (L - 1);
    const int row = (int(blockIdx.x) * 256 + tid) / L, at = min(row, a.M - 1);
    const int g = ll / a.S, first = ll % a.S * NPL, e0 = g * a.gs + first;
    const int mine_of = g < a.G ? min(max(a.gs - first, 0), NPL) : 0;       // experts of this lane
    const void* logits = static_cast<const uint8_t*>(a.logits) + size_t(at) * size_t(a.ld) * (TYPE == 2 ? 4 : 2);
    uint32_t flags = 0;
    float l[NPL], b[NPL];
    constexpr int kPer = TYPE == 2 ? 4 : 8;            // experts of 16 bytes
    bool loaded = false;
    if constexpr (NPL % kPer == 0) {
        if (a.wide) {
            loaded = true;
            u32x4 w[NPL / kPer];
            const uint8_t* from = static_cast<const uint8_t*>(logits) + size_t(mine_of ? e0 : 0) * (16 / kPer);
#pragma unroll
            for (int i = 0; i < NPL / kPer; ++i) w[i] = reinterpret_cast<const u32x4*>(from)[i];
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                const uint32_t v = w[i / kPer][i % kPer * (16 / kPer) / 4];
                l[i] = TYPE == 2 ? __uint_as_float(v) : TYPE == 1 ? f16_bits_to_f32(v >> (16 * (i & 1)) & 0xffffu)
                                                                 : __uint_as_float(i & 1 ? v & 0xffff0000u : v << 16);
                if (!mine_of) l[i] = -__builtin_huge_valf();
            }
        }
    }
    if (!loaded) {
#pragma unroll
        for (int i = 0; i < NPL; ++i) l[i] = route_logit<TYPE>(logits, i < mine_of ? e0 + i : 0);
#pragma unroll
        for (int i = 0; i < NPL; ++i) l[i] = i < mine_of ? l[i] : -__builtin_huge_valf();
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i)
        if (l[i] != l[i]) flags |= kRouteNan;
    // scores and what the experts are picked by
    const bool softmax = a.score == ORNITH_SCORE_SOFTMAX;
    double c[NPL], total = 1.0;
    float mx = -__builtin_huge_valf();                 // (a renormalised softmax's weights are relative to its picks)
    if (softmax && (a.bias || !a.renormalize || (a.two && a.Gk < a.G))) {
#pragma unroll
        for (int i = 0; i < NPL; ++i) mx = fmaxf(mx, l[i]);
        mx = lanes_maxf(mx, L);
    }
    if (a.bias) {
#pragma unroll
        for (int i = 0; i < NPL; ++i) b[i] = a.bias[i < mine_of ? e0 + i : 0];
    }
    if (softmax && (a.bias || !a.renormalize)) {
        total = 0.0;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            c[i] = l[i] > -__builtin_huge_valf() ? soft_mass(l[i], mx) : 0.0;
            total += c[i];
        }
        total = lanes_sum(total, L);
    }
    const double part = total > 0.0 ? rcp_d(total) : 0.0;
    if (!a.bias) {
#pragma unroll
        for (int i = 0; i < NPL; ++i) c[i] = l[i] > -__builtin_huge_valf() ? double(l[i]) : kNone;     // (NaN: none)
    } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            if (i < mine_of && !(b[i] < __builtin_huge_valf())) flags |= kRouteNan;
            const double s = softmax ? c[i] * part : sigmoid_d(l[i]), v = s + double(b[i]);
            c[i] = l[i] > -__builtin_huge_valf() && v > kNone ? v : kNone;
        }
    }
    if (a.Gk < a.G) {
        // the two largest c of the group, its score, and how many groups are ahead of it
        double m1 = kNone, m2 = kNone;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            m2 = max_d(m2, min_d(m1, c[i]));
            m1 = max_d(m1, c[i]);
        }
        struct Two { double a, b; };
        const Two best = lanes_fold(Two{m1, m2}, a.S,
            [](Two x, Two y) { return Two{max_d(x.a, y.a), max_d(min_d(x.a, y.a), max_d(x.b, y.b))}; },
            [](Two x, auto m) { return Two{across_d<decltype(m)::value>(x.a), across_d<decltype(m)::value>(x.b)}; });
        double score = best.a;
        if (a.two) {
            auto s = [&](double v) {
                if (!(v > kNone)) return 0.0;
                return a.bias ? v : softmax ? soft_mass(float(v), mx) : sigmoid_d(float(v));
            };
            score = best.a > kNone ? s(best.a) + s(best.b) : kNone;
        }
        __shared__ double s_score[256];                // (a row's are its wave's)
        s_score[tid] = score;
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const double* of = s_score + (tid - ll);
        int ahead = 0;
        for (int h = 0; h < a.G; ++h) {
            const double v = of[h * a.S];
            ahead += v > score || (v == score && h < g) ? 1 : 0;
        }
        if (ahead >= a.Gk) {
#pragma unroll
            for (int i = 0; i < NPL; ++i) c[i] = kNone;
        }
    }
    double mine = kNone;                               // lane r: the r-th pick
    if constexpr (L == 64) mine = route_pick<NPL, K>(c, e0, a.k);
    else {
#pragma unroll
        for (int i = 0; i < NPL; ++i) c[i] = c[i] > kNone ? route_key(c[i], e0 + i) : kNone;
        sort_d<NPL>(c);
        for (int r = 0; r < a.k; ++r) {
            const double m = lanes_max(c[0], L);
            const bool drop = c[0] == m;
#pragma unroll
            for (int i = 0; i + 1 < NPL; ++i) c[i] = drop ? c[i + 1] : c[i];
            c[NPL - 1] = drop ? kNone : c[NPL - 1];
            mine = ll == r ? m : mine;
        }
    }
    const bool picked = mine > kNone;
    const int id = picked ? route_id(mine) : -1;
    if (ll < a.k && !picked) flags |= kRouteFew;
    // weights, on the first P lanes: of a renormalised softmax relative to the largest that was picked
    constexpr int P = L == 64 ? K : L;
    const float lp = picked ? route_logit<TYPE>(logits, id) : -__builtin_huge_valf();
    double s = 0.0;
    if (softmax) {
        const float top = a.renormalize ? lanes_maxf(lp, P) : mx;
        s = picked ? soft_mass(lp, top) * (a.renormalize ? 1.0 : part) : 0.0;
    } else if (picked) s = sigmoid_d(lp);
    if (a.renormalize) {
        const double sum = lanes_sum(s, P);
        s = sum > 0.0 ? s * rcp_d(sum) : 0.0;
    }
    if (row < a.M) {
        if (ll < a.k) {
            const size_t to = size_t(row) * a.k + ll;
            a.weights[to] = float(s * a.scale);
            a.ids[to] = id;
        }
        flag_or(a.flags, flags);
    }
}

int pow2_from(int n) {
    int p = 1;
    while (p < n) p *= 2;
    return p;
}

template <int TYPE, int L> hipError_t route_rows(RouteArgs a, hipStream_t s) {
    a.S = L / pow2_from(a.G);
    const int npl = pow2_from((a.gs + a.S - 1) / a.S);
    const dim3 grid(unsigned((int64_t(a.M) * L + 255) / 256));
    constexpr int size = TYPE == 2 ? 4 : 2;
    a.wide = a.gs % npl == 0 && npl * size % 16 == 0 && a.ld * size % 16 == 0 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 &&
             a.gs * size % 16 == 0;
    auto go = [&](auto kernel) { timed_launch("route_experts", kernel, grid, dim3(256), 0, s, a); };
    auto of = [&](auto n) {
        constexpr int N = decltype(n)::value;
        if (L < 64 || a.k <= 8) go(route_kernel<TYPE, L, N, 8>);
        else go(route_kernel<TYPE, L, N, 32>);
    };
    if (npl <= 1) of(std::integral_constant<int, 1>{});
    else if (npl <= 2) of(std::integral_constant<int, 2>{});
    else if (npl <= 4) of(std::integral_constant<int, 4>{});
    else if constexpr (L == 64) {
        if (npl <= 8) of(std::integral_constant<int, 8>{});
        else if (npl <= 16) of(std::integral_constant<int, 16>{});
        else of(std::integral_constant<int, 32>{});
    }
    return hipGetLastError();
}

template <int TYPE> hipError_t route_lanes(const RouteArgs& a, hipStream_t s) {
    // The least lanes that leave each at most four experts (us, 16 / 32 / 64 lanes: 8192 rows of 16 experts, 2 picks,
    // 3.0 / 3.9 / 7.1; of 64, 6 picks, 4.0 / 5.0 / 7.4; of 128, 8 picks, - / 6.8 / 8.2)
    auto fits = [&](int L) {
        const int groups = pow2_from(a.G);
        return groups <= L && a.k <= L && (a.gs + L / groups - 1) / (L / groups) <= 4;
    };
    if (fits(16)) return route_rows<TYPE, 16>(a, s);
    if (fits(32)) return route_rows<TYPE, 32>(a, s);
    return route_rows<TYPE, 64>(a, s);
}

}  // namespace
}  // namespace ornith

using namespace ornith;

extern "C" hipError_t ornith_route_experts_launch(const void* logits, int logits_type, int M, int E, int64_t ld,
                                                  const void* bias, int score, int G, int Gk, int group_top, int k,
                                                  int renormalize, float scale, void* weights, void* ids, void* flags,
                                                  hipStream_t stream) {
    if (logits_type < 0 || logits_type > 2 || M < 0 || E < 1 || E > kRouteMaxE || ld < E || G < 1 || G > kRouteMaxG ||
        E % G || Gk < 1 || Gk > G || (group_top != 1 && group_top != 2) || k < 1 || k > kRouteMaxK ||
        k > Gk * (E / G) || (score != ORNITH_SCORE_SOFTMAX && score != ORNITH_SCORE_SIGMOID) ||
        (renormalize != 0 && renormalize != 1) || !std::isfinite(scale))
        return hipErrorInvalidValue;
    if (!M) return hipSuccess;
    const size_t size = logits_type == 2 ? 4 : 2, picks = size_t(M) * size_t(k) * 4;
    if (uint64_t(ld) > (uint64_t(1) << 62) / uint64_t(M)) return hipErrorInvalidValue;
    const Buffer buffers[] = {{logits, (size_t(M - 1) * size_t(ld) + size_t(E)) * size, size, false, false},
                              {bias, size_t(E) * 4, 4, false, true},
                              {weights, picks, 4, true, false},
                              {ids, picks, 4, true, false},
                              {flags, 4, 4, true, false}};
    if (!check_buffers(buffers)) return hipErrorInvalidValue;
    if (Gk == G) Gk = G = 1;                           // (every group stays)
    constexpr int kAtOnce = 1 << 24;                   // rows of a grid, which has less than 2^32 threads
    for (int64_t r = 0; r < M; r += kAtOnce) {
        const RouteArgs a{static_cast<const uint8_t*>(logits) + size_t(r) * size_t(ld) * size, ld,
                          static_cast<const float*>(bias), static_cast<float*>(weights) + r * k,
                          static_cast<int32_t*>(ids) + r * k, static_cast<uint32_t*>(flags),
                          int(M - r < kAtOnce ? M - r : kAtOnce), E, G, Gk, k, E / G, 0, false, score, group_top == 2,
                          renormalize, double(scale)};
        const hipError_t st = logits_type == 2 ? route_lanes<2>(a, stream)
                            : logits_type == 1 ? route_lanes<1>(a, stream) : route_lanes<0>(a, stream);
        if (st != hipSuccess) return st;
    }
    return hipSuccess;
}
