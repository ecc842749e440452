// Routing to experts from given logits (definition: include/ornith_route.h).
//
// A row on L lanes of a wave.  Values to pick by are fp64 numbers with the
// expert's id in their lowest ten bits, so no two are equal and a maximum over
// lanes is a pick; what those bits displace is below 2^-42 of the value.  An
// fp32 logit leaves 29 bits clear, so picks without a bias are exact.
#include <cmath>
#include "kernels.hpp"
#include "timing.hpp"
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
    int score, two, renormalize;
    double scale;
};

constexpr double kNone = -__builtin_huge_val();

template <int CTRL> __device__ __forceinline__ double dpp_d(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = uint32_t(dpp_i<CTRL>(int(uint32_t(b)))), hi = uint32_t(dpp_i<CTRL>(int(uint32_t(b >> 32))));
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
__device__ __forceinline__ double max_d(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ double lanes_max(double v, int N) {
    return lanes_fold(v, N, [](double a, double b) { return max_d(a, b); },
                      [](double x, auto m) { return across_d<decltype(m)::value>(x); });
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
// exp(l - mx) with mx the row's largest, and 1 / (1 + exp(-l))
__device__ __forceinline__ double soft_mass(float l, float mx) { return l == mx ? 1.0 : exp(double(l) - double(mx)); }
__device__ __forceinline__ double sigmoid_d(float l) { return 1.0 / (1.0 + exp(-fmax(double(l), -700.0))); }

// c with the id behind it: of two equal c the lower id is the larger.
__device__ __forceinline__ double route_key(double c, int id) {
    c = __builtin_fmin(__builtin_fmax(c, -0x1p1000), 0x1p1000) + 0.0;
    const uint64_t b = __builtin_bit_cast(uint64_t, c);
    const uint64_t low = (b >> 63) ? uint64_t(id) : uint64_t(1023 - id);
    return __builtin_bit_cast(double, (b & ~uint64_t(1023)) | low);
}
__device__ __forceinline__ int route_id(double key) {
    const uint64_t b = __builtin_bit_cast(uint64_t, key);
    return (b >> 63) ? int(b & 1023) : 1023 - int(b & 1023);
}

// Lane j of group g's S lanes holds the group's experts j, j + S, ...
template <int TYPE, int L, int NPL>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, ll = lane & (L - 1);
    const int row = (int(blockIdx.x) * 256 + tid) / L, at = min(row, a.M - 1);
    const int g = ll / a.S, j = ll % a.S;
    const void* logits = static_cast<const uint8_t*>(a.logits) + size_t(at) * size_t(a.ld) * (TYPE == 2 ? 4 : 2);
    uint32_t flags = 0;
    float l[NPL];
    float b[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        const int in = i * a.S + j;
        const bool have = g < a.G && in < a.gs;
        const int e = have ? g * a.gs + in : 0;
        l[i] = have ? route_logit<TYPE>(logits, e) : -__builtin_huge_valf();
        b[i] = have && a.bias ? a.bias[e] : 0.f;
    }
    float mx = -__builtin_huge_valf();
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        if (l[i] != l[i] || !(b[i] < __builtin_huge_valf())) flags |= kRouteNan;
        mx = fmaxf(mx, l[i]);
    }
    mx = float(lanes_max(double(mx), L));
    // scores and what the experts are picked by
    const bool softmax = a.score == ORNITH_SCORE_SOFTMAX;
    double c[NPL], total = 1.0;
    if (softmax && (a.bias || !a.renormalize)) {
        total = 0.0;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            c[i] = l[i] > -__builtin_huge_valf() ? soft_mass(l[i], mx) : 0.0;
            total += c[i];
        }
        total = lanes_sum(total, L);
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        if (!a.bias) c[i] = double(l[i]);
        else c[i] = (softmax ? soft_mass(l[i], mx) / total : sigmoid_d(l[i])) + double(b[i]);
        if (!(l[i] > -__builtin_huge_valf()) || !(c[i] > kNone)) c[i] = kNone;      // (NaN too)
    }
    if (a.Gk < a.G) {
        // the two largest c of the group, its score, and how many groups are ahead of it
        double m1 = kNone, m2 = kNone;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            m2 = max_d(m2, __builtin_fmin(m1, c[i]));
            m1 = max_d(m1, c[i]);
        }
        struct Two { double a, b; };
        const Two best = lanes_fold(Two{m1, m2}, a.S,
            [](Two x, Two y) { return Two{max_d(x.a, y.a), max_d(__builtin_fmin(x.a, y.a), max_d(x.b, y.b))}; },
            [](Two x, auto m) { return Two{across_d<decltype(m)::value>(x.a), across_d<decltype(m)::value>(x.b)}; });
        double score = best.a;
        if (a.two && best.b > kNone) {
            auto s = [&](double v) {
                return a.bias ? v : softmax ? soft_mass(float(v), mx) : sigmoid_d(float(v));
            };
            score = s(best.a) + s(best.b);
        } else if (a.two && best.a > kNone && !a.bias) {
            score = softmax ? soft_mass(float(best.a), mx) : sigmoid_d(float(best.a));
        }
        if (g >= a.G) score = kNone;
        __shared__ double s_score[256];
        s_score[tid] = score;
        __syncthreads();
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
#pragma unroll
    for (int i = 0; i < NPL; ++i)
        if (c[i] > kNone) c[i] = route_key(c[i], g * a.gs + i * a.S + j);
    // k picks; lane r keeps the r-th
    double mine = kNone;
    for (int r = 0; r < a.k; ++r) {
        double m = kNone;
#pragma unroll
        for (int i = 0; i < NPL; ++i) m = max_d(m, c[i]);
        m = lanes_max(m, L);
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (c[i] == m) c[i] = kNone;
        if (ll == r) mine = m;
    }
    const bool picked = mine > kNone;
    const int id = picked ? route_id(mine) : -1;
    if (ll < a.k && !picked) flags |= kRouteFew;
    // weights: of a renormalised softmax relative to the largest that was picked
    const float lp = picked ? route_logit<TYPE>(logits, id) : -__builtin_huge_valf();
    double s = 0.0;
    if (softmax) {
        const float top = a.renormalize ? float(lanes_max(double(lp), L)) : mx;
        s = picked ? soft_mass(lp, top) / (a.renormalize ? 1.0 : total) : 0.0;
    } else if (picked) s = sigmoid_d(lp);
    if (a.renormalize) {
        const double sum = lanes_sum(s, L);
        s = picked ? s / sum : 0.0;
    }
    if (row < a.M && ll < a.k) {
        const size_t to = size_t(row) * a.k + ll;
        a.weights[to] = float(s * a.scale);
        a.ids[to] = id;
        flag_or(a.flags, flags);
    } else if (row < a.M) flag_or(a.flags, flags);
}

int pow2_from(int n) {
    int p = 1;
    while (p < n) p *= 2;
    return p;
}

template <int TYPE, int L> hipError_t route_rows(RouteArgs a, hipStream_t s) {
    a.S = L / pow2_from(a.G);
    const int npl = (a.gs + a.S - 1) / a.S;
    const dim3 grid(unsigned((int64_t(a.M) * L + 255) / 256));
    auto go = [&](auto kernel) { timed_launch("route_experts", kernel, grid, dim3(256), 0, s, a); };
    if (npl <= 1) go(route_kernel<TYPE, L, 1>);
    else if (npl <= 2) go(route_kernel<TYPE, L, 2>);
    else if (npl <= 4) go(route_kernel<TYPE, L, 4>);
    else if (npl <= 8) go(route_kernel<TYPE, L, 8>);
    else if (npl <= 16) go(route_kernel<TYPE, L, 16>);
    else go(route_kernel<TYPE, L, 32>);
    return hipGetLastError();
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
                          int(M - r < kAtOnce ? M - r : kAtOnce), E, G, Gk, k, E / G, 0, score, group_top == 2,
                          renormalize, double(scale)};
        const hipError_t st = logits_type == 2 ? route_rows<2, 64>(a, stream)
                            : logits_type == 1 ? route_rows<1, 64>(a, stream) : route_rows<0, 64>(a, stream);
        if (st != hipSuccess) return st;
    }
    return hipSuccess;
}
