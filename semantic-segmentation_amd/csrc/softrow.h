// One pass over the logits of a row: running maximum, sum of exponentials, sum for the entropy, and the K largest logits.
#pragma once
#include "elem.h"
#include <float.h>
#include <type_traits>

constexpr float SR_LOG2E = 1.4426950408889634f, SR_LN2 = 0.6931471805599453f;
constexpr float SR_FAR = -1000.f;         // stands for any difference whose exponential is 0 (below -150) where the two are multiplied

// Butterfly over neighbouring lanes: the values of the two halves of a group of 2*O lanes whose halves hold one value each.
// Inside 16 lanes by DPP (quad permutes, then the mirrors of half rows and rows: the halves are uniform by then), across them by the row
// swaps of gfx950; an LDS permute instead costs about 100 cycles of latency each, and a top-8 over 64 lanes takes 96 in a row.
template <int O>
__device__ __forceinline__ void halves(int x, int& a, int& b) {
    if (O == 1) { a = x; b = __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, true); }
    else if (O == 2) { a = x; b = __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, true); }
    else if (O == 4) { a = x; b = __builtin_amdgcn_update_dpp(0, x, 0x141, 0xF, 0xF, true); }
    else if (O == 8) { a = x; b = __builtin_amdgcn_update_dpp(0, x, 0x140, 0xF, 0xF, true); }
    else if (O == 16) { const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false); a = r[0]; b = r[1]; }
    else { const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false); a = r[0]; b = r[1]; }
}
template <int O>
__device__ __forceinline__ void halves(float x, float& a, float& b) {
    int i, j;
    halves<O>(__float_as_int(x), i, j);
    a = __int_as_float(i);
    b = __int_as_float(j);
}
// fn<O>() for O = 1, 2, 4 ... LANES/2
template <int LANES, int O = 1, typename F>
__device__ __forceinline__ void butterfly(F&& fn) {
    if constexpr (O < LANES) {
        fn(std::integral_constant<int, O>());
        butterfly<LANES, O * 2>(fn);
    }
}
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
    butterfly<LANES>([&](auto o) { float a, b; halves<decltype(o)::value>(v, a, b); v = fmaxf(a, b); });
    return v;
}
template <int LANES>
__device__ __forceinline__ unsigned lanes_min(unsigned v) {
    butterfly<LANES>([&](auto o) { int a, b; halves<decltype(o)::value>((int)v, a, b); v = min((unsigned)a, (unsigned)b); });
    return v;
}

// With d = (z - m) log2 e:  s = sum 2^d,  t = sum d 2^d.  The running maximum starts at the lowest finite value, so a row of
// nothing but -inf keeps s == 0 and any finite logit makes s >= 1.  A NaN or +inf makes s NaN and nothing takes that back.
struct Soft {
    float m, s, t;
    __device__ __forceinline__ void clear() { m = -FLT_MAX; s = 0.f; t = 0.f; }
    // change of reference: d -> d + D, so s -> s 2^D and t -> (t + D s) 2^D
    __device__ __forceinline__ void shift_to(float mn) {
        const float D = fmaxf((m - mn) * SR_LOG2E, SR_FAR), f = __builtin_amdgcn_exp2f(D);
        t = fmaf(D, s, t) * f;
        s *= f;
        m = mn;
    }
    __device__ __forceinline__ void add(float z) {       // z <= m, or -inf, or NaN
        const float d = (z - m) * SR_LOG2E, e = __builtin_amdgcn_exp2f(d);
        s += e;
        t = fmaf(fmaxf(d, SR_FAR), e, t);
    }
    __device__ __forceinline__ void join(float om, float os, float ot) {
        const float mn = fmaxf(m, om);
        Soft o{om, os, ot};
        o.shift_to(mn);
        shift_to(mn);
        s += o.s;
        t += o.t;
    }
    // over LANES neighbouring lanes, the same bits in all of them
    template <int LANES>
    __device__ __forceinline__ void join_lanes() {
        butterfly<LANES>([&](auto o) {
            constexpr int O = decltype(o)::value;
            Soft b;
            halves<O>(m, m, b.m);
            halves<O>(s, s, b.s);
            halves<O>(t, t, b.t);
            join(b.m, b.s, b.t);
        });
    }
    __device__ __forceinline__ bool empty() const { return s == 0.f; }
    __device__ __forceinline__ float entropy(float log_s) const {
        if (empty()) return 0.f;
        const float h = log_s - SR_LN2 * t / s;
        return h < 0.f ? 0.f : h;                         // keeps a NaN
    }
};

// The instructions themselves: the compiler's forms first quieten their operands, whose bits might be a signalling NaN for all it
// knows.  (A row with a NaN gives no list: whatever the instructions make of it is not used.)
__device__ __forceinline__ float med3(float a, float b, float c) {
    float r;
    asm("v_med3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float larger(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// The K largest, descending; offered in ascending class order, so that of equal ones the lowest class stays in front.
template <int K>
struct Top {
    float v[K > 0 ? K : 1];
    int i[K > 0 ? K : 1];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < K; ++j) { v[j] = -INFINITY; i[j] = -1; }
    }
    __device__ __forceinline__ void offer(float z, int c) {
        bool g[K > 0 ? K : 1];
#pragma unroll
        for (int j = 0; j < K; ++j) g[j] = z > v[j];
#pragma unroll
        for (int j = K - 1; j > 0; --j) {
            i[j] = g[j - 1] ? i[j - 1] : (g[j] ? c : i[j]);
            v[j] = med3(v[j - 1], v[j], z);
        }
        if (K > 0) {
            i[0] = g[0] ? c : i[0];
            v[0] = larger(v[0], z);
        }
    }
    // The K largest of the lists of LANES neighbouring lanes, in every one of them: K times the best head, whose lane moves up.
    template <int LANES>
    __device__ __forceinline__ void join_lanes() {
        Top<K> r;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const float bv = lanes_max<LANES>(v[0]);
            const int bi = (int)lanes_min<LANES>(v[0] == bv ? (unsigned)i[0] : 0xffffffffu);       // -1, no class, is the largest
            const bool mine = bi >= 0 && i[0] == bi;
#pragma unroll
            for (int q = 0; q + 1 < K; ++q) {
                v[q] = mine ? v[q + 1] : v[q];
                i[q] = mine ? i[q + 1] : i[q];
            }
            v[K > 0 ? K - 1 : 0] = mine ? -INFINITY : v[K > 0 ? K - 1 : 0];
            i[K > 0 ? K - 1 : 0] = mine ? -1 : i[K > 0 ? K - 1 : 0];
            r.v[j] = bv;
            r.i[j] = bi;
        }
        *this = r;
    }
};

// log probability of an alternative: NaN in a row without a distribution, -inf where the row has no such class
__device__ __forceinline__ float top_log_p(float v, int i, const Soft& a, float log_s) {
    return a.s != a.s ? a.s : i < 0 ? -INFINITY : (v - a.m) - log_s;
}
__device__ __forceinline__ int64_t top_index(int i, const Soft& a) { return a.s != a.s ? -1 : i; }
