// Global gradient norm over many tensors, clipping by it, and the Adam update with the clip coefficient applied on the fly.
//
//   norm = scale * sqrt(sum g^2) (or scale * max |g|),  coef = min(1, max_norm / (norm + 1e-6)),  g <- g * coef
//
// Bound by HBM: the norm reads every gradient once, the second pass reads and writes it.  Two launches per call: the first
// leaves one fp64 partial per block, and every block of the second adds up the same partials in the same order and so knows
// the coefficient without a third launch, an atomic or a flag.
//
// Measured (kernel times): norm of 35.4 M fp32 elements alone 27 us, of 200 M bf16 elements 77 us (5.2 TB/s); 46 and 124 us right after the
// scaling or the update of the pass before, whose writes are leaving the caches meanwhile.  Scaling 51 us (284 MB) and 131 (800 MB); the
// Adam update of 35.4 M parameters with bf16 copy 183 to 196 us after the norm (1.06 GB, 5.4 to 5.8 TB/s).
#include "elem.h"
#include <math.h>
#include <algorithm>
#include <new>
#include <utility>
#include <vector>

namespace {

// Elements of one range that a block takes at a time: small ones spread few elements over more CUs (a launch of 100 tensors with 1.1 M
// elements: norm 5.4 us against 7.2 with chunks of 8192), lists of 35 and 200 M elements show no difference.
constexpr int CHUNK = 4096;
// 8 blocks of 4 waves per CU fill the chip; a block takes several chunks in a row.  With 4096 blocks the scaling of 200 M elements takes 139 us
// against 132, with 8192 171: each adds up all partials.
constexpr int MAX_BLOCKS = 2048;
// The ranges of one launch travel in its kernel arguments (4.0 of 4 KB), ten bytes each: 32 bits of distance from the first range, in
// elements, 32 bits of length and 16 bits of first chunk.  24 bytes each made three launches of what fits one; a launch costs the host 3 us.
constexpr int MAX_RANGES = 400;
constexpr int MAX_CHUNKS = 65535;         // of one launch
constexpr int64_t MAX_LENGTH = (int64_t)(MAX_CHUNKS / 2) * CHUNK;       // of one range; longer ones are several
constexpr int64_t MAX_ELEMS = (int64_t)1 << 42;

struct Group {
    char* base;
    int32_t at[MAX_RANGES];               // in elements from base
    uint32_t n[MAX_RANGES];
    uint16_t first[MAX_RANGES + 1];       // first chunk of range i
    int32_t n_ranges;
};
static_assert(sizeof(Group) <= 4032, "kernel arguments beside it: workspace, counts, threshold, result");

// Last range whose first chunk is <= chunk: every lane compares some, all loads at once.
__device__ __forceinline__ int find_range(const Group& g, int chunk) {
    const int lane = threadIdx.x & 63;
    int r = 0;
#pragma unroll
    for (int k = 0; k < MAX_RANGES; k += 64) {
        const int i = k + lane;
        r += __popcll(__ballot(i > 0 && i < g.n_ranges && (int)g.first[i < MAX_RANGES ? i : MAX_RANGES] <= chunk));
    }
    return r;
}

// Consecutive chunks of this block: the range is looked up once.  Every block has at least one (the grid has no more blocks).
struct Share { int first, last; };
__device__ __forceinline__ Share share_of(int n_chunks) {
    const int q = n_chunks / (int)gridDim.x, rest = n_chunks - q * (int)gridDim.x, b = blockIdx.x;
    const int first = b * q + (b < rest ? b : rest);
    return {first, first + q + (b < rest ? 1 : 0)};
}

// max that keeps a NaN (fmax drops it)
__device__ __forceinline__ double max_nan(double a, double b) { return (b > a || b != b) ? b : a; }

template <bool MAXNORM>
__device__ __forceinline__ double join(double a, double b) { return MAXNORM ? (a != a ? a : max_nan(a, b)) : a + b; }

// The same value in every lane of the block; a fixed order of additions.  `lds`: 4 doubles.
template <bool MAXNORM>
__device__ __forceinline__ double block_join(double v, double* lds) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = join<MAXNORM>(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return join<MAXNORM>(join<MAXNORM>(lds[0], lds[1]), join<MAXNORM>(lds[2], lds[3]));
}

template <int DT, bool MAXNORM>
__global__ __launch_bounds__(256) void partials_kernel(const Group g, double* ws) {
    typedef Elem<DT> E;
    __shared__ double lds[4];
    const int n_chunks = g.first[g.n_ranges];
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    auto take = [&](int k, float x) {
        if (MAXNORM) acc[k] = join<true>(acc[k], (double)fabsf(x));
        else acc[k] = __builtin_fma((double)x, (double)x, acc[k]);      // the product is exact: 24 + 24 bits
    };
    const Share sh = share_of(n_chunks);
    int r = find_range(g, sh.first);
    for (int ch = sh.first; ch < sh.last; ++ch) {
        while (ch >= g.first[r + 1]) ++r;
        const uint32_t off = (uint32_t)(ch - g.first[r]) * CHUNK, left = g.n[r] - off;
        const int n = left < CHUNK ? (int)left : CHUNK;
        const typename E::T* p = reinterpret_cast<const typename E::T*>(g.base) + g.at[r] + off;
        constexpr int IT = CHUNK / E::N / 256;                  // loads in flight before the first is used
        int i = threadIdx.x * E::N;
        for (; i + ((IT - 1) * 256 + 1) * E::N <= n; i += IT * 256 * E::N) {
            typename E::V v[IT];
#pragma unroll
            for (int it = 0; it < IT; ++it) v[it] = *reinterpret_cast<const typename E::V*>(p + i + it * 256 * E::N);
#pragma unroll
            for (int it = 0; it < IT; ++it)
#pragma unroll
                for (int k = 0; k < E::N; ++k) take(k & 3, E::up(v[it][k]));
        }
        for (; i + E::N <= n; i += 256 * E::N) {
            const typename E::V v = *reinterpret_cast<const typename E::V*>(p + i);
#pragma unroll
            for (int k = 0; k < E::N; ++k) take(k & 3, E::up(v[k]));
        }
        const int t = n / E::N * E::N + (int)threadIdx.x;
        if (t < n) take(0, E::up(p[t]));                                // fewer than one vector is left
    }
    const double v = join<MAXNORM>(join<MAXNORM>(acc[0], acc[1]), join<MAXNORM>(acc[2], acc[3]));
    const double s = block_join<MAXNORM>(v, lds);
    if (threadIdx.x == 0) ws[blockIdx.x] = s;
}

// The norm from the partials of all launches: lane t adds partials t, t + 256, ...; the same in every block.
template <bool MAXNORM>
__device__ __forceinline__ double total_norm(const double* ws, int n, float scale, double* lds) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) v = join<MAXNORM>(v, ws[i]);
    v = block_join<MAXNORM>(v, lds);
    return (double)scale * (MAXNORM ? v : sqrt(v));
}

__device__ __forceinline__ double clip_coef(double norm, float max_norm) {
    // an infinite threshold never clips (inf / inf would be NaN); a NaN norm stays NaN
    if (norm == norm && max_norm == INFINITY) return 1.0;
    const double c = (double)max_norm / (norm + 1e-6);
    return c > 1.0 ? 1.0 : c;
}

// A factor for fp32 values, rounded once to 24 bits: below 2^-100 in two, as one it would lose its last bits as a denormal (a norm of 1e39
// clipped to 1) while the values it multiplies are large.
struct Factor {
    float a, b;
    __device__ __forceinline__ explicit Factor(double c) {
        const bool small = c < 0x1p-100;                  // false for NaN
        a = (float)(small ? c * 0x1p100 : c);
        b = small ? 0x1p-100f : 1.f;
    }
    __device__ __forceinline__ float times(float x) const { return x * a * b; }
    __device__ __forceinline__ bool one() const { return a == 1.f && b == 1.f; }
};

__device__ __forceinline__ double any_norm(const double* ws, int n, int norm_type, float scale, double* lds) {
    return norm_type == 2 ? total_norm<false>(ws, n, scale, lds) : total_norm<true>(ws, n, scale, lds);
}

__global__ __launch_bounds__(256) void finish_kernel(const double* ws, int n, int norm_type, float scale, float* norm) {
    __shared__ double lds[4];
    const double v = any_norm(ws, n, norm_type, scale, lds);
    if (threadIdx.x == 0) norm[0] = (float)v;
}

template <int DT>
__global__ __launch_bounds__(256) void scale_kernel(const Group g, const double* ws, int n_ws, int norm_type, float max_norm, float* norm) {
    typedef Elem<DT> E;
    __shared__ double lds[4];
    const double total = any_norm(ws, n_ws, norm_type, 1.f, lds);
    if (blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)total;
    const Factor coef(clip_coef(total, max_norm));
    if (coef.one()) return;               // x * 1 is x
    const int n_chunks = g.first[g.n_ranges];
    const Share sh = share_of(n_chunks);
    int r = find_range(g, sh.last - 1);
    for (int ch = sh.last - 1; ch >= sh.first; --ch) {                  // backwards: what the norm read last is still in the cache
        while (ch < g.first[r]) --r;
        const uint32_t off = (uint32_t)(ch - g.first[r]) * CHUNK, left = g.n[r] - off;
        const int n = left < CHUNK ? (int)left : CHUNK;
        typename E::T* p = reinterpret_cast<typename E::T*>(g.base) + g.at[r] + off;
        constexpr int IT = CHUNK / E::N / 512;
        int i = threadIdx.x * E::N;
        for (; i + ((IT - 1) * 256 + 1) * E::N <= n; i += IT * 256 * E::N) {
            typename E::V v[IT];
#pragma unroll
            for (int it = 0; it < IT; ++it) v[it] = *reinterpret_cast<const typename E::V*>(p + i + it * 256 * E::N);
#pragma unroll
            for (int it = 0; it < IT; ++it) {
#pragma unroll
                for (int k = 0; k < E::N; ++k) v[it][k] = E::down(coef.times(E::up(v[it][k])));
                *reinterpret_cast<typename E::V*>(p + i + it * 256 * E::N) = v[it];
            }
        }
        for (; i + E::N <= n; i += 256 * E::N) {
            typename E::V* q = reinterpret_cast<typename E::V*>(p + i);
            typename E::V v = *q;
#pragma unroll
            for (int k = 0; k < E::N; ++k) v[k] = E::down(coef.times(E::up(v[k])));
            *q = v;
        }
        const int t = n / E::N * E::N + (int)threadIdx.x;
        if (t < n) p[t] = E::down(coef.times(E::up(p[t])));
    }
}

struct AdamArgs {
    int64_t n;
    float* p; const float* g; float* m; float* v;
    u16* w16;
    float lr1, beta1, beta1c, beta2, beta2c, bc2s, eps, weight_decay;      // lr / bias correction 1, 1 - beta, sqrt(bias correction 2)
};

// Adam with coupled L2, as torch.optim.Adam(weight_decay=...), on g * scale * coef.
__global__ __launch_bounds__(256) void adam_clipped_kernel(const AdamArgs d, const double* ws, int n_ws, int norm_type, float scale, float max_norm,
                                                           float* norm) {
    __shared__ double lds[4];
    const double total = any_norm(ws, n_ws, norm_type, scale, lds);
    if (blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)total;
    const Factor gs((double)scale * clip_coef(total, max_norm));
    auto update = [&](float& p, const float gr, float& m, float& v) {
        const float g = gs.times(gr) + d.weight_decay * p;
        m = d.beta1 * m + d.beta1c * g;
        v = d.beta2 * v + d.beta2c * g * g;
        p -= d.lr1 * (m / (sqrtf(v) / d.bc2s + d.eps));
    };
    u16* w16 = d.w16;
    const int64_t nv = d.n / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nv; i += (int64_t)gridDim.x * 256) {
        f32x4u* qp = reinterpret_cast<f32x4u*>(d.p) + i;
        f32x4u* qm = reinterpret_cast<f32x4u*>(d.m) + i;
        f32x4u* qv = reinterpret_cast<f32x4u*>(d.v) + i;
        f32x4u p = *qp, m = *qm, v = *qv;
        const f32x4u g = *(reinterpret_cast<const f32x4u*>(d.g) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float pk = p[k], mk = m[k], vk = v[k];
            update(pk, g[k], mk, vk);
            p[k] = pk; m[k] = mk; v[k] = vk;
        }
        *qp = p; *qm = m; *qv = v;
        if (w16) {
            typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(2)));
            u32x2u o;
            o[0] = pack_bf2(p[0], p[1]);
            o[1] = pack_bf2(p[2], p[3]);
            *reinterpret_cast<u32x2u*>(w16 + i * 4) = o;
        }
    }
    const int64_t t = nv * 4 + threadIdx.x;
    if (blockIdx.x == 0 && t < d.n) {
        update(d.p[t], d.g[t], d.m[t], d.v[t]);
        if (w16) w16[t] = (u16)f2bf_bits(d.p[t]);
    }
}

int blocks_for(int64_t chunks) { return (int)(chunks < MAX_BLOCKS ? chunks : MAX_BLOCKS); }

// Order in which the ranges are walked: as given while all of them are within reach of each other (32 bits of distance in elements of 2
// bytes), else by address, so that a launch ends where the next 4 GiB begin and not wherever the list jumps there and back.
struct Order {
    std::vector<int32_t> by_address;      // empty: as given
    int operator[](int i) const { return by_address.empty() ? i : by_address[i]; }
    // lo, hi: of the ranges' addresses; sorted: they ascend
    int make(const dsaspp_clip_desc& d, const char* who, uintptr_t lo, uintptr_t hi, bool sorted) {
        if (sorted || hi - lo < (1ull << 32)) return 0;
        try {
            by_address.resize(d.n_ranges);
        } catch (const std::bad_alloc&) {
            return dsaspp_set_error("%s: out of host memory", who);
        }
        for (int i = 0; i < d.n_ranges; ++i) by_address[i] = i;
        auto at = [&](int i) { return (uintptr_t)d.ranges[i].p; };
        std::sort(by_address.begin(), by_address.end(), [&](int a, int b) { return at(a) < at(b) || (at(a) == at(b) && a < b); });
        return 0;
    }
};

// Calls fn(dtype, group) for every launch the ranges need: up to MAX_RANGES ranges of one type each.  A range that begins where
// the one before it ends goes on with it: gradients that are views of one arena.
template <typename F>
void for_each_group(const dsaspp_clip_desc& d, const Order& order, F fn) {
    for (int dt = 0; dt < 3; ++dt) {
        const int64_t size = dt == 1 ? 4 : 2;
        Group g;
        int64_t chunks = 0;               // of the ranges in g
        const char* end = nullptr;
        g.n_ranges = 0;
        g.first[0] = 0;
        auto flush = [&]() {
            if (g.n_ranges) fn(dt, g);
            g.n_ranges = 0;
            chunks = 0;
            end = nullptr;
        };
        for (int i = 0; i < d.n_ranges; ++i) {
            const dsaspp_grad_range& range = d.ranges[order[i]];
            if (range.dtype != dt) continue;
            char* p = (char*)range.p;
            for (int64_t left = range.n; left > 0;) {
                const int64_t n = left < MAX_LENGTH ? left : MAX_LENGTH, more = (n + CHUNK - 1) / CHUNK;
                const int k = g.n_ranges - 1;
                if (k >= 0 && end == p && g.n[k] + n <= MAX_LENGTH && chunks + more <= MAX_CHUNKS) {
                    g.n[k] += (uint32_t)n;
                    chunks = g.first[k] + ((int64_t)g.n[k] + CHUNK - 1) / CHUNK;
                    g.first[k + 1] = (uint16_t)chunks;
                } else {
                    const int64_t at = k >= 0 ? (p - g.base) / size : 0;
                    // a distance that is no whole number of elements or needs more than 32 bits starts a launch of its own
                    if (g.n_ranges == MAX_RANGES || chunks + more > MAX_CHUNKS || (k >= 0 && ((p - g.base) % size != 0 || at != (int32_t)at))) flush();
                    if (g.n_ranges == 0) g.base = p;
                    g.at[g.n_ranges] = (int32_t)((p - g.base) / size);
                    g.n[g.n_ranges] = (uint32_t)n;
                    chunks += more;
                    g.first[++g.n_ranges] = (uint16_t)chunks;
                }
                p += n * size;
                end = p;
                left -= n;
            }
        }
        flush();
    }
}

int check(const dsaspp_clip_desc* d, const char* who, Order* order = nullptr) {
    DS_REQUIRE(d, "%s: null descriptor", who);
    DS_REQUIRE(d->n_ranges >= 0 && (d->n_ranges == 0 || d->ranges), "%s: bad list of ranges", who);
    DS_REQUIRE(d->norm_type == 2 || d->norm_type == 0, "%s: norm_type must be 2 (Euclidean) or 0 (largest magnitude), got %d", who, d->norm_type);
    DS_REQUIRE(d->scale > 0.f && d->scale < INFINITY, "%s: scale must be positive and finite", who);
    uintptr_t lo = UINTPTR_MAX, hi = 0, last = 0;
    bool sorted = true;
    for (int i = 0; i < d->n_ranges; ++i) {
        const dsaspp_grad_range& r = d->ranges[i];
        const uintptr_t p = (uintptr_t)r.p;
        lo = std::min(lo, p);
        hi = std::max(hi, p);
        sorted = sorted && p >= last;
        last = p;
        DS_REQUIRE(r.dtype >= 0 && r.dtype <= 2, "%s: range %d has dtype %d (0 = bf16, 1 = fp32, 2 = fp16)", who, i, r.dtype);
        DS_REQUIRE(r.p && r.n > 0 && r.n <= MAX_ELEMS, "%s: range %d is empty, too long or null", who, i);
        DS_REQUIRE(((uintptr_t)r.p & (r.dtype == 1 ? 3 : 1)) == 0, "%s: range %d is not aligned to its element type", who, i);
    }
    return order ? order->make(*d, who, lo, hi, sorted) : 0;
}

int64_t n_partials(const dsaspp_clip_desc& d, const Order& order) {
    int64_t n = 0;
    for_each_group(d, order, [&](int, const Group& g) { n += blocks_for(g.first[g.n_ranges]); });
    return n;
}

int check_used(const dsaspp_clip_desc* d, const char* who, int64_t used) {
    DS_REQUIRE(used < (1ll << 31), "%s: too many ranges", who);
    DS_REQUIRE(used == 0 || (d->ws && d->ws_len >= used && ((uintptr_t)d->ws & 7) == 0), "%s: the workspace needs %lld doubles", who, (long long)used);
    return 0;
}

int check_ws(const dsaspp_clip_desc* d, const char* who, Order* order, int64_t* used) {
    if (int rc = check(d, who, order)) return rc;
    *used = n_partials(*d, *order);
    return check_used(d, who, *used);
}

void launch_partials(const dsaspp_clip_desc& d, const Order& order, hipStream_t s) {
    double* ws = d.ws;
    for_each_group(d, order, [&](int dt, const Group& g) {
        const int nb = blocks_for(g.first[g.n_ranges]);
#define PARTIALS(DT)                                                                                                       \
        if (d.norm_type == 2) hipLaunchKernelGGL((partials_kernel<DT, false>), dim3(nb), dim3(256), 0, s, g, ws);          \
        else hipLaunchKernelGGL((partials_kernel<DT, true>), dim3(nb), dim3(256), 0, s, g, ws)
        if (dt == 0) { PARTIALS(0); } else if (dt == 1) { PARTIALS(1); } else { PARTIALS(2); }
#undef PARTIALS
        ws += nb;
    });
}

void launch_scale(const dsaspp_clip_desc& d, const Order& order, int used, hipStream_t s) {
    for_each_group(d, order, [&](int dt, const Group& g) {
        const int nb = blocks_for(g.first[g.n_ranges]);
        if (dt == 0) hipLaunchKernelGGL(scale_kernel<0>, dim3(nb), dim3(256), 0, s, g, d.ws, used, d.norm_type, d.max_norm, d.norm);
        else if (dt == 1) hipLaunchKernelGGL(scale_kernel<1>, dim3(nb), dim3(256), 0, s, g, d.ws, used, d.norm_type, d.max_norm, d.norm);
        else hipLaunchKernelGGL(scale_kernel<2>, dim3(nb), dim3(256), 0, s, g, d.ws, used, d.norm_type, d.max_norm, d.norm);
    });
}

// Norm and scaling of a few gradients in one block, without the second launch.  A range costs the block two trips to memory and 1024
// elements some 0.3 us: 8000 elements in 8 ranges take 6.9 us a pass against 9.9 us with two launches, 20000 take 10.4 against 10.2,
// 7000 in 30 ranges 14.4 against 11.
constexpr int64_t ONE_BLOCK = 8192;       // elements
constexpr int ONE_BLOCK_RANGES = 8;

template <int DT>
__global__ __launch_bounds__(1024) void clip_one_kernel(const Group g, int norm_type, float max_norm, float* norm) {
    typedef Elem<DT> E;
    __shared__ double lds[16];
    double acc = 0.0;
    for (int r = 0; r < g.n_ranges; ++r) {
        const typename E::T* p = reinterpret_cast<const typename E::T*>(g.base) + g.at[r];
        const int n = (int)g.n[r];
        for (int i = threadIdx.x; i < n; i += 1024) {
            const float x = E::up(p[i]);
            acc = norm_type == 2 ? __builtin_fma((double)x, (double)x, acc) : join<true>(acc, (double)fabsf(x));
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double other = __shfl_xor(acc, o, 64);
        acc = norm_type == 2 ? acc + other : join<true>(acc, other);
    }
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = acc;
    __syncthreads();                      // also: every element has been read before any is written
    acc = lds[0];
#pragma unroll
    for (int w = 1; w < 16; ++w) acc = norm_type == 2 ? acc + lds[w] : join<true>(acc, lds[w]);
    const double total = norm_type == 2 ? sqrt(acc) : acc;
    if (threadIdx.x == 0) norm[0] = (float)total;
    const Factor coef(clip_coef(total, max_norm));
    if (coef.one()) return;
    for (int r = 0; r < g.n_ranges; ++r) {
        typename E::T* p = reinterpret_cast<typename E::T*>(g.base) + g.at[r];
        const int n = (int)g.n[r];
        for (int i = threadIdx.x; i < n; i += 1024) p[i] = E::down(coef.times(E::up(p[i])));
    }
}

}  // namespace

extern "C" int dsaspp_grad_ranges_overlap(const dsaspp_clip_desc* d) {
    if (check(d, "grad_ranges_overlap")) return -1;
    std::vector<std::pair<uintptr_t, uintptr_t>> v;
    try {
        v.reserve(d->n_ranges);
    } catch (const std::bad_alloc&) {
        dsaspp_set_error("grad_ranges_overlap: out of host memory");
        return -1;
    }
    for (int i = 0; i < d->n_ranges; ++i) {
        const uintptr_t p = (uintptr_t)d->ranges[i].p;
        v.emplace_back(p, p + (uintptr_t)d->ranges[i].n * (d->ranges[i].dtype == 1 ? 4 : 2));
    }
    if (!std::is_sorted(v.begin(), v.end())) std::sort(v.begin(), v.end());
    for (size_t i = 1; i < v.size(); ++i)
        if (v[i].first < v[i - 1].second) return 1;
    return 0;
}

extern "C" int64_t dsaspp_grad_norm_workspace(const dsaspp_clip_desc* d) {
    Order order;
    if (check(d, "grad_norm_workspace", &order)) return -1;
    return n_partials(*d, order);
}

extern "C" int dsaspp_grad_norm_partials(const dsaspp_clip_desc* d, dsaspp_stream_t stream) {
    int64_t used = 0;
    Order order;
    if (int rc = check_ws(d, "grad_norm_partials", &order, &used)) return rc;
    launch_partials(*d, order, (hipStream_t)stream);
    DS_LAUNCH_CHECK("grad_norm_partials");
    return 0;
}

extern "C" int dsaspp_grad_norm_finish(const dsaspp_clip_desc* d, dsaspp_stream_t stream) {
    int64_t used = 0;
    Order order;
    if (int rc = check_ws(d, "grad_norm_finish", &order, &used)) return rc;
    DS_REQUIRE(d->norm, "grad_norm_finish: null output");
    hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, d->ws, (int)used, d->norm_type, d->scale, d->norm);
    DS_LAUNCH_CHECK("grad_norm_finish");
    return 0;
}

extern "C" int dsaspp_clip_scale(const dsaspp_clip_desc* d, dsaspp_stream_t stream) {
    int64_t used = 0;
    Order order;
    if (int rc = check_ws(d, "clip_scale", &order, &used)) return rc;
    DS_REQUIRE(d->norm, "clip_scale: null output");
    DS_REQUIRE(d->scale == 1.f, "clip_scale: scale must be 1");
    DS_REQUIRE(d->max_norm >= 0.f, "clip_scale: max_norm must be >= 0");
    if (d->n_ranges == 0) return dsaspp_grad_norm_finish(d, stream);
    launch_scale(*d, order, (int)used, (hipStream_t)stream);
    DS_LAUNCH_CHECK("clip_scale");
    return 0;
}

extern "C" int dsaspp_clip_grads(const dsaspp_clip_desc* d, dsaspp_stream_t stream) {
    Order order;
    if (int rc = check(d, "clip_grads", &order)) return rc;
    DS_REQUIRE(d->norm && d->scale == 1.f && d->max_norm >= 0.f, "clip_grads: null output, scale other than 1 or negative max_norm");
    int64_t total = 0, used = 0;
    int groups = 0, ranges = 0;
    for_each_group(*d, order, [&](int, const Group& g) {
        ++groups;
        ranges += g.n_ranges;
        used += blocks_for(g.first[g.n_ranges]);
        for (int i = 0; i < g.n_ranges; ++i) total += g.n[i];
    });
    if (int rc = check_used(d, "clip_grads", used)) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (groups == 0) return dsaspp_grad_norm_finish(d, stream);
    if (groups == 1 && ranges <= ONE_BLOCK_RANGES && total <= ONE_BLOCK) {
        for_each_group(*d, order, [&](int dt, const Group& g) {
            if (dt == 0) hipLaunchKernelGGL(clip_one_kernel<0>, dim3(1), dim3(1024), 0, s, g, d->norm_type, d->max_norm, d->norm);
            else if (dt == 1) hipLaunchKernelGGL(clip_one_kernel<1>, dim3(1), dim3(1024), 0, s, g, d->norm_type, d->max_norm, d->norm);
            else hipLaunchKernelGGL(clip_one_kernel<2>, dim3(1), dim3(1024), 0, s, g, d->norm_type, d->max_norm, d->norm);
        });
    } else {
        launch_partials(*d, order, s);
        launch_scale(*d, order, (int)used, s);
    }
    DS_LAUNCH_CHECK("clip_grads");
    return 0;
}

extern "C" int dsaspp_adam_step_clipped(const dsaspp_adam_clip_desc* a, const dsaspp_clip_desc* c, dsaspp_stream_t stream) {
    int64_t used = 0;
    Order order;
    DS_REQUIRE(a && a->n > 0 && a->n <= MAX_ELEMS, "adam_step_clipped: n must be positive");
    DS_REQUIRE(a->p && a->g && a->m && a->v && a->step >= 1, "adam_step_clipped: bad descriptor");
    DS_REQUIRE((((uintptr_t)a->p | (uintptr_t)a->g | (uintptr_t)a->m | (uintptr_t)a->v) & 3) == 0 && ((uintptr_t)a->w16 & 1) == 0,
               "adam_step_clipped: buffers must be aligned to their element type");
    if (int rc = check_ws(c, "adam_step_clipped", &order, &used)) return rc;
    DS_REQUIRE(c->norm && c->max_norm >= 0.f, "adam_step_clipped: null output or negative max_norm");
    const AdamArgs d = {a->n, a->p, a->g, a->m, a->v, reinterpret_cast<u16*>(a->w16),
                        (float)(a->lr / (1.0 - pow(a->beta1, (double)a->step))), (float)a->beta1, (float)(1.0 - a->beta1), (float)a->beta2,
                        (float)(1.0 - a->beta2), (float)sqrt(1.0 - pow(a->beta2, (double)a->step)), (float)a->eps, (float)a->weight_decay};
    int64_t nb = (a->n / 4 + 255) / 256;
    nb = nb < 1 ? 1 : nb > MAX_BLOCKS ? MAX_BLOCKS : nb;
    hipLaunchKernelGGL(adam_clipped_kernel, dim3((unsigned)nb), dim3(256), 0, (hipStream_t)stream, d, c->ws, (int)used, c->norm_type, c->scale,
                       c->max_norm, c->norm);
    DS_LAUNCH_CHECK("adam_step_clipped");
    return 0;
}
