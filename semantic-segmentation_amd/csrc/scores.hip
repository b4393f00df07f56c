// Log probability of a given label, entropy and the most probable classes of every row of a tensor of logits, and the gradient.
//
//   log_p[c] = z[c] - m - log s,  H = log s - (sum (z-m) e^(z-m)) / s,  m = max z, s = sum e^(z-m)
//   dz[c] = a [c == label] + sum_j t_j [c == top_j] - p[c] A - b p[c] (log_p[c] + H),   A = a + sum t_j
//
// Both directions are one pass over the logits and bound by HBM: maximum, sums and the K largest run along with the pass; the
// backward pass gets m, log s and H from the forward pass and never sums.  Two layouts, two kernels each: "rows" (the classes are
// contiguous: a group of lanes shares a row and reads 16 bytes per lane) and "planes" (class stride other than 1, NCHW: a lane owns
// P neighbouring pixels and walks the classes).
//
// Measured (kernel times): 4.2 M pixels of 19 fp32 planes with 3 alternatives 118 us (537 MB, 4.6 TB/s); 2.4 M pixels of 19 bf16 planes forward
// and backward 58 + 60 us (450 MB; the forward pass, with half the bytes in flight per load, 3.0 TB/s); 223729 rows of 150 bf16 classes with 3
// alternatives 32 us (79 MB; vector instructions, 11 of some 20 per class keep the alternatives in order); 8191 rows of 1203 fp32 classes 12 + 18 us.
#include "softrow.h"

namespace {

constexpr int PU = 4;                     // classes a lane has in flight

struct Args {
    dsaspp_scores_desc d;
    int64_t rows, plane;                  // d0*d1*d2, d1*d2
};

struct Row {
    int64_t i0, rem;                      // index along d0, index inside [d1][d2]
    int64_t off;                          // of class 0, in elements
};

__device__ __forceinline__ Row row_of(const Args& a, int64_t row) {
    Row r;
    if (a.plane == 1) {
        r.i0 = row;
        r.rem = 0;
        r.off = row * a.d.s0;
    } else {
        r.i0 = row / a.plane;
        r.rem = row - r.i0 * a.plane;
        const int64_t i1 = r.rem / a.d.d2;
        r.off = r.i0 * a.d.s0 + i1 * a.d.s1 + (r.rem - i1 * a.d.d2) * a.d.s2;
    }
    return r;
}

// class of the row's label, -1 for a row without one
__device__ __forceinline__ int label_of(const dsaspp_scores_desc& d, int64_t row) {
    if (!d.labels) return -1;
    const int64_t l = d.labels[row];
    return l != d.ignore_index && l >= 0 && l < d.n_class ? (int)l : -1;
}

__device__ __forceinline__ float label_log_p(int label, float z, const Soft& s, float log_s) {
    return label < 0 ? 0.f : s.empty() ? -INFINITY : (z - s.m) - log_s;
}

// m and log s for the backward pass; a row with nothing but -inf gets log s = +inf, which makes every p 0
__device__ __forceinline__ void store_stats(float* stats, int64_t row, const Soft& s, float log_s) {
    stats[2 * row] = s.empty() ? 0.f : s.m;
    stats[2 * row + 1] = s.empty() ? INFINITY : log_s;
}

typedef int64_t i64x2u __attribute__((ext_vector_type(2), aligned(8)));
// P neighbouring values of a row tensor (P = 1 or 4), 16 bytes at a time; np < P only at the end of a row of pixels
template <int P>
__device__ __forceinline__ void load_row(const float* p, int np, float (&f)[P]) {
    if (P > 1 && np == P) {
#pragma unroll
        for (int h = 0; h + 3 < P; h += 4) {
            const f32x4u v = *reinterpret_cast<const f32x4u*>(p + h);
#pragma unroll
            for (int k = 0; k < 4; ++k) f[h + k] = v[k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < P; ++k) f[k] = k < np ? p[k] : 0.f;
    }
}
template <int P>
__device__ __forceinline__ void load_row(const int64_t* p, int np, int64_t (&f)[P]) {
    if (P > 1 && np == P) {
#pragma unroll
        for (int h = 0; h + 1 < P; h += 2) {
            const i64x2u v = *reinterpret_cast<const i64x2u*>(p + h);
            f[h] = v[0];
            f[h + 1] = v[1];
        }
    } else {
#pragma unroll
        for (int k = 0; k < P; ++k) f[k] = k < np ? p[k] : 0;
    }
}
template <int P>
__device__ __forceinline__ void store_row(float* p, int np, const float (&f)[P]) {
    if (P > 1 && np == P) {
#pragma unroll
        for (int h = 0; h + 3 < P; h += 4) {
            const f32x4u v = {f[h], f[h + 1], f[h + 2], f[h + 3]};
            *reinterpret_cast<f32x4u*>(p + h) = v;
        }
    } else {
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (k < np) p[k] = f[k];
    }
}
template <int P>
__device__ __forceinline__ void store_row(int64_t* p, int np, const int64_t (&f)[P]) {
    if (P > 1 && np == P) {
#pragma unroll
        for (int h = 0; h + 1 < P; h += 2) {
            const i64x2u v = {f[h], f[h + 1]};
            *reinterpret_cast<i64x2u*>(p + h) = v;
        }
    } else {
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (k < np) p[k] = f[k];
    }
}
template <int P>
__device__ __forceinline__ void load_labels(const dsaspp_scores_desc& d, int64_t row, int np, int (&label)[P]) {
    if (!d.labels) {
#pragma unroll
        for (int q = 0; q < P; ++q) label[q] = -1;
        return;
    }
    int64_t l[P];
    load_row<P>(d.labels + row, np, l);
#pragma unroll
    for (int q = 0; q < P; ++q) label[q] = l[q] != d.ignore_index && l[q] >= 0 && l[q] < d.n_class ? (int)l[q] : -1;
}

// ---------------------------------------------------------------- rows: TPR lanes share a row
// The vector of N classes from c on; returns the class of its first element.  At the end of a row whose length is no multiple of N it
// is the row's last N classes instead, with those before c (another lane's) at -inf: wide loads for rows of any length >= N.
template <int DT>
__device__ __forceinline__ int load_classes(const typename Elem<DT>::T* z, int c, int V, float (&f)[Elem<DT>::N]) {
    typedef Elem<DT> E;
    if (V >= E::N) {
        const int base = c + E::N <= V ? c : V - E::N;
        const typename E::V v = *reinterpret_cast<const typename E::V*>(z + base);
#pragma unroll
        for (int k = 0; k < E::N; ++k) f[k] = base + k >= c ? E::up(v[k]) : -INFINITY;
        return base;
    }
#pragma unroll
    for (int k = 0; k < E::N; ++k) f[k] = k < V ? E::up(z[k]) : -INFINITY;
    return 0;
}

template <int K>
__device__ __forceinline__ void store_outputs(const Args& a, int64_t row, const Row& r, int label, float zl, const Soft& s, const Top<K>& top) {
    const dsaspp_scores_desc& d = a.d;
    const float log_s = logf(s.s);
    if (d.logp) d.logp[row] = label_log_p(label, zl, s, log_s);
    if (d.entropy) d.entropy[row] = s.entropy(log_s);
    if (d.stats) store_stats(d.stats, row, s, log_s);
#pragma unroll
    for (int j = 0; j < K; ++j)
        if (j < d.top_k) {
            const int64_t o = (r.i0 * d.top_k + j) * a.plane + r.rem;
            d.top_logp[o] = top_log_p(top.v[j], top.i[j], s, log_s);
            d.top_class[o] = top_index(top.i[j], s);
        }
}

template <int DT, int K, int TPR>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rows_fwd_kernel(const Args a) {
    typedef Elem<DT> E;
    constexpr int BLOCK = TPR > 256 ? TPR : 256, RPB = BLOCK / TPR, WAVES = TPR > 64 ? TPR / 64 : 1;
    __shared__ float ls[WAVES][3];
    __shared__ float lv[WAVES][K > 0 ? K : 1];
    __shared__ int li[WAVES][K > 0 ? K : 1];
    const dsaspp_scores_desc& d = a.d;
    const int V = d.n_class, lane = threadIdx.x % TPR;
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows; row += (int64_t)gridDim.x * RPB) {
        const Row r = row_of(a, row);
        const typename E::T* z = reinterpret_cast<const typename E::T*>(d.logits) + r.off;
        const int label = label_of(d, row);
        const float zl = label >= 0 ? E::up(z[label]) : 0.f;
        Soft s;
        Top<K> top;
        s.clear();
        top.clear();
        auto take = [&](const float* f, int n, int c) {
            float mx = f[0];
#pragma unroll
            for (int k = 1; k < n; ++k) mx = fmaxf(mx, f[k]);
            if (mx > s.m) s.shift_to(mx);
#pragma unroll
            for (int k = 0; k < n; ++k) {
                s.add(f[k]);
                top.offer(f[k], c + k);
            }
        };
        for (int c = lane * E::N; c < V; c += TPR * E::N) {
            float f[E::N];
            take(f, E::N, load_classes<DT>(z, c, V, f));
        }
        constexpr int G = TPR < 64 ? TPR : 64;
        s.template join_lanes<G>();
        top.template join_lanes<G>();
        if (TPR > 64) {
            const int wave = threadIdx.x >> 6, wl = threadIdx.x & 63;
            __syncthreads();              // the lists of the block's previous row have been read
            if (wl == 0) {
                ls[wave][0] = s.m; ls[wave][1] = s.s; ls[wave][2] = s.t;
#pragma unroll
                for (int j = 0; j < K; ++j) { lv[wave][j] = top.v[j]; li[wave][j] = top.i[j]; }
            }
            __syncthreads();
            if (wave != 0) continue;      // to the next row's first barrier, as wave 0 does after writing
            s.clear();
            top.clear();
            if (wl < WAVES) {
                s = Soft{ls[wl][0], ls[wl][1], ls[wl][2]};
#pragma unroll
                for (int j = 0; j < K; ++j) { top.v[j] = lv[wl][j]; top.i[j] = li[wl][j]; }
            }
            s.template join_lanes<WAVES>();
            top.template join_lanes<WAVES>();
        }
        if (lane == 0) store_outputs(a, row, r, label, zl, s, top);
    }
}

// Few long rows: gridDim.x blocks share a row, each leaving its running values and its K largest; then a wave per row joins them.
// One block of 1024 lanes takes 13.7 us for a row of 21841 bf16 classes, half of it the vector instructions of a single CU.
constexpr int MAX_SPLIT = 64;             // partials of a row, one per lane of the wave that joins them
constexpr int PART = 3 + 2 * DSASPP_SCORES_MAX_TOP;

template <int DT, int K>
__global__ __launch_bounds__(256) void rows_part_kernel(const Args a, const int span) {
    typedef Elem<DT> E;
    __shared__ float ls[4][3];
    __shared__ float lv[4][K > 0 ? K : 1];
    __shared__ int li[4][K > 0 ? K : 1];
    const dsaspp_scores_desc& d = a.d;
    const int64_t row = blockIdx.y;
    const Row r = row_of(a, row);
    const typename E::T* z = reinterpret_cast<const typename E::T*>(d.logits) + r.off;
    const int c0 = blockIdx.x * span, V = min(d.n_class, c0 + span);        // span is a multiple of 256 N: the last block alone is shorter
    Soft s;
    Top<K> top;
    s.clear();
    top.clear();
    for (int c = c0 + threadIdx.x * E::N; c < V; c += 256 * E::N) {
        float f[E::N];
        const int base = load_classes<DT>(z, c, V, f);
        float mx = f[0];
#pragma unroll
        for (int k = 1; k < E::N; ++k) mx = fmaxf(mx, f[k]);
        if (mx > s.m) s.shift_to(mx);
#pragma unroll
        for (int k = 0; k < E::N; ++k) {
            s.add(f[k]);
            top.offer(f[k], base + k);
        }
    }
    s.template join_lanes<64>();
    top.template join_lanes<64>();
    const int wave = threadIdx.x >> 6, wl = threadIdx.x & 63;
    if (wl == 0) {
        ls[wave][0] = s.m; ls[wave][1] = s.s; ls[wave][2] = s.t;
#pragma unroll
        for (int j = 0; j < K; ++j) { lv[wave][j] = top.v[j]; li[wave][j] = top.i[j]; }
    }
    __syncthreads();
    if (wave != 0) return;
    s.clear();
    top.clear();
    if (wl < 4) {
        s = Soft{ls[wl][0], ls[wl][1], ls[wl][2]};
#pragma unroll
        for (int j = 0; j < K; ++j) { top.v[j] = lv[wl][j]; top.i[j] = li[wl][j]; }
    }
    s.template join_lanes<4>();
    top.template join_lanes<4>();
    if (wl == 0) {
        float* o = d.ws + (row * gridDim.x + blockIdx.x) * PART;
        o[0] = s.m; o[1] = s.s; o[2] = s.t;
#pragma unroll
        for (int j = 0; j < K; ++j) { o[3 + 2 * j] = top.v[j]; o[4 + 2 * j] = __int_as_float(top.i[j]); }
    }
}

template <int DT, int K>
__global__ __launch_bounds__(64) void rows_join_kernel(const Args a, const int parts) {
    typedef Elem<DT> E;
    const dsaspp_scores_desc& d = a.d;
    const int64_t row = blockIdx.x;
    const Row r = row_of(a, row);
    const int label = label_of(d, row);
    const float zl = label >= 0 ? E::up(reinterpret_cast<const typename E::T*>(d.logits)[r.off + label]) : 0.f;
    Soft s;
    Top<K> top;
    s.clear();
    top.clear();
    if ((int)threadIdx.x < parts) {
        const float* o = d.ws + (row * parts + threadIdx.x) * PART;
        s = Soft{o[0], o[1], o[2]};
#pragma unroll
        for (int j = 0; j < K; ++j) { top.v[j] = o[3 + 2 * j]; top.i[j] = __float_as_int(o[4 + 2 * j]); }
    }
    s.template join_lanes<64>();
    top.template join_lanes<64>();
    if (threadIdx.x == 0) store_outputs(a, row, r, label, zl, s, top);
}

// what the gradient of one row needs besides its logits
template <int K>
struct Up {
    float m, log_s, h, a, b, A;
    float t[K > 0 ? K : 1];
    int label, top[K > 0 ? K : 1];
    bool live;
    // from the statistics, the label and the upstream gradients; g_top and the alternatives follow one by one
    __device__ __forceinline__ void start(float m_, float log_s_, float h_, int label_, float g_logp, float g_entropy) {
        m = m_;
        log_s = log_s_;
        h = h_;
        label = label_;
        a = label >= 0 ? g_logp : 0.f;
        b = g_entropy;
        A = a;
        live = a != 0.f || b != 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) { t[j] = 0.f; top[j] = -1; }
    }
    __device__ __forceinline__ void add_top(int j, int64_t cls, float g) {
        top[j] = (int)cls;
        // without alternatives because of a NaN: the gradient is NaN unless nothing flows back
        t[j] = cls >= 0 ? g : (log_s != log_s && g != 0.f) ? log_s : 0.f;
        A += t[j];
        live = live || t[j] != 0.f;
    }
    __device__ __forceinline__ void finish() { live = live && log_s != INFINITY; }        // +inf: every class masked out
    __device__ __forceinline__ float grad(float z, int c) const {
        const float lp = (z - m) - log_s, p = __builtin_amdgcn_exp2f(lp * SR_LOG2E);
        float g = -p * fmaf(b, fmaxf(lp, SR_FAR) + h, A);
        if (c == label) g += a;
#pragma unroll
        for (int j = 0; j < K; ++j)
            if (c == top[j]) g += t[j];
        return live ? g : 0.f;
    }
};

// For P neighbouring rows; np < P only at the end of a row of pixels (the rest is dead).
template <int K, int P>
__device__ __forceinline__ void load_up(const dsaspp_scores_desc& d, int64_t plane, int64_t row, int64_t i0, int64_t rem, int np, Up<K> (&u)[P]) {
    int label[P];
    float st[2 * P], h[P], ga[P], gb[P];
    load_labels<P>(d, row, np, label);
    if (P > 1 && np == P) {
#pragma unroll
        for (int h = 0; h + 3 < 2 * P; h += 4) {
            const f32x4u v = *reinterpret_cast<const f32x4u*>(d.stats + 2 * row + h);
#pragma unroll
            for (int k = 0; k < 4; ++k) st[h + k] = v[k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2 * P; ++k) st[k] = k < 2 * np ? d.stats[2 * row + k] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < P; ++q) { h[q] = 0.f; ga[q] = 0.f; gb[q] = 0.f; }
    if (d.g_logp) {
        if (d.g_logp_one) {
#pragma unroll
            for (int q = 0; q < P; ++q) ga[q] = d.g_logp[0];
        } else {
            load_row<P>(d.g_logp + row, np, ga);
        }
    }
    if (d.g_entropy) {
        load_row<P>(d.entropy + row, np, h);
        if (d.g_entropy_one) {
#pragma unroll
            for (int q = 0; q < P; ++q) gb[q] = d.g_entropy[0];
        } else {
            load_row<P>(d.g_entropy + row, np, gb);
        }
    }
#pragma unroll
    for (int q = 0; q < P; ++q) u[q].start(st[2 * q], st[2 * q + 1], h[q], label[q], ga[q], gb[q]);
#pragma unroll
    for (int j = 0; j < K; ++j)
        if (d.g_top && j < d.top_k) {
            const int64_t at = (i0 * d.top_k + j) * plane + rem;
            int64_t cls[P];
            float g[P];
            load_row<P>(d.top_class + at, np, cls);
            if (d.g_top_one) {
#pragma unroll
                for (int q = 0; q < P; ++q) g[q] = d.g_top[0];
            } else {
                load_row<P>(d.g_top + at, np, g);
            }
#pragma unroll
            for (int q = 0; q < P; ++q) u[q].add_top(j, cls[q], g[q]);
        }
#pragma unroll
    for (int q = 0; q < P; ++q) u[q].finish();
}

template <int DT, int K, int TPR>
__global__ __launch_bounds__(256) void rows_bwd_kernel(const Args a) {
    typedef Elem<DT> E;
    constexpr int RPB = 256 / TPR;
    const dsaspp_scores_desc& d = a.d;
    const int V = d.n_class, lane = threadIdx.x % TPR;
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows; row += (int64_t)gridDim.x * RPB) {
        const Row r = row_of(a, row);
        const typename E::T* z = reinterpret_cast<const typename E::T*>(d.logits) + r.off;
        typename E::T* o = reinterpret_cast<typename E::T*>(d.dlogits) + row * V;
        Up<K> us[1];
        load_up<K, 1>(d, a.plane, row, r.i0, r.rem, 1, us);
        const Up<K>& u = us[0];
        for (int c = lane * E::N; c < V; c += TPR * E::N) {
            float f[E::N];
            const int base = load_classes<DT>(z, c, V, f);
            if (base == c && V >= E::N) {
                typename E::V w;
#pragma unroll
                for (int k = 0; k < E::N; ++k) w[k] = E::down(u.grad(f[k], c + k));
                *reinterpret_cast<typename E::V*>(o + c) = w;
            } else {
#pragma unroll
                for (int k = 0; k < E::N; ++k)
                    if (base + k >= c && base + k < V) o[base + k] = E::down(u.grad(f[k], base + k));
            }
        }
    }
}

// ---------------------------------------------------------------- rows of few classes: a lane per row, by way of LDS
// A block's 256 rows are one piece of memory.  It is copied to LDS in 16-byte pieces, every lane takes its row from there (and leaves its
// gradient there), and no lanes have to be joined.  A row of a multiple of 8 classes gets 16 bytes of padding: its 64 lanes would meet in
// few LDS banks, and no 16-byte piece crosses its end.
constexpr int TILE_ROWS = 256, TILE_ROW_BYTES = 128;      // rows of up to 128 bytes: 36 KB of LDS, 4 blocks per CU

template <int DT, bool OUT>
__device__ __forceinline__ void copy_tile(char* tile, typename Elem<DT>::T* g, int total, int V, int stride) {
    typedef Elem<DT> E;
    constexpr int U = 4;
    const int nv = total / E::N, per_row = V / E::N;
    const bool padded = stride != V * (int)sizeof(typename E::T);
    auto place = [&](int i) {
        const int row = padded ? i / per_row : 0;
        return reinterpret_cast<typename E::V*>(tile + (padded ? row * stride + (i - row * per_row) * 16 : i * 16));
    };
    for (int i0 = threadIdx.x; i0 < nv; i0 += U * 256) {
        typename E::V v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * 256 < nv) v[u] = OUT ? *place(i0 + u * 256) : *reinterpret_cast<const typename E::V*>(g + (i0 + u * 256) * E::N);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * 256 < nv) {
                if (OUT) *reinterpret_cast<typename E::V*>(g + (i0 + u * 256) * E::N) = v[u];
                else *place(i0 + u * 256) = v[u];
            }
    }
    const int i = nv * E::N + (int)threadIdx.x;       // only without padding: a padded tile is whole pieces
    if (i < total) {
        if (OUT) g[i] = reinterpret_cast<const typename E::T*>(tile)[i];
        else reinterpret_cast<typename E::T*>(tile)[i] = g[i];
    }
}

template <int DT, int K>
__global__ __launch_bounds__(256) void tile_fwd_kernel(const Args a, const int stride) {
    typedef Elem<DT> E;
    extern __shared__ __attribute__((aligned(16))) char tile[];
    const dsaspp_scores_desc& d = a.d;
    const int V = d.n_class;
    const int64_t row0 = (int64_t)blockIdx.x * TILE_ROWS, row = row0 + threadIdx.x;
    const int n = a.rows - row0 < TILE_ROWS ? (int)(a.rows - row0) : TILE_ROWS;
    const int label = (int)threadIdx.x < n ? label_of(d, row) : -1;
    copy_tile<DT, false>(tile, const_cast<typename E::T*>(reinterpret_cast<const typename E::T*>(d.logits)) + row0 * V, n * V, V, stride);
    __syncthreads();
    if ((int)threadIdx.x >= n) return;
    const typename E::T* z = reinterpret_cast<const typename E::T*>(tile + threadIdx.x * stride);
    Soft s;
    Top<K> top;
    s.clear();
    top.clear();
    int c = 0;
    for (; c + PU <= V; c += PU) {
        float f[PU];
#pragma unroll
        for (int u = 0; u < PU; ++u) f[u] = E::up(z[c + u]);
        float mx = f[0];
#pragma unroll
        for (int u = 1; u < PU; ++u) mx = fmaxf(mx, f[u]);
        if (mx > s.m) s.shift_to(mx);
#pragma unroll
        for (int u = 0; u < PU; ++u) {
            s.add(f[u]);
            top.offer(f[u], c + u);
        }
    }
    for (; c < V; ++c) {
        const float f = E::up(z[c]);
        if (f > s.m) s.shift_to(f);
        s.add(f);
        top.offer(f, c);
    }
    store_outputs(a, row, row_of(a, row), label, label >= 0 ? E::up(z[label]) : 0.f, s, top);
}

template <int DT, int K>
__global__ __launch_bounds__(256) void tile_bwd_kernel(const Args a, const int stride) {
    typedef Elem<DT> E;
    extern __shared__ __attribute__((aligned(16))) char tile[];
    const dsaspp_scores_desc& d = a.d;
    const int V = d.n_class;
    const int64_t row0 = (int64_t)blockIdx.x * TILE_ROWS, row = row0 + threadIdx.x;
    const int n = a.rows - row0 < TILE_ROWS ? (int)(a.rows - row0) : TILE_ROWS;
    copy_tile<DT, false>(tile, const_cast<typename E::T*>(reinterpret_cast<const typename E::T*>(d.logits)) + row0 * V, n * V, V, stride);
    Up<K> u[1];
    if ((int)threadIdx.x < n) {
        const Row r = row_of(a, row);
        load_up<K, 1>(d, a.plane, row, r.i0, r.rem, 1, u);
    }
    __syncthreads();
    if ((int)threadIdx.x < n) {
        typename E::T* z = reinterpret_cast<typename E::T*>(tile + threadIdx.x * stride);
#pragma unroll 4
        for (int c = 0; c < V; ++c) z[c] = E::down(u[0].grad(E::up(z[c]), c));
    }
    __syncthreads();
    copy_tile<DT, true>(tile, reinterpret_cast<typename E::T*>(d.dlogits) + row0 * V, n * V, V, stride);
}

// ---------------------------------------------------------------- planes: a lane owns P neighbouring pixels
// P pixels of one class; np < P only at the end of a row of pixels (lanes past the end hold -inf)
template <int DT, int P>
__device__ __forceinline__ void load_px(const typename Elem<DT>::T* p, int np, float (&f)[P]) {
    typedef Elem<DT> E;
    if (P == 1) {
        f[0] = E::up(p[0]);
    } else if (np == P) {
        const typename E::V4 v = *reinterpret_cast<const typename E::V4*>(p);
#pragma unroll
        for (int k = 0; k < P; ++k) f[k] = E::up(v[k & 3]);
    } else {
#pragma unroll
        for (int k = 0; k < P; ++k) f[k] = k < np ? E::up(p[k]) : -INFINITY;
    }
}

// A class of the plane is one wide load per lane; PU of them are in flight before the first is used.  Bound by HBM.
template <int DT, int K, int P>
__global__ __launch_bounds__(256) void planes_fwd_kernel(const Args a, const int64_t groups, const int64_t per_row) {
    typedef Elem<DT> E;
    const dsaspp_scores_desc& d = a.d;
    const int V = d.n_class;
    for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < groups; g += (int64_t)gridDim.x * 256) {
        const int64_t line = g / per_row, i2 = (g - line * per_row) * P;
        const int64_t row = line * d.d2 + i2;
        const int np = d.d2 - i2 < P ? (int)(d.d2 - i2) : P;
        const Row r = row_of(a, row);
        const typename E::T* z = reinterpret_cast<const typename E::T*>(d.logits) + r.off;
        Soft s[P];
        Top<K> top[P];
        int label[P];
        float zl[P];
        load_labels<P>(d, row, np, label);
#pragma unroll
        for (int q = 0; q < P; ++q) { s[q].clear(); top[q].clear(); zl[q] = 0.f; }
        int c = 0;
        for (; c + PU <= V; c += PU) {
            float f[PU][P];
#pragma unroll
            for (int u = 0; u < PU; ++u) load_px<DT, P>(z + (c + u) * d.sc, np, f[u]);
#pragma unroll
            for (int q = 0; q < P; ++q) {
                float mx = f[0][q];
#pragma unroll
                for (int u = 1; u < PU; ++u) mx = fmaxf(mx, f[u][q]);
                if (mx > s[q].m) s[q].shift_to(mx);
#pragma unroll
                for (int u = 0; u < PU; ++u) {
                    s[q].add(f[u][q]);
                    top[q].offer(f[u][q], c + u);
                    zl[q] = label[q] == c + u ? f[u][q] : zl[q];       // a gather afterwards would touch a line per pixel
                }
            }
        }
        for (; c < V; ++c) {
            float f[P];
            load_px<DT, P>(z + c * d.sc, np, f);
#pragma unroll
            for (int q = 0; q < P; ++q) {
                if (f[q] > s[q].m) s[q].shift_to(f[q]);
                s[q].add(f[q]);
                top[q].offer(f[q], c);
                zl[q] = label[q] == c ? f[q] : zl[q];
            }
        }
        float log_s[P], o[P];
#pragma unroll
        for (int q = 0; q < P; ++q) log_s[q] = logf(s[q].s);
        if (d.logp) {
#pragma unroll
            for (int q = 0; q < P; ++q) o[q] = label_log_p(label[q], zl[q], s[q], log_s[q]);
            store_row<P>(d.logp + row, np, o);
        }
        if (d.entropy) {
#pragma unroll
            for (int q = 0; q < P; ++q) o[q] = s[q].entropy(log_s[q]);
            store_row<P>(d.entropy + row, np, o);
        }
        if (d.stats) {
            float lo[P], hi[P];           // (m, log s) pairs of the first and the second half of the pixels
#pragma unroll
            for (int q = 0; q < P; ++q) {
                float* half = 2 * q < P ? lo : hi;
                half[2 * q % P] = s[q].empty() ? 0.f : s[q].m;
                if (P > 1) half[(2 * q + 1) % P] = s[q].empty() ? INFINITY : log_s[q];
            }
            if (P > 1 && np == P) {
                store_row<P>(d.stats + 2 * row, P, lo);
                store_row<P>(d.stats + 2 * row + P, P, hi);
            } else {
#pragma unroll
                for (int q = 0; q < P; ++q)
                    if (q < np) store_stats(d.stats, row + q, s[q], log_s[q]);
            }
        }
#pragma unroll
        for (int j = 0; j < K; ++j)
            if (j < d.top_k) {
                const int64_t at = (r.i0 * d.top_k + j) * a.plane + r.rem;
                int64_t ti[P];
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    o[q] = top_log_p(top[q].v[j], top[q].i[j], s[q], log_s[q]);
                    ti[q] = top_index(top[q].i[j], s[q]);
                }
                store_row<P>(d.top_logp + at, np, o);
                store_row<P>(d.top_class + at, np, ti);
            }
    }
}

template <int DT, int K, int P>
__global__ __launch_bounds__(256) void planes_bwd_kernel(const Args a, const int64_t groups, const int64_t per_row) {
    typedef Elem<DT> E;
    const dsaspp_scores_desc& d = a.d;
    const int V = d.n_class;
    for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < groups; g += (int64_t)gridDim.x * 256) {
        const int64_t line = g / per_row, i2 = (g - line * per_row) * P;
        const int64_t row = line * d.d2 + i2;
        const int np = d.d2 - i2 < P ? (int)(d.d2 - i2) : P;
        const Row r = row_of(a, row);
        const typename E::T* z = reinterpret_cast<const typename E::T*>(d.logits) + r.off;
        typename E::T* o = reinterpret_cast<typename E::T*>(d.dlogits) + r.i0 * V * a.plane + r.rem;
        Up<K> u[P];
        load_up<K, P>(d, a.plane, row, r.i0, r.rem, np, u);
#pragma unroll PU
        for (int c = 0; c < V; ++c) {
            float f[P];
            load_px<DT, P>(z + c * d.sc, np, f);
#pragma unroll
            for (int q = 0; q < P; ++q) f[q] = u[q].grad(f[q], c);
            typename E::T* oc = o + c * a.plane;
            if (P == 4 && np == P) {
                typename E::V4 w;
#pragma unroll
                for (int q = 0; q < 4; ++q) w[q] = E::down(f[q < P ? q : 0]);
                *reinterpret_cast<typename E::V4*>(oc) = w;
            } else {
#pragma unroll
                for (int q = 0; q < P; ++q)
                    if (q < np) oc[q] = E::down(f[q]);
            }
        }
    }
}

// ---------------------------------------------------------------- host side
int check(const dsaspp_scores_desc* d, const char* who, Args* a) {
    DS_REQUIRE(d, "%s: null descriptor", who);
    DS_REQUIRE(d->dtype >= 0 && d->dtype <= 2, "%s: dtype must be 0 (bf16), 1 (fp32) or 2 (fp16), got %d", who, d->dtype);
    DS_REQUIRE(d->n_class > 0 && d->n_class < (1 << 30), "%s: n_class must be in [1, 2^30)", who);
    DS_REQUIRE(d->top_k >= 0 && d->top_k <= DSASPP_SCORES_MAX_TOP && d->top_k <= d->n_class, "%s: top_k must be in [0, %d] and at most n_class, got %d", who,
               DSASPP_SCORES_MAX_TOP, d->top_k);
    DS_REQUIRE(d->d0 > 0 && d->d1 > 0 && d->d2 > 0 && d->d0 < (1ll << 40) / d->d1 && d->d0 * d->d1 < (1ll << 40) / d->d2, "%s: bad row counts", who);
    DS_REQUIRE(d->s0 >= 0 && d->s1 >= 0 && d->s2 >= 0 && d->sc >= 0, "%s: negative stride", who);
    DS_REQUIRE(d->logits, "%s: null logits", who);
    DS_REQUIRE(((uintptr_t)d->logits & (d->dtype == 1 ? 3 : 1)) == 0, "%s: logits are not aligned to their element type", who);
    a->d = *d;
    a->plane = d->d1 * d->d2;
    a->rows = d->d0 * a->plane;
    return 0;
}

unsigned grid_for(int64_t blocks) { return (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)); }

// Pixels per lane, 4 or 1, where the pixels are contiguous.  Forward and 19 classes of 4.2 M pixels, 1 against 4: without alternatives
// 84 and 82 us (fp32), 48 and 47 (bf16); with one and what the backward pass needs 98 and 104, 88 and 76; with three 113 and 130, 107 and 112;
// with eight 163 and 207, 172 and 247: four lists of alternatives leave too few waves.  And 4 need enough pixels, us with 1 and with 4 without alternatives:
//              9 classes        19             60              150
//   fp32   1 M  13.8  12.5    20.5  18.8    50.0  44.2    132   121
//          2 M  23.6  20.9    36.5  33.9     112   120    245   261
//          4 M  39.5  35.8    84.2  81.6     208   222    467   524
//   bf16   1 M  10.7  10.1    15.3  16.6    30.5  35.1    80.8  104
//          2 M  18.2  19.1    26.5  28.2    64.2  76.3    161   202
//          4 M  32.2  30.1    47.5  46.6     135   141    311   330
// so many classes take 4 only in fp32 and below 2 M.
//
// Backward, 19 classes, one to three alternatives: 262144 pixels 16 against 18 us (fp32) and 10 against 13 (bf16), 400000 pixels 25 and 21, 19 and
// 16, 4.2 M 261 and 184, 180 and 97: writes of 16 or 8 bytes per lane; 150 classes of 4.2 M 1217 and 1156 (fp32), 1034 and 569 (bf16).  8 pixels of a
// 16-bit type per lane were slower at every top_k.
template <int DT, int K, bool BWD>
int px_per_lane(const Args& a) {
    const int64_t least = BWD ? 3 << 17 : DT == 1 ? 1 << 20 : 1 << 21;
    const bool many = !BWD && a.d.n_class > 32 && (DT != 1 || a.rows >= 1 << 21);
    return a.d.s2 == 1 && a.d.d2 >= 4 && (BWD || K <= 1) && a.rows >= least && !many ? 4 : 1;
}

template <int DT, int K, bool BWD>
void launch_planes(const Args& a, hipStream_t s) {
    const int P = px_per_lane<DT, K, BWD>(a);
    const int64_t per_row = (a.d.d2 + P - 1) / P, groups = a.d.d0 * a.d.d1 * per_row;
    const dim3 grid(grid_for((groups + 255) / 256)), block(256);
#define LAUNCH(P) \
    if constexpr (BWD) hipLaunchKernelGGL((planes_bwd_kernel<DT, K, P>), grid, block, 0, s, a, groups, per_row); \
    else hipLaunchKernelGGL((planes_fwd_kernel<DT, K, P>), grid, block, 0, s, a, groups, per_row)
    if constexpr (BWD || K <= 1) {
        if (P == 4) { LAUNCH(4); return; }
    }
    LAUNCH(1);
#undef LAUNCH
}

template <int DT, int K, int TPR, bool BWD>
void launch_rows_tpr(const Args& a, hipStream_t s) {
    constexpr int T = BWD && TPR > 256 ? 256 : TPR, BLOCK = T > 256 ? T : 256, RPB = BLOCK / T;
    const dim3 grid(grid_for((a.rows + RPB - 1) / RPB)), block(BLOCK);
    if constexpr (BWD) hipLaunchKernelGGL((rows_bwd_kernel<DT, K, T>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((rows_fwd_kernel<DT, K, TPR>), grid, block, 0, s, a);
}

// Blocks that share a row in the forward pass (1: none do).  Fewer than 128 rows leave half the CUs without a block; a block
// of a shared row keeps at least one vector per lane.
int row_parts(const dsaspp_scores_desc& d, int64_t rows) {
    const int n = d.dtype == 1 ? 4 : 8;
    if (d.sc != 1 || rows >= 128 || d.n_class < 4 * 256 * n) return 1;
    const int64_t most = d.n_class / (256 * n), want = 512 / rows;
    return (int)(most < want ? (most < MAX_SPLIT ? most : MAX_SPLIT) : (want < MAX_SPLIT ? want : MAX_SPLIT));
}
int part_span(const dsaspp_scores_desc& d, int parts) {        // classes of a part: whole rounds of the block, so that parts cover the row
    const int unit = 256 * (d.dtype == 1 ? 4 : 8), per = (d.n_class + parts - 1) / parts;
    return (per + unit - 1) / unit * unit;
}

// Lanes per row: 4 hold the lane butterflies and the ends of rows cheap (150 classes: 32 us with 4, 57 with 16, 183 with 64 for 223729 rows);
// more only as long as the rows are too few to fill the chip, and every lane keeps a vector (1203 classes, 8191 rows: 41 us with 4,
// 14 with 16, 12 with 64, 20 with 256).
//
// The backward pass joins nothing, and its writes gain from longer pieces per row: a vector per lane of 16 or 64 wherever there is one
// (150 classes: 103 us with 16 against 145 with 4; 1203 classes: 88 with 64, 97 with 16 and with 256; forward and backward pass).
template <int DT, int K, bool BWD>
void launch_rows(const Args& a, hipStream_t s) {
    const dsaspp_scores_desc& d = a.d;
    const int size = DT == 1 ? 4 : 2;
    const bool dense = (d.d2 == 1 || d.s2 == d.n_class) && (d.d1 == 1 || d.s1 == d.d2 * d.n_class) && (d.d0 == 1 || d.s0 == a.plane * d.n_class);
    // A lane per row by way of LDS from two blocks per CU on (a grid has fewer than 2^32 lanes).  19 fp32 classes, 3 alternatives, forward and backward:
    // 8192 rows 12.1 us against 9.1 with lanes sharing rows, 65536 rows 13.8 and 13.1, 1 M rows 70 and 116.
    if (dense && d.n_class * size <= TILE_ROW_BYTES && a.rows >= 512 * TILE_ROWS && a.rows < (1ll << 31)) {
        const int stride = d.n_class * size + (d.n_class % 8 == 0 ? 16 : 0);
        const dim3 grid((unsigned)((a.rows + TILE_ROWS - 1) / TILE_ROWS)), block(TILE_ROWS);
        if constexpr (BWD) hipLaunchKernelGGL((tile_bwd_kernel<DT, K>), grid, block, TILE_ROWS * stride, s, a, stride);
        else hipLaunchKernelGGL((tile_fwd_kernel<DT, K>), grid, block, TILE_ROWS * stride, s, a, stride);
        return;
    }
    if constexpr (!BWD) {
        const int parts = row_parts(a.d, a.rows);
        if (parts > 1) {
            const int span = part_span(a.d, parts), used = (a.d.n_class + span - 1) / span;
            hipLaunchKernelGGL((rows_part_kernel<DT, K>), dim3(used, (unsigned)a.rows), dim3(256), 0, s, a, span);
            hipLaunchKernelGGL((rows_join_kernel<DT, K>), dim3((unsigned)a.rows), dim3(64), 0, s, a, used);
            return;
        }
    }
    const int64_t vecs = (d.n_class + Elem<DT>::N - 1) / Elem<DT>::N;
    int tpr = BWD ? (vecs >= 128 ? 64 : vecs >= 16 ? 16 : 4) : 4;
    while (tpr < 1024 && tpr * 4 <= vecs && a.rows * tpr < 256 * 1024) tpr *= 4;
    if (tpr == 4) launch_rows_tpr<DT, K, 4, BWD>(a, s);
    else if (tpr == 16) launch_rows_tpr<DT, K, 16, BWD>(a, s);
    else if (tpr == 64) launch_rows_tpr<DT, K, 64, BWD>(a, s);
    else if (tpr == 256) launch_rows_tpr<DT, K, 256, BWD>(a, s);
    else launch_rows_tpr<DT, K, 1024, BWD>(a, s);
}

template <int DT, bool BWD>
void launch_k(const Args& a, int k, hipStream_t s) {
    const bool rows = a.d.sc == 1 || a.d.n_class == 1;
#define LAUNCH(K) rows ? launch_rows<DT, K, BWD>(a, s) : launch_planes<DT, K, BWD>(a, s)
    if (k == 0) LAUNCH(0);
    else if (k == 1) LAUNCH(1);
    else if (k <= 3) LAUNCH(3);
    else if (k <= 5) LAUNCH(5);
    else LAUNCH(8);
#undef LAUNCH
}

}  // namespace

extern "C" int64_t dsaspp_scores_workspace(const dsaspp_scores_desc* d) {
    Args a;
    if (check(d, "scores_workspace", &a)) return -1;
    const int parts = row_parts(*d, a.rows);
    return parts > 1 ? a.rows * parts * PART : 0;
}

extern "C" int dsaspp_scores_fwd(const dsaspp_scores_desc* d, dsaspp_stream_t stream) {
    Args a;
    if (int rc = check(d, "scores_fwd", &a)) return rc;
    DS_REQUIRE(!d->logp || d->labels, "scores_fwd: logp needs labels");
    DS_REQUIRE((d->top_k > 0) == (d->top_logp != nullptr) && (d->top_k > 0) == (d->top_class != nullptr), "scores_fwd: top_logp and top_class go with top_k > 0");
    DS_REQUIRE(d->logp || d->entropy || d->stats || d->top_k, "scores_fwd: nothing to compute");
    const int parts = row_parts(*d, a.rows);
    DS_REQUIRE(parts == 1 || (d->ws && ((uintptr_t)d->ws & 3) == 0 && d->ws_len >= a.rows * parts * PART), "scores_fwd: the workspace needs %lld floats",
               (long long)(a.rows * parts * PART));
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == 0) launch_k<0, false>(a, d->top_k, s);
    else if (d->dtype == 1) launch_k<1, false>(a, d->top_k, s);
    else launch_k<2, false>(a, d->top_k, s);
    DS_LAUNCH_CHECK("scores_fwd");
    return 0;
}

extern "C" int dsaspp_scores_bwd(const dsaspp_scores_desc* d, dsaspp_stream_t stream) {
    Args a;
    if (int rc = check(d, "scores_bwd", &a)) return rc;
    DS_REQUIRE(d->stats && d->dlogits, "scores_bwd: null stats or gradient");
    DS_REQUIRE(((uintptr_t)d->dlogits & (d->dtype == 1 ? 3 : 1)) == 0, "scores_bwd: dlogits is not aligned to its element type");
    DS_REQUIRE(d->g_logp || d->g_entropy || d->g_top, "scores_bwd: no upstream gradient");
    DS_REQUIRE(!d->g_logp || d->labels, "scores_bwd: g_logp needs labels");
    DS_REQUIRE(!d->g_entropy || d->entropy, "scores_bwd: g_entropy needs the entropy of the forward pass");
    DS_REQUIRE(!d->g_top || (d->top_k > 0 && d->top_class), "scores_bwd: g_top needs top_class of the forward pass");
    hipStream_t s = (hipStream_t)stream;
    const int k = d->g_top ? d->top_k : 0;
    if (d->dtype == 0) launch_k<0, true>(a, k, s);
    else if (d->dtype == 1) launch_k<1, true>(a, k, s);
    else launch_k<2, true>(a, k, s);
    DS_LAUNCH_CHECK("scores_bwd");
    return 0;
}
