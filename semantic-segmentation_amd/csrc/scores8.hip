// Class scores of logits at 1/8 resolution with the bilinear x8 upsample fused in (align_corners=False), and their gradient.
//
//   z[c] = hy r0[c] + ly r1[c],  r_i[c] = hx L[yi][x0][c] + lx L[yi][x1][c]     every product and sum rounded by itself
//   log_p, H, top as in scores.hip;  dL = adjoint of the interpolation of dz
//
// The full-resolution logits (76 bytes per pixel at 19 classes) never exist: a pixel costs its label and its outputs in HBM
// traffic and its classes in vector arithmetic, which is the bound.  As in the fused loss a lane owns one output column of a "cell" --
// the 8 x 8 output pixels that interpolate between the same four low-resolution pixels -- and walks its 8 rows with the
// x-interpolated corner rows in registers.  A block owns 8 x 4 cells and reads their 9 x 5 corner pixels once, into LDS.
// The backward pass leaves the sums of every block's 9 x 5 corner pixels in a workspace and a second kernel adds the one to four
// blocks that meet in a pixel (more on the border) in a fixed order: no atomics, equal inputs give equal bits.
#include "softrow.h"

namespace {

constexpr int TCX = 8, TCY = 4, PX = TCX + 1, PY = TCY + 1;
constexpr int NC_MAX = 32;

// Source coordinate of output index o as torch computes it: src = max(0.125*(o+0.5)-0.5, 0), i0 = floor(src), l1 = src - i0.
__device__ __forceinline__ void src_index(int o, int n, int& i0, int& i1, float& l1) {
    float s = 0.125f * ((float)o + 0.5f) - 0.5f;      // exact: multiples of 1/16
    s = fmaxf(s, 0.f);
    i0 = (int)s;
    i1 = i0 + (i0 < n - 1 ? 1 : 0);
    l1 = s - (float)i0;
}

__device__ __forceinline__ float mix(float h, float a, float l, float b) {
#pragma clang fp contract(off)
    return h * a + l * b;
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
    if (dtype == 1) return reinterpret_cast<const float*>(p)[i];
    const u16 x = reinterpret_cast<const u16*>(p)[i];
    return dtype == 0 ? Elem<0>::up(x) : Elem<2>::up(x);
}

struct Tile {
    int n, ci0, cj0;                                  // image, first cell column and row
    __device__ __forceinline__ Tile(int tile, int tiles_x, int tiles_y) {
        const int bx = tile % tiles_x, t = tile / tiles_x;
        n = t / tiles_y;
        ci0 = bx * TCX;
        cj0 = (t - n * tiles_y) * TCY;
    }
};

// The corner pixels of the tile's cells, fp32, CS floats apart; cell (i, j) of the tile has its corners at (j..j+1, i..i+1).
template <int CS>
__device__ __forceinline__ void stage(const dsaspp_scores8_desc& d, const Tile& t, float* corner) {
    const int nc = d.n_class, total = PX * PY * nc;
    const int64_t base = (int64_t)t.n * d.sn;
    const bool inner = d.sc == 1;                     // the fastest index of the walk is the contiguous one
    for (int i = threadIdx.x; i < total; i += 256) {
        int c, px, py;
        if (inner) {
            c = i % nc;
            const int p = i / nc;
            px = p % PX; py = p / PX;
        } else {
            px = i % PX;
            const int p = i / PX;
            py = p % PY; c = p / PY;
        }
        const int y = min(max(t.cj0 - 1 + py, 0), d.h - 1), x = min(max(t.ci0 - 1 + px, 0), d.w - 1);
        corner[(py * PX + px) * CS + c] = load_any(d.logits, base + y * d.sy + x * d.sx + c * d.sc, d.dtype);
    }
    __syncthreads();
}

// One output column: which it is, its weights and the LDS addresses of its four corners.
struct Column {
    int X, cj, py, px;
    bool ok;
    float lx, hx;
    int o00, o01, o10, o11;
    __device__ __forceinline__ Column(const dsaspp_scores8_desc& d, const Tile& t, int cs) {
        const int lane8 = threadIdx.x & 7;
        px = (threadIdx.x >> 3) & (TCX - 1);
        py = threadIdx.x >> 6;
        cj = t.cj0 + py;
        X = 8 * (t.ci0 + px) - 4 + lane8;
        ok = cj <= d.h && X >= 0 && X < 8 * d.w;
        int x0, x1;
        src_index(max(X, 0), d.w, x0, x1, lx);
        hx = 1.f - lx;
        // left of the first pixel's centre the first corner is the pixel itself: LDS column 1 of the first tile, as column 0
        const int c0 = min(max(x0 - (t.ci0 - 1), 0), PX - 1), c1 = min(max(x1 - (t.ci0 - 1), 0), PX - 1);
        int y0, y1;
        float l;
        src_index(max(8 * cj - 4, 0), d.h, y0, y1, l);
        const int r0 = min(max(y0 - (t.cj0 - 1), 0), PY - 1), r1 = min(max(y1 - (t.cj0 - 1), 0), PY - 1);
        o00 = (r0 * PX + c0) * cs; o01 = (r0 * PX + c1) * cs;
        o10 = (r1 * PX + c0) * cs; o11 = (r1 * PX + c1) * cs;
    }
};

template <int NC, bool EXACT, int K>
__global__ __launch_bounds__(256) void scores8_fwd_kernel(const dsaspp_scores8_desc d, const int tiles_x, const int tiles_y) {
    constexpr int CS = NC | 1;
    __shared__ float corner[PX * PY * CS];
    const Tile tl(blockIdx.x, tiles_x, tiles_y);
    stage<CS>(d, tl, corner);
    const Column q(d, tl, CS);
    if (!q.ok) return;
    const int nc = EXACT ? NC : d.n_class, H = 8 * d.h, W = 8 * d.w;
    float r0[NC], r1[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        r0[c] = mix(q.hx, corner[q.o00 + c], q.lx, corner[q.o01 + c]);
        r1[c] = mix(q.hx, corner[q.o10 + c], q.lx, corner[q.o11 + c]);
    }
    const int64_t image = (int64_t)tl.n * H * W;
    for (int r = 0; r < 8; ++r) {
        const int Y = 8 * q.cj - 4 + r;
        if (Y < 0 || Y >= H) continue;
        int y0, y1;
        float ly;
        src_index(Y, d.h, y0, y1, ly);
        const float hy = 1.f - ly;
        float z[NC];
        Top<K> top;
        top.clear();
        Soft s;
        s.clear();
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            z[c] = mix(hy, r0[c], ly, r1[c]);
            if (!EXACT) z[c] = c < nc ? z[c] : -INFINITY;
            s.m = fmaxf(s.m, z[c]);
            top.offer(z[c], c);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) s.add(z[c]);
        const float log_s = logf(s.s);
        const int64_t pix = (int64_t)Y * W + q.X;
        if (d.logp) {
            const int64_t l = d.labels[image + pix];
            const bool has = l != d.ignore_index && l >= 0 && l < nc;
            const int lc = has ? (int)l : 0;
            const float a = mix(q.hx, corner[q.o00 + lc], q.lx, corner[q.o01 + lc]);
            const float b = mix(q.hx, corner[q.o10 + lc], q.lx, corner[q.o11 + lc]);
            d.logp[image + pix] = !has ? 0.f : s.empty() ? -INFINITY : (mix(hy, a, ly, b) - s.m) - log_s;
        }
        if (d.entropy) d.entropy[image + pix] = s.entropy(log_s);
#pragma unroll
        for (int j = 0; j < K; ++j)
            if (j < d.top_k) {
                const int64_t o = ((int64_t)tl.n * d.top_k + j) * H * W + pix;
                d.top_logp[o] = top_log_p(top.v[j], top.i[j], s, log_s);
                d.top_class[o] = top_index(top.i[j], s);
            }
    }
}

__device__ __forceinline__ float row8_sum(float v) {
    // sum over the 8 lanes of a cell (an aligned 8-lane group inside a DPP row), result in every lane
    int x = __float_as_int(v);
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, true));    // quad_perm [1,0,3,2]
    x = __float_as_int(v);
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, true));    // quad_perm [2,3,0,1]
    x = __float_as_int(v);
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x141, 0xF, 0xF, true));   // row_half_mirror
    return v;
}

// HB: an upstream gradient of the entropy is there.  Per pixel and class  dz = 2^d (k0 + k1 d)  with d = (z - m) log2 e and per-pixel
// k0, k1; what falls on the label and on the alternatives is added to lane-private LDS columns instead of being selected by class.
template <int NC, bool EXACT, bool HB>
__global__ __launch_bounds__(256) void scores8_bwd_kernel(const dsaspp_scores8_desc d, const int tiles_x, const int tiles_y) {
    constexpr int CS = NC | 1, CELLS = TCX * TCY, KS = CELLS * CS;
    __shared__ float corner[PX * PY * CS];
    __shared__ float oh[2 * NC * 256];                // [corner row][class][lane]
    __shared__ float ct[4 * KS];                      // [corner][cell][class]
    const int tid = threadIdx.x, nc = EXACT ? NC : d.n_class, H = 8 * d.h, W = 8 * d.w;
    const Tile tl(blockIdx.x, tiles_x, tiles_y);
#pragma unroll
    for (int c = 0; c < 2 * NC; ++c) oh[c * 256 + tid] = 0.f;
    stage<CS>(d, tl, corner);
    const Column q(d, tl, CS);
    float g0[NC], g1[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) { g0[c] = 0.f; g1[c] = 0.f; }
    if (q.ok) {
        float r0[NC], r1[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            r0[c] = mix(q.hx, corner[q.o00 + c], q.lx, corner[q.o01 + c]);
            r1[c] = mix(q.hx, corner[q.o10 + c], q.lx, corner[q.o11 + c]);
        }
        const int64_t image = (int64_t)tl.n * H * W;
        for (int r = 0; r < 8; ++r) {
            const int Y = 8 * q.cj - 4 + r;
            if (Y < 0 || Y >= H) continue;
            int y0, y1;
            float ly;
            src_index(Y, d.h, y0, y1, ly);
            const float hy = 1.f - ly;
            const int64_t pix = (int64_t)Y * W + q.X;
            const float b = HB ? d.g_entropy[d.g_entropy_one ? 0 : image + pix] : 0.f;
            float a = 0.f, A;
            int label = -1;
            if (d.g_logp) {
                const int64_t l = d.labels[image + pix];
                if (l != d.ignore_index && l >= 0 && l < nc) {
                    label = (int)l;
                    a = d.g_logp[d.g_logp_one ? 0 : image + pix];
                }
            }
            A = a;
            bool live = a != 0.f || b != 0.f;
            if (d.g_top)
                for (int j = 0; j < d.top_k; ++j) {
                    const int64_t o = ((int64_t)tl.n * d.top_k + j) * H * W + pix;
                    const float g = d.g_top[d.g_top_one ? 0 : o];
                    live = live || g != 0.f;
                    if (d.top_class[o] >= 0) A += g;
                }
            if (!live) continue;
            float z[NC];
            Soft s;
            s.clear();
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                z[c] = mix(hy, r0[c], ly, r1[c]);
                if (!EXACT) z[c] = c < nc ? z[c] : -INFINITY;
                s.m = fmaxf(s.m, z[c]);
            }
            float e[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                z[c] = (z[c] - s.m) * SR_LOG2E;
                e[c] = __builtin_amdgcn_exp2f(z[c]);
                s.s += e[c];
                if (HB) {
                    z[c] = fmaxf(z[c], SR_FAR);
                    s.t = fmaf(z[c], e[c], s.t);
                }
            }
            if (s.empty()) continue;                  // every class masked out
            const float inv = 1.f / s.s;
            // log_p + H = (d ln2 - log s) + (log s - ln2 t / s) = ln2 (d - t / s)
            const float k1 = HB ? -b * SR_LN2 * inv : 0.f;
            const float k0 = HB ? -A * inv - k1 * (s.t * inv) : -A * inv;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float g = HB ? e[c] * fmaf(k1, z[c], k0) : e[c] * k0;
                g0[c] = fmaf(hy, g, g0[c]);
                g1[c] = fmaf(ly, g, g1[c]);
            }
            if (label >= 0) {
                oh[label * 256 + tid] += a * hy;
                oh[(NC + label) * 256 + tid] += a * ly;
            }
            if (d.g_top)
                for (int j = 0; j < d.top_k; ++j) {
                    const int64_t o = ((int64_t)tl.n * d.top_k + j) * H * W + pix;
                    const int64_t tc = d.top_class[o];
                    if (tc >= 0 && tc < nc) {
                        const float g = d.g_top[d.g_top_one ? 0 : o];
                        oh[(int)tc * 256 + tid] += g * hy;
                        oh[(NC + (int)tc) * 256 + tid] += g * ly;
                    }
                }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            g0[c] += oh[c * 256 + tid];
            g1[c] += oh[(NC + c) * 256 + tid];
        }
    }
    // the 8 columns of a cell together: corner (y, x0) gets the hx-weighted, (y, x1) the lx-weighted sum
    const int cell = tid >> 3, lane8 = tid & 7;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const float a00 = row8_sum(q.hx * g0[c]), a01 = row8_sum(q.lx * g0[c]);
        const float a10 = row8_sum(q.hx * g1[c]), a11 = row8_sum(q.lx * g1[c]);
        if ((c & 7) == lane8) {                       // cells outside the image store their zeros
            ct[0 * KS + cell * CS + c] = a00;
            ct[1 * KS + cell * CS + c] = a01;
            ct[2 * KS + cell * CS + c] = a10;
            ct[3 * KS + cell * CS + c] = a11;
        }
    }
    __syncthreads();
    // corner pixel (py, px) of the tile is corner 00 of cell (py, px), 01 of (py, px-1), 10 of (py-1, px), 11 of (py-1, px-1)
    float* out = d.ws + (int64_t)blockIdx.x * (PX * PY) * nc;
    for (int i = tid; i < PX * PY * nc; i += 256) {
        const int c = i % nc, p = i / nc, py = p / PX, px = p - py * PX;
        float v = 0.f;
        if (py < TCY && px < TCX) v += ct[0 * KS + (py * TCX + px) * CS + c];
        if (py < TCY && px > 0) v += ct[1 * KS + (py * TCX + px - 1) * CS + c];
        if (py > 0 && px < TCX) v += ct[2 * KS + ((py - 1) * TCX + px) * CS + c];
        if (py > 0 && px > 0) v += ct[3 * KS + ((py - 1) * TCX + px - 1) * CS + c];
        out[i] = v;
    }
}

// Positions along one axis whose sums belong to source pixel i of n: (tile, place in the tile), at most 6.  A cell stands for the
// pixels before clamping; what falls on -1 or n belongs to the border pixel.
template <int TC>
__device__ __forceinline__ int places(int i, int n, int tiles, int (&tile)[6], int (&at)[6]) {
    int k = 0;
#pragma unroll
    for (int e = -1; e <= 1; ++e) {                   // e = 0: the pixel itself; -1, 1: beyond the border
        if ((e < 0 && i != 0) || (e > 0 && i != n - 1)) continue;
        const int u = i + e + 1, b = u / TC, o = u - b * TC;
        if (b < tiles) { tile[k] = b; at[k] = o; ++k; }
        if (o == 0 && b > 0) { tile[k] = b - 1; at[k] = TC; ++k; }
    }
    return k;
}

__global__ __launch_bounds__(256) void scores8_gather_kernel(const dsaspp_scores8_desc d, const int tiles_x, const int tiles_y, const int64_t total) {
    const bool inner = d.gc == 1;
    for (int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x; idx < total; idx += (int64_t)gridDim.x * 256) {
        int64_t t = idx;
        int c, x, y;
        if (inner) {
            c = (int)(t % d.n_class); t /= d.n_class;
            x = (int)(t % d.w); t /= d.w;
            y = (int)(t % d.h); t /= d.h;
        } else {
            x = (int)(t % d.w); t /= d.w;
            y = (int)(t % d.h); t /= d.h;
            c = (int)(t % d.n_class); t /= d.n_class;
        }
        const int64_t n = t;
        int tx[6], ax[6], ty[6], ay[6];
        const int kx = places<TCX>(x, d.w, tiles_x, tx, ax), ky = places<TCY>(y, d.h, tiles_y, ty, ay);
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < 6; ++j)
#pragma unroll
            for (int i = 0; i < 6; ++i)
                if (j < ky && i < kx) v += d.ws[(((n * tiles_y + ty[j]) * tiles_x + tx[i]) * (PX * PY) + ay[j] * PX + ax[i]) * d.n_class + c];
        const int64_t o = n * d.gn + y * d.gy + x * d.gx + c * d.gc;
        if (d.g_dtype == 1) reinterpret_cast<float*>(d.dlogits)[o] = v;
        else reinterpret_cast<u16*>(d.dlogits)[o] = d.g_dtype == 0 ? Elem<0>::down(v) : Elem<2>::down(v);
    }
}

int check(const dsaspp_scores8_desc* d, const char* who, int* tx, int* ty, int64_t* tiles) {
    DS_REQUIRE(d, "%s: null descriptor", who);
    DS_REQUIRE(d->n_img > 0 && d->h > 0 && d->w > 0 && d->h < (1 << 20) && d->w < (1 << 20), "%s: bad geometry", who);
    DS_REQUIRE(d->n_class > 0 && d->n_class <= NC_MAX, "%s: n_class must be in [1, %d], got %d", who, NC_MAX, d->n_class);
    DS_REQUIRE(d->top_k >= 0 && d->top_k <= DSASPP_SCORES_MAX_TOP && d->top_k <= d->n_class, "%s: top_k must be in [0, %d] and at most n_class, got %d", who,
               DSASPP_SCORES_MAX_TOP, d->top_k);
    DS_REQUIRE(d->dtype >= 0 && d->dtype <= 2, "%s: dtype must be 0 (bf16), 1 (fp32) or 2 (fp16), got %d", who, d->dtype);
    DS_REQUIRE(d->sn >= 0 && d->sy >= 0 && d->sx >= 0 && d->sc >= 0, "%s: negative stride", who);
    *tx = (d->w + 1 + TCX - 1) / TCX;
    *ty = (d->h + 1 + TCY - 1) / TCY;
    *tiles = (int64_t)d->n_img * *tx * *ty;
    DS_REQUIRE(*tiles < (1ll << 31), "%s: too many pixels", who);
    return 0;
}

int check_logits(const dsaspp_scores8_desc* d, const char* who) {
    DS_REQUIRE(d->logits && ((uintptr_t)d->logits & (d->dtype == 1 ? 3 : 1)) == 0, "%s: logits are null or not aligned to their element type", who);
    return 0;
}

template <int NC, bool EX>
void launch_fwd(const dsaspp_scores8_desc& d, int tx, int ty, unsigned grid, hipStream_t s) {
#define LAUNCH(K) hipLaunchKernelGGL((scores8_fwd_kernel<NC, EX, K>), dim3(grid), dim3(256), 0, s, d, tx, ty)
    if (d.top_k == 0) LAUNCH(0);
    else if (d.top_k == 1) LAUNCH(1);
    else if (d.top_k <= 3) LAUNCH(3);
    else LAUNCH(8);
#undef LAUNCH
}

template <int NC, bool EX>
void launch_bwd(const dsaspp_scores8_desc& d, int tx, int ty, unsigned grid, hipStream_t s) {
    if (d.g_entropy) hipLaunchKernelGGL((scores8_bwd_kernel<NC, EX, true>), dim3(grid), dim3(256), 0, s, d, tx, ty);
    else hipLaunchKernelGGL((scores8_bwd_kernel<NC, EX, false>), dim3(grid), dim3(256), 0, s, d, tx, ty);
}

}  // namespace

// Cityscapes' 19 classes have their own instantiation, every other count the next multiple of 8: the class loops are unrolled
// registers, and the range checks of the inexact ones cost a select per class.
#define BY_CLASSES(F)                                        \
    if (d->n_class == 19) F(19, true);                       \
    else if (d->n_class <= 8) F(8, false);                   \
    else if (d->n_class <= 16) F(16, false);                 \
    else if (d->n_class <= 24) F(24, false);                 \
    else F(32, false)

extern "C" int dsaspp_scores8_fwd(const dsaspp_scores8_desc* d, dsaspp_stream_t stream) {
    int tx, ty;
    int64_t tiles;
    if (int rc = check(d, "scores8_fwd", &tx, &ty, &tiles)) return rc;
    if (int rc = check_logits(d, "scores8_fwd")) return rc;
    DS_REQUIRE(!d->logp || d->labels, "scores8_fwd: logp needs labels");
    DS_REQUIRE((d->top_k > 0) == (d->top_logp != nullptr) && (d->top_k > 0) == (d->top_class != nullptr), "scores8_fwd: top_logp and top_class go with top_k > 0");
    DS_REQUIRE(d->logp || d->entropy || d->top_k, "scores8_fwd: nothing to compute");
#define F(NC, EX) launch_fwd<NC, EX>(*d, tx, ty, (unsigned)tiles, (hipStream_t)stream)
    BY_CLASSES(F);
#undef F
    DS_LAUNCH_CHECK("scores8_fwd");
    return 0;
}

extern "C" int64_t dsaspp_scores8_workspace(const dsaspp_scores8_desc* d) {
    int tx, ty;
    int64_t tiles;
    if (check(d, "scores8_workspace", &tx, &ty, &tiles)) return -1;
    return tiles * (PX * PY) * d->n_class;
}

extern "C" int dsaspp_scores8_bwd(const dsaspp_scores8_desc* d, dsaspp_stream_t stream) {
    int tx, ty;
    int64_t tiles;
    if (int rc = check(d, "scores8_bwd", &tx, &ty, &tiles)) return rc;
    if (int rc = check_logits(d, "scores8_bwd")) return rc;
    DS_REQUIRE(d->g_logp || d->g_entropy || d->g_top, "scores8_bwd: no upstream gradient");
    DS_REQUIRE(!d->g_logp || d->labels, "scores8_bwd: g_logp needs labels");
    DS_REQUIRE(!d->g_top || (d->top_k > 0 && d->top_class), "scores8_bwd: g_top needs top_class of the forward pass");
    DS_REQUIRE(d->g_dtype >= 0 && d->g_dtype <= 2, "scores8_bwd: g_dtype must be 0 (bf16), 1 (fp32) or 2 (fp16), got %d", d->g_dtype);
    DS_REQUIRE(d->dlogits && ((uintptr_t)d->dlogits & (d->g_dtype == 1 ? 3 : 1)) == 0, "scores8_bwd: dlogits is null or not aligned to its element type");
    DS_REQUIRE(d->gn >= 0 && d->gy > 0 && d->gx > 0 && d->gc > 0, "scores8_bwd: bad gradient strides");
    DS_REQUIRE(d->ws && ((uintptr_t)d->ws & 3) == 0 && d->ws_len >= tiles * (PX * PY) * d->n_class, "scores8_bwd: the workspace needs %lld floats",
               (long long)(tiles * (PX * PY) * d->n_class));
    hipStream_t s = (hipStream_t)stream;
#define F(NC, EX) launch_bwd<NC, EX>(*d, tx, ty, (unsigned)tiles, s)
    BY_CLASSES(F);
#undef F
    const int64_t total = (int64_t)d->n_img * d->h * d->w * d->n_class;
    int64_t nb = (total + 255) / 256;
    if (nb > (1 << 20)) nb = 1 << 20;
    hipLaunchKernelGGL(scores8_gather_kernel, dim3((unsigned)nb), dim3(256), 0, s, *d, tx, ty, total);
    DS_LAUNCH_CHECK("scores8_bwd");
    return 0;
}
