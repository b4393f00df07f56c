// Class scores of logits at 1/8 resolution with the bilinear x8 upsample fused in (align_corners=False), and their gradient.
//
//   z[c] = hy r0[c] + ly r1[c],  r_i[c] = hx L[yi][x0][c] + lx L[yi][x1][c]     every product and sum rounded by itself
//   log_p, H, top as in scores.hip;  dL = adjoint of the interpolation of dz
//
// The full-resolution logits (76 bytes per pixel at 19 classes) never exist: a pixel costs its label and its outputs in HBM
// traffic and its classes in vector arithmetic, which is the bound.  As in the fused loss a lane owns one output column of a "cell" --
// the 8 x 8 output pixels that interpolate between the same four low-resolution pixels -- and walks its 8 rows with the
// x-interpolated corner rows in registers.  A block owns 8 x 4 cells and reads their 9 x 5 corner pixels once, into LDS; in the forward
// pass, which joins no lanes, its 64 columns begin at a multiple of 64 instead (10 x 5 corner pixels), so that a wave writes whole
// lines: 131 us against 144 at four pictures of 1024 x 2048, 19 classes, 3 alternatives.
//
// Measured there: 134 us, 446 MB, 3.3 TB/s.  Training with an entropy term, eight such pictures: 110 us forward (340 MB), 163 backward (400 MB)
// and 22 for the joining kernel; the vector units are busy 71 % and 85 % of the time.
// The backward pass leaves the sums of every block's 9 x 5 corner pixels in a workspace and a second kernel adds the one to four
// blocks that meet in a pixel (more on the border) in a fixed order: no atomics, equal inputs give equal bits.
#include "softrow.h"

namespace {

constexpr int TCX = 8, TCY = 4, PX = TCX + 1, PY = TCY + 1;
constexpr int PXF = PX + 1;               // of the forward pass, whose 64 columns begin at a multiple of 64: half a cell, seven, half a cell
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
// Returns the largest magnitude among them, NaN counting as the largest, for the whole block.  Lanes are dealt so that a lane computes
// one address and steps from there, all loads before the first use: with a division and two 64-bit products per load staging took an
// eighth of the block's vector instructions.
template <int CS, int PX, int DT>
__device__ __forceinline__ unsigned stage_typed(const dsaspp_scores8_desc& d, const Tile& t, float* corner) {
    typedef Elem<DT> E;
    const typename E::T* L = reinterpret_cast<const typename E::T*>(d.logits) + (int64_t)t.n * d.sn;
    const int nc = d.n_class;
    unsigned big = 0;
    auto line = [&](int py) { return min(max(t.cj0 - 1 + py, 0), d.h - 1) * d.sy; };
    auto column = [&](int px) { return min(max(t.ci0 - 1 + px, 0), d.w - 1) * d.sx; };
    auto keep = [&](float* to, typename E::T raw) {
        const float v = E::up(raw);
        big = max(big, __float_as_uint(v) & 0x7fffffffu);       // ordered as the magnitudes are, NaN above infinity
        *to = v;
    };
    if (d.sc == 1) {                                  // 32 lanes per pixel, 8 pixels of a line at a time; the rest of every line at the end
        const int c = threadIdx.x & 31, k8 = threadIdx.x >> 5;
        if (c < nc) {
            const bool last = k8 < PY;
            const typename E::T* from = L + column(k8) + c;
            typename E::T v[PY], w[PX - 8] = {};
#pragma unroll
            for (int py = 0; py < PY; ++py) v[py] = from[line(py)];
#pragma unroll
            for (int px = 8; px < PX; ++px)
                if (last) w[px - 8] = L[line(k8) + column(px) + c];
            float* to = corner + k8 * CS + c;
#pragma unroll
            for (int py = 0; py < PY; ++py) keep(to + py * PX * CS, v[py]);
#pragma unroll
            for (int px = 8; px < PX; ++px)
                if (last) keep(corner + (k8 * PX + px) * CS + c, w[px - 8]);
        }
    } else {                                          // a lane per pixel and fifth class
        constexpr int STEP = 5, IT = (CS + STEP - 1) / STEP;
        static_assert(STEP * PX * PY <= 256, "lanes of a block");
        const int c0 = threadIdx.x / (PX * PY), p = threadIdx.x - c0 * (PX * PY), py = p / PX;
        if (c0 < STEP) {
            const typename E::T* from = L + line(py) + column(p - py * PX) + c0 * d.sc;
            typename E::T v[IT];
#pragma unroll
            for (int k = 0; k < IT; ++k)
                if (c0 + k * STEP < nc) v[k] = from[k * STEP * d.sc];
            float* to = corner + p * CS + c0;
#pragma unroll
            for (int k = 0; k < IT; ++k)
                if (c0 + k * STEP < nc) keep(to + k * STEP, v[k]);
        }
    }
    return big;
}

template <int CS, int PX>
__device__ __forceinline__ float stage(const dsaspp_scores8_desc& d, const Tile& t, float* corner, unsigned* largest) {
    unsigned big;
    if (d.dtype == 1) big = stage_typed<CS, PX, 1>(d, t, corner);
    else if (d.dtype == 0) big = stage_typed<CS, PX, 0>(d, t, corner);
    else big = stage_typed<CS, PX, 2>(d, t, corner);
    big = ~lanes_min<64>(~big);
    if ((threadIdx.x & 63) == 0) largest[threadIdx.x >> 6] = big;
    __syncthreads();
    return __uint_as_float(max(max(largest[0], largest[1]), max(largest[2], largest[3])));
}

typedef __attribute__((address_space(3))) const float lds_float;

// One output column: which it is, its weights, where its four corners are in LDS and the rows of its cell.  A wave is one row of
// cells, so everything about rows is uniform.
template <int CS, int PX>
struct Column {
    int X, cj, r_begin, r_end;                        // rows 8 cj - 4 + [r_begin, r_end)
    bool ok;
    float lx, hx;
    int at;                                           // of the upper left corner; the others are one pixel right and one line down
    int to_x0, to_x1, to_y0, to_y1;                   // where the plain form reads instead, see logit()
    __device__ __forceinline__ Column(const dsaspp_scores8_desc& d, const Tile& t) {
        constexpr int from = PX == PXF ? 4 : 0;       // where in its first cell the wave's first column is
        const int u = (threadIdx.x & 63) + from, px = u >> 3, py = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        cj = t.cj0 + py;
        X = 8 * t.ci0 - 4 + u;
        ok = cj <= d.h && X >= 0 && X < 8 * d.w;
        r_begin = cj == 0 ? 4 : 0;
        r_end = cj == d.h ? 4 : 8;
        int x0, x1;
        src_index(max(X, 0), d.w, x0, x1, lx);
        hx = 1.f - lx;
        at = (py * PX + px) * CS;
        // Left of the first pixel's centre (and above it) torch reads pixels 0 and 1 with weights 1 and 0, the tile holds pixel 0 twice: the
        // same sum unless pixel 1 is not finite.
        to_x0 = x0 - (t.ci0 - 1 + px) > 0 ? CS : 0;
        to_x1 = (min(px + 1 + (x0 - (t.ci0 - 1 + px) > 0 && x1 > x0), PX - 1) - px) * CS;
        const int down = cj == 0 ? 1 : 0;
        to_y0 = down * PX * CS;
        to_y1 = (1 + (down && d.h > 1 ? 1 : 0)) * PX * CS;
    }
    // the address of the corners as one value: the compiler adds the array's own offset, beyond the range of an LDS instruction's, to every
    // class otherwise
    __device__ __forceinline__ const lds_float* corners(const float* corner) const {
        uint32_t p = (uint32_t)(uintptr_t)(lds_float*)(corner + at);
        asm("" : "+v"(p));
        return (const lds_float*)p;
    }
    // weight of the second corner row: (2 r + 1) / 16, but 0 above the first pixel's centre (exact in fp32 either way)
    __device__ __forceinline__ float ly(int r) const { return cj == 0 ? 0.f : 0.125f * (float)r + 0.0625f; }
    // the interpolated logit of one class, every product and sum rounded by itself
    __device__ __forceinline__ float logit(const float* corner, int c, float hy, float ly) const {
        const float* p = corner + at + c;
        return mix(hy, mix(hx, p[0], lx, p[CS]), ly, mix(hx, p[PX * CS], lx, p[PX * CS + CS]));
    }
    // the same from the very pixels that torch reads, for logits that may be infinite or NaN
    __device__ __forceinline__ float plain_logit(const float* corner, int c, float hy, float ly) const {
        const float* p = corner + at + c;
        return mix(hy, mix(hx, p[to_y0 + to_x0], lx, p[to_y0 + to_x1]), ly, mix(hx, p[to_y1 + to_x0], lx, p[to_y1 + to_x1]));
    }
};

// The short form of a column's arithmetic, for columns of tame logits whose two corner rows are alike enough.
//
// With M_i = max r_i, x0 = (r0 - M0) log2 e and dx = (r1 - M1) log2 e - x0 the logit of class c in output row r is
//   (z - up) log2 e = x(r) = x0 + ly(r) dx,   up = hy M0 + ly M1,
// at most 0 and linear in r, so its exponential is a geometric sequence down the 8 rows of a cell: e(r + 1) = e(r) 2^(dx / 8), one
// multiplication where an interpolation, a subtraction and an exponential (four issue slots) would be.  It asks for |dx| <= 48: then the
// sum of a row is at least 2^-48, and a term that starts below the normal range (2^-126) ends below 2^-78 and does not count.
// A step adds at most 3 half-steps of relative error (the factor's and the product's), seven of them 21.
//
// r0 and r1 are rounded as z's definition rounds them and the maximum is subtracted before the scaling, so a class that leads both rows has
// x = 0 and e = 1 to the bit, and the log probability of any class is taken from the same x: nothing but the class' own x and the sum enter,
// no reference rounded apart (one of them put half of all confident pixels above 0, by up to R half-steps).
//
// What the two forms round differently is z along y (2 half-steps of hy |r0| + ly |r1|) and x (subtraction, scaling, dx, x: 3 of the distance
// from the maximum and one of dx).  With M = max |M_i| and a class X below the maximum that is 2 (X + M) + 3 X + 34 half-steps in its logit:
// it falls out of the classes that count, but grows with M.  So columns with M from 64 on take the plain form, which has the errors of an
// fp32 log-softmax of z; below that a log probability, which has two such terms and the 23 half-steps of the exponentials, is off by up to
// 4 M + 92 + 5 (|log p| + H) half-steps more: for likely classes 2e-5 at M = 64, 8e-6 at M = 10.
// (With M up to 1e5, logits 3 units apart and 1e4 off zero had log probabilities 2e-3 off.)
// Blocks with logits beyond 1e5, and those with -inf or NaN, take the plain form too: four pictures of 1024 x 2048, 19 classes, 3 alternatives
// 267 us against 137, forward and backward pass of eight 843 against 270.
constexpr float ALIKE = 48.f, NEAR_ZERO = 64.f, TAME = 1.0e5f;
constexpr float PAD = -1.0e6f;            // x of the classes past the last one: below that of any tame logit

template <int NC>
struct Chain {
    float x0[NC], dx[NC], q[NC], e[NC];
    float M0, M1;
    // from the four corners; classes from nc on get exponentials of 0.  Returns whether the short form holds for this lane.
    template <bool EXACT, int CS, int PX>
    __device__ __forceinline__ bool start(const Column<CS, PX>& col, const float* corner, int nc) {
        const lds_float* p = col.corners(corner);
        M0 = M1 = -FLT_MAX;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            x0[c] = mix(col.hx, p[c], col.lx, p[CS + c]);
            dx[c] = mix(col.hx, p[PX * CS + c], col.lx, p[PX * CS + CS + c]);
            if (EXACT || c < nc) { M0 = fmaxf(M0, x0[c]); M1 = fmaxf(M1, dx[c]); }
        }
        const float ly = col.ly(col.r_begin), step = col.cj != 0 ? 0.125f : 0.f;
        float far = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const bool real = EXACT || c < nc;
            x0[c] = real ? (x0[c] - M0) * SR_LOG2E : PAD;
            dx[c] = real ? fmaf(dx[c] - M1, SR_LOG2E, -x0[c]) : 0.f;
            far = fmaxf(far, fabsf(dx[c]));
            q[c] = __builtin_amdgcn_exp2f(step * dx[c]);         // the topmost cells have ly = 0 throughout
            e[c] = __builtin_amdgcn_exp2f(fmaf(ly, dx[c], x0[c]));
        }
        far *= 8.f * step;
        return far <= ALIKE && largest() < NEAR_ZERO;
    }
    __device__ __forceinline__ float largest() const { return fmaxf(fabsf(M0), fabsf(M1)); }
    __device__ __forceinline__ float x(int c, float ly) const { return fmaf(ly, dx[c], x0[c]); }
    // the same bits for a class known at run time only: from the corners again, no register is indexed
    template <int CS, int PX>
    __device__ __forceinline__ float x_of(const Column<CS, PX>& col, const float* corner, int c, float ly) const {
        const float* p = corner + col.at + c;
        const float a = (mix(col.hx, p[0], col.lx, p[CS]) - M0) * SR_LOG2E;
        return fmaf(ly, fmaf(mix(col.hx, p[PX * CS], col.lx, p[PX * CS + CS]) - M1, SR_LOG2E, -a), a);
    }
};

// The K largest of a pixel in the short form.  A key is x with its five lowest bits replaced by the class, so that keeping K + 1
// keys in order is K + 1 instructions per class (one max, K medians of three) where values and classes apart take 4 K - 1.  Where
// two neighbours among them are closer than the roundings of x and of the key, the pixel's logits are offered again, exactly.
template <int K>
struct Keys {
    float v[K + 1];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j <= K; ++j) v[j] = -FLT_MAX;
    }
    __device__ __forceinline__ void offer(float x, int c) {
        const float k = __uint_as_float((__float_as_uint(x) & ~31u) | (unsigned)c);
#pragma unroll
        for (int j = K; j > 0; --j) v[j] = med3(v[j - 1], v[j], k);
        v[0] = larger(v[0], k);
    }
    __device__ __forceinline__ int cls(int j) const { return (int)(__float_as_uint(v[j]) & 31u); }
    // Two keys are in the logits' order if they are further apart than what may have moved them: up to 31 steps of the last place of x each
    // (the class for the bits that were there), together 124 half-steps of the larger magnitude; and the roundings of the two x, above, which
    // are 5 |x| + 2.9 M + 48 half-steps each in log2 units.
    static __device__ __forceinline__ float margin(float M) { return fmaf(M, 6.f * 0x1p-24f, 100.f * 0x1p-24f); }
    __device__ __forceinline__ bool unclear(int k, float near) const {
        int u = 0;                        // no short circuit: it would put each median into a block of its own, with every key kept for it
#pragma unroll
        for (int j = 0; j < K; ++j) u |= (int)(v[j] - v[j + 1] <= fmaf(fabsf(v[j + 1]), 140.f * 0x1p-24f, near)) & (int)(j < k);
        return u != 0;
    }
};

template <int NC, bool EXACT, int K>
__global__ __launch_bounds__(256, NC <= 19 ? (K == 0 ? 4 : 3) : 1) void scores8_fwd_kernel(const dsaspp_scores8_desc d, const int tiles_x,
                                                                                            const int tiles_y) {
    constexpr int CS = NC | 1;
    __shared__ float corner[PXF * PY * CS];
    __shared__ unsigned largest[4];
    const Tile tl(xcd_remap(blockIdx.x, gridDim.x), tiles_x, tiles_y);
    const Column<CS, PXF> q(d, tl);
    const int nc = EXACT ? NC : d.n_class, W = 8 * d.w;
    const int64_t plane = 64ll * d.h * d.w;
    const unsigned X = q.X;               // row bases are uniform, lanes differ in X alone
    int64_t at = tl.n * plane + (int64_t)(8 * q.cj - 4 + q.r_begin) * W;
    int64_t next = -1, after = -1;        // labels, two rows ahead; a cell has 4 or 8 rows
    if (q.ok && d.logp) {
        next = (d.labels + at)[X];
        after = (d.labels + at + W)[X];
    }
    const float R = stage<CS, PXF>(d, tl, corner, largest);
    if (!q.ok) return;
    Chain<NC> ch;
    const bool alike = ch.template start<EXACT>(q, corner, nc);
    const bool brief = R < TAME && __all(alike);
    const float near = Keys<K>::margin(ch.largest());
    auto rows = [&](auto form) {          // a loop for each form: together they would copy every class' registers at its start
        constexpr bool BRIEF = decltype(form)::value;
#pragma unroll 1
        for (int r = q.r_begin; r < q.r_end; ++r, at += W) {
            const float ly = q.ly(r), hy = 1.f - ly;
            const int64_t l = next;
            next = after;
            if (d.logp && r + 2 < q.r_end) after = (d.labels + at + 2 * W)[X];
            const int label = d.logp && l != d.ignore_index && l >= 0 && l < nc ? (int)l : -1;
            int top_i[K > 0 ? K : 1];
            float logp, h, sum, top_lp[K > 0 ? K : 1];
            if constexpr (BRIEF) {
                float s = 0.f, t = 0.f;
                Keys<K> keys;
                if (K > 0) keys.clear();
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const float x = ch.x(c, ly);
                    s += ch.e[c];
                    t = fmaf(x, ch.e[c], t);
                    if (K > 0) keys.offer(x, c);
                    ch.e[c] *= ch.q[c];
                }
                sum = s;
                const float log2_s = __builtin_amdgcn_logf(s);
                // between two rows with other leading classes the sum's error may exceed the class' distance from it
                logp = label < 0 ? 0.f : fminf(SR_LN2 * (ch.x_of(q, corner, max(label, 0), ly) - log2_s), 0.f);
                h = fmaxf(SR_LN2 * (log2_s - t * __builtin_amdgcn_rcpf(s)), 0.f);
                if (K > 0) {
#pragma unroll
                    for (int j = 0; j < K; ++j) top_i[j] = keys.cls(j);
                    if (keys.unclear(d.top_k, near)) {
                        Top<K> top;
                        top.clear();
#pragma unroll 1
                        for (int c = 0; c < nc; ++c) top.offer(q.logit(corner, c, hy, ly), c);
#pragma unroll
                        for (int j = 0; j < K; ++j) top_i[j] = top.i[j];
                    }
#pragma unroll
                    for (int j = 0; j < K; ++j)
                        if (j < d.top_k)          // descending as the logits are, whose near ties x may turn round
                            top_lp[j] = fminf(SR_LN2 * (ch.x_of(q, corner, top_i[j], ly) - log2_s), j > 0 ? top_lp[j > 0 ? j - 1 : 0] : 0.f);
                }
            } else {
                Top<K> top;
                Soft s;
                top.clear();
                s.clear();
                int best = 0;
#pragma unroll 1
                for (int c = 0; c < nc; ++c) {
                    const float z = q.plain_logit(corner, c, hy, ly);
                    best = z > s.m ? c : best;
                    s.m = fmaxf(s.m, z);
                    top.offer(z, c);
                }
#pragma unroll 1
                for (int c = 0; c < nc; ++c) s.add(q.plain_logit(corner, c, hy, ly));
                // relative to the reference of the short form: the backward pass, whose waves hold other columns, may take that for this one
                sum = s.s * __builtin_amdgcn_exp2f(fmaxf(ch.x_of(q, corner, best, ly), SR_FAR));
                const float log_s = logf(s.s);
                logp = label < 0 ? 0.f : s.empty() ? -INFINITY : (q.plain_logit(corner, label, hy, ly) - s.m) - log_s;
                h = s.entropy(log_s);
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    top_lp[j] = top_log_p(top.v[j], top.i[j], s, log_s);
                    top_i[j] = (int)top_index(top.i[j], s);
                }
            }
            if (d.logp) (d.logp + at)[X] = logp;
            if (d.entropy) (d.entropy + at)[X] = h;
            if (d.stats) (d.stats + at)[X] = sum;
#pragma unroll
            for (int j = 0; j < K; ++j)
                if (j < d.top_k) {
                    const int64_t o = at + ((int64_t)tl.n * (d.top_k - 1) + j) * plane;
                    (d.top_logp + o)[X] = top_lp[j];
                    (d.top_class + o)[X] = top_i[j];
                }
        }
    };
    if (brief) rows(std::true_type()); else rows(std::false_type());
}

// v of lane 7 - i of the 8 lanes of a cell (an aligned half of a DPP row)
__device__ __forceinline__ float mirror8(float v) {
    const int x = __float_as_int(v);
    return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x141, 0xF, 0xF, true));      // row_half_mirror
}
// sum over an aligned group of four lanes, in every one of them
__device__ __forceinline__ float quad_sum(float v) {
    int x = __float_as_int(v);
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, true));         // quad_perm [1,0,3,2]
    x = __float_as_int(v);
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, true));   // quad_perm [2,3,0,1]
}

// HB: an upstream gradient of the entropy is there.  Per pixel and class  dz = e (k0 + k1 x)  with e = 2^x, x = (z - up) log2 e for
// any reference up, and per-pixel k0, k1; what falls on the label and on the alternatives is added to lane-private LDS columns instead of
// being selected by class.
// KT (0, 3 or 8): room for the gradients of a pixel's alternatives.  All are asked for before the first is used, one by one they cost a
// trip to memory each, twice per row (five alternatives, three 1024 x 2048 pictures, forward and backward: 493 us against 350).
// The sum of the exponentials and the entropy come from the forward pass: 8 bytes per pixel for three instructions per class.
// With eight and an entropy gradient two waves per SIMD without spills are faster than three with (350 against 535 us).
template <int NC, bool EXACT, bool HB, int KT>
__global__ __launch_bounds__(256, NC <= 19 ? (HB && KT == 8 ? 2 : 3) : 1) void scores8_bwd_kernel(const dsaspp_scores8_desc d, const int tiles_x, const int tiles_y) {
    constexpr int CS = NC | 1, CELLS = TCX * TCY, KS = CELLS * CS;
    __shared__ float corner[PX * PY * CS];
    __shared__ float oh[2 * NC * 256];                // [corner row][class][lane]
    __shared__ float ct[4 * KS];                      // [corner][cell][class]
    __shared__ unsigned largest[4];
    const int tid = threadIdx.x, nc = EXACT ? NC : d.n_class, W = 8 * d.w;
    const int tile = xcd_remap(blockIdx.x, gridDim.x);
    const Tile tl(tile, tiles_x, tiles_y);
#pragma unroll
    for (int c = 0; c < 2 * NC; ++c) oh[c * 256 + tid] = 0.f;
    const Column<CS, PX> q(d, tl);
    const float R = stage<CS, PX>(d, tl, corner, largest);
    float g0[NC], g1[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) { g0[c] = 0.f; g1[c] = 0.f; }
    if (q.ok) {
        const int64_t plane = 64ll * d.h * d.w;
        const unsigned X = q.X;           // row bases are uniform, lanes differ in X alone
        int64_t at = tl.n * plane + (int64_t)(8 * q.cj - 4 + q.r_begin) * W;
        Chain<NC> ch;
        const bool alike = ch.template start<EXACT>(q, corner, nc);
        const bool brief = R < TAME && __all(alike);
        struct In { int64_t l; float a, b, s, h; };
        // An upstream gradient of one value is read like a dense one, at index 0 throughout: loads on either side of a branch would share
        // registers and wait for each other (30 us of 160 at the size below).
        const unsigned Xa = d.g_logp_one ? 0 : X, Xb = d.g_entropy_one ? 0 : X, Xt = d.g_top_one ? 0 : X;
        auto load = [&](int64_t p) {
            In v;
            v.l = d.g_logp ? (d.labels + p)[X] : -1;
            v.a = d.g_logp ? (d.g_logp + (d.g_logp_one ? 0 : p))[Xa] : 0.f;
            v.b = HB ? (d.g_entropy + (d.g_entropy_one ? 0 : p))[Xb] : 0.f;
            v.s = brief ? (d.stats + p)[X] : 0.f;
            v.h = HB && brief ? (d.entropy + p)[X] : 0.f;
            return v;
        };
        In next = load(at);
        auto rows = [&](auto form) {      // a loop for each form: together they would copy every class' registers at its start
            constexpr bool BRIEF = decltype(form)::value;
#pragma unroll 1
            for (int r = q.r_begin; r < q.r_end; ++r, at += W) {
                const float ly = q.ly(r), hy = 1.f - ly;
                const In in = next;
                if (r + 1 < q.r_end) next = load(at + W);         // on its way while this row is worked out
                const int label = d.g_logp && in.l != d.ignore_index && in.l >= 0 && in.l < nc ? (int)in.l : -1;
                const float a = label >= 0 ? in.a : 0.f, b = in.b;
                float A = a;
                bool live = a != 0.f || b != 0.f;
                constexpr int KR = KT > 0 ? KT : 1;
                constexpr bool EARLY = KT <= 3;           // their classes too: eight would not fit beside the row's arithmetic
                float gt[KR];
                int64_t ct_[KR];
                auto load_classes = [&]() {
#pragma unroll
                    for (int j = 0; j < KR; ++j) ct_[j] = j < d.top_k ? (d.top_class + at + ((int64_t)tl.n * (d.top_k - 1) + j) * plane)[X] : -1;
                };
                if (KT > 0) {
#pragma unroll
                    for (int j = 0; j < KR; ++j)
                        gt[j] = j >= d.top_k ? 0.f : (d.g_top + (d.g_top_one ? 0 : at + ((int64_t)tl.n * (d.top_k - 1) + j) * plane))[Xt];
                    if (EARLY || !BRIEF) load_classes();
#pragma unroll
                    for (int j = 0; j < KR; ++j) {
                        live = live || gt[j] != 0.f;
                        A += BRIEF || ct_[j] >= 0 ? gt[j] : 0.f;      // in the short form every pixel has its alternatives
                    }
                }
                // the label's sums are read now and written back after the row's arithmetic
                float* const o0 = oh + max(label, 0) * 256 + tid;
                const float w0 = o0[0], w1 = o0[NC * 256];
                if constexpr (BRIEF) {
                    // log_p + H = ln2 (x - log2 s + H / ln2), with the sum and the entropy of the forward pass
                    const float inv = live ? 1.f / in.s : 0.f;
                    const float k1 = HB ? -b * SR_LN2 * inv : 0.f;
                    const float k0 = HB ? -A * inv - k1 * (__builtin_amdgcn_logf(in.s) - in.h * SR_LOG2E) : -A * inv;
                    const float a0 = hy * k0, a1 = ly * k0;
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        if (HB) {
                            const float g = ch.e[c] * fmaf(k1, ch.x(c, ly), k0);
                            g0[c] = fmaf(hy, g, g0[c]);
                            g1[c] = fmaf(ly, g, g1[c]);
                        } else {
                            g0[c] = fmaf(a0, ch.e[c], g0[c]);
                            g1[c] = fmaf(a1, ch.e[c], g1[c]);
                        }
                        ch.e[c] *= ch.q[c];
                    }
                    if (!live) continue;
                } else {
                    if (!live) continue;
                    Soft s;
                    s.clear();
#pragma unroll 1
                    for (int c = 0; c < nc; ++c) s.m = fmaxf(s.m, q.plain_logit(corner, c, hy, ly));
#pragma unroll 1
                    for (int c = 0; c < nc; ++c) s.add(q.plain_logit(corner, c, hy, ly));
                    if (s.empty()) continue;              // every class masked out
                    const float inv = 1.f / s.s, k1 = HB ? -b * SR_LN2 * inv : 0.f, k0 = HB ? -A * inv - k1 * (s.t * inv) : -A * inv;
#pragma unroll 1
                    for (int c = 0; c < nc; ++c) {        // into the lane's own column, as the label below: no register is indexed
                        const float x = (q.plain_logit(corner, c, hy, ly) - s.m) * SR_LOG2E;
                        const float g = __builtin_amdgcn_exp2f(x) * fmaf(k1, fmaxf(x, SR_FAR), k0);
                        oh[c * 256 + tid] += hy * g;
                        oh[(NC + c) * 256 + tid] += ly * g;
                    }
                }
                if constexpr (BRIEF) {
                    if (label >= 0) {
                        o0[0] = fmaf(a, hy, w0);
                        o0[NC * 256] = fmaf(a, ly, w1);
                    }
                } else if (label >= 0) {                  // the loop above wrote the same columns
                    o0[0] += a * hy;
                    o0[NC * 256] += a * ly;
                }
                if (KT > 0) {
                    if (!EARLY && BRIEF) load_classes();
#pragma unroll
                    for (int j = 0; j < KR; ++j)
                        if (ct_[j] >= 0 && ct_[j] < nc) {
                            oh[(int)ct_[j] * 256 + tid] += gt[j] * hy;
                            oh[(NC + (int)ct_[j]) * 256 + tid] += gt[j] * ly;
                        }
                }
            }
        };
        if (brief) rows(std::true_type()); else rows(std::false_type());
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            g0[c] += oh[c * 256 + tid];
            g1[c] += oh[(NC + c) * 256 + tid];
        }
    }
    // The 8 columns of a cell together: corner (y, x0) gets the hx-weighted, (y, x1) the lx-weighted sum.  Two classes at a time: a lane of
    // the lower half takes its mirror's value of the first class and gives its own of the second, so that from then on the halves hold a
    // class each (11 instructions for what takes 16 class by class).
    const int cell = tid >> 3, lane8 = tid & 7;
    const bool hi = lane8 >= 4;
    const float hxm = mirror8(q.hx), lxm = mirror8(q.lx);
#pragma unroll
    for (int c = 0; c < NC; c += 2) {
        const float o0 = c + 1 < NC ? g0[c + 1 < NC ? c + 1 : c] : 0.f, o1 = c + 1 < NC ? g1[c + 1 < NC ? c + 1 : c] : 0.f;
        const float k0 = hi ? o0 : g0[c], k1 = hi ? o1 : g1[c], m0 = mirror8(hi ? g0[c] : o0), m1 = mirror8(hi ? g1[c] : o1);
        const float a00 = quad_sum(fmaf(hxm, m0, q.hx * k0)), a01 = quad_sum(fmaf(lxm, m0, q.lx * k0));
        const float a10 = quad_sum(fmaf(hxm, m1, q.hx * k1)), a11 = quad_sum(fmaf(lxm, m1, q.lx * k1));
        const int mine = c + (hi ? 1 : 0);
        if ((lane8 & 3) == (c / 2 & 3) && mine < NC) {         // cells outside the image store their zeros
            float* to = ct + cell * CS + mine;
            to[0 * KS] = a00;
            to[1 * KS] = a01;
            to[2 * KS] = a10;
            to[3 * KS] = a11;
        }
    }
    __syncthreads();
    // corner pixel (py, px) of the tile is corner 00 of cell (py, px), 01 of (py, px-1), 10 of (py-1, px), 11 of (py-1, px-1)
    float* out = d.ws + (int64_t)tile * (PX * PY) * nc;
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

// Positions along one axis, counted before clamping (pixel i is position i + 1, what lies beyond the border falls on the border pixel),
// and the tiles that hold a position: tile b has positions b TC .. (b + 1) TC.
struct Span {
    int first, last;
    __device__ __forceinline__ Span(int i, int n) : first(i == 0 ? 0 : i + 1), last(i == n - 1 ? n + 1 : i + 1) {}
};
template <int TC>
__device__ __forceinline__ int first_tile(int u) { return u > 0 ? (u - 1) / TC : 0; }

// One thread per class of a source pixel in GL lines, whose loads are all on their way before the first is added; classes fastest (as
// the workspace has them) or, for planes, pixels fastest.
constexpr int GL = 4;
__global__ __launch_bounds__(256) void scores8_gather_kernel(const dsaspp_scores8_desc d, const int tiles_x, const int tiles_y, const unsigned per_line,
                                                             const unsigned lines) {
    const bool inner = d.gc == 1;
    const unsigned i = blockIdx.x * 256 + threadIdx.x;
    if (i >= per_line) return;
    const int c = inner ? i % (unsigned)d.n_class : i / (unsigned)d.w, x = inner ? i / (unsigned)d.n_class : i % (unsigned)d.w;
    const Span sx(x, d.w);
    const int ux = x + 1, tx = ux / TCX, tile_len = PX * PY * d.n_class;
    const bool x0 = tx < tiles_x, x1 = tx > 0 && ux == tx * TCX;
    const int at0 = tx * tile_len + (ux - tx * TCX) * d.n_class + c, at1 = at0 - tile_len + TCX * d.n_class;       // inside a row of tiles
    for (unsigned line0 = blockIdx.y * GL; line0 < lines; line0 += gridDim.y * GL) {
        float v[GL][4];
        int image[GL], row[GL];           // of the lines: one division for all of them
        image[0] = line0 / (unsigned)d.h;
        row[0] = line0 - (unsigned)image[0] * (unsigned)d.h;
#pragma unroll
        for (int k = 1; k < GL; ++k) {
            const bool wrap = row[k - 1] + 1 == d.h;
            row[k] = wrap ? 0 : row[k - 1] + 1;
            image[k] = image[k - 1] + (wrap ? 1 : 0);
        }
        auto line_of = [&](int n, int uy, int ty) {               // the same for all lanes
            return d.ws + ((int64_t)n * tiles_y + ty) * tiles_x * tile_len + (uy - ty * TCY) * PX * d.n_class;
        };
#pragma unroll
        for (int k = 0; k < GL; ++k) {
#pragma unroll
            for (int m = 0; m < 4; ++m) v[k][m] = 0.f;
            if (line0 + k >= lines) continue;
            const int n = image[k], uy = row[k] + 1, ty = uy / TCY;
            if (ty < tiles_y) {
                const float* p = line_of(n, uy, ty);
                if (x0) v[k][0] = p[at0];
                if (x1) v[k][1] = p[at1];
            }
            if (ty > 0 && uy == ty * TCY) {
                const float* p = line_of(n, uy, ty - 1);
                if (x0) v[k][2] = p[at0];
                if (x1) v[k][3] = p[at1];
            }
        }
#pragma unroll
        for (int k = 0; k < GL; ++k) {
            if (line0 + k >= lines) break;
            const int n = image[k], y = row[k];
            float sum = (v[k][0] + v[k][1]) + (v[k][2] + v[k][3]);
            const Span sy(y, d.h);
            if (sy.last > sy.first || sx.last > sx.first) {       // border pixels: what fell beyond the border too
                for (int by = sy.first; by <= sy.last; ++by)
                    for (int bx = sx.first; bx <= sx.last; ++bx) {
                        if (by == y + 1 && bx == ux) continue;
                        for (int ty = first_tile<TCY>(by); ty <= by / TCY && ty < tiles_y; ++ty)
                            for (int t = first_tile<TCX>(bx); t <= bx / TCX && t < tiles_x; ++t)
                                sum += line_of(n, by, ty)[t * tile_len + (bx - t * TCX) * d.n_class + c];
                    }
            }
            const int64_t o = n * d.gn + y * d.gy + x * d.gx + c * d.gc;
            if (d.g_dtype == 1) reinterpret_cast<float*>(d.dlogits)[o] = sum;
            else reinterpret_cast<u16*>(d.dlogits)[o] = d.g_dtype == 0 ? Elem<0>::down(sum) : Elem<2>::down(sum);
        }
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
    DS_REQUIRE(*tiles < (1ll << 24), "%s: too many pixels for one launch (fewer than 2^32 lanes)", who);
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
    else if (d.top_k <= 5) LAUNCH(5);
    else LAUNCH(8);
#undef LAUNCH
}

template <int NC, bool EX>
void launch_bwd(const dsaspp_scores8_desc& d, int tx, int ty, unsigned grid, hipStream_t s) {
#define LAUNCH(HB, KT) hipLaunchKernelGGL((scores8_bwd_kernel<NC, EX, HB, KT>), dim3(grid), dim3(256), 0, s, d, tx, ty)
    const int k = d.g_top ? d.top_k : 0;
    if (d.g_entropy) {
        if (k == 0) LAUNCH(true, 0);
        else if (k <= 3) LAUNCH(true, 3);
        else LAUNCH(true, 8);
    } else {
        if (k == 0) LAUNCH(false, 0);
        else if (k <= 3) LAUNCH(false, 3);
        else LAUNCH(false, 8);
    }
#undef LAUNCH
}

}  // namespace

// Cityscapes' 19 classes have their own instantiation, every other count the next multiple of 8: the class loops are unrolled
// registers, and the range checks of the inexact ones cost a select per class.  Four pictures with 3 alternatives, and forward and backward pass of
// eight (us):  5 classes 108, 183;  16: 117, 259;  19: 130, 272;  20 to 24: 138, 359;  25 to 32: 176, 616.  The last is LDS: the backward pass keeps
// two sums per class and lane there, 88 KB in all at 32 classes, so that a CU has one block (three at 19 classes).
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
    DS_REQUIRE(d->logp || d->entropy || d->stats || d->top_k, "scores8_fwd: nothing to compute");
    tx = (d->w + TCX - 1) / TCX;                      // no tile for the half cell left of column 0
    tiles = (int64_t)d->n_img * tx * ty;
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
    DS_REQUIRE(d->stats, "scores8_bwd: null stats");
    DS_REQUIRE(!d->g_entropy || d->entropy, "scores8_bwd: g_entropy needs the entropy of the forward pass");
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
    const unsigned per_line = (unsigned)d->w * d->n_class;
    const unsigned lines = (unsigned)d->n_img * d->h;         // below 2^26: at least a tile of 4 lines' cells each
    const unsigned gy = (lines + GL - 1) / GL;
    hipLaunchKernelGGL(scores8_gather_kernel, dim3((per_line + 255) / 256, gy < 65535 ? gy : 65535), dim3(256), 0, s, *d, tx, ty, per_line, lines);
    DS_LAUNCH_CHECK("scores8_bwd");
    return 0;
}
