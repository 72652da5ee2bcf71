// Group norm with an activation (and optional dropout behind it) over ragged channels-last rows: X[M, C], cloud b owns rows
// seg_off[b] .. seg_off[b+1], group j the channels j*Cg .. (j+1)*Cg, Cg = C / G.  Per (cloud, group) with n = rows * Cg elements:
//   mean, biased var, r = (var + eps)^-1/2, xh = (x - mean) r, u = w xh + b, y = D phi(u)            (D: dropout, keep / (1 - p))
// First gradient:   g = dy D phi'(u), h = w g, dx = r (h - m(h) - xh m(h xh)), dw = sum_rows g xh, db = sum_rows g       (m: mean over n)
// Second gradient, cotangents P of dx, q of dw, s of db:
//   v = r (P - m(P) - xh m(P xh)),  gb = w v + q xh + s,  d(dy) = gb D phi',  ub = gb dy D phi''
//   X = -r (h m(P xh) + P m(h xh)) + q g + w ub
//   d(x) = r (X - m(X) - xh (m(X xh) + r (m(P h) - m(P) m(h) - m(P xh) m(h xh)))),  d(w) = sum_rows (g v + ub xh),  d(b) = sum_rows ub
// The simplest form: one workgroup per (cloud, group), one pass over the data per sum.
#include "group_norm.h"

#include <stdlib.h>

#include <algorithm>
#include <initializer_list>

namespace {

struct GN : gn::Norm {
    int act;
};

__device__ __forceinline__ float block_sum(float v, float* s_red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
    __syncthreads();
    return s_red[0] + s_red[1] + s_red[2] + s_red[3];
}

__device__ __forceinline__ float act_eval(int act, float u, float slope, float* d1, float* d2) {
    switch (act_family(act)) {
        case DD3D_FAM_LINEAR: return activate<DD3D_FAM_LINEAR, 2>(u, slope, d1, d2);
        case DD3D_FAM_SILU: return activate<DD3D_FAM_SILU, 2>(u, slope, d1, d2);
        default: return activate<DD3D_FAM_GELU, 2>(u, slope, d1, d2);
    }
}

__device__ __forceinline__ float drop_factor(const GN& a, int64_t row, int c) {
    if (!a.drop.key) return 1.f;
    const uint4 w = philox_block(philox_key(a.drop.key), (uint64_t)row * (uint64_t)((a.C + 3) / 4) + (uint64_t)(c / 4));
    const uint32_t r = (c & 3) == 0 ? w.x : (c & 3) == 1 ? w.y : (c & 3) == 2 ? w.z : w.w;
    return !a.drop.all && r >= a.drop.thr ? a.drop.scale : 0.f;
}
__device__ __forceinline__ float dropped(float d, float v) { return d == 0.f ? 0.f : d * v; }

__device__ __forceinline__ void cloud_rows(const GN& a, int b, int64_t* r0, int64_t* r1) {
    *r0 = min(max(a.seg[b], 0), a.M);
    *r1 = min(max(a.seg[b + 1], (int)*r0), a.M);
}

// rows of [0, M) that belong to no cloud are written as zeros
template <typename T>
__global__ __launch_bounds__(256) void k_zero_rest(GN a, T* Y, T* Y2) {
    const int64_t lo = a.B ? min(max(a.seg[0], 0), a.M) : 0, hi = a.B ? min(max(a.seg[a.B], (int)lo), a.M) : 0;
    const int64_t n0 = lo * a.C, n1 = (a.M - hi) * a.C;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n0 + n1; i += (int64_t)gridDim.x * 256) {
        const int64_t at = i < n0 ? i : hi * a.C + (i - n0);
        if (Y) Y[at] = narrow<T>(0.f);
        if (Y2) Y2[at] = narrow<T>(0.f);
    }
}

// what the gradients need of one element
struct Elem {
    float xh, w, dyd, g, h, d1, d2, D;
};
template <typename T>
__device__ __forceinline__ Elem element(const GN& a, const T* dY, const T* X, int64_t row, int c, float mean, float rstd) {
    Elem e;
    e.w = a.W ? load_param(a.W, a.pdt, c) : 1.f;
    e.xh = (widen(X[row * a.C + c]) - mean) * rstd;
    act_eval(a.act, e.w * e.xh + (a.Bi ? load_param(a.Bi, a.pdt, c) : 0.f), a.slope, &e.d1, &e.d2);
    e.D = drop_factor(a, row, c);
    e.dyd = dropped(e.D, widen(dY[row * a.C + c]));
    e.g = e.dyd * e.d1;
    e.h = e.g * e.w;
    return e;
}

template <typename T>
__global__ __launch_bounds__(256) void k_bwd_x(GN a, const T* dY, const T* X, const float* mean_in, const float* rstd_in, T* dX) {
    __shared__ float s_red[4];
    const int b = blockIdx.x / a.G, j = blockIdx.x % a.G;
    int64_t r0, r1;
    cloud_rows(a, b, &r0, &r1);
    const int64_t n = (r1 - r0) * a.Cg;
    if (n == 0) return;
    const float mean = mean_in[blockIdx.x], rstd = rstd_in[blockIdx.x];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t i = threadIdx.x; i < n; i += 256) {
        const Elem e = element(a, dY, X, r0 + i / a.Cg, j * a.Cg + (int)(i % a.Cg), mean, rstd);
        s1 += e.h;
        s2 += e.h * e.xh;
    }
    const float m1 = block_sum(s1, s_red) / (float)n, m2 = block_sum(s2, s_red) / (float)n;
    for (int64_t i = threadIdx.x; i < n; i += 256) {
        const int64_t row = r0 + i / a.Cg;
        const int c = j * a.Cg + (int)(i % a.Cg);
        const Elem e = element(a, dY, X, row, c, mean, rstd);
        dX[row * a.C + c] = narrow<T>(rstd * (e.h - m1 - e.xh * m2));
    }
}

// one workgroup per channel
template <typename T>
__global__ __launch_bounds__(256) void k_bwd_p(GN a, const T* dY, const T* X, const float* mean_in, const float* rstd_in, void* dW, void* dB) {
    __shared__ float s_red[4];
    const int c = blockIdx.x;
    float sw = 0.f, sb = 0.f;
    for (int b = 0; b < a.B; ++b) {
        int64_t r0, r1;
        cloud_rows(a, b, &r0, &r1);
        for (int64_t row = r0 + threadIdx.x; row < r1; row += 256) {
            const Elem e = element(a, dY, X, row, c, mean_in[(int64_t)b * a.G + c / a.Cg], rstd_in[(int64_t)b * a.G + c / a.Cg]);
            sw += e.g * e.xh;
            sb += e.g;
        }
    }
    sw = block_sum(sw, s_red);
    sb = block_sum(sb, s_red);
    if (threadIdx.x == 0) {
        if (dW) store_param(dW, a.pdt, c, sw);
        if (dB) store_param(dB, a.pdt, c, sb);
    }
}

template <typename T>
struct Second {
    const T* P;
    const void *q, *s;
};

struct Means {
    float mp, mp2, mph, m1, m2;
};

struct Elem2 {
    Elem e;
    float P, q, v, gb, ub, X;
};
template <typename T>
__device__ __forceinline__ Elem2 element2(const GN& a, const Second<T>& z, const T* dY, const T* X, int64_t row, int c, float mean, float rstd, const Means& m) {
    Elem2 o;
    o.e = element(a, dY, X, row, c, mean, rstd);
    o.P = z.P ? widen(z.P[row * a.C + c]) : 0.f;
    o.q = z.q ? load_param(z.q, a.pdt, c) : 0.f;
    o.v = rstd * (o.P - m.mp - o.e.xh * m.mp2);
    o.gb = o.e.w * o.v + o.q * o.e.xh + (z.s ? load_param(z.s, a.pdt, c) : 0.f);
    o.ub = o.gb * o.e.dyd * o.e.d2;
    o.X = -rstd * (o.e.h * m.mp2 + o.P * m.m2) + o.q * o.e.g + o.e.w * o.ub;
    return o;
}

// writes d(dy), d(x) and the five means of the (cloud, group) for the parameter kernel behind it
template <typename T>
__global__ __launch_bounds__(256) void k_bwd2_x(GN a, Second<T> z, const T* dY, const T* X, const float* mean_in, const float* rstd_in, T* ddY, T* ddX,
                                                Means* means) {
    __shared__ float s_red[4];
    const int b = blockIdx.x / a.G, j = blockIdx.x % a.G;
    int64_t r0, r1;
    cloud_rows(a, b, &r0, &r1);
    const int64_t n = (r1 - r0) * a.Cg;
    if (n == 0) return;
    const float mean = mean_in[blockIdx.x], rstd = rstd_in[blockIdx.x], inv = 1.f / (float)n;
    Means m = {0.f, 0.f, 0.f, 0.f, 0.f};
    for (int64_t i = threadIdx.x; i < n; i += 256) {
        const int64_t row = r0 + i / a.Cg;
        const int c = j * a.Cg + (int)(i % a.Cg);
        const Elem e = element(a, dY, X, row, c, mean, rstd);
        const float P = z.P ? widen(z.P[row * a.C + c]) : 0.f;
        m.mp += P, m.mp2 += P * e.xh, m.mph += P * e.h, m.m1 += e.h, m.m2 += e.h * e.xh;
    }
    m.mp = block_sum(m.mp, s_red) * inv, m.mp2 = block_sum(m.mp2, s_red) * inv, m.mph = block_sum(m.mph, s_red) * inv;
    m.m1 = block_sum(m.m1, s_red) * inv, m.m2 = block_sum(m.m2, s_red) * inv;
    if (threadIdx.x == 0) means[blockIdx.x] = m;
    float t1 = 0.f, t2 = 0.f;
    for (int64_t i = threadIdx.x; i < n; i += 256) {
        const Elem2 o = element2(a, z, dY, X, r0 + i / a.Cg, j * a.Cg + (int)(i % a.Cg), mean, rstd, m);
        t1 += o.X;
        t2 += o.X * o.e.xh;
    }
    t1 = block_sum(t1, s_red) * inv;
    t2 = block_sum(t2, s_red) * inv + rstd * (m.mph - m.mp * m.m1 - m.mp2 * m.m2);
    for (int64_t i = threadIdx.x; i < n; i += 256) {
        const int64_t row = r0 + i / a.Cg;
        const int c = j * a.Cg + (int)(i % a.Cg);
        const Elem2 o = element2(a, z, dY, X, row, c, mean, rstd, m);
        if (ddY) ddY[row * a.C + c] = narrow<T>(dropped(o.e.D, o.gb * o.e.d1));
        if (ddX) ddX[row * a.C + c] = narrow<T>(rstd * (o.X - t1 - o.e.xh * t2));
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_bwd2_p(GN a, Second<T> z, const T* dY, const T* X, const float* mean_in, const float* rstd_in, const Means* means,
                                                void* dW, void* dB) {
    __shared__ float s_red[4];
    const int c = blockIdx.x;
    float sw = 0.f, sb = 0.f;
    for (int b = 0; b < a.B; ++b) {
        int64_t r0, r1;
        cloud_rows(a, b, &r0, &r1);
        const int64_t at = (int64_t)b * a.G + c / a.Cg;
        for (int64_t row = r0 + threadIdx.x; row < r1; row += 256) {
            const Elem2 o = element2(a, z, dY, X, row, c, mean_in[at], rstd_in[at], means[at]);
            sw += o.e.g * o.v + o.ub * o.e.xh;
            sb += o.ub;
        }
    }
    sw = block_sum(sw, s_red);
    sb = block_sum(sb, s_red);
    if (threadIdx.x == 0) {
        if (dW) store_param(dW, a.pdt, c, sw);
        if (dB) store_param(dB, a.pdt, c, sb);
    }
}

inline int rest_blocks(int64_t M, int C) { return (int)(ceil_div64(M * C, 256) < 1024 ? ceil_div64(M * C, 256) : 1024); }

// argument checks shared by the three entry points; 0 = fill in `a` and go on
inline int check(int dtype, int64_t M, int C, const int32_t* seg, int B, int G, const void* W, const void* Bi, int pdt, int act, float slope, double p,
                 const int64_t* key, GN* a) {
    if (M < 0 || B < 0 || C <= 0 || G <= 0 || C % G != 0) return DD3D_EARG;
    if (M >= (1ll << 31) || C > 4096 || (int64_t)B * G >= (1ll << 31)) return DD3D_ESIZE;
    if (dtype < DD3D_F32 || dtype > DD3D_BF16 || (pdt != DD3D_F32 && pdt != dtype) || act < DD3D_ACT_NONE || act > DD3D_ACT_GELU) return DD3D_EARG;
    if (slope != slope || (B > 0 && !seg) || !make_drop(p, key, &a->drop)) return DD3D_EARG;
    a->M = (int)M, a->C = C, a->B = B, a->G = G, a->Cg = C / G, a->pdt = pdt, a->act = act, a->seg = seg, a->W = W, a->Bi = Bi;
    a->slope = act == DD3D_ACT_NONE ? 1.f : act == DD3D_ACT_RELU ? 0.f : slope;
    a->eps = 0.f;
    return 0;
}

// ---- launch geometry --------------------------------------------------------------------------------------------------------------
// windows of the whole batch: enough to fill the chip with the slabs of a row, never so many that joining them shows
inline int max_windows(int C) { return C >= 1024 ? 64 : C <= 64 ? 1024 : 65536 / C; }
constexpr int MIN_WINDOW = 512;

inline int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

inline gn::Div divide_by(int d) {
    gn::Div r;
    r.d = d, r.mul = d == 1 ? 0 : (uint32_t)((0x100000000ull + d - 1) / d);
    return r;
}

// K: quantities summed at once; nrs / nrl: vectors a thread holds
inline gn::Plan plan(const gn::Norm& a, int act, int esize, bool aligned, int K, int nrs, int nrl, bool params) {
    gn::Plan p;
    gn::Geo& g = p.g;
    p.fam = act_family(act);
    p.V = esize == 2 && aligned && a.Cg % 8 == 0 && a.Cg <= 2048 ? 8 : 4;
    const int m0 = 4 / gcd(a.Cg, 4);   // groups whose channels fill whole vectors of four
    p.al = aligned && a.C % p.V == 0 && m0 * a.Cg <= 4096;
    p.uni = p.al && a.Cg % p.V == 0;
    auto lanes = [&](int k) { return p.al || k >= a.G || k * a.Cg % 4 == 0 ? (k * a.Cg + p.V - 1) / p.V : (k * a.Cg + 6) / 4; };
    auto whole = [&](int k) { return k >= a.G ? a.G : p.al ? std::min(a.G, (k + m0 - 1) / m0 * m0) : k; };
    // Slab width: 64 bytes of a row at least (its neighbour reads the other half of the line into the same L2), doubled while a short
    // cloud still fits one chunk and 1024 workgroups remain to fill the chip.  fp32 forward, 128 channels, us at 64 / 128 / 256 / 512
    // bytes: 2560 clouds of 82 rows 106 / 65 / 52 / 58, 100 of 216 rows 13.7 / 15.3 / 19.8 / 28.7, 400 of 750 rows (long variant)
    // 87 / 96 / 112 / 123.
    const int kmin = whole((64 / esize + a.Cg - 1) / a.Cg);
    const int64_t mean = a.B ? a.M / a.B : 0;
    int k = kmin;
    p.size = 0;
    if (lanes(kmin) > 256) {
        p.size = 2;
    } else {
        for (int w = whole(2 * k); k < a.G && lanes(w) <= 64 && (int64_t)nrs * (256 / lanes(w)) >= mean && (int64_t)a.B * ((a.G + w - 1) / w) >= 1024; w = whole(2 * k)) k = w;
        if (p.uni && p.V == 4 && (int64_t)nrs * (256 / lanes(kmin)) < mean) p.size = 1;
    }
    if (getenv("GN_T")) p.size = p.uni && p.V == 4 ? atoi(getenv("GN_T")) : 0;
    if (getenv("GN_W")) k = whole(std::max(1, atoi(getenv("GN_W")) / a.Cg));
    const int threads = p.size == 2 ? 1024 : 256, nr = p.size == 1 ? nrl : nrs;
    g.k = k;
    g.nslab = (a.G + k - 1) / k;
    g.CL = lanes(k);
    g.RL = threads / g.CL;
    g.lcl = -1;
    for (int i = 0; i <= 6; ++i)
        if (g.CL == 1 << i) g.lcl = i;
    g.cw = p.uni ? a.Cg / p.V : a.Cg;
    g.fast = p.uni && g.lcl >= 0 && (g.cw & (g.cw - 1)) == 0;
    g.quads = (a.C + 3) / 4;
    g.dCL = divide_by(g.CL), g.dCg = divide_by(a.Cg);
    const int64_t cap = (int64_t)nr * g.RL;
    g.NW = (int)std::min<int64_t>(ceil_div64(a.M, MIN_WINDOW), max_windows(a.C));
    g.CH = g.NW ? (int)ceil_div64(a.M, g.NW) : 1;
    g.Tl = (int)std::max<int64_t>(std::max<int64_t>(2 * cap, 1024), g.CH);
    g.NW = a.M <= g.Tl ? 0 : (int)ceil_div64(a.M, g.CH);
    g.U = a.B;
    g.units = 0;
    p.blocks0 = (unsigned)(align_up64((int64_t)g.U + g.NW, 8) * g.nslab);
    p.blocks1 = (unsigned)(align_up64(g.NW, 8) * g.nslab);
    // LDS: row partials of kb quantities (or two buffers of the waves' sums, or the columns of one parameter gradient), the columns' totals
    // of kb quantities, the groups' sums of all
    const int ns = p.uni ? 1 : p.V, cols = g.CL * ns;
    g.kb = std::max(1, std::min(K, 8192 / (g.RL * cols)));
    g.red = g.fast ? 2 * K * (threads / 64) * g.k : g.kb * g.RL * cols;
    if (params) g.red = std::max(g.red, (g.lcl >= 0 ? threads / 64 : g.RL) * g.CL * p.V);
    p.lds = sizeof(float) * ((size_t)g.red + g.kb * cols + K * g.k);
    return p;
}

inline bool aligned16(std::initializer_list<const void*> ps) {
    uintptr_t m = 0;
    for (const void* p : ps) m |= (uintptr_t)p;
    return (m & 15) == 0;
}

template <typename T>
int zero(const GN& a, void* Y, hipStream_t st) {
    if (a.M) k_zero_rest<T><<<rest_blocks(a.M, a.C), 256, 0, st>>>(a, (T*)Y, nullptr);
    DD3D_CHECK_LAUNCH();
    return 0;
}

template <typename T>
int bwd(const GN& a, const void* dY, const void* X, const float* mean, const float* rstd, void* dX, void* dW, void* dB, hipStream_t st) {
    if (a.M && dX) {
        k_zero_rest<T><<<rest_blocks(a.M, a.C), 256, 0, st>>>(a, (T*)dX, nullptr);
        if (a.B) k_bwd_x<T><<<(unsigned)(a.B * a.G), 256, 0, st>>>(a, (const T*)dY, (const T*)X, mean, rstd, (T*)dX);
    }
    if (dW || dB) k_bwd_p<T><<<a.C, 256, 0, st>>>(a, (const T*)dY, (const T*)X, mean, rstd, dW, dB);
    DD3D_CHECK_LAUNCH();
    return 0;
}
template <typename T>
int bwd2(const GN& a, const void* P, const void* q, const void* s, const void* dY, const void* X, const float* mean, const float* rstd, void* ddY, void* ddX,
         void* dW, void* dB, void* ws, hipStream_t st) {
    const Second<T> z = {(const T*)P, q, s};
    if (a.M && (ddY || ddX)) k_zero_rest<T><<<rest_blocks(a.M, a.C), 256, 0, st>>>(a, (T*)ddY, (T*)ddX);
    if (a.B)
        k_bwd2_x<T><<<(unsigned)(a.B * a.G), 256, 0, st>>>(a, z, (const T*)dY, (const T*)X, mean, rstd, (T*)ddY, (T*)ddX, (Means*)ws);
    if (dW || dB) k_bwd2_p<T><<<a.C, 256, 0, st>>>(a, z, (const T*)dY, (const T*)X, mean, rstd, (const Means*)ws, dW, dB);
    DD3D_CHECK_LAUNCH();
    return 0;
}

}  // namespace

// See include/dd3d.h.
DD3D_API int64_t dd3d_group_norm_ws_bytes(int64_t M, int C, int B, int G, int order) {
    if (M < 0 || B < 0 || C <= 0 || G <= 0 || C % G != 0 || order < 0 || order > 2) return DD3D_EARG;
    if (M >= (1ll << 31) || C > 4096 || (int64_t)B * G >= (1ll << 31)) return DD3D_ESIZE;
    const int64_t slots = 2 * (M > MIN_WINDOW ? std::min<int64_t>(ceil_div64(M, MIN_WINDOW), max_windows(C)) : 0);
    if (order == 0) return slots * (G * 2 * (int64_t)sizeof(float) + (int64_t)sizeof(int));
    return order == 2 ? (int64_t)B * G * sizeof(Means) : 0;
}

DD3D_API int dd3d_group_norm_fwd(const void* X, int dtype, int64_t M, int C, const int32_t* seg_off, int B, int G, const void* weight, const void* bias,
                                 int pdtype, float eps, int act, float slope, double p, const int64_t* key, void* Y, float* mean, float* rstd, void* ws,
                                 int64_t ws_bytes, void* stream) {
    GN a;
    const int rc = check(dtype, M, C, seg_off, B, G, weight, bias, pdtype, act, slope, p, key, &a);
    if (rc) return rc;
    if (!(eps > 0.f) || (!mean != !rstd) || (M > 0 && (!X || !Y))) return DD3D_EARG;
    a.eps = eps;
    if (M == 0 && B == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    if (ws_bytes < dd3d_group_norm_ws_bytes(M, C, B, G, 0) || (ws_bytes > 0 && !ws)) return DD3D_EWS;
    if (B == 0) return dtype == DD3D_F32 ? zero<float>(a, Y, st) : zero<half_t>(a, Y, st);
    const gn::Plan q = plan(a, act, dtype == DD3D_F32 ? 4 : 2, aligned16({X, Y}), 2, gn::FWD_NRS, gn::FWD_NRL, false);
    return dtype == DD3D_F32   ? gn::launch_fwd<float>(a, q, X, Y, mean, rstd, (float*)ws, (int*)((float*)ws + 4ll * q.g.NW * G), st)
           : dtype == DD3D_F16 ? gn::launch_fwd<half_t>(a, q, X, Y, mean, rstd, (float*)ws, (int*)((float*)ws + 4ll * q.g.NW * G), st)
                               : gn::launch_fwd<bf16_t>(a, q, X, Y, mean, rstd, (float*)ws, (int*)((float*)ws + 4ll * q.g.NW * G), st);
}

DD3D_API int dd3d_group_norm_bwd(const void* dY, const void* X, int dtype, int64_t M, int C, const int32_t* seg_off, int B, int G, const void* weight,
                                 const void* bias, int pdtype, int act, float slope, double p, const int64_t* key, const float* mean, const float* rstd,
                                 void* dX, void* dweight, void* dbias, void* ws, int64_t ws_bytes, void* stream) {
    GN a;
    const int rc = check(dtype, M, C, seg_off, B, G, weight, bias, pdtype, act, slope, p, key, &a);
    if (rc) return rc;
    if ((M > 0 && (!X || !dY)) || (B > 0 && (!mean || !rstd))) return DD3D_EARG;
    hipStream_t st = (hipStream_t)stream;
    return dtype == DD3D_F32   ? bwd<float>(a, dY, X, mean, rstd, dX, dweight, dbias, st)
           : dtype == DD3D_F16 ? bwd<half_t>(a, dY, X, mean, rstd, dX, dweight, dbias, st)
                               : bwd<bf16_t>(a, dY, X, mean, rstd, dX, dweight, dbias, st);
}

DD3D_API int dd3d_group_norm_bwd2(const void* ggX, const void* ggW, const void* ggB, const void* dY, const void* X, int dtype, int64_t M, int C,
                                  const int32_t* seg_off, int B, int G, const void* weight, const void* bias, int pdtype, int act, float slope, double p,
                                  const int64_t* key, const float* mean, const float* rstd, void* ddY, void* ddX, void* ddweight, void* ddbias, void* ws,
                                  int64_t ws_bytes, void* stream) {
    GN a;
    const int rc = check(dtype, M, C, seg_off, B, G, weight, bias, pdtype, act, slope, p, key, &a);
    if (rc) return rc;
    if ((M > 0 && (!X || !dY)) || (B > 0 && (!mean || !rstd))) return DD3D_EARG;
    if (ws_bytes < dd3d_group_norm_ws_bytes(M, C, B, G, 2) || (B > 0 && !ws)) return DD3D_EWS;
    hipStream_t st = (hipStream_t)stream;
    return dtype == DD3D_F32   ? bwd2<float>(a, ggX, ggW, ggB, dY, X, mean, rstd, ddY, ddX, ddweight, ddbias, ws, st)
           : dtype == DD3D_F16 ? bwd2<half_t>(a, ggX, ggW, ggB, dY, X, mean, rstd, ddY, ddX, ddweight, ddbias, ws, st)
                               : bwd2<bf16_t>(a, ggX, ggW, ggB, dY, X, mean, rstd, ddY, ddX, ddweight, ddbias, ws, st);
}
