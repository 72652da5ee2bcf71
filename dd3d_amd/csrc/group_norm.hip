// Group norm with an activation (and optional dropout behind it) over ragged channels-last rows: X[M, C], cloud b owns rows
// seg_off[b] .. seg_off[b+1], group j the channels j*Cg .. (j+1)*Cg, Cg = C / G.  Per (cloud, group) with n = rows * Cg elements:
//   mean, biased var, r = (var + eps)^-1/2, xh = (x - mean) r, u = w xh + b, y = D phi(u)            (D: dropout, keep / (1 - p))
// First gradient:   g = dy D phi'(u), h = w g, dx = r (h - m(h) - xh m(h xh)), dw = sum_rows g xh, db = sum_rows g       (m: mean over n)
// Second gradient, cotangents P of dx, q of dw, s of db:
//   v = r (P - m(P) - xh m(P xh)),  gb = w v + q xh + s,  d(dy) = gb D phi',  ub = gb dy D phi''
//   X = -r (h m(P xh) + P m(h xh)) + q g + w ub
//   d(x) = r (X - m(X) - xh (m(X xh) + r (m(P h) - m(P) m(h) - m(P xh) m(h xh)))),  d(w) = sum_rows (g v + ub xh),  d(b) = sum_rows ub
// m(X) and m(X xh) follow from sums that one pass over the rows gives (group_norm.h).  The kernels: group_norm.h.  Here: argument checks, launch geometry, parameter gradients.
#include "group_norm.h"

#include <algorithm>
#include <initializer_list>

namespace {

// rows of [0, M) that belong to no cloud: all of them when there is no cloud
__global__ __launch_bounds__(256) void k_zero(uint32_t* y, int64_t words) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) y[i] = 0;
}
__global__ void k_zero_half(uint16_t* y, int64_t n) {
    if (threadIdx.x == 0 && n > 0) y[n - 1] = 0;   // the odd last element of a half-width matrix
}

__global__ __launch_bounds__(1024) void k_fold(gn::Norm a, gn::Geo g, gn::Work w, gn::Fold f) {
    __shared__ float lds[1024];
    gn::fold_slots<1024>(a, g, w, f, lds);
}

// ---- launch geometry --------------------------------------------------------------------------------------------------------------
// windows of the whole batch: enough to fill the chip with the slabs of a row, never so many that joining them shows
inline int max_windows(int C) { return C >= 1024 ? 64 : C <= 64 ? 1024 : 65536 / C; }
constexpr int MIN_WINDOW = 512, MAX_UNITS = 2048;
// Workgroups of a windows' launch: three a compute unit, all at once.  Seven clouds of 57 000 rows of 96 bf16 channels, forward / backward:
// 59 / 104 us, with 512 workgroups 70 / 124, with 2048 68 / 110 (a second round starts as the first ends).
constexpr int WINDOW_GROUPS = 768;

inline int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

inline gn::Div divide_by(int d) {
    gn::Div r;
    r.d = d, r.mul = d == 1 ? 0 : (uint32_t)((0x100000000ull + d - 1) / d);
    return r;
}

// workgroups that take whole clouds (times slabs): one a cloud, or as few as deal the clouds out evenly and stay below MAX_UNITS where each
// leaves its part of the parameter gradients, else below what a grid of at most 256 slabs and 2^32 threads holds (60 000 clouds of two
// rows of 128 fp32 channels, forward: 164 us, a workgroup each 209)
inline int cloud_units(int B, bool params) {
    const int most = params ? MAX_UNITS : 32768;
    return B > most ? (int)ceil_div64(B, ceil_div64(B, most)) : B;
}

// sums: quantities summed at once; nr: vectors a thread holds in the variants for short and long clouds; params: column_sums is called
constexpr int NR_STREAM[3] = {16, 16, 16};   // the second gradient walks long clouds twice: its slabs and windows are cut as if 16 rows were held
inline gn::Plan plan(const gn::Norm& a, int act, int esize, bool aligned, int sums, const int (&nr)[3], bool params) {
    gn::Plan p;
    gn::Geo& g = p.g;
    p.fam = act_family(act);
    // Eight channels of half width to a vector where one statistic serves them all.  Two of them (groups of four) cost more registers than the wide
    // accesses give: 2560 clouds of 82 x 128 bf16 in groups of four, forward / backward / second gradient 47 / 82 / 137 us in vectors of four, 49 / 95 / 187
    // in vectors of eight; 7 clouds of 300 000 x 96 in all 52 / 92 / 150 and 51 / 88 / 184; 400 clouds of 200 000 x 128 fp16 in all with dropout 76 / 132 / 183
    // and 68 / 117 / 175.
    p.V = esize == 2 && aligned && a.Cg % 8 == 0 && a.Cg <= 2048 ? 8 : 4;
    const int m0 = p.V / gcd(a.Cg, p.V);   // groups whose channels fill whole vectors
    p.al = aligned && a.C % p.V == 0 && m0 * a.Cg <= 4096;
    p.ns = p.al && a.Cg % p.V == 0 ? 1 : 4;
    auto lanes = [&](int k) { return p.al || k >= a.G || k * a.Cg % 4 == 0 ? (k * a.Cg + p.V - 1) / p.V : (k * a.Cg + 6) / 4; };
    auto whole = [&](int k) { return k >= a.G ? a.G : p.al ? std::min(a.G, (k + m0 - 1) / m0 * m0) : k; };
    // Slab width: 64 bytes of a row at least (its neighbour reads the other half of the line into the same L2), doubled while a short
    // cloud still fits one chunk and 1024 workgroups remain to fill the chip.  fp32 forward, 128 channels, us at 64 / 128 / 256 / 512
    // bytes: 2560 clouds of 82 rows 105 / 66 / 53 / 59, 100 of 216 rows 13.7 / 16.0 / 20.3 / 29.6, 400 of 750 rows (long variant)
    // 88 / 98 / 120 / 138.  Less than 64 bytes where that leaves less than 512 workgroups (97 clouds of 309 rows, 100 channels in groups of
    // 20, fp16: 31 us at 40 bytes, 44 at 80; backward 39 and 58).
    const int kmin = whole((64 / esize + a.Cg - 1) / a.Cg);
    const int64_t mean = a.B ? a.M / a.B : 0, shorter = nr[p.V == 8 ? 2 : 0];   // rows a thread holds, short variant
    int k = kmin;
    const int64_t pieces = a.B + std::min<int64_t>(a.M / MIN_WINDOW, WINDOW_GROUPS);   // clouds and windows
    while (k > 1 && pieces * ((a.G + k - 1) / k) < 512 && whole(k / 2) < k) k = whole(k / 2);
    p.size = 0;
    if (lanes(k) > 256) {
        p.size = 2;
    } else {
        for (int w = whole(2 * k); k < a.G && lanes(w) <= 64 && shorter * (256 / lanes(w)) >= mean && (int64_t)a.B * ((a.G + w - 1) / w) >= 1024; w = whole(2 * k)) k = w;
        if (p.ns == 1 && p.V == 4 && shorter * (256 / lanes(k)) < mean) p.size = 1;
    }
    const int threads = p.size == 2 ? 1024 : 256;
    g.k = k;
    g.nslab = (a.G + k - 1) / k;
    g.CL = lanes(k);
    g.RL = threads / g.CL;
    g.lcl = -1;
    for (int i = 0; i <= 6; ++i)
        if (g.CL == 1 << i) g.lcl = i;
    g.cw = std::max(1, a.Cg * p.ns / p.V);
    g.fast = p.al && g.lcl >= 0 && (p.ns == 1 ? (g.cw & (g.cw - 1)) == 0 : g.cw == 1);
    g.quads = (a.C + 3) / 4;
    g.dCL = divide_by(g.CL), g.dCg = divide_by(a.Cg);
    const int64_t cap = (p.size == 1 ? nr[1] : shorter) * g.RL;   // rows of a chunk
    g.NW = (int)std::min<int64_t>(std::min<int64_t>(ceil_div64(a.M, MIN_WINDOW), max_windows(a.C)), std::max(64, WINDOW_GROUPS / g.nslab));
    g.CH = g.NW ? (int)ceil_div64(a.M, g.NW) : 1;
    g.Tl = (int)std::max<int64_t>(2 * cap, g.CH);
    g.NW = a.M <= g.Tl ? 0 : (int)ceil_div64(a.M, g.CH);
    g.U = cloud_units(a.B, params);
    g.units = g.hold = 0;
    p.blocks0 = (unsigned)(align_up64((int64_t)g.U + g.NW, 8) * g.nslab);
    p.blocks1 = (unsigned)(align_up64(g.NW, 8) * g.nslab);
    // LDS: row partials of kb quantities (or two buffers of the waves' sums, or the columns of one parameter gradient), the columns' totals
    // of kb quantities, the groups' sums of all
    const int cols = g.CL * p.ns;
    g.kb = std::max(1, std::min(sums, 8192 / (g.RL * cols)));
    g.red = g.fast ? 2 * sums * (threads / 64) * g.k : g.kb * g.RL * cols;
    if (params) g.red = std::max(g.red, (g.lcl >= 0 ? threads / 64 : g.RL) * g.CL * p.V);
    p.lds = sizeof(float) * std::max<size_t>((size_t)g.red + g.kb * cols + std::max(sums, 3) * g.k, params ? threads : 0);
    return p;
}

// The workspace: piece sums, units' slots, pieces per window.  Sized by bounds that hold for every type and alignment.
struct Layout {
    int64_t part, slots, found, bytes;
};
inline Layout layout(int64_t M, int C, int B, int G, int order) {
    const int64_t windows = M > MIN_WINDOW ? std::min<int64_t>(ceil_div64(M, MIN_WINDOW), max_windows(C)) : 0;
    const int64_t units = order && B ? cloud_units(B, true) + windows : 0;
    Layout l;
    int64_t at = 0;
    auto take = [&](int64_t words) {
        const int64_t here = at;
        at = align_up64(at + words * 4, 256);
        return here;
    };
    l.part = take(2 * windows * G * (order == 2 ? 14 : order == 1 ? 2 : 3));
    l.slots = take(units * 2 * C);
    l.found = take(windows);
    l.bytes = at;
    return l;
}
inline gn::Work work_at(void* ws, const Layout& l, bool params) {
    char* p = (char*)ws;
    gn::Work w;
    w.part = (float*)(p + l.part), w.slots = params ? (float*)(p + l.slots) : nullptr, w.found = (int*)(p + l.found);
    return w;
}
inline gn::Fold fold_for(const gn::Norm& a, void* dw, void* db) { return gn::Fold{(unsigned)ceil_div64(2 * a.C, 8), dw, db}; }

inline bool aligned16(std::initializer_list<const void*> ps) {
    uintptr_t m = 0;
    for (const void* p : ps) m |= (uintptr_t)p;
    return (m & 15) == 0;
}

// argument checks shared by the three entry points; 0 = fill in `a`, take the statistics' flag off `act` and go on
inline int check(int dtype, int64_t M, int C, const int32_t* seg, int B, int G, const void* W, const void* Bi, int pdt, int& act, float slope, double p,
                 const int64_t* key, gn::Norm* a) {
    if (M < 0 || B < 0 || C <= 0 || G <= 0 || C % G != 0) return DD3D_EARG;
    if (M > gn::MOST || C > 4096 || (int64_t)B * G > gn::MOST) return DD3D_ESIZE;
    a->low = act >= 0 && (act & DD3D_ACT_LOW_MEANS);
    if (a->low) act &= ~DD3D_ACT_LOW_MEANS;
    if (dtype < DD3D_F32 || dtype > DD3D_BF16 || (pdt != DD3D_F32 && pdt != dtype) || act < DD3D_ACT_NONE || act > DD3D_ACT_GELU) return DD3D_EARG;
    if (slope != slope || (B > 0 && !seg) || !make_drop(p, key, &a->drop)) return DD3D_EARG;
    a->M = (int)M, a->C = C, a->B = B, a->G = G, a->Cg = C / G, a->pdt = pdt, a->seg = seg, a->W = W, a->Bi = Bi;
    a->slope = act == DD3D_ACT_NONE ? 1.f : act == DD3D_ACT_RELU ? 0.f : slope;
    a->eps = 0.f;
    return 0;
}

inline int zero(void* y, const gn::Norm& a, int esize, hipStream_t st) {
    const int64_t n = (int64_t)a.M * a.C, words = n * esize / 4;
    if (!y || n == 0) return 0;
    if (words) k_zero<<<(unsigned)std::min<int64_t>(ceil_div64(words, 256), 2048), 256, 0, st>>>((uint32_t*)y, words);
    if (n * esize % 4) k_zero_half<<<1, 64, 0, st>>>((uint16_t*)y, n);
    DD3D_CHECK_LAUNCH();
    return 0;
}
// parameter gradients of no cloud at all
inline int zero_params(const gn::Norm& a, void* dw, void* db, hipStream_t st) {
    if (!dw && !db) return 0;
    const gn::Fold f = fold_for(a, dw, db);
    k_fold<<<f.blocks, 1024, 0, st>>>(a, gn::Geo{}, gn::Work{}, f);
    DD3D_CHECK_LAUNCH();
    return 0;
}
inline int esize_of(int dtype) { return dtype == DD3D_F32 ? 4 : 2; }

}  // namespace

int gn::launch_fold(const Norm& a, const Plan& p, const Work& w, Fold f, hipStream_t st) {
    k_fold<<<f.blocks, 1024, 0, st>>>(a, p.g, w, f);
    DD3D_CHECK_LAUNCH();
    return 0;
}

// See include/dd3d.h.
DD3D_API int64_t dd3d_group_norm_ws_bytes(int64_t M, int C, int B, int G, int order) {
    if (M < 0 || B < 0 || C <= 0 || G <= 0 || C % G != 0 || order < 0 || order > 2) return DD3D_EARG;
    if (M > gn::MOST || C > 4096 || (int64_t)B * G > gn::MOST) return DD3D_ESIZE;
    return layout(M, C, B, G, order).bytes;
}

DD3D_API int dd3d_group_norm_fwd(const void* X, int dtype, int64_t M, int C, const int32_t* seg_off, int B, int G, const void* weight, const void* bias,
                                 int pdtype, float eps, int act, float slope, double p, const int64_t* key, void* Y, float* mean, float* rstd, void* ws,
                                 int64_t ws_bytes, void* stream) {
    gn::Norm a;
    const int rc = check(dtype, M, C, seg_off, B, G, weight, bias, pdtype, act, slope, p, key, &a);
    if (rc) return rc;
    if (!(eps >= 1.17549435e-38f && eps <= 3.4e38f) || (!mean != !rstd) || (M > 0 && (!X || !Y))) return DD3D_EARG;
    a.eps = eps;
    const Layout l = layout(M, C, B, G, 0);
    if (ws_bytes < l.bytes || (l.bytes > 0 && !ws)) return DD3D_EWS;
    hipStream_t st = (hipStream_t)stream;
    if (B == 0) return zero(Y, a, esize_of(dtype), st);
    const gn::Plan q = plan(a, act, esize_of(dtype), aligned16({X, Y}), 2, gn::NR_FWD, false);
    const gn::Work w = work_at(ws, l, false);
    return dtype == DD3D_F32   ? gn::launch_fwd<float>(a, q, X, Y, mean, rstd, w, st)
           : dtype == DD3D_F16 ? gn::launch_fwd<half_t>(a, q, X, Y, mean, rstd, w, st)
                               : gn::launch_fwd<bf16_t>(a, q, X, Y, mean, rstd, w, st);
}

DD3D_API int dd3d_group_norm_bwd(const void* dY, const void* X, int dtype, int64_t M, int C, const int32_t* seg_off, int B, int G, const void* weight,
                                 const void* bias, int pdtype, int act, float slope, double p, const int64_t* key, const float* mean, const float* rstd,
                                 void* dX, void* dweight, void* dbias, void* ws, int64_t ws_bytes, void* stream) {
    gn::Norm a;
    int rc = check(dtype, M, C, seg_off, B, G, weight, bias, pdtype, act, slope, p, key, &a);
    if (rc) return rc;
    if ((M > 0 && (!X || !dY)) || (B > 0 && (!mean || !rstd))) return DD3D_EARG;
    const Layout l = layout(M, C, B, G, 1);
    if (ws_bytes < l.bytes || (l.bytes > 0 && !ws)) return DD3D_EWS;
    hipStream_t st = (hipStream_t)stream;
    if (B == 0) {
        rc = zero(dX, a, esize_of(dtype), st);
        return rc ? rc : zero_params(a, dweight, dbias, st);
    }
    const bool params = dweight || dbias;
    if (!params && !dX) return 0;
    const gn::Plan q = plan(a, act, esize_of(dtype), aligned16({X, dY, dX}), 2, gn::NR_BWD, params);
    const gn::Work w = work_at(ws, l, params);
    const gn::Fold f = fold_for(a, dweight, dbias);
    return dtype == DD3D_F32   ? gn::launch_bwd<float>(a, q, dY, X, mean, rstd, dX, w, f, st)
         : dtype == DD3D_F16 ? gn::launch_bwd<half_t>(a, q, dY, X, mean, rstd, dX, w, f, st)
                             : gn::launch_bwd<bf16_t>(a, q, dY, X, mean, rstd, dX, w, f, st);
}

DD3D_API int dd3d_group_norm_bwd2(const void* ggX, const void* ggW, const void* ggB, const void* dY, const void* X, int dtype, int64_t M, int C,
                                  const int32_t* seg_off, int B, int G, const void* weight, const void* bias, int pdtype, int act, float slope, double p,
                                  const int64_t* key, const float* mean, const float* rstd, void* ddY, void* ddX, void* ddweight, void* ddbias, void* ws,
                                  int64_t ws_bytes, void* stream) {
    gn::Norm a;
    int rc = check(dtype, M, C, seg_off, B, G, weight, bias, pdtype, act, slope, p, key, &a);
    if (rc) return rc;
    if ((M > 0 && (!X || !dY)) || (B > 0 && (!mean || !rstd))) return DD3D_EARG;
    const Layout l = layout(M, C, B, G, 2);
    if (ws_bytes < l.bytes || (l.bytes > 0 && !ws)) return DD3D_EWS;
    hipStream_t st = (hipStream_t)stream;
    if (B == 0) {
        rc = zero(ddY, a, esize_of(dtype), st);
        if (!rc) rc = zero(ddX, a, esize_of(dtype), st);
        return rc ? rc : zero_params(a, ddweight, ddbias, st);
    }
    const bool params = ddweight || ddbias;
    if (!params && !ddY && !ddX) return 0;
    const gn::Plan q = plan(a, act, esize_of(dtype), aligned16({X, dY, ggX, ddY, ddX}), act_family(act) == DD3D_FAM_LINEAR ? 7 : 14, NR_STREAM, params);
    const gn::Work w = work_at(ws, l, params);
    const gn::Fold f = fold_for(a, ddweight, ddbias);
    return dtype == DD3D_F32   ? gn::launch_bwd2<float>(a, q, ggX, ggW, ggB, dY, X, mean, rstd, ddY, ddX, w, f, st)
         : dtype == DD3D_F16 ? gn::launch_bwd2<half_t>(a, q, ggX, ggW, ggB, dY, X, mean, rstd, ddY, ddX, w, f, st)
                             : gn::launch_bwd2<bf16_t>(a, q, ggX, ggW, ggB, dY, X, mean, rstd, ddY, ddX, w, f, st);
}
