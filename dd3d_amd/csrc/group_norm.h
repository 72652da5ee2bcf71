// Device code of the group norm (formulas: group_norm.hip), shared by its three passes and instantiated per row type and pass in group_norm_*.hip.
//
// The passes need sums over (cloud, group) before anything can be written, so a row has to be read twice unless it stays on chip in between.
// Large batches of fp32 rows are bound by HBM: 210 000 x 128 in 2560 clouds, SiLU, forward 50 us (4.3 TB/s), backward 84 (3.8); second
// gradient of 300 000 x 128 in 400 clouds, GELU, 222 (3.5, and 4.8 with what it reads twice).  Half-width rows are bound by vector instructions,
// which fill 99% of the SIMDs' cycles in the forward pass of 210 000 x 128 bf16 with GELU (45 us), as is the forward pass with GELU and dropout (400 000
// x 128 fp32: 119 us, 83%; 28 of a row's 198 instructions read spilled scalars back).  Layout of the work:
//   * a SLAB is a run of whole groups, 64 bytes of a row at least; a workgroup owns one slab of one cloud after another.  Thread t holds V
//     channels (one 16-byte vector) of the rows rl, rl + RL, ...: the rows of a chunk of NR * RL are loaded at once into registers, so up to
//     that many loads are in flight per thread, and stay there while the workgroup forms the sums -- HBM sees every row once.  Four waves
//     a workgroup: with sixteen the instructions that every wave spends on the sums outweighed the rows (2560 clouds of 82 rows of 128
//     channels, fp32 forward, before the sums went by lane exchanges: 97 us against 64).  Sixteen only where a slab has more than 256 vectors.
//   * a cloud longer than one chunk and up to `Tl` rows is walked again by the same workgroup (its slab mostly comes out of the caches).
//   * a longer cloud ("large") is cut by WINDOWS of CH rows of the whole batch; Tl >= CH, so a window meets at most two large clouds: the
//     one it begins in (slot 2w) and one that begins inside it (slot 2w + 1).  Windows write partial sums, a second launch joins them
//     (every workgroup for itself, in window order) and walks the rows again.  Which clouds are large is read from seg_off on the device.
// Sums are fp32: per thread over its rows, then lanes, waves, windows in a fixed order.  Variances come from differences to a mean
// at every level (thread, workgroup, windows), never from a mean of squares; and the mean of those differences is added to the mean they were
// taken to, so that neither the sum's roundings nor a reciprocal's stay in it: a constant cloud is centred to zeros.  Of fp32 rows a mean is held in
// two floats, as its rounding to one is a visible part of the spread of values that lie close together (3000 clouds, half of them of two or three rows,
// a group a channel: dx is 4.6e-6 off with one float, 2.2e-7 with two).  Values of half width cannot lie that close.
#pragma once
#include "feature_math.h"

namespace gn {

// Rows, clouds, and clouds times groups of one call: 65536 below 2^31, so that a counter which a loop has moved past its end by one step (a chunk of
// 4096 rows at most, or the 32768 clouds that lie between two of one workgroup) is still a positive 32-bit number.
constexpr int64_t MOST = (1ll << 31) - 65536;

struct Norm {
    int M, C, B, G, Cg, pdt;   // M, B <= MOST: row and cloud numbers fit 32 bits, element offsets do not
    const int* seg;
    const void *W, *Bi;
    float eps, slope;
    bool low;                  // behind the B * G means lie what their roundings left of them
    Drop drop;
};

// n / d for n, d < 2^16 as one wide product
struct Div {
    uint32_t mul;
    int d;
};
__device__ __forceinline__ int quot(int n, const Div& d) { return d.d == 1 ? n : (int)__umulhi((uint32_t)n, d.mul); }

// launch geometry (plan() in group_norm.hip); everything is uniform
struct Geo {
    int k, nslab;        // groups per slab, slabs
    int CL, RL, lcl;     // channel lanes (vectors per row of the slab), row lanes, log2(CL) if CL is a power of two <= 64, else -1
    int cw;              // columns of one group (a column: the channels of a vector that share a statistic)
    int fast;            // slabs, and groups wider than a vector, are powers of two of lanes: sums by lane exchanges
    int U, NW, CH, Tl;   // cloud units, windows, rows per window, longest cloud that one workgroup takes
    int units;           // of this launch
    int quads;           // ceil(C / 4)
    int kb;              // quantities reduced at once where the sums go through LDS
    int red;             // floats of LDS for them
    int hold;            // where in LDS (floats) the second gradient keeps a cloud's first chunk, 0: nowhere
    Div dCL, dCg;
};

// ---- one thread's V channels of one row --------------------------------------------------------------------------------------
template <typename T, int V>
struct Raw {
    uint32_t __attribute__((ext_vector_type(V * (int)sizeof(T) / 4))) u;
};
__device__ __forceinline__ float raw_get(const Raw<float, 4>& r, int i) { return __uint_as_float(r.u[i]); }
template <int V>
__device__ __forceinline__ float raw_get(const Raw<half_t, V>& r, int i) {
    const uint16_t h = (uint16_t)(r.u[i >> 1] >> ((i & 1) * 16));
    half_t f;
    __builtin_memcpy(&f, &h, 2);
    return (float)f;
}
template <int V>
__device__ __forceinline__ float raw_get(const Raw<bf16_t, V>& r, int i) {
    return __uint_as_float((i & 1) ? r.u[i >> 1] & 0xFFFF0000u : r.u[i >> 1] << 16);
}

// The same row to the compiler's eye new: what an earlier pass computed from it is computed again, not kept in registers (half a dozen
// values an element) until the later pass comes.
template <typename R>
__device__ __forceinline__ R again(R r) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r.u) / 4); ++i) {
        uint32_t v = r.u[i];
        asm volatile("" : "+v"(v));
        r.u[i] = v;
    }
    return r;
}

// ---- where this thread stands ---------------------------------------------------------------------------------------------------
// The compile-time side of a launch.  NS: statistics a vector needs -- 1 where it lies inside one group (Cg % V == 0), else one per channel.  AL:
// whole, aligned vectors.
// Vectors a thread holds in the three passes: vectors of four in the variants for short and for long clouds, vectors of eight; and the
// waves per SIMD that the registers of that many rows leave.  More rows spare a long cloud its second reading until registers run out
// (400 clouds of 750 rows of 128 fp32 channels, 8 against 16: forward 99 and 74 us, backward 152 and 126); clouds that fit 8 gain from the
// waves that 8 leave.
constexpr int NR_FWD[3] = {8, 16, 8}, NR_BWD[3] = {8, 16, 4}, NR_BWD2[3] = {4, 4, 2};

template <typename T_, int V_, bool AL_, int NS_, int FAM_, int THREADS_, int NR_>
struct Cfg {
    typedef T_ T;
    static constexpr int V = V_, FAM = FAM_, THREADS = THREADS_, NR = NR_, NS = NS_, WAVES = THREADS_ / 64;
    static constexpr int PER = V_ / NS_;   // channels that share a statistic
    static constexpr bool AL = AL_, LOW = sizeof(T_) == 4;   // LOW: means in two floats
    static constexpr int FWD_WAVES = THREADS_ > 256 || NR_ <= 8 ? 4 : 3, BWD_WAVES = THREADS_ > 256 ? 4 : NR_ > 8 ? 2 : 3,
                         BWD2_WAVES = THREADS_ > 256 ? 4 : NS_ == 1 ? 3 : 2;
    static constexpr int at(int i) { return i / PER; }
    typedef Raw<T_, V_> Row;
};

template <typename Z>
struct Spot {
    int unit, slab;
    int cl, rl, wave, lane;
    int s0, s1, gs;       // channels [s0, s1) of the slab, groups
    int c0, lo, hi;       // first channel of this thread, which of its V exist in the slab
    bool on;              // this thread has rows at all
    int buf;              // which half of the sums' LDS is next
    uint32_t off, step;   // bytes from a chunk's first row to this thread's first vector, and from one of its rows to the next
    uint32_t word;        // the same in blocks of random words
    int j[Z::NS];         // group (within the slab) of its channels
    float w[Z::V], b[Z::V];
};

// V values from channel c0 of a parameter vector; channels outside the slab [s0, s1) read one that is in it
template <int V>
__device__ __forceinline__ void load_params(const void* p, int pdt, int c0, int s0, int s1, float otherwise, float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = otherwise;
    if (!p) return;
    if (pdt == DD3D_F32) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = ((const float*)p)[min(max(c0 + i, s0), s1 - 1)];
    } else {
        uint16_t h[V];
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = ((const uint16_t*)p)[min(max(c0 + i, s0), s1 - 1)];
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = widen_bits(h[i], pdt);
    }
}

// consecutive workgroups go to consecutive XCDs: the slabs of one unit are eight workgroups apart, on one XCD, so lines that two slabs
// share are fetched into one L2
__device__ __forceinline__ bool place(const Geo& g, int& unit, int& slab, unsigned first = 0) {
    const int at = blockIdx.x - first, lo = at & 7, rest = at >> 3, hi = g.nslab == 1 ? rest : rest / g.nslab;
    slab = rest - hi * g.nslab;
    unit = hi * 8 + lo;
    return unit < g.units;
}

template <typename Z>
__device__ __forceinline__ void locate(const Norm& a, const Geo& g, int unit, int slab, Spot<Z>& s) {
    s.unit = unit, s.slab = slab;
    s.lane = threadIdx.x & 63, s.wave = threadIdx.x >> 6;
    s.rl = quot(threadIdx.x, g.dCL), s.cl = threadIdx.x - s.rl * g.CL;
    s.s0 = s.slab * g.k * a.Cg;
    s.gs = min(g.k, a.G - s.slab * g.k);
    s.s1 = s.s0 + s.gs * a.Cg;
    s.c0 = (s.s0 & ~3) + s.cl * Z::V;   // from a multiple of four, where the random words' blocks begin
    s.lo = s.s0 - s.c0, s.hi = s.s1 - s.c0;
    s.on = s.rl < g.RL && s.hi > 0;
    s.buf = 0;
    s.step = g.RL * a.C * (int)sizeof(typename Z::T);
    s.off = Z::AL && !s.on ? 0x40000000u : (uint32_t)(s.rl * a.C + s.c0) * (uint32_t)sizeof(typename Z::T);   // (a chunk is far below 2^30 bytes)
    s.word = s.rl * g.quads + s.c0 / 4;
#pragma unroll
    for (int i = 0; i < Z::NS; ++i) s.j[i] = min(quot(max(s.c0 + i * Z::PER - s.s0, 0), g.dCg), s.gs - 1);
    load_params<Z::V>(a.W, a.pdt, s.c0, s.s0, s.s1, 1.f, s.w);
    load_params<Z::V>(a.Bi, a.pdt, s.c0, s.s0, s.s1, 0.f, s.b);
}

// a value the compiler must not compute ahead of the loop it is used in: a chunk's eight offsets are one addition each, and kept over the
// whole kernel they would push the rows out of the registers
__device__ __forceinline__ uint32_t here(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

// 1 / sqrt(v) of a normal v > 0: the hardware's value and one Newton step, within about a half step of the exact one at a seventh of the
// instructions of a division by a square root
__device__ __forceinline__ float rsqrt_newton(float v) {
    const float r = __builtin_amdgcn_rsqf(v);
    return fmaf(r * 0.5f, fmaf(-v * r, r, 1.f), r);
}

// a result that is finished here, not moved behind a branch that only some launches take: everything it is made of would live until there
__device__ __forceinline__ float done(float v) {
    asm volatile("" : "+v"(v));
    return v;
}

// how far the means' second floats lie behind the first ones: multiplied where it is used, as two more scalars over a whole kernel push others out
__device__ __forceinline__ int64_t means(const Norm& a) {
    int b = a.B;
    asm volatile("" : "+s"(b));
    return (int64_t)b * a.G;
}

// ---- rows of a cloud ------------------------------------------------------------------------------------------------------------
struct Range {
    int r0, r1;
};
__device__ __forceinline__ Range cloud_rows(const Norm& a, int b) {
    // uniform, and kept in scalar registers: the compiler cannot know it of a value loaded through seg
    Range r;
    r.r0 = min(max(__builtin_amdgcn_readfirstlane(a.seg[b]), 0), a.M);
    r.r1 = min(max(__builtin_amdgcn_readfirstlane(a.seg[b + 1]), r.r0), a.M);
    return r;
}

// the cloud that row `at` belongs to (-1 or B: none): 64-ary search, every wave for itself
__device__ __forceinline__ int cloud_of(const Norm& a, int at) {
    int lo = 0, n = a.B + 1;   // seg[lo - 1] <= at < seg[lo + n], over the entries seg[0 .. B]
    const int lane = threadIdx.x & 63;
    while (n > 0) {
        const int step = (n + 63) / 64, i = lo + lane * step;
        const unsigned long long m = __ballot(i < lo + n && a.seg[min(i, a.B)] <= at);
        const int c = __popcll(m);   // entries lo, lo + step, .. are <= at for the first c lanes
        if (c == 0) break;
        const int first = lo + (c - 1) * step + 1, end = min(lo + n, lo + c * step);
        lo = first, n = end - first;
    }
    return __builtin_amdgcn_readfirstlane(lo) - 1;
}

// a window's part of a large cloud
struct Piece {
    int b, slot;
    Range all, part;
};
// the number of pieces; the first launch looks for them and notes the number in found[w], the later ones read it
template <bool LOOK>
__device__ __forceinline__ int window_pieces(const Norm& a, const Geo& g, int w, int* found, Piece (&p)[2]) {
    if (!LOOK && __builtin_amdgcn_readfirstlane(found[w]) == 0) return 0;
    const int a0 = w * g.CH, a1 = a0 + min(g.CH, a.M - a0);
    int n = 0;
    const int b0 = cloud_of(a, a0), b1 = cloud_of(a, a1 - 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int b = i ? b1 : b0;
        if (b < 0 || b >= a.B || (i && b1 == b0)) continue;
        const Range r = cloud_rows(a, b);
        if (r.r1 - r.r0 <= g.Tl) continue;
        Piece q;
        q.b = b, q.all = r, q.slot = 2 * w + (r.r0 < a0 ? 0 : 1);
        q.part.r0 = max(r.r0, a0), q.part.r1 = min(r.r1, a1);
        if (n) p[1] = q;
        else p[0] = q;
        ++n;
    }
    if (LOOK && threadIdx.x == 0) found[w] = n;   // (by every slab's workgroup, the same number)
    return n;
}
// the slots of a large cloud, in window order
__device__ __forceinline__ int piece_count(const Geo& g, const Range& r) { return (r.r1 - 1) / g.CH - r.r0 / g.CH + 1; }
__device__ __forceinline__ int piece_slot(const Geo& g, const Range& r, int i) { return 2 * (r.r0 / g.CH + i) + (i == 0 ? 1 : 0); }
__device__ __forceinline__ int piece_rows(const Geo& g, const Range& r, int i) {
    const int w0 = (r.r0 / g.CH + i) * g.CH;
    return min(r.r1 - w0, g.CH) - max(r.r0 - w0, 0);
}

// rows of [0, M) in no cloud: zeros, shared out over all workgroups of the launch
template <typename T>
__device__ __forceinline__ void zero_rest(const Norm& a, T* Y) {
    if (!Y) return;
    const int lo = min(max(a.seg[0], 0), a.M), hi = min(max(a.seg[a.B], lo), a.M);
    const int64_t n0 = (int64_t)lo * a.C, n = n0 + (int64_t)(a.M - hi) * a.C;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
        Y[i < n0 ? i : (int64_t)hi * a.C + (i - n0)] = narrow<T>(0.f);
}

// ---- lanes' sums without the LDS crossbar ---------------------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xF, 0xF, true));
}
// v + the value 16 (32) lanes away: a row swap of v with itself leaves the two halves of every pair side by side
__device__ __forceinline__ float add_row16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_row32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// sum over aligned blocks of `n` lanes (a power of two); all lanes of a block hold it
template <int K>
__device__ __forceinline__ void add_block(float (&v)[K], int n) {
    if (n > 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = dpp_add<0xB1>(v[k]);    // quad_perm 1 0 3 2
    if (n > 2)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = dpp_add<0x4E>(v[k]);    // quad_perm 2 3 0 1
    if (n > 4)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = dpp_add<0x141>(v[k]);   // row_half_mirror: the other quad of eight
    if (n > 8)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = dpp_add<0x140>(v[k]);   // row_mirror: the other eight of sixteen
    if (n > 16)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = add_row16(v[k]);
    if (n > 32)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = add_row32(v[k]);
}
// sum over the lanes that are equal modulo `n` (a power of two); all of them hold it
template <int K>
__device__ __forceinline__ void add_strided(float (&v)[K], int n) {
    if (n <= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = dpp_add<0xB1>(v[k]);
    if (n <= 2)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = dpp_add<0x4E>(v[k]);
    if (n <= 4)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = dpp_add<0x124>(v[k]);   // row_ror 4, then 8: the four lanes of a class in sixteen
    if (n <= 8)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = dpp_add<0x128>(v[k]);
    if (n <= 16)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = add_row16(v[k]);
    if (n <= 32)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = add_row32(v[k]);
}

// ---- sums -----------------------------------------------------------------------------------------------------------------------
// v[q][i], per thread and statistic -> the sum over the rows of the workgroup and the channels of the group that the statistic belongs to.  Lanes without rows bring zeros.
template <int K, typename Z>
__device__ __forceinline__ void group_sums(float (&v)[K][Z::NS], const Norm& a, const Geo& g, Spot<Z>& s, float* lds) {
    constexpr int NS = Z::NS;
    if (g.fast) {
        // the group's lanes, then the wave's row lanes; one value per wave and group through LDS.  Two buffers in turn: one barrier a call
        float t[K * NS];
#pragma unroll
        for (int q = 0; q < K * NS; ++q) t[q] = v[q / NS][q % NS];
        if (NS == 1) add_block(t, g.cw);
        add_strided(t, g.CL);
        float* red = lds + s.buf * (g.red >> 1);   // (a fixed half: calls of different K follow each other)
        s.buf ^= 1;
        if (s.lane < g.CL && (NS > 1 || (s.lane & (g.cw - 1)) == 0) && s.hi > 0) {
#pragma unroll
            for (int q = 0; q < K * NS; ++q)
                if (NS == 1 || q % NS * Z::PER < s.hi) red[(q / NS * Z::WAVES + s.wave) * g.k + s.j[q % NS]] = t[q];
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < K; ++q)
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                v[q][i] = 0.f;
#pragma unroll
                for (int p = 0; p < Z::WAVES; ++p) v[q][i] += red[(q * Z::WAVES + p) * g.k + s.j[i]];
            }
        return;
    }
    // through LDS: [row lane][column], summed per column, then per group
    const int cols = g.CL * NS, c_first = (s.s0 & 3) / Z::PER;   // the slab's first column
    float *tot = lds + g.red, *out = tot + g.kb * cols;
    for (int k0 = 0; k0 < K; k0 += g.kb) {
        const int kn = min(K - k0, g.kb);
        __syncthreads();
        if (s.rl < g.RL) {
#pragma unroll
            for (int q = 0; q < K; ++q)
                if (q >= k0 && q < k0 + kn) {
#pragma unroll
                    for (int i = 0; i < Z::NS; ++i) lds[((q - k0) * g.RL + s.rl) * cols + s.cl * Z::NS + i] = v[q][i];
                }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < kn * cols; c += Z::THREADS) {
            const int q = c / cols;
            const float* from = lds + q * g.RL * cols + (c - q * cols);
            float t = 0.f;
            for (int p = 0; p < g.RL; ++p) t += from[p * cols];
            tot[c] = t;
        }
        __syncthreads();
        // eight lanes a group
        for (int jb = threadIdx.x >> 3; jb < kn * s.gs; jb += Z::THREADS / 8) {
            const int q = jb / s.gs, j = jb - q * s.gs;
            float t = 0.f;
            for (int i = threadIdx.x & 7; i < g.cw; i += 8) t += tot[q * cols + c_first + j * g.cw + i];
            t += __shfl_xor(t, 1, 64);
            t += __shfl_xor(t, 2, 64);
            t += __shfl_xor(t, 4, 64);
            if ((threadIdx.x & 7) == 0) out[(k0 + q) * g.k + j] = t;
        }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < K; ++q)
#pragma unroll
        for (int i = 0; i < Z::NS; ++i) v[q][i] = out[q * g.k + s.j[i]];
}

// acc[q][i] per thread and channel -> slot[q * C + c], the sum over the workgroup's rows (parameter gradients, once a workgroup)
template <int K, typename Z>
__device__ __forceinline__ void column_sums(float (&acc)[K][Z::V], const Norm& a, const Geo& g, const Spot<Z>& s, float* lds, float* slot) {
    int np = g.RL;
    const int cols = g.CL * Z::V;
    if (g.lcl >= 0) {
        for (int o = g.CL; o < 64; o <<= 1) {
#pragma unroll
            for (int q = 0; q < K; ++q)
#pragma unroll
                for (int i = 0; i < Z::V; ++i) acc[q][i] += __shfl_xor(acc[q][i], o, 64);
        }
        np = Z::WAVES;
    }
    const int p = g.lcl >= 0 ? s.wave : s.rl;
    const bool writes = g.lcl >= 0 ? s.lane < g.CL : s.rl < g.RL;
#pragma unroll
    for (int q = 0; q < K; ++q) {
        __syncthreads();
        if (writes) {
#pragma unroll
            for (int i = 0; i < Z::V; ++i) lds[p * cols + s.cl * Z::V + i] = acc[q][i];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += Z::THREADS) {
            const int ch = (s.s0 & ~3) + c;
            float t = 0.f;
            for (int r = 0; r < np; ++r) t += lds[r * cols + c];
            if (ch >= s.s0 && ch < s.s1) slot[(int64_t)q * a.C + ch] = t;
        }
    }
}

// part[slot][G][K]: whether this thread's i-th statistic is the one that is written for its group
template <typename Z>
__device__ __forceinline__ bool writes_group(const Norm& a, const Spot<Z>& s, int i) {
    const int c = i * Z::PER;
    return s.rl == 0 && s.on && c >= s.lo && c < s.hi && s.j[i] * a.Cg == s.c0 + c - s.s0;
}
template <int K, typename Z>
__device__ __forceinline__ void put_part(float* part, int slot, const float (&v)[K][Z::NS], const Norm& a, const Geo& g, const Spot<Z>& s) {
#pragma unroll
    for (int i = 0; i < Z::NS; ++i)
        if (writes_group(a, s, i)) {
            float* to = part + ((int64_t)slot * a.G + s.slab * g.k + s.j[i]) * K;
#pragma unroll
            for (int q = 0; q < K; ++q) to[q] = v[q][i];
        }
}

// the sums of a large cloud's pieces, in window order: a wave a group, lanes over pieces
template <int K, typename Z>
__device__ __forceinline__ void join_parts(const float* part, const Range& r, float (&v)[K][Z::NS], const Norm& a, const Geo& g, const Spot<Z>& s, float* lds) {
    float* out = lds + g.red + g.kb * g.CL * Z::NS;
    const int n = piece_count(g, r);
    __syncthreads();
    for (int j = s.wave; j < s.gs; j += Z::WAVES) {
        float t[K];
#pragma unroll
        for (int q = 0; q < K; ++q) t[q] = 0.f;
        for (int o = s.lane; o < n; o += 64) {
            const float* from = part + ((int64_t)piece_slot(g, r, o) * a.G + s.slab * g.k + j) * K;
#pragma unroll
            for (int q = 0; q < K; ++q) t[q] += from[q];
        }
#pragma unroll
        for (int q = 0; q < K; ++q) {
            t[q] = wave_sum(t[q]);
            if (s.lane == 0) out[q * g.k + j] = t[q];
        }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < K; ++q)
#pragma unroll
        for (int i = 0; i < Z::NS; ++i) v[q][i] = out[q * g.k + s.j[i]];
}

// the random words of a thread's vector
template <int V>
struct Words {
    uint32_t w[V];

    __device__ __forceinline__ Words(const PhiloxKey& k, uint64_t block) {
#pragma unroll
        for (int h = 0; h < V / 4; ++h) {
            const uint4 r = philox_block(k, block + h);
            w[4 * h] = r.x, w[4 * h + 1] = r.y, w[4 * h + 2] = r.z, w[4 * h + 3] = r.w;
        }
    }
    __device__ __forceinline__ void drop(const Drop& d, float (&v)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = w[i] >= d.thr && !d.all ? v[i] * d.scale : 0.f;
    }
    __device__ __forceinline__ uint32_t bits(const Drop& d) const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) m |= w[i] >= d.thr && !d.all ? 1u << i : 0u;
        return m;
    }
};
// dropout of one row's values by kept bits, behind one uniform branch
template <int V>
__device__ __forceinline__ void drop_row(const Drop& d, uint32_t keep, float (&v)[V]) {
    if (!d.key) return;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = keep & (1u << i) ? v[i] * d.scale : 0.f;
}
__device__ __forceinline__ PhiloxKey drop_key(const Drop& d) {
    PhiloxKey k = {0, 0, 0, 0};
    if (d.key) k = philox_key(d.key);
    return k;
}

// The chunk of rows that begins at `from`, `left` rows before the end, as a buffer: an access past its last row, or by a thread without
// channels (whose offset lies past any chunk), reads zeros and writes nothing, so no access waits behind a branch and none needs its
// bounds computed.  Unaligned rows are moved element by element, under the thread's own bounds.
template <typename Z>
struct Chunk {
    typedef typename Z::T T;
    __amdgpu_buffer_rsrc_t buf;
    T* at;
    int left;

    __device__ __forceinline__ Chunk(const T* from, int C, int left_, const Geo& g) : at(const_cast<T*>(from)), left(left_) {
        if (Z::AL) buf = __builtin_amdgcn_make_buffer_rsrc(at, 0, min(left, Z::NR * g.RL) * C * (int)sizeof(T), 0x00020000);
    }
    __device__ __forceinline__ bool has(const Geo& g, const Spot<Z>& s, int n) const { return s.on && s.rl + n * g.RL < left; }

    // row n of the thread; off = here(s.off)
    __device__ __forceinline__ typename Z::Row load(const Geo& g, const Spot<Z>& s, uint32_t off, int n) const {
        typename Z::Row r;
        const uint32_t o = off + n * s.step;
        if constexpr (Z::AL && sizeof(r) == 16) {
            r.u = __builtin_amdgcn_raw_buffer_load_b128(buf, (int)o, 0, 0);
        } else if constexpr (Z::AL) {
            r.u = __builtin_amdgcn_raw_buffer_load_b64(buf, (int)o, 0, 0);
        } else {
            T e[Z::V];
#pragma unroll
            for (int i = 0; i < Z::V; ++i) e[i] = has(g, s, n) && i >= s.lo && i < s.hi ? ((const T*)((const char*)at + o))[i] : narrow<T>(0.f);
            __builtin_memcpy(&r, e, sizeof(r));
        }
        return r;
    }
    __device__ __forceinline__ void store(const Geo& g, const Spot<Z>& s, uint32_t off, int n, const float (&v)[Z::V]) const {
        typename Z::Row r;
        T e[Z::V];
        const uint32_t o = off + n * s.step;
#pragma unroll
        for (int i = 0; i < Z::V; ++i) e[i] = narrow<T>(v[i]);
        if constexpr (Z::AL) {
            __builtin_memcpy(&r, e, sizeof(r));
            if constexpr (sizeof(r) == 16) __builtin_amdgcn_raw_buffer_store_b128(r.u, buf, (int)o, 0, 0);
            else __builtin_amdgcn_raw_buffer_store_b64(r.u, buf, (int)o, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < Z::V; ++i)
                if (has(g, s, n) && i >= s.lo && i < s.hi) ((T*)((char*)at + o))[i] = e[i];
        }
    }
    // all rows of the thread
    __device__ __forceinline__ void load_all(const Geo& g, const Spot<Z>& s, typename Z::Row (&x)[Z::NR]) const {
        const uint32_t off = here(s.off);
#pragma unroll
        for (int n = 0; n < Z::NR; ++n)
            if (n * g.RL < left) x[n] = load(g, s, off, n);
    }
};
// element offset of row `base`, and its first block of random words
__device__ __forceinline__ int64_t row_at(const Norm& a, int base) { return (int64_t)base * a.C; }
__device__ __forceinline__ uint64_t words_at(const Geo& g, int base) { return (uint64_t)(uint32_t)base * (uint32_t)g.quads; }

// one row after the other: the scheduler would otherwise work on all of a chunk's rows at once and run out of registers
__device__ __forceinline__ void row_border() { __builtin_amdgcn_sched_barrier(0); }

// ---- the caller's workspace, and the parameter gradients in it --------------------------------------------------------------------
struct Work {
    float *part, *slots;   // pieces' sums; [units][2][C]
    int* found;            // pieces per window
};
struct Fold {
    unsigned blocks;       // workgroups (8 columns each) in front of the windows' launch
    void *dw, *db;
};

// out[q][c] = the sum over units of slots[unit][q][c] in a fixed order: eight columns a workgroup, THREADS / 8 row lanes, sixteen loads in
// flight a thread (latency is all there is to hide: 1300 units of 128 channels are 1.3 MB).
template <int THREADS>
__device__ __forceinline__ void fold_slots(const Norm& a, const Geo& g, const Work& w, const Fold& f, float* lds) {
    constexpr int LANES = THREADS / 8;
    const int cols = 2 * a.C, c = blockIdx.x * 8 + (threadIdx.x & 7), lane = threadIdx.x >> 3;
    float t = 0.f;
    if (c < cols) {
        const float* from = w.slots + c;
#pragma unroll 16
        for (int i = lane; i < g.U; i += LANES) t += from[(int64_t)i * cols];
#pragma unroll 8
        for (int i = lane; i < g.NW; i += LANES) {
            const float v = from[(int64_t)(g.U + i) * cols];   // read in any case: a load behind a branch would wait for the one before it
            t += w.found[i] ? v : 0.f;                         // (a window without a large cloud has written nothing)
        }
    }
    lds[threadIdx.x] = t;
    for (int n = LANES / 2; n > 0; n >>= 1) {
        __syncthreads();
        if (lane < n) lds[threadIdx.x] += lds[threadIdx.x + n * 8];
    }
    if (lane || c >= cols) return;
    void* to = c < a.C ? f.dw : f.db;
    if (to) store_param(to, a.pdt, c < a.C ? c : c - a.C, lds[threadIdx.x]);
}

// ---- forward --------------------------------------------------------------------------------------------------------------------
// The sum of squares about the mean, from the sums `e` of differences and `q` of their squares about a shift that lies shift = e / n below the mean.
// What is left below the roundings of q (2^-18: some sixty half steps) is nothing: of equal values only those are left.
__device__ __forceinline__ float about_mean(float q, float e, float shift) {
    const float r = fmaf(-e, shift, q);
    return r < q * 0x1p-18f ? 0.f : r;
}

// (x - mean) / standard deviation from x less the mean's first float; low: the second one times -rstd
template <typename Z>
__device__ __forceinline__ float normal(float d, float rstd, float low) {
    return Z::LOW ? fmaf(d, rstd, low) : d * rstd;
}

template <typename Z>
struct Fwd {
    typedef typename Z::T T;
    static constexpr int V = Z::V, NR = Z::NR, NS = Z::NS;
    const Norm& a;
    const Geo& g;
    Spot<Z>& s;
    const T* X;
    T* Y;
    float* lds;
    PhiloxKey key;

    // per-thread count, mean (mu + low) and centred sum of squares, joined with those of one more chunk
    __device__ __forceinline__ void add_rows(int all, const typename Z::Row (&z)[NR], const float (&k)[NS], float& cnt, float (&mu)[NS], float (&low)[NS], float (&m2)[NS]) {
        const int left = s.on ? all : 0;
        float n1 = 0.f, sx[NS], e[NS], q[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) sx[i] = e[i] = q[i] = 0.f;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            if (n * g.RL >= all) break;
            n1 += s.rl + n * g.RL < left ? (float)(V / NS) : 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) sx[Z::at(i)] += raw_get(z[n], i);   // (zeros past the end)
        }
        if (n1 == 0.f) return;
        // (reciprocals to a step: sx need only be near the chunk's mean, and is the reference where that is as near: equal values then leave nothing
        // in the mean's second float)
        const float inv = __builtin_amdgcn_rcpf(n1), sum = cnt + n1, part = n1 * __builtin_amdgcn_rcpf(sum), cross = cnt * part;
#pragma unroll
        for (int i = 0; i < NS; ++i) sx[i] = Z::LOW && fabsf(fmaf(sx[i], inv, -k[i])) <= fabsf(k[i]) * 0x1p-18f ? k[i] : sx[i] * inv;
#pragma unroll
        for (int n = 0; n < NR; ++n)
            if (s.rl + n * g.RL < left) {
                const typename Z::Row x = again(z[n]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = raw_get(x, i) - sx[Z::at(i)];
                    e[Z::at(i)] += d;
                    q[Z::at(i)] = fmaf(d, d, q[Z::at(i)]);
                }
            }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const float shift = e[i] * inv, m = sx[i] + shift, l = Z::LOW ? (sx[i] - m) + shift : 0.f, d = Z::LOW ? (m - mu[i]) + (l - low[i]) : m - mu[i];
            m2[i] += fmaf(d * cross, d, about_mean(q[i], e[i], shift));
            const float t = Z::LOW ? fmaf(d, part, low[i]) : d * part, next = mu[i] + t;
            low[i] = Z::LOW ? cnt > 0.f ? (mu[i] - next) + t : l : 0.f;
            mu[i] = cnt > 0.f ? next : m;   // (the first chunk's as it is)
        }
        cnt = sum;
    }

    // A value next to the mean that all threads of a group know: its first channel in the first row.  Sums over threads are of differences to it, so
    // that equal means add up to exactly that mean.
    __device__ __forceinline__ void reference(int row, float (&k)[NS]) {
        const T* at = X + row_at(a, row) + s.s0;
#pragma unroll
        for (int i = 0; i < NS; ++i) k[i] = widen(at[s.j[i] * a.Cg]);
    }

    // the thread's part -> v[0] + v[2] = mean, v[1] = centred sum of squares of its groups over `rows` rows
    __device__ __forceinline__ void join(int rows, const float (&k)[NS], float cnt, const float (&mu)[NS], const float (&low)[NS], const float (&m2)[NS], float (&v)[3][NS]) {
        const float inv = 1.f / ((float)rows * (float)a.Cg);
        float sum[1][NS], eq[2][NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) sum[0][i] = cnt * (Z::LOW ? (mu[i] - k[i]) + low[i] : mu[i] - k[i]);
        group_sums<1, Z>(sum, a, g, s, lds);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            v[0][i] = fmaf(sum[0][i], inv, k[i]);
            const float d = Z::LOW ? (mu[i] - v[0][i]) + low[i] : mu[i] - v[0][i];
            eq[0][i] = d * cnt;
            eq[1][i] = cnt > 0.f ? fmaf(eq[0][i], d, m2[i]) : 0.f;
        }
        group_sums<2, Z>(eq, a, g, s, lds);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const float shift = eq[0][i] * inv, m = v[0][i] + shift;
            v[1][i] = about_mean(eq[1][i], eq[0][i], shift);
            v[2][i] = Z::LOW ? (v[0][i] - m) + shift : 0.f;
            v[0][i] = m;
        }
    }

    // statistics of rows that take several chunks
    __device__ __forceinline__ void stats(const Range& r, float (&v)[3][NS]) {
        float cnt = 0.f, k[NS], mu[NS], low[NS], m2[NS];
        reference(r.r0, k);
#pragma unroll
        for (int i = 0; i < NS; ++i) mu[i] = low[i] = m2[i] = 0.f;
        for (int base = r.r0; base < r.r1; base += NR * g.RL) {
            typename Z::Row z[NR];
            Chunk<Z>(X + row_at(a, base), a.C, r.r1 - base, g).load_all(g, s, z);
            add_rows(r.r1 - base, z, k, cnt, mu, low, m2);
        }
        join(r.r1 - r.r0, k, cnt, mu, low, m2, v);
    }

    // 1 / standard deviation from v of a whole cloud of `rows` rows; `keep`: this workgroup writes the statistics
    __device__ __forceinline__ void finish(const float (&v)[3][NS], int b, int rows, bool keep, float* mean_out, float* rstd_out, float (&rstd)[NS]) {
        const float inv = 1.f / ((float)rows * (float)a.Cg);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            rstd[i] = rsqrt_newton(fmaf(v[1][i], inv, a.eps));
            if (mean_out && keep && writes_group(a, s, i)) {
                const int64_t at = (int64_t)b * a.G + s.slab * g.k + s.j[i];
                mean_out[at] = v[0][i], rstd_out[at] = rstd[i];
                if (Z::LOW && a.low) mean_out[at + means(a)] = v[2][i];
            }
        }
    }

    // y of rows that take several chunks
    __device__ __forceinline__ void apply(const Range& r, const float (&v)[3][NS], const float (&rstd)[NS]) {
        for (int base = r.r0; base < r.r1; base += NR * g.RL) {
            typename Z::Row z[NR];
            Chunk<Z>(X + row_at(a, base), a.C, r.r1 - base, g).load_all(g, s, z);
            rows_out(base, r.r1 - base, v, rstd, z);
        }
    }

    // a cloud that one chunk holds: its rows are read once
    __device__ __forceinline__ void short_cloud(const Range& r, int b, float* mean_out, float* rstd_out) {
        const int rows = r.r1 - r.r0;
        typename Z::Row z[NR];
        Chunk<Z>(X + row_at(a, r.r0), a.C, rows, g).load_all(g, s, z);
        float cnt = 0.f, k[NS], mu[NS], low[NS], m2[NS], v[3][NS], rstd[NS];
        reference(r.r0, k);
#pragma unroll
        for (int i = 0; i < NS; ++i) mu[i] = low[i] = m2[i] = 0.f;
        add_rows(rows, z, k, cnt, mu, low, m2);
        join(rows, k, cnt, mu, low, m2, v);
        finish(v, b, rows, true, mean_out, rstd_out, rstd);
        rows_out(r.r0, rows, v, rstd, z);
    }

    __device__ __forceinline__ void rows_out(int base, int all, const float (&v)[3][NS], const float (&rstd)[NS], const typename Z::Row (&z)[NR]) {
        const Chunk<Z> to(Y + row_at(a, base), a.C, all, g);
        const uint64_t words = words_at(g, base);
        const uint32_t off = here(s.off), word = here(s.word);
        float scale[V], low[NS];   // (of half-width rows one factor a channel: an operation less)
#pragma unroll
        for (int i = 0; i < V; ++i) scale[i] = rstd[Z::at(i)] * s.w[i];
#pragma unroll
        for (int i = 0; i < NS; ++i) low[i] = -v[2][i] * rstd[i];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            row_border();
            if (n * g.RL >= all) break;
            float y[V], d1, d2;
            const typename Z::Row x = again(z[n]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = raw_get(x, i) - v[0][Z::at(i)];
                const float u = Z::LOW ? fmaf(normal<Z>(d, rstd[Z::at(i)], low[Z::at(i)]), s.w[i], s.b[i]) : fmaf(d, scale[i], s.b[i]);
                y[i] = activate<Z::FAM, 0, sizeof(T) == 2>(u, a.slope, &d1, &d2);
            }
            if (a.drop.key) {
                Words<V>(key, words + (word + n * (uint32_t)(g.RL * g.quads))).drop(a.drop, y);
            }
            to.store(g, s, off, n, y);
        }
    }
};

// part [2 * NW][G][3]: mean, centred sum of squares and low part of the mean of a window's piece of a large cloud.  MODE 0: the clouds, and the windows' partial
// sums; MODE 1: the windows' rows
template <typename Z, int MODE>
__global__ __launch_bounds__(Z::THREADS, Z::FWD_WAVES) void k_fwd(Norm a, Geo g, const typename Z::T* X, typename Z::T* Y, float* mean_out, float* rstd_out,
                                                                                  float* part, int* found) {
    extern __shared__ __align__(16) float lds[];
    if (MODE == 0) zero_rest(a, Y);
    int unit, slab;
    if (!place(g, unit, slab)) return;
    const bool whole = MODE == 0 && unit < g.U;   // this unit's clouds, or a window's pieces
    Piece p[2];
    const int np = whole ? 0 : window_pieces<MODE == 0>(a, g, unit - (MODE == 0 ? g.U : 0), found, p);
    if (!whole && np == 0) return;
    Spot<Z> s;
    locate(a, g, unit, slab, s);
    Fwd<Z> f{a, g, s, X, Y, lds, drop_key(a.drop)};
    float v[3][Z::NS], rstd[Z::NS];
    for (int i = 0, b = s.unit;; ++i, b += g.U) {
        if (MODE == 0) {
            Range r;
            if (whole) {
                if (b >= a.B) break;
                r = cloud_rows(a, b);
                if (r.r1 - r.r0 > g.Tl) continue;
                if (r.r1 == r.r0) {   // no statistics: zeros
                    if (mean_out)
                        for (int j = threadIdx.x; j < s.gs; j += Z::THREADS) {
                            const int64_t at = (int64_t)b * a.G + s.slab * g.k + j;
                            mean_out[at] = rstd_out[at] = 0.f;
                            if (Z::LOW && a.low) mean_out[at + means(a)] = 0.f;
                        }
                    continue;
                }
            } else {
                if (i >= np) break;
                r = i ? p[1].part : p[0].part;
            }
            if (whole && r.r1 - r.r0 <= Z::NR * g.RL) {
                f.short_cloud(r, b, mean_out, rstd_out);
                continue;
            }
            f.stats(r, v);
            if (whole) {
                f.finish(v, b, r.r1 - r.r0, true, mean_out, rstd_out, rstd);
                f.apply(r, v, rstd);
            } else {
                put_part<3, Z>(part, i ? p[1].slot : p[0].slot, v, a, g, s);
            }
            continue;
        }
        if (i >= np) break;
        const Piece q = i ? p[1] : p[0];
        // the whole cloud's mean, then its centred sum of squares: a wave a group, lanes over pieces
        const int n = piece_count(g, q.all), rows = q.all.r1 - q.all.r0;
        float* out = lds + g.red + g.kb * g.CL * Z::NS;
        __syncthreads();
        for (int j = s.wave; j < s.gs; j += Z::WAVES) {
            const float* from = part + (s.slab * g.k + j) * 3;
            const auto piece = [&](int o) { return from + (int64_t)piece_slot(g, q.all, o) * a.G * 3; };
            const float inv = 1.f / (float)rows, k = piece(0)[0];
            float m = 0.f, e = 0.f, m2 = 0.f;
            for (int o = s.lane; o < n; o += 64) m = fmaf(piece(o)[0] - k, (float)piece_rows(g, q.all, o) * inv, m);
            m = k + wave_sum(m);
            for (int o = s.lane; o < n; o += 64) e = fmaf((piece(o)[0] - m) + piece(o)[2], (float)piece_rows(g, q.all, o) * inv, e);
            e = wave_sum(e);
            const float mean = m + e, low = Z::LOW ? (m - mean) + e : 0.f;
            for (int o = s.lane; o < n; o += 64) {
                const float* z = piece(o);
                const float d = (z[0] - mean) + (z[2] - low);
                m2 += fmaf(d * d, (float)piece_rows(g, q.all, o) * (float)a.Cg, z[1]);
            }
            m2 = wave_sum(m2);
            if (s.lane == 0) out[j] = mean, out[g.k + j] = m2, out[2 * g.k + j] = low;
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < Z::NS; ++h)
#pragma unroll
            for (int c = 0; c < 3; ++c) v[c][h] = out[c * g.k + s.j[h]];
        f.finish(v, q.b, rows, q.all.r0 == q.part.r0, mean_out, rstd_out, rstd);
        f.apply(q.part, v, rstd);
    }
}

// 1 / standard deviation for one row; zero for a row that is not there: what stands in for its values is read as zeros, which may lie as far from the
// mean as fp32 goes in units of the spread, and only times a finite number do its dy = 0 and P = 0 add nothing.
template <int NS>
__device__ __forceinline__ void row_rstd(const float (&rstd)[NS], bool there, float (&rs)[NS]) {
#pragma unroll
    for (int i = 0; i < NS; ++i) rs[i] = there ? rstd[i] : 0.f;
}

// the statistics of cloud b
template <typename Z>
__device__ __forceinline__ void read_stats(const Norm& a, const Geo& g, const Spot<Z>& s, int b, const float* mean_in, const float* rstd_in, float (&mean)[Z::NS],
                                           float (&rstd)[Z::NS], float (&low)[Z::NS]) {
    const int64_t at = (int64_t)b * a.G + s.slab * g.k;
#pragma unroll
    for (int i = 0; i < Z::NS; ++i) {
        mean[i] = mean_in[at + s.j[i]], rstd[i] = rstd_in[at + s.j[i]];
        low[i] = Z::LOW && a.low ? -mean_in[at + s.j[i] + means(a)] * rstd[i] : 0.f;
    }
}
// ---- first gradient -------------------------------------------------------------------------------------------------------------
// Bound by HBM and, at two to three waves per SIMD, by the latency of its loads; with dropout (400 000 x 128 fp32, GELU: 184 us, 3.3 TB/s) by having
// two waves only, whose vector instructions take 55% of the cycles; half-width rows by vector instructions (80 to 90%).  What a thread keeps of a
// row between the sums and the result: the normalised values and g (fp32 rows: in the registers the loaded rows had), or the rows as loaded and the
// bits dropout kept (half-width rows: half the registers, the derivative is computed again).
template <typename Z>
struct Bwd {
    typedef typename Z::T T;
    static constexpr int V = Z::V, NR = Z::NR, NS = Z::NS;
    static constexpr bool HOLD = sizeof(T) == 4;
    const Norm& a;
    const Geo& g;
    Spot<Z>& s;
    const T *dY, *X;
    T* dX;
    float* lds;
    PhiloxKey key;
    float mean[NS], rstd[NS], low[NS], par[2][V];   // low: what is left of the mean, times -rstd; parameter gradients of this thread's channels: dw, db

    struct Held {
        typename Z::Row x[NR], d[NR];
        float xh[HOLD ? NR : 1][V], gr[HOLD ? NR : 1][V];
        uint32_t keep[HOLD ? 1 : (NR * V + 31) / 32];
    };

    __device__ __forceinline__ void load_stats(int b, const float* mean_in, const float* rstd_in) {
        read_stats<Z>(a, g, s, b, mean_in, rstd_in, mean, rstd, low);
    }

    __device__ __forceinline__ void load(int base, int all, Held& h) {
        const Chunk<Z> cx(X + row_at(a, base), a.C, all, g), cd(dY + row_at(a, base), a.C, all, g);
        const uint32_t off = here(s.off);
#pragma unroll
        for (int n = 0; n < NR; ++n)   // row by row: the first can be worked on while the others are on their way
            if (n * g.RL < all) h.x[n] = cx.load(g, s, off, n), h.d[n] = cd.load(g, s, off, n);
    }

    // xh and g of one row
    __device__ __forceinline__ void element(const typename Z::Row& x, const float (&rs)[NS], float (&xh)[V], float (&gr)[V]) {   // gr: dy after dropout -> g
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float d1, d2;
            xh[i] = normal<Z>(raw_get(x, i) - mean[Z::at(i)], rs[Z::at(i)], low[Z::at(i)]);
            activate<Z::FAM, 1>(fmaf(xh[i], s.w[i], s.b[i]), a.slope, &d1, &d2);
            gr[i] *= d1;
        }
    }

    // the chunk's part of v = sums of h and h xh per group, and of the parameter gradients
    __device__ __forceinline__ void add_rows(int base, int all, Held& h, float (&v)[2][NS]) {
        const uint64_t words = words_at(g, base);
        const uint32_t word = here(s.word);
#pragma unroll
        for (int i = 0; i < (HOLD ? 1 : (NR * V + 31) / 32); ++i) h.keep[i] = 0;
#pragma unroll
        for (int n = 0; n < NR; ++n) {   // (a row past the end has dy = 0 and xh = 0, and adds nothing)
            row_border();
            if (n * g.RL >= all) break;
            float xh[V], gr[V], rs[NS];
            row_rstd(rstd, s.rl < all - n * g.RL, rs);
#pragma unroll
            for (int i = 0; i < V; ++i) gr[i] = raw_get(h.d[n], i);
            if (a.drop.key) {
                const Words<V> rnd(key, words + (word + n * (uint32_t)(g.RL * g.quads)));
                rnd.drop(a.drop, gr);
                if (!HOLD) h.keep[n * V / 32] |= rnd.bits(a.drop) << (n * V % 32);
            }
            element(h.x[n], rs, xh, gr);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float t = gr[i] * s.w[i];
                v[0][Z::at(i)] += t;
                v[1][Z::at(i)] = fmaf(t, xh[i], v[1][Z::at(i)]);
                par[0][i] = fmaf(gr[i], xh[i], par[0][i]);
                par[1][i] += gr[i];
                if (HOLD) h.xh[n][i] = xh[i], h.gr[n][i] = gr[i];
            }
        }
    }

    __device__ __forceinline__ void rows_out(int base, int all, const Held& h, bool fresh, const float (&m1)[NS], const float (&m2)[NS]) {
        const Chunk<Z> to(dX + row_at(a, base), a.C, all, g);
        const uint64_t words = words_at(g, base);
        const uint32_t off = here(s.off), word = here(s.word);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            row_border();
            if (n * g.RL >= all) break;
            float xh[V], gr[V], dx[V];
            if (HOLD && !fresh) {
#pragma unroll
                for (int i = 0; i < V; ++i) xh[i] = h.xh[n][i], gr[i] = h.gr[n][i];
            } else {
                const typename Z::Row x = again(h.x[n]), d = again(h.d[n]);
#pragma unroll
                for (int i = 0; i < V; ++i) gr[i] = raw_get(d, i);
                if (!fresh) drop_row<V>(a.drop, h.keep[HOLD ? 0 : n * V / 32] >> (n * V % 32), gr);
                else if (a.drop.key) Words<V>(key, words + (word + n * (uint32_t)(g.RL * g.quads))).drop(a.drop, gr);
                element(x, rstd, xh, gr);   // (a row past the end is not stored)
            }
#pragma unroll
            for (int i = 0; i < V; ++i) dx[i] = rstd[Z::at(i)] * fmaf(gr[i], s.w[i], -fmaf(xh[i], m2[Z::at(i)], m1[Z::at(i)]));
            to.store(g, s, off, n, dx);
        }
    }

    __device__ __forceinline__ void means(float (&v)[2][NS], int rows) {
        const float inv = 1.f / ((float)rows * (float)a.Cg);
#pragma unroll
        for (int i = 0; i < NS; ++i) v[0][i] *= inv, v[1][i] *= inv;
    }

    __device__ __forceinline__ void short_cloud(const Range& r) {
        const int rows = r.r1 - r.r0;
        Held h;
        float v[2][NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) v[0][i] = v[1][i] = 0.f;
        load(r.r0, rows, h);
        add_rows(r.r0, rows, h, v);
        if (!dX) return;
        group_sums<2, Z>(v, a, g, s, lds);
        means(v, rows);
        rows_out(r.r0, rows, h, false, v[0], v[1]);
    }

    __device__ __forceinline__ void sums(const Range& r, float (&v)[2][NS]) {
#pragma unroll
        for (int i = 0; i < NS; ++i) v[0][i] = v[1][i] = 0.f;
        for (int base = r.r0; base < r.r1; base += NR * g.RL) {
            Held h;
            load(base, r.r1 - base, h);
            add_rows(base, r.r1 - base, h, v);
        }
        group_sums<2, Z>(v, a, g, s, lds);
    }

    __device__ __forceinline__ void apply(const Range& r, const float (&m1)[NS], const float (&m2)[NS]) {
        for (int base = r.r0; base < r.r1; base += NR * g.RL) {
            Held h;
            load(base, r.r1 - base, h);
            rows_out(base, r.r1 - base, h, true, m1, m2);
        }
    }
};

// part [2 * NW][G][2]: sums of h and h xh over a piece; w.slots NULL: no parameter gradients asked for
template <typename Z, int MODE>
__global__ __launch_bounds__(Z::THREADS, Z::BWD_WAVES) void k_bwd(Norm a, Geo g, const typename Z::T* dY, const typename Z::T* X, const float* mean_in,
                                                                 const float* rstd_in, typename Z::T* dX, Work w, Fold fold) {
    extern __shared__ __align__(16) float lds[];
    if (MODE == 0) {
        zero_rest(a, dX);
    } else if (blockIdx.x < fold.blocks) {   // the windows' launch brings the parameter gradients along
        fold_slots<Z::THREADS>(a, g, w, fold, lds);
        return;
    }
    int unit, slab;
    if (!place(g, unit, slab, MODE == 0 ? 0 : fold.blocks)) return;
    const bool whole = MODE == 0 && unit < g.U;
    Piece p[2];
    const int np = whole ? 0 : window_pieces<MODE == 0>(a, g, unit - (MODE == 0 ? g.U : 0), w.found, p);
    if (!whole && np == 0) return;
    Spot<Z> s;
    locate(a, g, unit, slab, s);
    Bwd<Z> f{a, g, s, dY, X, dX, lds, drop_key(a.drop)};
#pragma unroll
    for (int i = 0; i < Z::V; ++i) f.par[0][i] = f.par[1][i] = 0.f;
    float v[2][Z::NS];
    for (int i = 0, b = unit;; ++i, b += g.U) {
        if (MODE == 0) {
            Range r;
            if (whole) {
                if (b >= a.B) break;
                r = cloud_rows(a, b);
                if (r.r1 - r.r0 > g.Tl || r.r1 == r.r0) continue;
            } else {
                if (i >= np) break;
                r = i ? p[1].part : p[0].part;
            }
            f.load_stats(whole ? b : i ? p[1].b : p[0].b, mean_in, rstd_in);
            if (whole && r.r1 - r.r0 <= Z::NR * g.RL) {
                f.short_cloud(r);
                continue;
            }
            f.sums(r, v);
            if (!whole) {
                put_part<2, Z>(w.part, i ? p[1].slot : p[0].slot, v, a, g, s);
            } else if (dX) {
                f.means(v, r.r1 - r.r0);
                f.apply(r, v[0], v[1]);
            }
            continue;
        }
        if (i >= np) break;
        const Piece q = i ? p[1] : p[0];
        f.load_stats(q.b, mean_in, rstd_in);
        join_parts<2, Z>(w.part, q.all, v, a, g, s, lds);
        f.means(v, q.all.r1 - q.all.r0);
        f.apply(q.part, v[0], v[1]);
    }
    if (MODE == 0 && w.slots) column_sums<2, Z>(f.par, a, g, s, lds, w.slots + (int64_t)unit * 2 * a.C);
}

// ---- second gradient ------------------------------------------------------------------------------------------------------------
// Three matrices in, two out, and 14 sums an element: fp32 rows by HBM where they are read twice (vector instructions take 75% of the cycles, with
// dropout 92%), half-width rows by vector instructions (all of them).  The three matrices stay as loaded; the activation's derivatives are computed
// again in every pass over them.
template <typename Z>
struct Bwd2 {
    typedef typename Z::T T;
    static constexpr int V = Z::V, NR = Z::NR, NS = Z::NS, KW = (NR * V + 31) / 32;
    const Norm& a;
    const Geo& g;
    Spot<Z>& s;
    const T *P, *dY, *X;
    T *ddY, *ddX;
    float* lds;
    PhiloxKey key;
    typename Z::Row* mine;                 // this thread's rows in LDS: [NR][x, dy, P], a workgroup's width apart; NULL: none
    float q[V], t[V];                      // cotangents of dw and db
    float mean[NS], rstd[NS], low[NS], par[2][V];   // low: what is left of the mean, times -rstd; d(w), d(b)

    struct Held {
        typename Z::Row x[NR], d[NR], p[NR];
        uint32_t keep[KW];
    };
    // Means over the cloud of h, h xh, P, P xh, P h, q g, q g xh; and, with e = w dy D phi'' and c = q xh + s, of w e {1, xh, xh xh, P, P xh}, e c,
    // e c xh.  ub = dy D phi'' gb is linear in the means of P and P xh that gb holds, so those seven give the means of w ub and w ub xh
    // without a second pass over the rows.
    enum { H, HX, MP, PX, PH, QG, QX, E0, E1, E2, EP, EPX, EC, ECX };
    static constexpr int KS = Z::FAM == DD3D_FAM_LINEAR ? 7 : 14;
    // A cloud's rows are needed twice, and what lies between has more of them in flight than the L2 holds (400 clouds of 750 rows of 128 fp32
    // channels: 972 MiB read instead of 439).  So LDS keeps the first chunk of a cloud and the registers its last: 242 us without, 227 with
    // the LDS alone, 222 and 701 MiB with both.  The other variants' registers are full already (vectors of eight, and sixteen waves
    // a workgroup, spill some with SiLU and GELU; one statistic a channel takes up to 241 at two waves a SIMD) and walk all rows twice.
    static constexpr bool HOLD = V == 4 && NS == 1 && Z::THREADS == 256;

    __device__ __forceinline__ void load_stats(int b, const float* mean_in, const float* rstd_in) {
        read_stats<Z>(a, g, s, b, mean_in, rstd_in, mean, rstd, low);
    }

    __device__ __forceinline__ void load(int base, int all, Held& h, bool from_lds) {
        if (!from_lds) load_rows(base, all, h);
#pragma unroll
        for (int i = 0; i < KW; ++i) h.keep[i] = 0;
        if (!a.drop.key) return;
        const uint64_t words = words_at(g, base);
        const uint32_t word = here(s.word);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            row_border();
            if (n * g.RL < all) h.keep[n * V / 32] |= Words<V>(key, words + (word + n * (uint32_t)(g.RL * g.quads))).bits(a.drop) << (n * V % 32);
        }
    }
    __device__ __forceinline__ void load_rows(int base, int all, Held& h) {
        const Chunk<Z> cx(X + row_at(a, base), a.C, all, g), cd(dY + row_at(a, base), a.C, all, g);
        const Chunk<Z> cp(P ? P + row_at(a, base) : X, a.C, P ? all : 0, g);   // (without P: an empty buffer, whose rows read as zeros)
        const uint32_t off = here(s.off);
#pragma unroll
        for (int n = 0; n < NR; ++n)   // row by row: the first can be worked on while the others are on their way
            if (n * g.RL < all) h.x[n] = cx.load(g, s, off, n), h.d[n] = cd.load(g, s, off, n), h.p[n] = cp.load(g, s, off, n);
    }

    // one row: values after dropout, and the activation's derivatives element by element
    struct RowOf {
        float x[V], p[V], dy[V], rs[NS];
    };
    __device__ __forceinline__ RowOf row_of(const typename Z::Row& x, const typename Z::Row& d, const typename Z::Row& p, uint32_t keep, bool there) {
        RowOf r;
        row_rstd(rstd, there, r.rs);
#pragma unroll
        for (int i = 0; i < V; ++i) r.x[i] = raw_get(x, i), r.dy[i] = raw_get(d, i), r.p[i] = raw_get(p, i);
        drop_row<V>(a.drop, keep, r.dy);
        return r;
    }
    struct Elem {
        float xh, p, dy, d1, d2;
    };
    __device__ __forceinline__ Elem element(const RowOf& r, int i) {
        Elem e;
        e.xh = normal<Z>(r.x[i] - mean[Z::at(i)], r.rs[Z::at(i)], low[Z::at(i)]);
        e.p = r.p[i], e.dy = r.dy[i];
        activate<Z::FAM, 2>(fmaf(e.xh, s.w[i], s.b[i]), a.slope, &e.d1, &e.d2);
        return e;
    }

    __device__ __forceinline__ void add_rows(int all, const Held& h, float (&v)[KS][NS], bool to_lds) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {   // (a row past the end has dy = P = xh = 0 and adds nothing)
            row_border();
            if (n * g.RL >= all) break;
            if (HOLD && to_lds) mine[3 * n * Z::THREADS] = h.x[n], mine[(3 * n + 1) * Z::THREADS] = h.d[n], mine[(3 * n + 2) * Z::THREADS] = h.p[n];
            const RowOf row = row_of(h.x[n], h.d[n], h.p[n], h.keep[n * V / 32] >> (n * V % 32), s.rl < all - n * g.RL);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                row_border();
                const int c = Z::at(i);
                const Elem e = element(row, i);
                const float gr = e.dy * e.d1, hh = gr * s.w[i], qg = gr * q[i];
                v[H][c] += hh;
                v[HX][c] = fmaf(hh, e.xh, v[HX][c]);
                v[MP][c] += e.p;
                v[PX][c] = fmaf(e.p, e.xh, v[PX][c]);
                v[PH][c] = fmaf(e.p, hh, v[PH][c]);
                v[QG][c] += qg;
                v[QX][c] = fmaf(qg, e.xh, v[QX][c]);
                if constexpr (KS > 7) {
                    const float w1 = e.dy * e.d2 * s.w[i], w2 = w1 * s.w[i], wx = w2 * e.xh, wc = w1 * fmaf(q[i], e.xh, t[i]);
                    v[E0][c] += w2;
                    v[E1][c] += wx;
                    v[E2][c] = fmaf(wx, e.xh, v[E2][c]);
                    v[EP][c] = fmaf(w2, e.p, v[EP][c]);
                    v[EPX][c] = fmaf(wx, e.p, v[EPX][c]);
                    v[EC][c] += wc;
                    v[ECX][c] = fmaf(wc, e.xh, v[ECX][c]);
                }
            }
        }
    }

    // cotangent of g
    __device__ __forceinline__ float gbar(const Elem& e, const float (&m)[KS][NS], int i, float& vv) {
        const int c = Z::at(i);
        vv = rstd[c] * (e.p - fmaf(e.xh, m[PX][c], m[MP][c]));
        return fmaf(s.w[i], vv, fmaf(q[i], e.xh, t[i]));
    }

    __device__ __forceinline__ void rows_out(int base, int all, const Held& h, const float (&m)[KS][NS], const float (&u)[2][NS], bool from_lds) {
        const Chunk<Z> to_y(ddY + row_at(a, base), a.C, all, g), to_x(ddX + row_at(a, base), a.C, all, g);
        const uint32_t off = here(s.off);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            row_border();
            if (n * g.RL >= all) break;
            float oy[V], ox[V];
            typename Z::Row x = again(h.x[n]), d = again(h.d[n]), p = again(h.p[n]);
            if (HOLD && from_lds) x = mine[3 * n * Z::THREADS], d = mine[(3 * n + 1) * Z::THREADS], p = mine[(3 * n + 2) * Z::THREADS];
            const uint32_t keep = h.keep[n * V / 32] >> (n * V % 32);
            const RowOf row = row_of(x, d, p, keep, s.rl < all - n * g.RL);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                row_border();
                const int c = Z::at(i);
                const Elem e = element(row, i);
                float vv;
                const float gb = gbar(e, m, i, vv), gr = e.dy * e.d1, hh = gr * s.w[i], ub = Z::FAM == DD3D_FAM_LINEAR ? 0.f : gb * e.dy * e.d2;
                const float X = fmaf(q[i], gr, s.w[i] * ub) - rstd[c] * fmaf(hh, m[PX][c], e.p * m[HX][c]);
                oy[i] = done(gb * e.d1);
                ox[i] = done(rstd[c] * (X - fmaf(e.xh, u[1][c], u[0][c])));
                par[0][i] += fmaf(gr, vv, ub * e.xh);
                par[1][i] += ub;
            }
            drop_row<V>(a.drop, keep, oy);
            if (ddY) to_y.store(g, s, off, n, oy);
            if (ddX) to_x.store(g, s, off, n, ox);
        }
    }

    __device__ __forceinline__ void means(float (&m)[KS][NS], int rows) {
        const float inv = 1.f / ((float)rows * (float)a.Cg);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < NS; ++i) m[k][i] *= inv;
    }
    // the mean of X, and what multiplies xh in d(x)
    __device__ __forceinline__ void finish(const float (&m)[KS][NS], float (&u)[2][NS]) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            u[0][i] = m[QG][i] - rstd[i] * fmaf(m[PX][i], m[H][i], m[HX][i] * m[MP][i]);
            u[1][i] = m[QX][i] + rstd[i] * (m[PH][i] - m[MP][i] * m[H][i] - 3.f * (m[PX][i] * m[HX][i]));
            if constexpr (KS > 7) {   // means of w ub, w ub xh
                u[0][i] += fmaf(rstd[i], m[EP][i] - fmaf(m[MP][i], m[E0][i], m[PX][i] * m[E1][i]), m[EC][i]);
                u[1][i] += fmaf(rstd[i], m[EPX][i] - fmaf(m[MP][i], m[E1][i], m[PX][i] * m[E2][i]), m[ECX][i]);
            }
        }
    }

    __device__ __forceinline__ void clear(float (&m)[KS][NS]) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < NS; ++i) m[k][i] = 0.f;
    }

    // Sums from the first chunk to the last, results from the last to the first.  HOLD: LDS keeps the first chunk's rows, h the last one's.
    __device__ __forceinline__ void sums(const Range& r, float (&m)[KS][NS], bool first_to_lds, Held& h) {
        clear(m);
        for (int base = r.r0; base < r.r1; base += NR * g.RL) {
            Held fresh;
            Held& rows = HOLD ? h : fresh;
            load(base, r.r1 - base, rows, false);
            add_rows(r.r1 - base, rows, m, first_to_lds && base == r.r0);
        }
        group_sums<KS, Z>(m, a, g, s, lds);
    }
    __device__ __forceinline__ void apply_held(const Range& r, const float (&m)[KS][NS], const float (&u)[2][NS], bool first_in_lds, Held& h) {
        const int chunk = NR * g.RL, last = r.r0 + (r.r1 - r.r0 - 1) / chunk * chunk;
        for (int base = last; base >= r.r0; base -= chunk) {
            const bool in_lds = first_in_lds && base == r.r0 && base != last;
            if (base != last) load(base, r.r1 - base, h, in_lds);
            rows_out(base, r.r1 - base, h, m, u, in_lds);
        }
    }
    __device__ __forceinline__ void apply(const Range& r, const float (&m)[KS][NS], const float (&u)[2][NS]) {
        for (int base = r.r0; base < r.r1; base += NR * g.RL) {
            Held h;
            load(base, r.r1 - base, h, false);
            rows_out(base, r.r1 - base, h, m, u, false);
        }
    }
};

// part [2 * NW][G][KS]: a piece's sums.  MODE 0: the clouds, and the windows' sums; MODE 1: the windows' rows
template <typename Z, int MODE>
__global__ __launch_bounds__(Z::THREADS, Z::BWD2_WAVES) void k_bwd2(Norm a, Geo g, const typename Z::T* P, const void* ggw, const void* ggb, const typename Z::T* dY,
                                                                   const typename Z::T* X, const float* mean_in, const float* rstd_in, typename Z::T* ddY,
                                                                   typename Z::T* ddX, Work w) {
    extern __shared__ __align__(16) float lds[];
    if (MODE == 0) {
        zero_rest(a, ddY);
        zero_rest(a, ddX);
    }
    int unit, slab;
    if (!place(g, unit, slab)) return;
    const bool whole = MODE == 0 && unit < g.U;
    Piece p[2];
    const int np = whole ? 0 : window_pieces<MODE == 0>(a, g, unit - (MODE == 0 ? g.U : 0), w.found, p);
    if (!whole && np == 0) return;
    Spot<Z> s;
    locate(a, g, unit, slab, s);
    typedef Bwd2<Z> F;
    F f{a, g, s, P, dY, X, ddY, ddX, lds, drop_key(a.drop), (typename Z::Row*)(lds + g.hold) + threadIdx.x};
    const bool held = F::HOLD && MODE == 0 && whole && g.hold;
    load_params<Z::V>(ggw, a.pdt, s.c0, s.s0, s.s1, 0.f, f.q);
    load_params<Z::V>(ggb, a.pdt, s.c0, s.s0, s.s1, 0.f, f.t);
#pragma unroll
    for (int i = 0; i < Z::V; ++i) f.par[0][i] = f.par[1][i] = 0.f;
    float m[F::KS][Z::NS], u[2][Z::NS];
    for (int i = 0, b = unit;; ++i, b += g.U) {
        if (MODE == 0) {
            Range r;
            if (whole) {
                if (b >= a.B) break;
                r = cloud_rows(a, b);
                if (r.r1 - r.r0 > g.Tl || r.r1 == r.r0) continue;
            } else {
                if (i >= np) break;
                r = i ? p[1].part : p[0].part;
            }
            f.load_stats(whole ? b : i ? p[1].b : p[0].b, mean_in, rstd_in);
            typename F::Held rows;
            f.sums(r, m, held, rows);
            if (!whole) {
                put_part<F::KS, Z>(w.part, i ? p[1].slot : p[0].slot, m, a, g, s);
                continue;
            }
            f.means(m, r.r1 - r.r0);
            f.finish(m, u);
            if constexpr (F::HOLD) f.apply_held(r, m, u, held, rows);
            else f.apply(r, m, u);
            continue;
        }
        if (i >= np) break;
        const Piece q = i ? p[1] : p[0];
        f.load_stats(q.b, mean_in, rstd_in);
        join_parts<F::KS, Z>(w.part, q.all, m, a, g, s, lds);
        f.means(m, q.all.r1 - q.all.r0);
        f.finish(m, u);
        f.apply(q.part, m, u);
    }
    // a window's parameter gradients belong to its rows' last pass
    if (w.slots && (MODE == 1 || whole)) column_sums<2, Z>(f.par, a, g, s, lds, w.slots + (int64_t)(MODE == 1 ? g.U + unit : unit) * 2 * a.C);
}

struct Plan {
    Geo g;
    int V, fam, size;            // size: 0 few rows a thread, 1 many, 2 sixteen waves (slabs of more than 256 vectors)
    bool al;
    int ns;
    unsigned blocks0, blocks1;   // workgroups of the first launch and of the windows' launches
    size_t lds;
};

template <typename T>
int launch_fwd(const Norm& a, const Plan& p, const void* X, void* Y, float* mean, float* rstd, const Work& w, hipStream_t st);
template <typename T>
int launch_bwd(const Norm& a, const Plan& p, const void* dY, const void* X, const float* mean, const float* rstd, void* dX, const Work& w, Fold f, hipStream_t st);
template <typename T>
int launch_bwd2(const Norm& a, const Plan& p, const void* P, const void* ggw, const void* ggb, const void* dY, const void* X, const float* mean, const float* rstd,
                void* ddY, void* ddX, const Work& w, Fold f, hipStream_t st);
int launch_fold(const Norm& a, const Plan& p, const Work& w, Fold f, hipStream_t st);   // (group_norm.hip)

}  // namespace gn
