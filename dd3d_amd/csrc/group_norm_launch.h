// Picks the compiled variant a plan names and launches it (included by each group_norm_*.hip for one row type).
#pragma once
#include "group_norm.h"

namespace gn {

template <typename Z>
struct Tag {
    typedef Z type;
};

// NRS / NRL / NR8: vectors a thread holds (NR_* in group_norm.h)
template <typename T, int NRS, int NRL, int V, bool AL, int NS, int FAM, typename F>
int with_size(const Plan& p, F f) {
    if (p.size == 2) {
        if constexpr (V == 4) return f(Tag<Cfg<T, V, AL, NS, FAM, 1024, NRS>>());
    }
    if constexpr (NS == 1 && V == 4) {
        if (p.size == 1) return f(Tag<Cfg<T, V, AL, NS, FAM, 256, NRL>>());
    }
    return f(Tag<Cfg<T, V, AL, NS, FAM, 256, NRS>>());
}
template <typename T, int NRS, int NRL, int V, bool AL, int NS, typename F>
int with_family(const Plan& p, F f) {
    return p.fam == DD3D_FAM_LINEAR ? with_size<T, NRS, NRL, V, AL, NS, DD3D_FAM_LINEAR>(p, f)
           : p.fam == DD3D_FAM_SILU ? with_size<T, NRS, NRL, V, AL, NS, DD3D_FAM_SILU>(p, f)
                                    : with_size<T, NRS, NRL, V, AL, NS, DD3D_FAM_GELU>(p, f);
}
template <typename T, int NRS, int NRL, int NR8, typename F>
int with_variant(const Plan& p, F f) {
    if constexpr (sizeof(T) == 2) {
        if (p.V == 8) return with_family<T, NR8, NR8, 8, true, 1>(p, f);
    }
    if (!p.al) return with_family<T, NRS, NRL, 4, false, 4>(p, f);
    return p.ns == 1 ? with_family<T, NRS, NRL, 4, true, 1>(p, f) : with_family<T, NRS, NRL, 4, true, 4>(p, f);
}

// LDS of a workgroup of the second gradient that keeps a chunk in it: a third of a compute unit's 160 KB, as its registers allow three
constexpr size_t HOLD_LDS = 53 * 1024;

template <typename K>
int set_lds(K kernel, size_t lds) {
    if (lds > 64 * 1024) DD3D_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    return 0;
}

template <typename T>
int launch_fwd(const Norm& a, const Plan& p, const void* X, void* Y, float* mean, float* rstd, const Work& w, hipStream_t st) {
    return with_variant<T, NR_FWD[0], NR_FWD[1], NR_FWD[2]>(p, [&](auto tag) {
        typedef typename decltype(tag)::type Z;
        int rc = set_lds(k_fwd<Z, 0>, p.lds);
        if (rc) return rc;
        Geo g = p.g;
        g.units = g.U + g.NW;
        k_fwd<Z, 0><<<p.blocks0, Z::THREADS, p.lds, st>>>(a, g, (const T*)X, (T*)Y, mean, rstd, w.part, w.found);
        if (g.NW) {
            rc = set_lds(k_fwd<Z, 1>, p.lds);
            if (rc) return rc;
            g.units = g.NW;
            k_fwd<Z, 1><<<p.blocks1, Z::THREADS, p.lds, st>>>(a, g, (const T*)X, (T*)Y, mean, rstd, w.part, w.found);
        }
        DD3D_CHECK_LAUNCH();
        return 0;
    });
}

template <typename T>
int launch_bwd(const Norm& a, const Plan& p, const void* dY, const void* X, const float* mean, const float* rstd, void* dX, const Work& w, Fold f, hipStream_t st) {
    return with_variant<T, NR_BWD[0], NR_BWD[1], NR_BWD[2]>(p, [&](auto tag) {
        typedef typename decltype(tag)::type Z;
        int rc = set_lds(k_bwd<Z, 0>, p.lds);
        if (rc) return rc;
        Geo g = p.g;
        g.units = g.U + g.NW;
        k_bwd<Z, 0><<<p.blocks0, Z::THREADS, p.lds, st>>>(a, g, (const T*)dY, (const T*)X, mean, rstd, (T*)dX, w, f);
        if (g.NW && dX) {
            rc = set_lds(k_bwd<Z, 1>, p.lds);
            if (rc) return rc;
            g.units = g.NW;
            if (!w.slots) f.blocks = 0;
            k_bwd<Z, 1><<<f.blocks + p.blocks1, Z::THREADS, p.lds, st>>>(a, g, (const T*)dY, (const T*)X, mean, rstd, (T*)dX, w, f);
        } else if (w.slots) {
            return launch_fold(a, p, w, f, st);
        }
        DD3D_CHECK_LAUNCH();
        return 0;
    });
}

template <typename T>
int launch_bwd2(const Norm& a, const Plan& p, const void* P, const void* ggw, const void* ggb, const void* dY, const void* X, const float* mean, const float* rstd,
                void* ddY, void* ddX, const Work& w, Fold f, hipStream_t st) {
    return with_variant<T, NR_BWD2[0], NR_BWD2[1], NR_BWD2[2]>(p, [&](auto tag) {
        typedef typename decltype(tag)::type Z;
        Geo g = p.g;
        const size_t chunk = 3 * Z::NR * sizeof(typename Z::Row) * Z::THREADS, with = align_up64(p.lds, 16) + chunk;
        const bool hold = Bwd2<Z>::HOLD && with <= HOLD_LDS;
        g.hold = hold ? (int)((with - chunk) / 4) : 0;
        const size_t lds = hold ? with : p.lds;
        int rc = set_lds(k_bwd2<Z, 0>, lds);
        if (rc) return rc;
        g.units = g.U + g.NW;
        k_bwd2<Z, 0><<<p.blocks0, Z::THREADS, lds, st>>>(a, g, (const T*)P, ggw, ggb, (const T*)dY, (const T*)X, mean, rstd, (T*)ddY, (T*)ddX, w);
        if (g.NW) {
            rc = set_lds(k_bwd2<Z, 1>, p.lds);
            if (rc) return rc;
            g.units = g.NW;
            k_bwd2<Z, 1><<<p.blocks1, Z::THREADS, p.lds, st>>>(a, g, (const T*)P, ggw, ggb, (const T*)dY, (const T*)X, mean, rstd, (T*)ddY, (T*)ddX, w);
        }
        DD3D_CHECK_LAUNCH();
        return w.slots ? launch_fold(a, p, w, f, st) : 0;
    });
}

}  // namespace gn
