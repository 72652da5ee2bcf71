// Dropout whose mask is never stored: element (row, c) is dropped iff its Philox word (feature_math.h) is below round(p 2^32), else scaled by
// 1 / (1 - p).  The gradient is the same map applied to the incoming gradient, so one kernel serves every order.  A dropped element is
// zero whatever it held (NaN and infinity included).
#include "feature_math.h"

namespace {

template <typename T>
struct Vec {   // 16 bytes of a row
    static constexpr int V = 16 / sizeof(T);
    T e[V];
};

// Whole 16-byte vectors of rows whose blocks of four words follow each other without gaps (C % 4 == 0): element i of the flat array has
// word i % 4 of block i / 4.  Ten rounds of two wide products for every four elements stay hidden behind HBM: 800 001 x 128 bf16 rows take
// 78 us (5.2 TB/s; element by element 154).  Four vectors a thread are loaded before the first is worked on.
template <typename T>
__global__ __launch_bounds__(256) void k_dropout_flat(const Vec<T>* X, int64_t n, Drop d, Vec<T>* Y) {
    constexpr int V = Vec<T>::V, U = 4;
    const PhiloxKey k = philox_key(d.key);
    const int64_t stride = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += U * stride) {
        Vec<T> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = X[min(i + u * stride, n - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = i + u * stride;
            if (at >= n) break;
            Vec<T> y;
#pragma unroll
            for (int h = 0; h < V / 4; ++h) {
                const uint4 w = philox_block(k, (uint64_t)at * (V / 4) + h);
                const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) y.e[4 * h + j] = narrow<T>(r[j] >= d.thr && !d.all ? widen(x[u].e[4 * h + j]) * d.scale : 0.f);
            }
            Y[at] = y;
        }
    }
}

// any width and alignment, from row row0 on: a thread a block of four words, its elements one by one
template <typename T>
__global__ __launch_bounds__(256) void k_dropout(const T* X, int64_t rows, int64_t C, int64_t row0, Drop d, T* Y) {
    const PhiloxKey k = philox_key(d.key);
    const int64_t quads = (C + 3) / 4, stride = (int64_t)gridDim.x * 256, rstep = stride / quads, qstep = stride - rstep * quads;
    int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / quads, q = i - row * quads;
    for (row += row0; row < rows;) {
        const uint4 w4 = philox_block(k, (uint64_t)(row * quads + q));
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        const int64_t at = row * C + q * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (q * 4 + j < C) Y[at + j] = narrow<T>(w[j] >= d.thr && !d.all ? widen(X[at + j]) * d.scale : 0.f);
        row += rstep, q += qstep;
        if (q >= quads) q -= quads, ++row;
    }
}

template <typename T>
void run(const T* X, int64_t rows, int64_t C, const Drop& d, T* Y, hipStream_t st) {
    constexpr int V = Vec<T>::V;
    int64_t row0 = 0;
    if (C % 4 == 0 && (((uintptr_t)X | (uintptr_t)Y) & 15) == 0) {
        // (as many rows as fill whole vectors: half widths with C % 8 == 4 leave an odd last row)
        row0 = C % V == 0 ? rows : rows / 2 * 2;
        const int64_t n = row0 * C / V, blocks = ceil_div64(n, 256 * 4);
        if (n) k_dropout_flat<T><<<(unsigned)(n < 256 * 1024 ? ceil_div64(n, 256) : blocks < 8192 ? blocks : 8192), 256, 0, st>>>((const Vec<T>*)X, n, d, (Vec<T>*)Y);
    }
    if (row0 < rows) {
        const int64_t blocks = ceil_div64((rows - row0) * ((C + 3) / 4), 256);
        k_dropout<T><<<(unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, st>>>(X, rows, C, row0, d, Y);
    }
}

// the key of the next call: key = {seed, call}, then call += 1, on the stream, so a replayed graph draws anew every time
__global__ void k_random_key(int64_t* state, int64_t* key) {
    const int64_t seed = state[0], call = state[1];
    key[0] = seed;
    key[1] = call;
    state[1] = (int64_t)((uint64_t)call + 1u);
}

}  // namespace

// See include/dd3d.h.
DD3D_API int dd3d_dropout(const void* X, int dtype, int64_t rows, int64_t C, double p, const int64_t* key, void* Y, void* stream) {
    Drop d;
    if (rows < 0 || C < 0 || dtype < DD3D_F32 || dtype > DD3D_BF16 || !make_drop(p, key, &d) || !key) return DD3D_EARG;
    if (C > 0 && rows > (1ll << 60) / C) return DD3D_ESIZE;
    if (rows == 0 || C == 0) return 0;
    if (!X || !Y) return DD3D_EARG;
    d.key = key;  // p == 0 keeps every element through the same kernel
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DD3D_F32) run((const float*)X, rows, C, d, (float*)Y, st);
    else if (dtype == DD3D_F16) run((const half_t*)X, rows, C, d, (half_t*)Y, st);
    else run((const bf16_t*)X, rows, C, d, (bf16_t*)Y, st);
    DD3D_CHECK_LAUNCH();
    return 0;
}

DD3D_API int dd3d_random_key(int64_t* state, int64_t* key, void* stream) {
    if (!state || !key) return DD3D_EARG;
    k_random_key<<<1, 1, 0, (hipStream_t)stream>>>(state, key);
    DD3D_CHECK_LAUNCH();
    return 0;
}
