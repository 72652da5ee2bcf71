// Dropout whose mask is never stored: element (row, c) is dropped iff its Philox word (feature_math.h) is below round(p 2^32), else scaled by
// 1 / (1 - p).  The gradient is the same map applied to the incoming gradient, so one kernel serves every order.  A dropped element is
// zero whatever it held (NaN and infinity included).
#include "feature_math.h"

namespace {

template <typename T>
__global__ __launch_bounds__(256) void k_dropout(const T* X, int64_t rows, int64_t C, Drop d, T* Y) {
    const PhiloxKey k = philox_key(d.key);
    const int64_t quads = (C + 3) / 4;
    const int64_t n = rows * quads;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const uint4 w4 = philox_block(k, (uint64_t)i);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        const int64_t row = i / quads;
        const int64_t c0 = (i - row * quads) * 4;
        for (int j = 0; j < 4 && c0 + j < C; ++j) {
            const int64_t at = row * C + c0 + j;
            Y[at] = narrow<T>(!d.all && w[j] >= d.thr ? widen(X[at]) * d.scale : 0.f);
        }
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
    const int64_t blocks = ceil_div64(rows * ((C + 3) / 4), 256);
    const unsigned grid = (unsigned)(blocks < 16384 ? blocks : 16384);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DD3D_F32) k_dropout<float><<<grid, 256, 0, st>>>((const float*)X, rows, C, d, (float*)Y);
    else if (dtype == DD3D_F16) k_dropout<half_t><<<grid, 256, 0, st>>>((const half_t*)X, rows, C, d, (half_t*)Y);
    else k_dropout<bf16_t><<<grid, 256, 0, st>>>((const bf16_t*)X, rows, C, d, (bf16_t*)Y);
    DD3D_CHECK_LAUNCH();
    return 0;
}

DD3D_API int dd3d_random_key(int64_t* state, int64_t* key, void* stream) {
    if (!state || !key) return DD3D_EARG;
    k_random_key<<<1, 1, 0, (hipStream_t)stream>>>(state, key);
    DD3D_CHECK_LAUNCH();
    return 0;
}
