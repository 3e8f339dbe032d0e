// Training operators: activations in 8 bits (include/ccsm_train_ops.h: ccsm_code8).
#include "ccsm_train_ops_common.h"

namespace ccsm_ops {

// Any width, stride and alignment: one lane per element, 32 lanes per block of the row; loads, code bytes and scale bytes are contiguous over
// the lanes whatever the base is.
template <typename T, int CODE>
__global__ __launch_bounds__(256) void act8_pack_kernel(const T* x, long long ldx, long long rows, int width, uint8_t* codes, long long ldc, uint8_t* scales, long long lds) {
    const int nb = (width + 31) >> 5;
    const int c = threadIdx.x & 31;
    for (long long b = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); b < rows * nb; b += (long long)gridDim.x * 8) {
        const long long r = b / nb;
        const int q = (int)(b % nb), col = 32 * q + c;
        const float v = col < width ? (float)x[r * ldx + col] : 0.f;
        float most = fabsf(v) < INFINITY ? fabsf(v) : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
        const unsigned s = scale_byte<CODE>(most);
        const float k = v * pow2_of_byte(254 - s);
        codes[r * ldc + col] = (uint8_t)encode4<CODE>(k, 0.f, 0.f, 0.f, largest_code<CODE, TypeOf<T>::v>(s));
        if (c == 0) scales[r * lds + q] = (uint8_t)s;
    }
}
template <typename T>
__global__ __launch_bounds__(256) void act8_unpack_kernel(Saved s, long long rows, int width, T* y, long long ldy) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * width; i += (long long)gridDim.x * 256) {
        const long long r = i / width;
        const int c = (int)(i % width);
        y[r * ldy + c] = (T)saved_at<T>(s, r, c);
    }
}

}  // namespace ccsm_ops
