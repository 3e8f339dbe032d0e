// Training operators: activations in 8 bits (include/ccsm_train_ops.h: ccsm_code8).
// Bound by memory: a lane takes 16 neighbouring values of a row (two or four 16-byte loads, whatever the row's alignment), the two lanes of a
// block of 32 exchange their largest magnitudes, and 16 codes leave as one aligned piece.  A power of two per block instead of any factor: the
// division and the values are exact, so packing values that came from codes gives the same codes, and a product can take them as bf16
// (or in the type that was packed) without a second rounding.
// Measured (86016 x 512 bf16, int8): packing 21.8 us (133 MB at 6.1 TB/s, part of it still in the last-level cache), values 32 us (4.2 TB/s).
#include "ccsm_train_ops_common.h"

namespace ccsm_ops {

template <typename T, int CODE>
__global__ __launch_bounds__(256) void act8_pack_kernel(const T* x, long long ldx, unsigned items, Div per_row, int width, uint8_t* codes, long long ldc, uint8_t* scales, long long lds) {
    const unsigned it = blockIdx.x * 256u + threadIdx.x;      // (a row has an even number of items: both lanes of a block are in or out)
    if (it >= items) return;
    const unsigned r = per_row.of(it), q = it - r * per_row.d;
    const int c = (int)(16 * q);
    float v[16];
    load_row<T, 16>(x + r * ldx + c, width - c, v);
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) most = fmaxf(most, fabsf(v[k]) < INFINITY ? fabsf(v[k]) : 0.f);
    most = fmaxf(most, __shfl_xor(most, 1));
    const unsigned s = scale_byte<CODE>(most);
    const float k = pow2_of_byte(254 - s), top = largest_code<CODE, TypeOf<T>::v>(s);
    uint4 o;
    o.x = encode4<CODE>(v[0] * k, v[1] * k, v[2] * k, v[3] * k, top);
    o.y = encode4<CODE>(v[4] * k, v[5] * k, v[6] * k, v[7] * k, top);
    o.z = encode4<CODE>(v[8] * k, v[9] * k, v[10] * k, v[11] * k, top);
    o.w = encode4<CODE>(v[12] * k, v[13] * k, v[14] * k, v[15] * k, top);
    *reinterpret_cast<uint4*>(codes + r * ldc + c) = o;
    if ((q & 1) == 0) scales[r * lds + (q >> 1)] = (uint8_t)s;
}
template <typename T, int CODE>
__global__ __launch_bounds__(256) void act8_unpack_kernel(const uint8_t* codes, long long ldc, const uint8_t* scales, long long lds, unsigned items, Div per_row, int width, T* y, long long ldy) {
    const unsigned it = blockIdx.x * 256u + threadIdx.x;
    if (it >= items) return;
    const unsigned r = per_row.of(it), q = it - r * per_row.d;
    const int c = (int)(16 * q);
    const uint4 u = *reinterpret_cast<const uint4*>(codes + r * ldc + c);
    const float k = pow2_of_byte(scales[r * lds + (q >> 1)]);
    float v[16];
    decode4<CODE>(u.x, k, *(float(*)[4])(v));
    decode4<CODE>(u.y, k, *(float(*)[4])(v + 4));
    decode4<CODE>(u.z, k, *(float(*)[4])(v + 8));
    decode4<CODE>(u.w, k, *(float(*)[4])(v + 12));
    store_row<T, 16>(y + r * ldy + c, width - c, v);
}

}  // namespace ccsm_ops
