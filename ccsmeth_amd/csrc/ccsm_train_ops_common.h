// Shared by the training operators' kernels (ccsm_train_ops*.hip): element types, activations and their slopes, 8-bit codes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ccsm_ops {

typedef _Float16 f16;
typedef __bf16 b16;

template <typename T> struct TypeOf;                       // the ccsm_type of an element type
template <> struct TypeOf<float> { static constexpr int v = 0; };
template <> struct TypeOf<f16> { static constexpr int v = 1; };
template <> struct TypeOf<b16> { static constexpr int v = 2; };

// N elements that are loaded and stored as one aligned piece of up to 16 bytes
template <typename T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };
// ... as the widest pieces that the hardware has, with the alignment of one element (gfx950 takes any)
template <typename T, int N> struct Loose { T v[N]; };

// N elements of a row from p on, of which the first `left` exist (the others: zeros, not written)
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* p, int left, float (&v)[N]) {
    if (left >= N) {
        const Loose<T, N> t = *reinterpret_cast<const Loose<T, N>*>(p);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = (float)t.v[k];
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = k < left ? (float)p[k] : 0.f;
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_row(T* p, int left, const float (&v)[N]) {
    if (left >= N) {
        Loose<T, N> t;
#pragma unroll
        for (int k = 0; k < N; ++k) t.v[k] = (T)v[k];
        *reinterpret_cast<Loose<T, N>*>(p) = t;
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) if (k < left) p[k] = (T)v[k];
    }
}

// N elements as they are (the ones behind `left`: zeros)
template <typename T, int N>
__device__ __forceinline__ Loose<T, N> raw_row(const T* p, int left) {
    if (left >= N) return *reinterpret_cast<const Loose<T, N>*>(p);
    Loose<T, N> t;
#pragma unroll
    for (int k = 0; k < N; ++k) t.v[k] = k < left ? p[k] : (T)0.f;
    return t;
}

// x / d for x < 2^31 by a multiplication: m = floor(2^(31 + s) / d) + 1, s = the bits of d - 1 (Granlund and Montgomery's method for 31 bits)
struct Div {
    unsigned d, m, s;
    static Div by(unsigned d) {
        unsigned s = 0;
        while ((1u << s) < d) ++s;
        return Div{d, (unsigned)(((unsigned long long)1 << (31 + s)) / d + 1), s};
    }
    __device__ __forceinline__ unsigned of(unsigned x) const { return __umulhi(2 * x, m) >> s; }
};

enum { kActNone = 0, kActRelu, kActTanh, kActSigmoid, kActGelu, kActSilu };

// FAST (16-bit tensors, whose results keep 11 bits at most): hardware exp2 and reciprocal (1 ulp each), and for gelu the rational form of erfc
// by Abramowitz and Stegun (7.1.26; |error| <= 1.5e-7): 14 instructions where the library's erff has more than 40, which was a sixth of
// a wide layer's time in the epilogue.  fp32 tensors take the accurate library functions.
template <bool FAST>
__device__ __forceinline__ float exp_(float x) { return FAST ? __expf(x) : expf(x); }
template <bool FAST>
__device__ __forceinline__ float rcp_(float x) { return FAST ? __builtin_amdgcn_rcpf(x) : 1.f / x; }
template <bool FAST>
__device__ __forceinline__ float sigmoid_(float z) { return rcp_<FAST>(1.f + exp_<FAST>(-z)); }
template <bool FAST>
__device__ __forceinline__ float tanh_(float z) {
    if (!FAST) return tanhf(z);
    // 1 - 2 / (1 + e^2z); below 2^-6 that loses bits (2^-24 / |z|), and z - z^3 / 3 is within 2^-27 z
    const float t = 1.f - 2.f * rcp_<true>(1.f + __builtin_amdgcn_exp2f(2.88539008f * z));
    return fabsf(z) < 0.015625f ? z - z * z * z * 0.33333333f : t;
}
// the normal distribution's Phi(z), and e^(-z^2 / 2) (the library's erfc keeps its relative accuracy in the lower tail)
template <bool FAST>
__device__ __forceinline__ float phi_(float z, float* e) {
    if (!FAST) {
        *e = expf(-0.5f * z * z);
        return 0.5f * erfcf(-z * 0.70710678118654752f);
    }
    *e = __builtin_amdgcn_exp2f(-0.72134752f * z * z);
    const float t = rcp_<true>(1.f + 0.23164190f * fabsf(z));      // (the formula's 0.3275911 |z| / sqrt 2; its coefficients halved)
    const float q = *e * t * (0.127414796f + t * (-0.142248368f + t * (0.7107068705f + t * (-0.7265760135f + t * 0.5307027145f))));
    return z >= 0.f ? 1.f - q : q;
}
template <bool FAST, int N>
__device__ __forceinline__ void act_all(float (&z)[N], int act) {
    float e;
    switch (act) {
        case kActRelu:
#pragma unroll
            for (int k = 0; k < N; ++k) z[k] = z[k] < 0.f ? 0.f : z[k];            // (a NaN stays one)
            break;
        case kActTanh:
#pragma unroll
            for (int k = 0; k < N; ++k) z[k] = tanh_<FAST>(z[k]);
            break;
        case kActSigmoid:
#pragma unroll
            for (int k = 0; k < N; ++k) z[k] = sigmoid_<FAST>(z[k]);
            break;
        case kActGelu:
#pragma unroll
            for (int k = 0; k < N; ++k) z[k] *= phi_<FAST>(z[k], &e);
            break;
        case kActSilu:
#pragma unroll
            for (int k = 0; k < N; ++k) z[k] *= sigmoid_<FAST>(z[k]);
            break;
        default: break;
    }
}
template <bool FAST>
__device__ __forceinline__ float slope_(float z, int act) {
    float e, a;
    switch (act) {
        case kActRelu: return z > 0.f ? 1.f : z <= 0.f ? 0.f : z;
        case kActTanh: {                                     // 1 - tanh^2 = 4 e / (1 + e)^2 with e = e^-2|z|: no cancellation for large |z|
            e = exp_<FAST>(-2.f * fabsf(z));
            a = rcp_<FAST>(1.f + e);
            return 4.f * e * a * a;
        }
        case kActSigmoid: {
            e = exp_<FAST>(-fabsf(z));
            a = rcp_<FAST>(1.f + e);
            return e * a * a;
        }
        case kActGelu: {
            a = phi_<FAST>(z, &e);
            return a + z * e * 0.3989422804f;
        }
        case kActSilu: a = sigmoid_<FAST>(z); return a * (1.f + z * (1.f - a));
        default: return 1.f;
    }
}

template <bool FAST, int N>
__device__ __forceinline__ void slope_all(float (&z)[N], int act) {
    switch (act) {
#define CCSM_SLOPES(A)                                               \
    case A:                                                          \
        _Pragma("unroll") for (int k = 0; k < N; ++k) z[k] = slope_<FAST>(z[k], A); \
        break;
        CCSM_SLOPES(kActRelu)
        CCSM_SLOPES(kActTanh)
        CCSM_SLOPES(kActSigmoid)
        CCSM_SLOPES(kActGelu)
        CCSM_SLOPES(kActSilu)
#undef CCSM_SLOPES
        default: break;
    }
}

// ---- 8-bit codes (ccsm_code8) ---------------------------------------------------------------------------------------
enum { kCodeNone = 0, kCodeInt8 = 1, kCodeE4m3 = 2 };

__device__ __forceinline__ float pow2_of_byte(unsigned b) { return __uint_as_float(b << 23); }      // 2^(b - 127), b in [1, 254]
// the scale byte of a block whose largest finite magnitude is `most`: the least e with most <= 127 2^e (448 2^e), read off most's exponent
// and fraction (127 = 1.984375 2^6, 448 = 1.75 2^8)
template <int CODE>
__device__ __forceinline__ unsigned scale_byte(float most) {
    const unsigned u = __float_as_uint(most), frac = u & 0x7fffffu;
    const int b = (int)(u >> 23) - (CODE == kCodeInt8 ? 6 : 8) + (frac > (CODE == kCodeInt8 ? 0x7e0000u : 0x600000u) ? 1 : 0);
    return b < 1 ? 1u : (unsigned)b;
}
// the largest code of a block: one that rounds up past the packed type's range has to stay below it (the topmost scale byte only)
template <int CODE, int TYPE>
__device__ __forceinline__ float largest_code(unsigned b) {
    const unsigned top = (TYPE == 1 ? 142u : 254u) + (CODE == kCodeInt8 ? -5 : -7);
    return b >= top ? (CODE == kCodeInt8 ? 63.f : 240.f) : (CODE == kCodeInt8 ? 127.f : 448.f);
}
// four values, already divided by 2^e, as four codes
template <int CODE>
__device__ __forceinline__ unsigned encode4(float a, float b, float c, float d, float top) {
    if (CODE == kCodeE4m3) {
        auto lim = [top](float v) { return fminf(fmaxf(v, -top), top); };
        auto fin = [](float v) { return fabsf(v) < INFINITY; };
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(lim(a), lim(b), 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(lim(c), lim(d), r, true);
        unsigned u = (unsigned)r;
        if (!fin(a)) u = (u & 0xffffff00u) | 0x7fu;
        if (!fin(b)) u = (u & 0xffff00ffu) | 0x7f00u;
        if (!fin(c)) u = (u & 0xff00ffffu) | 0x7f0000u;
        if (!fin(d)) u = (u & 0x00ffffffu) | 0x7f000000u;
        return u;
    }
    auto one = [top](float v) -> unsigned {
        const float q = fminf(fmaxf(__builtin_rintf(v), -top), top);
        return fabsf(v) < INFINITY ? (unsigned)(int)q & 0xffu : 0x80u;
    };
    return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
}
// four codes as the values they stand for
template <int CODE>
__device__ __forceinline__ void decode4(unsigned u, float scale, float (&v)[4]) {
    if (CODE == kCodeE4m3) {
        v[0] = __builtin_amdgcn_cvt_f32_fp8((int)u, 0) * scale;
        v[1] = __builtin_amdgcn_cvt_f32_fp8((int)u, 1) * scale;
        v[2] = __builtin_amdgcn_cvt_f32_fp8((int)u, 2) * scale;
        v[3] = __builtin_amdgcn_cvt_f32_fp8((int)u, 3) * scale;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int q = (int)(signed char)(u >> (8 * j));
        v[j] = q == -128 ? __builtin_nanf("") : (float)q * scale;
    }
}
// a matrix that a forward pass has kept, in the call's type or as codes
struct Saved {
    const void* data; long long ld; int code; const uint8_t* scales; long long lds;
};

}  // namespace ccsm_ops
