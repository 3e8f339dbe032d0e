// Training operators: the matrix product on the matrix cores.  out(i, j) = sum over k of P(i, k) Q(j, k), P and Q of 16-bit elements in device
// memory, fp32 accumulators.
//
// Tiles.  256 x 256 outputs by eight waves (2 x 4, one workgroup a CU) or 128 x 128 by four (2 x 2, two workgroups a CU); a wave owns a grid of 16 x 16
// tiles of v_mfma_f32_16x16x32 (the shape that costs least energy per flop here).  Q is the instruction's first operand, so that a lane ends with
// four neighbouring j of one i.
//
// Measured (16384 x 4096 x 4096 bf16): x w^T 400 to 430 us from card to card (1280 to 1373 TFLOP/s; the library's product: 442), d w 403 to 460, d^T x 389 to 440; at 1.95 GHz the matrix pipe is busy 66 % of the cycles.  Without the
// requests the loop takes 8 % fewer cycles, without the fragment reads as many as with them.
//
// Operands go from memory straight to LDS (buffer_load_dwordx4 ... lds, 1 KiB per wave and request) in chunks of 64 k, so that a row of an operand
// whose k is contiguous is read as whole 128-byte lines: with chunks of 32 k each line was fetched twice (75 instead of 38 M L2 requests for a 16384 x
// 4096 x 4096 product) and the requests alone took 1770 cycles per 32 k, matrix instructions or not.  Two chunks of P and three of Q are in LDS (all
// of its 160 KB): P's next chunk is requested two steps of 32 k before it is read, Q's next but one four.
//
// Two storage forms of an operand, by which index is contiguous in memory:
//   k (TR = false)   LDS rows of 64 k = 128 bytes; a fragment is one ds_read_b128 per lane; piece c (16 bytes) of row r lies at c ^ (r & 7)
//   i or j (TR)      LDS rows of the tile's i or j, one per k; a fragment is two ds_read_b64_tr_b16 (the LDS transposes 4 x 16 blocks); the
//                    32-byte piece p of row k lies at p ^ s(k), s = k & 3 | k >> 1 & 4: the eight rows that are read together lie in eight
//                    different parts of the 256 bytes of banks
// Both permutations are made on the source side (each lane requests the piece that belongs where its 16 bytes land).
//
// Ragged sizes: pieces beyond k's end get an offset outside the buffer resource and arrive as zeros; rows and columns beyond i's or j's end
// repeat the last ones, and their results are not written.  What the kernel needs: 16-byte aligned bases and row strides (multiples of 8
// elements), the contiguous extent a multiple of 8; other operands are staged first (stage_kernel).
#pragma once
#include <type_traits>

#include "ccsm_train_ops_common.h"

namespace ccsm_ops {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

// run: the compiler's own form.  tied: the accumulator stays in its registers (left to itself the compiler gives most products another destination and
// copies 200 accumulators a step around); what reads or writes such an accumulator by another instruction waits by itself (below).
template <typename E> struct Mfma;
template <> struct Mfma<f16> {
    static __device__ __forceinline__ f32x4 run(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void tied(s16x8 a, s16x8 b, f32x4& c) { asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b)); }
};
template <> struct Mfma<b16> {
    static __device__ __forceinline__ f32x4 run(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void tied(s16x8 a, s16x8 b, f32x4& c) { asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b)); }
};

// what a product's results go through: z = acc (* factor) + bias; y = act(z) + residual.  With `part`, the accumulators go there instead (split k)
struct Epilogue {
    const void* bias; const void* residual; long long ldr; void* y; long long ldy; void* pre; long long ldp; int act;
    const float* factor = nullptr;            // fp16: z = acc * *factor (+ bias), where an operand was multiplied by its inverse
};
struct Plane { const void* base; long long ld; };
struct ProductArgs {
    Plane P, Q;
    int M, N, K;
    int tiles_i, tiles_j, splits, depth;      // k of one split (a multiple of the kernel's chunk)
    float* part; long long part_ld;           // [split][M][part_ld]
    Epilogue ep;
};

// N results (i, j .. j + N - 1), of which the first `left` exist; bias and r = the residual's values of them
template <typename T, int N>
__device__ __forceinline__ void finish(const Epilogue& e, long long i, int j, int left, float (&z)[N], const float (&bias)[N], const Loose<T, N>& r) {
    constexpr bool fast = sizeof(T) == 2;
    if constexpr (std::is_same<T, f16>::value) {
        if (e.factor) {
            const float f = *e.factor;
#pragma unroll
            for (int k = 0; k < N; ++k) z[k] *= f;
        }
    }
    if (e.bias) {
#pragma unroll
        for (int k = 0; k < N; ++k) z[k] += bias[k];
    }
    if (e.pre) store_row<T, N>((T*)e.pre + i * e.ldp + j, left, z);
    act_all<fast, N>(z, e.act);
    if (e.residual) {
#pragma unroll
        for (int k = 0; k < N; ++k) z[k] += (float)r.v[k];
    }
    store_row<T, N>((T*)e.y + i * e.ldy + j, left, z);
}
// One operand's side: requests by NW waves (this one is number `wave` of them) for B rows or columns, and the fragments of this wave's W of them; ES =
// bytes of an element (a chunk is 128 / ES deep)
template <int ES, bool TR, int B, int W, int NW>
struct Side {
    static constexpr unsigned kChunk = B * 128;            // bytes
    static constexpr int kReq = kChunk / 1024 / NW;        // requests per wave and chunk
    static constexpr int kFrag = W / 16;
    unsigned off[kReq];                                    // byte offset of this lane's piece from the chunk's origin
    int kpos[kReq];                                        // its k within the chunk
    unsigned rd[TR ? kFrag : 2];                           // LDS byte offsets of the fragments (k contiguous: of the two halves of a chunk)

    __device__ __forceinline__ void init(const Plane& p, int at, int extent, int wave, int lane, int w0, unsigned lds) {
        constexpr int kPer = 16 / ES;                      // elements of a 16-byte piece
#pragma unroll
        for (int r = 0; r < kReq; ++r) {
            const int q = r * NW + wave;                   // request number within the chunk
            if (!TR) {
                const int row = q * 8 + (lane >> 3), c = (lane & 7) ^ (row & 7);
                const int i = at + row < extent ? row : extent - 1 - at;
                off[r] = (unsigned)(((long long)i * p.ld + kPer * c) * ES);
                kpos[r] = kPer * c;
            } else {
                constexpr int kRow = B / kPer;             // pieces per row
                const int k = (q * 64 + lane) / kRow, x = (q * 64 + lane) % kRow;
                const int c = ES == 2 ? (((x >> 1) ^ ((k & 3) | ((k >> 1) & 4))) << 1) | (x & 1) : ((x >> 2) ^ ((k >> 3) & 3)) << 2 | (x & 3);
                const int i = at + kPer * c < extent ? kPer * c : ((extent - 1) & ~(kPer - 1)) - at;
                off[r] = (unsigned)(((long long)k * p.ld + i) * ES);
                kpos[r] = k;
            }
        }
        if (!TR) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                rd[h] = lds + (unsigned)((w0 + (lane & 15)) * 128 + (((ES == 2 ? 4 * h + (lane >> 4) : 2 * (lane >> 4) + h) ^ (lane & 7)) << 4));
        } else if (ES == 2) {
            const int k = 8 * (lane >> 4) + ((lane & 15) >> 2), s = (k & 3) | ((k >> 1) & 4);
#pragma unroll
            for (int f = 0; f < kFrag; ++f) rd[f] = lds + (unsigned)(k * (2 * B) + (((w0 / 16 + f) ^ s) << 5) + (lane & 3) * 8);
        } else {
            const int g = lane >> 4;
#pragma unroll
            for (int f = 0; f < kFrag; ++f) rd[f] = lds + (unsigned)(8 * g * (4 * B) + (((w0 / 16 + f) ^ g) << 6) + (lane & 15) * 4);
        }
    }
    // request r of a chunk into LDS at `m0` (the wave's base of that request)
    __device__ __forceinline__ void request(int r, u32x4 srd, int left, unsigned m0) const {
        const unsigned o = kpos[r] < left ? off[r] : 0xffffffffu;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" :: "s"(m0), "v"(o), "s"(srd) : "memory");
    }
    // fragment f of half h (32 k) of the chunk at byte `base` of this operand's ring
    __device__ __forceinline__ s16x8 fragment(int f, int h, unsigned base) const {
        typedef __attribute__((address_space(3))) const s16x8* P8;
        typedef __attribute__((address_space(3))) s16x4* P4;
        if (!TR) return *(P8)(uintptr_t)(rd[h] + base + f * 2048);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P4)(uintptr_t)(rd[f] + base + h * 64 * B));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P4)(uintptr_t)(rd[f] + base + h * 64 * B + 8 * B));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    // ES = 4: the eight values of fragment f
    __device__ __forceinline__ void values(int f, unsigned base, float (&v)[8]) const {
        typedef __attribute__((address_space(3))) const f32x4* P4;
        typedef __attribute__((address_space(3))) const float* P1;
        if (!TR) {
            const f32x4 a = *(P4)(uintptr_t)(rd[0] + base + f * 2048), b = *(P4)(uintptr_t)(rd[1] + base + f * 2048);
#pragma unroll
            for (int q = 0; q < 4; ++q) { v[q] = a[q]; v[4 + q] = b[q]; }
            return;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = *(P1)(uintptr_t)(rd[f] + base + q * 4 * B);
    }
};
// where an operand's next chunk comes from
template <int ES, bool TR>
struct Cursor {
    const char* base;
    long long step;                                        // bytes from one chunk to the next
    int left;                                              // k left in the split, and behind it: everything out of range, zeros that nobody reads
    __device__ __forceinline__ u32x4 next(int* l) {
        const unsigned long long p = (unsigned long long)base;
        *l = left;
        base += step;
        left -= 128 / ES;
        return u32x4{(unsigned)p, (unsigned)(p >> 32) & 0xffffu, 0xfffffffeu, 0x00020000u};
    }
};
template <int ES, bool TR>
__device__ __forceinline__ Cursor<ES, TR> cursor(const Plane& p, int at, int k0, int k1) {
    return Cursor<ES, TR>{(const char*)p.base + (TR ? (long long)k0 * p.ld + at : (long long)at * p.ld + k0) * ES, (TR ? p.ld * (128 / ES) : 128 / ES) * ES, k1 - k0};
}
// Workgroups go to the eight XCDs in turn; each XCD takes one contiguous eighth of the tiles (its L2 holds their operands), in columns of eight tiles
// along i, so that the 32 tiles of an XCD that run together share eight strips of P and four of Q
struct Place { int i, j, split; };
__device__ __forceinline__ Place place_of(int b, int tiles_i, int tiles_j, int splits) {
    const int n = tiles_i * tiles_j * splits, each = n >> 3, over = n & 7, x = b & 7;
    int t = x * each + (x < over ? x : over) + (b >> 3);
    const int split = t / (tiles_i * tiles_j);
    t -= split * (tiles_i * tiles_j);
    const int band = t / (8 * tiles_j), in = t - band * 8 * tiles_j, rows = tiles_i - 8 * band < 8 ? tiles_i - 8 * band : 8;
    return Place{8 * band + in % rows, in / rows, split};
}

// Sums of products of values in pieces are NaN wherever an operand is infinite (its other pieces are NaN, and infinity times an empty piece is), or where
// the largest products pass fp32's range and smaller ones of the other sign do too.  A wave that finds a NaN among its results makes
// those sums again from one piece of each value: infinities, opposite infinities, infinity times zero and NaN then give what they give in fp32.
// Finite results cost the look (one instruction for two of them).  Again costs a 16 x 16 tile its contraction step by step: 21504 x 512 -> 768 takes 100 us
// more with one infinity, and 1.8 ms with an operand full of NaN.
//
// one piece of v: sign, exponent and seven bits; a NaN stays one, what is not zero does not become it
__device__ __forceinline__ short leading(float v) {
    const unsigned u = __float_as_uint(v), m = u & 0x7fffffffu;
    return (short)((m > 0x7f800000u ? 0x7fc0u : m != 0 && m < 0x00800000u ? 0x0080u : m >> 16) | (u >> 16 & 0x8000u));
}
__device__ __forceinline__ s16x8 leading8(const float (&v)[8]) {
    s16x8 p;
#pragma unroll
    for (int k = 0; k < 8; ++k) p[k] = leading(v[k]);
    return p;
}
__device__ __forceinline__ bool any_nan(const f32x4& v) { return __builtin_isunordered(v[0], v[1]) || __builtin_isunordered(v[2], v[3]); }
__device__ __forceinline__ void replace_nan(f32x4& v, const f32x4& by) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] != v[e] ? by[e] : v[e];
}
// the sums over [first, last) of a 16 x 16 tile from (i0, j0) on, from one piece of each fp32 value; straight from memory, with a bounds check each
template <bool TRP, bool TRQ>
__device__ __forceinline__ f32x4 tile_of_leading(Plane P, Plane Q, int i0, int j0, int M, int N, int first, int last, int lane) {
    const long long i = i0 + (lane & 15) < M ? i0 + (lane & 15) : M - 1, j = j0 + (lane & 15) < N ? j0 + (lane & 15) : N - 1;
    auto eight = [&](const Plane& s, bool tr, long long r, int k) {
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = k + q < last ? ((const float*)s.base)[tr ? (k + q) * s.ld + r : r * s.ld + k + q] : 0.f;
        return leading8(v);
    };
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
    for (int k0 = first; k0 < last; k0 += 32) {
        const int k = k0 + 8 * (lane >> 4);
        acc = Mfma<b16>::run(eight(Q, TRQ, j, k), eight(P, TRP, i, k), acc);
    }
    return acc;
}
// a wave's 16 FI x 16 FJ results from (i_wave, jw) on; again(i, j): what the NaN among those of a 16 x 16 tile are replaced by (fp32)
template <typename T, int FI, int FJ, int NW, typename Again>
__device__ __forceinline__ void store_tile(const ProductArgs& a, float* smem, int wave, int lane, int i_wave, int jw, int split, f32x4 (&acc)[FI][FJ], Again again) {
    // The results leave through the wave's own part of LDS, 32 rows of i at a time (rows 16 bytes longer than they need: the lanes' writes fall on
    // different banks), and from there in pieces of eight neighbours of a row.  A lane's column does not change, so its bias is loaded once; a
    // round's residual is loaded a round ahead (one load at a time, 128 loads one behind the other, took 170 of 640 us of a 16384 x 4096 x 4096
    // product).
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // (no request may still write LDS)
    constexpr int WJT = 16 * FJ, kRow = WJT + 4, kPer = WJT / 8, kIt = 32 * kPer / 64, kRowsIt = 64 / kPer;
    static_assert(NW * 32 * kRow * 4 <= (NW == 8 ? 160 : 80) * 1024 && 64 % kPer == 0, "the waves' rows fit into the stages");
    float* out = smem + wave * 32 * kRow;
    if constexpr (sizeof(T) == 4) {
        bool nan = false;
#pragma unroll
        for (int p = 0; p < FI; ++p)
#pragma unroll
            for (int q = 0; q < FJ; ++q) nan |= any_nan(acc[p][q]);
        if (__any(nan)) {                                  // (a row of tiles at a time, through the wave's part of LDS)
            f32x4* mine = (f32x4*)out + lane;
#pragma unroll 1
            for (int h = 0; h < FI; ++h) {
#pragma unroll
                for (int p = 0; p < FI; ++p) {
                    if (p != h) continue;
#pragma unroll
                    for (int q = 0; q < FJ; ++q) mine[64 * q] = acc[p][q];
                }
#pragma unroll 1
                for (int q = 0; q < FJ; ++q) {
                    f32x4 v = mine[64 * q];
                    if (!__any(any_nan(v)) || i_wave + 16 * h >= a.M || jw + 16 * q >= a.N) continue;
                    replace_nan(v, again(i_wave + 16 * h, jw + 16 * q));
                    mine[64 * q] = v;
                }
#pragma unroll
                for (int p = 0; p < FI; ++p) {
                    if (p != h) continue;
#pragma unroll
                    for (int q = 0; q < FJ; ++q) acc[p][q] = mine[64 * q];
                }
            }
        }
    }
    const int c = lane % kPer * 8, j = jw + c, left_j = a.N - j, iw = i_wave + lane / kPer;
    const bool res = !a.part && a.ep.residual && left_j > 0;
    float bias[8];
    if (!a.part && a.ep.bias && left_j > 0) load_row<T, 8>((const T*)a.ep.bias + j, left_j, bias);
    Loose<T, 8> r[2][kIt];
    auto residual = [&](int h, Loose<T, 8> (&o)[kIt]) {
        const T* p[kIt];
#pragma unroll
        for (int q = 0; q < kIt; ++q) {                    // (rows behind the last one read that one: no condition between the loads)
            const int i = iw + 32 * h + q * kRowsIt;
            p[q] = (const T*)a.ep.residual + (long long)(i < a.M ? i : a.M - 1) * a.ep.ldr + j;
        }
        if (left_j >= 8) {
#pragma unroll
            for (int q = 0; q < kIt; ++q) o[q] = *reinterpret_cast<const Loose<T, 8>*>(p[q]);
        } else {
#pragma unroll
            for (int q = 0; q < kIt; ++q) o[q] = raw_row<T, 8>(p[q], left_j);
        }
    };
    if (res) residual(0, r[0]);
#pragma unroll 1
    for (int h = 0; h < FI / 2; ++h) {
#pragma unroll
        for (int p = 0; p < FI; ++p) {
            if (p / 2 != h) continue;
#pragma unroll
            for (int q = 0; q < FJ; ++q) *(f32x4*)(out + (16 * (p & 1) + (lane & 15)) * kRow + 16 * q + 4 * (lane >> 4)) = acc[p][q];
        }
        if (res && h + 1 < FI / 2) residual(h + 1, r[1]);
        static_assert(kIt % 2 == 0, "two pieces at a time");
#pragma unroll
        for (int q0 = 0; q0 < kIt; q0 += 2) {              // (two pieces read at a time; all four at once do not fit into the registers)
            f32x4 u[2], v[2];
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const float* o = out + (lane / kPer + (q0 + d) * kRowsIt) * kRow + c;
                u[d] = *(const f32x4*)o;
                v[d] = *(const f32x4*)(o + 4);
            }
            if (left_j <= 0) continue;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const int i = iw + 32 * h + (q0 + d) * kRowsIt;
                if (i >= a.M) continue;
                if (a.part) {
                    float* g = a.part + ((long long)split * a.M + i) * a.part_ld + j;
                    *(f32x4*)g = u[d];
                    if (left_j > 4) *(f32x4*)(g + 4) = v[d];
                } else {
                    float z[8] = {u[d][0], u[d][1], u[d][2], u[d][3], v[d][0], v[d][1], v[d][2], v[d][3]};
                    finish<T, 8>(a.ep, i, j, left_j, z, bias, r[0][q0 + d]);
                }
            }
        }
#pragma unroll
        for (int q = 0; q < kIt; ++q) r[0][q] = r[1][q];
    }
}

template <typename T, bool TRP, bool TRQ, int BI, int BJ, int WI, int WJ>
__device__ __forceinline__ void product_mfma(const ProductArgs& a, int block) {
    constexpr int NW = WI * WJ, FI = BI / WI / 16, FJ = BJ / WJ / 16, HW = BI / WI;
    typedef Side<2, TRP, BI, HW, NW> SP;
    typedef Side<2, TRQ, BJ, BJ / WJ, NW> SQ;
    constexpr int kReq = SP::kReq;
    static_assert(SP::kReq == SQ::kReq, "the waits below count as many requests of each operand");
    extern __shared__ __attribute__((aligned(1024))) char ops_smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave / WJ, wj = wave % WJ;
    const Place at = place_of(block, a.tiles_i, a.tiles_j, a.splits);
    const int i0 = at.i * BI, j0 = at.j * BJ, split = at.split;
    const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)ops_smem;
    constexpr unsigned kP = SP::kChunk, kQ = SQ::kChunk, kQ0 = 2 * kP;      // LDS: P's two chunks, then Q's three
    const unsigned lq = lds + kQ0;
    SP sp;
    SQ sq;
    sp.init(a.P, i0, a.M, wave, lane, wi * HW, lds);
    sq.init(a.Q, j0, a.N, wave, lane, wj * (BJ / WJ), lq);
    const int first = split * a.depth, last = first + a.depth < a.K ? first + a.depth : a.K;
    Cursor<2, TRP> cp = cursor<2, TRP>(a.P, i0, first, last);
    Cursor<2, TRQ> cq = cursor<2, TRQ>(a.Q, j0, first, last);
    u32x4 srd;
    int left;
    auto request_p = [&](int r, unsigned base) { sp.request(r, srd, left, lds + base + (r * NW + wave) * 1024); };
    auto request_q = [&](int r, unsigned base) { sq.request(r, srd, left, lq + base + (r * NW + wave) * 1024); };

    f32x4 acc[FI][FJ];
#pragma unroll
    for (int p = 0; p < FI; ++p)
#pragma unroll
        for (int q = 0; q < FJ; ++q) {
            acc[p][q] = f32x4{0.f, 0.f, 0.f, 0.f};
            asm volatile("" : "+v"(acc[p][q]));            // (written here, far from the first product)
        }
    // Chunk c = steps 2c and 2c + 1.  The fragments of a step are read while the step before multiplies; one barrier a chunk, in front of step 2c + 1, behind
    // which chunk c + 1 has landed (every wave has waited for all but its last four requests) and chunk c has been read.  Its place in P's ring is
    // requested for chunk c + 2 in step 2c + 1, the one of chunk c - 1 in Q's ring for chunk c + 2 in step 2c.
    s16x8 fp[2][FI], fq[2][FJ];
    auto all_p = [&](unsigned base) {
        srd = cp.next(&left);
#pragma unroll
        for (int r = 0; r < kReq; ++r) request_p(r, base);
    };
    auto all_q = [&](unsigned base) {
        srd = cq.next(&left);
#pragma unroll
        for (int r = 0; r < kReq; ++r) request_q(r, base);
    };
    all_p(0);
    all_q(0);
    all_q(kQ);
    all_p(kP);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(2 * kReq) : "memory");
#pragma unroll
    for (int q = 0; q < FJ; ++q) fq[0][q] = sq.fragment(q, 0, 0);
#pragma unroll
    for (int p = 0; p < FI; ++p) fp[0][p] = sp.fragment(p, 0, 0);
    unsigned bp = 0, bq = 0, free_q = 2 * kQ;              // the current chunk's places in the rings, Q's free one
    constexpr int kReads = FI + FJ, kRows = FI == 8 ? 6 : FI;
    for (int c = first; c < last; c += 64) {
        srd = cq.next(&left);
#pragma unroll
        for (int p = 0; p < FI; ++p) {                     // fragments of the step's other half first, then requests, between rows of products
#pragma unroll
            for (int f = p * kReads / kRows; f < (p + 1) * kReads / kRows && f < kReads; ++f) {
                if (f < FJ) fq[1][f] = sq.fragment(f, 1, bq);
                else fp[1][f - FJ] = sp.fragment(f - FJ, 1, bp);
            }
#pragma unroll
            for (int q = 0; q < FJ; ++q) Mfma<T>::tied(fq[0][q], fp[0][p], acc[p][q]);
#pragma unroll
            for (int r = p * kReq / FI; r < (p + 1) * kReq / FI; ++r) request_q(r, free_q);
            __builtin_amdgcn_sched_barrier(0);             // (left to itself the compiler begins the next step's products here and waits for their operands)
        }
        free_q = bq;
        bq = bq == 2 * kQ ? 0 : bq + kQ;
        bp ^= kP;
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(kReq) : "memory");
        srd = cp.next(&left);
#pragma unroll
        for (int p = 0; p < FI; ++p) {
#pragma unroll
            for (int f = p * kReads / kRows; f < (p + 1) * kReads / kRows && f < kReads; ++f) {
                if (f < FJ) fq[0][f] = sq.fragment(f, 0, bq);
                else fp[0][f - FJ] = sp.fragment(f - FJ, 0, bp);
            }
#pragma unroll
            for (int q = 0; q < FJ; ++q) Mfma<T>::tied(fq[1][q], fp[1][p], acc[p][q]);
#pragma unroll
            for (int r = p * kReq / FI; r < (p + 1) * kReq / FI; ++r) request_p(r, bp ^ kP);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    asm volatile("s_nop 15\n\ts_nop 15");                    // the last products' results are there (16 passes at most), for whatever reads them below
#pragma unroll
    for (int p = 0; p < FI; ++p)
#pragma unroll
        for (int q = 0; q < FJ; ++q) asm volatile("" : "+v"(acc[p][q]));
    store_tile<T, FI, FJ, NW>(a, reinterpret_cast<float*>(ops_smem), wave, lane, i0 + wi * HW, j0 + wj * (BJ / WJ), split, acc, [](int, int) { return f32x4{}; });
}

// v as three bf16 values whose sum it is: the first eight bits cut off (so that no finite value becomes infinite), the rest rounded to nearest twice;
// an infinity's are infinity and NaN twice
__device__ __forceinline__ void three(float v, b16 (&p)[3]) {
    const float h = __uint_as_float(__float_as_uint(v) & 0xffff0000u), r = v - h;
    p[0] = __builtin_bit_cast(b16, (unsigned short)(__float_as_uint(v) >> 16));
    p[1] = (b16)r;
    p[2] = (b16)(r - (float)p[1]);
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
// the same for eight values, as three fragments: 44 instructions
__device__ __forceinline__ void three8(const float (&v)[8], s16x8 (&p)[3]) {
    unsigned o[3][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const unsigned a = __float_as_uint(v[2 * k]), b = __float_as_uint(v[2 * k + 1]);
        o[0][k] = __builtin_amdgcn_perm(b, a, 0x07060302u);       // the upper halves of both
        const f32x2 r{v[2 * k] - __uint_as_float(a & 0xffff0000u), v[2 * k + 1] - __uint_as_float(b & 0xffff0000u)};
        o[1][k] = __builtin_bit_cast(unsigned, __builtin_convertvector(r, b16x2));
        const f32x2 s{r[0] - __uint_as_float(o[1][k] << 16), r[1] - __uint_as_float(o[1][k] & 0xffff0000u)};
        o[2][k] = __builtin_bit_cast(unsigned, __builtin_convertvector(s, b16x2));
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) p[q] = __builtin_bit_cast(s16x8, u32x4{o[q][0], o[q][1], o[q][2], o[q][3]});
}
// eight values as two fragments, rounded to nearest twice
__device__ __forceinline__ void two8(const float (&v)[8], s16x8 (&p)[2]) {
    unsigned o[2][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        o[0][k] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{v[2 * k], v[2 * k + 1]}), b16x2));
        const f32x2 r{v[2 * k] - __uint_as_float(o[0][k] << 16), v[2 * k + 1] - __uint_as_float(o[0][k] & 0xffff0000u)};
        o[1][k] = __builtin_bit_cast(unsigned, __builtin_convertvector(r, b16x2));
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) p[q] = __builtin_bit_cast(s16x8, u32x4{o[q][0], o[q][1], o[q][2], o[q][3]});
}
// The fp32 product: the same tiles, rings and requests with chunks of 32 k; a fragment's eight values are read as fp32 and split into three bf16
// fragments in registers (5.5 instructions a value), and each pair of fragments is multiplied six times: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0); what is
// left out is below 2^-22 of each product, 2^-25 in the mean.  Bound by the matrix pipe: 192 instructions of 16 cycles a chunk and wave, beside 2100
// cycles of splitting.  (Three bf16 planes in memory, made by a kernel in front and multiplied by the 16-bit kernel: 18 us a 44 MB operand, and three
// times the requests: 21504 x 512 x 768 110 us.)
// Q's fragments of a chunk stay in registers; P's come one row of products ahead.  The next chunk's Q is read and split in the last row, each fragment
// behind its last product; the barrier stands in front of that row, when all of this chunk has been read.
template <bool TRP, bool TRQ, int BI, int BJ, int WI, int WJ>
__device__ __forceinline__ void product_f32(const ProductArgs& a, int block) {
    constexpr int NW = WI * WJ, FI = BI / WI / 16, FJ = BJ / WJ / 16, HW = BI / WI;
    typedef Side<4, TRP, BI, HW, NW> SP;
    typedef Side<4, TRQ, BJ, BJ / WJ, NW> SQ;
    constexpr int kReq = SP::kReq;
    static_assert(SP::kReq == SQ::kReq && kReq <= FI, "the waits below count as many requests of each operand");
    extern __shared__ __attribute__((aligned(1024))) char ops_smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave / WJ, wj = wave % WJ;
    const Place at = place_of(block, a.tiles_i, a.tiles_j, a.splits);
    const int i0 = at.i * BI, j0 = at.j * BJ;
    const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)ops_smem;
    constexpr unsigned kP = SP::kChunk, kQ = SQ::kChunk;
    const unsigned lq = lds + 2 * kP;
    SP sp;
    SQ sq;
    sp.init(a.P, i0, a.M, wave, lane, wi * HW, lds);
    sq.init(a.Q, j0, a.N, wave, lane, wj * (BJ / WJ), lq);
    const int first = at.split * a.depth, last = first + a.depth < a.K ? first + a.depth : a.K;
    Cursor<4, TRP> cp = cursor<4, TRP>(a.P, i0, first, last);
    Cursor<4, TRQ> cq = cursor<4, TRQ>(a.Q, j0, first, last);
    u32x4 srd;
    int left;
    auto request_p = [&](int r, unsigned base) { sp.request(r, srd, left, lds + base + (r * NW + wave) * 1024); };
    auto request_q = [&](int r, unsigned base) { sq.request(r, srd, left, lq + base + (r * NW + wave) * 1024); };
    auto all_p = [&](unsigned base) {
        srd = cp.next(&left);
#pragma unroll
        for (int r = 0; r < kReq; ++r) request_p(r, base);
    };
    auto all_q = [&](unsigned base) {
        srd = cq.next(&left);
#pragma unroll
        for (int r = 0; r < kReq; ++r) request_q(r, base);
    };
    f32x4 acc[FI][FJ];
#pragma unroll
    for (int p = 0; p < FI; ++p)
#pragma unroll
        for (int q = 0; q < FJ; ++q) acc[p][q] = f32x4{0.f, 0.f, 0.f, 0.f};
    all_p(0);
    all_q(0);
    all_q(kQ);
    all_p(kP);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(2 * kReq) : "memory");
    s16x8 fq[FJ][3], fp[2][3];
    float raw[8], rq[2][8];
#pragma unroll
    for (int q = 0; q < FJ; ++q) {
        sq.values(q, 0, raw);
        three8(raw, fq[q]);
    }
    sp.values(0, 0, raw);
    three8(raw, fp[0]);
    sp.values(1, 0, raw);
    unsigned bp = 0, bq = 0, free_q = 2 * kQ;              // the current chunk's places in the rings, Q's free one
    auto products = [&](int p, int q0, int q1) {           // six products of row p with the fragments [q0, q1): neighbours in time are independent of each other
        constexpr int kQ6[6] = {2, 0, 1, 1, 0, 0}, kP6[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
        for (int s = 0; s < 6; ++s)
#pragma unroll
            for (int q = q0; q < q1; ++q) acc[p][q] = Mfma<b16>::run(fq[q][kQ6[s]], fp[p & 1][kP6[s]], acc[p][q]);
    };
    // the order of a row: two vector instructions of the next fragment's splitting in the shadow of each matrix instruction.  (One behind the other, the two
    // waves of a SIMD split and multiply at the same times, and the step takes the sum of both: 90 us at 21504 x 512 x 768.)
    auto interleave = [&]() {
#pragma unroll
        for (int k = 0; k < 6 * FJ; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    for (int c = first; c < last; c += 32) {
        srd = cq.next(&left);
#pragma unroll
        for (int p = 0; p < FI - 1; ++p) {
            three8(raw, fp[(p + 1) & 1]);
            products(p, 0, FJ);
            interleave();
            if (p + 2 < FI) sp.values(p + 2, bp, raw);
            if (p < kReq) request_q(p, free_q);
        }
        if (kReq == FI) request_q(kReq - 1, free_q);
        free_q = bq;
        bq = bq == 2 * kQ ? 0 : bq + kQ;
        bp ^= kP;
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(kReq) : "memory");
        srd = cp.next(&left);
        sq.values(0, bq, rq[0]);
        sq.values(1, bq, rq[1]);
        sp.values(0, bp, raw);
#pragma unroll
        for (int q = 0; q < FJ; q += 2) {
            products(FI - 1, q, q + 2);
            three8(rq[0], fq[q]);
            three8(rq[1], fq[q + 1]);
            if (q + 2 < FJ) {
                sq.values(q + 2, bq, rq[0]);
                sq.values(q + 3, bq, rq[1]);
            }
        }
        three8(raw, fp[0]);
        sp.values(1, bp, raw);
#pragma unroll
        for (int r = 0; r < kReq; ++r) request_p(r, bp ^ kP);
        __builtin_amdgcn_sched_barrier(0);
    }
    store_tile<float, FI, FJ, NW>(a, reinterpret_cast<float*>(ops_smem), wave, lane, i0 + wi * HW, j0 + wj * (BJ / WJ), at.split, acc,
                                  [&](int i, int j) { return tile_of_leading<TRP, TRQ>(a.P, a.Q, i, j, a.M, a.N, first, last, lane); });
}

template <typename T, bool TRP, bool TRQ, int B>
__device__ __forceinline__ void product_of(const ProductArgs& a, int block) {
    if constexpr (sizeof(T) == 4) product_f32<TRP, TRQ, B, B, 2, B == 256 ? 4 : 2>(a, block);
    else product_mfma<T, TRP, TRQ, B, B, 2, B == 256 ? 4 : 2>(a, block);
}
template <typename T, bool TRP, bool TRQ, int B>
__global__ __launch_bounds__(B == 256 ? 512 : 256, B == 256 ? 1 : 2) void product_kernel(ProductArgs a) { product_of<T, TRP, TRQ, B>(a, blockIdx.x); }
// both products of a backward pass: the workgroups of the first (dx = d w), then those of the second (dw = d^T x), which fill the CUs that it leaves
template <typename T, int B>
__global__ __launch_bounds__(B == 256 ? 512 : 256, B == 256 ? 1 : 2) void product_pair_kernel(ProductArgs x, ProductArgs w, int first) {
    if ((int)blockIdx.x < first) product_of<T, false, true, B>(x, blockIdx.x);
    else product_of<T, true, true, B>(w, blockIdx.x - first);
}

// the splits' parts in order, and the epilogue; a lane takes four neighbours; workgroup `block` of `job.blocks`
struct JoinJob { const float* part; int splits; long long M; int N; long long ld; Epilogue ep; unsigned blocks; };
template <typename T>
__device__ __forceinline__ void product_join(const JoinJob& job, unsigned block) {
    const Epilogue& ep = job.ep;
    const long long M = job.M, ld = job.ld;
    const int N = job.N, nj = (N + 3) / 4;
    for (long long x = (long long)block * 256 + threadIdx.x; x < M * nj; x += (long long)job.blocks * 256) {
        const long long i = x / nj;
        const int j = (int)(x % nj) * 4;
        f32x4 v = *(const f32x4*)(job.part + i * ld + j);
#pragma unroll 8
        for (int s = 1; s < job.splits; ++s) v += *(const f32x4*)(job.part + ((long long)s * M + i) * ld + j);
        float z[4] = {v[0], v[1], v[2], v[3]}, bias[4];
        Loose<T, 4> r;
        if (ep.bias) load_row<T, 4>((const T*)ep.bias + j, N - j, bias);
        if (ep.residual) r = raw_row<T, 4>((const T*)ep.residual + i * ep.ldr + j, N - j);
        finish<T, 4>(ep, i, j, N - j, z, bias, r);
    }
}

// the values of eight codes; those behind the width are whatever the caller left there, NaN's too: zeros
__device__ __forceinline__ void decode8(int code, uint2 u, uint8_t scale, int left, float (&v)[8]) {
    const float k = pow2_of_byte(scale);
    float a[4], b[4];
    if (code == kCodeInt8) { decode4<kCodeInt8>(u.x, k, a); decode4<kCodeInt8>(u.y, k, b); }
    else { decode4<kCodeE4m3>(u.x, k, a); decode4<kCodeE4m3>(u.y, k, b); }
#pragma unroll
    for (int q = 0; q < 4; ++q) { v[q] = a[q]; v[4 + q] = b[q]; }
    if (left < 8) {
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = q < left ? v[q] : 0.f;
    }
}
// eight values of row r from column c on, zeros beyond the width
template <typename T>
__device__ __forceinline__ void load8(const Saved& s, long long r, int c, int width, float (&v)[8]) {
    if (s.code == kCodeNone) {
        load_row<T, 8>((const T*)s.data + r * s.ld + c, width - c, v);
        return;
    }
    decode8(s.code, *(const uint2*)((const uint8_t*)s.data + r * s.ld + c), s.scales[r * s.lds + (c >> 5)], width - c, v);      // (a code row covers whole blocks of 32)
}
// the same of R rows, all of them requested before the first is used
template <typename T, int R>
__device__ __forceinline__ void load8s(const Saved& s, const long long (&r)[R], int c, int width, float (&v)[R][8]) {
    if (s.code == kCodeNone && width - c >= 8) {
        Loose<T, 8> t[R];
#pragma unroll
        for (int q = 0; q < R; ++q) t[q] = *reinterpret_cast<const Loose<T, 8>*>((const T*)s.data + r[q] * s.ld + c);
#pragma unroll
        for (int q = 0; q < R; ++q) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[q][k] = (float)t[q].v[k];
        }
    } else if (s.code != kCodeNone) {
        uint2 t[R];
        uint8_t k[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            t[q] = *(const uint2*)((const uint8_t*)s.data + r[q] * s.ld + c);
            k[q] = s.scales[r[q] * s.lds + (c >> 5)];
        }
#pragma unroll
        for (int q = 0; q < R; ++q) decode8(s.code, t[q], k[q], width - c, v[q]);
    } else {
#pragma unroll
        for (int q = 0; q < R; ++q) load8<T>(s, r[q], c, width, v[q]);
    }
}

// kept matrices as rows of whole 16-byte pieces in the call's type (zeros behind the width); an item is eight values
struct StageJob { Saved from; long long items; int width; void* out; long long ld; };
template <typename T>
__device__ __forceinline__ void stage_items(const StageJob& a, const StageJob& b, unsigned block, unsigned blocks) {
    for (long long x = (long long)block * 256 + threadIdx.x; x < a.items + b.items; x += (long long)blocks * 256) {
        const bool first = x < a.items;
        const StageJob& job = first ? a : b;
        const long long i = first ? x : x - a.items;
        const int n = (int)(job.ld / 8);
        const long long r = i >> 32 ? i / n : (unsigned)i / (unsigned)n;
        const int c = (int)(i - r * n) * 8;
        float v[8];
        load8<T>(job.from, r, c, job.width, v);
        store_row<T, 8>((T*)job.out + r * job.ld + c, 8, v);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void stage_kernel(StageJob a, StageJob b) { stage_items<T>(a, b, blockIdx.x, gridDim.x); }

// The largest finite magnitude of each workgroup's part of an fp16 matrix, eight values a lane and four of those in flight.  Bound
// by memory: 16384 x 4096 in 37 us, 134 MB at 3.6 TB/s (that backward pass 945 -> 983 us, one of 43008 x 512 -> 768 138 -> 154, 4096 x 512 x 512 27 -> 35)
constexpr int kMosts = 256;
__global__ __launch_bounds__(1024) void most_kernel(const f16* p, long long ld, long long items, unsigned per_row, int width, float* most) {
    __shared__ float s[16];
    float a = 0.f;
    const long long all = (long long)gridDim.x * 1024;
    for (long long x = (long long)blockIdx.x * 1024 + threadIdx.x; x < items; x += 4 * all) {
        Loose<f16, 8> v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const long long i = x + all * q < items ? x + all * q : items - 1, r = i >> 32 ? i / per_row : (unsigned)i / per_row;
            const int c = (int)(i - r * per_row) * 8;
            v[q] = raw_row<f16, 8>(p + r * ld + c, width - c);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float u = fabsf((float)v[q].v[k]);
                a = fmaxf(a, u < INFINITY ? u : 0.f);
            }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) a = fmaxf(a, __shfl_xor(a, o));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 16; ++w) a = fmaxf(a, s[w]);
    most[blockIdx.x] = a;
}
// d = dy act'(z) in the call's type (16-bit types: rounded), and the column sums of 32 rows each.  One workgroup: 32 rows x 256 columns: 32 lanes of eight
// columns, eight rows at a time, four rows of a lane in flight.
// Rounding d: 16-bit products take 16-bit operands.  This rounding (half a step per factor, independent of each other) moves a gradient by as much as
// the rounding of the gradient itself does: together sqrt 2 times that.  The bias gradient takes d before it.
// fp16 has steps of 2^-24 below 2^-14 and ends at 65504, so d is multiplied by the power of two that brings dy's largest finite magnitude A to [2^14, 2^15)
// (a slope is at most 1.13), and the results by its inverse: down to 2^-28 A d keeps its eleven bits, below that steps of 2^-38 A, which a sum of M rows
// sees beside its result's own only where A |x| sqrt M is past 2^14.  (Without, the gradients of a mean loss over a large batch lost
// their bits: dy about 2^-16 and the sigmoid's slope, 16384 rows: an error of 5.3e-3 for 2.1e-4.)
// Bound by memory, and behind it by the slopes' instructions: 16384 x 4096 bf16 (gelu) 90 us, 400 MB at 4.5 TB/s; 43008 x 768 with z in e4m3 (silu)
// and 43008 x 512 codes of x behind it 50 us, 231 MB at 4.6.
// The workgroups behind the slopes' stage the products' other operands: one launch in front of both products.
struct SlopeJob { Saved dy, z; int act; long long M; int N; void* d; long long ldd; float* part; unsigned parts, blocks; const float* most; int mosts; float* factor; };
template <typename T>
__global__ __launch_bounds__(256) void slope_kernel(SlopeJob job, StageJob sa, StageJob sb) {
    if (blockIdx.x >= job.blocks) {
        stage_items<T>(sa, sb, blockIdx.x - job.blocks, gridDim.x - job.blocks);
        return;
    }
    const Saved &dy = job.dy, &z = job.z;
    const int act = job.act, N = job.N;
    const long long M = job.M, ldd = job.ldd;
    T* d = (T*)job.d;
    float* part = job.part;
    const unsigned by = blockIdx.x / job.parts, bx = blockIdx.x - by * job.parts;
    constexpr bool fast = sizeof(T) == 2;
    __shared__ float sum[8][256];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = (int)by * 256 + lane * 8;
    const long long m0 = (long long)bx * 32 + w;
    float acc[8] = {};
    const bool scaled = std::is_same<T, f16>::value && job.mosts;
    float most = 0.f, times = 1.f;
    if (scaled) {                                          // (every wave looks at all of them)
#pragma unroll
        for (int b = 0; b < kMosts; b += 64) most = fmaxf(most, job.most[min(b + (int)(threadIdx.x & 63), job.mosts - 1)]);
#pragma unroll
        for (int o = 32; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    }
    if (c < N) {
        float v[4][8], u[4][8];
        long long r[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) r[q] = m0 + 8 * q < M ? m0 + 8 * q : M - 1;      // (no condition between the loads)
        load8s<T, 4>(dy, r, c, N, v);
        if (act != kActNone) load8s<T, 4>(z, r, c, N, u);
        if (scaled) {
            const int e = (int)(__float_as_uint(most) >> 23) - 127;      // (fp16's values are normal in fp32)
            times = most > 0.f ? pow2_of_byte(127 + 14 - e) : 1.f;
            if (blockIdx.x == 0 && threadIdx.x == 0) *job.factor = 1.f / times;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (m0 + 8 * q >= M) break;
            if (act != kActNone) {
                slope_all<fast, 8>(u[q], act);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[q][k] = c + k < N ? v[q][k] * u[q][k] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] += v[q][k];
            if (scaled) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[q][k] *= times;
            }
            if (d) store_row<T, 8>(d + (m0 + 8 * q) * ldd + c, 8, v[q]);
        }
    }
    if (!part) return;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum[w][lane * 8 + k] = acc[k];
    __syncthreads();
    const int n = (int)(by * 256 + threadIdx.x);
    if (n >= N) return;
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) a += sum[k][threadIdx.x];
    part[(long long)bx * N + n] = a;
}

// ---- small products and few rows ------------------------------------------------------------------------------------
// The same products straight from memory into the matrix instructions' operands, without staging, LDS or a kernel in front: any type, alignment and
// storage form, an activation's slope included.  A wave owns 16 j x 16 MT i; a workgroup's eight waves share the contraction (kw of
// them) and the i between them; their sums are added in order through LDS.  fp32: the three bf16 parts of each operand are made in
// registers.
// For up to 64 rows it is bound by reading w once (1 x 512 x 768 bf16: 3.6 us; the tile kernel 9.8, four steps through LDS by six of 256 CUs); for
// small products by its one launch (the tile kernel's way takes up to three).
struct DirectArgs {
    Plane P, Z, Q;                // Z, act: P's elements are multiplied by act'(Z)
    int act;
    long long M, N, K;
    int kw;                       // waves along k: 1, 2, 4 or 8
    void* sums;                   // NULL, or (M): the sum over k of P(i, k), before its rounding
    Epilogue ep;                  // y NULL: the sums alone
};
template <typename T, int MT>
struct DirectRoom { f32x4 sum[8][MT][64]; float total[8][MT][16]; };
template <typename T, bool TRP, bool TRQ, int MT>
__device__ __forceinline__ void direct_product(const DirectArgs& a, DirectRoom<T, MT>& room, unsigned by) {
    typedef typename std::conditional<sizeof(T) == 4, b16, T>::type E;
    constexpr int NP = sizeof(T) == 4 ? 3 : 1, U = 4;
    constexpr bool fast = sizeof(T) == 2;
    auto& sum = room.sum;
    auto& total = room.total;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wk = wave & (a.kw - 1), wm = wave / a.kw, mw = 8 / a.kw;
    const long long j0 = (long long)blockIdx.x * 16, i0 = ((long long)by * mw + wm) * (16 * MT);
    const long long j = j0 + (lane & 15) < a.N ? j0 + (lane & 15) : a.N - 1;
    long long i[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) i[t] = i0 + 16 * t + (lane & 15) < a.M ? i0 + 16 * t + (lane & 15) : a.M - 1;
    f32x4 acc[MT];
    float tot[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) { acc[t] = f32x4{0.f, 0.f, 0.f, 0.f}; tot[t] = 0.f; }
    auto pieces = [](const Loose<T, 8>& v, s16x8 (&p)[NP]) {
        if constexpr (NP == 1) p[0] = __builtin_bit_cast(s16x8, v);
        else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                b16 o[3];
                three(v.v[k], o);
#pragma unroll
                for (int q = 0; q < 3; ++q) p[q][k] = __builtin_bit_cast(short, o[q]);
            }
        }
    };
    // eight neighbours along k of one row (TR: column) of a matrix, zeros behind its end.  TR: one address for all lanes and k, 32 bits for a lane's own
    // part (addresses of 64 bits for each of 72 loads do not fit into the registers); strides are below 2^21
    auto eight = [&](const Plane& s, bool tr, long long r, long long k0, unsigned kl) -> Loose<T, 8> {
        const long long k = k0 + kl;
        const int left = (int)(a.K - k < 8 ? a.K - k : 8);
        if (!tr) return raw_row<T, 8>((const T*)s.base + r * s.ld + k, left);
        Loose<T, 8> o;
        const char* p = (const char*)s.base + k0 * s.ld * (long long)sizeof(T);
        const unsigned own = (kl * (unsigned)s.ld + (unsigned)r) * (unsigned)sizeof(T);
#pragma unroll
        for (int q = 0; q < 8; ++q) o.v[q] = q < left ? *(const T*)(p + q * s.ld * (long long)sizeof(T) + own) : (T)0.f;
        return o;
    };
    // d = v act'(z) and its sum
    auto sloped = [&](const Loose<T, 8>& v, const Loose<T, 8>& z, float (&d)[8], float& t) {
#pragma unroll
        for (int q = 0; q < 8; ++q) d[q] = (float)z.v[q];
        slope_all<fast, 8>(d, a.act);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            d[q] = (float)v.v[q] * d[q];
            t += d[q];
        }
    };
    // 16-bit products of unrounded d: two bf16 pieces of d, whose range is fp32's (fp16 pieces lost a d below 2^-14 and made one above 65504 infinite),
    // with x as it is (bf16) or as the two bf16 pieces whose sum an fp16 value is.  What is left out of d is below 2^-16 of it.  (The tile kernels' d is
    // rounded once to its type, an error beside the result's own of as much.)  The second piece of a bf16 d costs 1 us of 25
    auto multiply_sloped = [&](const Loose<T, 8>& xv, const float (&d)[8], f32x4& c) {
        s16x8 y[2];
        two8(d, y);
        if constexpr (std::is_same<T, f16>::value) {
            float v[8];
            s16x8 x[2];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = (float)xv.v[q];
            two8(v, x);
            c = Mfma<b16>::run(x[1], y[1], c);
            c = Mfma<b16>::run(x[0], y[1], c);
            c = Mfma<b16>::run(x[1], y[0], c);
            c = Mfma<b16>::run(x[0], y[0], c);
        } else if constexpr (sizeof(T) == 2) {
            const s16x8 x = __builtin_bit_cast(s16x8, xv);
            c = Mfma<b16>::run(x, y[1], c);
            c = Mfma<b16>::run(x, y[0], c);
        }
    };
    auto multiply = [&](const s16x8 (&x)[NP], const Loose<T, 8>& p, f32x4& c) {
        s16x8 y[NP];
        pieces(p, y);
        if constexpr (NP == 3) {
            c = Mfma<E>::run(x[2], y[0], c);
            c = Mfma<E>::run(x[0], y[2], c);
            c = Mfma<E>::run(x[1], y[1], c);
            c = Mfma<E>::run(x[1], y[0], c);
            c = Mfma<E>::run(x[0], y[1], c);
        }
        c = Mfma<E>::run(x[0], y[0], c);
    };
    const bool slope = a.act != kActNone, want = a.sums != nullptr && blockIdx.x == 0;
    const int step = 32 * a.kw;
    long long k0 = 0;
    const unsigned kl = wk * 32 + 8 * (lane >> 4);
    if (!TRP && !TRQ && !slope) {       // four steps of whole pieces in flight
        for (; k0 + step * U <= a.K; k0 += step * U) {
            const long long k = k0 + kl;
            Loose<T, 8> qv[U], pv[U][MT];
#pragma unroll
            for (int u = 0; u < U; ++u) qv[u] = *reinterpret_cast<const Loose<T, 8>*>((const T*)a.Q.base + j * a.Q.ld + k + step * u);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < MT; ++t) pv[u][t] = *reinterpret_cast<const Loose<T, 8>*>((const T*)a.P.base + i[t] * a.P.ld + k + step * u);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s16x8 x[NP];
                pieces(qv[u], x);
#pragma unroll
                for (int t = 0; t < MT; ++t) multiply(x, pv[u][t], acc[t]);
            }
        }
    }
    for (; k0 < a.K; k0 += step) {
        Loose<T, 8> qv = {};
        s16x8 x[NP];
        if (a.ep.y) qv = eight(a.Q, TRQ, j, k0, kl);
        constexpr int G = TRP && MT > 2 ? 2 : MT;          // (rows in flight: four columns of each of P and Z, element by element, spill)
#pragma unroll
        for (int t0 = 0; t0 < MT; t0 += G) {
            Loose<T, 8> pv[G], zv[G];
#pragma unroll
            for (int t = 0; t < G; ++t) pv[t] = eight(a.P, TRP, i[t0 + t], k0, kl);
            if (slope) {
#pragma unroll
                for (int t = 0; t < G; ++t) zv[t] = eight(a.Z, TRP, i[t0 + t], k0, kl);
            }
            if (t0 == 0) pieces(qv, x);
            if (slope) {
#pragma unroll
                for (int t = 0; t < G; ++t) {
                    float d[8];
                    sloped(pv[t], zv[t], d, tot[t0 + t]);
                    if constexpr (sizeof(T) == 2) multiply_sloped(qv, d, acc[t0 + t]);
                    else {
#pragma unroll
                        for (int q = 0; q < 8; ++q) pv[t].v[q] = d[q];
                        multiply(x, pv[t], acc[t0 + t]);
                    }
                }
            } else {
#pragma unroll
                for (int t = 0; t < G; ++t) {
                    if (want) {
#pragma unroll
                        for (int q = 0; q < 8; ++q) tot[t0 + t] += (float)pv[t].v[q];
                    }
                    multiply(x, pv[t], acc[t0 + t]);
                }
            }
            if (G < MT) __builtin_amdgcn_sched_barrier(0);
        }
    }
    bool nan = false;
#pragma unroll
    for (int t = 0; t < MT; ++t) nan |= any_nan(acc[t]);
    if ((sizeof(T) == 4 || slope) && a.ep.y && __any(nan)) {      // (above: from one piece of each value)
        f32x4 again[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) again[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (k0 = 0; k0 < a.K; k0 += step) {
            const Loose<T, 8> qv = eight(a.Q, TRQ, j, k0, kl);
            float v[8], u[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = (float)qv.v[q];
            const s16x8 x = leading8(v);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const Loose<T, 8> pv = eight(a.P, TRP, i[t], k0, kl);
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = (float)pv.v[q];
                if (slope) {
                    const Loose<T, 8> zv = eight(a.Z, TRP, i[t], k0, kl);
#pragma unroll
                    for (int q = 0; q < 8; ++q) u[q] = (float)zv.v[q];
                    slope_all<fast, 8>(u, a.act);
#pragma unroll
                    for (int q = 0; q < 8; ++q) v[q] *= u[q];
                }
                again[t] = Mfma<b16>::run(x, leading8(v), again[t]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) replace_nan(acc[t], again[t]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) sum[wave][t][lane] = acc[t];
    if (want) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            tot[t] += __shfl_xor(tot[t], 16);
            tot[t] += __shfl_xor(tot[t], 32);
            if (lane < 16) total[wave][t][lane] = tot[t];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < mw * MT * 64; e += 512) {
        const int l = e & 63, t = (e >> 6) % MT, w = (e >> 6) / MT;
        const long long m = ((long long)by * mw + w) * (16 * MT) + 16 * t + (l & 15), n = j0 + 4 * (l >> 4);
        if (m >= a.M || n >= a.N || !a.ep.y) continue;
        const int left = (int)(a.N - n < 4 ? a.N - n : 4);
        f32x4 v = sum[w * a.kw][t][l];
        for (int q = 1; q < a.kw; ++q) v += sum[w * a.kw + q][t][l];
        float z[4] = {v[0], v[1], v[2], v[3]}, bias[4];
        Loose<T, 4> r;
        if (a.ep.bias) load_row<T, 4>((const T*)a.ep.bias + n, left, bias);
        if (a.ep.residual) r = raw_row<T, 4>((const T*)a.ep.residual + m * a.ep.ldr + n, left);
        finish<T, 4>(a.ep, m, (int)n, left, z, bias, r);
    }
    if (want)
        for (int e = threadIdx.x; e < mw * MT * 16; e += 512) {
            const int l = e & 15, t = (e >> 4) % MT, w = (e >> 4) / MT;
            const long long m = ((long long)by * mw + w) * (16 * MT) + 16 * t + l;
            if (m >= a.M) continue;
            float v = total[w * a.kw][t][l];
            for (int q = 1; q < a.kw; ++q) v += total[w * a.kw + q][t][l];
            ((T*)a.sums)[m] = (T)v;
        }
}
template <typename T, bool TRP, bool TRQ, int MT>
__global__ __launch_bounds__(512) void direct_kernel(DirectArgs a) {
    __shared__ DirectRoom<T, MT> room;
    direct_product<T, TRP, TRQ, MT>(a, room, blockIdx.y);
}
// both products of a small backward pass: the rows of workgroups of the first (dx = d w), then those of the second (dw = d^T x)
template <typename T, int MT>
__global__ __launch_bounds__(512) void direct_pair_kernel(DirectArgs x, DirectArgs w, unsigned first) {
    __shared__ DirectRoom<T, MT> room;
    if (blockIdx.y < first) direct_product<T, false, true, MT>(x, room, blockIdx.y);
    else direct_product<T, true, true, MT>(w, room, blockIdx.y - first);
}

}  // namespace ccsm_ops
