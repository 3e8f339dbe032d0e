// Training operators: products with an epilogue, and their gradients (include/ccsm_train_ops.h).
//   forward    y = act(x w^T + bias) + residual        i = rows of x, j = rows of w, contraction over `inner`
//   dx = d w                                           i = rows of d, j = columns of w, contraction over `outer`
//   dw = d^T x                                         i = columns of d, j = columns of x, contraction over `rows`
#include "ccsm_train_ops_common.h"

namespace ccsm_ops {

// One operand: element (free index i, contraction index k) at row i, column k of the stored matrix (TR: at row k, column i)
struct Operand { Saved m; int tr; };
struct Epilogue {
    const void* bias; const void* residual; long long ldr; void* y; long long ldy; void* pre; long long ldp; int act;
};

// Any sizes, strides and alignment: a 64 x 64 tile per workgroup of 256 threads, 4 x 4 outputs per thread, 16 contraction steps through LDS as
// fp32, fp32 FMA.
template <typename T>
__global__ __launch_bounds__(256) void product_fma_kernel(Operand A, Operand B, long long M, long long N, long long K, Epilogue ep) {
    __shared__ float sa[16][64 + 4], sb[16][64 + 4];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const long long i0 = (long long)blockIdx.y * 64, j0 = (long long)blockIdx.x * 64;
    float acc[4][4] = {};
    for (long long k0 = 0; k0 < K; k0 += 16) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int e = threadIdx.x + 256 * q;
            const int ka = A.tr ? e >> 6 : e & 15, ia = A.tr ? e & 63 : e >> 4, kb = B.tr ? e >> 6 : e & 15, jb = B.tr ? e & 63 : e >> 4;
            const long long k1 = k0 + ka, i = i0 + ia, k2 = k0 + kb, j = j0 + jb;
            sa[ka][ia] = k1 < K && i < M ? (A.tr ? saved_at<T>(A.m, k1, i) : saved_at<T>(A.m, i, k1)) : 0.f;
            sb[kb][jb] = k2 < K && j < N ? (B.tr ? saved_at<T>(B.m, k2, j) : saved_at<T>(B.m, j, k2)) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int b = 0; b < 4; ++b) acc[a][b] = fmaf(sa[k][ty * 4 + a], sb[k][tx * 4 + b], acc[a][b]);
        __syncthreads();
    }
    constexpr bool fast = sizeof(T) == 2;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const long long i = i0 + ty * 4 + a, j = j0 + tx * 4 + b;
            if (i >= M || j >= N) continue;
            const float z = acc[a][b] + (ep.bias ? (float)((const T*)ep.bias)[j] : 0.f);
            if (ep.pre) ((T*)ep.pre)[i * ep.ldp + j] = (T)z;
            float y = act_<fast>(z, ep.act);
            if (ep.residual) y += (float)((const T*)ep.residual)[i * ep.ldr + j];
            ((T*)ep.y)[i * ep.ldy + j] = (T)y;
        }
}

// d = dy act'(z), rounded to T (fp32: not at all): 16-bit products take 16-bit operands, and this rounding (half a step of T per factor,
// independent of each other) moves a gradient by less than the rounding of the gradient itself does.  The bias gradient takes d before it.
// One workgroup: 32 rows x 256 columns; part[row block][column] = the column's sum over the block's rows, joined in block order.
template <typename T>
__global__ __launch_bounds__(256) void slope_kernel(const T* dy, long long lddy, Saved z, int act, long long M, int N, T* d, long long ldd, float* part) {
    constexpr bool fast = sizeof(T) == 2;
    const long long m0 = (long long)blockIdx.x * 32;
    const int n = blockIdx.y * 256 + threadIdx.x;
    if (n >= N) return;
    float sum = 0.f;
    for (int r = 0; r < 32 && m0 + r < M; ++r) {
        const long long m = m0 + r;
        float v = (float)dy[m * lddy + n];
        if (act != kActNone) v *= slope_<fast>(saved_at<T>(z, m, n), act);
        if (d) d[m * ldd + n] = (T)v;
        sum += v;
    }
    if (part) part[(long long)blockIdx.x * N + n] = sum;
}
template <typename T>
__global__ __launch_bounds__(256) void column_join_kernel(const float* part, long long parts, int N, T* out) {
    // 256 threads = 32 columns x 8 slices of the parts; the slices are added in order
    __shared__ float s[8][33];
    const int c = threadIdx.x & 31, q = threadIdx.x >> 5, n = blockIdx.x * 32 + c;
    float a = 0.f;
    if (n < N)
        for (long long p = q; p < parts; p += 8) a += part[p * N + n];
    s[q][c] = a;
    __syncthreads();
    if (q == 0 && n < N) {
        for (int k = 1; k < 8; ++k) a += s[k][c];
        out[n] = (T)a;
    }
}
template <typename T>
__global__ __launch_bounds__(256) void fill_zero_kernel(T* p, long long ld, long long rows, int cols) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (long long)gridDim.x * 256) p[i / cols * ld + i % cols] = (T)0.f;
}

}  // namespace ccsm_ops
