// Training operators: products with an epilogue, and their gradients (include/ccsm_train_ops.h).
//   forward    y = act(x w^T + bias) + residual        i = rows of x, j = rows of w, contraction over `inner`
//   dx = d w                                           i = rows of d, j = columns of w, contraction over `outer`
//   dw = d^T x                                         i = columns of d, j = columns of x, contraction over `rows`
#include "ccsm_train_ops_mfma.h"

namespace ccsm_ops {

// the parts of a bias gradient in a fixed order: a workgroup takes eight columns, each lane every 32nd part; the 32 sums are added in order
struct ColumnJob { const float* part; int parts; int N; void* out; unsigned blocks; };
template <typename T>
__device__ __forceinline__ void column_join(const ColumnJob& job, unsigned block) {
    __shared__ float s[32][9];
    const int c = threadIdx.x & 7, q = threadIdx.x >> 3, n = (int)block * 8 + c;
    float a = 0.f;
    if (n < job.N) {
#pragma unroll 8
        for (int p = q; p < job.parts; p += 32) a += job.part[(long long)p * job.N + n];
    }
    s[q][c] = a;
    __syncthreads();
    if (q == 0 && n < job.N) {
        for (int k = 1; k < 32; ++k) a += s[k][c];
        ((T*)job.out)[n] = (T)a;
    }
}
// what is left to add up behind the products of a call, in one launch
template <typename T>
__global__ __launch_bounds__(256) void joins_kernel(ColumnJob c, JoinJob a, JoinJob b) {
    unsigned block = blockIdx.x;
    if (block < c.blocks) { column_join<T>(c, block); return; }
    block -= c.blocks;
    if (block < a.blocks) product_join<T>(a, block);
    else product_join<T>(b, block - a.blocks);
}
template <typename T>
__global__ __launch_bounds__(256) void fill_zero_kernel(T* p, long long ld, long long rows, int cols) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (long long)gridDim.x * 256) p[i / cols * ld + i % cols] = (T)0.f;
}

}  // namespace ccsm_ops
