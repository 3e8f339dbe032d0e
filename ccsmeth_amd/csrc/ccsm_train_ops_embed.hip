// Training operators: embedding lookup with scaling, and the table's gradient by sorted tokens (include/ccsm_train_ops.h).
//
// Gradient: dtable[v] = scale * sum of dy[i] over the tokens i with ids[i] = v.  The tokens are sorted by id with a stable radix sort (8 bits at
// most a pass), so that the rows of one sum lie next to each other in token order; each group of lanes then walks a piece of kPiece sorted
// tokens and adds rows up in fp32 registers.  A sum that lies inside a piece is written at once; what crosses a piece's border goes to two
// partial rows of the workspace (its head, its tail), which a second kernel adds in piece order.  No atomics: the order of a sum depends on the
// ids alone.
#include "ccsm_train_ops_common.h"

namespace ccsm_ops {

constexpr int kSortItems = 4096;        // tokens per workgroup of the sort: 256 threads x 16
constexpr int kPiece = 32;              // sorted tokens per group of lanes

__device__ __forceinline__ unsigned id_at(const void* ids, int type, long long i, long long rows) {      // rows: no token
    const long long v = type == 0 ? ((const uint8_t*)ids)[i] : type == 1 ? ((const int32_t*)ids)[i] : ((const int64_t*)ids)[i];
    return v >= 0 && v < rows ? (unsigned)v : (unsigned)rows;
}

template <typename T, int N>
__global__ __launch_bounds__(256) void lookup_kernel(const void* ids, int id_type, long long tokens, long long rows, int pieces, const T* table, long long ldt,
                                                     float scale, T* y, long long ldy) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < tokens * pieces; i += (long long)gridDim.x * 256) {
        const long long t = i / pieces;
        const int c = (int)(i % pieces) * N;
        const unsigned id = id_at(ids, id_type, t, rows);
        Vec<T, N> v;
        if (id < rows) v = *(const Vec<T, N>*)(table + (long long)id * ldt + c);
#pragma unroll
        for (int k = 0; k < N; ++k) v.v[k] = id < rows ? (T)((float)v.v[k] * scale) : (T)0.f;
        *(Vec<T, N>*)(y + t * ldy + c) = v;
    }
}

// ---- the sort -------------------------------------------------------------------------------------------------------
// counts[digit][block] of this pass's digit
__global__ __launch_bounds__(256) void sort_count_kernel(const void* ids, int id_type, const unsigned* keys, long long n, long long rows, int shift, int bins,
                                                         unsigned* counts) {
    __shared__ unsigned h[256];
    h[threadIdx.x] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * kSortItems;
    for (int q = 0; q < kSortItems / 256; ++q) {
        const long long i = base + q * 256 + threadIdx.x;
        if (i < n) atomicAdd(&h[((keys ? keys[i] : id_at(ids, id_type, i, rows)) >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    if ((int)threadIdx.x < bins) counts[(long long)threadIdx.x * gridDim.x + blockIdx.x] = h[threadIdx.x];
}
// exclusive running sum of c[0 .. n), in place, one workgroup
__global__ __launch_bounds__(1024) void sort_scan_kernel(unsigned* c, long long n) {
    __shared__ unsigned part[16];
    __shared__ unsigned carry;
    if (threadIdx.x == 0) carry = 0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (long long b = 0; b < n; b += 1024) {
        const long long i = b + threadIdx.x;
        const unsigned v = i < n ? c[i] : 0;
        unsigned s = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned t = __shfl_up(s, o);
            if (lane >= o) s += t;
        }
        if (lane == 63) part[wave] = s;
        __syncthreads();
        unsigned before = carry;
        for (int w = 0; w < wave; ++w) before += part[w];
        if (i < n) c[i] = before + s - v;
        __syncthreads();
        if (threadIdx.x == 1023) carry = before + s;
        __syncthreads();
    }
}
// a wave takes 1024 items in order, 64 at a time: a lane's place = the digit's next free place + how many lower lanes hold the same digit
__global__ __launch_bounds__(256) void sort_scatter_kernel(const void* ids, int id_type, const unsigned* keys, const unsigned* at, long long n, long long rows, int shift,
                                                           int bins, const unsigned* starts, unsigned* keys_out, unsigned* at_out) {
    __shared__ unsigned next[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = threadIdx.x; d < 1024; d += 256) (&next[0][0])[d] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * kSortItems + wave * 1024;
    auto key = [&](long long i) { return keys ? keys[i] : id_at(ids, id_type, i, rows); };
    for (int q = 0; q < 16; ++q) {
        const long long i = base + q * 64 + lane;
        if (i < n) atomicAdd(&next[wave][(key(i) >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    if ((int)threadIdx.x < bins) {
        unsigned s = starts[(long long)threadIdx.x * gridDim.x + blockIdx.x];
        for (int w = 0; w < 4; ++w) {
            const unsigned t = next[w][threadIdx.x];
            next[w][threadIdx.x] = s;
            s += t;
        }
    }
    __syncthreads();
    for (int q = 0; q < 16; ++q) {
        const long long i = base + q * 64 + lane;
        const bool in = i < n;
        const unsigned k = in ? key(i) : 0, d = (k >> shift) & (bins - 1);
        unsigned long long same = __ballot(in);
        for (int b = 1; b < bins; b <<= 1) {
            const unsigned long long on = __ballot((d & b) != 0);
            same &= (d & b) ? on : ~on;
        }
        const int before = __popcll(same & ((1ull << lane) - 1));
        const unsigned place = in ? next[wave][d] + before : 0;
        __builtin_amdgcn_wave_barrier();
        if (in && before == 0) next[wave][d] += __popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (in) {
            keys_out[place] = k;
            at_out[place] = at ? at[i] : (unsigned)i;
        }
    }
}

// ---- the sums -------------------------------------------------------------------------------------------------------
// group of lanes g = one piece of sorted tokens; lane l of the group = columns N l .. of the row
template <typename T, int N>
__global__ __launch_bounds__(256) void piece_sum_kernel(const unsigned* keys, const unsigned* at, long long n, long long rows, int lanes, int width, const T* dy,
                                                        long long lddy, float scale, T* dt, long long ldt, float* part) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long g = id / lanes;
    const int c = (int)(id % lanes) * N;
    const long long s = g * kPiece;
    if (s >= n) return;
    const long long e = s + kPiece < n ? s + kPiece : n;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    unsigned cur = keys[s];
    bool open = s > 0 && keys[s - 1] == cur;       // this sum began in an earlier piece
    auto flush = [&](bool goes_on) {
        if (cur >= rows) return;
        if (open || goes_on) {
            float* o = part + (2 * g + (open ? 0 : 1)) * (long long)width + c;
#pragma unroll
            for (int k = 0; k < N; ++k) o[k] = acc[k];
        } else {
            Vec<T, N> v;
#pragma unroll
            for (int k = 0; k < N; ++k) v.v[k] = (T)(acc[k] * scale);
            *(Vec<T, N>*)(dt + (long long)cur * ldt + c) = v;
        }
    };
    for (long long i = s; i < e; ++i) {
        const unsigned k = keys[i];
        if (k != cur) {
            flush(false);
            cur = k;
            open = false;
#pragma unroll
            for (int q = 0; q < N; ++q) acc[q] = 0.f;
        }
        if (k >= rows) break;                      // no tokens from here on
        const Vec<T, N> v = *(const Vec<T, N>*)(dy + (long long)at[i] * lddy + c);
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] += (float)v.v[q];
    }
    flush(cur < rows && e < n && keys[e] == cur);
}
// workgroups [0, pieces): the sum that starts in this piece and leaves it, if there is one: tail of the piece + heads of the following ones.
// workgroups from `pieces` on: rows of the table that no token names are zero.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const unsigned* keys, long long n, long long rows, int width, float scale, T* dt, long long ldt, const float* part,
                                                   long long pieces) {
    auto first_at_least = [&](unsigned v, long long lo) {
        long long hi = n;
        while (lo < hi) {
            const long long m = (lo + hi) >> 1;
            if (keys[m] < v) lo = m + 1; else hi = m;
        }
        return lo;
    };
    if (blockIdx.x >= pieces) {
        for (long long r = blockIdx.x - pieces; r < rows; r += gridDim.x - pieces) {
            const long long i = first_at_least((unsigned)r, 0);
            if (i < n && keys[i] == (unsigned)r) continue;
            for (int c = threadIdx.x; c < width; c += 256) dt[r * ldt + c] = (T)0.f;
        }
        return;
    }
    const long long g = blockIdx.x, e = (g + 1) * kPiece;
    if (e >= n) return;
    const unsigned k = keys[e - 1];
    if (k >= rows || keys[e] != k) return;
    const long long s = g * kPiece;
    if (keys[s] == k && s > 0 && keys[s - 1] == k) return;         // it began earlier
    const long long last = (first_at_least(k + 1, e) - 1) / kPiece;  // the piece of its last token
    for (int c = threadIdx.x; c < width; c += 256) {
        float a = part[(2 * g + 1) * (long long)width + c];
        for (long long p = g + 1; p <= last; ++p) a += part[2 * p * (long long)width + c];
        dt[(long long)k * ldt + c] = (T)(a * scale);
    }
}

}  // namespace ccsm_ops
