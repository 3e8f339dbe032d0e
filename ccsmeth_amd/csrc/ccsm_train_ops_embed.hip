// Training operators: embedding lookup with scaling, and the table's gradient by sorted tokens (include/ccsm_train_ops.h).
//
// Gradient: dtable[v] = scale * sum of dy[i] over the tokens i with ids[i] = v.  The tokens are sorted by id with a stable radix sort (8 bits at
// most a pass), so that the rows of one sum lie next to each other in token order; each group of lanes then walks a piece of kPiece sorted
// tokens and adds rows up in fp32 registers, eight rows in flight.  A sum that lies inside a piece is written at once; what crosses a piece's
// border goes to two partial rows of the workspace (its head, its tail), which a second kernel adds in a fixed order.  Rows of the table that no
// token names are marked by the sort's last pass (a byte for each row) and cleared by further workgroups of the sums' launch, so the table
// is written once.  No floating-point atomics: the order of a sum depends on the ids alone.
#include "ccsm_train_ops_common.h"

namespace ccsm_ops {

constexpr int kPiece = 32;              // sorted tokens per group of lanes

__device__ __forceinline__ unsigned id_at(const void* ids, int type, long long i, long long rows) {      // rows: no token
    const long long v = type == 0 ? ((const uint8_t*)ids)[i] : type == 1 ? ((const int32_t*)ids)[i] : ((const int64_t*)ids)[i];
    return v >= 0 && v < rows ? (unsigned)v : (unsigned)rows;
}

// one lane: N neighbouring values of one token's row
template <typename T, int N>
__global__ __launch_bounds__(256) void lookup_kernel(const void* ids, int id_type, unsigned items, Div pieces, long long rows, int width, const T* table, long long ldt,
                                                     float scale, T* y, long long ldy) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= items) return;
    const unsigned t = pieces.of(i);
    const int c = (int)(i - t * pieces.d) * N;
    const unsigned id = id_at(ids, id_type, t, rows);
    float v[N] = {};
    if (id < rows) load_row<T, N>(table + (long long)id * ldt + c, width - c, v);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] *= scale;
    if (id >= rows) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = 0.f;                  // (whatever the scale is)
    }
    store_row<T, N>(y + (long long)t * ldy + c, width - c, v);
}

// ---- the sort -------------------------------------------------------------------------------------------------------
// A workgroup takes 256 Q tokens, a wave 64 Q of them in order.  counts[digit][block] of this pass's digit; the first pass also clears the marks.
template <int Q>
__global__ __launch_bounds__(256) void sort_count_kernel(const void* ids, int id_type, const unsigned* keys, long long n, long long rows, int shift, int bins,
                                                         unsigned* counts, unsigned* marks, long long mark_words) {
    __shared__ unsigned h[256];
    h[threadIdx.x] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * (256 * Q);
    unsigned k[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const long long i = base + q * 256 + threadIdx.x;
        k[q] = i < n ? (keys ? keys[i] : id_at(ids, id_type, i, rows)) : 0;
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (base + q * 256 + threadIdx.x < n) atomicAdd(&h[(k[q] >> shift) & (bins - 1)], 1u);
    if (marks)
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < mark_words; i += (long long)gridDim.x * 256) marks[i] = 0;
    __syncthreads();
    if ((int)threadIdx.x < bins) counts[(long long)threadIdx.x * gridDim.x + blockIdx.x] = h[threadIdx.x];
}
// exclusive running sum of c[0 .. n), in place, one workgroup, four values a lane
__global__ __launch_bounds__(1024) void sort_scan_kernel(unsigned* c, long long n) {
    __shared__ unsigned part[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned carry = 0;
    for (long long b = 0; b < n; b += 4096) {
        const long long i = b + 4 * threadIdx.x;
        unsigned v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = i + k < n ? c[i + k] : 0;
        const unsigned mine = v[0] + v[1] + v[2] + v[3];
        unsigned s = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned t = __shfl_up(s, o);
            if (lane >= o) s += t;
        }
        if (lane == 63) part[wave] = s;
        __syncthreads();
        unsigned at = carry + s - mine;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            if (w < wave) at += part[w];
            carry += part[w];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (i + k < n) c[i + k] = at;
            at += v[k];
        }
        __syncthreads();
    }
}
// a lane's place = its digit's next free place + how many lower lanes hold the same digit
template <int Q>
__global__ __launch_bounds__(256) void sort_scatter_kernel(const void* ids, int id_type, const unsigned* keys, const unsigned* at, long long n, long long rows, int shift,
                                                           int bins, const unsigned* starts, unsigned* keys_out, unsigned* at_out, uint8_t* marks) {
    __shared__ unsigned next[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = threadIdx.x; d < 1024; d += 256) (&next[0][0])[d] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * (256 * Q) + wave * (64 * Q);
    unsigned k[Q], from[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const long long i = base + q * 64 + lane;
        k[q] = i < n ? (keys ? keys[i] : id_at(ids, id_type, i, rows)) : 0;
        from[q] = at && i < n ? at[i] : (unsigned)i;
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (base + q * 64 + lane < n) atomicAdd(&next[wave][(k[q] >> shift) & (bins - 1)], 1u);
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
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const bool in = base + q * 64 + lane < n;
        const unsigned d = (k[q] >> shift) & (bins - 1);
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
            keys_out[place] = k[q];
            at_out[place] = from[q];
            if (marks && k[q] < rows) marks[k[q]] = 1;
        }
    }
}

// ---- the sums -------------------------------------------------------------------------------------------------------
// workgroups [0, sums): a group of lanes = one piece of sorted tokens, a lane of it = N neighbouring columns.  The others clear the rows of the
// table that have no mark.
template <typename T, int N>
__global__ __launch_bounds__(256) void piece_sum_kernel(const unsigned* keys, const unsigned* at, long long n, long long rows, unsigned sums, Div lanes, int width, const T* dy,
                                                        long long lddy, float scale, T* dt, long long ldt, float* part, long long part_ld, const uint8_t* marks) {
    if (blockIdx.x >= sums) {
        // eight rows' marks at a time
        for (long long r0 = (blockIdx.x - sums) * 8ll; r0 < rows; r0 += (gridDim.x - sums) * 8ll)
            for (unsigned i = threadIdx.x; i < 8 * lanes.d; i += 256) {
                const unsigned q = lanes.of(i);
                const long long r = r0 + q;
                const int c = (int)(i - q * lanes.d) * N;
                const float z[N] = {};
                if (r < rows && !marks[r]) store_row<T, N>(dt + r * ldt + c, width - c, z);
            }
        return;
    }
    const unsigned id = blockIdx.x * 256u + threadIdx.x, g = lanes.of(id);
    const int c = (int)(id - g * lanes.d) * N;
    const long long s = (long long)g * kPiece;
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
            float* o = part + (2ll * g + (open ? 0 : 1)) * part_ld + c;
#pragma unroll
            for (int k = 0; k < N; k += 4) {
                if constexpr (N >= 4) *(Vec<float, 4>*)(o + k) = Vec<float, 4>{{acc[k], acc[k + 1], acc[k + 2], acc[k + 3]}};
                else o[k] = acc[k];
            }
        } else {
            float v[N];
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = acc[k] * scale;
            store_row<T, N>(dt + (long long)cur * ldt + c, width - c, v);
        }
    };
    constexpr int kAhead = 8;
    for (long long b = s; b < e; b += kAhead) {
        unsigned k[kAhead];
        float v[kAhead][N];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) k[q] = b + q < e ? keys[b + q] : (unsigned)rows;
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const long long i = b + q < e ? at[b + q] : 0;
            if (k[q] < rows) load_row<T, N>(dy + i * lddy + c, width - c, v[q]);
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            if (b + q >= e) break;
            if (k[q] != cur) {
                flush(false);
                cur = k[q];
                open = false;
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] = 0.f;
            }
            if (cur < rows) {
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] += v[q][j];
            }
        }
    }
    flush(e < n && keys[e] == cur);
}
// One workgroup per piece: the sum that starts in it and leaves it, if there is one = tail of the piece + heads of the following ones.  The lanes
// take four columns each and share the heads between them; their sums are added in order.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const unsigned* keys, long long n, long long rows, int width, float scale, T* dt, long long ldt, const float* part,
                                                   long long part_ld) {
    const long long g = blockIdx.x, s = g * kPiece, e = s + kPiece;
    if (e >= n) return;
    const unsigned k = keys[e - 1];
    if (k >= rows || keys[e] != k) return;
    if (keys[s] == k && s > 0 && keys[s - 1] == k) return;         // it began earlier
    long long lo = e + 1, hi = n;                                  // the first token behind the sum
    bool near = true;
    for (long long step = kPiece; lo < hi; step = near ? 4 * step : step) {            // (most sums are short: look nearby first, then further and further, then between)
        near = near && lo + step < hi;
        const long long m = near ? lo + step : (lo + hi) >> 1;
        if (keys[m] == k) lo = m + 1; else { hi = m; near = false; }
    }
    const long long last = (lo - 1) / kPiece;                      // the piece of its last token
    __shared__ Vec<float, 4> sum[256];
    const int cols = (width + 3) / 4, wide = cols < 256 ? cols : 256, slices = 256 / wide;
    const int slice = threadIdx.x / wide, lane = threadIdx.x % wide;
    for (int c0 = 0; c0 < cols; c0 += wide) {
        const int c = 4 * (c0 + lane);
        float a[4] = {};
        if (slice < slices && c < width) {
            if (slice == 0) {
                const Vec<float, 4> v = *(const Vec<float, 4>*)(part + (2 * g + 1) * part_ld + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) a[j] = v.v[j];
            }
#pragma unroll 8
            for (long long p = g + 1 + slice; p <= last; p += slices) {
                const Vec<float, 4> v = *(const Vec<float, 4>*)(part + 2 * p * part_ld + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) a[j] += v.v[j];
            }
        }
        __syncthreads();
        sum[threadIdx.x] = Vec<float, 4>{{a[0], a[1], a[2], a[3]}};
        __syncthreads();
        // halves are added together, slice by slice
        for (int w = 1; w < slices; w <<= 1) {
            if (slice < slices && slice % (2 * w) == 0 && slice + w < slices) {
                const Vec<float, 4> v = sum[threadIdx.x + w * wide];
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[threadIdx.x].v[j] += v.v[j];
            }
            __syncthreads();
        }
        if (slice == 0 && c < width) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = sum[threadIdx.x].v[j] * scale;
            store_row<T, 4>(dt + (long long)k * ldt + c, width - c, v);
        }
    }
}

}  // namespace ccsm_ops
