// Training operators: embedding lookup with scaling, and the table's gradient by sorted tokens (include/ccsm_train_ops.h).
//
// Gradient: dtable[v] = scale * sum of dy[i] over the tokens i with ids[i] = v.  The tokens are sorted by id with a stable radix sort (8 bits at
// most a pass), so that the rows of one sum lie next to each other in token order; each group of lanes then walks a piece of sorted tokens and adds
// rows up in fp32 registers, the next ones in flight.  A sum that lies inside a piece is written at once; what crosses a piece's
// border goes to two partial rows of the workspace (its head, its tail), which a second kernel adds in a fixed order.  Rows of the table that no
// token names are marked by the sort's last pass (a byte for each row) and cleared by further workgroups of the sums' launch, so the table
// is written once.  No floating-point atomics: the order of a sum depends on the ids alone.
//
// Tables of a few rows (bases, strands, segments) are not sorted for: every lane adds its tokens up in its own copy of the table's columns.
#include "ccsm_train_ops_common.h"

namespace ccsm_ops {

__device__ __forceinline__ unsigned id_at(const void* ids, int type, long long i, long long rows) {      // rows: no token
    const long long v = type == 0 ? ((const uint8_t*)ids)[i] : type == 1 ? ((const int32_t*)ids)[i] : ((const int64_t*)ids)[i];
    return v >= 0 && v < rows ? (unsigned)v : (unsigned)rows;
}

// a lane takes N neighbouring values of a token's row, four tokens (or parts of one) a workgroup apart: four ids, then four rows in flight.
// Bound by memory: 65536 x 1024 bf16 in 51 us, 268 MB read and written at 5.2 TB/s (a copy: 5.1)
template <typename T, int N>
__global__ __launch_bounds__(256) void lookup_kernel(const void* ids, int id_type, unsigned items, Div pieces, long long rows, int width, const T* table, long long ldt,
                                                     float scale, T* y, long long ldy) {
    constexpr int U = 4;
    const unsigned first = blockIdx.x * (256u * U) + threadIdx.x;
    unsigned t[U], id[U];
    int c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned i = first + 256u * u;
        t[u] = pieces.of(i < items ? i : 0);
        c[u] = (int)((i < items ? i : 0) - t[u] * pieces.d) * N;
        id[u] = id_at(ids, id_type, t[u], rows);
    }
    Loose<T, N> r[U];                                      // (no token: the table's first row, not used; no condition between the loads)
    if (width % N == 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) r[u] = *reinterpret_cast<const Loose<T, N>*>(table + (long long)(id[u] < rows ? id[u] : 0) * ldt + c[u]);
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u) r[u] = raw_row<T, N>(table + (long long)(id[u] < rows ? id[u] : 0) * ldt + c[u], width - c[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = id[u] < rows ? (float)r[u].v[k] * scale : 0.f;
        if (first + 256u * u < items) store_row<T, N>(y + (long long)t[u] * ldy + c[u], width - c[u], v);
    }
}

// ---- the sort -------------------------------------------------------------------------------------------------------
// A workgroup takes 256 Q tokens, a wave 64 Q of them in order.  Up to kFewBlocks workgroups each sums up the counts itself (counts[block][digit]: a lane per
// digit; a kernel for that alone took 10 us at 65536 tokens, the sums inside the scatter 3); above, that square of reads costs more than the kernel, and
// counts[digit][block] are scanned.  The first pass also clears the marks and the list's length.
constexpr int kFewBlocks = 128;
template <int Q>
__global__ __launch_bounds__(256) void sort_count_kernel(const void* ids, int id_type, const unsigned* keys, long long n, long long rows, int shift, int bins,
                                                         unsigned* counts, unsigned* marks, long long mark_words, unsigned* list) {
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
    if (marks && blockIdx.x == 0 && threadIdx.x == 0) *list = 0;
    if (marks)
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < mark_words; i += (long long)gridDim.x * 256) marks[i] = 0;
    __syncthreads();
    if ((int)threadIdx.x < bins) counts[gridDim.x <= kFewBlocks ? (long long)blockIdx.x * bins + threadIdx.x : (long long)threadIdx.x * gridDim.x + blockIdx.x] = h[threadIdx.x];
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
    __shared__ unsigned wave_sum[4], sums[2][256];
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
    unsigned start = 0;
    if (gridDim.x <= kFewBlocks) {
        unsigned all = 0;
        const int groups = 256 / bins, d = threadIdx.x & (bins - 1);                  // (bins: a power of two, at most 256; every lane sums up)
        for (int b0 = 0; b0 < (int)gridDim.x; b0 += 16 * groups) {                    // (uniform trips, loads without a condition: sixteen in flight)
            unsigned t[16];
            const int b = b0 + threadIdx.x / bins;
#pragma unroll
            for (int q = 0; q < 16; ++q) t[q] = starts[min(b + q * groups, (int)gridDim.x - 1) * bins + d];
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                all += b + q * groups < (int)gridDim.x ? t[q] : 0;
                start += b + q * groups < (int)blockIdx.x ? t[q] : 0;
            }
        }
        if (groups > 1) {
            sums[0][threadIdx.x] = all;
            sums[1][threadIdx.x] = start;
            __syncthreads();
            all = start = 0;
            for (int q = 0; q < groups && (int)threadIdx.x < bins; ++q) {
                all += sums[0][q * bins + threadIdx.x];
                start += sums[1][q * bins + threadIdx.x];
            }
        }
        unsigned s = all;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned t = __shfl_up(s, o);
            if (lane >= o) s += t;
        }
        if (lane == 63) wave_sum[wave] = s;
        __syncthreads();
        start += s - all;
        for (int w = 0; w < wave; ++w) start += wave_sum[w];
    } else {
        __syncthreads();
        if ((int)threadIdx.x < bins) start = starts[(long long)threadIdx.x * gridDim.x + blockIdx.x];
    }
    if ((int)threadIdx.x < bins) {
        unsigned s = start;
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
// Pieces of 32 sorted tokens, or of 8 where those would leave most of the chip idle (86016 x 72 fp16 in 32s are 378 waves of 32 rows each).
constexpr int kLongPiece = 32, kShortPiece = 8;
// Workgroups [0, sums) of a column block: `groups` groups of lanes with a piece of sorted tokens each, a lane = N neighbouring columns.  A sum that lies
// inside a piece is written at once.  What crosses pieces is put together in LDS by the group whose piece it starts in, and written if it ends in
// this workgroup; else it leaves as the workgroup's head or tail.  The other workgroups clear the rows of the table that have no mark.
// Measured (65536 x 1024 bf16 over 50000 rows, 15.5 thousand of them met, from memory): 70 us, 236 MB at 3.4 TB/s (84 with a
// condition on each row's load), the sort in front 26, the join behind 11.  Clearing first, or between the sums, took 5 and 25 us more; pieces of 8, 16,
// 64 tokens 7, 2, 25; eight more rows in flight spilled.
template <typename T, int N, int kPiece>
__global__ __launch_bounds__(256, 3) void piece_sum_kernel(const unsigned* keys, const unsigned* at, long long n, long long rows, unsigned sums, int groups, Div lanes, int width,
                                                        const T* dy, long long lddy, float scale, T* dt, long long ldt, float* part, long long part_ld, const uint8_t* marks,
                                                        unsigned* list) {
    const int c0 = blockIdx.y * 256 * N;
    if (blockIdx.x >= sums) {
        for (long long r0 = (blockIdx.x - sums) * 8ll; r0 < rows; r0 += (gridDim.x - sums) * 8ll)      // eight rows' marks at a time
            for (unsigned i = threadIdx.x; i < 8 * lanes.d; i += 256) {
                const unsigned q = lanes.of(i);
                const long long r = r0 + q;
                const int c = c0 + (int)(i - q * lanes.d) * N;
                const float z[N] = {};
                if (r < rows && c < width && !marks[r]) store_row<T, N>(dt + r * ldt + c, width - c, z);
            }
        return;
    }
    __shared__ float head[N][256], tail[N][256];
    __shared__ unsigned char kind[256];                    // of a group: 1 its head belongs to an earlier piece's sum, 2 the whole piece does and so does more, 4 it has a tail
    const int j = (int)lanes.of(threadIdx.x), c = c0 + ((int)threadIdx.x - j * (int)lanes.d) * N;
    const long long s = ((long long)blockIdx.x * groups + j) * kPiece;
    const bool on = j < groups && s < n && c < width;
    unsigned cur = 0;
    if (on) {
        const long long e = s + kPiece < n ? s + kPiece : n;
        constexpr int kAhead = 8;
        unsigned k[kAhead], from[kAhead];
        auto ahead = [&](long long b) {
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                k[q] = b + q < e ? keys[b + q] : (unsigned)rows;
                from[q] = b + q < e ? at[b + q] : 0;
            }
        };
        ahead(s);
        const bool whole = width - c >= N;
        const unsigned before = s > 0 ? keys[s - 1] : ~0u, after = e < n ? keys[e] : ~0u;
        float acc[N];
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] = 0.f;
        cur = k[0];
        bool open = before == cur && cur < rows;           // this sum began in an earlier piece
        unsigned char is = open ? 1 : 0;
        auto flush = [&](bool goes_on) {
            if (cur >= rows) return;
            if (open) {
#pragma unroll
                for (int q = 0; q < N; ++q) head[q][threadIdx.x] = acc[q];
                if (goes_on) is |= 2;
            } else if (goes_on) {
#pragma unroll
                for (int q = 0; q < N; ++q) tail[q][threadIdx.x] = acc[q];
                is |= 4;
            } else {
                float v[N];
#pragma unroll
                for (int q = 0; q < N; ++q) v[q] = acc[q] * scale;
                store_row<T, N>(dt + (long long)cur * ldt + c, width - c, v);
            }
        };
#pragma unroll 1
        for (long long b = s; b < e; b += kAhead) {
            Loose<T, N> v[kAhead];
            unsigned now[kAhead];
#pragma unroll
            for (int q = 0; q < kAhead; ++q) now[q] = k[q];
            if (now[0] < rows) {                           // (sorted: tokens of no row are the last ones)
                if (whole) {                               // eight loads without a condition between them
#pragma unroll
                    for (int q = 0; q < kAhead; ++q) v[q] = *reinterpret_cast<const Loose<T, N>*>(dy + (long long)from[q] * lddy + c);
                } else {
#pragma unroll
                    for (int q = 0; q < kAhead; ++q) v[q] = raw_row<T, N>(dy + (long long)from[q] * lddy + c, width - c);
                }
            }
            if (kPiece > kAhead && b + kAhead < e) ahead(b + kAhead);
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                if (b + q >= e) break;
                if (now[q] != cur) {
                    flush(false);
                    cur = now[q];
                    open = false;
#pragma unroll
                    for (int t = 0; t < N; ++t) acc[t] = 0.f;
                }
                if (cur < rows) {
#pragma unroll
                    for (int t = 0; t < N; ++t) acc[t] += (float)v[q].v[t];
                }
            }
        }
        flush(after == cur);
        kind[j] = is;                                      // (every lane of the group writes the same)
    }
    __syncthreads();                                       // (lanes without a piece stay for the barriers below)
    // head[j] <- what the pieces from j on add to a sum that is open in front of j: a scan from behind, in steps of 1, 2, 4 ... groups (one by one, 128
    // groups of two lanes took 16 us)
    const int live = (int)(((n - (long long)blockIdx.x * groups * kPiece) + kPiece - 1) / kPiece), end = live < groups ? live : groups;
    for (int d = 1; d < end; d <<= 1) {
        const bool more = on && j + d < end && (kind[j] & 2);
        float a[N];
        unsigned char is = 0;
        if (more) {
            is = kind[j + d];
#pragma unroll
            for (int q = 0; q < N; ++q) a[q] = head[q][threadIdx.x + d * (int)lanes.d];
        }
        __syncthreads();
        if (more) {
#pragma unroll
            for (int q = 0; q < N; ++q) head[q][threadIdx.x] += a[q];
            if (!(is & 2)) kind[j] &= 5;                   // (every lane of the group writes the same)
        }
        __syncthreads();
    }
    if (!on) return;
    if (kind[j] & 4) {                                     // the group's tail and what follows it
        float a[N];
        const bool inside = j + 1 < end, closed = inside && !(kind[j + 1] & 2);
#pragma unroll
        for (int q = 0; q < N; ++q) a[q] = tail[q][threadIdx.x] + (inside ? head[q][threadIdx.x + (int)lanes.d] : 0.f);
        if (closed) {
#pragma unroll
            for (int q = 0; q < N; ++q) a[q] *= scale;
            store_row<T, N>(dt + (long long)cur * ldt + c, width - c, a);
        } else {
            float* o = part + (2ll * blockIdx.x + 1) * part_ld + c;
#pragma unroll
            for (int q = 0; q < N; q += 4) *(Vec<float, 4>*)(o + q) = Vec<float, 4>{{a[q], a[q + 1], a[q + 2], a[q + 3]}};
            if (c == 0) list[1 + atomicAdd(list, 1u)] = blockIdx.x;      // (the order of the list does not matter: each of its sums is complete by itself)
        }
    }
    if (j == 0 && (kind[0] & 1)) {                         // the workgroup's head
        float* o = part + 2ll * blockIdx.x * part_ld + c;
#pragma unroll
        for (int q = 0; q < N; q += 4)
            *(Vec<float, 4>*)(o + q) = Vec<float, 4>{{head[q][threadIdx.x], head[q + 1][threadIdx.x], head[q + 2][threadIdx.x], head[q + 3][threadIdx.x]}};
    }
}
// The listed workgroups: the sum that leaves one = its tail + the heads of the following ones, as far as they begin with the same key.  A
// workgroup takes 256 columns of one at a time; four columns a lane, the heads shared between the slices of lanes, whose sums are added in a
// fixed order.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const unsigned* keys, long long n, int piece, int width, float scale, T* dt, long long ldt, const float* part,
                                                   long long part_ld, const unsigned* list, int chunks) {
    __shared__ Vec<float, 4> sum[256];
    const int cols = (width + 3) / 4, wide = cols < 64 ? cols : 64, slices = 256 / wide;
    const int slice = threadIdx.x / wide, lane = threadIdx.x % wide;
    const long long items = (long long)list[0] * chunks;
    for (long long it = blockIdx.x; it < items; it += gridDim.x) {
        const long long g = list[1 + it / chunks];
        const unsigned k = keys[(g + 1) * piece];
        long long last = g;                                        // the piece of its last token
        for (int more = 256; more == 256; last += more) {
            const long long i = (last + 1 + threadIdx.x) * piece;
            more = __syncthreads_count(i < n && keys[i] == k);     // (keys are sorted: the pieces that begin with k are the next ones)
        }
        const int c = 4 * ((int)(it % chunks) * 64 + lane);
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
        for (int w = 1; w < slices; w <<= 1) {                     // neighbours are added together
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

// ---- tables of few rows ----------------------------------------------------------------------------------------------
// A lane has four neighbouring columns of every row in LDS (rows x 16 bytes) and adds to them the tokens of its slice, `per` of them, each `slices`
// behind the last, eight in flight.  Then the slices of the workgroup are added up, and few_join_kernel adds the workgroups' tables.  No atomics; the
// order of a sum depends on the sizes and ids alone.  Two launches, where the sort's way has four at
// least.  Measured (fp32, us a call with its host part, sort -> here): 5 x 8 21 -> 13.6 at 21504 tokens, 48 -> 19.5 at a million; 2 x 1024 60 -> 30 at 21504.
// Larger tables leave too few waves on a CU (15 x 256 24 -> 19 at 21504 tokens, but 316 -> 442 at a million; 15 x 1024 37 -> 52).
constexpr int kFewIds = 15, kFewValues = 2048;             // (62 KB of LDS at most)
template <typename T>
__global__ __launch_bounds__(256) void few_sum_kernel(const void* ids, int id_type, long long n, int rows, int per, Div lanes, int slices, int width, const T* dy,
                                                      long long lddy, float* part, long long part_ld) {
    typedef Vec<float, 4> V;
    extern __shared__ __align__(16) char room[];
    V* tab = (V*)room;                                     // [rows][257]
    const int j = (int)lanes.of(threadIdx.x), lane = (int)threadIdx.x - j * (int)lanes.d, c = (int)blockIdx.y * 1024 + 4 * lane;
    for (int r = 0; r < rows; ++r) tab[r * 257 + threadIdx.x] = V{};
    const long long base = (long long)blockIdx.x * slices * per + j;
    if (j < slices && c < width) {
        for (int b = 0; b < per; b += 8) {
            unsigned id[8];
            Loose<T, 4> v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const long long t = base + (long long)(b + q) * slices;
                id[q] = t < n ? id_at(ids, id_type, t, rows) : (unsigned)rows;
                if (t < n) v[q] = raw_row<T, 4>(dy + t * lddy + c, width - c);
            }
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (id[q] < (unsigned)rows) {
                    V o = tab[id[q] * 257 + threadIdx.x];
#pragma unroll
                    for (int k = 0; k < 4; ++k) o.v[k] += (float)v[q].v[k];
                    tab[id[q] * 257 + threadIdx.x] = o;
                }
        }
    }
    __syncthreads();
    // `many` lanes for each four columns of a row: each adds slices g, g + many, ... into slice g, the first of them those
    const int cells = rows * (int)lanes.d, many = cells >= 256 ? 1 : 256 / cells < slices ? 256 / cells : slices;
    for (int pass = 0; pass < 2; ++pass) {
        const int step = pass ? 1 : many, end = pass ? many : slices, use = pass ? cells : cells * many;
        for (int e = threadIdx.x; e < use; e += 256) {
            const int g = e / cells, cell = e - g * cells, r = (int)lanes.of(cell), l = cell - r * (int)lanes.d;
            V o = tab[r * 257 + g * (int)lanes.d + l];
            for (int w = g + step; w < end; w += step) {
                const V a = tab[r * 257 + w * (int)lanes.d + l];
#pragma unroll
                for (int k = 0; k < 4; ++k) o.v[k] += a.v[k];
            }
            const int col = (int)blockIdx.y * 1024 + 4 * l;
            if (pass == 0) tab[r * 257 + g * (int)lanes.d + l] = o;
            else if (col < width) *(V*)(part + ((long long)blockIdx.x * rows + r) * part_ld + col) = o;
        }
        __syncthreads();
    }
}
// a workgroup: 16 lanes of four columns of the table, 16 slices of the parts
template <typename T>
__global__ __launch_bounds__(256) void few_join_kernel(const float* part, long long part_ld, int parts, int rows, int width, float scale, T* dt, long long ldt) {
    typedef Vec<float, 4> V;
    __shared__ V sum[16][16];
    const int lane = threadIdx.x & 15, slice = threadIdx.x >> 4;
    const long long quarter = part_ld / 4, cell = (long long)blockIdx.x * 16 + lane, all = rows * quarter;
    V o = {};
    if (cell < all)
#pragma unroll 4
        for (int p = slice; p < parts; p += 16) {
            const V a = *(const V*)(part + 4 * (p * all + cell));
#pragma unroll
            for (int k = 0; k < 4; ++k) o.v[k] += a.v[k];
        }
    sum[slice][lane] = o;
    __syncthreads();
    if (slice != 0 || cell >= all) return;
    for (int w = 1; w < 16; ++w) {
#pragma unroll
        for (int k = 0; k < 4; ++k) o.v[k] += sum[w][lane].v[k];
    }
    const long long r = cell / quarter;
    const int c = 4 * (int)(cell - r * quarter);
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = o.v[k] == 0.f ? 0.f : o.v[k] * scale;
    store_row<T, 4>(dt + r * ldt + c, width - c, v);
}

}  // namespace ccsm_ops
