// libccsm_train: the training operators' C-ABI (include/ccsm_train_ops.h).  Checks, workspace layout and launches; the kernels are in
// ccsm_train_ops_linear.hip, ccsm_train_ops_embed.hip and ccsm_train_ops_act8.hip.
#include <atomic>
#include <string>
#include <type_traits>

#include "../../include/ccsm_train_ops.h"
#include "ccsm_train_ops_act8.hip"
#include "ccsm_train_ops_embed.hip"
#include "ccsm_train_ops_linear.hip"

namespace {

using namespace ccsm_ops;

thread_local std::string g_err;
ccsm_status fail(ccsm_status s, const char* what) {
    try { g_err = what; } catch (...) {}
    return s;
}
ccsm_status hip_fail(hipError_t e, const char* what) {
    try { g_err = std::string(what) + ": " + hipGetErrorString(e); } catch (...) {}
    return CCSM_ERR_HIP;
}
#define REFUSE(cond, text) do { if (cond) return fail(CCSM_ERR_INVALID_ARG, text); } while (0)
#define LAUNCHED(what) do { hipError_t e_ = hipGetLastError(); if (e_ != hipSuccess) return hip_fail(e_, what); } while (0)

// makes `device` current for the call, and the caller's own again behind it
struct OnDevice {
    int before = -1;
    hipError_t err;
    explicit OnDevice(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device); else if (err == hipSuccess) before = -1;
    }
    ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
};
#define ON_DEVICE(device)                      \
    OnDevice on_device_(device);               \
    if (on_device_.err != hipSuccess) return hip_fail(on_device_.err, "hipSetDevice")

// Where direct_kernel takes a product.  Forward: at most 64 rows, or at most 2^27 multiplications whose contraction is short, since its steps follow each
// other without a tile's prefetch.  Measured (bf16 | fp32, us on the GPU, tile way -> direct): 512^3 10.4 -> 6.0 | 16.2 -> 8.9, 300 x 700 x 300
// 15.9 -> 6.2 | 12.8 -> 9.3; beyond: 1024^3 13.8 -> 24 | 30 -> 53; a contraction of 4096 (128 x 128 results) 11 -> 20.5 | 14.5 -> 39; results of
// 13377 x 768 (stored in pieces of 16 columns) 26 -> 51.  Backward: contractions of at most 512 and, both products together, three steps a CU,
// one workgroup each: 64 x 512 x 512 15.1 -> 11.3 | 19.3 -> 16.7, 500 x 2000 x 60 19.1 -> 15.3 | 23.9 -> 18.1; at two steps, 256 x 512 x 512, 15.5 -> 15.1 |
// 22 -> 19.7; at three, 300 x 500 x 400, 16.6 -> 21.4 | 22 -> 30, for gradients that keep what rounding d leaves; beyond: 512^3 16.2 -> 22.3 | 25 -> 31.
constexpr int64_t kFewRows = 64, kSmallProduct = 1 << 27, kSmallResult = 1 << 21, kShortForward = 1024, kShortBackward = 512, kBackwardSteps = 768;
constexpr int64_t kNarrow = 1 << 21;                              // row strides that the kernels' 32-bit offsets span
constexpr int64_t kMostRows = 0x7fffff00, kMostCols = 0x00ffff00;
// The tile kernels' offsets into an operand whose contraction index is contiguous: 255 rows and a row's 128 bytes, in the 32 bits of a buffer's extent.  A
// caller's own stride is below kNarrow; a staged copy (and d) is as wide as the contraction.  16 bits: 8421504 columns, fp32: 4210752
constexpr int64_t kExtent = 0xfffffffe;
// slope_kernel takes 32 rows x 256 columns a workgroup; a launch has less than 2^32 lanes, staging's workgroups among them
constexpr int64_t kSlopeBlocks = (1 << 24) - (1 << 16) - 1;

size_t size_of(int type) { return type == CCSM_TYPE_F32 ? 4 : 2; }
bool good_type(int t) { return t == CCSM_TYPE_F32 || t == CCSM_TYPE_F16 || t == CCSM_TYPE_BF16; }
bool off_by(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }
size_t up(size_t n, size_t a) { return (n + a - 1) / a * a; }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
unsigned grid_of(int64_t n, int64_t most = 1 << 20) { return (unsigned)(n < 1 ? 1 : n > most ? most : n); }

bool spanned(int64_t k, int type) { return 255 * (int64_t)up((size_t)k, 8) * (int64_t)size_of(type) + 128 <= kExtent; }

// scratch of a call, handed out piece by piece; without a base it only counts.  What the call takes beside it: the tile's edge (0: the small kernel) and
// the parts of each product's contraction (0: no such product), operands staged
struct Scratch {
    char* base = nullptr;
    size_t used = 0;
    int tile = 0, parts[2] = {0, 0}, staged = 0;
    template <typename T> T* take(size_t n) {
        T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used += up(n * sizeof(T), 256);
        return p;
    }
};
#define TYPED(type, ...)                                                       \
    do {                                                                       \
        if ((type) == CCSM_TYPE_F32) { typedef float T; __VA_ARGS__; }         \
        else if ((type) == CCSM_TYPE_F16) { typedef f16 T; __VA_ARGS__; }      \
        else { typedef b16 T; __VA_ARGS__; }                                   \
    } while (0)

// a matrix in memory: rows of `wide` bytes, `ld` bytes from one to the next
struct Held { const void* p; int64_t ld, rows, wide; };
Held held(const void* p, int64_t ld, int64_t rows, int64_t cols, size_t size) {      // (one row's stride may be anything)
    return Held{p, rows > 1 ? ld * (int64_t)size : 0, rows, cols * (int64_t)size};
}
// whether two of them share memory: their ranges meet, and they are not different columns of the same rows (of one row, the other's stride)
bool meet(const Held& a, const Held& b) {
    if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0) return false;
    const char *pa = (const char*)a.p, *pb = (const char*)b.p;
    if (pb >= pa + (a.rows - 1) * a.ld + a.wide || pa >= pb + (b.rows - 1) * b.ld + b.wide) return false;
    if (a.rows == 1 && b.rows == 1) return true;
    if (a.rows > 1 && b.rows > 1 && a.ld != b.ld) return true;
    const int64_t step = a.rows > 1 ? a.ld : b.ld, off = ((pb - pa) % step + step) % step;
    return off < a.wide || off + b.wide > step;
}
template <size_t NO, size_t NI>
bool shared(const Held (&out)[NO], const Held (&in)[NI]) {
    for (size_t o = 0; o < NO; ++o) {
        for (const Held& i : in) if (meet(out[o], i)) return true;
        for (size_t q = o + 1; q < NO; ++q) if (meet(out[o], out[q])) return true;
    }
    return false;
}

ccsm_status check_saved(const ccsm_saved& s, int type, int64_t width, const char* what) {
    REFUSE(!s.data, what);
    if (s.code == CCSM_CODE_NONE) {
        REFUSE(s.ld < width, "a kept matrix: ld is less than its width");
        REFUSE(off_by(s.data, size_of(type)), "a kept matrix is not aligned to its elements");
        return CCSM_OK;
    }
    REFUSE(s.code != CCSM_CODE_INT8 && s.code != CCSM_CODE_E4M3, "unknown code of a kept matrix");
    REFUSE(!s.scales, "a kept matrix in 8 bits needs its scales");
    REFUSE(s.ld % 32 != 0 || s.ld < (int64_t)up(width, 32) || s.lds < cdiv(width, 32), "a kept matrix in 8 bits: ld is a multiple of 32 and covers whole blocks, lds the blocks");
    REFUSE(off_by(s.data, 16), "a kept matrix in 8 bits is 16-byte aligned");
    return CCSM_OK;
}
Held held(const ccsm_saved& s, int64_t rows, int64_t cols, int type) {
    return s.code == CCSM_CODE_NONE ? held(s.data, s.ld, rows, cols, size_of(type)) : held(s.data, s.ld, rows, (int64_t)up((size_t)cols, 32), 1);
}
Held held_scales(const ccsm_saved& s, int64_t rows, int64_t cols) {
    return s.code == CCSM_CODE_NONE ? Held{nullptr, 0, 0, 0} : held(s.scales, s.lds, rows, cdiv(cols, 32), 1);
}
Saved saved_of(const ccsm_saved& s) { return Saved{s.data, s.ld, s.code, s.scales, s.lds}; }
Saved plain(const void* p, int64_t ld) { return Saved{p, ld, kCodeNone, nullptr, 0}; }

// An operand as the tile kernels take it: as it is where its rows consist of whole, aligned 16-byte pieces of the call's type, else a staged copy in the
// scratch (8-bit codes too: the values that they stand for)
bool whole_rows(const void* p, int64_t ld, int64_t width, int type) {
    const int64_t n = 16 / (int64_t)size_of(type);
    return !off_by(p, 16) && ld % n == 0 && width % n == 0 && ld < kNarrow;
}
// (both operands' copies in one launch: 3 us and a gap of 2 each)
struct Staging {
    StageJob jobs[2] = {};
    int count = 0;
    template <typename T> Plane of(const Saved& s, int64_t rows, int64_t width, Scratch& ws) {
        if (s.code == kCodeNone && whole_rows(s.data, s.ld, width, TypeOf<T>::v)) return Plane{s.data, s.ld};
        const int64_t ld = (int64_t)up(width, 8);
        T* out = ws.take<T>((size_t)rows * ld);
        jobs[count++] = StageJob{s, rows * ld / 8, (int)width, out, ld};
        ws.staged = count;
        return Plane{out, ld};
    }
    unsigned blocks() const { return grid_of(cdiv(jobs[0].items + jobs[1].items, 256), 1 << 16); }
    template <typename T> hipError_t launch(hipStream_t st) const {
        if (!count) return hipSuccess;
        stage_kernel<T><<<blocks(), 256, 0, st>>>(jobs[0], jobs[1]);
        return hipGetLastError();
    }
};

template <int B, typename F, typename... A>
hipError_t launch_tiles(F* f, std::atomic<uint64_t>& known, int64_t blocks, hipStream_t st, const A&... args) {
    constexpr int lds = 5 * B * 128;                    // two chunks of P, three of Q
    // an attribute of the function on each device: set once for each (setting it twice, from two threads, does no harm)
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const uint64_t bit = device < 64 ? (uint64_t)1 << device : 0;
    if (!(known.load(std::memory_order_relaxed) & bit)) {
        e = hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        known.fetch_or(bit, std::memory_order_relaxed);
    }
    f<<<(unsigned)blocks, B == 256 ? 512 : 256, lds, st>>>(args...);
    return hipGetLastError();
}
int64_t blocks_of(const ProductArgs& a) { return (int64_t)a.tiles_i * a.tiles_j * a.splits; }
template <typename T, bool TRP, bool TRQ, int B>
hipError_t launch_product(const ProductArgs& a, hipStream_t st) {
    static std::atomic<uint64_t> known{0};
    return launch_tiles<B>(&product_kernel<T, TRP, TRQ, B>, known, blocks_of(a), st, a);
}
template <typename T, int B>
hipError_t launch_pair(const ProductArgs& x, const ProductArgs& w, hipStream_t st) {
    static std::atomic<uint64_t> known{0};
    return launch_tiles<B>(&product_pair_kernel<T, B>, known, blocks_of(x) + blocks_of(w), st, x, w, (int)blocks_of(x));
}
// The tile and the number of parts of the contraction with the least estimated time.  The estimate: workgroups go in rounds, 256 of the large tile (one for
// each CU), 512 of the small one (two for each CU, and a round of up to 256 has them to itself); a round takes its chunks' measured time; parts cost a
// launch, their sums' way through memory, and a step of the join each.  Chunk times measured at 2048^3 and 4096 x 4096 x 1024 (us, 16 bits | fp32):
// large tile 1.3 | 4.5, small tile alone 0.55 | 1.4, in pairs 0.8 | 2.6.  Measured against the rule before (large tiles from 200 on, parts up to
// 512 workgroups), bf16 | fp32, us, before -> after: 4096 x 1024 x 1024 26.6 -> 14.1 | 61 -> 53; 2048^3 33 -> 23 | 101 -> 95; 30000 x 1800 x 600
// 92 -> 91 | 470 -> 372; 1024 x 4096 x 1024 26.3 -> 22.5 | 59 -> 57.
struct Shape { int tile, splits; };
struct Costs { double large, alone, pair, launch = 4, per_part = 0.08; };
Costs costs(bool f32) { return f32 ? Costs{4.5, 1.4, 2.6} : Costs{1.3, 0.55, 0.8}; }
Shape shape_of(int64_t M, int64_t N, int64_t chunks, bool f32) {
    const auto [large, alone, pair, launch, per_part] = costs(f32);
    const double sums = (double)M * (double)N * 8 / 6e6;     // (written and read at 6 TB/s)
    const int64_t tiles_big = cdiv(M, 256) * cdiv(N, 256), tiles_small = cdiv(M, 128) * cdiv(N, 128);
    Shape best{128, 1};
    double least = 0;
    for (int64_t s = 1; s <= 256 && (s == 1 || 2 * s <= chunks); s += s < 32 ? 1 : s / 8) {
        const double depth = (double)cdiv(chunks, s), join = s == 1 ? 0 : launch + per_part * (double)s + sums * (double)s;
        const int64_t big = tiles_big * s, small = tiles_small * s, rest = small % 512;
        if (s > 1 && small > 2048) break;
        const double in_big = (double)cdiv(big, 256) * large * depth + join;
        const double in_small = ((double)(small / 512) * pair + (rest == 0 ? 0 : rest <= 256 ? alone : pair)) * depth + join;
        if (s == 1 || in_small < least) { least = in_small; best = {128, (int)s}; }
        if (in_big < least) { least = in_big; best = {256, (int)s}; }
    }
    return best;
}
// the same of two products in one launch (M x N results over `chunks` each), whose workgroups share the CUs: the chunks of all of them, or the longest one
struct Pair { int tile, splits[2]; };
Pair pair_of(const int64_t (&M)[2], const int64_t (&N)[2], const int64_t (&chunks)[2], bool f32) {
    const auto [large, alone, pair, launch, per_part] = costs(f32);
    Pair best{128, {1, 1}};
    double least = -1;
    for (int tile = 128; tile <= 256; tile += 128) {
        int64_t tiles[2];
        for (int k = 0; k < 2; ++k) tiles[k] = cdiv(M[k], tile) * cdiv(N[k], tile);
        for (int64_t sx = 1; sx == 1 || (2 * sx <= chunks[0] && tiles[0] * sx <= 2048 && sx <= 64); sx += sx < 4 ? 1 : sx / 2)
            for (int64_t sw = 1; sw == 1 || (2 * sw <= chunks[1] && tiles[1] * sw <= 2048 && sw <= 256); sw += sw < 4 ? 1 : sw / 4 + 1) {
                const int64_t dx = cdiv(chunks[0], sx), dw = cdiv(chunks[1], sw), longest = dx > dw ? dx : dw, nx = tiles[0] * sx, nw = tiles[1] * sw;
                const int64_t slots = tile == 256 ? 256 : 512;
                const double chunk = tile == 256 ? large : nx + nw <= 256 ? alone : pair, alike = (double)longest * chunk;
                double t = (double)(nx * dx + nw * dw) / (double)slots * (tile == 256 ? large : pair);
                if (nx + nw > slots && (nx % slots || nw % slots)) t += 0.5 * (double)dw * chunk;      // (a last round that is half empty)
                if (t < alike) t = alike;
                if (sx > 1 || sw > 1) t += launch + per_part * (double)(sx > sw ? sx : sw);
                if (sx > 1) t += (double)M[0] * (double)N[0] * 8 * (double)sx / 6e6;
                if (sw > 1) t += (double)M[1] * (double)N[1] * 8 * (double)sw / 6e6;
                if (least < 0 || t < least) { least = t; best = {tile, {(int)sx, (int)sw}}; }
            }
    }
    return best;
}
// out(i, j) = sum over k P(i, k) Q(j, k) and the epilogue, in tiles and parts of that shape; with parts, what is left to add up goes to *join
template <typename T>
ProductArgs product_args(const Plane& p, const Plane& q, int64_t M, int64_t N, int64_t K, int64_t chunks, Shape shape, const Epilogue& ep, Scratch& ws, JoinJob* join) {
    ProductArgs a;
    a.P = p; a.Q = q;
    a.M = (int)M; a.N = (int)N; a.K = (int)K;
    a.ep = ep;
    a.tiles_i = (int)cdiv(M, shape.tile); a.tiles_j = (int)cdiv(N, shape.tile);
    a.depth = (int)(cdiv(chunks, shape.splits) * (128 / (int64_t)sizeof(T)));
    a.splits = (int)cdiv(K, a.depth);
    a.part_ld = (int64_t)up(N, 4);
    a.part = a.splits > 1 ? ws.take<float>((size_t)a.splits * M * a.part_ld) : nullptr;
    if (a.splits > 1) *join = JoinJob{a.part, a.splits, M, (int)N, a.part_ld, ep, grid_of(cdiv(M * cdiv(N, 4), 256), 1 << 16)};
    return a;
}
template <typename T> int64_t chunks_of(int64_t K) { return cdiv(K, 128 / (int64_t)sizeof(T)); }
template <typename T, bool TRP, bool TRQ>
hipError_t product(hipStream_t st, const Plane& p, const Plane& q, int64_t M, int64_t N, int64_t K, const Epilogue& ep, Scratch& ws, JoinJob* join, bool count) {
    const Shape shape = shape_of(M, N, chunks_of<T>(K), sizeof(T) == 4);
    const ProductArgs a = product_args<T>(p, q, M, N, K, chunks_of<T>(K), shape, ep, ws, join);
    ws.tile = shape.tile;
    ws.parts[TRP] = a.splits;
    if (count) return hipSuccess;
    return shape.tile == 256 ? launch_product<T, TRP, TRQ, 256>(a, st) : launch_product<T, TRP, TRQ, 128>(a, st);
}
template <typename T>
hipError_t joins(hipStream_t st, const ColumnJob& c, const JoinJob& a, const JoinJob& b) {
    const unsigned blocks = c.blocks + a.blocks + b.blocks;
    if (!blocks) return hipSuccess;
    joins_kernel<T><<<blocks, 256, 0, st>>>(c, a, b);
    return hipGetLastError();
}
#define TRY(x, what) do { hipError_t e_ = (x); if (e_ != hipSuccess) return hip_fail(e_, what); } while (0)

bool small_product(int64_t M, int64_t N, int64_t K) { return M * N <= kSmallResult && M * N * K <= kSmallProduct; }
int waves_along(int64_t K) {                                      // (a wave has a whole step of 32 at least)
    int kw = 1;
    while (kw < 8 && 32 * 2 * kw <= K) kw *= 2;
    return kw;
}
int64_t steps_of(int64_t M, int64_t N, int64_t K) {               // of all workgroups
    const int kw = waves_along(K);
    return cdiv(N, 16) * cdiv(M, 64 * (8 / kw)) * cdiv(K, 32 * kw);
}
DirectArgs direct_args(const Plane& p, const Plane& z, int act, const Plane& q, int64_t M, int64_t N, int64_t K, void* sums, const Epilogue& ep) {
    return DirectArgs{p, z, q, act, M, N, K, waves_along(K), sums, ep};
}
unsigned rows_of(const DirectArgs& a, int mt) { return (unsigned)cdiv(a.M, 16 * mt * (8 / a.kw)); }
template <typename T, bool TRP, bool TRQ>
hipError_t direct(hipStream_t st, const DirectArgs& a) {
    const int mt = a.M <= 16 ? 1 : 4;
    auto* f = mt == 1 ? &direct_kernel<T, TRP, TRQ, 1> : &direct_kernel<T, TRP, TRQ, 4>;
    f<<<dim3((unsigned)cdiv(a.N, 16), rows_of(a, mt)), 512, 0, st>>>(a);
    return hipGetLastError();
}
template <typename T>
hipError_t direct_pair(hipStream_t st, const DirectArgs& x, const DirectArgs& w) {      // (as many columns each)
    const int mt = x.M <= 16 && w.M <= 16 ? 1 : 4;
    auto* f = mt == 1 ? &direct_pair_kernel<T, 1> : &direct_pair_kernel<T, 4>;
    f<<<dim3((unsigned)cdiv(x.N, 16), rows_of(x, mt) + rows_of(w, mt)), 512, 0, st>>>(x, w, rows_of(x, mt));
    return hipGetLastError();
}

ccsm_status check_linear(const ccsm_linear* p) {
    REFUSE(!p, "linear: NULL argument");
    REFUSE(!good_type(p->type), "linear: unknown type");
    REFUSE(p->activation < CCSM_ACT_NONE || p->activation > CCSM_ACT_SILU, "linear: unknown activation");
    REFUSE(p->rows < 0 || p->rows > kMostRows || p->inner <= 0 || p->inner > kMostCols || p->outer <= 0 || p->outer > kMostCols, "linear: sizes out of range");
    REFUSE(p->rows > kFewRows && !spanned(p->inner, p->type), "linear: inner is too long for more than 64 rows");
    REFUSE(!p->w || (p->rows && (!p->x || !p->y)), "linear: x, w and y must be non-NULL");
    REFUSE(p->ldx < p->inner || p->ldw < p->inner || p->ldy < p->outer || (p->residual && p->ldr < p->outer) || (p->preact && p->ldp < p->outer), "linear: a row stride is less than the row's width");
    const size_t s = size_of(p->type);
    REFUSE(off_by(p->x, s) || off_by(p->w, s) || off_by(p->y, s) || off_by(p->bias, s) || off_by(p->residual, s) || off_by(p->preact, s), "linear: a pointer is not aligned to its elements");
    return CCSM_OK;
}
ccsm_status apart(const ccsm_linear* p) {
    const size_t s = size_of(p->type);
    const Held y = held(p->y, p->ldy, p->rows, p->outer, s), pre = held(p->preact, p->ldp, p->rows, p->outer, s), r = held(p->residual, p->ldr, p->rows, p->outer, s);
    const Held out[] = {y, pre}, in[] = {held(p->x, p->ldx, p->rows, p->inner, s), held(p->w, p->ldw, p->outer, p->inner, s), held(p->bias, p->outer, 1, p->outer, s)};
    REFUSE(shared(out, in) || meet(pre, r) || (meet(y, r) && (p->y != p->residual || (p->rows > 1 && p->ldy != p->ldr))), "linear: an output shares memory with another tensor");
    return CCSM_OK;
}
template <typename T>
ccsm_status linear_forward(const ccsm_linear* p, Scratch& ws, hipStream_t st, bool count) {
    const Epilogue ep{p->bias, p->residual, p->ldr, p->y, p->ldy, p->preact, p->ldp, p->activation};
    if (p->rows <= kFewRows || (p->inner <= kShortForward && small_product(p->rows, p->outer, p->inner))) {
        if (count) return CCSM_OK;
        TRY((direct<T, false, false>(st, direct_args(Plane{p->x, p->ldx}, Plane{p->x, p->ldx}, CCSM_ACT_NONE, Plane{p->w, p->ldw}, p->rows, p->outer, p->inner, nullptr, ep))), "linear_forward");
        return CCSM_OK;
    }
    Staging stage;
    const Plane x = stage.of<T>(plain(p->x, p->ldx), p->rows, p->inner, ws), w = stage.of<T>(plain(p->w, p->ldw), p->outer, p->inner, ws);
    if (!count) TRY(stage.launch<T>(st), "linear_forward");
    JoinJob join = {};
    TRY((product<T, false, false>(st, x, w, p->rows, p->outer, p->inner, ep, ws, &join, count)), "linear_forward");
    if (!count) TRY(joins<T>(st, ColumnJob{}, join, JoinJob{}), "linear_forward");
    return CCSM_OK;
}

ccsm_status check_grad(const ccsm_linear_grad* p) {
    REFUSE(!p, "linear_backward: NULL argument");
    REFUSE(!good_type(p->type), "linear_backward: unknown type");
    REFUSE(p->activation < CCSM_ACT_NONE || p->activation > CCSM_ACT_SILU, "linear_backward: unknown activation");
    REFUSE(p->rows < 0 || p->rows > kMostRows || p->inner <= 0 || p->inner > kMostCols || p->outer <= 0 || p->outer > kMostCols, "linear_backward: sizes out of range");
    const size_t s = size_of(p->type);
    REFUSE(off_by(p->dy, s) || off_by(p->w, s) || off_by(p->dx, s) || off_by(p->dw, s) || off_by(p->dbias, s), "linear_backward: a pointer is not aligned to its elements");
    if (p->rows) {
        REFUSE(!p->dy, "linear_backward: dy must be non-NULL");
        REFUSE(p->lddy < p->outer, "linear_backward: a row stride is less than the row's width");
        if (p->activation != CCSM_ACT_NONE) {
            ccsm_status e = check_saved(p->preact, p->type, p->outer, "linear_backward: an activation's slope needs the pre-activation");
            if (e != CCSM_OK) return e;
        }
        REFUSE(cdiv(p->rows, 32) * cdiv(p->outer, 256) > kSlopeBlocks, "linear_backward: more rows than a launch covers");
        REFUSE(p->dx && !spanned(p->outer, p->type), "linear_backward: outer is too long for dx");
        if (p->dx) REFUSE(!p->w || p->ldw < p->inner || p->lddx < p->inner, "linear_backward: dx needs w, and strides of at least inner");
        if (p->dw) {
            ccsm_status e = check_saved(p->x, p->type, p->inner, "linear_backward: dw needs x");
            if (e != CCSM_OK) return e;
        }
    }
    REFUSE(p->dw && p->lddw < p->inner, "linear_backward: a row stride is less than the row's width");
    return CCSM_OK;
}
ccsm_status apart(const ccsm_linear_grad* p) {
    const size_t s = size_of(p->type);
    const int64_t M = p->rows, K = p->inner, N = p->outer;
    const ccsm_saved none = {}, x = p->dw ? p->x : none, z = p->activation == CCSM_ACT_NONE ? none : p->preact;
    const Held out[] = {held(p->dx, p->lddx, M, K, s), held(p->dw, p->lddw, N, K, s), held(p->dbias, N, 1, N, s)};
    const Held in[] = {held(p->dy, p->lddy, M, N, s), held(p->dx ? p->w : nullptr, p->ldw, N, K, s), held(x, M, K, p->type), held_scales(x, M, K), held(z, M, N, p->type), held_scales(z, M, N)};
    REFUSE(shared(out, in), "linear_backward: an output shares memory with another tensor");
    return CCSM_OK;
}
template <typename T>
ccsm_status linear_backward(const ccsm_linear_grad* p, Scratch& ws, hipStream_t st, bool count) {
    const int64_t M = p->rows;
    const int K = p->inner, N = p->outer;
    if (M == 0) {
        if (count) return CCSM_OK;
        if (p->dw) fill_zero_kernel<T><<<grid_of(cdiv((int64_t)N * K, 256), 4096), 256, 0, st>>>((T*)p->dw, p->lddw, N, K);
        if (p->dbias) fill_zero_kernel<T><<<grid_of(cdiv(N, 256)), 256, 0, st>>>((T*)p->dbias, N, 1, N);
        LAUNCHED("linear_backward");
        return CCSM_OK;
    }
    Epilogue to_dx{nullptr, nullptr, 0, p->dx, p->lddx, nullptr, 0, kActNone}, to_dw{nullptr, nullptr, 0, p->dw, p->lddw, nullptr, 0, kActNone};
    const bool narrow = p->lddy < kNarrow && (!p->dx || p->ldw < kNarrow) && (p->activation == CCSM_ACT_NONE || p->preact.ld < kNarrow) && (!p->dw || p->x.ld < kNarrow);
    if (narrow && M <= kShortBackward && N <= kShortBackward && steps_of(M, K, N) + steps_of(N, K, M) <= kBackwardSteps) {
        // checkpoints are made values in a launch of their own: a lane would read them code by code along the rows (bf16, both operands in 8 bits, us a
        // backward pass: 512^3 52 -> 28, 64 x 512 x 512 43 -> 23)
        Staging stage;
        auto values = [&](const ccsm_saved& v, int width) { return v.code == kCodeNone ? Plane{v.data, v.ld} : stage.of<T>(saved_of(v), M, width, ws); };
        const Plane dy{p->dy, p->lddy}, z = p->activation == CCSM_ACT_NONE ? dy : values(p->preact, N), x = p->dw ? values(p->x, K) : dy;
        if (count) return CCSM_OK;
        TRY(stage.launch<T>(st), "linear_backward");
        const DirectArgs ax = direct_args(dy, z, p->activation, Plane{p->w, p->ldw}, M, K, N, nullptr, to_dx);
        const DirectArgs aw = direct_args(dy, z, p->activation, x, N, p->dw ? K : 1, M, p->dbias, to_dw);
        if (p->dx && p->dw) TRY(direct_pair<T>(st, ax, aw), "linear_backward: dx and dw");
        else if (p->dx) TRY((direct<T, false, true>(st, ax)), "linear_backward: dx");
        if (!(p->dx && p->dw) && (p->dw || p->dbias))              // (the bias gradient comes with dw's product, or by the same sums without it)
            TRY((direct<T, true, true>(st, aw)), "linear_backward: dw");
        return CCSM_OK;
    }
    // d as the products take it: dy itself where there is no activation and its rows are whole pieces
    const bool products = p->dx || p->dw;
    const Saved dy = plain(p->dy, p->lddy);
    const bool none = p->activation == CCSM_ACT_NONE, as_is = none && whole_rows(p->dy, p->lddy, N, TypeOf<T>::v), make = products && !as_is;
    const int64_t ldd = (int64_t)up(N, 8), parts = cdiv(M, 32);
    T* made = make ? ws.take<T>((size_t)M * ldd) : nullptr;
    const Plane d = make ? Plane{made, ldd} : Plane{p->dy, p->lddy};
    float* part = p->dbias ? ws.take<float>((size_t)parts * N) : nullptr;
    Staging stage;
    const Plane w = p->dx ? stage.of<T>(plain(p->w, p->ldw), N, K, ws) : Plane{}, x = p->dw ? stage.of<T>(saved_of(p->x), M, K, ws) : Plane{};
    const bool scaled = TypeOf<T>::v == CCSM_TYPE_F16 && make && !none;      // (d is dy itself without an activation)
    float *most = scaled ? ws.take<float>(kMosts) : nullptr, *factor = scaled ? ws.take<float>(1) : nullptr;
    to_dx.factor = to_dw.factor = factor;
    if (!count && (part || make)) {
        const int64_t items = M * cdiv(N, 8);
        const int mosts = scaled ? (int)grid_of(cdiv(items, 1024), kMosts) : 0;
        if (scaled) most_kernel<<<(unsigned)mosts, 1024, 0, st>>>((const f16*)p->dy, p->lddy, items, (unsigned)cdiv(N, 8), N, most);
        const SlopeJob job{dy, none ? dy : saved_of(p->preact), p->activation, M, N, made, ldd, part, (unsigned)parts, (unsigned)(parts * cdiv(N, 256)), most, mosts, factor};
        slope_kernel<T><<<job.blocks + (stage.count ? stage.blocks() : 0), 256, 0, st>>>(job, stage.jobs[0], stage.jobs[1]);
        LAUNCHED("linear_backward");
    } else if (!count) TRY(stage.launch<T>(st), "linear_backward");
    JoinJob join_x = {}, join_w = {};
    if (p->dx && p->dw) {
        const int64_t chunks[2] = {chunks_of<T>(N), chunks_of<T>(M)};
        const Pair both = pair_of({M, (int64_t)N}, {(int64_t)K, (int64_t)K}, chunks, sizeof(T) == 4);
        const ProductArgs ax = product_args<T>(d, w, M, K, N, chunks[0], Shape{both.tile, both.splits[0]}, to_dx, ws, &join_x);
        const ProductArgs aw = product_args<T>(d, x, N, K, M, chunks[1], Shape{both.tile, both.splits[1]}, to_dw, ws, &join_w);
        ws.tile = both.tile;
        ws.parts[0] = ax.splits;
        ws.parts[1] = aw.splits;
        if (!count) TRY((both.tile == 256 ? launch_pair<T, 256>(ax, aw, st) : launch_pair<T, 128>(ax, aw, st)), "linear_backward: dx and dw");
    } else if (p->dx) TRY((product<T, false, true>(st, d, w, M, K, N, to_dx, ws, &join_x, count)), "linear_backward: dx");
    else if (p->dw) TRY((product<T, true, true>(st, d, x, N, K, M, to_dw, ws, &join_w, count)), "linear_backward: dw");
    if (!count) TRY(joins<T>(st, part ? ColumnJob{part, (int)parts, N, p->dbias, (unsigned)cdiv(N, 8)} : ColumnJob{}, join_x, join_w), "linear_backward");
    return CCSM_OK;
}

// Rows of a call are taken in ranges of at most 2^30 items (a lane's work), so that an item's number fits 31 bits
constexpr int64_t kMostItems = (int64_t)1 << 30;
template <typename F>
void in_ranges(int64_t rows, int64_t per_row, F launch) {
    const int64_t step = kMostItems / per_row > 0 ? kMostItems / per_row : 1;
    for (int64_t r = 0; r < rows; r += step) launch(r, rows - r < step ? rows - r : step);
}

struct SortPlan { int bits, passes, digit, per_lane, piece, lanes, groups; int64_t blocks, sums; };
SortPlan sort_plan(int type, int64_t tokens, int64_t rows, int width) {
    SortPlan s;
    s.bits = 1;
    while (((int64_t)1 << s.bits) < rows + 1) ++s.bits;          // ids 0 .. rows (rows = no token)
    s.passes = (s.bits + 7) / 8;
    s.digit = (s.bits + s.passes - 1) / s.passes;
    s.per_lane = tokens <= 131072 ? 4 : 16;                      // 1024 tokens a workgroup up to kFewBlocks workgroups (19 -> 6 us a pass at 65536), then 4096
    s.blocks = cdiv(tokens, 256 * s.per_lane);
    const int64_t all = cdiv(width, 16 / (int64_t)size_of(type));
    s.piece = tokens / kLongPiece * all >= 65536 ? kLongPiece : kShortPiece;      // a wave for each SIMD at least
    s.lanes = (int)(all < 256 ? all : 256);
    s.groups = 256 / s.lanes;
    s.sums = cdiv(tokens, (int64_t)s.piece * s.groups);
    return s;
}
struct EmbedScratch { unsigned *keys[2], *at[2], *counts, *list, *marks; int64_t mark_words; float* part; int64_t part_ld; };
EmbedScratch embed_scratch(Scratch& ws, const SortPlan& s, int64_t tokens, int64_t rows, int width) {
    EmbedScratch e;
    for (int k = 0; k < 2; ++k) {
        e.keys[k] = ws.take<unsigned>(tokens);
        e.at[k] = ws.take<unsigned>(tokens);
    }
    e.counts = ws.take<unsigned>((size_t)s.blocks << s.digit);
    e.list = ws.take<unsigned>(1 + s.sums);
    e.mark_words = cdiv(rows, 4);
    e.marks = ws.take<unsigned>(e.mark_words);
    e.part_ld = (int64_t)up(width, 8);
    e.part = ws.take<float>((size_t)2 * s.sums * e.part_ld);
    return e;
}
// Tables of few rows, for their own two kernels.  Eight tokens of a slice at least, and enough to be worth a table's way through memory; four workgroups
// for each CU at most
bool few_rows(int64_t rows, int width) { return rows <= kFewIds && rows * width <= kFewValues; }
struct FewPlan { int lanes, slices, per; int64_t blocks, part_ld; unsigned columns; };
FewPlan few_plan(int64_t tokens, int64_t rows, int width) {
    FewPlan f;
    const int64_t all = cdiv(width, 4);
    f.columns = (unsigned)cdiv(all, 256);
    f.lanes = (int)(all < 256 ? all : 256);
    f.slices = 256 / f.lanes;
    const int64_t most = f.columns < 1024 ? 1024 / f.columns : 1, even = cdiv(tokens, f.slices * most), worth = cdiv(4 * rows, f.slices);
    f.per = (int)up((size_t)(even > worth ? even : worth), 8);
    f.blocks = cdiv(tokens, (int64_t)f.slices * f.per);
    f.part_ld = (int64_t)up(width, 4);
    return f;
}
template <typename T>
void few_sums(hipStream_t st, const FewPlan& f, const void* ids, int id_type, int64_t tokens, int rows, int width, const void* dy, int64_t lddy, float scale, void* dt,
              int64_t ldt, float* part) {
    few_sum_kernel<T><<<dim3((unsigned)f.blocks, f.columns), 256, (size_t)rows * 257 * 16, st>>>(ids, id_type, tokens, rows, f.per, Div::by((unsigned)f.lanes), f.slices, width,
                                                                                        (const T*)dy, lddy, part, f.part_ld);
    few_join_kernel<T><<<(unsigned)cdiv(rows * f.part_ld, 64), 256, 0, st>>>(part, f.part_ld, (int)f.blocks, rows, width, scale, (T*)dt, ldt);
}
Held held_ids(const void* ids, int id_type, int64_t tokens) { return held(ids, tokens, 1, tokens, id_type == CCSM_ID_U8 ? 1 : id_type == CCSM_ID_I32 ? 4 : 8); }
ccsm_status check_embedding(int type, int id_type, int64_t tokens, const void* ids, int64_t rows, int width) {
    REFUSE(!good_type(type), "embedding: unknown type");
    REFUSE(id_type < CCSM_ID_U8 || id_type > CCSM_ID_I64, "embedding: unknown type of ids");
    REFUSE(tokens < 0 || tokens > kMostRows || rows <= 0 || rows > kMostRows || width <= 0 || width > kMostCols, "embedding: sizes out of range");
    REFUSE(tokens * width > ((int64_t)1 << 37), "embedding: more values than a GPU holds");
    REFUSE(tokens && !ids, "embedding: ids must be non-NULL");
    REFUSE(off_by(ids, id_type == CCSM_ID_U8 ? 1 : id_type == CCSM_ID_I32 ? 4 : 8), "embedding: ids are not aligned to their elements");
    return CCSM_OK;
}
template <int Q>
void sort_pass(hipStream_t st, const SortPlan& s, const EmbedScratch& b, const void* ids, int id_type, int64_t tokens, int64_t rows, int pass, int k) {
    const unsigned *keys = pass ? b.keys[k] : nullptr, *at = pass ? b.at[k] : nullptr;
    const int bins = 1 << s.digit;
    sort_count_kernel<Q><<<(unsigned)s.blocks, 256, 0, st>>>(ids, id_type, keys, tokens, rows, pass * s.digit, bins, b.counts, pass ? nullptr : b.marks, b.mark_words, b.list);
    if (s.blocks > kFewBlocks) sort_scan_kernel<<<1, 1024, 0, st>>>(b.counts, s.blocks << s.digit);
    sort_scatter_kernel<Q><<<(unsigned)s.blocks, 256, 0, st>>>(ids, id_type, keys, at, tokens, rows, pass * s.digit, bins, b.counts, b.keys[k ^ 1], b.at[k ^ 1],
                                                               pass + 1 == s.passes ? (uint8_t*)b.marks : nullptr);
}
ccsm_status check_room(size_t need, const void* workspace, size_t have) {
    if (need && (!workspace || have < need)) return fail(CCSM_ERR_CAPACITY, "the workspace is too small");
    REFUSE(need && off_by(workspace, 256), "the workspace is not 256-byte aligned");
    return CCSM_OK;
}

}  // namespace

extern "C" {

const char* ccsm_train_ops_last_error(void) { return g_err.c_str(); }

size_t ccsm_train_linear_workspace(const ccsm_linear* p) {
    if (check_linear(p) != CCSM_OK || p->rows == 0) return 0;
    Scratch ws;
    TYPED(p->type, (void)linear_forward<T>(p, ws, nullptr, true));
    return ws.used;
}
ccsm_status ccsm_train_linear_forward(int device, const ccsm_linear* p, void* workspace, size_t workspace_bytes, void* stream) {
    ccsm_status e = check_linear(p);
    if (e != CCSM_OK || p->rows == 0) return e;
    if ((e = check_room(ccsm_train_linear_workspace(p), workspace, workspace_bytes)) != CCSM_OK || (e = apart(p)) != CCSM_OK) return e;
    ON_DEVICE(device);
    Scratch ws;
    ws.base = (char*)workspace;
    TYPED(p->type, return linear_forward<T>(p, ws, (hipStream_t)stream, false));
}

size_t ccsm_train_linear_backward_workspace(const ccsm_linear_grad* p) {
    if (check_grad(p) != CCSM_OK) return 0;
    Scratch ws;
    TYPED(p->type, (void)linear_backward<T>(p, ws, nullptr, true));
    return ws.used;
}
ccsm_status ccsm_train_linear_backward(int device, const ccsm_linear_grad* p, void* workspace, size_t workspace_bytes, void* stream) {
    ccsm_status e = check_grad(p);
    if (e != CCSM_OK) return e;
    if ((e = check_room(ccsm_train_linear_backward_workspace(p), workspace, workspace_bytes)) != CCSM_OK || (e = apart(p)) != CCSM_OK) return e;
    ON_DEVICE(device);
    Scratch ws;
    ws.base = (char*)workspace;
    TYPED(p->type, return linear_backward<T>(p, ws, (hipStream_t)stream, false));
}

static void way_of(const Scratch& ws, int32_t* way) { way[0] = ws.tile; way[1] = ws.parts[0]; way[2] = ws.parts[1]; way[3] = ws.staged; }
ccsm_status ccsm_train_linear_way(const ccsm_linear* p, int32_t* way) {
    const ccsm_status e = check_linear(p);
    if (e != CCSM_OK) return e;
    REFUSE(!way, "linear_way: NULL argument");
    Scratch ws;
    if (p->rows) TYPED(p->type, (void)linear_forward<T>(p, ws, nullptr, true));
    way_of(ws, way);
    return CCSM_OK;
}
ccsm_status ccsm_train_linear_backward_way(const ccsm_linear_grad* p, int32_t* way) {
    const ccsm_status e = check_grad(p);
    if (e != CCSM_OK) return e;
    REFUSE(!way, "linear_backward_way: NULL argument");
    Scratch ws;
    TYPED(p->type, (void)linear_backward<T>(p, ws, nullptr, true));
    way_of(ws, way);
    return CCSM_OK;
}

ccsm_status ccsm_train_embedding_forward(int device, int type, int id_type, int64_t tokens, const void* ids, int64_t rows, int32_t width,
                                         const void* table, int64_t ldt, float scale, void* y, int64_t ldy, void* stream) {
    ccsm_status e = check_embedding(type, id_type, tokens, ids, rows, width);
    if (e != CCSM_OK || tokens == 0) return e;
    REFUSE(!table || !y || ldt < width || ldy < width, "embedding: table and y must be non-NULL, their strides at least the width");
    REFUSE(off_by(table, size_of(type)) || off_by(y, size_of(type)), "embedding: a pointer is not aligned to its elements");
    const Held out[] = {held(y, ldy, tokens, width, size_of(type))}, in[] = {held(table, ldt, rows, width, size_of(type)), held_ids(ids, id_type, tokens)};
    REFUSE(shared(out, in), "embedding: y shares memory with another tensor");
    ON_DEVICE(device);
    hipStream_t st = (hipStream_t)stream;
    TYPED(type, constexpr int P = 16 / sizeof(T); const int64_t pieces = cdiv(width, P);
          in_ranges(tokens, pieces, [&](int64_t t, int64_t n) {
              const char* i = (const char*)ids + t * (id_type == CCSM_ID_U8 ? 1 : id_type == CCSM_ID_I32 ? 4 : 8);
              lookup_kernel<T, P><<<(unsigned)cdiv(n * pieces, 1024), 256, 0, st>>>(i, id_type, (unsigned)(n * pieces), Div::by((unsigned)pieces), rows, width, (const T*)table, ldt,
                                                                                 scale, (T*)y + t * ldy, ldy);
          }));
    LAUNCHED("embedding_forward");
    return CCSM_OK;
}

size_t ccsm_train_embedding_backward_workspace(int type, int64_t tokens, int64_t rows, int32_t width) {
    if (!good_type(type) || tokens <= 0 || tokens > kMostRows || rows <= 0 || rows > kMostRows || width <= 0 || width > kMostCols) return 0;
    Scratch ws;
    if (few_rows(rows, width)) {
        const FewPlan f = few_plan(tokens, rows, width);
        ws.take<float>((size_t)f.blocks * rows * f.part_ld);
    } else (void)embed_scratch(ws, sort_plan(type, tokens, rows, width), tokens, rows, width);
    return ws.used;
}
ccsm_status ccsm_train_embedding_backward(int device, int type, int id_type, int64_t tokens, const void* ids, int64_t rows, int32_t width,
                                          const void* dy, int64_t lddy, float scale, void* dtable, int64_t ldt, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    ccsm_status e = check_embedding(type, id_type, tokens, ids, rows, width);
    if (e != CCSM_OK) return e;
    REFUSE(!dtable || ldt < width || (tokens && (!dy || lddy < width)), "embedding: dy and dtable must be non-NULL, their strides at least the width");
    REFUSE(off_by(dtable, size_of(type)) || off_by(dy, size_of(type)), "embedding: a pointer is not aligned to its elements");
    if ((e = check_room(ccsm_train_embedding_backward_workspace(type, tokens, rows, width), workspace, workspace_bytes)) != CCSM_OK) return e;
    const Held out[] = {held(dtable, ldt, rows, width, size_of(type))}, in[] = {held(dy, lddy, tokens, width, size_of(type)), held_ids(ids, id_type, tokens)};
    REFUSE(shared(out, in), "embedding: dtable shares memory with another tensor");
    ON_DEVICE(device);
    hipStream_t st = (hipStream_t)stream;
    if (tokens == 0) {
        TYPED(type, fill_zero_kernel<T><<<grid_of(cdiv(rows * width, 256), 4096), 256, 0, st>>>((T*)dtable, ldt, rows, width));
        LAUNCHED("embedding_backward");
        return CCSM_OK;
    }
    Scratch ws;
    ws.base = (char*)workspace;
    if (few_rows(rows, width)) {
        const FewPlan f = few_plan(tokens, rows, width);
        float* part = ws.take<float>((size_t)f.blocks * rows * f.part_ld);
        TYPED(type, few_sums<T>(st, f, ids, id_type, tokens, (int)rows, width, dy, lddy, scale, dtable, ldt, part));
        LAUNCHED("embedding_backward");
        return CCSM_OK;
    }
    const SortPlan s = sort_plan(type, tokens, rows, width);
    const EmbedScratch b = embed_scratch(ws, s, tokens, rows, width);
    int k = 0;
    for (int pass = 0; pass < s.passes; ++pass, k ^= 1) {
        if (s.per_lane == 4) sort_pass<4>(st, s, b, ids, id_type, tokens, rows, pass, k);
        else sort_pass<16>(st, s, b, ids, id_type, tokens, rows, pass, k);
    }
    TYPED(type, constexpr int P = 16 / sizeof(T); const int chunks = (int)cdiv(width, 256);
          auto* f = s.piece == kLongPiece ? &piece_sum_kernel<T, P, kLongPiece> : &piece_sum_kernel<T, P, kShortPiece>;
          f<<<dim3((unsigned)s.sums + grid_of(cdiv(rows, 8), 4096), (unsigned)cdiv(width, 256 * P)), 256, 0, st>>>(
              b.keys[k], b.at[k], tokens, rows, (unsigned)s.sums, s.groups, Div::by((unsigned)s.lanes), width, (const T*)dy, lddy, scale, (T*)dtable, ldt, b.part, b.part_ld,
              (const uint8_t*)b.marks, b.list);
          if (s.sums > 1) join_kernel<T><<<grid_of(s.sums * chunks, 1024), 256, 0, st>>>(b.keys[k], tokens, s.piece * s.groups, width, scale, (T*)dtable, ldt, b.part, b.part_ld,
                                                                                         b.list, chunks));
    LAUNCHED("embedding_backward");
    return CCSM_OK;
}

ccsm_status ccsm_train_act8_pack(int device, int type, int code, int64_t rows, int32_t width, const void* x, int64_t ldx, void* codes,
                                 int64_t ldc, uint8_t* scales, int64_t lds, void* stream) {
    REFUSE(!good_type(type), "act8_pack: unknown type");
    REFUSE(code != CCSM_CODE_INT8 && code != CCSM_CODE_E4M3, "act8_pack: unknown code");
    REFUSE(rows < 0 || rows > kMostRows || width <= 0 || width > kMostCols, "act8_pack: sizes out of range");
    if (rows == 0) return CCSM_OK;
    REFUSE(!x || ldx < width || off_by(x, size_of(type)), "act8_pack: x must be non-NULL and aligned to its elements, its stride at least the width");
    ccsm_status e = check_saved(ccsm_saved{codes, ldc, code, scales, lds}, type, width, "act8_pack: codes must be non-NULL");
    if (e != CCSM_OK) return e;
    const ccsm_saved s{codes, ldc, code, scales, lds};
    const Held out[] = {held(s, rows, width, type), held_scales(s, rows, width)}, in[] = {held(x, ldx, rows, width, size_of(type))};
    REFUSE(shared(out, in), "act8_pack: codes or scales share memory with another tensor");
    ON_DEVICE(device);
    const int64_t per = 2 * cdiv(width, 32);
    TYPED(type, in_ranges(rows, per, [&](int64_t r, int64_t n) {
              auto* f = code == CCSM_CODE_INT8 ? &act8_pack_kernel<T, kCodeInt8> : &act8_pack_kernel<T, kCodeE4m3>;
              f<<<(unsigned)cdiv(n * per, 256), 256, 0, (hipStream_t)stream>>>((const T*)x + r * ldx, ldx, (unsigned)(n * per), Div::by((unsigned)per), width, (uint8_t*)codes + r * ldc,
                                                                              ldc, scales + r * lds, lds);
          }));
    LAUNCHED("act8_pack");
    return CCSM_OK;
}
ccsm_status ccsm_train_act8_unpack(int device, int type, int64_t rows, int32_t width, const ccsm_saved* s, void* y, int64_t ldy, void* stream) {
    REFUSE(!s, "act8_unpack: NULL argument");
    REFUSE(!good_type(type), "act8_unpack: unknown type");
    REFUSE(s->code != CCSM_CODE_INT8 && s->code != CCSM_CODE_E4M3, "act8_unpack: unknown code");
    REFUSE(rows < 0 || rows > kMostRows || width <= 0 || width > kMostCols, "act8_unpack: sizes out of range");
    if (rows == 0) return CCSM_OK;
    ccsm_status e = check_saved(*s, type, width, "act8_unpack: codes must be non-NULL");
    if (e != CCSM_OK) return e;
    REFUSE(!y || ldy < width || off_by(y, size_of(type)), "act8_unpack: y must be non-NULL and aligned to its elements, its stride at least the width");
    const Held out[] = {held(y, ldy, rows, width, size_of(type))}, in[] = {held(*s, rows, width, type), held_scales(*s, rows, width)};
    REFUSE(shared(out, in), "act8_unpack: y shares memory with another tensor");
    ON_DEVICE(device);
    const int64_t per = cdiv(width, 16);
    TYPED(type, in_ranges(rows, per, [&](int64_t r, int64_t n) {
              auto* f = s->code == CCSM_CODE_INT8 ? &act8_unpack_kernel<T, kCodeInt8> : &act8_unpack_kernel<T, kCodeE4m3>;
              f<<<(unsigned)cdiv(n * per, 256), 256, 0, (hipStream_t)stream>>>((const uint8_t*)s->data + r * s->ld, s->ld, s->scales + r * s->lds, s->lds, (unsigned)(n * per),
                                                                              Div::by((unsigned)per), width, (T*)y + r * ldy, ldy);
          }));
    LAUNCHED("act8_unpack");
    return CCSM_OK;
}

}  // extern "C"
