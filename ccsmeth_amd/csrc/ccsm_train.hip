// libccsm_train: the attbigru2s training step (forward with saved activations, backward, Adam) for gfx950, fp32.
// C-ABI in include/ccsm_train.h.  Dense products: the library's three-pass split-fp16 MFMA kernel (ccsm_train_gemm.hip; no BLAS library
// is linked - rounds 1-3 called rocBLAS SGEMM here, an A/B build still can: GemmCtx below); the recurrent part, gates, attention, loss,
// embedding scatter, dropout and the optimizer are the kernels below and in ccsm_train_seq.hip.  Activations are time-major: (T, M, features) with M = 2N rows
// (strand 1 rows first), so that a timestep of a direction is one contiguous (M, H) block and both strands share every product.
//
// Reference equations: ModelAttRNN.forward (models.py:89-150), torch.nn.GRU cell (gate order r, z, n), Attention
// (utils/attention.py:48-70), CrossEntropyLoss(weight) + clip_grad_norm_ + Adam (train_multigpu.py:212-216, 283-312).
#include <hip/hip_runtime.h>
#ifdef CCSM_TRAIN_WITH_ROCBLAS          // A/B build only (tools: hipcc -DCCSM_TRAIN_WITH_ROCBLAS ... -lrocblas): the product library links no BLAS
#include <rocblas/rocblas.h>
#else
typedef void* rocblas_handle;
typedef int rocblas_status;
constexpr int rocblas_status_success = 0, rocblas_status_internal_error = 6;
#endif

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>

#include "../../include/ccsm_train.h"
#include "../../include/ccsm_train_ops.h"
#include "ccsm_train_gemm.hip"

// Where a matrix product of the step runs.  The product library: ccsm_train_gemm.hip, the library's three-pass split-fp16 MFMA kernel, for
// every product ("own": 5.35 / 12.4 ms per step at batch 512 / 2048 against 5.72 / 13.8 with rocBLAS SGEMM, profiles/r04_h_train_gemm.log).
// A -DCCSM_TRAIN_WITH_ROCBLAS build (A/B runs) also holds the rounds 1-3 rocBLAS calls: CCSM_TRAIN_GEMM = own | rocblas | mixed (mixed: the
// library's kernel for row-major A, rocBLAS for the A^T B weight gradients), read at ccsm_train_create.
struct GemmCtx { hipStream_t st; unsigned* amax; rocblas_handle rb; int mode; };      // mode: 0 mixed, 1 own, 2 rocblas
typedef GemmCtx* blas_t;

namespace {

constexpr int T = 21, H = 256, G = 3 * H, H2 = 2 * H, NE = 8, F0 = 11, L = CCSM_LAYERS, NC = 2, NV = 5;

thread_local std::string g_err;
ccsm_status fail(ccsm_status s, const std::string& m) { g_err = m; return s; }
#define HIPCHK(x)                                                                                        \
    do {                                                                                                 \
        hipError_t e_ = (x);                                                                             \
        if (e_ != hipSuccess) return fail(CCSM_ERR_HIP, std::string(#x) + ": " + hipGetErrorString(e_)); \
    } while (0)
#define BLASCHK(x)                                                                                              \
    do {                                                                                                        \
        rocblas_status s_ = (x);                                                                                \
        if (s_ != rocblas_status_success) return fail(CCSM_ERR_HIP, std::string(#x) + ": rocblas status " + std::to_string((int)s_)); \
    } while (0)

// ---- flat parameter order ------------------------------------------------------------------------------------------
struct Offsets {
    int64_t embed, w_ih[L][2], w_hh[L][2], b_ih[L][2], b_hh[L][2], wa, ua, va, fcw, fcb, total;
    int64_t list[31];
    Offsets() {
        int64_t o = 0;
        int k = 0;
        auto take = [&](int64_t n) { int64_t r = o; list[k++] = o; o += n; return r; };
        embed = take(NV * NE);
        for (int l = 0; l < L; ++l)
            for (int d = 0; d < 2; ++d) {
                w_ih[l][d] = take((int64_t)G * (l == 0 ? F0 : H2));
                w_hh[l][d] = take((int64_t)G * H);
                b_ih[l][d] = take(G);
                b_hh[l][d] = take(G);
            }
        wa = take((int64_t)H * H2);
        ua = take((int64_t)H * H2);
        va = take(H);
        fcw = take((int64_t)NC * 2 * H2);
        fcb = take(NC);
        total = o;
        list[k] = o;
    }
};
const Offsets kOff;

// ---- small device helpers -------------------------------------------------------------------------------------------
__device__ __forceinline__ float sigmoidf_(float x) { return 1.0f / (1.0f + __expf(-x)); }
__device__ __forceinline__ uint64_t mix64(uint64_t z) {
    z += 0x9e3779b97f4a7c15ull;
    z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
    z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
    return z ^ (z >> 31);
}
__device__ __forceinline__ float uniform01(uint64_t seed, uint64_t stream, uint64_t idx) {
    const uint64_t r = mix64(mix64(seed ^ (stream * 0xd1342543de82ef95ull)) + idx);
    return (float)(r >> 40) * (1.0f / 16777216.0f);
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// x0[t][m][0..7] = embed[kmer[m][t]], [8] = ipd, [9] = pw, [10] = npass          (models.py:91-106)
__global__ void build_x0_kernel(const uint8_t* kmer, const float* ipd, const float* pw, const float* npass, const float* embed,
                                float* x0, int M) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= T * M) return;
    const int t = i / M, m = i % M;
    int b = kmer[m * T + t];
    b = b > 4 ? 4 : b;
    float* o = x0 + (size_t)i * F0;
#pragma unroll
    for (int e = 0; e < NE; ++e) o[e] = embed[b * NE + e];
    o[8] = ipd[m * T + t];
    o[9] = pw[m * T + t];
    o[10] = npass[m * T + t];
}

// h0 from the counter-based generator (DEVICE_RNG): N(0,1) by Box-Muller.  The counter is keyed by the GLOBAL site index
// (offset + site), then (layer-direction, strand, unit): a site draws the same states wherever it stands in a batch, and batches whose
// site ranges [offset, offset + N) do not overlap share no counter.  h0 layout: [2L][2N rows: strand-major][H].
__global__ void h0_rng_kernel(float* h0, int64_t n, int n_sites, uint64_t seed, uint64_t offset) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int h = (int)(i % H);
    const int64_t row = (i / H) % (2 * (int64_t)n_sites), k = i / ((int64_t)H * 2 * n_sites);
    const uint64_t site = offset + (uint64_t)(row % n_sites), strand = (uint64_t)(row / n_sites);
    const uint64_t c = 2 * ((((site * (2 * L) + (uint64_t)k) * 2 + strand) * H) + (uint64_t)h);
    const float u1 = fmaxf(uniform01(seed, 0x68300, c), 1e-7f), u2 = uniform01(seed, 0x68300, c + 1);
    h0[i] = sqrtf(-2.0f * __logf(u1)) * __cosf(6.283185307179586f * u2);
}

// What changes from step to step lives in device memory, so that a captured graph of the step can be replayed unchanged.
struct Ctl {
    uint64_t seed;       // dropout masks of this step
    float pos_weight;    // CrossEntropyLoss weight of class 1
    float wsum;          // sum of the batch's class weights (the loss is a weighted mean)
};

// y = x * mask / keep  (inverted dropout, mask from (seed, stream, element index))
__global__ void dropout_kernel(const float* x, float* y, int64_t n, float rate, const Ctl* ctl, uint64_t stream) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    y[i] = uniform01(ctl->seed, stream, (uint64_t)i) >= rate ? x[i] * (1.0f / (1.0f - rate)) : 0.0f;
}

// one GRU step of one direction: gi (M,G) = x_t W_ih^T (no bias yet), gh (M,G) = h_{t-1} W_hh^T (no bias yet)
//   r = s(gi_r + b_ir + gh_r + b_hr); z likewise; hp = gh_n + b_hn; n = tanh(gi_n + b_in + r * hp); h = (1 - z) n + z h_{t-1}
__global__ void gru_gate_fwd_kernel(const float* gi, const float* gh, const float* b_ih, const float* b_hh, const float* hprev,
                                    int ld_hprev, float* out, float* R, float* Z, float* Nn, float* HP, int M, int save) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= M * H) return;
    const int m = i / H, j = i % H;
    const float* a = gi + (size_t)m * G;
    const float* b = gh + (size_t)m * G;
    const float r = sigmoidf_(a[j] + b_ih[j] + b[j] + b_hh[j]);
    const float z = sigmoidf_(a[H + j] + b_ih[H + j] + b[H + j] + b_hh[H + j]);
    const float hp = b[2 * H + j] + b_hh[2 * H + j];
    const float n = tanhf(a[2 * H + j] + b_ih[2 * H + j] + r * hp);
    const float h = (1.0f - z) * n + z * hprev[(size_t)m * ld_hprev + j];
    out[(size_t)m * H2 + j] = h;
    if (save) { R[i] = r; Z[i] = z; Nn[i] = n; HP[i] = hp; }
}

// backward of that step.  Writes dgi = [dr, dz, dn], dgh = [dr, dz, dn * r], carry = dh * z; the caller then computes the three
// per-gate products dgh[gate] W_hh[gate] into cpart (one batched GEMM: three times the workgroups of a single K = 768 product,
// which left three quarters of the CUs idle at 1024 rows), and the next step's launch adds them up.
__global__ void gru_gate_bwd_kernel(const float* dout, float* carry, const float* cpart, const float* R, const float* Z, const float* Nn,
                                    const float* HP, const float* hprev, int ld_hprev, float* dgi, float* dgh, int M) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= M * H) return;
    const int m = i / H, j = i % H;
    // dh_t = d out_t + (dh_{t+1} z_{t+1}) + the three per-gate products dgh_{t+1}[gate] W_hh[gate] of the previous launch
    const size_t ps = (size_t)M * H;
    const float dh = dout[(size_t)m * H2 + j] + carry[i] + cpart[i] + cpart[ps + i] + cpart[2 * ps + i];
    const float r = R[i], z = Z[i], n = Nn[i], hp = HP[i];
    const float dn = dh * (1.0f - z) * (1.0f - n * n);
    const float dz = dh * (hprev[(size_t)m * ld_hprev + j] - n) * z * (1.0f - z);
    const float dr = dn * hp * r * (1.0f - r);
    float* a = dgi + (size_t)m * G;
    float* b = dgh + (size_t)m * G;
    a[j] = dr; a[H + j] = dz; a[2 * H + j] = dn;
    b[j] = dr; b[H + j] = dz; b[2 * H + j] = dn * r;
    carry[i] = dh * z;
}

// h_n = [forward final state = out[T-1][:, :H] | backward final state = out[0][:, H:]]            (models.py:135-137)
__global__ void gather_hn_kernel(const float* out2, float* hn, int M) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= M * H2) return;
    const int m = i / H2, k = i % H2;
    hn[i] = k < H ? out2[((size_t)(T - 1) * M + m) * H2 + k] : out2[(size_t)m * H2 + k];
}
__global__ void scatter_dhn_kernel(const float* dhn, float* dout2, int M) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= M * H2) return;
    const int m = i / H2, k = i % H2;
    float* p = k < H ? dout2 + ((size_t)(T - 1) * M + m) * H2 + k : dout2 + (size_t)m * H2 + k;
    *p += dhn[i];
}

// S[t][m][:] = tanh(q[m] + K[t][m]) in place of K; e[t][m] = va . S                (attention.py:69-70); one wave per (t, m)
__global__ void att_score_kernel(float* KS, const float* q, const float* va, float* e, int M) {
    const int row = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= T * M) return;
    const int m = row % M;
    float acc = 0.f;
#pragma unroll
    for (int c = 0; c < H / 64; ++c) {
        const int j = lane + 64 * c;
        const float s = tanhf(q[(size_t)m * H + j] + KS[(size_t)row * H + j]);
        KS[(size_t)row * H + j] = s;
        acc += va[j] * s;
    }
    acc = wave_sum(acc);
    if (lane == 0) e[row] = acc;
}
// a = softmax over t, per row m                                                  (attention.py:55)
__global__ void att_softmax_kernel(const float* e, float* a, int M) {
    const int m = blockIdx.x * blockDim.x + threadIdx.x;
    if (m >= M) return;
    float mx = -INFINITY;
    for (int t = 0; t < T; ++t) mx = fmaxf(mx, e[(size_t)t * M + m]);
    float den = 0.f;
    for (int t = 0; t < T; ++t) den += __expf(e[(size_t)t * M + m] - mx);
    for (int t = 0; t < T; ++t) a[(size_t)t * M + m] = __expf(e[(size_t)t * M + m] - mx) / den;
}
// c[m][k] = sum_t a[t][m] out2[t][m][k]                                          (attention.py:57-58)
__global__ void att_context_kernel(const float* a, const float* out2, float* c, int M) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= M * H2) return;
    const int m = i / H2;
    float acc = 0.f;
    for (int t = 0; t < T; ++t) acc += a[(size_t)t * M + m] * out2[(size_t)t * M * H2 + i];
    c[i] = acc;
}
// da[t][m] = dc[m] . out2[t][m]; one wave per (t, m)
__global__ void att_dalpha_kernel(const float* dc, const float* out2, float* da, int M) {
    const int row = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= T * M) return;
    const int m = row % M;
    float acc = 0.f;
#pragma unroll
    for (int c = 0; c < H2 / 64; ++c) acc += dc[(size_t)m * H2 + lane + 64 * c] * out2[(size_t)row * H2 + lane + 64 * c];
    acc = wave_sum(acc);
    if (lane == 0) da[row] = acc;
}
// de = a * (da - sum_t a da)   (softmax backward), in place of da
__global__ void att_dscore_kernel(const float* a, float* da, int M) {
    const int m = blockIdx.x * blockDim.x + threadIdx.x;
    if (m >= M) return;
    float s = 0.f;
    for (int t = 0; t < T; ++t) s += a[(size_t)t * M + m] * da[(size_t)t * M + m];
    for (int t = 0; t < T; ++t) da[(size_t)t * M + m] = a[(size_t)t * M + m] * (da[(size_t)t * M + m] - s);
}
// dSpre[t][m][j] = de[t][m] va[j] (1 - S^2) in place of S; dva_part[block][j] = sum over the block's 64 rows of de S (added up in block
// order by sum_partials_kernel: no float atomics anywhere in the step since round 4); dout2[t][m][k] = a[t][m] dc[m][k]
__global__ void att_dpre_kernel(float* S, const float* de, const float* va, float* dva_part, int rows) {
    const int j = threadIdx.x;                       // blockDim.x == H
    const int r0 = blockIdx.x * 64, r1 = min(rows, r0 + 64);
    float acc = 0.f;
    const float v = va[j];
    for (int r = r0; r < r1; ++r) {
        const float s = S[(size_t)r * H + j], d = de[r];
        acc += d * s;
        S[(size_t)r * H + j] = d * v * (1.0f - s * s);
    }
    dva_part[(size_t)blockIdx.x * H + j] = acc;
}
__global__ void att_dq_kernel(const float* dS, float* dq, int M) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= M * H) return;
    float acc = 0.f;
    for (int t = 0; t < T; ++t) acc += dS[(size_t)t * M * H + i];
    dq[i] = acc;
}
__global__ void att_dout_init_kernel(const float* a, const float* dc, float* dout2, int M) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (int64_t)T * M * H2) return;
    const int64_t row = i / H2;
    const int k = (int)(i % H2);
    const int m = (int)(row % M);
    dout2[i] = a[row] * dc[(size_t)m * H2 + k];
}

// feat[n] = [c[n] | c[N + n]] (dropout1 applied when rate > 0); logits = feat fc^T + b; p = softmax; weighted CE
//   loss_sum += w_y * -log p_y ; dlogits[n][c] = w_y (p_c - [c == y]) / wsum            (models.py:145-150, train_multigpu.py:212-214)
__global__ void fc_loss_kernel(const float* c, const float* fcw, const float* fcb, const int32_t* labels, const Ctl* ctl, float rate,
                               float* feat, float* logits, float* dlogits, float* loss_site, int N) {
    const int n = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (n >= N) return;
    const uint64_t seed = ctl->seed;
    const float pos_weight = ctl->pos_weight, wsum = ctl->wsum;
    float a0 = 0.f, a1 = 0.f;
    for (int k = lane; k < 2 * H2; k += 64) {
        float v = k < H2 ? c[(size_t)n * H2 + k] : c[(size_t)(N + n) * H2 + (k - H2)];
        if (rate > 0.f) v = uniform01(seed, 0xfc1, (uint64_t)n * 2 * H2 + k) >= rate ? v * (1.0f / (1.0f - rate)) : 0.0f;
        feat[(size_t)n * 2 * H2 + k] = v;
        a0 += v * fcw[k];
        a1 += v * fcw[2 * H2 + k];
    }
    a0 = wave_sum(a0) + fcb[0];
    a1 = wave_sum(a1) + fcb[1];
    if (lane == 0) {
        logits[2 * n] = a0;
        logits[2 * n + 1] = a1;
        if (labels != nullptr) {
            const float mx = fmaxf(a0, a1);
            const float lse = mx + __logf(__expf(a0 - mx) + __expf(a1 - mx));
            const int y = labels[n] != 0;
            const float w = y ? pos_weight : 1.0f;
            loss_site[n] = w * (lse - (y ? a1 : a0));         // added up in site order by sum_fixed_kernel
            if (dlogits != nullptr) {
                dlogits[2 * n] = w * (__expf(a0 - lse) - (y ? 0.f : 1.f)) / wsum;
                dlogits[2 * n + 1] = w * (__expf(a1 - lse) - (y ? 1.f : 0.f)) / wsum;
            }
        }
    }
}
// dc[m][k] from dlogits fc_w (through dropout1), db_fc = column sums of dlogits
__global__ void fc_bwd_kernel(const float* dlogits, const float* fcw, float rate, const Ctl* ctl, float* dc, float* dfcb, int N) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    const uint64_t seed = ctl->seed;
    if (i < NC) {
        float s = 0.f;
        for (int n = 0; n < N; ++n) s += dlogits[2 * n + i];
        dfcb[i] = s;
    }
    if (i >= N * 2 * H2) return;
    const int n = i / (2 * H2), k = i % (2 * H2);
    float g = dlogits[2 * n] * fcw[k] + dlogits[2 * n + 1] * fcw[2 * H2 + k];
    if (rate > 0.f) g = uniform01(seed, 0xfc1, (uint64_t)i) >= rate ? g * (1.0f / (1.0f - rate)) : 0.0f;
    const int m = k < H2 ? n : N + n;
    dc[(size_t)m * H2 + (k % H2)] = g;
}
// dembed_part[block][code][e] = sum over the block's 256 (t, m) entries with kmer[m][t] == code of dx0[t][m][e], each bin added up in
// entry order by one thread (fixed order); sum_partials_kernel adds the blocks
__global__ void embed_bwd_kernel(const float* dx0, const uint8_t* kmer, float* dembed_part, int M) {
    __shared__ float val[256][NE];
    __shared__ int code[256];
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    int b = -1;
    if (i < T * M) {
        const int t = i / M, m = i % M;
        b = kmer[m * T + t];
        b = b > 4 ? 4 : b;
#pragma unroll
        for (int e = 0; e < NE; ++e) val[threadIdx.x][e] = dx0[(size_t)i * F0 + e];
    }
    code[threadIdx.x] = b;
    __syncthreads();
    if (threadIdx.x < NV * NE) {
        const int bb = threadIdx.x / NE, e = threadIdx.x % NE;
        float acc = 0.f;
        for (int k = 0; k < 256; ++k)
            if (code[k] == bb) acc += val[k][e];
        dembed_part[(size_t)blockIdx.x * NV * NE + threadIdx.x] = acc;
    }
}
// part[block][c] = sum over the block's 32 rows of a[r][c]  (bias gradients: column sums of the (T*M, 768) gate-gradient blocks; the blocks
// are added up in order by sum_partials_kernel)
__global__ void colsum_kernel(const float* a, float* part, int rows, int cols) {
    const int r0 = blockIdx.x * 32, r1 = min(rows, r0 + 32);
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
        float acc = 0.f;
#pragma unroll 8
        for (int r = r0; r < r1; ++r) acc += a[(size_t)r * cols + c];
        part[(size_t)blockIdx.x * cols + c] = acc;
    }
}
// out[0] = sum of x[0 .. n) in a fixed order (one block: strided partial sums, then a tree)
__global__ void sum_fixed_kernel(const float* x, int n, float* out) {
    __shared__ float s[256];
    float acc = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) acc += x[i];
    s[threadIdx.x] = acc;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) s[threadIdx.x] += s[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[0] = s[0];
}
// out[i] = sum_k part[k][i]   (the per-timestep partial products of a weight gradient; the per-block partial sums of the reductions above)
__global__ void sum_partials_kernel(const float* part, float* out, int parts, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    float acc = 0.f;
    for (int k = 0; k < parts; ++k) acc += part[(size_t)k * n + i];
    out[i] = acc;
}
// torch.optim.Adam (no amsgrad, no weight decay): m, v moments, bias correction by step; g pre-scaled by `clip`
__global__ void adam_kernel(float* p, const float* g, float* m, float* v, int64_t n, float lr, float b1, float b2, float eps, float clip,
                            float bc1, float bc2) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const float gi = g[i] * clip;
    const float mi = b1 * m[i] + (1.0f - b1) * gi;
    const float vi = b2 * v[i] + (1.0f - b2) * gi * gi;
    m[i] = mi;
    v[i] = vi;
    p[i] -= (lr / bc1) * mi / (sqrtf(vi) / sqrtf(bc2) + eps);
}

inline dim3 blocks(int64_t n, int per = 256) { return dim3((unsigned)((n + per - 1) / per)); }

#include "ccsm_train_seq.hip"

}  // namespace

struct ccsm_trainer {
    int device = 0, max_sites = 0;
    blas_t blas = nullptr, blas1 = nullptr;            // per stream: the stream, one scale word, the rocBLAS handle, the mode
    GemmCtx gctx[2] = {{nullptr, nullptr, nullptr, 0}, {nullptr, nullptr, nullptr, 0}};
    float* nrm_part = nullptr;                         // 1024 partial sums of squares + the norm (ccsm_train_step) + the scale words below
    unsigned* amax_slot(int k) const { return reinterpret_cast<unsigned*>(nrm_part + 1027 + k); }    // 0, 1: dgi of direction 0 / 1; 2: dSpre; 3: dq
    bool own_any() const { return gctx[0].mode != 2; }
    hipStream_t stream = nullptr, stream1 = nullptr;       // stream1 / blas1: the backward direction of a layer
    hipEvent_t ev_fork = nullptr, ev_join = nullptr;
    float *params = nullptr, *grads = nullptr, *adam_m = nullptr, *adam_v = nullptr;
    bool own_grads = false;
    int64_t step = 0;
    // inputs
    uint8_t* kmer = nullptr;
    float *ipd = nullptr, *pw = nullptr, *npass = nullptr, *h0 = nullptr;
    int32_t* labels = nullptr;
    // activations
    float* x0 = nullptr;
    float* out[L] = {nullptr, nullptr, nullptr};
    float* xdrop[L] = {nullptr, nullptr, nullptr};     // dropout(out[l]) = input of layer l + 1 (rate > 0 only)
    float* sav[L][2][4];
    // activation_bits 8: the four gate arrays of every layer and direction are kept as int8 checkpoints (ccsm_train_act8_pack behind a direction's
    // forward, _unpack in front of its backward); the layers then share one set of fp32 arrays for each direction (sav[l] = sav[0])
    int act_bits = 32;
    uint8_t* codes[L][2][4];
    uint8_t* scales[L][2][4];
    float *gi[2] = {nullptr, nullptr}, *gh[2] = {nullptr, nullptr}, *dgi[2] = {nullptr, nullptr}, *dgh[2] = {nullptr, nullptr},
          *carry[2] = {nullptr, nullptr}, *cpart[2] = {nullptr, nullptr};            // per direction
    float *hn = nullptr, *q = nullptr, *KS = nullptr, *e = nullptr, *a = nullptr, *c = nullptr, *feat = nullptr, *logits = nullptr,
          *dlogits = nullptr, *loss = nullptr;
    float* red[2] = {nullptr, nullptr};               // per stream: per-block partial sums of the step's reductions (added up in a fixed order)
    float *dc = nullptr, *dq = nullptr, *dhn = nullptr, *dA = nullptr, *dB = nullptr;   // dA / dB: (T, M, 512) gradient ping-pong
    float* part[2] = {nullptr, nullptr};               // per direction: (T, 768, 512) per-timestep partial weight gradients
    std::vector<uint8_t> h_kmer;
    std::vector<float> h_f;
    Ctl* ctl = nullptr;                // device
    // captured step graphs, keyed by (sites, train, labels, dropout rate); a key's first call runs eagerly (rocBLAS loads its kernels)
    struct StepGraph { uint64_t key; int uses; hipGraphExec_t exec; };
    std::vector<StepGraph> graphs;
    bool use_graph = false;
    int sp20 = 0, sp21 = 0;            // timesteps per batched weight-gradient product (divisors of 20 / 21); 0 = by batch size
    uint4* whh_frag = nullptr;         // split fp16 B-operand fragments of every W_hh (ccsm_train_seq.hip), repacked every forward
    uint4* whh_t_frag = nullptr;       // ... and of every W_hh^T (the backward kernel's product dgh W_hh)
    int seq_mode = -1;                 // recurrent part: 1 = one fused launch per layer and direction (ccsm_train_seq.hip), 0 = one rocBLAS
                                       // product + gate kernel per timestep, -1 = by batch size (fused from 768 rows up: measured 4.13 vs
                                       // 3.92 ms per step at 256 sites, 5.73 vs 6.40 at 512, 13.6 vs 18.4 at 2048); CCSM_TRAIN_STEPWISE=0|1 forces
    long fused_fallbacks = 0;          // backward passes repeated stepwise because the fused kernel flagged saturation
    bool stepwise_bwd = false;         // CCSM_TRAIN_STEPWISE=bwd (tests): fused forward, stepwise backward - what a saturation fallback runs
    bool stepwise_for(int M) const { return seq_mode == 0 || (seq_mode < 0 && M < 768); }
    bool stepwise_bwd_for(int M) const { return stepwise_bwd || stepwise_for(M); }
};

namespace {

// row-major C(MxN) (+)= op(A) op(B): tA = A is stored K x M, tB = B is stored N x K
inline rocblas_status hip2rb(hipError_t e) { return e == hipSuccess ? rocblas_status_success : rocblas_status_internal_error; }
// row-major C(MxN) (+)= op(A) op(B): tA = A is stored K x M, tB = B is stored N x K.
// grad_a: A holds gradients (every product with tA does: A = dg^T; the backward products through a weight matrix say so themselves)
// amax_pre: a device word that already bounds max |A| (one scan of the gradient tensor serves every product that reads it)
rocblas_status rm_gemm(blas_t h, bool tA, bool tB, int M, int N, int K, float alpha, const float* A, int lda, const float* B,
                       int ldb, float beta, float* C, int ldc, bool grad_a = false, unsigned* amax_pre = nullptr) {
    const bool own = h->mode == 1 || (h->mode == 0 && !tA && M >= 128);
    if (own) return hip2rb(ccsm_train::gemm_s3(h->st, tA, tB, M, N, K, alpha, A, lda, 0, B, ldb, 0, beta, C, ldc, 0, 1,
                                               amax_pre ? amax_pre : (tA || grad_a) ? h->amax : nullptr, amax_pre == nullptr));
#ifdef CCSM_TRAIN_WITH_ROCBLAS
    return rocblas_sgemm(h->rb, tB ? rocblas_operation_transpose : rocblas_operation_none, tA ? rocblas_operation_transpose : rocblas_operation_none,
                         N, M, K, &alpha, B, ldb, A, lda, &beta, C, ldc);
#else
    return rocblas_status_internal_error;
#endif
}
// C_b (M x N) = A_b B_b for `batch` problems at element strides sA / sB / sC (row-major, no transposes; A = gate gradients)
rocblas_status rm_gemm_batched(blas_t h, int M, int N, int K, const float* A, int lda, long long sA, const float* B, int ldb, long long sB,
                               float* C, int ldc, long long sC, int batch) {
    if (h->mode == 1 || (h->mode == 0 && M >= 128))
        return hip2rb(ccsm_train::gemm_s3(h->st, false, false, M, N, K, 1.f, A, lda, sA, B, ldb, sB, 0.f, C, ldc, sC, batch, h->amax));
#ifdef CCSM_TRAIN_WITH_ROCBLAS
    const float one = 1.f, zero = 0.f;
    return rocblas_sgemm_strided_batched(h->rb, rocblas_operation_none, rocblas_operation_none, N, M, K, &one, B, ldb, (rocblas_stride)sB, A, lda,
                                         (rocblas_stride)sA, &zero, C, ldc, (rocblas_stride)sC, batch);
#else
    return rocblas_status_internal_error;
#endif
}

// C (m x n) = sum over `parts` row blocks of A_blk^T B_blk, A_blk = rows_per_part x m (lda), B_blk = rows_per_part x n (ldb): one
// batched product per block into `scratch` (parts x m x n) and a reduction, so that a weight gradient with a 21504-long inner
// dimension fills the chip instead of 24 workgroups.  `extra` slots of scratch beyond `parts` are summed too (filled by the caller).
rocblas_status atb_split(blas_t h, hipStream_t st, int m, int n, int rows_per_part, int parts, const float* A, int lda, const float* B,
                         int ldb, float* scratch, int extra, float* C, unsigned* amax_pre = nullptr) {
    rocblas_status s;
    if (h->mode == 1) {
        s = hip2rb(ccsm_train::gemm_s3(h->st, true, false, m, n, rows_per_part, 1.f, A, lda, (long long)rows_per_part * lda, B, ldb,
                                       (long long)rows_per_part * ldb, 0.f, scratch, n, (long long)m * n, parts, amax_pre ? amax_pre : h->amax,
                                       amax_pre == nullptr));
    } else {
#ifdef CCSM_TRAIN_WITH_ROCBLAS
        const float one = 1.f, zero = 0.f;
        s = rocblas_sgemm_strided_batched(h->rb, rocblas_operation_none, rocblas_operation_transpose, n, m, rows_per_part, &one, B, ldb,
                                          (rocblas_stride)rows_per_part * ldb, A, lda, (rocblas_stride)rows_per_part * lda, &zero, scratch, n,
                                          (rocblas_stride)m * n, parts);
#else
        s = rocblas_status_internal_error;
#endif
    }
    if (s != rocblas_status_success) return s;
    sum_partials_kernel<<<blocks((int64_t)m * n), 256, 0, st>>>(scratch, C, parts + extra, (int64_t)m * n);
    return rocblas_status_success;
}

ccsm_status upload_batch(ccsm_trainer* t, int N, const ccsm_batch* batch, const int32_t* labels, const ccsm_h0* h0) {
    const int M = 2 * N;
    t->h_kmer.resize((size_t)M * T);
    t->h_f.resize((size_t)M * T * 3);
    float* ipd = t->h_f.data();
    float* pw = ipd + (size_t)M * T;
    float* np = pw + (size_t)M * T;
    for (int s = 0; s < 2; ++s) {
        const ccsm_strand& st = batch->strand[s];
        if (!st.kmer || !st.ipd || !st.pw || !st.npass) return fail(CCSM_ERR_INVALID_ARG, "batch pointers must be non-NULL");
        const size_t o = (size_t)s * N * T;
        for (size_t i = 0; i < (size_t)N * T; ++i) {
            int b = batch->kmer_is_f32 ? (int)((const float*)st.kmer)[i] : (int)((const uint8_t*)st.kmer)[i];
            t->h_kmer[o + i] = (uint8_t)(b < 0 ? 4 : (b > 4 ? 4 : b));
            np[o + i] = batch->npass_per_base ? st.npass[i] : st.npass[i / T];
        }
        std::memcpy(ipd + o, st.ipd, sizeof(float) * (size_t)N * T);
        std::memcpy(pw + o, st.pw, sizeof(float) * (size_t)N * T);
    }
    HIPCHK(hipMemcpyAsync(t->kmer, t->h_kmer.data(), (size_t)M * T, hipMemcpyHostToDevice, t->stream));
    HIPCHK(hipMemcpyAsync(t->ipd, ipd, sizeof(float) * (size_t)M * T, hipMemcpyHostToDevice, t->stream));
    HIPCHK(hipMemcpyAsync(t->pw, pw, sizeof(float) * (size_t)M * T, hipMemcpyHostToDevice, t->stream));
    HIPCHK(hipMemcpyAsync(t->npass, np, sizeof(float) * (size_t)M * T, hipMemcpyHostToDevice, t->stream));
    if (labels) HIPCHK(hipMemcpyAsync(t->labels, labels, sizeof(int32_t) * (size_t)N, hipMemcpyHostToDevice, t->stream));
    const int64_t nh0 = (int64_t)2 * L * M * H;
    const int mode = h0 ? h0->mode : CCSM_H0_ZERO;
    if (mode == CCSM_H0_EXPLICIT) {
        if (!h0->h0[0] || !h0->h0[1]) return fail(CCSM_ERR_INVALID_ARG, "explicit h0 needs both tensors");
        for (int k = 0; k < 2 * L; ++k)
            for (int s = 0; s < 2; ++s)
                HIPCHK(hipMemcpyAsync(t->h0 + ((size_t)k * M + (size_t)s * N) * H, h0->h0[s] + (size_t)k * N * H, sizeof(float) * (size_t)N * H,
                                      hipMemcpyHostToDevice, t->stream));
    } else if (mode == CCSM_H0_ZERO) {
        HIPCHK(hipMemsetAsync(t->h0, 0, sizeof(float) * nh0, t->stream));
    } else if (mode == CCSM_H0_DEVICE_RNG) {
        h0_rng_kernel<<<blocks(nh0), 256, 0, t->stream>>>(t->h0, nh0, N, h0->seed, h0->offset);
    } else {
        return fail(CCSM_ERR_INVALID_ARG, "unknown h0 mode");
    }
    HIPCHK(hipStreamSynchronize(t->stream));      // the host staging vectors are reused by the next call
    return CCSM_OK;
}

// The two directions of a layer are independent: direction 0 runs on the trainer's stream, direction 1 on a second stream with
// its own rocBLAS handle, joined by events at the layer boundaries (a 1024-row recurrent product alone leaves a quarter of the
// CUs idle and is latency-bound).
ccsm_status fork(ccsm_trainer* t) {
    HIPCHK(hipEventRecord(t->ev_fork, t->stream));
    HIPCHK(hipStreamWaitEvent(t->stream1, t->ev_fork, 0));
    return CCSM_OK;
}
ccsm_status join(ccsm_trainer* t) {
    HIPCHK(hipEventRecord(t->ev_join, t->stream1));
    HIPCHK(hipStreamWaitEvent(t->stream, t->ev_join, 0));
    return CCSM_OK;
}

// the gates of one layer and direction into their checkpoints, or out of them again
ccsm_status keep_gates(ccsm_trainer* t, int M, int l, int d, bool back) {
    if (t->act_bits != 8) return CCSM_OK;
    hipStream_t st = d == 0 ? t->stream : t->stream1;
    for (int k = 0; k < 4; ++k) {
        const ccsm_saved s{t->codes[l][d][k], H, CCSM_CODE_INT8, t->scales[l][d][k], H / 32};
        const ccsm_status e = back ? ccsm_train_act8_unpack(t->device, CCSM_TYPE_F32, (int64_t)T * M, H, &s, t->sav[l][d][k], H, st)
                                   : ccsm_train_act8_pack(t->device, CCSM_TYPE_F32, CCSM_CODE_INT8, (int64_t)T * M, H, t->sav[l][d][k], H, t->codes[l][d][k], H, t->scales[l][d][k],
                                                          H / 32, st);
        if (e != CCSM_OK) return fail(e, std::string("the gates' checkpoints: ") + ccsm_train_ops_last_error());
    }
    return CCSM_OK;
}

ccsm_status forward_dir(ccsm_trainer* t, int M, int l, int d, const float* X, int in, bool train) {
    const float* P = t->params;
    blas_t blas = d == 0 ? t->blas : t->blas1;
    hipStream_t st = d == 0 ? t->stream : t->stream1;
    BLASCHK(rm_gemm(blas, false, true, T * M, G, in, 1.f, X, in, P + kOff.w_ih[l][d], in, 0.f, t->gi[d], G));
    if (!t->stepwise_for(M)) {     // all 21 steps in one launch (ccsm_train_seq.hip)
        gru_seq_fwd_kernel<<<(M + 31) / 32, 512, kSqLds, st>>>(t->gi[d], t->h0 + (size_t)(2 * l + d) * M * H, t->whh_frag + (size_t)(2 * l + d) * kSqFragPerDir,
                                                               P + kOff.b_ih[l][d], P + kOff.b_hh[l][d], t->out[l] + d * H, t->sav[l][d][0], t->sav[l][d][1],
                                                               t->sav[l][d][2], t->sav[l][d][3], M, d, train ? 1 : 0);
        HIPCHK(hipGetLastError());
        return train ? keep_gates(t, M, l, d, false) : CCSM_OK;
    }
    for (int s = 0; s < T; ++s) {
        const int tt = d == 0 ? s : T - 1 - s;
        const float* hprev;
        int ld;
        if (s == 0) { hprev = t->h0 + (size_t)(2 * l + d) * M * H; ld = H; }
        else { hprev = t->out[l] + (size_t)(d == 0 ? tt - 1 : tt + 1) * M * H2 + d * H; ld = H2; }
        BLASCHK(rm_gemm(blas, false, true, M, G, H, 1.f, hprev, ld, P + kOff.w_hh[l][d], H, 0.f, t->gh[d], G));
        const size_t so = (size_t)tt * M * H;
        gru_gate_fwd_kernel<<<blocks((int64_t)M * H), 256, 0, st>>>(t->gi[d] + (size_t)tt * M * G, t->gh[d], P + kOff.b_ih[l][d], P + kOff.b_hh[l][d],
                                                                   hprev, ld, t->out[l] + (size_t)tt * M * H2 + d * H, t->sav[l][d][0] + so,
                                                                   t->sav[l][d][1] + so, t->sav[l][d][2] + so, t->sav[l][d][3] + so, M, train ? 1 : 0);
    }
    return train ? keep_gates(t, M, l, d, false) : CCSM_OK;
}

ccsm_status forward(ccsm_trainer* t, int N, bool train, float rate, bool have_labels) {
    const int M = 2 * N;
    const float* P = t->params;
    hipStream_t st = t->stream;
    build_x0_kernel<<<blocks((int64_t)T * M), 256, 0, st>>>(t->kmer, t->ipd, t->pw, t->npass, P + kOff.embed, t->x0, M);
    if (!t->stepwise_for(M))
        for (int l = 0; l < L; ++l)
            for (int d = 0; d < 2; ++d)
                {
                    pack_whh_kernel<<<blocks(8 * (H / 16) * 3 * 64), 256, 0, st>>>(P + kOff.w_hh[l][d], t->whh_frag + (size_t)(2 * l + d) * kSqFragPerDir);
                    if (train) pack_whh_t_kernel<<<blocks(8 * (G / 16) * 64), 256, 0, st>>>(P + kOff.w_hh[l][d], t->whh_t_frag + (size_t)(2 * l + d) * kSqFragPerDir);
                }
    const bool drop = train && rate > 0.f;
    for (int l = 0; l < L; ++l) {
        const float* X = l == 0 ? t->x0 : (drop ? t->xdrop[l - 1] : t->out[l - 1]);
        const int in = l == 0 ? F0 : H2;
        ccsm_status s = fork(t);
        if (s != CCSM_OK) return s;
        for (int d = 0; d < 2; ++d) {
            s = forward_dir(t, M, l, d, X, in, train);
            if (s != CCSM_OK) return s;
        }
        s = join(t);
        if (s != CCSM_OK) return s;
        if (drop && l + 1 < L)
            dropout_kernel<<<blocks((int64_t)T * M * H2), 256, 0, st>>>(t->out[l], t->xdrop[l], (int64_t)T * M * H2, rate, t->ctl, 0xd0 + l);
    }
    const float* O2 = t->out[L - 1];
    gather_hn_kernel<<<blocks((int64_t)M * H2), 256, 0, st>>>(O2, t->hn, M);
    BLASCHK(rm_gemm(t->blas, false, true, M, H, H2, 1.f, t->hn, H2, P + kOff.wa, H2, 0.f, t->q, H));
    BLASCHK(rm_gemm(t->blas, false, true, T * M, H, H2, 1.f, O2, H2, P + kOff.ua, H2, 0.f, t->KS, H));
    att_score_kernel<<<blocks((int64_t)T * M, 4), 256, 0, st>>>(t->KS, t->q, P + kOff.va, t->e, M);
    att_softmax_kernel<<<blocks(M), 256, 0, st>>>(t->e, t->a, M);
    att_context_kernel<<<blocks((int64_t)M * H2), 256, 0, st>>>(t->a, O2, t->c, M);
    HIPCHK(hipMemsetAsync(t->loss, 0, 2 * sizeof(float), st));      // [loss sum | saturation flag of the fused backward kernels]
    fc_loss_kernel<<<blocks(N, 4), 256, 0, st>>>(t->c, P + kOff.fcw, P + kOff.fcb, have_labels ? t->labels : nullptr, t->ctl,
                                                 drop ? rate : 0.f, t->feat, t->logits, train ? t->dlogits : nullptr, t->red[0], N);
    if (have_labels) sum_fixed_kernel<<<1, 256, 0, st>>>(t->red[0], N, t->loss);
    HIPCHK(hipGetLastError());
    return CCSM_OK;
}

ccsm_status backward_dir(ccsm_trainer* t, int M, int l, int d, const float* dO, const float* X, int in) {
    const float* P = t->params;
    float* Gd = t->grads;
    blas_t blas = d == 0 ? t->blas : t->blas1;
    hipStream_t st = d == 0 ? t->stream : t->stream1;
    float *dgi = t->dgi[d], *dgh = t->dgh[d], *carry = t->carry[d], *part = t->part[d];
    // timesteps per batched weight-gradient product: measured best 2 / 3 up to 1024 sites per step (6.98 vs 8.30 ms at 512), 4 / 3 above
    // (the library's own kernel: one timestep per partial product - 20 / 21 problems of (768 / 128) x (n / 128) workgroups fill the chip)
    const bool own_atb = t->gctx[0].mode == 1;
    const int sp20 = t->sp20 ? t->sp20 : own_atb ? 1 : (M <= 2048 ? 2 : 4), sp21 = t->sp21 ? t->sp21 : own_atb ? 1 : 3;
    float* cpart = t->cpart[d];
    { const ccsm_status e = keep_gates(t, M, l, d, true); if (e != CCSM_OK) return e; }
    if (!t->stepwise_bwd_for(M)) {     // all 21 steps in one launch (ccsm_train_seq.hip)
        gru_seq_bwd_kernel<<<(M + 31) / 32, 512, kSbLds, st>>>(dO + d * H, t->out[l] + d * H, t->h0 + (size_t)(2 * l + d) * M * H,
                                                               t->whh_t_frag + (size_t)(2 * l + d) * kSqFragPerDir, t->sav[l][d][0], t->sav[l][d][1],
                                                               t->sav[l][d][2], t->sav[l][d][3], dgi, dgh, t->red[d], M, d,
                                                               reinterpret_cast<int*>(t->loss + 1));
        seq_bias_reduce_kernel<<<blocks(4 * H), 256, 0, st>>>(t->red[d], (M + 31) / 32, Gd + kOff.b_ih[l][d], Gd + kOff.b_hh[l][d]);
        HIPCHK(hipGetLastError());
    } else {
        HIPCHK(hipMemsetAsync(carry, 0, sizeof(float) * (size_t)M * H, st));
        HIPCHK(hipMemsetAsync(cpart, 0, sizeof(float) * (size_t)3 * M * H, st));
        for (int s = T - 1; s >= 0; --s) {
            const int tt = d == 0 ? s : T - 1 - s;
            const float* hprev;
            int ld;
            if (s == 0) { hprev = t->h0 + (size_t)(2 * l + d) * M * H; ld = H; }
            else { hprev = t->out[l] + (size_t)(d == 0 ? tt - 1 : tt + 1) * M * H2 + d * H; ld = H2; }
            const size_t so = (size_t)tt * M * H;
            gru_gate_bwd_kernel<<<blocks((int64_t)M * H), 256, 0, st>>>(dO + (size_t)tt * M * H2 + d * H, carry, cpart, t->sav[l][d][0] + so,
                                                                       t->sav[l][d][1] + so, t->sav[l][d][2] + so, t->sav[l][d][3] + so, hprev, ld,
                                                                       dgi + (size_t)tt * M * G, dgh + (size_t)tt * M * G, M);
            if (s > 0) {
                // cpart[g] (M x 256) = dgh_t[:, g*256 : (g+1)*256] W_hh[g*256 : (g+1)*256, :]
                BLASCHK(rm_gemm_batched(blas, M, H, H, dgh + (size_t)tt * M * G, G, H, P + kOff.w_hh[l][d], H, (long long)H * H, cpart, H, (long long)M * H, 3));
            }
        }
    }
    // one scan of this direction's gate gradients bounds every product that reads them (|dgh| <= |dgi| elementwise: dgh_n = r dgi_n)
    unsigned* am = nullptr;
    if (t->own_any()) {
        am = t->amax_slot(d);
        HIPCHK(ccsm_train::gemm_scan_amax(st, dgi, G, T * M, G, am));
    }
    // weight gradients over all steps at once
    float* dWhh = Gd + kOff.w_hh[l][d];
    float* last = part + (size_t)((T - 1) / sp20) * G * H;      // the h0 step's product goes to the slot after the batched ones
    if (d == 0) {
        BLASCHK(rm_gemm(blas, true, false, G, H, M, 1.f, dgh, G, t->h0 + (size_t)(2 * l) * M * H, H, 0.f, last, H, true, am));
        BLASCHK(atb_split(blas, st, G, H, M * sp20, (T - 1) / sp20, dgh + (size_t)M * G, G, t->out[l], H2, part, 1, dWhh, am));
    } else {
        BLASCHK(rm_gemm(blas, true, false, G, H, M, 1.f, dgh + (size_t)(T - 1) * M * G, G, t->h0 + (size_t)(2 * l + 1) * M * H, H, 0.f, last, H, true, am));
        BLASCHK(atb_split(blas, st, G, H, M * sp20, (T - 1) / sp20, dgh, G, t->out[l] + (size_t)M * H2 + H, H2, part, 1, dWhh, am));
    }
    BLASCHK(atb_split(blas, st, G, in, M * sp21, T / sp21, dgi, G, X, in, part, 0, Gd + kOff.w_ih[l][d], am));
    if (t->stepwise_bwd_for(M)) {      // (the fused backward kernel has accumulated the bias gradients already)
        const int nb = (int)blocks((int64_t)T * M, 32).x;
        colsum_kernel<<<nb, 256, 0, st>>>(dgi, t->red[d], T * M, G);
        sum_partials_kernel<<<blocks(G), 256, 0, st>>>(t->red[d], Gd + kOff.b_ih[l][d], nb, G);
        colsum_kernel<<<nb, 256, 0, st>>>(dgh, t->red[d], T * M, G);
        sum_partials_kernel<<<blocks(G), 256, 0, st>>>(t->red[d], Gd + kOff.b_hh[l][d], nb, G);
    }
    return CCSM_OK;
}

ccsm_status backward(ccsm_trainer* t, int N, float rate) {
    const int M = 2 * N;
    const float* P = t->params;
    float* Gd = t->grads;
    hipStream_t st = t->stream;
    const bool drop = rate > 0.f;
    HIPCHK(hipMemsetAsync(Gd, 0, sizeof(float) * kOff.total, st));
    // fc1 and dropout1
    BLASCHK(rm_gemm(t->blas, true, false, NC, 2 * H2, N, 1.f, t->dlogits, NC, t->feat, 2 * H2, 0.f, Gd + kOff.fcw, 2 * H2));
    fc_bwd_kernel<<<blocks((int64_t)N * 2 * H2), 256, 0, st>>>(t->dlogits, P + kOff.fcw, drop ? rate : 0.f, t->ctl, t->dc, Gd + kOff.fcb, N);
    // attention
    const float* O2 = t->out[L - 1];
    float* dO = t->dA;
    att_dalpha_kernel<<<blocks((int64_t)T * M, 4), 256, 0, st>>>(t->dc, O2, t->e, M);        // e <- da
    att_dscore_kernel<<<blocks(M), 256, 0, st>>>(t->a, t->e, M);                             // e <- de
    att_dout_init_kernel<<<blocks((int64_t)T * M * H2), 256, 0, st>>>(t->a, t->dc, dO, M);
    att_dpre_kernel<<<blocks((int64_t)T * M, 64), H, 0, st>>>(t->KS, t->e, P + kOff.va, t->red[0], T * M);   // KS <- dSpre
    sum_partials_kernel<<<blocks(H), 256, 0, st>>>(t->red[0], Gd + kOff.va, (int)blocks((int64_t)T * M, 64).x, H);
    att_dq_kernel<<<blocks((int64_t)M * H), 256, 0, st>>>(t->KS, t->dq, M);
    unsigned *am_s = nullptr, *am_q = nullptr;
    if (t->own_any()) {
        am_s = t->amax_slot(2); am_q = t->amax_slot(3);
        HIPCHK(ccsm_train::gemm_scan_amax(st, t->KS, H, T * M, H, am_s));
        HIPCHK(ccsm_train::gemm_scan_amax(st, t->dq, H, M, H, am_q));
    }
    { const int sp21 = t->sp21 ? t->sp21 : t->gctx[0].mode == 1 ? 1 : 3;
      BLASCHK(atb_split(t->blas, st, H, H2, M * sp21, T / sp21, t->KS, H, O2, H2, t->part[0], 0, Gd + kOff.ua, am_s)); }
    BLASCHK(rm_gemm(t->blas, false, false, T * M, H2, H, 1.f, t->KS, H, P + kOff.ua, H2, 1.f, dO, H2, true, am_s));
    BLASCHK(rm_gemm(t->blas, true, false, H, H2, M, 1.f, t->dq, H, t->hn, H2, 0.f, Gd + kOff.wa, H2, true, am_q));
    BLASCHK(rm_gemm(t->blas, false, false, M, H2, H, 1.f, t->dq, H, P + kOff.wa, H2, 0.f, t->dhn, H2, true, am_q));
    scatter_dhn_kernel<<<blocks((int64_t)M * H2), 256, 0, st>>>(t->dhn, dO, M);
    // GRU layers, top down
    float* dX = t->dB;
    for (int l = L - 1; l >= 0; --l) {
        const float* X = l == 0 ? t->x0 : (drop ? t->xdrop[l - 1] : t->out[l - 1]);
        const int in = l == 0 ? F0 : H2;
        ccsm_status s = fork(t);
        if (s != CCSM_OK) return s;
        for (int d = 0; d < 2; ++d) {
            s = backward_dir(t, M, l, d, dO, X, in);
            if (s != CCSM_OK) return s;
        }
        s = join(t);
        if (s != CCSM_OK) return s;
        for (int d = 0; d < 2; ++d)
            BLASCHK(rm_gemm(t->blas, false, false, T * M, in, G, 1.f, t->dgi[d], G, P + kOff.w_ih[l][d], in, d == 0 ? 0.f : 1.f, dX, in, true,
                            t->own_any() ? t->amax_slot(d) : nullptr));
        if (l == 0) {
            embed_bwd_kernel<<<blocks((int64_t)T * M), 256, 0, st>>>(dX, t->kmer, t->red[0], M);
            sum_partials_kernel<<<1, 256, 0, st>>>(t->red[0], Gd + kOff.embed, (int)blocks((int64_t)T * M).x, NV * NE);
        } else {
            if (drop) dropout_kernel<<<blocks((int64_t)T * M * H2), 256, 0, st>>>(dX, dX, (int64_t)T * M * H2, rate, t->ctl, 0xd0 + (l - 1));
            float* tmp = dO; dO = dX; dX = tmp;
        }
    }
    HIPCHK(hipGetLastError());
    return CCSM_OK;
}

template <typename Tp>
ccsm_status dalloc(Tp** p, size_t n) {
    HIPCHK(hipMalloc((void**)p, n * sizeof(Tp)));
    return CCSM_OK;
}

}  // namespace

extern "C" {

const char* ccsm_train_last_error(void) { return g_err.c_str(); }
int64_t ccsm_train_num_params(void) { return kOff.total; }
int ccsm_train_param_offsets(int64_t* offsets, int n) {
    if (!offsets || n < 31) return 1;
    for (int i = 0; i < 31; ++i) offsets[i] = kOff.list[i];
    return 0;
}

ccsm_status ccsm_train_create(const ccsm_weights* w, int device, int max_sites, float* d_grads, ccsm_trainer** out) {
    return ccsm_train_create_act(w, device, max_sites, d_grads, 32, out);
}
ccsm_status ccsm_train_create_act(const ccsm_weights* w, int device, int max_sites, float* d_grads, int activation_bits, ccsm_trainer** out) {
    if (!w || !out || max_sites <= 0) return fail(CCSM_ERR_INVALID_ARG, "weights, out must be non-NULL and max_sites > 0");
    if (activation_bits != 32 && activation_bits != 8) return fail(CCSM_ERR_INVALID_ARG, "activation_bits must be 32 or 8");
    *out = nullptr;
    HIPCHK(hipSetDevice(device));
    ccsm_trainer* t = new ccsm_trainer();
    t->device = device;
    t->max_sites = max_sites;
    t->act_bits = activation_bits;
    const size_t M = 2 * (size_t)max_sites;
    for (int l = 0; l < L; ++l)
        for (int d = 0; d < 2; ++d)
            for (int k = 0; k < 4; ++k) { t->sav[l][d][k] = nullptr; t->codes[l][d][k] = t->scales[l][d][k] = nullptr; }
#define TRY(x) do { ccsm_status s__ = (x); if (s__ != CCSM_OK) { ccsm_train_destroy(t); return s__; } } while (0)
    HIPCHK(hipStreamCreate(&t->stream));
    HIPCHK(hipStreamCreate(&t->stream1));
    HIPCHK(hipEventCreateWithFlags(&t->ev_fork, hipEventDisableTiming));
    HIPCHK(hipEventCreateWithFlags(&t->ev_join, hipEventDisableTiming));
    TRY(dalloc(&t->nrm_part, 1024 + 1 + 8));
    {
        int mode = 1;                                   // the library's own kernel
#ifdef CCSM_TRAIN_WITH_ROCBLAS
        const char* gm = std::getenv("CCSM_TRAIN_GEMM");
        mode = gm && std::strcmp(gm, "mixed") == 0 ? 0 : gm && std::strcmp(gm, "rocblas") == 0 ? 2 : 1;
#endif
        t->gctx[0] = GemmCtx{t->stream, reinterpret_cast<unsigned*>(t->nrm_part + 1025), nullptr, mode};
        t->gctx[1] = GemmCtx{t->stream1, reinterpret_cast<unsigned*>(t->nrm_part + 1026), nullptr, mode};
        t->blas = &t->gctx[0];
        t->blas1 = &t->gctx[1];
        HIPCHK(ccsm_train::gemm_s3_init());
#ifdef CCSM_TRAIN_WITH_ROCBLAS
        if (mode != 1) {
            if (rocblas_create_handle(&t->gctx[0].rb) != rocblas_status_success || rocblas_create_handle(&t->gctx[1].rb) != rocblas_status_success) {
                ccsm_train_destroy(t);
                return fail(CCSM_ERR_HIP, "rocblas_create_handle failed");
            }
            rocblas_set_stream(t->gctx[0].rb, t->stream);
            rocblas_set_stream(t->gctx[1].rb, t->stream1);
            rocblas_set_pointer_mode(t->gctx[0].rb, rocblas_pointer_mode_host);
            rocblas_set_pointer_mode(t->gctx[1].rb, rocblas_pointer_mode_host);
        }
#endif
    }
    TRY(dalloc(&t->params, kOff.total));
    TRY(dalloc(&t->adam_m, kOff.total));
    TRY(dalloc(&t->adam_v, kOff.total));
    if (d_grads) t->grads = d_grads; else { TRY(dalloc(&t->grads, kOff.total)); t->own_grads = true; }
    HIPCHK(hipMemset(t->adam_m, 0, sizeof(float) * kOff.total));
    HIPCHK(hipMemset(t->adam_v, 0, sizeof(float) * kOff.total));
    HIPCHK(hipStreamSynchronize(nullptr));      // (device memsets are asynchronous, on the NULL stream, which the trainer's own stream does not wait for)
    TRY(dalloc(&t->kmer, M * T));
    TRY(dalloc(&t->ipd, M * T)); TRY(dalloc(&t->pw, M * T)); TRY(dalloc(&t->npass, M * T));
    TRY(dalloc(&t->labels, (size_t)max_sites));
    TRY(dalloc(&t->h0, 2 * L * M * H + 32 * H));      // + 32 rows of slack everywhere the fused recurrent kernels read whole 32-row tiles
    TRY(dalloc(&t->x0, T * M * F0));
    for (int l = 0; l < L; ++l) {
        TRY(dalloc(&t->out[l], T * M * H2 + 32 * H2));
        if (l + 1 < L) TRY(dalloc(&t->xdrop[l], T * M * H2));
        for (int d = 0; d < 2; ++d)
            for (int k = 0; k < 4; ++k) {
                if (l == 0 || t->act_bits != 8) TRY(dalloc(&t->sav[l][d][k], T * M * H + 32 * H));
                else t->sav[l][d][k] = t->sav[0][d][k];
                if (t->act_bits == 8) { TRY(dalloc(&t->codes[l][d][k], T * M * H)); TRY(dalloc(&t->scales[l][d][k], T * M * (H / 32))); }
            }
    }
    for (int d = 0; d < 2; ++d) {
        TRY(dalloc(&t->gi[d], T * M * G + 32 * G));     // + 32 rows of slack: gru_seq_fwd_kernel reads whole 32-row tiles
        TRY(dalloc(&t->gh[d], M * G)); TRY(dalloc(&t->dgi[d], T * M * G)); TRY(dalloc(&t->dgh[d], T * M * G));
        TRY(dalloc(&t->carry[d], M * H)); TRY(dalloc(&t->cpart[d], 3 * M * H)); TRY(dalloc(&t->part[d], (size_t)T * G * H2));
        TRY(dalloc(&t->red[d], ((size_t)T * M / 32 + 2) * G));        // the largest user: colsum_kernel, 32 rows per block x 768 columns
    }
    TRY(dalloc(&t->hn, M * H2)); TRY(dalloc(&t->q, M * H)); TRY(dalloc(&t->KS, T * M * H)); TRY(dalloc(&t->e, T * M)); TRY(dalloc(&t->a, T * M));
    TRY(dalloc(&t->c, M * H2)); TRY(dalloc(&t->feat, (size_t)max_sites * 2 * H2)); TRY(dalloc(&t->logits, (size_t)max_sites * NC));
    TRY(dalloc(&t->dlogits, (size_t)max_sites * NC)); TRY(dalloc(&t->loss, 2)); TRY(dalloc(&t->ctl, 1));
    { const char* e = std::getenv("CCSM_TRAIN_SP20"); if (e) t->sp20 = std::atoi(e); e = std::getenv("CCSM_TRAIN_SP21"); if (e) t->sp21 = std::atoi(e);
      if (t->sp20 < 0 || (t->sp20 && (T - 1) % t->sp20)) t->sp20 = 0;
      if (t->sp21 < 0 || (t->sp21 && T % t->sp21)) t->sp21 = 0; }
    { const char* e = std::getenv("CCSM_TRAIN_GRAPH"); t->use_graph = e && e[0] == '1'; }   // opt-in: measured +1.5 % (the step is not launch-bound)
    { const char* e = std::getenv("CCSM_TRAIN_STEPWISE"); if (e && (e[0] == '0' || e[0] == '1')) t->seq_mode = e[0] == '1' ? 0 : 1; if (e && e[0] == 'b') t->stepwise_bwd = true; }
    TRY(dalloc(&t->whh_frag, (size_t)2 * L * kSqFragPerDir));
    TRY(dalloc(&t->whh_t_frag, (size_t)2 * L * kSqFragPerDir));
    HIPCHK(hipFuncSetAttribute(reinterpret_cast<const void*>(&gru_seq_bwd_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kSbLds));
    HIPCHK(hipFuncSetAttribute(reinterpret_cast<const void*>(&gru_seq_fwd_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kSqLds));
    TRY(dalloc(&t->dc, M * H2)); TRY(dalloc(&t->dq, M * H)); TRY(dalloc(&t->dhn, M * H2)); TRY(dalloc(&t->dA, T * M * H2 + 32 * H2)); TRY(dalloc(&t->dB, T * M * H2 + 32 * H2));
    // parameters: host tensors -> flat order
    std::vector<float> flat((size_t)kOff.total);
    auto put = [&](int64_t off, const float* src, int64_t n) { if (src) std::memcpy(flat.data() + off, src, sizeof(float) * (size_t)n); };
    bool ok = w->embed_weight && w->att_wa && w->att_ua && w->att_va && w->fc1_weight && w->fc1_bias;
    for (int l = 0; l < L; ++l)
        for (int d = 0; d < 2; ++d) ok = ok && w->weight_ih[l][d] && w->weight_hh[l][d] && w->bias_ih[l][d] && w->bias_hh[l][d];
    if (!ok) { ccsm_train_destroy(t); return fail(CCSM_ERR_INVALID_ARG, "every weight tensor must be non-NULL"); }
    put(kOff.embed, w->embed_weight, NV * NE);
    for (int l = 0; l < L; ++l)
        for (int d = 0; d < 2; ++d) {
            put(kOff.w_ih[l][d], w->weight_ih[l][d], (int64_t)G * (l == 0 ? F0 : H2));
            put(kOff.w_hh[l][d], w->weight_hh[l][d], (int64_t)G * H);
            put(kOff.b_ih[l][d], w->bias_ih[l][d], G);
            put(kOff.b_hh[l][d], w->bias_hh[l][d], G);
        }
    put(kOff.wa, w->att_wa, (int64_t)H * H2);
    put(kOff.ua, w->att_ua, (int64_t)H * H2);
    put(kOff.va, w->att_va, H);
    put(kOff.fcw, w->fc1_weight, (int64_t)NC * 2 * H2);
    put(kOff.fcb, w->fc1_bias, NC);
    HIPCHK(hipMemcpy(t->params, flat.data(), sizeof(float) * kOff.total, hipMemcpyHostToDevice));
    HIPCHK(hipStreamSynchronize(t->stream));
#undef TRY
    *out = t;
    return CCSM_OK;
}

void ccsm_train_destroy(ccsm_trainer* t) {
    if (!t) return;
    (void)hipSetDevice(t->device);
    float* fl[] = {t->params, t->adam_m, t->adam_v, t->own_grads ? t->grads : nullptr, t->ipd, t->pw, t->npass, t->h0, t->x0, t->gi[0], t->gi[1], t->gh[0], t->gh[1], t->dgi[0],
                   t->dgi[1], t->dgh[0], t->dgh[1], t->carry[0], t->carry[1], t->cpart[0], t->cpart[1], t->part[0], t->part[1], t->hn, t->q, t->KS, t->e, t->a, t->c, t->feat, t->logits, t->dlogits, t->loss, t->dc, t->dq, t->dhn, t->dA, t->dB};
    for (float* p : fl) if (p) (void)hipFree(p);
    for (int d = 0; d < 2; ++d) if (t->red[d]) (void)hipFree(t->red[d]);
    for (auto& c : t->graphs) if (c.exec) (void)hipGraphExecDestroy(c.exec);
    if (t->ctl) (void)hipFree(t->ctl);
    if (t->whh_frag) (void)hipFree(t->whh_frag);
    if (t->whh_t_frag) (void)hipFree(t->whh_t_frag);
    if (t->kmer) (void)hipFree(t->kmer);
    if (t->labels) (void)hipFree(t->labels);
    for (int l = 0; l < L; ++l) {
        if (t->out[l]) (void)hipFree(t->out[l]);
        if (t->xdrop[l]) (void)hipFree(t->xdrop[l]);
        for (int d = 0; d < 2; ++d)
            for (int k = 0; k < 4; ++k) {
                if (t->sav[l][d][k] && (l == 0 || t->act_bits != 8)) (void)hipFree(t->sav[l][d][k]);
                if (t->codes[l][d][k]) (void)hipFree(t->codes[l][d][k]);
                if (t->scales[l][d][k]) (void)hipFree(t->scales[l][d][k]);
            }
    }
#ifdef CCSM_TRAIN_WITH_ROCBLAS
    for (int k = 0; k < 2; ++k)
        if (t->gctx[k].rb) rocblas_destroy_handle(t->gctx[k].rb);
#endif
    if (t->nrm_part) (void)hipFree(t->nrm_part);
    if (t->ev_fork) (void)hipEventDestroy(t->ev_fork);
    if (t->ev_join) (void)hipEventDestroy(t->ev_join);
    if (t->stream1) (void)hipStreamDestroy(t->stream1);
    if (t->stream) (void)hipStreamDestroy(t->stream);
    delete t;
}

static ccsm_status run(ccsm_trainer* t, int n_sites, const ccsm_batch* batch, const int32_t* labels, const ccsm_h0* h0, float pos_weight,
                       bool train, float rate, uint64_t seed, float* loss, float* logits) {
    if (!t || !batch) return fail(CCSM_ERR_INVALID_ARG, "trainer and batch must be non-NULL");
    if (n_sites <= 0) return fail(CCSM_ERR_INVALID_ARG, "n_sites must be > 0");
    if (n_sites > t->max_sites) return fail(CCSM_ERR_CAPACITY, "n_sites exceeds max_sites");
    if (train && !labels) return fail(CCSM_ERR_INVALID_ARG, "training needs labels");
    if (!(rate >= 0.f && rate < 1.f)) return fail(CCSM_ERR_INVALID_ARG, "dropout_rate must be in [0, 1)");
    HIPCHK(hipSetDevice(t->device));
    ccsm_status s = upload_batch(t, n_sites, batch, labels, h0);
    if (s != CCSM_OK) return s;
    double wsum = 0.0;
    if (labels) for (int i = 0; i < n_sites; ++i) wsum += labels[i] != 0 ? (double)pos_weight : 1.0;
    const Ctl host_ctl = {seed, pos_weight, (float)wsum};
    HIPCHK(hipMemcpyAsync(t->ctl, &host_ctl, sizeof(Ctl), hipMemcpyHostToDevice, t->stream));
    HIPCHK(hipStreamSynchronize(t->stream));            // host_ctl is a stack object
    uint32_t rate_bits;
    std::memcpy(&rate_bits, &rate, 4);
    const uint64_t key = ((uint64_t)n_sites << 34) | ((uint64_t)(train ? 1 : 0) << 33) | ((uint64_t)(labels ? 1 : 0) << 32) | rate_bits;
    auto enqueue = [&]() -> ccsm_status {
        ccsm_status e = forward(t, n_sites, train, rate, labels != nullptr);
        if (e == CCSM_OK && train) e = backward(t, n_sites, rate);
        return e;
    };
    ccsm_trainer::StepGraph* g = nullptr;
    for (auto& c : t->graphs) if (c.key == key) g = &c;
    if (!t->use_graph) {
        s = enqueue();
        if (s != CCSM_OK) return s;
    } else if (g == nullptr) {                           // first call of this shape: eager (rocBLAS loads and tunes its kernels here)
        if (t->graphs.size() >= 16) {
            for (auto& c : t->graphs) if (c.exec) (void)hipGraphExecDestroy(c.exec);
            t->graphs.clear();
        }
        t->graphs.push_back({key, 1, nullptr});
        s = enqueue();
        if (s != CCSM_OK) return s;
    } else {
        if (g->exec == nullptr) {                        // second call: capture both streams' work into one graph
            hipGraph_t graph = nullptr;
            HIPCHK(hipStreamBeginCapture(t->stream, hipStreamCaptureModeThreadLocal));
            s = enqueue();
            hipError_t ce = hipStreamEndCapture(t->stream, &graph);
            if (s != CCSM_OK) { if (graph) (void)hipGraphDestroy(graph); return s; }
            if (ce != hipSuccess) return fail(CCSM_ERR_HIP, std::string("hipStreamEndCapture: ") + hipGetErrorString(ce));
            hipError_t ie = hipGraphInstantiate(&g->exec, graph, nullptr, nullptr, 0);
            (void)hipGraphDestroy(graph);
            if (ie != hipSuccess) { g->exec = nullptr; return fail(CCSM_ERR_HIP, std::string("hipGraphInstantiate: ") + hipGetErrorString(ie)); }
        }
        g->uses += 1;
        HIPCHK(hipGraphLaunch(g->exec, t->stream));
    }
    float lsum = 0.f;
    float lbuf[2] = {0.f, 0.f};
    HIPCHK(hipMemcpyAsync(lbuf, t->loss, 2 * sizeof(float), hipMemcpyDeviceToHost, t->stream));
    if (logits) HIPCHK(hipMemcpyAsync(logits, t->logits, sizeof(float) * (size_t)n_sites * NC, hipMemcpyDeviceToHost, t->stream));
    HIPCHK(hipStreamSynchronize(t->stream));
    lsum = lbuf[0];
    int sat = 0;
    std::memcpy(&sat, &lbuf[1], sizeof(int));
    if (train && sat && !t->stepwise_bwd_for(2 * n_sites)) {
        // a gate gradient left the range of the fused kernels' scaled fp16 operands (|.| > 14.6: e.g. a sum-reduced loss or a blown-up
        // fc1 layer): this step is repeated with the backward pass step by step in fp32.  The forward pass runs again first - the
        // backward pass overwrites the attention scores and keys it reads (e, KS) - with the same inputs, masks and initial states
        const bool keep = t->stepwise_bwd;
        t->stepwise_bwd = true;
        s = forward(t, n_sites, true, rate, labels != nullptr);
        if (s == CCSM_OK) s = backward(t, n_sites, rate);
        t->stepwise_bwd = keep;
        if (s != CCSM_OK) return s;
        HIPCHK(hipStreamSynchronize(t->stream));
        t->fused_fallbacks += 1;
    }
    if (loss) *loss = labels ? (float)(lsum / wsum) : 0.f;
    return CCSM_OK;
}

ccsm_status ccsm_train_forward_backward(ccsm_trainer* t, int n_sites, const ccsm_batch* batch, const int32_t* labels, const ccsm_h0* h0,
                                        float pos_weight, float dropout_rate, uint64_t dropout_seed, float* loss, float* logits) {
    return run(t, n_sites, batch, labels, h0, pos_weight, true, dropout_rate, dropout_seed, loss, logits);
}

ccsm_status ccsm_train_eval(ccsm_trainer* t, int n_sites, const ccsm_batch* batch, const int32_t* labels, const ccsm_h0* h0, float pos_weight,
                            float* loss, float* logits) {
    return run(t, n_sites, batch, labels, h0, pos_weight, false, 0.f, 0, loss, logits);
}

ccsm_status ccsm_train_step(ccsm_trainer* t, float lr, float beta1, float beta2, float eps, float max_norm, float* grad_norm) {
    if (!t) return fail(CCSM_ERR_INVALID_ARG, "trainer must be non-NULL");
    HIPCHK(hipSetDevice(t->device));
    float norm = 0.f;
    // |g|_2: per-block partial sums and a final block, both in a fixed order (the same gradients always give the same clip coefficient)
    ccsm_train::sumsq_partial_kernel<<<1024, 256, 0, t->stream>>>(t->grads, (long long)kOff.total, t->nrm_part);
    ccsm_train::sumsq_final_kernel<<<1, 256, 0, t->stream>>>(t->nrm_part, 1024, t->nrm_part + 1024);
    HIPCHK(hipMemcpyAsync(&norm, t->nrm_part + 1024, sizeof(float), hipMemcpyDeviceToHost, t->stream));
    HIPCHK(hipStreamSynchronize(t->stream));
    if (grad_norm) *grad_norm = norm;
    float clip = 1.f;
    if (max_norm > 0.f) {                                   // clip_grad_norm_: coef = max_norm / (norm + 1e-6), clamped to 1
        clip = max_norm / (norm + 1e-6f);
        if (clip > 1.f) clip = 1.f;
    }
    t->step += 1;
    const float bc1 = 1.0f - std::pow(beta1, (float)t->step), bc2 = 1.0f - std::pow(beta2, (float)t->step);
    adam_kernel<<<blocks(kOff.total), 256, 0, t->stream>>>(t->params, t->grads, t->adam_m, t->adam_v, kOff.total, lr, beta1, beta2, eps, clip, bc1, bc2);
    HIPCHK(hipGetLastError());
    HIPCHK(hipStreamSynchronize(t->stream));
    return CCSM_OK;
}

ccsm_status ccsm_train_grad_ptr(ccsm_trainer* t, float** d_grads) {
    if (!t || !d_grads) return fail(CCSM_ERR_INVALID_ARG, "NULL argument");
    *d_grads = t->grads;
    return CCSM_OK;
}
ccsm_status ccsm_train_get_params(ccsm_trainer* t, float* host_flat) {
    if (!t || !host_flat) return fail(CCSM_ERR_INVALID_ARG, "NULL argument");
    HIPCHK(hipSetDevice(t->device));
    HIPCHK(hipStreamSynchronize(t->stream));
    HIPCHK(hipMemcpy(host_flat, t->params, sizeof(float) * kOff.total, hipMemcpyDeviceToHost));
    return CCSM_OK;
}
ccsm_status ccsm_train_set_params(ccsm_trainer* t, const float* host_flat) {
    if (!t || !host_flat) return fail(CCSM_ERR_INVALID_ARG, "NULL argument");
    HIPCHK(hipSetDevice(t->device));
    HIPCHK(hipStreamSynchronize(t->stream));
    HIPCHK(hipMemcpy(t->params, host_flat, sizeof(float) * kOff.total, hipMemcpyHostToDevice));
    return CCSM_OK;
}
long ccsm_train_fused_fallbacks(const ccsm_trainer* t) { return t ? t->fused_fallbacks : 0; }

ccsm_status ccsm_train_selftest_gemm(int device, int t_a, int t_b, int M, int N, int K, float alpha, const float* A, int lda, const float* B,
                                     int ldb, float beta, float* C, int ldc, int grad_a) {
    if (!A || !B || !C || M <= 0 || N <= 0 || K <= 0) return fail(CCSM_ERR_INVALID_ARG, "selftest_gemm: bad arguments");
    HIPCHK(hipSetDevice(device));
    const size_t na = (size_t)(t_a ? K : M) * lda, nb = (size_t)(t_b ? N : K) * ldb, nc = (size_t)M * ldc;
    float *dA = nullptr, *dB = nullptr, *dC = nullptr;
    unsigned* amax = nullptr;
    HIPCHK(hipMalloc(&dA, na * 4)); HIPCHK(hipMalloc(&dB, nb * 4)); HIPCHK(hipMalloc(&dC, nc * 4)); HIPCHK(hipMalloc(&amax, 4));
    HIPCHK(hipMemcpy(dA, A, na * 4, hipMemcpyHostToDevice)); HIPCHK(hipMemcpy(dB, B, nb * 4, hipMemcpyHostToDevice));
    HIPCHK(hipMemcpy(dC, C, nc * 4, hipMemcpyHostToDevice));
    HIPCHK(ccsm_train::gemm_s3_init());
    HIPCHK(ccsm_train::gemm_s3(nullptr, t_a != 0, t_b != 0, M, N, K, alpha, dA, lda, 0, dB, ldb, 0, beta, dC, ldc, 0, 1, grad_a ? amax : nullptr));
    HIPCHK(hipDeviceSynchronize());
    HIPCHK(hipMemcpy(C, dC, nc * 4, hipMemcpyDeviceToHost));
    (void)hipFree(dA); (void)hipFree(dB); (void)hipFree(dC); (void)hipFree(amax);
    return CCSM_OK;
}

ccsm_status ccsm_train_get_grads(ccsm_trainer* t, float* host_flat) {
    if (!t || !host_flat) return fail(CCSM_ERR_INVALID_ARG, "NULL argument");
    HIPCHK(hipSetDevice(t->device));
    HIPCHK(hipStreamSynchronize(t->stream));
    HIPCHK(hipMemcpy(host_flat, t->grads, sizeof(float) * kOff.total, hipMemcpyDeviceToHost));
    return CCSM_OK;
}

}  // extern "C"
