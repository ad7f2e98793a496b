// linear.cu — the fully connected layer: y = act(x w + bias) + residual, and its backward pass.
//
//   forward   z = x w + bias,  y = act(z) + residual                    x [M,K], w [K,N] (in, out: as the framework stores weights)
//   backward  dz = dy act'(z);  dx = dz w^T;  dw = x^T dz;  dbias = sum over rows of dz
//
// Three ways, by size: a few rows on the CUDA cores with the weights streamed once (k_linear_few); small products in one launch on the CUDA
// cores (layer_small.cuh); the rest on the matrix engine (hgemm.cuh), f16 operands as they lie in memory, f32 ones as two f16 planes that
// kernels of this file make first.  Forward 4096 x 1024 -> 4096, f32, gelu, z kept: 121 us, 17 of them the planes; its backward pass
// 255 us: dz and its planes 40, x's 31, w's 8, bias 7, the two products 166.
#include "hgemm.cuh"
#include "layer_common.cuh"
#include "layer_host.h"
#include "layer_small.cuh"
#include "state.h"

namespace thc {

void *layer_scratch(const char *who, uint64_t bytes) {
    void *p = scratch_reserve(bytes);
    if (scratch_short(bytes)) { set_error("%s: library scratch had to grow inside the captured step: run the step once before capturing it", who); return nullptr; }
    return p;
}

bool layer_buffers(const char *who, const uint32_t *ins, const uint64_t *in_need, int n_in, int in_required,
                   const uint32_t *outs, const uint64_t *out_need, int n_out, int out_required, uint32_t inplace) {
    for (int side = 0; side < 2; side++) {
        const uint32_t *ids = side ? outs : ins;
        const uint64_t *need = side ? out_need : in_need;
        for (int i = 0; i < (side ? n_out : n_in); i++) {
            if (ids[i] == 0) {
                if (i < (side ? out_required : in_required)) { set_error("%s: a required buffer is missing", who); return false; }
                continue;
            }
            if (ids[i] >= THC_MAX_BUFS || !g.bufs[ids[i]].live) { set_error("%s: buffer id %u is not live", who, ids[i]); return false; }
            if (g.bufs[ids[i]].bytes < need[i]) { set_error("%s: buffer %u is too small", who, ids[i]); return false; }
        }
    }
    for (int i = 0; i < n_out; i++) {
        if (!outs[i]) continue;
        for (int j = 0; j < i; j++) if (outs[j] == outs[i]) { set_error("%s: two outputs are the same buffer %u", who, outs[i]); return false; }
        for (int j = 0; j < n_in; j++)
            if (ins[j] == outs[i] && !(i == 0 && (inplace >> j & 1u))) { set_error("%s: buffer %u is both input and output", who, outs[i]); return false; }
    }
    return true;
}

// ---- operands ----
// f32 operands become planes of x 2^s (hgemm.cuh).  The scale belongs to a row of memory, so that a row is read once, kept in
// registers while its largest value is found, and written as planes.  Where the contraction runs along those rows
// (x, dz and, for dx, w) the result is scaled back in the epilogue; where it runs across them, the other operand takes the
// inverse scales before it is split itself:
//   forward   w [K,N] by rows k: w' = w 2^s_k;           x' = x 2^-s_k, then scaled by its own rows m
//   dw        dz [M,N] by rows m: dz' = dz 2^s_m;        x' = x 2^-s_m, then scaled by its columns k (over m)
// Values below 2^-40 of the largest in their row (column) are rounded to that step.  An infinity in an f32 operand of the
// matrix engine gives NaN where it takes part, as in the framework's other contractions: its low part is no number.
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }       // -126 <= e <= 127; 0 at -127
__device__ __forceinline__ float finite_abs(float v) { v = fabsf(v); return v <= 3.402823466e38f ? v : 0.0f; }
// the exponent s that puts `top` into [2^14, 2^15); rows below 2^-112 keep fewer bits.  A row of zeros gets 127, whose way back is a factor
// of 0: what the other operand has beside it (a masked token's values) has no part in that operand's own scale.
__device__ __forceinline__ int scale_for(float top) {
    if (top == 0.0f) return 127;
    const int s = 14 - ((int)(__float_as_uint(top) >> 23) - 127);
    return s > 126 ? 126 : s;
}
// what a row's values are
template <typename T> struct RowsOf {                  // a matrix, its columns times 2^-shift
    const T *p; const int *shift; uint32_t cols;
    template <int VEC> __device__ void load(uint64_t row, uint32_t c, float (&v)[VEC]) const {
        load_vec<VEC>(p + row * cols + c, v);
        if (shift) {
#pragma unroll
            for (int j = 0; j < VEC; j++) v[j] *= pow2(-shift[c + j]);
        }
    }
};
template <typename T> struct GradOf {                  // dz = dy act'(z)
    const T *dy, *z; uint32_t cols, act;
    template <int VEC> __device__ void load(uint64_t row, uint32_t c, float (&v)[VEC]) const {
        load_vec<VEC>(dy + row * cols + c, v);
        if (act != THC_ACT_NONE) {
            float q[VEC];
            load_vec<VEC>(z + row * cols + c, q);
            act_slopes<VEC>(act, v, q);
        }
    }
};

struct Planes {
    __half *hi, *lo; uint64_t pitch; int *exps; float *sums;       // any may be null; exps null: unscaled
    uint32_t *clear; uint32_t n_clear;                             // words to be zeroed for a later kernel
};

__device__ __forceinline__ float block_max(float v, float *red) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < 8; w++) v = fmaxf(v, red[w]);
    return v;
}
// Blocks walk over rows, U units of VEC values a thread in registers; sums[block][cols] = the block's column sums.
template <class Src, int VEC, int U>
__global__ void __launch_bounds__(256)
k_split_rows(const Src src, const Planes out, uint32_t rows, uint32_t cols) {
    depend();
    __shared__ float red[8];
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < out.n_clear; i += gridDim.x * 256) out.clear[i] = 0;
    float sum[U][VEC];
#pragma unroll
    for (int i = 0; i < U; i++)
#pragma unroll
        for (int j = 0; j < VEC; j++) sum[i][j] = 0.0f;
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        float v[U][VEC];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < U; i++) {
            const uint32_t c = (threadIdx.x + 256u * i) * VEC;
            if (c < cols) {
                src.template load<VEC>(row, c, v[i]);
#pragma unroll
                for (int j = 0; j < VEC; j++) { top = fmaxf(top, finite_abs(v[i][j])); sum[i][j] += v[i][j]; }
            }
        }
        float scale = 1.0f;
        if (out.exps) {
            const int s = scale_for(block_max(top, red));
            if (threadIdx.x == 0) out.exps[row] = s;
            scale = pow2(s);
        }
        if (out.hi) {
#pragma unroll
            for (int i = 0; i < U; i++) {
                const uint32_t c = (threadIdx.x + 256u * i) * VEC;
                if (c >= cols) continue;
#pragma unroll
                for (int j = 0; j < VEC; j++) v[i][j] *= scale;
                store_planes<VEC>(out.hi + row * out.pitch + c, out.lo ? out.lo + row * out.pitch + c : nullptr, v[i]);
            }
        }
    }
    if (out.sums) {
#pragma unroll
        for (int i = 0; i < U; i++)
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const uint32_t c = (threadIdx.x + 256u * i) * VEC + j;
                if (c < cols) out.sums[(uint64_t)blockIdx.x * cols + c] = sum[i][j];
            }
    }
}
// rows longer than a block's registers: the values are made twice, the sums by k_grad_sums
template <class Src>
__global__ void __launch_bounds__(256)
k_split_long_rows(const Src src, const Planes out, uint32_t rows, uint32_t cols) {
    depend();
    __shared__ float red[8];
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < out.n_clear; i += gridDim.x * 256) out.clear[i] = 0;
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        float v[1], top = 0.0f;
        for (uint32_t c = threadIdx.x; c < cols; c += 256) { src.template load<1>(row, c, v); top = fmaxf(top, finite_abs(v[0])); }
        float scale = 1.0f;
        if (out.exps) {
            const int s = scale_for(block_max(top, red));
            if (threadIdx.x == 0) out.exps[row] = s;
            scale = pow2(s);
        }
        for (uint32_t c = threadIdx.x; c < cols; c += 256) {
            src.template load<1>(row, c, v);
            v[0] *= scale;
            store_planes<1>(out.hi + row * out.pitch + c, out.lo ? out.lo + row * out.pitch + c : nullptr, v);
        }
    }
}
template <class Src>
__global__ void __launch_bounds__(256)
k_grad_sums(const Src src, float *sums, uint32_t rows, uint32_t cols) {
    depend();
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float v[1], s = 0.0f;
    for (uint64_t row = blockIdx.y; row < rows; row += gridDim.y) { src.template load<1>(row, c, v); s += v[0]; }
    sums[(uint64_t)blockIdx.y * cols + c] = s;
}
// Scales by columns: the largest |x 2^-shift[row]| of each column, as bits (which order as the values do, so the order of the atomics does
// not matter), then the planes.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
k_col_tops(const T *x, const int *shift, uint32_t *tops, uint32_t rows, uint32_t cols) {
    depend();
    const uint32_t c = (blockIdx.x * 256 + threadIdx.x) * VEC;
    if (c >= cols) return;
    float top[VEC] = {};
#pragma unroll 8
    for (uint64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        float v[VEC];
        load_vec<VEC>(x + row * cols + c, v);
        const float f = pow2(-shift[row]);
#pragma unroll
        for (int j = 0; j < VEC; j++) top[j] = fmaxf(top[j], finite_abs(v[j] * f));
    }
#pragma unroll
    for (int j = 0; j < VEC; j++) atomicMax(tops + c + j, __float_as_uint(top[j]));
}
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
k_split_cols(const T *x, const int *shift, const uint32_t *tops, const Planes out, uint32_t rows, uint32_t cols) {
    depend();
    const uint32_t c = (blockIdx.x * 256 + threadIdx.x) * VEC;
    if (c >= cols) return;
    float scale[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        const int s = scale_for(__uint_as_float(tops[c + j]));
        if (blockIdx.y == 0) out.exps[c + j] = s;
        scale[j] = pow2(s);
    }
#pragma unroll 4
    for (uint64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        float v[VEC];
        load_vec<VEC>(x + row * cols + c, v);
        const float f = pow2(-shift[row]);
#pragma unroll
        for (int j = 0; j < VEC; j++) v[j] = v[j] * f * scale[j];
        store_planes<VEC>(out.hi + row * out.pitch + c, out.lo ? out.lo + row * out.pitch + c : nullptr, v);
    }
}

constexpr uint32_t ROW_VALUES = 8192;                  // a block of k_split_rows holds so many
template <class Src>
static void split_rows(const Src &src, const Planes &out, uint32_t rows, uint32_t cols, uint32_t blocks, const char *name) {
    profile_begin();
    if (cols > ROW_VALUES) {
        if (out.hi) { chain(k_split_long_rows<Src>, dim3(grid_for(rows, 1, 8)), 256, 0, src, out, rows, cols); after_launch(name); profile_begin(); }
        if (out.sums) { chain(k_grad_sums<Src>, dim3((cols + 255) / 256, blocks), 256, 0, src, out.sums, rows, cols); after_launch(name); }
        return;
    }
    if (cols % 4 == 0) {
        if (cols <= 1024) chain(k_split_rows<Src, 4, 1>, dim3(blocks), 256, 0, src, out, rows, cols);
        else if (cols <= 4096) chain(k_split_rows<Src, 4, 4>, dim3(blocks), 256, 0, src, out, rows, cols);
        else chain(k_split_rows<Src, 4, 8>, dim3(blocks), 256, 0, src, out, rows, cols);
    } else if (cols <= 1024) chain(k_split_rows<Src, 1, 4>, dim3(blocks), 256, 0, src, out, rows, cols);
    else chain(k_split_rows<Src, 1, 32>, dim3(blocks), 256, 0, src, out, rows, cols);
    after_launch(name);
}
static uint32_t split_blocks(uint32_t rows) { return rows < (1u << 30) ? rows : 1u << 30; }      // a row each
static uint32_t col_runs(uint32_t rows, uint32_t cols, uint32_t vec) {      // every how many rows a thread of k_col_tops looks: two blocks an SM, as the columns' maxima meet in atomics; eight rows a thread at least
    const uint32_t across = (cols / vec + 255) / 256, most = (rows + 7) / 8;
    uint32_t n = (uint32_t)g.sm_count * 2 / across;
    if (n > most) n = most;
    return n < 1 ? 1 : n > 65535 ? 65535 : n;
}

// scratch of one call, cut into pieces
struct Cut {
    uint64_t at = 0;
    uint8_t *base = nullptr;
    template <typename T> T *take(uint64_t n) { T *p = (T *)(base + at); at += (n * sizeof(T) + 255) & ~255ull; return p; }
};
// (rows of 64 values: the matrix engine may read them by blocks of 64 across)
static Planes take_planes(Cut &c, uint32_t rows, uint32_t cols, bool lo, bool exps, uint32_t n_exps) {
    Planes p{};
    p.pitch = (cols + 63u) & ~63ull;
    p.hi = c.take<__half>(rows * p.pitch * (lo ? 2 : 1));
    p.lo = lo ? p.hi + rows * p.pitch : nullptr;
    p.exps = exps ? c.take<int>(n_exps) : nullptr;
    return p;
}
static hg::Operand operand(const Planes &p, bool mn) { return hg::Operand{p.hi, p.pitch, p.lo ? (uint64_t)(p.lo - p.hi) : 0, mn}; }

// ---- epilogues: what a layer stores, and a gradient ----
template <typename T, int V, int R> __device__ __forceinline__ void store_rows(T *to, hg::Rows r, uint32_t n, uint32_t N, const float (&v)[R][V]) {
    T *p = to + (uint64_t)r.first * N + n;
    const uint64_t step = (uint64_t)r.step * N;
#pragma unroll
    for (uint32_t i = 0; i < R; i++, p += step) if (r.first + i * r.step < r.end) store_vec<V>(p, v[i]);
}
template <typename T, uint32_t ACT> struct LayerEpi {  // act(sum 2^-exps[m] + bias) + residual
    static constexpr bool mirrors = false, long_start = false, heavy = ACT == THC_ACT_GELU || ACT == THC_ACT_SILU;
    T *out, *z; const T *bias, *residual; const int *exps; uint32_t N;
    float bias_n[4];                                   // of the lane's columns
    __device__ bool wide() const { return N % 4 == 0; }
    __device__ float row_factor(uint32_t m) const { return exps ? pow2(-exps[m]) : 1.0f; }
    __device__ void touch(uint32_t m, uint32_t n, uint32_t cols) const { if (residual) hg::touch_row(residual + (uint64_t)m * N, n, cols, N); }
    template <int V> __device__ void column(uint32_t n) {
#pragma unroll
        for (int j = 0; j < V; j++) bias_n[j] = bias ? to_f32(bias[n + j]) : 0.0f;
    }
    template <int V> __device__ void fetch(uint32_t m, uint32_t n, float (&x)[V]) const { if (residual) load_vec<V>(residual + (uint64_t)m * N + n, x); }
    template <int V, int R> __device__ void put(hg::Rows r, uint32_t n, float (&v)[R][V], const float (&x)[R][V], uint32_t) const {
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int j = 0; j < V; j++) v[i][j] += bias_n[j];
        if (z) store_rows<T, V, R>(z, r, n, N, v);
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int j = 0; j < V; j++) { v[i][j] = act_value(ACT, v[i][j]); if (residual) v[i][j] += x[i][j]; }
        store_rows<T, V, R>(out, r, n, N, v);
    }
};
template <typename T, bool COLS> struct GradEpi {      // sum 2^(-exps[m] - col_exps[n])
    static constexpr bool mirrors = false, long_start = false, heavy = false;
    T *out; const int *exps, *col_exps; uint32_t N;
    int exp_n[4];
    __device__ bool wide() const { return N % 4 == 0; }
    __device__ float row_factor(uint32_t m) const { return !COLS && exps ? pow2(-exps[m]) : 1.0f; }
    __device__ void touch(uint32_t, uint32_t, uint32_t) const {}
    template <int V> __device__ void column(uint32_t n) {
        if constexpr (COLS) {
#pragma unroll
            for (int j = 0; j < V; j++) exp_n[j] = col_exps[n + j];
        }
    }
    template <int V> __device__ void fetch(uint32_t m, uint32_t, float (&x)[V]) const { if constexpr (COLS) x[0] = __int_as_float(exps[m]); }
    template <int V, int R> __device__ void put(hg::Rows r, uint32_t n, float (&v)[R][V], const float (&x)[R][V], uint32_t) const {
        if constexpr (COLS) {                          // up to 252 either way: two exact factors
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int j = 0; j < V; j++) { const int e = -__float_as_int(x[i][0]) - exp_n[j], h = e >> 1; v[i][j] = v[i][j] * pow2(h) * pow2(e - h); }
        }
        store_rows<T, V, R>(out, r, n, N, v);
    }
};

// ---- few rows: the weights are what is read, once, and the arithmetic is the CUDA cores' ----
// A cluster of eight blocks takes 32 V columns of w and all of K: each block an eighth of K, each of its eight warps every eighth row of that,
// a lane V neighbouring columns of MR rows of x.  The warps' sums meet in shared memory, the blocks' in the cluster's, in a fixed order;
// each block then finishes an eighth of the columns.  x comes through shared memory, FEW_K of its columns at a time.
// Bound by memory: K N values once.  V = 4: a lane copies its own weights to shared memory, FEW_RING groups of four rows ahead (16 KB
// of f16 or 32 KB of f32 in flight per block, and no registers: as plain loads the compiler kept two or three in flight, and 4096 x 4096 f32
// times one row took 32 us).  V = 1, for rows of w that are not aligned to four values: plain loads.
constexpr uint32_t FEW_K = 512, FEW_CLUSTER = 8, FEW_RING = 4;
template <typename T, int MR, int V> static constexpr uint32_t few_smem() {
    return FEW_K * MR * 4 + (V == 4 && 8 * FEW_RING * 4 * 32 * V * sizeof(T) > 8u * MR * 32 * V * 4 ? 8 * FEW_RING * 4 * 32 * V * (uint32_t)sizeof(T) : 8u * MR * 32 * V * 4);
}
template <typename T> __device__ __forceinline__ void copy4(uint32_t dst, const T *src) {
    if constexpr (sizeof(T) == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
template <typename T, int MR, int V>
__global__ void __cluster_dims__(1, FEW_CLUSTER, 1) __launch_bounds__(256)
k_linear_few(T *y, T *z, const T *x, const T *w, const T *bias, const T *residual, uint32_t M, uint32_t K, uint32_t N, uint32_t act) {
    depend();
    constexpr uint32_t COLS = 32 * V;
    extern __shared__ float few[];
    float (*xs)[MR] = reinterpret_cast<float (*)[MR]>(few);                      // [FEW_K]
    float (*sums)[MR][COLS] = reinterpret_cast<float (*)[MR][COLS]>(few + FEW_K * MR);   // [8], where the ring was
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, rank = blockIdx.y % FEW_CLUSTER;
    const uint32_t n = blockIdx.x * COLS + lane * V, m0 = blockIdx.y / FEW_CLUSTER * MR;
    const uint32_t share = (K + FEW_CLUSTER - 1) / FEW_CLUSTER, k_begin = rank * share < K ? rank * share : K, k_end = k_begin + share < K ? k_begin + share : K;
    const uint64_t down = (uint64_t)8 * N;
    // this lane's place in its warp's ring: row r of group g at + (g * 4 + r) * COLS values
    const T *ring = reinterpret_cast<const T *>(few + FEW_K * MR) + warp * (FEW_RING * 4 * COLS) + lane * V;
    float acc[MR][V];
#pragma unroll
    for (int i = 0; i < MR; i++)
#pragma unroll
        for (int j = 0; j < V; j++) acc[i][j] = 0.0f;
    for (uint32_t k0 = k_begin; k0 < k_end; k0 += FEW_K) {
        const uint32_t nk = k_end - k0 < FEW_K ? k_end - k0 : FEW_K;
        const uint32_t mine = n < N && warp < nk ? (nk - warp + 7) / 8 : 0;           // rows k0 + warp + 8 i
        const T *p = w + (uint64_t)(k0 + warp) * N + n;
        if constexpr (V == 4) {
#pragma unroll
            for (uint32_t gr = 0; gr < FEW_RING - 1; gr++) {
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) if (gr * 4 + r < mine) copy4(hg::smem32(ring + (gr * 4 + r) * COLS), p + (gr * 4 + r) * down);
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
        }
        __syncthreads();
        for (uint32_t u = threadIdx.x; u < MR * FEW_K; u += 256) {
            const uint32_t i = u / FEW_K, k = u % FEW_K;
            if (k < nk) xs[k][i] = m0 + i < M ? to_f32(x[(uint64_t)(m0 + i) * K + k0 + k]) : 0.0f;
        }
        __syncthreads();
        if constexpr (V == 4) {
            for (uint32_t i0 = 0, at = 0; i0 < mine; i0 += 4, at = (at + 1) % FEW_RING) {
                const uint32_t ahead = i0 + 4 * (FEW_RING - 1), to = (at + FEW_RING - 1) % FEW_RING;
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) if (ahead + r < mine) copy4(hg::smem32(ring + (to * 4 + r) * COLS), p + (ahead + r) * down);
                asm volatile("cp.async.commit_group;" ::: "memory");
                asm volatile("cp.async.wait_group %0;" ::"n"(FEW_RING - 1) : "memory");
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) {
                    if (i0 + r >= mine) break;
                    float v[V];
                    load_vec<V>(ring + (at * 4 + r) * COLS, v);
                    const float *xk = xs[warp + 8 * (i0 + r)];
#pragma unroll
                    for (int i = 0; i < MR; i++)
#pragma unroll
                        for (int j = 0; j < V; j++) acc[i][j] += xk[i] * v[j];
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        } else {
#pragma unroll 8
            for (uint32_t i0 = 0; i0 < mine; i0++) {
                const float v = to_f32(p[i0 * down]);
                const float *xk = xs[warp + 8 * i0];
#pragma unroll
                for (int i = 0; i < MR; i++) acc[i][0] += xk[i] * v;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MR; i++)
#pragma unroll
        for (int j = 0; j < V; j++) sums[warp][i][lane * V + j] = acc[i][j];
    __syncthreads();
    for (uint32_t u = threadIdx.x; u < MR * COLS; u += 256) {
        const uint32_t i = u / COLS, c = u % COLS;
        float s = sums[0][i][c];
#pragma unroll
        for (int q = 1; q < 8; q++) s += sums[q][i][c];
        sums[0][i][c] = s;
    }
    hg::cluster_sync();
    constexpr uint32_t MINE = COLS / FEW_CLUSTER;
    for (uint32_t u = threadIdx.x; u < MR * MINE; u += 256) {
        const uint32_t i = u / MINE, c = rank * MINE + u % MINE, col = blockIdx.x * COLS + c, m = m0 + i;
        const uint32_t here = hg::smem32(&sums[0][i][c]);
        float s = 0.0f;
#pragma unroll
        for (uint32_t r = 0; r < FEW_CLUSTER; r++) {
            float q;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(q) : "r"(hg::in_cta(here, r)) : "memory");
            s += q;
        }
        if (col >= N || m >= M) continue;
        const uint64_t at = (uint64_t)m * N + col;
        if (bias) s += to_f32(bias[col]);
        if (z) put_f32(z + at, s);
        s = act_value(act, s);
        if (residual) s += to_f32(residual[at]);
        put_f32(y + at, s);
    }
    hg::cluster_sync();                                // no block leaves while another reads its sums
}

// an f16 matrix as it is, or copied to a pitch that tile loads can take
static hg::Operand f16_operand(Cut &c, const __half *p, uint32_t rows, uint32_t cols, bool mn, bool copy) {
    if (cols % 8 == 0) return hg::Operand{p, cols, 0, mn};
    const Planes q = take_planes(c, rows, cols, false, false, 0);
    if (copy) split_rows(RowsOf<__half>{p, nullptr, cols}, q, rows, cols, split_blocks(rows), "layer_operand");
    return operand(q, mn);
}

template <typename T, int MR, int V>
static void few_rows_as(void *y, void *z, const void *x, const void *w, const void *bias, const void *residual, uint32_t M, uint32_t K, uint32_t N, uint32_t act) {
    static int seen = -1;
    if (first_on_device(seen)) THC_CUDA_OK(cudaFuncSetAttribute(k_linear_few<T, MR, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)few_smem<T, MR, V>()));
    layer_estimate(2.0 * M * K * N, ((double)K * N + (double)M * K + (double)M * N) * sizeof(T));
    chain(k_linear_few<T, MR, V>, dim3((N + 32 * V - 1) / (32 * V), (M + MR - 1) / MR * FEW_CLUSTER), 256, few_smem<T, MR, V>(), (T *)y, (T *)z, (const T *)x, (const T *)w, (const T *)bias, (const T *)residual, M, K, N, act);
}
// Up to how many rows the kernel above is taken, from 4096 x 4096 weights.  f32: 15 us for one row, 19 for eight, 37 for 16, 53 for 24, 68 for 32;
// the matrix engine, which splits the weights into planes first, 65 whatever the rows up to 128.  f16: 11 us for one row, 14 for
// four, 18 for eight; the engine 18.  Where rows of w are not aligned, the engine copies them first: 16 rows for either type.
template <typename T> static bool few_rows(void *y, void *z, const void *x, const void *w, const void *bias, const void *residual, uint32_t M, uint32_t K, uint32_t N, uint32_t act) {
    profile_begin();
    if (N % 4) {
        if (M > 16) return false;
        if (M <= 2) few_rows_as<T, 2, 1>(y, z, x, w, bias, residual, M, K, N, act);
        else few_rows_as<T, 8, 1>(y, z, x, w, bias, residual, M, K, N, act);
    } else {
        if (M > (sizeof(T) == 4 ? 24 : 4)) return false;
        if (M == 1) few_rows_as<T, 1, 4>(y, z, x, w, bias, residual, M, K, N, act);
        else if (M <= 4) few_rows_as<T, 4, 4>(y, z, x, w, bias, residual, M, K, N, act);
        else if constexpr (sizeof(T) == 4) few_rows_as<T, 8, 4>(y, z, x, w, bias, residual, M, K, N, act);
    }
    after_launch("linear_few");
    return true;
}

// Up to how many products (M K N) the one-launch kernels of layer_small.cuh are taken.  Forward, f32: 512 x 400 x 120 in 9 us, the engine with its
// operands' planes 16; 512 x 512 x 512 in 20 and 18; in f16 the engine needs no planes and is as fast at 64 x 64 x 64 (6 us), except for rows
// that it has to copy to an aligned pitch first (265 x 177 x 221 18 us).  Backward:
// f32 256^3 12 and 31 us, 512 x 400 x 120 22 and 35, 1024 x 400 x 120 44 and 37; f16 17 and 27, 29 and 30; with 2000 rows, over which dw sums,
// 32 and 34, 49 and 32.
constexpr double SMALL_FORWARD = 1e8, SMALL_FORWARD_COPIED = 2e7, SMALL_BACKWARD_F32 = 4e7, SMALL_BACKWARD_F16 = 2e7;
constexpr uint32_t SMALL_BACKWARD_ROWS = 1024;

template <typename T>
static bool linear_forward(void *y, void *z, const void *x, const void *w, const void *bias, const void *residual, uint32_t M, uint32_t K, uint32_t N, uint32_t act) {
    constexpr bool F = sizeof(T) == 4;
    if (few_rows<T>(y, z, x, w, bias, residual, M, K, N, act)) return true;
    if ((double)M * K * N <= (F ? SMALL_FORWARD : K % 8 || N % 8 ? SMALL_FORWARD_COPIED : 0)) {
        Small<T> S{};
        S.x = (const T *)x; S.w = (const T *)w; S.bias = (const T *)bias; S.residual = (const T *)residual; S.y = (T *)y; S.z_out = (T *)z;
        S.M = M; S.K = K; S.N = N; S.act = act;
        const uint32_t tiles = ((M + SMALL_ROWS - 1) / SMALL_ROWS) * ((N + 31) / 32), ranks = small_ranks(tiles, K, 8);
        layer_estimate(2.0 * M * K * N, ((double)K * N + (double)M * K + (double)M * N) * sizeof(T));
        profile_begin();
        chain_cluster(ranks, k_small_forward<T>, dim3(tiles, ranks), 128, 0, S);
        after_launch("linear_small");
        return true;
    }
    const hg::Plan plan = hg::plan(M, N, K, F, false);
    const int *exps = nullptr;
    Cut c;
    hg::Operand A{}, B{};
    float *partial = nullptr;
    for (int pass = 0; pass < 2; pass++) {             // the first pass measures
        if (pass) {
            c.base = (uint8_t *)layer_scratch("linear", c.at);
            if (!c.base && c.at) return false;
            c.at = 0;
        }
        partial = c.take<float>(plan.partial_bytes / 4);
        if constexpr (F) {
            const Planes pw = take_planes(c, K, N, true, true, K), px = take_planes(c, M, K, true, true, M);
            A = operand(px, false); B = operand(pw, true);
            exps = px.exps;
            if (pass) {
                split_rows(RowsOf<float>{(const float *)w, nullptr, N}, pw, K, N, split_blocks(K), "layer_operand");
                split_rows(RowsOf<float>{(const float *)x, pw.exps, K}, px, M, K, split_blocks(M), "layer_operand");
            }
        } else {
            A = f16_operand(c, (const __half *)x, M, K, false, pass);
            B = f16_operand(c, (const __half *)w, K, N, true, pass);
        }
    }
    const auto run = [&](auto epi) { hg::product(A, B, M, N, K, plan, partial, epi, false, "linear"); };
    T *ty = (T *)y, *tz = (T *)z;
    const T *tb = (const T *)bias, *tr = (const T *)residual;
    switch (act) {
        case THC_ACT_RELU: run(LayerEpi<T, THC_ACT_RELU>{ty, tz, tb, tr, exps, N, {}}); break;
        case THC_ACT_GELU: run(LayerEpi<T, THC_ACT_GELU>{ty, tz, tb, tr, exps, N, {}}); break;
        case THC_ACT_SILU: run(LayerEpi<T, THC_ACT_SILU>{ty, tz, tb, tr, exps, N, {}}); break;
        default:           run(LayerEpi<T, THC_ACT_NONE>{ty, tz, tb, tr, exps, N, {}}); break;
    }
    return true;
}

template <typename T>
static bool linear_backward(void *dx, void *dw, void *dbias, const void *dy, const void *z, const void *x, const void *w, uint32_t M, uint32_t K, uint32_t N, uint32_t act) {
    constexpr bool F = sizeof(T) == 4;
    if ((double)M * K * N <= (F ? SMALL_BACKWARD_F32 : SMALL_BACKWARD_F16) && M <= SMALL_BACKWARD_ROWS) {
        Small<T> S{};
        S.x = (const T *)x; S.w = (const T *)w; S.dy = (const T *)dy; S.z_in = (const T *)z; S.dx = (T *)dx; S.dw = (T *)dw; S.dbias = (T *)dbias;
        S.M = M; S.K = K; S.N = N; S.act = act;
        const uint32_t m = (M + SMALL_ROWS - 1) / SMALL_ROWS, k = (K + SMALL_ROWS - 1) / SMALL_ROWS, k32 = (K + 31) / 32, n = (N + 31) / 32;
        const uint32_t ranks = small_ranks((uint64_t)m * k32 + k * n, M > N ? M : N, 16);                  // (whatever is asked for)
        S.dx_tiles = dx ? m * k32 : 0;
        const uint32_t tiles = S.dx_tiles + (dw ? k * n : dbias ? n : 0);      // the bias's gradient comes from dw's first row of tiles
        layer_estimate(4.0 * M * K * N, 2.0 * ((double)K * N + (double)M * K + (double)M * N) * sizeof(T));
        profile_begin();
        chain_cluster(ranks, k_small_backward<T>, dim3(tiles, ranks), 128, 0, S);
        after_launch("linear_backward_small");
        return true;
    }
    const bool smooth = act == THC_ACT_GELU || act == THC_ACT_SILU;
    const bool scaled = F || smooth;                   // dz needs planes: f32, or f16 times a slope that is neither 0 nor 1
    const bool as_is = !F && act == THC_ACT_NONE && N % 8 == 0;
    const GradOf<T> grad{(const T *)dy, (const T *)z, N, act};
    const hg::Plan plan_x = hg::plan(M, K, N, scaled, false), plan_w = hg::plan(K, N, M, scaled, false);
    const uint32_t blocks = dbias ? grid_for(M, 1, 4) : split_blocks(M), sum_rows = N > ROW_VALUES ? (M < 16 ? M : 16) : blocks;
    Cut c;
    for (int pass = 0; pass < 2; pass++) {
        if (pass) {
            c.base = (uint8_t *)layer_scratch("linear_backward", c.at);
            if (!c.base && c.at) return false;
            c.at = 0;
        }
        float *partial = c.take<float>((plan_x.partial_bytes > plan_w.partial_bytes ? plan_x.partial_bytes : plan_w.partial_bytes) / 4);
        // dz, and its sums over rows
        Planes pz{};
        if (!as_is && (dx || dw)) pz = take_planes(c, M, N, scaled, scaled, M);
        if (scaled && dw) { pz.clear = c.take<uint32_t>(K); pz.n_clear = K; }
        pz.sums = dbias ? c.take<float>((uint64_t)sum_rows * N) : nullptr;
        if (pass && (pz.hi || pz.sums)) split_rows(grad, pz, M, N, N > ROW_VALUES && pz.sums ? sum_rows : blocks, "linear_backward_dz");
        if (pass && dbias) {
            profile_begin();
            chain(k_fold_rows<T>, dim3((N + 31) / 32, 1), 1024, 0, (T *)dbias, (T *)nullptr, (const float *)pz.sums, sum_rows, N);
            after_launch("linear_backward_bias");
        }
        const hg::Operand dz_k = as_is ? hg::Operand{(const __half *)dy, N, 0, false} : operand(pz, false);
        hg::Operand dz_mn = dz_k;
        dz_mn.mn = true;
        if (dx) {
            hg::Operand W{};
            const int *col_exps = nullptr;
            if constexpr (F) {
                const Planes pw = take_planes(c, K, N, true, true, K);
                if (pass) split_rows(RowsOf<float>{(const float *)w, nullptr, N}, pw, K, N, split_blocks(K), "layer_operand");
                W = operand(pw, false);
                col_exps = pw.exps;
            } else W = f16_operand(c, (const __half *)w, K, N, false, pass);
            if (pass) hg::product(dz_k, W, M, K, N, plan_x, partial, GradEpi<T, F>{(T *)dx, pz.exps, col_exps, K, {}}, false, "linear_backward_dx");
        }
        if (dw) {
            hg::Operand X{};
            const int *exps = nullptr;
            if (scaled) {                              // x takes dz's scales back
                const Planes px = take_planes(c, M, K, F, true, K);
                if (pass) {
                    const T *xs = (const T *)x;
                    const uint32_t vec = K % 4 == 0 ? 4 : 1;
                    const dim3 grid((K / vec + 255) / 256, col_runs(M, K, vec));
                    profile_begin();
                    if (vec == 4) {
                        chain(k_col_tops<T, 4>, grid, 256, 0, xs, pz.exps, pz.clear, M, K);
                        chain(k_split_cols<T, 4>, grid, 256, 0, xs, pz.exps, pz.clear, px, M, K);
                    } else {
                        chain(k_col_tops<T, 1>, grid, 256, 0, xs, pz.exps, pz.clear, M, K);
                        chain(k_split_cols<T, 1>, grid, 256, 0, xs, pz.exps, pz.clear, px, M, K);
                    }
                    after_launch("layer_operand");
                }
                X = operand(px, true);
                exps = px.exps;
            } else if constexpr (!F) X = f16_operand(c, (const __half *)x, M, K, true, pass);
            if (pass) hg::product(X, dz_mn, K, N, M, plan_w, partial, GradEpi<T, false>{(T *)dw, exps, nullptr, N, {}}, false, "linear_backward_dw");
        }
    }
    return true;
}

static bool linear_shape(const char *who, uint32_t M, uint32_t K, uint32_t N, uint32_t act, uint32_t dtype) {
    if (M == 0 || K == 0 || N == 0) { set_error("%s: empty shape", who); return false; }
    if (M > (1u << 30) || K > (1u << 30) || N > (1u << 30)) { set_error("%s: a dimension exceeds 2^30", who); return false; }
    if (dtype != THC_F32 && dtype != THC_F16) { set_error("%s: dtype %u is neither f32 nor f16", who, dtype); return false; }
    if (act > THC_ACT_SILU) { set_error("%s: unknown activation %u", who, act); return false; }
    return true;
}

}  // namespace thc

using namespace thc;

extern "C" {

int thvm_cuda_linear(uint32_t y, uint32_t z, uint32_t x, uint32_t w, uint32_t bias, uint32_t residual,
                     uint32_t M, uint32_t K, uint32_t N, uint32_t act, uint32_t dtype) {
    if (!linear_shape("linear", M, K, N, act, dtype)) return 1;
    const uint64_t sz = dtype == THC_F16 ? 2 : 4, mn = (uint64_t)M * N * sz;
    const uint32_t outs[2] = {y, z}, ins[4] = {x, w, bias, residual};
    const uint64_t out_need[2] = {mn, mn}, in_need[4] = {(uint64_t)M * K * sz, (uint64_t)K * N * sz, N * sz, mn};
    if (!layer_buffers("linear", ins, in_need, 4, 2, outs, out_need, 2, 1, 1u << 3)) return 1;
    const void *px = buf_checked(x, "linear(x)").ptr, *pw = buf_checked(w, "linear(w)").ptr;
    const void *pb = bias ? buf_checked(bias, "linear(bias)").ptr : nullptr, *pr = residual ? buf_checked(residual, "linear(residual)").ptr : nullptr;
    void *py = buf_for_output(y, "linear(y)", mn).ptr, *pz = z ? buf_for_output(z, "linear(z)", mn).ptr : nullptr;
    mark_device_written(y);
    if (z) mark_device_written(z);
    return (dtype == THC_F16 ? linear_forward<__half>(py, pz, px, pw, pb, pr, M, K, N, act) : linear_forward<float>(py, pz, px, pw, pb, pr, M, K, N, act)) ? 0 : 1;
}

int thvm_cuda_linear_backward(uint32_t dx, uint32_t dw, uint32_t dbias, uint32_t dy, uint32_t z, uint32_t x, uint32_t w,
                              uint32_t M, uint32_t K, uint32_t N, uint32_t act, uint32_t dtype) {
    if (!linear_shape("linear_backward", M, K, N, act, dtype)) return 1;
    if (!dx && !dw && !dbias) { set_error("linear_backward: no output asked for"); return 1; }
    if (act != THC_ACT_NONE && !z) { set_error("linear_backward: this activation needs the pre-activation z"); return 1; }
    if (dx && !w) { set_error("linear_backward: dx needs w"); return 1; }
    if (dw && !x) { set_error("linear_backward: dw needs x"); return 1; }
    if (act == THC_ACT_NONE) z = 0;
    const uint64_t sz = dtype == THC_F16 ? 2 : 4, mn = (uint64_t)M * N * sz, mk = (uint64_t)M * K * sz, kn = (uint64_t)K * N * sz;
    const uint32_t outs[3] = {dx, dw, dbias}, ins[4] = {dy, z, x, w};
    const uint64_t out_need[3] = {mk, kn, N * sz}, in_need[4] = {mn, mn, mk, kn};
    if (!layer_buffers("linear_backward", ins, in_need, 4, 1, outs, out_need, 3, 0, 0)) return 1;
    const void *pdy = buf_checked(dy, "linear_backward(dy)").ptr, *pz = z ? buf_checked(z, "linear_backward(z)").ptr : nullptr;
    const void *px = x ? buf_checked(x, "linear_backward(x)").ptr : nullptr, *pw = w ? buf_checked(w, "linear_backward(w)").ptr : nullptr;
    void *pdx = dx ? buf_for_output(dx, "linear_backward(dx)", mk).ptr : nullptr;
    void *pdw = dw ? buf_for_output(dw, "linear_backward(dw)", kn).ptr : nullptr;
    void *pdb = dbias ? buf_for_output(dbias, "linear_backward(dbias)", N * sz).ptr : nullptr;
    for (uint32_t id : outs) if (id) mark_device_written(id);
    return (dtype == THC_F16 ? linear_backward<__half>(pdx, pdw, pdb, pdy, pz, px, pw, M, K, N, act) : linear_backward<float>(pdx, pdw, pdb, pdy, pz, px, pw, M, K, N, act)) ? 0 : 1;
}

}  // extern "C"
