// layernorm.cu — layer norm over the last dim of a contiguous [rows, cols] tensor, forward and backward.
//
//   mean = sum x / cols,  rstd = 1 / sqrt(sum (x - mean)^2 / cols + eps),  y = (x - mean) rstd gamma + beta
//   xh = (x - mean) rstd,  g = dy gamma
//   dx = rstd (g - sum g / cols - xh sum(g xh) / cols),  dgamma = sum_rows dy xh,  dbeta = sum_rows dy
//
// All sums are f32 over f32 values whatever the storage type; only the stored results are rounded.  Both passes are
// bound by memory: forward reads x and writes y, backward reads x and dy and writes dx, each once.  16384 x 2048 f32: forward 45 us,
// 5.98 TB/s, 0.91 of the measured copy rate; backward 70 us, 5.73 TB/s, 0.87 (7 us of it add up 592 blocks' partial sums).
//
// A row belongs to a group of G threads, which keeps it in registers from the load to the store, so the deviation from
// the mean is summed in a second pass that costs no memory traffic.  The backward pass keeps, beside the row, the running
// column sums of dy xh and dy: a thread sees the same columns of every row its block visits.  Each block leaves one
// partial row of sums and k_fold_rows adds those in block order, so results do not depend on timing.
#include "layer_common.cuh"
#include "layer_host.h"
#include "state.h"

namespace thc {

// sum over the G threads of a row group; `red` has one slot per warp of the block
template <int G> __device__ __forceinline__ float group_sum(float v, float *red) {
    v = warp_sum(v);
    if constexpr (G > 32) {
        __syncthreads();                               // the slots' last readers are done
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < G / 32; w++) v += red[w];
    }
    return v;
}

// two sums at once
template <int G> __device__ __forceinline__ float2 group_sum2(float a, float b, float2 *red) {
    a = warp_sum(a); b = warp_sum(b);
    if constexpr (G > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int w = 0; w < G / 32; w++) { const float2 r = red[w]; a += r.x; b += r.y; }
    }
    return make_float2(a, b);
}

constexpr int NORM_BLOCK = 256;                        // threads of a block whose groups are single warps
// values of a row that a thread of the forward kernel holds: 32 where there are rows for all SMs, 8 where latency counts, with gamma and
// beta read beside x
constexpr int NORM_VALUES = 32, NORM_VALUES_FEW = 8;

// Forward.  G threads a row; blocks of G threads, or of NORM_BLOCK / 32 warps with a row each.
template <typename T, int VEC, int G, int VALUES>
__global__ void __launch_bounds__(G > 32 ? G : NORM_BLOCK)
k_norm(T *y, float *mean_out, float *rstd_out, const T *x, const T *gamma, const T *beta, uint32_t rows, uint32_t cols, float eps) {
    depend();
    constexpr int NV = VALUES / VEC;
    constexpr bool EARLY = VALUES == NORM_VALUES_FEW;
    __shared__ float red[G > 32 ? G / 32 : 1];
    const uint32_t t = G > 32 ? threadIdx.x : (threadIdx.x & 31u);
    const uint64_t row = G > 32 ? blockIdx.x : (uint64_t)blockIdx.x * (NORM_BLOCK / 32) + (threadIdx.x >> 5);
    if (row >= rows) return;                           // (whole warps, and only where a row is one warp's)
    const T *xr = x + row * cols;
    float v[NV][VEC], gm[EARLY ? NV : 1][VEC], bt[EARLY ? NV : 1][VEC];
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const uint32_t c = (t + (uint32_t)i * G) * VEC;
        if constexpr (EARLY) {
            if (gamma && c < cols) load_vec<VEC>(gamma + c, gm[i]);
            if (beta && c < cols) load_vec<VEC>(beta + c, bt[i]);
        }
        if (c < cols) load_vec<VEC>(xr + c, v[i]);
        else {
#pragma unroll
            for (int j = 0; j < VEC; j++) v[i][j] = 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < VEC; j++) s += v[i][j];
    const float mean = group_sum<G>(s, red) / (float)cols;
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++)
        if ((t + (uint32_t)i * G) * VEC < cols) {
#pragma unroll
            for (int j = 0; j < VEC; j++) { v[i][j] -= mean; q += v[i][j] * v[i][j]; }
        }
    const float rstd = 1.0f / sqrtf(group_sum<G>(q, red) / (float)cols + eps);
    T *yr = y + row * cols;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const uint32_t c = (t + (uint32_t)i * G) * VEC;
        if (c >= cols) continue;
        constexpr int AT = EARLY ? 1 : 0;
        if constexpr (!EARLY) {
            if (gamma) load_vec<VEC>(gamma + c, gm[0]);
            if (beta) load_vec<VEC>(beta + c, bt[0]);
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            float o = v[i][j] * rstd;
            if (gamma) o *= gm[AT * i][j];
            if (beta) o += bt[AT * i][j];
            v[i][j] = o;
        }
        store_vec<VEC>(yr + c, v[i]);
    }
    if (t == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
}

// Forward for rows that no block holds in registers: three passes over the row, the later two mostly from L2.
template <typename T>
__global__ void __launch_bounds__(1024)
k_norm_long(T *y, float *mean_out, float *rstd_out, const T *x, const T *gamma, const T *beta, uint32_t rows, uint32_t cols, float eps) {
    depend();
    __shared__ float red[32];
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * cols;
        float s = 0.0f;
        for (uint32_t c = threadIdx.x; c < cols; c += 1024) s += to_f32(xr[c]);
        const float mean = group_sum<1024>(s, red) / (float)cols;
        float q = 0.0f;
        for (uint32_t c = threadIdx.x; c < cols; c += 1024) { const float d = to_f32(xr[c]) - mean; q += d * d; }
        const float rstd = 1.0f / sqrtf(group_sum<1024>(q, red) / (float)cols + eps);
        for (uint32_t c = threadIdx.x; c < cols; c += 1024) {
            float o = (to_f32(xr[c]) - mean) * rstd;
            if (gamma) o *= to_f32(gamma[c]);
            if (beta) o += to_f32(beta[c]);
            put_f32(y + row * cols + c, o);
        }
        if (threadIdx.x == 0) {
            if (mean_out) mean_out[row] = mean;
            if (rstd_out) rstd_out[row] = rstd;
        }
    }
}

constexpr int NORM_BWD_VALUES = 8;                     // values of a row that a thread of the backward kernel holds

// Backward.  Blocks of R groups of G threads walk over the rows; partial[block][2][cols] gets the block's column sums.
template <typename T, int VEC, int G>
__global__ void __launch_bounds__(G > 32 ? G : NORM_BLOCK)
k_norm_bwd(T *dx, float *partial, const T *dy, const T *x, const T *gamma, const float *mean, const float *rstd, uint32_t rows, uint32_t cols) {
    depend();
    constexpr int NV = NORM_BWD_VALUES / VEC, R = G > 32 ? 1 : NORM_BLOCK / 32;
    __shared__ float2 red[G > 32 ? G / 32 : 1];
    __shared__ float fold[G > 32 ? 1 : NORM_BLOCK * NORM_BWD_VALUES];
    const uint32_t t = G > 32 ? threadIdx.x : (threadIdx.x & 31u), r0 = G > 32 ? 0u : threadIdx.x >> 5;
    float gm[NV][VEC], sg[NV][VEC], sb[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const uint32_t c = (t + (uint32_t)i * G) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; j++) { gm[i][j] = 1.0f; sg[i][j] = sb[i][j] = 0.0f; }
        if (gamma && c < cols) load_vec<VEC>(gamma + c, gm[i]);
    }
    const float inv = 1.0f / (float)cols;
    for (uint64_t row = (uint64_t)blockIdx.x * R + r0; row < rows; row += (uint64_t)gridDim.x * R) {
        const float mu = mean[row], rs = rstd[row];
        float xh[NV][VEC], d[NV][VEC];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const uint32_t c = (t + (uint32_t)i * G) * VEC;
            if (c < cols) { load_vec<VEC>(x + row * cols + c, xh[i]); load_vec<VEC>(dy + row * cols + c, d[i]); }
        }
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++)
            if ((t + (uint32_t)i * G) * VEC < cols) {
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    xh[i][j] = (xh[i][j] - mu) * rs;
                    sg[i][j] += d[i][j] * xh[i][j]; sb[i][j] += d[i][j];
                    d[i][j] *= gm[i][j];
                    s1 += d[i][j]; s2 += d[i][j] * xh[i][j];
                }
            }
        if (dx) {
            const float2 s = group_sum2<G>(s1, s2, red);
            const float m1 = s.x * inv, m2 = s.y * inv;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const uint32_t c = (t + (uint32_t)i * G) * VEC;
                if (c >= cols) continue;
#pragma unroll
                for (int j = 0; j < VEC; j++) d[i][j] = rs * (d[i][j] - m1 - xh[i][j] * m2);
                store_vec<VEC>(dx + row * cols + c, d[i]);
            }
        }
    }
    if (!partial) return;
    float *p = partial + (uint64_t)blockIdx.x * 2 * cols;
#pragma unroll
    for (int half = 0; half < 2; half++) {
        if constexpr (R > 1) {                         // the groups' sums in group order
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < VEC; j++) fold[threadIdx.x * NORM_BWD_VALUES + i * VEC + j] = half ? sb[i][j] : sg[i][j];
            __syncthreads();
            if (r0 == 0) {
#pragma unroll
                for (int i = 0; i < NV; i++)
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        float s = 0.0f;
                        for (int r = 0; r < R; r++) s += fold[(r * 32 + t) * NORM_BWD_VALUES + i * VEC + j];
                        if (half) sb[i][j] = s; else sg[i][j] = s;
                    }
            }
        }
        if (r0 == 0) {
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const uint32_t c = (t + (uint32_t)i * G) * VEC + (uint32_t)j;
                    if (c < cols) p[(uint64_t)half * cols + c] = half ? sb[i][j] : sg[i][j];
                }
        }
    }
}

// dx for rows that no block holds in registers: a pass for the two sums, a pass for the result
template <typename T>
__global__ void __launch_bounds__(1024)
k_norm_bwd_long(T *dx, const T *dy, const T *x, const T *gamma, const float *mean, const float *rstd, uint32_t rows, uint32_t cols) {
    depend();
    __shared__ float2 red[32];
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float mu = mean[row], rs = rstd[row];
        float s1 = 0.0f, s2 = 0.0f;
        for (uint32_t c = threadIdx.x; c < cols; c += 1024) {
            const float g = to_f32(dy[row * cols + c]) * (gamma ? to_f32(gamma[c]) : 1.0f);
            s1 += g; s2 += g * ((to_f32(x[row * cols + c]) - mu) * rs);
        }
        const float2 s = group_sum2<1024>(s1, s2, red);
        const float m1 = s.x / (float)cols, m2 = s.y / (float)cols;
        for (uint32_t c = threadIdx.x; c < cols; c += 1024) {
            const float g = to_f32(dy[row * cols + c]) * (gamma ? to_f32(gamma[c]) : 1.0f);
            put_f32(dx + row * cols + c, rs * (g - m1 - (to_f32(x[row * cols + c]) - mu) * rs * m2));
        }
    }
}
// column sums of the same: a block takes 256 columns and every gridDim.y-th row
template <typename T>
__global__ void __launch_bounds__(256)
k_norm_bwd_cols(float *partial, const T *dy, const T *x, const float *mean, const float *rstd, uint32_t rows, uint32_t cols) {
    depend();
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float sg = 0.0f, sb = 0.0f;
    for (uint64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float d = to_f32(dy[row * cols + c]);
        sg += d * ((to_f32(x[row * cols + c]) - mean[row]) * rstd[row]); sb += d;
    }
    partial[(uint64_t)blockIdx.y * 2 * cols + c] = sg;
    partial[((uint64_t)blockIdx.y * 2 + 1) * cols + c] = sb;
}

// ---- host ----
// threads of a row's group when each holds `values` of it: 32, 128, 256, 512 or 1024; 0 = none holds the row
static uint32_t norm_group(uint32_t cols, uint32_t values) {
    const uint32_t sizes[] = {32, 128, 256, 512, 1024};
    for (uint32_t g : sizes) if ((uint64_t)g * values >= cols) return g;
    return 0;
}

template <typename T, int VEC, int G, int VALUES>
static void norm_launch(void *y, float *mean, float *rstd, const void *x, const void *gamma, const void *beta, uint32_t rows, uint32_t cols, float eps) {
    const uint32_t per = G > 32 ? 1 : NORM_BLOCK / 32;
    chain(k_norm<T, VEC, G, VALUES>, dim3((rows + per - 1) / per), G > 32 ? G : NORM_BLOCK, 0, (T *)y, mean, rstd, (const T *)x, (const T *)gamma, (const T *)beta, rows, cols, eps);
}
template <typename T, int VEC, int VALUES>
static void norm_launch_g(uint32_t group, void *y, float *mean, float *rstd, const void *x, const void *gamma, const void *beta, uint32_t rows, uint32_t cols, float eps) {
    switch (group) {
        case 32:   norm_launch<T, VEC, 32, VALUES>(y, mean, rstd, x, gamma, beta, rows, cols, eps); break;
        case 128:  norm_launch<T, VEC, 128, VALUES>(y, mean, rstd, x, gamma, beta, rows, cols, eps); break;
        case 256:  norm_launch<T, VEC, 256, VALUES>(y, mean, rstd, x, gamma, beta, rows, cols, eps); break;
        case 512:  norm_launch<T, VEC, 512, VALUES>(y, mean, rstd, x, gamma, beta, rows, cols, eps); break;
        default:   norm_launch<T, VEC, 1024, VALUES>(y, mean, rstd, x, gamma, beta, rows, cols, eps); break;
    }
}
template <typename T>
static void norm_forward(void *y, float *mean, float *rstd, const void *x, const void *gamma, const void *beta, uint32_t rows, uint32_t cols, float eps) {
    constexpr int V = Vec16<T>::n;
    const uint32_t few = norm_group(cols, NORM_VALUES_FEW), group = norm_group(cols, NORM_VALUES);
    const bool wide = cols % V == 0;
    if (few && (uint64_t)rows * few <= (uint64_t)g.sm_count * 1024) {     // all rows at once, at half the GPU's threads
        if (wide) norm_launch_g<T, V, NORM_VALUES_FEW>(few, y, mean, rstd, x, gamma, beta, rows, cols, eps);
        else norm_launch_g<T, 1, NORM_VALUES_FEW>(few, y, mean, rstd, x, gamma, beta, rows, cols, eps);
    } else if (!group) chain(k_norm_long<T>, dim3(grid_for(rows, 1, 2)), 1024, 0, (T *)y, mean, rstd, (const T *)x, (const T *)gamma, (const T *)beta, rows, cols, eps);
    else if (wide) norm_launch_g<T, V, NORM_VALUES>(group, y, mean, rstd, x, gamma, beta, rows, cols, eps);
    else norm_launch_g<T, 1, NORM_VALUES>(group, y, mean, rstd, x, gamma, beta, rows, cols, eps);
}

template <typename T, int VEC, int G>
static void norm_bwd_launch(void *dx, float *partial, const void *dy, const void *x, const void *gamma, const float *mean, const float *rstd, uint32_t rows, uint32_t cols, uint32_t blocks) {
    chain(k_norm_bwd<T, VEC, G>, dim3(blocks), G > 32 ? G : NORM_BLOCK, 0, (T *)dx, partial, (const T *)dy, (const T *)x, (const T *)gamma, mean, rstd, rows, cols);
}
template <typename T, int VEC>
static void norm_bwd_launch_g(uint32_t group, void *dx, float *partial, const void *dy, const void *x, const void *gamma, const float *mean, const float *rstd, uint32_t rows, uint32_t cols, uint32_t blocks) {
    switch (group) {
        case 32:   norm_bwd_launch<T, VEC, 32>(dx, partial, dy, x, gamma, mean, rstd, rows, cols, blocks); break;
        case 128:  norm_bwd_launch<T, VEC, 128>(dx, partial, dy, x, gamma, mean, rstd, rows, cols, blocks); break;
        case 256:  norm_bwd_launch<T, VEC, 256>(dx, partial, dy, x, gamma, mean, rstd, rows, cols, blocks); break;
        case 512:  norm_bwd_launch<T, VEC, 512>(dx, partial, dy, x, gamma, mean, rstd, rows, cols, blocks); break;
        default:   norm_bwd_launch<T, VEC, 1024>(dx, partial, dy, x, gamma, mean, rstd, rows, cols, blocks); break;
    }
}
template <typename T>
static bool norm_backward(void *dx, void *dgamma, void *dbeta, const void *dy, const void *x, const void *gamma, const float *mean, const float *rstd, uint32_t rows, uint32_t cols) {
    const uint32_t group = norm_group(cols, NORM_BWD_VALUES);
    const bool sums = dgamma || dbeta;
    uint32_t n;
    float *partial = nullptr;
    profile_begin();
    if (group) {
        const uint32_t threads = group > 32 ? group : NORM_BLOCK, per = group > 32 ? 1 : NORM_BLOCK / 32;
        // 1024 threads an SM: the registers allow no more; and four rows a group at least, for the sums' sake
        n = grid_for((rows + 3) / 4, per, 1024 / threads);
        if (sums && !(partial = (float *)layer_scratch("layernorm_backward", (uint64_t)n * 2 * cols * sizeof(float)))) return false;
        if (cols % Vec16<T>::n == 0) norm_bwd_launch_g<T, Vec16<T>::n>(group, dx, partial, dy, x, gamma, mean, rstd, rows, cols, n);
        else norm_bwd_launch_g<T, 1>(group, dx, partial, dy, x, gamma, mean, rstd, rows, cols, n);
        after_launch("layernorm_backward");
    } else {
        n = rows < 16 ? rows : 16;
        if (sums) {                                    // first: dx may lie where dy or x does
            if (!(partial = (float *)layer_scratch("layernorm_backward", (uint64_t)n * 2 * cols * sizeof(float)))) return false;
            chain(k_norm_bwd_cols<T>, dim3((cols + 255) / 256, n), 256, 0, partial, (const T *)dy, (const T *)x, mean, rstd, rows, cols);
            after_launch("layernorm_backward_cols");
            profile_begin();
        }
        if (dx) {
            chain(k_norm_bwd_long<T>, dim3(grid_for(rows, 1, 2)), 1024, 0, (T *)dx, (const T *)dy, (const T *)x, (const T *)gamma, mean, rstd, rows, cols);
            after_launch("layernorm_backward");
        }
    }
    if (sums) {
        profile_begin();
        chain(k_fold_rows<T>, dim3((cols + 31) / 32, 2), 1024, 0, (T *)dgamma, (T *)dbeta, (const float *)partial, n, cols);
        after_launch("layernorm_fold");
    }
    return true;
}

}  // namespace thc

using namespace thc;

extern "C" {

int thvm_cuda_layernorm(uint32_t y, uint32_t mean, uint32_t rstd, uint32_t x, uint32_t gamma, uint32_t beta,
                        uint32_t rows, uint32_t cols, float eps, uint32_t dtype) {
    if (rows == 0 || cols == 0) { set_error("layernorm: empty shape"); return 1; }
    if (rows > (1u << 30) || cols > (1u << 30)) { set_error("layernorm: a dimension exceeds 2^30"); return 1; }
    if (dtype != THC_F32 && dtype != THC_F16) { set_error("layernorm: dtype %u is neither f32 nor f16", dtype); return 1; }
    if (!(eps >= 0.0f)) { set_error("layernorm: eps %g", (double)eps); return 1; }
    const uint64_t sz = dtype == THC_F16 ? 2 : 4, need = (uint64_t)rows * cols * sz;
    const uint32_t outs[3] = {y, mean, rstd}, ins[3] = {x, gamma, beta};
    const uint64_t out_need[3] = {need, (uint64_t)rows * 4, (uint64_t)rows * 4}, in_need[3] = {need, cols * sz, cols * sz};
    if (!layer_buffers("layernorm", ins, in_need, 3, 1, outs, out_need, 3, 1, 1u << 0)) return 1;
    const void *px = buf_checked(x, "layernorm(x)").ptr;
    const void *pg = gamma ? buf_checked(gamma, "layernorm(gamma)").ptr : nullptr, *pb = beta ? buf_checked(beta, "layernorm(beta)").ptr : nullptr;
    void *py = buf_for_output(y, "layernorm(y)", need).ptr;
    float *pm = mean ? (float *)buf_for_output(mean, "layernorm(mean)", (uint64_t)rows * 4).ptr : nullptr;
    float *pr = rstd ? (float *)buf_for_output(rstd, "layernorm(rstd)", (uint64_t)rows * 4).ptr : nullptr;
    for (uint32_t id : outs) if (id) mark_device_written(id);
    layer_estimate(8.0 * rows * cols, 2.0 * need);
    profile_begin();
    if (dtype == THC_F16) norm_forward<__half>(py, pm, pr, px, pg, pb, rows, cols, eps);
    else norm_forward<float>(py, pm, pr, px, pg, pb, rows, cols, eps);
    after_launch("layernorm");
    return 0;
}

int thvm_cuda_layernorm_backward(uint32_t dx, uint32_t dgamma, uint32_t dbeta, uint32_t dy, uint32_t x, uint32_t gamma,
                                 uint32_t mean, uint32_t rstd, uint32_t rows, uint32_t cols, uint32_t dtype) {
    if (rows == 0 || cols == 0) { set_error("layernorm_backward: empty shape"); return 1; }
    if (rows > (1u << 30) || cols > (1u << 30)) { set_error("layernorm_backward: a dimension exceeds 2^30"); return 1; }
    if (dtype != THC_F32 && dtype != THC_F16) { set_error("layernorm_backward: dtype %u is neither f32 nor f16", dtype); return 1; }
    if (!dx && !dgamma && !dbeta) { set_error("layernorm_backward: no output asked for"); return 1; }
    const uint64_t sz = dtype == THC_F16 ? 2 : 4, need = (uint64_t)rows * cols * sz;
    const uint32_t outs[3] = {dx, dgamma, dbeta}, ins[5] = {dy, x, mean, rstd, gamma};
    const uint64_t out_need[3] = {need, cols * sz, cols * sz}, in_need[5] = {need, need, (uint64_t)rows * 4, (uint64_t)rows * 4, cols * sz};
    if (!layer_buffers("layernorm_backward", ins, in_need, 5, 4, outs, out_need, 3, 0, 3u)) return 1;
    const void *pdy = buf_checked(dy, "layernorm_backward(dy)").ptr, *px = buf_checked(x, "layernorm_backward(x)").ptr;
    const float *pm = (const float *)buf_checked(mean, "layernorm_backward(mean)").ptr, *pr = (const float *)buf_checked(rstd, "layernorm_backward(rstd)").ptr;
    const void *pg = gamma ? buf_checked(gamma, "layernorm_backward(gamma)").ptr : nullptr;
    void *pdx = dx ? buf_for_output(dx, "layernorm_backward(dx)", need).ptr : nullptr;
    void *pdg = dgamma ? buf_for_output(dgamma, "layernorm_backward(dgamma)", cols * sz).ptr : nullptr;
    void *pdb = dbeta ? buf_for_output(dbeta, "layernorm_backward(dbeta)", cols * sz).ptr : nullptr;
    for (uint32_t id : outs) if (id) mark_device_written(id);
    layer_estimate(14.0 * rows * cols, 3.0 * need);
    return (dtype == THC_F16 ? norm_backward<__half>(pdx, pdg, pdb, pdy, px, pg, pm, pr, rows, cols) : norm_backward<float>(pdx, pdg, pdb, pdy, px, pg, pm, pr, rows, cols)) ? 0 : 1;
}

}  // extern "C"
