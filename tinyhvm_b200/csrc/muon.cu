// muon.cu — orthogonalisation of a matrix by Newton-Schulz products, and the optimizer step that applies it.
//
//   X = G / (|G|_F + 1e-7);  steps times:  A = X X^T (over the smaller side),  B = b A + c A A,  X = a X + B X
// with the quintic's coefficients a, b, c = 3.4445, -4.7750, 2.0315: X keeps G's singular vectors and its singular values
// move to the neighbourhood of 1.
//   mom = mu mom + g;  u = nesterov ? g + mu mom : mom;  p = p (1 - lr decay) - lr sqrt(max(1, rows / cols)) X(u)
#include <math.h>
#include "layer_common.cuh"
#include "layer_host.h"
#include "state.h"

namespace thc {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;

// mom and u, or a plain copy of x; partial[block] = the block's sum of squares, in double: squares of f32 values do not overflow it
__global__ void __launch_bounds__(256)
k_muon_update(float *u, float *mom, const float *grad, double *partial, float mu, int nesterov, uint64_t n) {
    __shared__ double red[8];
    double s = 0.0;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) {
        const float gr = grad[i];
        float v = gr;
        if (mom) { const float m = mu * mom[i] + gr; mom[i] = m; v = nesterov ? gr + mu * m : m; }
        u[i] = v;
        s += (double)v * v;
    }
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) { s = 0.0; for (int w = 0; w < 8; w++) s += red[w]; partial[blockIdx.x] = s; }
}
__global__ void __launch_bounds__(256)
k_muon_scale(float *x, const double *partial, uint32_t n_partial, uint64_t n) {
    __shared__ float inv;
    if (threadIdx.x == 0) { double s = 0.0; for (uint32_t i = 0; i < n_partial; i++) s += partial[i]; inv = (float)(1.0 / (sqrt(s) + 1e-7)); }
    __syncthreads();
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) x[i] *= inv;
}
// C = alpha P Q + beta D over 64 x 64 tiles, all f32; P (m,k) and Q (k,n) through element strides
__global__ void __launch_bounds__(256)
k_ns_product(float *C, const float *P, uint64_t pm, uint64_t pk, const float *Q, uint64_t qk, uint64_t qn, const float *D, float alpha, float beta, uint32_t M, uint32_t N, uint32_t K) {
    __shared__ float As[16][65], Bs[16][65];
    const uint32_t m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (uint32_t k0 = 0; k0 < K; k0 += 16) {
        for (uint32_t v = threadIdx.x; v < 1024; v += 256) {
            const uint32_t ma = pk == 1 ? v >> 4 : v & 63u, ka = pk == 1 ? v & 15u : v >> 6;
            const uint32_t nb = qk == 1 ? v >> 4 : v & 63u, kb = qk == 1 ? v & 15u : v >> 6;
            As[ka][ma] = m0 + ma < M && k0 + ka < K ? P[(m0 + ma) * pm + (k0 + ka) * pk] : 0.0f;
            Bs[kb][nb] = n0 + nb < N && k0 + kb < K ? Q[(n0 + nb) * qn + (k0 + kb) * qk] : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] += As[k][ty * 4 + i] * Bs[k][tx + 16 * j];
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
            if (m < M && n < N) { const uint64_t at = (uint64_t)m * N + n; C[at] = alpha * acc[i][j] + (D ? beta * D[at] : 0.0f); }
        }
}
__global__ void __launch_bounds__(256)
k_muon_apply(float *p, const float *x, float keep, float step, uint64_t n) {
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) p[i] = p[i] * keep - step * x[i];
}

// out (or the parameter step, when param is given) <- Newton-Schulz of grad or of the momentum update
static void newton_schulz(float *out, float *param, float *mom, const float *grad, uint32_t rows, uint32_t cols, uint32_t steps, float mu, int nesterov, float keep, float step) {
    const uint64_t n = (uint64_t)rows * cols;
    const uint32_t m = rows < cols ? rows : cols;
    const uint64_t nb = (n * 4 + 255) & ~255ull, mb = ((uint64_t)m * m * 4 + 255) & ~255ull;
    const unsigned blocks = grid_for(n, 256, 8);
    uint8_t *base = (uint8_t *)scratch_reserve(2 * nb + 2 * mb + blocks * sizeof(double));
    float *x = (float *)base, *x2 = (float *)(base + nb), *a = (float *)(base + 2 * nb), *b = (float *)(base + 2 * nb + mb);
    double *partial = (double *)(base + 2 * nb + 2 * mb);
    const bool wide = rows <= cols;
    profile_begin();
    k_muon_update<<<blocks, 256, 0, g.stream>>>(x, mom, grad, partial, mu, nesterov, n);
    after_launch("newton_schulz_update");
    k_muon_scale<<<blocks, 256, 0, g.stream>>>(x, partial, blocks, n);
    after_launch("newton_schulz_scale");
    const dim3 sq((m + 63) / 64, (m + 63) / 64), full((cols + 63) / 64, (rows + 63) / 64);
    for (uint32_t i = 0; i < steps; i++) {
        if (wide) k_ns_product<<<sq, 256, 0, g.stream>>>(a, x, cols, 1, x, 1, cols, nullptr, 1.0f, 0.0f, m, m, cols);
        else k_ns_product<<<sq, 256, 0, g.stream>>>(a, x, 1, cols, x, cols, 1, nullptr, 1.0f, 0.0f, m, m, rows);
        k_ns_product<<<sq, 256, 0, g.stream>>>(b, a, m, 1, a, m, 1, a, NS_C, NS_B, m, m, m);
        float *dst = (i + 1 == steps && !param) ? out : x2;
        if (wide) k_ns_product<<<full, 256, 0, g.stream>>>(dst, b, m, 1, x, cols, 1, x, 1.0f, NS_A, rows, cols, m);
        else k_ns_product<<<full, 256, 0, g.stream>>>(dst, x, cols, 1, b, m, 1, x, 1.0f, NS_A, rows, cols, m);
        after_launch("newton_schulz");
        float *t = x; x = x2; x2 = t;
    }
    if (param) { k_muon_apply<<<blocks, 256, 0, g.stream>>>(param, x, keep, step, n); after_launch("muon_apply"); }
}

static bool ns_shape(const char *who, uint32_t rows, uint32_t cols, uint32_t steps) {
    if (rows == 0 || cols == 0) { set_error("%s: empty shape", who); return false; }
    if (rows > (1u << 20) || cols > (1u << 20)) { set_error("%s: a dimension exceeds 2^20", who); return false; }
    if (steps < 1 || steps > 32) { set_error("%s: %u steps are not between 1 and 32", who, steps); return false; }
    return true;
}

}  // namespace thc

using namespace thc;

extern "C" {

int thvm_cuda_newton_schulz(uint32_t out, uint32_t x, uint32_t rows, uint32_t cols, uint32_t steps) {
    if (!ns_shape("newton_schulz", rows, cols, steps)) return 1;
    const uint64_t need = (uint64_t)rows * cols * 4;
    if (!layer_buffers("newton_schulz", &x, &need, 1, 1, &out, &need, 1, 1, 1u)) return 1;
    const float *px = (const float *)buf_checked(x, "newton_schulz(x)").ptr;
    float *po = (float *)buf_for_output(out, "newton_schulz(out)", need).ptr;
    mark_device_written(out);
    newton_schulz(po, nullptr, nullptr, px, rows, cols, steps, 0.0f, 0, 0.0f, 0.0f);
    return 0;
}

int thvm_cuda_muon_step(uint32_t param, uint32_t grad, uint32_t momentum, uint32_t rows, uint32_t cols,
                        float lr, float mu, float weight_decay, uint32_t nesterov, uint32_t steps) {
    if (!ns_shape("muon_step", rows, cols, steps)) return 1;
    const uint64_t need = (uint64_t)rows * cols * 4, needs[2] = {need, need};
    const uint32_t outs[2] = {param, momentum};
    if (!layer_buffers("muon_step", &grad, &need, 1, 1, outs, needs, 2, 2, 0)) return 1;
    const float *pg = (const float *)buf_checked(grad, "muon_step(grad)").ptr;
    float *pp = (float *)buf_checked(param, "muon_step(param)").ptr, *pm = (float *)buf_checked(momentum, "muon_step(momentum)").ptr;
    mark_device_written(param); mark_device_written(momentum);
    const double ratio = (double)rows / (double)cols;
    newton_schulz(nullptr, pp, pm, pg, rows, cols, steps, mu, nesterov != 0, (float)(1.0 - (double)lr * weight_decay), (float)((double)lr * sqrt(ratio > 1.0 ? ratio : 1.0)));
    return 0;
}

}  // extern "C"
