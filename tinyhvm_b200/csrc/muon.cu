// muon.cu — orthogonalisation of a matrix by Newton-Schulz products, and the optimizer step that applies it.
//
//   X = G / (|G|_F + 1e-7);  steps times:  A = X X^T (over the smaller side),  B = b A + c A A,  X = a X + B X
// with the quintic's coefficients a, b, c = 3.4445, -4.7750, 2.0315: X keeps G's singular vectors and its singular values
// move to the neighbourhood of 1.
//   mom = mu mom + g;  u = nesterov ? g + mu mom : mom;  p = p (1 - lr decay) - lr sqrt(max(1, rows / cols)) X(u)
#include <math.h>
#include "hgemm.cuh"
#include "layer_common.cuh"
#include "layer_host.h"
#include "state.h"

namespace thc {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;

// Planes hold 2^13 times the value: X and its square stay below 1.5 in magnitude, the polynomial below 3.45, so the largest is
// 28262 and the low part's step is 2^-37.
constexpr float PLANE = 8192.0f;

__device__ __forceinline__ void put_plane(__half *hi, __half *lo, uint64_t at, float v) {
    const __half h = __float2half_rn(v);
    hi[at] = h;
    lo[at] = __float2half_rn(v - __half2float(h));
}

// mom = mu mom + grad (when there is a momentum) and the sum of squares of the update: one partial per block, in double, which
// the squares of f32 values do not overflow
template <int VEC>
__global__ void __launch_bounds__(256)
k_muon_momentum(float *mom, const float *grad, double *partial, float mu, int nesterov, uint64_t n) {
    __shared__ double red[8];
    double s = 0.0;
    for (uint64_t i = (blockIdx.x * 256ull + threadIdx.x) * VEC; i < n; i += gridDim.x * 256ull * VEC) {
        float u[VEC];
        load_vec<VEC>(grad + i, u);
        if (mom) {
            float m[VEC];
            load_vec<VEC>(mom + i, m);
#pragma unroll
            for (int j = 0; j < VEC; j++) { m[j] = mu * m[j] + u[j]; u[j] = nesterov ? u[j] + mu * m[j] : m[j]; }
            store_vec<VEC>(mom + i, m);
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) s += (double)u[j] * u[j];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < 8; w++) s += red[w];
        partial[blockIdx.x] = s;
    }
}
// planes of the update over its norm; the update is made again from the gradient and the new momentum
template <int VEC>
__global__ void __launch_bounds__(256)
k_muon_planes(__half *hi, __half *lo, uint64_t pitch, const float *mom, const float *grad, const double *partial, uint32_t n_partial, float mu, int nesterov, uint32_t rows, uint32_t cols) {
    __shared__ double red[8];
    __shared__ float inv;
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < n_partial; i += 256) s += partial[i];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < 8; w++) s += red[w];
        inv = (float)(PLANE / (sqrt(s) + 1e-7));
    }
    __syncthreads();
    const float f = inv;
    const uint32_t per_row = cols / VEC;
    const uint64_t n = (uint64_t)rows * per_row;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) {
        const uint64_t row = i / per_row;
        const uint32_t c = (uint32_t)(i - row * per_row) * VEC;
        float u[VEC];
        load_vec<VEC>(grad + row * cols + c, u);
        if (mom) {
            float m[VEC];
            load_vec<VEC>(mom + row * cols + c, m);
#pragma unroll
            for (int j = 0; j < VEC; j++) u[j] = nesterov ? u[j] + mu * m[j] : m[j];
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) put_plane(hi, lo, row * pitch + c + j, u[j] * f);
    }
}

// ---- epilogues of the three products of a step (sums carry 2^26) ----
struct SquareEpi {                                     // A = X X^T
    static constexpr bool mirrors = true;
    __half *hi, *lo; uint64_t pitch;
    __device__ void column(uint32_t) const {}
    __device__ void mirror(uint32_t n, uint32_t m, float v) const { put_plane(hi, lo, n * pitch + m, v * (1.0f / PLANE)); }
    __device__ void put(uint32_t m, uint32_t n, float v, uint32_t) const { put_plane(hi, lo, m * pitch + n, v * (1.0f / PLANE)); }
};
struct PolyEpi {                                       // a I + b A + c A A
    static constexpr bool mirrors = true;
    __half *hi, *lo; const __half *a_hi, *a_lo; uint64_t pitch;
    __device__ void column(uint32_t) const {}
    __device__ float value(uint64_t at, float v) const { return NS_B * (__half2float(a_hi[at]) + __half2float(a_lo[at])) + NS_C * (v * (1.0f / PLANE)); }
    __device__ void mirror(uint32_t n, uint32_t m, float v) const { const uint64_t at = n * pitch + m; put_plane(hi, lo, at, value(at, v)); }
    __device__ void put(uint32_t m, uint32_t n, float v, uint32_t) const { const uint64_t at = m * pitch + n; put_plane(hi, lo, at, value(at, v) + (m == n ? NS_A * PLANE : 0.0f)); }
};
struct ApplyEpi {                                      // X = (a I + b A + c A A) X: planes for the next step, the result, or the parameters' step
    static constexpr bool mirrors = false;
    __half *hi, *lo; uint64_t pitch;
    float *out, *param; uint32_t cols; float keep, step;
    __device__ void column(uint32_t) const {}
    __device__ void mirror(uint32_t, uint32_t, float) const {}
    __device__ void put(uint32_t m, uint32_t n, float v, uint32_t) const {
        if (hi) { put_plane(hi, lo, m * pitch + n, v * (1.0f / PLANE)); return; }
        v *= 1.0f / (PLANE * PLANE);
        const uint64_t at = (uint64_t)m * cols + n;
        if (param) param[at] = param[at] * keep - step * v;
        else out[at] = v;
    }
};

// out (or the parameter step, when param is given) <- Newton-Schulz of grad or of the momentum update
static void newton_schulz(float *out, float *param, float *mom, const float *grad, uint32_t rows, uint32_t cols, uint32_t steps, float mu, int nesterov, float keep, float step) {
    const uint64_t n = (uint64_t)rows * cols;
    const bool wide = rows <= cols;
    const uint32_t m = wide ? rows : cols, k = wide ? cols : rows;
    const uint64_t px = (cols + 7u) & ~7ull, pm = (m + 7u) & ~7ull, x_bytes = (rows * px * 2 + 255) & ~255ull, m_bytes = (m * pm * 2 + 255) & ~255ull;
    const unsigned blocks = grid_for(n, 1024, 4);
    const hg::Plan square = hg::plan(m, m, k, false), poly = hg::plan(m, m, m, false), apply = hg::plan(rows, cols, m, true);
    uint8_t *base = (uint8_t *)scratch_reserve(4 * x_bytes + 4 * m_bytes + apply.partial_bytes + blocks * sizeof(double));
    __half *x[2][2], *a[2], *b[2];
    for (int i = 0; i < 2; i++) {
        for (int p = 0; p < 2; p++) x[i][p] = (__half *)(base + (2 * i + p) * x_bytes);
        a[i] = (__half *)(base + 4 * x_bytes + i * m_bytes);
        b[i] = (__half *)(base + 4 * x_bytes + (2 + i) * m_bytes);
    }
    float *partial = (float *)(base + 4 * x_bytes + 4 * m_bytes);
    double *norms = (double *)(base + 4 * x_bytes + 4 * m_bytes + ((apply.partial_bytes + 7) & ~7ull));
    profile_begin();
    if (n % 4 == 0) k_muon_momentum<4><<<blocks, 256, 0, g.stream>>>(mom, grad, norms, mu, nesterov, n);
    else k_muon_momentum<1><<<blocks, 256, 0, g.stream>>>(mom, grad, norms, mu, nesterov, n);
    after_launch("newton_schulz_norm");
    profile_begin();
    if (cols % 4 == 0) k_muon_planes<4><<<blocks, 256, 0, g.stream>>>(x[0][0], x[0][1], px, mom, grad, norms, blocks, mu, nesterov, rows, cols);
    else k_muon_planes<1><<<blocks, 256, 0, g.stream>>>(x[0][0], x[0][1], px, mom, grad, norms, blocks, mu, nesterov, rows, cols);
    after_launch("newton_schulz_planes");
    for (uint32_t i = 0; i < steps; i++) {
        __half **cur = x[i & 1], **next = x[(i & 1) ^ 1];
        const hg::Operand X{cur[0], cur[1], px, !wide}, A{a[0], a[1], pm, false}, B{b[0], b[1], pm, false};
        hg::product(X, X, m, m, k, square, nullptr, SquareEpi{a[0], a[1], pm}, true, "newton_schulz_square");
        hg::product(A, A, m, m, m, poly, nullptr, PolyEpi{b[0], b[1], a[0], a[1], pm}, true, "newton_schulz_poly");
        const bool last = i + 1 == steps;
        const ApplyEpi epi{last ? nullptr : next[0], next[1], px, out, param, cols, keep, step};
        const hg::Operand Xr{cur[0], cur[1], px, wide};                        // X across: the other way round than in its square
        if (wide) hg::product(B, Xr, rows, cols, m, apply, partial, epi, false, "newton_schulz_apply");
        else hg::product(Xr, B, rows, cols, m, apply, partial, epi, false, "newton_schulz_apply");
    }
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
