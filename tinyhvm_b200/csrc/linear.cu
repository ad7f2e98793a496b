// linear.cu — the fully connected layer: y = act(x w + bias) + residual, and its backward pass.
//
//   forward   z = x w + bias,  y = act(z) + residual                    x [M,K], w [K,N] (in, out: as the framework stores weights)
//   backward  dz = dy act'(z);  dx = dz w^T;  dw = x^T dz;  dbias = sum over rows of dz
#include "layer_common.cuh"
#include "layer_host.h"
#include "state.h"

namespace thc {

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

// ---- contraction on the CUDA cores: C(m,n) = sum_k A(m,k) B(k,n) through element strides ----
struct Strided { const void *p; uint64_t sm, sk; };    // sm: along m (or n), sk: along k
template <typename TA, typename TB, class Epi>
__global__ void __launch_bounds__(256)
k_product(Strided A, Strided B, Epi epi, uint32_t M, uint32_t N, uint32_t K) {
    __shared__ float As[16][65], Bs[16][65];
    const uint32_t m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (uint32_t k0 = 0; k0 < K; k0 += 16) {
        for (uint32_t u = threadIdx.x; u < 1024; u += 256) {
            // neighbouring threads walk along whichever index is dense
            const uint32_t ma = A.sk == 1 ? u >> 4 : u & 63u, ka = A.sk == 1 ? u & 15u : u >> 6;
            const uint32_t nb = B.sk == 1 ? u >> 4 : u & 63u, kb = B.sk == 1 ? u & 15u : u >> 6;
            As[ka][ma] = m0 + ma < M && k0 + ka < K ? to_f32(((const TA *)A.p)[(m0 + ma) * A.sm + (k0 + ka) * A.sk]) : 0.0f;
            Bs[kb][nb] = n0 + nb < N && k0 + kb < K ? to_f32(((const TB *)B.p)[(n0 + nb) * B.sm + (k0 + kb) * B.sk]) : 0.0f;
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
            if (m < M && n < N) epi(m, n, acc[i][j]);
        }
}

template <typename T> struct LinearEpi {
    T *y, *z; const T *bias, *residual; uint32_t act, N;
    __device__ void operator()(uint32_t m, uint32_t n, float v) const {
        const uint64_t at = (uint64_t)m * N + n;
        if (bias) v += to_f32(bias[n]);
        if (z) put_f32(z + at, v);
        v = act_value(act, v);
        if (residual) v += to_f32(residual[at]);
        put_f32(y + at, v);
    }
};
template <typename T> struct PlainEpi {
    T *c; uint32_t N;
    __device__ void operator()(uint32_t m, uint32_t n, float v) const { put_f32(c + (uint64_t)m * N + n, v); }
};

template <typename TA, typename TB, class Epi>
static void product(Strided A, Strided B, Epi epi, uint32_t M, uint32_t N, uint32_t K) {
    k_product<TA, TB, Epi><<<dim3((N + 63) / 64, (M + 63) / 64), 256, 0, g.stream>>>(A, B, epi, M, N, K);
}

// dz = dy act'(z) in f32
template <typename T>
__global__ void __launch_bounds__(256)
k_dz(float *dz, const T *dy, const T *z, uint32_t act, uint64_t n) {
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) dz[i] = to_f32(dy[i]) * (z ? act_slope(act, to_f32(z[i])) : 1.0f);
}
template <typename T>
__global__ void __launch_bounds__(256)
k_col_sums(T *out, const float *dz, uint32_t M, uint32_t N) {
    __shared__ float red[8][33];
    const uint32_t c = blockIdx.x * 32 + (threadIdx.x & 31u), q = threadIdx.x >> 5;
    float s = 0.0f;
    if (c < N) for (uint64_t m = q; m < M; m += 8) s += dz[m * N + c];
    red[q][threadIdx.x & 31u] = s;
    __syncthreads();
    if (q == 0 && c < N) {
        s = 0.0f;
        for (int i = 0; i < 8; i++) s += red[i][threadIdx.x];
        put_f32(out + c, s);
    }
}

template <typename T>
static void linear_forward(void *y, void *z, const void *x, const void *w, const void *bias, const void *residual, uint32_t M, uint32_t K, uint32_t N, uint32_t act) {
    profile_begin();
    product<T, T>(Strided{x, K, 1}, Strided{w, 1, N}, LinearEpi<T>{(T *)y, (T *)z, (const T *)bias, (const T *)residual, act, N}, M, N, K);
    after_launch("linear");
}

template <typename T>
static void linear_backward(void *dx, void *dw, void *dbias, const void *dy, const void *z, const void *x, const void *w, uint32_t M, uint32_t K, uint32_t N, uint32_t act) {
    const uint64_t mn = (uint64_t)M * N;
    float *dz = (float *)scratch_reserve(mn * 4);
    profile_begin();
    k_dz<T><<<grid_for(mn, 256, 8), 256, 0, g.stream>>>(dz, (const T *)dy, (const T *)z, act, mn);
    after_launch("linear_backward_dz");
    if (dbias) { k_col_sums<T><<<(N + 31) / 32, 256, 0, g.stream>>>((T *)dbias, dz, M, N); after_launch("linear_backward_bias"); }
    if (dx) { product<float, T>(Strided{dz, N, 1}, Strided{w, N, 1}, PlainEpi<T>{(T *)dx, K}, M, K, N); after_launch("linear_backward_dx"); }
    if (dw) { product<T, float>(Strided{x, 1, K}, Strided{dz, 1, N}, PlainEpi<T>{(T *)dw, N}, K, N, M); after_launch("linear_backward_dw"); }
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
    if (dtype == THC_F16) linear_forward<__half>(py, pz, px, pw, pb, pr, M, K, N, act);
    else linear_forward<float>(py, pz, px, pw, pb, pr, M, K, N, act);
    return 0;
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
    if (dtype == THC_F16) linear_backward<__half>(pdx, pdw, pdb, pdy, pz, px, pw, M, K, N, act);
    else linear_backward<float>(pdx, pdw, pdb, pdy, pz, px, pw, M, K, N, act);
    return 0;
}

}  // extern "C"
