// layer_common.cuh — what the layer operators (layernorm.cu, linear.cu, muon.cu) share: loads and stores of one to eight
// neighbouring values as f32, block sums, and the activations with their slopes.
//
// f16 values are rounded to nearest even when they are stored.  (The dispatch path rounds half up on the dropped bits,
// because it is compared bit for bit with the reference; these operators have no counterpart there.)
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "../../include/thvm_cuda.h"

namespace thc {

// Kernels of these operators follow one another as dependent launches (layer_host.h:chain): a kernel may be set up while the one before
// it still runs.  Each calls this before it touches memory: everything before is then finished and visible, and the kernel after may be set up.
__device__ __forceinline__ void depend() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void put_f32(float *p, float v) { *p = v; }
__device__ __forceinline__ void put_f32(__half *p, float v) { *p = __float2half_rn(v); }

// 16 bytes hold this many values
template <typename T> struct Vec16 { static constexpr int n = 16 / (int)sizeof(T); };

// V neighbouring values; p is aligned to V of them
template <int V> __device__ __forceinline__ void load_vec(const float *p, float (&v)[V]) {
    if constexpr (V == 4) { const float4 q = *reinterpret_cast<const float4 *>(p); v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w; }
    else { v[0] = *p; }
}
template <int V> __device__ __forceinline__ void load_vec(const __half *p, float (&v)[V]) {
    if constexpr (V == 8) {
        const uint4 q = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i])); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    } else if constexpr (V == 4) {
        const uint2 q = *reinterpret_cast<const uint2 *>(p);
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&q.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&q.y));
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    } else { v[0] = __half2float(*p); }
}
template <int V> __device__ __forceinline__ void store_vec(float *p, const float (&v)[V]) {
    if constexpr (V == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *p = v[0];
}
template <int V> __device__ __forceinline__ void store_vec(__half *p, const float (&v)[V]) {
    if constexpr (V == 8) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) { const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t *>(&h); }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else if constexpr (V == 4) {
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    } else { *p = __float2half_rn(v[0]); }
}
// hi = f16(x), lo = f16(x - hi): the planes of V neighbouring values (hgemm.cuh)
template <int V> __device__ __forceinline__ void store_planes(__half *hi, __half *lo, const float (&x)[V]) {
    float h[V], l[V];
#pragma unroll
    for (int j = 0; j < V; j++) { h[j] = __half2float(__float2half_rn(x[j])); l[j] = x[j] - h[j]; }
    store_vec<V>(hi, h);
    if (lo) store_vec<V>(lo, l);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Column sums of partial rows: partial[n][gridDim.y][cols] -> first (blockIdx.y 0) and second (1), 32 columns a block of 1024, every 32nd row a
// thread, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024)
k_fold_rows(T *first, T *second, const float *partial, uint32_t n, uint32_t cols) {
    depend();
    __shared__ float red[32][33];
    const uint32_t lane = threadIdx.x & 31u, q = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    T *out = blockIdx.y ? second : first;
    if (!out) return;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 4
        for (uint32_t i = q; i < n; i += 32) s += partial[((uint64_t)i * gridDim.y + blockIdx.y) * cols + c];
    }
    red[q][lane] = s;
    __syncthreads();
    s = warp_sum(red[lane][q]);                        // warp q: column q of the block
    if (lane == 0 && blockIdx.x * 32 + q < cols) put_f32(out + blockIdx.x * 32 + q, s);
}

// ---- activations (thvm_cuda_linear): value and slope at z ----
// Phi(z) = (1 + erf(z / sqrt 2)) / 2.  With t = |z| / sqrt 2, erfc(t) = 2^(-t p(t)); p is a polynomial of degree 7 fitted to
// -log2(erfc(t)) / t over [0, 4] so that erf's error is least at its largest (1.6e-8, with f32 arithmetic 7.5e-8; beyond 4, where
// erfc < 2e-8, t p(t) keeps growing).  One exponential and no branch, where erff has two; the lower tail keeps its relative accuracy.
__device__ __forceinline__ float normal_cdf(float z) {
    const float t = fabsf(z) * 0.70710678f;
    float p = 4.5354569e-05f;
    p = fmaf(p, t, -4.4547446e-04f);
    p = fmaf(p, t, 1.4893346e-03f);
    p = fmaf(p, t, 7.7480281e-04f);
    p = fmaf(p, t, -2.8253829e-02f);
    p = fmaf(p, t, 1.4848168e-01f);
    p = fmaf(p, t, 9.1841638e-01f);
    p = fmaf(p, t, 1.6279086f);
    const float half_erfc = 0.5f * exp2f(-t * p);
    return z < 0.0f ? half_erfc : 1.0f - half_erfc;
}
__device__ __forceinline__ float logistic(float z) { return __fdividef(1.0f, 1.0f + exp2f(-1.44269504f * z)); }
__device__ __forceinline__ float act_value(uint32_t act, float z) {
    switch (act) {
        case THC_ACT_RELU: return z > 0.0f ? z : 0.0f;                       // as the RELU op of the dispatch path: NaN gives 0
        case THC_ACT_GELU: return z * normal_cdf(z);
        case THC_ACT_SILU: return z * logistic(z);
        default:           return z;
    }
}
__device__ __forceinline__ float act_slope(uint32_t act, float z) {
    switch (act) {
        case THC_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case THC_ACT_GELU: return normal_cdf(z) + z * exp2f(-0.72134752f * z * z) * 0.39894228f;
        case THC_ACT_SILU: { const float s = logistic(z); return s * (1.0f + z * (1.0f - s)); }
        default:           return 1.0f;
    }
}
// v *= act'(z)
template <int V> __device__ __forceinline__ void act_slopes(uint32_t act, float (&v)[V], const float (&z)[V]) {
    if (act == THC_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < V; j++) v[j] *= act_slope(THC_ACT_RELU, z[j]);
    } else if (act == THC_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < V; j++) v[j] *= act_slope(THC_ACT_GELU, z[j]);
    } else if (act == THC_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < V; j++) v[j] *= act_slope(THC_ACT_SILU, z[j]);
    }
}

}  // namespace thc
