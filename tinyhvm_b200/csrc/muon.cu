// muon.cu — orthogonalisation of a matrix by Newton-Schulz products, and the optimizer step that applies it.
//
//   X = G / (|G|_F + 1e-7);  steps times:  A = X X^T (over the smaller side),  B = b A + c A A,  X = a X + B X
// with the quintic's coefficients a, b, c = 3.4445, -4.7750, 2.0315: X keeps G's singular vectors and its singular values
// move to the neighbourhood of 1.
// On the matrix engine a step is three products, with the matrices between them kept as the engine's f16 planes: A and B are symmetric and
// only made from the diagonal on.  Five steps: 4096 x 4096 3.9 ms (1374 GFLOP with
// the symmetry used: 353 TFLOP/s, 1060 of f16 products, the clock at its power limit); 1024 x 4096 390 us.
//   mom = mu mom + g;  u = nesterov ? g + mu mom : mom;  p = p (1 - lr decay) - lr sqrt(max(1, rows / cols)) X(u)
#include <math.h>
#include "hgemm.cuh"
#include "layer_common.cuh"
#include "layer_host.h"
#include "state.h"

namespace thc {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;

// Planes hold 2^13 times the value: X and its square stay below 1.5 in magnitude, b A + c A A below 2.9, so the largest is below 24000 and the
// low part's step is 2^-37.
constexpr float PLANE = 8192.0f;

// mom = mu mom + grad (when there is a momentum) and the sum of squares of the update: one partial per block, in double, which
// the squares of f32 values do not overflow
template <int VEC>
__global__ void __launch_bounds__(256)
k_muon_momentum(float *mom, const float *grad, double *partial, float mu, int nesterov, uint64_t n) {
    depend();
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
    depend();
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
        for (int j = 0; j < VEC; j++) u[j] *= f;
        store_planes<VEC>(hi + row * pitch + c, lo + row * pitch + c, u);
    }
}

// ---- epilogues of the three products of a step (sums carry 2^26) ----
template <int V, int R> __device__ __forceinline__ void put_planes(__half *hi, __half *lo, uint64_t pitch, hg::Rows r, uint32_t n, const float (&v)[R][V]) {
    const uint64_t at = r.first * pitch + n, step = r.step * pitch;
#pragma unroll
    for (uint32_t i = 0; i < R; i++) if (r.first + i * r.step < r.end) store_planes<V>(hi + at + i * step, lo + at + i * step, v[i]);
}
struct SquareEpi {                                     // A = X X^T
    static constexpr bool mirrors = true, long_start = false, heavy = false;
    __half *hi, *lo; uint64_t pitch; uint32_t side;
    __device__ bool wide() const { return side % 4 == 0; }
    __device__ float row_factor(uint32_t) const { return 1.0f / PLANE; }
    __device__ void touch(uint32_t, uint32_t, uint32_t) const {}
    template <int V> __device__ void column(uint32_t) const {}
    template <int V> __device__ void fetch(uint32_t, uint32_t, float (&)[V]) const {}
    template <int V, int R> __device__ void put(hg::Rows r, uint32_t n, float (&v)[R][V], const float (&)[R][V], uint32_t) const { put_planes<V, R>(hi, lo, pitch, r, n, v); }
    template <int V, int R> __device__ void mirror(hg::Rows r, uint32_t m, const float (&v)[R][V]) const { put_planes<V, R>(hi, lo, pitch, r, m, v); }
};
struct PolyEpi {                                       // b A + c A A
    static constexpr bool mirrors = true, long_start = false, heavy = false;
    __half *hi, *lo; const __half *a_hi, *a_lo; uint64_t pitch; uint32_t side;
    __device__ bool wide() const { return side % 4 == 0; }
    __device__ float row_factor(uint32_t) const { return 1.0f / PLANE; }
    __device__ void touch(uint32_t, uint32_t, uint32_t) const {}
    template <int V> __device__ void column(uint32_t) const {}
    template <int V> __device__ void fetch(uint32_t m, uint32_t n, float (&x)[V]) const {
        float l[V];
        load_vec<V>(a_hi + m * pitch + n, x);
        load_vec<V>(a_lo + m * pitch + n, l);
#pragma unroll
        for (int j = 0; j < V; j++) x[j] += l[j];
    }
    template <int V, int R> __device__ void put(hg::Rows r, uint32_t n, float (&v)[R][V], const float (&x)[R][V], uint32_t) const {
#pragma unroll
        for (uint32_t i = 0; i < R; i++)
#pragma unroll
            for (int j = 0; j < V; j++) v[i][j] = NS_B * x[i][j] + NS_C * v[i][j];
        put_planes<V, R>(hi, lo, pitch, r, n, v);
    }
    template <int V, int R> __device__ void mirror(hg::Rows r, uint32_t m, const float (&v)[R][V]) const { put_planes<V, R>(hi, lo, pitch, r, m, v); }
};
enum { NEXT, RESULT, STEP };
// X = a X + (b A + c A A) X: planes for the next step, the result, or the parameters' step.  a X is added here, in f32: it is most of the sum
// while the small singular values still grow, and the tensor core's truncation would be a share of it.
template <int TO> struct ApplyEpi {
    static constexpr bool mirrors = false, long_start = true, heavy = false;
    const __half *x_hi, *x_lo; __half *hi, *lo; uint64_t pitch;
    float *out; uint32_t cols; float keep, step;
    __device__ bool wide() const { return cols % 4 == 0; }
    __device__ void touch(uint32_t m, uint32_t n, uint32_t count) const { if constexpr (TO == STEP) hg::touch_row(out + (uint64_t)m * cols, n, count, cols); }
    __device__ float row_factor(uint32_t) const { return TO == NEXT ? 1.0f / PLANE : 1.0f / (PLANE * PLANE); }
    template <int V> __device__ void column(uint32_t) const {}
    template <int V> __device__ void fetch(uint32_t m, uint32_t n, float (&x)[V]) const {
        float l[V], p[V];
        load_vec<V>(x_hi + m * pitch + n, x);
        load_vec<V>(x_lo + m * pitch + n, l);
        if constexpr (TO == STEP) load_vec<V>(out + (uint64_t)m * cols + n, p);
#pragma unroll
        for (int j = 0; j < V; j++) {
            x[j] = (x[j] + l[j]) * (TO == NEXT ? NS_A : NS_A / PLANE);
            if constexpr (TO == STEP) x[j] = p[j] * keep - step * x[j];
        }
    }
    template <int V, int R> __device__ void put(hg::Rows r, uint32_t n, float (&v)[R][V], const float (&x)[R][V], uint32_t) const {
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int j = 0; j < V; j++) v[i][j] = TO == STEP ? x[i][j] - step * v[i][j] : x[i][j] + v[i][j];
        if constexpr (TO == NEXT) { put_planes<V, R>(hi, lo, pitch, r, n, v); return; }
        float *p = out + (uint64_t)r.first * cols + n;
        const uint64_t down = (uint64_t)r.step * cols;
#pragma unroll
        for (uint32_t i = 0; i < R; i++, p += down) if (r.first + i * r.step < r.end) store_vec<V>(p, v[i]);
    }
};

// ---- small matrices: one launch, everything in one cluster's shared memory ----
// The smaller side is at most 128, the larger 64 times the cluster (128 x 1024 157 us, 128 x 1536 205; on
// the engine 128 x 1600 177).  Block r of the cluster keeps every row of its own share of the larger
// side's columns, X_r (stored column by column), and A and B whole.  A step: P_r = X_r X_r^T by each block; A = sum of P_r, an equal share
// of rows by each block, written to all; B = a I + b A + c A A the same way; X_r = B X_r.  Three barriers of the cluster a step.  All in
// f32 on the CUDA cores: 0.03 GFLOP a step at 400 x 120 is nothing; what bounds it is the latency of the shared-memory reads with four warps a
// scheduler and of the exchange: 400 x 120, five steps, 100 us, of a step's 38000 cycles 8000 in the barriers, 8000 in adding and
// spreading A, 6000 in each of P and B, 9000 in B X.  As 15 launches of the matrix engine it takes 164 us.
constexpr uint32_t NS_SIDE = 128, NS_SHARE = 64, NS_PITCH = 132, NS_THREADS = 512, NS_WARPS = NS_THREADS / 32;
constexpr size_t NS_SMEM = (size_t)(NS_SHARE + 2 * NS_SIDE) * NS_PITCH * 4 + 32 * NS_SIDE * 4;     // X, A, B; parts of eight rows
struct NsSmall { float *out, *param, *mom; const float *grad; uint32_t rows, cols, steps; int nesterov; float mu, keep, step; };

__device__ __forceinline__ float4 remote4(const float *p, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(hg::in_cta(hg::smem32(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ void remote4(float *p, uint32_t rank, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(hg::in_cta(hg::smem32(p), rank)), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__global__ void __launch_bounds__(NS_THREADS, 1)
k_ns_small(const __grid_constant__ NsSmall S) {
    depend();
    extern __shared__ __align__(16) float ns[];
    float (*X)[NS_PITCH] = reinterpret_cast<float (*)[NS_PITCH]>(ns);                              // [NS_SHARE]: column, row
    float (*A)[NS_PITCH] = X + NS_SHARE, (*B)[NS_PITCH] = A + NS_SIDE;                             // [NS_SIDE]; B first holds P
    float4 *parts = reinterpret_cast<float4 *>(B + NS_SIDE);                                       // [4][8][32]
    __shared__ double red[NS_WARPS], norm;
    const uint32_t ranks = gridDim.y, rank = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const bool wide = S.rows <= S.cols;
    const uint32_t m = wide ? S.rows : S.cols, n = wide ? S.cols : S.rows, share = (n + ranks - 1) / ranks;
    const uint32_t c0 = rank * share, mine = c0 >= n ? 0 : n - c0 < share ? n - c0 : share;        // columns c0 .. c0 + mine
    const uint32_t padded = (share + 31u) & ~31u;          // columns kept: whole groups of 32
    // the update, its place in memory and its sum of squares; rows and columns beyond the matrix are zeros
    const auto place = [&](uint32_t c, uint32_t r) { return wide ? (uint64_t)r * S.cols + c0 + c : (uint64_t)(c0 + c) * S.cols + r; };
    const auto each = [&](auto f) {                        // lanes along memory
        for (uint32_t u = tid; u < padded * NS_SIDE; u += NS_THREADS) { const uint32_t c = wide ? u % padded : u / NS_SIDE, r = wide ? u / padded : u % NS_SIDE; f(c, r, c < mine && r < m); }
    };
    double sq = 0.0;
    each([&](uint32_t c, uint32_t r, bool in) {
        float v = 0.0f;
        if (in) {
            const uint64_t at = place(c, r);
            v = S.grad[at];
            if (S.mom) { const float g = v, q = S.mu * S.mom[at] + g; S.mom[at] = q; v = S.nesterov ? g + S.mu * q : q; }
        }
        X[c][r] = v;
        sq += (double)v * v;
    });
#pragma unroll
    for (int o = 16; o; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    if ((tid & 31) == 0) red[tid >> 5] = sq;
    __syncthreads();
    if (tid == 0) { double s = 0.0; for (uint32_t w = 0; w < NS_WARPS; w++) s += red[w]; norm = s; }
    hg::cluster_sync();
    double total = 0.0;
    for (uint32_t q = 0; q < ranks; q++) {
        double d;
        asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(d) : "r"(hg::in_cta(hg::smem32(&norm), q)) : "memory");
        total += d;
    }
    const float inv = (float)(1.0 / (sqrt(total) + 1e-7));
    each([&](uint32_t c, uint32_t r, bool) { X[c][r] *= inv; });
    const uint32_t band = NS_SIDE / ranks;                 // rows of A and of B that this block makes
    for (uint32_t step = 0; step < S.steps; step++) {
        __syncthreads();
        {   // P = X_r X_r^T: 8 x 4 sums a thread
            const uint32_t r0 = warp * 8, q0 = lane * 4;
            float acc[8][4] = {};
            if (r0 < m)
#pragma unroll 2
            for (uint32_t k = 0; k < mine; k++) {
                const float4 a0 = *reinterpret_cast<const float4 *>(&X[k][r0]), a1 = *reinterpret_cast<const float4 *>(&X[k][r0 + 4]), b = *reinterpret_cast<const float4 *>(&X[k][q0]);
                const float a[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
                for (int i = 0; i < 8; i++) { acc[i][0] += a[i] * b.x; acc[i][1] += a[i] * b.y; acc[i][2] += a[i] * b.z; acc[i][3] += a[i] * b.w; }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) *reinterpret_cast<float4 *>(&B[r0 + i][q0]) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
        }
        hg::cluster_sync();
        // this block's rows of A: the two halves of the block add the P of half of the ranks each, and write to half of them
        for (uint32_t i0 = 0; i0 < band; i0 += 8) {
            const uint32_t r = rank * band + i0 + (warp & 7u), c = lane * 4, side = warp >> 3, some = ranks / 2;
            float4 s = make_float4(0, 0, 0, 0);
#pragma unroll 8
            for (uint32_t q = side * some; q < (side + 1) * some; q++) { const float4 v = remote4(&B[r][c], q); s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w; }
            parts[tid] = s;
            __syncthreads();
            const float4 x = parts[tid & 255u], y = parts[(tid & 255u) + 256u];
            s = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
#pragma unroll 8
            for (uint32_t q = side * some; q < (side + 1) * some; q++) remote4(&A[r][c], q, s);
            __syncthreads();
        }
        hg::cluster_sync();
        // its rows of a I + b A + c A A: a warp sums a quarter of the contraction for two whole rows, the parts are added in order
        for (uint32_t i0 = 0; i0 < band; i0 += 8) {
            const uint32_t r0 = rank * band + i0 + (warp & 3u) * 2, k1 = (warp >> 2) * 32;
            float4 acc[2] = {make_float4(0, 0, 0, 0), make_float4(0, 0, 0, 0)};
            if (r0 < m)
#pragma unroll 2
                for (uint32_t k = k1; k < k1 + 32; k += 4) {
                    const float4 a0 = *reinterpret_cast<const float4 *>(&A[r0][k]), a1 = *reinterpret_cast<const float4 *>(&A[r0 + 1][k]);
                    const float u[4] = {a0.x, a0.y, a0.z, a0.w}, v[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float4 b = *reinterpret_cast<const float4 *>(&A[k + j][lane * 4]);
                        acc[0].x += u[j] * b.x; acc[0].y += u[j] * b.y; acc[0].z += u[j] * b.z; acc[0].w += u[j] * b.w;
                        acc[1].x += v[j] * b.x; acc[1].y += v[j] * b.y; acc[1].z += v[j] * b.z; acc[1].w += v[j] * b.w;
                    }
                }
#pragma unroll
            for (int i = 0; i < 2; i++) parts[((warp >> 2) * 8 + (warp & 3u) * 2 + i) * 32 + lane] = acc[i];
            __syncthreads();
            const uint32_t r = rank * band + i0 + (warp & 7u), c = lane * 4, side = warp >> 3, some = ranks / 2;
            float4 s = make_float4(0, 0, 0, 0);
#pragma unroll
            for (uint32_t w = 0; w < 4; w++) { const float4 v = parts[(w * 8 + (warp & 7u)) * 32 + lane]; s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w; }
            const float4 q = *reinterpret_cast<const float4 *>(&A[r][c]);
            s.x = NS_B * q.x + NS_C * s.x + (r == c ? NS_A : 0.0f); s.y = NS_B * q.y + NS_C * s.y + (r == c + 1 ? NS_A : 0.0f);
            s.z = NS_B * q.z + NS_C * s.z + (r == c + 2 ? NS_A : 0.0f); s.w = NS_B * q.w + NS_C * s.w + (r == c + 3 ? NS_A : 0.0f);
#pragma unroll 8
            for (uint32_t t = side * some; t < (side + 1) * some; t++) remote4(&B[r][c], t, s);
            __syncthreads();
        }
        hg::cluster_sync();
        // X_r = B X_r: 4 rows x 2 columns of every 32 a thread; B is symmetric to rounding, so its rows are read as columns.  The columns
        // are independent of one another and a warp's belong to it alone: they are replaced as they are done
        for (uint32_t q0 = warp * 2; q0 < mine; q0 += 2 * NS_WARPS) {
            const uint32_t r0 = lane * 4;
            float acc[2][4] = {};
#pragma unroll 2
            for (uint32_t k = 0; k < m; k += 4) {          // (rows and columns beyond m are zeros)
                const float4 x0 = *reinterpret_cast<const float4 *>(&X[q0][k]), x1 = *reinterpret_cast<const float4 *>(&X[q0 + 1][k]);
                const float u[4] = {x0.x, x0.y, x0.z, x0.w}, v[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4 b = *reinterpret_cast<const float4 *>(&B[k + j][r0]);
                    acc[0][0] += b.x * u[j]; acc[0][1] += b.y * u[j]; acc[0][2] += b.z * u[j]; acc[0][3] += b.w * u[j];
                    acc[1][0] += b.x * v[j]; acc[1][1] += b.y * v[j]; acc[1][2] += b.z * v[j]; acc[1][3] += b.w * v[j];
                }
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 2; j++) *reinterpret_cast<float4 *>(&X[q0 + j][r0]) = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
        }
    }
    __syncthreads();
    each([&](uint32_t c, uint32_t r, bool in) {
        if (!in) return;
        const uint64_t at = place(c, r);
        if (S.param) S.param[at] = S.param[at] * S.keep - S.step * X[c][r];
        else S.out[at] = X[c][r];
    });
    hg::cluster_sync();                                    // no block leaves while another may still write to it
}
// the cluster's size for a matrix, or 0 where it does not fit; 16 blocks need the GPU's consent
static uint32_t ns_small_ranks(uint32_t m, uint32_t n) {
    if (m > NS_SIDE || n > NS_SHARE * 16) return 0;
    static int most = 0, seen = -1;
    if (first_on_device(seen)) {
        most = 8;
        THC_CUDA_OK(cudaFuncSetAttribute(k_ns_small, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)NS_SMEM));
        THC_CUDA_OK(cudaFuncSetAttribute(k_ns_small, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        cudaLaunchConfig_t c{};
        cudaLaunchAttribute a[1];
        a[0].id = cudaLaunchAttributeClusterDimension;
        a[0].val.clusterDim.x = 1; a[0].val.clusterDim.y = 16; a[0].val.clusterDim.z = 1;
        c.gridDim = dim3(1, 16); c.blockDim = dim3(NS_THREADS); c.dynamicSmemBytes = NS_SMEM; c.attrs = a; c.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, k_ns_small, &c) == cudaSuccess && clusters > 0) most = 16;
        else cudaGetLastError();
    }
    return n <= NS_SHARE * (uint32_t)most ? (uint32_t)most : 0;
}

// out (or the parameter step, when param is given) <- Newton-Schulz of grad or of the momentum update
static bool newton_schulz(float *out, float *param, float *mom, const float *grad, uint32_t rows, uint32_t cols, uint32_t steps, float mu, int nesterov, float keep, float step) {
    const uint64_t n = (uint64_t)rows * cols;
    const bool wide = rows <= cols;
    const uint32_t m = wide ? rows : cols, k = wide ? cols : rows;
    if (const uint32_t ranks = ns_small_ranks(m, k)) {
        layer_estimate(2.0 * steps * m * m * (2.0 * k + m), 4.0 * rows * cols * (param ? 5 : 2));
        profile_begin();
        chain_cluster(ranks, k_ns_small, dim3(1, ranks), NS_THREADS, NS_SMEM, NsSmall{out, param, mom, grad, rows, cols, steps, nesterov, mu, keep, step});
        after_launch("newton_schulz_small");
        return true;
    }
    const uint64_t px = (cols + 63u) & ~63ull, pm = (m + 63u) & ~63ull, x_bytes = rows * px * 2, m_bytes = m * pm * 2;    // (multiples of 128)
    const unsigned blocks = grid_for(n, 1024, 4);
    const hg::Plan square = hg::plan(m, m, k, true, true), poly = hg::plan(m, m, m, true, true), apply = hg::plan(rows, cols, m, true, false);
    uint64_t partial_bytes = square.partial_bytes > poly.partial_bytes ? square.partial_bytes : poly.partial_bytes;
    if (apply.partial_bytes > partial_bytes) partial_bytes = apply.partial_bytes;
    uint8_t *base = (uint8_t *)layer_scratch(mom ? "muon_step" : "newton_schulz", 4 * x_bytes + 4 * m_bytes + ((partial_bytes + 7) & ~7ull) + blocks * sizeof(double));
    if (!base) return false;
    __half *x[2][2], *a[2], *b[2];
    for (int i = 0; i < 2; i++) {
        for (int p = 0; p < 2; p++) x[i][p] = (__half *)(base + (2 * i + p) * x_bytes);
        a[i] = (__half *)(base + 4 * x_bytes + i * m_bytes);
        b[i] = (__half *)(base + 4 * x_bytes + (2 + i) * m_bytes);
    }
    float *partial = (float *)(base + 4 * x_bytes + 4 * m_bytes);
    double *norms = (double *)(base + 4 * x_bytes + 4 * m_bytes + ((partial_bytes + 7) & ~7ull));
    profile_begin();
    if (n % 4 == 0) chain(k_muon_momentum<4>, dim3(blocks), 256, 0, mom, grad, norms, mu, nesterov, n);
    else chain(k_muon_momentum<1>, dim3(blocks), 256, 0, mom, grad, norms, mu, nesterov, n);
    after_launch("newton_schulz_norm");
    profile_begin();
    if (cols % 4 == 0) chain(k_muon_planes<4>, dim3(blocks), 256, 0, x[0][0], x[0][1], px, mom, grad, norms, blocks, mu, nesterov, rows, cols);
    else chain(k_muon_planes<1>, dim3(blocks), 256, 0, x[0][0], x[0][1], px, mom, grad, norms, blocks, mu, nesterov, rows, cols);
    after_launch("newton_schulz_planes");
    for (uint32_t i = 0; i < steps; i++) {
        __half **cur = x[i & 1], **next = x[(i & 1) ^ 1];
        const hg::Operand X{cur[0], px, rows * px, !wide}, A{a[0], pm, m * pm, false}, B{b[0], pm, m * pm, false};
        hg::product(X, X, m, m, k, square, partial, SquareEpi{a[0], a[1], pm, m}, true, "newton_schulz_square");
        hg::product(A, A, m, m, m, poly, partial, PolyEpi{b[0], b[1], a[0], a[1], pm, m}, true, "newton_schulz_poly");
        const hg::Operand Xr{cur[0], px, rows * px, wide};                     // X across: the other way round than in its square
        const auto run = [&](auto epi) { hg::product(wide ? B : Xr, wide ? Xr : B, rows, cols, m, apply, partial, epi, false, "newton_schulz_apply"); };
        if (i + 1 < steps) run(ApplyEpi<NEXT>{cur[0], cur[1], next[0], next[1], px, nullptr, cols, 0.0f, 0.0f});
        else if (param) run(ApplyEpi<STEP>{cur[0], cur[1], nullptr, nullptr, px, param, cols, keep, step});
        else run(ApplyEpi<RESULT>{cur[0], cur[1], nullptr, nullptr, px, out, cols, 0.0f, 0.0f});
    }
    return true;
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
    return newton_schulz(po, nullptr, nullptr, px, rows, cols, steps, 0.0f, 0, 0.0f, 0.0f) ? 0 : 1;
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
    return newton_schulz(nullptr, pp, pm, pg, rows, cols, steps, mu, nesterov != 0, (float)(1.0 - (double)lr * weight_decay), (float)((double)lr * sqrt(ratio > 1.0 ? ratio : 1.0))) ? 0 : 1;
}

}  // extern "C"
