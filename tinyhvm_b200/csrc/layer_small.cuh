// layer_small.cuh — products of the linear layer that are too small for the matrix engine, whose kernels cost some 10 us each with
// the operands' planes before them: one launch on the CUDA cores, forward, or both gradients and the bias's (included by linear.cu).
//
// A block of 128 threads makes 64 x 32 sums, 4 x 4 a thread, from slabs of 32 of the contraction in shared memory; the next slab is read
// into registers while one is used.  A cluster of S blocks splits the contraction and adds the parts through its shared memory, in
// rank order.  A slab's 32 products are summed by themselves before they go onto the total, so a sum has K / 32 roundings of its size, not K.
// dz = dy act'(z) is made where it is read.
#pragma once
#include "hgemm.cuh"

namespace thc {

enum { SMALL_Y, SMALL_DX, SMALL_DW };
template <typename T> struct Small {
    const T *x, *w, *dy, *z_in, *bias, *residual;
    T *y, *z_out, *dx, *dw, *dbias;
    uint32_t M, K, N, act, dx_tiles;                       // blocks below dx_tiles make dx, the others dw
};

// value of an operand at memory row r, column c of a [rows, cols] matrix
template <typename T> __device__ __forceinline__ float small_at(const T *p, uint32_t r, uint32_t c, uint32_t rows, uint32_t cols) {
    return r < rows && c < cols ? to_f32(p[(uint64_t)r * cols + c]) : 0.0f;
}
template <typename T> __device__ __forceinline__ float small_dz(const Small<T> &S, uint32_t m, uint32_t n) {
    if (m >= S.M || n >= S.N) return 0.0f;
    const uint64_t at = (uint64_t)m * S.N + n;
    const float d = to_f32(S.dy[at]);
    return S.act == THC_ACT_NONE ? d : d * act_slope(S.act, to_f32(S.z_in[at]));
}

constexpr uint32_t SMALL_ROWS = 64;
struct SmallShared { float a[32][SMALL_ROWS + 4], b[32][36], part[SMALL_ROWS][33], column[4][32]; };

// a float of a block of the cluster
__device__ __forceinline__ float small_part(uint32_t addr, uint32_t rank) {
    float p;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p) : "r"(hg::in_cta(addr, rank)));
    return p;
}

template <typename T, int MODE>
__device__ __forceinline__ void small_tile(const Small<T> &S, SmallShared &sh, uint32_t tile, uint32_t rank, uint32_t ranks) {
    // rows x cols = the result, depth = the contraction
    const uint32_t rows = MODE == SMALL_DW ? S.K : S.M, cols = MODE == SMALL_DX ? S.K : S.N, depth = MODE == SMALL_Y ? S.K : MODE == SMALL_DX ? S.N : S.M;
    const uint32_t across = (cols + 31) / 32, r0 = tile / across * SMALL_ROWS, c0 = tile % across * 32;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, tx = threadIdx.x & 7u, ty = threadIdx.x >> 3;
    const uint32_t slabs = (depth + 31) / 32, per = (slabs + ranks - 1) / ranks, first = rank * per < slabs ? rank * per : slabs, last = first + per < slabs ? first + per : slabs;
    float total[4][4] = {}, ra[16], rb[8], column = 0.0f;
    const auto read = [&](uint32_t slab) {
        const uint32_t d = slab * 32;
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) {                // lanes run along memory
            if constexpr (MODE == SMALL_Y) ra[i] = small_at(S.x, r0 + warp + 4 * i, d + lane, S.M, S.K);
            if constexpr (MODE == SMALL_DX) ra[i] = small_dz(S, r0 + warp + 4 * i, d + lane);
            if constexpr (MODE == SMALL_DW) ra[i] = S.dw ? small_at(S.x, d + warp + 4 * (i & 7), r0 + (i >> 3) * 32 + lane, S.M, S.K) : 0.0f;    // (for dbias alone there need be no x)
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t q = warp + 4 * i;
            if constexpr (MODE == SMALL_Y) rb[i] = small_at(S.w, d + q, c0 + lane, S.K, S.N);
            if constexpr (MODE == SMALL_DX) rb[i] = small_at(S.w, c0 + q, d + lane, S.K, S.N);
            if constexpr (MODE == SMALL_DW) { rb[i] = small_dz(S, d + q, c0 + lane); column += rb[i]; }
        }
    };
    if (first < last) read(first);
    for (uint32_t s = first; s < last; s++) {
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) { if constexpr (MODE == SMALL_DW) sh.a[warp + 4 * (i & 7)][(i >> 3) * 32 + lane] = ra[i]; else sh.a[lane][warp + 4 * i] = ra[i]; }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) { if constexpr (MODE == SMALL_DX) sh.b[lane][warp + 4 * i] = rb[i]; else sh.b[warp + 4 * i][lane] = rb[i]; }
        __syncthreads();
        if (s + 1 < last) read(s + 1);
        float acc[4][4] = {};
#pragma unroll
        for (int k = 0; k < 32; k++) {
            const float4 p = *reinterpret_cast<const float4 *>(&sh.a[k][4 * ty]), b = *reinterpret_cast<const float4 *>(&sh.b[k][4 * tx]);
            const float a[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
            for (int i = 0; i < 4; i++) { acc[i][0] += a[i] * b.x; acc[i][1] += a[i] * b.y; acc[i][2] += a[i] * b.z; acc[i][3] += a[i] * b.w; }
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) total[i][j] += acc[i][j];
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) sh.part[4 * ty + i][4 * tx + j] = total[i][j];
    if constexpr (MODE == SMALL_DW) sh.column[warp][lane] = column;
    hg::cluster_sync();                                    // (of one block too: its threads' parts)
    const uint32_t share = SMALL_ROWS * 32 / ranks;
    for (uint32_t u = threadIdx.x; u < share; u += 128) {
        const uint32_t e = rank * share + u, r = e >> 5, c = e & 31u, here = hg::smem32(&sh.part[r][c]);
        float p[8], v = 0.0f;                              // eight reads at once, not one after another
#pragma unroll
        for (uint32_t q = 0; q < 8; q++) p[q] = q < ranks ? small_part(here, q) : 0.0f;
#pragma unroll
        for (uint32_t q = 0; q < 8; q++) v += p[q];
        if (r0 + r >= rows || c0 + c >= cols) continue;
        const uint64_t at = (uint64_t)(r0 + r) * cols + c0 + c;
        if constexpr (MODE == SMALL_Y) {
            if (S.bias) v += to_f32(S.bias[c0 + c]);
            if (S.z_out) put_f32(S.z_out + at, v);
            v = act_value(S.act, v);
            if (S.residual) v += to_f32(S.residual[at]);
            put_f32(S.y + at, v);
        }
        if constexpr (MODE == SMALL_DX) put_f32(S.dx + at, v);
        if constexpr (MODE == SMALL_DW) if (S.dw) put_f32(S.dw + at, v);
    }
    if constexpr (MODE == SMALL_DW) {
        if (S.dbias && r0 == 0 && rank == 0 && threadIdx.x < 32 && c0 + lane < cols) {
            float p[8][4], v = 0.0f;
#pragma unroll
            for (uint32_t q = 0; q < 8; q++)
#pragma unroll
                for (int w = 0; w < 4; w++) p[q][w] = q < ranks ? small_part(hg::smem32(&sh.column[w][lane]), q) : 0.0f;
#pragma unroll
            for (uint32_t q = 0; q < 8; q++)
#pragma unroll
                for (int w = 0; w < 4; w++) v += p[q][w];
            put_f32(S.dbias + c0 + lane, v);
        }
    }
    hg::cluster_sync();                                    // no block leaves while another reads its parts
}

template <typename T>
__global__ void __launch_bounds__(128)
k_small_forward(const __grid_constant__ Small<T> S) {
    depend();
    __shared__ __align__(16) SmallShared sh;
    small_tile<T, SMALL_Y>(S, sh, blockIdx.x, blockIdx.y, gridDim.y);
}
template <typename T>
__global__ void __launch_bounds__(128)
k_small_backward(const __grid_constant__ Small<T> S) {
    depend();
    __shared__ __align__(16) SmallShared sh;
    if (blockIdx.x < S.dx_tiles) small_tile<T, SMALL_DX>(S, sh, blockIdx.x, blockIdx.y, gridDim.y);
    else small_tile<T, SMALL_DW>(S, sh, blockIdx.x - S.dx_tiles, blockIdx.y, gridDim.y);
}

// Blocks of a cluster: as many as leave a slab of the contraction to each, while `room` blocks an SM hold them all.
static uint32_t small_ranks(uint64_t tiles, uint32_t depth, uint32_t room) {
    uint32_t s = 1;
    while (s < 8 && tiles * s * 2 <= (uint64_t)g.sm_count * room && depth >= 64u * s) s *= 2;
    return s;
}

}  // namespace thc
