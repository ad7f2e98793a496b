// hgemm.cuh — products of f16 planes on the tensor cores, for the layer operators (included by linear.cu and muon.cu).
//
//   acc(m, n) = sum over k of A(m,k) B(n,k),   A = A_hi + A_lo,  B = B_hi + B_lo      (low planes optional)
//
// An f32 operand travels as two f16 planes of x 2^s: hi = f16(x 2^s) and lo = f16(x 2^s - hi).  f16 holds 11 bits, the
// remainder is at most half a step and has a sign, so hi + lo is x to 2^-24 relative, f32's own half step, as long as
// the scaled value is not so small that lo falls below f16's smallest step, 2^-24: the scale puts the largest value of a row in
// [2^14, 2^15), which leaves 2^-40 of that as the floor.  A B is then A_hi B_lo + A_lo B_hi + A_hi B_hi (the fourth
// product is below 2^-24): three f16 MMAs, where three tf32 MMAs would run at half their rate and keep 2^-21.
//
// The tensor core truncates when it adds to an accumulator, so a long sum drifts towards zero by about 2^-24 per add.
// Here an accumulator lives for 128 k only (1024 or 2048 without low planes): eight epilogue warps then take it from
// tensor memory and add it, rounded, to f32 sums in registers, while the MMAs of the next chunk fill the other of
// two accumulators.  Within a block of k the small products go first.
//
// A CTA pair (cta_group::2) computes a 256 x NT tile, NT = 256 or 128: each CTA holds 128 rows of A, half of B's
// columns, and the accumulators of its own rows.  Roles: warps 0-7 epilogue, warps 8 and 9 tile loads of A and of B, warp 10
// (first CTA) MMAs; 11 fills up their warpgroup.  The pairs are
// persistent and walk over the tiles, so the next tile's loads and MMAs run under this one's epilogue.
//
// Operands may lie either way round, as the matrix descriptors allow for f16: k along memory rows (boxes of 64 k x rows),
// or m / n along memory rows (boxes of 64 rows x 64 k), so nothing is ever transposed.
//
// What bounds it, measured: the tensor cores, and the power they draw.  8192 x 4096 x 4096 in f16 207 us, 1326 TFLOP/s, 0.80 of the measured
// burst rate (in a long loop the clock falls to 1.35 GHz: 250 to 270 us); 4096^3 in f32 358 us with the planes' making, 385 TFLOP/s, of which
// three f16 MMAs each make 1154.  A pair takes 1900 cycles for 64 k of three products, whose MMAs take 1536: the rest is the epilogue where the
// next tile's first two chunks do not hide it, and tile loads and MMAs sharing shared memory's bandwidth (without loads 1640).
//
// Every wait is bounded.  A wait that runs out raises status bit 8 and ends the kernel after its copies in flight.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <string.h>
#include "layer_common.cuh"
#include "layer_host.h"
#include "state.h"

namespace thc {
namespace hg {

constexpr uint32_t EPI_WARPS = 8, TMA_A_WARP = 8, TMA_B_WARP = 9, MMA_WARP = 10, THREADS = 384;
// 168 registers a thread at launch (65536 / 384, by eights); the epilogue's two warpgroups take from the third: 128 x 56 + 256 x 224 = 384 x 168
constexpr uint32_t EPI_REGS = 224, IO_REGS = 56;
constexpr uint32_t KB = 64;                                // k of a block: 128 bytes, the swizzle's width
constexpr uint32_t A_PLANE = 128 * 128;                    // bytes of one CTA's A plane of a block
constexpr uint32_t RING_BYTES = 196608, STAGING = EPI_WARPS * 4096;
constexpr uint32_t MAX_STAGES = 8;
constexpr uint32_t WAIT_LIMIT = 1u << 24;
constexpr int STATUS_TIMEOUT = 8;
// How an operand lies in memory, and its tile loads: k along rows, [planes][rows][k]; m / n along rows whose pitch is a multiple of 64,
// seen as [planes][blocks of 64][k][64]; or the latter with one plane and any pitch, a load per block.  (A load costs
// the issuing thread some 200 cycles: with one per plane and block the loads, not the MMAs, set the pace.)
enum : uint32_t { K_ROWS = 0, MN_BLOCKS = 1, MN_BOXES = 2 };

struct Shared {
    unsigned long long full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_empty[2];
    uint32_t tmem;
    int abort_flag;
};
constexpr size_t SMEM = 1024 + RING_BYTES + STAGING + sizeof(Shared);

struct Shape {
    uint32_t M, N, K;
    uint32_t row_tiles, col_tiles, tiles;                  // tiles: of all splits, below the diagonal left out when `upper`
    uint32_t blocks, split_blocks, chunk, lead;            // blocks of k: in all, per split, per chunk; how much longer a tile's first two are
    uint32_t split_tiles;                                  // tiles of a split
    uint32_t halves, stages, stage_bytes, half_bytes, a_bytes;   // a block of k is one or two times 64 k: a half holds A's and B's planes of 64 k
    uint32_t a_mode, b_mode, a_lo, b_lo, upper;
    int *status;
};
struct Maps { CUtensorMap a, b; };

// ---- PTX ----
__device__ __forceinline__ uint32_t smem32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) { uint32_t r; asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank)); return r; }
__device__ __forceinline__ uint32_t cluster_cta() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t cluster_addr) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
// false after WAIT_LIMIT polls or when another thread of this CTA gave up
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
    for (uint32_t it = 0; it < WAIT_LIMIT; ++it) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if ((it & 255u) == 255u && *abort_flag) return false;
    }
    *abort_flag = 1;
    return false;
}
// The same for the three threads that everything waits for: test_wait in a tight loop, as try_wait may park the thread and waking it
// takes several hundred cycles.
__device__ __forceinline__ bool bar_spin(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
    for (uint32_t it = 0; it < WAIT_LIMIT * 8u; ++it) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if ((it & 1023u) == 1023u && *abort_flag) return false;
    }
    *abort_flag = 1;
    return false;
}
// a box of the map into this CTA's shared memory, signalled on a barrier of the pair's first CTA
__device__ __forceinline__ void load_box3(uint32_t dst, const CUtensorMap *map, uint32_t bar, uint32_t x, uint32_t y) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"((int)x), "r"((int)y), "r"(0) : "memory");
}
__device__ __forceinline__ void load_box4(uint32_t dst, const CUtensorMap *map, uint32_t bar, uint32_t y, uint32_t z) {
    asm volatile("cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"((int)y), "r"((int)z), "r"(0) : "memory");
}
// One operand's tile of a block of k: all its planes, `blocks` x 64 of m / n where they run along memory rows.
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap *map, uint32_t bar, uint32_t mode, uint32_t blocks, uint32_t mn, uint32_t k) {
    if (mode == K_ROWS) load_box3(dst, map, bar, k, mn);
    else if (mode == MN_BLOCKS) load_box4(dst, map, bar, k, mn / 64u);
    else for (uint32_t j = 0; j < blocks; j++) load_box3(dst + j * 8192u, map, bar, mn + j * 64u, k);
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commit_both(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// 128-byte-swizzled operand.  k along rows: 8-row groups 1024 bytes apart.  m / n along rows: 64-value blocks 8192 bytes apart, groups of
// 8 k 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t mn) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(mn ? 8192u >> 4 : 1u) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void acc_load(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// `n` values of a row into L2
template <typename T> __device__ __forceinline__ void touch_row(const T *row, uint32_t from, uint32_t n, uint32_t end) {
    for (uint32_t i = from; i < from + n && i < end; i += 128u / sizeof(T)) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + i));
}

// The chunks of a tile: the first two are `lead` times as long, so that the MMAs have work while the epilogue warps finish the tile before.
// Twice, without low planes or where the epilogue adds more than the product is (Epi::long_start); else once: twice gains 8% at
// K = 1024, but sums of one sign would be off by 1.6e-6 instead of 0.6e-6.
__device__ __forceinline__ uint32_t chunk_end(uint32_t kb, uint32_t chunk, uint32_t lead) { return kb + (kb < 2 * lead * chunk ? lead * chunk : chunk); }

struct Tile { uint32_t m0, n0, z, blocks, block0; };
// Tiles in order: split, then bands of 8 row tiles, columns, rows of the band: the tiles in flight share few operand panels.
template <uint32_t NT> __device__ __forceinline__ Tile tile_of(const Shape &S, uint32_t t) {
    Tile r;
    uint32_t row, col;
    r.z = t / S.split_tiles;
    t -= r.z * S.split_tiles;
    if (S.upper) {                                         // row by row from the diagonal on
        row = 0; col = t;
        for (;;) {
            const uint32_t first = row * 256u / NT, n = S.col_tiles - first;
            if (col < n) { col += first; break; }
            col -= n; row++;
        }
    } else {
        const uint32_t band = t / (8u * S.col_tiles), v = t - band * 8u * S.col_tiles;
        const uint32_t h = S.row_tiles - band * 8u < 8u ? S.row_tiles - band * 8u : 8u;
        col = v / h; row = band * 8u + (v - col * h);
    }
    r.m0 = row * 256u; r.n0 = col * NT;
    r.block0 = r.z * S.split_blocks;
    r.blocks = S.blocks - r.block0 < S.split_blocks ? S.blocks - r.block0 : S.split_blocks;
    return r;
}

// Epi: what happens to finished sums, R rows (m, m + step, ...; those below M count) of V neighbouring columns at a time (V = 4 where
// Epi::wide() says that the result's rows allow it, else 1).  column<V>(n) sets up what belongs to the columns n, n+1, ...; fetch<V>(m, n, x)
// reads what a row's result needs from memory; row_factor(m), exact, goes onto a row's sums before all that; put<V, R>(rows, n, v, x, z) finishes the values
// in v and stores them.  With Epi::mirrors, mirror<V, R> stores finished values in the transposed place of a symmetric product: rows along n,
// V neighbouring values of m.
struct Rows { uint32_t first, step, end; };             // end: 0xffffffff where the caller knows that all are valid

// A block of 32 x 32 sums passes through shared memory, one warp's 4 KB, from "a lane holds a row" to "eight lanes hold a row" (or
// 32 lanes, V = 1).  16-byte chunk c of row r lies at chunk c ^ swap(r): whole rows, rows by chunk and columns by four are all read
// and written without bank conflicts.
//
// Four rows of a lane go together, so that their arithmetic overlaps.  What an epilogue does not do has to be left out when it is
// compiled: a branch over sixteen values is turned into sixteen predicated instructions, and with every choice made at run time a
// tile's epilogue took 18000 cycles, where the MMAs of K = 1024 take 8000 in f16.
__device__ __forceinline__ uint32_t swap(uint32_t r) { return (r ^ (r >> 2)) & 7u; }
template <int V, bool WHOLE, class Epi>
__device__ __forceinline__ void put_block(Epi &e, float *st, uint32_t lane, uint32_t m0, uint32_t n0, uint32_t rows, uint32_t N, uint32_t z) {
    const uint32_t M = WHOLE ? 0xffffffffu : rows;
    if constexpr (V == 4) {
        const uint32_t ro = lane >> 3, n = n0 + (lane & 7u) * 4u, b = (lane & 7u) ^ ro;
        if (!WHOLE && n >= N) return;
        e.template column<4>(n);
        float *p = st + ro * 32u;
        constexpr int TIMES = Epi::heavy ? 1 : 2;      // (gelu: 121 us as a loop, 127 unrolled; without an activation 103 and 104, f16 43 and 38)
#pragma unroll TIMES
        for (uint32_t t = 0; t < 8; t += 4) {          // row ro + 4 (t + i): swap of it = ro ^ (4 (i & 1)) ^ i ^ t
            float x[4][4], v[4][4];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
                if (m0 + ro + 4 * (t + i) < M) e.template fetch<4>(m0 + ro + 4 * (t + i), n, x[i]);
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const float4 q = *reinterpret_cast<const float4 *>(p + (t + i) * 128u + ((b ^ t ^ (((i & 1u) * 4u) ^ i)) << 2));
                v[i][0] = q.x; v[i][1] = q.y; v[i][2] = q.z; v[i][3] = q.w;
            }
            e.template put<4, 4>(Rows{m0 + ro + 4 * t, 4, M}, n, v, x, z);
            if constexpr (Epi::mirrors) {              // the finished values go back, for the mirror to store
#pragma unroll
                for (uint32_t i = 0; i < 4; i++)
                    *reinterpret_cast<float4 *>(p + (t + i) * 128u + ((b ^ t ^ (((i & 1u) * 4u) ^ i)) << 2)) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
            }
        }
    } else {
        const uint32_t n = n0 + lane;
        if (n >= N) return;
        e.template column<1>(n);
#pragma unroll 1
        for (uint32_t r0 = 0; r0 < 32u; r0 += 4) {
            float x[4][1], v[4][1];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                if (m0 + r0 + i < M) e.template fetch<1>(m0 + r0 + i, n, x[i]);
                v[i][0] = st[(r0 + i) * 32u + (((lane >> 2) ^ swap(r0 + i)) << 2) + (lane & 3u)];
            }
            e.template put<1, 4>(Rows{m0 + r0, 1, M}, n, v, x, z);
            if constexpr (Epi::mirrors) {
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) st[(r0 + i) * 32u + (((lane >> 2) ^ swap(r0 + i)) << 2) + (lane & 3u)] = v[i][0];
            }
        }
    }
}
template <int V, class Epi>
__device__ __forceinline__ void mirror_block(Epi &e, const float *st, uint32_t lane, uint32_t m0, uint32_t n0, uint32_t N) {
    constexpr uint32_t STEP = V == 4 ? 4 : 1;
    const uint32_t no = V == 4 ? lane >> 3 : 0u, mo = V == 4 ? (lane & 7u) * 4u : lane;
#pragma unroll 1
    for (uint32_t c0 = no; c0 < 32u; c0 += 4 * STEP) {
        float v[4][V];
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t c = c0 + i * STEP;
#pragma unroll
            for (uint32_t j = 0; j < V; j++) v[i][j] = st[(mo + j) * 32u + (((c >> 2) ^ swap(mo + j)) << 2) + (c & 3u)];
        }
        e.template mirror<V, 4>(Rows{n0 + c0, STEP, N}, m0 + mo, v);
    }
}
template <uint32_t NT, class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
k_hgemm(const __grid_constant__ Shape S, const __grid_constant__ Maps maps, const __grid_constant__ Epi epi) {
    extern __shared__ uint8_t raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    Shared &sh = *reinterpret_cast<Shared *>(base + RING_BYTES + STAGING);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, rank = cluster_cta();
    const uint32_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    volatile int *abort_flag = &sh.abort_flag;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < MAX_STAGES; s++) { bar_init(smem32(&sh.full[s]), 1); bar_init(smem32(&sh.empty[s]), 1); }
        for (int b = 0; b < 2; b++) { bar_init(smem32(&sh.acc_full[b]), 1); bar_init(smem32(&sh.acc_empty[b]), 2 * EPI_WARPS); }
        sh.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem32(&sh.tmem)), "r"(2u * NT) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    depend();
    const uint32_t tmem = sh.tmem;
    const uint32_t ring = smem32(base);
    constexpr uint32_t B_PLANE = NT / 2 * 128;             // bytes of this CTA's B plane of a block

    if (warp < EPI_WARPS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(EPI_REGS));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(IO_REGS));
    if (warp < EPI_WARPS) {
        // ================= epilogue: rows of this CTA, quadrant warp % 4; columns half warp / 4 =================
        constexpr uint32_t COLS = NT / 2;
        const uint32_t q = warp & 3u, half = warp >> 2;
        float *st = reinterpret_cast<float *>(base + RING_BYTES) + warp * 1024u;
        Epi e = epi;                                       // (keeps what belongs to the lane's columns)
        const bool wide = e.wide();
        bool ok = true;
        uint32_t c = 0;                                    // chunks so far
        for (uint32_t t = pair; t < S.tiles && ok; t += pairs) {
            const Tile T = tile_of<NT>(S, t);
            const uint32_t m0 = T.m0 + rank * 128u + q * 32u, n0 = T.n0 + half * COLS;
            if (m0 + lane < S.M) e.touch(m0 + lane, n0, COLS);         // what the result reads: into L2 while the sums are made
            float acc[COLS];
#pragma unroll
            for (uint32_t i = 0; i < COLS; i++) acc[i] = 0.0f;
            for (uint32_t kb = 0; kb < T.blocks && ok; kb = chunk_end(kb, S.chunk, S.lead), c++) {
                const uint32_t buf = c & 1u;
                ok = bar_wait(smem32(&sh.acc_full[buf]), (c >> 1) & 1u, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (uint32_t j = 0; j < COLS / 32; j++) {
                    uint32_t r[32];
                    acc_load(tmem + ((q * 32u) << 16) + buf * NT + half * COLS + j * 32u, r);
#pragma unroll
                    for (uint32_t i = 0; i < 32; i++) acc[j * 32 + i] += __uint_as_float(r[i]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive(in_cta(smem32(&sh.acc_empty[buf]), 0));
            }
            if (!ok) break;
            const float f = m0 + lane < S.M ? e.row_factor(m0 + lane) : 0.0f;
#pragma unroll 1
            for (uint32_t j = 0; j < COLS / 32; j++) {
                const uint32_t n1 = n0 + j * 32u;
                if (n1 >= S.N || m0 >= S.M) break;
                __syncwarp();
#pragma unroll
                for (uint32_t k = 0; k < COLS / 32; k++)           // (registers are picked by number, not by index)
                    if (k == j) {
#pragma unroll
                        for (uint32_t i = 0; i < 8; i++)
                            *reinterpret_cast<float4 *>(st + lane * 32u + ((i ^ swap(lane)) << 2)) = make_float4(acc[k * 32 + 4 * i] * f, acc[k * 32 + 4 * i + 1] * f, acc[k * 32 + 4 * i + 2] * f, acc[k * 32 + 4 * i + 3] * f);
                    }
                __syncwarp();
                bool above = false;
                if constexpr (Epi::mirrors) {
                    if (S.upper) {
                        if (n1 < m0) continue;                 // (blocks of 32 x 32: below the diagonal the mirror of one above writes)
                        above = n1 > m0;
                    }
                }
                if (wide && m0 + 32u <= S.M && n1 + 32u <= S.N) put_block<4, true>(e, st, lane, m0, n1, S.M, S.N, T.z);
                else if (wide) put_block<4, false>(e, st, lane, m0, n1, S.M, S.N, T.z);
                else put_block<1, false>(e, st, lane, m0, n1, S.M, S.N, T.z);
                if constexpr (Epi::mirrors) {
                    __syncwarp();
                    if (above) { if (wide) mirror_block<4>(e, st, lane, m0, n1, S.N); else mirror_block<1>(e, st, lane, m0, n1, S.N); }
                }
            }
        }
    } else if (warp == TMA_A_WARP || warp == TMA_B_WARP) {
        // ================= tile loads: one thread per CTA and operand =================
        if (lane == 0) {
            const bool is_a = warp == TMA_A_WARP;
            const CUtensorMap *map = is_a ? &maps.a : &maps.b;
            const uint32_t halves = S.halves, mode = is_a ? S.a_mode : S.b_mode, boxes = is_a ? 2u : NT / 128, width = is_a ? 128u : NT / 2, at = is_a ? 0u : S.a_bytes;
            bool ok = true;
            uint32_t it = 0, s = 0, use = 0;
            for (uint32_t t = pair; t < S.tiles && ok; t += pairs) {
                const Tile T = tile_of<NT>(S, t);
                const uint32_t mn = (is_a ? T.m0 : T.n0) + rank * width;
                for (uint32_t kb = 0; kb < T.blocks; kb++) {
                    if (use) ok = bar_spin(smem32(&sh.empty[s]), (use - 1) & 1u, abort_flag);
                    if (!ok) break;
                    if (is_a && rank == 0) bar_expect(smem32(&sh.full[s]), 2u * S.stage_bytes);
                    const uint32_t dst = ring + s * S.stage_bytes + at, bar = in_cta(smem32(&sh.full[s]), 0), k = (T.block0 + kb) * halves;
                    for (uint32_t h = 0; h < halves; h++) load_operand(dst + h * S.half_bytes, map, bar, mode, boxes, mn, (k + h) * KB);
                    it++;
                    if (++s == S.stages) { s = 0; use++; }
                }
            }
            if (!ok && rank == 0) {
                // give the copies in flight (both CTAs' signal here) time to land before shared memory is given up
                int never = 0;
                const uint32_t n = it < S.stages ? it : S.stages;
                for (uint32_t i = it - n; i < it; i++) bar_wait(smem32(&sh.full[i % S.stages]), (i / S.stages) & 1u, &never);
            }
        }
        __syncwarp();
    } else if (warp == MMA_WARP && rank == 0) {
        // ================= MMAs: one thread, for the pair =================
        if (lane == 0) {
            const uint32_t a_mn = S.a_mode != K_ROWS, b_mn = S.b_mode != K_ROWS;
            const uint32_t idesc = (1u << 4) | (a_mn << 15) | (b_mn << 16) | ((NT >> 3) << 17) | ((256u >> 4) << 24);   // f32 sums of f16 products
            const uint64_t step_a = a_mn ? 2048u >> 4 : 32u >> 4, step_b = b_mn ? 2048u >> 4 : 32u >> 4;                 // 16 k further
            const uint32_t lo = S.a_lo | S.b_lo << 1, halves = S.halves, chunk = S.chunk, lead = S.lead, stages = S.stages;
            const uint64_t a_first = operand_desc(ring, a_mn), b_first = operand_desc(ring + S.a_bytes, b_mn), half = S.half_bytes >> 4;
            bool ok = true;
            uint32_t s = 0, use = 0, c = 0;
            uint64_t at = 0;                               // of the stage, in the descriptors' units
            for (uint32_t t = pair; t < S.tiles && ok; t += pairs) {
                const Tile T = tile_of<NT>(S, t);
                for (uint32_t kb = 0; kb < T.blocks && ok; kb = chunk_end(kb, chunk, lead), c++) {
                    const uint32_t buf = c & 1u, d = tmem + buf * NT;
                    if (c >= 2) ok = bar_spin(smem32(&sh.acc_empty[buf]), ((c >> 1) - 1) & 1u, abort_flag);
                    const uint32_t next = chunk_end(kb, chunk, lead), end = (next < T.blocks ? next : T.blocks) - kb;
                    uint32_t more = 0;
                    for (uint32_t i = 0; i < end && ok; i++) {
                        ok = bar_spin(smem32(&sh.full[s]), use & 1u, abort_flag);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        uint64_t a_hi = a_first + at, b_hi = b_first + at;
                        for (uint32_t h = 0; h < halves; h++, a_hi += half, b_hi += half) {
                            if (lo & 1u) {
#pragma unroll
                                for (uint32_t k = 0; k < 4; k++) { mma(d, a_hi + (A_PLANE >> 4) + k * step_a, b_hi + k * step_b, idesc, more); more = 1; }
                            }
                            if (lo & 2u) {
#pragma unroll
                                for (uint32_t k = 0; k < 4; k++) { mma(d, a_hi + k * step_a, b_hi + (B_PLANE >> 4) + k * step_b, idesc, more); more = 1; }
                            }
#pragma unroll
                            for (uint32_t k = 0; k < 4; k++) { mma(d, a_hi + k * step_a, b_hi + k * step_b, idesc, more); more = 1; }
                        }
                        commit_both(smem32(&sh.empty[s]));
                        at += S.stage_bytes >> 4;
                        if (++s == stages) { s = 0; use++; at = 0; }
                    }
                    if (ok) commit_both(smem32(&sh.acc_full[buf]));
                }
            }
        }
        __syncwarp();
    }

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    if (threadIdx.x == 0 && sh.abort_flag) atomicOr(S.status, STATUS_TIMEOUT);
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2u * NT) : "memory");
    }
}

// Sums of a split product: partial[z][m][n] in split order, then the epilogue.
struct PartialEpi {
    static constexpr bool mirrors = false, long_start = false, heavy = false;
    float *partial; uint64_t mn; uint32_t N;
    __device__ bool wide() const { return N % 4 == 0; }
    __device__ float row_factor(uint32_t) const { return 1.0f; }
    __device__ void touch(uint32_t, uint32_t, uint32_t) const {}
    template <int V> __device__ void column(uint32_t) const {}
    template <int V> __device__ void fetch(uint32_t, uint32_t, float (&)[V]) const {}
    template <int V, int R> __device__ void put(Rows r, uint32_t n, const float (&v)[R][V], const float (&)[R][V], uint32_t z) const {
#pragma unroll
        for (uint32_t i = 0; i < R; i++) if (r.first + i * r.step < r.end) store_vec<V>(partial + z * mn + (uint64_t)(r.first + i * r.step) * N + n, v[i]);
    }
};
template <int V, class Epi>
__global__ void __launch_bounds__(256)
k_hgemm_fold(const float *partial, uint32_t splits, uint32_t M, uint32_t N, const __grid_constant__ Epi epi) {
    const uint32_t n = (blockIdx.x * 32 + (threadIdx.x & 31u)) * V;
    if (n >= N) return;
    depend();
    Epi e = epi;
    e.template column<V>(n);
    for (uint32_t m = blockIdx.y * 8 + (threadIdx.x >> 5); m < M; m += gridDim.y * 8) {
        float v[1][V], x[1][V];
        e.template fetch<V>(m, n, x[0]);
        load_vec<V>(partial + (uint64_t)m * N + n, v[0]);
        for (uint32_t z = 1; z < splits; z++) {
            float p[V];
            load_vec<V>(partial + ((uint64_t)z * M + m) * N + n, p);
#pragma unroll
            for (int j = 0; j < V; j++) v[0][j] += p[j];
        }
        const float f = e.row_factor(m);
#pragma unroll
        for (int j = 0; j < V; j++) v[0][j] *= f;
        e.template put<V, 1>(Rows{m, 1, M}, n, v, x, 0);
    }
}

// The same for a symmetric product, of which only the tiles from the diagonal on were made: a block of 256 threads takes 32 x 32 sums
// on or above it and writes them in both places.  Through shared memory as in the product's own epilogue, one warp's layout.
template <int V, class Epi>
__global__ void __launch_bounds__(256)
k_hgemm_fold_upper(const float *partial, uint32_t splits, uint32_t M, const __grid_constant__ Epi epi) {
    if (blockIdx.x < blockIdx.y) return;
    depend();
    __shared__ float st[32][33];
    const uint32_t m0 = blockIdx.y * 32, n0 = blockIdx.x * 32, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    Epi e = epi;
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
        const uint32_t m = m0 + warp + 8 * i, n = n0 + lane;
        float v = 0.0f;
        if (m < M && n < M) {
            for (uint32_t z = 0; z < splits; z++) v += partial[((uint64_t)z * M + m) * M + n];
            v *= e.row_factor(m);
        }
        st[warp + 8 * i][lane] = v;
    }
    __syncthreads();
    constexpr uint32_t PER = 32 / V;                       // threads a row
    for (uint32_t u = threadIdx.x; u < 32 * PER; u += 256) {
        const uint32_t r = u / PER, c = (u % PER) * V;
        if (m0 + r >= M || n0 + c >= M) continue;
        float x[1][V], v[1][V];
#pragma unroll
        for (uint32_t j = 0; j < V; j++) v[0][j] = st[r][c + j];
        e.template column<V>(n0 + c);
        e.template fetch<V>(m0 + r, n0 + c, x[0]);
        e.template put<V, 1>(Rows{m0 + r, 1, M}, n0 + c, v, x, 0);
#pragma unroll
        for (uint32_t j = 0; j < V; j++) st[r][c + j] = v[0][j];
    }
    __syncthreads();
    if (blockIdx.x > blockIdx.y)
        for (uint32_t u = threadIdx.x; u < 32 * PER; u += 256) {
            const uint32_t r = u / PER, c = (u % PER) * V;
            float v[1][V];
#pragma unroll
            for (uint32_t j = 0; j < V; j++) v[0][j] = st[c + j][r];
            if (n0 + r < M && m0 + c < M) e.template mirror<V, 1>(Rows{n0 + r, 1, M}, m0 + c, v);
        }
}

// ---- host ----
// One operand: one or two f16 planes of rows `pitch` values apart (a multiple of 8; base 16-byte aligned), the second `plane` values
// behind the first (0: there is none).  mn: the rows run along the operand's m or n, one row per k, and with two planes the pitch is
// a multiple of 64 and all of it may be read; otherwise along k.
struct Operand { const __half *p; uint64_t pitch, plane; bool mn; };

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// the operand's map and mode; rows: its m or n
static uint32_t operand_map(CUtensorMap *m, const Operand &o, uint32_t rows, uint32_t K, uint32_t tile_rows) {
    static EncodeTiled fn = nullptr;
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        THC_CUDA_OK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q));
        if (q != cudaDriverEntryPointSuccess) fatal("cuTensorMapEncodeTiled is not in this driver");
        fn = (EncodeTiled)p;
    }
    const uint32_t mode = !o.mn ? K_ROWS : o.pitch % 64 == 0 && (o.plane || rows % 64 == 0) ? MN_BLOCKS : MN_BOXES;
    const cuuint64_t planes = o.plane ? 2 : 1, pitch = o.pitch * 2, plane = o.plane ? o.plane * 2 : pitch;
    cuuint64_t dims[4], strides[3];
    cuuint32_t box[4];
    const cuuint32_t one[4] = {1, 1, 1, 1};
    if (mode == MN_BLOCKS) {
        dims[0] = 64; dims[1] = K; dims[2] = (rows + 63) / 64; dims[3] = planes;
        strides[0] = pitch; strides[1] = 128; strides[2] = plane;
        box[0] = 64; box[1] = KB; box[2] = tile_rows / 64; box[3] = (cuuint32_t)planes;
    } else {
        dims[0] = mode == K_ROWS ? K : rows; dims[1] = mode == K_ROWS ? rows : K; dims[2] = planes;
        strides[0] = pitch; strides[1] = plane;
        box[0] = 64; box[1] = mode == K_ROWS ? tile_rows : KB; box[2] = (cuuint32_t)planes;
    }
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, mode == MN_BLOCKS ? 4 : 3, const_cast<__half *>(o.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) fatal("tensor map of %u x %u values, pitch %llu: error %d", rows, K, (unsigned long long)o.pitch, (int)r);
    return mode;
}

struct Plan { uint32_t nt, splits; uint64_t partial_bytes; };
static uint32_t count_tiles(uint32_t M, uint32_t N, uint32_t nt, bool upper) {
    const uint32_t rows = (M + 255) / 256, cols = (N + nt - 1) / nt;
    uint32_t n = rows * cols;
    if (upper) { n = 0; for (uint32_t r = 0; r < rows; r++) n += cols - r * 256 / nt; }
    return n;
}
// Tile width and splits over K for an M x N product: the least time in cycles by what the parts of one cost, measured.  A block of 64 k
// with planes on both sides takes a pair 1900 cycles at 256 columns and 1500 at 128 (where issuing the MMAs is what takes long), one of
// 128 k without planes 1550 and 1200; a tile's epilogue, as far as the next tile does not hide it, 4000 and 2000; the second kernel
// that a split needs 9000, and the split's sums 3500 bytes a cycle, written and read.  4096 x 1024 x 4096: 64 wide tiles, 76 us; 128
// narrow ones in two rounds, 137 us.
static Plan plan(uint32_t M, uint32_t N, uint32_t K, bool planes, bool upper) {
    const uint32_t pairs = (uint32_t)g.sm_count / 2, blocks = (K + (planes ? 63 : 127)) / (planes ? 64 : 128);
    Plan best{256, 1, 0};
    double least = 0;
    for (uint32_t nt = 256; nt >= 128; nt -= 128) {
        const uint32_t tiles = count_tiles(M, N, nt, upper);
        const double block = planes ? (nt == 256 ? 1900 : 1500) : (nt == 256 ? 1550 : 1200), end = nt == 256 ? 4000 : 2000;
        for (uint32_t s = 1; s <= 16 && (s == 1 || 2 * s <= blocks); s++) {
            const double rounds = (double)(((uint64_t)tiles * s + pairs - 1) / pairs);
            double t = rounds * (((blocks + s - 1) / s) * block + end);
            if (s > 1) t += 9000 + (double)s * M * N * (upper ? 4.5 : 8) / 3500;
            if (least == 0 || t < least) { least = t; best = Plan{nt, s, s > 1 ? (uint64_t)s * M * N * 4 : 0}; }
        }
    }
    return best;
}

template <uint32_t NT, class Epi>
static void launch(const Shape &S, const Maps &maps, const Epi &epi, const char *name) {
    static int seen = -1;
    if (first_on_device(seen)) THC_CUDA_OK(cudaFuncSetAttribute(k_hgemm<NT, Epi>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM));
    layer_estimate(2.0 * S.M * S.N * S.K, (S.M + (double)S.N) * S.K * (S.a_lo | S.b_lo ? 4 : 2) + 4.0 * S.M * S.N);
    const uint32_t pairs = (uint32_t)g.sm_count / 2;
    profile_begin();
    chain(k_hgemm<NT, Epi>, dim3(2 * (S.tiles < pairs ? S.tiles : pairs)), THREADS, SMEM, S, maps, epi);
    after_launch(name);
}

// A (M rows) times B (N rows) over K.  `partial`: plan.partial_bytes of scratch.  `upper`: a symmetric product (A = B): tiles
// below the diagonal are left out and the epilogue mirrors the others.
template <class Epi>
static void product(const Operand &A, const Operand &B, uint32_t M, uint32_t N, uint32_t K, const Plan &p, float *partial, const Epi &epi, bool upper, const char *name) {
    Shape S;
    memset(&S, 0, sizeof S);
    S.M = M; S.N = N; S.K = K;
    S.row_tiles = (M + 255) / 256; S.col_tiles = (N + p.nt - 1) / p.nt;
    S.halves = A.plane || B.plane ? 1 : 2;
    S.blocks = (K + KB * S.halves - 1) / (KB * S.halves);
    S.split_blocks = (S.blocks + p.splits - 1) / p.splits;
    const uint32_t splits = (S.blocks + S.split_blocks - 1) / S.split_blocks;          // p.splits or fewer
    S.a_lo = A.plane != 0; S.b_lo = B.plane != 0;
    S.chunk = S.a_lo || S.b_lo ? 2 : 8;
    S.lead = !(S.a_lo || S.b_lo) || Epi::long_start ? 2 : 1;
    S.a_bytes = A_PLANE * (1 + S.a_lo);
    S.half_bytes = S.a_bytes + p.nt / 2 * 128 * (1 + S.b_lo);
    S.stage_bytes = S.half_bytes * S.halves;
    S.stages = RING_BYTES / S.stage_bytes;
    if (S.stages > MAX_STAGES) S.stages = MAX_STAGES;
    S.upper = upper;
    S.split_tiles = count_tiles(M, N, p.nt, upper);
    S.tiles = S.split_tiles * splits;
    S.status = g.dev_status;
    Maps maps;
    S.a_mode = operand_map(&maps.a, A, M, K, 128);
    S.b_mode = operand_map(&maps.b, B, N, K, p.nt / 2);
    if (splits > 1) {
        const PartialEpi pe{partial, (uint64_t)M * N, N};
        if (p.nt == 256) launch<256>(S, maps, pe, name); else launch<128>(S, maps, pe, name);
        profile_begin();
        if constexpr (Epi::mirrors) {
            const dim3 grid((N + 31) / 32, (M + 31) / 32);
            if (N % 4 == 0) chain(k_hgemm_fold_upper<4, Epi>, grid, 256, 0, (const float *)partial, splits, M, epi);
            else chain(k_hgemm_fold_upper<1, Epi>, grid, 256, 0, (const float *)partial, splits, M, epi);
        } else {
            const uint32_t down = (M + 7) / 8 < 4096 ? (M + 7) / 8 : 4096;
            if (N % 4 == 0) chain(k_hgemm_fold<4, Epi>, dim3((N + 127) / 128, down), 256, 0, (const float *)partial, splits, M, N, epi);
            else chain(k_hgemm_fold<1, Epi>, dim3((N + 31) / 32, down), 256, 0, (const float *)partial, splits, M, N, epi);
        }
        after_launch("layer_fold");
        return;
    }
    if (p.nt == 256) launch<256>(S, maps, epi, name); else launch<128>(S, maps, epi, name);
}

}  // namespace hg
}  // namespace thc
