// linear_xent.cu -- classifier product and softmax cross-entropy in one operator, forward and backward, in pieces of the
// vocabulary and without ever keeping the logits:
//
//   l[v][t]   = sum_d table[v][d] * x[d][t]
//   loss_t    = -log(exp(l[tgt] - lse_t) + 1e-10),  lse_t = log sum_v exp(l[v][t])
//   dl[v][t]  = (exp(l[v][t] - lse_t) - [v == tgt_t]) * grad_scale / S         (0 for a token without a target)
//   dx        = table^T dl         d_table += dl x^T
//
// Four matrix products on the tensor cores (fp32 accumulation):
//   stats     l, reduced on the fly to a (max, sum of exp) pair per token and tile of 256 vocabulary rows
//   dlogits   l once more for one piece of the vocabulary, turned into dl and written to scratch in 16 bits
//   dx        dl x table, added to an fp32 sum over the pieces
//   d_table   x x dl, added to the caller's fp32 gradient
// Writing the logits and reading them back would take longer than the second product: 12 bytes per logit (write, read, write
// dl) at 6.5 TB/s are 1.9 ps, 2 * 1024 operations at 1.5 PFLOP/s are 1.4 ps.
//
// Measured, 8192 tokens x 151936 rows x 1024 channels in bf16 (cuBLAS on this GPU: 1650 TFLOP/s in a burst, 1410 under the
// power cap), launches one after the other: stats 1.49 ms (1710 TFLOP/s), dlogits 2.15 (1190; it writes 5 GB of dl), dx 1.72
// (1490), d_table 3.13 for two products (1630).  Back to back under the power cap the whole call takes 9.6 to 10.1 ms, 1290
// TFLOP/s over the five products that it does and 780 over the three that the result cannot do without.
//
// Precision.  16-bit inputs enter the products as they are.  dl is rounded to 16 bits for dx, whose result is rounded to 16
// bits as well; d_table is an fp32 sum, so dl enters it as two 16-bit numbers, the rounded value and what the rounding left
// (17 bits and more), at the price of one more product.  fp32 inputs are split into two fp16 parts after scaling by a power of
// two that puts the tensor's largest magnitude at 2^13: 22 bits of every number above 2^-28 of the largest.  Every product is
// then low*high + high*low + high*high; what is dropped is below 2^-22 of a term.  Where dl is held in fp16 it is scaled by
// 2^14 (|dl| * S / grad_scale <= 1 becomes 16384 at most), so that the probabilities of a large vocabulary, 1e-5 and less, do
// not fall among fp16's subnormals.
//
// The accumulators of the tensor cores cut off what does not fit instead of rounding: every step of 16 along K takes half a
// unit of the last place from the sum on average, 3e-8 of it (measured: 1.2e-5 after 345 steps).  So fp32 results leave the
// accumulator after 32 steps and are added up in registers with rounding; the logits of fp32 inputs after 72 (leaving more often
// lets the matrix thread run less far ahead of the epilogue: dlogits 125 us against 108 for 4096 tokens over 9200 rows).
//
// A token without a target (id outside [0, V)) has zeros in place of its x, so that nothing it holds -- infinities and NaN
// included -- reaches d_table.
#include "common.cuh"
#include "tma.cuh"

#include <math.h>

namespace ane {

constexpr float LX_LOG2E = 1.4426950408889634f;

enum LxEpilogue { LX_STATS, LX_DLOGITS, LX_DX, LX_DTABLE };
// What a stage of the ring holds and what is done with it:
//   LX_PLAIN   A, B           one accumulator (the other one belongs to the next tile)
//   LX_WIDE    A, B, B'       B' = the next 256 rows of the output's columns: both accumulators make one 256 x 512 tile
//   LX_TWO     A, B, B'       B' = the low part of B: both products into one accumulator
//   LX_SPLIT   A, B, B', A'   fp32 inputs, A' and B' the low parts: A' B, A B' and A B into one accumulator
//   LX_NARROW  the same with tiles of 256 x 128
enum LxMode { LX_PLAIN, LX_WIDE, LX_TWO, LX_SPLIT, LX_NARROW };

constexpr int LX_CTA_M = 128;                            // rows of the tile in each block of a pair
constexpr int LX_BM = 2 * LX_CTA_M, LX_BN = 256, LX_BK = 64;      // one accumulator: M x N outputs of a pair; K elements per stage
constexpr int LX_BOX_BYTES = LX_CTA_M * LX_BK * 2;                // a block's 128 rows of one operand
constexpr int LX_EPI_WARPS = 8;                          // two for each 32 accumulator lanes, half of the columns each
constexpr int lx_acc_n(int mode) { return mode == LX_NARROW ? LX_BN / 2 : LX_BN; }
constexpr int LX_THREADS = 64 + 32 * LX_EPI_WARPS;       // copy warp, matrix warp, epilogue warps
constexpr int LX_RING_BOXES = 12;                        // of operands
constexpr int LX_STAGING_BYTES = 2 * 32 * 64;            // dlogits: an epilogue warp's 32 rows x 32 columns of both parts
constexpr size_t lx_smem(int epi) { return (size_t)LX_RING_BOXES * LX_BOX_BYTES + (epi == LX_DLOGITS ? LX_EPI_WARPS * LX_STAGING_BYTES : 0) + 1024; }
constexpr int LX_STEPS = 32;                             // of 16 along K that stay in an accumulator where an fp32 result is wanted
constexpr int LX_WAIT_LIMIT = 1 << 20;
constexpr float LX_HALF_SCALE = 16384.0f;                // of dl where it is held in fp16

struct LxMaps { CUtensorMap a[2], b[2], hi, lo; };       // operands and their low parts; dlogits: where dl goes
struct LxArgs {
    int kblocks;
    int splits;                // shares of the K blocks, each with its own sums (dx only)
    int span;                  // K blocks that one accumulator sums before its values move to registers
    int m_tiles, n_tiles;
    int m, n;                  // valid rows and columns of the output
    uint32_t idesc;
    // stats, dlogits: m = tokens, n = vocabulary rows of the piece from v0
    const void *targets;       // of the first token
    int id_u16, V, v0;
    const float *scales;       // fp32 inputs: {1 / scale of x, 1 / scale of the table}; else null
    float2 *part; int tile0;   // stats: [half vocabulary tile][ldt], this piece's first
    float *hit;                // stats: the target's logit per token
    const float *lse2;         // dlogits: lse * log2(e)
    int two_parts;             // dlogits: the low parts of dl are wanted
    float dscale;
    // dx: [split][column][ldt] sums; d_table: [column][D]
    float *out; size_t ldt; int first;
    float alpha;
    int half_type;             // 1 when the 16-bit operands are fp16
    ane_cuda_status *status;
};

// ------------------------------------------------------------------ tensor-core primitives
// Shared-memory operand descriptor, 128-byte swizzle.  K-major: rows of 64 K elements, eight rows per 1024-byte group.
// MN-major: 64 M (or N) elements per 128-byte row, one row per k, eight k per group, the next 64 M after `lead` bytes.
__device__ __forceinline__ uint64_t lx_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void lx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives on the barrier of this offset in both blocks of the pair once the matrix instructions issued so far are done.
__device__ __forceinline__ void lx_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void lx_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void lx_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Address of the first block's copy of a shared variable.
__device__ __forceinline__ uint32_t lx_in_leader(const void *p) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
    return r;
}
// Relaxed: what has to come before it are reads of the accumulator, which have completed (a release would wait for this
// thread's global stores as well, and hold the accumulator that long).
__device__ __forceinline__ void lx_arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A box into this block's shared memory, counted on a barrier of the pair's first block.
__device__ __forceinline__ void lx_load_box(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool lx_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void lx_pair_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 32 accumulator columns of this warp's 32 lanes: v[j] = column + j of the thread's own row.
__device__ __forceinline__ void lx_tmem_load(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
                 "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
                   "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ float lx_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void lx_add(float *p, float v) { asm volatile("red.global.add.f32 [%0], %1;" ::"l"(p), "f"(v) : "memory"); }

// Bounded wait that also ends when another role of the block gave up.
__device__ __forceinline__ bool lx_wait(uint64_t *bar, uint32_t parity, volatile int *abort) {
    for (int i = 0; i < LX_WAIT_LIMIT; i++) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort) return false;
    }
    *abort = 1;
    return false;
}

__device__ __forceinline__ int lx_target(const void *targets, int id_u16, int V, int t) {
    const int id = id_u16 ? (int)static_cast<const uint16_t *>(targets)[t] : static_cast<const int32_t *>(targets)[t];
    return id >= 0 && id < V ? id : -1;
}

// Two fp32 values -> their 16-bit roundings, and the roundings of what was left.
template <bool HALF> __device__ __forceinline__ void lx_split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    if constexpr (HALF) {
        const __half2 h = __floats2half2_rn(a, b);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
        hi = *reinterpret_cast<const uint32_t *>(&h);
        lo = *reinterpret_cast<const uint32_t *>(&l);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        const __nv_bfloat162 l = __floats2bfloat162_rn(a - __low2float(h), b - __high2float(h));
        hi = *reinterpret_cast<const uint32_t *>(&h);
        lo = *reinterpret_cast<const uint32_t *>(&l);
    }
}
__device__ __forceinline__ void lx_store_shared(uint32_t at, const uint32_t (&w)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}
// A box out of shared memory; columns and rows outside the matrix are left out.
__device__ __forceinline__ void lx_store_box(const CUtensorMap *map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(src) : "memory");
}

// The K blocks of one tile: the tile's share [k0, k1), in parts of `span`.
struct LxRange {
    int k0, k1, span, part, k;
    __device__ __forceinline__ LxRange(const LxArgs &a, int tile) {
        const int ks = tile / (a.m_tiles * a.n_tiles);
        k0 = (int)((long long)a.kblocks * ks / a.splits);
        k1 = (int)((long long)a.kblocks * (ks + 1) / a.splits);
        span = a.span;
        part = k = k0;
    }
    __device__ __forceinline__ bool done() const { return k >= k1; }
    __device__ __forceinline__ bool first() const { return k == part || k >= k1; }       // at the beginning of a part (or past the last)
    __device__ __forceinline__ void next() {
        if (++k == part + span) part = k;
    }
};

// ------------------------------------------------------------------ the product
// Pairs of blocks on neighbouring SMs work on accumulators of 256 x 256 outputs: each block holds 128 rows of A, 128 of B's 256
// rows and the accumulator of its own 128 output rows, and the matrix instructions of the first block read both blocks'
// operands.  In each block one thread copies operand boxes into a ring of stages; in the first block one thread issues the
// matrix instructions; eight warps take the accumulators over.
//
// A 256 x 256 tile wants 64 bytes per SM and clock from L2 and 256 x 512 wants 48, so the large products bring two boxes of B for
// each box of A (LX_WIDE, LX_TWO): d_table went from 1137 to 1414 TFLOP/s with it.  fp32 inputs need 43 with all four parts in one
// stage for their three products; a pass for each product took 708 us instead of 629 for the losses of 4096 tokens over 32000
// rows, 2440 instead of 2240 with gradients.  The second half of the distance was the
// matrix thread itself: with descriptors computed in vector registers a K block took 1450 clocks instead of the 1024 of its
// instructions (stats 1350 -> 1590 TFLOP/s with uniform registers).
template <int EPI, int MODE, bool HALF>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LX_THREADS, 1) lx_gemm_kernel(const __grid_constant__ LxMaps maps, const __grid_constant__ LxArgs a) {
    constexpr bool A_MN = EPI == LX_DTABLE, B_MN = EPI == LX_DX || EPI == LX_DTABLE;
    constexpr bool SPLIT = MODE == LX_SPLIT || MODE == LX_NARROW, LOW_B = MODE == LX_TWO || SPLIT, SUMS = SPLIT || EPI == LX_DX || EPI == LX_DTABLE;
    constexpr int ACC_N = lx_acc_n(MODE), COLS = ACC_N / 2;      // columns of an accumulator, of an epilogue warp
    constexpr int ACCS = MODE == LX_WIDE ? 2 : 1, TILE_N = ACCS * ACC_N;
    // a stage: A, one or two boxes of B, A'
    constexpr int B_BYTES = COLS * LX_BK * 2, B_BOXES = MODE == LX_PLAIN ? 1 : 2, LOW_A = LX_BOX_BYTES + B_BOXES * B_BYTES;
    constexpr int STAGE_BYTES = LOW_A + (SPLIT ? LX_BOX_BYTES : 0), STAGES = LX_RING_BOXES * LX_BOX_BYTES / STAGE_BYTES;
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;       // the same offset in both blocks
    // full and acc_empty are used in the first block only; the others are each block's own
    __shared__ uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], drained;
    __shared__ uint32_t tmem_at;
    __shared__ int give_up;
    volatile int *abort = &give_up;

    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; i++) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; i++) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 2 * LX_EPI_WARPS); }
        mbar_init(&drained, 1);
        give_up = 0;
        mbar_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        lx_fence_before();
    }
    __syncthreads();
    lx_pair_sync();
    lx_fence_after();
    const uint32_t tmem = tmem_at;
    dep_sync();                                           // nothing before this reads or writes global memory

    const int tiles = a.m_tiles * a.n_tiles * a.splits;
    uint32_t issued = 0;                                  // copy warp: K blocks whose copies were started

    // The copy warp and the matrix warp run their loops with all lanes, so that addresses and descriptors stay in uniform
    // registers, and elect one lane for the instructions that start something.
    if (warp == 0) {
        uint32_t st = 0, phase = 1;
        bool ok = true;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            const int mt = tile % a.m_tiles, nt = tile / a.m_tiles % a.n_tiles;
            const int am = mt * LX_BM + rank * LX_CTA_M, bn = nt * TILE_N + rank * COLS;
            for (LxRange r(a, tile); !r.done(); r.next()) {
                if (!(ok = __all_sync(0xffffffffu, lx_wait(&empty[st], phase, abort)))) break;
                if (lx_elect()) {
                    const int k = r.k * LX_BK;
                    const uint32_t sa = base + st * STAGE_BYTES, bar = lx_in_leader(&full[st]);
                    if (rank == 0) mbar_arrive_expect_tx(&full[st], 2 * STAGE_BYTES);
#pragma unroll
                    for (int h = 0; h < (SPLIT ? 2 : 1); h++) {
                        const uint32_t at = sa + h * LOW_A;
                        if constexpr (A_MN) {
#pragma unroll
                            for (int i = 0; i < LX_CTA_M / 64; i++) lx_load_box(at + i * 8192, &maps.a[h], am + i * 64, k, bar);
                        } else {
                            lx_load_box(at, &maps.a[h], k, am, bar);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < B_BOXES; h++) {
                        const CUtensorMap *map = &maps.b[LOW_B ? h : 0];
                        const uint32_t sb = sa + LX_BOX_BYTES + h * B_BYTES;
                        const int n = bn + (MODE == LX_WIDE ? h * ACC_N : 0);
                        if constexpr (B_MN) {
#pragma unroll
                            for (int i = 0; i < COLS / 64; i++) lx_load_box(sb + i * 8192, map, n + i * 64, k, bar);
                        } else {
                            lx_load_box(sb, map, k, n, bar);
                        }
                    }
                }
                __syncwarp();
                issued++;
                if (++st == STAGES) { st = 0; phase ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            uint32_t st = 0, phase = 0, turn = 0;
            bool ok = true;
            const uint64_t da = lx_desc(base, A_MN ? 8192 : 16), db = lx_desc(base, B_MN ? 8192 : 16);
            // the product of a stage's A (or A') and box `box` of B into accumulator `acc`
            auto product = [&](uint32_t stage, bool low_a, int box, uint32_t acc, bool more) {
                const uint64_t sa = da + (stage * (STAGE_BYTES >> 4) + (low_a ? LOW_A >> 4 : 0)), sb = db + (stage * (STAGE_BYTES >> 4) + ((LX_BOX_BYTES + box * B_BYTES) >> 4));
#pragma unroll
                for (int i = 0; i < LX_BK / 16; i++) lx_mma(tmem + acc * LX_BN, sa + i * (A_MN ? 128 : 2), sb + i * (B_MN ? 128 : 2), a.idesc, i > 0 || more);
            };
            auto wait = [&](uint64_t *bar, uint32_t parity) {
                ok = __all_sync(0xffffffffu, lx_wait(bar, parity, abort));
                lx_fence_after();
                return ok;
            };
            for (int tile = pair; tile < tiles && ok; tile += pairs) {
                if constexpr (MODE == LX_WIDE) {
                    // Both accumulators share every box of A.  They are taken over one after the other, so the first one runs ahead:
                    // by all stages but one at the beginning of a tile, where the second is still being read, and by two K blocks
                    // at the end.
                    const LxRange r(a, tile);
                    const int n = r.k1 - r.k0;
                    for (int i = 0; i < n && ok;) {
                        const int left = n - i, group = i == 0 ? (left < STAGES - 1 ? left : STAGES - 1) : left == 2 ? 2 : 1;
                        if (i == 0 && !wait(&acc_empty[0], ((turn >> 1) & 1) ^ 1)) break;
                        uint32_t s = st, ph = phase;
                        for (int j = 0; j < group; j++) {
                            if (!wait(&full[s], ph)) break;
                            if (lx_elect()) product(s, false, 0, 0, i + j > 0);
                            __syncwarp();
                            if (++s == STAGES) { s = 0; ph ^= 1; }
                        }
                        if (!ok) break;
                        if (i + group == n && lx_elect()) lx_commit(&acc_full[0]);
                        __syncwarp();
                        if (i == 0 && !wait(&acc_empty[1], ((turn >> 1) & 1) ^ 1)) break;
                        for (int j = 0; j < group; j++) {
                            if (lx_elect()) {
                                product(st, false, 1, 1, i + j > 0);
                                lx_commit(&empty[st]);
                            }
                            __syncwarp();
                            if (++st == STAGES) { st = 0; phase ^= 1; }
                        }
                        if (i + group == n && lx_elect()) lx_commit(&acc_full[1]);
                        __syncwarp();
                        i += group;
                    }
                    if (n > 0) turn += 2;
                } else {
                    bool more = false;
                    for (LxRange r(a, tile); !r.done();) {
                        if (r.first()) {
                            if (!wait(&acc_empty[turn & 1], ((turn >> 1) & 1) ^ 1)) break;
                            more = false;
                        }
                        if (!wait(&full[st], phase)) break;
                        r.next();
                        const bool last = r.first();                  // the accumulator is complete
                        if (lx_elect()) {
                            if constexpr (SPLIT) product(st, true, 0, turn & 1, more);
                            if constexpr (LOW_B) product(st, false, 1, turn & 1, more || SPLIT);
                            product(st, false, 0, turn & 1, more || LOW_B);
                            lx_commit(&empty[st]);
                            if (last) lx_commit(&acc_full[turn & 1]);
                        }
                        __syncwarp();
                        more = true;
                        turn += last;
                        if (++st == STAGES) { st = 0; phase ^= 1; }
                    }
                }
            }
            if (lx_elect()) lx_commit(&drained);              // also after a give-up: no instruction or arrival outlives the block
            __syncwarp();
        }
        mbar_wait_bounded(&drained, 0);
    } else {
        const int quad = warp & 3, row = quad * 32 + lane;   // a warp reads the accumulator lanes of its place in the group of four
        const int c0 = warp >= 2 + LX_EPI_WARPS / 2 ? COLS : 0;
        uint32_t turn = 0;
        bool ok = true;
        const float unscale = a.scales ? (EPI == LX_DTABLE ? a.scales[0] : EPI == LX_DX ? a.scales[1] : a.scales[0] * a.scales[1]) : 1.0f;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            const int mt = tile % a.m_tiles, nt = tile / a.m_tiles % a.n_tiles, ks = tile / (a.m_tiles * a.n_tiles);
            const int m = mt * LX_BM + rank * LX_CTA_M + row;
            const bool live = m < a.m;
            const LxRange range(a, tile);
            const bool none = range.k0 >= range.k1;          // a share without K blocks
            int id = -1;
            float lse2 = 0.0f;
            if constexpr (EPI == LX_STATS || EPI == LX_DLOGITS) id = live ? lx_target(a.targets, a.id_u16, a.V, m) : -1;
            if constexpr (EPI == LX_DLOGITS) lse2 = live ? a.lse2[m] : 0.0f;
            for (int h = 0; h < ACCS && ok; h++) {
                const int n0 = nt * TILE_N + h * ACC_N + c0;
                const int left = a.n - n0, cols = left < 0 ? 0 : left < COLS ? left : COLS;     // of this warp
                // This warp's columns into registers; the accumulator is free again before anything is computed.
                float v[COLS];
                if constexpr (SUMS) {
#pragma unroll
                    for (int j = 0; j < COLS; j++) v[j] = 0.0f;
                }
                for (int part = range.k0; part < range.k1; part += a.span, turn++) {
                    ok = __all_sync(0xffffffffu, lx_wait(&acc_full[turn & 1], (turn >> 1) & 1, abort));
                    if (!ok) break;
                    lx_fence_after();
                    const uint32_t t = tmem + (turn & 1) * LX_BN + c0 + ((uint32_t)(quad * 32) << 16);
#pragma unroll
                    for (int c = 0; c < COLS; c += 32) {
                        float w[32];
                        lx_tmem_load(t + c, w);
#pragma unroll
                        for (int j = 0; j < 32; j++) {
                            if constexpr (SUMS) v[c + j] += w[j];
                            else v[c + j] = w[j];
                        }
                    }
                    lx_fence_before();
                    __syncwarp();
                    if (lane == 0) lx_arrive_at(lx_in_leader(&acc_empty[turn & 1]));
                }
                if (!ok) break;
                if constexpr (EPI == LX_STATS) {
                    const int tgt = id >= 0 ? id - a.v0 - n0 : -1;     // column of this warp
                    const float k2 = unscale * LX_LOG2E;
                    if (__any_sync(0xffffffffu, tgt >= 0 && tgt < COLS)) {
                        float hit = 0.0f;
#pragma unroll
                        for (int j = 0; j < COLS; j++) hit = tgt == j ? v[j] : hit;
                        if (tgt >= 0 && tgt < COLS) a.hit[m] = hit * unscale;
                    }
                    if (cols < COLS) {
#pragma unroll
                        for (int j = 0; j < COLS; j++) if (j >= cols) v[j] = -INFINITY;
                    }
                    float top[4] = {v[0], v[1], v[2], v[3]}, sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int j = 4; j < COLS; j++) top[j & 3] = fmaxf(top[j & 3], v[j]);
                    const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * k2;
#pragma unroll
                    for (int j = 0; j < COLS; j++) sum[j & 3] += lx_exp2(fmaf(v[j], k2, -mx));
                    if (live && cols > 0) a.part[(size_t)(a.tile0 + (n0 / COLS)) * a.ldt + m] = make_float2(mx, (sum[0] + sum[1]) + (sum[2] + sum[3]));
                } else if constexpr (EPI == LX_DLOGITS) {
                    const int tgt = id >= 0 ? id - a.v0 - n0 : -1;
                    const float k2 = unscale * LX_LOG2E;
                    const float shift = log2f(a.dscale) - lse2;          // a power of two: exp2 brings it in
                    const bool mine = __any_sync(0xffffffffu, tgt >= 0 && tgt < COLS);
                    const int row0 = mt * LX_BM + rank * LX_CTA_M + quad * 32;
                    const uint32_t stage = base + STAGES * STAGE_BYTES + (warp - 2) * LX_STAGING_BYTES;
                    // 32 columns at a time through this warp's shared memory to the copy engine: 64-byte rows, swizzled as it
                    // expects them.  Straight to memory a lane writes its own row, 32 lines per instruction: this product took
                    // 22.2 us instead of 20.0 for one sequence over 9200 rows, 2.22 ms instead of 2.15 for 8192 tokens over
                    // 151936 (the whole call there: the same within its spread, the power cap sets it).
#pragma unroll
                    for (int c = 0; c < COLS; c += 32) {
                        if (c >= cols || row0 >= a.m) break;
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");     // the staging is free again
                        __syncwarp();
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            uint32_t hi[4], lo[4];
                            float e[8];
#pragma unroll
                            for (int j = 0; j < 8; j++) e[j] = lx_exp2(fmaf(v[c + q * 8 + j], k2, shift));
                            if (mine) {
#pragma unroll
                                for (int j = 0; j < 8; j++) e[j] = tgt == c + q * 8 + j ? e[j] - a.dscale : e[j];
                            }
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                lx_split2<HALF>(e[2 * j], e[2 * j + 1], hi[j], lo[j]);
                                if (id < 0) hi[j] = lo[j] = 0;           // a masked token: zeros, whatever its logits are
                            }
                            const uint32_t at = stage + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4);
                            lx_store_shared(at, hi);
                            lx_store_shared(at + LX_STAGING_BYTES / 2, lo);
                        }
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            lx_store_box(&maps.hi, stage, n0 + c, row0);
                            if (a.two_parts) lx_store_box(&maps.lo, stage + LX_STAGING_BYTES / 2, n0 + c, row0);
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                    }
                } else if (live) {
                    // dx: rows are tokens, columns are channels; d_table: rows are channels, columns vocabulary rows.  Either way
                    // the 32 lanes of a warp hold 32 neighbours of a contiguous row.
                    float *out = a.out + ((size_t)(EPI == LX_DX ? ks : 0) * a.n + n0) * a.ldt + m;
                    const float k = EPI == LX_DTABLE ? a.alpha * unscale : unscale;
                    if (EPI == LX_DX && a.first) {
#pragma unroll
                        for (int j = 0; j < COLS; j++) if (j < cols) out[(size_t)j * a.ldt] = v[j] * k;
                    } else if (!none) {
#pragma unroll
                        for (int j = 0; j < COLS; j++) if (j < cols) lx_add(out + (size_t)j * a.ldt, v[j] * k);
                    }
                }
            }
        }
    }
    if (EPI == LX_DLOGITS && warp >= 2 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
    lx_fence_before();
    __syncthreads();
    if (*abort && threadIdx.x == 0) {
        // copies still on their way into shared memory: every stage's last one, counted in the first block
        if (rank == 0)
            for (uint32_t i = issued > STAGES ? issued - STAGES : 0; i < issued; i++) mbar_wait_bounded(&full[i % STAGES], (i / STAGES) & 1);
        atomicAdd(&a.status->wait_giveups, 1);
    }
    __syncthreads();
    lx_pair_sync();                                       // the other block may still arrive on, or read from, this one's memory
    lx_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// ------------------------------------------------------------------ around the products
// fp32 inputs: the largest finite magnitude that each block finds in x (the first x_blocks; where a token has a target) or in the
// table, as the bits of a float, which compare like integers.
constexpr int LX_LARGEST_BLOCKS = 1184;
__global__ void __launch_bounds__(256) lx_largest_kernel(uint32_t *most, int x_blocks, const float *__restrict__ x, size_t nx, const float *__restrict__ table, size_t ne,
                                                         const void *__restrict__ targets, int id_u16, int V, int D, int S) {
    dep_sync();
    const bool of_x = blockIdx.x < x_blocks;
    const int first = of_x ? 0 : x_blocks, blocks = of_x ? x_blocks : gridDim.x - x_blocks;
    const float *p = of_x ? x : table;
    const size_t n = of_x ? nx : ne;
    uint32_t top = 0;
    const bool small = n <= 0xffffffffu;                     // 64-bit divisions are five times as long
    auto has_target = [&](size_t i) {
        const uint32_t j = (uint32_t)i;
        return lx_target(targets, id_u16, V, small ? (int)(j / ((uint32_t)D * S) * S + j % S) : (int)(i / ((size_t)D * S) * S + i % S)) >= 0;
    };
    auto look = [&](float f, size_t i) {
        const uint32_t u = __float_as_uint(f) & 0x7fffffffu;
        if (u > top && u < 0x7f800000u && (!of_x || has_target(i))) top = u;
    };
    const size_t step = (size_t)blocks * 256, at = (size_t)(blockIdx.x - first) * 256 + threadIdx.x, quads = aligned16(p) ? n / 4 : 0;
    for (size_t i = at; i < quads; i += 4 * step) {
        float4 q[4];
#pragma unroll
        for (int u = 0; u < 4; u++) q[u] = i + u * step < quads ? reinterpret_cast<const float4 *>(p)[i + u * step] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const size_t j = 4 * (i + u * step);
            look(q[u].x, j); look(q[u].y, j + 1); look(q[u].z, j + 2); look(q[u].w, j + 3);
        }
    }
    for (size_t i = 4 * quads + at; i < n; i += step) look(p[i], i);
    __shared__ uint32_t sh[8];
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; i++) top = sh[i] > top ? sh[i] : top;
        most[blockIdx.x] = top;
    }
}
// The exponent of the power of two that puts the largest magnitude of `blocks` blocks at 2^13.  256 threads; `sh` holds 8 words,
// each call its own.
__device__ __forceinline__ int lx_exponent(const uint32_t *most, int blocks, uint32_t *sh) {
    uint32_t top = 0;
    for (int i = threadIdx.x; i < blocks; i += 256) { const uint32_t u = most[i]; top = u > top ? u : top; }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) top = sh[i] > top ? sh[i] : top;
    const int e = 13 - ((int)(top >> 23) - 127);
    return top == 0 ? 0 : e > 60 ? 60 : e < -60 ? -60 : e;
}
__device__ __forceinline__ float lx_power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// Operands of the products.  The first `x_blocks` blocks: x of tokens [t0, t0 + tokens) -> [token][ld] 16-bit rows, zeros for
// tokens without a target.  The others: `rows` rows of the table -> [row][ld] with aligned ends; `flat`: rows without a gap on both
// sides (ld == D), eight elements at a time.  fp32 (most not null) scaled, as two parts; the first block leaves the inverse scales of
// x and of the table for the products.
template <typename T, typename H> struct LxPack {
    H *xh, *xl;
    const T *x;
    int x_blocks, t0, tokens, S;
    const void *targets; int id_u16, V;
    H *eh, *el;
    const T *table;
    int rows, flat;
    int D; size_t ld;
    const uint32_t *most; int most_x, most_table;      // blocks that looked at x, at the table
    float *scales;
};
template <typename T, typename H> __global__ void __launch_bounds__(256) lx_pack_kernel(const __grid_constant__ LxPack<T, H> p) {
    __shared__ float tile[32][33];
    __shared__ uint32_t sh[2][8];
    dep_sync();
    const int D = p.D, bx = blockIdx.x;
    const size_t ld = p.ld;
    const bool of_x = bx < p.x_blocks;
    float scale = 1.0f;
    if (p.most) {
        const auto exponent = [&](bool x, uint32_t *sh) { return lx_exponent(x ? p.most : p.most + p.most_x, x ? p.most_x : p.most_table, sh); };
        const int e = exponent(of_x, sh[0]);
        scale = lx_power(e);
        if (bx == 0) {
            const int other = exponent(!of_x, sh[1]);
            if (threadIdx.x == 0) { p.scales[of_x ? 0 : 1] = lx_power(-e); p.scales[of_x ? 1 : 0] = lx_power(-other); }
        }
    }
    if (of_x) {
        const int tiles = (p.tokens + 31) / 32, r0 = bx % tiles * 32, d0 = bx / tiles * 32;
        const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, t = r0 + tx;
        const bool live = t < p.tokens && lx_target(p.targets, p.id_u16, p.V, p.t0 + t) >= 0;
        const int b = (p.t0 + t) / p.S, s = (p.t0 + t) % p.S;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d = d0 + ty + 8 * i;
            tile[ty + 8 * i][tx] = live && d < D ? Elt<T>::to_f(p.x[((size_t)b * D + d) * p.S + s]) * scale : 0.0f;
        }
        __syncthreads();
        const int d = d0 + tx;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = r0 + ty + 8 * i;
            if (r < p.tokens && d < (int)ld) {
                const float v = tile[tx][ty + 8 * i];
                const H h = Elt<H>::from_f(v);
                p.xh[(size_t)r * ld + d] = h;
                if (p.xl) p.xl[(size_t)r * ld + d] = Elt<H>::from_f(v - Elt<H>::to_f(h));
            }
        }
        return;
    }
    const int first = bx - p.x_blocks, step = gridDim.x - p.x_blocks;
    if (sizeof(T) == 4 && p.flat) {
        const size_t n = (size_t)p.rows * D / 8;
        for (size_t i = (size_t)first * 256 + threadIdx.x; i < n; i += (size_t)step * 256) {
            float f[8], h[8];
            Elt<float>::unpack(reinterpret_cast<const uint4 *>(p.table)[2 * i], f);
            Elt<float>::unpack(reinterpret_cast<const uint4 *>(p.table)[2 * i + 1], f + 4);
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] *= scale;
            const uint4 q = Elt<H>::pack(f);
            Elt<H>::unpack(q, h);
            reinterpret_cast<uint4 *>(p.eh)[i] = q;
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] -= h[j];
            reinterpret_cast<uint4 *>(p.el)[i] = Elt<H>::pack(f);
        }
        return;
    }
    // eight columns of a row at a time: whole vectors out, single elements in (a row of the table starts anywhere).  With a block per
    // row the losses of 200 tokens over 32000 fp16 rows of 1001 took 92 us instead of 48.
    const uint32_t per = (uint32_t)(ld / 8);
    for (size_t i = (size_t)first * 256 + threadIdx.x; i < (size_t)p.rows * per; i += (size_t)step * 256) {
        const uint32_t r = (uint32_t)(i / per), d = (uint32_t)(i - (size_t)r * per) * 8;
        const T *src = p.table + (size_t)r * D + d;
        float f[8], h[8];
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = d + j < D ? Elt<T>::to_f(src[j]) * scale : 0.0f;
        const uint4 q = Elt<H>::pack(f);
        Elt<H>::unpack(q, h);
        reinterpret_cast<uint4 *>(p.eh)[i] = q;
        if (!p.el) continue;
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] -= h[j];
        reinterpret_cast<uint4 *>(p.el)[i] = Elt<H>::pack(f);
    }
}

// (max, sum) pairs of the vocabulary tiles -> lse and loss of TOK tokens per block: 1024 / TOK threads take turns at the tiles
// of a token and are joined in a fixed order.
template <int TOK>
__global__ void __launch_bounds__(1024) lx_join_kernel(float *__restrict__ lse2, float *__restrict__ loss_tok, const float2 *__restrict__ part, const float *__restrict__ hit,
                                                       const void *__restrict__ targets, int id_u16, int V, int tiles, int tokens, size_t ldt, ane_cuda_status *status) {
    constexpr int SL = 1024 / TOK;
    __shared__ float2 sh[SL][TOK + 1];
    dep_sync();
    const int cl = threadIdx.x % TOK, sl = threadIdx.x / TOK;
    const int t = blockIdx.x * TOK + cl;
    float m = -INFINITY, s = 0.0f;
    if (t < tokens)
        for (int i = sl; i < tiles; i += 4 * SL) {
            float2 p[4];
            float mn = m;
#pragma unroll
            for (int u = 0; u < 4; u++) p[u] = i + SL * u < tiles ? part[(size_t)(i + SL * u) * ldt + t] : make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int u = 0; u < 4; u++) mn = fmaxf(mn, p[u].x);
            s *= lx_exp2(m - mn);
#pragma unroll
            for (int u = 0; u < 4; u++) if (p[u].y != 0.0f) s += p[u].y * lx_exp2(p[u].x - mn);
            m = mn;
        }
    sh[sl][cl] = make_float2(m, s);
    __syncthreads();
    // warp w joins the slices of token w: SL / 32 per lane, then the lanes by a fixed tree
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (w >= TOK) return;
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < SL / 32; i++) top = fmaxf(top, sh[i * 32 + lane][w].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
    for (int i = 0; i < SL / 32; i++) {                                       // slices without a tile hold (-inf, 0)
        const float2 p = sh[i * 32 + lane][w];
        if (p.y != 0.0f) sum += p.y * lx_exp2(p.x - top);
    }
    sum = warp_sum(sum);
    const int token = blockIdx.x * TOK + w;
    if (lane != 0 || token >= tokens) return;
    const float l2 = top + log2f(sum);
    lse2[token] = l2;
    const int id = id_u16 ? (int)static_cast<const uint16_t *>(targets)[token] : static_cast<const int32_t *>(targets)[token];
    float loss = 0.0f;
    if (id >= 0 && id < V) {
        loss = -logf(exp2f(fmaf(hit[token], LX_LOG2E, -l2)) + 1e-10f);
        if (!isfinite(loss)) atomicAdd(&status->nonfinite, 1);
    } else if (id >= V) {
        atomicAdd(&status->oor_ids, 1);
    }
    loss_tok[token] = loss;
}

// loss_seq[b] = (sum_t loss_tok[b][t]) / S, fixed summation tree of 256 threads.
__device__ __forceinline__ void lx_sequence_loss(float *loss_seq, const float *loss_tok, int S, int b, float *sh) {
    const float *p = loss_tok + (size_t)b * S;
    float acc = 0.0f;
    for (int t = threadIdx.x; t < S; t += 256) acc += p[t];
    acc = warp_sum(acc);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        float s = 0.0f;
        for (int i = 0; i < 8; i++) s += sh[i];
        loss_seq[b] = s / (float)S;
    }
}

// dx[b][d][s] = alpha * sum over the shares of K, in order.  A token without a target has zeros, whatever the table holds.
template <typename T>
__global__ void __launch_bounds__(256) lx_finish_dx_kernel(T *__restrict__ dx, const float *__restrict__ sums, const void *__restrict__ targets, int id_u16, int V, int splits,
                                                           int t0, int tokens, int D, int S, size_t ldt, float alpha, float *loss_seq, const float *loss_tok, int seqs) {
    __shared__ float sh[8];
    dep_sync();
    const int by = loss_seq ? gridDim.y - 1 : gridDim.y;             // the last row of blocks: losses of the sequences
    if (blockIdx.y == by) {
        for (int b = blockIdx.x; b < seqs; b += gridDim.x) lx_sequence_loss(loss_seq, loss_tok, S, b, sh);
        return;
    }
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= tokens) return;
    const bool live = lx_target(targets, id_u16, V, t0 + t) >= 0;
    const int b = (t0 + t) / S, s = (t0 + t) % S;
    for (int d = blockIdx.y; d < D; d += by) {
        float v = 0.0f;
        for (int k = 0; k < splits; k++) v += sums[((size_t)k * D + d) * ldt + t];
        dx[((size_t)b * D + d) * S + s] = Elt<T>::from_f(live ? v * alpha : 0.0f);
    }
}

// ------------------------------------------------------------------ one to four tokens
// For so few tokens the operator is the table read once (and once more, with its gradient read and written, for the gradients):
// plain fp32 arithmetic on the elements as they are, bound by HBM.  A tile of the tensor cores would be 252 rows of nothing,
// and fp32 tables would have to be packed first.  The few logits of a row are kept for the second pass, [V][T].
// Against the tensor cores, 151936 rows x 1024 channels, losses / with gradients: fp32 1 token 123 / 434 against 453 / 1044 us,
// 4 tokens 187 / 592 against 464 / 1094 (9200 x 768: 18 / 46 against 36 / 87); bf16 1 token 60 / 440 against 76 / 498, 2 tokens
// 145 / 517 against 72 / 493.  Hence four tokens in fp32 and one in 16 bits.
constexpr int LF_TOKENS = 4;
constexpr size_t LF_SMEM = 96 << 10;                     // of x as fp32

template <typename T> __device__ __forceinline__ void lf_x_to_shared(float *xs, const T *x, const void *targets, int id_u16, int V, int tokens, int D, int S) {
    for (int i = threadIdx.x; i < tokens * D; i += blockDim.x) {
        const int t = i / D, d = i - t * D;
        xs[i] = lx_target(targets, id_u16, V, t) >= 0 ? Elt<T>::to_f(x[((size_t)(t / S) * D + d) * S + t % S]) : 0.0f;
    }
}

// A warp takes two rows at a time; per block a (max, sum) pair per token over its rows.
template <typename T, int VEC, int TOK>
__global__ void __launch_bounds__(256) lf_logits_kernel(float *__restrict__ logits, float2 *__restrict__ part, float *__restrict__ hit, const T *__restrict__ x,
                                                        const T *__restrict__ table, const void *__restrict__ targets, int id_u16, int V, int D, int S, size_t ldt) {
    extern __shared__ float xs[];
    __shared__ float2 sh[8][TOK];
    dep_sync();
    lf_x_to_shared(xs, x, targets, id_u16, V, TOK, D, S);
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int step = 2 * 8 * gridDim.x;
    float m[TOK], s[TOK];
#pragma unroll
    for (int t = 0; t < TOK; t++) { m[t] = -INFINITY; s[t] = 0.0f; }
    for (int v = 2 * (blockIdx.x * 8 + warp); v < V; v += step) {
        const T *row = table + (size_t)v * D, *next = v + 1 < V ? row + D : row;
        float a[2][TOK];
#pragma unroll
        for (int t = 0; t < TOK; t++) a[0][t] = a[1][t] = 0.0f;
#pragma unroll 2
        for (int d = lane * VEC; d < D; d += 32 * VEC) {
            Raw<T, VEC> r[2];
            r[0].load_stream(row + d);
            r[1].load_stream(next + d);
            float e[2][VEC];
            r[0].unpack(e[0]);
            r[1].unpack(e[1]);
#pragma unroll
            for (int t = 0; t < TOK; t++)
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const float q = xs[t * D + d + j];
                    a[0][t] = fmaf(e[0][j], q, a[0][t]);
                    a[1][t] = fmaf(e[1][j], q, a[1][t]);
                }
        }
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int t = 0; t < TOK; t++) a[r][t] = warp_sum(a[r][t]);
#pragma unroll
        for (int r = 0; r < 2; r++)
            if (v + r < V) {
#pragma unroll
                for (int t = 0; t < TOK; t++) {
                    const float l2 = a[r][t] * LX_LOG2E, mn = fmaxf(m[t], l2);
                    s[t] = s[t] * lx_exp2(m[t] - mn) + lx_exp2(l2 - mn);
                    m[t] = mn;
                    if (lane == t) {
                        if (logits) logits[(size_t)(v + r) * TOK + t] = a[r][t];
                        if (lx_target(targets, id_u16, V, t) == v + r) hit[t] = a[r][t];
                    }
                }
            }
    }
    if (lane == 0)
#pragma unroll
        for (int t = 0; t < TOK; t++) sh[warp][t] = make_float2(m[t], s[t]);
    __syncthreads();
    if (threadIdx.x < TOK) {
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; w++) top = fmaxf(top, sh[w][threadIdx.x].x);
#pragma unroll
        for (int w = 0; w < 8; w++) if (sh[w][threadIdx.x].y != 0.0f) sum += sh[w][threadIdx.x].y * lx_exp2(sh[w][threadIdx.x].x - top);
        part[(size_t)blockIdx.x * ldt + threadIdx.x] = make_float2(top, sum);
    }
}

// Rows [v0, v1) of a block, columns of blockIdx.y: d_table += dl x^T, and the block's share of dx, [chunk][TOK][D].
constexpr int LF_ROWS = 64;                              // dl of this many rows at a time
template <typename T, int VEC, int TOK>
__global__ void __launch_bounds__(256) lf_grads_kernel(float *__restrict__ dx_part, float *__restrict__ d_table, const float *__restrict__ logits, const float *__restrict__ lse2,
                                                       const T *__restrict__ x, const T *__restrict__ table, const void *__restrict__ targets, int id_u16, int V, int D, int S,
                                                       int chunk, float alpha) {
    __shared__ float dl[LF_ROWS][TOK];
    dep_sync();
    const int d = (blockIdx.y * 256 + threadIdx.x) * VEC;
    const bool live = d < D;
    float q[TOK][VEC], acc[TOK][VEC];
#pragma unroll
    for (int t = 0; t < TOK; t++)
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            acc[t][j] = 0.0f;
            q[t][j] = live && lx_target(targets, id_u16, V, t) >= 0 ? Elt<T>::to_f(x[((size_t)(t / S) * D + d + j) * S + t % S]) * alpha : 0.0f;
        }
    const int v0 = blockIdx.x * chunk, v1 = v0 + chunk < V ? v0 + chunk : V;
    for (int r0 = v0; r0 < v1; r0 += LF_ROWS) {
        const int rows = v1 - r0 < LF_ROWS ? v1 - r0 : LF_ROWS;
        __syncthreads();
        for (int i = threadIdx.x; i < rows * TOK; i += 256) {
            const int t = i % TOK, v = r0 + i / TOK, id = lx_target(targets, id_u16, V, t);
            const float p = lx_exp2(fmaf(logits[(size_t)r0 * TOK + i], LX_LOG2E, -lse2[t]));
            dl[i / TOK][t] = id < 0 ? 0.0f : id == v ? p - 1.0f : p;
        }
        __syncthreads();
        if (live) {
#pragma unroll 4
            for (int r = 0; r < rows; r++) {
                float k[TOK];
#pragma unroll
                for (int t = 0; t < TOK; t++) k[t] = dl[r][t];
                const size_t at = (size_t)(r0 + r) * D + d;
                if (dx_part) {
                    Raw<T, VEC> e;
                    float f[VEC];
                    e.load_stream(table + at);
                    e.unpack(f);
#pragma unroll
                    for (int t = 0; t < TOK; t++)
#pragma unroll
                        for (int j = 0; j < VEC; j++) acc[t][j] = fmaf(k[t], f[j], acc[t][j]);
                }
                if (d_table) {
                    if constexpr (VEC % 4 == 0) {
#pragma unroll
                        for (int h = 0; h < VEC; h += 4) {
                            float4 g = __ldcs(reinterpret_cast<const float4 *>(d_table + at + h));
#pragma unroll
                            for (int t = 0; t < TOK; t++) {
                                g.x = fmaf(k[t], q[t][h], g.x); g.y = fmaf(k[t], q[t][h + 1], g.y);
                                g.z = fmaf(k[t], q[t][h + 2], g.z); g.w = fmaf(k[t], q[t][h + 3], g.w);
                            }
                            __stcs(reinterpret_cast<float4 *>(d_table + at + h), g);
                        }
                    } else {
                        float g = d_table[at];
#pragma unroll
                        for (int t = 0; t < TOK; t++) g = fmaf(k[t], q[t][0], g);
                        d_table[at] = g;
                    }
                }
            }
        }
    }
    if (dx_part && live)
#pragma unroll
        for (int t = 0; t < TOK; t++)
#pragma unroll
            for (int j = 0; j < VEC; j++) dx_part[((size_t)blockIdx.x * TOK + t) * D + d + j] = acc[t][j];
}

// dx[b][d][s] = alpha * sum over the chunks, in order: eight slices of them per column.
template <typename T>
__global__ void __launch_bounds__(256) lf_finish_dx_kernel(T *__restrict__ dx, const float *__restrict__ part, const void *__restrict__ targets, int id_u16, int V, int chunks,
                                                           int tokens, int D, int S, float alpha) {
    __shared__ float sh[8][33];
    dep_sync();
    const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5, d = blockIdx.x * 32 + cl, t = blockIdx.y;
    float a = 0.0f;
    if (d < D)
#pragma unroll 4
        for (int i = sl; i < chunks; i += 8) a += part[((size_t)i * tokens + t) * D + d];
    sh[sl][cl] = a;
    __syncthreads();
    if (sl != 0 || d >= D) return;
    a = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) a += sh[i][cl];
    dx[((size_t)(t / S) * D + d) * S + t % S] = Elt<T>::from_f(lx_target(targets, id_u16, V, t) >= 0 ? a * alpha : 0.0f);
}

__global__ void __launch_bounds__(256) lx_loss_kernel(float *__restrict__ loss_seq, const float *__restrict__ loss_tok, int S) {
    __shared__ float sh[8];
    dep_sync();
    lx_sequence_loss(loss_seq, loss_tok, S, blockIdx.x, sh);
}

static inline int lx_div(long long a, long long b) { return (int)((a + b - 1) / b); }
static inline int lx_pairs() { return ctx().sm_count / 2; }

// Every kernel of the chain is a programmatic dependent launch: its blocks may be placed and set up their barriers and
// accumulators while the kernel before drains, and stop in dep_sync() until that one has completed.  A call has 4 to 8 short
// launches where the problem is small: 98 -> 81 us for one fp32 sequence over 9200 rows.
template <typename... KArgs, typename... Args>
static inline void lx_call(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = tuning("linear_xent_dep", 1) != 0;
    cfg.attrs = attr; cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);          // the error, if any, is picked up by ANE_LAUNCH_OK
}

template <int EPI, int MODE, bool HALF> static int lx_start_kernel(cudaStream_t st, const LxMaps &maps, const LxArgs &a) {
    static bool ready = false;
    if (!ready) {
        ANE_CUDA_TRY(cudaFuncSetAttribute(lx_gemm_kernel<EPI, MODE, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lx_smem(EPI)));
        ready = true;
    }
    const long long tiles = (long long)a.m_tiles * a.n_tiles * a.splits;
    const int pairs = tiles < lx_pairs() ? (int)tiles : lx_pairs();
    lx_call(lx_gemm_kernel<EPI, MODE, HALF>, dim3(2 * pairs), dim3(LX_THREADS), lx_smem(EPI), st, maps, a);
    ANE_LAUNCH_OK(1);
    return ANE_CUDA_OK;
}
// The type of the operands is the instruction's business; only dlogits writes 16-bit values itself.
template <int EPI, int MODE> static int lx_start(cudaStream_t st, const LxMaps &maps, const LxArgs &a) {
    constexpr bool WRITES = EPI == LX_DLOGITS, FP16_ONLY = WRITES && (MODE == LX_SPLIT || MODE == LX_NARROW);
    if (FP16_ONLY || (WRITES && a.half_type)) return lx_start_kernel<EPI, MODE, WRITES>(st, maps, a);
    return lx_start_kernel<EPI, MODE, FP16_ONLY>(st, maps, a);
}

// Time of a product of `tiles` accumulators of 256 x 256 (m x n of them), in K blocks of one accumulator: waves over the SM
// pairs.  A wide tile takes the time of 1.55 plain ones (clocks per K block, 512 for a plain accumulator's instructions: about
// 850 plain, 1300 wide).  Losses of 16 tokens over 151936 rows: 84 us wide, 101 plain; all of 8192 tokens: 10.3 against 10.4 ms.
// Split inputs take about two plain ones: four boxes for three products.
constexpr double LX_WIDE_COST = 1.55, LX_SPLIT_COST = 2.0;
static double lx_cost(int m, int n, int splits, bool split, bool *wide) {
    const double plain = lx_div((long long)m * n * splits, lx_pairs()) * (split ? LX_SPLIT_COST : 1.0), w = lx_div((long long)m * lx_div(n, 2) * splits, lx_pairs()) * LX_WIDE_COST;
    const bool is = !split && tuning("linear_xent_wide", w < plain) != 0;
    if (wide) *wide = is;
    return is ? w : plain;
}
// Tiles of 256 x 128 for products of split inputs with m x (n columns) outputs, where 256 x 256 ones leave pairs idle.  A narrow
// tile takes about 0.6 of the time.  Losses, 768 channels, 9200 rows, plain / narrow: 256 tokens 37.9 / 32.4 us (36 tiles for 74
// pairs), 512 40.6 / 39.9, 768 53.2 / 48.5, 1024 55.9 / 55.9, 2048 80.5 / 88.4.  d_table of 256 tokens (108 tiles): 21.9 / 17.7.
static bool lx_narrow(int m, int n) {
    return tuning("linear_xent_narrow", lx_div((long long)m * lx_div(n, LX_BN / 2), lx_pairs()) * 0.6 < lx_div((long long)m * lx_div(n, LX_BN), lx_pairs())) != 0;
}
// n_tiles of `a` counts accumulators; operands of one part may run wide.
template <int EPI> static int lx_launch(cudaStream_t st, const LxMaps &maps, LxArgs a, bool split, bool narrow = false) {
    if (narrow) return lx_start<EPI, LX_NARROW>(st, maps, a);
    if (split) return lx_start<EPI, LX_SPLIT>(st, maps, a);
    bool wide = false;
    lx_cost(a.m_tiles, a.n_tiles, a.splits, false, &wide);
    if (!wide) return lx_start<EPI, LX_PLAIN>(st, maps, a);
    a.n_tiles = lx_div(a.n_tiles, 2);
    return lx_start<EPI, LX_WIDE>(st, maps, a);
}

// K blocks after which an fp32 sum leaves the accumulator, with `products` steps for every 16 of K.
static int lx_span(int products) { return LX_STEPS * 16 / (products * LX_BK); }

// Instruction descriptor: fp32 accumulator, 16-bit operands of one type, their layouts, the tile.
static uint32_t lx_idesc(bool half_type, bool a_mn, bool b_mn, int acc_n = LX_BN) {
    const uint32_t f = half_type ? 0u : 1u;
    return 1u << 4 | f << 7 | f << 10 | (a_mn ? 1u : 0u) << 15 | (b_mn ? 1u : 0u) << 16 | (uint32_t)(acc_n >> 3) << 17 | (uint32_t)(LX_BM >> 4) << 24;
}

struct LxCall {
    cudaStream_t st;
    ane_dtype dtype;
    int id_u16, B, D, V, S;
    float *loss_seq, *loss_tok;
    void *dx;
    float *d_table;
    const void *x, *table, *targets;
    float grad_scale;
};

// Sizes of one call: tokens of a round, vocabulary tiles of a piece, shares of K for dx.
struct LxPlan { int chunk, piece_tiles, splits; bool narrow_dx; };

// A round has at most 8192 tokens.  A piece has as many vocabulary tiles as fill whole waves of the SM pairs best, counted in
// waves of K blocks over all pieces and products (with four K blocks for the start of a launch), while the two parts of dl
// stay within 768 MiB (128, 192, 384, 768 MiB: 12.0, 11.4, 10.8, 10.3 ms for 8192 tokens x 151936 rows x 1024
// channels under the power cap: a launch of dx has one tile per pair and nothing to hide its end behind).  dx has few tiles
// and a long K: where its tiles leave pairs idle, K is cut into shares.
static LxPlan lx_plan(int T_all, int D, int V, bool split, bool dx, bool d_table, bool two_parts) {
    LxPlan p;
    const int rounds = lx_div(T_all, 8192), pairs = lx_pairs();
    p.chunk = (int)round_up((size_t)lx_div(T_all, rounds), LX_BM);
    if (p.chunk > T_all) p.chunk = T_all;
    const int mt = lx_div(p.chunk, LX_BM), wide_dt = lx_div(D, LX_BN), vt = lx_div(V, LX_BN);
    p.narrow_dx = split && pairs / (mt * wide_dt) > 1;      // half as many shares to store and to add up: 19 us instead of 24 for 256 tokens, 768 channels
    const int dt = p.narrow_dx ? lx_div(D, LX_BN / 2) : wide_dt;
    const int kd = lx_div(D, LX_BK), kt = lx_div(p.chunk, LX_BK);
    long long most = (768ll << 20) / ((long long)p.chunk * LX_BN * (two_parts ? 4 : 2));
    if (most < 1) most = 1;
    if (most > vt) most = vt;
    double best = 1e300;
    p.piece_tiles = 1; p.splits = 1;
    for (int n = (int)most; n >= 1 && n >= (int)most / 4; n -= 1 + (int)most / 1024) {
        const int pieces = lx_div(vt, n);
        int splits = 1;
        if (dx) {
            splits = pairs / (mt * dt);
            if (splits > n) splits = n;                     // four K blocks per share at least
            if (splits < 1) splits = 1;
        }
        double cost = 0.0;
        for (int i = 0; i < 2; i++) {                       // the whole pieces and the last
            const int tiles = i ? vt - (pieces - 1) * n : n, times = i ? 1 : pieces - 1;
            double c = lx_cost(mt, tiles, 1, split, nullptr) * kd + 4;
            if (dx) c += lx_cost(mt, dt, splits, split, nullptr) * (p.narrow_dx ? 0.5 : 1.0) * lx_div((long long)tiles * 4, splits) + 4;
            if (d_table) c += (double)lx_div((long long)wide_dt * tiles, pairs) * (split ? LX_SPLIT_COST : LX_WIDE_COST) * kt + 4;
            cost += c * times;
        }
        if (cost < best * 0.999) { best = cost; p.piece_tiles = n; p.splits = splits; }
    }
    return p;
}

template <typename T, int VEC, int TOK> static int lf_run(const LxCall &c) {
    const bool grad = c.dx || c.d_table;
    const int D = c.D, V = c.V;
    const int blocks = lx_div(V, 16) < 4 * ctx().sm_count ? lx_div(V, 16) : 4 * ctx().sm_count;
    const int cols = lx_div(D, 256 * VEC);
    int chunks = lx_div(4 * ctx().sm_count, cols);
    if (chunks > lx_div(V, 8)) chunks = lx_div(V, 8);
    const int chunk = lx_div(V, chunks);
    chunks = lx_div(V, chunk);
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += round_up(bytes, 1024); return at; };
    const size_t o_tok = take(LF_TOKENS * 4), o_lse = take(LF_TOKENS * 4), o_hit = take(LF_TOKENS * 4), o_part = take((size_t)blocks * LF_TOKENS * 8);
    const size_t o_logits = take(grad ? (size_t)V * TOK * 4 : 0), o_dx = take(c.dx ? (size_t)chunks * TOK * D * 4 : 0);
    char *ws = static_cast<char *>(workspace(off));
    if (!ws) return fail(ANE_CUDA_ERR_NOMEM, "ane_cuda_linear_cross_entropy_dev: no scratch (%zu bytes)", off);
    float *loss_tok = c.loss_tok ? c.loss_tok : reinterpret_cast<float *>(ws + o_tok), *lse2 = reinterpret_cast<float *>(ws + o_lse), *hit = reinterpret_cast<float *>(ws + o_hit);
    float *logits = grad ? reinterpret_cast<float *>(ws + o_logits) : nullptr, *dxs = c.dx ? reinterpret_cast<float *>(ws + o_dx) : nullptr;
    float2 *part = reinterpret_cast<float2 *>(ws + o_part);
    const T *x = static_cast<const T *>(c.x), *table = static_cast<const T *>(c.table);
    static bool ready = false;
    if (!ready) {
        ANE_CUDA_TRY(cudaFuncSetAttribute(lf_logits_kernel<T, VEC, TOK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)LF_SMEM));
        ready = true;
    }
    lx_call(lf_logits_kernel<T, VEC, TOK>, dim3(blocks), dim3(256), (size_t)TOK * D * 4, c.st, logits, part, hit, x, table, c.targets, c.id_u16, V, D, c.S, (size_t)LF_TOKENS);
    lx_call(lx_join_kernel<4>, dim3(1), dim3(1024), 0, c.st, lse2, loss_tok, part, hit, c.targets, c.id_u16, V, blocks, TOK, (size_t)LF_TOKENS, ctx().status);
    ANE_LAUNCH_OK(2);
    const float alpha = c.grad_scale / (float)c.S;
    if (grad) {
        lx_call(lf_grads_kernel<T, VEC, TOK>, dim3(chunks, cols), dim3(256), 0, c.st, dxs, c.d_table, logits, lse2, x, table, c.targets, c.id_u16, V, D, c.S, chunk, alpha);
        ANE_LAUNCH_OK(1);
    }
    if (c.dx) {
        lx_call(lf_finish_dx_kernel<T>, dim3(lx_div(D, 32), TOK), dim3(256), 0, c.st, static_cast<T *>(c.dx), dxs, c.targets, c.id_u16, V, chunks, TOK, D, c.S, alpha);
        ANE_LAUNCH_OK(1);
    }
    lx_call(lx_loss_kernel, dim3(c.B), dim3(256), 0, c.st, c.loss_seq, loss_tok, c.S);
    ANE_LAUNCH_OK(1);
    return ANE_CUDA_OK;
}

template <typename T, typename H> static int lx_run(const LxCall &c) {
    if (c.B * c.S <= (sizeof(T) == 4 ? LF_TOKENS : 1) && (size_t)c.B * c.S * c.D * 4 <= LF_SMEM && c.V < (1 << 29) && tuning("linear_xent_few", 1)) {
        const bool vec = c.D % Elt<T>::VEC == 0 && aligned16(c.table) && aligned16(c.d_table);
        switch (c.B * c.S) {
            case 1: return vec ? lf_run<T, Elt<T>::VEC, 1>(c) : lf_run<T, 1, 1>(c);
            case 2: return vec ? lf_run<T, Elt<T>::VEC, 2>(c) : lf_run<T, 1, 2>(c);
            case 3: return vec ? lf_run<T, Elt<T>::VEC, 3>(c) : lf_run<T, 1, 3>(c);
            default: return vec ? lf_run<T, Elt<T>::VEC, 4>(c) : lf_run<T, 1, 4>(c);
        }
    }
    const bool split = sizeof(T) == 4;                       // fp32 inputs as two parts
    const ane_dtype part = c.dtype == ANE_BF16 ? ANE_BF16 : ANE_F16;
    const int half_type = part == ANE_F16;
    const bool grad = c.dx || c.d_table;
    const int T_all = c.B * c.S, D = c.D, V = c.V;
    const size_t ldd = round_up((size_t)D, 8);
    const bool pack_table = split || D % 8 || !aligned16(c.table);
    const bool need_lo = c.d_table || split;
    const LxPlan plan = lx_plan(T_all, D, V, split, c.dx != nullptr, c.d_table != nullptr, need_lo);
    const int chunk = plan.chunk, vp = plan.piece_tiles * LX_BN < V ? plan.piece_tiles * LX_BN : V, splits = plan.splits;
    const size_t ldt = round_up((size_t)chunk, 32), ldl = (size_t)plan.piece_tiles * LX_BN;
    // A table that has to be packed is packed once where that takes up to 256 MiB, else piece by piece.
    const size_t row_bytes = ldd * 2 * (split ? 2 : 1);
    const int vk = !pack_table ? 0 : (size_t)V * row_bytes <= ((size_t)256 << 20) ? V : vp;
    // statistics: the whole table in one launch, or piece by piece where it is packed so; a (max, sum) pair per epilogue warp's columns
    const int fstep = pack_table && vk < V ? vp : V;
    const bool narrow_stats = split && lx_narrow(lx_div(chunk, LX_BM), fstep);
    const int stat_cols = (narrow_stats ? lx_acc_n(LX_NARROW) : LX_BN) / 2, parts_n = lx_div(V, stat_cols);

    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += round_up(bytes, 1024); return at; };
    const size_t o_most = take(split ? LX_LARGEST_BLOCKS * 4 : 0), o_scales = take(8);
    const size_t o_tok = take(c.loss_tok ? 0 : (size_t)T_all * 4), o_lse = take(ldt * 4), o_hit = take(ldt * 4), o_part = take((size_t)parts_n * ldt * 8);
    const size_t o_xh = take((size_t)chunk * ldd * 2), o_xl = take(split ? (size_t)chunk * ldd * 2 : 0);
    const size_t o_eh = take((size_t)vk * ldd * 2), o_el = take(split ? (size_t)vk * ldd * 2 : 0);
    const size_t o_lh = take(grad ? (size_t)chunk * ldl * 2 : 0), o_ll = take(grad && need_lo ? (size_t)chunk * ldl * 2 : 0);
    const size_t o_dx = take(c.dx ? (size_t)splits * D * ldt * 4 : 0);
    char *ws = static_cast<char *>(workspace(off));
    if (!ws) return fail(ANE_CUDA_ERR_NOMEM, "ane_cuda_linear_cross_entropy_dev: no scratch (%zu bytes)", off);
    uint32_t *most = split ? reinterpret_cast<uint32_t *>(ws + o_most) : nullptr;
    float *scales = split ? reinterpret_cast<float *>(ws + o_scales) : nullptr;
    float *loss_tok = c.loss_tok ? c.loss_tok : reinterpret_cast<float *>(ws + o_tok);
    float *lse2 = reinterpret_cast<float *>(ws + o_lse), *hit = reinterpret_cast<float *>(ws + o_hit), *dxs = reinterpret_cast<float *>(ws + o_dx);
    float2 *parts = reinterpret_cast<float2 *>(ws + o_part);
    H *xh = reinterpret_cast<H *>(ws + o_xh), *xl = split ? reinterpret_cast<H *>(ws + o_xl) : nullptr;
    H *eh = reinterpret_cast<H *>(ws + o_eh), *el = split ? reinterpret_cast<H *>(ws + o_el) : nullptr;
    void *lh = ws + o_lh, *ll = need_lo ? ws + o_ll : nullptr;
    const size_t idb = c.id_u16 ? 2 : 4;
    ane_cuda_status *status = ctx().status;

    int most_x = 0, most_table = 0;
    if (split) {                                             // as many blocks as are resident at once, at least 4096 elements each
        const size_t nx = (size_t)T_all * D, ne = (size_t)V * D;
        const auto share = [](size_t n, int most) { return n / 4096 < 1 ? 1 : n / 4096 < (size_t)most ? (int)(n / 4096) : most; };
        most_x = share(nx, nx < ne ? LX_LARGEST_BLOCKS / 2 : LX_LARGEST_BLOCKS - share(ne, LX_LARGEST_BLOCKS / 2));
        most_table = share(ne, LX_LARGEST_BLOCKS - most_x);
        lx_call(lx_largest_kernel, dim3(most_x + most_table), dim3(256), 0, c.st, most, most_x, static_cast<const float *>(c.x), nx, static_cast<const float *>(c.table), ne, c.targets,
                c.id_u16, V, D, c.S);
        ANE_LAUNCH_OK(1);
    }
    // Packs tokens [t0, t0 + n_tok) of x and rows [v0, v0 + nv) of the table; either may be none.
    auto pack = [&](int t0, int n_tok, int v0, int nv) -> int {
        const T *from = static_cast<const T *>(c.table) + (size_t)v0 * D;
        const int flat = split && D % 8 == 0 && aligned16(from), x_blocks = lx_div(n_tok, 32) * lx_div(D, 32);
        const size_t want = ((size_t)nv * (ldd / 8) + 255) / 256;          // (ldd is D where it is flat)
        const LxPack<T, H> p = {xh, xl, static_cast<const T *>(c.x), x_blocks, t0, n_tok, c.S, c.targets, c.id_u16, V, eh, el, from, nv, flat, D, ldd, most, most_x, most_table, scales};
        lx_call(lx_pack_kernel<T, H>, dim3((unsigned)(x_blocks + (want < 4096 ? want : 4096))), dim3(256), 0, c.st, p);
        ANE_LAUNCH_OK(1);
        return ANE_CUDA_OK;
    };
    // Rows [v0, v0 + nv) of the table as 16-bit rows with `ld` elements between them; packs them where that is done piece by piece.
    const H *rows_hi = nullptr, *rows_lo = nullptr;
    size_t ld = ldd;
    auto table_rows = [&](int v0, int nv) -> int {
        if (!pack_table) {
            rows_hi = reinterpret_cast<const H *>(c.table) + (size_t)v0 * D;
            ld = (size_t)D;
            return ANE_CUDA_OK;
        }
        if (vk < V) if (int rc = pack(0, 0, v0, nv)) return rc;
        rows_hi = vk < V ? eh : eh + (size_t)v0 * ldd;
        rows_lo = !split ? nullptr : vk < V ? el : el + (size_t)v0 * ldd;
        return ANE_CUDA_OK;
    };
    // Operands; low parts that are null are not in use.
    auto maps_for = [&](LxMaps &m, const void *ah, const void *al, const void *bh, const void *bl, size_t arows, size_t acols, size_t lda, int abox, size_t brows, size_t bcols,
                        size_t ldb, int bbox) -> int {
        if (int rc = make_matrix_map(&m.a[0], part, ah, arows, acols, lda, abox)) return rc;
        if (int rc = make_matrix_map(&m.b[0], part, bh, brows, bcols, ldb, bbox)) return rc;
        if (al) if (int rc = make_matrix_map(&m.a[1], part, al, arows, acols, lda, abox)) return rc;
        if (bl) if (int rc = make_matrix_map(&m.b[1], part, bl, brows, bcols, ldb, bbox)) return rc;
        return ANE_CUDA_OK;
    };

    bool with_dx = false;                                    // the sequences' losses are made beside the last dx
    for (int t0 = 0; t0 < T_all; t0 += chunk) {
        const int n_tok = T_all - t0 < chunk ? T_all - t0 : chunk;
        const void *tg = static_cast<const char *>(c.targets) + (size_t)t0 * idb;
        // the whole table with the first tokens, where it stays packed
        if (int rc = pack(t0, n_tok, 0, t0 == 0 && pack_table && vk == V ? V : 0)) return rc;

        LxArgs a = {};
        a.kblocks = lx_div(D, LX_BK); a.splits = 1; a.span = split ? 3 * lx_span(3) : 1 << 20;
        a.m_tiles = lx_div(n_tok, LX_BM); a.m = n_tok;
        a.targets = tg; a.id_u16 = c.id_u16; a.V = V;
        a.scales = scales;
        a.part = parts; a.hit = hit; a.lse2 = lse2; a.ldt = ldt;
        a.half_type = half_type; a.dscale = half_type ? LX_HALF_SCALE : 1.0f;
        a.status = status;
        const auto forward_args = [&](int v0, int nv, bool narrow) {
            const int acc_n = lx_acc_n(narrow ? LX_NARROW : LX_PLAIN);
            a.n_tiles = lx_div(nv, acc_n); a.n = nv; a.v0 = v0;
            a.idesc = lx_idesc(half_type, false, false, acc_n);
        };
        for (int v0 = 0; v0 < V; v0 += fstep) {
            const int nv = V - v0 < fstep ? V - v0 : fstep;
            LxMaps m;
            if (int rc = table_rows(v0, nv)) return rc;
            if (int rc = maps_for(m, xh, xl, rows_hi, rows_lo, n_tok, D, ldd, LX_CTA_M, nv, D, ld, stat_cols)) return rc;
            forward_args(v0, nv, narrow_stats);
            a.tile0 = v0 / stat_cols;
            if (int rc = lx_launch<LX_STATS>(c.st, m, a, split, narrow_stats)) return rc;
        }
        // few tokens: more threads for each
        if (n_tok <= 1024) lx_call(lx_join_kernel<4>, dim3(lx_div(n_tok, 4)), dim3(1024), 0, c.st, lse2, loss_tok + t0, parts, hit, tg, c.id_u16, V, parts_n, n_tok, ldt, status);
        else lx_call(lx_join_kernel<32>, dim3(lx_div(n_tok, 32)), dim3(1024), 0, c.st, lse2, loss_tok + t0, parts, hit, tg, c.id_u16, V, parts_n, n_tok, ldt, status);
        ANE_LAUNCH_OK(1);
        if (!grad) continue;

        const float alpha = c.grad_scale / (float)c.S / a.dscale;
        for (int v0 = 0; v0 < V; v0 += vp) {
            const int nv = V - v0 < vp ? V - v0 : vp;
            const bool narrow = split && lx_narrow(a.m_tiles, nv);
            LxMaps m;
            if (int rc = table_rows(v0, nv)) return rc;
            if (int rc = maps_for(m, xh, xl, rows_hi, rows_lo, n_tok, D, ldd, LX_CTA_M, nv, D, ld, narrow ? LX_BN / 4 : LX_BN / 2)) return rc;
            forward_args(v0, nv, narrow);
            if (int rc = make_matrix_map(&m.hi, part, lh, n_tok, nv, ldl, 32, 32)) return rc;
            if (need_lo) if (int rc = make_matrix_map(&m.lo, part, ll, n_tok, nv, ldl, 32, 32)) return rc;
            a.two_parts = need_lo;
            if (int rc = lx_launch<LX_DLOGITS>(c.st, m, a, split, narrow)) return rc;
            if (c.dx) {
                LxArgs g = a;
                if (int rc = maps_for(m, lh, split ? ll : nullptr, rows_hi, rows_lo, n_tok, nv, ldl, LX_CTA_M, nv, D, ld, LX_BK)) return rc;
                g.kblocks = lx_div(nv, LX_BK); g.splits = splits;
                if (split) g.span = lx_span(3);              // a 16-bit dx does not show what the accumulator cuts off
                const int acc_n = lx_acc_n(plan.narrow_dx ? LX_NARROW : LX_PLAIN);
                g.n_tiles = lx_div(D, acc_n); g.n = D;
                g.idesc = lx_idesc(half_type, false, true, acc_n);
                g.out = dxs; g.first = v0 == 0;
                if (int rc = lx_launch<LX_DX>(c.st, m, g, split, plan.narrow_dx)) return rc;
            }
            if (c.d_table) {
                LxArgs g = a;
                // 16-bit inputs: both parts of dl beside one box of x, two steps for every 16 of K
                if (int rc = maps_for(m, xh, xl, lh, ll, n_tok, D, ldd, LX_BK, n_tok, nv, ldl, LX_BK)) return rc;
                g.span = lx_span(split ? 3 : 2);
                g.kblocks = lx_div(n_tok, LX_BK);
                g.m_tiles = lx_div(D, LX_BM); g.m = D;
                const bool narrow_e = split && lx_narrow(g.m_tiles, nv);
                const int acc_n = lx_acc_n(narrow_e ? LX_NARROW : LX_PLAIN);
                g.n_tiles = lx_div(nv, acc_n); g.n = nv;
                g.idesc = lx_idesc(half_type, true, true, acc_n);
                g.out = c.d_table + (size_t)v0 * D; g.ldt = (size_t)D; g.alpha = alpha;
                if (int rc = !split ? lx_start<LX_DTABLE, LX_TWO>(c.st, m, g) : narrow_e ? lx_start<LX_DTABLE, LX_NARROW>(c.st, m, g) : lx_start<LX_DTABLE, LX_SPLIT>(c.st, m, g)) return rc;
            }
        }
        if (c.dx) {
            const int by = D < 1024 ? D : 1024;
            with_dx = t0 + n_tok == T_all && c.B <= 4 * lx_div(n_tok, 256);      // a block takes a few sequences, one after the other
            lx_call(lx_finish_dx_kernel<T>, dim3(lx_div(n_tok, 256), by + with_dx), dim3(256), 0, c.st, static_cast<T *>(c.dx), dxs, c.targets, c.id_u16, V, splits, t0, n_tok, D, c.S, ldt,
                    alpha, with_dx ? c.loss_seq : nullptr, loss_tok, c.B);
            ANE_LAUNCH_OK(1);
        }
    }
    if (!with_dx) {
        lx_call(lx_loss_kernel, dim3(c.B), dim3(256), 0, c.st, c.loss_seq, loss_tok, c.S);
        ANE_LAUNCH_OK(1);
    }
    return ANE_CUDA_OK;
}

}  // namespace ane

using namespace ane;

extern "C" {

int ane_cuda_linear_cross_entropy_dev(void *stream, ane_dtype dtype, ane_idtype idtype, int B, int D, int V, int S, float *loss_seq, float *loss_tok, void *dx,
                                      float *d_table, const void *x, const void *table, const void *targets, float grad_scale) {
    ANE_REQUIRE_INIT();
    ANE_REQUIRE(loss_seq && x && table && targets, "%s: null pointer", __func__);
    ANE_REQUIRE(dtype_ok(dtype), "%s: bad dtype %d", __func__, (int)dtype);
    ANE_REQUIRE(idtype == ANE_ID_U16 || idtype == ANE_ID_I32, "%s: bad id type", __func__);
    ANE_REQUIRE(B >= 1 && D >= 1 && V >= 1 && S >= 1, "%s: bad shape B=%d D=%d V=%d S=%d", __func__, B, D, V, S);
    // up to 2^30, the sum of an index and a step over tokens or rows fits an int
    ANE_REQUIRE((long long)B * S <= 1 << 30 && V <= 1 << 30 && D <= 65536, "%s: more than 2^30 tokens or rows, or D above 65536", __func__);
    ANE_REQUIRE(!dx || dx != x, "%s: dx may not be x", __func__);
    const size_t e = dtype_size(dtype), xb = (size_t)B * D * S * e;
    ANE_CHECK_EXTENT(loss_seq, (size_t)B * 4); ANE_CHECK_EXTENT(loss_tok, (size_t)B * S * 4); ANE_CHECK_EXTENT(dx, xb); ANE_CHECK_EXTENT(x, xb);
    ANE_CHECK_EXTENT(table, (size_t)V * D * e); ANE_CHECK_EXTENT(d_table, (size_t)V * D * 4);
    ANE_CHECK_EXTENT(targets, (size_t)B * S * (idtype == ANE_ID_U16 ? 2 : 4));
    const LxCall c = {(cudaStream_t)stream, dtype, idtype == ANE_ID_U16, B, D, V, S, loss_seq, loss_tok, dx, d_table, x, table, targets, grad_scale};
    switch (dtype) {
        case ANE_F32: return lx_run<float, __half>(c);
        case ANE_BF16: return lx_run<__nv_bfloat16, __nv_bfloat16>(c);
        default: return lx_run<__half, __half>(c);
    }
}

}  // extern "C"
