// block_norm_ring.cuh -- backward pass of the norms around a block as a pipeline, for aligned rows, channels in multiples of
// 128 up to 1024, and many tokens.
//
// One block per SM, clusters of up to eight blocks that share the channels of a tile (128 bytes of tokens per row, 128 rows per
// block) and walk the tiles.  The copy engine fills a ring of three stages (x2, dy, f, dx2 of one tile).  While the per-token
// sums of tile j travel, the rows of tile j-1 are finished, so neither the copies nor the exchange stand in the way:
//
//   16 warps        sums of tile j | factors of tile j-1 arrive | sums of j on their way | rows of tile j-1 read again, written
//   exchange warp   sums of the tokens that this block owns, from all blocks of the cluster -> factors -> to all of them
//   copy warp       fills stages as they come free
//
// A lane holds one 32-bit word of a row (two 16-bit tokens, or one fp32), so the sums need no reduction inside a warp: 12
// accumulators against 48 with 16-byte vectors.  Sums and factors cross the cluster as asynchronous stores that complete a
// transaction barrier at their destination.  One slot for sums and one for factors are enough: a block sends the sums of tile
// j only after the factors of tile j-1 have arrived from all blocks, which is after these have read the sums of tile j-1.
#pragma once
#include "common.cuh"
#include "tma.cuh"

namespace ane {

constexpr int BR_WARPS = 16, BR_THREADS = (BR_WARPS + 2) * 32;       // + exchange warp, copy warp
constexpr int BR_ROWS = 128, BR_NR = BR_ROWS / BR_WARPS;             // rows of a block, of a warp
constexpr int BR_STAGES = 3, BR_BOX = BR_ROWS * 128;
constexpr uint32_t BR_WAIT_LIMIT = 1u << 20;

template <typename T> struct BrWord;      // one 32-bit word of a row
template <> struct BrWord<float> {
    static constexpr int W = 1;
    __device__ __forceinline__ static V<1> get(uint32_t w) { V<1> v; v.a = __uint_as_float(w); return v; }
    __device__ __forceinline__ static uint32_t put(const V<1> &v) { return __float_as_uint(v.a); }
};
template <> struct BrWord<__nv_bfloat16> {
    static constexpr int W = 2;
    __device__ __forceinline__ static V<2> get(uint32_t w) { V<2> v; v.p[0] = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); return v; }
    __device__ __forceinline__ static uint32_t put(const V<2> &v) {
        const __nv_bfloat162 q = __floats2bfloat162_rn(v.p[0].x, v.p[0].y);
        return *reinterpret_cast<const uint32_t *>(&q);
    }
};
template <> struct BrWord<__half> {
    static constexpr int W = 2;
    __device__ __forceinline__ static V<2> get(uint32_t w) { V<2> v; v.p[0] = __half22float2(*reinterpret_cast<const __half2 *>(&w)); return v; }
    __device__ __forceinline__ static uint32_t put(const V<2> &v) {
        const __half2 q = __floats2half2_rn(v.p[0].x, v.p[0].y);
        return *reinterpret_cast<const uint32_t *>(&q);
    }
};
__device__ __forceinline__ float br_hsum(const V<1> &v) { return v.a; }
__device__ __forceinline__ float br_hsum(const V<2> &v) { return v.p[0].x + v.p[0].y; }
__device__ __forceinline__ void br_store(float *p, const V<1> &v) { *p = v.a; }
__device__ __forceinline__ void br_store(float *p, const V<2> &v) { *reinterpret_cast<float2 *>(p) = v.p[0]; }
__device__ __forceinline__ void br_load(V<1> &v, const float *p) { v.a = *p; }
__device__ __forceinline__ void br_load(V<2> &v, const float *p) { v.p[0] = *reinterpret_cast<const float2 *>(p); }

__device__ __forceinline__ uint32_t br_at(uint32_t local, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}
// Stores a float in a block of the cluster and counts its bytes on that block's barrier.
__device__ __forceinline__ void br_send(uint32_t at, uint32_t bar, float v) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(at), "f"(v), "r"(bar) : "memory");
}
// Bounded wait, cluster scope; after a give-up anywhere in the block every wait returns at once and the rest of the work runs
// on whatever is there (in bounds), so that all warps still meet at their barriers.
__device__ __forceinline__ void br_wait(uint64_t *bar, uint32_t parity, volatile int *give_up) {
    for (uint32_t i = 0; i < BR_WAIT_LIMIT; i++) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (ok || *give_up) return;
    }
    *give_up = 1;
}

struct BrMaps { CUtensorMap t[4]; };         // x2, dy, f, dx2
struct BrLayout {                            // shared memory behind the ring
    float red[BR_WARPS][6][64];
    float mail[6 * 72];                      // [block][6][own tokens]: at most 64 tokens and a rounding per block
    float fac[4][64];
    uint64_t full[BR_STAGES], empty[BR_STAGES], mail_bar, fac_bar;
    int give_up;
};
constexpr size_t BR_SMEM = 1024 + (size_t)BR_STAGES * 4 * BR_BOX + sizeof(BrLayout);

// POST: there is a norm behind the block; DX2: a gradient arrives at x2.  (As conditions at run time inside the unrolled rows
// they cost a quarter of the instructions.)  Every block has all of its 128 rows: a condition per row, for a number of channels
// that is no multiple of 128, keeps the loads of the rows from being started together (198 -> 340 us; the cluster form takes
// 245).
template <typename T, bool POST, bool DX2>
__global__ void __launch_bounds__(BR_THREADS, 1)
block_norm_bwd_ring_kernel(const __grid_constant__ BrMaps maps, T *__restrict__ dx, T *__restrict__ df, float *__restrict__ partial, const float *__restrict__ w_post,
                           const float *__restrict__ gate, const float *__restrict__ w_pre, BnShape sh, int tiles, ane_cuda_status *status) {
    using Word = BrWord<T>;
    constexpr int W = Word::W, TW = 32 * W;
    extern __shared__ uint8_t raw[];
    uint8_t *ring = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);       // the same offset in every block
    BrLayout &L = *reinterpret_cast<BrLayout *>(ring + (size_t)BR_STAGES * 4 * BR_BOX);
    volatile int *give_up = &L.give_up;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const uint32_t blocks = bn_size(), rank = bn_rank();
    const int clusters = gridDim.x / blocks, first = blockIdx.x / blocks;
    const int n_items = first < tiles ? (tiles - first + clusters - 1) / clusters : 0;
    const int c0 = (int)rank * BR_ROWS;
    const int per_owner = (TW + (int)blocks - 1) / (int)blocks;
    const int own0 = (int)rank * per_owner, own = own0 >= TW ? 0 : TW - own0 < per_owner ? TW - own0 : per_owner;
    if (threadIdx.x == 0) {
        for (int i = 0; i < BR_STAGES; i++) { mbar_init(&L.full[i], 1); mbar_init(&L.empty[i], BR_WARPS); }
        mbar_init(&L.mail_bar, 1);
        mbar_init(&L.fac_bar, 1);
        L.give_up = 0;
        mbar_init_fence();
        if (own) mbar_arrive_expect_tx(&L.mail_bar, blocks * 6 * own * 4);
        mbar_arrive_expect_tx(&L.fac_bar, 4 * TW * 4);
    }
    __syncthreads();
    bn_cluster_arrive();
    bn_cluster_wait();
    dep_sync();

    int issued = 0;
    if (warp == BR_WARPS + 1) {
        if (lane == 0) {
            for (int it = 0; it < n_items && !*give_up; it++) {
                const int st = it % BR_STAGES, tile = first + it * clusters;
                br_wait(&L.empty[st], ((it / BR_STAGES) & 1) ^ 1, give_up);
                if (*give_up) break;
                const int b = tile / sh.tiles_per_seq, t0 = (tile - b * sh.tiles_per_seq) * TW;
                uint8_t *to = ring + (size_t)st * 4 * BR_BOX;
                mbar_arrive_expect_tx(&L.full[st], (DX2 ? 4 : 3) * BR_BOX);
                for (int i = 0; i < (DX2 ? 4 : 3); i++) tma_load_3d(to + i * BR_BOX, &maps.t[i], t0, c0, b, &L.full[st]);
                issued = it + 1;
            }
            // after a give-up: the copies in flight land before the block ends
            if (*give_up)
                for (int it = issued > BR_STAGES ? issued - BR_STAGES : 0; it < issued; it++) mbar_wait_bounded(&L.full[it % BR_STAGES], (it / BR_STAGES) & 1);
        }
    } else if (warp == BR_WARPS) {
        const BnBwd<64> factors = {1.0f / (float)sh.C, sh.eps, 1.0f, POST};      // alpha is in the sums already
        for (int it = 0; it < n_items && own; it++) {
            br_wait(&L.mail_bar, it & 1, give_up);
            if (__any_sync(0xffffffffu, *give_up)) break;
            if (lane == 0) mbar_arrive_expect_tx(&L.mail_bar, blocks * 6 * own * 4);
            __syncwarp();
            for (int j = lane; j < own; j += 32) {
                float s[6 * 64 - 63];                                     // 6 sums, 64 apart, as the functor reads them
#pragma unroll
                for (int k = 0; k < 6; k++) {
                    float a = 0.0f;
                    for (uint32_t r = 0; r < blocks; r++) a += L.mail[(r * 6 + k) * own + j];
                    s[64 * k] = a;
                }
                factors(s);
                for (uint32_t r = 0; r < blocks; r++) {
                    const uint32_t bar = br_at(smem_u32(&L.fac_bar), r);
#pragma unroll
                    for (int k = 0; k < 4; k++) br_send(br_at(smem_u32(&L.fac[k][own0 + j]), r), bar, s[64 * k]);
                }
            }
        }
    } else {
        const bool want_p = POST || gate;
        const int row0 = c0 + warp;                // rows row0, row0 + 16, ... of this warp
        // w_pre, and alpha * gate * w_post.  A gate per sequence: of sequence k1_of, read again when another one is needed (two
        // sets would not fit the registers).
        V<W> k2[BR_NR], k1[BR_NR];
        int k1_of = 0;
        auto load_k1 = [&](int b) {
            k1_of = b;
#pragma unroll
            for (int k = 0; k < BR_NR; k++) {
                const int c = row0 + k * BR_WARPS;
                float v = sh.alpha;
                if constexpr (POST) v *= __ldg(w_post + c);
                if (gate) v *= __ldg(gate + (size_t)b * sh.gate_stride + c);
                k1[k] = V<W>::splat(v);
            }
        };
#pragma unroll
        for (int k = 0; k < BR_NR; k++) k2[k] = V<W>::splat(__ldg(w_pre + row0 + k * BR_WARPS));
        load_k1(0);
        // this thread's share of the exchange: one sum over the warps, and where it goes
        static_assert(6 * TW <= BR_WARPS * 32, "one sum per thread");
        const bool sends = threadIdx.x < 6 * TW;
        const float *red_at = &L.red[0][sends ? threadIdx.x / TW : 0][threadIdx.x % TW];
        const int owner = (int)(threadIdx.x % TW) / per_owner, at_owner = (int)(threadIdx.x % TW) - owner * per_owner;
        const int own_there = TW - owner * per_owner < per_owner ? TW - owner * per_owner : per_owner;
        const uint32_t send_at = sends ? br_at(smem_u32(&L.mail[((int)rank * 6 + threadIdx.x / TW) * own_there + at_owner]), owner) : 0;
        const uint32_t send_bar = sends ? br_at(smem_u32(&L.mail_bar), owner) : 0;
        const size_t step = (size_t)BR_WARPS * sh.S;
        size_t base_last = 0;
        int tile_last = 0, b_last = 0;
        bool active_last = false;
        for (int it = 0; it <= n_items; it++) {
            const bool cur = it < n_items;
            const int tile = first + it * clusters, b = cur ? tile / sh.tiles_per_seq : b_last;
            const int t = (tile - b * sh.tiles_per_seq) * TW + lane * W;
            V<W> s[6];
            if (cur) {
                if (sh.gate_stride && k1_of != b) load_k1(b);
                br_wait(&L.full[it % BR_STAGES], (it / BR_STAGES) & 1, give_up);
                const uint32_t *w = reinterpret_cast<const uint32_t *>(ring + (size_t)(it % BR_STAGES) * 4 * BR_BOX) + warp * 32 + lane;
#pragma unroll
                for (int i = 0; i < 6; i++) s[i] = V<W>::splat(0.0f);
#pragma unroll
                for (int k = 0; k < BR_NR; k++) {
                    const uint32_t *r = w + k * BR_WARPS * 32;
                    const V<W> vx = Word::get(r[0]), va = vmul(Word::get(r[BR_BOX / 4]), k2[k]);
                    s[0] = vfma(vx, vx, s[0]);
                    s[1] = vfma(va, vx, s[1]);
                    if constexpr (POST) {
                        const V<W> vf = Word::get(r[2 * (BR_BOX / 4)]), vq = vmul(vf, k1[k]);
                        s[2] = vfma(vf, vf, s[2]);
                        if constexpr (DX2) s[3] = vfma(vq, Word::get(r[3 * (BR_BOX / 4)]), s[3]);
                        s[4] = vfma(vq, va, s[4]);
                        s[5] = vfma(vq, vx, s[5]);
                    }
                    }
            }
            V<W> r2, nk, rf, nj;
            if (it > 0) {
                br_wait(&L.fac_bar, (it - 1) & 1, give_up);
                br_load(r2, &L.fac[0][lane * W]);
                br_load(nk, &L.fac[1][lane * W]);
                br_load(rf, &L.fac[2][lane * W]);
                br_load(nj, &L.fac[3][lane * W]);
                if (threadIdx.x == 0 && !*give_up) mbar_arrive_expect_tx(&L.fac_bar, 4 * TW * 4);
            }
            if (cur) {
#pragma unroll
                for (int i = 0; i < 6; i++) br_store(&L.red[warp][i][lane * W], s[i]);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(BR_WARPS * 32) : "memory");
            if (cur && sends) {
                float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < BR_WARPS; i++) x[i & 3] += red_at[i * 6 * 64];
                br_send(send_at, send_bar, (x[0] + x[1]) + (x[2] + x[3]));
            }
            if (it > 0) {
                if (sh.gate_stride && k1_of != b_last) load_k1(b_last);
                const int st = (it - 1) % BR_STAGES;
                const uint32_t *w = reinterpret_cast<const uint32_t *>(ring + (size_t)st * 4 * BR_BOX) + warp * 32 + lane;
                float sums[2 * BR_NR];
                T *px = dx + base_last, *pf = df + base_last;
#pragma unroll
                for (int k = 0; k < BR_NR; k++) {
                    const uint32_t *r = w + k * BR_WARPS * 32;
                    const V<W> vx = Word::get(r[0]), vf = Word::get(r[2 * (BR_BOX / 4)]);
                    const V<W> u = vmul(Word::get(r[BR_BOX / 4]), r2);                     // dy * r_2
                    V<W> G;
                    if constexpr (DX2) G = vfma(u, k2[k], vfma(nk, vx, Word::get(r[3 * (BR_BOX / 4)])));
                    else G = vfma(u, k2[k], vmul(nk, vx));
                    const V<W> h = vmul(G, rf);
                    sums[2 * k] = br_hsum(vmul(u, vx));
                    sums[2 * k + 1] = br_hsum(vmul(h, vf));
                    if (active_last) {
                        __stcs(reinterpret_cast<unsigned int *>(px), Word::put(G));
                        __stcs(reinterpret_cast<unsigned int *>(pf), Word::put(vfma(h, k1[k], vmul(nj, vf))));
                    }
                    px += step;
                    pf += step;
                }
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&L.empty[st])) : "memory");
                // over the lanes: four steps exchange halves, the fifth adds; lanes with an even number write
                int at = 0;
#pragma unroll
                for (int off = 16, left = BR_NR; off > 1; off >>= 1, left >>= 1) {
                    const bool up = lane & off;
#pragma unroll
                    for (int i = 0; i < BR_NR; i++)
                        if (i < left) {
                            const float other = __shfl_xor_sync(0xffffffffu, up ? sums[i] : sums[i + left], off);
                            sums[i] = (up ? sums[i + left] : sums[i]) + other;
                        }
                    at += up ? left : 0;
                }
                sums[0] += __shfl_xor_sync(0xffffffffu, sums[0], 1);
                if (!(lane & 1) && ((at & 1) == 0 || want_p))
                    partial[((size_t)tile_last * sh.C + row0 + at / 2 * BR_WARPS) * 2 + (at & 1)] = sums[0];
            }
            if (cur) {
                base_last = ((size_t)b * sh.C + row0) * sh.S + t;
                tile_last = tile;
                b_last = b;
                active_last = t < sh.S;
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && *give_up) atomicAdd(&status->wait_giveups, 1);
    bn_cluster_leave();
    bn_cluster_wait();                       // a peer may still send to this block
}

}  // namespace ane
