// block_norm.cu -- the norms around a transformer block in one operator, forward and backward:
//
//   n  = f * r_f * w_post             r_f = 1 / sqrt(mean_c f^2 + eps)      (w_post NULL: n = f)
//   x2 = x + alpha * gate * n         rounded to the storage type            (gate NULL: 1)
//   y  = x2 * r_2 * w_pre             r_2 = 1 / sqrt(mean_c x2^2 + eps), from the rounded x2
//
// f is the block's output, x the residual stream, w_post the norm behind the block, w_pre the norm before the next one; gate
// is fp32, one value per channel or per (sequence, channel).  Tensors are [B][C][S], sums over c have stride S.
//
// Backward, with dy and dx2 the gradients of the two outputs:
//   a  = w_pre * dy,  k = r_2^3 * mean(a * x2)
//   G  = dx2 + r_2 * a - k * x2                                             = dx
//   q  = gate * w_post * f,  j = alpha * r_f^3 * mean(q * G)
//   df = alpha * r_f * gate * w_post * G - j * f                            (w_post NULL: alpha * gate * G)
//   dw_pre = sum dy * x2 * r_2,   P = alpha * sum f * r_f * G,   dw_post = gate * P,   dgate = w_post * P
// G is linear in quantities known per element, so mean(q * G) comes out of the same sweep as the other sums:
//   sum q G = sum q dx2 + r_2 sum q a - k sum q x2
// -- six sums over the channels in one sweep, one exchange, then the sweep that writes.
//
// Both directions move each tensor once at best (4 and 6 tensor passes) and do a few operations per element, so HBM is the
// floor; what they run into before it are the phases of a tile (loads, sums, exchange, stores), which a block goes through one
// after the other.  Measured, 32 sequences x 2048 tokens x 1024 channels in bf16 (82 and 123 us at the copy rate):
//   forward   115 us   one block of 512 threads per 32 tokens, two blocks per SM       (4.7 TB/s)
//             138      clusters of eight blocks of 256 threads, 128-byte rows
//             157      three sweeps through L2
//   backward  199 us   pipeline over clusters (block_norm_ring.cuh): 15 clusters of eight, 59 % of their issue slots busy  (4.0 TB/s)
//             245      one block of 512 threads per 32 tokens; clusters of eight, 128-byte rows: 250
//             380      two sweeps through L2
// Rows that break 16-byte alignment (5 x 1000 x 333 in fp16): 24 us over clusters of eight against 125 us in one block per tile.
#include "common.cuh"

#include <type_traits>

namespace ane {

constexpr int BN_THREADS = 256;
constexpr int BN_WARPS = BN_THREADS / 32;

struct BnShape {
    int B, C, S;
    int tiles_per_seq;
    int rows_per_seq;        // gate per sequence: blocks (= rows of partial sums) per sequence; 0: blocks walk all tiles
    int gate_stride;         // 0 or C
    float alpha, eps;
};

// Sum over the row groups of a warp (lanes of equal lane % LG), every lane gets the total.
template <int N, int LG> __device__ __forceinline__ V<N> bn_warp_sum(V<N> v) {
#pragma unroll
    for (int off = LG; off < 32; off <<= 1)
#pragma unroll
        for (int j = 0; j < N; j++) v.set(j, v.get(j) + __shfl_xor_sync(0xffffffffu, v.get(j), off));
    return v;
}
// Sum over the LG lanes of a row.
template <int LG> __device__ __forceinline__ float bn_row_sum(float v) {
#pragma unroll
    for (int off = LG / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// Per-token factors out of per-token sums, once per token and not once per thread (a root and a division are 25
// instructions): `tot` points at a token's sums, TW apart; the factors replace the first of them.
template <int TW> struct BnRms {                         // sum of squares -> 1 / rms
    static constexpr int FACTORS = 1;
    float inv_c, eps;
    __device__ __forceinline__ void operator()(float *tot) const { tot[0] = 1.0f / sqrtf(fmaf(tot[0], inv_c, eps)); }
};
// The six sums of the backward pass -> r_2, -k, r_f, -j.
template <int TW> struct BnBwd {
    static constexpr int FACTORS = 4;
    float inv_c, eps, alpha;
    bool post;
    __device__ __forceinline__ void operator()(float *tot) const {
        const float r2 = 1.0f / sqrtf(fmaf(tot[0], inv_c, eps));
        const float rf = post ? 1.0f / sqrtf(fmaf(tot[2 * TW], inv_c, eps)) : 1.0f;
        const float k = r2 * r2 * r2 * (tot[TW] * inv_c);
        const float j = post ? alpha * rf * rf * rf * (inv_c * (tot[3 * TW] + r2 * tot[4 * TW] - k * tot[5 * TW])) : 0.0f;
        tot[0] = r2;
        tot[TW] = -k;
        tot[2 * TW] = rf;
        tot[3 * TW] = -j;
    }
};

// NS per-token sums over the block, then their factors: each warp's total goes to shared memory, the warps are added in order.
// `red` holds [NS][warps][TW] floats, `tot` [NS][TW].  Ends with the factors in registers; `tot` is read until the next
// barrier.
template <int NS, int N, int LG, typename F> __device__ __forceinline__ void bn_block_sums(V<N> (&v)[NS], float *red, float *tot, F finish) {
    constexpr int TW = N * LG;
    const int lg = threadIdx.x % LG, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
#pragma unroll
    for (int s = 0; s < NS; s++) {
        v[s] = bn_warp_sum<N, LG>(v[s]);
        if (lane < LG) lanes_to_smem<N>(red + (s * BN_WARPS + warp) * TW + lg * N, v[s]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NS * TW; i += BN_THREADS) {
        const int s = i / TW, t = i % TW;
        float a = 0.0f;
#pragma unroll
        for (int w = 0; w < BN_WARPS; w++) a += red[(s * BN_WARPS + w) * TW + t];
        tot[i] = a;
    }
    __syncthreads();
    if (threadIdx.x < TW) finish(tot + threadIdx.x);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < F::FACTORS; s++) v[s] = lanes_from_smem<N>(tot + s * TW + lg * N);
}

// Any shape.  A block owns a [C x LG*VEC] token tile and sweeps the channels up to three times; what one sweep read the
// next finds in L2.  VEC = 1 covers rows that break 16-byte alignment, LG = 1 sequences of very few tokens, where
// neighbouring threads take neighbouring channels.
template <typename T, int VEC, int LG>
__global__ void __launch_bounds__(BN_THREADS)
block_norm_kernel(T *x2, T *y, const T *x, const T *f, const float *__restrict__ w_post, const float *__restrict__ gate,
                  const float *__restrict__ w_pre, BnShape sh) {
    constexpr int R = BN_THREADS / LG, TW = LG * VEC;
    __shared__ __align__(16) float red[BN_WARPS * TW];
    __shared__ __align__(16) float tot[TW];
    const int b = blockIdx.x / sh.tiles_per_seq;
    const int lg = threadIdx.x % LG, rg = threadIdx.x / LG;
    const int t = (blockIdx.x % sh.tiles_per_seq) * TW + lg * VEC;
    const bool active = t < sh.S;
    const size_t base = (size_t)b * sh.C * sh.S + t;
    const float inv_c = 1.0f / (float)sh.C;
    if (gate) gate += (size_t)b * sh.gate_stride;

    const BnRms<TW> rms = {inv_c, sh.eps};
    V<VEC> rf = V<VEC>::splat(1.0f);
    if (w_post) {
        V<VEC> ss[1] = {V<VEC>::splat(0.0f)};
        if (active)
#pragma unroll 4
            for (int c = rg; c < sh.C; c += R) {
                Raw<T, VEC> r;
                r.load(f + base + (size_t)c * sh.S);
                ss[0] = vfma(r.get(), r.get(), ss[0]);
            }
        bn_block_sums<1, VEC, LG>(ss, red, tot, rms);
        rf = ss[0];
    }
    V<VEC> ss[1] = {V<VEC>::splat(0.0f)};
    if (active)
#pragma unroll 4
        for (int c = rg; c < sh.C; c += R) {
            const size_t at = base + (size_t)c * sh.S;
            Raw<T, VEC> r, q;
            r.load(f + at);
            q.load(x + at);
            const float k = sh.alpha * (gate ? __ldg(gate + c) : 1.0f) * (w_post ? __ldg(w_post + c) : 1.0f);
            q.put(vfma_s(vmul(r.get(), rf), k, q.get()));
            q.store(x2 + at);
            ss[0] = vfma(q.get(), q.get(), ss[0]);
        }
    bn_block_sums<1, VEC, LG>(ss, red, tot, rms);
    const V<VEC> r2 = ss[0];
    if (active)
#pragma unroll 4
        for (int c = rg; c < sh.C; c += R) {
            const size_t at = base + (size_t)c * sh.S;
            Raw<T, VEC> q;
            q.load(x2 + at);                          // this thread's own stores
            q.put(vscale(vmul(q.get(), r2), __ldg(w_pre + c)));
            q.store(y + at);
        }
}

template <typename T, int VEC, int LG>
__global__ void __launch_bounds__(BN_THREADS)
block_norm_bwd_kernel(T *dx, T *df, float *__restrict__ partial, const T *dy, const T *dx2, const T *x2, const T *f,
                      const float *__restrict__ w_post, const float *__restrict__ gate, const float *__restrict__ w_pre, BnShape sh) {
    constexpr int R = BN_THREADS / LG, TW = LG * VEC;
    __shared__ __align__(16) float red[6 * BN_WARPS * TW];
    __shared__ __align__(16) float tot[6 * TW];
    const int lg = threadIdx.x % LG, rg = threadIdx.x / LG;
    const float inv_c = 1.0f / (float)sh.C;
    float *prow = partial + (size_t)blockIdx.x * 2 * sh.C;
    // tiles of this block: those of one sequence, or of all of them
    const int per = sh.rows_per_seq;
    const long long first = per ? (long long)(blockIdx.x / per) * sh.tiles_per_seq + blockIdx.x % per : blockIdx.x;
    const long long step = per ? per : gridDim.x;
    const long long end = per ? (long long)(blockIdx.x / per + 1) * sh.tiles_per_seq : (long long)sh.B * sh.tiles_per_seq;
    const bool want_p = w_post || gate;
    for (long long tile = first; tile < end; tile += step) {
        const int b = (int)(tile / sh.tiles_per_seq);
        const int t = (int)(tile % sh.tiles_per_seq) * TW + lg * VEC;
        const bool active = t < sh.S;
        const size_t base = (size_t)b * sh.C * sh.S + t;
        const float *g = gate ? gate + (size_t)b * sh.gate_stride : nullptr;
        V<VEC> s[6];
#pragma unroll
        for (int i = 0; i < 6; i++) s[i] = V<VEC>::splat(0.0f);
        if (active)
#pragma unroll 2
            for (int c = rg; c < sh.C; c += R) {
                const size_t at = base + (size_t)c * sh.S;
                Raw<T, VEC> rx, ry, rd, rf;
                rx.load(x2 + at);
                ry.load(dy + at);
                if (w_post) { rf.load(f + at); if (dx2) rd.load(dx2 + at); }
                const V<VEC> vx = rx.get(), va = vscale(ry.get(), __ldg(w_pre + c));
                s[0] = vfma(vx, vx, s[0]);
                s[1] = vfma(va, vx, s[1]);
                if (w_post) {
                    const V<VEC> vf = rf.get(), vq = vscale(vf, (g ? __ldg(g + c) : 1.0f) * __ldg(w_post + c));
                    s[2] = vfma(vf, vf, s[2]);
                    if (dx2) s[3] = vfma(vq, rd.get(), s[3]);
                    s[4] = vfma(vq, va, s[4]);
                    s[5] = vfma(vq, vx, s[5]);
                }
            }
        bn_block_sums<6, VEC, LG>(s, red, tot, BnBwd<TW>{inv_c, sh.eps, sh.alpha, w_post != nullptr});
        const V<VEC> r2 = s[0], nk = s[1], rms_f = s[2], nj = s[3];
        for (int c = rg; c < (sh.C + R - 1) / R * R; c += R) {     // whole warps stay together for the row sums
            float sum_q = 0.0f, sum_p = 0.0f;
            if (active && c < sh.C) {
                const size_t at = base + (size_t)c * sh.S;
                Raw<T, VEC> rx, ry, rd, rf;
                rx.load(x2 + at);
                ry.load(dy + at);
                if (dx2) rd.load(dx2 + at);
                rf.load(f + at);
                const V<VEC> vx = rx.get(), vy = ry.get(), vf = rf.get();
                const V<VEC> z = vmul(vx, r2);
                V<VEC> G = vfma(vscale(vy, __ldg(w_pre + c)), r2, vmul(nk, vx));
                if (dx2) G = vadd(G, rd.get());
                sum_q = vmul(vy, z).hsum();
                const float gw = (g ? __ldg(g + c) : 1.0f) * (w_post ? __ldg(w_post + c) : 1.0f);
                const V<VEC> u = vmul(vf, rms_f);
                sum_p = vmul(u, G).hsum();
                rx.put(G);
                rx.store(dx + at);
                rf.put(vfma(vscale(G, sh.alpha * gw), rms_f, vmul(nj, vf)));
                rf.store(df + at);
            }
            sum_q = bn_row_sum<LG>(sum_q);
            if (want_p) sum_p = bn_row_sum<LG>(sum_p);
            if (lg == 0 && c < sh.C) {
                float *p = prow + 2 * (size_t)c;
                if (tile == first) { p[0] = sum_q; p[1] = sum_p; }
                else { p[0] += sum_q; p[1] += sum_p; }
            }
        }
        __syncthreads();                              // tot is read until here, and rewritten by the next tile
    }
}

// ------------------------------------------------------------------ clusters
// The channels of a token tile are shared out over a cluster of up to eight blocks, each of which keeps its part of the tile
// on the SM (forward in registers, backward in shared memory) between the sweeps, so that every tensor crosses HBM once.  The
// per-token sums of the blocks meet in distributed shared memory and are added in block order.  Rows of 16-byte vectors; LG
// lanes per row, NV rows per thread.
__device__ __forceinline__ uint32_t bn_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t bn_size() { uint32_t r; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void bn_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void bn_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// An arrival that publishes nothing (a release would wait for this thread's stores to global memory).
__device__ __forceinline__ void bn_cluster_leave() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ float bn_peer(const float *p, uint32_t rank) {
    uint32_t at;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// Sums of N values a lane over the lanes that differ in the bits OFF, 2*OFF, ... 16.  As long as the count allows it a step
// exchanges halves: the lane with the bit set goes on with the upper half, so each step halves the work.  `first` is the index
// of the values that a lane ends up with; lanes that only hold copies drop out as writers.  -> number of values held.
template <int N, int OFF> struct BnFold {
    static constexpr bool HALVE = N % 8 == 0;
    static constexpr int LEFT = BnFold<HALVE ? N / 2 : N, 2 * OFF>::LEFT;
    __device__ __forceinline__ static void run(float *a, int lane, int &first, bool &writer) {
        const bool up = lane & OFF;
        if constexpr (HALVE) {
#pragma unroll
            for (int i = 0; i < N / 2; i++) {
                const float other = __shfl_xor_sync(0xffffffffu, up ? a[i] : a[i + N / 2], OFF);
                a[i] = (up ? a[i + N / 2] : a[i]) + other;
            }
            first += up ? N / 2 : 0;
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) a[i] += __shfl_xor_sync(0xffffffffu, a[i], OFF);
            writer = writer && !up;
        }
        BnFold<HALVE ? N / 2 : N, 2 * OFF>::run(a, lane, first, writer);
    }
};
template <int N> struct BnFold<N, 32> {
    static constexpr int LEFT = N;
    __device__ __forceinline__ static void run(float *, int, int &, bool &) {}
};

// NS per-token sums over the cluster, the warps' parts three sums at a time (`red` holds [3][warps][TW]: three blocks fit an SM
// then).  `mine` [NS][TW] is read by the other blocks until the next cluster barrier behind this call, so it is not reused
// before that.
template <int NS, int N, int LG, int THREADS, typename F> __device__ __forceinline__ void bn_cluster_sums(V<N> (&v)[NS], float *red, float *mine, float *tot, F finish) {
    constexpr int TW = N * LG, PER = NS < 3 ? NS : 3, WARPS = THREADS / 32;
    const int lg = threadIdx.x % LG, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const uint32_t blocks = bn_size();
#pragma unroll
    for (int s0 = 0; s0 < NS; s0 += PER) {
        float a[PER * N];
#pragma unroll
        for (int s = 0; s < PER; s++)
#pragma unroll
            for (int j = 0; j < N; j++) a[s * N + j] = v[s0 + s].get(j);
        int first = 0;
        bool writer = true;
        BnFold<PER * N, LG>::run(a, lane, first, writer);
        if (s0) __syncthreads();
        constexpr int LEFT = BnFold<PER * N, LG>::LEFT;
        static_assert(N == 1 || LEFT % 4 == 0, "whole 16-byte words");
        if constexpr (N == 1) {
#pragma unroll
            for (int s = 0; s < PER; s++) red[(s * WARPS + warp) * TW + lg] = a[s];
        } else if (writer) {
#pragma unroll
            for (int i = 0; i < LEFT; i += 4) {
                const int at = first + i;                         // value at % N of sum at / N
                *reinterpret_cast<float4 *>(red + ((at / N) * WARPS + warp) * TW + lg * N + at % N) = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
            }
        }
        __syncthreads();
        if constexpr (NS == 1 && N > 1 && TW <= 32) {
            if (blocks == 1) {
                // one block: every warp adds up the warps' parts itself, a lane per token, and no second barrier is needed (`red` is
                // not used again by the next exchange)
                float a = 0.0f;
                if (lane < TW) {
#pragma unroll
                    for (int w = 0; w < WARPS; w++) a += red[w * TW + lane];
                }
                finish(&a);
#pragma unroll
                for (int j = 0; j < N; j++) v[0].set(j, __shfl_sync(0xffffffffu, a, lg * N + j));
                return;
            }
        }
        for (int i = threadIdx.x; i < PER * TW; i += THREADS) {
            const int s = i / TW, t = i % TW;
            float a = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) a += red[(s * WARPS + w) * TW + t];
            mine[s0 * TW + i] = a;
        }
    }
    if (blocks > 1) {
        bn_cluster_arrive();
        bn_cluster_wait();
    } else if (NS > 1) {
        __syncthreads();
    }
    for (int i = threadIdx.x; i < NS * TW; i += THREADS) {     // for one block a thread's own entries again
        float a;
        if (blocks > 1) {
            float p[8];
#pragma unroll
            for (uint32_t r = 0; r < 8; r++) p[r] = r < blocks ? bn_peer(mine + i, r) : 0.0f;
            a = 0.0f;
#pragma unroll
            for (uint32_t r = 0; r < 8; r++) a += p[r];
        } else {
            a = mine[i];
        }
        tot[i] = a;
        if (NS == 1) finish(tot + i);                  // the thread that holds the sum
    }
    __syncthreads();
    if (NS > 1) {
        if (threadIdx.x < TW) finish(tot + threadIdx.x);
        __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < F::FACTORS; s++) v[s] = lanes_from_smem<N>(tot + s * TW + lg * N);
}

__device__ __forceinline__ void bn_copy16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void bn_copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A thread's own vectors of NT tensors, NV rows each: the first SM tensors in shared memory, filled by asynchronous copies that
// nobody else has to know of, the others in registers.
template <typename T, int VEC, int NT, int SM, int NV, int THREADS> struct BnStrip {
    static constexpr size_t BYTES = (size_t)SM * NV * THREADS * 16;
    uint4 *at;                                            // this thread's first entry
    Raw<T, VEC> r[NT - SM > 0 ? NT - SM : 1][NV];
    __device__ __forceinline__ BnStrip(uint4 *strip) : at(strip + threadIdx.x) {}
    __device__ __forceinline__ void fill(int tensor, int k, const T *p) {
        if (tensor < SM) bn_copy16(at + (tensor * NV + k) * THREADS, p); else r[tensor - SM][k].load_stream(p);
    }
    __device__ __forceinline__ void zero(int tensor, int k) {
        if (tensor < SM) at[(tensor * NV + k) * THREADS] = make_uint4(0, 0, 0, 0);
        else { V<VEC> z = V<VEC>::splat(0.0f); r[tensor - SM][k].put(z); }
    }
    __device__ __forceinline__ void done() { if (SM) bn_copies_done(); }
    __device__ __forceinline__ V<VEC> get(int tensor, int k) const {
        if constexpr (SM > 0) {
            if (tensor < SM) { Raw<T, VEC> q; q.v = at[(tensor * NV + k) * THREADS]; return q.get(); }
        }
        return r[tensor - SM][k].get();
    }
};

// A cluster per token tile.  LG lanes of VEC tokens per row, NV rows per thread; x2 takes x's place in the strip.
template <typename T, int VEC, int LG, int NV, int THREADS, int SM>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? (NV <= 8 || VEC == 1 ? 2 : 1) : NV * VEC <= 32 ? 4 : 2)
block_norm_cluster_kernel(T *x2, T *y, const T *x, const T *f, const float *__restrict__ w_post, const float *__restrict__ gate,
                          const float *__restrict__ w_pre, BnShape sh, int rows) {
    constexpr int R = THREADS / LG, TW = LG * VEC;
    extern __shared__ __align__(16) uint4 strips[];
    __shared__ __align__(16) float red[2][THREADS / 32 * TW], mine[2][TW], tot[TW];
    const int tile = blockIdx.x / bn_size(), c0 = (int)bn_rank() * rows, c = c0 + threadIdx.x / LG;
    const int end = c0 + rows < sh.C ? c0 + rows : sh.C;
    const int b = tile / sh.tiles_per_seq, t = (tile - b * sh.tiles_per_seq) * TW + (int)(threadIdx.x % LG) * VEC;
    const int n = t >= sh.S || c >= end ? 0 : (end - c + R - 1) / R;      // rows c, c + R, ... of this thread
    const size_t base = ((size_t)b * sh.C + c) * sh.S + t, step = (size_t)R * sh.S;
    const BnRms<TW> rms = {1.0f / (float)sh.C, sh.eps};
    BnStrip<T, VEC, 2, SM, NV, THREADS> strip(strips);    // x, f
    if (gate) gate += (size_t)b * sh.gate_stride;
    dep_sync();
#pragma unroll
    for (int k = 0; k < NV; k++) if (k < n) strip.fill(1, k, f + base + k * step);
#pragma unroll
    for (int k = 0; k < NV; k++) if (k < n) strip.fill(0, k, x + base + k * step);
    strip.done();
    V<VEC> ss[1] = {V<VEC>::splat(0.0f)}, r = V<VEC>::splat(1.0f);
    if (w_post) {
#pragma unroll
        for (int k = 0; k < NV; k++) if (k < n) { const V<VEC> v = strip.get(1, k); ss[0] = vfma(v, v, ss[0]); }
        bn_cluster_sums<1, VEC, LG, THREADS>(ss, red[0], mine[0], tot, rms);
        r = ss[0];
        ss[0] = V<VEC>::splat(0.0f);
    }
    Raw<T, VEC> z[NV];                                    // x2 as it is stored
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (k < n) {
            const float k1 = sh.alpha * (gate ? __ldg(gate + c + k * R) : 1.0f) * (w_post ? __ldg(w_post + c + k * R) : 1.0f);
            z[k].put(vfma_s(vmul(strip.get(1, k), r), k1, strip.get(0, k)));
            const V<VEC> v = z[k].get();
            ss[0] = vfma(v, v, ss[0]);
        }
    bn_cluster_sums<1, VEC, LG, THREADS>(ss, red[1], mine[1], tot, rms);
    bn_cluster_leave();                                   // this block has read its peers' sums
    // both results only now: a store before the exchange would have to land before its barrier opens
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (k < n) {
            z[k].store_stream(x2 + base + k * step);
            z[k].put(vscale(vmul(z[k].get(), ss[0]), __ldg(w_pre + c + k * R)));
            z[k].store_stream(y + base + k * step);
        }
    bn_cluster_wait();                                    // no block leaves while a peer may still read its sums
}

template <typename T, int VEC, int LG, int NV, int THREADS, int SM>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 1 : VEC == 1 ? 2 : NV <= 4 ? 3 : 1)
block_norm_bwd_cluster_kernel(T *dx, T *df, float *__restrict__ partial, const T *dy, const T *dx2, const T *x2, const T *f,
                              const float *__restrict__ w_post, const float *__restrict__ gate, const float *__restrict__ w_pre, BnShape sh, int rows) {
    constexpr int R = THREADS / LG, TW = LG * VEC;
    extern __shared__ __align__(16) uint4 strips[];
    __shared__ __align__(16) float red[3 * (THREADS / 32) * TW], mine[6 * TW], tot[6 * TW];
    const int tile = blockIdx.x / bn_size(), c0 = (int)bn_rank() * rows, c = c0 + threadIdx.x / LG;
    const int end = c0 + rows < sh.C ? c0 + rows : sh.C, lg = threadIdx.x % LG;
    const int b = tile / sh.tiles_per_seq, t = (tile - b * sh.tiles_per_seq) * TW + lg * VEC;
    const int n = t >= sh.S || c >= end ? 0 : (end - c + R - 1) / R;
    const size_t base = ((size_t)b * sh.C + c) * sh.S + t, step = (size_t)R * sh.S;
    const bool want_p = w_post || gate;
    const BnBwd<TW> factors = {1.0f / (float)sh.C, sh.eps, sh.alpha, w_post != nullptr};
    BnStrip<T, VEC, 4, SM, NV, THREADS> strip(strips);    // x2, dy, f, dx2
    if (gate) gate += (size_t)b * sh.gate_stride;
    dep_sync();
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (k < n) {
            const size_t i = base + k * step;
            if (dx2) strip.fill(3, k, dx2 + i); else strip.zero(3, k);
            strip.fill(0, k, x2 + i);
            strip.fill(1, k, dy + i);
            strip.fill(2, k, f + i);
        }
    float k1[NV], k2[NV];                                 // gate * w_post, w_pre
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (k < n) {
            k1[k] = (gate ? __ldg(gate + c + k * R) : 1.0f) * (w_post ? __ldg(w_post + c + k * R) : 1.0f);
            k2[k] = __ldg(w_pre + c + k * R);
        }
    strip.done();
    V<VEC> s[6];
#pragma unroll
    for (int i = 0; i < 6; i++) s[i] = V<VEC>::splat(0.0f);
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (k < n) {
            const V<VEC> vx = strip.get(0, k), va = vscale(strip.get(1, k), k2[k]);
            s[0] = vfma(vx, vx, s[0]);
            s[1] = vfma(va, vx, s[1]);
            if (w_post) {
                const V<VEC> vf = strip.get(2, k), vq = vscale(vf, k1[k]);
                s[2] = vfma(vf, vf, s[2]);
                s[3] = vfma(vq, strip.get(3, k), s[3]);
                s[4] = vfma(vq, va, s[4]);
                s[5] = vfma(vq, vx, s[5]);
            }
        }
    bn_cluster_sums<6, VEC, LG, THREADS>(s, red, mine, tot, factors);
    bn_cluster_leave();
    const V<VEC> r2 = s[0], nk = s[1], rms_f = s[2], nj = s[3];
    float sums[2 * NV];                                   // per row: dy x2 r2, f r_f G, over the thread's tokens
#pragma unroll
    for (int k = 0; k < NV; k++) {
        sums[2 * k] = sums[2 * k + 1] = 0.0f;
        if (k < n) {
            const V<VEC> vx = strip.get(0, k), vy = strip.get(1, k), vf = strip.get(2, k);
            const V<VEC> G = vfma(vscale(vy, k2[k]), r2, vfma(nk, vx, strip.get(3, k)));
            sums[2 * k] = vmul(vy, vmul(vx, r2)).hsum();
            sums[2 * k + 1] = vmul(vmul(vf, rms_f), G).hsum();
            Raw<T, VEC> out;
            out.put(G);
            out.store_stream(dx + base + k * step);
            out.put(vfma(vscale(G, sh.alpha * k1[k]), rms_f, vmul(nj, vf)));
            out.store_stream(df + base + k * step);
        }
    }
    // over the lanes of a row: each step exchanges halves, a lane ends with HELD of the sums, the first of them `first`
    constexpr int HELD = 2 * NV / LG;
    static_assert(HELD >= 1, "every step halves");
    int first = 0;
#pragma unroll
    for (int off = LG / 2, left = NV; off > 0; off >>= 1, left >>= 1) {
        const bool up = lg & off;
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (i < left) {
                const float other = __shfl_xor_sync(0xffffffffu, up ? sums[i] : sums[i + left], off);
                sums[i] = (up ? sums[i + left] : sums[i]) + other;
            }
        first += up ? left : 0;
    }
    float *prow = partial + (size_t)tile * sh.C * 2;
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const int ch = c + (first + i) / 2 * R, p = (first + i) & 1;
        if (ch < end && (p == 0 || want_p)) prow[2 * (size_t)ch + p] = sums[i];
    }
    bn_cluster_wait();
}

}  // namespace ane
#include "block_norm_ring.cuh"
namespace ane {

// ------------------------------------------------------------------ parameter gradients
// Sums of the rows of partials [row][C] of one group, in a fixed order: 32 channels x 8 slices of rows per block.  The sums
// stay in `sums` [group][C] for the kernel below; where a group is a sequence with a gate of its own, its dgate is finished
// here.  Rows of a group are consecutive; the last group may be shorter.
__global__ void __launch_bounds__(256)
block_norm_grad_kernel(const float2 *__restrict__ partial, long long all_rows, int rows, float2 *__restrict__ sums, float *__restrict__ dgate,
                       const float *__restrict__ w_post, int C, float alpha) {
    __shared__ float2 acc[8][32];
    dep_sync();
    const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cl;
    const size_t group = blockIdx.y;
    const long long left = all_rows - (long long)group * rows;
    const int have = left < rows ? (int)left : rows, per = (have + 7) / 8;
    const int r0 = sl * per, r1 = r0 + per < have ? r0 + per : have;
    const float2 *p = partial + group * rows * C;
    float2 s = make_float2(0.0f, 0.0f);
    if (c < C) {
        int r = r0;
        for (; r + 4 <= r1; r += 4) {
            float2 v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) v[u] = p[(size_t)(r + u) * C + c];
#pragma unroll
            for (int u = 0; u < 4; u++) { s.x += v[u].x; s.y += v[u].y; }
        }
        for (; r < r1; r++) { const float2 v = p[(size_t)r * C + c]; s.x += v.x; s.y += v.y; }
    }
    acc[sl][cl] = s;
    __syncthreads();
    if (sl != 0 || c >= C) return;
    s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 8; i++) { s.x += acc[i][cl].x; s.y += acc[i][cl].y; }
    s.y *= alpha;
    if (dgate) dgate[group * C + c] += w_post ? w_post[c] * s.y : s.y;
    sums[group * C + c] = s;
}

// The groups' sums, in order, into the parameter gradients.  A gate per sequence weighs each group's share of dw_post.
__global__ void __launch_bounds__(256)
block_norm_grad_join_kernel(const float2 *__restrict__ sums, int groups, float *__restrict__ dw_post, float *__restrict__ dgate, float *__restrict__ dw_pre,
                            const float *__restrict__ w_post, const float *__restrict__ gate, int gate_stride, int C) {
    __shared__ float2 acc[8][32];
    dep_sync();
    const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cl;
    const int per = (groups + 7) / 8;
    const int g0 = sl * per, g1 = g0 + per < groups ? g0 + per : groups;
    float2 s = make_float2(0.0f, 0.0f);
    if (c < C)
#pragma unroll 4
        for (int g = g0; g < g1; g++) {
            const float2 v = sums[(size_t)g * C + c];
            s.x += v.x;
            s.y += gate_stride ? v.y * gate[(size_t)g * gate_stride + c] : v.y;
        }
    acc[sl][cl] = s;
    __syncthreads();
    if (sl != 0 || c >= C) return;
    s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 8; i++) { s.x += acc[i][cl].x; s.y += acc[i][cl].y; }
    if (dw_pre) dw_pre[c] += s.x;
    if (dw_post) dw_post[c] += gate && !gate_stride ? gate[c] * s.y : s.y;
    if (dgate && !gate_stride) dgate[c] += w_post ? w_post[c] * s.y : s.y;
}

// Blocks of a cluster and channels of each; 0 blocks: no cluster form for this many channels.
struct BnSplit { int blocks, rows; };
static BnSplit bn_split(int C, int rows_most) {
    const int blocks = (C + rows_most - 1) / rows_most;
    if (blocks > 8) return {0, 0};
    return {blocks, (C + blocks - 1) / blocks};
}
template <typename... KArgs, typename... Args>
static inline void bn_call(void (*kernel)(KArgs...), dim3 grid, int threads, int cluster, size_t smem, cudaStream_t st, Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3((unsigned)threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = cluster ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);      // the error, if any, is picked up by ANE_LAUNCH_OK
}
// Clusters of `blocks` blocks that the device holds at once.
template <typename... KArgs> static int bn_resident(void (*kernel)(KArgs...), int threads, int blocks, size_t smem) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(blocks * ctx().sm_count)); cfg.blockDim = dim3((unsigned)threads); cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)blocks; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.attrs = &at; cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) { cudaGetLastError(); n = ctx().sm_count / (2 * blocks); }
    return n < 1 ? 1 : n;
}
// The pipelined backward form: up to eight blocks of 128 channels, and at least four tiles for every SM's block to walk (with
// fewer the pipeline is mostly filling and draining).
static bool bn_ring(int C, const BnSplit &sp, long long tiles) {
    return sp.blocks && C % 128 == 0 && (tuning("block_norm_cluster", 7) & 4) && tiles * sp.blocks >= 4LL * ctx().sm_count;
}
// The cluster form for a shape, if there is one.
//   many tiles   512 threads per block; 1024 channels to a block (forward 115 us against 138, backward 245 against 250, see above)
//   few tiles    256 threads, up to eight blocks per tile, so that more SMs take part (5 us for 256 tokens x 768 channels)
//   rows that break 16-byte alignment: element by element, 32 tokens per row, up to eight blocks per tile; blocks of 512 threads
//                above 1024 channels (8 x 2048 x 1001 in fp16: forward 105 us against 223 in sweeps, backward 186 against 490)
// -> BN_NONE: none (channels beyond eight blocks, or unaligned sequences so short that most lanes of a row would idle).
constexpr int BN_NONE = 1;
template <int V_, int LG_, int NV_, int TH_> struct BnForm { static constexpr int VEC = V_, LG = LG_, NV = NV_, THREADS = TH_; };
// BIG_LG: lanes per row of the large form (a thread has C / (512 / BIG_LG) rows); BIG_C: channels above which it is used.
template <typename T, bool FORWARD, typename Fn> static int bn_pick_cluster(bool vec, int B, int C, int S, Fn &&go) {
    constexpr int N = Elt<T>::VEC, BIG_LG = 4, BIG_C = FORWARD ? 0 : 512, BR = 512 / BIG_LG;
    const int knob = tuning("block_norm_cluster", 7);    // bits: 1 small form, 2 large form, 4 backward ring; 0: none
    if (!(knob & 3)) return BN_NONE;
    const long long big_tiles = (long long)B * ((S + BIG_LG * N - 1) / (BIG_LG * N));
    if (vec && C > BIG_C && C <= 4096 && (knob & 2) && big_tiles * ((C + 1023) / 1024) >= 2LL * ctx().sm_count) {
        if constexpr (BIG_C < 512) {
            if (C <= 256) return go(BnForm<N, BIG_LG, 256 / BR, 512>(), bn_split(C, 256));
            if (C <= 512) return go(BnForm<N, BIG_LG, 512 / BR, 512>(), bn_split(C, 512));
        }
        return go(BnForm<N, BIG_LG, 1024 / BR, 512>(), bn_split(C, 1024));
    }
    if (vec && C <= 1024) return go(BnForm<N, 8, 4, 256>(), bn_split(C, 256 / 8 * 4));
    if (vec && C <= 2048) return go(BnForm<N, 4, 4, 256>(), bn_split(C, 256 / 4 * 4));
    if (vec && C <= 4096) return go(BnForm<N, 4, 8, 256>(), bn_split(C, 256 / 4 * 8));
    if (!vec && S >= 16 && C <= 2048) {
        // forward, few channels, many tiles: the sweeps find their tile in L1 (333 x 64 x 1001 in fp16 88 us against 122, 40 channels
        // 14 against 22; in fp32 124 against 130)
        if (FORWARD && C <= 512 && (long long)B * ((S + 31) / 32) >= 8LL * ctx().sm_count) return BN_NONE;
        if (C <= 1024) return go(BnForm<1, 32, 16, 256>(), bn_split(C, 256 / 32 * 16));
        return go(BnForm<1, 32, 16, 512>(), bn_split(C, 512 / 32 * 16));
    }
    return BN_NONE;
}
// Blocks with more than the default shared memory ask for it once.
template <typename... KArgs> static int bn_allow(void (*kernel)(KArgs...), size_t smem, bool &ready) {
    if (!ready && smem) ANE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    ready = true;
    return ANE_CUDA_OK;
}

// LG lanes of VEC tokens per row of a tile for the kernels above.
template <typename T, typename Fn> static int bn_pick(bool vec, int S, Fn &&go) {
    if (vec) return go(std::integral_constant<int, Elt<T>::VEC>(), std::integral_constant<int, 8>());
    if (S >= 16) return go(std::integral_constant<int, 1>(), std::integral_constant<int, 32>());
    if (S >= 3) return go(std::integral_constant<int, 1>(), std::integral_constant<int, 4>());
    return go(std::integral_constant<int, 1>(), std::integral_constant<int, 1>());
}

}  // namespace ane

using namespace ane;

extern "C" {

int ane_cuda_block_norm_dev(void *stream, ane_dtype dtype, int B, int C, int S, void *x2, void *y, const void *x, const void *f, const float *w_post,
                            const float *gate, int gate_per_seq, const float *w_pre, float alpha, float eps) {
    ANE_REQUIRE_INIT();
    ANE_REQUIRE(x2 && y && x && f && w_pre, "%s: null pointer", __func__);
    ANE_REQUIRE(dtype_ok(dtype), "%s: bad dtype %d", __func__, (int)dtype);
    ANE_REQUIRE(B >= 1 && C >= 1 && S >= 1, "%s: bad shape B=%d C=%d S=%d", __func__, B, C, S);
    ANE_REQUIRE(gate_per_seq == 0 || (gate_per_seq == 1 && gate), "%s: gate_per_seq is 0, or 1 with a gate", __func__);
    ANE_REQUIRE(y != x2 && y != x && y != f && x2 != f, "%s: only x2 may be x", __func__);
    ANE_REQUIRE((long long)B * S < 0x7fffffffLL, "%s: too many tokens", __func__);
    const size_t bytes = (size_t)B * C * S * dtype_size(dtype);
    ANE_CHECK_EXTENT(x2, bytes); ANE_CHECK_EXTENT(y, bytes); ANE_CHECK_EXTENT(x, bytes); ANE_CHECK_EXTENT(f, bytes);
    ANE_CHECK_EXTENT(w_post, (size_t)C * 4); ANE_CHECK_EXTENT(w_pre, (size_t)C * 4); ANE_CHECK_EXTENT(gate, (size_t)(gate_per_seq ? B : 1) * C * 4);
    cudaStream_t st = (cudaStream_t)stream;
    BnShape sh = {B, C, S, 0, 0, gate_per_seq ? C : 0, alpha, eps};
    ANE_DISPATCH_DTYPE(dtype, T, {
        const bool vec = S % Elt<T>::VEC == 0 && aligned16(x2) && aligned16(y) && aligned16(x) && aligned16(f);
        const int rc = bn_pick_cluster<T, true>(vec, B, C, S, [&](auto form, BnSplit sp) -> int {
            using F = decltype(form);
            constexpr int SM = F::VEC == 1 ? 0 : F::THREADS == 512 ? 1 : 2;      // 512 threads: x in shared memory, f in registers
            constexpr size_t smem = BnStrip<T, F::VEC, 2, SM, F::NV, F::THREADS>::BYTES;
            static bool ready = false;
            const auto kernel = block_norm_cluster_kernel<T, F::VEC, F::LG, F::NV, F::THREADS, SM>;
            if (int e = bn_allow(kernel, smem, ready)) return e;
            sh.tiles_per_seq = (S + F::LG * F::VEC - 1) / (F::LG * F::VEC);
            bn_call(kernel, dim3((unsigned)B * (unsigned)sh.tiles_per_seq * (unsigned)sp.blocks), F::THREADS, sp.blocks, smem, st, (T *)x2, (T *)y, (const T *)x, (const T *)f, w_post, gate,
                    w_pre, sh, sp.rows);
            return ANE_CUDA_OK;
        });
        if (rc == ANE_CUDA_OK) { ANE_LAUNCH_OK(1); return ANE_CUDA_OK; }
        if (rc != BN_NONE) return rc;
        bn_pick<T>(vec, S, [&](auto v, auto lg) {
            constexpr int VEC = decltype(v)::value, LG = decltype(lg)::value;
            sh.tiles_per_seq = (S + VEC * LG - 1) / (VEC * LG);
            block_norm_kernel<T, VEC, LG><<<(unsigned)B * (unsigned)sh.tiles_per_seq, BN_THREADS, 0, st>>>((T *)x2, (T *)y, (const T *)x, (const T *)f, w_post, gate, w_pre, sh);
            return 0;
        });
    });
    ANE_LAUNCH_OK(1);
    return ANE_CUDA_OK;
}

int ane_cuda_block_norm_bwd_dev(void *stream, ane_dtype dtype, int B, int C, int S, void *dx, void *df, float *dw_post, float *dgate, float *dw_pre,
                                const void *dy, const void *dx2, const void *x2, const void *f, const float *w_post, const float *gate, int gate_per_seq,
                                const float *w_pre, float alpha, float eps) {
    ANE_REQUIRE_INIT();
    ANE_REQUIRE(dx && df && dy && x2 && f && w_pre, "%s: null pointer", __func__);
    ANE_REQUIRE(dtype_ok(dtype), "%s: bad dtype %d", __func__, (int)dtype);
    ANE_REQUIRE(B >= 1 && C >= 1 && S >= 1, "%s: bad shape B=%d C=%d S=%d", __func__, B, C, S);
    ANE_REQUIRE(gate_per_seq == 0 || (gate_per_seq == 1 && gate), "%s: gate_per_seq is 0, or 1 with a gate", __func__);
    ANE_REQUIRE((!dw_post || w_post) && (!dgate || gate), "%s: a gradient is asked for a weight or gate that is not given", __func__);
    ANE_REQUIRE(dx != df && dx != f && dx != x2 && dx != dy && df != x2 && df != dy && df != dx2, "%s: only dx may be dx2, and df may be f", __func__);
    ANE_REQUIRE((long long)B * S < 0x7fffffffLL, "%s: too many tokens", __func__);
    const size_t bytes = (size_t)B * C * S * dtype_size(dtype), gb = (size_t)(gate_per_seq ? B : 1) * C * 4;
    ANE_CHECK_EXTENT(dx, bytes); ANE_CHECK_EXTENT(df, bytes); ANE_CHECK_EXTENT(dy, bytes); ANE_CHECK_EXTENT(dx2, bytes); ANE_CHECK_EXTENT(x2, bytes);
    ANE_CHECK_EXTENT(f, bytes); ANE_CHECK_EXTENT(w_post, (size_t)C * 4); ANE_CHECK_EXTENT(w_pre, (size_t)C * 4); ANE_CHECK_EXTENT(dw_post, (size_t)C * 4);
    ANE_CHECK_EXTENT(dw_pre, (size_t)C * 4); ANE_CHECK_EXTENT(gate, gb); ANE_CHECK_EXTENT(dgate, gb);
    cudaStream_t st = (cudaStream_t)stream;
    BnShape sh = {B, C, S, 0, 0, gate_per_seq ? C : 0, alpha, eps};
    float2 *partial = nullptr, *sums = nullptr;
    long long all_rows = 0;          // of partial sums, and how many make a group
    int rows = 1, groups = 1;
    // Scratch for the partial rows and the groups' sums.  A group is a sequence where the gate is per sequence, else 64 rows.
    auto scratch = [&](long long n, int per_seq) -> int {
        all_rows = n;
        rows = per_seq ? per_seq : 64;
        groups = (int)((n + rows - 1) / rows);
        const size_t pbytes = round_up((size_t)n * C * sizeof(float2), 256);
        char *ws = static_cast<char *>(workspace(pbytes + (size_t)groups * C * sizeof(float2)));
        if (!ws) return fail(ANE_CUDA_ERR_NOMEM, "ane_cuda_block_norm_bwd_dev: no scratch");
        partial = reinterpret_cast<float2 *>(ws);
        sums = reinterpret_cast<float2 *>(ws + pbytes);
        return ANE_CUDA_OK;
    };
    ANE_DISPATCH_DTYPE(dtype, T, {
        const bool vec = S % Elt<T>::VEC == 0 && aligned16(dx) && aligned16(df) && aligned16(dy) && aligned16(dx2) && aligned16(x2) && aligned16(f);
        int rc = BN_NONE;
        constexpr int RTW = 32 * BrWord<T>::W;
        const BnSplit rsp = bn_split(C, BR_ROWS);
        const long long rtiles = (long long)B * ((S + RTW - 1) / RTW);
        if (vec && bn_ring(C, rsp, rtiles)) {
            BrMaps maps;
            const void *from[4] = {x2, dy, f, dx2};
            for (int i = 0; i < (dx2 ? 4 : 3); i++)
                if (int e = make_bcs_tensor_map(&maps.t[i], dtype, from[i], B, C, S, RTW, BR_ROWS)) return e;
            sh.tiles_per_seq = (S + RTW - 1) / RTW;
            if (int e = scratch(rtiles, gate_per_seq ? sh.tiles_per_seq : 0)) return e;
            auto go = [&](auto post, auto has) -> int {
                const auto kernel = block_norm_bwd_ring_kernel<T, decltype(post)::value, decltype(has)::value>;
                static int fit[9] = {};
                if (!fit[rsp.blocks]) {
                    ANE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)BR_SMEM));
                    fit[rsp.blocks] = bn_resident(kernel, BR_THREADS, rsp.blocks, BR_SMEM);
                }
                const int clusters = rtiles < fit[rsp.blocks] ? (int)rtiles : fit[rsp.blocks];
                bn_call(kernel, dim3((unsigned)(clusters * rsp.blocks)), BR_THREADS, rsp.blocks, BR_SMEM, st, maps, (T *)dx, (T *)df, reinterpret_cast<float *>(partial), w_post, gate, w_pre,
                        sh, (int)rtiles, ctx().status);
                return ANE_CUDA_OK;
            };
            rc = w_post ? (dx2 ? go(std::true_type(), std::true_type()) : go(std::true_type(), std::false_type()))
                        : (dx2 ? go(std::false_type(), std::true_type()) : go(std::false_type(), std::false_type()));
            if (rc != ANE_CUDA_OK) return rc;
        }
        if (rc == BN_NONE) rc = bn_pick_cluster<T, false>(vec, B, C, S, [&](auto form, BnSplit sp) -> int {
            using F = decltype(form);
            constexpr int SM = F::VEC == 1 ? 0 : F::THREADS == 512 ? 3 : 4;      // 512 threads: dx2 in registers
            constexpr size_t smem = BnStrip<T, F::VEC, 4, SM, F::NV, F::THREADS>::BYTES;
            static bool ready = false;
            const auto kernel = block_norm_bwd_cluster_kernel<T, F::VEC, F::LG, F::NV, F::THREADS, SM>;
            if (int e = bn_allow(kernel, smem, ready)) return e;
            sh.tiles_per_seq = (S + F::LG * F::VEC - 1) / (F::LG * F::VEC);
            if (int e = scratch((long long)B * sh.tiles_per_seq, gate_per_seq ? sh.tiles_per_seq : 0)) return e;
            bn_call(kernel, dim3((unsigned)B * (unsigned)sh.tiles_per_seq * (unsigned)sp.blocks), F::THREADS, sp.blocks, smem, st, (T *)dx, (T *)df, reinterpret_cast<float *>(partial),
                    (const T *)dy, (const T *)dx2, (const T *)x2, (const T *)f, w_post, gate, w_pre, sh, sp.rows);
            return ANE_CUDA_OK;
        });
        if (rc == BN_NONE) {
            rc = bn_pick<T>(vec, S, [&](auto v, auto lg) -> int {
                constexpr int VEC = decltype(v)::value, LG = decltype(lg)::value;
                sh.tiles_per_seq = (S + VEC * LG - 1) / (VEC * LG);
                // up to eight blocks per SM, each with a row of partial sums
                const long long most = 8LL * ctx().sm_count, tiles = (long long)B * sh.tiles_per_seq, want = (most + B - 1) / B;
                sh.rows_per_seq = !gate_per_seq ? 0 : (int)(want < sh.tiles_per_seq ? want : sh.tiles_per_seq);
                const long long blocks = gate_per_seq ? (long long)B * sh.rows_per_seq : tiles < most ? tiles : most;
                if (int e = scratch(blocks, sh.rows_per_seq)) return e;
                block_norm_bwd_kernel<T, VEC, LG><<<(unsigned)blocks, BN_THREADS, 0, st>>>((T *)dx, (T *)df, reinterpret_cast<float *>(partial), (const T *)dy, (const T *)dx2,
                                                                                         (const T *)x2, (const T *)f, w_post, gate, w_pre, sh);
                return ANE_CUDA_OK;
            });
        }
        if (rc != ANE_CUDA_OK) return rc;
    });
    ANE_LAUNCH_OK(1);
    if (dw_pre || dw_post || dgate) {
        // gridDim.y holds 65535 groups: more than that take further launches
        for (int g0 = 0; g0 < groups; g0 += 65535) {
            const int n = groups - g0 < 65535 ? groups - g0 : 65535;
            bn_call(block_norm_grad_kernel, dim3((C + 31) / 32, n), 256, 0, 0, st, partial + (size_t)g0 * rows * C, all_rows - (long long)g0 * rows, rows, sums + (size_t)g0 * C,
                    gate_per_seq && dgate ? dgate + (size_t)g0 * C : nullptr, w_post, C, alpha);
            ANE_LAUNCH_OK(1);
        }
        if (dw_pre || dw_post || (dgate && !gate_per_seq)) {
            bn_call(block_norm_grad_join_kernel, dim3((C + 31) / 32), 256, 0, 0, st, sums, groups, dw_post, dgate, dw_pre, w_post, gate, sh.gate_stride, C);
            ANE_LAUNCH_OK(1);
        }
    }
    return ANE_CUDA_OK;
}

}  // extern "C"
