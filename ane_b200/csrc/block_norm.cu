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
// Both directions move each tensor once at best (4 and 6 tensor passes) and do a few operations per element: HBM-bound.
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

// NS per-token sums over the block: each warp's total goes to shared memory, the warps are added in order.  `red` holds
// [NS][warps][TW] floats, `tot` [NS][TW].  Ends with the totals in registers and the arrays free for reuse.
template <int NS, int N, int LG> __device__ __forceinline__ void bn_block_sums(V<N> (&v)[NS], float *red, float *tot) {
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
#pragma unroll
    for (int s = 0; s < NS; s++) v[s] = lanes_from_smem<N>(tot + s * TW + lg * N);
}

template <int N> __device__ __forceinline__ V<N> bn_rms(const V<N> &sumsq, float inv_c, float eps) {
    V<N> r;
#pragma unroll
    for (int j = 0; j < N; j++) r.set(j, 1.0f / sqrtf(fmaf(sumsq.get(j), inv_c, eps)));
    return r;
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
        bn_block_sums<1, VEC, LG>(ss, red, tot);
        rf = bn_rms(ss[0], inv_c, sh.eps);
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
    bn_block_sums<1, VEC, LG>(ss, red, tot);
    const V<VEC> r2 = bn_rms(ss[0], inv_c, sh.eps);
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

// The six per-token sums of the backward pass -> the five per-token factors of the sweep that writes.
template <int N> struct BnFactors { V<N> r2, k, rf, j; };
template <int N> __device__ __forceinline__ BnFactors<N> bn_factors(const V<N> (&s)[6], bool post, float inv_c, float alpha, float eps) {
    BnFactors<N> o;
    o.r2 = bn_rms(s[0], inv_c, eps);
    o.rf = post ? bn_rms(s[2], inv_c, eps) : V<N>::splat(1.0f);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float r2 = o.r2.get(i), rf = o.rf.get(i);
        const float k = r2 * r2 * r2 * (s[1].get(i) * inv_c);
        o.k.set(i, k);
        o.j.set(i, post ? alpha * rf * rf * rf * (inv_c * (s[3].get(i) + r2 * s[4].get(i) - k * s[5].get(i))) : 0.0f);
    }
    return o;
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
        bn_block_sums<6, VEC, LG>(s, red, tot);
        const BnFactors<VEC> o = bn_factors<VEC>(s, w_post != nullptr, inv_c, sh.alpha, sh.eps);
        const V<VEC> nk = vscale(o.k, -1.0f), nj = vscale(o.j, -1.0f);
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
                const V<VEC> z = vmul(vx, o.r2);
                V<VEC> G = vfma(vscale(vy, __ldg(w_pre + c)), o.r2, vmul(nk, vx));
                if (dx2) G = vadd(G, rd.get());
                sum_q = vmul(vy, z).hsum();
                const float gw = (g ? __ldg(g + c) : 1.0f) * (w_post ? __ldg(w_post + c) : 1.0f);
                const V<VEC> u = vmul(vf, o.rf);
                sum_p = vmul(u, G).hsum();
                rx.put(G);
                rx.store(dx + at);
                rf.put(vfma(vscale(G, sh.alpha * gw), o.rf, vmul(nj, vf)));
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

// Sums of the rows of partials of one group (a sequence, or everything), in a fixed order: 32 channels x 8 slices of rows per
// block.  One group: the gradients are added to their buffers.  Several (gate per sequence): the sums stay in `sums`
// [group][2][C] for the kernel below, and dgate of the sequence is finished here.
__global__ void __launch_bounds__(256)
block_norm_grad_kernel(const float *__restrict__ partial, int rows, float *__restrict__ sums, float *__restrict__ dw_post, float *__restrict__ dgate,
                       float *__restrict__ dw_pre, const float *__restrict__ w_post, const float *__restrict__ gate, int C, float alpha) {
    __shared__ float2 acc[8][32];
    const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cl, group = blockIdx.y;
    const int per = (rows + 7) / 8;
    const int r0 = sl * per, r1 = r0 + per < rows ? r0 + per : rows;
    const float2 *p = reinterpret_cast<const float2 *>(partial) + (size_t)group * rows * C;
    float2 s = make_float2(0.0f, 0.0f);
    if (c < C) {
        int r = r0;
        for (; r + 8 <= r1; r += 8) {
            float2 v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] = p[(size_t)(r + u) * C + c];
#pragma unroll
            for (int u = 0; u < 8; u++) { s.x += v[u].x; s.y += v[u].y; }
        }
        for (; r < r1; r++) { const float2 v = p[(size_t)r * C + c]; s.x += v.x; s.y += v.y; }
    }
    acc[sl][cl] = s;
    __syncthreads();
    if (sl != 0 || c >= C) return;
    float q = 0.0f, a = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) { q += acc[i][cl].x; a += acc[i][cl].y; }
    a *= alpha;
    if (dgate) dgate[(sums ? (size_t)group * C : 0) + c] += w_post ? w_post[c] * a : a;
    if (sums) {
        sums[((size_t)group * 2) * C + c] = q;
        sums[((size_t)group * 2 + 1) * C + c] = a * gate[(size_t)group * C + c];
    } else {
        if (dw_pre) dw_pre[c] += q;
        if (dw_post) dw_post[c] += gate ? gate[c] * a : a;
    }
}

__global__ void __launch_bounds__(256)
block_norm_grad_join_kernel(const float *__restrict__ sums, int groups, float *__restrict__ dw_post, float *__restrict__ dw_pre, int C) {
    __shared__ float2 acc[8][32];
    const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cl;
    const int per = (groups + 7) / 8;
    const int g0 = sl * per, g1 = g0 + per < groups ? g0 + per : groups;
    float2 s = make_float2(0.0f, 0.0f);
    if (c < C)
#pragma unroll 4
        for (int g = g0; g < g1; g++) { s.x += sums[((size_t)g * 2) * C + c]; s.y += sums[((size_t)g * 2 + 1) * C + c]; }
    acc[sl][cl] = s;
    __syncthreads();
    if (sl != 0 || c >= C) return;
    float q = 0.0f, a = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) { q += acc[i][cl].x; a += acc[i][cl].y; }
    if (dw_pre) dw_pre[c] += q;
    if (dw_post) dw_post[c] += a;
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
    const int groups = gate_per_seq ? B : 1;
    int rows = 1;
    float *partial = nullptr, *sums = nullptr;
    ANE_DISPATCH_DTYPE(dtype, T, {
        const bool vec = S % Elt<T>::VEC == 0 && aligned16(dx) && aligned16(df) && aligned16(dy) && aligned16(dx2) && aligned16(x2) && aligned16(f);
        const int rc = bn_pick<T>(vec, S, [&](auto v, auto lg) {
            constexpr int VEC = decltype(v)::value, LG = decltype(lg)::value;
            sh.tiles_per_seq = (S + VEC * LG - 1) / (VEC * LG);
            // up to eight blocks per SM, each with a row of partial sums
            const long long most = 8LL * ctx().sm_count;
            if (gate_per_seq) {
                const long long want = (most + B - 1) / B;
                rows = sh.rows_per_seq = (int)(want < sh.tiles_per_seq ? want : sh.tiles_per_seq);
            } else {
                const long long tiles = (long long)B * sh.tiles_per_seq;
                rows = (int)(tiles < most ? tiles : most);
            }
            const size_t blocks = (size_t)rows * groups;
            const size_t pbytes = round_up(blocks * 2 * C * sizeof(float), 256);
            char *ws = static_cast<char *>(workspace(pbytes + (gate_per_seq ? (size_t)B * 2 * C * sizeof(float) : 0)));
            if (!ws) return fail(ANE_CUDA_ERR_NOMEM, "ane_cuda_block_norm_bwd_dev: no scratch");
            partial = reinterpret_cast<float *>(ws);
            sums = gate_per_seq ? reinterpret_cast<float *>(ws + pbytes) : nullptr;
            block_norm_bwd_kernel<T, VEC, LG><<<(unsigned)blocks, BN_THREADS, 0, st>>>((T *)dx, (T *)df, partial, (const T *)dy, (const T *)dx2, (const T *)x2,
                                                                                     (const T *)f, w_post, gate, w_pre, sh);
            return (int)ANE_CUDA_OK;
        });
        if (rc != ANE_CUDA_OK) return rc;
    });
    ANE_LAUNCH_OK(1);
    if (dw_pre || dw_post || dgate) {
        // gridDim.y holds 65535 groups: more sequences than that take further launches
        for (int g0 = 0; g0 < groups; g0 += 65535) {
            const int n = groups - g0 < 65535 ? groups - g0 : 65535;
            block_norm_grad_kernel<<<dim3((C + 31) / 32, n), 256, 0, st>>>(partial + (size_t)g0 * rows * 2 * C, rows, sums ? sums + (size_t)g0 * 2 * C : nullptr, dw_post,
                                                                          dgate ? dgate + (size_t)g0 * C : nullptr, dw_pre, w_post, gate ? gate + (size_t)g0 * C : nullptr, C, alpha);
            ANE_LAUNCH_OK(1);
        }
        if (sums && (dw_pre || dw_post)) {
            block_norm_grad_join_kernel<<<(C + 31) / 32, 256, 0, st>>>(sums, groups, dw_post, dw_pre, C);
            ANE_LAUNCH_OK(1);
        }
    }
    return ANE_CUDA_OK;
}

}  // extern "C"
