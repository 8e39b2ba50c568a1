// adam_multi.cu -- one Adam / AdamW step over a list of tensors, with the moments in 32 bits or in 8, and the conversion of
// 8-bit moments to fp32 and back.
//
// The update is the one of ane_cuda_adam_dev (the same IEEE operations in the same order).  An 8-bit moment is a code per
// element and an fp32 scale per 256 elements.  The codes are floats without infinities or NaN:
//   first moment    sign, 4 exponent bits (bias 7), 3 mantissa bits     largest 480
//   second moment         5 exponent bits (bias 15), 3 mantissa bits    largest 122880
// (a second moment spans the square of the range, hence the exponent bit in place of the sign).  With fp32's exponent field
// aligned over the code's, code << 20 read as a float is the value times a power of two, subnormals included, so decoding is
// a shift and two products, and encoding is one addition on the bits: 20 random bits added below the kept mantissa bits,
// then a shift.  That rounds up or down with the probability that keeps the mean.  Rounding to nearest would not do here:
// with beta2 = 0.95 a gradient of zero takes 5 % from v and codes are 6 to 12 % apart, so v would never come down again.
#include "common.cuh"

#include <math.h>
#include <string.h>
#include <vector>
#include <algorithm>

namespace ane {

constexpr int AM_THREADS = 256;
constexpr int AM_GROUP = 256;                     // elements that share a scale: one warp, eight per lane
constexpr int AM_CHUNK = AM_THREADS / 32 * AM_GROUP;   // elements of a block

// One tensor of a launch.  The list travels in the kernel's parameters (no copy to the device to wait for, and a captured
// graph holds it by value).
struct AmItem {
    float *w;
    const void *g;
    void *m, *v;
    float *ms, *vs;
    void *copy;
    size_t n;
    float wd;
    uint32_t key;
    uint32_t first_chunk;
    uint32_t vec;            // every pointer aligned for eight elements at a time
};
template <int CAP> struct AmList {
    int count;
    AmItem it[CAP];
};
struct AmScalars {
    float b1, b2, omb1, omb2, bc1, bc2, ibc1, ibc2, lr, eps, gscale;
    const float *clip;
    unsigned variant;
    int use_gscale, copy_dtype;
};

// The finaliser of MurmurHash3 (public domain, Appleby): every input bit reaches every output bit.
__host__ __device__ __forceinline__ uint32_t am_mix(uint32_t h) {
    h ^= h >> 16; h *= 0x85EBCA6Bu;
    h ^= h >> 13; h *= 0xC2B2AE35u;
    return h ^ (h >> 16);
}
__device__ __forceinline__ uint32_t am_hash(size_t place, uint32_t key) { return am_mix((uint32_t)place * 0x9E3779B1u + key); }

__device__ __forceinline__ float am_sqrt(float x) {
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool SECOND> struct Code8;
template <> struct Code8<false> {
    static constexpr float TOP = 480.0f;
    __device__ __forceinline__ static float decode(uint32_t c, float scale) {
        const float v = __fmul_rn(__fmul_rn(__uint_as_float((c & 127u) << 20), 0x1p120f), scale);
        return c & 128u ? -v : v;
    }
    __device__ __forceinline__ static uint32_t encode(float v, float inv, uint32_t r20) {
        const uint32_t c = (__float_as_uint(__fmul_rn(__fmul_rn(fabsf(v), inv), 0x1p-120f)) + r20) >> 20;
        return (c < 127u ? c : 127u) | (v < 0.0f ? 128u : 0u);
    }
};
template <> struct Code8<true> {
    static constexpr float TOP = 122880.0f;
    __device__ __forceinline__ static float decode(uint32_t c, float scale) {
        return __fmul_rn(__fmul_rn(__uint_as_float(c << 20), 0x1p112f), scale);
    }
    // A value above zero keeps a code above zero: m / sqrt(v) with v lost to rounding would be m / eps.
    __device__ __forceinline__ static uint32_t encode(float v, float inv, uint32_t r20) {
        const float y = __fmul_rn(__fmul_rn(fabsf(v), inv), 0x1p-112f);
        uint32_t c = (__float_as_uint(y) + r20) >> 20;
        c = c < 255u ? c : 255u;
        return c == 0u && y > 0.0f ? 1u : c;
    }
};

// Scale of a block from its largest magnitude over the warp.  Magnitudes compare as unsigned integers, and NaN above all, so
// a NaN or an infinity makes the whole block NaN instead of vanishing in a code.  A block below 2^-100 is zero: top / most
// would leave fp32's range.  Scale and inverse come from reciprocals (most * (1 / top), (1 / most) * top): the code of a value
// is defined by these roundings.
template <bool SECOND> __device__ __forceinline__ float am_scale(const float *v, float &inv) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) { const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu; most = a > most ? a : most; }
    float a = __uint_as_float(__reduce_max_sync(0xffffffffu, most));
    if (a < 0x1p-100f) a = 0.0f;
    inv = a > 0.0f ? __fmul_rn(__frcp_rn(a), Code8<SECOND>::TOP) : 0.0f;
    return a <= 3.402823466e38f ? __fmul_rn(a, 1.0f / Code8<SECOND>::TOP) : __uint_as_float(0x7fc00000u);
}

// Eight elements at p + i: whole when `full`, else those below n, the others 0.
template <typename T> __device__ __forceinline__ void am_load8(const T *p, size_t i, size_t n, bool full, float *f) {
    if (full) {
        if constexpr (sizeof(T) == 4) {
            Elt<T>::unpack(__ldcs(reinterpret_cast<const uint4 *>(p + i)), f);
            Elt<T>::unpack(__ldcs(reinterpret_cast<const uint4 *>(p + i) + 1), f + 4);
        } else {
            Elt<T>::unpack(__ldcs(reinterpret_cast<const uint4 *>(p + i)), f);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = i + j < n ? Elt<T>::to_f(p[i + j]) : 0.0f;
    }
}
template <typename T> __device__ __forceinline__ void am_store8(T *p, size_t i, size_t n, bool full, const float *f) {
    if (full) {
        if constexpr (sizeof(T) == 4) {
            __stcs(reinterpret_cast<uint4 *>(p + i), Elt<T>::pack(f));
            __stcs(reinterpret_cast<uint4 *>(p + i) + 1, Elt<T>::pack(f + 4));
        } else {
            __stcs(reinterpret_cast<uint4 *>(p + i), Elt<T>::pack(f));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) if (i + j < n) p[i + j] = Elt<T>::from_f(f[j]);
    }
}
__device__ __forceinline__ uint2 am_load_codes(const uint8_t *p, size_t i, size_t n, bool full) {
    if (full) return __ldcs(reinterpret_cast<const uint2 *>(p + i));
    uint2 c = make_uint2(0u, 0u);
#pragma unroll
    for (int j = 0; j < 8; j++) if (i + j < n) (j < 4 ? c.x : c.y) |= (uint32_t)p[i + j] << (8 * (j & 3));
    return c;
}
__device__ __forceinline__ void am_store_codes(uint8_t *p, size_t i, size_t n, bool full, uint2 c) {
    if (full) { __stcs(reinterpret_cast<uint2 *>(p + i), c); return; }
#pragma unroll
    for (int j = 0; j < 8; j++) if (i + j < n) p[i + j] = (uint8_t)((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
}
template <bool SECOND> __device__ __forceinline__ void am_decode8(uint2 c, float scale, float *f) {
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = Code8<SECOND>::decode(((j < 4 ? c.x : c.y) >> (8 * (j & 3))) & 255u, scale);
}

// A warp owns 256 consecutive elements of one tensor, a lane eight of them.  All loads of the lane are issued before the
// first use; nothing is kept between elements, so the kernel is a stream.
template <typename G, bool Q8, int CAP>
__global__ void __launch_bounds__(AM_THREADS) adam_multi_kernel(const __grid_constant__ AmList<CAP> list, const __grid_constant__ AmScalars s) {
    // the tensor of this block: the last whose first chunk is not behind it
    int lo = 0, hi = list.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (list.it[mid].first_chunk <= blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const AmItem &it = list.it[lo];
    const size_t n = it.n;
    const size_t group = (size_t)(blockIdx.x - it.first_chunk) * (AM_CHUNK / AM_GROUP) + threadIdx.x / 32;
    if (group * AM_GROUP >= n) return;                       // whole warps only
    const size_t i = group * AM_GROUP + (threadIdx.x & 31) * 8;
    const bool full = it.vec && i + 8 <= n;

    float w[8], g[8], m[8], v[8];
    am_load8(it.w, i, n, full, w);
    am_load8(static_cast<const G *>(it.g), i, n, full, g);
    if constexpr (Q8) {
        const uint2 cm = am_load_codes(static_cast<const uint8_t *>(it.m), i, n, full), cv = am_load_codes(static_cast<const uint8_t *>(it.v), i, n, full);
        am_decode8<false>(cm, it.ms[group], m);
        am_decode8<true>(cv, it.vs[group], v);
    } else {
        am_load8(static_cast<const float *>(it.m), i, n, full, m);
        am_load8(static_cast<const float *>(it.v), i, n, full, v);
    }
    const float clip = s.clip ? __ldg(s.clip) : 1.0f;        // a product with 1 changes nothing
    const float gscale = s.use_gscale ? s.gscale : 1.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float gj = __fmul_rn(__fmul_rn(g[j], gscale), clip);
        m[j] = __fadd_rn(__fmul_rn(s.b1, m[j]), __fmul_rn(s.omb1, gj));
        v[j] = __fadd_rn(__fmul_rn(s.b2, v[j]), __fmul_rn(__fmul_rn(s.omb2, gj), gj));
        if constexpr (Q8) {
            // The moments are exact to the bit, because codes are made of them; the step is not: approximate root and quotient
            // (2^-22) against 35 instructions an element more, where a byte-sized state leaves 60 in the time of its bytes.
            const float den = am_sqrt(v[j] * s.ibc2) + s.eps;
            const float step = __fdividef(m[j] * s.ibc1, den);
            w[j] -= s.lr * (s.variant == ANE_ADAM_STORIES ? step : fmaf(it.wd, w[j], step));
            continue;
        }
        const float mh = __fdiv_rn(m[j], s.bc1), vh = __fdiv_rn(v[j], s.bc2);
        const float den = __fadd_rn(__fsqrt_rn(vh), s.eps);
        if (s.variant == ANE_ADAM_STORIES) w[j] = __fsub_rn(w[j], __fdiv_rn(__fmul_rn(s.lr, mh), den));
        else w[j] = __fsub_rn(w[j], __fmul_rn(s.lr, __fadd_rn(__fdiv_rn(mh, den), __fmul_rn(it.wd, w[j]))));
    }
    am_store8(it.w, i, n, full, w);
    if (it.copy) {
        if (s.copy_dtype == ANE_BF16) am_store8(static_cast<__nv_bfloat16 *>(it.copy), i, n, full, w);
        else am_store8(static_cast<__half *>(it.copy), i, n, full, w);
    }
    if constexpr (Q8) {
        float im, iv;
        const float sm = am_scale<false>(m, im), sv = am_scale<true>(v, iv);
        if ((threadIdx.x & 31) == 0) { it.ms[group] = sm; it.vs[group] = sv; }
        uint32_t cm[2] = {0, 0}, cv[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t h = am_hash(i + j, it.key);
            cm[j / 4] |= Code8<false>::encode(m[j], im, h >> 12) << (8 * (j & 3));
            cv[j / 4] |= Code8<true>::encode(v[j], iv, h & 0xfffffu) << (8 * (j & 3));
        }
        am_store_codes(static_cast<uint8_t *>(it.m), i, n, full, make_uint2(cm[0], cm[1]));
        am_store_codes(static_cast<uint8_t *>(it.v), i, n, full, make_uint2(cv[0], cv[1]));
    } else {
        am_store8(static_cast<float *>(it.m), i, n, full, m);
        am_store8(static_cast<float *>(it.v), i, n, full, v);
    }
}

template <bool SECOND>
__global__ void __launch_bounds__(AM_THREADS) adam_state_unpack_kernel(size_t n, float *out, const uint8_t *codes, const float *scales, int vec) {
    const size_t group = (size_t)blockIdx.x * (AM_CHUNK / AM_GROUP) + threadIdx.x / 32;
    const size_t i = group * AM_GROUP + (threadIdx.x & 31) * 8;
    if (i >= n) return;
    const bool full = vec && i + 8 <= n;
    float f[8];
    am_decode8<SECOND>(am_load_codes(codes, i, n, full), scales[group], f);
    am_store8(out, i, n, full, f);
}

template <bool SECOND>
__global__ void __launch_bounds__(AM_THREADS) adam_state_pack_kernel(size_t n, uint8_t *codes, float *scales, const float *value, uint32_t key, int vec) {
    const size_t group = (size_t)blockIdx.x * (AM_CHUNK / AM_GROUP) + threadIdx.x / 32;
    if (group * AM_GROUP >= n) return;
    const size_t i = group * AM_GROUP + (threadIdx.x & 31) * 8;
    const bool full = vec && i + 8 <= n;
    float f[8], inv;
    am_load8(value, i, n, full, f);
    const float scale = am_scale<SECOND>(f, inv);
    if ((threadIdx.x & 31) == 0) scales[group] = scale;
    uint32_t c[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t h = am_hash(i + j, key);
        c[j / 4] |= Code8<SECOND>::encode(f[j], inv, SECOND ? h & 0xfffffu : h >> 12) << (8 * (j & 3));
    }
    am_store_codes(codes, i, n, full, make_uint2(c[0], c[1]));
}

static inline bool aligned_to(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <typename G, bool Q8, int CAP>
static int launch_items(cudaStream_t st, const AmItem *items, int count, const AmScalars &s) {
    static thread_local AmList<CAP> list;
    list.count = count;
    memcpy(list.it, items, sizeof(AmItem) * (size_t)count);
    const AmItem &last = items[count - 1];
    const unsigned chunks = last.first_chunk + (unsigned)((last.n + AM_CHUNK - 1) / AM_CHUNK);
    adam_multi_kernel<G, Q8, CAP><<<chunks, AM_THREADS, 0, st>>>(list, s);
    ANE_LAUNCH_OK(1);
    return ANE_CUDA_OK;
}

constexpr int AM_SMALL = 40, AM_LARGE = 400;      // 80 bytes a tensor: within 4 KB and 32 KB of kernel parameters

template <typename G, bool Q8>
static int launch_list(cudaStream_t st, AmItem *items, int count, const AmScalars &s) {
    for (int a = 0; a < count;) {
        uint64_t chunks = 0;
        int b = a;
        for (; b < count && b - a < AM_LARGE; b++) {
            const uint64_t more = (items[b].n + AM_CHUNK - 1) / AM_CHUNK;
            if (b > a && chunks + more > 0x7fffffffull) break;
            items[b].first_chunk = (uint32_t)chunks;
            chunks += more;
        }
        const int rc = b - a <= AM_SMALL ? launch_items<G, Q8, AM_SMALL>(st, items + a, b - a, s) : launch_items<G, Q8, AM_LARGE>(st, items + a, b - a, s);
        if (rc != ANE_CUDA_OK) return rc;
        a = b;
    }
    return ANE_CUDA_OK;
}

}  // namespace ane

using namespace ane;

extern "C" {

int ane_cuda_adam_multi_dev(void *stream, ane_adam_state state, ane_dtype g_dtype, ane_dtype copy_dtype, int count, const ane_adam_item *items, int t,
                            float lr, float b1, float b2, float eps, float gscale, const float *clip_dev, unsigned seed, unsigned flags) {
    ANE_REQUIRE_INIT();
    ANE_REQUIRE(count >= 0 && (items || count == 0), "%s: null list or negative count", __func__);
    ANE_REQUIRE(state == ANE_ADAM_STATE_F32 || state == ANE_ADAM_STATE_Q8, "%s: bad state type %d", __func__, (int)state);
    ANE_REQUIRE(dtype_ok(g_dtype), "%s: bad gradient dtype %d", __func__, (int)g_dtype);
    ANE_REQUIRE(t >= 1, "%s: step t must be >= 1 (got %d)", __func__, t);
    ANE_REQUIRE(flags == ANE_ADAM_STORIES || flags == ANE_ADAM_DYNAMIC, "%s: bad flags %u", __func__, flags);
    const bool q8 = state == ANE_ADAM_STATE_Q8;
    std::vector<AmItem> list;
    std::vector<std::pair<uintptr_t, uintptr_t>> written;
    list.reserve((size_t)count);
    for (int k = 0; k < count; k++) {
        const ane_adam_item &a = items[k];
        if (a.n == 0) continue;
        ANE_REQUIRE(a.n <= (size_t)AM_CHUNK * 0x7fffffffull, "%s: tensor %d is too large (%zu elements)", __func__, k, a.n);
        ANE_REQUIRE(a.w && a.g && a.m && a.v, "%s: null pointer in tensor %d", __func__, k);
        ANE_REQUIRE(!q8 || (a.m_scale && a.v_scale), "%s: tensor %d has 8-bit states and no scales", __func__, k);
        ANE_REQUIRE(!a.copy || copy_dtype == ANE_BF16 || copy_dtype == ANE_F16, "%s: the copy of the weights is bf16 or fp16 (got %d)", __func__, (int)copy_dtype);
        const size_t sb = q8 ? a.n : a.n * 4, cb = (a.n + AM_GROUP - 1) / AM_GROUP * 4;
        ANE_REQUIRE(aligned_to(a.w, 4) && aligned_to(a.g, dtype_size(g_dtype)) && (q8 || (aligned_to(a.m, 4) && aligned_to(a.v, 4))) &&
                        (!q8 || (aligned_to(a.m_scale, 4) && aligned_to(a.v_scale, 4))) && aligned_to(a.copy, 2),
                    "%s: a pointer of tensor %d is not aligned to its element", __func__, k);
        if (check_extents_on()) {
            ANE_CHECK_EXTENT(a.w, a.n * 4); ANE_CHECK_EXTENT(a.g, a.n * dtype_size(g_dtype));
            ANE_CHECK_EXTENT(a.m, sb); ANE_CHECK_EXTENT(a.v, sb); ANE_CHECK_EXTENT(a.copy, a.n * 2);
            if (q8) { ANE_CHECK_EXTENT(a.m_scale, cb); ANE_CHECK_EXTENT(a.v_scale, cb); }
            auto range = [&](const void *p, size_t bytes) { if (p) written.emplace_back((uintptr_t)p, (uintptr_t)p + bytes); };
            range(a.w, a.n * 4); range(a.m, sb); range(a.v, sb); range(a.copy, a.n * 2);
            if (q8) { range(a.m_scale, cb); range(a.v_scale, cb); }
        }
        AmItem d = {};
        d.w = a.w; d.g = a.g; d.m = a.m; d.v = a.v; d.ms = a.m_scale; d.vs = a.v_scale; d.copy = a.copy; d.n = a.n; d.wd = a.wd;
        d.key = am_mix(seed + 0x9E3779B9u * (uint32_t)k);
        const size_t sa = q8 ? 8 : 16;
        d.vec = aligned16(a.w) && aligned16(a.g) && aligned_to(a.m, sa) && aligned_to(a.v, sa) && aligned16(a.copy);
        list.push_back(d);
    }
    if (!written.empty()) {       // debug mode: two tensors that share memory would race
        std::sort(written.begin(), written.end());
        for (size_t k = 1; k < written.size(); k++)
            ANE_REQUIRE(written[k].first >= written[k - 1].second, "%s: two ranges that the step writes overlap", __func__);
    }
    if (list.empty()) return ANE_CUDA_OK;
    AmScalars s = {};
    s.b1 = b1; s.b2 = b2;
    s.omb1 = 1 - b1; s.omb2 = 1 - b2;
    s.bc1 = 1.0f - powf(b1, t);           // on the host, as ane_cuda_adam_dev
    s.bc2 = 1.0f - powf(b2, t);
    s.ibc1 = 1.0f / s.bc1; s.ibc2 = 1.0f / s.bc2;
    s.lr = lr; s.eps = eps; s.gscale = gscale;
    s.use_gscale = gscale != 1.0f;
    s.clip = clip_dev;
    s.variant = flags;
    s.copy_dtype = (int)copy_dtype;
    cudaStream_t st = (cudaStream_t)stream;
    ANE_DISPATCH_DTYPE(g_dtype, G, return q8 ? (launch_list<G, true>(st, list.data(), (int)list.size(), s)) : (launch_list<G, false>(st, list.data(), (int)list.size(), s)));
    return ANE_CUDA_OK;
}

int ane_cuda_adam_state_unpack_dev(void *stream, size_t n, float *out, const void *codes, const float *scales, int second) {
    ANE_REQUIRE_INIT();
    if (n == 0) return ANE_CUDA_OK;
    ANE_REQUIRE(out && codes && scales, "%s: null pointer", __func__);
    ANE_REQUIRE(second == 0 || second == 1, "%s: `second` is 0 or 1 (got %d)", __func__, second);
    ANE_REQUIRE(n <= (size_t)AM_CHUNK * 0x7fffffffull, "%s: too many elements", __func__);
    ANE_CHECK_EXTENT(out, n * 4); ANE_CHECK_EXTENT(codes, n); ANE_CHECK_EXTENT(scales, (n + AM_GROUP - 1) / AM_GROUP * 4);
    const unsigned blocks = (unsigned)((n + AM_CHUNK - 1) / AM_CHUNK);
    const int vec = aligned16(out) && aligned_to(codes, 8);
    cudaStream_t st = (cudaStream_t)stream;
    if (second) adam_state_unpack_kernel<true><<<blocks, AM_THREADS, 0, st>>>(n, out, static_cast<const uint8_t *>(codes), scales, vec);
    else adam_state_unpack_kernel<false><<<blocks, AM_THREADS, 0, st>>>(n, out, static_cast<const uint8_t *>(codes), scales, vec);
    ANE_LAUNCH_OK(1);
    return ANE_CUDA_OK;
}

int ane_cuda_adam_state_pack_dev(void *stream, size_t n, void *codes, float *scales, const float *value, int second, unsigned seed) {
    ANE_REQUIRE_INIT();
    if (n == 0) return ANE_CUDA_OK;
    ANE_REQUIRE(value && codes && scales, "%s: null pointer", __func__);
    ANE_REQUIRE(second == 0 || second == 1, "%s: `second` is 0 or 1 (got %d)", __func__, second);
    ANE_REQUIRE(n <= (size_t)AM_CHUNK * 0x7fffffffull, "%s: too many elements", __func__);
    ANE_CHECK_EXTENT(value, n * 4); ANE_CHECK_EXTENT(codes, n); ANE_CHECK_EXTENT(scales, (n + AM_GROUP - 1) / AM_GROUP * 4);
    const unsigned blocks = (unsigned)((n + AM_CHUNK - 1) / AM_CHUNK);
    const int vec = aligned16(value) && aligned_to(codes, 8);
    cudaStream_t st = (cudaStream_t)stream;
    const uint32_t key = am_mix(seed);
    if (second) adam_state_pack_kernel<true><<<blocks, AM_THREADS, 0, st>>>(n, static_cast<uint8_t *>(codes), scales, value, key, vec);
    else adam_state_pack_kernel<false><<<blocks, AM_THREADS, 0, st>>>(n, static_cast<uint8_t *>(codes), scales, value, key, vec);
    ANE_LAUNCH_OK(1);
    return ANE_CUDA_OK;
}

}  // extern "C"
