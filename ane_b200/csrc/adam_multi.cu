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
//
// Measured, 110 M parameters in 110 tensors: fp32 moments 28 bytes a parameter, 450 us, the copy rate; 8-bit moments with bf16
// gradients and copies 16 bytes a parameter, 340 us (5.2 TB/s): the arithmetic of the codes keeps the integer pipe busy 68 % of
// the time and the issue slots 74 %.
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
    float b1, b2, omb1, omb2, bc1, bc2, ibc1, ibc2, lr, eps, gscale, one;
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
constexpr uint32_t AM_GOLD = 0x9E3779B1u;
__device__ __forceinline__ float am_sqrt(float x) { float y; asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float am_rcp(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float2 am_two(float x) { return make_float2(x, x); }

// The step is bound by instruction issue beside 8-bit states (16 bytes an element, 50 instructions), so values go in pairs
// through the packed fp32 operations -- which round each half like the scalar ones -- and codes four to a word.
template <bool SECOND> struct Code8;
template <> struct Code8<false> {
    static constexpr float TOP = 480.0f;
    static constexpr float UP = 0x1p120f, DOWN = 0x1p-120f;
    // byte j of a word as a float's bits: the sign to bit 31, the code's seven bits to 26..20
    __device__ __forceinline__ static float bits(uint32_t word, int j) {
        return __uint_as_float((uint32_t)((int32_t)(word << (24 - 8 * j)) >> 4) & 0x87f00000u);
    }
    // y = value * inverse * 2^-120
    __device__ __forceinline__ static uint32_t encode(float v, float y, uint32_t r20) {
        const uint32_t c = ((__float_as_uint(y) & 0x7fffffffu) + r20) >> 20;
        return (c < 127u ? c : 127u) | (v < 0.0f ? 128u : 0u);
    }
};
template <> struct Code8<true> {
    static constexpr float TOP = 122880.0f;
    static constexpr float UP = 0x1p112f, DOWN = 0x1p-112f;
    __device__ __forceinline__ static float bits(uint32_t word, int j) {
        return __uint_as_float((8 * j < 20 ? word << (20 - 8 * j) : word >> (8 * j - 20)) & 0x0ff00000u);
    }
    // A value above zero keeps a code above zero: m / sqrt(v) with v lost to rounding would be m / eps.
    __device__ __forceinline__ static uint32_t encode(float, float y, uint32_t r20) {
        const uint32_t u = __float_as_uint(y) & 0x7fffffffu, c = (u + r20) >> 20, least = u < 1u ? u : 1u;
        return c < least ? least : c < 255u ? c : 255u;
    }
};

// Eight values of a lane.
typedef float2 Am8[4];
__device__ __forceinline__ float am_at(const Am8 &f, int j) { return j & 1 ? f[j >> 1].y : f[j >> 1].x; }

// Scale of a block from its largest magnitude over the warp.  Magnitudes compare as unsigned integers, and NaN above all, so
// a NaN or an infinity makes the whole block NaN instead of vanishing in a code.  A block below 2^-100 is zero: top / most
// would leave fp32's range.  Scale and inverse come from reciprocals (most * (1 / top), (1 / most) * top): the code of a value
// is defined by these roundings.
template <bool SECOND> __device__ __forceinline__ float am_scale(const Am8 &v, float &inv) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) { const uint32_t a = __float_as_uint(am_at(v, j)) & 0x7fffffffu; most = a > most ? a : most; }
    float a = __uint_as_float(__reduce_max_sync(0xffffffffu, most));
    if (a < 0x1p-100f) a = 0.0f;
    inv = a > 0.0f ? __fmul_rn(__frcp_rn(a), Code8<SECOND>::TOP) : 0.0f;
    return a <= 3.402823466e38f ? __fmul_rn(a, 1.0f / Code8<SECOND>::TOP) : __uint_as_float(0x7fc00000u);
}
template <bool SECOND> __device__ __forceinline__ void am_decode8(uint2 c, float scale, Am8 &f) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = i < 2 ? c.x : c.y;
        const float2 q = make_float2(Code8<SECOND>::bits(w, 2 * i & 3), Code8<SECOND>::bits(w, (2 * i & 3) + 1));
        f[i] = f2_mul(f2_mul(q, am_two(Code8<SECOND>::UP)), am_two(scale));
    }
}
// The random bits of element j of a lane whose first element hashes to h0: the upper 20 for the first moment, the lower 20
// for the second.
__device__ __forceinline__ uint32_t am_noise(uint32_t h0, int j) { return am_mix(h0 + (uint32_t)j * AM_GOLD); }
template <bool SECOND> __device__ __forceinline__ uint2 am_encode8(const Am8 &v, float inv, const uint32_t (&h)[8]) {
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 y = f2_mul(f2_mul(v[i], am_two(inv)), am_two(Code8<SECOND>::DOWN));
        c[2 * i] = Code8<SECOND>::encode(v[i].x, y.x, SECOND ? h[2 * i] & 0xfffffu : h[2 * i] >> 12);
        c[2 * i + 1] = Code8<SECOND>::encode(v[i].y, y.y, SECOND ? h[2 * i + 1] & 0xfffffu : h[2 * i + 1] >> 12);
    }
    return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
}

// Eight elements at p + i: whole when `full`, else those below n, the others 0.
template <typename T> __device__ __forceinline__ void am_load8(const T *p, size_t i, size_t n, bool full, Am8 &f) {
    if (full) {
        Elt<T>::unpack2(__ldcs(reinterpret_cast<const uint4 *>(p + i)), f);
        if constexpr (sizeof(T) == 4) Elt<T>::unpack2(__ldcs(reinterpret_cast<const uint4 *>(p + i) + 1), f + 2);
    } else {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = i + j < n ? Elt<T>::to_f(p[i + j]) : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = make_float2(v[2 * j], v[2 * j + 1]);
    }
}
template <typename T> __device__ __forceinline__ void am_store8(T *p, size_t i, size_t n, bool full, const Am8 &f) {
    if (full) {
        __stcs(reinterpret_cast<uint4 *>(p + i), Elt<T>::pack2(f));
        if constexpr (sizeof(T) == 4) __stcs(reinterpret_cast<uint4 *>(p + i) + 1, Elt<T>::pack2(f + 2));
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) if (i + j < n) p[i + j] = Elt<T>::from_f(am_at(f, j));
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

    Am8 w, g, m, v;
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
    for (int j = 0; j < 4; j++) {
        const float2 gj = f2_mul(f2_mul(g[j], am_two(gscale)), am_two(clip));
        // A sum of two rounded products.  A packed product and a packed add would be contracted into one fma, with one rounding
        // less; as a product with a 1 that the compiler does not know the add stays what it is.
        m[j] = f2_fma(f2_mul(am_two(s.b1), m[j]), am_two(s.one), f2_mul(am_two(s.omb1), gj));
        v[j] = f2_fma(f2_mul(am_two(s.b2), v[j]), am_two(s.one), f2_mul(f2_mul(am_two(s.omb2), gj), gj));
        if constexpr (Q8) {
            // The moments are exact to the bit, because codes are made of them; the step is not: approximate root and reciprocal
            // (2^-22 each) against 35 instructions an element more.
            const float2 vh = f2_mul(v[j], am_two(s.ibc2));
            const float2 den = f2_add(make_float2(am_sqrt(vh.x), am_sqrt(vh.y)), am_two(s.eps));
            float2 step = f2_mul(f2_mul(m[j], am_two(s.ibc1)), make_float2(am_rcp(den.x), am_rcp(den.y)));
            if (s.variant != ANE_ADAM_STORIES) step = f2_fma(am_two(it.wd), w[j], step);
            w[j] = f2_fma(am_two(-s.lr), step, w[j]);
        } else {
            auto one = [&](float w, float m, float v) {
                const float mh = __fdiv_rn(m, s.bc1), vh = __fdiv_rn(v, s.bc2);
                const float den = __fadd_rn(__fsqrt_rn(vh), s.eps);
                if (s.variant == ANE_ADAM_STORIES) return __fsub_rn(w, __fdiv_rn(__fmul_rn(s.lr, mh), den));
                return __fsub_rn(w, __fmul_rn(s.lr, __fadd_rn(__fdiv_rn(mh, den), __fmul_rn(it.wd, w))));
            };
            w[j] = make_float2(one(w[j].x, m[j].x, v[j].x), one(w[j].y, m[j].y, v[j].y));
        }
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
        uint32_t h[8];
        const uint32_t h0 = (uint32_t)i * AM_GOLD + it.key;
#pragma unroll
        for (int j = 0; j < 8; j++) h[j] = am_noise(h0, j);
        am_store_codes(static_cast<uint8_t *>(it.m), i, n, full, am_encode8<false>(m, im, h));
        am_store_codes(static_cast<uint8_t *>(it.v), i, n, full, am_encode8<true>(v, iv, h));
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
    Am8 f;
    am_decode8<SECOND>(am_load_codes(codes, i, n, full), scales[group], f);
    am_store8(out, i, n, full, f);
}

template <bool SECOND>
__global__ void __launch_bounds__(AM_THREADS) adam_state_pack_kernel(size_t n, uint8_t *codes, float *scales, const float *value, uint32_t key, int vec) {
    const size_t group = (size_t)blockIdx.x * (AM_CHUNK / AM_GROUP) + threadIdx.x / 32;
    if (group * AM_GROUP >= n) return;
    const size_t i = group * AM_GROUP + (threadIdx.x & 31) * 8;
    const bool full = vec && i + 8 <= n;
    Am8 f;
    float inv;
    am_load8(value, i, n, full, f);
    const float scale = am_scale<SECOND>(f, inv);
    if ((threadIdx.x & 31) == 0) scales[group] = scale;
    uint32_t h[8];
    const uint32_t h0 = (uint32_t)i * AM_GOLD + key;
#pragma unroll
    for (int j = 0; j < 8; j++) h[j] = am_noise(h0, j);
    am_store_codes(codes, i, n, full, am_encode8<SECOND>(f, inv, h));
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
    struct Range { uintptr_t from, to; bool written; };
    std::vector<Range> ranges;
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
            auto range = [&](const void *p, size_t bytes, bool written = true) { if (p) ranges.push_back({(uintptr_t)p, (uintptr_t)p + bytes, written}); };
            range(a.w, a.n * 4); range(a.m, sb); range(a.v, sb); range(a.copy, a.n * 2);
            range(a.g, a.n * dtype_size(g_dtype), false);
            if (q8) { range(a.m_scale, cb); range(a.v_scale, cb); }
        }
        AmItem d = {};
        d.w = a.w; d.g = a.g; d.m = a.m; d.v = a.v; d.ms = a.m_scale; d.vs = a.v_scale; d.copy = a.copy; d.n = a.n; d.wd = a.wd;
        d.key = am_mix(seed + 0x9E3779B9u * (uint32_t)k);
        const size_t sa = q8 ? 8 : 16;
        d.vec = aligned16(a.w) && aligned16(a.g) && aligned_to(a.m, sa) && aligned_to(a.v, sa) && aligned16(a.copy);
        list.push_back(d);
    }
    // debug mode: a tensor that shares memory with one that the step writes would race; gradients may share with each other
    std::sort(ranges.begin(), ranges.end(), [](const Range &a, const Range &b) { return a.from < b.from; });
    uintptr_t written_to = 0, any_to = 0;
    for (const Range &r : ranges) {
        ANE_REQUIRE(r.from >= (r.written ? any_to : written_to), "%s: two tensors overlap and the step writes one of them", __func__);
        any_to = std::max(any_to, r.to);
        if (r.written) written_to = std::max(written_to, r.to);
    }
    if (list.empty()) return ANE_CUDA_OK;
    AmScalars s = {};
    s.b1 = b1; s.b2 = b2;
    s.omb1 = 1 - b1; s.omb2 = 1 - b2;
    s.bc1 = 1.0f - powf(b1, t);           // on the host, as ane_cuda_adam_dev
    s.bc2 = 1.0f - powf(b2, t);
    s.ibc1 = 1.0f / s.bc1; s.ibc2 = 1.0f / s.bc2;
    s.one = 1.0f;
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
