// AdamW over a list of tensors and the norm of a list of gradients (CUDA cores, HBM-bound).
//
// One launch walks up to NT_LARGE tensors: their pointers travel in the kernel's parameters.  The tensors are cut into segments of
// 256 elements, the warps of the grid take segments in turn (each by itself: no barrier), and since a warp's segments only move
// forward, the tensor of the next one is found by stepping on from the last one's (of the first by bisection).  256 consecutive elements share the scale of an
// 8-bit moment, so its maximum is one shuffle reduction and nothing is read twice.  Arithmetic is float32; what the 8-bit
// moments are made of has one rounding per operation as written (no contraction), so their bytes follow from the inputs alone.
//
//   m' = b1 m + (1 - b1) g        v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
#include <cuda_fp8.h>
#include <float.h>
#include <math.h>
#include <type_traits>

#include "common.cuh"

namespace rdb {

constexpr int NORM_CHUNK = 8192;
constexpr int ADAMW_THREADS = 256;
static_assert(NORM_CHUNK == 8 * 4 * 256, "sumsq_kernel takes a chunk in four passes of its eight warps");
constexpr int SEG = RDB_ADAMW_BLOCK;      // elements per warp pass, and per scale of an 8-bit moment
static_assert(SEG == 256, "a warp pass is 32 lanes x 8 elements");

struct AdamwDesc {
    void *p;
    const void *g;
    float *master;
    void *m, *v;
    float *ms, *vs;
    float *step;
    int64_t n;
};

// NT tensors; first[i] is the first segment (AdamW) or chunk (norm) of tensor i, first[count] their number
template <int NT>
struct AdamwTable {
    AdamwDesc t[NT];
    uint32_t first[NT + 1];
    int32_t count;
    int32_t index0;                       // position of t[0] in the caller's list
};

struct AdamwScalars {
    float b1, omb1, b2, omb2, eps;
    bool fast;                            // see update_of
    double lr, ln_beta1, ln_beta2;         // natural logarithms; -inf for 0
    const float *lr_dev;                  // one float32 in device memory, or null: `lr`
    double weight_decay;
    uint32_t seed;
};

// ---- loads and stores of the 8 elements a lane owns: two groups of four, 128 apart (vector form), or eight single elements
// 32 apart (tensors that do not start on a vector boundary, and the ragged end of a tensor)
template <typename T> struct Vec4;
template <> struct Vec4<float> { using V = float4; };
template <> struct Vec4<__nv_bfloat16> { using V = uint2; };

template <bool VEC> __device__ __forceinline__ int elem_of(int lane, int j) {
    return VEC ? ((j >> 2) * 128 + lane * 4 + (j & 3)) : (j * 32 + lane);
}

template <bool VEC, typename T>
__device__ __forceinline__ void load8(T (&r)[8], const T *__restrict__ base, int lane, int left) {
    if (VEC) {
        using V = typename Vec4<T>::V;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const V v = *reinterpret_cast<const V *>(base + h * 128 + lane * 4);
            const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
            for (int k = 0; k < 4; ++k) r[h * 4 + k] = e[k];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = j * 32 + lane;
            T zero{};
            r[j] = e < left ? base[e] : zero;
        }
    }
}

template <bool VEC, typename T>
__device__ __forceinline__ void store8(T *__restrict__ base, const T (&r)[8], int lane, int left) {
    if (VEC) {
        using V = typename Vec4<T>::V;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            V v;
            T *e = reinterpret_cast<T *>(&v);
#pragma unroll
            for (int k = 0; k < 4; ++k) e[k] = r[h * 4 + k];
            *reinterpret_cast<V *>(base + h * 128 + lane * 4) = v;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = j * 32 + lane;
            if (e < left) base[e] = r[j];
        }
    }
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// First moment in 8 bits: float8 e4m3 times the scale that puts the block's largest magnitude at 448, rounded to nearest
// (off by at most 2^-4 of the value; b1 forgets it within a few steps).
__device__ __forceinline__ float2 e4m3_values(uint8_t c0, uint8_t c1) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((uint32_t)c0 | ((uint32_t)c1 << 8)), __NV_E4M3);
    return __half22float2(__half2(h));
}
__device__ __forceinline__ uint16_t e4m3_codes(float x0, float x1) { return __nv_cvt_float2_to_fp8x2(make_float2(x0, x1), __NV_SATFINITE, __NV_E4M3); }

// x / d with 1 / d at hand, correctly rounded: quotient, exact residual, one correction (P. Markstein, "Computation of elementary
// functions on the IBM RISC System/6000 processor", 1990).  The bytes of the second moment hang on every bit of it.
__device__ __forceinline__ float divide_by(float x, float d, float inv) {
    const float q = __fmul_rn(x, inv);
    return __fmaf_rn(__fmaf_rn(-q, d, x), inv, q);
}

constexpr float V_MOST = 3e38f;         // largest second moment in 8 bits: 1.9375 times its scale is still finite
__device__ __forceinline__ bool is_lost(float m, float v) { return !(fabsf(m) <= FLT_MAX && v <= V_MOST); }

// Second moment in 8 bits: no sign, 4 exponent bits (bias 15), 4 mantissa bits; byte 255 stands for 1.9375 and carries the
// block's maximum.  Shifted into a float32 the byte sits on top of exponent and mantissa, so its value is that float32 times
// 2^112 = 5.19e33 (subnormals included).  (1 - b2) is far below a step of any 8-bit format: rounding to nearest would leave v where it
// is however small the gradients become, so v is rounded to one of its two neighbours at random with the odds that keep its
// expectation: add 19 random bits below the byte and cut.  A positive v never becomes 0: it divides.
__device__ __forceinline__ uint32_t ue4m4_code(float q, float v, uint32_t r19) {
    uint32_t c = (__float_as_uint(__fmul_rn(q, 1.925929944387236e-34f)) + r19) >> 19;
    c = c > 255u ? 255u : c;
    return (c == 0u && v > 0.0f) ? 1u : c;
}

// Division and square root of the update, within 2^-21.  The fast forms take values below 2^-126 for 0.  A v below it then misses from the
// denominator with up to 2^-63 inv_root, so they are taken where eps is 2^21 times that (the usual 1e-8 is); an m below it has an
// update of at most 2^-126 / eps < 2^-84, which becomes 0.
constexpr float FAST_EPS = 2.2737368e-13f;     // 2^21 * 2^-63
__device__ __forceinline__ float update_of(float m, float v, float inv_root, float eps, bool fast) {
    if (fast) {
        float r, q;
        asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
        r = __fmaf_rn(r, inv_root, eps);
        asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(q) : "f"(m), "f"(r));
        return q;
    }
    return __fdiv_rn(m, __fmaf_rn(__fsqrt_rn(v), inv_root, eps));
}

struct StepScalars {
    float size, inv_root, decay, eps;
    bool fast;
};

// parameter (or its master) after the step
template <typename P, bool MASTER>
__device__ __forceinline__ void move(P &p8, float &w8, float m, float v, const StepScalars &c) {
    const float p = MASTER ? w8 : to_f32<P>(p8);
    const float q = __fmaf_rn(p, c.decay, -c.size * update_of(m, v, c.inv_root, c.eps, c.fast));
    if (MASTER) w8 = q;
    p8 = from_f32<P>(q);
}

__device__ __forceinline__ void new_moments(float &m, float &v, float g, const AdamwScalars &s) {
    m = __fadd_rn(__fmul_rn(m, s.b1), __fmul_rn(g, s.omb1));
    v = __fadd_rn(__fmul_rn(v, s.b2), __fmul_rn(__fmul_rn(g, g), s.omb2));
}

template <typename P, typename G, bool MASTER, bool VEC>
__device__ __forceinline__ void adamw_segment32(const AdamwDesc &d, int64_t at, int left, int lane, const AdamwScalars &s, float gscale,
                                                const StepScalars &c) {
    P p8[8];
    G g8[8];
    float m[8], v[8], w8[8];
    load8<VEC>(g8, reinterpret_cast<const G *>(d.g) + at, lane, left);
    load8<VEC>(m, const_cast<const float *>(reinterpret_cast<float *>(d.m)) + at, lane, left);
    load8<VEC>(v, const_cast<const float *>(reinterpret_cast<float *>(d.v)) + at, lane, left);
    if (MASTER) load8<VEC>(w8, const_cast<const float *>(d.master) + at, lane, left);
    else load8<VEC>(p8, const_cast<const P *>(reinterpret_cast<P *>(d.p)) + at, lane, left);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        new_moments(m[j], v[j], __fmul_rn(to_f32<G>(g8[j]), gscale), s);
        move<P, MASTER>(p8[j], w8[j], m[j], v[j], c);
    }
    store8<VEC>(reinterpret_cast<P *>(d.p) + at, p8, lane, left);
    if (MASTER) store8<VEC>(d.master + at, w8, lane, left);
    store8<VEC>(reinterpret_cast<float *>(d.m) + at, m, lane, left);
    store8<VEC>(reinterpret_cast<float *>(d.v) + at, v, lane, left);
}

// four bytes of a lane: words in the vector form, gathered bytes otherwise
template <bool VEC> __device__ __forceinline__ uint32_t load_bytes(const uint8_t *base, int h, int lane, int left) {
    if (VEC) return *reinterpret_cast<const uint32_t *>(base + h * 128 + lane * 4);
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int e = elem_of<false>(lane, h * 4 + k);
        w |= (e < left ? (uint32_t)base[e] : 0u) << (8 * k);
    }
    return w;
}
template <bool VEC> __device__ __forceinline__ void store_bytes(uint8_t *base, uint32_t w, int h, int lane, int left) {
    if (VEC) *reinterpret_cast<uint32_t *>(base + h * 128 + lane * 4) = w;
    else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int e = elem_of<false>(lane, h * 4 + k);
            if (e < left) base[e] = (uint8_t)(w >> (8 * k));
        }
    }
}

template <typename P, typename G, bool MASTER, bool VEC>
__device__ __forceinline__ void adamw_segment8(const AdamwDesc &d, int64_t at, int left, int lane, const AdamwScalars &s, float gscale,
                                               const StepScalars &c, uint32_t rseed) {
    P p8[8];
    G g8[8];
    float m[8], v[8], w8[8];
    uint8_t *mb = reinterpret_cast<uint8_t *>(d.m) + at, *vb = reinterpret_cast<uint8_t *>(d.v) + at;
    load8<VEC>(g8, reinterpret_cast<const G *>(d.g) + at, lane, left);
    uint32_t mw[2], vw[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        mw[h] = load_bytes<VEC>(mb, h, lane, left);
        vw[h] = load_bytes<VEC>(vb, h, lane, left);
    }
    if (MASTER) load8<VEC>(w8, const_cast<const float *>(d.master) + at, lane, left);
    else load8<VEC>(p8, const_cast<const P *>(reinterpret_cast<P *>(d.p)) + at, lane, left);
    float mscale = d.ms[at / SEG], vscale = d.vs[at / SEG];
    // byte << 19 as a float32 is the value times 2^-112: one product where the scale leaves room for 2^112
    const bool room = vscale < 16384.0f;
    const float vup = room ? __fmul_rn(vscale, 5.192296858534828e33f) : vscale;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float2 x0 = e4m3_values((uint8_t)mw[h], (uint8_t)(mw[h] >> 8)), x1 = e4m3_values((uint8_t)(mw[h] >> 16), (uint8_t)(mw[h] >> 24));
        m[h * 4] = __fmul_rn(x0.x, mscale);
        m[h * 4 + 1] = __fmul_rn(x0.y, mscale);
        m[h * 4 + 2] = __fmul_rn(x1.x, mscale);
        m[h * 4 + 3] = __fmul_rn(x1.y, mscale);
        const uint32_t b0 = (vw[h] & 0xFFu) << 19, b1 = (vw[h] & 0xFF00u) << 11, b2 = (vw[h] & 0xFF0000u) << 3, b3 = (vw[h] >> 5) & 0x7F80000u;
        const uint32_t b[4] = {b0, b1, b2, b3};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            v[h * 4 + k] = room ? __fmul_rn(__uint_as_float(b[k]), vup) : __fmul_rn(__fmul_rn(__uint_as_float(b[k]), 5.192296858534828e33f), vup);
    }
    float mmax = 0.0f, vmax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        new_moments(m[j], v[j], __fmul_rn(to_f32<G>(g8[j]), gscale), s);
        mmax = fmaxf(mmax, fabsf(m[j]));
        vmax = fmaxf(vmax, v[j]);
        move<P, MASTER>(p8[j], w8[j], m[j], v[j], c);
    }
    store8<VEC>(reinterpret_cast<P *>(d.p) + at, p8, lane, left);
    if (MASTER) store8<VEC>(d.master + at, w8, lane, left);
    mmax = warp_max(mmax);
    vmax = warp_max(vmax);
    const bool in_range = mmax <= FLT_MAX && vmax <= V_MOST;
    if (!in_range) {
        // Some element's moments have left the range: it is lost (first moment NaN from here on), and its block's others go on as if it were
        // not there.  An infinite scale would turn them all into 0 * infinity.
        mmax = vmax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (is_lost(m[j], v[j])) continue;
            mmax = fmaxf(mmax, fabsf(m[j]));
            vmax = fmaxf(vmax, v[j]);
        }
        mmax = warp_max(mmax);
        vmax = warp_max(vmax);
    }
    mscale = __fmul_rn(mmax, 1.0f / 448.0f);
    vscale = __fmul_rn(vmax, 1.0f / 1.9375f);
    const uint32_t h0 = (uint32_t)at * SQ5_N1 + rseed;
    // ordinary scales: multiply by the reciprocal (a NaN stays one); others divide, and a scale of zero gives zero, but NaN where an element is
    // lost: the first moment's code holds NaN.  (The second moment's has none: 255, the block's largest.  An element never has it NaN alone.)
    const bool easy = in_range && mscale > 1e-30f && vscale > 1e-30f && mscale < 1e30f && vscale < 1e30f;
    const float minv = easy ? __frcp_rn(mscale) : 0.0f, vinv = easy ? __frcp_rn(vscale) : 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float qm[4], qv[4];
        uint32_t code[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int j = h * 4 + k;
            if (easy) {
                qm[k] = divide_by(m[j], mscale, minv);
                qv[k] = divide_by(v[j], vscale, vinv);
            } else {
                qm[k] = is_lost(m[j], v[j]) ? NAN : mscale > 0.0f ? __fdiv_rn(m[j], mscale) : 0.0f;
                qv[k] = vscale > 0.0f ? __fdiv_rn(v[j], vscale) : 0.0f;
            }
            code[k] = ue4m4_code(qv[k], v[j], sq5_tail(h0 + (uint32_t)elem_of<VEC>(lane, j) * SQ5_N1) >> 13);
        }
        store_bytes<VEC>(mb, (uint32_t)e4m3_codes(qm[0], qm[1]) | ((uint32_t)e4m3_codes(qm[2], qm[3]) << 16), h, lane, left);
        store_bytes<VEC>(vb, code[0] | (code[1] << 8) | (code[2] << 16) | (code[3] << 24), h, lane, left);
    }
    if (lane == 0) {
        d.ms[at / SEG] = mscale;
        d.vs[at / SEG] = vscale;
    }
}

// the tensor that part `chunk` belongs to (the last one when there is none)
template <typename Table>
__device__ __forceinline__ int find_tensor(const Table &tab, uint32_t chunk) {
    int lo = 0, hi = tab.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.first[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// every tensor's step count, one more; a launch of its own, before any block of the update reads a count
template <int NT>
struct StepTable {
    float *step[NT];
    int32_t count;
};
template <int NT>
__global__ void adamw_count_kernel(const __grid_constant__ StepTable<NT> tab) {
    pdl_launch_dependents();
    pdl_wait();
    for (int i = threadIdx.x; i < tab.count; i += blockDim.x) *tab.step[i] += 1.0f;
}

template <typename P, typename G, bool MASTER, bool BITS8, int NT>
__global__ void __launch_bounds__(ADAMW_THREADS, 4)
adamw_kernel(const __grid_constant__ AdamwTable<NT> tab, const AdamwScalars s, const float *__restrict__ grad_scale) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const uint32_t warps = gridDim.x * (ADAMW_THREADS / 32);
    const float gscale = grad_scale ? *grad_scale : 1.0f;
    const uint32_t segs = tab.first[tab.count];
    StepScalars c{};
    c.eps = s.eps;
    c.fast = s.fast;
    float t_have = NAN;
    uint32_t g = blockIdx.x * (ADAMW_THREADS / 32) + (threadIdx.x >> 5);
    int ti = find_tensor(tab, g);
    for (; g < segs; g += warps) {
        while (g >= tab.first[ti + 1]) ++ti;
        const AdamwDesc &d = tab.t[ti];
        const float t = *d.step;
        if (t != t_have) {                // bias corrections of this step, in float64; tensors that began together share them
            const double lr = s.lr_dev ? (double)*s.lr_dev : s.lr;
            c.size = (float)(lr / -expm1((double)t * s.ln_beta1));            // 1 - beta^t
            c.inv_root = 1.0f / sqrtf((float)-expm1((double)t * s.ln_beta2));
            c.decay = (float)(1.0 - lr * s.weight_decay);
            t_have = t;
        }
        const int64_t at = (int64_t)(g - tab.first[ti]) * SEG;
        const int left = (int)(d.n - at < SEG ? d.n - at : SEG);
        constexpr uintptr_t PV = sizeof(P) * 4 - 1, GV = sizeof(G) * 4 - 1, SV = BITS8 ? 3 : 15;
        const bool vec = left == SEG && ((reinterpret_cast<uintptr_t>(d.p) & PV) | (reinterpret_cast<uintptr_t>(d.g) & GV) |
                                         (reinterpret_cast<uintptr_t>(d.m) & SV) | (reinterpret_cast<uintptr_t>(d.v) & SV) |
                                         (MASTER ? reinterpret_cast<uintptr_t>(d.master) & 15 : 0)) == 0;
        if (BITS8) {
            const uint32_t rseed = s.seed + (uint32_t)(int64_t)t * 0x9E3779B1u + (uint32_t)(tab.index0 + ti) * 0x85EBCA6Bu;
            if (vec) adamw_segment8<P, G, MASTER, true>(d, at, left, lane, s, gscale, c, rseed);
            else adamw_segment8<P, G, MASTER, false>(d, at, left, lane, s, gscale, c, rseed);
        } else {
            if (vec) adamw_segment32<P, G, MASTER, true>(d, at, left, lane, s, gscale, c);
            else adamw_segment32<P, G, MASTER, false>(d, at, left, lane, s, gscale, c);
        }
    }
}

// ---- norm ----------------------------------------------------------------------------------------------------------------
// Sum of squares: float32 within the 8 elements a lane reads at a time (float64 where their squares leave its range), float64 above; one
// partial sum per block in the workspace, added in block order by one block, so the result repeats run to run.  Bound by latency: at 80 M
// bf16 elements DRAM is 65 % busy, issue 38 %, 64 % of the warps resident (5.2 TB/s).
template <typename G> __device__ __forceinline__ double sum_of_squares(const G (&g)[8]) {
    float f = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f += to_f32<G>(g[j]) * to_f32<G>(g[j]);
    if (f > 1e-30f && f < 1e38f) return (double)f;
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(to_f32<G>(g[j])));
    if (f == 0.0f && top == 0.0f) return 0.0;              // gradients of rows that were not looked up
    double d = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) d += (double)to_f32<G>(g[j]) * (double)to_f32<G>(g[j]);
    return d;
}

template <typename G, int NT>
__global__ void __launch_bounds__(ADAMW_THREADS)
sumsq_kernel(const __grid_constant__ AdamwTable<NT> tab, double *__restrict__ partial) {
    __shared__ double sh[ADAMW_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t chunks = tab.first[tab.count];
    double acc = 0.0;
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int ti = find_tensor(tab, c);
        const AdamwDesc &d = tab.t[ti];
        const int64_t lo = (int64_t)(c - tab.first[ti]) * NORM_CHUNK;
        const int64_t hi = lo + NORM_CHUNK < d.n ? lo + NORM_CHUNK : d.n;
        const bool vec = (reinterpret_cast<uintptr_t>(d.g) & (sizeof(G) * 4 - 1)) == 0;
        const G *g = reinterpret_cast<const G *>(d.g);
        if (vec && hi - lo == NORM_CHUNK) {         // a whole chunk: four 256-element passes of the warp, all loads in flight
            G g8[4][8];
#pragma unroll
            for (int u = 0; u < 4; ++u) load8<true>(g8[u], g + lo + (warp * 4 + u) * SEG, lane, SEG);
#pragma unroll
            for (int u = 0; u < 4; ++u) acc += sum_of_squares(g8[u]);
            continue;
        }
        for (int64_t at = lo + warp * SEG; at < hi; at += (ADAMW_THREADS / 32) * SEG) {
            const int left = (int)(hi - at < SEG ? hi - at : SEG);
            G g8[8];
            if (vec && left == SEG) load8<true>(g8, g + at, lane, left);
            else load8<false>(g8, g + at, lane, left);
            acc += sum_of_squares(g8);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) sh[warp] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < ADAMW_THREADS / 32; ++i) t += sh[i];
        partial[blockIdx.x] = t;
    }
}

// norm, and the factor that brings it down to max_norm (1 when it is below; max_norm < 0: none asked for)
__global__ void __launch_bounds__(256) norm_finish_kernel(float *__restrict__ norm, float *__restrict__ coef, const double *__restrict__ partial,
                                                          int n, float max_norm) {
    __shared__ double sh[256];
    pdl_launch_dependents();
    pdl_wait();
    double a = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) a += partial[i];
    sh[threadIdx.x] = a;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const float nv = (float)sqrt(sh[0]);
        if (norm) *norm = nv;
        if (coef) {
            const float c = max_norm / (nv + 1e-6f);
            *coef = c > 1.0f ? 1.0f : c;          // not-a-number stays one
        }
    }
}

static int norm_blocks(uint32_t chunks) { return (int)(chunks < (uint32_t)RDB_NORM_BLOCKS ? (chunks ? chunks : 1) : RDB_NORM_BLOCKS); }

// ---- host ----------------------------------------------------------------------------------------------------------------
constexpr int NT_SMALL = 48, NT_LARGE = 384;      // tensors per launch: 3.5 KB or 26 KB of kernel parameters
static_assert(sizeof(AdamwTable<NT_LARGE>) + 512 < 32764, "kernel parameters");

template <int NT>
static int count_parts(AdamwTable<NT> *tab, int n, int index0, int part) {
    uint64_t c = 0;
    for (int i = 0; i < n; ++i) {
        tab->first[i] = (uint32_t)c;
        c += (uint64_t)cdiv64(tab->t[i].n, part);
        if (c >= (1ull << 32)) return RDB_ERR_TOO_LARGE;
    }
    tab->first[n] = (uint32_t)c;
    tab->count = n;
    tab->index0 = index0;
    return RDB_OK;
}

template <typename P, typename G, bool MASTER, bool BITS8, int NT>
static int launch_adamw(const rdb_adamw_lists &l, int n, int at, const AdamwScalars &s, const float *gs, cudaStream_t st) {
    AdamwTable<NT> tab;
    StepTable<NT> steps;
    for (int i = 0; i < n; ++i) {
        const int k = at + i;
        tab.t[i] = AdamwDesc{l.param[k], l.grad[k], MASTER ? l.master[k] : nullptr, l.exp_avg[k], l.exp_avg_sq[k], BITS8 ? l.exp_avg_scale[k] : nullptr,
                             BITS8 ? l.exp_avg_sq_scale[k] : nullptr, l.step[k], l.numel[k]};
        steps.step[i] = l.step[k];
    }
    int rc = count_parts(&tab, n, at, SEG);
    if (rc) return rc;
    steps.count = n;
    rc = launch_pdl(adamw_count_kernel<NT>, dim3(1), 256, 0, st, steps);
    if (rc) return rc;
    const uint32_t want = (tab.first[n] + ADAMW_THREADS / 32 - 1) / (ADAMW_THREADS / 32);
    if (want == 0) return RDB_OK;
    // Four blocks are resident per SM.  32-bit moments, bound by memory: many short blocks (69 M elements, float32: 4, 8, 16, 64
    // blocks per SM take 318, 307, 298, 287 us); 8-bit moments pay a block's float64 bias corrections more dearly (232, 229, 228, 251).
    const uint32_t cap = 148 * (BITS8 ? 16 : 64);
    return launch_pdl(adamw_kernel<P, G, MASTER, BITS8, NT>, dim3(want < cap ? want : cap), ADAMW_THREADS, 0, st, tab, s, gs);
}

template <typename P, typename G, bool MASTER, bool BITS8>
static int adamw_all(const rdb_adamw_lists &l, const AdamwScalars &s, const float *gs, cudaStream_t st) {
    const int n = (int)l.n;
    for (int i = 0; i < n;) {
        const int k = n - i < NT_LARGE ? n - i : NT_LARGE;
        const int rc = k <= NT_SMALL ? launch_adamw<P, G, MASTER, BITS8, NT_SMALL>(l, k, i, s, gs, st)
                                     : launch_adamw<P, G, MASTER, BITS8, NT_LARGE>(l, k, i, s, gs, st);
        if (rc) return rc;
        i += k;
    }
    return RDB_OK;
}

struct GradRef {
    const void *p;
    int64_t n;
};

template <typename G, int NT>
static int launch_sumsq(const GradRef *t, int n, double *partial, int *used, cudaStream_t st) {
    AdamwTable<NT> tab;
    for (int i = 0; i < n; ++i) {
        tab.t[i] = AdamwDesc{};
        tab.t[i].g = t[i].p;
        tab.t[i].n = t[i].n;
    }
    int rc = count_parts(&tab, n, 0, NORM_CHUNK);
    if (rc) return rc;
    *used = norm_blocks(tab.first[n]);
    return launch_pdl(sumsq_kernel<G, NT>, dim3(*used), ADAMW_THREADS, 0, st, tab, partial);
}

}  // namespace rdb

using namespace rdb;

extern "C" int rdb_adamw_step(const rdb_adamw_lists *lists, int param_dtype, int grad_dtype, int state_bits, const rdb_adamw_hyper *h,
                              const float *grad_scale, void *stream) {
    if (!lists || !h) return RDB_ERR_NULL;
    const rdb_adamw_lists &l = *lists;
    if (l.n < 0) return RDB_ERR_SHAPE;
    if (l.n == 0) return RDB_OK;
    if (l.n > (1 << 30)) return RDB_ERR_TOO_LARGE;
    if (!l.param || !l.grad || !l.exp_avg || !l.exp_avg_sq || !l.step || !l.numel) return RDB_ERR_NULL;
    if ((param_dtype != RDB_F32 && param_dtype != RDB_BF16) || (grad_dtype != RDB_F32 && grad_dtype != RDB_BF16)) return RDB_ERR_DTYPE;
    if (state_bits != 32 && state_bits != 8) return RDB_ERR_DTYPE;
    if (state_bits == 8 && (!l.exp_avg_scale || !l.exp_avg_sq_scale)) return RDB_ERR_NULL;
    if (!(h->beta1 >= 0.0 && h->beta1 < 1.0 && h->beta2 >= 0.0 && h->beta2 < 1.0) || !(h->eps >= 0.0)) return RDB_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(h->lr_dev) | reinterpret_cast<uintptr_t>(grad_scale)) & 3) return RDB_ERR_ALIGN;
    const bool master = l.master != nullptr;
    if (master && param_dtype != RDB_BF16) return RDB_ERR_UNSUPPORTED;
    const uintptr_t pm = dtype_size(param_dtype) - 1, gm = dtype_size(grad_dtype) - 1, sm = state_bits == 8 ? 0 : 3;
    for (int64_t i = 0; i < l.n; ++i) {
        if (l.numel[i] < 0) return RDB_ERR_SHAPE;
        if (!l.step[i]) return RDB_ERR_NULL;
        if (l.numel[i] == 0) continue;
        if (!l.param[i] || !l.grad[i] || !l.exp_avg[i] || !l.exp_avg_sq[i] || (master && !l.master[i])) return RDB_ERR_NULL;
        if (state_bits == 8 && (!l.exp_avg_scale[i] || !l.exp_avg_sq_scale[i])) return RDB_ERR_NULL;
        if ((reinterpret_cast<uintptr_t>(l.param[i]) & pm) || (reinterpret_cast<uintptr_t>(l.grad[i]) & gm) || (reinterpret_cast<uintptr_t>(l.exp_avg[i]) & sm) ||
            (reinterpret_cast<uintptr_t>(l.exp_avg_sq[i]) & sm) || (master && (reinterpret_cast<uintptr_t>(l.master[i]) & 3)) ||
            (reinterpret_cast<uintptr_t>(l.step[i]) & 3) ||
            (state_bits == 8 && ((reinterpret_cast<uintptr_t>(l.exp_avg_scale[i]) | reinterpret_cast<uintptr_t>(l.exp_avg_sq_scale[i])) & 3)))
            return RDB_ERR_ALIGN;
    }
    cudaStream_t st = (cudaStream_t)stream;
    AdamwScalars s;
    s.b1 = (float)h->beta1;
    s.omb1 = (float)(1.0 - h->beta1);
    s.b2 = (float)h->beta2;
    s.omb2 = (float)(1.0 - h->beta2);
    s.eps = (float)h->eps;
    s.fast = h->eps >= FAST_EPS / sqrt(1.0 - h->beta2);               // inv_root is largest at the first step
    s.lr = h->lr;
    s.ln_beta1 = log(h->beta1);
    s.ln_beta2 = log(h->beta2);
    s.lr_dev = h->lr_dev;
    s.weight_decay = h->weight_decay;
    s.seed = h->seed;
    const bool b8 = state_bits == 8;
#define RDB_ADAMW(P, G, M) (b8 ? adamw_all<P, G, M, true>(l, s, grad_scale, st) : adamw_all<P, G, M, false>(l, s, grad_scale, st))
    if (param_dtype == RDB_F32) return grad_dtype == RDB_F32 ? RDB_ADAMW(float, float, false) : RDB_ADAMW(float, __nv_bfloat16, false);
    if (master) return grad_dtype == RDB_F32 ? RDB_ADAMW(__nv_bfloat16, float, true) : RDB_ADAMW(__nv_bfloat16, __nv_bfloat16, true);
    return grad_dtype == RDB_F32 ? RDB_ADAMW(__nv_bfloat16, float, false) : RDB_ADAMW(__nv_bfloat16, __nv_bfloat16, false);
#undef RDB_ADAMW
}

extern "C" size_t rdb_grad_norm_workspace_bytes(int n) {
    const int64_t launches = (n > 0 ? cdiv64(n, NT_LARGE) : 0) + 1;     // one more: the two types' lists are filled apart
    return (size_t)launches * RDB_NORM_BLOCKS * sizeof(double);
}

extern "C" int rdb_grad_norm(float *norm, float *coef, const void *const *grads, const int64_t *numels, const int32_t *dtypes, int n,
                             float max_norm, void *workspace, size_t workspace_bytes, void *stream) {
    if (n < 0) return RDB_ERR_SHAPE;
    if (!norm && !coef) return RDB_ERR_NULL;
    if (n > 0 && (!grads || !numels || !dtypes)) return RDB_ERR_NULL;
    if (coef && !(max_norm >= 0.0f)) return RDB_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < rdb_grad_norm_workspace_bytes(n) || (reinterpret_cast<uintptr_t>(workspace) & 7)) return RDB_ERR_WORKSPACE;
    for (int i = 0; i < n; ++i) {
        if (dtypes[i] != RDB_F32 && dtypes[i] != RDB_BF16) return RDB_ERR_DTYPE;
        if (numels[i] < 0) return RDB_ERR_SHAPE;
        if (numels[i] > 0 && !grads[i]) return RDB_ERR_NULL;
        if (reinterpret_cast<uintptr_t>(grads[i]) & (dtype_size(dtypes[i]) - 1)) return RDB_ERR_ALIGN;
    }
    cudaStream_t st = (cudaStream_t)stream;
    double *partial = reinterpret_cast<double *>(workspace);
    int filled = 0;
    GradRef part[NT_LARGE];
    for (int dtype = RDB_F32; dtype <= RDB_BF16; ++dtype) {       // one launch holds gradients of one type
        int k = 0;
        for (int i = 0; i <= n; ++i) {
            if (i < n && (dtypes[i] != dtype || numels[i] == 0)) continue;
            if (k == NT_LARGE || (i == n && k > 0)) {
                int used = 0, rc;
                if (dtype == RDB_F32)
                    rc = k <= NT_SMALL ? launch_sumsq<float, NT_SMALL>(part, k, partial + filled, &used, st)
                                       : launch_sumsq<float, NT_LARGE>(part, k, partial + filled, &used, st);
                else
                    rc = k <= NT_SMALL ? launch_sumsq<__nv_bfloat16, NT_SMALL>(part, k, partial + filled, &used, st)
                                       : launch_sumsq<__nv_bfloat16, NT_LARGE>(part, k, partial + filled, &used, st);
                if (rc) return rc;
                filled += used;
                k = 0;
            }
            if (i < n) {
                part[k++] = GradRef{grads[i], numels[i]};
            }
        }
    }
    return launch_pdl(norm_finish_kernel, dim3(1), 256, 0, st, norm, coef, (const double *)partial, filled, max_norm);
}
