// AdamW (decoupled weight decay) over many tensors in one launch.
//
//   g = grad / grad_div;  m = b1 m + (1-b1) g;  v = b2 v + (1-b2) g^2
//   p = p (1 - lr wd) - lr / (1-b1^t) * m / (sqrt(v) / sqrt(1-b2^t) + eps)
//
// Every product and sum is one rounded fp32 operation in this order (no fused
// multiply-add), so a step can be reproduced bit for bit operation by operation
// (with 8-bit states but for the last bit of a quotient now and then, see quot2).
// The states m, v and the masters of all tensors lie in flat buffers, each
// tensor from a multiple of 256 values on.  States in 8 bits are m and sqrt(v)
// as e4m3 values times one fp32 scale per 256 values (largest magnitude / 448):
// sqrt(v) keeps the moment's range within e4m3's, and one above zero is never
// stored as zero, so that the next step does not divide by eps alone.
//
// With 32-bit states HBM bounds the step: 312 M bf16 weights with masters take
// 1.31 ms, 103 % of the measured copy rate.  With 8-bit states (10 bytes a value
// instead of 28) it is the instructions, 41 a value at 70 % of the issue slots:
// 0.58 ms, 84 % of that rate.
#include <cstring>

#include <cuda_fp8.h>

#include "common.cuh"
#include "f32x2.cuh"

namespace usaf {

constexpr int kAdamBlock = 256;      // values per scale, and the unit of the tensors' places

// each constant twice, as the operand of an f32x2 instruction
struct AdamwConsts {
    uint64_t b1, omb1, b2, omb2, inv_root2, eps, neg_step, gmul, one, half, neg_one, huge;
    bool usual;                      // eps: update_fast
    bool spread_m, spread_v;         // rounding of the codes: encode
    uint32_t seed_m, seed_v;
};
static uint64_t twice(float v) {
    uint32_t u;
    std::memcpy(&u, &v, 4);
    return (uint64_t)u << 32 | u;
}

// the tensors of one launch, passed by value: nothing on the device to keep or to update
template <int N> struct AdamwTable {
    int32_t n;
    int32_t first[N + 1];            // first run of blocks of each tensor in this launch
    void *p[N];
    const void *g[N];
    int64_t numel[N];
    int64_t start[N];                // first 256-value block in the flat buffers
    float keep[N];                   // 1 - lr * weight decay
};

// the caller's host arrays from one tensor on
struct AdamwList {
    void *const *p;
    const void *const *g;
    const int64_t *numel, *start;
    const double *decay;
};

struct AdamwState {
    float *master;
    void *m, *v;
    float *m_scale, *v_scale;
};

// four e4m3 values as two pairs, and back
__device__ __forceinline__ void unpack_e4m3(uint32_t u, uint64_t *p) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u >> 16 * k), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        p[k] = pair(f.x, f.y);
    }
}
__device__ __forceinline__ uint32_t pack_e4m3(const uint64_t *p) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(halves(p[0]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(halves(p[1]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
// a value between two codes becomes the upper one where its fraction and a number in
// [0, 1) reach 1: 16 bits of r for two values each, the second's in reversed order
__device__ __forceinline__ uint32_t pack_e4m3_spread(const uint64_t *p, uint32_t r) {
    const float2 a = halves(p[0]), b = halves(p[1]);
    uint32_t d;
    asm("cvt.rs.satfinite.e4m3x4.f32 %0, {%1, %2, %3, %4}, %5;"
        : "=r"(d)
        : "f"(b.y), "f"(b.x), "f"(a.y), "f"(a.x), "r"(r));
    return d;
}

// 8 values of T from memory as 4 pairs, and back; one by one where the tensor is
// not aligned or ends within them
template <typename T> __device__ __forceinline__ void load8(const T *p, bool whole, int n, uint64_t *v) {
    if (whole) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            unpack<T>(reinterpret_cast<const uint4 *>(p)[i], v + i * kPairs<T>);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = pair(2 * i < n ? to_f(p[2 * i]) : 0.0f, 2 * i + 1 < n ? to_f(p[2 * i + 1]) : 0.0f);
    }
}
template <typename T> __device__ __forceinline__ void store8(T *p, bool whole, int n, const uint64_t *v) {
    if (whole) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(p)[i] = pack<T>(v + i * kPairs<T>);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = halves(v[i]);
            if (2 * i < n) p[2 * i] = from_f<T>(f.x);
            if (2 * i + 1 < n) p[2 * i + 1] = from_f<T>(f.y);
        }
    }
}

// a + b by a multiply-add with a 1 that comes with the launch: f32x2 additions of
// f32x2 products, and multiply-adds with a known 1, were fused with the products
// (observed: the weights came out as a fused multiply-add's)
__device__ __forceinline__ uint64_t sum2(uint64_t a, uint64_t b, uint64_t one) { return fma2(a, one, b); }

// Root and quotient by an approximation and one corrected step (Markstein's
// method: the residual of the first result by a fused multiply-add, times the
// approximate reciprocal), two at a time, with a third of the instructions of the
// correctly rounded ones, which bound the step with 8-bit states.
//
// The root is the nearest value for radicands from 2^-125 on (compared for all 2^23
// significands at an even and an odd exponent, at thirteen places of the range; below,
// the residual is too small for a number), and of zero.  The quotient is within 1/2 + 2^-20 units in the
// last place: the reciprocal is off by 2^-23 at most and the first quotient by
// 1.5 * 2^-23, so what the correction leaves is their product, 2.3 * 2^-46, and only
// quotients that lie so close to the middle of two values may become the farther
// one (for numerators below 2^-101, whose residuals have fewer bits, within 2^-22 of the
// quotient).  update_fast says where these are used.
__device__ __forceinline__ float rsqrt_approx(float v) {
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return fminf(r, 9.3e18f);        // 2^-126 has 9.2e18; a root of zero is zero times this
}
__device__ __forceinline__ float rcp_approx(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ uint64_t root2(const AdamwConsts &c, uint64_t v) {
    const float2 w = halves(v);
    const uint64_t y = pair(rsqrt_approx(w.x), rsqrt_approx(w.y));
    const uint64_t s = mul2(v, y);
    return fma2(fma2(mul2(s, c.neg_one), s, v), mul2(y, c.half), s);
}
__device__ __forceinline__ uint64_t quot2(const AdamwConsts &c, uint64_t a, uint64_t b) {
    const float2 w = halves(b);
    const uint64_t y = pair(rcp_approx(w.x), rcp_approx(w.y));
    const uint64_t q = mul2(a, y);
    return fma2(fma2(mul2(q, c.neg_one), b, a), y, q);
}
__device__ __forceinline__ float warp_top(float v) {     // largest magnitude of the warp
    float r;
    asm("redux.sync.max.abs.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// the moments of 8 values with a new gradient
__device__ __forceinline__ void moments(const AdamwConsts &c, const uint64_t *g, uint64_t *m, uint64_t *v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint64_t gk = mul2(g[k], c.gmul);
        m[k] = sum2(mul2(m[k], c.b1), mul2(gk, c.omb1), c.one);
        v[k] = sum2(mul2(v[k], c.b2), mul2(mul2(gk, c.omb2), gk), c.one);
    }
}

// p with the roots of v: the step's second half
__device__ __forceinline__ uint64_t stepped(const AdamwConsts &c, float keep, uint64_t p, uint64_t up) {
    return sum2(mul2(p, pair(keep, keep)), mul2(up, c.neg_step), c.one);
}

// the step of 8 values with correctly rounded operations; root, where it is kept, is
// the largest number where v is infinite (such a value takes a step of zero)
template <bool KEPT>
__device__ __forceinline__ void update(const AdamwConsts &c, float keep, uint64_t *p, const uint64_t *m, const uint64_t *v,
                                       uint64_t *root) {
    constexpr float kMost = 0x1.fffffep63f;          // sqrt of the largest fp32 value
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 w = halves(v[k]), h = halves(m[k]);
        const float rx = __fsqrt_rn(w.x), ry = __fsqrt_rn(w.y);
        const float2 den = halves(sum2(mul2(pair(rx, ry), c.inv_root2), c.eps, c.one));
        p[k] = stepped(c, keep, p[k], pair(__fdiv_rn(h.x, den.x), __fdiv_rn(h.y, den.y)));
        if (KEPT) root[k] = pair(rx > kMost ? kMost : rx, ry > kMost ? kMost : ry);      // NaN stays
    }
}

__device__ __forceinline__ float top_nan(float a, float b) {     // the larger one, NaN where one is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The fast step of a block with 8-bit states: p, the roots and the block's largest
// root.  False where it may have changed a bit beside the quotient's last, and the
// block has to be stepped again by update: it holds where the largest root is zero or
// 2^-44 and above, so that one whose square is below 2^-125 becomes the lowest code
// either way; eps is larger than 2^25 times what such a root adds to it (c.usual); no
// v is near the range's upper end (a root of infinity comes out as NaN).
__device__ __forceinline__ bool update_fast(const AdamwConsts &c, float keep, uint64_t *p, const uint64_t *m,
                                            const uint64_t *v, uint64_t *root, float &top) {
    top = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        root[k] = root2(c, v[k]);
        p[k] = stepped(c, keep, p[k], quot2(c, m[k], sum2(mul2(root[k], c.inv_root2), c.eps, c.one)));
        const float2 w = halves(root[k]);
        top = top_nan(top, top_nan(w.x, w.y));
    }
    asm("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(top));
    return c.usual && (top == 0.0f || (top >= 0x1p-44f && top < 0x1p63f));
}
// the largest number among the block's roots: NaN takes no part in its scale
__device__ __forceinline__ float top_root(const uint64_t *root) {
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 w = halves(root[k]);
        top = fmaxf(top, fmaxf(w.x, w.y));
    }
    return warp_top(top);
}

// m and v of a lane's 8 values from their e4m3 codes and the block's scales, and
// back: the scales are the warp's largest magnitudes (av, of the roots) / 448
struct Codes {
    uint2 m, v;
    float m_scale, v_scale;
};
__device__ __forceinline__ void decode(const Codes &q, uint64_t *m, uint64_t *v) {
    unpack_e4m3(q.m.x, m);
    unpack_e4m3(q.m.y, m + 2);
    unpack_e4m3(q.v.x, v);
    unpack_e4m3(q.v.y, v + 2);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        m[k] = mul2(m[k], pair(q.m_scale, q.m_scale));
        v[k] = mul2(v[k], pair(q.v_scale, q.v_scale));
        v[k] = mul2(v[k], v[k]);
    }
}
//
// Codes lie 1/16 to 1/8 of a value apart.  A step moves m by w = (1 - b) / (1 - b^t) of
// the way to the gradient (bias-corrected), the root of v by half of that at most, so
// while w is 1/8 or more the nearest codes follow.  Later most steps move a value by
// less than half the distance of two codes: rounded to the nearest, a root would never
// fall (beta2 = 0.999, half of a block's gradients 30 times smaller from some step on:
// 11 times the 32-bit root 5000 steps later) and m would stop at a part of its way.
// So a value then becomes the upper code as often as its place between the two asks
// for: its fraction plus a number of the step and the value's place in the tensor,
// where the numbers of one place's steps are evenly spread (multiples of a golden
// ratio's or the like, mod 1, their bits exchanged by a hash of the place; in reversed
// order the low bits of an odd number's multiples, which are even as well).  Nothing
// is drawn at random and a step repeats bit for bit.
__device__ __forceinline__ Codes encode(const AdamwConsts &c, const uint64_t *m, const uint64_t *root, float av,
                                        uint32_t quad) {
    float am = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 h = halves(m[k]);
        am = fmaxf(am, fmaxf(fabsf(h.x), fabsf(h.y)));
    }
    am = warp_top(am);
    const float mm = am >= 1e-30f ? __fmul_rn(__frcp_rn(am), 448.0f) : 0.0f;
    const float mv = av >= 1e-30f ? __fmul_rn(__frcp_rn(av), 448.0f) : 0.0f;
    // a root above zero (3e-23 at least, of the smallest fp32 value) becomes no
    // less than the lowest code, 2^-9
    const float least = mv > 0.0f ? 0.001953125f : 0.0f;
    uint64_t a[4], b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        a[k] = mul2(m[k], pair(mm, mm));
        const float2 q = halves(mul2(root[k], pair(mv, mv))), any = halves(mul2(root[k], c.huge));
        b[k] = pair(fmaxf(q.x, fminf(any.x, least)), fmaxf(q.y, fminf(any.y, least)));
    }
    Codes q;
    auto place = [quad](int k) {             // quad: the place in the tensor / 4
        const uint32_t h = (quad + k) * 0x9E3779B1u;
        return h ^ h >> 15;
    };
    if (c.spread_m)
        q.m = make_uint2(pack_e4m3_spread(a, c.seed_m ^ place(0)), pack_e4m3_spread(a + 2, c.seed_m ^ place(1)));
    else
        q.m = make_uint2(pack_e4m3(a), pack_e4m3(a + 2));
    if (c.spread_v)
        q.v = make_uint2(pack_e4m3_spread(b, c.seed_v ^ place(0)), pack_e4m3_spread(b + 2, c.seed_v ^ place(1)));
    else
        q.v = make_uint2(pack_e4m3(b), pack_e4m3(b + 2));
    q.m_scale = mm > 0.0f ? __fmul_rn(am, (float)(1.0 / 448.0)) : 0.0f;
    q.v_scale = mv > 0.0f ? __fmul_rn(av, (float)(1.0 / 448.0)) : 0.0f;
    return q;
}

// A lane's values of the blocks ahead, on their way into its own slots of shared
// memory (16 bytes a slot, neighbouring threads' side by side): weights, gradients,
// and the codes of m and v in one slot.
template <typename P, typename G> struct AdamRing {
    static constexpr int SP = sizeof(P) / 2, SG = sizeof(G) / 2, S = SP + SG + 1;
    static constexpr int D = S <= 3 ? 4 : 3;             // 192 to 240 bytes a thread
    static constexpr int kBytes = D * S * 16 * 256;
    uint32_t base;
    __device__ __forceinline__ static void copy(uint32_t to, const void *from, bool half) {
        if (half) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
        else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    }
    __device__ __forceinline__ static uint4 read(uint32_t at) {
        uint4 u;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                     : "r"(at));
        return u;
    }
    __device__ __forceinline__ void fetch(int stage, bool any, const P *p, const G *g, const void *m, const void *v) const {
        const uint32_t at = base + stage * (S * 16 * 256);
        if (any) {
#pragma unroll
            for (int i = 0; i < SP; ++i) copy(at + i * 4096, reinterpret_cast<const uint4 *>(p) + i, false);
#pragma unroll
            for (int i = 0; i < SG; ++i) copy(at + (SP + i) * 4096, reinterpret_cast<const uint4 *>(g) + i, false);
            copy(at + (SP + SG) * 4096, m, true);
            copy(at + (SP + SG) * 4096 + 8, v, true);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    __device__ __forceinline__ static void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory"); }
    __device__ __forceinline__ void get(int stage, uint64_t *p, uint64_t *g, Codes &q) const {
        const uint32_t at = base + stage * (S * 16 * 256);
#pragma unroll
        for (int i = 0; i < SP; ++i) unpack<P>(read(at + i * 4096), p + i * kPairs<P>);
#pragma unroll
        for (int i = 0; i < SG; ++i) unpack<G>(read(at + (SP + i) * 4096), g + i * kPairs<G>);
        const uint4 u = read(at + (SP + SG) * 4096);
        q.m = make_uint2(u.x, u.y);
        q.v = make_uint2(u.z, u.w);
    }
};
__device__ __forceinline__ void store_codes(const AdamwState &s, const Codes &q, int64_t f, int64_t blk, int lane) {
    *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(s.m) + f) = q.m;
    *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(s.v) + f) = q.v;
    if (lane == 0) {
        s.m_scale[blk] = q.m_scale;
        s.v_scale[blk] = q.v_scale;
    }
}

// a lane's weights and new moments of a block, from memory; n < 8: the tensor ends
// within them, and what lies behind its end takes no part and stays as it is
template <typename P, typename G, bool EIGHT, bool MASTER>
__device__ __forceinline__ void load_block(const AdamwConsts &c, const AdamwState &s, const P *pp, const G *gg, int64_t f,
                                           int64_t blk, int n, bool whole, uint64_t *p, uint64_t *m, uint64_t *v) {
    uint64_t g[4];
    load8<G>(gg, whole, n, g);
    if (MASTER) load8<float>(s.master + f, true, 8, p);
    else load8<P>(pp, whole, n, p);
    if (EIGHT) {
        Codes q;
        q.m = *reinterpret_cast<const uint2 *>(static_cast<uint8_t *>(s.m) + f);
        q.v = *reinterpret_cast<const uint2 *>(static_cast<uint8_t *>(s.v) + f);
        q.m_scale = s.m_scale[blk];
        q.v_scale = s.v_scale[blk];
        decode(q, m, v);
    } else {
        load8<float>(static_cast<float *>(s.m) + f, true, 8, m);
        load8<float>(static_cast<float *>(s.v) + f, true, 8, v);
    }
    if (n < 8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 x = halves(m[k]), y = halves(v[k]);
            m[k] = pair(2 * k < n ? x.x : 0.0f, 2 * k + 1 < n ? x.y : 0.0f);
            v[k] = pair(2 * k < n ? y.x : 0.0f, 2 * k + 1 < n ? y.y : 0.0f);
        }
    }
    moments(c, g, m, v);
}
template <typename P, bool MASTER>
__device__ __forceinline__ void store_weights(const AdamwState &s, P *pp, int64_t f, int n, bool whole, const uint64_t *p) {
    store8<P>(pp, whole, n, p);
    if (MASTER) store8<float>(s.master + f, n == 8, n, p);
}

__device__ __forceinline__ int values_left(int64_t numel, int64_t i) {      // of a lane's 8
    return numel - i >= 8 ? 8 : numel - i > 0 ? (int)(numel - i) : 0;
}

// A warp steps a run of up to `run` blocks of 256 values one after another, 8
// values a lane: every load of a warp is of whole sectors and a block's scales are
// its lanes' maximum.  With 8-bit states a block takes as long to compute as its
// few bytes take to arrive, so they are fetched D - 1 blocks ahead (loaded where
// they are used, the warps waited for half of the time), and the scales of the
// run's 16 blocks at most lie in its lanes.
template <int N, typename P, typename G, bool EIGHT, bool MASTER>
__global__ void __launch_bounds__(256, 3)
adamw_kernel(const __grid_constant__ AdamwTable<N> tab, const __grid_constant__ AdamwState s,
             const __grid_constant__ AdamwConsts c, const int run) {
    extern __shared__ uint4 dyn[];
    wait_for_previous();
    const int u = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (u >= tab.first[tab.n]) return;
    int lo = 0, hi = tab.n;          // the last tensor that starts at or before this run
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.first[mid] <= u) lo = mid;
        else hi = mid;
    }
    using PM = std::conditional_t<MASTER, float, P>;     // where the exact weight is
    const int64_t rel = (int64_t)(u - tab.first[lo]) * run, numel = tab.numel[lo];
    const int64_t i = rel * kAdamBlock + lane * 8;
    const int64_t blk = tab.start[lo] + rel, f = blk * kAdamBlock + lane * 8;
    P *const p0 = static_cast<P *>(tab.p[lo]) + i;
    const G *const g0 = static_cast<const G *>(tab.g[lo]) + i;
    const float keep = tab.keep[lo];
    const uint32_t quad = (uint32_t)(i >> 2);
    const bool aligned = (((uintptr_t)p0 | (uintptr_t)g0) & 15) == 0;
    const int64_t left = (numel + kAdamBlock - 1) / kAdamBlock - rel;
    const int blocks = (int)(left < run ? left : run);
    uint32_t again = 0;              // blocks that update_fast does not hold for: bit r, of 16 at most
    if (EIGHT && aligned && numel - rel * kAdamBlock >= (int64_t)blocks * kAdamBlock) {
        using Ring = AdamRing<PM, G>;
        Ring ring;
        ring.base = (uint32_t)__cvta_generic_to_shared(dyn + threadIdx.x);
        const PM *from;
        if constexpr (MASTER) from = s.master + f;
        else from = p0;
        const uint8_t *m8 = static_cast<const uint8_t *>(s.m) + f, *v8 = static_cast<const uint8_t *>(s.v) + f;
        auto fetch = [&](int stage, int r) {
            const int64_t at = (int64_t)r * kAdamBlock;
            ring.fetch(stage, r < blocks, from + at, g0 + at, m8 + at, v8 + at);
        };
#pragma unroll
        for (int d = 0; d < Ring::D - 1; ++d) fetch(d, d);
        float scale = 0.0f;          // lanes 0-15: of m, 16-31: of v
        if ((lane & 15) < blocks) scale = (lane < 16 ? s.m_scale : s.v_scale)[blk + (lane & 15)];
        int stage = 0;
        P *pp = p0;
        int64_t at = f, b = blk;
        for (int r = 0; r < blocks; ++r) {
            fetch(stage == 0 ? Ring::D - 1 : stage - 1, r + Ring::D - 1);
            Ring::wait();
            uint64_t p[4], g[4], m[4], v[4], root[4];
            Codes q;
            ring.get(stage, p, g, q);
            q.m_scale = __shfl_sync(0xffffffffu, scale, r);
            q.v_scale = __shfl_sync(0xffffffffu, scale, 16 + r);
            decode(q, m, v);
            moments(c, g, m, v);
            float av;
            if (update_fast(c, keep, p, m, v, root, av)) {
                store_weights<P, MASTER>(s, pp, at, 8, true, p);
                store_codes(s, encode(c, m, root, av, quad + r * (kAdamBlock / 4)), at, b, lane);
            } else {
                again |= 1u << r;
            }
            stage = stage == Ring::D - 1 ? 0 : stage + 1;
            pp += kAdamBlock;
            at += kAdamBlock;
            ++b;
        }
    } else {
        for (int r = 0; r < blocks; ++r) {
            const int64_t at = (int64_t)r * kAdamBlock;
            const int n = values_left(numel, i + at);
            const bool whole = aligned && n == 8;
            uint64_t p[4], m[4], v[4], root[4];
            float av;
            load_block<P, G, EIGHT, MASTER>(c, s, p0 + at, g0 + at, f + at, blk + r, n, whole, p, m, v);
            if constexpr (EIGHT) {
                if (update_fast(c, keep, p, m, v, root, av)) {
                    store_weights<P, MASTER>(s, p0 + at, f + at, n, whole, p);
                    store_codes(s, encode(c, m, root, av, quad + r * (kAdamBlock / 4)), f + at, blk + r, lane);
                } else {
                    again |= 1u << r;
                }
            } else {
                update<false>(c, keep, p, m, v, root);
                store_weights<P, MASTER>(s, p0 + at, f + at, n, whole, p);
                store8<float>(static_cast<float *>(s.m) + f + at, n == 8, n, m);
                store8<float>(static_cast<float *>(s.v) + f + at, n == 8, n, v);
            }
        }
    }
    if constexpr (EIGHT) {
        for (; again; again &= again - 1) {          // rare, from the beginning: nothing of the block is stored yet
            const int r = __ffs(again) - 1;
            const int64_t at = (int64_t)r * kAdamBlock;
            const int n = values_left(numel, i + at);
            const bool whole = aligned && n == 8;
            uint64_t p[4], m[4], v[4], root[4];
            load_block<P, G, true, MASTER>(c, s, p0 + at, g0 + at, f + at, blk + r, n, whole, p, m, v);
            update<true>(c, keep, p, m, v, root);
            store_weights<P, MASTER>(s, p0 + at, f + at, n, whole, p);
            store_codes(s, encode(c, m, root, top_root(root), quad + r * (kAdamBlock / 4)), f + at, blk + r, lane);
        }
    }
}

template <int N, typename P, typename G, bool EIGHT, bool MASTER>
static int adamw_start(const AdamwTable<N> &tab, const AdamwState &s, const AdamwConsts &c, int run, cudaStream_t st) {
    auto kernel = adamw_kernel<N, P, G, EIGHT, MASTER>;
    const int smem = EIGHT ? AdamRing<std::conditional_t<MASTER, float, P>, G>::kBytes : 0;
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
        (void)cudaGetLastError();
        return USAF_ECUDA;
    }
    return launch_early(kernel, dim3(cdiv(tab.first[tab.n], 8)), 256, smem, st, tab, s, c, run) ? USAF_OK : USAF_ECUDA;
}

template <int N, typename P, typename G, bool EIGHT>
static int adamw_launch(const AdamwList &t, int at, int n, double lr, const AdamwState &s, const AdamwConsts &c,
                        cudaStream_t st) {
    AdamwTable<N> tab;
    int64_t values = 0, runs = 0;
    for (int i = 0; i < n; ++i) values += t.numel[at + i];
    // A warp looks its place up once for a run of up to 16 blocks (4 with 32-bit
    // states, which have no ring to fill), where that leaves the GPU (148 SMs of 24
    // warps) eight runs for each of its warps
    int run = 1;
    while (run < (EIGHT ? 16 : 4) && values >= (int64_t)kAdamBlock * 2 * run * 148 * 24 * 8) run *= 2;
    tab.n = n;
    for (int i = 0; i < n; ++i) {
        tab.first[i] = (int32_t)runs;
        tab.p[i] = t.p[at + i];
        tab.g[i] = t.g[at + i];
        tab.numel[i] = t.numel[at + i];
        tab.start[i] = t.start[at + i] / kAdamBlock;
        tab.keep[i] = (float)(1.0 - lr * t.decay[at + i]);
        runs += (t.numel[at + i] + kAdamBlock * run - 1) / (kAdamBlock * run);
        if (runs > 0x7fffffff) return USAF_EUNSUPPORTED;
    }
    tab.first[n] = (int32_t)runs;
    if (runs == 0) return USAF_OK;
    return s.master ? adamw_start<N, P, G, EIGHT, true>(tab, s, c, run, st)
                    : adamw_start<N, P, G, EIGHT, false>(tab, s, c, run, st);
}

template <typename P, typename G>
static int adamw_all(const AdamwList &t, int n, bool eight, double lr, const AdamwState &s,
                     const AdamwConsts &c, cudaStream_t st) {
    constexpr int kFew = 64, kMost = 640;    // 3 or 26 KB of the 32 KB that a launch takes by value
    for (int at = 0; at < n; at += kMost) {
        const int k = std::min(kMost, n - at);
        int rc;
        if (k <= kFew)
            rc = eight ? adamw_launch<kFew, P, G, true>(t, at, k, lr, s, c, st)
                       : adamw_launch<kFew, P, G, false>(t, at, k, lr, s, c, st);
        else
            rc = eight ? adamw_launch<kMost, P, G, true>(t, at, k, lr, s, c, st)
                       : adamw_launch<kMost, P, G, false>(t, at, k, lr, s, c, st);
        if (rc) return rc;
    }
    return USAF_OK;
}

}  // namespace usaf

using namespace usaf;

extern "C" int usaf_adamw(int32_t n_tensors, void *const *p, const void *const *g, const int64_t *numel,
                          const int64_t *start, const double *weight_decay, int32_t p_dtype, int32_t g_dtype,
                          float *master, int32_t bits, void *m, void *v, float *m_scale, float *v_scale,
                          double grad_div, int32_t step, double lr, double beta1, double beta2, double eps,
                          void *stream) {
    USAF_REQUIRE(n_tensors >= 0 && step >= 1 && (bits == 32 || bits == 8) && grad_div != 0.0);
    if (n_tensors == 0) return USAF_OK;
    USAF_REQUIRE(p && g && numel && start && weight_decay && m && v && (bits == 32 || (m_scale && v_scale)));
    USAF_REQUIRE((((uintptr_t)m | (uintptr_t)v | (uintptr_t)master) & 15) == 0);
    for (int i = 0; i < n_tensors; ++i)
        USAF_REQUIRE(numel[i] >= 0 && (numel[i] == 0 || (p[i] && g[i])) && start[i] >= 0 && start[i] % kAdamBlock == 0);
    const AdamwList tensors{p, g, numel, start, weight_decay};
    AdamwConsts c;
    c.b1 = twice((float)beta1);
    c.omb1 = twice((float)(1.0 - beta1));
    c.b2 = twice((float)beta2);
    c.omb2 = twice((float)(1.0 - beta2));
    const double inv_root2 = 1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step));
    c.inv_root2 = twice((float)inv_root2);
    c.usual = eps >= inv_root2 * 0x1p-37 && eps <= 0x1p60;     // a root of 2^-62.5 vanishes beside eps
    // codes are spread from the step on where a new gradient's weight is below 1/8
    // (encode); the multipliers, all odd: 2^16 times 0.6180, the golden ratio's inverse, and
    // 0.7549 and 0.5698, the inverse of the root of x^3 = x + 1 and its square
    const auto weight = [step](double b) { return (1.0 - b) / (1.0 - std::pow(b, (double)step)); };
    const auto seed = [step](uint32_t lo, uint32_t hi) {
        return (((uint32_t)step * lo) & 0xffffu) | ((uint32_t)step * hi) << 16;
    };
    c.spread_m = weight(beta1) < 0.125;
    c.spread_v = weight(beta2) < 0.125;
    c.seed_m = seed(0x91E1u, 0x9E37u);
    c.seed_v = seed(0x9E37u, 0xC13Fu);
    c.eps = twice((float)eps);
    c.neg_step = twice(-(float)(lr / (1.0 - std::pow(beta1, (double)step))));
    c.gmul = twice((float)(1.0 / grad_div));
    c.one = twice(1.0f);
    c.half = twice(0.5f);
    c.neg_one = twice(-1.0f);
    c.huge = twice(1e30f);
    const AdamwState s{master, m, v, m_scale, v_scale};
    const bool eight = bits == 8;
    cudaStream_t st = as_stream(stream);
    switch (p_dtype * 4 + g_dtype) {
        case USAF_F32 * 4 + USAF_F32: return adamw_all<float, float>(tensors, n_tensors, eight, lr, s, c, st);
        case USAF_BF16 * 4 + USAF_BF16: return adamw_all<__nv_bfloat16, __nv_bfloat16>(tensors, n_tensors, eight, lr, s, c, st);
        case USAF_BF16 * 4 + USAF_F32: return adamw_all<__nv_bfloat16, float>(tensors, n_tensors, eight, lr, s, c, st);
        case USAF_F16 * 4 + USAF_F16: return adamw_all<__half, __half>(tensors, n_tensors, eight, lr, s, c, st);
        case USAF_F16 * 4 + USAF_F32: return adamw_all<__half, float>(tensors, n_tensors, eight, lr, s, c, st);
        default: return USAF_EINVAL;
    }
}
