// AdamW (decoupled weight decay) over many tensors in one launch.
//
//   g = grad / grad_div;  m = b1 m + (1-b1) g;  v = b2 v + (1-b2) g^2
//   p = p (1 - lr wd) - lr / (1-b1^t) * m / (sqrt(v) / sqrt(1-b2^t) + eps)
//
// Every product and sum is one rounded fp32 operation in this order (no fused
// multiply-add), so a step can be reproduced bit for bit operation by operation.
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
// approximate reciprocal), two at a time.  Equal to the correctly rounded ones
// for every significand (2^24 of each of eleven exponents compared) down to a
// radicand of 2^-125, below which the residual is too small for a number; with a
// third of the instructions, which bound the step with 8-bit states.
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

// the step of 8 values: p, m and v are replaced, root is the new sqrt(v)
template <bool EIGHT>
__device__ __forceinline__ void step8(const AdamwConsts &c, float keep, uint64_t *g, uint64_t *p, uint64_t *m,
                                      uint64_t *v, uint64_t *root) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint64_t gk = mul2(g[k], c.gmul);
        m[k] = sum2(mul2(m[k], c.b1), mul2(gk, c.omb1), c.one);
        v[k] = sum2(mul2(v[k], c.b2), mul2(mul2(gk, c.omb2), gk), c.one);
        uint64_t up;
        if (EIGHT) {
            root[k] = root2(c, v[k]);
            up = quot2(c, m[k], sum2(mul2(root[k], c.inv_root2), c.eps, c.one));
        } else {
            const float2 w = halves(v[k]), h = halves(m[k]);
            root[k] = pair(__fsqrt_rn(w.x), __fsqrt_rn(w.y));
            const float2 den = halves(sum2(mul2(root[k], c.inv_root2), c.eps, c.one));
            up = pair(__fdiv_rn(h.x, den.x), __fdiv_rn(h.y, den.y));
        }
        p[k] = sum2(mul2(p[k], pair(keep, keep)), mul2(up, c.neg_step), c.one);
    }
}

// m and v of a lane's 8 values from their e4m3 codes and the block's scales, and
// back: the scales are the warp's largest magnitudes / 448
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
__device__ __forceinline__ Codes encode(const AdamwConsts &c, const uint64_t *m, const uint64_t *root) {
    float am = 0.0f, av = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 h = halves(m[k]), w = halves(root[k]);
        am = fmaxf(am, fmaxf(fabsf(h.x), fabsf(h.y)));
        av = fmaxf(av, fmaxf(w.x, w.y));
    }
    am = warp_top(am);
    av = warp_top(av);
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
    q.m = make_uint2(pack_e4m3(a), pack_e4m3(a + 2));
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

// A warp steps a run of up to `run` blocks of 256 values one after another, 8
// values a lane: every load of a warp is of whole sectors and a block's scales are
// its lanes' maximum.  With 8-bit states a block takes as long to compute as its
// few bytes take to arrive, so they are fetched D - 1 blocks ahead (loaded where
// they are used, the warps waited for half of the time), and the scales of the
// run's 16 blocks at most lie in its lanes.
template <int N, typename P, typename G, bool EIGHT, bool MASTER>
__global__ void __launch_bounds__(256, 3)
adamw_kernel(const __grid_constant__ AdamwTable<N> tab, const AdamwState s, const AdamwConsts c, const int run) {
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
    int64_t i = rel * kAdamBlock + lane * 8;
    int64_t blk = tab.start[lo] + rel, f = blk * kAdamBlock + lane * 8;
    P *pp = static_cast<P *>(tab.p[lo]) + i;
    const G *gg = static_cast<const G *>(tab.g[lo]) + i;
    const float keep = tab.keep[lo];
    const bool aligned = (((uintptr_t)pp | (uintptr_t)gg) & 15) == 0;
    const int64_t left = (numel + kAdamBlock - 1) / kAdamBlock - rel;
    const int blocks = (int)(left < run ? left : run);
    if (EIGHT && aligned && numel - rel * kAdamBlock >= (int64_t)blocks * kAdamBlock) {
        using Ring = AdamRing<PM, G>;
        Ring ring;
        ring.base = (uint32_t)__cvta_generic_to_shared(dyn + threadIdx.x);
        const PM *from;
        if constexpr (MASTER) from = s.master + f;
        else from = pp;
        const uint8_t *m8 = static_cast<const uint8_t *>(s.m) + f, *v8 = static_cast<const uint8_t *>(s.v) + f;
        auto fetch = [&](int stage, int r) {
            const int64_t at = (int64_t)r * kAdamBlock;
            ring.fetch(stage, r < blocks, from + at, gg + at, m8 + at, v8 + at);
        };
#pragma unroll
        for (int d = 0; d < Ring::D - 1; ++d) fetch(d, d);
        float scale = 0.0f;          // lanes 0-15: of m, 16-31: of v
        if ((lane & 15) < blocks) scale = (lane < 16 ? s.m_scale : s.v_scale)[blk + (lane & 15)];
        int stage = 0;
        for (int r = 0; r < blocks; ++r) {
            fetch(stage == 0 ? Ring::D - 1 : stage - 1, r + Ring::D - 1);
            Ring::wait();
            uint64_t p[4], g[4], m[4], v[4], root[4];
            Codes q;
            ring.get(stage, p, g, q);
            q.m_scale = __shfl_sync(0xffffffffu, scale, r);
            q.v_scale = __shfl_sync(0xffffffffu, scale, 16 + r);
            decode(q, m, v);
            step8<true>(c, keep, g, p, m, v, root);
            store8<P>(pp, true, 8, p);
            if (MASTER) store8<float>(s.master + f, true, 8, p);
            store_codes(s, encode(c, m, root), f, blk, lane);
            stage = stage == Ring::D - 1 ? 0 : stage + 1;
            pp += kAdamBlock;
            f += kAdamBlock;
            ++blk;
        }
        return;
    }
    for (int r = 0; r < blocks; ++r) {
        const int n = numel - i >= 8 ? 8 : numel - i > 0 ? (int)(numel - i) : 0;
        const bool whole = aligned && n == 8;
        float *m32 = static_cast<float *>(s.m) + f, *v32 = static_cast<float *>(s.v) + f;
        uint64_t p[4], g[4], m[4], v[4], root[4];
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
            load8<float>(m32, true, 8, m);
            load8<float>(v32, true, 8, v);
        }
        if (n < 8) {                 // what lies behind a tensor's end takes no part
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 x = halves(m[k]), y = halves(v[k]);
                m[k] = pair(2 * k < n ? x.x : 0.0f, 2 * k + 1 < n ? x.y : 0.0f);
                v[k] = pair(2 * k < n ? y.x : 0.0f, 2 * k + 1 < n ? y.y : 0.0f);
            }
        }
        step8<EIGHT>(c, keep, g, p, m, v, root);
        store8<P>(pp, whole, n, p);
        // the values behind a tensor's end stay as they are
        if (MASTER) store8<float>(s.master + f, n == 8, n, p);
        if (EIGHT) {
            store_codes(s, encode(c, m, root), f, blk, lane);
        } else {
            store8<float>(m32, n == 8, n, m);
            store8<float>(v32, n == 8, n, v);
        }
        pp += kAdamBlock;
        gg += kAdamBlock;
        f += kAdamBlock;
        i += kAdamBlock;
        ++blk;
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
    c.inv_root2 = twice((float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step))));
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
