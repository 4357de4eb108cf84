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
#include <cuda_fp8.h>

#include "common.cuh"
#include "f32x2.cuh"

namespace usaf {

constexpr int kAdamBlock = 256;      // values per scale, and the unit of the tensors' places

struct AdamwConsts {
    float b1, omb1, b2, omb2, inv_root2, eps, step_size, gmul;
};

// the tensors of one launch, passed by value: nothing on the device to keep or to update
template <int N> struct AdamwTable {
    int32_t n;
    int32_t first[N + 1];            // first 256-value block of each tensor in this launch
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

// a + b by scalar additions: an f32x2 addition of f32x2 products was fused with
// them (observed: the weights came out as a fused multiply-add's)
__device__ __forceinline__ uint64_t sum2(uint64_t a, uint64_t b) {
    const float2 x = halves(a), y = halves(b);
    return pair(__fadd_rn(x.x, y.x), __fadd_rn(x.y, y.y));
}

// A warp steps one block of 256 values, 8 a lane: every load of a warp is of
// whole sectors, all of a block's loads are on their way at once, and a block's
// scales are its lanes' maximum.
template <int N, typename P, typename G, bool EIGHT, bool MASTER>
__global__ void __launch_bounds__(256)
adamw_kernel(const __grid_constant__ AdamwTable<N> tab, const AdamwState s, const AdamwConsts c) {
    const int b = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (b >= tab.first[tab.n]) return;
    int lo = 0, hi = tab.n;          // the last tensor that starts at or before this block
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.first[mid] <= b) lo = mid;
        else hi = mid;
    }
    const int64_t rel = b - tab.first[lo], i = rel * kAdamBlock + lane * 8;
    const int64_t blk = tab.start[lo] + rel, f = blk * kAdamBlock + lane * 8;
    P *pp = static_cast<P *>(tab.p[lo]) + i;
    const G *gg = static_cast<const G *>(tab.g[lo]) + i;
    const int n = (int)max((int64_t)0, min((int64_t)8, tab.numel[lo] - i));
    const bool whole = n == 8 && (((uintptr_t)pp | (uintptr_t)gg) & 15) == 0;
    uint64_t p[4], g[4], m[4], v[4];
    load8<G>(gg, whole, n, g);
    if (MASTER) load8<float>(s.master + f, true, 8, p);
    else load8<P>(pp, whole, n, p);
    if (EIGHT) {
        const uint2 qm = *reinterpret_cast<const uint2 *>(static_cast<uint8_t *>(s.m) + f);
        const uint2 qv = *reinterpret_cast<const uint2 *>(static_cast<uint8_t *>(s.v) + f);
        const float sm = s.m_scale[blk], sv = s.v_scale[blk];
        unpack_e4m3(qm.x, m);
        unpack_e4m3(qm.y, m + 2);
        unpack_e4m3(qv.x, v);
        unpack_e4m3(qv.y, v + 2);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            m[k] = mul2(m[k], pair(sm, sm));
            v[k] = mul2(v[k], pair(sv, sv));
            v[k] = mul2(v[k], v[k]);
        }
    } else {
        load8<float>(static_cast<float *>(s.m) + f, true, 8, m);
        load8<float>(static_cast<float *>(s.v) + f, true, 8, v);
    }
    if (n < 8) {                     // what lies behind a tensor's end takes no part
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 a = halves(m[k]), b2 = halves(v[k]);
            m[k] = pair(2 * k < n ? a.x : 0.0f, 2 * k + 1 < n ? a.y : 0.0f);
            v[k] = pair(2 * k < n ? b2.x : 0.0f, 2 * k + 1 < n ? b2.y : 0.0f);
        }
    }
    const float keep = tab.keep[lo];
    uint64_t root[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        g[k] = mul2(g[k], pair(c.gmul, c.gmul));
        m[k] = sum2(mul2(m[k], pair(c.b1, c.b1)), mul2(g[k], pair(c.omb1, c.omb1)));
        v[k] = sum2(mul2(v[k], pair(c.b2, c.b2)), mul2(mul2(g[k], pair(c.omb2, c.omb2)), g[k]));
        const float2 w = halves(v[k]);
        root[k] = pair(__fsqrt_rn(w.x), __fsqrt_rn(w.y));
        const float2 den = halves(sum2(mul2(root[k], pair(c.inv_root2, c.inv_root2)), pair(c.eps, c.eps)));
        const float2 h = halves(m[k]);
        const uint64_t up = pair(__fdiv_rn(h.x, den.x), __fdiv_rn(h.y, den.y));
        p[k] = sum2(mul2(p[k], pair(keep, keep)), mul2(up, pair(-c.step_size, -c.step_size)));
    }
    store8<P>(pp, whole, n, p);
    if (n == 8) {
        if (MASTER) store8<float>(s.master + f, true, 8, p);
        if (!EIGHT) {
            store8<float>(static_cast<float *>(s.m) + f, true, 8, m);
            store8<float>(static_cast<float *>(s.v) + f, true, 8, v);
        }
    } else {                         // the values behind a tensor's end stay as they are
        if (MASTER) store8<float>(s.master + f, false, n, p);
        if (!EIGHT) {
            store8<float>(static_cast<float *>(s.m) + f, false, n, m);
            store8<float>(static_cast<float *>(s.v) + f, false, n, v);
        }
    }
    if (!EIGHT) return;
    float am = 0.0f, av = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 h = halves(m[k]), w = halves(root[k]);
        am = fmaxf(am, fmaxf(fabsf(h.x), fabsf(h.y)));
        av = fmaxf(av, fmaxf(w.x, w.y));
    }
    am = warp_max(am);
    av = warp_max(av);
    const float mm = am >= 1e-30f ? __fmul_rn(__frcp_rn(am), 448.0f) : 0.0f;
    const float mv = av >= 1e-30f ? __fmul_rn(__frcp_rn(av), 448.0f) : 0.0f;
    // below the lowest code 2^-9 a root above zero becomes that
    const float least = mv > 0.0f ? 0.001953125f : 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        m[k] = mul2(m[k], pair(mm, mm));
        const float2 w = halves(root[k]), q = halves(mul2(root[k], pair(mv, mv)));
        root[k] = pair(w.x > 0.0f ? fmaxf(q.x, least) : q.x, w.y > 0.0f ? fmaxf(q.y, least) : q.y);
    }
    *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(s.m) + f) = make_uint2(pack_e4m3(m), pack_e4m3(m + 2));
    *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(s.v) + f) = make_uint2(pack_e4m3(root), pack_e4m3(root + 2));
    if (lane == 0) {
        s.m_scale[blk] = mm > 0.0f ? __fmul_rn(am, (float)(1.0 / 448.0)) : 0.0f;
        s.v_scale[blk] = mv > 0.0f ? __fmul_rn(av, (float)(1.0 / 448.0)) : 0.0f;
    }
}

template <int N, typename P, typename G, bool EIGHT>
static int adamw_launch(const AdamwList &t, int at, int n, double lr, const AdamwState &s, const AdamwConsts &c,
                        cudaStream_t st) {
    AdamwTable<N> tab;
    int64_t blocks = 0;
    tab.n = n;
    for (int i = 0; i < n; ++i) {
        tab.first[i] = (int32_t)blocks;
        tab.p[i] = t.p[at + i];
        tab.g[i] = t.g[at + i];
        tab.numel[i] = t.numel[at + i];
        tab.start[i] = t.start[at + i] / kAdamBlock;
        tab.keep[i] = (float)(1.0 - lr * t.decay[at + i]);
        blocks += (t.numel[at + i] + kAdamBlock - 1) / kAdamBlock;
        if (blocks > 0x7fffffff) return USAF_EUNSUPPORTED;
    }
    tab.first[n] = (int32_t)blocks;
    if (blocks == 0) return USAF_OK;
    const unsigned grid = cdiv(blocks, 8);
    if (s.master) adamw_kernel<N, P, G, EIGHT, true><<<grid, 256, 0, st>>>(tab, s, c);
    else adamw_kernel<N, P, G, EIGHT, false><<<grid, 256, 0, st>>>(tab, s, c);
    USAF_CHECK_LAUNCH();
    return USAF_OK;
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
    c.b1 = (float)beta1;
    c.omb1 = (float)(1.0 - beta1);
    c.b2 = (float)beta2;
    c.omb2 = (float)(1.0 - beta2);
    c.inv_root2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
    c.eps = (float)eps;
    c.step_size = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    c.gmul = (float)(1.0 / grad_div);
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
