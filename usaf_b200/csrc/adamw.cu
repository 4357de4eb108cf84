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

struct AdamwState {
    float *master;
    void *m, *v;
    float *m_scale, *v_scale;
};

__device__ __forceinline__ float e4m3_to_f(uint8_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}
__device__ __forceinline__ uint8_t f_to_e4m3(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }

template <int N, typename P, typename G, bool EIGHT>
__global__ void __launch_bounds__(256)
adamw_kernel(const __grid_constant__ AdamwTable<N> tab, const AdamwState s, const AdamwConsts c) {
    __shared__ float red[2][8];
    int lo = 0, hi = tab.n;          // the last tensor that starts at or before this block
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.first[mid] <= (int)blockIdx.x) lo = mid;
        else hi = mid;
    }
    const int64_t rel = blockIdx.x - tab.first[lo], i = rel * kAdamBlock + threadIdx.x;
    const int64_t blk = tab.start[lo] + rel, f = blk * kAdamBlock + threadIdx.x;
    const bool in = i < tab.numel[lo];
    P *pp = static_cast<P *>(tab.p[lo]) + i;
    float g = 0.0f, p = 0.0f, m = 0.0f, v = 0.0f;
    if (in) {
        g = __fmul_rn(to_f(static_cast<const G *>(tab.g[lo])[i]), c.gmul);
        p = s.master ? s.master[f] : to_f(*pp);
        if (EIGHT) {
            m = __fmul_rn(e4m3_to_f(static_cast<uint8_t *>(s.m)[f]), s.m_scale[blk]);
            v = __fmul_rn(e4m3_to_f(static_cast<uint8_t *>(s.v)[f]), s.v_scale[blk]);
            v = __fmul_rn(v, v);
        } else {
            m = static_cast<float *>(s.m)[f];
            v = static_cast<float *>(s.v)[f];
        }
    }
    m = __fadd_rn(__fmul_rn(m, c.b1), __fmul_rn(g, c.omb1));
    v = __fadd_rn(__fmul_rn(v, c.b2), __fmul_rn(__fmul_rn(g, c.omb2), g));
    const float root = __fsqrt_rn(v);
    const float den = __fadd_rn(__fmul_rn(root, c.inv_root2), c.eps);
    p = __fsub_rn(__fmul_rn(p, tab.keep[lo]), __fmul_rn(__fdiv_rn(m, den), c.step_size));
    if (in) {
        if (s.master) s.master[f] = p;
        *pp = from_f<P>(p);
    }
    if (!EIGHT) {
        if (in) {
            static_cast<float *>(s.m)[f] = m;
            static_cast<float *>(s.v)[f] = v;
        }
        return;
    }
    float am = warp_max(fabsf(m)), av = warp_max(root);
    if ((threadIdx.x & 31) == 0) {
        red[0][threadIdx.x >> 5] = am;
        red[1][threadIdx.x >> 5] = av;
    }
    __syncthreads();
    am = av = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        am = fmaxf(am, red[0][k]);
        av = fmaxf(av, red[1][k]);
    }
    const float mm = am >= 1e-30f ? __fmul_rn(__frcp_rn(am), 448.0f) : 0.0f;
    const float mv = av >= 1e-30f ? __fmul_rn(__frcp_rn(av), 448.0f) : 0.0f;
    uint8_t qv = f_to_e4m3(__fmul_rn(root, mv));
    if (qv == 0 && root > 0.0f && mv > 0.0f) qv = 1;
    static_cast<uint8_t *>(s.m)[f] = f_to_e4m3(__fmul_rn(m, mm));
    static_cast<uint8_t *>(s.v)[f] = qv;
    if (threadIdx.x == 0) {
        s.m_scale[blk] = mm > 0.0f ? __fmul_rn(am, (float)(1.0 / 448.0)) : 0.0f;
        s.v_scale[blk] = mv > 0.0f ? __fmul_rn(av, (float)(1.0 / 448.0)) : 0.0f;
    }
}

template <int N, typename P, typename G, bool EIGHT>
static int adamw_launch(const usaf_adamw_tensor *t, int n, double lr, const AdamwState &s, const AdamwConsts &c,
                        cudaStream_t st) {
    AdamwTable<N> tab;
    int64_t blocks = 0;
    tab.n = n;
    for (int i = 0; i < n; ++i) {
        tab.first[i] = (int32_t)blocks;
        tab.p[i] = t[i].p;
        tab.g[i] = t[i].g;
        tab.numel[i] = t[i].numel;
        tab.start[i] = t[i].start / kAdamBlock;
        tab.keep[i] = (float)(1.0 - lr * t[i].weight_decay);
        blocks += (t[i].numel + kAdamBlock - 1) / kAdamBlock;
        if (blocks > 0x7fffffff) return USAF_EUNSUPPORTED;
    }
    tab.first[n] = (int32_t)blocks;
    if (blocks == 0) return USAF_OK;
    adamw_kernel<N, P, G, EIGHT><<<(unsigned)blocks, 256, 0, st>>>(tab, s, c);
    USAF_CHECK_LAUNCH();
    return USAF_OK;
}

template <typename P, typename G>
static int adamw_all(const usaf_adamw_tensor *t, int n, bool eight, double lr, const AdamwState &s,
                     const AdamwConsts &c, cudaStream_t st) {
    constexpr int kMost = 640;       // 26 KB of the 32 KB that a launch takes by value
    for (int at = 0; at < n; at += kMost) {
        const int k = std::min(kMost, n - at);
        const int rc = eight ? adamw_launch<kMost, P, G, true>(t + at, k, lr, s, c, st)
                             : adamw_launch<kMost, P, G, false>(t + at, k, lr, s, c, st);
        if (rc) return rc;
    }
    return USAF_OK;
}

}  // namespace usaf

using namespace usaf;

extern "C" int usaf_adamw(const usaf_adamw_tensor *tensors, int32_t n_tensors, int32_t p_dtype, int32_t g_dtype,
                          float *master, int32_t bits, void *m, void *v, float *m_scale, float *v_scale,
                          double grad_div, int32_t step, double lr, double beta1, double beta2, double eps,
                          void *stream) {
    USAF_REQUIRE(n_tensors >= 0 && step >= 1 && (bits == 32 || bits == 8) && grad_div != 0.0);
    if (n_tensors == 0) return USAF_OK;
    USAF_REQUIRE(tensors && m && v && (bits == 32 || (m_scale && v_scale)));
    for (int i = 0; i < n_tensors; ++i) {
        const usaf_adamw_tensor &t = tensors[i];
        USAF_REQUIRE(t.numel >= 0 && (t.numel == 0 || (t.p && t.g)) && t.start >= 0 && t.start % kAdamBlock == 0);
    }
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
