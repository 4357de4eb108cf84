// RMS norm of rows of H values and its backward pass.
//
//   s = round(x + res) (or x);  r = 1 / sqrt(mean(s^2) + eps);  y = s r w
//   g = dy w;  c = mean(g s r);  ds = r (g - s r c) + dsum;  dw = sum over rows of dy s r
//
// All sums, r and the products run in fp32; y, s, ds and dw are rounded once.
// dw is summed per CTA over the rows the CTA walks, written as a row of fp32
// partial sums, and a second kernel adds those rows in a fixed order: the
// result does not depend on timing.
#include "common.cuh"

namespace usaf {

constexpr int kNormMaxPartials = 296;   // two CTAs per SM
constexpr int kNormMaxH = 32768;        // fp32 dw sums of a row in shared memory

template <int NT> __device__ __forceinline__ float block_sum(float v, float *red) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) s += red[i];
    __syncthreads();
    return s;
}

// any width, stride and alignment: one CTA per row
template <typename T, typename W>
__global__ void __launch_bounds__(256)
norm_fwd_any(const T *__restrict__ x, int64_t ldx, const T *__restrict__ res, int64_t ldr,
             const W *__restrict__ w, int64_t rows, int H, float eps, T *__restrict__ sum,
             T *__restrict__ y, float *__restrict__ rstd) {
    __shared__ float red[8];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        float ss = 0.0f;
        for (int c = threadIdx.x; c < H; c += 256) {
            float v = to_f(x[row * ldx + c]);
            if (res) {
                const T t = from_f<T>(v + to_f(res[row * ldr + c]));
                sum[row * H + c] = t;
                v = to_f(t);
            }
            ss = fmaf(v, v, ss);
        }
        ss = block_sum<256>(ss, red);
        const float r = __frcp_rn(__fsqrt_rn(ss / (float)H + eps));
        // a thread reads back only the sums it wrote itself
        const T *s = res ? sum + row * H : x + row * ldx;
        for (int c = threadIdx.x; c < H; c += 256)
            y[row * H + c] = from_f<T>(to_f(s[c]) * r * to_f(w[c]));
        if (rstd && threadIdx.x == 0) rstd[row] = r;
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(256)
norm_bwd_any(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x, int64_t ldx,
             const W *__restrict__ w, const float *__restrict__ rstd, const T *__restrict__ dsum,
             int64_t ldds, int64_t rows, int H, T *__restrict__ dx, float *__restrict__ part) {
    extern __shared__ float acc[];      // [H] dw sums, a thread's own columns only
    __shared__ float red[8];
    if (part)
        for (int c = threadIdx.x; c < H; c += 256) acc[c] = 0.0f;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float r = rstd[row];
        float dot = 0.0f;
        for (int c = threadIdx.x; c < H; c += 256) {
            const float d = to_f(dy[row * lddy + c]), hat = to_f(x[row * ldx + c]) * r;
            dot = fmaf(d * to_f(w[c]), hat, dot);
            if (part) acc[c] = fmaf(d, hat, acc[c]);
        }
        dot = block_sum<256>(dot, red) / (float)H;
        for (int c = threadIdx.x; c < H; c += 256) {
            const float hat = to_f(x[row * ldx + c]) * r;
            float v = r * (to_f(dy[row * lddy + c]) * to_f(w[c]) - hat * dot);
            if (dsum) v += to_f(dsum[row * ldds + c]);
            dx[row * H + c] = from_f<T>(v);
        }
    }
    if (part)
        for (int c = threadIdx.x; c < H; c += 256) part[(int64_t)blockIdx.x * H + c] = acc[c];
}

// dw[c] = sum over the P partial rows: 32 columns a CTA, 8 warps over the rows,
// their sums added in warp order
template <typename W>
__global__ void __launch_bounds__(256) norm_dw_kernel(const float *__restrict__ part, int P, int H,
                                                      W *__restrict__ dw) {
    __shared__ float s[8][32];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
    float v = 0.0f;
    if (c < H)
        for (int p = k; p < P; p += 8) v += part[(int64_t)p * H + c];
    s[k][threadIdx.x & 31] = v;
    __syncthreads();
    if (k == 0 && c < H) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += s[i][threadIdx.x];
        dw[c] = from_f<W>(t);
    }
}

struct NormFwd {
    const void *x; int64_t ldx;
    const void *res; int64_t ldr;
    const void *w;
    int64_t rows; int H; float eps;
    void *sum, *y; float *rstd;
};

struct NormBwd {
    const void *dy; int64_t lddy;
    const void *x; int64_t ldx;
    const void *w; const float *rstd;
    const void *dsum; int64_t ldds;
    int64_t rows; int H;
    void *dx, *dw; float *part;
};

template <typename T, typename W> static int norm_fwd(const NormFwd &a, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 148 * 8);
    norm_fwd_any<T, W><<<grid, 256, 0, st>>>((const T *)a.x, a.ldx, (const T *)a.res, a.ldr, (const W *)a.w, a.rows,
                                             a.H, a.eps, (T *)a.sum, (T *)a.y, a.rstd);
    USAF_CHECK_LAUNCH();
    return USAF_OK;
}

template <typename T, typename W> static int norm_bwd(const NormBwd &a, cudaStream_t st) {
    const int P = (int)std::min<int64_t>(a.rows, kNormMaxPartials);
    float *part = a.dw ? a.part : nullptr;
    if (P) {
        const int smem = part ? a.H * 4 : 0;
        if (smem > 48 * 1024 &&
            cudaFuncSetAttribute(norm_bwd_any<T, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
            return USAF_ECUDA;
        norm_bwd_any<T, W><<<P, 256, smem, st>>>((const T *)a.dy, a.lddy, (const T *)a.x, a.ldx, (const W *)a.w, a.rstd,
                                                 (const T *)a.dsum, a.ldds, a.rows, a.H, (T *)a.dx, part);
        USAF_CHECK_LAUNCH();
    }
    if (a.dw) {
        norm_dw_kernel<W><<<cdiv(a.H, 32), 256, 0, st>>>(a.part, P, a.H, (W *)a.dw);
        USAF_CHECK_LAUNCH();
    }
    return USAF_OK;
}

}  // namespace usaf

using namespace usaf;

// the weight has the rows' dtype or fp32
#define NORM_DISPATCH(fn, args)                                                     \
    switch (dtype * 4 + w_dtype) {                                                  \
        case USAF_F32 * 4 + USAF_F32: return fn<float, float>(args, st);            \
        case USAF_BF16 * 4 + USAF_BF16: return fn<__nv_bfloat16, __nv_bfloat16>(args, st); \
        case USAF_BF16 * 4 + USAF_F32: return fn<__nv_bfloat16, float>(args, st);   \
        case USAF_F16 * 4 + USAF_F16: return fn<__half, __half>(args, st);          \
        case USAF_F16 * 4 + USAF_F32: return fn<__half, float>(args, st);           \
        default: return USAF_EINVAL;                                                \
    }

extern "C" int64_t usaf_rms_norm_workspace_bytes(int64_t rows, int32_t H) {
    if (rows < 0 || H < 1) return -1;
    return std::min<int64_t>(rows, kNormMaxPartials) * H * 4;
}

extern "C" int usaf_rms_norm_fwd(const void *x, int64_t ldx, const void *res, int64_t ldr, const void *w,
                                 int32_t dtype, int32_t w_dtype, int64_t rows, int32_t H, double eps, void *sum,
                                 void *y, float *rstd, void *stream) {
    USAF_REQUIRE(rows >= 0 && H >= 1 && eps >= 0.0);
    if (rows == 0) return USAF_OK;
    USAF_REQUIRE(x && w && y && ldx >= 0 && (res == nullptr) == (sum == nullptr) && (!res || ldr >= 0));
    if (H > kNormMaxH) return USAF_EUNSUPPORTED;
    cudaStream_t st = as_stream(stream);
    const NormFwd a{x, ldx, res, ldr, w, rows, H, (float)eps, sum, y, rstd};
    NORM_DISPATCH(norm_fwd, a)
}

extern "C" int usaf_rms_norm_bwd(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *w,
                                 const float *rstd, const void *dsum, int64_t ldds, int32_t dtype, int32_t w_dtype,
                                 int64_t rows, int32_t H, void *dx, void *dw, void *ws, void *stream) {
    USAF_REQUIRE(rows >= 0 && H >= 1);
    if (rows == 0 && !dw) return USAF_OK;
    USAF_REQUIRE(rows == 0 || (dy && x && w && rstd && dx && lddy >= 0 && ldx >= 0 && (!dsum || ldds >= 0)));
    USAF_REQUIRE(rows == 0 || !dw || ws);
    if (H > kNormMaxH) return USAF_EUNSUPPORTED;
    cudaStream_t st = as_stream(stream);
    const NormBwd a{dy, lddy, x, ldx, w, rstd, dsum, ldds, rows, H, dx, dw, (float *)ws};
    NORM_DISPATCH(norm_bwd, a)
}
