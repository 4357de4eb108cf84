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

constexpr int kNormMaxPartials = 592;   // four CTAs per SM
constexpr int kNormMaxBlock = 512;      // 128 registers a thread
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

// ---- rows in registers --------------------------------------------------------
// `tpr` threads (a power of two up to 32, or whole warps) hold one row, NV
// vectors of VN values each: vector i of thread t is columns (i tpr + t) VN ...,
// so that every load of a warp is contiguous.  A CTA holds blockDim / tpr rows
// at a time and walks down the rows with the weight kept in registers, each row
// read once.
template <typename T, int VN> struct alignas(sizeof(T) * VN) Vec { T v[VN]; };

template <typename T, int VN> __device__ __forceinline__ Vec<T, VN> load_vec(const T *p) {
    Vec<T, VN> r;
    constexpr int B = sizeof(T) * VN;
    if constexpr (B >= 16) {                 // 16 bytes a load (fp32 weights of 8 values: two)
#pragma unroll
        for (int i = 0; i < B / 16; ++i)
            reinterpret_cast<uint4 *>(&r)[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < VN; ++i) r.v[i] = p[i];
    }
    return r;
}

template <typename T, int VN> __device__ __forceinline__ void store_vec(T *p, const Vec<T, VN> &r) {
    if constexpr (sizeof(T) * VN == 16) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(&r);
    else
#pragma unroll
        for (int i = 0; i < VN; ++i) p[i] = r.v[i];
}

// sum over the row's threads, in the same order for each of them; `red` holds
// a value per warp, and rows alternate between two of them so that one barrier
// a row is enough
__device__ __forceinline__ float row_sum(float v, int tpr, int group, float *red) {
    for (int o = min(tpr, 32) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (tpr > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(tpr) : "memory");
        const int n = tpr >> 5;
        v = 0.0f;
        for (int i = 0; i < n; ++i) v += red[group * n + i];
    }
    return v;
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

// ---- rows ahead -----------------------------------------------------------------
// Aligned rows come through a ring in shared memory that every thread fills for
// itself by asynchronous copies: a thread has D - 1 rows' vectors on their way
// and reads back only what it copied, so no barrier and no register is spent on
// them.  384 bytes a thread keep about 100 KB in flight on an SM.
__device__ __forceinline__ void copy_ahead(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ uint4 ring_read(uint32_t at) {
    uint4 u;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(at));
    return u;
}
constexpr int ring_depth(int nv, int tensors) {
    const int d = 12 / (nv * tensors);
    return d > 6 ? 6 : d < 2 ? 2 : d;
}

// NT tensors' rows of one thread: `p[k]`, `ld[k]`; vector i of the row of turn n
template <typename T, int VN, int NV, int NT> struct RowRing {
    static constexpr int D = ring_depth(NV, NT);
    const T *p[NT];
    int64_t ld[NT];
    uint32_t base;               // this thread's 16 bytes of the first slot
    int tpr, t, H;
    int64_t rows;

    __device__ __forceinline__ uint32_t slot(int stage, int k, int i) const {
        return base + (uint32_t)(((stage * NT + k) * NV + i) * blockDim.x) * 16u;
    }
    __device__ __forceinline__ void fetch(int stage, int64_t row) const {
        if (row < rows) {
#pragma unroll
            for (int k = 0; k < NT; ++k)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = (i * tpr + t) * VN;
                    if (c < H) copy_ahead(slot(stage, k, i), p[k] + row * ld[k] + c);
                }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    __device__ __forceinline__ static void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory"); }
    // vector i of tensor k: from the ring, or for single values from memory
    __device__ __forceinline__ Vec<T, VN> get(int stage, int k, int i, int64_t row) const {
        Vec<T, VN> v;
        if constexpr (VN > 1) *reinterpret_cast<uint4 *>(&v) = ring_read(slot(stage, k, i));
        else v.v[0] = p[k][row * ld[k] + i * tpr + t];
        return v;
    }
};

template <typename T, typename W, int VN, int NV, bool RES>
__global__ void __launch_bounds__(kNormMaxBlock) norm_fwd_rows(const NormFwd a, int tpr) {
    __shared__ float red[2][32];
    extern __shared__ uint4 dyn[];
    const int group = threadIdx.x / tpr, t = threadIdx.x - group * tpr, groups = blockDim.x / tpr;
    using Ring = RowRing<T, VN, NV, RES ? 2 : 1>;
    Ring ring;
    ring.p[0] = static_cast<const T *>(a.x);
    ring.ld[0] = a.ldx;
    if constexpr (RES) {
        ring.p[1] = static_cast<const T *>(a.res);
        ring.ld[1] = a.ldr;
    }
    ring.base = (uint32_t)__cvta_generic_to_shared(dyn + threadIdx.x);
    ring.tpr = tpr;
    ring.t = t;
    ring.H = a.H;
    ring.rows = a.rows;
    const int64_t step = (int64_t)gridDim.x * groups;
    const int64_t start = (int64_t)blockIdx.x * groups;
    if constexpr (VN > 1)
#pragma unroll
        for (int d = 0; d < Ring::D - 1; ++d) ring.fetch(d, start + d * step + group);
    Vec<W, VN> wv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * tpr + t) * VN;
        if (c < a.H) wv[i] = load_vec<W, VN>(static_cast<const W *>(a.w) + c);
    }
    const float inv_h = 1.0f / (float)a.H;
    int flip = 0, stage = 0;
    // every thread takes every turn: the shuffles and barriers are for whole groups
    for (int64_t base = start; base < a.rows; base += step) {
        const int64_t row = base + group;
        const bool in = row < a.rows;
        if constexpr (VN > 1) {
            ring.fetch(stage == 0 ? Ring::D - 1 : stage - 1, row + (Ring::D - 1) * step);
            Ring::wait();
        }
        Vec<T, VN> v[NV];
        float ss = 0.0f;
        if (in) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * tpr + t) * VN;
                if (c < a.H) {
                    v[i] = ring.get(stage, 0, i, row);
                    if constexpr (RES) {
                        const Vec<T, VN> q = ring.get(stage, RES ? 1 : 0, i, row);
#pragma unroll
                        for (int k = 0; k < VN; ++k) v[i].v[k] = from_f<T>(to_f(v[i].v[k]) + to_f(q.v[k]));
                        store_vec<T, VN>(static_cast<T *>(a.sum) + row * a.H + c, v[i]);
                    }
#pragma unroll
                    for (int k = 0; k < VN; ++k) ss = fmaf(to_f(v[i].v[k]), to_f(v[i].v[k]), ss);
                }
            }
        }
        ss = row_sum(ss, tpr, group, red[flip]);
        flip ^= 1;
        stage = stage == Ring::D - 1 ? 0 : stage + 1;
        const float r = __frcp_rn(__fsqrt_rn(ss * inv_h + a.eps));
        if (in) {
            if (a.rstd && t == 0) a.rstd[row] = r;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * tpr + t) * VN;
                if (c < a.H) {
                    Vec<T, VN> o;
#pragma unroll
                    for (int k = 0; k < VN; ++k) o.v[k] = from_f<T>(to_f(v[i].v[k]) * r * to_f(wv[i].v[k]));
                    store_vec<T, VN>(static_cast<T *>(a.y) + row * a.H + c, o);
                }
            }
        }
    }
}

template <typename T, typename W, int VN, int NV, bool DSUM, bool DW>
__global__ void __launch_bounds__(kNormMaxBlock) norm_bwd_rows(const NormBwd a, int tpr) {
    __shared__ float red[2][32];
    extern __shared__ uint4 dyn[];           // the ring; at the end [groups][H] sums, where a CTA has several rows
    const int group = threadIdx.x / tpr, t = threadIdx.x - group * tpr, groups = blockDim.x / tpr;
    using Ring = RowRing<T, VN, NV, DSUM ? 3 : 2>;
    Ring ring;
    ring.p[0] = static_cast<const T *>(a.x);
    ring.ld[0] = a.ldx;
    ring.p[1] = static_cast<const T *>(a.dy);
    ring.ld[1] = a.lddy;
    if constexpr (DSUM) {
        ring.p[2] = static_cast<const T *>(a.dsum);
        ring.ld[2] = a.ldds;
    }
    ring.base = (uint32_t)__cvta_generic_to_shared(dyn + threadIdx.x);
    ring.tpr = tpr;
    ring.t = t;
    ring.H = a.H;
    ring.rows = a.rows;
    const int64_t step = (int64_t)gridDim.x * groups;
    const int64_t start = (int64_t)blockIdx.x * groups;
    if constexpr (VN > 1)
#pragma unroll
        for (int d = 0; d < Ring::D - 1; ++d) ring.fetch(d, start + d * step + group);
    Vec<W, VN> wv[NV];
    float acc[DW ? NV : 1][VN];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * tpr + t) * VN;
        if (c < a.H) wv[i] = load_vec<W, VN>(static_cast<const W *>(a.w) + c);
        if constexpr (DW)
#pragma unroll
            for (int k = 0; k < VN; ++k) acc[i][k] = 0.0f;
    }
    const float inv_h = 1.0f / (float)a.H;
    int flip = 0, stage = 0;
    float r = start + group < a.rows ? a.rstd[start + group] : 0.0f;
    for (int64_t base = start; base < a.rows; base += step) {
        const int64_t row = base + group;
        const bool in = row < a.rows;
        const float r_next = row + step < a.rows ? a.rstd[row + step] : 0.0f;
        if constexpr (VN > 1) {
            ring.fetch(stage == 0 ? Ring::D - 1 : stage - 1, row + (Ring::D - 1) * step);
            Ring::wait();
        }
        float dot = 0.0f;
        if (in) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * tpr + t) * VN;
                if (c < a.H) {
                    const Vec<T, VN> x = ring.get(stage, 0, i, row), d = ring.get(stage, 1, i, row);
#pragma unroll
                    for (int k = 0; k < VN; ++k) {
                        dot = fmaf(to_f(d.v[k]) * to_f(wv[i].v[k]), to_f(x.v[k]), dot);
                        if constexpr (DW) acc[i][k] = fmaf(to_f(d.v[k]), to_f(x.v[k]) * r, acc[i][k]);
                    }
                }
            }
        }
        // hat c = s r mean(g s r): s times this
        const float along = row_sum(dot, tpr, group, red[flip]) * inv_h * r * r * r;
        flip ^= 1;
        if (in) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * tpr + t) * VN;
                if (c < a.H) {               // read again: cheaper than the registers to keep them
                    const Vec<T, VN> x = ring.get(stage, 0, i, row), d = ring.get(stage, 1, i, row);
                    Vec<T, VN> o;
                    float v[VN];
#pragma unroll
                    for (int k = 0; k < VN; ++k)
                        v[k] = fmaf(to_f(d.v[k]) * to_f(wv[i].v[k]), r, -along * to_f(x.v[k]));
                    if constexpr (DSUM) {
                        const Vec<T, VN> s = ring.get(stage, DSUM ? 2 : 0, i, row);
#pragma unroll
                        for (int k = 0; k < VN; ++k) v[k] += to_f(s.v[k]);
                    }
#pragma unroll
                    for (int k = 0; k < VN; ++k) o.v[k] = from_f<T>(v[k]);
                    store_vec<T, VN>(static_cast<T *>(a.dx) + row * a.H + c, o);
                }
            }
        }
        stage = stage == Ring::D - 1 ? 0 : stage + 1;
        r = r_next;
    }
    if constexpr (DW) {
        float *part = a.part + (int64_t)blockIdx.x * a.H, *fold = reinterpret_cast<float *>(dyn);
        float *to = groups > 1 ? fold + (int64_t)group * a.H : part;
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();                     // the ring is read; its space takes the sums
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + t) * VN;
            if (c < a.H)
#pragma unroll
                for (int k = 0; k < VN; ++k) to[c + k] = acc[i][k];
        }
        if (groups > 1) {
            __syncthreads();
            for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
                float v = 0.0f;
                for (int g = 0; g < groups; ++g) v += fold[g * a.H + c];
                part[c] = v;
            }
        }
    }
}

// ---- any width, stride and alignment ---------------------------------------------
// one CTA per row, rows wider than the registers of a CTA or not aligned: read twice
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

// dw[c] = sum over the P partial rows: 32 columns a CTA, 32 warps over the rows
// (a few loads each, all in flight), their sums added in warp order
template <typename W>
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float *__restrict__ part, int P, int H,
                                                       W *__restrict__ dw) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (c < H) {
#pragma unroll 10
        for (int p = k; p < P; p += 32) v += part[(int64_t)p * H + c];
    }
    s[k][lane] = v;
    __syncthreads();
    v = warp_sum(s[lane][k]);                // warp k adds column k of the CTA
    if (lane == 0 && blockIdx.x * 32 + k < H) dw[blockIdx.x * 32 + k] = from_f<W>(v);
}

// How the rows are cut: vectors of 16 bytes where every row starts on a 16-byte
// boundary, else single values; NV vectors a thread, threads a row, threads a CTA.
struct RowPlan {
    int vn, nv, tpr, block;
};

template <typename T> static RowPlan plan_rows(int H, bool aligned) {
    RowPlan p{aligned ? 16 / (int)sizeof(T) : 1, 8, 0, 0};
    const int n = (H + p.vn - 1) / p.vn;     // vectors of a row
    if (aligned) p.nv = n <= 4 ? 1 : n <= 2 * kNormMaxBlock ? 2 : 4;
    const int t = (n + p.nv - 1) / p.nv;
    if (t > 32) {
        p.tpr = (t + 31) / 32 * 32;
    } else {
        p.tpr = 1;
        while (p.tpr < t) p.tpr *= 2;
    }
    p.block = p.tpr >= 256 ? p.tpr : 256 / p.tpr * p.tpr;
    if (p.tpr > kNormMaxBlock) p.nv = 0;     // too wide for a CTA's registers
    return p;
}

static bool on16(const void *p, int64_t ld_bytes) { return ((uintptr_t)p | (uintptr_t)ld_bytes) % 16 == 0; }

// CTAs that fit the SMs at once by shared memory and `regs` registers a thread,
// or fewer where the rows are fewer
static int row_grid(const RowPlan &p, int smem, int regs, int64_t rows, int most) {
    const int per_sm = std::max(1, std::min({227 * 1024 / (smem + 1024 + 256), 65536 / (regs * p.block),
                                             2048 / p.block}));
    const int groups = p.block / p.tpr;
    return (int)std::min<int64_t>((rows + groups - 1) / groups, std::min(148 * per_sm, most));
}

template <typename K> static bool allow_smem(K kernel, int smem) {
    if (smem + 256 <= 48 * 1024 ||       // 256 bytes are the reduction's
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess)
        return true;
    (void)cudaGetLastError();
    return false;
}

template <typename T, typename W, int VN, int NV, bool RES>
static int fwd_launch(const NormFwd &a, const RowPlan &p, cudaStream_t st) {
    constexpr int NT = RES ? 2 : 1;
    const int smem = VN > 1 ? NV * NT * ring_depth(NV, NT) * 16 * p.block : 0;
    if (!allow_smem(norm_fwd_rows<T, W, VN, NV, RES>, smem)) return USAF_ECUDA;
    const int grid = row_grid(p, smem, NV == 4 ? 128 : 64, a.rows, 1 << 30);
    norm_fwd_rows<T, W, VN, NV, RES><<<grid, p.block, smem, st>>>(a, p.tpr);
    USAF_CHECK_LAUNCH();
    return USAF_OK;
}

template <typename T, typename W, int VN, int NV>
static int fwd_launch(const NormFwd &a, const RowPlan &p, cudaStream_t st) {
    return a.res ? fwd_launch<T, W, VN, NV, true>(a, p, st) : fwd_launch<T, W, VN, NV, false>(a, p, st);
}

template <typename T, typename W> static int norm_fwd(const NormFwd &a, cudaStream_t st) {
    constexpr int N = 16 / (int)sizeof(T);
    const int64_t row = (int64_t)a.H * sizeof(T);
    const bool aligned = on16(a.x, a.ldx * sizeof(T)) && on16(a.y, row) && on16(a.w, 0) &&
                         (!a.res || (on16(a.res, a.ldr * sizeof(T)) && on16(a.sum, row)));
    const RowPlan p = plan_rows<T>(a.H, aligned);
    if (p.vn > 1) {
        if (p.nv == 1) return fwd_launch<T, W, N, 1>(a, p, st);
        if (p.nv == 2) return fwd_launch<T, W, N, 2>(a, p, st);
        if (p.nv == 4) return fwd_launch<T, W, N, 4>(a, p, st);
    } else if (p.nv) {
        return fwd_launch<T, W, 1, 8>(a, p, st);
    }
    const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 148 * 8);
    norm_fwd_any<T, W><<<grid, 256, 0, st>>>((const T *)a.x, a.ldx, (const T *)a.res, a.ldr, (const W *)a.w, a.rows,
                                             a.H, a.eps, (T *)a.sum, (T *)a.y, a.rstd);
    USAF_CHECK_LAUNCH();
    return USAF_OK;
}

// the partial rows of a launch: P of them
template <typename T, typename W, int VN, int NV, bool DSUM, bool DW>
static int bwd_launch(const NormBwd &a, const RowPlan &p, int *P, cudaStream_t st) {
    constexpr int NT = DSUM ? 3 : 2;
    const int groups = p.block / p.tpr, fold = DW && groups > 1 ? groups * a.H * 4 : 0;
    const int smem = std::max(VN > 1 ? NV * NT * ring_depth(NV, NT) * 16 * p.block : 0, fold);
    if (!allow_smem(norm_bwd_rows<T, W, VN, NV, DSUM, DW>, smem)) return USAF_ECUDA;
    const int grid = row_grid(p, smem, NV == 4 ? 128 : 64, a.rows, DW ? kNormMaxPartials : 1 << 30);
    norm_bwd_rows<T, W, VN, NV, DSUM, DW><<<grid, p.block, smem, st>>>(a, p.tpr);
    USAF_CHECK_LAUNCH();
    *P = grid;
    return USAF_OK;
}

template <typename T, typename W, int VN, int NV>
static int bwd_launch(const NormBwd &a, const RowPlan &p, int *P, cudaStream_t st) {
    if (a.dw)
        return a.dsum ? bwd_launch<T, W, VN, NV, true, true>(a, p, P, st) : bwd_launch<T, W, VN, NV, false, true>(a, p, P, st);
    return a.dsum ? bwd_launch<T, W, VN, NV, true, false>(a, p, P, st) : bwd_launch<T, W, VN, NV, false, false>(a, p, P, st);
}

template <typename T, typename W> static int bwd_rows(const NormBwd &a, int *P, cudaStream_t st) {
    constexpr int N = 16 / (int)sizeof(T);
    const bool aligned = on16(a.x, a.ldx * sizeof(T)) && on16(a.dy, a.lddy * sizeof(T)) && on16(a.w, 0) &&
                         on16(a.dx, (int64_t)a.H * sizeof(T)) && (!a.dsum || on16(a.dsum, a.ldds * sizeof(T)));
    const RowPlan p = plan_rows<T>(a.H, aligned);
    if (p.vn > 1) {
        if (p.nv == 1) return bwd_launch<T, W, N, 1>(a, p, P, st);
        if (p.nv == 2) return bwd_launch<T, W, N, 2>(a, p, P, st);
        if (p.nv == 4) return bwd_launch<T, W, N, 4>(a, p, P, st);
    } else if (p.nv) {
        return bwd_launch<T, W, 1, 8>(a, p, P, st);
    }
    const int smem = a.dw ? a.H * 4 : 0;
    if (smem + 256 > 48 * 1024 && cudaFuncSetAttribute(norm_bwd_any<T, W>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kNormMaxH * 4) != cudaSuccess) {
        (void)cudaGetLastError();
        return USAF_ECUDA;
    }
    *P = (int)std::min<int64_t>(a.rows, kNormMaxPartials);
    norm_bwd_any<T, W><<<*P, 256, smem, st>>>((const T *)a.dy, a.lddy, (const T *)a.x, a.ldx, (const W *)a.w, a.rstd,
                                              (const T *)a.dsum, a.ldds, a.rows, a.H, (T *)a.dx, a.dw ? a.part : nullptr);
    USAF_CHECK_LAUNCH();
    return USAF_OK;
}

template <typename T, typename W> static int norm_bwd(const NormBwd &a, cudaStream_t st) {
    int P = 0;
    if (a.rows) {
        const int rc = bwd_rows<T, W>(a, &P, st);
        if (rc) return rc;
    }
    if (a.dw) {
        norm_dw_kernel<W><<<cdiv(a.H, 32), 1024, 0, st>>>(a.part, P, a.H, (W *)a.dw);
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
