// RMS norm of rows of H values and its backward pass.
//
//   s = round(x + res) (or x);  r = 1 / sqrt(mean(s^2) + eps);  y = s r w
//   g = dy w;  c = mean(g s r);  ds = r (g - s r c) + dsum;  dw = sum over rows of dy s r
//
// All sums, r and the products run in fp32; y, s, ds and dw are rounded once.
// dw is summed per CTA over the rows the CTA walks, written as a row of fp32
// partial sums, and a second kernel adds those rows in a fixed order: the
// result does not depend on timing.
//
// HBM bounds both passes: with rows of 8192 x 2048 bf16 (and the residual) the
// forward pass takes 20 us and the backward pass 21 us, with dw 27, where the
// bytes take 20.8 at the measured copy rate; 262144 x 128: 22 and 32 (36) against
// 20.8 and 31.1; 4096 x 6144: 18 and 25 (31) against 15.6 and 23.4 (one after
// another in a graph, over three sets of rows).
#include "common.cuh"
#include "f32x2.cuh"

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

// ---- rows of whole 16-byte vectors ------------------------------------------------
// `tpr` threads (a power of two up to 32, or whole warps) hold one row, NV
// vectors of 16 bytes each: vector i of thread t is the row's vector i tpr + t, so
// that every load of a warp is contiguous.  A CTA holds blockDim / tpr rows at a
// time and walks down the rows with the weight in registers.
//
// A row costs few bytes and many instructions (counted: the first form of these
// kernels issued 45 a value in the backward pass and was bound by that), so
// products run in pairs (f32x2), 16-bit values are taken apart by a shift and a
// mask and put together two at a time, and addresses are carried along.

// the weight of the columns of one vector of rows
template <typename T, typename W> __device__ __forceinline__ void load_weight(const W *w, uint64_t *p) {
    constexpr int N = 2 * kPairs<T>;
    uint4 u[N * sizeof(W) / 16];
#pragma unroll
    for (int i = 0; i < (int)(N * sizeof(W) / 16); ++i) u[i] = reinterpret_cast<const uint4 *>(w)[i];
#pragma unroll
    for (int i = 0; i < (int)(N * sizeof(W) / 16); ++i) unpack<W>(u[i], p + i * kPairs<W>);
}

// Sum over the row's threads, the same bits for each of them.  `red` holds 16
// values a group, those behind its warps zero; rows alternate between two of
// them, so that one barrier a row is enough.
__device__ __forceinline__ float row_sum(float v, int tpr, int group, float (*red)[16]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < tpr) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (tpr > 32) {
        if ((threadIdx.x & 31) == 0) red[group][(threadIdx.x - group * tpr) >> 5] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(tpr) : "memory");
        v = 0.0f;
        for (int i = 0; i * 128 < tpr; ++i) {
            const float4 q = *reinterpret_cast<const float4 *>(&red[group][4 * i]);
            v += (q.x + q.y) + (q.z + q.w);
        }
    }
    return v;
}

// Rows ahead: NT tensors' rows come through a ring in shared memory that every
// thread fills for itself by asynchronous copies: it has D - 1 rows' vectors on
// their way and reads back only what it copied, so no barrier and no register is
// spent on them.  12 slots of 16 bytes a thread are 1024 threads' share of an
// SM's shared memory.  A slot's 16 bytes of neighbouring threads lie side by side:
// with each thread's slots together instead, the copies' scattered writes made the
// forward pass of 8192 x 2048 rows take 28 us instead of 21.
constexpr int ring_depth(int nv, int tensors, int slots) {
    const int d = slots / (nv * tensors);
    return d > 6 ? 6 : d < 2 ? 2 : d;
}
constexpr int kFwdSlots = 12, kBwdSlots = 16;   // the backward pass's registers leave 3 CTAs of 256 an SM
constexpr int ring_slots(int nv, int tensors, int slots) { return ring_depth(nv, tensors, slots) * nv * tensors; }

template <typename T, int NV, int NT, int SLOTS> struct RowRing {
    static constexpr int D = ring_depth(NV, NT, SLOTS);
    const char *p[NT];           // this thread's first vector of the next row to fetch
    int64_t ahead[NT];           // bytes from a turn's row to the next turn's
    int64_t row, step, rows;     // the next row to fetch
    uint32_t base, in_at, out_at, slot;   // slot: bytes of a slot of all threads
    int hop;                     // bytes between a thread's vectors
    uint32_t has;                // bit i: vector i lies in the row

    __device__ __forceinline__ void open(uint4 *dyn, int tpr, int t, int H, int64_t first, int64_t step_, int64_t rows_) {
        row = first;
        step = step_;
        rows = rows_;
        hop = tpr * 16;
        has = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((i * tpr + t) * 2 * kPairs<T> < H) has |= 1u << i;
        base = in_at = out_at = (uint32_t)__cvta_generic_to_shared(dyn + threadIdx.x);
        slot = blockDim.x * 16;
    }
    __device__ __forceinline__ void tensor(int k, const void *q, int64_t ld, int t) {
        p[k] = static_cast<const char *>(q) + row * ld * (int64_t)sizeof(T) + t * 16;
        ahead[k] = step * ld * (int64_t)sizeof(T);
    }
    __device__ __forceinline__ uint32_t next(uint32_t at) const {
        return at == base + (D - 1) * NV * NT * slot ? base : at + NV * NT * slot;
    }
    __device__ __forceinline__ void fetch() {
        if (row < rows) {
#pragma unroll
            for (int k = 0; k < NT; ++k)
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (has >> i & 1)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(in_at + (k * NV + i) * slot),
                                     "l"(p[k] + i * hop)
                                     : "memory");
        }
#pragma unroll
        for (int k = 0; k < NT; ++k) p[k] += ahead[k];
        row += step;
        in_at = next(in_at);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    __device__ __forceinline__ void fill() {
#pragma unroll
        for (int d = 0; d < D - 1; ++d) fetch();
    }
    // one more row on its way, the turn's row is there
    __device__ __forceinline__ void turn() {
        fetch();
        asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
    }
    __device__ __forceinline__ uint4 get(int k, int i) const {
        uint4 u;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                     : "r"(out_at + (k * NV + i) * slot));
        return u;
    }
    __device__ __forceinline__ void done() { out_at = next(out_at); }
};

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

// a CTA's sum of column c: a partial one, or where it is the only CTA, dw itself
template <typename W> __device__ __forceinline__ void put_dw(const NormBwd &a, int c, float v) {
    if (gridDim.x == 1) static_cast<W *>(a.dw)[c] = from_f<W>(v);
    else a.part[(int64_t)blockIdx.x * a.H + c] = v;
}

template <typename T, typename W, int NV, bool RES>
__global__ void __launch_bounds__(kNormMaxBlock) norm_fwd_rows(const NormFwd a, int tpr) {
    __shared__ alignas(16) float red[2][8][16];
    extern __shared__ uint4 dyn[];
    constexpr int N2 = kPairs<T>;
    const int group = threadIdx.x / tpr, t = threadIdx.x - group * tpr, groups = blockDim.x / tpr;
    for (int i = threadIdx.x; i < 256; i += blockDim.x) (&red[0][0][0])[i] = 0.0f;
    __syncthreads();
    wait_for_previous();
    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t row = (int64_t)blockIdx.x * groups + group;
    RowRing<T, NV, RES ? 2 : 1, kFwdSlots> ring;
    ring.open(dyn, tpr, t, a.H, row, step, a.rows);
    ring.tensor(0, a.x, a.ldx, t);
    if constexpr (RES) ring.tensor(1, a.res, a.ldr, t);
    ring.fill();
    uint64_t w[NV][N2];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (ring.has >> i & 1) load_weight<T, W>(static_cast<const W *>(a.w) + (i * tpr + t) * 2 * N2, w[i]);
    const float inv_h = 1.0f / (float)a.H;
    const int64_t out = step * a.H * (int64_t)sizeof(T);
    char *y = static_cast<char *>(a.y) + row * a.H * (int64_t)sizeof(T) + t * 16;
    char *sum = RES ? static_cast<char *>(a.sum) + row * a.H * (int64_t)sizeof(T) + t * 16 : nullptr;
    int flip = 0;
    // every thread takes every turn: the shuffles and barriers are for whole groups
    for (int64_t base = (int64_t)blockIdx.x * groups; base < a.rows; base += step) {
        const bool in = row < a.rows;
        ring.turn();
        uint4 v[NV];
        uint64_t ss = 0;
        if (in) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (ring.has >> i & 1) {
                    uint64_t x[N2];
                    v[i] = ring.get(0, i);
                    unpack<T>(v[i], x);
                    if constexpr (RES) {
                        uint64_t q[N2];
                        unpack<T>(ring.get(RES ? 1 : 0, i), q);
#pragma unroll
                        for (int k = 0; k < N2; ++k) q[k] = add2(x[k], q[k]);
                        v[i] = pack<T>(q);
                        *reinterpret_cast<uint4 *>(sum + i * ring.hop) = v[i];
                        unpack<T>(v[i], x);
                    }
#pragma unroll
                    for (int k = 0; k < N2; ++k) ss = fma2(x[k], x[k], ss);
                }
            }
        }
        const float2 h = halves(ss);
        const float r = __frcp_rn(__fsqrt_rn(row_sum(h.x + h.y, tpr, group, red[flip]) * inv_h + a.eps));
        flip ^= 1;
        ring.done();
        if (in) {
            if (a.rstd && t == 0) a.rstd[row] = r;
            const uint64_t r2 = pair(r, r);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (ring.has >> i & 1) {
                    uint64_t x[N2];
                    unpack<T>(v[i], x);
#pragma unroll
                    for (int k = 0; k < N2; ++k) x[k] = mul2(mul2(x[k], r2), w[i][k]);
                    *reinterpret_cast<uint4 *>(y + i * ring.hop) = pack<T>(x);
                }
            }
        }
        row += step;
        y += out;
        if constexpr (RES) sum += out;
    }
}

template <typename T, typename W, int NV, bool DSUM, bool DW>
__global__ void __launch_bounds__(kNormMaxBlock) norm_bwd_rows(const NormBwd a, int tpr) {
    __shared__ alignas(16) float red[2][8][16];
    extern __shared__ uint4 dyn[];           // the ring; at the end [groups][H] sums, where a CTA has several rows
    constexpr int N2 = kPairs<T>;
    const int group = threadIdx.x / tpr, t = threadIdx.x - group * tpr, groups = blockDim.x / tpr;
    for (int i = threadIdx.x; i < 256; i += blockDim.x) (&red[0][0][0])[i] = 0.0f;
    __syncthreads();
    wait_for_previous();
    if constexpr (DW) let_next_start();
    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t row = (int64_t)blockIdx.x * groups + group;
    RowRing<T, NV, DSUM ? 3 : 2, kBwdSlots> ring;
    ring.open(dyn, tpr, t, a.H, row, step, a.rows);
    ring.tensor(0, a.x, a.ldx, t);
    ring.tensor(1, a.dy, a.lddy, t);
    if constexpr (DSUM) ring.tensor(2, a.dsum, a.ldds, t);
    ring.fill();
    uint64_t w[NV][N2], acc[DW ? NV : 1][N2];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (ring.has >> i & 1) load_weight<T, W>(static_cast<const W *>(a.w) + (i * tpr + t) * 2 * N2, w[i]);
        if constexpr (DW)
#pragma unroll
            for (int k = 0; k < N2; ++k) acc[i][k] = 0;
    }
    const float inv_h = 1.0f / (float)a.H;
    const int64_t out = step * a.H * (int64_t)sizeof(T);
    char *dx = static_cast<char *>(a.dx) + row * a.H * (int64_t)sizeof(T) + t * 16;
    int flip = 0;
    float r = row < a.rows ? a.rstd[row] : 0.0f;
    for (int64_t base = (int64_t)blockIdx.x * groups; base < a.rows; base += step) {
        const bool in = row < a.rows;
        row += step;
        const float r_next = row < a.rows ? a.rstd[row] : 0.0f;
        ring.turn();
        const uint64_t r2 = pair(r, r);
        uint64_t dot = 0;
        if (in) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (ring.has >> i & 1) {
                    uint64_t x[N2], d[N2];
                    unpack<T>(ring.get(0, i), x);
                    unpack<T>(ring.get(1, i), d);
#pragma unroll
                    for (int k = 0; k < N2; ++k) {
                        dot = fma2(mul2(d[k], w[i][k]), x[k], dot);
                        if constexpr (DW) acc[i][k] = fma2(d[k], mul2(x[k], r2), acc[i][k]);
                    }
                }
            }
        }
        const float2 h = halves(dot);
        const float along = row_sum(h.x + h.y, tpr, group, red[flip]) * inv_h * r;     // mean(g s r)
        flip ^= 1;
        if (in) {
            const uint64_t back = pair(-along, -along);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (ring.has >> i & 1) {     // read again: cheaper than the registers to keep them
                    uint64_t x[N2], d[N2];
                    unpack<T>(ring.get(0, i), x);
                    unpack<T>(ring.get(1, i), d);
#pragma unroll
                    for (int k = 0; k < N2; ++k)
                        x[k] = mul2(fma2(mul2(x[k], r2), back, mul2(d[k], w[i][k])), r2);
                    if constexpr (DSUM) {
                        unpack<T>(ring.get(DSUM ? 2 : 0, i), d);
#pragma unroll
                        for (int k = 0; k < N2; ++k) x[k] = add2(x[k], d[k]);
                    }
                    *reinterpret_cast<uint4 *>(dx + i * ring.hop) = pack<T>(x);
                }
            }
        }
        ring.done();
        dx += out;
        r = r_next;
    }
    if constexpr (DW) {
        float *part = a.part + (int64_t)blockIdx.x * a.H, *fold = reinterpret_cast<float *>(dyn);
        const bool folds = groups > 1 || gridDim.x == 1;
        float *to = (folds ? fold + group * a.H : part) + t * 2 * N2;
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();                     // the ring is read; its space takes the sums
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (ring.has >> i & 1)
#pragma unroll
                for (int k = 0; k < N2; k += 2) {
                    const float2 x = halves(acc[i][k]), y = halves(acc[i][k + 1]);
                    reinterpret_cast<float4 *>(to + i * tpr * 2 * N2)[k / 2] = make_float4(x.x, x.y, y.x, y.y);
                }
        if (folds) {
            __syncthreads();
            for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
                float v = 0.0f;
                for (int g = 0; g < groups; ++g) v += fold[g * a.H + c];
                put_dw<W>(a, c, v);
            }
        }
    }
}

// ---- dense rows of any width --------------------------------------------------------
// Rows that lie behind one another but do not start on 16-byte boundaries: a tile
// of so many rows that its bytes do (8 rows of an odd number of 16-bit values)
// comes into shared memory in 16-byte copies, `per` threads take a row there value
// by value, and the results leave from where the inputs lay, in 16-byte stores.
// dw is summed by columns, a thread's own ones, over each tile's rows.  Forward /
// backward with dw, against a CTA a row: 20000 x 771 bf16 21 / 47 us (48 / 80),
// 260000 x 35 15 / 35 (279 / 422); bound by instructions, single values' accesses
// to shared memory among them (78 % of the issue slots forward).
template <typename T> __device__ __forceinline__ void tile_in(T *to, const T *from, int n) {
    const int nv = n * (int)sizeof(T) / 16;
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    for (int i = threadIdx.x; i < nv; i += 256)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + i * 16),
                     "l"(reinterpret_cast<const uint4 *>(from) + i)
                     : "memory");
    for (int i = nv * 16 / (int)sizeof(T) + threadIdx.x; i < n; i += 256) to[i] = from[i];
}
template <typename T> __device__ __forceinline__ void tile_out(T *to, const T *from, int n) {
    const int nv = n * (int)sizeof(T) / 16;
    for (int i = threadIdx.x; i < nv; i += 256)
        reinterpret_cast<uint4 *>(to)[i] = reinterpret_cast<const uint4 *>(from)[i];
    for (int i = nv * 16 / (int)sizeof(T) + threadIdx.x; i < n; i += 256) to[i] = from[i];
}
__device__ __forceinline__ void tile_ready() {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
}
__device__ __forceinline__ float lane_sum(float v, int per) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < per) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// shared memory: one tile of R rows for each tensor, then w [H] fp32 (and the dw sums,
// at most 256 or H)
constexpr int kTileRows = 256;

template <typename T, typename W, bool RES>
__global__ void __launch_bounds__(256, 5) norm_fwd_tile(const NormFwd a, int R, int per) {
    extern __shared__ uint4 dyn[];
    T *t0 = reinterpret_cast<T *>(dyn), *t1 = t0 + R * a.H;
    float *w = reinterpret_cast<float *>(RES ? t1 + R * a.H : t1);
    wait_for_previous();
    for (int c = threadIdx.x; c < a.H; c += 256) w[c] = to_f(static_cast<const W *>(a.w)[c]);
    const int l = threadIdx.x & (per - 1), g = threadIdx.x / per, groups = 256 / per;
    const float inv_h = 1.0f / (float)a.H;
    for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < a.rows; row0 += (int64_t)gridDim.x * R) {
        const int nr = (int)min((int64_t)R, a.rows - row0), n = nr * a.H;
        const int64_t at = row0 * a.H;
        tile_in(t0, static_cast<const T *>(a.x) + at, n);
        if (RES) tile_in(t1, static_cast<const T *>(a.res) + at, n);
        tile_ready();
        for (int r0 = 0; r0 < nr; r0 += groups) {
            const int r = r0 + g;
            T *x = t0 + r * a.H, *y = RES ? t1 + r * a.H : x;
            float ss = 0.0f;
            if (r < nr)
                for (int c = l; c < a.H; c += per) {
                    float v = to_f(x[c]);
                    if (RES) {
                        x[c] = from_f<T>(v + to_f(y[c]));
                        v = to_f(x[c]);
                    }
                    ss = fmaf(v, v, ss);
                }
            const float rs = __frcp_rn(__fsqrt_rn(lane_sum(ss, per) * inv_h + a.eps));
            if (r < nr) {
                if (a.rstd && l == 0) a.rstd[row0 + r] = rs;
                for (int c = l; c < a.H; c += per) y[c] = from_f<T>(to_f(x[c]) * rs * w[c]);
            }
        }
        __syncthreads();
        if (RES) tile_out(static_cast<T *>(a.sum) + at, t0, n);
        tile_out(static_cast<T *>(a.y) + at, RES ? t1 : t0, n);
        __syncthreads();
    }
}

template <typename T, typename W, bool DSUM, bool DW>
__global__ void __launch_bounds__(256, 5) norm_bwd_tile(const NormBwd a, int R, int per) {
    extern __shared__ uint4 dyn[];
    __shared__ float rstd[kTileRows];
    T *tx = reinterpret_cast<T *>(dyn), *td = tx + R * a.H, *ts = td + R * a.H;
    float *w = reinterpret_cast<float *>(DSUM ? ts + R * a.H : ts), *acc = w + a.H;
    wait_for_previous();
    if constexpr (DW) let_next_start();
    // threads by columns for dw: of a narrow row several take every parts-th row
    const int wide = (a.H + 31) / 32 * 32, parts = wide <= 128 ? 256 / wide : 1;
    const int part = parts > 1 ? threadIdx.x / wide : 0, col = threadIdx.x - part * wide;
    for (int c = threadIdx.x; c < a.H; c += 256) w[c] = to_f(static_cast<const W *>(a.w)[c]);
    if (DW)
        for (int c = threadIdx.x; c < parts * a.H; c += 256) acc[c] = 0.0f;
    const int l = threadIdx.x & (per - 1), g = threadIdx.x / per, groups = 256 / per;
    const float inv_h = 1.0f / (float)a.H;
    for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < a.rows; row0 += (int64_t)gridDim.x * R) {
        const int nr = (int)min((int64_t)R, a.rows - row0), n = nr * a.H;
        const int64_t at = row0 * a.H;
        tile_in(tx, static_cast<const T *>(a.x) + at, n);
        tile_in(td, static_cast<const T *>(a.dy) + at, n);
        if (DSUM) tile_in(ts, static_cast<const T *>(a.dsum) + at, n);
        for (int r = threadIdx.x; r < nr; r += 256) rstd[r] = a.rstd[row0 + r];
        tile_ready();
        if (DW) {
            if (part < parts)
                for (int c = col; c < a.H; c += 256) {
                    float v = 0.0f;
#pragma unroll 4
                    for (int r = part; r < nr; r += parts)
                        v = fmaf(to_f(td[r * a.H + c]), to_f(tx[r * a.H + c]) * rstd[r], v);
                    acc[part * a.H + c] += v;
                }
            __syncthreads();
        }
        for (int r0 = 0; r0 < nr; r0 += groups) {
            const int r = r0 + g;
            const T *x = tx + r * a.H, *s = ts + r * a.H;
            T *d = td + r * a.H;
            float dot = 0.0f, rs = 0.0f;
            if (r < nr) {
                rs = rstd[r];
                for (int c = l; c < a.H; c += per) dot = fmaf(to_f(d[c]) * w[c], to_f(x[c]), dot);
            }
            const float along = lane_sum(dot, per) * inv_h * rs;                       // mean(g s r)
            if (r < nr)
                for (int c = l; c < a.H; c += per) {
                    float v = rs * fmaf(to_f(x[c]) * rs, -along, to_f(d[c]) * w[c]);
                    if (DSUM) v += to_f(s[c]);
                    d[c] = from_f<T>(v);
                }
        }
        __syncthreads();
        tile_out(static_cast<T *>(a.dx) + at, td, n);
        __syncthreads();
    }
    if (DW)
        for (int c = threadIdx.x; c < a.H; c += 256) {
            float v = 0.0f;
            for (int k = 0; k < parts; ++k) v += acc[k * a.H + c];
            put_dw<W>(a, c, v);
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
             int64_t ldds, int64_t rows, int H, T *__restrict__ dx, float *__restrict__ part, W *__restrict__ dw) {
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
        for (int c = threadIdx.x; c < H; c += 256) {
            if (gridDim.x == 1) dw[c] = from_f<W>(acc[c]);
            else part[(int64_t)blockIdx.x * H + c] = acc[c];
        }
}

// dw[c] = sum over the P partial rows: 32 columns a CTA, 32 warps over the rows
// (a few loads each, all in flight), their sums added in warp order
template <typename W>
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float *part, int P, int H, W *dw) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float v = 0.0f;
    wait_for_previous();
    if (c < H) {
#pragma unroll 10
        for (int p = k; p < P; p += 32) v += part[(int64_t)p * H + c];
    }
    s[k][lane] = v;
    __syncthreads();
    v = warp_sum(s[lane][k]);                // warp k adds column k of the CTA
    if (lane == 0 && blockIdx.x * 32 + k < H) dw[blockIdx.x * 32 + k] = from_f<W>(v);
}

// How rows of n 16-byte vectors are cut: vectors a thread, threads a row, threads
// a CTA.  More vectors a thread let the work of a turn (addresses, the sum over
// the threads) serve more bytes and leave fewer warps to wait for one another;
// the backward pass's dw sums cost 8 registers each.  Measured (us, forward /
// backward with dw, bf16): n = 256 (8192 rows, residual) two vectors 24.1 / 26.3,
// three 23.5 / 33.9; n = 512 (4000 rows) two 15.1 / 24.3, four 13.5 / 23.1; n = 640
// (5000 rows) three 20.9 / 33.0, four 19.0 / 29.9; n = 768 (4096 rows) two 20.5 / 34.4,
// three 18.8 / 31.1, four 20.3 / 31.9; n = 1024 (3000 rows) two 20.2 / 35.8, four
// 17.9 / 29.7.  So two up to 256, then three or four, whichever leaves fewer idle
// lanes, four above 768.
struct RowPlan {
    int nv, tpr, block;
};

static RowPlan plan_rows(int n) {
    const auto idle = [n](int nv) { return (n + 32 * nv - 1) / (32 * nv) * 32 * nv - n; };
    RowPlan p{n <= 4 ? 1 : n <= 256 ? 2 : n <= 768 && idle(3) <= idle(4) ? 3 : 4, 1, 0};
    const int t = (n + p.nv - 1) / p.nv;
    if (t > 32) p.tpr = (t + 31) / 32 * 32;
    else
        while (p.tpr < t) p.tpr *= 2;
    p.block = p.tpr >= 256 ? p.tpr : 256 / p.tpr * p.tpr;
    if (p.tpr > kNormMaxBlock) p.nv = 0;     // too wide for a CTA's registers
    return p;
}

static bool on16(const void *p, int64_t ld_bytes) { return ((uintptr_t)p | (uintptr_t)ld_bytes) % 16 == 0; }

// CTAs that fit the SMs at once by shared memory and `regs` registers a thread,
// or fewer where the rows are fewer
static int row_grid(const RowPlan &p, int smem, int regs, int64_t rows, int most) {
    const int per_sm = std::max(1, std::min({227 * 1024 / (smem + 2048), 65536 / (regs * p.block), 2048 / p.block}));
    const int groups = p.block / p.tpr;
    return (int)std::min<int64_t>((rows + groups - 1) / groups, std::min(148 * per_sm, most));
}

// Tiles of dense rows: R rows (0: too wide), threads a row (each of 16 values or
// more: what a row costs beside them, a sum, a root and addresses, was 150 of 229
// instructions with 32 threads to 131 values), bytes of shared memory.
// About 8 KB a tensor, so that several CTAs an SM load, compute and store at
// different times; at most 64 KB in all, three CTAs an SM: with few rows to a large tile
// most warps have none, and a CTA a row is as fast (8000 x 2050 bf16 with a residual
// forward, 41 KB: 40 us; 8000 x 2051, whose tile would take 74 KB, a CTA a row: 38).
struct TilePlan {
    int R, per, smem;
};

static TilePlan plan_tile(int H, int size, int tensors, bool backward) {
    TilePlan t{16 / size, 32, 0};            // rows until the bytes are a multiple of 16
    while (t.R > 1 && (int64_t)H * size * (t.R / 2) % 16 == 0) t.R /= 2;
    t.R *= std::max(1, std::min(kTileRows, 8192 / (H * size)) / t.R);
    while (t.per > 1 && t.per * 16 >= H && t.per * t.R >= 512) t.per /= 2;      // and the tile's rows for 256 threads
    // whether dw is wanted does not choose the kernel: dx has the same bits either way
    const int64_t smem = (int64_t)tensors * t.R * H * size + H * 4 + (backward ? std::max(256, H) * 4 : 0);
    if (smem > 64 * 1024) t.R = 0;
    t.smem = (int)smem;
    return t;
}

static int tile_grid(const TilePlan &t, int64_t rows, int most) {
    const int per_sm = std::max(1, std::min(227 * 1024 / (t.smem + 2048), 5));
    return (int)std::min<int64_t>((rows + t.R - 1) / t.R, std::min(148 * per_sm, most));
}

template <typename K> static bool allow_smem(K kernel, int smem) {
    if (smem + 1024 <= 48 * 1024 ||          // static arrays take up to 1024 bytes more
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess)
        return true;
    (void)cudaGetLastError();
    return false;
}

template <typename T, typename W, int NV, bool RES>
static int fwd_launch(const NormFwd &a, const RowPlan &p, cudaStream_t st) {
    const int smem = ring_slots(NV, RES ? 2 : 1, kFwdSlots) * 16 * p.block;
    if (!allow_smem(norm_fwd_rows<T, W, NV, RES>, smem)) return USAF_ECUDA;
    const int grid = row_grid(p, smem, NV == 4 ? 128 : NV == 3 ? 80 : 64, a.rows, 1 << 30);
    return launch_early(norm_fwd_rows<T, W, NV, RES>, dim3(grid), p.block, smem, st, a, p.tpr) ? USAF_OK : USAF_ECUDA;
}

template <typename T, typename W, int NV> static int fwd_launch(const NormFwd &a, const RowPlan &p, cudaStream_t st) {
    return a.res ? fwd_launch<T, W, NV, true>(a, p, st) : fwd_launch<T, W, NV, false>(a, p, st);
}

template <typename T, typename W> static int norm_fwd(const NormFwd &a, cudaStream_t st) {
    const int64_t bytes = (int64_t)a.H * sizeof(T);
    if (on16(a.x, a.ldx * sizeof(T)) && on16(a.y, bytes) && on16(a.w, 0) &&
        (!a.res || (on16(a.res, a.ldr * sizeof(T)) && on16(a.sum, 0)))) {
        const RowPlan p = plan_rows((int)(bytes / 16));
        if (p.nv == 1) return fwd_launch<T, W, 1>(a, p, st);
        if (p.nv == 2) return fwd_launch<T, W, 2>(a, p, st);
        if (p.nv == 3) return fwd_launch<T, W, 3>(a, p, st);
        if (p.nv == 4) return fwd_launch<T, W, 4>(a, p, st);
    }
    const bool dense = a.ldx == a.H && (!a.res || a.ldr == a.H) && on16(a.x, 0) && on16(a.y, 0) &&
                       (!a.res || (on16(a.res, 0) && on16(a.sum, 0)));
    const TilePlan t = plan_tile(a.H, sizeof(T), a.res ? 2 : 1, false);
    if (dense && t.R) {
        auto kernel = a.res ? norm_fwd_tile<T, W, true> : norm_fwd_tile<T, W, false>;
        if (!allow_smem(kernel, t.smem)) return USAF_ECUDA;
        return launch_early(kernel, dim3(tile_grid(t, a.rows, 1 << 30)), 256, t.smem, st, a, t.R, t.per) ? USAF_OK
                                                                                                          : USAF_ECUDA;
    }
    const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 148 * 8);
    norm_fwd_any<T, W><<<grid, 256, 0, st>>>((const T *)a.x, a.ldx, (const T *)a.res, a.ldr, (const W *)a.w, a.rows,
                                             a.H, a.eps, (T *)a.sum, (T *)a.y, a.rstd);
    USAF_CHECK_LAUNCH();
    return USAF_OK;
}

// the launches write P partial rows of dw
template <typename T, typename W, int NV, bool DSUM, bool DW>
static int bwd_launch(const NormBwd &a, const RowPlan &p, int *P, cudaStream_t st) {
    const int groups = p.block / p.tpr, fold = DW ? groups * a.H * 4 : 0;
    const int smem = std::max(ring_slots(NV, DSUM ? 3 : 2, kBwdSlots) * 16 * p.block, fold);
    if (!allow_smem(norm_bwd_rows<T, W, NV, DSUM, DW>, smem)) return USAF_ECUDA;
    // up to four turns in one CTA, which then needs no reduction of partial sums
    const int grid = DW && a.rows <= 4 * groups
                         ? 1
                         : row_grid(p, smem, NV == 4 ? 128 : NV == 3 ? 104 : 80, a.rows, DW ? kNormMaxPartials : 1 << 30);
    if (!launch_early(norm_bwd_rows<T, W, NV, DSUM, DW>, dim3(grid), p.block, smem, st, a, p.tpr)) return USAF_ECUDA;
    *P = grid;
    return USAF_OK;
}

template <typename T, typename W, int NV>
static int bwd_launch(const NormBwd &a, const RowPlan &p, int *P, cudaStream_t st) {
    if (a.dw) return a.dsum ? bwd_launch<T, W, NV, true, true>(a, p, P, st) : bwd_launch<T, W, NV, false, true>(a, p, P, st);
    return a.dsum ? bwd_launch<T, W, NV, true, false>(a, p, P, st) : bwd_launch<T, W, NV, false, false>(a, p, P, st);
}

template <typename T, typename W> static int bwd_rows(const NormBwd &a, int *P, cudaStream_t st) {
    const int64_t bytes = (int64_t)a.H * sizeof(T);
    if (on16(a.x, a.ldx * sizeof(T)) && on16(a.dy, a.lddy * sizeof(T)) && on16(a.w, 0) && on16(a.dx, bytes) &&
        on16(a.dw ? a.part : nullptr, 0) && (!a.dsum || on16(a.dsum, a.ldds * sizeof(T)))) {
        const RowPlan p = plan_rows((int)(bytes / 16));
        if (p.nv == 1) return bwd_launch<T, W, 1>(a, p, P, st);
        if (p.nv == 2) return bwd_launch<T, W, 2>(a, p, P, st);
        if (p.nv == 3) return bwd_launch<T, W, 3>(a, p, P, st);
        if (p.nv == 4) return bwd_launch<T, W, 4>(a, p, P, st);
    }
    const bool dense = a.ldx == a.H && a.lddy == a.H && (!a.dsum || a.ldds == a.H) && on16(a.x, 0) && on16(a.dy, 0) &&
                       on16(a.dx, 0) && (!a.dsum || on16(a.dsum, 0));
    const TilePlan t = plan_tile(a.H, sizeof(T), a.dsum ? 3 : 2, true);
    if (dense && t.R) {
        auto kernel = a.dw ? (a.dsum ? norm_bwd_tile<T, W, true, true> : norm_bwd_tile<T, W, false, true>)
                           : (a.dsum ? norm_bwd_tile<T, W, true, false> : norm_bwd_tile<T, W, false, false>);
        if (!allow_smem(kernel, t.smem)) return USAF_ECUDA;
        *P = tile_grid(t, a.rows, a.dw ? kNormMaxPartials : 1 << 30);
        return launch_early(kernel, dim3(*P), 256, t.smem, st, a, t.R, t.per) ? USAF_OK : USAF_ECUDA;
    }
    const int smem = a.dw ? a.H * 4 : 0;
    if (!allow_smem(norm_bwd_any<T, W>, smem)) return USAF_ECUDA;
    *P = (int)std::min<int64_t>(a.rows, kNormMaxPartials);
    norm_bwd_any<T, W><<<*P, 256, smem, st>>>((const T *)a.dy, a.lddy, (const T *)a.x, a.ldx, (const W *)a.w, a.rstd,
                                              (const T *)a.dsum, a.ldds, a.rows, a.H, (T *)a.dx, a.dw ? a.part : nullptr,
                                              (W *)a.dw);
    USAF_CHECK_LAUNCH();
    return USAF_OK;
}

template <typename T, typename W> static int norm_bwd(const NormBwd &a, cudaStream_t st) {
    int P = 0;
    if (a.rows) {
        const int rc = bwd_rows<T, W>(a, &P, st);
        if (rc) return rc;
    }
    if (a.dw && P != 1) {                    // one CTA has written dw itself
        if (!launch_early(norm_dw_kernel<W>, dim3(cdiv(a.H, 32)), 1024, 0, st, (const float *)a.part, P, a.H,
                          (W *)a.dw))
            return USAF_ECUDA;
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
