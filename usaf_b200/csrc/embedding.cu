// Embedding lookup y[t] = scale W[id_t] and the gradient of the table,
// dW[v] = scale * (sum of dy[t] over the tokens t with id_t = v, ascending t).
//
// The gradient takes three launches:
//   1. sort: one cluster of 8 CTAs sorts the (token, position) pairs by a stable
//      radix sort (digits of up to 9 bits, so two passes for a table of up to
//      2^18 rows); the other clusters of the same launch write the table's zeros,
//      which is where the time goes (V x H values against tokens x H);
//   2. sum: the sorted positions are cut into chunks of 32, whatever tokens they
//      hold, so that a frequent token spreads over many warps; a warp adds the
//      rows of its chunk in fp32, writes the rows of tokens that lie in the chunk
//      as a whole and leaves fp32 partial sums of the first and the last token
//      where these go on in a neighbour;
//   3. join: the chunk in which such a token begins adds the partial sums of the
//      chunks it runs through, in chunk order.
// Nothing is added atomically: the sums' order is that of the positions.
#include <cooperative_groups.h>

#include "common.cuh"
#include "f32x2.cuh"

namespace cg = cooperative_groups;

namespace usaf {

__device__ __forceinline__ int64_t token_id(const void *ids, int ids64, int64_t t) {
    return ids64 ? static_cast<const int64_t *>(ids)[t] : (int64_t) static_cast<const int32_t *>(ids)[t];
}

// ---- rows in registers ------------------------------------------------------
// A lane holds N = 16 / sizeof(T) values of a slab of 32 N columns: 16
// consecutive bytes where the rows are 16-byte aligned (VEC), else every 32nd
// column.
template <typename T> constexpr int kLaneN = 16 / (int)sizeof(T);

template <typename T, bool VEC>
__device__ __forceinline__ void load_lane(const T *__restrict__ row, int c0, int lane, int H, float *v) {
    constexpr int N = kLaneN<T>;
    if (VEC) {
        const int c = c0 + lane * N;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (c < H) u = *reinterpret_cast<const uint4 *>(row + c);
        const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = to_f(t[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int c = c0 + lane + 32 * k;
            v[k] = c < H ? to_f(row[c]) : 0.0f;
        }
    }
}

// the lane's columns: c0 + lane * N + k (VEC) or c0 + lane + 32 k
template <typename T, bool VEC> __device__ __forceinline__ int lane_col(int c0, int lane, int k) {
    return VEC ? c0 + lane * kLaneN<T> + k : c0 + lane + 32 * k;
}

// ---- forward ------------------------------------------------------------------
// one warp per token and up to 4 slabs; a token outside the table reads as
// zeros and sets the error word
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
embed_fwd_kernel(const void *__restrict__ ids, int ids64, int64_t tokens, const T *__restrict__ table, int64_t V,
                 int H, float scale, T *__restrict__ out, int32_t *__restrict__ err) {
    constexpr int N = kLaneN<T>, S = 4;
    const int groups = (H + 32 * N * S - 1) / (32 * N * S);
    const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const int64_t t = item / groups;
    if (t >= tokens) return;
    const int c0 = (int)(item % groups) * 32 * N * S;
    const int64_t id = token_id(ids, ids64, t);
    const bool ok = id >= 0 && id < V;
    if (!ok && lane == 0 && c0 == 0 && err) atomicOr(err, USAF_ERR_BAD_INDEX);
    float v[S][N];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        if (ok) load_lane<T, VEC>(table + id * H, c0 + s * 32 * N, lane, H, v[s]);
        else
#pragma unroll
            for (int k = 0; k < N; ++k) v[s][k] = 0.0f;
    }
    T *o = out + t * H;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        if (VEC) {
            uint4 u;
            T *w = reinterpret_cast<T *>(&u);
#pragma unroll
            for (int k = 0; k < N; ++k) w[k] = from_f<T>(v[s][k] * scale);
            const int c = c0 + s * 32 * N + lane * N;
            if (c < H) *reinterpret_cast<uint4 *>(o + c) = u;
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int c = c0 + s * 32 * N + lane + 32 * k;
                if (c < H) o[c] = from_f<T>(v[s][k] * scale);
            }
        }
    }
}

// ---- backward: sort and zeros ---------------------------------------------------
constexpr int kSortCtas = 8, kSortThreads = 1024, kSortWarps = 32, kMaxBins = 512;
constexpr int kChunk = 32;      // sorted positions a warp adds up

struct SortArgs {
    const void *ids; int ids64;
    int64_t V, pad;
    uint32_t tokens;
    int passes, width;          // digits of `width` bits
    uint32_t *key[2], *pos[2];  // pass i writes buffer i & 1
    int32_t *err;
    char *zero; int64_t zero_bytes;   // the gradient to clear, or none
};

__device__ __forceinline__ void zero_fill(char *p, int64_t n, int64_t tid, int64_t threads) {
    const int64_t head = min(n, (int64_t)(-(uintptr_t)p & 15));
    for (int64_t i = tid; i < head; i += threads) p[i] = 0;
    p += head;
    n -= head;
    const uint4 z = make_uint4(0, 0, 0, 0);
    for (int64_t i = tid; i < n / 16; i += threads) reinterpret_cast<uint4 *>(p)[i] = z;
    for (int64_t i = n / 16 * 16 + tid; i < n; i += threads) p[i] = 0;
}

// padding and tokens outside the table sort behind the table's rows, as row V
__device__ __forceinline__ uint32_t sort_key(const SortArgs &a, uint32_t j) {
    const int64_t id = token_id(a.ids, a.ids64, j);
    if (id < 0 || id >= a.V) {
        if (a.err) atomicOr(a.err, USAF_ERR_BAD_INDEX);
        return (uint32_t)a.V;
    }
    return id == a.pad ? (uint32_t)a.V : (uint32_t)id;
}

// Each CTA of the first cluster owns a contiguous eighth of the pairs, each of
// its warps a contiguous part of that.  A pass counts the digits per warp
// (equal digits of 32 pairs found by match), scans the counts over warps, CTAs
// (distributed shared memory) and digits, and moves every pair to its place:
// stable, since a warp walks its pairs in order.
__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads)
embed_sort_kernel(const SortArgs a) {
    extern __shared__ uint32_t hist[];                 // [32 warps][bins], then total [bins], base [bins]
    let_next_start();
    if (blockIdx.x >= kSortCtas) {
        zero_fill(a.zero, a.zero_bytes, (int64_t)(blockIdx.x - kSortCtas) * kSortThreads + threadIdx.x,
                  (int64_t)(gridDim.x - kSortCtas) * kSortThreads);
        return;
    }
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int bins = 1 << a.width;
    uint32_t *total = hist + kSortWarps * bins, *base = total + bins;
    __shared__ uint32_t scan[16];
    const uint32_t part = (a.tokens + kSortCtas * kSortWarps * 32 - 1) / (kSortCtas * kSortWarps * 32) * 32;
    const uint64_t first = (uint64_t)(blockIdx.x * kSortWarps + warp) * part;
    const uint32_t b = (uint32_t)min(first, (uint64_t)a.tokens), e = (uint32_t)min(first + part, (uint64_t)a.tokens);
    uint32_t *mine = hist + warp * bins;
    for (int pass = 0; pass < a.passes; ++pass) {
        const uint32_t *ksrc = a.key[(pass + 1) & 1], *psrc = a.pos[(pass + 1) & 1];
        uint32_t *kdst = a.key[pass & 1], *pdst = a.pos[pass & 1];
        const int shift = pass * a.width;
        for (int i = tid; i < kSortWarps * bins; i += kSortThreads) hist[i] = 0;
        __syncthreads();
        for (uint32_t j0 = b; j0 < e; j0 += 32) {
            const uint32_t j = j0 + lane;
            uint32_t d = bins;
            if (j < e) d = ((pass ? ksrc[j] : sort_key(a, j)) >> shift) & (bins - 1);
            const uint32_t same = __match_any_sync(0xffffffffu, d);
            if (j < e && lane == __ffs(same) - 1) mine[d] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
        if (tid < bins) {
            uint32_t run = 0;
            for (int w = 0; w < kSortWarps; ++w) {
                const uint32_t t = hist[w * bins + tid];
                hist[w * bins + tid] = run;
                run += t;
            }
            total[tid] = run;
        }
        cluster.sync();
        uint32_t all = 0, before = 0, inc = 0;
        if (tid < kMaxBins) {                          // whole warps; bins <= kMaxBins
            if (tid < bins) {
#pragma unroll
                for (int c = 0; c < kSortCtas; ++c) {
                    const uint32_t t = cluster.map_shared_rank(total, c)[tid];
                    if (c < (int)blockIdx.x) before += t;
                    all += t;
                }
            }
            inc = all;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += t;
            }
            if (lane == 31) scan[warp] = inc;
        }
        __syncthreads();
        if (tid < bins) {
            uint32_t add = 0;
            for (int w = 0; w < warp; ++w) add += scan[w];
            base[tid] = add + inc - all + before;
        }
        __syncthreads();
        for (uint32_t j0 = b; j0 < e; j0 += 32) {
            const uint32_t j = j0 + lane;
            uint32_t d = bins, key = 0;
            if (j < e) {
                key = pass ? ksrc[j] : sort_key(a, j);
                d = (key >> shift) & (bins - 1);
            }
            const uint32_t same = __match_any_sync(0xffffffffu, d);
            uint32_t to = 0;
            if (j < e) to = base[d] + mine[d] + __popc(same & ((1u << lane) - 1));
            __syncwarp();
            if (j < e) {
                if (lane == __ffs(same) - 1) mine[d] += __popc(same);
                kdst[to] = key;
                pdst[to] = pass ? psrc[j] : j;
            }
            __syncwarp();
        }
        cluster.sync();                                // the pass's pairs are in place, `total` is read
    }
}

// ---- backward: sums -----------------------------------------------------------
// the lane's 16 / sizeof(T) sums into its columns of a row of the gradient
template <typename T, typename G, bool VEC>
__device__ __forceinline__ void put_row(G *__restrict__ g, int c0, int lane, int H, const uint64_t *acc, float scale,
                                        int add) {
    constexpr int N2 = kPairs<T>;
    const uint64_t by = pair(scale, scale);
    if constexpr (VEC) {             // one or two vectors
        const int c = c0 + lane * 2 * N2;
        if (c >= H) return;
        uint4 *to = reinterpret_cast<uint4 *>(g + c);
#pragma unroll
        for (int i = 0; i < N2 / kPairs<G>; ++i) {
            uint64_t v[kPairs<G>];
            if (add) unpack<G>(to[i], v);
#pragma unroll
            for (int k = 0; k < kPairs<G>; ++k) {
                const uint64_t s = acc[i * kPairs<G> + k];
                v[k] = add ? fma2(s, by, v[k]) : mul2(s, by);
            }
            to[i] = pack<G>(v);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N2; ++k) {
            const float2 h = halves(acc[k]);
            const int c = c0 + lane + 64 * k;
            if (c < H) g[c] = from_f<G>(add ? fmaf(h.x, scale, to_f(g[c])) : h.x * scale);
            if (c + 32 < H) g[c + 32] = from_f<G>(add ? fmaf(h.y, scale, to_f(g[c + 32])) : h.y * scale);
        }
    }
}

// One warp per chunk and slab.  The chunk's rows come through a ring of kAhead
// slots of 16 bytes a lane in shared memory, filled by asynchronous copies (of 16
// bytes, or of 4 where fp32 rows are not aligned), so that 15 rows are on their
// way whatever the tokens are; 16-bit rows that are not aligned are loaded eight at
// a time.
constexpr int kAhead = 16;

template <typename T, typename G, bool VEC>
__global__ void __launch_bounds__(256)
embed_sum_kernel(const T *__restrict__ dy, const uint32_t *__restrict__ key, const uint32_t *__restrict__ pos,
                 uint32_t tokens, uint32_t V, int H, float scale, int add, G *__restrict__ grad,
                 float *__restrict__ part) {
    extern __shared__ uint4 dyn[];   // [kAhead][256 threads]
    constexpr int N = kLaneN<T>, N2 = N / 2;
    wait_for_previous();
    let_next_start();
    const int slabs = (H + 32 * N - 1) / (32 * N);
    const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const int64_t chunk = item / slabs;
    const int c0 = (int)(item % slabs) * 32 * N;
    const uint32_t b = (uint32_t)min((uint64_t)chunk * kChunk, (uint64_t)tokens);
    const int n = (int)min((uint32_t)kChunk, tokens - b);
    if (n <= 0) return;
    const uint32_t k_l = lane < n ? key[b + lane] : V, p_l = lane < n ? pos[b + lane] : 0;
    const uint32_t before = b ? key[b - 1] : V, after = b + n < tokens ? key[b + n] : V;
    const int live = __popc(__ballot_sync(0xffffffffu, k_l < V));     // row V sorts behind the others
    if (!live) return;
    uint4 *ring = dyn + threadIdx.x;
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(ring);
    auto fetch = [&](int i) {        // row i of the chunk into slot i % kAhead
        if constexpr (VEC || sizeof(T) == 4) {
            const uint32_t p = __shfl_sync(0xffffffffu, p_l, i & 31), to = at + (i % kAhead) * 4096;
            if (i < live) {
                const T *row = dy + (int64_t)p * H + c0;
                if constexpr (VEC) {
                    if (c0 + lane * N < H)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(row + lane * N) : "memory");
                } else {
#pragma unroll
                    for (int k = 0; k < N; ++k)
                        if (c0 + lane + 32 * k < H)
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 4 * k),
                                         "l"(row + lane + 32 * k)
                                         : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    };
    for (int i = 0; i < kAhead - 1; ++i) fetch(i);
    uint64_t acc[N2];
    uint32_t cur = V, first = V;
    for (int i = 0; i <= live; ++i) {
        const uint32_t k_i = __shfl_sync(0xffffffffu, k_l, i & 31);
        if (i == live || k_i != cur) {
            if (i > 0) {             // the row of `cur` is complete in this chunk
                const bool from = cur == before && cur == first, on = i == live && live == n && cur == after;
                if (!from && !on) {
                    put_row<T, G, VEC>(grad + (int64_t)cur * H, c0, lane, H, acc, scale, add);
                } else {             // slot 0: begun before this chunk, 1: begins in it
                    put_row<T, float, VEC>(part + (chunk * 2 + (from ? 0 : 1)) * H, c0, lane, H, acc, 1.0f, 0);
                }
            } else {
                first = k_i;
            }
            if (i == live) break;
            cur = k_i;
#pragma unroll
            for (int k = 0; k < N2; ++k) acc[k] = 0;
        }
        if constexpr (!VEC && sizeof(T) == 2) {
            if (i % 8 == 0) {
                T v[8][N];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t p = __shfl_sync(0xffffffffu, p_l, i + j);
                    if (i + j < live)
#pragma unroll
                        for (int k = 0; k < N; ++k)
                            v[j][k] = c0 + lane + 32 * k < H ? dy[(int64_t)p * H + c0 + lane + 32 * k] : T();
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (i + j < live) {
                        uint4 u;
#pragma unroll
                        for (int k = 0; k < N; ++k) reinterpret_cast<T *>(&u)[k] = v[j][k];
                        ring[((i + j) % kAhead) * 256] = u;
                    }
            }
        } else {
            fetch(i + kAhead - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        }
        uint64_t v[N2];
        unpack<T>(ring[(i % kAhead) * 256], v);
#pragma unroll
        for (int k = 0; k < N2; ++k) acc[k] = add2(acc[k], v[k]);
    }
}

// A CTA looks at 8 chunks, one a warp: where a chunk's last token begins in it and
// goes on, the chunks that it runs through are counted.  A token of few chunks is
// joined by its warp, 32 columns at a time; of many (a run of hundreds of partial
// sums) by all 8 warps, each a contiguous part, which are then added in order.
template <typename G>
__global__ void __launch_bounds__(256)
embed_join_kernel(const uint32_t *__restrict__ key, uint32_t tokens, uint32_t V, int H, float scale, int add,
                  G *__restrict__ grad, const float *__restrict__ part, int64_t chunks) {
    __shared__ float s[8][32];
    __shared__ int follow[8];
    __shared__ uint32_t token[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kFew = 12;
    auto put = [&](uint32_t k, int c, float v) {
        G *g = grad + (int64_t)k * H + c;
        *g = from_f<G>(add ? fmaf(v, scale, to_f(*g)) : v * scale);
    };
    wait_for_previous();
    const int64_t mine = (int64_t)blockIdx.x * 8 + warp;
    int n = 0;
    if (mine < chunks - 1) {
        const uint32_t b = (uint32_t)(mine * kChunk), e = b + kChunk;
        const uint32_t k = key[e - 1];
        if (k < V && key[e] == k && !(key[b] == k && b > 0 && key[b - 1] == k)) {
            for (;;) {               // chunks that begin with this token
                const uint64_t p = (uint64_t)e + (uint64_t)(n + lane) * kChunk;
                const int got = __popc(__ballot_sync(0xffffffffu, p < tokens && key[p] == k));
                n += got;
                if (got < 32) break;
            }
        }
        if (n > 0 && n <= kFew) {
            for (int c = blockIdx.y * 32 + lane; c < H; c += gridDim.y * 32) {
                float v[kFew + 1];
#pragma unroll
                for (int i = 0; i <= kFew; ++i)
                    v[i] = i <= n ? part[((mine + i) * 2 + (i == 0 ? 1 : 0)) * H + c] : 0.0f;
                float t = v[0];
#pragma unroll
                for (int i = 1; i <= kFew; ++i)
                    if (i <= n) t += v[i];
                put(k, c, t);
            }
            n = 0;
        }
        if (lane == 0) token[warp] = k;
    }
    if (lane == 0) follow[warp] = n;
    __syncthreads();
    for (int w = 0; w < 8; ++w) {
        const int m = follow[w] + 1, each = (m + 7) / 8;
        if (m == 1) continue;
        const int64_t chunk = (int64_t)blockIdx.x * 8 + w;
        for (int c = blockIdx.y * 32 + lane; c - lane < H; c += gridDim.y * 32) {
            float v = 0.0f;
            if (c < H) {
#pragma unroll 8
                for (int i = warp * each; i < min(m, (warp + 1) * each); ++i)
                    v += part[((chunk + i) * 2 + (i == 0 ? 1 : 0)) * H + c];
            }
            s[warp][lane] = v;
            __syncthreads();
            if (warp == 0 && c < H) {
                float t = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) t += s[i][lane];
                put(token[w], c, t);
            }
            __syncthreads();
        }
    }
}

struct EmbedBwd {
    const void *dy, *ids; int ids64;
    int64_t tokens, V; int H; float scale; int64_t pad; int add;
    void *grad, *ws; int32_t *err;
};

static inline int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

static int64_t embed_ws_bytes(int64_t tokens, int H) {
    const int64_t chunks = (tokens + kChunk - 1) / kChunk;
    return 4 * up256(tokens * 4) + (chunks > 1 ? chunks * 2 * H * 4 : 0);
}

template <typename T, typename G> static int embed_bwd(const EmbedBwd &a, cudaStream_t st) {
    SortArgs s;
    s.ids = a.ids;
    s.ids64 = a.ids64;
    s.V = a.V;
    s.pad = a.pad;
    s.tokens = (uint32_t)a.tokens;
    char *w = static_cast<char *>(a.ws);
    for (int i = 0; i < 2; ++i) {
        s.key[i] = reinterpret_cast<uint32_t *>(w + (2 * i) * up256(a.tokens * 4));
        s.pos[i] = reinterpret_cast<uint32_t *>(w + (2 * i + 1) * up256(a.tokens * 4));
    }
    float *part = reinterpret_cast<float *>(w + 4 * up256(a.tokens * 4));
    int bits = 1;                                      // of row V, the last key
    while ((a.V >> bits) != 0) ++bits;
    s.passes = (bits + 8) / 9;
    s.width = (bits + s.passes - 1) / s.passes;
    s.err = a.err;
    s.zero = static_cast<char *>(a.grad);
    s.zero_bytes = a.add ? 0 : a.V * (int64_t)a.H * (int64_t)sizeof(G);
    // two CTAs per SM write zeros, fewer where that is less than 16 KB each
    const int64_t fill = std::min<int64_t>(36, (s.zero_bytes + kSortCtas * 16384 - 1) / (kSortCtas * 16384));
    const int bins = 1 << s.width, smem = (kSortWarps + 2) * bins * 4;
    if (smem > 48 * 1024 && cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (kSortWarps + 2) * kMaxBins * 4) != cudaSuccess) {
        (void)cudaGetLastError();
        return USAF_ECUDA;
    }
    embed_sort_kernel<<<(unsigned)(kSortCtas * (1 + fill)), kSortThreads, smem, st>>>(s);
    USAF_CHECK_LAUNCH();
    if (a.tokens == 0) return USAF_OK;
    const uint32_t *key = s.key[(s.passes - 1) & 1], *pos = s.pos[(s.passes - 1) & 1];
    const int64_t chunks = (a.tokens + kChunk - 1) / kChunk;
    const int slabs = (a.H + 32 * kLaneN<T> - 1) / (32 * kLaneN<T>);
    const unsigned grid = cdiv(chunks * slabs, 8);
    // 16-byte vectors of dy's rows, of the gradient's and of the partial sums
    const bool vec = ((uintptr_t)a.dy | (uintptr_t)a.grad | (uintptr_t)a.ws) % 16 == 0 && (int64_t)a.H * sizeof(T) % 16 == 0;
    auto sum = vec ? embed_sum_kernel<T, G, true> : embed_sum_kernel<T, G, false>;
    const int ring = kAhead * 256 * 16;
    if (cudaFuncSetAttribute(sum, cudaFuncAttributeMaxDynamicSharedMemorySize, ring) != cudaSuccess) {
        (void)cudaGetLastError();
        return USAF_ECUDA;
    }
    if (!launch_early(sum, dim3(grid), 256, ring, st, (const T *)a.dy, key, pos, (uint32_t)a.tokens, (uint32_t)a.V, a.H,
                      a.scale, a.add, (G *)a.grad, part))
        return USAF_ECUDA;
    if (chunks > 1) {
        const dim3 jgrid(cdiv(chunks - 1, 8), (unsigned)std::min((a.H + 31) / 32, 64));
        if (!launch_early(embed_join_kernel<G>, jgrid, 256, 0, st, key, (uint32_t)a.tokens, (uint32_t)a.V, a.H, a.scale,
                          a.add, (G *)a.grad, (const float *)part, chunks))
            return USAF_ECUDA;
    }
    return USAF_OK;
}

template <typename T>
static void embed_fwd(const void *ids, int ids64, int64_t tokens, const void *table, int64_t V, int H, float scale,
                      void *out, int32_t *err, cudaStream_t st) {
    const int group = 32 * kLaneN<T> * 4;
    const unsigned grid = cdiv(tokens * ((H + group - 1) / group), 8);
    const bool vec = ((uintptr_t)table | (uintptr_t)out) % 16 == 0 && (int64_t)H * sizeof(T) % 16 == 0;
    if (vec)
        embed_fwd_kernel<T, true><<<grid, 256, 0, st>>>(ids, ids64, tokens, (const T *)table, V, H, scale, (T *)out, err);
    else
        embed_fwd_kernel<T, false><<<grid, 256, 0, st>>>(ids, ids64, tokens, (const T *)table, V, H, scale, (T *)out, err);
}

}  // namespace usaf

using namespace usaf;

// positions and rows are 32-bit in the sort; a launch has at most 2^31 - 1 CTAs
constexpr int64_t kMostTokens = (int64_t)1 << 30, kMostRows = (int64_t)1 << 30;

extern "C" int usaf_embedding_fwd(const void *ids, int32_t ids_bits, int64_t tokens, const void *table, int32_t dtype,
                                  int64_t V, int32_t H, double scale, void *out, int32_t *err, void *stream) {
    USAF_REQUIRE(tokens >= 0 && V >= 0 && H >= 1 && (ids_bits == 32 || ids_bits == 64));
    if (tokens == 0) return USAF_OK;
    USAF_REQUIRE(ids && (table || V == 0) && out);
    if (tokens > kMostTokens || tokens * ((H + 511) / 512) > ((int64_t)1 << 33)) return USAF_EUNSUPPORTED;
    cudaStream_t st = as_stream(stream);
    const int wide = ids_bits == 64;
    switch (dtype) {
        case USAF_F32: embed_fwd<float>(ids, wide, tokens, table, V, H, (float)scale, out, err, st); break;
        case USAF_BF16: embed_fwd<__nv_bfloat16>(ids, wide, tokens, table, V, H, (float)scale, out, err, st); break;
        case USAF_F16: embed_fwd<__half>(ids, wide, tokens, table, V, H, (float)scale, out, err, st); break;
        default: return USAF_EINVAL;
    }
    USAF_CHECK_LAUNCH();
    return USAF_OK;
}

extern "C" int64_t usaf_embedding_workspace_bytes(int64_t tokens, int64_t V, int32_t H) {
    if (tokens < 0 || V < 0 || H < 1) return -1;
    return embed_ws_bytes(tokens, H);
}

extern "C" int usaf_embedding_bwd(const void *dy, const void *ids, int32_t ids_bits, int64_t tokens, int32_t dtype,
                                  int64_t V, int32_t H, double scale, int64_t padding_idx, int32_t accumulate,
                                  void *grad, int32_t grad_dtype, void *ws, int32_t *err, void *stream) {
    USAF_REQUIRE(tokens >= 0 && V >= 0 && H >= 1 && (ids_bits == 32 || ids_bits == 64));
    USAF_REQUIRE((grad || V == 0) && (tokens == 0 || (dy && ids && ws)));
    if (tokens > kMostTokens || V > kMostRows || (tokens / kChunk + 1) * ((H + 127) / 128) > ((int64_t)1 << 33))
        return USAF_EUNSUPPORTED;
    cudaStream_t st = as_stream(stream);
    const EmbedBwd a{dy, ids, ids_bits == 64, tokens, V, H, (float)scale, padding_idx, accumulate, grad, ws, err};
    switch (dtype * 4 + grad_dtype) {
        case USAF_F32 * 4 + USAF_F32: return embed_bwd<float, float>(a, st);
        case USAF_BF16 * 4 + USAF_BF16: return embed_bwd<__nv_bfloat16, __nv_bfloat16>(a, st);
        case USAF_BF16 * 4 + USAF_F32: return embed_bwd<__nv_bfloat16, float>(a, st);
        case USAF_F16 * 4 + USAF_F16: return embed_bwd<__half, __half>(a, st);
        case USAF_F16 * 4 + USAF_F32: return embed_bwd<__half, float>(a, st);
        default: return USAF_EINVAL;
    }
}
