// Embedding lookup y[t] = scale W[id_t] and the gradient of the table,
// dW[v] = scale * (sum of dy[t] over the tokens t with id_t = v, ascending t).
//
// The gradient takes four launches, each set up while the one before runs:
//   1. sort: one cluster of 8 CTAs sorts the (token, position) pairs by a stable
//      radix sort (digits of up to 9 bits, so two passes for a table of fewer than
//      2^18 rows: the number of rows is a key of its own, of padding);
//      zeros: on the other SMs at the same time, the table's gradient is cleared,
//      which is where the time goes (V x H values against tokens x H);
//   2. sum: the sorted positions are cut into chunks of 32, whatever tokens they
//      hold, so that a frequent token spreads over many warps; a warp adds the
//      rows of its chunk in fp32, writes the rows of tokens that lie in the chunk
//      as a whole and leaves fp32 partial sums of the first and the last token
//      where these go on in a neighbour;
//   3. join: the chunk in which such a token begins adds the partial sums of the
//      chunks it runs through, in chunk order.
// Nothing is added atomically: the sums' order is that of the positions.
// 8192 tokens of a 151936 x 2048 bf16 table: 117 us with the lookup (10), of which
// the zeros are 84, where the bytes take 109 at the measured copy rate; 16384 live
// tokens of 1001 fp32 values added to a gradient: sort 23, sums 28, joins 10.
#include <cooperative_groups.h>

#include "common.cuh"
#include "f32x2.cuh"

namespace cg = cooperative_groups;

namespace usaf {

__device__ __forceinline__ int64_t token_id(const void *ids, int ids64, int64_t t) {
    return ids64 ? static_cast<const int64_t *>(ids)[t] : (int64_t) static_cast<const int32_t *>(ids)[t];
}

// ---- forward ------------------------------------------------------------------
// A lane holds N = 16 / sizeof(T) values of a slab of 32 N columns: 16
// consecutive bytes where the rows are 16-byte aligned (VEC), else every 32nd
// column.  One warp takes a token and up to 8 slabs, all loaded before the first
// is stored; a token outside the table reads as zeros and sets the error word.
template <typename T> constexpr int kLaneN = 16 / (int)sizeof(T);
constexpr int kFwdSlabs = 8;

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
embed_fwd_kernel(const void *ids, int ids64, int64_t tokens, const T *table, int64_t V, int H, float scale, T *out,
                 int32_t *err) {
    constexpr int N = kLaneN<T>, S = kFwdSlabs;
    wait_for_previous();
    const int groups = (H + 32 * N * S - 1) / (32 * N * S);
    const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const int64_t t = item / groups;
    if (t >= tokens) return;
    const int c0 = (int)(item % groups) * 32 * N * S;
    const int64_t id = token_id(ids, ids64, t);
    const bool ok = id >= 0 && id < V;
    if (!ok && lane == 0 && c0 == 0 && err) atomicOr(err, USAF_ERR_BAD_INDEX);
    const T *row = table + (ok ? id * H : 0);
    T *o = out + t * H;
    if constexpr (VEC) {
        uint4 u[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int c = c0 + s * 32 * N + lane * N;
            u[s] = make_uint4(0, 0, 0, 0);
            if (ok && c < H) u[s] = *reinterpret_cast<const uint4 *>(row + c);
        }
        const uint64_t by = pair(scale, scale);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int c = c0 + s * 32 * N + lane * N;
            uint64_t v[kPairs<T>];
            unpack<T>(u[s], v);
#pragma unroll
            for (int k = 0; k < kPairs<T>; ++k) v[k] = mul2(v[k], by);
            if (c < H) *reinterpret_cast<uint4 *>(o + c) = pack<T>(v);
        }
    } else {
        T v[S * N];
#pragma unroll
        for (int k = 0; k < S * N; ++k) v[k] = ok && c0 + lane + 32 * k < H ? row[c0 + lane + 32 * k] : from_f<T>(0.0f);
#pragma unroll
        for (int k = 0; k < S * N; ++k)
            if (c0 + lane + 32 * k < H) o[c0 + lane + 32 * k] = from_f<T>(to_f(v[k]) * scale);
    }
}

// ---- backward: sort and zeros ---------------------------------------------------
constexpr int kSortCtas = 8, kSortThreads = 1024, kSortWarps = 32, kMaxBins = 512;
constexpr int kRound = 8;       // pairs a lane loads at once
constexpr int kChunk = 32;      // sorted positions a warp adds up

struct SortArgs {
    const void *ids; int ids64;
    int64_t V, pad;
    uint32_t tokens;
    int passes, width;          // digits of `width` bits
    uint2 *pairs[2];            // (key, position); pass i writes buffer i & 1
    int32_t *err;
};

// A CTA clears its 32 KB of the gradient, so many CTAs one after another: 86 us
// for 622 MB, as the runtime's memset; CTAs that walk through all of it, one or two
// an SM, took 103 us, and whole clusters of the sort's launch 240.  It runs beside
// the sort, which it does not need; its last CTAs wait for the sort, so that what
// waits for the zeros has both.
constexpr int kZeroTile = 32768, kZeroThreads = 512;

__global__ void __launch_bounds__(kZeroThreads) embed_zero_kernel(char *p, int64_t n) {
    const int64_t head = min(n, (int64_t)(-(uintptr_t)p & 15)), tile = blockIdx.x;
    let_next_start();
    if (tile == 0 && threadIdx.x < head) p[threadIdx.x] = 0;
    p += head;
    n -= head;
    uint4 *v = reinterpret_cast<uint4 *>(p);
#pragma unroll
    for (int i = 0; i < kZeroTile / 16 / kZeroThreads; ++i) {
        const int64_t at = tile * (kZeroTile / 16) + i * kZeroThreads + threadIdx.x;
        if (at < n / 16) v[at] = make_uint4(0, 0, 0, 0);
    }
    if (tile == n / kZeroTile && threadIdx.x < (n & 15)) p[n - 1 - threadIdx.x] = 0;
    if (blockIdx.x + 1 == gridDim.x) wait_for_previous();
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

// the lanes of the warp with this lane's digit: a vote per bit (match_any, which
// does the same, took 4.5 us for 4 digits a lane of 32 warps, the votes under 1)
__device__ __forceinline__ uint32_t same_digit(uint32_t d, int bits) {
    uint32_t same = 0xffffffffu;
    for (int i = 0; i < bits; ++i) {
        const uint32_t set = __ballot_sync(0xffffffffu, d >> i & 1);
        same &= d >> i & 1 ? set : ~set;
    }
    return same;
}

// Each CTA of the cluster owns a contiguous eighth of the pairs, each of
// its warps a contiguous part of that.  A pass counts the digits per warp, scans
// the counts over warps, CTAs (distributed shared memory) and digits, and moves
// every pair to its place: stable, since a warp walks its pairs in order.
__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads)
embed_sort_kernel(const SortArgs a) {
    extern __shared__ uint32_t hist[];                 // [32 warps][bins]; total, base [bins]; sums [4][bins]
    wait_for_previous();             // before the zeros may start: all that was enqueued before has ended
    let_next_start();
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int bins = 1 << a.width;
    uint32_t *total = hist + kSortWarps * bins, *base = total + bins, *sums = base + bins;
    __shared__ uint32_t scan[16];
    const uint32_t part = (a.tokens + kSortCtas * kSortWarps * 32 - 1) / (kSortCtas * kSortWarps * 32) * 32;
    const uint64_t first = (uint64_t)(blockIdx.x * kSortWarps + warp) * part;
    const uint32_t b = (uint32_t)min(first, (uint64_t)a.tokens), e = (uint32_t)min(first + part, (uint64_t)a.tokens);
    uint32_t *mine = hist + warp * bins;
    const bool once = part <= 32 * kRound;              // a warp's pairs stay in its registers for a pass
    const int split = min(4, kSortThreads / bins);      // threads that scan a digit's counts of the warps
    for (int pass = 0; pass < a.passes; ++pass) {
        const uint2 *src = a.pairs[(pass + 1) & 1];
        uint2 *dst = a.pairs[pass & 1];
        const int shift = pass * a.width;
        uint2 item[kRound];                             // and the lanes with the same digit
        uint32_t same[kRound];
#pragma unroll
        for (int r = 0; r < kRound; ++r) item[r] = make_uint2(0, 0);
        auto load = [&](uint32_t j0) {
#pragma unroll
            for (int r = 0; r < kRound; ++r) {
                const uint32_t j = j0 + 32 * r + lane;
                if (j < e) item[r] = pass ? src[j] : make_uint2(sort_key(a, j), j);
            }
        };
        for (int i = tid; i < kSortWarps * bins; i += kSortThreads) hist[i] = 0;
        if (once) load(b);
        __syncthreads();
        for (uint32_t j0 = b; j0 < e; j0 += 32 * kRound) {
            if (!once) load(j0);
#pragma unroll
            for (int r = 0; r < kRound; ++r) {
                if (j0 + 32 * r >= e) break;
                const bool in = j0 + 32 * r + lane < e;
                const uint32_t d = (item[r].x >> shift) & (bins - 1);
                same[r] = same_digit(d, a.width) & __ballot_sync(0xffffffffu, in);
                if (in && lane == __ffs(same[r]) - 1) mine[d] += __popc(same[r]);
                __syncwarp();
            }
        }
        __syncthreads();
        {                                               // a digit's counts: `split` threads, in whole warps
            const int d = tid & (bins - 1), q = tid >> a.width, each = kSortWarps / split;
            uint32_t run = 0;
            if (q < split) {
#pragma unroll 8
                for (int w = q * each; w < (q + 1) * each; ++w) run += hist[w * bins + d];
                sums[q * bins + d] = run;
            }
            __syncthreads();
            if (q < split) {
                uint32_t at = 0;
                for (int k = 0; k < q; ++k) at += sums[k * bins + d];
                if (q == split - 1) total[d] = at + run;
#pragma unroll 8
                for (int w = q * each; w < (q + 1) * each; ++w) {
                    const uint32_t t = hist[w * bins + d];
                    hist[w * bins + d] = at;
                    at += t;
                }
            }
        }
        cluster.sync();
        uint32_t all = 0, before = 0, inc = 0;
        if (tid < kMaxBins) {                          // whole warps; bins <= kMaxBins
            if (tid < bins) {
                uint32_t t[kSortCtas];
#pragma unroll
                for (int c = 0; c < kSortCtas; ++c) t[c] = cluster.map_shared_rank(total, c)[tid];
#pragma unroll
                for (int c = 0; c < kSortCtas; ++c) {
                    if (c < (int)blockIdx.x) before += t[c];
                    all += t[c];
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
        for (uint32_t j0 = b; j0 < e; j0 += 32 * kRound) {
            if (!once) load(j0);
#pragma unroll
            for (int r = 0; r < kRound; ++r) {
                if (j0 + 32 * r >= e) break;
                const bool in = j0 + 32 * r + lane < e;
                const uint32_t d = (item[r].x >> shift) & (bins - 1);
                if (!once) same[r] = same_digit(d, a.width) & __ballot_sync(0xffffffffu, in);
                const uint32_t to = base[d] + mine[d] + __popc(same[r] & ((1u << lane) - 1));
                __syncwarp();
                if (in) {
                    if (lane == __ffs(same[r]) - 1) mine[d] += __popc(same[r]);
                    dst[to] = item[r];
                }
                __syncwarp();
            }
        }
        cluster.sync();                                // the pass's pairs are in place, `total` is read
    }
}

// Up to 512 pairs of a table of up to 2^23 - 2 rows: key and position fit 32 bits
// together, and one CTA counts for every pair those that are smaller, 4 a load.
// The cluster's passes and barriers take 12 us whatever they sort.
constexpr int kFewTokens = 512;
constexpr int64_t kFewRows = (1 << 23) - 2;

__global__ void __launch_bounds__(2 * kFewTokens) embed_sort_few_kernel(const SortArgs a, uint2 *sorted) {
    __shared__ alignas(16) uint32_t keys[kFewTokens];
    wait_for_previous();
    let_next_start();
    // two threads a pair, each over every other four keys
    const uint32_t j = threadIdx.x >> 1, half = threadIdx.x & 1;
    const uint32_t key = j < a.tokens ? sort_key(a, j) : 0, mine = j < a.tokens ? key << 9 | j : 0xffffffffu;
    if (half == 0) keys[j] = mine;
    __syncthreads();
    uint32_t to = 0;
    const uint32_t n = (a.tokens + 3) / 4;              // what lies behind the tokens is larger than any
#pragma unroll 4
    for (uint32_t i = half; i < n; i += 2) {
        const uint4 k = reinterpret_cast<const uint4 *>(keys)[i];
        to += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
    }
    to += __shfl_xor_sync(0xffffffffu, to, 1);
    if (half == 0 && j < a.tokens) sorted[to] = make_uint2(key, j);
}

// ---- backward: sums -----------------------------------------------------------
// A slab is 32 lanes times NV vectors of 16 bytes of T; a lane's values are those
// of vectors lane, 32 + lane, ... (VEC), else every 32nd column.  From a slot of the
// ring that holds a row of X (T, or the gradient's fp32) of the slab, `shift` bytes
// behind the slot's beginning:
template <typename T, typename X, int NV, bool VEC>
__device__ __forceinline__ void read_slot(const char *slot, int shift, int c0, int lane, int H, uint64_t *v) {
    constexpr int N2 = kPairs<T>, R = N2 / kPairs<X>;
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < R; ++i)
                unpack<X>(reinterpret_cast<const uint4 *>(slot)[(j * 32 + lane) * R + i], v + j * N2 + i * kPairs<X>);
    } else {
        const X *t = reinterpret_cast<const X *>(slot + shift) + lane;
#pragma unroll
        for (int k = 0; k < NV * N2; ++k) {
            const int c = c0 + lane + 64 * k;
            v[k] = pair(c < H ? to_f(t[64 * k]) : 0.0f, c + 32 < H ? to_f(t[64 * k + 32]) : 0.0f);
        }
    }
}

// the lane's sums into its columns of a row
template <typename T, typename X, int NV, bool VEC>
__device__ __forceinline__ void put_row(X *row, int c0, int lane, int H, const uint64_t *v) {
    constexpr int N2 = kPairs<T>;
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = c0 + (j * 32 + lane) * 2 * N2;
            if (c < H)
#pragma unroll
                for (int i = 0; i < N2 / kPairs<X>; ++i)
                    reinterpret_cast<uint4 *>(row + c)[i] = pack<X>(v + j * N2 + i * kPairs<X>);
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV * N2; ++k) {
            const float2 h = halves(v[k]);
            const int c = c0 + lane + 64 * k;
            if (c < H) row[c] = from_f<X>(h.x);
            if (c + 32 < H) row[c + 32] = from_f<X>(h.y);
        }
    }
}

// One warp per chunk and slab.  The chunk's rows come through a ring of kAhead
// slots in shared memory, filled by asynchronous copies of 16 bytes, so that many
// rows are on their way whatever the tokens are; where the sums are added to a
// gradient, its row follows a token's last row through the same ring (loaded where
// it was needed, its latency once a token took two thirds of the time).  Of a row
// that is not aligned the 16-byte vectors around the slab are fetched: each holds
// a value of the row, so it lies in the tensor's memory.
template <int NV> constexpr int kAhead = NV == 1 ? 16 : 8;
template <typename T, typename G, int NV, bool VEC>
constexpr int kSlot = 512 * NV * (int)(sizeof(G) / sizeof(T)) + (VEC ? 0 : 16);

template <typename T, typename G, int NV, bool VEC>
__global__ void __launch_bounds__(256)
embed_sum_kernel(const T *dy, const uint2 *sorted, uint32_t tokens, uint32_t V, int H, float scale, int add, G *grad,
                 float *part) {
    constexpr int N = kLaneN<T> * NV, N2 = N / 2, D = kAhead<NV>, S = kSlot<T, G, NV, VEC>;
    extern __shared__ uint4 dyn[];   // [8 warps][D][S bytes]
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
    const uint2 own = lane < n ? sorted[b + lane] : make_uint2(V, 0);
    const uint32_t k_l = own.x, p_l = own.y;
    const uint32_t before = b ? sorted[b - 1].x : V, after = b + n < tokens ? sorted[b + n].x : V;
    const int live = __popc(__ballot_sync(0xffffffffu, k_l < V));     // row V sorts behind the others
    if (!live) return;
    // bit i: position i is its token's last in this chunk; begun before it, going on behind it
    const uint32_t follows = __shfl_down_sync(0xffffffffu, k_l, 1), first = __shfl_sync(0xffffffffu, k_l, 0);
    const uint32_t last = __ballot_sync(0xffffffffu, lane < live && (lane == live - 1 || follows != k_l));
    const uint32_t from = __ballot_sync(0xffffffffu, k_l == first && first == before);
    const uint32_t on = __ballot_sync(0xffffffffu, live == n && k_l == after);
    const uint32_t whole = last & ~from & ~on, with = add ? whole : 0;    // rows to write; gradient rows to read first
    char *ring = reinterpret_cast<char *>(dyn) + (threadIdx.x >> 5) * (D * S);
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
    const int width = min(32 * N, H - c0);
    const char *dy0 = reinterpret_cast<const char *>(dy + c0), *grad0 = reinterpret_cast<const char *>(grad + c0);
    // bytes that a row begins behind a 16-byte boundary (32 bits hold what matters)
    auto shift_of = [&](const char *base, uint32_t row, int size) {
        return VEC ? 0 : (int)(((uint32_t)(uintptr_t)base + row * (uint32_t)H * (uint32_t)size) & 15);
    };
    auto copy_row = [&](int slot, const char *base, uint32_t row, int size, int most) {
        const int shift = shift_of(base, row, size), bytes = width * size + shift;
        const char *src = base + (int64_t)row * H * size - shift + lane * 16;
#pragma unroll
        for (int i = 0; i <= most; ++i)
            if (lane * 16 + 512 * i < bytes && (i < most || !VEC))
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + slot * S + 512 * i), "l"(src + 512 * i)
                             : "memory");
    };
    int f_row = 0, f_slot = 0;       // next to fetch: the row of position f_row, or the gradient row behind it
    bool f_grad = false;
    auto fetch = [&] {
        if (f_row < live) {
            const uint32_t r = __shfl_sync(0xffffffffu, f_grad ? k_l : p_l, f_row);
            if (f_grad) copy_row(f_slot, grad0, r, sizeof(G), NV * (int)(sizeof(G) / sizeof(T)));
            else copy_row(f_slot, dy0, r, sizeof(T), NV);
            f_grad = !f_grad && (with >> f_row & 1);
            f_row += !f_grad;
            f_slot = (f_slot + 1) % D;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int slot = 0;
    // the next slot is there, and every lane has read the one that is filled now
    auto next = [&] {
        asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
        __syncwarp();
        fetch();
        const char *s = ring + slot * S;
        slot = (slot + 1) % D;
        return s;
    };
    for (int i = 0; i < D - 1; ++i) fetch();
    uint64_t acc[N2], v[N2];
#pragma unroll
    for (int k = 0; k < N2; ++k) acc[k] = 0;
    for (int i = 0; i < live; ++i) {
        const int shift = VEC ? 0 : shift_of(dy0, __shfl_sync(0xffffffffu, p_l, i), sizeof(T));
        read_slot<T, T, NV, VEC>(next(), shift, c0, lane, H, v);
#pragma unroll
        for (int k = 0; k < N2; ++k) acc[k] = add2(acc[k], v[k]);
        if (last >> i & 1) {
            if (whole >> i & 1) {
                const uint32_t token = __shfl_sync(0xffffffffu, k_l, i);
                const uint64_t by = pair(scale, scale);
                if (add) {
                    read_slot<T, G, NV, VEC>(next(), shift_of(grad0, token, sizeof(G)), c0, lane, H, v);
#pragma unroll
                    for (int k = 0; k < N2; ++k) acc[k] = fma2(acc[k], by, v[k]);
                } else {
#pragma unroll
                    for (int k = 0; k < N2; ++k) acc[k] = mul2(acc[k], by);
                }
                put_row<T, G, NV, VEC>(grad + (int64_t)token * H, c0, lane, H, acc);
            } else {                 // slot 0: begun before this chunk, 1: begins in it
                put_row<T, float, NV, VEC>(part + (chunk * 2 + (from >> i & 1 ? 0 : 1)) * H, c0, lane, H, acc);
            }
#pragma unroll
            for (int k = 0; k < N2; ++k) acc[k] = 0;
        }
    }
}

// A CTA looks at 8 chunks, one a warp: where a chunk's last token begins in it and
// goes on, the chunks that it runs through are counted.  A token of few chunks is
// joined by its warp, 128 columns a CTA; of many (a run of hundreds of partial
// sums) by all 8 warps, each a contiguous part, which are then added in order.
template <typename G>
__global__ void __launch_bounds__(256)
embed_join_kernel(const uint2 *sorted, uint32_t tokens, uint32_t V, int H, float scale, int add, G *grad,
                  const float *part, int64_t chunks) {
    __shared__ float s[8][128];
    __shared__ int follow[8];
    __shared__ uint32_t token[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kFew = 16;
    const int c0 = blockIdx.y * 128 + lane;             // columns c0, c0 + 32, c0 + 64, c0 + 96
    auto put = [&](uint32_t k, int c, float v) {
        G *g = grad + (int64_t)k * H + c;
        *g = from_f<G>(add ? fmaf(v, scale, to_f(*g)) : v * scale);
    };
    // partial sums [i0, i1) of a token that begins in `chunk`, in order
    auto sums = [&](int64_t chunk, int i0, int i1, float *t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = 0.0f;
#pragma unroll 4
        for (int i = i0; i < i1; ++i) {
            const float *p = part + ((chunk + i) * 2 + (i == 0 ? 1 : 0)) * H;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c0 + 32 * j < H) t[j] += p[c0 + 32 * j];
        }
    };
    float t[4];
    wait_for_previous();
    const int64_t mine = (int64_t)blockIdx.x * 8 + warp;
    int n = 0;
    if (mine < chunks - 1) {
        const uint32_t b = (uint32_t)(mine * kChunk), e = b + kChunk;
        // the keys around, and those that the chunks behind begin with
        const uint32_t k = sorted[e - 1].x, front = sorted[b].x, before = b ? sorted[b - 1].x : V;
        uint64_t p = (uint64_t)e + (uint64_t)lane * kChunk;
        uint32_t ahead = p < tokens ? sorted[p].x : V;
        if (k < V && !(front == k && before == k)) {
            for (;;) {
                const int got = __popc(__ballot_sync(0xffffffffu, ahead == k));
                n += got;
                if (got < 32) break;
                p += 32 * kChunk;
                ahead = p < tokens ? sorted[p].x : V;
            }
        }
        if (n > 0 && n <= kFew) {
            sums(mine, 0, n + 1, t);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c0 + 32 * j < H) put(k, c0 + 32 * j, t[j]);
            n = 0;
        }
        if (lane == 0) token[warp] = k;
    }
    if (lane == 0) follow[warp] = n;
    __syncthreads();
    for (int w = 0; w < 8; ++w) {
        const int m = follow[w] + 1, each = (m + 7) / 8;
        if (m == 1) continue;
        sums((int64_t)blockIdx.x * 8 + w, min(m, warp * each), min(m, (warp + 1) * each), t);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[warp][lane + 32 * j] = t[j];
        __syncthreads();
        if (threadIdx.x < 128 && blockIdx.y * 128 + threadIdx.x < H) {
            float v = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) v += s[i][threadIdx.x];
            put(token[w], blockIdx.y * 128 + threadIdx.x, v);
        }
        __syncthreads();
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
    return 2 * up256(tokens * 8) + (chunks > 1 ? chunks * 2 * H * 4 : 0);
}

template <typename T, typename G, int NV, bool VEC>
static int sum_launch(const EmbedBwd &a, const uint2 *sorted, int64_t chunks, float *part, cudaStream_t st) {
    constexpr int smem = 8 * kAhead<NV> * kSlot<T, G, NV, VEC>, slab = 32 * NV * kLaneN<T>;
    auto kernel = embed_sum_kernel<T, G, NV, VEC>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
        (void)cudaGetLastError();
        return USAF_ECUDA;
    }
    const unsigned grid = cdiv(chunks * ((a.H + slab - 1) / slab), 8);
    return launch_early(kernel, dim3(grid), 256, smem, st, (const T *)a.dy, sorted, (uint32_t)a.tokens, (uint32_t)a.V, a.H,
                        a.scale, a.add, (G *)a.grad, part)
               ? USAF_OK
               : USAF_ECUDA;
}

template <typename T, typename G> static int embed_bwd(const EmbedBwd &a, cudaStream_t st) {
    SortArgs s;
    s.ids = a.ids;
    s.ids64 = a.ids64;
    s.V = a.V;
    s.pad = a.pad;
    s.tokens = (uint32_t)a.tokens;
    char *w = static_cast<char *>(a.ws);
    for (int i = 0; i < 2; ++i) s.pairs[i] = reinterpret_cast<uint2 *>(w + i * up256(a.tokens * 8));
    float *part = reinterpret_cast<float *>(w + 2 * up256(a.tokens * 8));
    int bits = 1;                                      // of row V, the last key
    while ((a.V >> bits) != 0) ++bits;
    s.passes = (bits + 8) / 9;
    s.width = (bits + s.passes - 1) / s.passes;
    s.err = a.err;
    const int bins = 1 << s.width, smem = (kSortWarps + 6) * bins * 4;
    if (smem > 47 * 1024 && cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (kSortWarps + 6) * kMaxBins * 4) != cudaSuccess) {
        (void)cudaGetLastError();
        return USAF_ECUDA;
    }
    const int64_t zero = a.add ? 0 : a.V * (int64_t)a.H * (int64_t)sizeof(G);
    if (a.tokens == 0) {             // nothing sorted: nothing that the zeros may start beside
        if (zero && cudaMemsetAsync(a.grad, 0, (size_t)zero, st) != cudaSuccess) {
            (void)cudaGetLastError();
            return USAF_ECUDA;
        }
        return USAF_OK;
    }
    const bool few = a.tokens <= kFewTokens && a.V <= kFewRows;
    if (!(few ? launch_early(embed_sort_few_kernel, dim3(1), 2 * kFewTokens, 0, st, s, s.pairs[0])
              : launch_early(embed_sort_kernel, dim3(kSortCtas), kSortThreads, smem, st, s)))
        return USAF_ECUDA;
    if (zero && !launch_early(embed_zero_kernel, dim3(cdiv(zero + 1, kZeroTile)), kZeroThreads, 0, st, (char *)a.grad, zero))
        return USAF_ECUDA;
    const uint2 *sorted = s.pairs[few ? 0 : (s.passes - 1) & 1];
    const int64_t chunks = (a.tokens + kChunk - 1) / kChunk;
    const bool vec = ((uintptr_t)a.dy | (uintptr_t)a.grad | (uintptr_t)a.ws) % 16 == 0 && (int64_t)a.H * sizeof(T) % 16 == 0;
    // Two vectors a lane halve what a row costs beside its bytes (16384 rows of 1001
    // fp32 values added to a gradient: 28 us against 37); one where that would leave an
    // SM fewer than 16 warps to have rows on their way (8192 rows of 2048 bf16: the
    // pass 123 us against 129)
    const int wide = 64 * kLaneN<T>;
    const bool two = a.H > wide / 2 && chunks * ((a.H + wide - 1) / wide) >= 148 * 16;
    auto sum = two ? (vec ? sum_launch<T, G, 2, true> : sum_launch<T, G, 2, false>)
                   : (vec ? sum_launch<T, G, 1, true> : sum_launch<T, G, 1, false>);
    if (const int rc = sum(a, sorted, chunks, part, st)) return rc;
    if (chunks > 1) {
        const dim3 jgrid(cdiv(chunks - 1, 8), cdiv(a.H, 128));
        if (!launch_early(embed_join_kernel<G>, jgrid, 256, 0, st, sorted, (uint32_t)a.tokens, (uint32_t)a.V, a.H, a.scale,
                          a.add, (G *)a.grad, (const float *)part, chunks))
            return USAF_ECUDA;
    }
    return USAF_OK;
}

template <typename T>
static int embed_fwd(const void *ids, int ids64, int64_t tokens, const void *table, int64_t V, int H, float scale,
                      void *out, int32_t *err, cudaStream_t st) {
    const int group = 32 * kLaneN<T> * kFwdSlabs;
    const unsigned grid = cdiv(tokens * ((H + group - 1) / group), 8);
    const bool vec = ((uintptr_t)table | (uintptr_t)out) % 16 == 0 && (int64_t)H * sizeof(T) % 16 == 0;
    return launch_early(vec ? embed_fwd_kernel<T, true> : embed_fwd_kernel<T, false>, dim3(grid), 256, 0, st, ids, ids64,
                        tokens, (const T *)table, V, H, scale, (T *)out, err)
               ? USAF_OK
               : USAF_ECUDA;
}

}  // namespace usaf

using namespace usaf;

// positions and rows are 32-bit in the sort; a launch has at most 2^31 - 1 CTAs
constexpr int64_t kMostTokens = (int64_t)1 << 30, kMostRows = (int64_t)1 << 30;
constexpr int32_t kMostWidth = 1 << 22;

extern "C" int usaf_embedding_fwd(const void *ids, int32_t ids_bits, int64_t tokens, const void *table, int32_t dtype,
                                  int64_t V, int32_t H, double scale, void *out, int32_t *err, void *stream) {
    USAF_REQUIRE(tokens >= 0 && V >= 0 && H >= 1 && (ids_bits == 32 || ids_bits == 64));
    if (tokens == 0) return USAF_OK;
    USAF_REQUIRE(ids && (table || V == 0) && out);
    if (H > kMostWidth || tokens > kMostTokens || tokens * ((H + 511) / 512) > ((int64_t)1 << 33)) return USAF_EUNSUPPORTED;
    cudaStream_t st = as_stream(stream);
    const int wide = ids_bits == 64;
    switch (dtype) {
        case USAF_F32: return embed_fwd<float>(ids, wide, tokens, table, V, H, (float)scale, out, err, st);
        case USAF_BF16: return embed_fwd<__nv_bfloat16>(ids, wide, tokens, table, V, H, (float)scale, out, err, st);
        case USAF_F16: return embed_fwd<__half>(ids, wide, tokens, table, V, H, (float)scale, out, err, st);
        default: return USAF_EINVAL;
    }
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
    if (tokens > kMostTokens || V > kMostRows || H > kMostWidth ||
        (tokens / kChunk + 1) * ((H + 127) / 128) > ((int64_t)1 << 33))
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
