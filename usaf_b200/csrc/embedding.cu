// Embedding lookup y[t] = scale W[id_t] and the gradient of the table,
// dW[v] = scale * (sum of dy[t] over the tokens t with id_t = v, ascending t).
#include "common.cuh"

namespace usaf {

__device__ __forceinline__ int64_t token_id(const void *ids, int ids64, int64_t t) {
    return ids64 ? static_cast<const int64_t *>(ids)[t] : (int64_t) static_cast<const int32_t *>(ids)[t];
}

// one warp per token; a token outside the table reads as zeros and sets the error word
template <typename T>
__global__ void __launch_bounds__(256)
embed_fwd_kernel(const void *__restrict__ ids, int ids64, int64_t tokens, const T *__restrict__ table, int64_t V,
                 int H, float scale, T *__restrict__ out, int32_t *__restrict__ err) {
    const int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (t >= tokens) return;
    const int64_t id = token_id(ids, ids64, t);
    const bool ok = id >= 0 && id < V;
    if (!ok && lane == 0 && err) atomicOr(err, USAF_ERR_BAD_INDEX);
    for (int c = lane; c < H; c += 32) out[t * H + c] = from_f<T>(ok ? to_f(table[id * H + c]) * scale : 0.0f);
}

// one warp per token: the first token of an id sums the rows of all its tokens
template <typename T, typename G>
__global__ void __launch_bounds__(256)
embed_bwd_kernel(const T *__restrict__ dy, const void *__restrict__ ids, int ids64, int64_t tokens, int64_t V, int H,
                 float scale, int64_t pad, int add, G *__restrict__ grad, int32_t *__restrict__ err) {
    const int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (t >= tokens) return;
    const int64_t id = token_id(ids, ids64, t);
    if (id < 0 || id >= V) {
        if (lane == 0 && err) atomicOr(err, USAF_ERR_BAD_INDEX);
        return;
    }
    if (id == pad) return;
    for (int64_t j = 0; j < t; j += 32) {
        const bool same = j + lane < t && token_id(ids, ids64, j + lane) == id;
        if (__any_sync(0xffffffffu, same)) return;
    }
    for (int c0 = 0; c0 < H; c0 += 256) {
        float acc[8] = {};
        for (int64_t j = t; j < tokens; j += 32) {
            const bool same = j + lane < tokens && token_id(ids, ids64, j + lane) == id;
            for (uint32_t m = __ballot_sync(0xffffffffu, same); m; m &= m - 1) {
                const int64_t row = j + __ffs(m) - 1;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int c = c0 + lane + 32 * k;
                    if (c < H) acc[k] += to_f(dy[row * H + c]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int c = c0 + lane + 32 * k;
            if (c < H) {
                G *p = grad + id * H + c;
                *p = from_f<G>(add ? fmaf(acc[k], scale, to_f(*p)) : acc[k] * scale);
            }
        }
    }
}

struct EmbedBwd {
    const void *dy, *ids; int ids64;
    int64_t tokens, V; int H; float scale; int64_t pad; int add;
    void *grad, *ws; int32_t *err;
};

template <typename T, typename G> static int embed_bwd(const EmbedBwd &a, cudaStream_t st) {
    if (!a.add && cudaMemsetAsync(a.grad, 0, (size_t)a.V * a.H * sizeof(G), st) != cudaSuccess) return USAF_ECUDA;
    if (a.tokens) {
        embed_bwd_kernel<T, G><<<cdiv(a.tokens * 32, 256), 256, 0, st>>>((const T *)a.dy, a.ids, a.ids64, a.tokens, a.V,
                                                                        a.H, a.scale, a.pad, a.add, (G *)a.grad, a.err);
        USAF_CHECK_LAUNCH();
    }
    return USAF_OK;
}

}  // namespace usaf

using namespace usaf;

extern "C" int usaf_embedding_fwd(const void *ids, int32_t ids_bits, int64_t tokens, const void *table, int32_t dtype,
                                  int64_t V, int32_t H, double scale, void *out, int32_t *err, void *stream) {
    USAF_REQUIRE(tokens >= 0 && V >= 0 && H >= 1 && (ids_bits == 32 || ids_bits == 64));
    if (tokens == 0) return USAF_OK;
    USAF_REQUIRE(ids && (table || V == 0) && out);
    cudaStream_t st = as_stream(stream);
    const unsigned grid = cdiv(tokens * 32, 256);
    const int wide = ids_bits == 64;
    switch (dtype) {
        case USAF_F32: embed_fwd_kernel<float><<<grid, 256, 0, st>>>(ids, wide, tokens, (const float *)table, V, H, (float)scale, (float *)out, err); break;
        case USAF_BF16: embed_fwd_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(ids, wide, tokens, (const __nv_bfloat16 *)table, V, H, (float)scale, (__nv_bfloat16 *)out, err); break;
        case USAF_F16: embed_fwd_kernel<__half><<<grid, 256, 0, st>>>(ids, wide, tokens, (const __half *)table, V, H, (float)scale, (__half *)out, err); break;
        default: return USAF_EINVAL;
    }
    USAF_CHECK_LAUNCH();
    return USAF_OK;
}

extern "C" int64_t usaf_embedding_workspace_bytes(int64_t tokens, int64_t V, int32_t H) {
    if (tokens < 0 || V < 0 || H < 1) return -1;
    return 0;
}

extern "C" int usaf_embedding_bwd(const void *dy, const void *ids, int32_t ids_bits, int64_t tokens, int32_t dtype,
                                  int64_t V, int32_t H, double scale, int64_t padding_idx, int32_t accumulate,
                                  void *grad, int32_t grad_dtype, void *ws, int32_t *err, void *stream) {
    USAF_REQUIRE(tokens >= 0 && V >= 0 && H >= 1 && (ids_bits == 32 || ids_bits == 64));
    USAF_REQUIRE((grad || V == 0) && (tokens == 0 || (dy && ids)));
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
