// Attention over the 4-bit paged cache: the plainest form, a CTA for each query head and token.
//
//   s_t = scale * q . (z_t + n_t s_t),   out = sum_t softmax(s)_t (z'_t + n'_t s'_t)
//
// One pass with a running maximum and sum; a tile of 16 tokens at a time, eight threads a token for the scores, a thread per
// channel (or two) for the values.
#include "mk36_kv4.cuh"

namespace mk36 {

struct Kv4AttnParams {
    Kv4View cache;
    const void* q;
    void* out;
    long long q_row, q_token, q_head;
    int query_heads, tokens, group;
    float scale;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_attention_simple_kernel(const Kv4AttnParams p) {
    __shared__ float s_q[D], s_score[kKv4Tile];
    const int head = blockIdx.x % p.query_heads, i = blockIdx.x / p.query_heads % p.tokens, row = blockIdx.x / p.query_heads / p.tokens;
    const T* q = static_cast<const T*>(p.q) + row * p.q_row + i * p.q_token + head * p.q_head;
    for (int c = threadIdx.x; c < D; c += blockDim.x) s_q[c] = to_float<T>(q[c]);
    const int seen = kv4_length(p.cache, row) - p.tokens + i + 1;
    float top = -INFINITY, sum = 0.f, acc[2] = {0.f, 0.f};
    __syncthreads();
    for (int first = 0; first < seen; first += kKv4Tile) {
        int slot, inner;
        fdivmod(first / kKv4Tile, p.cache.tiles_per_page, slot, inner);
        long long page = p.cache.table[(long long)row * p.cache.row_pages + slot];
        const bool lost = page < 0 || page >= p.cache.pages;
        if (lost) page = 0;
        const unsigned char* tile = p.cache.pool + ((page * p.cache.kv_heads + head / p.group) * (long long)p.cache.tiles_per_page.d + inner) * p.cache.tile_bytes;
        const unsigned char* param = tile + 2 * kv4_code_bytes(D);
        const int t = threadIdx.x / 8;
        float dot = 0.f, scale, zero;
        for (int c = threadIdx.x % 8 * 8; c < D; c += 64) {
            const unsigned word = *reinterpret_cast<const unsigned*>(tile + kv4_key_word<D>(t, c));
            kv4_unpack(reinterpret_cast<const Kv4Param<T>*>(param)[t * (D / kKv4Group) + c / kKv4Group], scale, zero);
            for (int k = 0; k < 8; ++k) dot = fmaf(s_q[c + k], fmaf((float)((word >> (4 * k)) & 15u), scale, zero), dot);
        }
        for (int off = 1; off < 8; off <<= 1) dot += __shfl_xor_sync(kFullMask, dot, off);
        if (threadIdx.x % 8 == 0) s_score[t] = first + t < seen ? (lost ? __uint_as_float(0x7fc00000u) : dot * p.scale) : -INFINITY;
        __syncthreads();
        float now = top;
        for (int k = 0; k < kKv4Tile; ++k) now = fmaxf(now, s_score[k]);
        const float base = now == -INFINITY ? 0.f : now, corr = expf(top - base);
        top = now;
        sum *= corr;
        acc[0] *= corr, acc[1] *= corr;
        for (int k = 0; k < kKv4Tile && first + k < seen; ++k) {
            const float w = expf(s_score[k] - base);
            sum += w;
            for (int x = 0, c = threadIdx.x; c < D; ++x, c += 128) {
                const unsigned word = *reinterpret_cast<const unsigned*>(tile + kv4_value_word<D>(k, c & ~7));
                kv4_unpack(reinterpret_cast<const Kv4Param<T>*>(param + kv4_param_bytes(D, sizeof(T)))[k * (D / kKv4Group) + c / kKv4Group], scale, zero);
                acc[x] = fmaf(w, fmaf((float)((word >> (4 * (c & 7))) & 15u), scale, zero), acc[x]);
            }
        }
        __syncthreads();
    }
    T* out = static_cast<T*>(p.out) + (long long)blockIdx.x * D;
    for (int x = 0, c = threadIdx.x; c < D; ++x, c += 128) out[c] = from_float<T>(sum == 0.f ? 0.f : acc[x] / sum);
}

static int kv4_attention_params(const mk36_kv4_cache* c, const mk36_kv4_attention_args* a, Kv4AttnParams* p) {
    const char* what = "kv4_attention_decode";
    const int rc = kv4_view(c, what, &p->cache);
    if (rc != MK36_OK) return rc;
    if (!a) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (!a->q || !a->out) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: NULL tensor pointer", what);
    if (a->query_heads <= 0 || a->tokens <= 0) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: sizes must be positive", what);
    if (a->query_heads % c->kv_heads != 0) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: query_heads must be divisible by kv_heads", what);
    if (!(a->scale - a->scale == 0.0f)) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: scale must be finite", what);
    if ((long long)c->rows * a->tokens * a->query_heads > 0x7fffffffLL) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 query heads", what);
    const int elem = kv4_elem(c->dtype);
    if (reinterpret_cast<uintptr_t>(a->q) % elem != 0 || reinterpret_cast<uintptr_t>(a->out) % elem != 0)
        MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: q and out must be aligned to their elements", what);
    p->q = a->q;
    p->out = a->out;
    p->q_row = a->q_row, p->q_token = a->q_token, p->q_head = a->q_head;
    p->query_heads = a->query_heads;
    p->tokens = a->tokens;
    p->group = a->query_heads / c->kv_heads;
    p->scale = a->scale;
    return MK36_OK;
}

template <typename T>
static int kv4_attention_launch(const Kv4AttnParams& p, int d, cudaStream_t s) {
    const unsigned ctas = (unsigned)((long long)p.cache.rows * p.tokens * p.query_heads);
    if (d == 64) kv4_attention_simple_kernel<T, 64><<<ctas, 128, 0, s>>>(p);
    else if (d == 128) kv4_attention_simple_kernel<T, 128><<<ctas, 128, 0, s>>>(p);
    else kv4_attention_simple_kernel<T, 256><<<ctas, 128, 0, s>>>(p);
    MK36_CUDA_OK(cudaGetLastError());
    return MK36_OK;
}

}  // namespace mk36

using namespace mk36;

extern "C" size_t mk36_kv4_attention_workspace_bytes(const mk36_kv4_cache* cache, const mk36_kv4_attention_args* args) {
    Kv4AttnParams p{};
    return kv4_attention_params(cache, args, &p) == MK36_OK ? 16 : 0;
}

extern "C" int mk36_kv4_attention_decode(const mk36_kv4_cache* cache, const mk36_kv4_attention_args* args, void* workspace,
                                         size_t workspace_bytes, void* stream) {
    Kv4AttnParams p{};
    const int rc = kv4_attention_params(cache, args, &p);
    if (rc != MK36_OK) return rc;
    if (!workspace || workspace_bytes < mk36_kv4_attention_workspace_bytes(cache, args))
        MK36_FAIL(MK36_ERR_WORKSPACE, "kv4_attention_decode: workspace of %zu bytes is too small", workspace_bytes);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (cache->dtype) {
        case MK36_BF16: return kv4_attention_launch<__nv_bfloat16>(p, cache->head_dim, s);
        case MK36_F16: return kv4_attention_launch<__half>(p, cache->head_dim, s);
        default: return kv4_attention_launch<float>(p, cache->head_dim, s);
    }
}
