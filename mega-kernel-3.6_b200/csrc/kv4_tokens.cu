// Appending tokens to the 4-bit paged cache (quantisation) and reading them back.
//
// A group of 64 channels of one token and head becomes a scale s = (max - min) / 15 and a zero point z = min, both in the
// activations' type, and codes n = round((x - z) / s); the cache then stands for z + n s.  Both directions move each byte
// once and are bound by memory: a thread has eight consecutive channels (16 bytes of a 2-byte type on one side, one 32-bit
// word of codes on the other), eight threads a group, whose minimum and maximum take three shuffles.
//
// Codes and scales follow from exact arithmetic.  In fp32 that needs a second look only where the quotient lies next to a
// border between two codes (or the scale next to one between two values of its type); there the thread does it again in fp64.
#include <type_traits>

#include "mk36_kv4.cuh"

namespace mk36 {

struct Kv4TokenParams {
    Kv4View cache;
    unsigned char* k;  // append reads k and v, read writes them
    unsigned char* v;
    const int* cu;      // null: `tokens` of every row
    long long tokens, total;
    long long k_row, k_token, k_head, v_row, v_token, v_head;  // elements
    int wide;  // 1: every eight channels lie on a 16-byte boundary
    FastDiv per_row;
};

// Row and position of token i; false where it belongs to no row.
__device__ __forceinline__ bool kv4_place(const Kv4TokenParams& p, long long i, int& row, int& local, int& position) {
    int n;
    if (!p.cu) {
        fdivmod((int)i, p.per_row, row, local);
        n = (int)p.tokens;
    } else {
        int lo = 0, hi = p.cache.rows;  // the last row that starts at or before i
        if (i < p.cu[0] || i >= p.cu[hi]) return false;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.cu[mid] <= i) lo = mid;
            else hi = mid;
        }
        row = lo;
        local = (int)i - p.cu[lo];
        n = p.cu[lo + 1] - p.cu[lo];
        if (local >= n) return false;
    }
    position = kv4_length(p.cache, row) - n + local;
    return true;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool wide, float (&f)[8]) {
    if (wide) {
        unpack8(load_chunk8<T>(p), f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_float<T>(p[i]);
    }
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, bool wide, const float (&f)[8]) {
    if (wide) {
        uint4 r;
        unsigned* w = &r.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned*>(&h);
        }
        *reinterpret_cast<uint4*>(p) = r;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(f[i]);
    }
}
__device__ __forceinline__ void store8(__half* p, bool wide, const float (&f)[8]) {
    if (wide) {
        uint4 r;
        unsigned* w = &r.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned*>(&h);
        }
        *reinterpret_cast<uint4*>(p) = r;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __float2half_rn(f[i]);
    }
}
__device__ __forceinline__ void store8(float* p, bool wide, const float (&f)[8]) {
    if (wide) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = f[i];
    }
}

// (high - low) / 15 rounded once to T, in fp64 throughout: the difference of two values of T is exact there or off by a part in
// 2^53, far from where it could change the rounding to 24 bits or fewer.
__device__ __forceinline__ float scale_exact(float low, float high, const __nv_bfloat16*) {
    return __bfloat162float(__double2bfloat16(((double)high - (double)low) / 15.0));
}
__device__ __forceinline__ float scale_exact(float low, float high, const __half*) {
    return __half2float(__double2half(((double)high - (double)low) / 15.0));
}
__device__ __forceinline__ float scale_exact(float low, float high, const float*) {
    return (float)(((double)high - (double)low) / 15.0);
}

// The same by way of fp32 where that cannot differ: the fp32 quotient is within 4 steps of the exact one, so both round alike unless
// they lie around the middle between two neighbours of T.
__device__ __forceinline__ float scale_of(float low, float high, const __nv_bfloat16* t) {
    const float q = (high - low) * (1.0f / 15.0f);
    const unsigned rest = __float_as_uint(q) & 0xffffu;
    if (!(q >= 1e-30f) || q > 1e37f || rest - 0x7ff8u <= 0x10u) return scale_exact(low, high, t);
    return __bfloat162float(__float2bfloat16_rn(q));
}
__device__ __forceinline__ float scale_of(float low, float high, const __half* t) {
    const float q = (high - low) * (1.0f / 15.0f);
    const unsigned rest = __float_as_uint(q) & 0x1fffu;
    if (!(q >= 6.2e-5f) || rest - 0xff8u <= 0x10u) return scale_exact(low, high, t);  // below: f16 subnormals, fewer bits
    return __half2float(__float2half_rn(q));
}
__device__ __forceinline__ float scale_of(float low, float high, const float* t) { return scale_exact(low, high, t); }

__device__ __noinline__ unsigned code_exact(float x, float zero, float scale) {
    const double n = rint(((double)x - (double)zero) / (double)scale);
    return n > 0.0 ? (n < 15.0 ? (unsigned)n : 15u) : 0u;
}

// y = (x - zero) * (1 / scale) in fp32 is off by less than 2e-5 for codes up to 16: the difference and the product are off by
// 2^-24 each, the reciprocal by 2^-23.
__device__ __forceinline__ unsigned code_of(float x, float zero, float scale, float inv) {
    const float y = (x - zero) * inv;
    const float n = rintf(y);
    if (!(fabsf(y - n) < 0.4999f)) return code_exact(x, zero, scale);
    return n > 0.0f ? (n < 15.0f ? (unsigned)n : 15u) : 0u;
}

template <typename T>
__device__ __forceinline__ void write_param(unsigned char* p, float scale, float zero, bool fine) {
    if (sizeof(T) == 4) {
        *reinterpret_cast<float2*>(p) = make_float2(scale, zero);
    } else {
        constexpr unsigned kNan = std::is_same<T, __half>::value ? 0x7e007e00u : 0x7fc07fc0u;
        T two[2] = {from_float<T>(scale), from_float<T>(zero)};
        *reinterpret_cast<unsigned*>(p) = fine ? *reinterpret_cast<const unsigned*>(two) : kNan;
    }
}

// One of 2 * kv_heads * D / 8 pieces of a token: keys of all heads, then values.
template <typename T, int D>
struct Kv4Piece {
    const T* dense;             // its channels in k or v
    unsigned char *word, *param;  // its codes and its group's parameters in the cache
    bool placed, in_pool;
};

template <typename T, int D>
__device__ __forceinline__ bool kv4_piece(const Kv4TokenParams& p, long long unit, int pieces, Kv4Piece<T, D>& out) {
    const long long i = unit / pieces;
    int piece = (int)(unit - i * pieces);
    int row, local, position;
    if (i >= p.total || !kv4_place(p, i, row, local, position)) return false;
    const bool is_k = piece < pieces / 2;
    if (!is_k) piece -= pieces / 2;
    const int head = piece / (D / 8), c = piece % (D / 8) * 8;
    const long long at = is_k ? (p.cu ? i * p.k_token : row * p.k_row + local * p.k_token) + head * p.k_head
                              : (p.cu ? i * p.v_token : row * p.v_row + local * p.v_token) + head * p.v_head;
    out.dense = reinterpret_cast<const T*>(is_k ? p.k : p.v) + at + c;
    out.placed = position >= 0;
    out.in_pool = false;
    out.word = out.param = nullptr;
    if (out.placed) {
        int slot, inner;
        fdivmod(position / kKv4Tile, p.cache.tiles_per_page, slot, inner);
        const long long page = p.cache.table[(long long)row * p.cache.row_pages + slot];
        if (page >= 0 && page < p.cache.pages) {
            out.in_pool = true;
            unsigned char* tile = p.cache.pool + ((page * p.cache.kv_heads + head) * (long long)p.cache.tiles_per_page.d + inner) * p.cache.tile_bytes;
            const int t = position % kKv4Tile;
            out.word = tile + (is_k ? kv4_key_word<D>(t, c) : kv4_value_word<D>(t, c));
            out.param = tile + 2 * kv4_code_bytes(D) + (is_k ? 0 : kv4_param_bytes(D, sizeof(T))) + (t * (D / kKv4Group) + c / kKv4Group) * 2 * sizeof(T);
        }
    }
    return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4TokenParams p) {
    const int pieces = 2 * p.cache.kv_heads * (D / 8);
    const long long unit = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    Kv4Piece<T, D> piece;
    // the eight threads of a group take the same way; the warp stays together for the shuffles
    const bool go = kv4_piece<T, D>(p, unit, pieces, piece) && piece.in_pool;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (go) load8<T>(piece.dense, p.wide != 0, f);
    float low = f[0], high = f[0], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        low = fminf(low, f[i]);
        high = fmaxf(high, f[i]);
        sum += f[i] * 0.0f;  // NaN as soon as one is an infinity or a NaN
    }
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
        low = fminf(low, __shfl_xor_sync(kFullMask, low, off));
        high = fmaxf(high, __shfl_xor_sync(kFullMask, high, off));
        sum += __shfl_xor_sync(kFullMask, sum, off);
    }
    if (!go) return;
    const bool fine = sum == 0.0f;
    const float nan = __uint_as_float(0x7fc00000u);
    const float zero = fine ? low + 0.0f : nan;  // -0 becomes 0
    const float scale = fine ? scale_of(low, high, static_cast<const T*>(nullptr)) : nan;
    unsigned word = 0;
    if (fine && scale > 0.0f) {
        // a scale whose reciprocal fp32 does not hold well makes every quotient an infinity or NaN here, or is far from 1e-30
        const float inv = scale >= 1e-30f ? 1.0f / scale : nan;
#pragma unroll
        for (int i = 0; i < 8; ++i) word |= code_of(f[i], zero, scale, inv) << (4 * i);
    }
    *reinterpret_cast<unsigned*>(piece.word) = word;
    if (threadIdx.x % 8 == 0) write_param<T>(piece.param, scale, zero, fine);
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4TokenParams p) {
    const int pieces = 2 * p.cache.kv_heads * (D / 8);
    const long long unit = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    Kv4Piece<T, D> piece;
    if (!kv4_piece<T, D>(p, unit, pieces, piece)) return;
    float f[8];
    if (piece.in_pool) {
        const unsigned word = *reinterpret_cast<const unsigned*>(piece.word);
        float scale, zero;
        kv4_unpack(*reinterpret_cast<const Kv4Param<T>*>(piece.param), scale, zero);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = fmaf((float)((word >> (4 * i)) & 15u), scale, zero);
    } else {
        const float fill = piece.placed ? __uint_as_float(0x7fc00000u) : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = fill;
    }
    store8(const_cast<T*>(piece.dense), p.wide != 0, f);
}

int kv4_view(const mk36_kv4_cache* c, const char* what, Kv4View* v) {
    if (!c) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: cache is NULL", what);
    if (!c->pool || !c->page_table || !c->lengths) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: NULL tensor pointer", what);
    if (c->dtype != MK36_BF16 && c->dtype != MK36_F16 && c->dtype != MK36_F32) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: unsupported dtype %d", what, c->dtype);
    if (c->pages <= 0 || c->kv_heads <= 0 || c->rows <= 0 || c->row_pages <= 0 || c->page_size <= 0)
        MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: sizes must be positive", what);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256", what);
    if (c->page_size % kKv4Tile != 0) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: page_size must be a multiple of %d", what, kKv4Tile);
    if (c->pages > 0x7fffffffLL) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 pages", what);
    const long long capacity = (long long)c->row_pages * c->page_size;
    if (capacity > 0x7fffff00LL) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: more than 2^31 - 256 tokens in a row", what);
    if (reinterpret_cast<uintptr_t>(c->pool) % 16 != 0) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: the pool must be 16-byte aligned", what);
    v->pool = static_cast<unsigned char*>(c->pool);
    v->table = c->page_table;
    v->lengths = c->lengths;
    v->pages = c->pages;
    v->kv_heads = c->kv_heads;
    v->rows = c->rows;
    v->row_pages = c->row_pages;
    v->capacity = (int)capacity;
    v->tiles_per_page = make_fastdiv((unsigned)(c->page_size / kKv4Tile));
    v->tile_bytes = (unsigned)kv4_tile_bytes(c->head_dim, kv4_elem(c->dtype));
    return MK36_OK;
}

template <typename T, int D>
static int kv4_tokens_launch(const Kv4TokenParams& p, bool append, cudaStream_t s, const char* what) {
    const long long threads = p.total * (2ll * p.cache.kv_heads * (D / 8));
    const long long ctas = (threads + 255) / 256;
    if (ctas > 0x7fffffffLL) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: too many tokens for one call", what);
    if (append) kv4_append_kernel<T, D><<<(unsigned)ctas, 256, 0, s>>>(p);
    else kv4_read_kernel<T, D><<<(unsigned)ctas, 256, 0, s>>>(p);
    MK36_CUDA_OK(cudaGetLastError());
    return MK36_OK;
}

template <typename T>
static int kv4_tokens_head_dim(const Kv4TokenParams& p, int d, bool append, cudaStream_t s, const char* what) {
    if (d == 64) return kv4_tokens_launch<T, 64>(p, append, s, what);
    if (d == 128) return kv4_tokens_launch<T, 128>(p, append, s, what);
    return kv4_tokens_launch<T, 256>(p, append, s, what);
}

static int kv4_tokens(const mk36_kv4_cache* c, const mk36_kv4_tokens* t, bool append, void* stream, const char* what) {
    Kv4TokenParams p{};
    const int rc = kv4_view(c, what, &p.cache);
    if (rc != MK36_OK) return rc;
    if (!t) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: tokens is NULL", what);
    if (t->tokens < 0) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: tokens must not be negative", what);
    if (t->tokens == 0) return MK36_OK;
    if (!t->k || !t->v) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: NULL tensor pointer", what);
    p.total = t->cu_tokens ? t->tokens : t->tokens * c->rows;
    if (t->tokens > 0x7fffffffLL || p.total > 0x7fffffffLL) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: too many tokens for one call", what);
    p.k = static_cast<unsigned char*>(t->k);
    p.v = static_cast<unsigned char*>(t->v);
    p.cu = t->cu_tokens;
    p.tokens = t->tokens;
    p.k_row = t->k_row, p.k_token = t->k_token, p.k_head = t->k_head;
    p.v_row = t->v_row, p.v_token = t->v_token, p.v_head = t->v_head;
    const int elem = kv4_elem(c->dtype);
    if (reinterpret_cast<uintptr_t>(t->k) % elem != 0 || reinterpret_cast<uintptr_t>(t->v) % elem != 0)
        MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: k and v must be aligned to their elements", what);
    const long long strides = (t->cu_tokens ? 0 : t->k_row | t->v_row) | t->k_token | t->k_head | t->v_token | t->v_head;
    p.wide = (reinterpret_cast<uintptr_t>(t->k) | reinterpret_cast<uintptr_t>(t->v) | (uintptr_t)(strides * elem)) % 16 == 0;
    p.per_row = make_fastdiv((unsigned)t->tokens);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (c->dtype) {
        case MK36_BF16: return kv4_tokens_head_dim<__nv_bfloat16>(p, c->head_dim, append, s, what);
        case MK36_F16: return kv4_tokens_head_dim<__half>(p, c->head_dim, append, s, what);
        default: return kv4_tokens_head_dim<float>(p, c->head_dim, append, s, what);
    }
}

}  // namespace mk36

using namespace mk36;

extern "C" int mk36_kv4_append(const mk36_kv4_cache* cache, const mk36_kv4_tokens* tokens, void* stream) {
    return kv4_tokens(cache, tokens, true, stream, "kv4_append");
}

extern "C" int mk36_kv4_read(const mk36_kv4_cache* cache, const mk36_kv4_tokens* tokens, void* stream) {
    return kv4_tokens(cache, tokens, false, stream, "kv4_read");
}
