// Appending tokens to the 4-bit paged cache (quantisation) and reading them back.
//
// A group of 64 channels of one token and head becomes a scale s = (max - min) / 15 and a zero point z = min, both in the
// activations' type, and codes n = round((x - z) / s); the cache then stands for z + n s.  Both directions move each byte once.  An
// append has 16 channels for a thread (32 bytes of a 2-byte type on one side, two 32-bit words of codes on the other), four threads a
// group, whose minimum and maximum travel as one pair through two shuffles; a read has eight.
//
// Codes and scales follow from exact arithmetic (fp32: from 64 bits), whatever the order of operations in fp32 would give: see codes_of and
// scale_of.
//
// What bounds them: reading back, memory and instructions alike (32768 tokens of 2 heads of 256 in bf16: 86 MB in 16.3 us, 5.3 TB/s; in fp32
// 155 MB in 36 us, 4.3 TB/s); appending, instructions (28.7 us, 3.0 TB/s; 26.2 us in f16, where fewer values lie half way between codes; fp32 41.9
// us, 3.7 TB/s).
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
    int cta_tokens;
    int clear;  // read: zeros behind the last row's tokens
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

// Eight channels as they lie in memory.
template <typename T>
__device__ __forceinline__ Chunk8<T> load8(const T* p, bool wide) {
    if (wide) return load_chunk8<T>(p);
    Chunk8<T> c;
    T* x = reinterpret_cast<T*>(&c);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
    return c;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool wide, const Chunk8<T>& c) {
    if (wide) {
        *reinterpret_cast<Chunk8<T>*>(p) = c;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = reinterpret_cast<const T*>(&c)[i];
    }
}

// zero + code * scale, rounded once.  In two-byte types two at a time: 0x..0n or'ed to a power of two is that plus n, and a fused
// product and sum of the types' own rounds once.
template <typename T2>
__device__ __forceinline__ void dequantise_pairs(unsigned word, unsigned param, unsigned power, uint4& out) {
    const unsigned scale = __byte_perm(param, param, 0x1010), zero = __byte_perm(param, param, 0x3232);
    unsigned n[4];  // codes i and i + 4
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned x = (word >> (4 * i) & 0x000f000fu) | power;
        const T2 v = __hfma2(__hsub2(*reinterpret_cast<const T2*>(&x), *reinterpret_cast<const T2*>(&power)), *reinterpret_cast<const T2*>(&scale),
                             *reinterpret_cast<const T2*>(&zero));
        n[i] = *reinterpret_cast<const unsigned*>(&v);
    }
    out = make_uint4(__byte_perm(n[0], n[1], 0x5410), __byte_perm(n[2], n[3], 0x5410), __byte_perm(n[0], n[1], 0x7632), __byte_perm(n[2], n[3], 0x7632));
}
__device__ __forceinline__ void dequantise(unsigned word, const Kv4Param<__nv_bfloat16>& p, Chunk8<__nv_bfloat16>& out) {
    dequantise_pairs<__nv_bfloat162>(word, p.raw, 0x43004300u, out.raw);  // 128
}
__device__ __forceinline__ void dequantise(unsigned word, const Kv4Param<__half>& p, Chunk8<__half>& out) {
    dequantise_pairs<__half2>(word, p.raw, 0x64006400u, out.raw);  // 1024
}
__device__ __forceinline__ void dequantise(unsigned word, const Kv4Param<float>& p, Chunk8<float>& out) {
    float* f = reinterpret_cast<float*>(&out);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = fmaf((float)(word >> (4 * i) & 15u), p.scale, p.zero);
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

// Values in registers: an array passed by its address would be stored to memory by every thread, called or not.
__device__ __noinline__ unsigned four_exact(float4 x, float zero, float scale) {
    return code_exact(x.x, zero, scale) | code_exact(x.y, zero, scale) << 4 | code_exact(x.z, zero, scale) << 8 | code_exact(x.w, zero, scale) << 12;
}
__device__ __forceinline__ unsigned codes_exact(const float (&x)[8], float zero, float scale) {
    return four_exact(make_float4(x[0], x[1], x[2], x[3]), zero, scale) | four_exact(make_float4(x[4], x[5], x[6], x[7]), zero, scale) << 16;
}

constexpr float kRoundUp = 12582912.0f;  // 1.5 * 2^23: added, it rounds to a whole number, halves to even, and leaves that in the low bits

// Whole numbers below 16, as floats, to a word of eight half bytes: sums of four are exact.
__device__ __forceinline__ unsigned pack_codes(const float (&n)[8]) {
    const float low = fmaf(n[3], 4096.0f, fmaf(n[2], 256.0f, fmaf(n[1], 16.0f, n[0]))), high = fmaf(n[7], 4096.0f, fmaf(n[6], 256.0f, fmaf(n[5], 16.0f, n[4])));
    return __byte_perm(__float_as_uint(low + kRoundUp), __float_as_uint(high + kRoundUp), 0x5410);
}

// Codes of two-byte values.  n = the whole number nearest to (x - zero) / scale by way of an approximate reciprocal is right, or next to
// it where the quotient lies at a border: what is left, r = (x - zero) - n scale, says so, because it is exact.  (n scale has 15
// bits at most; x - zero has 24 and is off by e at most half its last place; half the scale is a multiple of that place.)
// Values half way between two codes are common, one in some hundred of bf16: about every second warp has one.
template <typename T>
__device__ __forceinline__ unsigned codes_of(const float (&x)[8], float zero, float scale, float inv, const T*) {
    const float half = 0.5f * scale;
    const f32x2 zeros = pair_of(-zero, -zero), scales = pair_of(-scale, -scale), invs = pair_of(inv, inv), up = pair_of(kRoundUp, kRoundUp),
                down = pair_of(-kRoundUp, -kRoundUp);
    float n[8], r[8];
    f32x2 m[4];  // n of i and i + 4
    bool border = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2 d = add_pair(pair_of(x[i], x[i + 4]), zeros);
        m[i] = add_pair(fma_pair(d, invs, up), down);
        const f32x2 rest = fma_pair(m[i], scales, d);
        r[i] = first_of(rest), r[i + 4] = second_of(rest);
        border |= fabsf(r[i]) >= half;
        border |= fabsf(r[i + 4]) >= half;
    }
    if (border) {
#pragma unroll
        for (int i = 0; i < 4; ++i) n[i] = first_of(m[i]), n[i + 4] = second_of(m[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (fabsf(r[i]) >= half) {
                const float d = x[i] - zero, part = x[i] - d, e = (part - zero) + (x[i] - (d + part));  // what the difference lost
                const float way = copysignf(1.0f, r[i]), over = fmaf(way, e, fabsf(r[i]) - half);       // its sign is exact
                const bool odd = __float_as_uint(n[i] + kRoundUp) & 1u;
                if (over > 0.0f || (over == 0.0f && odd)) n[i] += way;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = pair_of(n[i], n[i + 4]);
    }
    // the word's two halves at once: sums of four whole numbers below 16 are exact
    const f32x2 word = add_pair(fma_pair(m[3], pair_of(4096.0f, 4096.0f), fma_pair(m[2], pair_of(256.0f, 256.0f), fma_pair(m[1], pair_of(16.0f, 16.0f), m[0]))), up);
    return __byte_perm(__float_as_uint(first_of(word)), __float_as_uint(second_of(word)), 0x5410);
}

// Codes of fp32 values: neither the difference nor the product is exact, so near a border fp64 decides.  The quotient is off by less than
// 2e-5: difference, product and reciprocal by 2^-23 or less each.
__device__ __forceinline__ unsigned codes_of(const float (&x)[8], float zero, float scale, float inv, const float*) {
    float n[8], furthest = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = (x[i] - zero) * inv;
        n[i] = (y + kRoundUp) - kRoundUp;
        furthest = fmaxf(furthest, fabsf(y - n[i]));
    }
    return furthest < 0.4999f ? pack_codes(n) : codes_exact(x, zero, scale);
}

// Codes of a group's part, two words of eight: what both kinds share.
template <typename T>
__device__ __forceinline__ uint2 two_words(const float (&x)[16], float zero, float high, float scale) {
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
    if (sizeof(T) == 4) inv = 1.0f / scale;
    const float(&first)[8] = *reinterpret_cast<const float(*)[8]>(&x[0]);
    const float(&second)[8] = *reinterpret_cast<const float(*)[8]>(&x[8]);
    if (!(scale > 0.0f)) return make_uint2(0u, 0u);
    // scales of a few units of the smallest number, whose quotients may be far beyond 15, and what the reciprocal does not hold
    if (!(scale >= 1e-30f && (high - zero) * inv <= 15.4f)) return make_uint2(codes_exact(first, zero, scale), codes_exact(second, zero, scale));
    return make_uint2(codes_of(first, zero, scale, inv, static_cast<const T*>(nullptr)), codes_of(second, zero, scale, inv, static_cast<const T*>(nullptr)));
}

// Least and greatest of the 64 values of four lanes, 16 of each; NaN if one is a NaN.
__device__ __forceinline__ void least_greatest(const float (&f)[16], const Chunk8<float> (&)[2], float& low, float& high) {
    low = high = f[0];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        low = fminf(low, f[i]);
        high = fmaxf(high, f[i]);
        sum = fmaf(f[i], 0.0f, sum);  // NaN as soon as one is an infinity or a NaN
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
        low = fminf(low, __shfl_xor_sync(kFullMask, low, off));
        high = fmaxf(high, __shfl_xor_sync(kFullMask, high, off));
        sum += __shfl_xor_sync(kFullMask, sum, off);
    }
    low += sum;
    high += sum;
}
template <typename T2, typename T>
__device__ __forceinline__ void least_greatest_pairs(const Chunk8<T> (&c)[2], float& low, float& high) {
    const T2 *x = reinterpret_cast<const T2*>(&c[0]), *y = reinterpret_cast<const T2*>(&c[1]);
    T2 a = __hmin2_nan(__hmin2_nan(__hmin2_nan(x[0], x[1]), __hmin2_nan(x[2], x[3])), __hmin2_nan(__hmin2_nan(y[0], y[1]), __hmin2_nan(y[2], y[3])));
    const T2 b = __hmax2_nan(__hmax2_nan(__hmax2_nan(x[0], x[1]), __hmax2_nan(x[2], x[3])), __hmax2_nan(__hmax2_nan(y[0], y[1]), __hmax2_nan(y[2], y[3])));
    // the least and the greatest, less its sign, travel as one pair
    a.x = __hmin_nan(a.x, a.y);
    a.y = __hneg(__hmax_nan(b.x, b.y));
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) a = __hmin2_nan(a, __shfl_xor_sync(kFullMask, a, off));
    low = to_float<T>(a.x);
    high = -to_float<T>(a.y);
}
__device__ __forceinline__ void least_greatest(const float (&)[16], const Chunk8<__nv_bfloat16> (&c)[2], float& low, float& high) {
    least_greatest_pairs<__nv_bfloat162>(c, low, high);
}
__device__ __forceinline__ void least_greatest(const float (&)[16], const Chunk8<__half> (&c)[2], float& low, float& high) {
    least_greatest_pairs<__half2>(c, low, high);
}

template <typename T>
__device__ __forceinline__ void write_param(unsigned char* p, float scale, float zero, bool fine) {
    if (sizeof(T) == 4) {
        const float nan = __uint_as_float(0x7fc00000u);
        *reinterpret_cast<float2*>(p) = fine ? make_float2(scale, zero) : make_float2(nan, nan);
    } else {
        constexpr unsigned kNan = std::is_same<T, __half>::value ? 0x7e007e00u : 0x7fc07fc0u;
        T two[2] = {from_float<T>(scale), from_float<T>(zero)};
        *reinterpret_cast<unsigned*>(p) = fine ? *reinterpret_cast<const unsigned*>(two) : kNan;
    }
}

// A token has pieces of 8 channels (read) or 16 (append): keys of all heads, then values.  A CTA takes p.cta_tokens consecutive tokens
// and 32 of the pieces: a lane keeps its piece, a warp takes every fourth token.  Where a token's codes go is looked up once, by one
// thread.
constexpr int kTokThreads = 128, kTokWarps = kTokThreads / 32, kMaxCtaTokens = 32, kBatch = 2;  // kBatch: loads of a lane of the read that are on their way together

struct Kv4Where {
    long long dense[2];      // elements from the start of k and of v
    unsigned char* word[2];  // the token's place in the tile of head 0, of key codes and of value codes; null: nowhere
    unsigned char* param;
    int t;                   // token of the tile; -1: before the row's start, 16: behind the last row
};

template <typename T, int D>
__device__ __forceinline__ void kv4_find(const Kv4TokenParams& p, long long i, Kv4Where& w) {
    int row, local, position;
    w.word[0] = w.word[1] = w.param = nullptr;
    w.dense[0] = i * p.k_token, w.dense[1] = i * p.v_token;
    w.t = kKv4Tile;
    if (i >= p.total) return;
    if (!kv4_place(p, i, row, local, position)) {
        if (p.clear) w.t = -1;
        return;
    }
    if (!p.cu) w.dense[0] = row * p.k_row + local * p.k_token, w.dense[1] = row * p.v_row + local * p.v_token;
    w.t = position < 0 ? -1 : position % kKv4Tile;
    if (position < 0) return;
    int slot, inner;
    fdivmod(position / kKv4Tile, p.cache.tiles_per_page, slot, inner);
    const long long page = p.cache.table[(long long)row * p.cache.row_pages + slot];
    if (page < 0 || page >= p.cache.pages) return;
    unsigned char* tile = p.cache.pool + (page * p.cache.kv_heads * p.cache.tiles_per_page.d + inner) * (long long)p.cache.tile_bytes;
    w.word[0] = tile + kv4_key_word<D>(w.t, 0);
    w.word[1] = tile + kv4_value_word<D>(w.t, 0);
    w.param = tile + 2 * kv4_code_bytes(D) + w.t * (D / kKv4Group * 2 * (int)sizeof(T));
}

// A lane's piece: what of its places does not depend on the token.
template <typename T, int D, int kChannels>
struct Kv4Piece {
    bool there;
    int of;  // 0 keys, 1 values
    T* dense;
    long long word, param;
    const Kv4Where* where;

    __device__ __forceinline__ Kv4Piece(const Kv4TokenParams& p, const Kv4Where* w) {
        int piece = blockIdx.y * 32 + (threadIdx.x & 31);
        const int half = p.cache.kv_heads * (D / kChannels);
        there = piece < 2 * half;
        of = piece < half ? 0 : 1;
        piece -= of * half;
        const int head = piece / (D / kChannels), c = piece % (D / kChannels) * kChannels;
        const long long tile = (long long)head * p.cache.tiles_per_page.d * p.cache.tile_bytes;
        dense = reinterpret_cast<T*>(of ? p.v : p.k) + head * (of ? p.v_head : p.k_head) + c;
        word = tile + (of ? kv4_value_word<D>(0, c) - kv4_value_word<D>(0, 0) : kv4_key_word<D>(0, c));
        param = tile + of * kv4_param_bytes(D, sizeof(T)) + c / kKv4Group * 2 * (int)sizeof(T);
        where = w;
    }
    __device__ __forceinline__ T* dense_at(int token) const { return dense + where[token].dense[of]; }
    __device__ __forceinline__ unsigned* word_at(int token) const { return reinterpret_cast<unsigned*>(where[token].word[of] + word); }
    __device__ __forceinline__ unsigned char* param_at(int token) const { return where[token].param + param; }
};

// A warp requests its next token before it works on this one; 64 registers (two-byte types), eight CTAs an SM (32768 tokens: 28.7 us; two tokens requested and
// then worked on, 29.6, and 31.4 with one fp32 operation an instruction).
template <typename T, int D>
__global__ void __launch_bounds__(kTokThreads, sizeof(T) == 4 ? 6 : 8) kv4_append_kernel(const __grid_constant__ Kv4TokenParams p) {
    __shared__ Kv4Where s_where[kMaxCtaTokens];
    if ((int)threadIdx.x < p.cta_tokens) kv4_find<T, D>(p, (long long)blockIdx.x * p.cta_tokens + threadIdx.x, s_where[threadIdx.x]);
    const Kv4Piece<T, D, 16> piece(p, s_where);  // four lanes have a group
    __syncthreads();
    Chunk8<T> next[2];
    auto request = [&](int token) {
        zero_chunk8<T>(next[0]);
        zero_chunk8<T>(next[1]);
        if (token < p.cta_tokens && piece.there && s_where[token].param) {
            const T* src = piece.dense_at(token);
            next[0] = load8<T>(src, p.wide != 0);
            next[1] = load8<T>(src + 8, p.wide != 0);
        }
    };
    request(threadIdx.x >> 5);
#pragma unroll 1
    for (int token = threadIdx.x >> 5; token < p.cta_tokens; token += kTokWarps) {
        const Chunk8<T> chunk[2] = {next[0], next[1]};
        request(token + kTokWarps);  // on its way while this one is worked on
        if (!s_where[token].param) continue;  // all of the warp
        float f[16], low, high;
        unpack8(chunk[0], *reinterpret_cast<float(*)[8]>(&f[0]));
        unpack8(chunk[1], *reinterpret_cast<float(*)[8]>(&f[8]));
        least_greatest(f, chunk, low, high);
        const bool fine = fabsf(low) < INFINITY && fabsf(high) < INFINITY;
        const float zero = low + 0.0f;  // -0 becomes 0
        const float scale = fine ? scale_of(low, high, static_cast<const T*>(nullptr)) : 0.0f;
        const uint2 words = two_words<T>(f, zero, high, scale);
        __syncwarp();
        if (!piece.there) continue;
        if (piece.of == 0) {
            *reinterpret_cast<uint2*>(piece.word_at(token)) = words;
        } else {
            piece.word_at(token)[0] = words.x;
            piece.word_at(token)[D / 16] = words.y;  // four units on: the next eight channels' lane
        }
        if (threadIdx.x % 4 == 0) write_param<T>(piece.param_at(token), scale, zero, fine);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kTokThreads) kv4_read_kernel(const __grid_constant__ Kv4TokenParams p) {
    __shared__ Kv4Where s_where[kMaxCtaTokens];
    if ((int)threadIdx.x < p.cta_tokens) kv4_find<T, D>(p, (long long)blockIdx.x * p.cta_tokens + threadIdx.x, s_where[threadIdx.x]);
    const Kv4Piece<T, D, 8> piece(p, s_where);
    __syncthreads();
    if (!piece.there) return;
#pragma unroll 1
    for (int first = threadIdx.x >> 5; first < p.cta_tokens; first += kTokWarps * kBatch) {
        unsigned word[kBatch];
        Kv4Param<T> param[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int token = first + b * kTokWarps;
            if (token < p.cta_tokens && s_where[token].param) {
                word[b] = *piece.word_at(token);
                param[b] = *reinterpret_cast<const Kv4Param<T>*>(piece.param_at(token));
            }
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int token = first + b * kTokWarps;
            if (token >= p.cta_tokens || s_where[token].t == kKv4Tile) continue;  // behind the last row's tokens: left as it was
            Chunk8<T> out;
            if (s_where[token].param) {
                dequantise(word[b], param[b], out);
            } else {
                const T fill = from_float<T>(s_where[token].t < 0 ? 0.0f : __uint_as_float(0x7fc00000u));
#pragma unroll
                for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(&out)[i] = fill;
            }
            store8(piece.dense_at(token), p.wide != 0, out);
        }
    }
}

int kv4_view(const mk36_kv4_cache* c, const char* what, Kv4View* v) {
    if (!c) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: cache is NULL", what);
    if (!c->pool || !c->page_table || !c->lengths) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: NULL tensor pointer", what);
    if (c->dtype != MK36_BF16 && c->dtype != MK36_F16 && c->dtype != MK36_F32) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: unsupported dtype %d", what, c->dtype);
    if (c->pages <= 0 || c->kv_heads <= 0 || c->rows <= 0 || c->row_pages <= 0 || c->page_size <= 0)
        MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: sizes must be positive", what);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256", what);
    if (c->page_size % kKv4Tile != 0) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: page_size must be a multiple of %d", what, kKv4Tile);
    if (c->kv_heads > 1 << 20) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: too many heads", what);
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
static int kv4_tokens_launch(Kv4TokenParams p, bool append, cudaStream_t s, const char* what) {
    const DeviceInfo* info = current_device_info();
    if (!info) return MK36_ERR_LAUNCH;
    const long long groups = (2ll * p.cache.kv_heads * (D / (append ? 16 : 8)) + 31) / 32;
    if (groups > 65535) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: too many heads", what);
    // 32 tokens a CTA; fewer where that would leave SMs without work
    p.cta_tokens = kMaxCtaTokens;
    while (p.cta_tokens > kTokWarps && p.total * groups < p.cta_tokens * 8ll * info->sm_count) p.cta_tokens /= 2;
    const dim3 ctas((unsigned)((p.total + p.cta_tokens - 1) / p.cta_tokens), (unsigned)groups);
    if (append) kv4_append_kernel<T, D><<<ctas, kTokThreads, 0, s>>>(p);
    else kv4_read_kernel<T, D><<<ctas, kTokThreads, 0, s>>>(p);
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
    p.clear = t->clear_rest;
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
