// The paged cache that holds keys and values in 4 bits: where everything lies.
//
// A page holds page_size tokens of every KV head.  Its unit is the tile: 16 consecutive tokens of one KV head, in one
// contiguous block, pool[page][kv_head][tile_of_page][tile_bytes]:
//     key codes 8 D | value codes 8 D | key parameters | value parameters
// A code is 4 bits; a group of 64 channels of a token shares a scale and a zero point in the activations' type (parameters:
// [16 tokens][D / 64 groups]{scale, zero}), and an entry stands for zero + code * scale.
//
// Codes lie in the order in which mma.sync.m16n8k16 takes them, so that a warp reads a tile with consecutive vectors, lane
// after lane, and turns a 32-bit word into two operand registers with two masks each: the half with bits 0x000n is the
// subnormal n * 2^-24, exactly.  Lane = 4 g + j:
//   * keys (A: 16 tokens x 16 channels): lane reads tokens g and g + 8, and of each group of 64 the channels 16 j .. 16 j + 15;
//   * values (A: 16 channels x 16 tokens): lane reads tokens 2 j, 2 j + 1, 2 j + 8, 2 j + 9, and of each group the channels
//     8 g .. 8 g + 7.
// Eight consecutive channels of a token are one 32-bit word in both, so a token is written without touching its neighbours.
#pragma once

#include "mk36_common.cuh"

namespace mk36 {

constexpr int kKv4Tile = 16;   // tokens of a tile
constexpr int kKv4Group = 64;  // channels that share a scale and a zero point

__host__ __device__ constexpr int kv4_code_bytes(int d) { return 8 * d; }                    // of the keys, or of the values, of a tile
__host__ __device__ constexpr int kv4_param_bytes(int d, int elem) { return d * elem / 2; }  // 16 tokens * d / 64 groups * 2
__host__ __device__ constexpr int kv4_tile_bytes(int d, int elem) { return 16 * d + d * elem; }

inline int kv4_elem(int dtype) { return dtype == MK36_F32 ? 4 : 2; }

// What every kernel over the cache needs.
struct Kv4View {
    unsigned char* pool;
    const int* table;    // [rows][row_pages]
    const int* lengths;  // [rows]
    long long pages;
    int kv_heads, rows, row_pages;
    int capacity;  // tokens that a row of the table can hold
    FastDiv tiles_per_page;
    unsigned tile_bytes;
};

// Fills the view; returns MK36_OK or an error with its text set.  `what` names the operator.
int kv4_view(const mk36_kv4_cache* c, const char* what, Kv4View* v);

#if defined(__CUDACC__)

__device__ __forceinline__ int kv4_length(const Kv4View& v, int row) {
    return max(0, min(v.lengths[row], v.capacity));
}

// Byte of the 32-bit word with the key codes of channels c .. c + 7 (c a multiple of eight) of token t of a tile.
template <int D>
__device__ __forceinline__ int kv4_key_word(int t, int c) {
    constexpr int kUnit = D >= 128 ? 16 : 8;
    const int inside = (c / kKv4Group) * 8 + ((c & 8) >> 1);
    const int vec = inside / kUnit;
    return ((t >> 3) * (D / 8 / kUnit) + vec) * (32 * kUnit) + ((t & 7) * 4 + (c % kKv4Group) / 16) * kUnit + inside % kUnit;
}

// The same of the value codes.
template <int D>
__device__ __forceinline__ int kv4_value_word(int t, int c) {
    constexpr int kUnit = D / 16;
    const int quarter = (t & 1) | ((t >> 3) << 1);
    return kv4_code_bytes(D) + quarter * (32 * kUnit) + (((c % kKv4Group) / 8) * 4 + ((t & 7) >> 1)) * kUnit + (c / kKv4Group) * 4;
}

// Scale and zero point of a group, as they lie in the cache.
template <typename T>
struct Kv4Param {
    unsigned raw;
};
template <>
struct Kv4Param<float> {
    float scale, zero;
};

__device__ __forceinline__ void kv4_unpack(const Kv4Param<__nv_bfloat16>& p, float& scale, float& zero) {
    scale = __uint_as_float(p.raw << 16);
    zero = __uint_as_float(p.raw & 0xffff0000u);
}
__device__ __forceinline__ void kv4_unpack(const Kv4Param<__half>& p, float& scale, float& zero) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p.raw));
    scale = f.x;
    zero = f.y;
}
__device__ __forceinline__ void kv4_unpack(const Kv4Param<float>& p, float& scale, float& zero) {
    scale = p.scale;
    zero = p.zero;
}

// Two fp32 operations an instruction, each rounded as one alone would be.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair_of(float x, float y) {
    f32x2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}
__device__ __forceinline__ float first_of(f32x2 v) { return __uint_as_float((unsigned)v); }
__device__ __forceinline__ float second_of(f32x2 v) { return __uint_as_float((unsigned)(v >> 32)); }
__device__ __forceinline__ f32x2 add_pair(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 fma_pair(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ f32x2 mul_pair(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

#endif  // __CUDACC__

}  // namespace mk36
