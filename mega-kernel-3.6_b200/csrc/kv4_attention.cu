// Attention over the 4-bit paged cache, for the last token or the last few of every row.
//
// Mathematics.  A key entry stands for z + n s with a code n of 4 bits and s, z of its group of 64 channels, a value entry likewise:
//     score_t = sum_groups s_tg (q_g . n_tg) + z_tg sum(q_g)          out_c = sum_t (p_t s'_tg) n'_tc + sum_t p_t z'_tg
// so scales and zero points never touch an element: keys get theirs on the products of a group, values on the weights.  What is left
// per element is to turn codes into operands, and there f16 helps: the bits 0x000n are the subnormal n 2^-24, 0x00n0 is n 2^-20, so
// a 32-bit word of eight codes becomes four operand registers with four masks and one shift (five instructions for eight codes).  The
// factor 16 of every second register goes into q (keys) or into the result (values).
//   q is scaled by a power of two so that its largest channel is in [2^14, 2^15), exact for bf16 and for f16.  Weights times scales
// are divided by the power of two of the largest scale met so far, so that f16 holds them whatever the size of the values; they are held
// in two halves (hi + lo, 22 bits), because what the codes stand for has a zero point: the error of a rounded weight would be
// multiplied by a code of 0 .. 15 where the value itself may be near zero.
//
// Work.  Four warps a CTA, two CTAs an SM.  A warp takes a tile (16 tokens of a KV head) on its own: scores as MMAs of 16 tokens x 16
// channels by 8 columns (the query heads and tokens that share the KV head), a transposition of the 16 x 8 scores inside the warp,
// running maximum and sum, values as MMAs of 16 channels x 16 tokens.  Tiles come through a ring of the warp's own, one bulk copy
// each (a tile is contiguous), so that nothing but the end of a segment needs the other warps.  All tiles of all rows and heads form one line
// that is cut into as many equal pieces as there are CTAs; a piece that ends inside a row leaves a partial result, and a second launch
// joins those.
#include <math.h>

#include <type_traits>

#include "mk36_kv4.cuh"
#include "mk36_mma.cuh"
#include "mk36_ring.cuh"

namespace mk36 {

#ifndef KA_CTAS
#define KA_CTAS 2
#endif
#ifndef KA_STEP
#define KA_STEP 2
#endif
constexpr int kKaWarps = 4;
constexpr int kKaThreads = kKaWarps * 32;
constexpr int kKaMinTiles = 8;     // fewest tiles of a piece: two a warp
constexpr int kKaJoinThreads = 256;

struct Kv4AttnParams {
    Kv4View cache;
    const void* q;
    void* out;
    float* partial;
    long long q_row, q_token, q_head;
    int query_heads, tokens, group, columns;  // group: query heads of a KV head; columns: group * tokens
    int blocks;                               // pieces of the columns, 8 or 16 each
    int streams;                              // kv_heads * blocks: passes over a row
    int ctas, wide_q;
    float scale;
    FastDiv fd_blocks, fd_group, fd_streams;
};

// Partial results: per (CTA, first or last segment) and column the sums, then maximum (of scores in units of log 2) and sum of weights.
__host__ __device__ constexpr int ka_slot_floats(int d, int nt) { return 8 * nt * (d + 4); }

// What their registers leave room for.
__host__ __device__ constexpr int ka_ctas_per_sm(bool fp32, int nt) { return fp32 || nt == 2 ? 2 : KA_CTAS; }
__host__ __device__ constexpr int ka_step(bool fp32, int nt) { return fp32 || nt == 2 ? 1 : KA_STEP; }


template <typename T, int D, int NT>
struct KaConfig {
    static constexpr int kGroups = D / kKv4Group;
    static constexpr int kTile = kv4_tile_bytes(D, sizeof(T));
    static constexpr int kQParts = sizeof(T) == 4 ? 2 : 1;
    static constexpr int kCtas = ka_ctas_per_sm(sizeof(T) == 4, NT);
    static constexpr int kFoldRow = D + 8;  // the lanes of a store (g, j), rows j apart, fall into 32 banks
    static constexpr int kFold = kKaWarps * 4 * kFoldRow * 4;
    static constexpr int kOperands = NT * kQParts * kGroups * 4 * 32 * 8;  // of the queries
    static constexpr int kStats = (kKaWarps * 8 * NT * 2 + 8 * NT * kGroups * 2) * 4;
    static constexpr int kRoom = 232448 / kCtas - 1024 - kFold - kOperands - kStats - 512;
    // tiles a warp takes together: two where the registers allow it
    static constexpr int kStep = ka_step(sizeof(T) == 4, NT);
    static constexpr int kMost = kRoom / (kKaWarps * kTile);
    static constexpr int kStages = kMost < 8 ? kMost : 8;
    static constexpr int kSmem = kKaWarps * kStages * kTile + kFold + kOperands + kStats + kKaWarps * kStages * 8;
    static_assert(kStages > kStep, "no room for a ring");
};

__device__ __forceinline__ unsigned movmatrix(unsigned a) {
    unsigned d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// lane (g, j) holds (row g, columns 2 j, 2 j + 1) of an 8 x 8 block of fp32; afterwards (column g, rows 2 j, 2 j + 1).
__device__ __forceinline__ void transpose8(float& x, float& y) {
    const unsigned a = __float_as_uint(x), b = __float_as_uint(y);
    const unsigned lo = movmatrix(__byte_perm(a, b, 0x5410)), hi = movmatrix(__byte_perm(a, b, 0x7632));
    x = __uint_as_float(__byte_perm(lo, hi, 0x5410));
    y = __uint_as_float(__byte_perm(lo, hi, 0x7632));
}

// D += A B, 16 x 16 by 16 x 8; not volatile, so that the compiler may place it
__device__ __forceinline__ void ka_mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}

// x - h, one instruction
__device__ __forceinline__ float minus_half(float x, __half h) {
    float d;
    asm("fma.rn.f32.f16 %0, %1, %2, %3;" : "=f"(d) : "h"(*reinterpret_cast<const unsigned short*>(&h)), "h"((unsigned short)0xbc00), "f"(x));
    return d;
}

// hi and lo halves of two fp32 values: 22 bits together
__device__ __forceinline__ void split_half(float x, float y, unsigned& hi, unsigned& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    hi = *reinterpret_cast<const unsigned*>(&h);
    lo = pack_half(minus_half(x, __low2half(h)), minus_half(y, __high2half(h)));
}

// The two-byte types' parameters are worked on as they lie: pairs of halves in a word.
template <typename T>
struct KaPair;
template <>
struct KaPair<__nv_bfloat16> {
    static constexpr unsigned kExponent = 0x7f80u, kTop = 255u;
    static constexpr int kShift = 7, kLeast = 23, kBias = 127;
    // scales as f16, 2^(unit - bias) as 2^7: a shift of the exponents.  Scales 2^21 times smaller than that become 0.
    static __device__ __forceinline__ unsigned scales(unsigned w, int unit) {
        const unsigned c = (unsigned)(unit - 22) * 0x00800080u;
        return __vmaxu2(w, c) * 8u - c * 8u;
    }
    static __device__ __forceinline__ unsigned pack(float x, float y) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const unsigned*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(unsigned w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
};
template <>
struct KaPair<__half> {
    static constexpr unsigned kExponent = 0x7c00u, kTop = 31u;
    static constexpr int kShift = 10, kLeast = 7, kBias = 15;
    static __device__ __forceinline__ unsigned scales(unsigned w, int unit) {
        const unsigned f = (unsigned)(22 - unit + 15) * 0x04000400u;  // 2^(22 - unit), twice
        const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&f));
        return *reinterpret_cast<const unsigned*>(&h);
    }
    static __device__ __forceinline__ unsigned pack(float x, float y) { return pack_half(x, y); }
    static __device__ __forceinline__ float2 unpack(unsigned w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
};

template <typename T>
__device__ __forceinline__ void ka_mma_params(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    if (std::is_same<T, __nv_bfloat16>::value) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        ka_mma(d, a0, a1, a2, a3, b0, b1);
    }
}

__device__ __forceinline__ __half2 as_half2(unsigned w) { return *reinterpret_cast<const __half2*>(&w); }
__device__ __forceinline__ unsigned as_word(__half2 h) { return *reinterpret_cast<const unsigned*>(&h); }

// 2^e, e in [-126, 127]
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// 2^e <= most < 2^(e + 1), within what pow2 takes on either side
__device__ __forceinline__ int ka_exponent(float most) { return min(max((int)(__float_as_uint(most) >> 23), 14), 254) - 127; }

template <int N>
__device__ __forceinline__ void lds_words(const unsigned char* p, unsigned (&w)[N]) {
    if (N == 1) {
        w[0] = *reinterpret_cast<const unsigned*>(p);
    } else if (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[N > 1 ? 1 : 0] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * i);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    }
}

// Which halves of a pair of tokens t, t + 1 lie below `end`.
__device__ __forceinline__ unsigned ka_keep(int t, int end) { return (t < end ? 0x0000ffffu : 0u) | (t + 1 < end ? 0xffff0000u : 0u); }

// Weights (two halves) times scales, again in two halves: the product rounded, and what the rounding left plus the weights' second halves.
__device__ __forceinline__ void ka_weigh(unsigned ph, unsigned pl, unsigned scale, unsigned& hi, unsigned& lo) {
    const __half2 h = __hmul2(as_half2(ph), as_half2(scale));
    hi = as_word(h);
    lo = as_word(__hfma2(as_half2(pl), as_half2(scale), __hfma2(as_half2(ph), as_half2(scale), __hneg2(h))));
}

// The least unit, and what a sum in units of it is multiplied by.
template <typename T>
__device__ __forceinline__ int ka_least_unit() {
    if constexpr (sizeof(T) == 4) return 1;
    else return KaPair<T>::kLeast;
}
template <typename T>
__device__ __forceinline__ float ka_unit_value(int unit) {
    if constexpr (sizeof(T) == 4) return pow2(unit - 127);
    else return pow2(unit - KaPair<T>::kBias - 7);
}

// Scales and zero points of a token's groups.
template <typename T, int G>
__device__ __forceinline__ void load_params(const unsigned char* p, float (&s)[G], float (&z)[G]) {
    unsigned w[G * sizeof(T) / 2];
    lds_words(p, w);
#pragma unroll
    for (int i = 0; i < G; ++i) {
        if (sizeof(T) == 4) {
            s[i] = __uint_as_float(w[(2 * i) % (G * (int)sizeof(T) / 2)]);
            z[i] = __uint_as_float(w[(2 * i + 1) % (G * (int)sizeof(T) / 2)]);
        } else {
            Kv4Param<typename std::conditional<sizeof(T) == 4, __half, T>::type> one{w[i]};
            kv4_unpack(one, s[i], z[i]);
        }
    }
}

// A place in the line of all tiles: row, pass over the row (KV head and block of columns), tile.
struct KaCursor {
    int row, stream, tile, tiles;
};

__device__ __forceinline__ int ka_tiles(const Kv4View& v, int row) { return (kv4_length(v, row) + kKv4Tile - 1) / kKv4Tile; }

__device__ __forceinline__ void ka_advance(const Kv4AttnParams& p, KaCursor& c, int by) {
    c.tile += by;
    while (c.row < p.cache.rows && c.tile >= c.tiles) {
        c.tile -= c.tiles;
        if (++c.stream == p.streams) {
            c.stream = 0;
            c.tiles = 0;
            while (++c.row < p.cache.rows && (c.tiles = ka_tiles(p.cache, c.row)) == 0) {
            }
        }
    }
}

// All CTAs cut the line alike: tiles of all rows, and the piece length.  Every thread calls it; s: 32 words.
template <int kThreads>
__device__ __forceinline__ int ka_line(const Kv4AttnParams& p, int rows, int* s) {
    int mine = 0;  // the whole line is below 2^31 tiles, which the host sees to
    for (int r = threadIdx.x; r < rows; r += kThreads) mine += ka_tiles(p.cache, r);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(kFullMask, mine, off);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = mine;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) sum += s[w];
    return sum * p.streams;
}

__device__ __forceinline__ int ka_piece(int total, int ctas) {
    return max(kKaMinTiles, (int)(((unsigned)total + (unsigned)ctas - 1u) / (unsigned)ctas));
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kKaThreads, KaConfig<T, D, NT>::kCtas) kv4_attention_kernel(const __grid_constant__ Kv4AttnParams p) {
    using C = KaConfig<T, D, NT>;
    constexpr int G = C::kGroups, QP = C::kQParts;
    constexpr bool kWide = sizeof(T) == 4;
    constexpr int kStep = C::kStep;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int s_scan[kKaWarps], s_start[2], s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
    unsigned char* ring = smem + warp * C::kStages * C::kTile;
    float* s_fold = reinterpret_cast<float*>(smem + kKaWarps * C::kStages * C::kTile);
    uint4* s_qf = reinterpret_cast<uint4*>(s_fold + C::kFold / 4);  // [NT][QP][G][2][32]: operand registers of the queries, of two MMAs each
    float* s_max = reinterpret_cast<float*>(s_qf) + C::kOperands / 4;  // [warp][8 NT]
    float* s_sum = s_max + kKaWarps * 8 * NT;           // [warp][8 NT]
    float* s_most = s_sum + kKaWarps * 8 * NT;          // [G][8 NT]: largest |q|
    float* s_qsum = s_most + G * 8 * NT;                // [8 NT][G]
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(s_qsum + 8 * NT * G) + warp * C::kStages;
    if (lane == 0) {
        for (int i = 0; i < C::kStages; ++i) mbar_init(&bars[i], 1);
        mbar_init_fence();
    }
    if (threadIdx.x == 0) s_abort = 0;
    asm volatile("griddepcontrol.launch_dependents;");  // the join may be set up while this runs; it waits for the end of the grid

    // ---- this CTA's piece of the line
    const int total = ka_line<kKaThreads>(p, p.cache.rows, s_scan);
    const int piece = ka_piece(total, p.ctas);
    if ((long long)blockIdx.x * piece >= total) return;
    const int begin = blockIdx.x * piece, end = total - begin < piece ? total : begin + piece;
    {
        // the row that holds tile `begin`: rows in batches of a thread each
        int before = 0;
        const int target = fdiv(begin, p.fd_streams);  // begin's row has before * streams <= begin < (before + tiles) * streams
        for (int base = 0;; base += kKaThreads) {
            const int r = base + threadIdx.x;
            const int n = r < p.cache.rows ? ka_tiles(p.cache, r) : 0;
            int inc = n;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int x = __shfl_up_sync(kFullMask, inc, off);
                if (lane >= off) inc += x;
            }
            __syncthreads();
            if (lane == 31) s_scan[warp] = inc;
            __syncthreads();
            int all = 0, lower = before;
#pragma unroll
            for (int w = 0; w < kKaWarps; ++w) {
                if (w < warp) lower += s_scan[w];
                all += s_scan[w];
            }
            const int first = lower + inc - n;
            if (first <= target && target < first + n) s_start[0] = r, s_start[1] = first;
            before += all;
            if (before > target || base + kKaThreads >= p.cache.rows) break;
        }
        __syncthreads();
    }
    KaCursor start;
    start.row = s_start[0];
    start.tiles = ka_tiles(p.cache, start.row);
    {
        const int off = begin - s_start[1] * p.streams;
        start.stream = (unsigned)off / (unsigned)start.tiles;
        start.tile = off - start.stream * start.tiles;
    }

    // ---- the ring: this warp's tiles are begin + warp, begin + warp + kKaWarps, ...  Lane i looks up where the i-th of the next 32 lies,
    // a batch ahead, so that no request waits for the table
    KaCursor place = start;
    int place_at = begin + warp + kKaWarps * lane;
    if (place_at < end) ka_advance(p, place, warp + kKaWarps * lane);
    auto look_up = [&]() -> const unsigned char* {
        const unsigned char* src = nullptr;  // null: the table names no page of the pool
        if (place_at < end) {
            int slot, inner;
            fdivmod(place.tile, p.cache.tiles_per_page, slot, inner);
            const long long page = p.cache.table[(long long)place.row * p.cache.row_pages + slot];
            if (page >= 0 && page < p.cache.pages)
                src = p.cache.pool + ((page * p.cache.kv_heads + fdiv(place.stream, p.fd_blocks)) * (int)p.cache.tiles_per_page.d + inner) * C::kTile;
            place_at += 32 * kKaWarps;
            if (place_at < end) ka_advance(p, place, 32 * kKaWarps);
        }
        return src;
    };
    const unsigned char *src_now = look_up(), *src_next = nullptr;
    int requested = 0;
    unsigned lost = 0;  // bit s: stage s holds another tile, because the table names none
    auto request = [&](int stage) {
        if (begin + warp + requested * kKaWarps >= end) return;
        if (requested % 32 == 0) {
            if (requested > 0) src_now = src_next;
            src_next = look_up();
        }
        const unsigned char* src = reinterpret_cast<const unsigned char*>(__shfl_sync(kFullMask, reinterpret_cast<unsigned long long>(src_now), requested % 32));
        lost = (lost & ~(1u << stage)) | (src ? 0u : 1u << stage);
        if (lane == 0) {
            mbar_arrive_expect_tx(&bars[stage], C::kTile);
            bulk_copy_g2s(ring + stage * C::kTile, src ? src : p.cache.pool, C::kTile, &bars[stage]);
        }
        ++requested;
    };
    __syncwarp();
    for (int i = 0; i < C::kStages; ++i) request(i);

    int stage = 0, use = 0;
    bool dead = false;  // a wait has run out: outputs from here on are NaN
    int at = begin + warp, segment = begin;
    KaCursor now = start;  // the tile at `segment`
    while (segment < end) {
        const int segment_end = end - segment < now.tiles - now.tile ? end : segment + (now.tiles - now.tile);
        const bool whole = now.tile == 0 && segment_end - segment == now.tiles;
        const int length = kv4_length(p.cache, now.row);
        const int kv_head = fdiv(now.stream, p.fd_blocks), block = now.stream - kv_head * p.blocks;
        const int row = now.row;

        // ---- the queries of this pass.  A warp prepares one group of 64 channels of every column (lane: column g, channels 16 j .. + 15);
        // the operand registers stay in shared memory, where every tile takes them from.
        float mult[NT];             // factor of column g's scores, in units of log 2
        float q_sum[NT][2][kWide ? G : 1];  // fp32: sums over the groups' channels of columns 2 j, 2 j + 1
        unsigned q_zero[NT][2];     // two-byte types: the sums of column g as operand registers, against the zero points
        int limit[NT][2], own_limit[NT];  // positions that the columns 2 j, 2 j + 1 see, and column g
        {
            float q[NT][16];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int column = (block * NT + nt) * 8 + g, token = fdiv(column, p.fd_group);
                own_limit[nt] = length - p.tokens + 1 + token;
#pragma unroll
                for (int i = 0; i < 16; ++i) q[nt][i] = 0.f;
                if (warp >= G) continue;
                float most = 0.f;
                if (column < p.columns) {
                    const T* src = static_cast<const T*>(p.q) + row * p.q_row + token * p.q_token + (kv_head * p.group + column - token * p.group) * p.q_head +
                                   warp * kKv4Group + 16 * j;
                    if (p.wide_q) {
                        float f[2][8];
                        unpack8(load_chunk8<T>(src), f[0]);
                        unpack8(load_chunk8<T>(src + 8), f[1]);
#pragma unroll
                        for (int i = 0; i < 16; ++i) q[nt][i] = f[i >> 3][i & 7];
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) q[nt][i] = to_float<T>(src[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(q[nt][i]));
                most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 1));
                most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 2));
                if (j == 0) s_most[warp * 8 * NT + nt * 8 + g] = most;
            }
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (warp >= G) continue;
                float most = 0.f;
#pragma unroll
                for (int gr = 0; gr < G; ++gr) most = fmaxf(most, s_most[gr * 8 * NT + nt * 8 + g]);
                const float up = copysignf(pow2(14 - ka_exponent(most)), p.scale);  // the scale's sign goes into q
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    q[nt][i] *= up;
                    sum += q[nt][i];
                }
                sum += __shfl_xor_sync(kFullMask, sum, 1);
                sum += __shfl_xor_sync(kFullMask, sum, 2);
                if (j == 0) s_qsum[(nt * 8 + g) * G + warp] = sum * pow2(-24);
#pragma unroll
                for (int w = 0; w < 2; ++w) {  // MMA m takes the codes 2 (m % 2), + 1, + 4, + 5 of word m / 2
                    const float* x = &q[nt][8 * w];
                    uint4 hi, lo;
                    split_half(x[0], x[4], hi.x, lo.x);
                    split_half(x[1] * 0.0625f, x[5] * 0.0625f, hi.y, lo.y);
                    split_half(x[2], x[6], hi.z, lo.z);
                    split_half(x[3] * 0.0625f, x[7] * 0.0625f, hi.w, lo.w);
                    s_qf[(((nt * QP) * G + warp) * 2 + w) * 32 + lane] = hi;
                    if (QP == 2) s_qf[(((nt * QP + QP - 1) * G + warp) * 2 + w) * 32 + lane] = lo;
                }
            }
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float most = 0.f;
#pragma unroll
                for (int gr = 0; gr < G; ++gr) most = fmaxf(most, s_most[gr * 8 * NT + nt * 8 + g]);
                // not 0, so that a score of -infinity stays one
                mult[nt] = fmaxf(ldexpf(fabsf(p.scale) * 1.4426950408889634f, 24 - 14 + ka_exponent(most)), 1e-37f);
                // what belongs to a column, for the lanes that hold it in the products' layout: columns 2 j, 2 j + 1
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    limit[nt][c] = __shfl_sync(kFullMask, own_limit[nt], (2 * j + c) * 4);
                    if constexpr (kWide) {
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) q_sum[nt][c][gr] = s_qsum[(nt * 8 + 2 * j + c) * G + gr];
                    }
                }
                if constexpr (!kWide) {
                    // k = 0..3 and 4..7 (and 8..15 for bf16): the sums of the groups, in two parts (four) that add up to 22 bits (32)
                    float x[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) x[i] = 2 * (j & 1) + i < G ? s_qsum[(nt * 8 + g) * G + (2 * (j & 1) + i) % G] : 0.f;
                    if (std::is_same<T, __half>::value) x[0] *= pow2(16), x[1] *= pow2(16);  // room for f16's second part; taken back below
                    unsigned part[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        part[i] = KaPair<T>::pack(x[0], x[1]);
                        const float2 f = KaPair<T>::unpack(part[i]);
                        x[0] -= f.x, x[1] -= f.y;
                    }
                    const bool second = j >> 1;
                    q_zero[nt][0] = second ? part[1] : part[0];
                    q_zero[nt][1] = std::is_same<T, __half>::value ? 0u : (second ? part[3] : part[2]);
                }
            }
        }
        int sees_all = length;  // every column sees the positions below this
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sees_all = min(sees_all, min(limit[nt][0], limit[nt][1]));
        sees_all = min(sees_all, __shfl_xor_sync(kFullMask, sees_all, 1));
        sees_all = min(sees_all, __shfl_xor_sync(kFullMask, sees_all, 2));

        // zero_sum: the zero points' part, of column g for every group (fp32), or as an MMA leaves it: row g % 4 (the group), columns 2 j, 2 j + 1
        constexpr int Z = kWide ? G : 4;
        float o[NT][G][4][4], zero_sum[NT][Z], top[NT], limit_top[NT], shift[NT], weight_sum[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            top[nt] = limit_top[nt] = -INFINITY;
            shift[nt] = weight_sum[nt] = 0.f;
#pragma unroll
            for (int i = 0; i < Z; ++i) zero_sum[nt][i] = 0.f;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[nt][gr][m][i] = 0.f;
            }
        }
        int unit = ka_least_unit<T>(), unit_limit = -1;  // exponent field of the scale that the values' sums are in units of; none yet

        while (at < segment_end) {
            // kStep tiles together: their chains of dependent instructions run side by side.  A tile that is not there counts as one that
            // nothing is seen of.
            const unsigned char* codes[kStep];
            int first[kStep], count = 0;
#pragma unroll
            for (int u = 0; u < kStep; ++u) {
                codes[u] = codes[0];
                first[u] = 0x3fffff00;
                if (u == 0 || at + u * kKaWarps < segment_end) {
                    ++count;
                    const int st = stage + u < C::kStages ? stage + u : stage + u - C::kStages;
                    if (!dead && !mbar_wait(&bars[st], (use + (st < stage)) & 1, &s_abort)) dead = true;
                    if (lost >> st & 1u) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) weight_sum[nt] = __uint_as_float(0x7fc00000u);
                    }
                    codes[u] = ring + st * C::kTile;
                    first[u] = (now.tile + (at - segment) + u * kKaWarps) * kKv4Tile;
                }
            }
            at += count * kKaWarps;
            dead = __any_sync(kFullMask, dead);
            if (dead) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) weight_sum[nt] = __uint_as_float(0x7fc00000u);
                continue;
            }

            // ---- scores
            float s[kStep][NT][4];
#pragma unroll
            for (int u = 0; u < kStep; ++u) {
                const unsigned char* params = codes[u] + 2 * kv4_code_bytes(D);
                constexpr int kUnit = D >= 128 ? 16 : 8, kVecs = D / 8 / kUnit, kWords = kUnit / 4;
                unsigned a[kVecs][kWords], a8[kVecs][kWords];  // tokens g and g + 8
#pragma unroll
                for (int v = 0; v < kVecs; ++v) {
                    lds_words(codes[u] + (v * 32 + lane) * kUnit, a[v]);
                    lds_words(codes[u] + ((kVecs + v) * 32 + lane) * kUnit, a8[v]);
                }
                float ks[2][G], kz[2][G];
                load_params<T, G>(params + g * (G * 2 * (int)sizeof(T)), ks[0], kz[0]);
                load_params<T, G>(params + (g + 8) * (G * 2 * (int)sizeof(T)), ks[1], kz[1]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[u][nt][i] = 0.f;
                if constexpr (!kWide) {  // zero points times sums of the queries: one MMA, tokens x groups by groups x columns
                    unsigned z[2][G > 1 ? 2 : 1];  // of tokens g and g + 8: groups 2 (j % 2) and the next
                    lds_words(params + (g * G + (2 * (j & 1)) % G) * 4, z[0]);
                    lds_words(params + ((g + 8) * G + (2 * (j & 1)) % G) * 4, z[1]);
                    const unsigned a0 = __byte_perm(z[0][0], z[0][G > 1 ? 1 : 0], 0x7632), a1 = __byte_perm(z[1][0], z[1][G > 1 ? 1 : 0], 0x7632);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        ka_mma_params<T>(s[u][nt], a0, a1, a0, a1, q_zero[nt][0], q_zero[nt][1]);
                        if (std::is_same<T, __half>::value) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[u][nt][i] *= pow2(-16);
                        }
                    }
                }
                float acc[NT][G][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int gr = 0; gr < G; ++gr)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[nt][gr][i] = 0.f;
#pragma unroll
                for (int w = 0; w < 2; ++w) {  // the groups' chains side by side: an MMA does not wait for the one before it
                    uint4 b[NT][QP][G];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int part = 0; part < QP; ++part)
#pragma unroll
                            for (int gr = 0; gr < G; ++gr) b[nt][part][gr] = s_qf[(((nt * QP + part) * G + gr) * 2 + w) * 32 + lane];
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) {
                            const int v = gr / (kWords / 2), x = 2 * (gr % (kWords / 2)) + w;
                            const unsigned wa = a[v][x] >> (8 * m), wb = a8[v][x] >> (8 * m);
                            const unsigned a0 = wa & 0x000f000fu, a1 = wb & 0x000f000fu, a2 = wa & 0x00f000f0u, a3 = wb & 0x00f000f0u;
#pragma unroll
                            for (int part = 0; part < QP; ++part)
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
                                    ka_mma(acc[nt][gr], a0, a1, a2, a3, m ? b[nt][part][gr].z : b[nt][part][gr].x, m ? b[nt][part][gr].w : b[nt][part][gr].y);
                        }
                    }
                }
#pragma unroll
                for (int gr = 0; gr < G; ++gr)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if constexpr (kWide) s[u][nt][i] = fmaf(kz[i >> 1][gr], q_sum[nt][i & 1][gr], s[u][nt][i]);
                            s[u][nt][i] = fmaf(ks[i >> 1][gr], acc[nt][gr][i], s[u][nt][i]);
                        }
            }
            bool edge[kStep];
#pragma unroll
            for (int u = 0; u < kStep; ++u) {
                edge[u] = first[u] + kKv4Tile > sees_all;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (edge[u]) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (first[u] + g + 8 * (i >> 1) >= limit[nt][i & 1]) s[u][nt][i] = -INFINITY;
                    }
                    // from (tokens g, g + 8; columns 2 j, 2 j + 1) to (tokens 2 j, 2 j + 1, + 8, + 9; column g)
                    transpose8(s[u][nt][0], s[u][nt][1]);
                    transpose8(s[u][nt][2], s[u][nt][3]);
                }
            }

            // ---- scales of the values of the lane's four tokens.  The sums are kept in units of a scale's power of two, so that f16 holds
            // weights times scales, and the unit is raised when a scale is 2^4 times larger (2^9 for fp32).  The exponents' bits or'ed
            // together are no smaller than the largest; only where that says so, it is looked for.
            unsigned sw[kStep][2][G];  // two-byte types: pairs of tokens
            float vs[kStep][4][kWide ? G : 1], vz[kStep][4][kWide ? G : 1];
            bool larger = false;
#pragma unroll
            for (int u = 0; u < kStep; ++u) {
                const unsigned char* v_params = codes[u] + 2 * kv4_code_bytes(D) + kv4_param_bytes(D, sizeof(T));
                if constexpr (!kWide) {
                    unsigned w[4][G], bits = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) lds_words(v_params + (2 * j + (i & 1) + 8 * (i >> 1)) * (G * 4), w[i]);
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) sw[u][0][gr] = __byte_perm(w[0][gr], w[1][gr], 0x5410), sw[u][1][gr] = __byte_perm(w[2][gr], w[3][gr], 0x5410);
                    if (edge[u]) {  // behind the row's end anything may lie
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const unsigned keep = ka_keep(first[u] + 2 * j + 8 * x, length);
#pragma unroll
                            for (int gr = 0; gr < G; ++gr) sw[u][x][gr] &= keep;
                        }
                    }
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) bits |= sw[u][0][gr] | sw[u][1][gr];
                    larger |= (int)((bits | bits >> 16) & KaPair<T>::kExponent) > unit_limit * (1 << KaPair<T>::kShift);
                } else {
                    unsigned bits = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int t = 2 * j + (i & 1) + 8 * (i >> 1);
                        load_params<T, G>(v_params + t * (G * 8), vs[u][i], vz[u][i]);
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) {
                            if (edge[u] && first[u] + t >= length) vs[u][i][gr] = vz[u][i][gr] = 0.f;
                            bits |= __float_as_uint(vs[u][i][gr]);
                        }
                    }
                    larger |= (int)(bits >> 23) > unit_limit;
                }
            }

            // ---- maximum.  Weights are taken relative to `top`, which follows the maximum only when that is 2^4 times larger: then, and not
            // with every tile, what has been summed is brought to the new one.
            float most[NT];
            bool moved = larger, poisoned = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float m = -INFINITY;
#pragma unroll
                for (int u = 0; u < kStep; ++u) m = fmaxf(m, fmaxf(fmaxf(s[u][nt][0], s[u][nt][1]), fmaxf(s[u][nt][2], s[u][nt][3])));
                m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 1));
                m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 2));
                most[nt] = m;
                moved |= m > limit_top[nt];
            }
            if (__any_sync(kFullMask, moved)) {
                float down = 1.f;
                if (__any_sync(kFullMask, larger)) {
                    int largest = 0;  // an exponent field; that of a NaN is no size: other columns may not see it
                    if constexpr (!kWide) {
#pragma unroll
                        for (int i = 0; i < kStep * 4 * G; ++i) {
                            const unsigned f = (sw[i / 4 / G][i / 2 / G % 2][i / 2 % G] >> (16 * (i & 1)) & KaPair<T>::kExponent) >> KaPair<T>::kShift;
                            if (f == KaPair<T>::kTop) poisoned = true;
                            else largest = max(largest, (int)f);
                        }
                        poisoned = __any_sync(kFullMask, poisoned);
                    } else {
#pragma unroll
                        for (int i = 0; i < kStep * 4; ++i)
#pragma unroll
                            for (int gr = 0; gr < G; ++gr) {
                                const int f = (int)(__float_as_uint(vs[i / 4][i % 4][gr]) >> 23);
                                if (f < 255) largest = max(largest, min(f, 253));
                            }
                    }
                    largest = __reduce_max_sync(kFullMask, largest);
                    if (largest > unit) {
                        down = pow2(max(unit - largest, -126));
                        unit = largest;
                    }
                    unit_limit = min(unit + (kWide ? 8 : 3), 254);  // the exponent of a NaN is always beyond it
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float m = fmaxf(top[nt], most[nt]);
                    const float corr = m == -INFINITY ? 0.f : exp2f((top[nt] - m) * mult[nt]);  // nothing has been summed without a maximum
                    top[nt] = m;
                    limit_top[nt] = m == -INFINITY ? m : m + 4.f / mult[nt];
                    shift[nt] = m == -INFINITY ? 0.f : -m * mult[nt];
                    weight_sum[nt] *= corr;
                    const float k0 = __shfl_sync(kFullMask, corr, 8 * j), k1 = __shfl_sync(kFullMask, corr, 8 * j + 4);
                    const float c0 = k0 * down, c1 = k1 * down;
                    if constexpr (kWide) {
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) zero_sum[nt][gr] *= corr;
                    } else {
                        zero_sum[nt][0] *= k0, zero_sum[nt][1] *= k1;
                    }
#pragma unroll
                    for (int gr = 0; gr < G; ++gr)
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            o[nt][gr][m][0] *= c0, o[nt][gr][m][1] *= c1;
                            o[nt][gr][m][2] *= c0, o[nt][gr][m][3] *= c1;
                        }
                }
            }

            // fp32: the difference first, which is exact where it matters
#pragma unroll
            for (int u = 0; u < kStep; ++u)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[u][nt][i] = kWide ? exp2f((s[u][nt][i] - (top[nt] == -INFINITY ? 0.f : top[nt])) * mult[nt]) : exp2_approx(fmaf(s[u][nt][i], mult[nt], shift[nt]));

            // ---- weights times scales, in two halves; the zero points' part
#pragma unroll
            for (int u = 0; u < kStep; ++u) {
                const unsigned char* v_params = codes[u] + 2 * kv4_code_bytes(D) + kv4_param_bytes(D, sizeof(T));
                unsigned hi[NT][G][2], lo[NT][G][2];
                if constexpr (!kWide) {
                    unsigned scale[2][G];
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) scale[x][gr] = KaPair<T>::scales(sw[u][x][gr], unit);
                    if (std::is_same<T, __nv_bfloat16>::value && poisoned) {  // the shift of exponents does not do for a NaN
#pragma unroll
                        for (int x = 0; x < 2; ++x)
#pragma unroll
                            for (int gr = 0; gr < G; ++gr) {
                                const float2 f = KaPair<T>::unpack(sw[u][x][gr]);
                                scale[x][gr] = pack_half(f.x * pow2(134 - unit), f.y * pow2(134 - unit));
                            }
                    }
                    unsigned z[4], za[2];
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[i] = *reinterpret_cast<const unsigned*>(v_params + ((2 * j + (i & 1) + 8 * (i >> 1)) * G + g % G) * 4);
                    za[0] = __byte_perm(z[0], z[1], 0x7632), za[1] = __byte_perm(z[2], z[3], 0x7632);
                    if (edge[u]) {  // nothing behind the row's end, and no NaN, which a weight of 0 would let through: its scale is a NaN too
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            unsigned keep = ka_keep(first[u] + 2 * j + 8 * x, length);
                            if ((za[x] & KaPair<T>::kExponent) == KaPair<T>::kExponent) keep &= 0xffff0000u;
                            if ((za[x] >> 16 & KaPair<T>::kExponent) == KaPair<T>::kExponent) keep &= 0x0000ffffu;
                            za[x] &= keep;
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        weight_sum[nt] += (s[u][nt][0] + s[u][nt][1]) + (s[u][nt][2] + s[u][nt][3]);
                        unsigned ph[2], pl[2];
                        split_half(s[u][nt][0], s[u][nt][1], ph[0], pl[0]);
                        split_half(s[u][nt][2], s[u][nt][3], ph[1], pl[1]);
                        if (std::is_same<T, __nv_bfloat16>::value) {  // operands of one type: the weights once more, as two bf16 (16 bits)
                            unsigned bh[2], bl[2];
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                bh[x] = KaPair<__nv_bfloat16>::pack(s[u][nt][2 * x], s[u][nt][2 * x + 1]);
                                const float2 f = KaPair<__nv_bfloat16>::unpack(bh[x]);
                                bl[x] = KaPair<__nv_bfloat16>::pack(s[u][nt][2 * x] - f.x, s[u][nt][2 * x + 1] - f.y);
                            }
                            ka_mma_params<T>(*reinterpret_cast<float(*)[4]>(zero_sum[nt]), za[0], 0u, za[1], 0u, bl[0], bl[1]);
                            ka_mma_params<T>(*reinterpret_cast<float(*)[4]>(zero_sum[nt]), za[0], 0u, za[1], 0u, bh[0], bh[1]);
                        } else {
                            ka_mma_params<T>(*reinterpret_cast<float(*)[4]>(zero_sum[nt]), za[0], 0u, za[1], 0u, pl[0], pl[1]);
                            ka_mma_params<T>(*reinterpret_cast<float(*)[4]>(zero_sum[nt]), za[0], 0u, za[1], 0u, ph[0], ph[1]);
                        }
                        if (edge[u]) {  // what the column does not see may be a NaN
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const unsigned keep = ka_keep(first[u] + 2 * j + 8 * x, own_limit[nt]);
#pragma unroll
                                for (int gr = 0; gr < G; ++gr) ka_weigh(ph[x], pl[x], scale[x][gr] & keep, hi[nt][gr][x], lo[nt][gr][x]);
                            }
                        } else {
#pragma unroll
                            for (int x = 0; x < 2; ++x)
#pragma unroll
                                for (int gr = 0; gr < G; ++gr) ka_weigh(ph[x], pl[x], scale[x][gr], hi[nt][gr][x], lo[nt][gr][x]);
                        }
                    }
                } else {
                    const float shrink = pow2(127 - unit);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        weight_sum[nt] += (s[u][nt][0] + s[u][nt][1]) + (s[u][nt][2] + s[u][nt][3]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (edge[u] && first[u] + 2 * j + (i & 1) + 8 * (i >> 1) >= own_limit[nt]) {
#pragma unroll
                                for (int gr = 0; gr < G; ++gr) vs[u][i][gr] = vz[u][i][gr] = 0.f;  // NT is 1: no other column of this lane
                            }
#pragma unroll
                            for (int gr = 0; gr < G; ++gr) zero_sum[nt][gr] = fmaf(s[u][nt][i], vz[u][i][gr], zero_sum[nt][gr]);
                            s[u][nt][i] *= shrink;
                        }
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) {
                            split_half(s[u][nt][0] * vs[u][0][gr], s[u][nt][1] * vs[u][1][gr], hi[nt][gr][0], lo[nt][gr][0]);
                            split_half(s[u][nt][2] * vs[u][2][gr], s[u][nt][3] * vs[u][3][gr], hi[nt][gr][1], lo[nt][gr][1]);
                        }
                    }
                }

                // ---- values
                constexpr int kUnit = D / 16;
                unsigned v[4][G];
#pragma unroll
                for (int i = 0; i < 4; ++i) lds_words(codes[u] + kv4_code_bytes(D) + (i * 32 + lane) * kUnit, v[i]);
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    unsigned a[4][4];
#pragma unroll
                    for (int m = 0; m < 4; ++m) {  // rows g and g + 8: channels 8 g + c and 8 g + c + 2, c = 0, 1 (x 16), 4, 5 (x 16)
                        const unsigned pick = m < 2 ? 0x5410u : 0x7632u, mask = m & 1 ? 0x00f000f0u : 0x000f000fu;
                        const unsigned near = __byte_perm(v[0][gr], v[1][gr], pick), far = __byte_perm(v[2][gr], v[3][gr], pick);
                        a[m][0] = near & mask, a[m][1] = near >> 8 & mask, a[m][2] = far & mask, a[m][3] = far >> 8 & mask;
                    }
                    if (sizeof(T) == 4) {  // chains of two, added up in fp32: the tensor core cuts off where an addition rounds
                        float acc[NT][4][4];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int m = 0; m < 4; ++m)
#pragma unroll
                                for (int i = 0; i < 4; ++i) acc[nt][m][i] = 0.f;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int m = 0; m < 4; ++m) ka_mma(acc[nt][m], a[m][0], a[m][1], a[m][2], a[m][3], lo[nt][gr][0], lo[nt][gr][1]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int m = 0; m < 4; ++m) ka_mma(acc[nt][m], a[m][0], a[m][1], a[m][2], a[m][3], hi[nt][gr][0], hi[nt][gr][1]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int m = 0; m < 4; ++m) add_tile(o[nt][gr][m], acc[nt][m]);
                    } else {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int m = 0; m < 4; ++m) ka_mma(o[nt][gr][m], a[m][0], a[m][1], a[m][2], a[m][3], lo[nt][gr][0], lo[nt][gr][1]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int m = 0; m < 4; ++m) ka_mma(o[nt][gr][m], a[m][0], a[m][1], a[m][2], a[m][3], hi[nt][gr][0], hi[nt][gr][1]);
                    }
                }
            }

            __syncwarp();  // every lane has read the stages
            for (int u = 0; u < count; ++u) {
                request(stage);
                if (++stage == C::kStages) stage = 0, ++use;
            }
        }

        // ---- the end of a segment: the warps' sums meet
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            weight_sum[nt] += __shfl_xor_sync(kFullMask, weight_sum[nt], 1);
            weight_sum[nt] += __shfl_xor_sync(kFullMask, weight_sum[nt], 2);
            if constexpr (kWide) {
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    zero_sum[nt][gr] += __shfl_xor_sync(kFullMask, zero_sum[nt][gr], 1);
                    zero_sum[nt][gr] += __shfl_xor_sync(kFullMask, zero_sum[nt][gr], 2);
                }
            }
            if (j == 0) {
                const int c = (warp * NT + nt) * 8 + g;
                s_max[c] = top[nt] * mult[nt];
                s_sum[c] = weight_sum[nt];
            }
        }
        __syncthreads();
        const float grow = ka_unit_value<T>(unit);
        const long long slot = 2ll * blockIdx.x + (segment > begin ? 1 : 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {  // the columns 2 j + c of all warps; a warp then adds one of them up
                float m = -INFINITY;
#pragma unroll
                for (int w = 0; w < kKaWarps; ++w) m = fmaxf(m, s_max[(w * NT + nt) * 8 + 2 * j + c]);
                const float own = s_max[(warp * NT + nt) * 8 + 2 * j + c];
                const float weight = own == -INFINITY ? 0.f : exp2f(own - m);
                // channel 8 g + i of a group at 8 i + g
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    const float zero = kWide ? __shfl_sync(kFullMask, zero_sum[nt][gr % Z], (2 * j + c) * 4) : __shfl_sync(kFullMask, zero_sum[nt][c], gr * 4 + j);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int m4 = (k >> 2) * 2 + (k & 1), half = (k >> 1) & 1;  // channel 8 g + k lies in these registers
                        const float sum = fmaf(o[nt][gr][m4][2 * half + c] * (m4 & 1 ? 0x1p20f : 0x1p24f), grow, zero);
                        s_fold[(warp * 4 + j) * C::kFoldRow + gr * kKv4Group + k * 8 + g] = sum * weight;
                    }
                }
                __syncthreads();
                const int mine = 2 * warp + c, column = (block * NT + nt) * 8 + mine;
                if (column < p.columns) {
                    float most = -INFINITY, sum = 0.f;
#pragma unroll
                    for (int w = 0; w < kKaWarps; ++w) most = fmaxf(most, s_max[(w * NT + nt) * 8 + mine]);
#pragma unroll
                    for (int w = 0; w < kKaWarps; ++w) {
                        const int x = (w * NT + nt) * 8 + mine;
                        sum += s_max[x] == -INFINITY ? s_sum[x] : exp2f(s_max[x] - most) * s_sum[x];  // without a maximum the sum is 0 or NaN
                    }
                    const int token = fdiv(column, p.fd_group), head = kv_head * p.group + column - token * p.group;
                    T* out = static_cast<T*>(p.out) + (((long long)row * p.tokens + token) * p.query_heads + head) * D;
                    float* part = p.partial + slot * ka_slot_floats(D, NT) + (nt * 8 + mine) * (D + 4);
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const int channel = i * 32 + lane, at = channel / kKv4Group * kKv4Group + channel % 8 * 8 + channel % kKv4Group / 8;
                        float value = 0.f;
#pragma unroll
                        for (int w = 0; w < kKaWarps; ++w) value += s_fold[(w * 4 + warp) * C::kFoldRow + at];
                        if (whole) out[channel] = from_float<T>(sum == 0.f ? 0.f : value * inv);
                        else part[channel] = value;
                    }
                    if (!whole && lane < 2) part[D + lane] = lane ? sum : most;
                }
                __syncthreads();
            }
        }
        now.tile = now.tiles - 1;
        ka_advance(p, now, 1);
        segment = segment_end;
    }
    if (dead && lane == 0) {  // copies that are still on the way have to land before the CTA leaves
        for (int i = 0; i < C::kStages && i < requested; ++i) {
            const int last = (requested - 1 - i) / C::kStages;
            const unsigned long long t0 = global_timer_ns();
            while (!mbar_try_wait(&bars[i], last & 1) && global_timer_ns() - t0 <= kWaitLimitNs) {
            }
        }
    }
}

// Joins the partial results of rows that several CTAs worked on; a CTA for each query head, token and 64 channels.  Rows without a token
// get zeros.  A warp takes every eighth partial result, kBatch of them in flight together, with a running maximum of its own.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kKaJoinThreads) kv4_attention_join_kernel(const __grid_constant__ Kv4AttnParams p) {
    constexpr int kWarps = kKaJoinThreads / 32, kBatch = 5;
    __shared__ float2 s_out[kWarps][32];
    __shared__ float s_max[kWarps], s_sum[kWarps];
    __shared__ int s_scan[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = blockIdx.x % (D / 64), output = blockIdx.x / (D / 64);
    const int head = output % p.query_heads, rest = output / p.query_heads;
    const int token = rest % p.tokens, row = rest / p.tokens;
    const int tiles = ka_tiles(p.cache, row);
    T* out = static_cast<T*>(p.out) + (long long)output * D + part * 64;
    if (tiles == 0) {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // no CTA of this grid ends before the grid ahead of it
        if (threadIdx.x < 64) out[threadIdx.x] = from_float<T>(0.f);
        return;
    }
    const int kv_head = fdiv(head, p.fd_group), column = token * p.group + head - kv_head * p.group;
    const int block = column / (8 * NT);
    const int before = ka_line<kKaJoinThreads>(p, row, s_scan), total = ka_line<kKaJoinThreads>(p, p.cache.rows, s_scan);
    const int piece = ka_piece(total, p.ctas);
    const int first = before + (kv_head * p.blocks + block) * tiles;
    const int cta0 = (unsigned)first / (unsigned)piece, cta1 = (unsigned)(first + tiles - 1) / (unsigned)piece;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (cta0 == cta1) return;  // that CTA has written the output
    const float* base = p.partial + (column - block * 8 * NT) * (D + 4);
    float top = -INFINITY, sum = 0.f;
    float2 acc = make_float2(0.f, 0.f);
    for (int c0 = cta0 + warp; c0 <= cta1; c0 += kWarps * kBatch) {
        float2 stats[kBatch], value[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int c = c0 + i * kWarps;
            stats[i] = make_float2(-INFINITY, 0.f);
            value[i] = make_float2(0.f, 0.f);
            if (c <= cta1) {
                const float* x = base + (2ll * c + (first > c * piece ? 1 : 0)) * ka_slot_floats(D, NT);
                stats[i] = __ldcg(reinterpret_cast<const float2*>(x + D));
                value[i] = __ldcg(reinterpret_cast<const float2*>(x + part * 64) + lane);
            }
        }
        float now = top;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) now = fmaxf(now, stats[i].x);
        const float base_now = now == -INFINITY ? 0.f : now, corr = exp2f(top - base_now);
        sum *= corr, acc.x *= corr, acc.y *= corr;
        top = now;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const float own = exp2f(stats[i].x - base_now);
            sum += stats[i].x == -INFINITY ? stats[i].y : own * stats[i].y;  // without a maximum the sum is 0 or NaN
            acc.x = fmaf(own, value[i].x, acc.x), acc.y = fmaf(own, value[i].y, acc.y);
        }
    }
    s_out[warp][lane] = acc;
    if (lane == 0) s_max[warp] = top, s_sum[warp] = sum;
    __syncthreads();
    if (warp != 0) return;
    float all_top = -INFINITY, all = 0.f;
    float2 value = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all_top = fmaxf(all_top, s_max[w]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const float own = s_max[w] == -INFINITY ? 0.f : exp2f(s_max[w] - all_top);
        all += s_max[w] == -INFINITY ? s_sum[w] : own * s_sum[w];
        value.x = fmaf(own, s_out[w][lane].x, value.x), value.y = fmaf(own, s_out[w][lane].y, value.y);
    }
    const float inv = all == 0.f ? 0.f : 1.f / all;
    out[2 * lane] = from_float<T>(all == 0.f ? 0.f : value.x * inv);
    out[2 * lane + 1] = from_float<T>(all == 0.f ? 0.f : value.y * inv);
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
    if ((long long)c->rows * a->tokens > 0x7fffffffLL || (long long)c->rows * a->tokens * a->query_heads > 0x1fffffffLL)
        MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: more than 2^29 - 1 query heads", what);
    const int elem = kv4_elem(c->dtype);
    if (reinterpret_cast<uintptr_t>(a->q) % elem != 0 || reinterpret_cast<uintptr_t>(a->out) % elem != 0)
        MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: q and out must be aligned to their elements", what);
    p->q = a->q;
    p->out = a->out;
    p->q_row = a->q_row, p->q_token = a->q_token, p->q_head = a->q_head;
    p->wide_q = (reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)((a->q_row | a->q_token | a->q_head) * elem)) % 16 == 0;
    p->query_heads = a->query_heads;
    p->tokens = a->tokens;
    p->group = a->query_heads / c->kv_heads;
    p->columns = p->group * a->tokens;
    p->scale = a->scale;
    return MK36_OK;
}

// Two blocks of eight columns a pass where there are more than eight, so that a tile is read and unpacked once for both.  fp32 takes one:
// its queries and weights are held in two halves each, which leaves no registers for a second.
static int ka_blocks_of_eight(const Kv4AttnParams& p, int dtype) { return dtype != MK36_F32 && p.columns > 8 ? 2 : 1; }

static int ka_grid(Kv4AttnParams* p, int dtype, int page_size) {
    const DeviceInfo* info = current_device_info();
    if (!info) return MK36_ERR_LAUNCH;
    const int nt = ka_blocks_of_eight(*p, dtype);
    p->blocks = (p->columns + 8 * nt - 1) / (8 * nt);
    p->streams = p->cache.kv_heads * p->blocks;
    p->fd_blocks = make_fastdiv((unsigned)p->blocks), p->fd_group = make_fastdiv((unsigned)p->group), p->fd_streams = make_fastdiv((unsigned)p->streams);
    const double line = (double)p->cache.rows * p->cache.row_pages * (page_size / kKv4Tile) * p->streams;
    if (line > 2e9) MK36_FAIL(MK36_ERR_UNSUPPORTED, "kv4_attention_decode: the table holds more than 2e9 tiles of 16 tokens, heads and query blocks");
    const long long most = (long long)line;
    const long long ctas = (most + kKaMinTiles - 1) / kKaMinTiles, resident = (long long)info->sm_count * ka_ctas_per_sm(dtype == MK36_F32, nt);
    p->ctas = (int)(ctas < resident ? ctas : resident);
    return MK36_OK;
}

template <typename T, int D, int NT>
static int kv4_attention_launch(const Kv4AttnParams& p, cudaStream_t s) {
    using C = KaConfig<T, D, NT>;
    const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kv4_attention_kernel<T, D, NT>), C::kSmem);
    if (rc != MK36_OK) return rc;
    kv4_attention_kernel<T, D, NT><<<p.ctas, kKaThreads, C::kSmem, s>>>(p);
    MK36_CUDA_OK(cudaGetLastError());
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)((long long)p.cache.rows * p.tokens * p.query_heads * (D / 64)));
    config.blockDim = dim3(kKaJoinThreads);
    config.stream = s;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    MK36_CUDA_OK(cudaLaunchKernelEx(&config, kv4_attention_join_kernel<T, D, NT>, p));
    return MK36_OK;
}

template <typename T>
static int kv4_attention_head_dim(const Kv4AttnParams& p, int d, int nt, cudaStream_t s) {
    if (nt == 2) {
        if (d == 64) return kv4_attention_launch<T, 64, sizeof(T) == 4 ? 1 : 2>(p, s);
        if (d == 128) return kv4_attention_launch<T, 128, sizeof(T) == 4 ? 1 : 2>(p, s);
        return kv4_attention_launch<T, 256, sizeof(T) == 4 ? 1 : 2>(p, s);
    }
    if (d == 64) return kv4_attention_launch<T, 64, 1>(p, s);
    if (d == 128) return kv4_attention_launch<T, 128, 1>(p, s);
    return kv4_attention_launch<T, 256, 1>(p, s);
}

}  // namespace mk36

using namespace mk36;

static size_t ka_workspace(const Kv4AttnParams& p, int d, int nt) { return 2ull * p.ctas * ka_slot_floats(d, nt) * sizeof(float); }

extern "C" size_t mk36_kv4_attention_workspace_bytes(const mk36_kv4_cache* cache, const mk36_kv4_attention_args* args) {
    Kv4AttnParams p{};
    if (kv4_attention_params(cache, args, &p) != MK36_OK || ka_grid(&p, cache->dtype, cache->page_size) != MK36_OK) return 0;
    return ka_workspace(p, cache->head_dim, ka_blocks_of_eight(p, cache->dtype));
}

extern "C" int mk36_kv4_attention_decode(const mk36_kv4_cache* cache, const mk36_kv4_attention_args* args, void* workspace,
                                         size_t workspace_bytes, void* stream) {
    Kv4AttnParams p{};
    int rc = kv4_attention_params(cache, args, &p);
    if (rc != MK36_OK) return rc;
    rc = ka_grid(&p, cache->dtype, cache->page_size);
    if (rc != MK36_OK) return rc;
    const int nt = ka_blocks_of_eight(p, cache->dtype);
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < ka_workspace(p, cache->head_dim, nt))
        MK36_FAIL(MK36_ERR_WORKSPACE, "kv4_attention_decode: workspace of %zu bytes is too small or not 16-byte aligned", workspace_bytes);
    p.partial = static_cast<float*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (cache->dtype) {
        case MK36_BF16: return kv4_attention_head_dim<__nv_bfloat16>(p, cache->head_dim, nt, s);
        case MK36_F16: return kv4_attention_head_dim<__half>(p, cache->head_dim, nt, s);
        default: return kv4_attention_head_dim<float>(p, cache->head_dim, nt, s);
    }
}
