// Attention over the 4-bit paged cache, for the last token or the last few of every row.
//
// Mathematics.  A key entry stands for z + n s with a code n of 4 bits and s, z of its group of 64 channels, a value entry likewise:
//     score_t = sum_groups s_tg (q_g . n_tg) + z_tg sum(q_g)          out_c = sum_t (p_t s'_tg) n'_tc + sum_t p_t z'_tg
// so scales and zero points never touch an element: keys get theirs on the products of a group, values on the weights, and the two sums
// with zero points are small matrix products of their own (tokens x groups by groups x columns; groups x tokens by tokens x columns).
// What is left per element is to turn codes into operands, and there f16 helps: the bits 0x000n are the subnormal n 2^-24, 0x00n0 is
// n 2^-20, so a 32-bit word of eight codes becomes four operand registers with four masks and one shift.  The factor 16 of every
// second register goes into q (keys) or into the result (values).
//   * q is scaled by a power of two so that its largest channel is in [2^14, 2^15): exact for bf16 and f16 values, but for what lies below steps of
//     2^-35 of that channel.  A group whose largest channel is smaller than 2^-12 of it has a power of its own (its keys may be as much larger), and
//     the groups' products are then brought together in fp32.
//   * Weights times scales are formed in fp32 and brought into f16's range by a power of two for each group of channels and each column, chosen
//     by the largest such product so far: not by the largest scale, which may be that of a token without weight, of another group, or of a token
//     that this query does not see.  They are held in two halves (hi + lo, 22 bits, and down to 2^-34 of the largest): a rounded weight's error would be
//     multiplied by a code of 0 .. 15 where the value itself, with its zero point, may be near zero.  (One half: 6 us of 78 less at 48 long
//     rows, and an error of 2^-11 of the codes' size.)
//   * Weights at the zero points are of the operands' type: two halves of f16 (22 bits, and down to 2^-35 of the largest weight) or of bf16 (16 bits; the
//     output has 8, and what lies next to the middle between two neighbours may go to the other one); fp32 multiplies them as they are.
//   * fp32 splits its queries the same way, takes codes less 8, and adds up short chains of products in fp32 (its error against 64 bits
//     is 2e-7 to 5e-7 of the output, that of sums in fp32 throughout 2e-7 to 9e-7).
//
// Work.  Four warps a CTA, three CTAs an SM (heads of 256).  A warp takes a tile (16 tokens of a KV head) on its own: scores as MMAs of 16
// tokens x 16 channels by 8 columns (the query heads and tokens that share the KV head), a transposition of the 16 x 8 scores inside
// the warp, weights relative to a maximum that moves only when it has to, values as MMAs of 16 channels x 16 tokens.  Tiles come through a
// ring of the warp's own, one bulk copy each (a tile is contiguous), so that nothing but the end of a segment needs the other warps.  All
// tiles of all rows and heads form one line that is cut into as many equal pieces as there are CTAs; a piece that ends inside a row
// leaves a partial result, and a second launch, set up while the first still runs, joins those.
//
// What bounds it.  Short rows: latency, 8.9 us for one row of 700 tokens.  Many long rows: not memory (tiles that all lie in L2 take 97 % of
// the time) but the SMs: 642 instructions a tile, half of them masks, shifts and permutations that issue every other cycle, 51 MMAs
// of 8 cycles; issue slots, that pipe, the tensor cores and shared memory are each 40 to 60 % busy, with three warps a scheduler.  48 rows
// of 2000 to 40000 tokens, 16 / 2 heads of 256: 273 MB in 78.1 us, 3.5 TB/s, whatever the size of the values; 24 / 4 heads, three tokens, 12 rows: 43.2 us.
#include <math.h>

#include <type_traits>

#include "mk36_kv4.cuh"
#include "mk36_mma.cuh"
#include "mk36_ring.cuh"

namespace mk36 {

constexpr int kKaWarps = 4;
constexpr int kKaThreads = kKaWarps * 32;
constexpr int kKaMinTiles = kKaWarps;  // fewest tiles of a piece: one a warp (one row of 700 tokens, when it was chosen: 9.6 us; two a warp 12.6, four 14.8)

struct Kv4AttnParams {
    Kv4View cache;
    const void* q;
    void* out;
    float* partial;
    long long q_row, q_token, q_head;
    int query_heads, tokens, group, columns;  // group: query heads of a KV head; columns: group * tokens
    int blocks;                               // of eight columns
    int streams;                              // kv_heads * blocks: passes over a row
    int ctas, wide_q, join_wide;
    float scale;
    FastDiv fd_blocks, fd_group, fd_streams;
};

// Partial results: per (CTA, first or last segment) and column the sums, then maximum (of scores in units of log 2) and sum of weights.
__host__ __device__ constexpr int ka_slot_floats(int d) { return 8 * (d + 4); }

// As many as their registers leave room for without spills (heads of 128 in three: 74 us where four take 69; heads of 256 in four, which
// spill: 110 us where three take 78).
__host__ __device__ constexpr int ka_ctas_per_sm(bool fp32, int d) { return fp32 ? (d == 64 ? 3 : 2) : (d == 256 ? 3 : 4); }

template <typename T, int D>
struct KaConfig {
    static constexpr int kGroups = D / kKv4Group;
    static constexpr int kTile = kv4_tile_bytes(D, sizeof(T));
    static constexpr int kQParts = sizeof(T) == 4 ? 2 : 1;
    static constexpr int kCtas = ka_ctas_per_sm(sizeof(T) == 4, D);
    static constexpr int kFoldRow = D + 8;  // the lanes of a store (g, j), rows j apart, fall into 32 banks
    static constexpr int kFold = kKaWarps * 4 * kFoldRow * 4;
    static constexpr int kOperands = kQParts * kGroups * 4 * 32 * 8;  // of the queries
    static constexpr int kStats = (kKaWarps * 8 * 2 + 8 * kGroups * 3) * 4;
    static constexpr int kRoom = 232448 / kCtas - 1024 - kFold - kOperands - kStats - 512;
    static constexpr int kMost = kRoom / (kKaWarps * kTile);
    static constexpr int kStages = kMost < 8 ? kMost : 8;
    static constexpr int kSmem = kKaWarps * kStages * kTile + kFold + kOperands + kStats + kKaWarps * kStages * 8;
    static_assert(kStages >= 2, "no room for a ring");
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
    static constexpr unsigned kExponent = 0x7f80u;
    static __device__ __forceinline__ unsigned pack(float x, float y) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const unsigned*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(unsigned w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
};
template <>
struct KaPair<__half> {
    static constexpr unsigned kExponent = 0x7c00u;
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

// e of a positive number in [2^e, 2^(e + 1))
__device__ __forceinline__ int exponent_of(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }

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

// Weights are at most 2^(kLift + kLag).  f16 has them in two halves, for the zero points, and needs room below; the others hold them as fp32 and
// as two bf16, and need room above: with weights of at most 1 no sum is larger than the values are.
template <typename T>
constexpr int kLift = std::is_same<T, __half>::value ? 10 : -4;
constexpr int kLag = 4;
constexpr float kNoTop = -3e38f;  // below every score but -infinity, which then has a weight of 0; sums without a maximum are 0 or NaN, and finite factors keep them
constexpr int kMostQ = 100;  // queries larger than 2^100 have products in units of 2^100: the factor to log 2 units stays finite
// Weights times scales of a group: the largest one is brought to 2^9 .. 2^10 and may grow to 2^15 before that is done again, by a power of two of
// at most 2^(120 - kLift - kLag), so that its product with a weight is finite.
constexpr int kAim = 9;
template <typename T>
constexpr int kMostUp = 120 - kLift<T> - kLag;

// A group's scale out of its word of the two-byte types' parameters.
template <typename T>
__device__ __forceinline__ float ka_scale(unsigned w) {
    if constexpr (std::is_same<T, __half>::value) return __low2float(as_half2(w));
    else return __uint_as_float(w << 16);
}

// fp32 takes codes less 8 as whole numbers in f16 (`times`: 1, or 16 for the upper half bytes).  Sums of them are no larger than they need to
// be, so that what the tensor core cuts off stays at the size of fp32's own rounding; subnormals 0 .. 15 are one instruction less.
__device__ __forceinline__ unsigned ka_centred(unsigned code, int times) {
    const unsigned c = times == 1 ? 0x64086408u : 0x64806480u;  // 1024 + 8, 1024 + 128
    return as_word(__hsub2(as_half2(code | 0x64006400u), as_half2(c)));
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
            Kv4Param<typename std::conditional<sizeof(T) == 4, __half, T>::type> one{w[i]};  // fp32 does not come here
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

// All CTAs, and the join, cut the line alike.
__device__ __forceinline__ int ka_piece(int total, int ctas) {
    return max(kKaMinTiles, (int)(((unsigned)total + (unsigned)ctas - 1u) / (unsigned)ctas));
}

// Tiles of the whole line, below 2^31 as the host sees to.  Every thread of a CTA calls it; s: a word for each warp.
template <int kWarps>
__device__ __forceinline__ int ka_line(const Kv4AttnParams& p, int* s) {
    int mine = 0;
    for (int r = threadIdx.x; r < p.cache.rows; r += kWarps * 32) mine += ka_tiles(p.cache, r);
    mine = __reduce_add_sync(kFullMask, mine);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = mine;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += s[w];
    return sum * p.streams;
}

// The piece [begin, end) of the line that belongs to CTA `cta`, and the tile it begins at; false where nothing is left for that CTA.  Every
// thread of a CTA calls it; s: a word for each warp, and three.
template <int kWarps>
__device__ __forceinline__ bool ka_begin(const Kv4AttnParams& p, int cta, int* s, int& piece, int& begin, int& end, KaCursor& start) {
    constexpr int kThreads = kWarps * 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *s_scan = s, *s_start = s + kWarps;
    int all = 0, before = 0;
    if (p.cache.rows > kThreads) {
        all = ka_line<kWarps>(p, s_scan);
        piece = ka_piece(all, p.ctas);
        if ((long long)cta * piece >= all) return false;
    }
    for (int base = 0;; base += kThreads) {  // rows in batches of a thread each
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
        int batch = 0, lower = before;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) lower += s_scan[w];
            batch += s_scan[w];
        }
        if (p.cache.rows <= kThreads) all = batch * p.streams;
        piece = ka_piece(all, p.ctas);
        if ((long long)cta * piece >= all) return false;  // the whole CTA, in its first batch
        begin = cta * piece, end = all - begin < piece ? all : begin + piece;
        // begin's row has first * streams <= begin < (first + n) * streams
        const int target = fdiv(begin, p.fd_streams), first = lower + inc - n;
        if (first <= target && target < first + n) s_start[0] = r, s_start[1] = first, s_start[2] = n;
        before += batch;
        if (before > target || base + kThreads >= p.cache.rows) break;
    }
    __syncthreads();
    start.row = s_start[0];
    start.tiles = s_start[2];
    const int off = begin - s_start[1] * p.streams;
    start.stream = (unsigned)off / (unsigned)start.tiles;
    start.tile = off - start.stream * start.tiles;
    return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(kKaThreads, KaConfig<T, D>::kCtas) kv4_attention_kernel(const __grid_constant__ Kv4AttnParams p) {
    using C = KaConfig<T, D>;
    constexpr int G = C::kGroups, QP = C::kQParts;
    constexpr bool kWide = sizeof(T) == 4;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int s_scan[kKaWarps + 3], s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
    unsigned char* ring = smem + warp * C::kStages * C::kTile;
    float* s_fold = reinterpret_cast<float*>(smem + kKaWarps * C::kStages * C::kTile);
    uint4* s_qf = reinterpret_cast<uint4*>(s_fold + C::kFold / 4);  // [QP][G][2][32]: operand registers of the queries, of two MMAs each
    float* s_max = reinterpret_cast<float*>(s_qf) + C::kOperands / 4;  // [warp][8]
    float* s_sum = s_max + kKaWarps * 8;           // [warp][8]
    float* s_most = s_sum + kKaWarps * 8;          // [G][8]: largest |q|
    float* s_qsum = s_most + G * 8;                // [8][G]
    float* s_qunit = s_qsum + 8 * G;               // [8][G]: unit of a group's products, where they have units of their own
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(s_qunit + 8 * G) + warp * C::kStages;
    if (lane == 0) {
        for (int i = 0; i < C::kStages; ++i) mbar_init(&bars[i], 1);
        mbar_init_fence();
    }
    if (threadIdx.x == 0) s_abort = 0;
    asm volatile("griddepcontrol.launch_dependents;");  // the join may be set up while this runs; it waits for the end of the grid

    int begin, end;
    KaCursor start;
    {
        int piece;
        if (!ka_begin<kKaWarps>(p, blockIdx.x, s_scan, piece, begin, end, start)) return;
    }

    // A warp prepares one group of 64 channels of every column's query (lane: column g, channels 16 j .. + 15).  They are requested a
    // segment ahead.
    Chunk8<T> q_raw[2];
    auto request_queries = [&](const KaCursor& c) {
        const int kv_head = fdiv(c.stream, p.fd_blocks), block = c.stream - kv_head * p.blocks;
        const int column = block * 8 + g, token = fdiv(column, p.fd_group);
        zero_chunk8<T>(q_raw[0]);
        zero_chunk8<T>(q_raw[1]);
        if (warp < G && column < p.columns) {
            const T* src = static_cast<const T*>(p.q) + c.row * p.q_row + token * p.q_token + (kv_head * p.group + column - token * p.group) * p.q_head +
                           warp * kKv4Group + 16 * j;
            if (p.wide_q) {
                q_raw[0] = load_chunk8<T>(src);
                q_raw[1] = load_chunk8<T>(src + 8);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) reinterpret_cast<T*>(&q_raw[i >> 3])[i & 7] = src[i];
            }
        }
    };
    request_queries(start);

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
    auto request = [&](int stage) {
        if (begin + warp + requested * kKaWarps >= end) return;
        if (requested % 32 == 0) {
            if (requested > 0) src_now = src_next;
            src_next = look_up();
        }
        const unsigned char* src = reinterpret_cast<const unsigned char*>(__shfl_sync(kFullMask, reinterpret_cast<unsigned long long>(src_now), requested % 32));
        if (src) {
            if (lane == 0) {
                mbar_arrive_expect_tx(&bars[stage], C::kTile);
                bulk_copy_g2s(ring + stage * C::kTile, src, C::kTile, &bars[stage]);
            }
        } else {  // a tile of NaN: it reaches the queries that see it, like any other
            for (int i = lane; i < C::kTile / 16; i += 32) reinterpret_cast<uint4*>(ring + stage * C::kTile)[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the stage's next copy
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[stage]);
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

        // ---- the queries of this pass: the operand registers stay in shared memory, where every tile takes them from
        float mult;                     // factor of column g's scores, in units of log 2
        float q_sum[2][kWide ? G : 1];  // fp32: sums over the groups' channels of columns 2 j, 2 j + 1
        unsigned q_zero[2];             // two-byte types: the sums of column g as operand registers, against the zero points
        bool apart = false;             // groups' products have units of their own: of a column, their largest channels are far apart, or it is very large
        int limit[2], own_limit;        // positions that the columns 2 j, 2 j + 1 see, and column g
        {
            float q[16];
            const int column = block * 8 + g, token = fdiv(column, p.fd_group);
            own_limit = min(length, length - p.tokens + 1 + token);
            float f[2][8], most = 0.f;
            unpack8(q_raw[0], f[0]);
            unpack8(q_raw[1], f[1]);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                q[i] = f[i >> 3][i & 7];
                most = fmaxf(most, fabsf(q[i]));
            }
            most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 1));
            most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 2));
            if (warp < G && j == 0) s_most[warp * 8 + g] = most;
            __syncthreads();
            most = 0.f;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) most = fmaxf(most, s_most[gr * 8 + g]);
            // The unit of the column's products: such that the groups' own units are within 2^-126 .. 2^127 of it.
            const int all = ka_exponent(most);
            int unit = all, column_unit = min(all, kMostQ);
#pragma unroll
            for (int gr = 0; G > 1 && gr < G; ++gr) {
                const float own = s_most[gr * 8 + g];
                if (own > 0.f && own < 0x1p-12f * most) {
                    column_unit = min(column_unit, ka_exponent(own) + 126);
                    if (gr == warp) unit = ka_exponent(own);
                }
            }
            if (warp < G) {
                const float up = copysignf(pow2(14 - unit), p.scale);  // the scale's sign goes into q
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    q[i] *= up;
                    sum += q[i];
                }
                sum += __shfl_xor_sync(kFullMask, sum, 1);
                sum += __shfl_xor_sync(kFullMask, sum, 2);
                if (j == 0) {
                    s_qsum[g * G + warp] = sum * pow2(-24);
                    s_qunit[g * G + warp] = pow2(unit - column_unit);
                }
#pragma unroll
                for (int w = 0; w < 2; ++w) {  // MMA m takes the codes 2 (m % 2), + 1, + 4, + 5 of word m / 2
                    const float* x = &q[8 * w];
                    uint4 hi, lo;
                    split_half(x[0], x[4], hi.x, lo.x);
                    split_half(x[1] * 0.0625f, x[5] * 0.0625f, hi.y, lo.y);
                    split_half(x[2], x[6], hi.z, lo.z);
                    split_half(x[3] * 0.0625f, x[7] * 0.0625f, hi.w, lo.w);
                    s_qf[(warp * 2 + w) * 32 + lane] = hi;
                    if (QP == 2) s_qf[(((QP - 1) * G + warp) * 2 + w) * 32 + lane] = lo;
                }
            }
            __syncthreads();
            // not 0, so that a score of -infinity stays one, but as near as can be, so that any other score times a scale of 0 is
            mult = fmaxf(ldexpf(fabsf(p.scale) * 1.4426950408889634f, 24 - 14 + column_unit), __uint_as_float(1u));
#pragma unroll
            for (int gr = 0; gr < G; ++gr) apart |= s_qunit[g * G + gr] != 1.f;
            apart = __any_sync(kFullMask, apart);  // in all warps alike: each looks at all columns
            // what belongs to a column, for the lanes that hold it in the products' layout: columns 2 j, 2 j + 1
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                limit[c] = __shfl_sync(kFullMask, own_limit, (2 * j + c) * 4);
                if constexpr (kWide) {
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) q_sum[c][gr] = s_qsum[(2 * j + c) * G + gr];
                }
            }
            if constexpr (!kWide) {
                // k = 0..3 and 4..7 (and 8..15 for bf16): the sums of the groups, in two parts (four) that add up to 22 bits (32)
                float x[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) x[i] = 2 * (j & 1) + i < G ? s_qsum[g * G + (2 * (j & 1) + i) % G] : 0.f;
                if (std::is_same<T, __half>::value) x[0] *= pow2(16), x[1] *= pow2(16);  // room for f16's second part; taken back below
                unsigned part[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    part[i] = KaPair<T>::pack(x[0], x[1]);
                    const float2 f = KaPair<T>::unpack(part[i]);
                    x[0] -= f.x, x[1] -= f.y;
                }
                const bool second = j >> 1;
                q_zero[0] = second ? part[1] : part[0];
                q_zero[1] = std::is_same<T, __half>::value ? 0u : (second ? part[3] : part[2]);
            }
        }
        int sees_all = min(limit[0], limit[1]);  // every column sees the positions below this
        sees_all = min(sees_all, __shfl_xor_sync(kFullMask, sees_all, 1));
        sees_all = min(sees_all, __shfl_xor_sync(kFullMask, sees_all, 2));

        // zero_sum: the zero points' part, of column g for every group (fp32), or as an MMA leaves it: row g % 4 (the group), columns 2 j, 2 j + 1
        constexpr int Z = kWide ? G : 4;
        // top: the score that weights are relative to, no further than kLag below the maximum; up: the power of two of weights times scales, of column g
        float o[G][4][4], zero_sum[Z], up[G], top = kNoTop, weight_sum = 0.f;
#pragma unroll
        for (int i = 0; i < Z; ++i) zero_sum[i] = 0.f;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            up[gr] = pow2(kMostUp<T>);
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[gr][m][i] = 0.f;
        }
        // Brings the sums of the codes down by a factor for each group, of column g.
        auto bring_down = [&](const float (&by)[G]) {
            bool some = false;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) some |= by[gr] != 1.f;
            if (!__any_sync(kFullMask, some)) return;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                const float c0 = __shfl_sync(kFullMask, by[gr], 8 * j), c1 = __shfl_sync(kFullMask, by[gr], 8 * j + 4);
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    o[gr][m][0] *= c0, o[gr][m][1] *= c1;
                    o[gr][m][2] *= c0, o[gr][m][3] *= c1;
                }
            }
        };

        bool fresh = true;  // no tile has been summed yet
        for (; at < segment_end; at += kKaWarps) {
            if (!dead && !mbar_wait(&bars[stage], use & 1, &s_abort)) dead = true;
            dead = __any_sync(kFullMask, dead);
            if (dead) {
                weight_sum = __uint_as_float(0x7fc00000u);
                continue;
            }
            const unsigned char *codes = ring + stage * C::kTile, *params = codes + 2 * kv4_code_bytes(D), *v_params = params + kv4_param_bytes(D, sizeof(T));
            const int first = (now.tile + (at - segment)) * kKv4Tile;

            // ---- scores
            float s[4] = {0.f, 0.f, 0.f, 0.f};
            constexpr int kKeyUnit = D >= 128 ? 16 : 8, kVecs = D / 8 / kKeyUnit, kWords = kKeyUnit / 4;
            unsigned keys[kVecs][kWords], keys8[kVecs][kWords];  // tokens g and g + 8
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                lds_words(codes + (v * 32 + lane) * kKeyUnit, keys[v]);
                lds_words(codes + ((kVecs + v) * 32 + lane) * kKeyUnit, keys8[v]);
            }
            float ks[2][G], kz[2][G];
            load_params<T, G>(params + g * (G * 2 * (int)sizeof(T)), ks[0], kz[0]);
            load_params<T, G>(params + (g + 8) * (G * 2 * (int)sizeof(T)), ks[1], kz[1]);
            if constexpr (!kWide) {  // zero points times sums of the queries: one MMA, tokens x groups by groups x columns
                unsigned z[2][G > 1 ? 2 : 1];  // of tokens g and g + 8: groups 2 (j % 2) and the next
                lds_words(params + (g * G + (2 * (j & 1)) % G) * 4, z[0]);
                lds_words(params + ((g + 8) * G + (2 * (j & 1)) % G) * 4, z[1]);
                const unsigned a0 = __byte_perm(z[0][0], z[0][G > 1 ? 1 : 0], 0x7632), a1 = __byte_perm(z[1][0], z[1][G > 1 ? 1 : 0], 0x7632);
                ka_mma_params<T>(s, a0, a1, a0, a1, q_zero[0], q_zero[1]);
                if (std::is_same<T, __half>::value) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[i] *= pow2(-16);
                }
            }
            float acc[G][4];
#pragma unroll
            for (int gr = 0; gr < G; ++gr)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[gr][i] = 0.f;
#pragma unroll
            for (int w = 0; w < 2; ++w) {  // the groups' chains side by side: an MMA does not wait for the one before it
                uint4 b[QP][G];
#pragma unroll
                for (int part = 0; part < QP; ++part)
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) b[part][gr] = s_qf[((part * G + gr) * 2 + w) * 32 + lane];
#pragma unroll
                for (int m = 0; m < 2; ++m) {
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        const int v = gr / (kWords / 2), x = 2 * (gr % (kWords / 2)) + w;
                        const unsigned wa = keys[v][x] >> (8 * m), wb = keys8[v][x] >> (8 * m);
                        const unsigned a0 = wa & 0x000f000fu, a1 = wb & 0x000f000fu, a2 = wa & 0x00f000f0u, a3 = wb & 0x00f000f0u;
                        if constexpr (kWide) {
                            const unsigned c0 = ka_centred(a0, 1), c1 = ka_centred(a1, 1), c2 = ka_centred(a2, 16), c3 = ka_centred(a3, 16);
                            float sum[4] = {0.f, 0.f, 0.f, 0.f};
                            ka_mma(sum, c0, c1, c2, c3, m ? b[1][gr].z : b[1][gr].x, m ? b[1][gr].w : b[1][gr].y);
                            ka_mma(sum, c0, c1, c2, c3, m ? b[0][gr].z : b[0][gr].x, m ? b[0][gr].w : b[0][gr].y);
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[gr][i] = fmaf(sum[i], 0x1p-24f, acc[gr][i]);  // room for scales of any size
                        } else {
                            ka_mma(acc[gr], a0, a1, a2, a3, m ? b[0][gr].z : b[0][gr].x, m ? b[0][gr].w : b[0][gr].y);
                        }
                    }
                }
            }
            if (apart) {  // zero points in fp32 too
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float* unit = &s_qunit[(2 * j + (i & 1)) * G];
                    const float* sum = &s_qsum[(2 * j + (i & 1)) * G];
                    s[i] = 0.f;
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        s[i] = fmaf((kWide ? fmaf(8.f, ks[i >> 1][gr], kz[i >> 1][gr]) : kz[i >> 1][gr]) * unit[gr], sum[gr], s[i]);
                        s[i] = fmaf(ks[i >> 1][gr] * unit[gr], acc[gr][i], s[i]);
                    }
                }
            } else {
#pragma unroll
                for (int gr = 0; gr < G; ++gr)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (kWide) s[i] = fmaf(fmaf(8.f, ks[i >> 1][gr], kz[i >> 1][gr]), q_sum[i & 1][gr], s[i]);
                        s[i] = fmaf(ks[i >> 1][gr], acc[gr][i], s[i]);
                    }
            }
            const bool edge = first + kKv4Tile > sees_all;
            if (edge) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (first + g + 8 * (i >> 1) >= limit[i & 1]) s[i] = -INFINITY;
            }
            // from (tokens g, g + 8; columns 2 j, 2 j + 1) to (tokens 2 j, 2 j + 1, + 8, + 9; column g)
            transpose8(s[0], s[1]);
            transpose8(s[2], s[3]);

            // ---- maximum.  `top` follows it only when it is 2^kLag times larger: then, and not with every tile, what has been summed is brought
            // to the new one.  Differences of scores come first: they are exact where they matter, for scores of any size.
            float most = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
            if (__any_sync(kFullMask, (most - top) * mult > (float)kLag)) {
                most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 1));
                most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 2));
                const float next = fmaxf(top, most), drop = (next - top) * mult;
                top = next;
                if (!fresh) {
                    const float corr = exp2f(-drop);
                    weight_sum *= corr;
                    if constexpr (kWide) {
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) zero_sum[gr] *= corr;
                    } else {
                        zero_sum[0] *= __shfl_sync(kFullMask, corr, 8 * j), zero_sum[1] *= __shfl_sync(kFullMask, corr, 8 * j + 4);
                    }
                    // weights get smaller, and `up` grows by as much as far as it goes and in whole powers of two; the rest is the sums'
                    const int by = (int)fminf(drop, 1000.f);
                    const float part = exp2f((float)by - drop);
                    float rest[G];
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        const int e = exponent_of(up[gr]), n = min(e + by, kMostUp<T>);
                        up[gr] = pow2(n);
                        rest[gr] = pow2(max(n - e - by, -126)) * part;
                    }
                    bring_down(rest);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const f32x2 x = fma_pair(add_pair(pair_of(s[i], s[i + 1]), pair_of(-top, -top)), pair_of(mult, mult), pair_of((float)kLift<T>, (float)kLift<T>));
                s[i] = kWide ? exp2f(first_of(x)) : exp2_approx(first_of(x)), s[i + 1] = kWide ? exp2f(second_of(x)) : exp2_approx(second_of(x));
            }
            weight_sum += (s[0] + s[1]) + (s[2] + s[3]);

            // ---- scales of the values of the lane's four tokens; what the column does not see may be anything, a NaN too
            unsigned vw[4][kWide ? 1 : G];
            float vs[4][kWide ? G : 1], vz[4][kWide ? G : 1];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 2 * j + (i & 1) + 8 * (i >> 1);
                if constexpr (kWide) load_params<T, G>(v_params + t * (G * 8), vs[i], vz[i]);
                else lds_words(v_params + t * (G * 4), vw[i]);
            }
            if (edge) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (first + 2 * j + (i & 1) + 8 * (i >> 1) >= own_limit) {
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) {
                            if constexpr (kWide) vs[i][gr] = vz[i][gr] = 0.f;
                            else vw[i][gr] = 0u;
                        }
                    }
            }
            auto scale_of = [&](int i, int gr) {
                if constexpr (kWide) return vs[i][gr];
                else return ka_scale<T>(vw[i][gr]);
            };

            // ---- weights times scales, in two halves.  They are what has to lie in f16's range, whatever weights and scales are by themselves: in
            // units of their own for each group and column.  Where one goes beyond, the units are chosen again.
            unsigned hi[G][2], lo[G][2];
#pragma unroll 1
            for (int turn = 0;; ++turn) {
                __half2 largest = __float2half2_rn(0.f);
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const f32x2 weights = mul_pair(pair_of(s[2 * x], s[2 * x + 1]), pair_of(up[gr], up[gr]));
                        const f32x2 both = mul_pair(weights, pair_of(scale_of(2 * x, gr), scale_of(2 * x + 1, gr)));
                        split_half(first_of(both), second_of(both), hi[gr][x], lo[gr][x]);
                        largest = __hmax2(largest, __habs2(as_half2(hi[gr][x])));
                    }
                }
                const bool fits = __hbleu2(largest, __float2half2_rn(32768.f));
                if (turn == 1 || __all_sync(kFullMask, fits)) break;
                float by[G];
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    float m = 0.f;  // 2^-20 of the largest, which is finite
#pragma unroll
                    for (int i = 0; i < 4; ++i) m = fmaxf(m, fabsf(s[i] * 0x1p-20f * scale_of(i, gr)));
                    m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 1));
                    m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 2));
                    const int e = exponent_of(up[gr]), size = exponent_of(m) + 20;
                    const int n = m == 0.f ? e : max(min(e, kAim - size), -126);
                    up[gr] = pow2(n);
                    by[gr] = pow2(max(n - e, -126));
                }
                if (!fresh) bring_down(by);
            }
            fresh = false;

            // ---- the zero points' part
            if constexpr (kWide) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) zero_sum[gr] = fmaf(s[i], fmaf(8.f, vs[i][gr], vz[i][gr]), zero_sum[gr]);
            } else {
                unsigned z[4], za[2];
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = *reinterpret_cast<const unsigned*>(v_params + ((2 * j + (i & 1) + 8 * (i >> 1)) * G + g % G) * 4);
                za[0] = __byte_perm(z[0], z[1], 0x7632), za[1] = __byte_perm(z[2], z[3], 0x7632);
                if (edge) {  // nothing behind the row's end, and no NaN, which a weight of 0 would let through: its scale is a NaN too
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        unsigned keep = ka_keep(first + 2 * j + 8 * x, length);
                        if ((za[x] & KaPair<T>::kExponent) == KaPair<T>::kExponent) keep &= 0xffff0000u;
                        if ((za[x] >> 16 & KaPair<T>::kExponent) == KaPair<T>::kExponent) keep &= 0x0000ffffu;
                        za[x] &= keep;
                    }
                }
                unsigned ph[2], pl[2];  // operands of one type: two halves of f16 (22 bits) or two of bf16 (16 bits)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                        ph[x] = KaPair<T>::pack(s[2 * x], s[2 * x + 1]);
                        const float2 f = KaPair<T>::unpack(ph[x]);
                        pl[x] = KaPair<T>::pack(s[2 * x] - f.x, s[2 * x + 1] - f.y);
                    } else {
                        split_half(s[2 * x], s[2 * x + 1], ph[x], pl[x]);
                    }
                }
                ka_mma_params<T>(zero_sum, za[0], 0u, za[1], 0u, pl[0], pl[1]);
                ka_mma_params<T>(zero_sum, za[0], 0u, za[1], 0u, ph[0], ph[1]);
            }

            // ---- values
            unsigned v[4][G];
#pragma unroll
            for (int i = 0; i < 4; ++i) lds_words(codes + kv4_code_bytes(D) + (i * 32 + lane) * (D / 16), v[i]);
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                unsigned a[4][4];
#pragma unroll
                for (int m = 0; m < 4; ++m) {  // rows g and g + 8: channels 8 g + c and 8 g + c + 2, c = 0, 1 (x 16), 4, 5 (x 16)
                    const unsigned pick = m < 2 ? 0x5410u : 0x7632u, mask = m & 1 ? 0x00f000f0u : 0x000f000fu;
                    const unsigned near = __byte_perm(v[0][gr], v[1][gr], pick), far = __byte_perm(v[2][gr], v[3][gr], pick);
                    a[m][0] = near & mask, a[m][1] = near >> 8 & mask, a[m][2] = far & mask, a[m][3] = far >> 8 & mask;
                    if constexpr (kWide) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) a[m][i] = ka_centred(a[m][i], m & 1 ? 16 : 1);
                    }
                }
                if (sizeof(T) == 4) {  // chains of two, added up in fp32: the tensor core cuts off where an addition rounds
                    float acc[4][4];
#pragma unroll
                    for (int m = 0; m < 4; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[m][i] = 0.f;
#pragma unroll
                    for (int m = 0; m < 4; ++m) ka_mma(acc[m], a[m][0], a[m][1], a[m][2], a[m][3], lo[gr][0], lo[gr][1]);
#pragma unroll
                    for (int m = 0; m < 4; ++m) ka_mma(acc[m], a[m][0], a[m][1], a[m][2], a[m][3], hi[gr][0], hi[gr][1]);
#pragma unroll
                    for (int m = 0; m < 4; ++m) add_tile(o[gr][m], acc[m]);
                } else {
#pragma unroll
                    for (int m = 0; m < 4; ++m) ka_mma(o[gr][m], a[m][0], a[m][1], a[m][2], a[m][3], lo[gr][0], lo[gr][1]);
#pragma unroll
                    for (int m = 0; m < 4; ++m) ka_mma(o[gr][m], a[m][0], a[m][1], a[m][2], a[m][3], hi[gr][0], hi[gr][1]);
                }
            }

            __syncwarp();  // every lane has read the stage
            request(stage);
            if (++stage == C::kStages) stage = 0, ++use;
        }

        KaCursor next = now;
        next.tile = next.tiles - 1;
        if (segment_end < end) {
            ka_advance(p, next, 1);
            request_queries(next);
        }

        // ---- the end of a segment: the warps' sums meet
        weight_sum += __shfl_xor_sync(kFullMask, weight_sum, 1);
        weight_sum += __shfl_xor_sync(kFullMask, weight_sum, 2);
        if constexpr (kWide) {
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                zero_sum[gr] += __shfl_xor_sync(kFullMask, zero_sum[gr], 1);
                zero_sum[gr] += __shfl_xor_sync(kFullMask, zero_sum[gr], 2);
            }
        }
        if (j == 0) {
            const int c = warp * 8 + g;
            s_max[c] = fminf(fmaxf(top * mult, kNoTop), -kNoTop);
            s_sum[c] = weight_sum;
        }
        __syncthreads();
        const long long slot = 2ll * blockIdx.x + (segment > begin ? 1 : 0);
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // the columns 2 j + c of all warps; a warp then adds one of them up
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < kKaWarps; ++w) m = fmaxf(m, s_max[w * 8 + 2 * j + c]);
            const float own = s_max[warp * 8 + 2 * j + c];
            const float weight = exp2f(own - m);
            // channel 8 g + i of a group at 8 i + g
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                const float back = __uint_as_float(0x7f000000u - __float_as_uint(__shfl_sync(kFullMask, up[gr], (2 * j + c) * 4)));  // 1 / up
                const float zero = kWide ? __shfl_sync(kFullMask, zero_sum[gr % Z], (2 * j + c) * 4) : __shfl_sync(kFullMask, zero_sum[c], gr * 4 + j);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int m4 = (k >> 2) * 2 + (k & 1), half = (k >> 1) & 1;  // channel 8 g + k lies in these registers
                    const float sum = fmaf(o[gr][m4][2 * half + c] * ((m4 & 1 ? 0.0625f : 1.f) * (kWide ? 1.f : 0x1p24f)), back, zero);
                    s_fold[(warp * 4 + j) * C::kFoldRow + gr * kKv4Group + k * 8 + g] = sum * weight;
                }
            }
            __syncthreads();
            const int mine = 2 * warp + c, column = block * 8 + mine;
            if (column < p.columns) {
                float most = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < kKaWarps; ++w) most = fmaxf(most, s_max[w * 8 + mine]);
#pragma unroll
                for (int w = 0; w < kKaWarps; ++w) {
                    const int x = w * 8 + mine;
                    sum += exp2f(s_max[x] - most) * s_sum[x];
                }
                const int token = fdiv(column, p.fd_group), head = kv_head * p.group + column - token * p.group;
                T* out = static_cast<T*>(p.out) + (((long long)row * p.tokens + token) * p.query_heads + head) * D;
                float* part = p.partial + slot * ka_slot_floats(D) + mine * (D + 4);
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
        now = next;
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

// Adds partial results (maximum and sum of weights; sums of two channels) to what a warp has so far.
template <int N>
__device__ __forceinline__ void ka_join(const float2 (&stats)[N], const float2 (&value)[N], float& top, float& sum, float2& acc) {
    float now = top;
#pragma unroll
    for (int i = 0; i < N; ++i) now = fmaxf(now, stats[i].x);
    const float base = now == -INFINITY ? 0.f : now, corr = exp2f(top - base);
    sum *= corr, acc.x *= corr, acc.y *= corr;
    top = now;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float own = exp2f(stats[i].x - base);
        sum = fmaf(own, stats[i].y, sum);
        acc.x = fmaf(own, value[i].x, acc.x), acc.y = fmaf(own, value[i].y, acc.y);
    }
}

// The same for the partial results of the CTAs c0, c0 + step, ... up to cta1: kBatch of them, all requested at once.
template <int kBatch, int D>
__device__ __forceinline__ void ka_join_batch(const float* values, const float* both, int first, int piece, int c0, int step, int cta1, int lane,
                                              float& top, float& sum, float2& acc) {
    float2 stats[kBatch], value[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        const int c = min(c0 + i * step, cta1);  // loads without a branch; one too many counts for nothing
        const long long slot = (2ll * c + (first > c * piece ? 1 : 0)) * ka_slot_floats(D);
        stats[i] = __ldcg(reinterpret_cast<const float2*>(both + slot));
        value[i] = __ldcg(reinterpret_cast<const float2*>(values + slot) + lane);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (c0 + i * step > cta1) stats[i] = make_float2(-INFINITY, 0.f), value[i] = make_float2(0.f, 0.f);
    ka_join<kBatch>(stats, value, top, sum, acc);
}

// Joins the partial results of passes that several CTAs worked on; rows without a token get zeros.  Two forms, as ka_grid chooses: few
// passes, cut into very many pieces, or any others.
//
// Few passes: a CTA of 32 warps takes 64 channels of one query head and token.  A warp takes every 32nd partial result, kBatch of them in
// flight together, with a running maximum of its own: a round trip for a batch is 2 to 3 us (one row of 32768 tokens, 16 / 2 heads of 256,
// 205 partial results for each: 15.9 us for the call with the cache in L2, 19.8 with the other form; one of 700 tokens 8.0 and 8.5).
constexpr int kKaWideWarps = 32;

template <typename T, int D>
__global__ void __launch_bounds__(kKaWideWarps * 32) kv4_attention_join_wide_kernel(const __grid_constant__ Kv4AttnParams p) {
    constexpr int kBatch = 4, kParts = D / 64;  // 4: with 3, 32 registers, two CTAs crowd on an SM (18.8 us instead of 16.7)
    __shared__ float2 s_out[kKaWideWarps][32];
    __shared__ float s_max[kKaWideWarps], s_sum[kKaWideWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int output = blockIdx.x / kParts, part = blockIdx.x % kParts;
    const int head = output % p.query_heads, rest = output / p.query_heads;
    const int token = rest % p.tokens, row = rest / p.tokens;
    T* out = static_cast<T*>(p.out) + (long long)output * D + part * 64;
    int mine = 0, mine_before = 0;  // tiles of all rows, and of those before this one; every warp sums them up
    for (int r = lane; r < p.cache.rows; r += 32) {
        const int n = ka_tiles(p.cache, r);
        mine += n;
        mine_before += r < row ? n : 0;
    }
    const int tiles = ka_tiles(p.cache, row);
    const int total = __reduce_add_sync(kFullMask, mine) * p.streams, before = __reduce_add_sync(kFullMask, mine_before) * p.streams;
    const int kv_head = fdiv(head, p.fd_group), column = token * p.group + head - kv_head * p.group;
    const int block = column / 8;
    const int piece = ka_piece(total, p.ctas);
    const int first = before + (kv_head * p.blocks + block) * tiles;
    const int cta0 = (unsigned)first / (unsigned)piece, cta1 = (unsigned)(first + max(tiles, 1) - 1) / (unsigned)piece;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // no CTA of this grid ends before the grid ahead of it
    if (tiles == 0) {
        if (warp == 0) out[2 * lane] = out[2 * lane + 1] = from_float<T>(0.f);
        return;
    }
    if (cta0 == cta1) return;  // that CTA has written the output
    const float* base = p.partial + (column - block * 8) * (D + 4);
    float top = -INFINITY, sum = 0.f;
    float2 acc = make_float2(0.f, 0.f);
    for (int c0 = cta0 + warp; c0 <= cta1; c0 += kKaWideWarps * kBatch)
        ka_join_batch<kBatch, D>(base + part * 64, base + D, first, piece, c0, kKaWideWarps, cta1, lane, top, sum, acc);
    s_out[warp][lane] = acc;
    if (lane == 0) s_max[warp] = top, s_sum[warp] = sum;
    __syncthreads();
    if (warp != 0) return;
    const float peer_max = s_max[lane], peer_sum = s_sum[lane];  // each lane looks at one of the warps
    const float all_top = warp_max(peer_max);
    const float peer_own = peer_max == -INFINITY ? 0.f : exp2f(peer_max - all_top);
    const float all = warp_sum(peer_max == -INFINITY ? peer_sum : peer_own * peer_sum);
    float2 value = make_float2(0.f, 0.f);
#pragma unroll 8
    for (int i = 0; i < kKaWideWarps; ++i) {
        const float own = __shfl_sync(kFullMask, peer_own, i);
        const float2 x = s_out[i][lane];
        value.x = fmaf(own, x.x, value.x), value.y = fmaf(own, x.y, value.y);
    }
    const float inv = all == 0.f ? 0.f : 1.f / all;
    out[2 * lane] = from_float<T>(all == 0.f ? 0.f : value.x * inv);
    out[2 * lane + 1] = from_float<T>(all == 0.f ? 0.f : value.y * inv);
}

// Any others: a CTA for each cut of the line, and those of one pass share its eight columns and their groups of 64 channels.  Passes that
// are whole cost nothing (a CTA of a few warps for each query head took 35 us where this takes 24: 256 rows of 500 tokens, 16 / 2 heads of
// 128; 57 and 23 for 1024 rows of 7; but 46.8 and 47.6 for eight rows of 32768, and 42.9 and 43.2 for 12 rows of 27B heads with three tokens).  With eight partial results in flight for a warp, not three, 74 registers leave room for three CTAs an SM: 30 us.
constexpr int kKaJoinWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kKaJoinWarps * 32) kv4_attention_join_cuts_kernel(const __grid_constant__ Kv4AttnParams p) {
    constexpr int kBatch = 3, kParts = D / 64, kItems = 8 * kParts;
    __shared__ float2 s_out[kKaJoinWarps][32];
    __shared__ float s_max[kKaJoinWarps], s_sum[kKaJoinWarps];
    __shared__ int s_scan[kKaJoinWarps + 3];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int piece, begin, end;
    KaCursor start;
    const bool cut = ka_begin<kKaJoinWarps>(p, blockIdx.x, s_scan, piece, begin, end, start) && start.tile > 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // no CTA of this grid ends before the grid ahead of it
    for (int row = blockIdx.x; row < p.cache.rows; row += gridDim.x) {
        if (ka_tiles(p.cache, row) != 0) continue;
        const long long n = (long long)p.tokens * p.query_heads * D;
        T* out = static_cast<T*>(p.out) + row * n;
        for (long long i = threadIdx.x; i < n; i += kKaJoinWarps * 32) out[i] = from_float<T>(0.f);
    }
    if (!cut) return;
    const int first = begin - start.tile, cta0 = (unsigned)first / (unsigned)piece, cta1 = (unsigned)(first + start.tiles - 1) / (unsigned)piece;
    const int share = min(1 << (31 - __clz(cta1 - cta0)), kItems);  // CTAs that work on the segment
    const int index = blockIdx.x - cta0 - 1;
    if (index >= share) return;
    const int items = kItems / share, turns = max(kKaJoinWarps / items, 1), turn = warp % turns;
    const int kv_head = fdiv(start.stream, p.fd_blocks), block = start.stream - kv_head * p.blocks;
    for (int i = warp / turns; i < items; i += kKaJoinWarps / turns) {  // more than once only where turns is 1
        const int item = index * items + i, mine = item / kParts, part = item % kParts, column = block * 8 + mine;
        const float* base = p.partial + mine * (D + 4);
        float top = -INFINITY, sum = 0.f;
        float2 acc = make_float2(0.f, 0.f);
        for (int c0 = cta0 + turn; c0 <= cta1 && column < p.columns; c0 += turns * kBatch)
            ka_join_batch<kBatch, D>(base + part * 64, base + D, first, piece, c0, turns, cta1, lane, top, sum, acc);
        if (turns > 1) {
            s_out[warp][lane] = acc;
            if (lane == 0) s_max[warp] = top, s_sum[warp] = sum;
            __syncthreads();
            if (turn == 0) {
                float2 stats[1], value[1];
                for (int w = warp + 1; w < warp + turns; ++w) {
                    stats[0] = make_float2(s_max[w], s_sum[w]), value[0] = s_out[w][lane];
                    ka_join<1>(stats, value, top, sum, acc);
                }
            }
        }
        if (turn == 0 && column < p.columns) {
            const int token = fdiv(column, p.fd_group), head = kv_head * p.group + column - token * p.group;
            T* out = static_cast<T*>(p.out) + (((long long)start.row * p.tokens + token) * p.query_heads + head) * D + part * 64;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            out[2 * lane] = from_float<T>(sum == 0.f ? 0.f : acc.x * inv);
            out[2 * lane + 1] = from_float<T>(sum == 0.f ? 0.f : acc.y * inv);
        }
    }
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

static int ka_grid(Kv4AttnParams* p, const mk36_kv4_cache* c) {
    const DeviceInfo* info = current_device_info();
    if (!info) return MK36_ERR_LAUNCH;
    // Columns beyond eight take passes of their own.  (Two blocks of eight in one pass, which reads and unpacks a tile once for both, need
    // all 255 registers: two CTAs an SM instead of three.  27B, three tokens, twelve rows: 52.5 us so, 43.0 in passes of eight; heads
    // of 128 channels with 16 columns or more were up to a tenth faster so.)
    p->blocks = (p->columns + 7) / 8;
    p->streams = p->cache.kv_heads * p->blocks;
    p->fd_blocks = make_fastdiv((unsigned)p->blocks), p->fd_group = make_fastdiv((unsigned)p->group), p->fd_streams = make_fastdiv((unsigned)p->streams);
    const double line = (double)p->cache.rows * p->cache.row_pages * (c->page_size / kKv4Tile) * p->streams;
    if (line > 2e9) MK36_FAIL(MK36_ERR_UNSUPPORTED, "kv4_attention_decode: the table holds more than 2e9 tiles of 16 tokens, heads and query blocks");
    const long long most = (long long)line;
    const long long ctas = (most + kKaMinTiles - 1) / kKaMinTiles, resident = (long long)info->sm_count * ka_ctas_per_sm(c->dtype == MK36_F32, c->head_dim);
    p->ctas = (int)(ctas < resident ? ctas : resident);
    // The wide form of the join: more than 64 pieces a pass when the table is full (4 rows, 16 / 2 heads of 128, 74 pieces: 13.7 us, 15.2 with
    // the other; 2 rows, 24 / 4 heads of 256, 55 pieces: 29.5 and 28.9; 8 rows, 16 / 2 heads of 256, 28 pieces: 54.7 and 47.6), or an SM for each CTA of both launches.  Either way there
    // are at most two such CTAs for each SM.
    const long long outputs = (long long)p->cache.rows * p->tokens * p->query_heads;
    p->join_wide = p->ctas > 64ll * p->cache.rows * p->streams || p->ctas + outputs * (c->head_dim / 64) <= info->sm_count;
    return MK36_OK;
}

template <typename T, int D>
static int kv4_attention_launch(const Kv4AttnParams& p, cudaStream_t s) {
    using C = KaConfig<T, D>;
    const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kv4_attention_kernel<T, D>), C::kSmem);
    if (rc != MK36_OK) return rc;
    kv4_attention_kernel<T, D><<<p.ctas, kKaThreads, C::kSmem, s>>>(p);
    MK36_CUDA_OK(cudaGetLastError());
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(p.join_wide ? (unsigned)(p.cache.rows * p.tokens * p.query_heads * (D / 64)) : (unsigned)p.ctas);
    config.blockDim = dim3(p.join_wide ? kKaWideWarps * 32 : kKaJoinWarps * 32);
    config.stream = s;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    MK36_CUDA_OK(cudaLaunchKernelEx(&config, p.join_wide ? kv4_attention_join_wide_kernel<T, D> : kv4_attention_join_cuts_kernel<T, D>, p));
    return MK36_OK;
}

template <typename T>
static int kv4_attention_head_dim(const Kv4AttnParams& p, int d, cudaStream_t s) {
    if (d == 64) return kv4_attention_launch<T, 64>(p, s);
    if (d == 128) return kv4_attention_launch<T, 128>(p, s);
    return kv4_attention_launch<T, 256>(p, s);
}

static size_t ka_workspace(const Kv4AttnParams& p, int d) { return 2ull * p.ctas * ka_slot_floats(d) * sizeof(float); }

}  // namespace mk36

using namespace mk36;

extern "C" size_t mk36_kv4_attention_workspace_bytes(const mk36_kv4_cache* cache, const mk36_kv4_attention_args* args) {
    Kv4AttnParams p{};
    if (kv4_attention_params(cache, args, &p) != MK36_OK || ka_grid(&p, cache) != MK36_OK) return 0;
    return ka_workspace(p, cache->head_dim);
}

extern "C" int mk36_kv4_attention_decode(const mk36_kv4_cache* cache, const mk36_kv4_attention_args* args, void* workspace,
                                         size_t workspace_bytes, void* stream) {
    Kv4AttnParams p{};
    int rc = kv4_attention_params(cache, args, &p);
    if (rc != MK36_OK) return rc;
    rc = ka_grid(&p, cache);
    if (rc != MK36_OK) return rc;
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < ka_workspace(p, cache->head_dim))
        MK36_FAIL(MK36_ERR_WORKSPACE, "kv4_attention_decode: workspace of %zu bytes is too small or not 16-byte aligned", workspace_bytes);
    p.partial = static_cast<float*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (cache->dtype) {
        case MK36_BF16: return kv4_attention_head_dim<__nv_bfloat16>(p, cache->head_dim, s);
        case MK36_F16: return kv4_attention_head_dim<__half>(p, cache->head_dim, s);
        default: return kv4_attention_head_dim<float>(p, cache->head_dim, s);
    }
}
