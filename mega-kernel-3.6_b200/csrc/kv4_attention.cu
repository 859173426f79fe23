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

#include "mk36_kv4.cuh"
#include "mk36_mma.cuh"
#include "mk36_ring.cuh"

namespace mk36 {

constexpr int kKaWarps = 4;
constexpr int kKaThreads = kKaWarps * 32;
constexpr int kKaCtasPerSm = 2;
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
};

// Partial results: per (CTA, first or last segment) and column the sums, then maximum (of scores in units of log 2) and sum of weights.
__host__ __device__ constexpr int ka_slot_floats(int d, int nt) { return 8 * nt * (d + 4); }

template <typename T, int D, int NT>
struct KaConfig {
    static constexpr int kGroups = D / kKv4Group;
    static constexpr int kTile = kv4_tile_bytes(D, sizeof(T));
    static constexpr int kFoldRow = D + 4;  // lanes 8 j + g of a store fall into 32 banks
    static constexpr int kFold = kKaWarps * 8 * kFoldRow * 4;
    static constexpr int kStats = kKaWarps * 8 * NT * (2 + kGroups) * 4;
    static constexpr int kRoom = 232448 / kKaCtasPerSm - 1024 - kFold - kStats - 512;
    static constexpr int kMost = kRoom / (kKaWarps * kTile);
    static constexpr int kStages = kMost < 8 ? kMost : 8;
    static constexpr int kSmem = kKaWarps * kStages * kTile + kFold + kStats + kKaWarps * kStages * 8;
    static constexpr int kQParts = sizeof(T) == 4 ? 2 : 1;
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

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}

// hi and lo halves of two fp32 values: 22 bits together
__device__ __forceinline__ void split_half(float x, float y, unsigned& hi, unsigned& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const unsigned*>(&h);
    lo = pack_half(x - f.x, y - f.y);
}

// 2^e, e in [-126, 127]
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

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
__device__ __forceinline__ long long ka_line(const Kv4AttnParams& p, int rows, int* s) {
    int mine = 0;  // tiles of a pass over every row: below 2^31 as long as rows * capacity / 16 is, which the host checks
    for (int r = threadIdx.x; r < rows; r += kThreads) mine += ka_tiles(p.cache, r);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(kFullMask, mine, off);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = mine;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) sum += s[w];
    return (long long)sum * p.streams;
}

__device__ __forceinline__ long long ka_piece(long long total, int ctas) {
    const long long each = (total + ctas - 1) / ctas;
    return each < kKaMinTiles ? kKaMinTiles : each;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kKaThreads, kKaCtasPerSm) kv4_attention_kernel(const __grid_constant__ Kv4AttnParams p) {
    using C = KaConfig<T, D, NT>;
    constexpr int G = C::kGroups, QP = C::kQParts;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int s_scan[kKaWarps], s_start[2], s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
    unsigned char* ring = smem + warp * C::kStages * C::kTile;
    float* s_fold = reinterpret_cast<float*>(smem + kKaWarps * C::kStages * C::kTile);
    float* s_max = s_fold + C::kFold / 4;               // [warp][8 NT]
    float* s_sum = s_max + kKaWarps * 8 * NT;           // [warp][8 NT]
    float* s_zero = s_sum + kKaWarps * 8 * NT;          // [warp][8 NT][G]
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(s_zero + kKaWarps * 8 * NT * G) + warp * C::kStages;
    if (lane == 0) {
        for (int i = 0; i < C::kStages; ++i) mbar_init(&bars[i], 1);
        mbar_init_fence();
    }
    if (threadIdx.x == 0) s_abort = 0;
    asm volatile("griddepcontrol.launch_dependents;");  // the join may be set up while this runs; it waits for the end of the grid

    // ---- this CTA's piece of the line
    const long long total = ka_line<kKaThreads>(p, p.cache.rows, s_scan);
    const long long piece = ka_piece(total, p.ctas);
    const long long begin = blockIdx.x * piece, end = min(total, begin + piece);
    if (begin >= end) return;
    {
        // the row that holds tile `begin`: rows in batches of a thread each
        int before = 0;
        const int target = (int)(begin / p.streams);  // begin's row has before * streams <= begin < (before + tiles) * streams
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
        const int off = (int)(begin - (long long)s_start[1] * p.streams);
        start.stream = off / start.tiles;
        start.tile = off - start.stream * start.tiles;
    }

    // ---- the ring: this warp's tiles are begin + warp, begin + warp + kKaWarps, ...
    KaCursor ahead = start;  // the tile to be requested next
    long long ahead_at = begin + warp;
    ka_advance(p, ahead, warp);
    int ahead_page = 0;
    auto page_of = [&]() {
        return ahead_at < end ? p.cache.table[(long long)ahead.row * p.cache.row_pages + fdiv(ahead.tile, p.cache.tiles_per_page)] : 0;
    };
    ahead_page = page_of();
    int requested = 0;
    unsigned lost = 0;  // bit s: stage s holds another page's tile, because the table names none
    auto request = [&](int stage) {
        if (ahead_at >= end) return;
        const bool bad = ahead_page < 0 || ahead_page >= p.cache.pages;
        lost = (lost & ~(1u << stage)) | (bad ? 1u << stage : 0u);
        if (lane == 0) {
            const int per = (int)p.cache.tiles_per_page.d;
            const int inner = ahead.tile - fdiv(ahead.tile, p.cache.tiles_per_page) * per;
            const long long page = bad ? 0 : ahead_page;
            const unsigned char* src = p.cache.pool + ((page * p.cache.kv_heads + ahead.stream / p.blocks) * per + inner) * C::kTile;
            mbar_arrive_expect_tx(&bars[stage], C::kTile);
            bulk_copy_g2s(ring + stage * C::kTile, src, C::kTile, &bars[stage]);
        }
        ++requested;
        ka_advance(p, ahead, kKaWarps);
        ahead_at += kKaWarps;
        ahead_page = page_of();
    };
    __syncwarp();
    for (int i = 0; i < C::kStages; ++i) request(i);

    int stage = 0, use = 0;
    bool dead = false;  // a wait has run out: outputs from here on are NaN
    long long at = begin + warp, segment = begin;
    KaCursor now = start;  // the tile at `segment`
    while (segment < end) {
        const long long segment_end = min(end, segment + (now.tiles - now.tile));
        const bool whole = now.tile == 0 && segment + now.tiles == segment_end;
        const int length = kv4_length(p.cache, now.row);
        const int kv_head = now.stream / p.blocks, block = now.stream - kv_head * p.blocks;
        const int row = now.row;

        // ---- the queries of this pass: column g of each n-tile, this lane's channels of every group
        unsigned qf[NT][QP][G][4][2];
        float q_sum[NT][2][G], mult[NT][2];
        int limit[NT][2], own_limit[NT];  // positions that the columns 2 j, 2 j + 1 see, and column g
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int column = (block * NT + nt) * 8 + g;
            float q[G][16], most = 0.f;
            const int token = column / p.group, head = kv_head * p.group + column - token * p.group;
            const T* src = static_cast<const T*>(p.q) + row * p.q_row + token * p.q_token + head * p.q_head + 16 * j;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    if (column < p.columns) {
                        const T* x = src + gr * kKv4Group + half * 8;
                        if (p.wide_q) {
                            unpack8(load_chunk8<T>(x), f);
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i) f[i] = to_float<T>(x[i]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        q[gr][half * 8 + i] = f[i];
                        most = fmaxf(most, fabsf(f[i]));
                    }
                }
            }
            most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 1));
            most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 2));
            const int e = min(max((int)(__float_as_uint(most) >> 23), 14), 254) - 127;  // 2^e <= most < 2^(e + 1)
            const float up = pow2(14 - e);
            float sum[G];
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                sum[gr] = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    q[gr][i] *= up;
                    sum[gr] += q[gr][i];
                }
                sum[gr] += __shfl_xor_sync(kFullMask, sum[gr], 1);
                sum[gr] += __shfl_xor_sync(kFullMask, sum[gr], 2);
#pragma unroll
                for (int m = 0; m < 4; ++m) {  // MMA m takes the codes 2 (m % 2), + 1, + 4, + 5 of word m / 2
                    const int c = (m >> 1) * 8 + (m & 1) * 2;
                    if (QP == 1) {
                        qf[nt][0][gr][m][0] = pack_half(q[gr][c], q[gr][c + 4]);
                        qf[nt][0][gr][m][1] = pack_half(q[gr][c + 1] * 0.0625f, q[gr][c + 5] * 0.0625f);
                    } else {
                        split_half(q[gr][c], q[gr][c + 4], qf[nt][0][gr][m][0], qf[nt][QP - 1][gr][m][0]);
                        split_half(q[gr][c + 1] * 0.0625f, q[gr][c + 5] * 0.0625f, qf[nt][0][gr][m][1], qf[nt][QP - 1][gr][m][1]);
                    }
                }
            }
            own_limit[nt] = length - p.tokens + 1 + token;
            // what belongs to a column goes to the lanes that hold it in the scores' layout: columns 2 j, 2 j + 1
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int from = (2 * j + c) * 4;
#pragma unroll
                for (int gr = 0; gr < G; ++gr) q_sum[nt][c][gr] = __shfl_sync(kFullMask, sum[gr], from) * pow2(-24);
                const int e_c = __shfl_sync(kFullMask, e, from);
                mult[nt][c] = ldexpf(p.scale * 1.4426950408889634f, 24 - 14 + e_c);
                limit[nt][c] = __shfl_sync(kFullMask, own_limit[nt], from);
            }
        }
        int sees_all = length;  // every column sees the positions below this
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sees_all = min(sees_all, min(limit[nt][0], limit[nt][1]));
        sees_all = min(sees_all, __shfl_xor_sync(kFullMask, sees_all, 1));
        sees_all = min(sees_all, __shfl_xor_sync(kFullMask, sees_all, 2));

        float o[NT][G][4][4], zero_sum[NT][G], top[NT], weight_sum[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            top[nt] = -INFINITY;
            weight_sum[nt] = 0.f;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                zero_sum[nt][gr] = 0.f;
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[nt][gr][m][i] = 0.f;
            }
        }
        int unit = 1;  // exponent field of the power of two that weights times scales are divided by

        for (; at < segment_end; at += kKaWarps) {
            const int tile = now.tile + (int)(at - segment);
            if (!dead && !mbar_wait(&bars[stage], use & 1, &s_abort)) dead = true;
            dead = __any_sync(kFullMask, dead);
            if (dead || (lost >> stage & 1u)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) weight_sum[nt] = __uint_as_float(0x7fc00000u);
            }
            if (dead) continue;
            const unsigned char* codes = ring + stage * C::kTile;
            const unsigned char* params = codes + 2 * kv4_code_bytes(D);

            // ---- scores
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[nt][i] = 0.f;
            {
                float ks[2][G], kz[2][G];
                load_params<T, G>(params + g * (G * 2 * (int)sizeof(T)), ks[0], kz[0]);
                load_params<T, G>(params + (g + 8) * (G * 2 * (int)sizeof(T)), ks[1], kz[1]);
                constexpr int kUnit = D >= 128 ? 16 : 8, kVecs = D / 8 / kUnit, kWords = kUnit / 4;
#pragma unroll
                for (int v = 0; v < kVecs; ++v) {
                    unsigned a[kWords], b[kWords];
                    lds_words(codes + (v * 32 + lane) * kUnit, a);
                    lds_words(codes + ((kVecs + v) * 32 + lane) * kUnit, b);
#pragma unroll
                    for (int x = 0; x < kWords / 2; ++x) {
                        const int gr = v * (kWords / 2) + x;
                        float acc[NT][4];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            const unsigned wa = a[2 * x + (m >> 1)] >> (8 * (m & 1)), wb = b[2 * x + (m >> 1)] >> (8 * (m & 1));
                            const unsigned a0 = wa & 0x000f000fu, a1 = wb & 0x000f000fu, a2 = wa & 0x00f000f0u, a3 = wb & 0x00f000f0u;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int part = 0; part < QP; ++part)
                                    mma_16816<__half>(acc[nt], a0, a1, a2, a3, qf[nt][part][gr][m][0], qf[nt][part][gr][m][1]);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                s[nt][i] += fmaf(ks[i >> 1][gr], acc[nt][i], kz[i >> 1][gr] * q_sum[nt][i & 1][gr]);
                    }
                }
            }
            const int first = tile * kKv4Tile;
            const bool edge = first + kKv4Tile > sees_all;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[nt][i] *= mult[nt][i & 1];
                    if (edge && first + g + 8 * (i >> 1) >= limit[nt][i & 1]) s[nt][i] = -INFINITY;
                }
                // from (tokens g, g + 8; columns 2 j, 2 j + 1) to (tokens 2 j, 2 j + 1, + 8, + 9; column g)
                transpose8(s[nt][0], s[nt][1]);
                transpose8(s[nt][2], s[nt][3]);
            }

            // ---- scales and zero points of the values of the lane's four tokens
            float vs[4][G], vz[4][G];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 2 * j + (i & 1) + 8 * (i >> 1);
                load_params<T, G>(params + kv4_param_bytes(D, sizeof(T)) + t * (G * 2 * (int)sizeof(T)), vs[i], vz[i]);
                if (edge && first + t >= length) {  // behind the row's end anything may lie
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) vs[i][gr] = vz[i][gr] = 0.f;
                }
            }
            unsigned largest = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int gr = 0; gr < G; ++gr) largest = max(largest, __float_as_uint(vs[i][gr]));
            largest = max(largest, __shfl_xor_sync(kFullMask, largest, 1));
            largest = max(largest, __shfl_xor_sync(kFullMask, largest, 2));
            const int unit_now = max(unit, min((int)(largest >> 23), 253));

            // ---- running maximum; what has been summed is brought to it
            float corr[NT];
            bool moved = unit_now != unit;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float m = fmaxf(fmaxf(s[nt][0], s[nt][1]), fmaxf(s[nt][2], s[nt][3]));
                m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 1));
                m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 2));
                m = fmaxf(m, top[nt]);
                const float base = m == -INFINITY ? 0.f : m;
                corr[nt] = exp2_approx(top[nt] - base);
                moved |= m != top[nt];
                top[nt] = m;
#pragma unroll
                for (int i = 0; i < 4; ++i) s[nt][i] = sizeof(T) == 4 ? exp2f(s[nt][i] - base) : exp2_approx(s[nt][i] - base);
            }
            if (__any_sync(kFullMask, moved)) {
                const float down = pow2(max(unit - unit_now, -126));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    weight_sum[nt] *= corr[nt];
                    const float c0 = __shfl_sync(kFullMask, corr[nt], 8 * j) * down, c1 = __shfl_sync(kFullMask, corr[nt], 8 * j + 4) * down;
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        zero_sum[nt][gr] *= corr[nt];
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            o[nt][gr][m][0] *= c0, o[nt][gr][m][1] *= c1;
                            o[nt][gr][m][2] *= c0, o[nt][gr][m][3] *= c1;
                        }
                    }
                }
                unit = unit_now;
            }
            const float shrink = pow2(127 - unit);

            // ---- values
            constexpr int kUnit = D / 16;
            unsigned v[4][G];
#pragma unroll
            for (int i = 0; i < 4; ++i) lds_words(codes + kv4_code_bytes(D) + (i * 32 + lane) * kUnit, v[i]);
            unsigned hi[NT][G][2], lo[NT][G][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                weight_sum[nt] += (s[nt][0] + s[nt][1]) + (s[nt][2] + s[nt][3]);
                auto weigh = [&](const float (&scale)[4][G], const float (&zero)[4][G]) {
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        float add = s[nt][0] * zero[0][gr];
#pragma unroll
                        for (int i = 1; i < 4; ++i) add = fmaf(s[nt][i], zero[i][gr], add);
                        zero_sum[nt][gr] += add;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nt][i] *= shrink;
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        split_half(s[nt][0] * scale[0][gr], s[nt][1] * scale[1][gr], hi[nt][gr][0], lo[nt][gr][0]);
                        split_half(s[nt][2] * scale[2][gr], s[nt][3] * scale[3][gr], hi[nt][gr][1], lo[nt][gr][1]);
                    }
                };
                if (edge) {  // what the column does not see may be a NaN, which a weight of 0 would let through
                    float scale[4][G], zero[4][G];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool seen = first + 2 * j + (i & 1) + 8 * (i >> 1) < own_limit[nt];
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) scale[i][gr] = seen ? vs[i][gr] : 0.f, zero[i][gr] = seen ? vz[i][gr] : 0.f;
                    }
                    weigh(scale, zero);
                } else {
                    weigh(vs, vz);
                }
            }
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
#pragma unroll
                for (int m = 0; m < 4; ++m) {  // rows g and g + 8: channels 8 g + c and 8 g + c + 2, c = 0, 1 (x 16), 4, 5 (x 16)
                    const unsigned pick = m < 2 ? 0x5410u : 0x7632u, mask = m & 1 ? 0x00f000f0u : 0x000f000fu;
                    const unsigned near = __byte_perm(v[0][gr], v[1][gr], pick), far = __byte_perm(v[2][gr], v[3][gr], pick);
                    const unsigned a0 = near & mask, a1 = near >> 8 & mask, a2 = far & mask, a3 = far >> 8 & mask;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (sizeof(T) == 4) {  // chains of two, added up in fp32: the tensor core cuts off where an addition rounds
                            float acc[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_16816<__half>(acc, a0, a1, a2, a3, lo[nt][gr][0], lo[nt][gr][1]);
                            mma_16816<__half>(acc, a0, a1, a2, a3, hi[nt][gr][0], hi[nt][gr][1]);
                            add_tile(o[nt][gr][m], acc);
                        } else {
                            mma_16816<__half>(o[nt][gr][m], a0, a1, a2, a3, lo[nt][gr][0], lo[nt][gr][1]);
                            mma_16816<__half>(o[nt][gr][m], a0, a1, a2, a3, hi[nt][gr][0], hi[nt][gr][1]);
                        }
                    }
                }
            }

            __syncwarp();  // every lane has read the stage
            request(stage);
            if (++stage == C::kStages) stage = 0, ++use;
        }

        // ---- the end of a segment: the warps' sums meet
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            weight_sum[nt] += __shfl_xor_sync(kFullMask, weight_sum[nt], 1);
            weight_sum[nt] += __shfl_xor_sync(kFullMask, weight_sum[nt], 2);
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                zero_sum[nt][gr] += __shfl_xor_sync(kFullMask, zero_sum[nt][gr], 1);
                zero_sum[nt][gr] += __shfl_xor_sync(kFullMask, zero_sum[nt][gr], 2);
            }
            if (j == 0) {
                const int c = (warp * NT + nt) * 8 + g;
                s_max[c] = top[nt];
                s_sum[c] = weight_sum[nt];
#pragma unroll
                for (int gr = 0; gr < G; ++gr) s_zero[c * G + gr] = zero_sum[nt][gr];
            }
        }
        __syncthreads();
        const float grow = pow2(unit - 127);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float weight[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float m = -INFINITY;
#pragma unroll
                for (int w = 0; w < kKaWarps; ++w) m = fmaxf(m, s_max[(w * NT + nt) * 8 + 2 * j + c]);
                const float own = s_max[(warp * NT + nt) * 8 + 2 * j + c];
                weight[c] = own == -INFINITY ? 0.f : exp2f(own - m) * grow;
            }
            // channel 8 g + i of a group at 8 i + g: the 32 lanes of a store fall into 32 banks
#pragma unroll
            for (int gr = 0; gr < G; ++gr)
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c = i & 1, channel = (m >> 1) * 4 + (m & 1) + 2 * (i >> 1);
                        s_fold[(warp * 8 + 2 * j + c) * C::kFoldRow + gr * kKv4Group + channel * 8 + g] = o[nt][gr][m][i] * (m & 1 ? 0x1p20f : 0x1p24f) * weight[c];
                    }
            __syncthreads();
            const long long slot = 2ll * blockIdx.x + (segment > begin ? 1 : 0);
            float* part = p.partial + slot * ka_slot_floats(D, NT) + nt * 8 * (D + 4);
            for (int i = threadIdx.x; i < 8 * D; i += kKaThreads) {
                const int c = i / D, channel = i - c * D;
                const int column = (block * NT + nt) * 8 + c;
                if (column >= p.columns) break;  // columns ascend with i
                const int place = channel / kKv4Group * kKv4Group + channel % 8 * 8 + channel % kKv4Group / 8;
                float m = -INFINITY, sum = 0.f, value = 0.f;
#pragma unroll
                for (int w = 0; w < kKaWarps; ++w) m = fmaxf(m, s_max[(w * NT + nt) * 8 + c]);
#pragma unroll
                for (int w = 0; w < kKaWarps; ++w) {
                    const int x = (w * NT + nt) * 8 + c;
                    const float own = s_max[x] == -INFINITY ? (s_sum[x] == 0.f ? 0.f : s_sum[x]) : exp2f(s_max[x] - m);
                    sum = fmaf(own, s_sum[x], sum);
                    value += s_fold[(w * 8 + c) * C::kFoldRow + place] + own * s_zero[x * G + channel / kKv4Group];
                }
                if (whole) {
                    const int token = column / p.group, head = kv_head * p.group + column - token * p.group;
                    T* out = static_cast<T*>(p.out) + (((long long)row * p.tokens + token) * p.query_heads + head) * D;
                    out[channel] = from_float<T>(sum == 0.f ? 0.f : value / sum);
                } else {
                    part[c * (D + 4) + channel] = value;
                    if (channel < 2) part[c * (D + 4) + D + channel] = channel ? sum : m;
                }
            }
            __syncthreads();
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

// Joins the partial results of rows that several CTAs worked on; a CTA for each query head and token.  Rows without a token get zeros.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kKaJoinThreads) kv4_attention_join_kernel(const __grid_constant__ Kv4AttnParams p) {
    __shared__ float s_out[kKaJoinThreads / 32][D];
    __shared__ int s_scan[kKaJoinThreads / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.x % p.query_heads, rest = blockIdx.x / p.query_heads;
    const int token = rest % p.tokens, row = rest / p.tokens;
    const int tiles = ka_tiles(p.cache, row);
    T* out = static_cast<T*>(p.out) + (long long)blockIdx.x * D;
    if (tiles == 0) {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // no CTA of this grid ends before the grid ahead of it
        for (int c = threadIdx.x; c < D; c += kKaJoinThreads) out[c] = from_float<T>(0.f);
        return;
    }
    const int kv_head = head / p.group, column = token * p.group + head - kv_head * p.group;
    const int block = column / (8 * NT);
    const long long before = ka_line<kKaJoinThreads>(p, row, s_scan), total = ka_line<kKaJoinThreads>(p, p.cache.rows, s_scan);
    const long long piece = ka_piece(total, p.ctas);
    const long long first = before + (long long)(kv_head * p.blocks + block) * tiles;
    const long long cta0 = first / piece, cta1 = (first + tiles - 1) / piece;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (cta0 == cta1) return;  // that CTA has written the output
    const float* base = p.partial + (column - block * 8 * NT) * (D + 4);
    auto part_of = [&](long long cta) { return base + (2 * cta + (first > cta * piece ? 1 : 0)) * ka_slot_floats(D, NT); };
    float top = -INFINITY;
    for (long long c = cta0 + lane; c <= cta1; c += 32) top = fmaxf(top, __ldcg(part_of(c) + D));
    top = warp_max(top);
    constexpr int kPer = D / 32;
    float acc[kPer], sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
#pragma unroll 4
    for (long long c = cta0 + warp; c <= cta1; c += kKaJoinThreads / 32) {
        const float* x = part_of(c);
        const float m = __ldcg(x + D), part_sum = __ldcg(x + D + 1);
        const float own = m == -INFINITY ? (part_sum == 0.f ? 0.f : part_sum) : exp2f(m - top);
        sum = fmaf(own, part_sum, sum);
#pragma unroll
        for (int i = 0; i < kPer; ++i) acc[i] = fmaf(own, __ldcg(x + i * 32 + lane), acc[i]);
    }
    __shared__ float s_sum[kKaJoinThreads / 32];
#pragma unroll
    for (int i = 0; i < kPer; ++i) s_out[warp][i * 32 + lane] = acc[i];
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += kKaJoinThreads) {
        float value = 0.f, all = 0.f;
#pragma unroll
        for (int w = 0; w < kKaJoinThreads / 32; ++w) {
            value += s_out[w][c];
            all += s_sum[w];
        }
        out[c] = from_float<T>(all == 0.f ? 0.f : value / all);
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
    if ((long long)c->rows * a->tokens > 0x7fffffffLL || (long long)c->rows * a->tokens * a->query_heads > 0x7fffffffLL)
        MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 query heads", what);
    if ((long long)c->rows * c->row_pages * (c->page_size / kKv4Tile) > 0x7fffffffLL)
        MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: the table holds more than 2^31 - 1 tiles of 16 tokens", what);
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
    const long long most = (long long)p->cache.rows * p->cache.row_pages * (page_size / kKv4Tile) * p->streams;
    const long long ctas = (most + kKaMinTiles - 1) / kKaMinTiles, resident = (long long)info->sm_count * kKaCtasPerSm;
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
    config.gridDim = dim3((unsigned)((long long)p.cache.rows * p.tokens * p.query_heads));
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
