// k_attn.hip -- attention of one new token of each row over a paged cache:
// out[s, h] = sum_t p_t v_t, p = softmax over t in (pos - window, pos] of scale * q[s, h] . k_t.
//
// One pass over the cells with the running maximum and sum of the softmax.  A cell is read
// once for all the query heads that share it, and both products run on the matrix cores: 32 tokens by
// up to 16 heads (16 tokens of a 32-bit cache).  Bytes bound it: 512 bytes of k and v of a
// token take some 6 cycles of a CU's four matrix cores and 55 of its share of the memory.
//
// 32-bit accuracy from 16-bit products: q and p are 32-bit and are split into parts of the
// cache's type, whose products with a cell are exact in the 32-bit sums.  bf16: three parts of 8
// bits, nothing is lost.  f16: q is first scaled by a power of two to 2^13..2^14 and p by 2^13, so that
// two parts hold 22 bits (a relative 2^-23) of all that matters beside the largest.  f32
// caches use the f32 matrix instruction.
//
// The layout needs no shared memory between the two products: lane l = 16 g + c of the
// scores' tile holds head c and tokens 4g .. 4g+3, just what the second product's right
// operand wants as its elements of the summed index, whose order is free.  So v's rows are
// loaded for these tokens, 16 bytes of a row per lane, and a lane transposes its
// 8 tokens x 8 values by byte permutations in registers.
//
// Measured (bf16, 8 cache heads of 128, 32 query heads; a page copy of the same size runs at 6.0 TB/s):
// one row of 131,072 tokens 102 us (5.2 TB/s), 30 rows of 1 to 8,192 tokens 92 to 106 us by the card
// (4.9 to 5.7 TB/s); 64 rows of a window of 512, heads of 64, 19.5 us (3.6 TB/s, 3.8 us of it the launch); f32, 16 heads of
// 128, 7 rows of 600 to 3,000 tokens 45 to 55 us by the run (4.1 to 5.0 TB/s); one row of 900 tokens 9.9 us, where the page
// table's, q's and the first cells' latencies and the join follow each other.  In the long ones the matrix cores are busy a
// tenth of the time, the vector units a fifth: the rest waits for memory.  A prompt's rows each read their cells again,
// through the caches: 2,048 rows from position 0 take 690 us, from 8,000 on 5.1 ms.
#include "sw_attn.h"

#define AT_NT 256
#define AT_NW (AT_NT / 64)
#define AT_BLOCKS 512                     // two blocks on each CU
#define AT_MIN 4                          // chunks of a part: one a wave
#define AT_ROW 12
// Beyond so many rows they are dealt whole, a block of each cache head a row, without counting them (32 query heads, 8
// of 128).  That suits a prompt's rows (257 from position 0: 35 us, counted 71; 2,048: 690 and 1,270) and rows of like
// lengths (257 of 1 to 500 tokens: 56 us, counted 63).  It does not suit a row far longer than the others, which stays with its
// one block: 257 rows of 1 to 500 and one of 65,536 take 950 us, counted 128.
#define AT_COUNT 256
// A row's parts, up to this many, are joined by the block that finishes last (one launch), else by k_attn_join
#define AT_FUSE 64

// bytes of a lane per row: 16-byte pieces first, then 8 and 4; the byte of row `rr` at dword w
template <int RB>
__host__ __device__ constexpr int at_vbyte(int w, int rr) {
    const int full = RB / 256, rem = RB % 256, x = w - 4 * full;
    return x < 0 ? (w / 4) * 256 + rr * 16 + (w % 4) * 4
         : rem >= 128 ? (x < 2 ? full * 256 + rr * 8 + x * 4 : full * 256 + 128 + rr * 4)
                      : full * 256 + rr * 4;
}
// parts of 8 values: three bf16 (by truncation: each takes the next 8 bits, exact) or two f16
template <int TYPE>
struct AtParts { static constexpr int n = TYPE == SW_KV_BF16 ? 3 : 2; };
template <int TYPE>
__device__ __forceinline__ void at_split(const float (&x)[8], sw_u32x4 (&o)[AtParts<TYPE>::n]) {
    if constexpr (TYPE == SW_KV_BF16) {
        uint32_t b[8], m[8], z[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            b[i] = __builtin_bit_cast(uint32_t, x[i]);
            const float r1 = x[i] - __builtin_bit_cast(float, b[i] & 0xFFFF0000u);
            m[i] = __builtin_bit_cast(uint32_t, r1);
            z[i] = __builtin_bit_cast(uint32_t, r1 - __builtin_bit_cast(float, m[i] & 0xFFFF0000u));
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            o[0][i] = __builtin_amdgcn_perm(b[2 * i + 1], b[2 * i], 0x07060302);
            o[1][i] = __builtin_amdgcn_perm(m[2 * i + 1], m[2 * i], 0x07060302);
            o[2][i] = __builtin_amdgcn_perm(z[2 * i + 1], z[2 * i], 0x07060302);
        }
    } else {
        sw_half8 hi, lo;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            hi[i] = (_Float16)x[i];
            lo[i] = (_Float16)(x[i] - (float)hi[i]);
        }
        o[0] = __builtin_bit_cast(sw_u32x4, hi);
        o[1] = __builtin_bit_cast(sw_u32x4, lo);
    }
}
template <int TYPE>
__device__ __forceinline__ sw_f32x4 at_mfma(sw_u32x4 a, sw_u32x4 b, sw_f32x4 c) {
    if constexpr (TYPE == SW_KV_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(sw_bf16x8, a), __builtin_bit_cast(sw_bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(sw_half8, a), __builtin_bit_cast(sw_half8, b), c, 0, 0, 0);
}

// the same over 16 of the summed index: elements 4 (l / 16) + 0 .. 3 of a lane
typedef _Float16 at_half4 __attribute__((ext_vector_type(4)));
typedef short at_short4 __attribute__((ext_vector_type(4)));
template <int TYPE>
__device__ __forceinline__ sw_f32x4 at_mfma16(uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1, sw_f32x4 c) {
    const uint2 a = make_uint2(a0, a1), b = make_uint2(b0, b1);
    if constexpr (TYPE == SW_KV_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(at_short4, a), __builtin_bit_cast(at_short4, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(at_half4, a), __builtin_bit_cast(at_half4, b), c, 0, 0, 0);
}

// Tokens of a wave's chunk: two tiles; one where two would leave room for one block on a CU and one for two
// (bf16 heads of 224 and 256 spill at two: 127 us against 106 for 8 rows of 8192 tokens).  bf16 heads of 160 and f16 of 256
// spill 11 and 6 registers at two and are no better off at one: 49 rows of 469 tokens 24.0 us against 30.4 and 33.4
// against 41.6, 8 rows of 8192 68 against 71 and 106 against 104.
__host__ __device__ constexpr int at_chunk(int type, int dh) {
    return type == SW_KV_F32 || (dh > 160 && (type == SW_KV_F16 || dh <= 192)) ? 16 : 32;
}
__host__ __device__ constexpr int at_blocks_cu(int type, int dh) {
    return (type == SW_KV_F32 && dh > 160) || (type == SW_KV_BF16 && dh > 192) ? 1 : 2;
}

// (the same in every lane: kept in scalar registers)
__device__ __forceinline__ int at_uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t at_uni(int64_t x) {
    return (int64_t)(((uint64_t)(uint32_t)at_uni((int)(x >> 32)) << 32) | (uint32_t)at_uni((int)x));
}
// Row s's position, -1 for a row without cells to look for
__device__ __forceinline__ int at_pos(const SwRows &r, int s) {
    const int sq = r.seq ? r.seq[s] : s;
    return sq < 0 || sq >= r.n_seqs ? -1 : r.pos[s];
}
// A row's cells as chunks of CT tokens: n of them from chunk c0.
struct AtRow { int first, last, c0, n; };
__device__ __forceinline__ AtRow at_row(const SwKv &c, const SwRows &r, int pos, int window, int CT) {
    AtRow w;
    w.first = window > 0 && pos >= window ? pos - window + 1 : 0;
    w.last = min(pos, (r.max_pages << c.psh) - 1);                     // (the host keeps that below 2^30)
    w.c0 = w.first / CT;
    w.n = w.last < w.first ? 0 : w.last / CT - w.c0 + 1;
    return w;
}

// The least chunks of a part: one a wave, and a part's chunks take a wave a third of a microsecond each, its outputs
// the join some 30 KB a microsecond, so the longest row's (mx chunks) are no shorter than where the two
// together are least.
__host__ __device__ inline int at_least(int64_t mx, int G, int dh) {
    const int best = (int)sqrtf((float)mx * (float)((G < 16 ? G : 16) * dh) / 2500.f);
    return best < AT_MIN ? AT_MIN : best;
}

// How the rows' chunks are dealt to the B blocks of a cache head.  Laid end to end they are N, and
// block b takes those from b q to (b + 1) q, whatever rows they fall in: parts of rows, joined
// at the end, and the same work for each block however the lengths differ.  Or whole rows (b, b + B,
// ...), where that is less: a row costs a block its chunks and about AT_ROW more for its beginning
// and end, a join as much again.  The lengths are on the device alone, so each wave counts them, 64
// rows at a time; up to 64 rows their positions then stay in registers.
struct AtPlan {
    int64_t N, q;
    bool whole;
    int pos, n;                                                        // lane i: row i's position and chunks (S <= 64)
    uint32_t upto;                                                     //         the chunks of rows up to it
};
__device__ __forceinline__ AtPlan at_plan(const SwKv &c, const SwRows &r, int S, int Hq, int window, int CT, int B, int fuse) {
    AtPlan p = {};
    if (S > AT_COUNT) { p.whole = true; return p; }
    const int lane = threadIdx.x & 63;
    int64_t mx = 0;
    p.N = 0;
    if (S == 1) {
        p.pos = at_uni(at_pos(r, 0));
        p.n = at_row(c, r, p.pos, window, CT).n;
        p.upto = (uint32_t)p.n;
        p.N = mx = p.n;
    } else
    for (int i0 = 0; i0 < S; i0 += 64) {                               // (the host keeps 64 rows below 2^32 chunks)
        p.pos = i0 + lane < S ? at_pos(r, i0 + lane) : -1;
        p.n = at_row(c, r, p.pos, window, CT).n;
        p.upto = sw_wave_scan((uint32_t)p.n);
        p.N += (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)p.upto, 63);
        const int m = at_uni((int)sw_wave_max((uint32_t)p.n));
        mx = m > mx ? m : mx;
    }
    p.q = (p.N + B - 1) / B;
    const int best = at_uni(at_least(mx, Hq / c.Hkv, c.dh));
    if (p.q < best) p.q = best;
    if (fuse && B > AT_FUSE && p.q * (AT_FUSE - 2) < mx) p.q = (mx + AT_FUSE - 3) / (AT_FUSE - 2);      // (no row has more parts)
    p.whole = ((S + B - 1) / B) * (AT_ROW + mx) <= p.q + AT_ROW * (2 + S / B);
    return p;
}
// the row in which chunk `at` (below N) of all lies, and the chunks of rows before it
__device__ __forceinline__ int at_find(const AtPlan &plan, const SwKv &c, const SwRows &r, int S, int window, int CT, int64_t at,
                                       int64_t &before) {
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    uint32_t upto = plan.upto;
    int n = plan.n, i0 = 0;
    for (;; i0 += 64) {
        if (S > 64) {
            n = i0 + lane < S ? at_row(c, r, at_pos(r, i0 + lane), window, CT).n : 0;
            upto = sw_wave_scan((uint32_t)n);
        }
        const int64_t all = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        if (base + all > at || i0 + 64 >= S) break;
        base += all;
    }
    const int i = __builtin_ctzll(__ballot((int64_t)upto > at - base) | (1ull << 63));
    before = base + (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(upto - (uint32_t)n), i);
    return i0 + i;
}

// What one block writes for another of the same launch goes through to memory and is read from there,
// eight bytes at a time (agent-scope accesses): no cache has to be written back or dropped for it, as a
// fence would, 20 us and more over a launch of 512 blocks.  The writer waits for its
// stores before it counts itself done.
__device__ __forceinline__ void at_put(float *p, float a, float b) {
    const uint64_t v = ((uint64_t)__builtin_bit_cast(uint32_t, b) << 32) | __builtin_bit_cast(uint32_t, a);
    __hip_atomic_store((uint64_t *)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 at_get(const float *p) {
    const uint64_t v = __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__builtin_bit_cast(float, (uint32_t)v), __builtin_bit_cast(float, (uint32_t)(v >> 32)));
}

// Parts that are written, of the split row that begins in a block (no two begin in one): counted up by
// its blocks, and zero again when the last has joined them.  Launches are in one stream's order.
static __device__ int g_at_done[AT_BLOCKS];

// One block per cache head (16 query heads of it) and share of the rows' chunks; of a row's part a
// wave takes every 4th chunk, its k of the next chunk and v of the next chunk in flight while
// it computes.
template <int TYPE, int NB>
__global__ __launch_bounds__(AT_NT, at_blocks_cu(TYPE, 32 * NB)) void k_attn(SwKv c, SwRows r, const float *__restrict__ q, int S, int Hq, float sc0,
                                                                int window, float *__restrict__ out, float *__restrict__ part, int B, int fuse) {
    constexpr bool F32 = TYPE == SW_KV_F32;
    constexpr int DH = 32 * NB, ES = F32 ? 4 : 2, RB = DH * ES, CT = at_chunk(TYPE, DH);
    constexpr int NT = CT / 16, NS = RB / 64, ND = RB / 64, NTOK = 4 * NT, NO = DH / 16;
    constexpr int NP = F32 ? 1 : AtParts<TYPE>::n, QN = NP * NS * 64, QI = (NS * 64 + AT_NT - 1) / AT_NT;
    constexpr int LD = DH + 4;                                         // a head's row in the waves' join
    constexpr int SHJ = AT_NW * 16 * LD * 4, SHB = QN * 16 > SHJ ? QN * 16 : SHJ;
    static_assert(SHJ >= AT_FUSE * 16 * 4 + AT_NT * 16, "the parts' weights and sums");
    __shared__ __align__(16) char sh[SHB];
    __shared__ float s_m[AT_NW][16], s_l[AT_NW][16], s_q[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = at_uni(tid >> 6), g = lane >> 4, cl = lane & 15;
    const int G = Hq / c.Hkv, gt = (G + 15) >> 4, per_s = c.Hkv * gt;
    const int hg = blockIdx.x % per_s, b = blockIdx.x / per_s;
    const int hk = hg / gt, h0 = hk * G + (hg % gt) * 16, nh = min(16, G - (hg % gt) * 16);
    const AtPlan plan = at_plan(c, r, S, Hq, window, CT, B, fuse);
    auto row_at = [&](int s) { return at_row(c, r, S <= 64 ? __builtin_amdgcn_readlane(plan.pos, s) : at_uni(at_pos(r, s)), window, CT); };
    for (int64_t s = b + (int64_t)B * tid; s < S; s += (int64_t)B * AT_NT)             // rows without any cell: zeros
        if (at_row(c, r, at_pos(r, (int)s), window, CT).n == 0)
            for (int i = 0; i < nh * DH; i += 4) *(sw_f32x4 *)(out + (s * Hq + h0) * DH + i) = sw_f32x4{0.f, 0.f, 0.f, 0.f};
    int64_t at = (int64_t)b * plan.q, end = at + plan.q < plan.N ? at + plan.q : plan.N, before = 0;
    if (!plan.whole && at >= end) return;
    int s = plan.whole ? b : at_find(plan, c, r, S, window, CT, at, before);
    const int pmask = (1 << c.psh) - 1;
    const char *kb = (const char *)c.k + (int64_t)hk * c.hs * ES + g * 16;
    const char *vb = (const char *)c.v + (int64_t)hk * c.hs * ES;
    sw_u32x4 *sq = (sw_u32x4 *)sh;

    for (; s < S && (plan.whole || at < end); s += plan.whole ? B : 1) {
        const AtRow w = row_at(s);
        if (w.n == 0) continue;
        // this block's chunks of the row
        const int from = plan.whole ? 0 : (int)(at - before), len = plan.whole ? w.n : (int)(end - at < w.n - from ? end - at : w.n - from);
        const int c1 = w.c0 + from + len;
        int ch = w.c0 + from + wave;
        const int64_t begin = before;
        before += w.n;
        at += len;
        // ---- q's rows on their way, then the first chunk's cells
        const float *qrow = q + ((int64_t)s * Hq + h0) * DH;
        sw_f32x4 qx[QI][F32 ? 1 : 2];
#pragma unroll
        for (int i = 0; i < QI; i++) {
            const int d = ((tid + i * AT_NT) >> 6) * (64 / ES) + g * (16 / ES);
#pragma unroll
            for (int j = 0; j < (F32 ? 1 : 2); j++) {
                qx[i][j] = sw_f32x4{0.f, 0.f, 0.f, 0.f};
                if (tid + i * AT_NT < NS * 64 && cl < nh) qx[i][j] = *(const sw_f32x4 *)(qrow + cl * DH + d + 4 * j);
            }
        }
        const int seq = r.seq ? r.seq[s] : s;
        struct Pages { int k[NT], v[NT]; };
        auto pages = [&](int x) {
            Pages p;
            const int t0 = x * CT;
            if (pmask >= CT - 1) {                                     // one page, read once for the wave
                const int y = __builtin_amdgcn_readfirstlane(sw_page(c, r, seq, t0));
#pragma unroll
                for (int t = 0; t < NT; t++) p.k[t] = p.v[t] = y;
            } else {
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    p.k[t] = sw_page(c, r, seq, t0 + 16 * t + cl);
                    p.v[t] = sw_page(c, r, seq, t0 + 16 * t + 4 * g);
                }
            }
            return p;
        };
        sw_u32x4 K[NT][NS];
        uint32_t V[NTOK][ND];
        // (a page that leads nowhere: page 0's cells are read in its place and weigh nothing)
        auto load_k = [&](int x, const Pages &p) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const char *a = kb + ((int64_t)max(p.k[t], 0) * c.ps + (int64_t)((x * CT + 16 * t + cl) & pmask) * c.ts) * ES;
#pragma unroll
                for (int i = 0; i < NS; i++) K[t][i] = *(const sw_u32x4 *)(a + i * 64);
            }
        };
        auto load_v = [&](int x, const Pages &p) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const char *a = vb + ((int64_t)max(p.v[t], 0) * c.ps + (int64_t)((x * CT + 16 * t + 4 * g + j) & pmask) * c.ts) * ES;
                    uint32_t (&d)[ND] = V[4 * t + j];
#pragma unroll
                    for (int u = 0; u < RB / 256; u++) {
                        const sw_u32x4 y = *(const sw_u32x4 *)(a + u * 256 + cl * 16);
#pragma unroll
                        for (int e = 0; e < 4; e++) d[4 * u + e] = y[e];
                    }
                    constexpr int w0 = 4 * (RB / 256), b0 = RB / 256 * 256;
                    if constexpr (RB % 256 >= 128) {
                        const uint2 y = *(const uint2 *)(a + b0 + cl * 8);
                        d[w0] = y.x; d[w0 + 1] = y.y;
                    }
                    if constexpr (RB % 128 == 64) d[ND - 1] = *(const uint32_t *)(a + RB - 64 + cl * 4);
                }
        };
        Pages p, pn;
        if (ch < c1) {
            p = pages(ch);
            pn = ch + AT_NW < c1 ? pages(ch + AT_NW) : p;
            load_k(ch, p);
            load_v(ch, p);
        }
        // ---- q's parts in the right operand's order: [part][step][lane] of 16 bytes
        float sc = sc0;
        int up = 0;                                                    // the power of two that q is scaled by
        if constexpr (TYPE == SW_KV_F16) {
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < QI; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(qx[i][j / 4][j % 4]));
            mx = sw_max4(mx);
            __syncthreads();                                           // (the row before is done with)
            if (lane < 16) s_m[wave][cl] = mx;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < AT_NW; i++) mx = fmaxf(mx, s_m[i][cl]);
            up = mx > 0.f && mx < INFINITY ? 13 - ilogbf(mx) : 0;      // (-114 to 162: no float holds them all)
            sc = ldexpf(sc0, -up);
            if (fabsf(sc) == INFINITY && fabsf(sc0) < INFINITY) sc = copysignf(3.402823466e38f, sc0);   // (a score of 0 stays one)
        } else {
            __syncthreads();                                           // (the row before is done with)
        }
#pragma unroll
        for (int i = 0; i < QI; i++) {
            if (tid + i * AT_NT >= NS * 64) break;
            if constexpr (F32) {
                sq[tid + i * AT_NT] = __builtin_bit_cast(sw_u32x4, qx[i][0]);
            } else {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = TYPE == SW_KV_F16 ? ldexpf(qx[i][j / 4][j % 4], up) : qx[i][j / 4][j % 4];
                sw_u32x4 o[NP];
                at_split<TYPE>(x, o);
#pragma unroll
                for (int u = 0; u < NP; u++) sq[u * NS * 64 + tid + i * AT_NT] = o[u];
            }
        }
        __syncthreads();

        sw_f32x4 O[NO];
#pragma unroll
        for (int i = 0; i < NO; i++) O[i] = sw_f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;                                  // head cl: the maximum, this lane's part of the sum
        for (; ch < c1; ch += AT_NW) {
            const bool more = ch + AT_NW < c1;
            Pages pnn = pn;
            if (ch + 2 * AT_NW < c1) pnn = pages(ch + 2 * AT_NW);
            // scores of the chunk's tokens 16 t + 4 g + j for head cl
            sw_f32x4 Sc[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                Sc[t] = sw_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    if constexpr (F32) {
                        const sw_f32x4 a = __builtin_bit_cast(sw_f32x4, K[t][i]), y = __builtin_bit_cast(sw_f32x4, sq[i * 64 + lane]);
#pragma unroll
                        for (int e = 0; e < 4; e++) Sc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], y[e], Sc[t], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int u = 0; u < NP; u++) Sc[t] = at_mfma<TYPE>(K[t][i], sq[(u * NS + i) * 64 + lane], Sc[t]);
                    }
                }
            }
            if (more) load_k(ch + AT_NW, pn);
            bool ok = ch * CT >= w.first && ch * CT + CT - 1 <= w.last;
#pragma unroll
            for (int t = 0; t < NT; t++) ok = ok && p.v[t] >= 0;
            const bool full = __all(ok);
            float x[NTOK], mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[4 * t + j] = Sc[t][j] * sc;
                    if (!full) {
                        const int tok = ch * CT + 16 * t + 4 * g + j;
                        if (tok < w.first || tok > w.last || p.v[t] < 0) {
                            x[4 * t + j] = -INFINITY;
#pragma unroll
                            for (int e = 0; e < ND; e++) V[4 * t + j][e] = 0;
                        }
                    }
                    mx = fmaxf(mx, x[4 * t + j]);
                }
            const float nm = fmaxf(m, sw_max4(mx));
            if (__any(nm > m)) {                                       // some head's maximum grew
                const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - nm);
                l = l * f;
#pragma unroll
                for (int i = 0; i < NO; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) O[i][j] = O[i][j] * f;
                m = nm;
            }
            const float base = m == -INFINITY ? 0.f : TYPE == SW_KV_F16 ? m - 13.f : m;
            float pr[NTOK];
#pragma unroll
            for (int j = 0; j < NTOK; j++) {
                pr[j] = __builtin_amdgcn_exp2f(x[j] - base);
                l = l + pr[j];
            }
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int e = 0; e < ND; e++)
                        O[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, V[j][e]), pr[j], O[e], 0, 0, 0);
            } else {
                float p8[8];
#pragma unroll
                for (int j = 0; j < 8; j++) p8[j] = j < NTOK ? pr[j] : 0.f;
                sw_u32x4 P[NP];
                at_split<TYPE>(p8, P);
#pragma unroll
                for (int e = 0; e < 2 * ND; e++) {
                    uint32_t a[4];
#pragma unroll
                    for (int i = 0; i < NTOK / 2; i++)
                        a[i] = __builtin_amdgcn_perm(V[2 * i + 1][e / 2], V[2 * i][e / 2], e & 1 ? 0x07060302 : 0x05040100);
#pragma unroll
                    for (int u = 0; u < NP; u++) {
                        if constexpr (NT == 2) O[e] = at_mfma<TYPE>(sw_u32x4{a[0], a[1], a[2], a[3]}, P[u], O[e]);
                        else O[e] = at_mfma16<TYPE>(a[0], a[1], P[u][0], P[u][1], O[e]);
                    }
                }
            }
            if (more) load_v(ch + AT_NW, pn);
            p = pn;
            pn = pnn;
        }
        // ---- the waves join: outputs relative to the block's maximum, summed in the waves' order
        l = sw_sum4(l);
        __syncthreads();                                               // q's parts (and the maxima of q) are done with
        if (g == 0) { s_m[wave][cl] = m; s_l[wave][cl] = l; }
        __syncthreads();
        float M = s_m[0][cl];
#pragma unroll
        for (int i = 1; i < AT_NW; i++) M = fmaxf(M, s_m[i][cl]);
        const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
        float *so = (float *)sh + wave * 16 * LD + cl * LD;
#pragma unroll
        for (int e = 0; e < NO; e++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int d = F32 ? at_vbyte<RB>(e, 4 * g + j) / 4 : at_vbyte<RB>(e / 2, 4 * g + j) / 2 + (e & 1);
                so[d] = O[e][j] * f;
            }
        const bool all = len == w.n;
        float *prow = all ? nullptr : part + ((int64_t)(b + s) * Hq + h0) * (DH + 4);      // (one more for each row or block)
        if (tid < 16) {
            float L = 0.f;
#pragma unroll
            for (int i = 0; i < AT_NW; i++) L = __builtin_fmaf(s_l[i][tid], s_m[i][tid] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[i][tid] - M), L);
            s_q[tid] = L;
            if (!all && tid < nh) at_put(prow + tid * (DH + 4), M, L);
        }
        __syncthreads();
        for (int i = tid; i < nh * (DH / 4); i += AT_NT) {
            const int h = i / (DH / 4), d = i % (DH / 4) * 4;
            sw_f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < AT_NW; v++) {
                const sw_f32x4 y = *(const sw_f32x4 *)((float *)sh + (v * 16 + h) * LD + d);
#pragma unroll
                for (int e = 0; e < 4; e++) a[e] = a[e] + y[e];
            }
            if (!all) {
                at_put(prow + h * (DH + 4) + 4 + d, a[0], a[1]);
                at_put(prow + h * (DH + 4) + 6 + d, a[2], a[3]);
            } else {
                const float L = s_q[h];
#pragma unroll
                for (int e = 0; e < 4; e++) a[e] = L == 0.f ? 0.f : a[e] / L;
                *(sw_f32x4 *)(out + ((int64_t)s * Hq + h0 + h) * DH + d) = a;
            }
        }
        if (all || !fuse) continue;
        // ---- the last of the row's blocks joins its parts, in their order
        const int b0 = (int)(begin / plan.q), parts = (int)((before - 1) / plan.q) - b0 + 1;
        int *done = g_at_done + hg * B + b0;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                                               // the block's part is in memory
        if (tid == 0) s_q[0] = __hip_atomic_fetch_add(done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1 ? 1.f : 0.f;
        __syncthreads();
        if (s_q[0] == 0.f) continue;
        if (tid == 0) __hip_atomic_store(done, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int64_t prs = (int64_t)Hq * (DH + 4);                    // from a part to the next
        const float *p0 = part + ((int64_t)(b0 + s) * Hq + h0) * (DH + 4);
        float *s_f = (float *)sh;                                      // [part][head] weights
        sw_f32x4 *s_o = (sw_f32x4 *)(sh + AT_FUSE * 16 * 4);
        const int items = nh * (DH / 4), ng = items < AT_NT ? AT_NT / items : 1;       // groups of parts, where few values
        const int it0 = ng > 1 ? tid % items : tid, gr = ng > 1 ? tid / items : 0;
        for (int i0 = 0; i0 < items; i0 += AT_NT) {
            const int it = i0 + it0, h = it / (DH / 4), d = it % (DH / 4) * 4;
            const bool mine = it < items && gr < ng;
            const float *po = p0 + h * (DH + 4) + 4 + d;
            sw_f32x4 a = {0.f, 0.f, 0.f, 0.f};
            for (int j0 = gr; j0 < parts || j0 == gr; j0 += 8 * ng) {
                float2 y[8], z[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    y[j] = z[j] = make_float2(0.f, 0.f);
                    if (mine && j0 + j * ng < parts) {
                        y[j] = at_get(po + (j0 + j * ng) * prs);
                        z[j] = at_get(po + (j0 + j * ng) * prs + 2);
                    }
                }
                if (i0 == 0 && j0 == gr) {                             // (meanwhile) the parts' weights, 16 threads a head
                    const int hh = tid >> 4;
                    float2 ml[AT_FUSE / 16];
                    float M2 = -INFINITY, L = 0.f;
#pragma unroll
                    for (int i = 0; i < AT_FUSE / 16; i++) {
                        ml[i] = make_float2(-INFINITY, 0.f);
                        if (hh < nh && (tid & 15) + 16 * i < parts) ml[i] = at_get(p0 + ((tid & 15) + 16 * i) * prs + hh * (DH + 4));
                        M2 = fmaxf(M2, ml[i].x);
                    }
                    for (int o = 8; o; o >>= 1) M2 = fmaxf(M2, __shfl_xor(M2, o));
#pragma unroll
                    for (int i = 0; i < AT_FUSE / 16; i++) {
                        const float x = ml[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[i].x - M2);
                        if (hh < nh) s_f[((tid & 15) + 16 * i) * 16 + hh] = x;
                        L = __builtin_fmaf(ml[i].y, x, L);
                    }
                    for (int o = 8; o; o >>= 1) L = L + __shfl_xor(L, o);
                    __syncthreads();                                   // (s_q[0] is read)
                    if ((tid & 15) == 0 && hh < nh) s_q[hh] = L;
                    __syncthreads();
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float x = mine && j0 + j * ng < parts ? s_f[(j0 + j * ng) * 16 + h] : 0.f;
                    a[0] = __builtin_fmaf(y[j].x, x, a[0]);
                    a[1] = __builtin_fmaf(y[j].y, x, a[1]);
                    a[2] = __builtin_fmaf(z[j].x, x, a[2]);
                    a[3] = __builtin_fmaf(z[j].y, x, a[3]);
                }
            }
            if (ng > 1) {
                s_o[tid] = a;
                __syncthreads();
                for (int i = 1; i < ng && gr == 0; i++) {
                    const sw_f32x4 y = s_o[i * items + it];
#pragma unroll
                    for (int e = 0; e < 4; e++) a[e] = a[e] + y[e];
                }
            }
            if (mine && gr == 0) {
                const float L = s_q[h];
#pragma unroll
                for (int e = 0; e < 4; e++) a[e] = L == 0.f ? 0.f : a[e] / L;
                *(sw_f32x4 *)(out + ((int64_t)s * Hq + h0 + h) * DH + d) = a;
            }
        }
    }
}

// The parts of a row's head joined: part [block + row][head] of (maximum, sum, -, -, the
// output's values).  A part's weight first, one part a thread; then dh / 4 threads take four values of
// every (AT_NT / (dh / 4))-th part, and their sums meet in order.
__global__ __launch_bounds__(AT_NT) void k_attn_join(SwKv c, SwRows r, int S, int Hq, int window, int CT, const float *__restrict__ part,
                                                     int B, float *__restrict__ out) {
    __shared__ float s_f[AT_BLOCKS], s_r[AT_NW];
    __shared__ sw_f32x4 s_o[AT_NT];
    const int tid = threadIdx.x, s = blockIdx.x / Hq, h = blockIdx.x % Hq, nd = c.dh / 4, ng = AT_NT / nd;
    const int n = at_row(c, r, at_uni(at_pos(r, s)), window, CT).n;
    if (n == 0) return;
    const AtPlan plan = at_plan(c, r, S, Hq, window, CT, B, 0);
    if (plan.whole) return;
    int64_t before = 0;                                                // the chunks of rows before it
    for (int i0 = 0; i0 < s; i0 += 64) {
        const int i = i0 + (tid & 63);
        before += (uint32_t)__builtin_amdgcn_readlane((int)sw_wave_scan(i < s ? (uint32_t)at_row(c, r, at_pos(r, i), window, CT).n : 0u), 63);
    }
    const int b0 = (int)(before / plan.q), parts = (int)((before + n - 1) / plan.q) - b0 + 1;
    if (parts < 2) return;
    const int64_t row = (int64_t)Hq * (c.dh + 4);                      // from a part to the next
    const float *p = part + ((int64_t)(b0 + s) * Hq + h) * (c.dh + 4);
    float M = -INFINITY, L = 0.f;
    for (int i = tid; i < parts; i += AT_NT) {
        s_f[i] = p[i * row];
        M = fmaxf(M, s_f[i]);
    }
    for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    if ((tid & 63) == 0) s_r[tid >> 6] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < AT_NW; i++) M = fmaxf(M, s_r[i]);
    __syncthreads();
    for (int i = tid; i < parts; i += AT_NT) {
        const float f = s_f[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_f[i] - M);
        s_f[i] = f;
        L = __builtin_fmaf(p[i * row + 1], f, L);
    }
    for (int o = 32; o; o >>= 1) L = L + __shfl_xor(L, o);
    if ((tid & 63) == 0) s_r[tid >> 6] = L;
    __syncthreads();
    const int gr = tid / nd, d = tid % nd * 4;
    sw_f32x4 a = {0.f, 0.f, 0.f, 0.f};
    if (gr < ng) {
#pragma unroll 4
        for (int i = gr; i < parts; i += ng) {
            const sw_f32x4 v = *(const sw_f32x4 *)(p + i * row + 4 + d);
            const float f = s_f[i];
#pragma unroll
            for (int e = 0; e < 4; e++) a[e] = __builtin_fmaf(v[e], f, a[e]);
        }
        s_o[tid] = a;
    }
    __syncthreads();
    if (tid >= nd) return;
    L = 0.f;
#pragma unroll
    for (int i = 0; i < AT_NW; i++) L = L + s_r[i];
    for (int i = 1; i < ng; i++) {
        const sw_f32x4 v = s_o[i * nd + tid];
#pragma unroll
        for (int e = 0; e < 4; e++) a[e] = a[e] + v[e];
    }
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] = L == 0.f ? 0.f : a[e] / L;
    *(sw_f32x4 *)(out + (int64_t)blockIdx.x * c.dh + d) = a;
}

// cells of the longest row there can be
static int64_t at_cells(const SwKv &c, const SwRows &r, int window) {
    const int64_t cells = (int64_t)r.max_pages << c.psh, most = (int64_t)window + at_chunk(c.type, c.dh);
    return window > 0 && most < cells ? most : cells;                  // (a window begins anywhere in a chunk)
}
int64_t sw_attn_row_chunks(const SwKv &c, const SwRows &r) {
    const int CT = at_chunk(c.type, c.dh);
    return (((int64_t)r.max_pages << c.psh) + CT - 1) / CT;
}
// Blocks of a cache head: so many that all of them are AT_BLOCKS, no more than rows or least parts for them.
static int at_blocks(const SwKv &c, const SwRows &r, int Hq, int window, int S) {
    if (S > AT_COUNT) return S;
    const int per_s = c.Hkv * ((Hq / c.Hkv + 15) / 16), CT = at_chunk(c.type, c.dh);
    const int64_t most = (S * (at_cells(c, r, window) / CT + 1) + AT_MIN - 1) / AT_MIN, n = AT_BLOCKS / per_s;
    const int64_t use = S > most ? S : most;
    return (int)(n < 1 ? 1 : n < use ? n : use);
}
int64_t sw_attn_part_floats(const SwKv &c, const SwRows &r, int Hq, int window, int S) {
    const int B = at_blocks(c, r, Hq, window, S);
    return B > 1 && S <= AT_COUNT ? (int64_t)(B + S) * Hq * (c.dh + 4) : 0;
}

template <int TYPE, int NB>
static void at_launch(hipStream_t st, unsigned grid, const SwKv &c, const SwRows &r, const float *q, int S, int Hq, float sc, int window,
                      float *out, float *part, int B, int fuse) {
    SW_LAUNCH((k_attn<TYPE, NB>), dim3(grid), dim3(AT_NT), 0, st, c, r, q, S, Hq, sc, window, out, part, B, fuse);
}
template <int TYPE>
static void at_dispatch(hipStream_t st, unsigned grid, const SwKv &c, const SwRows &r, const float *q, int S, int Hq, float sc,
                        int window, float *out, float *part, int B, int fuse) {
    switch (c.dh / 32) {
    case 1: at_launch<TYPE, 1>(st, grid, c, r, q, S, Hq, sc, window, out, part, B, fuse); break;
    case 2: at_launch<TYPE, 2>(st, grid, c, r, q, S, Hq, sc, window, out, part, B, fuse); break;
    case 3: at_launch<TYPE, 3>(st, grid, c, r, q, S, Hq, sc, window, out, part, B, fuse); break;
    case 4: at_launch<TYPE, 4>(st, grid, c, r, q, S, Hq, sc, window, out, part, B, fuse); break;
    case 5: at_launch<TYPE, 5>(st, grid, c, r, q, S, Hq, sc, window, out, part, B, fuse); break;
    case 6: at_launch<TYPE, 6>(st, grid, c, r, q, S, Hq, sc, window, out, part, B, fuse); break;
    case 7: at_launch<TYPE, 7>(st, grid, c, r, q, S, Hq, sc, window, out, part, B, fuse); break;
    default: at_launch<TYPE, 8>(st, grid, c, r, q, S, Hq, sc, window, out, part, B, fuse); break;
    }
}

int sw_launch_attn(hipStream_t st, const SwKv &c, const SwRows &r, const float *q, int Hq, float scale, int window, float *out,
                   int S, float *part) {
    if (c.dh < 32 || c.dh > 256 || c.dh % 32) return -1;
    const int B = at_blocks(c, r, Hq, window, S);
    const int64_t grid = (int64_t)B * c.Hkv * ((Hq / c.Hkv + 15) / 16);
    if ((int64_t)S * Hq >= (int64_t)1 << 31 || grid >= (int64_t)1 << 31 || (B > 1 && S <= AT_COUNT && !part))
        return -1;
    const float sc = (float)((double)scale * 1.4426950408889634074);   // the softmax in powers of two
    // over more blocks the join in the same launch pays where no row can have many parts: below 72 KB of them (112
    // rows of one token, 3 cache heads of 96: 13.2 -> 8.5 us; 8 rows, 13 parts of 12 heads of 128, 80 KB: 19.2 ->
    // 20.1), 160 KB of many rows (32 rows, 23 parts of 8 heads of 192, 138 KB: 56.1 -> 52.8)
    const int G = Hq / c.Hkv, nh = G < 16 ? G : 16;
    const int64_t mx = at_cells(c, r, window) / at_chunk(c.type, c.dh) + 1;              // chunks of the longest row there can be
    const int64_t parts = mx / at_least(mx, G, c.dh) + 2;
    const int fuse = B <= AT_FUSE || S > AT_COUNT || (parts <= AT_FUSE && parts * nh * c.dh <= (S < 32 ? 18432 : 40960));
    if (c.type == SW_KV_F32) at_dispatch<SW_KV_F32>(st, (unsigned)grid, c, r, q, S, Hq, sc, window, out, part, B, fuse);
    else if (c.type == SW_KV_BF16) at_dispatch<SW_KV_BF16>(st, (unsigned)grid, c, r, q, S, Hq, sc, window, out, part, B, fuse);
    else at_dispatch<SW_KV_F16>(st, (unsigned)grid, c, r, q, S, Hq, sc, window, out, part, B, fuse);
    if (!fuse)
        SW_LAUNCH(k_attn_join, dim3((unsigned)(S * Hq)), dim3(AT_NT), 0, st, c, r, S, Hq, window, at_chunk(c.type, c.dh), part, B, out);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
