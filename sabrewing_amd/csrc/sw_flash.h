// sw_flash.h -- one pass of a softmax over cells staged in LDS, for a wave's 32 columns.
//
// A column is a query (a head of a row).  A wave holds 32 of them in registers and takes the cells in
// tiles of 32 tokens, both products on the 32 x 32 matrix instructions:
//   scores   S[token][column] = K . Q     (16 registers: column l % 32, token 8 (j / 4) + 4 (l / 32) + j % 4)
//   outputs  O[value][column] += V^T . P  (the scores' layout is the right operand as it stands: the order
//            of the summed index is free, so a lane's 16 weights stay where they are)
// The tiles come from memory straight into LDS, without registers between, several ahead of the
// one in work.  Of a row's 16-byte pieces, piece i of token t lies at i ^ x(t), so that neither the scores'
// reads (one piece of 32 tokens) nor the outputs' (32 pieces of a token) meet on a bank; the
// loading lanes pick their source address accordingly.  An output's operand wants 8 tokens of a value
// where memory has 8 values of a token: a lane reads 8 x 8 and transposes them by byte permutations.
//
// The waves of a block share columns, tokens or values: WC of them have 32 columns each and read
// the same tile, and 4 / WC groups of them take every (4 / WC)-th tile.  Or (SPLIT > 1, where queries and outputs of a cell's width
// do not fit a wave's registers) SPLIT waves have the same columns: each takes a share of the scores' sums, which they exchange
// through LDS, and of the outputs' values.
#ifndef SW_FLASH_H
#define SW_FLASH_H
#include "sw_attn.h"

typedef float fl_f32x16 __attribute__((ext_vector_type(16)));

#define FL_NT 256
#define FL_NW 4

__device__ __forceinline__ int fl_uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t fl_uni(int64_t x) {
    return (int64_t)(((uint64_t)(uint32_t)fl_uni((int)(x >> 32)) << 32) | (uint32_t)fl_uni((int)x));
}
__device__ __forceinline__ float fl_max2(float x) {                    // over the two lanes of a column
    const uint2 a = sw_pair<32>(__builtin_bit_cast(uint32_t, x));
    return fmaxf(__builtin_bit_cast(float, a.x), __builtin_bit_cast(float, a.y));
}
__device__ __forceinline__ float fl_sum2(float x) {
    const uint2 a = sw_pair<32>(__builtin_bit_cast(uint32_t, x));
    return __builtin_bit_cast(float, a.x) + __builtin_bit_cast(float, a.y);
}
template <int TYPE>
__device__ __forceinline__ fl_f32x16 fl_mfma(sw_u32x4 a, sw_u32x4 b, fl_f32x16 c) {
    if constexpr (TYPE == SW_KV_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(sw_bf16x8, a), __builtin_bit_cast(sw_bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(sw_half8, a), __builtin_bit_cast(sw_half8, b), c, 0, 0, 0);
}

// 16 bytes of each lane's address into LDS, lane l's at `lds` + 16 l.  The wave counts the load
// with its others (vmcnt); fl_wait waits for all but the last N.
__device__ __forceinline__ void fl_load16(const void *g, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(lds), "v"(g) : "memory");
}
template <int N> __device__ __forceinline__ void fl_wait() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }
__device__ __forceinline__ void fl_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t fl_lds_addr(const void *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)p;
}
static __device__ const sw_u32x4 g_fl_zero = {0, 0, 0, 0};             // the source of pieces that a cell does not have

// A token's page: entries of the table are read through the scalar cache (a vector load would wait for every
// tile on its way).  p[k] is the page of tokens t0 + 8 k .. + 7 of a tile, -1 where it leads nowhere.
struct FlPages { int p[4]; bool ok; };
__device__ __forceinline__ int fl_entry(const int *table, int i) {
    int x;
    const int *a = table + i;
    asm volatile("s_load_dword %0, %1, 0x0\n\ts_waitcnt lgkmcnt(0)" : "=s"(x) : "s"(a) : "memory");
    return x;
}
__device__ __forceinline__ FlPages fl_pages(const int *table, int max_pages, int n_pages, int psh, int t0) {
    FlPages g;
    g.ok = true;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (k == 0 || psh == 3 || (psh == 4 && k == 2)) {
            const int i = (t0 + 8 * k) >> psh;
            int x = -1;
            if (i < max_pages) x = fl_entry(table, i);
            g.p[k] = x >= 0 && x < n_pages ? x : -1;
            g.ok = g.ok && g.p[k] >= 0;
        } else {
            g.p[k] = g.p[k - 1];
        }
    }
    return g;
}

// parts of 8 values: one (to nearest), three bf16 (by truncation, each takes the next 8 bits: exact) or two f16
template <int TYPE, int NP>
__device__ __forceinline__ void fl_split(const float (&x)[8], sw_u32x4 (&o)[NP]) {
    if constexpr (NP == 1) {
        if constexpr (TYPE == SW_KV_BF16) {
            sw_bf16x8 h;
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = (__bf16)x[i];
            o[0] = __builtin_bit_cast(sw_u32x4, h);
        } else {
            sw_half8 h;
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = (_Float16)x[i];
            o[0] = __builtin_bit_cast(sw_u32x4, h);
        }
    } else if constexpr (TYPE == SW_KV_BF16) {
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

// A wave's 32 columns.  NP: parts that a 32-bit q and the weights are split into (1: 16-bit queries, one
// rounding of the weights).  DK: values of a query, a multiple of 32; DV: of an output; INK: a cell's
// first DV values of k are its v.  AHEAD: dwords of a row that a lane reads at once (8 rows of them), and twice the scores' steps read
// ahead: registers for it.
template <int TYPE, int NP, int DK, int DV, bool INK, int SPLIT = 1, int AHEAD = 4>
struct Fl {
    static constexpr bool F32 = TYPE == SW_KV_F32;
    static constexpr int ES = F32 ? 4 : 2, RBK = DK * ES, RBV = INK ? RBK : DV * ES;                   // bytes of a row of k, of v
    static constexpr int NCK = RBK / 16, NCV = DV * ES / 16;
    static constexpr int TB = 32 * RBK + (INK ? 0 : 32 * RBV);                                         // bytes of a tile
    static constexpr int DKS = RBK / 32 / SPLIT, DVW = DV / SPLIT, NO = DVW / 32, VB = DVW * ES;       // a wave's share: steps of the scores, values
    static_assert(RBK / 32 % SPLIT == 0 && (SPLIT == 1 || (DVW % 64 == 0 && RBK % 128 == 0)), "whole shares");
    static constexpr int XB = SPLIT > 1 ? 4096 : 0;                                                    // bytes of a wave in the exchange
    // where a piece of a row lies: its low bits turned by the token
    static constexpr int MK = NCK % 8 == 0 ? 7 : 3, MV = INK ? MK : NCV % 8 == 0 ? 7 : 3;
    template <int M> static __device__ __forceinline__ int turn(int t) { return M == 7 ? t & 7 : (t >> 1) & 3; }
    // weights are kept below 2^OFF; a maximum may lag behind by LAG powers of two (a running maximum that grows costs a pass
    // over the outputs; 16-bit weights hold 2^8 as well as 1, in parts they may not)
    static constexpr float LAG = NP == 1 && !F32 ? 8.f : 0.f;
    static constexpr float OFF = TYPE != SW_KV_F16 ? 0.f : NP == 1 ? 7.f : 13.f;

    sw_u32x4 Q[F32 ? 1 : NP][DKS];
    fl_f32x16 O[NO];
    float m, l, sc;
    static constexpr int KB = MK == 3 ? 2 : 4 / SPLIT;                 // this lane's places in a tile's row of k: they repeat
    int kb[KB], share;                                                 // after KB steps (every SPLIT-th is the wave's)

    __device__ __forceinline__ void begin(float scale, int share_ = 0) {
        const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
        m = -INFINITY;
        l = 0.f;
        sc = scale;
#pragma unroll
        for (int i = 0; i < NO; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) O[i][j] = 0.f;
#pragma unroll
        for (int i = 0; i < KB; i++) kb[i] = c * RBK + (((2 * (SPLIT * i + share_) + h) ^ turn<MK>(c)) * 16);
        share = share_;
    }
    // 8 values 16 i + 8 h .. of a 32-bit query (f32 cells: 4 of them, 8 i + 4 h ..); f16 in parts: called after scale_up
    __device__ __forceinline__ void query(int i, const float (&x)[8]) {
        if constexpr (!F32) {
            sw_u32x4 o[NP];
            fl_split<TYPE, NP>(x, o);
#pragma unroll
            for (int u = 0; u < NP; u++) Q[u][i] = o[u];
        }
    }

    // the scores of the tile at `t`, times the scale
    __device__ __forceinline__ void scores(const char *t, float (&x)[16], char *xch, int wave) const {
        fl_f32x16 s = {};
#pragma unroll
        for (int i = 0; i < DKS; i++) {
            const sw_u32x4 a = *(const sw_u32x4 *)(t + kb[i % KB] + i / KB * (KB * SPLIT * 32));
            if constexpr (F32) {
                const sw_f32x4 y = __builtin_bit_cast(sw_f32x4, a), z = __builtin_bit_cast(sw_f32x4, Q[0][i]);
#pragma unroll
                for (int e = 0; e < 4; e++) s = __builtin_amdgcn_mfma_f32_32x32x2f32(y[e], z[e], s, 0, 0, 0);
            } else {
#pragma unroll
                for (int u = 0; u < NP; u++) s = fl_mfma<TYPE>(a, Q[u][i], s);
            }
            if (i % (2 * AHEAD) == 2 * AHEAD - 1) __builtin_amdgcn_sched_barrier(0);     // (reads of the whole row ahead would spill)
        }
        if constexpr (SPLIT > 1) {                                     // the shares in their order: the same sum in every wave
            sw_f32x4 *to = (sw_f32x4 *)xch + (threadIdx.x & 63);
#pragma unroll
            for (int j = 0; j < 4; j++) to[(wave * 4 + j) * 64] = sw_f32x4{s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]};
            __syncthreads();
            const int w0 = wave - share;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                sw_f32x4 y = to[(w0 * 4 + j) * 64];
#pragma unroll
                for (int k = 1; k < SPLIT; k++) {
                    const sw_f32x4 z = to[((w0 + k) * 4 + j) * 64];
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] = y[e] + z[e];
                }
#pragma unroll
                for (int e = 0; e < 4; e++) s[4 * j + e] = y[e];
            }
        }
#pragma unroll
        for (int j = 0; j < 16; j++) x[j] = s[j] * sc;
    }

    // scores (masked ones -INFINITY) to weights; the outputs follow a maximum that grew
    __device__ __forceinline__ void weights(float (&x)[16]) {
        float mx = x[0];
#pragma unroll
        for (int j = 1; j < 16; j++) mx = fmaxf(mx, x[j]);
        const float nm = fl_max2(mx);
        if (__any(nm > m + LAG)) {
            const float n = fmaxf(m, nm), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - n);
            l = l * f;
#pragma unroll
            for (int i = 0; i < NO; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) O[i][j] = O[i][j] * f;
            m = n;
        }
        const float base = m == -INFINITY ? 0.f : m - OFF;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            x[j] = __builtin_amdgcn_exp2f(x[j] - base);
            l = l + x[j];
        }
    }

    static __device__ __forceinline__ uint32_t infinite(uint32_t w) {   // all ones in the halves (or whole) that are no finite number
        if constexpr (F32) return (w & 0x7F800000u) == 0x7F800000u ? 0xFFFFFFFFu : 0u;
        constexpr uint32_t E = TYPE == SW_KV_BF16 ? 0x7F80u : 0x7C00u;
        return ((w & E) == E ? 0xFFFFu : 0u) | ((w & (E << 16)) == E << 16 ? 0xFFFF0000u : 0u);
    }

    // O += V^T P
    __device__ __forceinline__ void outputs(const char *t, const float (&p)[16]) {
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));                                 // (the places are taken anew for each tile, not kept)
        const int c = lane & 31, h = lane >> 5;
        if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int x = MV == 7 ? 4 * h + j % 4 : 2 * h + ((j % 4) >> 1);
                group_f32<AHEAD, 0, 0>(t + (8 * (j / 4) + j % 4 + 4 * h) * RBV, x, c, p[j]);
                if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int mm = 0; mm < 2; mm++) {
                float p8[8];
#pragma unroll
                for (int j = 0; j < 8; j++) p8[j] = p[8 * mm + j];
                sw_u32x4 P[NP];
                fl_split<TYPE, NP>(p8, P);
                group<AHEAD, 0, 0>(t + 16 * mm * RBV + 4 * h * RBV, c, h, P);
            }
        }
    }
    // Infinities and NaN among the values of a tile's v, in wave w of n's share, become 0 (a weight of 0 times one of them is none);
    // the tokens that had one are marked in `bad`.
    static __device__ __forceinline__ void clean(char *t, int w, int n, uint32_t *bad) {
        char *v = INK ? t : t + 32 * RBK;
        uint32_t met = 0;
#pragma unroll 1
        for (int i = w * 64 + (threadIdx.x & 63); i < 32 * NCV; i += n * 64) {
            const int tok = i / NCV;
            sw_u32x4 *a = (sw_u32x4 *)(v + tok * RBV + (i - tok * NCV) * 16);
            sw_u32x4 y = *a;
            uint32_t any = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t x = infinite(y[e]);
                any |= x;
                y[e] = y[e] & ~x;
            }
            if (any) { *a = y; met |= 1u << tok; }
        }
        if (met) atomicOr(bad, met);
    }
    // the values from byte B0 on (output tiles from O0 on), W dwords of a row a lane
    template <int W, int B0, int O0>
    __device__ __forceinline__ void group(const char *t, int c, int h, const sw_u32x4 (&P)[NP]) {
        if constexpr (B0 + 32 * 4 * W <= VB) {
            uint32_t v[8][W];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int x = MV == 7 ? 4 * h + k % 4 : 2 * h + ((k % 4) >> 1);
                const char *a = t + (8 * (k / 4) + k % 4) * RBV + B0 + (((c * W / 4) ^ x) * 16 + (c * W % 4) * 4);
                if constexpr (W == 4) {
                    const sw_u32x4 y = *(const sw_u32x4 *)a;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[k][e] = y[e];
                } else if constexpr (W == 2) {
                    const uint2 y = *(const uint2 *)a;
                    v[k][0] = y.x; v[k][1] = y.y;
                } else v[k][0] = *(const uint32_t *)a;
            }
#pragma unroll
            for (int e = 0; e < 2 * W; e++) {
                sw_u32x4 a;
#pragma unroll
                for (int i = 0; i < 4; i++) a[i] = __builtin_amdgcn_perm(v[2 * i + 1][e / 2], v[2 * i][e / 2], e & 1 ? 0x07060302 : 0x05040100);
#pragma unroll
                for (int u = 0; u < NP; u++) O[O0 + e] = fl_mfma<TYPE>(a, P[u], O[O0 + e]);
            }
            __builtin_amdgcn_sched_barrier(0);
            group<W, B0 + 128 * W, O0 + 2 * W>(t, c, h, P);
        } else if constexpr (W > 1) {
            group<W / 2, B0, O0>(t, c, h, P);
        } else if constexpr (B0 < VB) {                                // 32 values left: two bytes a lane
            uint32_t v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int x = MV == 7 ? 4 * h + k % 4 : 2 * h + ((k % 4) >> 1);
                v[k] = *(const uint16_t *)(t + (8 * (k / 4) + k % 4) * RBV + B0 + (((c / 8) ^ x) * 16 + c % 8 * 2));
            }
            sw_u32x4 a;
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = v[2 * i] | (v[2 * i + 1] << 16);
#pragma unroll
            for (int u = 0; u < NP; u++) O[O0] = fl_mfma<TYPE>(a, P[u], O[O0]);
        }
    }
    template <int W, int B0, int O0>
    __device__ __forceinline__ void group_f32(const char *row, int x, int c, float p) {
        if constexpr (B0 + 32 * 4 * W <= VB) {
            uint32_t v[W];
            const char *a = row + B0 + (((c * W / 4) ^ x) * 16 + (c * W % 4) * 4);
            if constexpr (W == 4) {
                const sw_u32x4 y = *(const sw_u32x4 *)a;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = y[e];
            } else if constexpr (W == 2) {
                const uint2 y = *(const uint2 *)a;
                v[0] = y.x; v[1] = y.y;
            } else v[0] = *(const uint32_t *)a;
#pragma unroll
            for (int e = 0; e < W; e++)
                O[O0 + e] = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(float, v[e]), p, O[O0 + e], 0, 0, 0);
            group_f32<W, B0 + 128 * W, O0 + W>(row, x, c, p);
        } else if constexpr (W > 1) group_f32<W / 2, B0, O0>(row, x, c, p);
    }

    // One tile.  whole: every column attends to all of its tokens, else seen(token of the tile) says it for this lane's column, and bit k of
    // bad that token k's v is no number: whoever attends to it has no meaningful output.
    template <class Seen>
    __device__ __forceinline__ void tile(const char *t, bool whole, uint32_t bad, Seen seen, char *xch, int wave) {
        float x[16];
        scores(t, x, xch, wave);
        if (!whole) {
            const int h4 = (threadIdx.x & 32) >> 3;
            uint32_t met = 0;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int k = 8 * (j / 4) + h4 + j % 4;
                const bool s = seen(k);
                if (!s) x[j] = -INFINITY;
                else met |= bad >> k & 1;
            }
            if (met) l = NAN;
        }
        weights(x);
        outputs((INK ? t : t + 32 * RBK) + (SPLIT > 1 ? share * VB : 0), x);
    }

    // Where an output's values lie: tile o's row r is value d0 + T r + e of a group of values that T tiles share (groups of 256
    // values (f32: 128), 128, 64 and 32), tile o being its e-th.
    struct Map { int d0[NO], tiles[NO], e[NO]; };
    static constexpr Map map() {
        Map m = {};
        int d = 0, w = F32 ? AHEAD : 2 * AHEAD;
        for (int at = 0; at < NO; at += w) {
            while (d + 32 * w > DVW) w /= 2;
            for (int e = 0; e < w; e++) { m.d0[at + e] = d; m.tiles[at + e] = w; m.e[at + e] = e; }
            d += 32 * w;
        }
        return m;
    }
};

// A block's work on one item: tiles ta .. tb - 1, dealt to its WT groups of waves in turn; NS tiles of a group in LDS (`sh`).
// issue(tile, LDS address): the wave's share of a tile's loads, NL of them, and whether every page of it is there;
// whole(tile) (alike in the waves that share a tile), seen(tile, token): the mask; columns: this wave has some (with SPLIT every
// wave takes part); xch: LDS of the exchange; s_bad: two words a group.
template <int WC, int WT, int SPLIT, int NS, int NL, class F, class Issue, class Whole, class Seen>
__device__ __forceinline__ void fl_run(F &f, char *sh, char *xch, uint32_t *s_bad, int ta, int tb, int wave, bool columns, Issue issue, Whole whole, Seen seen) {
    static_assert(WT == 1 || SPLIT == 1, "groups of waves do not exchange");
    constexpr int TB = F::TB;
    constexpr bool shared = WC * SPLIT > 1;
    const int wt = WT == 1 ? 0 : wave / WC, all = (tb - ta + WT - 1) / WT, n = (tb - ta - wt + WT - 1) / WT;     // tiles of the longest group, of this one
    char *mine = sh + wt * NS * TB;
    s_bad += 2 * wt;
    const uint32_t lds = fl_lds_addr(mine);
    const bool first = (threadIdx.x & 63) == 0 && (WT > 1 && WC == 1 ? true : wave % (WC * SPLIT) == 0);       // of its group
    if (first) s_bad[0] = 0;                                           // (the item before is done with it)
    uint32_t there = 0;                                                // bit s: all pages of the tile in place s are there
    auto load = [&](int i, int s) {
        const bool ok = issue(ta + wt + i * WT, lds + s * TB);
        there = ok ? there | 1u << s : there & ~(1u << s);
    };
#pragma unroll 1
    for (int i = 0; i < NS - 1; i++)
        if (i < n) load(i, i);
    int s = 0;                                                         // the place of tile i
#pragma unroll 1
    for (int i = 0; i < all; i++) {
        if (NS == 1) {
            if (shared) __syncthreads();                               // (every wave of the group has read the tile before)
            else fl_wait_lds();
            if (i < n) load(i, 0);
        }
        if (NS < 3 || i + NS - 2 >= n) fl_wait<0>();
        else fl_wait<(NS < 3 ? 0 : NS - 2) * NL>();
        const int t = ta + wt + i * WT;
        const bool whl = i >= n || (((there >> s) & 1) && whole(t));
        bool all_whole = whl;
        if (!shared) fl_wait_lds();
        else if (WT > 1) all_whole = __syncthreads_and(whl);
        else __syncthreads();
        if (NS > 1 && i + NS - 1 < n) load(i + NS - 1, s == 0 ? NS - 1 : s - 1);
        if (first) s_bad[(i + 1) & 1] = 0;
        uint32_t bad = 0;
        if (!all_whole) {
            if (!whl) f.clean(mine + s * TB, WT == 1 ? wave : wave % WC, WC * SPLIT, s_bad + (i & 1));
            if (shared) __syncthreads();
            else fl_wait_lds();
            bad = s_bad[i & 1];
        }
        if (SPLIT > 1 || (i < n && columns)) f.tile(mine + s * TB, whl, bad, [&](int k) { return seen(t, k); }, xch, wave);
        s = s + 1 == NS ? 0 : s + 1;
    }
}

// The end of an item: the groups' outputs of a column joined in their order and given to put(column, value, four
// outputs, maximum, sum).  sh: LDS of fl_end_bytes, free.
template <class F, int NW>
constexpr int fl_end_bytes() { return NW * 32 * (F::DVW / 4 + 4) * 4; }
template <int WC, int WT, int SPLIT, class F, class Put>
__device__ __forceinline__ void fl_end(F &f, char *sh, float (*s_m)[32], float (*s_l)[32], int wave, Put put) {
    constexpr int DVW = F::DVW, LD = DVW / 4 + 4, NO = F::NO, NT = WC * WT * SPLIT * 64;
    constexpr auto map = F::map();
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
    const float l = fl_sum2(f.l);
    __syncthreads();                                                   // the tiles are done with
    if (h == 0) { s_m[wave][c] = f.m; s_l[wave][c] = l; }
    __syncthreads();
    float g = 1.f;
    if constexpr (WT > 1) {
        float M = f.m;
#pragma unroll
        for (int i = 0; i < WT; i++) M = fmaxf(M, s_m[i * WC + wave % WC][c]);
        g = f.m == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(f.m - M);
    }
    float *so = (float *)sh + (wave * 32 + c) * LD;
#pragma unroll
    for (int q = 0; q < 4; q++) {
#pragma unroll
        for (int o = 0; o < NO; o++) {
            const int T = map.tiles[o], at = map.d0[o] / 4 + map.e[o];
#pragma unroll
            for (int j = 0; j < 4; j++) so[at + T * (4 * h + j)] = WT > 1 ? f.O[o][4 * q + j] * g : f.O[o][4 * q + j];
        }
        __syncthreads();
        // (column, share, four values): the shares of a column are waves side by side
#pragma unroll 1
        for (int i = tid; i < WC * 32 * SPLIT * (DVW / 16); i += NT) {
            const int v = i % (SPLIT * (DVW / 16)), col = i / (SPLIT * (DVW / 16)), sp = v / (DVW / 16), d = v % (DVW / 16) * 4;
            const int w = (col >> 5) * SPLIT + sp;
            sw_f32x4 a = *(const sw_f32x4 *)((const float *)sh + (w * 32 + (col & 31)) * LD + d);
            float mx = s_m[w][col & 31], sum = s_l[w][col & 31];
            if constexpr (WT > 1) {
#pragma unroll
                for (int k = 1; k < WT; k++) {
                    const sw_f32x4 y = *(const sw_f32x4 *)((const float *)sh + ((w + k * WC) * 32 + (col & 31)) * LD + d);
#pragma unroll
                    for (int e = 0; e < 4; e++) a[e] = a[e] + y[e];
                    mx = fmaxf(mx, s_m[w + k * WC][col & 31]);
                }
                sum = 0.f;
#pragma unroll
                for (int k = 0; k < WT; k++) {
                    const float x = s_m[w + k * WC][col & 31];
                    sum = __builtin_fmaf(s_l[w + k * WC][col & 31], x == -INFINITY ? (mx == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(x - mx), sum);
                }
            }
            // the quarter's value d: which group of values it is in
            int d0 = 0, T8 = 0;
#pragma unroll
            for (int o = 0; o < NO; o++)
                if (map.e[o] == 0 && map.d0[o] / 4 <= d) { d0 = map.d0[o]; T8 = map.tiles[o] * 8; }
            put(col, sp * DVW + d0 + T8 * q + d - d0 / 4, a, mx, sum);
        }
        __syncthreads();
    }
}

// How items' tiles are dealt to B blocks: laid end to end they are N, and block b takes those from b q to (b + 1) q, whatever
// items they fall in.  count(i): the tiles of item i (evaluated 64 items at a time, a lane each).  `least`: no fewer
// tiles a block.
struct FlDeal { int64_t N, q; };
template <class Count>
__device__ __forceinline__ FlDeal fl_deal(int items, int B, int least, Count count) {
    const int lane = threadIdx.x & 63;
    FlDeal d = {0, 0};
    for (int i0 = 0; i0 < items; i0 += 64)
        d.N += (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)sw_wave_scan(i0 + lane < items ? (uint32_t)count(i0 + lane) : 0u), 63);
    d.q = (d.N + B - 1) / B;
    if (d.q < least) d.q = least;
    return d;
}
// the item in which tile `at` (below N) of all lies, and the tiles of items before it
template <class Count>
__device__ __forceinline__ int fl_find(int items, int64_t at, int64_t &before, Count count) {
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    for (int i0 = 0;; i0 += 64) {
        const uint32_t n = i0 + lane < items ? (uint32_t)count(i0 + lane) : 0u, upto = sw_wave_scan(n);
        const int64_t all = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        if (base + all > at || i0 + 64 >= items) {
            const int i = __builtin_ctzll(__ballot((int64_t)upto > at - base) | (1ull << 63));
            before = base + (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(upto - n), i);
            return i0 + i;
        }
        base += all;
    }
}
// the tiles of items before item i
template <class Count>
__device__ __forceinline__ int64_t fl_before(int i, Count count) {
    const int lane = threadIdx.x & 63;
    int64_t n = 0;
    for (int i0 = 0; i0 < i; i0 += 64)
        n += (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)sw_wave_scan(i0 + lane < i ? (uint32_t)count(i0 + lane) : 0u), 63);
    return n;
}
#endif
