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
// where memory has 8 values of a token: transposing reads bring them so.
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
// the lane, for places in LDS that are taken anew for each tile: kept, they would take the registers that the queries need
template <bool KEEP = false>
__device__ __forceinline__ int fl_lane() {
    int lane = threadIdx.x & 63;
    if (!KEEP) asm volatile("" : "+v"(lane));
    return lane;
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
// the same from a scalar base and a lane's 32-bit offset
__device__ __forceinline__ void fl_load16(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds), "v"(off), "s"(base) : "memory");
}
template <int N> __device__ __forceinline__ void fl_wait() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }
__device__ __forceinline__ void fl_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t fl_lds_addr(const void *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)p;
}
// LDS at an address (tiles begin on 256 bytes, so that a piece's turn is an exclusive or of the whole address)
template <class T> __device__ __forceinline__ T fl_lds(uint32_t a) { return *(const __attribute__((address_space(3))) T *)(uintptr_t)a; }
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

// By how much (an exclusive or) a row's pieces are turned in LDS, whose 64 banks are 16 pieces.  The scores read one piece of 16 tokens at a time: M 15, 7
// and 3 for rows of whole 256 bytes, odd 128 and odd 64 (where 1, 2 and 4 rows begin on different banks by themselves).  The outputs read four pieces
// of four tokens: 12, 4 and 0 for the same rows; 7 does for them too, where one row serves both.  Each is linear in t's bits.
template <int M>
__device__ __forceinline__ constexpr int fl_turn(int t) {
    return M == 15 ? t & 15 : M == 7 ? (t & 2) << 1 | (t & 4) >> 1 | (t & 8) >> 3 : M == 3 ? (t >> 2) & 3 : M == 12 ? 4 * (t & 3) : M == 4 ? 2 * (t & 2) : 0;
}
// Rows of NCH 16-byte pieces from `base` on, `step` bytes apart (below 2^26), into a tile at `to`: wave w of W's share, N loads of it.
// M: the pieces' turn by token.
template <int NCH, int M, int W, int N>
__device__ __forceinline__ void fl_rows(const char *base, uint32_t step, int w, int lane, uint32_t to) {
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int kk = (N * W > NCH / 2) ? min(k * W + w, NCH / 2 - 1) : k * W + w;
        if constexpr (64 % NCH == 0) {                                 // a load is some whole rows: a part of the turn is the wave's
            constexpr int RP = 64 / NCH;
            const uint32_t off = lane / NCH * step + ((lane % NCH ^ fl_turn<M>(lane / NCH) ^ fl_turn<M>(kk * RP)) * 16);
            fl_load16(base + (int64_t)kk * RP * step, off, to + kk * 1024);
        } else {
            const int p = kk * 64 + lane, tok = p / NCH, ch = (p - tok * NCH) ^ fl_turn<M>(tok);
            fl_load16(base, tok * step + ch * 16, to + kk * 1024);
        }
    }
}
// The same from pages that end inside the tile, or rows far apart or shorter than the tile's (real pieces of them, then zeros): cell
// of token t0 + k in page g.p[k / 8].
template <int NCH, int M, int W, int N>
__device__ __forceinline__ void fl_rows_any(const char *pool, const FlPages &g, int64_t page, int64_t step, int t0, int pmask, int real, int w, int lane,
                                            uint32_t to) {
#pragma unroll 1
    for (int k = 0; k < N; k++) {
        const int kk = min(k * W + w, NCH / 2 - 1), p = kk * 64 + lane, tok = p / NCH, ch = (p - tok * NCH) ^ fl_turn<M>(tok);
        const int g01 = tok & 8 ? g.p[1] : g.p[0], g23 = tok & 8 ? g.p[3] : g.p[2], x = tok & 16 ? g23 : g01;
        const char *a = pool + (int64_t)max(x, 0) * page + (int64_t)((t0 + tok) & pmask) * step + ch * 16;
        fl_load16(ch < real ? a : (const char *)&g_fl_zero, to + kk * 1024);
    }
}

// x plus two 16-bit values
template <int TYPE>
__device__ __forceinline__ float fl_sum(uint32_t w, float x) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    if constexpr (TYPE == SW_KV_BF16) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w), b2{(__bf16)1.f, (__bf16)1.f}, x, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(sw_half2, w), sw_half2{(_Float16)1.f, (_Float16)1.f}, x, false);
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
// rounding of the weights; k_latent.hip says what it costs and saves).  DK: values of a query, a multiple of 32; DV: of an output; INK: a cell's
// first DV values of k are its v.  How much is read ahead of the products goes by the registers that queries and outputs leave: a
// spilled one is a load in the loop, and waiting for it waits for every tile on its way (k_tree.hip: where that is so).
template <int TYPE, int NP, int DK, int DV, bool INK, int SPLIT = 1>
struct Fl {
    static constexpr bool F32 = TYPE == SW_KV_F32;
    static constexpr int AHEAD = 2;                                    // f32 cells: dwords of a row that a lane reads at once, 4 rows of them
    static constexpr int ES = F32 ? 4 : 2, RBK = DK * ES, RBV = INK ? RBK : DV * ES;                   // bytes of a row of k, of v
    static constexpr int NCK = RBK / 16, NCV = DV * ES / 16;
    static constexpr int TB = 32 * RBK + (INK ? 0 : 32 * RBV);                                         // bytes of a tile
    static constexpr int DKS = RBK / 32 / SPLIT, DVW = DV / SPLIT, NO = DVW / 32, VB = DVW * ES;       // a wave's share: steps of the scores, values
    static_assert(RBK / 32 % SPLIT == 0 && (SPLIT == 1 || (DVW % 64 == 0 && RBK % 128 == 0)), "whole shares");
    static_assert(SPLIT == 1 || SPLIT == 2 || SPLIT == 4, "pairs");
    static constexpr int HELD = (F32 ? 1 : NP) * DKS * 4 + NO * 16;
    static constexpr bool KEEP = HELD <= 128;                          // room for places in LDS
    static constexpr int PIPE = HELD <= 144 ? 2 : 1, QB = HELD <= 144 && NP == 1 && !F32 ? 4 : 2, VT = HELD <= 144 ? 4 : 2;
    // bytes of a wave in the exchange, and of 32 columns: a share's sums of scores; the columns' weights and maxima
    static constexpr int XB = SPLIT > 1 ? 4096 + (2048 + SPLIT * 128) / SPLIT + 16 : 0;
    // how a row's pieces are turned
    static constexpr int MK = NCK % 16 == 0 ? 15 : NCK % 8 == 0 ? 7 : 3;
    static constexpr int MV = INK ? MK : F32 ? (NCV % 16 == 0 ? 15 : NCV % 8 == 0 ? 7 : 3) : NCV % 16 == 0 ? 12 : NCV % 8 == 0 ? 4 : 0;
    static_assert(!INK || MK == 7, "a turn that serves both reads");
    // weights are kept below 2^OFF; a maximum may lag behind by LAG powers of two (a running maximum that grows costs a pass
    // over the outputs; 16-bit weights hold 2^8 as well as 1, in parts they may not)
    static constexpr float LAG = NP == 1 && !F32 ? 8.f : 0.f;
    static constexpr float OFF = TYPE != SW_KV_F16 ? 0.f : NP == 1 ? 7.f : 13.f;

    sw_u32x4 Q[F32 ? 1 : NP][DKS];
    fl_f32x16 O[NO];
    float m, l, sc;
    static constexpr int KB = MK == 3 ? 2 : (MK == 15 ? 8 : 4) / SPLIT;// a lane's places in a tile's row of k repeat after KB steps
    int share;                                                         // (every SPLIT-th step is the wave's)

    // scale: of the scores, in powers of two.  Its sign (and a scale of 0) goes into the queries, see query().
    __device__ __forceinline__ void begin(float scale, int share_ = 0) {
        m = -INFINITY;
        l = 0.f;
        sc = scale == 0.f ? 1.f : fabsf(scale);
#pragma unroll
        for (int i = 0; i < NO; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) O[i][j] = 0.f;
        share = share_;
    }
    static __device__ __forceinline__ uint32_t signed_by(uint32_t w, float scale) {   // two 16-bit values (or one of 32) times the scale's sign
        return scale == 0.f ? 0u : scale < 0.f ? w ^ (F32 ? 0x80000000u : 0x80008000u) : w;
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

    // the scores of the tile at `t` (a wave's share of their sums), not yet times the scale, added to s
    __device__ __forceinline__ void dot(const char *t, fl_f32x16 &s) const {
        // QB steps' operands are read while the QB before are multiplied
        constexpr int NB = (DKS + QB - 1) / QB;
        const int lane = fl_lane<KEEP>(), c = lane & 31, h = lane >> 5;
        const uint32_t row = fl_lds_addr(t) + c * RBK + (((2 * share + h) ^ fl_turn<MK>(c)) * 16);
        uint32_t kb[KB];
#pragma unroll
        for (int i = 0; i < KB; i++) kb[i] = row ^ (32 * SPLIT * i);
        sw_u32x4 a[2][QB];
        auto read = [&](int b) {
#pragma unroll
            for (int k = 0; k < QB; k++)
                if (b * QB + k < DKS) a[b & 1][k] = fl_lds<sw_u32x4>(kb[(b * QB + k) % KB] + (b * QB + k) / KB * (KB * SPLIT * 32));
        };
        read(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if (b + 1 < NB) read(b + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < QB; k++) {
                const int i = b * QB + k;
                if (i >= DKS) break;
                if constexpr (F32) {
                    const sw_f32x4 y = __builtin_bit_cast(sw_f32x4, a[b & 1][k]), z = __builtin_bit_cast(sw_f32x4, Q[0][i]);
#pragma unroll
                    for (int e = 0; e < 4; e++) s = __builtin_amdgcn_mfma_f32_32x32x2f32(y[e], z[e], s, 0, 0, 0);
                } else {
#pragma unroll
                    for (int u = 0; u < NP; u++) s = fl_mfma<TYPE>(a[b & 1][k], Q[u][i], s);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
    }
    // scores (masked ones -INFINITY) to weights; the outputs follow a maximum that grew.  (16-bit weights are summed as they are rounded, in outputs().)
    static constexpr bool SUMS = !F32 && NP == 1;
    __device__ __forceinline__ void weights(const fl_f32x16 &s, float (&x)[16]) {
        float mx = s[0];
#pragma unroll
        for (int j = 1; j < 16; j++) mx = fmaxf(mx, s[j]);
        const float nm = fl_max2(mx);
        if (__any(LAG == 0.f ? nm > m : (nm - m) * sc > LAG)) {
            const float n = fmaxf(m, nm), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - n) * sc);
            l = l * f;
#pragma unroll
            for (int i = 0; i < NO; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) O[i][j] = O[i][j] * f;
            m = n;
        }
        const float base = m == -INFINITY ? 0.f : OFF - m * sc;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            x[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], sc, base));
            if constexpr (!SUMS) l = l + x[j];
        }
    }

    static __device__ __forceinline__ uint32_t infinite(uint32_t w) {   // all ones in the halves (or whole) that are no finite number
        if constexpr (F32) return (w & 0x7F800000u) == 0x7F800000u ? 0xFFFFFFFFu : 0u;
        constexpr uint32_t E = TYPE == SW_KV_BF16 ? 0x7F80u : 0x7C00u;
        return ((w & E) == E ? 0xFFFFu : 0u) | ((w & (E << 16)) == E << 16 ? 0xFFFF0000u : 0u);
    }

    // O += V^T P.  Operands are read while those before are multiplied; the first are in `first`.
    // 16-bit cells: an operand is 32 values of 16 tokens, 8 of a lane, where memory has the values side by side: two transposing reads, by which 16
    // lanes fetch 4 tokens' 16 values and each gets one value of the four.  VT operands at a time, output tile o values 32 o ...
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    // f32 cells: a lane's piece of a row (AHEAD values) is an operand of as many tiles; four tokens at a time, groups of values by rising width
    static constexpr int NG = NO + 1;
    struct Steps { int n, b0[NG], w[NG], o0[NG]; };
    static constexpr Steps steps() {
        Steps s = {};
        int b = 0, o = 0, w = AHEAD;
        while (b < VB) {
            while (b + 128 * w > VB) w /= 2;
            s.b0[s.n] = b; s.w[s.n] = w; s.o0[s.n] = o; s.n++;
            b += 128 * w;
            o += w;
        }
        return s;
    }
    static constexpr int NST = F32 ? 4 * steps().n : (2 * NO + VT - 1) / VT;
    struct Piece { uint32_t v[F32 ? 4 * AHEAD : 4 * VT]; };
    static __device__ __forceinline__ void read(const char *t, int step, Piece &p) {
        const int lane = fl_lane<KEEP>();
        if constexpr (F32) {
            constexpr Steps S = steps();
            const int lot = step / S.n, g = step % S.n, w = S.w[g], c = lane & 31, h = lane >> 5;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int x = fl_turn<MV>(8 * lot + k) ^ fl_turn<MV>(4 * h);
                const char *row = t + (8 * lot + k + 4 * h) * RBV + S.b0[g];
                if (w == 2) {
                    const uint2 y = *(const uint2 *)(row + ((c >> 1) ^ x) * 16 + (c & 1) * 8);
                    p.v[AHEAD * k] = y.x; p.v[AHEAD * k + 1] = y.y;
                } else p.v[AHEAD * k] = *(const uint32_t *)(row + ((c >> 2) ^ x) * 16 + (c & 3) * 4);
            }
        } else {
            const int k = 4 * (lane >> 5) + ((lane & 15) >> 2), d = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), x = fl_turn<MV>(k);
            const uint32_t row = fl_lds_addr(t) + k * RBV + (lane & 1) * 8 + (d ^ x) * 16;
#pragma unroll
            for (int i = 0; i < VT; i++) {
                const int at = step * VT + i, lot = at / NO, o = at % NO;
                if (at >= 2 * NO) break;
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    constexpr int W = MV == 12 ? 4 : MV == 0 ? 1 : 2;  // (operands of the pieces that are turned among themselves)
                    const uint32_t a = (row ^ (64 * (o % W) ^ 16 * fl_turn<MV>(8 * b))) + (16 * lot + 8 * b) * RBV + 64 * W * (o / W);
                    const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(uintptr_t)a);
                    const uint2 z = __builtin_bit_cast(uint2, y);
                    p.v[4 * i + 2 * b] = z.x; p.v[4 * i + 2 * b + 1] = z.y;
                }
            }
        }
    }
    // (p, or where they are operands already, P)
    typedef sw_u32x4 Weights[2][F32 ? 1 : NP];
    __device__ __forceinline__ void outputs(const char *t, const float (&p)[16], Weights &P, Piece &first) {
        Piece v[PIPE];
        v[0] = first;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < NST; s++) {
            if (PIPE == 1 && s > 0) read(t, s, v[0]);
            if (PIPE == 2 && s + 1 < NST) read(t, s + 1, v[(s + 1) % PIPE]);
            __builtin_amdgcn_sched_barrier(0);
            Piece &y = v[s % PIPE];
            if constexpr (F32) {
                constexpr Steps S = steps();
                const int lot = s / S.n, g = s % S.n;
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int e = 0; e < S.w[g]; e++)
                        O[S.o0[g] + e] = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(float, y.v[AHEAD * k + e]), p[4 * lot + k], O[S.o0[g] + e], 0, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < VT; i++) {
                    const int at = s * VT + i, lot = at / NO, o = at % NO;
                    if (at >= 2 * NO) break;
                    if (o == 0 && SPLIT == 1) {
                        float p8[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) p8[j] = p[8 * lot + j];
                        fl_split<TYPE, NP>(p8, P[lot]);
                        if constexpr (SUMS)
#pragma unroll
                            for (int j = 0; j < 4; j++) l = fl_sum<TYPE>(P[lot][0][j], l);
                    }
                    const sw_u32x4 a = {y.v[4 * i], y.v[4 * i + 1], y.v[4 * i + 2], y.v[4 * i + 3]};
#pragma unroll
                    for (int u = 0; u < NP; u++) O[o] = fl_mfma<TYPE>(a, P[lot][u], O[o]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
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
    // One tile.  whole: every column attends to all of its tokens, else seen(token of the tile) says it for this lane's column, and bit k of
    // bad that token k's v is no number: whoever attends to it has no meaningful output.
    template <class Seen>
    __device__ __forceinline__ void tile(const char *t, bool whole, uint32_t bad, Seen seen) {
        fl_f32x16 s = {};
        dot(t, s);
        alone(t, whole, bad, seen, s);
    }
    template <class Seen>
    __device__ __forceinline__ void alone(const char *t, bool whole, uint32_t bad, Seen seen, fl_f32x16 &s) {
        const char *v = INK ? t : t + 32 * RBK;
        if (!whole) {
            const int h4 = (threadIdx.x & 32) >> 3;
            uint32_t met = 0;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int k = 8 * (j / 4) + h4 + j % 4;
                const bool in = seen(k);
                s[j] = in ? s[j] : -INFINITY;
                met |= in ? bad >> k & 1 : 0u;
            }
            if (met) l = NAN;
        }
        Piece first;
        read(v, 0, first);
        __builtin_amdgcn_sched_barrier(0);
        float x[16];
        Weights P;
        weights(s, x);
        outputs(v, x, P, first);
    }
    // Columns that SPLIT waves share: each wave has a share of the scores' sums of all 32 tokens, which it puts into LDS (sums).  Behind a
    // barrier each takes all sums of its own tokens (QT quads of a lane), makes their weights and puts those into LDS as the outputs'
    // operand, which all read behind another (weigh).  A maximum that grew too far (the waves' lags alike) is rare: then the waves
    // put their maxima there too and make the weights again.
    static constexpr int QT = 4 / SPLIT;
    __device__ __forceinline__ void sums(const char *t, char *xch, int wave) const {
        fl_f32x16 s = {};
        dot(t, s);
        sw_f32x4 *to = (sw_f32x4 *)(xch + (wave - share) * XB) + fl_lane<KEEP>();
#pragma unroll
        for (int j = 0; j < 4; j++) to[(share * 4 + j) * 64] = sw_f32x4{s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]};
    }
    template <class Seen>
    __device__ __forceinline__ void weigh(const char *t, bool whole, uint32_t bad, Seen seen, char *xch, int wave, int odd) {
        static_assert(SPLIT == 1 || SUMS, "16-bit weights");
        const int lane = fl_lane<KEEP>(), c = lane & 31, h4 = (lane & 32) >> 3;
        const char *v = (INK ? t : t + 32 * RBK) + share * VB;
        char *mine = xch + (wave - share) * XB;                        // of the columns: the shares' sums, the weights, the maxima, two flags
        const sw_f32x4 *all = (const sw_f32x4 *)mine + lane;
        uint2 *w = (uint2 *)(mine + SPLIT * 4096) + lane * 2;
        float *top = (float *)(mine + SPLIT * 4096 + 2048) + c;
        int *grew = (int *)(xch + SPLIT * 4096 + 2048 + SPLIT * 128);  // (of all columns: the block's first)
        float x[4 * QT], mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < QT; q++) {
            sw_f32x4 y = all[(share * QT + q) * 64];
#pragma unroll
            for (int k = 1; k < SPLIT; k++) {
                const sw_f32x4 z = all[(k * 4 + share * QT + q) * 64];
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = y[e] + z[e];
            }
#pragma unroll
            for (int e = 0; e < 4; e++) x[4 * q + e] = y[e];
        }
        if (!whole) {
            uint32_t met = 0;
#pragma unroll
            for (int j = 0; j < 4 * QT; j++) {
                const int k = 8 * (share * QT + j / 4) + h4 + j % 4;
                const bool in = seen(k);
                x[j] = in ? x[j] : -INFINITY;
                met |= in ? bad >> k & 1 : 0u;
            }
            if (met) l = NAN;
        }
#pragma unroll
        for (int j = 0; j < 4 * QT; j++) mx = fmaxf(mx, x[j]);
        mx = fl_max2(mx);
        auto put = [&](float &add) {                                   // this wave's tokens' weights and their sum
            const float base = m == -INFINITY ? 0.f : OFF - m * sc;
            add = 0.f;
#pragma unroll
            for (int q = 0; q < QT; q++) {
                float p8[8] = {};
#pragma unroll
                for (int e = 0; e < 4; e++) p8[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[4 * q + e], sc, base));
                sw_u32x4 o[1];
                fl_split<TYPE, 1>(p8, o);
                add = fl_sum<TYPE>(o[0][0], fl_sum<TYPE>(o[0][1], add));
                const int quad = share * QT + q;
                w[(quad >> 1) * 128 + (quad & 1)] = make_uint2(o[0][0], o[0][1]);
            }
        };
        float add;
        if (__any((mx - m) * sc > LAG) && lane == 0) grew[odd] = 1;
        if (wave == 0 && lane == 0) grew[odd ^ 1] = 0;                 // (read last before the barrier before)
        put(add);
        Piece first;
        read(v, 0, first);
        __syncthreads();
        if (__builtin_expect(grew[odd], 0)) {
            if (lane < 32) top[share * 32] = mx;
            __syncthreads();
            float n = m;
#pragma unroll
            for (int k = 0; k < SPLIT; k++) n = fmaxf(n, top[k * 32]);
            const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - n) * sc);
            l = l * f;
#pragma unroll
            for (int i = 0; i < NO; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) O[i][j] = O[i][j] * f;
            m = n;
            put(add);
            __syncthreads();
        }
        l = l + add;
        Weights P;
#pragma unroll
        for (int i = 0; i < 2; i++) P[i][0] = *(const sw_u32x4 *)(w + i * 128);
        const float none[16] = {};
        outputs(v, none, P, first);
    }

    // Where an output's values lie: tile o's row r is value d0 + T r + e of a group of values that T tiles share (f32: groups of 64 and 32
    // values; else T is 1), tile o being its e-th.
    struct Map { int d0[NO], tiles[NO], e[NO]; };
    static constexpr Map map() {
        Map m = {};
        int d = 0, w = F32 ? AHEAD : 1;
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
// whole(tile) (alike in the waves that share a tile), seen(tile, token): the mask; columns: this wave has some; s_bad: two words a group.
template <int WC, int WT, int NS, int NL, class F, class Issue, class Whole, class Seen>
__device__ __forceinline__ void fl_run(F &f, char *sh, uint32_t *s_bad, int ta, int tb, int wave, bool columns, Issue issue, Whole whole, Seen seen) {
    constexpr int TB = F::TB;
    constexpr bool shared = WC > 1;
    const int wt = WT == 1 ? 0 : wave / WC, all = (tb - ta + WT - 1) / WT, n = (tb - ta - wt + WT - 1) / WT;     // tiles of the longest group, of this one
    char *mine = sh + wt * NS * TB;
    s_bad += 2 * wt;
    const uint32_t lds = fl_lds_addr(mine);
    const bool first = (threadIdx.x & 63) == 0 && (WT > 1 && WC == 1 ? true : wave % WC == 0);       // of its group
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
            if (!whl) f.clean(mine + s * TB, WT == 1 ? wave : wave % WC, WC, s_bad + (i & 1));
            if (shared) __syncthreads();
            else fl_wait_lds();
            bad = s_bad[i & 1];
        }
        if (i < n && columns) f.tile(mine + s * TB, whl, bad, [&](int k) { return seen(t, k); });
        s = s + 1 == NS ? 0 : s + 1;
    }
}

// The same for WC groups of SPLIT waves that share columns, all of one tile; xch: LDS of the exchange.  Two barriers a tile: the outputs of one and the
// sums of the next lie between the same two, where the waves' products fill each other's waits.
template <int WC, int SPLIT, int NS, int NL, class F, class Issue, class Whole, class Seen>
__device__ __forceinline__ void fl_run_split(F &f, char *sh, char *xch, uint32_t *s_bad, int ta, int tb, int wave, Issue issue, Whole whole, Seen seen) {
    static_assert(NS >= 3, "a tile in the outputs, one in the sums, one on its way");
    constexpr int TB = F::TB;
    const int n = tb - ta;
    const uint32_t lds = fl_lds_addr(sh);
    const bool first = threadIdx.x == 0;
    if (first) {
        int *grew = (int *)(xch + SPLIT * 4096 + 2048 + SPLIT * 128);
        grew[0] = grew[1] = 0;
        s_bad[0] = 0;                                                  // (the item before is done with them)
    }
    uint32_t there = 0;                                                // bit s: all pages of the tile in place s are there
    auto load = [&](int i, int s) {
        const bool ok = issue(ta + i, lds + s * TB);
        there = ok ? there | 1u << s : there & ~(1u << s);
    };
#pragma unroll 1
    for (int i = 0; i < NS - 1; i++)
        if (i < n) load(i, i);
    if (NS - 2 >= n) fl_wait<0>();
    else fl_wait<(NS - 2) * NL>();
    __syncthreads();                                                   // the first tile is there
    f.sums(sh, xch, wave);
    int s = 0;                                                         // the place of tile i
#pragma unroll 1
    for (int i = 0; i < n; i++) {
        if (i + NS - 2 >= n) fl_wait<0>();
        else fl_wait<(NS - 3) * NL>();
        __syncthreads();                                               // tile i + 1 and the sums of i are there, tile i - 1 is read
        if (i + NS - 1 < n) load(i + NS - 1, s == 0 ? NS - 1 : s - 1);
        if (first) s_bad[(i + 1) & 1] = 0;
        char *t = sh + s * TB;
        const bool whl = ((there >> s) & 1) && whole(ta + i);
        uint32_t bad = 0;
        if (!whl) {
            f.clean(t, wave, WC * SPLIT, s_bad + (i & 1));
            __syncthreads();
            bad = s_bad[i & 1];
        }
        f.weigh(t, whl, bad, [&](int k) { return seen(ta + i, k); }, xch, wave, i & 1);
        s = s + 1 == NS ? 0 : s + 1;
        if (i + 1 < n) f.sums(sh + s * TB, xch, wave);
    }
}

// The end of an item: the groups' outputs of a column joined in their order and given to put(column, value, four
// outputs, maximum, sum), rows of 32 values or more at a time, so that they are written as whole lines.  sh: LDS of fl_end_bytes, free.
template <class F> constexpr int fl_end_row() { return 32 * (F::F32 ? 2 : 1) + 4; }
template <class F, int NW>
constexpr int fl_end_bytes() { return NW * 32 * fl_end_row<F>() * 4; }
template <int WC, int WT, int SPLIT, class F, class Put>
__device__ __forceinline__ void fl_end(F &f, char *sh, float (*s_m)[32], float (*s_l)[32], int wave, Put put) {
    constexpr int LD = fl_end_row<F>(), NO = F::NO;
    constexpr auto map = F::map();
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
    const float l = fl_sum2(f.l), m = f.m * f.sc;                      // (from here on the maximum is times the scale; with SPLIT the sums are of shares)
    __syncthreads();                                                   // the tiles are done with
    if (h == 0) { s_m[wave][c] = m; s_l[wave][c] = l; }
    __syncthreads();
    float g = 1.f;
    if constexpr (WT > 1) {
        float M = m;
#pragma unroll
        for (int i = 0; i < WT; i++) M = fmaxf(M, s_m[i * WC + wave % WC][c]);
        g = m == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(m - M);
    }
    const float *all = (const float *)sh;
    float *so = (float *)sh + (wave * 32 + c) * LD;
#pragma unroll
    for (int o0 = 0; o0 < NO; o0++) {                                  // T tiles share a row of 32 T values
        if (map.e[o0]) continue;
        const int T = map.tiles[o0], d0 = map.d0[o0];
#pragma unroll
        for (int e = 0; e < T; e++)
#pragma unroll
            for (int j = 0; j < 16; j++) so[T * (8 * (j / 4) + 4 * h + j % 4) + e] = WT > 1 ? f.O[o0 + e][j] * g : f.O[o0 + e][j];
        if constexpr (WT == 1) {                                       // a wave's own columns
            fl_wait_lds();
#pragma unroll 1
            for (int i = 0; i < 4 * T; i++) {
                const int k = i * 64 + lane, col = k / (8 * T), d = k % (8 * T) * 4, wc = wave / SPLIT;
                const sw_f32x4 a = *(const sw_f32x4 *)(all + (wave * 32 + col) * LD + d);
                float sum = s_l[wc * SPLIT][col];
#pragma unroll
                for (int k2 = 1; k2 < SPLIT; k2++) sum = sum + s_l[wc * SPLIT + k2][col];
                put(wc * 32 + col, (wave % SPLIT) * F::DVW + d0 + d, a, s_m[wave][col], sum);
            }
            fl_wait_lds();
        } else {
            __syncthreads();
#pragma unroll 1
            for (int i = tid; i < WC * 32 * 8 * T; i += WC * WT * 64) {
                const int col = i / (8 * T), d = i % (8 * T) * 4, w = col >> 5;
                sw_f32x4 a = *(const sw_f32x4 *)(all + (w * 32 + (col & 31)) * LD + d);
                float mx = s_m[w][col & 31], sum = 0.f;
#pragma unroll
                for (int k = 1; k < WT; k++) {
                    const sw_f32x4 y = *(const sw_f32x4 *)(all + ((w + k * WC) * 32 + (col & 31)) * LD + d);
#pragma unroll
                    for (int e = 0; e < 4; e++) a[e] = a[e] + y[e];
                    mx = fmaxf(mx, s_m[w + k * WC][col & 31]);
                }
#pragma unroll
                for (int k = 0; k < WT; k++) {
                    const float x = s_m[w + k * WC][col & 31];
                    sum = __builtin_fmaf(s_l[w + k * WC][col & 31], x == -INFINITY ? (mx == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(x - mx), sum);
                }
                put(col, d0 + d, a, mx, sum);
            }
            __syncthreads();
        }
    }
    if (WT == 1) __syncthreads();                                      // (the next item's tiles take the same LDS)
}

// A block's parts: of the item that it goes on with, and of the one that it begins and does not end (an item's tiles from `from` on).  An
// item's part k is then 2 k - 1 places behind its first.
__device__ __forceinline__ int64_t fl_slot(int b, int from) { return 2 * (int64_t)b + (from == 0); }
// Parts of one column joined, in their order: part k at p + max(0, 2 k - 1) * step holds its maximum and sum, then (behind 4) DV outputs.  A wave
// takes 256 values from v0 on, 4 a lane; where DV / 4 lanes are a part of a wave, its parts take turns.  Weights are a lane's each, 64
// parts at a time.  Returns the outputs divided by the sum (0 where there is none).
template <int DV>
__device__ __forceinline__ sw_f32x4 fl_join(const float *p, int64_t step, int parts, int v0) {
    constexpr int ND = DV / 4, SUB = ND <= 32 && (ND & (ND - 1)) == 0 ? 64 / ND : 1;
    const int lane = threadIdx.x & 63, sub = SUB > 1 ? lane / ND : 0, d = v0 + (SUB > 1 ? lane % ND : lane) * 4;
    const bool mine = d < DV;
    sw_f32x4 a = {0.f, 0.f, 0.f, 0.f};
    float M = -INFINITY, L = 0.f;
    parts = fl_uni(parts);
    for (int k0 = 0; k0 < parts; k0 += 64) {
        const int top = min(64, parts - k0);
        constexpr int LOT = 8;                                         // outputs on their way, the first while the weights are made (16: 2 us more for many columns)
        sw_f32x4 y[LOT];
        auto fetch = [&](int k) {
#pragma unroll
            for (int i = 0; i < LOT; i++)
                if (k + i * SUB < top) y[i] = *(const sw_f32x4 *)(p + max(0, 2 * (k0 + min(k + i * SUB + sub, top - 1)) - 1) * step + 4 + (mine ? d : 0));
        };
        float m = -INFINITY, l = 0.f;
        if (k0 + lane < parts) {
            const float2 z = *(const float2 *)(p + max(0, 2 * (k0 + lane) - 1) * step);
            m = z.x; l = z.y;
        }
        fetch(0);
        float n = fmaxf(M, m);
#pragma unroll
        for (int o = 32; o; o >>= 1) n = fmaxf(n, __shfl_xor(n, o));
        const float g = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(M - n);                          // (nothing summed before: any factor)
        const float w = m == -INFINITY ? (n == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(m - n);
        float s = l * w;
#pragma unroll
        for (int o = 32; o; o >>= 1) s = s + __shfl_xor(s, o);
        L = __builtin_fmaf(L, g, s);
        M = n;
#pragma unroll
        for (int e = 0; e < 4; e++) a[e] = a[e] * g;
        for (int k = 0;;) {
#pragma unroll
            for (int i = 0; i < LOT; i++) {
                if (k + i * SUB >= top) break;
                const int at = k + i * SUB + sub;
                const float f = __shfl(w, at & 63);
#pragma unroll
                for (int e = 0; e < 4; e++) a[e] = at < top ? __builtin_fmaf(y[i][e], f, a[e]) : a[e];
            }
            k += LOT * SUB;
            if (k >= top) break;
            fetch(k);
        }
    }
#pragma unroll
    for (int o = ND; o < 64 && SUB > 1; o <<= 1)
#pragma unroll
        for (int e = 0; e < 4; e++) a[e] = a[e] + __shfl_xor(a[e], o);
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] = L == 0.f ? 0.f : a[e] * inv;
    return a;
}

// Blocks of a join of `of` such groups of columns, `all` of one: waves take several columns where they would not all run at once, and
// find their place among the items once (16 trees' join 27 -> 16 us, and as much with half or twice the blocks).
inline int fl_join_blocks(int all, int64_t of) {
    const int64_t n = 1024 / (of < 1 ? 1 : of);
    return n < 1 ? 1 : n < all ? (int)n : all;
}

// The least tiles of a block: a tile takes it some 2 us, and the outputs of a part (cols columns of all blocks that share its tokens) are written and
// read again at some 4 TB/s, so with N tiles in all the two are least together where q^2 = N cols values 8 bytes / 8 MB.
__device__ __forceinline__ int fl_least(int64_t N, int64_t values) {
    const int q = (int)sqrtf((float)N * (float)values * 1e-6f);
    return q < 1 ? 1 : q;
}

// How items' tiles are dealt to B blocks: laid end to end they are N, and block b takes those from b q to (b + 1) q, whatever
// items they fall in.  count(i): the tiles of item i (evaluated 64 items at a time, a lane each).  `values`: outputs of an item (fl_least).
struct FlDeal { int64_t N, q; };
template <class Count>
__device__ __forceinline__ FlDeal fl_deal(int items, int B, int64_t values, Count count) {
    const int lane = threadIdx.x & 63;
    FlDeal d = {0, 0};
    for (int i0 = 0; i0 < items; i0 += 64)
        d.N += (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)sw_wave_scan(i0 + lane < items ? (uint32_t)count(i0 + lane) : 0u), 63);
    d.q = (d.N + B - 1) / B;
    const int least = fl_uni(fl_least(d.N, values));
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
