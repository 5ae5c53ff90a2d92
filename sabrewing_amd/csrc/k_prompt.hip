// k_prompt.hip -- latent attention of a prompt's tokens, the expanded form: keys Wk[h] c_t and values Wv[h] c_t of every token
// are made once, then out[s, h] = sum_t p_t v_t, p = softmax over t <= start + s of scale * q[s, h] . (k_t, r_t).
//
// Bf16, 32 heads of 128 + 64 and 128, rank 512: 2,048 tokens from position 6,000 on 433 to 476 us by the card (362 GFLOP, 836 to 760 TFLOP/s).  Traced,
// where the launches take longer than back to back: the gathering 9.5, the expansion 112 (67 GFLOP: eight lots of 64 values are few to fill the pipe),
// the attention 358 (295 GFLOP: matrix instructions half of the cycles, vector ones -- exponentials -- the rest).  Heads of 192 and 256 are held as 256, one block
// a CU: 747 us with 192 + 64 and 128, 1,108 with 256 + 64 and 256.  300 tokens of 16 heads from the beginning 33 us, its three launches' begins
// and ends.
//
// Three launches: cells gathered from their pages, keys and values of some heads expanded, their attention.  Against the
// absorbed form a pair of tokens costs 2 (nope + rope + v) instead of 2 (2 rank + rope) operations, and a token 2 rank (nope + v) once.
//
// Keys and values are held in f16, whatever the cache's type: 11 bits, where bf16's 8 would add errors as large as the
// output's own rounding three times over.  (Outputs of 32 bits have no more: 24 would be three times the products.)  f16's range is met by powers of two: |k_d| <= |Wk_d| |c_t| (their 2-norms), so each
// head's keys are scaled by 2^(15 - a - b), a and b the exponents of the largest |Wk_d| and |c_t|, which keeps them
// below 2^15; a sum of many terms stays some 2^8 below that bound, and what is more than 2^20 smaller than the largest, of whichever
// token, loses bits.  Values alike; queries are scaled to 2^13.  The rotary part stays as the cache has it.
#include "sw_flash.h"

#define LP_NT 256
#define LP_ROPE 64

template <int TYPE> __device__ __forceinline__ float lp_float(uint32_t w, int hi) {
    if constexpr (TYPE == SW_KV_BF16) return __builtin_bit_cast(float, hi ? w & 0xFFFF0000u : w << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(hi ? w >> 16 : w));
}
// e with x < 2^e for a sum of squares x^2, in 64 bits: whatever finite values of 16 bits are squared, it is finite, and 0 where they all are
#define LP_LEAST -140
__device__ __forceinline__ int lp_exp(double x2) { return x2 > 0.0 ? (ilogb(x2) + 2) >> 1 : LP_LEAST; }
// a + b of the lanes BY (16, 32) apart: of a in the lower of the two, of b in the upper
template <int BY>
__device__ __forceinline__ double lp_halves(double a, double b) {
    const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
    if constexpr (BY == 16) {
        const auto lo = __builtin_amdgcn_permlane16_swap(x.x, y.x, false, false), hi = __builtin_amdgcn_permlane16_swap(x.y, y.y, false, false);
        return __builtin_bit_cast(double, make_uint2((uint32_t)lo[0], (uint32_t)hi[0])) + __builtin_bit_cast(double, make_uint2((uint32_t)lo[1], (uint32_t)hi[1]));
    } else {
        const auto lo = __builtin_amdgcn_permlane32_swap(x.x, y.x, false, false), hi = __builtin_amdgcn_permlane32_swap(x.y, y.y, false, false);
        return __builtin_bit_cast(double, make_uint2((uint32_t)lo[0], (uint32_t)hi[0])) + __builtin_bit_cast(double, make_uint2((uint32_t)lo[1], (uint32_t)hi[1]));
    }
}
// x plus the value of the lane that a rotation in rows of 16 lanes brings
template <int DPP>
__device__ __forceinline__ double lp_turned(double x) {
    const uint2 u = __builtin_bit_cast(uint2, x);
    return x + __builtin_bit_cast(double, make_uint2((uint32_t)__builtin_amdgcn_update_dpp(0, (int)u.x, DPP, 0xF, 0xF, false),
                                                     (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u.y, DPP, 0xF, 0xF, false)));
}
// a wave's largest exponent
__device__ __forceinline__ int lp_max(int e) { return (int)sw_wave_max((uint32_t)(e + 1024)) - 1024; }

// Blocks 0 .. tiles - 1: 32 cells side by side in xl [tokens][rank] and xr [tokens][64] (zeros where there is no cell or no value), te: the
// exponent of the tile's largest norm, re: of its largest rotary value, vm: which tokens have a cell.  Blocks behind them, LP_PARTS for a head's keys and as many for its
// values: we, the exponent of the largest norm of a share of the rows of Wk or Wv.  Values that are no numbers do not count in a
// norm.  A wave takes its 8 rows at once: one wait.
#define LP_PARTS 8
template <int TYPE>
__global__ __launch_bounds__(LP_NT) void k_prompt_gather(SwLatent c, const int *__restrict__ pages, int max_pages, int T, const uint16_t *__restrict__ wk,
                                                         const uint16_t *__restrict__ wv, int nope, int vd, uint16_t *__restrict__ xl,
                                                         uint16_t *__restrict__ xr, int *__restrict__ te, int *__restrict__ re, uint32_t *__restrict__ vm,
                                                         int *__restrict__ we) {
    constexpr int NW = LP_NT / 64, N = 32 / NW;
    __shared__ int s_n[NW];
    __shared__ float s_r[NW];
    __shared__ uint32_t s_v[NW];
    const int tid = threadIdx.x, lane = tid & 63, wave = fl_uni(tid >> 6), tiles = (T + 31) / 32;
    double ss[N];                                                      // of each row
    float turned = 0.f;
    uint32_t there = 0;
    // (every lane reads, those behind a row's end its last values, which do not count)
    const bool in = 8 * lane < c.rank;
    const int at = min(8 * lane, c.rank - 8), rat = c.rank + max(0, min(8 * lane, c.rope - 8));
    sw_u32x4 a[N];
    auto finite = [](uint32_t y, int k) {
        const float f = lp_float<TYPE>(y, k);
        return fabsf(f) < INFINITY ? f : 0.f;
    };
    auto squares = [&](sw_u32x4 y, bool count) {
        double x = 0.0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const double g = finite(y[e / 2], e & 1);
            x = __builtin_fma(g, g, x);
        }
        return count && in ? x : 0.0;
    };
    if ((int)blockIdx.x < tiles) {
        const int t0 = blockIdx.x * 32 + wave * N, pmask = (1 << c.psh) - 1;
        const int pg = min(t0 + (lane & (N - 1)), T - 1) >> c.psh;
        int page = pages[min(pg, max_pages - 1)];
        if (t0 + (lane & (N - 1)) >= T || pg >= max_pages || page >= c.n_pages) page = -1;
        there = (uint32_t)__ballot(lane < N && page >= 0);
        sw_u32x4 b[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int p = max(__builtin_amdgcn_readlane(page, i), 0);
            const uint16_t *cell = (const uint16_t *)c.p + (int64_t)p * c.ps + (int64_t)((t0 + i) & pmask) * c.ts;
            a[i] = *(const sw_u32x4 *)(cell + at);
            b[i] = *(const sw_u32x4 *)(cell + (c.rope ? rat : 0));
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const bool cell = there >> i & 1;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                a[i][e] = cell ? a[i][e] : 0u;
                b[i][e] = cell && 8 * lane < c.rope ? b[i][e] : 0u;
            }
            if (in) *(sw_u32x4 *)(xl + (int64_t)(t0 + i) * c.rank + 8 * lane) = a[i];
            if (lane < LP_ROPE / 8) *(sw_u32x4 *)(xr + (int64_t)(t0 + i) * LP_ROPE + 8 * lane) = b[i];
            ss[i] = squares(a[i], true);
#pragma unroll
            for (int e = 0; e < 8; e++) turned = fmaxf(turned, fabsf(finite(b[i][e / 2], e & 1)));
        }
        turned = __builtin_bit_cast(float, sw_wave_max(__builtin_bit_cast(uint32_t, turned)));         // (none is negative)
    } else {
        const int k = (blockIdx.x - tiles) / LP_PARTS, part = (blockIdx.x - tiles) % LP_PARTS, h = k >> 1, n = k & 1 ? vd : nope;
        const uint16_t *w = (k & 1 ? wv : wk) + (int64_t)h * n * c.rank;
        const int i0 = part * (n / LP_PARTS) + wave * N, end = (part + 1) * (n / LP_PARTS);           // (n: a multiple of 32, at most 256)
#pragma unroll
        for (int i = 0; i < N; i++) a[i] = *(const sw_u32x4 *)(w + (int64_t)min(i0 + i, n - 1) * c.rank + at);
#pragma unroll
        for (int i = 0; i < N; i++) ss[i] = squares(a[i], i0 + i < end);
    }
    // the rows' sums: halves and quarters of the rows go to halves and quarters of the lanes, whose 16 lanes add up two rows each
    static_assert(N == 8, "rows of a wave");
#pragma unroll
    for (int i = 0; i < 4; i++) ss[i] = lp_halves<32>(ss[i], ss[i + 4]);
#pragma unroll
    for (int i = 0; i < 2; i++) ss[i] = lp_turned<0x121>(lp_turned<0x122>(lp_turned<0x124>(lp_turned<0x128>(lp_halves<16>(ss[i], ss[i + 2])))));
    int best = lp_max(max(lp_exp(ss[0]), lp_exp(ss[1])));
    if (lane == 0) { s_n[wave] = best; s_r[wave] = turned; s_v[wave] = there << (wave * N); }
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int i = 1; i < NW; i++) { best = max(best, s_n[i]); turned = fmaxf(turned, s_r[i]); }
        if ((int)blockIdx.x < tiles) {
            te[blockIdx.x] = best;
            re[blockIdx.x] = turned > 0.f ? ilogbf(turned) + 1 : LP_LEAST;
            vm[blockIdx.x] = s_v[0] | s_v[1] | s_v[2] | s_v[3];
        }
        else we[blockIdx.x - tiles] = best;
    }
}

// Keys and values of heads h0 .. of H: [head][tokens][np or vp] in f16, times 2^eh, the values behind nope or vd zeros (eh[2 H]: the
// exponent of the largest rotary value of all tokens).  A block takes 128 outputs by 128 tokens, both in LDS by 64 of the summed values, one lot ahead; a wave 64 by 64 of them.  A die's blocks share
// a range of tokens (they stay in its cache) and go through all heads.
#define LE_K 64
#define LE_TILE (128 * LE_K * 2)
template <int TYPE>
__global__ __launch_bounds__(LP_NT, 2) void k_prompt_expand(const uint16_t *__restrict__ xl, const int *__restrict__ te, const int *__restrict__ re,
                                                            const int *__restrict__ we, int T32, int H, int rank, const uint16_t *__restrict__ wk, const uint16_t *__restrict__ wv, int nope, int vd,
                                                            int np, int vp, int heads, int h0, uint16_t *__restrict__ kb, uint16_t *__restrict__ vb,
                                                            int *__restrict__ eh) {
    __shared__ __align__(16) char sh[2 * 2 * LE_TILE];
    __shared__ int s_e[LP_NT / 64], s_r[LP_NT / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = fl_uni(tid >> 6), c = lane & 31, g = lane >> 5;
    const int tk = (np + 127) / 128, tv = (vp + 127) / 128, nt = (T32 + 127) / 128, per = (nt + 7) / 8;
    const int die = blockIdx.x & 7, j0 = blockIdx.x >> 3, tt = die * per + j0 % per, y0 = j0 / per;
    if (tt >= nt || y0 >= heads * (tk + tv)) return;
    const int hl = y0 / (tk + tv), by = y0 % (tk + tv), h = h0 + hl, kv = by >= tk, n = kv ? vd : nope, pad = kv ? vp : np;
    const int o0 = (kv ? by - tk : by) * 128, s0 = tt * 128;
    const uint16_t *W = (kv ? wv : wk) + (int64_t)h * n * rank;
    // rows o0 .. of W and s0 .. of xl (the last in the place of those behind), 8 pieces of 16 bytes each, turned by the row
    uint32_t wo[4], xo[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int r = (k * 4 + wave) * 8 + (lane >> 3), p = (lane & 7) ^ fl_turn<7>(r);
        wo[k] = (uint32_t)min(o0 + r, n - 1) * rank * 2 + p * 16;
        xo[k] = (uint32_t)min(r, T32 - 1 - s0) * rank * 2 + p * 16;
    }
    const char *xb = (const char *)(xl + (int64_t)s0 * rank);
    const uint32_t lds = fl_lds_addr(sh);
    auto load = [&](int i) {
#pragma unroll
        for (int k = 0; k < 4; k++) fl_load16((const char *)W + i * (LE_K * 2), wo[k], lds + (i & 1) * 2 * LE_TILE + (k * 4 + wave) * 1024);
#pragma unroll
        for (int k = 0; k < 4; k++) fl_load16(xb + i * (LE_K * 2), xo[k], lds + (i & 1) * 2 * LE_TILE + LE_TILE + (k * 4 + wave) * 1024);
    };
    load(0);
    int e = LP_LEAST, r = LP_LEAST;
    for (int i = tid; i < T32 / 32; i += LP_NT) { e = max(e, te[i]); r = max(r, re[i]); }
    e = lp_max(e);
    r = lp_max(r);
    if (lane == 0) { s_e[wave] = e; s_r[wave] = r; }
    __syncthreads();
    int w = LP_LEAST;
#pragma unroll
    for (int i = 0; i < LP_NT / 64; i++) { e = max(e, s_e[i]); r = max(r, s_r[i]); }
#pragma unroll
    for (int i = 0; i < LP_PARTS; i++) w = max(w, we[(2 * h + kv) * LP_PARTS + i]);
    e = min(max(15 - e - w, -120), 120);
    if (tid == 0 && tt == 0) { eh[2 * h + kv] = e; eh[2 * H] = r; }    // (every block the same)
    fl_f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = fl_f32x16{};
    const int wo0 = (wave & 1) * 64, ws0 = (wave >> 1) * 64, steps = rank / LE_K;
#pragma unroll 1
    for (int i = 0; i < steps; i++) {
        fl_wait<0>();
        __syncthreads();                                               // lot i is there, lot i - 1 read
        if (i + 1 < steps) load(i + 1);
        const char *A = sh + (i & 1) * 2 * LE_TILE, *B = A + LE_TILE;
#pragma unroll
        for (int k = 0; k < LE_K / 16; k++) {
            sw_u32x4 a[2], b[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                a[u] = *(const sw_u32x4 *)(A + (wo0 + 32 * u + c) * (LE_K * 2) + (((2 * k + g) ^ fl_turn<7>(c)) * 16));
                b[u] = *(const sw_u32x4 *)(B + (ws0 + 32 * u + c) * (LE_K * 2) + (((2 * k + g) ^ fl_turn<7>(c)) * 16));
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int v = 0; v < 2; v++) acc[u][v] = fl_mfma<TYPE>(a[u], b[v], acc[u][v]);
        }
    }
    const float f = ldexpf(1.f, e);
    uint16_t *y = (kv ? vb : kb) + (int64_t)hl * T32 * pad;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int s = s0 + ws0 + 32 * j + c;
        if (s >= T32) continue;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int o = o0 + wo0 + 32 * i;
            if (o >= pad) break;
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                uint32_t p[4];
#pragma unroll
                for (int q = 0; q < 4; q++) p[q] = o < n ? (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)(acc[i][j][r + q] * f)) : 0u;
                *(uint2 *)(y + (int64_t)s * pad + o + 2 * r + 4 * g) = make_uint2(p[0] | (p[1] << 16), p[2] | (p[3] << 16));
            }
        }
    }
}

// 32 rows of a head a wave; a tile holds 32 tokens' keys (their expanded part), values and rotary parts
template <int TYPE, int NOPE, int DV>
struct LpFl : Fl<SW_KV_F16, 1, NOPE, DV, false> {
    using Base = Fl<SW_KV_F16, 1, NOPE, DV, false>;
    static constexpr int ROPE_AT = Base::TB, TB = Base::TB + 32 * LP_ROPE * 2;
    sw_u32x4 R[LP_ROPE / 16];                                          // the queries' rotary part, scaled as the other is with its keys
    int lift;                                                          // or 2^lift less (lifts: in any of the wave's columns)
    bool lifts;
    template <class Seen>
    __device__ __forceinline__ void tile(const char *t, bool whole, uint32_t bad, Seen seen) {
        const int lane = fl_lane<Base::KEEP>(), c = lane & 31, h = lane >> 5;
        fl_f32x16 s = {};
        sw_u32x4 r[LP_ROPE / 16];
#pragma unroll
        for (int i = 0; i < LP_ROPE / 16; i++) r[i] = *(const sw_u32x4 *)(t + ROPE_AT + c * (LP_ROPE * 2) + (((2 * i + h) ^ fl_turn<7>(c)) * 16));
        this->dot(t, s);
        if (__builtin_expect(lifts, 0))
#pragma unroll
            for (int j = 0; j < 16; j++) s[j] = ldexpf(s[j], -lift);
#pragma unroll
        for (int i = 0; i < LP_ROPE / 16; i++) s = fl_mfma<TYPE>(r[i], R[i], s);
        if (__builtin_expect(lifts, 0))
#pragma unroll
            for (int j = 0; j < 16; j++) s[j] = ldexpf(s[j], lift);
        this->alone(t, whole, bad, seen, s);
    }
};
// blocks a CU (with 32 rows a block, heads of 128 + 128 and of 256 + 64 take registers for one all the same)
template <int NOPE, int DV> constexpr int lp_occ() { return NOPE / 4 + DV / 2 <= 112 ? 2 : 1; }
template <int TYPE, int NOPE, int DV, int WC> constexpr int lp_ns() {
    constexpr int n = (lp_occ<NOPE, DV>() == 2 ? 78 : 156) * 1024 / (FL_NW / WC * LpFl<TYPE, NOPE, DV>::TB);
    return n < 1 ? 1 : n > 3 ? 3 : n;
}
template <int TYPE, int NOPE, int DV, int WC>
__global__ __launch_bounds__(FL_NT, (lp_occ<NOPE, DV>())) void k_prompt(const uint16_t *__restrict__ kb, const uint16_t *__restrict__ vb,
                                                                       const uint16_t *__restrict__ xr, const uint32_t *__restrict__ vm,
                                                                       const int *__restrict__ eh, int T32, int start, int S, int nope, int vd, int rope,
                                                                       const uint16_t *__restrict__ q, int H, int h0, int heads, float sc0,
                                                                       void *__restrict__ out, int of32) {
    using F = LpFl<TYPE, NOPE, DV>;
    constexpr int ROWS = 32 * WC, WT = FL_NW / WC, NS = lp_ns<TYPE, NOPE, DV, WC>();
    constexpr int LK = (F::NCK / 2 + WC - 1) / WC, LV = (F::NCV / 2 + WC - 1) / WC, LR = (LP_ROPE / 16 + WC - 1) / WC, NL = LK + LV + LR;
    constexpr int SHT = WT * NS * F::TB, SHB = SHT > fl_end_bytes<F, FL_NW>() ? SHT : fl_end_bytes<F, FL_NW>();
    static_assert(SHB <= 157 * 1024 && (NS < 3 ? 0 : NS - 2) * NL < 64, "LDS, and loads that a wave can count");
    __shared__ __align__(256) char sh[SHB];
    __shared__ float s_m[FL_NW][32], s_l[FL_NW][32];
    __shared__ uint32_t s_bad[2 * FL_NW];
    const int tid = threadIdx.x, lane = tid & 63, wave = fl_uni(tid >> 6), wc = wave % WC, cl = lane & 31, h2 = lane >> 5;
    // the longest rows first; a head's blocks 8 apart where the heads are a multiple of 8 (its keys and values in one L2)
    const int hl = blockIdx.x % heads, h = h0 + hl, r0 = ((int)(gridDim.x / heads) - 1 - (int)(blockIdx.x / heads)) * ROWS;
    const int row = r0 + wc * 32 + cl, last = start + min(r0 + ROWS, S) - 1, tiles = (last >> 5) + 1;
    F f;
    // ---- the queries
    const uint16_t *qp = q + ((int64_t)min(row, S - 1) * H + h) * (nope + rope);
    sw_u32x4 raw[F::DKS];
    float mx = 0.f;
#pragma unroll
    for (int k = 0; k < F::DKS; k++) {
        raw[k] = sw_u32x4{0, 0, 0, 0};
        if (16 * k + 8 * h2 < nope) raw[k] = *(const sw_u32x4 *)(qp + 16 * k + 8 * h2);
#pragma unroll
        for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(lp_float<TYPE>(raw[k][e / 2], e & 1)));
    }
    sw_u32x4 rr[LP_ROPE / 16];
    float mr = 0.f;
#pragma unroll
    for (int k = 0; k < LP_ROPE / 16; k++) {
        rr[k] = sw_u32x4{0, 0, 0, 0};
        if (16 * k + 8 * h2 < rope) rr[k] = *(const sw_u32x4 *)(qp + nope + 16 * k + 8 * h2);
#pragma unroll
        for (int e = 0; e < 8; e++) mr = fmaxf(mr, fabsf(lp_float<TYPE>(rr[k][e / 2], e & 1)));
    }
    mx = fl_max2(mx);
    mr = fl_max2(mr);
    // The scores are to be 2^E times as large, of both parts: the keys are 2^ek times, the queries 2^(E - ek) -- up to 2^13 -- and the
    // rotary queries, whose keys are as they were, 2^E, where the sum of their products then stays far below f32's largest (er).  But they are
    // 2^15 at most in f16 (2^120 in bf16).  Where that binds, E follows while the first part's queries keep their bits (2^1 and
    // what is 2^15 below it); else the rotary scores are made 2^lift smaller and lifted.
    const int ek = eh[2 * h], ev = eh[2 * h + 1], er = eh[2 * H];
    const bool nx = mx > 0.f && mx < INFINITY, nr = mr > 0.f && mr < INFINITY;
    int E = min(max(nx ? 13 - ilogbf(mx) + ek : ek, -120), 120), Er = E;
    if (nr) {
        E = max(min(E, 99 - ilogbf(mr) - er), -120);
        Er = min(E, (TYPE == SW_KV_BF16 ? 120 : 14) - ilogbf(mr));
        if (E - Er <= 12) E = Er;
    }
    f.lift = E - Er;
    f.lifts = __any(f.lift != 0);
    const float sg = sc0 < 0.f ? -1.f : sc0 == 0.f ? 0.f : 1.f;       // (the scale's sign, or none: see Fl::begin)
    f.begin(ldexpf(sc0, -E));
#pragma unroll
    for (int k = 0; k < F::DKS; k++) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = sg * ldexpf(lp_float<TYPE>(raw[k][e / 2], e & 1), E - ek);
        f.query(k, y);
    }
#pragma unroll
    for (int k = 0; k < LP_ROPE / 16; k++) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = sg * ldexpf(lp_float<TYPE>(rr[k][e / 2], e & 1), Er);
        sw_u32x4 o[1];
        fl_split<TYPE, 1>(y, o);
        f.R[k] = o[0];
    }
    bool every = true;                                                 // no token without a cell before the last tile
    for (int i = tid; i < tiles - 1; i += FL_NT) every = every && vm[i] == 0xFFFFFFFFu;
    every = __syncthreads_and(every);
    const char *kp = (const char *)(kb + (int64_t)hl * T32 * NOPE), *vp = (const char *)(vb + (int64_t)hl * T32 * DV);
    auto issue = [&](int tile, uint32_t lds) {
        const int lane_ = fl_lane<F::KEEP>();
        fl_rows<F::NCK, F::MK, WC, LK>(kp + (int64_t)tile * (32 * NOPE * 2), NOPE * 2, wc, lane_, lds);
        fl_rows<F::NCV, F::MV, WC, LV>(vp + (int64_t)tile * (32 * DV * 2), DV * 2, wc, lane_, lds + 32 * F::RBK);
        fl_rows<LP_ROPE / 8, 7, WC, LR>((const char *)xr + (int64_t)tile * (32 * LP_ROPE * 2), LP_ROPE * 2, wc, lane_, lds + F::ROPE_AT);
        return every || fl_entry((const int *)vm, tile) == -1;
    };
    auto whole = [&](int tile) { return tile * 32 + 31 <= start + r0 && tile < tiles - 1; };
    auto seen = [&](int tile, int k) { return tile * 32 + k <= start + row && ((vm[tile] >> k) & 1); };
    fl_run<WC, WT, NS, NL>(f, sh, s_bad, 0, tiles, wave, true, issue, whole, seen);
    fl_end<WC, WT, 1>(f, sh, s_m, s_l, wave, [&](int col, int d, sw_f32x4 a, float, float sum) {
        const int s = r0 + col;
        if (s >= S || d >= vd) return;
#pragma unroll
        for (int e = 0; e < 4; e++) a[e] = sum == 0.f ? 0.f : ldexpf(a[e] * (1.f / sum), -ev);
        const int64_t at = ((int64_t)s * H + h) * vd + d;
        if (of32) *(sw_f32x4 *)((float *)out + at) = a;
        else {
            uint32_t p[4];
#pragma unroll
            for (int e = 0; e < 4; e++) p[e] = TYPE == SW_KV_BF16 ? (uint32_t)sw_bf16_rne(a[e]) : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a[e]);
            *(uint2 *)((uint16_t *)out + at) = make_uint2(p[0] | (p[1] << 16), p[2] | (p[3] << 16));
        }
    });
}

// ------------------------------------------------------------------ scratch and launches ----
// heads expanded at a time: as many as a GiB holds, and one at least (beyond 2^20 tokens of 256 + 256 that is more, up to 4 GiB)
struct LpPlan { int64_t T32, xl, xr, te, re, vm, we, eh, kb, vb, total; int heads, np, vp; };
static LpPlan lp_plan(const SwLatent &c, int H, int nope, int vd, int64_t T) {
    LpPlan p;
    p.T32 = (T + 31) / 32 * 32;
    p.np = nope <= 64 ? 64 : nope <= 128 ? 128 : 256;
    p.vp = vd <= 64 ? 64 : vd <= 128 ? 128 : 256;
    const int64_t one = p.T32 * (p.np + p.vp) * 2, most = ((int64_t)1 << 30) / one;
    p.heads = (int)(most < 1 ? 1 : most < H ? most : H);
    int64_t at = 0;
    auto take = [&](int64_t n) { const int64_t x = at; at += (n + 255) / 256 * 256; return x; };
    p.xl = take(p.T32 * c.rank * 2);
    p.xr = take(p.T32 * LP_ROPE * 2);
    p.te = take(p.T32 / 8);
    p.re = take(p.T32 / 8);
    p.vm = take(p.T32 / 8);
    p.we = take((int64_t)H * 8 * LP_PARTS);
    p.eh = take((int64_t)H * 8 + 4);
    p.kb = take(p.heads * p.T32 * p.np * 2);
    p.vb = take(p.heads * p.T32 * p.vp * 2);
    p.total = at;
    return p;
}
int64_t sw_latent_prompt_bytes(const SwLatent &c, int H, int nope, int vd, int64_t T) { return lp_plan(c, H, nope, vd, T).total; }

struct LpArgs { const uint16_t *kb, *vb, *xr; const uint32_t *vm; const int *eh; int T32, start, S, nope, vd, rope; const uint16_t *q; int H, h0, heads; float sc; void *out; int of32; };
template <int TYPE, int NOPE, int DV, int WC>
static void lp_launch(hipStream_t st, const LpArgs &a) {
    const int64_t grid = (int64_t)a.heads * ((a.S + 32 * WC - 1) / (32 * WC));
    SW_LAUNCH((k_prompt<TYPE, NOPE, DV, WC>), dim3((unsigned)grid), dim3(FL_NT), 0, st, a.kb, a.vb, a.xr, a.vm, a.eh, a.T32, a.start, a.S, a.nope, a.vd, a.rope,
              a.q, a.H, a.h0, a.heads, a.sc, a.out, a.of32);
}
template <int TYPE, int NOPE, int DV>
static void lp_form(hipStream_t st, const LpArgs &a) {
    // 128 rows a block where that fills the chip, else 32 rows whose tokens the waves share
    const bool wide = (int64_t)a.heads * ((a.S + 127) / 128) >= 256;
    if (wide) lp_launch<TYPE, NOPE, DV, 4>(st, a);
    else lp_launch<TYPE, NOPE, DV, 1>(st, a);
}
template <int TYPE, int NOPE>
static void lp_values(hipStream_t st, const LpArgs &a) {
    if (a.vd <= 64) lp_form<TYPE, NOPE, 64>(st, a);
    else if (a.vd <= 128) lp_form<TYPE, NOPE, 128>(st, a);
    else lp_form<TYPE, NOPE, 256>(st, a);
}
template <int TYPE>
static int lp_run(hipStream_t st, const SwLatent &c, const int *pages, int max_pages, int start, const void *wk, const void *wv, int nope, int vd, const void *q,
                  int H, float sc, void *out, int out_f32, int S, char *A) {
    const int T = start + S;
    const LpPlan p = lp_plan(c, H, nope, vd, T);
    uint16_t *xl = (uint16_t *)(A + p.xl), *xr = (uint16_t *)(A + p.xr), *kb = (uint16_t *)(A + p.kb), *vb = (uint16_t *)(A + p.vb);
    int *te = (int *)(A + p.te), *re = (int *)(A + p.re), *we = (int *)(A + p.we), *eh = (int *)(A + p.eh);
    uint32_t *vm = (uint32_t *)(A + p.vm);
    SW_LAUNCH(k_prompt_gather<TYPE>, dim3((unsigned)(p.T32 / 32 + 2 * H * LP_PARTS)), dim3(LP_NT), 0, st, c, pages, max_pages, T, (const uint16_t *)wk, (const uint16_t *)wv,
              nope, vd, xl, xr, te, re, vm, we);
    for (int h0 = 0; h0 < H; h0 += p.heads) {
        const int heads = H - h0 < p.heads ? H - h0 : p.heads, blocks = (p.np + 127) / 128 + (p.vp + 127) / 128;
        const int64_t per = (p.T32 / 32 + 31) / 32;                     // lots of 128 tokens of a die
        SW_LAUNCH(k_prompt_expand<TYPE>, dim3((unsigned)(8 * per * heads * blocks)), dim3(LP_NT), 0, st, xl, te, re, we, (int)p.T32, H, c.rank,
                  (const uint16_t *)wk, (const uint16_t *)wv, nope, vd, p.np, p.vp, heads, h0, kb, vb, eh);
        const LpArgs a = {kb, vb, xr, vm, eh, (int)p.T32, start, S, nope, vd, c.rope, (const uint16_t *)q, H, h0, heads, sc, out, out_f32};
        if (nope <= 64) lp_values<TYPE, 64>(st, a);
        else if (nope <= 128) lp_values<TYPE, 128>(st, a);
        else lp_values<TYPE, 256>(st, a);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int sw_launch_latent_prompt(hipStream_t st, const SwLatent &c, const int *pages, int max_pages, int start, const void *wk, const void *wv, int nope, int vd,
                            const void *q, int H, float scale, void *out, int out_f32, int S, void *scratch) {
    const float sc = (float)((double)scale * 1.4426950408889634074);   // the softmax in powers of two
    if (c.type == SW_KV_BF16) return lp_run<SW_KV_BF16>(st, c, pages, max_pages, start, wk, wv, nope, vd, q, H, sc, out, out_f32, S, (char *)scratch);
    return lp_run<SW_KV_F16>(st, c, pages, max_pages, start, wk, wv, nope, vd, q, H, sc, out, out_f32, S, (char *)scratch);
}
