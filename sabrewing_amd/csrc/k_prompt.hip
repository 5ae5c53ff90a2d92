// k_prompt.hip -- latent attention of a prompt's tokens, the expanded form: keys Wk[h] c_t and values Wv[h] c_t of every token
// are made once, then out[s, h] = sum_t p_t v_t, p = softmax over t <= start + s of scale * q[s, h] . (k_t, r_t).
//
// Three launches: cells gathered from their pages, keys and values of some heads expanded, their attention.  Against the
// absorbed form a pair of tokens costs 2 (nope + rope + v) instead of 2 (2 rank + rope) operations, and a token 2 rank (nope + v) once.
//
// Keys and values are held in f16, whatever the cache's type: 11 bits, where bf16's 8 would add errors as large as the
// output's own rounding three times over.  f16's range is met by powers of two: |k_d| <= |Wk_d| |c_t| (their 2-norms), so each
// head's keys are scaled by 2^(15 - a - b), a and b the exponents of the largest |Wk_d| and |c_t|, which keeps them
// below 2^15; a sum of many terms stays some 2^8 below that bound, and what is more than 2^20 smaller than the largest loses bits.
// Values alike; queries are scaled to 2^13.  The rotary part stays as the cache has it.
#include "sw_flash.h"

#define LP_NT 256
#define LP_ROPE 64

template <int TYPE> __device__ __forceinline__ float lp_float(uint32_t w, int hi) {
    if constexpr (TYPE == SW_KV_BF16) return __builtin_bit_cast(float, hi ? w & 0xFFFF0000u : w << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(hi ? w >> 16 : w));
}
// e with x < 2^e for a finite sum of squares x^2; far from the ends of f32
__device__ __forceinline__ int lp_exp(float x2) {
    const float x = sqrtf(x2);
    return x > 0.f ? min(max(ilogbf(x) + 1, -100), 100) : -100;
}

// Blocks 0 .. tiles - 1: 32 cells side by side in xl [tokens][rank] and xr [tokens][64] (zeros where there is no cell or no value), te: the
// exponent of the tile's largest norm, vm: which tokens have a cell.  Blocks behind them: we[2 h + kv], the exponent of a head's
// largest row norm of Wk or Wv.  Values that are no numbers do not count in a norm.
template <int TYPE>
__global__ __launch_bounds__(LP_NT) void k_prompt_gather(SwLatent c, const int *__restrict__ pages, int max_pages, int T, const uint16_t *__restrict__ wk,
                                                         const uint16_t *__restrict__ wv, int nope, int vd, uint16_t *__restrict__ xl,
                                                         uint16_t *__restrict__ xr, int *__restrict__ te, uint32_t *__restrict__ vm, int *__restrict__ we) {
    __shared__ float s_n[LP_NT / 64];
    __shared__ uint32_t s_v;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, tiles = (T + 31) / 32;
    float best = 0.f;
    auto square = [](sw_u32x4 y) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float f = lp_float<TYPE>(y[e], i), g = fabsf(f) < INFINITY ? f : 0.f;
                ss = __builtin_fmaf(g, g, ss);
            }
        return ss;
    };
    if ((int)blockIdx.x < tiles) {
        if (tid == 0) s_v = 0;
        __syncthreads();
#pragma unroll 2
        for (int i = wave; i < 32; i += LP_NT / 64) {
            const int t = blockIdx.x * 32 + i, pg = t >> c.psh;
            int page = -1;
            if (t < T && pg < max_pages) page = pages[pg];
            if (page >= c.n_pages) page = -1;
            const uint16_t *cell = (const uint16_t *)c.p + (int64_t)max(page, 0) * c.ps + (int64_t)(t & ((1 << c.psh) - 1)) * c.ts;
            sw_u32x4 a = {0, 0, 0, 0}, b = a;
            if (page >= 0 && 8 * lane < c.rank) a = *(const sw_u32x4 *)(cell + 8 * lane);
            if (page >= 0 && 8 * lane < c.rope) b = *(const sw_u32x4 *)(cell + c.rank + 8 * lane);
            if (8 * lane < c.rank) *(sw_u32x4 *)(xl + (int64_t)t * c.rank + 8 * lane) = a;
            if (lane < LP_ROPE / 8) *(sw_u32x4 *)(xr + (int64_t)t * LP_ROPE + 8 * lane) = b;
            float ss = square(a);
            for (int o = 32; o; o >>= 1) ss = ss + __shfl_xor(ss, o);
            best = fmaxf(best, ss);
            if (lane == 0 && page >= 0) atomicOr(&s_v, 1u << i);
        }
    } else {
        const int k = blockIdx.x - tiles, h = k >> 1, n = k & 1 ? vd : nope;
        const uint16_t *w = (k & 1 ? wv : wk) + (int64_t)h * n * c.rank;
#pragma unroll 4
        for (int i = wave; i < n; i += LP_NT / 64) {
            float ss = 8 * lane < c.rank ? square(*(const sw_u32x4 *)(w + (int64_t)i * c.rank + 8 * lane)) : 0.f;
            for (int o = 32; o; o >>= 1) ss = ss + __shfl_xor(ss, o);
            best = fmaxf(best, ss);
        }
    }
    if (lane == 0) s_n[wave] = best;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int i = 1; i < LP_NT / 64; i++) best = fmaxf(best, s_n[i]);
        if ((int)blockIdx.x < tiles) { te[blockIdx.x] = lp_exp(best); vm[blockIdx.x] = s_v; }
        else we[blockIdx.x - tiles] = lp_exp(best);
    }
}

// Keys and values of heads h0 ..: [head][tokens][n] in f16, times 2^eh.  A wave takes 64 outputs by 64 tokens, its
// operands straight from memory; a block 128 by 128.
template <int TYPE>
__global__ __launch_bounds__(LP_NT) void k_prompt_expand(const uint16_t *__restrict__ xl, const int *__restrict__ te, const int *__restrict__ we, int T32,
                                                         int rank, const uint16_t *__restrict__ wk, const uint16_t *__restrict__ wv, int nope, int vd,
                                                         int h0, uint16_t *__restrict__ kb, uint16_t *__restrict__ vb, int *__restrict__ eh) {
    __shared__ int s_e[LP_NT / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = fl_uni(tid >> 6), c = lane & 31, g = lane >> 5;
    const int tk = (nope + 127) / 128, tv = (vd + 127) / 128, hl = blockIdx.y / (tk + tv), by = blockIdx.y % (tk + tv), h = h0 + hl;
    const int kv = by >= tk, n = kv ? vd : nope;
    int e = -100;
    for (int i = tid; i < T32 / 32; i += LP_NT) e = max(e, te[i]);
    for (int o = 32; o; o >>= 1) e = max(e, __shfl_xor(e, o));
    if (lane == 0) s_e[wave] = e;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LP_NT / 64; i++) e = max(e, s_e[i]);
    e = min(max(15 - e - we[2 * h + kv], -120), 120);
    if (tid == 0 && blockIdx.x == 0) eh[2 * h + kv] = e;
    const int o0 = (kv ? by - tk : by) * 128 + (wave & 1) * 64, s0 = blockIdx.x * 128 + (wave >> 1) * 64;
    if (o0 >= n || s0 >= T32) return;
    const uint16_t *wp[2], *xp[2];
#pragma unroll
    for (int i = 0; i < 2; i++) wp[i] = (kv ? wv : wk) + ((int64_t)h * n + min(o0 + 32 * i + c, n - 1)) * rank + 8 * g;
#pragma unroll
    for (int i = 0; i < 2; i++) xp[i] = xl + (int64_t)min(s0 + 32 * i + c, T32 - 1) * rank + 8 * g;
    fl_f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = fl_f32x16{};
#pragma unroll 2
    for (int k = 0; k < rank; k += 16) {
        sw_u32x4 a[2], b[2];
#pragma unroll
        for (int i = 0; i < 2; i++) a[i] = *(const sw_u32x4 *)(wp[i] + k);
#pragma unroll
        for (int i = 0; i < 2; i++) b[i] = *(const sw_u32x4 *)(xp[i] + k);
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = fl_mfma<TYPE>(a[i], b[j], acc[i][j]);
    }
    const float f = ldexpf(1.f, e);
    uint16_t *y = (kv ? vb : kb) + (int64_t)hl * T32 * n;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int s = s0 + 32 * j + c;
        if (s >= T32) continue;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (o0 + 32 * i >= n) break;
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                uint32_t p[4];
#pragma unroll
                for (int q = 0; q < 4; q++) p[q] = __builtin_bit_cast(uint16_t, (_Float16)(acc[i][j][r + q] * f));
                *(uint2 *)(y + (int64_t)s * n + o0 + 32 * i + 2 * r + 4 * g) = make_uint2(p[0] | (p[1] << 16), p[2] | (p[3] << 16));
            }
        }
    }
}

// 32 rows of a head a wave; a tile holds 32 tokens' keys (their expanded part), values and rotary parts
template <int TYPE, int NOPE, int DV>
struct LpFl : Fl<SW_KV_F16, 1, NOPE, DV, false> {
    using Base = Fl<SW_KV_F16, 1, NOPE, DV, false>;
    static constexpr int ROPE_AT = Base::TB, TB = Base::TB + 32 * LP_ROPE * 2;
    sw_u32x4 R[LP_ROPE / 16];
    float scr;
    template <class Seen>
    __device__ __forceinline__ void tile(const char *t, bool whole, uint32_t bad, Seen seen, char *, int) {
        const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
        fl_f32x16 s = {};
#pragma unroll
        for (int i = 0; i < LP_ROPE / 16; i++)
            s = fl_mfma<TYPE>(*(const sw_u32x4 *)(t + ROPE_AT + c * (LP_ROPE * 2) + (((2 * i + h) ^ (c & 7)) * 16)), R[i], s);
        float x[16];
        this->scores(t, x, nullptr, 0);
#pragma unroll
        for (int j = 0; j < 16; j++) x[j] = __builtin_fmaf(s[j], scr, x[j]);
        if (!whole) {
            uint32_t met = 0;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int k = 8 * (j / 4) + 4 * h + j % 4;
                const bool in = seen(k);
                if (!in) x[j] = -INFINITY;
                else met |= bad >> k & 1;
            }
            if (met) this->l = NAN;
        }
        this->weights(x);
        this->outputs(t + 32 * Base::RBK, x);
    }
};
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
    __shared__ __align__(16) char sh[SHB];
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
    mx = fl_max2(mx);
    const int up = mx > 0.f && mx < INFINITY ? 13 - ilogbf(mx) : 0;
    const int ek = eh[2 * h], ev = eh[2 * h + 1];
    f.begin(ldexpf(sc0, -up - ek));
    f.scr = sc0;
#pragma unroll
    for (int k = 0; k < F::DKS; k++) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = ldexpf(lp_float<TYPE>(raw[k][e / 2], e & 1), up);
        f.query(k, y);
    }
#pragma unroll
    for (int k = 0; k < LP_ROPE / 16; k++) {
        f.R[k] = sw_u32x4{0, 0, 0, 0};
        if (16 * k + 8 * h2 < rope) f.R[k] = *(const sw_u32x4 *)(qp + nope + 16 * k + 8 * h2);
    }
    const char *kp = (const char *)(kb + (int64_t)hl * T32 * nope), *vp = (const char *)(vb + (int64_t)hl * T32 * vd);
    auto issue = [&](int tile, uint32_t lds) {
        int lane_ = lane;
        asm volatile("" : "+v"(lane_));                                // (the pieces' places are taken anew, not kept in registers)
        auto rows = [&](const char *src, int nch, int real, bool turn7, int loads, uint32_t to) {
            src += (int64_t)tile * 32 * real * 16;
#pragma unroll
            for (int k = 0; k < loads; k++) {
                const int kk = min(k * WC + wc, nch / 2 - 1), p = kk * 64 + lane_, tok = p / nch;
                const int ch = (p - tok * nch) ^ (turn7 ? tok & 7 : (tok >> 1) & 3);
                fl_load16(ch < real ? src + (tok * real + ch) * 16 : (const char *)&g_fl_zero, to + kk * 1024);
            }
        };
        rows(kp, F::NCK, nope / 8, F::MK == 7, LK, lds);
        rows(vp, F::NCV, vd / 8, F::MV == 7, LV, lds + 32 * F::RBK);
        rows((const char *)xr, LP_ROPE / 8, LP_ROPE / 8, true, LR, lds + F::ROPE_AT);
        return fl_entry((const int *)vm, tile) == -1;
    };
    auto whole = [&](int tile) { return tile * 32 + 31 <= start + r0; };
    auto seen = [&](int tile, int k) { return tile * 32 + k <= start + row && ((vm[tile] >> k) & 1); };
    fl_run<WC, WT, 1, NS, NL>(f, sh, nullptr, s_bad, 0, tiles, wave, true, issue, whole, seen);
    fl_end<WC, WT, 1>(f, sh, s_m, s_l, wave, [&](int col, int d, sw_f32x4 a, float, float sum) {
        const int s = r0 + col;
        if (s >= S || d >= vd) return;
#pragma unroll
        for (int e = 0; e < 4; e++) a[e] = sum == 0.f ? 0.f : ldexpf(a[e] / sum, -ev);
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
// heads expanded at a time: what they take stays about a GiB
struct LpPlan { int64_t T32, xl, xr, te, vm, we, eh, kb, vb, total; int heads; };
static LpPlan lp_plan(const SwLatent &c, int H, int nope, int vd, int64_t T) {
    LpPlan p;
    p.T32 = (T + 31) / 32 * 32;
    const int64_t one = p.T32 * (nope + vd) * 2, most = ((int64_t)1 << 30) / one;
    p.heads = (int)(most < 1 ? 1 : most < H ? most : H);
    int64_t at = 0;
    auto take = [&](int64_t n) { const int64_t x = at; at += (n + 255) / 256 * 256; return x; };
    p.xl = take(p.T32 * c.rank * 2);
    p.xr = take(p.T32 * LP_ROPE * 2);
    p.te = take(p.T32 / 8);
    p.vm = take(p.T32 / 8);
    p.we = take((int64_t)H * 8);
    p.eh = take((int64_t)H * 8);
    p.kb = take(p.heads * p.T32 * nope * 2);
    p.vb = take(p.heads * p.T32 * vd * 2);
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
    int *te = (int *)(A + p.te), *we = (int *)(A + p.we), *eh = (int *)(A + p.eh);
    uint32_t *vm = (uint32_t *)(A + p.vm);
    SW_LAUNCH(k_prompt_gather<TYPE>, dim3((unsigned)(p.T32 / 32 + 2 * H)), dim3(LP_NT), 0, st, c, pages, max_pages, T, (const uint16_t *)wk, (const uint16_t *)wv,
              nope, vd, xl, xr, te, vm, we);
    for (int h0 = 0; h0 < H; h0 += p.heads) {
        const int heads = H - h0 < p.heads ? H - h0 : p.heads, blocks = (nope + 127) / 128 + (vd + 127) / 128;
        SW_LAUNCH(k_prompt_expand<TYPE>, dim3((unsigned)((p.T32 + 127) / 128), (unsigned)(heads * blocks)), dim3(LP_NT), 0, st, xl, te, we, (int)p.T32, c.rank,
                  (const uint16_t *)wk, (const uint16_t *)wv, nope, vd, h0, kb, vb, eh);
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
