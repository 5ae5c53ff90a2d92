// k_latent.hip -- latent attention: a token's keys and values of every head come from one vector of `rank` values and
// `rope` turned ones, the cell of a paged cache.  Here: cells written, products for each head into the latent space and out of
// it, and the absorbed form of the attention, out[s, h] = sum_t p_t c_t, p = softmax over t <= pos[s] of
// scale * q[s, h] . (c_t, r_t), for queries that are in the latent space already.
#include "sw_flash.h"

// ------------------------------------------------------------------ cells and queries of new tokens ----
__device__ __forceinline__ void lt_angle(double freq, int pos, float factor, float &cs, float &sn) {
    double t = (double)pos * freq * 0.15915494309189533577;            // full turns, in 64 bits: far positions
    t = t - rint(t);
    sincospif((float)(t + t), &sn, &cs);
    cs = cs * factor;
    sn = sn * factor;
}
template <int TYPE>
__device__ __forceinline__ uint32_t lt_pack(float a, float b) {
    if constexpr (TYPE == SW_KV_BF16) return (uint32_t)sw_bf16_rne(a) | ((uint32_t)sw_bf16_rne(b) << 16);
    else return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16);
}
// eight values of a rotary part whose pairs are 4 u .. 4 u + 3: read as its halves' values 4 u .. 4 u + 3 or
// (interleaved) as 8 u .. 8 u + 7, turned (np pairs of the part, all or none: none are written as they are), and written in the same places
struct LtPairs { sw_f32x4 a, b; };
__device__ __forceinline__ LtPairs lt_read(const float *x, int u, int dims, bool inter) {
    LtPairs p;
    p.a = *(const sw_f32x4 *)(x + (inter ? 8 * u : 4 * u));
    p.b = *(const sw_f32x4 *)(x + (inter ? 8 * u + 4 : dims / 2 + 4 * u));
    return p;
}
template <int TYPE>
__device__ __forceinline__ void lt_turn(LtPairs p, int u, int dims, int np, bool inter, const float *s_cs, const float *s_sn, uint16_t *to) {
    const sw_f32x4 cs = *(const sw_f32x4 *)(s_cs + 4 * u), sn = *(const sw_f32x4 *)(s_sn + 4 * u);
    float x[4], y[4], v[4], w[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        x[e] = inter ? (e < 2 ? p.a[2 * e] : p.b[2 * e - 4]) : p.a[e];
        y[e] = inter ? (e < 2 ? p.a[2 * e + 1] : p.b[2 * e - 3]) : p.b[e];
        v[e] = np ? __builtin_fmaf(x[e], cs[e], -(y[e] * sn[e])) : x[e];
        w[e] = np ? __builtin_fmaf(y[e], cs[e], x[e] * sn[e]) : y[e];
    }
    if (inter) {
        *(sw_u32x4 *)(to + 8 * u) = sw_u32x4{lt_pack<TYPE>(v[0], w[0]), lt_pack<TYPE>(v[1], w[1]), lt_pack<TYPE>(v[2], w[2]), lt_pack<TYPE>(v[3], w[3])};
    } else {
        *(uint2 *)(to + 4 * u) = make_uint2(lt_pack<TYPE>(v[0], v[1]), lt_pack<TYPE>(v[2], v[3]));
        *(uint2 *)(to + dims / 2 + 4 * u) = make_uint2(lt_pack<TYPE>(w[0], w[1]), lt_pack<TYPE>(w[2], w[3]));
    }
}
// Blocks (row, y): y = 0 the row's cell, others UNITS units of eight values a thread of its query heads; the row's angles are taken once a block, in 64
// bits.  Bound by bytes: 1,024 rows of 128 heads (128 + 64), 151 MB, 36 us or 4.2 TB/s; one row of 16 heads 4.9 us, a launch.
#define LA_NT 256
template <int TYPE, int UNITS>
__global__ __launch_bounds__(LA_NT) void k_latent_append(SwLatent c, SwRows r, SwRope rope, const float *__restrict__ ckv, int64_t ldc,
                                                         const float *__restrict__ norm, float eps, const float *__restrict__ q, int64_t ldq, int H,
                                                         int nope, uint16_t *__restrict__ qn, int64_t nrs, int64_t nhs, uint16_t *__restrict__ qr,
                                                         int64_t rrs, int64_t rhs) {
    __shared__ __align__(16) float s_cs[32], s_sn[32];
    const int tid = threadIdx.x, s = blockIdx.x, dims = c.rope;
    const int pos = r.pos[s];
    if (pos < 0) return;
    const bool inter = rope.interleaved;
    auto angles = [&] {
        if (tid < rope.np) lt_angle(rope.freq[tid], pos, rope.factor, s_cs[tid], s_sn[tid]);
        __syncthreads();
    };
    if (blockIdx.y == 0) {                                             // wave 0 the latent, wave 1 the rotary part
        if (tid >= 128) { if (dims) __syncthreads(); return; }
        const float *x = ckv + (int64_t)s * ldc;
        const int lane = tid & 63, page = sw_page_of(r, c.n_pages, c.psh, r.seq ? r.seq[s] : s, pos);
        uint16_t *cell = (uint16_t *)c.p + (int64_t)page * c.ps + (int64_t)(pos & ((1 << c.psh) - 1)) * c.ts;
        sw_f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
        LtPairs p = {a, a};
        if (tid < 64 && 8 * lane < c.rank) { a = *(const sw_f32x4 *)(x + 8 * lane); b = *(const sw_f32x4 *)(x + 8 * lane + 4); }
        if (tid >= 64 && 8 * lane < dims) p = lt_read(x + c.rank, lane, dims, inter);
        if (dims) angles();
        if (tid < 64) {
            if (norm) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 4; e++) ss = __builtin_fmaf(a[e], a[e], __builtin_fmaf(b[e], b[e], ss));
                for (int o = 32; o; o >>= 1) ss = ss + __shfl_xor(ss, o);
                const float inv = 1.f / sqrtf(ss / (float)c.rank + eps);
                if (8 * lane < c.rank)
#pragma unroll
                    for (int e = 0; e < 4; e++) { a[e] = a[e] * inv * norm[8 * lane + e]; b[e] = b[e] * inv * norm[8 * lane + 4 + e]; }
            }
            if (page >= 0 && 8 * lane < c.rank)
                *(sw_u32x4 *)(cell + 8 * lane) = sw_u32x4{lt_pack<TYPE>(a[0], a[1]), lt_pack<TYPE>(a[2], a[3]), lt_pack<TYPE>(b[0], b[1]), lt_pack<TYPE>(b[2], b[3])};
        } else if (page >= 0 && 8 * lane < dims) {
            lt_turn<TYPE>(p, lane, dims, rope.np, inter, s_cs, s_sn, cell + c.rank);
        }
        return;
    }
    const int per = (nope + dims) / 8, units = H * per, u0 = (blockIdx.y - 1) * UNITS * LA_NT + tid;
    const float *x = q + (int64_t)s * ldq;
    LtPairs p[UNITS];
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        const int u = u0 + i * LA_NT, h = u / per, k = u - h * per;
        if (u >= units) break;
        const float *xh = x + (int64_t)h * (nope + dims);
        if (8 * k < nope) p[i] = {*(const sw_f32x4 *)(xh + 8 * k), *(const sw_f32x4 *)(xh + 8 * k + 4)};
        else p[i] = lt_read(xh + nope, k - nope / 8, dims, inter);
    }
    if (dims) angles();
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        const int u = u0 + i * LA_NT, h = u / per, k = u - h * per;
        if (u >= units) break;
        if (8 * k < nope)
            *(sw_u32x4 *)(qn + s * nrs + h * nhs + 8 * k) = sw_u32x4{lt_pack<TYPE>(p[i].a[0], p[i].a[1]), lt_pack<TYPE>(p[i].a[2], p[i].a[3]),
                                                                     lt_pack<TYPE>(p[i].b[0], p[i].b[1]), lt_pack<TYPE>(p[i].b[2], p[i].b[3])};
        else lt_turn<TYPE>(p[i], k - nope / 8, dims, rope.np, inter, s_cs, s_sn, qr + s * rrs + h * rhs);
    }
}

template <int TYPE>
static int la_launch(hipStream_t st, const SwLatent &c, const SwRows &r, const SwRope &rope, const float *ckv, int64_t ldc, const float *norm, float eps,
                     const float *q, int64_t ldq, int H, int nope, const SwHeads &qn, const SwHeads &qr, int S) {
    const int64_t units = (int64_t)H * (nope + c.rope) / 8;
    // four units a thread where the rows alone fill the chip
    const int n = S * ((units + 4 * LA_NT - 1) / (4 * LA_NT)) >= 512 ? 4 : 1;
    const dim3 grid((unsigned)S, (unsigned)(1 + (units + n * LA_NT - 1) / (n * LA_NT)));
    if (n == 4)
        SW_LAUNCH((k_latent_append<TYPE, 4>), grid, dim3(LA_NT), 0, st, c, r, rope, ckv, ldc, norm, eps, q, ldq, H, nope, (uint16_t *)qn.p, qn.rs, qn.hs,
                  (uint16_t *)qr.p, qr.rs, qr.hs);
    else
        SW_LAUNCH((k_latent_append<TYPE, 1>), grid, dim3(LA_NT), 0, st, c, r, rope, ckv, ldc, norm, eps, q, ldq, H, nope, (uint16_t *)qn.p, qn.rs, qn.hs,
                  (uint16_t *)qr.p, qr.rs, qr.hs);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int sw_launch_latent_append(hipStream_t st, const SwLatent &c, const SwRows &r, const SwRope &rope, const float *ckv, int64_t ldc, const float *norm,
                            float eps, const float *q, int64_t ldq, int H, int nope, const SwHeads &qn, const SwHeads &qr, int S) {
    if (c.type == SW_KV_BF16) return la_launch<SW_KV_BF16>(st, c, r, rope, ckv, ldc, norm, eps, q, ldq, H, nope, qn, qr, S);
    return la_launch<SW_KV_F16>(st, c, r, rope, ckv, ldc, norm, eps, q, ldq, H, nope, qn, qr, S);
}

// ------------------------------------------------------------------ a product for each head ----
// y[s, h] = W[h] x[s, h]: a wave takes OT x 32 outputs of a head and TT x 32 rows on the 32 x 32 matrix instructions, operands
// straight from memory (a row of W is read by one wave, or from the caches by the few that share its outputs).  Up to 64 rows a wave takes 32 by 32,
// as there are few waves; beyond 64 by 64, half the reads.  Bound by W's bytes: 128 heads of 512 x 128, one row 6.0 us (16.8 MB, 2.8 TB/s with the
// launch), 64 rows of 128 x 512 with 32-bit outputs 11.0 us (29 MB), 256 rows 22 us
// and of 512 x 128 27 us (67 and 59 MB, 195 and 156 TFLOP/s).  Two steps' operands at a time instead of eight: 6.6 and 12.7.
#define LH_NT 256
template <int TYPE, bool YF32, int OT, int TT>
__global__ __launch_bounds__(LH_NT) void k_latent_heads(const uint16_t *__restrict__ x, int64_t xrs, int64_t xhs, const uint16_t *__restrict__ W, int H,
                                                        int n_in, int n_out, void *__restrict__ y, int64_t yrs, int64_t yhs, int S) {
    const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
    const int to = (n_out / 32 + OT - 1) / OT, ts = (S + 32 * TT - 1) / (32 * TT);
    // a die takes neighbouring blocks: those of a head's other rows find its W in their cache
    const unsigned n8 = gridDim.x & ~7u, block = blockIdx.x < n8 ? (blockIdx.x & 7) * (n8 >> 3) + (blockIdx.x >> 3) : blockIdx.x;
    const int64_t w = (int64_t)block * (LH_NT / 64) + fl_uni((int)(threadIdx.x >> 6));
    if (w >= (int64_t)H * to * ts) return;
    const int o0 = (int)(w % to) * OT * 32, s0 = (int)(w / to % ts) * TT * 32, h = (int)(w / to / ts);
    const uint16_t *wp[OT], *xp[TT];
#pragma unroll
    for (int i = 0; i < OT; i++) wp[i] = W + ((int64_t)h * n_out + min(o0 + 32 * i + c, n_out - 1)) * n_in + 8 * g;
#pragma unroll
    for (int i = 0; i < TT; i++) xp[i] = x + min(s0 + 32 * i + c, S - 1) * xrs + h * xhs + 8 * g;
    fl_f32x16 acc[OT][TT];
#pragma unroll
    for (int i = 0; i < OT; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) acc[i][j] = fl_f32x16{};
    // KC steps' operands are fetched while those before are multiplied: a wave has 16 loads or more on their way
    constexpr int KC = 8 / OT;
    const int steps = n_in / 16;
    sw_u32x4 a[2][KC][OT], b[2][KC][TT];
    auto fetch = [&](int k0, int to) {
#pragma unroll
        for (int u = 0; u < KC; u++) {
            const int k = min(k0 + u, steps - 1) * 16;
#pragma unroll
            for (int i = 0; i < OT; i++) a[to][u][i] = *(const sw_u32x4 *)(wp[i] + k);
#pragma unroll
            for (int i = 0; i < TT; i++) b[to][u][i] = *(const sw_u32x4 *)(xp[i] + k);
        }
    };
    auto multiply = [&](int k0, int from) {
#pragma unroll
        for (int u = 0; u < KC; u++) {
            if (k0 + u >= steps) break;
#pragma unroll
            for (int i = 0; i < OT; i++)
#pragma unroll
                for (int j = 0; j < TT; j++) acc[i][j] = fl_mfma<TYPE>(a[from][u][i], b[from][u][j], acc[i][j]);
        }
    };
    fetch(0, 0);
#pragma unroll 1
    for (int k = 0; k < steps; k += 2 * KC) {
        if (k + KC < steps) fetch(k + KC, 1);
        multiply(k, 0);
        if (k + KC >= steps) break;
        if (k + 2 * KC < steps) fetch(k + 2 * KC, 0);
        multiply(k + KC, 1);
    }
#pragma unroll
    for (int j = 0; j < TT; j++) {
        const int s = s0 + 32 * j + c;
        if (s >= S) continue;
#pragma unroll
        for (int i = 0; i < OT; i++) {
            if (o0 + 32 * i >= n_out) break;
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int64_t at = s * yrs + h * yhs + o0 + 32 * i + 2 * e + 4 * g;
                if constexpr (YF32) *(sw_f32x4 *)((float *)y + at) = sw_f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
                else *(uint2 *)((uint16_t *)y + at) = make_uint2(lt_pack<TYPE>(acc[i][j][e], acc[i][j][e + 1]), lt_pack<TYPE>(acc[i][j][e + 2], acc[i][j][e + 3]));
            }
        }
    }
}
template <int TYPE, bool YF32, int OT, int TT>
static void lh_launch(hipStream_t st, const SwHeads &x, const void *W, int H, int n_in, int n_out, const SwHeads &y, int S) {
    const int64_t waves = (int64_t)H * ((n_out / 32 + OT - 1) / OT) * ((S + 32 * TT - 1) / (32 * TT));
    SW_LAUNCH((k_latent_heads<TYPE, YF32, OT, TT>), dim3((unsigned)((waves + 3) / 4)), dim3(LH_NT), 0, st, (const uint16_t *)x.p, x.rs, x.hs, (const uint16_t *)W, H,
              n_in, n_out, y.p, y.rs, y.hs, S);
}
template <int TYPE, bool YF32>
static void lh_form(hipStream_t st, const SwHeads &x, const void *W, int H, int n_in, int n_out, const SwHeads &y, int S) {
    if (S <= 64) lh_launch<TYPE, YF32, 1, 1>(st, x, W, H, n_in, n_out, y, S);
    else lh_launch<TYPE, YF32, 2, 2>(st, x, W, H, n_in, n_out, y, S);
}
int sw_launch_latent_heads(hipStream_t st, int type, const SwHeads &x, const void *W, int H, int n_in, int n_out, const SwHeads &y, int y_f32, int S) {
    if (type == SW_KV_BF16) {
        if (y_f32) lh_form<SW_KV_BF16, true>(st, x, W, H, n_in, n_out, y, S);
        else lh_form<SW_KV_BF16, false>(st, x, W, H, n_in, n_out, y, S);
    } else {
        if (y_f32) lh_form<SW_KV_F16, true>(st, x, W, H, n_in, n_out, y, S);
        else lh_form<SW_KV_F16, false>(st, x, W, H, n_in, n_out, y, S);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// ------------------------------------------------------------------ the absorbed form ----
// Heads are the columns, a cell is key and value of all of them: 2 (2 rank + rope) operations a head for 2 (rank + rope) bytes.  Queries and outputs of 512
// values by 32 columns are more than a wave's registers, so that waves share columns (sw_flash.h).  Rows' tiles are laid end to end and dealt to
// 256 blocks as trees' are.  Bf16, rank 512 + 64: 32 rows of 128 heads over 100 to 16,384 cells 139 to 158 us by the lengths drawn: matrix
// instructions a quarter of the cycles, vector ones 16 %, LDS 27 %, the rest waits at two barriers a tile of eight waves on a CU; the join's 12 us
// within.  One row of 16 heads over 1,500 cells 18 us: a chain of waits, and the join's launch.
//
// The softmax's weights are rounded once to the cells' type, 8 bits in bf16.  Weights in two parts double the second product, 13 us
// more (158 -> 171) without what their exchange would add; they would bring the outputs' error, relative to 64 bits, from 0.0019 to the 0.0017 that
// the outputs' own rounding to bf16 leaves.  attn_paged and attn_tree, whose outputs are of 32 bits, keep 24.
#define LN_ROPE 64                                                     // a cell's rotary part in LDS: the rest of it zeros
#define LN_SPLIT 256                                                   // beyond so many rows none is split: rows of like lengths fill the chip (of ragged ones the longest is waited for)
// waves that share 32 heads (a share of the outputs is whole pairs of 32 values), and tiles in LDS
template <int R> constexpr int ln_split() { return R % 256 == 0 ? 4 : 2; }
template <int TYPE, int R> using LnFl = Fl<TYPE, 1, R + LN_ROPE, R, true, ln_split<R>()>;
template <int R, int WC> constexpr int ln_ns() {
    constexpr int n = (156 * 1024 - WC * ln_split<R>() * 5 * 1024) / (32 * (R + LN_ROPE) * 2);
    return n > 4 ? 4 : n;
}
struct LnRow { int seq, last; };                                       // (last: -1 for every free place, so that it has no tiles)
__device__ __forceinline__ LnRow ln_row(const SwLatent &c, const SwRows &r, int s) {
    LnRow x;
    x.seq = r.seq ? r.seq[s] : s;
    x.last = x.seq < 0 || x.seq >= r.n_seqs ? -1 : max(-1, min(r.pos[s], (r.max_pages << c.psh) - 1));
    return x;
}
template <int TYPE, int R, int WC>
__global__ __launch_bounds__((64 * WC * ln_split<R>())) void k_latent(SwLatent c, SwRows r, const uint16_t *__restrict__ q, int S, int H, float sc,
                                                                uint16_t *__restrict__ out, float *__restrict__ part, int B) {
    using F = LnFl<TYPE, R>;
    constexpr int SPLIT = ln_split<R>(), NW = WC * SPLIT, NT = 64 * NW;
    constexpr int CW = 32 * WC, NS = ln_ns<R, WC>(), NL = (F::NCK / 2 + NW - 1) / NW;
    constexpr int SHT = NS * F::TB + NW * F::XB, SHB = SHT > fl_end_bytes<F, NW>() ? SHT : fl_end_bytes<F, NW>();
    static_assert(SHB <= 157 * 1024 && (NS < 3 ? 0 : NS - 2) * NL < 64, "LDS, and loads that a wave can count");
    __shared__ __align__(256) char sh[SHB];
    __shared__ float s_m[NW][32], s_l[NW][32];
    __shared__ uint32_t s_bad[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = fl_uni(tid >> 6), wc = wave / SPLIT, share = wave % SPLIT, cl = lane & 31, h2 = lane >> 5;
    const int per = (H + CW - 1) / CW, hg = blockIdx.x % per, b = blockIdx.x / per, c0 = hg * CW, nh = min(CW, H - c0), width = c.rank + c.rope;
    auto count = [&](int s) { return (ln_row(c, r, s).last >> 5) + 1; };
    const int blocks = B ? B : S;
    for (int s = b; s < S; s += blocks)                                // rows without any cell: zeros
        if (ln_row(c, r, s).last < 0)
            for (int k = tid; k < nh * (R / 8); k += NT) *(sw_u32x4 *)(out + ((int64_t)s * H + c0) * R + 8 * k) = sw_u32x4{0, 0, 0, 0};
    int64_t at = 0, end = 1, before = 0;
    int s = b;
    if (B) {
        const FlDeal deal = fl_deal(S, B, (int64_t)H * R, count);
        at = (int64_t)b * deal.q;
        end = at + deal.q < deal.N ? at + deal.q : deal.N;
        if (at >= end) return;
        s = fl_find(S, at, before, count);
    }
    const int pmask = (1 << c.psh) - 1;
    F f;
    for (; at < end; s++) {
        LnRow x = ln_row(c, r, s);
        x.seq = fl_uni(x.seq); x.last = fl_uni(x.last);
        const int tiles = (x.last >> 5) + 1;
        if (!B) { end = tiles; if (tiles == 0) return; }
        if (tiles == 0) continue;
        const int from = (int)(at - before), len = (int)(end - at < tiles - from ? end - at : tiles - from);
        before += tiles;
        at += len;
        const int head = c0 + wc * 32 + cl;
        const uint16_t *qp = q + ((int64_t)s * H + head) * width;
        f.begin(sc, share);
#pragma unroll
        for (int k = 0; k < F::DKS; k++) {
            sw_u32x4 y = {0, 0, 0, 0};
            const int d = 16 * (SPLIT * k + share) + 8 * h2;
            if (head < H && d < width) y = *(const sw_u32x4 *)(qp + d);
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = F::signed_by(y[e], sc);
            f.Q[0][k] = y;
        }
        const int *table = r.table + (int64_t)x.seq * r.max_pages;
        auto issue = [&](int tile, uint32_t lds) {
            const int t0 = tile * 32;
            const FlPages g = fl_pages(table, r.max_pages, c.n_pages, c.psh, t0);
            if (c.psh >= 5 && width == R + LN_ROPE && c.ts < 1 << 25)  // one page, whole rows, not far apart
                fl_rows<F::NCK, F::MK, NW, NL>((const char *)c.p + ((int64_t)max(g.p[0], 0) * c.ps + (int64_t)(t0 & pmask) * c.ts) * 2, (uint32_t)c.ts * 2,
                                               wave, lane, lds);
            else
                fl_rows_any<F::NCK, F::MK, NW, NL>((const char *)c.p, g, c.ps * 2, c.ts * 2, t0, pmask, width / 8, wave, lane, lds);
            return g.ok;
        };
        auto whole = [&](int tile) { return tile * 32 + 31 <= x.last; };
        auto seen = [&](int tile, int k) {
            const int tok = tile * 32 + k, pg = tok >> c.psh;
            const int page = pg < r.max_pages ? table[pg] : -1;
            return tok <= x.last && page >= 0 && page < c.n_pages;
        };
        fl_run_split<WC, SPLIT, NS, NL>(f, sh, sh + NS * F::TB, s_bad, from, from + len, wave, issue, whole, seen);
        const bool all = len == tiles;
        float *pp = all ? nullptr : part + ((int64_t)hg * 2 * B + fl_slot(b, from)) * CW * (R + 4);
        fl_end<WC, 1, SPLIT>(f, sh, s_m, s_l, wave, [&](int col, int d, sw_f32x4 a, float mx, float sum) {
            if (col >= nh) return;
            if (all) {
#pragma unroll
                for (int e = 0; e < 4; e++) a[e] = sum == 0.f ? 0.f : a[e] * (1.f / sum);
                *(uint2 *)(out + ((int64_t)s * H + c0 + col) * R + d) = make_uint2(lt_pack<TYPE>(a[0], a[1]), lt_pack<TYPE>(a[2], a[3]));
            } else {
                float *o = pp + col * (R + 4);
                *(sw_f32x4 *)(o + 4 + d) = a;
                if (d == 0) { o[0] = mx; o[1] = sum; }
            }
        });
        if (!B) return;
    }
}

// The parts of a row's heads joined: a wave 256 values of a head at a time
template <int TYPE, int R>
__global__ __launch_bounds__(FL_NT) void k_latent_join(SwLatent c, SwRows r, int S, int H, const float *__restrict__ part, int B, int CW,
                                                       uint16_t *__restrict__ out) {
    constexpr int NV = (R + 255) / 256;
    const int s = blockIdx.y, k0 = fl_uni((int)(blockIdx.x * FL_NW + (threadIdx.x >> 6)));
    auto count = [&](int i) { return (ln_row(c, r, i).last >> 5) + 1; };
    const int tiles = count(s);
    if (tiles == 0 || k0 >= H * NV) return;
    const FlDeal deal = fl_deal(S, B, (int64_t)H * R, count);
    const int64_t before = fl_before(s, count);
    const int b0 = (int)(before / deal.q), parts = (int)((before + tiles - 1) / deal.q) - b0 + 1;
    if (parts < 2) return;
    for (int k = k0; k < H * NV; k += gridDim.x * FL_NW) {
        const int head = k / NV, v0 = k % NV * 256, d = v0 + (threadIdx.x & 63) * 4;
        const sw_f32x4 a = fl_join<R>(part + (((int64_t)(head / CW) * 2 * B + fl_slot(b0, 0)) * CW + head % CW) * (R + 4), (int64_t)CW * (R + 4), parts, v0);
        if (d < R && (threadIdx.x & 63) * 4 < R) *(uint2 *)(out + ((int64_t)s * H + head) * R + d) = make_uint2(lt_pack<TYPE>(a[0], a[1]), lt_pack<TYPE>(a[2], a[3]));
    }
}

// Columns of a block (32 times wc) and blocks of each group of heads; 0: a block a row.  64 columns a block where there are more than 32: 128 heads 151 us
// at the time, in blocks of 128 columns (half the reads of cells, queries in LDS for want of registers) 20 more, with two waves to share 64 columns 40 more.
struct LnPlan { int wc, groups, B; };
static LnPlan ln_plan(const SwLatent &c, const SwRows &r, int H, int S) {
    LnPlan p;
    p.wc = H <= 32 ? 1 : 2;
    p.groups = (H + 32 * p.wc - 1) / (32 * p.wc);
    const int64_t tiles = ((((int64_t)r.max_pages << c.psh) + 31) / 32) * S;
    const int n = 256 / p.groups;
    p.B = S > LN_SPLIT ? 0 : (int)(n < 1 ? 1 : n < tiles ? n : tiles);
    return p;
}
int64_t sw_latent_part_floats(const SwLatent &c, const SwRows &r, int H, int S) {
    const LnPlan p = ln_plan(c, r, H, S);
    return p.B > 1 ? (int64_t)p.groups * 2 * p.B * 32 * p.wc * (c.rank + 4) : 0;
}
template <int TYPE, int R>
static int ln_launch(hipStream_t st, const SwLatent &c, const SwRows &r, const uint16_t *q, int H, float sc, uint16_t *out, int S, float *part) {
    const LnPlan p = ln_plan(c, r, H, S);
    const int64_t grid = (int64_t)(p.B ? p.B : S) * p.groups;
    if (grid >= (int64_t)1 << 31 || (p.B > 1 && !part)) return -1;
    if (p.wc == 1) SW_LAUNCH((k_latent<TYPE, R, 1>), dim3((unsigned)grid), dim3(64 * ln_split<R>()), 0, st, c, r, q, S, H, sc, out, part, p.B);
    else SW_LAUNCH((k_latent<TYPE, R, 2>), dim3((unsigned)grid), dim3(128 * ln_split<R>()), 0, st, c, r, q, S, H, sc, out, part, p.B);
    if (p.B > 1) {
        constexpr int NV = (R + 255) / 256;
        SW_LAUNCH((k_latent_join<TYPE, R>), dim3((unsigned)fl_join_blocks((H * NV + FL_NW - 1) / FL_NW, S), (unsigned)S), dim3(FL_NT), 0, st, c, r, S, H, part, p.B, 32 * p.wc, out);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
template <int TYPE>
static int ln_dispatch(hipStream_t st, const SwLatent &c, const SwRows &r, const uint16_t *q, int H, float sc, uint16_t *out, int S, float *part) {
    switch (c.rank) {
    case 128: return ln_launch<TYPE, 128>(st, c, r, q, H, sc, out, S, part);
    case 256: return ln_launch<TYPE, 256>(st, c, r, q, H, sc, out, S, part);
    case 384: return ln_launch<TYPE, 384>(st, c, r, q, H, sc, out, S, part);
    case 512: return ln_launch<TYPE, 512>(st, c, r, q, H, sc, out, S, part);
    }
    return -1;
}
int sw_launch_latent(hipStream_t st, const SwLatent &c, const SwRows &r, const void *q, int H, float scale, void *out, int S, float *part) {
    const float sc = (float)((double)scale * 1.4426950408889634074);   // the softmax in powers of two
    if (c.type == SW_KV_BF16) return ln_dispatch<SW_KV_BF16>(st, c, r, (const uint16_t *)q, H, sc, (uint16_t *)out, S, part);
    return ln_dispatch<SW_KV_F16>(st, c, r, (const uint16_t *)q, H, sc, (uint16_t *)out, S, part);
}
