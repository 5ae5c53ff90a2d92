// k_tree.hip -- attention of trees of drafted tokens over a paged cache: row s is a node of a tree,
// out[s, h] = sum_t p_t v_t, p = softmax over t < base (within the window) and the cells base + j that bit j of
// sees[s] names, of scale * q[s, h] . k_t.
//
// A tree's nodes and the query heads of a cache head are the columns of one product, so that its cells are read once.  32-bit queries and weights
// meet 16-bit cells in parts of the cells' type, products exact in 32-bit sums (bf16 three parts, f16 two): that is what bounds a batch, each
// cell costing three times the matrix instructions, and splitting the weights about as many cycles of vector instructions.
// Trees' tiles are laid end to end and dealt to the blocks in equal shares, the parts of a tree joined by a second launch.  Bf16, 32 heads over 8
// of 128: 16 trees of up to 26 nodes over 500 to 12,000 cells 147 to 164 us by the lengths drawn (matrix instructions 36 % of the cycles, vector
// 35 %); one tree of 8 nodes over 700 cells 24 us, 19 of them a chain of waits in 22 blocks of one tile a cache head, 6 the join, over 60,000
// cells 73 us (3.4 TB/s).  8 trees over up to 6,000 f32 cells 154 us.  Two parts of a weight (16 bits) took 8 us less and doubled the error.
//
// Registers: bf16 of 256 (both forms), and with up to 32 columns bf16 of 128 and 192 and f16 of 224, spill 14 to 43 of them, those of 256 within the
// tiles' loop (a reload waits for the tiles on their way: time, not results).  f32 of 96, 128 and 160 and f16 of 160 with up to 32 columns run
// one block a CU where tr_occ allows two, and have half of the blocks waiting.
#include "sw_flash.h"

// tree i: its rows, and the cells that any of them may attend to
struct TrTree { int row, n, base, seq, first, last; };
__device__ __forceinline__ TrTree tr_tree(const SwKv &c, const SwTrees &t, int i, int S, int window) {
    TrTree x;
    x.row = t.first[i];
    const int end = t.first[i + 1];
    x.n = x.row < 0 || x.row >= S || end <= x.row ? 0 : min(min(end, S) - x.row, t.max_nodes);
    x.base = t.base[i];
    x.seq = t.seq ? t.seq[i] : i;
    const int limit = (t.max_pages << c.psh) - 1;                      // (the host keeps that below 2^30)
    x.first = window > 0 && x.base >= window ? x.base - window + 1 : 0;
    x.last = x.base < 0 || x.seq < 0 || x.seq >= t.n_seqs || x.n == 0 ? -1 : min(min(x.base, limit) + x.n - 1, limit);
    return x;
}
// tiles of 32 cells that columns from c0 on (G a node) of a tree have to take
__device__ __forceinline__ int tr_tiles(const TrTree &x, int G, int c0) {
    return x.last < x.first || x.n * G <= c0 ? 0 : (x.last >> 5) - (x.first >> 5) + 1;
}

// outputs of a tree with all its nodes
__host__ __device__ inline int64_t tr_values(const SwTrees &t, int Hq, int dh) { return (int64_t)t.max_nodes * Hq * dh; }
template <int TYPE> constexpr int tr_np() { return TYPE == SW_KV_F32 ? 1 : TYPE == SW_KV_BF16 ? 3 : 2; }
template <int TYPE, int DH> using TrFl = Fl<TYPE, tr_np<TYPE>(), DH, DH, false>;
template <int TYPE, int DH> constexpr int tr_occ() {
    return tr_np<TYPE>() * TrFl<TYPE, DH>::DKS * 4 + TrFl<TYPE, DH>::NO * 16 <= 176 ? 2 : 1;
}
template <int TYPE, int DH, int WC> constexpr int tr_ns() {
    constexpr int n = (tr_occ<TYPE, DH>() == 2 ? 78 : 156) * 1024 / (FL_NW / WC * TrFl<TYPE, DH>::TB);
    return n < 1 ? 1 : n > 4 ? 4 : n;
}
// the fewest waves that share columns: one, or two where four tiles do not fit in LDS
template <int TYPE, int DH> constexpr int tr_wc() { return 4 * TrFl<TYPE, DH>::TB <= 156 * 1024 ? 1 : 2; }

template <int TYPE, int DH, int WC>
__global__ __launch_bounds__(FL_NT, (tr_occ<TYPE, DH>())) void k_tree(SwKv c, SwTrees t, const float *__restrict__ q, int S, int Hq, float sc0,
                                                                    int window, float *__restrict__ out, float *__restrict__ part, int B) {
    using F = TrFl<TYPE, DH>;
    constexpr int CW = 32 * WC, NS = tr_ns<TYPE, DH, WC>(), WT = FL_NW / WC, ES = F::ES;
    constexpr int LK = (F::NCK / 2 + WC - 1) / WC, LV = (F::NCV / 2 + WC - 1) / WC;                    // loads of a wave
    constexpr int SHT = WT * NS * F::TB, SHB = SHT > fl_end_bytes<F, FL_NW>() ? SHT : fl_end_bytes<F, FL_NW>();
    static_assert(SHB <= 158 * 1024 && (NS < 3 ? 0 : NS - 2) * (LK + LV) < 64, "LDS, and loads that a wave can count");
    __shared__ __align__(256) char sh[SHB];
    __shared__ float s_m[FL_NW][32], s_l[FL_NW][32];
    __shared__ uint32_t s_bad[2 * FL_NW];
    __shared__ int s_lo;
    const int tid = threadIdx.x, lane = tid & 63, wave = fl_uni(tid >> 6), wc = wave % WC, cl = lane & 31, h = lane >> 5;
    const int G = Hq / c.Hkv, ncg = (t.max_nodes * G + CW - 1) / CW, per = c.Hkv * ncg;
    const int hg = blockIdx.x % per, b = blockIdx.x / per, hk = hg / ncg, c0 = hg % ncg * CW;
    auto count = [&](int i) { return tr_tiles(tr_tree(c, t, i, S, window), G, c0); };
    for (int i = b; i < t.n_trees; i += B) {                           // trees without any cell: zeros
        const TrTree x = tr_tree(c, t, i, S, window);
        if (x.last < x.first)
            for (int k = tid; k < min(CW, x.n * G - c0) * (DH / 4); k += FL_NT) {
                const int ci = c0 + k / (DH / 4);
                *(sw_f32x4 *)(out + ((int64_t)(x.row + ci / G) * Hq + hk * G + ci % G) * DH + k % (DH / 4) * 4) = sw_f32x4{0.f, 0.f, 0.f, 0.f};
            }
    }
    const FlDeal deal = fl_deal(t.n_trees, B, tr_values(t, Hq, c.dh), count);
    int64_t at = (int64_t)b * deal.q, before = 0;
    const int64_t end = at + deal.q < deal.N ? at + deal.q : deal.N;
    if (at >= end) return;
    int i = fl_find(t.n_trees, at, before, count);
    const int pmask = (1 << c.psh) - 1;
    const char *kp = (const char *)c.k + (int64_t)hk * c.hs * ES, *vp = (const char *)c.v + (int64_t)hk * c.hs * ES;
    const int64_t psb = c.ps * ES, tsb = c.ts * ES;
    const bool near = tsb < (int64_t)1 << 26;
    F f;
    for (; at < end; i++) {
        TrTree x = tr_tree(c, t, i, S, window);
        x.row = fl_uni(x.row); x.n = fl_uni(x.n); x.base = fl_uni(x.base); x.seq = fl_uni(x.seq); x.first = fl_uni(x.first); x.last = fl_uni(x.last);
        const int tiles = tr_tiles(x, G, c0);
        if (tiles == 0) continue;
        const int from = (int)(at - before), len = (int)(end - at < tiles - from ? end - at : tiles - from);
        const int ta = (x.first >> 5) + from;
        before += tiles;
        at += len;
        // this lane's column
        const int ci = c0 + wc * 32 + cl, node = ci / G, row = x.row + node;
        const bool mine = node < x.n;
        const float *qp = q + ((int64_t)row * Hq + hk * G + ci % G) * DH;
        uint64_t sees = 0;
        int lo = 0;                                                    // the column's first cell
        if (mine) {
            sees = t.sees[row];
            if (window > 0) lo = max(0, max(t.pos[row], x.base) - window + 1);
        }
        float sc = sc0;
        int up = 0;                                                    // the power of two that f16 queries are scaled by
        if constexpr (TYPE == SW_KV_F16) {
            float mx = 0.f;
#pragma unroll
            for (int k = 0; k < F::DKS; k++)
#pragma unroll
                for (int j = 0; j < 2; j++)
                    if (mine) {
                        const sw_f32x4 y = *(const sw_f32x4 *)(qp + 16 * k + 8 * h + 4 * j);
#pragma unroll
                        for (int e = 0; e < 4; e++) mx = fmaxf(mx, fabsf(y[e]));
                    }
            mx = fl_max2(mx);
            up = mx > 0.f && mx < INFINITY ? 13 - ilogbf(mx) : 0;
            sc = ldexpf(sc0, -up);
            if (fabsf(sc) == INFINITY && fabsf(sc0) < INFINITY) sc = copysignf(3.402823466e38f, sc0);
        }
        f.begin(sc);
#pragma unroll
        for (int k = 0; k < F::DKS; k++) {
            if constexpr (F::F32) {
                sw_f32x4 y = {0.f, 0.f, 0.f, 0.f};
                if (mine) y = *(const sw_f32x4 *)(qp + 8 * k + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; e++) f.Q[0][k][e] = F::signed_by(__builtin_bit_cast(uint32_t, (float)y[e]), sc);
            } else {
                float y[8];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    sw_f32x4 z = {0.f, 0.f, 0.f, 0.f};
                    if (mine) z = *(const sw_f32x4 *)(qp + 16 * k + 8 * h + 4 * j);
#pragma unroll
                    for (int e = 0; e < 4; e++) y[4 * j + e] = TYPE == SW_KV_F16 ? ldexpf(z[e], up) : z[e];
#pragma unroll
                    for (int e = 0; e < 4; e++) y[4 * j + e] = sc == 0.f ? 0.f : sc < 0.f ? -y[4 * j + e] : y[4 * j + e];
                }
                f.query(k, y);
            }
        }
        const int *table = t.table + (int64_t)x.seq * t.max_pages;
        const bool columns = c0 + wc * 32 < x.n * G;
        auto issue = [&](int tile, uint32_t lds) {
            const int t0 = tile * 32;
            int lane_ = lane;
            if constexpr (WC < 4) asm volatile("" : "+v"(lane_));      // (the pieces' places are taken anew, not kept in registers)
            const FlPages g = fl_pages(table, t.max_pages, c.n_pages, c.psh, t0);
            if (near && c.psh >= 5) {                                  // one page, rows not far apart
                const int64_t at = (int64_t)max(g.p[0], 0) * psb + (int64_t)(t0 & pmask) * tsb;
                fl_rows<F::NCK, F::MK, WC, LK>(kp + at, (uint32_t)tsb, wc, lane_, lds);
                fl_rows<F::NCV, F::MV, WC, LV>(vp + at, (uint32_t)tsb, wc, lane_, lds + 32 * F::RBK);
            } else {
                fl_rows_any<F::NCK, F::MK, WC, LK>(kp, g, psb, tsb, t0, pmask, F::NCK, wc, lane_, lds);
                fl_rows_any<F::NCV, F::MV, WC, LV>(vp, g, psb, tsb, t0, pmask, F::NCV, wc, lane_, lds + 32 * F::RBK);
            }
            return g.ok;
        };
        int lo_all = 0;                                                // the last cell at which a column's window begins
        if (window > 0) {
            __syncthreads();
            if (tid == 0) s_lo = 0;
            __syncthreads();
            if (mine) atomicMax(&s_lo, lo);
            __syncthreads();
            lo_all = fl_uni(s_lo);
        }
        auto whole = [&](int tile) { return tile * 32 + 31 < x.base && tile * 32 >= lo_all; };
        auto seen = [&](int tile, int k) {
            const int tok = tile * 32 + k, j = tok - x.base;
            const int pg = tok >> c.psh;
            const int page = pg < t.max_pages ? table[pg] : -1;
            return tok <= x.last && page >= 0 && page < c.n_pages && (j < 0 ? tok >= lo : j < x.n && ((sees >> j) & 1));
        };
        fl_run<WC, WT, NS, LK + LV>(f, sh, s_bad, ta, ta + len, wave, columns, issue, whole, seen);
        const bool all = len == tiles;
        float *pp = all ? nullptr : part + ((int64_t)hg * 2 * B + fl_slot(b, from)) * CW * (DH + 4);
        fl_end<WC, WT, 1>(f, sh, s_m, s_l, wave, [&](int col, int d, sw_f32x4 a, float mx, float sum) {
            const int ck = c0 + col;
            if (ck >= x.n * G) return;
            if (all) {
#pragma unroll
                for (int e = 0; e < 4; e++) a[e] = sum == 0.f ? 0.f : a[e] * (1.f / sum);
                *(sw_f32x4 *)(out + ((int64_t)(x.row + ck / G) * Hq + hk * G + ck % G) * DH + d) = a;
            } else {
                float *o = pp + col * (DH + 4);
                *(sw_f32x4 *)(o + 4 + d) = a;
                if (d == 0) { o[0] = mx; o[1] = sum; }
            }
        });
    }
}

// The parts of a tree's columns joined: a wave a column at a time
template <int DH>
__global__ __launch_bounds__(FL_NT) void k_tree_join(SwKv c, SwTrees t, int S, int Hq, int window, const float *__restrict__ part, int B,
                                                     int CW, int nb, float *__restrict__ out) {
    const int G = Hq / c.Hkv, ncg = (t.max_nodes * G + CW - 1) / CW, lane = threadIdx.x & 63;
    const int hg = blockIdx.x / nb, i = blockIdx.y, hk = hg / ncg, c0 = hg % ncg * CW, col0 = fl_uni((int)(blockIdx.x % nb * FL_NW + (threadIdx.x >> 6)));
    auto count = [&](int k) { return tr_tiles(tr_tree(c, t, k, S, window), G, c0); };
    const TrTree x = tr_tree(c, t, i, S, window);
    const int tiles = tr_tiles(x, G, c0);
    if (tiles == 0 || c0 + col0 >= x.n * G) return;
    const FlDeal deal = fl_deal(t.n_trees, B, tr_values(t, Hq, c.dh), count);
    const int64_t before = fl_before(i, count);
    const int b0 = (int)(before / deal.q), parts = (int)((before + tiles - 1) / deal.q) - b0 + 1;
    if (parts < 2) return;
    for (int col = col0; col < min(CW, x.n * G - c0); col += nb * FL_NW) {
        const sw_f32x4 a = fl_join<DH>(part + (((int64_t)hg * 2 * B + fl_slot(b0, 0)) * CW + col) * (DH + 4), (int64_t)CW * (DH + 4), parts, 0);
        const int ck = c0 + col;
        if (lane < DH / 4) *(sw_f32x4 *)(out + ((int64_t)(x.row + ck / G) * Hq + hk * G + ck % G) * DH + lane * 4) = a;
    }
}

// Columns of a block and blocks of each of their groups, by max_nodes and n_trees: what is placed is known on the device alone, so that 8 nodes in a
// place for 32 take the form for more than 32 columns.  Up to 32 columns: a wave has them all and four take tiles in turn (one tile a wave
// in flight costs less than three idle waves).  Beyond, four waves have 32 each and read one tile.  Two blocks a CU where registers allow.
struct TrPlan { int wc, groups, B; };
template <int TYPE, int DH>
static TrPlan tr_plan(const SwKv &c, const SwTrees &t, int Hq) {
    TrPlan p;
    const int cols = t.max_nodes * (Hq / c.Hkv);
    p.wc = cols <= 32 ? tr_wc<TYPE, DH>() : 4;
    p.groups = c.Hkv * ((cols + 32 * p.wc - 1) / (32 * p.wc));
    const int64_t tiles = ((((int64_t)t.max_pages << c.psh) + 31) / 32 + 1) * t.n_trees;
    const int n = 256 * tr_occ<TYPE, DH>() / p.groups;
    p.B = (int)(n < 1 ? 1 : n < tiles ? n : tiles);
    return p;
}
template <int TYPE, int DH>
static int64_t tr_part(const SwKv &c, const SwTrees &t, int Hq) {
    const TrPlan p = tr_plan<TYPE, DH>(c, t, Hq);
    return p.B > 1 ? (int64_t)p.groups * 2 * p.B * 32 * p.wc * (DH + 4) : 0;
}
template <int TYPE, int DH>
static int tr_launch(hipStream_t st, const SwKv &c, const SwTrees &t, const float *q, int S, int Hq, float sc, int window, float *out, float *part) {
    const TrPlan p = tr_plan<TYPE, DH>(c, t, Hq);
    if (p.B > 1 && !part) return -1;
    const dim3 grid((unsigned)(p.B * p.groups));
    if (p.wc == 4) SW_LAUNCH((k_tree<TYPE, DH, 4>), grid, dim3(FL_NT), 0, st, c, t, q, S, Hq, sc, window, out, part, p.B);
    else SW_LAUNCH((k_tree<TYPE, DH, tr_wc<TYPE, DH>()>), grid, dim3(FL_NT), 0, st, c, t, q, S, Hq, sc, window, out, part, p.B);
    if (p.B > 1) {
        const int CW = 32 * p.wc, nb = fl_join_blocks(CW / FL_NW, (int64_t)p.groups * t.n_trees);
        SW_LAUNCH((k_tree_join<DH>), dim3((unsigned)(p.groups * nb), (unsigned)t.n_trees), dim3(FL_NT), 0, st, c, t, S, Hq, window, part, p.B, CW, nb, out);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

#define TR_DISPATCH(CALL)                                                                                      \
    switch (c.dh / 32) {                                                                                       \
    case 1: return CALL(32); case 2: return CALL(64); case 3: return CALL(96); case 4: return CALL(128);       \
    case 5: return CALL(160); case 6: return CALL(192); case 7: return CALL(224); default: return CALL(256);   \
    }
template <int TYPE>
static int64_t tr_part_of(const SwKv &c, const SwTrees &t, int Hq) {
#define TR_CALL(DH) (tr_part<TYPE, DH>(c, t, Hq))
    TR_DISPATCH(TR_CALL)
#undef TR_CALL
}
template <int TYPE>
static int tr_launch_of(hipStream_t st, const SwKv &c, const SwTrees &t, const float *q, int S, int Hq, float sc, int window, float *out, float *part) {
#define TR_CALL(DH) (tr_launch<TYPE, DH>(st, c, t, q, S, Hq, sc, window, out, part))
    TR_DISPATCH(TR_CALL)
#undef TR_CALL
}
int64_t sw_attn_tree_part_floats(const SwKv &c, const SwTrees &t, int Hq) {
    return c.type == SW_KV_F32 ? tr_part_of<SW_KV_F32>(c, t, Hq) : c.type == SW_KV_BF16 ? tr_part_of<SW_KV_BF16>(c, t, Hq) : tr_part_of<SW_KV_F16>(c, t, Hq);
}
int sw_launch_attn_tree(hipStream_t st, const SwKv &c, const SwTrees &t, const float *q, int Hq, float scale, int window, float *out, int S,
                        float *part) {
    if (c.dh < 32 || c.dh > 256 || c.dh % 32) return -1;
    const float sc = (float)((double)scale * 1.4426950408889634074);   // the softmax in powers of two
    if (c.type == SW_KV_F32) return tr_launch_of<SW_KV_F32>(st, c, t, q, S, Hq, sc, window, out, part);
    if (c.type == SW_KV_BF16) return tr_launch_of<SW_KV_BF16>(st, c, t, q, S, Hq, sc, window, out, part);
    return tr_launch_of<SW_KV_F16>(st, c, t, q, S, Hq, sc, window, out, part);
}
