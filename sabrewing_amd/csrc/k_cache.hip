// k_cache.hip -- writing the paged cache: the projection's heads normalised, turned and
// appended, and pages copied.
#include "sw_attn.h"

// Two forms of the append; both hold a head's pairs of values in a lane's registers, so a turn and
// all but one reduction of a head's sum of squares stay there.  The angle pos * freq[i] and its distance
// to the next full turn are taken in 64 bits: at position 10^6 a 32-bit product is 0.06 radians off.
__device__ __forceinline__ void rp_angle(double freq, int pos, float factor, float &cs, float &sn) {
    double t = (double)pos * freq * 0.15915494309189533577;                      // full turns
    t = t - rint(t);
    sincospif((float)(t + t), &sn, &cs);
    cs = cs * factor;
    sn = sn * factor;
}

#define RP_NT 256
// The form for any pairs (two halves of a part whose halves are no multiple of 4 values) and norm weights that do not begin
// on 16 bytes: a wave a head, a lane the pairs lane and lane + 64.  Each head takes its angles again: 2048 rows of 32 + 2 x
// 8 heads of 128 take 34 to 35 us (18.5 in the other form), one row and 48 what a launch takes.
template <int TYPE>
__global__ __launch_bounds__(RP_NT) void k_qk_rope_any(SwKv c, SwRows r, const int *__restrict__ turn_at, SwRope rope,
                                                          const float *__restrict__ qkv, int64_t ld, const float *__restrict__ wq, const float *__restrict__ wk, float eps,
                                                          int Hq, float *__restrict__ q_out) {
    const int lane = threadIdx.x & 63, s = blockIdx.x;
    const int H = Hq + 2 * c.Hkv, h = blockIdx.y * (RP_NT / 64) + (threadIdx.x >> 6);
    const int pos = r.pos[s];
    if (pos < 0 || h >= H) return;
    const int turn = turn_at ? turn_at[s] : pos;
    const int page = sw_page(c, r, r.seq ? r.seq[s] : s, pos);
    const int64_t cell = (int64_t)page * c.ps + (int64_t)(pos & ((1 << c.psh) - 1)) * c.ts;
    float cs[2], sn[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int i = lane + 64 * j;
        cs[j] = 1.f; sn[j] = 0.f;
        if (i < rope.np) rp_angle(rope.freq[i], turn, rope.factor, cs[j], sn[j]);
    }
    const float *x = qkv + (int64_t)s * ld;
    const bool is_v = h >= Hq + c.Hkv;
    const float *w = h < Hq ? wq : is_v ? nullptr : wk;
    float a[2], b[2], ss = 0.f;
    int ia[2], ib[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int i = lane + 64 * j;
        const bool half = !is_v && i < rope.np && !rope.interleaved;
        ia[j] = half ? i : 2 * i;
        ib[j] = half ? i + rope.np : 2 * i + 1;
        a[j] = b[j] = 0.f;
        if (i < c.dh / 2) { a[j] = x[h * c.dh + ia[j]]; b[j] = x[h * c.dh + ib[j]]; }
        ss = __builtin_fmaf(a[j], a[j], __builtin_fmaf(b[j], b[j], ss));
    }
    if (w) {
        for (int o = 32; o; o >>= 1) ss += __shfl_xor(ss, o);
        const float inv = 1.f / sqrtf(ss / (float)c.dh + eps);
#pragma unroll
        for (int j = 0; j < 2; j++)
            if (lane + 64 * j < c.dh / 2) { a[j] = a[j] * inv * w[ia[j]]; b[j] = b[j] * inv * w[ib[j]]; }
    }
#pragma unroll
    for (int j = 0; j < 2; j++) {
        if (lane + 64 * j >= c.dh / 2) continue;
        float ra = a[j], rb = b[j];
        if (!is_v && lane + 64 * j < rope.np) {
            ra = __builtin_fmaf(a[j], cs[j], -(b[j] * sn[j]));
            rb = __builtin_fmaf(b[j], cs[j], a[j] * sn[j]);
        }
        if (h < Hq) {
            float *q = q_out + ((int64_t)s * Hq + h) * c.dh;
            q[ia[j]] = ra;
            q[ib[j]] = rb;
        } else if (page >= 0) {
            const int64_t at = cell + (int64_t)(is_v ? h - Hq - c.Hkv : h - Hq) * c.hs;
            sw_kv_store<TYPE>(is_v ? c.v : c.k, at + ia[j], ra);
            sw_kv_store<TYPE>(is_v ? c.v : c.k, at + ib[j], rb);
        }
    }
}

// four values in the cache's type, side by side
template <int TYPE>
__device__ __forceinline__ void rp_store4(void *p, int64_t i, const float (&f)[4]) {
    if constexpr (TYPE == SW_KV_F32) {
        *(sw_f32x4 *)((float *)p + i) = sw_f32x4{f[0], f[1], f[2], f[3]};
    } else {
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
            h[e] = TYPE == SW_KV_BF16 ? (uint32_t)sw_bf16_rne(f[e]) : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[e]);
        *(uint2 *)((uint16_t *)p + i) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
    }
}
// x over the 2^n lanes of a head (n 2 to 5): quads, halves of a row of 16, rows, two rows
__device__ __forceinline__ float rp_sum(float x, int lanes) {
    auto dpp = [](float f, auto ctrl) {
        return f + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, f), decltype(ctrl)::v, 0xF, 0xF, false));
    };
    x = dpp(x, SwIc<0xB1>{});
    x = dpp(x, SwIc<0x4E>{});
    if (lanes > 4) x = dpp(x, SwIc<0x141>{});
    if (lanes > 8) x = dpp(x, SwIc<0x140>{});
    if (lanes > 16) {
        const uint2 a = sw_pair<16>(__builtin_bit_cast(uint32_t, x));
        x = __builtin_bit_cast(float, a.x) + __builtin_bit_cast(float, a.y);
    }
    return x;
}

// The form by 16 bytes: a lane holds 8 values of a head, 4 pairs -- 4u .. 4u + 3 of each half, or (interleaved,
// and what is not turned) 8u .. 8u + 7 -- and dh / 8 lanes (of a power of two) a head.  A block takes a row,
// or where rows are few a part of its heads; the row's angles are taken once, a thread each, into
// LDS while the first PB rounds of heads are on their way.  Bytes bound it: 2048 rows of 32 + 2 x 8 heads
// of 128 (92 MB) take 18.5 us (5.0 TB/s; 37.9 us by single values), 48 rows and one row what a launch takes,
// 4.5 us.
template <int TYPE, int PB>
__global__ __launch_bounds__(RP_NT) void k_qk_rope(SwKv c, SwRows r, const int *__restrict__ turn_at, SwRope rope,
                                                   const float *__restrict__ qkv, int64_t ld, const float *__restrict__ wq, const float *__restrict__ wk, float eps, int Hq,
                                                   float *__restrict__ q_out, int lanes) {
    __shared__ __align__(16) float s_cs[128], s_sn[128];
    const int tid = threadIdx.x, s = blockIdx.x, H = Hq + 2 * c.Hkv, per = RP_NT / lanes;      // heads a round
    const int u = tid & (lanes - 1), h0 = blockIdx.y * PB * per + tid / lanes;
    const int pos = r.pos[s];
    if (pos < 0) return;
    const int turn = turn_at ? turn_at[s] : pos;
    // this lane's places in a turned head: ia .. ia + 3 and ib .. ib + 3
    const bool turned = 4 * u < rope.np, halves = turned && !rope.interleaved;
    const int ia = halves ? 4 * u : 8 * u, ib = halves ? rope.np + 4 * u : 8 * u + 4;
    const bool in = 8 * u < c.dh;
    const float *x = qkv + (int64_t)s * ld;
    sw_f32x4 xa[PB], xb[PB];
#pragma unroll
    for (int j = 0; j < PB; j++) {
        const int h = h0 + j * per;
        xa[j] = xb[j] = sw_f32x4{0.f, 0.f, 0.f, 0.f};
        if (in && h < H) {
            const bool is_v = h >= Hq + c.Hkv;
            xa[j] = *(const sw_f32x4 *)(x + h * c.dh + (is_v ? 8 * u : ia));
            xb[j] = *(const sw_f32x4 *)(x + h * c.dh + (is_v ? 8 * u + 4 : ib));
        }
    }
    const int page = sw_page(c, r, r.seq ? r.seq[s] : s, pos);
    if (tid < rope.np) rp_angle(rope.freq[tid], turn, rope.factor, s_cs[tid], s_sn[tid]);
    __syncthreads();
    const sw_f32x4 cs = *(const sw_f32x4 *)(s_cs + 4 * u), sn = *(const sw_f32x4 *)(s_sn + 4 * u);     // (used below np alone)
    const int64_t cell = (int64_t)page * c.ps + (int64_t)(pos & ((1 << c.psh) - 1)) * c.ts;
#pragma unroll
    for (int j = 0; j < PB; j++) {
        const int h = h0 + j * per;
        const bool is_q = h < Hq, is_v = h >= Hq + c.Hkv;
        float a[4], b[4], ss = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            a[e] = xa[j][e];
            b[e] = xb[j][e];
            ss = __builtin_fmaf(a[e], a[e], __builtin_fmaf(b[e], b[e], ss));
        }
        ss = rp_sum(ss, lanes);                                        // (all lanes: heads are whole groups of them)
        if (!in || h >= H) continue;
        const float *w = is_q ? wq : is_v ? nullptr : wk;
        if (w) {
            const float inv = 1.f / sqrtf(ss / (float)c.dh + eps);
            const sw_f32x4 ga = *(const sw_f32x4 *)(w + ia), gb = *(const sw_f32x4 *)(w + ib);
#pragma unroll
            for (int e = 0; e < 4; e++) { a[e] = a[e] * inv * ga[e]; b[e] = b[e] * inv * gb[e]; }
        }
        if (!is_v && turned) {
            if (halves) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float p = a[e], q = b[e];
                    a[e] = __builtin_fmaf(p, cs[e], -(q * sn[e]));
                    b[e] = __builtin_fmaf(q, cs[e], p * sn[e]);
                }
            } else {                                                   // pairs (a0 a1) (a2 a3) (b0 b1) (b2 b3)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float p = a[e], q = a[e + 1], y = b[e], z = b[e + 1];
                    if (4 * u + e / 2 < rope.np) {
                        a[e] = __builtin_fmaf(p, cs[e / 2], -(q * sn[e / 2]));
                        a[e + 1] = __builtin_fmaf(q, cs[e / 2], p * sn[e / 2]);
                    }
                    if (4 * u + 2 + e / 2 < rope.np) {
                        b[e] = __builtin_fmaf(y, cs[2 + e / 2], -(z * sn[2 + e / 2]));
                        b[e + 1] = __builtin_fmaf(z, cs[2 + e / 2], y * sn[2 + e / 2]);
                    }
                }
            }
        }
        if (is_q) {
            float *q = q_out + ((int64_t)s * Hq + h) * c.dh;
            *(sw_f32x4 *)(q + ia) = sw_f32x4{a[0], a[1], a[2], a[3]};
            *(sw_f32x4 *)(q + ib) = sw_f32x4{b[0], b[1], b[2], b[3]};
        } else if (page >= 0) {
            const int64_t at = cell + (int64_t)(is_v ? h - Hq - c.Hkv : h - Hq) * c.hs;
            rp_store4<TYPE>(is_v ? c.v : c.k, at + (is_v ? 8 * u : ia), a);
            rp_store4<TYPE>(is_v ? c.v : c.k, at + (is_v ? 8 * u + 4 : ib), b);
        }
    }
}

template <int TYPE>
static int rp_launch(hipStream_t st, const SwKv &c, const SwRows &r, const int *at, const SwRope &rope, const float *qkv, int64_t ld, const float *wq,
                     const float *wk, float eps, int Hq, float *q_out, int S) {
    const int H = Hq + 2 * c.Hkv;
    if ((!rope.interleaved && rope.np % 4) || (((uintptr_t)wq | (uintptr_t)wk) & 15)) {
        SW_LAUNCH(k_qk_rope_any<TYPE>, dim3((unsigned)S, (unsigned)((H + 3) / 4)), dim3(RP_NT), 0, st, c, r, at, rope, qkv, ld, wq, wk, eps, Hq,
                  q_out);
    } else {
        const int lanes = c.dh <= 32 ? 4 : c.dh <= 64 ? 8 : c.dh <= 128 ? 16 : 32, rounds = (H * lanes + RP_NT - 1) / RP_NT;
        // four rounds of heads a block where the rows alone fill the chip, else one (an angle is taken by more blocks)
        if ((int64_t)S * ((rounds + 3) / 4) >= 512)
            SW_LAUNCH((k_qk_rope<TYPE, 4>), dim3((unsigned)S, (unsigned)((rounds + 3) / 4)), dim3(RP_NT), 0, st, c, r, at, rope, qkv, ld, wq, wk,
                      eps, Hq, q_out, lanes);
        else
            SW_LAUNCH((k_qk_rope<TYPE, 1>), dim3((unsigned)S, (unsigned)rounds), dim3(RP_NT), 0, st, c, r, at, rope, qkv, ld, wq, wk, eps, Hq,
                      q_out, lanes);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int sw_launch_qk_rope_append(hipStream_t st, const SwKv &c, const SwRows &r, const int *at, const SwRope &rope, const float *qkv, int64_t ld,
                             const float *wq, const float *wk, float eps, int Hq, float *q_out, int S) {
    if (c.type == SW_KV_F32) return rp_launch<SW_KV_F32>(st, c, r, at, rope, qkv, ld, wq, wk, eps, Hq, q_out, S);
    if (c.type == SW_KV_BF16) return rp_launch<SW_KV_BF16>(st, c, r, at, rope, qkv, ld, wq, wk, eps, Hq, q_out, S);
    return rp_launch<SW_KV_F16>(st, c, r, at, rope, qkv, ld, wq, wk, eps, Hq, q_out, S);
}

// A page is n2 x n1 runs of `run` 16-byte pieces (one run where its cells lie side by side).
// The pairs and the pools' addresses travel with the launch: nothing to upload, and a
// recorded copy keeps its own.  A piece a thread: bytes bound it, 1.6 GB in 267 us (6.0 TB/s; 307 us with four
// pieces a thread), a fork's 28 MB in 7.1 us.
struct SwCopy {
    void *pool[2 * SW_COPY_LAYERS];
    int src[SW_COPY_PAIRS], dst[SW_COPY_PAIRS];
};
#define KC_NT 256
__global__ __launch_bounds__(KC_NT) void k_kv_copy(SwCopy a, int64_t ps, int n1, int64_t s1, int64_t s2, int run, int total) {
    const int i = blockIdx.x * KC_NT + threadIdx.x;
    if (i >= total) return;
    const int row = i / run, at = i - row * run, r2 = row / n1, r1 = row - r2 * n1;
    sw_u32x4 *pool = (sw_u32x4 *)a.pool[blockIdx.z];
    const int64_t off = r2 * s2 + r1 * s1 + at;
    pool[a.dst[blockIdx.y] * ps + off] = pool[a.src[blockIdx.y] * ps + off];
}

int sw_launch_kv_copy(hipStream_t st, const SwKv *layers, int n_layers, const int *src, const int *dst, int n) {
    if (n < 1 || n > SW_COPY_PAIRS || n_layers < 1 || n_layers > SW_COPY_LAYERS) return -1;
    const SwKv &c = layers[0];
    const int per = c.type == SW_KV_F32 ? 4 : 8, P = 1 << c.psh;         // elements of a piece
    int64_t d = c.dh, run = d, s1 = c.ts, s2 = c.hs;
    int n1 = P, n2 = c.Hkv;
    if (c.ts == d) {                                  // tokens of a head side by side
        run = d * P; s1 = c.hs; n1 = c.Hkv; n2 = 1; s2 = 0;
        if (c.hs == run || c.Hkv == 1) { run *= c.Hkv; n1 = 1; }
    } else if (c.hs == d || c.Hkv == 1) {             // heads of a token side by side
        run = d * c.Hkv; s1 = c.ts; n1 = P; n2 = 1; s2 = 0;
        if (c.ts == run) { run *= P; n1 = 1; }
    }
    const int64_t total = run / per * n1 * n2;
    if (total >= (int64_t)1 << 31) return -1;
    SwCopy a = {};
    for (int l = 0; l < n_layers; l++) { a.pool[2 * l] = layers[l].k; a.pool[2 * l + 1] = layers[l].v; }
    for (int i = 0; i < n; i++) { a.src[i] = src[i]; a.dst[i] = dst[i]; }
    SW_LAUNCH(k_kv_copy, dim3((unsigned)((total + KC_NT - 1) / KC_NT), (unsigned)n, (unsigned)(2 * n_layers)), dim3(KC_NT), 0, st, a,
              c.ps / per, n1, s1 / per, s2 / per, (int)(run / per), (int)total);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// A tree's accepted path and its cells.  The walk takes a ballot a step (a node a lane) and is taken by every wave of every
// layer's block: nothing to wait for.  A path's nodes rise, so node path[i]'s cell lies at or behind its place i and is
// nobody's place before i: a thread moves one piece of 16 bytes of all cells in turn, eight reads and then their writes.
// Bound by the launch and a chain of waits: 48 layers of 8 heads of 128, one tree of 16 nodes 5.4 us, 32 of 64 nodes 5.8.
#define TC_NT 256
struct SwCommit { void *pool[2 * SW_COPY_LAYERS]; };
__global__ __launch_bounds__(TC_NT) void k_tree_commit(SwCommit a, SwKv c, SwTrees t, const int *__restrict__ parent, const int *__restrict__ draft,
                                                       const int *__restrict__ tok, int *__restrict__ path, int *__restrict__ count,
                                                       int *__restrict__ next, int S, int es, int run) {
    __shared__ int64_t s_src[64], s_dst[64];
    const int tid = threadIdx.x, lane = tid & 63, i = blockIdx.x;
    const int row = t.first[i], end = t.first[i + 1], base = t.base[i], seq = t.seq ? t.seq[i] : i;
    const int n = base < 0 || row < 0 || row >= S || end <= row ? 0 : min(min(end, S) - row, t.max_nodes);
    const bool node = lane < n;
    const int p = node ? parent[row + lane] : -2, d = node ? draft[row + lane] : 0, k = node ? tok[row + lane] : 0;
    int at = 0, len = n ? 1 : 0, mine = -1;
    if (lane == 0 && n) mine = 0;
    while (n) {
        const int pick = __builtin_amdgcn_readlane(k, at);
        const uint64_t kids = __ballot(lane > at && p == at && d == pick);
        if (!kids) break;
        at = __builtin_ctzll(kids);
        if (lane == len) mine = at;
        len++;
    }
    if (blockIdx.y == 0 && tid < 64) {
        if (lane < t.max_nodes) path[(int64_t)i * t.max_nodes + lane] = mine;
        if (lane == 0) {
            count[i] = len;
            next[i] = n ? __builtin_amdgcn_readlane(k, at) : -1;
        }
    }
    // the cells that move: their offsets, side by side
    const SwRows r = {nullptr, nullptr, t.table, t.n_seqs, t.max_pages};
    const int64_t from = (int64_t)base + mine, to = (int64_t)base + lane;
    int pf = -1, pt = -1;
    if (mine > lane && from < (int64_t)t.max_pages << c.psh) { pf = sw_page(c, r, seq, (int)from); pt = sw_page(c, r, seq, (int)to); }
    const bool moves = pf >= 0 && pt >= 0;
    const uint64_t all = __ballot(moves);
    const int cells = __builtin_popcountll(all), pmask = (1 << c.psh) - 1;
    if (moves && tid < 64) {
        const int x = __builtin_popcountll(all & ((1ull << lane) - 1));
        s_src[x] = (pf * c.ps + (from & pmask) * c.ts) * es;
        s_dst[x] = (pt * c.ps + (to & pmask) * c.ts) * es;
    }
    if (!cells) return;
    __syncthreads();
    const int pieces = 2 * c.Hkv * run;                                // of 16 bytes: both pools, heads of `run`
    for (int x = tid; x < pieces; x += TC_NT) {
        const int v = x >= c.Hkv * run, y = x - v * c.Hkv * run, h = y / run;
        char *pool = (char *)a.pool[2 * blockIdx.y + v] + h * c.hs * es + (y - h * run) * 16;
        for (int j0 = 0; j0 < cells; j0 += 8) {
            sw_u32x4 b[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j0 + j < cells) b[j] = *(const sw_u32x4 *)(pool + s_src[j0 + j]);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j0 + j < cells) *(sw_u32x4 *)(pool + s_dst[j0 + j]) = b[j];
        }
    }
}

int sw_launch_tree_commit(hipStream_t st, const SwKv *layers, int n_layers, const SwTrees &t, const int *parent, const int *draft, const int *tok,
                          int *path, int *count, int *next, int S) {
    if (n_layers < 1 || n_layers > SW_COPY_LAYERS) return -1;
    SwCommit a = {};
    for (int l = 0; l < n_layers; l++) { a.pool[2 * l] = layers[l].k; a.pool[2 * l + 1] = layers[l].v; }
    const int es = layers[0].type == SW_KV_F32 ? 4 : 2;
    SW_LAUNCH(k_tree_commit, dim3((unsigned)t.n_trees, (unsigned)n_layers), dim3(TC_NT), 0, st, a, layers[0], t, parent, draft, tok, path, count,
              next, S, es, layers[0].dh * es / 16);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
