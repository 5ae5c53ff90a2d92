// k_sample.hip -- a token of each row of logits from a given random number.
//
// Weights are whole numbers, w_i = rint(2^42 exp((l_i - max) / T)), the exponential in 64
// bits: their sums are exact in 64-bit integers, so no order of threads or atomics changes a
// pick, and up to 2^20 of them fit.  (In floats a sum of 10^5 weights is 1e-6 off, and some
// row of a large batch picks the neighbour.)  The tokens in order of falling logit, equal ones by
// rising index -- a token's code, (order bits of its logit, ~index), in falling order; top-k
// keeps the first k, top-p the shortest beginning of those with at least top_p of their sum, min-p the
// weights of at least min_p of the largest: each keeps a beginning of that order, so the
// kept set is one least code and one least weight.  The pick is the lowest index at which the
// running sum of kept weights, in order of index, passes u times their sum.
//
// A block per row, in passes over it (the first SP_CACHE tiles stay in LDS, the rest of a
// larger row comes from the caches again), each for what the settings need:
//   the largest logit, from the maxima of 256 groups of the row's tokens;
//   a top-k of up to SP_MAXK: the k-th largest group maximum bounds the k-th largest logit from
//     below and little more than k logits reach it; they are listed, and all the rest is
//     done on the list, a thread a token (as is min-p alone, where few weights reach it);
//   one of up to SP_LIST: the threads' own maxima bound it, and where that leaves too many for the list,
//     a histogram of counts says which bins hold the first k;
//   else a histogram over the distance to the largest logit, of counts for top-k, then of
//     weights for top-p; the tokens of the bin in which the beginning ends are listed and ranked;
//   the kept weights of each group of tiles, then tile by tile of the group in which the sum passes.
// Weights are what costs in the passes over all of a large row (some 20 64-bit operations each).
//
// Measured: one row of 32,000 logits, top-k 50, 11.5 us; 8 of 128,000: greedy 7, top-k 50 20, top-k 500 37, top-k
// 1000 59, top-p alone 91, no limit 41.  200 rows of 131,072 of all settings 108 us (0.97 TB/s), which is what one
// row of top-p takes: 45 us the histogram of weights (47 cycles of an LDS atomic for a wave), 29 us the
// groups' sums (64-bit operations), the rest the row's reading three times.  A row of a batch has a CU to
// itself, so up to 256 rows take no longer than the slowest of them, and few rows leave most CUs idle.  (One register of
// 128 spills.)
#include "sw_attn.h"
#include "sw_gate.h"

#define SP_NT 1024
#define SP_NW (SP_NT / 64)
#define SP_TILE (4 * SP_NT)
#define SP_CACHE 8                        // tiles in LDS: 128 KB
#define SP_BINS 2048
#define SP_LIST 1024                      // a thread each
#define SP_GROUPS 256
#define SP_MAXK 192                       // (at random, 355 tokens reach the 192nd of 256 maxima,
#define SP_MAXK2 600                      // 900 the 600th of the threads' 1024)
#define SP_STEPS 512
#define SP_GROUPS_OF_TILES 16
#define SP_ONE 4398046511104.0            // 2^42
#define SP_FAR 43.1                       // log2 of the largest weight over one that rounds to 0
#define SP_SCALE 47.0f                    // bins per halving (47 x 43.1 < SP_BINS)

typedef unsigned long long u64;
typedef u64 u64x4 __attribute__((ext_vector_type(4)));
typedef float sp_f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// 2^(j / 32) and 2^(j / 512), rounded to nearest
__constant__ double SP_POW2[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0,
};
__constant__ double SP_POW2F[16] = {
    0x1.0000000000000p+0, 0x1.0058c86da1c0ap+0, 0x1.00b1afa5abcbfp+0, 0x1.010ab5b2cbd11p+0,
    0x1.0163da9fb3335p+0, 0x1.01bd1e77170b4p+0, 0x1.02168143b0281p+0, 0x1.027003103b10ep+0,
    0x1.02c9a3e778061p+0, 0x1.032363d42b027p+0, 0x1.037d42e11bbccp+0, 0x1.03d7411915a8ap+0,
    0x1.04315e86e7f85p+0, 0x1.048b9b35659d8p+0, 0x1.04e5f72f654b1p+0, 0x1.0540727fc1762p+0,
};
struct SpShared {
    sw_f32x4 tile[SP_CACHE * SP_NT];
    u64 hist[SP_BINS];                    // (also the weights beside a short list, the tiles' sums by wave)
    u64 item[SP_LIST];
    float group[SP_GROUPS];
    u64 part[SP_NW], found, before;
    double pow2[SP_STEPS];                // 2^(42 + j / SP_STEPS)
    int n, bin, pick;
    float fmax, bound;
};
struct SpRow {
    const float *v;
    int V, ntile;
    float fmax, c32;                      // the largest logit; bins of distance to it by logit
    double m64, c64;
    float lf;                             // kept so far: logits above lf, and equal ones up to index li
    int li;
};

// tile k of the row, this thread's four (NaN behind its end)
__device__ __forceinline__ sw_f32x4 sp_load(const SpRow &r, int k) {
    const int i = k * SP_TILE + 4 * (int)threadIdx.x;
    if (i + 4 <= r.V) return *(const sp_f32x4u *)(r.v + i);
    sw_f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = i + e < r.V ? r.v[i + e] : NAN;
    return x;
}
// f(four logits, the first's index, tile) over all of the row; tiles beyond LDS are loaded four ahead
template <class F>
__device__ __forceinline__ void sp_each(const SpShared &sh, const SpRow &r, F f) {
    const int i0 = 4 * (int)threadIdx.x;
    sw_f32x4 x[4];
    if (r.ntile > SP_CACHE)
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = sp_load(r, min(SP_CACHE + j, r.ntile - 1));
#pragma unroll 1
    for (int k = 0; k < min(r.ntile, SP_CACHE); k++) f(sh.tile[k * SP_NT + threadIdx.x], k * SP_TILE + i0, k);
#pragma unroll 1
    for (int k = SP_CACHE; k < r.ntile; k++) {
        const sw_f32x4 y = x[0];
#pragma unroll
        for (int j = 0; j < 3; j++) x[j] = x[j + 1];
        if (k + 4 < r.ntile) x[3] = sp_load(r, k + 4);
        f(y, k * SP_TILE + i0, k);
    }
}

__device__ __forceinline__ u64 sp_code(float f, int i) { return ((u64)ord_f32(f + 0.0f) << 32) | (0xFFFFFFFFu - (uint32_t)i); }
__device__ __forceinline__ float sp_unkey(uint32_t o) { return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7FFFFFFFu : ~o); }
// log2(largest weight / weight) in bins
__device__ __forceinline__ float sp_dist(float f, const SpRow &r) {
    return f == r.fmax ? 0.f : fminf(r.fmax - f, 3.402823466e38f) * r.c32;           // (of finite ones the difference may not be)
}
__device__ __forceinline__ bool sp_kept(float f, int i, const SpRow &r) { return (f > r.lf) | ((f == r.lf) & (i <= r.li)); }
// 2^42 2^((f - max) c) to the nearest whole number: 512 steps of a halving from a table, the rest
// (at most 2^-10 of one) by the exponential's series to the third power, 9e-15 off.  For what is kept;
// infinities count as the largest float, which m64 is then
__device__ __forceinline__ u64 sp_weight(float f, const SpRow &r, const SpShared &sh) {
    constexpr double L = 0.69314718055994530942 / SP_STEPS, MAGIC = 6755399441055744.0;   // 1.5 * 2^52: rounds to whole numbers
    const double x = (double)__builtin_amdgcn_fmed3f(f, -3.402823466e38f, 3.402823466e38f) - r.m64;
    const double t = __builtin_fma(x, r.c64, MAGIC);
    const int k = (int)(uint32_t)__builtin_bit_cast(u64, t);
    const double z = __builtin_fma(x, r.c64, MAGIC - t);
    const double p = __builtin_fma(z, __builtin_fma(z, __builtin_fma(z, L * L * L / 6, L * L / 2), L), 1.0);
    const u64 b = __builtin_bit_cast(u64, sh.pow2[k & (SP_STEPS - 1)]);       // its exponent lowered by whole halvings
    const uint32_t hi = (uint32_t)(b >> 32) + ((uint32_t)(k & -SP_STEPS) << 11);
    const double w = __builtin_fma(p, __builtin_bit_cast(double, ((u64)hi << 32) | (uint32_t)b), 4503599627370496.0);
    return __builtin_bit_cast(u64, w) & 0xFFFFFFFFFFFFFull;
}
// the weights of the four with `on`, 0 for the others (side by side: each is a chain of 64-bit operations)
__device__ __forceinline__ void sp_weights(const sw_f32x4 &x, const bool (&on)[4], const SpRow &r, const SpShared &sh, u64 (&w)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        w[e] = sp_weight(x[e], r, sh);
        if (!on[e]) w[e] = 0;
    }
}

// a 64-bit value moved in a row of 16 lanes or to the next rows, 0 where nothing comes from
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ u64 sp_dpp(u64 x) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xF, false);
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 sp_wave_sum(u64 v) {           // (row rotations by 8, 4, 2, 1, then the rows)
    v += sp_dpp<0x128>(v);
    v += sp_dpp<0x124>(v);
    v += sp_dpp<0x122>(v);
    v += sp_dpp<0x121>(v);
    uint2 lo = sw_pair<16>((uint32_t)v), hi = sw_pair<16>((uint32_t)(v >> 32));
    v = (((u64)hi.x << 32) | lo.x) + (((u64)hi.y << 32) | lo.y);
    lo = sw_pair<32>((uint32_t)v);
    hi = sw_pair<32>((uint32_t)(v >> 32));
    return (((u64)hi.x << 32) | lo.x) + (((u64)hi.y << 32) | lo.y);
}
__device__ __forceinline__ u64 sp_wave_scan(u64 v) {          // sums up to each lane (shifts by 1, 2, 4, 8, then the rows' last)
    v += sp_dpp<0x111>(v);
    v += sp_dpp<0x112>(v);
    v += sp_dpp<0x114>(v);
    v += sp_dpp<0x118>(v);
    v += sp_dpp<0x142, 0xA>(v);
    v += sp_dpp<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ float sp_wave_max(float x) {
    auto ror = [](float f, auto n) {
        return fmaxf(f, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, f), 0x120 + decltype(n)::v, 0xF, 0xF, false)));
    };
    x = ror(x, SwIc<8>{});
    x = ror(x, SwIc<4>{});
    x = ror(x, SwIc<2>{});
    x = ror(x, SwIc<1>{});
    return sw_max4(x);
}
// the block's sum, and with `before` the sum of the threads before this one
__device__ __forceinline__ u64 sp_block_sum(SpShared &sh, u64 v, u64 *before = nullptr) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 x = before ? sp_wave_scan(v) : sp_wave_sum(v);
    __syncthreads();
    if (lane == 63) sh.part[wave] = x;
    __syncthreads();
    u64 t = 0;
    if (before) *before = x - v;
#pragma unroll
    for (int q = 0; q < SP_NW; q++) {
        if (before && q < wave) *before += sh.part[q];
        t += sh.part[q];
    }
    return t;
}

// hist[b] += w for the four with `on` (a wave whose first ones share a bin, as in a row of equal logits,
// adds up its lanes of a bin first)
__device__ __forceinline__ void sp_add(SpShared &sh, const bool (&on)[4], const int (&b)[4], const u64 (&w)[4]) {
    const u64 any = __ballot(on[0]);
    const int b0 = __builtin_amdgcn_readlane(b[0], any ? __builtin_ctzll(any) : 0);
    if (__popcll(any) > 8 && __ballot(on[0] && b[0] != b0) == 0) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const u64 v = sp_wave_sum(on[e] && b[e] == b0 ? w[e] : 0);
            if ((threadIdx.x & 63) == 0) atomicAdd(&sh.hist[b0], v);
            if (on[e] && b[e] != b0) atomicAdd(&sh.hist[b[e]], w[e]);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (on[e]) atomicAdd(&sh.hist[b[e]], w[e]);
}
__device__ __forceinline__ void sp_clear(SpShared &sh) {
    __syncthreads();
    sh.hist[threadIdx.x] = sh.hist[threadIdx.x + SP_NT] = 0;
    __syncthreads();
}
// The bin in which the histogram's sum, from bin 0 (up: from the last), reaches limit(its total), and
// the sum before it; -1: never.
template <class F>
__device__ __forceinline__ int sp_find(SpShared &sh, F limit_of, u64 &limit, u64 &before, bool up = false) {
    const int t = threadIdx.x, b0 = up ? SP_BINS - 1 - 2 * t : 2 * t, b1 = up ? b0 - 1 : b0 + 1;
    __syncthreads();
    const u64 a = sh.hist[b0], b = sh.hist[b1];
    if (t == 0) sh.bin = -1;
    u64 at;
    limit = limit_of(sp_block_sum(sh, a + b, &at));
    if (at < limit && at + a + b >= limit) {
        const bool first = at + a >= limit;
        sh.bin = first ? b0 : b1;
        sh.before = first ? at : at + a;
    }
    __syncthreads();
    before = sh.before;
    return sh.bin;
}
// the tokens with `on` of the wave's four into the list (beyond its end they are counted)
__device__ __forceinline__ void sp_list(SpShared &sh, const bool (&on)[4], const sw_f32x4 &x, int i) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const u64 b = __ballot(on[e]);
        if (!b) continue;
        int at = 0;
        if ((int)(threadIdx.x & 63) == __builtin_ctzll(b)) at = atomicAdd(&sh.n, (int)__popcll(b));
        at = __builtin_amdgcn_readlane(at, __builtin_ctzll(b)) +
             (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
        if (on[e] && at < SP_LIST) sh.item[at] = sp_code(x[e], i + e);
    }
}
__device__ __forceinline__ u64 sp_share(double part, u64 total, u64 least) {      // ceil(part * total), at least `least`
    const double x = ceil(part * (double)total);
    return x > (double)least ? (u64)x : least;
}
__device__ __forceinline__ u64 sp_target(float u, u64 total) {                    // floor(u * total), below total
    const double x = (double)u * (double)total;
    const u64 t = x > 0.0 ? (u64)x : 0;
    return t < total ? t : total - 1;
}

// Of the threads with `on`, in order of rising bin and in a bin of falling code: the code at which the sum of
// w reaches limit (0: nowhere).  A histogram finds the bin, its few are ranked.
__device__ __forceinline__ u64 sp_border(SpShared &sh, bool on, int bin, u64 code, u64 w, u64 limit) {
    sp_clear(sh);                                                     // (the list is read)
    if (on) atomicAdd(&sh.hist[bin], w);
    u64 left, at;
    const int b = sp_find(sh, [&](u64) { return limit; }, left, at);
    if (b < 0) return 0;
    on = on && bin == b;
    if (threadIdx.x == 0) { sh.n = 0; sh.found = 0; }
    __syncthreads();
    if (on) {
        const int i = atomicAdd(&sh.n, 1);
        sh.item[i] = code;
        sh.hist[i] = w;
    }
    __syncthreads();
    if (on) {
        const int n = sh.n;
#pragma unroll 4
        for (int j = 0; j < n; j++) at += sh.item[j] > code ? sh.hist[j] : 0;
        if (at < limit && at + w >= limit) sh.found = code;
    }
    __syncthreads();
    return sh.found;
}

// The code at which the beginning ends, among the kept: after `limit` tokens, or (mass) with the token
// at which the weights' sum reaches `limit`; `before`: what counts of the bins before `bin`.  The bin's
// tokens are narrowed by bits of the code until the list takes them.
__device__ __forceinline__ u64 sp_cut(SpShared &sh, const SpRow &r, int bin, u64 limit, u64 before, bool mass) {
    u64 prefix = 0, mask = 0;
    int shift = 64;
    const float lo = (float)bin, hi = bin == SP_BINS - 1 ? NAN : (float)(bin + 1);     // (the last bin has no end)
    for (bool list = true;;) {
        if (!list) sp_clear(sh);
        __syncthreads();
        if (threadIdx.x == 0) { sh.n = 0; sh.found = 0; }
        __syncthreads();
        sp_each(sh, r, [&](const sw_f32x4 &x, int i, int) {
            bool on[4], any = false;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float d = sp_dist(x[e], r);
                on[e] = (d >= lo) & !(d >= hi);
                any |= on[e];
            }
            if (!__any(any)) return;
#pragma unroll
            for (int e = 0; e < 4; e++) on[e] = on[e] && sp_kept(x[e], i + e, r);
            if (mask)
#pragma unroll
                for (int e = 0; e < 4; e++) on[e] = on[e] && (sp_code(x[e], i + e) & mask) == prefix;
            if (list) {
                sp_list(sh, on, x, i);
                return;
            }
            u64 w[4] = {1, 1, 1, 1};
            int b[4];
            if (mass) sp_weights(x, on, r, sh, w);
#pragma unroll
            for (int e = 0; e < 4; e++) b[e] = (int)(sp_code(x[e], i + e) >> shift) & (SP_BINS - 1);
            sp_add(sh, on, b, w);
        });
        __syncthreads();
        if (list) {
            if (sh.n <= SP_LIST) break;
            shift = shift > 11 ? shift - 11 : 0;                      // 2048 ways by the next bits
        } else {
            u64 more, left;
            const int b = sp_find(sh, [&](u64) { return limit - before; }, left, more, true);
            before += more;
            prefix |= (u64)b << shift;
            mask |= (u64)(SP_BINS - 1) << shift;
        }
        list = !list;
    }
    u64 c = 0, w = 0;                                                 // 2048 parts of the bin
    int part = 0;
    const bool on = (int)threadIdx.x < sh.n;
    if (on) {
        c = sh.item[threadIdx.x];
        const float f = sp_unkey((uint32_t)(c >> 32));
        w = mass ? sp_weight(f, r, sh) : 1;
        part = min((int)((sp_dist(f, r) - lo) * SP_BINS), SP_BINS - 1);
    }
    return sp_border(sh, on, part, c, w, limit - before);
}

__global__ __launch_bounds__(SP_NT) void k_sample(const float *__restrict__ logits, int V, SwSample p, const float *__restrict__ u,
                                                  int *__restrict__ tok) {
    __shared__ SpShared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, s = blockIdx.x;
    SpRow r;
    r.v = logits + (int64_t)s * V;
    r.V = V;
    r.ntile = (V + SP_TILE - 1) / SP_TILE;
    const float temp = p.temp ? p.temp[s] : 1.f, us = u[s], f0 = r.v[0];
    int k = p.top_k ? p.top_k[s] : 0;
    const float top_p = p.top_p ? p.top_p[s] : 1.f, min_p = p.min_p ? p.min_p[s] : 0.f;
    if (k <= 0 || k >= V) k = 0;
    if (tid < SP_STEPS) sh.pow2[tid] = SP_POW2[tid >> 4] * SP_POW2F[tid & 15] * SP_ONE;
    // ---- the largest logit: each thread's first, in order of index
    float best = -INFINITY;
    int bi = -1;
    auto take = [&](const sw_f32x4 &x, int t) {
        if (t < SP_CACHE) sh.tile[t * SP_NT + tid] = x;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (x[e] > best) { best = x[e]; bi = t * SP_TILE + 4 * tid + e; }
    };
    const int whole = V / SP_TILE;
    const sw_f32x4 last = sp_load(r, r.ntile - 1);
    for (int k0 = 0; k0 < whole; k0 += 8) {                           // (past the last: that one again)
        sw_f32x4 x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = *(const sp_f32x4u *)(r.v + min(k0 + j, whole - 1) * SP_TILE + 4 * tid);
#pragma unroll
        for (int j = 0; j < 8; j++) take(x[j], min(k0 + j, whole - 1));
    }
    if (whole < r.ntile) take(last, whole);
    {   // (a group: 16 lanes of a wave hold the maxima of their four)
        const float g = sw_max4(best);
        if (lane < 16) sh.group[wave * 16 + lane] = g;
    }
    const bool by_p = top_p < 1.f, by_k = k > 0 && k <= SP_MAXK;
    const bool few = temp > 0.f && (by_k || (!k && !by_p && min_p > 0.f));
    __syncthreads();
    if (wave == 0) {
        const sw_f32x4 g = ((const sw_f32x4 *)sh.group)[lane];
        const float top = sp_wave_max(fmaxf(fmaxf(g[0], g[1]), fmaxf(g[2], g[3])));
        float bound = -INFINITY;
        int some = 0;                                                 // groups that hold anything
#pragma unroll
        for (int e = 0; e < 4; e++) some += (int)__popcll(__ballot(g[e] > -INFINITY));
        if (few && by_k && top < INFINITY && some >= k) {
            // the k-th largest of the groups, or a little less: halving the range between a bound that k
            // groups reach and one that fewer do
            float least = fminf(fminf(g[0], g[1]), fminf(g[2], g[3]));
            least = -sp_wave_max(-least);
            float lo = least, hi = top, at = lo > -INFINITY ? 0.5f * lo + 0.5f * top : top - 1.f;
            for (int step = 0; step < 40; step++) {
                int n = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) n += (int)__popcll(__ballot(g[e] >= at));
                if (n >= k) lo = at; else hi = at;
                if (n >= k && n <= k + (step < 6 ? 3 : 8)) break;
                at = lo > -INFINITY ? 0.5f * lo + 0.5f * hi : top - 2.f * (top - hi);
                if (at == lo || at == hi || !(at > -INFINITY)) break;
            }
            bound = lo;
        }
        if (lane == 0) {
            sh.fmax = top;
            sh.bound = bound;
            sh.n = 0;
            sh.pick = 0x7FFFFFFF;
        }
    }
    __syncthreads();
    r.fmax = sh.fmax;
    if (!(temp > 0.f) || r.fmax == -INFINITY) {                       // greedy, or nothing to draw from
        if (best == r.fmax && bi >= 0) atomicMin(&sh.pick, bi);
        __syncthreads();
        if (tid == 0) tok[s] = f0 != f0 || r.fmax == -INFINITY ? 0 : sh.pick;
        return;
    }
    r.m64 = (double)fminf(r.fmax, 3.402823466e38f);
    r.c64 = SP_STEPS * 1.4426950408889634074 / (double)temp;
    r.c32 = fminf((float)(SP_SCALE * 1.4426950408889634074 / (double)temp), 3.402823466e38f);
    // what rounds to no weight is not kept: logits more than SP_FAR halvings below the largest.  In 64 bits, and no
    // lower than that: at temperatures near 0 a neighbour of the largest can be 1000 halvings away
    {
        const double far = r.m64 - SP_FAR * 0.69314718055994530942 * (double)temp;
        float lo = (float)far;                                        // (the float below it, and below the largest logit)
        if ((double)lo > far || lo >= r.fmax) {
            const int b = __builtin_bit_cast(int, lo);
            lo = __builtin_bit_cast(float, lo > 0.f ? b - 1 : lo < 0.f ? b + 1 : (int)0x80000001);
        }
        r.lf = r.fmax == INFINITY ? 3.402823466e38f : lo;
        r.li = -1;
    }
    const u64 least_w = min_p > 0.f ? (u64)ceil(fmin((double)min_p, 1.0) * SP_ONE) : 0;

    // ---- few tokens can be kept: list them and stay there
    int listed = -1;                                                  // tokens of the list, where it holds all that can be kept
    if (few) {
        float bound = sh.bound;                                       // the list's tokens reach it
        if (!by_p && min_p > 0.f) {                                   // (a little lower: the weights decide)
            const float lo = r.fmax - (0.05f - log2f(fminf(min_p, 1.f))) * 0.6931472f * temp;
            bound = fmaxf(bound, lo - 1e-6f * fabsf(lo));
        }
        sp_each(sh, r, [&](const sw_f32x4 &x, int i, int) {
            if (__all(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) < bound)) return;
            bool on[4];
#pragma unroll
            for (int e = 0; e < 4; e++) on[e] = (x[e] >= bound) & (x[e] > r.lf);
            sp_list(sh, on, x, i);
        });
        __syncthreads();
        const int n = sh.n;
        if (n <= 64) {                                                // one wave does the rest
            if (wave) return;
            u64 code = 0, w = 0, at = 0;
            int rank = 0;
            if (lane < n) {
                code = sh.item[lane];
                w = sp_weight(sp_unkey((uint32_t)(code >> 32)), r, sh);
            }
            for (int j0 = 0; j0 < n; j0 += 8)                         // (lanes behind the list hold 0)
#pragma unroll
            for (int j = j0; j < j0 + 8; j++) {
                const u64 cj = ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(code >> 32), j) << 32) |
                               (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)code, j);
                const u64 wj = ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(w >> 32), j) << 32) |
                               (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)w, j);
                rank += cj > code;
                at += cj > code ? wj : 0;
            }
            if (lane >= n || (k && rank >= k)) w = 0;
            if (by_p && at >= sp_share((double)top_p, sp_wave_sum(w), 1)) w = 0;
            if (w < least_w) w = 0;
            const u64 target = sp_target(us, sp_wave_sum(w));
            u64 sum = 0;                                              // the kept weights up to this index
            for (int j0 = 0; j0 < n; j0 += 8)
#pragma unroll
            for (int j = j0; j < j0 + 8; j++) {
                const uint32_t cj = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)code, j);
                const u64 wj = ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(w >> 32), j) << 32) |
                               (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)w, j);
                sum += cj >= (uint32_t)code ? wj : 0;
            }
            // the least index past the target: the one token whose own weight crosses it
            if (w && sum > target && sum - w <= target) tok[s] = (int)(0xFFFFFFFFu - (uint32_t)code);
            return;
        }
        if (n <= SP_LIST) listed = n;
    }
    if (listed < 0) {
        // bins as fine as the range of the row's first tiles allows (what lies below is in the last one)
        {
            float m = INFINITY;
            for (int t = 0; t < min(r.ntile, SP_CACHE); t++) {
                const sw_f32x4 x = sh.tile[t * SP_NT + tid];
                m = fminf(fminf(fminf(m, x[0]), fminf(x[1], x[2])), x[3]);
            }
            m = -sp_wave_max(-m);
            __syncthreads();
            if (lane == 0) sh.group[wave] = m;
            __syncthreads();
            float lo = sh.group[0];
#pragma unroll
            for (int q = 1; q < SP_NW; q++) lo = fminf(lo, sh.group[q]);
            r.c32 = fminf(fmaxf(r.c32, (SP_BINS - 1) / (r.fmax - fmaxf(lo, r.lf))), 3.402823466e38f);
        }
        if (k) {
            // the k-th largest of the threads' maxima bounds the k-th largest token from below: all above `bound` (the
            // end of a bin, or a little lower) are looked at
            float bound = -INFINITY;
            auto end_of = [&](int b) {
                const float x = r.fmax - (float)(b + 1) / r.c32;
                return b < SP_BINS - 1 && r.fmax < INFINITY ? x - 1e-6f * (fabsf(x) + fabsf(r.fmax)) : -INFINITY;
            };
            u64 limit, before;
            if (k <= SP_LIST) {
                sp_clear(sh);
                if (best > r.lf) atomicAdd(&sh.hist[min((int)sp_dist(best, r), SP_BINS - 1)], 1ull);
                const int b = sp_find(sh, [&](u64) { return (u64)k; }, limit, before);
                if (b >= 0) bound = end_of(b);
            }
            // a list of these, if they are few enough; else they are counted by bin, and the k-th token's bin is the
            // last of the list, or its tokens are ranked
            for (bool count = k > SP_MAXK2, again = false;; again = count, count = true) {
                if (count) {
                    sp_clear(sh);
                    sp_each(sh, r, [&](const sw_f32x4 &x, int i, int) {
                        if (__all(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) < bound)) return;
                        bool on[4];
                        int d[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            d[e] = min((int)sp_dist(x[e], r), SP_BINS - 1);
                            on[e] = (x[e] > r.lf) & (x[e] >= bound);
                        }
                        const u64 one[4] = {1, 1, 1, 1};
                        sp_add(sh, on, d, one);
                    });
                    const int b = sp_find(sh, [&](u64) { return (u64)k; }, limit, before);
                    if (b >= 0 && !again && before + sh.hist[b] <= SP_LIST - 8) {
                        bound = fmaxf(bound, end_of(b));
                    } else if (b >= 0) {
                        const u64 c = sp_cut(sh, r, b, limit, before, false);
                        r.lf = sp_unkey((uint32_t)(c >> 32));
                        r.li = (int)(0xFFFFFFFFu - (uint32_t)c);
                    }
                    if (k > SP_LIST) break;
                }
                __syncthreads();
                if (tid == 0) sh.n = 0;
                __syncthreads();
                sp_each(sh, r, [&](const sw_f32x4 &x, int i, int) {
                    if (__all(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) < bound)) return;
                    bool on[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) on[e] = sp_kept(x[e], i + e, r) & (x[e] >= bound);
                    sp_list(sh, on, x, i);
                });
                __syncthreads();
                if (sh.n <= SP_LIST) {
                    listed = sh.n;
                    break;
                }
            }
        }
    }
    if (listed >= 0) {
        u64 code = 0, w = 0;
        int d = 0;
        if (tid < listed) {
            code = sh.item[tid];
            const float f = sp_unkey((uint32_t)(code >> 32));
            w = sp_weight(f, r, sh);
            d = min((int)sp_dist(f, r), SP_BINS - 1);
        }
        if (k && k < listed && code < sp_border(sh, tid < listed, d, code, 1, (u64)k)) w = 0;
        if (by_p) {
            const u64 limit = sp_share((double)top_p, sp_block_sum(sh, w), 1);
            if (code < sp_border(sh, w != 0, d, code, w, limit)) w = 0;
        }
        if (w < least_w) w = 0;
        // the pick: the same in order of index
        const int bits = 32 - __builtin_clz(V), shift = bits > 11 ? bits - 11 : 0;
        const u64 target = sp_target(us, sp_block_sum(sh, w));
        const u64 c = sp_border(sh, w != 0, (int)((0xFFFFFFFFu - (uint32_t)code) >> shift) & (SP_BINS - 1), (uint32_t)code, w, target + 1);
        if (tid == 0) tok[s] = (int)(0xFFFFFFFFu - (uint32_t)c);
        return;
    }

    // ---- top-p: the least token that is kept, by weights
    if (by_p) {
        sp_clear(sh);
        sp_each(sh, r, [&](const sw_f32x4 &x, int i, int) {
            bool on[4], any = false;
            int d[4];
            u64 w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                on[e] = sp_kept(x[e], i + e, r);
                d[e] = on[e] ? min((int)sp_dist(x[e], r), SP_BINS - 1) : 0;
                any |= on[e];
            }
            if (!__any(any)) return;
            sp_weights(x, on, r, sh, w);
            sp_add(sh, on, d, w);
        });
        u64 limit, before;
        const int b = sp_find(sh, [&](u64 total) { return sp_share((double)top_p, total, 1); }, limit, before);
        if (b >= 0) {
            const u64 c = sp_cut(sh, r, b, limit, before, true);
            r.lf = sp_unkey((uint32_t)(c >> 32));
            r.li = (int)(0xFFFFFFFFu - (uint32_t)c);
        }
    }
    // ---- the kept weights by group of tiles, in order of index: hist[group][wave]
    const int per = (r.ntile + SP_GROUPS_OF_TILES - 1) / SP_GROUPS_OF_TILES;
    auto kept4 = [&](const sw_f32x4 &x, int i) -> u64x4 {
        bool on[4], any = false;
        u64x4 w = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            on[e] = sp_kept(x[e], i + e, r);
            any |= on[e];
        }
        if (__any(any)) {
            u64 v[4];
            sp_weights(x, on, r, sh, v);
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = v[e];
            if (least_w)
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = v[e] < least_w ? 0 : v[e];
        }
        return w;
    };
    __syncthreads();
    u64 acc = 0;
    int left = per, group = 0;
    sp_each(sh, r, [&](const sw_f32x4 &x, int i, int t) {
        const u64x4 w = kept4(x, i);
        acc += (w[0] + w[1]) + (w[2] + w[3]);
        if (--left && t + 1 < r.ntile) return;
        const u64 v = sp_wave_sum(acc);
        if (lane == 0) sh.hist[group * SP_NW + wave] = v;
        acc = 0;
        left = per;
        group++;
    });
    __syncthreads();
    u64 base, mine = 0;
    if (tid < group)
#pragma unroll
        for (int q = 0; q < SP_NW; q++) mine += sh.hist[tid * SP_NW + q];
    u64 target = sp_target(us, sp_block_sum(sh, mine, &base));
    if (base <= target && target < base + mine) { sh.bin = tid; sh.before = base; }
    __syncthreads();
    target -= sh.before;
    // ---- that group's tiles one by one
    for (int t = sh.bin * per; t < r.ntile; t++) {
        const sw_f32x4 x = t < SP_CACHE ? sh.tile[t * SP_NT + tid] : sp_load(r, t);
        const u64x4 w = kept4(x, t * SP_TILE + 4 * tid);
        const u64 sum = (w[0] + w[1]) + (w[2] + w[3]);
        u64 at;
        const u64 all = sp_block_sum(sh, sum, &at);
        if (all <= target) { target -= all; continue; }
        if (at <= target && target < at + sum) {
            int e = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                at += w[j];
                e += at <= target;
            }
            tok[s] = t * SP_TILE + 4 * tid + e;
        }
        return;
    }
}

int sw_launch_sample(hipStream_t st, const float *logits, int S, int V, const SwSample &p, const float *u, int *tok) {
    SW_LAUNCH(k_sample, dim3((unsigned)S), dim3(SP_NT), 0, st, logits, V, p, u, tok);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
