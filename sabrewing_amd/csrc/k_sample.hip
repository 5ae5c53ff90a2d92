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
//   the largest logit;
//   a top-k of up to SP_LIST / 2: the k-th largest of the threads' own maxima bounds the k-th
//     largest logit from below and little more than k logits reach it; they are listed, and all the
//     rest is done on the list (as is min-p alone, where few weights reach it);
//   else a histogram over the distance to the largest logit, of counts for top-k, then of
//     weights for top-p; the tokens of the bin in which the beginning ends are listed and ranked;
//   the kept weights of each tile, then of the one tile in which the sum passes.
// Weights are what costs in the passes over all of a large row (some 20 64-bit operations each).
#include "sw_attn.h"
#include "sw_gate.h"

#define SP_NT 1024
#define SP_NW (SP_NT / 64)
#define SP_TILE (4 * SP_NT)
#define SP_CACHE 8                        // tiles in LDS: 128 KB
#define SP_BINS 2048
#define SP_LIST 512
#define SP_MAXTILES 256                   // 2^20 logits
#define SP_ONE 4398046511104.0            // 2^42
#define SP_FAR 43.5f                      // log2 of the largest weight over one that rounds to 0
#define SP_SCALE 47.0f                    // bins per halving

typedef unsigned long long u64;
typedef float sp_f32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct SpShared {
    sw_f32x4 tile[SP_CACHE * SP_NT];
    u64 hist[SP_BINS];                    // (also the tiles' sums)
    u64 code[SP_LIST], weight[SP_LIST];
    u64 part[SP_NW], found, before, acc;
    double pow2[32];                      // 2^(42 + j / 32)
    int n, bin, pick;
};
struct SpRow {
    const float *v;
    int V, ntile;
    float fmax, c32;                      // the largest logit; log2(e) / T
    double m64, c64;
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
// f(logit, index) over all of the row, four tiles' loads ahead; done(tile) after each tile
template <class F, class G>
__device__ __forceinline__ void sp_each(const SpShared &sh, const SpRow &r, F f, G done) {
    for (int k0 = 0; k0 < r.ntile; k0 += 4) {
        sw_f32x4 x[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (k0 + j < r.ntile) x[j] = k0 < SP_CACHE ? sh.tile[(k0 + j) * SP_NT + threadIdx.x] : sp_load(r, k0 + j);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (k0 + j >= r.ntile) break;
            const int i = (k0 + j) * SP_TILE + 4 * (int)threadIdx.x;
#pragma unroll
            for (int e = 0; e < 4; e++) f(x[j][e], i + e);
            done(k0 + j);
        }
    }
}

__device__ __forceinline__ u64 sp_code(float f, int i) { return ((u64)ord_f32(f + 0.0f) << 32) | (0xFFFFFFFFu - (uint32_t)i); }
// log2(largest weight / weight), for bins and for what has no weight: NaN or infinite then
__device__ __forceinline__ float sp_dist(float f, const SpRow &r) { return f == r.fmax ? 0.f : (r.fmax - f) * r.c32; }
__device__ __forceinline__ int sp_bin(float d) { return (int)(d * SP_SCALE); }            // d in [0, SP_FAR]: below SP_BINS
// 2^42 2^((f - max) c) to the nearest whole number: 32 steps of a halving from a table, the rest (at
// most 2^-6 of one) by the exponential's series to the fifth power, 2e-15 off
__device__ __forceinline__ u64 sp_weight(float f, const SpRow &r, const SpShared &sh) {
    constexpr double L = 0.69314718055994530942 / 32, MAGIC = 6755399441055744.0;         // 1.5 * 2^52: rounds to whole numbers
    if (f == r.fmax) return (u64)SP_ONE;
    const double x = (double)f - r.m64;
    const double t = __builtin_fma(x, r.c64, MAGIC);
    const int k = (int)(uint32_t)__builtin_bit_cast(u64, t);
    const double z = __builtin_fma(x, r.c64, MAGIC - t);
    const double p = __builtin_fma(z, __builtin_fma(z, __builtin_fma(z, __builtin_fma(z, __builtin_fma(z, L * L * L * L * L / 120, L * L * L * L / 24),
                                                                                      L * L * L / 6), L * L / 2), L), 1.0);
    const double w = __builtin_fma(p, __builtin_ldexp(sh.pow2[k & 31], k >> 5), 4503599627370496.0);
    return __builtin_bit_cast(u64, w) & 0xFFFFFFFFFFFFFull;
}

__device__ __forceinline__ u64 sp_wave_sum(u64 v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// the block's sum, and with `before` the sum of the threads before this one
__device__ __forceinline__ u64 sp_block_sum(SpShared &sh, u64 v, u64 *before = nullptr) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 x = v;
    if (before) {
        for (int o = 1; o < 64; o <<= 1) { const u64 t = __shfl_up(x, o); if (lane >= o) x += t; }
    } else {
        x = sp_wave_sum(x);
    }
    __syncthreads();
    if (lane == 63) sh.part[wave] = x;
    __syncthreads();
    u64 t = 0;
    if (before) *before = x - v;
    for (int q = 0; q < SP_NW; q++) {
        if (before && q < wave) *before += sh.part[q];
        t += sh.part[q];
    }
    return t;
}

// hist[b] += w for the lanes with `on` (lanes of one bin, a row of equal logits say, in one addition)
__device__ __forceinline__ void sp_add(SpShared &sh, bool on, int b, u64 w) {
    const u64 any = __ballot(on);
    if (!any) return;
    const int b0 = __builtin_amdgcn_readlane(b, __builtin_ctzll(any));
    if (__ballot(on && b != b0) == 0 && __popcll(any) > 4) {
        w = sp_wave_sum(on ? w : 0);
        if ((threadIdx.x & 63) == 0) atomicAdd(&sh.hist[b0], w);
    } else if (on) {
        atomicAdd(&sh.hist[b], w);
    }
}
__device__ __forceinline__ void sp_clear(SpShared &sh) {
    __syncthreads();
    sh.hist[threadIdx.x] = sh.hist[threadIdx.x + SP_NT] = 0;
    __syncthreads();
}
// The bin in which the histogram's sum, from bin 0 (up: from the last), reaches `limit`, and the sum
// before it; -1: never.
__device__ __forceinline__ int sp_find(SpShared &sh, u64 limit, u64 &before, bool up = false) {
    const int t = threadIdx.x, b0 = up ? SP_BINS - 1 - 2 * t : 2 * t, b1 = up ? b0 - 1 : b0 + 1;
    __syncthreads();
    const u64 a = sh.hist[b0], b = sh.hist[b1];
    if (t == 0) sh.bin = -1;
    u64 at;
    sp_block_sum(sh, a + b, &at);
    if (at < limit && at + a + b >= limit) {
        const bool first = at + a >= limit;
        sh.bin = first ? b0 : b1;
        sh.before = first ? at : at + a;
    }
    __syncthreads();
    before = sh.before;
    return sh.bin;
}
// the lanes with `on` into the list (beyond its end they are counted)
__device__ __forceinline__ void sp_list(SpShared &sh, bool on, u64 code, u64 w) {
    const u64 any = __ballot(on);
    if (!any) return;
    const int lane = threadIdx.x & 63, first = __builtin_ctzll(any);
    int at = 0;
    if (lane == first) at = atomicAdd(&sh.n, (int)__popcll(any));
    at = __builtin_amdgcn_readlane(at, first) + (int)__popcll(any & ((1ull << lane) - 1));
    if (on && at < SP_LIST) { sh.code[at] = code; sh.weight[at] = w; }
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

// The code at which the beginning ends, among codes >= least: after `limit` tokens, or (mass) with the
// token at which the weights' sum reaches `limit`.  The histogram's bin holding it is narrowed by bits of
// the code until the list takes its tokens.  `over`: what counts, of the whole beginning.
__device__ u64 sp_cut(SpShared &sh, const SpRow &r, int bin, u64 limit, u64 before, bool mass, u64 least, u64 &over) {
    u64 prefix = 0, mask = 0;
    int shift = 64;
    for (;;) {
        __syncthreads();
        if (threadIdx.x == 0) { sh.n = 0; sh.found = 0; sh.acc = 0; }
        __syncthreads();
        sp_each(sh, r, [&](float f, int i) {
            const float d = sp_dist(f, r);
            const u64 c = sp_code(f, i);
            const bool on = d <= SP_FAR && sp_bin(d) == bin && (c & mask) == prefix && c >= least;
            u64 w = 1;
            if (mass && __any(on)) w = sp_weight(f, r, sh);
            sp_list(sh, on, c, w);
        }, [](int) {});
        __syncthreads();
        if (sh.n <= SP_LIST) break;
        shift = shift > 11 ? shift - 11 : 0;                          // 2048 ways by the next bits
        sp_clear(sh);
        sp_each(sh, r, [&](float f, int i) {
            const float d = sp_dist(f, r);
            const u64 c = sp_code(f, i);
            const bool on = d <= SP_FAR && sp_bin(d) == bin && (c & mask) == prefix && c >= least;
            u64 w = 1;
            if (mass && __any(on)) w = sp_weight(f, r, sh);
            sp_add(sh, on, (int)(c >> shift) & (SP_BINS - 1), w);
        }, [](int) {});
        u64 more;
        const int b = sp_find(sh, limit - before, more, true);
        before += more;
        prefix |= (u64)b << shift;
        mask |= (u64)(SP_BINS - 1) << shift;
    }
    const int n = sh.n, t = threadIdx.x;
    if (t < n) {
        const u64 c = sh.code[t], w = sh.weight[t];
        u64 at = before;
        for (int j = 0; j < n; j++)
            if (sh.code[j] > c) at += sh.weight[j];
        if (at < limit && at + w >= limit) { sh.found = c; sh.acc = at + w; }
    }
    __syncthreads();
    over = sh.acc;
    return sh.found;
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
    // ---- the largest logit: each thread's first, in order of index
    float best = -INFINITY;
    int bi = -1;
    for (int k0 = 0; k0 < r.ntile; k0 += 4) {
        sw_f32x4 x[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (k0 + j < r.ntile) x[j] = sp_load(r, k0 + j);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (k0 + j >= r.ntile) break;
            if (k0 < SP_CACHE) sh.tile[(k0 + j) * SP_NT + tid] = x[j];
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (x[j][e] > best) { best = x[j][e]; bi = (k0 + j) * SP_TILE + 4 * tid + e; }
        }
    }
    u64 top = bi < 0 ? 0 : sp_code(best, bi);
    for (int o = 32; o; o >>= 1) { const u64 t = __shfl_xor(top, o); top = t > top ? t : top; }
    if (lane == 0) sh.part[wave] = top;
    if (tid < 32) sh.pow2[tid] = exp2((double)tid / 32) * SP_ONE;
    __syncthreads();
    for (int q = 0; q < SP_NW; q++) top = sh.part[q] > top ? sh.part[q] : top;
    const int arg = top ? (int)(0xFFFFFFFFu - (uint32_t)top) : 0;
    if (!(temp > 0.f) || !top) {                                      // greedy, or nothing to draw from
        if (tid == 0) tok[s] = f0 != f0 ? 0 : arg;
        return;
    }
    {
        const uint32_t o = (uint32_t)(top >> 32);                     // back from the order bits
        r.fmax = __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
    }
    r.m64 = (double)r.fmax;
    r.c64 = 32 * 1.4426950408889634074 / (double)temp;                // (in steps of 1/32 halving)
    r.c32 = (float)(1.4426950408889634074 / (double)temp);
    const double least_w = min_p > 0.f ? fmin((double)min_p, 1.0) * SP_ONE : 0.0;

    // ---- few tokens can be kept: list them and stay there
    const bool by_p = top_p < 1.f;
    if ((k > 0 && k <= SP_LIST / 2) || (!k && !by_p && min_p > 0.f)) {
        int bound = SP_BINS - 1;
        if (k) {
            sp_clear(sh);
            const float d = sp_dist(best, r);
            sp_add(sh, bi >= 0 && d <= SP_FAR, bi >= 0 && d <= SP_FAR ? sp_bin(d) : 0, 1);
            u64 before;
            const int b = sp_find(sh, (u64)k, before);
            if (b >= 0) bound = b;
        }
        if (!by_p && min_p > 0.f) bound = min(bound, sp_bin(fminf(-log2f(fminf(min_p, 1.f)) + 0.05f, SP_FAR)) + 1);
        __syncthreads();
        if (tid == 0) { sh.n = 0; sh.pick = 0x7FFFFFFF; }
        __syncthreads();
        sp_each(sh, r, [&](float f, int i) {
            const float d = sp_dist(f, r);
            const bool on = d <= SP_FAR && sp_bin(d) <= bound;
            u64 w = 0;
            if (__any(on)) w = sp_weight(f, r, sh);
            sp_list(sh, on, sp_code(f, i), w);
        }, [](int) {});
        __syncthreads();
        const int n = sh.n;
        if (n <= SP_LIST) {
            u64 code = 0, w = 0, at = 0;
            int rank = 0;
            if (tid < n) {
                code = sh.code[tid];
                w = sh.weight[tid];
                for (int j = 0; j < n; j++)
                    if (sh.code[j] > code) { rank++; at += sh.weight[j]; }
            }
            bool kept = tid < n && (!k || rank < k);
            if (by_p) {
                const u64 total = sp_block_sum(sh, kept ? w : 0);
                kept = kept && at < sp_share((double)top_p, total, 1);
            }
            kept = kept && (double)w >= least_w;
            const u64 total = sp_block_sum(sh, kept ? w : 0);
            const u64 target = sp_target(us, total);
            __syncthreads();
            if (tid < n && !kept) sh.weight[tid] = 0;
            __syncthreads();
            if (kept && w) {                                          // the kept weights up to this index
                u64 sum = 0;
                for (int j = 0; j < n; j++)
                    if ((uint32_t)sh.code[j] >= (uint32_t)code) sum += sh.weight[j];
                if (sum > target) atomicMin(&sh.pick, (int)(0xFFFFFFFFu - (uint32_t)code));
            }
            __syncthreads();
            if (tid == 0) tok[s] = sh.pick;
            return;
        }
    }

    // ---- the least code that is kept
    u64 least = 0, total = 0;
    if (k) {
        sp_clear(sh);
        sp_each(sh, r, [&](float f, int) {
            const float d = sp_dist(f, r);
            sp_add(sh, d <= SP_FAR, d <= SP_FAR ? sp_bin(d) : 0, 1);
        }, [](int) {});
        u64 before, n;
        const int b = sp_find(sh, (u64)k, before);
        if (b >= 0) least = sp_cut(sh, r, b, (u64)k, before, false, 0, n);
    }
    if (by_p) {
        sp_clear(sh);
        u64 sum = 0;
        sp_each(sh, r, [&](float f, int i) {
            const float d = sp_dist(f, r);
            const bool on = d <= SP_FAR && sp_code(f, i) >= least;
            u64 w = 0;
            if (__any(on)) w = sp_weight(f, r, sh);
            if (!on) w = 0;
            sum += w;
            sp_add(sh, on, on ? sp_bin(d) : 0, w);
        }, [](int) {});
        total = sp_block_sum(sh, sum);
        u64 before, over;
        const u64 limit = sp_share((double)top_p, total, 1);
        const int b = sp_find(sh, limit, before);
        if (b >= 0) {
            const u64 c = sp_cut(sh, r, b, limit, before, true, least, over);
            least = c > least ? c : least;
        }
    }
    // ---- the kept weights by tile, in order of index
    __syncthreads();
    if (tid < SP_MAXTILES) sh.hist[tid] = 0;
    __syncthreads();
    u64 w4 = 0;
    sp_each(sh, r, [&](float f, int i) {
        const bool on = sp_dist(f, r) <= SP_FAR && sp_code(f, i) >= least;
        if (!__any(on)) return;
        const u64 w = sp_weight(f, r, sh);
        if (on && (double)w >= least_w) w4 += w;
    }, [&](int t) {
        if (__any(w4 != 0)) {
            const u64 x = sp_wave_sum(w4);
            if (lane == 0) atomicAdd(&sh.hist[t], x);
        }
        w4 = 0;
    });
    __syncthreads();
    u64 before;
    const u64 mine = tid < r.ntile ? sh.hist[tid] : 0;
    total = sp_block_sum(sh, mine, &before);
    const u64 target = sp_target(us, total);
    if (before <= target && target < before + mine) { sh.bin = tid; sh.before = before; }
    __syncthreads();
    const int t = sh.bin;
    const u64 base = sh.before;
    // ---- the tile's four of each thread
    const sw_f32x4 x = t < SP_CACHE ? sh.tile[t * SP_NT + tid] : sp_load(r, t);
    u64 w[4], sum = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const bool on = sp_dist(x[e], r) <= SP_FAR && sp_code(x[e], t * SP_TILE + 4 * tid + e) >= least;
        w[e] = on ? sp_weight(x[e], r, sh) : 0;
        if ((double)w[e] < least_w) w[e] = 0;
        sum += w[e];
    }
    u64 at;
    sp_block_sum(sh, sum, &at);
    at += base;
    if (at <= target && target < at + sum) {
        int e = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            at += w[j];
            e += at <= target;
        }
        tok[s] = t * SP_TILE + 4 * tid + e;
    }
}

int sw_launch_sample(hipStream_t st, const float *logits, int S, int V, const SwSample &p, const float *u, int *tok) {
    SW_LAUNCH(k_sample, dim3((unsigned)S), dim3(SP_NT), 0, st, logits, V, p, u, tok);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
