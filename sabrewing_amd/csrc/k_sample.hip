// k_sample.hip -- a token of each row of logits from a given random number.
//
// Weights are whole numbers, w_i = rint(2^42 exp((l_i - max) / T)), the exponential in 64
// bits: their sums are exact in 64-bit integers, so no order of threads or atomics changes a
// pick, and up to 2^20 of them fit.  (In floats a sum of 10^5 weights is 1e-6 off, and some row of a
// large batch picks the neighbour.)  The tokens in order of falling logit, equal ones by
// rising index; top-k keeps the first k, top-p the shortest beginning of those with at least
// top_p of their sum, min-p the weights of at least min_p of the largest: each keeps a
// beginning of that order, so the kept set is one threshold (a logit, and how many of its
// equals).  The pick is the lowest index at which the running sum of kept weights, in order
// of index, passes u times their sum.
#include "sw_attn.h"
#include "sw_gate.h"

#define SP_NT 1024
#define SP_ONE 4398046511104.0            // 2^42

typedef unsigned long long u64;

struct SpRow { uint32_t top; float fmax; double c; };                // the largest key, its logit, log2(e) / T
// order bits of a logit, 0 for NaN (-0 and +0 equal)
__device__ __forceinline__ uint32_t sp_key(float f) { return f == f ? ord_f32(f + 0.0f) : 0u; }
__device__ __forceinline__ u64 sp_weight(float f, const SpRow &r) {
    if (!(f > -INFINITY)) return 0;                                  // masked, or NaN
    if (f == r.fmax) return (u64)SP_ONE;                             // (also +inf, where the difference has no value)
    return (u64)rint(exp2(((double)f - (double)r.fmax) * r.c) * SP_ONE);
}

__device__ __forceinline__ u64 sp_block_sum(u64 v, u64 *part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if (lane == 0) part[wave] = v;
    __syncthreads();
    u64 t = 0;
    for (int q = 0; q < SP_NT / 64; q++) t += part[q];
    return t;
}

// The beginning of the order that ends where `limit` tokens (by_mass: less than `limit` of
// weight before the token) are reached, among the first keys >= floor_key (and of those equal
// to it the first floor_n): its last key, how many tokens of that key it has, and its weight.
__device__ void sp_select(const float *v, int V, const SpRow &r, int by_mass, u64 limit, u64 *mass, u64 *count, uint32_t &key,
                          u64 &n_eq, u64 &sum) {
    __shared__ u64 s_before[2];
    __shared__ uint32_t s_digit;
    uint32_t prefix = 0, mask = 0;
    u64 mass_before = 0, count_before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += SP_NT) mass[i] = count[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < V; i += SP_NT) {
            const float f = v[i];
            const uint32_t k = sp_key(f);
            if (k && (k & mask) == prefix) {
                atomicAdd(&count[(k >> shift) & 255], 1ull);
                atomicAdd(&mass[(k >> shift) & 255], sp_weight(f, r));
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            u64 m = mass_before, n = count_before;
            int d = 255, last = 255;
            for (; d >= 0; d--) {                    // the digit in which the limit is reached
                if (!count[d]) continue;
                last = d;
                if ((by_mass ? m + mass[d] : n + count[d]) >= limit) break;
                m += mass[d];
                n += count[d];
            }
            if (d < 0) { m -= mass[last]; n -= count[last]; }        // never reached: all of it
            s_digit = (uint32_t)last;
            s_before[0] = m;
            s_before[1] = n;
        }
        __syncthreads();
        mass_before = s_before[0];
        count_before = s_before[1];
        prefix |= s_digit << shift;
        mask |= 255u << shift;
    }
    const uint32_t d = prefix & 255;
    const u64 n = count[d], w = n ? mass[d] / n : 0;                 // equal keys: equal weights
    u64 take = n;
    if (!by_mass) take = limit > count_before ? (limit - count_before < n ? limit - count_before : n) : 0;
    else if (w) {
        const u64 need = limit > mass_before ? (limit - mass_before + w - 1) / w : 0;
        take = need < n ? need : n;
    }
    key = prefix;
    n_eq = take;
    sum = mass_before + take * w;
    __syncthreads();
}

__global__ __launch_bounds__(SP_NT) void k_sample(const float *__restrict__ logits, int V, SwSample p, const float *__restrict__ u,
                                                  int *__restrict__ tok) {
    __shared__ u64 part[SP_NT / 64], mass[256], count[256];
    __shared__ int s_pick;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, s = blockIdx.x;
    const float *v = logits + (int64_t)s * V;
    const float temp = p.temp ? p.temp[s] : 1.f;
    const int k = p.top_k ? p.top_k[s] : 0;
    const float top_p = p.top_p ? p.top_p[s] : 1.f, min_p = p.min_p ? p.min_p[s] : 0.f;
    u64 best = 0;
    for (int i = tid; i < V; i += SP_NT) {
        const u64 x = ((u64)sp_key(v[i]) << 32) | (0xFFFFFFFFu - (uint32_t)i);
        best = x > best ? x : best;
    }
    for (int o = 32; o; o >>= 1) { const u64 t = __shfl_xor(best, o); best = t > best ? t : best; }
    if (lane == 0) part[wave] = best;
    __syncthreads();
    for (int q = 0; q < SP_NT / 64; q++) best = part[q] > best ? part[q] : best;
    const uint32_t top = (uint32_t)(best >> 32);
    const int arg = (int)(0xFFFFFFFFu - (uint32_t)best);
    const float fmax = v[arg];
    if (!(temp > 0.f) || fmax != fmax || fmax == -INFINITY) {        // greedy, or nothing to draw from
        const float f0 = v[0];
        if (tid == 0) tok[s] = f0 != f0 ? 0 : arg;
        return;
    }
    SpRow r = {top, fmax, 1.4426950408889634074 / (double)temp};
    uint32_t key = 0;                        // kept: keys above it and its first n_eq equals
    u64 n_eq = 0, sum = 0;
    bool all = true;
    if (k > 0 && k < V) { sp_select(v, V, r, 0, (u64)k, mass, count, key, n_eq, sum); all = false; }
    if (top_p < 1.f) {
        if (all) {
            u64 w = 0;
            for (int i = tid; i < V; i += SP_NT) w += sp_weight(v[i], r);
            sum = sp_block_sum(w, part);
        }
        const double want = top_p > 0.f ? ceil((double)top_p * (double)sum) : 1.0;
        uint32_t key2;
        u64 n2, sum2;
        sp_select(v, V, r, 1, want < 1.0 ? 1ull : (u64)want, mass, count, key2, n2, sum2);
        if (all || key2 > key || (key2 == key && n2 < n_eq)) { key = key2; n_eq = n2; }
        all = false;
    }
    // min-p as a bound on the weight
    const double least = min_p > 0.f ? fmin((double)min_p, 1.0) * SP_ONE : 0.0;
    // the kept weights in order of index, tile by tile: their sum first, then the place of u * sum
    u64 total = 0, target = 0;
    for (int pass = 0; pass < 2; pass++) {
        u64 run = 0, eq = 0;
        for (int i0 = 0; i0 < V; i0 += SP_NT) {
            const int i = i0 + tid;
            const float f = i < V ? v[i] : NAN;
            const uint32_t kk = sp_key(f);
            // the index among the equals of the threshold
            const u64 is_eq = __ballot(!all && kk == key && kk);
            __syncthreads();
            if (lane == 0) part[wave] = __popcll(is_eq);
            __syncthreads();
            u64 rank = eq + __popcll(is_eq & ((1ull << lane) - 1));
            for (int q = 0; q < wave; q++) rank += part[q];
            for (int q = 0; q < SP_NT / 64; q++) eq += part[q];
            u64 w = kk && (all || kk > key || (kk == key && rank < n_eq)) ? sp_weight(f, r) : 0;
            if ((double)w < least) w = 0;
            if (pass == 0) { run += w; continue; }
            u64 x = w;                       // inclusive sums of the wave, then of the block
            for (int o = 1; o < 64; o <<= 1) { const u64 t = __shfl_up(x, o); if (lane >= o) x += t; }
            __syncthreads();
            if (lane == 63) part[wave] = x;
            if (tid == 0) s_pick = 0x7FFFFFFF;
            __syncthreads();
            u64 before = run;
            for (int q = 0; q < wave; q++) before += part[q];
            for (int q = 0; q < SP_NT / 64; q++) run += part[q];
            if (w && before + x > target) atomicMin(&s_pick, i);
            __syncthreads();
            if (s_pick != 0x7FFFFFFF) {
                if (tid == 0) tok[s] = s_pick;
                return;
            }
        }
        if (pass == 0) {
            total = sp_block_sum(run, part);
            const double t = (double)u[s] * (double)total;
            target = t > 0.0 ? (u64)t : 0;
            if (target >= total) target = total - 1;                 // u outside [0, 1)
        }
    }
    if (tid == 0) tok[s] = arg;              // (not reached: the last kept weight passes the target)
}

int sw_launch_sample(hipStream_t st, const float *logits, int S, int V, const SwSample &p, const float *u, int *tok) {
    SW_LAUNCH(k_sample, dim3((unsigned)S), dim3(SP_NT), 0, st, logits, V, p, u, tok);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
