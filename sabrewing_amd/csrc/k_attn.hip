// k_attn.hip -- attention of one new token of each row over a paged cache:
// out[s, h] = sum_t p_t v_t, p = softmax over t in (pos - window, pos] of scale * q[s, h] . k_t.
#include "sw_attn.h"

// One block per (row, head), a wave per token in turn, a lane 1 to 4 of the head's values;
// each wave keeps the running maximum, sum and output of its tokens, and the waves join at
// the end.  All in 32 bits.
#define AT_NT 256
template <int TYPE>
__global__ __launch_bounds__(AT_NT) void k_attn(SwKv c, SwRows r, const float *__restrict__ q, int Hq, float scale, int window,
                                                float *__restrict__ out) {
    __shared__ float sm[4], sl[4], so[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, s = blockIdx.x, h = blockIdx.y;
    const int hk = h / (Hq / c.Hkv), pos = r.pos[s], sq = r.seq ? r.seq[s] : s;
    const int first = window > 0 && pos >= window ? pos - window + 1 : 0;
    const int last = min(pos, (r.max_pages << c.psh) - 1);             // (the host keeps that below 2^30)
    const int64_t row = ((int64_t)s * Hq + h) * c.dh;
    float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) qv[j] = lane + 64 * j < c.dh ? q[row + lane + 64 * j] : 0.f;
    for (int t = first + wave; t <= last; t += 4) {
        const int page = sw_page(c, r, sq, t);
        if (page < 0) continue;
        const int64_t cell = (int64_t)page * c.ps + (int64_t)hk * c.hs + (int64_t)(t & ((1 << c.psh) - 1)) * c.ts;
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (lane + 64 * j < c.dh) d = __builtin_fmaf(qv[j], sw_kv_load<TYPE>(c.k, cell + lane + 64 * j), d);
        for (int k = 32; k; k >>= 1) d += __shfl_xor(d, k);
        d = d * scale;
        const float nm = d > m || d != d ? d : m;
        if (nm == -INFINITY) continue;                             // no weight yet
        const float f = m == nm ? 1.f : expf(m - nm), p = expf(d - nm);
        l = __builtin_fmaf(l, f, p);
        m = nm;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (lane + 64 * j < c.dh) o[j] = __builtin_fmaf(o[j], f, p * sw_kv_load<TYPE>(c.v, cell + lane + 64 * j));
    }
    if (lane == 0) { sm[wave] = m; sl[wave] = l; }
#pragma unroll
    for (int j = 0; j < 4; j++) so[wave][lane + 64 * j] = o[j];
    __syncthreads();
    if ((int)threadIdx.x >= c.dh) return;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int w = 0; w < 4; w++) M = sm[w] > M || sm[w] != sm[w] ? sm[w] : M;
    for (int w = 0; w < 4; w++) {
        if (sl[w] == 0.f && sm[w] == -INFINITY) continue;          // a wave without tokens
        const float f = expf(sm[w] - M);
        L = __builtin_fmaf(sl[w], f, L);
        O = __builtin_fmaf(so[w][threadIdx.x], f, O);
    }
    out[row + threadIdx.x] = L == 0.f ? 0.f : O / L;
}

int sw_launch_attn(hipStream_t st, const SwKv &c, const SwRows &r, const float *q, int Hq, float scale, int window, float *out,
                   int S) {
    const dim3 grid((unsigned)S, (unsigned)Hq);
    if (c.type == SW_KV_F32) SW_LAUNCH(k_attn<SW_KV_F32>, grid, dim3(AT_NT), 0, st, c, r, q, Hq, scale, window, out);
    else if (c.type == SW_KV_BF16) SW_LAUNCH(k_attn<SW_KV_BF16>, grid, dim3(AT_NT), 0, st, c, r, q, Hq, scale, window, out);
    else SW_LAUNCH(k_attn<SW_KV_F16>, grid, dim3(AT_NT), 0, st, c, r, q, Hq, scale, window, out);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
