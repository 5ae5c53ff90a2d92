// k_cache.hip -- writing the paged cache: the projection's heads normalised, turned and
// appended, and pages copied.
#include "sw_attn.h"

// A wave takes a row's heads one after the other, a lane the pairs lane and lane + 64 of a
// head, so both values of a turn, and a head's sum of squares but for one reduction, are
// in its registers.  Pair i < np of the turned part is values (i, i + np) or, interleaved,
// (2i, 2i + 1); the values behind it pass through as pairs (2i, 2i + 1), as all of v's do.
// The angle pos * freq[i] and its distance to the next full turn are taken in 64 bits: at
// position 10^6 a 32-bit product is 0.06 radians off.
#define RP_NT 256
template <int TYPE>
__global__ __launch_bounds__(RP_NT) void k_qk_rope_append(SwKv c, SwRows r, SwRope rope, const float *__restrict__ qkv, int64_t ld,
                                                          const float *__restrict__ wq, const float *__restrict__ wk, float eps,
                                                          int Hq, float *__restrict__ q_out, int hpw) {
    const int lane = threadIdx.x & 63, s = blockIdx.x;
    const int H = Hq + 2 * c.Hkv, h0 = (blockIdx.y * (RP_NT / 64) + (threadIdx.x >> 6)) * hpw;
    const int pos = r.pos[s];
    if (pos < 0 || h0 >= H) return;
    const int page = sw_page(c, r, r.seq ? r.seq[s] : s, pos);
    const int64_t cell = (int64_t)page * c.ps + (int64_t)(pos & ((1 << c.psh) - 1)) * c.ts;
    float cs[2], sn[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int i = lane + 64 * j;
        cs[j] = 1.f; sn[j] = 0.f;
        if (i < rope.np) {
            double t = (double)pos * rope.freq[i] * 0.15915494309189533577;      // full turns
            t = t - rint(t);
            sincospif((float)(t + t), &sn[j], &cs[j]);
            cs[j] = cs[j] * rope.factor;
            sn[j] = sn[j] * rope.factor;
        }
    }
    const float *x = qkv + (int64_t)s * ld;
    for (int h = h0; h < min(h0 + hpw, H); h++) {
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
}

int sw_launch_qk_rope_append(hipStream_t st, const SwKv &c, const SwRows &r, const SwRope &rope, const float *qkv, int64_t ld,
                             const float *wq, const float *wk, float eps, int Hq, float *q_out, int S) {
    const int H = Hq + 2 * c.Hkv, hpw = 1;
    const dim3 grid((unsigned)S, (unsigned)((H + RP_NT / 64 * hpw - 1) / (RP_NT / 64 * hpw)));
    if (c.type == SW_KV_F32) SW_LAUNCH(k_qk_rope_append<SW_KV_F32>, grid, dim3(RP_NT), 0, st, c, r, rope, qkv, ld, wq, wk, eps, Hq, q_out, hpw);
    else if (c.type == SW_KV_BF16) SW_LAUNCH(k_qk_rope_append<SW_KV_BF16>, grid, dim3(RP_NT), 0, st, c, r, rope, qkv, ld, wq, wk, eps, Hq, q_out, hpw);
    else SW_LAUNCH(k_qk_rope_append<SW_KV_F16>, grid, dim3(RP_NT), 0, st, c, r, rope, qkv, ld, wq, wk, eps, Hq, q_out, hpw);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// A page is n2 x n1 runs of `run` 16-byte pieces (one run where its cells lie side by side).
// The pairs and the pools' addresses travel with the launch: nothing to upload, and a
// recorded copy keeps its own.
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
