// sw_attn.h -- the paged cache as its kernels see it (k_cache.hip, k_attn.hip).
#ifndef SW_ATTN_H
#define SW_ATTN_H
#include "sw_hip.h"

enum { SW_KV_F32 = 0, SW_KV_BF16 = 1, SW_KV_F16 = 2 };

// One layer's pools of k and v: cell (page, head, slot) holds head_dim values at
// page * ps + head * hs + slot * ts (elements of the pool's type, 64-bit offsets: a long
// cache passes 32 bits).  page_size = 1 << psh.
struct SwKv {
    void *k, *v;
    int type, n_pages, psh, Hkv, dh;
    int64_t ps, hs, ts;
};
// Row s of a batch: position pos[s] (negative: no row) of sequence seq[s] (null: s), whose
// token t lies in page table[seq * max_pages + (t >> psh)], slot t & (page_size - 1).
struct SwRows {
    const int *pos, *seq, *table;
    int n_seqs, max_pages;
};

// the page of token t of sequence q, or -1 where the table or its entry leads nowhere
__device__ __forceinline__ int sw_page(const SwKv &c, const SwRows &r, int q, int t) {
    const int i = t >> c.psh;
    if (q < 0 || q >= r.n_seqs || t < 0 || i >= r.max_pages) return -1;
    const int p = r.table[(int64_t)q * r.max_pages + i];
    return p >= 0 && p < c.n_pages ? p : -1;
}

// f32 to the cache's type, to nearest even (a NaN stays one)
__device__ __forceinline__ uint16_t sw_bf16_rne(float f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, f);
    return f != f ? (uint16_t)(u >> 16 | 0x40) : (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1)) >> 16);
}
template <int TYPE>
__device__ __forceinline__ void sw_kv_store(void *p, int64_t i, float f) {
    if constexpr (TYPE == SW_KV_F32) ((float *)p)[i] = f;
    else if constexpr (TYPE == SW_KV_BF16) ((uint16_t *)p)[i] = sw_bf16_rne(f);
    else ((_Float16 *)p)[i] = (_Float16)f;
}

// A value and its partner's 16 or 32 lanes away (as a pair in no order): each swap exchanges
// the rows of 16, or the halves, of two registers.  (The second register is hidden from the
// compiler, which takes the swap of a register with itself for no change.)
template <int BY>
__device__ __forceinline__ uint2 sw_pair(uint32_t a) {
    uint32_t b = a;
    asm("" : "+v"(b));
    const auto r = BY == 16 ? __builtin_amdgcn_permlane16_swap(a, b, false, false) : __builtin_amdgcn_permlane32_swap(a, b, false, false);
    return make_uint2((uint32_t)r[0], (uint32_t)r[1]);
}
// sums up to each lane of a wave (shifts by 1, 2, 4, 8 in rows of 16, then the rows' last), the wave's maximum
__device__ __forceinline__ uint32_t sw_wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
    return v;
}
__device__ __forceinline__ uint32_t sw_wave_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xF, 0xF, false));
    uint2 p = sw_pair<16>(v);
    v = max(p.x, p.y);
    p = sw_pair<32>(v);
    return max(p.x, p.y);
}
// over the four lanes 16 apart
__device__ __forceinline__ float sw_max4(float x) {
    const uint2 a = sw_pair<16>(__builtin_bit_cast(uint32_t, x));
    const uint2 b = sw_pair<32>(__builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a.x), __builtin_bit_cast(float, a.y))));
    return fmaxf(__builtin_bit_cast(float, b.x), __builtin_bit_cast(float, b.y));
}
__device__ __forceinline__ float sw_sum4(float x) {
    const uint2 a = sw_pair<16>(__builtin_bit_cast(uint32_t, x));
    const uint2 b = sw_pair<32>(__builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a.x) + __builtin_bit_cast(float, a.y)));
    return __builtin_bit_cast(float, b.x) + __builtin_bit_cast(float, b.y);
}

// ---- launch wrappers (async on `st`) ----
// (k_cache.hip) the q and k heads of S projected rows normalised (wq, wk null: not) and
// turned (np pairs of a head, freq in radians per position), q to q_out, k and v to the cache
struct SwRope { const double *freq; int np, interleaved; float factor; };
int sw_launch_qk_rope_append(hipStream_t st, const SwKv &c, const SwRows &r, const SwRope &rope, const float *qkv, int64_t ld,
                             const float *wq, const float *wk, float eps, int Hq, float *q_out, int S);
// pages src[i] to dst[i] of n_layers caches of one geometry (host arrays, n <= SW_COPY_PAIRS,
// n_layers <= SW_COPY_LAYERS: they travel with the launch)
#define SW_COPY_PAIRS 256
#define SW_COPY_LAYERS 64
int sw_launch_kv_copy(hipStream_t st, const SwKv *layers, int n_layers, const int *src, const int *dst, int n);
// (k_attn.hip) one token of each row against its sequence's cells (pos - window, pos]; part:
// scratch of sw_attn_part_floats floats, 16-byte aligned (0: none)
int64_t sw_attn_row_chunks(const SwKv &c, const SwRows &r);           // chunks of the longest row there can be: 64 rows' fit 32 bits
int64_t sw_attn_part_floats(const SwKv &c, const SwRows &r, int Hq, int window, int S);
int sw_launch_attn(hipStream_t st, const SwKv &c, const SwRows &r, const float *q, int Hq, float scale, int window, float *out,
                   int S, float *part);
// (k_sample.hip) a pick of each row of logits; each setting may be null
struct SwSample { const float *temp; const int *top_k; const float *top_p, *min_p; };
int sw_launch_sample(hipStream_t st, const float *logits, int S, int V, const SwSample &p, const float *u, int *tok);
#endif
