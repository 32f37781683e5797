// tg_kvq_attn.cu — attention of many tokens over the paged 4-bit key/value cache.
//
//   s_r = scale * q . k_r over the rows r up to the token's own, p = softmax(s),
//   out = sum_r p_r v_r
// in one pass over the rows: the running maximum m and sum l of exp(s - m) are kept with
// the output, which is rescaled when m grows.  fp32 throughout.
//
// One warp per (token, head): 32 rows at a time, a row per lane for the scores, the
// dimensions 32b + l per lane for the sum.
#include "tg_serve.cuh"

namespace tg {

namespace {

constexpr int WARPS = 4;

struct AttnKvqArgs {
    KvqCache c;
    KvqBatch b;
    int T, NH;
    const void* q;
    long long qs;
    void* out;
    long long os;
    float scale;   // times log2(e)
};

template <int DT, int NB>
__global__ void __launch_bounds__(32 * WARPS) k_kvq_attn(AttnKvqArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int HD = 32 * NB;
    __shared__ float s_q[WARPS][HD];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const long long w = (long long)blockIdx.x * WARPS + wid;
    const int t = (int)(w / a.NH), h = (int)(w % a.NH), j = h / (a.NH / a.c.nkv);
    if (t >= a.T) return;
    const int b = kvq_find_seq(a.b, t, lane);
    const int s0 = a.b.q_start[b], s1 = a.b.q_start[b + 1];
    if (t < s0 || t >= s1) return;
    if (t - s0 >= a.b.max_new) {
        if (lane == 0) kvq_flag(a.b, TGX_KVQ_BAD_NEW);
        return;
    }
    long long rows = (long long)a.b.kv_lens[b] - (s1 - t) + 1;
    const long long cap = (long long)a.b.max_pages * a.c.pt;
    if (rows > cap) {
        if (lane == 0) kvq_flag(a.b, TGX_KVQ_BAD_LENGTH);
        rows = cap;
    }
    const T* q = reinterpret_cast<const T*>(a.q) + (size_t)t * a.qs + (size_t)h * HD;
    float* sq = s_q[wid];
#pragma unroll
    for (int i = 0; i < NB; i++) sq[32 * i + lane] = to_f32(q[32 * i + lane]);
    __syncwarp();
    float m = -INFINITY, l = 0.0f, o[NB];
#pragma unroll
    for (int i = 0; i < NB; i++) o[i] = 0.0f;
    for (int r0 = 0; r0 < rows; r0 += 32) {
        const int r = r0 + lane;
        int page = -1;
        if (r < rows) {
            page = a.b.table[(size_t)b * a.b.max_pages + r / a.c.pt];
            if (page < 0 || page >= a.c.n_pages) {
                kvq_flag(a.b, TGX_KVQ_BAD_PAGE);
                page = -1;
            }
        }
        const uint8_t* gr = page >= 0 ? kvq_granule(a.c, page, j, r % a.c.pt) : nullptr;
        const int tk = r & 15;
        float s = -INFINITY;
        if (gr) {
            const uint16_t* sc = reinterpret_cast<const uint16_t*>(gr + 16 * HD) + tk * NB;
            s = 0.0f;
            for (int i = 0; i < NB; i++) {
                float dot = 0.0f;
                for (int c = 0; c < 4; c++) {
                    const uint32_t x = *reinterpret_cast<const uint32_t*>(gr + ((tk >> 3) * 32 + (tk & 7) * 4 + c) * (HD / 8) + 4 * i);
#pragma unroll
                    for (int n = 0; n < 8; n++)   // halfword e = n / 4, nibble n % 4
                        dot = fmaf(sq[32 * i + 8 * (n & 3) + 2 * c + (n >> 2)], (float)((int)(x >> (4 * n) & 15) - 8), dot);
                }
                s = fmaf(dot, __half2float(__ushort_as_half(sc[i])), s);
            }
            s *= a.scale;
        }
        float top = s;
#pragma unroll
        for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float mn = fmaxf(m, top);
        const bool any = mn > -INFINITY;
        const float p = any && gr ? exp2f(s - mn) : 0.0f;
        const float f = any ? exp2f(m - mn) : 1.0f;
        m = mn;
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < NB; i++) o[i] *= f;
        const unsigned long long g64 = (unsigned long long)gr;
        for (int n = 0; n < 32; n++) {
            const uint8_t* gn = (const uint8_t*)__shfl_sync(0xffffffffu, g64, n);
            const float pn = __shfl_sync(0xffffffffu, p, n);
            if (!gn) continue;
            const int tn = (r0 + n) & 15, hc = (tn >> 3) * 32 + ((tn & 7) >> 1);
            const uint16_t* sc = reinterpret_cast<const uint16_t*>(gn + 17 * HD) + ((tn >> 3) * 4 + ((tn & 7) >> 1)) * NB * 2 + (tn & 1);
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const uint32_t x = *reinterpret_cast<const uint16_t*>(gn + 8 * HD + (hc + 4 * (lane & 7)) * (HD / 8) + 4 * i + 2 * (tn & 1));
                o[i] = fmaf(pn * __half2float(__ushort_as_half(sc[2 * i])), (float)((int)(x >> (4 * (lane >> 3)) & 15) - 8), o[i]);
            }
        }
    }
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    T* out = reinterpret_cast<T*>(a.out) + (size_t)t * a.os + (size_t)h * HD;
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
#pragma unroll
    for (int i = 0; i < NB; i++) from_f32(o[i] * inv, out[32 * i + lane]);
}

template <int DT>
cudaError_t launch_attn(const AttnKvqArgs& a, cudaStream_t s) {
    const unsigned grid = (unsigned)(((long long)a.T * a.NH + WARPS - 1) / WARPS);
    switch (a.c.hd / 32) {
#define TG_CASE(n) case n: k_kvq_attn<DT, n><<<grid, 32 * WARPS, 0, s>>>(a); break;
        TG_CASE(1) TG_CASE(2) TG_CASE(3) TG_CASE(4) TG_CASE(5) TG_CASE(6) TG_CASE(7) TG_CASE(8)
#undef TG_CASE
    }
    return cudaGetLastError();
}

}  // namespace

}  // namespace tg

extern "C" size_t tgx_kvq_attention_scratch_bytes(const tgx_kvq_cache* cache, const tgx_kvq_batch* batch, int n_tokens,
                                                  int n_heads) {
    if (!cache || !batch || n_tokens < 0 || n_heads <= 0 || cache->n_kv_heads <= 0 || n_heads % cache->n_kv_heads) return 0;
    return 256;
}

extern "C" int tgx_kvq_attention(const tgx_kvq_cache* cache, const tgx_kvq_batch* batch, int dtype, int n_tokens,
                                 const void* q, long long q_stride, int n_heads, void* out, long long out_stride,
                                 float scale, void* scratch, size_t scratch_bytes, void* stream) {
    const char* fn = "tgx_kvq_attention";
    int rc = tg::kvq_check(fn, cache, batch);
    if (rc != TG_OK) return rc;
    if (!q || !out || !scratch) return tg::serve_fail(TG_EINVAL, fn, "null pointer");
    if (dtype < TGX_F32 || dtype > TGX_F16) return tg::serve_fail(TG_EINVAL, fn, "unknown dtype");
    if (n_tokens < 0 || n_heads <= 0 || n_heads % cache->n_kv_heads || n_heads / cache->n_kv_heads > 32)
        return tg::serve_fail(TG_EINVAL, fn, "n_heads must be a multiple of n_kv_heads, at most 32 per kv head");
    const long long w = (long long)n_heads * cache->head_dim;
    if (q_stride < w || out_stride < w || (q_stride | out_stride) % 4)
        return tg::serve_fail(TG_EINVAL, fn, "strides must cover a row and be multiples of 4 elements");
    const size_t al = 4 * tg::elem_bytes(dtype);
    if (!tg::aligned(q, al) || !tg::aligned(out, al)) return tg::serve_fail(TG_EINVAL, fn, "rows must be 4-element aligned");
    if (!tg::aligned(scratch, 256) || scratch_bytes < tgx_kvq_attention_scratch_bytes(cache, batch, n_tokens, n_heads))
        return tg::serve_fail(TG_EINVAL, fn, "scratch must be 256-byte aligned, of tgx_kvq_attention_scratch_bytes");
    if ((long long)n_tokens * n_heads / tg::WARPS >= 0x7fffffffll)
        return tg::serve_fail(TG_EINVAL, fn, "too many tokens for one call");
    if (!(scale >= 0.0f) || scale > 3e38f) return tg::serve_fail(TG_EINVAL, fn, "scale must be finite and not negative");
    tg::ServeDevice dev(fn, cache->pages);
    if (dev.rc != TG_OK || n_tokens == 0) return dev.rc;
    const float sc = (scale > 0.0f ? scale : 1.0f / sqrtf((float)cache->head_dim)) * 1.44269504088896340736f;
    tg::AttnKvqArgs a{tg::kvq_cache(*cache), tg::kvq_batch(*batch), n_tokens, n_heads, q, q_stride, out, out_stride, sc};
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e = dtype == TGX_F32    ? tg::launch_attn<TGX_F32>(a, s)
                    : dtype == TGX_BF16 ? tg::launch_attn<TGX_BF16>(a, s)
                                        : tg::launch_attn<TGX_F16>(a, s);
    return e == cudaSuccess ? TG_OK : tg::serve_fail(TG_ECUDA, fn, cudaGetErrorString(e));
}
