// tg_kvq.cu — appending to the paged 4-bit key/value cache, and reading it back.
//
// Per new token: q and k heads RMS-normalised and rotated, k and v quantised to blocks of
// 32 (m = the value of the largest magnitude, the first of several; scale fp16(m / -8);
// code = min(15, floor(8.5 - 8 x / m))) and written at the token's row of its page.
//
// A code is cut at a border, so a rounding in front of it can move a value by a whole
// step.  Keys are therefore computed in 64 bits from the inputs to the code (B200 has full
// 64-bit rate to spare beside the memory traffic); values are exact in any width.  q has no
// borders: fp32, rounded once to its type.
//
// One warp per (token, head): lane l holds dimensions 32b + l, so block b is one value per
// lane.  Bound by memory; what it has to move is q in and out, k and v in, codes out.
#include "tg_serve.cuh"

namespace tg {

namespace {

constexpr int WARPS = 8;

struct AppendArgs {
    KvqCache c;
    KvqBatch b;
    int T, NH;
    const void *q, *k, *v;
    long long qs, ks, vs;
    const float *q_norm, *k_norm, *cos, *sin;
    float eps;
    int n_pos;
    const int32_t* positions;
    void* q_out;
};

// The other half's value of x's dimension: dimension d + 16 NB (d below the middle) or
// d - 16 NB, of every value of the lane.  NB even: the same lane's block b +- NB / 2; odd:
// lane ^ 16's.
template <int NB, typename T>
__device__ __forceinline__ void other_half(const T (&x)[NB], T (&o)[NB], int lane) {
    if constexpr (NB % 2 == 0) {
#pragma unroll
        for (int b = 0; b < NB; b++) o[b] = x[(b + NB / 2) % NB];
    } else {
        T y[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) y[b] = __shfl_xor_sync(0xffffffffu, x[b], 16);
        // lane < 16: dimension 32b + l pairs with block b + (NB - 1) / 2 or b - (NB + 1) / 2,
        // that is b + (NB - 1) / 2 modulo NB; lane >= 16: b + (NB + 1) / 2 modulo NB
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const T lo = y[(b + (NB - 1) / 2) % NB], hi = y[(b + (NB + 1) / 2) % NB];
            o[b] = lane < 16 ? lo : hi;
        }
    }
}

template <int NB, typename T, typename W>
__device__ __forceinline__ void norm_rotate(T (&x)[NB], const float* w, float eps, const float* cos, const float* sin,
                                            int pos, int lane, W rsqrt_of) {
    constexpr int HD = 32 * NB;
    if (w) {
        T ss = 0;
#pragma unroll
        for (int b = 0; b < NB; b++) ss += x[b] * x[b];
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const T r = rsqrt_of(ss / HD + (T)eps);
#pragma unroll
        for (int b = 0; b < NB; b++) x[b] = x[b] * r * (T)w[32 * b + lane];
    }
    if (cos) {
        T o[NB];
        other_half<NB>(x, o, lane);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int d = 32 * b + lane, i = d < HD / 2 ? d : d - HD / 2;
            const T c = cos[(size_t)pos * (HD / 2) + i], s = sin[(size_t)pos * (HD / 2) + i];
            x[b] = d < HD / 2 ? x[b] * c - o[b] * s : x[b] * c + o[b] * s;
        }
    }
}

// One block, a value per lane: the lane's code, and the scale's bits.
__device__ __forceinline__ int quant_block(double x, uint16_t& scale) {
    const double a = fabs(x);
    double top = a;   // NaN and infinities: found by the vote below
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    const unsigned at = __ballot_sync(0xffffffffu, a == top);
    const double m = __shfl_sync(0xffffffffu, x, at ? __ffs(at) - 1 : 0);
    const __half d = __float2half_rn(__double2float_rn(m) * -0.125f);
    const bool bad = __any_sync(0xffffffffu, !(a <= 1.7e308)) || __hisinf(d);
    scale = bad ? (uint16_t)0x7e00 : __half_as_ushort(d);
    if (bad || m == 0.0) return 8;
    const int q = (int)floor(8.5 - 8.0 * x / m);
    return q > 15 ? 15 : q < 0 ? 0 : q;
}

template <int DT, int NB>
__global__ void __launch_bounds__(32 * WARPS) k_kvq_append(AppendArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int HD = 32 * NB;
    const int lane = threadIdx.x & 31, items = a.NH + 2 * a.c.nkv;
    const long long w = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
    const int t = (int)(w / items), it = (int)(w % items);
    if (t >= a.T) return;
    const KvqPlace p = kvq_place(a.b, a.c, t, lane);
    if (!p.mine) return;
    int pos = a.positions ? a.positions[t] : (int)p.row;
    bool ok = p.row >= 0;
    if (ok && a.cos && (pos < 0 || pos >= a.n_pos)) {
        if (lane == 0) kvq_flag(a.b, TGX_KVQ_BAD_POSITION);
        ok = false;
    }
    if (it < a.NH) {
        T* dst = reinterpret_cast<T*>(a.q_out) + ((size_t)t * a.NH + it) * HD;
        float x[NB];
        if (ok) {
            const T* src = reinterpret_cast<const T*>(a.q) + (size_t)t * a.qs + (size_t)it * HD;
#pragma unroll
            for (int b = 0; b < NB; b++) x[b] = to_f32(src[32 * b + lane]);
            norm_rotate<NB>(x, a.q_norm, a.eps, a.cos, a.sin, pos, lane,
                            [](float v) { return __fdiv_rn(1.0f, __fsqrt_rn(v)); });
        } else {
#pragma unroll
            for (int b = 0; b < NB; b++) x[b] = 0.0f;
        }
#pragma unroll
        for (int b = 0; b < NB; b++) from_f32(x[b], dst[32 * b + lane]);
        return;
    }
    if (!ok) return;
    const bool is_k = it < a.NH + a.c.nkv;
    const int j = is_k ? it - a.NH : it - a.NH - a.c.nkv;
    const T* src = is_k ? reinterpret_cast<const T*>(a.k) + (size_t)t * a.ks + (size_t)j * HD
                        : reinterpret_cast<const T*>(a.v) + (size_t)t * a.vs + (size_t)j * HD;
    double x[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) x[b] = to_f32(src[32 * b + lane]);
    if (is_k)
        norm_rotate<NB>(x, a.k_norm, a.eps, a.cos, a.sin, pos, lane, [](double v) { return 1.0 / sqrt(v); });
    uint8_t* gr = kvq_granule(a.c, p.page, j, p.tok);
    const int tk = p.tok & 15, h = tk >> 3;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        uint16_t sc;
        const unsigned code = quant_block(x[b], sc);
        // nibbles i = 0 .. 3 of the dimensions l, l + 8, l + 16, l + 24 into lane l < 8
        unsigned v = code | __shfl_down_sync(0xffffffffu, code, 8) << 4;
        v |= __shfl_down_sync(0xffffffffu, v, 16) << 8;
        if (lane < 8) {
            const int g = is_k ? tk & 7 : lane, c = is_k ? lane >> 1 : (tk & 7) >> 1, e = is_k ? lane & 1 : tk & 1;
            uint8_t* codes = gr + (is_k ? 0 : 8 * HD);
            *reinterpret_cast<uint16_t*>(codes + (h * 32 + g * 4 + c) * (HD / 8) + b * 4 + e * 2) = (uint16_t)v;
        }
        if (lane == 0) {
            uint16_t* scales = reinterpret_cast<uint16_t*>(gr + 16 * HD);
            scales[is_k ? tk * NB + b : HD / 2 + ((h * 4 + ((tk & 7) >> 1)) * NB + b) * 2 + (tk & 1)] = sc;
        }
    }
}

template <int NB>
__global__ void __launch_bounds__(32 * WARPS) k_kvq_read(KvqCache c, KvqBatch bt, int T, float* k_out, float* v_out) {
    constexpr int HD = 32 * NB;
    const int lane = threadIdx.x & 31, items = 2 * c.nkv;
    const long long w = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
    const int t = (int)(w / items), it = (int)(w % items);
    if (t >= T) return;
    const bool is_k = it < c.nkv;
    float* out = is_k ? k_out : v_out;
    if (!out) return;
    const int j = is_k ? it : it - c.nkv;
    const KvqPlace p = kvq_place(bt, c, t, lane);
    if (!p.mine) return;
    out += ((size_t)t * c.nkv + j) * HD;
    const uint8_t* gr = kvq_granule(c, p.page, j, p.tok);
    const int tk = p.tok & 15, h = tk >> 3;
    const int g = is_k ? tk & 7 : lane & 7, cc = is_k ? (lane & 7) >> 1 : (tk & 7) >> 1, e = is_k ? lane & 1 : tk & 1;
    const uint8_t* codes = gr + (is_k ? 0 : 8 * HD) + (h * 32 + g * 4 + cc) * (HD / 8) + e * 2;
    const uint16_t* scales = reinterpret_cast<const uint16_t*>(gr + 16 * HD) +
                             (is_k ? tk * NB : HD / 2 + (h * 4 + ((tk & 7) >> 1)) * NB * 2 + (tk & 1));
#pragma unroll
    for (int b = 0; b < NB; b++) {
        float x = 0.0f;
        if (p.row >= 0) {
            const int q = (*reinterpret_cast<const uint16_t*>(codes + 4 * b) >> (4 * (lane >> 3))) & 15;
            x = __half2float(__ushort_as_half(scales[is_k ? b : 2 * b])) * (float)(q - 8);
        }
        out[32 * b + lane] = x;
    }
}

template <int DT>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t s) {
    const long long warps = (long long)a.T * (a.NH + 2 * a.c.nkv);
    const unsigned grid = (unsigned)((warps + WARPS - 1) / WARPS);
    switch (a.c.hd / 32) {
#define TG_CASE(n) case n: k_kvq_append<DT, n><<<grid, 32 * WARPS, 0, s>>>(a); break;
        TG_CASE(1) TG_CASE(2) TG_CASE(3) TG_CASE(4) TG_CASE(5) TG_CASE(6) TG_CASE(7) TG_CASE(8)
#undef TG_CASE
    }
    return cudaGetLastError();
}

}  // namespace

}  // namespace tg

extern "C" size_t tgx_kvq_page_bytes(int n_kv_heads, int head_dim, int page_tokens) {
    if (n_kv_heads <= 0 || n_kv_heads > 4096 || head_dim < 32 || head_dim > 256 || head_dim % 32 || page_tokens < 16 ||
        page_tokens > 1024 || page_tokens % 16)
        return 0;
    return (size_t)n_kv_heads * (page_tokens / 16) * tg::gran_bytes(head_dim);
}

extern "C" int tgx_kvq_append(const tgx_kvq_cache* cache, const tgx_kvq_batch* batch, int dtype, int n_tokens,
                              const void* q, long long q_stride, const void* k, long long k_stride, const void* v,
                              long long v_stride, int n_heads, const float* q_norm, const float* k_norm, float eps,
                              const float* rope_cos, const float* rope_sin, int n_pos, const int32_t* positions,
                              void* q_out, void* stream) {
    const char* fn = "tgx_kvq_append";
    int rc = tg::kvq_check(fn, cache, batch);
    if (rc != TG_OK) return rc;
    if (!k || !v || (n_heads && (!q || !q_out)) || (!rope_cos) != (!rope_sin))
        return tg::serve_fail(TG_EINVAL, fn, "null pointer");
    if (dtype < TGX_F32 || dtype > TGX_F16) return tg::serve_fail(TG_EINVAL, fn, "unknown dtype");
    if (n_tokens < 0 || n_heads < 0 || n_heads > 65536 || (rope_cos && n_pos <= 0) || !(eps >= 0.0f))
        return tg::serve_fail(TG_EINVAL, fn, "bad n_tokens, n_heads, n_pos or eps");
    const long long kvw = (long long)cache->n_kv_heads * cache->head_dim, qw = (long long)n_heads * cache->head_dim;
    if (q_stride < (n_heads ? qw : 0) || k_stride < kvw || v_stride < kvw || (q_stride | k_stride | v_stride) % 4)
        return tg::serve_fail(TG_EINVAL, fn, "strides must cover a row and be multiples of 4 elements");
    const size_t al = 4 * tg::elem_bytes(dtype);
    if (!tg::aligned(q, al) || !tg::aligned(k, al) || !tg::aligned(v, al) || !tg::aligned(q_out, al))
        return tg::serve_fail(TG_EINVAL, fn, "rows must be 4-element aligned");
    if ((long long)n_tokens * (n_heads + 2 * cache->n_kv_heads) / tg::WARPS >= 0x7fffffffll)
        return tg::serve_fail(TG_EINVAL, fn, "too many tokens for one call");
    tg::ServeDevice dev(fn, cache->pages);
    if (dev.rc != TG_OK || n_tokens == 0) return dev.rc;
    tg::AppendArgs a{tg::kvq_cache(*cache), tg::kvq_batch(*batch), n_tokens, n_heads, q, k, v, q_stride, k_stride,
                     v_stride, q_norm, k_norm, rope_cos, rope_sin, eps, n_pos, positions, q_out};
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e = dtype == TGX_F32    ? tg::launch_append<TGX_F32>(a, s)
                    : dtype == TGX_BF16 ? tg::launch_append<TGX_BF16>(a, s)
                                        : tg::launch_append<TGX_F16>(a, s);
    return e == cudaSuccess ? TG_OK : tg::serve_fail(TG_ECUDA, fn, cudaGetErrorString(e));
}

extern "C" int tgx_kvq_read(const tgx_kvq_cache* cache, const tgx_kvq_batch* batch, int n_tokens, float* k_out,
                            float* v_out, void* stream) {
    const char* fn = "tgx_kvq_read";
    int rc = tg::kvq_check(fn, cache, batch);
    if (rc != TG_OK) return rc;
    if (n_tokens < 0) return tg::serve_fail(TG_EINVAL, fn, "bad n_tokens");
    if ((long long)n_tokens * 2 * cache->n_kv_heads / tg::WARPS >= 0x7fffffffll)
        return tg::serve_fail(TG_EINVAL, fn, "too many tokens for one call");
    tg::ServeDevice dev(fn, cache->pages);
    if (dev.rc != TG_OK || n_tokens == 0) return dev.rc;
    const tg::KvqCache c = tg::kvq_cache(*cache);
    const tg::KvqBatch b = tg::kvq_batch(*batch);
    const unsigned grid = (unsigned)(((long long)n_tokens * 2 * c.nkv + tg::WARPS - 1) / tg::WARPS);
    cudaStream_t s = (cudaStream_t)stream;
    switch (c.hd / 32) {
#define TG_CASE(n) case n: tg::k_kvq_read<n><<<grid, 32 * tg::WARPS, 0, s>>>(c, b, n_tokens, k_out, v_out); break;
        TG_CASE(1) TG_CASE(2) TG_CASE(3) TG_CASE(4) TG_CASE(5) TG_CASE(6) TG_CASE(7) TG_CASE(8)
#undef TG_CASE
    }
    SERVE_LAUNCHED(fn);
    return TG_OK;
}
