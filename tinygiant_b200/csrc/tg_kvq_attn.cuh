// tg_kvq_attn.cuh — what the two attention kernels over the 4-bit cache share: their
// arguments, a sequence's share of a call, codes as fp16.
#pragma once
#include "tg_serve.cuh"

namespace tg {

struct AttnKvqArgs {
    KvqCache c;
    KvqBatch b;
    int T, NH, R;       // R = NH / nkv
    const void* q;
    long long qs;
    void* out;
    long long os;
    float scale;        // times log2(e)
    uint32_t k1024;     // fp16 1024 twice
    int workers;
    float* slots;       // [workers][2] partial results: m, l [rows], O [rows][HD]
    int* heads;         // [workers][2][4] what a slot holds: kind, token row base, kv head, query rows
    const int* only;    // [B][nkv] or null: sequences without a nonzero word are left out
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

// Two codes of the lower (bits 0 .. 3 of each halfword) or the upper nibbles (4 .. 7) as
// fp16: code - 8, or, RAW, code * 2^-24 and code * 2^-20.
// `k1024` is 1024 twice, in a register: one three-input operation then masks and merges.
template <bool RAW>
__device__ __forceinline__ uint32_t codes_lo(uint32_t x, uint32_t k1024) {
    if constexpr (RAW) return x & 0x000f000fu;
    uint32_t y;
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(y) : "r"(x), "r"(k1024));
    return as_u32(__hadd2(as_h2(y), __float2half2_rn(-1032.0f)));
}
template <bool RAW>
__device__ __forceinline__ uint32_t codes_hi(uint32_t x, uint32_t k1024) {
    if constexpr (RAW) return x & 0x00f000f0u;
    uint32_t y;
    asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xEA;" : "=r"(y) : "r"(x), "r"(k1024));
    return as_u32(__hfma2(as_h2(y), __float2half2_rn(0.0625f), __float2half2_rn(-72.0f)));
}

// 2^score is taken as fma(raw score, fac, offset - fac * reference) while the reference is small, and
// from the difference of the raw scores where it is so large that fp32 would round the exponent away.
constexpr float FAR = 65536.0f;
// A row's factor from raw scores to exponents, kept where products with it are neither 0 nor infinite for
// sums of at most 2^33: beyond these bounds scores are all alike, or one is all there is.
__device__ __forceinline__ float bounded_fac(float x) { return fminf(fmaxf(x, 0x1p-120f), 0x1p120f); }

constexpr uint32_t NO_GRANULE = 0xffffffffu;

// N words, in the widest loads that their alignment allows.
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4*>(&w[i]) = *reinterpret_cast<const uint4*>(p + 4 * i);
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) *reinterpret_cast<uint2*>(&w[i]) = *reinterpret_cast<const uint2*>(p + 4 * i);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
    }
}
// N fp16 scales as floats.
template <int N>
__device__ __forceinline__ void load_scales(float (&d)[N], const uint8_t* p) {
    if constexpr (N % 2 == 0) {
        uint32_t w[N / 2];
        load_words<N / 2>(w, p);
#pragma unroll
        for (int i = 0; i < N; i++) d[i] = i & 1 ? __high2float(as_h2(w[i / 2])) : __low2float(as_h2(w[i / 2]));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) d[i] = __half2float(*reinterpret_cast<const __half*>(p + 2 * i));
    }
}
__device__ __forceinline__ float2 load2(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 load2(const __nv_bfloat16* p) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
}
__device__ __forceinline__ float2 load2(const __half* p) { return __half22float2(*reinterpret_cast<const __half2*>(p)); }

// A sequence's share of the call.
struct SeqInfo {
    int s0, n;          // first new token, how many are attended for
    long long len;      // cached rows within the table
    int off;            // new token i sees the rows below off + i + 1 (may be negative)
    int tiles, grans;   // row tiles per kv head; units per tile (at least one)
};

__device__ __forceinline__ long long quotient(long long x, long long y) {
    if ((x | y) < 0x100000000ll) return (uint32_t)x / (uint32_t)y;
    return x / y;
}

__device__ __forceinline__ SeqInfo seq_info(const AttnKvqArgs& a, int b, int tile_rows) {
    SeqInfo s;
    const int s0 = a.b.q_start[b], s1 = a.b.q_start[b + 1];
    s.s0 = s0;
    s.n = s0 >= 0 && s1 > s0 && s1 <= a.T ? s1 - s0 : 0;
    const long long cap = (long long)a.b.max_pages * a.c.pt, len = a.b.kv_lens[b];
    const long long off = len - s.n;
    s.off = (int)(off < -(1ll << 30) ? -(1ll << 30) : off);
    s.len = len < 0 ? 0 : len > cap ? cap : len;
    s.n = min(s.n, a.b.max_new);
    if (a.only) {
        int any = 0;
        for (int j = 0; j < a.c.nkv; j++) any |= a.only[(size_t)b * a.c.nkv + j];
        if (!any) s.n = 0;
    }
    s.tiles = (int)(((long long)s.n * a.R + tile_rows - 1) / tile_rows);
    s.grans = max(1, (int)((s.len + 15) >> 4));
    return s;
}

// The 256-row tiles of tg_kvq_tc.cu: whether they take the call, their scratch, and the launch
// (which leaves sequences with a scale that is not finite, marked in its scratch, to the other
// kernel: *only then points at the marks).
bool attn_tc_takes(int dtype, const KvqCache& c, const KvqBatch& b, int T, int R);
size_t attn_tc_scratch(const KvqCache& c, const KvqBatch& b, int T, int R);
cudaError_t launch_attn_tc(int dtype, const AttnKvqArgs& a, void* scratch, const int** only, cudaStream_t s);

}  // namespace tg
