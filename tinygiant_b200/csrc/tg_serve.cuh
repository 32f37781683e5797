// tg_serve.cuh — what the batched serving operators share: element types, the paged
// cache's layout and a token's place in it, argument checks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/tinygiant.h"
#include "tg_internal.h"

namespace tg {

// ---------------------------------------------------------------- element types
template <int DT> struct Elem;
template <> struct Elem<TGX_F32> { using T = float; };
template <> struct Elem<TGX_BF16> { using T = __nv_bfloat16; };
template <> struct Elem<TGX_F16> { using T = __half; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f32(float x, float& o) { o = x; }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16& o) { o = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_f32(float x, __half& o) { o = __float2half_rn(x); }

inline int elem_bytes(int dtype) { return dtype == TGX_F32 ? 4 : 2; }

// ---------------------------------------------------------------- the paged cache
// A granule is 16 tokens of one kv head: 18 * HD bytes (include/tinygiant.h).
struct KvqCache {
    uint8_t* pages;
    int n_pages, pt, nkv, hd;
    size_t page_bytes;
};
struct KvqBatch {
    int B, max_pages, max_new;
    const int32_t* q_start;
    const int32_t* kv_lens;
    const int32_t* table;
    int32_t* status;
};

__device__ __forceinline__ void kvq_flag(const KvqBatch& b, int bit) {
    if (b.status) atomicOr(b.status, bit);
}

__host__ __device__ inline int gran_bytes(int hd) { return 18 * hd; }

// Granule of token `tok` (in its page) of kv head j of page `page`.
__device__ __forceinline__ uint8_t* kvq_granule(const KvqCache& c, int page, int j, int tok) {
    return c.pages + (size_t)page * c.page_bytes + (size_t)(j * (c.pt >> 4) + (tok >> 4)) * gran_bytes(c.hd);
}

// The sequence of token t: the last b with q_start[b] <= t, found by the whole warp, 32
// probes a step.  Any contents of q_start give some b in [0, B).
__device__ __forceinline__ int kvq_find_seq(const KvqBatch& b, int t, int lane) {
    int lo = 0, hi = b.B;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) >> 5, i = lo + lane * step;
        const unsigned le = __ballot_sync(0xffffffffu, i < hi && (lane == 0 || b.q_start[i] <= t));
        lo += (31 - __clz(le)) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

struct KvqPlace {
    int seq;
    long long row;   // cache row, or -1 where the token has none
    int page, tok;
    bool mine;       // the token belongs to a sequence
};

// Token t's row and page, by the whole warp.  `flag` reports what does not fit.
__device__ __forceinline__ KvqPlace kvq_place(const KvqBatch& b, const KvqCache& c, int t, int lane) {
    KvqPlace p{0, -1, 0, 0, false};
    p.seq = kvq_find_seq(b, t, lane);
    const int s0 = b.q_start[p.seq], s1 = b.q_start[p.seq + 1];
    if (t < s0 || t >= s1) return p;
    p.mine = true;
    const long long row = (long long)b.kv_lens[p.seq] - (s1 - t);
    if (row < 0 || row >= (long long)b.max_pages * c.pt) {
        if (lane == 0) kvq_flag(b, TGX_KVQ_BAD_LENGTH);
        return p;
    }
    const int r = (int)row, at = r / c.pt;   // max_pages * pt fits 32 bits
    p.page = b.table[(size_t)p.seq * b.max_pages + at];
    p.tok = r - at * c.pt;
    if (p.page < 0 || p.page >= c.n_pages) {
        if (lane == 0) kvq_flag(b, TGX_KVQ_BAD_PAGE);
        return p;
    }
    p.row = row;
    return p;
}

// ---------------------------------------------------------------- host side
inline KvqCache kvq_cache(const tgx_kvq_cache& c) {
    return KvqCache{(uint8_t*)c.pages, c.n_pages, c.page_tokens, c.n_kv_heads, c.head_dim,
                    tgx_kvq_page_bytes(c.n_kv_heads, c.head_dim, c.page_tokens)};
}
inline KvqBatch kvq_batch(const tgx_kvq_batch& b) {
    return KvqBatch{b.n_seqs, b.max_pages, b.max_new, b.q_start, b.kv_lens, b.page_table, b.status};
}

inline int serve_fail(int code, const char* fn, const std::string& msg) {
    return set_error(code, (std::string(fn) + ": " + msg).c_str());
}

inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// The shared checks of the cache and the batch: TG_OK or the error, reported.
inline int kvq_check(const char* fn, const tgx_kvq_cache* c, const tgx_kvq_batch* b) {
    if (!c || !b || !c->pages || !b->q_start || !b->kv_lens || !b->page_table)
        return serve_fail(TG_EINVAL, fn, "null pointer");
    if (!tgx_kvq_page_bytes(c->n_kv_heads, c->head_dim, c->page_tokens) || c->n_pages <= 0)
        return serve_fail(TG_EINVAL, fn,
                          "bad cache (n_pages, n_kv_heads > 0; head_dim a multiple of 32 up to 256; page_tokens a "
                          "multiple of 16 up to 1024)");
    if (!aligned(c->pages, 16)) return serve_fail(TG_EINVAL, fn, "pages must be 16-byte aligned");
    if (b->n_seqs <= 0 || b->max_pages <= 0 || b->max_new <= 0)
        return serve_fail(TG_EINVAL, fn, "n_seqs, max_pages and max_new must be positive");
    if ((long long)b->max_pages * c->page_tokens > 0x7fffffffll - 65536)
        return serve_fail(TG_EINVAL, fn, "max_pages * page_tokens is beyond 32 bits");
    return TG_OK;
}

// Makes the device that holds `p` current for the call: kernels run where the data is,
// whatever device the caller has selected.
struct ServeDevice {
    int prev = -1, rc = TG_OK;
    ServeDevice(const char* fn, const void* p) {
        cudaPointerAttributes at{};
        if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
            cudaGetLastError();
            int n = 0;
            if (cudaGetDeviceCount(&n) != cudaSuccess || n <= 0) {
                cudaGetLastError();
                rc = serve_fail(TG_ENODEV, fn, "no CUDA device");
            } else {
                rc = serve_fail(TG_EINVAL, fn, "not device memory");
            }
            return;
        }
        if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) {
            rc = serve_fail(TG_EINVAL, fn, "not device memory");
            return;
        }
        int cur = -1;
        if (cudaGetDevice(&cur) == cudaSuccess && cur != at.device && cudaSetDevice(at.device) == cudaSuccess) prev = cur;
    }
    ~ServeDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

#define SERVE_LAUNCHED(fn)                                                                        \
    do {                                                                                          \
        cudaError_t e_ = cudaGetLastError();                                                      \
        if (e_ != cudaSuccess) return tg::serve_fail(TG_ECUDA, fn, cudaGetErrorString(e_));       \
    } while (0)

}  // namespace tg
