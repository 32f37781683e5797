// tg_i8.cu — 8-bit integer matrix product with a scale per token and per output channel.
//
//   a = rint(127 y / max |y|), sa = max |y| / 127 per row (y = x, or RMSNorm(x) * w)
//   out[m][n] = (sum_k a[m][k] w[n][k]) * (sa[m] * sw[n]) (+ residual[m][n])
// The integer sum is exact in 32 bits for k <= 131072.
//
// The RMSNorm's own factor cancels in the codes: it only scales sa, so one pass finds max
// |y| and the sum of squares.  A code is cut at borders k + 1/2: it is first taken in fp32
// and, where that lands near a border, decided again in 64 bits, so codes are the
// definition's.
#include <cuda.h>

#include <cmath>

#include "tg_mbar.cuh"
#include "tg_serve.cuh"

namespace tg {

namespace {

struct QuantArgs {
    const void* x;
    long long xs;
    int rows, cols, kp;
    const float* norm;
    float eps;
    int8_t* codes;
    float* scales;
};

// A row's type: its elements, how many make a piece, and an element's value.  fp32 taken as a 16-bit
// type (TGX_FROM_F32) is rounded to it, unless it is finite and the rounding is not; its pieces are
// the 16-bit type's, so that both give the same sums.
template <int DT> struct Row {
    using T = typename Elem<DT & ~TGX_FROM_F32>::T;
    static constexpr int V = 16 / sizeof(T);
    __device__ __forceinline__ static float value(T x) { return to_f32(x); }
};
template <int DT> struct Rounded {
    using T = float;
    static constexpr int V = 8;
    __device__ __forceinline__ static float value(float x) {
        typename Elem<DT>::T r;
        from_f32(x, r);
        return fabsf(to_f32(r)) <= 3.4028235e38f ? to_f32(r) : x;
    }
};
template <> struct Row<TGX_BF16 | TGX_FROM_F32> : Rounded<TGX_BF16> {};
template <> struct Row<TGX_F16 | TGX_FROM_F32> : Rounded<TGX_F16> {};

// A piece of x as floats, and its norm weights: in 16-byte loads (ALL), or element by element with
// zeros behind the row.
template <int DT, bool ALL, int V>
__device__ __forceinline__ void load_piece(float (&v)[V], const typename Row<DT>::T* x, int at, int cols) {
    using T = typename Row<DT>::T;
    if constexpr (ALL) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < V; i += N) {
            const uint4 u = *reinterpret_cast<const uint4*>(x + at + i);
            const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int y = 0; y < N; y++) v[i + y] = Row<DT>::value(t[y]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = at + i < cols ? Row<DT>::value(x[at + i]) : 0.0f;
    }
}
template <bool NORM, bool ALL, int V>
__device__ __forceinline__ void load_norm(float (&w)[V], const float* norm, int at, int cols) {
    if constexpr (NORM && ALL) {
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(&w[i]) = *reinterpret_cast<const float4*>(norm + at + i);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) w[i] = NORM ? (at + i < cols ? norm[at + i] : 0.0f) : 1.0f;
    }
}

__device__ __forceinline__ float max_nan(float x, float y) {   // NaN if either is
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}

// rint(127 x w / top) in 64 bits: 127 x is exact, x w and the quotient round at 2^-53.
__device__ __noinline__ int i8_code_exact(float x, float w, double top) { return (int)rint((double)x * w * 127.0 / top); }

// The codes of a piece, packed: rint(127 y / top) for y = x (or x * w, unrounded), |y| <= top, in
// exact arithmetic.  Adding 1.5 * 2^23 rounds the fp32 quotient to a whole number, ties to even,
// and leaves it in the low byte.  That quotient is off by less than 2^-15, so only what comes
// that close to a border (2 in 10000, for a margin of 1e-4) needs the 64-bit one; so does x next to
// 0 under a w whose w * inv is beyond fp32, which leaves an infinity or NaN here.
template <int V>
__device__ __forceinline__ void i8_codes(uint32_t (&c)[V / 4], const float (&x)[V], const float (&w)[V], double top, float inv) {
    float t[V], far = 0.0f;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float r = x[i] * (w[i] * inv);
        t[i] = __fadd_rn(r, 12582912.0f);
        far = max_nan(far, fabsf(r - __fsub_rn(t[i], 12582912.0f)));
    }
    if (!(far < 0.4999f)) {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (!(fabsf(x[i] * (w[i] * inv) - __fsub_rn(t[i], 12582912.0f)) < 0.4999f))
                t[i] = __int_as_float(i8_code_exact(x[i], w[i], top));
    }
#pragma unroll
    for (int i = 0; i < V; i += 4)
        c[i / 4] = __byte_perm(__byte_perm(__float_as_uint(t[i]), __float_as_uint(t[i + 1]), 0x0040),
                               __byte_perm(__float_as_uint(t[i + 2]), __float_as_uint(t[i + 3]), 0x0040), 0x5410);
}

// G warps per row, two passes: the largest |y| and the sum of squares, then the codes.  The
// largest y = x * w has to be exact: its fp32 rounding is found first, then what the rounding
// lost, in the pieces that hold it.  The second pass reads the row again, from L1: rolled loops
// over it beat rows held in registers, whose unrolled code did not fit the instruction cache
// (8100 x 2048 bf16 behind a norm: 41 to 56 us).
//
// Bound by the instructions, 26 issue slots an element, for many rows (8100 x 2048 bf16 behind a norm: 21 us): a
// warp each and no barrier (G = 1).  For few rows, by latency: a CTA each (G = 8).
template <int DT, bool NORM, bool VEC, int G>
__global__ void __launch_bounds__(256, 4) k_i8_rows(QuantArgs a) {
    using T = typename Row<DT>::T;
    constexpr int V = Row<DT>::V, NT = 32 * G;
    static_assert(G == 1 || G == 8, "a warp or a CTA of 256 threads per row");
    __shared__ float s_hi[8], s_ss[8];
    __shared__ double s_top[8];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the product's weights may come
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int row = G == 1 ? blockIdx.x * 8 + wid : blockIdx.x, tid = G == 1 ? lane : threadIdx.x;
    if (row >= a.rows) return;
    const T* x = reinterpret_cast<const T*>(a.x) + (size_t)row * a.xs;
    const int pieces = a.kp / V;
    const int whole = VEC ? a.cols / V : 0;   // pieces that load in one go
    float hi = 0.0f, ss = 0.0f;               // hi: NaN once a value is
    uint32_t where = 0;                       // the thread's pieces whose largest is hi; bit 31: those from 31 on
    // f(values, weights, first column, its number) of every piece of the row that the thread owns
    auto each = [&](auto&& f) {
        float v[V], w[V];
        int i = 0, c = tid;
#pragma unroll 2
        for (; c < whole; c += NT, i++) {
            load_piece<DT, true>(v, x, c * V, a.cols);
            load_norm<NORM, true>(w, a.norm, c * V, a.cols);
            f(v, w, c * V, min(i, 31));
        }
#pragma unroll 1
        for (; c < pieces; c += NT, i++) {
            load_piece<DT, false>(v, x, c * V, a.cols);
            load_norm<NORM, false>(w, a.norm, c * V, a.cols);
            f(v, w, c * V, min(i, 31));
        }
    };
    each([&](const float (&v)[V], const float (&w)[V], int, int at) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            top = max_nan(top, fabsf(NORM ? __fmul_rn(v[i], w[i]) : v[i]));
            if (NORM) ss = fmaf(v[i], v[i], ss);
        }
        where = top > hi ? 1u << at : top == hi ? where | 1u << at : where;
        hi = max_nan(hi, top);
    });
    const float own = hi;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        if (NORM) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    if constexpr (G > 1) {
        if (lane == 0) s_hi[wid] = hi, s_ss[wid] = ss;
        __syncthreads();
        ss = 0.0f;
#pragma unroll
        for (int i = 0; i < G; i++) {
            hi = max_nan(hi, s_hi[i]);
            ss += s_ss[i];
        }
    }
    const bool poor = !(hi <= 3.4028235e38f);
    double top = hi;
    bool exact = false;   // codes from 64-bit quotients throughout
    if (NORM && hi > 0.0f && !poor) {
        double y = 0.0;   // the largest in 64 bits, where it may be
        exact = hi < 1e-30f;   // what such products lose is beyond fp32, too
        auto largest = [&](const float (&v)[V], const float (&w)[V]) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (exact || fabsf(__fmul_rn(v[i], w[i])) == hi) y = fmax(y, fabs((double)v[i] * w[i]));
        };
        if (exact || (own == hi && where >> 31)) {
            each([&](const float (&v)[V], const float (&w)[V], int, int) { largest(v, w); });
        } else if (own == hi) {   // few pieces, mostly one
#pragma unroll 1
            for (uint32_t left = where; left; left &= left - 1) {
                const int c = (tid + (__ffs(left) - 1) * NT) * V;
                float v[V], w[V];
                load_piece<DT, false>(v, x, c, a.cols);
                load_norm<NORM, false>(w, a.norm, c, a.cols);
                largest(v, w);
            }
        }
        __syncwarp();
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) y = fmax(y, __shfl_xor_sync(0xffffffffu, y, o));
        if constexpr (G > 1) {
            if (lane == 0) s_top[wid] = y;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < G; i++) y = fmax(y, s_top[i]);
        }
        top = y;
    }
    const float topf = __double2float_rn(top), inv = __fdiv_rn(127.0f, topf);
    const bool none = poor || !(topf <= 3.4028235e38f) || top == 0.0;
    exact |= !(inv <= 3.4028235e38f);   // 127 / top overflows for a top this small
    int8_t* out = a.codes + (size_t)row * a.kp;
    each([&](const float (&v)[V], const float (&w)[V], int at, int) {
        uint32_t c[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; i++) c[i] = 0;
        if (!none && !exact) i8_codes(c, v, w, top, inv);
        if (!none && exact)
#pragma unroll
            for (int i = 0; i < V; i++) c[i / 4] |= (uint32_t)(i8_code_exact(v[i], w[i], top) & 255) << (8 * (i % 4));
        if constexpr (V == 8)
            *reinterpret_cast<uint2*>(out + at) = make_uint2(c[0], c[1]);
        else
            *reinterpret_cast<uint32_t*>(out + at) = c[0];
    });
    if (tid == 0) {
        float s = __fdiv_rn(topf, 127.0f);
        if (NORM) s *= __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)a.cols), a.eps)));
        a.scales[row] = poor || !(topf <= 3.4028235e38f) ? __int_as_float(0x7fc00000) : s;
    }
}

// ---------------------------------------------------------------- the product
//
// tcgen05.mma kind::i8, int32 accumulators in TMEM.  The weights' rows (output channels) are
// the MMA's 128 rows and the tokens its columns, so a lane of the epilogue is a channel:
// outputs of 32 neighbouring channels leave together for any stride, sw[n] is one register,
// and few tokens cost few columns.  Operands come by TMA, K in steps of 128 bytes, 128-byte
// swizzle, into a ring of stages; rows and bytes beyond the matrices are filled with zeros.
//
// Warps 0 .. 7 are the epilogue (TMEM lanes 32 (w % 4) .., every second 16 columns), warp 8
// issues the copies, warp 9 the MMAs.  A CTA walks its tiles; with two accumulators the
// epilogue of one runs behind the MMAs of the next.  Where there are fewer tiles than SMs, K is split over the CTAs of a
// cluster: each puts its int32 sums into its own shared memory, and every CTA adds up and
// finishes every splits-th column, exactly, whatever the split.
//
// Many tokens (8100 x 5120 x 2048: 64 us, 2.6 Pop/s) are bound by the operands' way from L2: a
// stage is 48 KB for 512 cycles of MMAs, 15.6 TB/s over all SMs, 62 bytes a cycle and SM.  Pairs
// of CTAs on tiles of 256 x 256 (cta_group::2, 32 KB a stage, the second CTA passing on its full
// barriers by remote arrivals) were right but took 136 us.
//
// The first copies of weights are issued before the quantiser in front has finished.
// Every wait is bounded; where one expires the tile's outputs become NaN, copies and MMAs in
// flight are waited for (bounded) and the TMEM is freed.
struct MatArgs {
    const float* sa;
    const float* sw;
    int M, N;
    const void* res;
    long long rs;
    void* out;
    long long os;
    int tn;       // tokens per tile, a multiple of 16 up to 256
    int ksteps;   // 128-byte steps of a row
    int stages;
    int splits;   // CTAs of a cluster that share a tile
};

constexpr int TM = 128;           // channels per tile
constexpr int KB = 128;           // bytes of K per stage
constexpr int MAX_STAGES = 12;
constexpr int MAX_SPLITS = 4;     // larger clusters of one CTA per SM wait for room in a GPC: 8 took 20 us where 4 take 15
constexpr int EW = 8;             // epilogue warps
constexpr int GT = 32 * (EW + 2); // threads
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, uint64_t* mbar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            saddr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(saddr(mbar))
        : "memory");
}

template <int DT>
__global__ void __launch_bounds__(GT, 1)
    k_i8_mma(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mx, MatArgs g) {
    using T = typename Elem<DT>::T;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_free[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    __shared__ __align__(16) float s_sa[2][256];   // the tokens' scales of a tile
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    volatile int* failed = &s_failed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nt = (g.N + TM - 1) / TM, mt = (g.M + g.tn - 1) / g.tn, tiles = nt * mt;
    const int rank = (int)blockIdx.x % g.splits, first = (int)blockIdx.x / g.splits, stride = (int)gridDim.x / g.splits;
    const int k0 = (int)((long long)g.ksteps * rank / g.splits), k1 = (int)((long long)g.ksteps * (rank + 1) / g.splits);
    const int stage_bytes = TM * KB + g.tn * KB;
    uint32_t cols = 32;
    while ((int)cols < 2 * g.tn) cols *= 2;

    if (tid == 0) {
        for (int i = 0; i < g.stages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_free[i], 32 * EW);
        }
        s_failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;");
    }
    if (warp == EW + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&s_tmem)), "r"(cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;

    if (warp == EW) {
        if (lane == 0) {
            // x is the quantiser's: only weights may be fetched before it has finished
            const int steps = k1 - k0, n_mine = first < tiles ? (tiles - first + stride - 1) / stride : 0;
            const int ahead = min(g.stages, n_mine * steps);
            for (int f = 0, k = 0, tile = first; f < ahead; f++) {
                mbar_expect(&full[f], stage_bytes);
                tma_load(sm + f * stage_bytes, &mw, (k0 + k) * KB, tile % nt * TM, &full[f]);
                if (++k == steps) k = 0, tile += stride;
            }
            asm volatile("griddepcontrol.wait;" ::: "memory");
            // one thread feeds the ring: stage and phase are counted, not divided out
            int issued = 0, s = 0;
            uint32_t phase = 1;   // of `empty`: a fresh barrier's wait for it passes
            bool ok = true;
            for (int tile = first; tile < tiles && ok; tile += stride) {
                const int y = tile % nt * TM, my = tile / nt * g.tn;
                for (int k = k0; k < k1; k++) {
                    uint8_t* at = sm + s * stage_bytes;
                    if (issued >= ahead) {
                        ok = mbar_wait(&empty[s], phase, failed);
                        if (!ok) break;
                        mbar_expect(&full[s], stage_bytes);
                        tma_load(at, &mw, k * KB, y, &full[s]);
                    }
                    tma_load(at + TM * KB, &mx, k * KB, my, &full[s]);
                    issued++;
                    if (++s == g.stages) s = 0, phase ^= 1;
                }
            }
            if (*failed || !ok)   // everything that is under way lands before the CTA ends
                for (int i = max(0, issued - g.stages); i < issued; i++) mbar_drain(&full[i % g.stages], (i / g.stages) & 1);
        }
    } else if (warp == EW + 1) {
        {
            // D int32, A and B signed, K-major, N = tn, M = 128
            const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(g.tn >> 3) << 17) | ((TM >> 4) << 24);
            int f = 0, i = 0, s = 0;
            uint32_t phase = 0;
            const uint64_t da0 = sw128_desc(saddr(sm)), db0 = sw128_desc(saddr(sm + TM * KB));
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            bool ok = true;   // the warp is in step throughout; one lane issues
            for (int tile = first; tile < tiles && ok; tile += stride, i++) {
                if (i >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&acc_free[i & 1], ((i >> 1) - 1) & 1, failed));
                const uint32_t d = tm + (i & 1) * (cols / 2);
                uint32_t add = 0;   // the tile's first product overwrites
                for (int k = k0; k < k1 && ok; k++, f++) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&full[s], phase, failed));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t at = (uint64_t)(uint32_t)(s * (stage_bytes >> 4));
                    const uint64_t da = da0 + at, db = db0 + at;
                    if (elect_one()) {
#pragma unroll
                        for (int x = 0; x < KB / 32; x++)
                            asm volatile(
                                "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                                "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                                "l"(da + 2 * x), "l"(db + 2 * x), "r"(idesc), "r"(x ? 1u : add));
                        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                                         saddr(&empty[s]))
                                     : "memory");
                    }
                    __syncwarp();
                    add = 1;
                    if (++s == g.stages) s = 0, phase ^= 1;
                }
                if (ok && elect_one())
                    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                                     saddr(&acc_full[i & 1]))
                                 : "memory");
            }
            if (!ok)   // the last stages' MMAs
                for (int x = max(0, f - g.stages); x < f; x++) mbar_drain(&empty[x % g.stages], (x / g.stages) & 1);
        }
    } else {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const int quad = warp & 3, side = warp >> 2;
        int i = 0;
        for (int tile = first; tile < tiles; tile += stride, i++) {
            const int m0 = tile / nt * g.tn, n = tile % nt * TM + 32 * quad + lane;
            const bool n_ok = n < g.N;
            const float sw = n_ok ? g.sw[n] : 0.0f;
            float* sa = s_sa[i & 1];   // the other one may still be read
            if (tid < g.tn) sa[tid] = m0 + tid < g.M ? g.sa[m0 + tid] : 0.0f;
            asm volatile("bar.sync 1, %0;" ::"n"(32 * EW) : "memory");
            const bool ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[i & 1], (i >> 1) & 1, failed));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t d = tmem + (i & 1) * (cols / 2) + ((uint32_t)(32 * quad) << 16);
            if (g.splits > 1) {
                // own sums to shared memory (its stages are no longer in use), [column][channel]
                int* part = reinterpret_cast<int*>(sm);
                for (int c = 16 * side; c < g.tn && ok; c += 32) {
                    uint32_t v[16];
                    tmem_ld<16>(v, d + c);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int x = 0; x < 16; x++) part[(c + x) * TM + 32 * quad + lane] = (int)v[x];
                }
                break;   // one tile per cluster
            }
            T* out = reinterpret_cast<T*>(g.out) + (size_t)(m0 + 16 * side) * g.os + n;
            if (!g.res && ok && m0 + g.tn <= g.M && tile % nt * TM + TM <= g.N) {   // nothing to ask per output
                for (int c = 16 * side; c < g.tn; c += 32) {
                    uint32_t v[16];
                    tmem_ld<16>(v, d + c);
                    float s[16];
#pragma unroll
                    for (int x = 0; x < 16; x += 4) *reinterpret_cast<float4*>(&s[x]) = *reinterpret_cast<const float4*>(sa + c + x);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    T* to = out;
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        from_f32((float)(int)v[x] * (s[x] * sw), *to);
                        to += g.os;
                    }
                    out += 32 * g.os;
                }
            } else {
                const T* res = g.res ? reinterpret_cast<const T*>(g.res) + (size_t)(m0 + 16 * side) * g.rs + n : nullptr;
                for (int c = 16 * side; c < g.tn && m0 + c < g.M; c += 32) {
                    uint32_t v[16];
                    tmem_ld<16>(v, d + c);
                    const int left = n_ok ? g.M - m0 - c : 0;   // columns with an output
                    float r[16], s[16];
#pragma unroll
                    for (int x = 0; x < 16; x++) r[x] = res && x < left ? to_f32(res[x * g.rs]) : 0.0f;
#pragma unroll
                    for (int x = 0; x < 16; x += 4) *reinterpret_cast<float4*>(&s[x]) = *reinterpret_cast<const float4*>(sa + c + x);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    T* to = out;
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        float o = (float)(int)v[x] * (s[x] * sw);
                        if (res) o += r[x];
                        if (!ok) o = __int_as_float(0x7fc00000);
                        if (x < left) from_f32(o, *to);
                        to += g.os;
                    }
                    out += 32 * g.os;
                    if (res) res += 32 * g.rs;
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            mbar_arrive(&acc_free[i & 1]);
        }
    }
    __syncwarp();
    if (g.splits > 1) {   // every CTA's sums are in shared memory
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (warp < EW && first < tiles) {
            const int m0 = first / nt * g.tn, quad = warp & 3, row = 32 * quad + lane, n = first % nt * TM + row;
            const float sw = n < g.N ? g.sw[n] : 0.0f;
            uint32_t peer[MAX_SPLITS], bad = 0;
#pragma unroll
            for (int r = 0; r < MAX_SPLITS; r++) {
                const int p = r < g.splits ? r : 0;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer[r]) : "r"(saddr(sm) + row * 4), "r"(p));
            }
            {
                uint32_t at;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(saddr(&s_failed)), "r"(lane % g.splits));
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(bad) : "r"(at) : "memory");
                bad = __any_sync(0xffffffffu, bad != 0);
            }
            T* out = reinterpret_cast<T*>(g.out) + (size_t)m0 * g.os + n;
            const T* res = g.res ? reinterpret_cast<const T*>(g.res) + (size_t)m0 * g.rs + n : nullptr;
            const int end = min(g.tn, g.M - m0);
#pragma unroll 2
            for (int c = rank + g.splits * (warp >> 2); c < end; c += 2 * g.splits) {
                uint32_t v[MAX_SPLITS];
#pragma unroll
                for (int r = 0; r < MAX_SPLITS; r++) {
                    v[r] = 0;
                    if (r < g.splits)
                        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v[r]) : "r"(peer[r] + c * TM * 4) : "memory");
                }
                const float q = res && n < g.N ? to_f32(res[(size_t)c * g.rs]) : 0.0f;
                int acc = 0;
#pragma unroll
                for (int r = 0; r < MAX_SPLITS; r++) acc += (int)v[r];
                if (n < g.N) {
                    float o = (float)acc * (s_sa[0][c] * sw);
                    if (res) o += q;
                    if (bad) o = __int_as_float(0x7fc00000);
                    from_f32(o, out[(size_t)c * g.os]);
                }
            }
        }
        // nobody leaves while its sums may still be read
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == EW + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
}

// ---------------------------------------------------------------- its launch
constexpr int SMEM_MAX = 227 * 1024 - 4096;   // beside the barriers and the scales

struct MatPlan {
    int tn, splits, stages, ctas;
};

// The tile's tokens and the split of K, by an estimate in SM cycles: a K step of 128 bytes
// takes the MMAs' 2 per token (128 at least: the weights' tile is read through shared memory)
// or its bytes' way at about 32 bytes a cycle and SM, whichever is longer; a tile's last
// columns leave at about 8 a token, and a split adds its exchange.
MatPlan plan_mat(int M, int N, int kp, int sms) {
    const int nt = (N + TM - 1) / TM, kt = (kp + KB - 1) / KB;
    MatPlan best{};
    double best_cost = 1e300;
    for (int tn = 16; tn <= 256; tn += 16) {
        if (tn > 16 && tn - 16 >= M) break;   // wider than the tokens
        const long long tiles = (long long)nt * ((M + tn - 1) / tn);
        const double step = fmax(fmax(2.0 * tn, 128.0), (TM * KB + tn * KB) / 32.0);
        for (int s = 1; s <= MAX_SPLITS && s <= kt; s++) {
            if (s > 1 && (tiles * s > sms || tn * TM * 4 > SMEM_MAX - 1024)) break;
            const long long waves = (tiles * s + sms - 1) / sms;
            const double cost = (double)waves * ((kt + s - 1) / s) * step + 8.0 * tn + (s > 1 ? 1500.0 + 4.0 * tn : 0.0);
            if (cost < best_cost) {
                best_cost = cost;
                const long long ctas = tiles * s < sms ? tiles * s : sms;
                best = MatPlan{tn, s, 0, (int)ctas};
            }
        }
    }
    const int stage = TM * KB + best.tn * KB;
    best.stages = (SMEM_MAX - 1024) / stage;
    if (best.stages > MAX_STAGES) best.stages = MAX_STAGES;
    return best;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeTiled)p;
    }();
    return fn;
}

// int8 rows of kp bytes, copied in boxes of 128 bytes by `box` rows.
bool row_map(CUtensorMap* m, const void* base, int rows, int kp, int box) {
    const cuuint64_t dims[2] = {(cuuint64_t)kp, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)kp};
    const cuuint32_t boxes[2] = {KB, (cuuint32_t)box}, ones[2] = {1, 1};
    return encode_tiled()(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 0;
    return sms;
}

template <int DT>
cudaError_t launch_mat(MatArgs g, const int8_t* x, const int8_t* w, int kp, cudaStream_t s) {
    const int sms = sm_count();
    if (!sms || !encode_tiled()) return cudaErrorNotSupported;
    const MatPlan p = plan_mat(g.M, g.N, kp, sms);
    g.tn = p.tn;
    g.splits = p.splits;
    g.stages = p.stages;
    g.ksteps = (kp + KB - 1) / KB;
    CUtensorMap mw, mx;
    if (!row_map(&mw, w, g.N, kp, TM) || !row_map(&mx, x, g.M, kp, p.tn)) return cudaErrorInvalidValue;
    const int ring = p.stages * (TM * KB + p.tn * KB), part = p.splits > 1 ? p.tn * TM * 4 : 0;
    const int smem = (ring > part ? ring : part) + 1024;
    // the same limit in every call: it is the kernel's, shared with other threads' calls of other sizes
    cudaError_t e = cudaFuncSetAttribute(k_i8_mma<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.ctas);
    cfg.blockDim = dim3(GT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, k_i8_mma<DT>, mw, mx, g);
}

template <int DT>
cudaError_t launch_rows(const QuantArgs& a, cudaStream_t s) {
    constexpr int E = sizeof(typename Row<DT>::T);
    const bool vec = ((uintptr_t)a.x | (uintptr_t)(a.xs * E) | (uintptr_t)a.norm) % 16 == 0;
    // a warp per row once that fills the device (148 SMs of 24 such warps) and rows are no longer
    // than a few thousand: 8100 x 2048 bf16 took 41 us a CTA each
    if (a.rows >= 2048 && a.kp <= 8192) {
        const int grid = (a.rows + 7) / 8;
        if (a.norm)
            vec ? k_i8_rows<DT, true, true, 1><<<grid, 256, 0, s>>>(a) : k_i8_rows<DT, true, false, 1><<<grid, 256, 0, s>>>(a);
        else
            vec ? k_i8_rows<DT, false, true, 1><<<grid, 256, 0, s>>>(a) : k_i8_rows<DT, false, false, 1><<<grid, 256, 0, s>>>(a);
    } else if (a.norm) {
        vec ? k_i8_rows<DT, true, true, 8><<<a.rows, 256, 0, s>>>(a) : k_i8_rows<DT, true, false, 8><<<a.rows, 256, 0, s>>>(a);
    } else {
        vec ? k_i8_rows<DT, false, true, 8><<<a.rows, 256, 0, s>>>(a) : k_i8_rows<DT, false, false, 8><<<a.rows, 256, 0, s>>>(a);
    }
    return cudaGetLastError();
}

cudaError_t launch_rows(int dtype, const QuantArgs& a, cudaStream_t s) {
    switch (dtype) {
        case TGX_F32: return launch_rows<TGX_F32>(a, s);
        case TGX_BF16: return launch_rows<TGX_BF16>(a, s);
        case TGX_F16: return launch_rows<TGX_F16>(a, s);
        case TGX_BF16 | TGX_FROM_F32: return launch_rows<TGX_BF16 | TGX_FROM_F32>(a, s);
        default: return launch_rows<TGX_F16 | TGX_FROM_F32>(a, s);
    }
}

// Whether the rows may be of that type, and the bytes of an element.
bool row_type(int dtype) {
    return (dtype >= TGX_F32 && dtype <= TGX_F16) || dtype == (TGX_BF16 | TGX_FROM_F32) || dtype == (TGX_F16 | TGX_FROM_F32);
}
int row_elem(int dtype) { return dtype & TGX_FROM_F32 ? 4 : elem_bytes(dtype); }

size_t r256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

}  // namespace tg

extern "C" size_t tgx_i8_row_bytes(int cols) { return cols > 0 && cols <= 131072 ? ((size_t)cols + 15) & ~(size_t)15 : 0; }

extern "C" int tgx_i8_quantize_rows(int dtype, const void* x, long long x_stride, int rows, int cols,
                                    const float* norm_w, float eps, int8_t* codes, float* scales, void* stream) {
    const char* fn = "tgx_i8_quantize_rows";
    if (!x || !codes || !scales) return tg::serve_fail(TG_EINVAL, fn, "null pointer");
    if (!tg::row_type(dtype)) return tg::serve_fail(TG_EINVAL, fn, "unknown dtype");
    if (rows < 0 || !tgx_i8_row_bytes(cols) || x_stride < cols || !(eps >= 0.0f))
        return tg::serve_fail(TG_EINVAL, fn, "bad rows, cols (1 .. 131072), stride or eps");
    if (!tg::aligned(codes, 16) || !tg::aligned(x, tg::row_elem(dtype)))
        return tg::serve_fail(TG_EINVAL, fn, "codes must be 16-byte aligned, x to its elements");
    tg::ServeDevice dev(fn, x);
    if (dev.rc != TG_OK || rows == 0) return dev.rc;
    tg::QuantArgs a{x, x_stride, rows, cols, (int)tgx_i8_row_bytes(cols), norm_w, eps, codes, scales};
    cudaError_t e = tg::launch_rows(dtype, a, (cudaStream_t)stream);
    return e == cudaSuccess ? TG_OK : tg::serve_fail(TG_ECUDA, fn, cudaGetErrorString(e));
}

extern "C" size_t tgx_i8_matmul_scratch_bytes(int m, int n, int k) {
    if (m < 0 || n <= 0 || !tgx_i8_row_bytes(k)) return 0;
    return tg::r256((size_t)m * tgx_i8_row_bytes(k)) + tg::r256((size_t)m * 4) + 256;
}

extern "C" int tgx_i8_matmul(int dtype, const void* x, long long x_stride, int m, int k, const float* norm_w, float eps,
                             const int8_t* w_codes, const float* w_scales, int n, const void* residual,
                             long long res_stride, void* out, long long out_stride, void* scratch, size_t scratch_bytes,
                             void* stream) {
    const char* fn = "tgx_i8_matmul";
    if (!x || !w_codes || !w_scales || !out || !scratch) return tg::serve_fail(TG_EINVAL, fn, "null pointer");
    if (!tg::row_type(dtype)) return tg::serve_fail(TG_EINVAL, fn, "unknown dtype");
    if (m < 0 || n <= 0 || !tgx_i8_row_bytes(k) || x_stride < k || out_stride < n || (residual && res_stride < n) ||
        !(eps >= 0.0f))
        return tg::serve_fail(TG_EINVAL, fn, "bad m, n, k (1 .. 131072), stride or eps");
    const int type = dtype & ~TGX_FROM_F32;   // of out and residual
    const size_t e1 = tg::elem_bytes(type);
    if (!tg::aligned(w_codes, 16) || !tg::aligned(x, tg::row_elem(dtype)) || !tg::aligned(out, e1) || !tg::aligned(residual, e1))
        return tg::serve_fail(TG_EINVAL, fn, "w_codes must be 16-byte aligned, x, residual and out to their elements");
    if (!tg::aligned(scratch, 256) || scratch_bytes < tgx_i8_matmul_scratch_bytes(m, n, k))
        return tg::serve_fail(TG_EINVAL, fn, "scratch must be 256-byte aligned, of tgx_i8_matmul_scratch_bytes");
    tg::ServeDevice dev(fn, x);
    if (dev.rc != TG_OK || m == 0) return dev.rc;
    cudaStream_t s = (cudaStream_t)stream;
    const int kp = (int)tgx_i8_row_bytes(k);
    int8_t* codes = (int8_t*)scratch;
    float* scales = (float*)((uint8_t*)scratch + tg::r256((size_t)m * kp));
    tg::QuantArgs qa{x, x_stride, m, k, kp, norm_w, eps, codes, scales};
    cudaError_t e = tg::launch_rows(dtype, qa, s);
    if (e != cudaSuccess) return tg::serve_fail(TG_ECUDA, fn, cudaGetErrorString(e));
    tg::MatArgs g{scales, w_scales, m, n, residual, res_stride, out, out_stride, 0, 0, 0, 0};
    e = type == TGX_F32    ? tg::launch_mat<TGX_F32>(g, codes, w_codes, kp, s)
        : type == TGX_BF16 ? tg::launch_mat<TGX_BF16>(g, codes, w_codes, kp, s)
                           : tg::launch_mat<TGX_F16>(g, codes, w_codes, kp, s);
    return e == cudaSuccess ? TG_OK : tg::serve_fail(TG_ECUDA, fn, cudaGetErrorString(e));
}
