// tg_kvq_attn.cu — attention of many tokens over the paged 4-bit key/value cache.
//
//   s_r = scale * q . k_r over the rows r up to the token's own, p = softmax(s),
//   out = sum_r p_r v_r
// in one pass over the rows: a running reference m (the maximum, or within 2^4 of it), the
// sum l of exp2(s - m) and the output, rescaled when the scores leave m's range.
//
// Both products run on the tensor cores with the codes as the other operand, mma m16n8k16:
//   K: rows 16 cached tokens, columns 8 query rows (heads of the kv head x new tokens), k 16
//      dimensions; a block's sum enters the score times the block's scale, in fp32.
//   V: rows 16 dimensions, columns the query rows, k 16 tokens; a block's scale goes into the
//      probability, p * d, per block.
// fp32 inputs keep 22 bits of q and of p * d as two fp16 pieces, each an mma of its own; for
// 16-bit types one piece (11 bits) is as fine as the output.  The pieces stay in fp16's range
// by powers of two: q's rows are scaled to 2^13 .. 2^14, p to 2^6 at its maximum, V scales to
// 2^2 .. 2^5 at the largest met so far (vexp; O is rescaled when a larger one comes).
//
// Codes become fp16 by masks.  For 16-bit types a nibble masked into the low byte of a
// halfword IS the number code * 2^-24 (a subnormal; 2^-20 for the nibble above it): eight
// codes cost four ANDs and a shift.  The upper nibbles' factor 16 is taken off q, and off the
// output; the codes' offset of 8 is -8 sum q in the scores' first accumulator and, for V, one
// more mma per block whose other operand is -8 * 2^-24 throughout.  The tensor cores align
// products by exponent fields, which subnormals leave 2^6 .. 2^10 above their values, so sums
// are good to about 2^-17: below 16-bit outputs, too coarse for fp32.  There the nibbles go
// into the low bits of 1024 and one half-precision operation more makes them code - 8.
//
// Work: an item is (sequence, kv head, tile of 8 * NT query rows), its units the granules
// of 16 tokens (18 * HD contiguous bytes).  All items' units in one line are cut into equal
// parts, one per worker (a CTA of W warps), whatever the lengths: a worker walks the items of
// its part.  Each of its warps takes every W-th granule, through a ring of its own that
// cp.async keeps STAGES deep, and the W results meet in shared memory.  An item that lies in
// one part is finished there; the others' parts go to scratch and k_kvq_join adds them in
// order, so results repeat exactly.
//
// Bound by memory for few query rows: a granule is 2304 bytes at HD 128, about 100 cycles of
// an SM's share of the bandwidth, against 40 to 80 of its tensor cores.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "tg_serve.cuh"

namespace tg {

namespace {

constexpr int DEEP_WARPS = 4;         // warps of a worker that share an item
constexpr float P_EXP = 6.0f;        // p is held times 2^P_EXP
constexpr float P_SLACK = 4.0f;      // and may exceed that by 2^P_SLACK before m moves
constexpr int V_LOW = 2, V_HIGH = 5; // V scales are held in 2^V_LOW .. 2^V_HIGH at the largest: 2^(6 + 4 + 5) < 65504

struct AttnKvqArgs {
    KvqCache c;
    KvqBatch b;
    int T, NH, R;       // R = NH / nkv
    const void* q;
    long long qs;
    void* out;
    long long os;
    float scale;        // times log2(e)
    int workers;
    float* slots;       // [workers][2] partial results: m, l [rows], O [rows][HD]
    int* heads;         // [workers][2][4] what a slot holds: kind, token row base, kv head, query rows
};

// Slot kinds: nothing; a part that its item goes on behind; the item's last part.
enum { SLOT_NONE = 0, SLOT_MORE = 1, SLOT_LAST = 2 };

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {   // an 8 x 8 tile of halves across the warp
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

// Two codes of the lower (bits 0 .. 3 of each halfword) or the upper nibbles (4 .. 7) as
// fp16: code - 8, or, RAW, code * 2^-24 and code * 2^-20.
template <bool RAW>
__device__ __forceinline__ uint32_t codes_lo(uint32_t x) {
    if constexpr (RAW) return x & 0x000f000fu;
    return as_u32(__hadd2(as_h2((x & 0x000f000fu) | 0x64006400u), __float2half2_rn(-1032.0f)));
}
template <bool RAW>
__device__ __forceinline__ uint32_t codes_hi(uint32_t x) {
    if constexpr (RAW) return x & 0x00f000f0u;
    return as_u32(__hfma2(as_h2((x & 0x00f000f0u) | 0x64006400u), __float2half2_rn(0.0625f), __float2half2_rn(-72.0f)));
}

// A sequence's share of the call.
struct SeqInfo {
    int s0, n;          // first new token, how many are attended for
    long long len;      // cached rows within the table
    int off;            // new token i sees the rows below off + i + 1 (may be negative)
    int tiles, grans;   // row tiles per kv head; units per tile (at least one)
};

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
    s.tiles = (int)(((long long)s.n * a.R + tile_rows - 1) / tile_rows);
    s.grans = max(1, (int)((s.len + 15) >> 4));
    return s;
}

template <int NB> constexpr int stages() { return NB <= 4 ? 4 : 3; }

// Shared memory of a CTA of W warps: the rings, which the joining of the warps reuses.
template <int NB, int NT>
constexpr int attn_smem(int W) {
    const int ring = W * stages<NB>() * 18 * 32 * NB, join = W * 8 * NT * (32 * NB + 4) * 4;
    return ring > join ? ring : join;
}

template <int DT, int NB, int NT>
__global__ void __launch_bounds__(32 * DEEP_WARPS) k_kvq_attn(AttnKvqArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int HD = 32 * NB, GB = 18 * HD, ST = stages<NB>(), KS = 2 * NB, ROWS = 8 * NT;
    constexpr int PC = DT == TGX_F32 ? 2 : 1;    // fp16 pieces of q and of p * d
    constexpr bool RAW = PC == 1;                // codes as subnormals
    constexpr int OC = RAW ? NB : 1;             // offset accumulators
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ long long s_scan[8];
    __shared__ long long s_base;
    __shared__ int s_seq;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, W = blockDim.x >> 5;
    const int g = lane >> 2, c = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- the plan: every worker adds up all sequences' units and finds where its part begins.
    // Thread t owns sequences [t * per, ...), so a prefix over the threads is one over them.
    const int per = (a.b.B + (int)blockDim.x - 1) / (int)blockDim.x;
    long long mine = 0;
    for (int i = 0; i < per; i++) {
        const int b = tid * per + i;
        if (b < a.b.B) {
            const SeqInfo s = seq_info(a, b, ROWS);
            mine += (long long)s.tiles * s.grans * a.c.nkv;
            if (blockIdx.x == 0 && (long long)a.b.kv_lens[b] > (long long)a.b.max_pages * a.c.pt)
                kvq_flag(a.b, TGX_KVQ_BAD_LENGTH);
            if (blockIdx.x == 0 && (long long)a.b.q_start[b + 1] - a.b.q_start[b] > a.b.max_new)
                kvq_flag(a.b, TGX_KVQ_BAD_NEW);
        }
    }
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[wid] = incl;
    __syncthreads();
    long long before = 0, total = 0;
    for (int i = 0; i < W; i++) {
        if (i < wid) before += s_scan[i];
        total += s_scan[i];
    }
    // at least one granule per warp of a worker: short work goes to fewer workers
    const long long used = max(1ll, min((long long)a.workers, (total + W - 1) / W));
    const long long w = blockIdx.x;
    long long u = w < used ? total * w / used : total;
    const long long u_end = w < used ? total * (w + 1) / used : total;
    if (tid < 2) {   // no slots yet
        a.heads[((size_t)w * 2 + tid) * 4] = SLOT_NONE;
    }
    if (u >= u_end) return;
    if (u >= before + incl - mine && u < before + incl) {
        long long x = before + incl - mine;
        int b = tid * per;
        for (;; b++) {
            const SeqInfo s = seq_info(a, b, ROWS);
            const long long n = (long long)s.tiles * s.grans * a.c.nkv;
            if (u < x + n) break;
            x += n;
        }
        s_seq = b;
        s_base = x;
    }
    __syncthreads();
    int b = s_seq;
    long long base = s_base;   // units in front of sequence b

    uint8_t* ring = sm + wid * ST * GB;
    while (u < u_end) {
        const SeqInfo si = seq_info(a, b, ROWS);
        const long long units = (long long)si.tiles * si.grans * a.c.nkv;
        if (u >= base + units) {
            base += units;
            b++;
            continue;
        }
        const int item = (int)((u - base) / si.grans), g0 = (int)((u - base) % si.grans);
        const int rt = item / a.c.nkv, j = item % a.c.nkv;   // kv heads innermost
        const int g1 = (int)min((long long)si.grans, g0 + (u_end - u));
        u += g1 - g0;
        const int row0 = rt * ROWS, nrows = min(ROWS, si.n * a.R - row0);   // query rows of the item

        // ---- the query rows as B operands: lane (g, c) holds row g's dimensions 16s + 2c, + 1
        // and + 8, and the rows' factors, limits and offsets for the columns 2c, 2c + 1
        uint32_t qf[NT][PC][KS][2];
        float corr[NT][NB][2], fac[NT][2];
        int lim[NT][2], lim_min = 0x7fffffff, lim_max = 0;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int r = 8 * n + g;
            const bool ok = r < nrows;
            const int rho = row0 + r;
            const T* src = reinterpret_cast<const T*>(a.q) + (size_t)(si.s0 + (ok ? rho / a.R : 0)) * a.qs +
                           (size_t)(j * a.R + (ok ? rho % a.R : 0)) * HD;
            float x[KS][4], top = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    x[s][h] = ok ? to_f32(src[16 * s + 8 * (h >> 1) + 2 * c + (h & 1)]) : 0.0f;
                    top = fmaxf(top, fabsf(x[s][h]));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^-e: top into 2^13 .. 2^14 (in two factors: e reaches beyond fp32's exponents)
            int e = top > 0.0f && top <= 3.4e38f ? ilogbf(top) - 13 : 0;
            e = max(e, -110);
            const float up1 = scalbnf(1.0f, -(e / 2)), up2 = scalbnf(1.0f, -(e - e / 2));
            float sums[NB];
#pragma unroll
            for (int i = 0; i < NB; i++) sums[i] = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float y0 = x[s][2 * h] * up1 * up2, y1 = x[s][2 * h + 1] * up1 * up2;
                    sums[s >> 1] += y0 + y1;
                    const float m = RAW && h ? 0.0625f : 1.0f;   // the upper nibbles' codes count 16 times
                    const __half2 hi = __floats2half2_rn(y0 * m, y1 * m);
                    qf[n][0][s][h] = as_u32(hi);
                    if constexpr (PC == 2)
                        qf[n][1][s][h] =
                            as_u32(__floats2half2_rn(y0 * m - __low2float(hi), y1 * m - __high2float(hi)));
                }
            float f = a.scale * (RAW ? 0x1p24f : 1.0f);
            f = scalbnf(f, e);
            int l = (int)max(0ll, min(si.len, (long long)si.off + (ok ? rho / a.R : 0) + 1));
            if (!ok) l = 0x7fffffff;   // rows beyond the item: any scores will do
#pragma unroll
            for (int k = 0; k < 2; k++) {
                fac[n][k] = __shfl_sync(0xffffffffu, f, 4 * (2 * c + k));
                lim[n][k] = __shfl_sync(0xffffffffu, l, 4 * (2 * c + k));
            }
            lim_min = min(lim_min, l);
            lim_max = max(lim_max, ok ? l : 0);
#pragma unroll
            for (int i = 0; i < NB; i++) {
                float t = sums[i];
                t += __shfl_xor_sync(0xffffffffu, t, 1);
                t += __shfl_xor_sync(0xffffffffu, t, 2);
                t = RAW ? t * (-8.0f * 0x1p-24f) : 0.0f;
#pragma unroll
                for (int k = 0; k < 2; k++) corr[n][i][k] = __shfl_sync(0xffffffffu, t, 4 * (2 * c + k));
            }
        }
#pragma unroll
        for (int o = 16; o >= 4; o >>= 1) {
            lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, o));
            lim_max = max(lim_max, __shfl_xor_sync(0xffffffffu, lim_max, o));
        }

        // ---- this warp's granules: g0 + wid, + W, ... below the last visible row
        const int gl = min(g1, (lim_max + 15) >> 4);
        const int nk = gl > g0 + wid ? (gl - g0 - wid + W - 1) / W : 0;
        const int gpp = a.c.pt >> 4;
        // lane l: where granule 32 x + l of this warp lies, or -1
        auto find = [&](int x) -> long long {
            const int k = 32 * x + lane;
            if (k >= nk) return -1;
            const int gi = g0 + wid + k * W, pi = gi / gpp;
            const int page = a.b.table[(size_t)b * a.b.max_pages + pi];
            if (page < 0 || page >= a.c.n_pages) {
                kvq_flag(a.b, TGX_KVQ_BAD_PAGE);
                return -1;
            }
            return (long long)((size_t)page * a.c.page_bytes + (size_t)(j * gpp + gi - pi * gpp) * GB);
        };
        long long at_cur = find(0), at_next = find(1);
        auto issue = [&](int k) {   // one commit group per call
            const long long at = __shfl_sync(0xffffffffu, (k >> 5) & 1 ? at_next : at_cur, k & 31);
            if (k < nk && at >= 0) {
                const uint8_t* src = a.c.pages + at;
                const uint32_t dst = smem_addr(ring + (k % ST) * GB);
#pragma unroll
                for (int i = 0; i < (GB / 16 + 31) / 32; i++) {
                    const int o = 32 * i + lane;
                    if (o < GB / 16)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 16 * o), "l"(src + 16 * o)
                                     : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };

        float m[NT][2], l[NT][2], o[NT][2 * NB][4], oc[NT][OC][4];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int k = 0; k < 2; k++) m[n][k] = -INFINITY, l[n][k] = 0.0f;
#pragma unroll
            for (int t = 0; t < 2 * NB; t++)
#pragma unroll
                for (int k = 0; k < 4; k++) o[n][t][k] = 0.0f;
#pragma unroll
            for (int t = 0; t < OC; t++)
#pragma unroll
                for (int k = 0; k < 4; k++) oc[n][t][k] = 0.0f;
        }
        int vexp = -100;                         // V scales are held times 2^-vexp
        __half2 vmul = __float2half2_rn(0.0f);   // that factor (two of them: 2^-vexp may leave fp16)
        __half2 vmul2 = vmul;

#pragma unroll
        for (int k = 0; k < ST - 1; k++) issue(k);
        for (int k = 0; k < nk; k++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
            __syncwarp();
            const long long at = __shfl_sync(0xffffffffu, (k >> 5) & 1 ? at_next : at_cur, k & 31);
            // the lanes' places: two sets of 32, the one behind refilled when the front moves on
            if ((k & 31) == 0 && k) {
                if ((k >> 5) & 1) at_cur = find((k >> 5) + 1);
                else at_next = find((k >> 5) + 1);
            }
            issue(k + ST - 1);
            if (at < 0) continue;
            const uint8_t* gr = ring + (k % ST) * GB;
            const int t0 = (g0 + wid + k * W) * 16;

            // ---- scores
            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int x = 0; x < 4; x++) sc[n][x] = 0.0f;
            const uint32_t* kc = reinterpret_cast<const uint32_t*>(gr) + lane * NB;   // chunk (h, g, c): word h * 32 * NB
            const __half* ks = reinterpret_cast<const __half*>(gr + 16 * HD) + g * NB;
            uint32_t kw[2][NB];
            float kd[2][NB];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if constexpr (NB % 4 == 0) {
#pragma unroll
                    for (int i = 0; i < NB; i += 4)
                        *reinterpret_cast<uint4*>(&kw[h][i]) = *reinterpret_cast<const uint4*>(kc + h * 32 * NB + i);
                } else if constexpr (NB % 2 == 0) {
#pragma unroll
                    for (int i = 0; i < NB; i += 2)
                        *reinterpret_cast<uint2*>(&kw[h][i]) = *reinterpret_cast<const uint2*>(kc + h * 32 * NB + i);
                } else {
#pragma unroll
                    for (int i = 0; i < NB; i++) kw[h][i] = kc[h * 32 * NB + i];
                }
                if constexpr (NB % 2 == 0) {
#pragma unroll
                    for (int i = 0; i < NB; i += 2) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(ks + h * 8 * NB + i));
                        kd[h][i] = f.x;
                        kd[h][i + 1] = f.y;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < NB; i++) kd[h][i] = __half2float(ks[h * 8 * NB + i]);
                }
            }
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const uint32_t w0 = kw[0][i], w1 = kw[1][i], x0 = w0 >> 8, x1 = w1 >> 8;
                const uint32_t a0[4] = {codes_lo<RAW>(w0), codes_lo<RAW>(w1), codes_hi<RAW>(w0), codes_hi<RAW>(w1)};
                const uint32_t a1[4] = {codes_lo<RAW>(x0), codes_lo<RAW>(x1), codes_hi<RAW>(x0), codes_hi<RAW>(x1)};
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float acc[4] = {corr[n][i][0], corr[n][i][1], corr[n][i][0], corr[n][i][1]};
#pragma unroll
                    for (int p = 0; p < PC; p++) {
                        mma16816(acc, a0, qf[n][p][2 * i][0], qf[n][p][2 * i][1]);
                        mma16816(acc, a1, qf[n][p][2 * i + 1][0], qf[n][p][2 * i + 1][1]);
                    }
                    sc[n][0] = fmaf(kd[0][i], acc[0], sc[n][0]);
                    sc[n][1] = fmaf(kd[0][i], acc[1], sc[n][1]);
                    sc[n][2] = fmaf(kd[1][i], acc[2], sc[n][2]);
                    sc[n][3] = fmaf(kd[1][i], acc[3], sc[n][3]);
                }
            }

            // ---- p = 2^(s - m + P_EXP); m moves when a score is beyond its slack
            bool over = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int x = 0; x < 4; x++) sc[n][x] *= fac[n][x & 1];
            if (t0 + 16 > lim_min) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        if (t0 + g + 8 * (x >> 1) >= lim[n][x & 1]) sc[n][x] = -INFINITY;
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int x = 0; x < 4; x++) over |= sc[n][x] > m[n][x & 1] + P_SLACK;

            // ---- V scales: pairs of tokens, the lane's own; larger ones than fit, or not finite?
            const uint32_t* vs = reinterpret_cast<const uint32_t*>(gr + 17 * HD) + c * NB;
            uint32_t vd[2][NB];
            __half2 vtop = __float2half2_rn(0.0f);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if constexpr (NB % 4 == 0) {
#pragma unroll
                    for (int i = 0; i < NB; i += 4)
                        *reinterpret_cast<uint4*>(&vd[h][i]) = *reinterpret_cast<const uint4*>(vs + h * 4 * NB + i);
                } else {
#pragma unroll
                    for (int i = 0; i < NB; i++) vd[h][i] = vs[h * 4 * NB + i];
                }
#pragma unroll
                for (int i = 0; i < NB; i++) vtop = __hmax2_nan(vtop, __habs2(as_h2(vd[h][i])));
            }
            const float vt = fmaxf(__low2float(vtop), __high2float(vtop));
            const bool vnan = !(__low2float(vtop) <= 65504.0f) || !(__high2float(vtop) <= 65504.0f);
            // rows behind the limits hold anything: their NaN must not reach a product
            const bool odd = __any_sync(0xffffffffu, over || vnan || vt > scalbnf(1.0f, V_HIGH + vexp));
            bool mend = false;
            if (odd) {
                mend = __any_sync(0xffffffffu, vnan);
                float top = vnan ? 0.0f : vt;
                if (mend) {   // the largest finite one
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int i = 0; i < NB; i++) {
                            const float x = fabsf(__low2float(as_h2(vd[h][i]))), y = fabsf(__high2float(as_h2(vd[h][i])));
                            if (x <= 65504.0f) top = fmaxf(top, x);
                            if (y <= 65504.0f) top = fmaxf(top, y);
                        }
                }
#pragma unroll
                for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                float vf = 1.0f;
                if (top > scalbnf(1.0f, V_HIGH + vexp)) {
                    const int e = max(ilogbf(top) - V_LOW, -30);
                    vf = scalbnf(1.0f, max(vexp - e, -126));
                    vexp = e;
                    vmul = __float2half2_rn(scalbnf(1.0f, -(vexp / 2)));
                    vmul2 = __float2half2_rn(scalbnf(1.0f, -(vexp - vexp / 2)));
                }
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int k2 = 0; k2 < 2; k2++) {
                        float t = fmaxf(sc[n][k2], sc[n][k2 + 2]);
#pragma unroll
                        for (int x = 16; x >= 4; x >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
                        const float mn = fmaxf(m[n][k2], t);
                        const float f = mn == m[n][k2] ? 1.0f : ex2(m[n][k2] - mn);
                        m[n][k2] = mn;
                        l[n][k2] *= f;
                        const float of = f * vf;
#pragma unroll
                        for (int t2 = 0; t2 < 2 * NB; t2++) {
                            o[n][t2][k2] *= of;
                            o[n][t2][k2 + 2] *= of;
                        }
#pragma unroll
                        for (int t2 = 0; t2 < OC; t2++) {
                            oc[n][t2][k2] *= of;
                            oc[n][t2][k2 + 2] *= of;
                        }
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < NB; i++) vd[h][i] = as_u32(__hmul2(__hmul2(as_h2(vd[h][i]), vmul), vmul2));

            // ---- p in pieces, transposed: lane (g, c) gets row g's tokens 2c, 2c + 1 of each half
            uint32_t ph[NT][PC][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float p[4];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    // nothing seen yet leaves m at -inf: masked scores are 0, NaN stays NaN
                    p[x] = sc[n][x] == -INFINITY ? 0.0f : ex2(sc[n][x] - (m[n][x & 1] - P_EXP));
                    l[n][x & 1] += p[x];
                    // beside a NaN a probability that fp16 would lose stays above zero
                    if (mend && sc[n][x] > -INFINITY) p[x] = fmaxf(p[x], 0x1p-24f);
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const __half2 hi = __floats2half2_rn(p[2 * h], p[2 * h + 1]);
                    ph[n][0][h] = transpose8(as_u32(hi));
                    if constexpr (PC == 2)
                        ph[n][1][h] = transpose8(
                            as_u32(__floats2half2_rn(p[2 * h] - __low2float(hi), p[2 * h + 1] - __high2float(hi))));
                }
            }

            // ---- O += (p d) V
            const uint32_t* vc = reinterpret_cast<const uint32_t*>(gr + 8 * HD) + lane * NB;
            uint32_t vw[2][NB];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if constexpr (NB % 4 == 0) {
#pragma unroll
                    for (int i = 0; i < NB; i += 4)
                        *reinterpret_cast<uint4*>(&vw[h][i]) = *reinterpret_cast<const uint4*>(vc + h * 32 * NB + i);
                } else if constexpr (NB % 2 == 0) {
#pragma unroll
                    for (int i = 0; i < NB; i += 2)
                        *reinterpret_cast<uint2*>(&vw[h][i]) = *reinterpret_cast<const uint2*>(vc + h * 32 * NB + i);
                } else {
#pragma unroll
                    for (int i = 0; i < NB; i++) vw[h][i] = vc[h * 32 * NB + i];
                }
            }
            constexpr uint32_t M8 = 0x80088008u, M8H = 0x80808080u;   // -8 * 2^-24, -8 * 2^-20
            const uint32_t ones[4] = {M8, M8H, M8, M8H};
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const uint32_t w0 = vw[0][i], w1 = vw[1][i], x0 = w0 >> 8, x1 = w1 >> 8;
                // rows g: the lower nibbles' dimensions; rows g + 8: the upper ones'
                const uint32_t a0[4] = {codes_lo<RAW>(w0), codes_hi<RAW>(w0), codes_lo<RAW>(w1), codes_hi<RAW>(w1)};
                const uint32_t a1[4] = {codes_lo<RAW>(x0), codes_hi<RAW>(x0), codes_lo<RAW>(x1), codes_hi<RAW>(x1)};
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    uint32_t pb[PC][2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const __half2 d = as_h2(vd[h][i]), p0 = as_h2(ph[n][0][h]);
                        __half2 hi = __hmul2(p0, d);
                        if constexpr (PC == 2) {
                            // what the product lost, and the lower piece's
                            __half2 lo = __hfma2(as_h2(ph[n][1][h]), d, __hfma2(p0, d, __hneg2(hi)));
                            if (mend) lo = as_u32(p0) & 0x7fffu ? lo : __halves2half2(__float2half_rn(0.0f), __high2half(lo));
                            if (mend) lo = as_u32(p0) & 0x7fff0000u ? lo : __halves2half2(__low2half(lo), __float2half_rn(0.0f));
                            pb[1][h] = as_u32(lo);
                        }
                        if (mend) {
                            if (!(as_u32(p0) & 0x7fffu)) hi = __halves2half2(__float2half_rn(0.0f), __high2half(hi));
                            if (!(as_u32(p0) & 0x7fff0000u)) hi = __halves2half2(__low2half(hi), __float2half_rn(0.0f));
                        }
                        pb[0][h] = as_u32(hi);
                    }
#pragma unroll
                    for (int p = 0; p < PC; p++) {
                        mma16816(o[n][2 * i], a0, pb[p][0], pb[p][1]);
                        mma16816(o[n][2 * i + 1], a1, pb[p][0], pb[p][1]);
                        if constexpr (RAW) mma16816(oc[n][i], ones, pb[p][0], pb[p][1]);
                    }
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // ---- the warps meet: m, l and O of every query row, in shared memory
        const bool whole = g0 == 0 && g1 == si.grans;
        constexpr int PR = HD + 4;   // floats per row: O, then m and l
        float* js = reinterpret_cast<float*>(sm) + wid * ROWS * PR;
        __syncthreads();
        const float back = scalbnf(1.0f, min(max((RAW ? 24 : 0) - 6 + vexp, -126), 127));   // out of the units of p, the codes and vexp
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float lt = l[n][k];
#pragma unroll
                for (int x = 16; x >= 4; x >>= 1) lt += __shfl_xor_sync(0xffffffffu, lt, x);
                float* row = js + (8 * n + 2 * c + k) * PR;
#pragma unroll
                for (int i = 0; i < NB; i++)
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        row[32 * i + 16 * t + g] = (o[n][2 * i + t][k] + oc[n][RAW ? i : 0][k]) * back;
                        row[32 * i + 16 * t + 8 + g] =
                            (o[n][2 * i + t][k + 2] + oc[n][RAW ? i : 0][k + 2]) * (RAW ? 0.0625f : 1.0f) * back;
                    }
                if (g == 0) {
                    row[HD] = m[n][k];
                    row[HD + 1] = lt * 0x1p-6f;
                }
            }
        __syncthreads();
        const int slot = (int)w * 2 + (g0 == 0 ? 1 : 0);
        for (int i = tid; i < ROWS * (HD / 4); i += blockDim.x) {
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
            if (r >= nrows) continue;
            const float* p = reinterpret_cast<const float*>(sm) + r * PR;
            float mm = -INFINITY, ll = 0.0f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int v = 0; v < W; v++) mm = fmaxf(mm, p[v * ROWS * PR + HD]);
            for (int v = 0; v < W; v++) {
                const float* pv = p + v * ROWS * PR;
                const float f = pv[HD] == mm ? 1.0f : ex2(pv[HD] - mm);
                const float4 y = *reinterpret_cast<const float4*>(pv + d);
                x.x = fmaf(f, y.x, x.x);
                x.y = fmaf(f, y.y, x.y);
                x.z = fmaf(f, y.z, x.z);
                x.w = fmaf(f, y.w, x.w);
                ll = fmaf(f, pv[HD + 1], ll);
            }
            if (whole) {
                const int rho = row0 + r;
                T* dst = reinterpret_cast<T*>(a.out) + (size_t)(si.s0 + rho / a.R) * a.os + (size_t)(j * a.R + rho % a.R) * HD + d;
                const float inv = ll == 0.0f ? 0.0f : __fdiv_rn(1.0f, ll);
                from_f32(x.x * inv, dst[0]);
                from_f32(x.y * inv, dst[1]);
                from_f32(x.z * inv, dst[2]);
                from_f32(x.w * inv, dst[3]);
            } else {
                float* dst = a.slots + ((size_t)slot * ROWS + r) * PR;
                *reinterpret_cast<float4*>(dst + d) = x;
                if (d == 0) dst[HD] = mm, dst[HD + 1] = ll;
            }
        }
        if (!whole && tid == 0) {
            int* h = a.heads + (size_t)slot * 4;
            h[0] = g1 == si.grans ? SLOT_LAST : SLOT_MORE;
            h[1] = si.s0 + row0 / a.R;               // token and head of the first query row
            h[2] = j * a.R + row0 % a.R;
            h[3] = nrows;
        }
        __syncthreads();
    }
}

// One CTA per (worker, query row of an item): where the worker's second slot begins an item,
// the parts of the following workers are added to it up to the item's last.
template <int DT, int NB, int NT>
__global__ void __launch_bounds__(128) k_kvq_join(AttnKvqArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int HD = 32 * NB, ROWS = 8 * NT, PR = HD + 4;
    __shared__ float s_o[4][HD], s_l[4], s_m[4];
    __shared__ int s_n;
    const int w = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int* h = a.heads + ((size_t)w * 2 + 1) * 4;
    if (h[0] == SLOT_NONE || r >= h[3]) return;
    if (wid == 0) {   // workers behind w up to the one with the item's last part
        int n = 1;
        for (int x = w + 1; x < a.workers; x += 32) {
            const int v = x + lane;
            const int kind = v < a.workers ? a.heads[(size_t)v * 8] : SLOT_LAST;
            const unsigned last = __ballot_sync(0xffffffffu, kind != SLOT_MORE);
            if (last) {
                n += __ffs(last);
                break;
            }
            n += 32;
        }
        if (lane == 0) s_n = n;
    }
    __syncthreads();
    const int n = s_n;   // parts: the second slot of w, then the first slots of w + 1, ...
    auto part = [&](int i) { return a.slots + ((size_t)(i == 0 ? 2 * w + 1 : 2 * (w + i)) * ROWS + r) * PR; };
    float m = -INFINITY, l = 0.0f, o[NB];
#pragma unroll
    for (int i = 0; i < NB; i++) o[i] = 0.0f;
    for (int i = tid; i < n; i += 128) m = fmaxf(m, part(i)[HD]);
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    if (lane == 0) s_m[wid] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
#pragma unroll 4
    for (int i = wid; i < n; i += 4) {
        const float* p = part(i);
        const float f = p[HD] == m ? 1.0f : ex2(p[HD] - m);
        l = fmaf(f, p[HD + 1], l);
#pragma unroll
        for (int x = 0; x < NB; x++) o[x] = fmaf(f, p[32 * x + lane], o[x]);
    }
#pragma unroll
    for (int x = 0; x < NB; x++) s_o[wid][32 * x + lane] = o[x];
    if (lane == 0) s_l[wid] = l;
    __syncthreads();
    l = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    const int rho = h[2] % a.R + r;   // query row counted from the first token of the tile
    T* dst = reinterpret_cast<T*>(a.out) + (size_t)(h[1] + rho / a.R) * a.os + (size_t)(h[2] / a.R * a.R + rho % a.R) * HD;
    for (int d = tid; d < HD; d += 128) from_f32(((s_o[0][d] + s_o[1][d]) + (s_o[2][d] + s_o[3][d])) * inv, dst[d]);
}

// ---------------------------------------------------------------- launching
// Up to this many query rows per kv head, a worker's warps share an item (one row tile, the
// granules dealt out); with more, every warp is a worker of its own.
constexpr int DEEP_ROWS = 32;
constexpr int MAX_DEV = 64;
constexpr int MAX_SMS = 160;


constexpr int workers_per_sm(int warps) { return warps > 1 ? 4 : 12; }

// A second tile of 8 query rows takes the same unpacked codes: worth it where there are the
// rows for it and the registers (fp32 holds q and p twice).
constexpr bool two_tiles(int dt, int nb) { return nb <= (dt == TGX_F32 ? 3 : 4); }

struct Shape {
    int warps, nt, workers;
};

// Workers and their row tiles for these bounds; at most `have` workers are resident.
Shape shape_of(const KvqCache& c, const KvqBatch& b, int R, bool two, int have_one, int have_deep) {
    Shape sh;
    const long long rows = (long long)b.max_new * R;
    sh.warps = rows <= DEEP_ROWS ? DEEP_WARPS : 1;
    sh.nt = rows > 8 && two ? 2 : 1;
    // no more workers than there can be granules for their warps
    const long long most = (long long)b.B * c.nkv * ((rows + 8 * sh.nt - 1) / (8 * sh.nt)) *
                           (((long long)b.max_pages * c.pt + 15) / 16);
    const long long have = sh.warps > 1 ? have_deep : have_one, want = (most + sh.warps - 1) / sh.warps;
    sh.workers = (int)(want < have ? want : have);
    return sh;
}

size_t head_bytes(int workers) { return ((size_t)workers * 32 + 255) & ~(size_t)255; }
size_t attn_scratch(const Shape& sh, int hd) {
    return head_bytes(sh.workers) + (size_t)sh.workers * 2 * 8 * sh.nt * (hd + 4) * 4;
}

template <int DT, int NB, int NT>
int attn_workers(int W) {   // resident CTAs of the device, per kernel and CTA size
    static std::mutex mu;
    static int known[MAX_DEV][2] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEV) return 0;
    std::lock_guard<std::mutex> lock(mu);
    int& n = known[dev][W > 1];
    if (!n) {
        int sms = 0, per = 0;
        const int smem = attn_smem<NB, NT>(W);
        if (cudaFuncSetAttribute(k_kvq_attn<DT, NB, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 attn_smem<NB, NT>(DEEP_WARPS)) != cudaSuccess ||
            cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, k_kvq_attn<DT, NB, NT>, 32 * W, smem) != cudaSuccess)
            return 0;
        n = std::min(sms, MAX_SMS) * std::max(1, std::min(per, workers_per_sm(W)));
    }
    return n;
}

template <int DT, int NB, int NT>
cudaError_t launch_attn_t(AttnKvqArgs a, int W, int workers, cudaStream_t s) {
    a.workers = workers;
    k_kvq_attn<DT, NB, NT><<<workers, 32 * W, attn_smem<NB, NT>(W), s>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(workers, 8 * NT);
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_kvq_join<DT, NB, NT>, a);
}

template <int DT, int NB>
cudaError_t launch_attn_nb(AttnKvqArgs a, void* scratch, size_t scratch_bytes, cudaStream_t s) {
    constexpr int NT2 = two_tiles(DT, NB) ? 2 : 1;
    const bool nt2 = NT2 == 2 && (long long)a.b.max_new * a.R > 8;
    const int one = nt2 ? attn_workers<DT, NB, NT2>(1) : attn_workers<DT, NB, 1>(1);
    const int deep = nt2 ? attn_workers<DT, NB, NT2>(DEEP_WARPS) : attn_workers<DT, NB, 1>(DEEP_WARPS);
    if (!one || !deep) return cudaErrorUnknown;
    const Shape sh = shape_of(a.c, a.b, a.R, NT2 == 2, one, deep);
    if (scratch_bytes < attn_scratch(sh, a.c.hd)) return cudaErrorInvalidValue;
    a.heads = reinterpret_cast<int*>(scratch);
    a.slots = reinterpret_cast<float*>((uint8_t*)scratch + head_bytes(sh.workers));
    return nt2 ? launch_attn_t<DT, NB, NT2>(a, sh.warps, sh.workers, s)
               : launch_attn_t<DT, NB, 1>(a, sh.warps, sh.workers, s);
}

#define TG_NB(DT, F, ...)                     \
    switch (a.c.hd / 32) {                    \
        case 1: return F<DT, 1>(__VA_ARGS__); \
        case 2: return F<DT, 2>(__VA_ARGS__); \
        case 3: return F<DT, 3>(__VA_ARGS__); \
        case 4: return F<DT, 4>(__VA_ARGS__); \
        case 5: return F<DT, 5>(__VA_ARGS__); \
        case 6: return F<DT, 6>(__VA_ARGS__); \
        case 7: return F<DT, 7>(__VA_ARGS__); \
        default: return F<DT, 8>(__VA_ARGS__); \
    }

template <int DT>
cudaError_t launch_t(const AttnKvqArgs& a, void* scratch, size_t n, cudaStream_t s) { TG_NB(DT, launch_attn_nb, a, scratch, n, s) }

cudaError_t launch_attn(int dtype, const AttnKvqArgs& a, void* scratch, size_t n, cudaStream_t s) {
    return dtype == TGX_F32    ? launch_t<TGX_F32>(a, scratch, n, s)
           : dtype == TGX_BF16 ? launch_t<TGX_BF16>(a, scratch, n, s)
                               : launch_t<TGX_F16>(a, scratch, n, s);
}

}  // namespace

}  // namespace tg

extern "C" size_t tgx_kvq_attention_scratch_bytes(const tgx_kvq_cache* cache, const tgx_kvq_batch* batch, int n_tokens,
                                                  int n_heads) {
    if (!cache || !batch || n_tokens < 0 || n_heads <= 0 || n_heads > 32 * 4096 ||
        !tgx_kvq_page_bytes(cache->n_kv_heads, cache->head_dim, cache->page_tokens) || n_heads % cache->n_kv_heads ||
        batch->n_seqs <= 0 || batch->max_pages <= 0 || batch->max_new <= 0)
        return 0;
    const tg::KvqCache c = tg::kvq_cache(*cache);
    const tg::KvqBatch b = tg::kvq_batch(*batch);
    size_t most = 0;   // of any type, on any device
    for (int two = 0; two < 2; two++)
        most = std::max(most, tg::attn_scratch(tg::shape_of(c, b, n_heads / c.nkv, two, tg::MAX_SMS * tg::workers_per_sm(1),
                                                            tg::MAX_SMS * tg::workers_per_sm(tg::DEEP_WARPS)), c.hd));
    return most;
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
    if ((long long)n_tokens * n_heads >= 0x7fffffffll)
        return tg::serve_fail(TG_EINVAL, fn, "too many tokens for one call");
    if (!(scale >= 0.0f) || scale > 3e38f) return tg::serve_fail(TG_EINVAL, fn, "scale must be finite and not negative");
    tg::ServeDevice dev(fn, cache->pages);
    if (dev.rc != TG_OK || n_tokens == 0) return dev.rc;
    const float sc = (scale > 0.0f ? scale : 1.0f / sqrtf((float)cache->head_dim)) * 1.44269504088896340736f;
    tg::AttnKvqArgs a{tg::kvq_cache(*cache), tg::kvq_batch(*batch), n_tokens, n_heads, n_heads / cache->n_kv_heads, q,
                      q_stride, out, out_stride, sc, 0, nullptr, nullptr};
    cudaError_t e = tg::launch_attn(dtype, a, scratch, scratch_bytes, (cudaStream_t)stream);
    return e == cudaSuccess ? TG_OK : tg::serve_fail(TG_ECUDA, fn, cudaGetErrorString(e));
}
