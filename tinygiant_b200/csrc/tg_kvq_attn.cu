// tg_kvq_attn.cu — attention of many tokens over the paged 4-bit key/value cache.
//
//   s_r = scale * q . k_r over the rows r up to the token's own, p = softmax(s),
//   out = sum_r p_r v_r
// in one pass over the rows: a running reference m (the maximum, or within 2^4 of it), the
// sum l of exp2(s - m) and the output, rescaled when the scores leave m's range.  All three are fp32.
//
// Both products run on the tensor cores with the codes as the other operand, mma m16n8k16:
//   K: rows 16 cached tokens, columns 8 query rows (heads of the kv head x new tokens), k 16
//      dimensions; a block's sum enters the score times the block's scale, in fp32.
//   V: rows 16 dimensions, columns the query rows, k 16 tokens; a block's scale goes into the
//      probability, p * d, per block.
// fp32 inputs keep 22 bits of q and of p * d as two fp16 pieces, each an mma of its own; for
// 16-bit types one piece (11 bits) is as fine as the output.  The pieces stay in fp16's range
// by powers of two: q's rows are scaled to 2^13 .. 2^14, p to 2^6 at its maximum, V scales to
// 2^2 .. 2^5 at the largest met so far among the rows that the item sees (vexp; O is rescaled when
// a larger one comes).  So a probability below 2^-31 of its row's largest counts as 0.
//
// Codes become fp16 by masks: a nibble in the low bits of 1024, and one half-precision
// operation makes it code - 8.  K's codes with 16-bit types go without the second: a nibble
// masked into the low byte of a halfword IS the number code * 2^-24 (a subnormal; 2^-20 for
// the nibble above it).  The upper nibbles' factor 16 is taken off q, and the codes' offset is
// -8 sum q, the scores' first accumulator.  (The tensor cores align products by exponent
// fields, which subnormals leave 2^6 .. 2^10 above their values, so such a sum is good to about
// 2^-17 of sum |q| 16 d: enough for a score behind 16-bit inputs, too coarse for fp32, and for
// V, where sum 8 p d would have to cancel.)
//
// Work: an item is (sequence, kv head, tile of 8 * NT query rows) over the sequence's granules
// of 16 tokens (18 * HD contiguous bytes).  A worker is a CTA of W warps.  All items in one line are
// cut into one part per worker, whatever the lengths, and a worker walks the items of its part;
// few items are each cut into equal parts, a worker each.  Each of its warps takes every W-th pair of granules, through a ring of its own that
// cp.async keeps STAGES deep, and the W results meet in shared memory.  An item that lies in
// one part is finished there; the others' parts go to scratch and k_kvq_join adds them in
// order, so results repeat exactly.
//
// A granule is 2304 bytes at HD 128, about 100 cycles of an SM's share of the bandwidth, against 40
// to 80 of its tensor cores.  Bound by the latency of a warp's chain (scores, exponentials,
// transpose, sums) that 11 warps an SM do not hide: 128 streams of up to 12000 rows, bf16, take 126 us,
// 4.4 TB/s; at 32 of them issue is at 50%, DRAM at 40%, the tensor pipe at 16%.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "tg_kvq_attn.cuh"

namespace tg {

namespace {

constexpr int DEEP_WARPS = 4;         // warps of a worker that share an item
constexpr float P_EXP = 6.0f;        // p is held times 2^P_EXP
constexpr float P_SLACK = 4.0f;      // and may exceed that by 2^P_SLACK before m moves
constexpr int V_LOW = 2, V_HIGH = 5; // V scales are held in 2^V_LOW .. 2^V_HIGH at the largest: 2^(6 + 4 + 5) < 65504

// What beginning an item costs beside its granules, in a warp's granules: about 5 us measured
// (queries, first copies, joining the warps), against 0.6 us for a granule.
constexpr int OPEN_UNITS = 8;

// Slot kinds: nothing; a part that its item goes on behind; the item's last part.
constexpr int MAX_SMS = 160;
constexpr int workers_per_sm(int warps) { return warps > 1 ? 4 : 12; }
constexpr int MAX_WORKERS = MAX_SMS * workers_per_sm(1);

enum { SLOT_NONE = 0, SLOT_MORE = 1, SLOT_LAST = 2 };

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a b + c
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                         const float (&e)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(e[0]), "f"(e[1]), "f"(e[2]), "f"(e[3]));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {   // an 8 x 8 tile of halves across the warp
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Four CTAs of four warps per SM (128 registers a thread) where that leaves nothing to spill.
constexpr int min_ctas(int nb, int nt) { return nb <= 3 && nt == 1 ? 4 : nb * nt <= 4 ? 3 : 2; }

constexpr int STAGES = 3;
constexpr int U = 2;   // granules of a stage, and of a step of the loop

// Shared memory of a CTA of W warps: the rings, which the joining of the warps reuses, then
// the query rows' operands, factors and limits.
template <int NB, int NT>
constexpr int attn_ring(int W) {
    const int ring = W * STAGES * U * 18 * 32 * NB, join = W * 8 * NT * (32 * NB + 4) * 4;
    return ring > join ? ring : join;
}
template <int NB, int NT>
constexpr int attn_smem(int W) {
    return attn_ring<NB, NT>(W) + NT * 2 * NB * 512 + 8 * NT * (NB + 2) * 4;
}

// Exclusive prefix of v over the CTA's threads; `total` gets the sum.
__device__ __forceinline__ long long block_sum(long long v, long long& total, long long* s_scan, int W) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    long long incl = v, before = 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[wid] = incl;
    __syncthreads();
    total = 0;
    for (int i = 0; i < W; i++) {
        if (i < wid) before += s_scan[i];
        total += s_scan[i];
    }
    __syncthreads();
    return before + incl - v;
}

template <int DT, int NB, int NT>
__global__ void __launch_bounds__(32 * DEEP_WARPS, min_ctas(NB, NT)) k_kvq_attn(AttnKvqArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int HD = 32 * NB, GB = 18 * HD, ST = STAGES, KS = 2 * NB, ROWS = 8 * NT;
    constexpr int PC = DT == TGX_F32 ? 2 : 1;    // fp16 pieces of q and of p * d
    constexpr bool RAW = PC == 1;                // K's codes as subnormals
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ long long s_scan[DEEP_WARPS];
    __shared__ long long s_base;
    __shared__ int s_seq;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, W = blockDim.x >> 5;
    const int g = lane >> 2, c = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- the plan, made by every worker for itself.  Thread t owns sequences [t * per, ...), so
    // a prefix over the threads is one over them.  Units: granules, and OPEN for each item, what
    // beginning another item costs.
    const int per = (a.b.B + (int)blockDim.x - 1) / (int)blockDim.x, w = blockIdx.x;
    const int OPEN = OPEN_UNITS * W;
    long long mine = 0, grans = 0, before, total, total_grans, items = 0;
    for (int i = 0; i < per; i++) {
        const int b = tid * per + i;
        if (b < a.b.B) {
            const SeqInfo s = seq_info(a, b, ROWS);
            const long long n = (long long)s.tiles * a.c.nkv;
            mine += n;
            grans += n * s.grans;
            if (w == 0 && (long long)a.b.kv_lens[b] > (long long)a.b.max_pages * a.c.pt) kvq_flag(a.b, TGX_KVQ_BAD_LENGTH);
            const int s0 = a.b.q_start[b], s1 = a.b.q_start[b + 1];
            if (w == 0 && (s0 < 0 || s1 < s0 || s1 > a.T || s1 - s0 > a.b.max_new)) kvq_flag(a.b, TGX_KVQ_BAD_NEW);
        }
    }
    if (tid < 2) a.heads[((size_t)w * 2 + tid) * 4] = SLOT_NONE;   // no slots yet
    block_sum(mine, items, s_scan, W);
    block_sum(grans, total_grans, s_scan, W);
    int b, item, g0, g1;            // the piece at hand: sequence, item in it, granules
    long long u = 0, u_end = 0, base = 0;
    // One line of all items cut into equal parts, or each item in parts of its own, of at most
    // `quota` granules, where that is no longer than a part of the line and a second beginning in it.
    const int step = U * W;
    const long long room = a.workers - items;
    const long long quota = room > 0 ? max(1ll, quotient(quotient(total_grans, room) + step, step)) * step : 0;
    const bool few = room > 0 && quota <= quotient(total_grans + items * OPEN, a.workers) + OPEN;
    if (few) {
        auto parts = [&](const SeqInfo& s) { return (int)quotient(s.grans + quota - 1, quota); };
        mine = 0;
        for (int i = 0; i < per; i++) {
            const int b = tid * per + i;
            if (b < a.b.B) {
                const SeqInfo s = seq_info(a, b, ROWS);
                mine += (long long)s.tiles * a.c.nkv * parts(s);
            }
        }
        before = block_sum(mine, total, s_scan, W);
        if (w >= total) return;
        if (w >= before && w < before + mine) {
            long long x = before;
            int b = tid * per;
            for (;; b++) {
                const SeqInfo s = seq_info(a, b, ROWS);
                const long long n = (long long)s.tiles * a.c.nkv * parts(s);
                if (w < x + n) break;
                x += n;
            }
            s_seq = b;
            s_base = x;
        }
        __syncthreads();
        b = s_seq;
        const SeqInfo s = seq_info(a, b, ROWS);
        const int n = parts(s), part = (int)(w - s_base) % n;
        item = (int)(w - s_base) / n;
        g0 = (int)((long long)s.grans * part / n);
        g1 = (int)((long long)s.grans * (part + 1) / n);
    } else {   // one line, cut into equal parts
        mine = grans + mine * OPEN;
        before = block_sum(mine, total, s_scan, W);
        const long long share = quotient(total, a.workers), more = total - share * a.workers;   // one unit more
        u = share * w + min((long long)w, more);
        u_end = u + share + (w < more ? 1 : 0);
        if (u >= u_end) return;
        if (u >= before && u < before + mine) {
            long long x = before;
            int b = tid * per;
            for (;; b++) {
                const SeqInfo s = seq_info(a, b, ROWS);
                const long long n = (long long)s.tiles * a.c.nkv * (s.grans + OPEN);
                if (u < x + n) break;
                x += n;
            }
            s_seq = b;
            s_base = x;
        }
        __syncthreads();
        b = s_seq;
        base = s_base;   // units in front of sequence b
    }

    uint8_t* ring = sm + wid * ST * U * GB;
    uint32_t* s_q = reinterpret_cast<uint32_t*>(sm + attn_ring<NB, NT>(W));   // q's operands, [tile][piece][NB][lane][4]
    float* s_corr = reinterpret_cast<float*>(s_q + NT * PC * KS * 64);        // [row][NB]
    float* s_fac = s_corr + ROWS * NB;
    int* s_lim = reinterpret_cast<int*>(s_fac + ROWS);
    const uint32_t k1024 = a.k1024;
    do {
        const SeqInfo si = seq_info(a, b, ROWS);
        if (!few) {
            const int each = si.grans + OPEN;
            const long long units = (long long)si.tiles * a.c.nkv * each;
            if (u >= base + units) {
                base += units;
                b++;
                continue;
            }
            item = (int)quotient(u - base, each);
            const int x = (int)(u - base - (long long)item * each);
            const int y = (int)min((long long)each, x + (u_end - u));
            u += y - x;
            g0 = max(0, x - OPEN);
            g1 = y - OPEN;
            if (g1 <= g0) continue;   // units of its beginning only: the next worker begins it
        }
        const int rt = item / a.c.nkv, j = item % a.c.nkv;   // kv heads innermost
        const int row0 = rt * ROWS, nrows = min(ROWS, si.n * a.R - row0);   // query rows of the item

        // rows that new token i attends to: those below its limit
        auto limit = [&](int i) { return (int)max(0ll, min(si.len, (long long)si.off + i + 1)); };
        const int lim_min = limit(row0 / a.R), lim_max = limit((row0 + nrows - 1) / a.R);

        // ---- this warp's granules below the last visible row: U from g0 + U wid on, U from
        // g0 + U (wid + W) on, ..., in nk steps
        const int gl = min(g1, (lim_max + 15) >> 4);
        const int nk = gl > g0 + U * wid ? (gl - g0 - U * wid + U * W - 1) / (U * W) : 0;
        const int gpp = a.c.pt >> 4;
        // lane l: the 32 x + l'th of them, counted through all pages, or NO_GRANULE
        auto find = [&](int x) -> uint32_t {
            const int k = 32 * x + lane, gi = g0 + U * (wid + k / U * W) + k % U;
            if (gi >= gl) return NO_GRANULE;
            const int pi = gi / gpp;
            const int page = a.b.table[(size_t)b * a.b.max_pages + pi];
            if (page < 0 || page >= a.c.n_pages) {
                kvq_flag(a.b, TGX_KVQ_BAD_PAGE);
                return NO_GRANULE;
            }
            return ((uint32_t)page * a.c.nkv + j) * gpp + (gi - pi * gpp);
        };
        // two sets of 32; the one behind is refilled when the front has moved on
        uint32_t at_even = find(0), at_odd = find(1);
        uint32_t there = 0;   // U bits per step: the granules that exist, the step issued last lowest
        // one commit group per call; a granule that does not exist becomes zeros
        auto issue = [&](int k) {
            const uint8_t* src[U];
            uint32_t size[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t at = __shfl_sync(0xffffffffu, k * U & 32 ? at_odd : at_even, (k * U + u) & 31);
                const bool ok = at != NO_GRANULE;   // none behind the last step either
                there = there << 1 | (ok ? 1u : 0u);
                size[u] = ok ? 16 : 0;
                src[u] = a.c.pages + (size_t)(ok ? at : 0) * GB;
            }
            const uint32_t dst = smem_addr(ring + (k % ST) * (U * GB)) + 16 * lane;
            constexpr int C = GB / 16;   // pieces of a granule
#pragma unroll
            for (int i = 0; i < (U * C + 31) / 32; i++) {
                const int o = 32 * i + lane;
                const int first = 32 * i / C, last = min(U * C - 1, 32 * i + 31) / C;   // granules of the lanes
                const int u = first == last ? first : o >= last * C ? last : first;
                const uint8_t* from = (first == last ? src[first] : o >= last * C ? src[last] : src[first]) + 16 * (o - u * C);
                const uint32_t n = first == last ? size[first] : o >= last * C ? size[last] : size[first];
                if (32 * i + 32 <= U * C || o < U * C)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 512 * i), "l"(from), "r"(n)
                                 : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int k = 0; k < ST - 1; k++) issue(k);

        // ---- the query rows as B operands: lane (g, c) holds row g's dimensions 16s + 2c, + 1
        // and + 8, and the rows' factors, limits and offsets for the columns 2c, 2c + 1.  A warp
        // makes every W-th row's, for all; lane l takes the pairs of dimensions 2l + 64x, + 1.
        for (int r = wid; r < ROWS; r += W) {
            const bool ok = r < nrows;
            const int rho = row0 + r;
            const T* src = reinterpret_cast<const T*>(a.q) + (size_t)(si.s0 + (ok ? rho / a.R : 0)) * a.qs +
                           (size_t)(j * a.R + (ok ? rho % a.R : 0)) * HD;
            constexpr int NP = (NB + 1) / 2;
            float2 x[NP];
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < NP; i++) {
                x[i] = make_float2(0.0f, 0.0f);
                if (ok && (NB % 2 == 0 || 64 * i + 2 * lane < HD)) x[i] = load2(src + 64 * i + 2 * lane);
                top = fmaxf(top, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
            }
#pragma unroll
            for (int y = 16; y >= 1; y >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, y));
            // 2^-e: top into 2^13 .. 2^14, from its exponent field (e down to -113 for tiny ones).  The
            // factor is two powers of two: e reaches beyond fp32's exponents
            const int field = (int)(__float_as_uint(top) >> 23);
            const int e = field == 255 || top == 0.0f ? 0 : max(field - 127, -100) - 13, half = e / 2;
            const float up1 = __uint_as_float((uint32_t)(127 - half) << 23), up2 = __uint_as_float((uint32_t)(127 - (e - half)) << 23);
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int d = 64 * i + 2 * lane, s = d / 16, h = d / 8 % 2, cc = d / 2 % 4, word = 2 * s + h;
                const float y0 = x[i].x * up1 * up2, y1 = x[i].y * up1 * up2;
                const float m = RAW && h ? 0.0625f : 1.0f;   // the upper nibbles' codes count 16 times
                const __half2 hi = __floats2half2_rn(y0 * m, y1 * m);
                uint32_t* to = s_q + ((r / 8 * PC) * NB + word / 4) * 128 + (r % 8 * 4 + cc) * 4 + word % 4;
                float sum = y0 + y1;
#pragma unroll
                for (int y = 8; y >= 1; y >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, y);
                if (NB % 2 == 0 || d < HD) {
                    to[0] = as_u32(hi);
                    if constexpr (PC == 2)
                        to[NB * 128] = as_u32(__floats2half2_rn(y0 * m - __low2float(hi), y1 * m - __high2float(hi)));
                    if (lane % 16 == 0) s_corr[r * NB + d / 32] = sum * (-8.0f * 0x1p-24f);
                }
            }
            if (lane == 0) {
                s_fac[r] = bounded_fac(a.scale * (RAW ? 0x1p24f : 1.0f) * __uint_as_float((uint32_t)(127 + half) << 23) *
                                       __uint_as_float((uint32_t)(127 + e - half) << 23));
                s_lim[r] = ok ? limit(rho / a.R) : 0x7fffffff;   // rows beyond the item: any scores will do
            }
        }
        __syncthreads();
        uint32_t qf[NT][PC][KS][2];
        float corr[NT][NB][4], fac[NT][2];
        int lim[NT][2], lim_g[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int p = 0; p < PC; p++)
#pragma unroll
                for (int i = 0; i < NB; i++) {
                    const uint4 v = *reinterpret_cast<const uint4*>(s_q + ((n * PC + p) * NB + i) * 128 + lane * 4);
                    qf[n][p][2 * i][0] = v.x;
                    qf[n][p][2 * i][1] = v.y;
                    qf[n][p][2 * i + 1][0] = v.z;
                    qf[n][p][2 * i + 1][1] = v.w;
                }
            lim_g[n] = s_lim[8 * n + g];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                fac[n][k] = s_fac[8 * n + 2 * c + k];
                lim[n][k] = s_lim[8 * n + 2 * c + k];
#pragma unroll
                for (int i = 0; i < NB; i++) {
                    corr[n][i][k] = s_corr[(8 * n + 2 * c + k) * NB + i];
                    // a register of its own: the accumulator's four are read together
                    asm volatile("mov.f32 %0, %1;" : "=f"(corr[n][i][k + 2]) : "f"(corr[n][i][k]));
                }
            }
        }

        float m[NT][2], off[NT][2], l[NT][2], o[NT][2 * NB][4];   // m in raw scores; off = P_EXP - m * fac
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int k = 0; k < 2; k++) m[n][k] = -INFINITY, off[n][k] = INFINITY, l[n][k] = 0.0f;
#pragma unroll
            for (int t = 0; t < 2 * NB; t++)
#pragma unroll
                for (int k = 0; k < 4; k++) o[n][t][k] = 0.0f;
        }
        int vexp = 0;                            // V scales are held times 2^-vexp
        __half2 vmul = __float2half2_rn(1.0f);   // that factor
        uint32_t vlim = 0;                       // fp16 bits of 2^(V_HIGH + vexp), the largest scale that fits; none yet

#pragma unroll 1
        for (int k = 0; k < nk; k++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
            __syncwarp();
            if (k && (k * U & 31) == 0) {
                if (k * U & 32) at_even = find(k * U / 32 + 1);
                else at_odd = find(k * U / 32 + 1);
            }
            issue(k + ST - 1);
            const uint32_t have = there >> ((ST - 1) * U);   // bit U - 1 - u: granule u of this step
            const uint8_t* step = ring + (k % ST) * (U * GB);
            const int t0 = (g0 + U * (wid + k * W)) * 16;

            // ---- scores
            float sc[U][NT][4];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint8_t* gr = step + u * GB;
                uint32_t kw[2][NB];
                float kd[2][NB];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    load_words<NB>(kw[h], gr + (h * 32 + lane) * NB * 4);
                    load_scales<NB>(kd[h], gr + 16 * HD + (h * 8 + g) * NB * 2);
                }
#pragma unroll
                for (int i = 0; i < NB; i++) {
                    const uint32_t w0 = kw[0][i], w1 = kw[1][i], x0 = w0 >> 8, x1 = w1 >> 8;
                    const uint32_t a0[4] = {codes_lo<RAW>(w0, k1024), codes_lo<RAW>(w1, k1024), codes_hi<RAW>(w0, k1024),
                                            codes_hi<RAW>(w1, k1024)};
                    const uint32_t a1[4] = {codes_lo<RAW>(x0, k1024), codes_lo<RAW>(x1, k1024), codes_hi<RAW>(x0, k1024),
                                            codes_hi<RAW>(x1, k1024)};
                    constexpr float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        float acc[4];
                        if constexpr (RAW)
                            mma16816(acc, a0, qf[n][0][2 * i][0], qf[n][0][2 * i][1], corr[n][i]);
                        else
                            mma16816(acc, a0, qf[n][0][2 * i][0], qf[n][0][2 * i][1], none);
                        mma16816(acc, a1, qf[n][0][2 * i + 1][0], qf[n][0][2 * i + 1][1]);
#pragma unroll
                        for (int p = 1; p < PC; p++) {
                            mma16816(acc, a0, qf[n][p][2 * i][0], qf[n][p][2 * i][1]);
                            mma16816(acc, a1, qf[n][p][2 * i + 1][0], qf[n][p][2 * i + 1][1]);
                        }
#pragma unroll
                        for (int x = 0; x < 4; x++)
                            sc[u][n][x] = i ? fmaf(kd[x >> 1][i], acc[x], sc[u][n][x]) : kd[x >> 1][i] * acc[x];
                    }
                }
            }

            // ---- t = (s - m) * fac + P_EXP; is one beyond the slack in m's range?
            float t[U][NT][4];
            constexpr uint32_t ALL = (1u << U) - 1;
            const bool edge = t0 + 16 * U > lim_min || (have & ALL) != ALL;
            auto sees = [&](int u, int n, int x) {   // whether the column's row attends to the lane's token
                return t0 + 16 * u + g + 8 * (x >> 1) < lim[n][x & 1] && (have >> (U - 1 - u) & 1);
            };
            auto place = [&] {
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int x = 0; x < 4; x++) t[u][n][x] = fmaf(sc[u][n][x], fac[n][x & 1], off[n][x & 1]);
                if (edge) {
#pragma unroll
                    for (int u = 0; u < U; u++)
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int x = 0; x < 4; x++)
                                if (!sees(u, n, x)) t[u][n][x] = -INFINITY;
                }
            };
            place();
            float top_t = t[0][0][0];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int x = 0; x < 4; x++) top_t = fmaxf(top_t, t[u][n][x]);
            bool odd = top_t > P_EXP + P_SLACK;

            // ---- V scales: does one not fit, or is not finite?  A word of two for each lane.
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < (NB + 3) / 4; i++) {
                    const int x = 32 * i + lane;
                    if (NB % 4 == 0 || x < 8 * NB) {
                        const uint32_t v = *reinterpret_cast<const uint32_t*>(step + u * GB + 17 * HD + 4 * x) & 0x7fff7fffu;
                        odd |= max(v & 0xffffu, v >> 16) > vlim;
                    }
                }
            bool mend = false;
            if (__any_sync(0xffffffffu, odd)) {
                // What no row of the item sees (an earlier use of the page may have left it) must not choose vexp;
                // nor, beyond fp16 in its units, meet a probability of 0.
                const int left = s_lim[nrows - 1] - t0;
                bool nan = left < 16 * U;
                float top = 0.0f;   // the largest finite one
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int i = 0; i < (NB + 3) / 4; i++) {
                        const int x = 32 * i + lane;
                        if (x < 8 * NB) {
                            uint32_t w = *reinterpret_cast<const uint32_t*>(step + u * GB + 17 * HD + 4 * x);
                            const int seen = left - (16 * u + x / NB * 2);   // of the word's two tokens
                            w = seen >= 2 ? w : seen == 1 ? w & 0xffffu : 0u;
                            const __half2 v = __habs2(as_h2(w));
                            const float v0 = __low2float(v), v1 = __high2float(v);
                            nan |= !(v0 <= 65504.0f) || !(v1 <= 65504.0f);
                            top = fmaxf(top, fmaxf(v0 <= 65504.0f ? v0 : 0.0f, v1 <= 65504.0f ? v1 : 0.0f));
                        }
                    }
                mend = __any_sync(0xffffffffu, nan);
#pragma unroll
                for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                float vf = 1.0f;
                if (top > __half2float(__ushort_as_half((uint16_t)vlim))) {
                    const int e = min(max(ilogbf(top) - V_LOW, -14), 13);
                    vf = scalbnf(1.0f, vexp - e);
                    vexp = e;
                    vmul = __float2half2_rn(scalbnf(1.0f, -e));
                    vlim = V_HIGH + e >= 16 ? 0x7bffu : (uint32_t)__half_as_ushort(__float2half_rn(scalbnf(1.0f, V_HIGH + e)));
                }
                bool beyond = false;
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int k2 = 0; k2 < 2; k2++) {
                        float mn = m[n][k2];
#pragma unroll
                        for (int u = 0; u < U; u++)
#pragma unroll
                            for (int h = 0; h < 2; h++)
                                if (sees(u, n, k2 + 2 * h)) mn = fmaxf(mn, sc[u][n][k2 + 2 * h]);
#pragma unroll
                        for (int x = 16; x >= 4; x >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, x));
                        const float f = mn == m[n][k2] ? 1.0f : ex2((m[n][k2] - mn) * fac[n][k2]);
                        m[n][k2] = mn;
                        const bool far = mn != -INFINITY && fabsf(mn * fac[n][k2]) > FAR;
                        off[n][k2] = far ? INFINITY : P_EXP - mn * fac[n][k2];   // far: every step comes here
                        beyond |= far;
                        l[n][k2] *= f;
                        const float of = f * vf;
#pragma unroll
                        for (int t2 = 0; t2 < 2 * NB; t2++) {
                            o[n][t2][k2] *= of;
                            o[n][t2][k2 + 2] *= of;
                        }
                    }
                }
                place();
                if (__any_sync(0xffffffffu, beyond)) {
#pragma unroll
                    for (int u = 0; u < U; u++)
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int x = 0; x < 4; x++)
                                if (sees(u, n, x)) t[u][n][x] = fmaf(sc[u][n][x] - m[n][x & 1], fac[n][x & 1], P_EXP);
                }
            }

#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint8_t* gr = step + u * GB;
                // ---- p in pieces, transposed: lane (g, c) gets row g's tokens 2c, 2c + 1 of each half
                uint32_t ph[NT][PC][2];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float p[4];
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        p[x] = ex2(t[u][n][x]);
                        l[n][x & 1] += p[x];
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
                uint32_t vd[2][NB], vw[2][NB];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    load_words<NB>(vd[h], gr + 17 * HD + (h * 4 + c) * NB * 4);
                    load_words<NB>(vw[h], gr + 8 * HD + (h * 32 + lane) * NB * 4);
#pragma unroll
                    for (int i = 0; i < NB; i++) vd[h][i] = as_u32(__hmul2(as_h2(vd[h][i]), vmul));
                }
                // a block held as NaN may lie behind a row's limit, where it must not meet even a
                // probability of 0
                auto keep = [&](int n, int h, uint32_t d) {
                    if (!mend) return d;
                    const int seen = lim_g[n] - (t0 + 16 * u + 8 * h + 2 * c);
                    return seen >= 2 ? d : seen == 1 ? d & 0xffffu : 0u;
                };
                if constexpr (NT == 1) {
                    if (mend)
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int i = 0; i < NB; i++) vd[h][i] = keep(0, h, vd[h][i]);
                }
#pragma unroll
                for (int i = 0; i < NB; i++) {
                    const uint32_t w0 = vw[0][i], w1 = vw[1][i], x0 = w0 >> 8, x1 = w1 >> 8;
                    // rows g: the lower nibbles' dimensions; rows g + 8: the upper ones'
                    const uint32_t a0[4] = {codes_lo<false>(w0, k1024), codes_hi<false>(w0, k1024),
                                            codes_lo<false>(w1, k1024), codes_hi<false>(w1, k1024)};
                    const uint32_t a1[4] = {codes_lo<false>(x0, k1024), codes_hi<false>(x0, k1024),
                                            codes_lo<false>(x1, k1024), codes_hi<false>(x1, k1024)};
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        uint32_t pb[PC][2];
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const __half2 d = as_h2(NT == 1 ? vd[h][i] : keep(n, h, vd[h][i])), p0 = as_h2(ph[n][0][h]);
                            const __half2 hi = __hmul2(p0, d);
                            pb[0][h] = as_u32(hi);
                            // what the product lost, and the lower piece's
                            if constexpr (PC == 2)
                                pb[1][h] = as_u32(__hfma2(as_h2(ph[n][1][h]), d, __hfma2(p0, d, __hneg2(hi))));
                        }
#pragma unroll
                        for (int p = 0; p < PC; p++) {
                            mma16816(o[n][2 * i], a0, pb[p][0], pb[p][1]);
                            mma16816(o[n][2 * i + 1], a1, pb[p][0], pb[p][1]);
                        }
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
        const float back = scalbnf(1.0f, vexp - 6);   // out of the units of p and vexp
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
                        row[32 * i + 16 * t + g] = o[n][2 * i + t][k] * back;
                        row[32 * i + 16 * t + 8 + g] = o[n][2 * i + t][k + 2] * back;
                    }
                if (g == 0) {
                    row[HD] = m[n][k] * fac[n][k];
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
    } while (u < u_end);
}

// Adding up the parts of an item: the second slot of the worker w that begins it, then the
// first slots of w + 1, ... up to the item's last.
constexpr int JT = 256, JW = JT / 32;

template <int HD, int ROWS>
__device__ __forceinline__ const float* join_part(const AttnKvqArgs& a, int w, int i, int r) {
    return a.slots + ((size_t)(i == 0 ? 2 * w + 1 : 2 * (w + i)) * ROWS + r) * (HD + 4);
}

// Where row r of the item that begins with head h (kind, token, head, rows) belongs.
template <typename T>
__device__ __forceinline__ T* join_out(const AttnKvqArgs& a, const int4& h, int r) {
    const int rho = h.z % a.R + r;   // query row counted from the first token of the tile
    return reinterpret_cast<T*>(a.out) + (size_t)(h.y + rho / a.R) * a.os +
           (size_t)(h.z / a.R * a.R + rho % a.R) * a.c.hd;
}

// Up to a few parts per item: a CTA per worker, a warp per query row.
template <int DT, int NB, int NT>
__global__ void __launch_bounds__(JT) k_kvq_join(AttnKvqArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int HD = 32 * NB, ROWS = 8 * NT;
    const int w = blockIdx.x, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 h = *reinterpret_cast<const int4*>(a.heads + ((size_t)w * 2 + 1) * 4);
    if (h.x == SLOT_NONE) return;
    for (int r = threadIdx.x >> 5; r < h.w; r += JW) {
        float m = -INFINITY, l = 0.0f, o[NB];
#pragma unroll
        for (int x = 0; x < NB; x++) o[x] = 0.0f;
        for (int i0 = 0;; i0 += 32) {   // 32 parts at a time, a lane looking at each
            const int i = i0 + lane;
            const bool in = w + i < a.workers;
            const int kind = i == 0 ? SLOT_MORE : in ? a.heads[(size_t)(w + i) * 8] : SLOT_LAST;
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (in) ml = *reinterpret_cast<const float2*>(join_part<HD, ROWS>(a, w, i, r) + HD);   // of an empty slot, too
            const unsigned last = __ballot_sync(0xffffffffu, kind != SLOT_MORE);
            const int n = last ? __ffs(last) : 32;
            float mn = lane < n ? ml.x : -INFINITY;
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, x));
            mn = fmaxf(mn, m);
            const float back = mn == m ? 1.0f : ex2(m - mn);
            const float f = lane >= n ? 0.0f : ml.x == mn ? 1.0f : ex2(ml.x - mn);
            m = mn;
            l = fmaf(l, back, lane < n ? f * ml.y : 0.0f);
#pragma unroll
            for (int x = 0; x < NB; x++) o[x] *= back;
#pragma unroll 4
            for (int y = 0; y < n; y++) {
                const float* p = join_part<HD, ROWS>(a, w, i0 + y, r);
                const float fy = __shfl_sync(0xffffffffu, f, y);
#pragma unroll
                for (int x = 0; x < NB; x++) o[x] = fmaf(fy, p[32 * x + lane], o[x]);
            }
            if (last) break;
        }
#pragma unroll
        for (int x = 16; x >= 1; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
        const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
        T* dst = join_out<T>(a, h, r);
#pragma unroll
        for (int x = 0; x < NB; x++) from_f32(o[x] * inv, dst[32 * x + lane]);
    }
}

// Few items of many parts: a CTA per (item, query row), its warps dealing out the parts.
template <int DT, int NB, int NT>
__global__ void __launch_bounds__(JT) k_kvq_join_wide(AttnKvqArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int HD = 32 * NB, ROWS = 8 * NT;
    __shared__ float s_o[JW][HD], s_l[JW], s_m[JW], s_f[MAX_WORKERS];
    __shared__ uint8_t s_kind[MAX_WORKERS], s_tail[MAX_WORKERS];
    __shared__ int s_w, s_n;
    const int item = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int w = tid; w < a.workers; w += JT) {
        s_kind[w] = (uint8_t)a.heads[(size_t)w * 8];
        s_tail[w] = (uint8_t)a.heads[(size_t)w * 8 + 4];
    }
    __syncthreads();
    if (wid == 0) {   // the item'th worker that begins one, and the parts up to the last
        int w = -1, seen = 0, n = 0;
        for (int x = 0; x < a.workers && w < 0; x += 32) {
            const unsigned begins = __ballot_sync(0xffffffffu, x + lane < a.workers && s_tail[x + lane] != SLOT_NONE);
            if (seen + __popc(begins) > item) w = x + __fns(begins, 0, item - seen + 1);
            seen += __popc(begins);
        }
        if (w >= 0) {
            n = 1;
            for (int x = w + 1;; x += 32) {
                const unsigned last = __ballot_sync(0xffffffffu, x + lane >= a.workers || s_kind[x + lane] != SLOT_MORE);
                if (last) {
                    n += __ffs(last);
                    break;
                }
                n += 32;
            }
        }
        if (lane == 0) s_w = w, s_n = n;
    }
    __syncthreads();
    const int w = s_w, n = min(s_n, a.workers - max(w, 0));
    if (w < 0) return;
    const int4 h = *reinterpret_cast<const int4*>(a.heads + ((size_t)w * 2 + 1) * 4);
    if (r >= h.w) return;
    float m = -INFINITY;
    for (int i = tid; i < n; i += JT) m = fmaxf(m, join_part<HD, ROWS>(a, w, i, r)[HD]);
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    if (lane == 0) s_m[wid] = m;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < JW; x++) m = fmaxf(m, s_m[x]);
    float l = 0.0f, o[NB];
    for (int i = tid; i < n; i += JT) {
        const float2 ml = *reinterpret_cast<const float2*>(join_part<HD, ROWS>(a, w, i, r) + HD);
        s_f[i] = ml.x == m ? 1.0f : ex2(ml.x - m);
        l = fmaf(s_f[i], ml.y, l);
    }
#pragma unroll
    for (int x = 0; x < NB; x++) o[x] = 0.0f;
    __syncthreads();
#pragma unroll 8
    for (int i = wid; i < n; i += JW) {
        const float* p = join_part<HD, ROWS>(a, w, i, r);
        const float f = s_f[i];
#pragma unroll
        for (int x = 0; x < NB; x++) o[x] = fmaf(f, p[32 * x + lane], o[x]);
    }
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
    for (int x = 0; x < NB; x++) s_o[wid][32 * x + lane] = o[x];
    if (lane == 0) s_l[wid] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int x = 0; x < JW; x++) l += s_l[x];
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    T* dst = join_out<T>(a, h, r);
    for (int d = tid; d < HD; d += JT) {
        float x = 0.0f;
#pragma unroll
        for (int y = 0; y < JW; y++) x += s_o[y][d];
        from_f32(x * inv, dst[d]);
    }
}

// ---------------------------------------------------------------- launching
// Up to this many query rows per kv head, a worker's warps share an item (one row tile, the
// granules dealt out); with more, every warp is a worker of its own.
constexpr int DEEP_ROWS = 32;
constexpr int MAX_DEV = 64;

// A second tile of 8 query rows takes the same unpacked codes: worth it where there are the
// rows for it and the registers (fp32 holds q and p twice).
constexpr bool two_tiles(int dt, int nb) { return nb <= (dt == TGX_F32 ? 3 : 4); }

struct Shape {
    int warps, nt, workers;
    int wide;   // items for the wide join, 0 for the other
};

// Query rows per kv head that the launch is made for.  Behind the tiles of tg_kvq_tc.cu these are a
// decode step's (sequences that it leaves for their scales may have more, and take longer).
long long shape_rows(const KvqBatch& b, int R, bool left) { return left ? R : (long long)b.max_new * R; }

// Workers and their row tiles for these bounds; at most `have` workers are resident.
Shape shape_of(const KvqCache& c, const KvqBatch& b, long long rows, bool left, bool two, int have_one, int have_deep) {
    Shape sh;
    sh.warps = rows <= DEEP_ROWS ? DEEP_WARPS : 1;
    sh.nt = rows > 8 && two ? 2 : 1;
    // no more workers than there can be granules for their warps
    const long long items = (long long)b.B * c.nkv * ((rows + 8 * sh.nt - 1) / (8 * sh.nt));
    const long long most = items * (((long long)b.max_pages * c.pt + 15) / 16);
    const long long have = sh.warps > 1 ? have_deep : have_one, want = (most + sh.warps - 1) / sh.warps;
    sh.workers = (int)(want < have ? want : have);
    // many parts per item: 14 us -> see k_kvq_join_wide
    sh.wide = items * 16 < sh.workers && !left ? (int)items : 0;   // a bound on the items, so not for what is left
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
cudaError_t launch_attn_t(AttnKvqArgs a, const Shape& sh, cudaStream_t s) {
    a.workers = sh.workers;
    k_kvq_attn<DT, NB, NT><<<sh.workers, 32 * sh.warps, attn_smem<NB, NT>(sh.warps), s>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = sh.wide ? dim3(sh.wide, 8 * NT) : dim3(sh.workers);
    cfg.blockDim = dim3(JT);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, sh.wide ? k_kvq_join_wide<DT, NB, NT> : k_kvq_join<DT, NB, NT>, a);
}

template <int DT, int NB>
cudaError_t launch_attn_nb(AttnKvqArgs a, void* scratch, size_t scratch_bytes, cudaStream_t s) {
    constexpr int NT2 = two_tiles(DT, NB) ? 2 : 1;
    const bool left = a.only != nullptr, nt2 = NT2 == 2 && shape_rows(a.b, a.R, left) > 8;
    const int one = nt2 ? attn_workers<DT, NB, NT2>(1) : attn_workers<DT, NB, 1>(1);
    const int deep = nt2 ? attn_workers<DT, NB, NT2>(DEEP_WARPS) : attn_workers<DT, NB, 1>(DEEP_WARPS);
    if (!one || !deep) return cudaErrorUnknown;
    const Shape sh = shape_of(a.c, a.b, shape_rows(a.b, a.R, left), left, NT2 == 2, one, deep);
    if (scratch_bytes < attn_scratch(sh, a.c.hd)) return cudaErrorInvalidValue;
    a.heads = reinterpret_cast<int*>(scratch);
    a.slots = reinterpret_cast<float*>((uint8_t*)scratch + head_bytes(sh.workers));
    return nt2 ? launch_attn_t<DT, NB, NT2>(a, sh, s) : launch_attn_t<DT, NB, 1>(a, sh, s);
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

cudaError_t launch_attn(int dtype, AttnKvqArgs a, void* scratch, size_t n, cudaStream_t s) {
    if (attn_tc_takes(dtype, a.c, a.b, a.T, a.R)) {
        const size_t tc = attn_tc_scratch(a.c, a.b, a.T, a.R);
        if (n < tc) return cudaErrorInvalidValue;
        cudaError_t e = launch_attn_tc(dtype, a, scratch, &a.only, s);
        if (e != cudaSuccess) return e;
        scratch = (uint8_t*)scratch + tc;
        n -= tc;
    }
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
    const int R = n_heads / c.nkv;
    size_t most = 0;   // of any type, on any device
    for (int two = 0; two < 2; two++)
        for (int left = 0; left < 2; left++)
            most = std::max(most, tg::attn_scratch(tg::shape_of(c, b, tg::shape_rows(b, R, left), left, two,
                                                                tg::MAX_SMS * tg::workers_per_sm(1),
                                                                tg::MAX_SMS * tg::workers_per_sm(tg::DEEP_WARPS)), c.hd));
    return most + tg::attn_tc_scratch(c, b, n_tokens, R);
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
                      q_stride, out, out_stride, sc, 0x64006400u, 0, nullptr, nullptr, nullptr};
    cudaError_t e = tg::launch_attn(dtype, a, scratch, scratch_bytes, (cudaStream_t)stream);
    return e == cudaSuccess ? TG_OK : tg::serve_fail(TG_ECUDA, fn, cudaGetErrorString(e));
}
