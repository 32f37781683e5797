// tg_kvq_tc.cu — attention of prompts over the paged 4-bit cache: many query rows per kv head, on
// tcgen05, for 16-bit types and heads of 64 or 128.
//
// A CTA has 256 query rows (new tokens x heads of one kv head) as two tiles of 128, and walks
// the rows they see in tiles of 64 tokens:
//   S = Q K^T     kind::f16, 128 x 64 fp32 in TMEM, two of them per query tile
//   p = 2^(s - m) a thread per query row, reading its TMEM lane; P goes back over S as fp16
//   O += P V      A from TMEM, B the transposed V tile
// Codes are turned into fp16 values once per CTA and tile, code * d rounded to 11 bits, by four
// warps that read the granules straight into registers (the next tile's while this one's are
// converted) and write the 128-byte-swizzled operands; a ring of six slots holds K, V, K, ...
// The layout of the cache makes both K-major operands of 4-byte pieces that 32 lanes store
// without a bank conflict: two dimensions of a token for K, two tokens of a dimension for V.
// The scores of a tile are issued before the softmax of the one in front is waited for, so the
// softmax warps go from tile to tile (with one S per query tile and tiles of 128 tokens they
// waited: 254 us instead of TCUS for three prompts of up to 1500 tokens behind up to 2500).
//
// m moves, and O in TMEM is rescaled, only when a row's scores leave 2^SLACK of it.  q rows, K
// and V are held in fp16 times powers of two: q's largest in 2^13 .. 2^14, the largest scale of
// the sequence's head in 2^7 .. 2^8 (found by k_kvq_scan in front, which also marks sequences
// with a scale that is not finite: a NaN behind a row's limit must not meet a probability of 0,
// so those are left to tg_kvq_attn.cu's kernel).
//
// Every wait is bounded; where one expires the CTA's outputs become NaN.
#include "tg_kvq_attn.cuh"
#include "tg_mbar.cuh"

namespace tg {

namespace {

constexpr int QT = 128;          // query rows of a tile
constexpr int TK = 64;           // tokens of a tile: a granule per conversion warp
constexpr int SLOTS = 6;
constexpr int SW = 8, DW = 4;    // softmax and conversion warps; one more for the MMAs
constexpr int THREADS = 32 * (SW + DW + 1);
constexpr float P_EXP = 6.0f, SLACK = 8.0f;   // p is held times 2^6, and up to 2^14: fp16 reaches 2^16

struct TcArgs {
    AttnKvqArgs a;
    const int* marks;      // [B][nkv]
    const int2* exps;      // [B][nkv] exponents of K and V
};

__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add));
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(
            d),
        "r"(a), "l"(b), "r"(idesc), "r"(add));
}
__device__ __forceinline__ void commit(uint64_t* m) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(saddr(m)) : "memory");
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }   // -126 .. 127

// The largest scale magnitudes of every (sequence, kv head)'s cached rows as exponents, and whether
// one of them is not finite.
__global__ void __launch_bounds__(512) k_kvq_scan(AttnKvqArgs a, int* marks, int2* exps) {
    __shared__ unsigned s_top[2];
    const int j = blockIdx.x, b = blockIdx.y, hd = a.c.hd, nb = hd / 32;
    const SeqInfo si = seq_info(a, b, 2 * QT);
    if (threadIdx.x < 2) s_top[threadIdx.x] = 0;
    __syncthreads();
    const int parts = 2 * hd / 16, gpp = a.c.pt >> 4;   // 16-byte parts of a granule's scales: K's, then V's
    unsigned top[2] = {0, 0};
    if (si.tiles) {
        const long long n = (si.len + 15) / 16 * parts;
#pragma unroll 4
        for (long long x = threadIdx.x; x < n; x += blockDim.x) {
            const int gi = (int)(x / parts), part = (int)(x - (long long)gi * parts), pi = gi / gpp;
            const int page = a.b.table[(size_t)b * a.b.max_pages + pi];
            if (page < 0 || page >= a.c.n_pages) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(kvq_granule(a.c, page, j, (gi - pi * gpp) * 16) + 16 * hd + 16 * part);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            const bool is_v = part >= hd / 16;
            const int left = (int)min(16ll, si.len - 16ll * gi);   // tokens of the granule
            unsigned most = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int at = (is_v ? part - hd / 16 : part) * 8 + i;   // which half of K's or V's
                // V's pairs: [h][c][block][e]
                const int tok = is_v ? at / (2 * nb) * 2 + (at & 1) : at / nb;
                const unsigned u = w[i / 2] >> (16 * (i & 1)) & 0x7fffu;
                if (tok < left) most = max(most, u);
            }
            top[0] = is_v ? top[0] : max(top[0], most);
            top[1] = is_v ? max(top[1], most) : top[1];
        }
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        top[i] = __reduce_max_sync(0xffffffffu, top[i]);
        if ((threadIdx.x & 31) == 0) atomicMax(&s_top[i], top[i]);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int e[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float f = __half2float(__ushort_as_half((unsigned short)min(s_top[i], 0x7bffu)));
            e[i] = f > 0.0f ? max(ilogbf(f) - 7, -14) : 0;
        }
        marks[b * a.c.nkv + j] = s_top[0] >= 0x7c00u || s_top[1] >= 0x7c00u;
        exps[b * a.c.nkv + j] = make_int2(e[0], e[1]);
    }
}

template <int DT, int NB>
__global__ void __launch_bounds__(THREADS, 1) k_kvq_tc(TcArgs t) {
    using T = typename Elem<DT>::T;
    const AttnKvqArgs& a = t.a;
    constexpr int HD = 32 * NB, ATOM = QT * 128;               // bytes of 64 dimensions of 128 rows
    constexpr int Q_BYTES = NB / 2 * ATOM, SLOT = 4096 * NB, K_ATOM = TK * 128;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t q_full, full[SLOTS], empty[SLOTS], s_full[2][2], p_ready[2][2], pv_done[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    __shared__ __align__(4) uint8_t s_valid[8][DW];   // [tile % 8][conversion warp]: whether its granule exists
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, j = blockIdx.y, b = blockIdx.z;

    const SeqInfo si = seq_info(a, b, 2 * QT);
    const int rt = si.tiles - 1 - (int)blockIdx.x;   // the longest first
    if (rt < 0) return;
    for (int x = 0; x < a.c.nkv; x++)
        if (t.marks[b * a.c.nkv + x]) return;
    const int row0 = rt * 2 * QT, nrows = min(2 * QT, si.n * a.R - row0);
    auto limit = [&](int i) { return (int)max(0ll, min(si.len, (long long)si.off + i + 1)); };
    const int seen = limit((row0 + nrows - 1) / a.R), tiles = (seen + TK - 1) / TK;
    const int2 ex = t.exps[b * a.c.nkv + j];
    uint8_t* const s_q = sm;
    uint8_t* const ring = sm + 2 * Q_BYTES;

    if (tid == 0) {
        mbar_init(&q_full, 32 * SW);
        for (int i = 0; i < SLOTS; i++) mbar_init(&full[i], 32 * DW), mbar_init(&empty[i], 1);
        for (int i = 0; i < 2; i++) {
            for (int x = 0; x < 2; x++) mbar_init(&s_full[i][x], 1), mbar_init(&p_ready[i][x], QT);
            mbar_init(&pv_done[i], 1);
        }
        s_failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;");
    }
    if (warp == SW + DW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&s_tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;   // S (and P) of query tile q at 128 q + 64 (tile & 1), O at 256 + 128 q
    volatile int* failed = &s_failed;

    if (warp < SW) {
        // ================================ a thread per query row
        const int q = warp >> 2, r = (warp & 3) * 32 + lane, x0 = q * QT;
        const bool ok = x0 + r < nrows;
        const int rho = row0 + x0 + (ok ? r : 0);
        const int lim = ok ? limit(rho / a.R) : 0x7fffffff;
        const int lim_min = x0 < nrows ? limit((row0 + x0) / a.R) : 0x7fffffff;
        float fac;
        {
            const T* src = reinterpret_cast<const T*>(a.q) + (size_t)(si.s0 + rho / a.R) * a.qs + (size_t)(j * a.R + rho % a.R) * HD;
            auto load4 = [&](float (&v)[4], int d) {
                struct alignas(4 * sizeof(T)) Vec { T t[4]; };
                const Vec u = *reinterpret_cast<const Vec*>(src + d);
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = ok ? to_f32(u.t[i]) : 0.0f;
            };
            float top = 0.0f;
#pragma unroll 8
            for (int d = 0; d < HD; d += 4) {
                float v[4];
                load4(v, d);
                top = fmaxf(fmaxf(top, fmaxf(fabsf(v[0]), fabsf(v[1]))), fmaxf(fabsf(v[2]), fabsf(v[3])));
            }
            // 2^-e: the largest into 2^13 .. 2^14; in two factors, as e reaches beyond fp32's exponents
            const int field = (int)(__float_as_uint(top) >> 23);
            const int e = field == 255 || top == 0.0f ? 0 : max(field - 127, -100) - 13, half = e / 2;
            const float up1 = pow2(-half), up2 = pow2(-(e - half));
            uint8_t* to = s_q + q * Q_BYTES + r * 128;
#pragma unroll 4
            for (int d = 0; d < HD; d += 8) {
                float v[4], w[4];
                load4(v, d);
                load4(w, d + 4);
                uint4 u;
                u.x = as_u32(__floats2half2_rn(v[0] * up1 * up2, v[1] * up1 * up2));
                u.y = as_u32(__floats2half2_rn(v[2] * up1 * up2, v[3] * up1 * up2));
                u.z = as_u32(__floats2half2_rn(w[0] * up1 * up2, w[1] * up1 * up2));
                u.w = as_u32(__floats2half2_rn(w[2] * up1 * up2, w[3] * up1 * up2));
                *reinterpret_cast<uint4*>(to + d / 64 * ATOM + ((d % 64 / 8) ^ (r & 7)) * 16) = u;
            }
            fac = a.scale * pow2(half) * pow2(e - half) * pow2(ex.x);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&q_full);
        }
        const uint32_t s_at = tmem + q * 128 + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t o_at = tmem + 256 + q * 128 + ((uint32_t)((warp & 3) * 32) << 16);
        float m = -INFINITY, off = 0.0f, l = 0.0f;
        bool good = true;
        for (int i = 0; i < tiles && good; i++) {
            good = __all_sync(0xffffffffu, mbar_wait(&s_full[q][i & 1], i >> 1 & 1, failed));
            if (!good) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t have = *reinterpret_cast<const volatile uint32_t*>(s_valid[i & 7]), s_i = s_at + (i & 1) * TK;
            const int t0 = i * TK;
            uint32_t v[2][32];
            tmem_ld<32>(v[0], s_i);
            tmem_ld<32>(v[1], s_i + 32);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            const bool edge = t0 + TK > lim_min || have != 0x01010101u;
            if (edge) {
#pragma unroll
                for (int x = 0; x < TK; x++)   // hidden from the row, or not in the cache
                    if (t0 + x >= lim || !(have >> (x / 16 * 8) & 1)) v[x / 32][x % 32] = __float_as_uint(-INFINITY);
            }
            float top = -INFINITY;
#pragma unroll
            for (int x = 0; x < TK; x++) top = fmaxf(top, __uint_as_float(v[x / 32][x % 32]));
            top = top == -INFINITY ? top : top * fac;
            if (__any_sync(0xffffffffu, top > m + SLACK)) {
                const float mn = fmaxf(m, top), f = mn == m ? 1.0f : ex2(m - mn);
                m = mn;
                off = m == -INFINITY ? 0.0f : P_EXP - m;
                l *= f;
                if (i) {
                    good = __all_sync(0xffffffffu, mbar_wait(&pv_done[q], (i - 1) & 1, failed));   // O is at rest
                    if (!good) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t w[32];
                        tmem_ld<32>(w, o_at + c);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int x = 0; x < 32; x++) w[x] = __float_as_uint(__uint_as_float(w[x]) * f);
                        tmem_st(o_at + c, w);
                    }
                }
            }
            uint32_t p[32];
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < 32; x++) {
                float y[2];
#pragma unroll
                for (int z = 0; z < 2; z++) {
                    const float s = __uint_as_float(v[x / 16][2 * (x % 16) + z]);
                    y[z] = ex2(fmaf(s, fac, off));
                    sum[z] += y[z];
                }
                p[x] = as_u32(__floats2half2_rn(y[0], y[1]));
            }
            l += sum[0] + sum[1];
            tmem_st(s_i, p);   // over scores that have been read
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            mbar_arrive(&p_ready[q][i & 1]);
        }
        if (good && tiles) good = __all_sync(0xffffffffu, mbar_wait(&pv_done[q], (tiles - 1) & 1, failed));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const float inv = !good ? __int_as_float(0x7fc00000) : l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
        const float v2 = pow2(ex.y);
        T* dst = reinterpret_cast<T*>(a.out) + (size_t)(si.s0 + rho / a.R) * a.os + (size_t)(j * a.R + rho % a.R) * HD;
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
            uint32_t v[32];
            if (tiles) {
                tmem_ld<32>(v, o_at + c);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            } else {
#pragma unroll
                for (int x = 0; x < 32; x++) v[x] = 0u;
            }
            if (ok) {
                struct alignas(4 * sizeof(T)) Vec { T t[4]; };
#pragma unroll
                for (int x = 0; x < 32; x += 4) {
                    Vec u;
#pragma unroll
                    for (int y = 0; y < 4; y++) from_f32(__uint_as_float(v[x + y]) * v2 * inv, u.t[y]);
                    *reinterpret_cast<Vec*>(dst + c + x) = u;
                }
            }
        }
    } else if (warp < SW + DW) {
        // ================================ codes into operands: a granule of each tile per warp
        const int dw = warp - SW, g = lane >> 2, c = lane & 3, gpp = a.c.pt >> 4;
        const __half2 kmul = __float2half2_rn(pow2(-ex.x)), vmul = __float2half2_rn(pow2(-ex.y));
        const uint32_t k1024 = a.k1024;
        uint32_t kw[2][NB], vw[2][NB], ks[2][NB / 2], vs[2][NB];   // [half]
        const uint8_t* at = nullptr;
        bool there = true;
        auto find = [&](int i) {   // the tile's granule; none behind the last row that is seen
            const int gi = i * (TK / 16) + dw;
            at = nullptr;
            there = true;
            if (gi * 16 >= seen) return;   // hidden by the rows' limits
            const int pi = gi / gpp, page = a.b.table[(size_t)b * a.b.max_pages + pi];
            there = page >= 0 && page < a.c.n_pages;
            if (there)
                at = kvq_granule(a.c, page, j, (gi - pi * gpp) * 16);
            else if (lane == 0)
                kvq_flag(a.b, TGX_KVQ_BAD_PAGE);
        };
        auto load_k = [&] {
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int y = 0; y < NB; y++) kw[h][y] = 0;
#pragma unroll
                for (int y = 0; y < NB / 2; y++) ks[h][y] = 0;
                if (at) {
                    load_words<NB>(kw[h], at + (h * 32 + lane) * NB * 4);
                    load_words<NB / 2>(ks[h], at + 16 * HD + (h * 8 + g) * NB * 2);
                }
            }
        };
        auto load_v = [&](int i) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int y = 0; y < NB; y++) vw[h][y] = vs[h][y] = 0;
                if (at) {
                    load_words<NB>(vw[h], at + 8 * HD + (h * 32 + lane) * NB * 4);
                    load_words<NB>(vs[h], at + 17 * HD + (h * 4 + c) * NB * 4);
                    // rows behind the last hold anything
                    const long long left = si.len - (i * TK + dw * 16 + 8 * h + 2 * c);
                    if (left < 2)
#pragma unroll
                        for (int y = 0; y < NB; y++) vs[h][y] &= left == 1 ? 0xffffu : 0u;
                }
            }
        };
        int slot = 0;
        uint32_t phase = 1;   // of `empty`: a fresh barrier's wait for it passes
        auto next = [&] {
            if (++slot == SLOTS) slot = 0, phase ^= 1;
        };
        // the lane's four code pairs of a word
        auto codes = [&](uint32_t (&z)[4], uint32_t w) {
            const uint32_t x = w >> 8;
            z[0] = codes_lo<false>(w, k1024), z[1] = codes_hi<false>(w, k1024);
            z[2] = codes_lo<false>(x, k1024), z[3] = codes_hi<false>(x, k1024);
        };
        bool good = true;
        if (tiles) {
            find(0);
            load_k();
        }
        for (int i = 0; i < tiles; i++) {
            load_v(i);
            if (lane == 0) s_valid[i & 7][dw] = there ? 1 : 0;
            good = mbar_wait(&empty[slot], phase, failed);
            if (!good) break;
            uint8_t* to = ring + slot * SLOT;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint8_t* row = to + (dw * 16 + 8 * h + g) * 128 + 4 * c;
#pragma unroll
                for (int y = 0; y < NB; y++) {
                    const __half2 pair = as_h2(ks[h][y / 2]);
                    const __half2 d = __hmul2(y & 1 ? __high2half2(pair) : __low2half2(pair), kmul);
                    uint32_t z[4];
                    codes(z, kw[h][y]);
#pragma unroll
                    for (int n = 0; n < 4; n++)
                        *reinterpret_cast<uint32_t*>(row + y / 2 * K_ATOM + (((y % 2) * 4 + n) ^ g) * 16) = as_u32(__hmul2(as_h2(z[n]), d));
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&full[slot]);
            next();
            if (i + 1 < tiles) {
                find(i + 1);
                load_k();
            }
            good = mbar_wait(&empty[slot], phase, failed);
            if (!good) break;
            to = ring + slot * SLOT;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint8_t* row = to + g * 128 + ((dw * 2 + h) ^ g) * 16 + 4 * c;   // 16 bytes: 8 tokens
#pragma unroll
                for (int y = 0; y < NB; y++) {
                    const __half2 d = __hmul2(as_h2(vs[h][y]), vmul);
                    uint32_t z[4];
                    codes(z, vw[h][y]);
#pragma unroll
                    for (int n = 0; n < 4; n++)
                        *reinterpret_cast<uint32_t*>(row + (32 * y + 8 * n) * 128) = as_u32(__hmul2(as_h2(z[n]), d));
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&full[slot]);
            next();
        }
    } else if (tiles) {
        // ================================ the MMAs
        constexpr uint32_t IDESC_S = (1u << 4) | ((TK >> 3) << 17) | ((QT >> 4) << 24);
        constexpr uint32_t IDESC_O = (1u << 4) | ((HD >> 3) << 17) | ((QT >> 4) << 24);
        const uint64_t dq = sw128_desc(saddr(s_q)), dr = sw128_desc(saddr(ring));
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        // the warp is in step throughout; one lane issues
        auto scores = [&](int q, int i, int slot, bool last) {
            const uint32_t d = tm + q * 128 + (i & 1) * TK;
            const uint64_t x = dq + (q * Q_BYTES >> 4), y = dr + (slot * SLOT >> 4);
            if (elect_one()) {
#pragma unroll
                for (int s = 0; s < 2 * NB; s++)
                    mma_f16_ss(d, x + ((s / 4 * ATOM + s % 4 * 32) >> 4), y + ((s / 4 * K_ATOM + s % 4 * 32) >> 4), IDESC_S, s > 0);
                commit(&s_full[q][i & 1]);
                if (last) commit(&empty[slot]);
            }
            __syncwarp();
        };
        auto values = [&](int q, int i, int slot, bool last) {
            const uint32_t d = tm + 256 + q * 128, x = tm + q * 128 + (i & 1) * TK;
            const uint64_t y = dr + (slot * SLOT >> 4);
            if (elect_one()) {
#pragma unroll
                for (int s = 0; s < TK / 16; s++) mma_f16_ts(d, x + 8 * s, y + (s * 32 >> 4), IDESC_O, i > 0 || s > 0);
                commit(&pv_done[q]);
                if (last) commit(&empty[slot]);
            }
            __syncwarp();
        };
        auto fence = [] { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); };
        int kslot = 0, vslot = 1;                // of K of the next tile, and V of this one
        uint32_t kphase = 0, vphase = 0;
        auto step = [](int& slot, uint32_t& phase) {
            slot += 2;
            if (slot >= SLOTS) slot -= SLOTS, phase ^= 1;
        };
        auto wait = [&](uint64_t* m, uint32_t parity) { return (bool)__all_sync(0xffffffffu, mbar_wait(m, parity, failed)); };
        bool good = wait(&q_full, 0) && wait(&full[0], 0);
        if (good) {
            fence();
            scores(0, 0, 0, false);
            scores(1, 0, 0, true);
            step(kslot, kphase);
        }
        for (int i = 0; i < tiles && good; i++) {
            const bool more = i + 1 < tiles;
            if (more) good = wait(&full[kslot], kphase);
            for (int q = 0; q < 2 && good; q++) {
                if (more) {   // the next scores go into the other half of S, which O's last sum has read
                    fence();
                    scores(q, i + 1, kslot, q == 1);
                }
                good = (q || wait(&full[vslot], vphase)) && wait(&p_ready[q][i & 1], i >> 1 & 1);
                if (!good) break;
                fence();
                values(q, i, vslot, q == 1);
            }
            step(kslot, kphase);
            step(vslot, vphase);
        }
        if (!good) {   // what is under way ends before the TMEM is freed: one more commit behind it all
            if (elect_one()) commit(&q_full);
            const long long t0 = clock64();
            while (!mbar_try(&q_full, 1) && clock64() - t0 < WAIT_CYCLES / 16) {
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == SW + DW) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

size_t r256(size_t n) { return (n + 255) & ~(size_t)255; }

template <int DT, int NB>
cudaError_t launch_tc(const TcArgs& t, cudaStream_t s) {
    constexpr int smem = 2 * (NB / 2) * QT * 128 + SLOTS * 4096 * NB + 1024;
    cudaError_t e = cudaFuncSetAttribute(k_kvq_tc<DT, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const long long rows = (long long)t.a.b.max_new * t.a.R;
    k_kvq_tc<DT, NB><<<dim3((unsigned)((rows + 2 * QT - 1) / (2 * QT)), t.a.c.nkv, t.a.b.B), THREADS, smem, s>>>(t);
    return cudaGetLastError();
}

}  // namespace

// Where a tile of 256 rows is mostly full, and there are CTAs for about half of the SMs: few
// tiles over a long cache are cut along the cache by the other kernel.
bool attn_tc_takes(int dtype, const KvqCache& c, const KvqBatch& b, int R) {
    const long long rows = (long long)b.max_new * R, items = (rows + 2 * QT - 1) / (2 * QT) * c.nkv * b.B;
    return dtype != TGX_F32 && (c.hd == 64 || c.hd == 128) && rows >= QT && items >= 64 && c.nkv <= 65535 && b.B <= 65535;
}

size_t attn_tc_scratch(const KvqCache& c, const KvqBatch& b) {
    return r256((size_t)c.nkv * b.B * 4) + r256((size_t)c.nkv * b.B * 8);
}

cudaError_t launch_attn_tc(int dtype, const AttnKvqArgs& a, void* scratch, const int** only, cudaStream_t s) {
    int* marks = reinterpret_cast<int*>(scratch);
    int2* exps = reinterpret_cast<int2*>((uint8_t*)scratch + r256((size_t)a.c.nkv * a.b.B * 4));
    k_kvq_scan<<<dim3(a.c.nkv, a.b.B), 512, 0, s>>>(a, marks, exps);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const TcArgs t{a, marks, exps};
    *only = marks;   // `only` may be a's own
    if (dtype == TGX_BF16) return a.c.hd == 128 ? launch_tc<TGX_BF16, 4>(t, s) : launch_tc<TGX_BF16, 2>(t, s);
    return a.c.hd == 128 ? launch_tc<TGX_F16, 4>(t, s) : launch_tc<TGX_F16, 2>(t, s);
}

}  // namespace tg
