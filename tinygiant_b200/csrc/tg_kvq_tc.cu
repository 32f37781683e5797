// tg_kvq_tc.cu — attention of prompts over the paged 4-bit cache: many query rows per kv head, on
// tcgen05, for 16-bit types and heads of 64 or 128.
//
// A CTA has 256 query rows (new tokens x heads of one kv head) as two tiles of 128, and walks
// the rows they see in tiles of 64 tokens:
//   S = Q K^T     kind::f16, 128 x 64 fp32 in TMEM, two of them per query tile
//   p = 2^(s - m) a thread per query row, reading its TMEM lane; P goes back over S as fp16
//   O += P V      A from TMEM, B the transposed V tile
// Codes are turned into fp16 values once per CTA and tile, code * d rounded to 11 bits, by eight
// warps, four for K and four for V, that read the granules straight into registers (the next
// tile's while this one's are converted) and write the 128-byte-swizzled operands; a ring of six
// slots holds K, V, K, ...  The layout of the cache makes both K-major operands of 4-byte pieces
// that 32 lanes store without a bank conflict: two dimensions of a token for K, two tokens of a
// dimension for V.  The scores of a tile are issued before the softmax of the one in front is
// waited for, so the softmax warps go from tile to tile.
//
// Three prompts of up to 1500 tokens behind up to 2500 (32 heads over 4 kv heads of 128): 139 us,
// 10 of them k_kvq_scan's and 8 the empty pass of the other kernel.  A pair of tiles takes 1950
// cycles: its MMAs about 64 each whether N is 64 or 128 (1536 in all), its exponentials 1024.
// Measured on the way: 254 us with tiles of 128 tokens and one S per query tile; 246 with four
// conversion warps, query rows read and written a row a thread (34000 cycles before the first
// tile, 7000 now) and a sequence's items next to one another instead of in order of the rows they
// see; 156 with one warp that issues for both query tiles.  Tiles of 128 tokens, which halve the
// score MMAs, measured 157 to 183 us again: without a second S a query tile's softmax and MMAs
// take turns.
//
// m moves, and O in TMEM is rescaled, only when a row's scores leave 2^SLACK of it.  m, l and O are
// fp32.  q rows, K, V and P are held in fp16, the tensor cores' type, 11 bits like the 16-bit inputs (and
// more than bf16's), times powers of two: q's largest in 2^13 .. 2^14, the largest scale of the
// sequence's head in 2^7 .. 2^8, so blocks more than 2^21 below it have fewer bits
// (found by k_kvq_scan in front, which also marks sequences
// with a scale that is not finite: a NaN behind a row's limit must not meet a probability of 0,
// so those are left to tg_kvq_attn.cu's kernel).
//
// Every wait is bounded; where one expires the CTA's outputs become NaN.
#include "tg_kvq_attn.cuh"
#include "tg_mbar.cuh"

namespace tg {

namespace {

constexpr int QT = 128;          // query rows of a tile
constexpr int TK = 64;           // tokens of a tile: K or V of a granule per conversion warp
constexpr int SLOTS = 6;
// A sequence of so few query rows is the other kernel's, which cuts it along the cache: 40 sequences
// of 3000 rows next to a prompt of 1000 take 67 us instead of 138 with 8 query rows, 112 with 32,
// but 175 instead of 139 with 64.
constexpr int FEW = 32;
constexpr int SW = 8, DW = 8;    // softmax and conversion warps; four more, two of them for the MMAs
constexpr int THREADS = 32 * (SW + DW + 4);
constexpr float P_EXP = 6.0f, SLACK = 8.0f;   // p is held times 2^6, and up to 2^14: fp16 reaches 2^16

struct TcArgs {
    AttnKvqArgs a;
    const int* marks;      // [B][nkv]
    const int2* exps;      // [B][nkv] exponents of K and V
    const int2* order;     // the items (sequence, tile of 256 rows) by the rows they see, the most first
    const int* items;      // how many
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
__device__ __forceinline__ void commit(uint32_t m) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(m) : "memory");
}
// Two fp32 numbers an instruction.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t z;
    asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(x), "f"(y));
    return z;
}
__device__ __forceinline__ float2 unpack2(uint64_t x) {
    float2 z;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(z.x), "=f"(z.y) : "l"(x));
    return z;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t z;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(z) : "l"(a), "l"(b), "l"(c));
    return z;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t z;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(z) : "l"(a), "l"(b));
    return z;
}
// The exponent by which a row of q is divided, from its largest magnitude.
__device__ __forceinline__ int q_exp(unsigned top) {
    const int field = (int)(top >> 23);
    return field == 255 || top == 0 ? 0 : max(field - 127, -100) - 13;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }   // -126 .. 127

// Rows of the cache that the last row of tile rt sees.
__device__ __forceinline__ int item_seen(const AttnKvqArgs& a, const SeqInfo& si, int rt) {
    const int last = min((rt + 1) * 2 * QT, si.n * a.R) - 1;
    return (int)max(0ll, min(si.len, (long long)si.off + last / a.R + 1));
}

// The largest scale magnitudes of every (sequence, kv head)'s cached rows as exponents, and whether
// one of them is not finite; and the order of the items: an item's place is the number of those
// that see more.
__global__ void __launch_bounds__(1024) k_kvq_scan(AttnKvqArgs a, int* marks, int2* exps, int2* order, int* items, int cap) {
    __shared__ unsigned s_top[2];
    const int j = blockIdx.x, b = blockIdx.y, hd = a.c.hd, lb = hd == 128 ? 2 : 1;   // 2^lb blocks a row
    const SeqInfo si = seq_info(a, b, 2 * QT);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (j == a.c.nkv) {   // the items of the sequence, a warp each
        const int lane = threadIdx.x & 31, rt_step = blockDim.x / 32;
        for (int rt = threadIdx.x / 32; rt < si.tiles || (b == 0 && rt == threadIdx.x / 32); rt += rt_step) {
            const int mine = rt < si.tiles ? item_seen(a, si, rt) : 0;
            int rank = 0, all = 0;
            for (int x = lane; x < a.b.B; x += 32) {
                const SeqInfo sx = seq_info(a, x, 2 * QT);
                int lo = 0, hi = sx.tiles;   // the first that is in front of mine: they see more and more
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1, see = item_seen(a, sx, mid);
                    const bool front = see > mine || (see == mine && (x < b || (x == b && mid > rt)));
                    if (front)
                        hi = mid;
                    else
                        lo = mid + 1;
                }
                rank += sx.tiles - lo, all += sx.tiles;
            }
            rank = __reduce_add_sync(0xffffffffu, rank), all = __reduce_add_sync(0xffffffffu, all);
            if (lane == 0 && rt < si.tiles && rank < cap) order[rank] = make_int2(b, rt);
            if (threadIdx.x == 0 && b == 0) *items = min(all, cap);   // more than cap: q_start goes back
        }
        return;
    }
    if (threadIdx.x < 2) s_top[threadIdx.x] = 0;
    __syncthreads();
    const int parts = 2 * hd / 16, gpp = a.c.pt >> 4;   // 16-byte parts of a granule's scales: K's, then V's
    unsigned top[2] = {0, 0};
    const bool few = si.n * a.R <= FEW;
    if (!few) {
        // a granule's parts are neighbouring threads'; four granules a thread at a time
        const int per = (int)blockDim.x / parts, part = (int)threadIdx.x % parts, grans = (int)((si.len + 15) / 16);
        const bool is_v = part >= hd / 16;
        unsigned most = 0;
        for (int g0 = (int)threadIdx.x / parts; g0 < grans && (int)threadIdx.x < per * parts; g0 += 4 * per) {
            uint4 v[4];
            int page[4];
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const int gi = g0 + y * per;
                page[y] = gi < grans ? a.b.table[(size_t)b * a.b.max_pages + gi / gpp] : -1;
            }
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const int gi = g0 + y * per;
                v[y] = make_uint4(0, 0, 0, 0);
                if (page[y] >= 0 && page[y] < a.c.n_pages)
                    v[y] = *reinterpret_cast<const uint4*>(kvq_granule(a.c, page[y], j, gi % gpp * 16) + 16 * hd + 16 * part);
            }
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const uint32_t w[4] = {v[y].x, v[y].y, v[y].z, v[y].w};
                const long long left = si.len - 16ll * (g0 + y * per);   // tokens of the granule
                if (left >= 16) {
#pragma unroll
                    for (int i = 0; i < 4; i++) most = max(most, max(w[i] & 0x7fffu, w[i] >> 16 & 0x7fffu));
                    continue;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int at = (is_v ? part - hd / 16 : part) * 8 + i;   // which half of K's or V's
                    // V's pairs: [h][c][block][e]
                    const int tok = is_v ? (at >> (1 + lb)) * 2 + (at & 1) : at >> lb;
                    if (tok < left) most = max(most, w[i / 2] >> (16 * (i & 1)) & 0x7fffu);
                }
            }
        }
        top[0] = is_v ? 0 : most;
        top[1] = is_v ? most : 0;
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
        marks[b * a.c.nkv + j] = few || s_top[0] >= 0x7c00u || s_top[1] >= 0x7c00u;
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
    __shared__ __align__(8) uint64_t s_bars[17 + 2 * SLOTS];
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    __shared__ __align__(4) uint8_t s_valid[8][TK / 16];   // [tile % 8]: whether its granules exist
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t bars = saddr_kept(s_bars), q_full = bars;
    // of tile i, one for the even and one for the odd: a parity tells neighbouring phases apart only, and
    // nothing says that tile i - 2's arrival is there before that of the scores of tile i
    auto pv_done = [&](int q, int i) { return bars + 8 + 8 * q + (i & 1) * (112 + 16 * SLOTS); };
    auto s_full = [&](int q, int i) { return bars + 24 + 16 * q + 8 * (i & 1); };    // of tile i
    auto p_ready = [&](int q, int i) { return bars + 56 + 16 * q + 8 * (i & 1); };
    auto full = [&](int slot) { return bars + 88 + 8 * slot; };
    auto empty = [&](int slot) { return bars + 88 + 8 * SLOTS + 8 * slot; };
    auto o_done = [&](int q) { return bars + 88 + 16 * SLOTS + 8 * q; };   // O's last sum
    auto at_rest = [&](int q) { return bars + 104 + 16 * SLOTS + 8 * q; };  // all that was issued, where a wait failed

    const int item = blockIdx.x / a.c.nkv, j = blockIdx.x % a.c.nkv;   // the longest first
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (item >= *t.items) return;
    const int b = t.order[item].x, rt = t.order[item].y;
    const SeqInfo si = seq_info(a, b, 2 * QT);
    for (int x = 0; x < a.c.nkv; x++)
        if (t.marks[b * a.c.nkv + x]) return;
    const int row0 = rt * 2 * QT, nrows = min(2 * QT, si.n * a.R - row0);
    auto limit = [&](int i) { return (int)max(0ll, min(si.len, (long long)si.off + i + 1)); };
    const int seen = limit((row0 + nrows - 1) / a.R), tiles = (seen + TK - 1) / TK;
    const int2 ex = t.exps[b * a.c.nkv + j];
    uint8_t* const s_q = sm;
    uint8_t* const ring = sm + 2 * Q_BYTES;

    if (tid == 0) {
        mbar_init(&s_bars[0], 32 * SW);
        for (int i = 1; i < 7; i++) mbar_init(&s_bars[i], 1);
        for (int i = 7; i < 11; i++) mbar_init(&s_bars[i], QT);
        for (int i = 0; i < SLOTS; i++) mbar_init(&s_bars[11 + i], 16 * DW), mbar_init(&s_bars[11 + SLOTS + i], 2);
        for (int i = 0; i < 6; i++) mbar_init(&s_bars[11 + 2 * SLOTS + i], 1);
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

    // 640 threads start with 96 registers each (61440): 256 x 120 + 256 x 80 + 128 x 72 are 60416
    if (warp < SW) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
        // ================================ a thread per query row
        const int q = warp >> 2, r = (warp & 3) * 32 + lane, x0 = q * QT;
        const bool ok = x0 + r < nrows;
        const int rho = row0 + (ok ? x0 + r : 0);   // rows behind the last are the item's first, and not written back
        const int lim = ok ? limit(rho / a.R) : 0x7fffffff;
        const int lim_min = x0 < nrows ? limit((row0 + x0) / a.R) : 0x7fffffff;
        constexpr int RPI = 128 / HD, LPR = 32 / RPI;   // rows that a warp reads at once, 4 elements a lane
        const int lr = lane / LPR, ld = lane % LPR * 4; // its row of those, and dimension
        uint8_t* const s_row = s_q + q * Q_BYTES + (r - lane) * 128;   // rows of this warp
        auto piece = [&](int row) { return s_row + row * 128 + ld / 64 * ATOM + ((ld % 64 / 8) ^ (row & 7)) * 16 + (ld & 4) * 2; };
        auto row_at = [&](long long stride) {   // of the thread's row of q or out
            return (si.s0 + rho / a.R) * stride + (j * a.R + rho % a.R) * HD;
        };
        struct alignas(4 * sizeof(T)) Vec { T t[4]; };
        float fac, l;
        {
            unsigned top = 0;
            const int lr = lane / LPR, ld = lane % LPR * 4;   // the lane's row of those, and dimension
            const long long at = row_at(a.qs);
#pragma unroll
            for (int y0 = 0; y0 < LPR; y0 += 16) {
                Vec u[16];
#pragma unroll
                for (int y = 0; y < 16; y++)
                    u[y] = *reinterpret_cast<const Vec*>(reinterpret_cast<const T*>(a.q) + __shfl_sync(0xffffffffu, at, (y0 + y) * RPI + lr) + ld);
#pragma unroll
                for (int y = 0; y < 16; y++) {
                    const int row = (y0 + y) * RPI + lr;
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = to_f32(u[y].t[i]);
                    unsigned most = __float_as_uint(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))));
                    if (RPI == 1) {
                        most = __reduce_max_sync(0xffffffffu, most);
                    } else {
#pragma unroll
                        for (int x = 1; x < LPR; x *= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, x));
                    }
                    // 2^-e: the largest into 2^13 .. 2^14; in two factors, as e reaches beyond fp32's exponents
                    const int e = q_exp(most), half = e / 2;
                    const float up1 = pow2(-half), up2 = pow2(-(e - half));
                    uint2 w;
                    w.x = as_u32(__floats2half2_rn(v[0] * up1 * up2, v[1] * up1 * up2));
                    w.y = as_u32(__floats2half2_rn(v[2] * up1 * up2, v[3] * up1 * up2));
                    *reinterpret_cast<uint2*>(piece(row)) = w;
                    most = __shfl_sync(0xffffffffu, most, lane % RPI * LPR);
                    if (lane / RPI == y0 + y) top = most;   // of the thread's own row
                }
            }
            const int e = q_exp(top), half = e / 2;
            fac = bounded_fac(a.scale * pow2(half) * pow2(e - half) * pow2(ex.x));
            // an infinity's scores may all be -inf, which below is a row without a token to attend to
            l = top >> 23 == 255 && lim > 0 ? __int_as_float(0x7fc00000) : 0.0f;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(q_full);
        }
        const uint32_t s_at = tmem + q * 128 + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t o_at = tmem + 256 + q * 128 + ((uint32_t)((warp & 3) * 32) << 16);
        // in raw scores: the reference m, and from where on they leave its range
        float m = -INFINITY, above = -INFINITY, off = 0.0f;
        bool good = true;
        for (int i = 0; i < tiles && good; i++) {
            good = __all_sync(0xffffffffu, mbar_wait(s_full(q, i), i >> 1 & 1, failed));
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
                asm volatile("");   // a branch: 64 predicated compares cost every tile otherwise
#pragma unroll
                for (int x = 0; x < TK; x++)   // hidden from the row, or not in the cache
                    if (t0 + x >= lim || !(have >> (x / 16 * 8) & 1)) v[x / 32][x % 32] = __float_as_uint(-INFINITY);
            }
            float top = -INFINITY;
#pragma unroll
            for (int x = 0; x < TK; x++) top = fmaxf(top, __uint_as_float(v[x / 32][x % 32]));
            if (__any_sync(0xffffffffu, top > above)) {
                const float mn = fmaxf(m, top), f = mn == m ? 1.0f : ex2((m - mn) * fac);
                m = mn;
                const bool far = __any_sync(0xffffffffu, m != -INFINITY && fabsf(m * fac) > FAR);
                above = far ? -INFINITY : m + __fdividef(SLACK, fac);   // far: every tile comes here
                off = m == -INFINITY ? 0.0f : far ? P_EXP : P_EXP - m * fac;
                l *= f;
                if (i) {
                    good = __all_sync(0xffffffffu, mbar_wait(pv_done(q, i - 1), (i - 1) >> 1 & 1, failed));   // O is at rest
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
                if (far) {
                    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
                    for (int x = 0; x < TK; x++) v[x / 32][x % 32] = __float_as_uint(__uint_as_float(v[x / 32][x % 32]) - base);
                }
            }
            uint32_t p[32];
            uint64_t sum = 0;   // fp32 sums of the even and odd columns
            const uint64_t fac2 = pack2(fac, fac), off2 = pack2(off, off);
#pragma unroll
            for (int x = 0; x < 32; x++) {
                const float2 s = unpack2(fma2(pack2(__uint_as_float(v[x / 16][2 * (x % 16)]), __uint_as_float(v[x / 16][2 * (x % 16) + 1])), fac2, off2));
                const float y0 = ex2(s.x), y1 = ex2(s.y);
                sum = add2(sum, pack2(y0, y1));
                p[x] = as_u32(__floats2half2_rn(y0, y1));
            }
            l += unpack2(sum).x + unpack2(sum).y;
            tmem_st(s_i, p);   // over scores that have been read
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            mbar_arrive(p_ready(q, i));
        }
        // a barrier of its own, which completes once: no phase to take for another
        if (good && tiles) good = __all_sync(0xffffffffu, mbar_wait(o_done(q), 0, failed));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const float inv = !good ? __int_as_float(0x7fc00000) : l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
        const float v2 = pow2(ex.y);
        // through shared memory, where q is done with, so that a warp writes whole rows
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
#pragma unroll
            for (int x = 0; x < 32; x += 8) {
                struct alignas(16) Vec8 { T t[8]; } u;
#pragma unroll
                for (int y = 0; y < 8; y++) from_f32(__uint_as_float(v[x + y]) * v2 * inv, u.t[y]);
                *reinterpret_cast<Vec8*>(s_row + lane * 128 + c / 64 * ATOM + (((c + x) % 64 / 8) ^ (lane & 7)) * 16) = u;
            }
        }
        __syncwarp();
        const long long to = ok ? row_at(a.os) : -1;
#pragma unroll 8
        for (int y = 0; y < LPR; y++) {
            const int row = y * RPI + lr;
            const long long at = __shfl_sync(0xffffffffu, to, row);
            if (at >= 0) *reinterpret_cast<Vec*>(reinterpret_cast<T*>(a.out) + at + ld) = *reinterpret_cast<const Vec*>(piece(row));
        }
    } else if (warp < SW + DW) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        // ================================ codes into operands: K's or V's of a granule per warp and tile
        const int dw = warp - SW, gt = dw & 3, g = lane >> 2, c = lane & 3, gpp = a.c.pt >> 4;
        const bool is_v = dw >= DW / 2;
        const __half2 mul = __float2half2_rn(pow2(is_v ? -ex.y : -ex.x));
        const uint32_t k1024 = a.k1024;
        struct Raw {
            uint32_t w[2][NB], s[2][NB];   // of the granule's two halves: codes, and scales (K's: half as many)
            bool there;
        } cur, nxt;
        // the page table's entry and the granule of its page of the next tile's granule; the page is read a tile ahead
        const int* entry = a.b.table + (size_t)b * a.b.max_pages + gt / gpp;
        int gp = gt % gpp, ahead = gp, page = 0, tok = gt * 16;
        auto read_page = [&](int t) {
            while (ahead >= gpp) ahead -= gpp, entry++;
            page = t < seen ? *entry : 0;   // what lies behind the last row that is seen, the rows' limits hide
        };
        auto load = [&](Raw& x) {
            const bool in = tok < seen;
            x.there = !in || (page >= 0 && page < a.c.n_pages);
            if (!x.there && lane == 0) kvq_flag(a.b, TGX_KVQ_BAD_PAGE);
#pragma unroll
            for (int y = 0; y < 2 * NB; y++) x.w[y / NB][y % NB] = x.s[y / NB][y % NB] = 0;
            if (in && x.there) {
                const uint8_t* at = kvq_granule(a.c, page, j, gp * 16);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (is_v) {
                        load_words<NB>(x.w[h], at + 8 * HD + (h * 32 + lane) * NB * 4);
                        load_words<NB>(x.s[h], at + 17 * HD + (h * 4 + c) * NB * 4);
                    } else {
                        load_words<NB>(x.w[h], at + (h * 32 + lane) * NB * 4);
                        uint32_t (&half)[NB / 2] = reinterpret_cast<uint32_t (&)[NB / 2]>(x.s[h]);
                        load_words<NB / 2>(half, at + 16 * HD + (h * 8 + g) * NB * 2);
                    }
                }
            }
            gp += TK / 16, ahead = gp;
            tok += TK;
            read_page(tok);
            gp = ahead;
        };
        int slot = is_v;
        uint32_t phase = 1;   // of `empty`: a fresh barrier's wait for it passes
        // the lane's four code pairs of a word
        auto codes = [&](uint32_t (&z)[4], uint32_t w) {
            const uint32_t x = w >> 8;
            z[0] = codes_lo<false>(w, k1024), z[1] = codes_hi<false>(w, k1024);
            z[2] = codes_lo<false>(x, k1024), z[3] = codes_hi<false>(x, k1024);
        };
        read_page(tok);
        load(cur);
#pragma unroll 2
        for (int i = 0; i < tiles; i++) {
            load(nxt);
            if (lane == 0 && !is_v) s_valid[i & 7][gt] = cur.there ? 1 : 0;
            if (!mbar_wait(empty(slot), phase, failed)) break;
            if (!is_v) {
                uint8_t* row = ring + slot * SLOT + (gt * 16 + g) * 128 + 4 * c;
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int y = 0; y < NB; y++) {
                        const __half2 pair = as_h2(cur.s[h][y / 2]);
                        const __half2 d = __hmul2(y & 1 ? __high2half2(pair) : __low2half2(pair), mul);
                        uint32_t z[4];
                        codes(z, cur.w[h][y]);
#pragma unroll
                        for (int n = 0; n < 4; n++)
                            *reinterpret_cast<uint32_t*>(row + h * 1024 + y / 2 * K_ATOM + (((y % 2) * 4 + n) ^ g) * 16) = as_u32(__hmul2(as_h2(z[n]), d));
                    }
            } else {
                const long long left = si.len - (i * TK + gt * 16);   // rows behind the last hold anything
                if (left < 16)
#pragma unroll
                    for (int y = 0; y < 2 * NB; y++) {
                        const int t = y / NB * 8 + 2 * c;
                        if (t + 1 >= left) cur.s[y / NB][y % NB] &= t < left ? 0xffffu : 0u;
                    }
                uint8_t* row = ring + slot * SLOT + g * 128 + 4 * c;   // 16 bytes: 8 tokens
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int y = 0; y < NB; y++) {
                        const __half2 d = __hmul2(as_h2(cur.s[h][y]), mul);
                        uint32_t z[4];
                        codes(z, cur.w[h][y]);
#pragma unroll
                        for (int n = 0; n < 4; n++)
                            *reinterpret_cast<uint32_t*>(row + ((gt * 2 + h) ^ g) * 16 + (32 * y + 8 * n) * 128) = as_u32(__hmul2(as_h2(z[n]), d));
                    }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(full(slot));
            if ((slot += 2) >= SLOTS) slot -= SLOTS, phase ^= 1;
            cur = nxt;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp < SW + DW + 2 && tiles) {
            // ================================ the MMAs, a warp per query tile
            const int q = __shfl_sync(0xffffffffu, warp, 0) - SW - DW;
            constexpr uint32_t IDESC_S = (1u << 4) | ((TK >> 3) << 17) | ((QT >> 4) << 24);
            constexpr uint32_t IDESC_O = (1u << 4) | ((HD >> 3) << 17) | ((QT >> 4) << 24);
            const uint64_t dq = sw128_desc(saddr(s_q)), dr = sw128_desc(saddr(ring));
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            // the warp is in step throughout; one lane issues
            auto scores = [&](int i, int slot) {
                const uint32_t d = tm + q * 128 + (i & 1) * TK;
                const uint64_t x = dq + (q * Q_BYTES >> 4), y = dr + (slot * SLOT >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int s = 0; s < 2 * NB; s++)
                        mma_f16_ss(d, x + ((s / 4 * ATOM + s % 4 * 32) >> 4), y + ((s / 4 * K_ATOM + s % 4 * 32) >> 4), IDESC_S, s > 0);
                    commit(s_full(q, i));
                    commit(empty(slot));
                }
                __syncwarp();
            };
            auto values = [&](int i, int slot) {
                const uint32_t d = tm + 256 + q * 128, x = tm + q * 128 + (i & 1) * TK;
                const uint64_t y = dr + (slot * SLOT >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int s = 0; s < TK / 16; s++) mma_f16_ts(d, x + 8 * s, y + (s * 32 >> 4), IDESC_O, i > 0 || s > 0);
                    commit(pv_done(q, i));
                    if (i + 1 == tiles) commit(o_done(q));
                    commit(empty(slot));
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
            auto wait = [&](uint32_t m, uint32_t parity) { return (bool)__all_sync(0xffffffffu, mbar_wait(m, parity, failed)); };
            bool good = wait(q_full, 0) && wait(full(0), 0);
            if (good) {
                fence();
                scores(0, 0);
                step(kslot, kphase);
            }
            for (int i = 0; i < tiles && good; i++) {
                if (i + 1 < tiles) {   // the next scores go into the other half of S, which O's last sum has read
                    good = wait(full(kslot), kphase);
                    if (!good) break;
                    fence();
                    scores(i + 1, kslot);
                }
                good = wait(full(vslot), vphase) && wait(p_ready(q, i), i >> 1 & 1);
                if (!good) break;
                fence();
                values(i, vslot);
                step(kslot, kphase);
                step(vslot, vphase);
            }
            if (!good) {   // what is under way ends before the TMEM is freed: one more commit behind it all
                if (elect_one()) commit(at_rest(q));
                const long long t0 = clock64();
                while (!mbar_try(at_rest(q), 0) && clock64() - t0 < WAIT_CYCLES) {
                }
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == SW + DW) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

size_t r256(size_t n) { return (n + 255) & ~(size_t)255; }

// Items that T tokens of B sequences have at most.
long long item_cap(const KvqBatch& b, int T, int R) { return (long long)T * R / (2 * QT) + b.B; }

template <int DT, int NB>
cudaError_t launch_tc(const TcArgs& t, cudaStream_t s) {
    constexpr int smem = 2 * (NB / 2) * QT * 128 + SLOTS * 4096 * NB + 1024;
    cudaError_t e = cudaFuncSetAttribute(k_kvq_tc<DT, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(item_cap(t.a.b, t.a.T, t.a.R) * t.a.c.nkv));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_kvq_tc<DT, NB>, t);
}

}  // namespace

// Where a tile of 256 rows is mostly full, and there are CTAs for about half of the SMs: few
// tiles over a long cache are cut along the cache by the other kernel.
bool attn_tc_takes(int dtype, const KvqCache& c, const KvqBatch& b, int T, int R) {
    const long long rows = (long long)b.max_new * R, items = (rows + 2 * QT - 1) / (2 * QT) * c.nkv * b.B;
    return dtype != TGX_F32 && (c.hd == 64 || c.hd == 128) && rows >= QT && items >= 64 && c.nkv <= 65535 && b.B <= 65535 &&
           item_cap(b, T, R) * c.nkv <= 0x7fffffff;
}

size_t attn_tc_scratch(const KvqCache& c, const KvqBatch& b, int T, int R) {
    return r256((size_t)c.nkv * b.B * 4) + r256((size_t)c.nkv * b.B * 8) + r256((size_t)item_cap(b, T, R) * 8) + 256;
}

cudaError_t launch_attn_tc(int dtype, const AttnKvqArgs& a, void* scratch, const int** only, cudaStream_t s) {
    uint8_t* at = (uint8_t*)scratch;
    auto take = [&](size_t n) {
        void* p = at;
        at += r256(n);
        return p;
    };
    const int cap = (int)item_cap(a.b, a.T, a.R);
    int* marks = (int*)take((size_t)a.c.nkv * a.b.B * 4);
    int2* exps = (int2*)take((size_t)a.c.nkv * a.b.B * 8);
    int2* order = (int2*)take((size_t)cap * 8);
    int* items = (int*)take(4);
    k_kvq_scan<<<dim3(a.c.nkv + 1, a.b.B), 1024, 0, s>>>(a, marks, exps, order, items, cap);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const TcArgs t{a, marks, exps, order, items};
    *only = marks;   // `only` may be a's own
    if (dtype == TGX_BF16) return a.c.hd == 128 ? launch_tc<TGX_BF16, 4>(t, s) : launch_tc<TGX_BF16, 2>(t, s);
    return a.c.hd == 128 ? launch_tc<TGX_F16, 4>(t, s) : launch_tc<TGX_F16, 2>(t, s);
}

}  // namespace tg
