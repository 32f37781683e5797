// tg_kvq.cu — appending to the paged 4-bit key/value cache, and reading it back.
//
// Per new token: q and k heads RMS-normalised and rotated, k and v quantised to blocks of
// 32 (m = the value of the largest magnitude, the first of several; scale fp16(m / -8);
// code = min(15, floor(8.5 - 8 x / m))) and written at the token's row of its page.
//
// A code is cut at a border, so a rounding in front of it can move a value by a whole
// step.  Values are exact in 32 bits, and their code comes from an fp32 quotient that is right
// or one too high: the sign of (code - 8.5) m + 8 x, one fused operation, decides.  Keys are the
// definition's in 64 bits: computed in 32 with a bound on the error, and where a code, the
// largest value or the rounding of a scale is within that bound of turning out otherwise (about
// one pair of heads in 20), once more in 64.  All in 64 bits took 141 us for 13077 tokens of 32
// and 4 heads of 128 in bf16, which now take 90.  q has no borders: fp32, rounded once to its type.
//
// 16 lanes per head, 2 NB = HD / 16 dimensions in a row per lane, so the other half of a
// rotated pair is 8 lanes away, and a block of 32 is 16 / NB lanes.  A warp takes pairs of heads
// of one kind of one token: angles and norm weights are loaded once for them.  Bound by instructions
// for many tokens: those 13077 take 69 M warp instructions, 33 issue slots an element of q, k and v,
// where their bytes would take 39 us.  By latency for few.
#include <algorithm>

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
    int per_token;   // warps that share a token's pairs of heads
};

// N elements in a row as floats, and back; 4 at a time (rows are 4-element aligned), 2, or 1.
template <int N, typename T>
__device__ __forceinline__ void load_row(float (&v)[N], const T* p) {
    constexpr int W = N % 4 == 0 ? 4 : N % 2 == 0 ? 2 : 1;
    struct alignas(W * sizeof(T)) Vec { T t[W]; };
#pragma unroll
    for (int i = 0; i < N; i += W) {
        const Vec u = *reinterpret_cast<const Vec*>(p + i);
#pragma unroll
        for (int x = 0; x < W; x++) v[i + x] = to_f32(u.t[x]);
    }
}
// The same for norm weights and angles, which may begin at any element.
template <int N>
__device__ __forceinline__ void load_table(float (&v)[N], const float* p) {
    if ((uintptr_t)p % (N % 4 == 0 ? 16 : 8) == 0) {
        load_row(v, p);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = p[i];
    }
}
template <int N, typename T>
__device__ __forceinline__ void store_row(T* p, const float (&v)[N]) {
    constexpr int W = N % 4 == 0 ? 4 : N % 2 == 0 ? 2 : 1;
    struct alignas(W * sizeof(T)) Vec { T t[W]; };
#pragma unroll
    for (int i = 0; i < N; i += W) {
        Vec u;
#pragma unroll
        for (int x = 0; x < W; x++) from_f32(v[i + x], u.t[x]);
        *reinterpret_cast<Vec*>(p + i) = u;
    }
}

__device__ __forceinline__ float inv_sqrt(float v) { return __fdiv_rn(1.0f, __fsqrt_rn(v)); }
__device__ __forceinline__ double inv_sqrt(double v) { return 1.0 / sqrt(v); }

__device__ __forceinline__ float max_nan(float x, float y) {   // NaN if either is
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}

// x: the lane's N dimensions of a head of 16 lanes; w: their norm weights, or null.  Returns the
// mean square plus eps (1 without a norm).
template <int N, typename T>
__device__ __forceinline__ T norm_head(T (&x)[N], const float* w, float eps) {
    if (!w) return 1;
    T ss = 0;
#pragma unroll
    for (int i = 0; i < N; i++) ss += x[i] * x[i];
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const T mean = ss / (16 * N) + (T)eps, r = inv_sqrt(mean);
    float wn[N];
    load_table(wn, w);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = x[i] * r * (T)wn[i];
    return mean;
}
// cs / sn: the lane's angles.  Returns the largest magnitude of the lane's cosines and sines, 1 at least.
template <int N, typename T>
__device__ __forceinline__ float rotate_head(T (&x)[N], const float* cs, const float* sn, int lane) {
    if (!cs) return 1.0f;
    float c[N], s[N], most = 1.0f;
    load_table(c, cs);
    load_table(s, sn);
#pragma unroll
    for (int i = 0; i < N; i++) most = fmaxf(most, fmaxf(fabsf(c[i]), fabsf(s[i])));
#pragma unroll
    for (int i = 0; i < N; i++) {
        const T y = __shfl_xor_sync(0xffffffffu, x[i], 8);
        const T a = x[i] * (T)c[i], b = y * (T)s[i];
        x[i] = lane & 8 ? a + b : a - b;
    }
    return most;
}

// A code is left in the low bits of 1.5 * 2^23 + code.  Packs a lane's N of them, elements N q and
// on of the block: nibble i of halfword e of word x is element 8i + 2x + e.
template <int N>
__device__ __forceinline__ void pack(uint32_t (&word)[4], const float (&t)[N], int q) {
#pragma unroll
    for (int i = 0; i < 4; i++) word[i] = 0;
    if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2)
            word[i % 8 / 2] |= __byte_perm(__float_as_uint(t[i]), __float_as_uint(t[i + 1]), 0x5410) << (4 * (i / 8));
#pragma unroll
        for (int i = 0; i < 4; i++) word[i] <<= N / 2 * q;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const int dd = N * q + i;
            const uint32_t v = __byte_perm(__float_as_uint(t[i]), __float_as_uint(t[i + 1]), 0x5410) << (4 * (dd / 8));
#pragma unroll
            for (int y = 0; y < 4; y++) word[y] |= y == dd % 8 / 2 ? v : 0u;
        }
    }
}
template <int L>
__device__ __forceinline__ void share(uint32_t (&word)[4]) {   // the whole block's on each of its L lanes
#pragma unroll
    for (int o = 1; o < L; o <<= 1)
#pragma unroll
        for (int i = 0; i < 4; i++) word[i] |= __shfl_xor_sync(0xffffffffu, word[i], o);
}

// The block's codes from its values, N of them in this lane, L lanes in a row per block (a power
// of two), packed; and the scale's bits.  x is exact, or off by up to `off` (FUZZY): `again` then
// says that the exact values may give something else.  T double: x is exact, too.
template <int N, int L, bool FUZZY, typename T>
__device__ __forceinline__ uint16_t quant_block(const T (&x)[N], int lane, uint32_t (&word)[4], float off, bool& again) {
    float f[N], top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        f[i] = (float)x[i];
        top = max_nan(top, fabsf(f[i]));
    }
#pragma unroll
    for (int o = 1; o < L; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    // the first value of that magnitude
    T m = 0;
    bool has = false;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = N - 1; i >= 0; i--)
            if (fabsf(f[i]) == top) m = x[i], has = true;
    } else {   // equal in 32 bits need not be in 64
        T best = -1;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (fabsf(f[i]) == top && fabs(x[i]) > best) best = fabs(x[i]), m = x[i], has = true;
        T most = best;
#pragma unroll
        for (int o = 1; o < L; o <<= 1) most = fmax(most, __shfl_xor_sync(0xffffffffu, most, o));
        has = has && best == most;
    }
    const unsigned who = __ballot_sync(0xffffffffu, has) >> (lane & ~(L - 1)) & (unsigned)((1ull << L) - 1);
    m = __shfl_sync(0xffffffffu, m, (lane & ~(L - 1)) + (who ? __ffs(who) - 1 : 0));
    const __half d = __float2half_rn((float)m * -0.125f);
    const bool bad = !(top <= 3.4028235e38f) || __hisinf(d), plain = !bad && top > 0.0f;
    float wide = 0.0f;   // how far a quotient may be off, beside its own roundings
    if constexpr (FUZZY) {
        // off bounds the roundings of each value, x's and m's; their common factor, 1e-6
        wide = off * __fdiv_rn(16.0f, top);
        const float lo = top * (1.0f - 1e-6f) - off, hi = top * (1.0f + 1e-6f) + off;
        int count = 0;
#pragma unroll
        for (int i = 0; i < N; i++) count += fabsf(f[i]) >= top - 2.0f * off;
        // rivals of the largest in other lanes: smaller ones show there, equal ones here
        again = count > 1 || (count == 1 && !has) || __popc(who) > 1 || !plain || !(top > 1e-20f) ||
                __half_as_ushort(__float2half_rn(lo * 0.125f)) != __half_as_ushort(__float2half_rn(hi * 0.125f));
    }
    constexpr float MAGIC = 12582912.0f;
    // tiny ones out of the way of underflow, exactly
    const bool tiny = !FUZZY && __any_sync(0xffffffffu, top < 1e-20f && top > 0.0f);
    const T up = tiny && top < 1e-20f ? (T)0x1p100 : (T)1;
    const T m8 = m * up * (T)0.125;
    const float inv = plain ? __fdiv_rn(-1.0f, (float)m8) : 0.0f;
    const T sign = m8 > 0 ? (T)1 : (T)-1;
    float t[N], far = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        // floor(8.5 - 8 x / m): that less a half, rounded
        if constexpr (FUZZY) {
            const float v = __fmaf_rn(f[i], inv, 8.0f);
            t[i] = __fadd_rn(v, MAGIC);
            far = fmaxf(far, fabsf(v - __fsub_rn(t[i], MAGIC)));
        } else {
            const T xs = tiny ? x[i] * up : x[i];
            // right, or one more within 1e-4 of the next
            t[i] = __fadd_rn(__fmaf_rn((float)xs, inv, 8.0001f), MAGIC);
            const T over = fma((T)(__fsub_rn(t[i], MAGIC) - 8.5f), m8, xs);
            if (over * sign > 0) t[i] -= 1.0f;
        }
        t[i] = plain ? fminf(fmaxf(t[i], MAGIC), MAGIC + 15.0f) : MAGIC + 8.0f;
    }
    if (FUZZY) again |= far > 0.4999f - wide;
    pack<N>(word, t, lane % L);
    share<L>(word);
    return bad ? (uint16_t)0x7e00 : __half_as_ushort(d);
}

// One block's words and scale into token tk's (of 16) place in its granule.  q: the lane among
// its block's L.
template <int NB, int L, bool K>
__device__ __forceinline__ void put_block(uint8_t* gr, int tk, int b, int q, const uint32_t (&word)[4], uint16_t scale) {
    constexpr int HD = 32 * NB;
    const int h = tk >> 3, c = (tk & 7) >> 1, e = tk & 1;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (i % L != q) continue;
        if constexpr (K) {   // word i belongs to chunk (h, g, i), g the token
            *reinterpret_cast<uint32_t*>(gr + (h * 32 + (tk & 7) * 4 + i) * (HD / 8) + 4 * b) = word[i];
        } else {             // its halfwords to chunks (h, 2i, c) and (h, 2i + 1, c)
            uint8_t* at = gr + 8 * HD + (h * 32 + 8 * i + c) * (HD / 8) + 4 * b + 2 * e;
            *reinterpret_cast<uint16_t*>(at) = (uint16_t)word[i];
            *reinterpret_cast<uint16_t*>(at + HD / 2) = (uint16_t)(word[i] >> 16);
        }
    }
    if (q == 0) {
        uint16_t* scales = reinterpret_cast<uint16_t*>(gr + 16 * HD);
        scales[K ? tk * NB + b : HD / 2 + ((h * 4 + c) * NB + b) * 2 + e] = scale;
    }
}

template <int NB, bool K, typename T>
__device__ __forceinline__ void quant_head(const T (&x)[2 * NB], uint8_t* gr, int tk, int lane, bool put, T* s_x) {
    constexpr int N = 2 * NB;
    uint32_t word[4];
    bool again;
    if constexpr (16 % NB == 0) {
        constexpr int L = 16 / NB;
        const uint16_t d = quant_block<N, L, false>(x, lane, word, 0.0f, again);
        if (put) put_block<NB, L, K>(gr, tk, lane % 16 / L, lane % L, word, d);
    } else {
        // blocks that end inside a lane's dimensions: through shared memory to 2 values of 16 lanes
#pragma unroll
        for (int i = 0; i < N; i++) s_x[lane * N + i] = x[i];
        __syncwarp();
#pragma unroll 1
        for (int b = 0; b < NB; b++) {
            T y[2];
#pragma unroll
            for (int i = 0; i < 2; i++) y[i] = s_x[lane / 16 * 16 * N + 32 * b + lane % 16 * 2 + i];
            const uint16_t d = quant_block<2, 16, false>(y, lane, word, 0.0f, again);
            if (put) put_block<NB, 16, K>(gr, tk, b, lane % 16, word, d);
        }
        __syncwarp();
    }
}

// A key's head in 64 bits.
template <int NB>
__device__ __noinline__ void key_exact(const float (&x)[2 * NB], const float* w, float eps, const float* cs, const float* sn,
                                       uint8_t* gr, int tk, int lane, bool put, double* s_x) {
    double z[2 * NB];
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) z[i] = x[i];
    norm_head(z, w, eps);
    rotate_head(z, cs, sn, lane);
    quant_head<NB, true>(z, gr, tk, lane, put, s_x);
}

// A key's head: in 32 bits where that is sure to give the same.
template <int NB>
__device__ __forceinline__ void key_head(const float (&x)[2 * NB], const float* w, float eps, const float* cs, const float* sn,
                                         uint8_t* gr, int tk, int lane, bool put, double* s_x) {
    bool again = true;
    if constexpr (16 % NB == 0) {
        constexpr int N = 2 * NB, L = 16 / NB;
        float y[N], top = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) y[i] = x[i];
        const float mean = norm_head(y, w, eps);
#pragma unroll
        for (int i = 0; i < N; i++) top = fmaxf(top, fabsf(y[i]));
        top *= rotate_head(y, cs, sn, lane);
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // a value's roundings, each 2^-24: two of the norm on both of the pair (at most top each),
        // two products, a sum of up to 1.5 top: 2 * 3 + 1.5 of them, less than 5e-7 top, where top
        // has the largest cosine or sine as a factor if that is above 1
        uint32_t word[4];
        const uint16_t d = quant_block<N, L, true>(y, lane, word, 5e-7f * top, again);
        // squares next to the smallest numbers have roundings beyond the common factor's 1e-6
        again = __any_sync(0xffffffffu, again || !(mean > 1e-30f));
        if (!again && put) put_block<NB, L, true>(gr, tk, lane % 16 / L, lane % L, word, d);
    }
    if (again) key_exact<NB>(x, w, eps, cs, sn, gr, tk, lane, put, s_x);
}

// Pairs of heads that are under way for a warp, in shared memory.
constexpr int held_pairs(int nb) { return 16 % nb ? 1 : nb <= 4 ? 4 : 2; }

// q: x' = r (x w cos -+ y w' sin), y and w' the pair's other half's.  The products of weights and
// angles are the same for all of a token's heads.  With NB even a lane holds NB dimensions of each
// half (both of every rotated pair), else 2 NB in a row.
template <int NB>
struct QTables {
    static constexpr bool SPLIT = NB % 2 == 0;
    float cl[NB], sl[NB], ch[NB], sh[NB];   // lower' = r (x cl - y sl), upper' = r (y ch + x sh)

    __device__ __forceinline__ static int lower(int l) { return SPLIT ? l * NB : 2 * l * NB; }
    __device__ __forceinline__ static int upper(int l) { return SPLIT ? (16 + l) * NB : (2 * l + 1) * NB; }

    __device__ __forceinline__ void load(const float* cs, const float* sn, const float* w, int l) {
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const int a = lower(l) + i, b = upper(l) + i;
            if constexpr (SPLIT) {
                const float c = cs ? cs[a] : 1.0f, s = cs ? sn[a] : 0.0f, wl = w ? w[a] : 1.0f, wh = w ? w[b] : 1.0f;
                cl[i] = wl * c, sl[i] = wh * s, ch[i] = wh * c, sh[i] = wl * s;
            } else {   // the partner of dimension d is d +- HD / 2, in lane l ^ 8
                const int half = 16 * NB, pa = a < half ? a : a - half, pb = b < half ? b : b - half;
                const float sign = l & 8 ? 1.0f : -1.0f;
                cl[i] = (cs ? cs[pa] : 1.0f) * (w ? w[a] : 1.0f);
                sl[i] = (cs ? sign * sn[pa] : 0.0f) * (w ? w[a < half ? a + half : a - half] : 1.0f);
                ch[i] = (cs ? cs[pb] : 1.0f) * (w ? w[b] : 1.0f);
                sh[i] = (cs ? sign * sn[pb] : 0.0f) * (w ? w[b < half ? b + half : b - half] : 1.0f);
            }
        }
    }
    __device__ __forceinline__ void apply(float (&x)[NB], float (&y)[NB], float r) const {
#pragma unroll
        for (int i = 0; i < NB; i++) {
            if constexpr (SPLIT) {
                const float a = x[i], b = y[i];
                x[i] = r * fmaf(-b, sl[i], a * cl[i]);
                y[i] = r * fmaf(a, sh[i], b * ch[i]);
            } else {
                const float a = __shfl_xor_sync(0xffffffffu, x[i], 8), b = __shfl_xor_sync(0xffffffffu, y[i], 8);
                x[i] = r * fmaf(a, sl[i], x[i] * cl[i]);
                y[i] = r * fmaf(b, sh[i], y[i] * ch[i]);
            }
        }
    }
};

template <int DT, int NB>
__global__ void __launch_bounds__(32 * WARPS, NB <= 4 ? 3 : NB <= 7 ? 2 : 1) k_kvq_append(AppendArgs a) {
    using T = typename Elem<DT>::T;
    using Q = QTables<NB>;
    constexpr int HD = 32 * NB, N = 2 * NB, HELD = held_pairs(NB);
    constexpr int CE = NB % 2 ? 2 : 4, CP = CE * sizeof(T);   // elements and bytes of a copy
    __shared__ __align__(16) T s_row[WARPS][HELD][2 * HD];
    __shared__ double s_buf[16 % NB ? WARPS * 32 * N : 1];
    const int lane = threadIdx.x & 31, l = lane & 15, side = lane >> 4, wid = threadIdx.x >> 5;
    const int qp = (a.NH + 1) / 2, kp = (a.c.nkv + 1) / 2, pairs = qp + 2 * kp, step = a.per_token;
    const uint32_t w = blockIdx.x * WARPS + wid;
    const int t = (int)(w / (uint32_t)step);
    if (t >= a.T) return;
    int p = (int)(w - (uint32_t)t * step);   // pairs p, p + step, ...: of q's heads, k's, v's
    const T* q = reinterpret_cast<const T*>(a.q) + (size_t)t * a.qs;
    const T* k = reinterpret_cast<const T*>(a.k) + (size_t)t * a.ks;
    const T* v = reinterpret_cast<const T*>(a.v) + (size_t)t * a.vs;
    int next = p, slot_in = 0;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(&s_row[wid][0][side * HD + CE * l]);
    auto fetch = [&] {   // the next pair's two rows, 16 lanes each; a head that is not there: the last one's
        if (next < pairs) {
            const bool is_q = next < qp, is_k = next < qp + kp;
            const int head = min(2 * (next - (is_q ? 0 : is_k ? qp : qp + kp)) + side, (is_q ? a.NH : a.c.nkv) - 1);
            const T* from = (is_q ? q : is_k ? k : v) + (CE * l + head * HD);
            const uint32_t to = ring + slot_in * (2 * HD * (int)sizeof(T));
#pragma unroll
            for (int i = 0; i < HD / (16 * CE); i++)
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to + 16 * CP * i), "l"(from + 16 * CE * i), "n"(CP)
                             : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        next += step;
        slot_in = slot_in + 1 == HELD ? 0 : slot_in + 1;
    };
#pragma unroll
    for (int i = 0; i < (HELD > 1 ? HELD - 1 : 1); i++) fetch();
    const KvqPlace at = kvq_place(a.b, a.c, t, lane);
    const int pos = a.positions ? a.positions[t] : (int)at.row;
    bool ok = at.row >= 0;
    if (ok && a.cos && (pos < 0 || pos >= a.n_pos)) {
        if (lane == 0) kvq_flag(a.b, TGX_KVQ_BAD_POSITION);
        ok = false;
    }
    const size_t angle = ok ? (size_t)pos * (HD / 2) : 0;
    const float* cs = a.cos ? a.cos + angle : nullptr;
    const float* sn = a.cos ? a.sin + angle : nullptr;
    Q tab;
    if (p < qp) tab.load(cs, sn, a.q_norm, l);
    T* out = reinterpret_cast<T*>(a.q_out) + ((size_t)t * a.NH + 2 * p + side) * HD;
    double* buf = s_buf + (16 % NB ? wid * 32 * N : 0);
    const bool turns = ok && (a.cos || a.q_norm);   // q is rotated or normalised
    int slot = 0;
#pragma unroll 1
    for (; p < pairs; p += step, slot = slot + 1 == HELD ? 0 : slot + 1) {
        if constexpr (HELD > 1) fetch();
        asm volatile("cp.async.wait_group %0;" ::"n"(HELD - 1) : "memory");
        __syncwarp();
        const T* row = &s_row[wid][slot][side * HD];
        if (!at.mine) {
            // a row behind the last sequence: nothing but the copies to wait for
        } else if (p < qp) {
            float x[NB], y[NB], r = 1.0f;
            load_row(x, row + Q::lower(l));
            load_row(y, row + Q::upper(l));
            if (a.q_norm) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < NB; i++) ss = fmaf(x[i], x[i], fmaf(y[i], y[i], ss));
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                r = rsqrtf(fmaf(ss, 1.0f / HD, a.eps));
            }
            tab.apply(x, y, r);
            if (!turns && ok) {   // as they are: a value must not have met its partner's infinity or NaN times 0
                load_row(x, row + Q::lower(l));
                load_row(y, row + Q::upper(l));
            } else if (!turns) {
#pragma unroll
                for (int i = 0; i < NB; i++) x[i] = y[i] = 0.0f;
            }
            if (2 * p + side < a.NH) {
                store_row(out + Q::lower(l), x);
                store_row(out + Q::upper(l), y);
            }
            out += 2 * step * HD;
        } else if (ok) {
            const bool is_k = p < qp + kp;
            const int head = 2 * (is_k ? p - qp : p - qp - kp) + side;
            uint8_t* gr = kvq_granule(a.c, at.page, min(head, a.c.nkv - 1), at.tok);
            float x[N];
            load_row(x, row + l * N);
            if (is_k)
                key_head<NB>(x, a.k_norm ? a.k_norm + l * N : nullptr, a.eps, cs ? cs + (l & 7) * N : nullptr, sn + (l & 7) * N,
                             gr, at.tok & 15, lane, head < a.c.nkv, buf);
            else
                quant_head<NB, false>(x, gr, at.tok & 15, lane, head < a.c.nkv, reinterpret_cast<float*>(buf));
        }
        __syncwarp();   // the slot is free again
        if constexpr (HELD == 1) fetch();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// A warp takes every per_token'th (key or value, kv head) of a token; lane l holds dimensions
// 32b + l.  A nibble and an element a lane and load: bound by its instructions (13077 tokens of 4
// heads of 128: 20 us, 3.0 TB/s of codes in and fp32 out).
template <int NB>
__global__ void __launch_bounds__(32 * WARPS) k_kvq_read(KvqCache c, KvqBatch bt, int T, int per_token, float* k_out, float* v_out) {
    constexpr int HD = 32 * NB;
    const int lane = threadIdx.x & 31, items = 2 * c.nkv;
    const uint32_t w = blockIdx.x * WARPS + (threadIdx.x >> 5);
    const int t = (int)(w / (uint32_t)per_token);
    if (t >= T) return;
    const KvqPlace p = kvq_place(bt, c, t, lane);
    if (!p.mine) return;
    const int tk = p.tok & 15, h = tk >> 3;
#pragma unroll 4
    for (int it = (int)(w - (uint32_t)t * per_token); it < items; it += per_token) {
        const bool is_k = it < c.nkv;
        float* out = is_k ? k_out : v_out;
        if (!out) continue;
        const int j = is_k ? it : it - c.nkv;
        out += ((size_t)t * c.nkv + j) * HD + lane;
        const uint8_t* gr = kvq_granule(c, p.page, j, p.tok);
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
            out[32 * b] = x;
        }
    }
}

template <int DT, int NB>
cudaError_t launch_append(AppendArgs a, cudaStream_t s) {
    // a warp per pair of heads while that leaves the device room (148 SMs of 24 such warps), down
    // to one per token, for one look-up of the token's place and one set of tables
    const int pairs = (a.NH + 1) / 2 + 2 * ((a.c.nkv + 1) / 2);
    a.per_token = std::max(1, std::min(pairs, 148 * 24 / a.T));
    const unsigned grid = (unsigned)(((long long)a.T * a.per_token + WARPS - 1) / WARPS);
    k_kvq_append<DT, NB><<<grid, 32 * WARPS, 0, s>>>(a);
    return cudaGetLastError();
}

template <int DT>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t s) {
    switch (a.c.hd / 32) {
        case 1: return launch_append<DT, 1>(a, s);
        case 2: return launch_append<DT, 2>(a, s);
        case 3: return launch_append<DT, 3>(a, s);
        case 4: return launch_append<DT, 4>(a, s);
        case 5: return launch_append<DT, 5>(a, s);
        case 6: return launch_append<DT, 6>(a, s);
        case 7: return launch_append<DT, 7>(a, s);
        default: return launch_append<DT, 8>(a, s);
    }
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
    if (!tg::aligned(q_norm, 4) || !tg::aligned(k_norm, 4) || !tg::aligned(rope_cos, 4) || !tg::aligned(rope_sin, 4) ||
        !tg::aligned(positions, 4))
        return tg::serve_fail(TG_EINVAL, fn, "norm weights, angles and positions must be aligned to their elements");
    if ((long long)n_tokens * (n_heads + 2 * cache->n_kv_heads) >= 0x7fff0000ll)
        return tg::serve_fail(TG_EINVAL, fn, "too many tokens for one call");
    tg::ServeDevice dev(fn, cache->pages);
    if (dev.rc != TG_OK || n_tokens == 0) return dev.rc;
    tg::AppendArgs a{tg::kvq_cache(*cache), tg::kvq_batch(*batch), n_tokens, n_heads, q, k, v, q_stride, k_stride,
                     v_stride, q_norm, k_norm, rope_cos, rope_sin, eps, n_pos, positions, q_out, 0};
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
    if ((long long)n_tokens * 2 * cache->n_kv_heads >= 0x7fff0000ll)
        return tg::serve_fail(TG_EINVAL, fn, "too many tokens for one call");
    tg::ServeDevice dev(fn, cache->pages);
    if (dev.rc != TG_OK || n_tokens == 0) return dev.rc;
    const tg::KvqCache c = tg::kvq_cache(*cache);
    const tg::KvqBatch b = tg::kvq_batch(*batch);
    // as many warps per token as fill the device, for one look-up of the token's place in each
    const int per_token = std::max(1, std::min(2 * c.nkv, 148 * 48 / n_tokens));
    const unsigned grid = (unsigned)(((long long)n_tokens * per_token + tg::WARPS - 1) / tg::WARPS);
    cudaStream_t s = (cudaStream_t)stream;
    switch (c.hd / 32) {
#define TG_CASE(n) case n: tg::k_kvq_read<n><<<grid, 32 * tg::WARPS, 0, s>>>(c, b, n_tokens, per_token, k_out, v_out); break;
        TG_CASE(1) TG_CASE(2) TG_CASE(3) TG_CASE(4) TG_CASE(5) TG_CASE(6) TG_CASE(7) TG_CASE(8)
#undef TG_CASE
    }
    SERVE_LAUNCHED(fn);
    return TG_OK;
}
