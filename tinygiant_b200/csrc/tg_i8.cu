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
#include "tg_serve.cuh"

namespace tg {

namespace {

constexpr int QT = 256;   // threads of the row quantiser

struct QuantArgs {
    const void* x;
    long long xs;
    int rows, cols, kp;
    const float* norm;
    float eps;
    int8_t* codes;
    float* scales;
};

// rint(127 y / top) for y = x (or x * w, unrounded), |y| <= top, in exact arithmetic: the
// fp32 quotient is off by less than 2^-15, so only values that close to a border need the
// 64-bit one (127 x is exact there; x * w * 127 and the quotient round at 2^-53).
__device__ __forceinline__ int i8_code(float x, float w, double top, float inv) {
    const float r = x * w * inv;
    const float c = rintf(r);
    if (fabsf(fabsf(r - c) - 0.5f) > 1e-3f) return (int)c;
    return (int)rint((double)x * w * 127.0 / top);
}

template <int DT, bool NORM>
__global__ void __launch_bounds__(QT) k_i8_rows(QuantArgs a) {
    using T = typename Elem<DT>::T;
    __shared__ double s_top[QT / 32];
    __shared__ float s_ss[QT / 32];
    __shared__ int s_bad;
    const int row = blockIdx.x, tid = threadIdx.x;
    const T* x = reinterpret_cast<const T*>(a.x) + (size_t)row * a.xs;
    double top = 0.0;
    float ss = 0.0f;
    bool bad = false;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    for (int i = tid; i < a.cols; i += QT) {
        const float v = to_f32(x[i]);
        bad |= !(fabsf(v) <= 3.4028235e38f);
        double y = v;
        if (NORM) {
            const float w = a.norm[i];
            bad |= !(fabsf(w) <= 3.4028235e38f);
            y *= w;
            ss += v * v;
        }
        top = fmax(top, fabs(y));
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    if (bad) s_bad = 1;
    if ((tid & 31) == 0) {
        s_top[tid >> 5] = top;
        s_ss[tid >> 5] = ss;
    }
    __syncthreads();
    ss = 0.0f;
#pragma unroll
    for (int i = 0; i < QT / 32; i++) {
        top = fmax(top, s_top[i]);
        ss += s_ss[i];
    }
    bad = s_bad || !(top <= 3.4028234663852886e38);
    const float topf = __double2float_rn(top), inv = __fdiv_rn(127.0f, topf);
    int8_t* out = a.codes + (size_t)row * a.kp;
    // 127 / top overflows for a top this small: quotients then come from 64 bits
    const bool tiny = !(inv <= 3.4028235e38f);
    for (int i = tid; i < a.kp; i += QT) {
        int c = 0;
        if (i < a.cols && !bad && top > 0.0) {
            const float v = to_f32(x[i]), w = NORM ? a.norm[i] : 1.0f;
            c = tiny ? (int)rint((double)v * w * 127.0 / top) : i8_code(v, w, top, inv);
        }
        out[i] = (int8_t)c;
    }
    if (tid == 0) {
        float s = __fdiv_rn(topf, 127.0f);
        if (NORM) s *= __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)a.cols), a.eps)));
        a.scales[row] = bad ? __int_as_float(0x7fc00000) : s;
    }
}

struct MatArgs {
    const int8_t* a;
    const float* sa;
    const int8_t* w;
    const float* sw;
    int M, N, kp;
    const void* res;
    long long rs;
    void* out;
    long long os;
};

template <int DT>
__global__ void __launch_bounds__(256) k_i8_dot(MatArgs g) {
    using T = typename Elem<DT>::T;
    const int lane = threadIdx.x & 31, n = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (n >= g.N) return;
    for (int m = blockIdx.y; m < g.M; m += gridDim.y) {
        const int4* a = reinterpret_cast<const int4*>(g.a + (size_t)m * g.kp);
        const int4* w = reinterpret_cast<const int4*>(g.w + (size_t)n * g.kp);
        int acc = 0;
        for (int i = lane; i < g.kp / 16; i += 32) {
            const int4 u = a[i], v = w[i];
            acc = __dp4a(u.x, v.x, acc);
            acc = __dp4a(u.y, v.y, acc);
            acc = __dp4a(u.z, v.z, acc);
            acc = __dp4a(u.w, v.w, acc);
        }
        acc = __reduce_add_sync(0xffffffffu, acc);
        if (lane == 0) {
            float o = (float)acc * (g.sa[m] * g.sw[n]);
            if (g.res) o += to_f32(reinterpret_cast<const T*>(g.res)[(size_t)m * g.rs + n]);
            from_f32(o, reinterpret_cast<T*>(g.out)[(size_t)m * g.os + n]);
        }
    }
}

template <int DT>
cudaError_t launch_rows(const QuantArgs& a, cudaStream_t s) {
    if (a.norm)
        k_i8_rows<DT, true><<<a.rows, QT, 0, s>>>(a);
    else
        k_i8_rows<DT, false><<<a.rows, QT, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_rows(int dtype, const QuantArgs& a, cudaStream_t s) {
    return dtype == TGX_F32 ? launch_rows<TGX_F32>(a, s)
                            : dtype == TGX_BF16 ? launch_rows<TGX_BF16>(a, s) : launch_rows<TGX_F16>(a, s);
}

size_t r256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

}  // namespace tg

extern "C" size_t tgx_i8_row_bytes(int cols) { return cols > 0 && cols <= 131072 ? ((size_t)cols + 15) & ~(size_t)15 : 0; }

extern "C" int tgx_i8_quantize_rows(int dtype, const void* x, long long x_stride, int rows, int cols,
                                    const float* norm_w, float eps, int8_t* codes, float* scales, void* stream) {
    const char* fn = "tgx_i8_quantize_rows";
    if (!x || !codes || !scales) return tg::serve_fail(TG_EINVAL, fn, "null pointer");
    if (dtype < TGX_F32 || dtype > TGX_F16) return tg::serve_fail(TG_EINVAL, fn, "unknown dtype");
    if (rows < 0 || !tgx_i8_row_bytes(cols) || x_stride < cols || !(eps >= 0.0f))
        return tg::serve_fail(TG_EINVAL, fn, "bad rows, cols (1 .. 131072), stride or eps");
    if (!tg::aligned(codes, 16) || !tg::aligned(x, tg::elem_bytes(dtype)))
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
    if (dtype < TGX_F32 || dtype > TGX_F16) return tg::serve_fail(TG_EINVAL, fn, "unknown dtype");
    if (m < 0 || n <= 0 || !tgx_i8_row_bytes(k) || x_stride < k || out_stride < n || (residual && res_stride < n) ||
        !(eps >= 0.0f))
        return tg::serve_fail(TG_EINVAL, fn, "bad m, n, k (1 .. 131072), stride or eps");
    const size_t e1 = tg::elem_bytes(dtype);
    if (!tg::aligned(w_codes, 16) || !tg::aligned(x, e1) || !tg::aligned(out, e1) || !tg::aligned(residual, e1))
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
    tg::MatArgs g{codes, scales, w_codes, w_scales, m, n, kp, residual, res_stride, out, out_stride};
    const dim3 grid((n + 7) / 8, m < 4096 ? m : 4096);
    if (dtype == TGX_F32)
        tg::k_i8_dot<TGX_F32><<<grid, 256, 0, s>>>(g);
    else if (dtype == TGX_BF16)
        tg::k_i8_dot<TGX_BF16><<<grid, 256, 0, s>>>(g);
    else
        tg::k_i8_dot<TGX_F16><<<grid, 256, 0, s>>>(g);
    SERVE_LAUNCHED(fn);
    return TG_OK;
}
