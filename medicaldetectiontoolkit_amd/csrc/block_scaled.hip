// block_scaled.hip -- tensors into 8-bit and 4-bit block-scaled codes and back, and the convolution epilogue that keeps an 8-bit copy (gfx950).
//
// All of it is HBM-bound streaming: a block of 32 values is held by 8 lanes (4 fp32 values each) or 4 lanes (8 values of 16 bits each), 16 bytes a
// lane and load, and its maximum is two quad permutes (and one half-row mirror) of the lanes' own maxima -- no LDS, no second pass over the data.  What they reach (a copy of
// 1 GiB: 5.0 TB/s, read and written): 5.5 TB/s for the epilogue and the read-back of 75.5 M values with a residual (192 + 58 us), 5.7 for 94 M 16-bit values into 4 bits and back
// (48 + 38 us).
#include "block_scaled.h"

namespace {

using namespace mdt_bs;

constexpr int THREADS = 256;

// GV values from index i on, zero behind n
template <typename T>
__device__ __forceinline__ void load_group(const T *__restrict__ x, long long i, long long n, float (&v)[Io<T>::GV])
{
    constexpr int GV = Io<T>::GV;
    if (i + GV <= n) {
        const typename Io<T>::vec t = *reinterpret_cast<const typename Io<T>::vec *>(x + i);
#pragma unroll
        for (int k = 0; k < GV; ++k) v[k] = Io<T>::to_f(t[k]);
    } else {
#pragma unroll
        for (int k = 0; k < GV; ++k) v[k] = i + k < n ? Io<T>::to_f(x[i + k]) : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store_group(T *__restrict__ x, long long i, long long n, const T (&v)[Io<T>::GV])
{
    constexpr int GV = Io<T>::GV;
    if (i + GV <= n) {
        typename Io<T>::vec t;
#pragma unroll
        for (int k = 0; k < GV; ++k) t[k] = v[k];
        *reinterpret_cast<typename Io<T>::vec *>(x + i) = t;
    } else {
#pragma unroll
        for (int k = 0; k < GV; ++k) if (i + k < n) x[i + k] = v[k];
    }
}

// one lane's GV values (of a block held by 32 / GV lanes) -> its codes, and the block's scale byte by the first of the lanes
template <int GV, bool RELU>
__device__ __forceinline__ void quantize8_group(const float (&v)[GV], long long i, long long n, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales)
{
    unsigned mb = 0;
#pragma unroll
    for (int k = 0; k < GV; ++k) {
        const float t = RELU && v[k] < 0.0f ? 0.0f : v[k];
        mb = umax(mb, __float_as_uint(t) & 0x7fffffffu);
    }
    mb = group_max<BLOCK / GV>(mb);
    const int b = scale_byte<typename std::conditional<RELU, Q255, Q127>::type>(mb);
    const float inv = inv_scale(b == 255 ? 0 : b);
    unsigned w[GV / 4];
#pragma unroll
    for (int q = 0; q < GV / 4; ++q) {
        w[q] = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float x = v[q * 4 + k];
            int c;
            if (RELU) {
                c = (int)rintf((x > 0.0f ? x : 0.0f) * inv);
                c = x > 0.0f && c < 1 ? 1 : c;
                if (b == 255) c = x > 0.0f ? 1 : 0;
            } else {
                c = b == 255 ? 0 : (int)rintf(x * inv);
            }
            w[q] |= ((unsigned)c & 255u) << (8 * k);
        }
    }
    if (i + GV <= n) {
        typedef unsigned uvec __attribute__((ext_vector_type(GV / 4), aligned(4)));
        uvec t;
#pragma unroll
        for (int q = 0; q < GV / 4; ++q) t[q] = w[q];
        *reinterpret_cast<uvec *>(codes + i) = t;
    } else {
#pragma unroll
        for (int k = 0; k < GV; ++k) if (i + k < n) codes[i + k] = (uint8_t)(w[k / 4] >> (8 * (k % 4)));
    }
    if (i % BLOCK == 0 && i < n) scales[i / BLOCK] = (uint8_t)b;
}

// One group a thread: 75.5 M fp32 values in 67 us, 5.7 TB/s, and of 16 bits in 38 (4 groups a thread: 67 and 41).
template <typename T, bool RELU>
__global__ __launch_bounds__(THREADS) void act8_quantize_kernel(const T *__restrict__ x, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, long long n)
{
    constexpr int GV = Io<T>::GV;
    const long long i = ((long long)blockIdx.x * THREADS + threadIdx.x) * GV;
    float v[GV];
    load_group<T>(x, i, n, v);
    quantize8_group<GV, RELU>(v, i, n, codes, scales);
}

// U groups a thread, loaded before the first is used
template <typename T, bool RELU, int U>
__global__ __launch_bounds__(THREADS) void act8_restore_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, T *__restrict__ x, long long n)
{
    constexpr int GV = Io<T>::GV;
    typedef unsigned uvec __attribute__((ext_vector_type(GV / 4), aligned(4)));
    const long long g0 = (long long)blockIdx.x * (THREADS * U) + threadIdx.x;
    unsigned w[U][GV / 4];
    int b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = (g0 + u * THREADS) * GV;
        b[u] = i < n ? scales[i / BLOCK] : 0;
        if (i + GV <= n) {
            const uvec t = *reinterpret_cast<const uvec *>(codes + i);
#pragma unroll
            for (int q = 0; q < GV / 4; ++q) w[u][q] = t[q];
        } else {
#pragma unroll
            for (int q = 0; q < GV / 4; ++q) {
                w[u][q] = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) if (i + q * 4 + k < n) w[u][q] |= (unsigned)codes[i + q * 4 + k] << (8 * k);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        T v[GV];
#pragma unroll
        for (int k = 0; k < GV; ++k) {
            const unsigned c = w[u][k / 4] >> (8 * (k % 4)) & 255u;
            v[k] = read_back<T>(RELU ? (float)c : (float)(int8_t)c, b[u]);
        }
        store_group<T>(x, (g0 + u * THREADS) * GV, n, v);
    }
}

// y = act((x + bias) + residual), rounded to fp32 after each sum as mdt_bias_act_forward does, and y's codes.  Channel of element i: CL i % C, else
// (i / inner) % C; the workgroup's first element is divided in 64 bits once, the rest by multiplication.  y may alias x and the residual.
template <bool CL, bool RES, bool RELU, int U>
__global__ __launch_bounds__(THREADS) void bias_act_act8_kernel(float *y, const float *x, const float *__restrict__ bias, const float *res, uint8_t *__restrict__ codes,
                                                                uint8_t *__restrict__ scales, long long n, long long inner, FastDiv fc, FastDiv fi)
{
    const long long i0 = (long long)blockIdx.x * (THREADS * U * 4);
    const unsigned C = fc.d;
    const unsigned q0 = CL ? (unsigned)(i0 % C) : (unsigned)(i0 / inner % C), r0 = CL ? 0u : (unsigned)(i0 % inner);
    float v[U][4], r[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = i0 + (u * THREADS + threadIdx.x) * 4;
        load_group<float>(x, i, n, v[u]);
        if (RES) load_group<float>(res, i, n, r[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned l = (u * THREADS + threadIdx.x) * 4;
        const long long i = i0 + l;
        unsigned c = 0;
        if (CL) { c = q0 + l; c -= fc.div(c) * C; }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (!CL) { c = q0 + fi.div(r0 + l + k); c -= fc.div(c) * C; }
            float t = v[u][k] + bias[c];
            if (RES) t = t + r[u][k];
            if (RELU) t = t > 0.0f ? t : 0.0f;
            v[u][k] = i + k < n ? t : 0.0f;
            if (CL) c = c + 1 == C ? 0 : c + 1;
        }
        store_group<float>(y, i, n, v[u]);
        quantize8_group<4, RELU>(v[u], i, n, codes, scales);
    }
}

// ---- 4 bits ------------------------------------------------------------------------------------------------------------------------

// rows of k values, cut into blocks of their own (the last one padded with zeros): group g of a row's kb * (32 / GV) belongs to row g / groups.  75.5 M fp32 values in
// 60 us, 5.7 TB/s (4 groups a thread: 61).
template <typename T>
__global__ __launch_bounds__(THREADS) void mx4_quantize_kernel(const T *__restrict__ x, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, long long row0, unsigned total,
                                                               long long k, FastDiv groups)
{
    constexpr int GV = Io<T>::GV, LPB = BLOCK / GV;
    const unsigned g = blockIdx.x * THREADS + threadIdx.x, row = groups.div(g), col = (g - row * groups.d) * GV;
    float v[GV] = {};
    if (g < total) load_group<T>(x + (row0 + row) * k, col, k, v);
    int b;
    const unsigned w = quantize4_group<GV>(v, b);
    if (g >= total) return;
    const long long at = row0 * groups.d + g;                                    // groups of all rows are consecutive: GV / 2 bytes each
    if (GV == 8) reinterpret_cast<unsigned *>(codes)[at] = w;
    else reinterpret_cast<uint16_t *>(codes)[at] = (uint16_t)w;
    if (g % LPB == 0) scales[at / LPB] = (uint8_t)b;
}

template <typename T, int U>
__global__ __launch_bounds__(THREADS) void mx4_dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, T *__restrict__ x, long long row0,
                                                                 unsigned total, long long k, FastDiv groups)
{
    constexpr int GV = Io<T>::GV, LPB = BLOCK / GV;
    const unsigned g0 = blockIdx.x * (THREADS * U) + threadIdx.x;
    unsigned w[U];
    int b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned g = g0 + u * THREADS;
        w[u] = 0;
        b[u] = 0;
        if (g < total) {
            const long long at = row0 * groups.d + g;
            w[u] = GV == 8 ? reinterpret_cast<const unsigned *>(codes)[at] : reinterpret_cast<const uint16_t *>(codes)[at];
            b[u] = scales[at / LPB];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned g = g0 + u * THREADS, row = groups.div(g), col = (g - row * groups.d) * GV;
        if (g >= total) continue;
        v2f p[4];
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 0);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 1);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 2);
        p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 3);
        T v[GV];
#pragma unroll
        for (int j = 0; j < GV; ++j) v[j] = read_back<T>(p[j / 2][j % 2], b[u]);
        if (col < k) store_group<T>(x + (row0 + row) * k, col, k, v);
    }
}

// Where codes are read or the epilogue adds a second stream, 4 groups a thread keep enough loads in flight on a full card (75.5 M values: restore 80 -> 66 us, 4 bits to fp32
// 100 -> 76, the epilogue 153 -> 128); a small tensor is spread over more workgroups instead (4 M values: 6 us either way, the launch).
constexpr long long FULL = 256LL * 8 * THREADS * 4;

template <typename T>
int quantize8(const void *x, uint8_t *codes, uint8_t *scales, long long n, int relu, hipStream_t s)
{
    const long long groups = (n + BLOCK - 1) / BLOCK * (BLOCK / Io<T>::GV);
    const dim3 grid((unsigned)((groups + THREADS - 1) / THREADS));
    if (relu) act8_quantize_kernel<T, true><<<grid, THREADS, 0, s>>>((const T *)x, codes, scales, n);
    else act8_quantize_kernel<T, false><<<grid, THREADS, 0, s>>>((const T *)x, codes, scales, n);
    return launch_check();
}

template <typename T>
int restore8(const uint8_t *codes, const uint8_t *scales, void *x, long long n, int relu, hipStream_t s)
{
    const long long groups = (n + Io<T>::GV - 1) / Io<T>::GV;
    const int u = groups >= FULL ? 4 : 1;
    const dim3 grid((unsigned)((groups + THREADS * u - 1) / (THREADS * u)));
    T *p = (T *)x;
    if (relu && u == 4) act8_restore_kernel<T, true, 4><<<grid, THREADS, 0, s>>>(codes, scales, p, n);
    else if (relu) act8_restore_kernel<T, true, 1><<<grid, THREADS, 0, s>>>(codes, scales, p, n);
    else if (u == 4) act8_restore_kernel<T, false, 4><<<grid, THREADS, 0, s>>>(codes, scales, p, n);
    else act8_restore_kernel<T, false, 1><<<grid, THREADS, 0, s>>>(codes, scales, p, n);
    return launch_check();
}

template <bool CL, bool RES, int U>
void bias_act_act8_launch(dim3 grid, hipStream_t s, float *y, const float *x, const float *bias, const float *res, uint8_t *codes, uint8_t *scales, long long n, long long inner,
                          FastDiv fc, FastDiv fi, int relu)
{
    if (relu) bias_act_act8_kernel<CL, RES, true, U><<<grid, THREADS, 0, s>>>(y, x, bias, res, codes, scales, n, inner, fc, fi);
    else bias_act_act8_kernel<CL, RES, false, U><<<grid, THREADS, 0, s>>>(y, x, bias, res, codes, scales, n, inner, fc, fi);
}

// rows in chunks whose groups fit 31 bits
template <typename T, bool QUANT>
int mx4_rows(const void *x, uint8_t *codes, uint8_t *scales, long long rows, long long k, hipStream_t s)
{
    const long long groups = (k + BLOCK - 1) / BLOCK * (BLOCK / Io<T>::GV);
    if (groups > (1LL << 30)) return MDT_ERR_UNSUPPORTED;
    const long long step = (1LL << 30) / groups;
    for (long long r = 0; r < rows; r += step) {
        const long long take = rows - r < step ? rows - r : step, total = take * groups;
        const int u = !QUANT && total >= FULL ? 4 : 1;
        const dim3 grid((unsigned)((total + THREADS * u - 1) / (THREADS * u)));
        const FastDiv fd((unsigned)groups);
        if (QUANT) {
            mx4_quantize_kernel<T><<<grid, THREADS, 0, s>>>((const T *)x, codes, scales, r, (unsigned)total, k, fd);
        } else {
            if (u == 4) mx4_dequantize_kernel<T, 4><<<grid, THREADS, 0, s>>>(codes, scales, (T *)x, r, (unsigned)total, k, fd);
            else mx4_dequantize_kernel<T, 1><<<grid, THREADS, 0, s>>>(codes, scales, (T *)x, r, (unsigned)total, k, fd);
        }
        const int rc = launch_check();
        if (rc != MDT_OK) return rc;
    }
    return MDT_OK;
}

inline bool misaligned(const void *p, int a) { return ((uintptr_t)p & (a - 1)) != 0; }

}  // namespace

extern "C" {

int mdt_act8_quantize(const void *x, void *codes, void *scales, long long n, int dtype, int relu, void *stream)
{
    if (n < 0 || n > (1LL << 33) || (n > 0 && (!x || !codes || !scales)) || misaligned(codes, 4)) return MDT_ERR_INVALID_ARGUMENT;
    if (n == 0) return MDT_OK;
    const hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case MDT_DTYPE_F32: return quantize8<float>(x, (uint8_t *)codes, (uint8_t *)scales, n, relu, s);
        case MDT_DTYPE_BF16: return quantize8<__bf16>(x, (uint8_t *)codes, (uint8_t *)scales, n, relu, s);
        case MDT_DTYPE_F16: return quantize8<_Float16>(x, (uint8_t *)codes, (uint8_t *)scales, n, relu, s);
    }
    return MDT_ERR_INVALID_ARGUMENT;
}

int mdt_act8_restore(const void *codes, const void *scales, void *x, long long n, int dtype, int relu, void *stream)
{
    if (n < 0 || n > (1LL << 33) || (n > 0 && (!x || !codes || !scales)) || misaligned(codes, 4)) return MDT_ERR_INVALID_ARGUMENT;
    if (n == 0) return MDT_OK;
    const hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case MDT_DTYPE_F32: return restore8<float>((const uint8_t *)codes, (const uint8_t *)scales, x, n, relu, s);
        case MDT_DTYPE_BF16: return restore8<__bf16>((const uint8_t *)codes, (const uint8_t *)scales, x, n, relu, s);
        case MDT_DTYPE_F16: return restore8<_Float16>((const uint8_t *)codes, (const uint8_t *)scales, x, n, relu, s);
    }
    return MDT_ERR_INVALID_ARGUMENT;
}

int mdt_bias_act_act8_forward(float *y, const float *x, const float *bias, const float *residual, void *codes, void *scales, long long n, int channels, long long inner, int relu,
                              void *stream)
{
    if (n < 0 || n > (1LL << 33) || channels < 1 || channels > (1 << 24) || inner < 1 || inner > (1LL << 30) || (n > 0 && (!y || !x || !bias || !codes || !scales)) || misaligned(codes, 4))
        return MDT_ERR_INVALID_ARGUMENT;
    if (n == 0) return MDT_OK;
    const hipStream_t s = (hipStream_t)stream;
    const long long groups = (n + BLOCK - 1) / BLOCK * 8;
    const int u = groups >= FULL ? 4 : 1;
    const dim3 grid((unsigned)((groups + THREADS * u - 1) / (THREADS * u)));
    const FastDiv fc((unsigned)channels), fi((unsigned)inner);
    uint8_t *c = (uint8_t *)codes, *sc = (uint8_t *)scales;
    if (inner == 1) {
        if (residual && u == 4) bias_act_act8_launch<true, true, 4>(grid, s, y, x, bias, residual, c, sc, n, inner, fc, fi, relu);
        else if (residual) bias_act_act8_launch<true, true, 1>(grid, s, y, x, bias, residual, c, sc, n, inner, fc, fi, relu);
        else if (u == 4) bias_act_act8_launch<true, false, 4>(grid, s, y, x, bias, residual, c, sc, n, inner, fc, fi, relu);
        else bias_act_act8_launch<true, false, 1>(grid, s, y, x, bias, residual, c, sc, n, inner, fc, fi, relu);
    } else {
        if (residual) bias_act_act8_launch<false, true, 1>(dim3((unsigned)((groups + THREADS - 1) / THREADS)), s, y, x, bias, residual, c, sc, n, inner, fc, fi, relu);
        else bias_act_act8_launch<false, false, 1>(dim3((unsigned)((groups + THREADS - 1) / THREADS)), s, y, x, bias, residual, c, sc, n, inner, fc, fi, relu);
    }
    return launch_check();
}

int mdt_mx4_quantize(const void *x, void *codes, void *scales, long long rows, long long k, int dtype, void *stream)
{
    if (rows < 0 || k < 1 || rows > (1LL << 40) / k || (rows > 0 && (!x || !codes || !scales)) || misaligned(codes, 4)) return MDT_ERR_INVALID_ARGUMENT;
    const hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case MDT_DTYPE_F32: return mx4_rows<float, true>(x, (uint8_t *)codes, (uint8_t *)scales, rows, k, s);
        case MDT_DTYPE_BF16: return mx4_rows<__bf16, true>(x, (uint8_t *)codes, (uint8_t *)scales, rows, k, s);
        case MDT_DTYPE_F16: return mx4_rows<_Float16, true>(x, (uint8_t *)codes, (uint8_t *)scales, rows, k, s);
    }
    return MDT_ERR_INVALID_ARGUMENT;
}

int mdt_mx4_dequantize(const void *codes, const void *scales, void *x, long long rows, long long k, int dtype, void *stream)
{
    if (rows < 0 || k < 1 || rows > (1LL << 40) / k || (rows > 0 && (!x || !codes || !scales)) || misaligned(codes, 4)) return MDT_ERR_INVALID_ARGUMENT;
    const hipStream_t s = (hipStream_t)stream;
    uint8_t *c = (uint8_t *)const_cast<void *>(codes), *sc = (uint8_t *)const_cast<void *>(scales);
    switch (dtype) {
        case MDT_DTYPE_F32: return mx4_rows<float, false>(x, c, sc, rows, k, s);
        case MDT_DTYPE_BF16: return mx4_rows<__bf16, false>(x, c, sc, rows, k, s);
        case MDT_DTYPE_F16: return mx4_rows<_Float16, false>(x, c, sc, rows, k, s);
    }
    return MDT_ERR_INVALID_ARGUMENT;
}

}  // extern "C"
