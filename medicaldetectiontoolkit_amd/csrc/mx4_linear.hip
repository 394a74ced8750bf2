// mx4_linear.hip -- act(x W^T + bias) with both operands in 4-bit block-scaled codes (gfx950).
//
// The matrix units take 4-bit codes and one scale byte per 32 of them as they are (K = 64 of a 32 x 32 tile an instruction), products and sums in
// fp32.  x is rounded to codes first (mx4_quantize_kernel), W is kept in codes.
#include "block_scaled.h"

namespace {

using namespace mdt_bs;

constexpr int WAVES = 4;
constexpr int THREADS = 64 * WAVES;

// a wave's 32 x 32 tile over the block range of its split; lane l: row / column l % 32, block kb + l / 32.  A block beyond the row's end multiplies
// zero codes.
__global__ __launch_bounds__(THREADS) void mx4_gemm_kernel(const uint8_t *__restrict__ xc, const uint8_t *__restrict__ xs, const uint8_t *__restrict__ wc, const uint8_t *__restrict__ ws,
                                                           float *__restrict__ part, long long M, int N, long long kb, long long kb_per)
{
    const int l = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long m0 = ((long long)blockIdx.x * WAVES + wave) * 32;
    if (m0 >= M) return;
    const long long m = m0 + (l & 31);
    const int n = blockIdx.y * 32 + (l & 31);
    const long long b0 = (long long)blockIdx.z * kb_per, b1 = b0 + kb_per < kb ? b0 + kb_per : kb;
    v16f acc = {};
    for (long long b = b0; b < b1; b += 2) {
        const long long at = b + (l >> 5);
        v8i A = {}, B = {};
        int sa = 127, sb = 127;
        if (at < b1) {
            if (m < M) {
                *reinterpret_cast<v4u *>(&A) = *reinterpret_cast<const v4u *>(xc + (m * kb + at) * 16);
                sa = xs[m * kb + at];
            }
            if (n < N) {
                *reinterpret_cast<v4u *>(&B) = *reinterpret_cast<const v4u *>(wc + (n * kb + at) * 16);
                sb = ws[n * kb + at];
            }
        }
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, acc, 4, 4, 0, sa, 0, sb);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const long long row = m0 + 8 * (i / 4) + 4 * (l >> 5) + i % 4;
        if (row < M && n < N) part[((long long)blockIdx.z * M + row) * N + n] = acc[i];
    }
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_finish_kernel(const float *__restrict__ part, const float *__restrict__ bias, T *__restrict__ y, long long mn, int N, int splits, int relu)
{
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    if (e >= mn) return;
    float t = 0.0f;
    for (int k = 0; k < splits; ++k) t = t + part[k * mn + e];
    if (bias != nullptr) t = t + bias[e % N];
    if (relu) t = t < 0.0f ? 0.0f : t;
    y[e] = Io<T>::from_f(t);
}

inline long long blocks_of(long long k) { return (k + BLOCK - 1) / BLOCK; }

inline long long splits_of(long long rows, long long k, int n)
{
    const long long tiles = (rows + 127) / 128 * ((n + 31) / 32), kb = blocks_of(k);
    long long s = 512 / tiles;
    if (s < 1) s = 1;
    if (s > (kb + 7) / 8) s = (kb + 7) / 8;
    return s;
}

inline size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace

extern "C" {

size_t mdt_mx4_linear_workspace_bytes(long long rows, long long k, int n)
{
    if (rows < 1 || k < 1 || n < 1) return 256;
    const long long kb = blocks_of(k);
    return up256((size_t)(rows * kb * 16)) + up256((size_t)(rows * kb)) + (size_t)(splits_of(rows, k, n) * rows * n) * 4 + 256;
}

int mdt_mx4_linear(const void *x, int dtype, const void *w_codes, const void *w_scales, const float *bias, void *y, long long rows, long long k, int n, int relu, void *workspace,
                   size_t workspace_bytes, void *stream)
{
    if (rows < 0 || k < 1 || n < 1 || n > (1 << 20) || k > (1LL << 30) || rows > (1LL << 30) || rows > (1LL << 36) / k || rows > (1LL << 31) / n || (rows > 0 && (!x || !w_codes || !w_scales || !y))) return MDT_ERR_INVALID_ARGUMENT;
    if (dtype != MDT_DTYPE_F32 && dtype != MDT_DTYPE_BF16 && dtype != MDT_DTYPE_F16) return MDT_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)w_codes & 15) != 0) return MDT_ERR_INVALID_ARGUMENT;
    if (rows == 0) return MDT_OK;
    if (workspace == nullptr || workspace_bytes < mdt_mx4_linear_workspace_bytes(rows, k, n)) return MDT_ERR_WORKSPACE_TOO_SMALL;
    const hipStream_t s = (hipStream_t)stream;
    const long long kb = blocks_of(k), splits = splits_of(rows, k, n), per = (kb + splits - 1) / splits;
    uint8_t *xc = (uint8_t *)workspace, *xs = xc + up256((size_t)(rows * kb * 16));
    float *part = (float *)(xs + up256((size_t)(rows * kb)));
    const int rc = mdt_mx4_quantize(x, xc, xs, rows, k, dtype, stream);
    if (rc != MDT_OK) return rc;
    const dim3 grid((unsigned)((rows + 32 * WAVES - 1) / (32 * WAVES)), (unsigned)((n + 31) / 32), (unsigned)splits);
    mx4_gemm_kernel<<<grid, THREADS, 0, s>>>(xc, xs, (const uint8_t *)w_codes, (const uint8_t *)w_scales, part, rows, n, kb, per);
    const long long mn = rows * n;
    const dim3 fg((unsigned)((mn + 255) / 256));
    switch (dtype) {
        case MDT_DTYPE_F32: mx4_finish_kernel<float><<<fg, 256, 0, s>>>(part, bias, (float *)y, mn, n, (int)splits, relu); break;
        case MDT_DTYPE_BF16: mx4_finish_kernel<__bf16><<<fg, 256, 0, s>>>(part, bias, (__bf16 *)y, mn, n, (int)splits, relu); break;
        default: mx4_finish_kernel<_Float16><<<fg, 256, 0, s>>>(part, bias, (_Float16 *)y, mn, n, (int)splits, relu); break;
    }
    return launch_check();
}

}  // extern "C"
