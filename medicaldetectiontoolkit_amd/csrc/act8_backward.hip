// act8_backward.hip -- backward pass of a 1x1(x1) convolution from the 8-bit copies of its input and output (gfx950).
//
// Rows are voxels (channels-last).  With x^ the kept input (code * 2^e), m = (kept output code > 0) the ReLU's mask and W [co][ci]:
//   g = gy . m            gbias[o] = sum_v g[v][o]
//   gx[v][i] = sum_o g[v][o] W[o][i]                gw[o][i] = sum_v g[v][o] x^[v][i]
//
// Both products run on the bf16 matrix units with fp32 accumulation and lose nothing that fp32 would keep: a float is the exact sum of three bf16
// numbers (each the nearest to what the ones before leave), x^ IS a bf16 number, so gw takes 3 matrix instructions a tile and gx 6 (the three products
// left out are at most 2^-24 of the whole, of either sign).
#include "block_scaled.h"

namespace {

using namespace mdt_bs;

constexpr int WAVES = 4;
constexpr int THREADS = 64 * WAVES;

// two floats' upper halves as one register of two bf16
__device__ __forceinline__ unsigned pack_hi(float lo, float hi) { return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u); }

// two floats rounded to bf16 (to nearest even, one instruction) and what is left of each; the differences are exact
__device__ __forceinline__ unsigned round2(float &a, float &b)
{
    const v2f t = {a, b};
    const unsigned p = __builtin_bit_cast(unsigned, __builtin_convertvector(t, v2bf));
    a = a - __uint_as_float(p << 16);
    b = b - __uint_as_float(p & 0xffff0000u);
    return p;
}

// 8 floats -> their three bf16 pieces: |mid| <= 2^-8 |x|, |lo| <= 2^-17 |x|, hi + mid + lo = x
struct Split8 { v8bf hi, mid, lo; };
__device__ __forceinline__ Split8 split8(const float (&v)[8])
{
    v4u p[3];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float a = v[2 * q], b = v[2 * q + 1];
#pragma unroll
        for (int k = 0; k < 3; ++k) p[k][q] = round2(a, b);
    }
    return {__builtin_bit_cast(v8bf, p[0]), __builtin_bit_cast(v8bf, p[1]), __builtin_bit_cast(v8bf, p[2])};
}

__device__ __forceinline__ float code_value(unsigned c, bool is_relu, int b) { return (is_relu ? (float)c : (float)(int8_t)c) * scale_of(b); }

// ---- gw and gbias: partial sums over ranges of voxels --------------------------------------------------------------------------------
// matrix tile 32 x 32 (M = co, N = ci, K = 16 voxels): lane l holds row / column l % 32 and voxels 8 (l / 32) ...
__global__ __launch_bounds__(THREADS) void wgrad_kernel(const float *__restrict__ gy, const uint8_t *__restrict__ yc, const uint8_t *__restrict__ xc, const uint8_t *__restrict__ xs,
                                                        float *__restrict__ part_w, float *__restrict__ part_b, long long V, int ci, int co, int x_relu, long long per_split)
{
    __shared__ float s_acc[WAVES][32 * 32];
    __shared__ float s_b[WAVES][64];
    const int l = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int m = blockIdx.y * 32 + (l & 31), n = blockIdx.z * 32 + (l & 31);
    const long long v0 = (long long)blockIdx.x * per_split, v1 = v0 + per_split < V ? v0 + per_split : V;
    v16f acc = {};
    float bsum = 0.0f;
    for (long long v = v0 + wave * 16; v < v1; v += WAVES * 16) {
        float g[8], x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const long long r = v + 8 * (l >> 5) + j;
            const bool in = r < v1;
            g[j] = in && m < co ? gy[r * co + m] : 0.0f;
            if (yc != nullptr && in && m < co) g[j] = yc[r * co + m] ? g[j] : 0.0f;
            const long long at = r * ci + n;
            x[j] = in && n < ci ? code_value(xc[at], x_relu, xs[at >> 5]) : 0.0f;
            bsum = bsum + g[j];
        }
        const Split8 a = split8(g);
        v4u xb;
#pragma unroll
        for (int q = 0; q < 4; ++q) xb[q] = pack_hi(x[2 * q], x[2 * q + 1]);
        const v8bf b = __builtin_bit_cast(v8bf, xb);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.lo, b, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.mid, b, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b, acc, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s_acc[wave][(8 * (i / 4) + 4 * (l >> 5) + i % 4) * 32 + (l & 31)] = acc[i];
    s_b[wave][l] = bsum;
    __syncthreads();
    for (int t = threadIdx.x; t < 32 * 32; t += THREADS) {
        const int o = blockIdx.y * 32 + t / 32, i = blockIdx.z * 32 + t % 32;
        if (o < co && i < ci) part_w[((long long)blockIdx.x * co + o) * ci + i] = (s_acc[0][t] + s_acc[1][t]) + (s_acc[2][t] + s_acc[3][t]);
    }
    if (blockIdx.z == 0 && threadIdx.x < 32 && blockIdx.y * 32 + threadIdx.x < co) {
        float s = 0.0f;
        for (int w = 0; w < WAVES; ++w) s = s + (s_b[w][threadIdx.x] + s_b[w][threadIdx.x + 32]);
        part_b[(long long)blockIdx.x * co + blockIdx.y * 32 + threadIdx.x] = s;
    }
}

// out[e] = sum over the splits of part[split][e], 32 elements a workgroup and 8 ranges of splits, in a fixed order; elements [0, nw) are gw's, the rest gbias's
__global__ __launch_bounds__(256) void reduce_kernel(const float *__restrict__ part_w, const float *__restrict__ part_b, float *__restrict__ gw, float *__restrict__ gb, long long nw,
                                                     int nb, int splits)
{
    __shared__ float s[8][32];
    const int lane = threadIdx.x & 31, range = threadIdx.x >> 5;
    const long long e = (long long)blockIdx.x * 32 + lane;
    const bool is_w = e < nw;
    const float *p = is_w ? part_w + e : part_b + (e - nw);
    const long long step = is_w ? nw : nb;
    float acc = 0.0f;
    if (e < nw + nb)
        for (int k = range; k < splits; k += 8) acc = acc + p[k * step];
    s[range][lane] = acc;
    __syncthreads();
    if (range == 0 && e < nw + nb) {
        float t = 0.0f;
        for (int r = 0; r < 8; ++r) t = t + s[r][lane];
        if (is_w) { if (gw != nullptr) gw[e] = t; }
        else if (gb != nullptr) gb[e - nw] = t;
    }
}

// ---- gx (and g) ------------------------------------------------------------------------------------------------------------------------
// matrix tile 32 x 32 (M = voxels, N = ci, K = 16 of co); a wave's tile each
__global__ __launch_bounds__(THREADS) void dgrad_kernel(const float *__restrict__ gy, const uint8_t *__restrict__ yc, const float *__restrict__ w, float *__restrict__ gx,
                                                        float *__restrict__ g_out, long long V, int ci, int co)
{
    const int l = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long vbase = ((long long)blockIdx.x * WAVES + wave) * 32, r = vbase + (l & 31);
    const int n = blockIdx.y * 32 + (l & 31);
    v16f acc = {};
    for (int k0 = 0; k0 < co; k0 += 16) {
        const int k = k0 + 8 * (l >> 5);
        float g[8], b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            g[j] = r < V && k + j < co ? gy[r * co + k + j] : 0.0f;
            if (yc != nullptr && r < V && k + j < co) g[j] = yc[r * co + k + j] ? g[j] : 0.0f;
            if (g_out != nullptr && blockIdx.y == 0 && r < V && k + j < co) g_out[r * co + k + j] = g[j];
            b[j] = n < ci && k + j < co ? w[(long long)(k + j) * ci + n] : 0.0f;
        }
        const Split8 A = split8(g), B = split8(b);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.lo, B.hi, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.hi, B.lo, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.mid, B.mid, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.mid, B.hi, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.hi, B.mid, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.hi, B.hi, acc, 0, 0, 0);
    }
    if (gx == nullptr) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const long long row = vbase + 8 * (i / 4) + 4 * (l >> 5) + i % 4;
        if (row < V && n < ci) gx[row * ci + n] = acc[i];
    }
}

// voxels a workgroup of wgrad_kernel sums: enough workgroups for the card, not so many that the partial sums outweigh the inputs
inline long long wgrad_split(long long V, int ci, int co)
{
    const long long tiles = (long long)((co + 31) / 32) * ((ci + 31) / 32);
    long long splits = 1 + 2048 / tiles;
    const long long most = (V + 255) / 256;
    if (splits > most) splits = most;
    const long long per = (V + splits - 1) / splits;
    return (per + 15) / 16 * 16;
}

}  // namespace

extern "C" {

size_t mdt_conv1x1_act8_backward_workspace_bytes(long long n_voxels, int c_in, int c_out)
{
    if (n_voxels < 1 || c_in < 1 || c_out < 1 || c_in > 65536 || c_out > 65536) return 256;
    const long long per = wgrad_split(n_voxels, c_in, c_out), splits = (n_voxels + per - 1) / per;
    return (size_t)(splits * ((long long)c_in * c_out + c_out)) * 4 + 256;
}

int mdt_conv1x1_act8_backward(const float *gy, const float *w, const void *x_codes, const void *x_scales, int x_relu, const void *y_codes, float *gx, float *gw, float *gbias, float *g,
                              long long n_voxels, int c_in, int c_out, void *workspace, size_t workspace_bytes, void *stream)
{
    if (n_voxels < 0 || n_voxels > (1LL << 30) || c_in < 1 || c_out < 1 || c_in > 65536 || c_out > 65536) return MDT_ERR_INVALID_ARGUMENT;
    const hipStream_t s = (hipStream_t)stream;
    const bool sums = gw != nullptr || gbias != nullptr;
    if (n_voxels > 0 && (!gy || (gx && !w) || (gw && (!x_codes || !x_scales)))) return MDT_ERR_INVALID_ARGUMENT;
    const long long per = n_voxels > 0 ? wgrad_split(n_voxels, c_in, c_out) : 16, splits = (n_voxels + per - 1) / per;
    if (sums && n_voxels > 0 && (workspace == nullptr || workspace_bytes < mdt_conv1x1_act8_backward_workspace_bytes(n_voxels, c_in, c_out))) return MDT_ERR_WORKSPACE_TOO_SMALL;
    const long long nw = (long long)c_in * c_out;
    float *part_w = (float *)workspace, *part_b = part_w + splits * nw;
    if (n_voxels > 0 && (gx || g)) {
        const dim3 grid((unsigned)((n_voxels + 32 * WAVES - 1) / (32 * WAVES)), gx ? (unsigned)((c_in + 31) / 32) : 1u);
        dgrad_kernel<<<grid, THREADS, 0, s>>>(gy, (const uint8_t *)y_codes, w, gx, g, n_voxels, c_in, c_out);
    }
    if (sums) {
        if (n_voxels > 0) {
            const dim3 grid((unsigned)splits, (unsigned)((c_out + 31) / 32), gw ? (unsigned)((c_in + 31) / 32) : 1u);
            wgrad_kernel<<<grid, THREADS, 0, s>>>(gy, (const uint8_t *)y_codes, (const uint8_t *)x_codes, (const uint8_t *)x_scales, part_w, part_b, n_voxels, c_in, c_out, x_relu, per);
        }
        reduce_kernel<<<dim3((unsigned)((nw + c_out + 31) / 32)), 256, 0, s>>>(part_w, part_b, gw, gbias, nw, c_out, (int)splits);
    }
    return launch_check();
}

}  // extern "C"
