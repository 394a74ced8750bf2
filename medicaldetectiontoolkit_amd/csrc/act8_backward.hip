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

// floats of one wave's LDS tiles: 32 voxels of gradients (and a row's overhang; gx's rows take the same place later), 32 of bf16 inputs (and theirs)
__host__ __device__ constexpr int fused_rows_floats(int mt, int ci, int co) { return 32 * (co > ci ? co : ci) + 32 * mt; }
__host__ __device__ constexpr int fused_wave_floats(int mt, int nt, int ci, int co) { return (fused_rows_floats(mt, ci, co) + (32 * ci + 32 * nt) / 2 + 3) / 4 * 4; }

// ---- both products in one pass, for few channels --------------------------------------------------------------------------------------------
// A wave takes 32 voxels at a time and needs no other wave: their 32 co gradients are one contiguous run, loaded 16 bytes a lane, masked, and put into the
// wave's own LDS tile as they are; their 32 ci input codes are ci whole blocks.  From the tile gw takes columns (M = co, N = ci, K = voxel) and gx takes rows
// (M = ci, N = voxel, K = co), both cut into bf16 pieces in registers; gw stays in registers over all of a wave's voxels.  gx's tile replaces the gradients in LDS
// and leaves as the contiguous run that it is, like g.
// Loads and stores share one in-order counter: the next chunk's loads are issued before this chunk's stores and every chunk issues the same number of
// stores, so that the wait for the loads does not wait for the stores behind them.
// Entries of the tiles behind co or ci hold whatever follows in LDS: they only reach rows and columns that are not stored, except along gx's sum, where
// they are set to zero.
template <int MT, int NT, bool G_OUT>
__global__ __launch_bounds__(THREADS, MT * NT <= 3 ? 2 : 1) void fused_kernel(const float *__restrict__ gy, const uint8_t *__restrict__ yc, const float *__restrict__ w,
                                                                             const uint8_t *__restrict__ xc, const uint8_t *__restrict__ xs, float *__restrict__ gx,
                                                                             float *__restrict__ g_out, float *__restrict__ part_w, float *__restrict__ part_b, long long V, int ci, int co,
                                                                             int x_relu)
{
    extern __shared__ v4u smem[];
    const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = l >> 5, lo = l & 31;
    const int KS = (co + 15) / 16;
    v4u *wp = smem;                                                              // [NT][KS][3][64] pieces of W in fragment order
    float *gs = reinterpret_cast<float *>(smem + NT * KS * 3 * 64) + wave * fused_wave_floats(MT, NT, ci, co);
    uint16_t *xb = reinterpret_cast<uint16_t *>(gs + fused_rows_floats(MT, ci, co));
    for (int t = threadIdx.x; t < NT * KS * 64; t += THREADS) {
        const int ll = t & 63, n = (t / 64 / KS) * 32 + (ll & 31), k = (t / 64 % KS) * 16 + 8 * (ll >> 5);
        float b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = n < ci && k + j < co ? w[(k + j) * ci + n] : 0.0f;
        const Split8 B = split8(b);
        v4u *to = wp + (t / 64) * 3 * 64 + ll;
        to[0] = __builtin_bit_cast(v4u, B.hi);
        to[64] = __builtin_bit_cast(v4u, B.mid);
        to[128] = __builtin_bit_cast(v4u, B.lo);
    }
    __syncthreads();

    const long long chunks = (V + 31) / 32, full = V / 32, step = (long long)gridDim.x * WAVES;
    long long chunk = (long long)blockIdx.x * WAVES + wave;
    v4f G[4 * MT];
    unsigned Y[4 * MT], X[4 * NT];
    int S[4 * NT];
    // lanes behind the run's end repeat its last 16 bytes (and store them to the same place again)
    auto at_gy = [&](unsigned lane, int q) { return min(q * 64 + lane, 8u * co - 1); };
    auto at_x = [&](unsigned lane, int q) { return min(q * 64 + lane, 8u * ci - 1); };
    // the lane's number, kept from the optimiser: it would hold every address that it computes from it in a register of its own over the loop
    auto lane = [&] {
        unsigned v = l;
        asm volatile("" : "+v"(v));
        return v;
    };
    auto load = [&](long long c) {
        const unsigned ln = lane();
        if (yc != nullptr) {
            const uint8_t *py = yc + c * 32 * co;
#pragma unroll
            for (int q = 0; q < 4 * MT; ++q) Y[q] = *reinterpret_cast<const unsigned *>(py + 4 * at_gy(ln, q));
        }
        const uint8_t *px = xc + c * 32 * ci, *ps = xs + c * ci;
#pragma unroll
        for (int q = 0; q < 4 * NT; ++q) {
            X[q] = *reinterpret_cast<const unsigned *>(px + 4 * at_x(ln, q));
            S[q] = ps[at_x(ln, q) >> 3];
        }
        const float *pg = gy + c * 32 * co;
#pragma unroll
        for (int q = 0; q < 4 * MT; ++q) G[q] = *reinterpret_cast<const Io<float>::vec *>(pg + 4 * at_gy(ln, q));
    };
    // the last chunk where it is short: value by value, straight into the tiles
    auto fill_short = [&](long long c) {
        for (int e = l; e < 32 * co; e += 64) {
            const long long at = c * 32 * co + e;
            float t = 0.0f;
            if (at < V * co) {
                t = yc == nullptr || yc[at] ? gy[at] : 0.0f;
                if (G_OUT) g_out[at] = t;
            }
            gs[e] = t;
        }
        for (int e = l; e < 32 * ci; e += 64) {
            const long long at = c * 32 * ci + e;
            xb[e] = at < V * ci ? (uint16_t)(__float_as_uint(code_value(xc[at], x_relu, xs[at >> 5])) >> 16) : (uint16_t)0;
        }
    };
    auto fence = [] {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    v16f acc[MT][NT];
    float bsum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        bsum[m] = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = v16f{};
    }
    if (chunk < full) load(chunk);
    for (; chunk < chunks; chunk += step) {
        const bool whole = chunk < full;
        if (whole) {
            const unsigned ln = lane();
#pragma unroll
            for (int q = 0; q < 4 * MT; ++q) {
                if (yc != nullptr) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) G[q][j] = (Y[q] >> (8 * j) & 255u) ? G[q][j] : 0.0f;
                }
                *reinterpret_cast<v4f *>(gs + 4 * at_gy(ln, q)) = G[q];
            }
#pragma unroll
            for (int q = 0; q < 4 * NT; ++q) {
                float t[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) t[j] = code_value(X[q] >> (8 * j) & 255u, x_relu, S[q]);
                uint2 p;
                p.x = pack_hi(t[0], t[1]);
                p.y = pack_hi(t[2], t[3]);
                *reinterpret_cast<uint2 *>(xb + 4 * at_x(ln, q)) = p;
            }
        } else {
            fill_short(chunk);
        }
        if (chunk + step < full) load(chunk + step);
        fence();
        // gw and gbias
        const unsigned lg = lane(), og = 8 * (lg >> 5) * co + (lg & 31), ox = 8 * (lg >> 5) * ci + (lg & 31);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            v8bf B[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                v4u p;
#pragma unroll
                for (int q = 0; q < 4; ++q) p[q] = (unsigned)xb[ox + (ks * 16 + 2 * q) * ci + n * 32] | (unsigned)xb[ox + (ks * 16 + 2 * q + 1) * ci + n * 32] << 16;
                B[n] = __builtin_bit_cast(v8bf, p);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float a[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) a[j] = gs[og + (ks * 16 + j) * co + m * 32];
                bsum[m] = bsum[m] + (((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7])));
                const Split8 A = split8(a);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.lo, B[n], acc[m][n], 0, 0, 0);
                    acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.mid, B[n], acc[m][n], 0, 0, 0);
                    acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.hi, B[n], acc[m][n], 0, 0, 0);
                }
            }
        }
        // gx
        v16f d[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) d[n] = v16f{};
        for (int ks = 0; ks < KS; ++ks) {
            const int k = ks * 16 + 8 * half;
            const float *row = gs + lo * co + k;
            float b[8];
            if (co % 4 == 0) {
                *reinterpret_cast<v4f *>(b) = *reinterpret_cast<const v4f *>(row);
                *reinterpret_cast<v4f *>(b + 4) = *reinterpret_cast<const v4f *>(row + 4);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) b[j] = row[j];
            }
            if (ks * 16 + 16 > co) {
#pragma unroll
                for (int j = 0; j < 8; ++j) b[j] = k + j < co ? b[j] : 0.0f;
            }
            const Split8 B = split8(b);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const v4u *p = wp + (n * KS + ks) * 3 * 64 + l;
                const v8bf hi = __builtin_bit_cast(v8bf, p[0]), mid = __builtin_bit_cast(v8bf, p[64]), low = __builtin_bit_cast(v8bf, p[128]);
                d[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(low, B.hi, d[n], 0, 0, 0);
                d[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi, B.lo, d[n], 0, 0, 0);
                d[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(mid, B.mid, d[n], 0, 0, 0);
                d[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(mid, B.hi, d[n], 0, 0, 0);
                d[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi, B.mid, d[n], 0, 0, 0);
                d[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi, B.hi, d[n], 0, 0, 0);
            }
        }
        if (G_OUT && whole) {
            float *pg = g_out + chunk * 32 * co;
            const unsigned ln = lane();
#pragma unroll
            for (int q = 0; q < 4 * MT; ++q) *reinterpret_cast<Io<float>::vec *>(pg + 4 * at_gy(ln, q)) = *reinterpret_cast<const v4f *>(gs + 4 * at_gy(ln, q));
        }
        fence();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = n * 32 + 8 * q + 4 * half;
                float *to = gs + lo * ci + c;
                if (ci % 4 == 0) {
                    if (c < ci) *reinterpret_cast<v4f *>(to) = v4f{d[n][4 * q], d[n][4 * q + 1], d[n][4 * q + 2], d[n][4 * q + 3]};
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) if (c + j < ci) to[j] = d[n][4 * q + j];
                }
            }
        fence();
        float *px = gx + chunk * 32 * ci;
        if (whole) {
            const unsigned ln = lane();
#pragma unroll
            for (int q = 0; q < 4 * NT; ++q) *reinterpret_cast<Io<float>::vec *>(px + 4 * at_x(ln, q)) = *reinterpret_cast<const v4f *>(gs + 4 * at_x(ln, q));
        } else {
            for (int e = l; e < (V - chunk * 32) * ci; e += 64) px[e] = gs[e];
        }
        fence();
    }
    // the four waves' sums, in wave order
    float *sum = reinterpret_cast<float *>(smem), *sumb = sum + 32 * 32 * MT * NT;
#pragma unroll 1
    for (int turn = 0; turn < WAVES; ++turn) {
        __syncthreads();
        if (wave != turn) continue;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const float b2 = bsum[m] + __shfl_xor(bsum[m], 32);
            if (half == 0) sumb[m * 32 + lo] = turn == 0 ? b2 : sumb[m * 32 + lo] + b2;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float *to = sum + ((m * 32 + 8 * (i / 4) + 4 * half + i % 4) * NT + n) * 32 + lo;
                    *to = turn == 0 ? acc[m][n][i] : *to + acc[m][n][i];
                }
        }
    }
    __syncthreads();
    for (int t = threadIdx.x; t < co * ci; t += THREADS) part_w[(long long)blockIdx.x * co * ci + t] = sum[(t / ci) * 32 * NT + t % ci];
    for (int t = threadIdx.x; t < co; t += THREADS) part_b[(long long)blockIdx.x * co + t] = sumb[t];
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

struct FusedPlan { int mt, nt, lds, blocks; };

// the one-pass kernel's plan, mt = 0 where it does not apply
inline FusedPlan fused_plan(long long V, int ci, int co)
{
    FusedPlan p = {(co + 31) / 32, (ci + 31) / 32, 0, 0};
    const int tiles = co <= 160 && ci <= 160 ? p.mt * p.nt : 99;
    if (tiles > 10) return {0, 0, 0, 0};
    const int ks = (co + 15) / 16;
    p.lds = p.nt * ks * 3 * 1024 + WAVES * fused_wave_floats(p.mt, p.nt, ci, co) * 4;
    const int sums = (1024 * tiles + 32 * p.mt) * 4;
    if (p.lds < sums) p.lds = sums;
    if (p.lds > 160 * 1024) return {0, 0, 0, 0};
    const int per_cu = tiles <= 3 ? 2 : 1, fit = 160 * 1024 / p.lds, at_once = 256 * (fit < per_cu ? fit : per_cu);
    const long long want = (V + 32 * WAVES - 1) / (32 * WAVES);
    p.blocks = (int)(want < at_once ? want : at_once);
    return p;
}

struct FusedArgs { const float *gy; const uint8_t *yc; const float *w; const uint8_t *xc, *xs; float *gx, *g, *part_w, *part_b; long long V; int ci, co, x_relu; };

template <int MT, int NT>
int fused_launch(const FusedPlan &p, const FusedArgs &a, hipStream_t s)
{
    const auto kernel = a.g != nullptr ? fused_kernel<MT, NT, true> : fused_kernel<MT, NT, false>;
    if (hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, p.lds) != hipSuccess) return MDT_ERR_LAUNCH_FAILED;
    kernel<<<p.blocks, THREADS, p.lds, s>>>(a.gy, a.yc, a.w, a.xc, a.xs, a.gx, a.g, a.part_w, a.part_b, a.V, a.ci, a.co, a.x_relu);
    return MDT_OK;
}

int fused_run(const FusedPlan &p, const FusedArgs &a, hipStream_t s)
{
    switch (p.mt * 10 + p.nt) {
        case 11: return fused_launch<1, 1>(p, a, s);
        case 12: return fused_launch<1, 2>(p, a, s);
        case 13: return fused_launch<1, 3>(p, a, s);
        case 14: return fused_launch<1, 4>(p, a, s);
        case 15: return fused_launch<1, 5>(p, a, s);
        case 21: return fused_launch<2, 1>(p, a, s);
        case 22: return fused_launch<2, 2>(p, a, s);
        case 23: return fused_launch<2, 3>(p, a, s);
        case 24: return fused_launch<2, 4>(p, a, s);
        case 25: return fused_launch<2, 5>(p, a, s);
        case 31: return fused_launch<3, 1>(p, a, s);
        case 32: return fused_launch<3, 2>(p, a, s);
        case 33: return fused_launch<3, 3>(p, a, s);
        case 41: return fused_launch<4, 1>(p, a, s);
        case 42: return fused_launch<4, 2>(p, a, s);
        case 51: return fused_launch<5, 1>(p, a, s);
        case 52: return fused_launch<5, 2>(p, a, s);
    }
    return MDT_ERR_UNSUPPORTED;
}

}  // namespace

extern "C" {

size_t mdt_conv1x1_act8_backward_workspace_bytes(long long n_voxels, int c_in, int c_out)
{
    if (n_voxels < 1 || c_in < 1 || c_out < 1 || c_in > 65536 || c_out > 65536) return 256;
    const long long per = wgrad_split(n_voxels, c_in, c_out);
    long long splits = (n_voxels + per - 1) / per;
    const FusedPlan p = fused_plan(n_voxels, c_in, c_out);
    if (p.blocks > splits) splits = p.blocks;
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
    const FusedPlan p = n_voxels > 0 && gx && gw ? fused_plan(n_voxels, c_in, c_out) : FusedPlan{0, 0, 0, 0};
    if (p.mt > 0) {
        float *part_w = (float *)workspace, *part_b = part_w + p.blocks * nw;
        const FusedArgs a = {gy, (const uint8_t *)y_codes, w, (const uint8_t *)x_codes, (const uint8_t *)x_scales, gx, g, part_w, part_b, n_voxels, c_in, c_out, x_relu};
        const int rc = fused_run(p, a, s);
        if (rc != MDT_OK) return rc;
        reduce_kernel<<<dim3((unsigned)((nw + c_out + 31) / 32)), 256, 0, s>>>(part_w, part_b, gw, gbias, nw, c_out, p.blocks);
        return launch_check();
    }
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
