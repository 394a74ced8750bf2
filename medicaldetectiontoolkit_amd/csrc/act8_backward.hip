// act8_backward.hip -- backward pass of a 1x1(x1) convolution from the 8-bit copies of its input and output (gfx950).
//
// Rows are voxels (channels-last).  With x^ the kept input (code * 2^e), m = (kept output code > 0) the ReLU's mask and W [co][ci]:
//   g = gy . m            gbias[o] = sum_v g[v][o]
//   gx[v][i] = sum_o g[v][o] W[o][i]                gw[o][i] = sum_v g[v][o] x^[v][i]
//
// Both products run on the bf16 matrix units with fp32 accumulation and lose nothing that fp32 would keep: a float is the exact sum of three bf16
// numbers (each the nearest to what the ones before leave), x^ IS a bf16 number, so gw takes 3 matrix instructions a tile and gx 6 (the three products
// left out are at most 2^-24 of the whole, of either sign).  That holds from 2^-110 to the largest float; smaller ones are off by less than 2^-133, half a
// step of the smallest bf16 numbers.
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

// round2 for the first piece: a finite value that would round to an infinity (from 3.3962e38 on) gets the largest bf16 number (mid is up to 2^-7 of it then).  An infinity leaves one for
// the next piece and a NaN is left over, so neither becomes finite.  One instruction a value.
__device__ __forceinline__ unsigned first2(float &a, float &b)
{
    const float big = Largest<__bf16>::v;
    float p = __builtin_amdgcn_fmed3f(a, -big, big), q = __builtin_amdgcn_fmed3f(b, -big, big);
    const v2f t = {p, q};
    const unsigned w = __builtin_bit_cast(unsigned, __builtin_convertvector(t, v2bf));
    a = a - __uint_as_float(w << 16);
    b = b - __uint_as_float(w & 0xffff0000u);
    return w;
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
        for (int k = 0; k < 3; ++k) p[k][q] = k == 0 ? first2(a, b) : round2(a, b);
    }
    return {__builtin_bit_cast(v8bf, p[0]), __builtin_bit_cast(v8bf, p[1]), __builtin_bit_cast(v8bf, p[2])};
}

__device__ __forceinline__ float code_value(unsigned c, bool is_relu, int b) { return (is_relu ? (float)c : (float)(int8_t)c) * scale_of(b); }

struct Args { const float *gy; const uint8_t *yc; const float *w; const uint8_t *xc, *xs; float *gx, *g, *part_w, *part_b; long long V; int ci, co, x_relu; };

// ---- any number of channels: one product a workgroup, tiles through LDS ------------------------------------------------------------------------
// Both kernels cut what they load into bf16 pieces once, put the pieces into LDS with the summed axis innermost (32 entries and 8 of padding a row: the
// 16-byte reads and writes of neighbouring rows fall into different banks) and hold the next step's loads in registers meanwhile.  4 waves, WM x WN of
// them with TM x TN matrix tiles of 32 x 32 each.
// 1620 voxels 1536 -> 384: 43 us, 400 TFLOP/s of the 9 products of pieces, and 5 us for the joining (both launches in a queue of calls: 43 - 47 us).  The cutting, which every tile repeats for its rows (a quarter of
// the VALU's slots), and the waits at two workgroups a CU bound it.  Pieces cut once by a launch of their own and multiplied from L2 without LDS took 10 + 34 us
// here and twice the time for long narrow maps.
constexpr int KSTEP = 32, KROW = KSTEP + 8;

__device__ __forceinline__ v8bf row_of(const uint16_t *p) { return __builtin_bit_cast(v8bf, *reinterpret_cast<const v4u *>(p)); }

// A run of values from base[first] on, read 4 at a time at 32-bit offsets without branches (so that the number of loads in flight stays known and a wait for
// one does not become a wait for all): where 4 values would pass the end of the array, the last 4 are read, and fix() moves them to their places, zeros behind.
struct Run {
    long long first;        // of the base: the run's first element, or the array's fourth last
    int delta, last;        // the run's first element and the last 4 of the array, counted from the base
    __device__ __forceinline__ Run(long long at, long long n)
    {
        first = at < n - 4 ? at : n - 4;
        delta = (int)(at - first);
        const long long rest = n - 4 - first;
        last = rest < (1 << 30) ? (int)rest : 1 << 30;
    }
    __device__ __forceinline__ unsigned at(int off) const { return (unsigned)min(off + delta, last); }
    __device__ __forceinline__ v4f fix(v4f v, int off) const
    {
        const int d = off + delta - last;
        const bool one = d > 0 && (d & 1), two = d > 0 && (d & 2), none = d >= 4;
        v = v4f{one ? v[1] : v[0], one ? v[2] : v[1], one ? v[3] : v[2], one ? 0.0f : v[3]};
        v = v4f{two ? v[2] : v[0], two ? v[3] : v[1], two ? 0.0f : v[2], two ? 0.0f : v[3]};
        return v4f{none ? 0.0f : v[0], none ? 0.0f : v[1], none ? 0.0f : v[2], none ? 0.0f : v[3]};
    }
    __device__ __forceinline__ unsigned fix(unsigned v, int off) const
    {
        const int d = off + delta - last;
        return d <= 0 ? v : d < 4 ? v >> (8 * d) : 0u;
    }
};
__device__ __forceinline__ v4f get4(const float *p) { return *reinterpret_cast<const Io<float>::vec *>(p); }
__device__ __forceinline__ unsigned get4(const uint8_t *p)
{
    typedef unsigned una __attribute__((aligned(1)));
    return *reinterpret_cast<const una *>(p);
}
__device__ __forceinline__ v4f masked(v4f g, unsigned m)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = (m >> (8 * j) & 255u) ? g[j] : 0.0f;
    return g;
}
// 4 floats -> 4 entries of each of the three pieces' planes
__device__ __forceinline__ void put4(uint16_t *to, int plane, v4f v)
{
    float a = v[0], b = v[1], c = v[2], d = v[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        uint2 p;
        p.x = k == 0 ? first2(a, b) : round2(a, b);
        p.y = k == 0 ? first2(c, d) : round2(c, d);
        *reinterpret_cast<uint2 *>(to + k * plane) = p;
    }
}

// gx (and g).  M = ci, N = voxel, K = co: a lane ends up with 4 consecutive channels of one voxel.  Workgroup `id` of ranges of voxels x ci tiles x k_splits
// ranges of co, whose sums are joined later.
struct DgradGrid { int ci_tiles, k_splits, k_per; long long groups; float *to; };
template <int WM, int TM, int WN, int TN>
__device__ __forceinline__ void dgrad_tile(uint16_t *smem, const Args &a, const DgradGrid &grid, unsigned id)
{
    constexpr int BM = WM * TM * 32, BN = WN * TN * 32, GP = BN / 32, WG = BM / 64, DEPTH = TM * TN > 1 ? 1 : 2;    // DEPTH: steps loaded ahead
    const uint8_t *__restrict__ yc = a.yc;
    float *__restrict__ g_out = a.g;
    const long long V = a.V;
    const int ci = a.ci, co = a.co;
    uint16_t *s_w = smem, *s_g = smem + 3 * BM * KROW;
    const int t = threadIdx.x, l = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), half = l >> 5, lo = l & 31;
    // the tiles of one range of voxels follow each other on one XCD (workgroups go to the 8 XCDs in turn), whose L2 then holds the range's gradients; every XCD
    // gets as many tiles (whole ranges for each: 1620 voxels 384 -> 1536 in 70 us, not 57)
    const unsigned turn = id % 8 * (unsigned)(grid.groups / 8) + id / 8, tile = turn % (grid.ci_tiles * grid.k_splits);
    const int ct = tile % grid.ci_tiles, split = tile / grid.ci_tiles, kb = split * grid.k_per, ke = min(kb + grid.k_per, co);
    const long long v0 = (long long)(turn / (grid.ci_tiles * grid.k_splits)) * BN;
    if (v0 >= V || kb >= co) return;
    float *__restrict__ gx = grid.to + split * V * ci;
    // gradients: 8 lanes a row of 32, row gr + 32 i; weights: a lane a column, a wave (or two) 8 rows
    const int c0 = ct * BM, gr = t >> 3, gk = (t & 7) * 4, wn = t % BM, wk = wave / (BM / 64) * 8;
    const Run run(v0 * co, V * co);
    const bool ragged = v0 + BN + 4 >= V;                                        // 4 values of a row may pass the array's end (rows may be as short as 1)
    const float *__restrict__ gy = a.gy + run.first, *__restrict__ w = a.w + min(c0 + wn, ci - 1);
    if (yc != nullptr) yc += run.first;
    v4f G[DEPTH][GP];
    unsigned Y[DEPTH][GP];
    float W[DEPTH][WG][8];
    auto load = [&](v4f (&G)[GP], unsigned (&Y)[GP], float (&W)[WG][8], int k0) {
        if (yc != nullptr) {
#pragma unroll
            for (int i = 0; i < GP; ++i) Y[i] = get4(yc + run.at((i * 32 + gr) * co + k0 + gk));
        }
#pragma unroll
        for (int i = 0; i < GP; ++i) G[i] = get4(gy + run.at((i * 32 + gr) * co + k0 + gk));
#pragma unroll
        for (int i = 0; i < WG; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) W[i][j] = w[(long long)min(k0 + wk + i * (THREADS / BM) * 8 + j, ke - 1) * ci];
    };
    v16f acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = v16f{};
    const int wm = wave / WN * TM * 32, wv = wave % WN * TN * 32;
    auto step = [&](v4f (&G)[GP], unsigned (&Y)[GP], float (&W)[WG][8], int k0) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < GP; ++i) {
            v4f g = G[i];
            if (ragged) g = run.fix(g, (i * 32 + gr) * co + k0 + gk);
            if (yc != nullptr) g = masked(g, ragged ? run.fix(Y[i], (i * 32 + gr) * co + k0 + gk) : Y[i]);
            if (k0 + KSTEP > ke) {
#pragma unroll
                for (int j = 0; j < 4; ++j) g[j] = k0 + gk + j < ke ? g[j] : 0.0f;
            }
            put4(s_g + (i * 32 + gr) * KROW + gk, BN * KROW, g);
            if (g_out != nullptr && ct == 0) {
                const long long v = v0 + i * 32 + gr;
                float *to = g_out + v * co + k0 + gk;
                const int left = ke - k0 - gk;
                if (v < V) {
                    if (left >= 4) *reinterpret_cast<Io<float>::vec *>(to) = g;
                    else
#pragma unroll
                        for (int j = 0; j < 3; ++j) if (j < left) to[j] = g[j];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < WG; ++i) {
            if (k0 + KSTEP > ke) {
#pragma unroll
                for (int j = 0; j < 8; ++j) W[i][j] = k0 + wk + i * (THREADS / BM) * 8 + j < ke ? W[i][j] : 0.0f;
            }
            const Split8 p = split8(W[i]);
            uint16_t *to = s_w + wn * KROW + wk + i * (THREADS / BM) * 8;
            *reinterpret_cast<v4u *>(to) = __builtin_bit_cast(v4u, p.hi);
            *reinterpret_cast<v4u *>(to + BM * KROW) = __builtin_bit_cast(v4u, p.mid);
            *reinterpret_cast<v4u *>(to + 2 * BM * KROW) = __builtin_bit_cast(v4u, p.lo);
        }
        if (k0 + DEPTH * KSTEP < ke) load(G, Y, W, k0 + DEPTH * KSTEP);
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            v8bf A[TM][3], B[TN][3];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
#pragma unroll
                for (int m = 0; m < TM; ++m) A[m][p] = row_of(s_w + (p * BM + wm + m * 32 + lo) * KROW + ks * 16 + 8 * half);
#pragma unroll
                for (int n = 0; n < TN; ++n) B[n][p] = row_of(s_g + (p * BN + wv + n * 32 + lo) * KROW + ks * 16 + 8 * half);
            }
            // small products first; each pass over the tiles leaves every accumulator time to settle
#pragma unroll
            for (int e = 0; e < 6; ++e) {
                constexpr int PA[6] = {2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
                for (int m = 0; m < TM; ++m)
#pragma unroll
                    for (int n = 0; n < TN; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[m][PA[e]], B[n][PB[e]], acc[m][n], 0, 0, 0);
            }
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) if (kb + d * KSTEP < ke) load(G[d], Y[d], W[d], kb + d * KSTEP);
    for (int k0 = kb; k0 < ke; k0 += DEPTH * KSTEP) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) if (k0 + d * KSTEP < ke) step(G[d], Y[d], W[d], k0 + d * KSTEP);
    }
#pragma unroll
    for (int n = 0; n < TN; ++n) {
        const long long v = v0 + wv + n * 32 + lo;
        if (v >= V) continue;
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = c0 + wm + m * 32 + 8 * q + 4 * half;
                float *to = gx + v * ci + c;
                if (c + 4 <= ci) *reinterpret_cast<Io<float>::vec *>(to) = v4f{acc[m][n][4 * q], acc[m][n][4 * q + 1], acc[m][n][4 * q + 2], acc[m][n][4 * q + 3]};
                else
#pragma unroll
                    for (int j = 0; j < 3; ++j) if (c + j < ci) to[j] = acc[m][n][4 * q + j];
            }
    }
}

// gw and gbias, partial sums over ranges of voxels.  M = co, N = ci, K = voxel: a thread loads 4 channels of 4 voxels and turns them in registers.
struct WgradGrid { int co_tiles, ci_tiles; long long per, splits, groups; };
template <int WM, int TM, int WN, int TN, bool EVEN>
__device__ __forceinline__ void wgrad_tile(uint16_t *smem, const Args &a, const WgradGrid &grid, unsigned id)
{
    constexpr int BM = WM * TM * 32, BN = WN * TN * 32, GU = BM / 4 * 8, XU = BN / 4 * 8;
    constexpr bool APART = GU + XU <= THREADS;                                   // few enough units for a thread to load one kind only
    const uint8_t *__restrict__ yc = a.yc;
    const long long V = a.V;
    const int ci = a.ci, co = a.co, x_relu = a.x_relu;
    uint16_t *s_g = smem, *s_x = smem + 3 * BM * KROW;
    const int t = threadIdx.x, l = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), half = l >> 5, lo = l & 31;
    const unsigned turn = id % 8 * (unsigned)(grid.groups / 8) + id / 8, tile = turn % (grid.co_tiles * grid.ci_tiles);
    const long long split = turn / (grid.co_tiles * grid.ci_tiles);
    if (split >= grid.splits) return;
    const int bx = tile % grid.ci_tiles, by = tile / grid.ci_tiles;
    const long long v0 = split * grid.per, v1 = v0 + grid.per < V ? v0 + grid.per : V;
    const bool do_g = t < GU, do_x = a.xc != nullptr && (APART ? t >= GU && t < GU + XU : t < XU);
    const int ux = APART ? t - GU : t;
    // neighbouring lanes take neighbouring voxels of the same channels: 8 of them fill a row of LDS
    const int gc = t / 8 * 4, gv = t % 8 * 4, xn = ux / 8 * 4, xv = ux % 8 * 4, c0 = by * BM, n0 = bx * BN;
    const long long last_scale = (V * ci - 1) >> 5;
    struct Ahead { v4f G[4]; unsigned Y[4], X[4]; int S[4], S3[4]; } ahead[2];    // two steps' loads
    // channels behind co or ci belong to the next voxels and end in rows and columns that are not stored
    auto load = [&](Ahead &h, long long v) {
        if (do_g) {
            const Run run(v * co, V * co);
            if (yc != nullptr) {
#pragma unroll
                for (int j = 0; j < 4; ++j) h.Y[j] = get4(yc + run.first + run.at((gv + j) * co + c0 + gc));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) h.G[j] = get4(a.gy + run.first + run.at((gv + j) * co + c0 + gc));
        }
        if (do_x) {
            const Run run(v * ci, V * ci);                                       // v is a multiple of 32: the run begins with a block
            const uint8_t *ps = a.xs + (v * ci >> 5);
            const int most = (int)min(last_scale - (v * ci >> 5), 1LL << 30);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int off = (xv + j) * ci + n0 + xn;
                h.X[j] = get4(a.xc + run.first + run.at(off));
                h.S[j] = ps[(unsigned)min(off >> 5, most)];
                if (!EVEN) h.S3[j] = ps[(unsigned)min((off + 3) >> 5, most)];    // 4 values may reach into the next block
            }
        }
    };
    v16f acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = v16f{};
    v4f bsum = {};
    const int wm = wave / WN * TM * 32, wx = wave % WN * TN * 32;
    auto step = [&](Ahead &h, long long v) {
        const bool ragged = v + KSTEP + 4 >= V;
        __syncthreads();
        if (do_g) {
            const Run run(v * co, V * co);
            v4f g[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int off = (gv + j) * co + c0 + gc;
                g[j] = ragged ? run.fix(h.G[j], off) : h.G[j];
                if (yc != nullptr) g[j] = masked(g[j], ragged ? run.fix(h.Y[j], off) : h.Y[j]);
                if (v + KSTEP > v1 && v + gv + j >= v1) g[j] = v4f{};
            }
            bsum = bsum + ((g[0] + g[1]) + (g[2] + g[3]));
#pragma unroll
            for (int c = 0; c < 4; ++c) put4(s_g + (gc + c) * KROW + gv, BM * KROW, v4f{g[0][c], g[1][c], g[2][c], g[3][c]});
        }
        if (do_x) {
            const Run run(v * ci, V * ci);
            float f[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int off = (xv + j) * ci + n0 + xn;
                const unsigned x = ragged ? run.fix(h.X[j], off) : h.X[j];
#pragma unroll
                for (int c = 0; c < 4; ++c) f[j][c] = code_value(x >> (8 * c) & 255u, x_relu, EVEN || (off & 31) + c < 32 ? h.S[j] : h.S3[j]);
                if (v + KSTEP > v1 && v + xv + j >= v1) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) f[j][c] = 0.0f;
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint2 p;
                p.x = pack_hi(f[0][c], f[1][c]);
                p.y = pack_hi(f[2][c], f[3][c]);
                *reinterpret_cast<uint2 *>(s_x + (xn + c) * KROW + xv) = p;
            }
        }
        if (v + 2 * KSTEP < v1) load(h, v + 2 * KSTEP);
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            v8bf A[TM][3], B[TN];
#pragma unroll
            for (int n = 0; n < TN; ++n) B[n] = row_of(s_x + (wx + n * 32 + lo) * KROW + ks * 16 + 8 * half);
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int m = 0; m < TM; ++m) A[m][p] = row_of(s_g + (p * BM + wm + m * 32 + lo) * KROW + ks * 16 + 8 * half);
#pragma unroll
            for (int p = 2; p >= 0; --p)
#pragma unroll
                for (int m = 0; m < TM; ++m)
#pragma unroll
                    for (int n = 0; n < TN; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[m][p], B[n], acc[m][n], 0, 0, 0);
        }
    };
    load(ahead[0], v0);
    if (v0 + KSTEP < v1) load(ahead[1], v0 + KSTEP);
    for (long long v = v0; v < v1; v += 2 * KSTEP) {
        step(ahead[0], v);
        if (v + KSTEP < v1) step(ahead[1], v + KSTEP);
    }
    float *pw = a.part_w + split * co * ci;
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int o = by * BM + wm + m * 32 + 8 * (i / 4) + 4 * half + i % 4, c = bx * BN + wx + n * 32 + lo;
                if (o < co && c < ci) pw[(long long)o * ci + c] = acc[m][n][i];
            }
    if (bx != 0) return;
    __syncthreads();
    float *s_b = reinterpret_cast<float *>(s_g);                                 // [8 voxel groups][BM]
    if (do_g) *reinterpret_cast<v4f *>(s_b + t % 8 * BM + gc) = bsum;
    __syncthreads();
    if (t < BM && by * BM + t < co) {
        float b = 0.0f;
#pragma unroll
        for (int g = 0; g < 8; ++g) b = b + s_b[g * BM + t];
        a.part_b[split * co + by * BM + t] = b;
    }
}

// arrays of less than 4 values, which the loads of 4 above cannot read: an element of gx or gw a thread, gbias and g in plain loops
__global__ __launch_bounds__(THREADS) void conv1x1_bwd_act8_tiny(Args a, float *__restrict__ gw, float *__restrict__ gb)
{
    const long long e = (long long)blockIdx.x * THREADS + threadIdx.x, nx = a.V * a.ci, nw = (long long)a.co * a.ci, ng = a.V * a.co;
    auto g_at = [&](long long v, int o) { return a.yc == nullptr || a.yc[v * a.co + o] ? a.gy[v * a.co + o] : 0.0f; };
    float t = 0.0f;
    if (e < nx) {
        if (a.gx == nullptr) return;
        for (int o = 0; o < a.co; ++o) t = t + g_at(e / a.ci, o) * a.w[(long long)o * a.ci + e % a.ci];
        a.gx[e] = t;
    } else if (e < nx + nw) {
        if (gw == nullptr) return;
        const int o = (int)((e - nx) / a.ci), i = (int)((e - nx) % a.ci);
        for (long long v = 0; v < a.V; ++v) t = t + g_at(v, o) * code_value(a.xc[v * a.ci + i], a.x_relu, a.xs[(v * a.ci + i) >> 5]);
        gw[e - nx] = t;
    } else if (e < nx + nw + a.co) {
        if (gb == nullptr) return;
        for (long long v = 0; v < a.V; ++v) t = t + g_at(v, (int)(e - nx - nw));
        gb[e - nx - nw] = t;
    } else if (e < nx + nw + a.co + ng && a.g != nullptr) {
        const long long i = e - nx - nw - a.co;
        a.g[i] = g_at(i / a.co, (int)(i % a.co));
    }
}

// one launch for the two products, which do not depend on each other: the first groups sum voxels, the others channels
template <int W0, int W1, int W2, int W3, int D0, int D1, int D2, int D3, bool EVEN>
__global__ __launch_bounds__(THREADS, 2) void conv1x1_bwd_act8_products(Args a, WgradGrid wg, DgradGrid dg)
{
    constexpr int LW = (W0 * W1 * 3 + W2 * W3) * 32 * KROW, LD = (D0 * D1 + D2 * D3) * 3 * 32 * KROW;
    __shared__ __attribute__((aligned(16))) uint16_t smem[LW > LD ? LW : LD];
    if (blockIdx.x < wg.groups) wgrad_tile<W0, W1, W2, W3, EVEN>(smem, a, wg, blockIdx.x);
    else dgrad_tile<D0, D1, D2, D3>(smem, a, dg, blockIdx.x - (unsigned)wg.groups);
}

// out[e] = sum over the splits of part[split][e] in a fixed order, for up to three arrays at once.  A workgroup sums 1024 >> log_r elements, each in 1 << log_r
// interleaved ranges of splits: the fewest that make two workgroups a CU (512 partial sums of 18 x 72 weights in 8 ranges: 21 us, in 32: 5 us; 13 partial sums of 384 x 1536 weights
// in 8: 13.5 us, in 1: 8 us).
struct Joined { const float *part; float *out; long long n; int splits, log_r; long long groups; };
__global__ __launch_bounds__(1024) void conv1x1_bwd_act8_join(Joined j0, Joined j1, Joined j2)
{
    __shared__ float s[1024];
    long long id = blockIdx.x;
    Joined j = j0;
    if (id >= j0.groups) { id -= j0.groups; j = j1; if (id >= j1.groups) { id -= j1.groups; j = j2; } }
    const int per = 1024 >> j.log_r, lane = threadIdx.x & (per - 1), range = threadIdx.x >> (10 - j.log_r), R = 1 << j.log_r;
    const long long e = id * per + lane;
    float acc = 0.0f;
    if (e < j.n) {
        const float *p = j.part + e;
        int k = range;
        for (; k + 3 * R < j.splits; k += 4 * R) {
            const float a = p[k * j.n], b = p[(k + R) * j.n], c = p[(k + 2 * R) * j.n], d = p[(k + 3 * R) * j.n];
            acc = acc + ((a + b) + (c + d));
        }
        for (; k < j.splits; k += R) acc = acc + p[k * j.n];
    }
    s[threadIdx.x] = acc;
    __syncthreads();
    if (range != 0 || e >= j.n) return;
    acc = 0.0f;
    for (int r = 0; r < R; ++r) acc = acc + s[r * per + lane];
    j.out[e] = acc;
}

inline Joined joined(const float *part, float *out, long long n, long long splits)
{
    Joined j = {part, out, out ? n : 0, (int)splits, 0, 0};
    while (j.log_r < 5 && (j.n >> (10 - j.log_r)) < 512 && (splits >> j.log_r) > 4) ++j.log_r;
    j.groups = (j.n + (1024 >> j.log_r) - 1) / (1024 >> j.log_r);
    return j;
}

int join_run(const Joined &a, const Joined &b, const Joined &c, hipStream_t s)
{
    const long long groups = a.groups + b.groups + c.groups;
    if (groups >= (1LL << 22)) return MDT_ERR_UNSUPPORTED;                        // 2^32 threads are the most of a launch
    if (groups > 0) conv1x1_bwd_act8_join<<<dim3((unsigned)groups), 1024, 0, s>>>(a, b, c);
    return MDT_OK;
}

// ---- no product wanted: the mask and the sum of columns -----------------------------------------------------------------------------------------
// g = gy . m and gbias for a layer whose products other kernels take (a window, a stride).  5 bytes read and 4 written a value: 1 M x 18 in 34 us, 5.0 TB/s.
// A workgroup walks over its run of quads of values in steps of `active` quads, a multiple of the period after which quads begin at the same channel again: a thread's 4
// sums belong to the same 4 channels throughout, whatever the number of channels, as long as the period fits into a workgroup.
constexpr int SUM_ROWS = 1024;                                                   // partial sums of a channel at most (1 M x 18: 512 34.2 us, 1024 34.1, 2048 38.5; 100000 x 257: 80, 56, 55)

template <bool MASK>
__global__ __launch_bounds__(THREADS) void act8_mask_sum_quads(const float *__restrict__ gy, const uint8_t *__restrict__ yc, float *__restrict__ g, float *__restrict__ part, long long n,
                                                               int C, int active, long long per)
{
    __shared__ __attribute__((aligned(16))) float s[4 * THREADS];
    const int t = threadIdx.x;
    const long long nq = n / 4, q0 = blockIdx.x * per, q1 = min(q0 + per, nq);
    v4f sum = {};
    if (t < active)
        for (long long q = q0 + t; q < q1; q += 4 * active) {
            v4f v[4];
            unsigned m[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const long long at = 4 * min(q + u * active, nq - 1);
                if (MASK) m[u] = get4(yc + at);
                v[u] = get4(gy + at);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (q + u * active >= q1) break;
                if (MASK) v[u] = masked(v[u], m[u]);
                if (g != nullptr) *reinterpret_cast<Io<float>::vec *>(g + 4 * (q + u * active)) = v[u];
                sum = sum + v[u];
            }
        }
    *reinterpret_cast<v4f *>(s + 4 * t) = sum;
    __syncthreads();
    const int behind = blockIdx.x == gridDim.x - 1 ? (int)(n - 4 * nq) : 0;        // values behind the last quad
    for (int c = t; c < C; c += THREADS) {
        float b = 0.0f;
        for (int e = c; e < 4 * active; e += C) b = b + s[e];
        for (int k = 0; k < behind; ++k) {
            const long long e = 4 * nq + k;
            if (e % C != c) continue;
            const float v = !MASK || yc[e] ? gy[e] : 0.0f;
            if (g != nullptr) g[e] = v;
            b = b + v;
        }
        if (part != nullptr) part[(long long)blockIdx.x * C + c] = b;
    }
}

// channels whose period is longer than a workgroup: a thread a column
template <bool MASK>
__global__ __launch_bounds__(THREADS) void act8_mask_sum_columns(const float *__restrict__ gy, const uint8_t *__restrict__ yc, float *__restrict__ g, float *__restrict__ part, long long V,
                                                                 int C, long long per)
{
    const int c = blockIdx.x * THREADS + threadIdx.x;
    const long long v0 = blockIdx.y * per, v1 = min(v0 + per, V);
    if (c >= C) return;
    float sum = 0.0f;
    for (long long r = v0; r < v1; r += 4) {
        float v[4];
        uint8_t m[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const long long at = min(r + u, V - 1) * C + c;
            if (MASK) m[u] = yc[at];
            v[u] = gy[at];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (r + u >= v1) break;
            if (MASK && !m[u]) v[u] = 0.0f;
            if (g != nullptr) g[(r + u) * C + c] = v[u];
            sum = sum + v[u];
        }
    }
    if (part != nullptr) part[blockIdx.y * (long long)C + c] = sum;
}

struct SumPlan { int active, rows; long long per; };                              // active 0: a thread a column

inline SumPlan sum_plan(long long V, int C)
{
    SumPlan p;
    const int period = C % 4 == 0 ? C / 4 : C % 2 == 0 ? C / 2 : C;
    p.active = period <= THREADS ? THREADS / period * period : 0;
    const long long units = p.active ? (V * C + 4LL * p.active - 1) / (4LL * p.active) : V, columns = (C + THREADS - 1) / THREADS, most = p.active ? SUM_ROWS : (SUM_ROWS + columns - 1) / columns;
    const long long rows = (units + 3) / 4 < most ? (units + 3) / 4 : most;
    const long long each = (units + rows - 1) / rows;
    p.per = p.active ? each * p.active : each;
    p.rows = (int)((units + each - 1) / each);
    return p;
}

template <bool MASK>
void sum_run(const SumPlan &p, const Args &a, hipStream_t s)
{
    if (p.active) act8_mask_sum_quads<MASK><<<p.rows, THREADS, 0, s>>>(a.gy, a.yc, a.g, a.part_b, a.V * a.co, a.co, p.active, p.per);
    else act8_mask_sum_columns<MASK><<<dim3((a.co + THREADS - 1) / THREADS, p.rows), THREADS, 0, s>>>(a.gy, a.yc, a.g, a.part_b, a.V, a.co, p.per);
}

// floats of one wave's LDS tiles: 32 voxels of gradients (and a row's overhang; gx's rows take the same place later), 32 of bf16 inputs (and theirs)
__host__ __device__ constexpr int fused_rows_floats(int mt, int ci, int co) { return 32 * (co > ci ? co : ci) + 32 * mt; }
__host__ __device__ constexpr int fused_wave_floats(int mt, int nt, int ci, int co) { return (fused_rows_floats(mt, ci, co) + (32 * ci + 32 * nt) / 2 + 3) / 4 * 4; }

// regions of LDS for the waves' sums at the end: 9 tiles for each of 4 waves are 147 KB
__host__ __device__ constexpr int fused_regions(int tiles) { return tiles <= 9 ? WAVES : 2; }

// ---- both products in one pass, for few channels --------------------------------------------------------------------------------------------
// A wave takes 32 voxels at a time and needs no other wave: their 32 co gradients are one contiguous run, loaded 16 bytes a lane, masked, and put into the
// wave's own LDS tile as they are; their 32 ci input codes are ci whole blocks.  From the tile gw takes columns (M = co, N = ci, K = voxel) and gx takes rows
// (M = ci, N = voxel, K = co), both cut into bf16 pieces in registers; gw stays in registers over all of a wave's voxels.  gx's tile replaces the gradients in LDS
// and leaves as the contiguous run that it is, like g.
// Used while gw takes at most 10 tiles of 32 x 32 of a side of at most 160 (what registers hold): narrow layers gain (100000 voxels 32 -> 160: 48 us, tiled 70; 36 -> 144: 59,
// 67; 144 -> 36: 56, 68), square ones are equal (64 -> 64: 53, 50; 96 -> 64: 47, 45; 64 -> 96: 45, 48).
// 1 M voxels 18 -> 72 with g: 163 us, 4.8 TB/s of its 155 us floor; 72 -> 18: 118 us, 4.0 TB/s (floor 95); 131072 voxels 36 -> 144 with g: 70 us (floor 39), 144 -> 36: 59 (24): memory, and the waits of a wave's chunk where no other wave covers
// them.  A call of few voxels is one chunk's chain of loads, LDS and products: 32 voxels 8 us.
// Loads and stores share one in-order counter: the next chunk's loads are issued before this chunk's stores and every chunk issues the same number of
// stores, so that the wait for the loads does not wait for the stores behind them.
// Entries of the tiles behind co or ci hold whatever follows in LDS: they only reach rows and columns that are not stored, except along gx's sum, where
// they are set to zero.
template <int MT, int NT, bool G_OUT>
__global__ __launch_bounds__(THREADS, MT * NT <= 3 ? 2 : 1) void conv1x1_bwd_act8_fused(const float *__restrict__ gy, const uint8_t *__restrict__ yc, const float *__restrict__ w,
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
    const long long chunks = (V + 31) / 32, full = V / 32, step = (long long)gridDim.x * WAVES, last_scale = (V * ci - 1) >> 5;
    long long chunk = (long long)blockIdx.x * WAVES + wave;
    v4f G[4 * MT];
    unsigned Y[4 * MT], X[4 * NT];
    int S[4 * NT];
    // lanes behind the chunk's end repeat its last 16 bytes (and store them to the same place again)
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
        const Run rg(c * 32 * co, V * co), rx(c * 32 * ci, V * ci);
        // 16 bytes behind the chunk's end or the array's: the last ones again
        const int g0 = 4 * ln + rg.delta, x0 = 4 * ln + rx.delta, g1 = min(32 * co - 4 + rg.delta, rg.last), x1 = min(32 * ci - 4 + rx.delta, rx.last);
        const int s0 = ln >> 3, s1 = (int)min(last_scale - c * ci, ci - 1LL);
        const float *pg = gy + rg.first;
        const uint8_t *py = yc + rg.first, *px = xc + rx.first, *ps = xs + c * ci;
        if (yc != nullptr) {
#pragma unroll
            for (int q = 0; q < 4 * MT; ++q) Y[q] = get4(py + (unsigned)min(g0 + q * 256, g1));
        }
#pragma unroll
        for (int q = 0; q < 4 * NT; ++q) {
            X[q] = get4(px + (unsigned)min(x0 + q * 256, x1));
            S[q] = ps[(unsigned)min(s0 + q * 8, s1)];
        }
#pragma unroll
        for (int q = 0; q < 4 * MT; ++q) G[q] = get4(pg + (unsigned)min(g0 + q * 256, g1));
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
    if (chunk < chunks) load(chunk);
    for (int t = threadIdx.x; t < NT * KS * 64; t += THREADS) {
        const int ll = t & 63, n = (t / 64 / KS) * 32 + (ll & 31), k = (t / 64 % KS) * 16 + 8 * (ll >> 5);
        float b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = w[min(k + j, co - 1) * ci + min(n, ci - 1)];
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = n < ci && k + j < co ? b[j] : 0.0f;
        const Split8 B = split8(b);
        v4u *to = wp + (t / 64) * 3 * 64 + ll;
        to[0] = __builtin_bit_cast(v4u, B.hi);
        to[64] = __builtin_bit_cast(v4u, B.mid);
        to[128] = __builtin_bit_cast(v4u, B.lo);
    }
    __syncthreads();
    for (; chunk < chunks; chunk += step) {
        const bool whole = chunk < full;
        const unsigned lp = lane();
        if (!whole) {
            const Run rg(chunk * 32 * co, V * co), rx(chunk * 32 * ci, V * ci);
#pragma unroll
            for (int q = 0; q < 4 * MT; ++q) {
                G[q] = rg.fix(G[q], 4 * at_gy(lp, q));
                if (yc != nullptr) Y[q] = rg.fix(Y[q], 4 * at_gy(lp, q));
            }
#pragma unroll
            for (int q = 0; q < 4 * NT; ++q) {
                X[q] = rx.fix(X[q], 4 * at_x(lp, q));
            }
        }
#pragma unroll
        for (int q = 0; q < 4 * MT; ++q) {
            if (yc != nullptr) G[q] = masked(G[q], Y[q]);
            *reinterpret_cast<v4f *>(gs + 4 * at_gy(lp, q)) = G[q];
        }
#pragma unroll
        for (int q = 0; q < 4 * NT; ++q) {
            float t[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = code_value(X[q] >> (8 * j) & 255u, x_relu, S[q]);
            if (!whole) {                                                        // a scale of NaN must not reach the voxels behind the last one
                const int left = (int)(V - chunk * 32) * ci - 4 * (int)at_x(lp, q);
#pragma unroll
                for (int j = 0; j < 4; ++j) t[j] = j < left ? t[j] : 0.0f;
            }
            uint2 p;
            p.x = pack_hi(t[0], t[1]);
            p.y = pack_hi(t[2], t[3]);
            *reinterpret_cast<uint2 *>(xb + 4 * at_x(lp, q)) = p;
        }
        if (chunk + step < chunks) load(chunk + step);
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
        if (G_OUT) {
            float *pg = g_out + chunk * 32 * co;
            if (whole) {
                const unsigned ln = lane();
#pragma unroll
                for (int q = 0; q < 4 * MT; ++q) *reinterpret_cast<Io<float>::vec *>(pg + 4 * at_gy(ln, q)) = *reinterpret_cast<const v4f *>(gs + 4 * at_gy(ln, q));
            } else {
                for (int e = l; e < (V - chunk * 32) * co; e += 64) pg[e] = gs[e];
            }
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
    // the four waves' sums, in wave order: a region of LDS each, or one for two waves where four would not fit (one region, written in turn, took 7 us of a call's end)
    constexpr int REGIONS = fused_regions(MT * NT), REGION = 1024 * MT * NT + 32 * MT;
    float *sum = reinterpret_cast<float *>(smem) + wave % REGIONS * REGION, *sumb = sum + 1024 * MT * NT;
#pragma unroll
    for (int turn = 0; turn < WAVES / REGIONS; ++turn) {
        __syncthreads();
        if (wave / REGIONS != turn) continue;
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
    const float *all = reinterpret_cast<const float *>(smem);
    auto total = [&](int at) {
        float r = all[at];
#pragma unroll
        for (int k = 1; k < REGIONS; ++k) r = r + all[k * REGION + at];
        return r;
    };
    for (int t = threadIdx.x; t < co * ci; t += THREADS) part_w[(long long)blockIdx.x * co * ci + t] = total((t / ci) * 32 * NT + t % ci);
    for (int t = threadIdx.x; t < co; t += THREADS) part_b[(long long)blockIdx.x * co + t] = total(1024 * MT * NT + t);
}

// Tiles of the two products.  gx: 128 channels x 128 voxels where that gives a workgroup a CU (20000 voxels 300 -> 400: 108 us, 64 x 64 124; 100000 voxels 200 -> 250: 205,
// 264), else 128 x 64, or 64 x 64 where 128 would be padded (1620 voxels 1536 -> 384: 128 x 64 46 us, 64 x 64 52; 16384 voxels 72 -> 288: 31, 36; 6480 voxels 192 -> 768: 57,
// 48); where even those leave CUs idle, the sum over co is split (at least 4 steps each; 400 voxels 1000 -> 1000: 30 us, unsplit 63, twice as many ranges 32) and joined with gw's.  gw: 64 or
// 128 along each axis; its sum is split so that both products together fill whole rounds of the two workgroups that a CU holds, at least 128 of them and at least 128
// voxels each (1620 voxels 1536 -> 384: 13 ranges 64 us, 11 of them 50; 6480 voxels 192 -> 768: 43 ranges 68 us, 17 52).  Figures of whole calls, host work included.  The rules for both
// sums hold at these sizes; 1300 voxels 1000 -> 1000 they cost 8 us (63 -> 71).
struct Plan { int w_m, w_n, d_m, d_n; WgradGrid wg; DgradGrid dg; };
inline Plan plan_of(long long V, int ci, int co)
{
    Plan p;
    p.w_m = co > 64 ? 128 : 64;
    p.w_n = ci > 64 ? 128 : 64;
    WgradGrid &w = p.wg;
    w.co_tiles = (co + p.w_m - 1) / p.w_m;
    w.ci_tiles = (ci + p.w_n - 1) / p.w_n;
    DgradGrid &d = p.dg;
    const long long big = ((V + 127) / 128) * ((ci + 127) / 128);
    p.d_n = ci > 64 && big >= 256 ? 128 : 64;
    p.d_m = p.d_n == 128 || (ci + 63) / 64 % 2 == 0 ? 128 : 64;
    d.ci_tiles = (ci + p.d_m - 1) / p.d_m;
    const long long ranges = (V + p.d_n - 1) / p.d_n, now = ranges * d.ci_tiles;
    const int steps = (co + KSTEP - 1) / KSTEP;
    long long ks = (now + 255) / now;
    if (ks > steps / 4) ks = steps / 4;
    if (ks < 1) ks = 1;
    d.k_per = (int)((steps + ks - 1) / ks) * KSTEP;
    d.k_splits = (co + d.k_per - 1) / d.k_per;
    d.groups = (ranges * d.ci_tiles * d.k_splits + 7) / 8 * 8;
    const long long tiles = (long long)w.co_tiles * w.ci_tiles, most = (V + 127) / 128;
    const long long rounds = (d.groups + 128 + 511) / 512;
    long long splits = (rounds * 512 - d.groups) / tiles;
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    w.per = ((V + splits - 1) / splits + KSTEP - 1) / KSTEP * KSTEP;
    w.splits = (V + w.per - 1) / w.per;
    w.groups = (w.splits * tiles + 7) / 8 * 8;
    d.to = nullptr;
    return p;
}

template <int W0, int W1, int W2, int W3>
void products_launch(const Plan &p, const Args &a, hipStream_t s)
{
    const dim3 grid((unsigned)(p.wg.groups + p.dg.groups));
    const bool even = a.ci % 4 == 0;                                            // 4 input codes of a voxel lie in one block
    const auto kernel = p.d_n == 128 ? (even ? conv1x1_bwd_act8_products<W0, W1, W2, W3, 2, 2, 2, 2, true> : conv1x1_bwd_act8_products<W0, W1, W2, W3, 2, 2, 2, 2, false>)
                      : p.d_m == 128 ? (even ? conv1x1_bwd_act8_products<W0, W1, W2, W3, 2, 2, 2, 1, true> : conv1x1_bwd_act8_products<W0, W1, W2, W3, 2, 2, 2, 1, false>)
                                     : (even ? conv1x1_bwd_act8_products<W0, W1, W2, W3, 2, 1, 2, 1, true> : conv1x1_bwd_act8_products<W0, W1, W2, W3, 2, 1, 2, 1, false>);
    kernel<<<grid, THREADS, 0, s>>>(a, p.wg, p.dg);
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
    const int sums = fused_regions(tiles) * (1024 * tiles + 32 * p.mt) * 4;
    if (p.lds < sums) p.lds = sums;
    if (p.lds > 160 * 1024) return {0, 0, 0, 0};
    const int per_cu = tiles <= 3 ? 2 : 1, fit = 160 * 1024 / p.lds, at_once = 256 * (fit < per_cu ? fit : per_cu);
    const long long want = (V + 32 * WAVES - 1) / (32 * WAVES);
    p.blocks = (int)(want < at_once ? want : at_once);
    return p;
}

template <int MT, int NT>
int fused_launch(const FusedPlan &p, const Args &a, hipStream_t s)
{
    const auto kernel = a.g != nullptr ? conv1x1_bwd_act8_fused<MT, NT, true> : conv1x1_bwd_act8_fused<MT, NT, false>;
    if (p.lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, p.lds) != hipSuccess) return MDT_ERR_LAUNCH_FAILED;
    kernel<<<p.blocks, THREADS, p.lds, s>>>(a.gy, a.yc, a.w, a.xc, a.xs, a.gx, a.g, a.part_w, a.part_b, a.V, a.ci, a.co, a.x_relu);
    return MDT_OK;
}

int fused_run(const FusedPlan &p, const Args &a, hipStream_t s)
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
    const Plan q = plan_of(n_voxels, c_in, c_out);
    const FusedPlan p = fused_plan(n_voxels, c_in, c_out);
    const long long one = (long long)c_in * c_out + c_out, tiled = q.wg.splits * one + (q.dg.k_splits > 1 ? q.dg.k_splits * n_voxels * c_in : 0);
    const long long fused = p.blocks * one, sums = (long long)sum_plan(n_voxels, c_out).rows * c_out, more = tiled > fused ? tiled : fused;
    return (size_t)(more > sums ? more : sums) * 4 + 256;
}

int mdt_conv1x1_act8_backward(const float *gy, const float *w, const void *x_codes, const void *x_scales, int x_relu, const void *y_codes, float *gx, float *gw, float *gbias, float *g,
                              long long n_voxels, int c_in, int c_out, void *workspace, size_t workspace_bytes, void *stream)
{
    if (n_voxels < 0 || n_voxels > (1LL << 30) || c_in < 1 || c_out < 1 || c_in > 65536 || c_out > 65536) return MDT_ERR_INVALID_ARGUMENT;
    const hipStream_t s = (hipStream_t)stream;
    const bool sums = gw != nullptr || gbias != nullptr;
    const long long V = n_voxels, nw = (long long)c_in * c_out;
    const Joined none = {nullptr, nullptr, 0, 0, 0, 0};
    if (V == 0) {                                                                // sums over no voxels
        const int rc = join_run(joined(nullptr, gw, nw, 0), joined(nullptr, gbias, c_out, 0), none, s);
        return rc != MDT_OK ? rc : launch_check();
    }
    if (!gy || (gx && !w) || (gw && (!x_codes || !x_scales)) || ((uintptr_t)x_codes & 3) || ((uintptr_t)y_codes & 3)) return MDT_ERR_INVALID_ARGUMENT;
    if ((sums || gx) && (workspace == nullptr || workspace_bytes < mdt_conv1x1_act8_backward_workspace_bytes(V, c_in, c_out))) return MDT_ERR_WORKSPACE_TOO_SMALL;
    Args a = {gy, (const uint8_t *)y_codes, w, (const uint8_t *)x_codes, (const uint8_t *)x_scales, gx, g, (float *)workspace, nullptr, V, c_in, c_out, x_relu};
    const FusedPlan f = gx && gw ? fused_plan(V, c_in, c_out) : FusedPlan{0, 0, 0, 0};
    if (f.mt > 0 && V * c_in >= 4 && V * c_out >= 4) {
        a.part_b = a.part_w + f.blocks * nw;
        if (f.blocks == 1) {                                                     // nothing to join
            a.part_w = gw;
            if (gbias) a.part_b = gbias;
        }
        const int rc = fused_run(f, a, s);
        if (rc != MDT_OK || f.blocks == 1) return rc != MDT_OK ? rc : launch_check();
        const int rj = join_run(joined(a.part_w, gw, nw, f.blocks), joined(a.part_b, gbias, c_out, f.blocks), none, s);
        return rj != MDT_OK ? rj : launch_check();
    }
    if (V * c_in < 4 || V * c_out < 4) {
        const long long n = V * c_in + nw + c_out + V * c_out;
        conv1x1_bwd_act8_tiny<<<dim3((unsigned)((n + THREADS - 1) / THREADS)), THREADS, 0, s>>>(a, gw, gbias);
        return launch_check();
    }
    if (gx == nullptr && (g != nullptr || gw == nullptr)) {
        if (g == nullptr && gbias == nullptr) return launch_check();
        const SumPlan sp = sum_plan(V, c_out);
        a.part_b = gbias ? a.part_w : nullptr;
        if (y_codes) sum_run<true>(sp, a, s);
        else sum_run<false>(sp, a, s);
        const int rc = join_run(joined(a.part_b, gbias, c_out, sp.rows), none, none, s);
        if (rc != MDT_OK || gw == nullptr) return rc != MDT_OK ? rc : launch_check();
        a.g = g = nullptr;
        gbias = nullptr;
    }
    Plan p = plan_of(V, c_in, c_out);
    a.part_b = a.part_w + p.wg.splits * nw;
    float *part_x = a.part_b + p.wg.splits * c_out;
    if (gw == nullptr) {                                                         // gbias alone: one column of tiles without inputs
        a.xc = nullptr;
        p.wg.groups = sums ? (p.wg.splits * p.wg.co_tiles + 7) / 8 * 8 : 0;
        p.wg.ci_tiles = 1;
    }
    if (gx == nullptr) {
        p.dg.groups = 0;
        p.dg.k_splits = 1;
    }
    p.dg.to = p.dg.k_splits > 1 ? part_x : gx;
    if (p.wg.groups + p.dg.groups >= (1LL << 24)) return MDT_ERR_UNSUPPORTED;    // 2^32 threads are the most of a launch
    if (p.wg.groups + p.dg.groups > 0) {
        if (p.w_m == 128 && p.w_n == 128) products_launch<2, 2, 2, 2>(p, a, s);
        else if (p.w_m == 128) products_launch<4, 1, 1, 2>(p, a, s);
        else if (p.w_n == 128) products_launch<1, 2, 4, 1>(p, a, s);
        else products_launch<2, 1, 2, 1>(p, a, s);
    }
    const int rj = join_run(joined(a.part_w, gw, nw, p.wg.splits), joined(a.part_b, gbias, c_out, p.wg.splits),
                            p.dg.k_splits > 1 ? joined(part_x, gx, V * c_in, p.dg.k_splits) : none, s);
    return rj != MDT_OK ? rj : launch_check();
}

}  // extern "C"
