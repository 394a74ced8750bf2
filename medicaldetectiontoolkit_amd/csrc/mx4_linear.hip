// mx4_linear.hip -- act(x W^T + bias) with both operands in 4-bit block-scaled codes (gfx950).
//
// The matrix units take 4-bit codes and one scale byte per 32 of them as they are (16 x 16 outputs, 128 summed values an instruction), products exact and sums
// in fp32.  W is kept in codes; x is rounded to codes on its way into the product, in one launch and without scratch memory, so x is read once and nothing
// else of its size is moved.
//
// Work goes in chunks of 256 summed values = 8 blocks.  A lane (r = lane % 16, q = lane / 16) holds blocks 2q and 2q + 1 of row r: 32 bytes of codes and 2 of
// scales.  x's come from LDS, where the lanes that loaded x put its codes (a row of a chunk is 64 lanes of 4 floats, or 32 lanes of 8 values of 16 bits, so a
// block's maximum is a few lane permutes).  W's come straight from memory into registers: for few rows of x from W as it is kept, where the 64 lanes of a
// load touch 16 rows and cost 64 requests; for more rows from a copy in the lanes' order, one contiguous kilobyte a load, that a first launch makes in the
// workspace (the 2D head, 10000 x 9408 -> 768: 151 us without the copy, 5 + 87 us with it).  With W as the first operand a lane ends up with 4 consecutive
// outputs of one row.
//
// Two shapes of the same loop:
//   narrow   every wave sums its own chunks (w, w + 8, ...) of a 16 x 16 TN tile, without any barrier, and the 8 waves' sums are joined in LDS at the end: few
//            outputs a row, or few rows, where only the summed axis is long
//   wide     the 8 waves share one 16 TM x 128 TN tile's x and take 16 TN columns each: many rows and many columns, where x must not be rounded again for
//            each range of columns
// What bounds them: x's bytes, and beside them the rounding and the waits of a chunk's barrier at 8 waves a CU.  4000 x 5292 -> 144, fp32: 4 + 25 us (x alone 17);
// 10000 x 9408 -> 768, bf16: 5 + 87 us, 1.6 PFLOP/s (x alone 38).  Two chunks of loads in flight in the wide shape: 96 us for 92 (9000 x 9000 -> 300) and spills at 768
// columns; 96 rows x half the columns a workgroup: 137 us for 95.
#include "block_scaled.h"

namespace {

using namespace mdt_bs;

constexpr int WAVES = 8;
constexpr int THREADS = 64 * WAVES;
constexpr int CHUNK = 256, CHUNK_BLOCKS = CHUNK / BLOCK;
constexpr int ROW_BYTES = CHUNK / 2 + 16;                   // a row of codes in LDS, padded: 16-byte reads of neighbouring rows fall into different banks


// a number that the optimiser takes for a new one: it would hold every address that it computes from a lane's number in a register of its own over the loop
__device__ __forceinline__ int fresh(int v)
{
    asm volatile("" : "+v"(v));
    return v;
}

// one lane's fragment of 16 rows of W for a chunk: blocks 2q and 2q + 1 of its row
struct Frag { v4u c[2]; unsigned s; };

// W as it is kept.  Loads take no branches (the number of loads in flight stays known, and a wait for one does not become a wait for all): rows behind the last one
// repeat it, blocks behind a row's end repeat its last one (x's codes are zero there) and get a finite scale.
template <bool ONE>                                         // ONE: rows of a single block
struct WKept {
    const uint8_t *codes, *scales;
    int mine, most, kb, q;                                   // in blocks: the lane's row within the tile, the last row
    __device__ __forceinline__ WKept(const uint8_t *wc, const uint8_t *ws, int n0, int n, int blocks, int l) : kb(blocks), q(l >> 4)
    {
        const int from = min(n0, n - 1);
        codes = wc + (long long)from * blocks * 16;
        scales = ws + (long long)from * blocks;
        mine = l % 16 * blocks;
        most = min(n - 1 - from, 1023) * blocks;             // more than a tile's rows
    }
    __device__ __forceinline__ void load(Frag &f, int t, int c) const
    {
        typedef uint16_t u16una __attribute__((aligned(1)));
        const int off = min(fresh(mine) + t * 16 * kb, most), b = c * CHUNK_BLOCKS + 2 * q;
        f.c[0] = *reinterpret_cast<const v4u *>(codes + (unsigned)(off + min(b, kb - 1)) * 16u);
        if (!ONE) f.c[1] = *reinterpret_cast<const v4u *>(codes + (unsigned)(off + min(b + 1, kb - 1)) * 16u);
        if (ONE) f.c[1] = v4u{};
        if (ONE) f.s = scales[(unsigned)off];
        else f.s = *reinterpret_cast<const u16una *>(scales + (unsigned)(off + min(b, kb - 2)));
    }
    __device__ __forceinline__ unsigned scale(const Frag &f, int c) const
    {
        const int b = c * CHUNK_BLOCKS + 2 * q;
        if ((c + 1) * CHUNK_BLOCKS <= kb) return f.s;
        return b + 1 < kb ? f.s : b < kb ? (ONE ? f.s : f.s >> 8) | 127u << 8 : 127u | 127u << 8;
    }
};

// the copy in the lanes' order: codes [tiles of 16 rows][chunks][2][64 lanes][16 bytes], scales [tiles][chunks][64 lanes][2]; zero codes and finite scales behind W's
// rows and behind a row's end
struct WTiled {
    const uint8_t *codes, *scales;
    int chunks;
    unsigned l;
    __device__ __forceinline__ WTiled(const uint8_t *tc, const uint8_t *ts, int n0, int n, int blocks, int lane) : chunks((blocks + CHUNK_BLOCKS - 1) / CHUNK_BLOCKS), l(lane)
    {
        const int tiles = (n + 15) / 16;
        first = min(n0 / 16, tiles - 1);
        most = tiles - 1 - first;
        codes = tc;
        scales = ts;
    }
    int first, most;                                         // tiles behind the last one repeat it
    __device__ __forceinline__ void load(Frag &f, int t, int c) const
    {
        const long long at = (long long)(first + min(t, most)) * chunks + c;
        const uint8_t *pc = codes + at * 2048, *ps = scales + at * 128;
        f.c[0] = *reinterpret_cast<const v4u *>(pc + l * 16u);
        f.c[1] = *reinterpret_cast<const v4u *>(pc + l * 16u + 1024);
        f.s = *reinterpret_cast<const uint16_t *>(ps + l * 2u);
    }
    __device__ __forceinline__ unsigned scale(const Frag &f, int) const { return f.s; }
};

// a workgroup of 64 lanes x 4: one 16-row tile of 4 chunks
__global__ __launch_bounds__(256) void mx4_tile_weights(const uint8_t *__restrict__ wc, const uint8_t *__restrict__ ws, uint8_t *__restrict__ tc, uint8_t *__restrict__ ts, int n, int kb,
                                                           int chunks)
{
    const int c = blockIdx.x * 4 + (threadIdx.x >> 6), l = threadIdx.x & 63, tile = blockIdx.y;
    if (c >= chunks) return;
    // read 8 lanes a row (128 consecutive bytes), write where the fragment order wants the 16 bytes
    const long long to = (long long)tile * chunks + c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = h * 8 + l / 8, p = l % 8, row = tile * 16 + r, b = c * CHUNK_BLOCKS + p;
        const bool in = row < n && b < kb;
        const v4u v = in ? *reinterpret_cast<const v4u *>(wc + ((long long)row * kb + b) * 16) : v4u{};
        *reinterpret_cast<v4u *>(tc + to * 2048 + p % 2 * 1024 + (p / 2 * 16 + r) * 16) = v;
        ts[to * 128 + (p / 2 * 16 + r) * 2 + p % 2] = in ? ws[(long long)row * kb + b] : 127;
    }
}

__device__ __forceinline__ v8i operand(v4u c)
{
    v8i v = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (int)c[j];
    return v;
}

template <int STEP>
__device__ __forceinline__ v4f mfma4(v4u w, unsigned ws, v4u x, unsigned xs, v4f acc)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(x), acc, 4, 4, STEP, (int)ws, STEP, (int)xs);
}

// x's rows of one wave: LPR lanes a row of a chunk, 64 / LPR rows a load.  Loads take no branches here either: GV values that would pass the array's end are
// read from its last GV and moved to their places, values behind a row's end are set to zero, rows behind the last one hold anything.
template <typename T, int LOADS, bool TINY>                  // TINY: the whole array may be shorter than one load
struct XRows {
    static constexpr int GV = Io<T>::GV, LPR = CHUNK / GV, PER = 64 / LPR;      // 64 lanes and 1 row, or 32 lanes and 2 rows
    typedef typename Io<T>::vec vec;
    const T *base;
    long long k;
    int off, step, last, at;                                                     // the lane's first value, PER rows, the array's last GV (tiny: its length), the place in the chunk
    bool ragged, tiny;
    __device__ __forceinline__ XRows(const T *x, long long row0, long long rows, long long kk, int l) : k(kk)
    {
        const long long total = rows * kk, first = row0 * kk;
        tiny = TINY && total < GV;
        const long long from = tiny ? 0 : first < total - GV ? first : total - GV;
        base = x + from;
        at = l % LPR * GV;
        off = (int)(first - from) + l / LPR * (int)kk + at;
        step = PER * (int)kk;
        const long long rest = total - GV - from;
        last = tiny ? (int)total : rest < (1 << 28) ? (int)rest : 1 << 28;                           // more than a tile's values (48 rows of 2^22)
        ragged = row0 + LOADS * PER + GV >= rows;
    }
    __device__ __forceinline__ vec load(int i, int k0) const
    {
        if (TINY && tiny) {
            vec v;
#pragma unroll
            for (int j = 0; j < GV; ++j) v[j] = off + i * step + k0 + j < last ? base[off + i * step + k0 + j] : (T)0.0f;
            return v;
        }
        return *reinterpret_cast<const vec *>(reinterpret_cast<const char *>(base) + (unsigned)min(fresh(off) + i * step + k0, last) * (unsigned)sizeof(T));
    }
    __device__ __forceinline__ void values(float (&v)[GV], const vec &t, int i, int k0) const
    {
#pragma unroll
        for (int j = 0; j < GV; ++j) v[j] = Io<T>::to_f(t[j]);
        if (ragged && !(TINY && tiny)) {
            const int d = fresh(off) + i * step + k0 - last;
#pragma unroll
            for (int bit = 1; bit < GV; bit *= 2) {
                const bool move = d > 0 && (d & bit);
#pragma unroll
                for (int j = 0; j < GV; ++j) v[j] = move ? (j + bit < GV ? v[j + bit] : 0.0f) : v[j];
            }
#pragma unroll
            for (int j = 0; j < GV; ++j) v[j] = d < GV ? v[j] : 0.0f;
        }
        if (k0 + CHUNK > k) {
            const int left = (int)k - k0 - fresh(at);
#pragma unroll
            for (int j = 0; j < GV; ++j) v[j] = j < left ? v[j] : 0.0f;
        }
    }
    // quantize4_group without the detour over float: the maximum of 16-bit patterns, two at a time, and the conversion from the type itself
    static __device__ __forceinline__ unsigned round16(const vec &t, int &b)
    {
        typedef uint16_t u2 __attribute__((ext_vector_type(2)));
        const v4u whole = __builtin_bit_cast(v4u, t);
        const unsigned p[4] = {whole[0], whole[1], whole[2], whole[3]};             // (a bit_cast of a vector's element would take the first one)
        u2 m = __builtin_bit_cast(u2, p[0] & 0x7fff7fffu);
#pragma unroll
        for (int j = 1; j < 4; ++j) m = __builtin_elementwise_max(m, __builtin_bit_cast(u2, p[j] & 0x7fff7fffu));
        const unsigned top = group_max<BLOCK / GV>(umax(m[0], m[1]));
        b = scale_byte<Q6>(sizeof(T) == 2 && std::is_same<T, __bf16>::value ? top << 16 : __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)top)));
        const float s = scale_of(b == 255 ? 127 : b);
        unsigned w = 0;
        if constexpr (std::is_same<T, __bf16>::value) {
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2bf, p[0]), s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2bf, p[1]), s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2bf, p[2]), s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2bf, p[3]), s, 3);
        } else if constexpr (std::is_same<T, _Float16>::value) {
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2h, p[0]), s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2h, p[1]), s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2h, p[2]), s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2h, p[3]), s, 3);
        }
        return w;                                                                // (a block of scale 255 multiplies as NaN whatever its codes)
    }
    // codes and scales of load i into LDS rows `row` on
    __device__ __forceinline__ void put(uint8_t *codes, uint8_t *scales, const vec &t, int i, int k0, int row, int l) const
    {
        int b;
        unsigned w;
        if (GV == 8 && !ragged && k0 + CHUNK <= k) {
            w = round16(t, b);
        } else {
            float v[GV];
            values(v, t, i, k0);
            w = quantize4_group<GV>(v, b);
        }
        const int r = row + l / LPR, c = l % LPR;
        if (GV == 8) *reinterpret_cast<unsigned *>(codes + r * ROW_BYTES + c * 4) = w;
        else *reinterpret_cast<uint16_t *>(codes + r * ROW_BYTES + c * 2) = (uint16_t)w;
        if (c % (BLOCK / GV) == 0) scales[r * CHUNK_BLOCKS + c / (BLOCK / GV)] = (uint8_t)b;
    }
};

__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <typename T>
__device__ __forceinline__ T finish(float v, float add, int relu)
{
    v = v + add;
    if (relu) v = v < 0.0f ? 0.0f : v;
    return Io<T>::from_f(v);
}

template <typename T, int TN, class W, bool TINY>
__global__ __launch_bounds__(THREADS, 2) void mx4_linear_narrow(const T *__restrict__ x, const uint8_t *__restrict__ wc, const uint8_t *__restrict__ ws, const float *__restrict__ bias,
                                                            T *__restrict__ y, long long rows, long long k, int n, int n_tiles, int relu)
{
    constexpr int LOADS = 16 / (64 / (CHUNK / Io<T>::GV)), LDS_X = 16 * (ROW_BYTES + CHUNK_BLOCKS), LDS_SUM = 16 * TN * 16 * 4;
    typedef XRows<T, LOADS, TINY> R;
    __shared__ __attribute__((aligned(16))) uint8_t smem[WAVES * (LDS_X > LDS_SUM ? LDS_X : LDS_SUM)];
    const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = l >> 4, r = l & 15;
    const long long row0 = (long long)(blockIdx.x / n_tiles) * 16;
    const int n0 = (int)(blockIdx.x % n_tiles) * 16 * TN, kb = (int)((k + BLOCK - 1) / BLOCK), chunks = (kb + CHUNK_BLOCKS - 1) / CHUNK_BLOCKS;
    uint8_t *codes = smem + wave * LDS_X, *scales = codes + 16 * ROW_BYTES;
    const R xr(x, row0, rows, k, l);
    const W wr(wc, ws, n0, n, kb, l);
    v4f acc[TN];
#pragma unroll
    for (int t = 0; t < TN; ++t) acc[t] = v4f{};
    typename R::vec X[LOADS];
    Frag F[TN];
    // loads of x that hold a row at all; the codes of the other rows are whatever LDS holds and end in outputs that are not stored
    const int mine = (int)min(rows - row0, 16LL), some = (mine + R::PER - 1) / R::PER;
    auto load = [&](int c) {
        if (some == LOADS) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) X[i] = xr.load(i, c * CHUNK);
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) if (i < some) X[i] = xr.load(i, c * CHUNK);
        }
#pragma unroll
        for (int t = 0; t < TN; ++t) wr.load(F[t], t, c);
    };
    if (wave < chunks) load(wave);
    for (int c = wave; c < chunks; c += WAVES) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) if (i < some) xr.put(codes, scales, X[i], i, c * CHUNK, i * R::PER, l);
        wave_fence();
        const v4u x0 = *reinterpret_cast<const v4u *>(codes + r * ROW_BYTES + q * 32), x1 = *reinterpret_cast<const v4u *>(codes + r * ROW_BYTES + q * 32 + 16);
        const unsigned xs = *reinterpret_cast<const uint16_t *>(scales + r * CHUNK_BLOCKS + q * 2);
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            const unsigned s = wr.scale(F[t], c);
            acc[t] = mfma4<0>(F[t].c[0], s, x0, xs, acc[t]);
            acc[t] = mfma4<1>(F[t].c[1], s, x1, xs, acc[t]);
        }
#pragma unroll
        for (int t = 0; t < TN; ++t) asm volatile("" : "+v"(acc[t]) : : "memory");        // the products stay ahead of the loads into their operands
        if (c + WAVES < chunks) load(c + WAVES);
        wave_fence();
    }
    __syncthreads();
    float *sum = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int t = 0; t < TN; ++t) *reinterpret_cast<v4f *>(sum + ((wave * 16 + r) * TN + t) * 16 + q * 4) = acc[t];
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * TN * 16; e += THREADS) {
        const int col = n0 + e % (TN * 16);
        const long long row = row0 + e / (TN * 16);
        if (row >= rows || col >= n) continue;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v = v + sum[w * 16 * TN * 16 + e];
        y[row * n + col] = finish<T>(v, bias != nullptr ? bias[col] : 0.0f, relu);
    }
}

template <typename T, int TM, int TN>
__global__ __launch_bounds__(THREADS, 2) void mx4_linear_wide(const T *__restrict__ x, const uint8_t *__restrict__ wc, const uint8_t *__restrict__ ws, const float *__restrict__ bias,
                                                          T *__restrict__ y, long long rows, long long k, int n, int n_tiles, int relu)
{
    constexpr int BM = 16 * TM, MINE = BM / WAVES, LOADS = MINE / (64 / (CHUNK / Io<T>::GV));    // MINE: rows of x a wave rounds
    typedef XRows<T, LOADS, false> R;
    static_assert(LOADS * R::PER == MINE, "whole loads");
    __shared__ __attribute__((aligned(16))) uint8_t s_codes[2][BM * ROW_BYTES], s_scales[2][BM * CHUNK_BLOCKS];
    const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = l >> 4, r = l & 15;
    const long long row0 = (long long)(blockIdx.x / n_tiles) * BM;
    const int n0 = ((int)(blockIdx.x % n_tiles) * WAVES + wave) * 16 * TN, kb = (int)((k + BLOCK - 1) / BLOCK), chunks = (kb + CHUNK_BLOCKS - 1) / CHUNK_BLOCKS;
    const R xr(x, row0 + wave * MINE < rows ? row0 + wave * MINE : rows - 1, rows, k, l);
    const WTiled wr(wc, ws, n0, n, kb, l);
    v4f acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int t = 0; t < TN; ++t) acc[m][t] = v4f{};
    typename R::vec X[LOADS];
    Frag F[TN];
    // past the last chunk the last one is loaded and rounded again, into a buffer that nobody reads: no branch around a load
    auto load_x = [&](int i, int c) { X[i] = xr.load(i, min(c, chunks - 1) * CHUNK); };
    auto put_x = [&](int i, int c) { xr.put(s_codes[c & 1], s_scales[c & 1], X[i], i, min(c, chunks - 1) * CHUNK, wave * MINE + i * R::PER, l); };
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load_x(i, 0);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) put_x(i, 0);
    // in the loop's own order, for which its waits are counted
#pragma unroll
    for (int t = 0; t < TN; ++t) {
        wr.load(F[t], t, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = t * LOADS / TN; i < (t + 1) * LOADS / TN; ++i) load_x(i, 1);
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    for (int c = 0; c < chunks; ++c) {
        const uint8_t *codes = s_codes[c & 1], *scales = s_scales[c & 1];
        v4u x0[TM], x1[TM];
        unsigned xs[TM];
#pragma unroll
        for (int m = 0; m < TM; ++m) {
            x0[m] = *reinterpret_cast<const v4u *>(codes + (m * 16 + r) * ROW_BYTES + q * 32);
            x1[m] = *reinterpret_cast<const v4u *>(codes + (m * 16 + r) * ROW_BYTES + q * 32 + 16);
            xs[m] = *reinterpret_cast<const uint16_t *>(scales + (m * 16 + r) * CHUNK_BLOCKS + q * 2);
        }
#pragma unroll
        for (int t = 0; t < TN; ++t) {
#pragma unroll
            for (int m = 0; m < TM; ++m) acc[m][t] = mfma4<0>(F[t].c[0], F[t].s, x0[m], xs[m], acc[m][t]);
#pragma unroll
            for (int m = 0; m < TM; ++m) acc[m][t] = mfma4<1>(F[t].c[1], F[t].s, x1[m], xs[m], acc[m][t]);
            // the products stay here and the next chunk's loads behind them, so that the loads can take the same registers
#pragma unroll
            for (int m = 0; m < TM; ++m) asm volatile("" : "+v"(acc[m][t]) : : "memory");
            wr.load(F[t], t, min(c + 1, chunks - 1));
            // a share of the next chunk's rounding between the products, which run beside it
#pragma unroll
            for (int i = t * LOADS / TN; i < (t + 1) * LOADS / TN; ++i) {
                put_x(i, c + 1);
                load_x(i, c + 2);
            }
        }
        __syncthreads();
    }
    float add[TN][4];
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) add[t][j] = bias != nullptr ? bias[min(n0 + t * 16 + q * 4 + j, n - 1)] : 0.0f;
#pragma unroll
    for (int m = 0; m < TM; ++m) {
        const long long row = row0 + m * 16 + r;
        if (row >= rows) continue;
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            typedef T out __attribute__((ext_vector_type(4), aligned(sizeof(T))));
            const int col = n0 + t * 16 + q * 4;
            out v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = finish<T>(acc[m][t][j], add[t][j], relu);
            T *to = y + row * n + col;
            if (col + 4 <= n) *reinterpret_cast<out *>(to) = v;
            else
#pragma unroll
                for (int j = 0; j < 3; ++j) if (col + j < n) to[j] = v[j];
        }
    }
}

struct Call { const void *x; const uint8_t *wc, *ws; const float *bias; void *y; long long rows, k; int n, relu; hipStream_t s; };

template <typename T, int TN, class W, bool TINY>
int narrow(const Call &a)
{
    const int tiles = (a.n + 16 * TN - 1) / (16 * TN);
    const long long groups = (a.rows + 15) / 16 * tiles;
    if (groups >= (1LL << 23)) return MDT_ERR_UNSUPPORTED;                         // 2^32 threads are the most of a launch
    mx4_linear_narrow<T, TN, W, TINY><<<dim3((unsigned)groups), THREADS, 0, a.s>>>((const T *)a.x, a.wc, a.ws, a.bias, (T *)a.y, a.rows, a.k, a.n, tiles, a.relu);
    return launch_check();
}

template <typename T, int TM, int TN>
int wide(const Call &a)
{
    const int tiles = (a.n + 128 * TN - 1) / (128 * TN);
    const long long groups = (a.rows + 16 * TM - 1) / (16 * TM) * tiles;
    if (groups >= (1LL << 23)) return MDT_ERR_UNSUPPORTED;
    mx4_linear_wide<T, TM, TN><<<dim3((unsigned)groups), THREADS, 0, a.s>>>((const T *)a.x, a.wc, a.ws, a.bias, (T *)a.y, a.rows, a.k, a.n, tiles, a.relu);
    return launch_check();
}

struct Tiled { int chunks, tiles; size_t codes, bytes; };
inline Tiled tiled_of(long long k, int n)
{
    Tiled t;
    t.chunks = (int)((k + CHUNK - 1) / CHUNK);
    t.tiles = (n + 15) / 16;
    t.codes = (size_t)t.chunks * t.tiles * 2048;
    t.bytes = t.codes + (size_t)t.chunks * t.tiles * 128;
    return t;
}
// The wide shape for many columns and many rows; for few rows only where the sum is long (1500 x 5000 -> 500, fp32: 27 us, narrow 39; 1000 x 2000 -> 300,
// fp16: 18 us, narrow 13).  Its W is copied into the lanes' order, the narrow one's where rows and sum make up for the launch (600 x 5292 -> 144: 23 us, else
// 29; 4000 x 144 -> 144: 18 us, else 13).
inline bool is_wide(long long rows, long long k, int n) { return n > 144 && (rows >= 2048 || (rows >= 512 && k >= 4096)); }
inline bool copies_w(long long rows, long long k, int n) { return is_wide(rows, k, n) || (rows >= 256 && k >= 4096); }

template <typename T, int TM>
int wide_by_columns(const Call &a, int ranges)
{
    switch ((a.n + 128 * ranges - 1) / (128 * ranges)) {
        case 1: case 2: return wide<T, TM, 2>(a);
        case 3: return wide<T, TM, 3>(a);
        case 4: return wide<T, TM, 4>(a);
        case 5: return wide<T, TM, 5>(a);
        default: return wide<T, TM, 6>(a);
    }
}

// as few ranges of columns as still give many CUs a workgroup: each range rounds x again (at least 48 / 96 / 192 workgroups: 400 x 3000 -> 200 14.5 / 11.4 / 14.7 us,
// 600 x 5292 -> 144 18 / 18 / 27, 50 x 9408 -> 768 23 / 19.5 / 20)
template <typename T, class W>
int narrow_by_columns(const Call &a)
{
    const long long row_tiles = (a.rows + 15) / 16;
    if (a.n > 48 && row_tiles * ((a.n + 143) / 144) >= 96) return narrow<T, 9, W, false>(a);
    if (a.n > 16 && row_tiles * ((a.n + 47) / 48) >= 96) return narrow<T, 3, W, false>(a);
    return narrow<T, 1, W, false>(a);
}

template <typename T>
int run(Call a, uint8_t *workspace)
{
    if (copies_w(a.rows, a.k, a.n)) {
        const Tiled t = tiled_of(a.k, a.n);
        mx4_tile_weights<<<dim3((t.chunks + 3) / 4, t.tiles), 256, 0, a.s>>>(a.wc, a.ws, workspace, workspace + t.codes, a.n, (int)((a.k + BLOCK - 1) / BLOCK), t.chunks);
        a.wc = workspace;
        a.ws = workspace + t.codes;
        if (!is_wide(a.rows, a.k, a.n)) return narrow_by_columns<T, WTiled>(a);
        const int ranges = (a.n + 767) / 768;
        // 16 rows a workgroup while that gives a CU few of them, else 48: a turn of the short ones takes about 6 / 10 of a long one's (2500 x 9408 -> 768: 56 us, 80)
        const long long short_turns = ((a.rows + 15) / 16 * ranges + 255) / 256, long_turns = ((a.rows + 47) / 48 * ranges + 255) / 256;
        return 6 * short_turns < 10 * long_turns ? wide_by_columns<T, 1>(a, ranges) : wide_by_columns<T, 3>(a, ranges);
    }
    if (a.rows * a.k < Io<T>::GV) return narrow<T, 1, WKept<true>, true>(a);
    return a.k <= BLOCK ? narrow_by_columns<T, WKept<true>>(a) : narrow_by_columns<T, WKept<false>>(a);
}

}  // namespace

extern "C" {

size_t mdt_mx4_linear_workspace_bytes(long long rows, long long k, int n)
{
    if (rows < 1 || k < 1 || n < 1 || k > (1 << 22) || n > (1 << 20)) return 0;
    return copies_w(rows, k, n) ? tiled_of(k, n).bytes : 0;
}

int mdt_mx4_linear(const void *x, int dtype, const void *w_codes, const void *w_scales, const float *bias, void *y, long long rows, long long k, int n, int relu, void *workspace,
                   size_t workspace_bytes, void *stream)
{
    if (rows < 0 || k < 1 || n < 1 || n > (1 << 20) || k > (1 << 22) || rows > (1LL << 30) || (rows > 0 && (!x || !w_codes || !w_scales || !y))) return MDT_ERR_INVALID_ARGUMENT;
    if (dtype != MDT_DTYPE_F32 && dtype != MDT_DTYPE_BF16 && dtype != MDT_DTYPE_F16) return MDT_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)w_codes & 15) != 0 || ((uintptr_t)workspace & 15) != 0) return MDT_ERR_INVALID_ARGUMENT;
    if (rows == 0) return MDT_OK;
    const size_t need = mdt_mx4_linear_workspace_bytes(rows, k, n);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return MDT_ERR_WORKSPACE_TOO_SMALL;
    const Call a = {x, (const uint8_t *)w_codes, (const uint8_t *)w_scales, bias, y, rows, k, n, relu, (hipStream_t)stream};
    switch (dtype) {
        case MDT_DTYPE_F32: return run<float>(a, (uint8_t *)workspace);
        case MDT_DTYPE_BF16: return run<__bf16>(a, (uint8_t *)workspace);
        default: return run<_Float16>(a, (uint8_t *)workspace);
    }
}

}  // extern "C"
