// Products in 8-bit integers: y[r][n] = s[r] t[n] sum_k q[r][k] w[n][k] (+ bias[n]), with a scale for each row ("token") of x and for
// each output channel.  The frozen head of a teacher; beside subreg_linear_fwd (fp32, trained heads).
//   s[r] = max_k |x[r][k]| / 127, q = rint(x * (127 / max)): the codes use the whole range of their row, the step is half a unit of s.
//   The sum is exact: |q w| <= 2^14, dim <= 131071 keeps it inside 32 bits, so no rounding depends on the order of K.
#include "rows_common.h"

#include <type_traits>

namespace subreg {

typedef __attribute__((ext_vector_type(4))) int i32x4;

constexpr int I8_PITCH = 128;            // codes of x in the workspace: rows padded with zeros to whole 128-byte lines
constexpr float I8_FLOOR = 0x1p-100f;    // smallest row maximum: 127 / max stays finite

static inline long long round_up(long long a, long long b) { return (a + b - 1) / b * b; }

// scale and 1 / step of a row whose largest magnitude has the bits `top` (as integers a NaN's bits are above infinity's: both are seen)
__device__ __forceinline__ float row_inverse(unsigned top, float* scale) {
    const bool bad = top >= 0x7f800000u;
    const float amax = fmaxf(__uint_as_float(top), I8_FLOOR);
    *scale = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(amax, 127.f);
    return bad ? 0.f : __fdiv_rn(127.f, amax);
}
// |x inv| < 127.5 by the choice of inv; in a bad row inv = 0, and the conversion of 0 x infinity = NaN is 0 too
__device__ __forceinline__ int code_of(float x, float inv) { return __float2int_rn(x * inv); }

// NT threads (a wave or a block of 256) per row, the row in registers: one read of x, 16 bytes a load, codes of a load in one store
// (loads that overlap at the row's end write the same codes twice).  Bound by memory: 8192 x 4096 bf16 in 17 us, 5.9 TB/s (most of x
// comes from the last-level cache when it was just written).
template <typename T, int NT, int NV>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, long long x_stride, int rows, int dim,
                                                            signed char* __restrict__ codes, long long codes_stride,
                                                            float* __restrict__ scale) {
    constexpr int N = RowVec<T>::N;
    __shared__ unsigned red[16];
    const int lane = threadIdx.x % NT;
    const long long r = (long long)blockIdx.x * (256 / NT) + threadIdx.x / NT;
    if (r >= rows) return;                            // (whole waves; a block of one row never)
    const T* row = x + r * x_stride;
    RowVec<T> v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i].load(row, RowVec<T>::at(i * NT + lane, dim));
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) top = max(top, __float_as_uint(v[i].get(e)) & 0x7fffffffu);
    if constexpr (NT == 64) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    } else {
        top = block_reduce(top, red, 0u, [](unsigned a, unsigned b) { return max(a, b); });
    }
    float sc;
    const float inv = row_inverse(top, &sc);
    if (lane == 0) scale[r] = sc;
    signed char* out = codes + r * codes_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = i * NT + lane;
        signed char q[N];
#pragma unroll
        for (int e = 0; e < N; ++e) q[e] = (signed char)code_of(v[i].get(e), inv);
        if (c * N < dim) __builtin_memcpy(out + RowVec<T>::at(c, dim), q, N);
    }
    for (long long k = dim + lane; k < codes_stride; k += NT) out[k] = 0;
}

// rows shorter than a load, or too long for registers (two reads)
template <typename T>
__global__ __launch_bounds__(256) void quantize_any_rows_kernel(const T* __restrict__ x, long long x_stride, int dim,
                                                                 signed char* __restrict__ codes, long long codes_stride,
                                                                 float* __restrict__ scale) {
    __shared__ unsigned red[16];
    const long long r = blockIdx.x;
    const T* row = x + r * x_stride;
    unsigned top = 0;
    for (int k = threadIdx.x; k < dim; k += 256) top = max(top, __float_as_uint(ElemTraits<T>::to_float(row[k])) & 0x7fffffffu);
    top = block_reduce(top, red, 0u, [](unsigned a, unsigned b) { return max(a, b); });
    float sc;
    const float inv = row_inverse(top, &sc);
    if (threadIdx.x == 0) scale[r] = sc;
    signed char* out = codes + r * codes_stride;
    for (long long k = threadIdx.x; k < codes_stride; k += 256)
        out[k] = k < dim ? (signed char)code_of(ElemTraits<T>::to_float(row[k]), inv) : 0;
}

// codes copied to rows of the padded pitch (x given as codes, weights whose rows start anywhere): a thread per 16 bytes, which are read
// at any address; the bytes of a row's last ones behind `dim`, and those that would be read past the last row, become 0.  At most
// PAD_GRID blocks, which go round: a thread for every 16 bytes of the largest call (64 GB and more of codes) would be a grid of 2^32.
constexpr unsigned PAD_GRID = 1 << 18;

__global__ __launch_bounds__(256) void pad_codes_kernel(const signed char* __restrict__ x, long long x_stride, int rows, int dim,
                                                        signed char* __restrict__ codes, int pitch) {
    const unsigned per = (unsigned)pitch / 16;
    const unsigned long long all = (unsigned long long)rows * per;
    for (unsigned long long id = (unsigned long long)blockIdx.x * 256 + threadIdx.x; id < all; id += (unsigned long long)gridDim.x * 256) {
        const unsigned long long r = id / per;
        const int k = (int)(id - r * per) * 16, left = dim - k;          // left: bytes of the row from here
        const signed char* from = x + (long long)r * x_stride;
        i32x4 v = {0, 0, 0, 0};
        if (left >= 16) {
            __builtin_memcpy(&v, from + k, 16);
        } else if (left > 0) {
            unsigned long long lo = 0, hi = 0;
#pragma unroll
            for (int i = 0; i < 15; ++i)
                if (i < left) (i < 8 ? lo : hi) |= (unsigned long long)(unsigned char)from[k + i] << (8 * (i & 7));
            v = i32x4{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
        }
        *(i32x4*)(codes + (long long)r * pitch + k) = v;
    }
}

// 16 bytes of a weight row; bytes at or past `dim` come as zeros and are not read
__device__ __forceinline__ i32x4 load_codes_tail(const signed char* row, int k, int dim) {
    i32x4 v = {0, 0, 0, 0};
    signed char b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = k + i < dim ? row[k + i] : 0;
    __builtin_memcpy(&v, b, 16);
    return v;
}

// ---------------------------------------------------------------- one row: every wave a few channels
// Bound by the one read of the weights.  A wave holds the codes of x in registers (16 of every 1024 a lane, KV times) and reads whole weight
// rows, 1 KiB of consecutive bytes a load, R rows at a time; four-byte dot products, then the lanes' sums are added crosswise: log2 R
// exchanges halve the rows a lane stands for, after that each lane adds for one row only.  The next rows' loads are in flight meanwhile.
// A row's last 16 bytes are read where a load would pass its end (their codes that an earlier load has are 0): no read past a row.
// GEMV_GRID blocks are all that fit at once (four waves a SIMD); 1 x 4096 x 32768, weights from memory, with the quantiser's launch:
// 33.1 us on 1024 blocks, 36.0 on 2048; the MFMA kernel below 37, the tiles 41.
constexpr int GEMV_GRID = 1024, GEMV_MOST = 8192;                   // longest row: 32 registers of codes, 64 of weights

template <typename T, int KV, int R>
__global__ __launch_bounds__(256, 4) void linear_int8_gemv_kernel(const signed char* __restrict__ q, const float* __restrict__ s,
                                                                  const signed char* __restrict__ w, long long w_stride,
                                                                  const float* __restrict__ t, const float* __restrict__ bias,
                                                                  T* __restrict__ y, int dim, int out) {
    const int lane = threadIdx.x & 63, wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = gridDim.x * 4;
    unsigned at[KV];
#pragma unroll
    for (int v = 0; v < KV; ++v) at[v] = (unsigned)min((v * 64 + lane) * 16, dim - 16);
    i32x4 f[R][KV];
    auto load = [&](int n0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const signed char* row = w + (long long)min(n0 + r, out - 1) * w_stride;      // (wave-uniform)
#pragma unroll
            for (int v = 0; v < KV; ++v) __builtin_memcpy(&f[r][v], row + at[v], 16);
        }
    };
    int n0 = wave * R;
    if (n0 >= out) return;
    int code[KV][4];
    const float sx = s[0];
#pragma unroll
    for (int v = 0; v < KV; ++v) {
        i32x4 c;
        __builtin_memcpy(&c, q + at[v], 16);
        const int skip = (v * 64 + lane) * 16 - (int)at[v];          // codes that the load before has (16 or more: all)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = min(max(skip - 4 * i, 0), 4);
            code[v][i] = n == 4 ? 0 : (int)((unsigned)c[i] >> (8 * n) << (8 * n));
        }
    }
    load(n0);
    while (true) {
        int acc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            acc[r] = 0;
#pragma unroll
            for (int v = 0; v < KV; ++v)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[r] = __builtin_amdgcn_sdot4(code[v][i], f[r][v][i], acc[r], false);
        }
        const int done = n0;
        n0 += waves * R;
        load(n0 < out ? n0 : done);                                  // (no branch around loads)
        int mine = 0, o = 32;                                        // mine: the row (of R) this lane ends up with
#pragma unroll
        for (int half = R / 2; half > 0; half /= 2, o /= 2) {
            const bool up = lane & o;
#pragma unroll
            for (int r = 0; r < half; ++r) {
                const int keep = up ? acc[r + half] : acc[r], give = up ? acc[r] : acc[r + half];
                acc[r] = keep + __shfl_xor(give, o);
            }
            mine += up ? half : 0;
        }
#pragma unroll
        for (; o > 0; o /= 2) acc[0] += __shfl_xor(acc[0], o);
        const int n = done + mine;
        if ((lane & (64 / R - 1)) == 0 && n < out)
            y[n] = ElemTraits<T>::from_float((float)acc[0] * sx * t[n] + (bias ? bias[n] : 0.f));
        if (n0 >= out) break;
    }
}

// ---------------------------------------------------------------- few rows: the weights' stream
// y for rows <= 16 MT: bound by the one read of the weights, so they go from memory straight to the MFMAs' registers.  A block of W waves
// takes 16 NT channels; its waves take every W-th 128-byte chunk of K (two loads a lane; 64 consecutive bytes of 16 rows each) and add up
// through LDS.  The next chunk's loads - the next group's first ones at the end - are in flight under this one's MFMAs.  Any address and
// pitch of the weights.
// Blocks and K: 16 NT channels a block so that there are 256 blocks or more, four waves, eight where K is cut for 64 channels (4096 long, us
// with the quantiser, NT = 1 | 2 | 4: 64 x 4096 16.4 | 19.5 | 25.9; 64 x 8192 26.8 | 19.9 | 27.4; 48 x 16384 - | 28.9 | 27.0).  More than
// one chunk in flight behind the current one is slower (48 x 16384: 31): the registers cost waves.
// 48 x 4096 x 16384 moves its 67 MB in 20 us, 3.3 TB/s, and 16 rows in 16 us: the codes of x, read again by every block, or the one chunk in
// flight are the rest.  K % 128 != 0 costs more than its bytes: 48 x 2880 x 32768 52 us, K = 2944 41; 64 rows 63 and 47 - the last chunk is read byte
// by byte, and in the instances with MT = 3, 4 and NT = 4, W = 8 spills 43 and 110 registers.
constexpr int ROWS_MOST = 64, ROWS_GRID = 1024;

template <typename T, int MT, int NT, int W>
__global__ __launch_bounds__(64 * W, 2) void linear_int8_rows_kernel(
    const signed char* __restrict__ x, long long x_stride, const float* __restrict__ x_scale, const signed char* __restrict__ w,
    long long w_stride, const float* __restrict__ t, const float* __restrict__ bias, T* __restrict__ y, int rows, int dim, int out,
    int groups) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    i32x4* const part = (i32x4*)smem;                               // [W][NT * MT][64]
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int full = dim / 128;
    const int chunks = (full - wid + W - 1) / W;                    // whole chunks of this wave: wid, wid + W, ...

    struct Frag { i32x4 v[2]; };
    auto load_w = [&](Frag (&f)[NT], int n0, int c) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const signed char* p = w + (long long)min(n0 + j * 16 + l16, out - 1) * w_stride + c * 128 + g * 16;
            __builtin_memcpy(&f[j].v[0], p, 16);
            __builtin_memcpy(&f[j].v[1], p + 64, 16);
        }
    };
    auto load_x = [&](Frag (&f)[MT], int c) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int r = min(i * 16 + l16, rows - 1);
            const signed char* p = x + r * x_stride + c * 128 + g * 16;
            f[i].v[0] = *(const i32x4*)p;
            f[i].v[1] = *(const i32x4*)(p + 64);
        }
    };
    // Group g begins at chunk W g of K and goes round: with a pitch that is a multiple of the memory channels' interleave, blocks that all
    // walk K in the same order ask a few channels at a time.  (The sums are integers: any order is the same.)
    auto chunk_of = [&](int grp, int i) {                           // the i-th of this wave's chunks
        const int c = wid + i * W + (int)((unsigned)grp * W % (unsigned)max(full, 1));
        return c >= full ? c - full : c;
    };
    // (the codes of x are loaded with the weights: loads return in order, so codes asked for behind the next weights would wait for those)
    Frag cur[NT], curx[MT];
    if (chunks > 0) {
        load_x(curx, chunk_of(blockIdx.x, 0));
        load_w(cur, (int)blockIdx.x * 16 * NT, chunk_of(blockIdx.x, 0));
    }
    for (int grp = blockIdx.x; grp < groups; grp += gridDim.x) {
        const int n0 = grp * 16 * NT;
        i32x4 acc[NT][MT];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[j][i] = i32x4{0, 0, 0, 0};
        auto mma = [&](const Frag (&fw)[NT], const Frag (&fx)[MT]) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[j].v[s], fx[i].v[s], acc[j][i], 0, 0, 0);
        };
        const int g_next = grp + (int)gridDim.x < groups ? grp + (int)gridDim.x : grp;           // (at the very end the same again)
        for (int i = 0; i < chunks; ++i) {
            const bool more = i + 1 < chunks;
            const int g_of = more ? grp : g_next, c = chunk_of(g_of, more ? i + 1 : 0);
            mma(cur, curx);
            load_x(curx, c);
            load_w(cur, g_of * 16 * NT, c);
        }
        if (full * 128 < dim && full % W == wid) {                  // the row's last bytes: the codes of x are 0 behind them
            Frag fw[NT], fx[MT];
            load_x(fx, full);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int n = min(n0 + j * 16 + l16, out - 1);
                const signed char* row = w + (long long)n * w_stride;
#pragma unroll
                for (int h = 0; h < 2; ++h) fw[j].v[h] = load_codes_tail(row, full * 128 + h * 64 + g * 16, dim);
            }
            mma(fw, fx);
        }
        if (grp != (int)blockIdx.x) __syncthreads();                // (the last group's sums have been read)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) part[(wid * NT * MT + j * MT + i) * 64 + lane] = acc[j][i];
        __syncthreads();
        for (int e = tid; e < NT * MT * 64; e += 64 * W) {
            i32x4 sum = part[e];
#pragma unroll
            for (int v = 1; v < W; ++v) sum += part[v * NT * MT * 64 + e];
            const int tile = e >> 6, m = (tile % MT) * 16 + (e & 15), n = n0 + (tile / MT) * 16 + 4 * ((e >> 4) & 3);
            if (m >= rows) continue;
            const float sm = x_scale[m];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (n + c < out)
                    y[(long long)m * out + n + c] = ElemTraits<T>::from_float((float)sum[c] * sm * t[n + c] + (bias ? bias[n + c] : 0.f));
        }
    }
}

// ---------------------------------------------------------------- many rows: tiles through LDS
// Tile of y: TM = 32 FM rows x TN = 32 FN channels, four waves of (16 FM) x (16 FN), K in stages of 128 bytes, two LDS buffers.
// v_mfma_i32_16x16x64_i8: an operand lane holds row lane % 16, bytes 16 (lane / 16) .. + 15 of 64; the weights are the first operand, so
// a result lane holds row m = lane % 16 of x and the channels n = 4 (lane / 16) + i: four neighbours of y, one store.
// LDS row = 128 bytes = eight 16-byte slots; chunk c of row r sits in slot c ^ (r & 7), so the 16 rows of a fragment read meet every
// bank group twice (the minimum for 1 KiB).  The permutation is made by the source addresses of the LDS-DMA, inside a 128-byte line.
// Schedule of a stage (two k-steps): the reads of the second k-step run under the MFMAs of the first; the barrier stands in the MIDDLE
// of the second k-step's MFMAs, and behind it the DMA of the stage after next and the reads of the next stage's first k-step run under
// the other half.  A DMA has a whole stage of MFMAs to land.
// 8192 x 4096 x 8192 takes 229 - 238 us (2.3 P operations a second; a large library product of 8-bit integers: 2.2).  What bounds it: the same
// kernel without the DMA takes 186, without the fragment reads 214, without both and the barrier 169, of which 145 are the MFMAs - at 1.8
// GHz, where the clock is 2.0 with everything on and 2.4 at rest: the costs add up, as power does.  Four stages of 64 bytes with three
// in flight are slower (a whole call 267 against 245), and other places of the DMAs in the stage make no difference.
// D = C + A B with C and D the same accumulator registers.  As an asm statement because hipcc (ROCm 7.2) gives the builtin's result
// other registers than its addend and copies between them (376 copies beside the 128 MFMAs of a stage).  The operands come from LDS reads
// (the compiler waits for those before the statement); before the results are read, settle_acc() below lets the last one retire.
__device__ __forceinline__ void mfma_acc(i32x4& c, const i32x4& a, const i32x4& b) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

template <int FM, int FN> struct TileShape {
    static constexpr int TM = 32 * FM, TN = 32 * FN, BUF = (TM + TN) * 128, LDS = 2 * BUF, NP = (TM + TN) / 32;
};

template <int FM, int FN, typename T>
__global__ __launch_bounds__(256, FM * FN > 16 ? 1 : FM * FN > 8 ? 2 : 3) void linear_int8_tile_kernel(
    const signed char* __restrict__ q, int q_stride, const float* __restrict__ s, const signed char* __restrict__ w, int w_stride,
    const float* __restrict__ t, const float* __restrict__ bias, T* __restrict__ y, int rows, int dim, int out) {
    using S = TileShape<FM, FN>;
    constexpr int NP = S::NP, NPX = S::TM / 32;                     // 1-KiB DMA pieces (8 rows) of a wave: NPX of x, the rest of w
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    // tiles dealt to the XCDs in contiguous runs, and within a run in blocks of 8 tile rows: neighbours in time share L2 lines
    int tile_m, tile_n;
    {
        const int nm = (rows + S::TM - 1) / S::TM, nn = (out + S::TN - 1) / S::TN;
        const int n = gridDim.x, id = blockIdx.x, q8 = n / 8, r8 = n % 8, xcd = id % 8, slot = id / 8;
        const int v = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + slot;
        const int band = v / (8 * nn), in = v - band * 8 * nn, h = min(8, nm - band * 8);
        tile_m = band * 8 + in % h;
        tile_n = in / h;
    }
    const int m0 = tile_m * S::TM, n0 = tile_n * S::TN;

    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;
    const char* qb = (const char*)q + (long long)m0 * q_stride;
    const char* wb = (const char*)w + (long long)n0 * w_stride;
    const int chunk = ((lane & 7) ^ (lane >> 3)) << 4;
    unsigned off[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int r = (wid + 4 * (p < NPX ? p : p - NPX)) * 8 + (lane >> 3);
        off[p] = p < NPX ? (unsigned)min(r, rows - 1 - m0) * (unsigned)q_stride : (unsigned)min(r, out - 1 - n0) * (unsigned)w_stride;
    }
    const int wlast = (dim + 15) / 16 * 16 - 16;                    // last chunk of a weight row that may be read (the codes of x are 0 there)
    auto dma = [&](int p, int kx, int kw, int buf) {
        if (p < NPX) dma16(qb, off[p] + (unsigned)kx, lds0 + buf + (wid + 4 * p) * 1024);
        else dma16(wb, off[p] + (unsigned)kw, lds0 + buf + S::TM * 128 + (wid + 4 * (p - NPX)) * 1024);
    };
    auto kx_of = [&](int st) { return st * 128 + chunk; };
    auto kw_of = [&](int st) { return min(st * 128 + chunk, wlast); };

    const int stages = (dim + 127) / 128;
#pragma unroll
    for (int p = 0; p < NP; ++p) dma(p, kx_of(0), kw_of(0), 0);
    if (stages > 1) {
#pragma unroll
        for (int p = 0; p < NP; ++p) dma(p, kx_of(1), kw_of(1), S::BUF);
    }

    const int wm = wid & 1, wn = wid >> 1;
    const int xa = (wm * FM * 16 + l16) * 128 + ((g ^ (l16 & 7)) << 4);
    const int wa = (S::TM + wn * FN * 16 + l16) * 128 + ((g ^ (l16 & 7)) << 4);
    i32x4 acc[FN][FM], fx[2][FM], fw[2][FN];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[j][i] = i32x4{0, 0, 0, 0};
    // read r of a k-step: the first weight fragment, all of x, the other weight fragments
    auto rd = [&](int r, int set, int buf) {
        const int x6 = set ? 64 : 0;
        if (r == 0) fw[set][0] = *(const i32x4*)(smem + buf + (wa ^ x6));
        else if (r <= FM) fx[set][r - 1] = *(const i32x4*)(smem + buf + (xa ^ x6) + (r - 1) * 2048);
        else fw[set][r - FM] = *(const i32x4*)(smem + buf + (wa ^ x6) + (r - FM) * 2048);
    };
    auto mma = [&](int e, int set) {
        const int j = e / FM, i = e % FM;
        mfma_acc(acc[j][i], fw[set][j], fx[set][i]);
    };
    auto settle_acc = [&]() {                                       // (every access of acc before this stays before, every one behind it behind)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int i = 0; i < FM; ++i) asm volatile("" : "+a"(acc[j][i]));
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int i = 0; i < FM; ++i) asm volatile("" : "+a"(acc[j][i]));
    };
    constexpr int NM = FM * FN, NR = FM + FN, HALF = NM / 2;
    auto other = [](int buf) { return buf ? 0 : S::BUF; };
    auto stage = [&](int st, int buf, auto next_c, auto dma_c) {
        constexpr bool NEXT = decltype(next_c)::value, DMA = decltype(dma_c)::value;
        int rdone = 0;
#pragma unroll
        for (int e = 0; e < NM; ++e) {
            mma(e, 0);
            while ((e + 1) * NR / NM > rdone) {
                rd(rdone++, 1, buf);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int e = 0; e < HALF; ++e) mma(e, 1);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (NEXT) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        }
        const int kx = kx_of(st + 2), kw = kw_of(st + 2);
        int rn = 0, dn = 0;
#pragma unroll
        for (int e = HALF; e < NM; ++e) {
            mma(e, 1);
            if constexpr (NEXT) {
                while ((e + 1 - HALF) * NR / (NM - HALF) > rn) {
                    rd(rn++, 0, other(buf));
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (DMA) {
                while ((e + 1 - HALF) * NP / (NM - HALF) > dn) {
                    dma(dn++, kx, kw, buf);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    using Yes = std::integral_constant<bool, true>;
    using No = std::integral_constant<bool, false>;
    if (stages > 1) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(NP) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int r = 0; r < NR; ++r) rd(r, 0, 0);
    settle_acc();                                                    // the zeros are in the accumulators before the first MFMA adds to them
    int st = 0, buf = 0;
    for (; st + 2 < stages; ++st, buf = other(buf)) stage(st, buf, Yes{}, Yes{});
    if (st + 1 < stages) {
        stage(st, buf, Yes{}, No{});
        buf = other(buf);
    }
    stage(st, buf, No{}, No{});

    settle_acc();

    // four neighbours of y per lane and (i, j); the scales are in registers before the first store (a load behind a store would wait)
    typedef __attribute__((ext_vector_type(4))) T T4;
    const bool whole = m0 + S::TM <= rows && n0 + S::TN <= out && (out & 3) == 0;
    float sm[FM];
    f32x4 tn[FN], bn[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) sm[i] = s[min(m0 + (wm * FM + i) * 16 + l16, rows - 1)];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = n0 + (wn * FN + j) * 16 + 4 * g;
#pragma unroll
        for (int c = 0; c < 4; ++c) tn[j][c] = t[min(n + c, out - 1)];
#pragma unroll
        for (int c = 0; c < 4; ++c) bn[j][c] = bias ? bias[min(n + c, out - 1)] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int m = m0 + (wm * FM + i) * 16 + l16;
        T* row = y + (long long)m * out + n0 + 4 * g;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            T v[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = ElemTraits<T>::from_float((float)acc[j][i][c] * sm[i] * tn[j][c] + bn[j][c]);
            const int nl = (wn * FN + j) * 16;
            if (whole) {
                *(T4*)(row + nl) = T4{v[0], v[1], v[2], v[3]};
            } else if (m < rows) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (n0 + nl + 4 * g + c < out) row[nl + c] = v[c];
            }
        }
    }
}

template <typename T>
static void launch_quantize(const T* x, long long x_stride, int rows, int dim, signed char* codes, long long codes_stride, float* scale,
                            hipStream_t s) {
    constexpr int N = RowVec<T>::N;
    const int loads = (dim + N - 1) / N, four = (int)(((long long)rows + 3) / 4);
#define SUBREG_QUANT(NT, NV, GRID) \
    hipLaunchKernelGGL((quantize_rows_kernel<T, NT, NV>), GRID, 256, 0, s, x, x_stride, rows, dim, codes, codes_stride, scale)
    if (dim < N || loads > 256 * 16)
        hipLaunchKernelGGL(quantize_any_rows_kernel<T>, rows, 256, 0, s, x, x_stride, dim, codes, codes_stride, scale);
    else if (loads <= 64 * 2) SUBREG_QUANT(64, 2, four);
    else if (loads <= 64 * 4) SUBREG_QUANT(64, 4, four);
    else if (loads <= 64 * 8) SUBREG_QUANT(64, 8, four);
    else if (loads <= 256 * 4) SUBREG_QUANT(256, 4, rows);
    else if (loads <= 256 * 8) SUBREG_QUANT(256, 8, rows);
    else SUBREG_QUANT(256, 16, rows);
#undef SUBREG_QUANT
}

static int quantize(const void* x, long long x_stride, int dtype, int rows, int dim, signed char* codes, long long codes_stride,
                    float* scale, hipStream_t s) {
    SUBREG_FOR_FLOAT(dtype, launch_quantize<T>((const T*)x, x_stride, rows, dim, codes, codes_stride, scale, s))
    return launch_status();
}

}  // namespace subreg

using namespace subreg;

extern "C" int subreg_quantize_rows(const void* x, long long x_stride, int dtype, int rows, int dim, signed char* codes,
                                    long long codes_stride, float* scale, void* stream) {
    SUBREG_CHECK_ARG(x && codes && scale && rows > 0 && rows <= MAX_ROWS && dim > 0 && dim <= MAX_COLUMNS && x_stride >= 0 && codes_stride >= dim && float_dtype(dtype));
    return quantize(x, x_stride, dtype, rows, dim, codes, codes_stride, scale, (hipStream_t)stream);
}

static void pad_codes(const signed char* x, long long x_stride, int rows, int dim, signed char* codes, long long pitch, hipStream_t s) {
    const unsigned long long blocks = ((unsigned long long)rows * (pitch / 16) + 255) / 256;
    hipLaunchKernelGGL(pad_codes_kernel, blocks < PAD_GRID ? (unsigned)blocks : PAD_GRID, 256, 0, s, x, x_stride, rows, dim, codes, (int)pitch);
}

// the weight as the tile kernel reads it: rows at multiples of 16 bytes, 32-bit offsets inside a tile
static bool weight_direct(const signed char* w, long long w_stride) {
    return ((size_t)w & 15) == 0 && w_stride % 16 == 0 && w_stride <= (1 << 22);
}

extern "C" long long subreg_linear_int8_ws_bytes(int rows, int dim, int out, int x_dtype, const signed char* weight, long long w_stride) {
    if (rows <= 0 || rows > MAX_ROWS || dim <= 0 || dim > SUBREG_I8_MAX_DIM || out <= 0 || out > MAX_ROWS || w_stride < 0 || !(float_dtype(x_dtype) || x_dtype == SUBREG_I8))
        return SUBREG_EINVAL;
    const long long pitch = round_up(dim, I8_PITCH);
    return round_up(rows * pitch, 256) + round_up(4ll * rows, 256) + (rows <= ROWS_MOST || weight_direct(weight, w_stride) ? 0 : round_up(out * pitch, 256));
}

template <int FM, int FN, typename T>
static int launch_tiles(const signed char* q, int pitch, const float* s, const signed char* w, int w_stride, const float* t,
                        const float* bias, void* y, int rows, int dim, int out, hipStream_t st) {
    using S = TileShape<FM, FN>;
    static std::atomic<unsigned long long> ready{0};
    auto kern = linear_int8_tile_kernel<FM, FN, T>;
    const int rc = ensure_dynamic_lds((const void*)kern, S::LDS, ready);
    if (rc) return rc;
    const long long tiles = (long long)((rows + S::TM - 1) / S::TM) * ((out + S::TN - 1) / S::TN);
    if (tiles >= 1ll << 24) return SUBREG_EUNSUPPORTED;             // (a grid of 2^32 threads)
    hipLaunchKernelGGL(kern, (unsigned)tiles, 256, S::LDS, st, q, pitch, s, w, w_stride, t, bias, (T*)y, rows, dim, out);
    return launch_status();
}

template <typename T, int MT, int NT, int W>
static int launch_rows_kernel(const signed char* x, long long x_stride, const float* x_scale, const signed char* w, long long w_stride,
                              const float* t, const float* bias, T* y, int rows, int dim, int out, hipStream_t st) {
    static std::atomic<unsigned long long> ready{0};
    auto kern = linear_int8_rows_kernel<T, MT, NT, W>;
    constexpr int lds = W * NT * MT * 1024;
    const int rc = ensure_dynamic_lds((const void*)kern, lds, ready);
    if (rc) return rc;
    const int groups = (out + 16 * NT - 1) / (16 * NT);
    hipLaunchKernelGGL(kern, groups < ROWS_GRID ? groups : ROWS_GRID, 64 * W, lds, st, x, x_stride, x_scale, w, w_stride, t, bias, y, rows,
                       dim, out, groups);
    return launch_status();
}

template <typename T, int KV, int R>
static int launch_gemv(const signed char* q, const float* sx, const signed char* w, long long w_stride, const float* t, const float* bias,
                       T* y, int dim, int out, hipStream_t st) {
    const int blocks = (int)(((long long)out + 4 * R - 1) / (4 * R));
    hipLaunchKernelGGL((linear_int8_gemv_kernel<T, KV, R>), blocks < GEMV_GRID ? blocks : GEMV_GRID, 256, 0, st, q, sx, w, w_stride, t, bias,
                       y, dim, out);
    return launch_status();
}

extern "C" int subreg_linear_int8(const void* x, long long x_stride, int x_dtype, const float* x_scale, const signed char* weight,
                                  long long w_stride, const float* w_scale, const float* bias, void* y, int y_dtype, int rows,
                                  int dim, int out, void* ws, long long ws_bytes, void* stream) {
    SUBREG_CHECK_ARG(x && weight && w_scale && y && ws && rows > 0 && rows <= MAX_ROWS && dim > 0 && dim <= SUBREG_I8_MAX_DIM);
    SUBREG_CHECK_ARG(out > 0 && out <= MAX_ROWS);
    SUBREG_CHECK_ARG(x_stride >= 0 && w_stride >= 0 && float_dtype(y_dtype) && (float_dtype(x_dtype) || x_dtype == SUBREG_I8));
    SUBREG_CHECK_ARG((x_dtype == SUBREG_I8) == (x_scale != nullptr) && ((size_t)ws & 255) == 0);
    SUBREG_CHECK_ARG(ws_bytes >= subreg_linear_int8_ws_bytes(rows, dim, out, x_dtype, weight, w_stride));
    hipStream_t st = (hipStream_t)stream;
    const long long pitch = round_up(dim, I8_PITCH);
    signed char* q = (signed char*)ws;
    float* s = (float*)(q + round_up(rows * pitch, 256));
    if (x_dtype == SUBREG_I8) {
        pad_codes((const signed char*)x, x_stride, rows, dim, q, pitch, st);
    } else {
        const int rc = quantize(x, x_stride, x_dtype, rows, dim, q, pitch, s, st);
        if (rc) return rc;
    }
    const float* sx = x_dtype == SUBREG_I8 ? x_scale : s;
    if (rows == 1 && dim >= 16 && dim <= GEMV_MOST) {
        SUBREG_FOR_FLOAT(y_dtype, {
            if (dim <= 1024) return (launch_gemv<T, 1, 8>(q, sx, weight, w_stride, w_scale, bias, (T*)y, dim, out, st));
            if (dim <= 2048) return (launch_gemv<T, 2, 8>(q, sx, weight, w_stride, w_scale, bias, (T*)y, dim, out, st));
            if (dim <= 4096) return (launch_gemv<T, 4, 4>(q, sx, weight, w_stride, w_scale, bias, (T*)y, dim, out, st));
            return (launch_gemv<T, 8, 2>(q, sx, weight, w_stride, w_scale, bias, (T*)y, dim, out, st));
        })
    }
    // (short rows of many channels: the tiles' longer runs win - 64 x 1024 x 32768 16.4 us against 26.3)
    if (rows <= ROWS_MOST && !(dim < 2048 && out >= 16384 && weight_direct(weight, w_stride))) {
        const int mt = (rows + 15) / 16;
        SUBREG_FOR_FLOAT(y_dtype, {
            auto few = [&](auto nt, auto w) -> int {
                constexpr int NT = decltype(nt)::value, W = decltype(w)::value;
                if (mt == 1) return launch_rows_kernel<T, 1, NT, W>(q, pitch, sx, weight, w_stride, w_scale, bias, (T*)y, rows, dim, out, st);
                if (mt == 2) return launch_rows_kernel<T, 2, NT, W>(q, pitch, sx, weight, w_stride, w_scale, bias, (T*)y, rows, dim, out, st);
                if (mt == 3) return launch_rows_kernel<T, 3, NT, W>(q, pitch, sx, weight, w_stride, w_scale, bias, (T*)y, rows, dim, out, st);
                return launch_rows_kernel<T, 4, NT, W>(q, pitch, sx, weight, w_stride, w_scale, bias, (T*)y, rows, dim, out, st);
            };
            using std::integral_constant;
            if (out >= 256 * 64) return few(integral_constant<int, 4>{}, integral_constant<int, 8>{});
            if (out >= 256 * 32) return few(integral_constant<int, 2>{}, integral_constant<int, 4>{});
            return few(integral_constant<int, 1>{}, integral_constant<int, 4>{});
        })
    }
    if (!weight_direct(weight, w_stride)) {
        signed char* wp = (signed char*)s + round_up(4ll * rows, 256);
        pad_codes(weight, w_stride, out, dim, wp, pitch, st);
        weight = wp;
        w_stride = pitch;
    }
    // Tiles.  256 x 256 (a block a CU) does a tile's work in 1 / 1.2 of the time of four 128 x 128 ones, but in whole rounds of the 256 CUs:
    // us, 256 | 128: 8192 x 4096 x 4096 128 | 161; 3000 x 4096 x 5000 (240 tiles, one round) 70 | 73; 5000 x 2048 x 5000 (400, two) 81 | 75.
    // Where 128 x 128 makes 256 tiles or fewer, 64 x 128, and 64 x 64 where those do not fill the chip (128 | 64 x 128 | 64 x 64:
    // 2048 x 4096 x 2048 32.8 | 30.9 | 36.0; 1024 x 1024 x 4096 13.4 | 12.7 | 13.3; 333 x 1111 x 5003 22.0 | 19.5 | 19.0;
    // 128 x 4096 x 4096 26.0 | 23.1 | 20.3).
    auto tiles = [&](int tm, int tn) { return (long long)((rows + tm - 1) / tm) * ((out + tn - 1) / tn); };
    const long long n128 = tiles(128, 128);
    SUBREG_FOR_FLOAT(y_dtype, {
        if (20 * ((tiles(256, 256) + 255) / 256 * 256) <= 6 * n128)
            return launch_tiles<8, 8, T>(q, (int)pitch, sx, weight, (int)w_stride, w_scale, bias, y, rows, dim, out, st);
        if (n128 > 256) return launch_tiles<4, 4, T>(q, (int)pitch, sx, weight, (int)w_stride, w_scale, bias, y, rows, dim, out, st);
        if (tiles(64, 128) >= 256) return launch_tiles<2, 4, T>(q, (int)pitch, sx, weight, (int)w_stride, w_scale, bias, y, rows, dim, out, st);
        return launch_tiles<2, 2, T>(q, (int)pitch, sx, weight, (int)w_stride, w_scale, bias, y, rows, dim, out, st);
    })
    return SUBREG_EINVAL;
}
