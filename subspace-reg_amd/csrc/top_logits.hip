// The largest logits of a row, sorted, equal ones by the lower index: what a teacher's answer is kept as.
#include "rows_common.h"

namespace subreg {

// Keys: unsigned integers in the order of the numbers (sign bit set for positives, all bits flipped for negatives); -0 is +0, a NaN is
// above +infinity.  16-bit types have 16-bit keys.  value(): the number of a key (a zero comes back as +0, any NaN as one NaN).
template <typename T> struct TopKey;
template <> struct TopKey<float> {
    static constexpr int BITS = 32;
    static __device__ __forceinline__ unsigned of(float v) {
        const unsigned u = __float_as_uint(v);
        if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
        if ((u & 0x7fffffffu) == 0) return 0x80000000u;
        return u & 0x80000000u ? ~u : u | 0x80000000u;
    }
    static __device__ __forceinline__ float value(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
};
template <typename T, unsigned INF> struct TopKey16 {
    static constexpr int BITS = 16;
    static __device__ __forceinline__ unsigned of(T v) {
        const unsigned u = __builtin_bit_cast(unsigned short, v);
        if ((u & 0x7fffu) > INF) return 0xffffu;
        if ((u & 0x7fffu) == 0) return 0x8000u;
        return u & 0x8000u ? u ^ 0xffffu : u | 0x8000u;
    }
    static __device__ __forceinline__ T value(unsigned k) {
        return __builtin_bit_cast(T, (unsigned short)(k & 0x8000u ? k & 0x7fffu : k ^ 0xffffu));
    }
};
template <> struct TopKey<__bf16> : TopKey16<__bf16, 0x7f80u> {};
template <> struct TopKey<_Float16> : TopKey16<_Float16, 0x7c00u> {};

// One block per row, the row read once:
//   1. every thread keeps the largest logit of what it read;
//   2. a wave finds a key t that at least `top` threads' maxima reach, so at least `top` logits do (bit by bit over the NT maxima; stops
//      as soon as between top and 2 top of them reach it);
//   3. the 16 bytes that held the maximum of a thread that reaches t are read again (little more than `top` of them; all of a thread's
//      loads where two of them reach t), and logits with a key >= t are listed in LDS; each takes the place that the count of larger (key, lower index) pairs gives it.
// More than CAP candidates (ties, masked rows): select_exact.
// Nothing of the row is held: at 64 registers a thread eight blocks of 256 share a CU, and the chain 2 - 3 of some (5 us) runs under the
// reads of others: 2048 rows of 32000 bf16 in 27 us, 4.9 TB/s, what a large copy reaches.  With the row in registers (512 threads, 8 loads each, four blocks a CU in step) they took 40.
constexpr int CAP = 1024;
constexpr int TOP_SHORT = 512;

typedef unsigned long long u64;
__device__ __forceinline__ u64 pair_of(unsigned key, int v) { return (u64)key << 32 | (0xffffffffu - (unsigned)v); }

// atomicAdd on LDS, one instruction: of atomicAdd with an addend of each lane's own hipcc makes a loop over the wave's lanes
__device__ __forceinline__ int lds_add(int* p, int n) {
    const unsigned at = (unsigned)(size_t)(__attribute__((address_space(3))) int*)p;
    int old;
    asm volatile("ds_add_rtn_u32 %0, %1, %2\n\ts_waitcnt lgkmcnt(0)" : "=&v"(old) : "v"(at), "v"(n) : "memory");
    return old;
}

// the row's answer
template <typename T> struct TopOut {
    T* values;
    long long* indices;
    __device__ __forceinline__ void put(int place, u64 me) const {
        values[place] = TopKey<T>::value((unsigned)(me >> 32));
        indices[place] = 0xffffffffu - (unsigned)me;
    }
};

// how many of list[0..n) are larger than `me`; the list is padded with zeros to a multiple of 8 (eight reads in flight, not one)
__device__ __forceinline__ int count_larger(const u64* list, int n, u64 me) {
    int place = 0;
#pragma unroll 1
    for (int j = 0; j < n; j += 8) {
        u64 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = list[j + i];
#pragma unroll
        for (int i = 0; i < 8; ++i) place += x[i] > me;
    }
    return place;
}
__device__ __forceinline__ void pad_list(u64* list, int n, int lane) {
    if (lane < 7 && (n + lane) % 8 != 0 && n / 8 == (n + lane) / 8) list[n + lane] = 0;
}

// place of each of n listed pairs (n <= CAP); the first `top` are written.  The list is complete when this is called (and padded here).
template <int NT, typename OUT>
__device__ __forceinline__ void write_places(u64* list, int n, int top, const OUT& out) {
    pad_list(list, n, threadIdx.x);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) {
        const u64 me = list[i];
        const int place = count_larger(list, n, me);
        if (place < top) out.put(place, me);
    }
}

// any row: the key of the top-th largest bit by bit (BITS counts over the row), everything above it, then of those equal to it the
// first ones in the order of their indices
template <typename T, int NT, typename OUT>
__device__ __forceinline__ void select_exact(const T* row, int vocab, int top, const OUT& out, u64* list, int* red, int* filled) {
    unsigned t = 0;
    for (int b = TopKey<T>::BITS - 1; b >= 0; --b) {
        const unsigned want = t | (1u << b);
        int n = 0;
        for (int v = threadIdx.x; v < vocab; v += NT) n += TopKey<T>::of(row[v]) >= want;
        n = block_reduce(n, red, 0, [](int a, int c) { return a + c; });
        if (n >= top) t = want;
    }
    __syncthreads();
    if (threadIdx.x == 0) *filled = 0;
    __syncthreads();
    for (int v = threadIdx.x; v < vocab; v += NT) {
        const unsigned key = TopKey<T>::of(row[v]);
        if (key > t) list[atomicAdd(filled, 1)] = pair_of(key, v);                     // fewer than top of them
    }
    __syncthreads();
    int have = *filled;
    for (int v0 = 0; v0 < vocab && have < top; v0 += NT) {
        const int v = v0 + threadIdx.x;
        const bool eq = v < vocab && TopKey<T>::of(row[v]) == t;
        const u64 in = __ballot(eq);
        const int before = __popcll(in & ((1ull << (threadIdx.x & 63)) - 1));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __popcll(in);
        __syncthreads();
        int off = have, all = 0;
        for (int w = 0; w < NT / 64; ++w) {
            if (w < (int)(threadIdx.x >> 6)) off += red[w];
            all += red[w];
        }
        if (eq && off + before < top) list[off + before] = pair_of(t, v);
        have += all;
    }
    __syncthreads();
    write_places<NT>(list, top, top, out);
}

// What a thread keeps of its loads: the largest logit and the load that held it, the largest of all its other loads, and whether there was
// a NaN (float maxima pass over those; the largest magnitude, as an integer, shows them).  Three instructions a logit, where the key of
// each would be ten, and five a load.
template <typename T> struct TopSeen {
    float best = -INFINITY, second = -INFINITY;
    unsigned mag = 0;
    int at;
    bool any = false;
    template <typename USE> __device__ __forceinline__ void see(const RowVec<T>& x, int c, USE use) {
        float m = -INFINITY;
#pragma unroll
        for (int e = 0; e < RowVec<T>::N; ++e) {
            const float f = x.get(e);
            m = fmaxf(m, use(e) ? f : -INFINITY);
            mag = max(mag, use(e) ? __float_as_uint(f) & 0x7fffffffu : 0u);
            any |= use(e);
        }
        const bool more = m > best;
        second = more ? best : fmaxf(second, m);
        at = more ? c : at;
        best = fmaxf(best, m);
    }
    __device__ __forceinline__ bool nan() const { return mag > 0x7f800000u; }
    __device__ __forceinline__ unsigned key() const {                // 0: nothing seen (below every key: -infinity's is 1 or more)
        if (!any) return 0;
        return nan() ? (TopKey<T>::BITS == 32 ? 0xffffffffu : 0xffffu) : TopKey<T>::of(ElemTraits<T>::from_float(best));
    }
    __device__ __forceinline__ bool others_reach(unsigned t) const { return nan() || TopKey<T>::of(ElemTraits<T>::from_float(second)) >= t; }
};

template <typename T, int NT>
__global__ __launch_bounds__(NT, NT == 1024 ? 4 : 8) void top_logits_kernel(const T* __restrict__ z, long long stride, int vocab,
                                                                            int top, T* __restrict__ values,
                                                                            long long* __restrict__ indices) {
    using V = RowVec<T>;
    constexpr int N = V::N, DEEP = 8;                 // loads a thread has in flight
    __shared__ int red[16];
    __shared__ __attribute__((aligned(16))) u64 list[CAP + 8];
    __shared__ unsigned maxima[NT];
    __shared__ int one[NT];
    __shared__ unsigned short many[NT];
    __shared__ int filled, n_one, n_many;
    __shared__ unsigned border;
    const long long r = blockIdx.x;
    const int tid = threadIdx.x;
    const T* row = z + r * stride;
    const TopOut<T> out{values + r * top, indices + r * top};
    const int loads = (vocab + N - 1) / N;

    TopSeen<T> seen;
    seen.at = tid;
    for (int c0 = 0; c0 < loads; c0 += DEEP * NT) {
        V x[DEEP];
#pragma unroll
        for (int i = 0; i < DEEP; ++i) x[i].load(row, V::at(c0 + i * NT + tid, vocab));
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < DEEP; ++i) {
            const int c = c0 + i * NT + tid;
            if ((c0 + (i + 1) * NT) * N <= vocab) {
                seen.see(x[i], c, [](int) { return true; });
            } else {
                const int skip = V::skip(c, vocab);
                seen.see(x[i], c, [skip](int e) { return e >= skip; });
            }
        }
    }
    const unsigned mx = seen.key();
    if (tid == 0) filled = n_one = n_many = 0;
    maxima[tid] = mx;
    __syncthreads();
    unsigned t = 0;
    if (2 * top > min(loads, NT)) {
        // few threads hold anything (one load each: NT >= 2 top, so loads < NT): their maxima say little, the border is sought among all logits
        V x;
        unsigned key[N];
        const int skip = V::skip(tid, vocab);
        x.load(row, V::at(tid, vocab));
#pragma unroll
        for (int e = 0; e < N; ++e) key[e] = e >= skip ? TopKey<T>::of(x.elem(e)) : 0;
        for (int b = TopKey<T>::BITS - 1; b >= 0; --b) {
            const unsigned want = t | (1u << b);
            int n = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) n += key[i] >= want;
            n = block_reduce(n, red, 0, [](int a, int c) { return a + c; });
            if (n >= top) {
                t = want;
                if (n <= 2 * top) break;
            }
        }
    } else {
        if (tid < 64) {
            unsigned m[NT / 64];
#pragma unroll
            for (int i = 0; i < NT / 64; ++i) m[i] = maxima[i * 64 + tid];
            for (int b = TopKey<T>::BITS - 1; b >= 0; --b) {
                const unsigned want = t | (1u << b);
                int n = 0;
#pragma unroll
                for (int i = 0; i < NT / 64; ++i) n += __popcll(__ballot(m[i] >= want));
                if (n >= top) {
                    t = want;
                    if (n <= 2 * top) break;
                }
            }
            if (tid == 0) border = t;
        }
        __syncthreads();
        t = border;
    }
    t = max(t, 1u);                                   // (0 stands for nothing)
    // loads to be read again, dealt to all threads: the one that held a thread's maximum, or all of a thread's where another reaches t too
    if (mx >= t) {
        if (seen.others_reach(t)) many[atomicAdd(&n_many, 1)] = (unsigned short)tid;
        else one[atomicAdd(&n_one, 1)] = seen.at;
    }
    __syncthreads();
    const int ones = n_one, each = (loads + NT - 1) / NT, all = ones + n_many * each;
    for (int p = tid; p < all; p += NT) {
        int c;
        if (p < ones) {
            c = one[p];
        } else {
            const int h = (p - ones) / each;
            c = many[h] + (p - ones - h * each) * NT;
        }
        const int at = V::at(c, vocab), skip = V::skip(c, vocab);
        V x;
        x.load(row, at);
        unsigned hits = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) hits |= (e >= skip && TopKey<T>::of(x.elem(e)) >= t ? 1u : 0u) << e;
        if (hits == 0) continue;
        int i = lds_add(&filled, __popc(hits));
        x.forget();
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (hits >> e & 1) {
                if (i < CAP) list[i] = pair_of(TopKey<T>::of(x.elem(e)), at + e);
                ++i;
            }
    }
    __syncthreads();
    const int n = filled;
    if (n > CAP) select_exact<T, NT>(row, vocab, top, out, list, red, &filled);
    else write_places<NT>(list, n, top, out);
}

// short rows: one wave per row, its keys in registers
template <typename T>
__global__ __launch_bounds__(256) void top_short_kernel(const T* __restrict__ z, long long stride, int rows, int vocab, int top,
                                                        T* __restrict__ values, long long* __restrict__ indices) {
    constexpr int NK = TOP_SHORT / 64;
    __shared__ __attribute__((aligned(16))) u64 lists[4][TOP_SHORT + 8];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long long r = (long long)blockIdx.x * 4 + w;
    if (r >= rows) return;
    const T* row = z + r * stride;
    unsigned key[NK];
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        const T x = row[min(i * 64 + lane, vocab - 1)];
        key[i] = i * 64 + lane < vocab ? TopKey<T>::of(x) : 0;       // (0: below every key)
    }
    unsigned t = 0;
    for (int b = TopKey<T>::BITS - 1; b >= 0; --b) {
        const unsigned want = t | (1u << b);
        int n = 0;
#pragma unroll
        for (int i = 0; i < NK; ++i) n += __popcll(__ballot(key[i] >= want));
        if (n >= top) {
            t = want;
            if (n <= top + top / 2) break;
        }
    }
    t = max(t, 1u);
    const TopOut<T> out{values + r * top, indices + r * top};
    u64* list = lists[w];
    int n = 0;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        const u64 in = __ballot(key[i] >= t);
        if (key[i] >= t) list[n + __popcll(in & ((1ull << lane) - 1))] = pair_of(key[i], i * 64 + lane);
        n += __popcll(in);
    }
    pad_list(list, n, lane);
    __builtin_amdgcn_wave_barrier();
    __threadfence_block();
    for (int i = lane; i < n; i += 64) {
        const u64 me = list[i];
        const int place = count_larger(list, n, me);
        if (place < top) out.put(place, me);
    }
}

template <typename T>
static int launch_top(const T* z, long long stride, int rows, int vocab, int top, T* values, long long* indices, hipStream_t s) {
    const long long loads = ((long long)vocab + RowVec<T>::N - 1) / RowVec<T>::N;
    if (vocab <= TOP_SHORT) {
        hipLaunchKernelGGL(top_short_kernel<T>, (int)(((long long)rows + 3) / 4), 256, 0, s, z, stride, rows, vocab, top, values, indices);
        return launch_status();
    }
#define SUBREG_TOP(NT) hipLaunchKernelGGL((top_logits_kernel<T, NT>), rows, NT, 0, s, z, stride, vocab, top, values, indices)
    // Threads: twice `top` at least (the border is found among their maxima), at most 32 loads each, and 16 where there is a block per
    // CU at most, so that a row's latency counts: 1 row of 50000 bf16 takes 11.0 | 8.8 | 9.8 us on 256 | 512 | 1024 threads, of 32000
    // 7.6 | 7.5 | 10.3, of 128000 15.8 | 10.8 | 11.2.  (A row cut into 16 parts for as many blocks and joined by a second launch: 11.2 -
    // 12.5 us for all of these.)
    const bool few = rows <= 256;
    if (loads > 512 * 32) SUBREG_TOP(1024);
    else if (loads > 256 * (few ? 16 : 32) || top > 128) SUBREG_TOP(512);
    else SUBREG_TOP(256);
#undef SUBREG_TOP
    return launch_status();
}

}  // namespace subreg

using namespace subreg;

extern "C" int subreg_top_logits(const void* logits, long long stride, int dtype, int rows, int vocab, int top, void* values,
                                 long long* indices, void* stream) {
    SUBREG_CHECK_ARG(logits && values && indices && rows > 0 && rows <= MAX_ROWS && vocab > 0 && vocab <= MAX_COLUMNS && stride >= 0);
    SUBREG_CHECK_ARG(top >= 1 && top <= vocab && top <= SUBREG_TOP_MAX);
    SUBREG_FOR_FLOAT(dtype, return launch_top<T>((const T*)logits, stride, rows, vocab, top, (T*)values, indices, (hipStream_t)stream))
    return SUBREG_EINVAL;
}
