// The largest logits of a row, sorted, equal ones by the lower index: what a teacher's answer is kept as.
#include "rows_common.h"

namespace subreg {

// Keys: unsigned integers in the order of the numbers (sign bit set for positives, all bits flipped for negatives); -0 is +0, a NaN is
// above +infinity.  16-bit types have 16-bit keys.
template <typename T> struct TopKey;
template <> struct TopKey<float> {
    static constexpr int BITS = 32;
    static __device__ __forceinline__ unsigned of(float v) {
        const unsigned u = __float_as_uint(v);
        if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
        if ((u & 0x7fffffffu) == 0) return 0x80000000u;
        return u & 0x80000000u ? ~u : u | 0x80000000u;
    }
};
template <typename T, unsigned INF> struct TopKey16 {
    static constexpr int BITS = 16;
    static __device__ __forceinline__ unsigned of(T v) {
        const unsigned u = __builtin_bit_cast(unsigned short, v);
        if ((u & 0x7fffu) > INF) return 0xffffu;
        if ((u & 0x7fffu) == 0) return 0x8000u;
        return u & 0x8000u ? u ^ 0xffffu : u | 0x8000u;
    }
};
template <> struct TopKey<__bf16> : TopKey16<__bf16, 0x7f80u> {};
template <> struct TopKey<_Float16> : TopKey16<_Float16, 0x7c00u> {};

// Exact selection: the key of the top-th largest is found bit by bit (BITS counts over the row); then everything above it, and of
// those equal to it the first ones, are listed and each takes the place that the count of larger (key, lower index) pairs gives it.
template <typename T>
__global__ __launch_bounds__(256) void top_logits_kernel(const T* __restrict__ z, long long stride, int vocab, int top,
                                                         T* __restrict__ values, long long* __restrict__ indices) {
    __shared__ int red[16];
    __shared__ unsigned long long list[SUBREG_TOP_MAX];
    __shared__ int filled;
    const long long r = blockIdx.x;
    const T* row = z + r * stride;
    unsigned t = 0;
    for (int b = TopKey<T>::BITS - 1; b >= 0; --b) {
        const unsigned want = t | (1u << b);
        int n = 0;
        for (int v = threadIdx.x; v < vocab; v += 256) n += TopKey<T>::of(row[v]) >= want;
        n = block_reduce(n, red, 0, [](int a, int c) { return a + c; });
        if (n >= top) t = want;
    }
    if (threadIdx.x == 0) filled = 0;
    __syncthreads();
    for (int v = threadIdx.x; v < vocab; v += 256) {
        const unsigned key = TopKey<T>::of(row[v]);
        if (key > t) list[atomicAdd(&filled, 1)] = (unsigned long long)key << 32 | (0xffffffffu - (unsigned)v);   // < top of them
    }
    __syncthreads();
    int have = filled;
    for (int v0 = 0; v0 < vocab && have < top; v0 += 256) {          // ties in the order of their indices
        const int v = v0 + threadIdx.x;
        const bool eq = v < vocab && TopKey<T>::of(row[v]) == t;
        const unsigned long long in = __ballot(eq);
        const int before = __popcll(in & ((1ull << (threadIdx.x & 63)) - 1));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __popcll(in);
        __syncthreads();
        int off = have, all = 0;
        for (int w = 0; w < 4; ++w) {
            if (w < (int)(threadIdx.x >> 6)) off += red[w];
            all += red[w];
        }
        if (eq && off + before < top) list[off + before] = (unsigned long long)t << 32 | (0xffffffffu - (unsigned)v);
        have += all;
    }
    __syncthreads();
    if ((int)threadIdx.x < top) {
        const unsigned long long me = list[threadIdx.x];
        int rank = 0;
        for (int j = 0; j < top; ++j) rank += list[j] > me;
        const unsigned v = 0xffffffffu - (unsigned)me;
        values[r * top + rank] = row[v];
        indices[r * top + rank] = v;
    }
}

}  // namespace subreg

using namespace subreg;

extern "C" int subreg_top_logits(const void* logits, long long stride, int dtype, int rows, int vocab, int top, void* values,
                                 long long* indices, void* stream) {
    SUBREG_CHECK_ARG(logits && values && indices && rows > 0 && vocab > 0 && stride >= 0);
    SUBREG_CHECK_ARG(top >= 1 && top <= vocab && top <= SUBREG_TOP_MAX);
    SUBREG_FOR_FLOAT(dtype, hipLaunchKernelGGL(top_logits_kernel<T>, rows, 256, 0, (hipStream_t)stream, (const T*)logits, stride,
                                               vocab, top, (T*)values, indices))
    return launch_status();
}
