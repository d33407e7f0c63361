// Shared pieces of the teacher / student operators (linear_int8.hip, top_logits.hip, distill.hip).
#pragma once
#include "subreg_common.h"

namespace subreg {

template <> struct ElemTraits<_Float16> {
    static constexpr int DT = SUBREG_F16;
    static __device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 from_float(float v) { return (_Float16)v; }
};

constexpr int MAX_COLUMNS = 1 << 30;      // of a row: column arithmetic stays inside 32 bits
constexpr int MAX_ROWS = (1 << 22) - 1;   // of a call: a grid has fewer than 2^32 threads, and a row up to 1024 of them

inline bool float_dtype(int dt) { return dt == SUBREG_F32 || dt == SUBREG_BF16 || dt == SUBREG_F16; }
inline int dtype_bytes(int dt) { return dt == SUBREG_F32 ? 4 : dt == SUBREG_I8 ? 1 : 2; }

// calls F<T>() with the element type of a SUBREG_* float code
#define SUBREG_FOR_FLOAT(dt, ...)               \
    switch (dt) {                                \
        case SUBREG_F32: { using T = float; __VA_ARGS__; break; }      \
        case SUBREG_BF16: { using T = __bf16; __VA_ARGS__; break; }    \
        case SUBREG_F16: { using T = _Float16; __VA_ARGS__; break; }   \
        default: return SUBREG_EINVAL;           \
    }

// block reductions over blockDim.x threads (a multiple of 64, <= 1024); result in every thread; `red`: 16 entries of LDS
template <typename F, typename OP>
__device__ __forceinline__ F block_reduce(F v, F* red, F neutral, OP op) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o));
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, nw = blockDim.x >> 6;
    if (nw == 1) return v;
    __syncthreads();                                  // (a previous reduction's readers are done with `red`)
    if (lane == 0) red[wid] = v;
    __syncthreads();
    v = lane < nw ? red[lane] : neutral;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o));
    return __shfl(v, 0);
}

// 16 bytes of a row of n >= N elements, N to a load, without a branch (a load inside a divergent branch is waited for inside it, one
// after the other).  Load c covers the elements c N ... - or, where that passes the row's end, the row's last N: its first `skip`
// elements then belong to the load before it (skip >= N: all of them do).  Any alignment of the row: the hardware takes vector
// accesses at element addresses.
template <typename T> struct RowVec {
    static constexpr int N = 16 / sizeof(T);
    typedef __attribute__((ext_vector_type(N))) T V;
    typedef __attribute__((ext_vector_type(4))) unsigned U;
    U raw;
    static __device__ __forceinline__ int at(int c, int n) { return min(c * N, n - N); }
    static __device__ __forceinline__ int skip(int c, int n) { return max(c * N - (n - N), 0); }
    // (a 32-bit byte offset from the row's address, which all lanes share: one register a load in flight, not two)
    static __device__ __forceinline__ unsigned bytes(int at) { return (unsigned)at * (unsigned)sizeof(T); }
    __device__ __forceinline__ void load(const T* row, int at) { __builtin_memcpy(&raw, (const char*)row + bytes(at), 16); }
    __device__ __forceinline__ void store(T* row, int at) const { __builtin_memcpy((char*)row + bytes(at), &raw, 16); }
    __device__ __forceinline__ T elem(int e) const { return __builtin_bit_cast(V, raw)[e]; }
    __device__ __forceinline__ float get(int e) const { return ElemTraits<T>::to_float(elem(e)); }
    // past the caches (STREAM), for matrices that no cache holds until their next reader
    typedef U __attribute__((aligned(1))) UA;
    template <bool STREAM> __device__ __forceinline__ void load_as(const T* row, int at) {
        if constexpr (STREAM) raw = __builtin_nontemporal_load((const UA*)((const char*)row + bytes(at)));
        else load(row, at);
    }
    template <bool STREAM> __device__ __forceinline__ void store_as(T* row, int at) const {
        if constexpr (STREAM) __builtin_nontemporal_store(raw, (UA*)((char*)row + bytes(at)));
        else store(row, at);
    }
    // between two uses of a held row: what the first use unpacked is unpacked again (kept, it would take twice the registers)
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(raw)); }
};

}  // namespace subreg
