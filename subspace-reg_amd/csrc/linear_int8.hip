// Products in 8-bit integers: y[r][n] = s[r] t[n] sum_k q[r][k] w[n][k] (+ bias[n]), with a scale for each row ("token") of x and for
// each output channel.  The frozen head of a teacher; beside subreg_linear_fwd (fp32, trained heads).
//   s[r] = max_k |x[r][k]| / 127, q = rint(x * (127 / max)): the codes use the whole range of their row, the step is half a unit of s.
//   The sum is exact: |q w| <= 2^14, dim <= 131071 keeps it inside 32 bits, so no rounding depends on the order of K.
#include "rows_common.h"

namespace subreg {

typedef __attribute__((ext_vector_type(4))) int i32x4;

constexpr int I8_PITCH = 128;            // codes of x in the workspace: rows padded with zeros to whole 128-byte lines
constexpr float I8_FLOOR = 0x1p-100f;    // smallest row maximum: 127 / max stays finite

static inline long long round_up(long long a, long long b) { return (a + b - 1) / b * b; }

// one block per row: maximum of the magnitudes as integers (a NaN's bits are above infinity's, so both are seen), then the codes
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, long long x_stride, int dim,
                                                            signed char* __restrict__ codes, long long codes_stride,
                                                            float* __restrict__ scale) {
    __shared__ unsigned red[16];
    const long long r = blockIdx.x;
    const T* row = x + r * x_stride;
    unsigned top = 0;
    for (int k = threadIdx.x; k < dim; k += 256) top = max(top, __float_as_uint(ElemTraits<T>::to_float(row[k])) & 0x7fffffffu);
    top = block_reduce(top, red, 0u, [](unsigned a, unsigned b) { return max(a, b); });
    const bool bad = top >= 0x7f800000u;
    const float amax = fmaxf(__uint_as_float(top), I8_FLOOR);
    const float inv = bad ? 0.f : __fdiv_rn(127.f, amax);
    if (threadIdx.x == 0) scale[r] = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(amax, 127.f);
    signed char* out = codes + r * codes_stride;
    for (long long k = threadIdx.x; k < codes_stride; k += 256) {
        const float v = k < dim && !bad ? rintf(ElemTraits<T>::to_float(row[k]) * inv) : 0.f;
        out[k] = (signed char)(int)fminf(fmaxf(v, -127.f), 127.f);
    }
}

// x given as codes: rows copied to the padded pitch
__global__ __launch_bounds__(256) void pad_codes_kernel(const signed char* __restrict__ x, long long x_stride, int dim,
                                                        signed char* __restrict__ codes, long long codes_stride) {
    const long long r = blockIdx.x;
    for (long long k = threadIdx.x; k < codes_stride; k += 256) codes[r * codes_stride + k] = k < dim ? x[r * x_stride + k] : 0;
}

// 16 bytes of a weight row at any address; bytes at or past `dim` come as zeros and are not read
__device__ __forceinline__ i32x4 load_codes_tail(const signed char* row, int k, int dim) {
    i32x4 v = {0, 0, 0, 0};
    if (k + 16 <= dim) {
        __builtin_memcpy(&v, row + k, 16);
    } else {
        signed char b[16];
        for (int i = 0; i < 16; ++i) b[i] = k + i < dim ? row[k + i] : 0;
        __builtin_memcpy(&v, b, 16);
    }
    return v;
}

// one wave per 16 x 16 tile of y; operands straight from global memory.  A fragment of v_mfma_i32_16x16x64_i8: lane holds row
// lane % 16, bytes k = 16 (lane / 16) ... + 15; result lane holds column lane % 16, rows 4 (lane / 16) + i.
template <typename T>
__global__ __launch_bounds__(256) void linear_int8_kernel(const signed char* __restrict__ q, long long q_stride,
                                                          const float* __restrict__ s, const signed char* __restrict__ w,
                                                          long long w_stride, const float* __restrict__ t,
                                                          const float* __restrict__ bias, T* __restrict__ y, int rows, int dim,
                                                          int out) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const long long n0 = ((long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16, m0 = (long long)blockIdx.y * 16;
    if (n0 >= out) return;
    const signed char* qa = q + min(m0 + l16, (long long)rows - 1) * q_stride;
    const signed char* wb = w + min(n0 + l16, (long long)out - 1) * w_stride;
    i32x4 acc = {0, 0, 0, 0};
    for (int k = g * 16; k - g * 16 < dim; k += 64) {
        const i32x4 a = *(const i32x4*)(qa + k);
        const i32x4 b = load_codes_tail(wb, k, dim);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc, 0, 0, 0);
    }
    const long long n = n0 + l16;
    if (n >= out) return;
    const float tn = t[n], bn = bias ? bias[n] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long m = m0 + 4 * g + i;
        if (m < rows) {
            float v = (float)acc[i] * s[m] * tn;
            if (bias) v += bn;
            y[m * out + n] = ElemTraits<T>::from_float(v);
        }
    }
}

static int quantize(const void* x, long long x_stride, int dtype, int rows, int dim, signed char* codes, long long codes_stride,
                    float* scale, hipStream_t s) {
    SUBREG_FOR_FLOAT(dtype, hipLaunchKernelGGL(quantize_rows_kernel<T>, rows, 256, 0, s, (const T*)x, x_stride, dim, codes,
                                               codes_stride, scale))
    return launch_status();
}

}  // namespace subreg

using namespace subreg;

extern "C" int subreg_quantize_rows(const void* x, long long x_stride, int dtype, int rows, int dim, signed char* codes,
                                    long long codes_stride, float* scale, void* stream) {
    SUBREG_CHECK_ARG(x && codes && scale && rows > 0 && dim > 0 && x_stride >= 0 && codes_stride >= dim && float_dtype(dtype));
    return quantize(x, x_stride, dtype, rows, dim, codes, codes_stride, scale, (hipStream_t)stream);
}

extern "C" long long subreg_linear_int8_ws_bytes(int rows, int dim, int out, int x_dtype) {
    if (rows <= 0 || dim <= 0 || dim > SUBREG_I8_MAX_DIM || out <= 0 || !(float_dtype(x_dtype) || x_dtype == SUBREG_I8))
        return SUBREG_EINVAL;
    return round_up(rows * round_up(dim, I8_PITCH), 256) + round_up(4ll * rows, 256);
}

extern "C" int subreg_linear_int8(const void* x, long long x_stride, int x_dtype, const float* x_scale, const signed char* weight,
                                  long long w_stride, const float* w_scale, const float* bias, void* y, int y_dtype, int rows,
                                  int dim, int out, void* ws, long long ws_bytes, void* stream) {
    SUBREG_CHECK_ARG(x && weight && w_scale && y && ws && rows > 0 && dim > 0 && dim <= SUBREG_I8_MAX_DIM && out > 0);
    SUBREG_CHECK_ARG(x_stride >= 0 && w_stride >= 0 && float_dtype(y_dtype) && (float_dtype(x_dtype) || x_dtype == SUBREG_I8));
    SUBREG_CHECK_ARG((x_dtype == SUBREG_I8) == (x_scale != nullptr) && ((size_t)ws & 255) == 0);
    SUBREG_CHECK_ARG(ws_bytes >= subreg_linear_int8_ws_bytes(rows, dim, out, x_dtype));
    hipStream_t st = (hipStream_t)stream;
    const long long pitch = round_up(dim, I8_PITCH);
    signed char* q = (signed char*)ws;
    float* s = (float*)(q + round_up(rows * pitch, 256));
    if (x_dtype == SUBREG_I8) {
        hipLaunchKernelGGL(pad_codes_kernel, rows, 256, 0, st, (const signed char*)x, x_stride, dim, q, pitch);
    } else {
        const int rc = quantize(x, x_stride, x_dtype, rows, dim, q, pitch, s, st);
        if (rc) return rc;
    }
    const float* sx = x_dtype == SUBREG_I8 ? x_scale : s;
    const dim3 grid((out + 63) / 64, (rows + 15) / 16);
    SUBREG_FOR_FLOAT(y_dtype, hipLaunchKernelGGL(linear_int8_kernel<T>, grid, 256, 0, st, q, pitch, sx, weight, w_stride, w_scale,
                                                 bias, (T*)y, rows, dim, out))
    return launch_status();
}
