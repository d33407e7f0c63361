// Distillation from a teacher's top logits with the labels' cross entropy, loss and gradient in one pass over the student's logits.
//   p = softmax over a row's kept entries of t / T;  e_v = exp((z_v - m) / T), S = sum_v e_v;  likewise at T = 1 for the labels
//   KL = sum_j p_j (log p_j - (z_{i_j} - m) / T + log S);        CE = log S_1 - (z_y - m)
//   T KL = sum_j p_j ((t_j - t_m) - (z_{i_j} - m)) + T (log S - log P): what a row's term is kept as (T^2 alone overflows before the loss
//   does, and a difference over T where a kept entry's logit is masked by the type's lowest number)
//   d(a T^2 KL)/dz_v = a T (e_v / S - sum_{j: i_j = v} p_j);     d(b CE)/dz_v = b (e1_v / S_1 - [v = y])
// Every row needs its maximum and two sums before its first gradient is known, so a row is read, reduced and written by one block, and
// held in its registers in between: each logit is read once and each gradient written once.  Bound by memory: 4096 x 32000 bf16 with
// labels at T = 2, a tenth of the rows masked, in 103 us, 4.9 TB/s, what a large copy reaches; 1024 x 131072 in 139 us, 3.6 TB/s, for
// there one row fills a CU and its exponentials run alone.
// All exponents are x_v = z_v c - m c (c = log2(e) / T, one fused operation, m c rounded once and common to the row): its error is one
// rounding of x_v, and the common one cancels in every quotient - while |m c| <= FAR: the rounding of m c is then at most 2^-5 in an
// exponent (at 1e10, a mask's value, it would be 512, and e no number).  Rows whose maximum is further out take distill_any_row, which
// subtracts first.  Where T is a power of two, e1 = e^T by squarings (one instruction
// each, where a second exponential is five).
#include "rows_common.h"

#include <type_traits>

namespace subreg {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float FAR = 0x1p20f;
constexpr int COUNT_INLINE = 2048;       // up to so many entries every block counts for itself
constexpr int COUNT_BLOCKS = 256;        // at most, of the counting kernel

struct DistillArgs {
    const void* z;
    const void* tv;
    const long long* ti;
    const long long* target;
    long long z_stride, tv_stride, ti_stride, ignore;
    int rows, vocab, top, reduction, flags, count_blocks, count_rows, squarings;
    float c_t, inv_t, kd, ce, temp;      // c_t = log2(e) / T
    const float* gs;
    long long gs_stride;
    float* loss;
    void* dz;
    float* row_kd;                       // [rows] T KL of the row (SUM / MEAN)
    float* row_ce;
    int* counts;                         // [count_blocks][2] rows with entries | with a label (MEAN)
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// a product that is rounded: the difference of two such is 0 where they are equal (fused with the subtraction it would be the rounding
// error of one of them, which for masked rows' maxima is large)
__device__ __forceinline__ float rounded_product(float x, float y) {
#pragma clang fp contract(off)
    return x * y;
}

// (the teacher's type is a template argument of every kernel: looked up at run time, 64 x 60 takes 11.6 us for 10.8, its backward 7.3 for 6.6,
// and 512 x 151936 81 for 79; 4096 x 32000 is level)
template <typename TV>
__device__ __forceinline__ bool entry_kept(const DistillArgs& a, long long r, int j, float& v, long long& idx) {
    idx = a.ti[r * a.ti_stride + j];
    v = ElemTraits<TV>::to_float(((const TV*)a.tv)[r * a.tv_stride + j]);
    return idx >= 0 && !(v == -INFINITY);
}

// a thread's share (thread `tid` of `nt`) of the numbers of rows with entries and with a label: from the counting kernel's sums, or, where
// the call is so small that every row's entries cost less than another launch, from the entries themselves
template <typename TV, bool INLINE>
__device__ __forceinline__ void row_counts(const DistillArgs& a, int tid, int nt, int& n_kd, int& n_ce) {
    if (!INLINE || a.count_blocks) {
        for (int b = tid; b < a.count_blocks; b += nt) {
            n_kd += a.counts[2 * b];
            n_ce += a.counts[2 * b + 1];
        }
        return;
    }
    for (int r = tid; r < a.rows; r += nt) {
        bool any = false;
#pragma unroll 4
        for (int j = 0; j < a.top; ++j) {
            float v;
            long long idx;
            any |= entry_kept<TV>(a, r, j, v, idx);
        }
        n_kd += any;
        n_ce += a.target && a.target[r] != a.ignore;
    }
}

template <typename TV>
__global__ __launch_bounds__(256) void distill_count_kernel(DistillArgs a) {
    __shared__ int red[16];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    int kd = 0, ce = 0;
    for (int i = wid; i < a.count_rows; i += 4) {
        const long long r = (long long)blockIdx.x * a.count_rows + i;
        if (r >= a.rows) break;
        bool any = false;
        for (int j = lane; j < a.top; j += 64) {
            float v;
            long long idx;
            any |= entry_kept<TV>(a, r, j, v, idx);
        }
        kd += __any(any) ? 1 : 0;
        ce += a.target && a.target[r] != a.ignore ? 1 : 0;
    }
    auto add = [](int p, int q) { return p + q; };
    kd = block_reduce(lane == 0 ? kd : 0, red, 0, add);
    ce = block_reduce(lane == 0 ? ce : 0, red, 0, add);
    if (threadIdx.x == 0) {
        a.counts[2 * blockIdx.x] = kd;
        a.counts[2 * blockIdx.x + 1] = ce;
    }
}

// loss[0] from the rows' terms, in a fixed order; the rows that have a term are counted by its value (a row without one holds NO_TERM,
// which no KL and no cross entropy can be)
constexpr float NO_TERM = -INFINITY;
__global__ __launch_bounds__(1024) void distill_finish_kernel(DistillArgs a) {
    __shared__ double red[4][16];
    double v[4] = {0, 0, 0, 0};
#pragma unroll 4
    for (int r = threadIdx.x; r < a.rows; r += 1024) {
        const float kd = a.row_kd[r], ce = a.row_ce[r];
        if (kd != NO_TERM) { v[0] += (double)kd; v[2] += 1.0; }
        if (ce != NO_TERM) { v[1] += (double)ce; v[3] += 1.0; }
    }
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v[k] += __shfl_xor(v[k], o);
        if (lane == 0) red[k][wid] = v[k];
    }
    __syncthreads();
    if (threadIdx.x < 64) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = red[k][lane & 15];
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) v[k] += __shfl_xor(v[k], o);
        }
        if (lane == 0) {
            const bool mean = a.reduction == SUBREG_MEAN;
            const double kd = mean ? v[0] / fmax(v[2], 1.0) : v[0], ce = mean ? v[1] / fmax(v[3], 1.0) : v[1];
            a.loss[0] = (float)((double)a.kd * a.temp * kd + (double)a.ce * ce);
        }
    }
}

// any row: shorter than a load, or with a maximum too far from 0 for the products above (rows of nothing but masks, infinities, NaN).
// NT threads of one row; reads it three times, from the caches after the first.
template <typename T, typename TV, int NT, bool INLINE>
__device__ __forceinline__ void distill_any_row(const DistillArgs& a, long long r) {
    __shared__ float red[16];
    __shared__ int redi[16];
    __shared__ float s_p[SUBREG_TOP_MAX + 1];
    __shared__ int s_i[SUBREG_TOP_MAX + 1];          // vocabulary entry, -1: none; the label is entry `top`
    const int tid = threadIdx.x;
    const float g = a.gs ? a.gs[r * a.gs_stride] : 1.f;
    __syncthreads();
    const T* z = (const T*)a.z + r * a.z_stride;
    T* dz = a.dz ? (T*)a.dz + r * a.vocab : nullptr;
    auto add = [](float p, float q) { return p + q; };
    auto addi = [](int p, int q) { return p + q; };
    auto mx = [](float p, float q) { return fmaxf(p, q); };

    // the teacher's share
    int state = 0;
    float tm = -INFINITY;
    for (int j = tid; j < a.top; j += NT) {
        float v;
        long long idx;
        if (!entry_kept<TV>(a, r, j, v, idx)) continue;
        state += 1 + (idx >= a.vocab ? 1 << 16 : 0);
        tm = fmaxf(tm, v);
    }
    state = block_reduce(state, redi, 0, addi);
    const bool kd_on = (state & 0xffff) != 0, bad = state >> 16 != 0;
    long long y = -1;
    bool ce_on = false, bad_y = false;
    if (a.target) {
        y = a.target[r];
        ce_on = y != a.ignore;
        bad_y = ce_on && (y < 0 || y >= a.vocab);
        if (!ce_on || bad_y) y = -1;
    }
    float cnt_kd = 1.f, cnt_ce = 1.f;
    if (a.reduction == SUBREG_MEAN && dz) {
        int n_kd = 0, n_ce = 0;
        row_counts<TV, INLINE>(a, tid, NT, n_kd, n_ce);
        cnt_kd = (float)max(1, block_reduce(n_kd, redi, 0, addi));
        cnt_ce = (float)max(1, block_reduce(n_ce, redi, 0, addi));
    }
    float* out = a.reduction == SUBREG_NONE ? a.loss : nullptr;
    if (!kd_on && !ce_on) {
        if (dz)
            for (int v = tid; v < a.vocab; v += NT) dz[v] = ElemTraits<T>::from_float(0.f);
        if (tid == 0 && a.loss) {
            if (out) out[r] = 0.f;
            else { a.row_kd[r] = NO_TERM; a.row_ce[r] = NO_TERM; }
        }
        return;
    }
    tm = block_reduce(tm, red, -INFINITY, mx);
    float ps = 0.f;
    for (int j = tid; j < a.top; j += NT) {
        float v;
        long long idx;
        const bool kept = entry_kept<TV>(a, r, j, v, idx);
        s_p[j] = kept ? expf((v - tm) * a.inv_t) : 0.f;
        s_i[j] = kept && idx < a.vocab ? (int)idx : -1;
        ps += s_p[j];
    }
    ps = block_reduce(ps, red, 0.f, add);
    for (int j = tid; j < a.top; j += NT) s_p[j] = kd_on ? s_p[j] / ps : 0.f;
    if (tid == 0) {
        s_p[a.top] = 0.f;
        s_i[a.top] = (int)y;
    }

    // the student's softmax
    float m = -INFINITY;
    for (int v = tid; v < a.vocab; v += NT) m = fmaxf(m, ElemTraits<T>::to_float(z[v]));
    m = block_reduce(m, red, -INFINITY, mx);
    float se = 0.f, s1 = 0.f;
    for (int v = tid; v < a.vocab; v += NT) {
        const float d = ElemTraits<T>::to_float(z[v]) - m;
        se += exp2_fast(d * a.c_t);
        if (ce_on && !(a.squarings == 0)) s1 += exp2_fast(d * LOG2E);
    }
    se = block_reduce(se, red, 0.f, add);
    s1 = (a.squarings == 0) ? se : block_reduce(s1, red, 0.f, add);

    if (a.loss) {
        float term = 0.f;
        for (int j = tid; j < a.top; j += NT) {
            const float p = s_p[j];
            if (s_i[j] < 0 || p == 0.f) continue;
            const float tv = ElemTraits<TV>::to_float(((const TV*)a.tv)[r * a.tv_stride + j]);
            term += p * (((tv - tm) - (ElemTraits<T>::to_float(z[s_i[j]]) - m)) + a.temp * (logf(se) - logf(ps)));
        }
        term = block_reduce(term, red, 0.f, add);
        if (tid == 0) {
            if (bad) term = NAN;
            const float ce = !ce_on ? 0.f : bad_y ? NAN : logf(s1) - (ElemTraits<T>::to_float(z[y]) - m);
            if (out) out[r] = a.kd * a.temp * term + a.ce * ce;
            else { a.row_kd[r] = kd_on ? term : NO_TERM; a.row_ce[r] = ce_on ? ce : NO_TERM; }
        }
    }
    if (!dz) return;
    const float ckd = bad ? NAN : kd_on ? g * a.kd * a.temp / cnt_kd : 0.f;
    const float cce = bad_y ? NAN : ce_on ? g * a.ce / cnt_ce : 0.f;
    const float akd = ckd / se, ace = cce / s1;
    auto grad = [&](float zv, float pv, float hot) {
        const float d = zv - m;
        const float et = exp2_fast(d * a.c_t), e1 = (a.squarings == 0) ? et : exp2_fast(d * LOG2E);
        float o = 0.f;
        if (kd_on) o = akd * et - ckd * pv;
        if (ce_on) o += ace * e1 - cce * hot;
        return o;
    };
    for (int v = tid; v < a.vocab; v += NT) dz[v] = ElemTraits<T>::from_float(grad(ElemTraits<T>::to_float(z[v]), 0.f, 0.f));
    __syncthreads();                                     // the row's stores are done: its entries and the label are written again
    for (int j = tid; j <= a.top; j += NT) {
        const int v = s_i[j];
        if (v < 0) continue;
        float pv = 0.f;
        bool first = true;
        for (int i = 0; i <= a.top; ++i)
            if (s_i[i] == v) {
                if (i < j) first = false;
                pv += s_p[i];
            }
        if (first) dz[v] = ElemTraits<T>::from_float(grad(ElemTraits<T>::to_float(z[v]), pv, v == (int)y ? 1.f : 0.f));
    }
}

template <typename T, typename TV>
__global__ __launch_bounds__(256) void distill_any_kernel(DistillArgs a) {
    const long long r = blockIdx.x;
    if ((a.flags & SUBREG_DISTILL_SKIP_UNIT) && a.gs[r * a.gs_stride] == 1.f) return;
    distill_any_row<T, TV, 256, true>(a, r);
}

// NT threads per row, NV loads of 16 bytes a thread in registers; NV = 0: the row streamed with a running maximum and sum a thread (few
// registers, any length): the loss alone, and rows that do not fit the registers, which are then read a second time.  SQ: squarings from e to e1 (-1: a second exponential; 0: T = 1, or no
// labels).  The first wave does the teacher's side while the others' loads are in flight.
template <typename T, typename TV, int NT, int NV, int SQ, bool STREAM = false>
__global__ __launch_bounds__(NT) void distill_row_kernel(DistillArgs a) {
    using V = RowVec<T>;
    constexpr int N = V::N, EPL = SUBREG_TOP_MAX / 64;              // entries a lane
    __shared__ float red[16], red1[16];
    __shared__ float s_p[SUBREG_TOP_MAX + 1];
    __shared__ int s_i[SUBREG_TOP_MAX + 1];          // vocabulary entry, -1: none; the label is entry `top`
    __shared__ float s_cnt[2];
    const long long r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float g = a.gs ? a.gs[r * a.gs_stride] : 1.f;
    if ((a.flags & SUBREG_DISTILL_SKIP_UNIT) && g == 1.f) return;
    const T* z = (const T*)a.z + r * a.z_stride;
    T* dz = a.dz ? (T*)a.dz + r * a.vocab : nullptr;
    const int vocab = a.vocab, top = a.top;

    // which terms the row has (every wave for itself)
    float tv[EPL];
    int ti[EPL];
    bool kept = false, bad = false;
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
        const int j = q * 64 + lane;
        ti[q] = -1;
        tv[q] = -INFINITY;
        if (q * 64 < top) {
            float v;
            long long idx;
            const bool k = entry_kept<TV>(a, r, min(j, top - 1), v, idx) && j < top;
            kept |= k;
            bad |= k && idx >= vocab;
            if (k) { tv[q] = v; ti[q] = idx < vocab ? (int)idx : -1; }
        }
    }
    const bool kd_on = __any(kept);
    bad = __any(bad);
    long long y = -1;
    bool ce_on = false, bad_y = false;
    if (a.target) {
        y = a.target[r];
        ce_on = y != a.ignore;
        bad_y = ce_on && (y < 0 || y >= vocab);
        if (!ce_on || bad_y) y = -1;
    }
    float* out = a.reduction == SUBREG_NONE ? a.loss : nullptr;
    if (!kd_on && !ce_on) {
        if (dz) {
            V zero;
            zero.raw = typename V::U{0, 0, 0, 0};
            for (int c = tid; c * N < vocab; c += NT) zero.store(dz, V::at(c, vocab));
        }
        if (tid == 0 && a.loss) {
            if (out) out[r] = 0.f;
            else { a.row_kd[r] = NO_TERM; a.row_ce[r] = NO_TERM; }
        }
        return;
    }
    V x[NV ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i].template load_as<STREAM>(z, V::at(i * NT + tid, vocab));

    // the teacher's shares (first wave) and the counts (last wave)
    float p[EPL], tm = -INFINITY, ps = 0.f, z_at[EPL], z_y = 0.f;
    if (wid == 0) {
#pragma unroll
        for (int q = 0; q < EPL; ++q) tm = fmaxf(tm, tv[q]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) tm = fmaxf(tm, __shfl_xor(tm, o));
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
            p[q] = tv[q] == -INFINITY ? 0.f : expf((tv[q] - tm) * a.inv_t);
            ps += p[q];
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) ps += __shfl_xor(ps, o);
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
            const int j = q * 64 + lane;
            p[q] = kd_on ? p[q] / ps : 0.f;
            z_at[q] = 0.f;
            if (j < top) {
                s_p[j] = p[q];
                s_i[j] = ti[q];
                if (ti[q] >= 0) z_at[q] = ElemTraits<T>::to_float(z[ti[q]]);
            }
        }
        if (y >= 0) z_y = ElemTraits<T>::to_float(z[y]);
        if (lane == 0) {
            s_p[top] = 0.f;
            s_i[top] = (int)y;
        }
    }
    if (wid == NT / 64 - 1 && dz) {
        int n_kd = 0, n_ce = 0;
        if (a.reduction == SUBREG_MEAN) {
            row_counts<TV, NT == 64>(a, lane, 64, n_kd, n_ce);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                n_kd += __shfl_xor(n_kd, o);
                n_ce += __shfl_xor(n_ce, o);
            }
        }
        if (lane == 0) {
            s_cnt[0] = (float)max(n_kd, 1);
            s_cnt[1] = (float)max(n_ce, 1);
        }
    }
    if constexpr (NT == 64) __syncthreads();         // (a block of one wave passes no barrier in its reductions, which order s_cnt elsewhere)

    // the student's softmax
    auto add = [](float p, float q) { return p + q; };
    auto larger = [](float p, float q) { return fmaxf(p, q); };
    auto exps = [&](float v, float mc, float mc1, float& et, float& e1) {
        et = exp2_fast(fmaf(v, a.c_t, -mc));
        if constexpr (SQ < 0) {
            e1 = exp2_fast(fmaf(v, LOG2E, -mc1));
        } else {
            e1 = et;
#pragma unroll
            for (int k = 0; k < SQ; ++k) e1 *= e1;
        }
    };
    float se = 0.f, s1 = 0.f;
    // load c (of thread 0: first) into the sums; elements that another load covers count 0
    auto sum = [&](V& l, int first, int c, float mc, float mc1) {
        l.forget();
        if ((first + NT) * N <= vocab) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float et, e1;
                exps(l.get(e), mc, mc1, et, e1);
                se += et;
                if constexpr (SQ != 0) s1 += e1;
            }
        } else {
            const int skip = V::skip(c, vocab);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float et, e1;
                exps(l.get(e), mc, mc1, et, e1);
                se += e >= skip ? et : 0.f;
                if constexpr (SQ != 0) s1 += e >= skip ? e1 : 0.f;
            }
        }
    };
    // (a running maximum starts at a floor that is not FAR, so that a thread that sees nothing but masks of -infinity or any large number
    // has sums relative to the floor: 0, or what is left of numbers near it)
    const float floor_m = -FAR / fmaxf(a.c_t, LOG2E);
    float m = NV ? -INFINITY : floor_m;
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) m = fmaxf(m, x[i].get(e));
    } else {
        constexpr int DEEP = 4;
        const int loads = (vocab + N - 1) / N;
        for (int c0 = 0; c0 < loads; c0 += DEEP * NT) {
            V l[DEEP];
#pragma unroll
            for (int i = 0; i < DEEP; ++i) l[i].load(z, V::at(c0 + i * NT + tid, vocab));
            const float mc_was = rounded_product(m, a.c_t), mc1_was = rounded_product(m, LOG2E);
#pragma unroll
            for (int i = 0; i < DEEP; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) m = fmaxf(m, l[i].get(e));
            const float mc = rounded_product(m, a.c_t), mc1 = rounded_product(m, LOG2E);
            se *= exp2_fast(mc_was - mc);
            if constexpr (SQ != 0) s1 *= exp2_fast(SQ < 0 ? mc1_was - mc1 : (mc_was - mc) * (float)(1 << max(SQ, 0)));
#pragma unroll
            for (int i = 0; i < DEEP; ++i)
                if ((c0 + i * NT) < loads) sum(l[i], c0 + i * NT, c0 + i * NT + tid, mc, mc1);
        }
    }
    const float mc_own = rounded_product(m, a.c_t), mc1_own = rounded_product(m, LOG2E);
    m = block_reduce(m, red, -INFINITY, larger);
    const float mc = rounded_product(m, a.c_t), mc1 = rounded_product(m, LOG2E);
    if (!(m > floor_m && fabsf(mc) <= FAR && fabsf(mc1) <= FAR)) {
        distill_any_row<T, TV, NT, NT == 64>(a, r);
        return;
    }
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) sum(x[i], i * NT, i * NT + tid, mc, mc1);
    } else {
        se *= exp2_fast(mc_own - mc);
        if constexpr (SQ != 0) s1 *= exp2_fast(SQ < 0 ? mc1_own - mc1 : (mc_own - mc) * (float)(1 << max(SQ, 0)));
    }
    se = block_reduce(se, red, 0.f, add);
    s1 = SQ == 0 ? se : block_reduce(s1, red1, 0.f, add);

    constexpr float LN2 = 0.69314718055994530942f;
    if (a.loss && wid == 0) {
        const float off = fmaf(m, a.c_t, -mc);       // what rounding m c left out: common to the exponents, but not to z - m
        const float t_ls = a.temp * LN2 * (log2f(se) - off - log2f(ps));
        float term = 0.f;
#pragma unroll
        for (int q = 0; q < EPL; ++q)
            if (p[q] > 0.f || p[q] != p[q])
                term += p[q] * (((tv[q] - tm) - (z_at[q] - m)) + t_ls);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) term += __shfl_xor(term, o);
        if (lane == 0) {
            if (bad) term = NAN;
            float ce = 0.f;
            if (ce_on) {
                const float off1 = SQ < 0 ? fmaf(m, LOG2E, -mc1) : off * (float)(1 << max(SQ, 0));
                ce = bad_y ? NAN : (log2f(s1) - off1) * LN2 - (z_y - m);
            }
            if (out) out[r] = a.kd * a.temp * term + a.ce * ce;
            else { a.row_kd[r] = kd_on ? term : NO_TERM; a.row_ce[r] = ce_on ? ce : NO_TERM; }
        }
    }
    if (dz) {
        const float ckd = bad ? NAN : kd_on ? g * a.kd * a.temp / s_cnt[0] : 0.f;
        const float cce = bad_y ? NAN : ce_on ? g * a.ce / s_cnt[1] : 0.f;
        const float akd = ckd / se, ace = cce / s1;          // (a term that the row does not have: 0)
        auto grad = [&](V& l, int c) {
            l.forget();
            typename V::V o;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float et, e1;
                exps(l.get(e), mc, mc1, et, e1);
                o[e] = ElemTraits<T>::from_float(SQ == 0 ? (akd + ace) * et : fmaf(ace, e1, akd * et));
            }
            V w;
            w.raw = __builtin_bit_cast(typename V::U, o);
            if (c * N < vocab) w.template store_as<STREAM>(dz, V::at(c, vocab));   // (where loads overlap, the same values twice)
        };
        int tid_again = tid;
        asm volatile("" : "+v"(tid_again));              // (the stores' offsets are made where they are used)
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) grad(x[i], i * NT + tid_again);
        } else {                                         // (a row too long for the registers: read a second time)
            constexpr int DEEP = 4;
            const int loads = (vocab + N - 1) / N;
            for (int c0 = 0; c0 < loads; c0 += DEEP * NT) {
                V l[DEEP];
#pragma unroll
                for (int i = 0; i < DEEP; ++i) l[i].load(z, V::at(c0 + i * NT + tid_again, vocab));
#pragma unroll
                for (int i = 0; i < DEEP; ++i) grad(l[i], c0 + i * NT + tid_again);
            }
        }
        __syncthreads();                                     // the row's stores are done: its entries and the label are written again
        for (int j = tid; j <= top; j += NT) {
            const int v = s_i[j];
            if (v < 0) continue;
            float pv = 0.f;
            bool first = true;
            for (int i = 0; i <= top; ++i)
                if (s_i[i] == v) {
                    if (i < j) first = false;
                    pv += s_p[i];
                }
            if (!first) continue;
            float et, e1, o = 0.f;
            exps(ElemTraits<T>::to_float(z[v]), mc, mc1, et, e1);
            o = akd * et - ckd * pv;
            o += ace * e1 - (v == (int)y ? cce : 0.f);
            dz[v] = ElemTraits<T>::from_float(o);
        }
    }
}

template <typename T, typename TV, int SQ>
static void launch_rows(const DistillArgs& a, hipStream_t s) {
    const long long loads = ((long long)a.vocab + RowVec<T>::N - 1) / RowVec<T>::N;
    // logits and gradient that the last-level cache (256 MB) does not hold together go past it: 4096 x 32000 bf16 140 -> 121 us a call,
    // 1024 x 131072 162 -> 152; 512 x 32000, which it holds, 30.6 -> 29.8
    const bool stream = (long long)a.rows * a.vocab * (long long)sizeof(T) >= (128ll << 20);
#define SUBREG_STREAM(NT, NV)                                                                                       \
    if (stream) hipLaunchKernelGGL((distill_row_kernel<T, TV, NT, NV, SQ, true>), a.rows, NT, 0, s, a);             \
    else SUBREG_ROWS(NT, NV)
#define SUBREG_ROWS(NT, NV) hipLaunchKernelGGL((distill_row_kernel<T, TV, NT, NV, SQ>), a.rows, NT, 0, s, a)
    if (a.vocab < RowVec<T>::N) {
        hipLaunchKernelGGL((distill_any_kernel<T, TV>), a.rows, 256, 0, s, a);
    } else if (loads <= 64) {
        SUBREG_ROWS(64, 1);
    } else if (loads <= 64 * 2) {
        SUBREG_ROWS(64, 2);
    } else if (!a.dz || loads > 1024 * 16) {
        SUBREG_ROWS(256, 0);
    } else if (loads <= 256 * 4) {
        SUBREG_ROWS(256, 4);
    } else if (loads <= 256 * 8) {
        SUBREG_ROWS(256, 8);
    } else if (loads <= 256 * 16) {
        SUBREG_STREAM(256, 16);
    } else if (loads <= 512 * 16) {
        SUBREG_STREAM(512, 16);
    } else {
        SUBREG_STREAM(1024, 16);
    }
#undef SUBREG_ROWS
#undef SUBREG_STREAM
}

template <typename TZ>
static int distill_launch(const DistillArgs& a, int values_dtype, hipStream_t s) {
    const bool count = a.reduction == SUBREG_MEAN && a.dz && a.count_blocks && !(a.flags & SUBREG_DISTILL_COUNTED);
    SUBREG_FOR_FLOAT(values_dtype, {
        if (count) hipLaunchKernelGGL(distill_count_kernel<T>, a.count_blocks, 256, 0, s, a);
        switch (a.target ? a.squarings : 0) {
            case 0: launch_rows<TZ, T, 0>(a, s); break;
            case 1: launch_rows<TZ, T, 1>(a, s); break;
            case 2: launch_rows<TZ, T, 2>(a, s); break;
            default: launch_rows<TZ, T, -1>(a, s); break;
        }
    })
    if (a.loss && a.reduction != SUBREG_NONE) hipLaunchKernelGGL(distill_finish_kernel, 1, 1024, 0, s, a);
    return launch_status();
}

}  // namespace subreg

using namespace subreg;

static inline long long distill_align(long long b) { return (b + 255) / 256 * 256; }

extern "C" long long subreg_distill_ws_bytes(int rows) {
    if (rows <= 0 || rows > MAX_ROWS) return SUBREG_EINVAL;
    return 2 * distill_align(4ll * rows) + distill_align(8 * COUNT_BLOCKS);
}

extern "C" int subreg_distill_loss(const subreg_distill_desc* d, void* stream) {
    SUBREG_CHECK_ARG(d && d->logits && d->top_values && d->top_indices && (d->loss || d->dlogits));
    SUBREG_CHECK_ARG(d->rows > 0 && d->rows <= MAX_ROWS && d->vocab > 0 && d->vocab <= MAX_COLUMNS && d->top >= 1 && d->top <= SUBREG_TOP_MAX);
    SUBREG_CHECK_ARG(d->logits_stride >= 0 && d->values_stride >= 0 && d->indices_stride >= 0 && d->grad_scale_stride >= 0);
    SUBREG_CHECK_ARG(float_dtype(d->dtype) && float_dtype(d->values_dtype) && d->temperature >= 1e-30f && d->temperature <= 1e15f);
    constexpr double MOST = 1e30 * (1.0 + 0x1p-20);   // (of numbers rounded to fp32)
    SUBREG_CHECK_ARG(fabs((double)d->kd_weight) * d->temperature * fmax(d->temperature, 1.0) <= MOST && fabs((double)d->ce_weight) <= MOST);
    SUBREG_CHECK_ARG(d->reduction >= SUBREG_NONE && d->reduction <= SUBREG_MEAN);
    SUBREG_CHECK_ARG(!(d->flags & SUBREG_DISTILL_SKIP_UNIT) || (d->grad_scale && d->dlogits && !d->loss));
    SUBREG_CHECK_ARG(d->ws && ((size_t)d->ws & 255) == 0 && d->ws_bytes >= subreg_distill_ws_bytes(d->rows));
    DistillArgs a;
    a.z = d->logits; a.tv = d->top_values; a.ti = d->top_indices; a.target = d->target;
    a.z_stride = d->logits_stride; a.tv_stride = d->values_stride; a.ti_stride = d->indices_stride; a.ignore = d->ignore_index;
    a.rows = d->rows; a.vocab = d->vocab; a.top = d->top; a.reduction = d->reduction; a.flags = d->flags;
    a.squarings = d->temperature == 1.f ? 0 : d->temperature == 2.f ? 1 : d->temperature == 4.f ? 2 : -1;
    a.count_rows = (int)((((long long)d->rows + COUNT_BLOCKS - 1) / COUNT_BLOCKS + 3) / 4 * 4);
    a.count_blocks = (int)(((long long)d->rows + a.count_rows - 1) / a.count_rows);
    const int small = 128 * (16 / dtype_bytes(d->dtype));            // (the kernels for short rows know how)
    if ((long long)d->rows * d->top <= COUNT_INLINE && d->vocab <= small) a.count_blocks = 0;
    a.temp = d->temperature; a.inv_t = 1.f / d->temperature; a.c_t = (float)(1.4426950408889634 / (double)d->temperature);
    a.kd = d->kd_weight; a.ce = d->ce_weight;
    a.gs = d->grad_scale; a.gs_stride = d->grad_scale_stride; a.loss = d->loss; a.dz = d->dlogits;
    char* ws = (char*)d->ws;
    a.row_kd = (float*)ws;
    a.row_ce = (float*)(ws + distill_align(4ll * d->rows));
    a.counts = (int*)(ws + 2 * distill_align(4ll * d->rows));
    SUBREG_FOR_FLOAT(d->dtype, return distill_launch<T>(a, d->values_dtype, (hipStream_t)stream))
    return SUBREG_EINVAL;
}
