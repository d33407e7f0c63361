// Distillation from a teacher's top logits with the labels' cross entropy, loss and gradient in one pass over the student's logits.
//   p = softmax over a row's kept entries of t / T;  e_v = exp((z_v - m) / T), S = sum_v e_v;  likewise at T = 1 for the labels
//   KL = sum_j p_j (log p_j - (z_{i_j} - m) / T + log S);        CE = log S_1 - (z_y - m)
//   d(a T^2 KL)/dz_v = a T (e_v / S - sum_{j: i_j = v} p_j);     d(b CE)/dz_v = b (e1_v / S_1 - [v = y])
// Every row needs its maximum and two sums before its first gradient is known, so a row is read, reduced and written by one block.
#include "rows_common.h"

namespace subreg {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int COUNT_ROWS = 64;           // rows whose entries one block of the counting kernel looks at

struct DistillArgs {
    const void* z;
    const void* tv;
    const long long* ti;
    const long long* target;
    long long z_stride, tv_stride, ti_stride, ignore;
    int rows, vocab, top, reduction, flags, same_t, count_blocks;
    float c_t, inv_t, kd, ce, temp;      // c_t = log2(e) / T
    const float* gs;
    long long gs_stride;
    float* loss;
    void* dz;
    float* row_kd;                       // [rows] KL of the row (SUM / MEAN)
    float* row_ce;
    int* counts;                         // [count_blocks][2] rows with entries | with a label (MEAN)
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename TV>
__device__ __forceinline__ bool entry_kept(const DistillArgs& a, long long r, int j, float& v, long long& idx) {
    idx = a.ti[r * a.ti_stride + j];
    v = ElemTraits<TV>::to_float(((const TV*)a.tv)[r * a.tv_stride + j]);
    return idx >= 0 && !(v == -INFINITY);
}

template <typename TV>
__global__ __launch_bounds__(256) void distill_count_kernel(DistillArgs a) {
    __shared__ int red[16];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    int kd = 0, ce = 0;
    for (int i = wid; i < COUNT_ROWS; i += 4) {
        const long long r = (long long)blockIdx.x * COUNT_ROWS + i;
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

// loss[0] from the rows' terms, in a fixed order
__global__ __launch_bounds__(1024) void distill_finish_kernel(DistillArgs a) {
    __shared__ double red[16];
    double kd = 0, ce = 0, n_kd = 0, n_ce = 0;
    for (int r = threadIdx.x; r < a.rows; r += 1024) {
        kd += (double)a.row_kd[r];
        ce += (double)a.row_ce[r];
    }
    auto add = [](double p, double q) { return p + q; };
    kd = block_reduce(kd, red, 0.0, add);
    ce = block_reduce(ce, red, 0.0, add);
    if (a.reduction == SUBREG_MEAN) {
        for (int b = threadIdx.x; b < a.count_blocks; b += 1024) {
            n_kd += a.counts[2 * b];
            n_ce += a.counts[2 * b + 1];
        }
        n_kd = block_reduce(n_kd, red, 0.0, add);
        n_ce = block_reduce(n_ce, red, 0.0, add);
        kd /= fmax(n_kd, 1.0);
        ce /= fmax(n_ce, 1.0);
    }
    if (threadIdx.x == 0) a.loss[0] = (float)((double)a.kd * a.temp * a.temp * kd + (double)a.ce * ce);
}

template <typename T, typename TV>
__global__ __launch_bounds__(256) void distill_row_kernel(DistillArgs a) {
    __shared__ float red[16];
    __shared__ int redi[16];
    __shared__ float s_p[SUBREG_TOP_MAX + 1];
    __shared__ int s_i[SUBREG_TOP_MAX + 1];          // vocabulary entry, -1: none; the label is entry `top`
    const long long r = blockIdx.x;
    const int tid = threadIdx.x;
    const float g = a.gs ? a.gs[r * a.gs_stride] : 1.f;
    if ((a.flags & SUBREG_DISTILL_SKIP_UNIT) && g == 1.f) return;
    const T* z = (const T*)a.z + r * a.z_stride;
    T* dz = a.dz ? (T*)a.dz + r * a.vocab : nullptr;
    auto add = [](float p, float q) { return p + q; };
    auto addi = [](int p, int q) { return p + q; };
    auto mx = [](float p, float q) { return fmaxf(p, q); };

    // the teacher's share
    float tv = -INFINITY;
    long long ti = -1;
    const bool kept = tid < a.top && entry_kept<TV>(a, r, tid, tv, ti);
    const bool wild = kept && ti >= a.vocab;
    const int state = block_reduce((kept ? 1 : 0) + (wild ? 1 << 16 : 0), redi, 0, addi);
    const bool kd_on = (state & 0xffff) != 0;
    bool bad = state >> 16 != 0;
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
        for (int b = tid; b < a.count_blocks; b += 256) {
            n_kd += a.counts[2 * b];
            n_ce += a.counts[2 * b + 1];
        }
        cnt_kd = (float)max(1, block_reduce(n_kd, redi, 0, addi));
        cnt_ce = (float)max(1, block_reduce(n_ce, redi, 0, addi));
    }
    float* out = a.reduction == SUBREG_NONE ? a.loss : nullptr;
    if (!kd_on && !ce_on) {
        if (dz)
            for (int v = tid; v < a.vocab; v += 256) dz[v] = ElemTraits<T>::from_float(0.f);
        if (tid == 0 && a.loss) {
            if (out) out[r] = 0.f;
            else { a.row_kd[r] = 0.f; a.row_ce[r] = 0.f; }
        }
        return;
    }
    const float tm = block_reduce(kept ? tv : -INFINITY, red, -INFINITY, mx);
    float p = kept ? expf((tv - tm) * a.inv_t) : 0.f;
    const float ps = block_reduce(p, red, 0.f, add);
    p = kd_on ? p / ps : 0.f;
    if (tid < a.top) {
        s_p[tid] = p;
        s_i[tid] = kept && !wild ? (int)ti : -1;
    }
    if (tid == 0) {
        s_p[a.top] = 0.f;
        s_i[a.top] = (int)y;
    }

    // the student's softmax
    float m = -INFINITY;
    for (int v = tid; v < a.vocab; v += 256) m = fmaxf(m, ElemTraits<T>::to_float(z[v]));
    m = block_reduce(m, red, -INFINITY, mx);
    float se = 0.f, s1 = 0.f;
    for (int v = tid; v < a.vocab; v += 256) {
        const float d = ElemTraits<T>::to_float(z[v]) - m;
        se += exp2_fast(d * a.c_t);
        if (ce_on && !a.same_t) s1 += exp2_fast(d * LOG2E);
    }
    se = block_reduce(se, red, 0.f, add);
    s1 = a.same_t ? se : block_reduce(s1, red, 0.f, add);

    if (a.loss) {
        float term = 0.f;
        if (kept && !wild && !(p == 0.f))
            term = p * (((tv - tm) - (ElemTraits<T>::to_float(z[ti]) - m)) * a.inv_t + (logf(se) - logf(ps)));
        term = block_reduce(term, red, 0.f, add);
        if (tid == 0) {
            if (bad) term = NAN;
            const float ce = !ce_on ? 0.f : bad_y ? NAN : logf(s1) - (ElemTraits<T>::to_float(z[y]) - m);
            if (out) out[r] = a.kd * a.temp * a.temp * term + a.ce * ce;
            else { a.row_kd[r] = term; a.row_ce[r] = ce; }
        }
    }
    if (!dz) return;
    const float ckd = bad ? NAN : kd_on ? g * a.kd * a.temp / cnt_kd : 0.f;
    const float cce = bad_y ? NAN : ce_on ? g * a.ce / cnt_ce : 0.f;
    const float akd = ckd / se, ace = cce / s1;
    auto grad = [&](float zv, float pv, float hot) {
        const float d = zv - m;
        const float et = exp2_fast(d * a.c_t), e1 = a.same_t ? et : exp2_fast(d * LOG2E);
        float o = 0.f;
        if (kd_on) o = akd * et - ckd * pv;
        if (ce_on) o += ace * e1 - cce * hot;
        return o;
    };
    for (int v = tid; v < a.vocab; v += 256) dz[v] = ElemTraits<T>::from_float(grad(ElemTraits<T>::to_float(z[v]), 0.f, 0.f));
    __syncthreads();                                     // the row's stores are done: its entries and the label are written again
    for (int j = tid; j <= a.top; j += 256) {
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

template <typename TZ>
static int distill_launch(const DistillArgs& a, int values_dtype, hipStream_t s) {
    const bool count = a.reduction == SUBREG_MEAN && !(a.flags & SUBREG_DISTILL_COUNTED);
    SUBREG_FOR_FLOAT(values_dtype, {
        if (count) hipLaunchKernelGGL(distill_count_kernel<T>, a.count_blocks, 256, 0, s, a);
        hipLaunchKernelGGL((distill_row_kernel<TZ, T>), a.rows, 256, 0, s, a);
    })
    if (a.loss && a.reduction != SUBREG_NONE) hipLaunchKernelGGL(distill_finish_kernel, 1, 1024, 0, s, a);
    return launch_status();
}

}  // namespace subreg

using namespace subreg;

static inline long long distill_align(long long b) { return (b + 255) / 256 * 256; }

extern "C" long long subreg_distill_ws_bytes(int rows) {
    if (rows <= 0) return SUBREG_EINVAL;
    const long long blocks = ((long long)rows + COUNT_ROWS - 1) / COUNT_ROWS;
    return 2 * distill_align(4ll * rows) + distill_align(8 * blocks);
}

extern "C" int subreg_distill_loss(const subreg_distill_desc* d, void* stream) {
    SUBREG_CHECK_ARG(d && d->logits && d->top_values && d->top_indices && (d->loss || d->dlogits));
    SUBREG_CHECK_ARG(d->rows > 0 && d->vocab > 0 && d->vocab <= MAX_COLUMNS && d->top >= 1 && d->top <= SUBREG_TOP_MAX);
    SUBREG_CHECK_ARG(d->logits_stride >= 0 && d->values_stride >= 0 && d->indices_stride >= 0 && d->grad_scale_stride >= 0);
    SUBREG_CHECK_ARG(float_dtype(d->dtype) && float_dtype(d->values_dtype) && d->temperature > 0.f && d->temperature <= 3.0e38f);
    SUBREG_CHECK_ARG(d->reduction >= SUBREG_NONE && d->reduction <= SUBREG_MEAN);
    SUBREG_CHECK_ARG(!(d->flags & SUBREG_DISTILL_SKIP_UNIT) || (d->grad_scale && d->dlogits && !d->loss));
    SUBREG_CHECK_ARG(d->ws && ((size_t)d->ws & 255) == 0 && d->ws_bytes >= subreg_distill_ws_bytes(d->rows));
    DistillArgs a;
    a.z = d->logits; a.tv = d->top_values; a.ti = d->top_indices; a.target = d->target;
    a.z_stride = d->logits_stride; a.tv_stride = d->values_stride; a.ti_stride = d->indices_stride; a.ignore = d->ignore_index;
    a.rows = d->rows; a.vocab = d->vocab; a.top = d->top; a.reduction = d->reduction; a.flags = d->flags;
    a.same_t = d->temperature == 1.f;
    a.count_blocks = (int)(((long long)d->rows + COUNT_ROWS - 1) / COUNT_ROWS);
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
