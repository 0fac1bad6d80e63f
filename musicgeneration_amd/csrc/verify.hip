// Verification of drafted tokens (speculative sampling) from given uniforms.
//
//   test i (in order, i < n): the draft's token x_i stays while u_i q_i(x_i) < p_i(x_i); a = the number that stay
//   then one token is drawn from  w = max(p_a - q_a, 0)  (a < n)  or  w = p_a  (a = n, or where the former is zero):
//   the smallest class c with  w_0 + .. + w_c > u_last (w_0 + .. + w_{V-1})
//   no draft distribution: q is the one-hot of the drafted token.  A value that is not a positive finite number weighs 0,
//   and a token of such a p does not stay.
//
// Bound by reading one row of p and one of q per sequence: one workgroup per sequence reads them ONCE for the total, and
// then only walks down: 16 slices -> the slice that holds the target, its 16 sub-slices -> the sub-slice, 64 classes at
// a time (1/16 + 1/256 of the row again, from L2).  Sums are fp64: a class of a 50k vocabulary weighs 2e-5, an fp32
// running sum would shift its borders by up to 1e-3 of that.  No atomics; the summation order is fixed.
// Measured: 128 sequences x 50257 classes fp32 (51 MB): 16 to 17 us of kernel (a copy of the bytes: 10); 4 sequences of
// 618 classes, where the chain of dependent steps is all there is: 6 us.  Few sequences leave most of the chip idle (1 of
// 50257 classes: 14 us in graph replays, 8: 15, 128: 19, in bf16 18).
#include "mgx_common.h"

namespace {

constexpr int NW = 16;

template <typename T>
struct Row {
    const T *p, *q;          // q NULL: nothing is taken off but the one-hot at `lost`
    long long lost;          // class whose weight is dropped, -1: none
    // positive and finite: classes 7 and 8 (denormal, normal) of v_cmp_class_f32
    __device__ __forceinline__ double clean(float x) const { return __builtin_amdgcn_classf(x, 0x180) ? (double)x : 0.0; }
    __device__ __forceinline__ double weight(float pv, float qv, long c) const {
        const double d = fmax(clean(pv) - clean(qv), 0.0);
        return c == lost ? 0.0 : d;
    }
    __device__ __forceinline__ double at(long c) const { return weight(to_f32(p[c]), q ? to_f32(q[c]) : 0.f, c); }
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// this wave's sum over classes [c0, c1): U independent loads in flight per lane
template <typename T>
__device__ __forceinline__ double slice_sum(const Row<T>& row, long c0, long c1, int lane) {
    constexpr int U = 16;
    double s[2] = {0.0, 0.0};
    long c = c0 + lane;
    for (; c + 64 * (U - 1) < c1; c += 64 * U) {
        float pv[U], qv[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            pv[k] = to_f32(row.p[c + 64 * k]);
            qv[k] = 0.f;
        }
        if (row.q) {
#pragma unroll
            for (int k = 0; k < U; ++k) qv[k] = to_f32(row.q[c + 64 * k]);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) s[k & 1] += row.weight(pv[k], qv[k], c + 64 * k);
    }
    for (; c < c1; c += 64) s[0] += row.at(c);
    return wave_sum64(s[0] + s[1]);
}

// The slice of the NW sums whose running total passes `target` (the last one with weight if none does), and the total
// before it.  Every thread computes the same.
__device__ __forceinline__ int pick(const double* sums, double target, double& before) {
    double run = before;
    int last = 0;
    double at_last = before;
    for (int w = 0; w < NW; ++w) {
        if (run + sums[w] > target) {
            before = run;
            return w;
        }
        if (sums[w] > 0.0) last = w, at_last = run;
        run += sums[w];
    }
    before = at_last;
    return last;
}

template <typename T, typename I>
__global__ __launch_bounds__(64 * NW) void verify_draft_kernel(const T* __restrict__ target, const T* __restrict__ draft,
                                                                const I* __restrict__ tokens, const float* __restrict__ u,
                                                                const int* __restrict__ counts, I* __restrict__ out,
                                                                int* __restrict__ accepted, int k, long V, long tsb,
                                                                long tsr, long dsb, long dsr) {
    __shared__ int s_acc;
    __shared__ double sums[NW];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const T* tp = target + b * tsb;
    const T* dp = draft ? draft + b * dsb : nullptr;
    const I* x = tokens + (long)b * k;
    const float* ub = u + (long)b * (k + 1);
    const int n = counts ? max(0, min(counts[b], k)) : k;
    if (w == 0) {
        int a = n;
        for (int i0 = 0; i0 < n; i0 += 64) {
            const int i = i0 + lane;
            bool fails = false;
            if (i < n) {
                const long long c = (long long)x[i];
                fails = true;                          // a class outside the vocabulary has p = 0
                if (c >= 0 && c < V) {
                    const double pv = to_f32(tp[i * tsr + c]), qv = dp ? to_f32(dp[i * dsr + c]) : 1.f;
                    fails = !((double)ub[i] * qv < pv && pv > 0.0 && pv < (double)INFINITY);
                }
            }
            const unsigned long long m = __ballot(fails);
            if (m) {
                a = i0 + __ffsll(m) - 1;
                break;
            }
        }
        if (lane == 0) s_acc = a;
    }
    __syncthreads();
    const int a = s_acc;
    Row<T> row{tp + a * tsr, nullptr, -1};
    if (a < n) {
        if (dp) row.q = dp + a * dsr;
        else row.lost = (long long)x[a];
    }
    const double draw = ub[k];
    const long part = (V + NW - 1) / NW, c0 = min(w * part, V), c1 = min(c0 + part, V);
    for (int pass = 0; pass < 2; ++pass) {
        const double s = slice_sum(row, c0, c1, lane);
        if (lane == 0) sums[w] = s;
        __syncthreads();
        double total = 0.0;
        for (int i = 0; i < NW; ++i) total += sums[i];
        if (total > 0.0 || a == n) break;              // (the same in every thread)
        row.q = nullptr;                               // nothing is left over: draw from p
        row.lost = -1;
        __syncthreads();
    }
    double total = 0.0;
    for (int i = 0; i < NW; ++i) total += sums[i];
    const double goal = draw * total;
    double before = 0.0;
    const long s0 = min(pick(sums, goal, before) * part, V), s1 = min(s0 + part, V);
    __syncthreads();
    const long sub = (s1 - s0 + NW - 1) / NW, d0 = min(s0 + w * sub, s1), d1 = min(d0 + sub, s1);
    const double ss = slice_sum(row, d0, d1, lane);
    if (lane == 0) sums[w] = ss;
    __syncthreads();
    if (w == 0) {
        const long e0 = min(s0 + pick(sums, goal, before) * sub, s1), e1 = min(e0 + sub, s1);
        long found = -1, last = 0;
        double run = before;
        for (long c = e0; c < e1 && found < 0; c += 64) {          // uniform over the wave
            const double v = c + lane < e1 ? row.at(c + lane) : 0.0;
            double scan = v;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double left = __shfl_up(scan, o, 64);
                if (lane >= o) scan += left;
            }
            const unsigned long long over = __ballot(v > 0.0 && run + scan > goal), some = __ballot(v > 0.0);
            if (over) found = c + __ffsll(over) - 1;
            if (some) last = c + 63 - __clzll(some);
            run += __shfl(scan, 63, 64);
        }
        if (found < 0) found = last;
        for (int i = lane; i <= k; i += 64) out[(long)b * (k + 1) + i] = i < a ? x[i] : (I)(i == a ? found : -1);
        if (lane == 0) accepted[b] = a;
    }
}

}  // namespace

extern "C" int mgx_verify_draft(const void* target, const void* draft, const void* tokens, int tokens_are_int64,
                                const float* uniforms, const int* counts, void* out, int* accepted, int B, int k, long V,
                                long target_stride_b, long target_stride_row, long draft_stride_b, long draft_stride_row,
                                int dtype, void* stream) {
    MGX_REQUIRE(target && uniforms && out && accepted && (tokens || k == 0), MGX_EINVAL, "mgx_verify_draft: null pointer");
    MGX_REQUIRE(B > 0 && k >= 0 && V > 0 && V < (1L << 31), MGX_EINVAL, "mgx_verify_draft: B=%d k=%d V=%ld", B, k, V);
    MGX_REQUIRE(dtype == MGX_F32 || dtype == MGX_BF16, MGX_EINVAL, "mgx_verify_draft: bad dtype %d", dtype);
    MGX_REQUIRE(grid_fits(B, 64 * NW), MGX_EUNSUPPORTED, "mgx_verify_draft: B=%d", B);
    hipStream_t st = (hipStream_t)stream;
#define MGX_VERIFY(T_, I_)                                                                                              \
    hipLaunchKernelGGL((verify_draft_kernel<T_, I_>), dim3(B), dim3(64 * NW), 0, st, (const T_*)target,                 \
                       (const T_*)draft, (const I_*)tokens, uniforms, counts, (I_*)out, accepted, k, V, target_stride_b, \
                       target_stride_row, draft_stride_b, draft_stride_row)
    if (dtype == MGX_F32) {
        if (tokens_are_int64) MGX_VERIFY(float, long long);
        else MGX_VERIFY(float, int);
    } else {
        if (tokens_are_int64) MGX_VERIFY(bf16_t, long long);
        else MGX_VERIFY(bf16_t, int);
    }
#undef MGX_VERIFY
    MGX_CHECK_LAUNCH("verify_draft");
    return MGX_OK;
}
