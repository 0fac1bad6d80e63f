// Attention of new rows over a shared prefix and the sequences' own pages.
//
//   row r of sequence b (n_b rows; lens[b] own keys, the new rows' included) sits at i = P + lens[b] - n_b + r and sees the
//   P keys of the prefix and its own keys up to its own index:
//   out = sum_j softmax_j(scale q.k_j + slope_h (j - i)) v_j          zeros where there is no key to see
//   Key j of the prefix is row j % page of page prefix[j / page], own key j that of page table[b][j / page]; a page outside
//   the pool hides its keys.  Softmax statistics and sums are fp32.
#include "mgx_common.h"

namespace {

struct PagedArgs {
    const void *q, *kc, *vc;
    void* out;
    const int *table, *lens, *cu, *prefix;
    const float* slopes;
    int B, R, Hq, Hkv, dh, page, n_pages, width, P, max_rows, max_len;
    long T, qs;                                   // rows, elements from one row of q to the next
    float scale;
};

// sequence, row in it, rows of it, whether row t belongs to one
__device__ __forceinline__ bool find_row(const PagedArgs& a, long t, int& b, int& r, int& n) {
    if (!a.cu) {
        b = (int)(t / a.R);
        r = (int)(t - (long)b * a.R);
        n = a.R;
        return true;
    }
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= t) lo = mid;
        else hi = mid;
    }
    b = lo;
    r = (int)t - a.cu[b];
    n = a.cu[b + 1] - a.cu[b];
    return r >= 0 && r < n;
}

// One workgroup of 4 waves per (row, head); a key row is spread over lpr lanes, 16 bytes each.
template <typename T>
__global__ __launch_bounds__(256) void paged_attn_row_kernel(const PagedArgs a, int lpr) {
    constexpr int N = 16 / sizeof(T);
    __shared__ float part[4][256 + 2];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const long t = blockIdx.x;
    const int h = blockIdx.y, hk = h / (a.Hq / a.Hkv);
    int b, r, n;
    const bool real = find_row(a, t, b, r, n);
    const int own = real ? min(max(a.lens[b] - n + r + 1, 0), a.width * a.page) : 0;
    const int keys = real ? a.P + own : 0, i = keys - 1;
    const int sub = lane / lpr, ch = lane % lpr, rpl = 64 / lpr;
    const bool has = ch * N < a.dh;
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    float q[N], acc[N], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        q[k] = has && real ? to_f32(((const T*)a.q)[t * a.qs + (long)h * a.dh + ch * N + k]) : 0.f;
        acc[k] = 0.f;
    }
    for (int j0 = w * rpl; j0 < keys; j0 += 4 * rpl) {
        const int j = j0 + sub, jo = j - a.P;
        int pg = -1;
        if (j < keys) pg = jo < 0 ? a.prefix[j / a.page] : a.table[(long)b * a.width + jo / a.page];
        const bool see = (unsigned)pg < (unsigned)a.n_pages;
        const long at = (((long)pg * a.Hkv + hk) * a.page + (jo < 0 ? j : jo) % a.page) * a.dh + ch * N;
        float s = 0.f, v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            v[k] = see && has ? to_f32(((const T*)a.vc)[at + k]) : 0.f;
            s = fmaf(q[k], see && has ? to_f32(((const T*)a.kc)[at + k]) : 0.f, s);
        }
        for (int o = 1; o < lpr; o <<= 1) s += __shfl_xor(s, o, 64);
        if (see) {
            s = s * a.scale + slope * (float)(j - i);
            const float mn = fmaxf(m, s);
            const float alpha = mn == -INFINITY ? 1.f : expf(m - mn), p = mn == -INFINITY ? 0.f : expf(s - mn);
            l = l * alpha + p;
            m = mn;
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] = fmaf(p, v[k], acc[k] * alpha);
        }
    }
    for (int o = lpr; o < 64; o <<= 1) {
        const float m2 = __shfl_xor(m, o, 64), l2 = __shfl_xor(l, o, 64), mn = fmaxf(m, m2);
        const float a1 = mn == -INFINITY ? 1.f : expf(m - mn), a2 = mn == -INFINITY ? 1.f : expf(m2 - mn);
        l = l * a1 + l2 * a2;
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = acc[k] * a1 + __shfl_xor(acc[k], o, 64) * a2;
        m = mn;
    }
    if (sub == 0 && has) {
#pragma unroll
        for (int k = 0; k < N; ++k) part[w][ch * N + k] = acc[k];
        if (ch == 0) part[w][256] = m, part[w][257] = l;
    }
    __syncthreads();
    if (tid < a.dh) {
        const float mm = fmaxf(fmaxf(part[0][256], part[1][256]), fmaxf(part[2][256], part[3][256]));
        float num = 0.f, den = 0.f;
        for (int ww = 0; ww < 4; ++ww) {
            const float f = part[ww][256] == mm ? 1.f : expf(part[ww][256] - mm);
            num = fmaf(part[ww][tid], f, num);
            den = fmaf(part[ww][257], f, den);
        }
        ((T*)a.out)[(t * a.Hq + h) * a.dh + tid] = from_f32<T>(den == 0.f ? 0.f : num / den);
    }
}

}  // namespace

extern "C" long mgx_paged_attn_workspace_floats(long T, int B, int Hq, int Hkv, int dh, int prefix_len, int max_rows,
                                                int max_len, int dtype) {
    return 0;
}

extern "C" int mgx_paged_attn(const void* q, long q_row_stride, const void* kcache, const void* vcache, const int* table,
                              const int* lens, const int* cu_rows, const float* slopes, const int* prefix, void* out,
                              float* workspace, long T, int B, int R, int Hq, int Hkv, int dh, int page, int n_pages,
                              int width, int prefix_len, int max_rows, int max_len, float scale, int dtype, void* stream) {
    MGX_REQUIRE(q && kcache && vcache && table && lens && out, MGX_EINVAL, "mgx_paged_attn: null pointer");
    MGX_REQUIRE(T > 0 && T < (1L << 31) && B > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && dh > 0 && page > 0 && n_pages > 0 &&
                    width > 0,
                MGX_EINVAL, "mgx_paged_attn: T=%ld B=%d Hq=%d Hkv=%d dh=%d page=%d pages=%d width=%d", T, B, Hq, Hkv, dh,
                page, n_pages, width);
    MGX_REQUIRE(cu_rows || (R > 0 && (long)B * R == T), MGX_EINVAL, "mgx_paged_attn: B=%d x R=%d rows, got %ld", B, R, T);
    MGX_REQUIRE(prefix_len >= 0 && (prefix || prefix_len == 0), MGX_EINVAL, "mgx_paged_attn: prefix of %d keys", prefix_len);
    MGX_REQUIRE((long)page * width + prefix_len < (1L << 30), MGX_EUNSUPPORTED, "mgx_paged_attn: more than 2^30 keys");
    MGX_REQUIRE(max_rows > 0 && max_len > 0, MGX_EINVAL, "mgx_paged_attn: max_rows=%d max_len=%d", max_rows, max_len);
    MGX_REQUIRE(dtype == MGX_F32 || dtype == MGX_BF16, MGX_EINVAL, "mgx_paged_attn: bad dtype %d", dtype);
    const int N = dtype == MGX_F32 ? 4 : 8;
    MGX_REQUIRE(dh % N == 0 && dh <= 256, MGX_EUNSUPPORTED, "mgx_paged_attn: head dim %d must be a multiple of %d up to 256", dh, N);
    MGX_REQUIRE(q_row_stride >= (long)Hq * dh && q_row_stride % N == 0, MGX_EINVAL, "mgx_paged_attn: row stride %ld", q_row_stride);
    MGX_REQUIRE((((uintptr_t)q | (uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)out) & 15) == 0, MGX_EINVAL,
                "mgx_paged_attn: tensors must be 16-byte aligned");
    MGX_REQUIRE(Hq <= 65535, MGX_EUNSUPPORTED, "mgx_paged_attn: Hq=%d", Hq);
    const PagedArgs a{q, kcache, vcache, out, table, lens, cu_rows, prefix, slopes, B, R, Hq, Hkv, dh, page, n_pages, width,
                      prefix_len, max_rows, max_len, T, q_row_stride, scale};
    int lpr = 1;
    while (lpr * N < dh) lpr *= 2;
    const dim3 grid((unsigned)T, Hq);
    if (dtype == MGX_F32) hipLaunchKernelGGL((paged_attn_row_kernel<float>), grid, dim3(256), 0, (hipStream_t)stream, a, lpr);
    else hipLaunchKernelGGL((paged_attn_row_kernel<bf16_t>), grid, dim3(256), 0, (hipStream_t)stream, a, lpr);
    MGX_CHECK_LAUNCH("paged_attn");
    return MGX_OK;
}
