// Rotary positions in every form a model family uses, and the filing of rotated keys in a paged cache.
//
//   interleaved: pairs (x[2i], x[2i+1]);  half: pairs (x[i], x[i + rd/2]);  i < rd/2, the other dh - rd values pass through
//   y[a] = x[a] cos_i(p) - x[b] sin_i(p),  y[b] = x[b] cos_i(p) + x[a] sin_i(p)          p = the row's position
//   transposed (sin negated): the gradient.  Arithmetic in fp32, one rounding to the storage type at the end.
//
// Both kernels are bound by HBM: every value is read and written once.  Work split: a "unit" is what one thread turns
// for one head - one 16-byte vector (interleaved), or the two vectors of a pair of halves - and one thread takes the
// same unit of HPT heads of one row.  The angles (4 bytes each of cos and sin per pair, twice the bytes of a bf16 value
// pair) are then loaded once for HPT heads instead of once per head, and HPT vectors are in flight.  Consecutive lanes
// take consecutive units, then head groups, so a wave's request covers whole heads (128 bytes and more).
// Measured (a copy of 1 GiB moves 5.15 TB/s): q | k heads of 16 x 2048 rows, 16 heads of 64, bf16: 26 us = 5.1 TB/s;
// prompts of 16.5 k rows, 32 + 2 x 8 heads of 128, rotated and filed: 78.7 us = 5.15 TB/s; one row for each of 64 sequences:
// 4.5 us, of which the launch, two dependent loads (length, page) and the row's own are nearly all.  Sizes off the 16-byte
// grid (bf16, half layout, 40 of 80 values turned) take units of one value: 1.8 TB/s, rotated or filed (32 of 80: 3.8).
#include "mgx_common.h"

namespace {

// N consecutive values as one access: 16 bytes where the launcher found sizes, strides and pointers to be multiples of
// that, single values (N <= 2) otherwise.
template <typename T, int N>
struct Vals {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Vals<T, N> load_vals(const T* p) {
    Vals<T, N> r;
    if constexpr (N * sizeof(T) == 16) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(p);
        __builtin_memcpy(&r, &x, 16);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) r.v[k] = p[k];
    }
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_vals(T* p, const Vals<T, N>& r) {
    if constexpr (N * sizeof(T) == 16) {
        f32x4 x;
        __builtin_memcpy(&x, &r, 16);
        *reinterpret_cast<f32x4*>(p) = x;
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) p[k] = r.v[k];
    }
}

// The cos and sin a unit needs: N/2 pairs (interleaved) or N pairs (half).
template <int N, bool HALF>
struct Angles {
    static constexpr int P = HALF ? N : N / 2;
    float c[P], s[P];
};
template <int N, bool HALF>
__device__ __forceinline__ Angles<N, HALF> load_angles(const float* cs, const float* sn, int first, float sign) {
    Angles<N, HALF> a;
    constexpr int P = Angles<N, HALF>::P;
#pragma unroll
    for (int k = 0; k < P; ++k) {
        a.c[k] = cs[first + k];
        a.s[k] = sn[first + k] * sign;
    }
    return a;
}

// Geometry of the units of one head: `turn` of them rotate, the rest copy one vector each.
template <int N, bool HALF>
struct Units {
    int rd, dh, turn, all;
    __host__ __device__ Units(int rd_, int dh_) : rd(rd_), dh(dh_) {
        turn = HALF ? rd / (2 * N) : rd / N;
        all = turn + (dh - rd) / N;
    }
    // first value of unit u, and for a rotating unit of the half layout its partner rd/2 further
    __device__ __forceinline__ int at(int u) const { return u < turn ? u * N : rd + (u - turn) * N; }
    __device__ __forceinline__ int pair(int u) const { return u * (HALF ? N : N / 2); }
};

template <typename T, int N>
__device__ __forceinline__ void turn_interleaved(Vals<T, N>& x, const Angles<N, false>& a) {
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
        const float p = to_f32(x.v[2 * k]), q = to_f32(x.v[2 * k + 1]);
        x.v[2 * k] = from_f32<T>(p * a.c[k] - q * a.s[k]);
        x.v[2 * k + 1] = from_f32<T>(q * a.c[k] + p * a.s[k]);
    }
}
template <typename T, int N>
__device__ __forceinline__ void turn_half(Vals<T, N>& x, Vals<T, N>& y, const Angles<N, true>& a) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float p = to_f32(x.v[k]), q = to_f32(y.v[k]);
        x.v[k] = from_f32<T>(p * a.c[k] - q * a.s[k]);
        y.v[k] = from_f32<T>(q * a.c[k] + p * a.s[k]);
    }
}

constexpr int HPT = 4;        // heads per thread

struct RotaryArgs {
    const void* x;
    void* y;
    const float *cs, *sn;
    const void* pos;                                  // NULL: position = s
    int pos64, S, H, dh, rd, table_rows;
    long rows, xsb, xss, xsh, ysb, yss, ysh;
    float sign;
};

template <typename T, int N, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
    const Units<N, HALF> un(a.rd, a.dh);
    const int groups = (a.H + HPT - 1) / HPT, per_row = groups * un.all;
    const long e = (long)blockIdx.x * 256 + threadIdx.x;
    const long row = e / per_row;
    if (row >= a.rows) return;
    const int in_row = (int)(e - row * per_row);
    const int g = in_row / un.all, u = in_row - g * un.all;
    const long b = row / a.S;
    const int s = (int)(row - b * a.S);
    const bool turns = u < un.turn;
    if (!turns && a.x == a.y) return;                 // in place: what is not rotated stays
    long p = s;
    if (a.pos) p = a.pos64 ? reinterpret_cast<const long long*>(a.pos)[row] : reinterpret_cast<const int*>(a.pos)[row];
    p = p < 0 ? 0 : p >= a.table_rows ? a.table_rows - 1 : p;
    Angles<N, HALF> an;
    if (turns) an = load_angles<N, HALF>(a.cs + p * (a.rd / 2), a.sn + p * (a.rd / 2), un.pair(u), a.sign);
    const int h0 = g * HPT, nh = min(HPT, a.H - h0);
    const T* x = reinterpret_cast<const T*>(a.x) + b * a.xsb + s * a.xss + h0 * a.xsh + un.at(u);
    T* y = reinterpret_cast<T*>(a.y) + b * a.ysb + s * a.yss + h0 * a.ysh + un.at(u);
    Vals<T, N> lo[HPT], hi[HPT];
#pragma unroll
    for (int h = 0; h < HPT; ++h)
        if (h < nh) {
            lo[h] = load_vals<T, N>(x + h * a.xsh);
            if (HALF && turns) hi[h] = load_vals<T, N>(x + h * a.xsh + a.rd / 2);
        }
#pragma unroll
    for (int h = 0; h < HPT; ++h)
        if (h < nh) {
            if (turns) {
                if constexpr (HALF) turn_half<T, N>(lo[h], hi[h], an);
                else turn_interleaved<T, N>(lo[h], an);
            }
            store_vals<T, N>(y + h * a.ysh, lo[h]);
            if (HALF && turns) store_vals<T, N>(y + h * a.ysh + a.rd / 2, hi[h]);
        }
}

// ---- rotation and filing -----------------------------------------------------------------------------------------
// Row t of the packed projection [q heads | k heads | v heads] belongs to sequence b; its own index is
// lens[b] - n_b + r (lens counts the new rows), its position offset + index.  q goes out rotated, k (rotated) and v to
// slot index % page of page table[b][index / page].  A page outside the pool, an index outside the table and rows behind
// the last sequence file nothing (such rows' q is zero).
struct AppendArgs {
    const void* qkv;
    void *q, *kc, *vc;
    const int *table, *lens, *cu;                     // cu NULL: R rows for every sequence
    const float *cs, *sn;                             // NULL: no rotation, and q is not written
    int B, R, Hq, Hkv, dh, rd, page, n_pages, width, table_rows, offset;
    long T;
};

template <typename T, int N, bool HALF>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a) {
    const Units<N, HALF> un(a.rd, a.dh);
    const int first = a.cs ? 0 : a.Hq;                // no rotation: q stays where it is
    const int H = a.Hq + 2 * a.Hkv;
    const int groups = (H - first + HPT - 1) / HPT, per_row = groups * un.all;
    const long e = (long)blockIdx.x * 256 + threadIdx.x;
    const long t = e / per_row;
    if (t >= a.T) return;
    const int in_row = (int)(e - t * per_row);
    const int g = in_row / un.all, u = in_row - g * un.all;
    int b, r, n;
    bool real = true;
    if (a.cu) {                                       // the last sequence that begins at or before row t
        int lo = 0, hi = a.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.cu[mid] <= t) lo = mid;
            else hi = mid;
        }
        b = lo;
        r = (int)t - a.cu[b];
        n = a.cu[b + 1] - a.cu[b];
        real = r >= 0 && r < n;
    } else {
        b = (int)(t / a.R);
        r = (int)(t - (long)b * a.R);
        n = a.R;
    }
    const int index = min(max(a.lens[b], -(1 << 29)), 1 << 30) - n + r;      // (no sum of an absurd length overflows)
    T* kdst = nullptr;
    T* vdst = nullptr;
    if (real && index >= 0 && index / a.page < a.width) {
        const int pg = a.table[(long)b * a.width + index / a.page];
        if ((unsigned)pg < (unsigned)a.n_pages) {
            const long slot = ((long)pg * a.Hkv * a.page + index % a.page) * a.dh;      // head 0 of this key
            kdst = reinterpret_cast<T*>(a.kc) + slot;
            vdst = reinterpret_cast<T*>(a.vc) + slot;
        }
    }
    const bool turns = u < un.turn;                   // (the half layout's units move two vectors, v's too)
    Angles<N, HALF> an;
    if (turns && a.cs) {
        const long at = (long)a.offset + index;
        const long p = at < 0 ? 0 : at >= a.table_rows ? a.table_rows - 1 : at;
        an = load_angles<N, HALF>(a.cs + p * (a.rd / 2), a.sn + p * (a.rd / 2), un.pair(u), 1.f);
    }
    const int h0 = first + g * HPT, nh = min(HPT, H - h0);
    const int d0 = un.at(u);
    const T* x = reinterpret_cast<const T*>(a.qkv) + (t * H + h0) * a.dh + d0;
    Vals<T, N> lo[HPT], hi[HPT];
#pragma unroll
    for (int h = 0; h < HPT; ++h)
        if (h < nh) {
            lo[h] = load_vals<T, N>(x + h * a.dh);
            if (HALF && turns) hi[h] = load_vals<T, N>(x + h * a.dh + a.rd / 2);
        }
#pragma unroll
    for (int h = 0; h < HPT; ++h)
        if (h < nh) {
            const int head = h0 + h;
            T* dst;
            if (head < a.Hq) dst = reinterpret_cast<T*>(a.q) + (t * a.Hq + head) * a.dh;
            else if (head < a.Hq + a.Hkv) dst = kdst ? kdst + (long)(head - a.Hq) * a.page * a.dh : nullptr;
            else dst = vdst ? vdst + (long)(head - a.Hq - a.Hkv) * a.page * a.dh : nullptr;
            if (!dst) continue;
            if (turns && a.cs && head < a.Hq + a.Hkv) {
                if constexpr (HALF) turn_half<T, N>(lo[h], hi[h], an);
                else turn_interleaved<T, N>(lo[h], an);
            }
            if (!real) {
#pragma unroll
                for (int k = 0; k < N; ++k) lo[h].v[k] = hi[h].v[k] = from_f32<T>(0.f);
            }
            store_vals<T, N>(dst + d0, lo[h]);
            if (HALF && turns) store_vals<T, N>(dst + d0 + a.rd / 2, hi[h]);
        }
}

// cos and sin of position * freq[i], scaled by `amplitude`.  The angle and its functions are taken in 64 bits: at
// position 131072 an fp32 angle is off by up to 2^-8 rad.
__global__ __launch_bounds__(256) void rope_tables_kernel(const double* __restrict__ freq, float* __restrict__ cs,
                                                           float* __restrict__ sn, long n, int half, double amplitude) {
    const long e = (long)blockIdx.x * 256 + threadIdx.x;
    if (e >= n * half) return;
    const long p = e / half;
    double s, c;
    sincos((double)p * freq[e - p * half], &s, &c);
    cs[e] = (float)(c * amplitude);
    sn[e] = (float)(s * amplitude);
}

// units that move 16 bytes need every offset they touch to be a multiple of that
inline bool wide_units(int dh, int rd, int half, int N) { return dh % N == 0 && (half ? rd / 2 : rd) % N == 0; }

template <typename A>
int launch_units(void (*k)(const A), const A& a, long threads, const char* name, hipStream_t st) {
    const long blocks = (threads + 255) / 256;
    MGX_REQUIRE(grid_fits(blocks, 256), MGX_EUNSUPPORTED, "%s: too many rows", name);
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(256), 0, st, a);
    MGX_CHECK_LAUNCH(name);
    return MGX_OK;
}

template <typename T, int N, bool HALF>
int launch_rotary(const RotaryArgs& a, hipStream_t st) {
    const Units<N, HALF> un(a.rd, a.dh);
    return launch_units(rotary_kernel<T, N, HALF>, a, a.rows * ((a.H + HPT - 1) / HPT) * un.all, "rotary", st);
}
template <typename T, int N, bool HALF>
int launch_append(const AppendArgs& a, hipStream_t st) {
    const Units<N, HALF> un(a.rd, a.dh);
    const int heads = (a.cs ? a.Hq : 0) + 2 * a.Hkv;
    return launch_units(paged_append_kernel<T, N, HALF>, a, a.T * ((heads + HPT - 1) / HPT) * un.all, "paged_append", st);
}

inline bool multiple16(long elements, int dtype) { return elements % (dtype == MGX_F32 ? 4 : 8) == 0; }

}  // namespace

extern "C" int mgx_rope_tables(const double* freq, float* cos_tab, float* sin_tab, long n, int half, double amplitude,
                               void* stream) {
    MGX_REQUIRE(freq && cos_tab && sin_tab, MGX_EINVAL, "mgx_rope_tables: null pointer");
    MGX_REQUIRE(n > 0 && half > 0 && n <= (1L << 38) / half, MGX_EINVAL, "mgx_rope_tables: n=%ld half=%d", n, half);
    const long blocks = (n * half + 255) / 256;
    MGX_REQUIRE(grid_fits(blocks, 256), MGX_EUNSUPPORTED, "mgx_rope_tables: n=%ld half=%d", n, half);
    hipLaunchKernelGGL(rope_tables_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, freq, cos_tab,
                       sin_tab, n, half, amplitude);
    MGX_CHECK_LAUNCH("rope_tables");
    return MGX_OK;
}

extern "C" int mgx_rotary(const void* x, void* y, const float* cos_tab, const float* sin_tab, const void* positions,
                          int positions_are_int64, int B, int S, int H, int dh, int rd, int table_rows, long xsb, long xss,
                          long xsh, long ysb, long yss, long ysh, int half_layout, int transposed, int dtype,
                          void* stream) {
    MGX_REQUIRE(x && y && cos_tab && sin_tab, MGX_EINVAL, "mgx_rotary: null pointer");
    MGX_REQUIRE(B > 0 && S > 0 && H > 0 && dh > 0, MGX_EINVAL, "mgx_rotary: B=%d S=%d H=%d dh=%d", B, S, H, dh);
    MGX_REQUIRE(rd >= 2 && rd % 2 == 0 && rd <= dh, MGX_EINVAL, "mgx_rotary: rotary dim %d of head dim %d", rd, dh);
    MGX_REQUIRE(half_layout || dh % 2 == 0, MGX_EUNSUPPORTED, "mgx_rotary: interleaved layout needs an even head dim");
    MGX_REQUIRE(table_rows > 0 && (positions || S <= table_rows), MGX_EINVAL, "mgx_rotary: S=%d beyond %d table rows", S,
                table_rows);
    MGX_REQUIRE(dtype == MGX_F32 || dtype == MGX_BF16, MGX_EINVAL, "mgx_rotary: bad dtype %d", dtype);
    MGX_REQUIRE(x != y || (xsb == ysb && xss == yss && xsh == ysh), MGX_EINVAL, "mgx_rotary: in place needs equal strides");
    const RotaryArgs a{x,  y,  cos_tab,    sin_tab,     positions, positions_are_int64, S,   H,   dh,
                       rd, table_rows, (long)B * S, xsb, xss,       xsh,                 ysb, yss, ysh,
                       transposed ? -1.f : 1.f};
    hipStream_t st = (hipStream_t)stream;
    bool wide = wide_units(dh, rd, half_layout, dtype == MGX_F32 ? 4 : 8) && (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
    for (long stride : {xsb, xss, xsh, ysb, yss, ysh}) wide = wide && multiple16(stride, dtype);
    if (dtype == MGX_F32) {
        if (wide) return half_layout ? launch_rotary<float, 4, true>(a, st) : launch_rotary<float, 4, false>(a, st);
        return half_layout ? launch_rotary<float, 1, true>(a, st) : launch_rotary<float, 2, false>(a, st);
    }
    if (wide) return half_layout ? launch_rotary<bf16_t, 8, true>(a, st) : launch_rotary<bf16_t, 8, false>(a, st);
    return half_layout ? launch_rotary<bf16_t, 1, true>(a, st) : launch_rotary<bf16_t, 2, false>(a, st);
}

extern "C" int mgx_paged_append(const void* qkv, void* q_out, void* kcache, void* vcache, const int* table, const int* lens,
                                const int* cu_rows, const float* cos_tab, const float* sin_tab, long T, int B, int R,
                                int Hq, int Hkv, int dh, int rd, int page, int n_pages, int width, int table_rows,
                                int offset, int half_layout, int dtype, void* stream) {
    MGX_REQUIRE(qkv && kcache && vcache && table && lens, MGX_EINVAL, "mgx_paged_append: null pointer");
    MGX_REQUIRE((cos_tab != nullptr) == (sin_tab != nullptr) && (!cos_tab || q_out), MGX_EINVAL,
                "mgx_paged_append: cos, sin and q_out go together");
    MGX_REQUIRE(T > 0 && T < (1L << 30) && B > 0 && Hq > 0 && Hkv > 0 && dh > 0 && page > 0 && n_pages > 0 && width > 0,
                MGX_EINVAL, "mgx_paged_append: T=%ld B=%d Hq=%d Hkv=%d dh=%d page=%d pages=%d width=%d", T, B, Hq, Hkv, dh,
                page, n_pages, width);
    MGX_REQUIRE(cu_rows || (R > 0 && (long)B * R == T), MGX_EINVAL, "mgx_paged_append: B=%d x R=%d rows, got %ld", B, R, T);
    MGX_REQUIRE((long)page * width < (1L << 30), MGX_EUNSUPPORTED, "mgx_paged_append: table beyond 2^30 keys");
    MGX_REQUIRE(offset >= 0, MGX_EINVAL, "mgx_paged_append: offset %d", offset);
    MGX_REQUIRE(dtype == MGX_F32 || dtype == MGX_BF16, MGX_EINVAL, "mgx_paged_append: bad dtype %d", dtype);
    const int N = dtype == MGX_F32 ? 4 : 8;
    MGX_REQUIRE(dh % N == 0, MGX_EUNSUPPORTED, "mgx_paged_append: head dim %d must be a multiple of %d", dh, N);
    MGX_REQUIRE((((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)kcache | (uintptr_t)vcache) & 15) == 0, MGX_EINVAL,
                "mgx_paged_append: tensors must be 16-byte aligned");
    if (!cos_tab) rd = dh, half_layout = 0;           // plain copies: any unit will do
    MGX_REQUIRE(rd >= 2 && rd % 2 == 0 && rd <= dh, MGX_EINVAL, "mgx_paged_append: rotary dim %d of head dim %d", rd, dh);
    MGX_REQUIRE(!cos_tab || table_rows > 0, MGX_EINVAL, "mgx_paged_append: empty tables");
    const AppendArgs a{qkv, q_out, kcache, vcache, table, lens, cu_rows, cos_tab, sin_tab, B, R, Hq, Hkv, dh, rd, page,
                       n_pages, width, table_rows, offset, T};
    hipStream_t st = (hipStream_t)stream;
    const bool wide = wide_units(dh, rd, half_layout, N);
    if (dtype == MGX_F32) {
        if (wide) return half_layout ? launch_append<float, 4, true>(a, st) : launch_append<float, 4, false>(a, st);
        return half_layout ? launch_append<float, 1, true>(a, st) : launch_append<float, 2, false>(a, st);
    }
    if (wide) return half_layout ? launch_append<bf16_t, 8, true>(a, st) : launch_append<bf16_t, 8, false>(a, st);
    return half_layout ? launch_append<bf16_t, 1, true>(a, st) : launch_append<bf16_t, 2, false>(a, st);
}
