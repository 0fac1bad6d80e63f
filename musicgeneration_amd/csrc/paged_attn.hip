// Attention of new rows over a shared prefix and the sequences' own pages.
//
//   row r of sequence b (n_b rows; lens[b] own keys, the new rows' included) sits at i = P + lens[b] - n_b + r and sees the
//   P keys of the prefix and its own keys up to its own index:
//   out = sum_j softmax_j(scale q.k_j + slope_h (j - i)) v_j          zeros where there is no key to see
//   Key j of the prefix is row j % page of page prefix[j / page], own key j that of page table[b][j / page]; a page outside
//   the pool hides its keys.  Softmax statistics and sums are fp32.
//
// Keys are numbered through, the prefix's 0..P-1 first.  A work item is (rows, key range): up to 32, 128 or 256 of the rows
// that read one K/V head - the G = Hq / Hkv query heads of a group are rows of the same tile - against a range of keys.
//   own items     rows of one sequence, its own keys (all keys, where the prefix is not taken apart)
//   prefix items  rows of the WHOLE batch, prefix keys: K and V of the prefix are read once per row tile of the batch
// Every product is arranged as K . Q^T and V^T . P^T on MFMA tiles: the row (query) is on the lane, so a row's maximum and
// sum need one or two exchanges between lanes per tile, and P goes from the first product's accumulators to the second's
// operand without leaving the registers (the order of the keys in it is free, V is read in the same one).  Two bodies:
//   private  <= 16 or 32 rows (16x16 tiles): memory bound.  The waves take alternate 32-key tiles, each through LDS of its
//            own with the next tile's loads in flight in registers: no barrier in the loop; waves are joined once at the end.
//            Four waves, or eight where few items have long ranges; two for fp32 heads wider than 128 (LDS).
//   shared   32 or 64 rows a wave (32x32 tiles), 128 or 256 in all: 64-key tiles in LDS, double buffered, shared by the
//            four waves.
// Ranges of one row are joined by a second kernel from unnormalised fp32 sums with their maxima (fixed order).
//
// bf16 weights: the private tiles take them into the product with V in two bf16 parts (15 bits or more); the shared tiles round
// them to bf16, and divide by the sum of the rounded ones.  Two parts there were measured: 128 x 6 rows behind 16385 keys 139
// -> 181 us, the prompts 378 -> 488, so they keep the rounding of the training attention (attn_mfma.hip).
//
// Measured (library product of 8192^3 bf16: 1172 TFLOP/s; copy: 5.15 TB/s; graph replays of calls one after another):
//   64 sequences x 1 row, 32 + 8 heads of 128, prefix 8192, own <= 1024     52 us   (own keys alone 36: 3.7 TB/s; prefix alone
//                                                                           32; together they overlap in part)
//   128 sequences x 6 rows, 20 + 4 heads of 64, prefix 16385, own <= 2006   143 us  479 TFLOP/s (137 to 154 from box to box and run
//                                                                           to run): a SIMD issues in 70 % of its busy cycles, its
//                                                                           matrix unit works in 29 %; 1.65 waves a SIMD
//   9 prompts of 1..1500 rows, 16 + 2 heads of 128, behind 4001 keys        381 us  673 TFLOP/s: issue 56 %, matrix unit 31 %; 1.51
//                                                                           waves a SIMD (852 row tiles on 512 slots: the second
//                                                                           round leaves slots empty)
//   1 prompt of 4096 / 8192 rows, 32 + 8 heads of 128, no prefix            228 / 709 us  604 / 776 TFLOP/s
//   16 sequences x 1 row, 8 heads of 64, own <= 2048                        14.5 us of kernel, 16 a call (one key each instead: 6 to 7)
//   1 sequence, 8 heads of 128, 30001 keys                                  36 us   (3.4 TB/s with the join)
//   16 sequences x 1 row, 8 heads of 256, own <= 2048                       43 us   (3.1 TB/s)
//   9 prompts of 1..1500 rows, 16 + 2 heads of 256, behind 4001 keys        1.04 to 1.12 ms 458 TFLOP/s
//   the prompts in fp32, heads of 128 / 64                                  3.08 / 1.44 ms  83 / 89 TFLOP/s (library product 154)
//   24 x 3 rows fp32, 12 + 4 heads of 64, prefix 1000, own <= 703           16 + 4 us: latency
// A launch whose items hold one key takes 5.6 us (1 sequence) to 8 us (64, heads of 128): the beginning (length, page, keys:
// three dependent loads) and the end of an item.  That is what limits splitting; the plan reckons 5 us an item.
#include "attn_mfma_common.h"

namespace {

struct PagedArgs {
    const void *q, *kc, *vc;
    void* out;
    const int *table, *lens, *cu, *prefix;
    const float* slopes;
    float *acc, *ml;                              // joined later: [split][row][dh] sums, [split][row][2] maximum (log2), sum
    int B, R, Hq, Hkv, dh, page, shift, n_pages, width, P;
    long T, qs;                                   // rows, elements from one row of q to the next
    float scale;
    // plan
    int share, Sp, So, chunk_p, chunk_o, rt_p, rt_o;
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

// Waves of a workgroup.  Four, two workgroups a CU: against eight (256 rows share a tile, half the reads from L2) prompts of
// dh 128 take 396 instead of 405 us and those of dh 64 243 instead of 280 - one group's barriers and softmax under the
// other's products, and a finer end.
constexpr int NW = 4;
constexpr unsigned NONE = 0xFFFFFFFFu;
constexpr float NEG = -1.0e30f;       // a running maximum before any key: finite, so differences stay numbers

// Where numbered key j lies, in rows of the pool, in two steps, so that the page number is loaded a tile before it is
// needed (a wait for it where it is loaded would wait for the tile's keys, too): the page's number - of key end - 1 behind
// the end, so that nothing is masked; end > 0 -, and the row, NONE where the key is hidden or not before `end`.
__device__ __forceinline__ unsigned page_of(const PagedArgs& a, const int* own, int j, int end) {
    j = min(j, end - 1);
    const bool pre = j < a.P;
    const int jj = pre ? j : j - a.P;
    return (unsigned)(pre ? a.prefix : own)[a.shift >= 0 ? jj >> a.shift : jj / a.page];
}
__device__ __forceinline__ unsigned slot_of(const PagedArgs& a, int hk, unsigned pg, int j, int end) {
    const int jj = j < a.P ? j : j - a.P;
    const int in_page = a.shift >= 0 ? jj & (a.page - 1) : jj % a.page;
    return j < end && pg < (unsigned)a.n_pages ? (pg * a.Hkv + hk) * a.page + in_page : NONE;
}

// ---- LDS images and matrix products per storage type ------------------------------------------------------------------
template <typename T, int DH> struct Prod;

template <int DH> struct Prod<bf16_t, DH> {       // v_mfma_f32_32x32x16_bf16; image of attn_mfma_common.h
    static constexpr int CH = DH / 8;             // 16-byte chunks per row
    static constexpr int KB = 32 * DH * 2, VB = KB;           // bytes of 32 rows
    typedef bf16x8 QFrag;
    static constexpr int NQ = DH / 16;
    const LaneAddr<DH> la;
    __device__ __forceinline__ Prod(int lane) : la(lane) {}
    // which 16-byte piece of 8 rows x 8 chunks a lane moves: eight consecutive lanes - the unit a ds_write_b128 is serviced
    // in - take four chunks of two rows, 2 x 64 bytes on different banks
    __device__ static __forceinline__ void piece(int lane, int& row, int& ch) {
        row = 2 * (lane >> 4) + ((lane >> 2) & 1);
        ch = (lane & 3) | ((lane >> 1) & 4);
    }
    __device__ static __forceinline__ int koff(int row, int ch) { return Img<DH>::off(row, ch); }
    __device__ static __forceinline__ int voff(int row, int ch) { return Img<DH>::off(row, ch); }
    __device__ static __forceinline__ int qchunk(int ks, int h5) { return 2 * ks + h5; }
    // Fragments are read a group ahead of the products (left alone, the compiler reads one, waits for it and multiplies: an
    // LDS latency per product), the first V fragments before the softmax.
    template <int NB, int RW>
    __device__ __forceinline__ void scores(const char* K, const QFrag (&q)[RW][NQ], f32x16 (&s)[RW][NB]) const {
        constexpr int GR = 4 / RW, NG = NB * NQ / GR;   // groups of fragments for four or eight products, one group ahead
        bf16x8 k[2][GR];
        auto read = [&](int gr) {
#pragma unroll
            for (int i = 0; i < GR; ++i) k[gr & 1][i] = lds_read16(K + la.row_read((gr * GR + i) / NQ, (gr * GR + i) % NQ));
        };
        read(0);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
            if (gr + 1 < NG) read(gr + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < GR; ++i) {
                const int tb = (gr * GR + i) / NQ, ks = (gr * GR + i) % NQ;
#pragma unroll
                for (int w = 0; w < RW; ++w) s[w][tb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[gr & 1][i], q[w][ks], s[w][tb], 0, 0, 0);
            }
        }
    }
    struct VAhead {
        bf16x8 f[DH / 32];
    };
    __device__ __forceinline__ VAhead vread(const char* V, int tb, int s2) const {
        VAhead v;
#pragma unroll
        for (int d = 0; d < DH / 32; ++d) v.f[d] = lds_read_tr_pair(V + la.tr_read(tb, s2, 0, d), V + la.tr_read(tb, s2, 1, d));
        return v;
    }
    // P is rounded to bf16 for the product (2^-8 relative each, signs independent; two parts cost a third of the time, see
    // above) and so for the sum, so that the weights add up to one; two values an instruction
    template <int NB, int RW>
    __device__ __forceinline__ void weigh(const char* V, VAhead now, const f32x16 (&p)[RW][NB], f32x16 (&o)[RW][DH / 32],
                                          float (&l)[RW]) const {
        const bf16x2 one = {(bf16_t)1.f, (bf16_t)1.f};
#pragma unroll
        for (int step = 0; step < 2 * NB; ++step) {
            VAhead next = now;
            if (step + 1 < 2 * NB) next = vread(V, (step + 1) >> 1, (step + 1) & 1);
            bf16x8 pf[RW];
#pragma unroll
            for (int w = 0; w < RW; ++w) {
                pf[w] = pack8(p[w][step >> 1], 8 * (step & 1));
#pragma unroll
                for (int k = 0; k < 8; k += 2) l[w] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{pf[w][k], pf[w][k + 1]}, one, l[w], false);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                for (int w = 0; w < RW; ++w) o[w][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(now.f[d], pf[w], o[w][d], 0, 0, 0);
            now = next;
        }
    }
    // values that are not finite become 0; whether there was one
    __device__ static __forceinline__ bool finite_only(f32x4& x) {
        bool bad = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            unsigned w = __float_as_uint(x[k]);
            const bool lo = (w & 0x7F80u) == 0x7F80u, hi = (w & 0x7F800000u) == 0x7F800000u;
            w = (lo ? 0u : w & 0xFFFFu) | (hi ? 0u : w & 0xFFFF0000u);
            x[k] = __uint_as_float(w);
            bad |= lo || hi;
        }
        return bad;
    }
};

template <int DH> struct Prod<float, DH> {        // v_mfma_f32_32x32x2_f32: the parity mode, products exact to fp32
    static constexpr int CH = DH / 4;
    static constexpr int VS = DH + 8;             // V row stride: rows 4 apart (the two half-waves) lie 32 banks apart
    static constexpr int KB = 32 * DH * 4, VB = 32 * VS * 4;
    typedef f32x4 QFrag;
    static constexpr int NQ = DH / 8;
    const int l31, h5;
    __device__ __forceinline__ Prod(int lane) : l31(lane & 31), h5(lane >> 5) {}
    __device__ static __forceinline__ void piece(int lane, int& row, int& ch) { row = lane >> 3, ch = lane & 7; }
    __device__ static __forceinline__ int koff(int row, int ch) { return row * DH * 4 + 16 * (ch ^ (row & 15)); }
    __device__ static __forceinline__ int voff(int row, int ch) { return row * VS * 4 + 16 * ch; }
    // the reduced index may be taken in any order: half-wave h5 owns chunk 2 c + h5, four steps of one value each
    __device__ static __forceinline__ int qchunk(int ks, int h) { return 2 * ks + h; }
    template <int NB, int RW>
    __device__ __forceinline__ void scores(const char* K, const QFrag (&q)[RW][NQ], f32x16 (&s)[RW][NB]) const {
#pragma unroll
        for (int c = 0; c < NQ; ++c)
#pragma unroll
            for (int tb = 0; tb < NB; ++tb) {
                const f32x4 k = *reinterpret_cast<const f32x4*>(K + tb * KB + koff(l31, 2 * c + h5));
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int w = 0; w < RW; ++w) s[w][tb] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[w][c][e], s[w][tb], 0, 0, 0);
            }
    }
    struct VAhead {};
    __device__ __forceinline__ VAhead vread(const char*, int, int) const { return {}; }
    template <int NB, int RW>
    __device__ __forceinline__ void weigh(const char* V, VAhead, const f32x16 (&p)[RW][NB], f32x16 (&o)[RW][DH / 32], float (&l)[RW]) const {
#pragma unroll
        for (int tb = 0; tb < NB; ++tb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float* v = reinterpret_cast<const float*>(V + tb * VB) + (8 * (r >> 2) + 4 * h5 + (r & 3)) * VS + l31;
#pragma unroll
                for (int w = 0; w < RW; ++w) l[w] += p[w][tb][r];
#pragma unroll
                for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                    for (int w = 0; w < RW; ++w) o[w][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[32 * d], p[w][tb][r], o[w][d], 0, 0, 0);
            }
    }
    __device__ static __forceinline__ bool finite_only(f32x4& x) {
        bool bad = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool is = (__float_as_uint(x[k]) & 0x7F800000u) == 0x7F800000u;
            x[k] = is ? 0.f : x[k];
            bad |= is;
        }
        return bad;
    }
};

// ---- 16x16 tiles: RT x 16 rows a wave, 32 keys at a time ----------------------------------------------------------------
template <typename T, int DH> struct Prod16;

template <int DH> struct Prod16<bf16_t, DH> {     // v_mfma_f32_16x16x32_bf16
    static constexpr int CH = DH / 8, G8 = 8 * DH * 2;
    static constexpr int KB = 32 * DH * 2, VB = KB;
    typedef bf16x8 QFrag;
    static constexpr int NQ = DH / 32;
    int k0, v0;
    // 8-row x 32-column sub-tiles of 512 bytes; the XOR spreads the four rows of equal row & 3 over a 64-byte line (row
    // reads of 16 rows) and puts rows 0-3 and 4-7 on different 32-byte halves (transposed reads): both conflict-free
    __device__ static __forceinline__ int swap(int row) { return 2 * ((row >> 2) & 1) | ((row >> 3) & 1); }
    __device__ static __forceinline__ int koff(int row, int ch) {
        return G8 * (row >> 3) + 512 * (ch >> 2) + 64 * (row & 7) + 16 * ((ch & 3) ^ swap(row));
    }
    __device__ static __forceinline__ int voff(int row, int ch) { return koff(row, ch); }
    __device__ static __forceinline__ void piece(int lane, int& row, int& ch) { Prod<bf16_t, DH>::piece(lane, row, ch); }
    __device__ static __forceinline__ bool finite_only(f32x4& x) { return Prod<bf16_t, DH>::finite_only(x); }
    __device__ __forceinline__ Prod16(int lane) {
        const int l15 = lane & 15, g = lane >> 4, q = l15 >> 2, p = l15 & 3;
        k0 = koff(l15, g);
        v0 = koff(4 * g + q, p >> 1) + 8 * (p & 1);
    }
    __device__ static __forceinline__ int qchunk(int ks, int g) { return 4 * ks + g; }
    // keys 16 kt + .. against the rows of q (fragments ahead of the products: see Prod)
    template <int RT>
    __device__ __forceinline__ void scores(const char* K, const QFrag (&q)[RT][NQ], f32x4 (&s)[RT][2]) const {
        bf16x8 k[NQ][2];
#pragma unroll
        for (int ks = 0; ks < NQ; ++ks)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) k[ks][kt] = lds_read16(K + k0 + 2 * G8 * kt + 512 * ks);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < NQ; ++ks)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) s[rt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[ks][kt], q[rt][ks], s[rt][kt], 0, 0, 0);
    }
    static constexpr int AH = 4;                  // V fragments read ahead
    struct VAhead {
        bf16x8 f[AH];
    };
    __device__ __forceinline__ VAhead vread(const char* V, int d0) const {
        VAhead v;
#pragma unroll
        for (int d = 0; d < AH; ++d) v.f[d] = vfrag(V, d0 + d);
        return v;
    }
    // p = hi + lo: hi the upper 16 bits of p, lo the rest, rounded to bf16 and larger by 2^-24 hi, so that it is not zero: V
    // values that are infinite come out as such
    __device__ static __forceinline__ void split(const f32x4 (&p)[2], bf16x8& hi, bf16x8& lo) {
        f32x4 top;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned a = __float_as_uint(p[k >> 1][2 * (k & 1)]), b = __float_as_uint(p[k >> 1][2 * (k & 1) + 1]);
            top[k] = __uint_as_float(__builtin_amdgcn_perm(b, a, 0x07060302u));
        }
        __builtin_memcpy(&hi, &top, 16);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float x = p[k >> 2][k & 3];
            lo[k] = (bf16_t)fmaf(__uint_as_float(__float_as_uint(x) & 0xFFFF0000u), -0x1.fffffep-1f, x);
        }
    }
    __device__ __forceinline__ bf16x8 vfrag(const char* V, int d) const {
        const char* at = V + (v0 ^ (32 * (d & 1))) + 512 * (d >> 1);
        return lds_read_tr_pair(at, at + 2 * G8);
    }
    // P goes into the product in two bf16 parts, so that it keeps 15 bits and more (the rest's rounding: 2^-8 of at most 2^-7 of
    // p), as in decode's fp32 products.  These bodies wait for memory: 16 sequences of up to 2048 keys take 16.1 instead of 15.3
    // us for it, the other cases 0 to 3 % more.
    template <int RT>
    __device__ __forceinline__ void weigh(const char* V, VAhead now, const f32x4 (&p)[RT][2], f32x4 (&o)[RT][DH / 16]) const {
        bf16x8 hi[RT], lo[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) split(p[rt], hi[rt], lo[rt]);
#pragma unroll
        for (int d0 = 0; d0 < DH / 16; d0 += AH) {
            VAhead next = now;
            if (d0 + AH < DH / 16) next = vread(V, d0 + AH);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int part = 0; part < 2; ++part)          // (the two products of an accumulator lie AH apart)
#pragma unroll
                for (int d = 0; d < AH; ++d)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        o[rt][d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(now.f[d], part ? lo[rt] : hi[rt], o[rt][d0 + d], 0, 0, 0);
            now = next;
        }
    }
};

template <int DH> struct Prod16<float, DH> {      // v_mfma_f32_16x16x4_f32
    static constexpr int CH = DH / 4;
    static constexpr int VS = DH + 4;             // V row stride: the four rows a request reads, 4 apart, lie 16 banks apart
    static constexpr int KB = 32 * DH * 4, VB = 32 * VS * 4;
    typedef f32x4 QFrag;
    static constexpr int NQ = DH / 16;
    const int l15, g;
    __device__ __forceinline__ Prod16(int lane) : l15(lane & 15), g(lane >> 4) {}
    __device__ static __forceinline__ int koff(int row, int ch) { return row * DH * 4 + 16 * (ch ^ (row & 15)); }
    __device__ static __forceinline__ int voff(int row, int ch) { return row * VS * 4 + 16 * ch; }
    __device__ static __forceinline__ void piece(int lane, int& row, int& ch) { row = lane >> 3, ch = lane & 7; }
    __device__ static __forceinline__ bool finite_only(f32x4& x) { return Prod<float, DH>::finite_only(x); }
    __device__ static __forceinline__ int qchunk(int ks, int g_) { return 4 * ks + g_; }
    template <int RT>
    __device__ __forceinline__ void scores(const char* K, const QFrag (&q)[RT][NQ], f32x4 (&s)[RT][2]) const {
#pragma unroll
        for (int c = 0; c < NQ; ++c)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const f32x4 k = *reinterpret_cast<const f32x4*>(K + koff(16 * kt + l15, 4 * c + g));
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        s[rt][kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], q[rt][c][e], s[rt][kt], 0, 0, 0);
            }
    }
    __device__ __forceinline__ float value(const char* V, int kt, int r, int d) const {
        return reinterpret_cast<const float*>(V)[(16 * kt + 4 * g + r) * VS + l15 + 16 * d];
    }
    struct VAhead {};
    __device__ __forceinline__ VAhead vread(const char*, int) const { return {}; }
    template <int RT>
    __device__ __forceinline__ void weigh(const char* V, VAhead, const f32x4 (&p)[RT][2], f32x4 (&o)[RT][DH / 16]) const {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int d = 0; d < DH / 16; ++d) {
                    const float v = value(V, kt, r, d);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) o[rt][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[rt][kt][r], o[rt][d], 0, 0, 0);
                }
    }
};

// ROWS keys' K and V on their way from the pool to LDS, spread over NWS waves.  A request of a wave is 8 rows x 128 bytes;
// request m of a tile covers rows 8 (m / (CH / 8)) and on, chunks 8 (m % (CH / 8)) and on: LDS addresses of one lane differ
// by constants from request to request.
template <typename P_, typename T, int DH, int ROWS, int NWS>
struct Stage {
    static constexpr int N = ROWS * P_::CH / 64 / NWS, W = P_::CH / 8;
    f32x4 k[N], v[N];
    int r0, c0;
    __device__ __forceinline__ Stage(int lane, int w) {
        P_::piece(lane, r0, c0);
        if constexpr (NWS > 1) {                  // wave w takes requests w N .. w N + N - 1
            r0 += 8 * (w * N / W);
            c0 += 8 * (w * N % W);
        }
    }
    // (N is a multiple of W or the other way round, so a wave's requests are a rectangle)
    __device__ __forceinline__ int row(int n) const { return r0 + 8 * (n / W); }
    __device__ __forceinline__ int chunk(int n) const { return c0 + 8 * (n % W); }
    // at: lane r's slot_of the tile's key r.  Rows that are nowhere read row 0 and are zeroed, so no load is masked.
    __device__ __forceinline__ void load(const PagedArgs& a, unsigned at, bool whole) {
        const unsigned bytes = a.dh * (unsigned)sizeof(T);
        const unsigned safe = at == NONE ? 0u : at;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const unsigned ch = 16u * chunk(n);
            const size_t off = (size_t)__shfl(safe, row(n), 64) * bytes + (whole || ch < bytes ? ch : 0u);
            k[n] = *reinterpret_cast<const f32x4*>((const char*)a.kc + off);
            v[n] = *reinterpret_cast<const f32x4*>((const char*)a.vc + off);
        }
    }
    __device__ __forceinline__ void clean(const PagedArgs& a, unsigned at) {
        const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const bool keep = __shfl(at, row(n), 64) != NONE && 16 * chunk(n) < a.dh * (int)sizeof(T);
            k[n] = keep ? k[n] : z;
            v[n] = keep ? v[n] : z;
        }
    }
    __device__ __forceinline__ bool v_finite_only() {
        bool bad = false;
#pragma unroll
        for (int n = 0; n < N; ++n) bad |= P_::finite_only(v[n]);
        return __any(bad);
    }
    __device__ __forceinline__ void store(char* K, char* V) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            *reinterpret_cast<f32x4*>(K + P_::koff(row(n), chunk(n))) = k[n];
            *reinterpret_cast<f32x4*>(V + P_::voff(row(n), chunk(n))) = v[n];
        }
    }
};

template <typename T, typename QFrag>
__device__ __forceinline__ QFrag load_q(const PagedArgs& a, const T* row, int ch) {
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (row && ch * 16 < a.dh * (int)sizeof(T)) x = *reinterpret_cast<const f32x4*>((const char*)row + ch * 16);
    if (a.scale < 0.f) {                                 // the scale's sign moves into q, exactly
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = __uint_as_float(__float_as_uint(x[k]) ^ (sizeof(T) == 2 ? 0x80008000u : 0x80000000u));
    }
    QFrag q;
    __builtin_memcpy(&q, &x, 16);
    return q;
}

// One wave's RW x 32 rows, row 32 i + (lane & 31) on two lanes (lane ^ 32 holds the other half of the keys of a tile).
template <typename T, int DH, int RW>
struct Rows {
    typedef Prod<T, DH> P_;
    typename P_::QFrag q[RW][P_::NQ];
    f32x16 o[RW][DH / 32];
    float m[RW], l[RW], bias[RW], c;      // running maximum (raw scores), sum, slope in raw-score units; |scale| * log2e
    int limit[RW], at[RW];                // last key the row sees, its position
    int first_limit, last_limit;          // the smallest and largest limit of the wave's rows

    __device__ __forceinline__ void begin(const PagedArgs& a) { c = fmaxf(fabsf(a.scale) * LOG2E, 1e-30f); }
    // row: this lane's row i of q (element pointer at its head), or NULL
    __device__ __forceinline__ void begin_row(const PagedArgs& a, int i, const T* row, int h5, float slope, int limit_, int at_) {
        bias[i] = slope * LOG2E / c;
        limit[i] = limit_;
        at[i] = at_;
        m[i] = NEG;
        l[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < P_::NQ; ++ks) q[i][ks] = load_q<T, typename P_::QFrag>(a, row, P_::qchunk(ks, h5));
#pragma unroll
        for (int d = 0; d < DH / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][d][r] = 0.f;
    }
    // NB blocks of 32 keys from j0 on; seen: the keys that are somewhere
    template <int NB, bool ALIBI>
    __device__ __forceinline__ void take(const P_& pr, const char* K, const char* V, int j0, unsigned long long seen, int h5) {
        f32x16 s[RW][NB];
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            const float lb = ALIBI ? bias[i] * (float)(j0 + 4 * h5 - at[i]) : 0.f;
#pragma unroll
            for (int tb = 0; tb < NB; ++tb)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[i][tb][r] = ALIBI ? fmaf(bias[i], (float)(32 * tb + (r & 3) + 8 * (r >> 2)), lb) : 0.f;
        }
        pr.template scores<NB, RW>(K, q, s);
        const typename P_::VAhead va = pr.vread(V, 0, 0);
        const unsigned long long all = NB == 2 ? ~0ull : 0xFFFFFFFFull;
        if (seen != all || j0 + 32 * NB - 1 > first_limit) {          // uniform
            const unsigned long long mine = seen >> (4 * h5);
#pragma unroll
            for (int i = 0; i < RW; ++i) {
                const int dj = limit[i] - j0 - 4 * h5;
#pragma unroll
                for (int tb = 0; tb < NB; ++tb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int kk = 32 * tb + (r & 3) + 8 * (r >> 2);
                        if (kk > dj || !((mine >> kk) & 1)) s[i][tb][r] = -INFINITY;
                    }
            }
        }
        float mx[RW];
        bool grown = false;
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            float x = s[i][0][0];
#pragma unroll
            for (int tb = 0; tb < NB; ++tb)
#pragma unroll
                for (int r = 0; r < 16; ++r) x = fmaxf(x, s[i][tb][r]);
            mx[i] = half_swap_max(x);
            grown |= (mx[i] - m[i]) * c > RESCALE_LOG2;
        }
        // A row's stale maximum stays until it has grown by more than 2^8: weights are then at most 2^8, which fp32 sums and
        // bf16 weights hold with the same relative precision.  Each row for itself: what another row of the wave holds (NaN,
        // infinities) does not change its result.
        if (__any(grown)) {
#pragma unroll
            for (int i = 0; i < RW; ++i) {
                const float mn = (mx[i] - m[i]) * c > RESCALE_LOG2 ? mx[i] : m[i];
                const float alpha = fast_exp2((m[i] - mn) * c);
                m[i] = mn;
                l[i] *= alpha;
#pragma unroll
                for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[i][d][r] *= alpha;
            }
        }
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            const float mc = m[i] * c;
#pragma unroll
            for (int tb = 0; tb < NB; ++tb)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[i][tb][r] = fast_exp2(fmaf(s[i][tb][r], c, -mc));
        }
        pr.template weigh<NB, RW>(V, va, s, o, l);
    }
    // Keys j0 .. j0+31, whose V values that are not finite were left out: rows that see such a key have them added (an infinity
    // times a weight is the infinity).
    __device__ __forceinline__ void spoil(const PagedArgs& a, const int* own, int hk, int j0, int end, int h5) {
        for (int j = j0; j < min(j0 + 32, end); ++j) {
            const unsigned kr = slot_of(a, hk, page_of(a, own, j, end), j, end);
            if (kr == NONE) continue;
            const T* v = (const T*)a.vc + (size_t)kr * a.dh;
#pragma unroll
            for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at_d = 32 * d + 8 * (r >> 2) + 4 * h5 + (r & 3);
                    const float x = at_d < a.dh ? to_f32(v[at_d]) : 0.f;
                    const bool bad = !(fabsf(x) < INFINITY);
#pragma unroll
                    for (int i = 0; i < RW; ++i)
                        if (bad && j <= limit[i]) o[i][d][r] += x;
                }
        }
    }
};

// over the four 16-lane groups, each of which holds other keys of the same 16 rows
__device__ __forceinline__ float quarter_max(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return half_swap_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarter_sum(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return half_swap_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// RT x 16 rows of a wave: row 16 rt + (lane & 15) on four lanes.
template <typename T, int DH, int RT>
struct Rows16 {
    typedef Prod16<T, DH> P_;
    typename P_::QFrag q[RT][P_::NQ];
    f32x4 o[RT][DH / 16];
    float m[RT], l[RT], bias[RT], c;
    int limit[RT], at[RT], first_limit, last_limit;

    __device__ __forceinline__ void begin(const PagedArgs& a) { c = fmaxf(fabsf(a.scale) * LOG2E, 1e-30f); }
    __device__ __forceinline__ void begin_row(const PagedArgs& a, int rt, const T* row, int g, float slope, int limit_, int at_) {
        bias[rt] = slope * LOG2E / c;
        limit[rt] = limit_;
        at[rt] = at_;
        m[rt] = NEG;
        l[rt] = 0.f;
#pragma unroll
        for (int ks = 0; ks < P_::NQ; ++ks) q[rt][ks] = load_q<T, typename P_::QFrag>(a, row, P_::qchunk(ks, g));
#pragma unroll
        for (int d = 0; d < DH / 16; ++d) o[rt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // 32 keys from j0 on (see Rows::take)
    __device__ __forceinline__ void take(const P_& pr, const char* K, const char* V, int j0, unsigned seen, int g) {
        f32x4 s[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const float lb = bias[rt] * (float)(j0 + 4 * g - at[rt]);
#pragma unroll
                for (int r = 0; r < 4; ++r) s[rt][kt][r] = fmaf(bias[rt], (float)(16 * kt + r), lb);
            }
        pr.template scores<RT>(K, q, s);
        const typename P_::VAhead va = pr.vread(V, 0);
        const bool mask = seen != 0xFFFFFFFFu || j0 + 31 > first_limit;          // uniform
        bool grown = false;
        float mx[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (mask) {
                const int dj = limit[rt] - j0 - 4 * g;
                const unsigned mine = seen >> (4 * g);
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (16 * kt + r > dj || !((mine >> (16 * kt + r)) & 1)) s[rt][kt][r] = -INFINITY;
            }
            float x = s[rt][0][0];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) x = fmaxf(x, s[rt][kt][r]);
            mx[rt] = quarter_max(x);
            grown |= (mx[rt] - m[rt]) * c > RESCALE_LOG2;
        }
        if (__any(grown)) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float mn = (mx[rt] - m[rt]) * c > RESCALE_LOG2 ? mx[rt] : m[rt];      // (see Rows::take)
                const float alpha = fast_exp2((m[rt] - mn) * c);
                m[rt] = mn;
                l[rt] *= alpha;
#pragma unroll
                for (int d = 0; d < DH / 16; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[rt][d][r] *= alpha;
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float mc = m[rt] * c;
            float sum = 0.f;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[rt][kt][r] = fast_exp2(fmaf(s[rt][kt][r], c, -mc));
                    sum += s[rt][kt][r];
                }
            l[rt] += sum;
        }
        pr.template weigh<RT>(V, va, s, o);
    }
    __device__ __forceinline__ void spoil(const PagedArgs& a, const int* own, int hk, int j0, int end, int g) {      // see Rows::spoil
        for (int j = j0; j < min(j0 + 32, end); ++j) {
            const unsigned kr = slot_of(a, hk, page_of(a, own, j, end), j, end);
            if (kr == NONE) continue;
            const T* v = (const T*)a.vc + (size_t)kr * a.dh;
#pragma unroll
            for (int d = 0; d < DH / 16; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at_d = 16 * d + 4 * g + r;
                    const float x = at_d < a.dh ? to_f32(v[at_d]) : 0.f;
                    const bool bad = !(fabsf(x) < INFINITY);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        if (bad && j <= limit[rt]) o[rt][d][r] += x;
                }
        }
    }
};

template <typename T>
__device__ __forceinline__ void put4(T* p, const float* x) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    } else {
        bf16x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (bf16_t)x[k];
        *reinterpret_cast<bf16x4*>(p) = v;
    }
}

struct Item {
    bool prefix, direct;         // prefix: rows of the whole batch, prefix keys; direct: the output itself, nothing to join
    int b, hk, rt, rts, split;   // row tile and tiles in the grid; split: slot among the parts that are joined
    int k0, k1, n, first;        // key range, rows of the sequence, position of its first new row
    long row0;                   // first row (of q) of the sequence
};

// a length as the device holds it, kept where sums with it do not overflow (longer tables are refused)
__device__ __forceinline__ int sane(int len) { return min(max(len, -(1 << 29)), 1 << 30); }

__device__ __forceinline__ bool own_item(const PagedArgs& a, int id, Item& it) {
    it.prefix = false;
    it.rts = a.rt_o;
    const unsigned per_head = a.So, per_tile = per_head * a.Hkv, per_seq = per_tile * a.rt_o;
    unsigned rest = id;
    it.b = rest / per_seq;
    rest -= it.b * per_seq;
    it.rt = a.rt_o == 1 ? 0 : rest / per_tile;
    rest -= it.rt * per_tile;
    it.hk = per_head == 1 ? rest : rest / per_head;
    it.split = rest - it.hk * per_head;
    it.row0 = (long)it.b * a.R;
    it.n = a.R;
    if (a.cu) {                                   // (offsets that are none stay inside the rows)
        it.row0 = min(max((long)a.cu[it.b], 0L), a.T);
        it.n = (int)(min(max((long)a.cu[it.b + 1], it.row0), a.T) - it.row0);
    }
    const int last = sane(a.lens[it.b]);
    it.first = a.P + last - it.n;
    it.direct = !a.share && a.So == 1;
    const int base = a.share ? a.P : 0, end = a.P + min(max(last, 0), a.width * a.page);
    // ranges of chunk_o keys, the last one open: it takes what a longer sequence than announced has left
    it.k0 = base + it.split * a.chunk_o;
    it.k1 = it.split == a.So - 1 ? end : min(end, it.k0 + a.chunk_o);
    it.split += a.share ? a.Sp : 0;
    return it.n > 0 && (it.k0 < it.k1 || it.split == (a.share ? a.Sp : 0));
}
__device__ __forceinline__ int own_parts(const PagedArgs& a, int own) {         // the own parts that exist, at least one
    const int keys = a.share ? own : a.P + own;
    return min(max((keys + a.chunk_o - 1) / a.chunk_o, 1), a.So);
}
__device__ __forceinline__ void prefix_item(const PagedArgs& a, int id, Item& it) {
    // the row tiles of one (head, range) on one XCD (workgroup n runs on XCD n % 8), so that its L2 serves all but the first
    const int pairs = a.Hkv * a.Sp, x = id & 7, rest = id >> 3;
    it.prefix = true;
    it.direct = false;
    it.rts = a.rt_p;
    it.rt = rest % a.rt_p;
    const int pair = (rest / a.rt_p) * 8 + x;
    it.hk = pair < pairs ? pair % a.Hkv : -1;
    it.split = pair / a.Hkv;
    it.b = 0;
    it.row0 = 0;
    it.n = (int)a.T;
    it.first = a.P;
    it.k0 = it.split * a.chunk_p;
    it.k1 = min(a.P, it.k0 + a.chunk_p);
}

// this lane's row of an item: its row of q (NULL: none), head, last key it sees, position
template <typename T>
__device__ __forceinline__ const T* item_row(const PagedArgs& a, const Item& it, int rho, int G, long& t, int& h, int& limit, int& at) {
    const int r = (unsigned)rho / (unsigned)G;
    t = it.row0 + r;
    h = it.hk * G + rho - r * G;
    limit = at = a.P - 1;
    if (rho >= it.n * G || t >= a.T) return nullptr;
    if (!it.prefix) {
        at = it.first + r;
        limit = max(at, a.P - 1);
    } else if (a.slopes) {
        int b, rb, n;
        if (find_row(a, t, b, rb, n)) at = a.P + sane(a.lens[b]) - n + rb;
    }
    return (const T*)a.q + t * a.qs + (long)h * a.dh;
}
// the smallest and largest last key of rows rho0 .. rho0 + rows - 1 of an item (limits ascend with the row)
__device__ __forceinline__ void item_limits(const PagedArgs& a, const Item& it, int rho0, int rows, int G, int& lo, int& hi) {
    const int total = it.n * G;
    lo = hi = a.P - 1;
    if (rho0 >= total) lo = 0x7FFFFFFF, hi = -1;
    else if (!it.prefix) {
        lo = max(it.first + (int)((unsigned)rho0 / (unsigned)G), a.P - 1);
        hi = max(it.first + (int)((unsigned)(min(rho0 + rows, total) - 1) / (unsigned)G), a.P - 1);
    }
}

template <typename T, int DH, int RT, int NWP>
__device__ __forceinline__ void private_item(const PagedArgs& a, const Item& it, char* smem) {
    typedef Prod16<T, DH> P_;
    constexpr int TR = 16 * RT, STEP = 32 * NWP;
    // A tile is loaded while the last one is multiplied, but for fp32 heads of 256, whose 256 registers of it would be spilled
    // over the products: 16 sequences x 8 heads, own <= 2048, 444 us ahead and 139 not, 24 x 3 rows behind 1000 keys 213 / 111
    constexpr bool AHEAD = DH * sizeof(T) <= 512;
    const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4, l31 = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), G = a.Hq / a.Hkv;
    const P_ pr(lane);
    char* K = smem + w * (P_::KB + P_::VB);
    char* V = K + P_::KB;
    const int* own = a.table + (long)it.b * a.width;
    for (int rt = it.rt; rt * TR < it.n * G; rt += it.rts) {
        Rows16<T, DH, RT> rows;
        rows.begin(a);
        item_limits(a, it, rt * TR, TR, G, rows.first_limit, rows.last_limit);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            long t;
            int h, limit, at;
            const T* row = item_row<T>(a, it, rt * TR + 16 * i + l15, G, t, h, limit, at);
            rows.begin_row(a, i, row, g, a.slopes && row ? a.slopes[h] : 0.f, limit, at);
        }
        const int end = min(it.k1, rows.last_limit + 1);
        const bool whole = a.dh == DH;
        Stage<P_, T, DH, 32, 1> st(lane, 0);
        int j = it.k0 + 32 * w, odd_first = 0x7FFFFFFF, odd_last = -1;
        unsigned kr = NONE, page = 0;
        if (j < end) {
            kr = slot_of(a, it.hk, page_of(a, own, j + l31, end), j + l31, end);
            page = page_of(a, own, j + STEP + l31, end);
            if (AHEAD) st.load(a, kr, whole);
        }
        while (j < end) {
            if (!AHEAD) st.load(a, kr, whole);
            const unsigned seen = (unsigned)__ballot(kr != NONE);
            if (seen != 0xFFFFFFFFu || !whole) st.clean(a, kr);
            if (j + 31 > rows.first_limit && st.v_finite_only()) {      // (0 x inf must not reach rows that do not see the key)
                odd_first = min(odd_first, j);
                odd_last = j;
            }
            st.store(K, V);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int j0 = j;
            j += STEP;
            if (j < end) {
                kr = slot_of(a, it.hk, page, j + l31, end);
                page = page_of(a, own, j + STEP + l31, end);
                if (AHEAD) st.load(a, kr, whole);
            }
            rows.take(pr, K, V, j0, seen, g);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        for (j = odd_first; j <= odd_last; j += STEP) rows.spoil(a, own, it.hk, j, end, g);
        // join the waves: sums relative to each wave's maximum, through LDS (over the tiles)
        constexpr int LD = DH + 4;
        float* part = reinterpret_cast<float*>(smem);                   // [NWP][TR][LD]
        float* stat = part + NWP * TR * LD;                             // [NWP][TR][2]
        const int nr = min(TR, it.n * G - rt * TR);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int r = 16 * i + l15;
            const float lt = quarter_sum(rows.l[i]);
            if (r < nr) {
                float* dst = part + (w * TR + r) * LD + 4 * g;
#pragma unroll
                for (int d = 0; d < DH / 16; ++d) *reinterpret_cast<f32x4*>(dst + 16 * d) = rows.o[i][d];
                if (g == 0) {
                    stat[(w * TR + r) * 2] = rows.m[i] * rows.c;
                    stat[(w * TR + r) * 2 + 1] = lt;
                }
            }
        }
        __syncthreads();
        const int quads = a.dh / 4;
        for (int e = tid; e < nr * quads; e += 64 * NWP) {
            const int rr = e / quads, d0 = 4 * (e - rr * quads);
            const int rho = rt * TR + rr, r = (unsigned)rho / (unsigned)G;
            const long tt = it.row0 + r;
            if (tt >= a.T) continue;
            float mm = stat[rr * 2], x[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
#pragma unroll
            for (int ww = 1; ww < NWP; ++ww) mm = fmaxf(mm, stat[(ww * TR + rr) * 2]);
#pragma unroll
            for (int ww = 0; ww < NWP; ++ww) {
                const float f = fast_exp2(stat[(ww * TR + rr) * 2] - mm);
                den = fmaf(stat[(ww * TR + rr) * 2 + 1], f, den);
                const f32x4 p = *reinterpret_cast<const f32x4*>(part + (ww * TR + rr) * LD + d0);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = fmaf(p[k], f, x[k]);
            }
            const long orow = tt * a.Hq + it.hk * G + rho - r * G;
            if (it.direct) {
                const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] *= inv;
                put4((T*)a.out + orow * a.dh + d0, x);
            } else {
                const long slot = (long)it.split * a.T * a.Hq + orow;
                put4(a.acc + slot * a.dh + d0, x);
                if (d0 == 0) {
                    a.ml[2 * slot] = mm;
                    a.ml[2 * slot + 1] = den;
                }
            }
        }
        __syncthreads();
    }
}

template <typename T, int DH, int RW, bool ALIBI>
__device__ __forceinline__ void shared_item(const PagedArgs& a, const Item& it, char* smem) {
    typedef Prod<T, DH> P_;
    constexpr int TB = 2 * (P_::KB + P_::VB);                           // one 64-key buffer: K, then V
    constexpr int TR = 32 * RW * NW;
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h5 = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), G = a.Hq / a.Hkv;
    const P_ pr(lane);
    int* odd = reinterpret_cast<int*>(smem + 2 * TB);                   // first and last key of the tiles with V values left out
    const int* own = a.table + (long)it.b * a.width;
    for (int rt = it.rt; rt * TR < it.n * G; rt += it.rts) {
        Rows<T, DH, RW> rows;
        rows.begin(a);
        item_limits(a, it, rt * TR + 32 * RW * w, 32 * RW, G, rows.first_limit, rows.last_limit);
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            long t;
            int h, limit, at;
            const T* row = item_row<T>(a, it, rt * TR + 32 * (RW * w + i) + l31, G, t, h, limit, at);
            rows.begin_row(a, i, row, h5, a.slopes && row ? a.slopes[h] : 0.f, limit, at);
        }
        // the range ends behind the last key any row of the workgroup sees; masked keys begin behind the first row's
        int sure, end;
        item_limits(a, it, rt * TR, TR, G, sure, end);
        end = min(it.k1, end + 1);
        sure = it.prefix ? it.k1 : sure + 1;
        const int ntiles = end > it.k0 ? (end - it.k0 + 63) / 64 : 0;
        if (tid == 0) odd[0] = 0x7FFFFFFF, odd[1] = -1;
        Stage<P_, T, DH, 64, NW> st(lane, w);
        const bool whole = a.dh == DH;
        unsigned long long seen = 0, seen_next = 0;
        // tiles are walked from the last one back (see attn_mfma.hip: with slopes the largest scores come first); at step n
        // tile n is consumed, n + 1 filed in LDS, n + 2 fetched and the page numbers of n + 3 looked up
        auto tile_of = [&](int n) { return it.k0 + (ntiles - 1 - n) * 64; };
        auto lookup = [&](int n) { return page_of(a, own, max(tile_of(n), it.k0) + lane, end); };
        auto slot = [&](int n, unsigned page) { return slot_of(a, it.hk, page, tile_of(n) + lane, end); };
        auto file = [&](int n, unsigned kr) {
            seen_next = __ballot(kr != NONE);
            if (seen_next != ~0ull || !whole) st.clean(a, kr);
            char* B = smem + (n & 1) * TB;
            if (tile_of(n) + 63 >= sure && st.v_finite_only() && lane == 0) {      // (0 x inf must not reach rows that do not see the key)
                atomicMin(&odd[0], tile_of(n));
                atomicMax(&odd[1], tile_of(n) + 63);
            }
            st.store(B, B + 2 * P_::KB);
        };
        unsigned kr = NONE, page = 0;
        __syncthreads();
        if (ntiles > 0) {
            kr = slot(0, lookup(0));
            st.load(a, kr, whole);
            page = lookup(1);
            file(0, kr);
            seen = seen_next;
            if (ntiles > 1) {
                kr = slot(1, page);
                page = lookup(2);
                st.load(a, kr, whole);
            }
        }
        __syncthreads();
        for (int n = 0; n < ntiles; ++n) {
            const int j0 = tile_of(n);
            if (n + 1 < ntiles) file(n + 1, kr);
            if (n + 2 < ntiles) {
                kr = slot(n + 2, page);
                page = lookup(n + 3);
                st.load(a, kr, whole);
            }
            const char* B = smem + (n & 1) * TB;
            if (j0 <= rows.last_limit)                                  // uniform in the wave
                rows.template take<2, ALIBI>(pr, B, B + 2 * P_::KB, j0, seen, h5);
            seen = seen_next;
            __syncthreads();
        }
        for (int j = odd[0]; j <= odd[1]; j += 32) rows.spoil(a, own, it.hk, j, end, h5);
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            long t;
            int h, limit, at;
            if (!item_row<T>(a, it, rt * TR + 32 * (RW * w + i) + l31, G, t, h, limit, at)) continue;
            const float den = half_swap_sum(rows.l[i]);          // (both lanes of a row are here)
            const long orow = t * a.Hq + h;
            const long slot = (long)it.split * a.T * a.Hq + orow;
            const float inv = it.direct ? (den == 0.f ? 0.f : 1.f / den) : 1.f;
#pragma unroll
            for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d0 = 32 * d + 8 * g + 4 * h5;
                    if (d0 >= a.dh) continue;
                    float x[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] = rows.o[i][d][4 * g + k] * inv;
                    if (it.direct) put4((T*)a.out + orow * a.dh + d0, x);
                    else put4(a.acc + slot * a.dh + d0, x);
                }
            if (!it.direct && h5 == 0) {
                a.ml[2 * slot] = rows.m[i] * rows.c;
                a.ml[2 * slot + 1] = den;
            }
        }
        __syncthreads();                                                // (odd, before the next rows)
    }
}

// BODY: 0 / 1 private with 16 / 32 rows, 2 / 3 shared with 32 / 64 rows a wave, 4 private with 16 rows and eight waves (where
// the LDS holds their tiles): few items of long sequences, each of which one workgroup takes without a join.  (Sixteen waves
// for heads of 64: 16 sequences of up to 8000 keys 53 instead of 37 us, 128 registers a lane are too few.)
template <typename T, int DH, int BODY>
constexpr int waves_of() {
    if (DH == 256 && sizeof(T) == 4) return 2;
    return BODY == 4 && 8 * (Prod16<T, DH>::KB + Prod16<T, DH>::VB) <= 136 * 1024 ? 8 : NW;
}
template <typename T, int DH, int BODY>
constexpr int body_smem() {
    if (BODY == 2 || BODY == 3) return 4 * (Prod<T, DH>::KB + Prod<T, DH>::VB) + 16;
    const int nw = waves_of<T, DH, BODY>(), tiles = nw * (Prod16<T, DH>::KB + Prod16<T, DH>::VB);
    const int join = nw * (BODY == 1 ? 32 : 16) * (DH + 4 + 2) * 4;
    return tiles > join ? tiles : join;
}

// rows of no sequence (ragged rows before the first or behind the last one): zeros, 64 workgroups
constexpr int CLEARERS = 64;
template <typename T>
__device__ __forceinline__ void clear_rows(const PagedArgs& a, int wg) {
    const long width = (long)a.Hq * a.dh / 4, first = min(max((long)a.cu[0], 0L), a.T), last = min(max((long)a.cu[a.B], first), a.T);
    const long n = (first + a.T - last) * width;
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (long e = (long)wg * blockDim.x + threadIdx.x; e < n; e += (long)CLEARERS * blockDim.x)
        put4((T*)a.out + 4 * (e < first * width ? e : e + (last - first) * width), zero);
}

// ALIBI: slopes (shared items; the private ones, which wait for memory, add a slope of 0)
template <typename T, int DH, int BODY, bool ALIBI>
__device__ __forceinline__ void run_item(const PagedArgs& a, const Item& it, char* smem) {
    if constexpr (BODY == 2 || BODY == 3) shared_item<T, DH, BODY - 1, ALIBI>(a, it, smem);
    else private_item<T, DH, BODY == 1 ? 2 : 1, waves_of<T, DH, BODY>()>(a, it, smem);
}
// Prefix items first, then own items, in one launch: the former are bound by arithmetic, the latter by memory, and a CU holds
// one of each.
template <typename T, int DH, int BODY_P, int BODY_O, bool ALIBI>
__global__ __launch_bounds__((64 * waves_of<T, DH, BODY_O>()), (BODY_O == 4 ? waves_of<T, DH, BODY_O>() / 4 : DH * sizeof(T) <= 256 ? 2 : 1)) void paged_attn_kernel(const PagedArgs a, int items_p, int items) {
    extern __shared__ __attribute__((aligned(16))) char paged_smem[];
    Item it;
    const int id = blockIdx.x;
    if (id >= items) {
        clear_rows<T>(a, id - items);
        return;
    }
    if (id < items_p) {
        prefix_item(a, id, it);
        if (it.hk < 0) return;                                          // (whole workgroups, before any barrier)
        run_item<T, DH, BODY_P, ALIBI>(a, it, paged_smem);
    } else {
        if (!own_item(a, id - items_p, it)) return;
        run_item<T, DH, BODY_O, ALIBI>(a, it, paged_smem);
    }
}

// The parts of every row joined: 4 values a thread, 2^lq threads a row; where rows are few and parts many, L threads take
// every L-th part and are joined through LDS.
template <typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedArgs a, int lq, int L) {
    __shared__ float part[256][6];
    const int tid = threadIdx.x, q = tid & ((1 << lq) - 1), i = (tid >> lq) & (L - 1), rows = 256 >> lq;      // L, rows: powers of two
    const long row = (long)blockIdx.x * (rows / L) + (tid >> lq) / L;
    const int d0 = 4 * q;
    int b, r, n;
    float x[4] = {0.f, 0.f, 0.f, 0.f}, mm = NEG, den = 0.f;
    const bool real = row < a.T * a.Hq && d0 < a.dh && find_row(a, row / a.Hq, b, r, n);      // (others are cleared by the item launch)
    if (real) {
        const int own = min(max(a.lens[b], 0), a.width * a.page), parts = (a.share ? a.Sp : 0) + own_parts(a, own);
        const long step = a.T * a.Hq;
#pragma unroll 4
        for (int s = i; s < parts; s += L) {
            const long slot = s * step + row;
            const float m = a.ml[2 * slot], l = a.ml[2 * slot + 1];
            const f32x4 p = *reinterpret_cast<const f32x4*>(a.acc + slot * a.dh + d0);
            const float mn = fmaxf(mm, m), f0 = fast_exp2(mm - mn), f1 = fast_exp2(m - mn);
            mm = mn;
            den = den * f0 + l * f1;
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = x[k] * f0 + p[k] * f1;
        }
    }
    if (L > 1) {
        part[tid][0] = mm;
        part[tid][1] = den;
#pragma unroll
        for (int k = 0; k < 4; ++k) part[tid][2 + k] = x[k];
        __syncthreads();
        if (!real || i > 0) return;
        for (int o = 1; o < L; ++o) {
            const float* y = part[tid + (o << lq)];
            const float mn = fmaxf(mm, y[0]), f0 = fast_exp2(mm - mn), f1 = fast_exp2(y[0] - mn);
            mm = mn;
            den = den * f0 + y[1] * f1;
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = x[k] * f0 + y[2 + k] * f1;
        }
    }
    if (!real) return;
    const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] *= inv;
    put4((T*)a.out + row * a.dh + d0, x);
}

// ---- the split: how rows and keys become work items -------------------------------------------------------------------
struct Plan {
    int share, Sp, So, chunk_p, chunk_o, rt_p, rt_o, body_p, body_o;
};

inline long ceil_div(long a, long b) { return (a + b - 1) / b; }

// Into how many parts (1..64) a key range of `keys` keys goes, for `base` items of which `slots` workgroups run at once.
// A part costs 5 us of beginning and end and `key` us a key where the chip is full (`solo` us where it is not); `beside` us
// of other work share the launch.  The time is that of the rounds of parts or of all work spread evenly, whichever is more;
// `row_us` us for writing and reading one part of all rows; the join launch, where one part alone would not need it.
inline int parts_of(long base, long keys, long unit, int slots, double key, double solo, double beside, double row_us, bool join,
                    int& chunk, double& least) {
    int best = 1;
    least = 1e30;
    for (int s = 1; s <= 64; ++s) {
        const long c = ceil_div(ceil_div(keys, s), unit) * unit, n = ceil_div(keys, c);
        if (n != s) continue;
        const long rounds = base * s / slots, rest = base * s % slots;
        const double items = rounds * (5.0 + c * key) + (rest ? 5.0 + c * (rest * 2 <= slots ? solo : key) : 0.0);
        const double even = (double)base * s / slots * (5.0 + c * key) + beside;
        const double cost = (items > even ? items : even) + (s > 1 || !join ? s * row_us : 0.0) + (s > 1 && join ? 4.0 : 0.0);
        if (cost < least) least = cost, best = s, chunk = (int)c;
    }
    return best;
}

Plan plan_of(long T, int B, int Hq, int Hkv, int dh, int P, int max_rows, int max_len, int dtype) {
    max_rows = max_rows < T ? max_rows : (int)T;       // (hints: what is beyond any table or batch says nothing)
    const int room = P < 1 << 30 ? (1 << 30) - P : 1;
    max_len = max_len < room ? max_len : room;
    Plan p = {};
    const long G = Hq / Hkv, rows = (long)max_rows * G;
    const int bytes = dtype == MGX_F32 ? 4 : 2, DH = dh <= 64 ? 64 : dh <= 128 ? 128 : 256;
    // 64 rows a wave share the reads, the page look-ups and the staging of a tile (bf16 heads of 64: prefix items of 3840 rows
    // and 16385 keys: 129 -> 112 us); with 128 sums a row more they would not fit two waves a SIMD
    // Heads of 256, one workgroup a CU: 32 private rows a wave spill (16 sequences x 32 rows: 47 instead of 32 us); shared tiles
    // from 192 rows of a sequence on (16 sequences behind 2000 keys: 64 rows 47 instead of 36 us, 128 52 / 51, 256 84 / 88, long
    // prompts 1.06 / 2.46 ms), not in fp32 (LDS), and not for a prefix, beside own items (256 rows x 8192 keys 165 / 152 us)
    auto body_of = [&](long r) { return DH == 256 ? (r < 192 || bytes == 4 ? 0 : 2) : r <= 16 ? 0 : r <= 32 ? 1 : bytes == 2 && DH == 64 && r >= 192 ? 3 : 2; };
    auto tile_rows = [](int body) { return body == 4 ? 16L : body >= 2 ? 32L * NW * (body - 1) : 16L * (body + 1); };
    const double row_us = T * Hq * (dh + 2.0) * 8.0 / 4.2e6;
    const double key_bytes = 2.0 * dh * bytes;
    // Own lengths are taken to be half of the announced maximum on average (a prefix read once for each sequence comes from
    // L2, at twice the rate: the same half).  Four waves alone stream 25 bytes/ns (fp32, whose products take
    // as long as its loads, 14), the chip 5 bytes/ps.  Shared items: us a key
    // as measured with two workgroups a CU (128 rows of dh 128: 2.6 us for 64 keys); alone a workgroup takes 0.6 of that,
    // beside own items 0.8.
    auto parts = [&](long base, long keys, int body, bool join, double beside, int& chunk, double& us) {
        if (body == 2 || body == 3) {
            const double key = bytes == 4 ? (DH == 64 ? 0.11 : 0.22) : body == 3 ? 0.047 : DH == 64 ? 0.028 : 0.04;
            return parts_of(base, keys, 64, DH == 256 || (bytes == 4 && DH == 128) ? 256 : 512, key, (beside > 0.0 ? 0.8 : 0.6) * key, beside,
                            row_us, join, chunk, us);
        }
        const int groups = body == 4 ? 2 : 1, slots = (DH == 256 ? 256 : 512) / groups;       // (waves_of / 4)
        return parts_of(base, keys, 128 * groups, slots, 0.5 * key_bytes * slots / 5.0e6, (bytes == 4 ? 1.8 : 1.0) * key_bytes / (25.0e3 * groups), beside,
                        row_us, join, chunk, us);
    };
    auto own = [&](Plan& o, int body, long keys, bool join, double& us) {
        o.body_o = body;
        o.rt_o = (int)ceil_div(rows, tile_rows(body));
        const long full = T * G / tile_rows(body) + B, tiles = (long)B * o.rt_o < full ? (long)B * o.rt_o : full;      // ragged rows
        o.So = parts(Hkv * tiles, keys, body, join, 0.0, o.chunk_o, us);
    };
    double us, wide_us = 1e30, apart_us = 1e30;
    own(p, body_of(rows), (long)max_len + P, true, us);
    p.body_p = p.body_o;
    if (p.body_o == 0 && DH * bytes <= 256) {
        Plan w = p;
        own(w, 4, (long)max_len + P, true, wide_us);
        if (wide_us < us) p = w, us = wide_us;
    }
    // Taking the prefix apart packs the rows of all sequences into its tiles and reads it once; it costs the join.  A
    // sequence whose rows fill a tile by themselves has nothing to gain.
    if (P > 0 && B > 1 && T * G < 128L * B) {
        Plan s = p;
        double own_us, prefix_us;
        s.share = 1;
        s.body_p = DH == 256 ? 0 : body_of(T * G);
        int body = body_of(rows);
        if (s.body_p == 1 || body > s.body_p) body = s.body_p;           // (fewer instances: a body of more rows takes less)
        if (s.body_p == 3 && body == 2) body = 3;
        own(s, body, max_len, false, own_us);
        s.rt_p = (int)ceil_div(T * G, tile_rows(s.body_p));
        s.Sp = parts((long)Hkv * s.rt_p, P, s.body_p, false, 0.5 * B * Hkv * (double)max_len * key_bytes / 5.0e6, s.chunk_p, prefix_us);
        apart_us = (prefix_us > own_us ? prefix_us : own_us) + 4.0;
        if (apart_us < us) p = s;
    }
    // Row tiles of a sequence beyond what a launch holds go to the same workgroups in turn (many ragged sequences with no
    // closer bound of their rows than all of them).
    const long most = 0xFFFFFFFFL / (p.body_o == 4 ? 512 : 256) - CLEARERS - (p.share ? ceil_div((long)Hkv * p.Sp, 8) * 8 * p.rt_p : 0);
    const long fit = most / ((long)B * Hkv * p.So);
    if (p.rt_o > fit) p.rt_o = fit > 1 ? (int)fit : 1;
    return p;
}

template <typename T, int DH, int BODY_P, int BODY_O, bool ALIBI>
int launch_items(const PagedArgs& a, long items_p, long items_o, hipStream_t st) {
    constexpr int sp = body_smem<T, DH, BODY_P>(), so = body_smem<T, DH, BODY_O>(), smem = sp > so ? sp : so;
    static_assert(smem <= 160 * 1024, "LDS of a CU");
    const long items = items_p + items_o, grid = items + (a.cu ? CLEARERS : 0);
    MGX_REQUIRE(grid_fits(grid, 64 * waves_of<T, DH, BODY_O>()), MGX_EUNSUPPORTED, "mgx_paged_attn: too many work items");
    if (smem > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(paged_attn_kernel<T, DH, BODY_P, BODY_O, ALIBI>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, smem);
        MGX_REQUIRE(e == hipSuccess, MGX_ELAUNCH, "mgx_paged_attn: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL((paged_attn_kernel<T, DH, BODY_P, BODY_O, ALIBI>), dim3((unsigned)grid), dim3((64 * waves_of<T, DH, BODY_O>())), smem, st, a,
                       (int)items_p, (int)items);
    MGX_CHECK_LAUNCH("paged_attn");
    return MGX_OK;
}

template <typename T, int DH, int BODY_P, bool ALIBI>
int launch_wide(const PagedArgs& a, int body_o, long items_p, long items_o, hipStream_t st) {
    return body_o >= 2   ? launch_items<T, DH, BODY_P, BODY_P, ALIBI>(a, items_p, items_o, st)
           : body_o == 1 ? launch_items<T, DH, BODY_P, 1, ALIBI>(a, items_p, items_o, st)
                         : launch_items<T, DH, BODY_P, 0, ALIBI>(a, items_p, items_o, st);
}

template <typename T>
int launch_join(const PagedArgs& a, hipStream_t st) {
    int lq = 0, L = 1;
    while (4 << lq < a.dh) ++lq;
    const long rows = a.T * a.Hq;
    const int parts = (a.share ? a.Sp : 0) + a.So;
    while ((rows << lq) * L < 65536 && (L << lq) < 256 && 2 * L <= parts) L *= 2;       // a wave on each SIMD
    const long blocks = ceil_div(rows, (256 >> lq) / L);
    MGX_REQUIRE(grid_fits(blocks, 256), MGX_EUNSUPPORTED, "mgx_paged_attn: too many rows");
    hipLaunchKernelGGL(paged_join_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, a, lq, L);
    MGX_CHECK_LAUNCH("paged_join");
    return MGX_OK;
}

template <typename T, int DH>
int launch_paged(const PagedArgs& a, const Plan& p, hipStream_t st) {
    const long ip = p.share ? ceil_div((long)a.Hkv * p.Sp, 8) * 8 * p.rt_p : 0, io = (long)a.B * a.Hkv * p.rt_o * p.So;
    int rc;
    if constexpr (DH == 256) {
        if constexpr (sizeof(T) == 2) {
            if (p.body_p == 2) rc = a.slopes ? launch_items<T, DH, 2, 2, true>(a, ip, io, st) : launch_items<T, DH, 2, 2, false>(a, ip, io, st);
            else rc = launch_items<T, DH, 0, 0, true>(a, ip, io, st);
        } else rc = launch_items<T, DH, 0, 0, true>(a, ip, io, st);
    } else {
        constexpr int TALL = sizeof(T) == 2 && DH == 64 ? 3 : 2;          // (body 3: bf16 heads of 64 alone)
        if (p.body_p == 3) rc = a.slopes ? launch_wide<T, DH, TALL, true>(a, p.body_o, ip, io, st) : launch_wide<T, DH, TALL, false>(a, p.body_o, ip, io, st);
        else if (p.body_p == 2) rc = a.slopes ? launch_wide<T, DH, 2, true>(a, p.body_o, ip, io, st) : launch_wide<T, DH, 2, false>(a, p.body_o, ip, io, st);
        else if (p.body_o == 4) rc = launch_items<T, DH, 4, 4, true>(a, ip, io, st);
        else rc = p.body_p == 1 ? launch_items<T, DH, 1, 1, true>(a, ip, io, st) : launch_items<T, DH, 0, 0, true>(a, ip, io, st);
    }
    return rc || (!p.share && p.So == 1) ? rc : launch_join<T>(a, st);
}

}  // namespace

extern "C" long mgx_paged_attn_workspace_floats(long T, int B, int Hq, int Hkv, int dh, int prefix_len, int max_rows,
                                                int max_len, int dtype) {
    if (T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || dh <= 0 || max_rows <= 0 || max_len <= 0 || prefix_len < 0) return 0;
    const Plan p = plan_of(T, B, Hq, Hkv, dh, prefix_len, max_rows, max_len, dtype);
    if (!p.share && p.So == 1) return 0;
    return (p.So + p.Sp) * T * Hq * (dh + 2L);
}

extern "C" int mgx_paged_attn_plan(long T, int B, int Hq, int Hkv, int dh, int prefix_len, int max_rows, int max_len, int dtype,
                                   int* plan) {
    MGX_REQUIRE(plan, MGX_EINVAL, "mgx_paged_attn_plan: null pointer");
    MGX_REQUIRE(T > 0 && B > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && dh > 0 && dh <= 256 && max_rows > 0 && max_len > 0 &&
                    prefix_len >= 0 && (dtype == MGX_F32 || dtype == MGX_BF16),
                MGX_EINVAL, "mgx_paged_attn_plan: T=%ld B=%d Hq=%d Hkv=%d dh=%d prefix=%d max_rows=%d max_len=%d dtype=%d", T, B, Hq,
                Hkv, dh, prefix_len, max_rows, max_len, dtype);
    const Plan p = plan_of(T, B, Hq, Hkv, dh, prefix_len, max_rows, max_len, dtype);
    const int out[7] = {p.share, p.body_p, p.body_o, p.Sp, p.So, p.chunk_p, p.chunk_o};
    for (int i = 0; i < 7; ++i) plan[i] = out[i];
    return MGX_OK;
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
    MGX_REQUIRE(fabsf(scale) < 0x1p127f, MGX_EINVAL, "mgx_paged_attn: scale %g", scale);        // (times log2 e: an fp32 number)
    MGX_REQUIRE(dtype == MGX_F32 || dtype == MGX_BF16, MGX_EINVAL, "mgx_paged_attn: bad dtype %d", dtype);
    const int N = dtype == MGX_F32 ? 4 : 8;
    MGX_REQUIRE(dh % N == 0 && dh <= 256, MGX_EUNSUPPORTED, "mgx_paged_attn: head dim %d must be a multiple of %d up to 256", dh, N);
    MGX_REQUIRE(q_row_stride >= (long)Hq * dh && q_row_stride % N == 0, MGX_EINVAL, "mgx_paged_attn: row stride %ld", q_row_stride);
    MGX_REQUIRE((((uintptr_t)q | (uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)out) & 15) == 0, MGX_EINVAL,
                "mgx_paged_attn: tensors must be 16-byte aligned");
    MGX_REQUIRE(Hq <= 65535 && T * Hq < (1L << 30), MGX_EUNSUPPORTED, "mgx_paged_attn: T=%ld rows of Hq=%d heads", T, Hq);
    const Plan p = plan_of(T, B, Hq, Hkv, dh, prefix_len, max_rows, max_len, dtype);
    MGX_REQUIRE(workspace || (!p.share && p.So == 1), MGX_EINVAL, "mgx_paged_attn: no workspace");
    MGX_REQUIRE((long)n_pages * Hkv * page < 0xFFFFFFFFL, MGX_EUNSUPPORTED, "mgx_paged_attn: pool of more than 2^32 rows");
    PagedArgs a = {};
    a.q = q, a.kc = kcache, a.vc = vcache, a.out = out;
    a.table = table, a.lens = lens, a.cu = cu_rows, a.prefix = prefix, a.slopes = slopes;
    a.B = B, a.R = R, a.Hq = Hq, a.Hkv = Hkv, a.dh = dh, a.page = page, a.n_pages = n_pages, a.width = width, a.P = prefix_len;
    a.shift = (page & (page - 1)) ? -1 : __builtin_ctz(page);
    a.T = T, a.qs = q_row_stride, a.scale = scale;
    a.share = p.share, a.Sp = p.Sp, a.So = p.So, a.chunk_p = p.chunk_p, a.chunk_o = p.chunk_o;
    a.rt_p = p.rt_p, a.rt_o = p.rt_o;
    hipStream_t st = (hipStream_t)stream;
    a.acc = workspace;
    a.ml = workspace + (p.So + p.Sp) * T * Hq * (long)dh;
    if (dtype == MGX_F32) return dh <= 64 ? launch_paged<float, 64>(a, p, st) : dh <= 128 ? launch_paged<float, 128>(a, p, st) : launch_paged<float, 256>(a, p, st);
    return dh <= 64 ? launch_paged<bf16_t, 64>(a, p, st) : dh <= 128 ? launch_paged<bf16_t, 128>(a, p, st) : launch_paged<bf16_t, 256>(a, p, st);
}
