// Activation checkpoints in 8 bits and their use in the backward pass.
//
// A row's values go in groups of 32 with a scale 2^e and are kept as e4m3:
//   e = the least integer with max |x| <= 448 2^e, held to [-110, 119],
//   q = e4m3(x 2^-e) to nearest even,  x8 = q 2^e.
// A value costs 1 + 1/32 bytes.  The scale being a power of two, x 2^-e, q 2^e
// and x8 as bf16 are exact, so the backward's products on bf16 matrix
// instructions see x8 itself: the rounding to e4m3 (half a step: 2^-4 of the
// value, or 2^-10 2^e for small ones) is the only one.  e >= -110 keeps every x8
// a normal bf16; e <= 119 a finite fp32 (values past 448 2^119 saturate).  NaN
// and infinities are kept as NaN and leave the group's scale to the others.
#include "rowbuf.h"
#include <type_traits>
#include "../../include/ptcg_amd_kernels.h"

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int GRP = 32;

// 8 consecutive values of a row, as one access of any alignment (the hardware
// takes dword and wider accesses at any byte), or, past `left` of a row's last
// piece (TAIL), singly
template <typename T, int N> struct Packed { T v[N]; } __attribute__((packed));
template <bool TAIL> __device__ __forceinline__ void ld8(const float* p, int left, float (&x)[8]) {
    if (!TAIL || left >= 8) {
        const Packed<float, 8> a = *reinterpret_cast<const Packed<float, 8>*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = a.v[i];
    } else
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < left ? p[i] : 0.f;
}
template <bool TAIL> __device__ __forceinline__ void ld8(const __bf16* p, int left, float (&x)[8]) {
    if (!TAIL || left >= 8) {
        const Packed<unsigned, 4> a = *reinterpret_cast<const Packed<unsigned, 4>*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(i % 2 ? a.v[i / 2] & 0xffff0000u : a.v[i / 2] << 16);
    } else
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < left ? (float)p[i] : 0.f;
}
template <bool TAIL> __device__ __forceinline__ void st8(float* p, int left, const float (&x)[8]) {
    if (!TAIL || left >= 8) {
        Packed<float, 8> a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a.v[i] = x[i];
        *reinterpret_cast<Packed<float, 8>*>(p) = a;
    } else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = x[i];
}
template <bool TAIL> __device__ __forceinline__ void st8(__bf16* p, int left, const float (&x)[8]) {
    if (!TAIL || left >= 8) {
        Packed<unsigned, 4> a;
#pragma unroll
        for (int i = 0; i < 4; ++i) a.v[i] = __builtin_bit_cast(unsigned, bf16x2{(__bf16)x[2 * i], (__bf16)x[2 * i + 1]});
        *reinterpret_cast<Packed<unsigned, 4>*>(p) = a;
    } else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = (__bf16)x[i];
}
template <bool TAIL> __device__ __forceinline__ uint2 ldq8(const uint8_t* p, int left) {
    if (!TAIL || left >= 8) {
        const Packed<unsigned, 2> a = *reinterpret_cast<const Packed<unsigned, 2>*>(p);
        return make_uint2(a.v[0], a.v[1]);
    }
    uint2 r = make_uint2(0u, 0u);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < left) (i < 4 ? r.x : r.y) |= (unsigned)p[i] << (8 * (i & 3));
    return r;
}
template <bool TAIL> __device__ __forceinline__ void stq8(uint8_t* p, int left, uint2 v) {
    if (!TAIL || left >= 8) {
        Packed<unsigned, 2> a;
        a.v[0] = v.x;
        a.v[1] = v.y;
        *reinterpret_cast<Packed<unsigned, 2>*>(p) = a;
    } else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = (uint8_t)((i < 4 ? v.x : v.y) >> (8 * (i & 3)));
}

__device__ __forceinline__ float scale_of(int e) { return __int_as_float((e + 127) << 23); }   // 2^e, |e| < 127

// 8 codes as the values they stand for
__device__ __forceinline__ void values8(uint2 q, float w, float (&x)[8]) {
    const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8(q.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(q.x, true);
    const floatx2 c = __builtin_amdgcn_cvt_pk_f32_fp8(q.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(q.y, true);
    x[0] = a[0] * w; x[1] = a[1] * w; x[2] = b[0] * w; x[3] = b[1] * w;
    x[4] = c[0] * w; x[5] = c[1] * w; x[6] = d[0] * w; x[7] = d[1] * w;
}

// Elementwise kernels: a thread owns 8 consecutive values of a row (4 threads a
// group); a workgroup 256 consecutive ones of the rows laid end to end, `cpr`
// pieces a row (a multiple of 4, so that a group's threads are lanes of a quad).
struct Piece { long row; int col, left; bool ok; };
__device__ __forceinline__ Piece piece_of(long rows, int d, int cpr) {
    const long first = (long)blockIdx.x * 256, row0 = first / cpr;
    const unsigned p = (unsigned)(first - row0 * cpr) + threadIdx.x, dr = p / (unsigned)cpr;
    Piece r;
    r.row = row0 + dr;
    r.col = (int)(p - dr * (unsigned)cpr) * 8;
    r.left = d - r.col;
    r.ok = r.row < rows && r.left > 0;
    return r;
}

template <typename T, bool TAIL>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ x, long ldx, long rows, int d, int cpr,
        uint8_t* __restrict__ q, long ldq, uint8_t* __restrict__ sc, long lds) {
    const Piece p = piece_of(rows, d, cpr);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    if (p.ok) ld8<TAIL>(x + p.row * ldx + p.col, p.left, v);
    unsigned top = 0;    // bits of max |x| over finite values: integer order is float order
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned b = __float_as_uint(v[i]) & 0x7fffffffu;
        top = max(top, b < 0x7f800000u ? b : 0u);
    }
    top = max(top, (unsigned)__shfl_xor((int)top, 1, 64));
    top = max(top, (unsigned)__shfl_xor((int)top, 2, 64));
    // 448 = 1.75 2^8
    int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(-110, min(119, e));
    const float w = scale_of(-e);
    uint2 r;
    unsigned h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = v[i] * w;
        h[i] = __float_as_uint(fabsf(y) > 448.f && fabsf(v[i]) < INFINITY ? copysignf(448.f, y)
                               : fabsf(v[i]) < INFINITY ? y : NAN);
    }
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(h[0]), __uint_as_float(h[1]), lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(h[2]), __uint_as_float(h[3]), lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(h[4]), __uint_as_float(h[5]), hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(h[6]), __uint_as_float(h[7]), hi, true);
    r.x = (unsigned)lo; r.y = (unsigned)hi;
    if (!p.ok) return;
    stq8<TAIL>(q + p.row * ldq + p.col, p.left, r);
    if ((p.col & (GRP - 1)) == 0) sc[p.row * lds + p.col / GRP] = (uint8_t)(e + 127);
}

template <typename T, bool TAIL>
__global__ __launch_bounds__(256) void unpack_kernel(const uint8_t* __restrict__ q, long ldq,
        const uint8_t* __restrict__ sc, long lds, long rows, int d, int cpr, T* __restrict__ x, long ldx) {
    const Piece p = piece_of(rows, d, cpr);
    if (!p.ok) return;
    float v[8];
    values8(ldq8<TAIL>(q + p.row * ldq + p.col, p.left), scale_of((int)sc[p.row * lds + p.col / GRP] - 127), v);
    st8<TAIL>(x + p.row * ldx + p.col, p.left, v);
}

// z8 -> dz = dy gelu'(z8) and, where asked, a = gelu(z8): the byte stands in for
// the two activations a GELU layer's backward reads
template <typename T, bool TAIL>
__global__ __launch_bounds__(256) void gelu_bwd_kernel(const uint8_t* __restrict__ q, long ldq,
        const uint8_t* __restrict__ sc, long lds, long rows, int d, int cpr, const T* dy, long lddy, T* dz,
        long lddz, T* __restrict__ act, long lda) {
    const Piece p = piece_of(rows, d, cpr);
    if (!p.ok) return;
    float g[8], z[8], a[8];
    ld8<TAIL>(dy + p.row * lddy + p.col, p.left, g);
    values8(ldq8<TAIL>(q + p.row * ldq + p.col, p.left), scale_of((int)sc[p.row * lds + p.col / GRP] - 127), z);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float gd;
        pt_gelu_both(z[i], a[i], gd);
        g[i] *= gd;
    }
    st8<TAIL>(dz + p.row * lddz + p.col, p.left, g);
    if (act) st8<TAIL>(act + p.row * lda + p.col, p.left, a);
}

// ------------------------------------------------------- weight gradient
// dW (n, k) = dY^T x8 over the rows, db = column sums of dY.  Both operands
// have the reduction as their outer dimension, so both fragments come from
// row-major LDS tiles by ds_read_b64_tr_b16 (4 rows of 16 columns to a lane's
// 4 values); x8 becomes bf16 on the way into LDS, exactly.  fp32 dY is split
// into three bf16 terms (8 bits each, by truncation, together exact above
// 2^-102): 3 products against an x8 that needs no splitting, where two fp32
// operands take 6.
// A workgroup owns a TM x TN tile of dW and a range of the rows (splits leave
// partial tiles, added in split order by dw_reduce_kernel); its waves own
// TM / 2 x 64 each.  Steps of TK rows go through registers, two steps ahead of
// their use, into the half of a double buffer that the products left a barrier
// ago.  Splits also make the partial column sums.
constexpr int TK = 32, PADB = 16;

struct DwArgs {
    const void* dy; long lddy;
    const uint8_t* q; long ldq;
    const uint8_t* sc; long lds;
    float* dw; float* db;
    float* part;          // [splits][pstride]: dW (n, k), then the n column sums
    long pstride;
    int rows, k, n, splits, chunk, tn, tm;
};

__device__ __forceinline__ bf16x8 frag_tr(const __bf16* s, int st, int lane) {
    typedef __attribute__((address_space(3))) bf16x4* lds4;
    // rows 8 (lane / 32) + 0..7 of 16, columns lane % 32
    const int i = lane & 15;
    const __bf16* a = s + (8 * (lane >> 5) + (i >> 2)) * st + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)a);
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(a + 4 * st));
    return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

__device__ __forceinline__ float trunc_bf16(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }

// 8 values of dY as they were loaded, 8 codes.  Bounds hold per dword: a row
// whose bytes are no whole dwords loses its last ones where the descriptor
// ends, so the matrix's last rows come singly then (ONE).
template <typename T> struct Raw8;
template <> struct Raw8<float> {
    pt_uintx4 w[2];
    template <bool ONE> __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, int off) {
        w[0] = ld_buf16(rs, off);
        w[1] = ld_buf16(rs, off + 16);
    }
    __device__ __forceinline__ float at(int i) const { return __uint_as_float(w[i / 4][i % 4]); }
};
template <> struct Raw8<__bf16> {
    pt_uintx4 w;
    template <bool ONE> __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, int off) {
        if constexpr (!ONE) w = ld_buf16(rs, off);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = ld_buf2(rs, off + 4 * i) | ld_buf2(rs, off + 4 * i + 2) << 16;
    }
    __device__ __forceinline__ float at(int i) const {
        return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
};
template <bool ONE> __device__ __forceinline__ pt_uintx2 codes8(__amdgpu_buffer_rsrc_t rs, int off) {
    if constexpr (!ONE) return ld_buf8(rs, off);
    pt_uintx2 r = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i / 4] |= ld_buf1(rs, off + i) << (8 * (i % 4));
    return r;
}

template <typename T, int TM, int TN> struct DwCfg {
    static constexpr int NP = sizeof(T) == 4 ? 3 : 1;          // bf16 terms of dY
    static constexpr int NTH = 2 * TN;                         // 2 x TN / 64 waves
    static constexpr int SA = TM + PADB, SB = TN + PADB;
    static constexpr int BUF = NP * TK * SA + TK * SB;         // one half of the double buffer
    static constexpr int RA = NTH / (TM / 8), RB = NTH / (TN / 8);   // rows of a staging pass
    static constexpr int PA = TK / RA, PB = TK / RB;
    static constexpr size_t LDS = 2 * (size_t)BUF * 2;
    static_assert(TK % RA == 0 && TK % RB == 0 && LDS >= (size_t)RA * TM * 4, "staging passes, column sums");
};

// WHOLE: rows of dy and q are whole dwords
template <typename T, bool WHOLE, int TM, int TN>
__global__ __launch_bounds__(2 * TN) void dw_kernel(const DwArgs g) {
    typedef DwCfg<T, TM, TN> C;
    constexpr int NP = C::NP, SA = C::SA, SB = C::SB, MT = TM / 64;
    extern __shared__ __align__(16) char smem[];
    __bf16* lds = reinterpret_cast<__bf16*>(smem);      // [2] of A [NP][TK][SA], B [TK][SB]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // consecutive tiles of one row range on one XCD: its L2 serves their shared operands
    int b;
    {
        const int nblk = gridDim.x, x = blockIdx.x & 7, per = nblk >> 3, rem = nblk & 7;
        b = x * per + min(x, rem) + (blockIdx.x >> 3);
    }
    const int it = b % g.tn; b /= g.tn;
    const int ot = b % g.tm, sp = b / g.tm;
    const int o0 = ot * TM, i0 = it * TN;
    const int r0 = sp * g.chunk, r1 = min(g.rows, r0 + g.chunk);
    const int wm = (wave & 1) * (TM / 2), wn = (wave >> 1) * 64;
    const bool sums = it == 0 && g.db;

    // staging: a thread owns 8 columns of rows ra + RA u of dY and rb + RB u of
    // x8.  What it reads of a row past column n (k) reaches only outputs that
    // are not stored; rows past the range come as zeros.
    const int ca = tid % (TM / 8) * 8, ra = tid / (TM / 8);
    const int cb = tid % (TN / 8) * 8, rb = tid / (TN / 8);
    const RowBuf ya = {static_cast<const char*>(g.dy) + (long)o0 * sizeof(T), (int)g.lddy * (int)sizeof(T),
                       (g.n - o0) * (int)sizeof(T)};
    const RowBuf xq = {reinterpret_cast<const char*>(g.q) + i0, (int)g.ldq, g.k - i0};
    const RowBuf xs = {reinterpret_cast<const char*>(g.sc) + i0 / GRP, (int)g.lds, (g.k - i0 + GRP - 1) / GRP};
    int offa[C::PA], offq[C::PB], offs[C::PB];
#pragma unroll
    for (int u = 0; u < C::PA; ++u)
        offa[u] = o0 + ca < g.n ? (ra + C::RA * u) * ya.ld + ca * (int)sizeof(T) : PT_NOWHERE;
#pragma unroll
    for (int u = 0; u < C::PB; ++u) {
        offq[u] = i0 + cb < g.k ? (rb + C::RB * u) * xq.ld + cb : PT_NOWHERE;
        offs[u] = i0 + cb < g.k ? (rb + C::RB * u) * xs.ld + cb / GRP : PT_NOWHERE;
    }
    struct Set { Raw8<T> a[C::PA]; pt_uintx2 xb[C::PB]; unsigned xe[C::PB]; } set[2];
    float csum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) csum[i] = 0.f;
    // inlined by order: as a call, the sets lie in scratch (29 777 x 634 x 64 fp32:
    // 688 us against 32)
    auto fetch = [&](int r, Set& f) __attribute__((always_inline)) {
        // three rows more than the step has: the last dword of its last row is inside,
        // for rows of one byte too
        const auto ry = ya.rows(r, r1, TK + 3), rq = xq.rows(r, r1, TK + 3), rs = xs.rows(r, r1, TK + 3);
        if (WHOLE || r + TK + 2 < r1) {
#pragma unroll
            for (int u = 0; u < C::PA; ++u) f.a[u].template load<false>(ry, offa[u]);
#pragma unroll
            for (int u = 0; u < C::PB; ++u) f.xb[u] = codes8<false>(rq, offq[u]);
        } else {
#pragma unroll
            for (int u = 0; u < C::PA; ++u) f.a[u].template load<true>(ry, offa[u]);
#pragma unroll
            for (int u = 0; u < C::PB; ++u) f.xb[u] = codes8<true>(rq, offq[u]);
        }
#pragma unroll
        for (int u = 0; u < C::PB; ++u) f.xe[u] = ld_buf1(rs, offs[u]);
    };
    auto put = [&](auto sum, __bf16* As, const Set& f) __attribute__((always_inline)) {
        __bf16* Bs = As + NP * TK * SA;
#pragma unroll
        for (int u = 0; u < C::PA; ++u) {
            bf16x8 h[NP];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v = f.a[u].at(i);
                if constexpr (sum) csum[i] += v;
                if constexpr (NP == 1) h[0][i] = (__bf16)v;
                else {
                    const float t0 = trunc_bf16(v);
                    v -= t0;
                    const float t1 = trunc_bf16(v);
                    h[0][i] = (__bf16)t0;
                    h[1][i] = (__bf16)t1;
                    h[2][i] = (__bf16)(v - t1);
                }
            }
#pragma unroll
            for (int p = 0; p < NP; ++p) *reinterpret_cast<bf16x8*>(As + (p * TK + ra + C::RA * u) * SA + ca) = h[p];
        }
#pragma unroll
        for (int u = 0; u < C::PB; ++u) {
            const float w = scale_of((int)f.xe[u] - 127);   // rows past the range: 0 times 0
            const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.xb[u][0], w, false);
            const bf16x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.xb[u][0], w, true);
            const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.xb[u][1], w, false);
            const bf16x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.xb[u][1], w, true);
            *reinterpret_cast<bf16x8*>(Bs + (rb + C::RB * u) * SB + cb) =
                bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
        }
    };
    floatx16 acc[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[m][n][e] = 0.f;
    // One step: the products of buffer `cur`, with step `set` going into buffer
    // `nxt` and step r on its way into `set` between them: products, LDS traffic,
    // loads and the operands' conversion take turns in one wave's instruction
    // stream (the groups below), where phase by phase the products would stand
    // still in the others (all waves meet at the same barrier).
    auto step = [&](auto sum, const __bf16* cur, __bf16* nxt, Set& f, int r) __attribute__((always_inline)) {
        const __bf16* Bs = cur + NP * TK * SA;
        bf16x8 af[TK / 16][NP][MT], bf[TK / 16][2];
        auto read = [&](int k) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < 2; ++n) bf[k][n] = frag_tr(Bs + 16 * k * SB + wn + 32 * n, SB, lane);
#pragma unroll
            for (int p = NP - 1; p >= 0; --p)
#pragma unroll
                for (int m = 0; m < MT; ++m) af[k][p][m] = frag_tr(cur + (p * TK + 16 * k) * SA + wm + 32 * m, SA, lane);
        };
        read(0);
        put(sum, nxt, f);
        fetch(r, f);
        read(1);
#pragma unroll
        for (int k = 0; k < TK / 16; ++k)
#pragma unroll
            for (int p = NP - 1; p >= 0; --p)     // small terms first
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
                        acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[k][p][m], bf[k][n], acc[m][n], 0, 0, 0);
        constexpr int FR = 2 * (2 + NP * MT), MF = NP * MT * 2;   // LDS reads and products of 16 rows
        __builtin_amdgcn_sched_group_barrier(0x100, FR, 0);
#pragma unroll
        for (int i = 0; i < MF; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, (FR + MF - 1) / MF, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
        }
#pragma unroll
        for (int i = 0; i < MF; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        }
        __syncthreads();
    };
    // step t sits in buffer t % 2 while steps t + 1 and t + 2 are on their way
    auto walk = [&](auto sum) __attribute__((always_inline)) {
        fetch(r0, set[0]);
        put(sum, lds, set[0]);
        fetch(r0 + TK, set[1]);
        fetch(r0 + 2 * TK, set[0]);
        __syncthreads();
        for (int r = r0; r < r1; r += 2 * TK) {
            step(sum, lds, lds + C::BUF, set[1], r + 3 * TK);
            step(sum, lds + C::BUF, lds, set[0], r + 4 * TK);   // past the range: zeros
        }
    };
    if (r0 < r1) {
        if (sums) walk(std::true_type());
        else walk(std::false_type());
    }
    float* out = g.splits > 1 ? g.part + sp * g.pstride : g.dw;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int col = i0 + wn + 32 * n + (lane & 31);
            if (col >= g.k) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = o0 + wm + 32 * m + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
                if (row < g.n) out[(long)row * g.k + col] = acc[m][n][e];
            }
        }
    if (!sums) return;
    // column sums: the RA threads of a column piece add in row order
    float* cs = reinterpret_cast<float*>(smem);     // [RA][TM]; the loop ended in a barrier
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[ra * TM + ca + i] = csum[i];
    __syncthreads();
    for (int c = tid; c < TM && o0 + c < g.n; c += C::NTH) {
        float s = 0.f;
        for (int i = 0; i < C::RA; ++i) s += cs[i * TM + c];
        if (g.splits > 1) g.part[sp * g.pstride + (long)g.n * g.k + o0 + c] = s;
        else g.db[o0 + c] = s;
    }
}

// Adds the splits' partials (dW, then db): a thread takes 4 consecutive values
// of every SG-th split, SG groups of a workgroup meet in LDS, in order.  Few
// outputs with many splits need the groups (one thread walking 200 splits of a
// 128 x 128 dW waits for its loads in line: 60 000 x 128 x 128 bf16 62 us, both
// launches, against 17.5 with 16 groups).
template <int SG> __global__ __launch_bounds__(256) void dw_reduce_kernel(const DwArgs g) {
    __shared__ float4 sh[256];
    constexpr int CW = 256 / SG;
    const int c = threadIdx.x % CW, grp = threadIdx.x / CW;
    const long i = ((long)blockIdx.x * CW + c) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < g.pstride) {
#pragma unroll 8
        for (int p = grp; p < g.splits; p += SG) {
            const float4 x = *reinterpret_cast<const float4*>(g.part + p * g.pstride + i);
            s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
        }
    }
    if constexpr (SG > 1) {
        sh[threadIdx.x] = s;
        __syncthreads();
        if (grp > 0) return;
#pragma unroll
        for (int k = 1; k < SG; ++k) {
            const float4 x = sh[k * CW + c];
            s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
        }
    }
    const long nk = (long)g.n * g.k;
    if (i + 4 <= nk && ((uintptr_t)g.dw & 15) == 0) {
        *reinterpret_cast<float4*>(g.dw + i) = s;
        return;
    }
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (i + e < nk) g.dw[i + e] = v[e];
        else if (g.db && i + e < nk + g.n) g.db[i + e - nk] = v[e];
    }
}

// ------------------------------------------------------------------- host
int cu_count() {
    int dev = 0, cu = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cu, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cu <= 0)
        return 256;
    return cu;
}

// Tiles and splits of the rows.  One workgroup per CU (a second one shares its
// matrix cores and doubles the partials: 37 391 x 256 x 1 024 fp32 77 us with
// one, 95 with two).  128 x 256 tiles read the narrower operand half as often as
// 128 x 128 ones (62 us against 72, 20 000 x 1 024 x 1 024 bf16); a dW of few
// tiles takes 128 x 128, whose partials are half as many bytes (60 000 x 256 x
// 256 bf16: 40 us against 50).  256 x 256 in bf16 (16 products of 12 LDS reads a
// step) gains 14% of the products and costs another 33 MB of partials: from
// rows * in * out = 4e10 on (65 539 x 4 096 x 1 024: 537 us against 625;
// 20 000 x 1 024 x 1 024: 70 against 63).  In fp32 its accumulators leave too
// few registers for the three terms; in bf16, rows that are no whole dwords make it
// spill 38 a lane.  At least 4 steps a split.
struct DwPlan { int big_m, big_n, tm, tn, splits, chunk; long pstride; };
DwPlan dw_plan(int rows, int k, int n, int bf16) {
    DwPlan p;
    p.big_n = k > 128 && (long)n * k > 256 * 256;
    p.big_m = bf16 && p.big_n && n > 128 && (double)rows * n * k > 4e10;
    p.tm = pt_cdiv(n, p.big_m ? 256 : 128);
    p.tn = pt_cdiv(k, p.big_n ? 256 : 128);
    const long tiles = (long)p.tm * p.tn;
    long sp = cu_count() / tiles;
    const long most = rows / (4 * TK);
    if (sp > most) sp = most;
    if (sp < 1) sp = 1;
    p.chunk = rows > 0 ? pt_cdiv(pt_cdiv(rows, sp), TK) * TK : TK;
    p.splits = rows > 0 ? pt_cdiv(rows, p.chunk) : 1;
    p.pstride = ((long)n * k + n + 3) / 4 * 4;
    return p;
}

bool al(const void* p, int a) { return ((uintptr_t)p & (a - 1)) == 0; }

int check_rows(const char* who, int rows, int d, int64_t ldq, int64_t lds) {
    PT_REQUIRE(rows >= 0 && d >= 1, "%s: rows=%d d=%d", who, rows, d);
    PT_REQUIRE(ldq >= d && lds >= pt_cdiv(d, GRP), "%s: row strides %lld (codes), %lld (scales) below d=%d", who,
               (long long)ldq, (long long)lds, d);
    // a launch holds fewer than 2^32 threads, four a group
    PT_REQUIRE((long)rows * ((d + (long)GRP - 1) / GRP) < (1LL << 30), "%s: %d rows of %d are too many", who, rows, d);
    return PTCG_OK;
}
int grid_for(int rows, int d, int* cpr) {
    *cpr = pt_cdiv(d, GRP) * (GRP / 8);
    return pt_cdiv((long)rows * *cpr, 256);
}

template <typename T>
int pack(const void* x, long ldx, int rows, int d, uint8_t* q, long ldq, uint8_t* sc, long lds, hipStream_t s) {
    int cpr;
    const int grid = grid_for(rows, d, &cpr);
    auto kern = d % 8 ? pack_kernel<T, true> : pack_kernel<T, false>;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(256), 0, s, static_cast<const T*>(x), ldx, (long)rows, d, cpr, q, ldq,
                       sc, lds);
    PT_LAUNCH_CHECK();
    return PTCG_OK;
}
template <typename T>
int unpack(const uint8_t* q, long ldq, const uint8_t* sc, long lds, int rows, int d, void* x, long ldx,
           hipStream_t s) {
    int cpr;
    const int grid = grid_for(rows, d, &cpr);
    auto kern = d % 8 ? unpack_kernel<T, true> : unpack_kernel<T, false>;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(256), 0, s, q, ldq, sc, lds, (long)rows, d, cpr, static_cast<T*>(x),
                       ldx);
    PT_LAUNCH_CHECK();
    return PTCG_OK;
}
template <typename T>
int gelu(const uint8_t* q, long ldq, const uint8_t* sc, long lds, int rows, int d, const void* dy, long lddy,
         void* dz, long lddz, void* act, long lda, hipStream_t s) {
    int cpr;
    const int grid = grid_for(rows, d, &cpr);
    auto kern = d % 8 ? gelu_bwd_kernel<T, true> : gelu_bwd_kernel<T, false>;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(256), 0, s, q, ldq, sc, lds, (long)rows, d, cpr,
                       static_cast<const T*>(dy), lddy, static_cast<T*>(dz), lddz, static_cast<T*>(act), lda);
    PT_LAUNCH_CHECK();
    return PTCG_OK;
}
template <typename T, bool WHOLE, int TM, int TN> int launch_dw(const DwArgs& g, hipStream_t s) {
    typedef DwCfg<T, TM, TN> C;
    auto kern = dw_kernel<T, WHOLE, TM, TN>;
    if (C::LDS > 64 * 1024)
        PT_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)C::LDS));
    hipLaunchKernelGGL(kern, dim3((unsigned)((long)g.tm * g.tn * g.splits)), dim3(C::NTH), C::LDS, s, g);
    PT_LAUNCH_CHECK();
    return PTCG_OK;
}
template <typename T, bool WHOLE> int dw_tiles(const DwArgs& g, const DwPlan& p, hipStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (p.big_m) return launch_dw<T, WHOLE, 256, 256>(g, s);
    return p.big_n ? launch_dw<T, WHOLE, 128, 256>(g, s) : launch_dw<T, WHOLE, 128, 128>(g, s);
}
template <typename T> int dw(const DwArgs& g, const DwPlan& p, hipStream_t s) {
    const bool whole = g.k % 4 == 0 && (sizeof(T) == 4 || g.n % 2 == 0);
    PT_TRY(whole ? (dw_tiles<T, true>(g, p, s)) : (dw_tiles<T, false>(g, p, s)));
    if (p.splits > 1) {
        // enough workgroups for two per CU or so
        const long quads = g.pstride / 4;
        if (quads >= 512 * 256 || g.splits < 8)
            hipLaunchKernelGGL(dw_reduce_kernel<1>, dim3(pt_cdiv(quads, 256)), dim3(256), 0, s, g);
        else if (quads >= 128 * 256 || g.splits < 32)
            hipLaunchKernelGGL(dw_reduce_kernel<4>, dim3(pt_cdiv(quads, 64)), dim3(256), 0, s, g);
        else
            hipLaunchKernelGGL(dw_reduce_kernel<16>, dim3(pt_cdiv(quads, 16)), dim3(256), 0, s, g);
        PT_LAUNCH_CHECK();
    }
    return PTCG_OK;
}

int check_dw(const char* who, int rows, int in, int out) {
    PT_REQUIRE(rows >= 0 && rows < (1 << 30) && in >= 1 && out >= 1, "%s: rows=%d in=%d out=%d", who, rows, in, out);
    PT_REQUIRE((long)in * out < (1LL << 36) && (long)pt_cdiv(in, 128) * pt_cdiv(out, 128) < (1LL << 22),
               "%s: in=%d out=%d are too large", who, in, out);
    return PTCG_OK;
}
int64_t dw_need(int rows, int in, int out, int bf16) {
    const DwPlan p = dw_plan(rows, in, out, bf16);
    return p.splits > 1 ? (int64_t)p.splits * p.pstride * 4 : 0;
}

}  // namespace

extern "C" int ptcg_kernel_ckpt8_pack(const void* x, int64_t ldx, int bf16, int rows, int d, uint8_t* q, int64_t ldq,
                                      uint8_t* scales, int64_t lds, void* stream) {
    PT_TRY(check_rows("ckpt8_pack", rows, d, ldq, lds));
    PT_REQUIRE(ldx >= d, "ckpt8_pack: row stride %lld below d=%d", (long long)ldx, d);
    if (rows == 0) return PTCG_OK;
    PT_REQUIRE(x && q && scales, "ckpt8_pack: null buffer");
    return bf16 ? pack<__bf16>(x, ldx, rows, d, q, ldq, scales, lds, (hipStream_t)stream)
                : pack<float>(x, ldx, rows, d, q, ldq, scales, lds, (hipStream_t)stream);
}

extern "C" int ptcg_kernel_ckpt8_unpack(const uint8_t* q, int64_t ldq, const uint8_t* scales, int64_t lds, int rows,
                                        int d, void* x, int64_t ldx, int bf16, void* stream) {
    PT_TRY(check_rows("ckpt8_unpack", rows, d, ldq, lds));
    PT_REQUIRE(ldx >= d, "ckpt8_unpack: row stride %lld below d=%d", (long long)ldx, d);
    if (rows == 0) return PTCG_OK;
    PT_REQUIRE(x && q && scales, "ckpt8_unpack: null buffer");
    return bf16 ? unpack<__bf16>(q, ldq, scales, lds, rows, d, x, ldx, (hipStream_t)stream)
                : unpack<float>(q, ldq, scales, lds, rows, d, x, ldx, (hipStream_t)stream);
}

extern "C" int ptcg_kernel_ckpt8_gelu_bwd(const uint8_t* q, int64_t ldq, const uint8_t* scales, int64_t lds, int rows,
                                          int d, const void* dy, int64_t lddy, void* dz, int64_t lddz, void* act,
                                          int64_t lda, int bf16, void* stream) {
    PT_TRY(check_rows("ckpt8_gelu_bwd", rows, d, ldq, lds));
    PT_REQUIRE(lddy >= d && lddz >= d && (!act || lda >= d), "ckpt8_gelu_bwd: a row stride is below d=%d", d);
    if (rows == 0) return PTCG_OK;
    PT_REQUIRE(q && scales && dy && dz, "ckpt8_gelu_bwd: null buffer");
    PT_REQUIRE(dz != dy || lddz == lddy, "ckpt8_gelu_bwd: dz over dy takes its row stride, %lld, not %lld",
               (long long)lddy, (long long)lddz);
    PT_REQUIRE(!act || (act != dy && act != dz), "ckpt8_gelu_bwd: act is dy or dz");
    return bf16 ? gelu<__bf16>(q, ldq, scales, lds, rows, d, dy, lddy, dz, lddz, act, lda, (hipStream_t)stream)
                : gelu<float>(q, ldq, scales, lds, rows, d, dy, lddy, dz, lddz, act, lda, (hipStream_t)stream);
}

extern "C" int64_t ptcg_kernel_ckpt8_dw_ws_bytes(int rows, int in, int out, int bf16) {
    if (check_dw("ckpt8_dw_ws_bytes", rows, in, out) != PTCG_OK) return -1;
    return dw_need(rows, in, out, bf16);
}

extern "C" int ptcg_kernel_ckpt8_dw(int rows, int in, int out, const void* dY, int64_t lddy, int bf16,
                                    const uint8_t* q, int64_t ldq, const uint8_t* scales, int64_t lds, float* dW,
                                    float* db, void* workspace, int64_t workspace_bytes, void* stream) {
    PT_TRY(check_dw("ckpt8_dw", rows, in, out));
    PT_TRY(check_rows("ckpt8_dw", rows, in, ldq, lds));
    PT_REQUIRE(lddy >= out, "ckpt8_dw: row stride %lld below out=%d", (long long)lddy, out);
    PT_REQUIRE(lddy < (1 << 23) && ldq < (1 << 23) && lds < (1 << 23), "ckpt8_dw: a row stride is 2^23 or more");
    PT_REQUIRE(dW && (rows == 0 || (dY && q && scales)), "ckpt8_dw: null buffer");
    const int64_t need = dw_need(rows, in, out, bf16);
    PT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && al(workspace, 16)),
               "ckpt8_dw: workspace of %lld bytes, need %lld (16 B aligned)", (long long)workspace_bytes,
               (long long)need);
    const DwPlan p = dw_plan(rows, in, out, bf16);
    DwArgs g{};
    g.dy = dY; g.lddy = lddy; g.q = q; g.ldq = ldq; g.sc = scales; g.lds = lds;
    g.dw = dW; g.db = db; g.part = static_cast<float*>(workspace);
    g.rows = rows; g.k = in; g.n = out; g.splits = p.splits; g.chunk = p.chunk; g.tm = p.tm; g.tn = p.tn;
    g.pstride = p.pstride;
    return bf16 ? dw<__bf16>(g, p, (hipStream_t)stream) : dw<float>(g, p, (hipStream_t)stream);
}
