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
#include "common.h"
#include "../../include/ptcg_amd_kernels.h"

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int GRP = 32;

// 8 consecutive values of a row; VEC: 16 B (fp32: 2 x 16 B) aligned and whole,
// else single loads of those below `left`
template <bool VEC> __device__ __forceinline__ void ld8(const float* p, int left, float (&x)[8]) {
    if constexpr (VEC) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < left ? p[i] : 0.f;
}
template <bool VEC> __device__ __forceinline__ void ld8(const __bf16* p, int left, float (&x)[8]) {
    if constexpr (VEC) {
        const bf16x8 a = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
    } else
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < left ? (float)p[i] : 0.f;
}
template <bool VEC> __device__ __forceinline__ void st8(float* p, int left, const float (&x)[8]) {
    if constexpr (VEC) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = x[i];
}
template <bool VEC> __device__ __forceinline__ void st8(__bf16* p, int left, const float (&x)[8]) {
    if constexpr (VEC) {
        bf16x8 a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = (__bf16)x[i];
        *reinterpret_cast<bf16x8*>(p) = a;
    } else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = (__bf16)x[i];
}
template <bool VEC> __device__ __forceinline__ uint2 ldq8(const uint8_t* p, int left) {
    if constexpr (VEC) return *reinterpret_cast<const uint2*>(p);
    uint2 r = make_uint2(0u, 0u);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < left) (i < 4 ? r.x : r.y) |= (unsigned)p[i] << (8 * (i & 3));
    return r;
}
template <bool VEC> __device__ __forceinline__ void stq8(uint8_t* p, int left, uint2 v) {
    if constexpr (VEC) *reinterpret_cast<uint2*>(p) = v;
    else
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

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ x, long ldx, long rows, int d, int cpr,
        uint8_t* __restrict__ q, long ldq, uint8_t* __restrict__ sc, long lds) {
    const Piece p = piece_of(rows, d, cpr);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    if (p.ok) ld8<VEC>(x + p.row * ldx + p.col, p.left, v);
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
    stq8<VEC>(q + p.row * ldq + p.col, p.left, r);
    if ((p.col & (GRP - 1)) == 0) sc[p.row * lds + p.col / GRP] = (uint8_t)(e + 127);
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void unpack_kernel(const uint8_t* __restrict__ q, long ldq,
        const uint8_t* __restrict__ sc, long lds, long rows, int d, int cpr, T* __restrict__ x, long ldx) {
    const Piece p = piece_of(rows, d, cpr);
    if (!p.ok) return;
    float v[8];
    values8(ldq8<VEC>(q + p.row * ldq + p.col, p.left), scale_of((int)sc[p.row * lds + p.col / GRP] - 127), v);
    st8<VEC>(x + p.row * ldx + p.col, p.left, v);
}

// z8 -> dz = dy gelu'(z8) and, where asked, a = gelu(z8): the byte stands in for
// the two activations a GELU layer's backward reads
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void gelu_bwd_kernel(const uint8_t* __restrict__ q, long ldq,
        const uint8_t* __restrict__ sc, long lds, long rows, int d, int cpr, const T* dy, long lddy, T* dz,
        long lddz, T* __restrict__ act, long lda) {
    const Piece p = piece_of(rows, d, cpr);
    if (!p.ok) return;
    float g[8], z[8], a[8];
    ld8<VEC>(dy + p.row * lddy + p.col, p.left, g);
    values8(ldq8<VEC>(q + p.row * ldq + p.col, p.left), scale_of((int)sc[p.row * lds + p.col / GRP] - 127), z);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float gd;
        pt_gelu_both(z[i], a[i], gd);
        g[i] *= gd;
    }
    st8<VEC>(dz + p.row * lddz + p.col, p.left, g);
    if (act) st8<VEC>(act + p.row * lda + p.col, p.left, a);
}

// ------------------------------------------------------- weight gradient
// dW (n, k) = dY^T x8 over the rows, db = column sums of dY.  Both operands
// have the reduction as their outer dimension, so both fragments come from
// row-major LDS tiles by ds_read_b64_tr_b16 (4 rows of 16 columns to a lane's
// 4 values); x8 becomes bf16 on the way into LDS, exactly.  fp32 dY is split
// into three bf16 terms (8 bits each, by truncation, together exact above
// 2^-102): 3 products against an x8 that needs no splitting, where two fp32
// operands take 6.
// A workgroup of 4 waves owns a TM x TN tile of dW and a range of the rows
// (splits leave partial tiles, added in split order by dw_reduce_kernel);
// splits also make the partial column sums.
constexpr int TM = 128, TN = 128, TK = 32, PADB = 16;

struct DwArgs {
    const void* dy; long lddy;
    const uint8_t* q; long ldq;
    const uint8_t* sc; long lds;
    float* dw; float* db;
    float* part;          // [splits][n][k], then [splits][n] column sums
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

// VEC: rows of dy and q are 16 / 8 B aligned with n, k multiples of 8
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dw_kernel(const DwArgs g) {
    constexpr int NP = sizeof(T) == 4 ? 3 : 1;          // bf16 terms of dY
    constexpr int SA = TM + PADB, SB = TN + PADB;
    extern __shared__ __align__(16) char smem[];
    __bf16* As = reinterpret_cast<__bf16*>(smem);       // [NP][TK][SA]
    __bf16* Bs = As + NP * TK * SA;                     // [TK][SB]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int b = blockIdx.x;
    const int it = b % g.tn; b /= g.tn;
    const int ot = b % g.tm, sp = b / g.tm;
    const int o0 = ot * TM, i0 = it * TN;
    const int r0 = sp * g.chunk, r1 = min(g.rows, r0 + g.chunk);
    const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const T* dy = static_cast<const T*>(g.dy);
    const bool sums = it == 0;

    // staging: thread owns column piece pc (8 columns) of rows pr, pr + 16
    const int pc = (tid & 15) * 8, pr = tid >> 4;
    float a[2][8], csum[8];
    uint2 xb[2];
    int xe[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) csum[i] = 0.f;
    auto fetch = [&](int r) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = r + pr + 16 * u;
            const bool ok = row < r1;
            const int la = ok ? g.n - (o0 + pc) : 0, lb = ok ? g.k - (i0 + pc) : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) a[u][i] = 0.f;
            xb[u] = make_uint2(0u, 0u);
            xe[u] = 127;
            if (la > 0) ld8<VEC>(dy + (long)row * g.lddy + o0 + pc, la, a[u]);
            if (lb > 0) {
                xb[u] = ldq8<VEC>(g.q + (long)row * g.ldq + i0 + pc, lb);
                xe[u] = g.sc[(long)row * g.lds + (i0 + pc) / GRP];
            }
        }
    };
    floatx16 acc[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[m][n][e] = 0.f;
    if (r0 < r1) fetch(r0);
    for (int r = r0; r < r1; r += TK) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = pr + 16 * u;
            bf16x8 h[NP];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v = a[u][i];
                if (sums) csum[i] += v;
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
            for (int p = 0; p < NP; ++p) *reinterpret_cast<bf16x8*>(As + (p * TK + row) * SA + pc) = h[p];
            const float w = scale_of(xe[u] - 127);
            const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(xb[u].x, w, false);
            const bf16x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(xb[u].x, w, true);
            const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(xb[u].y, w, false);
            const bf16x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(xb[u].y, w, true);
            *reinterpret_cast<bf16x8*>(Bs + row * SB + pc) = bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
        }
        __syncthreads();
        if (r + TK < r1) fetch(r + TK);
#pragma unroll
        for (int kk = 0; kk < TK; kk += 16) {
            bf16x8 bf[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) bf[n] = frag_tr(Bs + kk * SB + wn + 32 * n, SB, lane);
#pragma unroll
            for (int p = NP - 1; p >= 0; --p)     // small terms first
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const bf16x8 af = frag_tr(As + (p * TK + kk) * SA + wm + 32 * m, SA, lane);
#pragma unroll
                    for (int n = 0; n < 2; ++n)
                        acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af, bf[n], acc[m][n], 0, 0, 0);
                }
        }
    }
    float* out = g.splits > 1 ? g.part + (long)sp * g.n * g.k : g.dw;
#pragma unroll
    for (int m = 0; m < 2; ++m)
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
    if (!sums || !g.db) return;
    // column sums: the 16 threads of a column piece add in row order
    __syncthreads();
    float* cs = reinterpret_cast<float*>(smem);     // [16][TM]
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[pr * TM + pc + i] = csum[i];
    __syncthreads();
    if (tid < TM && o0 + tid < g.n) {
        float s = 0.f;
        for (int i = 0; i < 16; ++i) s += cs[i * TM + tid];
        if (g.splits > 1) g.part[(long)g.splits * g.n * g.k + (long)sp * g.n + o0 + tid] = s;
        else g.db[o0 + tid] = s;
    }
}

__global__ __launch_bounds__(256) void dw_reduce_kernel(const DwArgs g) {
    const long nk = (long)g.n * g.k, i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i < nk) {
        float s = 0.f;
#pragma unroll 8
        for (int p = 0; p < g.splits; ++p) s += g.part[p * nk + i];
        g.dw[i] = s;
    } else if (g.db && i < nk + g.n) {
        const float* c = g.part + g.splits * nk + (i - nk);
        float s = 0.f;
        for (int p = 0; p < g.splits; ++p) s += c[(long)p * g.n];
        g.db[i - nk] = s;
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

// splits of the rows: two workgroups per CU, at least 8 steps each
struct DwPlan { int tm, tn, splits, chunk; };
DwPlan dw_plan(int rows, int k, int n) {
    DwPlan p;
    p.tm = pt_cdiv(n, TM);
    p.tn = pt_cdiv(k, TN);
    const long tiles = (long)p.tm * p.tn;
    long sp = (2 * cu_count()) / tiles;
    const long most = rows / (8 * TK);
    if (sp > most) sp = most;
    if (sp < 1) sp = 1;
    p.chunk = rows > 0 ? pt_cdiv(pt_cdiv(rows, sp), TK) * TK : TK;
    p.splits = rows > 0 ? pt_cdiv(rows, p.chunk) : 1;
    return p;
}

bool al(const void* p, int a) { return ((uintptr_t)p & (a - 1)) == 0; }

int check_rows(const char* who, int rows, int d, int64_t ldq, int64_t lds) {
    PT_REQUIRE(rows >= 0 && d >= 1, "%s: rows=%d d=%d", who, rows, d);
    PT_REQUIRE(ldq >= d && lds >= pt_cdiv(d, GRP), "%s: row strides %lld (codes), %lld (scales) below d=%d", who,
               (long long)ldq, (long long)lds, d);
    PT_REQUIRE((long)rows * pt_cdiv(d, GRP) < (1LL << 36), "%s: %d rows of %d are too many", who, rows, d);
    return PTCG_OK;
}
int grid_for(int rows, int d, int* cpr) {
    *cpr = pt_cdiv(d, GRP) * (GRP / 8);
    return pt_cdiv((long)rows * *cpr, 256);
}
// whether 8 values can move as 16 bytes of T (fp32: twice)
template <typename T> bool vec8(const void* p, long ld) { return al(p, 16) && ld % (16 / (int)sizeof(T)) == 0; }
bool vecq(const void* q, long ldq, int d) { return al(q, 8) && ldq % 8 == 0 && d % 8 == 0; }

template <typename T>
int pack(const void* x, long ldx, int rows, int d, uint8_t* q, long ldq, uint8_t* sc, long lds, hipStream_t s) {
    int cpr;
    const int grid = grid_for(rows, d, &cpr);
    auto kern = vecq(q, ldq, d) && vec8<T>(x, ldx) ? pack_kernel<T, true> : pack_kernel<T, false>;
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
    auto kern = vecq(q, ldq, d) && vec8<T>(x, ldx) ? unpack_kernel<T, true> : unpack_kernel<T, false>;
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
    const bool vec = vecq(q, ldq, d) && vec8<T>(dy, lddy) && vec8<T>(dz, lddz) && (!act || vec8<T>(act, lda));
    auto kern = vec ? gelu_bwd_kernel<T, true> : gelu_bwd_kernel<T, false>;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(256), 0, s, q, ldq, sc, lds, (long)rows, d, cpr,
                       static_cast<const T*>(dy), lddy, static_cast<T*>(dz), lddz, static_cast<T*>(act), lda);
    PT_LAUNCH_CHECK();
    return PTCG_OK;
}
template <typename T> int dw(const DwArgs& g, const DwPlan& p, hipStream_t s) {
    constexpr int NP = sizeof(T) == 4 ? 3 : 1;
    constexpr size_t lds = (size_t)(NP * TK * (TM + PADB) + TK * (TN + PADB)) * 2;
    static_assert(lds >= 16 * TM * 4 && lds <= 64 * 1024, "the column sums reuse the tiles");
    const bool vec = vecq(g.q, g.ldq, g.k) && vec8<T>(g.dy, g.lddy) && g.n % 8 == 0;
    auto kern = vec ? dw_kernel<T, true> : dw_kernel<T, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)((long)p.tm * p.tn * p.splits)), dim3(256), lds, s, g);
    PT_LAUNCH_CHECK();
    if (p.splits > 1) {
        hipLaunchKernelGGL(dw_reduce_kernel, dim3(pt_cdiv((long)g.n * g.k + g.n, 256)), dim3(256), 0, s, g);
        PT_LAUNCH_CHECK();
    }
    return PTCG_OK;
}

int check_dw(const char* who, int rows, int in, int out) {
    PT_REQUIRE(rows >= 0 && rows < (1 << 30) && in >= 1 && out >= 1, "%s: rows=%d in=%d out=%d", who, rows, in, out);
    PT_REQUIRE((long)in * out < (1LL << 36) && (long)pt_cdiv(in, TN) * pt_cdiv(out, TM) < (1LL << 22),
               "%s: in=%d out=%d are too large", who, in, out);
    return PTCG_OK;
}
int64_t dw_need(int rows, int in, int out) {
    const DwPlan p = dw_plan(rows, in, out);
    return p.splits > 1 ? (int64_t)p.splits * ((int64_t)in * out + out) * 4 : 0;
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
    return bf16 ? gelu<__bf16>(q, ldq, scales, lds, rows, d, dy, lddy, dz, lddz, act, lda, (hipStream_t)stream)
                : gelu<float>(q, ldq, scales, lds, rows, d, dy, lddy, dz, lddz, act, lda, (hipStream_t)stream);
}

extern "C" int64_t ptcg_kernel_ckpt8_dw_ws_bytes(int rows, int in, int out, int bf16) {
    if (check_dw("ckpt8_dw_ws_bytes", rows, in, out) != PTCG_OK) return -1;
    return dw_need(rows, in, out);
}

extern "C" int ptcg_kernel_ckpt8_dw(int rows, int in, int out, const void* dY, int64_t lddy, int bf16,
                                    const uint8_t* q, int64_t ldq, const uint8_t* scales, int64_t lds, float* dW,
                                    float* db, void* workspace, int64_t workspace_bytes, void* stream) {
    PT_TRY(check_dw("ckpt8_dw", rows, in, out));
    PT_TRY(check_rows("ckpt8_dw", rows, in, ldq, lds));
    PT_REQUIRE(lddy >= out, "ckpt8_dw: row stride %lld below out=%d", (long long)lddy, out);
    PT_REQUIRE(dW && (rows == 0 || (dY && q && scales)), "ckpt8_dw: null buffer");
    const int64_t need = dw_need(rows, in, out);
    PT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && al(workspace, 16)),
               "ckpt8_dw: workspace of %lld bytes, need %lld (16 B aligned)", (long long)workspace_bytes,
               (long long)need);
    const DwPlan p = dw_plan(rows, in, out);
    DwArgs g{};
    g.dy = dY; g.lddy = lddy; g.q = q; g.ldq = ldq; g.sc = scales; g.lds = lds;
    g.dw = dW; g.db = db; g.part = static_cast<float*>(workspace);
    g.rows = rows; g.k = in; g.n = out; g.splits = p.splits; g.chunk = p.chunk; g.tm = p.tm; g.tn = p.tn;
    return bf16 ? dw<__bf16>(g, p, (hipStream_t)stream) : dw<float>(g, p, (hipStream_t)stream);
}
