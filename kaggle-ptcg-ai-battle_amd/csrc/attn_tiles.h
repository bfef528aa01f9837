// Shared by the attention kernels over rows of heads: operand fragments, LDS
// tiles, 32 x 32 products and rows' way out (each includer's own copies, as
// everything is in its unnamed namespace), and the host's checks of layouts.
#pragma once
#include "rowbuf.h"
#include "../../include/ptcg_amd_kernels.h"

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// A: the operator's arguments, with the heads a kv head serves in G and gmagic
// (r / G = umulhi(r, gmagic) for r G < 2^32, G > 1)
template <class A> __device__ __forceinline__ int head_div(const A& a, int r) {
    return a.G == 1 ? r : (int)__umulhi((unsigned)r, a.gmagic);
}
// element offset of flattened query row r of kv head kvh (before the sample's)
template <class A>
__device__ __forceinline__ long row_off(const A& a, const PtcgHeadLayout& l, int kvh, int r) {
    const int qi = head_div(a, r), g = r - qi * a.G;
    return (long)qi * l.sl + (long)(kvh * a.G + g) * l.sh;
}

// Workgroups go to the 8 XCDs in turn; consecutive logical indexes on one XCD
// share a sample's keys in its L2.
__device__ __forceinline__ int xcd_block(int b, int nblk) {
    const int x = b & 7, per = nblk >> 3, rem = nblk & 7;
    return x * per + min(x, rem) + (b >> 3);
}

__device__ __forceinline__ float half_swap(float v) { return __shfl_xor(v, 32, 64); }

// ------------------------------------------------------------- fragments
template <typename T> constexpr int planes() { return sizeof(T) == 4 ? 3 : 1; }

// x[0..8) as bf16 terms
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&t)[3]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        t[0][i] = (__bf16)x[i];
        const float r = x[i] - (float)t[0][i];
        t[1][i] = (__bf16)r;
        t[2][i] = (__bf16)(r - (float)t[1][i]);
    }
}
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&t)[1]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[0][i] = (__bf16)x[i];
}

// c += a b by terms, small ones first
__device__ __forceinline__ void mma(const bf16x8 (&a)[1], const bf16x8 (&b)[1], floatx16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], c, 0, 0, 0);
}
__device__ __forceinline__ void mma(const bf16x8 (&a)[3], const bf16x8 (&b)[3], floatx16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[2], b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], c, 0, 0, 0);
}

// 8 consecutive values as they lie in memory
template <typename T> struct Chunk;
template <> struct Chunk<__bf16> {
    pt_uintx4 w;
    __device__ __forceinline__ void terms(bf16x8 (&t)[1]) const { t[0] = __builtin_bit_cast(bf16x8, w); }
    __device__ __forceinline__ void load(const __bf16* p) { w = *reinterpret_cast<const pt_uintx4*>(p); }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, int off) { w = ld_buf16(rs, off); }
    __device__ __forceinline__ void zero() { w = pt_uintx4{0, 0, 0, 0}; }
    __device__ __forceinline__ void keep(bool ok) { w = ok ? w : pt_uintx4{0, 0, 0, 0}; }
    __device__ __forceinline__ float at(int i) const {
        return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
};
template <> struct Chunk<float> {
    pt_uintx4 w[2];
    __device__ __forceinline__ void terms(bf16x8 (&t)[3]) const {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = at(i);
        split8(x, t);
    }
    __device__ __forceinline__ void load(const float* p) {
        w[0] = *reinterpret_cast<const pt_uintx4*>(p);
        w[1] = *reinterpret_cast<const pt_uintx4*>(p + 4);
    }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, int off) {
        w[0] = ld_buf16(rs, off);
        w[1] = ld_buf16(rs, off + 16);
    }
    __device__ __forceinline__ void zero() { w[0] = w[1] = pt_uintx4{0, 0, 0, 0}; }
    __device__ __forceinline__ void keep(bool ok) {
        w[0] = ok ? w[0] : pt_uintx4{0, 0, 0, 0};
        w[1] = ok ? w[1] : pt_uintx4{0, 0, 0, 0};
    }
    __device__ __forceinline__ float at(int i) const { return __uint_as_float(w[i / 4][i % 4]); }
};

// a lane's row as an operand: chunk c holds dims 16 c + 8 (lane / 32) + 0..7
template <typename T, int DH> struct Row {
    bf16x8 f[DH / 16][planes<T>()];
    // dims past dh, or no row: zeros
    __device__ __forceinline__ void load(const T* row, bool ok, int dh, int h) {
        Chunk<T> x[DH / 16];
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) {
            x[c].zero();
            if (ok && 16 * c + 8 * h < dh) x[c].load(row + 16 * c + 8 * h);
        }
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) x[c].terms(f[c]);
    }
    // the loads end here: in a loop that first uses them the compiler would wait for
    // everything on its way, each time round
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int c = 0; c < DH / 16; ++c)
#pragma unroll
            for (int p = 0; p < planes<T>(); ++p) asm volatile("" : "+v"(f[c][p]));
    }
};

// LDS rows are ST elements apart and chunk c (8 values) of a row lies at
// c ^ swz(row).  Both keep the row reads (16 rows' chunk c) and the transposed
// reads (4 rows' 4 chunks) on 64 different banks.  PAD (128 wide): 64 bytes of
// padding move 4 successive rows to different quarters of the banks and only
// the low two bits of c are turned, so that most of an operand's addresses are
// one register and a constant (the backward has none to spare); without, a tile
// of 128 keys and values leaves room for a second workgroup (a token against
// 50 001 keys: 43 us against 53).
template <int DH, bool PAD> struct Lds {
    static_assert(!PAD || DH == 128, "");
    static constexpr int ST = PAD ? DH + 32 : DH;
    static __device__ __forceinline__ int swz(int row) {
        if constexpr (PAD || DH == 32) return row >> 2 & 3;
        else if constexpr (DH == 64) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
        else return (row & 3) << 2 | (row >> 2 & 3);
    }
    // element offset of chunk 2 c + h of a row
    static __device__ __forceinline__ int chunk_at(int row, int h, int c) {
        if constexpr (PAD) return row * ST + 8 * ((2 * (c & 1) + h) ^ swz(row)) + 32 * (c >> 1);
        else return row * ST + (8 * (h ^ swz(row)) ^ 16 * c);
    }
    // element offset of column group dt (32 columns), chunk ch of it
    static __device__ __forceinline__ int group_at(int row, int ch, int dt) {
        if constexpr (PAD) return row * ST + 8 * (ch ^ swz(row)) + 32 * dt;
        else return row * ST + (8 * (ch ^ swz(row)) ^ 32 * dt);
    }
};

// S = X Y^T of 32 LDS rows of X (PS elements between its planes) against the
// lanes' rows
template <typename T, int DH, bool PAD, int PS>
__device__ __forceinline__ floatx16 mma_rows(const __bf16* xs, const Row<T, DH>& y, int lane) {
    floatx16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int c = 0; c < DH / 16; ++c) {
        bf16x8 a[planes<T>()];
#pragma unroll
        for (int p = 0; p < planes<T>(); ++p)
            a[p] = *reinterpret_cast<const bf16x8*>(xs + p * PS + Lds<DH, PAD>::chunk_at(lane & 31, lane >> 5, c));
        mma(a, y.f[c], s);
    }
    return s;
}

// the same against rows that lie in LDS too (one plane)
template <int DH, bool PAD>
__device__ __forceinline__ floatx16 mma_rows_lds(const __bf16* xs, const __bf16* ys, int lane) {
    floatx16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int c = 0; c < DH / 16; ++c) {
        const int at = Lds<DH, PAD>::chunk_at(lane & 31, lane >> 5, c);
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(xs + at),
                                                    *reinterpret_cast<const bf16x8*>(ys + at), s, 0, 0, 0);
    }
    return s;
}

// c += X^T P over 32 LDS rows of X: c[dt] is columns 32 dt .. of X; P's register
// r stands for row 8 (r / 4) + 4 h + r % 4.  bf16: P is rounded to bf16 for the
// product (by up to 2^-8 of each, as the stored operands are); its fp32 values make
// the softmax's sum.  Gradients are then off by 2.3e-3 to 2.5e-3 (relative L2),
// where rounding an exact one to bf16 gives 1.65e-3; a second term of P for
// samples of up to 64 keys took 1% off that and cost 12% (8 192 x 64 x 97: 277 us
// against 247, by its registers).
template <typename T, int DH, bool PAD, int PS>
__device__ __forceinline__ void mma_tr(const __bf16* xs, const floatx16& p, floatx16 (&c)[DH / 32], int lane) {
    typedef __attribute__((address_space(3))) bf16x4* lds4;
    const int i = lane & 15, r0 = 4 * (lane >> 5) + (i >> 2), ch = 2 * (lane >> 4 & 1) + (i >> 1 & 1);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        float x[8];
        bf16x8 b[planes<T>()];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = p[8 * kb + e];
        split8(x, b);
#pragma unroll
        for (int dt = 0; dt < DH / 32; ++dt) {
            bf16x8 a[planes<T>()];
#pragma unroll
            for (int pl = 0; pl < planes<T>(); ++pl) {
                const __bf16* q = xs + pl * PS + 16 * kb * Lds<DH, PAD>::ST + 4 * (i & 1);
                const lds4 p0 = (lds4)(q + Lds<DH, PAD>::group_at(r0, ch, dt));
                const lds4 p1 = (lds4)(q + Lds<DH, PAD>::group_at(r0 + 8, ch, dt));
                const bf16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(p0);
                const bf16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(p1);
                a[pl] = bf16x8{u[0], u[1], u[2], u[3], w[0], w[1], w[2], w[3]};
            }
            mma(a, b, c[dt]);
        }
    }
}

// A tile of BR rows on its way through registers into LDS: chunks of 8 values,
// thread t takes chunks t, t + NTH, ...  Loads are issued well before the
// barrier that publishes them.
template <typename T, int DH, bool PAD, int BR, int NTH> struct Stage {
    static constexpr int CPR = DH / 8, NCH = BR * CPR / NTH, RPP = NTH / CPR, PS = BR * Lds<DH, PAD>::ST;
    static_assert(BR * CPR % NTH == 0 && NTH % CPR == 0, "whole chunks per thread");
    Chunk<T> r[NCH];
    // byte offset of the thread's first chunk; chunk i is i * RPP rows on
    static __device__ __forceinline__ int first(int ld, int dh, int tid) {
        return tid % CPR * 8 < dh ? tid / CPR * ld + tid % CPR * 8 * (int)sizeof(T) : PT_NOWHERE;
    }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, int off, int ld) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) r[i].load(rs, off + i * (RPP * ld));
    }
    // rows of the flattened query matrix of kv head kvh, from row0; the last
    // row stands in for rows past it
    template <class A>
    __device__ __forceinline__ void load_q(const A& a, const PtcgHeadLayout& l, const T* base, int kvh, int row0,
                                           int len, int tid) {
        const int col = min(tid % CPR * 8, a.dh - 8);
#pragma unroll
        for (int i = 0; i < NCH; ++i)
            r[i].load(base + row_off(a, l, kvh, min(row0 + tid / CPR + i * RPP, len - 1)) + col);
    }
    __device__ __forceinline__ void put(__bf16* s, int tid, int i, bool ok) const {
        const int row = tid / CPR + i * RPP;
        bf16x8 t[planes<T>()];
        r[i].terms(t);
#pragma unroll
        for (int p = 0; p < planes<T>(); ++p)
            *reinterpret_cast<pt_uintx4*>(s + p * PS + row * Lds<DH, PAD>::ST + 8 * (tid % CPR ^ Lds<DH, PAD>::swz(row))) =
                ok ? __builtin_bit_cast(pt_uintx4, t[p]) : pt_uintx4{0, 0, 0, 0};
    }
    __device__ __forceinline__ void store(__bf16* s, int tid) const {
#pragma unroll
        for (int i = 0; i < NCH; ++i) put(s, tid, i, true);
    }
    // rows below `rows`, columns below dh; zeros besides
    __device__ __forceinline__ void store_q(__bf16* s, int tid, int rows, int dh) const {
#pragma unroll
        for (int i = 0; i < NCH; ++i) put(s, tid, i, tid / CPR + i * RPP < rows && tid % CPR * 8 < dh);
    }
};

// a lane's 4 consecutive output values
__device__ __forceinline__ void st4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ void st4(__bf16* p, float a, float b, float c, float d) {
    *reinterpret_cast<bf16x4*>(p) = bf16x4{(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
}
// row (lane % 32) of a transposed accumulator, times f
template <typename T, int DH>
__device__ __forceinline__ void store_row(T* row, const floatx16 (&o)[DH / 32], float f, int dh, int h) {
#pragma unroll
    for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int d = 32 * dt + 8 * b + 4 * h;
            if (d < dh)
                st4(row + d, o[dt][4 * b] * f, o[dt][4 * b + 1] * f, o[dt][4 * b + 2] * f, o[dt][4 * b + 3] * f);
        }
}

// A wave's 32 rows of a transposed accumulator to memory, times each row's f, by
// way of LDS (ws: 32 padded rows): whole rows of 16 bytes a lane instead of 8
// bytes here and there.
template <typename T, int DH> struct Out {
    static constexpr int E = 16 / sizeof(T), CPR = DH / E, ST = DH + E, WAVE = 32 * ST;
    static __device__ __forceinline__ void turn(T* ws, const floatx16 (&o)[DH / 32], float f, int lane) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        store_row<T, DH>(ws + (lane & 31) * ST, o, f, DH, lane >> 5);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    // rows r0 .. of kv head kvh, those below `rows`
    template <class A>
    static __device__ __forceinline__ void query_rows(const A& a, const PtcgHeadLayout& l, T* out, int kvh, int r0,
                                                      int rows, const floatx16 (&o)[DH / 32], float f, T* ws,
                                                      int lane) {
        turn(ws, o, f, lane);
#pragma unroll
        for (int i = 0; i < 32 * CPR / 64; ++i) {
            const int c = i * 64 + lane, row = c / CPR, col = c % CPR * E;
            if (r0 + row < rows && col < a.dh)
                *reinterpret_cast<pt_uintx4*>(out + row_off(a, l, kvh, r0 + row) + col) =
                    *reinterpret_cast<const pt_uintx4*>(ws + row * ST + col);
        }
    }
    // key rows key0 .. of a matrix at base, row stride sl
    static __device__ __forceinline__ void key_rows(T* base, long sl, int key0, int keys, int dh,
                                                    const floatx16 (&o)[DH / 32], float f, T* ws, int lane) {
        turn(ws, o, f, lane);
#pragma unroll
        for (int i = 0; i < 32 * CPR / 64; ++i) {
            const int c = i * 64 + lane, row = c / CPR, col = c % CPR * E;
            if (key0 + row < keys && col < dh)
                *reinterpret_cast<pt_uintx4*>(base + (long)(key0 + row) * sl + col) =
                    *reinterpret_cast<const pt_uintx4*>(ws + row * ST + col);
        }
    }
};

constexpr size_t max3(size_t a, size_t b, size_t c) { return a > b ? (a > c ? a : c) : (b > c ? b : c); }
// elements (bf16) of a tile of BR rows
template <typename T, int DH, bool PAD, int BR> constexpr int tile_elems() {
    return planes<T>() * BR * Lds<DH, PAD>::ST;
}

// ------------------------------------------------------------------- host
int cu_count() {
    int dev = 0, cu = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cu, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cu <= 0)
        return 256;
    return cu;
}

bool layout_ok(const PtcgHeadLayout& l, int e) {
    return l.sn >= 0 && l.sl >= 0 && l.sh >= 0 && l.sn % e == 0 && l.sl % e == 0 && l.sh % e == 0;
}

// Whether no two elements of an output share an address.  Packed, the host knows
// no row count (rows only bounds a sample's): a row's heads have to lie within the
// row stride, or else two rows, the fewest that a batch of more than one row may
// hold, within the head stride.
bool layout_apart(const PtcgHeadLayout& l, bool packed, int n, int rows, int heads, int dh) {
    if (n <= 0 || rows <= 0) return true;       // no element
    if (packed) {
        const bool many = n > 1 || rows > 1;
        if (heads <= 1) return !many || l.sl >= dh;
        if (l.sh < dh) return false;
        if (!many) return true;
        return l.sh <= l.sl ? l.sh <= (l.sl - dh) / (heads - 1) : l.sl >= dh && l.sl <= l.sh - dh;
    }
    int64_t st[3] = {n > 1 ? l.sn : -1, rows > 1 ? l.sl : -1, heads > 1 ? l.sh : -1};
    int64_t ex[3] = {n, rows, heads};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (st[j] < st[i]) {
                const int64_t t = st[i]; st[i] = st[j]; st[j] = t;
                const int64_t u = ex[i]; ex[i] = ex[j]; ex[j] = u;
            }
    int64_t span = dh;
    for (int i = 0; i < 3; ++i) {
        if (st[i] < 0) continue;
        if (st[i] < span || (ex[i] > 1 && st[i] > (1LL << 50) / (ex[i] - 1))) return false;
        span = st[i] * (ex[i] - 1) + span;
    }
    return true;
}

// A pool of pages and its table; strides multiples of e elements.
int check_pages(const PtcgPages& g, int n, int kv_heads, int dh, int e, const char* who) {
    PT_REQUIRE(g.pages >= 0 && g.page >= 1 && g.per_seq >= 0, "%s: %d pages of %d rows, %d a sequence", who, g.pages,
               g.page, g.per_seq);
    PT_REQUIRE((int64_t)g.page * g.per_seq < (1LL << 30), "%s: sequences of 2^30 rows or more", who);
    PT_REQUIRE(n <= 1 || g.table_sn >= g.per_seq, "%s: page tables overlap", who);
    PT_REQUIRE(layout_ok(g.k, e) && layout_ok(g.v, e), "%s: page strides must be non-negative multiples of %d elements",
               who, e);
    PT_REQUIRE(n == 0 || g.per_seq == 0 || g.table, "%s: no page table", who);
    PT_REQUIRE(g.pages == 0 || (g.kp && g.vp), "%s: no pool", who);
    return PTCG_OK;
}

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename K> int lds_attr(K kernel, size_t bytes) {
    if (bytes > 64 * 1024)
        PT_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return PTCG_OK;
}

}  // namespace
