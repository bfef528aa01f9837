// Norms of queries and keys for each head with the position rotation in the same
// pass, its gradient, and the same on the way into a cache of pages.
//
//   n = x w / sqrt(mean x^2 + eps),  y = R(p) n  (R on the first rot elements)
// Backward, r = 1 / sqrt(mean x^2 + eps), R^T the turn by the negative angle:
//   dn = R^T dy,  dw = sum dn x r,  dx = r (dn w - x r^2 mean(dn w x)).
//
// All of it is bound by its bytes.  A head's row is a group of LP lanes (a power
// of two); a lane holds VW pairs: of the turning part the pairs' two elements, of
// the rest 2 VW neighbours, so every access is a vector of VW elements, 16 bytes
// where widths, strides and addresses let it.  The statistics are a sum over the
// group.  An angle's cosine and sine serve a group for all the heads of its row
// that it walks (hg groups a row share them): no table is read.  512 x 97 rows of 4 + 4
// heads of 64 in fp32: forward 35 us (5.8 TB/s, read and written), backward 58 (5.2); 65 539 rows
// of 8 + 2 heads of 128 in bf16: 70 (4.8) and 113 (4.5); 134 MB of new rows into pages and as much
// written: 58 (4.6).
//
// Angles: position times frequency and the reduction to a quarter turn are 64
// bit (five instructions a pair and row); a 32-bit product would lose 2^-24 of
// the angle, a tenth of a radian at a position of a million.  What is left, at
// most pi / 4, goes through the Taylor polynomials of sine and cosine to y^9 and
// y^10, whose first terms left out are below 2^-28 there.
#include "attn_tiles.h"

#include <math.h>

#include <type_traits>

namespace {

constexpr int NTH = 256;

struct RopeArgs {
    int n, l, H, KV, dh, rot;
    int rows;
    int lps, hgs;                 // log2 of the lanes a head and the groups a row
    PtcgHeadLayout q, k, v, qo, ko;
    const float *wq, *wk;
    float eps, mag, inv_dh;
    const double* freq;
    const int* pos;
    // into the cache
    const int *q_off, *len;
    PtcgPages pg;
};

template <typename T, int VW> struct VecOf { typedef T type __attribute__((ext_vector_type(VW))); };
template <typename T> struct VecOf<T, 1> { typedef T type; };

// a lane's 2 VW elements of a head, as they lie in memory
template <typename T, int VW> struct Pairs {
    typedef typename VecOf<T, VW>::type V;
    V a, b;
    __device__ __forceinline__ void load(const T* p, int oa, int ob) {
        a = *reinterpret_cast<const V*>(p + oa);
        b = *reinterpret_cast<const V*>(p + ob);
    }
    __device__ __forceinline__ void store(T* p, int oa, int ob) const {
        *reinterpret_cast<V*>(p + oa) = a;
        *reinterpret_cast<V*>(p + ob) = b;
    }
    __device__ __forceinline__ void get(float (&x)[2 * VW]) const {
        if constexpr (VW == 1) {
            x[0] = (float)a;
            x[1] = (float)b;
        } else {
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                x[e] = (float)a[e];
                x[VW + e] = (float)b[e];
            }
        }
    }
    __device__ __forceinline__ void set(const float (&x)[2 * VW]) {
        if constexpr (VW == 1) {
            a = (T)x[0];
            b = (T)x[1];
        } else {
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                a[e] = (T)x[e];
                b[e] = (T)x[VW + e];
            }
        }
    }
};

// mag cos and mag sin of p freq (freq in radians)
__device__ __forceinline__ void cos_sin(double p, double freq, float mag, float& c, float& s) {
    const double t = p * freq * 0.15915494309189535;          // turns
    const double q = rint(4.0 * t);
    const float y = (float)((t - 0.25 * q) * 6.283185307179586);
    const float z = y * y;
    const float sn = fmaf(y * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), y);
    const float cs = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24),
                                  -0.5f), 1.f);
    const int k = (int)(q - 4.0 * floor(0.25 * q));           // quarter turns
    c = mag * (k & 1 ? (k & 2 ? sn : -sn) : (k & 2 ? -cs : cs));
    s = mag * (k & 1 ? (k & 2 ? -cs : cs) : (k & 2 ? -sn : sn));
}

// a lane's place in a head: offsets of its two vectors, and whether they turn
template <int VW, bool INTER> struct Unit {
    int oa, ob, first;     // first: its first pair
    bool live, turns;
    __device__ __forceinline__ Unit(int u, int dh, int rot) {
        live = u * 2 * VW < dh;
        turns = u * 2 * VW < rot;
        first = u * VW;
        if (turns && !INTER) {
            oa = u * VW;
            ob = oa + rot / 2;
        } else {
            oa = u * 2 * VW;
            ob = oa + VW;
        }
    }
    // pair e's elements in x
    static __device__ __forceinline__ int lo(int e) { return INTER ? 2 * e : e; }
    static __device__ __forceinline__ int hi(int e) { return INTER ? 2 * e + 1 : VW + e; }
};

template <int VW, bool INTER>
__device__ __forceinline__ void angles(const RopeArgs& a, const Unit<VW, INTER>& u, int p, float (&c)[VW],
                                       float (&s)[VW]) {
#pragma unroll
    for (int e = 0; e < VW; ++e) {
        c[e] = 1.f;
        s[e] = 0.f;
        if (u.turns) cos_sin(p, a.freq[u.first + e], a.mag, c[e], s[e]);
    }
}
// x turned by the angles (sign 1) or back (sign -1)
template <int VW, bool INTER>
__device__ __forceinline__ void turn(float (&x)[2 * VW], const float (&c)[VW], const float (&s)[VW], bool turns,
                                     float sign) {
    typedef Unit<VW, INTER> U;
    if (!turns) return;
#pragma unroll
    for (int e = 0; e < VW; ++e) {
        const float x0 = x[U::lo(e)], x1 = x[U::hi(e)], sn = sign * s[e];
        x[U::lo(e)] = x0 * c[e] - x1 * sn;
        x[U::hi(e)] = x0 * sn + x1 * c[e];
    }
}

// sum over a group of 2^lps lanes; up to 16 of them within the vector unit
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
    return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float group_sum(float v, int lps) {
    if (lps > 0) v = dpp_add<0xb1>(v);      // neighbours
    if (lps > 1) v = dpp_add<0x4e>(v);      // pairs of a quad
    if (lps > 2) v = dpp_add<0x141>(v);     // the other quad of 8, mirrored: its lanes are alike by now
    if (lps > 3) v = dpp_add<0x140>(v);     // the other 8 of 16
    for (int o = 16; o < 1 << lps; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// 1 / sqrt(v) to an ulp, of values whose root the instruction flushes too
__device__ __forceinline__ float rsqrt_of(float v) {
    const bool tiny = v < 1.1754944e-38f;
    const float r = __builtin_amdgcn_rsqf(tiny ? v * 0x1p64f : v);
    return tiny ? r * 0x1p32f : r;
}

// Which sample a row of packed matrices belongs to: the last whose first row is
// not past it (samples without rows are passed over).  -1: none, or past the
// rows a sample may have.
__device__ __forceinline__ int packed_sample(const int* off, int n, int lq, int row, int& j, int& m) {
    int lo = 0, hi = n;          // off[lo] <= row < off[hi], as far as there is such a place
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (off[mid] <= row) lo = mid;
        else hi = mid;
    }
    j = row - off[lo];
    m = min(lq, off[lo + 1] - off[lo]);
    return j >= 0 && j < m ? lo : -1;
}

// CACHE: k and v go to pages.  U heads' loads are on their way at once.
template <typename T, int VW, bool INTER, bool CACHE>
__global__ __launch_bounds__(NTH) void rope_fwd_kernel(const RopeArgs a, const T* q, const T* k, const T* v, T* qo,
                                                       T* ko) {
    constexpr int U = 4;
    const int tid = threadIdx.x, g = tid >> a.lps, hg = g & ((1 << a.hgs) - 1);
    const int row = blockIdx.x * (NTH >> (a.lps + a.hgs)) + (g >> a.hgs);
    if (row >= a.rows) return;
    const Unit<VW, INTER> u(tid & ((1 << a.lps) - 1), a.dh, a.rot);
    int i = row / a.l, j = row - i * a.l, p = j;
    long page = -1;
    int pr = 0;
    if constexpr (CACHE) {
        int m = a.l;
        if (a.q_off) i = packed_sample(a.q_off, a.n, a.l, row, j, m);
        if (i < 0) return;
        p = a.len[i] - m + j;
        if (p >= 0 && p / a.pg.page < a.pg.per_seq) {
            const int e = a.pg.table[i * a.pg.table_sn + p / a.pg.page];
            if (e >= 0 && e < a.pg.pages) page = e;
            pr = p % a.pg.page;
        }
    }
    if (a.pos) p = a.pos[row];
    const bool packed = CACHE && a.q_off;
    auto at = [&](const PtcgHeadLayout& l) { return packed ? row * l.sl : i * l.sn + j * l.sl; };
    const long kj = CACHE ? page * a.pg.k.sn + pr * a.pg.k.sl : at(a.ko);
    float c[VW], s[VW];
    angles<VW, INTER>(a, u, p, c, s);
    // The heads of q, of k, and (copied) of v, groups of the row in turn from head h0 on.
    const int HG = 1 << a.hgs;
    auto heads = [&](const T* src, long ssh, T* dst, long dsh, int n, int h0, const float* w, auto turns) {
        float wv[2 * VW];
#pragma unroll
        for (int e = 0; e < 2 * VW; ++e)
            wv[e] = decltype(turns)::value && u.live && w ? w[e < VW ? u.oa + e : u.ob + e - VW] : 1.f;
        for (int h = h0; h < n; h += U << a.hgs) {
            Pairs<T, VW> x[U];
#pragma unroll
            for (int t = 0; t < U; ++t)
                if (u.live && h + (t << a.hgs) < n) x[t].load(src + (h + (t << a.hgs)) * ssh, u.oa, u.ob);
#pragma unroll
            for (int t = 0; t < U; ++t) {
                if (h + (t << a.hgs) >= n) break;
                if constexpr (decltype(turns)::value) {
                    float y[2 * VW];
#pragma unroll
                    for (int e = 0; e < 2 * VW; ++e) y[e] = 0.f;
                    if (u.live) x[t].get(y);
                    if (w) {
                        float ss = 0.f;
#pragma unroll
                        for (int e = 0; e < 2 * VW; ++e) ss = fmaf(y[e], y[e], ss);
                        const float r = rsqrt_of(group_sum(ss, a.lps) * a.inv_dh + a.eps);
#pragma unroll
                        for (int e = 0; e < 2 * VW; ++e) y[e] *= r * wv[e];
                    }
                    turn<VW, INTER>(y, c, s, u.turns, 1.f);
                    x[t].set(y);
                }
                if (u.live) x[t].store(dst + (h + (t << a.hgs)) * dsh, u.oa, u.ob);
            }
        }
    };
    auto from = [&](int before) { return (hg - before) & (HG - 1); };
    heads(q + at(a.q), a.q.sh, qo + at(a.qo), a.qo.sh, a.H, hg, a.wq, std::true_type());
    if (!CACHE || page >= 0)
        heads(k + at(a.k), a.k.sh, (CACHE ? static_cast<T*>(a.pg.kp) : ko) + kj, CACHE ? a.pg.k.sh : a.ko.sh, a.KV,
              from(a.H), a.wk, std::true_type());
    if constexpr (CACHE)
        if (page >= 0)
            heads(v + at(a.v), a.v.sh, static_cast<T*>(a.pg.vp) + page * a.pg.v.sn + pr * a.pg.v.sl, a.pg.v.sh, a.KV,
                  from(a.H + a.KV), nullptr, std::false_type());
}

// Backward.  Workgroups walk the rows with a stride, so that a thread's part of
// dw stays in registers; its sums over the workgroup's groups meet in LDS in group
// order, over the workgroups in rope_dw_kernel.
template <typename T, int VW, bool INTER>
__global__ __launch_bounds__(NTH) void rope_bwd_kernel(const RopeArgs a, const T* __restrict__ q,
        const T* __restrict__ k, const T* __restrict__ dqo, const T* __restrict__ dko, T* __restrict__ dq,
        T* __restrict__ dk, float* __restrict__ part) {
    constexpr int U = 2;
    __shared__ float acc[NTH * 4 * VW];
    const int tid = threadIdx.x, g = tid >> a.lps, hg = g & ((1 << a.hgs) - 1), lane = tid & ((1 << a.lps) - 1);
    const Unit<VW, INTER> u(lane, a.dh, a.rot);
    const int per = NTH >> (a.lps + a.hgs), HG = 1 << a.hgs;
    float gq[2 * VW], gk[2 * VW];
#pragma unroll
    for (int e = 0; e < 2 * VW; ++e) gq[e] = gk[e] = 0.f;
    for (int row = blockIdx.x * per + (g >> a.hgs); row < a.rows; row += gridDim.x * per) {
        const int i = row / a.l, j = row - i * a.l, p = a.pos ? a.pos[row] : j;
        float c[VW], s[VW];
        angles<VW, INTER>(a, u, p, c, s);
        auto at = [&](const PtcgHeadLayout& l) { return i * l.sn + j * l.sl; };
        auto heads = [&](const T* xs, T* dx, long xsh, const T* dy, long ysh, int n, int h0, const float* w,
                         float (&gw)[2 * VW]) {
            float wv[2 * VW];
#pragma unroll
            for (int e = 0; e < 2 * VW; ++e) wv[e] = u.live && w ? w[e < VW ? u.oa + e : u.ob + e - VW] : 1.f;
            for (int h = h0; h < n; h += U << a.hgs) {
                Pairs<T, VW> x[U], d[U];
#pragma unroll
                for (int t = 0; t < U; ++t) {
                    if (!u.live || h + (t << a.hgs) >= n) continue;
                    d[t].load(dy + (h + (t << a.hgs)) * ysh, u.oa, u.ob);
                    if (w) x[t].load(xs + (h + (t << a.hgs)) * xsh, u.oa, u.ob);
                }
#pragma unroll
                for (int t = 0; t < U; ++t) {
                    if (h + (t << a.hgs) >= n) break;
                    float y[2 * VW];
#pragma unroll
                    for (int e = 0; e < 2 * VW; ++e) y[e] = 0.f;
                    if (u.live) d[t].get(y);
                    turn<VW, INTER>(y, c, s, u.turns, -1.f);
                    if (w) {
                        float xv[2 * VW], ss = 0.f, sd = 0.f;
#pragma unroll
                        for (int e = 0; e < 2 * VW; ++e) xv[e] = 0.f;
                        if (u.live) x[t].get(xv);
#pragma unroll
                        for (int e = 0; e < 2 * VW; ++e) {
                            ss = fmaf(xv[e], xv[e], ss);
                            sd = fmaf(y[e] * wv[e], xv[e], sd);
                        }
                        ss = group_sum(ss, a.lps);
                        sd = group_sum(sd, a.lps);
                        const float r = rsqrt_of(ss * a.inv_dh + a.eps), m = r * r * (sd * a.inv_dh);
#pragma unroll
                        for (int e = 0; e < 2 * VW; ++e) {
                            gw[e] += y[e] * (xv[e] * r);
                            y[e] = r * (y[e] * wv[e] - xv[e] * m);
                        }
                    }
                    d[t].set(y);
                    if (u.live) d[t].store(dx + (h + (t << a.hgs)) * xsh, u.oa, u.ob);
                }
            }
        };
        heads(q + at(a.q), dq + at(a.q), a.q.sh, dqo + at(a.qo), a.qo.sh, a.H, hg, a.wq, gq);
        heads(k + at(a.k), dk + at(a.k), a.k.sh, dko + at(a.ko), a.ko.sh, a.KV, (hg - a.H) & (HG - 1), a.wk, gk);
    }
    if (!part) return;
    // column e of q (then of k) over the groups
    const int G = NTH >> a.lps;
#pragma unroll
    for (int e = 0; e < 2 * VW; ++e) {
        const int at = e < VW ? u.oa + e : u.ob + e - VW;
        if (u.live) {
            acc[g * 2 * a.dh + at] = gq[e];
            acc[g * 2 * a.dh + a.dh + at] = gk[e];
        }
    }
    __syncthreads();
    for (int col = tid; col < 2 * a.dh; col += NTH) {
        float t = 0.f;
        for (int x = 0; x < G; ++x) t += acc[x * 2 * a.dh + col];
        part[(long)blockIdx.x * 2 * a.dh + col] = t;
    }
}

// dw from the workgroups' parts: 16 columns a workgroup, 64 threads down a column
__global__ __launch_bounds__(1024) void rope_dw_kernel(const float* __restrict__ part, int nblk, int dh,
                                                       float* __restrict__ dwq, float* __restrict__ dwk) {
    __shared__ double sh[64][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
    double t = 0;       // the parts' sums are long and of both signs
    if (col < 2 * dh)
#pragma unroll 4
        for (int b = r; b < nblk; b += 64) t += part[(long)b * 2 * dh + col];
    sh[r][c] = t;
    __syncthreads();
    if (r > 0 || col >= 2 * dh) return;
    for (int x = 1; x < 64; ++x) t += sh[x][c];
    float* out = col < dh ? dwq : dwk;
    if (out) out[col < dh ? col : col - dh] = (float)t;
}

// ------------------------------------------------------------------- host
int ilog2_up(int x) {
    int s = 0;
    while (1 << s < x) ++s;
    return s;
}

// The widest vector that widths, strides and addresses allow.
int vector_width(const RopeArgs& a, int es, const PtcgHeadLayout* const* lays, int nl, const void* const* ptrs,
                 int np) {
    for (int vw = 16 / es; vw > 1; vw /= 2) {
        bool ok = a.dh % (2 * vw) == 0 && a.rot % (2 * vw) == 0;
        for (int i = 0; i < nl; ++i) ok = ok && lays[i]->sn % vw == 0 && lays[i]->sl % vw == 0 && lays[i]->sh % vw == 0;
        for (int i = 0; i < np; ++i) ok = ok && (uintptr_t)ptrs[i] % (vw * es) == 0;
        if (ok) return vw;
    }
    return 1;
}

// Groups a row: as few as make 1 024 threads a CU, since each makes the row's angles anew
// and a group that walks several heads has their loads on their way together.  (With groups for 4 096:
// 65 539 bf16 rows of 8 + 2 heads of 128 forward 74 us for 70, backward 116 for 112; 49 664 of 4 + 4 of
// 64 42 for 21 and 70 for 37.  The backward launches no more than 1 024 threads a CU, see bwd_blocks.)
void set_groups(RopeArgs& a, int vw, int heads) {
    a.lps = ilog2_up((a.dh + 2 * vw - 1) / (2 * vw));
    const long want = (long)cu_count() * 1024;     // threads
    a.hgs = 0;
    while (a.lps + a.hgs < 8 && (1 << a.hgs) < heads && ((long)a.rows << (a.lps + a.hgs)) < want) ++a.hgs;
}

// A launch holds fewer than 2^32 threads (the backward's grid is bounded as it is).
int check_launch(const RopeArgs& a, const char* who) {
    PT_REQUIRE(((int64_t)a.rows << (a.lps + a.hgs)) <= (1LL << 32) - NTH,
               "%s: too many rows: %d of %d lanes a head", who, a.rows, 1 << a.lps);
    return PTCG_OK;
}
int check_rope(const PtcgRope& r, int dh, const char* who) {
    PT_REQUIRE(r.rot >= 0 && r.rot <= dh && r.rot % 2 == 0, "%s: %d turning elements of a head of %d", who, r.rot, dh);
    PT_REQUIRE(r.interleaved == 0 || r.interleaved == 1, "%s: interleaved=%d", who, r.interleaved);
    PT_REQUIRE(r.rot == 0 || r.freq, "%s: no frequencies", who);
    PT_REQUIRE(r.rot == 0 || (r.mag > -1e30f && r.mag < 1e30f), "%s: mag must be finite", who);
    return PTCG_OK;
}
int check_head(int heads, int kv_heads, int dh, int bf16, float eps, const char* who) {
    PT_REQUIRE(heads >= 1 && kv_heads >= 0, "%s: %d heads and %d kv heads", who, heads, kv_heads);
    PT_REQUIRE(heads < (1 << 20) && kv_heads < (1 << 20), "%s: too many heads", who);
    PT_REQUIRE(dh >= 2 && dh <= 128 && dh % 2 == 0, "%s: head width %d is not even, 2 to 128", who, dh);
    PT_REQUIRE(bf16 == 0 || bf16 == 1, "%s: bf16=%d", who, bf16);
    PT_REQUIRE(eps >= 0.f && eps < 1e30f, "%s: eps must be finite and not negative", who);
    return PTCG_OK;
}
int check_qk(const PtcgQkRope* d, const char* who) {
    PT_REQUIRE(d, "%s: null descriptor", who);
    PT_REQUIRE(d->n >= 0 && d->l >= 0, "%s: negative size n=%d l=%d", who, d->n, d->l);
    PT_REQUIRE((int64_t)d->n * d->l < (1 << 30), "%s: too many rows", who);
    PT_TRY(check_head(d->heads, d->kv_heads, d->dh, d->bf16, d->eps, who));
    PT_TRY(check_rope(d->rope, d->dh, who));
    PT_REQUIRE(layout_ok(d->q, 1) && layout_ok(d->qo, 1) && (!d->kv_heads || (layout_ok(d->k, 1) && layout_ok(d->ko, 1))),
               "%s: negative stride", who);
    return PTCG_OK;
}
bool aligned(const void* p, int es) { return (uintptr_t)p % es == 0; }

RopeArgs qk_args(const PtcgQkRope* d) {
    RopeArgs a = {};
    a.n = d->n; a.l = d->l; a.H = d->heads; a.KV = d->kv_heads; a.dh = d->dh; a.rot = d->rope.rot;
    a.rows = d->n * d->l;
    a.q = d->q; a.k = d->k; a.qo = d->qo; a.ko = d->ko;
    a.wq = d->wq; a.wk = d->wk;
    a.eps = d->eps; a.mag = d->rope.mag; a.inv_dh = 1.f / d->dh;
    a.freq = d->rope.freq; a.pos = d->rope.pos;
    return a;
}

template <typename T, int VW, bool INTER, bool CACHE>
int launch_rope(const RopeArgs& a, const void* q, const void* k, const void* v, void* qo, void* ko, hipStream_t s) {
    hipLaunchKernelGGL((rope_fwd_kernel<T, VW, INTER, CACHE>), dim3(pt_cdiv((long)a.rows << (a.lps + a.hgs), NTH)),
                       dim3(NTH), 0, s, a, static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                       static_cast<T*>(qo), static_cast<T*>(ko));
    PT_LAUNCH_CHECK();
    return PTCG_OK;
}
template <typename T, bool CACHE>
int rope_vw(const RopeArgs& a, int vw, bool inter, const void* q, const void* k, const void* v, void* qo, void* ko,
            hipStream_t s) {
#define PT_ROPE_VW(W) \
    return inter ? launch_rope<T, W, true, CACHE>(a, q, k, v, qo, ko, s) : launch_rope<T, W, false, CACHE>(a, q, k, v, qo, ko, s)
    if constexpr (sizeof(T) == 2)
        if (vw == 8) PT_ROPE_VW(8);
    if (vw == 4) PT_ROPE_VW(4);
    if (vw == 2) PT_ROPE_VW(2);
    PT_ROPE_VW(1);
#undef PT_ROPE_VW
}

template <typename T, int VW, bool INTER>
int launch_bwd(const RopeArgs& a, int nblk, const void* q, const void* k, const void* dqo, const void* dko, void* dq,
               void* dk, float* part, hipStream_t s) {
    hipLaunchKernelGGL((rope_bwd_kernel<T, VW, INTER>), dim3(nblk), dim3(NTH), 0, s, a, static_cast<const T*>(q),
                       static_cast<const T*>(k), static_cast<const T*>(dqo), static_cast<const T*>(dko),
                       static_cast<T*>(dq), static_cast<T*>(dk), part);
    PT_LAUNCH_CHECK();
    return PTCG_OK;
}
template <typename T>
int bwd_vw(const RopeArgs& a, int nblk, int vw, bool inter, const void* q, const void* k, const void* dqo,
           const void* dko, void* dq, void* dk, float* part, hipStream_t s) {
#define PT_ROPE_VW(W)                                                                                      \
    return inter ? launch_bwd<T, W, true>(a, nblk, q, k, dqo, dko, dq, dk, part, s)                       \
                 : launch_bwd<T, W, false>(a, nblk, q, k, dqo, dko, dq, dk, part, s)
    if constexpr (sizeof(T) == 2)
        if (vw == 8) PT_ROPE_VW(8);
    if (vw == 4) PT_ROPE_VW(4);
    if (vw == 2) PT_ROPE_VW(2);
    PT_ROPE_VW(1);
#undef PT_ROPE_VW
}

// workgroups of the backward, at most: each leaves a part of dw, and walks its rows (four times as many:
// 118 us for 113 over the 65 539 rows above, 43 for 37 over the 49 664)
int bwd_blocks(const PtcgQkRope* d) {
    const long rows = (long)d->n * d->l;
    const long most = 4L * cu_count();
    return (int)(rows < most ? rows : most);
}

}  // namespace

extern "C" int ptcg_rope_frequencies(int rot, double base, int scaling, double factor, double length, double fast,
                                     double slow, double* freq, float* mag) {
    PT_REQUIRE(rot >= 0 && rot % 2 == 0, "rope_frequencies: %d turning elements", rot);
    PT_REQUIRE((rot == 0 || freq) && mag, "rope_frequencies: null buffer");
    PT_REQUIRE(base > 1.0 && base < 1e300, "rope_frequencies: the base must be finite, above 1");
    PT_REQUIRE(scaling >= 0 && scaling <= 3, "rope_frequencies: scaling=%d", scaling);
    PT_REQUIRE(scaling == 0 || (factor >= 1.0 && factor < 1e300), "rope_frequencies: the factor must be finite, 1 or more");
    PT_REQUIRE(scaling != 3 || (length > 0.0 && length < 1e300 && slow >= 0.0 && fast > slow && fast < 1e300),
               "rope_frequencies: by parts takes a length above 0 and 0 <= slow < fast");
    const double b = scaling == 2 && rot > 2 ? base * pow(factor, (double)rot / (rot - 2)) : base;
    for (int i = 0; i < rot / 2; ++i) {
        double f = pow(b, -2.0 * i / rot);
        if (scaling == 1) f /= factor;
        if (scaling == 3) {
            const double turns = length * f / (2.0 * M_PI);
            double keep = (turns - slow) / (fast - slow);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
            f = f * keep + f / factor * (1.0 - keep);
        }
        freq[i] = f;
    }
    *mag = scaling == 3 ? (float)(0.1 * log(factor) + 1.0) : 1.f;
    return PTCG_OK;
}

extern "C" int ptcg_kernel_qk_norm_rope_fwd(const PtcgQkRope* d, const void* q, const void* k, void* qo, void* ko,
                                            void* stream) {
    const char* who = "qk_norm_rope_fwd";
    PT_TRY(check_qk(d, who));
    RopeArgs a = qk_args(d);
    if (a.rows == 0) return PTCG_OK;
    PT_REQUIRE(q && qo && (a.KV == 0 || (k && ko)), "%s: null buffer", who);
    const int es = d->bf16 ? 2 : 4;
    PT_REQUIRE(aligned(q, es) && aligned(qo, es) && (a.KV == 0 || (aligned(k, es) && aligned(ko, es))),
               "%s: buffers off their type's alignment", who);
    PT_REQUIRE(layout_apart(d->qo, false, d->n, d->l, d->heads, d->dh), "%s: rows of qo overlap", who);
    PT_REQUIRE(a.KV == 0 || layout_apart(d->ko, false, d->n, d->l, d->kv_heads, d->dh), "%s: rows of ko overlap", who);
    auto same = [](const PtcgHeadLayout& x, const PtcgHeadLayout& y) {
        return x.sn == y.sn && x.sl == y.sl && x.sh == y.sh;
    };
    PT_REQUIRE((q != qo || same(d->q, d->qo)) && (a.KV == 0 || k != ko || same(d->k, d->ko)),
               "%s: in place only with one layout", who);
    if (a.KV == 0) { a.k = a.q; a.ko = a.qo; k = q; ko = qo; }
    const PtcgHeadLayout* lays[] = {&a.q, &a.k, &a.qo, &a.ko};
    const void* ptrs[] = {q, k, qo, ko};
    const int vw = vector_width(a, es, lays, 4, ptrs, 4);
    set_groups(a, vw, a.H + a.KV);
    PT_TRY(check_launch(a, who));
    const hipStream_t s = (hipStream_t)stream;
    return d->bf16 ? rope_vw<__bf16, false>(a, vw, d->rope.interleaved, q, k, nullptr, qo, ko, s)
                   : rope_vw<float, false>(a, vw, d->rope.interleaved, q, k, nullptr, qo, ko, s);
}

extern "C" int64_t ptcg_kernel_qk_norm_rope_bwd_ws_bytes(const PtcgQkRope* d) {
    if (check_qk(d, "qk_norm_rope_bwd_ws_bytes") != PTCG_OK) return -1;
    return d->wq || d->wk ? (int64_t)bwd_blocks(d) * 2 * d->dh * 4 : 0;
}

extern "C" int ptcg_kernel_qk_norm_rope_bwd(const PtcgQkRope* d, const void* q, const void* k, const void* dqo,
                                            const void* dko, void* dq, void* dk, float* dwq, float* dwk,
                                            void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "qk_norm_rope_bwd";
    PT_TRY(check_qk(d, who));
    RopeArgs a = qk_args(d);
    const hipStream_t s = (hipStream_t)stream;
    const bool kv = a.KV > 0;
    PT_REQUIRE((dwq == nullptr || d->wq) && (dwk == nullptr || d->wk), "%s: a weight's gradient without its weight", who);
    const bool dw = dwq || dwk;
    const int64_t need = dw ? ptcg_kernel_qk_norm_rope_bwd_ws_bytes(d) : 0;
    PT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && al16(workspace)),
               "%s: workspace of %lld bytes, need %lld (16 B aligned)", who, (long long)workspace_bytes,
               (long long)need);
    if (a.rows > 0) {
        PT_REQUIRE(dqo && dq && (!kv || (dko && dk)) && (!d->wq || q) && (!kv || !d->wk || k), "%s: null buffer", who);
        const int es = d->bf16 ? 2 : 4;
        for (const void* p : {q, k, dqo, dko, (const void*)dq, (const void*)dk})
            PT_REQUIRE(aligned(p, es), "%s: buffers off their type's alignment", who);
        PT_REQUIRE(layout_apart(d->q, false, d->n, d->l, d->heads, d->dh),
                   "%s: rows of dq overlap (a broadcast q has no gradient layout)", who);
        PT_REQUIRE(!kv || layout_apart(d->k, false, d->n, d->l, d->kv_heads, d->dh),
                   "%s: rows of dk overlap (a broadcast k has no gradient layout)", who);
        if (!kv) { a.k = a.q; a.ko = a.qo; k = q; dko = dqo; dk = dq; }
        const PtcgHeadLayout* lays[] = {&a.q, &a.k, &a.qo, &a.ko};
        const void* ptrs[] = {q, k, dqo, dko, dq, dk};
        const int vw = vector_width(a, es, lays, 4, ptrs, 6);
        set_groups(a, vw, a.H + a.KV);
        const long full = pt_cdiv((long)a.rows << (a.lps + a.hgs), NTH);
        const int nblk = (int)(full < bwd_blocks(d) ? full : bwd_blocks(d));
        float* part = dw ? static_cast<float*>(workspace) : nullptr;
        PT_TRY(d->bf16 ? bwd_vw<__bf16>(a, nblk, vw, d->rope.interleaved, q, k, dqo, dko, dq, dk, part, s)
                       : bwd_vw<float>(a, nblk, vw, d->rope.interleaved, q, k, dqo, dko, dq, dk, part, s));
        if (!dw) return PTCG_OK;
        hipLaunchKernelGGL(rope_dw_kernel, dim3(pt_cdiv(2 * a.dh, 16)), dim3(1024), 0, s, part, nblk, a.dh, dwq, dwk);
        PT_LAUNCH_CHECK();
        return PTCG_OK;
    }
    if (dw) {     // no rows: sums of nothing
        hipLaunchKernelGGL(rope_dw_kernel, dim3(pt_cdiv(2 * a.dh, 16)), dim3(1024), 0, s, (const float*)nullptr, 0, a.dh,
                           dwq, dwk);
        PT_LAUNCH_CHECK();
    }
    return PTCG_OK;
}

extern "C" int ptcg_kernel_paged_append(const PtcgPagedAppend* d, const void* q, const void* k, const void* v,
                                        void* qo, void* stream) {
    const char* who = "paged_append";
    PT_REQUIRE(d, "%s: null descriptor", who);
    PT_REQUIRE(d->n >= 0 && d->lq >= 0 && (!d->q_off || d->rows >= 0), "%s: negative size n=%d lq=%d rows=%d", who, d->n,
               d->lq, d->rows);
    const int64_t rows = d->q_off ? (int64_t)d->rows : (int64_t)d->n * d->lq;
    PT_REQUIRE(rows < (1 << 30), "%s: too many rows", who);
    PT_TRY(check_head(d->heads, d->kv_heads, d->dh, d->bf16, d->eps, who));
    PT_REQUIRE(d->kv_heads >= 1, "%s: %d kv heads", who, d->kv_heads);
    PT_TRY(check_rope(d->rope, d->dh, who));
    PT_TRY(check_pages(d->cache, d->n, d->kv_heads, d->dh, 1, who));
    PT_REQUIRE(layout_apart(d->cache.k, false, d->cache.pages, d->cache.page, d->kv_heads, d->dh) &&
                   layout_apart(d->cache.v, false, d->cache.pages, d->cache.page, d->kv_heads, d->dh),
               "%s: rows of the pages overlap", who);
    PT_REQUIRE((q == nullptr) == (qo == nullptr), "%s: q and qo are given together", who);
    PT_REQUIRE((!q || (layout_ok(d->q, 1) && layout_ok(d->qo, 1))) && layout_ok(d->k, 1) && layout_ok(d->v, 1),
               "%s: negative stride", who);
    if (d->n == 0 || d->lq == 0 || rows == 0) return PTCG_OK;
    PT_REQUIRE(k && v && d->len, "%s: null buffer", who);
    const int es = d->bf16 ? 2 : 4;
    for (const void* p : {q, k, v, (const void*)qo, (const void*)d->cache.kp, (const void*)d->cache.vp})
        PT_REQUIRE(aligned(p, es), "%s: buffers off their type's alignment", who);
    PT_REQUIRE(!q || layout_apart(d->qo, d->q_off, d->n, d->lq, d->heads, d->dh), "%s: rows of qo overlap", who);
    PT_REQUIRE(q != qo || !q || (d->q.sn == d->qo.sn && d->q.sl == d->qo.sl && d->q.sh == d->qo.sh),
               "%s: in place only with one layout", who);
    RopeArgs a = {};
    a.n = d->n; a.l = d->lq; a.H = q ? d->heads : 0; a.KV = d->kv_heads; a.dh = d->dh; a.rot = d->rope.rot;
    a.rows = (int)rows;
    a.q = q ? d->q : d->k; a.k = d->k; a.v = d->v; a.qo = q ? d->qo : d->k;
    a.wq = d->wq; a.wk = d->wk;
    a.eps = d->eps; a.mag = d->rope.mag; a.inv_dh = 1.f / d->dh;
    a.freq = d->rope.freq; a.pos = d->rope.pos;
    a.q_off = d->q_off; a.len = d->len;
    a.pg = d->cache;
    const PtcgHeadLayout* lays[] = {&a.q, &a.k, &a.v, &a.qo, &a.pg.k, &a.pg.v};
    const void* ptrs[] = {q, k, v, qo, a.pg.kp, a.pg.vp};
    const int vw = vector_width(a, es, lays, 6, ptrs, 6);
    set_groups(a, vw, a.H + 2 * a.KV);
    PT_TRY(check_launch(a, who));
    const hipStream_t s = (hipStream_t)stream;
    return d->bf16 ? rope_vw<__bf16, true>(a, vw, d->rope.interleaved, q, k, v, qo, nullptr, s)
                   : rope_vw<float, true>(a, vw, d->rope.interleaved, q, k, v, qo, nullptr, s);
}
