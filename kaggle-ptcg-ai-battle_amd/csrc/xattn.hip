// Cross attention: query rows against an encoder's key / value rows of another
// length, shared kv heads, key masks, padded or packed samples; fp32 or bf16.
//
// Forward, per (sample, query head), over the kept keys j:
//   s_ij = scale q_i . k_j,  m_i = max_j s_ij,  l_i = sum_j exp(s_ij - m_i),
//   o_i = sum_j exp(s_ij - m_i) v_j / l_i,  lse_i = m_i + log l_i,
// in one pass over the keys: a tile's larger maximum rescales what is summed.
// Backward, with P_ij = exp(s_ij - lse_i) and D_i = do_i . o_i:
//   dv_j = sum_i P_ij do_i,  dS_ij = P_ij (do_i . v_j - D_i),
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,
// dk and dv summed over the query heads that share the kv head, in row order.
// A query that keeps no key, or whose kept scores are all -inf: o = 0, lse =
// -inf, and it adds to no gradient.
//
// Layout.  The G = heads / kv_heads query heads of a kv head are one matrix of
// lq * G rows (row r is query r / G, head r % G), so a single token's heads
// fill one tile and a gradient's sum over the heads is a sum over rows.  All
// products run as 32 x 32 tiles of v_mfma_f32_32x32x16_bf16, computed
// transposed: S^T = K Q^T leaves query lane % 32 of keys {8 (r / 4) +
// 4 (lane / 32) + r % 4} in register r, which is a B operand of O^T = V^T P^T
// over the same order of the keys, so P goes from accumulators to the next
// product without passing through LDS, and a query's maximum and sum are
// in-lane but for one exchange of the halves.  The A operand V^T comes from
// row-major LDS by ds_read_b64_tr_b16 (4 keys of 16 columns to a lane's 4
// values).
// fp32 operands are split into three bf16 terms (x = x0 + x1 + x2, 8 bits each,
// exact above 2^-102) that lie in LDS as three planes; a product is six term
// products, small ones first: 6 / 16 of the time of v_mfma_f32_32x32x2_f32.
// With |x1| <= 2^-8 |x| and |x2| <= 2^-17 |x|, the three left out (x1 y2, x2 y1,
// x2 y2) come to 2^-24 |x y| at most, one rounding of fp32.  An infinite operand becomes NaN in the products.
#include "attn_tiles.h"

#include <type_traits>

namespace {

// the descriptor as the kernels take it
struct XArgs {
    int n, lq, lk, H, KV, G, dh;
    unsigned gmagic;              // r / G = umulhi(r, gmagic) for r G < 2^32 (G > 1)
    float scale, scale2;          // scale2 = scale * log2(e): exponentials are exp2
    PtcgHeadLayout q, k, v, o;
    const int *q_off, *k_off, *k_len;
    const float* keep;
    long keep_sn;
    bool sorted;                  // place_of
};

struct Sample { long q, k, v, o, keep; int ql, kl; };   // element offsets of row 0, and row counts

// Row counts come from device memory: they are held to the host's bounds.
__device__ __forceinline__ Sample sample_of(const XArgs& a, int i) {
    Sample s;
    s.ql = a.lq; s.kl = a.lk;
    if (a.q_off) {
        const int r0 = a.q_off[i];
        s.ql = max(0, min(a.lq, a.q_off[i + 1] - r0));
        s.q = r0 * a.q.sl; s.o = r0 * a.o.sl;
    } else {
        s.q = i * a.q.sn; s.o = i * a.o.sn;
    }
    if (a.k_off) {
        const int r0 = a.k_off[i];
        s.kl = max(0, min(a.lk, a.k_off[i + 1] - r0));
        s.k = r0 * a.k.sl; s.v = r0 * a.v.sl; s.keep = r0;
    } else {
        s.k = i * a.k.sn; s.v = i * a.v.sn; s.keep = i * a.keep_sn;
        if (a.k_len) s.kl = max(0, min(a.lk, a.k_len[i]));
    }
    return s;
}

// Which (sample, rest) a workgroup works on.  Samples whose lengths only the
// device knows (`sorted`: up to 64 of them) are taken in the order of a tile's
// cost, longest first, without gaps: workgroups start in index order, and a long
// one that starts last runs alone (16 packed samples of 376 .. 1 501 rows and
// 1 001 .. 4 003 keys on 512 places, forward and backward: 1.00 ms against 1.30
// in index order).  Indexes past the last tile: i = -1.
struct Place { int i, rest; };
template <class Cost, class Tiles>
__device__ __forceinline__ Place place_of(const XArgs& a, bool sorted, int b, int nblk, int per_sample, Cost cost,
                                          Tiles tiles) {
    Place p;
    if (!sorted) {
        const int l = xcd_block(b, nblk);
        p.i = l / per_sample;
        p.rest = l - p.i * per_sample;
        return p;
    }
    const int lane = threadIdx.x & 63;
    const Sample s = sample_of(a, min(lane, a.n - 1));
    const int c = lane < a.n ? cost(s) : -1, t = lane < a.n ? tiles(s) : 0;
    int first = 0;
    for (int j = 0; j < a.n; ++j) {
        const int cj = __builtin_amdgcn_readlane(c, j), tj = __builtin_amdgcn_readlane(t, j);
        if (cj > c || (cj == c && j < lane)) first += tj;
    }
    const unsigned long long m = __ballot(b >= first && b < first + t);
    p.i = m ? __builtin_ctzll(m) : -1;
    p.rest = m ? b - __builtin_amdgcn_readlane(first, __builtin_ctzll(m)) : 0;
    return p;
}

// A tile of keys and values on its way: masked rows enter LDS as zeros, so that
// what they hold, NaN too, reaches no product; kf holds 0 or -inf per key.
template <typename T, int DH, bool PAD, int BK, int NTH> struct KvTile {
    typedef Stage<T, DH, PAD, BK, NTH> St;
    static_assert(BK <= NTH, "a thread per key flag");
    St k, v;
    float kp[St::NCH], kfr;
    RowBuf kb, vb, keep;
    int ko, vo, kend;
    bool masks;
    __device__ __forceinline__ void init(const XArgs& a, const Sample& s, const T* kp_, const T* vp, int kvh,
                                         int kend_, int tid) {
        constexpr int es = sizeof(T);
        kb = {reinterpret_cast<const char*>(kp_ + s.k + (long)kvh * a.k.sh), (int)a.k.sl * es, a.dh * es};
        vb = {reinterpret_cast<const char*>(vp + s.v + (long)kvh * a.v.sh), (int)a.v.sl * es, a.dh * es};
        keep = {reinterpret_cast<const char*>(a.keep + s.keep), 4, 4};
        masks = a.keep != nullptr;
        ko = St::first(kb.ld, a.dh, tid);
        vo = St::first(vb.ld, a.dh, tid);
        kend = kend_;
    }
    __device__ __forceinline__ void fetch(int row0, int tid) {
        const auto rk = kb.rows(row0, kend, BK), rv = vb.rows(row0, kend, BK);
        k.load(rk, ko, kb.ld);
        v.load(rv, vo, vb.ld);
        kfr = row0 + tid < kend ? 1.f : 0.f;
        if (masks) {
            const auto rm = keep.rows(row0, kend, BK);
#pragma unroll
            for (int i = 0; i < St::NCH; ++i) kp[i] = __uint_as_float(ld_buf4(rm, 4 * (tid / St::CPR + i * St::RPP)));
            kfr = __uint_as_float(ld_buf4(rm, 4 * tid));
        }
    }
    __device__ __forceinline__ void store(__bf16* Ks, __bf16* Vs, float* kf, int tid) const {
        if (masks) {
#pragma unroll
            for (int i = 0; i < St::NCH; ++i) {
                k.put(Ks, tid, i, kp[i] != 0.f);
                v.put(Vs, tid, i, kp[i] != 0.f);
            }
        } else {
            k.store(Ks, tid);
            v.store(Vs, tid);
        }
        if (tid < BK) kf[tid] = kfr != 0.f ? 0.f : -INFINITY;
    }
};

// the last kept key of [k0, kend), plus one (k0 if none): tiles behind a
// sample's valid prefix are not read.  A wave's part; the workgroup's is the
// largest of its waves'.
__device__ __forceinline__ int last_kept(const float* keep, int k0, int kend, int nth) {
    int last = k0;
    for (int j = k0 + (int)threadIdx.x; j - (int)(threadIdx.x & 63) < kend; j += nth) {
        const unsigned long long m = __ballot(j < kend && keep[min(j, kend - 1)] != 0.f);
        if (m) last = j - (int)(threadIdx.x & 63) + 64 - __builtin_clzll(m);
    }
    return last;
}

// ---------------------------------------------------------------- forward
// A workgroup owns 32 NW query rows; KS waves share a row block and split each
// tile of KS * KT keys (few rows against many keys), joined in LDS at the end.
// nsplit > 1: workgroups also split the keys, each leaving an unnormalised
// partial with its maximum and sum for xattn_join_kernel.
template <typename T, int DH, int NW, int KS, int KT> struct FwdCfg {
    static constexpr int NTH = 64 * NW * KS, BQ = 32 * NW, BK = KT * KS;
    static constexpr int TILE = tile_elems<T, DH, false, BK>();
    // One buffer: what a second one saves in barriers it costs in workgroups a CU
    // holds (with tiles of 64 keys, 8 192 x 64 x 97, 64 wide: 293 us against 333; a
    // token against 50 001 keys 39 against 46).
    static constexpr size_t PAIR = 4 * (size_t)TILE;   // bytes
    static constexpr size_t JOIN = (size_t)NW * (KS - 1) * (DH * 32 + 64) * sizeof(float);
    static constexpr size_t OUT = (size_t)NW * Out<T, DH>::WAVE * sizeof(T);   // the rows' way out
    static constexpr size_t BUFS = max3(PAIR, JOIN, OUT);
    static constexpr size_t LDS = BUFS + BK * sizeof(float) + 64;
};
// Waves a SIMD holds, for the register allocator: two (of 256 registers each)
// let one wave's softmax run beside the other's products.
template <typename T, int DH> constexpr int min_waves() { return sizeof(T) == 2 || DH <= 64 ? 2 : 1; }
// the backward holds two operands' rows; with a tile four times a wave's part
// (SPLIT waves along it) also on its way, one wave's registers.  Some spill all
// the same (registers a lane, by the compiler): the joint backward in fp32 64 wide
// 12 to 41, dk and dv in fp32 64 wide 2 to 29 and 128 wide up to 59, in bf16 128
// wide with two waves along the keys 24 and 68.
template <typename T, int DH, int SPLIT> constexpr int bwd_waves() {
    return DH * planes<T>() <= 64 || (SPLIT <= 2 && min_waves<T, DH>() == 2) ? 2 : 1;
}

template <typename T, int DH, int NW, int KS, int KT>
__global__ __launch_bounds__(64 * NW * KS, (min_waves<T, DH>())) void xattn_fwd_kernel(const XArgs a,
        const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, T* __restrict__ out,
        float* __restrict__ lse, float* __restrict__ part, int qtiles, int nsplit, int split_keys) {
    typedef FwdCfg<T, DH, NW, KS, KT> C;
    typedef KvTile<T, DH, false, C::BK, C::NTH> Kv;
    constexpr int PS = Kv::St::PS;
    extern __shared__ __align__(256) char smem[];
    __bf16* tiles = reinterpret_cast<__bf16*>(smem);
    float* kfs = reinterpret_cast<float*>(smem + C::BUFS);
    int* sh = reinterpret_cast<int*>(smem + C::LDS - 64);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const int qw = wave % NW, kw = wave / NW;
    const Place pl = place_of(a, a.sorted && nsplit == 1, blockIdx.x, gridDim.x, a.KV * qtiles * nsplit,
                              [](const Sample& x) { return x.kl; },
                              [&](const Sample& x) { return (x.ql * a.G + C::BQ - 1) / C::BQ * a.KV; });
    if (pl.i < 0) return;
    const int i = pl.i;
    const Sample s = sample_of(a, i);
    const int qtn = a.sorted && nsplit == 1 ? (s.ql * a.G + C::BQ - 1) / C::BQ : qtiles;
    const int qt = pl.rest % qtn, sp = pl.rest / qtn % nsplit, kvh = pl.rest / qtn / nsplit;
    const int rows = s.ql * a.G;
    if (qt * C::BQ >= rows) return;
    const int r = qt * C::BQ + 32 * qw + (lane & 31);
    const bool rok = r < rows;

    const int k0 = sp * split_keys;
    int kend = min(s.kl, k0 + split_keys);
    Kv kv;
    kv.init(a, s, k, v, kvh, kend, tid);
    if (k0 < kend) kv.fetch(k0, tid);       // on its way while the masks are looked through

    Row<T, DH> qf;
    qf.load(q + s.q + (rok ? row_off(a, a.q, kvh, r) : 0), rok, a.dh, h);

    float m2 = -INFINITY, l = 0.f;   // running maximum (of s scale2) and this half's sum
    floatx16 o[DH / 32];
#pragma unroll
    for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;

    if (a.keep && k0 < kend) {
        const int last = last_kept(a.keep + s.keep, k0, kend, C::NTH);
        if (lane == 0) sh[wave] = last;
        __syncthreads();
        kend = k0;
#pragma unroll
        for (int w = 0; w < NW * KS; ++w) kend = max(kend, sh[w]);
        kend = __builtin_amdgcn_readfirstlane(kend);
        kv.kend = kend;
    }
    const int nt = kend > k0 ? (kend - k0 + C::BK - 1) / C::BK : 0;

    auto tile = [&](int t, const __bf16* Ks, const float* kf) {
        const __bf16* Vs = Ks + C::TILE;
        const int row0 = k0 + t * C::BK + kw * KT;
        if (row0 >= kend) return;
        const bool masked = a.keep || row0 + KT > kend;
        floatx16 sc[KT / 32];
        float mt = -INFINITY;
#pragma unroll
        for (int j = 0; j < KT / 32; ++j)
            sc[j] = mma_rows<T, DH, false, PS>(Ks + (kw * KT + 32 * j) * Lds<DH, false>::ST, qf, lane);
        if (masked) {
#pragma unroll
            for (int j = 0; j < KT / 32; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 f = *reinterpret_cast<const float4*>(kf + kw * KT + 32 * j + 8 * e + 4 * h);
                    sc[j][4 * e] += f.x; sc[j][4 * e + 1] += f.y; sc[j][4 * e + 2] += f.z; sc[j][4 * e + 3] += f.w;
                }
        }
#pragma unroll
        for (int j = 0; j < KT / 32; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) mt = fmaxf(mt, sc[j][e]);
        mt = fmaxf(mt, half_swap(mt));
        const float mn = fmaxf(m2, mt * a.scale2);
        if (__any(mn > m2)) {
            const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m2 - mn);
            l *= al;
#pragma unroll
            for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[dt][e] *= al;
            m2 = mn;
        }
        const float ms = m2 == -INFINITY ? 0.f : m2;
#pragma unroll
        for (int j = 0; j < KT / 32; ++j) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                sc[j][e] = __builtin_amdgcn_exp2f(fmaf(sc[j][e], a.scale2, -ms));
                l += sc[j][e];
            }
            mma_tr<T, DH, false, PS>(Vs + (kw * KT + 32 * j) * Lds<DH, false>::ST, sc[j], o, lane);
        }
    };
    if (nt > 0) {
        kv.store(tiles, tiles + C::TILE, kfs, tid);
        if (nt > 1) kv.fetch(k0 + C::BK, tid);
        __syncthreads();
    }
    for (int t = 0; t < nt; ++t) {
        tile(t, tiles, kfs);
        __syncthreads();
        if (t + 1 < nt) {
            kv.store(tiles, tiles + C::TILE, kfs, tid);
            if (t + 2 < nt) kv.fetch(k0 + (t + 2) * C::BK, tid);
            __syncthreads();
        }
    }
    l += half_swap(l);

    // the key waves' results join in LDS, in wave order
    if constexpr (KS > 1) {
        float* jb = reinterpret_cast<float*>(smem);
        constexpr int JS = DH * 32 + 64;
        if (kw > 0) {
            float* p = jb + (size_t)((kw - 1) * NW + qw) * JS;
#pragma unroll
            for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) p[(dt * 16 + e) * 64 + lane] = o[dt][e];
            if (h == 0) {
                p[DH * 32 + lane] = m2;
                p[DH * 32 + 32 + lane] = l;
            }
        }
        __syncthreads();
        for (int w = 1; w < KS && kw == 0; ++w) {
            const float* p = jb + (size_t)((w - 1) * NW + qw) * JS;
            const float mw = p[DH * 32 + (lane & 31)], lw = p[DH * 32 + 32 + (lane & 31)];
            const float mn = fmaxf(m2, mw), ms = mn == -INFINITY ? 0.f : mn;
            const float f0 = __builtin_amdgcn_exp2f(m2 - ms), f1 = __builtin_amdgcn_exp2f(mw - ms);
            l = l * f0 + lw * f1;
            m2 = mn;
#pragma unroll
            for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[dt][e] = o[dt][e] * f0 + p[(dt * 16 + e) * 64 + lane] * f1;
        }
    }
    if constexpr (KS > 1) {
        __syncthreads();     // the joined buffers become the rows' way out
        if (kw > 0) return;
    }
    const int qi = head_div(a, rok ? r : 0), head = kvh * a.G + (rok ? r : 0) - qi * a.G;
    const long row = ((long)i * a.H + head) * a.lq + qi;
    if (nsplit > 1) {
        if (!rok) return;
        const long R = (long)a.n * a.H * a.lq;
        float* p = part + ((long)sp * R + row) * a.dh;
        store_row<float, DH>(p, o, 1.f, a.dh, h);
        if (h == 0) {
            float* ml = part + (long)nsplit * R * a.dh + ((long)sp * R + row) * 2;
            ml[0] = m2;
            ml[1] = l;
        }
        return;
    }
    // no key kept, or every kept score -inf: the sum is 0 (scores of NaN leave the
    // maximum at -inf too, but a sum of NaN); with no key kept no tile was read,
    // whatever the query holds
    const bool none = m2 == -INFINITY && l == 0.f;
    if (none) {
#pragma unroll
        for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
    }
    if (lse && rok && h == 0) lse[row] = none ? -INFINITY : m2 * LN2 + logf(l);
    Out<T, DH>::query_rows(a, a.o, out + s.o, kvh, qt * C::BQ + 32 * qw, rows, o, none ? 0.f : 1.f / l,
                           reinterpret_cast<T*>(smem) + qw * Out<T, DH>::WAVE, lane);
}

// Joins the key splits.  Groups of LG lanes (4 columns each) take a row's splits
// in turn, `per_row` groups a row, and meet in LDS in group order (one wave
// walking 56 splits waits them in line: 13.6 us for 32 rows of 128; one row a
// workgroup whatever its splits: 17 us more for 17 208 rows of 8 splits).
constexpr int JOIN_NTH = 512;
template <typename T, int LG>
__global__ __launch_bounds__(JOIN_NTH) void xattn_join_kernel(const XArgs a, const float* __restrict__ part,
        T* __restrict__ out, float* __restrict__ lse, int nsplit, int per_row) {
    constexpr int NG = JOIN_NTH / LG;
    __shared__ float4 sh[JOIN_NTH];
    __shared__ float2 shm[NG];
    const int tid = threadIdx.x, grp = tid / LG, c = tid % LG, g0 = grp & (per_row - 1);
    const long R = (long)a.n * a.H * a.lq, row = (long)blockIdx.x * (NG / per_row) + grp / per_row;
    const bool live = row < R;
    const int qi = live ? (int)(row % a.lq) : 0, head = live ? (int)(row / a.lq % a.H) : 0;
    const int i = live ? (int)(row / a.lq / a.H) : 0;
    const Sample s = sample_of(a, i);
    const float2* ml = reinterpret_cast<const float2*>(part + (long)nsplit * R * a.dh);
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    // one more split, or one more group: maximum em, sum el, values x
    auto add = [&](float em, float el, const float4& x) {
        const float mn = fmaxf(m, em), ms = mn == -INFINITY ? 0.f : mn;
        const float f0 = __builtin_amdgcn_exp2f(m - ms), f1 = __builtin_amdgcn_exp2f(em - ms);
        m = mn;
        l = l * f0 + el * f1;
        acc.x = acc.x * f0 + x.x * f1; acc.y = acc.y * f0 + x.y * f1;
        acc.z = acc.z * f0 + x.z * f1; acc.w = acc.w * f0 + x.w * f1;
    };
    if (live && qi < s.ql) {
#pragma unroll 4
        for (int p = g0; p < nsplit; p += per_row) {
            const float2 e = ml[p * R + row];
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (4 * c < a.dh) x = *reinterpret_cast<const float4*>(part + (p * R + row) * a.dh + 4 * c);
            add(e.x, e.y, x);
        }
    }
    sh[tid] = acc;
    if (c == 0) shm[grp] = make_float2(m, l);
    __syncthreads();
    if (g0 > 0 || !live || qi >= s.ql) return;
    for (int g = 1; g < per_row; ++g) {
        const float2 e = shm[grp + g];
        add(e.x, e.y, sh[(grp + g) * LG + c]);
    }
    const bool none = m == -INFINITY && l == 0.f;
    const float f = none ? 0.f : 1.f / l;
    if (none) acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (4 * c < a.dh)
        st4(out + s.o + (long)qi * a.o.sl + (long)head * a.o.sh + 4 * c, acc.x * f, acc.y * f, acc.z * f, acc.w * f);
    if (lse && c == 0) lse[row] = none ? -INFINITY : m * LN2 + logf(l);
}

// --------------------------------------------------------------- backward
// dQ: the forward's shape.  Per 32 keys S^T and dP^T = V dO^T with queries on
// lanes, dS^T in registers, dQ^T += K^T dS^T.  Also leaves D_i (from the
// stored o: in bf16 its rounding moves D by up to 2^-8 of terms that average out)
// for the dK / dV kernel, in row order of lse.
template <typename T, int DH, int NW, int KS, int KT> struct DqCfg {
    static constexpr int NTH = 64 * NW * KS, BQ = 32 * NW, BK = KT * KS;
    static constexpr int TILE = tile_elems<T, DH, DH == 128, BK>();
    static constexpr size_t PAIR = 4 * (size_t)TILE;   // bytes
    static constexpr size_t JOIN = (size_t)NW * (KS - 1) * DH * 32 * sizeof(float);
    static constexpr size_t OUT = (size_t)NW * Out<T, DH>::WAVE * sizeof(T);   // the rows' way out
    static constexpr size_t BUFS = max3(PAIR, JOIN, OUT);
    static constexpr size_t LDS = BUFS + BK * sizeof(float) + 64;
};

// what the backward reads and writes; part: the splits' (nsplit > 1)
template <typename T> struct Grads {
    const T *q, *k, *v, *out, *dout;
    const float* lse;
    T *dq, *dk, *dv;
    float *delta, *part;
};
// one workgroup's share of a sample: its tile, split and kv head
struct Share { int i, tile, sp, kvh; };

template <typename T, int DH, int NW, int KS, int KT>
__device__ __forceinline__ void dq_body(const XArgs& a, const Grads<T>& p, const Share& w, int nsplit,
                                        int split_keys, char* smem) {
    typedef DqCfg<T, DH, NW, KS, KT> C;
    typedef KvTile<T, DH, DH == 128, C::BK, C::NTH> Kv;
    constexpr int PS = Kv::St::PS;
    __bf16* tiles = reinterpret_cast<__bf16*>(smem);
    float* kfs = reinterpret_cast<float*>(smem + C::BUFS);
    int* sh = reinterpret_cast<int*>(smem + C::LDS - 64);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const int qw = wave % NW, kw = wave / NW;
    const int i = w.i, qt = w.tile, sp = w.sp, kvh = w.kvh;
    const Sample s = sample_of(a, i);
    const T *q = p.q, *k = p.k, *v = p.v, *out = p.out, *dout = p.dout;
    const float* lse = p.lse;
    T* dq = p.dq;
    float *delta = p.delta, *part = p.part;
    const int rows = s.ql * a.G;
    if (qt * C::BQ >= rows) return;
    const int r = qt * C::BQ + 32 * qw + (lane & 31);
    const bool rok = r < rows;

    const int k0 = sp * split_keys;
    int kend = min(s.kl, k0 + split_keys);
    Kv kv;
    kv.init(a, s, k, v, kvh, kend, tid);
    if (k0 < kend) kv.fetch(k0, tid);

    Row<T, DH> qf, df;
    qf.load(q + s.q + (rok ? row_off(a, a.q, kvh, r) : 0), rok, a.dh, h);
    const long oo = s.o + (rok ? row_off(a, a.o, kvh, r) : 0);
    float D = 0.f;
#pragma unroll
    for (int c = 0; c < DH / 16; ++c) {
        Chunk<T> x, y;
        x.zero();
        y.zero();
        if (rok && 16 * c + 8 * h < a.dh) {
            x.load(dout + oo + 16 * c + 8 * h);
            y.load(out + oo + 16 * c + 8 * h);
        }
        x.terms(df.f[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) D += x.at(e) * y.at(e);
    }
    D += half_swap(D);
    const int qi = head_div(a, rok ? r : 0), head = kvh * a.G + (rok ? r : 0) - qi * a.G;
    const long lrow = ((long)i * a.H + head) * a.lq + qi;
    const float lr = rok ? lse[lrow] : -INFINITY;
    const bool none = lr == -INFINITY;
    const float l2 = none ? INFINITY : lr * LOG2E;
    if (rok && kw == 0 && h == 0 && sp == 0) delta[lrow] = D;

    if (a.keep && k0 < kend) {
        const int last = last_kept(a.keep + s.keep, k0, kend, C::NTH);
        if (lane == 0) sh[wave] = last;
        __syncthreads();
        kend = k0;
#pragma unroll
        for (int w = 0; w < NW * KS; ++w) kend = max(kend, sh[w]);
        kend = __builtin_amdgcn_readfirstlane(kend);
        kv.kend = kend;
    }
    const int nt = kend > k0 ? (kend - k0 + C::BK - 1) / C::BK : 0;

    floatx16 g[DH / 32];
#pragma unroll
    for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) g[dt][e] = 0.f;
    auto tile = [&](int t, const __bf16* Ks, const float* kf) {
        const __bf16* Vs = Ks + C::TILE;
#pragma unroll 1
        for (int j = 0; j < KT / 32; ++j) {
            const int kr = kw * KT + 32 * j, row0 = k0 + t * C::BK + kr;
            if (row0 >= kend) break;
            const bool masked = a.keep || row0 + 32 > kend;
            floatx16 sc = mma_rows<T, DH, DH == 128, PS>(Ks + kr * Lds<DH, DH == 128>::ST, qf, lane);
            const floatx16 dp = mma_rows<T, DH, DH == 128, PS>(Vs + kr * Lds<DH, DH == 128>::ST, df, lane);
            if (masked) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 f = *reinterpret_cast<const float4*>(kf + kr + 8 * e + 4 * h);
                    sc[4 * e] += f.x; sc[4 * e + 1] += f.y; sc[4 * e + 2] += f.z; sc[4 * e + 3] += f.w;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e)
                sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], a.scale2, -l2)) * (dp[e] - D);
            mma_tr<T, DH, DH == 128, PS>(Ks + kr * Lds<DH, DH == 128>::ST, sc, g, lane);
        }
    };
    if (nt > 0) {
        kv.store(tiles, tiles + C::TILE, kfs, tid);
        if (nt > 1) kv.fetch(k0 + C::BK, tid);
        __syncthreads();
    }
    for (int t = 0; t < nt; ++t) {
        tile(t, tiles, kfs);
        __syncthreads();
        if (t + 1 < nt) {
            kv.store(tiles, tiles + C::TILE, kfs, tid);
            if (t + 2 < nt) kv.fetch(k0 + (t + 2) * C::BK, tid);
            __syncthreads();
        }
    }
    if constexpr (KS > 1) {
        float* jb = reinterpret_cast<float*>(smem);
        if (kw > 0) {
            float* p = jb + (size_t)((kw - 1) * NW + qw) * DH * 32;
#pragma unroll
            for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) p[(dt * 16 + e) * 64 + lane] = g[dt][e];
        }
        __syncthreads();
        for (int w = 1; w < KS && kw == 0; ++w) {
            const float* p = jb + (size_t)((w - 1) * NW + qw) * DH * 32;
#pragma unroll
            for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) g[dt][e] += p[(dt * 16 + e) * 64 + lane];
        }
        __syncthreads();
        if (kw > 0) return;
    }
    if (none) {
#pragma unroll
        for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) g[dt][e] = 0.f;
    }
    if (nsplit > 1) {
        if (rok) store_row<float, DH>(part + ((long)sp * a.n * a.H * a.lq + lrow) * a.dh, g, 1.f, a.dh, h);
        return;
    }
    Out<T, DH>::query_rows(a, a.q, dq + s.q, kvh, qt * C::BQ + 32 * qw, rows, g, a.scale,
                           reinterpret_cast<T*>(smem) + qw * Out<T, DH>::WAVE, lane);
}

// dK and dV: a workgroup owns 32 NK keys of one kv head, a wave 32 of them, and
// walks the flattened query rows in tiles of QS * QT (QS waves share a key
// block and split each tile).  S = Q K^T and dP = dO V^T with keys on lanes;
// dV^T += dO^T P and dK^T += Q^T dS read dO and Q transposed from LDS.
template <typename T, int DH, int NK, int QS, int QT> struct DkvCfg {
    static constexpr int NTH = 64 * NK * QS, BKEY = 32 * NK, BQ = QT * QS;
    static constexpr int TILE = tile_elems<T, DH, DH == 128, BQ>();
    static constexpr size_t PAIR = 4 * (size_t)TILE;   // bytes
    static constexpr size_t JOIN = (size_t)NK * (QS - 1) * 2 * DH * 32 * sizeof(float);
    static constexpr size_t OUT = (size_t)NK * Out<T, DH>::WAVE * sizeof(T);   // the rows' way out
    static constexpr size_t BUFS = max3(PAIR, JOIN, OUT);
    // 128 wide in bf16, the values' rows stay in LDS: with them, dK and dV in
    // registers two waves a SIMD would spill (558 us against 460, 16 packed samples of up to 1 501 x 4 003)
    static constexpr bool VLDS = sizeof(T) == 2 && DH == 128 && QS == 1;
    static constexpr size_t VROWS = VLDS ? (size_t)BKEY * Lds<DH, DH == 128>::ST * 2 : 0;
    static constexpr size_t LDS = BUFS + VROWS + 2 * BQ * sizeof(float) + 16;
};

// OWN: D_i made here from o and do (nothing of the dQ kernel's is read)
template <typename T, int DH, int NK, int QS, int QT, bool OWN>
__device__ __forceinline__ void dkv_body(const XArgs& a, const Grads<T>& g, const Share& w, int nsplit,
                                         int split_rows, char* smem) {
    typedef DkvCfg<T, DH, NK, QS, QT> C;
    typedef Stage<T, DH, DH == 128, C::BQ, C::NTH> St;
    __bf16* tiles = reinterpret_cast<__bf16*>(smem);
    float* lss = reinterpret_cast<float*>(smem + C::BUFS + C::VROWS);   // log-sum-exp and D of the buffer's rows
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const int kwv = wave % NK, qs = wave / NK;
    const int i = w.i, kt = w.tile, sp = w.sp, kvh = w.kvh;
    const Sample s = sample_of(a, i);
    const T *q = g.q, *k = g.k, *v = g.v, *out = g.out, *dout = g.dout;
    const float *lse = g.lse, *delta = g.delta;
    T *dk = g.dk, *dv = g.dv;
    float* part = g.part;
    const int kall = a.k_off ? s.kl : a.lk;     // padded rows past k_len get zeros
    if (kt * C::BKEY >= kall) return;
    const int key = kt * C::BKEY + 32 * kwv + (lane & 31);
    const bool kin = key < kall;
    const bool kok = key < s.kl && (!a.keep || a.keep[s.keep + key] != 0.f);

    typedef Lds<DH, DH == 128> L;
    Row<T, DH> kfr, vfr;
    __bf16* Vl = reinterpret_cast<__bf16*>(smem + C::BUFS) + 32 * kwv * L::ST;
    const long ko = s.k + (kin ? (long)key * a.k.sl + (long)kvh * a.k.sh : 0);
    const long vo = s.v + (kin ? (long)key * a.v.sl + (long)kvh * a.v.sh : 0);
    kfr.load(k + ko, kok, a.dh, h);
    vfr.load(v + vo, kok, a.dh, h);
    if constexpr (C::VLDS) {     // this wave's 32 rows, read by itself alone
#pragma unroll
        for (int c = 0; c < DH / 16; ++c)
            *reinterpret_cast<bf16x8*>(Vl + L::chunk_at(lane & 31, h, c)) = vfr.f[c][0];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    floatx16 gk[DH / 32], gv[DH / 32];
#pragma unroll
    for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) gk[dt][e] = gv[dt][e] = 0.f;

    // rows [r0, rows) of this split; a block that keeps no key has no gradient
    const int r0 = sp * split_rows;
    const int rows = __syncthreads_or(kok) ? min(s.ql * a.G, r0 + split_rows) : 0;
    const int nt = rows > r0 ? (rows - r0 + C::BQ - 1) / C::BQ : 0;
    St qs_, ds_, os_;
    float lr = 0.f, dr = 0.f;
    int rown = 0;     // rows of the fetched tile
    auto fetch = [&](int t) {
        const int row0 = r0 + t * C::BQ;
        rown = rows - row0;
        qs_.load_q(a, a.q, q + s.q, kvh, row0, rows, tid);
        ds_.load_q(a, a.o, dout + s.o, kvh, row0, rows, tid);
        if constexpr (OWN) os_.load_q(a, a.o, out + s.o, kvh, row0, rows, tid);
        if (tid < C::BQ) {
            const int r = min(row0 + tid, rows - 1);
            const int qi = head_div(a, r), head = kvh * a.G + r - qi * a.G;
            const long lrow = ((long)i * a.H + head) * a.lq + qi;
            lr = lse[lrow];
            if constexpr (!OWN) dr = delta[lrow];
        }
    };
    auto store = [&](__bf16* Qs, float* ls) {
        // Past the end q's last row stays, which the log-sum-exp of +inf below takes
        // out: its scores are infinite only where the row's own are, where zeros
        // against a key of -inf would make NaN of that key's gradients.
        qs_.store_q(Qs, tid, C::BQ, a.dh);
        ds_.store_q(Qs + C::TILE, tid, rown, a.dh);
        if (tid < C::BQ) {
            // exp2(s - inf) = 0: rows past the end, and rows that keep no key, add nothing
            const bool live = tid < rown;
            ls[tid] = live && lr != -INFINITY ? lr * LOG2E : INFINITY;
            if constexpr (!OWN) ls[C::BQ + tid] = live ? dr : 0.f;
        }
        if constexpr (OWN) {
            // a row's chunks lie in CPR neighbouring lanes
#pragma unroll
            for (int c = 0; c < St::NCH; ++c) {
                float D = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) D += ds_.r[c].at(e) * os_.r[c].at(e);
                if (tid % St::CPR * 8 >= a.dh) D = 0.f;
#pragma unroll
                for (int o = 1; o < St::CPR; o <<= 1) D += __shfl_xor(D, o, 64);
                const int row = tid / St::CPR + c * St::RPP;
                if (tid % St::CPR == 0) ls[C::BQ + row] = row < rown ? D : 0.f;
            }
        }
    };
    auto tile = [&](int t, const __bf16* Qs, const float* ls) {
        const __bf16* Ds = Qs + C::TILE;
        const float* dl = ls + C::BQ;
#pragma unroll 1
        for (int j = 0; j < QT / 32; ++j) {
            const int qr = qs * QT + 32 * j;
            if (r0 + t * C::BQ + qr >= rows) break;
            floatx16 p = mma_rows<T, DH, DH == 128, St::PS>(Qs + qr * Lds<DH, DH == 128>::ST, kfr, lane);
            floatx16 d;
            if constexpr (C::VLDS) d = mma_rows_lds<DH, DH == 128>(Ds + qr * L::ST, Vl, lane);
            else d = mma_rows<T, DH, DH == 128, St::PS>(Ds + qr * L::ST, vfr, lane);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float4 lf = *reinterpret_cast<const float4*>(ls + qr + 8 * e + 4 * h);
                const float4 df = *reinterpret_cast<const float4*>(dl + qr + 8 * e + 4 * h);
                const float lv[4] = {lf.x, lf.y, lf.z, lf.w}, dv4[4] = {df.x, df.y, df.z, df.w};
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    // a masked key's lane goes along: its columns are cleared at the end
                    const float pe = __builtin_amdgcn_exp2f(fmaf(p[4 * e + x], a.scale2, -lv[x]));
                    p[4 * e + x] = pe;
                    d[4 * e + x] = pe * (d[4 * e + x] - dv4[x]);
                }
            }
            mma_tr<T, DH, DH == 128, St::PS>(Ds + qr * Lds<DH, DH == 128>::ST, p, gv, lane);
            mma_tr<T, DH, DH == 128, St::PS>(Qs + qr * Lds<DH, DH == 128>::ST, d, gk, lane);
        }
    };
    if (nt > 0) {
        fetch(0);
        store(tiles, lss);
        if (nt > 1) fetch(1);
        __syncthreads();
    }
    for (int t = 0; t < nt; ++t) {
        tile(t, tiles, lss);
        __syncthreads();
        if (t + 1 < nt) {
            store(tiles, lss);
            if (t + 2 < nt) fetch(t + 2);
            __syncthreads();
        }
    }
    if constexpr (QS > 1) {
        float* jb = reinterpret_cast<float*>(smem);
        __syncthreads();
        if (qs > 0) {
            float* p = jb + (size_t)((qs - 1) * NK + kwv) * 2 * DH * 32;
#pragma unroll
            for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    p[(dt * 16 + e) * 64 + lane] = gk[dt][e];
                    p[DH * 32 + (dt * 16 + e) * 64 + lane] = gv[dt][e];
                }
        }
        __syncthreads();
        for (int w = 1; w < QS && qs == 0; ++w) {
            const float* p = jb + (size_t)((w - 1) * NK + kwv) * 2 * DH * 32;
#pragma unroll
            for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    gk[dt][e] += p[(dt * 16 + e) * 64 + lane];
                    gv[dt][e] += p[DH * 32 + (dt * 16 + e) * 64 + lane];
                }
        }
        __syncthreads();
        if (qs > 0) return;
    }
    if (!kok) {   // a masked key's gradient is zero, whatever the rows hold
#pragma unroll
        for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) gk[dt][e] = gv[dt][e] = 0.f;
    }
    if (nsplit > 1) {
        const long R = (long)a.n * a.KV * a.lk, row = ((long)i * a.KV + kvh) * a.lk + key;
        if (kin) {
            store_row<float, DH>(part + ((long)sp * 2 * R + row) * a.dh, gk, 1.f, a.dh, h);
            store_row<float, DH>(part + ((long)sp * 2 * R + R + row) * a.dh, gv, 1.f, a.dh, h);
        }
        return;
    }
    const int key0 = kt * C::BKEY + 32 * kwv;
    T* ws = reinterpret_cast<T*>(smem) + kwv * Out<T, DH>::WAVE;
    Out<T, DH>::key_rows(dk + s.k + (long)kvh * a.k.sh, a.k.sl, key0, kall, a.dh, gk, a.scale, ws, lane);
    Out<T, DH>::key_rows(dv + s.v + (long)kvh * a.v.sh, a.v.sl, key0, kall, a.dh, gv, 1.f, ws, lane);
}

template <typename T, int DH, int NW, int KS, int KT>
__global__ __launch_bounds__(64 * NW * KS, (bwd_waves<T, DH, KS>())) void xattn_dq_kernel(const XArgs a,
        const Grads<T> p, int qtiles, int nsplit, int split_keys) {
    typedef DqCfg<T, DH, NW, KS, KT> C;
    extern __shared__ __align__(256) char smem[];
    const bool sorted = a.sorted && nsplit == 1;
    const auto tiles = [&](const Sample& x) { return (x.ql * a.G + C::BQ - 1) / C::BQ; };
    const Place pl = place_of(a, sorted, blockIdx.x, gridDim.x, a.KV * qtiles * nsplit,
                              [](const Sample& x) { return x.kl; }, [&](const Sample& x) { return tiles(x) * a.KV; });
    if (pl.i < 0) return;
    const int qtn = sorted ? tiles(sample_of(a, pl.i)) : qtiles;
    dq_body<T, DH, NW, KS, KT>(a, p, {pl.i, pl.rest % qtn, pl.rest / qtn % nsplit, pl.rest / qtn / nsplit}, nsplit,
                               split_keys, smem);
}

template <typename T, int DH, int NK, int QS, int QT>
__global__ __launch_bounds__(64 * NK * QS, (bwd_waves<T, DH, QS>())) void xattn_dkv_kernel(const XArgs a,
        const Grads<T> p, int ktiles, int nsplit, int split_rows) {
    typedef DkvCfg<T, DH, NK, QS, QT> C;
    extern __shared__ __align__(256) char smem[];
    const bool sorted = a.sorted && nsplit == 1;
    const auto tiles = [&](const Sample& x) { return ((a.k_off ? x.kl : a.lk) + C::BKEY - 1) / C::BKEY; };
    const Place pl = place_of(a, sorted, blockIdx.x, gridDim.x, a.KV * ktiles * nsplit,
                              [](const Sample& x) { return x.ql; }, [&](const Sample& x) { return tiles(x) * a.KV; });
    if (pl.i < 0) return;
    const int ktn = sorted ? tiles(sample_of(a, pl.i)) : ktiles;
    dkv_body<T, DH, NK, QS, QT, false>(a, p, {pl.i, pl.rest % ktn, pl.rest / ktn % nsplit, pl.rest / ktn / nsplit},
                                       nsplit, split_rows, smem);
}

// Both in one launch, a sample's head's workgroups of either kind next to each
// other: what one reads the other finds in the caches, and a small problem's two
// halves run side by side (43 samples of 78 x 151, 40 wide, bf16, forward and
// backward: 19 us against 24).
template <typename T, int DH, int NW, int KS, int KT, int NK, int QS, int QT>
__global__ __launch_bounds__(256, (bwd_waves<T, DH, (KS > QS ? KS : QS)>())) void xattn_bwd_kernel(const XArgs a,
        const Grads<T> p, int qtiles, int ktiles) {
    static_assert(NW * KS == 4 && NK * QS == 4, "256 threads");
    extern __shared__ __align__(256) char smem[];
    const int per = qtiles + ktiles, l = xcd_block(blockIdx.x, gridDim.x), u = l / per, t = l - u * per;
    const int i = u / a.KV, kvh = u - i * a.KV;
    if (t < qtiles) dq_body<T, DH, NW, KS, KT>(a, p, {i, t, 0, kvh}, 1, 0x7fffffff, smem);
    else dkv_body<T, DH, NK, QS, QT, true>(a, p, {i, t - qtiles, 0, kvh}, 1, 0x7fffffff, smem);
}

// adds the splits' parts of dq, or of dk and dv, in split order: 4 columns a thread
template <typename T>
__global__ __launch_bounds__(256) void xattn_sum_q_kernel(const XArgs a, const float* __restrict__ part,
        T* __restrict__ dq, int nsplit) {
    const int c4 = a.dh / 4;
    const long R = (long)a.n * a.H * a.lq, at = (long)blockIdx.x * 256 + threadIdx.x, row = at / c4;
    if (row >= R) return;
    const int c = (int)(at - row * c4) * 4;
    const int qi = (int)(row % a.lq), head = (int)(row / a.lq % a.H), i = (int)(row / a.lq / a.H);
    const Sample s = sample_of(a, i);
    if (qi >= s.ql) return;
    float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int p = 0; p < nsplit; ++p) {
        const float4 x = *reinterpret_cast<const float4*>(part + (p * R + row) * a.dh + c);
        g.x += x.x; g.y += x.y; g.z += x.z; g.w += x.w;
    }
    st4(dq + s.q + (long)qi * a.q.sl + (long)head * a.q.sh + c, g.x * a.scale, g.y * a.scale, g.z * a.scale,
        g.w * a.scale);
}
template <typename T>
__global__ __launch_bounds__(256) void xattn_sum_kv_kernel(const XArgs a, const float* __restrict__ part,
        T* __restrict__ dk, T* __restrict__ dv, int nsplit) {
    const int c4 = a.dh / 4;
    const long R = (long)a.n * a.KV * a.lk, at = (long)blockIdx.x * 256 + threadIdx.x, both = at / c4;
    if (both >= 2 * R) return;
    const bool isv = both >= R;
    const long row = isv ? both - R : both;
    const int c = (int)(at - both * c4) * 4;
    const int key = (int)(row % a.lk), kvh = (int)(row / a.lk % a.KV), i = (int)(row / a.lk / a.KV);
    const Sample s = sample_of(a, i);
    if (key >= (a.k_off ? s.kl : a.lk)) return;
    float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int p = 0; p < nsplit; ++p) {
        const float4 x = *reinterpret_cast<const float4*>(part + (2 * p * R + both) * a.dh + c);
        g.x += x.x; g.y += x.y; g.z += x.z; g.w += x.w;
    }
    if (isv) st4(dv + s.v + (long)key * a.v.sl + (long)kvh * a.v.sh + c, g.x, g.y, g.z, g.w);
    else
        st4(dk + s.k + (long)key * a.k.sl + (long)kvh * a.k.sh + c, g.x * a.scale, g.y * a.scale, g.z * a.scale,
            g.w * a.scale);
}

// ------------------------------------------------------------------- host
// Waves along a workgroup's rows (or keys); the rest of the four split the other
// axis.  Four along the other axis take a tile of 128 rows, which in fp32 (three
// planes) fits LDS up to 64 wide.
int waves_for(long rows, bool bf16, int dh) { return rows <= 32 && (bf16 || dh <= 64) ? 1 : rows <= 64 ? 2 : 4; }

// workgroups of four waves that run at once
long at_once(const PtcgCrossAttn* d) { return (d->bf16 || d->dh <= 64 ? 2L : 1L) * cu_count(); }

// Whether the waves of few rows stay without partners along the keys: with more
// workgroups than run at once, smaller ones fill the CUs as well, wait for fewer
// waves at a barrier and join nothing.  Forward: 8 192 x 64 x 97, 64 wide, bf16
// 223 us against 245; 512 of them fp32 50 against 53, 128 wide 115 against 154;
// 2 000 x 8 x 150, 8 heads, fp32 264 against 733 (a tile of four waves' keys
// leaves LDS for one workgroup a CU).  In bf16 a long walk of one wave costs more
// than that (200 x 8 heads, one row, 1 000 keys: 90 us against 78).
bool lone_waves(const PtcgCrossAttn* d, int waves, long blocks) {
    return waves < 4 && blocks > at_once(d) && (!d->bf16 || d->lk <= 512);
}

// whether workgroups go by place_of's order: more of them than run at once
bool sorted_places(const PtcgCrossAttn* d, long blocks) {
    return d->n > 1 && d->n <= 64 && (d->q_off || d->k_off || d->k_len) && blocks > at_once(d);
}

// Splits of a long axis (keys; rows for dk and dv), where the other axis' work-
// groups leave CUs idle: `per_cu` workgroups a CU, at least two tiles each, and
// only from so many tiles on that the joining launch costs less than it saves
// (an fp32 tile takes twice a bf16 one's time).
struct Split { int n, len; };
Split split_of(long blocks, int len, int tile, int per_cu, bool bf16) {
    Split p = {1, len > 0 ? len : 1};
    const int cu = cu_count(), tiles = pt_cdiv(len, tile);
    if (blocks >= cu || blocks <= 0 || tiles < (bf16 ? 6 : 4)) return p;
    const long want = (per_cu * (long)cu + blocks - 1) / blocks;
    const int per = pt_cdiv(tiles, want < tiles / 2 ? want : tiles / 2);
    p.len = per * tile;
    p.n = pt_cdiv(len, p.len);
    return p;
}

// The forward takes four workgroups a CU: samples differ in length, and the
// shorter ones' last splits have nothing to do (two in fp32 128 wide, as many as
// run at once).  Up to 32 rows, in fp32 128 wide 64, against 1 024 keys and more go
// in lone waves that each walk a split of their own (one row against 50 001 keys,
// 4 samples, 8 heads on 2: 128 wide bf16 40 us against 43, fp32 123 against 163; 64
// wide bf16 24 against 28, fp32 49 against 76).  Fewer keys, or more rows, are
// joined as fast in LDS (6 samples of 8 x 667, 8 heads, fp32 15.0 us against 16.5;
// 2 of 60 x 8 000, bf16 18.3 against 20.3).
struct Plan { int nw, qtiles; Split s; bool sorted, lone; };
Plan fwd_plan(const PtcgCrossAttn* d) {
    Plan p;
    const long rows = (long)d->lq * (d->heads / d->kv_heads);
    p.nw = waves_for(rows, d->bf16, d->dh);
    p.qtiles = pt_cdiv(rows, 32 * p.nw);
    const long blocks = (long)d->n * d->kv_heads * p.qtiles;
    p.lone = d->lk >= 1024 && (p.nw == 1 || (p.nw == 2 && !d->bf16 && d->dh > 64));
    p.s = split_of(blocks, d->lk, p.lone ? 32 : p.nw == 1 ? 128 : 64, d->bf16 || d->dh <= 64 ? 4 : 2, d->bf16);
    if (p.s.n == 1) p.lone = lone_waves(d, p.nw, blocks);
    p.sorted = sorted_places(d, blocks);
    return p;
}
// backward: keys split for dq, rows for dk and dv
struct BwdPlan {
    int nw, nk;
    bool qlone, klone;      // waves without partners along the other axis
    bool both;              // one launch for both
    bool sorted;
    Split q, k;
    int64_t delta, part;    // workspace floats
};
BwdPlan bwd_plan(const PtcgCrossAttn* d) {
    BwdPlan p;
    const long G = d->heads / d->kv_heads, rows = d->lq * G, pairs = (long)d->n * d->kv_heads;
    p.nw = waves_for(rows, d->bf16, d->dh);
    p.nk = waves_for(d->lk, d->bf16, d->dh);
    long qb = pairs * pt_cdiv(rows, 32 * p.nw), kb = pairs * pt_cdiv(d->lk, 32 * p.nk);
    p.qlone = lone_waves(d, p.nw, qb);
    if (p.qlone) p.nw = 2;      // one of them as in the forward gains nothing: its registers spill
    // dk and dv with few keys (500 x 64 x 60, 8 heads, 64 wide: bf16 77 us against
    // 99, both gradients), or rows of one tile, whose staging two waves share as
    // well as four (2 000 x 8 x 150, bf16: 471 against 608; not 128 wide, where two
    // waves' spill: 200 samples of 1 x 1 000, 604 against 520)
    p.klone = kb > at_once(d) && (d->lk <= 64 || (rows <= 32 && d->dh <= 64));
    if (p.klone) {
        p.nk = 2;
        kb = pairs * pt_cdiv(d->lk, 64);
    }
    p.q = split_of(qb, d->lk, p.nw == 1 ? 128 : 64, 2, d->bf16);
    p.k = split_of(kb, (int)rows, p.nk == 1 ? 128 : 64, 2, d->bf16);
    p.sorted = sorted_places(d, qb > kb ? qb : kb);
    // One launch up to three rounds of workgroups (128 x 64 x 97, 4 heads, 64 wide,
    // fp32: 38 us against 43 of two launches); of more, the two kernels' own shapes
    // win (512 of them: 151 against 133).  128 wide the pair's registers do not
    // suffice: in bf16 it spills (150 samples of 39 x 78, 8 heads on one kv head,
    // forward and backward: 69 us against 46), in fp32 the compiler moved staging
    // offsets to accumulation registers where only the lanes with a query row run,
    // and the other lanes' later tiles were lost.
    p.both = rows > 0 && d->lk > 0 && p.q.n == 1 && p.k.n == 1 && p.nw > 1 && p.nk > 1 && !p.sorted && !p.qlone &&
             !p.klone && qb + kb <= 3 * at_once(d) && d->dh <= 64;
    const int64_t R = (int64_t)d->n * d->heads * d->lq, RK = pairs * d->lk;
    p.delta = (R + 3) / 4 * 4;
    const int64_t q = p.q.n > 1 ? p.q.n * R * d->dh : 0, k = p.k.n > 1 ? p.k.n * 2 * RK * d->dh : 0;
    p.part = q > k ? q : k;      // dq's are added up before dk's and dv's are made
    return p;
}

int check_desc(const PtcgCrossAttn* d, const char* who) {
    PT_REQUIRE(d, "%s: null descriptor", who);
    PT_REQUIRE(d->n >= 0 && d->lq >= 0 && d->lk >= 0, "%s: negative size n=%d lq=%d lk=%d", who, d->n, d->lq, d->lk);
    PT_REQUIRE(d->heads >= 1 && d->kv_heads >= 1 && d->heads % d->kv_heads == 0,
               "%s: %d heads over %d kv heads", who, d->heads, d->kv_heads);
    PT_REQUIRE(d->dh >= 8 && d->dh <= 128 && d->dh % 8 == 0, "%s: head width %d is not a multiple of 8 up to 128", who,
               d->dh);
    PT_REQUIRE(d->bf16 == 0 || d->bf16 == 1, "%s: bf16=%d", who, d->bf16);
    PT_REQUIRE(d->scale > 0.f && d->scale < 1e30f, "%s: scale must be positive and finite", who);
    PT_REQUIRE(!(d->k_off && d->k_len), "%s: packed keys (k_off) take no k_len", who);
    PT_REQUIRE(!d->keep || d->k_off || d->n <= 1 || d->keep_sn >= 0, "%s: negative keep stride", who);
    const int e = d->bf16 ? 8 : 4;
    PT_REQUIRE(layout_ok(d->q, e) && layout_ok(d->k, e) && layout_ok(d->v, e) && layout_ok(d->o, e),
               "%s: strides must be non-negative multiples of 16 bytes", who);
    PT_REQUIRE((d->k.sl | d->v.sl) < (1 << 22), "%s: key rows 2^22 elements apart or more", who);
    const int64_t G = d->heads / d->kv_heads, rows = (int64_t)d->lq * G;
    PT_REQUIRE(rows * G < (1LL << 32) && rows < (1LL << 31) - 256 && d->lk < (1 << 30),
               "%s: lq=%d lk=%d with %d heads a kv head is too long", who, d->lq, d->lk, (int)G);
    // a bounded tile reads zeros past its rows, which holds for rows that do not
    // reach into one another
    PT_REQUIRE((d->lk <= 1 && !d->k_off) ||
                   ((d->k.sl == 0 || d->k.sl >= d->dh) && (d->v.sl == 0 || d->v.sl >= d->dh)),
               "%s: key rows overlap", who);
    // a launch holds fewer than 2^32 threads, 256 a tile of 128 rows or keys
    PT_REQUIRE((double)d->n * d->kv_heads * (double)(rows / 128 + d->lk / 128 + 2) < (double)(1 << 24) &&
                   (double)d->n * d->heads * d->lq < 4294967296.0,
               "%s: too many tiles", who);
    return PTCG_OK;
}

XArgs to_args(const PtcgCrossAttn* d, bool sorted) {
    XArgs a;
    a.n = d->n; a.lq = d->lq; a.lk = d->lk; a.H = d->heads; a.KV = d->kv_heads;
    a.G = d->heads / d->kv_heads; a.dh = d->dh;
    a.gmagic = (unsigned)((1ULL << 32) / a.G + 1);
    a.scale = d->scale; a.scale2 = d->scale * LOG2E;
    a.q = d->q; a.k = d->k; a.v = d->v; a.o = d->o;
    if (d->lk <= 1 && !d->k_off) a.k.sl = a.v.sl = d->dh;     // one row: any stride was given
    a.q_off = d->q_off; a.k_off = d->k_off; a.k_len = d->k_len;
    a.keep = d->keep; a.keep_sn = d->keep_sn;
    a.sorted = sorted;
    return a;
}

template <typename T, int DH, int NW, int KS, int KT>
int launch_fwd(const XArgs& a, const Plan& p, const void* q, const void* k, const void* v, void* out, float* lse,
               float* part, hipStream_t s) {
    typedef FwdCfg<T, DH, NW, KS, KT> C;
    auto kern = xattn_fwd_kernel<T, DH, NW, KS, KT>;
    PT_TRY(lds_attr(kern, C::LDS));
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.n * a.KV * (long)p.qtiles * p.s.n)), dim3(C::NTH), C::LDS, s, a,
                       static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                       static_cast<T*>(out), lse, part, p.qtiles, p.s.n, p.s.len);
    PT_LAUNCH_CHECK();
    if (p.s.n > 1) {
        constexpr int NG = JOIN_NTH / (DH / 4);
        int per_row = 1;
        while (per_row < NG && per_row * 4 < p.s.n) per_row *= 2;     // four splits a group
        hipLaunchKernelGGL((xattn_join_kernel<T, DH / 4>), dim3(pt_cdiv((long)a.n * a.H * a.lq, NG / per_row)),
                           dim3(JOIN_NTH), 0, s, a, part, static_cast<T*>(out), lse, p.s.n, per_row);
        PT_LAUNCH_CHECK();
    }
    return PTCG_OK;
}

template <typename T, int DH>
int fwd_nw(const XArgs& a, const Plan& p, const void* q, const void* k, const void* v, void* out, float* lse,
           float* part, hipStream_t s) {
    if constexpr (sizeof(T) == 2 || DH <= 64)
        if (p.nw == 1)
            return p.lone ? launch_fwd<T, DH, 1, 1, 32>(a, p, q, k, v, out, lse, part, s)
                          : launch_fwd<T, DH, 1, 4, 32>(a, p, q, k, v, out, lse, part, s);
    if (p.nw == 2)
        return p.lone ? launch_fwd<T, DH, 2, 1, 32>(a, p, q, k, v, out, lse, part, s)
                      : launch_fwd<T, DH, 2, 2, 32>(a, p, q, k, v, out, lse, part, s);
    return launch_fwd<T, DH, 4, 1, 64>(a, p, q, k, v, out, lse, part, s);
}

template <typename T, int DH, int NW, int KS, int KT>
int launch_dq(const XArgs& a, const BwdPlan& p, const Grads<T>& g, hipStream_t s) {
    typedef DqCfg<T, DH, NW, KS, KT> C;
    auto kern = xattn_dq_kernel<T, DH, NW, KS, KT>;
    PT_TRY(lds_attr(kern, C::LDS));
    const int qtiles = pt_cdiv((long)a.lq * a.G, C::BQ);
    hipLaunchKernelGGL(kern, dim3((unsigned)((long)a.n * a.KV * qtiles * p.q.n)), dim3(C::NTH), C::LDS, s, a, g,
                       qtiles, p.q.n, p.q.len);
    PT_LAUNCH_CHECK();
    if (p.q.n > 1) {
        hipLaunchKernelGGL(xattn_sum_q_kernel<T>, dim3(pt_cdiv((long)a.n * a.H * a.lq * (a.dh / 4), 256)), dim3(256),
                           0, s, a, g.part, g.dq, p.q.n);
        PT_LAUNCH_CHECK();
    }
    return PTCG_OK;
}

template <typename T, int DH, int NK, int QS, int QT>
int launch_dkv(const XArgs& a, const BwdPlan& p, const Grads<T>& g, hipStream_t s) {
    typedef DkvCfg<T, DH, NK, QS, QT> C;
    auto kern = xattn_dkv_kernel<T, DH, NK, QS, QT>;
    PT_TRY(lds_attr(kern, C::LDS));
    const int ktiles = pt_cdiv(a.lk, C::BKEY);
    hipLaunchKernelGGL(kern, dim3((unsigned)((long)a.n * a.KV * ktiles * p.k.n)), dim3(C::NTH), C::LDS, s, a, g,
                       ktiles, p.k.n, p.k.len);
    PT_LAUNCH_CHECK();
    if (p.k.n > 1) {
        hipLaunchKernelGGL(xattn_sum_kv_kernel<T>, dim3(pt_cdiv(2L * a.n * a.KV * a.lk * (a.dh / 4), 256)), dim3(256),
                           0, s, a, g.part, g.dk, g.dv, p.k.n);
        PT_LAUNCH_CHECK();
    }
    return PTCG_OK;
}

template <typename T, int DH, int NW, int KS, int KT, int NK, int QS, int QT>
int launch_bwd(const XArgs& a, const Grads<T>& g, hipStream_t s) {
    typedef DqCfg<T, DH, NW, KS, KT> CQ;
    typedef DkvCfg<T, DH, NK, QS, QT> CK;
    constexpr size_t LDS = CQ::LDS > CK::LDS ? CQ::LDS : CK::LDS;
    auto kern = xattn_bwd_kernel<T, DH, NW, KS, KT, NK, QS, QT>;
    PT_TRY(lds_attr(kern, LDS));
    const int qtiles = pt_cdiv((long)a.lq * a.G, CQ::BQ), ktiles = pt_cdiv(a.lk, CK::BKEY);
    hipLaunchKernelGGL(kern, dim3((unsigned)((long)a.n * a.KV * (qtiles + ktiles))), dim3(256), LDS, s, a, g, qtiles,
                       ktiles);
    PT_LAUNCH_CHECK();
    return PTCG_OK;
}

template <typename T, int DH>
int bwd(const XArgs& a, const BwdPlan& p, const Grads<T>& g, hipStream_t s) {
    constexpr bool ONE = sizeof(T) == 2 || DH <= 64;      // waves_for
    // the rows of a step of dk / dv: 32 where the registers hold no more on their way
    constexpr int QT = DH * planes<T>() >= 128 ? 32 : 64;
    if constexpr (DH <= 64)
        if (p.both) {
            if (p.nw == 2)
                return p.nk == 2 ? launch_bwd<T, DH, 2, 2, 32, 2, 2, 32>(a, g, s)
                                 : launch_bwd<T, DH, 2, 2, 32, 4, 1, QT>(a, g, s);
            return p.nk == 2 ? launch_bwd<T, DH, 4, 1, 64, 2, 2, 32>(a, g, s)
                             : launch_bwd<T, DH, 4, 1, 64, 4, 1, QT>(a, g, s);
        }
    if (a.lq > 0) {
        if constexpr (ONE)
            if (p.nw == 1) PT_TRY((launch_dq<T, DH, 1, 4, 32>(a, p, g, s)));
        if (p.nw == 2)
            PT_TRY(p.qlone ? (launch_dq<T, DH, 2, 1, 32>(a, p, g, s)) : (launch_dq<T, DH, 2, 2, 32>(a, p, g, s)));
        if (p.nw == 4) PT_TRY((launch_dq<T, DH, 4, 1, 64>(a, p, g, s)));
    }
    if (a.lk > 0) {
        if constexpr (ONE)
            if (p.nk == 1) return launch_dkv<T, DH, 1, 4, 32>(a, p, g, s);
        if (p.nk == 2) return p.klone ? launch_dkv<T, DH, 2, 1, 32>(a, p, g, s) : launch_dkv<T, DH, 2, 2, 32>(a, p, g, s);
        return launch_dkv<T, DH, 4, 1, QT>(a, p, g, s);
    }
    return PTCG_OK;
}
template <typename T>
int bwd_dh(int dh, const XArgs& a, const BwdPlan& p, const void* q, const void* k, const void* v, const void* out,
           const float* lse, const void* dout, void* dq, void* dk, void* dv, float* ws, hipStream_t s) {
    const Grads<T> g = {static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                        static_cast<const T*>(out), static_cast<const T*>(dout), lse, static_cast<T*>(dq),
                        static_cast<T*>(dk), static_cast<T*>(dv), ws, ws + p.delta};
    return dh <= 32 ? bwd<T, 32>(a, p, g, s) : dh <= 64 ? bwd<T, 64>(a, p, g, s) : bwd<T, 128>(a, p, g, s);
}

int64_t ws_need(const PtcgCrossAttn* d, int backward) {
    const int64_t R = (int64_t)d->n * d->heads * d->lq;
    if (backward) {
        const BwdPlan p = bwd_plan(d);
        return (p.delta + p.part) * 4;
    }
    if (R == 0) return 0;
    const Plan p = fwd_plan(d);
    return p.s.n > 1 ? (int64_t)p.s.n * R * (d->dh + 2) * 4 : 0;
}

}  // namespace

extern "C" int64_t ptcg_kernel_cross_attention_ws_bytes(const PtcgCrossAttn* d, int backward) {
    if (check_desc(d, "cross_attention_ws_bytes") != PTCG_OK) return -1;
    return ws_need(d, backward);
}

extern "C" int ptcg_kernel_cross_attention_fwd(const PtcgCrossAttn* d, const void* q, const void* k, const void* v,
                                               void* out, float* lse, void* workspace, int64_t workspace_bytes,
                                               void* stream) {
    PT_TRY(check_desc(d, "cross_attention_fwd"));
    if ((int64_t)d->n * d->lq == 0) return PTCG_OK;
    PT_REQUIRE(q && out && (d->lk == 0 || (k && v)), "cross_attention_fwd: null buffer");
    PT_REQUIRE(al16(q) && al16(k) && al16(v) && al16(out), "cross_attention_fwd: buffers must be 16 B aligned");
    PT_REQUIRE(layout_apart(d->o, d->q_off, d->n, d->lq, d->heads, d->dh),
               "cross_attention_fwd: rows of the output overlap");
    const int64_t need = ws_need(d, 0);
    PT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && al16(workspace)),
               "cross_attention_fwd: workspace of %lld bytes, need %lld (16 B aligned)", (long long)workspace_bytes,
               (long long)need);
    const Plan p = fwd_plan(d);
    const XArgs a = to_args(d, p.sorted);
    float* part = static_cast<float*>(workspace);
    const hipStream_t s = (hipStream_t)stream;
    if (d->bf16)
        return d->dh <= 32   ? fwd_nw<__bf16, 32>(a, p, q, k, v, out, lse, part, s)
               : d->dh <= 64 ? fwd_nw<__bf16, 64>(a, p, q, k, v, out, lse, part, s)
                             : fwd_nw<__bf16, 128>(a, p, q, k, v, out, lse, part, s);
    return d->dh <= 32   ? fwd_nw<float, 32>(a, p, q, k, v, out, lse, part, s)
           : d->dh <= 64 ? fwd_nw<float, 64>(a, p, q, k, v, out, lse, part, s)
                         : fwd_nw<float, 128>(a, p, q, k, v, out, lse, part, s);
}

extern "C" int ptcg_kernel_cross_attention_bwd(const PtcgCrossAttn* d, const void* q, const void* k, const void* v,
                                               const void* out, const float* lse, const void* dout, void* dq,
                                               void* dk, void* dv, void* workspace, int64_t workspace_bytes,
                                               void* stream) {
    PT_TRY(check_desc(d, "cross_attention_bwd"));
    if (d->n == 0 || (d->lq == 0 && d->lk == 0)) return PTCG_OK;
    PT_REQUIRE(d->lq == 0 || (q && out && lse && dout && dq), "cross_attention_bwd: null buffer");
    PT_REQUIRE(d->lk == 0 || (k && v && dk && dv), "cross_attention_bwd: null buffer");
    PT_REQUIRE(al16(q) && al16(k) && al16(v) && al16(out) && al16(dout) && al16(dq) && al16(dk) && al16(dv),
               "cross_attention_bwd: buffers must be 16 B aligned");
    PT_REQUIRE(layout_apart(d->q, d->q_off, d->n, d->lq, d->heads, d->dh),
               "cross_attention_bwd: rows of dq overlap (a broadcast q has no gradient layout)");
    PT_REQUIRE(layout_apart(d->k, d->k_off, d->n, d->lk, d->kv_heads, d->dh) &&
                   layout_apart(d->v, d->k_off, d->n, d->lk, d->kv_heads, d->dh),
               "cross_attention_bwd: rows of dk or dv overlap (broadcast keys have no gradient layout)");
    const int64_t need = ws_need(d, 1);
    PT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && al16(workspace)),
               "cross_attention_bwd: workspace of %lld bytes, need %lld (16 B aligned)", (long long)workspace_bytes,
               (long long)need);
    const BwdPlan p = bwd_plan(d);
    const XArgs a = to_args(d, p.sorted);
    float* ws = static_cast<float*>(workspace);
    const hipStream_t s = (hipStream_t)stream;
    return d->bf16 ? bwd_dh<__bf16>(d->dh, a, p, q, k, v, out, lse, dout, dq, dk, dv, ws, s)
                   : bwd_dh<float>(d->dh, a, p, q, k, v, out, lse, dout, dq, dk, dv, ws, s);
}
