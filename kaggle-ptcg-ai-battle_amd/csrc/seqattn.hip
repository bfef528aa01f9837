// Causal attention along time, with a window and a few first tokens that stay
// visible: new rows over a cache of pages (chunks and single tokens), and whole
// sequences with their gradient.
//
// Row i of place p_i sees the keys j <= p_i with p_i - j < window or j < sinks:
//   s_ij = scale q_i . k_j,  m_i = max_j s_ij,  l_i = sum_j exp(s_ij - m_i),
//   o_i = sum_j exp(s_ij - m_i) v_j / l_i,  lse_i = m_i + log l_i,
// in one pass over the keys that any row of a tile sees: tiles of the first tokens,
// then tiles from the first row's window on to the last row's place.
// A row that sees no key, or whose seen scores are all -inf: o = 0, lse = -inf.
//
// Rows, fragments and products as in the attention to other states (attn_tiles.h):
// the G = heads / kv_heads query heads of a kv head are one matrix of rows, query r
// / G and head r % G of row r; S^T = K Q^T leaves a query on a lane and its
// scores in registers, which are an operand of O^T = V^T P^T as they are.
#include "attn_tiles.h"

#include <limits.h>

#include <type_traits>

namespace {

// the descriptors as the kernels take them
struct SArgs {
    int n, lq, H, KV, G, dh;
    unsigned gmagic;              // head_div
    float scale, scale2;          // scale2 = scale * log2(e): exponentials are exp2
    int window, sinks;            // window: INT_MAX where there is none
    PtcgHeadLayout q, k, v, o;    // k, v: rows of sequences, or of pages
    const int *q_off, *len;
    // pages
    const int* table;
    long table_sn;
    int pages, page, per_seq;
    int all_rows;                 // rows of the packed matrices
    unsigned pmagic;              // key / page = umulhi(key, pmagic) >> pshift (page > 1)
    int pshift;
};

// A sequence: element offsets of row 0, its live rows, the rows that are written (a
// padded one's dead rows too), its keys, and the place of row 0.
struct Seq { long q, o, k, v; const int* table; int ql, rows, kl, p0; };

// Counts come from device memory: they are held to the host's bounds.
template <bool PAGED> __device__ __forceinline__ Seq seq_of(const SArgs& a, int i) {
    Seq s = {};
    s.ql = s.rows = a.lq;
    if (a.q_off) {
        const int r0 = max(0, a.q_off[i]);
        s.ql = s.rows = max(0, min(a.lq, min(a.q_off[i + 1], a.all_rows) - r0));
        s.q = r0 * a.q.sl; s.o = r0 * a.o.sl;
        if constexpr (!PAGED) { s.k = r0 * a.k.sl; s.v = r0 * a.v.sl; }
    } else {
        s.q = i * a.q.sn; s.o = i * a.o.sn;
        if constexpr (!PAGED) {
            s.k = i * a.k.sn; s.v = i * a.v.sn;
            if (a.len) s.ql = max(0, min(a.lq, a.len[i]));
        }
    }
    s.kl = s.ql;
    if constexpr (PAGED) {
        const int n = max(0, a.len[i]);
        s.p0 = n - s.ql;
        s.kl = min(n, a.per_seq * a.page);
        s.table = a.table + i * a.table_sn;
    }
    return s;
}

// Key blocks (of BK keys) that rows of places plo .. phi see: the first hb, then
// nt - hb from block tw on; keys from kend on are seen by none of them.
struct Range {
    int hb, tw, nt, kend;
    __device__ __forceinline__ int block(int t) const { return t < hb ? t : tw + t - hb; }
};
template <int BK> __device__ __forceinline__ Range range_of(const SArgs& a, int plo, int phi, int kl) {
    Range r = {0, 0, 0, 0};
    r.kend = min(phi + 1, kl);
    if (r.kend <= 0) return r;
    const int te = (r.kend + BK - 1) / BK;
    r.tw = min(max(0, max(plo, 0) - a.window + 1) / BK, te);
    r.hb = min((min(a.sinks, r.kend) + BK - 1) / BK, r.tw);
    r.nt = r.hb + te - r.tw;
    return r;
}
// places of the live rows among flattened rows r0 .. r1 - 1; none: hi < 0
struct Places { int lo, hi; };
__device__ __forceinline__ Places places_of(const SArgs& a, const Seq& s, int r0, int r1) {
    const int q0 = head_div(a, r0), q1 = min(head_div(a, r1 - 1), s.ql - 1);
    return {s.p0 + q0, q1 < q0 ? -1 : s.p0 + q1};
}

// A workgroup's piece of work: key blocks t0 .. t1 - 1 (of those the tile has) of a row
// tile of a sequence; where the tile is shared with other workgroups, the place of this
// piece among the parts, its tile's number among all and, with the tile's first piece,
// the shared ones' count.
struct Work { int i, qt, t0, t1, part, tile, per, next; };

// Splitting.  Row tiles, each as long as its sequence's longest (K_i key blocks of T_i
// tiles), are laid end to end and cut into `slots` stretches of `per` blocks, one for
// each workgroup that runs at once: however many tiles there are and however they
// differ, all workgroups read the same number of keys.  A stretch may hold the end of a
// tile, whole tiles, and the beginning of one; a tile that is cut leaves a part in each
// of its stretches for the joining kernel: the stretch's first part, or its second
// where the tile begins within the stretch.  The lengths are on the device
// alone: every wave counts for itself, 64 sequences at a time.  (Packed sequences that are not
// cut are gone through in the same way to find a tile: 16 384 of up to 12 rows, 4 heads of 64, fp32,
// take 2.0 ms forward, padded 0.26; 512 of up to 97 67 us and 63.)
// (Counts of blocks fit 32 bits: the host splits nothing else.)
struct Cut { int all, per, tiles; };

// inclusive sum over the lanes, in the vector unit alone (by way of LDS the planning took 2 us
// of a token's call)
__device__ __forceinline__ int lane_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);      // 1, 2, 4, 8 lanes up in rows of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);      // lane 15 to row 1, 47 to row 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);      // lane 31 to rows 2 and 3
    return x;
}

template <bool PAGED, int BQ, int BK, bool ALIGNED> struct Deal {
    int t, k, to, tt;      // of 64 sequences on the lanes: tiles, blocks; pieces and tiles up to and with it
    int per;               // blocks a stretch, or a piece at most; 0: a piece is a tile
    // pieces of a tile, or blocks where tiles are laid end to end
    __device__ __forceinline__ int units() const { return per == 0 ? 1 : ALIGNED ? (k + per - 1) / per : k; }
    __device__ __forceinline__ void load(const SArgs& a, int i0) {
        const int i = i0 + (threadIdx.x & 63);
        t = 0;
        k = 1;
        if (i < a.n) {
            const Seq s = seq_of<PAGED>(a, i);
            t = (s.rows * a.G + BQ - 1) / BQ;
            const Places p = {s.p0, s.p0 + s.ql - 1};
            // the blocks of all rows, and of a tile of rows in a window; a tile that sees nothing is one too
            k = range_of<BK>(a, p.lo, p.hi, s.kl).nt;
            if (a.window < INT_MAX - 4 * BQ)
                k = min(k, (a.window + (BQ + a.G - 2) / a.G) / BK + 2 + (min(a.sinks, s.kl) + BK - 1) / BK);
            k = max(k, 1);
        }
    }
    __device__ __forceinline__ void place() {
        to = lane_sum(t * units());
        tt = lane_sum(t);
    }
    // up to 64 sequences stay on the lanes
    __device__ __forceinline__ Cut cut(const SArgs& a, int slots, int least) {
        int all = 0, tiles = 0;
        for (int i0 = 0; i0 < a.n; i0 += 64) {
            load(a, i0);
            all += __builtin_amdgcn_readlane(lane_sum(t * k), 63);
            tiles += __builtin_amdgcn_readlane(lane_sum(t), 63);
        }
        if constexpr (ALIGNED) {
            // sum t ceil(k / per) <= slots for certain from here on (slots > tiles); fewer by search
            per = max(1, (int)((long)all / max(1, slots - tiles)) + 1);
            if (a.n <= 64) {
                int lo = max(1, all / slots);
                while (per - lo > 1 + lo / 16) {
                    const int mid = lo + (per - lo) / 2;
                    if (__builtin_amdgcn_readlane(lane_sum(t * ((k + mid - 1) / mid)), 63) <= slots) per = mid;
                    else lo = mid;
                }
            }
            per = max(per, least);
            all = slots;
        } else {
            per = max(least, (int)(((long)all + slots - 1) / slots));
        }
        if (a.n <= 64) place();
        return {all, per, tiles};
    }
    // the work from b on, up to end
    __device__ __forceinline__ Work at(const SArgs& a, int b, int end) {
        int before = 0, tiles = 0;
        for (int i0 = 0; i0 < a.n; i0 += 64) {
            if (per == 0 || a.n > 64) {
                load(a, i0);
                place();
            }
            const int hi = before + to;
            const unsigned long long m = __ballot(b >= hi - t * units() && b < hi);
            if (m) {
                const int w = __builtin_ctzll(m);
                const int uw = __builtin_amdgcn_readlane(units(), w), nt = __builtin_amdgcn_readlane(t, w);
                const int kw = __builtin_amdgcn_readlane(k, w);
                const int off = b - (__builtin_amdgcn_readlane(hi, w) - nt * uw), q = off / uw, u = off - q * uw;
                Work r;
                r.i = i0 + w;
                r.qt = nt - 1 - q;                          // the last tile first: its rows see the most
                r.tile = tiles + __builtin_amdgcn_readlane(tt, w) - nt + q;
                r.part = -1;
                r.per = per;
                r.next = end;
                if (per == 0) {
                    r.t0 = 0;
                    r.t1 = INT_MAX;
                } else if constexpr (ALIGNED) {
                    r.per = (kw + uw - 1) / uw;
                    r.t0 = u * r.per;
                    r.t1 = r.t0 + r.per;
                    if (uw > 1) r.part = 2 * b;
                } else {
                    r.t0 = u;
                    r.t1 = min(kw, u + (end - b));
                    r.next = b + (r.t1 - u);
                    const int first = b - u;                 // the tile's first block
                    if (first / per != (first + kw - 1) / per) r.part = b / per * 2 + (b % per != 0);
                }
                return r;
            }
            before += __builtin_amdgcn_readlane(to, 63);
            tiles += __builtin_amdgcn_readlane(tt, 63);
        }
        return {-1, 0, 0, 0, -1, 0, 0, end};
    }
};
// the same in scalar registers, as it is one for all lanes
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ Work uniform(const Work& w) {
    return {uniform(w.i), uniform(w.qt), uniform(w.t0), uniform(w.t1), uniform(w.part), uniform(w.tile), uniform(w.per),
            uniform(w.next)};
}
__device__ __forceinline__ Cut uniform(const Cut& c) { return {uniform(c.all), uniform(c.per), uniform(c.tiles)}; }
// What the joining kernel is told: a tile's sequence, number in it, first part and how many
// (1: nothing to join); before the first, how many tiles there are.
struct Joint { int i, qt, part, parts; };
// a part's rows, unnormalised, then their maxima and sums
__host__ __device__ constexpr long part_floats(int prow, int dh) { return ((long)prow * (dh + 2) + 3) / 4 * 4; }

// Scores of keys that a row of place p does not see become -inf, whatever they are:
// register e is key k0 + 8 (e / 4) + e % 4.  last: the lesser of p and the last key.
__device__ __forceinline__ void hide(const SArgs& a, floatx16& s, int k0, int p, int last) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int j = k0 + 8 * (e / 4) + e % 4;
        const bool see = j <= last && (p - j < a.window || j < a.sinks);
        s[e] = see ? s[e] : -INFINITY;
    }
}
// the same of keys of no page: 32 keys' bits
__device__ __forceinline__ void hide_bits(floatx16& s, unsigned none, int h) {
    const unsigned mine = none >> 4 * h;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = mine & 1u << (8 * (e / 4) + e % 4) ? -INFINITY : s[e];
}
// whether some row of places lo .. hi does not see all of keys k0 .. k0 + nk - 1, or none
// of them does
__device__ __forceinline__ bool some_hidden(const SArgs& a, int k0, int nk, int lo, int hi) {
    return k0 + nk - 1 > lo || (hi - k0 >= a.window && k0 + nk > a.sinks);
}
__device__ __forceinline__ bool all_hidden(const SArgs& a, int k0, int nk, int lo, int hi) {
    return k0 > hi || (lo - (k0 + nk - 1) >= a.window && k0 >= a.sinks);
}

// the page of a sequence that key lies in
__device__ __forceinline__ int page_of(const SArgs& a, int key) {
    return a.page == 1 ? key : (int)(__umulhi((unsigned)key, a.pmagic) >> a.pshift);      // exact below 2^31
}
// (kend > 0.  For keys that are not there the last one's entry is read; no branches, here
// and around loads: regions of some lanes in loops that fill the registers cost more, and
// the compiler has lost registers at their ends.)
__device__ __forceinline__ int entry_of(const SArgs& a, const Seq& s, int key, int kend) {
    return s.table[page_of(a, min(key, kend - 1))];
}
// p where ok, else an address that can be read
template <typename T> __device__ __forceinline__ const T* where(bool ok, const T* p, const T* other) {
    return ok ? p : other;
}
// The kernel's first argument, read again from memory where this is called: around a loop
// over pieces of work the compiler would hold all of it in scalar registers, which do
// not suffice.
__device__ __forceinline__ const SArgs& args_again() {
    typedef const __attribute__((address_space(4))) SArgs* ArgP;
    ArgP p = (ArgP)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const SArgs*)p;
}

// the larger of both halves' values
__device__ __forceinline__ float half_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// the thread's number, for the compiler not the same each time: nothing made from it is
// held in registers around the pieces of work
__device__ __forceinline__ int thread_again() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// A running softmax of the rows on lanes: m2, a bound of the scores (s scale2) so far
// that was their maximum when it was last set, and this half's sum l of exp2(s scale2 -
// m2).  Where a score passes m2 by 8 or more, m2 moves up and what is summed is
// rescaled; below, exponentials reach 2^8, which costs fp32 sums and bf16 products
// nothing, and the rescaling (a multiplication per output) falls away in most tiles.
constexpr float SLACK = 8.f;
template <int DH> struct Soft {
    float m2, l;
    floatx16 o[DH / 32];
    __device__ __forceinline__ void init() {
        m2 = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
    }
    // a lane's largest score
    template <int N> static __device__ __forceinline__ float top(const floatx16 (&sc)[N]) {
        float mt = -INFINITY;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) mt = fmaxf(mt, sc[j][e]);
        return mt;
    }
    // what is summed is rescaled where new scores, at most mt on this lane, pass the bound
    __device__ __forceinline__ void raise(float mt, float scale2) {
        mt = half_max(mt);
        const float mn = fmaxf(m2, mt * scale2);
        if (__any(mn > m2 + SLACK)) {
            const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m2 - mn);
            l *= al;
#pragma unroll
            for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[dt][e] *= al;
            m2 = mn;
        }
    }
    // scores to exponentials
    __device__ __forceinline__ void exps(floatx16& sc, float scale2) {
        const float ms = m2 == -INFINITY ? 0.f : m2;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], scale2, -ms));
            l += sc[e];
        }
    }
    template <int N> __device__ __forceinline__ void step(floatx16 (&sc)[N], float scale2) {
        raise(top(sc), scale2);
#pragma unroll
        for (int j = 0; j < N; ++j) exps(sc[j], scale2);
    }
    // elements e0 .. e0 + n - 1 of 32 keys' scores to exponentials, and those to the values'
    // operand
    __device__ __forceinline__ void exps_of(floatx16& sc, bf16x8 (&p)[2], float scale2, float ms, int e0, int n) {
#pragma unroll
        for (int e = e0; e < e0 + n; ++e) {
            sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], scale2, -ms));
            l += sc[e];
            p[e / 8][e % 8] = (__bf16)sc[e];
        }
    }
};

// The order of instructions is the source's from here to the next such line: left to
// itself the compiler reads an operand just before its product and waits, or keeps so
// many on their way that registers spill.
__device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0); }

// S^T of 64 keys in LDS (bf16), a product at a time
template <int DH>
__device__ __forceinline__ void scores(const __bf16* ks, const Row<__bf16, DH>& q, floatx16 (&sc)[2], int lane) {
    typedef Lds<DH, false> L;
    constexpr int N = DH / 8, AHEAD = 4;       // operands on their way
    bf16x8 x[N];
    auto read = [&](int i) {
        x[i] = *reinterpret_cast<const bf16x8*>(ks + 32 * (i & 1) * L::ST + L::chunk_at(lane & 31, lane >> 5, i >> 1));
    };
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[j][e] = 0.f;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) read(i);
    pin();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        sc[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[i], q.f[i >> 1][0], sc[i & 1], 0, 0, 0);
        if (i + AHEAD < N) read(i + AHEAD);
        pin();
    }
}

// o^T += V^T P of 32 keys in LDS (bf16) and their exponentials p, in the same way
template <int DH, class Side>
__device__ __forceinline__ void values(const __bf16* vs, const bf16x8 (&p)[2], floatx16 (&o)[DH / 32], int lane,
                                       Side side) {
    typedef __attribute__((address_space(3))) bf16x4* lds4;
    typedef Lds<DH, false> L;
    constexpr int N = DH / 16, DT = DH / 32, AHEAD = 2;
    const int i15 = lane & 15, r0 = 4 * (lane >> 5) + (i15 >> 2), ch = 2 * (lane >> 4 & 1) + (i15 >> 1 & 1);
    bf16x4 u[N], w[N];
    auto read = [&](int i) {
        const __bf16* q = vs + 16 * (i / DT) * L::ST + 4 * (i15 & 1);
        u[i] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(q + L::group_at(r0, ch, i % DT)));
        w[i] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(q + L::group_at(r0 + 8, ch, i % DT)));
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) read(i);
    pin();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bf16x8 x = bf16x8{u[i][0], u[i][1], u[i][2], u[i][3], w[i][0], w[i][1], w[i][2], w[i][3]};
        o[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, p[i / DT], o[i % DT], 0, 0, 0);
        if (i + AHEAD < N) read(i + AHEAD);
        side(i);
        pin();
    }
}

// What a tile's rows come to: their output, or their split's part for the joining
// kernel (unnormalised, with maximum and sum).  rows: rows of the sequence.
template <typename T, int DH, int BQ>
__device__ __forceinline__ void finish(const SArgs& a, const Seq& s, int i, int kvh, int tile0, int row0, Soft<DH>& f,
                                       T* out, float* lse, float* part, int prow, T* ws, int lane) {
    const int rows = s.rows * a.G, r = row0 + (lane & 31), h = lane >> 5;
    const bool rok = r < rows;
    if (part) {
        if (!rok) return;
        store_row<float, DH>(part + (long)(r - tile0) * a.dh, f.o, 1.f, a.dh, h);
        if (h == 0) {
            float* ml = part + (long)prow * a.dh + (r - tile0) * 2;
            ml[0] = f.m2;
            ml[1] = f.l;
        }
        return;
    }
    // nothing seen, or every seen score -inf: the sum is 0 (scores of NaN leave the
    // maximum at -inf too, but a sum of NaN)
    const bool none = f.m2 == -INFINITY && f.l == 0.f;
    if (none) {
#pragma unroll
        for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) f.o[dt][e] = 0.f;
    }
    if (lse && rok && h == 0) {
        const int qi = head_div(a, r), head = kvh * a.G + r - qi * a.G;
        lse[((long)i * a.H + head) * a.lq + qi] = none ? -INFINITY : f.m2 * LN2 + logf(f.l);
    }
    Out<T, DH>::query_rows(a, a.o, out + s.o, kvh, row0, rows, f.o, none ? 0.f : 1.f / f.l, ws, lane);
}

// ---------------------------------------------------------- tiles of many rows
// A tile of BK keys and values on its way through registers into LDS; keys that
// are not there (past kend, of no page) enter as zeros and, of no page, with a
// flag of -inf.  Rows of one matrix: bounded loads; of pages: each row by its own
// page-table entry, looked up a block ahead.
template <typename T, int DH, bool PAD, int BK, int NTH, bool PAGED> struct KvRegs {
    typedef Stage<T, DH, PAD, BK, NTH> St;
    static_assert(BK <= NTH, "a thread per key flag");
    St k, v;
    RowBuf kb, vb;
    int ko, vo;
    int ent[St::NCH], entf;
    float kfr;
    unsigned ok;
    __device__ __forceinline__ void init(const SArgs& a, const Seq& s, const T* kp, const T* vp, int kvh, int tid) {
        if constexpr (!PAGED) {
            constexpr int es = sizeof(T);
            kb = {reinterpret_cast<const char*>(kp + s.k + (long)kvh * a.k.sh), (int)a.k.sl * es, a.dh * es};
            vb = {reinterpret_cast<const char*>(vp + s.v + (long)kvh * a.v.sh), (int)a.v.sl * es, a.dh * es};
            ko = St::first(kb.ld, a.dh, tid);
            vo = St::first(vb.ld, a.dh, tid);
        }
    }
    // the page-table entries that fetch(block) will need
    __device__ __forceinline__ void look(const SArgs& a, const Seq& s, int block, int kend, int tid) {
        if constexpr (PAGED) {
#pragma unroll
            for (int i = 0; i < St::NCH; ++i) ent[i] = entry_of(a, s, block * BK + tid / St::CPR + i * St::RPP, kend);
            entf = entry_of(a, s, block * BK + tid, kend);
        }
    }
    // q: an address that can be read
    __device__ __forceinline__ void fetch(const SArgs& a, const Seq& s, const T* kp, const T* vp, const T* q, int kvh,
                                          int block, int kend, int tid) {
        if constexpr (!PAGED) {
            const auto rk = kb.rows(block * BK, kend, BK), rv = vb.rows(block * BK, kend, BK);
            k.load(rk, ko, kb.ld);
            v.load(rv, vo, vb.ld);
        } else {
            const int col = tid % St::CPR * 8;
            ok = 0;
            kfr = ((tid < BK) & (block * BK + tid < kend) & ((unsigned)entf >= (unsigned)a.pages)) ? -INFINITY : 0.f;
#pragma unroll
            for (int i = 0; i < St::NCH; ++i) {
                const int key = block * BK + tid / St::CPR + i * St::RPP;
                // what is not there: any address that can be read, dropped in store
                const bool there = (key < kend) & (col < a.dh) & ((unsigned)ent[i] < (unsigned)a.pages);
                const int off = key - page_of(a, key) * a.page;
                ok |= there ? 1u << i : 0u;
                k.r[i].load(where(there, kp + (long)ent[i] * a.k.sn + (long)off * a.k.sl + (long)kvh * a.k.sh + col, q));
                v.r[i].load(where(there, vp + (long)ent[i] * a.v.sn + (long)off * a.v.sl + (long)kvh * a.v.sh + col, q));
            }
        }
    }
    __device__ __forceinline__ void store(__bf16* Ks, __bf16* Vs, float* kf, int* bad, int tid) const {
#pragma unroll
        for (int i = 0; i < St::NCH; ++i) {
            k.put(Ks, tid, i, !PAGED || (ok >> i & 1));
            v.put(Vs, tid, i, !PAGED || (ok >> i & 1));
        }
        if constexpr (PAGED)
            if (tid < BK) {
                kf[tid] = kfr;
                if (kfr != 0.f) *bad = 1;      // from this tile on the flags are looked at
            }
    }
};

// 16 bytes a lane from memory into LDS, lane L's to base + 16 L; zeros past the
// descriptor's end.  Issued from assembly so that the compiler does not tie LDS reads
// to loads on their way; who reads waits (arrived) and meets the others at a barrier.
// The load may not read a descriptor's word within five wait states of its v_readfirstlane,
// nor M0 within one of its move, and the compiler adds none in here: the move and four more.
// (M0 is named as written: the warning that it is a reserved register is what this file means.)
#pragma clang diagnostic ignored "-Winline-asm"
#define PT_WAIT_M0 "s_nop 3\n\t"
typedef int intx4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void to_lds(intx4 rs, const __bf16* base, int off) {
    const unsigned at = (unsigned)(uintptr_t)base;      // LDS offset: low bits of the generic address
    asm volatile("s_mov_b32 m0, %0\n\t" PT_WAIT_M0 "buffer_load_dwordx4 %1, %2, 0 offen lds"
                 :: "s"(__builtin_amdgcn_readfirstlane(at)), "v"(off), "s"(rs) : "memory", "m0");
}
// this wave's pieces have arrived
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A tile of BK key or value rows by 16-byte pieces straight into LDS (bf16): waves bring WR
// rows each that lie in one matrix, or in one page (whose size is a multiple of
// them).  A piece's place in LDS is its lane's, so the lane chooses the chunk that
// belongs there.
template <int DH, int BK, int NW, bool PAGED> struct KvDma {
    typedef Lds<DH, false> L;
    static constexpr int CPR = DH / 8, RPI = 64 / CPR;                     // rows an instruction
    static constexpr int WR = BK / NW, NI = WR / RPI;      // rows, instructions a wave
    static_assert(BK % NW == 0 && WR % RPI == 0, "whole instructions");
    int off[NI], ld, width, row;
    const char* base;
    // rows of layout l; row0: the sequence's first (one matrix)
    __device__ __forceinline__ void init(const SArgs& a, const Seq& s, const __bf16* x, int kvh, const PtcgHeadLayout& l,
                                         long row0, int tid) {
        const int lane = tid & 63;
        row = __builtin_amdgcn_readfirstlane(tid >> 6) * WR;
        ld = (int)l.sl * 2;
        width = 2 * a.dh;
        base = reinterpret_cast<const char*>(x + (PAGED ? 0 : row0) + (long)kvh * l.sh);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = i * RPI + lane / CPR, c = (lane % CPR) ^ L::swz(row + r);
            off[i] = 8 * c < a.dh ? r * ld + 16 * c : PT_NOWHERE;
        }
    }
    static __device__ __forceinline__ intx4 rsrc(const char* p, int bytes) {
        const unsigned long long x = (unsigned long long)p;
        return intx4{__builtin_amdgcn_readfirstlane((int)(unsigned)x),
                     __builtin_amdgcn_readfirstlane((int)(unsigned)(x >> 32)), __builtin_amdgcn_readfirstlane(bytes),
                     0x00020000};
    }
    // ent: the page that the wave's rows lie in
    __device__ __forceinline__ void fetch(const SArgs& a, const PtcgHeadLayout& l, int block, int kend, int ent,
                                          __bf16* to) const {
        const int key = block * BK + row;
        int n = max(0, min(kend - key, WR));
        const char* p = base;
        if constexpr (PAGED) {
            const bool is = (unsigned)ent < (unsigned)a.pages;
            if (!is) n = 0;
            const long e = is ? ent : 0, at = is ? key - page_of(a, key) * a.page : 0;
            p += (e * l.sn + at * l.sl) * 2;
        } else {
            p += (long)key * ld;
        }
        const intx4 rs = rsrc(p, n ? (n - 1) * ld + width : 0);
#pragma unroll
        for (int i = 0; i < NI; ++i) to_lds(rs, to + (row + i * RPI) * L::ST, off[i]);
    }
};

template <typename T, int DH, int NW, bool DMA> struct TileCfg {
    static constexpr int NTH = 64 * NW, BQ = 32 * NW, BK = 64;
    static constexpr int TILE = tile_elems<T, DH, false, BK>();
    static constexpr size_t PAIR = (DMA ? 2 : 1) * 4 * (size_t)TILE;   // bytes
    static constexpr size_t OUT = (size_t)NW * Out<T, DH>::WAVE * sizeof(T);
    static constexpr size_t BUFS = PAIR > OUT ? PAIR : OUT;
    static constexpr size_t LDS = BUFS + BK * sizeof(float) + 64;
};
template <typename T, int DH> constexpr int waves_simd() { return sizeof(T) == 2 || DH <= 64 ? 2 : 1; }

// Workgroup b of `pairs` (sequence, kv head) pairs with `per` pieces each, the longest
// first.  Workgroups go to the 8 XCDs in turn: a pair's pieces stay on one XCD, whose L2
// then holds their keys, pairs are dealt out to the XCDs one by one (sequences
// differ in length: with neighbours on one XCD a third of the CUs' time was idle), and an XCD
// takes so many pairs at once that their long pieces come before their short ones.
// Where pairs are few or of lengths that only the device knows (spread), a pair's pieces go
// to all XCDs instead (8 packed sequences of 2 heads, one pair or two an XCD: dk and dv
// 756 us against 570).
struct Share { int pair, piece; };
__device__ __forceinline__ Share share_of(int b, int pairs, int per, bool spread) {
    const int full = spread || pairs < 32 ? 0 : pairs >> 3, x = b & 7, idx = b >> 3;
    if (idx < full * per) {
        const int most = (127 + per) / per, g = idx / (most * per), n = min(most, full - g * most), r = idx - g * most * per;
        return {(g * most + r % n) * 8 + x, r / n};
    }
    const int r = b - 8 * full * per, pair = r / per;     // one after the other, over all XCDs
    return {8 * full + pair, r - pair * per};
}

// How workgroups get their work, as the host decided: even: every sequence has qtiles row
// tiles and nothing is split; split: `slots` stretches a kv head; else a row tile each
// (tiles: at most so many).
struct Plan { int slots, tiles, qtiles, least, prow; bool even, split; };

// A workgroup's work, one call of f after the other; js: what the joining kernel is told.
template <bool PAGED, int BQ, int BK, bool ALIGNED, class F>
__device__ __forceinline__ void work_through(const SArgs& a, const Plan& pl, Joint* js, F f) {
    Deal<PAGED, BQ, BK, ALIGNED> d;
    d.per = 0;
    Work w;
    int kvh, b = 0, end = 1;
    if (pl.even) {
        const Share sh = share_of(blockIdx.x, a.n * a.KV, pl.qtiles, false);
        kvh = sh.pair % a.KV;
        w = {sh.pair / a.KV, pl.qtiles - 1 - sh.piece, 0, INT_MAX, -1, 0, 0, 1};
    } else if (!pl.split) {
        kvh = blockIdx.x % a.KV;             // unequal tiles are spread over the XCDs
        b = blockIdx.x / a.KV;
        end = b + 1;
    } else {
        const int l = xcd_block(blockIdx.x, gridDim.x);
        kvh = l / pl.slots;
        const Cut c = uniform(d.cut(a, pl.slots, pl.least));
        if (l == 0 && threadIdx.x == 0) js[0].i = c.tiles <= pl.tiles ? c.tiles : 0;     // more: q_off does not ascend
        const long first = (long)(l - kvh * pl.slots) * (ALIGNED ? 1 : c.per);      // past the end: no work
        b = first < c.all ? (int)first : c.all;
        end = min(c.all - b, ALIGNED ? 1 : c.per) + b;
    }
    while (b < end) {
        if (!pl.even) w = uniform(d.at(a, b, end));
        if (w.i < 0) break;
        f(w, kvh);
        b = w.next;
        if (b < end) __syncthreads();        // the next one's tiles take the place of these rows' way out
    }
}
// whether a piece of a tile of nt key blocks leaves a part; the tile's first piece notes
// what there is to join
__device__ __forceinline__ bool shared_tile(Joint* js, const Work& w, int kvh, int nt, int tiles) {
    const bool cut = w.part >= 0 && (w.t0 > 0 || nt > w.t1);
    if (w.per > 0 && w.t0 == 0 && w.tile < tiles && kvh == 0 && threadIdx.x == 0)
        js[1 + w.tile] = {w.i, w.qt, w.part, cut ? 1 + (nt - w.t1 + w.per - 1) / w.per : 1};
    return cut;
}

// A workgroup owns 32 NW rows and walks their key blocks (or its split of them).
// DMA: tiles go straight into one of two buffers while the other is worked on, one
// barrier a tile; else through registers into one buffer.  Bound by its products, two
// workgroups a CU taking turns at them: 4 sequences to 2 048 new rows over 30 000 keys, 8 heads of
// 128 on 2, bf16, 542 to 563 us (915 to 950 TFLOP/s).  Whole sequences of 4 096, 2 198, 3 371 and 1 473
// rows padded to 4 096, 8 heads of 128: 143 us (503), bound by unequal tiles: these are not cut where there are
// as many as workgroups run at once, and the longest, of 64 key blocks, takes 1.8 times an XCD's mean load.
// In fp32 the operands' terms and six products a product: 512 sequences up to 97, 4 heads of 64, 62 us.
template <typename T, int DH, int NW, bool PAGED, bool DMA>
__global__ __launch_bounds__(64 * NW, (waves_simd<T, DH>())) void seq_fwd_kernel(const SArgs a_, const T* __restrict__ q,
        const T* __restrict__ k, const T* __restrict__ v, T* __restrict__ out, float* __restrict__ lse,
        float* __restrict__ part, const Plan pl) {
    typedef TileCfg<T, DH, NW, DMA> C;
    typedef KvRegs<T, DH, false, 64, C::NTH, PAGED> Kv;
    constexpr int BK = C::BK, BQ = C::BQ, PS = BK * Lds<DH, false>::ST;
    extern __shared__ __align__(256) char smem[];
    __bf16* tiles = reinterpret_cast<__bf16*>(smem);
    float* kf = reinterpret_cast<float*>(smem + C::BUFS);
    int* bad = reinterpret_cast<int*>(smem + C::LDS - 64);
    Joint* const js = reinterpret_cast<Joint*>(part);      // then the parts
    work_through<PAGED, BQ, BK, false>(a_, pl, js, [&](const Work& w, int kvh) {
    const SArgs& a = args_again();
    const int tid = thread_again(), lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5;
    const Seq s = seq_of<PAGED>(a, w.i);
    const int rows = s.rows * a.G, tile0 = w.qt * BQ;
    const Places pt = places_of(a, s, tile0, min(tile0 + BQ, rows));
    const Range rg = range_of<BK>(a, pt.lo, pt.hi, s.kl);
    const int t0 = w.t0, t1 = min(rg.nt, w.t1);
    const bool joined = shared_tile(js, w, kvh, rg.nt, pl.tiles);
    if (t0 > 0 && t0 >= rg.nt) return;
    if (PAGED && tid == 0) *bad = 0;

    const int r0 = tile0 + 32 * wave, r = r0 + (lane & 31);
    const bool rok = r < rows;
    // rows past the last stand at its place, dead ones see nothing
    const int qr = head_div(a, min(r, rows - 1)), p = s.p0 + qr, last = qr < s.ql ? min(p, rg.kend - 1) : -1;
    const int q0 = __builtin_amdgcn_readfirstlane(qr), q1 = __builtin_amdgcn_readlane(qr, 31);
    const bool live = r0 < rows, sees = live && q0 < s.ql, dead = q1 >= s.ql;
    const int wlo = s.p0 + q0, whi = s.p0 + min(q1, s.ql - 1);
    Row<T, DH> qf;
    qf.load(q + s.q + (rok ? row_off(a, a.q, kvh, r) : 0), rok, a.dh, h);
    Soft<DH> f;
    f.init();

    qf.settle();
    // tile t's block from Ks on; nopage: its keys of no page, by lanes
    auto tile = [&](int t, const __bf16* Ks, unsigned long long nopage) {
        const __bf16* Vs = Ks + C::TILE;
        const int key0 = rg.block(t) * BK;
        if (!sees || all_hidden(a, key0, BK, wlo, whi)) return;
        // a half that is not seen costs no products
        bool half[BK / 32];
        floatx16 sc[BK / 32];
#pragma unroll
        for (int j = 0; j < BK / 32; ++j) {
            half[j] = !all_hidden(a, key0 + 32 * j, 32, wlo, whi);
            if (half[j]) {
                sc[j] = mma_rows<T, DH, false, PS>(Ks + 32 * j * Lds<DH, false>::ST, qf, lane);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[j][e] = -INFINITY;
            }
        }
        if (dead || key0 + BK > rg.kend || some_hidden(a, key0, BK, wlo, whi)) {
#pragma unroll
            for (int j = 0; j < BK / 32; ++j) hide(a, sc[j], key0 + 32 * j + 4 * h, p, last);
        }
        if (PAGED && nopage) {
#pragma unroll
            for (int j = 0; j < BK / 32; ++j) hide_bits(sc[j], (unsigned)(nopage >> 32 * j), h);
        }
        f.step(sc, a.scale2);
#pragma unroll
        for (int j = 0; j < BK / 32; ++j)
            if (half[j]) mma_tr<T, DH, false, PS>(Vs + 32 * j * Lds<DH, false>::ST, sc[j], f.o, lane);
    };
    if constexpr (DMA) {
        static_assert(sizeof(T) == 2 && BK == 64, "");
        typedef KvDma<DH, BK, NW, PAGED> Dma;
        Dma kk, kv;
        kk.init(a, s, k, kvh, a.k, s.k, tid);
        kv.init(a, s, v, kvh, a.v, s.v, tid);
        // the page of the wave's rows of tile t: 64 tiles' on the lanes, looked up at once (a
        // scalar load a tile would make every LDS read behind it wait for it)
        int ents = 0, ents0 = t0 - 64;
        auto entry = [&](int t) {
            if constexpr (PAGED) {
                if (t - ents0 >= 64) {
                    ents0 = t;
                    ents = entry_of(a, s, rg.block(min(t + lane, t1 - 1)) * BK + kk.row, rg.kend);
                }
                return __builtin_amdgcn_readlane(ents, t - ents0);
            }
            return 0;
        };
        auto fetch = [&](int t, __bf16* to) {
            const int e = entry(t);
            kk.fetch(a, a.k, rg.block(t), rg.kend, e, to);
            kv.fetch(a, a.v, rg.block(t), rg.kend, e, to + C::TILE);
        };
        auto lacks = [&](int t) {       // a lane per key
            const int key = rg.block(t) * BK + lane;
            return (key < rg.kend) & ((unsigned)entry_of(a, s, key, rg.kend) >= (unsigned)a.pages);
        };
        if (t0 < t1) {
            fetch(t0, tiles);
            bool some = false;         // any key of no page: only then tiles look for them
            if constexpr (PAGED) {
                for (int t = t0 + wave; t < t1; t += NW) some |= lacks(t);
                some = __syncthreads_or(some);
            }
            constexpr int E = 16 / (DH / 16);       // elements in a product's shadow
            // tile t, at `at` of the two places
            auto turn = [&](int t, auto at) {
                constexpr int AT = decltype(at)::value;
                arrived();
                __syncthreads();       // everyone's pieces of tile t are here, and tile t - 1 is done with
                if (t + 1 < t1) fetch(t + 1, tiles + (1 - AT) * 2 * C::TILE);
                const int key0 = rg.block(t) * BK;
                if (!sees || all_hidden(a, key0, BK, wlo, whi)) return;
                const __bf16 *Ks = tiles + AT * 2 * C::TILE, *Vs = Ks + C::TILE;
                floatx16 sc[2];
                scores<DH>(Ks, qf, sc, lane);
                if (dead || key0 + BK > rg.kend || some_hidden(a, key0, BK, wlo, whi)) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) hide(a, sc[j], key0 + 32 * j + 4 * h, p, last);
                }
                if (PAGED && some) {
                    const unsigned long long nopage = __ballot(lacks(t));
                    if (nopage) {
                        hide_bits(sc[0], (unsigned)nopage, h);
                        hide_bits(sc[1], (unsigned)(nopage >> 32), h);
                    }
                }
                f.raise(f.top(sc), a.scale2);
                const float ms = f.m2 == -INFINITY ? 0.f : f.m2;
                bf16x8 pa[2], pb[2];
                f.exps_of(sc[0], pa, a.scale2, ms, 0, 16);
                // the second half's exponentials in the shadow of the first half's products
                values<DH>(Vs, pa, f.o, lane, [&](int i) { f.exps_of(sc[1], pb, a.scale2, ms, i * E, E); });
                values<DH>(Vs + 32 * Lds<DH, false>::ST, pb, f.o, lane, [](int) {});
            };
            for (int t = t0; t < t1; t += 2) {
                turn(t, std::integral_constant<int, 0>());
                if (t + 1 < t1) turn(t + 1, std::integral_constant<int, 1>());
            }
        }
        __syncthreads();           // the buffers become the rows' way out
    } else {
        __bf16 *Ks = tiles, *Vs = tiles + C::TILE;
        Kv kv;
        kv.init(a, s, k, v, kvh, tid);
        auto fetch = [&](int t) {
            kv.fetch(a, s, k, v, q, kvh, rg.block(t), rg.kend, tid);
            if (t + 1 < t1) kv.look(a, s, rg.block(t + 1), rg.kend, tid);
        };
        if (t0 < t1) {
            kv.look(a, s, rg.block(t0), rg.kend, tid);
            fetch(t0);
            __syncthreads();      // *bad is cleared
            kv.store(Ks, Vs, kf, bad, tid);
            if (t0 + 1 < t1) fetch(t0 + 1);
            __syncthreads();
        }
        for (int t = t0; t < t1; ++t) {
            unsigned long long nopage = 0;
            if (PAGED && *bad) nopage = __ballot(kf[lane] != 0.f);
            tile(t, Ks, nopage);
            __syncthreads();
            if (t + 1 < t1) {
                kv.store(Ks, Vs, kf, bad, tid);
                if (t + 2 < t1) fetch(t + 2);
                __syncthreads();
            }
        }
    }
    f.l += half_swap(f.l);
    float* pp = joined ? part + 4 * (1 + pl.tiles) + ((long)w.part * a.KV + kvh) * part_floats(pl.prow, a.dh) : nullptr;
    if (live)
        finish<T, DH, BQ>(a, s, w.i, kvh, tile0, r0, f, out, lse, pp, pl.prow,
                          reinterpret_cast<T*>(smem) + wave * Out<T, DH>::WAVE, lane);
    });
}

// ------------------------------------------------------------ few rows
// Up to 32 rows (a token's heads) against their keys: bound by reading the keys.
// Waves of a workgroup take the 32-key blocks in turn and share nothing until the
// end.  A lane holds a key's row as an operand straight from memory; the values go
// through the wave's own part of LDS, to be read transposed.  The next block's rows
// are on their way into the same registers while a block is worked on.  8 tokens over up to
// 131 072 keys, 8 heads of 128 on 2, bf16: 156 us, 4.5 TB/s; 256 over up to 8 000, 8 heads of 64: 224
// us, 4.8 TB/s; 16 over up to 1 000, 4 heads of 64, fp32: 14.4 us, latency.
template <typename T, int DH, int KS> struct TokenCfg {
    static constexpr int NTH = 64 * KS, BQ = 32, BK = 32;
    static constexpr int TILE = tile_elems<T, DH, false, BK>();
    static constexpr size_t VALS = (size_t)KS * TILE * 2;
    static constexpr int JS = DH * 32 + 64;      // floats of a wave's part
    static constexpr size_t LDS = max3(VALS, (size_t)(KS - 1) * JS * sizeof(float), Out<T, DH>::WAVE * sizeof(T));
};

template <typename T, int DH, int KS, bool PAGED>
__global__ __launch_bounds__(64 * KS, (waves_simd<T, DH>())) void seq_token_kernel(const SArgs a_,
        const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, T* __restrict__ out,
        float* __restrict__ lse, float* __restrict__ part, const Plan pl) {
    typedef TokenCfg<T, DH, KS> C;
    typedef Lds<DH, false> L;
    constexpr int BK = C::BK, BQ = C::BQ, PS = BK * L::ST;
    extern __shared__ __align__(256) char smem[];
    Joint* const js = reinterpret_cast<Joint*>(part);      // then the parts
    work_through<PAGED, BQ, BK, true>(a_, pl, js, [&](const Work& w, int kvh) {
    const SArgs& a = args_again();
    const int tid = thread_again(), lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5;
    __bf16* Vs = reinterpret_cast<__bf16*>(smem) + wave * C::TILE;
    const Seq s = seq_of<PAGED>(a, w.i);
    const int rows = s.rows * a.G, tile0 = w.qt * BQ;
    const Places pt = places_of(a, s, tile0, min(tile0 + BQ, rows));
    const Range rg = range_of<BK>(a, pt.lo, pt.hi, s.kl);
    const int t0 = w.t0, t1 = min(rg.nt, w.t1);
    const bool joined = shared_tile(js, w, kvh, rg.nt, pl.tiles);
    if (t0 > 0 && t0 >= rg.nt) return;

    const int r = tile0 + (lane & 31);
    const bool rok = r < rows;
    const int qr = head_div(a, min(r, rows - 1)), p = s.p0 + qr, last = qr < s.ql ? min(p, rg.kend - 1) : -1;
    Row<T, DH> qf;
    qf.load(q + s.q + (rok ? row_off(a, a.q, kvh, r) : 0), rok, a.dh, h);
    Soft<DH> f;
    f.init();

    Chunk<T> kc[DH / 16], vc[DH / 16];
    int ent = 0;
    bool nopage = false, here = false;
    auto look = [&](int t) {
        if constexpr (PAGED) ent = entry_of(a, s, rg.block(t) * BK + (lane & 31), rg.kend);
    };
    auto fetch = [&](int t) {
        const int key = rg.block(t) * BK + (lane & 31);
        bool there = key < rg.kend;
        long ka, va;
        if constexpr (PAGED) {
            nopage = there & ((unsigned)ent >= (unsigned)a.pages);
            there = there & ((unsigned)ent < (unsigned)a.pages);
            const int off = key - page_of(a, key) * a.page;
            ka = (long)ent * a.k.sn + (long)off * a.k.sl;
            va = (long)ent * a.v.sn + (long)off * a.v.sl;
        } else {
            ka = s.k + (long)key * a.k.sl;
            va = s.v + (long)key * a.v.sl;
        }
        // rows and columns that are not there: any address that can be read, then zeros
        const T *kr = k + ka + (long)kvh * a.k.sh + 8 * h, *vr = v + va + (long)kvh * a.v.sh + 8 * h;
#pragma unroll
        for (int c = 0; c < DH / 16; ++c)
            kc[c].load(where(there & (16 * c + 8 * h < a.dh), kr + 16 * c, q));
#pragma unroll
        for (int c = 0; c < DH / 16; ++c)
            vc[c].load(where(there & (16 * c + 8 * h < a.dh), vr + 16 * c, q));
        here = there;
    };
    int t = t0 + wave;
    if (t < t1) {
        look(t);
        fetch(t);
        if (t + KS < t1) look(t + KS);
    }
    for (; t < t1; t += KS) {
        const int key0 = rg.block(t) * BK;
        floatx16 sc[1];
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[0][e] = 0.f;
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) {
            bf16x8 x[planes<T>()];
            kc[c].keep(here & (16 * c + 8 * h < a.dh));
            kc[c].terms(x);
            mma(x, qf.f[c], sc[0]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");     // the last block's values are read
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) {
            bf16x8 x[planes<T>()];
            vc[c].keep(here & (16 * c + 8 * h < a.dh));
            vc[c].terms(x);
#pragma unroll
            for (int pn = 0; pn < planes<T>(); ++pn)
                *reinterpret_cast<bf16x8*>(Vs + pn * PS + L::chunk_at(lane & 31, h, c)) = x[pn];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const unsigned none = PAGED ? (unsigned)__ballot(nopage) : 0;
        if (t + KS < t1) {
            fetch(t + KS);
            if (t + 2 * KS < t1) look(t + 2 * KS);
        }
        hide(a, sc[0], key0 + 4 * h, p, last);
        if (none) hide_bits(sc[0], none, h);
        f.step(sc, a.scale2);
        mma_tr<T, DH, false, PS>(Vs, sc[0], f.o, lane);
    }
    f.l += half_swap(f.l);

    // the waves' parts join in LDS, in wave order
    if constexpr (KS > 1) {
        __syncthreads();
        float* jb = reinterpret_cast<float*>(smem);
        if (wave > 0) {
            float* x = jb + (size_t)(wave - 1) * C::JS;
#pragma unroll
            for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) x[(dt * 16 + e) * 64 + lane] = f.o[dt][e];
            if (h == 0) {
                x[DH * 32 + lane] = f.m2;
                x[DH * 32 + 32 + lane] = f.l;
            }
        }
        __syncthreads();
        if (wave > 0) return;
        for (int u = 1; u < KS; ++u) {
            const float* x = jb + (size_t)(u - 1) * C::JS;
            const float mw = x[DH * 32 + (lane & 31)], lw = x[DH * 32 + 32 + (lane & 31)];
            const float mn = fmaxf(f.m2, mw), ms = mn == -INFINITY ? 0.f : mn;
            const float f0 = __builtin_amdgcn_exp2f(f.m2 - ms), f1 = __builtin_amdgcn_exp2f(mw - ms);
            f.l = f.l * f0 + lw * f1;
            f.m2 = mn;
#pragma unroll
            for (int dt = 0; dt < DH / 32; ++dt) {
#pragma unroll
                for (int e = 0; e < 16; ++e) f.o[dt][e] = f.o[dt][e] * f0 + x[(dt * 16 + e) * 64 + lane] * f1;
                pin();      // not all the reads at once, whose registers would spill
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // before the parts become the rows' way out
    }
    float* pp = joined ? part + 4 * (1 + pl.tiles) + ((long)w.part * a.KV + kvh) * part_floats(pl.prow, a.dh) : nullptr;
    finish<T, DH, BQ>(a, s, w.i, kvh, tile0, tile0, f, out, lse, pp, pl.prow, reinterpret_cast<T*>(smem), lane);
    });
}

// ---------------------------------------------------------------- joining
// Joins the splits of a row tile: a workgroup takes some rows of a (tile, kv head);
// groups of LG lanes (4 columns each) take a row's splits in turn, per_row groups a
// row, and meet in LDS in group order.  4.0 to 5.5 us for tokens, 16 for a chunk of 8 192 rows
// 128 wide in 57 MB of parts.
constexpr int JOIN_NTH = 512;
template <typename T, int LG, bool PAGED, int BQ>
__global__ __launch_bounds__(JOIN_NTH) void seq_join_kernel(const SArgs a, const float* __restrict__ part,
        T* __restrict__ out, float* __restrict__ lse, const Plan pl, int per_row, int rgroups) {
    constexpr int NG = JOIN_NTH / LG;
    __shared__ float4 sh[JOIN_NTH];
    __shared__ float2 shm[NG];
    const int tid = threadIdx.x, grp = tid / LG, c = tid % LG, g0 = grp & (per_row - 1);
    const int rg_ = blockIdx.x % rgroups, kvh = blockIdx.x / rgroups % a.KV, tile = blockIdx.x / rgroups / a.KV;
    const Joint* js = reinterpret_cast<const Joint*>(part);
    if (tile >= js[0].i) return;
    const Joint w = js[1 + tile];
    if (w.parts <= 1) return;        // made by one workgroup
    const Seq s = seq_of<PAGED>(a, w.i);
    const int rows = s.rows * a.G, tile0 = w.qt * BQ;
    const int row = rg_ * (NG / per_row) + grp / per_row, r = tile0 + row;
    const bool live = row < BQ && r < rows;
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
    if (live) {
        // the first part's place, then the first places of the stretches after it
        const float* p0 = part + 4 * (1 + pl.tiles);
#pragma unroll 4
        for (int u = g0; u < w.parts; u += per_row) {
            const long at = u == 0 ? w.part : ((w.part >> 1) + u) * 2;
            const float* x = p0 + (at * a.KV + kvh) * part_floats(pl.prow, a.dh);
            const float2 e = *reinterpret_cast<const float2*>(x + (long)pl.prow * a.dh + 2 * row);
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            if (4 * c < a.dh) y = *reinterpret_cast<const float4*>(x + (long)row * a.dh + 4 * c);
            add(e.x, e.y, y);
        }
    }
    sh[tid] = acc;
    if (c == 0) shm[grp] = make_float2(m, l);
    __syncthreads();
    if (g0 > 0 || !live) return;
    for (int g = 1; g < per_row; ++g) {
        const float2 e = shm[grp + g];
        add(e.x, e.y, sh[(grp + g) * LG + c]);
    }
    const int qi = head_div(a, r), head = kvh * a.G + r - qi * a.G;
    const bool none = m == -INFINITY && l == 0.f;
    const float f = none ? 0.f : 1.f / l;
    if (none) acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (4 * c < a.dh)
        st4(out + s.o + (long)qi * a.o.sl + (long)head * a.o.sh + 4 * c, acc.x * f, acc.y * f, acc.z * f, acc.w * f);
    if (lse && c == 0) lse[((long)w.i * a.H + head) * a.lq + qi] = none ? -INFINITY : m * LN2 + logf(l);
}

// --------------------------------------------------------------- backward
// With P_ij = exp(s_ij - lse_i) and D_i = do_i . o_i over the pairs that see each other:
//   dv_j = sum_i P_ij do_i,  dS_ij = P_ij (do_i . v_j - D_i),
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,
// dk and dv summed over the query heads that share the kv head, in row order.
template <typename T> struct Grads {
    const T *q, *k, *v, *out, *dout;
    const float* lse;
    T *dq, *dk, *dv;
    float2* stats;
    float* part;
};

// Both products of 32 LDS rows that a tile begins with (bf16): s0 = X0 Y0^T, s1 = X1
// Y1^T, Y1 a lane's rows in registers or (YLDS) in LDS; side(c) goes into step c's shadow.
template <int DH, bool YLDS, class Side>
__device__ __forceinline__ void products(const __bf16* x0, const __bf16* x1, const Row<__bf16, DH>& y0,
                                         const Row<__bf16, DH>& y1, const __bf16* yl, floatx16& s0, floatx16& s1,
                                         int lane, Side side) {
    typedef Lds<DH, false> L;
    constexpr int N = DH / 16, AHEAD = 2;
    bf16x8 a0[N], a1[N], b1[N];
    auto read = [&](int c) {
        const int at = L::chunk_at(lane & 31, lane >> 5, c);
        a0[c] = *reinterpret_cast<const bf16x8*>(x0 + at);
        a1[c] = *reinterpret_cast<const bf16x8*>(x1 + at);
        if constexpr (YLDS) b1[c] = *reinterpret_cast<const bf16x8*>(yl + at);
    };
#pragma unroll
    for (int e = 0; e < 16; ++e) s0[e] = s1[e] = 0.f;
#pragma unroll
    for (int c = 0; c < AHEAD; ++c) read(c);
    pin();
#pragma unroll
    for (int c = 0; c < N; ++c) {
        s0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a0[c], y0.f[c][0], s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a1[c], YLDS ? b1[c] : y1.f[c][0], s1, 0, 0, 0);
        if (c + AHEAD < N) read(c + AHEAD);
        side(c);
        pin();
    }
}

// dQ: the forward's shape.  Per 32 keys S^T and dP^T = V dO^T with queries on
// lanes, dS^T in registers, dQ^T += K^T dS^T.  Also leaves each row's log-sum-exp (in
// units of exp2; +inf for a row that sees nothing) and D_i for the dK / dV kernel, in
// the order of its rows.  D_i is do_i . o_i of the output as it was stored; in bf16 its
// rounding is the largest error of short rows' gradients (9 keys: 3.3e-3 in relative L2, 2.4e-3
// without it), so there D_i is summed along the keys as well, for dK / dV, and for dQ too
// where one tile holds all keys of the rows.  The forward's four sequences, 8 heads of 128, bf16:
// 200 us (540 TFLOP/s in three products; its tiles and their unequal load); 512 sequences up to 97, 4
// heads of 64, fp32: 81 us.
template <typename T, int DH, int NW> struct DqCfg {
    static constexpr bool DMA = sizeof(T) == 2, PAD = DH == 128 && !DMA;
    static constexpr int NTH = 64 * NW, BQ = 32 * NW, BK = 64;
    static constexpr int TILE = tile_elems<T, DH, PAD, BK>();
    static constexpr size_t PAIR = (DMA ? 2 : 1) * 4 * (size_t)TILE;   // bytes
    static constexpr size_t OUT = (size_t)NW * Out<T, DH>::WAVE * sizeof(T);
    static constexpr size_t LDS = PAIR > OUT ? PAIR : OUT;
};
template <typename T, int DH, int NW>
__global__ __launch_bounds__(64 * NW, (waves_simd<T, DH>())) void seq_dq_kernel(const SArgs a_, const Grads<T> g,
                                                                               const Plan pl) {
    typedef DqCfg<T, DH, NW> C;
    typedef KvRegs<T, DH, C::PAD, C::BK, C::NTH, false> Kv;
    typedef Lds<DH, C::PAD> L;
    constexpr int PS = Kv::St::PS, BK = C::BK, BQ = C::BQ;
    extern __shared__ __align__(256) char smem[];
    __bf16* tiles = reinterpret_cast<__bf16*>(smem);
    work_through<false, BQ, BK, false>(a_, pl, nullptr, [&](const Work& w, int kvh) {
    const SArgs& a = args_again();
    const int tid = thread_again(), lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5;
    const Seq s = seq_of<false>(a, w.i);
    const int rows = s.rows * a.G, tile0 = w.qt * BQ;
    if (tile0 >= rows) return;
    const Places pt = places_of(a, s, tile0, min(tile0 + BQ, rows));
    const Range rg = range_of<BK>(a, pt.lo, pt.hi, s.kl);

    const int r0 = tile0 + 32 * wave, r = r0 + (lane & 31);
    const bool rok = r < rows;
    const int qr = head_div(a, min(r, rows - 1)), last = qr < s.ql ? min(qr, rg.kend - 1) : -1;
    const int q0 = __builtin_amdgcn_readfirstlane(qr), q1 = __builtin_amdgcn_readlane(qr, 31);
    const bool live = r0 < rows, sees = live && q0 < s.ql, dead = q1 >= s.ql;
    const int wlo = q0, whi = min(q1, s.ql - 1);

    Row<T, DH> qf, df;
    qf.load(g.q + s.q + (rok ? row_off(a, a.q, kvh, r) : 0), rok, a.dh, h);
    const long oo = s.o + (rok ? row_off(a, a.o, kvh, r) : 0);
    float D = 0.f;
#pragma unroll
    for (int c = 0; c < DH / 16; ++c) {
        Chunk<T> x, y;
        x.zero();
        y.zero();
        if (rok && 16 * c + 8 * h < a.dh) {
            x.load(g.dout + oo + 16 * c + 8 * h);
            y.load(g.out + oo + 16 * c + 8 * h);
        }
        x.terms(df.f[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) D += x.at(e) * y.at(e);
    }
    D += half_swap(D);
    const int qi = head_div(a, rok ? r : 0), head = kvh * a.G + (rok ? r : 0) - qi * a.G;
    const long lrow = ((long)w.i * a.H + head) * a.lq + qi;
    const float lr = rok && qr < s.ql ? g.lse[lrow] : -INFINITY;
    const bool none = lr == -INFINITY;
    const float l2 = none ? INFINITY : lr * LOG2E;
    float Dx = 0.f;      // bf16: D_i again, as sum_j P_ij (do_i . v_j)

    floatx16 acc[DH / 32];
#pragma unroll
    for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;
    qf.settle();
    df.settle();
    // sums: Dx alone
    auto tile = [&](int t, const __bf16* Ks, auto only) {
        constexpr bool sums = decltype(only)::value;
        const __bf16* Vs = Ks + C::TILE;
        // half a tile at a time: with both halves' dS on their way the kernel spills 128 wide
        // (251 us against 204 over the four sequences above)
#pragma unroll 1
        for (int j = 0; j < BK / 32; ++j) {
            const int key0 = rg.block(t) * BK + 32 * j;
            if (!sees || key0 >= rg.kend || all_hidden(a, key0, 32, wlo, whi)) continue;
            floatx16 sc, dp;
            if constexpr (C::DMA) {
                products<DH, false>(Ks + 32 * j * L::ST, Vs + 32 * j * L::ST, qf, df, nullptr, sc, dp, lane, [](int) {});
            } else {
                sc = mma_rows<T, DH, C::PAD, PS>(Ks + 32 * j * L::ST, qf, lane);
                dp = mma_rows<T, DH, C::PAD, PS>(Vs + 32 * j * L::ST, df, lane);
            }
            if (dead || key0 + 32 > rg.kend || some_hidden(a, key0, 32, wlo, whi)) hide(a, sc, key0 + 4 * h, qr, last);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], a.scale2, -l2));
                if constexpr (C::DMA) Dx = fmaf(sc[e], dp[e], Dx);
                if (sums) continue;
                sc[e] *= dp[e] - D;
            }
            if (!sums) mma_tr<T, DH, C::PAD, PS>(Ks + 32 * j * L::ST, sc, acc, lane);
        }
    };
    if constexpr (C::DMA) {
        KvDma<DH, BK, NW, false> kk, kv;
        kk.init(a, s, g.k, kvh, a.k, s.k, tid);
        kv.init(a, s, g.v, kvh, a.v, s.v, tid);
        auto fetch = [&](int t) {
            __bf16* to = tiles + (t & 1) * 2 * C::TILE;
            kk.fetch(a, a.k, rg.block(t), rg.kend, 0, to);
            kv.fetch(a, a.v, rg.block(t), rg.kend, 0, to + C::TILE);
        };
        if (rg.nt > 0) fetch(0);
        for (int t = 0; t < rg.nt; ++t) {
            arrived();
            __syncthreads();       // everyone's pieces of tile t are here, and tile t - 1 is done with
            if (t + 1 < rg.nt) fetch(t + 1);
            if (rg.nt == 1) {      // all keys are here: dq from the better D as well
                tile(t, tiles, std::true_type());
                D = Dx + half_swap(Dx);
                Dx = 0.f;
            }
            tile(t, tiles + (t & 1) * 2 * C::TILE, std::false_type());
        }
        __syncthreads();           // the buffers become the rows' way out
    } else {
        Kv kv;
        kv.init(a, s, g.k, g.v, kvh, tid);
        auto fetch = [&](int t) { kv.fetch(a, s, g.k, g.v, g.q, kvh, rg.block(t), rg.kend, tid); };
        if (rg.nt > 0) {
            fetch(0);
            kv.store(tiles, tiles + C::TILE, nullptr, nullptr, tid);
            if (rg.nt > 1) fetch(1);
            __syncthreads();
        }
        for (int t = 0; t < rg.nt; ++t) {
            tile(t, tiles, std::false_type());
            __syncthreads();
            if (t + 1 < rg.nt) {
                kv.store(tiles, tiles + C::TILE, nullptr, nullptr, tid);
                if (t + 2 < rg.nt) fetch(t + 2);
                __syncthreads();
            }
        }
    }
    if constexpr (C::DMA) D = Dx + half_swap(Dx);
    if (rok && h == 0) g.stats[((long)w.i * a.KV + kvh) * a.lq * a.G + r] = make_float2(l2, D);
    if (!live) return;
    if (none) {
#pragma unroll
        for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;
    }
    Out<T, DH>::query_rows(a, a.q, g.dq + s.q, kvh, r0, rows, acc, a.scale,
                           reinterpret_cast<T*>(smem) + wave * Out<T, DH>::WAVE, lane);
    });
}

// How dK / dV's work is cut.  Key tiles of 32 NK keys; the rows that see one are cut into
// pieces where the tiles alone do not fill the card (`nears` pieces of `near` rows), and
// where a window has first tokens the rows past its reach (far rows), which
// see none but the tiles that hold these (`first` of them), are `chunks` more
// pieces of `chunk` rows.  A tile in pieces leaves a part of each, `nears` of every tile
// that is cut (`cut` of them, from the first on), then the far ones; seq_sum_kernel adds
// them up in that order.
struct DkvPlan {
    int ktiles, first, chunks, chunk, nears, near, cut;
    __host__ __device__ __forceinline__ int pieces() const { return ktiles * nears + first * chunks; }
    __host__ __device__ __forceinline__ int parts() const { return cut * nears + first * chunks; }
};

// rows that see the key tile from key0: near ones up to `far`, far ones from there on (where
// these are cut off: else all are near)
struct Rows { int lo, far, hi; };
__device__ __forceinline__ Rows rows_of(const SArgs& a, const Seq& s, int key0, int nk, bool off) {
    Rows r;
    r.lo = min(key0, s.ql) * a.G;
    const int reach = a.window > s.ql - key0 - nk ? s.ql : min(s.ql, key0 + nk - 1 + a.window);
    r.far = reach * a.G;
    r.hi = key0 < a.sinks ? s.ql * a.G : r.far;
    if (!off) r.far = r.hi;
    return r;
}

// A tile of BQ query rows with their dO rows and statistics straight into LDS (bf16):
// pieces of both operands are dealt out to the waves.  Past the last row the last one
// stands in; its scores are masked.
template <int DH, int BQ, int NW> struct QDma {
    typedef Lds<DH, false> L;
    static constexpr int CPR = DH / 8, RPI = 64 / CPR, PER = BQ / RPI, NI = 2 * PER / NW;   // pieces an operand, a wave
    static_assert(2 * PER % NW == 0 && PER % NI == 0, "a wave's pieces are of one operand");
    static constexpr int FULL = 0x7fffffe0;      // the host has seen that offsets stay below
    intx4 rs, st;
    int wave, sl, sh, rows, row[NI], col[NI];
    bool isd;
    __device__ __forceinline__ void init(const SArgs& a, const Seq& s, const __bf16* q, const __bf16* d,
                                         const float2* stats, int kvh, int rows_, int tid) {
        const int lane = tid & 63;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        isd = wave * NI >= PER;
        const PtcgHeadLayout& l = isd ? a.o : a.q;
        sl = (int)l.sl * 2;
        sh = (int)l.sh * 2;
        rows = rows_;
        const __bf16* p = isd ? d + s.o : q + s.q;
        rs = KvDma<DH, 64, 4, false>::rsrc(reinterpret_cast<const char*>(p + (long)kvh * a.G * l.sh), FULL);
        st = KvDma<DH, 64, 4, false>::rsrc(reinterpret_cast<const char*>(stats), rows * 8);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            row[i] = (wave * NI + i) % PER * RPI + lane / CPR;
            const int c = (lane % CPR) ^ L::swz(row[i]);
            col[i] = 8 * c < a.dh ? 16 * c : PT_NOWHERE;
        }
    }
    __device__ __forceinline__ void fetch(const SArgs& a, int row0, __bf16* Qs, __bf16* Ds, float* ls, int lane) const {
        __bf16* to = isd ? Ds : Qs;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = min(row0 + row[i], rows - 1), qi = head_div(a, r);
            const int off = col[i] == PT_NOWHERE ? PT_NOWHERE : qi * sl + (r - qi * a.G) * sh + col[i];
            to_lds(rs, to + (wave * NI + i) % PER * RPI * L::ST, off);
        }
        if (wave < BQ / 32) {     // 32 rows' two numbers
            const unsigned at = (unsigned)(uintptr_t)(ls + wave * 64);
            asm volatile("s_mov_b32 m0, %0\n\t" PT_WAIT_M0 "buffer_load_dword %1, %2, 0 offen lds"
                         :: "s"(__builtin_amdgcn_readfirstlane(at)), "v"((row0 + wave * 32) * 8 + lane * 4), "s"(st)
                         : "memory", "m0");
        }
    }
};

template <typename T, int DH, int NK, bool DMA> struct DkvCfg {
    static constexpr bool PAD = DH == 128 && !DMA;
    static constexpr int NTH = 64 * NK, BKEY = 32 * NK;
    // the rows of a step: 32 where the registers hold no more on their way
    static constexpr int BQ = DH * planes<T>() >= 128 || NK < 4 ? 32 : 64;
    static constexpr int TILE = tile_elems<T, DH, PAD, BQ>();
    static constexpr size_t PAIR = (DMA ? 2 : 1) * 4 * (size_t)TILE;   // bytes
    static constexpr size_t OUT = (size_t)NK * Out<T, DH>::WAVE * sizeof(T);
    static constexpr size_t BUFS = PAIR > OUT ? PAIR : OUT;
    // 128 wide in bf16, the values' rows stay in LDS: with them, dK and dV in
    // registers two waves a SIMD would spill
    static constexpr bool VLDS = sizeof(T) == 2 && DH == 128;
    static constexpr size_t VROWS = VLDS ? (size_t)BKEY * Lds<DH, PAD>::ST * 2 : 0;
    static constexpr size_t LDS = BUFS + VROWS + 2 * 2 * BQ * sizeof(float);
};
template <typename T, int DH> constexpr int dkv_waves() {
    return DH * planes<T>() <= 64 || waves_simd<T, DH>() == 2 ? 2 : 1;
}

// dK and dV: a workgroup owns 32 NK keys of one kv head, a wave 32 of them, and
// walks the flattened query rows that see them.  S = Q K^T and dP = dO V^T with
// keys on lanes; dV^T += dO^T P and dK^T += Q^T dS read dO and Q transposed from LDS.
// The forward's four sequences, 8 heads of 128, bf16: 251 to 256 us (570 TFLOP/s in four products),
// bound by unequal tiles as well: the first keys' is seen by 128 blocks of rows, where an XCD's mean load
// is 70; 512 sequences up to 97, 4 heads of 64, fp32: 87 us.
template <typename T, int DH, int NK, bool DMA>
__global__ __launch_bounds__(64 * NK, (dkv_waves<T, DH>())) void seq_dkv_kernel(const SArgs a, const Grads<T> g,
                                                                               const DkvPlan pl) {
    typedef DkvCfg<T, DH, NK, DMA> C;
    typedef Stage<T, DH, C::PAD, C::BQ, C::NTH> St;
    typedef Lds<DH, C::PAD> L;
    constexpr int BQ = C::BQ;
    extern __shared__ __align__(256) char smem[];
    __bf16* tiles = reinterpret_cast<__bf16*>(smem);
    float* stats = reinterpret_cast<float*>(smem + C::BUFS + C::VROWS);   // log-sum-exp and D of the rows
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    // a (sequence, kv head)'s pieces: far chunks of its first key tiles, then near rows of all
    const int fars = pl.first * pl.chunks;
    const Share sh = share_of(blockIdx.x, a.n * a.KV, pl.pieces(), a.q_off != nullptr);
    const int u = sh.pair, i = u / a.KV, kvh = u - i * a.KV, x = sh.piece - fars;
    const bool isfar = x < 0;
    const int kt = isfar ? sh.piece / pl.chunks : x / pl.nears, ch = isfar ? sh.piece % pl.chunks : x % pl.nears;
    const Seq s = seq_of<false>(a, i);
    const int kall = s.rows;          // a padded sequence's dead rows get zeros
    if (kt * C::BKEY >= kall) return;
    const int key0 = kt * C::BKEY, kw = key0 + 32 * __builtin_amdgcn_readfirstlane(wave), key = kw + (lane & 31);
    const bool kin = key < kall, kok = key < s.kl;
    const Rows rr = rows_of(a, s, key0, C::BKEY, kt < pl.first);
    // this piece's rows; a tile's first piece is there even without rows
    const int r0 = isfar ? rr.far + ch * pl.chunk : rr.lo + ch * pl.near, end = isfar ? rr.hi : rr.far;
    int rows = isfar ? (ch + 1 == pl.chunks ? end : min(end, r0 + pl.chunk))
                     : (ch + 1 == pl.nears ? end : min(end, r0 + pl.near));
    if (r0 >= rows && (isfar || ch > 0)) return;
    if (key0 >= s.kl) rows = r0;

    Row<T, DH> kfr, vfr;
    __bf16* Vl = reinterpret_cast<__bf16*>(smem + C::BUFS) + 32 * wave * L::ST;
    const long ko = s.k + (kin ? (long)key * a.k.sl + (long)kvh * a.k.sh : 0);
    const long vo = s.v + (kin ? (long)key * a.v.sl + (long)kvh * a.v.sh : 0);
    kfr.load(g.k + ko, kok, a.dh, h);
    vfr.load(g.v + vo, kok, a.dh, h);
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

    const int nt = rows > r0 ? (rows - r0 + BQ - 1) / BQ : 0;
    const float2* sg = g.stats + (long)u * a.lq * a.G;
    kfr.settle();
    if constexpr (!C::VLDS) vfr.settle();
    auto tile = [&](int t, const __bf16* Qs, const __bf16* Ds, const float* ls) {
#pragma unroll 1
        for (int j = 0; j < BQ / 32; ++j) {
            const int qr = 32 * j, row0 = r0 + t * BQ + qr;
            if (row0 >= rows) break;
            const int plo = head_div(a, row0), phi = head_div(a, min(row0 + 31, rows - 1));
            if (kw >= s.kl || all_hidden(a, kw, 32, plo, phi)) continue;
            floatx16 p, d;
            if constexpr (DMA) {
                products<DH, C::VLDS>(Qs + qr * L::ST, Ds + qr * L::ST, kfr, vfr, Vl, p, d, lane, [](int) {});
            } else {
                p = mma_rows<T, DH, C::PAD, St::PS>(Qs + qr * L::ST, kfr, lane);
                if constexpr (C::VLDS) d = mma_rows_lds<DH, C::PAD>(Ds + qr * L::ST, Vl, lane);
                else d = mma_rows<T, DH, C::PAD, St::PS>(Ds + qr * L::ST, vfr, lane);
            }
            if (row0 + 32 > rows || some_hidden(a, kw, 32, plo, phi)) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int r = row0 + 8 * (e / 4) + 4 * h + e % 4, at = head_div(a, r);
                    const bool see = r < rows && key <= at && (at - key < a.window || key < a.sinks);
                    p[e] = see ? p[e] : -INFINITY;
                }
            }
            // a key that is not there goes along: its columns are cleared at the end
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float* x4 = ls + 2 * (qr + 8 * e + 4 * h);
                const float4 x0 = *reinterpret_cast<const float4*>(x4), x1 = *reinterpret_cast<const float4*>(x4 + 4);
                const float lv[4] = {x0.x, x0.z, x1.x, x1.z}, dv[4] = {x0.y, x0.w, x1.y, x1.w};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    p[4 * e + c] = __builtin_amdgcn_exp2f(fmaf(p[4 * e + c], a.scale2, -lv[c]));
                    d[4 * e + c] -= dv[c];
                }
            }
            if constexpr (DMA) {
                constexpr int E = 16 / (DH / 16);       // elements in a product's shadow
                bf16x8 pb[2], db[2];
#pragma unroll
                for (int e = 0; e < 16; ++e) pb[e / 8][e % 8] = (__bf16)p[e];
                values<DH>(Ds + qr * L::ST, pb, gv, lane, [&](int c) {
#pragma unroll
                    for (int e = c * E; e < (c + 1) * E; ++e) db[e / 8][e % 8] = (__bf16)(p[e] * d[e]);
                });
                values<DH>(Qs + qr * L::ST, db, gk, lane, [](int) {});
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) d[e] *= p[e];
                mma_tr<T, DH, C::PAD, St::PS>(Ds + qr * L::ST, p, gv, lane);
                mma_tr<T, DH, C::PAD, St::PS>(Qs + qr * L::ST, d, gk, lane);
            }
        }
    };
    if constexpr (DMA) {
        QDma<DH, BQ, NK> qd;
        if (nt > 0) qd.init(a, s, g.q, g.dout, sg, kvh, rows, tid);
        auto fetch = [&](int t) {
            __bf16* to = tiles + (t & 1) * 2 * C::TILE;
            qd.fetch(a, r0 + t * BQ, to, to + C::TILE, stats + (t & 1) * 2 * BQ, lane);
        };
        if (nt > 0) fetch(0);
        for (int t = 0; t < nt; ++t) {
            arrived();
            __syncthreads();       // everyone's pieces of tile t are here, and tile t - 1 is done with
            if (t + 1 < nt) fetch(t + 1);
            const __bf16* from = tiles + (t & 1) * 2 * C::TILE;
            tile(t, from, from + C::TILE, stats + (t & 1) * 2 * BQ);
        }
        __syncthreads();           // the buffers become the rows' way out
    } else {
        St qs_, ds_;
        float2 lr = make_float2(0.f, 0.f);
        auto fetch = [&](int t) {
            const int row0 = r0 + t * BQ;
            qs_.load_q(a, a.q, g.q + s.q, kvh, row0, rows, tid);
            ds_.load_q(a, a.o, g.dout + s.o, kvh, row0, rows, tid);
            if (tid < BQ) lr = sg[min(row0 + tid, rows - 1)];
        };
        auto store = [&]() {
            qs_.store_q(tiles, tid, BQ, a.dh);
            ds_.store_q(tiles + C::TILE, tid, BQ, a.dh);
            if (tid < BQ) reinterpret_cast<float2*>(stats)[tid] = lr;
        };
        if (nt > 0) {
            fetch(0);
            store();
            if (nt > 1) fetch(1);
            __syncthreads();
        }
        for (int t = 0; t < nt; ++t) {
            tile(t, tiles, tiles + C::TILE, stats);
            __syncthreads();
            if (t + 1 < nt) {
                store();
                if (t + 2 < nt) fetch(t + 2);
                __syncthreads();
            }
        }
    }
    if (!kok) {   // a dead key's gradient is zero, whatever the rows hold
#pragma unroll
        for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) gk[dt][e] = gv[dt][e] = 0.f;
    }
    if (kt < pl.cut) {
        const int at = isfar ? pl.cut * pl.nears + kt * pl.chunks + ch : kt * pl.nears + ch;
        float* p = g.part + (((long)u * pl.parts() + at) * C::BKEY + 32 * wave + (lane & 31)) * 2 * a.dh;
        if (kin) {
            store_row<float, DH>(p, gk, 1.f, a.dh, h);
            store_row<float, DH>(p + a.dh, gv, 1.f, a.dh, h);
        }
        return;
    }
    T* ws = reinterpret_cast<T*>(smem) + wave * Out<T, DH>::WAVE;
    Out<T, DH>::key_rows(g.dk + s.k + (long)kvh * a.k.sh, a.k.sl, kw, kall, a.dh, gk, a.scale, ws, lane);
    Out<T, DH>::key_rows(g.dv + s.v + (long)kvh * a.v.sh, a.v.sl, kw, kall, a.dh, gv, 1.f, ws, lane);
}

// the parts of the cut tiles' dk and dv, in order of their rows: 4 columns a thread and turn.  4 to 13 us
constexpr int SUM_BLOCKS = 1 << 16;      // parts may come to 2^32 threads and more: workgroups walk them
template <typename T>
__global__ __launch_bounds__(256) void seq_sum_kernel(const SArgs a, const float* __restrict__ part,
        T* __restrict__ dk, T* __restrict__ dv, const DkvPlan pl, int bkey) {
    const int c4 = a.dh / 4, per = pl.cut * bkey;       // keys a (sequence, kv head)
    const long all = (long)a.n * a.KV * per * 2 * c4;
    for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < all; at += (long)gridDim.x * 256) {
        const long both = at / c4;
        const int c = (int)(at - both * c4) * 4, isv = (int)(both & 1), u = (int)(both / 2 / per);
        const int key = (int)(both / 2 - (long)u * per);
        const int i = u / a.KV, kvh = u - i * a.KV, kt = key / bkey;
        const Seq s = seq_of<false>(a, i);
        if (key >= s.rows) continue;
        const Rows r = rows_of(a, s, kt * bkey, bkey, kt < pl.first);
        // the pieces that have rows
        const bool dead = kt * bkey >= s.kl;
        const int nn = dead || pl.nears == 1 ? 1 : max(1, min(pl.nears, (r.far - r.lo + pl.near - 1) / pl.near));
        const int nf = dead || kt >= pl.first ? 0 : min(pl.chunks, (r.hi - r.far + pl.chunk - 1) / pl.chunk);
        const float* p = part + (((long)u * pl.parts() * bkey + key % bkey) * 2 + isv) * a.dh + c;
        const long one = (long)bkey * 2 * a.dh;
        float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](int first, int n) {
#pragma unroll 4
            for (int x = 0; x < n; ++x) {
                const float4 y = *reinterpret_cast<const float4*>(p + (first + x) * one);
                g.x += y.x; g.y += y.y; g.z += y.z; g.w += y.w;
            }
        };
        add(kt * pl.nears, nn);
        add(pl.cut * pl.nears + kt * pl.chunks, nf);
        const float f = isv ? 1.f : a.scale;
        T* o = isv ? dv + s.v + (long)key * a.v.sl + (long)kvh * a.v.sh
                   : dk + s.k + (long)key * a.k.sl + (long)kvh * a.k.sh;
        st4(o + c, g.x * f, g.y * f, g.z * f, g.w * f);
    }
}

// ------------------------------------------------------------------- host
// packed_rows: the rows that packed sequences have in all; -1: not known
int check_common(int n, int l, int heads, int kv_heads, int dh, int bf16, float scale, int window, int sinks,
                 const PtcgHeadLayout& q, const PtcgHeadLayout& o, int64_t packed_rows, const char* who) {
    PT_REQUIRE(n >= 0 && l >= 0, "%s: negative size: %d sequences of %d rows", who, n, l);
    PT_REQUIRE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, "%s: %d heads over %d kv heads", who, heads,
               kv_heads);
    PT_REQUIRE(dh >= 8 && dh <= 128 && dh % 8 == 0, "%s: head width %d is not a multiple of 8 up to 128", who, dh);
    PT_REQUIRE(bf16 == 0 || bf16 == 1, "%s: bf16=%d", who, bf16);
    PT_REQUIRE(scale > 0.f && scale < 1e30f, "%s: scale must be positive and finite", who);
    PT_REQUIRE(window >= 0 && sinks >= 0, "%s: window=%d sinks=%d", who, window, sinks);
    const int e = bf16 ? 8 : 4;
    PT_REQUIRE(layout_ok(q, e) && layout_ok(o, e), "%s: strides must be non-negative multiples of 16 bytes", who);
    // (8 bytes of statistics a row within 2^31)
    const int64_t G = heads / kv_heads, rows = (int64_t)l * G;
    PT_REQUIRE(l < (1 << 30) && rows * G < (1LL << 32) && rows < (1LL << 28) - 64,
               "%s: %d rows of %d heads a kv head are too long", who, l, (int)G);
    // A launch holds fewer than 2^32 threads, 256 a tile of rows at most (32 rows or more) and two tiles'
    // for what of a sequence fills none; dk / dv's pieces, of 64 keys or more, are fewer.
    double tiles = (double)n * (double)(rows / 32 + 2);
    if (packed_rows >= 0) {      // no more than the rows there are make
        const double t = (double)packed_rows * G / 32 + 2.0 * n;
        if (t < tiles) tiles = t;
    }
    PT_REQUIRE(tiles * kv_heads < (double)(1 << 24), "%s: too many rows", who);
    return PTCG_OK;
}
int check_paged(const PtcgPagedAttn* d, const char* who) {
    PT_REQUIRE(d, "%s: null descriptor", who);
    PT_TRY(check_common(d->n, d->lq, d->heads, d->kv_heads, d->dh, d->bf16, d->scale, d->window, d->sinks, d->q, d->o,
                        d->q_off ? d->rows : -1, who));
    PT_REQUIRE(!d->q_off || (d->rows >= 0 && d->rows < (1 << 30)), "%s: rows=%d", who, d->rows);
    PT_TRY(check_pages(d->cache, d->n, d->kv_heads, d->dh, d->bf16 ? 8 : 4, who));
    return PTCG_OK;
}
int check_window(const PtcgWindowAttn* d, const char* who) {
    PT_REQUIRE(d, "%s: null descriptor", who);
    PT_TRY(check_common(d->n, d->l, d->heads, d->kv_heads, d->dh, d->bf16, d->scale, d->window, d->sinks, d->q, d->o,
                        -1, who));
    const int e = d->bf16 ? 8 : 4;
    PT_REQUIRE(layout_ok(d->k, e) && layout_ok(d->v, e), "%s: strides must be non-negative multiples of 16 bytes", who);
    PT_REQUIRE(!(d->off && d->len), "%s: packed sequences (off) take no len", who);
    PT_REQUIRE((d->k.sl | d->v.sl) < (1 << 22), "%s: key rows 2^22 elements apart or more", who);
    // a bounded tile reads zeros past its rows, which holds for rows that do not
    // reach into one another
    PT_REQUIRE((d->l <= 1 && !d->off) ||
                   ((d->k.sl == 0 || d->k.sl >= d->dh) && (d->v.sl == 0 || d->v.sl >= d->dh)),
               "%s: key rows overlap", who);
    return PTCG_OK;
}

SArgs base_args(int n, int l, int heads, int kv_heads, int dh, float scale, int window, int sinks) {
    SArgs a = {};
    a.n = n; a.lq = l; a.H = heads; a.KV = kv_heads; a.G = heads / kv_heads; a.dh = dh;
    a.gmagic = (unsigned)((1ULL << 32) / a.G + 1);
    a.scale = scale; a.scale2 = scale * LOG2E;
    a.window = window > 0 ? window : INT_MAX;
    a.sinks = sinks;
    return a;
}
SArgs paged_args(const PtcgPagedAttn* d) {
    SArgs a = base_args(d->n, d->lq, d->heads, d->kv_heads, d->dh, d->scale, d->window, d->sinks);
    a.q = d->q; a.o = d->o; a.k = d->cache.k; a.v = d->cache.v;
    a.q_off = d->q_off; a.len = d->len; a.all_rows = d->rows;
    a.table = d->cache.table; a.table_sn = d->n > 1 ? d->cache.table_sn : 0;
    a.pages = d->cache.pages; a.page = d->cache.page; a.per_seq = d->cache.per_seq;
    // m = ceil(2^(31 + b) / page) with 2^(b - 1) < page <= 2^b: m < 2^32, and key m / 2^(31 +
    // b) is above key / page by less than key / 2^31 / page < 1 / page
    int b = 1;
    while ((1LL << b) < a.page) ++b;
    a.pmagic = (unsigned)(((1ULL << (31 + b)) + a.page - 1) / a.page);
    a.pshift = b - 1;
    return a;
}
SArgs window_args(const PtcgWindowAttn* d) {
    SArgs a = base_args(d->n, d->l, d->heads, d->kv_heads, d->dh, d->scale, d->window, d->sinks);
    a.q = d->q; a.o = d->o; a.k = d->k; a.v = d->v;
    if (d->l <= 1 && !d->off) a.k.sl = a.v.sl = d->dh;     // one row: any stride was given
    a.q_off = d->off; a.len = d->len; a.all_rows = INT_MAX;
    return a;
}

// Which kernel and how it is split.  Up to 32 rows a (sequence, kv head): the kernel of
// few rows, its four waves along the keys where a sequence may have more than four blocks
// of 32.  Else tiles of 64 or 128 rows.
struct Form {
    bool token;
    bool dma;        // tiles straight into LDS: bf16 rows of one matrix, or of pages that a wave's rows never leave
    int waves;       // along the keys (token), along the rows else
    int bq, bk;
    Plan p;
};
// keys: the most that a row tile may see, as far as the host knows
Form form_of(const SArgs& a, int64_t packed_rows, int64_t keys, bool bf16, bool may_split) {
    Form f;
    const int64_t rows = (int64_t)a.lq * a.G;
    f.token = rows <= 32;
    // Up to 64 rows of whole sequences take two waves, up to 64 wide (512 x 64 rows, 4 heads of 64: 37 us against
    // 42 in fp32, 18 against 20 in bf16; of 128 in bf16 35 against 33).  Over pages, whose keys are many, four
    // waves bring the tiles faster (256 chunks of 48 rows over 2 000 keys, 64 wide: 178 us against 215 in fp32,
    // in bf16 50 against 51, in pages of 24 rows 67 against 82; 128 wide 106 against 173).
    f.waves = f.token ? (keys > 128 ? 4 : 1) : !a.page && rows <= 64 && a.dh <= 64 ? 2 : 4;
    f.bq = f.token ? 32 : 32 * f.waves;
    f.dma = bf16;
    if (a.page) {
        auto fits = [&](const PtcgHeadLayout& l) { return l.sl < (1 << 22) && (l.sl == 0 || l.sl >= a.dh); };
        f.dma = f.dma && a.page % 16 == 0 && fits(a.k) && fits(a.v);      // a wave's of 64 keys
    }
    f.bk = f.token ? 32 : 64;
    const int qtiles = pt_cdiv(rows, f.bq);
    int64_t tiles = (int64_t)a.n * qtiles;
    if (a.q_off) {       // no more than the rows there are make
        const int64_t t = packed_rows * a.G / f.bq + a.n;
        if (t < tiles) tiles = t;
    }
    // Where row tiles do not fill the card, stretches of keys do, one for each workgroup that
    // runs at once.  A stretch is four blocks at least (a token's: one a
    // wave), and costs a second launch.
    const int64_t fill = (bf16 || a.dh <= 64 ? 2 : 1) * (int64_t)cu_count();
    f.p.least = 4;
    f.p.split = may_split && tiles * a.KV < fill && keys >= 4 * f.p.least * f.bk &&
                (tiles + 1) * (keys / f.bk + 8) < (1LL << 30);
    f.p.tiles = (int)tiles;
    f.p.slots = (int)(f.p.split ? (fill / a.KV > 1 ? fill / a.KV : 1) : tiles);
    // a token's pieces: at least a second one for each tile that is cut
    if (f.p.split && f.token && f.p.slots < 2 * tiles) f.p.slots = (int)(2 * tiles);
    f.p.qtiles = qtiles;
    f.p.even = !a.q_off && !f.p.split;
    f.p.prow = (int)(rows < f.bq ? rows : f.bq);
    return f;
}
Form paged_form(const PtcgPagedAttn* d, const SArgs& a) {
    int64_t keys = (int64_t)a.per_seq * a.page;
    if (d->window > 0 && (int64_t)d->window + d->sinks + d->lq < keys) keys = (int64_t)d->window + d->sinks + d->lq;
    return form_of(a, d->rows, keys, d->bf16, true);
}
Form window_form(const PtcgWindowAttn* d, const SArgs& a) {
    return form_of(a, (int64_t)d->n * d->l, d->l, d->bf16, true);
}
int64_t part_bytes(const Form& f, const SArgs& a) {
    return f.p.split ? 16 * (1 + (int64_t)f.p.tiles) + 2 * (int64_t)f.p.slots * a.KV * part_floats(f.p.prow, a.dh) * 4 : 0;
}

template <typename T, int DH, bool PAGED, int BQ>
int launch_join(const SArgs& a, const Form& f, void* out, float* lse, const float* part, hipStream_t s) {
    constexpr int LG = DH / 4, NG = JOIN_NTH / LG;
    // four splits a group of lanes, as many as tiles have if they are alike
    int per_row = 1;
    while (per_row < NG && (int64_t)per_row * 4 * f.p.tiles < f.p.slots) per_row *= 2;
    const int rgroups = pt_cdiv(f.p.prow, NG / per_row);
    hipLaunchKernelGGL((seq_join_kernel<T, LG, PAGED, BQ>), dim3((unsigned)((int64_t)f.p.tiles * a.KV * rgroups)),
                       dim3(JOIN_NTH), 0, s, a, part, static_cast<T*>(out), lse, f.p, per_row, rgroups);
    PT_LAUNCH_CHECK();
    return PTCG_OK;
}

template <typename T, int DH, int NW, bool PAGED, bool DMA>
int launch_tiles(const SArgs& a, const Form& f, const void* q, const void* k, const void* v, void* out, float* lse,
                 float* part, hipStream_t s) {
    typedef TileCfg<T, DH, NW, DMA> C;
    auto kern = seq_fwd_kernel<T, DH, NW, PAGED, DMA>;
    PT_TRY(lds_attr(kern, C::LDS));
    hipLaunchKernelGGL(kern, dim3((unsigned)((int64_t)f.p.slots * a.KV)), dim3(C::NTH), C::LDS, s, a,
                       static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                       static_cast<T*>(out), lse, part, f.p);
    PT_LAUNCH_CHECK();
    return f.p.split ? launch_join<T, DH, PAGED, C::BQ>(a, f, out, lse, part, s) : PTCG_OK;
}
template <typename T, int DH, int KS, bool PAGED>
int launch_token(const SArgs& a, const Form& f, const void* q, const void* k, const void* v, void* out, float* lse,
                 float* part, hipStream_t s) {
    typedef TokenCfg<T, DH, KS> C;
    auto kern = seq_token_kernel<T, DH, KS, PAGED>;
    PT_TRY(lds_attr(kern, C::LDS));
    hipLaunchKernelGGL(kern, dim3((unsigned)((int64_t)f.p.slots * a.KV)), dim3(C::NTH), C::LDS, s, a,
                       static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                       static_cast<T*>(out), lse, part, f.p);
    PT_LAUNCH_CHECK();
    return f.p.split ? launch_join<T, DH, PAGED, C::BQ>(a, f, out, lse, part, s) : PTCG_OK;
}
template <typename T, int DH, bool PAGED>
int launch_form(const SArgs& a, const Form& f, const void* q, const void* k, const void* v, void* out, float* lse,
                float* part, hipStream_t s) {
    if (f.token)
        return f.waves == 4 ? launch_token<T, DH, 4, PAGED>(a, f, q, k, v, out, lse, part, s)
                            : launch_token<T, DH, 1, PAGED>(a, f, q, k, v, out, lse, part, s);
    if constexpr (sizeof(T) == 2)
        if (f.dma) {
            if constexpr (!PAGED && DH <= 64)
                if (f.waves == 2) return launch_tiles<T, DH, 2, PAGED, true>(a, f, q, k, v, out, lse, part, s);
            return launch_tiles<T, DH, 4, PAGED, true>(a, f, q, k, v, out, lse, part, s);
        }
    if constexpr (sizeof(T) == 4 || PAGED) {
        if constexpr (!PAGED && DH <= 64)
            if (f.waves == 2) return launch_tiles<T, DH, 2, PAGED, false>(a, f, q, k, v, out, lse, part, s);
        return launch_tiles<T, DH, 4, PAGED, false>(a, f, q, k, v, out, lse, part, s);
    }
    return PTCG_OK;
}
template <bool PAGED>
int run_fwd(const SArgs& a, const Form& f, bool bf16, const void* q, const void* k, const void* v, void* out, float* lse,
            float* part, hipStream_t s) {
    if (bf16)
        return a.dh <= 32   ? launch_form<__bf16, 32, PAGED>(a, f, q, k, v, out, lse, part, s)
               : a.dh <= 64 ? launch_form<__bf16, 64, PAGED>(a, f, q, k, v, out, lse, part, s)
                            : launch_form<__bf16, 128, PAGED>(a, f, q, k, v, out, lse, part, s);
    return a.dh <= 32   ? launch_form<float, 32, PAGED>(a, f, q, k, v, out, lse, part, s)
           : a.dh <= 64 ? launch_form<float, 64, PAGED>(a, f, q, k, v, out, lse, part, s)
                        : launch_form<float, 128, PAGED>(a, f, q, k, v, out, lse, part, s);
}

// The backward's launches: row tiles for dq; key tiles, and chunks of the rows that see
// first tokens alone, for dk and dv.
struct BwdPlan {
    int nw, nk;
    Plan q;
    DkvPlan k;
    bool dma;                // dk / dv's tiles straight into LDS
    int64_t stats, part;     // workspace floats
};
BwdPlan bwd_plan(const PtcgWindowAttn* d, const SArgs& a) {
    BwdPlan p = {};
    const int64_t rows = (int64_t)a.lq * a.G;
    // Two waves for up to 64 rows as in the forward, but where their instance spills (512 x 64 rows, 4 heads,
    // both gradients: 32 wide 56 us against 64 in fp32, 32 against 36 in bf16, 64 wide 49 against 52; in fp32
    // 64 and 128 wide, where it spilled, 111 us against 108 and 404 against 375; 128 wide in bf16 92 against 91)
    p.nw = rows <= 64 && a.dh <= (d->bf16 ? 64 : 32) ? 2 : 4;
    p.q.qtiles = pt_cdiv(rows, 32 * p.nw);
    p.q.tiles = p.q.slots = a.n * p.q.qtiles;
    p.q.even = !a.q_off;
    // short fp32 sequences, more of them than run at once: two waves wait for less (512 x 97, 4 heads,
    // 64 wide: 87 us against 97; of row tiles the same costs 8 to 30% more)
    p.nk = (a.lq <= 64 || (!d->bf16 && a.lq <= 128 && a.n * a.KV > 2 * cu_count())) && (d->bf16 || a.dh <= 64) ? 2 : 4;
    const int bkey = 32 * p.nk;
    p.k.ktiles = pt_cdiv(a.lq, bkey);
    // Far rows are cut off where one tile's would take longer than two key tiles' near ones, in
    // at most 16 pieces; with more than two such tiles there is work for many workgroups as it is.
    const int64_t reach = ((int64_t)bkey + a.window) * a.G, far = rows - reach;
    const bool firsts = a.sinks > 0 && a.window < a.lq;
    if (firsts && a.sinks <= 2 * bkey && far > reach) p.k.first = pt_cdiv(a.sinks, bkey);
    // Where key tiles are fewer than the workgroups that run at once, their near rows are
    // cut as well, so that the pieces are about as many; of 256 rows at least, and no
    // more parts than four times the workgroups.  (1 500 rows of 8 heads on one, 128 wide, 12 tiles: dk
    // and dv 2 446 us uncut, 173 cut in fp32, 438 and 44 in bf16; 4 x 1 000 rows of 8 heads, 64 wide,
    // 256 tiles: 116 and 75 in fp32, 34 and 38 in bf16, which is left whole from a tile a CU on.)
    const int64_t span = rows < reach || (firsts && !p.k.first) ? rows : reach, pairs = (int64_t)a.n * a.KV;
    const int64_t fill = (d->bf16 || a.dh <= 64 ? 2 : 1) * (int64_t)cu_count();
    p.k.nears = 1;
    p.k.near = INT_MAX;
    if (pairs * p.k.ktiles < (d->bf16 ? cu_count() : fill)) {
        int64_t all = 0;
        for (int t = 0; t < p.k.ktiles; ++t) {
            const int64_t left = rows - (int64_t)t * bkey * a.G;
            all += left < span ? left : span;
        }
        int64_t near = all * pairs / fill;
        if (near < span * pairs * p.k.ktiles / (4 * fill)) near = span * pairs * p.k.ktiles / (4 * fill);
        if (near < 256) near = 256;
        near = (near + 63) / 64 * 64;
        if (near < span) {
            p.k.near = (int)near;
            p.k.nears = pt_cdiv(span, near);
        }
    }
    if (p.k.first) {
        int64_t chunk = p.k.nears > 1 ? p.k.near : reach;
        if (chunk < far / 16) chunk = far / 16;
        chunk = (chunk + 63) / 64 * 64;
        p.k.chunk = (int)chunk;
        p.k.chunks = pt_cdiv(far, chunk);
    }
    p.k.cut = p.k.nears > 1 ? p.k.ktiles : p.k.first;
    p.stats = ((int64_t)a.n * a.H * a.lq * 2 + 3) / 4 * 4;
    auto near31 = [&](const PtcgHeadLayout& l) {     // a kv head's rows of a sequence within 2^31 bytes
        return l.sl < (1LL << 30) && l.sh < (1LL << 30) && ((int64_t)a.lq * l.sl + (int64_t)a.G * l.sh) * 2 < 0x7fffff00LL;
    };
    p.dma = d->bf16 && near31(a.q) && near31(a.o);
    p.part = pairs * p.k.parts() * bkey * 2 * a.dh;
    return p;
}

template <typename T, int DH, int NW> int launch_dq(const SArgs& a, const BwdPlan& p, const Grads<T>& g, hipStream_t s) {
    typedef DqCfg<T, DH, NW> C;
    auto kern = seq_dq_kernel<T, DH, NW>;
    PT_TRY(lds_attr(kern, C::LDS));
    hipLaunchKernelGGL(kern, dim3((unsigned)((int64_t)p.q.slots * a.KV)), dim3(C::NTH), C::LDS, s, a, g, p.q);
    PT_LAUNCH_CHECK();
    return PTCG_OK;
}
template <typename T, int DH, int NK, bool DMA>
int launch_dkv(const SArgs& a, const BwdPlan& p, const Grads<T>& g, hipStream_t s) {
    typedef DkvCfg<T, DH, NK, DMA> C;
    auto kern = seq_dkv_kernel<T, DH, NK, DMA>;
    PT_TRY(lds_attr(kern, C::LDS));
    const int64_t pairs = (int64_t)a.n * a.KV;
    hipLaunchKernelGGL(kern, dim3((unsigned)(pairs * p.k.pieces())), dim3(C::NTH), C::LDS, s, a,
                       g, p.k);
    PT_LAUNCH_CHECK();
    if (p.k.cut) {
        const int64_t blocks = (pairs * p.k.cut * C::BKEY * 2 * (a.dh / 4) + 255) / 256;
        hipLaunchKernelGGL(seq_sum_kernel<T>, dim3((unsigned)(blocks < SUM_BLOCKS ? blocks : SUM_BLOCKS)), dim3(256), 0, s,
                           a, g.part, g.dk, g.dv, p.k, C::BKEY);
        PT_LAUNCH_CHECK();
    }
    return PTCG_OK;
}
template <typename T, int DH> int run_bwd(const SArgs& a, const BwdPlan& p, const Grads<T>& g, hipStream_t s) {
    if constexpr (DH <= (sizeof(T) == 2 ? 64 : 32))
        PT_TRY(p.nw == 2 ? (launch_dq<T, DH, 2>(a, p, g, s)) : (launch_dq<T, DH, 4>(a, p, g, s)));
    else PT_TRY((launch_dq<T, DH, 4>(a, p, g, s)));
    if constexpr (sizeof(T) == 2)
        if (p.dma)
            return p.nk == 2 ? launch_dkv<T, DH, 2, true>(a, p, g, s) : launch_dkv<T, DH, 4, true>(a, p, g, s);
    if constexpr (sizeof(T) == 2 || DH <= 64)
        if (p.nk == 2) return launch_dkv<T, DH, 2, false>(a, p, g, s);
    return launch_dkv<T, DH, 4, false>(a, p, g, s);
}
template <typename T>
int bwd_dh(const SArgs& a, const BwdPlan& p, const void* q, const void* k, const void* v, const void* out,
           const float* lse, const void* dout, void* dq, void* dk, void* dv, float* ws, hipStream_t s) {
    const Grads<T> g = {static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                        static_cast<const T*>(out), static_cast<const T*>(dout), lse, static_cast<T*>(dq),
                        static_cast<T*>(dk), static_cast<T*>(dv), reinterpret_cast<float2*>(ws), ws + p.stats};
    return a.dh <= 32 ? run_bwd<T, 32>(a, p, g, s) : a.dh <= 64 ? run_bwd<T, 64>(a, p, g, s) : run_bwd<T, 128>(a, p, g, s);
}

}  // namespace

extern "C" int64_t ptcg_kernel_paged_attention_ws_bytes(const PtcgPagedAttn* d) {
    if (check_paged(d, "paged_attention_ws_bytes") != PTCG_OK) return -1;
    if (d->n == 0 || d->lq == 0) return 0;
    const SArgs a = paged_args(d);
    return part_bytes(paged_form(d, a), a);
}

extern "C" int ptcg_kernel_paged_attention(const PtcgPagedAttn* d, const void* q, void* out, float* lse, void* workspace,
                                           int64_t workspace_bytes, void* stream) {
    const char* who = "paged_attention";
    PT_TRY(check_paged(d, who));
    if (d->n == 0 || d->lq == 0 || (d->q_off && d->rows == 0)) return PTCG_OK;
    PT_REQUIRE(q && out && d->len, "%s: null buffer", who);
    PT_REQUIRE(al16(q) && al16(out) && al16(d->cache.kp) && al16(d->cache.vp), "%s: buffers must be 16 B aligned", who);
    PT_REQUIRE(layout_apart(d->o, d->q_off, d->n, d->lq, d->heads, d->dh), "%s: rows of the output overlap", who);
    const SArgs a = paged_args(d);
    const Form f = paged_form(d, a);
    const int64_t need = part_bytes(f, a);
    PT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && al16(workspace)),
               "%s: workspace of %lld bytes, need %lld (16 B aligned)", who, (long long)workspace_bytes,
               (long long)need);
    return run_fwd<true>(a, f, d->bf16, q, d->cache.kp, d->cache.vp, out, lse, static_cast<float*>(workspace),
                         (hipStream_t)stream);
}

extern "C" int64_t ptcg_kernel_window_attention_ws_bytes(const PtcgWindowAttn* d, int backward) {
    if (check_window(d, "window_attention_ws_bytes") != PTCG_OK) return -1;
    if (d->n == 0 || d->l == 0) return 0;
    const SArgs a = window_args(d);
    if (backward) {
        const BwdPlan p = bwd_plan(d, a);
        return (p.stats + p.part) * 4;
    }
    return part_bytes(window_form(d, a), a);
}

extern "C" int ptcg_kernel_window_attention_fwd(const PtcgWindowAttn* d, const void* q, const void* k, const void* v,
                                                void* out, float* lse, void* workspace, int64_t workspace_bytes,
                                                void* stream) {
    const char* who = "window_attention_fwd";
    PT_TRY(check_window(d, who));
    if (d->n == 0 || d->l == 0) return PTCG_OK;
    PT_REQUIRE(q && k && v && out, "%s: null buffer", who);
    PT_REQUIRE(al16(q) && al16(k) && al16(v) && al16(out), "%s: buffers must be 16 B aligned", who);
    PT_REQUIRE(layout_apart(d->o, d->off, d->n, d->l, d->heads, d->dh), "%s: rows of the output overlap", who);
    const SArgs a = window_args(d);
    const Form f = window_form(d, a);
    const int64_t need = part_bytes(f, a);
    PT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && al16(workspace)),
               "%s: workspace of %lld bytes, need %lld (16 B aligned)", who, (long long)workspace_bytes,
               (long long)need);
    return run_fwd<false>(a, f, d->bf16, q, k, v, out, lse, static_cast<float*>(workspace), (hipStream_t)stream);
}

extern "C" int ptcg_kernel_window_attention_bwd(const PtcgWindowAttn* d, const void* q, const void* k, const void* v,
                                                const void* out, const float* lse, const void* dout, void* dq, void* dk,
                                                void* dv, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "window_attention_bwd";
    PT_TRY(check_window(d, who));
    if (d->n == 0 || d->l == 0) return PTCG_OK;
    PT_REQUIRE(q && k && v && out && lse && dout && dq && dk && dv, "%s: null buffer", who);
    PT_REQUIRE(al16(q) && al16(k) && al16(v) && al16(out) && al16(dout) && al16(dq) && al16(dk) && al16(dv),
               "%s: buffers must be 16 B aligned", who);
    PT_REQUIRE(layout_apart(d->q, d->off, d->n, d->l, d->heads, d->dh),
               "%s: rows of dq overlap (a broadcast q has no gradient layout)", who);
    PT_REQUIRE(layout_apart(d->k, d->off, d->n, d->l, d->kv_heads, d->dh) &&
                   layout_apart(d->v, d->off, d->n, d->l, d->kv_heads, d->dh),
               "%s: rows of dk or dv overlap (broadcast keys have no gradient layout)", who);
    const SArgs a = window_args(d);
    const BwdPlan p = bwd_plan(d, a);
    const int64_t need = (p.stats + p.part) * 4;
    PT_REQUIRE(workspace && workspace_bytes >= need && al16(workspace),
               "%s: workspace of %lld bytes, need %lld (16 B aligned)", who, (long long)workspace_bytes,
               (long long)need);
    float* ws = static_cast<float*>(workspace);
    const hipStream_t s = (hipStream_t)stream;
    return d->bf16 ? bwd_dh<__bf16>(a, p, q, k, v, out, lse, dout, dq, dk, dv, ws, s)
                   : bwd_dh<float>(a, p, q, k, v, out, lse, dout, dq, dk, dv, ws, s);
}
