// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
//   out[t] = scale table[id_t],   dtable[v] = scale sum_{t : id_t = v} dout[t]
//
// An id outside [0, vocab) is padding: its row of out is zeros and it adds to
// no gradient.  Both directions move bytes and little else: the forward reads
// an id and a table row and writes a row of out; the backward reads every live
// row of dout once and writes every row of dtable once (untouched ones as
// zeros).
//
// Backward.  The tokens are sorted by id (stable: equal ids keep token order),
// a row of the table then owns a run of the sorted list and adds its tokens in
// that order, so the sums do not depend on scheduling.  Adding by atomics
// instead costs a read-modify-write per element and token, in an order that
// changes; equal ids then queue on the same lines.
// Sort: least significant digit first, 1 digit of up to 11 bits where the
// vocabulary fits, else digits of up to 9 bits; per digit a count per
// workgroup, a scan over the workgroups, and a placement whose ranks within a
// wave come from ballots.
// Runs longer than CHUNK tokens (frequent ids) are added in CHUNK-aligned
// pieces of the sorted list by groups of lanes of their own and folded in order,
// so one frequent id does not hold a single group for its whole run.
#include "common.h"
#include "../../include/ptcg_amd_kernels.h"

namespace {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int CHUNK = 64;        // tokens a group adds on its own
constexpr int MAXB = 256;        // workgroups of a sort pass (tiles grow past it)
constexpr int BITS1 = 11, BITS2 = 9;

// VW values of a row, as floats
template <int VW> struct Vals { float v[VW]; };
template <int VW> __device__ __forceinline__ Vals<VW> ld(const float* p) {
    Vals<VW> r;
    if constexpr (VW == 1) r.v[0] = *p;
    else
#pragma unroll
        for (int i = 0; i < VW; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(p + i);
            r.v[i] = x.x; r.v[i + 1] = x.y; r.v[i + 2] = x.z; r.v[i + 3] = x.w;
        }
    return r;
}
template <int VW> __device__ __forceinline__ Vals<VW> ld(const __bf16* p) {
    Vals<VW> r;
    if constexpr (VW == 1) r.v[0] = (float)*p;
    else if constexpr (VW == 4) {
        const bf16x4 x = *reinterpret_cast<const bf16x4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[i] = (float)x[i];
    } else {
        const bf16x8 x = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = (float)x[i];
    }
    return r;
}
template <int VW> __device__ __forceinline__ void st(float* p, const Vals<VW>& r) {
    if constexpr (VW == 1) *p = r.v[0];
    else
#pragma unroll
        for (int i = 0; i < VW; i += 4)
            *reinterpret_cast<float4*>(p + i) = make_float4(r.v[i], r.v[i + 1], r.v[i + 2], r.v[i + 3]);
}
template <int VW> __device__ __forceinline__ void st(__bf16* p, const Vals<VW>& r) {
    if constexpr (VW == 1) *p = (__bf16)r.v[0];
    else if constexpr (VW == 4)
        *reinterpret_cast<bf16x4*>(p) = bf16x4{(__bf16)r.v[0], (__bf16)r.v[1], (__bf16)r.v[2], (__bf16)r.v[3]};
    else {
        bf16x8 x;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (__bf16)r.v[i];
        *reinterpret_cast<bf16x8*>(p) = x;
    }
}

// ---------------------------------------------------------------- forward
// A workgroup moves FWD_U * 256 consecutive VW-wide pieces of out, FWD_U of
// them in flight per thread.
constexpr int FWD_U = 4;
template <typename TT, typename TO, int VW>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const int* __restrict__ ids, long rows,
        const TT* __restrict__ table, long ldt, int vocab, int cpr, float scale, TO* __restrict__ out, long ldo) {
    const long first = (long)blockIdx.x * (256 * FWD_U);
    const long row0 = first / cpr;
    const unsigned rem0 = (unsigned)(first - row0 * cpr);
    Vals<VW> x[FWD_U];
    long at[FWD_U];
#pragma unroll
    for (int u = 0; u < FWD_U; ++u) {
        const unsigned p = rem0 + u * 256 + threadIdx.x, dr = p / (unsigned)cpr;
        const int col = (int)(p - dr * (unsigned)cpr) * VW;
        const long row = row0 + dr;
        at[u] = -1;
        if (row < rows) {
            at[u] = row * ldo + col;
            const int id = ids[row];
            if ((unsigned)id < (unsigned)vocab) x[u] = ld<VW>(table + (long)id * ldt + col);
            else
#pragma unroll
                for (int i = 0; i < VW; ++i) x[u].v[i] = 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < FWD_U; ++u) {
        if (at[u] < 0) continue;
#pragma unroll
        for (int i = 0; i < VW; ++i) x[u].v[i] *= scale;
        st<VW>(out + at[u], x[u]);
    }
}

// ------------------------------------------------------------------- sort
// One digit pass over `n` tokens (n_dev: its device count after the first pass
// dropped the padding); pos null: the first pass, token t's position is t and
// ids outside the vocabulary are dropped.
struct SortPass {
    const int* keys; const int* pos;
    const int* n_dev;
    int n, vocab, shift, bits, tile, nb;
    int* cnt;     // [bins][nb]
    int* tot;     // [bins]
    int* out_keys; int* out_pos;
    int* starts;  // one-digit sorts: first sorted position of each id, [vocab + 1] (else null)
    int* live;    // first pass: tokens kept
};

__device__ __forceinline__ int pass_n(const SortPass& p) { return p.n_dev ? min(*p.n_dev, p.n) : p.n; }
// digit of token t, -1 if it is dropped
__device__ __forceinline__ int digit_of(const SortPass& p, int t, int n, int& key) {
    if (t >= n) return -1;
    key = p.keys[t];
    if (!p.pos && (unsigned)key >= (unsigned)p.vocab) return -1;
    return (key >> p.shift) & ((1 << p.bits) - 1);
}

__global__ __launch_bounds__(256) void sort_count_kernel(const SortPass p) {
    extern __shared__ int hist[];
    const int bins = 1 << p.bits, n = pass_n(p);
    for (int i = threadIdx.x; i < bins; i += 256) hist[i] = 0;
    __syncthreads();
    const int t0 = blockIdx.x * p.tile;
    for (int o = threadIdx.x; o < p.tile; o += 256) {
        int key;
        const int d = digit_of(p, t0 + o, n, key);
        if (d >= 0) atomicAdd(&hist[d], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += 256) p.cnt[(long)i * p.nb + blockIdx.x] = hist[i];
}

// one wave per digit: exclusive scan over the workgroups' counts
__global__ __launch_bounds__(256) void sort_scan_kernel(const SortPass p) {
    const int lane = threadIdx.x & 63, bin = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (bin >= 1 << p.bits) return;
    int* c = p.cnt + (long)bin * p.nb;
    int run = 0;
    for (int b0 = 0; b0 < p.nb; b0 += 64) {
        const int v = b0 + lane < p.nb ? c[b0 + lane] : 0;
        int s = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(s, o, 64);
            if (lane >= o) s += x;
        }
        if (b0 + lane < p.nb) c[b0 + lane] = run + s - v;
        run += __shfl(s, 63, 64);
    }
    if (lane == 0) p.tot[bin] = run;
}

// Placement.  A wave owns a quarter of the workgroup's tile and walks it 64
// tokens at a time: a token's place is its digit's base, plus the digit's
// tokens before it in earlier workgroups, waves and batches, plus those in
// lower lanes of its batch.
__global__ __launch_bounds__(256) void sort_place_kernel(const SortPass p) {
    extern __shared__ int sm[];
    const int bins = 1 << p.bits, n = pass_n(p);
    int* cnt = sm;               // [4][bins]
    int* part = sm + 4 * bins;   // [256]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < 4 * bins; i += 256) cnt[i] = 0;
    __syncthreads();
    const int per = p.tile / 4, w0 = blockIdx.x * p.tile + wave * per;
    for (int o = lane; o < per; o += 64) {
        int key;
        const int d = digit_of(p, w0 + o, n, key);
        if (d >= 0) atomicAdd(&cnt[wave * bins + d], 1);
    }
    // exclusive scan of the digits' totals: thread t owns bpt consecutive digits
    const int bpt = (bins + 255) / 256, d0 = tid * bpt;
    int sum = 0;
    for (int i = 0; i < bpt; ++i)
        if (d0 + i < bins) sum += p.tot[d0 + i];
    part[tid] = sum;
    __syncthreads();
    for (int o = 1; o < 256; o <<= 1) {
        const int x = tid >= o ? part[tid - o] : 0;
        __syncthreads();
        part[tid] += x;
        __syncthreads();
    }
    int base = part[tid] - sum;
    if (tid == 255 && blockIdx.x == 0 && p.live) *p.live = part[255];
    for (int i = 0; i < bpt; ++i) {
        const int d = d0 + i;
        if (d >= bins) break;
        if (p.starts && blockIdx.x == 0 && d < p.vocab) p.starts[d] = base;
        int run = base + p.cnt[(long)d * p.nb + blockIdx.x];
        base += p.tot[d];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int c = cnt[w * bins + d];
            cnt[w * bins + d] = run;
            run += c;
        }
    }
    if (p.starts && blockIdx.x == 0 && tid == 255) p.starts[p.vocab] = part[255];
    __syncthreads();
    volatile int* my = cnt + wave * bins;
    for (int o = 0; o < per; o += 64) {
        const int t = w0 + o + lane;
        int key = 0;
        const int d = digit_of(p, t, n, key);
        unsigned long long same = __ballot(d >= 0);
        for (int i = 0; i < p.bits; ++i) {
            const unsigned long long b = __ballot((d >> i) & 1);
            same &= ((d >> i) & 1) ? b : ~b;
        }
        if (d >= 0) {
            const int rank = __popcll(same & ((1ull << lane) - 1));
            const int at = my[d] + rank;
            __builtin_amdgcn_wave_barrier();
            if (rank == 0) my[d] = at + __popcll(same);
            p.out_keys[at] = key;
            p.out_pos[at] = p.pos ? p.pos[t] : t;
        }
    }
}

// sorts of several digits: first sorted position of each id, by binary search
__global__ __launch_bounds__(256) void sort_starts_kernel(const int* __restrict__ keys,
        const int* __restrict__ live, int vocab, int* __restrict__ starts) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v > vocab) return;
    int lo = 0, hi = *live;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (keys[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    starts[v] = lo;
}

// --------------------------------------------------------------- gradient
struct GradArgs {
    const int* keys; const int* pos; const int* starts; const int* live;
    long ldo, ldt;
    int vocab, d, lpr, lpr_shift, ncc, nchunks;   // lpr: lanes of a group; ncc: column blocks of lpr * VW
    float scale;
    float* dtable;
    float* part;    // [nchunks][2][d]: a chunk's piece of the run it continues, and of the one it starts
};

// sum of dout rows of sorted tokens [a, b) at columns col.., in order, 8 in flight
template <typename TO, int VW>
__device__ __forceinline__ Vals<VW> run_sum(const TO* __restrict__ dout, const GradArgs& g, int a, int b, int col) {
    Vals<VW> s;
#pragma unroll
    for (int i = 0; i < VW; ++i) s.v[i] = 0.f;
    int t = a;
    for (; t + 8 <= b; t += 8) {
        int at[8];
        Vals<VW> x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) at[u] = g.pos[t + u];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = ld<VW>(dout + at[u] * g.ldo + col);
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int i = 0; i < VW; ++i) s.v[i] += x[u].v[i];
    }
    if (t < b) {
        int at[8];
        Vals<VW> x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) at[u] = g.pos[min(t + u, b - 1)];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = ld<VW>(dout + at[u] * g.ldo + col);
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int i = 0; i < VW; ++i) s.v[i] += t + u < b ? x[u].v[i] : 0.f;
    }
    return s;
}

// One group of lpr lanes per (table row, column block), then per (chunk, column
// block); rows whose run is longer than CHUNK are left to the chunks.
template <typename TO, int VW>
__global__ __launch_bounds__(256) void embed_grad_kernel(const TO* __restrict__ dout, const GradArgs g) {
    const int gl = threadIdx.x & (g.lpr - 1);
    const long item = ((long)blockIdx.x << (8 - g.lpr_shift)) + (threadIdx.x >> g.lpr_shift);
    const long cold = (long)g.vocab * g.ncc;
    const long j = item < cold ? item : item - cold;
    const long r = j / g.ncc;
    const int col = ((int)(j - r * g.ncc) * g.lpr + gl) * VW;
    if (col >= g.d) return;
    if (item < cold) {
        const int a = g.starts[r], b = g.starts[r + 1];
        if (b - a > CHUNK) return;
        Vals<VW> s = run_sum<TO, VW>(dout, g, a, b, col);
#pragma unroll
        for (int i = 0; i < VW; ++i) s.v[i] *= g.scale;
        st<VW>(g.dtable + r * g.ldt + col, s);
        return;
    }
    const int live = *g.live;
    if (r >= g.nchunks || r * CHUNK >= live) return;
    const int a = (int)r * CHUNK, b = min(a + CHUNK, live);
    float* part = g.part + r * 2 * g.d + col;
    const int v0 = g.keys[a], s0 = g.starts[v0], e0 = g.starts[v0 + 1];
    if (e0 - s0 > CHUNK && s0 < a) st<VW>(part, run_sum<TO, VW>(dout, g, a, min(e0, b), col));
    const int v1 = g.keys[b - 1], s1 = g.starts[v1], e1 = g.starts[v1 + 1];
    if (e1 - s1 > CHUNK && s1 >= a) st<VW>(part + g.d, run_sum<TO, VW>(dout, g, s1, b, col));
}

// The chunk a long run starts in folds its pieces: groups take every 256 / lpr th
// piece in order, then add in group order.
template <int VW>
__global__ __launch_bounds__(256) void embed_fold_kernel(const GradArgs g) {
    __shared__ float sh[256 * VW];
    const int gl = threadIdx.x & (g.lpr - 1), grp = threadIdx.x >> g.lpr_shift, ng = 256 >> g.lpr_shift;
    const int c = blockIdx.x / g.ncc, cc = blockIdx.x - c * g.ncc;
    const int live = *g.live;
    if ((long)c * CHUNK >= live) return;
    const int a = c * CHUNK, b = min(a + CHUNK, live);
    const int v = g.keys[b - 1], s0 = g.starts[v], e0 = g.starts[v + 1];
    if (e0 - s0 <= CHUNK || s0 < a) return;      // the same for the whole workgroup
    const int pieces = (e0 - 1) / CHUNK - c + 1;
    const int col = (cc * g.lpr + gl) * VW;
    Vals<VW> s;
#pragma unroll
    for (int i = 0; i < VW; ++i) s.v[i] = 0.f;
    if (col < g.d) {
#pragma unroll 8
        for (int k = grp; k < pieces; k += ng) {
            const Vals<VW> x = ld<VW>(g.part + ((long)(c + k) * 2 + (k == 0)) * g.d + col);
#pragma unroll
            for (int i = 0; i < VW; ++i) s.v[i] += x.v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < VW; ++i) sh[i * 256 + threadIdx.x] = s.v[i];
    __syncthreads();
    if (grp > 0 || col >= g.d) return;
    for (int k = 1; k < ng; ++k)
#pragma unroll
        for (int i = 0; i < VW; ++i) s.v[i] += sh[i * 256 + k * g.lpr + gl];
#pragma unroll
    for (int i = 0; i < VW; ++i) s.v[i] *= g.scale;
    st<VW>(g.dtable + (long)v * g.ldt + col, s);
}

// ------------------------------------------------------------------- host
int bits_for(int vocab) {
    int b = 1;
    while (b < 31 && (1LL << b) < vocab) ++b;
    return b;
}

struct SortPlan { int passes, bits, tile, nb, bins; };
SortPlan sort_plan(long rows, int vocab) {
    SortPlan p;
    const int nb = bits_for(vocab);
    p.passes = nb <= BITS1 ? 1 : (nb + BITS2 - 1) / BITS2;
    p.bits = (nb + p.passes - 1) / p.passes;
    p.bins = 1 << p.bits;
    p.tile = 1024;
    if (rows > (long)MAXB * 1024) p.tile = pt_cdiv(pt_cdiv(rows, MAXB), 1024) * 1024;
    p.nb = rows > 0 ? pt_cdiv(rows, p.tile) : 1;
    return p;
}

// workspace in ints: keys and positions (twice for several digits), counts,
// totals, starts, live, then the chunks' pieces (16 B aligned)
struct Ws { long keys, pos, keys2, pos2, cnt, tot, starts, live, part, total; };
Ws ws_layout(long rows, int vocab, int d) {
    const SortPlan p = sort_plan(rows, vocab);
    Ws w;
    long at = 0;
    auto take = [&](long n) { const long r = at; at += (n + 3) / 4 * 4; return r; };
    w.keys = take(rows); w.pos = take(rows);
    w.keys2 = p.passes > 1 ? take(rows) : 0;
    w.pos2 = p.passes > 1 ? take(rows) : 0;
    w.cnt = take((long)p.bins * p.nb);
    w.tot = take(p.bins);
    w.starts = take((long)vocab + 1);
    w.live = take(1);
    w.part = take(rows > CHUNK ? (long)pt_cdiv(rows, CHUNK) * 2 * d : 0);
    w.total = at;
    return w;
}

bool fits(const void* p, long ld, int esize, int vw) {
    return ((uintptr_t)p % (size_t)(vw * esize < 16 ? vw * esize : 16)) == 0 && ld % vw == 0;
}

template <typename TT, typename TO, int VW>
int launch_fwd(const int* ids, long rows, const void* table, long ldt, int vocab, int d, float scale, void* out,
               long ldo, hipStream_t s) {
    const int cpr = d / VW;
    const long blocks = (rows * cpr + 256 * FWD_U - 1) / (256 * FWD_U);
    PT_REQUIRE(blocks < (1LL << 31), "embedding_fwd: %ld rows of %d are too many", rows, d);
    hipLaunchKernelGGL((embed_fwd_kernel<TT, TO, VW>), dim3((unsigned)blocks), dim3(256), 0, s, ids, rows,
                       static_cast<const TT*>(table), ldt, vocab, cpr, scale, static_cast<TO*>(out), ldo);
    PT_LAUNCH_CHECK();
    return PTCG_OK;
}

template <typename TT, typename TO>
int fwd(const int* ids, long rows, const void* table, long ldt, int vocab, int d, float scale, void* out, long ldo,
        hipStream_t s) {
    const int te = sizeof(TT), oe = sizeof(TO);
    // 16 bytes of the narrower side per thread where both sides allow it, else
    // 4 values, else single ones (odd widths and strides)
    if ((te == 2 || oe == 2) && d % 8 == 0 && fits(table, ldt, te, 8) && fits(out, ldo, oe, 8))
        return launch_fwd<TT, TO, 8>(ids, rows, table, ldt, vocab, d, scale, out, ldo, s);
    if (d % 4 == 0 && fits(table, ldt, te, 4) && fits(out, ldo, oe, 4))
        return launch_fwd<TT, TO, 4>(ids, rows, table, ldt, vocab, d, scale, out, ldo, s);
    return launch_fwd<TT, TO, 1>(ids, rows, table, ldt, vocab, d, scale, out, ldo, s);
}

template <typename TO, int VW>
int launch_grad(const TO* dout, GradArgs g, long rows, hipStream_t s) {
    const int cpr = g.d / VW;
    g.lpr = 1;
    g.lpr_shift = 0;
    while (g.lpr < 64 && g.lpr < cpr) {
        g.lpr <<= 1;
        ++g.lpr_shift;
    }
    g.ncc = pt_cdiv(cpr, g.lpr);
    g.nchunks = rows > CHUNK ? pt_cdiv(rows, CHUNK) : 0;
    const long items = ((long)g.vocab + g.nchunks) * g.ncc, per = 256 >> g.lpr_shift;
    PT_REQUIRE((items + per - 1) / per < (1LL << 31) && (long)g.nchunks * g.ncc < (1LL << 31),
               "embedding_bwd: %d rows of %d are too many", g.vocab, g.d);
    hipLaunchKernelGGL((embed_grad_kernel<TO, VW>), dim3((unsigned)((items + per - 1) / per)), dim3(256), 0, s, dout,
                       g);
    PT_LAUNCH_CHECK();
    if (g.nchunks) {
        hipLaunchKernelGGL(embed_fold_kernel<VW>, dim3((unsigned)(g.nchunks * g.ncc)), dim3(256), 0, s, g);
        PT_LAUNCH_CHECK();
    }
    return PTCG_OK;
}

template <typename TO>
int grad(const void* dout, const GradArgs& g, long rows, hipStream_t s) {
    const TO* x = static_cast<const TO*>(dout);
    if (sizeof(TO) == 2 && g.d % 8 == 0 && fits(x, g.ldo, 2, 8) && fits(g.dtable, g.ldt, 4, 4))
        return launch_grad<TO, 8>(x, g, rows, s);
    if (g.d % 4 == 0 && fits(x, g.ldo, sizeof(TO), 4) && fits(g.dtable, g.ldt, 4, 4))
        return launch_grad<TO, 4>(x, g, rows, s);
    return launch_grad<TO, 1>(x, g, rows, s);
}

int check_sizes(const char* who, int64_t rows, int vocab, int d) {
    PT_REQUIRE(rows >= 0 && rows < (1LL << 30), "%s: %lld rows", who, (long long)rows);
    PT_REQUIRE(vocab >= 1 && d >= 1 && d <= 65536, "%s: vocab=%d d=%d", who, vocab, d);
    return PTCG_OK;
}

}  // namespace

extern "C" int ptcg_kernel_embedding_fwd(const int32_t* ids, int64_t rows, const void* table, int64_t ldt,
                                         int table_bf16, int vocab, int d, float scale, void* out, int64_t ldo,
                                         int out_bf16, void* stream) {
    PT_TRY(check_sizes("embedding_fwd", rows, vocab, d));
    if (rows == 0) return PTCG_OK;
    PT_REQUIRE(ids && table && out, "embedding_fwd: null buffer");
    PT_REQUIRE(ldt >= d && ldo >= d, "embedding_fwd: row strides %lld, %lld below d=%d", (long long)ldt,
               (long long)ldo, d);
    const hipStream_t s = (hipStream_t)stream;
    if (table_bf16)
        return out_bf16 ? fwd<__bf16, __bf16>(ids, rows, table, ldt, vocab, d, scale, out, ldo, s)
                        : fwd<__bf16, float>(ids, rows, table, ldt, vocab, d, scale, out, ldo, s);
    return out_bf16 ? fwd<float, __bf16>(ids, rows, table, ldt, vocab, d, scale, out, ldo, s)
                    : fwd<float, float>(ids, rows, table, ldt, vocab, d, scale, out, ldo, s);
}

extern "C" int64_t ptcg_kernel_embedding_bwd_ws_bytes(int64_t rows, int vocab, int d) {
    if (check_sizes("embedding_bwd_ws_bytes", rows, vocab, d) != PTCG_OK) return -1;
    return ws_layout(rows, vocab, d).total * 4;
}

extern "C" int ptcg_kernel_embedding_bwd(const int32_t* ids, int64_t rows, const void* dout, int64_t ldo, int bf16,
                                         int vocab, int d, float scale, float* dtable, int64_t ldt, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
    PT_TRY(check_sizes("embedding_bwd", rows, vocab, d));
    PT_REQUIRE(dtable && (rows == 0 || (ids && dout)), "embedding_bwd: null buffer");
    PT_REQUIRE(ldt >= d && ldo >= d, "embedding_bwd: row strides %lld, %lld below d=%d", (long long)ldt,
               (long long)ldo, d);
    const Ws w = ws_layout(rows, vocab, d);
    PT_REQUIRE(workspace && workspace_bytes >= w.total * 4 && ((uintptr_t)workspace & 15) == 0,
               "embedding_bwd: workspace of %lld bytes, need %lld (16 B aligned)", (long long)workspace_bytes,
               (long long)(w.total * 4));
    const hipStream_t s = (hipStream_t)stream;
    int* ws = static_cast<int*>(workspace);
    const SortPlan p = sort_plan(rows, vocab);
    SortPass a{};
    a.keys = ids; a.pos = nullptr; a.n_dev = nullptr;
    a.n = (int)rows; a.vocab = vocab; a.bits = p.bits; a.tile = p.tile; a.nb = p.nb;
    a.cnt = ws + w.cnt; a.tot = ws + w.tot;
    a.starts = p.passes == 1 ? ws + w.starts : nullptr;
    const size_t place_lds = (4 * (size_t)p.bins + 256) * sizeof(int);
    for (int k = 0; k < p.passes; ++k) {
        a.shift = k * p.bits;
        a.live = k == 0 ? ws + w.live : nullptr;
        const bool odd = (p.passes - 1 - k) & 1;      // the last pass ends in keys / pos
        a.out_keys = ws + (odd ? w.keys2 : w.keys);
        a.out_pos = ws + (odd ? w.pos2 : w.pos);
        hipLaunchKernelGGL(sort_count_kernel, dim3(a.nb), dim3(256), p.bins * sizeof(int), s, a);
        PT_LAUNCH_CHECK();
        hipLaunchKernelGGL(sort_scan_kernel, dim3(pt_cdiv(p.bins, 4)), dim3(256), 0, s, a);
        PT_LAUNCH_CHECK();
        hipLaunchKernelGGL(sort_place_kernel, dim3(a.nb), dim3(256), place_lds, s, a);
        PT_LAUNCH_CHECK();
        a.keys = a.out_keys; a.pos = a.out_pos; a.n_dev = ws + w.live;
    }
    if (p.passes > 1) {
        hipLaunchKernelGGL(sort_starts_kernel, dim3(pt_cdiv((long)vocab + 1, 256)), dim3(256), 0, s, ws + w.keys,
                           ws + w.live, vocab, ws + w.starts);
        PT_LAUNCH_CHECK();
    }
    GradArgs g{};
    g.keys = ws + w.keys; g.pos = ws + w.pos; g.starts = ws + w.starts; g.live = ws + w.live;
    g.ldo = ldo; g.ldt = ldt; g.vocab = vocab; g.d = d; g.scale = scale; g.dtable = dtable;
    g.part = reinterpret_cast<float*>(ws + w.part);
    return bf16 ? grad<__bf16>(dout, g, rows, s) : grad<float>(dout, g, rows, s);
}
