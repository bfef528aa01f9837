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
// an order that the list alone gives, not scheduling.  Adding by atomics
// instead costs a read-modify-write per element and token, in an order that
// changes; equal ids then queue on the same lines.
// Sort: least significant digit first, 1 digit of up to 11 bits where the
// vocabulary fits, else digits of up to 9 bits; per digit a count per
// workgroup, a scan over the workgroups, and a placement whose ranks within a
// wave come from ballots.  Where the counts are few the placement scans them (a
// launch less: 48 107 tokens of 3 606 ids, two digits of 6 bits, 36 us against 40;
// 90 000 of 50 000, two of 8 bits on 176 workgroups, would take 10 more).  Passes
// are chains of waits more than work: tiles of 512 tokens take 1.5 us less than
// 1 024 of them at 49 152.
// Up to RANK_ROWS tokens each token counts the tokens before it instead (one
// launch for the three of every digit).
// Runs longer than LONG tokens (frequent ids) are added in CHUNK-aligned
// pieces of the sorted list by groups of lanes of their own, and the pieces in a
// fixed order (embed_fold_kernel), so one frequent id does not hold a single
// group for its whole run.  Where a run is cut depends on where it lies, that is
// on the tokens of smaller ids; shorter runs are added in token order.
#include "model.h"
#include "../../include/ptcg_amd_kernels.h"

namespace {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Tokens of one id: up to LONG a group of lanes adds in line; more are added in
// pieces by CHUNK (49 152 tokens, 64 wide, of a Zipf law over 2 048 ids: 34 us
// against 41 with 64 and 64; with 32 and 32 ids of 24 on average lose 3%)
constexpr int LONG = 40, CHUNK = 32;
constexpr int MAXB = 1024;        // workgroups of a sort pass (tiles grow past it)
constexpr int BITS1 = 11, BITS2 = 9;
constexpr int SMALL = 100000;    // tokens up to which a sort pass has twice the workgroups
constexpr int FEW = 8192;        // counts up to which every placing workgroup adds them up itself
constexpr int RANK_ROWS = 4096;  // 16 KB of keys in LDS; 4 096 compares a token

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

// the same as it lies in memory, so that a load in flight takes no more
// registers than its bytes
template <typename T, int VW> struct Raw {
    T v[VW] __attribute__((aligned(sizeof(T) * VW < 16 ? sizeof(T) * VW : 16)));
};
template <typename T, int VW> __device__ __forceinline__ Raw<T, VW> ldraw(const T* p) {
    return *reinterpret_cast<const Raw<T, VW>*>(p);
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
    int* cnt;     // [nb][bins]
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
    for (int i = threadIdx.x; i < bins; i += 256) p.cnt[(long)blockIdx.x * bins + i] = hist[i];
}

// exclusive scan over the workgroups' counts of each digit: a workgroup takes 64
// digits, 16 waves a run of the counting workgroups each
__global__ __launch_bounds__(1024) void sort_scan_kernel(const SortPass p) {
    __shared__ int sums[16][64];
    const int bins = 1 << p.bits, lane = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
    const int per = (p.nb + 15) / 16, b0 = min(w * per, p.nb), b1 = min(b0 + per, p.nb);
    int* c = p.cnt + d;
    int run = 0;
    if (d < bins) {
#pragma unroll 8
        for (int b = b0; b < b1; ++b) run += c[(long)b * bins];
    }
    sums[w][lane] = run;
    __syncthreads();
    int base = 0;
    for (int k = 0; k < 16; ++k) {
        if (k == w) run = base;
        base += sums[k][lane];
    }
    if (d >= bins) return;
#pragma unroll 8
    for (int b = b0; b < b1; ++b) {
        const int v = c[(long)b * bins];
        c[(long)b * bins] = run;
        run += v;
    }
    if (w == 0) p.tot[d] = base;
}

// Placement (SCAN: with the scan).  A wave owns a quarter of the workgroup's tile and walks it 64
// tokens at a time: a token's place is its digit's base, plus the digit's
// tokens before it in earlier workgroups, waves and batches, plus those in
// lower lanes of its batch.
template <int U, bool SCAN> __global__ __launch_bounds__(256) void sort_place_kernel(const SortPass p) {
    extern __shared__ int sm[];
    const int bins = 1 << p.bits, n = pass_n(p);
    int* cnt = sm;               // [4][bins]
    int* tot = sm + 4 * bins;    // [bins]
    int* before = tot + bins;    // [bins], SCAN alone
    int* part = before + (SCAN ? bins : 0);   // [4]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // what the previous launches left, all of it on its way before anything waits
    constexpr int PT = (1 << BITS1) / 256;
    int tv[PT], mv[PT];
    const int* mine = p.cnt + (long)blockIdx.x * bins;
    if constexpr (!SCAN)
#pragma unroll
        for (int i = 0; i < PT; ++i) {
            const int d = min(tid + 256 * i, bins - 1);
            tv[i] = p.tot[d];
            mv[i] = mine[d];
        }
    for (int i = tid; i < (SCAN ? 6 : 4) * bins; i += 256) cnt[i] = 0;
    // U batches' keys at a time (a wave's quarter is a multiple of 64 U tokens)
    const int per = p.tile / 4, w0 = blockIdx.x * p.tile + wave * per;
    int key[U], dig[U];
    auto load = [&](int o) {
#pragma unroll
        for (int u = 0; u < U; ++u) dig[u] = digit_of(p, w0 + o + 64 * u + lane, n, key[u]);
    };
    load(0);
    __syncthreads();
    if constexpr (SCAN) {
        // each digit's counts of all workgroups and of those before this one
        const int w = min(bins, 256), g = tid / w, ng = 256 / w;
        for (int d = tid % w; d < bins; d += w) {
            int all = 0, pre = 0;
#pragma unroll 8
            for (int b = g; b < p.nb; b += ng) {
                const int c = p.cnt[(long)b * bins + d];
                all += c;
                pre += b < (int)blockIdx.x ? c : 0;
            }
            atomicAdd(&tot[d], all);
            atomicAdd(&before[d], pre);
        }
    }
    for (int o = 0; o < per; o += 64 * U) {
        if (o > 0) load(o);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (dig[u] >= 0) atomicAdd(&cnt[wave * bins + dig[u]], 1);
    }
    // exclusive scan of the digits' totals: thread t adds up bpt consecutive digits
    const int bpt = (bins + 255) / 256, d0 = tid * bpt;
    if constexpr (!SCAN)
#pragma unroll
        for (int i = 0; i < PT; ++i)
            if (tid + 256 * i < bins) tot[tid + 256 * i] = tv[i];
    __syncthreads();
    int sum = 0;
    for (int i = 0; i < bpt; ++i)
        if (d0 + i < bins) sum += tot[d0 + i];
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(inc, o, 64);
        if (lane >= o) inc += x;
    }
    if (lane == 63) part[wave] = inc;
    __syncthreads();
    int base = inc - sum, all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) base += part[w];
        all += part[w];
    }
    for (int i = 0; i < bpt; ++i) {
        if (d0 + i >= bins) break;
        const int v = tot[d0 + i];
        tot[d0 + i] = base;
        base += v;
    }
    if (blockIdx.x == 0 && tid == 0) {
        if (p.live) *p.live = all;
        if (p.starts) p.starts[p.vocab] = all;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PT; ++i) {
        const int d = tid + 256 * i;
        if (d >= bins) break;
        const int at = tot[d];
        if (p.starts && blockIdx.x == 0 && d < p.vocab) p.starts[d] = at;
        int run = at + (SCAN ? before[d] : mv[i]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int c = cnt[w * bins + d];
            cnt[w * bins + d] = run;
            run += c;
        }
    }
    __syncthreads();
    for (int o = 0; o < per; o += 64 * U) {
        if (per > 64 * U) load(o);
        int at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int d = dig[u];
            unsigned long long same = __ballot(d >= 0);
            for (int i = 0; i < p.bits; ++i) {
                const unsigned long long b = __ballot((d >> i) & 1);
                same &= ((d >> i) & 1) ? b : ~b;
            }
            const int rank = __popcll(same & ((1ull << lane) - 1));
            int* c = sm + wave * bins + max(d, 0);
            at[u] = *c + rank;      // every lane reads before the digit's first lane moves it on
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (d >= 0 && rank == 0) *c = at[u] + __popcll(same);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (dig[u] >= 0) {
                const int t = w0 + o + 64 * u + lane;
                p.out_keys[at[u]] = key[u];
                p.out_pos[at[u]] = p.pos ? p.pos[t] : t;
            }
    }
}

// A token's place is the number of tokens with a smaller id, or with its id and
// a smaller position; padding goes last.  A workgroup places 64 tokens, each of
// its waves counting over a quarter of all of them.
__global__ __launch_bounds__(256) void sort_rank_kernel(const int* __restrict__ ids, int rows, int vocab,
        int* __restrict__ out_keys, int* __restrict__ out_pos, int* __restrict__ live) {
    __shared__ __align__(16) unsigned keys[RANK_ROWS];
    __shared__ int part[4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, t0 = blockIdx.x * 64, t = t0 + lane;
    const int all = (rows + 15) / 16 * 16;
    constexpr unsigned PAD = 0x80000000u, NONE = 0xffffffffu;   // above every id; past the end
    int kept = 0;
    for (int j = tid; j < all; j += 256) {
        const int id = j < rows ? ids[j] : 0;
        const bool ok = j < rows && (unsigned)id < (unsigned)vocab;
        keys[j] = ok ? (unsigned)id : j < rows ? PAD : NONE;
        kept += ok;
    }
    if (blockIdx.x == 0) {
        for (int o = 32; o > 0; o >>= 1) kept += __shfl_xor(kept, o, 64);
        if (lane == 0) part[wave][0] = kept;
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) *live = part[0][0] + part[1][0] + part[2][0] + part[3][0];
    const unsigned mine = keys[min(t, rows - 1)];
    const int j0 = wave * (all / 4), j1 = j0 + all / 4;
    int n = 0;
    for (int j = j0; j < j1; j += 4) {
        const uint4 k = *reinterpret_cast<const uint4*>(keys + j);
        // tokens before this workgroup's win ties, those after it lose them
        const unsigned m = j < t0 ? mine + 1 : mine;
        n += (k.x < m) + (k.y < m) + (k.z < m) + (k.w < m);
        if (j >= t0 && j < t0 + 64)
            n += (k.x == mine && j < t) + (k.y == mine && j + 1 < t) + (k.z == mine && j + 2 < t) +
                 (k.w == mine && j + 3 < t);
    }
    __syncthreads();
    part[wave][lane] = n;
    __syncthreads();
    if (wave > 0 || t >= rows) return;
    const int at = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
    out_keys[at] = (int)mine;
    out_pos[at] = t;
}

// first sorted position of each id, by binary search (a sort of one digit leaves
// them itself)
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

// sums of dout rows of sorted tokens [a, b) at CB column pieces `step` apart, in
// order; several rows in flight (past the end the last one again, not added)
template <typename TO, int VW, int CB>
__device__ __forceinline__ void run_sum(const TO* __restrict__ dout, const GradArgs& g, int a, int b,
                                        const int (&col)[CB], Vals<VW> (&s)[CB]) {
    constexpr int U = VW * sizeof(TO) * CB <= 16 ? 8 : 4;
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int i = 0; i < VW; ++i) s[c].v[i] = 0.f;
    for (int t = a; t < b; t += U) {
        int at[U];
        Raw<TO, VW> x[U][CB];
#pragma unroll
        for (int u = 0; u < U; ++u) at[u] = g.pos[min(t + u, b - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < CB; ++c) x[u][c] = ldraw<TO, VW>(dout + at[u] * g.ldo + col[c]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < CB; ++c)
#pragma unroll
                for (int i = 0; i < VW; ++i) s[c].v[i] += t + u < b ? (float)x[u][c].v[i] : 0.f;
    }
}

// One group of lpr lanes per (table row, column block of CB * lpr * VW), then per
// (chunk, column block); rows whose run is longer than LONG are left to the
// chunks.  Wide rows take two pieces a lane (CB = 2): a row of few tokens is a
// chain of dependent loads, and half as many groups walk it (300 007 tokens of
// 1 024 bf16 values, 100 003 ids: 250 us against 269 with one piece).
template <typename TO, int VW, int CB>
__global__ __launch_bounds__(256) void embed_grad_kernel(const TO* __restrict__ dout, const GradArgs g) {
    const int gl = threadIdx.x & (g.lpr - 1);
    const long item = ((long)blockIdx.x << (8 - g.lpr_shift)) + (threadIdx.x >> g.lpr_shift);
    const long cold = (long)g.vocab * g.ncc;
    const long j = item < cold ? item : item - cold;
    const long r = j / g.ncc;
    int col[CB];
    bool ok[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) {
        const int x = (((int)(j - r * g.ncc) * CB + c) * g.lpr + gl) * VW;
        ok[c] = x < g.d;
        col[c] = ok[c] ? x : 0;
    }
    if (!ok[0]) return;
    Vals<VW> s[CB];
    if (item < cold) {
        const int a = g.starts[r], b = g.starts[r + 1];
        if (b - a > LONG) return;
        run_sum<TO, VW, CB>(dout, g, a, b, col, s);
#pragma unroll
        for (int c = 0; c < CB; ++c) {
#pragma unroll
            for (int i = 0; i < VW; ++i) s[c].v[i] *= g.scale;
            if (ok[c]) st<VW>(g.dtable + r * g.ldt + col[c], s[c]);
        }
        return;
    }
    const int live = *g.live;
    if (r >= g.nchunks || r * CHUNK >= live) return;
    const int a = (int)r * CHUNK, b = min(a + CHUNK, live);
    float* part = g.part + r * 2 * g.d;
    const int v0 = g.keys[a], s0 = g.starts[v0], e0 = g.starts[v0 + 1];
    if (e0 - s0 > LONG && s0 < a) {
        run_sum<TO, VW, CB>(dout, g, a, min(e0, b), col, s);
#pragma unroll
        for (int c = 0; c < CB; ++c)
            if (ok[c]) st<VW>(part + col[c], s[c]);
    }
    const int v1 = g.keys[b - 1], s1 = g.starts[v1], e1 = g.starts[v1 + 1];
    if (e1 - s1 > LONG && s1 >= a) {
        run_sum<TO, VW, CB>(dout, g, s1, b, col, s);
#pragma unroll
        for (int c = 0; c < CB; ++c)
            if (ok[c]) st<VW>(part + g.d + col[c], s[c]);
    }
}

constexpr int FOLD = 512;
// The chunk a long run starts in folds its pieces: groups take every FOLD / lpr th
// piece in order, then add in group order.
template <int VW>
__global__ __launch_bounds__(FOLD) void embed_fold_kernel(const GradArgs g) {
    __shared__ float sh[FOLD * VW];
    const int gl = threadIdx.x & (g.lpr - 1), grp = threadIdx.x >> g.lpr_shift, ng = FOLD >> g.lpr_shift;
    const int c = blockIdx.x / g.ncc, cc = blockIdx.x - c * g.ncc;
    const int live = *g.live;
    if ((long)c * CHUNK >= live) return;
    const int a = c * CHUNK, b = min(a + CHUNK, live);
    const int v = g.keys[b - 1], s0 = g.starts[v], e0 = g.starts[v + 1];
    if (e0 - s0 <= LONG || s0 < a) return;      // the same for the whole workgroup
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
    for (int i = 0; i < VW; ++i) sh[i * FOLD + threadIdx.x] = s.v[i];
    __syncthreads();
    if (grp > 0 || col >= g.d) return;
    for (int k = 1; k < ng; ++k)
#pragma unroll
        for (int i = 0; i < VW; ++i) s.v[i] += sh[i * FOLD + k * g.lpr + gl];
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

struct SortPlan { int passes, bits, tile, nb, bins; bool scan; };   // passes 0: by rank
SortPlan sort_plan(long rows, int vocab) {
    SortPlan p;
    const int nb = bits_for(vocab);
    p.passes = nb <= BITS1 ? 1 : (nb + BITS2 - 1) / BITS2;
    if (rows <= RANK_ROWS) {
        p = SortPlan{};
        return p;
    }
    p.bits = (nb + p.passes - 1) / p.passes;
    p.bins = 1 << p.bits;
    p.tile = rows <= SMALL ? 512 : 1024;
    if (rows > (long)MAXB * 1024) p.tile = pt_cdiv(pt_cdiv(rows, MAXB), 1024) * 1024;
    p.nb = pt_cdiv(rows, p.tile);
    p.scan = (long)p.bins * p.nb > FEW;
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
    w.live = take(4);
    w.part = take(rows > LONG ? (long)pt_cdiv(rows, CHUNK) * 2 * d : 0);
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
    PT_REQUIRE(blocks < (1LL << 24), "embedding_fwd: %ld rows of %d are too many", rows, d);   // 2^32 threads
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

// A group's lanes and the launches over a table's rows and the sorted list's chunks
struct GradPlan { int vw, lpr, lpr_shift, cb, ncc, fold_ncc, nchunks; long blocks; };
GradPlan grad_plan(const void* dout, long ldo, int bf16, int vocab, int d, const float* dtable, long ldt, long rows) {
    GradPlan p;
    const int e = bf16 ? 2 : 4;
    p.vw = d % 4 || !fits(dout, ldo, e, 4) || !fits(dtable, ldt, 4, 4) ? 1
           : bf16 && d % 8 == 0 && fits(dout, ldo, e, 8)               ? 8
                                                                        : 4;
    const int cpr = d / p.vw;
    p.lpr = 1;
    p.lpr_shift = 0;
    while (p.lpr < 64 && p.lpr < cpr) {
        p.lpr <<= 1;
        ++p.lpr_shift;
    }
    p.fold_ncc = pt_cdiv(cpr, p.lpr);      // the fold's column blocks; the sums' are cb times as wide
    p.cb = p.fold_ncc > 1 ? 2 : 1;
    p.ncc = pt_cdiv(p.fold_ncc, p.cb);
    p.nchunks = rows > LONG ? pt_cdiv(rows, CHUNK) : 0;
    const long items = ((long)vocab + p.nchunks) * p.ncc, per = 256 >> p.lpr_shift;
    p.blocks = (items + per - 1) / per;
    return p;
}

template <typename TO, int VW> int launch_grad(const TO* dout, GradArgs g, const GradPlan& p, hipStream_t s) {
    auto kern = p.cb == 2 ? embed_grad_kernel<TO, VW, 2> : embed_grad_kernel<TO, VW, 1>;
    g.lpr = p.lpr; g.lpr_shift = p.lpr_shift; g.ncc = p.ncc; g.nchunks = p.nchunks;
    hipLaunchKernelGGL(kern, dim3((unsigned)p.blocks), dim3(256), 0, s, dout, g);
    PT_LAUNCH_CHECK();
    if (g.nchunks) {
        g.ncc = p.fold_ncc;
        hipLaunchKernelGGL(embed_fold_kernel<VW>, dim3((unsigned)(g.nchunks * g.ncc)), dim3(FOLD), 0, s, g);
        PT_LAUNCH_CHECK();
    }
    return PTCG_OK;
}

template <typename TO> int grad(const void* dout, const GradArgs& g, const GradPlan& p, hipStream_t s) {
    const TO* x = static_cast<const TO*>(dout);
    if constexpr (sizeof(TO) == 2)
        if (p.vw == 8) return launch_grad<TO, 8>(x, g, p, s);
    return p.vw == 4 ? launch_grad<TO, 4>(x, g, p, s) : launch_grad<TO, 1>(x, g, p, s);
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
    // a launch holds fewer than 2^32 threads
    const GradPlan gp = grad_plan(dout, ldo, bf16, vocab, d, dtable, ldt, rows);
    PT_REQUIRE(gp.blocks < (1LL << 24) && (long)gp.nchunks * gp.fold_ncc < (1LL << 32) / FOLD,
               "embedding_bwd: %lld tokens and a table of %d rows of %d are too many", (long long)rows, vocab, d);
    const hipStream_t s = (hipStream_t)stream;
    int* ws = static_cast<int*>(workspace);
    const SortPlan p = sort_plan(rows, vocab);
    if (p.passes == 0 && rows > 0) {
        hipLaunchKernelGGL(sort_rank_kernel, dim3(pt_cdiv(rows, 64)), dim3(256), 0, s, ids, (int)rows, vocab,
                           ws + w.keys, ws + w.pos, ws + w.live);
        PT_LAUNCH_CHECK();
    }
    if (rows == 0) PT_TRY(pt_fill_zero(reinterpret_cast<float*>(ws + w.live), 4, s));
    SortPass a{};
    a.keys = ids; a.pos = nullptr; a.n_dev = nullptr;
    a.n = (int)rows; a.vocab = vocab; a.bits = p.bits; a.tile = p.tile; a.nb = p.nb;
    a.cnt = ws + w.cnt; a.tot = ws + w.tot;
    a.starts = p.passes == 1 ? ws + w.starts : nullptr;
    const size_t place_lds = ((p.scan ? 5 : 6) * (size_t)p.bins + 4) * sizeof(int);
    for (int k = 0; k < p.passes; ++k) {
        a.shift = k * p.bits;
        a.live = k == 0 ? ws + w.live : nullptr;
        const bool odd = (p.passes - 1 - k) & 1;      // the last pass ends in keys / pos
        a.out_keys = ws + (odd ? w.keys2 : w.keys);
        a.out_pos = ws + (odd ? w.pos2 : w.pos);
        hipLaunchKernelGGL(sort_count_kernel, dim3(a.nb), dim3(256), p.bins * sizeof(int), s, a);
        PT_LAUNCH_CHECK();
        if (p.scan) {
            hipLaunchKernelGGL(sort_scan_kernel, dim3(pt_cdiv(p.bins, 64)), dim3(1024), 0, s, a);
            PT_LAUNCH_CHECK();
        }
        auto place = p.tile == 512 ? (p.scan ? sort_place_kernel<2, false> : sort_place_kernel<2, true>)
                                   : (p.scan ? sort_place_kernel<4, false> : sort_place_kernel<4, true>);
        hipLaunchKernelGGL(place, dim3(a.nb), dim3(256), place_lds, s, a);
        PT_LAUNCH_CHECK();
        a.keys = a.out_keys; a.pos = a.out_pos; a.n_dev = ws + w.live;
    }
    if (p.passes != 1) {
        hipLaunchKernelGGL(sort_starts_kernel, dim3(pt_cdiv((long)vocab + 1, 256)), dim3(256), 0, s, ws + w.keys,
                           ws + w.live, vocab, ws + w.starts);
        PT_LAUNCH_CHECK();
    }
    GradArgs g{};
    g.keys = ws + w.keys; g.pos = ws + w.pos; g.starts = ws + w.starts; g.live = ws + w.live;
    g.ldo = ldo; g.ldt = ldt; g.vocab = vocab; g.d = d; g.scale = scale; g.dtable = dtable;
    g.part = reinterpret_cast<float*>(ws + w.part);
    return bf16 ? grad<__bf16>(dout, g, gp, s) : grad<float>(dout, g, gp, s);
}
