// qdb_sample.cu - next-token sampling from given random numbers: temperature,
// top-k, top-p and min-p per row.
//
// With z_i = (l_i - max l) / T and weights w_i = exp(z_i), tokens ordered by
// (logit descending, index ascending), token i stays when
//   its rank is below top_k,
//   the weights before it sum to less than top_p * (sum over the top_k), and
//   w_i >= min_p;
// the token drawn is the first kept one, in index order, at which the running
// sum of the kept weights exceeds uniform * (their total). NaN logits count as
// -inf.
//
// Sums are 64-bit integers: w is rounded to a multiple of 2^-45 (a token more
// than 31.5 T below the maximum is never drawn), so a sum over up to 2^18 tokens
// is exact and independent of the order of the atomics. The weights themselves
// are off by up to 2^-42.6 of each (a polynomial cut after degree 5) and that
// rounding, 2^-46 of the largest; a border between two tokens is off by the sum
// of these.
// (uniform = 0 asks for the first kept token of any weight above zero: there
// every such token counts 1.)
//
// A row is read from HBM once: a cluster of up to 8 CTAs (as many as leave each
// at least 16K tokens) keeps it in shared memory as order-preserving integers.
//   1. maximum (and the greedy token) over the cluster
//   2. the first CTA collects a histogram of the logits below the maximum (2048
//      bins as far down as weights are above zero) and from it the bin in which
//      the top_k or the top_p ends at the latest
//   3. the tokens down to that bin, if at most 2048, go to the first CTA, which
//      sorts them, cuts exactly, sorts the rest by index and draws
// Where more tokens than that may stay (a flat distribution), only the bins
// that hold the end of the top_k, then of the top_p, go to the first CTA, which
// finds the last token that stays; every CTA then draws from its own tokens.
// Bins of more than 2048 (many equal logits) are cut by a radix selection. All
// ways take the same integer weights, so they give the same token.
//
// Measured, 151936 f32 logits a row: one row with top_k 50 and top_p 0.95 12.6 us
// (4.7 us greedy, 40 us top_p alone), 64 rows of mixed parameters 49 us, 18 rows of
// top_k 50 17 us. Reading the logits would take 0.1 and 6 us: what bounds it is
// one row's own chain of passes and cluster barriers (1000 clocks each). Clocks of
// a row with top_p alone, 73500 in all: start 2000, logits and maximum 6900, the
// pass that weighs and counts all tokens 14200 (16 warps of an SM: its 45
// instructions per token alone would be 6700), barrier and merge of the histograms
// 5200, bins of the cut 5900, their keys 1600, the pass that weighs the tokens
// above them 16900, sort and cut 9600, the sum below 5000, the draw 6200. A mixed
// batch waits for such rows. A first version, one CTA per row and the logits read
// again in every pass, took 609 and 3176 us. (40 bytes of the 64 registers spill.)
#include <cooperative_groups.h>
#include <math.h>
#include <stdio.h>

#include "qdb_kernels.h"
#include "qdb_paged.cuh"

namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;
constexpr int ST = 512, SW = ST / 32;       // threads and warps per CTA
constexpr int SC = 8;                       // CTAs per cluster, at most
constexpr int BINS = 2048, LIST = 2048;     // histogram bins; tokens the first CTA takes
constexpr int SLICE = QDB_SAMPLE_MAX_VOCAB / SC;  // tokens per CTA, at most
constexpr double S_ONE = 35184372088832.0;  // 2^45
constexpr float S_REACH = 31.5f;            // exp(-31.5) = 2^-45.4: what lies further down is left out

template <int TYPE>
__device__ __forceinline__ float widen(uint32_t bits) {
    return TYPE == QDB_TYPE_F32 ? __uint_as_float(bits) : TYPE == QDB_TYPE_F16 ? QdbHalf::lo(bits) : QdbBf16::lo(bits);
}

// Order-preserving integer of a logit: 0 for NaN and -inf (never drawn); -0
// and +0 are equal.
__device__ __forceinline__ uint32_t logit_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);  // (-0 becomes +0)
    const uint32_t k = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
    return k - 0x00800000u <= 0xff000000u ? k : 0u;  // from the lowest number (0x00800000) to +inf (0xff800000)
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float(k ^ ((uint32_t)((int)~k >> 31) | 0x80000000u));
}

template <typename X>
__device__ __forceinline__ X warp_scan(X v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const X y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}

struct Pick {     // of one digit of the radix selection
    int digit;
    unsigned ties;
    u64 above;    // count or weight above the digit
};

enum Way { ALL_LISTED, K_BIN, P_BINS, RADIX };
struct Plan {     // what the CTAs do next: bins lo .. hi go to the list
    int way, lo, hi;
};

struct alignas(16) SampleSmem {
    union {
        struct {
            unsigned n[BINS], f[BINS];  // tokens; their places within the bin, in 1 / 4096, added up
            // (also the scratch of a sorting list, which goes on into f)
        } hist;
        u64 val[LIST];
    };
    union {
        u64 list[LIST];
        struct {
            u64 w[256], lead_w[256];
            unsigned n[256], lead_n[256];
        } dig;
    };
    double exp2_16[16];  // 2^(45 + i / 16): a warp's reads have no bank conflict
    u64 scan[SW + 1];
    float scan_f[SW + 1];
    u64 best[SC], total[SC];
    uint32_t low[SC];
    u64 weight;      // first CTA: a sum of weights
    unsigned count;  // tokens in the list
    unsigned offset;
    u64 cut;         // the last token that stays
    int lo, hi;      // first CTA
    uint32_t ends[2];
    Plan plan;
    Pick pick;
};

// Exclusive prefix over the CTA; *all = the sum.
template <typename X>
__device__ __forceinline__ X block_scan(X v, X *buf, int lane, int warp, X *all) {
    const X in = warp_scan(v, lane);
    __syncthreads();
    if (lane == 31) buf[warp] = in;
    __syncthreads();
    X pre = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < SW; w++) {
        if (w < warp) pre += buf[w];
        sum += buf[w];
    }
    *all = sum;
    return pre + in - v;
}

// n2 (a power of two, at least 64) values, all different but for zeros, in
// descending order. Up to 128 by counting the larger ones of each; more by
// buckets of equal width, in which each value counts the larger ones (583 values:
// 5300 clocks, the bitonic network 15900); where a bucket has too many for that
// (equal logits), by a bitonic network, whose steps over distances up to 32 stay
// within 64 values of one warp. scratch: BINS + 2 words.
__device__ void sort_down(u64 *x, int n2, unsigned *scratch, unsigned *scan, int t) {
    __syncthreads();
    if (n2 <= 128) {
        const u64 mine = t < n2 ? x[t] : 0;
        const int m = __syncthreads_count(mine != 0);
        int at = 0;
        if (mine)
#pragma unroll 8
            for (int i = 0; i < n2; i += 2) {
                const ulonglong2 y = *reinterpret_cast<const ulonglong2 *>(x + i);
                at += (y.x > mine) + (y.y > mine);
            }
        __syncthreads();
        if (mine) x[at] = mine;
        if (t >= m && t < n2) x[t] = 0;
        __syncthreads();
        return;
    }
    constexpr int MINE = LIST / ST, FULL = 32;
    static_assert(BINS == ST * MINE, "a thread has as many buckets as values");
    u64 v[MINE];
    unsigned hi = 0, lo = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < MINE; e++) {
        v[e] = t + e * ST < n2 ? x[t + e * ST] : 0;
        if (v[e]) hi = max(hi, (unsigned)(v[e] >> 32)), lo = min(lo, (unsigned)(v[e] >> 32));
        scratch[t + e * ST] = 0;
    }
    unsigned *ends = scratch + BINS;
    if (t == 0) ends[0] = 0, ends[1] = 0xffffffffu;
    __syncthreads();
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo = __reduce_min_sync(0xffffffffu, lo);
    if ((t & 31) == 0) {
        atomicMax(ends, hi);
        atomicMin(ends + 1, lo);
    }
    __syncthreads();
    hi = ends[0];
    const float per = (float)BINS / ((float)(hi - ends[1]) + 1.f);  // (monotone: rounding moves no value past another)
    int bucket[MINE];
    unsigned slot[MINE];
    bool full = false;
#pragma unroll
    for (int e = 0; e < MINE; e++) {
        bucket[e] = min(BINS - 1, (int)((float)(hi - (unsigned)(v[e] >> 32)) * per));
        slot[e] = v[e] ? atomicAdd(scratch + bucket[e], 1u) : 0;
        full |= slot[e] >= FULL;
    }
    if (!__syncthreads_or(full)) {
        const uint4 c = reinterpret_cast<const uint4 *>(scratch)[t];
        unsigned m;
        const unsigned first = block_scan<unsigned>(c.x + c.y + c.z + c.w, scan, t & 31, t >> 5, &m);
        reinterpret_cast<uint4 *>(scratch)[t] = make_uint4(first, first + c.x, first + c.x + c.y, first + c.x + c.y + c.z);
        if (t == 0) scratch[BINS] = m;
        __syncthreads();
        unsigned at[MINE];
#pragma unroll
        for (int e = 0; e < MINE; e++)
            if (v[e]) x[at[e] = scratch[bucket[e]] + slot[e]] = v[e];
        for (int i = m + t; i < n2; i += ST) x[i] = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < MINE; e++) {
            if (!v[e]) continue;
            const unsigned b0 = scratch[bucket[e]], b1 = scratch[bucket[e] + 1];
            at[e] = b0;
            for (unsigned i = b0; i < b1; i++) at[e] += x[i] > v[e];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < MINE; e++)
            if (v[e]) x[at[e]] = v[e];
        __syncthreads();
        return;
    }
    for (int k = 2; k <= n2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int p = t; p < n2 / 2; p += ST) {
                const int i = 2 * p - (p & (j - 1)), q = i + j;
                const u64 a = x[i], b = x[q];
                if ((a < b) == ((i & k) == 0)) x[i] = b, x[q] = a;
            }
            // (the next step is over j / 2, or over k where this one was over 1)
            if (j > 32 || (j == 1 && k > 32)) __syncthreads();
            else __syncwarp();
        }
    __syncthreads();
}

// What a row's parameters ask for: 0 the largest logit, 1 the threads' maxima
// and a short list, 2 passes over all its tokens. C: CTAs of its cluster.
struct Asked {
    float T, top_p, min_p;
    int top_k;
    __device__ __forceinline__ Asked(const QdbSampleArgs &a, int row)
        : T(a.temperature ? a.temperature[row] : 1.f), top_p(a.top_p ? a.top_p[row] : 1.f),
          min_p(a.min_p ? a.min_p[row] : 0.f), top_k(a.top_k ? a.top_k[row] : 0) {}
    __device__ __forceinline__ bool greedy() const { return !(T > 0.f) || top_p <= 0.f || min_p > 1.f || top_k == 1; }
    __device__ __forceinline__ int work(int C) const { return greedy() ? 0 : top_k > 0 && top_k <= C * ST / 4 ? 1 : 2; }
};

// Where not all clusters run at once, those that start first take the rows with
// the most work: the cluster's row, ordered so within its 128 rows (64 rows of
// mixed parameters: 67 us in the rows' own order, 56 so).
__device__ __forceinline__ int heavy_first(const QdbSampleArgs &a, int at, int C, int lane) {
    const int first = at & ~127;
    int nth = at - first, work[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int row = first + e * 32 + lane;
        work[e] = row < a.rows ? Asked(a, row).work(C) : -1;
    }
    for (int w = 2; w >= 0; w--)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const unsigned b = __ballot_sync(0xffffffffu, work[e] == w);
            if (nth < __popc(b)) {
                const unsigned hit = __ballot_sync(0xffffffffu, (b >> lane & 1) && __popc(b & ((1u << lane) - 1)) == nth);
                return first + e * 32 + __ffs(hit) - 1;
            }
            nth -= __popc(b);
        }
    return at;  // (not reached)
}

template <int TYPE>
__global__ void __launch_bounds__(ST, 2) sample_kernel(const QdbSampleArgs a, int slice, bool ordered) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    SampleSmem &sm = *reinterpret_cast<SampleSmem *>(smem_raw);
    uint32_t *keys = reinterpret_cast<uint32_t *>(smem_raw + sizeof(SampleSmem));
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    int row = blockIdx.x / C;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.vocab;
    const int base = min(V, rank * slice), n = min(V, base + slice) - base;  // this CTA's tokens
    SampleSmem *lead = cl.map_shared_rank(&sm, 0);
    for (int i = t; i < BINS; i += ST) sm.hist.n[i] = 0, sm.hist.f[i] = 0;
    if (t == 0) sm.weight = 0, sm.count = 0, sm.total[0] = 0;
    if (t < 16) sm.exp2_16[t] = exp2(45.0 + t / 16.0);
    cl.barrier_arrive();  // (waited for before the first access to another CTA's memory)
    pdl_enter();
    if (ordered) row = heavy_first(a, row, C, lane);
    const size_t out_at = (a.step ? (size_t)*a.step * a.rows : 0) + row;
    const Asked ask(a, row);
    const float T = ask.T, top_p = ask.top_p, min_p = ask.min_p;
    const int top_k = ask.top_k;
    const float u = a.uniform[out_at];

    // ---- 1. the row into shared memory; its maximum
    // (thread t has tokens 4 t .. 4 t + 3, those 4 ST further on, and so on)
    u64 best = 0;
    uint32_t bk = 0, bi = 0;      // this thread's largest key, its first place
    uint32_t low = 0xffffffffu;   // smallest key above 0, less 1
    {
        constexpr int ES = TYPE == QDB_TYPE_F32 ? 4 : 2;
        const char *src = (const char *)a.logits + ((size_t)row * a.row_stride + base) * ES;
        const bool vec = ((uintptr_t)src & (4 * ES - 1)) == 0;
        constexpr int B = 4;  // loads in flight
        for (int i = t * 4; i < n; i += B * ST * 4) {
            uint4 x[B];
#pragma unroll
            for (int e = 0; e < B; e++) {
                const int j = i + e * ST * 4;
                const char *at = src + (size_t)j * ES;
                if (vec && j + 4 <= n) {
                    if (ES == 4) {
                        x[e] = ldg_stream(at);
                    } else {
                        const uint2 y = *reinterpret_cast<const uint2 *>(at);
                        x[e] = make_uint4(y.x & 0xffffu, y.x >> 16, y.y & 0xffffu, y.y >> 16);
                    }
                } else {
                    uint32_t w[4];
#pragma unroll
                    for (int f = 0; f < 4; f++)
                        w[f] = j + f >= n ? (TYPE == QDB_TYPE_F32 ? 0xff800000u : TYPE == QDB_TYPE_F16 ? 0xfc00u : 0xff80u)
                               : ES == 4  ? reinterpret_cast<const uint32_t *>(src)[j + f]
                                          : (uint32_t) reinterpret_cast<const uint16_t *>(src)[j + f];  // (-inf behind the end)
                    x[e] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
#pragma unroll
            for (int e = 0; e < B; e++) {
                const int j = i + e * ST * 4;
                if (j >= n) break;
                uint32_t k[4] = {logit_key(widen<TYPE>(x[e].x)), logit_key(widen<TYPE>(x[e].y)),
                                 logit_key(widen<TYPE>(x[e].z)), logit_key(widen<TYPE>(x[e].w))};
                if (a.mask_eos)
#pragma unroll
                    for (int f = 0; f < 4; f++)
                        if (base + j + f == QDB_ENDOFTEXT || base + j + f == QDB_IM_END) k[f] = 0;
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    if (k[f] > bk) bk = k[f], bi = j + f;
                    low = min(low, k[f] - 1);  // (0 wraps round: not counted)
                }
                *reinterpret_cast<uint4 *>(keys + j) = make_uint4(k[0], k[1], k[2], k[3]);
            }
        }
        if (bk) best = (u64)bk << 32 | (0xffffffffu - (uint32_t)(base + bi));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 y = __shfl_xor_sync(0xffffffffu, best, o);
        best = y > best ? y : best;
    }
    low = __reduce_min_sync(0xffffffffu, low);
    if (lane == 0) sm.scan[warp] = best, sm.scan_f[warp] = __uint_as_float(low);
    __syncthreads();
    cl.barrier_wait();
    if (t < C) {
        for (int w = 0; w < SW; w++) {
            best = sm.scan[w] > best ? sm.scan[w] : best;
            low = min(low, __float_as_uint(sm.scan_f[w]));
        }
        SampleSmem *o = cl.map_shared_rank(&sm, t);
        o->best[rank] = best;
        o->low[rank] = low;
    }
    cl.sync();
    for (int r = 0; r < C; r++) {
        best = sm.best[r] > best ? sm.best[r] : best;
        low = min(low, sm.low[r]);
    }
    if (best == 0 || ask.greedy()) {
        if (rank == 0 && t == 0) a.tokens[out_at] = best ? (int)(0xffffffffu - (uint32_t)best) : -1;
        return;
    }
    const uint32_t kmax = (uint32_t)(best >> 32);
    const float fmax = key_logit(kmax);
    const bool top_inf = isinf(fmax);  // (then only tokens that share it weigh)
    const double lmax = top_inf ? 0.0 : (double)fmax;
    const bool k_on = top_k > 0 && top_k < V, p_on = top_p < 1.f, first = !(u > 0.f);
    // 2^45 exp((l - max) / T) = 2^45 2^(y / 16) by 2^(i / 16) from the table times a
    // polynomial of degree 5 in x = y - i, |x| <= 1/2 (the next term is below 2^-42)
    const double c16 = 16.0 * 1.4426950408889634074 / (double)T;
    constexpr double E1 = 0.69314718055994530942 / 16, E2 = E1 * E1 / 2, E3 = E2 * E1 / 3, E4 = E3 * E1 / 4, E5 = E4 * E1 / 5;
    // keys below `least` (logits more than `reach` below the maximum) weigh
    // nothing; with an infinite maximum only those that share it weigh
    const float reach = S_REACH * T, bottom = fmax - reach;
    const uint32_t least = isnan(bottom) ? kmax : max(1u, min(kmax, logit_key(bottom)));
    auto weightless = [&](uint32_t k) { return k < least; };
    auto real_weight = [&](uint32_t k) -> double {  // without a branch: 0 where it is weightless
        const double d = (double)(top_inf ? 0.f : key_logit(k)) - lmax, magic = 6755399441055744.0;  // 1.5 * 2^52
        const double y = fma(d, c16, magic);
        const int i = __double2loint(y);
        const double x = fma(d, c16, magic - y);
        double e = fma(x, E5, E4);
        e = fma(x, e, E3);
        e = fma(x, e, E2);
        e = fma(x, e, E1);
        e = fma(x, e, 1.0) * sm.exp2_16[i & 15];
        e = __hiloint2double(__double2hiint(e) + ((i >> 4) << 20), __double2loint(e));
        return weightless(k) ? 0.0 : e;
    };
    auto whole_weight = [&](double w) -> u64 {  // rounded to an integer (below 2^51)
        return (u64)__double_as_longlong(w + 4503599627370496.0) & ((1ull << 52) - 1);
    };
    auto weight = [&](uint32_t k) { return whole_weight(real_weight(k)); };
    // The same as a double: a thread's up to 64 tokens add up to an exact integer
    // below 2^52, without the 64-bit additions' instructions.
    auto whole = [&](double w) { return (w + 4503599627370496.0) - 4503599627370496.0; };
    // Calls f(i, k) for this CTA's tokens i .. i + 3 with keys k[4], whose
    // arithmetic then overlaps (0 behind the end).
    auto each4 = [&](auto f) {
        for (int i = t * 4; i < n; i += ST * 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(keys + i);
            const uint32_t k[4] = {x.x, x.y, x.z, x.w};
            f(i, k);
        }
    };
    auto token_of = [&](uint32_t k, int i) { return (u64)k << 32 | (0xffffffffu - (uint32_t)(base + i)); };
    auto token = [&](int i) { return (u64)keys[i] << 32 | (0xffffffffu - (uint32_t)(base + i)); };
    auto warp_total = [&](u64 v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    // Tokens to the first CTA's list (in any order): each CTA collects in its own
    // list, then sends it; a barrier of the cluster has to follow.
    auto open_list = [&] {
        if (rank) {
            __syncthreads();
            if (t == 0) sm.count = 0;
            __syncthreads();
        }
    };
    auto push = [&](uint32_t k, int i) {
        const unsigned at = atomicAdd(&sm.count, 1u);
        if (at < LIST) sm.list[at] = token_of(k, i);
    };
    auto send_list = [&] {
        if (rank) {
            __syncthreads();
            if (t == 0) sm.offset = atomicAdd(&lead->count, sm.count);
            __syncthreads();
            const unsigned at = sm.offset;
            for (int i = t; i < (int)min(sm.count, (unsigned)LIST); i += ST)
                if (at + i < LIST) lead->list[at + i] = sm.list[i];
        }
    };
    auto gather = [&](uint32_t from, auto take) {  // those that `take` wants, none below `from`
        open_list();
        if (bk >= from)  // (else this thread has no key from there on)
            each4([&](int i, const uint32_t *k) {
                bool yes[4];
#pragma unroll
                for (int e = 0; e < 4; e++) yes[e] = take(k[e], i + e);
                if (!(yes[0] | yes[1] | yes[2] | yes[3])) return;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (yes[e]) push(k[e], i + e);
            });
        send_list();
    };
    // First CTA: sorts the list; returns its length.
    auto sort_list = [&](int *n2) {
        const int m = min((int)sm.count, LIST);
        *n2 = 64;
        while (*n2 < m) *n2 <<= 1;
        for (int i = m + t; i < *n2; i += ST) sm.list[i] = 0;
        sort_down(sm.list, *n2, sm.hist.n, reinterpret_cast<unsigned *>(sm.scan), t);  // (the histogram has been used)
        return m;
    };
    constexpr int PT = BINS / ST;  // bins, or list entries, of a thread
    u64 cut = 0, min_cut = 0;      // tokens from here up stay (by top_k and top_p, by min_p)
    int way = RADIX;

    // ---- 2. histogram: how far down the kept tokens can go
    const float span = fminf(reach, fmax - key_logit(low + 1)), s = span > 0.f ? BINS * 4096.f / span : 0.f;
    auto place_of = [&](uint32_t k) { return min(BINS * 4096 - 1, (int)((fmax - key_logit(k)) * s)); };
    auto bin_of = [&](uint32_t k) { return place_of(k) >> 12; };
    // The smallest key from `least` on that `in` holds for (it holds for larger
    // ones and for kmax), found by the warp 32 at a time.
    auto first_key = [&](auto in) {
        uint32_t lo = least, width = kmax - least + 1;  // the key is in [lo, lo + width)
        while (width > 1) {
            const uint32_t step = (width + 31) / 32;
            const u64 end = (u64)(lane + 1) * step;  // lane's group: does its last key qualify?
            const bool yes = end >= width || in(lo + (uint32_t)end - 1);
            const uint32_t g = __ffs(__ballot_sync(0xffffffffu, yes)) - 1;
            lo += g * step;
            width = min(step, width - g * step);
        }
        return lo;
    };
    // The smallest key of bins 0 .. bin: mostly one of the 32 about where it should be
    // (2000 clocks less than the search).
    auto bin_start = [&](int bin) {
        const uint32_t low = logit_key(fmax - (float)(bin + 1) * (4096.f / s)) - 16;
        if (low >= least && low < kmax - 32) {
            const unsigned in = __ballot_sync(0xffffffffu, bin_of(low + lane) <= bin);
            if (in && !(in & 1)) return low + __ffs(in) - 1;
        }
        return first_key([&](uint32_t k) { return bin_of(k) <= bin; });
    };
    // min_p as a cut
    if (min_p > 0.f && !first) {
        const double floor_w = (double)min_p * S_ONE;
        min_cut = (u64)first_key([&](uint32_t k) { return real_weight(k) >= floor_w; }) << 32;
    }
    // warp w owns indices [w * per, (w + 1) * per) of the slice
    const int per = ((n + SW - 1) / SW + 127) & ~127, i0 = min(n, warp * per), i1 = min(n, i0 + per);
    // The weight of this warp's tokens that `take` wants (weights are computed
    // only where some lane has one).
    auto range_sum = [&](auto take) {
        double sum = 0.0;
        for (int i = i0 + lane * 4; i - lane * 4 < i1; i += 128) {
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (i < i1) x = *reinterpret_cast<const uint4 *>(keys + i);
            const uint32_t k[4] = {x.x, x.y, x.z, x.w};
            bool yes[4];
#pragma unroll
            for (int e = 0; e < 4; e++) yes[e] = take(k[e], i + e);
            if (!__any_sync(0xffffffffu, yes[0] | yes[1] | yes[2] | yes[3])) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double w = whole(real_weight(k[e]));
                sum += yes[e] ? w : 0.0;
            }
        }
        return warp_total((u64)sum);
    };
    u64 range = 0;           // of the tokens that stay, if known
    bool have_range = false;
    // ---- 3. First CTA: cuts the list exactly, sorts what stays by index and
    // draws.
    auto draw_listed = [&] {
        int n2;
        const int m = sort_list(&n2);
        // (logit descending, index ascending): thread t has entries t * PT ..
        u64 w[PT], mine = 0, total;
#pragma unroll
        for (int e = 0; e < PT; e++) {
            const int i = t * PT + e;
            w[e] = i < m && (!k_on || i < top_k) ? weight((uint32_t)(sm.list[i] >> 32)) : 0;
            mine += w[e];
        }
        u64 before = block_scan<u64>(mine, sm.scan, lane, warp, &total);
        const u64 whole = k_on ? total : sm.weight;
        const u64 goal = p_on ? (u64)ceil((double)top_p * (double)whole) : ~0ull;
        // kept ones as index << 46 | weight (at most 2^45), in ascending order
        // of the index: complemented for the descending sort
#pragma unroll
        for (int e = 0; e < PT; e++) {
            const int i = t * PT + e;
            u64 x = 0;
            if (w[e] && before < goal) {
                const u64 c = sm.list[i];
                if (c >= min_cut) x = ~((u64)(0xffffffffu - (uint32_t)c) << 46 | w[e]);
            }
            before += w[e];
            if (i < n2) sm.val[i] = x;
        }
        sort_down(sm.val, n2, reinterpret_cast<unsigned *>(sm.list), reinterpret_cast<unsigned *>(sm.scan), t);
        mine = 0;
#pragma unroll
        for (int e = 0; e < PT; e++) {
            const u64 x = t * PT + e < n2 ? sm.val[t * PT + e] : 0;
            w[e] = x ? ~x & ((1ull << 46) - 1) : 0;
            mine += w[e];
        }
        before = block_scan<u64>(mine, sm.scan, lane, warp, &total);
        const double x = (double)u * (double)total;
        u64 want = x < (double)total ? (u64)x : total;
        if (want >= total) want = total - 1;
#pragma unroll
        for (int e = 0; e < PT; e++) {
            if (w[e] && before <= want && want < before + w[e]) a.tokens[out_at] = (int)(~sm.val[t * PT + e] >> 46);
            before += w[e];
        }
    };
    unsigned cn = 0, all_n;  // first CTA: tokens and (in f32) weight ahead of this thread's bins
    float cw = 0.f, all_w;
    // Adds up the cluster's histograms with their places: each CTA its share of the
    // bins, into the first CTA's.
    auto merge = [&] {
        if (C == 1) return;
        const int share = BINS / C;
        for (int i = t; i < 2 * share; i += ST) {
            const int bin = rank * share + (i < share ? i : i - share);
            unsigned sum = 0;
#pragma unroll
            for (int r = 0; r < SC; r++)
                if (r < C) {
                    const SampleSmem *o = cl.map_shared_rank(&sm, r);
                    sum += i < share ? o->hist.n[bin] : o->hist.f[bin];
                }
            if (i < share) lead->hist.n[bin] = sum;
            else lead->hist.f[bin] = sum;
        }
        cl.sync();
    };
    // First CTA: counts (and weights, of merged histograms) ahead of each thread's
    // bins. A bin's weight is taken as its tokens times the weight at their mean
    // place: off by less than 2^-14, since weights within a bin differ by at most a
    // factor of 1.016.
    float bin_w[PT];
    auto collect = [&](bool weights) {
        static_assert(PT == 4, "a thread's bins are one vector");
        uint4 bn = reinterpret_cast<const uint4 *>(sm.hist.n)[t], bf = reinterpret_cast<const uint4 *>(sm.hist.f)[t];
        if (!weights) {
#pragma unroll
            for (int r = 1; r < SC; r++)
                if (r < C) {
                    const uint4 y = reinterpret_cast<const uint4 *>(cl.map_shared_rank(&sm, r)->hist.n)[t];
                    bn.x += y.x, bn.y += y.y, bn.z += y.z, bn.w += y.w;
                }
            reinterpret_cast<uint4 *>(sm.hist.n)[t] = bn;
        }
        cn = block_scan<unsigned>(bn.x + bn.y + bn.z + bn.w, reinterpret_cast<unsigned *>(sm.scan), lane, warp, &all_n);
        if (weights) {
            const unsigned cnt[PT] = {bn.x, bn.y, bn.z, bn.w}, pl[PT] = {bf.x, bf.y, bf.z, bf.w};
            const float c = s > 0.f ? -1.4426950408889634f / T / s * 4096.f : 0.f;  // log2 of the weight per bin
            float w = 0.f;
#pragma unroll
            for (int e = 0; e < PT; e++) {
                const float at = (float)(t * PT + e) + (cnt[e] ? (float)pl[e] / ((float)cnt[e] * 4096.f) : 0.f);
                bin_w[e] = cnt[e] ? (float)cnt[e] * exp2f(at * c) : 0.f;
                w += bin_w[e];
            }
            cw = block_scan<float>(w, sm.scan_f, lane, warp, &all_w);
        }
    };
    // First CTA: sm.hi = the bin in which the count reaches top_k (or the last one).
    auto k_bin = [&] {
        int lim = BINS - 1;
        unsigned x = cn;
#pragma unroll
        for (int e = 0; e < PT; e++) {
            x += sm.hist.n[t * PT + e];
            if (lim == BINS - 1 && x >= (unsigned)top_k) lim = t * PT + e;
        }
        if (t == 0) sm.hi = BINS - 1;
        __syncthreads();
        lim = __reduce_min_sync(0xffffffffu, lim);
        if (lane == 0) atomicMin(&sm.hi, lim);
        __syncthreads();
    };
    // First CTA: `way` and its bins to every CTA.
    auto tell = [&](int way, int lo, int hi) {
        if (t < C) cl.map_shared_rank(&sm, t)->plan = Plan{way, lo, hi};
    };
    // A top_k that is small beside the number of threads: the top_k-th largest of
    // the threads' largest keys is a lower bound of the top_k-th key, and few
    // tokens lie above it.
    if (k_on && !first && top_k <= C * ST / 4) {
        // (four bins taken together: a quarter of the reads from the other CTAs, and a
        // list that is hardly longer)
        static_assert(PT == 4, "a thread has four bins");
        if (bk >= least) atomicAdd(&sm.hist.n[bin_of(bk) / PT], 1u);
        cl.sync();
        if (rank == 0) {
            unsigned here = sm.hist.n[t];
#pragma unroll
            for (int r = 1; r < SC; r++)
                if (r < C) here += cl.map_shared_rank(&sm, r)->hist.n[t];
            if (t == 0) sm.hi = BINS - 1;
            unsigned all;
            const unsigned before = block_scan<unsigned>(here, reinterpret_cast<unsigned *>(sm.scan), lane, warp, &all);
            if (before < (unsigned)top_k && (unsigned)top_k <= before + here) sm.hi = t * PT + PT - 1;
            __syncthreads();
            tell(ALL_LISTED, 0, sm.hi);
        }
        cl.sync();
        const uint32_t from = bin_start(sm.plan.hi);
        gather(from, [&](uint32_t k, int) { return k >= from; });
        cl.sync();
        const bool fits = lead->count <= LIST;
        cl.barrier_arrive();
        if (fits && rank == 0) draw_listed();
        cl.barrier_wait();  // (nobody leaves while the first CTA's count may be read)
        if (fits) return;
        // many equal logits: start again with all tokens counted
        for (int i = t; i < BINS; i += ST) sm.hist.n[i] = 0, sm.hist.f[i] = 0;
        if (t == 0) sm.count = 0;
        cl.sync();
    }
    if ((k_on || p_on) && !first) {
        const bool need_w = p_on && (!k_on || top_k > LIST);
        double mine = 0.0;
        each4([&](int, const uint32_t *k) {
            int b[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                b[e] = place_of(k[e]);
                b[e] = weightless(k[e]) ? -1 : b[e];
            }
            if (need_w && !k_on)
#pragma unroll
                for (int e = 0; e < 4; e++) mine += whole(real_weight(k[e]));
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (b[e] < 0) continue;
                atomicAdd(&sm.hist.n[b[e] >> 12], 1u);
                if (need_w) atomicAdd(&sm.hist.f[b[e] >> 12], (unsigned)b[e] & 4095u);
            }
        });
        if (p_on && !k_on) {
            const u64 sum = warp_total((u64)mine);
            if (lane == 0) atomicAdd(&lead->weight, sum);
        }
        cl.sync();
        if (need_w) merge();
        // First CTA: bins lo .. hi that hold the end of the top_p for a given
        // total weight. The f32 weights are taken to be off by up to 2^-11 (what was
        // found is checked).
        auto p_bins = [&](u64 whole) {
            const float goal = (float)((double)top_p * (double)whole / S_ONE);
            float w = cw;
            int lo = BINS - 1, hi = BINS - 1;
#pragma unroll
            for (int e = 0; e < PT; e++) {
                w += bin_w[e];
                if (lo == BINS - 1 && w * (1.f + 1.f / 2048) >= goal) lo = t * PT + e;
                if (hi == BINS - 1 && w * (1.f - 1.f / 2048) >= goal) hi = t * PT + e;
            }
            if (t == 0) sm.lo = sm.hi = BINS - 1;
            __syncthreads();
            lo = __reduce_min_sync(0xffffffffu, lo);
            hi = __reduce_min_sync(0xffffffffu, hi);
            if (lane == 0) {
                atomicMin(&sm.lo, lo);
                atomicMin(&sm.hi, hi);
            }
            __syncthreads();
        };
        if (rank == 0) {
            collect(need_w);
            if (k_on) k_bin();
            else p_bins(sm.weight);
            // tokens down to hi, and in lo .. hi
            const int hi = sm.hi, lo = k_on ? hi : sm.lo;
            auto upto = [&](int bin, unsigned *dst) {
                if (bin / PT != t) return;
                unsigned x = cn;
                for (int b = t * PT; b <= bin; b++) x += sm.hist.n[b];
                *dst = x;
            };
            unsigned *to = reinterpret_cast<unsigned *>(sm.scan);
            __syncthreads();
            if (t == 0) to[0] = 0;
            __syncthreads();
            upto(hi, to + 1);
            if (lo > 0) upto(lo - 1, to);
            __syncthreads();
            const unsigned ahead = to[0], down = to[1];
            tell(down <= LIST ? ALL_LISTED : down - ahead > LIST ? RADIX : k_on ? K_BIN : P_BINS, lo, hi);
            if (t == 0) sm.pick.above = ahead;
        }
        cl.sync();
        way = sm.plan.way;
        if (way == K_BIN) {  // the end of the top_k
            const uint32_t from = bin_start(sm.plan.hi), to = sm.plan.hi ? bin_start(sm.plan.hi - 1) : kmax + 1;
            gather(from, [&](uint32_t k, int) { return (k >= from) & (k < to); });
            cl.sync();
            if (rank == 0) {
                int n2;
                const int m = sort_list(&n2);
                // (an empty bin: the tokens that weigh are fewer than top_k, so all of them stay)
                const u64 last = m ? sm.list[min(m, top_k - (int)sm.pick.above) - 1] : (u64)least << 32;
                if (t < C) cl.map_shared_rank(&sm, t)->cut = last;
                __syncthreads();
                if (t == 0) sm.count = 0;
            }
            cl.sync();
            cut = sm.cut;
            if (top_k <= LIST) {
                way = ALL_LISTED;
            } else if (p_on) {  // the weight of the top_k, then the bins of the top_p
                u64 w = 0;
                each4([&](int i, const uint32_t *k) {
#pragma unroll
                    for (int e = 0; e < 4; e++) w += token_of(k[e], i + e) >= cut ? weight(k[e]) : 0;
                });
                w = warp_total(w);
                if (lane == 0) atomicAdd(&lead->weight, w);
                cl.sync();
                if (rank == 0) {
                    p_bins(sm.weight);
                    tell(P_BINS, sm.lo, sm.hi);
                }
                cl.sync();
                way = P_BINS;
            }
        }
        if (way == P_BINS) {  // the end of the top_p
            // keys from .. to - 1 are in bins lo .. hi (the ends found side by side)
            const uint32_t end = warp & 1 ? (sm.plan.lo ? bin_start(sm.plan.lo - 1) : kmax + 1) : bin_start(sm.plan.hi);
            if (lane == 0 && warp < 2) sm.ends[warp] = end;
            open_list();
            __syncthreads();
            const uint32_t from = sm.ends[0], to = sm.ends[1];
            // one pass: the weight of the tokens above those bins, and the bins' tokens
            const u64 w = range_sum([&](uint32_t k, int i) {
                const bool in = (k >= from) & (token_of(k, i) >= cut);
                if (in & (k < to)) push(k, i);
                return in & (k >= to);
            });
            if (lane == 0) atomicAdd(&lead->total[0], w);
            send_list();
            cl.sync();
            if (rank == 0) {
                int n2;
                const bool fits = sm.count <= LIST;
                const int m = sort_list(&n2);
                u64 x[PT], mine = 0, all;
#pragma unroll
                for (int e = 0; e < PT; e++) {
                    const int i = t * PT + e;
                    x[e] = i < m ? weight((uint32_t)(sm.list[i] >> 32)) : 0;
                    mine += x[e];
                }
                const u64 goal = (u64)ceil((double)top_p * (double)sm.weight), ahead = sm.total[0];
                u64 before = ahead + block_scan<u64>(mine, sm.scan, lane, warp, &all);
                const bool good = fits && m > 0 && ahead < goal && ahead + all >= goal;
#pragma unroll
                for (int e = 0; e < PT; e++) {
                    if (x[e] && before < goal && before + x[e] >= goal && good) sm.cut = sm.list[t * PT + e];
                    before += x[e];
                }
                __syncthreads();
                const u64 last = sm.cut;
                __syncthreads();
                if (t < C) {
                    cl.map_shared_rank(&sm, t)->cut = last;
                    cl.map_shared_rank(&sm, t)->plan = Plan{good ? P_BINS : RADIX, 0, 0};
                }
            }
            cl.sync();
            way = sm.plan.way;
            if (way == P_BINS) {
                cut = sm.cut;
                if (!min_cut) {  // the sum goes on with the last bins' tokens
                    range = w + range_sum([&](uint32_t k, int i) { return (k < to) & (token_of(k, i) >= cut); });
                    have_range = true;
                }
            }
        }
        if (way == ALL_LISTED) {
            const uint32_t from = cut ? least : bin_start(sm.plan.hi);
            gather(from, [&](uint32_t k, int i) { return (k >= from) & (token_of(k, i) >= cut); });
            cl.sync();
            if (rank == 0) draw_listed();
            return;
        }
    }

    auto cluster_sum = [&](u64 v, u64 *ahead) {  // over the cluster; *ahead: over the CTAs before this one
        cl.sync();
        if (t < C) cl.map_shared_rank(&sm, t)->total[rank] = v;
        cl.sync();
        u64 sum = 0, pre = 0;
        for (int r = 0; r < C; r++) {
            if (r < rank) pre += sm.total[r];
            sum += sm.total[r];
        }
        if (ahead) *ahead = pre;
        return sum;
    };
    if ((k_on || p_on) && way == RADIX) {
        // ---- radix selection: most significant digit first, the digit in which
        // the running count (or weight) from the top reaches the target; of the
        // tokens from `cut` up. Ends in the last token that stays.
        auto select = [&](bool by_weight, u64 target) {
            uint32_t prefix = 0;
            u64 above = 0;
            unsigned n_tie = 0;
            for (int sh = 24; sh >= 0; sh -= 8) {
                for (int i = t; i < 256; i += ST) sm.dig.n[i] = sm.dig.lead_n[i] = 0, sm.dig.w[i] = sm.dig.lead_w[i] = 0;
                cl.sync();
                for (int i = t; i < n; i += ST) {
                    const uint32_t k = keys[i];
                    if (!k || token(i) < cut || (sh < 24 && (k >> (sh + 8)) != (prefix >> (sh + 8)))) continue;
                    atomicAdd(&sm.dig.n[(k >> sh) & 255], 1u);
                    if (by_weight && !weightless(k)) atomicAdd(&sm.dig.w[(k >> sh) & 255], weight(k));
                }
                __syncthreads();
                for (int i = t; i < 256; i += ST)
                    if (sm.dig.n[i]) {
                        atomicAdd(&lead->dig.lead_n[i], sm.dig.n[i]);
                        if (by_weight) atomicAdd(&lead->dig.lead_w[i], sm.dig.w[i]);
                    }
                cl.sync();
                if (rank == 0) {  // thread t: digit 255 - t
                    u64 x = 0, all;
                    unsigned y = 0;
                    if (t < 256) y = sm.dig.lead_n[255 - t], x = by_weight ? sm.dig.lead_w[255 - t] : (u64)y;
                    const u64 before = above + block_scan<u64>(x, sm.scan, lane, warp, &all);
                    if (t == 0) sm.lo = 0, sm.hi = 256;
                    __syncthreads();
                    if (y) atomicMax(&sm.lo, t);                                 // the lowest digit holds the rest
                    if (y && before + x >= target) atomicMin(&sm.hi, t);
                    __syncthreads();
                    if (t == min(sm.lo, sm.hi))
                        for (int r = 0; r < C; r++) cl.map_shared_rank(&sm, r)->pick = Pick{255 - t, y, before};
                }
                cl.sync();
                prefix |= (uint32_t)sm.pick.digit << sh;
                above = sm.pick.above;
                n_tie = sm.pick.ties;
            }
            const u64 each = by_weight ? (weightless(prefix) ? 0 : weight(prefix)) : 1, left = target > above ? target - above : 0;
            u64 m = each ? (left + each - 1) / each : n_tie;  // of its ties, by index
            m = m < 1 ? 1 : m > n_tie ? n_tie : m;
            // the m-th of them
            unsigned mine = 0, here;
            for (int i = i0 + lane; i < i1; i += 32) mine += keys[i] == prefix && token(i) >= cut;
            mine = __reduce_add_sync(0xffffffffu, mine);
            unsigned pre = block_scan<unsigned>(lane == 0 ? mine : 0u, reinterpret_cast<unsigned *>(sm.scan), lane, warp, &here);
            u64 ahead;
            cluster_sum(here, &ahead);
            unsigned run = __shfl_sync(0xffffffffu, pre, 0) + (unsigned)ahead;
            if (run < m && m <= run + mine)
                for (int i = i0; i < i1; i += 32) {
                    const bool tie = i + lane < i1 && keys[i + lane] == prefix && token(i + lane) >= cut;
                    const unsigned same = __ballot_sync(0xffffffffu, tie);
                    if (tie && run + __popc(same & ((1u << lane) - 1)) + 1 == m)
                        for (int r = 0; r < C; r++) cl.map_shared_rank(&sm, r)->cut = token(i + lane);
                    run += __popc(same);
                }
            cl.sync();
            cut = sm.cut;
        };
        if (k_on && !cut) select(false, (u64)top_k);
        if (p_on) {
            u64 w = 0;
            for (int i = t; i < n; i += ST)
                if (!weightless(keys[i]) && token(i) >= cut) w += weight(keys[i]);
            u64 all;
            block_scan<u64>(w, sm.scan, lane, warp, &all);
            all = cluster_sum(all, nullptr);
            select(true, (u64)ceil((double)top_p * (double)all));
        }
    }
    // ---- draw in index order from the tokens where they are
    cut = cut > min_cut ? cut : min_cut;
    auto kept_weight = [&](uint32_t k, int i) -> u64 {
        if (first) {  // any weight above zero counts 1
            if (!k || token_of(k, i) < cut) return 0;
            const double w = k == kmax ? 1.0 : top_inf ? 0.0 : exp(((double)key_logit(k) - lmax) / (double)T);
            return (u64)(w > 0.0 && !(w < (double)min_p));
        }
        return token_of(k, i) < cut ? 0 : weight(k);
    };
    auto four = [&](int i, u64 *w) {  // of tokens i .. i + 3 of this warp's range; returns their sum
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (i < i1) x = *reinterpret_cast<const uint4 *>(keys + i);
        w[0] = kept_weight(x.x, i);
        w[1] = kept_weight(x.y, i + 1);
        w[2] = kept_weight(x.z, i + 2);
        w[3] = kept_weight(x.w, i + 3);
        return (w[0] + w[1]) + (w[2] + w[3]);
    };
    u64 sum = range, w[4];
    if (first) {
        for (int i = i0; i < i1; i += 128) sum += four(i + lane * 4, w);
        sum = warp_total(sum);
    } else if (!have_range) {
        sum = range_sum([&](uint32_t k, int i) { return (k >= least) & (token_of(k, i) >= cut); });
    }
    u64 all, run;
    u64 pre = block_scan<u64>(lane == 0 ? sum : 0, sm.scan, lane, warp, &all);
    const u64 total = cluster_sum(all, &run);
    run += __shfl_sync(0xffffffffu, pre, 0);
    const double x = (double)u * (double)total;
    u64 want = x > 0.0 ? (x < (double)total ? (u64)x : total) : 0;
    if (want >= total) want = total - 1;
    if (run <= want && want < run + sum) {  // this warp holds the token
        for (int i = i0; i < i1; i += 128) {
            const u64 mine = four(i + lane * 4, w), upto = run + warp_scan(mine, lane);
            const unsigned hit = __ballot_sync(0xffffffffu, upto > want);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    u64 at = upto - mine;
                    int e = 0;
                    while (e < 3 && (at += w[e]) <= want) e++;
                    a.tokens[out_at] = base + i + lane * 4 + e;
                }
                break;
            }
            run = __shfl_sync(0xffffffffu, upto, 31);
        }
    }
}

template <int TYPE>
cudaError_t launch(const QdbSampleArgs &a, cudaStream_t st) {
    // at least 16K tokens per CTA. 50257 tokens, top_k 50 / top_p alone: one row 11.5 /
    // 28.4 us, 64 rows 16.4 / 45; with 8K 10.4 / 23.8 and 29.7 / 63 (the clusters no
    // longer all run at once), with 32K 13.5 / 43 and 15.2 / 48
    int C = 1;
    while (C < SC && a.vocab > C * 16384) C <<= 1;
    const int slice = ((a.vocab + C - 1) / C + 31) & ~31;
    const size_t smem = sizeof(SampleSmem) + (size_t)slice * 4;
    // the limit belongs to the kernel, not to this call: always the largest, so that
    // calls of other sizes from other threads find it high enough
    constexpr size_t most = sizeof(SampleSmem) + (size_t)SLICE * 4;
    static_assert(SLICE >= 16384 && SLICE % 32 == 0 && most <= 227 * 1024, "a CTA's tokens fit its shared memory");
    cudaError_t e = cudaFuncSetAttribute(sample_kernel<TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e != cudaSuccess) return e;
    int dev = 0, sms = 0;
    if ((e = cudaGetDevice(&dev)) != cudaSuccess ||
        (e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess)
        return e;
    const bool ordered = (a.temperature || a.top_k || a.top_p || a.min_p) && (long long)a.rows * C > 2 * sms;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.rows * C);
    cfg.blockDim = dim3(ST);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = QDB_PDL;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, sample_kernel<TYPE>, a, slice, ordered);
}

}  // namespace

cudaError_t qdb_launch_sample(const QdbSampleArgs &a, int type, cudaStream_t st) {
    if (type == QDB_TYPE_F32) return launch<QDB_TYPE_F32>(a, st);
    if (type == QDB_TYPE_F16) return launch<QDB_TYPE_F16>(a, st);
    return launch<QDB_TYPE_BF16>(a, st);
}

extern "C" int qdb_sample(const void *logits, int type, long long row_stride, int rows, int vocab,
                          const qdb_sampling *s, int *tokens_out, void *stream) {
    qdb_set_error("");
    char m[256];
    auto refuse = [&](const char *fmt, long long x) {
        snprintf(m, sizeof(m), fmt, x);
        return qdb_set_error(m);
    };
    if (type != QDB_TYPE_F32 && type != QDB_TYPE_F16 && type != QDB_TYPE_BF16)
        return refuse("qdb_sample: logit type %lld", type);
    if (rows < 0 || rows > (1 << 20)) return refuse("qdb_sample: %lld rows", rows);
    if (vocab <= 0 || vocab > QDB_SAMPLE_MAX_VOCAB) return refuse("qdb_sample: vocabulary of %lld (1..262144)", vocab);
    if (row_stride && row_stride < vocab) return refuse("qdb_sample: row stride %lld", row_stride);
    if (rows == 0) return 0;
    if (!logits || !s || !s->uniform || !tokens_out) return qdb_set_error("qdb_sample: null argument");
    const int es = type == QDB_TYPE_F32 ? 4 : 2;
    const QdbNamedPtr ps[] = {{logits, "logits", es}, {s->temperature, "temperature"}, {s->top_k, "top_k"},
                              {s->top_p, "top_p"}, {s->min_p, "min_p"}, {s->uniform, "uniform"},
                              {tokens_out, "tokens_out"}};
    if (qdb_check_device_ptrs("qdb_sample", ps, 7)) return -1;
    const QdbSampleArgs a{logits, row_stride ? row_stride : vocab, rows, vocab, s->temperature, s->top_k, s->top_p,
                          s->min_p, s->uniform, 0, tokens_out, nullptr};
    const cudaError_t e = qdb_launch_sample(a, type, (cudaStream_t)stream);
    if (e != cudaSuccess) {
        snprintf(m, sizeof(m), "qdb_sample: %s", cudaGetErrorString(e));
        return qdb_set_error(m);
    }
    return 0;
}
