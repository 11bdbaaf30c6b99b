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
// than 31.5 T below the maximum is never drawn), so a sum over up to 2^18 tokens is exact, independent
// of the order of the atomics, and a border between two tokens is off by at
// most 2^-46 of the largest weight per token summed. (uniform = 0 asks for the
// first kept token of any weight above zero: there every such token counts 1.)
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
constexpr double S_ONE = 35184372088832.0;  // 2^45
constexpr float S_REACH = 31.5f;            // exp(-31.5) = 2^-45.4: what lies further down is left out

template <int TYPE>
__device__ __forceinline__ float widen(uint32_t bits) {
    return TYPE == QDB_TYPE_F32 ? __uint_as_float(bits) : TYPE == QDB_TYPE_F16 ? QdbHalf::lo(bits) : QdbBf16::lo(bits);
}

// Order-preserving integer of a logit: 0 for NaN and -inf (never drawn); -0
// and +0 are equal.
__device__ __forceinline__ uint32_t logit_key(float v) {
    if (isnan(v) || v == -INFINITY) return 0u;
    uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
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

struct SampleSmem {
    union {
        struct {
            unsigned n[BINS];
            float w[BINS];
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
    double exp2_64[64];  // 2^(45 + i / 64)
    u64 scan[SW + 1];
    float scan_f[SW + 1];
    u64 best[SC], total[SC];
    uint32_t low[SC];
    u64 weight;      // first CTA: a sum of weights
    unsigned count;  // first CTA: tokens in the list
    u64 cut;         // the last token that stays
    int lo, hi;      // first CTA
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

// n2 (a power of two) values in descending order.
__device__ void sort_down(u64 *x, int n2, int t) {
    for (int k = 2; k <= n2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int p = t; p < n2 / 2; p += ST) {
                const int i = 2 * p - (p & (j - 1)), q = i + j;
                const u64 a = x[i], b = x[q];
                if ((a < b) == ((i & k) == 0)) x[i] = b, x[q] = a;
            }
        }
    __syncthreads();
}

template <int TYPE>
__global__ void __launch_bounds__(ST, 2) sample_kernel(const QdbSampleArgs a, int slice) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    SampleSmem &sm = *reinterpret_cast<SampleSmem *>(smem_raw);
    uint32_t *keys = reinterpret_cast<uint32_t *>(smem_raw + sizeof(SampleSmem));
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank(), row = blockIdx.x / C;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.vocab;
    const int base = min(V, rank * slice), n = min(V, base + slice) - base;  // this CTA's tokens
    SampleSmem *lead = cl.map_shared_rank(&sm, 0);
    for (int i = t; i < BINS; i += ST) sm.hist.n[i] = 0, sm.hist.w[i] = 0.f;
    if (t == 0) sm.weight = 0, sm.count = 0;
    if (t < 64) sm.exp2_64[t] = exp2(45.0 + t / 64.0);
    cl.barrier_arrive();  // (waited for before the first access to another CTA's memory)
    pdl_enter();
    const size_t out_at = (a.step ? (size_t)*a.step * a.rows : 0) + row;
    const float T = a.temperature ? a.temperature[row] : 1.f;
    const int top_k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f;
    const float u = a.uniform[out_at];

    // ---- 1. the row into shared memory; its maximum
    u64 best = 0;
    uint32_t low = 0xffffffffu;
    {
        constexpr int ES = TYPE == QDB_TYPE_F32 ? 4 : 2, PER = 16 / ES;
        const char *src = (const char *)a.logits + ((size_t)row * a.row_stride + base) * ES;
        auto put = [&](int i, uint32_t bits) {
            uint32_t k = logit_key(widen<TYPE>(bits));
            if (a.mask_eos && (base + i == QDB_ENDOFTEXT || base + i == QDB_IM_END)) k = 0;
            keys[i] = k;
            const u64 c = (u64)k << 32 | (0xffffffffu - (uint32_t)(base + i));
            if (k) best = c > best ? c : best, low = min(low, k);
        };
        int from = 0;
        if (((uintptr_t)src & 15) == 0) {
            from = n / PER * PER;
#pragma unroll 4
            for (int i = t * PER; i < from; i += ST * PER) {
                const uint4 x = ldg_stream(src + (size_t)i * ES);
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < PER; e++) put(i + e, ES == 4 ? w[e] : (w[e / 2] >> (16 * (e & 1))) & 0xffffu);
            }
        }
#pragma unroll 4
        for (int i = from + t; i < n; i += ST)
            put(i, ES == 4 ? reinterpret_cast<const uint32_t *>(src)[i] : (uint32_t) reinterpret_cast<const uint16_t *>(src)[i]);
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
    if (best == 0 || !(T > 0.f) || top_p <= 0.f || min_p > 1.f || top_k == 1) {
        if (rank == 0 && t == 0) a.tokens[out_at] = best ? (int)(0xffffffffu - (uint32_t)best) : -1;
        return;
    }
    const uint32_t kmax = (uint32_t)(best >> 32);
    const float fmax = key_logit(kmax);
    const double lmax = (double)fmax, floor_w = (double)min_p * S_ONE;
    const bool k_on = top_k > 0 && top_k < V, p_on = top_p < 1.f, first = !(u > 0.f);
    // 2^45 exp((l - max) / T) by 2^(i / 64) from the table times a polynomial of
    // degree 4 in the rest (below 0.0055: the next term is 2^-44 of the weight)
    const double c64 = 64.0 * 1.4426950408889634074 / (double)T;
    auto real_weight = [&](uint32_t k) -> double {
        if (k == kmax) return S_ONE;
        const double d = (double)key_logit(k) - lmax, magic = 6755399441055744.0;  // 1.5 * 2^52
        const double y = fma(d, c64, magic);
        const int i = __double2loint(y);
        const double x = fma(d, c64, magic - y) * (0.69314718055994530942 / 64.0);
        double e = fma(x, 1.0 / 24, 1.0 / 6);
        e = fma(x, e, 0.5);
        e = fma(x, e, 1.0);
        e = fma(x, e, 1.0) * sm.exp2_64[i & 63];
        return __hiloint2double(__double2hiint(e) + ((i >> 6) << 20), __double2loint(e));
    };
    auto whole_weight = [&](double w) -> u64 {  // rounded to an integer (below 2^51)
        return (u64)__double_as_longlong(w + 4503599627370496.0) & ((1ull << 52) - 1);
    };
    auto weight = [&](uint32_t k) { return whole_weight(real_weight(k)); };
    const float reach = S_REACH * T;  // logits further below the maximum weigh nothing
    auto weightless = [&](uint32_t k) { return !k || (k != kmax && !(fmax - key_logit(k) <= reach)); };
    auto token = [&](int i) { return (u64)keys[i] << 32 | (0xffffffffu - (uint32_t)(base + i)); };
    auto warp_total = [&](u64 v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    // Tokens that `take` wants to the first CTA's list (in any order); a
    // barrier of the cluster has to follow.
    auto gather = [&](auto take) {
        for (int i0 = warp * 32; i0 < n; i0 += ST) {
            const bool yes = i0 + lane < n && take(i0 + lane);
            const unsigned m = __ballot_sync(0xffffffffu, yes);
            if (!m) continue;
            unsigned at = 0;
            if (lane == 0) at = atomicAdd(&lead->count, __popc(m));
            at = __shfl_sync(0xffffffffu, at, 0) + __popc(m & ((1u << lane) - 1));
            if (yes && at < LIST) lead->list[at] = token(i0 + lane);
        }
    };
    // First CTA: sorts the list; returns its length.
    auto sort_list = [&](int *n2) {
        const int m = min((int)sm.count, LIST);
        *n2 = 32;
        while (*n2 < m) *n2 <<= 1;
        for (int i = m + t; i < *n2; i += ST) sm.list[i] = 0;
        sort_down(sm.list, *n2, t);
        return m;
    };
    constexpr int PT = BINS / ST;  // bins, or list entries, of a thread
    u64 cut = 0;                   // tokens from here up stay
    int way = RADIX;

    // ---- 2. histogram: how far down the kept tokens can go
    const float span = fminf(reach, fmax - key_logit(low)), s = span > 0.f ? (float)BINS / span : 0.f;
    auto bin_of = [&](uint32_t k) { return k == kmax ? 0 : min(BINS - 1, (int)((fmax - key_logit(k)) * s)); };
    if ((k_on || p_on) && !first) {
        const bool need_w = p_on && (!k_on || top_k > LIST);
        u64 sum = 0;
        const float c = -1.4426950408889634f / T;
#pragma unroll 4
        for (int i = t; i < n; i += ST) {
            const uint32_t k = keys[i];
            if (weightless(k)) continue;
            const int b = bin_of(k);
            atomicAdd(&sm.hist.n[b], 1u);
            if (need_w) {
                atomicAdd(&sm.hist.w[b], k == kmax ? 1.f : exp2f((fmax - key_logit(k)) * c));
                if (!k_on) sum += weight(k);
            }
        }
        if (p_on && !k_on) {
            sum = warp_total(sum);
            if (lane == 0) atomicAdd(&lead->weight, sum);
        }
        __syncthreads();
        if (rank)
            for (int i = t; i < BINS; i += ST)
                if (sm.hist.n[i]) {
                    atomicAdd(&lead->hist.n[i], sm.hist.n[i]);
                    if (need_w) atomicAdd(&lead->hist.w[i], sm.hist.w[i]);
                }
        cl.sync();
        unsigned cn = 0, all_n;  // first CTA: tokens and (in f32) weight ahead of this thread's bins
        float cw = 0.f, all_w;
        // First CTA: bins lo .. hi that hold the end of the top_p for a given
        // total weight. The f32 sums are taken to be off by up to 2^-11 (more only
        // where bins hold thousands of tokens: what was found is checked).
        auto p_bins = [&](u64 whole) {
            const float goal = (float)((double)top_p * (double)whole / S_ONE);
            float w = cw;
            int lo = BINS - 1, hi = BINS - 1;
#pragma unroll
            for (int e = PT - 1; e >= 0; e--) {
                float x = w;
                for (int f = 0; f <= e; f++) x += sm.hist.w[t * PT + f];
                if (x * (1.f + 1.f / 2048) >= goal) lo = t * PT + e;
                if (x * (1.f - 1.f / 2048) >= goal) hi = t * PT + e;
            }
            if (t == 0) sm.lo = sm.hi = BINS - 1;
            __syncthreads();
            atomicMin(&sm.lo, lo);
            atomicMin(&sm.hi, hi);
            __syncthreads();
        };
        auto tell = [&](int way, int lo, int hi) {  // first CTA
            if (t < C) cl.map_shared_rank(&sm, t)->plan = Plan{way, lo, hi};
        };
        if (rank == 0) {
#pragma unroll
            for (int e = 0; e < PT; e++) cn += sm.hist.n[t * PT + e], cw += sm.hist.w[t * PT + e];
            cn = block_scan<unsigned>(cn, reinterpret_cast<unsigned *>(sm.scan), lane, warp, &all_n);
            cw = block_scan<float>(cw, sm.scan_f, lane, warp, &all_w);
            if (k_on) {  // the bin in which the count is reached
                int lim = BINS - 1;
                unsigned x = cn;
#pragma unroll
                for (int e = 0; e < PT; e++) {
                    x += sm.hist.n[t * PT + e];
                    if (lim == BINS - 1 && x >= (unsigned)top_k) lim = t * PT + e;
                }
                if (t == 0) sm.hi = BINS - 1;
                __syncthreads();
                atomicMin(&sm.hi, lim);
                __syncthreads();
            } else {
                p_bins(sm.weight);
            }
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
            const int bin = sm.plan.hi;
            gather([&](int i) { return !weightless(keys[i]) && bin_of(keys[i]) == bin; });
            cl.sync();
            if (rank == 0) {
                int n2;
                const int m = sort_list(&n2);
                const u64 last = sm.list[min(m, top_k - (int)sm.pick.above) - 1];
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
                for (int i = t; i < n; i += ST)
                    if (!weightless(keys[i]) && token(i) >= cut) w += weight(keys[i]);
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
            const int lo = sm.plan.lo, hi = sm.plan.hi;
            u64 w = 0;
#pragma unroll 2
            for (int i = t; i < n; i += ST) {
                const uint32_t k = keys[i];
                if (!weightless(k) && bin_of(k) < lo && token(i) >= cut) w += weight(k);
            }
            w = warp_total(w);
            if (t == 0 && rank == 0) sm.total[0] = 0;
            cl.sync();
            if (lane == 0) atomicAdd(&lead->total[0], w);
            gather([&](int i) {
                if (weightless(keys[i]) || token(i) < cut) return false;
                const int b = bin_of(keys[i]);
                return b >= lo && b <= hi;
            });
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
            if (way == P_BINS) cut = sm.cut;
        }
        if (way == ALL_LISTED) {
            // ---- 3. the tokens that may stay to the first CTA
            const int hi = sm.plan.hi;
            gather([&](int i) { return !weightless(keys[i]) && (cut ? token(i) >= cut : bin_of(keys[i]) <= hi); });
            cl.sync();
            if (rank) return;
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
                    if (!(real_weight((uint32_t)(c >> 32)) < floor_w)) x = ~((u64)(0xffffffffu - (uint32_t)c) << 46 | w[e]);
                }
                before += w[e];
                if (i < n2) sm.val[i] = x;
            }
            sort_down(sm.val, n2, t);
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
    // warp w owns indices [w * per, (w + 1) * per) of the slice
    const int per = ((n + SW - 1) / SW + 31) & ~31, i0 = min(n, warp * per), i1 = min(n, i0 + per);
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
    auto kept_weight = [&](int i) -> u64 {
        const uint32_t k = i < i1 ? keys[i] : 0u;
        if (!k || token(i) < cut) return 0;
        if (first) {  // any weight above zero counts 1
            const double w = k == kmax ? 1.0 : exp(((double)key_logit(k) - lmax) / (double)T);
            return (u64)(w > 0.0 && !(w < (double)min_p));
        }
        if (weightless(k)) return 0;
        const double w = real_weight(k);
        return w < floor_w ? 0 : whole_weight(w);
    };
    u64 sum = 0;
#pragma unroll 4
    for (int i = i0; i < i1; i += 32) sum += kept_weight(i + lane);
    sum = warp_total(sum);
    u64 all, run;
    u64 pre = block_scan<u64>(lane == 0 ? sum : 0, sm.scan, lane, warp, &all);
    const u64 total = cluster_sum(all, &run);
    run += __shfl_sync(0xffffffffu, pre, 0);
    const double x = (double)u * (double)total;
    u64 want = x > 0.0 ? (x < (double)total ? (u64)x : total) : 0;
    if (want >= total) want = total - 1;
    if (run <= want && want < run + sum) {  // this warp holds the token
        for (int i = i0; i < i1; i += 32) {
            const u64 w = warp_scan(kept_weight(i + lane), lane);
            const unsigned hit = __ballot_sync(0xffffffffu, run + w > want);
            if (hit) {
                if (lane == 0) a.tokens[out_at] = base + i + __ffs(hit) - 1;
                break;
            }
            run += __shfl_sync(0xffffffffu, w, 31);
        }
    }
}

template <int TYPE>
cudaError_t launch(const QdbSampleArgs &a, cudaStream_t st) {
    // at least 16K tokens per CTA: below that the cluster's barriers cost more
    // than the shorter passes save
    int C = 1;
    while (C < SC && a.vocab > C * 16384) C <<= 1;
    const int slice = ((a.vocab + C - 1) / C + 31) & ~31;
    const size_t smem = sizeof(SampleSmem) + (size_t)slice * 4;
    cudaError_t e = cudaFuncSetAttribute(sample_kernel<TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
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
    return cudaLaunchKernelEx(&cfg, sample_kernel<TYPE>, a, slice);
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
    if ((uintptr_t)logits % es) return qdb_set_error("qdb_sample: logits are not aligned to their type");
    const QdbNamedPtr ps[] = {{logits, "logits"}, {s->temperature, "temperature"}, {s->top_k, "top_k"},
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
