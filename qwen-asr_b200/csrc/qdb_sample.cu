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
// More tokens than that (a flat distribution) are cut by a radix selection on
// the integers, digit by digit over the cluster, and drawn where they are. Both
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
    unsigned above_n, ties;
    u64 above;    // count or weight above the digit
};

struct SampleSmem {
    union {
        struct {
            unsigned n[BINS];
            float w[BINS];
        } hist;
        u64 list[LIST];
    };
    union {
        u64 val[LIST];
        struct {
            u64 w[256], lead_w[256];
            unsigned n[256], lead_n[256];
        } dig;
    };
    u64 scan[SW + 1];
    float scan_f[SW + 1];
    u64 best[SC], total[SC];
    uint32_t low[SC];
    unsigned ties[SC];
    u64 weight;      // first CTA: sum of all weights
    unsigned count;  // first CTA: tokens in the list
    int limit;       // last bin that goes to the list, -1: too many
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
__global__ void __launch_bounds__(ST) sample_kernel(const QdbSampleArgs a, int slice) {
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
    const double lmax = (double)fmax, dT = (double)T, floor_w = (double)min_p;
    const bool k_on = top_k > 0 && top_k < V, p_on = top_p < 1.f, first = !(u > 0.f);
    auto real_weight = [&](uint32_t k) { return k == kmax ? 1.0 : exp(((double)key_logit(k) - lmax) / dT); };
    auto weight = [&](uint32_t k) -> u64 {  // in units of 2^-45
        return k ? __double2ull_rn(real_weight(k) * S_ONE) : 0;
    };
    const float reach = S_REACH * T;  // logits further below the maximum weigh nothing
    auto weightless = [&](uint32_t k) { return !k || (k != kmax && !(fmax - key_logit(k) <= reach)); };

    // ---- 2. histogram: how far down the kept tokens can go
    if ((k_on || p_on) && !first) {
        const float span = fminf(reach, fmax - key_logit(low)), s = span > 0.f ? (float)BINS / span : 0.f;
        auto bin_of = [&](uint32_t k) { return k == kmax ? 0 : min(BINS - 1, (int)((fmax - key_logit(k)) * s)); };
        u64 sum = 0;
        const float c = -1.4426950408889634f / T;
        for (int i = t; i < n; i += ST) {
            const uint32_t k = keys[i];
            if (weightless(k)) continue;
            const int b = bin_of(k);
            atomicAdd(&sm.hist.n[b], 1u);
            if (!k_on) {
                atomicAdd(&sm.hist.w[b], k == kmax ? 1.f : exp2f((fmax - key_logit(k)) * c));
                sum += weight(k);
            }
        }
        if (!k_on) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) atomicAdd(&lead->weight, sum);
        }
        __syncthreads();
        if (rank)
            for (int i = t; i < BINS; i += ST)
                if (sm.hist.n[i]) {
                    atomicAdd(&lead->hist.n[i], sm.hist.n[i]);
                    if (!k_on) atomicAdd(&lead->hist.w[i], sm.hist.w[i]);
                }
        cl.sync();
        if (rank == 0) {
            constexpr int PT = BINS / ST;
            unsigned cn = 0, all_n;
            float cw = 0.f, all_w;
#pragma unroll
            for (int e = 0; e < PT; e++) cn += sm.hist.n[t * PT + e], cw += sm.hist.w[t * PT + e];
            if (t == 0) sm.limit = BINS - 1;
            cn = block_scan<unsigned>(cn, reinterpret_cast<unsigned *>(sm.scan), lane, warp, &all_n);
            cw = block_scan<float>(cw, sm.scan_f, lane, warp, &all_w);
            // (the f32 sums of up to 2048 bins of up to 2048 tokens are off by
            // less than 2^-11; bins with more tokens end in the other way anyhow)
            const float goal = (float)((double)top_p * (double)sm.weight / S_ONE) * (1.f + 1.f / 2048);
            int lim = BINS;
#pragma unroll
            for (int e = 0; e < PT; e++) {
                cn += sm.hist.n[t * PT + e];
                cw += sm.hist.w[t * PT + e];
                if (lim == BINS && (k_on ? cn >= (unsigned)top_k : cw >= goal)) lim = t * PT + e;
            }
            atomicMin(&sm.limit, lim);
            __syncthreads();
            const int limit = sm.limit;
            if (limit / PT == t) {  // the tokens down to it
                for (int e = PT - 1; t * PT + e > limit; e--) cn -= sm.hist.n[t * PT + e];
                sm.count = cn;
            }
            __syncthreads();
            if (t < C) cl.map_shared_rank(&sm, t)->limit = sm.count > LIST ? -1 : limit;
            __syncthreads();
            if (t == 0) sm.count = 0;
        }
        cl.sync();
        const int limit = sm.limit;
        if (limit >= 0) {
            // ---- 3. those tokens to the first CTA
            for (int i0 = warp * 32; i0 < n; i0 += ST) {
                const uint32_t k = i0 + lane < n ? keys[i0 + lane] : 0u;
                const bool take = !weightless(k) && bin_of(k) <= limit;
                const unsigned m = __ballot_sync(0xffffffffu, take);
                if (!m) continue;
                unsigned at = 0;
                if (lane == 0) at = atomicAdd(&lead->count, __popc(m));
                at = __shfl_sync(0xffffffffu, at, 0) + __popc(m & ((1u << lane) - 1));
                if (take && at < LIST) lead->list[at] = (u64)k << 32 | (0xffffffffu - (uint32_t)(base + i0 + lane));
            }
            cl.sync();
            if (rank) return;
            const int m = min((int)sm.count, LIST);
            int n2 = 32;
            while (n2 < m) n2 <<= 1;
            for (int i = m + t; i < n2; i += ST) sm.list[i] = 0;
            sort_down(sm.list, n2, t);
            constexpr int PT = LIST / ST;
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

    // ---- many tokens: (cut, ties): keys above cut stay, and the first `ties`
    // (by index) equal to it
    uint32_t cut = 0;
    unsigned ties = 0xffffffffu;
    if ((k_on || p_on)) {
        if (rank == 0)
            for (int i = t; i < 256; i += ST) sm.dig.lead_n[i] = 0, sm.dig.lead_w[i] = 0;
        cl.sync();
    }
    // Most significant digit first: the digit in which the running count (or
    // weight) from the top reaches the target. Elements: keys >= lim.
    auto select = [&](bool by_weight, u64 target, uint32_t lim, unsigned lim_ties) {
        uint32_t prefix = 0;
        u64 above = 0;
        unsigned above_n = 0, n_tie = 0;
        for (int sh = 24; sh >= 0; sh -= 8) {
            for (int i = t; i < 256; i += ST) sm.dig.n[i] = 0, sm.dig.w[i] = 0;
            __syncthreads();
            for (int i = t; i < n; i += ST) {
                const uint32_t k = keys[i];
                if (!k || k < lim || (sh < 24 && (k >> (sh + 8)) != (prefix >> (sh + 8)))) continue;
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
            if (rank == 0) {
                if (t == 0) {
                    Pick p{0, above_n, 0, above};
                    int lowest = 0;
                    while (!sm.dig.lead_n[lowest]) lowest++;
                    for (int d = 255; d >= lowest; d--) {
                        if (!sm.dig.lead_n[d]) continue;
                        const u64 add = by_weight ? sm.dig.lead_w[d] : (u64)sm.dig.lead_n[d];
                        p.digit = d;
                        p.ties = sm.dig.lead_n[d];
                        if (p.above + add >= target || d == lowest) break;  // (the lowest holds the rest)
                        p.above += add;
                        p.above_n += p.ties;
                    }
                    for (int r = 0; r < C; r++) cl.map_shared_rank(&sm, r)->pick = p;
                }
                __syncthreads();
                for (int i = t; i < 256; i += ST) sm.dig.lead_n[i] = 0, sm.dig.lead_w[i] = 0;
            }
            cl.sync();
            prefix |= (uint32_t)sm.pick.digit << sh;
            above = sm.pick.above;
            above_n = sm.pick.above_n;
            n_tie = sm.pick.ties;
        }
        const u64 each = by_weight ? (weightless(prefix) ? 0 : weight(prefix)) : 1, left = target > above ? target - above : 0;
        u64 m = each ? (left + each - 1) / each : n_tie;
        if (m < 1) m = 1;
        if (m > n_tie) m = n_tie;
        if (prefix == lim && m > lim_ties) m = lim_ties;
        cut = prefix;
        ties = (unsigned)m;
    };
    auto cluster_sum = [&](u64 v, u64 *ahead) {  // over the cluster; *ahead: over the CTAs before this one
        cl.sync();
        if (t < C) cl.map_shared_rank(&sm, t)->total[rank] = v;
        cl.sync();
        u64 s = 0, pre = 0;
        for (int r = 0; r < C; r++) {
            if (r < rank) pre += sm.total[r];
            s += sm.total[r];
        }
        if (ahead) *ahead = pre;
        return s;
    };
    if (k_on) select(false, (u64)top_k, 0, 0xffffffffu);
    if (p_on) {
        u64 w = 0, all;
        for (int i = t; i < n; i += ST)
            if (keys[i] > cut && !weightless(keys[i])) w += weight(keys[i]);
        block_scan<u64>(w, sm.scan, lane, warp, &all);
        all = cluster_sum(all, nullptr);
        if (cut && !weightless(cut)) all += (u64)ties * weight(cut);
        select(true, (u64)ceil((double)top_p * (double)all), cut, ties);
    }
    // ---- draw in index order: warp w owns indices [w * per, (w + 1) * per) of the slice
    const int per = ((n + SW - 1) / SW + 31) & ~31, i0 = min(n, warp * per), i1 = min(n, i0 + per);
    unsigned tie0 = 0;
    if (cut) {
        unsigned mine = 0, all;
        for (int i = i0 + lane; i < i1; i += 32) mine += keys[i] == cut;
        mine = __reduce_add_sync(0xffffffffu, mine);
        const unsigned pre = block_scan<unsigned>(lane == 0 ? mine : 0u, reinterpret_cast<unsigned *>(sm.scan), lane, warp, &all);
        u64 ahead;
        cluster_sum(all, &ahead);
        tie0 = __shfl_sync(0xffffffffu, pre, 0) + (unsigned)ahead;
    }
    auto kept_weight = [&](int i, unsigned &before) -> u64 {  // of index i, if kept; before: ties ahead of this step
        const uint32_t k = i < i1 ? keys[i] : 0u;
        const unsigned same = __ballot_sync(0xffffffffu, k == cut && k);
        const bool tie = k == cut && before + __popc(same & ((1u << lane) - 1)) < ties;
        before += __popc(same);
        if (!k || !(k > cut || tie) || (!first && weightless(k))) return 0;
        const double w = real_weight(k);
        if (w < floor_w) return 0;
        return first ? (u64)(w > 0.0) : __double2ull_rn(w * S_ONE);
    };
    u64 sum = 0;
    unsigned seen = tie0;
    for (int i = i0; i < i1; i += 32) sum += kept_weight(i + lane, seen);
    u64 all;
    const u64 lane_pre = block_scan<u64>(sum, sm.scan, lane, warp, &all);
    u64 run;
    const u64 total = cluster_sum(all, &run);
    run += __shfl_sync(0xffffffffu, lane_pre, 0);
    sum = __shfl_sync(0xffffffffu, lane_pre + sum, 31) - __shfl_sync(0xffffffffu, lane_pre, 0);
    const double x = (double)u * (double)total;
    u64 want = x > 0.0 ? (x < (double)total ? (u64)x : total) : 0;
    if (want >= total) want = total - 1;
    if (run <= want && want < run + sum) {  // this warp holds the token
        seen = tie0;
        for (int i = i0; i < i1; i += 32) {
            const u64 w = warp_scan(kept_weight(i + lane, seen), lane);
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
