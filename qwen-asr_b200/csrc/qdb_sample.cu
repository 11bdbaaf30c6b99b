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
// Sums are 64-bit integers: w is rounded to a multiple of 2^-45 (a token below
// that is never drawn), so a sum over up to 2^18 tokens is exact, independent
// of the order of the atomics, and a border between two tokens is off by at
// most 2^-46 of the largest weight per token summed. (uniform = 0 asks for the
// first kept token of any weight above zero: there every such token counts 1.)
#include <math.h>
#include <stdio.h>

#include "qdb_kernels.h"
#include "qdb_paged.cuh"

namespace {

typedef unsigned long long u64;
constexpr int SM_THREADS = 1024, SM_WARPS = SM_THREADS / 32;
constexpr double SM_ONE = 35184372088832.0;  // 2^45

template <int TYPE>
__device__ __forceinline__ float load_logit(const void *p, size_t i) {
    float v;
    if (TYPE == QDB_TYPE_F32) v = reinterpret_cast<const float *>(p)[i];
    else if (TYPE == QDB_TYPE_F16) v = QdbHalf::lo(reinterpret_cast<const uint16_t *>(p)[i]);
    else v = QdbBf16::lo(reinterpret_cast<const uint16_t *>(p)[i]);
    return v;
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

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One CTA per row; the logits are read again from L2 in every pass.
template <int TYPE>
__global__ void __launch_bounds__(SM_THREADS) sample_kernel(const QdbSampleArgs a) {
    pdl_enter();
    __shared__ u64 hw[256];
    __shared__ unsigned hc[256];
    __shared__ u64 part[SM_WARPS + 1];
    __shared__ u64 s_best, s_total, s_before;
    __shared__ unsigned s_cbefore;
    __shared__ int s_digit, s_tok;
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.vocab;
    const size_t shift_row = (a.step ? (size_t)*a.step * a.rows : 0) + row;
    const char *base = (const char *)a.logits + (size_t)row * a.row_stride * (TYPE == QDB_TYPE_F32 ? 4 : 2);
    int *dst = a.tokens + shift_row;
    auto key_of = [&](int i) -> uint32_t {
        if (a.mask_eos && (i == QDB_ENDOFTEXT || i == QDB_IM_END)) return 0u;
        return logit_key(load_logit<TYPE>(base, i));
    };
    if (t == 0) s_best = 0;
    __syncthreads();
    u64 best = 0;
    for (int i = t; i < V; i += SM_THREADS) {
        const uint32_t k = key_of(i);
        const u64 c = ((u64)k << 32) | (0xffffffffu - (uint32_t)i);
        if (k && c > best) best = c;
    }
    atomicMax(&s_best, best);
    __syncthreads();
    best = s_best;
    const float T = a.temperature ? a.temperature[row] : 1.f;
    int top_k = a.top_k ? a.top_k[row] : 0;
    float top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f;
    const float u = a.uniform[shift_row];
    if (best == 0 || !(T > 0.f) || top_p <= 0.f || min_p > 1.f || top_k == 1) {
        if (t == 0) *dst = best ? (int)(0xffffffffu - (uint32_t)best) : -1;
        return;
    }
    const uint32_t kmax = (uint32_t)(best >> 32);
    const double lmax = (double)key_logit(kmax), dT = (double)T;
    auto weight = [&](uint32_t k) -> u64 {  // exp((l - max) / T) in units of 2^-45
        if (k == kmax) return (u64)SM_ONE;
        if (k == 0) return 0;
        return __double2ull_rn(exp(((double)key_logit(k) - lmax) / dT) * SM_ONE);
    };
    const bool first = !(u > 0.f);
    auto above_floor = [&](uint32_t k) { return k == kmax || !(exp(((double)key_logit(k) - lmax) / dT) < (double)min_p); };

    // (cut, ties): keys above cut stay, and the first `ties` (by index) equal to it
    uint32_t cut = 0;
    unsigned ties = 0xffffffffu;
    // Most significant digit first: the digit in which the running count (or
    // weight) from the top reaches the target. Elements: keys > lim, or the
    // first lim_ties equal to it (lim = 0: all).
    auto select = [&](bool by_weight, u64 target, uint32_t lim, unsigned lim_ties, uint32_t &o_cut, unsigned &o_ties) {
        uint32_t prefix = 0;
        u64 before = 0;       // count or weight above the current prefix range
        unsigned cbefore = 0; // count above it
        for (int sh = 24; sh >= 0; sh -= 8) {
            for (int i = t; i < 256; i += SM_THREADS) hw[i] = 0, hc[i] = 0;
            __syncthreads();
            for (int i = t; i < V; i += SM_THREADS) {
                const uint32_t k = key_of(i);
                if (!k || k < lim || (sh < 24 && (k >> (sh + 8)) != (prefix >> (sh + 8)))) continue;
                atomicAdd(&hc[(k >> sh) & 255], 1u);
                if (by_weight) atomicAdd(&hw[(k >> sh) & 255], weight(k));
            }
            __syncthreads();
            if (t == 0) {
                u64 s = before;
                unsigned c = cbefore;
                int d = 255, pick = -1;
                for (; d >= 0; d--) {
                    if (!hc[d]) continue;
                    u64 add = by_weight ? hw[d] : (u64)hc[d];
                    pick = d;
                    if (s + add >= target) break;
                    bool more = false;
                    for (int e = d - 1; e >= 0; e--) more |= hc[e] != 0;
                    if (!more) break;  // fewer than asked for: the last digit holds the rest
                    s += add;
                    c += hc[d];
                }
                s_digit = pick;
                s_before = s;
                s_cbefore = c;
            }
            __syncthreads();
            prefix |= (uint32_t)s_digit << sh;
            before = s_before;
            cbefore = s_cbefore;
            __syncthreads();
        }
        // prefix is the key at which the target is reached; hc of its digit = its ties
        const unsigned n_tie = hc[prefix & 255];
        const u64 each = by_weight ? weight(prefix) : 1;
        const u64 left = target > before ? target - before : 0;
        u64 m = each ? (left + each - 1) / each : n_tie;
        if (m < 1) m = 1;
        if (m > n_tie) m = n_tie;
        if (prefix == lim && m > lim_ties) m = lim_ties;
        o_cut = prefix;
        o_ties = (unsigned)m;
        __syncthreads();
    };
    if (top_k > 0 && top_k < V) select(false, (u64)top_k, 0, 0xffffffffu, cut, ties);
    if (top_p < 1.f) {  // (NaN: off)
        if (t == 0) s_total = 0;
        __syncthreads();
        u64 w = 0;
        for (int i = t; i < V; i += SM_THREADS) {
            const uint32_t k = key_of(i);
            if (k > cut) w += weight(k);
        }
        w = warp_sum64(w);
        if (lane == 0) atomicAdd(&s_total, w);
        __syncthreads();
        u64 total = s_total + (cut ? (u64)ties * weight(cut) : 0);
        __syncthreads();
        const u64 target = (u64)ceil((double)top_p * (double)total);
        uint32_t c2;
        unsigned t2;
        select(true, target, cut, ties, c2, t2);
        cut = c2;
        ties = t2;
    }
    // ---- draw in index order: warp w owns indices [w * per, (w + 1) * per)
    const int per = ((V + SM_WARPS - 1) / SM_WARPS + 31) & ~31, i0 = warp * per, i1 = min(V, i0 + per);
    unsigned n = 0;
    for (int i = i0 + lane; i < i1; i += 32) n += key_of(i) == cut && cut;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) part[warp] = n;
    __syncthreads();
    unsigned tie0 = 0;
    for (int w = 0; w < warp; w++) tie0 += (unsigned)part[w];
    __syncthreads();
    auto kept_weight = [&](int i, unsigned &rank) -> u64 {  // weight of index i if kept; rank: ties before this step
        const uint32_t k = i < i1 ? key_of(i) : 0u;
        const unsigned same = __ballot_sync(0xffffffffu, k == cut && k);
        const bool tie = k == cut && rank + __popc(same & ((1u << lane) - 1)) < ties;
        rank += __popc(same);
        if (!k || !(k > cut || tie) || !above_floor(k)) return 0;
        return first ? (u64)(k == kmax || exp(((double)key_logit(k) - lmax) / dT) > 0.0) : weight(k);
    };
    u64 sum = 0;
    unsigned rank = tie0;
    for (int i = i0; i < i1; i += 32) sum += kept_weight(i + lane, rank);
    sum = warp_sum64(sum);
    if (lane == 0) part[warp] = sum;
    if (t == 0) s_tok = -1;
    __syncthreads();
    u64 total = 0, run = 0;
    for (int w = 0; w < SM_WARPS; w++) {
        if (w < warp) run += part[w];
        total += part[w];
    }
    const double x = (double)u * (double)total;
    u64 target = x > 0.0 ? (x < (double)total ? (u64)x : total) : 0;
    if (target >= total) target = total - 1;
    if (run <= target && target < run + sum) {  // this warp holds the token
        rank = tie0;
        for (int i = i0; i < i1; i += 32) {
            u64 w = kept_weight(i + lane, rank);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 y = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= o) w += y;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, run + w > target);
            if (hit) {
                if (lane == 0) *dst = i + __ffs(hit) - 1;
                break;
            }
            run += __shfl_sync(0xffffffffu, w, 31);
        }
    }
}

}  // namespace

cudaError_t qdb_launch_sample(const QdbSampleArgs &a, int type, cudaStream_t st) {
    const dim3 grid(a.rows), block(SM_THREADS);
    if (type == QDB_TYPE_F32) return pdl_launch(sample_kernel<QDB_TYPE_F32>, grid, block, 0, st, a);
    if (type == QDB_TYPE_F16) return pdl_launch(sample_kernel<QDB_TYPE_F16>, grid, block, 0, st, a);
    return pdl_launch(sample_kernel<QDB_TYPE_BF16>, grid, block, 0, st, a);
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
