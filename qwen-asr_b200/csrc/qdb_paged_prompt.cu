// qdb_paged_prompt.cu - causal attention of packed prompts over a paged KV
// cache on the tensor cores (tcgen05).
//
// A CTA owns one key head and one block of a sequence's new rows: two tiles of
// 128 MMA rows (row r = position r / G, head r % G of the group), which share
// every K and V tile of 128 keys. It is bound by the tensor cores and by the
// exponentials (128 x 128 of them per tile take as long on the special
// function units as the tile's two products take on the tensor cores), so
// neither may wait for the other: the two row tiles run half a step apart, and
// a row tile's next scores are there before its softmax of this tile ends.
//   warps 0-3, 4-7  softmax of tile 0, 1: thread = row = TMEM lane
//   warp 8          issues S = Q K^T      (two warps, since waiting for the next
//   warp 9          issues O += P V        operands takes half as long as a product)
//   warps 10, 11    copy Q and the pages of K (ring of 2 tiles), of V (ring of 3):
//                   two, since a page of 16 positions takes as many instructions as
//                   one of 128
// TMEM: S (128 columns, read into registers at once, so one serves both row
// tiles in turn), P0, P1 (64 columns of packed 16-bit pairs, the A operand of
// the second product), O0, O1 (128 columns each). No product waits for another
// one's TMEM columns but through the softmax.
// V is used as loaded (keys along K, dims along N).
//   m, l            running maximum and sum per row in f32; O is rescaled only
//                   when the maximum grows by more than 2^8, so numerator and
//                   denominator always share one m
//   P               rounded to the cache's type (the type of V's own rounding)
// Keys behind a row's position count nothing, whatever the cache holds there:
// scores are replaced by -inf, and in the tiles that some row sees only in part
// the values behind the last visible key and non-finite values are cleared
// before the product (the latter are added back to the rows that do see them).
#include <math.h>

#include "qdb_kernels.h"
#include "qdb_paged.cuh"

namespace {

constexpr int PT_THREADS = 384;
constexpr int PT_N = 128;                 // keys per tile
constexpr int PT_KS = 2, PT_VS = 3;       // K and V tiles in shared memory
constexpr uint32_t PT_HALF = 128 * 128;   // bytes of [128 rows][64 dims]
constexpr uint32_t PT_TILE = 2 * PT_HALF;
constexpr int PT_PART = 3;                // tiles that some row sees only in part: 256 positions touch 3
constexpr float PT_RAISE = 8.0f;          // log2 growth of the maximum that is let pass

struct PromptSmem {
    unsigned char q[2][PT_TILE];
    unsigned char k[PT_KS][PT_TILE], v[PT_VS][PT_TILE];
    unsigned long long q_full, k_full[PT_KS], k_empty[PT_KS], v_full[PT_VS], v_empty[PT_VS], s_full[2], s_read, p_full[2], o_done[2], drain[2];
    unsigned long long v_part[PT_PART], v_clean[PT_PART];  // V of the tiles seen in part: landed, cleared
    uint32_t tmem;
    int abort;
    int nonfinite;
};

// ---- tcgen05
// Shared-memory operand, 128-byte swizzle, 8-row groups 1024 bytes apart
// (start >> 4, leading offset >> 4 at bit 16, stride offset >> 4 at bit 32,
// version 1 at 46, layout 2 at 61). K-major ignores the leading offset; in the
// MN-major form (V) it is the distance of the next 64 dims.
__device__ __forceinline__ uint64_t op_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | (uint64_t)((lead >> 4) & 0x3fffu) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// f32 accumulator (bit 4), A and B f16 or bf16 (bits 7, 10), B MN-major (bit
// 16), N / 8 at 17, M / 16 at 24.
template <typename T>
__device__ constexpr uint32_t op_kind(bool b_mn) {
    return (1u << 4) | (T::code == QDB_TYPE_BF16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) |
           (128u / 8) << 17 | (128u / 16) << 24;
}
// Eight products of K = 16: D (+)= A B over 128 dims (or keys). a, b: operand
// descriptors (or A's TMEM column) of the first; all offsets are constants, so
// the issuing warp has little to compute between two products.
template <bool ACC>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t kind) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a),
        "l"(b), "r"(kind), "n"(ACC ? 1 : 0)
        : "memory");
}
template <bool ACC>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t kind) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
        "r"(a), "l"(b), "r"(kind), "n"(ACC ? 1 : 0)
        : "memory");
}
__device__ __forceinline__ bool elect() {
    uint32_t r;
    asm volatile("{ .reg .pred q; elect.sync _|q, 0xffffffff; selp.u32 %0, 1, 0, q; }" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

#define R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define I8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
// 32 columns of this thread's lane, waited for.
__device__ __forceinline__ void tm_ld32(uint32_t a, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
        : R8(v, 0), R8(v, 8), R8(v, 16), R8(v, 24)
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void tm_ld64(uint32_t a, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,"
        "%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
        : R8(v, 0), R8(v, 8), R8(v, 16), R8(v, 24), R8(v, 32), R8(v, 40), R8(v, 48), R8(v, 56)
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t a, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
        I8(v, 0), I8(v, 8), I8(v, 16), I8(v, 24)
        : "memory");
}
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// Two f32 at a time.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// Bounded wait that also ends when another role has given up.
__device__ __forceinline__ bool wait_on(PromptSmem &sm, uint32_t bar, unsigned parity, int *err) {
    if (bar_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (!bar_try(bar, parity)) {
        if (*reinterpret_cast<volatile int *>(&sm.abort)) return false;
        if (clock64() - t0 > QDB_SPIN_LIMIT_CYCLES) {
            set_error(err, QDB_ERR_BARRIER_TIMEOUT);
            *reinterpret_cast<volatile int *>(&sm.abort) = 1;
            return false;
        }
    }
    return true;
}

// The CTA's block of rows.
struct Block {
    int b, row0, n, pos0;  // sequence, its first row here, rows (positions) here, position of the first
    bool any;
};

// Blocks of bq rows: sequence b's begin at number q_starts[b] / bq + b, which
// leaves room for every sequence's last, partly filled block (the numbers
// behind it are empty). The blocks with the longest histories come first.
__device__ Block find_block(const QdbPagedAttnArgs &a, int bq, int i, int lane) {
    Block k{0, 0, 0, 0, false};
    const int n = a.bt.n_seqs, step = a.bt.step ? *a.bt.step : 0;
    int lo = 0;
    if (a.bt.q_starts) {  // the last sequence that begins at or before i, 32 candidates at a time
        for (int size = n; size > 1;) {
            const int d = (size + 31) / 32, mid = lo + lane * d;
            const bool in = lane * d < size && max(a.bt.q_starts[mid], 0) / bq + mid <= i;
            const int last = 31 - __clz(__ballot_sync(0xffffffffu, in) | 1u);
            size = min(d, size - last * d);
            lo += last * d;
        }
    } else {
        lo = i;
        if (lo >= n) return k;
    }
    const int len = paged_len(a.bt, lo, a.kv.page_shift, step);
    int first, last;
    paged_rows(a.bt, lo, first, last);
    const int j = a.bt.q_starts ? i - (first / bq + lo) : 0, blocks = (last - first + bq - 1) / bq;
    if (j < 0 || j >= blocks) return k;
    const int at = (blocks - 1 - j) * bq;
    k.b = lo;
    k.row0 = first + at;
    k.n = min(bq, last - first - at);
    k.pos0 = len - (last - first) + at;
    k.any = true;
    return k;
}

template <typename T>
__global__ void __launch_bounds__(PT_THREADS, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv, const __grid_constant__ QdbPagedAttnArgs a) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    PromptSmem &sm = *reinterpret_cast<PromptSmem *>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int Hkv = a.kv.kv_heads, G = a.heads / Hkv, QP = 128 / G;  // positions per row tile
    const int g = blockIdx.x % Hkv;
    int *err = a.bt.err;
    if (t == 0) {
        bar_init(smem_u32(&sm.q_full), 1);
        for (int s = 0; s < PT_KS; s++) {
            bar_init(smem_u32(&sm.k_full[s]), 1);
            bar_init(smem_u32(&sm.k_empty[s]), 1);
        }
        for (int s = 0; s < PT_VS; s++) {
            bar_init(smem_u32(&sm.v_full[s]), 1);
            bar_init(smem_u32(&sm.v_empty[s]), 1);
        }
        for (int x = 0; x < 2; x++) {
            bar_init(smem_u32(&sm.s_full[x]), 1);
            bar_init(smem_u32(&sm.p_full[x]), 128);
            bar_init(smem_u32(&sm.o_done[x]), 1);
        }
        bar_init(smem_u32(&sm.s_read), 128);
        for (int k = 0; k < PT_PART; k++) {
            bar_init(smem_u32(&sm.v_part[k]), 1);
            bar_init(smem_u32(&sm.v_clean[k]), 256);
        }
        bar_init(smem_u32(&sm.drain[0]), 1);
        bar_init(smem_u32(&sm.drain[1]), 1);
        sm.abort = 0;
        sm.nonfinite = 0;
        fence_bar_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mq) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
    }
    __syncthreads();
    pdl_enter();
    const Block blk = find_block(a, 2 * QP, blockIdx.x / Hkv, lane);
    if (!blk.any) return;
    // tile x: rows of positions [x * QP, x * QP + nx); keys it needs, in tiles
    const int n0 = min(blk.n, QP), n1 = blk.n - n0;
    const int end0 = max(blk.pos0 + n0, 0), end1 = n1 > 0 ? max(blk.pos0 + blk.n, 0) : 0;
    const int t0 = (end0 + PT_N - 1) / PT_N, t1 = (end1 + PT_N - 1) / PT_N, tiles = max(t0, t1), end = max(end0, end1);
    // tiles from here on are not seen whole by every row
    const int special = max(blk.pos0 + 1, 0) / PT_N;
    // (after the wait for the kernel before: a CTA of it that shares the SM must
    // never find the columns taken by one that waits for it)
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // (the copying warps do not wait for the columns: barrier 1 is for the others)
    tc_before();
    if (warp < 10) asm volatile("bar.sync 1, 320;" ::: "memory");
    tc_after();
    const uint32_t tm = sm.tmem;
    // registers as launched (168 x 384) shared out anew: 208 x 256 + 88 x 128
    if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < 8) {
        // ------------------------------------------------ softmax of row tile x
        const int x = warp >> 2, r = t & 127, nx = x ? n1 : n0, nt = x ? t1 : t0;
        const int i = r / G;  // position in the tile
        const int pos = blk.pos0 + x * QP + i;
        const bool real = i < nx && i < QP;
        const int whole = max(blk.pos0 + x * QP + 1, 0) / PT_N;  // tiles before this one need no mask
        const uint32_t ts = tm + ((uint32_t)(32 * (warp & 3)) << 16), tp = ts + 128 + x * 64, to = ts + 256 + x * 128;
        const float c = a.scale * 1.4426950408889634f;
        constexpr float shift = T::code == QDB_TYPE_F16 ? 6.f : 0.f;  // keeps f16 weights down to 2^-30 of the largest
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        // Half x of V's dims of a tile that some row sees only in part.
        auto clear_v = [&](int j) {
            if (!wait_on(sm, smem_u32(&sm.v_part[j - special]), 0, err)) return false;
            uint4 *v = reinterpret_cast<uint4 *>(sm.v[j % PT_VS] + x * PT_HALF);
            bool odd = false, wrote = false;
#pragma unroll
            for (int e = r; e < (int)(PT_HALF / 16); e += 128) {
                // 16 bytes of key e / 8 (the swizzle moves them within their row only)
                uint4 w = v[e];
                if (j * PT_N + (e >> 3) >= end) {
                    v[e] = make_uint4(0u, 0u, 0u, 0u);
                    wrote = true;
                } else if (T::any_nonfinite(w.x) | T::any_nonfinite(w.y) | T::any_nonfinite(w.z) | T::any_nonfinite(w.w)) {
                    v[e] = make_uint4(T::clear_nonfinite(w.x), T::clear_nonfinite(w.y), T::clear_nonfinite(w.z),
                                      T::clear_nonfinite(w.w));
                    odd = wrote = true;
                }
            }
            if (odd) {
                *reinterpret_cast<volatile int *>(&sm.nonfinite) = 1;
                __threadfence_block();
            }
            if (wrote) fence_async();
            bar_arrive(smem_u32(&sm.v_clean[j - special]));
            return true;
        };
        // The output product of tile j - 1 has read P and written O.
        auto done_before = [&](int j) {
            const bool done = __all_sync(0xffffffffu, wait_on(sm, smem_u32(&sm.o_done[x]), (j - 1) & 1, err));
            tc_after();
            return done;
        };
        for (int j = 0; j < tiles; j++) {
            if (j >= special) {  // (before the scores are there: the output product waits for both halves)
                ok = __all_sync(0xffffffffu, clear_v(j));
                if (!ok) break;
            }
            if (j >= nt) continue;  // (the other row tile's last one)
            ok = wait_on(sm, smem_u32(&sm.s_full[x]), j & 1, err);
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            tc_after();
            float s[128];
            tm_ld64(ts, reinterpret_cast<uint32_t *>(s));
            tm_ld64(ts + 64, reinterpret_cast<uint32_t *>(s + 64));
            tc_before();
            bar_arrive(smem_u32(&sm.s_read));
            if (j >= whole) {
                const int seen = pos - j * PT_N;  // keys 0 .. seen of this tile
#pragma unroll
                for (int e = 0; e < 128; e++) s[e] = e <= seen ? s[e] : -INFINITY;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 128; e += 8)
#pragma unroll
                for (int k = 0; k < 4; k++) mx[k] = max3(mx[k], s[e + 2 * k], s[e + 2 * k + 1]);
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            const bool up = top > m && (m == -INFINITY || (top - m) * c > PT_RAISE);
            if (__any_sync(0xffffffffu, up)) {
                const float f = up ? (m == -INFINITY ? 0.f : ex2((m - top) * c)) : 1.f;
                if (up) m = top;
                l *= f;
                if (j > 0) {
                    ok = done_before(j);
                    if (!ok) break;
#pragma unroll 1
                    for (int k = 0; k < 128; k += 32) {
                        uint32_t o[32];
                        tm_ld32(to + k, o);
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tm_st32(to + k, o);
                    }
                }
            }
            const float mc = m == -INFINITY ? 0.f : m * c - shift;
            const uint64_t c2 = pair(c, c), mc2 = pair(-mc, -mc);
            uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
            for (int k = 0; k < 128; k += 64) {
                uint32_t p[32];
#pragma unroll
                for (int e = 0; e < 64; e += 2) {
                    const uint64_t x2 = fma2(pair(s[k + e], s[k + e + 1]), c2, mc2);
                    float p0, p1;
                    unpair(x2, p0, p1);
                    p0 = ex2(p0);
                    p1 = ex2(p1);
                    sum[(e / 2) & 1] = add2(sum[(e / 2) & 1], pair(p0, p1));
                    p[e / 2] = T::plain(p0, p1);
                }
                if (k == 0 && j > 0) {
                    ok = done_before(j);
                    if (!ok) break;
                }
                tm_st32(tp + k / 2, p);
            }
            {
                float s0, s1;
                unpair(add2(sum[0], sum[1]), s0, s1);
                l += s0 + s1;
            }
            if (!ok) break;
            tm_st_wait();
            tc_before();
            bar_arrive(smem_u32(&sm.p_full[x]));
        }
        if (ok && nt > 0) ok = wait_on(sm, smem_u32(&sm.o_done[x]), (nt - 1) & 1, err);
        if (ok && nt == 0 && tiles > 0) ok = wait_on(sm, smem_u32(&sm.q_full), 0, err);  // (its rows are reused below)
        ok = __all_sync(0xffffffffu, ok);
        if (ok && nx > 0) {
            tc_after();
            const float inv = l > 0.f ? 1.0f / l : (isnan(l) ? l : 0.f);
            const bool fix = sm.nonfinite != 0;  // (written before the products that o_done waited for)
            // rows go through the row tile's Q (all its scores are done): a row's 16
            // pieces of 16 bytes, exchanged by the row's number so that neither side
            // has bank conflicts, leave in whole rows
            unsigned char *stage = sm.q[x] + (warp & 3) * 32 * 256;
            const unsigned inv_g = (65536u + G - 1) / G;  // r / G = r * inv_g >> 16 for r < 128
            const float scale_o = l > 0.f || isnan(l) ? inv : 0.f;
            for (int part = 0; part < (a.lo ? 2 : 1); part++) {  // (hi, then lo of a bf16 pair)
                auto word = [&](uint32_t x, uint32_t y) {
                    const float u = __uint_as_float(x), v = __uint_as_float(y);
                    return a.lo ? QdbBf16::plain(pair_part(u, part), pair_part(v, part)) : T::plain(u, v);
                };
#pragma unroll 1
                for (int k = 0; k < 128; k += 64) {
                    uint32_t o[64];
                    if (nt > 0) {
                        tm_ld64(to + k, o);
                    } else {
#pragma unroll
                        for (int e = 0; e < 64; e++) o[e] = 0u;
                    }
#pragma unroll
                    for (int e = 0; e < 64; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * scale_o);
                    if (fix && real)  // non-finite values were left out of the products: add those this row sees
                        for (int key = special * PT_N; key <= pos; key++) {
                            const int page = paged_page(a.kv, a.bt, blk.b, key >> a.kv.page_shift);
                            if (page < 0) continue;
                            const uint16_t *v = a.kv.v + page * a.kv.page_stride + g * a.kv.head_stride +
                                                (key & ((1 << a.kv.page_shift) - 1)) * a.kv.pos_stride + k;
#pragma unroll
                            for (int e = 0; e < 64; e++) {
                                const float y = T::lo(v[e]);
                                if (!isfinite(y)) o[e] = __float_as_uint(__uint_as_float(o[e]) + y);
                            }
                        }
#pragma unroll
                    for (int e = 0; e < 64; e += 8)
                        *reinterpret_cast<uint4 *>(stage + lane * 256 + ((((k + e) / 8) ^ (lane & 7)) << 4)) =
                            make_uint4(word(o[e], o[e + 1]), word(o[e + 2], o[e + 3]), word(o[e + 4], o[e + 5]),
                                       word(o[e + 6], o[e + 7]));
                }
                __syncwarp();
#pragma unroll 4
                for (int e = 0; e < 32; e += 2) {  // two rows at a time
                    const int q = e + (lane >> 4), rr = 32 * (warp & 3) + q, ii = (int)((unsigned)rr * inv_g >> 16);
                    if (ii >= nx || ii >= QP) continue;
                    uint16_t *dst = (part ? a.lo : a.out) + (size_t)(blk.row0 + x * QP + ii) * a.out_stride + ((size_t)g * G + rr - ii * G) * QDB_HD;
                    *reinterpret_cast<uint4 *>(dst + (lane & 15) * 8) =
                        *reinterpret_cast<const uint4 *>(stage + q * 256 + (((lane & 15) ^ (q & 7)) << 4));
                }
                __syncwarp();  // (the rows have been read)
            }
        }
    } else if (warp < 10) {
        // ------------------------------------------------ products: warp 8 the scores, warp 9 the outputs
        // (the whole warp runs this together, with values that are the same in all
        // lanes, so that they stay in uniform registers, where the products' operands
        // have to be; one lane issues)
        const int T0 = __shfl_sync(0xffffffffu, t0, 0), T1 = __shfl_sync(0xffffffffu, t1, 0), TT = max(T0, T1);
        const int part = __shfl_sync(0xffffffffu, special, 0);
        const uint32_t tmu = __shfl_sync(0xffffffffu, tm, 0);
        if (TT > 0) {
            bool ok = true;
            const bool scores_warp = warp == 8, leader = elect();  // (a commit covers its own thread's products)
            const uint64_t q_desc = op_desc(smem_u32(sm.q[0]), 16), k_desc = op_desc(smem_u32(sm.k[0]), 16),
                           v_desc = op_desc(smem_u32(sm.v[0]), PT_HALF);
            constexpr uint64_t tile = PT_TILE >> 4;
            auto scores = [&](int x, int j) {  // S = Q_x K_j^T
                const uint64_t q = q_desc + x * tile, k = k_desc + (uint32_t)(j % PT_KS) * tile;
                if (leader) {
                    mma_ss<false>(tmu, q, k, op_kind<T>(false));
#pragma unroll
                    for (int e = 1; e < 8; e++) {
                        const uint64_t at = ((e >> 2) * PT_HALF + (e & 3) * 32) >> 4;
                        mma_ss<true>(tmu, q + at, k + at, op_kind<T>(false));
                    }
                    commit(smem_u32(&sm.s_full[x]));
                }
                __syncwarp();
            };
            auto output = [&](int x, int j) {  // O_x += P_x V_j
                const uint64_t v = v_desc + (uint32_t)(j % PT_VS) * tile;
                const uint32_t d = tmu + 256 + x * 128, p = tmu + 128 + x * 64;
                if (leader) {
                    if (j > 0) mma_ts<true>(d, p, v, op_kind<T>(true));
                    else mma_ts<false>(d, p, v, op_kind<T>(true));
#pragma unroll
                    for (int e = 1; e < 8; e++) mma_ts<true>(d, p + e * 8, v + e * (2048 >> 4), op_kind<T>(true));
                    commit(smem_u32(&sm.o_done[x]));
                }
                __syncwarp();
            };
            auto wait = [&](uint32_t bar, unsigned parity) { return __all_sync(0xffffffffu, wait_on(sm, bar, parity, err)); };
            // the tiles in the order 0(0) 1(0) 0(1) 1(1) ...; those a row tile does
            // not need are passed over
            int n = 0;
            if (scores_warp) ok = wait(smem_u32(&sm.q_full), 0);
            for (int j = 0; j < TT && ok; j++) {
                if (scores_warp) {
                    ok = wait(smem_u32(&sm.k_full[j % PT_KS]), (j / PT_KS) & 1);
                } else if (j < part) {
                    ok = wait(smem_u32(&sm.v_full[j % PT_VS]), (j / PT_VS) & 1);
                } else {  // V_j, which some row sees only in part, landed and was cleared
                    ok = wait(smem_u32(&sm.v_clean[j - part]), 0);
                }
                for (int x = 0; x < 2 && ok; x++) {
                    if (j >= (x ? T1 : T0)) continue;
                    if (scores_warp) {  // (the scores before have been read)
                        if (n) ok = wait(smem_u32(&sm.s_read), (n - 1) & 1);
                    } else {
                        ok = wait(smem_u32(&sm.p_full[x]), j & 1);
                    }
                    if (!ok) break;
                    tc_after();
                    if (scores_warp) scores(x, j);
                    else output(x, j);
                    n++;
                }
                if (ok && leader) commit(smem_u32(scores_warp ? &sm.k_empty[j % PT_KS] : &sm.v_empty[j % PT_VS]));
                __syncwarp();
            }
            if (!ok && n) {  // given up: the products in flight end before the CTA does
                if (leader) commit(smem_u32(&sm.drain[warp - 8]));
                __syncwarp();
                bar_wait(smem_u32(&sm.drain[warp - 8]), 0, err);
            }
        }
        __syncwarp();
    } else if (tiles > 0) {
        // ------------------------------------------------ copies: warp 10 Q and K, warp 11 V
        const bool is_v = warp == 11;
        const int rows = min(1 << a.kv.page_shift, PT_N), pieces = PT_N / rows, S = is_v ? PT_VS : PT_KS;
        unsigned long long *full = is_v ? sm.v_full : sm.k_full, *empty = is_v ? sm.v_empty : sm.k_empty;
        unsigned char *ring = is_v ? sm.v[0] : sm.k[0];
        const CUtensorMap *map = is_v ? &mv : &mk;
        auto look_up = [&](int j) {  // this lane's page of tile j
            const int key = j * PT_N + lane * rows;
            if (lane >= pieces || key >= end) return -1;
            const int p = paged_page(a.kv, a.bt, blk.b, key >> a.kv.page_shift);
            return p < 0 ? a.kv.n_pages : p;  // outside the pool: recorded, reads as zeros
        };
        int page = look_up(0);
        if (!is_v && lane == 0) {
            bar_expect(smem_u32(&sm.q_full), (n1 > 0 ? 4u : 2u) * 128u * G * QP);
            for (int x = 0; x < (n1 > 0 ? 2 : 1); x++)
                for (int half = 0; half < 2; half++)
                    asm volatile(
                        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
                        "{%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(sm.q[x]) + half * PT_HALF),
                        "l"(&mq), "r"(0), "r"(half), "r"(g * G), "r"(blk.row0 + x * QP), "r"(smem_u32(&sm.q_full))
                        : "memory");
        }
        __syncwarp();
        bool ok = true;
        int sent = 0;
        for (int j = 0; j < tiles; j++) {
            const int st = j % S, n = min(pieces, (end - j * PT_N + rows - 1) / rows);
            const int after = j + 1 < tiles ? look_up(j + 1) : -1;  // (not waited for before it is needed)
            if (j >= S) ok = __all_sync(0xffffffffu, wait_on(sm, smem_u32(&empty[st]), ((j / S) & 1) ^ 1, err));
            if (!ok) break;
            // (V of a tile seen in part lands on a barrier of its own, which the
            // clearing warps wait for, and which has one phase only)
            const uint32_t bar = smem_u32(is_v && j >= special ? &sm.v_part[j - special] : &full[st]);
            if (lane == 0) bar_expect(bar, (uint32_t)n * rows * 256u);
            __syncwarp();
            if (page >= 0) {
                const uint32_t dst = smem_u32(ring) + st * PT_TILE + lane * rows * 128;
                const int slot = (j * PT_N + lane * rows) & ((1 << a.kv.page_shift) - 1);
#pragma unroll
                for (int half = 0; half < 2; half++) load_half_page(dst + half * PT_HALF, map, slot, half, g, page, bar);
            }
            __syncwarp();
            page = after;
            sent = j + 1;
        }
        if (!ok && lane == 0) {  // given up: the copies in flight land first
            if (!is_v) bar_wait(smem_u32(&sm.q_full), 0, err);
            for (int j = max(0, sent - S); j < sent; j++)
                bar_wait(smem_u32(is_v && j >= special ? &sm.v_part[j - special] : &full[j % S]),
                         is_v && j >= special ? 0u : (unsigned)(j / S) & 1u, err);
        }
        __syncwarp();
    }
    tc_before();
    __syncthreads();
    if (warp == 8) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512) : "memory");
    }
}

// q as (64 dims, dim half, head, row): a copy brings G heads of QP rows.
int query_map(CUtensorMap *map, const QdbPagedAttnArgs &a, int type, int G) {
    return qdb_encode_map4(map, a.q, type, (uint64_t)a.heads, (uint64_t)a.bt.rows, (uint64_t)a.q_stride, (uint32_t)G,
                           (uint32_t)(128 / G));
}

template <typename T>
cudaError_t launch(const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, const QdbPagedAttnArgs &a,
                   cudaStream_t st) {
    const size_t smem = sizeof(PromptSmem) + 1024;
    cudaError_t e = cudaFuncSetAttribute(prompt_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const int G = a.heads / a.kv.kv_heads, bq = 2 * (128 / G);
    const long long blocks = a.bt.q_starts ? (long long)a.bt.rows / bq + a.bt.n_seqs : a.bt.n_seqs;
    if (blocks * a.kv.kv_heads > 2147483647ll) return cudaErrorInvalidConfiguration;
    return pdl_launch(prompt_kernel<T>, dim3((unsigned)(blocks * a.kv.kv_heads)), dim3(PT_THREADS), smem, st, mq, mk, mv, a);
}

}  // namespace

cudaError_t qdb_launch_paged_prompt(const QdbPagedAttnArgs &a, int type, cudaStream_t st) {
    CUtensorMap mq, mk, mv;
    const int page = 1 << a.kv.page_shift, rows = page < PT_N ? page : PT_N;
    if (query_map(&mq, a, type, a.heads / a.kv.kv_heads) || qdb_paged_map(&mk, a.kv.k, a.kv, type, rows, 1) ||
        qdb_paged_map(&mv, a.kv.v, a.kv, type, rows, 1))
        return cudaErrorInvalidValue;
    return type == QDB_TYPE_F16 ? launch<QdbHalf>(mq, mk, mv, a, st) : launch<QdbBf16>(mq, mk, mv, a, st);
}
