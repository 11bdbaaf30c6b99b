// qdb_paged_prompt.cu - causal attention of packed prompts over a paged KV
// cache on the tensor cores (tcgen05).
//
// A CTA owns one key head and one block of a sequence's new rows: two tiles of
// 128 MMA rows (row r = position r / G, head r % G of the group), which share
// every K and V tile of 128 keys. It is bound by the tensor cores and by the
// exponentials (128 x 128 of them per tile take as long on the special
// function units as the tile's two products take on the tensor cores), so the
// two row tiles alternate: while one's softmax runs, the other's products do.
//   warps 0-3, 4-7  softmax of tile 0, 1: thread = row = TMEM lane
//   warp 8          issues the products: S = Q K^T, then O += P V
//   warp 9          copies K and V pages (ring of 5 tiles) and Q
//   warps 10-11     clear what V holds behind the last visible key
// TMEM: S0, S1, O0, O1 (128 columns each); P replaces S as packed 16-bit pairs
// and is the A operand of the second product; V is used as loaded (keys along
// K, dims along N).
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
constexpr int PT_STAGES = 5;              // K and V tiles in flight
constexpr uint32_t PT_HALF = 128 * 128;   // bytes of [128 rows][64 dims]
constexpr uint32_t PT_TILE = 2 * PT_HALF;
constexpr int PT_PART = 3;                // tiles that some row sees only in part: 256 positions touch 3
constexpr float PT_RAISE = 8.0f;          // log2 growth of the maximum that is let pass

struct PromptSmem {
    unsigned char q[2][PT_TILE];
    unsigned char kv[PT_STAGES][PT_TILE];
    unsigned long long q_full, kv_full[PT_STAGES], kv_empty[PT_STAGES], s_full[2], p_full[2], o_full[2], drain;
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
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, uint32_t acc) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a),
        "l"(b), "r"(kind), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t kind, uint32_t acc) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
        "r"(a), "l"(b), "r"(kind), "r"(acc)
        : "memory");
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
__device__ Block find_block(const QdbPagedAttnArgs &a, int bq, int i) {
    Block k{0, 0, 0, 0, false};
    const int n = a.bt.n_seqs;
    int lo = 0;
    if (a.bt.q_starts) {
        int hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1, st = a.bt.q_starts[mid];
            if (max(st, 0) / bq + mid <= i) lo = mid;
            else hi = mid;
        }
    } else {
        lo = i;
        if (lo >= n) return k;
    }
    int first, last;
    paged_rows(a.bt, lo, first, last);
    const int j = a.bt.q_starts ? i - (first / bq + lo) : 0, blocks = (last - first + bq - 1) / bq;
    if (j < 0 || j >= blocks) return k;
    const int at = (blocks - 1 - j) * bq;
    const int len = paged_len(a.bt, lo, a.kv.page_shift, a.bt.step ? *a.bt.step : 0);
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
        for (int s = 0; s < PT_STAGES; s++) {
            bar_init(smem_u32(&sm.kv_full[s]), 1);
            bar_init(smem_u32(&sm.kv_empty[s]), 1);
        }
        for (int x = 0; x < 2; x++) {
            bar_init(smem_u32(&sm.s_full[x]), 1);
            bar_init(smem_u32(&sm.p_full[x]), 128);
            bar_init(smem_u32(&sm.o_full[x]), 1);
        }
        for (int k = 0; k < PT_PART; k++) {
            bar_init(smem_u32(&sm.v_part[k]), 1);
            bar_init(smem_u32(&sm.v_clean[k]), 64);
        }
        bar_init(smem_u32(&sm.drain), 1);
        sm.abort = 0;
        sm.nonfinite = 0;
        fence_bar_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mq) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
    }
    pdl_enter();
    const Block blk = find_block(a, 2 * QP, blockIdx.x / Hkv);
    if (!blk.any) return;
    // tile x: rows of positions [x * QP, x * QP + nx); keys it needs, in tiles
    const int n0 = min(blk.n, QP), n1 = blk.n - n0;
    const int end0 = max(blk.pos0 + n0, 0), end1 = n1 > 0 ? max(blk.pos0 + blk.n, 0) : 0;
    const int t0 = (end0 + PT_N - 1) / PT_N, t1 = (end1 + PT_N - 1) / PT_N, tiles = max(t0, t1), end = max(end0, end1);
    // tiles from here on are not seen whole by every row
    const int special = max(blk.pos0 + 1, 0) / PT_N;
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tm = sm.tmem;
    auto kv_full = [&](int i) { return smem_u32(&sm.kv_full[i % PT_STAGES]); };
    auto kv_empty = [&](int i) { return smem_u32(&sm.kv_empty[i % PT_STAGES]); };
    auto ring_par = [&](int i) { return (unsigned)(i / PT_STAGES) & 1u; };

    if (warp < 8) {
        // ------------------------------------------------ softmax of row tile x
        const int x = warp >> 2, r = t & 127, nx = x ? n1 : n0, nt = x ? t1 : t0;
        const int i = r / G, h = r - i * G;  // position in the tile, head of the group
        const int pos = blk.pos0 + x * QP + i;
        const bool real = i < nx && i < QP;
        const int whole = max(blk.pos0 + x * QP + 1, 0) / PT_N;  // tiles before this one need no mask
        const uint32_t ts = tm + x * 128 + ((uint32_t)(32 * (warp & 3)) << 16), to = ts + 256;
        const float c = a.scale * 1.4426950408889634f;
        constexpr float shift = T::code == QDB_TYPE_F16 ? 6.f : 0.f;  // keeps f16 weights down to 2^-30 of the largest
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < nt; j++) {
            ok = wait_on(sm, smem_u32(&sm.s_full[x]), j & 1, err);
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            tc_after();
            float s[128];
            tm_ld64(ts, reinterpret_cast<uint32_t *>(s));
            tm_ld64(ts + 64, reinterpret_cast<uint32_t *>(s + 64));
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
                if (j > 0) {  // S of this tile is there, so the product before it is done
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
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 128; k += 64) {
                uint32_t p[32];
#pragma unroll
                for (int e = 0; e < 64; e += 2) {
                    const float p0 = ex2(fmaf(s[k + e], c, -mc)), p1 = ex2(fmaf(s[k + e + 1], c, -mc));
                    sum[e & 2] += p0;
                    sum[(e & 2) + 1] += p1;
                    p[e / 2] = T::plain(p0, p1);
                }
                tm_st32(ts + k / 2, p);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tm_st_wait();
            tc_before();
            bar_arrive(smem_u32(&sm.p_full[x]));
        }
        if (ok && nt > 0) ok = wait_on(sm, smem_u32(&sm.o_full[x]), 0, err);
        ok = __all_sync(0xffffffffu, ok);
        if (ok && nx > 0) {
            tc_after();
            const float inv = l > 0.f ? 1.0f / l : (isnan(l) ? l : 0.f);
            uint16_t *dst = a.out + (size_t)(blk.row0 + x * QP + i) * a.out_stride + ((size_t)g * G + h) * QDB_HD;
            const bool fix = sm.nonfinite != 0;  // (written before the products that o_full waited for)
#pragma unroll 1
            for (int k = 0; k < 128; k += 32) {
                uint32_t o[32];
                if (nt > 0) {
                    tm_ld32(to + k, o);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0u;
                }
                if (!real) continue;
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = __float_as_uint(l > 0.f || isnan(l) ? __uint_as_float(o[e]) * inv : 0.f);
                if (fix)  // non-finite values were left out of the products: add those this row sees
                    for (int key = special * PT_N; key <= pos; key++) {
                        const int page = paged_page(a.kv, a.bt, blk.b, key >> a.kv.page_shift);
                        if (page < 0) continue;
                        const uint16_t *v = a.kv.v + page * a.kv.page_stride + g * a.kv.head_stride +
                                            (key & ((1 << a.kv.page_shift) - 1)) * a.kv.pos_stride + k;
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            const float y = T::lo(v[e]);
                            if (!isfinite(y)) o[e] = __float_as_uint(__uint_as_float(o[e]) + y);
                        }
                    }
#pragma unroll
                for (int e = 0; e < 32; e += 8)
                    *reinterpret_cast<uint4 *>(dst + k + e) =
                        make_uint4(T::plain(__uint_as_float(o[e]), __uint_as_float(o[e + 1])),
                                   T::plain(__uint_as_float(o[e + 2]), __uint_as_float(o[e + 3])),
                                   T::plain(__uint_as_float(o[e + 4]), __uint_as_float(o[e + 5])),
                                   T::plain(__uint_as_float(o[e + 6]), __uint_as_float(o[e + 7])));
            }
        }
    } else if (warp == 8) {
        // ------------------------------------------------ products
        if (lane == 0 && tiles > 0) {
            bool ok = true;
            int issued = 0;
            auto scores = [&](int x, int j) {  // S_x = Q_x K_j^T
                const uint32_t q = smem_u32(sm.q[x]), k = smem_u32(sm.kv[(2 * j) % PT_STAGES]);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    mma_ss(tm + x * 128, op_desc(q + (e >> 2) * PT_HALF + (e & 3) * 32, 16),
                           op_desc(k + (e >> 2) * PT_HALF + (e & 3) * 32, 16), op_kind<T>(false), e > 0);
                commit(smem_u32(&sm.s_full[x]));
                issued++;
            };
            auto output = [&](int x, int j) {  // O_x += P_x V_j
                const uint32_t v = smem_u32(sm.kv[(2 * j + 1) % PT_STAGES]);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    mma_ts(tm + 256 + x * 128, tm + x * 128 + e * 8, op_desc(v + e * 2048, PT_HALF), op_kind<T>(true),
                           j > 0 || e > 0);
            };
            ok = wait_on(sm, smem_u32(&sm.q_full), 0, err) && wait_on(sm, kv_full(0), 0, err);
            if (ok) {
                tc_after();
                if (t0 > 0) scores(0, 0);
                if (t1 > 0) scores(1, 0);
                commit(kv_empty(0));
            }
            for (int j = 0; j < tiles && ok; j++) {
                // V_j (and, where some row sees it only in part, cleared), and K_j+1
                ok = wait_on(sm, kv_full(2 * j + 1), ring_par(2 * j + 1), err);
                if (ok && j >= special) ok = wait_on(sm, smem_u32(&sm.v_clean[j - special]), 0, err);
                if (ok && j + 1 < tiles) ok = wait_on(sm, kv_full(2 * j + 2), ring_par(2 * j + 2), err);
                for (int x = 0; x < 2 && ok; x++) {
                    const int nt = x ? t1 : t0;
                    if (j >= nt) continue;
                    ok = wait_on(sm, smem_u32(&sm.p_full[x]), j & 1, err);
                    if (!ok) break;
                    tc_after();
                    output(x, j);
                    if (j + 1 < nt) scores(x, j + 1);  // (in issue order behind the product that reads P)
                    else commit(smem_u32(&sm.o_full[x]));
                }
                if (!ok) break;
                commit(kv_empty(2 * j + 1));
                if (j + 1 < tiles) commit(kv_empty(2 * j + 2));
            }
            if (!ok && issued) {  // given up: the products in flight end before the CTA does
                commit(smem_u32(&sm.drain));
                bar_wait(smem_u32(&sm.drain), 0, err);
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        // ------------------------------------------------ copies
        if (tiles > 0) {
            if (lane == 0) {
                bar_expect(smem_u32(&sm.q_full), (n1 > 0 ? 4u : 2u) * 128u * G * QP);
                for (int x = 0; x < (n1 > 0 ? 2 : 1); x++)
                    for (int half = 0; half < 2; half++)
                        asm volatile(
                            "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
                            "{%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(sm.q[x]) + half * PT_HALF),
                            "l"(&mq), "r"(0), "r"(half), "r"(g * G), "r"(blk.row0 + x * QP), "r"(smem_u32(&sm.q_full))
                            : "memory");
            }
            const int rows = min(1 << a.kv.page_shift, PT_N), pieces = PT_N / rows;
            bool ok = true;
            int sent = 0;
            for (int j = 0; j < tiles && ok; j++) {
                const int key = j * PT_N + lane * rows;
                const bool mine = lane < pieces && key < end;
                int page = 0;
                if (mine) {
                    page = paged_page(a.kv, a.bt, blk.b, key >> a.kv.page_shift);
                    if (page < 0) page = a.kv.n_pages;  // outside the pool: recorded, reads as zeros
                }
                const int n = min(pieces, (end - j * PT_N + rows - 1) / rows);
                for (int v = 0; v < 2 && ok; v++) {
                    const int i = 2 * j + v;
                    if (i >= PT_STAGES) ok = wait_on(sm, kv_empty(i), ring_par(i) ^ 1u, err);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    // (V of a tile seen in part lands on a barrier of its own, which the
                    // clearing warps wait for; the ring's barrier only keeps its count)
                    const bool part = v && j >= special;
                    const uint32_t bar = part ? smem_u32(&sm.v_part[j - special]) : kv_full(i);
                    if (lane == 0) {
                        bar_expect(bar, (uint32_t)n * rows * 256u);
                        if (part) bar_arrive(kv_full(i));
                    }
                    __syncwarp();
                    if (mine) {
                        const uint32_t dst = smem_u32(sm.kv[i % PT_STAGES]) + lane * rows * 128;
                        const int slot = key & ((1 << a.kv.page_shift) - 1);
#pragma unroll
                        for (int half = 0; half < 2; half++)
                            load_half_page(dst + half * PT_HALF, v ? &mv : &mk, slot, half, g, page, bar);
                    }
                    sent = i + 1;
                }
            }
            if (!ok && lane == 0) {  // given up: the copies in flight land first
                bar_wait(smem_u32(&sm.q_full), 0, err);
                for (int i = max(0, sent - PT_STAGES); i < sent; i++) {
                    bar_wait(kv_full(i), ring_par(i), err);
                    if ((i & 1) && i / 2 >= special) bar_wait(smem_u32(&sm.v_part[i / 2 - special]), 0, err);
                }
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------ V of the tiles that some row sees only in part
        const int u = t - 320;
        bool ok = true;
        for (int j = special; j < tiles && ok; j++) {
            const int i = 2 * j + 1;
            ok = __all_sync(0xffffffffu, wait_on(sm, smem_u32(&sm.v_part[j - special]), 0, err));
            if (!ok) break;
            unsigned char *v = sm.kv[i % PT_STAGES];
            bool odd = false;
#pragma unroll 4
            for (int e = u; e < (int)(PT_TILE / 16); e += 64) {
                // 16 bytes of key (e / 8) % 128 (the swizzle moves them within their row only)
                uint4 *at = reinterpret_cast<uint4 *>(v) + e;
                if (j * PT_N + ((e >> 3) & 127) >= end) {
                    *at = make_uint4(0u, 0u, 0u, 0u);
                } else {
                    uint4 w = *at;
                    if (T::any_nonfinite(w.x) | T::any_nonfinite(w.y) | T::any_nonfinite(w.z) | T::any_nonfinite(w.w)) {
                        odd = true;
                        w.x = T::clear_nonfinite(w.x);
                        w.y = T::clear_nonfinite(w.y);
                        w.z = T::clear_nonfinite(w.z);
                        w.w = T::clear_nonfinite(w.w);
                        *at = w;
                    }
                }
            }
            if (odd) {
                *reinterpret_cast<volatile int *>(&sm.nonfinite) = 1;
                __threadfence_block();
            }
            fence_async();
            bar_arrive(smem_u32(&sm.v_clean[j - special]));
        }
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
