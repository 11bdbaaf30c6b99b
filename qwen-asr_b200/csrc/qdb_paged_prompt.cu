// qdb_paged_prompt.cu - causal attention of packed prompts over a paged KV
// cache on the tensor cores (tcgen05).
//
// An item is one key head and one block of a sequence's new rows: two tiles of
// 128 MMA rows (row r = position r / G, head r % G of the group), which share
// every K and V tile of 128 keys. It is bound by the tensor cores and by the
// exponentials (128 x 128 of them per tile take as long on the special
// function units as the tile's two products take on the tensor cores), so
// neither may wait for the other: the two row tiles run half a step apart, and
// a row tile's next scores are there before its softmax of this tile ends.
//   warps 0-3, 4-7  softmax of tile 0, 1: thread = row = TMEM lane
//   warp 8          issues S = Q K^T      (two warps, since waiting for the next
//   warp 9          issues O += P V        operands takes half as long as a product),
//                   and clears what V holds behind the last visible key
//   warp 10         announces the items, copies Q and the pages of K (ring of 2 tiles)
//   warp 11         copies the pages of V (ring of 3)
// TMEM: S (128 columns, read into registers at once, so one serves both row
// tiles in turn), P0, P1 (64 columns of packed 16-bit pairs, the A operand of
// the second product), O0, O1 (128 columns each). No product waits for another
// one's TMEM columns but through the softmax.
// V is used as loaded (keys along K, dims along N).
// One CTA per SM walks through items, taking the next from the launch queue:
// its look-ups, copies and first scores run while the last one's output leaves.
//   m, l            running maximum and sum per row in f32; O is rescaled only
//                   when the maximum grows by more than 2^8, so numerator and
//                   denominator always share one m
//   P               rounded to the cache's type (the type of V's own rounding; error
//                   against 64 bits 1.1 to 1.3 times that of f32 arithmetic. A second
//                   half of P would need 64 more columns per row tile: 640 of 512)
// The roles' code together does not fit the instruction caches, and what runs
// once per item is fetched anew each time: loops over it are kept short and not
// unrolled, nothing is divided, non-finite values are dealt with after the
// stores. (64 prompts of 404 positions took 152 us with 83 KB of code, 99 with 58.)
// Measured, 16 heads on 8 key heads: 16384 positions bf16 813 us in short bursts
// (1.35 PFLOP/s), 950 run on and on, where power sets the clock; 3721 positions
// 55 us; 64 pieces of 30 to 130 rows behind up to 400 cached positions 38 us; one
// prompt of 404 13 us, most of it the chain of look-ups, copies and four tiles. A
// first version on the CUDA cores took 182 ms for the 16384, 1.7 ms for the pieces.
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
constexpr int PT_PART = 4;                // its barriers: more than such tiles in the ring
constexpr int PT_ITEMS = 4;               // announced items
constexpr float PT_RAISE = 8.0f;          // log2 growth of the maximum that is let pass

// One item's rows.
struct Block {
    int b, row0, n, pos0;  // sequence, its first row here, rows (positions) here, position of the first
    bool any;
};
struct Item {
    Block blk;
    int g;          // key head
    int nonfinite;  // set where values had to be cleared
};

struct PromptSmem {
    unsigned char q[2][PT_TILE];
    unsigned char k[PT_KS][PT_TILE], v[PT_VS][PT_TILE];
    unsigned long long q_full, q_empty, k_full[PT_KS], k_empty[PT_KS], v_full[PT_VS], v_empty[PT_VS];
    unsigned long long s_full[2], s_read, p_full[2], o_done[2], drain[2];
    unsigned long long v_clean[PT_PART];  // one half of a V tile seen in part is cleared
    unsigned long long item_full[PT_ITEMS], item_empty[PT_ITEMS];
    Item item[PT_ITEMS];
    alignas(16) uint64_t stolen[2];  // answer to a request for another CTA's number
    unsigned long long stolen_bar;
    uint32_t tmem;
    int abort;
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
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t kind, uint32_t more) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
        "r"(a), "l"(b), "r"(kind), "r"(more)
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
// Limit of the data waits in 32-bit cycles (well below where the counter comes
// round; qdb_set_wait_limit_paged_prompt).
__constant__ unsigned prompt_wait_limit = (unsigned)QDB_SPIN_LIMIT_CYCLES;

// Bounded wait that also ends when another role has given up. (Short: it is
// inlined at every wait. The error is recorded once, at the end.)
__device__ __forceinline__ bool wait_on(PromptSmem &sm, uint32_t bar, unsigned parity) {
    if (bar_test(bar, parity)) return true;
    const unsigned t0 = (unsigned)clock();
    do {
        if (*reinterpret_cast<volatile int *>(&sm.abort) || (unsigned)clock() - t0 >= prompt_wait_limit) {
            *reinterpret_cast<volatile int *>(&sm.abort) = 1;
            return false;
        }
    } while (!bar_try(bar, parity));
    return true;
}

// Blocks of bq rows: sequence b's begin at number q_starts[b] / bq + b, which
// leaves room for every sequence's last, partly filled block (the numbers
// behind it are empty). The blocks with the longest histories come first.
__device__ Block find_block(const QdbPagedAttnArgs &a, int bq, unsigned inv_bq, int i, int lane) {
    Block k{0, 0, 0, 0, false};
    const int n = a.bt.n_seqs, step = a.bt.step ? *a.bt.step : 0;
    int lo = 0;
    if (a.bt.q_starts) {  // the last sequence that begins at or before i, 32 candidates at a time
#pragma unroll 1
        for (int size = n; size > 1;) {
            const int d = (size + 31) / 32, mid = lo + lane * d;
            const bool in = lane * d < size && (int)__umulhi(max(a.bt.q_starts[mid], 0), inv_bq) + mid <= i;
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
    const int j = a.bt.q_starts ? i - ((int)__umulhi(first, inv_bq) + lo) : 0, blocks = __umulhi(last - first + bq - 1, inv_bq);
    if (j < 0 || j >= blocks) return k;
    const int at = (blocks - 1 - j) * bq;
    k.b = lo;
    k.row0 = first + at;
    k.n = min(bq, last - first - at);
    k.pos0 = len - (last - first) + at;
    k.any = true;
    return k;
}

// What the roles derive from a block.
struct Shape {
    int b, row0, pos0, g;
    int n0, n1;                    // positions of row tiles 0 and 1
    int t0, t1, tiles, end;        // key tiles they need, and all; keys
    int special, parts;            // first tile that some row does not see whole; number of such tiles
    __device__ __forceinline__ Shape(const Block &k, int g, int QP) : b(k.b), row0(k.row0), pos0(k.pos0), g(g) {
        n0 = min(k.n, QP);
        n1 = k.n - n0;
        const int end0 = max(pos0 + n0, 0), end1 = n1 > 0 ? max(pos0 + k.n, 0) : 0;
        t0 = (end0 + PT_N - 1) / PT_N;
        t1 = (end1 + PT_N - 1) / PT_N;
        tiles = max(t0, t1);
        end = max(end0, end1);
        special = max(pos0 + 1, 0) / PT_N;
        parts = max(tiles - special, 0);
    }
};

template <typename T, bool PAIR>  // PAIR: the output as a bf16 pair (a.out, a.lo)
__global__ void __launch_bounds__(PT_THREADS, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv, const __grid_constant__ QdbPagedAttnArgs a) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    PromptSmem &sm = *reinterpret_cast<PromptSmem *>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int Hkv = a.kv.kv_heads, G = a.heads / Hkv, QP = 128 / G;  // positions per row tile
    int *err = a.bt.err;
    if (t == 0) {
        bar_init(smem_u32(&sm.q_full), 1);
        bar_init(smem_u32(&sm.q_empty), 1);
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
            bar_init(smem_u32(&sm.drain[x]), 1);
        }
        bar_init(smem_u32(&sm.s_read), 128);
        for (int k = 0; k < PT_PART; k++) bar_init(smem_u32(&sm.v_clean[k]), 1);
        for (int k = 0; k < PT_ITEMS; k++) {
            bar_init(smem_u32(&sm.item_full[k]), 1);
            bar_init(smem_u32(&sm.item_empty[k]), 11);  // every warp but the announcing one
        }
        bar_init(smem_u32(&sm.stolen_bar), 1);
        sm.abort = 0;
        fence_bar_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mq) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
    }
    __syncthreads();
    pdl_enter();
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
    // Every role walks through the CTA's items on its own, as warp 10 announces
    // them, and keeps its own counts of the barriers' phases.
    bool ok = true;
    auto wait = [&](uint32_t bar, unsigned parity) { return __all_sync(0xffffffffu, wait_on(sm, bar, parity)); };
    int item = 0;
    Block blk;
    int g = 0;
    auto next_item = [&]() -> bool {  // the announced block; false: no more (or given up)
        const int k = item % PT_ITEMS;
        ok = wait(smem_u32(&sm.item_full[k]), (item / PT_ITEMS) & 1);
        if (!ok) return false;
        blk = sm.item[k].blk;
        g = sm.item[k].g;
        item++;
        return blk.any;
    };
    auto item_done = [&] {  // this warp no longer needs the announcement
        __syncwarp();
        if (lane == 0) bar_arrive(smem_u32(&sm.item_empty[(item - 1) % PT_ITEMS]));
    };

    // Half the dims of a V tile that some row sees only in part: behind the last
    // visible key they are zero, non-finite values are zero and noted.
    auto clear_v = [&](unsigned st, int half, int keys) {
        uint4 *v = reinterpret_cast<uint4 *>(sm.v[st] + half * PT_HALF);
        const int mine = keys * 8;  // 16 bytes of key e / 8 (the swizzle moves them within their row only)
        uint32_t acc = 0;
#pragma unroll 4
        for (int e = lane; e < (int)(PT_HALF / 16); e += 32) {
            uint4 w = v[e];
            if (e >= mine) v[e] = w = make_uint4(0u, 0u, 0u, 0u);
            acc |= T::zero_times(w.w, T::zero_times(w.z, T::zero_times(w.y, T::zero_times(w.x, 0))));
        }
        if (T::any_nonfinite(acc)) {
            *reinterpret_cast<volatile int *>(&sm.item[(item - 1) % PT_ITEMS].nonfinite) = 1;
            __threadfence_block();
#pragma unroll 1
            for (int e = lane; e < mine; e += 32) {
                const uint4 w = v[e];
                v[e] = make_uint4(T::clear_nonfinite(w.x), T::clear_nonfinite(w.y), T::clear_nonfinite(w.z),
                                  T::clear_nonfinite(w.w));
            }
        }
        fence_async();  // (before the product's reads, and the next copy into the stage)
        __syncwarp();
    };

    if (warp < 8) {
        // ------------------------------------------------ softmax of row tile x
        const int x = warp >> 2, r = t & 127;
        const unsigned inv_g = (65536u + G - 1) / G;  // n / G = n * inv_g >> 16 for n < 128
        const int i = (int)((unsigned)r * inv_g >> 16);  // position in the row tile
        const uint32_t ts = tm + ((uint32_t)(32 * (warp & 3)) << 16), tp = ts + 128 + x * 64, to = ts + 256 + x * 128;
        const float c = a.scale * 1.4426950408889634f;
        constexpr float shift = T::code == QDB_TYPE_F16 ? 6.f : 0.f;  // keeps f16 weights down to 2^-30 of the largest
        unsigned n_s = 0;  // score tiles of x before this item
        while (next_item()) {
            const Shape sh(blk, g, QP);
            const int *nonfinite = &sm.item[(item - 1) % PT_ITEMS].nonfinite;
            const int nx = x ? sh.n1 : sh.n0, nt = x ? sh.t1 : sh.t0;
            const int pos = sh.pos0 + x * QP + i;
            const bool real = i < nx && i < QP;
            const int whole = max(sh.pos0 + x * QP + 1, 0) / PT_N;  // tiles before this one need no mask
            float m = -INFINITY, l = 0.f;
            // The output product of tile j - 1 has read P and written O.
            auto done_before = [&](int j) {
                const bool done = wait(smem_u32(&sm.o_done[x]), (n_s + j - 1) & 1);
                tc_after();
                return done;
            };
            for (int j = 0; j < nt; j++) {
                ok = wait(smem_u32(&sm.s_full[x]), (n_s + j) & 1);
                if (!ok) break;
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
                if (!ok) break;
                float s0, s1;
                unpair(add2(sum[0], sum[1]), s0, s1);
                l += s0 + s1;
                tm_st_wait();
                tc_before();
                bar_arrive(smem_u32(&sm.p_full[x]));
            }
            if (ok && nt > 0) ok = done_before(nt);
            if (!ok) break;
            if (nx > 0) {
                if (nt == 0) {  // nothing to see for any row
                    uint32_t zero[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) zero[e] = 0u;
#pragma unroll 1
                    for (int k = 0; k < 128; k += 32) tm_st32(to + k, zero);
                    tm_st_wait();
                }
                const float scale_o = l > 0.f ? 1.0f / l : (isnan(l) ? l : 0.f);
                const bool fix = *reinterpret_cast<const volatile int *>(nonfinite) != 0;  // (written before the products)
                for (int part = 0; part < (PAIR ? 2 : 1); part++) {  // (hi, then lo of a bf16 pair)
                    auto word = [&](uint32_t y, uint32_t z) {
                        const float u = __uint_as_float(y), v = __uint_as_float(z);
                        return PAIR ? QdbBf16::plain(pair_part(u, part), pair_part(v, part)) : T::plain(u, v);
                    };
#pragma unroll 1
                    for (int k = 0; k < 128; k += 32) {
                        uint32_t o[32];
                        tm_ld32(to + k, o);
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * scale_o);
                        // (two lanes exchange pieces: each store writes whole 32-byte sectors)
                        const bool up = lane & 1;
                        const int rr0 = r & ~1, i0 = (int)((unsigned)rr0 * inv_g >> 16), i1 = (int)((unsigned)(rr0 + 1) * inv_g >> 16);
                        uint16_t *dst = (part ? a.lo : a.out) + (size_t)g * G * QDB_HD + k + (lane & 1) * 8;
                        uint16_t *d0 = dst + (size_t)(sh.row0 + x * QP + i0) * a.out_stride + (rr0 - i0 * G) * QDB_HD;
                        uint16_t *d1 = dst + (size_t)(sh.row0 + x * QP + i1) * a.out_stride + (rr0 + 1 - i1 * G) * QDB_HD;
                        const bool r0 = i0 < nx && i0 < QP, r1 = i1 < nx && i1 < QP;
#pragma unroll
                        for (int e = 0; e < 32; e += 16) {
                            uint32_t lo[4], hi[4];
#pragma unroll
                            for (int z = 0; z < 4; z++) {
                                const uint32_t p = word(o[e + 2 * z], o[e + 2 * z + 1]), q = word(o[e + 8 + 2 * z], o[e + 9 + 2 * z]);
                                const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? p : q, 1);
                                lo[z] = up ? got : p;
                                hi[z] = up ? q : got;
                            }
                            if (r0) *reinterpret_cast<uint4 *>(d0 + e) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                            if (r1) *reinterpret_cast<uint4 *>(d1 + e) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        }
                    }
                }
                if (fix) {  // non-finite values were left out of the products: add those each row sees
                    __syncwarp();
                    if (real) {
                        uint16_t *dst = a.out + (size_t)(sh.row0 + x * QP + i) * a.out_stride + ((size_t)g * G + r - i * G) * QDB_HD;
#pragma unroll 1
                        for (int key = sh.special * PT_N; key <= pos; key++) {
                            const int page = paged_page(a.kv, a.bt, sh.b, key >> a.kv.page_shift);
                            if (page < 0) continue;
                            const uint16_t *v = a.kv.v + page * a.kv.page_stride + g * a.kv.head_stride +
                                                (key & ((1 << a.kv.page_shift) - 1)) * a.kv.pos_stride;
#pragma unroll 1
                            for (int e = 0; e < QDB_HD; e++) {
                                const float y = T::lo(v[e]);
                                if (isfinite(y)) continue;
                                dst[e] = PAIR ? QdbBf16::plain1(QdbBf16::lo(dst[e]) + y) : T::plain1(T::lo(dst[e]) + y);
                            }
                        }
                    }
                }
            }
            tc_before();  // (O has been read: before the next item's first weights are announced)
            n_s += nt;
            item_done();
        }
        tm_st_wait();  // (where a wait ran out: before the columns are given back)
    } else if (warp < 10) {
        // ------------------------------------------------ products: warp 8 the scores, warp 9 the outputs
        // (the whole warp runs this together, with values that are the same in all
        // lanes, so that they stay in uniform registers, where the products' operands
        // have to be; one lane issues)
        const uint32_t tmu = __shfl_sync(0xffffffffu, tm, 0);
        const bool scores_warp = warp == 8, leader = elect();  // (a commit covers its own thread's products)
        const uint64_t q_desc = op_desc(smem_u32(sm.q[0]), 16), k_desc = op_desc(smem_u32(sm.k[0]), 16),
                       v_desc = op_desc(smem_u32(sm.v[0]), PT_HALF);
        constexpr uint64_t tile = PT_TILE >> 4;
        auto scores = [&](int x, unsigned st) {  // S = Q_x K^T
            const uint64_t q = q_desc + x * tile, k = k_desc + st * tile;
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
        auto output = [&](int x, unsigned st, bool more) {  // O_x (+)= P_x V
            const uint64_t v = v_desc + st * tile;
            const uint32_t d = tmu + 256 + x * 128, p = tmu + 128 + x * 64;
            if (leader) {
                mma_ts(d, p, v, op_kind<T>(true), more);
#pragma unroll
                for (int e = 1; e < 8; e++) mma_ts(d, p + e * 8, v + e * (2048 >> 4), op_kind<T>(true), 1);
                commit(smem_u32(&sm.o_done[x]));
            }
            __syncwarp();
        };
        unsigned st = 0, phase = 0;  // ring stage of the next tile, how often the ring has gone round (mod 2)
        unsigned n_part = 0, n_q = 0, n_s = 0, n_p0 = 0, n_p1 = 0;
        while (next_item()) {
            const Shape sh(blk, g, QP);
            const int T0 = __shfl_sync(0xffffffffu, sh.t0, 0), T1 = __shfl_sync(0xffffffffu, sh.t1, 0), TT = max(T0, T1);
            const int part = __shfl_sync(0xffffffffu, sh.special, 0);
            item_done();
            if (TT == 0) continue;
            if (scores_warp) ok = wait(smem_u32(&sm.q_full), n_q++ & 1);
            // row tiles 0 and 1 in turn, tile after tile
            for (int j = 0; j < TT && ok; j++) {
                ok = wait(smem_u32(scores_warp ? &sm.k_full[st] : &sm.v_full[st]), phase);
                if (!scores_warp && ok && j >= part) {  // warp 11 clears the other half
                    clear_v(st, 0, min(sh.end - j * PT_N, PT_N));
                    ok = wait(smem_u32(&sm.v_clean[n_part % PT_PART]), (n_part / PT_PART) & 1);
                    n_part++;
                }
#pragma unroll 1
                for (int x = 0; x < 2 && ok; x++) {
                    if (j >= (x ? T1 : T0)) continue;
                    if (scores_warp) {  // (the scores before have been read)
                        if (n_s) ok = wait(smem_u32(&sm.s_read), (n_s - 1) & 1);
                        n_s++;
                    } else {
                        ok = wait(smem_u32(&sm.p_full[x]), (x ? n_p1++ : n_p0++) & 1);
                    }
                    if (!ok) break;
                    tc_after();
                    if (scores_warp) scores(x, st);
                    else output(x, st, j > 0);
                }
                if (ok && leader) commit(smem_u32(scores_warp ? &sm.k_empty[st] : &sm.v_empty[st]));
                __syncwarp();
                if (++st == (scores_warp ? PT_KS : PT_VS)) st = 0, phase ^= 1;
            }
            if (!ok) break;
            if (scores_warp && leader) commit(smem_u32(&sm.q_empty));
            __syncwarp();
        }
        // the products and commits in flight end before the CTA does
        if (leader) commit(smem_u32(&sm.drain[warp - 8]));
        __syncwarp();
        bar_wait(smem_u32(&sm.drain[warp - 8]), 0, err);
        __syncwarp();
    } else {
        // ------------------------------------------------ copies: warp 10 Q and K (and the items), warp 11 V
        const bool is_v = warp == 11, leader = elect();
        const int rsh = min(a.kv.page_shift, 7), rows = 1 << rsh, pieces = PT_N >> rsh, S = is_v ? PT_VS : PT_KS;
        unsigned long long *full = is_v ? sm.v_full : sm.k_full, *empty = is_v ? sm.v_empty : sm.k_empty;
        const uint32_t ring = smem_u32(is_v ? sm.v[0] : sm.k[0]);
        const CUtensorMap *map = is_v ? &mv : &mk;
        unsigned n_tile = 0, n_q = 0, n_part = 0, st = 0, phase = 0;
        // The CTA's items: its own number, then those of CTAs that have not been
        // launched yet, taken from the launch queue until none is left. It asks for
        // the next one two tiles before this one's end: at once, a CTA with a heavy
        // item would keep a second one from those that will be free before it.
        int number = blockIdx.x;
        const unsigned inv_bq = 0xffffffffu / (2 * QP) + 1;  // n / bq = n * inv_bq >> 32 for n < 2^23, bq <= 256
        unsigned asked = 0, answered = 0;
        auto ask = [&] {
            if (leader) {
                fence_async();  // (the last answer has been read)
                bar_expect(smem_u32(&sm.stolen_bar), 16);
                asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                                 smem_u32(sm.stolen)),
                             "r"(smem_u32(&sm.stolen_bar))
                             : "memory");
            }
            __syncwarp();
            asked++;
        };
        auto answer = [&] {  // the number taken, or -1: none is left
            ok = wait(smem_u32(&sm.stolen_bar), answered & 1);
            if (!ok) return -1;
            answered++;
            const volatile uint64_t *w = sm.stolen;
            const uint64_t lo = w[0], hi = w[1];
            uint32_t got, x = 0;
            asm volatile(
                "{ .reg .b128 r; .reg .pred p; mov.b128 r, {%2, %3};\n\t"
                "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
                "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
                "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r; }"
                : "=r"(got), "=r"(x)
                : "l"(lo), "l"(hi));
            __syncwarp();
            return got ? (int)x : -1;
        };
        bool first = true;
        auto announce = [&]() -> bool {  // the next block that has rows
            for (;; first = false) {
                if (!first && number >= 0) {
                    if (asked == answered) ask();
                    number = answer();
                    if (!ok) return false;
                }
                Block k{0, 0, 0, 0, false};
                int kh = 0;
                if (number >= 0) {
                    const int blk_no = number / Hkv;
                    k = find_block(a, 2 * QP, inv_bq, blk_no, lane);
                    kh = number - blk_no * Hkv;
                    if (!k.any) continue;
                }
                const int s = item % PT_ITEMS;
                if (item >= PT_ITEMS) ok = wait(smem_u32(&sm.item_empty[s]), ((item / PT_ITEMS) & 1) ^ 1);
                if (!ok) return false;
                blk = k;
                g = kh;
                if (lane == 0) {
                    sm.item[s] = Item{k, g, 0};
                    bar_arrive(smem_u32(&sm.item_full[s]));
                }
                __syncwarp();
                item++;
                first = false;
                return k.any;
            }
        };
        while (is_v ? next_item() : announce()) {
            const Shape sh(blk, g, QP);
            auto look_up = [&](int j) {  // this lane's page of tile j
                const int key = j * PT_N + lane * rows;
                if (lane >= pieces || key >= sh.end) return -1;
                const int p = paged_page(a.kv, a.bt, sh.b, key >> a.kv.page_shift);
                return p < 0 ? a.kv.n_pages : p;  // outside the pool: recorded, reads as zeros
            };
            if (sh.tiles == 0) {
                if (is_v) item_done();
                continue;
            }
            int page = -1;
            const int end = __shfl_sync(0xffffffffu, sh.end, 0), head = __shfl_sync(0xffffffffu, g, 0);
            for (int j = -1; j < sh.tiles; j++) {
                const int after = j + 1 < sh.tiles ? look_up(j + 1) : -1;  // (not waited for before it is needed)
                if (j < 0) {
                    page = after;
                    continue;
                }
                const int n = min(pieces, (end - j * PT_N + rows - 1) >> rsh), slot = (j * PT_N) & ((1 << a.kv.page_shift) - 1);
                if (n_tile >= (unsigned)S) ok = wait(smem_u32(&empty[st]), phase ^ 1);
                if (!ok) break;
                // pieces one after the other, all operands the same in every lane
                const uint32_t dst = ring + st * PT_TILE, bar = smem_u32(&full[st]);
                if (leader) bar_expect(bar, (uint32_t)n * rows * 256u);
#pragma unroll 1
                for (int p = 0; p < n; p++) {
                    const int pg = __shfl_sync(0xffffffffu, page, p);
                    if (leader) {
                        load_half_page(dst + p * rows * 128, map, slot, 0, head, pg, bar);
                        load_half_page(dst + p * rows * 128 + PT_HALF, map, slot, 1, head, pg, bar);
                    }
                }
                __syncwarp();
                n_tile++;
                if (++st == (unsigned)S) st = 0, phase ^= 1;
                page = after;
                if (is_v) continue;
                if (j == 0) {  // Q, once the item before has no more use for its rows
                    if (n_q) ok = wait(smem_u32(&sm.q_empty), (n_q - 1) & 1);
                    if (!ok) break;
                    n_q++;
                    if (leader) {
                        bar_expect(smem_u32(&sm.q_full), (sh.n1 > 0 ? 4u : 2u) * 128u * G * QP);
                        for (int x = 0; x < (sh.n1 > 0 ? 2 : 1); x++)
                            for (int half = 0; half < 2; half++)
                                asm volatile(
                                    "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
                                    "[%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(sm.q[x]) + half * PT_HALF),
                                    "l"(&mq), "r"(0), "r"(half), "r"(head * G), "r"(sh.row0 + x * QP),
                                    "r"(smem_u32(&sm.q_full))
                                    : "memory");
                    }
                    __syncwarp();
                }
                if (j == max(sh.tiles - 2, 0)) ask();
            }
            if (!ok) break;
            if (is_v) {
                // (all of the item's tiles are on their way: those seen in part are its last
                // ones, no more than the ring holds, so none waits for another's clearing)
                for (int j = sh.special; j < sh.tiles; j++, n_part++) {
                    const unsigned k = n_tile - sh.tiles + j;
                    ok = wait(smem_u32(&sm.v_full[k % PT_VS]), (k / PT_VS) & 1);
                    if (!ok) break;
                    clear_v(k % PT_VS, 1, min(end - j * PT_N, PT_N));
                    if (leader) bar_arrive(smem_u32(&sm.v_clean[n_part % PT_PART]));
                }
                if (!ok) break;
                item_done();
            }
        }
        // what is in flight lands before the CTA ends, whatever role has given up
        // (none has: its copies have been waited for, and these checks find them there)
        const int ring_tiles = min(n_tile, (unsigned)S);
#pragma unroll 1
        for (int k = -2; k < ring_tiles; k++) {
            uint32_t bar = smem_u32(&sm.stolen_bar);
            unsigned parity = answered & 1;
            if (k == -2 && asked == answered) continue;
            if (k == -1) {
                if (!n_q) continue;
                bar = smem_u32(&sm.q_full), parity = (n_q - 1) & 1;
            } else if (k >= 0) {  // (the ring's tiles, the newest first)
                if (st-- == 0) st = S - 1, phase ^= 1;
                bar = smem_u32(&full[st]), parity = phase;
            }
            bar_wait(bar, parity, err);
        }
        __syncwarp();
    }
    tc_before();
    __syncthreads();
    if (t == 0 && sm.abort) set_error(err, QDB_ERR_BARRIER_TIMEOUT);
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

template <typename T, bool PAIR>
cudaError_t launch(const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, const QdbPagedAttnArgs &a,
                   cudaStream_t st) {
    const size_t smem = sizeof(PromptSmem) + 1024;
    cudaError_t e = cudaFuncSetAttribute(prompt_kernel<T, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const int G = a.heads / a.kv.kv_heads, bq = 2 * (128 / G);
    const long long blocks = a.bt.q_starts ? (long long)a.bt.rows / bq + a.bt.n_seqs : a.bt.n_seqs;
    if (blocks * a.kv.kv_heads > 2147483647ll) return cudaErrorInvalidConfiguration;
    return pdl_launch(prompt_kernel<T, PAIR>, dim3((unsigned)(blocks * a.kv.kv_heads)), dim3(PT_THREADS), smem, st, mq, mk, mv, a);
}

}  // namespace

extern "C" cudaError_t qdb_set_wait_limit_paged_prompt(long long cycles) {
    const unsigned c = (unsigned)(cycles < 3000000000ll ? cycles : 3000000000ll);
    return cudaMemcpyToSymbol(prompt_wait_limit, &c, sizeof(c));
}

cudaError_t qdb_launch_paged_prompt(const QdbPagedAttnArgs &a, int type, cudaStream_t st) {
    CUtensorMap mq, mk, mv;
    const int page = 1 << a.kv.page_shift, rows = page < PT_N ? page : PT_N;
    if (query_map(&mq, a, type, a.heads / a.kv.kv_heads) || qdb_paged_map(&mk, a.kv.k, a.kv, type, rows, 1) ||
        qdb_paged_map(&mv, a.kv.v, a.kv, type, rows, 1))
        return cudaErrorInvalidValue;
    if (a.lo)
        return type == QDB_TYPE_F16 ? launch<QdbHalf, true>(mq, mk, mv, a, st) : launch<QdbBf16, true>(mq, mk, mv, a, st);
    return type == QDB_TYPE_F16 ? launch<QdbHalf, false>(mq, mk, mv, a, st) : launch<QdbBf16, false>(mq, mk, mv, a, st);
}
