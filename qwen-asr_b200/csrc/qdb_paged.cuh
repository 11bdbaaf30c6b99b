// qdb_paged.cuh - the paged KV cache as the kernels see it: shared by the
// append, the one-token attention and the prompt attention.
//
// One layer's keys and values lie in pages of `page` positions; a sequence's
// positions [i * page, (i + 1) * page) are on page tables[b][i]. Element
// (page p, head g, slot s, dim d) is at p * page_stride + g * head_stride +
// s * pos_stride + d, so both [page][head][slot][128] and
// [page][slot][head][128] pools are read in place.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "../../include/qwen_asr_b200.h"
#include "qdb_common.cuh"

// Which check refused an access (err[1] of the caller's error words).
enum {
    QDB_CHECK_PAGE = 1,    // page id outside the pool: err[2] = sequence, err[3] = page id
    QDB_CHECK_TABLE = 2,   // behind the table's end: err[2] = sequence, err[3] = length (append: position)
    QDB_CHECK_ROPE = 3,    // position behind the rotation table: err[2] = sequence, err[3] = position
    QDB_CHECK_STARTS = 4,  // row range outside [0, rows] or backwards: err[2] = sequence, err[3] = its end
};

struct QdbPagedKV {
    uint16_t *k, *v;
    int n_pages, page_shift, kv_heads;
    long long page_stride, head_stride, pos_stride;
};

struct QdbPagedBatch {
    int n_seqs, rows;
    const int *q_starts;  // [n_seqs + 1], null: row b is sequence b
    const int *lens;      // [n_seqs] positions, the new rows among them
    const int *tables;    // [n_seqs][table_stride]
    int table_stride;
    int *err;         // nullable [4]
    const int *step;  // nullable: added to every length (a captured step's counter)
};

// 16-bit element types of cache, queries and output.
struct QdbHalf {
    static constexpr int code = QDB_TYPE_F16;
    static __device__ __forceinline__ float lo(uint32_t w) { return kvlo(w); }
    static __device__ __forceinline__ float hi(uint32_t w) { return kvhi(w); }
    // stores saturate at +-65504 (the cache's rule); NaN stays NaN
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return (uint32_t)one(a) | ((uint32_t)one(b) << 16);
    }
    static __device__ __forceinline__ uint16_t one(float f) { return isnan(f) ? (uint16_t)0x7fffu : f32_to_kv(f); }
    // without saturation: infinities stay
    static __device__ __forceinline__ uint16_t plain1(float f) { return __half_as_ushort(__float2half_rn(f)); }
    static __device__ __forceinline__ uint32_t plain(float a, float b) {
        const __half2 r = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    // acc + 0 * w of both halves: NaN from the first non-finite value on
    static __device__ __forceinline__ uint32_t zero_times(uint32_t w, uint32_t acc) {
        const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&w), __half2half2(__ushort_as_half(0)),
                                  *reinterpret_cast<const __half2 *>(&acc));
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    static __device__ __forceinline__ bool any_nonfinite(uint32_t w) {
        return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
    }
    static __device__ __forceinline__ uint32_t clear_nonfinite(uint32_t w) {
        if ((w & 0x7c00u) == 0x7c00u) w &= 0xffff0000u;
        if ((w & 0x7c000000u) == 0x7c000000u) w &= 0xffffu;
        return w;
    }
};
struct QdbBf16 {
    static constexpr int code = QDB_TYPE_BF16;
    static __device__ __forceinline__ float lo(uint32_t w) { return bf16lo(w); }
    static __device__ __forceinline__ float hi(uint32_t w) { return bf16hi(w); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    static __device__ __forceinline__ uint16_t one(float f) { return f32_to_bf16_rn(f); }
    static __device__ __forceinline__ uint16_t plain1(float f) { return one(f); }
    static __device__ __forceinline__ uint32_t plain(float a, float b) { return pack(a, b); }
    static __device__ __forceinline__ uint32_t zero_times(uint32_t w, uint32_t acc) {
        const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&w), __bfloat162bfloat162(__ushort_as_bfloat16(0)),
                                         *reinterpret_cast<const __nv_bfloat162 *>(&acc));
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    static __device__ __forceinline__ bool any_nonfinite(uint32_t w) {
        return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
    }
    static __device__ __forceinline__ uint32_t clear_nonfinite(uint32_t w) {
        if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
        if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
        return w;
    }
};

// Length of sequence b for reading: never negative, never behind its page table.
__device__ __forceinline__ int paged_len(const QdbPagedBatch &bt, int b, int page_shift, int step) {
    long long n = (long long)bt.lens[b] + step;
    const long long most = (long long)bt.table_stride << page_shift;
    if (n > most) {
        check_or_record(false, bt.err, QDB_CHECK_TABLE, b, n);
        n = most;
    }
    return n > 0 ? (int)n : 0;
}

// Rows [first, last) of sequence b, clamped to [0, rows] and never backwards.
__device__ __forceinline__ void paged_rows(const QdbPagedBatch &bt, int b, int &first, int &last) {
    if (!bt.q_starts) {
        first = b;
        last = b + 1;
        return;
    }
    first = bt.q_starts[b];
    last = bt.q_starts[b + 1];
    if (first < 0 || last > bt.rows || last < first) {
        check_or_record(false, bt.err, QDB_CHECK_STARTS, b, last);
        first = last = 0;
    }
}

// Page id of sequence b's i-th page, or -1 (recorded) when it is outside the pool.
__device__ __forceinline__ int paged_page(const QdbPagedKV &kv, const QdbPagedBatch &bt, int b, int i) {
    const int p = i < bt.table_stride ? bt.tables[(size_t)b * bt.table_stride + i] : -1;
    return check_or_record(p >= 0 && p < kv.n_pages, bt.err, QDB_CHECK_PAGE, b, p) ? p : -1;
}

// ---- barriers and tensor copies ----
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, unsigned n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, unsigned parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return ok != 0;
}
// (without waiting; bar_try may sleep until the phase ends)
__device__ __forceinline__ bool bar_test(uint32_t bar, unsigned parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return ok != 0;
}
// Bounded wait; false = ran out (recorded). The waits that drain a CTA's own
// copies or products before it exits take the fixed limit.
__device__ __forceinline__ bool bar_wait(uint32_t bar, unsigned parity, int *err, long long limit = QDB_SPIN_LIMIT_CYCLES) {
    if (bar_test(bar, parity)) return true;
    const long long t0 = clock64();
    do {
        if (clock64() - t0 >= limit) {
            set_error(err, QDB_ERR_BARRIER_TIMEOUT);
            return false;
        }
    } while (!bar_try(bar, parity));
    return true;
}
__device__ __forceinline__ void fence_bar_init() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
// Generic-proxy shared-memory accesses ordered before later asynchronous ones.
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The pools as 5-dimensional tensors (64 dims, slot, dim half, head, page):
// one copy brings `rows` slots of a page as two [rows][64] halves, each with
// rows of 128 bytes in the 128-byte swizzle.
__device__ __forceinline__ void load_page(uint32_t dst, const CUtensorMap *map, int slot, int head, int page,
                                          uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
        "%6}], [%7];" ::"r"(dst),
        "l"(map), "r"(0), "r"(slot), "r"(0), "r"(head), "r"(page), "r"(bar)
        : "memory");
}
// One half only, from a map of one half per copy.
__device__ __forceinline__ void load_half_page(uint32_t dst, const CUtensorMap *map, int slot, int half, int head,
                                               int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
        "%6}], [%7];" ::"r"(dst),
        "l"(map), "r"(0), "r"(slot), "r"(half), "r"(head), "r"(page), "r"(bar)
        : "memory");
}
// Host: writes that map. rows: slots per copy (at most the page size), halves: 1 or 2 per copy. 0 = ok.
int qdb_paged_map(CUtensorMap *map, const void *pool, const QdbPagedKV &kv, int type, int rows, int halves);
// Rows [rows][heads][128] of queries as (64 dims, dim half, head, row): a copy
// brings one half of box_heads heads of box_rows rows.
int qdb_encode_map4(CUtensorMap *map, const void *q, int type, uint64_t heads, uint64_t rows, uint64_t row_stride,
                    uint32_t box_heads, uint32_t box_rows);

// ---- host checks: refuses misaligned pointers, host pointers and pointers of
// another device than the current one (null pointers are left to the caller).
// 0 = ok.
struct QdbNamedPtr {
    const void *p;
    const char *name;
    int align = 4;
};
int qdb_check_device_ptrs(const char *fn, const QdbNamedPtr *ps, int n);

// ---- launchers (checked arguments) ----
struct QdbAppendArgs {
    QdbPagedKV kv;
    QdbPagedBatch bt;
    const void *qkv;
    long long row_stride;  // elements of the source type
    int heads;
    const float *q_norm, *k_norm;  // nullable
    float eps;
    const float2 *rope;  // nullable
    int rope_len;
    uint16_t *q_out;
    long long q_stride;
};
cudaError_t qdb_launch_paged_append(const QdbAppendArgs &a, int src_type, int kv_type, cudaStream_t st);

struct QdbPagedAttnArgs {
    QdbPagedKV kv;
    QdbPagedBatch bt;
    const uint16_t *q;
    long long q_stride;
    int heads;
    float scale;
    uint16_t *out;
    long long out_stride;
    uint16_t *lo;  // nullable: `out` receives the result as bf16 and lo its rest (hi + lo), whatever the cache's type
};
// One value of the bf16 pair: its hi part, or what that leaves.
__device__ __forceinline__ float pair_part(float v, bool lo) {
    const float hi = __uint_as_float((uint32_t)f32_to_bf16_rn(v) << 16);
    return lo ? v - hi : v;
}
// Scratch of one call at a time: partial results [2 * ctas][16][128] with their
// (m, l), and [ctas] counters, zero between calls.
struct QdbDecodeScratch {
    float *part;
    float2 *ml;
    unsigned *cnt;
    int ctas;
};
cudaError_t qdb_decode_scratch_alloc(int device, QdbDecodeScratch *s);  // on the current device
// Limit of the kernels' data waits in cycles, on the current device.
extern "C" cudaError_t qdb_set_wait_limit_paged_decode(long long cycles);
extern "C" cudaError_t qdb_set_wait_limit_paged_prompt(long long cycles);  // (at most 3e9)
cudaError_t qdb_launch_paged_decode(const QdbPagedAttnArgs &a, int type, const QdbDecodeScratch &ws, cudaStream_t st);
cudaError_t qdb_launch_paged_prompt(const QdbPagedAttnArgs &a, int type, cudaStream_t st);

struct QdbSampleArgs {
    const void *logits;
    long long row_stride;
    int rows, vocab;
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *uniform;
    int mask_eos;
    int *tokens;
    const int *step;  // nullable: uniform and tokens advance by *step * rows
};
cudaError_t qdb_launch_sample(const QdbSampleArgs &a, int type, cudaStream_t st);
