// qdb_paged.cu - paged KV cache: rotation and append of new positions; tensor
// maps of the pages; the C entry points of the paged operators and their checks.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math.h>
#include <stdio.h>

#include <new>

#include "qdb_kernels.h"
#include "qdb_paged.cuh"

namespace {

// ---------------------------------------------------------------- append
// y = x * rsqrt(mean(x^2) + eps) * w for query and key heads (where norms are
// given), then the rotation of the halves (a, b) -> (a c - b s, b c + a s)
// with (c, s) the position's table row; values as they are.

// Sequence of a row: the last b with q_starts[b] <= row (rows behind the last
// sequence: n_seqs).
__device__ __forceinline__ int row_sequence(const QdbPagedBatch &bt, int row) {
    if (!bt.q_starts) return row;
    int lo = 0, hi = bt.n_seqs;  // q_starts[lo] <= row < q_starts[hi + 1] as far as known
    if (bt.q_starts[hi] <= row) return bt.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (bt.q_starts[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

struct SrcF32 {};
// 8 consecutive source elements as they are, and widened.
template <typename S>
struct Raw8 {
    uint4 w;
    __device__ __forceinline__ void load(const void *p, size_t i) { w = ldg_stream(reinterpret_cast<const uint16_t *>(p) + i); }
    __device__ __forceinline__ void widen(float *v) const {
        v[0] = S::lo(w.x), v[1] = S::hi(w.x), v[2] = S::lo(w.y), v[3] = S::hi(w.y);
        v[4] = S::lo(w.z), v[5] = S::hi(w.z), v[6] = S::lo(w.w), v[7] = S::hi(w.w);
    }
};
template <>
struct Raw8<SrcF32> {
    uint4 w[2];
    __device__ __forceinline__ void load(const void *p, size_t i) {
        w[0] = ldg_stream(reinterpret_cast<const float *>(p) + i);
        w[1] = ldg_stream(reinterpret_cast<const float *>(p) + i + 4);
    }
    __device__ __forceinline__ void widen(float *v) const {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            v[4 * h] = __uint_as_float(w[h].x), v[4 * h + 1] = __uint_as_float(w[h].y);
            v[4 * h + 2] = __uint_as_float(w[h].z), v[4 * h + 3] = __uint_as_float(w[h].w);
        }
    }
};

// Bound by memory: every row is read once and written once. Eight lanes take a
// few head vectors of one row: lane i holds dims 8 i .. 8 i + 7 of both halves,
// the pairs that rotate together, so all loads and stores are 16 bytes. The row's
// sequence, position and page are looked up once for its vectors here, and the
// table row is read once. Measured: 26k rows of 32 vectors, bf16 to bf16, rotation
// only, 77 us (6.1 TB/s, 95 % of the copy) with four vectors, 87 with two, 96 with
// one (bound by the look-ups' instructions), 88 with eight; 3721 rows, f32 to f16,
// norms and rotation, 17.8 us (5.2 TB/s) with two, 25 with one, 21 with four; 64
// rows 4.4 us, which is the launch and the look-ups. Six CTAs per SM: 80 registers
// (of the 16-bit sources' four vectors 20 to 32 bytes spill).
constexpr int AP_THREADS = 128, AP_GROUPS = AP_THREADS / 8, AP_CTAS = 6;
template <typename S>
constexpr int ap_vecs = 4;
template <>
constexpr int ap_vecs<SrcF32> = 2;  // (twice the registers per vector)

template <typename S, typename T>
__global__ void __launch_bounds__(AP_THREADS, AP_CTAS) append_kernel(const QdbAppendArgs a, int units) {
    constexpr int U = ap_vecs<S>;
    pdl_enter();
    const int i8 = (threadIdx.x & 7) * 8, Hq = a.heads, Hkv = a.kv.kv_heads, slots = Hq + 2 * Hkv;
    const unsigned unit = blockIdx.x * AP_GROUPS + threadIdx.x / 8;  // (rows that fit the memory have fewer than 2^32)
    const int row = (int)(unit / (unsigned)units), s0 = (int)(unit - (unsigned)row * units) * U;
    const bool here = row < a.bt.rows;
    // the source does not depend on the look-ups: its loads go first
    Raw8<S> rx[U], ry[U];
#pragma unroll
    for (int u = 0; u < U; u++)
        if (here && s0 + u < slots) {
            const size_t at = (size_t)row * a.row_stride + (size_t)(s0 + u) * QDB_HD + i8;
            rx[u].load(a.qkv, at);
            ry[u].load(a.qkv, at + 64);
        }
    if (!here) return;
    const unsigned lanes = 0xffu << (threadIdx.x & 24);  // (the row's lanes leave together)
    const int b = row_sequence(a.bt, row);
    if (b >= a.bt.n_seqs) return;
    int first, last;
    paged_rows(a.bt, b, first, last);
    if (row < first || row >= last) return;
    const long long at64 = (long long)a.bt.lens[b] + (a.bt.step ? *a.bt.step : 0) - (last - row);
    if (at64 < 0) return;  // the sequence is shorter than its rows
    // a row that has no place in the page table, or cannot be rotated, is left out whole
    const bool held = at64 >> a.kv.page_shift < a.bt.table_stride;
    if (!check_or_record(held, a.bt.err, QDB_CHECK_TABLE, b, at64)) return;
    const int pos = (int)at64;
    if (a.rope && !check_or_record(pos < a.rope_len, a.bt.err, QDB_CHECK_ROPE, b, pos)) return;
    float4 cs[4];  // (cos, sin) of two pairs each
    if (a.rope && s0 < Hq + Hkv) {
        const float4 *p = reinterpret_cast<const float4 *>(a.rope + (size_t)pos * (QDB_HD / 2) + i8);
#pragma unroll
        for (int e = 0; e < 4; e++) cs[e] = p[e];
    }
    size_t at = 0;  // of the position in either pool
    bool paged = false;
    if (s0 + U > Hq) {
        const int page = paged_page(a.kv, a.bt, b, pos >> a.kv.page_shift);
        paged = page >= 0;
        at = page * a.kv.page_stride + (pos & ((1 << a.kv.page_shift) - 1)) * a.kv.pos_stride;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int slot = s0 + u;
        if (slot >= slots) break;
        float x[8], y[8];
        rx[u].widen(x);
        ry[u].widen(y);
        const float *w = slot < Hq ? a.q_norm : slot < Hq + Hkv ? a.k_norm : nullptr;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor_sync(lanes, ss, o);
            const float inv = 1.0f / sqrtf(ss / (float)QDB_HD + a.eps);
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 p = *reinterpret_cast<const float4 *>(w + i8 + e), q = *reinterpret_cast<const float4 *>(w + 64 + i8 + e);
                x[e] *= inv * p.x, x[e + 1] *= inv * p.y, x[e + 2] *= inv * p.z, x[e + 3] *= inv * p.w;
                y[e] *= inv * q.x, y[e + 1] *= inv * q.y, y[e + 2] *= inv * q.z, y[e + 3] *= inv * q.w;
            }
        }
        if (a.rope && slot < Hq + Hkv) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float4 r = cs[e / 2];
                const float x0 = x[e], x1 = x[e + 1];
                x[e] = x0 * r.x - y[e] * r.y;
                y[e] = y[e] * r.x + x0 * r.y;
                x[e + 1] = x1 * r.z - y[e + 1] * r.w;
                y[e + 1] = y[e + 1] * r.z + x1 * r.w;
            }
        }
        uint16_t *dst;
        if (slot < Hq) {
            dst = a.q_out + (size_t)row * a.q_stride + (size_t)slot * QDB_HD;
        } else {
            if (!paged) break;
            const bool is_k = slot < Hq + Hkv;
            dst = (is_k ? a.kv.k : a.kv.v) + at + (is_k ? slot - Hq : slot - Hq - Hkv) * a.kv.head_stride;
        }
        *reinterpret_cast<uint4 *>(dst + i8) =
            make_uint4(T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7]));
        *reinterpret_cast<uint4 *>(dst + 64 + i8) =
            make_uint4(T::pack(y[0], y[1]), T::pack(y[2], y[3]), T::pack(y[4], y[5]), T::pack(y[6], y[7]));
    }
}

}  // namespace

template <typename S>
static cudaError_t launch_append(const QdbAppendArgs &a, int kv_type, cudaStream_t st) {
    const int units = (a.heads + 2 * a.kv.kv_heads + ap_vecs<S> - 1) / ap_vecs<S>;  // of a row
    const long long groups = (long long)a.bt.rows * units;
    if (groups > 0xffffff00ll) return cudaErrorInvalidConfiguration;
    const dim3 grid((unsigned)((groups + AP_GROUPS - 1) / AP_GROUPS)), block(AP_THREADS);
    return kv_type == QDB_TYPE_F16 ? pdl_launch(append_kernel<S, QdbHalf>, grid, block, 0, st, a, units)
                                   : pdl_launch(append_kernel<S, QdbBf16>, grid, block, 0, st, a, units);
}

cudaError_t qdb_launch_paged_append(const QdbAppendArgs &a, int src_type, int kv_type, cudaStream_t st) {
    if (src_type == QDB_TYPE_F32) return launch_append<SrcF32>(a, kv_type, st);
    if (src_type == QDB_TYPE_F16) return launch_append<QdbHalf>(a, kv_type, st);
    return launch_append<QdbBf16>(a, kv_type, st);
}

cudaError_t qdb_decode_scratch_alloc(int device, QdbDecodeScratch *s) {
    cudaError_t e = cudaDeviceGetAttribute(&s->ctas, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = cudaMalloc((void **)&s->part, sizeof(float) * 2 * s->ctas * 16 * QDB_HD);
    if (e == cudaSuccess) e = cudaMalloc((void **)&s->ml, sizeof(float2) * 2 * s->ctas * 16);
    if (e == cudaSuccess) e = cudaMalloc((void **)&s->cnt, sizeof(unsigned) * s->ctas);
    if (e == cudaSuccess) e = cudaMemset(s->cnt, 0, sizeof(unsigned) * s->ctas);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e != cudaSuccess) {  // all or nothing
        cudaFree(s->part);
        cudaFree(s->ml);
        cudaFree(s->cnt);
        *s = {};
    }
    return e;
}

static int encode_map(CUtensorMap *map, const void *p, int type, int rank, const cuuint64_t *dims,
                      const cuuint64_t *strides, const cuuint32_t *box) {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult qr;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qr) == cudaSuccess &&
                        qr == cudaDriverEntryPointSuccess;
        return ok ? (PFN_cuTensorMapEncodeTiled_v12000)f : nullptr;
    }();
    if (!fn) return -1;
    const cuuint32_t es[5] = {1, 1, 1, 1, 1};
    return fn(map, type == QDB_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
              const_cast<void *>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0
               : -1;
}

int qdb_paged_map(CUtensorMap *map, const void *pool, const QdbPagedKV &kv, int type, int rows, int halves) {
    const cuuint64_t dims[5] = {64, (cuuint64_t)1 << kv.page_shift, 2, (cuuint64_t)kv.kv_heads, (cuuint64_t)kv.n_pages};
    const cuuint64_t strides[4] = {(cuuint64_t)kv.pos_stride * 2, 128, (cuuint64_t)kv.head_stride * 2,
                                   (cuuint64_t)kv.page_stride * 2};
    const cuuint32_t box[5] = {64, (cuuint32_t)rows, (cuuint32_t)halves, 1, 1};
    return encode_map(map, pool, type, 5, dims, strides, box);
}

int qdb_encode_map4(CUtensorMap *map, const void *q, int type, uint64_t heads, uint64_t rows, uint64_t row_stride,
                    uint32_t box_heads, uint32_t box_rows) {
    const cuuint64_t dims[4] = {64, 2, heads, rows};
    const cuuint64_t strides[3] = {128, 256, row_stride * 2};
    const cuuint32_t box[4] = {64, 1, box_heads, box_rows};
    return encode_map(map, q, type, 4, dims, strides, box);
}

// ---------------------------------------------------------------- C entry points
// The device of a pointer is checked before every launch: a host pointer, or
// one of another device than the current one, is refused instead of read.
static bool on_device(const void *p, int dev, const char *what, char *msg, size_t len) {
    cudaPointerAttributes at{};
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        snprintf(msg, len, "%s: %s", what, cudaGetErrorString(e));
        return false;
    }
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) {
        snprintf(msg, len, "%s is not a device pointer", what);
        return false;
    }
    if (at.type == cudaMemoryTypeDevice && at.device != dev) {
        snprintf(msg, len, "%s is on device %d, the current device is %d", what, at.device, dev);
        return false;
    }
    return true;
}

int qdb_check_device_ptrs(const char *fn, const QdbNamedPtr *ps, int n) {
    char msg[256], full[320];
    for (int i = 0; i < n; i++)
        if ((uintptr_t)ps[i].p % ps[i].align) {
            snprintf(full, sizeof(full), "%s: %s is not aligned to %d bytes", fn, ps[i].name, ps[i].align);
            return qdb_set_error(full);
        }
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) {
        cudaGetLastError();
        snprintf(full, sizeof(full), "%s: %s", fn, cudaGetErrorString(e));
        return qdb_set_error(full);
    }
    for (int i = 0; i < n; i++)
        if (ps[i].p && !on_device(ps[i].p, dev, ps[i].name, msg, sizeof(msg))) {
            snprintf(full, sizeof(full), "%s: %s", fn, msg);
            return qdb_set_error(full);
        }
    return 0;
}

#define REFUSE(cond, ...)                                     \
    do {                                                      \
        if (cond) {                                           \
            char m_[320];                                     \
            snprintf(m_, sizeof(m_), __VA_ARGS__);            \
            return qdb_set_error(m_);                         \
        }                                                     \
    } while (0)

static inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

static int check_kv(const char *fn, const qdb_paged_kv *kv, QdbPagedKV *o) {
    REFUSE(!kv || !kv->k || !kv->v, "%s: null cache", fn);
    REFUSE(kv->type != QDB_TYPE_F16 && kv->type != QDB_TYPE_BF16, "%s: cache type %d is not f16 or bf16", fn, kv->type);
    REFUSE(kv->n_pages <= 0 || kv->kv_heads <= 0, "%s: bad pool: %d pages of %d heads", fn, kv->n_pages, kv->kv_heads);
    int shift = 4;
    while (shift < 8 && (1 << shift) != kv->page_size) shift++;
    REFUSE((1 << shift) != kv->page_size, "%s: page size %d is not 16, 32, 64, 128 or 256", fn, kv->page_size);
    o->k = (uint16_t *)kv->k;
    o->v = (uint16_t *)kv->v;
    o->n_pages = kv->n_pages;
    o->page_shift = shift;
    o->kv_heads = kv->kv_heads;
    o->page_stride = kv->page_stride;
    o->head_stride = kv->head_stride;
    o->pos_stride = kv->pos_stride;
    if (!kv->page_stride && !kv->head_stride && !kv->pos_stride) {
        o->pos_stride = QDB_HD;
        o->head_stride = (long long)kv->page_size * QDB_HD;
        o->page_stride = o->head_stride * kv->kv_heads;
    }
    const long long st[3] = {o->page_stride, o->head_stride, o->pos_stride};
    for (long long s : st)
        REFUSE(s < QDB_HD || s % 8 || s >= (1ll << 38), "%s: cache stride %lld (needs a multiple of 8 from 128 up)", fn, s);
    REFUSE(!aligned16(kv->k) || !aligned16(kv->v), "%s: the cache must start on a 16-byte boundary", fn);
    return 0;
}

static int check_batch(const char *fn, const qdb_paged_batch *b, QdbPagedBatch *o) {
    REFUSE(!b, "%s: null batch", fn);
    REFUSE(b->n_seqs < 0 || b->rows < 0, "%s: negative size", fn);
    REFUSE(b->rows > (1 << 22), "%s: %d rows exceed the 4M-row limit", fn, b->rows);
    REFUSE(b->n_seqs > (1 << 20), "%s: %d sequences exceed the 1M limit", fn, b->n_seqs);
    *o = QdbPagedBatch{b->n_seqs, b->rows, b->q_starts, b->kv_lens, b->tables, b->table_stride, b->err, nullptr};
    if (!b->n_seqs || !b->rows) return 0;
    REFUSE(!b->kv_lens || !b->tables, "%s: null lengths or page tables", fn);
    REFUSE(b->table_stride <= 0 || b->table_stride > (1 << 22), "%s: page tables of %d entries", fn, b->table_stride);
    REFUSE(!b->q_starts && b->rows != b->n_seqs, "%s: %d rows of %d sequences need q_starts", fn, b->rows, b->n_seqs);
    return 0;
}

static int check_heads(const char *fn, int heads, int kv_heads) {
    REFUSE(heads <= 0 || heads % kv_heads || heads / kv_heads > 16 || heads > 1024,
           "%s: %d heads over %d key heads (needs a multiple, at most 16 each)", fn, heads, kv_heads);
    return 0;
}

static int launched(const char *fn, cudaError_t e) {
    REFUSE(e != cudaSuccess, "%s: %s", fn, cudaGetErrorString(e));
    return 0;
}

// Workspace of the one-token attention.
struct qdb_paged_workspace {
    int device;
    QdbDecodeScratch s;
};

extern "C" qdb_paged_workspace *qdb_paged_workspace_create(int device) {
    qdb_set_error("");
    const int n = qdb_device_count();
    if (device < 0 || device >= n) {
        char m[128];
        snprintf(m, sizeof(m), "CUDA device %d not available (%d visible)", device, n);
        qdb_set_error(m);
        return nullptr;
    }
    qdb_paged_workspace *ws = new (std::nothrow) qdb_paged_workspace{device, {}};
    if (!ws) {
        qdb_set_error("qdb_paged_workspace_create: out of memory");
        return nullptr;
    }
    int before = 0;
    cudaGetDevice(&before);
    cudaError_t e = cudaSetDevice(device);
    if (e == cudaSuccess) e = qdb_decode_scratch_alloc(device, &ws->s);
    cudaSetDevice(before);
    if (e != cudaSuccess) {
        char m[160];
        snprintf(m, sizeof(m), "qdb_paged_workspace_create: %s", cudaGetErrorString(e));
        qdb_set_error(m);
        qdb_paged_workspace_free(ws);
        return nullptr;
    }
    return ws;
}

extern "C" void qdb_paged_workspace_free(qdb_paged_workspace *ws) {
    if (!ws) return;
    cudaFree(ws->s.part);  // (cudaFree waits for the device's work)
    cudaFree(ws->s.ml);
    cudaFree(ws->s.cnt);
    delete ws;
}

extern "C" int qdb_paged_append(const qdb_paged_kv *kv, const qdb_paged_batch *batch, const void *qkv, int src_type,
                                long long row_stride, int heads, const float *q_norm, const float *k_norm, float eps,
                                const float *rope, int rope_len, void *q_out, long long q_stride, void *stream) {
    const char *fn = "qdb_paged_append";
    qdb_set_error("");
    QdbAppendArgs a{};
    if (check_kv(fn, kv, &a.kv) || check_batch(fn, batch, &a.bt) || check_heads(fn, heads, kv->kv_heads)) return -1;
    REFUSE(src_type != QDB_TYPE_F32 && src_type != QDB_TYPE_F16 && src_type != QDB_TYPE_BF16, "%s: source type %d", fn,
           src_type);
    if (!a.bt.n_seqs || !a.bt.rows) return 0;
    const long long width = (long long)(heads + 2 * kv->kv_heads) * QDB_HD;
    const int unit = src_type == QDB_TYPE_F32 ? 4 : 8;
    REFUSE(!qkv || !q_out, "%s: null rows", fn);
    REFUSE((row_stride && row_stride < width) || row_stride % unit, "%s: row stride %lld", fn, row_stride);
    REFUSE((q_stride && q_stride < (long long)heads * QDB_HD) || q_stride % 8, "%s: query stride %lld", fn, q_stride);
    REFUSE(!aligned16(qkv) || !aligned16(q_out) || !aligned16(q_norm) || !aligned16(k_norm) || !aligned16(rope),
           "%s: pointers must be on 16-byte boundaries", fn);
    REFUSE(rope && rope_len <= 0, "%s: rotation table of %d positions", fn, rope_len);
    const QdbNamedPtr ps[] = {{kv->k, "k"}, {kv->v, "v"}, {batch->q_starts, "q_starts"}, {batch->kv_lens, "kv_lens"},
                           {batch->tables, "tables"}, {batch->err, "err"}, {qkv, "qkv"}, {q_norm, "q_norm"},
                           {k_norm, "k_norm"}, {rope, "rope"}, {q_out, "q_out"}};
    if (qdb_check_device_ptrs(fn, ps, (int)(sizeof(ps) / sizeof(ps[0])))) return -1;
    a.qkv = qkv;
    a.row_stride = row_stride ? row_stride : width;
    a.heads = heads;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    a.rope = (const float2 *)rope;
    a.rope_len = rope_len;
    a.q_out = (uint16_t *)q_out;
    a.q_stride = q_stride ? q_stride : (long long)heads * QDB_HD;
    return launched(fn, qdb_launch_paged_append(a, src_type, kv->type, (cudaStream_t)stream));
}

// Checks of both attention forms; 1 = nothing to do.
static int check_attn(const char *fn, const qdb_paged_kv *kv, const qdb_paged_batch *batch, const void *q,
                      long long q_stride, int heads, float scale, void *out, long long out_stride,
                      QdbPagedAttnArgs *a) {
    if (check_kv(fn, kv, &a->kv) || check_batch(fn, batch, &a->bt) || check_heads(fn, heads, kv->kv_heads)) return -1;
    REFUSE(!(scale >= 0.f) || scale > 3e38f, "%s: scale %g", fn, (double)scale);
    if (!a->bt.n_seqs || !a->bt.rows) return 1;
    const long long width = (long long)heads * QDB_HD;
    REFUSE(!q || !out, "%s: null rows", fn);
    REFUSE((q_stride && q_stride < width) || q_stride % 8, "%s: query stride %lld", fn, q_stride);
    REFUSE((out_stride && out_stride < width) || out_stride % 8, "%s: output stride %lld", fn, out_stride);
    REFUSE(!aligned16(q) || !aligned16(out), "%s: rows must start on 16-byte boundaries", fn);
    const QdbNamedPtr ps[] = {{kv->k, "k"}, {kv->v, "v"}, {batch->q_starts, "q_starts"}, {batch->kv_lens, "kv_lens"},
                           {batch->tables, "tables"}, {batch->err, "err"}, {q, "q"}, {out, "out"}};
    if (qdb_check_device_ptrs(fn, ps, (int)(sizeof(ps) / sizeof(ps[0])))) return -1;
    a->q = (const uint16_t *)q;
    a->q_stride = q_stride ? q_stride : width;
    a->heads = heads;
    a->scale = scale > 0.f ? scale : 1.0f / sqrtf((float)QDB_HD);
    a->out = (uint16_t *)out;
    a->out_stride = out_stride ? out_stride : width;
    return 0;
}

extern "C" int qdb_paged_decode(const qdb_paged_kv *kv, const qdb_paged_batch *batch, const void *q,
                                long long q_stride, int heads, float scale, void *out, long long out_stride,
                                qdb_paged_workspace *ws, void *stream) {
    const char *fn = "qdb_paged_decode";
    qdb_set_error("");
    QdbPagedAttnArgs a{};
    REFUSE(batch && batch->q_starts, "%s: one row per sequence (q_starts must be null)", fn);
    REFUSE(!ws, "%s: null workspace", fn);
    const int rc = check_attn(fn, kv, batch, q, q_stride, heads, scale, out, out_stride, &a);
    if (rc) return rc < 0 ? -1 : 0;
    int dev = 0;
    cudaGetDevice(&dev);
    REFUSE((double)batch->n_seqs * batch->table_stride * kv->page_size / 16 * kv->kv_heads >= 2147483648.0,
           "%s: %d page tables of %d entries are too many positions for one call", fn, batch->n_seqs,
           batch->table_stride);
    REFUSE(ws->device != dev, "%s: the workspace is of device %d, the current device is %d", fn, ws->device, dev);
    return launched(fn, qdb_launch_paged_decode(a, kv->type, ws->s, (cudaStream_t)stream));
}

extern "C" int qdb_paged_prompt(const qdb_paged_kv *kv, const qdb_paged_batch *batch, const void *q,
                                long long q_stride, int heads, float scale, void *out, long long out_stride,
                                void *stream) {
    const char *fn = "qdb_paged_prompt";
    qdb_set_error("");
    QdbPagedAttnArgs a{};
    const int rc = check_attn(fn, kv, batch, q, q_stride, heads, scale, out, out_stride, &a);
    if (rc) return rc < 0 ? -1 : 0;
    return launched(fn, qdb_launch_paged_prompt(a, kv->type, (cudaStream_t)stream));
}
