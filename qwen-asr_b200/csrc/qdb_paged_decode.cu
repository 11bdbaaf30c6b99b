// qdb_paged_decode.cu - attention of one new token per sequence over a paged
// KV cache: o = softmax(scale q K^T) V for every query head.
//
// Every cached key and value is read once, so the pass is bound by HBM. The
// (sequence, key head) pairs' 16-key tiles form one list, sequence by
// sequence; it is cut into equal contiguous ranges, one per warp of a grid of
// one CTA per SM, whatever the lengths are. A warp runs its range on its own:
// its lane 0 keeps a ring of tiles in flight (one tensor copy for K, one for V
// per tile; the ring runs on across the pairs), and all query heads of the
// pair are computed together, 16 keys at a time, with a running maximum m and
// sum l per head in f32:
//   S^T = K q^T      (keys x heads: K as the row operand, ldmatrix)
//   P = 2^(S c - m)  (c = scale log2 e), rounded to the cache's type
//   O^T += V^T P^T   (dims x heads: V as the row operand, transposed ldmatrix;
//                     P^T by movmatrix from the S^T fragment)
// A pair that lies in several warps' ranges leaves partial (m, l, O); the
// CTA's parts are joined in shared memory, and where it spans CTAs the last
// one to arrive joins them, always in the order of the list, so the result
// does not depend on timing.
#include <math.h>

#include "qdb_kernels.h"
#include "qdb_paged.cuh"

namespace {

constexpr int DW = 8;             // warps per CTA
constexpr int TILE = 16;          // keys per tile (a page holds whole tiles)
constexpr int TILE_B = 4096;      // bytes of a tile's K (or V)
constexpr int MAX_G = 16;         // query heads per key head
constexpr float P_SHIFT = 8.0f;   // P is scaled by 2^8: f16 keeps weights down to 2^-32 of the largest

// Ring stages per warp: what shared memory leaves beside one partial per warp.
__host__ __device__ constexpr int ring_stages(int nt) { return nt == 1 ? 3 : 2; }

// A pair whose parts are all there: sequence, key head, first CTA, CTAs.
struct Whole {
    bool some;
    int b, g, c0, parts;
};

template <int NT>
struct DecodeSmem {
    static constexpr int NS = ring_stages(NT), H = 8 * NT;
    unsigned char ring[DW][NS][2][TILE_B];
    float head_part[DW][H][QDB_HD];  // the part of a pair that began in an earlier warp
    float2 ml[DW][2][H];             // (m, l) of the head part and of the last part
    unsigned long long full[DW][NS];
    long long scan[DW];
    int start[DW][3];                // sequence, key head, tile of each warp's first tile
    Whole todo;
};

__device__ __forceinline__ void ldsm4(uint32_t *r, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t *r, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <typename T>
__device__ __forceinline__ void mma16(float *c, const uint32_t *a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<QdbHalf>(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<QdbBf16>(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) { return exp2f(x); }

// A position in the list of tiles.
struct Cursor {
    int b, g, tile, nt, len;
};

// One joined part: head h's (m, l) and this lane's 4 dims.
struct Join {
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    __device__ __forceinline__ void add(float2 ml, float4 x) {
        const float mn = fmaxf(m, ml.x);
        const float f = m == mn ? 1.f : ex2(m - mn), w = ml.x == mn ? 1.f : ex2(ml.x - mn);
        l = l * f + ml.y * w;
        o[0] = o[0] * f + x.x * w;
        o[1] = o[1] * f + x.y * w;
        o[2] = o[2] * f + x.z * w;
        o[3] = o[3] * f + x.w * w;
        m = mn;
    }
};

template <typename T>
__device__ __forceinline__ void store_row4(uint16_t *dst, const Join &j) {
    const float inv = j.l > 0.f ? 1.0f / j.l : (isnan(j.l) ? j.l : 0.f);
    *reinterpret_cast<uint2 *>(dst) =
        make_uint2(T::pack(j.o[0] * inv, j.o[1] * inv), T::pack(j.o[2] * inv, j.o[3] * inv));
}

template <typename T, int NT>
__global__ void __launch_bounds__(DW * 32, 1)
    decode_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                  const __grid_constant__ QdbPagedAttnArgs a, const QdbDecodeScratch ws) {
    using S = DecodeSmem<NT>;
    constexpr int NS = S::NS;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    S &sm = *reinterpret_cast<S *>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int Hkv = a.kv.kv_heads, G = a.heads / Hkv, n = a.bt.n_seqs;
    const uint32_t full0 = smem_u32(sm.full[warp]);
    if (lane == 0) {
        for (int s = 0; s < NS; s++) bar_init(full0 + 8 * s, 1);
        fence_bar_init();
    }
    pdl_enter();
    const int step = a.bt.step ? *a.bt.step : 0;
    auto length = [&](int b) { return paged_len(a.bt, b, a.kv.page_shift, step); };

    // ---- the list: tiles before each thread's share of the sequences
    const int per = (n + DW * 32 - 1) / (DW * 32), b0 = min(n, t * per), b1 = min(n, b0 + per);
    long long mine = 0;
    for (int b = b0; b < b1; b++) {
        const int len = length(b);
        mine += (len + TILE - 1) / TILE;
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) sm.scan[warp] = upto;
    __syncthreads();
    long long total = 0, before = 0;
    for (int w = 0; w < DW; w++) {
        if (w < warp) before += sm.scan[w];
        total += sm.scan[w];
    }
    before += upto - mine;
    total *= Hkv;
    // rows of empty sequences are zero
    for (int b = blockIdx.x; b < n; b += gridDim.x)
        if (length(b) == 0)
            for (int i = t; i < a.heads * (QDB_HD / 8); i += DW * 32)
                *reinterpret_cast<uint4 *>(a.out + (size_t)b * a.out_stride + i * 8) = make_uint4(0u, 0u, 0u, 0u);
    if (total == 0) return;
    // CTAs that take part: all of them where there are more pairs than CTAs;
    // else a whole number per pair (equal lengths then need no join across
    // CTAs beyond the pair's own), each with at least 32 tiles (512 keys) on
    // average, below which a join costs more than the shorter range saves
    const long long avg = total / ((long long)n * Hkv);
    const long long np = (long long)n * Hkv;
    int ctas = ws.ctas;
    if (np <= ws.ctas) {
        long long k = avg / 32;
        if (k < 1) k = 1;
        if (k > ws.ctas / np) k = ws.ctas / np;
        ctas = (int)(np * k);
    }
    // (a tile for every warp: a range is empty only where one CTA does it all)
    if (ctas > total / DW) ctas = total >= DW ? (int)(total / DW) : 1;
    if ((int)blockIdx.x >= ctas) return;
    const long long nw = (long long)ctas * DW;
    auto first_of = [&](long long w) { return total * w / nw; };  // first tile of global warp w's range
    auto warp_of = [&](long long x) { return ((x + 1) * nw + total - 1) / total - 1; };  // its inverse
    const long long gw0 = (long long)blockIdx.x * DW;
    for (int w = 0; w < DW; w++) {
        const long long x = first_of(gw0 + w);
        if (x >= before * Hkv && x < (before + mine) * Hkv) {
            long long at = before * Hkv;
            for (int b = b0; b < b1; b++) {
                const int nt = (length(b) + TILE - 1) / TILE;
                if (x < at + (long long)nt * Hkv) {
                    sm.start[w][0] = b;
                    sm.start[w][1] = (int)((x - at) / nt);
                    sm.start[w][2] = (int)((x - at) % nt);
                    break;
                }
                at += (long long)nt * Hkv;
            }
        }
    }
    __syncthreads();

    const long long x0 = first_of(gw0 + warp), x1 = first_of(gw0 + warp + 1);
    const int count = (int)(x1 - x0);
    // ---- copies: lane 0 issues tile i + NS when tile i has been used
    Cursor pc, cc;
    auto seek = [&](Cursor &c) {  // the warp's first tile
        c.b = sm.start[warp][0];
        c.g = sm.start[warp][1];
        c.tile = sm.start[warp][2];
        c.len = length(c.b);
        c.nt = (c.len + TILE - 1) / TILE;
    };
    auto advance = [&](Cursor &c) {
        if (++c.tile < c.nt) return;
        c.tile = 0;
        if (++c.g < Hkv) return;
        c.g = 0;
        do {
            c.b++;
            c.len = c.b < n ? length(c.b) : 1;
        } while (c.len == 0);
        c.nt = (c.len + TILE - 1) / TILE;
    };
    const int tshift = a.kv.page_shift - 4, tmask = (1 << tshift) - 1;  // tiles per page
    unsigned char *ring = &sm.ring[warp][0][0][0];
    const uint32_t ring_u = smem_u32(ring);
    auto page_of = [&](const Cursor &c) {
        // (a page outside the pool is recorded and reads as zeros: coordinates
        // behind the tensor's end)
        const int p = paged_page(a.kv, a.bt, c.b, c.tile >> tshift);
        return p < 0 ? a.kv.n_pages : p;
    };
    auto issue = [&](int s, const Cursor &c, int page) {
        bar_expect(full0 + 8 * s, 2 * TILE_B);
        load_page(ring_u + s * 2 * TILE_B, &mk, (c.tile & tmask) * TILE, c.g, page, full0 + 8 * s);
        load_page(ring_u + s * 2 * TILE_B + TILE_B, &mv, (c.tile & tmask) * TILE, c.g, page, full0 + 8 * s);
    };
    int issued = 0, next_page = 0;
    if (count > 0) {
        seek(pc);
        cc = pc;
        if (lane == 0)
            for (; issued < min(NS, count); issued++) {
                issue(issued, pc, page_of(pc));
                advance(pc);
            }
        if (lane == 0 && issued < count) next_page = page_of(pc);
    }

    // ---- compute
    const float c = a.scale * 1.4426950408889634f;
    const int qr = lane >> 2, qc = lane & 3;  // fragment row and column pair
    float o[8][NT][4], m[NT][2], l[NT][2];
    uint32_t qf[8][NT][2];
    bool alive = true;
    int used = 0;
    bool has_head = false, has_last = false;  // partial results left in shared memory
    long long pair_lo = x0 - (count > 0 ? cc.tile : 0);  // list position of the current pair's first tile
    const uint32_t krow = (lane & 7) + ((lane >> 3) & 1) * 8, kch = lane >> 4;
    const uint32_t vrow = (lane & 7) + (lane >> 4) * 8, vch = (lane >> 3) & 1;
    for (int i = 0; i < count && alive; i++) {
        if (i == 0 || cc.tile == 0) {  // a new pair: its queries
            const uint16_t *q = a.q + (size_t)cc.b * a.q_stride + (size_t)cc.g * G * QDB_HD;
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const int h = j * 8 + qr;
#pragma unroll
                for (int ks = 0; ks < 8; ks++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        qf[ks][j][e] =
                            h < G ? *reinterpret_cast<const uint32_t *>(q + h * QDB_HD + ks * 16 + e * 8 + qc * 2) : 0u;
                m[j][0] = m[j][1] = -INFINITY;
                l[j][0] = l[j][1] = 0.f;
#pragma unroll
                for (int mt = 0; mt < 8; mt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[mt][j][e] = 0.f;
            }
        }
        const int s = i % NS;
        alive = bar_wait(full0 + 8 * s, (i / NS) & 1, a.bt.err);
        if (__any_sync(0xffffffffu, !alive)) {
            alive = false;
            break;
        }
        used = i + 1;
        const uint32_t kt = ring_u + s * 2 * TILE_B, vt = kt + TILE_B;
        float sc[NT][2][4];
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) sc[j][0][e] = sc[j][1][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 8; ks++) {
            uint32_t f[4];
            const uint32_t ch = ks * 2 + kch;
            ldsm4(f, kt + (ch >> 3) * 2048 + krow * 128 + (((ch & 7) ^ (krow & 7)) << 4));
#pragma unroll
            for (int j = 0; j < NT; j++) mma16<T>(sc[j][ks & 1], f, qf[ks][j][0], qf[ks][j][1]);
        }
        const int left = cc.len - cc.tile * TILE;  // valid keys of this tile
        if (left < TILE) {
            // values behind the end are whatever the page held: clear them
            for (int x = left * 16 + lane; x < TILE * 16; x += 32) {
                const int r = x >> 4, ch = x & 15;
                *reinterpret_cast<uint4 *>(ring + s * 2 * TILE_B + TILE_B + (ch >> 3) * 2048 + r * 128 +
                                           ((ch & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_async();
            __syncwarp();
        }
        uint32_t p[NT][2];
#pragma unroll
        for (int j = 0; j < NT; j++) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] = (sc[j][0][e] + sc[j][1][e]) * c;
                if (left < TILE && qr + (e >> 1) * 8 >= left) v[e] = -INFINITY;
            }
            float x0m = fmaxf(v[0], v[2]), x1m = fmaxf(v[1], v[3]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                x0m = fmaxf(x0m, __shfl_xor_sync(0xffffffffu, x0m, d));
                x1m = fmaxf(x1m, __shfl_xor_sync(0xffffffffu, x1m, d));
            }
            const bool up = x0m > m[j][0] || x1m > m[j][1];
            if (__any_sync(0xffffffffu, up)) {  // a maximum moved: rescale sum and output
                const float n0 = fmaxf(m[j][0], x0m), n1 = fmaxf(m[j][1], x1m);
                const float f0 = m[j][0] == n0 ? 1.f : ex2(m[j][0] - n0), f1 = m[j][1] == n1 ? 1.f : ex2(m[j][1] - n1);
                m[j][0] = n0;
                m[j][1] = n1;
                l[j][0] *= f0;
                l[j][1] *= f1;
#pragma unroll
                for (int mt = 0; mt < 8; mt++) {
                    o[mt][j][0] *= f0;
                    o[mt][j][1] *= f1;
                    o[mt][j][2] *= f0;
                    o[mt][j][3] *= f1;
                }
            }
            const float a0 = m[j][0] == -INFINITY ? 0.f : m[j][0] - P_SHIFT, a1 = m[j][1] == -INFINITY ? 0.f : m[j][1] - P_SHIFT;
            v[0] = ex2(v[0] - a0);
            v[1] = ex2(v[1] - a1);
            v[2] = ex2(v[2] - a0);
            v[3] = ex2(v[3] - a1);
            l[j][0] += v[0] + v[2];
            l[j][1] += v[1] + v[3];
            p[j][0] = transpose8(T::pack(v[0], v[1]));
            p[j][1] = transpose8(T::pack(v[2], v[3]));
        }
#pragma unroll
        for (int mt = 0; mt < 8; mt++) {
            uint32_t f[4];
            const uint32_t ch = mt * 2 + vch;
            ldsm4t(f, vt + (ch >> 3) * 2048 + vrow * 128 + (((ch & 7) ^ (vrow & 7)) << 4));
#pragma unroll
            for (int j = 0; j < NT; j++) mma16<T>(o[mt][j], f, p[j][0], p[j][1]);
        }
        __syncwarp();  // every lane has read the tile
        if (lane == 0 && issued < count) {
            issue(s, pc, next_page);
            advance(pc);
            if (++issued < count) next_page = page_of(pc);
        }
        // ---- the pair's last tile, or the range's
        const bool ends = cc.tile + 1 == cc.nt;
        if (ends || i + 1 == count) {
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], d);
            const bool begins = pair_lo >= x0;
            if (begins && ends) {  // the whole pair: its output rows
                uint16_t *dst = a.out + (size_t)cc.b * a.out_stride + (size_t)cc.g * G * QDB_HD;
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int h = j * 8 + qc * 2 + e;
                        if (h >= G) continue;
                        const float inv = l[j][e] > 0.f ? 1.0f / l[j][e] : (isnan(l[j][e]) ? l[j][e] : 0.f);
#pragma unroll
                        for (int mt = 0; mt < 8; mt++) {
                            dst[h * QDB_HD + mt * 16 + qr] = T::one(o[mt][j][e] * inv);
                            dst[h * QDB_HD + mt * 16 + 8 + qr] = T::one(o[mt][j][e + 2] * inv);
                        }
                    }
            } else {
                // a part: one that began earlier goes to head_part, the range's
                // last one (all tiles used by now) into the ring
                float *dst = begins ? reinterpret_cast<float *>(ring) : &sm.head_part[warp][0][0];
                if (begins) has_last = true;
                else has_head = true;
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int h = j * 8 + qc * 2 + e;
#pragma unroll
                        for (int mt = 0; mt < 8; mt++) {
                            dst[h * QDB_HD + mt * 16 + qr] = o[mt][j][e];
                            dst[h * QDB_HD + mt * 16 + 8 + qr] = o[mt][j][e + 2];
                        }
                        if (qr == 0) sm.ml[warp][begins ? 1 : 0][h] = make_float2(m[j][e] - P_SHIFT, l[j][e]);
                    }
            }
        }
        if (ends) pair_lo += cc.nt;
        if (i + 1 < count) advance(cc);
    }
    // a wait that ran out: the copies in flight land before the CTA goes on
    if (!alive && lane == 0)
        for (int i = used; i < issued; i++) bar_wait(full0 + 8 * (i % NS), (i / NS) & 1, a.bt.err);
    __syncthreads();

    // ---- join. The pair list positions of this warp's first and last pair
    // decide who joins: warp w the pair that begins in it and goes on behind
    // it, warp 0 also the one that came from an earlier CTA.
    const long long cta_lo = first_of(gw0), cta_hi = first_of(gw0 + DW);
    for (int turn = 0; turn < 2; turn++) {
        // turn 0: parts that began in an earlier CTA (warp 0's head part);
        // turn 1: pairs that begin in this warp's range and go on behind it
        Whole whole{false, 0, 0, 0, 0};
        const bool act = turn == 0 ? (warp == 0 && has_head) : has_last;
        int pb = 0, pg = 0, pnt = 0;
        long long lo = 0;
        if (act) {
            if (turn == 0) {
                pb = sm.start[0][0];
                pg = sm.start[0][1];
                lo = x0 - sm.start[0][2];
            } else {
                pb = cc.b;
                pg = cc.g;
                lo = x1 - 1 - cc.tile;
            }
            pnt = (length(pb) + TILE - 1) / TILE;
            const long long hi = lo + pnt;
            const long long last_w = warp_of(min(hi, cta_hi) - 1) - gw0;  // last warp of this CTA with a part
            const bool inside = lo >= cta_lo && hi <= cta_hi;
            const int c0 = (int)(warp_of(lo) / DW), c1 = (int)(warp_of(hi - 1) / DW);
            for (int h = 0; h < G; h++) {
                Join j;
                const float *src = turn ? reinterpret_cast<const float *>(ring) : &sm.head_part[0][0][0];
                j.add(sm.ml[warp][turn][h], *reinterpret_cast<const float4 *>(src + h * QDB_HD + lane * 4));
                for (int w = warp + 1; w <= (int)last_w; w++) {
                    if (first_of(gw0 + w) == first_of(gw0 + w + 1)) continue;  // an empty range
                    j.add(sm.ml[w][0][h], *reinterpret_cast<const float4 *>(&sm.head_part[w][h][lane * 4]));
                }
                if (inside) {
                    store_row4<T>(a.out + (size_t)pb * a.out_stride + ((size_t)pg * G + h) * QDB_HD + lane * 4, j);
                } else {
                    float *g = ws.part + ((size_t)(blockIdx.x * 2 + turn) * MAX_G + h) * 130;
                    *reinterpret_cast<float2 *>(g + lane * 4) = make_float2(j.o[0], j.o[1]);
                    *reinterpret_cast<float2 *>(g + lane * 4 + 2) = make_float2(j.o[2], j.o[3]);
                    if (lane == 0) *reinterpret_cast<float2 *>(g + QDB_HD) = make_float2(j.m, j.l);
                }
            }
            if (!inside) {
                __threadfence();
                __syncwarp();
                unsigned seen = 0;
                if (lane == 0) seen = atomicAdd(&ws.cnt[c0], 1u);
                seen = __shfl_sync(0xffffffffu, seen, 0);
                if (seen == (unsigned)(c1 - c0)) {  // the last of its parts
                    __threadfence();
                    whole = Whole{true, pb, pg, c0, c1 - c0 + 1};
                }
            }
        }
        // at most one warp has a pair to finish in each turn: the whole CTA does it
        if (t == 0) sm.todo.some = false;
        __syncthreads();
        if (whole.some && lane == 0) sm.todo = whole;
        __syncthreads();
        if (sm.todo.some) {
            const Whole wd = sm.todo;
            // warp: head warp % G and every pgc-th part, or heads warp, warp + 8, ...
            const int pgc = G <= DW ? DW / G : 1;
            float *sp = reinterpret_cast<float *>(&sm.ring[0][0][0][0] + 8192);  // free by now: [pgc][G][132]
            for (int h = G <= DW ? warp % G : warp; h < G; h += DW) {
                const int pg = G <= DW ? warp / G : 0;
                Join j;
                if (pg < pgc)
#pragma unroll 4
                    for (int i = pg; i < wd.parts; i += pgc) {
                        const float *g = ws.part + ((size_t)((wd.c0 + i) * 2 + (i == 0 ? 1 : 0)) * MAX_G + h) * 130;
                        const float2 x = __ldcg(reinterpret_cast<const float2 *>(g + lane * 4));
                        const float2 y = __ldcg(reinterpret_cast<const float2 *>(g + lane * 4 + 2));
                        j.add(__ldcg(reinterpret_cast<const float2 *>(g + QDB_HD)), make_float4(x.x, x.y, y.x, y.y));
                    }
                uint16_t *dst = a.out + (size_t)wd.b * a.out_stride + ((size_t)wd.g * G + h) * QDB_HD + lane * 4;
                if (pgc == 1) {
                    store_row4<T>(dst, j);
                } else if (pg < pgc) {
                    float *x = sp + (pg * G + h) * 132;
                    *reinterpret_cast<float4 *>(x + lane * 4) = make_float4(j.o[0], j.o[1], j.o[2], j.o[3]);
                    if (lane == 0) *reinterpret_cast<float2 *>(x + QDB_HD) = make_float2(j.m, j.l);
                }
            }
            if (pgc > 1) {
                __syncthreads();
                if (warp < G) {
                    Join j;
                    for (int i = 0; i < pgc; i++) {
                        const float *x = sp + (i * G + warp) * 132;
                        j.add(*reinterpret_cast<const float2 *>(x + QDB_HD), *reinterpret_cast<const float4 *>(x + lane * 4));
                    }
                    store_row4<T>(a.out + (size_t)wd.b * a.out_stride + ((size_t)wd.g * G + warp) * QDB_HD + lane * 4, j);
                }
            }
            if (t == 0) ws.cnt[wd.c0] = 0;
        }
        __syncthreads();
    }
}

template <typename T, int NT>
cudaError_t launch(const CUtensorMap &mk, const CUtensorMap &mv, const QdbPagedAttnArgs &a, const QdbDecodeScratch &ws,
                   cudaStream_t st) {
    const size_t smem = sizeof(DecodeSmem<NT>) + 1024;
    cudaError_t e = cudaFuncSetAttribute(decode_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    return pdl_launch(decode_kernel<T, NT>, dim3(ws.ctas), dim3(DW * 32), smem, st, mk, mv, a, ws);
}

}  // namespace

cudaError_t qdb_launch_paged_decode(const QdbPagedAttnArgs &a, int type, const QdbDecodeScratch &ws, cudaStream_t st) {
    CUtensorMap mk, mv;
    if (qdb_paged_map(&mk, a.kv.k, a.kv, type, TILE) || qdb_paged_map(&mv, a.kv.v, a.kv, type, TILE))
        return cudaErrorInvalidValue;
    const bool narrow = a.heads / a.kv.kv_heads <= 8;
    if (type == QDB_TYPE_F16)
        return narrow ? launch<QdbHalf, 1>(mk, mv, a, ws, st) : launch<QdbHalf, 2>(mk, mv, a, ws, st);
    return narrow ? launch<QdbBf16, 1>(mk, mv, a, ws, st) : launch<QdbBf16, 2>(mk, mv, a, ws, st);
}
