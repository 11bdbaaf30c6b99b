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
//   P = 2^(S c - m)  (c = scale log2 e), rounded to the cache's type (error against
//                     64 bits 1.25 times that of f32 arithmetic; as a pair of the
//                     type 1.00 times, but one short history 8.6 -> 8.8 us, 64 of
//                     them 30.6 -> 31.4)
//   O^T += V^T P^T   (dims x heads: V as the row operand, transposed ldmatrix;
//                     P^T by movmatrix from the S^T fragment)
// A pair that lies in several warps' ranges leaves partial (m, l, O); the
// CTA's parts are joined in shared memory, and where it spans CTAs the last
// one to arrive joins them, always in the order of the list, so the result
// does not depend on timing.
//
// Measured (L2 cold): 256 ragged sequences of 1 to 1500 tokens, 16 heads on 8
// key heads, bf16, 146 us, and 8 of 24000 to 32768, 32 heads on 4, 81 us: 90 %
// and 85 % of the copy bandwidth for their K and V bytes. 64 sequences of 404
// to 660, f16, 31 us against 21 for the bytes; one of 404 8.6 us against 0.3:
// the fixed chain of launch, lengths, page numbers, first tiles and the join
// over CTAs. A first version, one warp per (row, query head) with scalar
// products, took 734 us for the 256, 11.5 ms, 344 and 91 us.
#include <math.h>

#include <type_traits>

#include "qdb_kernels.h"
#include "qdb_paged.cuh"

namespace {

constexpr int DW = 8;             // warps per CTA
constexpr int TILE = 16;          // keys per tile (a page holds whole tiles)
constexpr int TILE_B = 4096;      // bytes of a tile's K (or V)
constexpr int MAX_G = 16;         // query heads per key head
// Tiles of a CTA, on average, below which a pair is not cut further. One sequence of
// 200 keys of 8 key heads: 8.1 us at 2 and 4, 9.5 at 8; four of 404: 8.8 at 2 and 4,
// 9.6 at 8; one of 1000 or 4000: the same at all three.
constexpr int MIN_TILES = 4;
// Tiles of a CTA from which the pairs' borders do not matter: 8 sequences of 24000
// to 32768 with 4 key heads 83 us on 128 CTAs, 80.8 on all 148; 20 of 20000 to 30000
// with 2 97.5 on 120, 90.9 on all; one of 100000 with 8 73 and 71.8.
constexpr int MANY_TILES = 128;
constexpr float P_SHIFT = 8.0f;   // P is scaled by 2^8: f16 keeps weights down to 2^-32 of the largest

// Ring stages per warp: what shared memory leaves beside one partial per warp.
__host__ __device__ constexpr int ring_stages(int nt) { return nt == 1 ? 3 : 2; }

// A pair with parts in this CTA: those of warps w0 (its last part, or where the
// pair came from an earlier CTA its head part) to w1 (head parts), and the CTAs
// c0 .. c1 that the pair lies in.
struct Group {
    int some, b, g, w0, w1, c0, c1;
};

template <int NT>
struct DecodeSmem {
    static constexpr int NS = ring_stages(NT), H = 8 * NT;
    unsigned char ring[DW][NS][2][TILE_B];
    union {
        float head_part[DW][H][QDB_HD];  // the part of a pair that began in an earlier warp
        struct {  // until the warps have found their first tiles
            int before[DW * 32];  // tiles of one key head ahead of each thread's share of the sequences
            int len0[DW * 32];    // length of the share's first sequence
        } find;
    };
    float2 ml[DW][2][H];             // (m, l) of the head part and of the last part
    unsigned long long full[DW][NS];
    int scan[DW];
    int start[4];                    // warp 0's first tile: sequence, key head, tile; the sequence's length
    Group grp[DW + 1];               // 0: came from an earlier CTA; 1 + w: begins in warp w and goes on
    int todo[2];                     // groups whose last part arrived here (-1: none)
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

// Joins parts 0 .. n-1 of one head, in their order: ml(i) = (m, l), row(i) = this
// lane's 4 dims; the weights are 2^(m_i - max).
struct Joined {
    float m, l, o[4];
    __device__ __forceinline__ void add(const float4 &x, float w) {
        o[0] = fmaf(x.x, w, o[0]);
        o[1] = fmaf(x.y, w, o[1]);
        o[2] = fmaf(x.z, w, o[2]);
        o[3] = fmaf(x.w, w, o[3]);
    }
};
__device__ __forceinline__ float part_weight(float m, float top) { return m == top ? 1.f : exp2f(m - top); }  // (also of -inf)
// Up to FEW parts: all loads at once, every lane weighs them all (64 sequences 32.4
// -> 30.6 us, one 9.1 -> 8.1 against reductions over the warp).
constexpr int FEW = DW;  // (the parts within a CTA)
template <typename ML, typename Row>
__device__ __forceinline__ Joined join_few(int n, ML ml, Row row) {
    float2 x[FEW];
    float4 r[FEW];
#pragma unroll
    for (int i = 0; i < FEW; i++) {
        x[i] = i < n ? ml(i) : make_float2(-INFINITY, 0.f);
        r[i] = i < n ? row(i) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    Joined j{x[0].x, 0.f, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i = 1; i < FEW; i++) j.m = fmaxf(j.m, x[i].x);
#pragma unroll
    for (int i = 0; i < FEW; i++) {
        if (i >= n) break;
        const float w = part_weight(x[i].x, j.m);
        j.l += x[i].y * w;
        j.add(r[i], w);
    }
    return j;
}
// Any number: the weights are computed one part per lane.
template <typename ML, typename Row>
__device__ __forceinline__ Joined join(int n, int lane, ML ml, Row row) {
    if (n <= FEW) return join_few(n, ml, row);
    Joined j{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
    for (int i = lane; i < n; i += 32) j.m = fmaxf(j.m, ml(i).x);
    j.m = warp_max(j.m);
    for (int i0 = 0; i0 < n; i0 += 32) {
        float w = 0.f, l = 0.f;
        if (i0 + lane < n) {
            const float2 x = ml(i0 + lane);
            w = part_weight(x.x, j.m);
            l = x.y * w;
        }
        j.l += warp_sum(l);
        const int k = min(32, n - i0);
#pragma unroll 8
        for (int i = 0; i < k; i++) j.add(row(i0 + i), __shfl_sync(0xffffffffu, w, i));
    }
    return j;
}

template <typename T, bool PAIR>
__device__ __forceinline__ void store_row4(const QdbPagedAttnArgs &a, size_t at, const Joined &j) {
    const float inv = j.l > 0.f ? 1.0f / j.l : (isnan(j.l) ? j.l : 0.f);
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = j.o[e] * inv;
    if constexpr (PAIR) {
        for (int p = 0; p < 2; p++)
            *reinterpret_cast<uint2 *>((p ? a.lo : a.out) + at) =
                make_uint2(QdbBf16::plain(pair_part(v[0], p), pair_part(v[1], p)),
                           QdbBf16::plain(pair_part(v[2], p), pair_part(v[3], p)));
    } else {
        *reinterpret_cast<uint2 *>(a.out + at) = make_uint2(T::plain(v[0], v[1]), T::plain(v[2], v[3]));
    }
}

template <typename T, int NT, bool PAIR>  // PAIR: the output as a bf16 pair (a.out, a.lo)
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
    if (t == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
    }
    pdl_enter();
    const int step = a.bt.step ? *a.bt.step : 0;
    auto length = [&](int b) { return paged_len(a.bt, b, a.kv.page_shift, step); };

    // ---- the list: tiles ahead of each thread's share of the sequences (the
    // host has checked that every count fits 31 bits)
    const int per = (n + DW * 32 - 1) / (DW * 32), b0 = min(n, t * per), b1 = min(n, b0 + per);
    int mine = 0;
    for (int b = b0; b < b1; b++) {
        const int len = length(b);
        if (b == b0) sm.find.len0[t] = len;
        mine += (len + TILE - 1) / TILE;
        if (len == 0 && b % gridDim.x == blockIdx.x)  // the row of an empty sequence is zero
            for (int i = 0; i < a.heads * QDB_HD / 8; i++) {
                *reinterpret_cast<uint4 *>(a.out + (size_t)b * a.out_stride + i * 8) = make_uint4(0u, 0u, 0u, 0u);
                if (PAIR) *reinterpret_cast<uint4 *>(a.lo + (size_t)b * a.out_stride + i * 8) = make_uint4(0u, 0u, 0u, 0u);
            }
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) sm.scan[warp] = upto;
    if (t <= DW) sm.grp[t].some = 0;
    if (t < 2) sm.todo[t] = -1;
    __syncthreads();
    int total = 0, before = upto - mine;
#pragma unroll
    for (int w = 0; w < DW; w++) {
        const int x = sm.scan[w];
        if (w < warp) before += x;
        total += x;
    }
    sm.find.before[t] = before;
    total *= Hkv;
    if (total == 0) return;
    // CTAs that take part: all of them where there are more pairs than CTAs, or
    // MANY_TILES for each; else a whole number per pair (equal lengths then need no
    // join beyond the pair's own), each with at least MIN_TILES tiles on average, and
    // no more than sqrt(16 tiles / G), at which the joining CTA reads as many bytes
    // of parts as each CTA has read of K and V (one history of 32000 with 16 heads
    // on one key head: 39.2 us with all 148 CTAs, 27.2 with these 44); never so many
    // that a warp would have no tile (a range is empty only where one CTA does it all)
    int ctas = ws.ctas;
    if ((long long)n * Hkv <= ctas) {
        const int np = n * Hkv;
        const int most = (int)sqrtf(16.f * (float)(total / np) / (float)G);
        if (ctas / np > most || total / ctas < MANY_TILES)
            ctas = np * max(1, min(min(ctas / np, most), total / (np * MIN_TILES)));
    }
    ctas = min(ctas, max(total / DW, 1));
    if ((int)blockIdx.x >= ctas) return;
    // warp w of the whole grid begins at tile first_of(w): share + 1 tiles for
    // each of the first `more` warps, share for the rest
    const int nw = ctas * DW, share = total / nw, more = total - share * nw;
    auto first_of = [&](int w) { return share * w + min(w, more); };
    auto cta_of = [&](int x) {  // the CTA whose range holds tile x
        const int y = more * (share + 1);
        return (x < y ? x / (share + 1) : more + (x - y) / share) / DW;
    };
    const int gw0 = blockIdx.x * DW, x0 = first_of(gw0 + warp), count = first_of(gw0 + warp + 1) - x0;
    __syncthreads();

    // ---- copies: lane 0 issues tile i + NS when tile i has been used
    Cursor pc{}, cc{};
    if (count > 0) {  // the warp's first tile: the last share that begins at or before it
        int i = 0;
#pragma unroll
        for (int d = DW * 16; d; d >>= 1)
            if (sm.find.before[i + d] * Hkv <= x0) i += d;
        int rel = x0 - sm.find.before[i] * Hkv, b = min(n, i * per), len = sm.find.len0[i], nt = (len + TILE - 1) / TILE;
        while (rel >= nt * Hkv) {
            rel -= nt * Hkv;
            len = length(++b);
            nt = (len + TILE - 1) / TILE;
        }
        pc = Cursor{b, rel / nt, rel % nt, nt, len};
        cc = pc;
        if (t == 0) {
            sm.start[0] = pc.b;
            sm.start[1] = pc.g;
            sm.start[2] = pc.tile;
            sm.start[3] = pc.len;
        }
    }
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
        // the first NS tiles' pages, and the one after them, are looked up side by side
        int page = 0;
        if (lane <= NS && lane < count) {
            for (int i = 0; i < lane; i++) advance(pc);
            page = page_of(pc);
            if (lane < NS) issue(lane, pc, page);
        }
        issued = min(NS, count);
        const int from = min(NS, count - 1);  // the cursor that goes on: tile NS
        pc.b = __shfl_sync(0xffffffffu, pc.b, from);
        pc.g = __shfl_sync(0xffffffffu, pc.g, from);
        pc.tile = __shfl_sync(0xffffffffu, pc.tile, from);
        pc.nt = __shfl_sync(0xffffffffu, pc.nt, from);
        pc.len = __shfl_sync(0xffffffffu, pc.len, from);
        next_page = __shfl_sync(0xffffffffu, page, from);
    }
    __syncthreads();  // (`find` makes room for head_part)

    // ---- compute
    const float c = a.scale * 1.4426950408889634f;
    const int qr = lane >> 2, qc = lane & 3;  // fragment row and column pair
    float o[8][NT][4], m[NT][2], l[NT][2];
    uint32_t qf[8][NT][2];
    bool alive = true;
    int used = 0;
    bool has_head = false, has_last = false;  // partial results left in shared memory
    int pair_lo = x0 - (count > 0 ? cc.tile : 0);  // list position of the current pair's first tile
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
        alive = bar_wait(full0 + 8 * s, (i / NS) & 1, a.bt.err, qdb_wait_limit_c);
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
            p[j][0] = transpose8(T::plain(v[0], v[1]));
            p[j][1] = transpose8(T::plain(v[2], v[3]));
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
                const size_t at = (size_t)cc.b * a.out_stride + (size_t)cc.g * G * QDB_HD;
                auto put = [&](size_t i, float v) {
                    if (!PAIR) {
                        a.out[at + i] = T::plain1(v);
                    } else {
                        a.out[at + i] = QdbBf16::plain1(v);
                        a.lo[at + i] = QdbBf16::plain1(pair_part(v, true));
                    }
                };
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int h = j * 8 + qc * 2 + e;
                        if (h >= G) continue;
                        const float inv = l[j][e] > 0.f ? 1.0f / l[j][e] : (isnan(l[j][e]) ? l[j][e] : 0.f);
#pragma unroll
                        for (int mt = 0; mt < 8; mt++) {
                            put(h * QDB_HD + mt * 16 + qr, o[mt][j][e] * inv);
                            put(h * QDB_HD + mt * 16 + 8 + qr, o[mt][j][e + 2] * inv);
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

    // ---- join: first the parts of this CTA, head by head over all warps
    if (lane == 0 && ((warp == 0 && has_head) || has_last)) {
        const int begin = first_of(gw0), end = first_of(gw0 + DW);
        auto put = [&](Group &gr, int b, int g, int w0, int lo, int len) {
            const int hi = lo + (len + TILE - 1) / TILE;
            int w1 = w0;
            while (w1 + 1 < DW && first_of(gw0 + w1 + 1) < hi) w1++;
            gr = Group{1, b, g, w0, w1, lo < begin ? cta_of(lo) : (int)blockIdx.x, hi > end ? cta_of(hi - 1) : (int)blockIdx.x};
        };
        if (warp == 0 && has_head) put(sm.grp[0], sm.start[0], sm.start[1], 0, x0 - sm.start[2], sm.start[3]);
        if (has_last) put(sm.grp[1 + warp], cc.b, cc.g, warp, x0 + count - 1 - cc.tile, cc.len);
    }
    __syncthreads();
    auto out_row = [&](const Group &gr, int h) {
        return (size_t)gr.b * a.out_stride + ((size_t)gr.g * G + h) * QDB_HD + lane * 4;
    };
    const unsigned groups = __ballot_sync(0xffffffffu, lane <= DW && sm.grp[lane <= DW ? lane : 0].some);
    const bool split = __any_sync(0xffffffffu, (groups >> lane & 1) && sm.grp[lane].c0 != sm.grp[lane].c1);
    int item = 0;
    for (unsigned left = groups; left; left &= left - 1) {
        const int k = __ffs(left) - 1;
        for (int h = 0; h < G; h++, item++) {
            if (item % DW != warp) continue;
            const Group gr = sm.grp[k];
            const Joined j = join_few(
                gr.w1 - gr.w0 + 1,
                [&](int i) { return sm.ml[gr.w0 + i][i == 0 && k ? 1 : 0][h]; },
                [&](int i) {
                    const float *src = i == 0 && k ? reinterpret_cast<const float *>(&sm.ring[gr.w0][0][0][0])
                                                   : &sm.head_part[gr.w0 + i][0][0];
                    return *reinterpret_cast<const float4 *>(src + h * QDB_HD + lane * 4);
                });
            if (gr.c0 == gr.c1) {
                store_row4<T, PAIR>(a, out_row(gr, h), j);
            } else {
                const size_t at = (size_t)(blockIdx.x * 2 + (k ? 1 : 0)) * MAX_G + h;
                *reinterpret_cast<float4 *>(ws.part + at * QDB_HD + lane * 4) = make_float4(j.o[0], j.o[1], j.o[2], j.o[3]);
                if (lane == 0) ws.ml[at] = make_float2(j.m, j.l);
            }
        }
    }
    if (!split) return;
    // ---- pairs over several CTAs (at most the first and the last of this one):
    // the CTA whose part arrives last joins them
    __syncthreads();
    if (t <= DW && sm.grp[t].some && sm.grp[t].c0 != sm.grp[t].c1) {
        const Group gr = sm.grp[t];
        unsigned before;  // (releases this CTA's parts, acquires the others')
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(ws.cnt + gr.c0) : "memory");
        if (before == (unsigned)(gr.c1 - gr.c0)) {
            sm.todo[t ? 1 : 0] = t;
            ws.cnt[gr.c0] = 0;  // nobody else comes
        }
    }
    __syncthreads();
    item = 0;
    for (int k = 0; k < 2; k++) {
        if (sm.todo[k] < 0) continue;
        const Group gr = sm.grp[sm.todo[k]];
        for (int h = 0; h < G; h++, item++) {
            if (item % DW != warp) continue;
            auto at = [&](int i) { return (size_t)((gr.c0 + i) * 2 + (i == 0 ? 1 : 0)) * MAX_G + h; };
            const Joined j = join(
                gr.c1 - gr.c0 + 1, lane, [&](int i) { return __ldcg(ws.ml + at(i)); },
                [&](int i) { return __ldcg(reinterpret_cast<const float4 *>(ws.part + at(i) * QDB_HD + lane * 4)); });
            store_row4<T, PAIR>(a, out_row(gr, h), j);
        }
    }
}

template <typename T, int NT, bool PAIR>
cudaError_t launch(const CUtensorMap &mk, const CUtensorMap &mv, const QdbPagedAttnArgs &a, const QdbDecodeScratch &ws,
                   cudaStream_t st) {
    const size_t smem = sizeof(DecodeSmem<NT>) + 1024;
    cudaError_t e = cudaFuncSetAttribute(decode_kernel<T, NT, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    return pdl_launch(decode_kernel<T, NT, PAIR>, dim3(ws.ctas), dim3(DW * 32), smem, st, mk, mv, a, ws);
}

}  // namespace

QDB_WAIT_LIMIT_SETTER(qdb_set_wait_limit_paged_decode)

cudaError_t qdb_launch_paged_decode(const QdbPagedAttnArgs &a, int type, const QdbDecodeScratch &ws, cudaStream_t st) {
    CUtensorMap mk, mv;
    if (qdb_paged_map(&mk, a.kv.k, a.kv, type, TILE, 2) || qdb_paged_map(&mv, a.kv.v, a.kv, type, TILE, 2))
        return cudaErrorInvalidValue;
    auto go = [&](auto pair) {
        constexpr bool P = decltype(pair)::value;
        const bool narrow = a.heads / a.kv.kv_heads <= 8;
        if (type == QDB_TYPE_F16)
            return narrow ? launch<QdbHalf, 1, P>(mk, mv, a, ws, st) : launch<QdbHalf, 2, P>(mk, mv, a, ws, st);
        return narrow ? launch<QdbBf16, 1, P>(mk, mv, a, ws, st) : launch<QdbBf16, 2, P>(mk, mv, a, ws, st);
    };
    return a.lo ? go(std::true_type()) : go(std::false_type());
}
