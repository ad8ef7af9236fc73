// A decode step whose slots share the first P positions and bring several new tokens each (drafts): rotation and append of
// the new rows, attention over the shared rows and the slot's own.  bf16, head dimension 64.
//
//   t = pos[b] + i is the position of token i of slot b; positions below P are rows of Kp, Vp (one copy for all slots), position
//   P + j is row j of the slot's cache.
#include <cuda.h>
#include <cuda_bf16.h>
#include <math.h>
#include <string.h>
#include "qlmb_common.cuh"
#include "qlmb_gemm.cuh"
#include "qlmb_attn.cuh"

namespace qlmb {

constexpr int PX_HD = 64;

// ------------------------------------------------------------------ rotation and append
// Four threads a head and row, each the dimensions 8 u .. 8 u + 7 and their partners 32 further: one head of q or k is rotated, one
// of v copied.  Bound by the launch at a few rows (2 KB a row and head group), by HBM beyond.
__global__ void __launch_bounds__(256) k_dec_rope_kv(bf16 *Qo, bf16 *Kc, bf16 *Vc, const bf16 *q, const bf16 *k, const bf16 *v, const float *cosb,
                                                     const float *sinb, const int *pos, int B, int n, int P, int Tm, int H, int KV, int Tr, int *errword)
{
    pdl_trigger();
    pdl_wait();
    const int heads = H + 2 * KV;
    const size_t g = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (g >= (size_t)B * n * heads * 4) return;
    const int u = (int)(g & 3);
    const size_t rh = g >> 2, row = rh / heads;
    const int hh = (int)(rh % heads), b = (int)(row / n), i = (int)(row % n);
    const long long t0 = pos[b], j0 = t0 - P;                          // the slot's first new token, its row of the cache
    if (j0 < 0 || j0 + n > Tm || t0 + n > Tr) {                        // a slot past its cache or the tables: left as it is
        if (u == 0 && hh == 0 && i == 0) report_bad_index(errword, 305, b, pos[b]);
        return;
    }
    const bf16 *src;
    bf16 *dst;
    const int KD = KV * PX_HD;
    const size_t crow = ((size_t)b * Tm + (size_t)(j0 + i)) * KD;
    if (hh < H) { const size_t o = (row * H + hh) * PX_HD; src = q + o; dst = Qo + o; }
    else if (hh < H + KV) { const int kh = hh - H; src = k + row * KD + kh * PX_HD; dst = Kc + crow + kh * PX_HD; }
    else { const int kh = hh - H - KV; src = v + row * KD + kh * PX_HD; dst = Vc + crow + kh * PX_HD; }
    src += 8 * u; dst += 8 * u;
    uint4 lo = *reinterpret_cast<const uint4 *>(src), hi = *reinterpret_cast<const uint4 *>(src + 32);
    if (hh < H + KV) {
        const float *cp = cosb + (size_t)(t0 + i) * 32 + 8 * u, *sp = sinb + (size_t)(t0 + i) * 32 + 8 * u;
        uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, c[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float2 cs = *reinterpret_cast<const float2 *>(cp + 2 * w), sn = *reinterpret_cast<const float2 *>(sp + 2 * w);
            const float x0 = __uint_as_float(a[w] << 16), x1 = __uint_as_float(a[w] & 0xffff0000u);
            const float y0 = __uint_as_float(c[w] << 16), y1 = __uint_as_float(c[w] & 0xffff0000u);
            const __nv_bfloat162 l2 = __floats2bfloat162_rn(x0 * cs.x - y0 * sn.x, x1 * cs.y - y1 * sn.y);
            const __nv_bfloat162 h2 = __floats2bfloat162_rn(y0 * cs.x + x0 * sn.x, y1 * cs.y + x1 * sn.y);
            a[w] = *reinterpret_cast<const uint32_t *>(&l2); c[w] = *reinterpret_cast<const uint32_t *>(&h2);
        }
        lo = make_uint4(a[0], a[1], a[2], a[3]); hi = make_uint4(c[0], c[1], c[2], c[3]);
    }
    *reinterpret_cast<uint4 *>(dst) = lo;
    *reinterpret_cast<uint4 *>(dst + 32) = hi;
}

// ------------------------------------------------------------------ attention
// Rows of queries of one kv head stand side by side in tiles of 16: the G = H / KV heads of a token, then the next token's.  An item
// is a tile and the keys its rows may see: a slot's own rows (tiles of the slot's n G rows), or the shared ones (tiles of all slots').
// Keys come in blocks of 32.  The blocks of all items, one after the other, are dealt out evenly to the warps of the device, a run
// each, whatever the slots' lengths: a warp goes through its run with a ring of asynchronous copies that does not stop at the
// items' borders, and leaves of each item that it meets a segment: output in fp32, normalised, and the logarithm (base 2) of its
// sum.  Segment number = item + warp, which no two share.  k_px_join adds the segments of a row up.
//
// Few slots and short prefixes take one launch of k_px_small instead.  Many blocks of shared keys go through k_px_tc, in pieces (128
// rows a tile, tcgen05), and only the slots' own through k_px_mma: see px_plan.
//
// Measured (12 heads, 12 kv heads unless stated; graph of calls, all launches): 1 slot after 512 keys 5.6 us, 8 slots of 4 tokens after
// 2048 10.9 us, 64 slots after 8192 31.8 us (101 MB, 3.2 TB/s), 64 slots of 5 tokens and 16 heads of 4 kv heads after 32768 91 us (96
// where k_px_mma waits for k_px_tc's end).  In the last k_px_tc has 75 us, 43 GFLOP at 573 TF/s: 168 M exponentials are 37 us of the
// special-function units; without them it takes 60 us, without any softmax 41 us, which is what its MMAs of 64 columns need.
constexpr int PX_WARPS = 12;                              // of a CTA, one CTA an SM: their rings fill its shared memory, and its registers
constexpr int PX_MAXB = 1024;                             // slots: every CTA keeps their positions and block counts
struct PxParams {
    alignas(64) CUtensorMap kc_map, vc_map, kp_map, vp_map;
    bf16 *O;
    float *lse;
    const bf16 *Q;
    const int *pos;
    float *seg_o, *seg_l;                     // [items + warps][16][64] and [items + warps][16]
    float *part_o, *part_l;                   // the shared keys' pieces of k_px_tc: [Sp][B*n*H][64] and [Sp][B*n*H]
    int *table;                               // for the join: blocks ahead of each slot's items [B + 1], then of a shared item, then a warp's
    int B, n, P, Tm, H, KV, G, win;
    int Sp, t_own, t_pre, warps, least;       // pieces of k_px_tc (0: the shared keys are items); tiles a (slot, kv head) / a kv head; blocks of a warp at least
    float scale_log2;                         // log2(e) / sqrt(64)
    int *errword;
};

__device__ __forceinline__ void px_mma(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A slot whose new tokens do not all lie in its cache (the first may see nothing of its own: pos = P - 1) is not touched.
__device__ __forceinline__ bool px_slot_ok(long long t0, int n, int P, int Tm) { return t0 - P >= -1 && t0 - P + n <= Tm; }
__device__ __forceinline__ bool px_nonfinite(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }

constexpr int PX_BLK = 32 * 128, PX_STAGE = 2 * PX_BLK;      // a block's keys; keys and values
constexpr int PX_Q = PX_WARPS * 2 * PX_STAGE, PX_RINGS = PX_Q + PX_WARPS * 16 * 128;      // two blocks a warp, then an item's queries a warp
static size_t px_smem(int B) { return (size_t)PX_RINGS + 256 + (size_t)(2 * B + 1) * sizeof(int); }
__device__ __forceinline__ void px_copy(uint32_t dst, const void *src, bool in)      // 16 bytes, zeros where !in
{ asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory"); }
__device__ __forceinline__ void px_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void px_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void px_ldm(uint32_t a, uint32_t v[4])
{ asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory"); }
__device__ __forceinline__ void px_ldmt(uint32_t a, uint32_t v[4])
{ asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory"); }

// The blocks of a slot's own keys: from its first visible one, in whole blocks, to the last new token's.
__device__ __forceinline__ int px_first(const PxParams &p, int t0) { return p.win > 0 ? max(0, t0 - p.win + 1 - p.P) & ~31 : 0; }
__device__ __forceinline__ int px_blocks(const PxParams &p, long long t0)
{
    if (!px_slot_ok(t0, p.n, p.P, p.Tm)) return 0;
    const int hi = (int)t0 + p.n - 1 - p.P;
    return hi < 0 ? 0 : (hi - px_first(p, (int)t0)) / 32 + 1;
}
// x / d for 0 <= x < 2^24: the quotient of the floats is off by one at most (a division of integers takes ten times as long)
__device__ __forceinline__ int px_div(int x, int d)
{
    int r = __float2int_rz(__fdividef((float)x, (float)d));
    const int left = x - r * d;
    return left < 0 ? r - 1 : left >= d ? r + 1 : r;
}
// 32 keys from kb on (the item's end at k1) and 16 rows: scores, the rows' running maxima (base 2) and sums, O.  A thread has rows g and g + 8,
// which see keys lo .. hi; every row of the tile sees alo .. ahi.
__device__ __forceinline__ void px_block(uint32_t sk, uint32_t sv, const uint32_t (&qa)[4][4], int kb, int k1, const int (&lo)[2], const int (&hi)[2], int alo, int ahi,
                                         float scale_log2, float (&m)[2], float (&l)[2], float (&oc)[8][4])
{
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    float s[4][4] = {};
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int h = 0; h < 2; h++) {                              // eight keys, dimensions 32 h .. 32 h + 31
            uint32_t w[4];
            px_ldm(sk + (8 * t + (lane & 7)) * 128 + (((4 * h + (lane >> 3)) ^ (lane & 7)) << 4), w);
            px_mma(s[t], qa[2 * h], w[0], w[1]);
            px_mma(s[t], qa[2 * h + 1], w[2], w[3]);
        }
    const bool edge = kb < alo || kb + 31 > ahi || kb + 32 > k1;   // some row does not see some key
    if (__builtin_expect(edge, 0)) {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int key = kb + 8 * t + 2 * q + (c & 1);
                if (key < lo[c >> 1] || key > hi[c >> 1] || key >= k1) s[t][c] = -INFINITY;
            }
    }
    float mn[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        float mx = fmaxf(fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1])),
                         fmaxf(fmaxf(s[2][2 * e], s[2][2 * e + 1]), fmaxf(s[3][2 * e], s[3][2 * e + 1])));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
        mn[e] = fmaxf(m[e], mx * scale_log2);
    }
    if (__any_sync(~0u, mn[0] > m[0] || mn[1] > m[1])) {            // a new maximum in some row
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float corr = ex2(m[e] - (mn[e] == -INFINITY ? 0.0f : mn[e]));
            m[e] = mn[e];
            l[e] *= corr;
#pragma unroll
            for (int j = 0; j < 8; j++) { oc[j][2 * e] *= corr; oc[j][2 * e + 1] *= corr; }
        }
    }
    uint32_t pa[2][4];                                             // weights in bf16, as every attention of the library has them
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const float mu = m[e] == -INFINITY ? 0.0f : m[e];          // nothing seen yet: every weight 0
        float sum[2] = {};
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const float p0 = ex2(fmaf(s[t][2 * e], scale_log2, -mu)), p1 = ex2(fmaf(s[t][2 * e + 1], scale_log2, -mu));
            sum[t & 1] += p0 + p1;
            const __nv_bfloat162 h2 = __floats2bfloat162_rn(p0, p1);
            pa[t >> 1][2 * (t & 1) + e] = *reinterpret_cast<const uint32_t *>(&h2);
        }
        l[e] += sum[0] + sum[1];
    }
    uint32_t vw[2][4][4];                                          // [16 keys][16 dimensions]: two pairs of operands
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) px_ldmt(sv + (16 * t + (lane & 15)) * 128 + (((2 * j + (lane >> 4)) ^ (lane & 7)) << 4), vw[t][j]);
    bool odd = false;                                              // an infinity or a NaN that some row must not see
    if (__builtin_expect(edge, 0)) {                               // keys behind the item's last are nobody's (a register holds keys 2 q and 2 q + 1 of eight)
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int key = kb + 16 * t + 8 * (k & 1) + 2 * q;
                const uint32_t in = (key < k1 ? 0xffffu : 0u) | (key + 1 < k1 ? 0xffff0000u : 0u);
#pragma unroll
                for (int j = 0; j < 4; j++) { vw[t][j][k] &= in; odd |= px_nonfinite(vw[t][j][k]); }
            }
    }
    if (__builtin_expect(!edge || !__any_sync(~0u, odd), 1)) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int j = 0; j < 4; j++) { px_mma(oc[2 * j], pa[t], vw[t][j][0], vw[t][j][1]); px_mma(oc[2 * j + 1], pa[t], vw[t][j][2], vw[t][j][3]); }
    } else {
        // 0 * inf is not 0: row by row, with the keys the row does not see taken as zeros
#pragma unroll 1
        for (int r = 0; r < 16; r++) {
            const int rlo = __shfl_sync(~0u, r < 8 ? lo[0] : lo[1], (r & 7) * 4), rhi = __shfl_sync(~0u, r < 8 ? hi[0] : hi[1], (r & 7) * 4);
#pragma unroll
            for (int t = 0; t < 2; t++) {
                uint32_t see[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int key = kb + 16 * t + 8 * h + 2 * q;
                    see[h] = (key >= rlo && key <= rhi && key < k1 ? 0xffffu : 0u) | (key + 1 >= rlo && key + 1 <= rhi && key + 1 < k1 ? 0xffff0000u : 0u);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    float c[4] = {};
                    px_mma(c, pa[t], vw[t][j >> 1][2 * (j & 1)] & see[0], vw[t][j >> 1][2 * (j & 1) + 1] & see[1]);
                    if (r == g) { oc[j][0] += c[0]; oc[j][1] += c[1]; }
                    if (r == g + 8) { oc[j][2] += c[2]; oc[j][3] += c[3]; }
                }
            }
        }
    }
}
// a place in the row of all blocks: item `sub` of slot b (b = B: of the shared keys), the block's first key, the item's last
struct PxCursor { int b, sub, key, last; };
__device__ __forceinline__ int px_ldcg(const int *p) { int v; asm volatile("ld.global.cg.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory"); return v; }

template <bool AHEAD> __global__ void __launch_bounds__(32 * PX_WARPS, 1) k_px_mma(const __grid_constant__ PxParams p)
{
    extern __shared__ __align__(1024) uint8_t px_s[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(px_s + PX_RINGS);                       // a ring's stages are full
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + 2 * PX_WARPS);
    int *plan = const_cast<int *>(abort_flag) + 1;                                        // first key and blocks of a shared item, blocks of a warp
    int *cum = reinterpret_cast<int *>(px_s + PX_RINGS + 256), *start = cum + p.B + 1;    // blocks of one item of each slot ahead of slot b; its first new position
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    if (smem_u32(px_s) & 1023u) {             // the swizzled blocks need a 1 KiB-aligned base
        if (tid == 0 && p.errword && atomicCAS(p.errword, 0, 201) == 0) { p.errword[1] = 130; p.errword[2] = (int)blockIdx.x; }
        pdl_wait();
        return;
    }
    if (tid == 0) {
        prefetch_map(&p.kc_map); prefetch_map(&p.vc_map);
        if (!p.Sp && p.P > 0) { prefetch_map(&p.kp_map); prefetch_map(&p.vp_map); }
        for (int i = 0; i < 2 * PX_WARPS; i++) mbar_init(smem_u32(&bars[i]), 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    pdl_trigger();
    // AHEAD: behind k_px_tc, which has waited before it let this kernel start and writes nothing that is read here, the wait comes last: SMs that
    // have no CTA of k_px_tc left begin with the slots' own keys.  (Reads pass by L1: copies, and the positions.)
    if (!AHEAD) pdl_wait();
    const int KT = p.KV * p.t_own;
    // ---- the slots' block counts, added up by the first warp
    if (warp == 0) {
        int carry = 0, first = 0x7fffffff;
        for (int b0 = 0; b0 < p.B; b0 += 32) {
            const int b = b0 + lane, t0 = b < p.B ? px_ldcg(p.pos + b) : 0, v = b < p.B ? px_blocks(p, t0) : 0;
            int x = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(~0u, x, o); if (lane >= o) x += y; }
            if (b < p.B) {
                start[b] = t0;
                cum[b] = carry + x - v;
                if (px_slot_ok(t0, p.n, p.P, p.Tm)) first = min(first, t0);
                else if (blockIdx.x == 0) report_bad_index(p.errword, 306, b, t0);
            }
            carry += __shfl_sync(~0u, x, 31);
        }
        first = __reduce_min_sync(~0u, first);
        if (lane == 0) {
            cum[p.B] = carry;
            // the shared keys that some row sees, the same for every item
            const int lo = p.win > 0 && first != 0x7fffffff ? max(0, first - p.win + 1) & ~31 : 0;
            const int n = p.Sp || lo >= p.P || first == 0x7fffffff ? 0 : (p.P - 1 - lo) / 32 + 1;
            const unsigned total = (unsigned)carry * KT + (unsigned)n * p.KV * p.t_pre;
            plan[0] = lo; plan[1] = n; plan[2] = (int)max((unsigned)p.least, (total + p.warps - 1) / p.warps);
        }
    }
    __syncthreads();
    const int rows_slot = p.n * p.G, lo_pre = plan[0], n_pre = plan[1];
    const unsigned own = (unsigned)cum[p.B] * KT, total = own + (unsigned)n_pre * p.KV * p.t_pre, per = plan[2];
    if (blockIdx.x == 0) {
        for (int b = tid; b <= p.B; b += 32 * PX_WARPS) p.table[b] = cum[b];
        if (tid == 0) { p.table[p.B + 1] = n_pre; p.table[p.B + 2] = (int)per; }
    }
    const unsigned me = blockIdx.x * PX_WARPS + warp;
    const unsigned from = me * per;                       // (the warps' number times per is little more than total: no overflow)
    if (from >= total) { if (AHEAD) pdl_wait(); return; }
    int count = (int)min(per, total - from);              // blocks of this warp
    // ---- the first of them
    const auto open = [&](PxCursor &c, int blk) {         // block blk of item (b, sub)
        if (c.b < p.B) { const int t0 = start[c.b]; c.key = px_first(p, t0) + 32 * blk; c.last = t0 + p.n - 1 - p.P; }
        else { c.key = lo_pre + 32 * blk; c.last = p.P - 1; }
    };
    PxCursor lc;
    {
        int blk;
        if (from < own) {
            int lo = 0, hi = p.B - 1;                     // the last slot that starts at or before it
            while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if ((unsigned)cum[mid] * KT <= from) lo = mid; else hi = mid - 1; }
            const unsigned off = from - (unsigned)cum[lo] * KT, nb = cum[lo + 1] - cum[lo];
            lc.b = lo; lc.sub = off / nb; blk = off % nb;
        } else { lc.b = p.B; lc.sub = (from - own) / n_pre; blk = (from - own) % n_pre; }
        open(lc, blk);
    }
    PxCursor cc = lc;
    // the next block; true where another item begins
    const auto step = [&](PxCursor &c) {
        c.key += 32;
        if (c.key <= c.last) return false;
        c.sub++;
        if (c.b < p.B && c.sub == KT) {
            c.sub = 0;
            do c.b++; while (c.b < p.B && cum[c.b + 1] == cum[c.b]);
        }
        open(c, 0);
        return true;
    };
    // row r of an item's tile: its place in O / 64 (-1: none) and its position
    const auto row_of = [&](int b, int sub, int r, int &t) {
        if (b < p.B) {
            const int kvh = px_div(sub, p.t_own), rr = (sub - kvh * p.t_own) * 16 + r, i = px_div(rr, p.G);
            t = start[b] + i;
            return rr < rows_slot ? (b * p.n + i) * p.H + kvh * p.G + rr - i * p.G : -1;
        }
        const int kvh = px_div(sub, p.t_pre), rr = (sub - kvh * p.t_pre) * 16 + r, token = px_div(rr, p.G), s = px_div(token, p.n);
        if (rr >= p.B * rows_slot || !px_slot_ok(start[s], p.n, p.P, p.Tm)) return -1;
        t = start[s] + token - s * p.n;
        return token * p.H + kvh * p.G + rr - token * p.G;
    };
    // ---- the ring; of an item's queries a lane has rows kr + 4 i, 16 bytes kc of the row
    const int kr = lane >> 3, kc = lane & 7;
    const uint32_t ring = smem_u32(px_s) + warp * (2 * PX_STAGE), sq = smem_u32(px_s) + PX_Q + warp * (16 * 128);
    const uint64_t *bar = bars + 2 * warp;
    int ls = 0, to_load = count;
    bool fresh = true;                                    // the block to be requested is the first of an item here
    int orow = -1, opos = 0;                              // of the item that was requested last: row lane % 16
    const auto load = [&]() {
        if (to_load > 0) {
            const bool mine = lc.b < p.B;
            const uint32_t d = ring + ls * PX_STAGE;
            if (elect_one()) {
                const uint32_t full = smem_u32(bar + ls);
                const int x = px_div(lc.sub, mine ? p.t_own : p.t_pre) * PX_HD, y = mine ? lc.b * p.Tm + lc.key : lc.key;
                mbar_expect_tx(full, 2 * PX_BLK);
                tma_load_2d(d, mine ? &p.kc_map : &p.kp_map, full, x, y);
                tma_load_2d(d + PX_BLK, mine ? &p.vc_map : &p.vp_map, full, x, y);
            }
            __syncwarp();
            if (fresh) {
                orow = row_of(lc.b, lc.sub, lane & 15, opos);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int o = __shfl_sync(~0u, orow, kr + 4 * i);
                    px_copy(sq + (kr + 4 * i) * 128 + ((kc ^ ((kr + 4 * i) & 7)) << 4), p.Q + (size_t)max(o, 0) * PX_HD + 8 * kc, o >= 0);
                }
            }
            if (--to_load > 0) fresh = step(lc);
        }
        ls ^= 1;
        px_commit();
    };
    load();
    int lo[2], hi[2], alo = 0, ahi = 0, stage = 0;        // the keys lo .. hi of the thread's two rows; those that every row of the tile sees
    bool live[2];
    uint32_t qa[4][4];
    float oc[8][4], m[2], l[2];
    bool begin = true;
    int bad = 0;
    uint32_t phase = 0;
    for (; count > 0; count--) {
        px_wait<0>();
        if ((bad = at_all_wait(smem_u32(bar + stage), phase, abort_flag, 131))) break;
        __syncwarp();
        const uint32_t sk = ring + stage * PX_STAGE, sv = sk + PX_BLK;
        phase ^= stage;
        stage ^= 1;
        const int kb = cc.key, k1 = cc.last + 1;
        if (begin) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int t = __shfl_sync(~0u, opos, g + 8 * e);
                live[e] = __shfl_sync(~0u, orow, g + 8 * e) >= 0;
                lo[e] = 0; hi[e] = -1;
                if (live[e]) {
                    hi[e] = cc.b < p.B ? t - p.P : p.P - 1;
                    if (p.win > 0) lo[e] = max(0, t - p.win + 1 - (cc.b < p.B ? p.P : 0));
                }
                if (lo[e] > hi[e]) { lo[e] = 0x7fffffff; hi[e] = -1; }
                m[e] = -INFINITY; l[e] = 0.0f;
            }
            alo = live[0] ? lo[0] : -1; ahi = live[0] ? hi[0] : 0x7fffffff;
            if (live[1]) { alo = max(alo, lo[1]); ahi = min(ahi, hi[1]); }
#pragma unroll
            for (int o = 16; o >= 4; o >>= 1) { alo = max(alo, __shfl_xor_sync(~0u, alo, o)); ahi = min(ahi, __shfl_xor_sync(~0u, ahi, o)); }
#pragma unroll
            for (int s = 0; s < 4; s++) px_ldm(sq + (lane & 15) * 128 + (((2 * s + (lane >> 4)) ^ (lane & 7)) << 4), qa[s]);
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int k = 0; k < 4; k++) oc[j][k] = 0.0f;
            __syncwarp();                                 // the queries are read
        }
        load();                                           // into the place of the block before this one
        px_block(sk, sv, qa, kb, k1, lo, hi, alo, ahi, p.scale_log2, m, l, oc);
        __syncwarp();                                                  // the block is read: the next copies may take its place
        const PxCursor was = cc;
        begin = count == 1 || step(cc);
        if (begin) {                                                   // this warp's segment of the item is whole
            const size_t seg = (size_t)(was.b < p.B ? (long long)was.b * KT + was.sub : (long long)p.B * KT + was.sub) + me;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                l[e] += __shfl_xor_sync(~0u, l[e], 1);
                l[e] += __shfl_xor_sync(~0u, l[e], 2);
                if (!live[e]) continue;
                const bool none = l[e] == 0.0f;                        // the join does not read such a segment's output
                if (q == 0) p.seg_l[seg * 16 + g + 8 * e] = none ? -INFINITY : (m[e] == -INFINITY ? 0.0f : m[e]) + __log2f(l[e]);
                if (none) continue;
                const float inv = __fdividef(1.0f, l[e]);
                float *d = p.seg_o + (seg * 16 + g + 8 * e) * PX_HD + 2 * q;
#pragma unroll
                for (int j = 0; j < 8; j++) *reinterpret_cast<float2 *>(d + 8 * j) = make_float2(oc[j][2 * e] * inv, oc[j][2 * e + 1] * inv);
            }
        }
    }
    px_wait<0>();
    at_give_up(bad, abort_flag, p.errword);
    if (*abort_flag)                                      // aborting: the copies under way must land before the CTA gives its shared memory back
        for (int i = 0; i < 2; i++)
            for (uint32_t k = 0; k < AT_WAIT_LIMIT && !at_test(smem_u32(bar + i), i < stage ? phase ^ 1u : phase); k++) {}
    if (AHEAD) pdl_wait();
}

// ------------------------------------------------------------------ the shared keys of many rows
// One CTA of 160 threads per (kv head, 128 rows, piece of the keys), three on an SM:
//
//   warp 0      one thread: K and V in steps of 64 keys through a three-stage TMA ring, S = Q K^T (128 x 64 x 64) and O += P V
//               (128 x 64 x 64) with tcgen05.mma
//   warps 1-4   softmax: a thread per row holds the 64 scores in registers, running maximum and sum in the exp2 domain, P as bf16
//               over the scores in tensor memory, O rescaled there when a row of the warp has a new maximum
//
// Every row sees every key, so there is no mask but at the end.  Scores and O take 128 columns of tensor memory and 64 scores
// 64 registers, so three CTAs share an SM: their phases wait on one another strictly (scores, weights, O), and the other two
// have the tensor core and the special-function unit meanwhile.  64 slots of 5 tokens, 16 heads, 4 kv heads, 32768 keys: 75.1 us; two
// CTAs an SM with the scores twice in tensor memory, so that a CTA's own phases overlap: 75.1 us; one CTA with two such tiles that
// take turns: 84.2 us.
constexpr int PT_M = 128, PT_N = 64, PT_NS = 3, PT_T = 160;
constexpr int PT_Q = PT_M * 128, PT_KV = PT_N * 128;      // bytes of the queries and of a step's keys (its values follow)
constexpr int PT_SMEM = PT_Q + PT_NS * 2 * PT_KV + 128;
struct PxTcParams {
    alignas(64) CUtensorMap k_map, v_map;
    const bf16 *Q;
    float *part_o, *part_l;                   // [pieces][B*n*H][64], [pieces][B*n*H]
    size_t all_rows;
    int rows, pieces, per, tiles, P, H, G;    // rows of a kv head; pieces of `per` steps, none of them empty; tiles of rows
    float scale_log2;
    int *errword;
};

__global__ void __launch_bounds__(PT_T, 3) k_px_tc(const __grid_constant__ PxTcParams p)
{
    extern __shared__ __align__(1024) uint8_t pt_s[];
    uint8_t *sQ = pt_s, *sKV = pt_s + PT_Q;
    uint64_t *bars = reinterpret_cast<uint64_t *>(sKV + PT_NS * 2 * PT_KV);
    uint64_t *q_full = bars, *s_full = bars + 1, *p_full = bars + 2, *o_full = bars + 3, *spare = bars + 4, *kv_full = bars + 5;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(kv_full + PT_NS);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (smem_u32(pt_s) & 1023u) {             // the swizzled tiles need a 1 KiB-aligned base
        if (threadIdx.x == 0 && p.errword && atomicCAS(p.errword, 0, 201) == 0) { p.errword[1] = 140; p.errword[2] = (int)blockIdx.x; }
        pdl_wait();
        return;
    }
    if (threadIdx.x == 0) {
        prefetch_map(&p.k_map); prefetch_map(&p.v_map);
        mbar_init(smem_u32(q_full), 4);
        mbar_init(smem_u32(s_full), 1);
        mbar_init(smem_u32(p_full), 4);
        mbar_init(smem_u32(o_full), 1);
        mbar_init(smem_u32(spare), 1);
        for (int i = 0; i < PT_NS; i++) mbar_init(smem_u32(&kv_full[i]), 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0) { tmem_alloc(smem_u32(tmem_slot), 128); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();                               // barriers and TMEM above are this kernel's own; its inputs come below
    pdl_trigger();
    const uint32_t tS = *tmem_slot, tO = tS + 64;

    // the row tiles of a piece, which read the same keys, side by side
    const int tile = (int)blockIdx.x % p.tiles, piece = (int)blockIdx.x / p.tiles % p.pieces, kvh = (int)blockIdx.x / p.tiles / p.pieces;
    const int t0 = piece * p.per, nt = min(p.per, (p.P + PT_N - 1) / PT_N - t0);

    if (warp == 0) {
        constexpr uint32_t IDESC_S = make_idesc(PT_M, PT_N, 0, 0), IDESC_PV = make_idesc(PT_M, PX_HD, 0, 1);
        int issued = 0;
        const auto load = [&](int t) {
            if (t < nt) {
                if (elect_one()) {
                    const uint32_t bar = smem_u32(&kv_full[t % PT_NS]), d = smem_u32(sKV + (t % PT_NS) * 2 * PT_KV);
                    mbar_expect_tx(bar, 2 * PT_KV);
                    tma_load_2d(d, &p.k_map, bar, kvh * PX_HD, (t0 + t) * PT_N);
                    tma_load_2d(d + PT_KV, &p.v_map, bar, kvh * PX_HD, (t0 + t) * PT_N);
                }
                __syncwarp();
                issued = t + 1;
            }
        };
        for (int t = 0; t < PT_NS; t++) load(t);
        // descriptors: an address is in their low bits, in units of 16 bytes
        const uint64_t q0 = make_desc(smem_u32(sQ), 16, 1024), k00 = make_desc(smem_u32(sKV), 16, 1024), v00 = make_desc(smem_u32(sKV) + PT_KV, 8192, 1024);
        int st = 0, bad = at_all_wait(smem_u32(q_full), 0, abort_flag, 141);
        uint32_t kv_phase = 0;
        for (int t = 0; !bad && t < nt; t++) {
            if ((bad = at_all_wait(smem_u32(&kv_full[st]), kv_phase, abort_flag, 142))) break;
            // P V of the last step has read the weights, over which the scores go, and its stage
            if (t > 0 && (bad = at_all_wait(smem_u32(o_full), (uint32_t)(t - 1) & 1u, abort_flag, 143))) break;
            tc_fence_after();
            const uint64_t k0 = k00 + (uint64_t)(st * (2 * PT_KV / 16)), v0 = v00 + (uint64_t)(st * (2 * PT_KV / 16));
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < PX_HD / 16; k++) tc_mma_bf16(tS, q0 + 2 * k, k0 + 2 * k, IDESC_S, k > 0);
                tc_commit(smem_u32(s_full));
            }
            __syncwarp();
            if (++st == PT_NS) { st = 0; kv_phase ^= 1; }
            if (t > 0) load(t - 1 + PT_NS);
            if ((bad = at_all_wait(smem_u32(p_full), (uint32_t)t & 1u, abort_flag, 144))) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < PT_N / 16; k++)
                    tc_mma_bf16_ta(tO, tS + k * 8, v0 + 128 * k, IDESC_PV, (t > 0 || k > 0) ? 1u : 0u);
                tc_commit(smem_u32(o_full));
            }
            __syncwarp();
        }
        at_give_up(bad, abort_flag, p.errword);
        if (*abort_flag) {                    // copies and MMAs under way end (bounded) before memory is given back
            for (int i = issued > PT_NS ? issued - PT_NS : 0; i < issued; i++)
                for (uint32_t k = 0; k < AT_WAIT_LIMIT && !at_test(smem_u32(&kv_full[i % PT_NS]), (uint32_t)(i / PT_NS) & 1u); k++) {}
            if (elect_one()) tc_commit(smem_u32(spare));
            __syncwarp();
            for (uint32_t k = 0; k < AT_WAIT_LIMIT && !at_test(smem_u32(spare), 0); k++) {}
        }
    } else {
        // a warp reaches the 32 lanes of tensor memory that its place in the warpgroup gives it
        const int q = warp & 3, r = q * 32 + lane, i = tile * PT_M + r;
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const bool live = i < p.rows, warp_live = tile * PT_M + q * 32 < p.rows;       // rows behind the last are neither computed nor stored
        const int token = px_div(min(i, p.rows - 1), p.G);
        const size_t at = (size_t)token * p.H + (size_t)kvh * p.G + (min(i, p.rows - 1) - token * p.G);       // the row's place in O / 64
        if (warp_live) {
            // the row into the 128-byte swizzle
            const uint4 *src = reinterpret_cast<const uint4 *>(p.Q + at * PX_HD);
            uint4 x[8];
#pragma unroll
            for (int c = 0; c < 8; c++) x[c] = src[c];
#pragma unroll
            for (int c = 0; c < 8; c++) *reinterpret_cast<uint4 *>(sQ + r * 128 + ((c ^ (r & 7)) << 4)) = live ? x[c] : make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(q_full));
        const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
        float m = -3e38f, l = 0.0f;
        int bad = 0;
        for (int t = 0; t < nt; t++) {
            if ((bad = at_all_wait(smem_u32(s_full), (uint32_t)t & 1u, abort_flag, 145))) break;
            if (warp_live) {
                tc_fence_after();
                uint32_t v[64];
                tmem_ld32(tS + lanes, v);
                tmem_ld32(tS + lanes + 32, v + 32);
                tmem_ld_wait();
                const int left = p.P - (t0 + t) * PT_N;
                if (left < PT_N) {
#pragma unroll
                    for (int j = 0; j < PT_N; j++) v[j] = j < left ? v[j] : 0xff800000u;
                }
                float mm[8];                            // eight chains: a step of one takes its instruction's latency
#pragma unroll
                for (int j = 0; j < 8; j++) mm[j] = fmaxf(__uint_as_float(v[j]), __uint_as_float(v[j + 8]));
#pragma unroll
                for (int j = 16; j < PT_N; j += 16)
#pragma unroll
                    for (int e = 0; e < 8; e++) mm[e] = fmaxf(fmaxf(mm[e], __uint_as_float(v[j + e])), __uint_as_float(v[j + 8 + e]));
                mm[0] = fmaxf(fmaxf(mm[0], mm[1]), mm[2]); mm[3] = fmaxf(fmaxf(mm[3], mm[4]), mm[5]);
                const float mx = fmaxf(fmaxf(mm[0], mm[3]), fmaxf(mm[6], mm[7])) * p.scale_log2;
                // A maximum that has grown by more than 2^8: O, to which nothing is being added now, is rescaled.  (Below that the weights
                // stay under 2^8, their rounding to bf16 is as large a part of them, and sums stay far from fp32's limits.)
                if (__any_sync(0xffffffffu, mx > m + 8.0f)) {
                    const float mn = fmaxf(m, mx), corr = ex2(m - mn);
                    m = mn;
                    l *= corr;
                    if (t > 0) {
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            uint32_t o[16];
                            tmem_ld16(tO + lanes + c * 16, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
                            tmem_st16(tO + lanes + c * 16, o);
                        }
                    }
                }
                const uint64_t negm2 = f2_pack(-m, -m);
                uint64_t rs[4] = {0, 0, 0, 0};          // pairs of 0.0f
                uint32_t pk[32];
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    float x0, x1;
                    f2_unpack(f2_fma(f2_packu(v[2 * j], v[2 * j + 1]), scale2, negm2), x0, x1);
                    const float p0 = ex2(x0), p1 = ex2(x1);
                    rs[j & 3] = f2_add(rs[j & 3], f2_pack(p0, p1));
                    const __nv_bfloat162 h2 = __floats2bfloat162_rn(p0, p1);
                    pk[j] = *reinterpret_cast<const uint32_t *>(&h2);
                }
                tmem_st32(tS + lanes, pk);
                float r0, r1;
                f2_unpack(f2_add(f2_add(rs[0], rs[1]), f2_add(rs[2], rs[3])), r0, r1);
                l += r0 + r1;
                tmem_st_wait();
                tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(p_full));
        }
        if (!bad) bad = at_all_wait(smem_u32(o_full), (uint32_t)(nt - 1) & 1u, abort_flag, 146);
        at_give_up(bad, abort_flag, p.errword);
        if (!bad && warp_live) {
            tc_fence_after();
            const bool some = live && l != 0.0f;        // l = 0: every score -inf; the join does not read such a piece
            const size_t po = (size_t)piece * p.all_rows + at;
            const float inv = 1.0f / l;
            float *dst = p.part_o + po * PX_HD;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t o[32];
                tmem_ld32(tO + lanes + c * 32, o);
                tmem_ld_wait();
                if (some)
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<float4 *>(dst + c * 32 + j) = make_float4(__uint_as_float(o[j]) * inv, __uint_as_float(o[j + 1]) * inv,
                                                                                   __uint_as_float(o[j + 2]) * inv, __uint_as_float(o[j + 3]) * inv);
            }
            if (live) p.part_l[po] = some ? m + log2f(l) : -INFINITY;
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 0) { tc_fence_after(); tmem_dealloc(tS, 128); }
}

// NW warps per row of O: its segments and pieces weighted by 2^(their logarithm - the largest), in a fixed order.
template <int NW> __global__ void __launch_bounds__(NW == 1 ? 128 : 32 * NW) k_px_join(const __grid_constant__ PxParams p)
{
    __shared__ float xs[NW == 1 ? 1 : NW][PX_HD + 1];
    const int lane = threadIdx.x & 31, part = NW == 1 ? 0 : threadIdx.x >> 5;
    const size_t rows = (size_t)p.B * p.n * p.H, at = NW == 1 ? (size_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    pdl_trigger();
    pdl_wait();
    if (at >= rows) return;
    const int token = px_div((int)at, p.H), h = (int)at - token * p.H, b = px_div(token, p.n), kvh = px_div(h, p.G), KT = p.KV * p.t_own;
    const int c0 = p.table[b], nb = p.table[b + 1] - c0, all = p.table[p.B], n_pre = p.table[p.B + 1];
    const unsigned per = p.table[p.B + 2];
    if (!px_slot_ok(p.pos[b], p.n, p.P, p.Tm)) return;
    // the row's segments of its slot's keys, then of the shared ones, then the pieces
    const int hg = h - kvh * p.G, rr = (token - b * p.n) * p.G + hg, rp = token * p.G + hg, so = kvh * p.t_own + rr / 16, sp = kvh * p.t_pre + rp / 16;
    const unsigned x0 = (unsigned)c0 * KT + (unsigned)so * nb, x1 = (unsigned)all * KT + (unsigned)sp * n_pre;
    const int w0 = x0 / per, s0 = nb ? (int)((x0 + nb - 1) / per) - w0 + 1 : 0;
    const int w1 = x1 / per, s1 = n_pre ? (int)((x1 + n_pre - 1) / per) - w1 + 1 : 0;
    const size_t g0 = ((size_t)b * KT + so + w0) * 16 + rr % 16, g1 = ((size_t)p.B * KT + sp + w1) * 16 + rp % 16;
    const int S = s0 + s1 + p.Sp;
    const auto place = [&](int s) { return s < s0 ? g0 + 16 * (size_t)s : s < s0 + s1 ? g1 + 16 * (size_t)(s - s0) : (size_t)(s - s0 - s1) * rows + at; };
    // half a warp has the 64 columns of a segment, eight are under way at a time, the first of them while the largest logarithm is
    // found; an empty one's output was not written
    const int half = lane >> 4, c4 = 4 * (lane & 15);
    float lg[4], mx = -INFINITY;
    float4 o[4];
    const auto fetch = [&](int k0) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int s = k0 + 2 * k + half;
            lg[k] = -INFINITY;
            o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (s < S) {
                const size_t pl = place(s);
                const bool seg = s < s0 + s1;
                lg[k] = (seg ? p.seg_l : p.part_l)[pl];
                o[k] = *reinterpret_cast<const float4 *>((seg ? p.seg_o : p.part_o) + pl * PX_HD + c4);
            }
        }
    };
    fetch(8 * part);
    for (int s = lane; s < S; s += 32) mx = fmaxf(mx, (s < s0 + s1 ? p.seg_l : p.part_l)[place(s)]);
#pragma unroll
    for (int i = 16; i; i >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, i));
    const float mref = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f, x[4] = {};
    for (int k0 = 8 * part; k0 < S; k0 += 8 * NW) {
        if (k0 != 8 * part) fetch(k0);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float w = ex2(lg[k] - mref);
            if (w == 0.0f) continue;
            sum += w; x[0] += w * o[k].x; x[1] += w * o[k].y; x[2] += w * o[k].z; x[3] += w * o[k].w;
        }
    }
    sum += __shfl_xor_sync(~0u, sum, 16);
#pragma unroll
    for (int k = 0; k < 4; k++) x[k] += __shfl_xor_sync(~0u, x[k], 16);
    if (NW > 1) {
        if (half == 0) {
#pragma unroll
            for (int k = 0; k < 4; k++) xs[part][c4 + k] = x[k];
            if (lane == 0) xs[part][PX_HD] = sum;
        }
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int w = 1; w < NW; w++) {
            sum += xs[w][PX_HD];
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] += xs[w][c4 + k];
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (half == 0) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0] * inv, x[1] * inv), c = __floats2bfloat162_rn(x[2] * inv, x[3] * inv);
        *reinterpret_cast<uint2 *>(p.O + at * PX_HD + c4) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&c));
    }
    if (p.lse && lane == 0) p.lse[at] = sum == 0.0f ? -INFINITY : (mref + log2f(sum)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ few slots, short prefixes
// One launch: a CTA per (slot, kv head, 16 rows) goes through the shared keys and the slot's own, twelve warps an equal run of blocks each,
// and joins the warps' maxima, sums and outputs in shared memory.  Shared keys are read once a slot, from L2.
constexpr int PS_SMEM = PX_Q + 16 * 128 + 256, PS_ROW = PX_HD + 4;      // rings, the tile's queries, barriers; a row of the join: O, maximum, sum
__global__ void __launch_bounds__(32 * PX_WARPS, 1) k_px_small(const __grid_constant__ PxParams p)
{
    extern __shared__ __align__(1024) uint8_t px_s[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(px_s + PX_Q + 16 * 128);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + 2 * PX_WARPS);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    if (smem_u32(px_s) & 1023u) {             // the swizzled blocks need a 1 KiB-aligned base
        if (tid == 0 && p.errword && atomicCAS(p.errword, 0, 201) == 0) { p.errword[1] = 132; p.errword[2] = (int)blockIdx.x; }
        pdl_wait();
        return;
    }
    if (tid == 0) {
        prefetch_map(&p.kc_map); prefetch_map(&p.vc_map);
        if (p.P > 0) { prefetch_map(&p.kp_map); prefetch_map(&p.vp_map); }
        for (int i = 0; i < 2 * PX_WARPS; i++) mbar_init(smem_u32(&bars[i]), 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    const int KT = p.KV * p.t_own, b = (int)blockIdx.x / KT, sub = (int)blockIdx.x - b * KT, kvh = px_div(sub, p.t_own), row0 = (sub - kvh * p.t_own) * 16;
    const int t0 = p.pos[b], rows = min(16, p.n * p.G - row0);
    if (!px_slot_ok(t0, p.n, p.P, p.Tm)) {
        if (sub == 0 && tid == 0) report_bad_index(p.errword, 306, b, t0);
        return;
    }
    const auto place = [&](int r, int &t) {               // row r: its place in O / 64, and its position
        const int i = px_div(row0 + r, p.G);
        t = t0 + i;
        return (size_t)(b * p.n + i) * p.H + kvh * p.G + row0 + r - i * p.G;
    };
    const int lo_pre = p.win > 0 ? max(0, t0 - p.win + 1) & ~31 : 0, n_pre = lo_pre < p.P ? (p.P - 1 - lo_pre) / 32 + 1 : 0;
    const int first = px_first(p, t0), blocks = n_pre + px_blocks(p, t0), w0 = blocks * warp / PX_WARPS, w1 = blocks * (warp + 1) / PX_WARPS;
    const uint32_t ring = smem_u32(px_s) + warp * (2 * PX_STAGE), sq = smem_u32(px_s) + PX_Q;
    uint64_t *bar = bars + 2 * warp;
    int next = w0;
    const auto load = [&]() {
        if (next < w1) {
            if (elect_one()) {
                const bool mine = next >= n_pre;
                const uint32_t full = smem_u32(bar + ((next - w0) & 1)), d = ring + ((next - w0) & 1) * PX_STAGE;
                const int x = kvh * PX_HD, y = mine ? b * p.Tm + first + 32 * (next - n_pre) : lo_pre + 32 * next;
                mbar_expect_tx(full, 2 * PX_BLK);
                tma_load_2d(d, mine ? &p.kc_map : &p.kp_map, full, x, y);
                tma_load_2d(d + PX_BLK, mine ? &p.vc_map : &p.vp_map, full, x, y);
            }
            __syncwarp();
            next++;
        }
    };
    load();
    if (tid < 128) {                          // 16 bytes each
        const int r = tid >> 3, c = tid & 7;
        int t;
        px_copy(sq + r * 128 + ((c ^ (r & 7)) << 4), p.Q + place(min(r, rows - 1), t) * PX_HD + 8 * c, r < rows);
    }
    px_commit();
    px_wait<0>();
    __syncthreads();
    uint32_t qa[4][4];
#pragma unroll
    for (int s = 0; s < 4; s++) px_ldm(sq + (lane & 15) * 128 + (((2 * s + (lane >> 4)) ^ (lane & 7)) << 4), qa[s]);
    float oc[8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    int lo[2], hi[2], alo = 0, ahi = 0, bad = 0;
    for (int j = w0; j < w1; j++) {
        const bool mine = j >= n_pre;
        if (j == w0 || j == n_pre) {          // the keys that the thread's rows see of these, and those that every row sees
            alo = -1; ahi = 0x7fffffff;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                int t;
                const int r = g + 8 * e;
                lo[e] = 0x7fffffff; hi[e] = -1;
                if (r >= rows) continue;
                place(r, t);
                hi[e] = mine ? t - p.P : p.P - 1;
                lo[e] = p.win > 0 ? max(0, t - p.win + 1 - (mine ? p.P : 0)) : 0;
                if (lo[e] > hi[e]) { lo[e] = 0x7fffffff; hi[e] = -1; }
                alo = max(alo, lo[e]); ahi = min(ahi, hi[e]);
            }
#pragma unroll
            for (int o = 16; o >= 4; o >>= 1) { alo = max(alo, __shfl_xor_sync(~0u, alo, o)); ahi = min(ahi, __shfl_xor_sync(~0u, ahi, o)); }
        }
        const int stage = (j - w0) & 1;
        load();                               // (its place was read in the round before)
        if ((bad = at_all_wait(smem_u32(bar + stage), (uint32_t)((j - w0) >> 1) & 1u, abort_flag, 133))) break;
        const uint32_t sk = ring + stage * PX_STAGE;
        px_block(sk, sk + PX_BLK, qa, mine ? first + 32 * (j - n_pre) : lo_pre + 32 * j, mine ? t0 + p.n - p.P : p.P, lo, hi, alo, ahi, p.scale_log2, m, l, oc);
        __syncwarp();                         // the block is read
    }
    at_give_up(bad, abort_flag, p.errword);
    if (*abort_flag)                          // aborting: the copies under way must land before the CTA gives its shared memory back
        for (int i = max(w0, next - 2); i < next; i++)
            for (uint32_t k = 0; k < AT_WAIT_LIMIT && !at_test(smem_u32(bar + ((i - w0) & 1)), (uint32_t)((i - w0) >> 1) & 1u); k++) {}
    __syncthreads();                          // the rings are free
    if (*abort_flag) return;
    float *xs = reinterpret_cast<float *>(px_s);
#pragma unroll
    for (int e = 0; e < 2; e++) {
        l[e] += __shfl_xor_sync(~0u, l[e], 1);
        l[e] += __shfl_xor_sync(~0u, l[e], 2);
        float *d = xs + (warp * 16 + g + 8 * e) * PS_ROW;
#pragma unroll
        for (int j = 0; j < 8; j++) *reinterpret_cast<float2 *>(d + 8 * j + 2 * q) = make_float2(oc[j][2 * e], oc[j][2 * e + 1]);
        if (q == 0) { d[PX_HD] = m[e]; d[PX_HD + 1] = l[e]; }
    }
    __syncthreads();
    if (tid >= 256) return;
    const int r = tid >> 4, c = 4 * (tid & 15);           // four columns of a row
    if (r >= rows) return;
    float mx = -INFINITY, sum = 0.0f, x[4] = {};
#pragma unroll
    for (int k = 0; k < PX_WARPS; k++) mx = fmaxf(mx, xs[(k * 16 + r) * PS_ROW + PX_HD]);
    const float mref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
    for (int k = 0; k < PX_WARPS; k++) {
        const float *d = xs + (k * 16 + r) * PS_ROW;
        if (d[PX_HD + 1] == 0.0f) continue;   // nothing seen, or all of it -inf
        const float w = ex2(d[PX_HD] - mref);
        const float4 v = *reinterpret_cast<const float4 *>(d + c);
        sum += w * d[PX_HD + 1]; x[0] += w * v.x; x[1] += w * v.y; x[2] += w * v.z; x[3] += w * v.w;
    }
    int t;
    const size_t at = place(r, t);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0] * inv, x[1] * inv), d2 = __floats2bfloat162_rn(x[2] * inv, x[3] * inv);
    *reinterpret_cast<uint2 *>(p.O + at * PX_HD + c) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&d2));
    if (p.lse && c == 0) p.lse[at] = sum == 0.0f ? -INFINITY : (mref + log2f(sum)) * 0.6931471805599453f;
}

// What a call needs: tiles, items, warps, pieces of k_px_tc (Sp of `per` steps of keys), bytes of the workspace's parts.
struct PxPlan { bool small; int t_own, t_pre, warps, Sp, per; size_t seg_o, seg_l, part_o, part_l, table, bytes; };
static PxPlan px_plan(int B, int n, int P, int Tm, int H, int KV, int win)
{
    PxPlan pl = {};
    const long long rows = (long long)B * n * (H / KV);
    // k_px_tc is a launch more, and as long for 16 rows as for 128; k_px_mma's warps take a block of 16 rows and 32 keys at a time.
    // Whole calls, k_px_mma alone and with k_px_tc, by blocks, slots with 64 keys of their own: 6144 (64 rows, 12 kv heads) 20.2 and 21.4 us,
    // 10240 (320 rows, 4) 22.9 and 22.7, 12288 (64 rows, 12) 26.1 and 25.1, 12800 (1280 rows, 4) 24.8 and 22.9, 15360 (320, 4) 29.6 and 23.7,
    // 24576 (16 rows, 12) 58 and 47, 49152 (one row, 12) 100 and 73; with 1000, which k_px_mma takes along: 10240 (320, 4) 21.6 and 27.8,
    // 12288 (64, 12) 47.8 and 50.7, 15360 (320, 4) 25.5 and 29.1, 16384 (128, 4) 24.4 and 27.0.  So the border moves with what the slots' caches
    // can hold (10560 blocks, 480 rows, 2 kv heads, caches of 36 rows: 27.5 and 22.6).  k_px_tc has no window.
    pl.t_own = (n * (H / KV) + 15) / 16;
    // k_px_small up to a CTA an SM and 2048 shared keys, or two and 512, unless it has a CTA for less than half of the SMs and a warp of it would
    // go through 8 blocks of keys more than one of k_px_mma, which deals them out evenly (if the caches are full: the host does not see how
    // full they are).  Us, it and k_px_mma with its join, slots with 64 / 1000 keys of their own, 12 kv heads: 1 slot after 512 keys 5.6 and
    // 8.4 / 7.6 and 9.0, after 2048 9.5 and 9.0 / 11.7 and 9.5 (and 4 less of the host, a launch and the workspace), after 4096 14.8 and 10.9; 12
    // slots after 1024 7.2 and 9.9 / 10.5 and 12.4; 16 slots of 8 tokens, 4 kv heads, after 2048 10.9 and 20.2; 20 slots (240 CTAs) after 128 8.2
    // and 9.9 / 14.7 and 16.3, after 512 10.9 and 9.9 / 16.0 and 16.5, after 1024 13.0 and 10.2; 36 slots (432) after 128 12.7 and 10.3.
    //   Longer caches, by the blocks a warp has more: 1 slot, no shared keys, 2000 of its own (5) 9.6 and 9.4, 4000 (10) 14.3 and 10.1, 16000
    // (38) 46.1 and 14.5; 4 slots (48 CTAs) 4000 (7) 14.8 and 12.3, 8000 (14) 25.8 and 17.2, 16000 (28) 47.7 and 40.5; a window of 1024 in 16000
    // (2) 6.2 and 8.2, of 4096 (10) 14.5 and 9.7.  From half of the SMs on k_px_small asks for as much as HBM gives: 6 slots (72 CTAs) 8000 26.8
    // and 31.3, 32000 93 and 135; 16 slots, 4 kv heads (64) 4000 14.8 and 12.9, 8000 26.2 and 27.8, 32000 90 and 83; 24 slots (288) 16000 180 and 254.
    const long long items = (long long)B * KV * pl.t_own, sms = sm_count(), most = win > 0 && (long long)win + n < (long long)P + Tm ? (long long)win + n : (long long)P + Tm;
    const long long dealt = (items * (Tm < most ? Tm : most) + KV * ((rows + 15) / 16) * (P < most ? P : most)) / sms;       // keys of an SM
    if (((items <= sms && P <= 2048) || (items <= 2 * sms && P <= 512)) && (2 * items >= sms || most - dealt <= 8 * 32 * PX_WARPS)) {
        pl.small = true;
        pl.bytes = 16;
        return pl;
    }
    const long long most_own = (long long)B * KV * pl.t_own * (Tm / 32 + 1);         // if the slots' caches are full
    const bool tc = P > 0 && win <= 0 && KV * ((rows + 15) / 16) * ((P + 31) / 32) > 8704 + (most_own < 4096 ? most_own : 4096);
    pl.t_pre = P > 0 && !tc ? (int)((rows + 15) / 16) : 0;
    pl.warps = sm_count() * PX_WARPS;
    if (tc) {
        const long long t = (P + PT_N - 1) / PT_N, ctas = KV * ((rows + PT_M - 1) / PT_M);
        long long s = 3LL * sm_count() / ctas;
        s = s < 1 ? 1 : s > t ? t : s;
        pl.per = (int)((t + s - 1) / s);
        pl.Sp = (int)((t + pl.per - 1) / pl.per);
    }
    const size_t segs = (size_t)B * KV * pl.t_own + (size_t)KV * pl.t_pre + pl.warps, all = (size_t)B * n * H;
    pl.seg_o = segs * 16 * PX_HD * sizeof(float);
    pl.seg_l = segs * 16 * sizeof(float);
    pl.part_o = (size_t)pl.Sp * all * PX_HD * sizeof(float);
    pl.part_l = ((size_t)pl.Sp * all * sizeof(float) + 15) / 16 * 16;
    pl.table = (size_t)(B + 3) * sizeof(int);
    pl.bytes = pl.seg_o + pl.seg_l + pl.part_o + pl.part_l + pl.table;
    return pl;
}
static bool px_shape_ok(int B, int n, int P, int Tm, int H, int KV)
{
    return B > 0 && B <= PX_MAXB && n > 0 && n <= 64 && P >= 0 && Tm > 0 && H > 0 && KV > 0 && H % KV == 0 && (long long)P + Tm < (1LL << 30) &&
           (long long)B * n * H < (1LL << 24) && (long long)H * 64 < (1LL << 20) &&
           (long long)B * Tm < (1LL << 31) - 64 &&                     // rows of the caches and blocks are counted in 32 bits
           (long long)B * KV * ((n * (H / KV) + 15) / 16) * (Tm / 32 + 2) + (long long)KV * (((long long)B * n * (H / KV) + 15) / 16) * (P / 32 + 2) < (1LL << 31);
}

}  // namespace qlmb
using namespace qlmb;

extern "C" int qlmb_dec_rope_kv(void *Qo, void *Kc, void *Vc, const void *q, const void *k, const void *v, const float *cosb, const float *sinb,
                                const int *pos, int B, int n, int P, int Tm, int H, int KV, int hd, int Tr, void *stream)
{
    QLMB_REQUIRE(Qo && Kc && Vc && q && k && v && cosb && sinb && pos, "qlmb_dec_rope_kv: NULL argument");
    QLMB_REQUIRE(hd == PX_HD, "qlmb_dec_rope_kv: head dimension %d (only 64 is built)", hd);
    QLMB_REQUIRE(n > 0 && P >= 0 && Tm > 0 && H > 0 && KV > 0 && Tr > 0, "qlmb_dec_rope_kv: bad shape n %d P %d Tm %d H %d KV %d Tr %d", n, P, Tm, H, KV, Tr);
    QLMB_REQUIRE((((uintptr_t)Qo | (uintptr_t)Kc | (uintptr_t)Vc | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)cosb | (uintptr_t)sinb) & 15) == 0,
                 "qlmb_dec_rope_kv: rows, caches and tables must be 16-byte aligned");
    if (B <= 0) return QLMB_OK;
    const unsigned long long total = (unsigned long long)B * n * ((unsigned long long)H + 2ull * KV) * 4, blocks = (total + 255) / 256;
    QLMB_REQUIRE(blocks < (1ull << 31), "qlmb_dec_rope_kv: %d slots of %d tokens are too many rows", B, n);
    QLMB_CUDA(pdl_launch_small(k_dec_rope_kv, dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), (bf16 *)Qo, (bf16 *)Kc, (bf16 *)Vc,
                               (const bf16 *)q, (const bf16 *)k, (const bf16 *)v, cosb, sinb, pos, B, n, P, Tm, H, KV, Tr, device_error_word()));
    QLMB_LAUNCH_CHECK("k_dec_rope_kv");
    return QLMB_OK;
}

extern "C" size_t qlmb_dec_attn_prefix_bytes(int B, int n, int P, int Tm, int H, int KV)
{
    if (!px_shape_ok(B, n, P, Tm, H, KV)) return 0;
    // For any window: where k_px_small takes a call without one it takes every one, else the widest is not its, and the rest of a plan asks only
    // whether there is a window.
    const size_t a = px_plan(B, n, P, Tm, H, KV, 0).bytes, b = px_plan(B, n, P, Tm, H, KV, P + Tm - 1).bytes;
    return a > b ? a : b;
}

extern "C" int qlmb_dec_attn_prefix(void *O, float *lse, const void *Q, const void *Kp, const void *Vp, const void *Kc, const void *Vc, const int *pos,
                                    int win, int B, int n, int P, int Tm, int H, int KV, int hd, void *ws, size_t ws_bytes, void *stream)
{
    QLMB_REQUIRE(O && Q && Kc && Vc && pos && (P == 0 || (Kp && Vp)), "qlmb_dec_attn_prefix: NULL argument");
    QLMB_REQUIRE(hd == PX_HD, "qlmb_dec_attn_prefix: head dimension %d (only 64 is built)", hd);
    if (B <= 0) return QLMB_OK;
    QLMB_REQUIRE(px_shape_ok(B, n, P, Tm, H, KV), "qlmb_dec_attn_prefix: bad shape B %d (up to %d) n %d P %d Tm %d H %d KV %d", B, PX_MAXB, n, P, Tm, H, KV);
    QLMB_REQUIRE((((uintptr_t)O | (uintptr_t)Q | (uintptr_t)Kp | (uintptr_t)Vp | (uintptr_t)Kc | (uintptr_t)Vc | (uintptr_t)ws) & 15) == 0,
                 "qlmb_dec_attn_prefix: rows, caches and workspace must be 16-byte aligned");
    if (win >= P + Tm) win = 0;                                        // hides nothing
    const PxPlan pl = px_plan(B, n, P, Tm, H, KV, win);
    QLMB_REQUIRE(pl.small || (ws && ws_bytes >= pl.bytes), "qlmb_dec_attn_prefix: a workspace of %zu bytes, %zu are needed", ws_bytes, pl.bytes);
    PxParams p;
    memset(&p, 0, sizeof p);
    const size_t rows = (size_t)B * n * H;
    char *w = (char *)ws;
    const unsigned long long width = (unsigned long long)KV * PX_HD;
    const struct { CUtensorMap *m; const void *base; unsigned long long rows; } maps[4] = {
        {&p.kc_map, Kc, (unsigned long long)B * Tm}, {&p.vc_map, Vc, (unsigned long long)B * Tm}, {&p.kp_map, Kp, (unsigned long long)P}, {&p.vp_map, Vp, (unsigned long long)P}};
    for (int i = 0; i < (P > 0 && !pl.Sp ? 4 : 2); i++) {
        const int rc = make_map(maps[i].m, maps[i].base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, width, maps[i].rows, width * 2, PX_HD, 32, CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc) return rc;
    }
    p.O = (bf16 *)O; p.lse = lse; p.Q = (const bf16 *)Q; p.pos = pos;
    p.seg_o = (float *)w; w += pl.seg_o;
    p.seg_l = (float *)w; w += pl.seg_l;
    p.part_o = (float *)w; w += pl.part_o;
    p.part_l = (float *)w; w += pl.part_l;
    p.table = (int *)w;
    p.B = B; p.n = n; p.P = P; p.Tm = Tm; p.H = H; p.KV = KV; p.G = H / KV;
    p.win = win;
    p.Sp = pl.Sp; p.t_own = pl.t_own; p.t_pre = pl.t_pre > 0 ? pl.t_pre : 1; p.warps = pl.warps; p.least = 2;
    p.scale_log2 = 1.4426950408889634f * 0.125f;
    p.errword = device_error_word();
    cudaStream_t st = as_stream(stream);
    static bool configured_dev[64];                                    // the attribute belongs to a device's copy of the kernel
    int dev = 0;
    QLMB_CUDA(cudaGetDevice(&dev));
    QLMB_REQUIRE(dev >= 0 && dev < 64, "device index %d", dev);
    if (!configured_dev[dev]) {
        QLMB_CUDA(cudaFuncSetAttribute(k_px_mma<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)px_smem(PX_MAXB)));
        QLMB_CUDA(cudaFuncSetAttribute(k_px_mma<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)px_smem(PX_MAXB)));
        QLMB_CUDA(cudaFuncSetAttribute(k_px_small, cudaFuncAttributeMaxDynamicSharedMemorySize, PS_SMEM));
        QLMB_CUDA(cudaFuncSetAttribute(k_px_tc, cudaFuncAttributeMaxDynamicSharedMemorySize, PT_SMEM));
        configured_dev[dev] = true;
    }
    if (pl.small) {
        QLMB_CUDA(pdl_launch_small(k_px_small, dim3((unsigned)(B * KV * pl.t_own)), dim3(32 * PX_WARPS), PS_SMEM, st, p));
        QLMB_LAUNCH_CHECK("k_px_small");
        return QLMB_OK;
    }
    if (pl.Sp) {
        PxTcParams t;
        memset(&t, 0, sizeof t);
        int rc = make_map(&t.k_map, Kp, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, width, (unsigned long long)P, width * 2, PX_HD, PT_N, CU_TENSOR_MAP_SWIZZLE_128B);
        if (!rc) rc = make_map(&t.v_map, Vp, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, width, (unsigned long long)P, width * 2, PX_HD, PT_N, CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc) return rc;
        t.Q = p.Q; t.part_o = p.part_o; t.part_l = p.part_l; t.all_rows = rows;
        t.rows = (int)(rows / KV); t.pieces = pl.Sp; t.per = pl.per; t.tiles = (t.rows + PT_M - 1) / PT_M;
        t.P = P; t.H = H; t.G = p.G; t.scale_log2 = p.scale_log2; t.errword = p.errword;
        QLMB_CUDA(pdl_launch(true, k_px_tc, dim3((unsigned)(t.tiles * t.pieces * KV)), dim3(PT_T), PT_SMEM, st, t));
        QLMB_LAUNCH_CHECK("k_px_tc");
    }
    QLMB_CUDA(pdl_launch_small(pl.Sp ? k_px_mma<true> : k_px_mma<false>, dim3((unsigned)(pl.warps / PX_WARPS)), dim3(32 * PX_WARPS), px_smem(B), st, p));
    QLMB_LAUNCH_CHECK("k_px_mma");
    // Eight warps a row where rows are few: one of a long prefix has a hundred segments.  Whole calls with one warp a row and with eight:
    // 384 rows 16.6 and 11.0 us, 768 rows 33.4 and 31.8, 5120 rows 96 and 114.
    if (rows <= 1024) QLMB_CUDA(pdl_launch(true, k_px_join<8>, dim3((unsigned)rows), dim3(256), 0, st, p));
    else QLMB_CUDA(pdl_launch(true, k_px_join<1>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, p));
    QLMB_LAUNCH_CHECK("k_px_join");
    return QLMB_OK;
}
