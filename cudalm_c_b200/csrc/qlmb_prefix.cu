// A decode step whose slots share the first P positions and bring several new tokens each (drafts): rotation and append of
// the new rows, attention over the shared rows and the slot's own.  bf16, head dimension 64.
//
//   t = pos[b] + i is the position of token i of slot b; positions below P are rows of Kp, Vp (one copy for all slots), position
//   P + j is row j of the slot's cache.
#include <cuda_bf16.h>
#include <math.h>
#include <stdlib.h>
#include "qlmb_common.cuh"
#include "qlmb_internal.h"

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
// The keys of a row are cut into pieces: the shared rows into Sp, the slot's own into So.  A piece of a tile of 16 query rows is
// one CTA's; it leaves the piece's output, normalised, and the logarithm (base 2) of its sum, and k_px_join adds the pieces up.
// Rows of one kv head that stand side by side: the G = H / KV heads of a token, then the next token's (prefix: of all slots).
struct PxParams {
    bf16 *O;
    float *lse;
    const bf16 *Q, *Kp, *Vp, *Kc, *Vc;
    const int *pos;
    float *part_o, *part_l;                   // [Sp + So][B*n*H][64] and [Sp + So][B*n*H]
    int B, n, P, Tm, H, KV, G, win;
    int Sp, So, own_items;                    // pieces of the shared and of the slots' own rows; items of the latter come first
    int rg_own, rg_pre, lw_own, lw_pre;       // groups of 2^lw tiles of 16 rows a (slot, kv head), resp. a kv head
    float scale_log2;                         // log2(e) / sqrt(64)
    int *errword;
};

__device__ __forceinline__ float px_ex2(float x)      // 2^x (ex2.approx: 2 ulp, -inf -> 0)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void px_mma(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A slot whose new tokens do not all lie in its cache (the first may see nothing of its own: pos = P - 1) is not touched.
__device__ __forceinline__ bool px_slot_ok(long long t0, int n, int P, int Tm) { return t0 - P >= -1 && t0 - P + n <= Tm; }
__device__ __forceinline__ bool px_nonfinite(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }

// A group of one, two or four tiles of 16 query rows against the keys of a piece: a warp has one tile, and where there are fewer than
// four they share the keys in blocks of 32, each with maximum, sum and output of its own, joined through shared memory at the end.
// A warp's blocks come through a ring of its own, three blocks of keys and values in 16-byte pieces whose place in the row is turned
// by the key; two are under way while one is multiplied on mma.m16n8k16.
constexpr int PX_NS = 3, PX_BLK = 32 * 128;              // stages, bytes of a block's keys (its values lie behind them)
constexpr int PX_SMEM = 4 * PX_NS * 2 * PX_BLK;
__device__ __forceinline__ uint32_t px_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void px_copy(uint32_t dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void px_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void px_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void px_ldm(uint32_t a, uint32_t v[4])
{ asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory"); }
__device__ __forceinline__ void px_ldmt(uint32_t a, uint32_t v[4])
{ asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory"); }

__global__ void __launch_bounds__(128, 2) k_px_mma(const __grid_constant__ PxParams p)
{
    extern __shared__ __align__(128) uint8_t px_s[];
    __shared__ float sm[4][16], sl[4][16];
    float (*so)[16][PX_HD + 4] = reinterpret_cast<float (*)[16][PX_HD + 4]>(px_s);       // at the end, over the rings
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    pdl_trigger();
    pdl_wait();
    const int KD = p.KV * PX_HD, rows_slot = p.n * p.G;
    const bool own = (int)blockIdx.x < p.own_items;
    int it = own ? blockIdx.x : blockIdx.x - p.own_items;
    int b = 0, kvh, rg, piece;
    const int npiece = own ? p.So : p.Sp, lw = own ? p.lw_own : p.lw_pre;
    const bf16 *K, *V;
    if (own) {
        piece = it % p.So; it /= p.So;
        rg = it % p.rg_own; it /= p.rg_own;
        kvh = it % p.KV; b = it / p.KV;
        K = p.Kc + (size_t)b * p.Tm * KD; V = p.Vc + (size_t)b * p.Tm * KD;
        if (!px_slot_ok(p.pos[b], p.n, p.P, p.Tm)) {
            if (threadIdx.x == 0 && kvh == 0 && rg == 0 && piece == 0) report_bad_index(p.errword, 306, b, p.pos[b]);
            return;
        }
    } else {
        rg = it % p.rg_pre; it /= p.rg_pre;               // groups that read the same keys side by side
        piece = it % p.Sp; kvh = it / p.Sp;
        K = p.Kp; V = p.Vp;
    }
    K += kvh * PX_HD; V += kvh * PX_HD;
    const int share = warp >> lw, shares = 4 >> lw, rt = (rg << lw) + (warp & ((1 << lw) - 1));      // the warp's part of the keys, its tile
    // the keys lo .. hi of the two rows this thread holds, and of the tile; orow: the row's place in O / 64, -1 where there is none
    int lo[2], hi[2];
    long long orow[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int rr = rt * 16 + g + 8 * e;
        lo[e] = 0; hi[e] = -1; orow[e] = -1;
        if (own) {
            if (rr < rows_slot) {
                const int i = rr / p.G, t = p.pos[b] + i;
                orow[e] = ((long long)b * p.n + i) * p.H + kvh * p.G + rr % p.G;
                hi[e] = t - p.P;
                if (p.win > 0) lo[e] = max(0, t - p.win + 1 - p.P);
            }
        } else if (rr < p.B * rows_slot) {
            const int token = rr / p.G, t0 = p.pos[token / p.n];
            if (px_slot_ok(t0, p.n, p.P, p.Tm)) {
                const int t = t0 + token % p.n;
                orow[e] = (long long)token * p.H + kvh * p.G + rr % p.G;
                hi[e] = p.P - 1;
                if (p.win > 0) lo[e] = max(0, t - p.win + 1);
            }
        }
        if (lo[e] > hi[e]) { lo[e] = 0x7fffffff; hi[e] = -1; }         // sees nothing here
    }
    int tlo = min(lo[0], lo[1]), thi = max(hi[0], hi[1]);
    int alo = orow[0] < 0 ? -1 : lo[0], ahi = orow[0] < 0 ? 0x7fffffff : hi[0];      // what every row of the tile sees
    if (orow[1] >= 0) { alo = max(alo, lo[1]); ahi = min(ahi, hi[1]); }
#pragma unroll
    for (int o = 16; o >= 4; o >>= 1) {
        tlo = min(tlo, __shfl_xor_sync(~0u, tlo, o)); thi = max(thi, __shfl_xor_sync(~0u, thi, o));
        alo = max(alo, __shfl_xor_sync(~0u, alo, o)); ahi = min(ahi, __shfl_xor_sync(~0u, ahi, o));
    }
    int k0 = 0, k1 = 0;                                                // keys of this piece: whole blocks of 32
    if (thi >= 0) {
        tlo &= ~31;
        const int nblk = (thi - tlo) / 32 + 1, per = (nblk + npiece - 1) / npiece;
        k0 = tlo + min(piece * per, nblk) * 32; k1 = min(thi + 1, tlo + min((piece + 1) * per, nblk) * 32);
    }
    const int step = 32 * shares;
    // a lane's pieces of a block: keys kr + 4 i, 16 bytes kc of the row
    const int kr = lane >> 3, kc = lane & 7;
    const uint32_t ring = px_addr(px_s) + warp * (PX_NS * 2 * PX_BLK);
    int lb = k0 + 32 * share, ls = 0;                                  // the next block to be requested, and its stage
    const auto load = [&]() {
        if (lb < k1) {
            const uint32_t d = ring + ls * (2 * PX_BLK) + kr * 128;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const size_t o = (size_t)min(lb + kr + 4 * i, k1 - 1) * KD + 8 * kc;      // keys behind the last: the last once more
                const uint32_t at = d + i * 512 + ((kc ^ ((kr + 4 * i) & 7)) << 4);
                px_copy(at, K + o);
                px_copy(at + PX_BLK, V + o);
            }
            lb += step;
        }
        ls = ls + 1 == PX_NS ? 0 : ls + 1;
        px_commit();
    };
    load(); load();
    uint32_t qa[4][4];
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int e = 0; e < 2; e++) qa[s][2 * h + e] = orow[e] >= 0 ? *reinterpret_cast<const uint32_t *>(p.Q + (size_t)orow[e] * PX_HD + 16 * s + 8 * h + 2 * q) : 0u;
    float oc[8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    int stage = 0;
    for (int kb = k0 + 32 * share; kb < k1; kb += step) {
        px_wait<1>();
        __syncwarp();
        load();                                                        // into the place of the block before this one
        const uint32_t sk = ring + stage * (2 * PX_BLK), sv = sk + PX_BLK;
        stage = stage + 1 == PX_NS ? 0 : stage + 1;
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
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int e = c >> 1, key = kb + 8 * t + 2 * q + (c & 1);
                s[t][c] *= p.scale_log2;
                if (edge && (key < lo[e] || key > hi[e] || key >= k1)) s[t][c] = -INFINITY;
                mx[e] = fmaxf(mx[e], s[t][c]);
            }
        float mu[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(~0u, mx[e], 1));
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(~0u, mx[e], 2));
            const float mn = fmaxf(m[e], mx[e]);
            mu[e] = mn == -INFINITY ? 0.0f : mn;                       // nothing seen yet: every weight 0
            const float corr = px_ex2(m[e] - mu[e]);
            m[e] = mn;
            l[e] *= corr;
#pragma unroll
            for (int j = 0; j < 8; j++) { oc[j][2 * e] *= corr; oc[j][2 * e + 1] *= corr; }
        }
        uint32_t pa[2][4];                                             // weights in bf16, as every attention of the library has them
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float p0 = px_ex2(s[t][2 * e] - mu[e]), p1 = px_ex2(s[t][2 * e + 1] - mu[e]);
                l[e] += p0 + p1;
                const __nv_bfloat162 h2 = __floats2bfloat162_rn(p0, p1);
                pa[t >> 1][2 * (t & 1) + e] = *reinterpret_cast<const uint32_t *>(&h2);
            }
        uint32_t vw[2][4][4];                                          // [16 keys][16 dimensions]: two pairs of operands
        bool odd = false;                                              // an infinity or a NaN that some row must not see
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                px_ldmt(sv + (16 * t + (lane & 15)) * 128 + (((2 * j + (lane >> 4)) ^ (lane & 7)) << 4), vw[t][j]);
                if (edge) odd |= px_nonfinite(vw[t][j][0]) | px_nonfinite(vw[t][j][1]) | px_nonfinite(vw[t][j][2]) | px_nonfinite(vw[t][j][3]);
            }
        if (!edge || !__any_sync(~0u, odd)) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int j = 0; j < 4; j++) { px_mma(oc[2 * j], pa[t], vw[t][j][0], vw[t][j][1]); px_mma(oc[2 * j + 1], pa[t], vw[t][j][2], vw[t][j][3]); }
        } else {
            // 0 * inf is not 0: row by row, with the keys the row does not see taken as zeros (a register holds keys 2 q and 2 q + 1 of eight)
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
        __syncwarp();                                                  // the block is read: the next copies may take its place
    }
    px_wait<0>();
    __syncthreads();
    // a thread holds columns 8 j + 2 q and the next of its rows
#pragma unroll
    for (int e = 0; e < 2; e++) {
        l[e] += __shfl_xor_sync(~0u, l[e], 1);
        l[e] += __shfl_xor_sync(~0u, l[e], 2);
        if (q == 0) { sm[warp][g + 8 * e] = m[e]; sl[warp][g + 8 * e] = l[e]; }
#pragma unroll
        for (int j = 0; j < 8; j++) *reinterpret_cast<float2 *>(&so[warp][g + 8 * e][8 * j + 2 * q]) = make_float2(oc[j][2 * e], oc[j][2 * e + 1]);
    }
    __syncthreads();
    // the tiles' rows, eight threads each, over the shares
    for (int tile = 0; tile < 1 << lw; tile++) {
    const int r = threadIdx.x >> 3, c8 = (threadIdx.x & 7) * 8, rr = ((rg << lw) + tile) * 16 + r;
    long long at = -1;
    if (own) { if (rr < rows_slot) at = ((long long)b * p.n + rr / p.G) * p.H + kvh * p.G + rr % p.G; }
    else if (rr < p.B * rows_slot && px_slot_ok(p.pos[rr / p.G / p.n], p.n, p.P, p.Tm)) at = (long long)(rr / p.G) * p.H + kvh * p.G + rr % p.G;
    if (at < 0) continue;
    float mm = -INFINITY;
    for (int w = tile; w < 4; w += 1 << lw) mm = fmaxf(mm, sm[w][r]);
    const float mref = mm == -INFINITY ? 0.0f : mm;
    float ll = 0.0f, a[8] = {};
    for (int w = tile; w < 4; w += 1 << lw) {
        if (sm[w][r] == -INFINITY && sl[w][r] == 0.0f) continue;       // this warp saw nothing (a NaN among the scores leaves a sum of NaN)
        const float f = px_ex2(sm[w][r] - mref);
        ll += sl[w][r] * f;
#pragma unroll
        for (int k = 0; k < 8; k++) a[k] += so[w][r][c8 + k] * f;
    }
    const bool none = ll == 0.0f;
    const float inv = none ? 0.0f : 1.0f / ll, lg = none ? -INFINITY : mref + log2f(ll);
    if (p.Sp + p.So == 1) {                                            // the only piece: its output is the row's
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const __nv_bfloat162 h2 = none ? __floats2bfloat162_rn(0.0f, 0.0f) : __floats2bfloat162_rn(a[2 * k] * inv, a[2 * k + 1] * inv);
            w[k] = *reinterpret_cast<const uint32_t *>(&h2);
        }
        *reinterpret_cast<uint4 *>(p.O + (size_t)at * PX_HD + c8) = make_uint4(w[0], w[1], w[2], w[3]);
        if (p.lse && c8 == 0) p.lse[at] = lg * 0.6931471805599453f;
        continue;
    }
    const size_t po = (size_t)(own ? p.Sp + piece : piece) * ((size_t)p.B * p.n * p.H) + (size_t)at;
    if (c8 == 0) p.part_l[po] = lg;
    if (none) continue;                                                // the join does not read it
    float *d = p.part_o + po * PX_HD + c8;
    *reinterpret_cast<float4 *>(d) = make_float4(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
    *reinterpret_cast<float4 *>(d + 4) = make_float4(a[4] * inv, a[5] * inv, a[6] * inv, a[7] * inv);
    }
}

// A warp per row of O: the pieces' outputs weighted by 2^(their logarithm - the largest), in ascending order.
__global__ void __launch_bounds__(128) k_px_join(const __grid_constant__ PxParams p)
{
    const int lane = threadIdx.x & 31;
    const size_t rows = (size_t)p.B * p.n * p.H, at = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    pdl_trigger();
    pdl_wait();
    if (at >= rows || !px_slot_ok(p.pos[at / ((size_t)p.n * p.H)], p.n, p.P, p.Tm)) return;
    const int S = p.Sp + p.So;
    float mx = -INFINITY;
    for (int s = lane; s < S; s += 32) mx = fmaxf(mx, p.part_l[s * rows + at]);
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
    const float mref = mx == -INFINITY ? 0.0f : mx;
    // half a warp has the 64 columns of a piece, four of its pieces are under way at a time; an empty one's output was not written
    const int half = lane >> 4, c4 = 4 * (lane & 15);
    float sum = 0.0f, x[4] = {};
    for (int s0 = 0; s0 < S; s0 += 32) {
        const float w = s0 + lane < S ? px_ex2(p.part_l[(s0 + lane) * rows + at] - mref) : 0.0f;
        for (int k0 = 0; k0 < 32 && s0 + k0 < S; k0 += 8) {
            float wk[4];
            float4 o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int s = k0 + 2 * k + half;
                wk[k] = __shfl_sync(~0u, w, s);
                o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (wk[k] != 0.0f) o[k] = *reinterpret_cast<const float4 *>(p.part_o + ((s0 + s) * rows + at) * PX_HD + c4);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) { sum += wk[k]; x[0] += wk[k] * o[k].x; x[1] += wk[k] * o[k].y; x[2] += wk[k] * o[k].z; x[3] += wk[k] * o[k].w; }
        }
    }
    sum += __shfl_xor_sync(~0u, sum, 16);
#pragma unroll
    for (int k = 0; k < 4; k++) x[k] += __shfl_xor_sync(~0u, x[k], 16);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (half == 0) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0] * inv, x[1] * inv), b = __floats2bfloat162_rn(x[2] * inv, x[3] * inv);
        *reinterpret_cast<uint2 *>(p.O + at * PX_HD + c4) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
    if (p.lse && lane == 0) p.lse[at] = sum == 0.0f ? -INFINITY : (mref + log2f(sum)) * 0.6931471805599453f;
}

// Pieces of a call.
struct PxPlan { int Sp, So, rg_own, rg_pre, lw_own, lw_pre, tc, per; };
static PxPlan px_plan(int B, int n, int P, int Tm, int H, int KV, int win)
{
    PxPlan pl = {};
    const long long rows = (long long)B * n * (H / KV);
    const auto tiles = [](long long rows, int *lw, int *rg) {
        const long long t = (rows + 15) / 16;
        *lw = t <= 1 ? 0 : t <= 2 ? 1 : 2;
        *rg = (int)((t + (1 << *lw) - 1) >> *lw);
    };
    tiles((long long)n * (H / KV), &pl.lw_own, &pl.rg_own);
    tiles(rows, &pl.lw_pre, &pl.rg_pre);
    const auto pieces = [](long long want, long long items, long long keys) {
        const long long most = (keys + 127) / 128, s = want / items;
        return (int)(s < 1 ? 1 : s > most ? (most < 1 ? 1 : most) : s);
    };
    int w1 = 3, w2 = 3, lim = 64;
    { const char *e = getenv("PX_W1"); if (e) w1 = atoi(e); e = getenv("PX_W2"); if (e) w2 = atoi(e); e = getenv("PX_LIM"); if (e) lim = atoi(e); }
    pl.So = pieces((long long)w1 * sm_count(), (long long)B * KV * pl.rg_own, Tm);
    if (P > 0) {
        pl.tc = rows > lim && win <= 0;
        if (pl.tc) {
            const int t = (P + 127) / 128, s = pieces(2LL * sm_count(), KV * ((rows + 127) / 128), P);
            pl.per = (t + s - 1) / s;
            pl.Sp = (t + pl.per - 1) / pl.per;
        } else
            pl.Sp = pieces((long long)w2 * sm_count(), (long long)KV * pl.rg_pre, P);
    }
    return pl;
}
static bool px_shape_ok(int B, int n, int P, int Tm, int H, int KV)
{
    return B > 0 && n > 0 && n <= 64 && P >= 0 && Tm > 0 && H > 0 && KV > 0 && H % KV == 0 && (long long)P + Tm < (1LL << 30) &&
           (long long)B * n * H < (1LL << 24) && (long long)H * 64 < (1LL << 20);
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
    const PxPlan pl = px_plan(B, n, P, Tm, H, KV, 0), pw = px_plan(B, n, P, Tm, H, KV, 1);
    const size_t S = (size_t)pl.So + (pl.Sp > pw.Sp ? pl.Sp : pw.Sp);
    return S * (size_t)B * n * H * (PX_HD + 1) * sizeof(float) + 16;
}

extern "C" int qlmb_dec_attn_prefix(void *O, float *lse, const void *Q, const void *Kp, const void *Vp, const void *Kc, const void *Vc, const int *pos,
                                    int win, int B, int n, int P, int Tm, int H, int KV, int hd, void *ws, size_t ws_bytes, void *stream)
{
    QLMB_REQUIRE(O && Q && Kc && Vc && pos && ws && (P == 0 || (Kp && Vp)), "qlmb_dec_attn_prefix: NULL argument");
    QLMB_REQUIRE(hd == PX_HD, "qlmb_dec_attn_prefix: head dimension %d (only 64 is built)", hd);
    if (B <= 0) return QLMB_OK;
    QLMB_REQUIRE(px_shape_ok(B, n, P, Tm, H, KV), "qlmb_dec_attn_prefix: bad shape B %d n %d P %d Tm %d H %d KV %d", B, n, P, Tm, H, KV);
    QLMB_REQUIRE((((uintptr_t)O | (uintptr_t)Q | (uintptr_t)Kp | (uintptr_t)Vp | (uintptr_t)Kc | (uintptr_t)Vc | (uintptr_t)ws) & 15) == 0,
                 "qlmb_dec_attn_prefix: rows, caches and workspace must be 16-byte aligned");
    const size_t need = qlmb_dec_attn_prefix_bytes(B, n, P, Tm, H, KV);
    QLMB_REQUIRE(ws_bytes >= need, "qlmb_dec_attn_prefix: a workspace of %zu bytes, %zu are needed", ws_bytes, need);
    const PxPlan pl = px_plan(B, n, P, Tm, H, KV, win);
    PxParams p = {};
    const size_t rows = (size_t)B * n * H;
    p.O = (bf16 *)O; p.lse = lse; p.Q = (const bf16 *)Q;
    p.Kp = (const bf16 *)Kp; p.Vp = (const bf16 *)Vp; p.Kc = (const bf16 *)Kc; p.Vc = (const bf16 *)Vc; p.pos = pos;
    p.part_o = (float *)ws; p.part_l = p.part_o + (size_t)(pl.Sp + pl.So) * rows * PX_HD;
    p.B = B; p.n = n; p.P = P; p.Tm = Tm; p.H = H; p.KV = KV; p.G = H / KV;
    p.win = win < (1 << 30) ? win : 0;                                 // such a window hides nothing
    p.Sp = pl.Sp; p.So = pl.So; p.rg_own = pl.rg_own; p.rg_pre = pl.rg_pre; p.lw_own = pl.lw_own; p.lw_pre = pl.lw_pre;
    const long long own_items = (long long)B * KV * pl.rg_own * pl.So, items = own_items + (pl.tc ? 0 : (long long)KV * pl.rg_pre * pl.Sp);
    QLMB_REQUIRE(items < (1LL << 31), "qlmb_dec_attn_prefix: %lld pieces are too many", items);
    p.own_items = (int)own_items;
    p.scale_log2 = 1.4426950408889634f * 0.125f;
    p.errword = device_error_word();
    cudaStream_t st = as_stream(stream);
    if (pl.tc) {
        const PrefixAttn px = {p.Q, p.part_o, p.part_l, rows, (int)(rows / KV), pl.Sp, pl.per};
        const int rc = attn_prefix_launch(px, Kp, Vp, P, H, KV, st);
        if (rc) return rc;
    }
    static bool configured_dev[64];                                    // the attribute belongs to a device's copy of the kernel
    int dev = 0;
    QLMB_CUDA(cudaGetDevice(&dev));
    QLMB_REQUIRE(dev >= 0 && dev < 64, "device index %d", dev);
    if (!configured_dev[dev]) {
        QLMB_CUDA(cudaFuncSetAttribute(k_px_mma, cudaFuncAttributeMaxDynamicSharedMemorySize, PX_SMEM));
        configured_dev[dev] = true;
    }
    QLMB_CUDA(pdl_launch_small(k_px_mma, dim3((unsigned)items), dim3(128), PX_SMEM, st, p));
    QLMB_LAUNCH_CHECK("k_px_mma");
    if (pl.Sp + pl.So > 1) {
        QLMB_CUDA(pdl_launch(true, k_px_join, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, p));
        QLMB_LAUNCH_CHECK("k_px_join");
    }
    return QLMB_OK;
}
