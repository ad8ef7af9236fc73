// A decode step whose slots share the first P positions and bring several new tokens each (drafts): rotation and append of
// the new rows, attention over the shared rows and the slot's own.  bf16, head dimension 64.
//
//   t = pos[b] + i is the position of token i of slot b; positions below P are rows of Kp, Vp (one copy for all slots), position
//   P + j is row j of the slot's cache.
#include <cuda_bf16.h>
#include <math.h>
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
    int Sp, So, own_items, rt_own, rt_pre;    // pieces; items of the slots' own rows come first; row tiles a (slot, kv head) / a kv head
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

// One tile of 16 query rows against the keys of a piece: four warps take blocks of 32 keys in turn, each with maximum, sum and
// output of its own, joined through shared memory at the end.  Products on mma.m16n8k16, fed from global memory without a
// detour: the order of the contracted dimension is free as long as both operands agree, so a thread takes 16 bytes of a key's
// row (dimensions 8 q .. and 32 + 8 q ..) where the instruction wants pairs, and of V eight neighbouring dimensions of each of
// its four keys, paired up by byte permutations.
__global__ void __launch_bounds__(128) k_px_mma(const __grid_constant__ PxParams p)
{
    __shared__ float so[4][16][PX_HD + 4];
    __shared__ float sm[4][16], sl[4][16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    pdl_trigger();
    pdl_wait();
    const int KD = p.KV * PX_HD, rows_slot = p.n * p.G;
    const bool own = (int)blockIdx.x < p.own_items;
    int it = own ? blockIdx.x : blockIdx.x - p.own_items;
    int b = 0, kvh, rt, piece, npiece;
    const bf16 *K, *V;
    if (own) {
        piece = it % p.So; it /= p.So; npiece = p.So;
        rt = it % p.rt_own; it /= p.rt_own;
        kvh = it % p.KV; b = it / p.KV;
        K = p.Kc + (size_t)b * p.Tm * KD; V = p.Vc + (size_t)b * p.Tm * KD;
        if (!px_slot_ok(p.pos[b], p.n, p.P, p.Tm)) {
            if (threadIdx.x == 0 && kvh == 0 && rt == 0 && piece == 0) report_bad_index(p.errword, 306, b, p.pos[b]);
            return;
        }
    } else {
        piece = it % p.Sp; it /= p.Sp; npiece = p.Sp;
        rt = it % p.rt_pre; kvh = it / p.rt_pre;
        K = p.Kp; V = p.Vp;
    }
    K += kvh * PX_HD; V += kvh * PX_HD;
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
    uint32_t qa[4][4];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        uint4 x = make_uint4(0, 0, 0, 0), y = x;
        if (orow[e] >= 0) {
            const bf16 *r = p.Q + (size_t)orow[e] * PX_HD + 8 * q;
            x = *reinterpret_cast<const uint4 *>(r); y = *reinterpret_cast<const uint4 *>(r + 32);
        }
        qa[0][e] = x.x; qa[0][2 + e] = x.y; qa[1][e] = x.z; qa[1][2 + e] = x.w;
        qa[2][e] = y.x; qa[2][2 + e] = y.y; qa[3][e] = y.z; qa[3][2 + e] = y.w;
    }
    float oc[8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    for (int kb = k0 + 32 * warp; kb < k1; kb += 128) {
        uint4 kx[4][2], vx[2][4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const bf16 *r = K + (size_t)min(kb + 8 * t + g, k1 - 1) * KD + 8 * q;
            kx[t][0] = *reinterpret_cast<const uint4 *>(r); kx[t][1] = *reinterpret_cast<const uint4 *>(r + 32);
        }
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int w = 0; w < 4; w++)
                vx[t][w] = *reinterpret_cast<const uint4 *>(V + (size_t)min(kb + 16 * t + 2 * q + (w & 1) + 8 * (w >> 1), k1 - 1) * KD + 8 * g);
        float s[4][4] = {};
#pragma unroll
        for (int t = 0; t < 4; t++) {
            px_mma(s[t], qa[0], kx[t][0].x, kx[t][0].y);
            px_mma(s[t], qa[1], kx[t][0].z, kx[t][0].w);
            px_mma(s[t], qa[2], kx[t][1].x, kx[t][1].y);
            px_mma(s[t], qa[3], kx[t][1].z, kx[t][1].w);
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
        bool odd = false;                                              // an infinity or a NaN that some row must not see
        if (edge) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int w = 0; w < 4; w++) odd |= px_nonfinite(vx[t][w].x) | px_nonfinite(vx[t][w].y) | px_nonfinite(vx[t][w].z) | px_nonfinite(vx[t][w].w);
            odd = __any_sync(~0u, odd);
        }
        if (!odd) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t w0[4] = {vx[t][0].x, vx[t][0].y, vx[t][0].z, vx[t][0].w}, w1[4] = {vx[t][1].x, vx[t][1].y, vx[t][1].z, vx[t][1].w};
                const uint32_t w2[4] = {vx[t][2].x, vx[t][2].y, vx[t][2].z, vx[t][2].w}, w3[4] = {vx[t][3].x, vx[t][3].y, vx[t][3].z, vx[t][3].w};
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                    px_mma(oc[j], pa[t], __byte_perm(w0[j >> 1], w1[j >> 1], sel), __byte_perm(w2[j >> 1], w3[j >> 1], sel));
                }
            }
        } else {
            // 0 * inf is not 0: row by row, with the keys the row does not see taken as zeros
            for (int r = 0; r < 16; r++) {
                const int rlo = __shfl_sync(~0u, r < 8 ? lo[0] : lo[1], (r & 7) * 4), rhi = __shfl_sync(~0u, r < 8 ? hi[0] : hi[1], (r & 7) * 4);
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    bool see[4];
#pragma unroll
                    for (int w = 0; w < 4; w++) { const int key = kb + 16 * t + 2 * q + (w & 1) + 8 * (w >> 1); see[w] = key >= rlo && key <= rhi && key < k1; }
                    const uint32_t *v0 = &vx[t][0].x, *v1 = &vx[t][1].x, *v2 = &vx[t][2].x, *v3 = &vx[t][3].x;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                        float c[4] = {};
                        px_mma(c, pa[t], __byte_perm(see[0] ? v0[j >> 1] : 0u, see[1] ? v1[j >> 1] : 0u, sel),
                               __byte_perm(see[2] ? v2[j >> 1] : 0u, see[3] ? v3[j >> 1] : 0u, sel));
                        if (r == g) { oc[j][0] += c[0]; oc[j][1] += c[1]; }
                        if (r == g + 8) { oc[j][2] += c[2]; oc[j][3] += c[3]; }
                    }
                }
            }
        }
    }
    // the four warps' shares; a thread holds columns 16 q .. 16 q + 15 of its rows (column 8 c + j of product j)
#pragma unroll
    for (int e = 0; e < 2; e++) {
        l[e] += __shfl_xor_sync(~0u, l[e], 1);
        l[e] += __shfl_xor_sync(~0u, l[e], 2);
        if (q == 0) { sm[warp][g + 8 * e] = m[e]; sl[warp][g + 8 * e] = l[e]; }
#pragma unroll
        for (int c = 0; c < 2; c++) {
            float *d = &so[warp][g + 8 * e][16 * q + 8 * c];
            *reinterpret_cast<float4 *>(d) = make_float4(oc[0][2 * e + c], oc[1][2 * e + c], oc[2][2 * e + c], oc[3][2 * e + c]);
            *reinterpret_cast<float4 *>(d + 4) = make_float4(oc[4][2 * e + c], oc[5][2 * e + c], oc[6][2 * e + c], oc[7][2 * e + c]);
        }
    }
    __syncthreads();
    const int r = threadIdx.x >> 3, c8 = (threadIdx.x & 7) * 8, rr = rt * 16 + r;
    long long at = -1;
    if (own) { if (rr < rows_slot) at = ((long long)b * p.n + rr / p.G) * p.H + kvh * p.G + rr % p.G; }
    else if (rr < p.B * rows_slot && px_slot_ok(p.pos[rr / p.G / p.n], p.n, p.P, p.Tm)) at = (long long)(rr / p.G) * p.H + kvh * p.G + rr % p.G;
    if (at < 0) return;
    float mm = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
    const float mref = mm == -INFINITY ? 0.0f : mm;
    float ll = 0.0f, a[8] = {};
#pragma unroll
    for (int w = 0; w < 4; w++) {
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
        return;
    }
    const size_t po = (size_t)(own ? p.Sp + piece : piece) * ((size_t)p.B * p.n * p.H) + (size_t)at;
    if (c8 == 0) p.part_l[po] = lg;
    if (none) return;                                                  // the join does not read it
    float *d = p.part_o + po * PX_HD + c8;
    *reinterpret_cast<float4 *>(d) = make_float4(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
    *reinterpret_cast<float4 *>(d + 4) = make_float4(a[4] * inv, a[5] * inv, a[6] * inv, a[7] * inv);
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
    float sum = 0.0f, x = 0.0f, y = 0.0f;
    for (int s0 = 0; s0 < S; s0 += 32) {
        const float w = s0 + lane < S ? px_ex2(p.part_l[(s0 + lane) * rows + at] - mref) : 0.0f;
        for (int k = 0; k < 32 && s0 + k < S; k++) {
            const float wk = __shfl_sync(~0u, w, k);
            if (wk == 0.0f) continue;                                  // an empty piece's output was not written
            const float2 o = *reinterpret_cast<const float2 *>(p.part_o + ((s0 + k) * rows + at) * PX_HD + 2 * lane);
            sum += wk; x += wk * o.x; y += wk * o.y;
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<__nv_bfloat162 *>(p.O + at * PX_HD + 2 * lane) = __floats2bfloat162_rn(x * inv, y * inv);
    if (p.lse && lane == 0) p.lse[at] = sum == 0.0f ? -INFINITY : (mref + log2f(sum)) * 0.6931471805599453f;
}

// Pieces of a call.
struct PxPlan { int Sp, So, rt_own, rt_pre, tc, per; };
static PxPlan px_plan(int B, int n, int P, int Tm, int H, int KV, int win)
{
    PxPlan pl = {};
    const long long want = 3LL * sm_count();
    const long long rows = (long long)B * n * (H / KV);
    pl.rt_own = (n * (H / KV) + 15) / 16;
    pl.rt_pre = (int)((rows + 15) / 16);
    const auto pieces = [](long long want, long long items, long long keys) {
        const long long most = (keys + 127) / 128, s = want / items;
        return (int)(s < 1 ? 1 : s > most ? (most < 1 ? 1 : most) : s);
    };
    pl.So = pieces(want, (long long)B * KV * pl.rt_own, Tm);
    if (P > 0) {
        pl.tc = rows > 16 && win <= 0;
        if (pl.tc) {
            const int tiles = (P + 127) / 128, s = pieces(2LL * sm_count(), KV * ((rows + 127) / 128), P);
            pl.per = (tiles + s - 1) / s;
            pl.Sp = (tiles + pl.per - 1) / pl.per;
        } else
            pl.Sp = pieces(want, (long long)KV * pl.rt_pre, P);
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
    p.Sp = pl.Sp; p.So = pl.So; p.rt_own = pl.rt_own; p.rt_pre = pl.rt_pre;
    const long long own_items = (long long)B * KV * pl.rt_own * pl.So, items = own_items + (pl.tc ? 0 : (long long)KV * pl.rt_pre * pl.Sp);
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
    QLMB_CUDA(pdl_launch_small(k_px_mma, dim3((unsigned)items), dim3(128), 0, st, p));
    QLMB_LAUNCH_CHECK("k_px_mma");
    if (pl.Sp + pl.So > 1) {
        QLMB_CUDA(pdl_launch(true, k_px_join, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, p));
        QLMB_LAUNCH_CHECK("k_px_join");
    }
    return QLMB_OK;
}
