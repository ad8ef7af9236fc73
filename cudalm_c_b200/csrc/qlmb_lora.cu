// Low-rank adapters of many requests beside a projection that their rows share:
//   Y[m] = base[m] + s_a (X[m] A_a^T) B_a,   a = adapter[m] (-1: Y[m] = base[m]),   A [n][R][K], B [n][R][N] bf16.
//
// Products on mma.m16n8k16, operands from global memory as they lie there: of X and A a thread takes eight neighbouring elements of K
// where the instruction wants pairs (the order of a contracted dimension is free as long as both operands agree), of B eight
// neighbouring columns of each of its four inner indices, paired up by byte permutations.
// A row's products depend on no other row: a tile's rows are multiplied by each adapter that occurs among them, and only the
// adapter's own rows are kept.  With the rows in the order of their adapters (`order`) most tiles have one.
// The R inner numbers of a row are sums in fp32; they enter the second product as two bf16 terms (bf16 rows) or three (fp32 rows), and
// so does X where it is fp32: 16 and 24 bits.
//
#include <cuda.h>
#include <cuda_bf16.h>
#include <string.h>
#include "qlmb_common.cuh"
#include "qlmb_gemm.cuh"
#include "qlmb_attn.cuh"
#include "qlmb_internal.h"

namespace qlmb {

constexpr int LR_RT = 64;                     // inner columns made at a time
constexpr int LR_UP = 512;                    // output columns of a CTA of k_lora_one

struct LoraParams {
    void *Y;
    const void *X, *base;
    const bf16 *A, *Bm;
    const float *scale;
    const int *adapter, *order;
    float *part;                              // [S][M][R]
    int M, K, N, R, adapters, S, kslice;
    int *errword;
};

__device__ __forceinline__ void lr_mma(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x, y as pairs of bf16: the nearest to them, then the nearest to what that leaves, and so on.  Two terms hold 16 bits, three all 24.  LIMIT: above
// bf16's largest number (an infinity too) every term but the last is that number; without it what is left is inf - inf, a NaN.
template <int TERMS, bool LIMIT> __device__ __forceinline__ void lr_split(float x, float y, uint32_t t[TERMS])
{
    const __nv_bfloat162 top = __halves2bfloat162(__ushort_as_bfloat16(0x7f7f), __ushort_as_bfloat16(0x7f7f));
#pragma unroll
    for (int k = 0; k < TERMS; k++) {
        __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        if (LIMIT && k + 1 < TERMS) h = __hmin2(__hmax2(h, __hneg2(top)), top);
        t[k] = *reinterpret_cast<const uint32_t *>(&h);
        x -= __uint_as_float(t[k] << 16); y -= __uint_as_float(t[k] & 0xffff0000u);
    }
}
__device__ __forceinline__ uint32_t lt_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void lt_copy(uint32_t dst, const void *src, bool in)      // 16 bytes, zeros where !in
{ asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory"); }
__device__ __forceinline__ void lt_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void lt_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// Loads that stay where they are written and pass by L1: k_lora_up reads ahead of its wait.
__device__ __forceinline__ int lr_ldcg(const int *p) { int v; asm volatile("ld.global.cg.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory"); return v; }
__device__ __forceinline__ uint4 lr_ldcg(const uint4 *p)
{ uint4 v; asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory"); return v; }
// Row of place j (of the tile order) and its adapter; -1, -1 behind the last row or for an index out of range, which is reported.
__device__ __forceinline__ void lr_row(const LoraParams &p, int j, int &m, int &a, bool report)
{
    m = a = -1;
    if (j >= p.M) return;
    m = p.order ? lr_ldcg(p.order + j) : j;
    if (m < 0 || m >= p.M) { if (report) report_bad_index(p.errword, 307, j, m); m = -1; return; }
    a = lr_ldcg(p.adapter + m);
    if (a < -1 || a >= p.adapters) { if (report) report_bad_index(p.errword, 307, m, a); a = -1; }
}

// c += X A^T for 16 rows (m0: row g, m1: row g + 8 of the thread, -1 for none) and NT tiles of 8 inner columns, over steps of 32 of K:
// kb, kb + stride, ... below k1.  UK steps are loaded before the first is multiplied.
template <bool F32, int NT, int UK, bool LIMIT>
__device__ __forceinline__ void lr_down_pass(const LoraParams &p, float (&c)[NT][4], const bf16 *A, int ncol, int m0, int m1, int kb, int k1, int stride)
{
    constexpr int XT = F32 ? 3 : 1;
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    for (; kb < k1; kb += UK * stride) {
        uint4 x[UK][2][F32 ? 2 : 1], b[UK][NT];
#pragma unroll
        for (int u = 0; u < UK; u++) {
            const int kk = kb + u * stride + 8 * q;
            const bool in = kk < k1;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                b[u][t] = make_uint4(0, 0, 0, 0);
                if (in && 8 * t < ncol) b[u][t] = *reinterpret_cast<const uint4 *>(A + (size_t)(8 * t + g) * p.K + kk);
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int mm = e ? m1 : m0;
#pragma unroll
                for (int h = 0; h < (F32 ? 2 : 1); h++) {
                    x[u][e][h] = make_uint4(0, 0, 0, 0);
                    if (in && mm >= 0) {
                        if (F32) x[u][e][h] = reinterpret_cast<const uint4 *>(reinterpret_cast<const float *>(p.X) + (size_t)mm * p.K + kk)[h];
                        else x[u][e][h] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const bf16 *>(p.X) + (size_t)mm * p.K + kk);
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UK; u++) {
            uint32_t xs[XT][2][4];                       // [term][row half][pair]
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (F32) {
                    const uint32_t f[8] = {x[u][e][0].x, x[u][e][0].y, x[u][e][0].z, x[u][e][0].w, x[u][e][F32].x, x[u][e][F32].y, x[u][e][F32].z, x[u][e][F32].w};
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        uint32_t t[XT];
                        lr_split<XT, LIMIT>(__uint_as_float(f[2 * w]), __uint_as_float(f[2 * w + 1]), t);
#pragma unroll
                        for (int i = 0; i < XT; i++) xs[i][e][w] = t[i];
                    }
                } else { xs[0][e][0] = x[u][e][0].x; xs[0][e][1] = x[u][e][0].y; xs[0][e][2] = x[u][e][0].z; xs[0][e][3] = x[u][e][0].w; }
            }
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = XT - 1; i >= 0; i--) {
                    const uint32_t a0[4] = {xs[i][0][0], xs[i][1][0], xs[i][0][1], xs[i][1][1]}, a1[4] = {xs[i][0][2], xs[i][1][2], xs[i][0][3], xs[i][1][3]};
                    lr_mma(c[t], a0, b[u][t].x, b[u][t].y);
                    lr_mma(c[t], a1, b[u][t].z, b[u][t].w);
                }
        }
    }
}

// The same from c = 0.  fp32 rows whose sums are no numbers are taken once more with limited terms (limits at all times: 7 % of 8192 fp32 rows).
template <bool F32, int NT, int UK>
__device__ __forceinline__ void lr_down(const LoraParams &p, float (&c)[NT][4], const bf16 *A, int ncol, int m0, int m1, int kb, int k1, int stride)
{
    lr_down_pass<F32, NT, UK, false>(p, c, A, ncol, m0, m1, kb, k1, stride);
    if (!F32) return;
    bool odd = false;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int k = 0; k < 4; k++) odd |= c[t][k] != c[t][k];
    if (__builtin_expect(!__any_sync(~0u, odd), 1)) return;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int k = 0; k < 4; k++) c[t][k] = 0.0f;
    lr_down_pass<F32, NT, 1, true>(p, c, A, ncol, m0, m1, kb, k1, stride);
}

// Columns n0 .. n0 + 63 of 16 rows: base + T B.  A thread asks for B's rows r0 + 2 q, + 1, + 8, + 9, columns n0 + 8 g .. n0 + 8 g + 7.
template <bool CG> __device__ __forceinline__ void lr_up_b(const LoraParams &p, int cur, int n0, int r0, uint4 (&b)[4])
{
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const int r = r0 + 2 * q + (w & 1) + 8 * (w >> 1), n = n0 + 8 * g;
        b[w] = make_uint4(0, 0, 0, 0);
        if (cur >= 0 && n < p.N && r < p.R) {
            const uint4 *src = reinterpret_cast<const uint4 *>(p.Bm + ((size_t)cur * p.R + r) * p.N + n);
            b[w] = CG ? lr_ldcg(src) : *src;
        }
    }
}
// T as bf16 terms in shared memory: [term][row][ldt] pairs, t0 = the pairs of row g
template <bool F32> __device__ __forceinline__ void lr_up_mul(const LoraParams &p, float (&c)[8][4], const uint4 (&b)[4], const uint32_t *t0, int ldt, int r0)
{
    constexpr int TT = F32 ? 3 : 2;
    const int q = threadIdx.x & 3;
    uint32_t ta[TT][4];
#pragma unroll
    for (int i = 0; i < TT; i++)
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int e = 0; e < 2; e++) ta[i][2 * h + e] = r0 + 8 * h < p.R ? t0[(i * 16 + 8 * e) * ldt + (r0 + 8 * h) / 2 + q] : 0u;
    const uint32_t *b0 = &b[0].x, *b1 = &b[1].x, *b2 = &b[2].x, *b3 = &b[3].x;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
        const uint32_t x = __byte_perm(b0[j >> 1], b1[j >> 1], sel), y = __byte_perm(b2[j >> 1], b3[j >> 1], sel);
#pragma unroll
        for (int i = TT - 1; i >= 0; i--) lr_mma(c[j], ta[i], x, y);
    }
}
// columns 16 q .. 16 q + 15 of the warp's 64 end up with a thread, for its two rows; `keep`: which of them are this adapter's
template <bool F32> __device__ __forceinline__ void lr_up_base(const LoraParams &p, uint4 (&base)[2][2][F32 ? 2 : 1], int n0, const int (&mrow)[2], const bool (&keep)[2])
{
    const int q = threadIdx.x & 3;
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int col = n0 + 16 * q + 8 * h;
            if (keep[e] && col < p.N)
#pragma unroll
                for (int k = 0; k < (F32 ? 2 : 1); k++)
                    base[e][h][k] = reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(p.base) + ((size_t)mrow[e] * p.N + col) * (F32 ? 4 : 2))[k];
        }
}
template <bool F32> __device__ __forceinline__ void lr_up_store(const LoraParams &p, const float (&c)[8][4], const uint4 (&base)[2][2][F32 ? 2 : 1], int cur, int n0,
                                                                    const int (&mrow)[2], const bool (&keep)[2])
{
    const int q = threadIdx.x & 3;
#pragma unroll
    for (int e = 0; e < 2; e++) {
        if (!keep[e] || (cur < 0 && p.Y == p.base)) continue;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int col = n0 + 16 * q + 8 * h;
            if (col >= p.N) continue;
            uint32_t w[8];
            const uint32_t *s = &base[e][h][0].x, *s2 = &base[e][h][F32 ? 1 : 0].x;
#pragma unroll
            for (int k = 0; k < 4; k++) { w[k] = s[k]; w[4 + k] = s2[k]; }
            if (cur >= 0) {
                if (F32) {
#pragma unroll
                    for (int k = 0; k < 8; k++) w[k] = __float_as_uint(__uint_as_float(w[k]) + c[k][2 * e + h]);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const __nv_bfloat162 h2 = __floats2bfloat162_rn(__uint_as_float(w[k] << 16) + c[2 * k][2 * e + h], __uint_as_float(w[k] & 0xffff0000u) + c[2 * k + 1][2 * e + h]);
                        w[k] = *reinterpret_cast<const uint32_t *>(&h2);
                    }
                }
            }
            uint4 *d = reinterpret_cast<uint4 *>(reinterpret_cast<char *>(p.Y) + ((size_t)mrow[e] * p.N + col) * (F32 ? 4 : 2));
            d[0] = make_uint4(w[0], w[1], w[2], w[3]);
            if (F32) d[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    }
}
template <bool F32> __device__ __forceinline__ void lr_up(const LoraParams &p, float (&c)[8][4], const uint32_t *t0, int ldt, int cur, int n0)
{
#pragma unroll 2
    for (int r0 = 0; r0 < p.R; r0 += 16) {
        uint4 b[4];
        lr_up_b<false>(p, cur, n0, r0, b);
        lr_up_mul<F32>(p, c, b, t0, ldt, r0);
    }
}

// ---- many rows that are fp32, out of order or of another rank.  A CTA of eight warps (four row groups of 16 times two halves of 32 columns) has 64 rows: the products' operands come
// through a ring of four stages in shared memory, a stage being 64 x 64 elements of X (or of the base) and of A (or B), in 16-byte
// pieces whose place is turned by the row.  First the inner numbers over K, 64 at a time, kept as bf16 terms; then Y, 64 columns at a
// time: the base lies in the stage, the sum takes its place there and leaves in whole pieces.
constexpr int LT_M = 64, LT_NS = 4, LT_W = 64 * 64 * 2;      // rows, stages, bytes of a stage's weights
template <bool F32> constexpr int lt_x() { return LT_M * 64 * (F32 ? 4 : 2); }
template <bool F32> static size_t lt_smem(int R) { return (size_t)LT_NS * (lt_x<F32>() + LT_W) + (size_t)(F32 ? 3 : 2) * LT_M * ((R + 15) / 16 * 8 + 4) * sizeof(uint32_t); }

__device__ __forceinline__ void lt_ldm(uint32_t a, uint32_t v[4])
{ asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory"); }
__device__ __forceinline__ void lt_ldmt(uint32_t a, uint32_t v[4])
{ asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory"); }

// SMALL (R <= 64): a warp keeps the terms of its 16 rows in registers while it goes through the columns.
// blockIdx.z: a tile's adapters are dealt out to LT_Z CTAs, so that the tiles at the border of two prompts take no longer than the others.
constexpr int LT_Z = 4;
template <bool B> struct LtFlag { static constexpr bool value = B; };
template <bool F32, bool SMALL> __global__ void __launch_bounds__(256, 2) k_lora_tile(const __grid_constant__ LoraParams p)
{
    constexpr int XT = F32 ? 3 : 1, TT = F32 ? 3 : 2, XB = lt_x<F32>(), STAGE = XB + LT_W, XP = F32 ? 16 : 8, EB = F32 ? 4 : 2;   // XP: pieces of a row of 64
    extern __shared__ __align__(128) uint8_t lt_s[];
    __shared__ int srow[LT_M];                            // the rows of the present adapter, -1 for the others
    uint32_t *ts = reinterpret_cast<uint32_t *>(lt_s + LT_NS * STAGE);       // [term][row][ldt] pairs of bf16
    const int ldt = (p.R + 15) / 16 * 8 + 4;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3, rg = (warp >> 1) * 16, nh = (warp & 1) * 32;
    pdl_trigger();
    pdl_wait();
    const int j0 = blockIdx.x * LT_M;
    int m[2], a[2];                                       // rows lane and lane + 32
#pragma unroll
    for (int e = 0; e < 2; e++) lr_row(p, j0 + lane + 32 * e, m[e], a[e], blockIdx.y == 0 && blockIdx.z == 0 && warp == 0);
    const int per = (p.N + 64 * gridDim.y - 1) / (64 * gridDim.y) * 64, c0 = blockIdx.y * per, c1 = min(p.N, c0 + per);
    if (c0 >= p.N) return;
    unsigned todo[2] = {__ballot_sync(~0u, a[0] >= 0), __ballot_sync(~0u, a[1] >= 0)};
    for (int nth = 0; todo[0] | todo[1]; nth++) {
        const int cur = todo[0] ? __shfl_sync(~0u, a[0], __ffs(todo[0]) - 1) : __shfl_sync(~0u, a[1], __ffs(todo[1]) - 1);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            todo[e] &= ~__ballot_sync(~0u, a[e] == cur);
            if (warp == 0 && nth % LT_Z == blockIdx.z) srow[lane + 32 * e] = a[e] == cur ? m[e] : -1;
        }
        if (nth % LT_Z != blockIdx.z) continue;
        __syncthreads();
        const float scale = p.scale[cur];
        const bf16 *A = p.A + (size_t)cur * p.R * p.K, *Bm = p.Bm + (size_t)cur * p.R * p.N;
        // A thread's pieces of a stage are the same in every step: rows xr + 256 / XP i of X (or the base), rows wr + 32 i of A (or B).
        constexpr int NX = LT_M * XP / 256;
        const int xr = tid / XP, xc = tid % XP, wr = tid >> 3, wc = tid & 7;
        const uint32_t s0 = lt_addr(lt_s), xd = s0 + xr * (XP * 16) + ((xc ^ (xr & 7)) << 4), wd = s0 + XB + wr * 128 + ((wc ^ (wr & 7)) << 4);
        int xrow[NX];
#pragma unroll
        for (int i = 0; i < NX; i++) xrow[i] = srow[xr + 256 / XP * i];
        // ---- inner numbers: 64 of K at a time, block of 64 inner columns by block
        int lrc, lk, ls;                                  // the next step to be requested, and its stage
        const auto load1 = [&]() {
            if (lrc < p.R) {
                const int k = lk + xc * (16 / EB), kw = lk + wc * 8;
                const uint32_t so = ls * STAGE;
#pragma unroll
                for (int i = 0; i < NX; i++) {
                    const bool in = xrow[i] >= 0 && k < p.K;
                    lt_copy(xd + so + i * (256 * 16), reinterpret_cast<const uint8_t *>(p.X) + (in ? ((size_t)xrow[i] * p.K + k) * EB : 0), in);
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int r = lrc + wr + 32 * i;
                    const bool in = r < p.R && kw < p.K;
                    lt_copy(wd + so + i * (32 * 128), A + (in ? (size_t)r * p.K + kw : 0), in);
                }
                lk += 64;
                if (lk >= p.K) { lk = 0; lrc += 64; }
            }
            ls = (ls + 1) % LT_NS;
            lt_commit();
        };
        float c[4][4] = {};
        const auto inner = [&](auto limit) {              // true where a sum is no number
            lrc = lk = ls = 0;
            for (int st = 0; st < LT_NS - 1; st++) load1();
            bool odd = false;
            for (int st = 0, rc = 0, k0 = 0; rc < p.R; st = (st + 1) % LT_NS) {
                lt_wait<LT_NS - 2>();
                __syncthreads();                              // the step has landed for everyone, and everyone is done with the one before
                load1();
                const uint8_t *sx = lt_s + st * STAGE, *sw = sx + XB;
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    uint32_t x[XT][4], w[2][4];
                    if (F32) {
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                const int r = rg + g + 8 * e, k = 16 * s + 8 * h + 2 * q;
                                const float2 f = *reinterpret_cast<const float2 *>(sx + r * 256 + (((k >> 2) ^ (r & 7)) << 4) + (k & 3) * 4);
                                uint32_t t[XT];
                                lr_split<XT, decltype(limit)::value>(f.x, f.y, t);
#pragma unroll
                                for (int i = 0; i < XT; i++) x[i][2 * h + e] = t[i];
                            }
                    } else {
                        const int r = rg + (lane & 15), cc = 2 * s + (lane >> 4);
                        lt_ldm(lt_addr(sx + r * 128 + ((cc ^ (r & 7)) << 4)), x[0]);
                    }
#pragma unroll
                    for (int t = 0; t < 2; t++) {             // two tiles of 8 inner columns: rows of A, their 16 elements of K in two pieces
                        const int r = nh + 16 * t + (lane & 7) + 8 * (lane >> 4), cc = 2 * s + ((lane >> 3) & 1);
                        lt_ldm(lt_addr(sw + r * 128 + ((cc ^ (r & 7)) << 4)), w[t]);
                    }
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = XT - 1; i >= 0; i--) lr_mma(c[t], x[i], w[t >> 1][2 * (t & 1)], w[t >> 1][2 * (t & 1) + 1]);
                }
                k0 += 64;
                if (k0 >= p.K) {                              // the block's sums are whole
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const int col = rc + nh + 8 * t;
                        if (col < p.R)
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                uint32_t v[TT];
                                lr_split<TT, true>(c[t][2 * e] * scale, c[t][2 * e + 1] * scale, v);
#pragma unroll
                                for (int i = 0; i < TT; i++) ts[(i * LT_M + rg + g + 8 * e) * ldt + col / 2 + q] = v[i];
                            }
#pragma unroll
                        for (int k = 0; k < 4; k++) { odd |= c[t][k] != c[t][k]; c[t][k] = 0.0f; }
                    }
                    k0 = 0; rc += 64;
                }
            }
            lt_wait<0>();
            return __syncthreads_or(odd);
        };
        if (inner(LtFlag<false>()) && F32) inner(LtFlag<true>());        // (as in lr_down)
        // ---- Y: 64 inner indices at a time, block of 64 columns by block; the base comes with a block's last step
        int ln = c0;
        lrc = 0; ls = 0;
        const auto load2 = [&]() {
            if (ln < c1) {
                const int n = ln + xc * (16 / EB), nw = ln + wc * 8;
                const uint32_t so = ls * STAGE;
                if (lrc + 64 >= p.R && n < c1)
#pragma unroll
                    for (int i = 0; i < NX; i++)
                        if (xrow[i] >= 0) lt_copy(xd + so + i * (256 * 16), reinterpret_cast<const uint8_t *>(p.base) + ((size_t)xrow[i] * p.N + n) * EB, true);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int r = lrc + wr + 32 * i;
                    const bool in = r < p.R && nw < c1;
                    lt_copy(wd + so + i * (32 * 128), Bm + (in ? (size_t)r * p.N + nw : 0), in);
                }
                lrc += 64;
                if (lrc >= p.R) { lrc = 0; ln += 64; }
            }
            ls = (ls + 1) % LT_NS;
            lt_commit();
        };
        for (int st = 0; st < LT_NS - 1; st++) load2();
        const auto terms = [&](int r0, uint32_t (&x)[TT][4]) {            // 16 inner numbers of rows g and g + 8 as an A operand
#pragma unroll
            for (int i = 0; i < TT; i++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int e = 0; e < 2; e++) x[i][2 * h + e] = r0 + 8 * h < p.R ? ts[(i * LT_M + rg + g + 8 * e) * ldt + (r0 + 8 * h) / 2 + q] : 0u;
        };
        uint32_t held[SMALL ? 4 : 1][TT][4];
        if (SMALL)
#pragma unroll
            for (int s = 0; s < 4; s++) terms(16 * s, held[SMALL ? s : 0]);
        for (int st = 0, rc = 0, n0 = c0; n0 < c1; st = (st + 1) % LT_NS) {
            lt_wait<LT_NS - 2>();
            __syncthreads();
            load2();
            uint8_t *sx = lt_s + st * STAGE;
            const uint8_t *sw = sx + XB;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                if (rc + 16 * s >= p.R) break;
                uint32_t w[2][4];
                if (!SMALL) terms(rc + 16 * s, held[0]);
                const uint32_t (&x)[TT][4] = held[SMALL ? s : 0];
#pragma unroll
                for (int t = 0; t < 2; t++) {             // two tiles of 8 columns: 16 rows of B
                    const int r = 16 * s + (lane & 15), cc = (nh >> 3) + 2 * t + (lane >> 4);
                    lt_ldmt(lt_addr(sw + r * 128 + ((cc ^ (r & 7)) << 4)), w[t]);
                }
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = TT - 1; i >= 0; i--) lr_mma(c[t], x[i], w[t >> 1][2 * (t & 1)], w[t >> 1][2 * (t & 1) + 1]);
            }
            rc += 64;
            if (rc >= p.R) {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int r = rg + g + 8 * e, col = nh + 8 * t + 2 * q;
                        uint8_t *d = sx + r * (XP * 16) + (((col * EB >> 4) ^ (r & 7)) << 4) + (col * EB & 15);
                        if (F32) {
                            float2 *f = reinterpret_cast<float2 *>(d);
                            *f = make_float2(f->x + c[t][2 * e], f->y + c[t][2 * e + 1]);
                        } else {
                            const uint32_t v = *reinterpret_cast<const uint32_t *>(d);
                            const __nv_bfloat162 h2 = __floats2bfloat162_rn(__uint_as_float(v << 16) + c[t][2 * e], __uint_as_float(v & 0xffff0000u) + c[t][2 * e + 1]);
                            *reinterpret_cast<uint32_t *>(d) = *reinterpret_cast<const uint32_t *>(&h2);
                        }
                        c[t][2 * e] = c[t][2 * e + 1] = 0.0f;
                    }
                __syncwarp();                             // the warp's own 16 x 32 numbers
#pragma unroll
                for (int i = lane; i < 16 * XP / 2; i += 32) {
                    const int r = rg + i / (XP / 2), cc = nh * EB / 16 + i % (XP / 2), row = srow[r], n = n0 + cc * (16 / EB);
                    if (row >= 0 && n < c1)
                        *reinterpret_cast<uint4 *>(reinterpret_cast<uint8_t *>(p.Y) + ((size_t)row * p.N + n) * EB) =
                            *reinterpret_cast<const uint4 *>(sx + r * (XP * 16) + ((cc ^ (r & 7)) << 4));
                }
                rc = 0; n0 += 64;
            }
        }
        lt_wait<0>();
        __syncthreads();
    }
    // rows without an adapter
    if (p.Y != p.base && blockIdx.z == 0)
        for (int r = warp; r < LT_M; r += 8) {
            const int row = __shfl_sync(~0u, r < 32 ? m[0] : m[1], r & 31), ad = __shfl_sync(~0u, r < 32 ? a[0] : a[1], r & 31);
            if (row < 0 || ad >= 0) continue;
            for (int n = c0 + lane * (16 / EB); n < c1; n += 32 * (16 / EB))
                *reinterpret_cast<uint4 *>(reinterpret_cast<uint8_t *>(p.Y) + ((size_t)row * p.N + n) * EB) =
                    *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(p.base) + ((size_t)row * p.N + n) * EB);
        }
}

// ---- many neighbouring rows in bf16, ranks of whole 16: tcgen05.  A pair is a tile of 128 rows and an adapter that occurs in it (rows without
// one, where Y is not the base, are such a pair, too); the pairs' blocks of 64 columns are dealt out evenly to the CTAs, one an SM.
//
//   warp 0      TMA into a ring of stages of 64 columns: X and A along K, then the base and B along N
//   warp 1      D = X A^T (128 x R), then for every block T B (128 x 64, T as two bf16 terms in tensor memory)
//   warps 2-9   D to T; of a block two groups of four warps take turns: a thread has a row, adds the sum to its base in the stage, and
//               the warp's rows leave by TMA (by plain stores where some are another adapter's)
//
// Tensor memory: T in columns 0 and 128, D in 256, which the blocks' sums (four of 64 columns) take over once D is read.
//
// 8192 rows on 9 adapters, K 768, N 1536, R 64: 22.6 us (63 MB, 2.8 TB/s; 64-row tiles on mma.sync 32.7).  Of a CTA's 27 k cycles in front of
// its end: counting adapters 5 k, the first pair's walk and copies 4 k, 12 steps of K 6 k (511 a step of 24 KB, what an SM gets from L2
// when all ask), D to T 2 k, 12 blocks 10 k.  Rows leaving by plain stores instead of TMA: 23.7; a fence behind those stores, which it
// then waits for: 26.
constexpr int LC_T = 320, LC_TILES = 8192, LC_NS = 8;
struct LcParams { alignas(64) CUtensorMap x_map, a_map, base_map, b_map, y_map; LoraParams l; int stages; };
static int lc_stage(int R) { return 128 * 128 + R * 128; }
static size_t lc_smem(int R, int stages) { return (size_t)stages * lc_stage(R) + LC_TILES + 512; }
static int lc_stages(int R) { const int s = (226 * 1024 - LC_TILES - 512) / lc_stage(R); return s < LC_NS ? s : LC_NS; }

// A warp's way through the pairs: the tile's adapters (row 32 k + lane), those that are still to come
struct LcWalk { int t, cur, a[4]; unsigned todo[4]; };
__device__ __forceinline__ void lc_ask(const LoraParams &p, int t, int (&a)[4])
{
#pragma unroll
    for (int k = 0; k < 4; k++) { const int row = 128 * t + 32 * k + (threadIdx.x & 31); a[k] = row < p.M ? p.adapter[row] : -2; }
}
__device__ __forceinline__ void lc_open(const LoraParams &p, LcWalk &w, const int (&v)[4], bool report)
{
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int row = 128 * w.t + 32 * k + (threadIdx.x & 31);
        w.a[k] = v[k];
        if (row < p.M && (v[k] < -1 || v[k] >= p.adapters)) { if (report) report_bad_index(p.errword, 307, row, v[k]); w.a[k] = -1; }
        if (w.a[k] == -1 && p.Y == p.base) w.a[k] = -2;
        w.todo[k] = __ballot_sync(~0u, w.a[k] != -2);
    }
}
__device__ __forceinline__ bool lc_pick(LcWalk &w)        // the tile's next adapter
{
    if (!(w.todo[0] | w.todo[1] | w.todo[2] | w.todo[3])) return false;
    const unsigned t = w.todo[0] ? w.todo[0] : w.todo[1] ? w.todo[1] : w.todo[2] ? w.todo[2] : w.todo[3];
    const int v = w.todo[0] ? w.a[0] : w.todo[1] ? w.a[1] : w.todo[2] ? w.a[2] : w.a[3];
    w.cur = __shfl_sync(~0u, v, __ffs(t) - 1);
#pragma unroll
    for (int k = 0; k < 4; k++) w.todo[k] &= ~__ballot_sync(~0u, w.a[k] == w.cur);
    return true;
}

__global__ void __launch_bounds__(LC_T, 1) k_lora_tc(const __grid_constant__ LcParams cp)
{
    extern __shared__ __align__(1024) uint8_t lc_s[];
    const LoraParams &p = cp.l;
    const int NS = cp.stages, STAGE = 128 * 128 + p.R * 128;
    uint8_t *cnt = lc_s + (size_t)NS * STAGE;             // adapters of a tile
    uint64_t *bars = reinterpret_cast<uint64_t *>(cnt + LC_TILES);
    uint64_t *full = bars, *empty = bars + LC_NS, *d2_full = empty + LC_NS, *d2_empty = d2_full + 4, *d1_full = d2_empty + 4, *t_full = d1_full + 1, *spare = t_full + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(spare + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *sum = const_cast<int *>(abort_flag) + 1, *begin = sum + 1;                  // pairs; the CTA's first tile, and pairs of it before the first
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (smem_u32(lc_s) & 1023u) {             // the swizzled tiles need a 1 KiB-aligned base
        if (tid == 0 && p.errword && atomicCAS(p.errword, 0, 201) == 0) { p.errword[1] = 160; p.errword[2] = (int)blockIdx.x; }
        pdl_wait();
        return;
    }
    if (tid == 0) {
        prefetch_map(&cp.x_map); prefetch_map(&cp.a_map); prefetch_map(&cp.base_map); prefetch_map(&cp.b_map);
        for (int i = 0; i < NS; i++) { mbar_init(smem_u32(&full[i]), 1); mbar_init(smem_u32(&empty[i]), 4); }
        for (int i = 0; i < 4; i++) { mbar_init(smem_u32(&d2_full[i]), 1); mbar_init(smem_u32(&d2_empty[i]), 4); }
        mbar_init(smem_u32(d1_full), 1);
        mbar_init(smem_u32(t_full), 8);
        mbar_init(smem_u32(spare), 1);
        *abort_flag = 0;
        *sum = 0; begin[0] = begin[1] = 0;
        fence_barrier_init();
    }
    if (warp == 0) { tmem_alloc(smem_u32(tmem_slot), 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();                               // barriers and TMEM above are this kernel's own; its inputs come below
    pdl_trigger();
    // ---- the tiles' adapters are counted, and the CTA's share found
    const int tiles = (p.M + 127) / 128, blocks = (p.N + 63) / 64;
    LcWalk w;
    {
        int mine = 0;
        for (int t = warp; t < tiles; t += 4 * (LC_T / 32)) {             // four tiles a warp at a time
            int v[4][4];
#pragma unroll
            for (int i = 0; i < 4; i++) lc_ask(p, t + i * (LC_T / 32), v[i]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                w.t = t + i * (LC_T / 32);
                if (w.t >= tiles) break;
                int n = 1;
                const int one = __shfl_sync(~0u, v[i][0], 0);             // mostly there is one adapter
                if (!__all_sync(~0u, v[i][0] == one && v[i][1] == one && v[i][2] == one && v[i][3] == one) || one < 0 || one >= p.adapters) {
                    lc_open(p, w, v[i], blockIdx.x == 0);
                    for (n = 0; lc_pick(w);) n++;
                }
                if (lane == 0) cnt[w.t] = (uint8_t)n;
                mine += n;
            }
        }
        if (lane == 0 && mine) atomicAdd(sum, mine);
    }
    __syncthreads();
    // (below 2^31, and in 32 bits: divisions in 64 took 1.2 us)
    const int units = *sum * blocks, share = units / (int)gridDim.x, over = units - share * (int)gridDim.x, me = blockIdx.x;
    const int u0 = share * me + min(me, over), u1 = u0 + share + (me < over), pair0 = u0 / blocks;
    if (warp == 0 && u0 < u1) {
        int before = 0;
        for (int t0 = 0; t0 < tiles; t0 += 32) {
            const int n = t0 + lane < tiles ? cnt[t0 + lane] : 0;
            int x = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(~0u, x, o); if (lane >= o) x += y; }
            const int at = before + x - n;
            if (at <= pair0 && pair0 < at + n) { begin[0] = t0 + lane; begin[1] = pair0 - at; }
            before += __shfl_sync(~0u, x, 31);
            if (before > pair0) break;
        }
    }
    __syncthreads();
    const uint32_t tT = *tmem_slot, tD = tT + 256;
    // the next pair, and its blocks b0 .. b1 - 1
    int u = u0, b0 = 0, b1 = 0, bad = 0, ask[4];
    const auto next = [&]() {
        if (u >= u1) return false;
        if (u == u0) {
            w.t = begin[0];
            lc_ask(p, w.t, ask);
            lc_open(p, w, ask, false);
            for (int i = begin[1]; i >= 0; i--) lc_pick(w);
            b0 = u0 - pair0 * blocks;
        } else {
            b0 = 0;
            if (!lc_pick(w)) {
                do w.t++; while (w.t + 1 < tiles && cnt[w.t] == 0);
                lc_ask(p, w.t, ask);
                lc_open(p, w, ask, false);
                lc_pick(w);
            }
        }
        b1 = min(blocks, b0 + u1 - u);
        u += b1 - b0;
        return true;
    };
    const int steps = (p.K + 63) / 64;
    int s = 0;                                // the stage, and how often the ring was gone through
    uint32_t phase = 0;
    const auto advance = [&](int n) { for (s += n; s >= NS; s -= NS) phase ^= 1; };

    if (warp == 0) {
        int issued = 0;
        while (!bad && next()) {
            const int n = (w.cur >= 0 ? steps : 0) + b1 - b0;
            for (int i = 0; i < n; i++) {
                if ((bad = at_all_wait(smem_u32(&empty[s]), phase ^ 1u, abort_flag, 161))) break;
                const bool inner = w.cur >= 0 && i < steps;
                const int x = 64 * (inner ? i : b0 + i - (w.cur >= 0 ? steps : 0));
                if (elect_one()) {
                    const uint32_t bar = smem_u32(&full[s]), d = smem_u32(lc_s + s * STAGE);
                    mbar_expect_tx(bar, w.cur >= 0 ? STAGE : 128 * 128);
                    tma_load_2d(d, inner ? &cp.x_map : &cp.base_map, bar, x, 128 * w.t);
                    if (w.cur >= 0) tma_load_2d(d + 128 * 128, inner ? &cp.a_map : &cp.b_map, bar, x, w.cur * p.R);
                }
                __syncwarp();
                issued++;
                advance(1);
            }
        }
        at_give_up(bad, abort_flag, p.errword);
        if (*abort_flag)                      // copies under way end (bounded) before memory is given back
            for (int i = issued > NS ? issued - NS : 0; i < issued; i++)
                for (uint32_t k = 0; k < AT_WAIT_LIMIT && !at_test(smem_u32(&full[i % NS]), (uint32_t)(i / NS) & 1u); k++) {}
    } else if (warp == 1) {
        const uint32_t IDESC_D = make_idesc(128, p.R, 0, 0);
        constexpr uint32_t IDESC_Y = make_idesc(128, 64, 0, 1);
        const uint64_t x00 = make_desc(smem_u32(lc_s), 16, 1024), a00 = make_desc(smem_u32(lc_s) + 128 * 128, 16, 1024), b00 = make_desc(smem_u32(lc_s) + 128 * 128, 8192, 1024);
        int nb = 0, np = 0;                   // blocks, pairs with an adapter
        while (!bad && next()) {
            const bool adapted = w.cur >= 0;
            for (int k = 0; k < 4 && !bad && adapted; k++) {             // D takes the place of the last pair's sums
                const int uses = (nb - k + 3) / 4;
                if (uses > 0) bad = at_all_wait(smem_u32(&d2_empty[k]), (uint32_t)(uses - 1) & 1u, abort_flag, 162);
            }
            for (int i = 0; i < steps && !bad && adapted; i++) {
                if ((bad = at_all_wait(smem_u32(&full[s]), phase, abort_flag, 163))) break;
                tc_fence_after();
                const uint64_t o = (uint64_t)(s * (STAGE / 16));
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; k++) tc_mma_bf16(tD, x00 + o + 2 * k, a00 + o + 2 * k, IDESC_D, i > 0 || k > 0);
                    for (int k = 0; k < 3; k++) mbar_arrive(smem_u32(&empty[s]));    // (a block's stage is given back by four warps)
                    tc_commit(smem_u32(&empty[s]));
                    if (i + 1 == steps) tc_commit(smem_u32(d1_full));
                }
                __syncwarp();
                advance(1);
            }
            if (bad || (adapted && (bad = at_all_wait(smem_u32(t_full), (uint32_t)np & 1u, abort_flag, 164)))) break;
            if (adapted) np++;
            // Blocks without an adapter, too, go through here: a wait tells a stage's turn from the one two before it only if the warp saw
            // the one in between.
            for (int b = b0; b < b1; b++, nb++) {
                const int buf = nb & 3;
                if ((bad = at_all_wait(smem_u32(&full[s]), phase, abort_flag, 165))) break;
                if (nb >= 4 && (bad = at_all_wait(smem_u32(&d2_empty[buf]), (uint32_t)(nb / 4 - 1) & 1u, abort_flag, 166))) break;
                tc_fence_after();
                const uint64_t o = (uint64_t)(s * (STAGE / 16));
                if (elect_one()) {
                    if (adapted) {
                        for (int k = 0; k < p.R / 16; k++) {
                            tc_mma_bf16_ta(tD + 64 * buf, tT + k * 8, b00 + o + 128 * k, IDESC_Y, k > 0);
                            tc_mma_bf16_ta(tD + 64 * buf, tT + 128 + k * 8, b00 + o + 128 * k, IDESC_Y, 1);
                        }
                        tc_commit(smem_u32(&d2_full[buf]));
                    } else mbar_arrive(smem_u32(&d2_full[buf]));
                }
                __syncwarp();
                advance(1);
            }
        }
        at_give_up(bad, abort_flag, p.errword);
        if (*abort_flag) {                    // MMAs under way end (bounded) before memory is given back
            if (elect_one()) tc_commit(smem_u32(spare));
            __syncwarp();
            for (uint32_t k = 0; k < AT_WAIT_LIMIT && !at_test(smem_u32(spare), 0); k++) {}
        }
    } else {
        // a warp reaches the 32 lanes of tensor memory that its place in the warpgroup gives it
        const int quarter = warp & 3, group = (warp - 2) >> 2, r = 32 * quarter + lane;
        const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
        int nb = 0, np = 0;
        while (!bad && next()) {
            const bool adapted = w.cur >= 0;
            const int own = quarter == 0 ? w.a[0] : quarter == 1 ? w.a[1] : quarter == 2 ? w.a[2] : w.a[3];
            const unsigned keep = __ballot_sync(~0u, own == w.cur);
            const bool whole = keep == __ballot_sync(~0u, 128 * w.t + r < p.M);      // (rows behind the last are not stored)
            if (adapted) {
                const float scale = p.scale[w.cur];
                if ((bad = at_all_wait(smem_u32(d1_full), (uint32_t)np & 1u, abort_flag, 167))) break;
                np++;
                tc_fence_after();
                for (int c = 32 * group; c < p.R; c += 64) {             // (columns from R on are read and written, not used)
                    uint32_t v[32], hi[16], lo[16];
                    tmem_ld32(tD + lanes + c, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        uint32_t t[2];
                        lr_split<2, true>(__uint_as_float(v[2 * k]) * scale, __uint_as_float(v[2 * k + 1]) * scale, t);
                        hi[k] = t[0]; lo[k] = t[1];
                    }
                    tmem_st16(tT + lanes + c / 2, hi);
                    tmem_st16(tT + 128 + lanes + c / 2, lo);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(t_full));
                advance(steps);
            }
            for (int b = b0; b < b1; b++, nb++) {
                const int buf = nb & 3;
                if ((nb & 1) != group) { advance(1); continue; }
                // (the sum first: then the stage has its turn, which the group alone, seeing every second one, could not tell from an earlier one)
                if ((bad = at_all_wait(smem_u32(&d2_full[buf]), (uint32_t)(nb / 4) & 1u, abort_flag, 168))) break;
                if ((bad = at_all_wait(smem_u32(&full[s]), phase, abort_flag, 169))) break;
                uint8_t *tile = lc_s + s * STAGE;
                if (adapted && keep) {
                    tc_fence_after();
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t v[32];
                        tmem_ld32(tD + 64 * buf + lanes + 32 * h, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            uint4 *d = reinterpret_cast<uint4 *>(tile + r * 128 + (((4 * h + c) ^ (r & 7)) << 4));
                            uint4 x = *d;
                            uint32_t *e = &x.x;
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const __nv_bfloat162 h2 = __floats2bfloat162_rn(__uint_as_float(e[k] << 16) + __uint_as_float(v[8 * c + 2 * k]),
                                                                                __uint_as_float(e[k] & 0xffff0000u) + __uint_as_float(v[8 * c + 2 * k + 1]));
                                e[k] = *reinterpret_cast<const uint32_t *>(&h2);
                            }
                            *d = x;
                        }
                    }
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&d2_empty[buf]));
                if (whole) {
                    fence_proxy_async();
                    __syncwarp();
                    if (keep && elect_one()) {
                        tma_store_2d(&cp.y_map, smem_u32(tile + 32 * quarter * 128), 64 * b, 128 * w.t + 32 * quarter);
                        bulk_commit();
                        bulk_wait_read();
                    }
                } else {
                    uint4 out[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int rr = 32 * quarter + 4 * i + (lane >> 3);
                        out[i] = *reinterpret_cast<const uint4 *>(tile + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
                    }
                    fence_proxy_async();                  // the next copy comes after these reads and writes (the fence waits for stores to Y, too)
                    bf16 *y = reinterpret_cast<bf16 *>(p.Y) + (size_t)(128 * w.t + 32 * quarter + (lane >> 3)) * p.N + 64 * b + 8 * (lane & 7);
                    if (64 * b + 8 * (lane & 7) < p.N)
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            if (keep >> (4 * i + (lane >> 3)) & 1) *reinterpret_cast<uint4 *>(y + (size_t)(4 * i) * p.N) = out[i];
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&empty[s]));
                advance(1);
            }
        }
        if (elect_one()) bulk_wait_all();
        __syncwarp();
        at_give_up(bad, abort_flag, p.errword);
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 0) { tc_fence_after(); tmem_dealloc(tT, 512); }
}

// ---- few rows, small adapters: one launch.  blockIdx.x = 16 tile + place: the CTA of a place that is the first of its adapter in the
// tile does that adapter's rows, every block of columns making the inner numbers for itself.  Eight warps share K, then the columns.
template <bool F32, int NT, int UK> __global__ void __launch_bounds__(256) k_lora_one(const __grid_constant__ LoraParams p)
{
    constexpr int TT = F32 ? 3 : 2;
    __shared__ float red[8][16][8 * NT + 2];
    __shared__ uint32_t ts[TT * 16 * (4 * NT + 4)];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3, ldt = (p.R + 15) / 16 * 8 + 4;
    pdl_trigger();
    pdl_wait();
    const int j0 = (int)blockIdx.x / 16 * 16, place = blockIdx.x % 16;
    int m, a;
    lr_row(p, j0 + (lane & 15), m, a, blockIdx.y == 0 && place == 0 && threadIdx.x < 16);
    const int cur = __shfl_sync(~0u, a, place);
    const unsigned mine = __ballot_sync(~0u, m >= 0 && a == cur) & 0xffffu;
    if (__ffs(mine) - 1 != place) return;
    const int rows[2] = {__shfl_sync(~0u, m, g), __shfl_sync(~0u, m, g + 8)};
    const bool keep[2] = {(mine >> g & 1) != 0, (mine >> (g + 8) & 1) != 0};
    if (cur >= 0) {
        float c[NT][4] = {};
        lr_down<F32, NT, UK>(p, c, p.A + (size_t)cur * p.R * p.K, p.R, keep[0] ? rows[0] : -1, keep[1] ? rows[1] : -1, 32 * warp, p.K, 256);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            *reinterpret_cast<float2 *>(&red[warp][g][8 * t + 2 * q]) = make_float2(c[t][0], c[t][1]);
            *reinterpret_cast<float2 *>(&red[warp][g + 8][8 * t + 2 * q]) = make_float2(c[t][2], c[t][3]);
        }
        __syncthreads();
        const float scale = p.scale[cur];
        for (int i = threadIdx.x; i < 16 * p.R / 2; i += 256) {
            const int r = i / (p.R / 2), col = 2 * (i % (p.R / 2));
            float x = 0.0f, y = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; k++) { const float2 v = *reinterpret_cast<const float2 *>(&red[k][r][col]); x += v.x; y += v.y; }
            uint32_t t[TT];
            lr_split<TT, true>(x * scale, y * scale, t);
#pragma unroll
            for (int k = 0; k < TT; k++) ts[(k * 16 + r) * ldt + col / 2] = t[k];
        }
        __syncthreads();
    }
    const int n1 = min(p.N, ((int)blockIdx.y + 1) * LR_UP);
    for (int n0 = blockIdx.y * LR_UP + 64 * warp; n0 < n1; n0 += 512) {
        uint4 base[2][2][F32 ? 2 : 1];
        lr_up_base<F32>(p, base, n0, rows, keep);
        float c[8][4] = {};
        if (cur >= 0) lr_up<F32>(p, c, ts + g * ldt, ldt, cur, n0);
        lr_up_store<F32>(p, c, base, cur, n0, rows, keep);
    }
}

// ---- few rows, large adapters: two launches, CTAs of places again; first the inner numbers in slices of K, then blocks of columns.
// (64 inner columns: two steps at a time of fp32 rows, 64.9 to 46.6 us at K 4040; of bf16 rows, 22.2 to 32.4 at K 4096, one.)
template <bool F32, int NT, int UK> __global__ void __launch_bounds__(128) k_lora_down(const __grid_constant__ LoraParams p)
{
    __shared__ float red[4][16][8 * NT + 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    pdl_wait();                               // ahead of the trigger: what ran before has ended when k_lora_up starts
    pdl_trigger();
    const int j0 = (int)blockIdx.x / 16 * 16, place = blockIdx.x % 16, r0 = blockIdx.z * (8 * NT), k0 = blockIdx.y * p.kslice, k1 = min(p.K, k0 + p.kslice);
    int m, a;
    lr_row(p, j0 + (lane & 15), m, a, blockIdx.y == 0 && blockIdx.z == 0 && place == 0 && threadIdx.x < 16);
    const int cur = __shfl_sync(~0u, a, place);
    const unsigned mine = __ballot_sync(~0u, a == cur) & 0xffffu;
    if (cur < 0 || __ffs(mine) - 1 != place) return;
    const int ra = __shfl_sync(~0u, m, g), rb = __shfl_sync(~0u, m, g + 8);
    float c[NT][4] = {};
    lr_down<F32, NT, UK>(p, c, p.A + ((size_t)cur * p.R + r0) * p.K, p.R - r0, mine >> g & 1 ? ra : -1, mine >> (g + 8) & 1 ? rb : -1, k0 + 32 * warp, k1, 128);
#pragma unroll
    for (int t = 0; t < NT; t++) {
        *reinterpret_cast<float2 *>(&red[warp][g][8 * t + 2 * q]) = make_float2(c[t][0], c[t][1]);
        *reinterpret_cast<float2 *>(&red[warp][g + 8][8 * t + 2 * q]) = make_float2(c[t][2], c[t][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * 8 * NT; i += 128) {
        const int r = i / (8 * NT), col = i % (8 * NT);
        if ((mine >> r & 1) && r0 + col < p.R)
            p.part[((size_t)blockIdx.y * p.M + j0 + r) * p.R + r0 + col] = (red[0][r][col] + red[1][r][col]) + (red[2][r][col] + red[3][r][col]);
    }
}
// k_lora_up starts while k_lora_down runs and requests what that does not write ahead of its wait: the rows' places, their base and
// B.  A place with one or two rows is multiplied by plain instructions, a lane having LC neighbouring columns: on tensor cores 14 or
// 15 rows of 16 would be nobody's, and the instructions around them bound it (64 rows on 64 adapters, K 4096, N 16384, R 16: 14.8 us
// instead of 16.2).  One with more goes through the tensor cores, the base in shared memory, and (NARROW, R <= 16) B for all of a warp's
// blocks of 64 columns requested first.  Now 17.3 us both launches (k_lora_down 8.7, k_lora_up 11.4 by themselves; 46 MB, 2.7 TB/s); a
// CTA a place and 1024 columns, which was two waves, 20.4; rings of copies a warp or a CTA with tensor cores only 24.7 and 27.3.
constexpr int LR_FEW = 2;
template <bool F32, bool NARROW> constexpr int lr_cols() { return NARROW && !F32 ? 1024 : 512; }        // columns of a CTA
template <bool F32, bool NARROW> constexpr int lr_pitch() { return lr_cols<F32, NARROW>() * (F32 ? 4 : 2) + 16; }       // bytes of a row of the base
template <bool F32, bool NARROW> static size_t lr_smem(int R) { return 16 * (size_t)lr_pitch<F32, NARROW>() + (size_t)(F32 ? 3 : 2) * 16 * ((R + 15) / 16 * 8 + 4) * sizeof(uint32_t); }

// A lane's LC columns of bf16 (LC = 8 or 4) as they lie, and of the rows
template <int LC> struct LrVec { uint32_t w[LC / 2]; };
template <int LC> __device__ __forceinline__ LrVec<LC> lr_ldv(const bf16 *p)
{
    LrVec<LC> v;
    if (LC == 8) { const uint4 x = lr_ldcg(reinterpret_cast<const uint4 *>(p)); v.w[0] = x.x; v.w[1] = x.y; v.w[LC / 2 - 2] = x.z; v.w[LC / 2 - 1] = x.w; }
    else asm volatile("ld.global.cg.v2.u32 {%0, %1}, [%2];" : "=r"(v.w[0]), "=r"(v.w[1]) : "l"(p) : "memory");
    return v;
}
// One or two rows of a place: blocks b0 .. b1 - 1 of 128 LC columns.  Whatever a block or 16 inner indices need next takes the
// registers' place as soon as they are used.
template <bool F32, int LC> __device__ __forceinline__ void lr_few(const LoraParams &p, float *tf, int j0, int cur, unsigned mine, int m, int b0, int b1, bool wait)
{
    constexpr int BW = F32 ? LC : LC / 2;                 // words of a row's base
    const bool two = (mine & (mine - 1)) != 0;
    const int place[2] = {__ffs(mine) - 1, two ? __ffs(mine & (mine - 1)) - 1 : __ffs(mine) - 1};
    const int row[2] = {__shfl_sync(~0u, m, place[0]), __shfl_sync(~0u, m, place[1])};
    int n = b0 * (128 * LC) + threadIdx.x * LC;
    const bf16 *B = p.Bm + (size_t)max(cur, 0) * p.R * p.N + n;
    LrVec<LC> b[16];
    uint32_t base[2][BW];
    // 16 rows of B from `from` on, `have` of them there
    const auto ask = [&](int r, const bf16 *&from, int have) { if (r < have) b[r] = lr_ldv<LC>(from); from += p.N; };
    const auto ask_base = [&](int n) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (n >= p.N || (e && !two)) continue;
#pragma unroll
            for (int k = 0; k < BW; k += LC / 2) {
                const LrVec<LC> v = lr_ldv<LC>(reinterpret_cast<const bf16 *>(reinterpret_cast<const uint32_t *>(p.base) + ((size_t)row[e] * p.N + n) / (F32 ? 1 : 2) + k));
#pragma unroll
                for (int i = 0; i < LC / 2; i++) base[e][k + i] = v.w[i];
            }
        }
    };
#pragma unroll
    for (int r = 0; r < 16; r++) b[r] = {};
    {
        const bf16 *from = B;
        const int have = cur >= 0 && n < p.N ? p.R : 0;
#pragma unroll
        for (int r = 0; r < 16; r++) ask(r, from, have);
    }
    ask_base(n);
    if (wait) pdl_wait();
    else __syncthreads();                     // the place before this one is done with tf
    if (cur >= 0) {
        const float scale = p.scale[cur];
        for (int i = threadIdx.x; i < (two ? 2 : 1) * p.R; i += 128) {
            const int e = i >= p.R, r = e ? i - p.R : i;
            float x = 0.0f;
            const float *src = p.part + (size_t)(j0 + place[e]) * p.R + r;
#pragma unroll 8
            for (int s = 0; s < p.S; s++) x += src[(size_t)s * p.M * p.R];
            tf[e * 256 + r] = x * scale;
        }
        __syncthreads();
    }
    for (int blk = b0; blk < b1; blk++, n += 128 * LC) {
        float c[2][LC] = {};
        if (cur >= 0)
            for (int r0 = 0; r0 < p.R; r0 += 16) {
                const bool end = r0 + 16 >= p.R, half = r0 + 8 >= p.R;
                if (end) B += 128 * LC;
                const bf16 *from = end ? B : B + (size_t)(r0 + 16) * p.N;
                const int have = end ? (blk + 1 < b1 && n + 128 * LC < p.N ? p.R : 0) : n < p.N ? p.R - r0 - 16 : 0;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    if (r < 8 || !half) {
                        float f[LC];
#pragma unroll
                        for (int k = 0; k < LC / 2; k++) { f[2 * k] = __uint_as_float(b[r].w[k] << 16); f[2 * k + 1] = __uint_as_float(b[r].w[k] & 0xffff0000u); }
                        const float t0 = tf[r0 + r];
#pragma unroll
                        for (int k = 0; k < LC; k++) c[0][k] = fmaf(t0, f[k], c[0][k]);
                        if (two) {
                            const float t1 = tf[256 + r0 + r];
#pragma unroll
                            for (int k = 0; k < LC; k++) c[1][k] = fmaf(t1, f[k], c[1][k]);
                        }
                    }
                    ask(r, from, have);
                }
            }
        uint32_t w[2][BW];
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int k = 0; k < BW; k++) {
                if (F32) w[e][k] = __float_as_uint(__uint_as_float(base[e][k]) + c[e][k]);
                else {
                    const __nv_bfloat162 h2 = __floats2bfloat162_rn(__uint_as_float(base[e][k] << 16) + c[e][2 * k], __uint_as_float(base[e][k] & 0xffff0000u) + c[e][2 * k + 1]);
                    w[e][k] = cur >= 0 ? *reinterpret_cast<const uint32_t *>(&h2) : base[e][k];
                }
            }
        if (blk + 1 < b1) ask_base(n + 128 * LC);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (n >= p.N || (e && !two)) continue;
            uint32_t *d = reinterpret_cast<uint32_t *>(p.Y) + ((size_t)row[e] * p.N + n) / (F32 ? 1 : 2);
#pragma unroll
            for (int k = 0; k < BW; k += 4) {
                if (BW >= 4) *reinterpret_cast<uint4 *>(d + k) = make_uint4(w[e][k], w[e][k + 1], w[e][BW >= 4 ? k + 2 : 0], w[e][BW >= 4 ? k + 3 : 0]);
                else *reinterpret_cast<uint2 *>(d) = make_uint2(w[e][0], w[e][1]);
            }
        }
    }
}
template <bool F32, bool NARROW, bool AHEAD> __global__ void __launch_bounds__(128, 4) k_lora_up(const __grid_constant__ LoraParams p)
{
    constexpr int TT = F32 ? 3 : 2, EB = F32 ? 4 : 2, UP = lr_cols<F32, NARROW>(), NB = UP / 256, PITCH = lr_pitch<F32, NARROW>(), PIECES = UP * EB / 16;
    extern __shared__ __align__(16) uint8_t lr_s[];
    uint32_t *ts = reinterpret_cast<uint32_t *>(lr_s + 16 * PITCH);       // [term][16][ldt] pairs of bf16
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3, ldt = (p.R + 15) / 16 * 8 + 4;
    pdl_trigger();
    if (!AHEAD) pdl_wait();
    const int j0 = (int)blockIdx.x / 16 * 16;
    int m, a;
    lr_row(p, j0 + (lane & 15), m, a, false);
    // The tile's places that have work (the first of each adapter), times blocks of columns, in equal shares to its 16 gridDim.y CTAs
    const unsigned same = __match_any_sync(~0u, m >= 0 ? a : -2) & 0xffffu;
    const unsigned work = __ballot_sync(~0u, m >= 0 && __ffs(same) - 1 == lane && !(a < 0 && p.Y == p.base));
    const int blocks = (p.N + UP - 1) / UP, total = __popc(work) * blocks, shares = 16 * gridDim.y, me = blockIdx.x % 16 * gridDim.y + blockIdx.y;
    const int u1 = (int)((long long)total * (me + 1) / shares);
    int u = (int)((long long)total * me / shares);
    if (u == u1) { if (AHEAD) pdl_wait(); return; }
    for (bool wait = AHEAD; u < u1; wait = false) {
        unsigned w = work;
        for (int k = u / blocks; k; k--) w &= w - 1;
        const int place = __ffs(w) - 1, b0 = u % blocks, b1 = min(blocks, b0 + u1 - u);
        u += b1 - b0;                         // this place's part of the share
        const int cur = __shfl_sync(~0u, a, place);
        const unsigned mine = __ballot_sync(~0u, m >= 0 && a == cur) & 0xffffu;
        if (__popc(mine) <= LR_FEW) { lr_few<F32, UP / 128>(p, reinterpret_cast<float *>(lr_s), j0, cur, mine, m, b0, b1, wait); continue; }
        if (!wait) __syncthreads();               // the place before this one is done with the shared memory
        uint4 b[NARROW ? NB : 1][4];
        const auto ask = [&](int c0) {            // B and the base of the CTA's columns
            if (NARROW)
#pragma unroll
                for (int i = 0; i < NB; i++) lr_up_b<true>(p, cur, c0 + 256 * i + 64 * warp, 0, b[NARROW ? i : 0]);
            for (int i = threadIdx.x; i < 16 * PIECES; i += 128) {
                const int r = i / PIECES, n = c0 + i % PIECES * (16 / EB), row = __shfl_sync(~0u, m, r);     // r: the warp's
                if ((mine >> r & 1) && n < p.N) lt_copy(lt_addr(lr_s + r * PITCH + i % PIECES * 16), reinterpret_cast<const uint8_t *>(p.base) + ((size_t)row * p.N + n) * EB, true);
            }
            lt_commit();
        };
        ask(b0 * UP);
        if (wait) pdl_wait();
        const int rows[2] = {__shfl_sync(~0u, m, g), __shfl_sync(~0u, m, g + 8)};
        const bool keep[2] = {(mine >> g & 1) != 0, (mine >> (g + 8) & 1) != 0};
        if (cur >= 0) {
            const float scale = p.scale[cur];
            for (int i = threadIdx.x; i < 16 * p.R / 2; i += 128) {
                const int r = i / (p.R / 2), col = 2 * (i % (p.R / 2));
                if (!(mine >> r & 1)) continue;
                float x = 0.0f, y = 0.0f;
                const float *src = p.part + (size_t)(j0 + r) * p.R + col;
#pragma unroll 8
                for (int s = 0; s < p.S; s++) { const float2 v = *reinterpret_cast<const float2 *>(src + (size_t)s * p.M * p.R); x += v.x; y += v.y; }
                uint32_t t[TT];
                lr_split<TT, true>(x * scale, y * scale, t);
#pragma unroll
                for (int k = 0; k < TT; k++) ts[(k * 16 + r) * ldt + col / 2] = t[k];
            }
        }
        for (int c0 = b0 * UP;;) {
            lt_wait<0>();
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const int n0 = c0 + 256 * i + 64 * warp;
                if (n0 >= p.N) break;
                float c[8][4] = {};
                if (cur >= 0) {
                    if (NARROW) lr_up_mul<F32>(p, c, b[NARROW ? i : 0], ts + g * ldt, ldt, 0);
                    else lr_up<F32>(p, c, ts + g * ldt, ldt, cur, n0);
                }
                uint4 base[2][2][F32 ? 2 : 1];
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int k = 0; k < (F32 ? 2 : 1); k++)
                            base[e][h][k] = *reinterpret_cast<const uint4 *>(lr_s + (g + 8 * e) * PITCH + (256 * i + 64 * warp + 16 * q + 8 * h) * EB + 16 * k);
                lr_up_store<F32>(p, c, base, cur, n0, rows, keep);
            }
            c0 += UP;
            if (c0 >= b1 * UP) break;
            __syncthreads();
            ask(c0);
        }
    }
}

// Which form, and the slices of K of LORA_TWO.  Us, on both sides of each border (bf16, M rows on so many adapters):
//   TILE (what TC does not take) above 2048 rows, of ranks up to 16 above 8192.  R 64: K 768, N 1536, rows in no order on 9 4096 24.0 as tiles
//                             and 41.2 as places, on 64 8192 52.3 and 82.8; K 2048, N 2048 on 64 4096 72.6 and 77.2; fp32, K 520, N 3664, 2660 / 8
//                             55.7 and 52.6.  fp32, R 16: K 3328, N 848, 2256 / 2 97.2 and 20.3; K 1024, N 1024, 8192 / 9 44.0 and 41.5;
//                             K 4096, N 4096 8192 / 9 162 and 101; K 2048, N 2048, 16384 / 9 109 and 126
//   ONE up to 256 rows, K R of 32768 and N of 2048 (or M N of 32768), where making the inner numbers once per 512 columns costs less
//                             than a launch.  K 768, N 768, R 16: 64 rows 4.8 instead of 6.2, 256 / 64 7.2 and 9.7, 512 / 64 10.5 and
//                             9.7; K 2048, N 2048, R 16: 64 / 64 7.2 and 8.1; K 768, N 4096, R 16: 8 / 8 4.5 and 5.5, 64 / 64 10.4 and
//                             7.4; K 768, N 16384, R 16: 1 row 5.7 and 5.5, 64 / 64 30.8 and 15.1
//                             K 768, N 1536, R 64 (K R 49152): 64 rows 14.2 and 10.3
//   ONE up to 32 rows, N of 2048 (4096 where M N is at most 32768) and K R of 65536: K 1024, N 1024, R 64: 1 row 7.5 and 9.2, 32 7.9 and 9.6; K 4096, R 16: N 768 1 row 5.5 and 5.5, 32 5.8
//                             and 6.7, N 4096 4 rows 6.2 and 5.6 (fp32 rows 2.4 more than LORA_TWO), and 4 us less of the host; K R 131072:
//                             K 4096, N 2048, R 32: 4 rows 13.0 and 6.9; K 2048, N 16384, R 24: 1 row 10.9 and 6.9
enum LoraForm { LORA_ONE, LORA_TWO, LORA_TILE, LORA_TC };
static LoraForm lora_form(int M, int K, int N, int R, int *S, int *kslice)
{
    *kslice = K; *S = 0;
    if (M > 8192 || (M > 2048 && R > 16)) return LORA_TILE;
    if (M <= 256 && R <= 64 && (long long)K * R <= (M <= 32 && N <= 4096 ? 65536 : 32768) && (N <= 2048 || (long long)M * N <= 32768)) return LORA_ONE;
    // Slices of K: as many CTAs as the device holds, if every row has a place; four times as many of at least 1024, since rows mostly share
    // their adapter with neighbours.  (R 64: fp32, K 4040, 895 / 1 64.9 and 34.3, with the loads below; bf16, K 4096, R 32, 1024 / 64 52.7 and
    // 37.8; slices of 384 where there was one of 768, 2048 / 8: 13.1 and 14.3.)
    long long s = (4LL * sm_count() + M - 1) / M;
    const long long most = (K + 511) / 512, more = (16LL * sm_count() + M - 1) / M;       // most: four warps with four steps of 32 each
    if (s < more) s = more < K / 1024 ? more : s > K / 1024 ? s : K / 1024;
    if (s > most) s = most;
    if (s < 1) s = 1;
    *kslice = (int)(((K + s - 1) / s + 127) / 128 * 128);
    *S = (K + *kslice - 1) / *kslice;
    return LORA_TWO;
}

// TC: bf16 rows that stand in their order, ranks of whole 16 (a tile of D and of B has no rows of the next adapter then), counts that fit
// 32 bits.  Us with it and without, rows in runs (M / adapters): K 768, N 1536, R 64: 512 / 8 11.0 and 14.8, 1024 / 4 9.9 and 17.8, 2048 / 8
// 12.0 and 22.1, 8192 / 9 22.6 and 32.7, 32768 / 9 57.7 and 91.7; R 256: 8192 / 3 29 and 127; K 768, N 768, R 16: 512 / 1 8.2 and 7.9, 1024 / 8
// 9.2 and 10.3, 8192 / 9 14.4 and 21.2.  Up to 2048 rows LORA_TWO's tiles of 16 are the better ones
//   where K is large, since every CTA makes the inner numbers of its pairs for itself: K 4096, N 4096: R 16 512 / 4 39 and 15, R 32 1024 / 64
//   57 and 53 (8192 / 9 61 and 91);
//   where rows come in no order with many adapters, or a small rank: K 768, N 1536, R 64: 512 / 8 14.6 and 21.6, 1024 / 16 28.9 and 39.4,
//   1024 / 32 47.9 and 44.7; K 768, N 768, R 16: 512 / 16 22.9 and 9.6, 512 / 64 67 and 9.3 (above 2048 the tiles of 64 are no better: K 768,
//   N 1536, R 64: 4096 / 64 255 and 581).
// Above them, up to 8192 rows of R 16, LORA_TWO's are so where K is large and N is not, whatever the rows' order: K 2048, N 2048: 2056 / 9 25.5 and
// 19.0, in no order 43.6 and 32.1, 4096 / 9 28.4 and 28.0; K 4096, N 1024: 4096 / 9 41.5 and 31.8; N 4096: 2056 / 9 44.5 and 25.3, 3300 / 9 47.2
// and 50.9; K 2048, N 6144: 3300 / 9 35.4 and 41.8; N 16384: K 4096, 2560 / 9 68 and 81; K 1536, N 1536: 2056 / 3 13.9 and 17.4.  Elsewhere it goes
// by the order, which the host does not see: K 768, N 768: 4096 / 9 11.8 and 19.8, 4096 / 64 19.0 and 20.0, 4096 / 200 31.6 and 20.7; in no order 34.9
// and 31.1, 164 and 40, 278 and 41 (8192 / 64 308 and 75).  Rows in no order come with `order`, and then take no TC.
static bool lora_tc_ok(int M, int K, int N, int R, int adapters)
{
    if (R == 16 && K >= 2048 && M <= 8192 && (long long)M * N <= 3000LL * K) return false;
    return R % 16 == 0 && (M > 2048 || (M >= 512 && K <= 1024 && R >= 32 && adapters <= 16)) && (M + 127) / 128 <= LC_TILES && (long long)M * ((N + 63) / 64) < (1LL << 31) &&
           (long long)adapters * R < (1LL << 31);
}

}  // namespace qlmb
using namespace qlmb;

static bool lora_shape_ok(int M, int K, int N, int R)
{
    return M > 0 && M < (1 << 24) && K > 0 && N > 0 && K < (1 << 24) && N < (1 << 24) && K % 8 == 0 && N % 8 == 0 && R >= 8 && R <= 256 && R % 8 == 0;
}
extern "C" size_t qlmb_lora_bytes(int M, int K, int N, int R)
{
    if (!lora_shape_ok(M, K, N, R)) return 0;
    int S, ks;
    return lora_form(M, K, N, R, &S, &ks) == LORA_TWO ? (size_t)S * M * R * sizeof(float) : 16;
}
static int lora_tc_launch(const LoraParams &p, cudaStream_t st)
{
    static bool configured_dev[64];                      // the attribute belongs to a device's copy of the kernel
    int dev = 0;
    QLMB_CUDA(cudaGetDevice(&dev));
    QLMB_REQUIRE(dev >= 0 && dev < 64, "device index %d", dev);
    if (!configured_dev[dev]) {
        QLMB_CUDA(cudaFuncSetAttribute(k_lora_tc, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        configured_dev[dev] = true;
    }
    LcParams c;
    memset(&c, 0, sizeof c);
    c.l = p;
    c.stages = lc_stages(p.R);
    const unsigned long long M = p.M, K = p.K, N = p.N, AR = (unsigned long long)p.adapters * p.R;
    const unsigned rank = (unsigned)p.R;
    const struct { CUtensorMap *m; const void *base; unsigned long long inner, rows; unsigned box; } maps[5] = {
        {&c.x_map, p.X, K, M, 128}, {&c.a_map, p.A, K, AR, rank}, {&c.base_map, p.base, N, M, 128}, {&c.b_map, p.Bm, N, AR, rank}, {&c.y_map, p.Y, N, M, 32}};
    for (int i = 0; i < 5; i++) {
        const int rc = make_map(maps[i].m, maps[i].base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, maps[i].inner, maps[i].rows, maps[i].inner * 2, 64, maps[i].box,
                                CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc) return rc;
    }
    const long long most = (long long)((p.M + 127) / 128) * ((p.N + 63) / 64);
    QLMB_CUDA(pdl_launch(true, k_lora_tc, dim3((unsigned)(most < sm_count() ? most : sm_count())), dim3(LC_T), lc_smem(p.R, c.stages), st, c));
    QLMB_LAUNCH_CHECK("k_lora_tc");
    return QLMB_OK;
}
template <bool F32> static int lora_launch(const LoraParams &p, LoraForm form, cudaStream_t st)
{
    if (form == LORA_TC) return lora_tc_launch(p, st);
    if (form == LORA_TILE) {
        static bool configured_dev[64];                  // the attribute belongs to a device's copy of the kernel
        int dev = 0;
        QLMB_CUDA(cudaGetDevice(&dev));
        QLMB_REQUIRE(dev >= 0 && dev < 64, "device index %d", dev);
        if (!configured_dev[dev]) {
            QLMB_CUDA(cudaFuncSetAttribute(k_lora_tile<F32, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lt_smem<F32>(64)));
            QLMB_CUDA(cudaFuncSetAttribute(k_lora_tile<F32, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lt_smem<F32>(256)));
            configured_dev[dev] = true;
        }
        const int tiles = (p.M + LT_M - 1) / LT_M, most = (p.N + 63) / 64;
        const int want = (3 * sm_count() / 2 + tiles / 2) / tiles;        // one to two CTAs an SM: each makes the inner numbers for itself
        const dim3 grid((unsigned)tiles, (unsigned)(want < 1 ? 1 : want > most ? most : want), LT_Z);
        QLMB_CUDA(pdl_launch_small(p.R <= 64 ? k_lora_tile<F32, true> : k_lora_tile<F32, false>, grid, dim3(256), lt_smem<F32>(p.R), st, p));
        QLMB_LAUNCH_CHECK("k_lora_tile");
        return QLMB_OK;
    }
    if (form == LORA_ONE) {
        const dim3 grid((unsigned)((p.M + 15) / 16 * 16), (unsigned)((p.N + LR_UP - 1) / LR_UP));
        QLMB_REQUIRE(grid.y < 65536, "qlmb_lora_add: N %d", p.N);
        QLMB_CUDA(pdl_launch_small(p.R <= 16 ? k_lora_one<F32, 2, 4> : k_lora_one<F32, 8, 1>, grid, dim3(256), 0, st, p));
        QLMB_LAUNCH_CHECK("k_lora_one");
        return QLMB_OK;
    }
    const bool narrow = p.R <= 16;
    // blocks of columns, and how many CTAs of k_lora_up there are to each 16 rows: as many as fit the device at once
    const int cols = narrow ? lr_cols<F32, true>() : lr_cols<F32, false>(), blocks = (p.N + cols - 1) / cols;
    const int each = (int)(((long long)blocks * p.M + 4 * sm_count() - 1) / (4 * sm_count()));
    const unsigned units = (unsigned)((p.M + 15) / 16 * 16);
    const dim3 gd(units, (unsigned)p.S, (unsigned)(narrow ? 1 : (p.R + LR_RT - 1) / LR_RT)), gu(units, (unsigned)((blocks + each - 1) / each));
    QLMB_REQUIRE(gd.y < 65536 && gu.y < 65536, "qlmb_lora_add: K %d, N %d", p.K, p.N);
    static bool configured_dev[64];
    int dev = 0;
    QLMB_CUDA(cudaGetDevice(&dev));
    QLMB_REQUIRE(dev >= 0 && dev < 64, "device index %d", dev);
    if (!configured_dev[dev]) {
        QLMB_CUDA(cudaFuncSetAttribute(k_lora_up<F32, true, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lr_smem<F32, true>(16)));
        QLMB_CUDA(cudaFuncSetAttribute(k_lora_up<F32, true, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lr_smem<F32, true>(16)));
        QLMB_CUDA(cudaFuncSetAttribute(k_lora_up<F32, false, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lr_smem<F32, false>(256)));
        QLMB_CUDA(cudaFuncSetAttribute(k_lora_up<F32, false, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lr_smem<F32, false>(256)));
        configured_dev[dev] = true;
    }
    QLMB_CUDA(pdl_launch_small(narrow ? k_lora_down<F32, 2, 4> : k_lora_down<F32, LR_RT / 8, F32 ? 2 : 1>, gd, dim3(128), 0, st, p));
    QLMB_LAUNCH_CHECK("k_lora_down");
    // behind k_lora_down, which waits before it lets this launch start (without early launches there is nothing to be ahead of)
    void (*up)(const LoraParams) = pdl_enabled() ? (narrow ? k_lora_up<F32, true, true> : k_lora_up<F32, false, true>)
                                                 : (narrow ? k_lora_up<F32, true, false> : k_lora_up<F32, false, false>);
    QLMB_CUDA(pdl_launch(true, up, gu, dim3(128), narrow ? lr_smem<F32, true>(p.R) : lr_smem<F32, false>(p.R), st, p));
    QLMB_LAUNCH_CHECK("k_lora_up");
    return QLMB_OK;
}
extern "C" int qlmb_lora_add(void *Y, const void *X, const void *base, int dtype, const void *A, const void *Bm, const float *scale, int adapters,
                             const int *adapter, const int *order, int M, int K, int N, int R, void *ws, size_t ws_bytes, void *stream)
{
    QLMB_REQUIRE(Y && X && base && A && Bm && scale && adapter, "qlmb_lora_add: NULL argument");
    QLMB_REQUIRE(dtype == QLMB_F32 || dtype == QLMB_BF16, "qlmb_lora_add: rows of type %d", dtype);
    if (M <= 0) return QLMB_OK;
    QLMB_REQUIRE(lora_shape_ok(M, K, N, R) && adapters > 0, "qlmb_lora_add: M %d, K %d and N %d (multiples of 8), rank %d (a multiple of 8 up to 256), %d adapters", M, K, N, R, adapters);
    QLMB_REQUIRE(Y != X, "qlmb_lora_add: Y is X (it may be the base)");
    QLMB_REQUIRE((((uintptr_t)Y | (uintptr_t)X | (uintptr_t)base | (uintptr_t)A | (uintptr_t)Bm | (uintptr_t)ws) & 15) == 0,
                 "qlmb_lora_add: rows, adapters and workspace must be 16-byte aligned");
    const size_t need = qlmb_lora_bytes(M, K, N, R);
    QLMB_REQUIRE(need <= 16 || (ws && ws_bytes >= need), "qlmb_lora_add: a workspace of %zu bytes, %zu are needed", ws_bytes, need);
    // Rows are read while others are written.
    const uintptr_t es = dtype == QLMB_F32 ? 4 : 2, y = (uintptr_t)Y, ny = (uintptr_t)M * N * es, x = (uintptr_t)X, b = (uintptr_t)base;
    QLMB_REQUIRE((y + ny <= x || x + (uintptr_t)M * K * es <= y) && (Y == base || y + ny <= b || b + ny <= y), "qlmb_lora_add: Y overlaps X, or the base without being it");
    LoraParams p = {Y, X, base, (const bf16 *)A, (const bf16 *)Bm, scale, adapter, order, (float *)ws, M, K, N, R, adapters, 0, 0, device_error_word()};
    LoraForm form = lora_form(M, K, N, R, &p.S, &p.kslice);
    if (dtype == QLMB_BF16 && !order && lora_tc_ok(M, K, N, R, adapters)) form = LORA_TC;
    return dtype == QLMB_F32 ? lora_launch<true>(p, form, as_stream(stream)) : lora_launch<false>(p, form, as_stream(stream));
}
