// Low-rank adapters of many requests beside a projection that their rows share:
//   Y[m] = base[m] + s_a (X[m] A_a^T) B_a,   a = adapter[m] (-1: Y[m] = base[m]),   A [n][R][K], B [n][R][N] bf16.
//
// Two launches: k_lora_down makes the R inner numbers of every row, in slices of K, k_lora_up adds the slices, multiplies by B and adds
// the base.  Both take tiles of 16 rows and go through the adapters that occur in the tile; a row's products depend on no other
// row, so a tile's 16 rows are multiplied by each adapter and only its own rows kept.  With the rows in the order of their
// adapters (`order`) most tiles have one.
// The inner numbers stay fp32: they enter the second product as two or three bf16 terms, so does X where it is fp32.
#include <cuda_bf16.h>
#include "qlmb_common.cuh"
#include "qlmb_internal.h"

namespace qlmb {

constexpr int LR_RT = 64;                     // inner columns of a CTA of k_lora_down
constexpr int LR_NT = 256;                    // output columns of a CTA of k_lora_up

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
// x, y as pairs of bf16: the nearest to them, then the nearest to what that leaves, and so on.  Two terms hold 16 bits, three all 24.
template <int TERMS> __device__ __forceinline__ void lr_split(float x, float y, uint32_t t[TERMS])
{
#pragma unroll
    for (int k = 0; k < TERMS; k++) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        t[k] = *reinterpret_cast<const uint32_t *>(&h);
        x -= __uint_as_float(t[k] << 16); y -= __uint_as_float(t[k] & 0xffff0000u);
    }
}
// Row of place j (of the tile order) and its adapter; -1, -1 behind the last row or for an index out of range, which is reported.
__device__ __forceinline__ void lr_row(const LoraParams &p, int j, int &m, int &a, bool report)
{
    m = a = -1;
    if (j >= p.M) return;
    m = p.order ? p.order[j] : j;
    if (m < 0 || m >= p.M) { if (report) report_bad_index(p.errword, 307, j, m); m = -1; return; }
    a = p.adapter[m];
    if (a < -1 || a >= p.adapters) { if (report) report_bad_index(p.errword, 307, m, a); a = -1; }
}

template <bool F32> __global__ void __launch_bounds__(128) k_lora_down(const __grid_constant__ LoraParams p)
{
    constexpr int XT = F32 ? 3 : 1;
    __shared__ float red[4][16][LR_RT + 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    pdl_trigger();
    pdl_wait();
    const int j0 = blockIdx.x * 16, r0 = blockIdx.z * LR_RT, k0 = blockIdx.y * p.kslice, k1 = min(p.K, k0 + p.kslice);
    int m, a;
    lr_row(p, j0 + (lane & 15), m, a, false);
    const int m0 = __shfl_sync(~0u, m, g), m1 = __shfl_sync(~0u, m, g + 8);
    unsigned left = __ballot_sync(~0u, a >= 0) & 0xffffu;
    while (left) {
        const int cur = __shfl_sync(~0u, a, __ffs(left) - 1);
        const unsigned mine = __ballot_sync(~0u, a == cur) & 0xffffu;
        left &= ~mine;
        float c[LR_RT / 8][4] = {};
        const bf16 *A = p.A + ((size_t)cur * p.R + r0) * p.K;
        for (int k = k0 + 32 * warp; k < k1; k += 128) {
            const int kk = k + 8 * q;
            const bool in = kk < k1;
            uint32_t x[XT][2][4];                        // [term][row half][pair]
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int mm = e ? m1 : m0;
                const bool live = in && mm >= 0 && (mine >> (g + 8 * e) & 1);
                if (F32) {
                    float4 u = make_float4(0, 0, 0, 0), v = u;
                    if (live) {
                        const float4 *s = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p.X) + (size_t)mm * p.K + kk);
                        u = s[0]; v = s[1];
                    }
                    const float f[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        uint32_t t[XT];
                        lr_split<XT>(f[2 * w], f[2 * w + 1], t);
#pragma unroll
                        for (int i = 0; i < XT; i++) x[i][e][w] = t[i];
                    }
                } else {
                    uint4 u = make_uint4(0, 0, 0, 0);
                    if (live) u = *reinterpret_cast<const uint4 *>(reinterpret_cast<const bf16 *>(p.X) + (size_t)mm * p.K + kk);
                    x[0][e][0] = u.x; x[0][e][1] = u.y; x[0][e][2] = u.z; x[0][e][3] = u.w;
                }
            }
#pragma unroll
            for (int t = 0; t < LR_RT / 8; t++) {
                uint4 b = make_uint4(0, 0, 0, 0);
                if (in && r0 + 8 * t < p.R) b = *reinterpret_cast<const uint4 *>(A + (size_t)(8 * t + g) * p.K + kk);
#pragma unroll
                for (int i = XT - 1; i >= 0; i--) {
                    const uint32_t a0[4] = {x[i][0][0], x[i][1][0], x[i][0][1], x[i][1][1]}, a1[4] = {x[i][0][2], x[i][1][2], x[i][0][3], x[i][1][3]};
                    lr_mma(c[t], a0, b.x, b.y);
                    lr_mma(c[t], a1, b.z, b.w);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < LR_RT / 8; t++) {
            *reinterpret_cast<float2 *>(&red[warp][g][8 * t + 2 * q]) = make_float2(c[t][0], c[t][1]);
            *reinterpret_cast<float2 *>(&red[warp][g + 8][8 * t + 2 * q]) = make_float2(c[t][2], c[t][3]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * LR_RT; i += 128) {
            const int r = i / LR_RT, col = i % LR_RT;
            if ((mine >> r & 1) && r0 + col < p.R)
                p.part[((size_t)blockIdx.y * p.M + j0 + r) * p.R + r0 + col] = (red[0][r][col] + red[1][r][col]) + (red[2][r][col] + red[3][r][col]);
        }
        __syncthreads();
    }
}

template <bool F32> __global__ void __launch_bounds__(128) k_lora_up(const __grid_constant__ LoraParams p)
{
    constexpr int TT = F32 ? 3 : 2;
    extern __shared__ float lr_t[];                      // [16][R + 4]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    pdl_trigger();
    pdl_wait();
    const int j0 = blockIdx.x * 16, n0 = blockIdx.y * LR_NT + warp * 64, ldt = p.R + 4;
    int m, a;
    lr_row(p, j0 + (lane & 15), m, a, blockIdx.y == 0 && threadIdx.x < 16);
    const int mrow[2] = {__shfl_sync(~0u, m, g), __shfl_sync(~0u, m, g + 8)};
    for (int i = threadIdx.x; i < 16 * p.R; i += 128) {
        const int r = i / p.R, col = i % p.R;
        int mm, aa;
        lr_row(p, j0 + r, mm, aa, false);
        float t = 0.0f;
        if (aa >= 0) {
            for (int s = 0; s < p.S; s++) t += p.part[((size_t)s * p.M + j0 + r) * p.R + col];
            t *= p.scale[aa];
        }
        lr_t[r * ldt + col] = t;
    }
    __syncthreads();
    unsigned left = __ballot_sync(~0u, m >= 0) & 0xffffu;
    while (left) {
        const int cur = __shfl_sync(~0u, a, __ffs(left) - 1);
        const unsigned mine = __ballot_sync(~0u, m >= 0 && a == cur) & 0xffffu;
        left &= ~mine;
        float c[8][4] = {};
        if (cur >= 0) {
            const bf16 *Bm = p.Bm + (size_t)cur * p.R * p.N + n0 + 8 * g;
            const bool in = n0 + 8 * g < p.N;
            for (int r0 = 0; r0 < p.R; r0 += 16) {
                uint32_t ta[TT][4];
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float2 v = make_float2(0.0f, 0.0f);
                        if (r0 + 8 * h < p.R) v = *reinterpret_cast<const float2 *>(lr_t + (g + 8 * e) * ldt + r0 + 8 * h + 2 * q);
                        uint32_t t[TT];
                        lr_split<TT>(v.x, v.y, t);
#pragma unroll
                        for (int i = 0; i < TT; i++) ta[i][2 * h + e] = t[i];
                    }
                uint4 b[4];
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const int r = r0 + 2 * q + (w & 1) + 8 * (w >> 1);
                    b[w] = make_uint4(0, 0, 0, 0);
                    if (in && r < p.R) b[w] = *reinterpret_cast<const uint4 *>(Bm + (size_t)r * p.N);
                }
                const uint32_t *b0 = &b[0].x, *b1 = &b[1].x, *b2 = &b[2].x, *b3 = &b[3].x;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                    const uint32_t x = __byte_perm(b0[j >> 1], b1[j >> 1], sel), y = __byte_perm(b2[j >> 1], b3[j >> 1], sel);
#pragma unroll
                    for (int i = TT - 1; i >= 0; i--) lr_mma(c[j], ta[i], x, y);
                }
            }
        }
        // columns 16 q .. 16 q + 15 of the warp's 64, rows g and g + 8
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (!(mine >> (g + 8 * e) & 1) || (cur < 0 && p.Y == p.base)) continue;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int col = n0 + 16 * q + 8 * h;
                if (col >= p.N) continue;
                const size_t at = (size_t)mrow[e] * p.N + col;
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; j++) f[j] = c[j][2 * e + h];
                if (F32) {
                    const float4 *s = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p.base) + at);
                    float4 *d = reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.Y) + at);
                    const float4 u = s[0], v = s[1];
                    d[0] = cur < 0 ? u : make_float4(u.x + f[0], u.y + f[1], u.z + f[2], u.w + f[3]);
                    d[1] = cur < 0 ? v : make_float4(v.x + f[4], v.y + f[5], v.z + f[6], v.w + f[7]);
                } else {
                    const uint4 u = *reinterpret_cast<const uint4 *>(reinterpret_cast<const bf16 *>(p.base) + at);
                    uint32_t w[4] = {u.x, u.y, u.z, u.w};
                    if (cur >= 0)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const __nv_bfloat162 h2 = __floats2bfloat162_rn(__uint_as_float(w[k] << 16) + f[2 * k], __uint_as_float(w[k] & 0xffff0000u) + f[2 * k + 1]);
                            w[k] = *reinterpret_cast<const uint32_t *>(&h2);
                        }
                    *reinterpret_cast<uint4 *>(reinterpret_cast<bf16 *>(p.Y) + at) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    }
}

// Slices of K: enough CTAs for the device, each warp at least one step of 32.
static void lora_plan(int M, int K, int R, int *S, int *kslice)
{
    const long long tiles = ((long long)M + 15) / 16 * ((R + LR_RT - 1) / LR_RT);
    long long s = (2LL * sm_count() + tiles - 1) / tiles;
    const long long most = (K + 127) / 128;
    if (s > most) s = most;
    if (s < 1) s = 1;
    *kslice = (int)(((K + s - 1) / s + 31) / 32 * 32);
    *S = (K + *kslice - 1) / *kslice;
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
    lora_plan(M, K, R, &S, &ks);
    return (size_t)S * M * R * sizeof(float);
}
extern "C" int qlmb_lora_add(void *Y, const void *X, const void *base, int dtype, const void *A, const void *Bm, const float *scale, int adapters,
                             const int *adapter, const int *order, int M, int K, int N, int R, void *ws, size_t ws_bytes, void *stream)
{
    QLMB_REQUIRE(Y && X && base && A && Bm && scale && adapter && ws, "qlmb_lora_add: NULL argument");
    QLMB_REQUIRE(dtype == QLMB_F32 || dtype == QLMB_BF16, "qlmb_lora_add: rows of type %d", dtype);
    if (M <= 0) return QLMB_OK;
    QLMB_REQUIRE(lora_shape_ok(M, K, N, R) && adapters > 0, "qlmb_lora_add: M %d, K %d and N %d (multiples of 8), rank %d (a multiple of 8 up to 256), %d adapters", M, K, N, R, adapters);
    QLMB_REQUIRE((((uintptr_t)Y | (uintptr_t)X | (uintptr_t)base | (uintptr_t)A | (uintptr_t)Bm | (uintptr_t)ws) & 15) == 0, "qlmb_lora_add: rows, adapters and workspace must be 16-byte aligned");
    const size_t need = qlmb_lora_bytes(M, K, N, R);
    QLMB_REQUIRE(ws_bytes >= need, "qlmb_lora_add: a workspace of %zu bytes, %zu are needed", ws_bytes, need);
    LoraParams p = {Y, X, base, (const bf16 *)A, (const bf16 *)Bm, scale, adapter, order, (float *)ws, M, K, N, R, adapters, 0, 0, device_error_word()};
    lora_plan(M, K, R, &p.S, &p.kslice);
    cudaStream_t st = as_stream(stream);
    const dim3 gd((unsigned)((M + 15) / 16), (unsigned)p.S, (unsigned)((R + LR_RT - 1) / LR_RT)), gu((unsigned)((M + 15) / 16), (unsigned)((N + LR_NT - 1) / LR_NT));
    QLMB_REQUIRE(gd.y < 65536 && gu.y < 65536, "qlmb_lora_add: K %d, N %d", K, N);
    QLMB_CUDA(pdl_launch_small(dtype == QLMB_F32 ? k_lora_down<true> : k_lora_down<false>, gd, dim3(128), 0, st, p));
    QLMB_LAUNCH_CHECK("k_lora_down");
    QLMB_CUDA(pdl_launch_small(dtype == QLMB_F32 ? k_lora_up<true> : k_lora_up<false>, gu, dim3(128), (size_t)16 * (R + 4) * sizeof(float), st, p));
    QLMB_LAUNCH_CHECK("k_lora_up");
    return QLMB_OK;
}
