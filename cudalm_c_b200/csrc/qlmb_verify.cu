// Verification of drafted tokens against the model's logits (speculative sampling), beside the pick of one token in qlmb_block.cu.
//
// Slot b has nd drafted tokens x_0 .. x_{nd-1} from distributions q_i and nd + 1 rows of logits; p_i = softmax(logits_i / T).
// Token i is taken when u_i q_i(x_i) < p_i(x_i).  At the first that is not, the slot ends with a token drawn from max(0, p_i - q_i)
// (from p_i where that is nothing), after the last with one from p_nd: the tokens are distributed as the model's own.
// The draw is the lowest token whose cumulated weight passes u times the whole; weights and sums are in 64 bits, for a draw next
// to a border is decided by them.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <math.h>
#include "qlmb_common.cuh"
#include "qlmb_internal.h"

namespace cg = cooperative_groups;

namespace qlmb {

constexpr int VF_C = 8;                       // CTAs of a slot: one cluster
constexpr int VF_T = 256;
constexpr int VF_W = VF_T / 32;
constexpr int VF_ROWS = 64;                   // rows of logits of a slot, at most

struct VerifyParams {
    int *out, *count;
    float *lp;
    const void *logits;
    const float *q, *u, *temp;
    const int *draft, *nd;
    int dtype, B, n, V;
    long long ld, ldq;                        // elements from a row of logits / of q to the next
    int *errword;
};

__device__ __forceinline__ float vf_ld(const void *p, int dtype, size_t i)
{
    return dtype == QLMB_F32 ? reinterpret_cast<const float *>(p)[i] : __bfloat162float(reinterpret_cast<const bf16 *>(p)[i]);
}
__device__ __forceinline__ double vf_warp_sum(double x)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

__global__ void __cluster_dims__(VF_C, 1, 1) __launch_bounds__(VF_T) k_dec_verify(const VerifyParams p)
{
    cg::cluster_group cl = cg::this_cluster();
    // of this CTA's share of a row: its maximum with the lowest index, whether something in it is no number to draw from, the
    // sums of exp((l - m) / T) and exp(l - m); of the row that ends the slot: the two sums of weights
    __shared__ float mx[VF_ROWS];
    __shared__ int arg[VF_ROWS], odd[VF_ROWS];
    __shared__ double st[VF_ROWS], s1[VF_ROWS], wsum[2], wpart[2][VF_W];
    __shared__ float gm[VF_ROWS];
    __shared__ int garg[VF_ROWS], gbad[VF_ROWS];
    __shared__ double gst[VF_ROWS], gs1[VF_ROWS];
    __shared__ float rv[VF_W];
    __shared__ int ri[VF_W], rodd[VF_W];
    __shared__ int end_row, end_kind;         // kind 0: draw after the drafts, 1: draw in place of a refused draft, 2: nothing to draw from
    const int b = blockIdx.x / VF_C, c = blockIdx.x % VF_C, tid = threadIdx.x, w = tid >> 5, ln = tid & 31, n = p.n;
    const int nd = p.nd ? p.nd[b] : n;
    int *out = p.out + (size_t)b * (n + 1);
    float *lp = p.lp + (size_t)b * (n + 1);
    if (nd < 0 || nd > n) {                   // no slot (the whole cluster leaves)
        if (c == 0) {
            if (tid == 0) { p.count[b] = 0; if (nd > n) report_bad_index(p.errword, 310, b, nd); }
            for (int i = tid; i <= n; i += VF_T) { out[i] = -1; lp[i] = 0.0f; }
        }
        return;
    }
    const float temp = p.temp[b];
    const bool greedy = !(temp > 0.0f);
    const double it = greedy ? 1.0 : 1.0 / (double)temp;
    const int slice = (p.V + VF_C - 1) / VF_C, v0 = min(c * slice, p.V), v1 = min(v0 + slice, p.V);
    const size_t row0 = (size_t)b * (n + 1) * (size_t)p.ld;
    for (int i = 0; i <= nd; i++) {
        const size_t base = row0 + (size_t)i * p.ld;
        float m = -INFINITY; int a = 0x7fffffff, bad = 0;
        for (int v = v0 + tid; v < v1; v += VF_T) {
            const float x = vf_ld(p.logits, p.dtype, base + v);
            bad |= !(x < INFINITY);
            if (x > m) { m = x; a = v; }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float om = __shfl_xor_sync(~0u, m, o); const int oa = __shfl_xor_sync(~0u, a, o);
            if (om > m || (om == m && oa < a)) { m = om; a = oa; }
            bad |= __shfl_xor_sync(~0u, bad, o);
        }
        if (ln == 0) { rv[w] = m; ri[w] = a; rodd[w] = bad; }
        __syncthreads();
        if (tid == 0) {
            for (int k = 1; k < VF_W; k++) {
                if (rv[k] > m || (rv[k] == m && ri[k] < a)) { m = rv[k]; a = ri[k]; }
                bad |= rodd[k];
            }
            mx[i] = m; arg[i] = a; odd[i] = bad;
        }
        __syncthreads();
    }
    cl.sync();
    for (int i = tid; i <= nd; i += VF_T) {
        float m = -INFINITY; int a = 0x7fffffff, bad = 0;
        for (int k = 0; k < VF_C; k++) {
            const float om = *cl.map_shared_rank(&mx[i], k); const int oa = *cl.map_shared_rank(&arg[i], k);
            if (om > m || (om == m && oa < a)) { m = om; a = oa; }
            bad |= *cl.map_shared_rank(&odd[i], k);
        }
        gm[i] = m; garg[i] = a; gbad[i] = bad || m == -INFINITY;
    }
    __syncthreads();
    for (int i = 0; i <= nd; i++) {
        const size_t base = row0 + (size_t)i * p.ld;
        const double m = gm[i];
        double a = 0.0, d = 0.0;
        if (!gbad[i])
            for (int v = v0 + tid; v < v1; v += VF_T) {
                const double x = (double)vf_ld(p.logits, p.dtype, base + v) - m;
                a += exp(x * it); d += exp(x);
            }
        a = vf_warp_sum(a); d = vf_warp_sum(d);
        if (ln == 0) { wpart[0][w] = a; wpart[1][w] = d; }
        __syncthreads();
        if (tid == 0) {
            a = d = 0.0;
            for (int k = 0; k < VF_W; k++) { a += wpart[0][k]; d += wpart[1][k]; }
            st[i] = a; s1[i] = d;
        }
        __syncthreads();
    }
    cl.sync();
    for (int i = tid; i <= nd; i += VF_T) {
        double a = 0.0, d = 0.0;
        for (int k = 0; k < VF_C; k++) { a += *cl.map_shared_rank(&st[i], k); d += *cl.map_shared_rank(&s1[i], k); }
        gst[i] = a; gs1[i] = d;
    }
    __syncthreads();
    if (tid == 0) {                           // every CTA of the slot comes to the same end
        int r = 0, kind = 0;
        for (; r <= nd; r++) {
            if (gbad[r]) { kind = 2; break; }
            if (r == nd) break;
            const int x = p.draft[(size_t)b * n + r];
            if (x < 0 || x >= p.V) { kind = 3; break; }
            if (greedy) { if (x != garg[r]) { kind = 1; break; } }
            else {
                const double e = exp(((double)vf_ld(p.logits, p.dtype, row0 + (size_t)r * p.ld + x) - (double)gm[r]) * it);
                const double qx = p.q ? (double)p.q[((size_t)b * n + r) * p.ldq + x] : 1.0;
                if (!((double)p.u[(size_t)b * (n + 1) + r] * qx * gst[r] < e)) { kind = 1; break; }
            }
        }
        end_row = r; end_kind = kind;
        if (c == 0 && kind == 2) report_bad_index(p.errword, 309, b, r);
        if (c == 0 && kind == 3) report_bad_index(p.errword, 308, b, p.draft[(size_t)b * n + r]);
    }
    __syncthreads();
    const int r = end_row, kind = end_kind;
    if (c == 0) {                             // what was taken, and the places behind the end
        for (int i = tid; i <= n; i += VF_T) {
            if (i == r && kind < 2) continue;
            int x = -1; float l = 0.0f;
            if (i < r) {
                x = p.draft[(size_t)b * n + i];
                l = (float)((double)vf_ld(p.logits, p.dtype, row0 + (size_t)i * p.ld + x) - (double)gm[i] - log(gs1[i]));
            }
            out[i] = x; lp[i] = l;
        }
        if (tid == 0) p.count[b] = kind < 2 ? r + 1 : r;
    }
    if (kind >= 2) { cl.sync(); return; }     // nobody reads this CTA's shared memory any more
    const size_t base = row0 + (size_t)r * p.ld;
    int pick = -1;
    if (greedy) {
        if (c == 0 && tid == 0) pick = garg[r];
    } else {
        const double m = gm[r], Z = gst[r];
        const float *qr = kind == 1 && p.q ? p.q + ((size_t)b * n + r) * p.ldq : nullptr;
        const int xr = kind == 1 && !p.q ? p.draft[(size_t)b * n + r] : -1;
        const auto weight = [&](int v, bool rest) {          // Z times the token's: no quotient to round
            double e = exp(((double)vf_ld(p.logits, p.dtype, base + v) - m) * it);
            if (rest) { if (qr) e = fmax(e - (double)qr[v] * Z, 0.0); else if (v == xr) e = 0.0; }
            return e;
        };
        // a warp's part of the share is one run of tokens
        const int sub = (v1 - v0 + VF_W - 1) / VF_W, w0 = min(v0 + w * sub, v1), w1 = min(w0 + sub, v1);
        double a = 0.0, d = 0.0;
        for (int v = w0 + ln; v < w1; v += 32) { a += weight(v, kind == 1); d += weight(v, false); }
        a = vf_warp_sum(a); d = vf_warp_sum(d);
        if (ln == 0) { wpart[0][w] = a; wpart[1][w] = d; }
        __syncthreads();
        if (tid == 0) {
            a = d = 0.0;
            for (int k = 0; k < VF_W; k++) { a += wpart[0][k]; d += wpart[1][k]; }
            wsum[0] = a; wsum[1] = d;
        }
        cl.sync();
        double W[2] = {0.0, 0.0};
        for (int k = 0; k < VF_C; k++) { W[0] += cl.map_shared_rank(wsum, k)[0]; W[1] += cl.map_shared_rank(wsum, k)[1]; }
        const int s = W[0] > 0.0 ? 0 : 1;     // nothing is left of p - q: from p
        const double target = (double)p.u[(size_t)b * (n + 1) + n] * W[s];
        // the share, then the run, whose end passes the target; the last with a weight where rounding leaves none
        double acc = 0.0, at = 0.0;
        int cta = -1;
        for (int k = 0; k < VF_C; k++) {
            const double x = cl.map_shared_rank(wsum, k)[s];
            if (x > 0.0) { cta = k; at = acc; if (acc + x > target) break; }
            acc += x;
        }
        if (cta == c) {
            int run = -1; double from = 0.0;
            acc = at;
            for (int k = 0; k < VF_W; k++) {
                const double x = wpart[s][k];
                if (x > 0.0) { run = k; from = acc; if (acc + x > target) break; }
                acc += x;
            }
            if (run == w) {
                int last = -1;
                for (int v = w0; v < w1 && pick < 0; v += 32) {
                    const double e = v + ln < w1 ? weight(v + ln, kind == 1 && s == 0) : 0.0;
                    double cum = e;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) { const double y = __shfl_up_sync(~0u, cum, o); if (ln >= o) cum += y; }
                    const unsigned some = __ballot_sync(~0u, e > 0.0), past = __ballot_sync(~0u, e > 0.0 && from + cum > target);
                    if (past) pick = v + __ffs(past) - 1;
                    if (some) last = v + 31 - __clz(some);
                    from += __shfl_sync(~0u, cum, 31);
                }
                if (pick < 0) pick = last;
                if (ln) pick = -1;
            }
        }
    }
    if (pick >= 0) {
        out[r] = pick;
        lp[r] = (float)((double)vf_ld(p.logits, p.dtype, base + pick) - (double)gm[r] - log(gs1[r]));
    }
    cl.sync();
}

}  // namespace qlmb
using namespace qlmb;

extern "C" int qlmb_dec_verify(int *out, int *count, float *lp, const void *logits, int lg_dtype, long long ld, const float *q, long long ldq,
                               const int *draft, const int *nd, const float *u, const float *temp, int B, int n, int V, void *stream)
{
    QLMB_REQUIRE(out && count && lp && logits && u && temp && (n == 0 || draft), "qlmb_dec_verify: NULL argument");
    QLMB_REQUIRE(lg_dtype == QLMB_F32 || lg_dtype == QLMB_BF16, "qlmb_dec_verify: logits of type %d", lg_dtype);
    QLMB_REQUIRE(n >= 0 && n < VF_ROWS && V > 0 && V < (1 << 30), "qlmb_dec_verify: n %d (0..%d), V %d", n, VF_ROWS - 1, V);
    QLMB_REQUIRE(ld >= V && (!q || ldq >= V), "qlmb_dec_verify: rows of %lld and %lld elements, %d tokens", ld, ldq, V);
    if (B <= 0) return QLMB_OK;
    QLMB_REQUIRE(B < (1 << 24), "qlmb_dec_verify: %d slots", B);
    VerifyParams p = {out, count, lp, logits, q, u, temp, draft, nd, lg_dtype, B, n, V, ld, ldq, device_error_word()};
    k_dec_verify<<<(unsigned)B * VF_C, VF_T, 0, as_stream(stream)>>>(p);
    QLMB_LAUNCH_CHECK("k_dec_verify");
    return QLMB_OK;
}
