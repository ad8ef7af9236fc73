// Verification of drafted tokens against the model's logits (speculative sampling), beside the pick of one token in qlmb_block.cu.
//
// Slot b has nd drafted tokens x_0 .. x_{nd-1} from distributions q_i and nd + 1 rows of logits.  With m_i the largest logit of row
// i, e_i(v) = exp((l_i(v) - m_i) / T) and Z_i their sum, token i is taken when u_i q_i(x_i) Z_i < e_i(x_i).  At the first that is not,
// the slot ends with a token drawn by the weights max(0, e_i - q_i Z_i) (by e_i where that is nothing), after the last with one drawn by
// e_nd: the tokens are distributed as the model's own.  The draw is the lowest token whose cumulated weight passes u times the whole.
// Weights are fp32, off by |l - m| / T 2^-23 (the two roundings of their exponent, which 1 / T enters in two parts: with one, all weights are off
// the same way) and 2^-22 (2^x).  A lane adds the 16 of a step in fp32, all further sums are 64 bits, so that the vocabulary's size does
// not matter to them.  Of 204800 draws from ten rows N(0, 2.5) at temperatures of 0.3 to 1.5 12 were not the exact ones' at V 16384, 27 at 130001.
//
// A slot is a cluster of eight CTAs, a row of logits is cut into runs, one a warp.  A lane keeps maximum, lowest index of it and
// the two sums (T, and 1 for the log-probability) of what it reads, rescaled as the maximum moves; lanes are joined at the end of a
// run, warps and CTAs through (distributed) shared memory.  The run that holds the draw is read once more.
//
// Measured over twelve sets of drafts (median, least and most; the rows that the longest slot reads): 1 slot of 16384 fp32 logits, four drafts
// 11.8 us (8.3 to 12.0; 1 to 5 rows), 64 of them, a third greedy, 14.4 (14.0 to 15.6; 4 or 5), bf16 17.1 (16.4 to 18.1), 32 of 130001, seven drafts
// 27.4 (19 to 49; 1 to 8), 8 of 65536 18.8 (18.8 to 19.2; 4 or 5).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <float.h>
#include <math.h>
#include "qlmb_common.cuh"
#include "qlmb_internal.h"

namespace cg = cooperative_groups;

namespace qlmb {

constexpr int VF_C = 8;                       // CTAs of a slot: one cluster
constexpr int VF_ROWS = 64;                   // rows of logits of a slot, at most
constexpr int VF_GROUP = 2;                   // rows of a round, at most

struct VerifyParams {
    int *out, *count;
    float *lp;
    const void *logits;
    const float *q, *u, *temp;
    const int *draft, *nd;
    int B, n, V, group;                       // group: rows that are read before the drafts among them are tested
    long long ld, ldq;                        // elements from a row of logits / of q to the next
    int *errword;
};

__device__ __forceinline__ float vf_ex2(float x)      // 2^x (ex2.approx: 2 ulp; 0 -> 1, -inf -> 0)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^(d it), it in two parts: hi below it, lo > 0 what hi leaves, so that an infinite d does not meet a 0
struct VfScale { float hi, lo; };
__device__ __forceinline__ VfScale vf_scale2(double it)
{
    VfScale s;
    s.hi = __double2float_rd(it);
    s.lo = fmaxf((float)(it - (double)s.hi), __uint_as_float(1u));
    return s;
}
__device__ __forceinline__ float vf_pow(float d, VfScale s) { return vf_ex2(fmaf(d, s.hi, d * s.lo)); }
template <bool BF> __device__ __forceinline__ float vf_ld(const void *p, size_t i)
{
    return BF ? __bfloat162float(reinterpret_cast<const bf16 *>(p)[i]) : reinterpret_cast<const float *>(p)[i];
}
// Four neighbouring logits, in one load where VEC; -inf from place `end` on.
template <bool BF, bool VEC> __device__ __forceinline__ float4 vf_ld4(const void *p, size_t base, int v, int end)
{
    float4 r = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (VEC && v + 4 <= end) {
        if (BF) {
            const uint2 w = *reinterpret_cast<const uint2 *>(reinterpret_cast<const bf16 *>(p) + base + v);
            return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
        }
        return *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + base + v);
    }
    if (v < end) r.x = vf_ld<BF>(p, base + v);
    if (v + 1 < end) r.y = vf_ld<BF>(p, base + v + 1);
    if (v + 2 < end) r.z = vf_ld<BF>(p, base + v + 2);
    if (v + 3 < end) r.w = vf_ld<BF>(p, base + v + 3);
    return r;
}
__device__ __forceinline__ double vf_warp_sum(double x)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

// A run or a row: its largest logit and the lowest index of it, the sums relative to it, whether all is finite or -inf.
struct VfPart { double st; float s1, m; int arg, odd; };

// 2^((a - b) it) for maxima a <= b, -inf for "none" (which have no sum)
__device__ __forceinline__ double vf_scale(float a, float b, double it) { return exp2((fmax((double)a, (double)-FLT_MAX) - fmax((double)b, (double)-FLT_MAX)) * it); }

template <bool BF, bool VEC, int VF_W> __global__ void __cluster_dims__(VF_C, 1, 1) __launch_bounds__(32 * VF_W, VF_W == 8 ? 4 : 7) k_dec_verify(const VerifyParams p)
{
    constexpr int VF_T = 32 * VF_W, RPL = VF_C * VF_W / 32;      // threads; runs of a row a lane looks at when they are joined
    cg::cluster_group cl = cg::this_cluster();
    __shared__ VfPart warp_part[VF_ROWS][VF_W], row_part[VF_ROWS];
    __shared__ double run_w[VF_GROUP][VF_C * VF_W];       // of the rows of a round: what the runs weigh, by the row's maximum
    __shared__ double wtot[VF_W], wleft[VF_W];            // of the row that ends the slot: the runs' weights behind a refused draft
    __shared__ int sx[VF_ROWS];               // the drafts, their logits, u q of each
    __shared__ float sl[VF_ROWS];
    __shared__ double suq[VF_ROWS];
    const int b = blockIdx.x / VF_C, c = blockIdx.x % VF_C, tid = threadIdx.x, w = tid >> 5, ln = tid & 31, n = p.n;
    pdl_trigger();
    pdl_wait();
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
    const float temp = p.temp[b], un = p.u[(size_t)b * (n + 1) + n];
    const bool greedy = !(temp > 0.0f);
    // (an infinite temperature: every logit but -inf has the weight 1, a mask of fp32's lowest number too)
    const double it = greedy ? 1.4426950408889634 : fmin(fmax(1.4426950408889634 / (double)temp, 1.5e-45), 1e38);
    const VfScale cT = vf_scale2(it);
    constexpr float c1 = 1.4426950408889634f;             // (log-probabilities are fp32 numbers)
    const bool unit = greedy || temp == 1.0f;             // the two sums are one
    // runs of whole groups of four
    const int run = ((p.V + 4 * VF_C * VF_W - 1) / (4 * VF_C * VF_W)) * 4;
    const int w0 = min((c * VF_W + w) * run, p.V), w1 = min(w0 + run, p.V);
    const size_t row0 = (size_t)b * (n + 1) * (size_t)p.ld;
    if (tid < nd) {
        const int x = p.draft[(size_t)b * n + tid];
        const bool in = x >= 0 && x < p.V;
        sx[tid] = x;
        sl[tid] = in ? vf_ld<BF>(p.logits, row0 + (size_t)tid * p.ld + x) : 0.0f;
        suq[tid] = (double)p.u[(size_t)b * (n + 1) + tid] * (p.q && in ? (double)p.q[((size_t)b * n + tid) * p.ldq + x] : 1.0);
    }
    const int steps = (run + 511) / 512;      // of a run: 16 logits a lane
    const auto fetch = [&](int i, int s, float4 d[4]) {   // step s of row i's run, on into the next rows
        if (s >= steps) { i += s / steps; s %= steps; }
        const size_t base = row0 + (size_t)i * p.ld;
#pragma unroll
        for (int k = 0; k < 4; k++) d[k] = vf_ld4<BF, VEC>(p.logits, base, w0 + s * 512 + 4 * ln + 128 * k, w1);
    };
    float4 x[4], y[4];
    fetch(0, 0, x);
    int r = 0, kind = -1, at = 0;             // at: the row's place in its round
    for (int i0 = 0; i0 <= nd; i0 += p.group) {
        const int i1 = min(i0 + p.group, nd + 1);
        // ---- this warp's run of the rows i0 .. i1 - 1; the next step is requested ahead, the next group's first one too
        const int total = steps * (i1 - i0);
        float m = -INFINITY;
        double st = 0.0, s1 = 0.0;
        int arg = 0x7fffffff;
        for (int s = 0; s < total; s++) {
            if (s + 1 < total || i1 <= nd) fetch(i0, s + 1, y);
            const int v = w0 + (s % steps) * 512 + 4 * ln;
            float mx[4];
#pragma unroll
            for (int k = 0; k < 4; k++) mx[k] = fmaxf(fmaxf(x[k].x, x[k].y), fmaxf(x[k].z, x[k].w));
            const float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            if (mn > m) {                     // a new maximum: its place (the lowest of equals)
                const float was = fmaxf(m, -FLT_MAX), d = was - fmaxf(mn, -FLT_MAX);
                st *= (double)vf_pow(d, cT);
                s1 *= (double)vf_ex2(d * c1);
                m = mn;
                const int k = mx[0] == mn ? 0 : mx[1] == mn ? 1 : mx[2] == mn ? 2 : 3;
                const float4 f = k == 0 ? x[0] : k == 1 ? x[1] : k == 2 ? x[2] : x[3];
                arg = v + 128 * k + (f.x == mn ? 0 : f.y == mn ? 1 : f.z == mn ? 2 : 3);
            }
            const float ref = fmaxf(m, -FLT_MAX);
            float pt = 0.0f, p1 = 0.0f;       // the step's 16
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float f[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
                for (int e = 0; e < 4; e++) {  // a NaN or +inf makes the sum a NaN
                    const float d = f[e] - ref;
                    pt += vf_pow(d, cT);
                    if (!unit) p1 += vf_ex2(d * c1);
                }
            }
            st += (double)pt;
            s1 += (double)p1;
            if (s % steps == steps - 1) {     // the end of a row's run
                if (unit) s1 = st;
                VfPart a;
                a.m = m;
                a.arg = arg;
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    const float om = __shfl_xor_sync(~0u, a.m, o); const int oa = __shfl_xor_sync(~0u, a.arg, o);
                    if (om > a.m || (om == a.m && oa < a.arg)) { a.m = om; a.arg = oa; }
                }
                a.odd = __any_sync(~0u, st != st);
                const float ref = fmaxf(m, -FLT_MAX), wref = fmaxf(a.m, -FLT_MAX);
                a.st = vf_warp_sum(st * (double)vf_pow(ref - wref, cT));
                a.s1 = (float)(s1 * (double)vf_ex2((ref - wref) * c1));
#pragma unroll
                for (int o = 16; o; o >>= 1) a.s1 += __shfl_xor_sync(~0u, a.s1, o);
                if (ln == 0) warp_part[i0 + s / steps][w] = a;
                m = -INFINITY; st = s1 = 0.0; arg = 0x7fffffff;
            }
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] = y[k];
        }
        cl.sync();
        for (int i = i0 + w; i < i1; i += VF_W) {         // a warp joins the runs of a row
            VfPart a[RPL], t;
#pragma unroll
            for (int k = 0; k < RPL; k++) a[k] = *cl.map_shared_rank(&warp_part[i][(RPL * ln + k) % VF_W], (RPL * ln + k) / VF_W);
            t = a[0];
#pragma unroll
            for (int k = 1; k < RPL; k++) {
                if (a[k].m > t.m) { t.m = a[k].m; t.arg = a[k].arg; }
                t.odd |= a[k].odd;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const float om = __shfl_xor_sync(~0u, t.m, o); const int oa = __shfl_xor_sync(~0u, t.arg, o);
                if (om > t.m || (om == t.m && oa < t.arg)) { t.m = om; t.arg = oa; }
            }
            t.odd = __any_sync(~0u, t.odd);
            double zt = 0.0, z1 = 0.0;
#pragma unroll
            for (int k = 0; k < RPL; k++) {
                const double x = a[k].st * vf_scale(a[k].m, t.m, it);
                zt += x;
                run_w[i - i0][RPL * ln + k] = vf_pow(a[k].m - t.m, cT) > 0.0f ? x : 0.0;      // 0: every weight of the run is 0 below
                z1 += (double)(a[k].s1 * vf_ex2((fmaxf(a[k].m, -FLT_MAX) - fmaxf(t.m, -FLT_MAX)) * c1));
            }
            t.st = vf_warp_sum(zt);
            t.s1 = (float)vf_warp_sum(z1);
            if (ln == 0) row_part[i] = t;
        }
        __syncthreads();
        // every warp of the slot comes to the same end: a lane looks at every 32nd row
        r = VF_ROWS; kind = -1;
        for (int i = i0 + ln; i < i1 && kind < 0; i += 32) {
            const VfPart &a = row_part[i];
            int k = -1;
            if (a.odd || a.m == -INFINITY) k = 2;
            else if (i == nd) k = 0;
            else if (sx[i] < 0 || sx[i] >= p.V) k = 3;
            else if (greedy ? sx[i] != a.arg : !(suq[i] * a.st < exp2(((double)sl[i] - (double)a.m) * it))) k = 1;
            if (k >= 0) { r = i; kind = k; }
        }
        const int first = __reduce_min_sync(~0u, r), who = __ffs(__ballot_sync(~0u, r == first)) - 1;
        kind = __shfl_sync(~0u, kind, who);
        r = first;
        at = r - i0;
        if (kind >= 0) break;
    }
    const size_t base = row0 + (size_t)r * p.ld;
    const VfPart row = row_part[min(r, VF_ROWS - 1)];
    int pick = -1;
    if (kind >= 2) {
    } else if (greedy) {
        if (c == 0 && tid == 0) pick = row.arg;
    } else {
        const bool rest = kind == 1;
        const float *qr = rest && p.q ? p.q + ((size_t)b * n + r) * p.ldq : nullptr;
        const int xr = rest && !p.q ? sx[r] : -1;
        const auto weight = [&](int v, bool rest) {
            double e = vf_pow(vf_ld<BF>(p.logits, base + v) - row.m, cT);
            if (rest) { if (qr) e = fmax(fma(-(double)qr[v], row.st, e), 0.0); else if (v == xr) e = 0.0; }
            return e;
        };
        // every warp of the slot finds the run whose end passes the target; the last with a weight where rounding leaves none
        double xs[RPL], mysum = 0.0, all = 0.0;
        if (qr) {                                         // what q leaves of each run
            double a = 0.0;
#pragma unroll 8
            for (int v = w0 + ln; v < w1; v += 32) a += weight(v, true);
            a = vf_warp_sum(a);
            if (ln == 0) wleft[w] = a;
            cl.sync();
#pragma unroll
            for (int k = 0; k < RPL; k++) { xs[k] = *cl.map_shared_rank(&wleft[(RPL * ln + k) % VF_W], (RPL * ln + k) / VF_W); mysum += xs[k]; }
            all = vf_warp_sum(mysum);
        } else if (rest) {                                // the refused draft's run without it: every warp adds it up for itself
            const int rx = xr / run, x1 = min((rx + 1) * run, p.V);
            double a = 0.0;
#pragma unroll 8
            for (int v = rx * run + ln; v < x1; v += 32) a += weight(v, true);
            a = vf_warp_sum(a);
#pragma unroll
            for (int k = 0; k < RPL; k++) { xs[k] = RPL * ln + k == rx ? a : run_w[at][RPL * ln + k]; mysum += xs[k]; }
            all = vf_warp_sum(mysum);
        }
        const bool left = all > 0.0;
        if (!left) {                                      // a draw behind the drafts, or nothing is left: by e
            mysum = 0.0;
#pragma unroll
            for (int k = 0; k < RPL; k++) { xs[k] = run_w[at][RPL * ln + k]; mysum += xs[k]; }
            all = vf_warp_sum(mysum);
        }
        const double target = (double)un * all;
        double cum = mysum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const double y = __shfl_up_sync(~0u, cum, o); if (ln >= o) cum += y; }
        const unsigned has = __ballot_sync(~0u, mysum > 0.0), over = __ballot_sync(~0u, mysum > 0.0 && cum > target);
        const int src = over ? __ffs(over) - 1 : 31 - __clz(has);
        int mine = 0;
        double from = 0.0, acc = cum - mysum;
        bool found = false;
#pragma unroll
        for (int k = 0; k < RPL; k++) {
            if (xs[k] > 0.0 && !found) { mine = RPL * ln + k; from = acc; found = acc + xs[k] > target; }
            acc += xs[k];
        }
        mine = __shfl_sync(~0u, mine, src);
        from = __shfl_sync(~0u, from, src);
        if (mine / VF_W == c) {
            // the CTA reads the run again: a lane has `each` neighbouring tokens
            const int r0 = min(mine * run, p.V), r1 = min(r0 + run, p.V), each = (r1 - r0 + VF_T - 1) / VF_T;
            const int l0 = min(r0 + tid * each, r1), l1 = min(l0 + each, r1);
            const bool held = each <= 4;                  // the weights stay in registers
            double e4[4];
            mysum = 0.0;
            int last = -1;
            if (held) {
#pragma unroll
                for (int k = 0; k < 4; k++) { e4[k] = l0 + k < l1 ? weight(l0 + k, left) : 0.0; mysum += e4[k]; if (e4[k] > 0.0) last = l0 + k; }
            } else
#pragma unroll 4
                for (int v = l0; v < l1; v++) { const double e = weight(v, left); mysum += e; if (e > 0.0) last = v; }
            cum = mysum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const double y = __shfl_up_sync(~0u, cum, o); if (ln >= o) cum += y; }
            if (ln == 31) wtot[w] = cum;
            __syncthreads();
            int mw = -1;
            acc = from;
            for (int k = 0; k < VF_W; k++) {
                const double t = wtot[k];
                if (t > 0.0) { mw = k; from = acc; if (acc + t > target) break; }
                acc += t;
            }
            if (mw == w) {
                const unsigned some = __ballot_sync(~0u, last >= 0), past = __ballot_sync(~0u, last >= 0 && from + cum > target);
                if (past ? ln == __ffs(past) - 1 : ln == 31 - __clz(some)) {
                    from += cum - mysum;
                    pick = last;
                    if (held) {
#pragma unroll
                        for (int k = 3; k >= 0; k--) {    // (the lowest that passes; the sums in the order of the loop below)
                            double x = from;
#pragma unroll
                            for (int j = 0; j <= k; j++) x += e4[j];
                            if (e4[k] > 0.0 && x > target) pick = l0 + k;
                        }
                    } else
                        for (int v = l0; v <= last; v++) {
                            const double e = weight(v, left);
                            from += e;
                            if (e > 0.0 && from > target) { pick = v; break; }
                        }
                }
            }
        }
    }
    if (pick >= 0) {
        out[r] = pick;
        lp[r] = (float)((double)vf_ld<BF>(p.logits, base + pick) - (double)row.m) - logf(row.s1);
    }
    if (c == 0) {                             // what was taken, and the places behind the end
        for (int i = tid; i <= n; i += VF_T) {
            if (i == r && kind < 2) continue;
            out[i] = i < r ? sx[i] : -1;
            lp[i] = i < r ? (float)((double)sl[i] - (double)row_part[i].m) - logf(row_part[i].s1) : 0.0f;
        }
        if (tid == 0) {
            p.count[b] = kind < 2 ? r + 1 : r;
            if (kind == 2) report_bad_index(p.errword, 309, b, r);
            if (kind == 3) report_bad_index(p.errword, 308, b, sx[r]);
        }
    }
    cl.sync();                                // nobody reads this CTA's shared memory any more
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
    // A round (a group of rows, the cluster's meeting, the test) costs about 2.5 us beside the reading, and rows behind the end are read for
    // nothing.  Means over eight sets of drafts (a call lasts as long as its longest slot, see k_dec_verify's figures), us.  Vocabularies of up
    // to 32768: four warps a CTA, so that the 64 clusters of a full server run at once, and two rows a round (64 slots of 16384, up to five
    // rows: 16.0; one row a round 18.3, all five 16.5, eight warps 23.5; 64 of 32768 21.7, eight warps 24.0).  Above: eight warps, and two
    // rows where drafts come with probabilities, since those are mostly taken (8 slots of 130048, up to five rows 29.6, one row 31.8, four
    // warps 42.6; 16 of 65536 21.5, 24.3 and 25.2), one where they do not (32 slots of 130001, up to eight rows: 26.8; two rows 29.4, four
    // warps 31.8).
    const bool wide = V > 32768, bf = lg_dtype == QLMB_BF16, vec = ld % 4 == 0 && ((uintptr_t)logits & (bf ? 7 : 15)) == 0;
    VerifyParams p = {out, count, lp, logits, q, u, temp, draft, nd, B, n, V, wide && !q ? 1 : 2, ld, ldq, device_error_word()};
    void (*kern)(const VerifyParams);
    if (wide) kern = bf ? (vec ? k_dec_verify<true, true, 8> : k_dec_verify<true, false, 8>) : (vec ? k_dec_verify<false, true, 8> : k_dec_verify<false, false, 8>);
    else kern = bf ? (vec ? k_dec_verify<true, true, 4> : k_dec_verify<true, false, 4>) : (vec ? k_dec_verify<false, true, 4> : k_dec_verify<false, false, 4>);
    QLMB_CUDA(pdl_launch_small(kern, dim3((unsigned)B * VF_C), dim3(wide ? 256 : 128), 0, as_stream(stream), p));
    QLMB_LAUNCH_CHECK("k_dec_verify");
    return QLMB_OK;
}
