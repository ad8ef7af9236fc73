"""The operators of a decode step for many requests at once (dec_rope_kv, dec_attn_prefix, dec_verify, lora_add): what their entry
points refuse, on the CPU, and their results against plain implementations in 64 bits, on the GPU.

Tolerances.  A rounding to bf16 is off by at most 2^-8 of the value, to fp32 by 2^-24.  Sums of n fp32 products are off by at most
n 2^-24 of the sum of the products' magnitudes (an accumulator that rounds towards zero: 2^-23)."""
import ctypes
import math

import numpy as np
import pytest
import torch

HD = 64
U16, U32 = 2.0 ** -8, 2.0 ** -24


# ------------------------------------------------------------------ refusals (no GPU)
def _lib():
    import cudalm_c_b200 as q
    return q.lib()


def test_refusals_of_the_entry_points():
    L, one, odd = _lib(), ctypes.c_void_p(4096), ctypes.c_void_p(4098)
    big = ctypes.c_size_t(1 << 40)

    def rope(Qo=one, hd=64, n=1, Tm=8, Tr=8, cos=one):
        return L.qlmb_dec_rope_kv(Qo, one, one, one, one, one, cos, one, one, 1, n, 0, Tm, 2, 2, hd, Tr, None)

    def attn(O=one, Kp=one, hd=64, B=1, n=1, P=8, Tm=8, H=2, KV=2, ws=one, nbytes=big):
        return L.qlmb_dec_attn_prefix(O, None, one, Kp, Kp, one, one, one, 0, B, n, P, Tm, H, KV, hd, ws, nbytes, None)

    def verify(out=one, dt=0, ld=16, q=one, ldq=16, draft=one, n=2, V=16):
        return L.qlmb_dec_verify(out, one, one, one, dt, ld, q, ldq, draft, None, one, one, 1, n, V, None)

    def lora(Y=ctypes.c_void_p(8192), X=one, dt=1, n=2, M=4, K=64, N=64, R=8, ws=one, nbytes=big):
        return L.qlmb_lora_add(Y, X, one, dt, one, one, one, n, one, None, M, K, N, R, ws, nbytes, None)

    cases = [
        (lambda: rope(Qo=None), b"NULL"), (lambda: rope(hd=128), b"head dimension"), (lambda: rope(n=0), b"bad shape"), (lambda: rope(Tm=0), b"bad shape"),
        (lambda: rope(Tr=0), b"bad shape"), (lambda: rope(Qo=odd), b"aligned"), (lambda: rope(cos=ctypes.c_void_p(4104)), b"aligned"),
        (lambda: attn(O=None), b"NULL"), (lambda: attn(Kp=None), b"NULL"), (lambda: attn(P=5000, ws=None), b"workspace"), (lambda: attn(hd=32), b"head dimension"),
        (lambda: attn(n=0), b"bad shape"), (lambda: attn(n=65), b"bad shape"), (lambda: attn(P=-1), b"bad shape"), (lambda: attn(H=3, KV=2), b"bad shape"),
        (lambda: attn(P=1 << 30), b"bad shape"), (lambda: attn(O=odd), b"aligned"), (lambda: attn(ws=odd), b"aligned"),
        (lambda: attn(P=5000, nbytes=ctypes.c_size_t(16)), b"workspace of 16 bytes"),
        (lambda: verify(out=None), b"NULL"), (lambda: verify(draft=None), b"NULL"), (lambda: verify(dt=2), b"type"), (lambda: verify(n=-1), b"n -1"),
        (lambda: verify(n=64), b"n 64"), (lambda: verify(V=0), b"V 0"), (lambda: verify(ld=15), b"rows of 15"), (lambda: verify(ldq=15), b"and 15"),
        (lambda: lora(Y=None), b"NULL"), (lambda: lora(ws=None, M=100, K=8192), b"workspace"), (lambda: lora(dt=7), b"type"), (lambda: lora(n=0), b"0 adapters"),
        (lambda: lora(K=60), b"multiples of 8"), (lambda: lora(N=63), b"multiples of 8"), (lambda: lora(R=12), b"rank 12"), (lambda: lora(R=264), b"rank 264"),
        (lambda: lora(R=0), b"rank 0"), (lambda: lora(Y=ctypes.c_void_p(8192), X=ctypes.c_void_p(8192)), b"Y is X"), (lambda: lora(Y=ctypes.c_void_p(8192), X=odd), b"aligned"), (lambda: lora(M=100, K=8192, nbytes=ctypes.c_size_t(4)), b"workspace of 4 bytes"),
    ]
    for i, (call, needle) in enumerate(cases):
        assert call() == 1, i
        assert needle in L.qlmb_last_error(), (i, needle, L.qlmb_last_error())
    # nothing to do is no error and touches no device
    assert L.qlmb_dec_rope_kv(*[one] * 9, 0, 1, 0, 8, 2, 2, 64, 8, None) == 0
    assert attn(B=0) == 0 and lora(M=0) == 0
    assert L.qlmb_dec_verify(one, one, one, one, 0, 16, one, 16, one, None, one, one, 0, 2, 16, None) == 0
    # workspaces: 0 where the shape is not supported
    for bad in ((0, 1, 8, 8, 2, 2), (1, 65, 8, 8, 2, 2), (1, 1, -1, 8, 2, 2), (1, 1, 8, 8, 3, 2), (1, 1, 1 << 30, 8, 2, 2), (1025, 2, 8, 8, 2, 2), (1024, 1, 8, 1 << 22, 2, 2)):
        assert L.qlmb_dec_attn_prefix_bytes(*bad) == 0, bad
    assert L.qlmb_dec_attn_prefix_bytes(2, 3, 100, 50, 4, 2) == 16 and L.qlmb_dec_attn_prefix_bytes(2, 3, 5000, 50, 4, 2) > 2 * 3 * 4 * 64 * 4
    for bad in ((0, 64, 64, 8), (4, 60, 64, 8), (4, 64, 64, 4), (4, 64, 64, 300)):
        assert L.qlmb_lora_bytes(*bad) == 0, bad
    assert L.qlmb_lora_bytes(5, 64, 128, 16) == 16 and L.qlmb_lora_bytes(105, 4096, 128, 16) >= 105 * 16 * 4


def test_refusals_of_the_mirrors():
    from cudalm_c_b200 import attn, block, linear
    bf = torch.bfloat16
    q, kp, kc, pos = torch.zeros(4, 128, dtype=bf), torch.zeros(8, 128, dtype=bf), torch.zeros(2, 8, 128, dtype=bf), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        attn.dec_attn_prefix(q, kp, kp, kc, kc, pos, 2)
    with pytest.raises(TypeError, match="pos"):
        attn.dec_attn_prefix(q, kp, kp, kc, kc, pos.long(), 2)
    with pytest.raises(TypeError, match="pos"):
        block.dec_rope_kv(q, q, q, kc, kc, kp, kp, [0, 0], 2)
    with pytest.raises(TypeError, match="logits"):
        block.dec_verify(torch.zeros(1, 2, 8, dtype=torch.float16), None, None, None)
    with pytest.raises(TypeError, match="X"):
        linear.lora_add(torch.zeros(1, 8, dtype=torch.float16), None, None, None, None, None)
    assert linear.lora_order(torch.tensor([2, -1, 0, 2, 0], dtype=torch.int32)).tolist() == [1, 2, 4, 0, 3]


# ------------------------------------------------------------------ plain implementations in 64 bits
def attn64(q, kp, vp, kc, vc, pos, H, win):
    """(o, lse, sum of weight * |v|, largest sum of |q k| / 8 of a row's keys) by a loop over tokens."""
    B, Tm, KD = kc.shape
    KV, P, n = KD // HD, kp.shape[0], q.shape[0] // pos.numel()
    G = H // KV
    o = torch.zeros(B * n, H, HD, dtype=torch.float64, device=q.device)
    lse = torch.full((B * n, H), -math.inf, dtype=torch.float64, device=q.device)
    absv, absqk = torch.zeros_like(o), torch.zeros_like(lse)
    for b, t0 in enumerate(pos.tolist()):
        for i in range(n):
            t = t0 + i
            lo = max(0, t - win + 1) if win > 0 else 0
            k = torch.cat((kp[lo:], kc[b, max(0, lo - P):t - P + 1])).double().view(-1, KV, HD)
            v = torch.cat((vp[lo:], vc[b, max(0, lo - P):t - P + 1])).double().view(-1, KV, HD)
            if k.shape[0] == 0:
                continue
            qq = q[b * n + i].double().view(KV, G, HD)
            s = torch.einsum("hgd,khd->hgk", qq, k) / 8.0
            w = torch.softmax(s, -1)
            o[b * n + i] = torch.einsum("hgk,khd->hgd", w, v).reshape(H, HD)
            absv[b * n + i] = torch.einsum("hgk,khd->hgd", w, v.abs()).reshape(H, HD)
            lse[b * n + i] = torch.logsumexp(s, -1).view(H)
            absqk[b * n + i] = (torch.einsum("hgd,khd->hgk", qq.abs(), k.abs()) / 8.0).amax(-1).view(H)
    return o, lse, absv, absqk


def check_attn(o, lse, want):
    wo, wl, absv, absqk = want
    # scores: 64 products, the scale, the difference to the maximum; 2^x to 2 ulp; weights to bf16; the sums over keys and pieces are
    # sums of like terms of relative error 2^-16 at most (thousands of keys in blocks); the output to bf16
    ds = 70 * 2 * U32 * absqk + 4 * U32 * (wl.abs().clamp(max=1e9) + absqk)
    tol = (U16 + 2.0 ** -16) * absv + 2 * ds[..., None] * absv + U16 * wo.abs() + 1e-30
    err = (o.double().view_as(wo) - wo).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    empty = wl == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    dl = (lse.double() - wl).abs()[~empty]
    assert bool((dl <= (ds + 2.0 ** -16 + 2 * U32 * wl.abs())[~empty]).all()), float(dl.max())


def make_attn(B, n, H, KV, P, Tm, seed, dev, spread=1.0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    bf = torch.bfloat16
    r = lambda *s: (torch.randn(*s, device=dev, generator=g) * spread).to(bf)
    return r(B * n, H * HD), r(P, KV * HD), r(P, KV * HD), r(B, Tm, KV * HD), r(B, Tm, KV * HD)


def ok(status=0):
    import cudalm_c_b200 as q
    torch.cuda.synchronize()
    assert q.lib().qlmb_check_device(None) == status, q.lib().qlmb_last_error()
    return q.lib().qlmb_last_error()


# ------------------------------------------------------------------ rotation and append
@pytest.mark.gpu
@pytest.mark.parametrize("B,n,H,KV,P,Tm", [(1, 1, 1, 1, 0, 1), (1, 1, 12, 12, 7, 9), (3, 5, 4, 2, 130, 40), (64, 4, 12, 3, 1000, 77), (2, 64, 3, 1, 0, 100)])
def test_rope_kv(cuda, B, n, H, KV, P, Tm):
    from cudalm_c_b200 import block
    q, k, v, Kc, Vc = make_attn(B, n, H, KV, B * n, Tm, 3, cuda)
    rs = np.random.RandomState(B + n)
    pos = P + rs.randint(0, Tm - n + 1, size=B)
    pos[0] = P + Tm - n                                    # the last rows of a cache
    cosb, sinb = block.rope_tables(P + Tm, HD, device=cuda)
    pt = torch.from_numpy(pos.astype(np.int32)).to(cuda)
    K0, V0, q0 = Kc.clone(), Vc.clone(), q.clone()
    got = block.dec_rope_kv(q, k, v, Kc, Vc, cosb, sinb, pt, H, P=P)
    ok()
    assert torch.equal(q, q0)
    t = (pt.long()[:, None] + torch.arange(n, device=cuda)).view(-1)
    slot = torch.arange(B, device=cuda).repeat_interleave(n)

    def turn(x):
        x = x.double().view(B * n, -1, 2, HD // 2)
        c, s = cosb[t].double()[:, None], sinb[t].double()[:, None]
        a, b = x[:, :, 0], x[:, :, 1]
        return torch.stack((a * c - b * s, b * c + a * s), 2).reshape(B * n, -1), torch.stack(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()), 2).reshape(B * n, -1)

    for have, src in ((got, q), (Kc[slot, t - P], k)):
        want, mag = turn(src)
        assert bool(((have.double() - want).abs() <= U16 * want.abs() + 3 * U32 * mag).all())
    assert torch.equal(Vc[slot, t - P], v)
    K0[slot, t - P], V0[slot, t - P] = Kc[slot, t - P], Vc[slot, t - P]
    assert torch.equal(K0, Kc) and torch.equal(V0, Vc)     # nothing else was written
    again = q.clone()
    assert block.dec_rope_kv(again, k, v, Kc, Vc, cosb, sinb, pt, H, P=P, out=again) is again and torch.equal(again, got)
    ok()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 2 ** 31 - 1, -2 ** 31, 19, 32 + 10 - 2])
def test_rope_kv_reports_a_slot_past_its_cache(cuda, bad):
    from cudalm_c_b200 import block
    P, Tm, n = 20, 12, 3
    q, k, v, Kc, Vc = make_attn(3, n, 2, 2, 9, Tm, 4, cuda)
    cosb, sinb = block.rope_tables(40, HD, device=cuda)
    pos = torch.tensor([P, bad, P + 1], dtype=torch.int32, device=cuda)
    K0, V0, out = Kc.clone(), Vc.clone(), torch.full_like(q, 7.0)
    block.dec_rope_kv(q, k, v, Kc, Vc, cosb, sinb, pos, 2, P=P, out=out)
    assert b"error code 201 (site 305" in ok(4)
    assert torch.equal(Kc[1], K0[1]) and torch.equal(Vc[1], V0[1]) and bool((out[3:6] == 7).all())
    assert torch.equal(Vc[0, :3], v[:3]) and torch.equal(Vc[2, 1:4], v[6:])


@pytest.mark.gpu
def test_rope_kv_stops_at_the_tables(cuda):
    from cudalm_c_b200 import block
    q, k, v, Kc, Vc = make_attn(1, 2, 1, 1, 2, 64, 5, cuda)
    cosb, sinb = block.rope_tables(31, HD, device=cuda)
    K0 = Kc.clone()
    block.dec_rope_kv(q, k, v, Kc, Vc, cosb, sinb, torch.tensor([30], dtype=torch.int32, device=cuda), 1)
    ok(4)
    assert torch.equal(Kc, K0)
    block.dec_rope_kv(q, k, v, Kc, Vc, cosb, sinb, torch.tensor([29], dtype=torch.int32, device=cuda), 1)
    ok()


# ------------------------------------------------------------------ attention
SHAPES = [
    # B, n, H, KV, P, Tm, win
    (1, 1, 1, 1, 0, 1, 0), (1, 1, 1, 1, 1, 1, 0), (1, 1, 12, 12, 512, 64, 0), (2, 1, 4, 4, 31, 33, 0), (3, 1, 4, 2, 32, 32, 0), (5, 2, 6, 2, 127, 65, 0),
    (8, 4, 12, 12, 300, 200, 0), (2, 3, 8, 1, 129, 40, 0), (7, 5, 16, 4, 1000, 130, 0), (64, 1, 12, 12, 640, 96, 0), (33, 5, 8, 2, 515, 64, 0), (1, 64, 8, 2, 257, 80, 0),
    (2, 16, 32, 2, 60, 100, 0), (4, 1, 2, 2, 4097, 20, 0), (1, 1, 2, 2, 3, 5000, 0), (16, 8, 8, 8, 0, 300, 0), (70, 3, 4, 4, 200, 30, 0), (1, 5, 1, 1, 20000, 9, 0),
    # shared keys of many rows (or very many of one) have a kernel of their own, joins of many rows and windows theirs
    (16, 5, 16, 4, 5003, 40, 0), (13, 5, 8, 8, 9857, 20, 0), (1, 1, 12, 12, 33003, 20, 0), (3, 64, 8, 2, 16448, 80, 0), (12, 5, 16, 2, 4800, 36, 0), (64, 5, 16, 4, 1217, 50, 0), (16, 5, 16, 4, 5003, 40, 4000),
    (300, 2, 4, 2, 40, 9, 0), (160, 3, 8, 2, 129, 40, 0), (400, 1, 2, 2, 0, 300, 0), (150, 2, 4, 4, 100, 50, 20), (37, 1, 4, 4, 2048, 33, 0), (37, 1, 4, 4, 2049, 33, 0), (5, 9, 8, 1, 700, 700, 100), (1024, 1, 2, 2, 40, 6, 0), (1024, 1, 1, 1, 13000, 3, 0),
    (3, 2, 4, 2, 100, 50, 1), (3, 4, 4, 2, 100, 50, 20), (6, 3, 2, 2, 400, 300, 128), (20, 5, 8, 2, 300, 64, 100), (2, 1, 2, 1, 64, 64, 2 ** 31 - 1), (9, 7, 3, 3, 5, 70, 33),
]


def positions(B, n, P, Tm, seed, dev):
    rs = np.random.RandomState(seed)
    pos = P + rs.randint(-1 if P else 0, Tm - n + 1, size=B)
    pos[0], pos[-1] = P + Tm - n, P + (-1 if P and B > 1 else 0) if B > 1 else P + Tm - n
    return torch.from_numpy(pos.astype(np.int32)).to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("B,n,H,KV,P,Tm,win", SHAPES)
def test_attention(cuda, B, n, H, KV, P, Tm, win):
    from cudalm_c_b200 import attn
    q, kp, vp, kc, vc = make_attn(B, n, H, KV, P, Tm, B * 7 + n, cuda)
    pos = positions(B, n, P, Tm, 11, cuda)
    for b, t in enumerate(pos.tolist()):                   # what lies behind a slot's last token is nobody's
        kc[b, t - P + n:] = math.nan
        vc[b, t - P + n:] = math.inf
    o, lse = attn.dec_attn_prefix(q, kp, vp, kc, vc, pos, H, win=win)
    ok()
    check_attn(o, lse, attn64(q, kp, vp, kc, vc, pos, H, win))
    o2, lse2 = attn.dec_attn_prefix(q, kp, vp, kc, vc, pos, H, win=win)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)   # the order of every sum is fixed


@pytest.mark.gpu
@pytest.mark.parametrize("B,n,H,KV,P,Tm,win", [(2, 4, 4, 2, 40, 30, 0), (9, 3, 16, 1, 200, 40, 0), (3, 4, 4, 2, 90, 60, 16), (40, 4, 4, 2, 300, 60, 64), (160, 4, 4, 2, 300, 60, 64), (160, 3, 16, 1, 200, 40, 0)])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_attention_keeps_infinities_to_those_who_see_them(cuda, B, n, H, KV, P, Tm, win, what):
    """The last new token's value (and with a window a row that only the first token still sees) is no number: the tokens that
    do not see it are as if it were 0."""
    from cudalm_c_b200 import attn
    q, kp, vp, kc, vc = make_attn(B, n, H, KV, P, Tm, 21, cuda)
    pos = P + torch.arange(B, device=cuda, dtype=torch.int32) % (Tm - n)
    clean = (kc.clone(), vc.clone(), kp.clone(), vp.clone())
    rows = torch.arange(B, device=cuda)
    kc[rows, (pos - P + n - 1).long()] = what
    vc[rows, (pos - P + n - 1).long()] = what
    seen = torch.zeros(B, n, dtype=torch.bool, device=cuda)
    seen[:, n - 1] = True
    if win:
        t = int(pos.max()) - win + 1                       # shared rows up to here are seen by few tokens or none
        hit = t if t < P else P - 1
        kp[hit], vp[hit] = what, what
        tt = pos[:, None] + torch.arange(n, device=cuda)
        seen |= (tt - win < hit) & (hit <= tt)
    o, lse = attn.dec_attn_prefix(q, kp, vp, kc, vc, pos, H, win=win)
    ok()
    o0, lse0 = attn.dec_attn_prefix(q, clean[2], clean[3], clean[0], clean[1], pos, H, win=win)
    s = seen.view(-1)
    assert bool(torch.isfinite(o[~s].float()).all()) and bool((~s).any())
    want = attn64(q, clean[2], clean[3], clean[0], clean[1], pos, H, win)
    check_attn(o[~s], lse[~s], tuple(x[~s] for x in want))
    if what != what:
        assert bool(torch.isnan(o[s].float()).all())


@pytest.mark.gpu
def test_attention_with_extreme_scores(cuda):
    """Scores of some 10^3 (one key has all the weight) and queries of 0 (all have the same)."""
    from cudalm_c_b200 import attn
    q, kp, vp, kc, vc = make_attn(4, 2, 4, 2, 333, 40, 5, cuda, spread=12.0)
    q[:2] = 0
    pos = positions(4, 2, 333, 40, 3, cuda)
    o, lse = attn.dec_attn_prefix(q, kp, vp, kc, vc, pos, 4)
    ok()
    check_attn(o, lse, attn64(q, kp, vp, kc, vc, pos, 4, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-2, 98, 130 - 3 + 1, 2 ** 31 - 1, -2 ** 31])
def test_attention_reports_a_slot_past_its_cache(cuda, bad):
    from cudalm_c_b200 import attn
    from cudalm_c_b200._lib import calls, lib, stream_ptr
    B, n, H, KV, P, Tm = 3, 3, 4, 2, 100, 30
    q, kp, vp, kc, vc = make_attn(B, n, H, KV, P, Tm, 8, cuda)
    pos = torch.tensor([P + 4, bad, P - 1], dtype=torch.int32, device=cuda)
    O, lse = torch.full_like(q, 7.0), torch.full((B * n, H), 7.0, device=cuda)
    nb = lib().qlmb_dec_attn_prefix_bytes(B, n, P, Tm, H, KV)
    ws = torch.empty(nb, dtype=torch.uint8, device=cuda)
    calls.dec_attn_prefix(O, lse, q, kp, vp, kc, vc, pos, 0, B, n, P, Tm, H, KV, 64, ws, nb, stream_ptr())
    assert b"error code 201 (site 306" in ok(4)
    assert bool((O[n:2 * n] == 7).all()) and bool((lse[n:2 * n] == 7).all())
    good = torch.tensor([P + 4, P, P - 1], dtype=torch.int32, device=cuda)
    o, l = attn.dec_attn_prefix(q, kp, vp, kc, vc, good, H)
    ok()
    for b in (0, 2):
        assert torch.equal(o[b * n:b * n + n], O[b * n:b * n + n]) and torch.equal(l[b * n:b * n + n], lse[b * n:b * n + n])


@pytest.mark.gpu
def test_attention_of_many_rows_at_its_borders(cuda):
    """Long shared keys of many rows: a slot past its cache is left as it is, scores of some 10^3 with the largest in the last key or
    the first, a shared value that is no number (seen by every row), a slot that sees nothing of its own."""
    from cudalm_c_b200 import attn
    from cudalm_c_b200._lib import calls, lib, stream_ptr
    B, n, H, KV, P, Tm = 16, 5, 16, 4, 5003, 12
    q, kp, vp, kc, vc = make_attn(B, n, H, KV, P, Tm, 18, cuda, spread=6.0)
    kp[0] *= 2
    kp[P - 1] *= 2
    q[:n] = 0
    pos = P + torch.arange(B, device=cuda, dtype=torch.int32) % (Tm - n) - 1
    pos[3] = P + Tm - n + 1
    O, lse = torch.full_like(q, 7.0), torch.full((B * n, H), 7.0, device=cuda)
    nb = lib().qlmb_dec_attn_prefix_bytes(B, n, P, Tm, H, KV)
    ws = torch.full((nb,), 255, dtype=torch.uint8, device=cuda)
    run = lambda: calls.dec_attn_prefix(O, lse, q, kp, vp, kc, vc, pos, 0, B, n, P, Tm, H, KV, 64, ws, nb, stream_ptr())
    run()
    assert b"error code 201 (site 306" in ok(4)
    assert bool((O[3 * n:4 * n] == 7).all()) and bool((lse[3 * n:4 * n] == 7).all())
    pos[3] = P
    run()
    ok()
    check_attn(O, lse, attn64(q, kp, vp, kc, vc, pos, H, 0))
    vp[77, 5] = math.inf                                   # kv head 0, dimension 5
    run()
    ok()
    o = O.float().view(B * n, KV, H // KV, HD)
    assert not bool(torch.isfinite(o[:n, 0, :, 5]).any())  # (queries of 0: every weight is the same)
    o[:, 0, :, 5] = 0                                      # elsewhere 0 * inf where the weight has gone to 0: no number, either
    assert bool(torch.isfinite(o).all())


@pytest.mark.gpu
def test_attention_of_slots_that_see_nothing(cuda):
    """No prefix and pos = -1: the first token sees nothing at all (zeros, -inf), the next one only itself."""
    from cudalm_c_b200 import attn
    for n in (1, 2):
        q, kp, vp, kc, vc = make_attn(3, n, 4, 2, 0, 9, 3, cuda)
        pos = torch.tensor([-1, 2, -1], dtype=torch.int32, device=cuda)
        for win in (0, 2):
            o, lse = attn.dec_attn_prefix(q, kp, vp, kc, vc, pos, 4, win=win)
            ok()
            check_attn(o, lse, attn64(q, kp, vp, kc, vc, pos, 4, win))
            assert bool((o[0] == 0).all()) and bool((lse[0] == -math.inf).all()) and bool(torch.isfinite(lse[n:2 * n]).all())


@pytest.mark.gpu
def test_attention_agrees_with_the_one_token_form(cuda):
    """Without a prefix and with one token a slot it is qlmb_dec_attn."""
    from cudalm_c_b200 import attn
    from cudalm_c_b200._lib import check, lib, ptr, stream_ptr
    B, H, KV, Tm = 5, 6, 3, 700
    q, _, _, kc, vc = make_attn(B, 1, H, KV, 0, Tm, 9, cuda)
    none = torch.empty(0, KV * HD, dtype=torch.bfloat16, device=cuda)
    pos = torch.tensor([0, 1, 255, 640, 699], dtype=torch.int32, device=cuda)
    for win in (0, 100):
        o, _ = attn.dec_attn_prefix(q, none, none, kc, vc, pos, H, win=win)
        ref = torch.empty_like(q)
        check(lib().qlmb_dec_attn(ptr(ref), ptr(q), ptr(kc), ptr(vc), ptr(pos), win, B, Tm, H, KV, 64, stream_ptr()))
        ok()
        want = attn64(q, none, none, kc, vc, pos, H, win)
        check_attn(o, want[1].float(), want)
        err = (o.double() - ref.double()).abs().view_as(want[0])
        assert bool((err <= 2 * (U16 + 2.0 ** -14) * (want[2] + want[0].abs())).all())


@pytest.mark.gpu
def test_attention_in_a_cache_past_32_bits(cuda):
    """Offsets of the last slot's rows lie beyond 2^32 bytes (and 2^31 elements)."""
    from cudalm_c_b200 import attn
    B, n, H, KV, P, Tm = 3, 2, 12, 12, 50, 1000000
    if torch.cuda.get_device_properties(0).total_memory < 40e9:
        pytest.skip("needs 10 GB")
    kc = torch.empty(B, Tm, KV * HD, dtype=torch.bfloat16, device=cuda)
    vc = torch.empty_like(kc)
    q, kp, vp, k1, v1 = make_attn(B, n, H, KV, P, 80, 10, cuda)
    win = 70                                               # the last 70 positions
    pos = torch.tensor([P + Tm - n, P + Tm - 40, P + Tm - n], dtype=torch.int32, device=cuda)
    kc[:, Tm - 120:] = 0
    vc[:, Tm - 120:] = 0
    kc[:, Tm - 80:], vc[:, Tm - 80:] = k1, v1
    o, lse = attn.dec_attn_prefix(q, kp, vp, kc, vc, pos, H, win=win)
    ok()
    # the same rows in a short cache: the positions of a window of 70 are all there
    short = torch.cat((torch.zeros_like(k1)[:, :40], k1), 1).contiguous(), torch.cat((torch.zeros_like(v1)[:, :40], v1), 1).contiguous()
    want = attn64(q, kp[:0], vp[:0], short[0], short[1], pos - P - Tm + 120, H, win)
    check_attn(o, lse, want)


# ------------------------------------------------------------------ verification
def verify64(logits, x, u, temp, q, nd, V):
    B, n1 = logits.shape[:2]
    n = n1 - 1
    out, count, lp = np.full((B, n1), -1, np.int64), np.zeros(B, np.int64), np.zeros((B, n1))
    lg = logits[:, :, :V].cpu().double().numpy()
    x, u, temp = x.cpu().numpy(), u.cpu().double().numpy(), temp.cpu().double().numpy()
    q = q.cpu().double().numpy() if q is not None else None
    nd = nd.cpu().numpy() if nd is not None else np.full(B, n)
    for b in range(B):
        for i in range(max(-1, nd[b]) + 1):
            row = lg[b, i]
            if not (row.max() > -np.inf and (row < np.inf).all()):
                break
            with np.errstate(over="ignore", under="ignore"):
                lsm = row - row.max()
                lsm = lsm - np.log(np.exp(lsm).sum())
                T = temp[b] if temp[b] > 0 else 1.0
                p = np.exp((row - row.max()) / T)          # Z times the probabilities: equal logits have weights of exactly 1
            Z = p.sum()
            if i < nd[b]:
                d = x[b, i]
                if not 0 <= d < V:
                    break
                if (row.argmax() == d) if temp[b] <= 0 else (u[b, i] * (q[b, i, d] if q is not None else 1.0) * Z < p[d]):
                    out[b, i], lp[b, i], count[b] = d, lsm[d], i + 1
                    continue
            w = p
            if i < nd[b] and temp[b] > 0:
                w = np.maximum(p - q[b, i, :V] * Z, 0) if q is not None else np.where(np.arange(V) == x[b, i], 0.0, p)
                w = w if w.sum() > 0 else p
            cum = np.cumsum(w)
            pick = row.argmax() if temp[b] <= 0 else np.nonzero(cum > u[b, n] * cum[-1])[0][0]
            out[b, i], lp[b, i], count[b] = pick, lsm[pick], i + 1
            break
    return out, count, lp


def make_verify(B, n, V, ld, dtype, dense, seed, dev, noise=0.6):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    lg = torch.full((B, n + 1, ld), 1e30, device=dev)      # columns behind the vocabulary are nobody's
    lg[:, :, :V] = torch.randn(B, n + 1, V, device=dev, generator=g) * 2.5
    lg = lg.to(dtype)
    temp = torch.rand(B, device=dev, generator=g) * 1.3 + 0.2
    temp[1::3] = 0.0
    tt = torch.where(temp > 0, temp, torch.ones_like(temp))[:, None, None]
    dl = (lg[:, :n, :V].float() + noise * torch.randn(B, n, V, device=dev, generator=g)) / tt
    q = torch.softmax(dl, -1)
    x = torch.empty(B, n, dtype=torch.int32, device=dev)
    if n:
        x = (dl - torch.log(-torch.log(torch.rand(B, n, V, device=dev, generator=g).clamp(1e-9, 1 - 1e-7)))).argmax(-1).int() if dense else dl.argmax(-1).int()
        x[1::3] = lg[1::3, :n, :V].float().argmax(-1).int()             # greedy slots take some
        if n > 1:
            x[1::6, n - 1] = (x[1::6, n - 1] + 1) % V
    u = torch.rand(B, n + 1, device=dev, generator=g)
    return lg, x.contiguous(), u, temp, q.contiguous() if dense else None


def check_verify(got, want):
    out, count, lp = (t.cpu().numpy() for t in got)
    assert np.array_equal(out, want[0]) and np.array_equal(count, want[1])
    # log-probabilities: fp32 numbers, the sum's terms to 2^-21 of themselves
    assert np.all(np.abs(lp - want[2]) <= U32 * np.abs(want[2]) + 2.0 ** -20 * (1 + np.abs(want[2])))


@pytest.mark.gpu
@pytest.mark.parametrize("B,n,V,ld", [(1, 0, 1, 1), (1, 1, 2, 2), (3, 4, 37, 37), (7, 3, 100, 128), (64, 4, 1000, 1001), (5, 8, 16384, 16384), (2, 63, 513, 520), (9, 2, 4099, 4100),
                                       (3, 5, 130001, 130048)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dense", [True, False])
@pytest.mark.parametrize("ragged", [True, False])
def test_verify(cuda, B, n, V, ld, dtype, dense, ragged):
    from cudalm_c_b200 import block
    lg, x, u, temp, q = make_verify(B, n, V, ld, dtype, dense, B + V, cuda)
    nd = torch.from_numpy(np.random.RandomState(V).randint(-1, n + 1, size=B).astype(np.int32)).to(cuda) if ragged else None
    got = block.dec_verify(lg, x, u, temp, q=q, nd=nd, V=V)
    ok()
    check_verify(got, verify64(lg, x, u, temp, q, nd, V))
    again = block.dec_verify(lg, x, u, temp, q=q, nd=nd, V=V)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.gpu
def test_verify_at_its_borders(cuda):
    """u at 0 and just below 1; equal distributions; a draft the model rules out; cut tokens; ties; very low and high temperatures."""
    from cudalm_c_b200 import block
    V, n = 300, 2
    B = 12
    g = torch.Generator(device=cuda)
    g.manual_seed(2)
    lg = torch.randn(B, n + 1, V, device=cuda, generator=g) * 2
    temp = torch.ones(B, device=cuda)
    u = torch.full((B, n + 1), 0.5, device=cuda)
    x = torch.randint(0, V, (B, n), device=cuda, generator=g, dtype=torch.int32)
    q = torch.softmax(lg[:, :n], -1)
    below = float(np.nextafter(np.float32(1), np.float32(0)))
    u[0], u[1] = 0.0, below
    lg[2, 0, int(x[2, 0])] = -math.inf                     # p(x) = 0, even u = 0 does not take it
    u[2] = 0.0
    lg[3, :, 5:] = -math.inf                               # five tokens are left
    lg[4, :, :] = 1.0                                      # all alike
    lg[5, :, 17] = 50.0                                    # one has everything
    x[5] = 17
    lg[6, 0, 40:44] = 99.0                                 # ties of a greedy slot: the lowest
    temp[6] = 0
    x[6, 0] = 41
    lg[7, 0, 40:44] = 99.0
    temp[7] = 0
    x[7, 0] = 40
    temp[8], temp[9] = 1e-30, 1e30
    lg[10] = torch.where(torch.rand(n + 1, V, device=cuda, generator=g) < 0.9, torch.full_like(lg[10], -3.4e38), lg[10])
    q[11] = 1.0                                            # nothing of p - q is left: from p
    u[11] = below
    got = block.dec_verify(lg, x, u, temp, q=q)
    ok()
    check_verify(got, verify64(lg, x, u, temp, q, None, V))
    assert got[0][6, 0] == 40 and got[1][6] == 1 and got[1][7] >= 2 and got[1][2] == 1 and int(got[0][2, 0]) != int(x[2, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 40001])
def test_verify_at_an_infinite_temperature(cuda, V):
    """Every token that is not cut has the same probability; a temperature that is no number picks the arg-max, as 0 does."""
    from cudalm_c_b200 import block
    B, n = 4, 2
    lg, x, u, temp, q = make_verify(B, n, V, V, torch.float32, False, 12, cuda)
    temp[:] = torch.tensor([math.inf, math.inf, math.nan, 3e38], device=cuda)
    lg[1, :, V // 2:] = -math.inf
    x[1] = V // 2 + 1
    x[2] = lg[2, :n].argmax(-1).int()
    got = block.dec_verify(lg, x, u, temp)
    ok()
    assert got[1][1] == 1 and int(got[0][1, 0]) == int(u[1, n].double() * (V // 2)) and got[1][2] == n + 1
    # finite logits: the oracle's own division by a large number is the same
    keep = torch.tensor([0, 3], device=cuda)
    check_verify(tuple(t[keep] for t in got), verify64(lg[keep], x[keep], u[keep], torch.full((2,), 1e30, device=cuda), None, None, V))


@pytest.mark.gpu
@pytest.mark.parametrize("what,site", [("nan", 309), ("inf", 309), ("none", 309), ("token", 308), ("negative", 308), ("count", 310)])
def test_verify_reports_what_it_cannot_use(cuda, what, site):
    from cudalm_c_b200 import block
    B, n, V = 3, 3, 200
    lg, x, u, temp, q = make_verify(B, n, V, V, torch.float32, True, 6, cuda)
    temp[:] = 0
    x[:] = lg[:, :n].argmax(-1).int()                      # everything is taken
    nd = torch.full((B,), n, dtype=torch.int32, device=cuda)
    if what == "nan":
        lg[1, 1, 100] = math.nan
    elif what == "inf":
        lg[1, 1, 100] = math.inf
    elif what == "none":
        lg[1, 1] = -math.inf
    elif what == "token":
        x[1, 1] = V
    elif what == "negative":
        x[1, 1] = -1
    else:
        nd[1] = n + 1
    out, count, lp = block.dec_verify(lg, x, u, temp, q=q, nd=nd)
    assert b"error code 201 (site %d" % site in ok(4)
    took = 0 if what == "count" else 1
    assert count.tolist() == [n + 1, took, n + 1]
    assert out[1].tolist() == x[1, :took].tolist() + [-1] * (n + 1 - took) and bool((lp[1, took:] == 0).all())


@pytest.mark.gpu
def test_verify_draws_the_models_distribution(cuda):
    """First tokens over many u are distributed as p, whatever q is: counts of 5 tokens within five standard deviations."""
    from cudalm_c_b200 import block
    V, B = 5, 20000
    g = torch.Generator(device=cuda)
    g.manual_seed(9)
    lg = torch.tensor([0.3, -1.0, 1.2, 0.0, -0.4], device=cuda).expand(B, 2, V).contiguous()
    q = torch.tensor([0.4, 0.3, 0.1, 0.1, 0.1], device=cuda).expand(B, 1, V).contiguous()
    x = torch.multinomial(q[:, 0], 1, replacement=True, generator=g).int()
    u = torch.rand(B, 2, device=cuda, generator=g)
    out, _, _ = block.dec_verify(lg, x, u, torch.ones(B, device=cuda), q=q)
    ok()
    p = torch.softmax(lg[0, 0].double(), -1).cpu()
    have = torch.bincount(out[:, 0].long().cpu(), minlength=V).double()
    assert bool(((have - B * p).abs() <= 5 * torch.sqrt(B * p * (1 - p))).all())


# ------------------------------------------------------------------ adapters
def lora64(X, base, A, Bm, scale, adapter):
    y, mag = base.double(), torch.zeros_like(base, dtype=torch.float64)
    for i in adapter.unique().tolist():
        if i < 0:
            continue
        r = torch.nonzero(adapter == i).flatten()
        x, a, b = X[r].double(), A[i].double(), Bm[i].double()
        y[r] += scale[i].double() * ((x @ a.t()) @ b)
        mag[r] = scale[i].double() * ((x.abs() @ a.abs().t()) @ b.abs())
    return y, mag


def make_lora(M, K, N, R, n, dtype, seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)
    return r(M, K).to(dtype), r(M, N).to(dtype), (r(n, R, K) * 0.1).bfloat16(), (r(n, R, N) * 0.1).bfloat16(), torch.rand(n, device=dev, generator=g) + 0.5


def check_lora(y, X, base, A, Bm, scale, adapter):
    want, mag = lora64(X, base, A, Bm, scale, adapter)
    K, R = A.shape[2], A.shape[1]
    # two sums and a few roundings in fp32; bf16 rows: the inner numbers to two bf16 terms (2^-16), the output to bf16
    if y.dtype == torch.float32:
        tol = (2 * (K + 3 * R) + 8) * U32 * mag + 2 * U32 * want.abs()
    else:
        tol = ((2 * (K + 2 * R) + 8) * U32 + 2.0 ** -16) * mag + U16 * want.abs() + U32 * want.abs()
    err = (y.double() - want).abs()
    assert bool((err <= tol + 1e-30).all()), float((err / (tol + 1e-30)).max())
    off = adapter == -1
    assert torch.equal(y[off], base[off])


LORA = [
    # M, K, N, R, adapters
    (1, 8, 8, 8, 1), (1, 768, 768, 8, 4), (3, 72, 136, 16, 2), (16, 64, 64, 64, 1), (17, 256, 512, 24, 5), (64, 768, 1536, 16, 64), (64, 1000, 200, 72, 7), (130, 512, 768, 256, 3),
    (333, 384, 264, 32, 10), (1000, 768, 768, 8, 40), (2, 4096, 16384, 16, 2), (70, 40, 1032, 40, 3),
    (2049, 72, 136, 8, 3), (2500, 768, 264, 64, 9), (2300, 256, 520, 136, 5), (4097, 512, 768, 16, 200), (257, 1024, 128, 64, 3),
    (2049, 72, 136, 24, 3), (32, 4096, 776, 16, 9), (31, 1016, 1032, 64, 31), (5, 8192, 520, 8, 2), (8200, 40, 136, 8, 3), (2100, 1032, 72, 16, 5), (600, 72, 136, 16, 3), (2304, 768, 520, 256, 4), (700, 64, 64, 32, 2), (5000, 136, 72, 48, 20), (512, 1024, 1544, 112, 1), (2180, 4104, 8, 16, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,R,n", LORA)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mode", ["runs", "mixed", "ordered", "none"])
def test_lora(cuda, M, K, N, R, n, dtype, mode):
    from cudalm_c_b200 import linear
    X, base, A, Bm, scale = make_lora(M, K, N, R, n, dtype, M + K, cuda)
    rs = np.random.RandomState(M + R)
    a = rs.randint(-1, n, size=M) if mode != "none" else np.full(M, -1)
    if mode == "runs":
        a = np.sort(a)[::-1].copy()
    if mode != "none":
        a[0] = n - 1
    adapter = torch.from_numpy(a.astype(np.int32)).to(cuda)
    order = linear.lora_order(adapter) if mode == "ordered" else None
    b0 = base.clone()
    y = linear.lora_add(X, base, A, Bm, scale, adapter, order=order)
    ok()
    assert torch.equal(base, b0)
    check_lora(y, X, base, A, Bm, scale, adapter)
    y2 = linear.lora_add(X, base, A, Bm, scale, adapter, order=order, out=base)          # in place
    ok()
    assert y2 is base and torch.equal(y2, y)


@pytest.mark.gpu
def test_lora_keeps_one_adapters_infinities_from_other_rows(cuda):
    from cudalm_c_b200 import linear
    X, base, A, Bm, scale = make_lora(40, 256, 320, 16, 3, torch.bfloat16, 1, cuda)
    adapter = torch.arange(40, device=cuda, dtype=torch.int32) % 3
    X[1] = math.inf                                        # a row of adapter 1
    A[2, 3], Bm[2, 5] = math.nan, math.inf
    y = linear.lora_add(X, base, A, Bm, scale, adapter)
    ok()
    clean = adapter != 2
    clean[1] = False
    assert bool(torch.isfinite(y[clean].float()).all()) and not bool(torch.isfinite(y[adapter == 2].float()).any())
    fixed = torch.where(clean, adapter, torch.full_like(adapter, -1))
    check_lora(torch.where(clean[:, None], y, base), X, base, A, Bm, scale, fixed)


@pytest.mark.gpu
@pytest.mark.parametrize("place", ["new", "in place"])
def test_lora_of_many_rows_keeps_adapters_apart(cuda, place):
    """Tiles with several adapters, with rows without one and with an adapter out of range: an adapter's infinities stay with its rows,
    a row whose adapter is no adapter keeps its base and is reported."""
    from cudalm_c_b200 import linear
    X, base, A, Bm, scale = make_lora(1300, 256, 320, 32, 5, torch.bfloat16, 4, cuda)
    adapter = torch.full((1300,), 3, device=cuda, dtype=torch.int32)
    adapter[100:300] = 1
    adapter[300:310] = torch.arange(10, device=cuda, dtype=torch.int32) % 5
    adapter[310:700] = -1
    adapter[900:1000] = 0
    adapter[1000:1024] = 2
    adapter[1030], adapter[1299] = 5, -2
    A[2, 3], Bm[2, 5], X[120] = math.nan, math.inf, math.inf
    out = base.clone() if place == "in place" else None
    b = out if out is not None else base
    y = linear.lora_add(X, b, A, Bm, scale, adapter, out=out)
    assert b"error code 201 (site 307" in ok(4)
    fixed = adapter.clone()
    fixed[1030], fixed[1299] = -1, -1
    odd = adapter == 2
    odd[120] = True
    assert not bool(torch.isfinite(y[odd].float()).any()) and bool(torch.isfinite(y[~odd].float()).all())
    fixed[odd] = -1
    check_lora(torch.where(odd[:, None], base, y), X, base, A, Bm, scale, fixed)


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["adapter", "negative", "order"])
def test_lora_reports_what_is_out_of_range(cuda, where):
    from cudalm_c_b200 import linear
    M = 21
    X, base, A, Bm, scale = make_lora(M, 64, 128, 8, 2, torch.float32, 2, cuda)
    adapter = torch.arange(M, device=cuda, dtype=torch.int32) % 2
    order = torch.arange(M, device=cuda, dtype=torch.int32)
    out = torch.full_like(base, 7.0)
    if where == "order":
        order[19] = M
    else:
        adapter[19] = 2 if where == "adapter" else -5
    linear.lora_add(X, base, A, Bm, scale, adapter, order=order, out=out)
    assert b"error code 201 (site 307" in ok(4)
    assert torch.equal(out[19], torch.full_like(out[19], 7.0) if where == "order" else base[19])
    keep = torch.arange(M, device=cuda) != 19
    check_lora(out[keep], X[keep], base[keep], A, Bm, scale, adapter[keep])


# ------------------------------------------------------------------ streams, graphs, all together
def _step(s):
    """One layer's part of a step that verifies drafts: adapted queries, rotation and append, attention, adapted output, the test."""
    from cudalm_c_b200 import attn, block, linear
    qa = linear.lora_add(s["x"], s["q"], s["A"], s["Bm"], s["scale"], s["adapter"], order=s["order"])
    qr = block.dec_rope_kv(qa, s["k"], s["v"], s["kc"], s["vc"], s["cos"], s["sin"], s["pos"], s["H"], P=s["P"])
    o, lse = attn.dec_attn_prefix(qr, s["kp"], s["vp"], s["kc"], s["vc"], s["pos"], s["H"])
    f = linear.lora_add(o, s["x"], s["A"], s["Bm"], s["scale"], s["adapter"], order=s["order"])
    logits = block.gemm_nt(f, s["emb"]).view(s["B"], s["n"], -1)
    out, count, lp = block.dec_verify(logits, s["draft"], s["u"], s["temp"])
    return qa, qr, o, lse, f, logits, out, count, lp


def _state(dev, seed, B=6, n=3, H=4, KV=2, P=150, Tm=64, V=512):
    from cudalm_c_b200 import block, linear
    D = H * HD
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)
    s = dict(B=B, n=n, H=H, P=P)
    _, s["kp"], s["vp"], s["kc"], s["vc"] = make_attn(B, n, H, KV, P, Tm, seed, dev)
    s["x"], s["q"] = r(B * n, D).bfloat16(), r(B * n, D).bfloat16()
    s["k"], s["v"] = r(B * n, KV * HD).bfloat16(), r(B * n, KV * HD).bfloat16()
    s["A"], s["Bm"], s["scale"] = (r(3, 16, D) * 0.1).bfloat16(), (r(3, 16, D) * 0.1).bfloat16(), torch.rand(3, device=dev, generator=g) + 0.5
    s["adapter"] = (torch.arange(B, device=dev, dtype=torch.int32) % 4 - 1).repeat_interleave(n).contiguous()
    s["order"] = linear.lora_order(s["adapter"])
    s["cos"], s["sin"] = block.rope_tables(P + Tm, HD, device=dev)
    s["pos"] = P + (torch.arange(B, device=dev, dtype=torch.int32) * 7) % (Tm - n)
    s["emb"] = (r(V, D) * 0.1).bfloat16()
    s["draft"] = torch.randint(0, V, (B, n - 1), device=dev, generator=g, dtype=torch.int32)
    s["u"], s["temp"] = torch.rand(B, n, device=dev, generator=g), torch.rand(B, device=dev, generator=g) + 0.5
    s["temp"][0] = 0
    return s


@pytest.mark.gpu
def test_the_operators_together(cuda):
    s = _state(cuda, 31)
    qa, qr, o, lse, f, logits, out, count, lp = _step(s)
    ok()
    check_lora(qa, s["x"], s["q"], s["A"], s["Bm"], s["scale"], s["adapter"])
    check_attn(o, lse, attn64(qr, s["kp"], s["vp"], s["kc"], s["vc"], s["pos"], s["H"], 0))
    check_lora(f, o, s["x"], s["A"], s["Bm"], s["scale"], s["adapter"])
    check_verify((out, count, lp), verify64(logits, s["draft"], s["u"], s["temp"], None, None, logits.shape[2]))


@pytest.mark.gpu
def test_two_graphs_and_two_streams(cuda):
    """Two captured steps replayed at the same time on two streams, new inputs in their buffers, and eager calls beside them: each
    call has scratch of its own."""
    states = [_state(cuda, 41), _state(cuda, 42, B=9, n=2, H=6, KV=3, P=700, Tm=40)]
    want = [[t.clone() for t in _step(s)] for s in states]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in states:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(_step(s))
        graphs.append(gr)
    torch.cuda.synchronize()
    for _ in range(20):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    ok()
    for got, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))
    fresh = _state(cuda, 43)
    w = [t.clone() for t in _step(fresh)]
    for k, t in fresh.items():
        if torch.is_tensor(t):
            states[0][k].copy_(t)
    with torch.cuda.stream(streams[0]):
        streams[0].wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
    with torch.cuda.stream(streams[1]):
        streams[1].wait_stream(torch.cuda.default_stream())
        eager = _step(fresh)
    ok()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], w)) and all(torch.equal(a, b) for a, b in zip(eager, w))


def test_the_mirrors_look_at_their_arguments():
    """calls.sizes: letters bind sizes, digits are powers of two, '?' may be None; whatever does not hold gives None."""
    from cudalm_c_b200._lib import calls
    f, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    look = lambda *a: calls.sizes(-1, torch.float32, *a)
    assert look(f, "ab", None, "?xy", torch.int32, i, "a") == (4, 8) and look(f, "b3") == (4,) and look(None, "?a") == () and look(f[:0], "ab") == (0, 8)
    for bad in ((f, "aa"), (f, "a"), (f, "abc"), (f.t(), "ab"), (f, "ab", f[:3], "ab"), (f, "a4"), (f.double(), "ab"), (3, "ab"), ([1.0], "a"), (None, "a"), (f, "a!"),
                (torch.int32, f, "ab"), (f[:, ::2], "ab")):
        assert look(*bad) is None, bad
    assert calls.sizes(0, torch.float32, f, "ab") is None
    with pytest.raises(TypeError):
        calls.sizes()
    with pytest.raises(TypeError):
        calls.sizes("x", f, "ab")


@pytest.mark.gpu
def test_the_large_forms_on_two_streams(cuda):
    """The tensor-core kernels (512 columns of tensor memory a CTA, 128 a CTA three times an SM), clusters and rings beside one another on two
    streams, eager and captured: results bit for bit those of calls one after the other."""
    from cudalm_c_b200 import attn, block, linear
    at = make_attn(16, 5, 16, 4, 5003, 40, 51, cuda)
    pos = positions(16, 5, 5003, 40, 52, cuda)
    big = make_lora(2500, 768, 264, 16, 5, torch.bfloat16, 53, cuda)
    wide = make_lora(2300, 256, 520, 128, 3, torch.float32, 54, cuda)
    few = make_lora(40, 4096, 2048, 16, 40, torch.bfloat16, 55, cuda)
    a_big = (torch.arange(2500, device=cuda, dtype=torch.int32) // 300) % 6 - 1
    a_wide = (torch.arange(2300, device=cuda, dtype=torch.int32) // 37) % 3
    a_few = torch.arange(40, device=cuda, dtype=torch.int32)
    lg, x, u, temp, q = make_verify(3, 4, 40001, 40001, torch.float32, True, 56, cuda)
    ops = [lambda: attn.dec_attn_prefix(at[0], at[1], at[2], at[3], at[4], pos, 16), lambda: (linear.lora_add(*big, a_big),), lambda: (linear.lora_add(*wide, a_wide),),
           lambda: (linear.lora_add(*few, a_few),), lambda: block.dec_verify(lg, x, u, temp, q=q)]
    want = [f() for f in ops]
    ok()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(6):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append([f() for f in (ops if k == 0 else ops[::-1])])
    ok()
    for k in range(2):
        for step in got[k]:
            for a, b in zip(step if k == 0 else step[::-1], want):
                assert all(torch.equal(p, r) for p, r in zip(a, b))
    graphs = []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got[k] = [f() for f in (ops if k == 0 else ops[::-1])]
        graphs.append(g)
    for _ in range(6):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    ok()
    for k in range(2):
        for a, b in zip(got[k] if k == 0 else got[k][::-1], want):
            assert all(torch.equal(p, r) for p, r in zip(a, b))


@pytest.mark.gpu
def test_the_first_call_of_a_process_may_be_captured(cuda):
    """Nothing was set up before: the device error word and the kernels' attributes are made while the stream is captured."""
    import os
    import subprocess
    import sys
    code = """
import sys; sys.path.insert(0, "tests")
import torch
from cudalm_c_b200 import block
x = torch.randn(2, 3, 300, device="cuda"); d = torch.zeros(2, 2, device="cuda", dtype=torch.int32)
u, t = torch.rand(2, 3, device="cuda"), torch.ones(2, device="cuda"); torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = block.dec_verify(x, d, u, t)
g.replay(); torch.cuda.synchronize()
want = block.dec_verify(x, d, u, t); torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, want)); print("equal")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "equal" in r.stdout, r.stderr[-2000:]


# ------------------------------------------------------------------ long caches of few slots
def test_long_caches_are_dealt_out_to_the_whole_device():
    """One launch of a CTA per (slot, kv head, 16 rows) only where its warps have few blocks of keys more than dealt out evenly: few slots
    with long caches have a workspace.  The workspace is enough for every window."""
    L = _lib()
    size = L.qlmb_dec_attn_prefix_bytes
    # B, n, P, Tm, H, KV
    for few in ((1, 1, 512, 1024, 12, 12), (8, 4, 2048, 1024, 12, 12), (1, 1, 0, 1, 1, 1), (12, 1, 0, 4000, 12, 12)):
        assert size(*few) == 16, few
    for long in ((1, 1, 512, 32768, 12, 12), (1, 1, 0, 8000, 1, 1), (4, 1, 512, 16000, 12, 12), (1, 5, 0, 65536, 16, 4)):
        assert size(*long) > 1000, long


@pytest.mark.gpu
@pytest.mark.parametrize("B,n,H,KV,P,Tm", [(1, 1, 12, 12, 512, 5000), (2, 3, 8, 2, 40, 9000), (1, 5, 4, 4, 0, 4100)])
@pytest.mark.parametrize("win", [0, 1, 100, 2500, 4000, -1])
def test_attention_in_long_caches_of_few_slots(cuda, B, n, H, KV, P, Tm, win):
    """On both sides of the border between one launch and three, which a window moves (-1: the widest that hides something)."""
    from cudalm_c_b200 import attn
    q, kp, vp, kc, vc = make_attn(B, n, H, KV, P, Tm, 61, cuda)
    pos = positions(B, n, P, Tm, 62, cuda)
    win = P + Tm - 1 if win < 0 else win
    o, lse = attn.dec_attn_prefix(q, kp, vp, kc, vc, pos, H, win=win)
    ok()
    check_attn(o, lse, attn64(q, kp, vp, kc, vc, pos, H, win))


@pytest.mark.gpu
def test_attention_dealt_out_in_a_cache_past_32_bits(cuda):
    """As test_attention_in_a_cache_past_32_bits, with a window too wide for one launch: the same rows in a short cache give the same."""
    from cudalm_c_b200 import attn
    B, n, H, KV, P, Tm, win, keep = 3, 2, 12, 12, 50, 1000000, 5000, 5200
    if torch.cuda.get_device_properties(0).total_memory < 40e9:
        pytest.skip("needs 10 GB")
    kc = torch.empty(B, Tm, KV * HD, dtype=torch.bfloat16, device=cuda)
    vc = torch.empty_like(kc)
    q, kp, vp, k1, v1 = make_attn(B, n, H, KV, P, keep, 63, cuda)
    kc[:, Tm - keep:], vc[:, Tm - keep:] = k1, v1
    pos = torch.tensor([P + Tm - n, P + Tm - 40, P + Tm - n - 130], dtype=torch.int32, device=cuda)
    o, lse = attn.dec_attn_prefix(q, kp, vp, kc, vc, pos, H, win=win)
    ok()
    check_attn(o, lse, attn64(q, kp[:0], vp[:0], k1, v1, pos - P - Tm + keep, H, win))


# ------------------------------------------------------------------ the device error word
_BLOCKING = """
import sys; sys.path.insert(0, "tests")
import ctypes, torch
from cudalm_c_b200 import block, lib
x = torch.randn(2, 3, 300, device="cuda"); d = torch.zeros(2, 2, device="cuda", dtype=torch.int32)
u, t = torch.rand(2, 3, device="cuda"), torch.zeros(2, device="cuda")
x[1, 0, 7] = float("nan"); torch.cuda.synchronize()
rt, st = ctypes.CDLL("libcudart.so.12"), ctypes.c_void_p()
assert rt.cudaStreamCreate(ctypes.byref(st)) == 0                # waits for the legacy stream, unlike torch's own
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(st.value)):
    out = block.dec_verify(x, d, u, t)
g.replay(); torch.cuda.synchronize()
assert lib().qlmb_check_device(None) == 4 and b"site 309" in lib().qlmb_last_error(), lib().qlmb_last_error()
assert lib().qlmb_check_device(None) == 0
print("reported")
"""


def _fresh_process(code):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    return subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=200)


@pytest.mark.gpu
def test_the_error_word_may_be_made_while_a_blocking_stream_is_captured(cuda):
    """The first call of a process, on a stream of plain cudaStreamCreate that is being captured: the word exists and is reported into."""
    r = _fresh_process(_BLOCKING)
    assert r.returncode == 0 and "reported" in r.stdout, r.stderr[-2000:]


# ------------------------------------------------------------------ adapters: values that are not finite, in every form
FORMS = [
    # M, K, N, R, adapters, order: one launch; two launches with one or two rows of an adapter, with more, of a larger rank; tiles of 64 rows; of 128
    (20, 72, 136, 8, 3, False), (24, 72, 136, 64, 3, False), (40, 1032, 4104, 16, 37, False), (40, 1032, 4104, 16, 4, False), (40, 1032, 2056, 72, 37, False), (40, 1032, 2056, 72, 4, True),
    (300, 256, 136, 16, 5, False), (2100, 72, 136, 24, 5, False), (2100, 136, 72, 48, 5, True), (2060, 72, 136, 136, 5, True), (600, 72, 136, 32, 5, False), (2100, 264, 72, 128, 5, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,R,n,ordered", FORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lora_takes_infinities_for_what_they_are(cuda, M, K, N, R, n, ordered, dtype):
    """Adapters of positive numbers: a row with an infinity is that infinity throughout, one with the type's largest number, which the
    adapter makes small, is finite."""
    from cudalm_c_b200 import linear
    X, base, A, Bm, scale = make_lora(M, K, N, R, n, dtype, 71, cuda)
    X, A, Bm = X.abs() + 0.125, A.abs() + 0.125, Bm.abs() + 0.125
    adapter = (torch.arange(M, device=cuda, dtype=torch.int32) * 7) % n
    top = torch.finfo(dtype).max
    A[:, :, 5] = 2.0 ** -100
    up, down, large = 3, M - 1, M // 2
    X[up, 9], X[down, K - 1] = math.inf, -math.inf
    X[large] = 0
    X[large, 5] = top
    order = linear.lora_order(adapter) if ordered else None
    y = linear.lora_add(X, base, A, Bm, scale, adapter, order=order)
    ok()
    assert bool((y[up] == math.inf).all()) and bool((y[down] == -math.inf).all())
    odd = torch.zeros(M, dtype=torch.bool, device=cuda)
    odd[up] = odd[down] = True
    check_lora(torch.where(odd[:, None], base, y), X, base, A, Bm, scale, torch.where(odd, torch.full_like(adapter, -1), adapter))


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,R,n,ordered", FORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("place", ["new", "in place"])
def test_lora_keeps_infinities_apart_in_every_form(cuda, M, K, N, R, n, ordered, dtype, place):
    """An adapter with a NaN and an infinity and a row of infinities reach nobody else's rows, nor do rows without an adapter."""
    from cudalm_c_b200 import linear
    X, base, A, Bm, scale = make_lora(M, K, N, R, n, dtype, 72, cuda)
    adapter = (torch.arange(M, device=cuda, dtype=torch.int32) * 5) % (n + 1) - 1
    A[2, 3], Bm[2, 5], X[1] = math.nan, math.inf, math.inf
    if M > 100:
        adapter[64:96] = 1                                 # tiles with several adapters, and a whole piece of one
        X[70] = math.nan
    order = linear.lora_order(adapter) if ordered else None
    out = base.clone() if place == "in place" else None
    b = out if out is not None else base
    y = linear.lora_add(X, b, A, Bm, scale, adapter, order=order, out=out)
    ok()
    odd = adapter == 2
    odd[1] = adapter[1] >= 0
    if M > 100:
        odd[70] = True
    assert bool(torch.isfinite(y[~odd].float()).all()) and not bool(torch.isfinite(y[odd].float()).any())
    check_lora(torch.where(odd[:, None], base, y), X, base, A, Bm, scale, torch.where(odd, torch.full_like(adapter, -1), adapter))


# ------------------------------------------------------------------ verification: sums of large vocabularies, masks at any temperature
@pytest.mark.gpu
@pytest.mark.parametrize("low,T", [(-2.8125, 1.0), (-1.5, 1.0), (-1.40625, 0.5)])
def test_verify_sums_a_large_vocabulary(cuda, low, T):
    """128 tokens of every 2^16 ahead of the others, which are equal: a lane of a warp has one or more of the former and some 2000 of the
    latter.  A draft is taken and refused as its u lies 2^-19 on
    either side of its probability: weights are off by 2^-21.7 (the exponent's two roundings, 2^x to 2 ulp), a step's 16 terms in fp32 by
    (2 + .. + 16) / 16 2^-24 = 2^-20.9."""
    from cudalm_c_b200 import block
    V = 1 << 22
    lg = torch.full((2, 2, V), low, device=cuda)
    lg.view(2, 2, -1, 1 << 16)[:, :, :, :128] = 0
    ahead = 128 * (V >> 16)
    p0 = 1.0 / (ahead + (V - ahead) * math.exp(low / T))
    u = torch.tensor([[p0 * (1 - 2.0 ** -19), 0.5], [p0 * (1 + 2.0 ** -19), 0.5]], dtype=torch.float64, device=cuda).float()
    x = torch.zeros(2, 1, dtype=torch.int32, device=cuda)
    out, count, lp = block.dec_verify(lg, x, u, torch.full((2,), T, device=cuda))
    ok()
    assert count.tolist() == [2, 1] and int(out[0, 0]) == 0 and int(out[1, 0]) > 0
    z1 = math.log(ahead + (V - ahead) * math.exp(low))     # log-probabilities at temperature 1
    want = torch.tensor([-z1, float(lg[1, 0, int(out[1, 0])]) - z1], dtype=torch.float64)
    have = torch.stack((lp[0, 0], lp[1, 0])).cpu().double()
    assert bool(((have - want).abs() <= 2.0 ** -20 * (1 + want.abs())).all()), (have, want)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 40001])
def test_verify_masks_of_the_lowest_number(cuda, V):
    """Logits of fp32's lowest number have no weight at ordinary temperatures, large ones too, and that of any other number at an infinite one."""
    from cudalm_c_b200 import block
    B = 6
    lg, x, u, temp, _ = make_verify(B, 0, V, V, torch.float32, False, 81, cuda)
    lg[:, 0, :V - 7] = torch.finfo(torch.float32).min
    temp[:] = torch.tensor([1.0, 1e-30, 1e30, 1e36, math.inf, math.inf], device=cuda)
    out, count, lp = block.dec_verify(lg, x, u, temp)
    ok()
    want = verify64(lg[:4], x[:4], u[:4], temp[:4], None, None, V)
    check_verify((out[:4], count[:4], lp[:4]), want)
    # all weights 1 (to 2^-20, the masked ones): the token is the one in which u V falls
    for b in (4, 5):
        assert abs(int(out[b, 0]) - float(u[b, 0]) * V) <= 1 + V * 2.0 ** -19


def test_the_mirrors_keep_few_sizes():
    """Batches and prompts change from step to step: what the mirrors keep by shape has an end."""
    from cudalm_c_b200 import attn, linear
    for i in range(1, 3000):
        assert attn._prefix_bytes(0, 1, 1, i, 64, 1, 1) > 0 and linear._lora_bytes(0, i, 64, 64, 8) > 0
    assert attn._prefix_bytes(0, 1, 65, 8, 8, 2, 2) == 0 and linear._lora_bytes(0, 4, 60, 64, 8) == 0
    assert attn._prefix_bytes.cache_info().currsize <= 1024 and linear._lora_bytes.cache_info().currsize <= 1024


def test_lora_refuses_a_result_over_its_rows():
    """Rows are read while others are written: Y may be the base as a whole, nothing else."""
    L, ws = _lib(), ctypes.c_void_p(1 << 30)

    def lora(Y, X, base, dtype=1, M=4, K=64, N=128):
        return L.qlmb_lora_add(ctypes.c_void_p(Y), ctypes.c_void_p(X), ctypes.c_void_p(base), dtype, ws, ws, ws, 2, ws, None, M, K, N, 8, ws, ctypes.c_size_t(1 << 30), None)

    big, far = 1 << 20, 1 << 24
    # Y of 4 x 128 and X of 4 x 64 bf16: 1024 and 512 bytes
    for y, x, base, dtype in ((big, big + 1008, far, 1), (big, big - 496, far, 1), (big, big + 2032, far, 0), (big, far, big + 1008, 1), (big, far, big - 16, 1), (big, big + 256, big, 1)):
        assert lora(y, x, base, dtype) == 1 and b"overlaps" in L.qlmb_last_error(), (y, x, base, dtype, L.qlmb_last_error())


@pytest.mark.gpu
def test_an_empty_batch(cuda):
    """A step without slots gives empty results, as lora_add does; rows without slots and slots without rows are refused."""
    from cudalm_c_b200 import attn, block, linear
    bf = torch.bfloat16
    q, k, kp, kc = (torch.zeros(s, dtype=bf, device=cuda) for s in ((0, 256), (0, 128), (9, 128), (0, 8, 128)))
    pos, tab = torch.zeros(0, dtype=torch.int32, device=cuda), torch.zeros(16, 32, device=cuda)
    assert block.dec_rope_kv(q, k, k, kc, kc, tab, tab, pos, 4, P=9).shape == (0, 256)
    o, lse = attn.dec_attn_prefix(q, kp, kp, kc, kc, pos, 4)
    assert o.shape == (0, 256) and o.dtype == bf and lse.shape == (0, 4) and lse.dtype == torch.float32
    out, count, lp = block.dec_verify(torch.zeros(0, 3, 50, device=cuda), torch.zeros(0, 2, dtype=torch.int32, device=cuda), torch.zeros(0, 3, device=cuda), torch.zeros(0, device=cuda))
    assert out.shape == lp.shape == (0, 3) and count.shape == (0,) and out.dtype == count.dtype == torch.int32
    A = torch.zeros(2, 8, 256, dtype=bf, device=cuda)
    assert linear.lora_add(q, q, A, A, torch.zeros(2, device=cuda), pos).shape == (0, 256)
    ok()
    rows, one = torch.zeros(2, 256, dtype=bf, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    for args in ((rows, kp, kp, kc, kc, pos, 4), (q, kp, kp, torch.zeros(1, 8, 128, dtype=bf, device=cuda), torch.zeros(1, 8, 128, dtype=bf, device=cuda), one, 4)):
        with pytest.raises(ValueError, match="dec_attn_prefix"):
            attn.dec_attn_prefix(*args)


_COLD = """
import sys; sys.path.insert(0, "tests")
import torch
from cudalm_c_b200 import attn, linear
import test_serving as t
dev = torch.device("cuda:0")
calls = []
for B, n, H, KV, P, Tm in ((2, 2, 4, 2, 100, 40), (40, 4, 4, 2, 300, 60), (16, 5, 16, 4, 5003, 40)):
    at = t.make_attn(B, n, H, KV, P, Tm, 91, dev)
    pos = t.positions(B, n, P, Tm, 92, dev)
    calls.append((lambda at=at, pos=pos, H=H: attn.dec_attn_prefix(*at, pos, H), lambda o, lse, at=at, pos=pos, H=H: t.check_attn(o, lse, t.attn64(*at, pos, H, 0))))
bf, f32 = torch.bfloat16, torch.float32
for M, K, N, R, n, dt in ((20, 72, 136, 8, 3, bf), (40, 1032, 4104, 16, 37, bf), (40, 1032, 2056, 72, 4, f32), (2100, 72, 136, 24, 5, f32), (2100, 136, 72, 72, 5, bf),
                          (2100, 264, 72, 128, 5, bf)):
    lo = t.make_lora(M, K, N, R, n, dt, 93, dev)
    ad = (torch.arange(M, device=dev, dtype=torch.int32) * 3) % n
    calls.append((lambda lo=lo, ad=ad: (linear.lora_add(*lo, ad),), lambda y, lo=lo, ad=ad: t.check_lora(y, *lo, ad)))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = [f() for f, _ in calls]
g.replay(); t.ok()
for (f, check), out in zip(calls, got):
    assert all(torch.equal(a, b) for a, b in zip(out, f()))
    check(*out)
t.ok(); print("equal")
"""


@pytest.mark.gpu
def test_every_form_may_be_captured_before_it_ever_ran(cuda):
    """The first calls of a process under capture, for every kernel with an attribute or tensor maps of its own."""
    r = _fresh_process(_COLD)
    assert r.returncode == 0 and "equal" in r.stdout, r.stderr[-2000:]


# ------------------------------------------------------------------ adapters: rows without one in the tiles of 128
@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,R,n", [(4200, 136, 1544, 16, 3), (4200, 2056, 1544, 16, 3), (6000, 72, 2056, 32, 2), (5000, 64, 1032, 256, 4), (4100, 200, 4104, 176, 1), (3000, 1032, 520, 64, 9), (20000, 72, 72, 16, 2)])
@pytest.mark.parametrize("mode", ["mixed", "runs", "first", "every other tile"])
def test_lora_tiles_with_rows_without_an_adapter(cuda, M, K, N, R, n, mode):
    """Pairs of a tile and no adapter, with more blocks of columns than the ring has stages, in front of and between pairs with one."""
    from cudalm_c_b200 import linear
    X, base, A, Bm, scale = make_lora(M, K, N, R, n, torch.bfloat16, M + N, cuda)
    rs = np.random.RandomState(M + R)
    a = rs.randint(-1, n, size=M)
    if mode == "runs":
        a = np.sort(a)
    elif mode == "first":
        a = np.where(np.arange(M) % 128 < 5, -1, a)
    elif mode == "every other tile":
        a = np.where(np.arange(M) // 128 % 2 == 0, -1, np.arange(M) // 256 % n)
    adapter = torch.from_numpy(a.astype(np.int32)).to(cuda)
    b0 = base.clone()
    for _ in range(3):
        y = linear.lora_add(X, base, A, Bm, scale, adapter)
        ok()
        check_lora(y, X, base, A, Bm, scale, adapter)
    assert torch.equal(base, b0)
    y2 = linear.lora_add(X, base, A, Bm, scale, adapter, out=base)
    ok()
    assert torch.equal(y2, y)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,R,n", [(2180, 4104, 8, 32, 2), (4200, 2056, 1544, 16, 3), (4100, 2048, 1496, 16, 9), (3000, 2048, 2056, 16, 70), (8200, 2048, 72, 16, 5), (2049, 2040, 264, 16, 40)])
@pytest.mark.parametrize("mode", ["runs", "mixed"])
def test_lora_of_many_rows_and_a_large_k(cuda, M, K, N, R, n, mode):
    """Both sides of the border between tiles of 128 rows and two launches."""
    test_lora(cuda, M, K, N, R, n, torch.bfloat16, mode)
