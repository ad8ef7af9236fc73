"""What the operators of a decode step for many requests at once are timed on.

A case is one of four calls, by its "op":

  append   block.dec_rope_kv: queries and keys of the slots' new tokens rotated, keys and values appended to the slots' caches
  prefix   attn.dec_attn_prefix: attention of the new tokens over a prefix that all slots share and each slot's own rows
  verify   block.dec_verify: drafted tokens tested against the model's logits, with the token that follows them
  lora     linear.lora_add: every row's own low-rank adapter beside a projection that the rows share

Every operator has its plain form here, in elementary torch operations (`own` false), and its definition in 64 bits
(`exact`).  Inputs are synthetic: activations, queries, keys and values N(0, 1), adapters N(0, 0.02), logits with the spread
of a trained head and drafts from a distribution near the model's.
"""
import math

import numpy as np
import torch

own = False

HD = 64                                     # the framework's head dimension
DTYPES = {"bf16": (torch.bfloat16, 2), "f32": (torch.float32, 4)}


def listed():
    return [
        # one new token of one user: launch latency
        dict(name="append_b1", op="append", B=1, n=1, H=12, KV=12, P=512, fill=64, Tm=1024),
        # a full server, four drafted tokens and the one before them in every slot
        dict(name="append_b64_n5", op="append", B=64, n=5, H=16, KV=4, P=8192, fill=1024, Tm=2048),
        # one user behind a short system prompt: the smallest call
        dict(name="prefix_b1_p512", op="prefix", B=1, n=1, H=12, KV=12, P=512, fill=64, Tm=1024, win=0),
        # a small batch that verifies three drafted tokens
        dict(name="prefix_b8_n4_p2048", op="prefix", B=8, n=4, H=12, KV=12, P=2048, fill=333, Tm=1024, win=0),
        # a full server, one token a slot, a long instruction in front of all of them
        dict(name="prefix_b64_p8192", op="prefix", B=64, n=1, H=12, KV=12, P=8192, fill=512, Tm=1024, win=0),
        # questions about one long document, drafted tokens, grouped heads: the largest
        dict(name="prefix_b64_n5_p32768", op="prefix", B=64, n=5, H=16, KV=4, P=32768, fill=1024, Tm=2048, win=0),
        # one user, four drafts from a small model that hands over its probabilities
        dict(name="verify_b1_v16384", op="verify", B=1, n=4, V=16384, ld=16384, dtype="f32", draft="dense", temps="sample", ragged=False),
        # a full server: greedy and sampling slots side by side, fewer drafts in some
        dict(name="verify_b64_v16384", op="verify", B=64, n=4, V=16384, ld=16384, dtype="f32", draft="dense", temps="mixed", ragged=True),
        # a large vocabulary whose head is padded, drafts looked up in the text so far (no probabilities)
        dict(name="verify_b32_v130001", op="verify", B=32, n=7, V=130001, ld=130048, dtype="f32", draft="point", temps="sample", ragged=False),
        # one row of one user at the model's width
        dict(name="lora_1x768x768_r8", op="lora", M=1, K=768, N=768, R=8, adapters=4, used=1, dtype="bf16", grouped=True),
        # a full server, every slot its own adapter, beside a large matrix
        dict(name="lora_64x4096x16384_r16", op="lora", M=64, K=4096, N=16384, R=16, adapters=64, used=64, dtype="bf16", grouped=False),
        # prompts of several users in one batch of rows
        dict(name="lora_8192x768x1536_r64", op="lora", M=8192, K=768, N=1536, R=64, adapters=16, used=9, dtype="bf16", grouped=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "prefix", "prefix", "verify", "verify", "lora", "lora"))
    if op in ("append", "prefix"):
        kv = rng.choice((1, 2, 4, 8, 12))
        g = rng.choice((1, 1, 2, 3, 4, 8))
        while kv * g > 32:
            g -= 1
        fill = _log(rng, 1, 2048)
        c = dict(op=op, B=_log(rng, 1, 64), n=rng.choice((1, 1, 2, 3, 5, 8, 16)), H=kv * g, KV=kv, P=_log(rng, 1, 32768) if rng.random() < 0.9 else 0,
                 fill=fill, Tm=fill + rng.choice((16, 17, 1000)))
        if op == "append":
            return c
        c["win"] = rng.choice((0, 0, 0, 256, 4096))
        while c["B"] * c["n"] * c["H"] * (c["P"] + fill) > 64 * 5 * 16 * 33000:       # the largest listed case's work
            c["B"] = max(1, c["B"] // 2)
            c["P"] = c["P"] * 3 // 4
        return c
    if op == "verify":
        V = _log(rng, 100, 131072)
        c = dict(op=op, B=_log(rng, 1, 64), n=rng.choice((0, 1, 2, 4, 5, 8)), V=V, ld=V + rng.choice((0, 0, 1, 64)), dtype=rng.choice(("f32", "f32", "bf16")),
                 draft=rng.choice(("dense", "point")), temps=rng.choice(("sample", "greedy", "mixed")), ragged=rng.random() < 0.5)
        while c["B"] * (c["n"] + 1) * V > 32 * 8 * 130048:
            c["B"] = max(1, c["B"] // 2)
        return c
    K, N = 8 * _log(rng, 16, 512), 8 * _log(rng, 16, 2048)
    M = _log(rng, 1, 8192)
    R = 8 * rng.choice((1, 2, 2, 3, 4, 8, 16))
    while M * (K + 2 * N) > 64 * 8192 * 64:                                             # keeps to a few hundred MB
        M = max(1, M // 2)
    adapters = _log(rng, 1, 64)
    return dict(op=op, M=M, K=K, N=N, R=R, adapters=adapters, used=max(1, min(adapters, M, _log(rng, 1, 64))), dtype=rng.choice(("bf16", "bf16", "f32")),
                grouped=rng.random() < 0.7)


def _positions(c, seed):
    """Absolute position of every slot's first new token: the slots joined at different times."""
    rs = np.random.RandomState(seed % (2 ** 31))
    hi = max(1, c["fill"])
    return c["P"] + rs.randint(hi // 2, hi, size=c["B"])


def _adapters(c, seed):
    """Every row's adapter (-1: none), in runs of rows (prompts) or one by one (slots)."""
    rs = np.random.RandomState((seed + 1) % (2 ** 31))
    ids = rs.permutation(c["adapters"])[:c["used"]]
    if c["grouped"]:
        cuts = np.sort(rs.randint(0, c["M"] + 1, size=c["used"] - 1)) if c["used"] > 1 else np.zeros(0, int)
        a = ids[np.searchsorted(cuts, np.arange(c["M"]), side="right")]
        if c["M"] > 64 and c["used"] > 1:
            a = np.where(a == ids[-1], -1, a)             # one request without an adapter
    else:
        a = ids[rs.randint(0, c["used"], size=c["M"])] if c["used"] < c["M"] else ids[np.arange(c["M"]) % c["used"]]
    return a.astype(np.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    s, op = dict(case), case["op"]
    bf = torch.bfloat16

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    if op in ("append", "prefix"):
        B, n, kd = s["B"], s["n"], s["KV"] * HD
        pos = _positions(case, seed)
        s["pos"] = torch.from_numpy(pos.astype(np.int32)).to(dev)
        s["q"] = randn(B * n, s["H"] * HD).to(bf)
        s["kc"], s["vc"] = (torch.empty(B, s["Tm"], kd, dtype=bf, device=dev) for _ in range(2))
        for b in range(B):                                # slot by slot: no fp32 copy of the whole cache
            for x in (s["kc"], s["vc"]):
                x[b] = randn(s["Tm"], kd)
        if op == "append":
            s["k"], s["v"] = (randn(B * n, kd).to(bf) for _ in range(2))
            rows = s["P"] + s["Tm"]
            ang = torch.arange(rows, dtype=torch.float64)[:, None] * (10000.0 ** (-torch.arange(HD // 2, dtype=torch.float64) * 2.0 / HD))[None, :]
            s["cos"], s["sin"] = ang.cos().float().to(dev), ang.sin().float().to(dev)
        else:
            s["kp"], s["vp"] = (randn(s["P"], kd).to(bf) for _ in range(2))
    elif op == "verify":
        B, n, V = s["B"], s["n"], s["V"]
        lg = torch.zeros(B, n + 1, s["ld"], device=dev)
        lg[:, :, :V] = randn(B, n + 1, V) * 2.5
        s["logits"] = lg.to(DTYPES[s["dtype"]][0])
        t = torch.rand(B, device=dev, generator=g) * 1.2 + 0.3
        if s["temps"] == "greedy":
            t.zero_()
        elif s["temps"] == "mixed":
            t[::3] = 0.0
        s["temp"] = t
        tt = torch.where(t > 0, t, torch.full_like(t, 0.5))[:, None, None]
        dl = (s["logits"][:, :n, :V].float() + 0.6 * randn(B, n, V)) / tt
        q = torch.softmax(dl, -1)
        if n == 0:
            s["x"] = torch.zeros(B, 0, dtype=torch.int32, device=dev)
        elif s["draft"] == "dense":
            s["x"] = torch.argmax(dl - torch.log(-torch.log(torch.rand(B, n, V, device=dev, generator=g).clamp(1e-9, 1 - 1e-7))), -1).int()
        else:
            s["x"] = dl.argmax(-1).int()
        s["q"] = q.contiguous() if s["draft"] == "dense" else None
        s["u"] = torch.rand(B, n + 1, device=dev, generator=g)
        s["nd"] = torch.randint(0, n + 1, (B,), device=dev, generator=g, dtype=torch.int32) if s["ragged"] else None
        del lg, dl, q
    elif op == "lora":
        M, K, N, R = (s[k] for k in "MKNR")
        dt = DTYPES[s["dtype"]][0]
        s["x"], s["base"] = randn(M, K).to(dt), randn(M, N).to(dt)
        s["a"], s["b"] = (randn(s["adapters"], R, K) * 0.02).to(bf), (randn(s["adapters"], R, N) * 0.02).to(bf)
        s["scale"] = torch.rand(s["adapters"], device=dev, generator=g) * 2.0 + 0.5
        a = _adapters(case, seed)
        s["adapter"] = torch.from_numpy(a).to(dev)
        # what a serving program keeps for as long as its batch stays the same: the rows in the order of their adapters
        s["order"] = None if s["grouped"] else torch.from_numpy(np.argsort(a, kind="stable").astype(np.int32)).to(dev)
        s["groups"] = [(int(i), torch.from_numpy(np.nonzero(a == i)[0]).to(dev)) for i in np.unique(a) if i >= 0]
    else:
        raise ValueError(op)
    return s


def run(s):
    return {"append": _append, "prefix": _prefix, "verify": _verify, "lora": _lora}[s["op"]](s)


def _append(s):
    if own:
        from cudalm_c_b200 import block
        q = block.dec_rope_kv(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["cos"], s["sin"], s["pos"], s["H"], P=s["P"])
        return {"q": q, "kc": s["kc"], "vc": s["vc"]}
    B, n, hf = s["B"], s["n"], HD // 2
    t = s["pos"].long()[:, None] + torch.arange(n, device=s["pos"].device)
    c, sn = s["cos"][t].view(B * n, 1, hf), s["sin"][t].view(B * n, 1, hf)

    def rotate(x):
        x = x.float().view(B * n, -1, HD)
        a, b = x[..., :hf], x[..., hf:]
        return torch.cat((a * c - b * sn, b * c + a * sn), -1).view(B * n, -1).bfloat16()

    slot = torch.arange(B, device=t.device)[:, None].expand(B, n)
    s["kc"][slot, t - s["P"]] = rotate(s["k"]).view(B, n, -1)
    s["vc"][slot, t - s["P"]] = s["v"].view(B, n, -1)
    return {"q": rotate(s["q"]), "kc": s["kc"], "vc": s["vc"]}


def _prefix(s):
    if own:
        from cudalm_c_b200 import attn
        o, lse = attn.dec_attn_prefix(s["q"], s["kp"], s["vp"], s["kc"], s["vc"], s["pos"], s["H"], win=s["win"])
        return {"o": o, "lse": lse}
    B, n, H, KV, P, Tm, win = (s[k] for k in ("B", "n", "H", "KV", "P", "Tm", "win"))
    G, dev = H // KV, s["q"].device
    q = s["q"].float().view(B, n, KV, G, HD) * (1.0 / math.sqrt(HD))
    t = s["pos"].long()[:, None] + torch.arange(n, device=dev)                                   # [B, n]
    # the shared rows: one product per head for the rows of all slots
    sp = torch.matmul(q.permute(2, 0, 1, 3, 4).reshape(KV, B * n * G, HD), s["kp"].float().view(P, KV, HD).permute(1, 2, 0))
    sp = sp.view(KV, B, n, G, P).permute(1, 0, 2, 3, 4)
    # the slots' own rows
    so = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(B, KV, n * G, HD), s["kc"].float().view(B, Tm, KV, HD).permute(0, 2, 3, 1))
    so = so.view(B, KV, n, G, Tm)
    j = torch.arange(Tm, device=dev) + P
    hide = j[None, None, :] > t[:, :, None]
    if win > 0:
        sp = sp.masked_fill((torch.arange(P, device=dev)[None, None, :] <= (t - win)[:, :, None])[:, None, :, None, :], -math.inf)
        hide = hide | (j[None, None, :] <= (t - win)[:, :, None])
    so = so.masked_fill(hide[:, None, :, None, :], -math.inf)
    m = so.amax(-1, keepdim=True)
    if P:
        m = torch.maximum(m, sp.amax(-1, keepdim=True))
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    sp, so = torch.exp(sp - m), torch.exp(so - m)
    l = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)                                      # [B, KV, n, G, 1]
    o = torch.matmul(sp.permute(1, 0, 2, 3, 4).reshape(KV, B * n * G, P), s["vp"].float().view(P, KV, HD).permute(1, 0, 2))
    o = o.view(KV, B, n, G, HD).permute(1, 0, 2, 3, 4)
    o = o + torch.matmul(so.reshape(B, KV, n * G, Tm), s["vc"].float().view(B, Tm, KV, HD).permute(0, 2, 1, 3)).view(B, KV, n, G, HD)
    o = torch.where(l > 0, o / l, torch.zeros_like(o))
    lse = (m + torch.log(l)).squeeze(-1)
    return {"o": o.permute(0, 2, 1, 3, 4).reshape(B * n, H * HD).bfloat16(), "lse": lse.permute(0, 2, 1, 3).reshape(B * n, H)}


def _verify(s):
    B, n, V = s["B"], s["n"], s["V"]
    if own:
        from cudalm_c_b200 import block
        out, count, lp = block.dec_verify(s["logits"], s["x"], s["u"], s["temp"], q=s["q"], nd=s["nd"], V=V)
        return {"out": out, "count": count, "lp": lp}
    dev = s["logits"].device
    lg = s["logits"][:, :, :V].double()
    m, top = lg.amax(-1, keepdim=True), lg.argmax(-1)                                            # [B, n + 1]
    greedy = (s["temp"] <= 0)[:, None]
    T = torch.where(s["temp"] > 0, s["temp"], torch.ones_like(s["temp"])).double()[:, None, None]
    e = torch.exp((lg - m) / T)
    p = e / e.sum(-1, keepdim=True)
    nd = s["nd"].long() if s["nd"] is not None else torch.full((B,), n, dtype=torch.long, device=dev)
    x = s["x"].long()
    ends = torch.arange(n, device=dev)[None, :] >= nd[:, None]
    px = torch.gather(p[:, :n], 2, x[:, :, None]).squeeze(-1)
    qx = torch.gather(s["q"], 2, x[:, :, None]).squeeze(-1).double() if s["q"] is not None else torch.ones_like(px)
    ok = torch.where(greedy, x == top[:, :n], s["u"][:, :n].double() * qx < px) & ~ends
    r = torch.cumprod(ok.long(), -1).sum(-1)                                                     # tokens accepted
    slot = torch.arange(B, device=dev)
    pr = p[slot, r]
    tested = r < nd
    w = pr
    if n:
        at = r.clamp(max=n - 1)
        if s["q"] is not None:
            rest = torch.clamp(pr - s["q"][slot, at].double(), min=0.0)
        else:
            rest = pr.scatter(1, x[slot, at][:, None], 0.0)
        w = torch.where((tested & (rest.sum(-1) > 0))[:, None], rest, pr)
    cum = torch.cumsum(w, -1)
    pick = (cum > (s["u"][:, n].double() * cum[:, -1])[:, None]).int().argmax(-1)
    pick = torch.where(greedy[:, 0], top[slot, r], pick)
    i = torch.arange(n + 1, device=dev)[None, :]
    tok = torch.cat((x, torch.zeros(B, 1, dtype=torch.long, device=dev)), -1)
    tok = torch.where(i < r[:, None], tok, torch.where(i == r[:, None], pick[:, None], torch.full_like(tok, -1)))
    lz = m.squeeze(-1) + torch.log(torch.exp(lg - m).sum(-1))
    lp = torch.gather(lg, 2, tok.clamp(min=0)[:, :, None]).squeeze(-1) - lz
    return {"out": tok.int(), "count": (r + 1).int(), "lp": torch.where(tok >= 0, lp, torch.zeros_like(lp)).float()}


def _lora(s):
    if own:
        from cudalm_c_b200 import linear
        # fp32 rows are added to where they are, as below, where float() makes no copy of them
        out = s["base"] if s["base"].dtype == torch.float32 else None
        return linear.lora_add(s["x"], s["base"], s["a"], s["b"], s["scale"], s["adapter"], order=s["order"], out=out)
    y = s["base"].float()
    for i, rows in s["groups"]:
        t = torch.matmul(s["x"][rows].float(), s["a"][i].float().t())
        y[rows] += torch.matmul(t, s["b"][i].float()) * s["scale"][i]
    return y.to(s["base"].dtype)


def work(case):
    c, op = case, case["op"]
    if op == "append":
        rows = c["B"] * c["n"]
        return {"bytes": rows * ((2 * c["H"] + 4 * c["KV"]) * HD * 2 + HD * 4) + c["B"] * 4, "flops": rows * (c["H"] + c["KV"]) * HD * 3}
    if op == "prefix":
        rows = c["B"] * c["n"]
        mine = 0.75 * c["fill"] + 0.5 * (c["n"] + 1)                                             # own rows that a token sees, on average
        shared = c["P"]
        if c["win"] > 0:
            shared = max(0.0, min(c["P"], c["win"] - mine))
            mine = min(mine, c["win"])
        last = min(mine + 0.5 * (c["n"] - 1), c["Tm"])                                           # rows that some token of the slot sees
        return {"bytes": int(2 * 2 * c["KV"] * HD * (shared + c["B"] * last) + rows * c["H"] * (HD * 2 * 2 + 4)),
                "flops": int(4 * HD * rows * c["H"] * (shared + mine))}
    if op == "verify":
        size = DTYPES[c["dtype"]][1]
        # logits up to the row that ends a slot: every second draft fails or is missing, more or less
        rows = sum(0.5 ** i for i in range(c["n"] + 1))
        q = 4 if c["draft"] == "dense" and c["n"] and c["temps"] != "greedy" else 0
        return {"bytes": int(c["B"] * c["V"] * (rows * size + 0.5 * q) + c["B"] * (c["n"] + 1) * 16), "flops": int(c["B"] * c["V"] * rows * 20)}
    size = DTYPES[c["dtype"]][1]
    return {"bytes": c["M"] * (c["K"] + 2 * c["N"]) * size + c["used"] * c["R"] * (c["K"] + c["N"]) * 2 + c["M"] * 4,
            "flops": 2 * c["M"] * c["R"] * (c["K"] + c["N"])}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f8 = torch.float64
    if op == "append":
        host = {k: s[k].to("cpu", f8).numpy() for k in ("q", "k", "v", "cos", "sin")}
        t = (s["pos"].cpu().numpy()[:, None] + np.arange(s["n"])[None, :]).reshape(-1)
        slot = np.repeat(np.arange(s["B"]), s["n"])
        z = np.exp(1j * np.arctan2(host["sin"][t], host["cos"][t])) * np.hypot(host["sin"][t], host["cos"][t])

        def turn(x):
            h = x.reshape(len(t), -1, 2, HD // 2)
            y = (h[:, :, 0] + 1j * h[:, :, 1]) * z[:, None, :]
            return np.stack((y.real, y.imag), 2).reshape(x.shape)

        kc, vc = (s[k].to("cpu", f8).numpy() for k in ("kc", "vc"))
        kc[slot, t - s["P"]] = turn(host["k"])
        vc[slot, t - s["P"]] = host["v"]
        return {"q": turn(host["q"]), "kc": kc, "vc": vc}
    if op == "prefix":
        B, n, H, KV, P = (s[k] for k in ("B", "n", "H", "KV", "P"))
        G = H // KV
        o = torch.zeros(B, n, H, HD, dtype=f8, device=s["q"].device)
        lse = torch.full((B, n, H), -math.inf, dtype=f8, device=s["q"].device)
        q = s["q"].view(B, n, H, HD)
        pos = s["pos"].tolist()
        for b in range(B):
            for i in range(n):
                t = pos[b] + i
                lo = max(0, t - s["win"] + 1) if s["win"] > 0 else 0
                k = torch.cat((s["kp"][lo:], s["kc"][b, max(0, lo - P):t - P + 1])).to(f8).view(-1, KV, HD)
                v = torch.cat((s["vp"][lo:], s["vc"][b, max(0, lo - P):t - P + 1])).to(f8).view(-1, KV, HD)
                if k.shape[0] == 0:
                    continue
                w = torch.einsum("hgd,khd->hgk", q[b, i].to(f8).view(KV, G, HD), k) / 8.0
                lse[b, i] = torch.logsumexp(w, -1).view(H)
                o[b, i] = torch.einsum("hgk,khd->hgd", torch.softmax(w, -1), v).reshape(H, HD)
        return {"o": o.view(B * n, H * HD), "lse": lse.view(B * n, H)}
    if op == "verify":
        B, n, V = s["B"], s["n"], s["V"]
        out, count, lp = np.full((B, n + 1), -1, np.int32), np.zeros(B, np.int32), np.zeros((B, n + 1))
        x, u, temp = s["x"].cpu().numpy(), s["u"].cpu().numpy().astype(np.float64), s["temp"].cpu().numpy().astype(np.float64)
        nd = s["nd"].cpu().numpy() if s["nd"] is not None else np.full(B, n)
        for b in range(B):
            for i in range(n + 1):
                lg = s["logits"][b, i, :V].to("cpu", f8).numpy()
                lsm = lg - lg.max()
                lsm -= math.log(math.fsum(np.exp(lsm)))
                if temp[b] > 0:
                    p = np.exp((lg - lg.max()) / temp[b])
                    p /= p.sum()
                last = i == nd[b]
                if not last:
                    d = x[b, i]
                    qd = float(s["q"][b, i, d]) if s["q"] is not None else 1.0
                    if (lg.argmax() == d) if temp[b] <= 0 else (u[b, i] * qd < p[d]):
                        out[b, i], lp[b, i] = d, lsm[d]
                        continue
                if temp[b] <= 0:
                    pick = int(lg.argmax())
                else:
                    w = p
                    if not last:
                        if s["q"] is not None:
                            w = np.maximum(p - s["q"][b, i].to("cpu", f8).numpy(), 0.0)
                        else:
                            w = p.copy()
                            w[x[b, i]] = 0.0
                        if not w.sum() > 0:
                            w = p
                    cum = np.cumsum(w)
                    pick = int(np.searchsorted(cum, u[b, n] * cum[-1], side="right"))
                out[b, i], lp[b, i], count[b] = pick, lsm[pick], i + 1
                break
        return {"out": out, "count": count, "lp": lp}
    y = s["base"].to(f8)
    a = s["adapter"].long()
    for i in range(s["adapters"]):
        mine = (a == i).to(f8)[:, None]
        d = torch.einsum("mr,rn->mn", torch.einsum("mk,rk->mr", s["x"].to(f8) * mine, s["a"][i].to(f8)), s["b"][i].to(f8))
        y = y + d * s["scale"][i].to(f8)
    return y
