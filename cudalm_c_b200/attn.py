"""Host-side mirror of the reference's attention operators (e_attn, cudalm.cu:3705-3730, and the
attention part of gpu_backward, cudalm.cu:5918-5960) over the C ABI."""
from functools import lru_cache

import torch

from ._lib import calls, check, device_index, lib, need, ptr, stream_ptr


def attn_fwd(Q, K, V, B, T, H, KV, win=0):
    """Causal attention: Q [B*T, H*64], K, V [B*T, KV*64] bf16 -> O bf16, lse [B, H, T] fp32."""
    O = torch.empty_like(Q)
    lse = torch.empty(B, H, T, dtype=torch.float32, device=Q.device)
    calls.attn_fwd(O, lse, Q, K, V, B, T, H, KV, 64, win, stream_ptr())
    return O, lse


def attn_bwd(Q, K, V, O, dA, lse, B, T, H, KV, win=0, rope=None):
    """Gradients of attn_fwd's inputs: dQ, dK, dV (bf16) and drow = rowsum(dA * O) [B, H, T].  With rope = (cos, sin) tables
    dQ and dK are rotated back, i.e. gradients of what block.rope was applied to."""
    dQ, dK, dV = torch.empty_like(Q), torch.empty_like(K), torch.empty_like(V)
    drow = torch.empty(B, H, T, dtype=torch.float32, device=Q.device)
    if rope is None:
        calls.attn_bwd(dQ, dK, dV, drow, Q, K, V, O, dA, lse, B, T, H, KV, 64, win, stream_ptr())
    else:
        check(lib().qlmb_attn_bwd_rope(ptr(dQ), ptr(dK), ptr(dV), ptr(drow), ptr(Q), ptr(K), ptr(V), ptr(O), ptr(dA), ptr(lse),
                                       ptr(rope[0]), ptr(rope[1]), B, T, H, KV, 64, win, stream_ptr()))
    return dQ, dK, dV, drow


@lru_cache(maxsize=1024)                                 # a ctypes call, 2 us; a server's shapes change from step to step
def _prefix_bytes(dev, *shape):
    """Bytes of dec_attn_prefix's scratch on a device, for (B, n, P, Tm, H, KV)."""
    return lib().qlmb_dec_attn_prefix_bytes(*shape)


def _dec_attn_prefix_args(Q, Kp, Vp, Kc, Vc, pos, H):
    bf = torch.bfloat16
    B = need("pos", pos, torch.int32, None).shape[0]
    Tm, KD = need("Kc", Kc, bf, B, None, None).shape[1:]
    need("Vc", Vc, bf, B, Tm, KD)
    P = need("Kp", Kp, bf, None, KD).shape[0]
    need("Vp", Vp, bf, P, KD)
    rows = need("Q", Q, bf, None, H * 64).shape[0]
    raise ValueError("dec_attn_prefix: %d rows of queries for %d slots, keys of %d columns, a cache of %d rows" % (rows, B, KD, Tm))


def dec_attn_prefix(Q, Kp, Vp, Kc, Vc, pos, H, win=0):
    """Attention of a decode step over a prefix that the slots share: Q [B*n, H*64], Kp and Vp [P, KD], caches Kc and Vc [B, Tm, KD]
    bf16, pos [B] int32 = absolute position of each slot's first new token (its cache row is pos - P).  Returns O [B*n, H*64] bf16 and
    the scores' log-sum-exp [B*n, H] fp32."""
    dev = device_index()
    got = calls.sizes(dev, torch.bfloat16, Q, "rw", Kc, "btk", Vc, "btk", Kp, "pk", Vp, "pk", torch.int32, pos, "b")
    if got is None or not (got[1] == H * 64 and got[4] % 64 == 0 and (got[0] % got[2] == 0 < got[0] if got[2] else got[0] == 0)):
        _dec_attn_prefix_args(Q, Kp, Vp, Kc, Vc, pos, H)
    rows, _, B, Tm, KD, P = got
    if B == 0:
        return torch.empty_like(Q), Q.new_empty((0, H), dtype=torch.float32)
    shape = (B, rows // B, P, Tm, H, KD // 64)
    nbytes = _prefix_bytes(dev, *shape)
    O = torch.empty_like(Q)
    lse = torch.empty_strided((rows, H), (H, 1), dtype=torch.float32, device=Q.device)         # (torch.empty: 0.9 us more)
    ws = Q.new_empty(nbytes + 1 >> 1) if nbytes > 16 else None
    calls.dec_attn_prefix(O, lse, Q, Kp, Vp, Kc, Vc, pos, win, *shape, 64, ws, nbytes, stream_ptr())
    return O, lse
