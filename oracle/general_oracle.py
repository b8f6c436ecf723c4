"""General attention (other key lengths, shared key heads, position bias) in 64 bits.

``attend`` computes the definition of ``cross_attention`` and ``relative_attention`` with
plain torch operations in float64, forward and gradients, and beside every result how far a
kernel may be off that keeps to the documented roundings:

* a value rounded to bfloat16 is off by at most ``eps / 2 = 2**-8`` of itself;
* probabilities (and dS) are rounded to bfloat16 before they are multiplied with V, dO, Q
  or K, so their products are off by at most ``2**-8`` of the sum of absolute products;
* delta = rowsum(O o dO) uses the rounded O; where the bias's gradient is wanted, O and the
  probabilities that made it have 16 bits instead (``exact``);
* exponentials, 32-bit sums and scores are off by less than ``2**-12`` of a probability.
"""
import math

import torch

HALF = 2.0 ** -8    # half a step of bfloat16, relative
FINE = 2.0 ** -12   # exponentials and 32-bit arithmetic
PAIR = 2.0 ** -16   # half a step of a value held as two of bfloat16


def bucket_of(relative, buckets, max_distance, both):
    """Bucket of relative positions (an int64 tensor, key minus query), by whole numbers."""
    side = buckets // 2 if both else buckets
    m = side // 2

    def one(r):
        if r < m:
            return r
        b = m
        while b < side - 1 and r ** (side - m) * m ** (b + 1 - m) >= max_distance ** (b + 1 - m) * m ** (side - m):
            b += 1
        return b

    table = torch.tensor([one(r) for r in range(max_distance + 1)], device=relative.device)
    d = (relative.abs() if both else (-relative).clamp(min=0)).clamp(max=max_distance)
    return table[d] + (side * (relative > 0) if both else 0)


def attend(q, k, v, do=None, bias=None, max_distance=128, both=False, causal=False, offsets=0, lengths=None, scale=None,
           exact=None):
    """``{"o", "lse", "dq", "dk", "dv", "dbias"}`` -> (value, allowed error), float64.

    q [B, Hq, Sq, D], k and v [B, Hkv, Sk, D]; lengths and offsets: lists or numbers."""
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    G = Hq // Hkv
    dev = q.device
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    exact = bias is not None and do is not None if exact is None else exact
    lengths = [Sk] * B if lengths is None else [min(max(int(n), 0), Sk) for n in lengths]
    offsets = [int(o) for o in offsets] if hasattr(offsets, "__len__") else [offsets] * B
    j = torch.arange(Sk, device=dev)
    i = torch.arange(Sq, device=dev)
    seen = torch.zeros(B, 1, Sq, Sk, dtype=torch.bool, device=dev)
    bucket = torch.zeros(B, Sq, Sk, dtype=torch.int64, device=dev)
    for b in range(B):
        r = j[None, :] - (i[:, None] + offsets[b])
        seen[b, 0] = (j < lengths[b])[None, :] & ((r <= 0) if causal else torch.ones_like(r, dtype=torch.bool))
        if bias is not None:
            bucket[b] = bucket_of(r, bias.shape[0], max_distance, both)
    key_in = seen.any(2)[:, 0]  # keys that someone sees; the others may hold anything
    qd = q.detach().double()
    kd = torch.where(key_in[:, None, :, None], k.detach().double(), 0.0).repeat_interleave(G, 1)
    vd = torch.where(key_in[:, None, :, None], v.detach().double(), 0.0).repeat_interleave(G, 1)
    s = qd @ kd.transpose(-1, -2) * scale
    if bias is not None:
        s = s + bias.detach().double()[bucket].permute(0, 3, 1, 2)
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True) if Sk else torch.full((B, Hq, Sq, 1), -math.inf, dtype=torch.float64, device=dev)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    o = p @ vd
    o_err = HALF * o.abs() + (HALF + FINE) * (p @ vd.abs()) + 1e-7
    lse = ((torch.where(top == -math.inf, 0.0, top) + torch.log(total)) / math.log(2.0))[..., 0]
    out = {"o": (o, o_err), "lse": (lse, FINE + 1e-6 * lse.abs())}
    if do is None:
        return out
    dd = do.detach().double()
    dp = dd @ vd.transpose(-1, -2)
    delta = (dd * o).sum(-1, keepdim=True)
    part = PAIR if exact else HALF
    delta_err = (dd.abs() * (part * o.abs() + (part + FINE) * (p @ vd.abs()))).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    sure = FINE * (p * (dp.abs() + delta.abs())) + p * delta_err  # of dS in 32 bits
    ds_err = HALF * ds.abs() + (1 + HALF) * sure
    def fold(x):  # heads that share a key head
        return x.view(B, Hkv, G, Sk, D).sum(2)
    dq, dq_err = ds @ kd * scale, ds_err @ kd.abs() * abs(scale)
    dk, dk_err = fold(ds.transpose(-1, -2) @ qd) * scale, fold(ds_err.transpose(-1, -2) @ qd.abs()) * abs(scale)
    dv, dv_err = fold(p.transpose(-1, -2) @ dd), fold((HALF + FINE) * (p.transpose(-1, -2) @ dd.abs()))
    for name, x, err in (("dq", dq, dq_err), ("dk", dk, dk_err), ("dv", dv, dv_err)):
        out[name] = (x, err + HALF * x.abs() + 1e-7)
    if bias is not None:
        db, db_err = (torch.zeros(Hq, bias.shape[0], dtype=torch.float64, device=dev) for _ in range(2))
        for b in range(B):
            place = bucket[b].reshape(1, -1).expand(Hq, -1)
            db.scatter_add_(1, place, ds[b].reshape(Hq, -1))
            db_err.scatter_add_(1, place, sure[b].reshape(Hq, -1))
        out["dbias"] = (db.t(), (db_err + HALF * db.abs()).t() + 1e-7)
    return out
