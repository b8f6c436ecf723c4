"""Cases that measure cross attention and attention with a learned relative position bias.

Both come in the forms that a program uses: a step of a few tokens over states or a cache
that are already there, a prompt (forward alone) and a training step (forward and backward).
``run`` computes a case either in its plain form, with elementary torch operations in 32
bits, or, where ``own`` is true, through the package's public functions.
"""
import math

import torch

own = False

_CARD = "cuda"


# ------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------
def _cross(name, form, B, Hq, Hkv, Sq, Sk, D, ragged, layout):
    return {"name": name, "op": "cross", "form": form, "B": B, "Hq": Hq, "Hkv": Hkv, "Sq": Sq, "Sk": Sk, "D": D,
            "ragged": ragged, "layout": layout}


def _relative(name, form, B, Hq, Hkv, Sq, Sk, D, ragged, layout, causal, buckets, distance):
    return {"name": name, "op": "relative", "form": form, "B": B, "Hq": Hq, "Hkv": Hkv, "Sq": Sq, "Sk": Sk, "D": D,
            "ragged": ragged, "layout": layout, "causal": causal, "buckets": buckets, "distance": distance}


def listed():
    return [
        # one token of one sequence over a short encoded text: latency alone
        _cross("cross step small", "step", 1, 12, 12, 1, 77, 64, False, "bhsd"),
        # one token of each of 64 sequences over encoded audio, a cache of encoder keys and values
        _cross("cross step batch", "step", 64, 16, 16, 1, 1500, 64, True, "bhsd"),
        # a few tokens over a very long source, key heads shared by 8 query heads, few rows in all
        _cross("cross step long", "step", 2, 32, 4, 3, 50001, 128, True, "bshd"),
        # decoder prompts over padded sources
        _cross("cross prompt", "prompt", 16, 20, 20, 224, 1500, 64, True, "bshd"),
        # image positions that look at a short text: few keys, many queries
        _cross("cross train short keys", "train", 8, 10, 10, 4096, 77, 64, False, "bshd"),
        # an encoder-decoder's training step with shared key heads and padded sources
        _cross("cross train", "train", 4, 32, 8, 2048, 4001, 128, True, "bshd"),
        # one new token of one short sequence
        _relative("relative step small", "step", 1, 8, 8, 1, 40, 64, False, "bhsd", True, 32, 128),
        # one new token of each of 32 sequences over their caches, of different lengths
        _relative("relative step batch", "step", 32, 16, 16, 1, 2048, 64, True, "bhsd", True, 32, 128),
        # a chunk of new tokens over a cache with shared key heads
        _relative("relative chunk", "chunk", 2, 32, 8, 500, 8192, 128, True, "bhsd", True, 32, 128),
        # an encoder over padded sentences
        _relative("relative encoder", "prompt", 16, 12, 12, 512, 512, 64, True, "bshd", False, 32, 128),
        # its training step, an odd length
        _relative("relative encoder train", "train", 8, 12, 12, 1000, 1000, 64, True, "bshd", False, 32, 128),
        # a decoder's training step at the longer end
        _relative("relative decoder train", "train", 2, 16, 16, 4096, 4096, 128, False, "bshd", True, 64, 256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


#: Most score entries (batch x query heads x queries x keys) of a drawn case, and most of its
#: multiply-adds: those of the largest listed case, a little less.
_MOST_SCORES = 4 * 32 * 2048 * 4001 * 0.9


def draw(rng):
    while True:
        op = rng.choice(["cross", "relative"])
        form = rng.choice(["step", "prompt", "train"] if op == "cross" else ["step", "chunk", "prompt", "train"])
        group = rng.choice([1, 1, 2, 4, 8])
        hkv = rng.choice([1, 2, 3, 4, 8, 12, 16])
        c = {"op": op, "form": form, "Hq": group * hkv, "Hkv": hkv, "D": rng.choice([32, 40, 64, 64, 80, 96, 128, 128]),
             "ragged": rng.random() < 0.6, "layout": rng.choice(["bhsd", "bshd"])}
        if form == "step":
            c.update(B=_log(rng, 1, 96), Sq=rng.choice([1, 1, 1, 2, 3, 4]), Sk=_log(rng, 16, 32768))
        elif op == "cross":
            c.update(B=_log(rng, 1, 16), Sq=_log(rng, 16, 8192), Sk=_log(rng, 16, 8192))
        else:
            c.update(B=_log(rng, 1, 16), Sq=_log(rng, 16, 4096))
            c["Sk"] = c["Sq"] if form != "chunk" else c["Sq"] + _log(rng, 16, 8192)
        if op == "relative":
            c["causal"] = True if form in ("step", "chunk") else rng.random() < 0.5
            c["buckets"], c["distance"] = rng.choice([(32, 128), (32, 128), (64, 256), (16, 64), (128, 800)])
        scores = c["B"] * c["Hq"] * c["Sq"] * c["Sk"]
        states = c["B"] * c["Hkv"] * c["Sk"]
        # a training step computes 3.5 times a forward's products: the cap holds for both
        if scores > _MOST_SCORES or (form != "train" and scores * c["D"] > 3 * _MOST_SCORES * 128):
            continue
        if form == "step" and states * c["D"] > 64 * 16 * 1500 * 64:
            continue
        return c


# ------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------
def _lengths(case):
    """The key lengths of a padded batch: spread from a quarter of the longest to the longest."""
    B, Sk, least = case["B"], case["Sk"], case["Sq"] if case["form"] in ("step", "chunk") and case["op"] == "relative" else 1
    if B == 1:
        return [max(least, (Sk * 7) // 8)]
    low = max(least, Sk // 4)
    return [low + ((Sk - low) * b) // (B - 1) for b in range(B)]


def prepare(case, seed):
    g = torch.Generator(device=_CARD).manual_seed(seed)
    B, Hq, Hkv, Sq, Sk, D = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    relative, train = case["op"] == "relative", case["form"] == "train"

    def tensor(H, S, size=1.0):
        shape = (B, S, H, D) if case["layout"] == "bshd" else (B, H, S, D)
        t = (torch.randn(shape, device=_CARD, generator=g) * size).to(torch.bfloat16)
        return t.transpose(1, 2) if case["layout"] == "bshd" else t

    s = {"case": dict(case), "lengths": None, "offset": 0}
    # attention with a position bias is used without a scale: its queries are small instead
    s["q"], s["k"], s["v"] = tensor(Hq, Sq, D ** -0.5 if relative else 1.0), tensor(Hkv, Sk), tensor(Hkv, Sk)
    s["scale"] = 1.0 if relative else None
    if case["ragged"]:
        order = torch.randperm(B, device=_CARD, generator=g)
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=_CARD)[order].contiguous()
    if relative:
        s["bias"] = (torch.randn(case["buckets"], Hq, device=_CARD, generator=g) * 1.5).to(torch.bfloat16)
        if case["form"] in ("step", "chunk"):  # the new tokens are the last ones of each sequence
            s["offset"] = s["lengths"] - Sq if case["ragged"] else Sk - Sq
    if train:
        s["do"] = tensor(Hq, Sq)
        for n in ("q", "k", "v", "bias"):
            if n in s:
                s[n].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------
def _buckets(relative, case):
    """The bucket of each relative position (key's minus query's), from the definition."""
    n, first = case["buckets"], 0
    if not case["causal"]:  # both directions: half of the buckets for each
        n //= 2
        first = (relative > 0).long() * n
        distance = relative.abs()
    else:
        distance = (-relative).clamp(min=0)
    exact_ones = n // 2
    # whole results of the logarithms' quotient stay on their side of the border
    far = torch.log(distance.double().clamp(min=1) / exact_ones) / math.log(case["distance"] / exact_ones)
    far = exact_ones + torch.floor(far * (n - exact_ones) + 1e-9).long()
    return first + torch.where(distance < exact_ones, distance, far.clamp(max=n - 1))


def _plain(s):
    case = s["case"]
    B, Hq, Hkv, Sq, Sk, D = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    G, train, relative = Hq // Hkv, case["form"] == "train", case["op"] == "relative"
    scale = s["scale"] if s["scale"] is not None else D ** -0.5
    q = s["q"].detach().float().reshape(B, Hkv, G * Sq, D)
    k, v = s["k"].detach().float(), s["v"].detach().float()
    scores = (q @ k.transpose(-1, -2)).view(B, Hq, Sq, Sk) * scale
    keys = torch.arange(Sk, device=_CARD)
    visible = None
    if s["lengths"] is not None:
        visible = (keys < s["lengths"][:, None]).view(B, 1, 1, Sk)
    if relative:
        start = s["offset"].view(-1, 1, 1) if torch.is_tensor(s["offset"]) else s["offset"]
        position = torch.arange(Sq, device=_CARD).view(1, Sq, 1) + start
        apart = keys.view(1, 1, Sk) - position  # [1 or B, Sq, Sk]
        bucket = _buckets(apart, case)
        scores = scores + s["bias"].detach().float()[bucket].permute(0, 3, 1, 2)
        if case["causal"]:
            seen = (apart <= 0)[:, None]
            visible = seen if visible is None else visible & seen
    if visible is not None:
        scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    o = (p.view(B, Hkv, G * Sq, Sk) @ v).view(B, Hq, Sq, D).to(torch.bfloat16)
    if not train:
        return [o]
    do = s["do"].float().reshape(B, Hkv, G * Sq, D)
    rows = p.view(B, Hkv, G * Sq, Sk)
    dv = rows.transpose(-1, -2) @ do
    dp = (do @ v.transpose(-1, -2))
    ds = rows * (dp - (dp * rows).sum(-1, keepdim=True))
    dq = ((ds @ k) * scale).view(B, Hq, Sq, D)
    dk = (ds.transpose(-1, -2) @ q) * scale
    grads = [dq.to(torch.bfloat16), dk.to(torch.bfloat16), dv.to(torch.bfloat16)]
    if relative:
        # each diagonal's sum: with the rows upside down and padded, rows read one element
        # shorter put a diagonal's entries under one another
        wide = torch.nn.functional.pad(ds.view(B, Hq, Sq, Sk).sum(0).flip(1), (0, Sq)).view(Hq, -1)
        diagonals = wide[:, :Sq * (Sq + Sk - 1)].view(Hq, Sq, Sq + Sk - 1).sum(1)
        apart = torch.arange(Sq + Sk - 1, device=_CARD) - (Sq - 1)
        table = torch.zeros(Hq, case["buckets"], device=_CARD)
        table.index_add_(1, _buckets(apart, case), diagonals)
        grads.append(table.t().contiguous().to(torch.bfloat16))
    return [o] + grads


def _own(s):
    import fastflashattention_b200 as ffa
    case = s["case"]
    shared = case["Hq"] != case["Hkv"]
    leaves = [s["q"], s["k"], s["v"]]
    if case["op"] == "cross":
        o = ffa.cross_attention(*leaves, key_lengths=s["lengths"], scale=s["scale"], enable_gqa=shared)
    else:
        o = ffa.relative_attention(*leaves, s["bias"], max_distance=case["distance"], is_causal=case["causal"],
                                   query_offset=s["offset"], key_lengths=s["lengths"], scale=s["scale"],
                                   enable_gqa=shared)
        leaves.append(s["bias"])
    if case["form"] != "train":
        return [o]
    return [o.detach(), *torch.autograd.grad(o, leaves, s["do"])]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------
def _bucket_table(n, distance, reach):
    """The bucket of each distance 0..reach on one side, in whole numbers: bucket m + j starts at
    the least r with (r / m) ** (n - m) >= (distance / m) ** j."""
    m, out, b = n // 2, [], 0
    for r in range(reach + 1):
        if r < m:
            b = r
        else:
            b = max(b, m)
            while b < n - 1 and r ** (n - m) * m ** (b + 1 - m) >= distance ** (b + 1 - m) * m ** (n - m):
                b += 1
        out.append(b)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    B, Hq, Hkv, Sq, Sk, D = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    G, train, relative = Hq // Hkv, case["form"] == "train", case["op"] == "relative"
    scale = s["scale"] if s["scale"] is not None else 1.0 / math.sqrt(D)
    lengths = s["lengths"].tolist() if case["ragged"] else [Sk] * B
    if relative:
        both = not case["causal"]
        sides = case["buckets"] // 2 if both else case["buckets"]
        reach = case["distance"]
        side = torch.tensor(_bucket_table(sides, case["distance"], reach), device=_CARD)
        starts = s["offset"].tolist() if torch.is_tensor(s["offset"]) else [s["offset"]] * B
    o = torch.zeros(B, Hq, Sq, D, dtype=torch.float64, device=_CARD)
    grads = [torch.zeros_like(s[n], dtype=torch.float64) for n in ("q", "k", "v")] if train else []
    dbias = torch.zeros(case["buckets"], Hq, dtype=torch.float64, device=_CARD) if train and relative else None
    step = max(1, int(2 ** 28 // (G * Sk)))  # queries at a time
    for b in range(B):
        n = lengths[b]
        if relative:
            j = torch.arange(n, device=_CARD)
        for h in range(Hkv):
            heads = slice(h * G, (h + 1) * G)
            k, v = s["k"][b, h, :n].detach().double(), s["v"][b, h, :n].detach().double()
            for i0 in range(0, Sq, step):
                rows = slice(i0, min(Sq, i0 + step))
                q = s["q"][b, heads, rows].detach().double()
                x = torch.einsum("gid,jd->gij", q, k) * scale
                if relative:
                    r = j[None, :] - (torch.arange(rows.start, rows.stop, device=_CARD)[:, None] + starts[b])
                    bucket = side[(r.abs() if both else (-r).clamp(min=0)).clamp(max=reach)]
                    if both:
                        bucket = bucket + sides * (r > 0)
                    x = x + s["bias"].detach().double()[bucket][..., heads].permute(2, 0, 1)
                    if case["causal"]:
                        x = x.masked_fill((r > 0)[None], -math.inf)
                p = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
                del x
                o[b, heads, rows] = torch.einsum("gij,jd->gid", p, v)
                if train:
                    do = s["do"][b, heads, rows].double()
                    inner = (do * o[b, heads, rows]).sum(-1, keepdim=True)
                    ds = p * (torch.einsum("gid,jd->gij", do, v) - inner)
                    grads[0][b, heads, rows] = torch.einsum("gij,jd->gid", ds, k) * scale
                    grads[1][b, h, :n] += torch.einsum("gij,gid->jd", ds, q) * scale
                    grads[2][b, h, :n] += torch.einsum("gij,gid->jd", p, do)
                    if relative:
                        place = bucket.reshape(1, -1).expand(G, -1)
                        dbias[:, heads] += torch.zeros(G, case["buckets"], dtype=torch.float64, device=_CARD).scatter_add_(
                            1, place, ds.reshape(G, -1)).t()
    return [o] + grads + ([dbias] if dbias is not None else [])


# ------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------
def work(case):
    B, Hq, Hkv, Sq, Sk, D = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    lengths = _lengths(case) if case["ragged"] else [Sk] * B
    pairs = keys = 0
    for n in lengths:
        if case.get("causal"):
            first = {"step": n - Sq, "chunk": n - Sq}.get(case["form"], 0)  # position of the first query
            whole = max(0, min(Sq, n - first))  # queries before the last key
            pairs += whole * (first + 1) + whole * (whole - 1) // 2 + (Sq - whole) * n
        else:
            pairs += Sq * n
        keys += n
    queries, states = B * Hq * Sq * D * 2, Hkv * keys * D * 2
    table = case.get("buckets", 0) * Hq * 2
    flops = 4 * pairs * Hq * D
    if case["form"] == "train":  # q, dO, O and dQ; k, v, dK and dV; the table and its gradient; 3.5 times the products
        return {"bytes": 4 * queries + 2 * states + 2 * B * Hkv * Sk * D * 2 + 2 * table, "flops": 3.5 * flops}
    return {"bytes": 2 * queries + 2 * states + table, "flops": flops}
