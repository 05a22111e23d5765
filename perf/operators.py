"""The paged key-value cache operators, as cases that can be timed and compared.

A serving program keeps keys and values in a pool of pages.  Each step appends
the new tokens' rows (`paged_append`, `paged_append_rope`), attends from one new
token per sequence over what the sequence has cached (`paged_attention`, which
can also add up the attention weight each cached token received) and, where the
cache outgrows its budget, keeps the tokens with the most weight
(`paged_evict`).

Shapes (torch, row-major): pools (P, KH, PS, E); block table (B, MP) int32, the
page of each run of PS slots, outside [0, P) for no page; lengths (B,) int32;
q (B, QH, 1, E); new k, v (B, KH, T, E); weights (B, KH, MP·PS) float32.

`run` computes an operator from elementary torch operations, or, where `own` is
true, calls the package.
"""
import math
import pathlib
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def _nnop():
    if "nnop" in sys.modules:
        return sys.modules["nnop"]
    root = str(pathlib.Path(__file__).resolve().parent.parent / "onionop.jl_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import nnop
    return nnop


# --------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of a batch: the rows of 64 new tokens, rotated and stored
        dict(name="append one token", op="append", dtype="bf16", B=64, QH=32, KH=8, E=128, T=1, PS=16,
             longest=8192, shortest=1, rope=True),
        # a batch of prompts padded to one length, rotated and stored
        dict(name="append prompts", op="append", dtype="bf16", B=4, QH=32, KH=8, E=128, T=8192, PS=16,
             longest=0, shortest=0, rope=True),
        # a chunk of a prompt without rotation, full precision, odd pages
        dict(name="append chunk f32", op="append", dtype="f32", B=8, QH=16, KH=16, E=64, T=511, PS=24,
             longest=1001, shortest=0, rope=False),
        # one user, a short conversation: latency
        dict(name="attend short", op="attend", dtype="bf16", B=1, QH=32, KH=8, E=128, PS=16,
             longest=77, shortest=77, weigh=False),
        # a serving batch of mixed lengths
        dict(name="attend batch", op="attend", dtype="bf16", B=64, QH=32, KH=8, E=128, PS=16,
             longest=8192, shortest=1, weigh=False),
        # one user, a very long document
        dict(name="attend long", op="attend", dtype="f16", B=1, QH=32, KH=8, E=128, PS=64,
             longest=131067, shortest=131067, weigh=False),
        # every query head with its own keys, narrow heads, odd pages
        dict(name="attend all heads", op="attend", dtype="f16", B=8, QH=16, KH=16, E=64, PS=20,
             longest=4096, shortest=513, weigh=False),
        # full precision
        dict(name="attend f32", op="attend", dtype="f32", B=2, QH=8, KH=4, E=64, PS=16,
             longest=2047, shortest=512, weigh=False),
        # a serving batch that also keeps each token's accumulated weight
        dict(name="attend and weigh", op="attend", dtype="bf16", B=16, QH=32, KH=8, E=128, PS=32,
             longest=8192, shortest=100, weigh=True),
        # a small cache cut to a quarter
        dict(name="evict small", op="evict", dtype="f16", B=2, KH=4, E=64, PS=16, longest=512, shortest=100,
             budget=128, recent=32),
        # a serving batch cut to a quarter of its longest
        dict(name="evict batch", op="evict", dtype="bf16", B=16, KH=8, E=128, PS=16, longest=8192, shortest=1500,
             budget=2048, recent=256),
        # one very long document
        dict(name="evict long", op="evict", dtype="bf16", B=1, KH=8, E=128, PS=64, longest=131067, shortest=131067,
             budget=8192, recent=1024),
    ]


def _near(rng, low, high):
    """A whole number spread over the logarithm of low..high."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    E = rng.choice([16, 32, 64, 128, 128])
    KH = rng.choice([1, 2, 3, 4, 8, 16])
    PS = rng.choice([8, 16, 16, 20, 32, 64, 128])
    case = dict(op=op, dtype=dtype, E=E, KH=KH, PS=PS)
    row = KH * E * _SIZE[dtype] * 2                       # bytes of one cached token
    if op == "append":
        group = rng.choice([1, 2, 4, 7, 8])
        B = _near(rng, 1, 64)
        most = min(8192, 300_000_000 // (row * B * (1 + group)))
        T = 1 if rng.random() < 0.4 else _near(rng, 2, max(2, most))
        longest = _near(rng, 1, 4096)
        case |= dict(B=B, QH=KH * group, T=T, longest=longest, shortest=rng.randint(0, longest),
                     rope=rng.random() < 0.6)
    elif op == "attend":
        group = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 24])
        B = _near(rng, 1, 128)
        longest = _near(rng, 1, max(1, min(131072, 400_000_000 // (row * B))))
        case |= dict(B=B, QH=KH * group, longest=longest, shortest=rng.randint(0, longest),
                     weigh=rng.random() < 0.4)
    else:
        B = _near(rng, 1, 32)
        longest = _near(rng, 2, max(2, min(131072, 400_000_000 // (row * B))))
        budget = _near(rng, 1, max(1, longest))
        case |= dict(B=B, longest=longest, shortest=rng.randint(0, longest), budget=budget,
                     recent=rng.randint(0, budget))
    return case


def _lengths(case):
    """The sequences' lengths, from the longest to the shortest in even steps."""
    B, hi, lo = case["B"], case["longest"], case["shortest"]
    return [hi - (hi - lo) * b // max(1, B - 1) for b in range(B)]


def _new(case):
    """How many of the T padded new rows of each sequence are tokens."""
    B, T = case["B"], case["T"]
    return [T - (T // 2) * b // B for b in range(B)]


# -------------------------------------------------------------------- inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    B, KH, E, PS = case["B"], case["KH"], case["E"], case["PS"]

    def randn(*shape, dtype=dtype):
        return torch.randn(*shape, device=dev, dtype=dtype, generator=g)

    order = torch.randperm(B, device=dev, generator=g)
    lengths = torch.tensor(_lengths(case), device=dev, dtype=torch.int32)[order].contiguous()
    slots = case["longest"] + case.get("T", 0)
    MP = -(-slots // PS) + 1
    DP = -(-case["budget"] // PS) if case["op"] == "evict" else 0
    P = B * (MP + DP)
    pages = torch.randperm(P, device=dev, generator=g).to(torch.int32)
    s = dict(case=case, lengths=lengths, table=pages[:B * MP].view(B, MP).contiguous(),
             k_cache=randn(P, KH, PS, E), v_cache=randn(P, KH, PS, E))
    if case["op"] == "append":
        T, QH = case["T"], case["QH"]
        s["k"], s["v"] = randn(B, KH, T, E), randn(B, KH, T, E)
        s["n_new"] = torch.tensor(_new(case), device=dev, dtype=torch.int32)[order].contiguous()
        if case["rope"]:
            s["q"] = randn(B, QH, T, E)
            freq = 10000.0 ** (-torch.arange(0, E, 2, device=dev, dtype=torch.float64) / E)
            at = lengths[:, None].double() + torch.arange(T, device=dev, dtype=torch.float64)
            angle = at[..., None] * torch.cat([freq, freq])
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    elif case["op"] == "attend":
        # a few times the unit scale, so that some keys get most of the weight
        s["q"] = 2 * randn(B, case["QH"], 1, E)
        if case["weigh"]:
            s["weights"] = torch.rand(B, KH, MP * PS, device=dev, generator=g)
    else:
        s["new_table"] = pages[B * MP:].view(B, DP).contiguous()
        # accumulated weights: most small, few large, some tokens never looked at
        w = torch.exp(2 * randn(B, KH, MP * PS, dtype=torch.float32))
        s["weights"] = torch.where(torch.rand(w.shape, device=dev, generator=g) < 0.1, torch.zeros_like(w), w)
    return s


# ----------------------------------------------------------------- operators

def run(state):
    op = state["case"]["op"]
    if op == "append":
        return _append(state)
    return _attend(state) if op == "attend" else _evict(state)


def _rotate(x, cos, sin):
    """Each pair (i, i + E/2) of x by the angle of index i, in 32 bits."""
    half = x.shape[-1] // 2
    a, b = x[..., :half].float(), x[..., half:].float()
    c, s = cos[:, None, :, :half], sin[:, None, :, :half]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(x.dtype)


def _append(st):
    rope = st["case"]["rope"]
    if own:
        nnop = _nnop()
        args = st["k_cache"], st["v_cache"], st["table"], st["lengths"]
        if rope:
            q, lengths = nnop.paged_append_rope(st["q"], st["k"], st["v"], *args, cos=st["cos"], sin=st["sin"],
                                                n_new=st["n_new"])
            return dict(q=q, lengths=lengths, k_cache=st["k_cache"], v_cache=st["v_cache"])
        lengths = nnop.paged_append(st["k"], st["v"], *args, n_new=st["n_new"])
        return dict(lengths=lengths, k_cache=st["k_cache"], v_cache=st["v_cache"])
    k, v, table = st["k"], st["v"], st["table"]
    B, KH, T, E = k.shape
    PS = st["k_cache"].shape[2]
    out = {}
    if rope:
        out["q"] = _rotate(st["q"], st["cos"], st["sin"])
        k = _rotate(k, st["cos"], st["sin"])
    t = torch.arange(T, device=k.device)
    b, t = torch.nonzero(t < st["n_new"][:, None], as_tuple=True)
    slot = st["lengths"].long()[b] + t
    page = table.long()[b, slot // PS]
    st["k_cache"][page, :, slot % PS] = k[b, :, t]
    st["v_cache"][page, :, slot % PS] = v[b, :, t]
    return dict(out, lengths=st["lengths"] + st["n_new"], k_cache=st["k_cache"], v_cache=st["v_cache"])


def _gather(pool, table):
    """The pages of each sequence one after the other: (B, KH, MP·PS, E) in 32 bits."""
    x = pool[table.long()].float()                         # (B, MP, KH, PS, E)
    B, MP, KH, PS, E = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, KH, MP * PS, E)


def _attend(st):
    q, table, lengths = st["q"], st["table"], st["lengths"]
    weights = st.get("weights")
    if own:
        o, lse = _nnop()._paged_attention(q, st["k_cache"], st["v_cache"], table, lengths, weights=weights)
        return dict(o=o, lse=lse) if weights is None else dict(o=o, lse=lse, weights=weights)
    B, QH, _, E = q.shape
    KH = st["k_cache"].shape[1]
    k, v = _gather(st["k_cache"], table), _gather(st["v_cache"], table)
    live = (torch.arange(k.shape[2], device=q.device) < lengths[:, None])[:, None, :, None]
    k, v = torch.where(live, k, 0.0), torch.where(live, v, 0.0)
    scale = torch.tensor(1.0 / math.sqrt(E)).to(q.dtype).float().item()   # flash_attention's scale
    s = torch.matmul(q.view(B, KH, QH // KH, E).float(), k.transpose(2, 3)) * scale
    s = s.masked_fill(~live.transpose(2, 3), -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)                # a sequence without tokens
    p = torch.exp(s - m)
    l = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(l == 0, 1.0, l)
    o = torch.matmul(p, v).to(q.dtype).view(B, QH, 1, E)
    lse = (m + torch.log(l)).view(B, QH, 1)
    if weights is None:
        return dict(o=o, lse=lse)
    weights += p.sum(dim=2)
    return dict(o=o, lse=lse, weights=weights)


def _evict(st):
    case, weights, lengths = st["case"], st["weights"], st["lengths"]
    budget, recent = case["budget"], case["recent"]
    if own:
        lengths, weights, kept = _nnop().paged_evict(st["k_cache"], st["v_cache"], st["table"], st["new_table"],
                                                     lengths, weights, budget=budget, recent=recent)
        return dict(lengths=lengths, weights=weights, kept=kept, k_cache=st["k_cache"], v_cache=st["v_cache"])
    B, KH, S = weights.shape
    PS, DP = st["k_cache"].shape[2], st["new_table"].shape[1]
    n = lengths[:, None, None]
    at = torch.arange(S, device=weights.device)
    # the last `recent` tokens first, then the others by weight, the lower slot first among equals
    w = torch.where(at < n, torch.where(at >= n - recent, math.inf, weights), -math.inf)
    best = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :budget]
    fewer = torch.clamp(n, max=budget)
    there = torch.arange(best.shape[-1], device=at.device) < fewer
    kept = torch.sort(torch.where(there, best, S), dim=-1).values
    there = kept < S
    kept = torch.nn.functional.pad(torch.where(there, kept, -1), (0, budget - kept.shape[-1]), value=-1)
    there = kept >= 0
    b, h, i = torch.nonzero(there, as_tuple=True)
    j = kept[b, h, i]
    new_weights = torch.zeros(B, KH, DP * PS, device=at.device)
    new_weights[b, h, i] = weights[b, h, j]
    src, dst = st["table"].long()[b, j // PS], st["new_table"].long()[b, i // PS]
    for pool in (st["k_cache"], st["v_cache"]):
        pool[dst, h, i % PS] = pool[src, h, j % PS]
    return dict(lengths=torch.clamp(lengths, max=budget), weights=new_weights, kept=kept.to(torch.int32),
                k_cache=st["k_cache"], v_cache=st["v_cache"])


# ------------------------------------------------------------ what it has to do

def work(case):
    B, KH, E, PS = case["B"], case["KH"], case["E"], case["PS"]
    size, lens = _SIZE[case["dtype"]], _lengths(case)
    if case["op"] == "append":
        T, rows = case["T"], sum(_new(case))
        nbytes = 2 * 2 * rows * KH * E * size + 4 * (rows + 3 * B)
        flops = 0
        if case["rope"]:
            # both halves of a position's angles are alike: one is needed
            nbytes += 2 * B * T * case["QH"] * E * size + 2 * 4 * B * T * (E // 2)
            flops = 3 * (B * T * case["QH"] + rows * KH) * E
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "attend":
        QH, rows = case["QH"], sum(lens)
        nbytes = 2 * rows * KH * E * size + 2 * B * QH * E * size + 4 * B * QH + 4 * (B + sum(-(-n // PS) for n in lens))
        nbytes += 8 * rows * KH if case["weigh"] else 0
        return {"bytes": nbytes, "flops": 4 * rows * QH * E}
    kept = sum(min(n, case["budget"]) for n in lens)
    DP = -(-case["budget"] // PS)
    return {"bytes": 2 * 2 * kept * KH * E * size + 4 * KH * sum(lens) + 4 * B * KH * (DP * PS + case["budget"]) + 8 * B,
            "flops": 0}


# ------------------------------------------------------------ the definition, in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    n = st["lengths"].tolist()
    table = st["table"].cpu()
    PS, B, KH, E = case["PS"], case["B"], case["KH"], case["E"]
    dev = st["k_cache"].device

    def places(b, slots, tab):
        """Pages and rows of the slots of sequence b."""
        slots = torch.as_tensor(slots, dtype=torch.int64)
        return tab[b].long()[slots // PS].to(dev), (slots % PS).to(dev)

    if case["op"] == "append":
        new = st["n_new"].tolist()
        k, v = st["k"].double(), st["v"].double()
        out = {}
        if case["rope"]:
            half = E // 2
            turn = torch.complex(st["cos"][..., :half].double(), st["sin"][..., :half].double())[:, None]

            def rotate(x):
                z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
                return torch.cat([z.real, z.imag], -1)
            out["q"], k = rotate(st["q"].double()), rotate(k)
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        for b in range(B):
            page, row = places(b, range(n[b], n[b] + new[b]), table)
            kc[page, :, row] = k[b, :, :new[b]].transpose(0, 1)
            vc[page, :, row] = v[b, :, :new[b]].transpose(0, 1)
        lengths = torch.tensor([a + c for a, c in zip(n, new)], dtype=torch.int32, device=dev)
        return dict(out, lengths=lengths, k_cache=kc, v_cache=vc)
    if case["op"] == "attend":
        QH = case["QH"]
        scale = torch.tensor(1.0 / math.sqrt(E)).to(st["q"].dtype).double().item()
        o = torch.zeros(B, KH, QH // KH, E, dtype=torch.float64, device=dev)
        lse = torch.full((B, KH, QH // KH), -math.inf, dtype=torch.float64, device=dev)
        weights = st["weights"].double() if case["weigh"] else None
        q = st["q"].double().view(B, KH, QH // KH, E)
        for b in range(B):
            if n[b] == 0:
                continue
            page, row = places(b, range(n[b]), table)
            k, v = st["k_cache"][page, :, row].double(), st["v_cache"][page, :, row].double()    # (n, KH, E)
            s = torch.einsum("hge,nhe->hgn", q[b], k) * scale
            lse[b] = torch.logsumexp(s, -1)
            p = torch.softmax(s, -1)
            o[b] = torch.einsum("hgn,nhe->hge", p, v)
            if weights is not None:
                weights[b, :, :n[b]] += p.sum(1)
        out = dict(o=o.view(B, QH, 1, E), lse=lse.view(B, QH, 1))
        return out if weights is None else dict(out, weights=weights)
    budget, recent = case["budget"], case["recent"]
    new_table = st["new_table"].cpu()
    weights = torch.zeros(B, KH, new_table.shape[1] * PS, dtype=torch.float64, device=dev)
    kept = torch.full((B, KH, budget), -1, dtype=torch.int32, device=dev)
    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    for b in range(B):
        last = min(recent, budget, n[b])
        old = n[b] - last
        count = min(n[b], budget)
        for h in range(KH):
            w = st["weights"][b, h, :n[b]].double()
            # by falling weight, then by rising slot
            order = sorted(range(old), key=lambda i, w=w[:old].tolist(): (-w[i], i))[:count - last]
            keep = torch.tensor(sorted(order) + list(range(old, n[b])), dtype=torch.int64)
            kept[b, h, :count] = keep.to(dev)
            weights[b, h, :count] = w[keep.to(dev)]
            (src, row), (dst, to) = places(b, keep, table), places(b, range(count), new_table)
            kc[dst, h, to] = st["k_cache"][src, h, row].double()
            vc[dst, h, to] = st["v_cache"][src, h, row].double()
    return dict(lengths=torch.clamp(st["lengths"], max=budget), weights=weights, kept=kept, k_cache=kc, v_cache=vc)
