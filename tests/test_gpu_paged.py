"""GPU parity of the paged key-value cache (paged_append, paged_append_rope,
paged_attention, paged_evict) against the float64 oracle.

Every slot that a call has no business reading (behind the lengths, in pages of no
table) holds NaN or Inf, so a stray read shows.  Tolerances are element by element
and follow from the arithmetic (u = 2^-24, the half step of fp32): a dot product
over E terms of sum |q_e k_e| <= S is off by at most (2E + 16)·u·S (the tensor cores
may truncate: two half steps a term), exp adds 2^-22 relative, a sum over n slots in
runs of 16 adds (80 + n/16)·u of the sum of magnitudes, the 16-bit kernels split a
probability into two 16-bit terms (2^-16), and the result is rounded once
(finfo.eps/2)."""
import math

import numpy as np
import pytest

from _util import to_dev, to_np, torch_dtype
from oracle import nnop_oracle as orc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


class Cache:
    """Pools with `spare` pages of no table, a table in random order, poison outside
    the lengths; the same as float64 / int numpy arrays."""

    def __init__(self, seed, dtype, KH, E, PS, lengths, *, MP=None, spare=3, bad=None, clean=False):
        import torch
        rng = self.rng = np.random.default_rng(seed)
        B = len(lengths)
        MP = max(1, -(-max(lengths) // PS)) + 1 if MP is None else MP
        P = B * MP + spare
        self.table = rng.permutation(P)[:B * MP].reshape(B, MP).astype(np.int32)
        pools = rng.standard_normal((2, P, KH, PS, E)).astype(np.float32)
        if not clean:
            live = np.zeros((P, PS), bool)
            for b, n in enumerate(lengths):
                j = np.arange(min(max(n, 0), MP * PS))
                live[self.table[b, j // PS], j % PS] = True
            at = np.nonzero(~live)
            pools[0][at[0], :, at[1]] = np.nan
            pools[1][at[0], :, at[1]] = rng.choice([np.nan, np.inf, -np.inf], (len(at[0]), 1, 1))
        if bad is not None:
            bad(self.table, P)
        self.dtype, self.P, self.KH, self.PS, self.E, self.B, self.MP = dtype, P, KH, PS, E, B, MP
        self.k, self.v = to_dev(pools[0], dtype), to_dev(pools[1], dtype)
        self.t = torch.from_numpy(self.table).cuda()
        self.lengths = np.asarray(lengths, np.int32)
        self.n = torch.from_numpy(self.lengths).cuda()

    @property
    def args(self):
        return self.k, self.v, self.t, self.n

    def np(self):
        return to_np(self.k), to_np(self.v), self.table, self.lengths


def attention_oracle(q, kc, vc, table, lengths, dtype):
    """(o, lse, w) and how far off each element may be."""
    B, QH, _, E = q.shape
    P, KH, PS, _ = kc.shape
    G = QH // KH
    scale = orc.attention_scale(E, dtype)
    o, lse, w = orc.paged_attention(q, kc, vc, table, lengths, scale=scale)
    tol_o, tol_l, tol_w = np.zeros_like(o), np.zeros_like(lse), np.zeros_like(w)
    half = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    for b in range(B):
        n = orc.paged_length(lengths, b, table, PS)
        slots = np.arange(n)
        page, row = orc.paged_places(table, b, slots, P, PS)
        slots, page, row = (x[page >= 0] for x in (slots, page, row))
        if not slots.size:
            continue
        k, v = (c[page, :, row] for c in (kc, vc))
        qb = q[b].reshape(KH, G, E)
        S = np.einsum("hge,nhe->hgn", np.abs(qb), np.abs(k)).max(-1) * scale             # (KH, G)
        p = np.exp(np.einsum("hge,nhe->hgn", qb, k) * scale - lse[b].reshape(KH, G, 1))
        mag = np.einsum("hgn,nhe->hge", p, np.abs(v))
        rel_p = (2 * E + 16) * U * S + 2.0 ** -22
        run = (80 + n / 16) * U
        split = 0 if dtype == "f32" else 2.0 ** -16
        tol_o[b] = (mag * (2 * rel_p + 2 * run + split)[..., None]).reshape(QH, 1, E) + half * np.abs(o[b])
        tol_l[b] = (rel_p + run).reshape(QH, 1) + 4 * U * np.abs(lse[b])
        tol_w[b][:, slots] = (p * (2 * rel_p + run + 16 * U)[..., None]).sum(1)
    return (o, lse, w), (tol_o + 1e-30, tol_l, tol_w + 1e-30)


def near(got, want, tol, what):
    got = to_np(got)
    fine = np.isfinite(want)
    same = np.array_equal(np.isfinite(got), fine) and np.array_equal(got[~fine], want[~fine])
    assert same, f"{what}: values that are not finite, at others' places"
    over = np.abs(got - np.where(fine, want, 0))[fine] - np.broadcast_to(tol, want.shape)[fine]
    assert not over.size or over.max() <= 0, f"{what}: {over.max():.3g} over its tolerance"


def check_attention(c, QH, *, weigh=False, scale_q=1.0):
    import torch

    import nnop
    q = to_dev(scale_q * c.rng.standard_normal((c.B, QH, 1, c.E)), c.dtype)
    w = torch.from_numpy(c.rng.random((c.B, c.KH, c.MP * c.PS)).astype(np.float32)).cuda() if weigh else None
    w0 = None if w is None else to_np(w)
    o, lse = nnop._paged_attention(q, *c.args, weights=w)
    torch.cuda.synchronize()
    (o_o, lse_o, w_o), (tol_o, tol_l, tol_w) = attention_oracle(to_np(q), *c.np(), c.dtype)
    near(o, o_o, tol_o, "o")
    near(lse, lse_o, tol_l, "lse")
    if weigh:
        near(w, w0 + w_o, tol_w + U * np.abs(w0 + w_o), "weights")
        assert np.array_equal(to_np(w)[w_o == 0], w0[w_o == 0])
    return q, o, lse


LENGTHS = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("E", [16, 32, 64, 128])
@pytest.mark.parametrize("QH,KH", [(1, 1), (4, 2), (6, 2), (8, 1), (10, 1), (48, 2)])
def test_attention_small(dtype, E, QH, KH):
    check_attention(Cache(E + QH, dtype, KH, E, 16, LENGTHS), QH, weigh=QH > 4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("PS", [1, 3, 8, 20, 64, 333])
def test_attention_page_sizes(dtype, PS):
    check_attention(Cache(PS, dtype, 2, 64, PS, [0, 1, 332, 333, 334, 700]), 6, weigh=True)


@pytest.mark.parametrize("dtype,E,QH,KH", [("f32", 128, 8, 2), ("bf16", 128, 32, 8), ("f16", 64, 3, 3), ("f16", 128, 128, 1),
                                           ("bf16", 32, 5, 1)])
@pytest.mark.parametrize("lengths", [[20011], [5000, 0, 0, 12345, 3], [1] * 300 + [4000]])
def test_attention_split_over_ctas(dtype, E, QH, KH, lengths):
    check_attention(Cache(len(lengths), dtype, KH, E, 16, lengths), QH, weigh=True, scale_q=3.0)


def _holes(table, P):
    table[0, :] = -1
    table[1, 1::2] = [-1, P, 2**31 - 1, -2**31][:table[1, 1::2].size]
    table[2, -1] = P + 5


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_skips_slots_without_a_page(dtype):
    check_attention(Cache(5, dtype, 2, 64, 8, [64, 62, 64, 10], MP=8, bad=_holes), 4, weigh=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_lengths_outside_the_table(dtype):
    import torch
    c = Cache(6, dtype, 1, 32, 16, [48, 48, 48], MP=3)
    c.lengths = np.array([49, 2**31 - 1, -5], np.int32)
    c.n = torch.from_numpy(c.lengths).cuda()
    check_attention(c, 2, weigh=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attention_peaks_and_far_scores(dtype):
    """One key far above the others, then all scores far below zero, late in the cache."""
    c = Cache(8, dtype, 1, 64, 16, [1500, 1500])
    for b in range(2):
        at = [777, 1490][b]
        c.k[c.table[b, at // 16], 0, at % 16] = 6.0
    import torch

    import nnop
    q = torch.full((2, 4, 1, 64), 2.0, device="cuda", dtype=torch_dtype(dtype))
    q[:, 2:] = -2.0
    o, lse = nnop._paged_attention(q, *c.args)
    (o_o, lse_o, _), (tol_o, tol_l, _) = attention_oracle(to_np(q), *c.np(), dtype)
    near(o, o_o, tol_o, "o")
    near(lse, lse_o, tol_l, "lse")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_infinite_scores(dtype):
    """A row whose every score is -Inf counts as empty; one +Inf or NaN score makes
    the row NaN, as it does in a softmax; other rows keep their values."""
    import torch

    import nnop
    c = Cache(9, dtype, 1, 16, 16, [70, 70, 70], clean=True)
    c.k[:] = 1.0
    q = torch.ones(3, 2, 1, 16, device="cuda", dtype=torch_dtype(dtype))
    q[0, 0] = -math.inf
    c.k[int(c.table[1, 2]), 0, 3, 5] = math.nan
    c.k[int(c.table[2, 0]), 0, 0, 0] = math.inf
    w = torch.zeros(3, 1, c.MP * c.PS, device="cuda")
    o, lse = nnop._paged_attention(q, *c.args, weights=w)
    assert not o[0, 0].any() and lse[0, 0] == -math.inf
    assert torch.isfinite(o[0, 1]).all() and torch.isnan(o[1]).all() and torch.isnan(o[2]).all()
    assert torch.allclose(w[0, 0, :70], torch.full((70,), 1 / 70, device="cuda"), rtol=1e-5) and not w[0, 0, 70:].any()


@pytest.mark.parametrize("layout", ["interleaved", "rows first", "wide"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(dtype, layout):
    """Both pools in one tensor, slots before heads, or rows with a gap."""
    import torch

    import nnop
    c = Cache(10, dtype, 3, 32, 10, [25, 40, 0, 7])
    flat = c.k.clone(), c.v.clone()
    if layout == "interleaved":
        both = torch.stack([c.k, c.v], 1)
        c.k, c.v = both[:, 0], both[:, 1]
    elif layout == "rows first":
        c.k, c.v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (c.k, c.v))
    else:
        c.k, c.v = (torch.cat([x, torch.full_like(x, math.nan)], -1)[..., :32] for x in (c.k, c.v))
    assert not c.k.is_contiguous()
    q, o, lse = check_attention(c, 6, weigh=True)
    again = nnop._paged_attention(q, *flat, c.t, c.n)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
    k, v = (to_dev(c.rng.standard_normal((4, 3, 5, 32)), dtype) for _ in range(2))
    n1 = nnop.paged_append(k, v, *c.args)
    n2 = nnop.paged_append(k, v, *flat, c.t, c.n)
    assert torch.equal(n1, n2)
    for a, b in zip((c.k, c.v), flat):
        assert torch.equal(a.contiguous().view(torch.uint8), b.view(torch.uint8))
    new_table = torch.tensor([[p] for p in sorted(set(range(c.P)) - set(c.table.ravel().tolist()))[:3] + [-1]],
                             dtype=torch.int32, device="cuda")
    w = torch.rand(4, 3, c.MP * 10, device="cuda")
    r1 = nnop.paged_evict(*c.args[:3], new_table, n1, w, budget=9, recent=2)
    r2 = nnop.paged_evict(*flat, c.t, new_table, n1, w, budget=9, recent=2)
    assert all(torch.equal(a, b) for a, b in zip(r1, r2))
    for a, b in zip((c.k, c.v), flat):
        assert torch.equal(a.contiguous().view(torch.uint8), b.view(torch.uint8))


def test_unaligned_and_strided_inputs():
    """q, k, v may be views of any stride and start; the table and lengths too."""
    import torch

    import nnop
    c = Cache(11, "bf16", 2, 64, 16, [30, 41])
    raw = to_dev(c.rng.standard_normal(2 * 4 * 64 + 1), "bf16")
    q = raw[1:].view(2, 4, 1, 64)
    o, lse = nnop._paged_attention(q, *c.args)
    t = torch.stack([c.t, c.t], -1)[..., 0]
    n = torch.stack([c.n, c.n], -1)[..., 0]
    o2, lse2 = nnop._paged_attention(q.clone(), c.k, c.v, t, n)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    k = to_dev(c.rng.standard_normal((2, 2, 64, 3)), "bf16").transpose(2, 3)
    nnop.paged_append(k, k, c.k, c.v, t, n)
    page, row = int(c.table[0, 1]), 14
    assert torch.equal(c.k[page, :, row], k[0, :, 0])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_matches_flash_attention(dtype):
    """A contiguous cache is a pool of one page per sequence."""
    import torch

    import nnop
    rng = np.random.default_rng(12)
    B, QH, KH, L, E = 3, 8, 2, 500, 64
    q, k, v = (to_dev(rng.standard_normal(s), dtype) for s in ((B, QH, 1, E), (B, KH, L, E), (B, KH, L, E)))
    mask = torch.zeros(B, L, dtype=torch.bool, device="cuda")
    lengths = [500, 123, 1]
    for b, n in enumerate(lengths):
        mask[b, :n] = True
    table = torch.arange(B, device="cuda", dtype=torch.int32)[:, None]
    o, lse = nnop._paged_attention(q, k, v, table, torch.tensor(lengths, device="cuda", dtype=torch.int32))
    o2, lse2 = nnop._flash_attention(q, k, v, causal=False, kpad_mask=mask)
    rtol = 1e-5 if dtype == "f32" else 2 ** -6     # the older kernel rounds its probabilities to 16 bits: 2^-8 twice, and o
    assert (o.float() - o2.float()).norm() <= rtol * o2.float().norm()
    assert torch.allclose(lse, lse2, rtol=1e-5, atol=1e-5)


def test_attention_same_bits_again_and_on_another_stream():
    import torch

    import nnop
    c = Cache(13, "bf16", 4, 128, 16, [3000, 77, 0, 1200])
    q = to_dev(c.rng.standard_normal((4, 16, 1, 128)), "bf16")
    w = torch.zeros(4, 4, c.MP * 16, device="cuda")
    first = nnop._paged_attention(q, *c.args, weights=w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        w2 = torch.zeros_like(w)
        again = nnop._paged_attention(q, *c.args, weights=w2)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, again)) and torch.equal(w, w2)


def test_captured_step_follows_the_lengths():
    """A captured decode step (append, attend, weigh) replays with the lengths and
    tables that the device holds then, two graphs beside each other."""
    import torch

    import nnop
    c = Cache(14, "f16", 2, 64, 8, [20, 5, 0], clean=True)
    q, k, v = (to_dev(c.rng.standard_normal((3, h, 1, 64)), "f16") for h in (4, 2, 2))
    cos, sin = nnop.LlamaRotaryEmbedding(64)(torch.arange(3, device="cuda", dtype=torch.float32)[:, None])

    def step(kc, vc, w, n):
        qr, n2 = nnop.paged_append_rope(q, k, v, kc, vc, c.t, n, cos=cos, sin=sin)
        o, lse = nnop._paged_attention(qr, kc, vc, c.t, n2, weights=w)
        return o, lse, n2
    graphs = []
    for _ in range(2):
        own = [c.k.clone(), c.v.clone(), torch.zeros(3, 2, c.MP * 8, device="cuda"), c.n.clone()]
        step(*[x.clone() for x in own])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*own)
            own[3].copy_(out[2])
        graphs.append((g, own, out))
    eager = [c.k.clone(), c.v.clone(), torch.zeros(3, 2, c.MP * 8, device="cuda"), c.n.clone()]
    for _ in range(4):
        want = step(*eager)
        eager[3].copy_(want[2])
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, (g, _, _) in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for _, own, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            assert all(torch.equal(a, b) for a, b in zip(own, eager))


def test_offsets_past_32_bits():
    """Pages whose elements lie past 2^31 and 2^32."""
    import torch

    import nnop
    KH, PS, E = 8, 16, 128
    per = KH * PS * E
    P = 2**32 // per + 40
    k, v = (torch.empty(P, KH, PS, E, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    pages = [2**31 // per - 1, 2**31 // per + 1, 2**32 // per - 1, 2**32 // per + 3, P - 1]
    rng = np.random.default_rng(15)
    rows = to_dev(rng.standard_normal((2, 1, KH, len(pages) * PS, E)), "bf16")
    table = torch.tensor([pages], device="cuda", dtype=torch.int32)
    n = nnop.paged_append(rows[0], rows[1], k, v, table, torch.zeros(1, device="cuda", dtype=torch.int32))
    assert n.tolist() == [len(pages) * PS]
    small = [torch.stack([x[p] for p in pages]) for x in (k, v)]
    assert torch.equal(small[0].transpose(0, 1).reshape(KH, -1, E), rows[0, 0])
    q = to_dev(rng.standard_normal((1, 16, 1, E)), "bf16")
    order = torch.arange(len(pages), device="cuda", dtype=torch.int32)[None]
    w, w2 = (torch.zeros(1, KH, len(pages) * PS, device="cuda") for _ in range(2))
    a, b = nnop._paged_attention(q, k, v, table, n, weights=w), nnop._paged_attention(q, *small, order, n, weights=w2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(w, w2)
    to = torch.tensor([[P - 3, 0]], device="cuda", dtype=torch.int32)
    _, _, kept = nnop.paged_evict(k, v, table, to, n, w, budget=20, recent=3)
    for h in (0, KH - 1):
        rows_kept = rows[0, 0, h, kept[0, h].long()]
        assert torch.equal(k[P - 3, h], rows_kept[:16]) and torch.equal(k[0, h, :4], rows_kept[16:])


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("E,T,PS", [(16, 1, 1), (32, 5, 3), (64, 40, 16), (128, 17, 20)])
@pytest.mark.parametrize("rope", [False, True])
def test_append(dtype, E, T, PS, rope):
    import torch

    import nnop
    MP = 4
    c = Cache(E + T, dtype, 2, E, PS, [0, 1, 2, 0, 3], MP=MP)
    c.lengths = np.array([0, 1, MP * PS - 1, MP * PS + 9, -3], np.int32)     # the last two: full, and taken as empty
    c.n = torch.from_numpy(c.lengths).cuda()
    n_new = np.array([T, max(T - 1, 0), T, T, T + 100], np.int32)
    k, v = (to_dev(c.rng.standard_normal((5, 2, T, E)), dtype) for _ in range(2))
    new = torch.from_numpy(n_new).cuda()
    want = k
    before = c.np()
    if rope:
        q = to_dev(c.rng.standard_normal((5, 6, T, E)), dtype)
        cos, sin = nnop.LlamaRotaryEmbedding(E)(torch.arange(5 * T, device="cuda", dtype=torch.float32).view(5, T))
        qr, n2 = nnop.paged_append_rope(q, k, v, *c.args, cos=cos, sin=sin, n_new=new)
        q2, want = nnop.llama_rope(q, k, cos=cos, sin=sin)
        assert torch.equal(qr, q2)
    else:
        n2 = nnop.paged_append(k, v, *c.args, n_new=new)
    kc, vc, n_o = orc.paged_append(to_np(want), to_np(v), *before, n_new)
    assert n2.tolist() == n_o.tolist() and c.n.tolist() == c.lengths.tolist()
    assert np.array_equal(to_np(c.k), kc, equal_nan=True) and np.array_equal(to_np(c.v), vc, equal_nan=True)


def test_append_one_table_of_angles_for_all_and_no_rows():
    import torch

    import nnop
    c = Cache(20, "bf16", 2, 64, 16, [3, 9])
    q, k, v = (to_dev(c.rng.standard_normal((2, h, 4, 64)), "bf16") for h in (4, 2, 2))
    cos, sin = nnop.LlamaRotaryEmbedding(64)(torch.arange(4, device="cuda", dtype=torch.float32)[None])
    k1, v1 = c.k.clone(), c.v.clone()
    qr, _ = nnop.paged_append_rope(q, k, v, *c.args, cos=cos, sin=sin)
    q2, n2 = nnop.paged_append_rope(q, k, v, k1, v1, c.t, c.n, cos=cos.repeat(2, 1, 1), sin=sin.repeat(2, 1, 1))
    assert torch.equal(qr, q2) and n2.tolist() == [7, 13]
    assert torch.equal(k1.view(torch.uint8), c.k.view(torch.uint8))
    zero = torch.zeros(2, device="cuda", dtype=torch.int32)
    assert torch.equal(nnop.paged_append(k, v, *c.args, n_new=zero), c.n)
    assert torch.equal(nnop.paged_append(k[:, :, :0], v[:, :, :0], *c.args), c.n)
    assert torch.equal(k1.view(torch.uint8), c.k.view(torch.uint8))


def test_append_drops_rows_without_a_page():
    import torch

    import nnop
    c = Cache(21, "f16", 1, 32, 4, [2, 2, 2], MP=3, bad=lambda t, P: t.__setitem__((slice(None), 1), [-1, P, 2**31 - 1]))
    k, v = (to_dev(c.rng.standard_normal((3, 1, 9, 32)), "f16") for _ in range(2))
    kc, vc, n_o = orc.paged_append(to_np(k), to_np(v), *c.np())
    n = nnop.paged_append(k, v, *c.args)
    assert n.tolist() == n_o.tolist() == [11, 11, 11]
    assert np.array_equal(to_np(c.k), kc, equal_nan=True) and np.array_equal(to_np(c.v), vc, equal_nan=True)


# ------------------------------------------------------------------- evict

def check_evict(c, w, budget, recent, *, new_cols=None, bad=None):
    import torch

    import nnop
    free = np.setdiff1d(np.arange(c.P), c.table)
    cols = -(-budget // c.PS) if new_cols is None else new_cols
    new_table = free[:c.B * cols].reshape(c.B, cols).astype(np.int32)
    if bad is not None:
        bad(new_table)
    want = orc.paged_evict(*c.np()[:3], new_table, c.lengths, w, budget=budget, recent=recent)
    n, nw, kept = nnop.paged_evict(*c.args[:3], torch.from_numpy(new_table).cuda(), c.n, torch.from_numpy(w).cuda(),
                                   budget=budget, recent=recent)
    torch.cuda.synchronize()
    assert np.array_equal(kept.cpu().numpy(), want[4])
    assert np.array_equal(n.cpu().numpy(), want[2])
    assert np.array_equal(nw.cpu().numpy(), want[3], equal_nan=True)
    assert np.array_equal(to_np(c.k), want[0], equal_nan=True) and np.array_equal(to_np(c.v), want[1], equal_nan=True)
    return new_table, kept


def _weights(c, kind):
    shape = (c.B, c.KH, c.MP * c.PS)
    if kind == "spread":
        w = np.exp(2 * c.rng.standard_normal(shape))
    elif kind == "ties":
        w = c.rng.integers(0, 4, shape).astype(float)
    elif kind == "equal":
        w = np.ones(shape)
    elif kind == "close":            # equal in all but the last bits
        w = 1 + c.rng.integers(0, 8, shape) * 2.0 ** -23
    else:
        w = c.rng.choice([0.0, -0.0, 1.0, -1.0, 1e-45, -1e-45, 3e38, -3e38, math.inf, -math.inf, math.nan], shape)
    return w.astype(np.float32)


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "close", "special"])
@pytest.mark.parametrize("budget,recent", [(0, 0), (1, 0), (1, 1), (50, 0), (50, 50), (64, 17), (333, 100), (2000, 5)])
def test_evict(kind, budget, recent):
    lengths = [0, 1, 49, 50, 51, 64, 65, 1000, 1999, 2000, 2100]
    c = Cache(budget + recent, "bf16", 2, 32, 16, lengths, spare=11 * 126, clean=True)
    check_evict(c, _weights(c, kind), budget, recent)


@pytest.mark.parametrize("dtype,E", [("f32", 16), ("f32", 128), ("bf16", 128), ("f16", 16), ("f16", 64)])
@pytest.mark.parametrize("PS", [1, 7, 16])
def test_evict_types_and_pages(dtype, E, PS):
    c = Cache(E + PS, dtype, 3, E, PS, [100, 7, 0, 64], spare=4 * 40)
    w = _weights(c, "spread")
    for b, n in enumerate(c.lengths):
        w[b, :, n:] = math.nan           # behind the length nothing counts
    check_evict(c, w, 30, 4)


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "special"])
def test_evict_long(kind):
    """Rows whose slots a cluster of CTAs shares, the second much shorter than its table."""
    c = Cache(31, "f16", 2, 16, 64, [70001, 33333], spare=400, clean=True)
    check_evict(c, _weights(c, kind), 9001, 100)


@pytest.mark.parametrize("kind", ["spread", "ties"])
def test_evict_rows_larger_than_shared_memory(kind):
    """Many rows leave a CTA each; a share that does not fit its shared memory is read again
    in every pass.  All sequences share their pages."""
    import torch

    import nnop
    rng = np.random.default_rng(33)
    B, KH, E, PS, MP, budget = 40, 2, 16, 64, 900, 5000
    cols = -(-budget // PS)
    P = MP + B * cols
    kc, vc = (to_dev(rng.standard_normal((P, KH, PS, E)), "f16") for _ in range(2))
    table = np.repeat(np.arange(MP, dtype=np.int32)[None], B, 0)
    new_table = (MP + np.arange(B * cols, dtype=np.int32)).reshape(B, cols)
    lengths = np.array([57600, 49157, 49152] + [7] * (B - 3), np.int32)
    w = np.exp(rng.standard_normal((B, KH, MP * PS))) if kind == "spread" else rng.integers(0, 3, (B, KH, MP * PS))
    w = w.astype(np.float32)
    want = orc.paged_evict(to_np(kc), to_np(vc), table, new_table, lengths, w, budget=budget, recent=11)
    got = nnop.paged_evict(kc, vc, *(torch.from_numpy(x).cuda() for x in (table, new_table, lengths, w)), budget=budget,
                           recent=11)
    assert np.array_equal(got[2].cpu().numpy(), want[4]) and np.array_equal(got[1].cpu().numpy(), want[3])
    assert np.array_equal(to_np(kc), want[0]) and np.array_equal(to_np(vc), want[1])


def test_captured_eviction():
    """A captured eviction replays with the weights and lengths that the device holds then."""
    import torch

    import nnop
    c = Cache(34, "bf16", 2, 32, 16, [40000, 900], spare=2 * 20, clean=True)
    free = np.setdiff1d(np.arange(c.P), c.table)[:40].reshape(2, 20).astype(np.int32)
    new_table, w = torch.from_numpy(free).cuda(), torch.rand(2, 2, c.MP * 16, device="cuda")
    call = lambda: nnop.paged_evict(c.k, c.v, c.t, new_table, c.n, w, budget=300, recent=20)  # noqa: E731
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for n in ([40000, 900], [12, 300], [0, 31234]):
        c.lengths = np.array(n, np.int32)
        c.n.copy_(torch.from_numpy(c.lengths))
        w.copy_(torch.rand_like(w))
        want = orc.paged_evict(*c.np()[:3], free, c.lengths, w.cpu().numpy(), budget=300, recent=20)
        g.replay()
        assert np.array_equal(out[2].cpu().numpy(), want[4]) and np.array_equal(out[0].cpu().numpy(), want[2])
        assert np.array_equal(out[1].cpu().numpy(), want[3]) and np.array_equal(to_np(c.v), want[1])


def test_evict_at_every_size_of_shared_memory():
    """Tables whose keys ask for shared memory from below to above what needs leave, each in
    a process of its own: leave that an earlier call got must not hide one that is missing."""
    import subprocess
    import sys
    code = """
import sys, torch
sys.path.insert(0, {path!r})
import nnop
MP = int(sys.argv[1])
i32 = dict(device='cuda', dtype=torch.int32)
k = torch.zeros(MP + 1, 1, 16, 16, device='cuda')
t = torch.arange(MP, **i32)[None]
w = torch.arange(MP * 16, device='cuda', dtype=torch.float32).view(1, 1, -1)
_, _, kept = nnop.paged_evict(k, k.clone(), t, torch.tensor([[MP]], **i32), torch.tensor([MP * 16], **i32), w, budget=16)
assert kept.flatten().tolist() == list(range(MP * 16 - 16, MP * 16))
"""
    import pathlib
    path = str(pathlib.Path(__file__).resolve().parent.parent / "onionop.jl_b200")
    runs = [subprocess.Popen([sys.executable, "-c", code.format(path=path), str(mp)], stderr=subprocess.PIPE, text=True)
            for mp in (100, 200, 320, 400, 512, 1900, 2500, 4000)]
    for r in runs:
        _, err = r.communicate(timeout=300)
        assert r.returncode == 0, err[-1000:]


def test_evictions_side_by_side():
    """Two streams evict different sequences of one pool at once."""
    import torch

    import nnop
    c = Cache(35, "f16", 4, 64, 16, [9000, 3000], spare=2 * 30, clean=True)
    free = np.setdiff1d(np.arange(c.P), c.table)[:60].reshape(2, 30).astype(np.int32)
    w = c.rng.random((2, 4, c.MP * 16)).astype(np.float32)
    want = orc.paged_evict(*c.np()[:3], free, c.lengths, w, budget=480, recent=7)
    new_table, wd = torch.from_numpy(free).cuda(), torch.from_numpy(w).cuda()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for b, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(nnop.paged_evict(c.k, c.v, c.t[b:b + 1], new_table[b:b + 1], c.n[b:b + 1], wd[b:b + 1], budget=480,
                                        recent=7))
    torch.cuda.synchronize()
    for i, k in ((0, 2), (1, 3), (2, 4)):
        assert np.array_equal(torch.cat([x[i] for x in got]).cpu().numpy(), want[k])
    assert np.array_equal(to_np(c.k), want[0]) and np.array_equal(to_np(c.v), want[1])


def test_evict_keeps_shared_pages_and_drops_what_has_no_page():
    c = Cache(32, "bf16", 2, 64, 8, [60, 60, 60], spare=30, clean=True)
    c.table[1, :4] = c.table[0, :4]              # a prefix that two sequences share
    c.table[2, 3] = -1
    import torch
    c.t = torch.from_numpy(c.table).cuda()
    old = c.k[torch.from_numpy(c.table[:2].astype(np.int64)).cuda()].clone()

    def bad(t):
        t[2, 1] = c.P
    check_evict(c, _weights(c, "spread"), 24, 8, bad=bad)
    assert torch.equal(old, c.k[torch.from_numpy(c.table[:2].astype(np.int64)).cuda()])


# ------------------------------------------------------- together, and refusals

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_run_of_decode_steps(dtype):
    """A prompt appended, then steps of append, attend, weigh, with an eviction when
    the cache is over its budget: every call against the oracle on the same state."""
    import torch

    import nnop
    rng = np.random.default_rng(40)
    B, QH, KH, E, PS, MP, budget, recent = 3, 8, 2, 64, 8, 8, 24, 8
    P = 2 * B * MP
    halves = rng.permutation(P).reshape(2, B, MP).astype(np.int32)
    tables = [torch.from_numpy(h).cuda() for h in halves]
    kc, vc = (torch.full((P, KH, PS, E), math.nan, device="cuda", dtype=torch_dtype(dtype)) for _ in range(2))
    n = torch.zeros(B, device="cuda", dtype=torch.int32)
    pos = torch.zeros(B, device="cuda", dtype=torch.int32)
    w = torch.zeros(B, KH, MP * PS, device="cuda")
    emb, use, evictions = nnop.LlamaRotaryEmbedding(E), 0, 0
    for step in range(40):
        T = 21 if step == 0 else 1
        n_new = torch.tensor([21, 13, 1] if step == 0 else [1, 1, step % 2], device="cuda", dtype=torch.int32)
        q, k, v = (to_dev(rng.standard_normal((B, h, T, E)), dtype) for h in (QH, KH, KH))
        cos, sin = emb((pos[:, None] + torch.arange(T, device="cuda")).float())
        before = to_np(kc), to_np(vc)
        qr, n2 = nnop.paged_append_rope(q, k, v, kc, vc, tables[use], n, cos=cos, sin=sin, n_new=n_new)
        q_o, k_o = nnop.llama_rope(q, k, cos=cos, sin=sin)
        want = orc.paged_append(to_np(k_o), to_np(v), *before, halves[use], n.cpu().numpy(), n_new.cpu().numpy())
        assert torch.equal(qr, q_o) and np.array_equal(n2.cpu().numpy(), want[2])
        assert np.array_equal(to_np(kc), want[0], equal_nan=True) and np.array_equal(to_np(vc), want[1], equal_nan=True)
        n, pos = n2, pos + n_new
        q1 = qr[torch.arange(B), :, (n_new.long() - 1).clamp(min=0)][:, :, None]
        w0 = to_np(w)
        o, lse = nnop._paged_attention(q1, kc, vc, tables[use], n, weights=w)
        (o_o, lse_o, w_o), (tol_o, tol_l, tol_w) = attention_oracle(to_np(q1), to_np(kc), to_np(vc), halves[use],
                                                                   n.cpu().numpy(), dtype)
        near(o, o_o, tol_o, "o")
        near(lse, lse_o, tol_l, "lse")
        near(w, w0 + w_o, tol_w + U * np.abs(w0 + w_o), "weights")
        if int(n.max()) > budget + 6:
            args = to_np(kc), to_np(vc), halves[use], halves[1 - use], n.cpu().numpy(), w.cpu().numpy()
            n, w, kept = nnop.paged_evict(kc, vc, tables[use], tables[1 - use], n, w, budget=budget, recent=recent)
            want = orc.paged_evict(*args, budget=budget, recent=recent)
            assert np.array_equal(kept.cpu().numpy(), want[4]) and np.array_equal(w.cpu().numpy(), want[3])
            assert np.array_equal(to_np(kc), want[0], equal_nan=True)
            use, evictions = 1 - use, evictions + 1
    assert evictions >= 2


def test_refusals():
    import torch

    import nnop
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    i32 = torch.int32
    kc, vc, t, n = z(4, 2, 16, 64), z(4, 2, 16, 64), z(2, 2, dt=i32), z(2, dt=i32)
    q, k, w = z(2, 4, 1, 64), z(2, 2, 3, 64), z(2, 2, 32, dt=torch.float32)
    cos = z(1, 3, 64, dt=torch.float32)
    E, S = nnop.NNopError, nnop.NNopShapeError
    att, app, ev = nnop.paged_attention, nnop.paged_append, nnop.paged_evict

    def refused(kind, text, fn, *a, **kw):
        with pytest.raises(kind, match=text):
            fn(*a, **kw)
    refused(S, "of one shape", att, q, kc, vc[:3], t, n)
    refused(E, "share a dtype", att, q, kc, vc.half(), t, n)
    refused(S, "block_table must be", att, q, kc, vc, t[:1], n)
    refused(E, "must be int32", att, q, kc, vc, t.long(), n)
    refused(E, "must be int32", att, q, kc, vc, t, n.long())
    refused(S, "same strides", att, q, kc, vc.transpose(1, 2).contiguous().transpose(1, 2), t, n)
    refused(S, "must be contiguous", att, q, *(x.transpose(2, 3).contiguous().transpose(2, 3) for x in (kc, vc)), t, n)
    refused(S, "q must be", att, z(2, 4, 2, 64), kc, vc, t, n)
    refused(S, "Embedding dim of Q", att, z(2, 4, 1, 32), kc, vc, t, n)
    refused(S, "must be divisible", att, z(2, 3, 1, 64), kc, vc, t, n)
    refused(E, "dtype of the caches", att, q.half(), kc, vc, t, n)
    refused(S, "weights must have shape", att, q, kc, vc, t, n, weights=w[:, :, :31])
    refused(E, "contiguous float32", att, q, kc, vc, t, n, weights=w.double())
    refused(E, "contiguous float32", att, q, kc, vc, t, n, weights=w.transpose(0, 1).contiguous().transpose(0, 1))
    refused(E, "has no gradient", att, q.clone().requires_grad_(), kc, vc, t, n)
    refused(E, "CUDA tensors only", att, q.cpu(), kc, vc, t, n)
    refused(S, "power-of-2", att, z(2, 4, 1, 48), z(4, 2, 16, 48), z(4, 2, 16, 48), t, n)
    refused(E, "16-byte aligned", att, q, *(z(4 * 2048 + 1)[1:].view(4, 2, 16, 64) for _ in range(2)), t, n)
    refused(S, "k and v must be", app, k[:, :1], k[:, :1], kc, vc, t, n)
    refused(E, "dtype of the caches", app, k.half(), k.half(), kc, vc, t, n)
    refused(S, "n_new must be", app, k, k, kc, vc, t, n, n_new=n[:1])
    refused(E, "n_new must be int32", app, k, k, kc, vc, t, n, n_new=n.long())
    refused(S, "expanded cache", app, k, k, *(z(1, 2, 16, 64).expand(4, -1, -1, -1) for _ in range(2)), t, n)
    refused(E, "has no gradient", app, k.clone().requires_grad_(), k, kc, vc, t, n)
    refused(S, "q must be", nnop.paged_append_rope, z(2, 4, 2, 64), k, k, kc, vc, t, n, cos=cos, sin=cos)
    refused(S, "cos/sin", nnop.paged_append_rope, z(2, 4, 3, 64), k, k, kc, vc, t, n, cos=cos[:, :2], sin=cos[:, :2])
    refused(E, "takes q, cos and sin", nnop.paged_append_rope, None, k, k, kc, vc, t, n, cos=cos, sin=cos)
    refused(S, "recent", ev, kc, vc, t, t, n, w, budget=33)
    refused(S, "recent", ev, kc, vc, t, t, n, w, budget=3, recent=4)
    refused(S, "new_table must be", ev, kc, vc, t, t[:1], n, w, budget=3)
    refused(E, "new_table must be int32", ev, kc, vc, t, t.long(), n, w, budget=3)
    refused(S, "weights must have shape", ev, kc, vc, t, t, n, w[:, :1], budget=3)
    refused(E, "must be float32", ev, kc, vc, t, t, n, w.half(), budget=3)
    with torch.no_grad():
        assert not att(q.clone().requires_grad_(), kc, vc, t, n).any()


def test_empty_calls():
    import torch

    import nnop
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    i32 = torch.int32
    kc = z(4, 2, 16, 64)
    none = nnop.paged_attention(z(0, 4, 1, 64), kc, kc, z(0, 2, dt=i32), z(0, dt=i32))
    assert none.shape == (0, 4, 1, 64)
    # a table without columns, and a pool without pages: every sequence is empty
    seven = torch.full((3,), 7, device="cuda", dtype=i32)
    for pool, table in ((kc, z(3, 0, dt=i32)), (kc[:0], z(3, 2, dt=i32))):
        o, lse = nnop._paged_attention(z(3, 4, 1, 64) + 1, pool, pool, table, seven)
        assert not o.any() and bool((lse == -math.inf).all())
        n = nnop.paged_append(z(3, 2, 2, 64), z(3, 2, 2, 64), pool, pool, table, seven)
        assert n.tolist() == [9 if table.shape[1] else 0] * 3
    n, w, kept = nnop.paged_evict(kc, kc, z(3, 0, dt=i32), z(3, 1, dt=i32), seven, z(3, 2, 0, dt=torch.float32), budget=5)
    assert n.tolist() == [0, 0, 0] and not w.any() and bool((kept == -1).all())
