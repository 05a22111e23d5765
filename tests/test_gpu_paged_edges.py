"""The paged key-value cache at its edges: precision that only a cancelling sum
shows, values that are not finite, and shapes that take a kernel variant of their
own.  Helpers and tolerances: test_gpu_paged.py (u = 2^-24, the half step of fp32)."""
import math

import numpy as np
import pytest

from _util import to_dev, to_np, torch_dtype
from test_gpu_paged import Cache, U, check_attention

pytestmark = pytest.mark.gpu

HALF = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_probabilities_enter_the_sum_with_32_bits(dtype):
    """Two keys whose values cancel to 2^-16 of themselves, so that o shows the bits of
    the probabilities that the rounding of o hides elsewhere.

    Scores are exact (one product of two 16-bit numbers; the scale is 1/4): 0 and -x, so
    the weights are 1 and p = exp(-x).  p is off by ex2's 2^-22, by 2^-21 for what its
    split into terms may drop (f16: 2^-10 of it is left by the first, rounded towards zero,
    and 2^-11 of that by the second; bf16: 2^-7, 2^-7 and 2^-8), and by 4u·x for the rounding of its argument; v1 + p·v2 by
    two half steps of its larger addend, twice (later terms are 2^-8 of it: 1/16 more);
    the division and the rounding of o by their share of o, half a step of f16's smallest
    (2^-25) where o is that small."""
    import torch

    import nnop
    B, E = 256, 16
    dt = torch_dtype(dtype)
    rng = np.random.default_rng(50)
    cast = lambda a: torch.from_numpy(np.asarray(a, np.float64)).to(dt).double().numpy()  # noqa: E731
    xq, xk = cast(rng.uniform(0.3, 1.0, B)), cast(rng.uniform(0.3, 3.0, B))
    if dtype == "f32":                       # a product that fits 24 bits there too
        xq, xk = (np.round(a * 256) / 256 for a in (xq, xk))
    x = xq * xk / 4
    p = np.exp(-x)[:, None]
    v1 = cast(rng.uniform(1, 2, (B, 512)))
    v2 = cast(-v1 / p)
    best = np.argsort(np.abs(v1 + p * v2), axis=1)[:, :E]
    v1, v2 = np.take_along_axis(v1, best, 1), np.take_along_axis(v2, best, 1)
    q, k, v = np.zeros((B, 1, 1, E)), np.zeros((B, 1, 16, E)), np.zeros((B, 1, 16, E))
    q[:, 0, 0, 3], k[:, 0, 1, 3] = xq, -xk
    v[:, 0, 0], v[:, 0, 1] = v1, v2
    k[:, :, 2:] = v[:, :, 2:] = math.nan
    table = torch.arange(B, device="cuda", dtype=torch.int32)[:, None]
    o = nnop.paged_attention(to_dev(q, dtype), to_dev(k, dtype), to_dev(v, dtype), table,
                             torch.full((B,), 2, device="cuda", dtype=torch.int32))
    want = (v1 + p * v2) / (1 + p)
    a2 = p * np.abs(v2)
    tol = (a2 * (2.0 ** -22 + 2.0 ** -21 + 4 * U * x[:, None]) + 4 * U * np.maximum(np.abs(v1), a2) * (1 + 2.0 ** -4)) / (1 + p)
    tol += (HALF[dtype] + 2.0 ** -20) * np.abs(want) + (2.0 ** -25 if dtype == "f16" else 0)
    over = np.abs(to_np(o)[:, 0, 0] - want) / tol
    assert over.max() <= 1, f"{over.max():.3g} times its tolerance"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("PS", [8, 16])
@pytest.mark.parametrize("n", [45, 20000])
def test_weights_of_a_row_that_is_not_finite(dtype, PS, n):
    """One NaN score makes every attended slot's weight NaN; slots without a page are not
    attended to and keep what they have, to the bit."""
    import torch

    import nnop
    MP = -(-n // PS)
    pages = np.arange(MP, dtype=np.int32)[None].copy()
    pages[0, 1], pages[0, MP // 2], pages[0, -1] = -1, MP, 2 ** 31 - 1
    kc, vc = (torch.randn(MP, 2, PS, 32, device="cuda").to(torch_dtype(dtype)) for _ in range(2))
    kc[0, 1, 3, 5] = math.nan                       # slot 3 of the second head
    q = torch.ones(1, 4, 1, 32, device="cuda", dtype=torch_dtype(dtype))
    w = torch.full((1, 2, MP * PS), -0.0, device="cuda")
    nnop.paged_attention(q, kc, vc, torch.from_numpy(pages).cuda(), torch.tensor([n], device="cuda", dtype=torch.int32),
                         weights=w)
    attended = np.isin(np.arange(MP * PS) // PS, [1, MP // 2, MP - 1], invert=True) & (np.arange(MP * PS) < n)
    w = w.cpu().numpy()[0]
    assert np.isnan(w[1, attended]).all() and (w[0, attended] > 0).all()
    assert (w[:, ~attended].view(np.uint32) == 0x80000000).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [2, 40000])
def test_weights_below_the_smallest_normal_number(dtype, n):
    """A key 95 below the others in score: its weight is exp(-95) / (n - 1), 5.5e-42 for two
    keys.  fp32 holds it in steps of 2^-149, and so do o (fp32, where only that key has a
    value) and the weights of every type.  Half a step each from exp, the division and
    the sum over two heads: 4 steps; and the rounding of the score, 137·2u·ln 2 of it."""
    import torch

    import nnop
    kc, vc = (torch.zeros(1, 1, n, 16, device="cuda", dtype=torch_dtype(dtype)) for _ in range(2))
    kc[0, 0, 1, 2] = -95.0
    big = {"f32": 2.0 ** 126, "bf16": 2.0 ** 126, "f16": 0.0}[dtype]
    vc[0, 0, 1] = big
    q = torch.zeros(1, 2, 1, 16, device="cuda", dtype=torch_dtype(dtype))
    q[..., 2] = 4.0                                 # the scale is 1/4
    w = torch.zeros(1, 1, n, device="cuda")
    o = nnop.paged_attention(q, kc, vc, torch.zeros(1, 1, device="cuda", dtype=torch.int32),
                             torch.tensor([n], device="cuda", dtype=torch.int32), weights=w)
    p = math.exp(-95) / (n - 1)
    assert abs(float(w[0, 0, 1]) - 2 * p) <= 4 * 2.0 ** -149 + 2 * p * 200 * U
    assert torch.allclose(w[0, 0, 2:], torch.tensor(2 / (n - 1), device="cuda"), rtol=1e-5)
    if dtype == "f32":
        # the numerator's exp(-95) alone is in steps of 2^-149
        assert np.abs(to_np(o) - p * big).max() <= 2 * 2.0 ** -149 * big / (n - 1) + p * big * 200 * U


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [48, 5000])
def test_weights_of_far_scores(dtype, n):
    """Equal scores s of about 2000 (exact: the scale is 1/4): every weight is 1/n, whatever
    the rounding of s·log2(e) (1.7e-4 in a weight) that weight and sum share.  Off by ex2's
    2^-22 in both, the division's and the sum's (80 + n/16)·u."""
    import torch

    import nnop
    B = 16
    k = np.zeros((B, 1, n, 16))
    k[:, 0, :, 0] = 125.0 + np.arange(B)[:, None] / 16 * 3
    q = np.zeros((B, 1, 1, 16))
    q[..., 0] = 64.0
    w = torch.zeros(B, 1, n, device="cuda")
    nnop.paged_attention(to_dev(q, dtype), to_dev(k, dtype), to_dev(np.zeros_like(k), dtype),
                         torch.arange(B, device="cuda", dtype=torch.int32)[:, None],
                         torch.full((B,), n, device="cuda", dtype=torch.int32), weights=w)
    assert np.abs(to_np(w) * n - 1).max() <= 2 * 2.0 ** -22 + 4 * U + (80 + n / 16) * U


def _state(MP=3, n=(20, 5)):
    """q, the new rows k and v, pools, a table, lengths and weights of two sequences."""
    import torch
    B, QH, KH, E, PS = 2, 4, 2, 64, 16
    r = lambda *s: torch.randn(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    kc, vc = r(2 * B * MP, KH, PS, E), r(2 * B * MP, KH, PS, E)
    t = torch.arange(2 * B * MP, device="cuda", dtype=torch.int32).view(2, B, MP)
    return (r(B, QH, 1, E), r(B, KH, 1, E), r(B, KH, 1, E), kc, vc, t,
            torch.tensor(n, device="cuda", dtype=torch.int32), torch.rand(B, KH, MP * PS, device="cuda"))


def test_writes_count_as_changes_in_place():
    """A backward pass that saved a pool or the weights does not go on with what a call
    has written there since; tensors of inference mode, which have no version, work."""
    import torch

    import nnop
    q, k, v, kc, vc, t, n, w = _state()
    cos, sin = nnop.LlamaRotaryEmbedding(64)(n[:, None].float())
    calls = [(lambda: nnop.paged_append(k, v, kc, vc, t[0], n), (kc, vc)),
             (lambda: nnop.paged_append_rope(q, k, v, kc, vc, t[0], n, cos=cos, sin=sin), (kc, vc)),
             (lambda: nnop.paged_attention(q, kc, vc, t[0], n, weights=w), (w,)),
             (lambda: nnop.paged_evict(kc, vc, t[0], t[1], n, w, budget=4), (kc, vc))]
    for call, written in calls:
        for x in written:
            y = torch.ones_like(x, requires_grad=True)
            z = (x[:1] * y[:1]).sum()                # saves a view of x
            call()
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                z.backward()
    y = torch.ones_like(kc, requires_grad=True)
    z = (kc * y).sum()
    nnop.paged_attention(q, kc, vc, t[0], n, weights=w)      # only reads the pools
    z.backward()
    with torch.inference_mode():
        q, k, v, kc, vc, t, n, w = _state()
        nnop.paged_append(k, v, kc, vc, t[0], n)
        nnop.paged_attention(q, kc, vc, t[0], n, weights=w)
        nnop.paged_evict(kc, vc, t[0], t[1], n, w, budget=4)


def test_tangents_are_refused():
    """A forward-mode tangent would be dropped without a word."""
    import torch
    from torch.autograd import forward_ad

    import nnop
    q, k, v, kc, vc, t, n, w = _state()
    cos, sin = nnop.LlamaRotaryEmbedding(64)(n[:, None].float())
    with torch.no_grad(), forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))  # noqa: E731
        for call in (lambda: nnop.paged_append(dual(k), v, kc, vc, t[0], n),
                     lambda: nnop.paged_append_rope(dual(q), k, v, kc, vc, t[0], n, cos=cos, sin=sin),
                     lambda: nnop.paged_attention(q, kc, dual(vc), t[0], n),
                     lambda: nnop.paged_attention(q, kc, vc, t[0], n, weights=dual(w)),
                     lambda: nnop.paged_evict(dual(kc), vc, t[0], t[1], n, w, budget=4)):
            with pytest.raises(nnop.NNopError, match="no forward-mode derivative"):
                call()
        nnop.paged_attention(q, kc, vc, t[0], n, weights=w)


@pytest.mark.parametrize("budget", [32, 40])
def test_documented_decode_loop_keeps_its_tokens(budget):
    """The decode step of INTEGRATION.md as it stands there, over several evictions: every
    token lands behind the ones before it and is attended to, none is dropped."""
    import pathlib
    import re

    import torch

    import nnop
    text = (pathlib.Path(__file__).resolve().parent.parent / "INTEGRATION.md").read_text()
    setup, step = [b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "held" in b]
    B, QH, KH, E, page_size, recent = 2, 4, 2, 64, 16, 8
    r = lambda h: torch.randn(B, h, 1, E, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    ns = dict(torch=torch, nnop=nnop, B=B, KH=KH, page_size=page_size, budget=budget, recent=recent,
              free=torch.randperm(64, device="cuda").int(), emb=nnop.LlamaRotaryEmbedding(E))
    ns["k_cache"], ns["v_cache"] = (torch.full((64, KH, page_size, E), math.nan, device="cuda", dtype=torch.bfloat16)
                                    for _ in range(2))
    exec(setup, ns)
    evictions, held = 0, 0
    for pos in range(150):
        q, k, v = r(QH), r(KH), r(KH)
        ns.update(q=q, k=k, v=v, positions=torch.full((B,), pos, device="cuda", dtype=torch.int32))
        exec(step, ns)
        held += 1
        assert not ns["o"].isnan().any()
        evicted = ns["lengths"].tolist() != [held] * B
        if evicted:
            assert ns["lengths"].tolist() == [budget] * B
            evictions, held = evictions + 1, budget
        # the newest token, among the last `recent` even after an eviction
        table, at = ns["table"], held - 1
        for b in range(B):
            assert torch.equal(ns["v_cache"][table[b, at // page_size], :, at % page_size], v[b, :, 0])
        assert (ns["weights"][:, :, at] > 0).all()
    assert evictions >= 3


# ------------------------------------------- kernel variants that take shapes of their own

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("E", [16, 32, 64, 128])
@pytest.mark.parametrize("group", [1, 8, 12, 16, 24, 40])
@pytest.mark.parametrize("PS", [1, 3, 8, 20])
def test_pages_that_do_not_hold_whole_tiles(dtype, E, group, PS):
    """Pages that no tile of 16 keys fits: every width and group (one or two head tiles a
    warp, one or two warps a key group), parts of one tile and sequences split over CTAs."""
    check_attention(Cache(E + group + PS, dtype, 1, E, PS, [0, 1, 333, 700]), group, weigh=group != 8)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("E,group", [(16, 40), (32, 12), (64, 2), (128, 12), (128, 24)])
@pytest.mark.parametrize("PS", [7, 8])
def test_odd_pages_split_over_ctas(dtype, E, group, PS):
    check_attention(Cache(E + group, dtype, 2, E, PS, [9001, 0, 3000]), 2 * group, weigh=True, scale_q=3.0)


@pytest.mark.parametrize("dtype,group", [("f32", 3), ("f32", 12), ("bf16", 3), ("f16", 12), ("bf16", 24), ("f16", 40)])
@pytest.mark.parametrize("E", [32, 128])
@pytest.mark.parametrize("PS", [3, 8, 16, 32])
def test_tables_with_holes(dtype, group, E, PS):
    """Entries without a page among pages that are there, at the ends and one after
    another, within a warp's step and over a split."""
    MP = -(-3000 // PS)

    def holes(table, P):
        table[0, 1::2] = np.resize([-1, P, 2 ** 31 - 1, -2 ** 31], table[0, 1::2].shape)
        table[1, 2:5], table[1, -3:], table[1, MP // 2] = -7, P, -1
        table[2, 0], table[2, 1:4:2] = P + 1, -1
        table[3, :] = -1
    check_attention(Cache(E + PS, dtype, 1, E, PS, [MP * PS, 3000 - 1, 77, 500], MP=MP, bad=holes), group, weigh=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("E,group,PS", [(16, 1, 16), (32, 12, 3), (64, 40, 16), (128, 4, 16), (128, 4, 20)])
@pytest.mark.parametrize("n", [1, 30, 20000])
def test_values_that_are_not_finite(dtype, E, group, PS, n):
    """An infinite element of v in an attended slot makes its column of o that infinity,
    whatever the bits of the slot's weight; NaN, or both infinities, make it NaN; the other
    columns keep their values."""
    import torch

    import nnop
    c = Cache(60, dtype, 1, E, PS, [n, n])
    q = to_dev(c.rng.standard_normal((2, group, 1, E)), dtype)
    put = lambda b, slot, e, x: c.v[int(c.table[b, slot // PS]), 0, slot % PS].__setitem__(e, x)  # noqa: E731
    before, _ = nnop._paged_attention(q, *c.args)
    put(0, 0, 0, math.inf), put(0, n - 1, 1, -math.inf), put(0, n // 2, 2, math.nan)
    for slot in range(min(n, 40)):
        put(0, slot, 3, math.inf)
    put(0, n // 2, 4, math.inf), put(0, n - 1, 4, -math.inf)
    if n > 1:
        put(0, 0, 4, -math.inf)
    o, _ = nnop._paged_attention(q, *c.args)
    assert torch.equal(o[1], before[1]) and torch.equal(o[0, :, :, 5:], before[0, :, :, 5:])
    o = to_np(o)[0, :, 0]
    assert (o[:, 0] == math.inf).all() and (o[:, 1] == -math.inf).all() and np.isnan(o[:, 2]).all()
    assert (o[:, 3] == math.inf).all()
    assert np.isnan(o[:, 4]).all() if n > 1 else (o[:, 4] == -math.inf).all()
