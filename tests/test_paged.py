"""CPU checks of the paged key-value cache: the oracle against the attention
oracle and by hand, the refusals of the C ABI before any launch, and the
arithmetic that finds a slot's page and shares a ragged batch out."""
import ctypes as C

import numpy as np
import pytest

from oracle import nnop_oracle as orc


def _table(rng, B, MP, spare=0):
    return rng.permutation(B * MP + spare)[:B * MP].reshape(B, MP).astype(np.int32)


def test_oracle_attention_is_attention_of_the_last_token():
    """A cache laid out in pages and attention over the same rows agree."""
    rng = np.random.default_rng(0)
    B, QH, KH, E, PS, MP = 3, 6, 2, 16, 5, 4
    table = _table(rng, B, MP, 2)
    kc, vc = rng.standard_normal((2, B * MP + 2, KH, PS, E))
    q = rng.standard_normal((B, QH, 1, E))
    lengths = np.array([20, 1, 13])
    o, lse, w = orc.paged_attention(q, kc, vc, table, lengths, scale=0.25)
    for b, n in enumerate(lengths):
        k, v = (np.stack([c[table[b, j // PS], :, j % PS] for j in range(n)], axis=1)[None] for c in (kc, vc))
        o2, lse2 = orc.attention_fwd(q[b:b + 1], k, v, causal=False, scale=0.25)
        assert np.allclose(o[b], o2[0], atol=1e-14) and np.allclose(lse[b], lse2[0], atol=1e-14)
        assert np.allclose(w[b].sum(-1), QH // KH) and not w[b][:, n:].any()


def test_oracle_append_then_attend_grows_the_sequence():
    rng = np.random.default_rng(1)
    B, KH, E, PS, MP, T = 2, 1, 16, 3, 3, 4
    table = _table(rng, B, MP)
    kc, vc = np.zeros((2, B * MP, KH, PS, E))
    k, v = rng.standard_normal((2, B, KH, T, E))
    kc, vc, lengths = orc.paged_append(k, v, kc, vc, table, np.array([0, 7]), np.array([4, 4]))
    assert list(lengths) == [4, 9]                      # the second is cut at its 9 slots
    assert np.array_equal(kc[table[0, 1], 0, 0], k[0, 0, 3])
    assert np.array_equal(vc[table[1, 2], 0, 2], v[1, 0, 1])


def test_oracle_evict_by_hand():
    kc = np.arange(8, dtype=np.float64).reshape(4, 1, 2, 1)    # pages of two slots: slot j of page p holds 2p + j
    table, new_table = np.array([[0, 1]]), np.array([[3, 2]])
    w = np.array([[[2, 5, 5, 1]]], np.float32)
    k2, _, n, nw, kept = orc.paged_evict(kc, kc, table, new_table, np.array([4]), w, budget=2, recent=1)
    assert list(kept[0, 0]) == [1, 3] and list(n) == [2] and list(nw[0, 0]) == [5, 1, 0, 0]
    assert k2[3, 0, 0, 0] == 1 and k2[3, 0, 1, 0] == 3
    _, _, n, nw, kept = orc.paged_evict(kc, kc, table, new_table, np.array([3]), w, budget=4, recent=1)
    assert list(kept[0, 0]) == [0, 1, 2, -1] and list(n) == [3] and list(nw[0, 0]) == [2, 5, 5, 0]


def test_page_division():
    """The kernels' division by the page size (a multiplication) is exact below 2^31."""
    rng = np.random.default_rng(2)
    for d in [1, 2, 3, 5, 7, 16, 20, 24, 64, 100, 127, 129, 641, 6700417, 2**30 - 1, 2**30, 2**30 + 1, 2**31 - 1024,
              *map(int, rng.integers(1, 2**31 - 1, 200))]:
        s = 0
        while s < 31 and (1 << s) < d:
            s += 1
        m = ((2**32 * ((1 << s) - d)) // d + 1) % 2**32
        near = [x for k in (0, 1, 2, 2**31 // d - 1, 2**31 // d) for x in (k * d - 1, k * d, k * d + 1)]
        n = np.array([x for x in [*near, 2**31 - 1, *rng.integers(0, 2**31, 200)] if 0 <= x < 2**31], np.uint64)
        hi = (n * np.uint64(m)) >> np.uint64(32)
        assert np.all(hi + n < 2**32)                       # the kernels' 32-bit sum
        assert np.array_equal((hi + n) >> np.uint64(s), n // np.uint64(d)), d


def _segments(lens, heads, ctas, unit, extra, parts):
    """The kernels' split, restated: for each part its segments (b, h, c0, c1) and, per
    (b, h), what owner() says of its first and last chunk."""
    total, some = sum(-(-n // unit) for n in lens), sum(n > 0 for n in lens)
    extra = extra if total * heads > ctas else 0
    chunks = [-(-n // unit) + extra if n else 0 for n in lens]
    units = sum(chunks) * heads
    G, parts = min(ctas, units), min(parts, units)
    where = [(b, h, c) for b, n in enumerate(chunks) for h in range(heads) for c in range(n)]
    segments = []
    for p in range(parts):
        u, u1 = units * p // parts, units * (p + 1) // parts
        mine = []
        if u < u1:
            b, h, c0 = where[u]
            if c0 <= extra:
                u, c0 = u - c0, 0
            while u < u1:
                c1 = min(chunks[b], c0 + u1 - u)
                if c1 <= extra and c1 < chunks[b]:
                    break
                mine.append((b, h, c0, c1))
                u += c1 - c0
                if u < u1:
                    b, h, c0 = where[u]
                    assert c0 == 0
        segments.append(mine)
    first = {bh: i for i, bh in reversed(list(enumerate(w[:2] for w in where)))}

    def owner(e):
        return ((e + 1) * G + units - 1) // units - 1
    owners = {(b, h): (owner(u + extra), owner(u + chunks[b] - 1)) for (b, h), u in first.items()}
    return segments, owners, extra, chunks


@pytest.mark.parametrize("ctas", [1, 7, 444])
@pytest.mark.parametrize("extra", [0, 1, 4, 9])
def test_split_covers_every_chunk_once(ctas, extra):
    """Whatever the lengths: every chunk with slots in one part, the parts of a (b, h) in
    consecutive CTAs from the first to the last that owner() names, so that each CTA has
    at most one part that begins inside a (b, h) and one that ends inside."""
    rng = np.random.default_rng(ctas + extra)
    for trial in range(25):
        lens = [int(n) for n in rng.integers(0, [1, 3, 40, 700][trial % 4] + 1, rng.integers(1, 12))]
        heads = int(rng.integers(1, 5))
        segments, owners, ex, chunks = _segments(lens, heads, ctas, 16, extra, ctas)
        got = {}
        for c, mine in enumerate(segments):
            assert sum(c0 > 0 for _, _, c0, _ in mine) <= 1 and sum(c1 < chunks[b] for b, _, _, c1 in mine) <= 1
            for b, h, c0, c1 in mine:
                got.setdefault((b, h), []).append((c, c0, c1))
        assert set(got) == set(owners) == {(b, h) for b, n in enumerate(lens) if n for h in range(heads)}
        for (b, h), parts in got.items():
            assert (parts[0][0], parts[-1][0]) == owners[b, h]
            assert [p[0] for p in parts] == list(range(parts[0][0], parts[-1][0] + 1))
            assert parts[0][1] == 0 and parts[-1][2] == chunks[b]
            assert all(x[2] == y[1] for x, y in zip(parts, parts[1:])) and (len(parts) == 1 or parts[0][2] > ex)
        # any other number of parts covers the chunks too (the second launch's)
        seen = [(b, h, c) for mine in _segments(lens, heads, ctas, 16, extra, 3 * ctas + 1)[0]
                for b, h, c0, c1 in mine for c in range(max(c0, ex), c1)]
        assert sorted(seen) == [(b, h, c) for b, n in enumerate(chunks) for h in range(heads) for c in range(ex, n)]


D = C.c_void_p(4096)      # never dereferenced: every call below is refused before a launch


def _append(lib, *, q=None, k=D, v=D, cos=None, sin=None, qo=None, kc=D, vc=D, table=D, lengths=D, new=C.c_void_p(8192),
            E=64, T=1, QH=0, KH=2, B=1, cb=1, P=4, PS=16, MP=2, ps=2048, hs=1024, rs=64, dtype=2):
    return lib.nnop_paged_append(q, k, v, cos, sin, None, qo, kc, vc, table, lengths, new, E, T, QH, KH, B, cb, P, PS, MP,
                                 ps, hs, rs, dtype, None)


def _attend(lib, *, q=D, kc=D, vc=D, table=D, lengths=D, weights=None, o=D, lse=D, ws=D, nbytes=1 << 40, E=64, QH=4,
            KH=2, B=1, P=4, PS=16, MP=2, ps=2048, hs=1024, rs=64, dtype=2):
    return lib.nnop_paged_attention_fwd(q, kc, vc, table, lengths, weights, o, lse, ws, nbytes, E, QH, KH, B, P, PS, MP,
                                        ps, hs, rs, dtype, None)


def _evict(lib, *, kc=D, vc=D, table=D, new_table=D, lengths=D, weights=D, new=C.c_void_p(8192), nw=C.c_void_p(8192), kept=D,
           E=64, KH=2, B=1, P=4, PS=16, MP=2, NP=1, ps=2048, hs=1024, rs=64, budget=8, recent=2, dtype=2):
    return lib.nnop_paged_evict(kc, vc, table, new_table, lengths, weights, new, nw, kept, E, KH, B, P, PS, MP, NP, ps, hs,
                                rs, budget, recent, dtype, None)


@pytest.mark.parametrize("call", [_append, _attend, _evict])
def test_cache_refusals(call):
    from nnop._lib import lib
    assert call(lib, dtype=3) == -2
    assert call(lib, E=48) == -1 and b"power-of-2" in lib.nnop_last_error()
    assert call(lib, E=8) == -1 and call(lib, E=256) == -1
    assert call(lib, PS=0) == -1 and call(lib, MP=-1) == -1 and call(lib, P=-1) == -1 and call(lib, KH=0) == -1
    assert call(lib, B=-1) == -1 and call(lib, B=65536) == -1
    assert call(lib, PS=1 << 20, MP=1 << 11) == -1          # 2^31 slots
    assert call(lib, P=1 << 31) == -1
    assert call(lib, ps=2044) == -6 and call(lib, rs=60) == -6 and call(lib, hs=-64) == -1
    assert call(lib, kc=C.c_void_p(4100)) == -6
    assert call(lib, kc=None) == -3 and call(lib, table=None) == -3 and call(lib, lengths=None) == -3
    assert call(lib, B=0) == 0                              # nothing to do


def test_append_refusals():
    from nnop._lib import lib
    assert _append(lib, T=-1) == -1 and _append(lib, QH=-1) == -1
    assert _append(lib, cos=D) == -3                        # cos without sin
    assert _append(lib, q=D, QH=4, qo=D) == -3              # q without cos and sin
    assert _append(lib, q=D) == -3                          # q without heads
    assert _append(lib, QH=4, cos=D, sin=D) == -3
    assert _append(lib, cos=D, sin=D, B=3, cb=2) == -1
    assert _append(lib, new=None) == -3 and _append(lib, new=D) == -3
    assert _append(lib, k=None) == -3 and _append(lib, k=C.c_void_p(8)) == -6


def test_attention_refusals():
    from nnop._lib import lib
    assert _attend(lib, QH=3) == -1 and b"must be divisible by number of KV heads `2`" in lib.nnop_last_error()
    assert _attend(lib, q=None) == -3 and _attend(lib, lse=None) == -3 and _attend(lib, ws=None) == -3
    need = lib.nnop_paged_attention_fwd_workspace_size(64, 4, 2, 1, 16, 2, 0, 2)
    assert need > 0 and _attend(lib, nbytes=need - 1) == -4
    assert _attend(lib, ws=C.c_void_p(4096 + 16)) == -6 and _attend(lib, q=C.c_void_p(8)) == -6
    assert _attend(lib, B=65535, QH=65534, KH=2, PS=1 << 20, MP=1 << 10) == -1      # 2^62 scores
    # with weights the workspace also holds a score per query head and slot
    assert lib.nnop_paged_attention_fwd_workspace_size(64, 4, 2, 1, 16, 2, 1, 2) >= need + 4 * 32 * 4


def test_evict_refusals():
    from nnop._lib import lib
    assert _evict(lib, budget=17) == -1                     # 16 slots in the new table
    assert _evict(lib, budget=-1, recent=0) == -1 and _evict(lib, recent=9) == -1 and _evict(lib, recent=-1) == -1
    assert _evict(lib, new=None) == -3 and _evict(lib, new=D) == -3 and _evict(lib, nw=D) == -3
    assert _evict(lib, kept=None) == -3 and _evict(lib, weights=None) == -3 and _evict(lib, new_table=None) == -3


def test_no_cpu_fallback():
    import torch

    import nnop
    pool, table, n = torch.zeros(2, 1, 16, 16), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: nnop.paged_append(pool[:1], pool[:1], pool, pool, table, n),
                 lambda: nnop.paged_attention(pool[:1, :, :1], pool, pool, table, n),
                 lambda: nnop.paged_evict(pool, pool, table, table, n, torch.zeros(1, 1, 16), budget=1)):
        with pytest.raises(nnop.NNopError, match="CUDA tensors only"):
            call()
