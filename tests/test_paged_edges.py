"""CPU checks around the paged key-value cache: the package on a torch without CUDA,
what the C ABI refuses at its limits, and the documented bindings."""
import os
import pathlib
import re
import subprocess
import sys

from test_paged import _append, _attend, _evict

ROOT = pathlib.Path(__file__).resolve().parent.parent


def test_package_imports_on_a_torch_without_cuda():
    """Such a torch lacks the raw stream call; the package imports and refuses per call."""
    code = """
import torch
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    del torch._C._cuda_getCurrentRawStream
import nnop
pool, i32 = torch.zeros(2, 1, 16, 16), torch.int32
try:
    nnop.paged_attention(pool[:1, :, :1], pool, pool, torch.zeros(1, 1, dtype=i32), torch.zeros(1, dtype=i32))
except nnop.NNopError as e:
    assert "CUDA tensors only" in str(e)
else:
    raise SystemExit("not refused")
"""
    env = dict(os.environ, PYTHONPATH=str(ROOT / "onionop.jl_b200"), CUDA_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-1000:]


def test_evict_refuses_what_its_counters_do_not_hold():
    """The choice of slots goes through a row in steps of up to 8192 slots (a cluster of 8
    CTAs of 1024 threads) with 32-bit counters: the last step ends past the last slot, so
    8192 slots fewer than 2^31 are the most.  The calls at the limit are refused for a
    missing array, none is launched."""
    from nnop._lib import lib
    assert 2 ** 31 - 8192 - 1 + 8192 <= 2 ** 31 - 1
    for pages in ({"MP": 2 ** 21 - 1}, {"NP": 2 ** 21 - 1}, {"NP": 2 ** 21 - 7}, {"MP": 2 ** 21 - 7}):
        assert _evict(lib, PS=1024, kept=None, **pages) == -1, pages
        assert b"2^31 - 8192 slots" in lib.nnop_last_error()
    for pages in ({"MP": 2 ** 21 - 8}, {"NP": 2 ** 21 - 8}):
        assert _evict(lib, PS=1024, kept=None, **pages) == -3
    # the other calls' counters step by at most 1024
    assert _append(lib, PS=1024, MP=2 ** 21 - 1, new=None) == -3 and _attend(lib, PS=1024, MP=2 ** 21 - 1, lse=None) == -3


def test_append_refuses_to_write_the_lengths_over_the_counts():
    """Other blocks still read n_new while new_lengths is written."""
    import ctypes as C

    from nnop._lib import lib
    a, b = C.c_void_p(4096), C.c_void_p(8192)
    call = lambda n_new, new: lib.nnop_paged_append(None, a, a, None, None, n_new, None, a, a, a, a, new,  # noqa: E731
                                                    64, 1, 0, 2, 1, 1, 4, 16, 2, 2048, 1024, 64, 2, None)
    assert call(b, b) == -3 and b"lengths or n_new" in lib.nnop_last_error()


def _split(text):
    """The arguments of a Julia call: what lies between commas outside all brackets."""
    parts, depth, last = [], 0, 0
    for i, c in enumerate(text):
        depth += (c in "([{") - (c in ")]}")
        if c == "," and depth == 0:
            parts.append(text[last:i])
            last = i + 1
    return [p.strip() for p in [*parts, text[last:]] if p.strip()]


def _ccalls():
    """(name, return type, argument types, arguments) of each ccall in the documented binding."""
    text = (ROOT / "INTEGRATION.md").read_text()
    for block in re.findall(r"```julia\n(.*?)```", text, re.S):
        block = re.sub(r"#.*", "", block)
        for m in re.finditer(r"ccall\(", block):
            depth, i = 1, m.end()
            while depth:
                depth += (block[i] == "(") - (block[i] == ")")
                i += 1
            target, result, types, *args = _split(block[m.end():i - 1])
            yield re.match(r"\(:(\w+), libnnop\)", target)[1], result, _split(types[1:-1]), args


def test_documented_bindings_have_the_signatures_of_the_library():
    """Julia's ccall pairs types and arguments as they are written: one argument for each
    type, no splat.  The paged calls are all bound."""
    import ctypes as C

    from nnop._lib import SIGNATURES
    kinds = {"Int64": C.c_int64, "Cint": C.c_int, "Csize_t": C.c_size_t, "Float32": C.c_float, "Cstring": C.c_char_p}
    of = lambda t: C.c_void_p if re.fullmatch(r"(Cu)?Ptr\{\w+\}", t) else kinds[t]  # noqa: E731
    seen = set()
    for name, result, types, args in _ccalls():
        res, argtypes = SIGNATURES[name]
        assert not any(a.endswith("...") for a in args), name
        assert len(types) == len(args) == len(argtypes), name
        assert [of(t) for t in types] == list(argtypes) and of(result) == res, name
        seen.add(name)
    assert {n for n in SIGNATURES if n.startswith("nnop_paged")} <= seen


def test_page_division_and_split_as_compiled(tmp_path):
    """FastDiv and the split's start() and owner() themselves, compiled for the host:
    against division, and against a walk over all units."""
    import ctypes as C

    import numpy as np
    from nnop import _build
    src, so = tmp_path / "split.cu", tmp_path / "split.so"
    src.write_text("""
        #include "paged.cuh"
        using namespace nnop::paged;
        extern "C" void divide(uint32_t d, const uint32_t* n, uint32_t* out, int count) {
            const FastDiv f(d);
            for (int i = 0; i < count; ++i) out[i] = f.div(n[i]);
        }
        extern "C" long long start(long long units, int c, int G) { return Split::start(units, c, G); }
        extern "C" int owner(long long units, int G, long long e) {
            Split s{};
            s.units = units, s.G = G;
            return s.owner(e);
        }
    """)
    subprocess.run([_build.nvcc(), *_build.NVCC_FLAGS, "-shared", str(src), "-o", str(so)], check=True, timeout=300)
    lib = C.CDLL(str(so))
    lib.divide.argtypes = [C.c_uint32, C.c_void_p, C.c_void_p, C.c_int]
    lib.start.argtypes, lib.start.restype = [C.c_longlong, C.c_int, C.c_int], C.c_longlong
    lib.owner.argtypes = [C.c_longlong, C.c_int, C.c_longlong]
    rng = np.random.default_rng(3)
    for d in [1, 2, 3, 5, 7, 16, 20, 24, 64, 127, 129, 641, 6700417, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1024,
              *map(int, rng.integers(1, 2 ** 31 - 1, 100))]:
        near = [x for k in (0, 1, 2, 2 ** 31 // d - 1, 2 ** 31 // d) for x in (k * d - 1, k * d, k * d + 1)]
        n = np.array([x for x in [*near, 2 ** 31 - 1, *rng.integers(0, 2 ** 31, 200)] if 0 <= x < 2 ** 31], np.uint32)
        out = np.zeros_like(n)
        lib.divide(d, n.ctypes.data, out.ctypes.data, len(n))
        assert np.array_equal(out, n // np.uint32(d)), d
    for units, G in [(1, 1), (7, 7), (7, 3), (443, 443), (444, 444), (1000, 444), (12345, 444), (3, 1), (99999, 296)]:
        starts = [lib.start(units, c, G) for c in range(G + 1)]
        assert starts[0] == 0 and starts[-1] == units and all(a < b for a, b in zip(starts, starts[1:]))
        owners = np.searchsorted(starts, np.arange(units), side="right") - 1
        assert [lib.owner(units, G, e) for e in range(units)] == owners.tolist()
    for units, G in [(9 * 10 ** 15, 444), (2 ** 40 + 12345, 444)]:          # past 32 bits, at the most the host lets through
        for c in (0, 1, 100, 443):
            a, b = lib.start(units, c, G), lib.start(units, c + 1, G)
            assert a == units * c // G and b == units * (c + 1) // G
            assert lib.owner(units, G, a) == c == lib.owner(units, G, b - 1)
