"""Host side of the pair-stream operators: the generator's oracle, argument checks, the C ABI's refusals."""
import ctypes as C
import random
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from fold_cp_ops_b200 import _lib
from fold_cp_ops_b200.workflows import pair_stream as P
from oracle.pair_oracle import keep_mask, philox4x32_10, rms_norm, rms_norm_grad

INCLUDE = Path(__file__).resolve().parent.parent / "include"
BF16 = 0


class Dropout(C.Structure):
    _fields_ = [("seed", C.c_uint64), ("offset", C.c_uint32), ("keep", C.c_uint32), ("device_seed", C.c_void_p),
                ("shared", C.c_int32), ("origin_b", C.c_int32), ("origin_i", C.c_int32), ("origin_j", C.c_int32)]


class Tensor4(C.Structure):
    _fields_ = [("data", C.c_void_p), ("stride_b", C.c_int64), ("stride_i", C.c_int64), ("stride_j", C.c_int64)]


class NormDesc(C.Structure):
    _fields_ = [("b", C.c_int32), ("i", C.c_int32), ("j", C.c_int32), ("d", C.c_int32), ("dtype", C.c_int32),
                ("weight_dtype", C.c_int32), ("group", C.c_int32), ("eps", C.c_float), ("dropout", Dropout)]


class EmbedDesc(C.Structure):
    _fields_ = [("tokens", C.c_int64), ("d", C.c_int32), ("rows", C.c_int32), ("index_bits", C.c_int32),
                ("dtype", C.c_int32), ("table_dtype", C.c_int32), ("scale", C.c_float)]


def refused(name, pat, *args):
    """The C entry refuses: pointers that are no structs stand for addresses that it must not reach."""
    args = [C.byref(a) if isinstance(a, C.Structure) else None if a is None else C.c_void_p(a) for a in args]
    with pytest.raises(ValueError, match=pat):
        _lib.check(getattr(_lib.load(), name)(*args), name)


# ------------------------------------------------------------------------------------------------
# the oracle itself
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("counter,key,words", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_the_oracles_generator_gives_the_published_known_answers(counter, key, words):
    assert tuple(int(w) for w in philox4x32_10(counter, key)) == words


def test_the_oracles_mask_keeps_the_share_and_repeats_along_the_shared_axis():
    shape, p = (2, 48, 40, 96), 0.25
    n = np.prod(shape)
    mask, gain = keep_mask(shape, p, 1 << 40, 3)
    # a binomial share: five standard deviations
    assert abs(mask.double().mean().item() - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5 and gain == 65536 / 49152
    rows, _ = keep_mask(shape, p, 7, 0, "rows")
    cols, _ = keep_mask(shape, p, 7, 0, "columns")
    assert torch.equal(rows, rows[:, :1].expand(shape)) and torch.equal(cols, cols[:, :, :1].expand(shape))
    whole, _ = keep_mask(shape, p, 7, 5)
    block, _ = keep_mask((1, 10, 20, 96), p, 7, 5, origin=(1, 30, 15))
    assert torch.equal(block, whole[1:, 30:40, 15:35])


def test_the_oracles_gradient_is_that_of_differences():
    """Central differences of the 64-bit norm with step 1e-5: truncation about h^2 = 1e-10 and rounding about 1e-16 / h."""
    g = torch.Generator().manual_seed(3)
    z, w, dy, dz = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 7), (7,), (3, 7), (3, 7)))
    f = lambda z, w: (rms_norm(z, w, 1e-3) * dy).sum() + (z * dz).sum()  # noqa: E731
    got, _, got_w, _ = rms_norm_grad(z, w, 1e-3, dy, dz)
    h = 1e-5
    for k in range(z.numel()):
        step = torch.zeros(z.numel(), dtype=torch.float64)
        step[k] = h
        step = step.reshape(z.shape)
        assert abs((f(z + step, w) - f(z - step, w)) / (2 * h) - got.reshape(-1)[k]) < 1e-7
    for k in range(7):
        step = torch.zeros(7, dtype=torch.float64)
        step[k] = h
        assert abs((f(z, w + step) - f(z, w - step)) / (2 * h) - got_w[k]) < 1e-7


# ------------------------------------------------------------------------------------------------
# C ABI
# ------------------------------------------------------------------------------------------------
def test_library_exports_every_symbol_of_the_pair_header():
    header = (INCLUDE / "pair_stream_sm100.h").read_text()
    assert set(re.findall(r"\b(pair_sm100_[a-z_0-9]+)\s*\(", header)) == set(_lib.PAIR_SYMBOLS)
    lib = C.CDLL(str(_lib.library_path()))
    assert all(hasattr(lib, s) for s in _lib.PAIR_SYMBOLS)


def test_ctypes_mirrors_match_the_pair_headers_structs(tmp_path):
    import shutil
    import subprocess

    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    mirrors = {"pair_dropout": Dropout, "pair_tensor": Tensor4, "pair_norm_desc": NormDesc, "pair_embed_desc": EmbedDesc}
    header = (INCLUDE / "pair_stream_sm100.h").read_text()
    assert set(re.findall(r"typedef struct (\w+) \{", header)) == set(mirrors)
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "pair_stream_sm100.h"', 'int main(void) {']
    want = []
    for name, mirror in mirrors.items():
        lines.append(f'  printf("%zu\\n", sizeof(struct {name}));')
        want.append(C.sizeof(mirror))
        for f, _ in mirror._fields_:
            lines.append(f'  printf("%zu\\n", offsetof(struct {name}, {f}));')
            want.append(getattr(mirror, f).offset)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-I", str(INCLUDE), str(src), "-o", str(exe)], check=True, capture_output=True)
    assert [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()] == want


def test_the_packed_dropout_has_the_headers_layout():
    drop = P.PairDropout(0.25, seed=0x8123456789ABCDEF, offset=7, shared="columns", origin=(3, 4, 5))
    assert P._record(drop, None) == (bytes(Dropout(0x8123456789ABCDEF, 7, 49152, None, 2, 3, 4, 5)), None)
    assert P._record(None, None) == P._record(P.PairDropout(1e-6), None) == (b"", None)


def test_the_host_module_was_built_from_these_sources(monkeypatch):
    from fold_cp_ops_b200 import build

    host = _lib.pair_host()
    assert host.build_id() == build.source_digest()
    monkeypatch.setattr(_lib, "_pair", None)
    monkeypatch.setattr(build, "source_digest", lambda: "0" * 32)
    with pytest.raises(_lib.TrimulLibraryError, match="was not built from the sources"):
        _lib.pair_host()


def _norm(**kw):
    d = NormDesc(1, 2, 3, 64, BF16, BF16, 0, 1e-5, Dropout(keep=65536))
    for k, v in kw.items():
        setattr(d.dropout if k in ("keep", "shared", "origin_b", "origin_i") else d, k, v)
    return d


@pytest.mark.parametrize("kw,pat", [
    (dict(d=0), "not a pair tensor"), (dict(i=-1), "not a pair tensor"), (dict(d=8193), "above 8192"),
    (dict(b=1 << 15, i=1 << 15, j=2), "2\\^31"), (dict(i=1 << 30, b=1 << 30), "2\\^31"), (dict(dtype=3), "unknown type"),
    (dict(weight_dtype=-1), "unknown type"), (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=1e-40), "eps"), (dict(eps=float("inf")), "eps"), (dict(keep=65537), "65536"), (dict(shared=3), "shared"),
    (dict(origin_i=-1), "origin"), (dict(keep=1, origin_b=65536), "batch entries"),
    (dict(group=16), "group"), (dict(d=96, group=64), "does not divide"),
])
def test_norm_refusals_of_the_c_entry(kw, pat):
    """Every refusal comes before anything is launched: the pointers are never read."""
    d, t = _norm(**kw), Tensor4(4096, 64, 64, 64)
    refused("pair_sm100_add_norm", pat, d, t, None, 4096, 4096, 4096, 4096, None)
    if "group" not in kw:
        refused("pair_sm100_add_norm_grad", pat, d, t, None, None, 4096, 4096, None, None, None, None)


def test_refusals_of_buffers_that_their_elements_do_not_fit():
    t = Tensor4(4096, 64, 64, 64)
    for args in ((Tensor4(4097, 64, 64, 64), None, 4096, 4096, 4096, None), (t, Tensor4(4097, 64, 64, 64), 4096, 4096, 4096, None),
                 (t, None, 4097, 4096, 4096, None), (t, None, 4096, 4097, 4096, None), (t, None, 4096, 4096, 4097, None)):
        refused("pair_sm100_add_norm", "not aligned", _norm(), *args, None)
    refused("pair_sm100_add_norm", "not aligned", _norm(dtype=2), Tensor4(4098, 64, 64, 64), None, 4096, 4096, 4096, None, None)
    refused("pair_sm100_add_norm_grad", "not aligned", _norm(), t, Tensor4(4097, 64, 64, 64), None, 4096, 4096, None, None, None, None)
    refused("pair_sm100_add_norm_grad", "not aligned", _norm(), t, None, None, 4096, 4096, None, 4097, 4096, None)
    d = EmbedDesc(10, 64, 5, 64, BF16, BF16, 1.0)
    refused("pair_sm100_embed", "not aligned", d, 4100, 4096, None, 4096, None)
    refused("pair_sm100_embed", "not aligned", d, 4096, 4096, 4097, 4096, None)
    refused("pair_sm100_embed_grad", "not aligned", d, 4096, 4096, 4097, 4096, None)


def test_norm_refusals_of_missing_buffers():
    d, t = _norm(), Tensor4(4096, 64, 64, 64)
    for args, pat in (((None, 4096, 4096, None, None), "come together"), ((None, None, 4096, 4096, None), "come together"),
                      ((None, None, None, None, None), "no output")):
        refused("pair_sm100_add_norm", pat, d, t, *args, None)
    refused("pair_sm100_add_norm", "update is NULL", d, None, None, 4096, 4096, 4096, None, None)
    refused("pair_sm100_add_norm", "needs y and scales", _norm(group=64), t, None, 4096, 4096, 4096, None, None)
    refused("pair_sm100_add_norm", "16-byte boundaries", _norm(group=32), Tensor4(4098, 64, 64, 64), None, 4096, 4096, 4096, 4096, None)
    refused("pair_sm100_add_norm", "16-byte boundaries", _norm(group=32), Tensor4(4096, 64, 64, 65), None, 4096, 4096, 4096, 4096, None)
    for args, pat in (((None, 4096, 4096, 4096, 4096), "weight is NULL"), ((4096, None, None, None, None), "no output"),
                      ((4096, 4096, None, 4096, None), "workspace"), ((4096, 4096, None, 4096, 4100), "workspace")):
        refused("pair_sm100_add_norm_grad", pat, d, t, None, None, *args, None)


@pytest.mark.parametrize("kw,pat", [
    (dict(tokens=-1), "tokens"), (dict(tokens=1 << 31), "2\\^31"), (dict(d=0), "width"), (dict(d=9000), "8192"),
    (dict(rows=0), "table rows"), (dict(index_bits=16), "32 nor 64"), (dict(dtype=5), "unknown type"),
    (dict(table_dtype=5), "unknown type"),
])
def test_embedding_refusals_of_the_c_entry(kw, pat):
    d = EmbedDesc(10, 64, 5, 64, BF16, BF16, 1.0)
    for k, v in kw.items():
        setattr(d, k, v)
    refused("pair_sm100_embed", pat, d, 4096, 4096, None, 4096, None)
    refused("pair_sm100_embed_grad", pat, d, 4096, 4096, 4096, 4096, None)


def test_quotients_by_multiplication_are_exact():
    """The kernels' row arithmetic: floor(n m / 2^(31+l)) with m = ceil(2^(31+l) / d) for every 0 <= n < 2^31."""
    rng = random.Random(1)
    divisors = [1, 2, 3, 5, 7, 8, 96, 197, 1023, 1024, 1025, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, (1 << 31) - 1]
    for d in divisors + [rng.randrange(1, 1 << 31) for _ in range(300)]:
        shift = max(0, (d - 1).bit_length())
        m = ((1 << (31 + shift)) + d - 1) // d
        assert m < 1 << 32
        for n in [0, 1, d - 1, d, (1 << 31) - 1] + [rng.randrange(1 << 31) for _ in range(50)] + \
                 [k for q in (1, 5, ((1 << 31) - 1) // d) for k in (q * d - 1, q * d) if 0 <= k < 1 << 31]:
            assert (n * m) >> (31 + shift) == n // d


# ------------------------------------------------------------------------------------------------
# the front door
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kw", [dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(p=0.5, shared="i"), dict(p=0.5, seed=-1),
                                dict(p=0.5, seed=1 << 64), dict(p=0.5, offset=1 << 32), dict(p=0.5, origin=(0, 0)),
                                dict(p=0.5, origin=(0, -1, 0)), dict(p=0.5, seed=torch.zeros(2, dtype=torch.int64))])
def test_dropout_refusals(kw):
    with pytest.raises(ValueError):
        P.PairDropout(**kw)


def test_dropout_keeps_the_nearest_of_65536():
    assert P.PairDropout(0.0).keep == 65536 and P.PairDropout(1.0).keep == 0
    assert P.PairDropout(0.25).keep == 49152 and P.PairDropout(0.1).keep == 58982


def test_there_is_no_cpu_path():
    x, w = torch.zeros(2, 3, 4, 8), torch.ones(8)
    for call in (lambda: P.dropout_add(x, x), lambda: P.add_rms_norm(x, None, w), lambda: P.add_rms_norm_fp8(x, x, w, group=None),
                 lambda: P.pair_embedding(torch.zeros(3, dtype=torch.int64), w[None])):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_the_alias_package_reaches_the_pair_stream():
    from fold_cp_ops.workflows import pair_stream as alias

    assert alias is P
