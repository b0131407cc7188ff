"""The kernels that the block-scaled products are compiled to (CPU): each is one that a call can reach by the library's rule."""
import re
import subprocess

import pytest

from _blocks import plan
from h3_tp2_amd import _lib

CUS = (64, 256, 304)
ROWS = sorted({int(2 ** (i / 4)) for i in range(0, 84)} | {16, 17, 32, 33, 64, 65, 128, 129})
CHANNELS = (16, 400, 1536, 2064, 4096, 5376, 6160, 13008, 16000, 21504, 43008)
EXPERTS = (1, 3, 16, 32, 300)


@pytest.fixture(scope="module")
def compiled():
    """The kernels of the built library: (channels, tokens, non-temporal, by expert), with fp16 and bias."""
    names = subprocess.run(["nm", "-C", _lib.LIB_PATH], check=True, capture_output=True, text=True).stdout
    out = {}
    for line in names.splitlines():
        m = re.search(r"__device_stub__gemm_blocks_(?:small|tile)_kernel<.*?(Small|Big)Tile<([^>]*)>, (\w+), (\w+), (\w+)>", line)
        if m:
            kind, dims, fp16, bias, grouped = m.groups()
            d = [x.strip() for x in dims.split(",")]
            wn, wm, ni, nj = (int(x) for x in d[:4])
            key = (16 * ni * wn, 16 * nj * wm, d[-1] == "true", grouped == "true")
            out.setdefault(key, set()).add((tuple(d), fp16 == "true", bias == "true"))
    assert out, "no block-scaled product in the built library"
    return out


@pytest.fixture(scope="module")
def reached():
    dense = {plan(M, N, 1, False, g)[:2] for M in ROWS for N in CHANNELS for g in CUS}
    experts = {plan(M, N, e, True, g)[:2] for M in ROWS for N in CHANNELS for e in EXPERTS for g in CUS}
    return {False: dense, True: experts}


def test_every_kernel_is_reached(compiled, reached):
    lost = [k for k in compiled if k[:2] not in reached[k[3]]]
    assert not lost, lost
    # a bias goes with the dense product only; the hint with 16 rows or fewer there
    assert not [k for k, v in compiled.items() if k[3] and any(b for _, _, b in v)]
    assert [k for k in compiled if k[2] and not k[3]] == [(32, 16, True, False)]


def test_every_form_has_its_kernels(compiled, reached):
    """Both output types of each form that a rule gives, with and without a bias for the dense product."""
    for grouped, tiles in reached.items():
        for t in tiles:
            got = {(f, b) for _, f, b in compiled.get((*t, False, grouped), ())}
            assert got == {(f, b) for f in (False, True) for b in ((False,) if grouped else (False, True))}, (t, grouped, got)
