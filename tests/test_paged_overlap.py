"""Results of the paged cache's entry points that lie over what other rows, groups or layers still read: refused on the
host, without a GPU (every call carries an invalid argument, so it returns before any HIP call)."""
import ctypes

import pytest

import inferno_amd as ia
from test_paged_args import FAKE, cache, evict, reorder, select

OVERLAP = 3
FAR = FAKE + (1 << 16)


@pytest.mark.parametrize("off", [4, 12, -4, -12])
def test_evict_lengths(off):
    """lens_out may be cache->lens, but another row's length must not be written before it is read."""
    assert evict(cache(), lo=FAKE + off) == OVERLAP
    assert evict(cache(), lo=FAKE, n=0) == 6  # the same: the next check's
    assert evict(cache(), lo=FAKE + (16 if off > 0 else -16), n=0) == 6  # beside them


@pytest.mark.parametrize("name", ["tok", "par", "out", "fo"])
@pytest.mark.parametrize("off", [4, 28, -4, -28])
def test_select_results_over_the_inputs_in_part(name, off):
    """The results may be the inputs, but not lie over another group's: [2, 4] each."""
    apart = dict(scores=FAR, fin=FAR + 4096, eos=1)
    assert select(**apart, **{name: FAR + off}) == OVERLAP
    assert select(**apart, **{name: FAR + 4096 + off}) == OVERLAP
    assert select(**apart, **{name: FAR}, n=64) == 6
    assert select(**apart, **{name: FAR + 4096}, n=64) == 6
    assert select(**apart, **{name: FAR + (32 if off > 0 else -32)}, n=64) == 6


@pytest.mark.parametrize("what", ["table", "lens", "parents", "spare"])
@pytest.mark.parametrize("result", ["out", "spare_out"])
def test_reorder_results_over_the_inputs(what, result):
    """Tables, lengths, parents and spare pages are read by every layer's workgroups while the new ones are written."""
    size = dict(table=64, lens=16, parents=16, spare=16)[what]
    mine = dict(out=64, spare_out=16)[result]
    for off in (0, 4, size - 4, 4 - mine):
        c, kw = cache(), dict(parents=FAKE, spare=FAKE, out=FAKE + 4096, spare_out=FAKE + 8192)
        kw[result] = FAR + off
        if what in ("table", "lens"):
            c = cache(**{what: FAR})
        else:
            kw[what] = FAR
        assert reorder(c, **kw) == OVERLAP
    assert reorder(cache(), out=FAR, spare_out=FAR + 60) == OVERLAP  # one over the other
    assert reorder(cache(), out=FAR, spare_out=FAR - 12) == OVERLAP
