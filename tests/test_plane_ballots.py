"""The ballots plane_kernel (bgt_amd/csrc/scan_plane.hip) hands out, at every width it is compiled for: lane l of a wave keeps the
ballot of column l and one bounded store per wave and row takes them to the bit planes.  Bit-exact against the oracle
(reference pbwt.c:129-170, bgt.c:735-757): genotypes come from the planes themselves, counts from their popcounts."""
import numpy as np
import pytest

import orc
import scenarios
from test_hip_parity import oracle_scan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import bgt_amd
    assert bgt_amd.device_count() > 0, bgt_amd.last_error()
    return bgt_amd


@pytest.fixture(scope="module")
def narrow():
    """m = 20,000 haplotypes: eight waves a workgroup."""
    return orc.encode_pbf(scenarios.ld_matrix(np.random.default_rng(31), 45, 20000, n_founders=7, switch=0.1), 2, 4)


@pytest.fixture(scope="module")
def wide():
    """m = 150,000 haplotypes: twelve waves a workgroup (three workgroups of eight waves do not fit a CU's LDS)."""
    return orc.encode_pbf(scenarios.ld_matrix(np.random.default_rng(32), 11, 150000, n_founders=7, switch=0.02), 2, 3)


def check(hip, data, n_samples, n_sel, threads, cpt):
    hip.force_kernels(hip.hip.FORCE_PLANE_SPLIT)
    pbf = hip.HipPbf.from_bytes(data)
    rd = hip.HipReader(pbf)
    smp = np.sort(np.random.default_rng(n_sel).choice(n_samples, n_sel, replace=False))
    cols = np.stack([2 * smp, 2 * smp + 1], 1).reshape(-1).astype(np.int32)
    rd.select(cols)
    rows = orc.Pbf(data).n
    oc, ogt = oracle_scan(data, 0, rows, cols=cols)
    # the whole file, ranges that begin and end inside a checkpoint block, one row (the last: a block may hold a single one)
    for a, b in ((0, rows), (1, rows - 1), (rows // 2, rows // 2 + 1), (rows - 1, rows)):
        c, g = rd.scan(a, b, want_gt=True)
        geo = rd.geometry()
        assert rd.path()["plane_split"] and (geo["threads"], geo["cols_per_thread"]) == (threads, cpt), (rd.path(), geo)
        assert np.array_equal(c, oc[a:b]) and np.array_equal(g, ogt[a:b]), (a, b, geo)
    assert np.array_equal(rd.scan(0, rows), oc)                          # counts alone: the planes stay in the reader's buffers
    rd.close()
    pbf.close()


# n_sel samples take ceil(n_sel / 32) ballots: the last wave that has any is partly filled, waves behind it have none
@pytest.mark.parametrize("n_sel,cpt", [(33, 4), (32 * 57 + 5, 8), (32 * 81 + 1, 12), (32 * 143 + 7, 20), (32 * 250 + 9, 32), (8192, 32)])
def test_every_width_of_eight_waves(hip, narrow, n_sel, cpt):
    check(hip, narrow, 10000, n_sel, 512, cpt)


@pytest.mark.parametrize("n_sel,cpt", [(32 * 41 + 3, 4), (32 * 85 + 1, 8), (32 * 133 + 30, 12), (32 * 178 + 2, 16), (32 * 200 + 31, 20), (7680, 20)])
def test_every_width_of_twelve_waves(hip, wide, n_sel, cpt):
    check(hip, wide, 75000, n_sel, 768, cpt)
