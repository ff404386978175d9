"""The checker's own computeSortedMarkers and computeAlignmentTable, which bench.py's CPU leg runs where the reference itself is not
built: the table against a python restatement, the aligner's results with and without the sorted markers."""
import numpy as np
import pytest

from shasta_amd import abi
from tests import host_support, support, table_checks


@pytest.mark.parametrize("read_count, count", [(1, 0), (2, 1), (37, 400), (211, 3000)])
def test_alignment_table(oracle_lib, read_count, count):
    rows = table_checks.random_alignment_data(np.random.default_rng(11), read_count, count)
    toc, values, seconds = oracle_lib.alignment_table(rows, read_count)
    toc_expected, values_expected = host_support.alignment_table_expected(read_count, rows)
    assert np.array_equal(toc, toc_expected) and np.array_equal(values, values_expected) and seconds > 0


def test_alignment_table_refuses_a_read_that_does_not_exist(oracle_lib):
    rows = table_checks.random_alignment_data(np.random.default_rng(12), 10, 20)
    with pytest.raises(RuntimeError):
        oracle_lib.alignment_table(rows, 5)


def test_sorted_markers_change_no_alignment(oracle_lib):
    toc, kmer, data7 = support.small_marker_set(n_reads=60, genome_markers=4000, seed=7)
    candidates = oracle_lib.lowhash0(toc, data7, None, abi.default_lowhash0_params(minBucketSize=2, maxBucketSize=30)).candidates[:120]
    assert len(candidates) > 20
    options = abi.default_align4_options(minAlignedMarkerCount=40)
    plain = oracle_lib.align4_batch(toc, data7, candidates, options, threads=2)
    assert len(plain.alignment_data) > 0
    assert oracle_lib.compute_sorted_markers(toc, data7, threads=3) > 0
    try:
        support.same_align(oracle_lib.align4_batch(toc, data7, candidates, options, threads=2), plain)
        other = data7.copy()                                       # (other markers: the sorted ones are not theirs)
        support.same_align(oracle_lib.align4_batch(toc, other, candidates, options, threads=2), plain)
    finally:
        oracle_lib.drop_sorted_markers()
    support.same_align(oracle_lib.align4_batch(toc, data7, candidates, options, threads=2), plain)
