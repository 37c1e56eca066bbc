"""Figures that bench.py takes from a stored capture belong to the kernel sources that are here."""
import benchlib


def test_dram_traffic_is_of_this_kernel_source():
    """Otherwise the benchmark's roofline loses its traffic (and its physical fraction): keep the hashed files, or take the
    capture again and store it with the new hash."""
    assert benchlib.spmm_kernel_source_hash() == benchlib.SPMM_DRAM_TRAFFIC["kernel_source"]
    for width in (32, 128, 256):
        assert benchlib.spmm_dram_traffic(22, width) > 0
