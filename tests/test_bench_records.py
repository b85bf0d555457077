"""CPU test of the figures that bench.py quotes from recorded captures."""
import importlib.util
import os

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_dram_traffic_of_the_main_kernel_is_quoted():
    """The record of the main decode kernel was taken on the sources as they are: a change to them asks for a new capture,
    a change to other kernels must not touch the files its digest covers."""
    spec = importlib.util.spec_from_file_location("fa_bench", os.path.join(ROOT, "bench.py"))
    bench = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(bench)
    traffic, source = bench.recorded_traffic(bench.main_kernel_name(3), "profile_small")
    assert traffic is not None, source
    for name in ("abi.cu", "cache_ops.cu", "rope_append.cu", "paged_attn.cu", "sample.cu", "serving.cuh"):
        assert name not in bench.KERNEL_SOURCES
