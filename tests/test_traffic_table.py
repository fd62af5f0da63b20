"""The benchmark's DRAM traffic comes from profiler captures, each tied to the sources that it was taken from: an edit
of those files takes the figure away until the capture is renewed."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_captures_are_of_these_sources():
    sys.path.insert(0, ROOT)
    import bench
    for kernel in ("run_kernel", "tbe_forward_kernel"):
        traffic, source = bench.measured_traffic(kernel, "target", 1245184)
        assert traffic is not None and traffic > 0, "%s: %s" % (kernel, source)
