"""Rules that the library's sources keep where no run would show the fault."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onegpu-csharp_b200", "csrc")


def test_memory_is_cleared_for_every_stream():
    """cudaMemset returns before it is done, in a stream that the devices' non-blocking streams do not wait for: counters
    are cleared by device_zeros, which waits."""
    calls = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = re.sub(r"//[^\n]*", "", open(path, encoding="utf-8").read())
        calls += [(os.path.basename(path), text[m.start():].split(";")[1].strip()) for m in re.finditer(r"\bcudaMemset\(", text)]
    assert len(calls) == 1 and "cudaStreamSynchronize(cudaStreamLegacy)" in calls[0][1], calls
