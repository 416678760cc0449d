"""How the library uses HIP streams: what its sources may not do."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "genozip_amd", "csrc")


def sources():
    for f in sorted(os.listdir(CSRC)):
        yield f, open(os.path.join(CSRC, f)).read()


def test_nothing_runs_on_the_null_stream():
    """a copy or a fill on the null stream waits for whatever its hardware queue holds - another handle's long chain included: every one names
    the handle's own stream (hipMemcpyFromSymbol / ToSymbol: debug builds' counters only)"""
    for f, text in sources():
        for m in re.finditer(r"\b(hipMemcpy|hipMemset|hipMemcpyDtoH|hipMemcpyHtoD|hipDeviceSynchronize)\s*\(", text):
            raise AssertionError("%s: %s" % (f, text[max(0, m.start() - 60):m.end() + 60]))
        for m in re.finditer(r"hipLaunchKernelGGL\s*\(([^;]*?)\);", text, re.S):
            args = re.sub(r"\([^()]*(\([^()]*\)[^()]*)*\)", "()", m.group(1)).split(",")
            assert len(args) > 4 and args[4].strip() not in ("0", "NULL", "nullptr"), (f, m.group(0)[:120])
