"""How the library uses HIP streams: what its sources may not do (CPU), the long leaves' launches against the oracle (CPU stand-in), and a
process whose streams all share ONE hardware queue (GPU)."""
import os
import re
import subprocess
import sys

import pytest

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


def test_streams_have_one_priority_and_kernels_wait_for_nobody():
    """the runtime maps streams onto a few hardware queues: a kernel that waits on the device for one of another stream may sit in front of it in
    the same queue and then never ends, and streams of different priorities are no way out. No stream asks for a priority, no kernel sleeps in a loop"""
    for f, text in sources():
        for word in ("CreateWithPriority", "StreamPriorityRange", "__builtin_amdgcn_s_sleep", "s_sleep "):
            assert word not in text, (f, word)
    for d in ("genozip_amd", "tools", "."):
        for f in os.listdir(os.path.join(ROOT, d)):
            if f.endswith(".py"):
                text = open(os.path.join(ROOT, d, f)).read()
                assert not re.search(r"Stream\([^)]*priority|is_high_priority_stream", text), f


@pytest.mark.parametrize("n", [65537, 131072, 200001, 720001])
def test_long_leaf_in_position_chunks(emul_engine, oracle, n):
    """leaves of 2, 2, 4 and 11 position chunks: the chain's state goes from launch to launch through the checkpoint the two share, a launch takes
    one chunk or several, the `low` kernels follow launch by launch"""
    from genozip_amd import synth
    data = synth.quality_diverse(11, (n + 149) // 150).tobytes()[:n]
    assert len(data) == n
    short = synth.quality_diverse(12, 40).tobytes()                       # (and a short leaf beside it, in one piece)
    got = emul_engine.compress_many([(16, data), (16, short)])
    assert got[0] == oracle.codec_compress(16, data) and got[1] == oracle.codec_compress(16, short)


ONE_QUEUE = """
import sys
sys.path[:0] = [%r, %r, %r]
import parity, pyoracle
from genozip_amd import synth
from genozip_amd.codec import Engine
E, O = Engine(device=0), pyoracle.Oracle()
data = synth.quality_diverse(7, 6000).tobytes()                            # 900 KB: 14 position chunks, the chain in several launches
items = [(c, data) for c in (16, 17, 18, 19, 6, 7)] + [(16, data[:3000])]
for rep in range(2):
    got = E.compress_many(items)
    for (c, d), g in zip(items, got):
        assert g == O.codec_compress(c, d), c
    print("codecs", rep, flush=True)
parity.fastq_zip(E, O, 2500, n_calls=2)                                    # QUAL coded ahead on the second handle
assert E.L.gz_chain_fallbacks(E.h) == 0
E.close()
print("ONE QUEUE OK", flush=True)
"""


@pytest.mark.gpu
def test_one_hardware_queue():
    """a process that has ONE hardware queue for all its streams: everything the library queues on its streams still runs, in the order it was
    queued - the oracle's bytes, no batch run twice (a kernel that waited on the device for another stream's would stand in its way for ever)"""
    code = ONE_QUEUE % (ROOT, os.path.join(ROOT, "oracle"), os.path.join(ROOT, "tests"))
    p = subprocess.run([sys.executable, "-u", "-c", code], env=dict(os.environ, GPU_MAX_HW_QUEUES="1"), stdout=subprocess.PIPE, stderr=subprocess.PIPE, timeout=100)
    assert p.returncode == 0 and b"ONE QUEUE OK" in p.stdout, p.stdout.decode()[-1000:] + p.stderr.decode()[-3000:]


@pytest.mark.gpu
def test_handles_of_several_threads(oracle):
    """six host threads, a handle each, long and short leaves at the same time: more streams than hardware queues, and chains that would ask for
    more whole compute units than the process gives away - the oracle's bytes on every handle, round after round"""
    import threading
    from genozip_amd import synth
    from genozip_amd.codec import Engine
    data = [synth.quality_diverse(40 + t, 1500 + 300 * t).tobytes() for t in range(6)]     # 225 - 450 KB: 4 - 7 position chunks
    want = [[oracle.codec_compress(c, d) for c in (16, 17)] for d in data]
    bad = []

    def work(t):
        E = Engine(device=0)
        try:
            for rep in range(3):
                got = E.compress_many([(16, data[t])] * 9 + [(17, data[t])] * 9)
                if got != [want[t][0]] * 9 + [want[t][1]] * 9:
                    bad.append((t, rep))
            if E.L.gz_chain_fallbacks(E.h):
                bad.append((t, "a batch ran twice"))
        except Exception as e:                                            # (a thread's exception would go unseen)
            bad.append((t, repr(e)))
        finally:
            E.close()
    ts = [threading.Thread(target=work, args=(t,)) for t in range(6)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad, bad
