"""What the head's products read, on the CPU: the library's host code makes its launches into a recorder, and every load of
every operand has to lie inside the operand, and the operand inside the call's buffers."""
import json
import os
import random
import shutil
import subprocess
import sys

import pytest

from cudnntest_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def recorder(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    so = str(tmp_path_factory.mktemp("recorder") / "launch_recorder.so")
    subprocess.check_call([cxx, "-O1", "-std=c++17", "-shared", "-fPIC", "-o", so, os.path.join(HERE, "host", "launch_recorder.cpp")])
    return so


def complaints(recorder, calls):
    r = subprocess.run([sys.executable, os.path.join(HERE, "launch_reach.py"), recorder, _lib.LIB_PATH], input=json.dumps(calls),
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    return json.loads(r.stdout)


def test_second_pass_over_two_values_stays_in_its_row(recorder):
    """dw of 256-wide tiles where half a row of dl is an odd multiple of 128 wide: the second pass starts half a row in."""
    sizes = [(174, 8327, 1091), (208, 7800, 1373), (124, 6000, 1392), (152, 9592, 1323), (256, 8192, 1024 + 128), (200, 16, 140000)]
    assert complaints(recorder, [("backward", dt, *s) for s in sizes for dt in (1, 2)]) == []


def test_reads_of_small_and_large_problems(recorder):
    """Sizes over the whole range, odd ones and pieces of the vocabulary among them, in every type and direction."""
    r = random.Random(5)
    log = lambda lo, hi: max(lo, min(hi, int(lo * (hi / lo) ** r.random())))
    calls = [(k, dt, *s) for k in ("forward", "backward") for dt in (0, 1, 2)
             for s in ((1, 1, 1), (1, 3, 2), (65, 129, 257), (250, 4096, 1000), (777, 1003, 10007), (2048, 2048, 32000), (1030, 24, 70000))]
    for _ in range(150):
        calls.append((r.choice(("forward", "backward")), r.randrange(3), log(1, 6000), log(1, 10000), log(1, 150000)))
        calls.append(("linear", r.randrange(3), log(1, 6000), log(1, 9000), log(1, 26000)))
    assert complaints(recorder, calls) == []
