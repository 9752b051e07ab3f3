"""CPU checks around the sequence-cache kernels: the backend's error word, and loads of kernels that are placed early."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sam3.cpp_b200", "csrc")


def _sources():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*")) + glob.glob(os.path.join(CSRC, "*.h"))):
        with open(path) as f:
            yield os.path.basename(path), re.sub(r"//[^\n]*", "", f.read())


def test_bits_of_wrong_data_mean_nothing_else():
    """The error word: a bit that names wrong data (an index, a page, a batch) is never also a kernel's timeout."""
    data, waits = {}, {}
    for name, text in _sources():
        for what, bit in re.findall(r"\b(\w*E[Rr][Rr]_?\w*)\s*=\s*1\s*<<\s*(\d+)", text):
            (data if what.startswith("kErr") or what.startswith("kOpErr") else waits).setdefault(int(bit), []).append((name, what))
    assert not set(data) & set(waits), {b: data[b] + waits[b] for b in set(data) & set(waits)}
    assert len(data) == sum(len(v) for v in data.values()) == 3 and sum(len(v) for v in waits.values()) > 20


def test_kernels_placed_early_read_through_coherent_loads():
    """Kernels that wait_for_stream() are on the GPU before the kernel in front has written its results: read-only loads
    ask for memory that nothing writes from a kernel's start to its end."""
    files = [(name, text) for name, text in _sources() if "wait_for_stream()" in text]
    assert len(files) >= 4
    for name, text in files:
        assert "__ldg" not in text and "global.nc" not in text, name
