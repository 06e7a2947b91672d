"""Every translation unit whose kernels can give up on a wait has a status word: the library's status call reads all of them and
the reset clears all of them."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "batchlas_b200", "csrc")


def test_every_status_word_is_read_and_cleared():
    defined = []
    for path in glob.glob(os.path.join(CSRC, "*.cu")):
        if os.path.basename(path) != "status.cu":
            defined += re.findall(r"^int (\w+_device_status(?:_clear)?)\([^)]*\) \{", open(path).read(), re.M)
    words = {n for n in defined if not n.endswith("_clear")}
    assert len(words) >= 8 and {w + "_clear" for w in words} == set(defined) - words
    aggregate = open(os.path.join(CSRC, "status.cu")).read()
    for name in defined:      # declared once and used
        assert len(re.findall(rf"\b{name}\b", aggregate)) >= 2, name


def test_units_with_bounded_waits_have_a_word():
    for path in glob.glob(os.path.join(CSRC, "*.cu")):
        text = open(path).read()
        if re.search(r"\bmbar_wait(_limit)?\(|launch_umma<", text) and os.path.basename(path) not in ("status.cu", "peak.cu"):
            assert re.search(r"_device_status\(int\* out\) \{ return read_device_status_word\(out\); \}", text), path
