"""CPU: a kernel's dynamic shared-memory limit is never set to the size of one launch: a second thread's smaller launch would
lower it between another thread's setting and its launch, which then fails.  Limits are raised once (SmemLimit), or under a
lock and never lowered."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "flashsvd_b200" / "csrc"


def test_limits_are_raised_once_or_under_a_lock():
    found = 0
    for path in sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh"), *CSRC.glob("*.h")]):
        text = path.read_text()
        for m in re.finditer(r"cudaFuncSetAttribute\(", text):
            found += 1
            before = text[max(0, m.start() - 600):m.start()]
            at_creation = "g_smem_optin - 1024" in text[m.start():m.start() + 140]   # the same number at every call
            assert path.name == "fsvd_smem.h" or "lock_guard" in before or at_creation, f"{path.name}: {text[m.start():m.start() + 120]}"
    assert found >= 2


def test_the_limit_of_a_launch_of_any_size_is_the_device_s():
    for name in ("fsvd_kv8.cu", "fsvd_sample.cu"):
        text = (CSRC / name).read_text()
        assert "SmemLimit" in text and re.search(r"\.raise\((KERNEL|kernels\[which\])\)", text), name
