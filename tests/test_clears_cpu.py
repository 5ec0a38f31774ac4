"""Device memory is cleared where the runtime's stream is ordered with it."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ammon_b200", "csrc")


def test_no_clear_on_the_default_stream():
    """A plain cudaMemset is ordered with neither the runtime's stream nor the peers that are about
    to write; clear_device is."""
    found = []
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            code = re.sub(r"//[^\n]*", "", f.read())
        found += [name] * len(re.findall(r"\bcudaMemset\s*\(", code))
    assert not found
