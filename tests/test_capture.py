"""No operator that a caller may capture into a graph records a memset (such nodes have left wrong values on replays after the first)."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "unet_amd" / "csrc"


def test_only_the_network_engine_enqueues_memsets():
    found = {f.name for f in CSRC.glob("*.h*") if re.search(r"hip(Memset|MemsetD)\w*\s*\(", f.read_text())}
    assert found <= {"engine.hip"}, found
