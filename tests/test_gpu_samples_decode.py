"""The C++ sample driver's decode-step commands: their known-answer checks pass and their lines parse."""
import re
import subprocess
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

BIN = Path(__file__).resolve().parent.parent / "optimized_rocwmma_samples_b200" / "b2sq_samples"
LINE = re.compile(r"^\[(?P<tag>[\w -]+)\] .*?\s+(?P<ms>[0-9.e+-]+) ms\s+(?P<val>[0-9.e+-]+) GB/s$")


@pytest.mark.parametrize("command,want", [("kv4", {"KV4-Append": 2, "KV4-Attention": 2, "KV4-Evict": 2}),
                                          ("moe_layer", {"MoE-Layer": 2})])
def test_decode_samples(cuda_device, command, want):
    assert BIN.exists(), "build the package first (python -m optimized_rocwmma_samples_b200.build)"
    res = subprocess.run([str(BIN), command], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    tags = [m["tag"] for m in map(LINE.match, res.stdout.splitlines()) if m]
    assert {t: tags.count(t) for t in want} == want and "FAILED" not in res.stdout
