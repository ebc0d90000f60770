"""The CPU baseline without the reference's library: the oracle's functions."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_port_with_heads_wider_than_the_model():
    """The attention's output has heads x head_dim values, more than the
    model's width here; a process of its own, so that a write past a buffer
    ends it and not the tests."""
    code = """
from oracle import cpu_baseline
cpu_baseline._setup_ref = lambda: None
for _ in range(3):
    r = cpu_baseline.measure(D=64, H=64, KVH=8, hd=64, E=4, K=2, inter=64, V=128, gs=32, ctx=64, window=16)
assert r["kind"] == "port" and r["tok_s"] > 0
print("done")
"""
    p = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and "done" in p.stdout, p.stderr[-500:]
