"""Arguments that the C entry points of the sequence layers have to survive, whatever they hold."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROBE = """
import sys
sys.path.insert(0, {root!r})
import ctypes
import dm_amd_bootstrap
from dm_amd.runtime import hip
good = dict(Tq=1000, Tk=1000, B=2, H=8, Hk=2, dh=64)
floats = lambda **k: hip.lib().ddpm_packed_attn_dkv_floats(ctypes.byref(hip.PackedAttnDesc(**dict(good, **k))))
assert floats() > 0
for bad in (dict(B=-2, Tk=0), dict(B=-9, Tk=1000), dict(B=-1), dict(Tk=-1), dict(Tq=-1), dict(H=0), dict(Hk=0), dict(Hk=-2), dict(H=-8), dict(B=2 ** 31 - 1, Tk=2 ** 31 - 1),
            dict(B=2 ** 31 - 2, Tk=0)):
    assert floats(**bad) == 0, bad
assert hip.lib().ddpm_packed_attn_dkv_floats(None) == 0
print("survived")
"""


def test_workspace_size_of_wrong_descriptors():
    """no workspace for what the backward pass refuses; a count of no workgroups was divided by (a process of its own: that ends it)"""
    r = subprocess.run([sys.executable, "-c", PROBE.format(root=ROOT)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "survived" in r.stdout, (r.returncode, r.stderr[-500:])
