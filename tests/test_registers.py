"""Registers of the built kernels, from the metadata of the library's gfx950 code objects (CPU: nothing runs)."""
import re
import subprocess

from test_wait_states import library_code_objects

READELF = '/opt/rocm/llvm/bin/llvm-readelf'


def _kernels():
    """{kernel: vector registers that it spills}"""
    found = {}
    for code in library_code_objects():
        notes = subprocess.run([READELF, '--notes', '-'], input=code, capture_output=True, check=True).stdout.decode()
        for kernel in re.split(r'\n\s+- \.agpr_count:', notes)[1:]:
            found[re.search(r'\.name:\s+(\S+)', kernel).group(1)] = int(re.search(r'\.vgpr_spill_count:\s+(\d+)', kernel).group(1))
    return found


def test_the_normalisation_spills_at_1024_lanes_only():
    """A streaming kernel whose registers spill moves them through memory beside its rows."""
    norms = {name: spilled for name, spilled in _kernels().items() if 'layer_norm' in name and 'gated' not in name}
    assert len(norms) > 100
    spilling = [name for name, spilled in norms.items() if spilled and 'Li1024E' not in name]
    assert not spilling, spilling
