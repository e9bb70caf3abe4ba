"""What the compiler makes of the device code, where a result hangs on it: compiled here for gfx950,
nothing is run."""
import os
import re
import subprocess

import pytest

from tabby_amd import build


def _assembly(tmp_path, source):
    """Kernel name -> its instructions, one to an entry."""
    try:
        hipcc = build._hipcc()
    except RuntimeError:
        pytest.skip("hipcc is needed to look at the compiled code")
    out = os.path.join(tmp_path, "device.s")
    flags = [f for f in build.HIPCC_FLAGS if f != "-shared"]
    r = subprocess.run([hipcc, *flags, "--cuda-device-only", "-S", "-o", out, os.path.join(build.CSRC, source)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    with open(out) as f:
        text = f.read()
    kernels = {}
    for name in re.findall(r"^\s*\.amdhsa_kernel (\S+)", text, re.M):
        body = text.split(f"\n{name}:", 1)[1].split(f".section\t.rodata", 1)[0]
        kernels[name] = [line.split(";")[0].split() for line in body.splitlines() if re.match(r"\s+[a-z]", line)]
    assert kernels
    return kernels


def test_the_waves_of_a_selection_exchange_their_lists_in_order(tmp_path):
    # A wave lists entries in LDS and then publishes their count; another that sees the count reads the entries. LDS
    # keeps the order of a wave's own accesses (ds_); flat ones reach it another way, which has no order with those.
    rows = {n: code for n, code in _assembly(tmp_path, "beam_select.hip").items() if "beam_row_kernel" in n}
    assert len(rows) == 18
    for name, code in rows.items():
        assert any(i[0] == "ds_write_b64" for i in code), name
        assert not [i for i in code if i[0].startswith("flat_")], name
