"""Buffers that a caller may give as input and output at once are not declared free of aliases to the compiler, read off
its own intermediate code; no GPU."""
import os
import re
import subprocess

import pytest

from karume_amd import build


@pytest.mark.parametrize("source,kernel,count,one_buffer", [
    ("rotary.hip", "rope_pieces_kernel", 4, (0, 4)), ("rotary.hip", "rope_rows_kernel", 2, (0, 4)),
    ("kv4_cache.hip", "kv4_append_kernel", 12, (6, 7))])
def test_in_place_buffers_may_alias(tmp_path, source, kernel, count, one_buffer):
    if not os.path.exists(build.HIPCC):
        pytest.skip("no compiler")
    out = tmp_path / "device.ll"
    subprocess.run([build.HIPCC, *build.FLAGS, "--offload-device-only", "-emit-llvm", "-S", os.path.join(build.CSRC, source),
                    "-o", str(out)], check=True, capture_output=True)
    found = re.findall(rf"^define [^@]*amdgpu_kernel void @\w*{kernel}\w*\((.*)\) .*\{{$", out.read_text(), re.MULTILINE)
    assert len(found) == count
    for arguments in found:
        parts = re.split(r", (?=ptr|i\d|float|%|\{)", arguments)
        for at in one_buffer:
            assert parts[at].startswith("ptr") and "noalias" not in parts[at], parts[at]
        assert any("noalias" in p for p in parts)   # (the other buffers are: the attribute is found where it stands)
