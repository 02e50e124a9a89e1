"""What the compiler makes of the paged attention's registers, from the assembly
of this package's own sources (hipcc cross-compiles without a GPU)."""

import concurrent.futures as cf
import os
import subprocess

import pytest

from mtplx_amd import build

SOURCES = ["paged_attn.hip", "paged_attn_window.hip", "paged_attn_shared.hip"]


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no hipcc")
def test_no_spilled_tuple_is_split(tmp_path):
    """A tuple of registers of which three were spilled to memory and one was
    kept in an accumulator register came back without the fourth where a matrix
    instruction reloaded it into other accumulator registers (a chunk kernel at
    head dim 256: wrong scores). The compiler marks such halves."""
    def assembly(src):
        out = tmp_path / (src + ".s")
        subprocess.run([build.HIPCC, *build.flags_for(src), "--cuda-device-only", "-S",
                        os.path.join(build.CSRC, src), "-o", str(out)], check=True, capture_output=True)
        return out.read_text()

    with cf.ThreadPoolExecutor(len(SOURCES)) as pool:
        for src, text in zip(SOURCES, pool.map(assembly, SOURCES)):
            assert "mfma" in text and "Reload Reuse" not in text, src
