"""What scans or rebuilds the library's kernels does so with the flags that the library is built with: another flag is other code, with other
registers (packed fp32 instructions: thousands in conv.hip with them, none without)."""
import os
import re
from concurrent.futures import ThreadPoolExecutor

import helpers as H  # noqa: F401  (puts the repo root on sys.path)
from test_isa_cpu import ROOT, _tool
from vitta_amd import build

FILES = ["conv_b3.hip", "conv.hip", "conv_sk.hip", "head.hip", "tam_branch.hip", "gemm.hip", "scores.hip"]


def test_shipped_kernels_have_no_wide_buffer_store_followed_by_a_write_of_its_data_registers():
    t = _tool()
    assert t.COMMAND[1:len(build.CFLAGS) + 1] == build.CFLAGS
    with ThreadPoolExecutor(4) as pool:
        texts = list(pool.map(t.assembly, [os.path.join(ROOT, "vitta_amd", "csrc", f) for f in FILES]))
    for f, asm in zip(FILES, texts):
        assert "s_endpgm" in asm, f
        assert t.scan(asm, 2) == [], f
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", asm), f


def test_every_recipe_for_the_library_uses_its_flags():
    flags = " ".join(build.NO_PACKED_F32)
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    for line in text.splitlines():
        if line.startswith("hipcc"):
            assert flags in line, line
    variant = open(os.path.join(ROOT, "tools", "debug", "mkvariant.sh")).read()
    assert "build.CFLAGS" in variant and "-O3" not in variant
