"""The block attention's main loop as the compiler lays it out.  Its waits count
loads: a wave that waits until kLoads are left must have issued exactly kLoads
vector loads since the tile it waits for, and no wait of the compiler's own may
empty the queue.  The device code is compiled to assembly (no GPU needed)."""
from __future__ import annotations

import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "comfyui-turing-utils_amd", "csrc")
# 16-byte loads of 64 keys' K and V^T by 256 lanes, and a tile's scale
LOADS = {128: 64 * 128 * 3 // 4096 + 1, 64: 64 * 64 * 3 // 4096 + 1}


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{(head_dim, causal, split): [instructions of each basic block]}"""
    flags = re.search(r"^HIPFLAGS = ((?:.*\\\n)*.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M).group(1)
    out = tmp_path_factory.mktemp("asm") / "block_attn.s"
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *flags.replace("\\\n", " ").split(), "--offload-device-only", "-S",
                    "block_attn.hip", "-o", str(out)], cwd=CSRC, check=True, timeout=300)
    text = out.read_text()
    found = {}
    for m in re.finditer(r"^_ZN2tu12_GLOBAL__N_117block_attn_kernelILi(\d+)ELb([01])ELb([01])E\S*:", text, re.M):
        body = text[m.end():text.index(".Lfunc_end", m.end())]
        found[tuple(map(int, m.groups()))] = [
            [ln.strip().split(";")[0] for ln in b.splitlines() if re.match(r"\t[a-z]", ln)]
            for b in re.split(r"^\.LBB[0-9_]+:", body, flags=re.M)]
    assert len(found) == 8
    return found


@pytest.mark.parametrize("d,causal,split", [(d, c, s) for d in (64, 128) for c in (0, 1) for s in (0, 1)])
def test_main_loop_counts_its_loads(kernels, d, causal, split):
    mfmas = 52 if d == 128 else 28
    blocks = kernels[d, causal, split]
    starts = [n for n, b in enumerate(blocks) if sum(i.startswith("v_mfma") for i in b) == mfmas]
    assert len(starts) == 1, starts
    # to the barrier that ends an interval (a rescaling of the sums is a branch in between)
    last = next(n for n in range(starts[0], len(blocks)) if any("s_barrier" in i for i in blocks[n]))
    loop = [i for b in blocks[starts[0]:last + 1] for i in b]
    loop = loop[:next(n for n, i in enumerate(loop) if "s_barrier" in i)]
    vector = [i for i in loop if re.match(r"(buffer|global|flat|scratch)_", i)]
    assert len(vector) == LOADS[d] and all(i.startswith("buffer_load") for i in vector), vector
    assert sum(i.rstrip().endswith("lds") for i in vector) == LOADS[d] - 1, vector
    assert not any(i.startswith("s_load") for i in loop)
    waits = [int(n) for i in loop if i.startswith("s_waitcnt") for n in re.findall(r"vmcnt\((\d+)\)", i)]
    assert waits == [LOADS[d]], waits
