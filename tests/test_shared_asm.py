"""Static check of the gfx950 code of attention over shared pages (hipcc -S here, no GPU). Its tiles go from memory to LDS by
themselves, into places that other waves have written before (zeros beyond a narrow head's width, a segment's last sums): a wave
sends for a tile only behind a barrier that all waves reach with their own LDS writes done. So on no path from an LDS write to a
tile's load may a barrier be missing.

A data-flow pass over the basic blocks of each kernel: whether something has been written since the last barrier; at a join, if
it has on either side."""
import os
import re
import shutil
import subprocess

import pytest

from test_wide_gemm_asm import blocks, parse

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "comfy-quant-bench_amd", "csrc", "mq_attn_shared.hip")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
KERNEL = re.compile(r"^(_ZN2mq12_GLOBAL__N_118attn_shared_kernel\w+):")


def unguarded(ins):
    """Indices of tiles' loads that an LDS write reaches without a barrier between them, and the number of such loads."""
    bl, succ = blocks(ins)
    dirty, todo, bad, loads = [False] * len(bl), list(range(len(bl))), set(), set()
    while todo:
        k = todo.pop()
        d = dirty[k]
        for i in bl[k]:
            kind, op, _, _ = ins[i]
            if kind != "op":
                continue
            if op.startswith("ds_write") or op.startswith("ds_store"):
                d = True
            elif op == "s_barrier":
                d = False
            elif op == "global_load_lds_dwordx4":
                loads.add(i)
                if d:
                    bad.add(i)
        for n in succ[k]:
            if d and not dirty[n]:
                dirty[n] = True
                todo.append(n)
    return bad, len(loads)


def test_the_check_itself():
    code = ["ds_write_b128 v0, v[4:7]", "s_cbranch_vccnz .LBB0_2", "s_barrier", ".LBB0_2:", "global_load_lds_dwordx4 v[2:3], off", "s_endpgm"]
    assert unguarded(parse(code)) == ({4}, 1)           # past the barrier by the branch
    assert unguarded(parse([c for c in code if "cbranch" not in c])) == (set(), 1)
    loop = [".LBB0_1:", "global_load_lds_dwordx4 v[2:3], off", "ds_write_b128 v0, v[4:7]", "s_cbranch_vccnz .LBB0_1", "s_endpgm"]
    assert unguarded(parse(loop)) == ({1}, 1)


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
def test_tiles_are_sent_for_behind_a_barrier(tmp_path):
    import build

    out = str(tmp_path / "shared.s")
    subprocess.run([HIPCC, *build.flags(), "--cuda-device-only", "-S", SRC, "-o", out], check=True, capture_output=True)
    kernels, name = {}, None
    with open(out) as f:
        for line in f:
            m = KERNEL.match(line)
            if m:
                name = m.group(1)
                kernels[name] = []
            elif line.startswith(".Lfunc_end"):
                name = None
            elif name:
                kernels[name].append(line.rstrip("\n"))
    assert len(kernels) == 12
    for name, body in kernels.items():
        bad, loads = unguarded(parse(body))
        assert loads > 0 and not bad, (name, sorted(bad))
