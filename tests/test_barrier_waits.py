"""The assembly hipcc writes for the tensor and row-table kernels: on every path to a workgroup
barrier the wave has waited for its LDS stores.  hipcc 7.2 leaves that wait out in front of a
barrier at a loop's head that the back edge reaches with stores under way.  The training operators'
kernels place their plain barriers behind the stores (a vote such as __syncthreads_or may stand at a
head: it has an LDS store and a barrier behind it of its own); the assembly of every source is
searched for barriers without the wait."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vings_mono_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["-O3", "-std=c++17", "--offload-arch=gfx950", "-fno-slp-vectorize", "-Xclang", "-target-feature", "-Xclang",
         "-packed-fp32-ops", "-S", "--cuda-device-only"]


def barriers_without_wait(asm):
    """[(kernel, block)] of barriers that some path reaches with an LDS access not waited for."""
    found = []
    for kernel in re.finditer(r"^(_Z\w+):.*?\n(.*?)\.Lfunc_end", asm, re.S | re.M):
        blocks, order, cur = {"entry": []}, ["entry"], "entry"
        for line in kernel.group(2).split("\n"):
            line = line.split(";")[0].strip()
            label = re.match(r"(\.LBB\w+):", line)
            if label:
                cur = label.group(1)
                blocks[cur] = []
                order.append(cur)
            elif line and not line.startswith("."):
                blocks[cur].append(line)
        pending, changed = dict.fromkeys(order, False), True
        while changed:
            changed = False
            for k, block in enumerate(order):
                under_way, falls_through = pending[block], True
                for text in blocks[block]:
                    op = text.split()[0]
                    if op.startswith("ds_") and not op.startswith(("ds_bpermute", "ds_permute", "ds_swizzle")):
                        under_way = True
                    elif op == "s_waitcnt" and re.search(r"lgkmcnt\(0\)|s_waitcnt\s+0$", text):
                        under_way = False
                    elif op == "s_barrier" and under_way and (kernel.group(1), block) not in found:
                        found.append((kernel.group(1), block))
                    targets = [text.split()[1]] if op.startswith(("s_cbranch", "s_branch")) else []
                    falls_through = op not in ("s_branch", "s_endpgm")
                    for target in targets:
                        if under_way and not pending.get(target, True):
                            pending[target] = changed = True
                    if not falls_through:
                        break
                if falls_through and k + 1 < len(order) and under_way and not pending[order[k + 1]]:
                    pending[order[k + 1]] = changed = True
    return found


def test_the_check_sees_a_missing_wait():
    loop = "_Zk:\n\tds_write_b32 v0, v1\n\ts_waitcnt lgkmcnt(0)\n.LBB0_1:\n\ts_barrier\n\tds_write_b32 v0, v1\n%s" \
           "\ts_cbranch_scc1 .LBB0_1\n\ts_endpgm\n.Lfunc_end0:\n"
    assert barriers_without_wait(loop % "") == [("_Zk", ".LBB0_1")]
    assert barriers_without_wait(loop % "\ts_waitcnt lgkmcnt(0)\n") == []


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason="no hipcc")
@pytest.mark.parametrize("source", ["row_table", "grad_norm", "sparse_adam"])
def test_every_barrier_waits_for_lds_stores(source, tmp_path):
    out = tmp_path / "kernels.s"
    strict = ["-ffp-contract=off"] if source == "sparse_adam" else []
    subprocess.run([HIPCC, *FLAGS, *strict, "-o", str(out), os.path.join(CSRC, source + ".hip")], check=True,
                   stderr=subprocess.DEVNULL)
    asm = out.read_text()
    assert asm.count("s_barrier") > 0
    assert barriers_without_wait(asm) == []


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason="no hipcc")
@pytest.mark.parametrize("source", ["grad_norm", "sparse_adam"])
def test_no_kernel_spills_to_scratch(source, tmp_path):
    out = tmp_path / "kernels.s"
    strict = ["-ffp-contract=off"] if source in STRICT else []
    subprocess.run([HIPCC, *FLAGS, *strict, "-o", str(out), os.path.join(CSRC, source + ".hip")], check=True,
                   stderr=subprocess.DEVNULL)
    sizes = re.findall(r"\.amdhsa_kernel (\S+).*?\.amdhsa_private_segment_fixed_size (\d+)", out.read_text(), re.S)
    assert sizes and [kernel for kernel, size in sizes if size != "0"] == []


STRICT = ("surfel_project", "sparse_adam", "splat_step", "loop_rectify", "splat_knn")     # as in the Makefile
OTHERS = sorted(f[:-4] for f in os.listdir(CSRC) if f.endswith(".hip"))
OTHERS = [s for s in OTHERS if s not in ("row_table", "grad_norm", "sparse_adam")]


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason="no hipcc")
@pytest.mark.parametrize("source", OTHERS)
def test_every_barrier_of_the_other_sources_waits_for_lds_stores(source, tmp_path):
    out = tmp_path / "kernels.s"
    strict = ["-ffp-contract=off"] if source in STRICT else []
    subprocess.run([HIPCC, *FLAGS, *strict, "-o", str(out), os.path.join(CSRC, source + ".hip")], check=True,
                   stderr=subprocess.DEVNULL)
    assert barriers_without_wait(out.read_text()) == []


@pytest.mark.parametrize("source", ["row_table.hip", "grad_norm.hip", "grad_norm.hpp", "sparse_adam.hip", "radix_sort.hpp"])
def test_no_loop_of_the_training_operators_begins_with_a_barrier(source):
    text = open(os.path.join(CSRC, source)).read()
    heads = re.findall(r"\b(?:for|while) \([^{}]*\) \{\s*__syncthreads\(\);", text) + \
        re.findall(r"\bdo \{\s*__syncthreads\(\);", text)
    assert heads == []
