"""The layer operators' kernels as built: orders of instructions that their waits count on, read from the code object."""
import os
import re
import subprocess

import pytest

from conftest import pkg
from mx_kernels import SIZES, kernels_of, round_of, widths

MX = pkg("mx")


@pytest.fixture(scope="module")
def listing(tmp_path_factory):
    """{kernel: its instructions} of the built library."""
    if not os.path.exists(MX.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    at = tmp_path_factory.mktemp("code")
    llvm = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")
    fat, code = str(at / "fat"), str(at / "code")
    subprocess.run([f"{llvm}/llvm-objcopy", "--dump-section", f".hip_fatbin={fat}", MX.LIB_PATH, str(at / "copy")], check=True)
    subprocess.run([f"{llvm}/clang-offload-bundler", "--unbundle", "--type=o", f"--input={fat}", f"--output={code}",
                    "--targets=hipv4-amdgcn-amd-amdhsa--gfx950"], check=True)
    text = subprocess.run([f"{llvm}/llvm-objdump", "-d", "--no-show-raw-insn", code], check=True, capture_output=True, text=True).stdout
    kernels = {}
    for part in re.split(r"\n(?=[0-9a-f]+ <)", text):
        head = re.match(r"[0-9a-f]+ <(\w+)>:", part)
        if head:
            kernels[head.group(1)] = [line.split("//")[0].strip() for line in part.split("\n")[1:]]
    return kernels


def first_loads(instructions):
    """From the first direct load to LDS to the barrier after it: "lds" and "load" for buffer loads, a number for a wait."""
    events, begun = [], False
    for i in instructions:
        if i.startswith("buffer_load"):
            events.append("lds" if i.endswith(" lds") else "load")
            begun = begun or events[-1] == "lds"
        elif begun and i.startswith("s_waitcnt") and "vmcnt" in i:
            events.append(int(re.search(r"vmcnt\((\d+)\)", i).group(1)))
        elif begun and i.startswith("s_barrier"):
            break
    return events


def test_few_rows_wait_counts_the_loads_behind_x(listing):
    """few_kernel waits for all but the weight's first 2 + 2 U loads: right where x's direct loads come before those."""
    few = {n: i for n, i in listing.items() if "few_kernel" in n}
    assert len(few) == 12
    for name, instructions in few.items():
        events = first_loads(instructions)
        u = int(re.search(r"few_kernelI.*Li[48]ELi(\d)ELi", name).group(1))
        first = events.index("load")
        assert "lds" not in events[first:], name
        assert events.count("load") == events[-1] == 2 + 2 * u, (name, events)


def test_few_rows_first_loads_wait_for_none(listing):
    """Up to the wait for x nothing waits for memory: the weight's first loads go out behind x's, not when x is there."""
    for name, instructions in listing.items():
        if "few_kernel" in name:
            events = first_loads(instructions)
            # the last of x's loads, the wait of the later rounds (all of x, no weight on its way) and then the weight's
            tail = events[events.index("load"):]
            assert [e for e in tail if e != "load"] == [tail[-1]], (name, events)


def test_every_kernel_that_is_built_is_reached_and_tested(listing):
    """The sizes of the product tests take every kernel of the library, and no kernel is built that none of them can take."""
    built = set()
    for name in listing:
        m = re.match(r"_ZN5ns_mx\d+(few|tile)_kernelI(?:f|NS_\d\w+?E)(Li.*)EE", name)
        if m:
            built.add((m.group(1), *(int(v) for v in re.findall(r"Li(\d+)E", m.group(2) + "E"))))
    reached = {k for size in SIZES for k in kernels_of(*size)}
    assert built == reached
    for kernel in reached:
        at, r = widths(kernel), round_of(kernel)
        assert min(at) <= max(128, r // 4) or kernel[:3] == ("few", kernel[1], 4)
        assert r in at and (max(at) > 2 * r or kernel[0] == "few" and kernel[2] == 2)


def test_tiles_first_loads_come_stage_by_stage(listing):
    """The first wait of a tile with three places or more leaves the loads of all stages but the first in flight: right where
    each stage's loads, from the same rows one stage further, are issued together."""
    seen = 0
    for name, instructions in listing.items():
        m = re.match(r".*tile_kernelI(?:f|NS_\d\w+?E)Li(\d)ELi(\d+)ELi(\d+)ELi(\d)ELi(\d)ELi(\d+)ELi(\d)ELi(\d)EE", name)
        if not m or int(m.group(7)) < 3:
            continue
        fmt, bm, bn, wm, wn, bk, p, _ = (int(v) for v in m.groups())
        each = (bm * bk * (1 if fmt == 8 else 0.5) + bn * bk / 2) / 1024 / (wm * wn)     # direct loads of a wave and stage
        assert each == int(each)
        each = int(each)
        loads, wait = [], None
        for i in instructions:
            if i.startswith("buffer_load"):
                assert i.endswith(" lds"), name
                loads.append(re.match(r"\S+ (v\d+), (s\[\d+:\d+\])", i).groups())
            elif i.startswith("s_waitcnt") and "vmcnt" in i:
                wait = int(re.search(r"vmcnt\((\d+)\)", i).group(1))
            elif i.startswith("s_barrier"):
                break
        stages = loads[-(p - 1) * each:]
        stages = [sorted(stages[s * each:(s + 1) * each]) for s in range(p - 1)]
        assert wait == (p - 2) * each and all(s == stages[0] for s in stages) and len(set(stages[0])) == each, (name, loads)
        seen += 1
    assert seen == 9     # three tiles, three types
