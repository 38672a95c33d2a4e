"""CPU: a warpgroup changes its share of registers (setmaxnreg) by one instruction that all four of its warps execute: PTX leaves anything
else undefined. Read from the sources: what such an instruction stands under may ask for a warp only by its warpgroup, and no warpgroup
meets two of them."""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "faie2-flashnext_b200", "csrc")
FILES = [f for f in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))) if "setmaxnreg" in open(f).read()]


def splits(text):
    """(instruction, the conditions it stands under) of every setmaxnreg; those of an else branch are the ones that its ifs asked before."""
    text = re.sub(r"//[^\n]*", "", text)
    found, stack, chain, at = [], [], [], 0
    for m in re.finditer(r"[{}]|setmaxnreg\.(dec|inc)", re.sub(r'"\{|\}"|\{[^{}\n]*\}', lambda q: " " * len(q.group()), text)):
        before = text[at:m.start()]
        if m.group() == "{":
            head = before.strip().split(";")[-1].strip()
            cond = re.search(r"\bif\s*(?:constexpr\s*)?\((.*)\)\s*$", head, re.S)
            own = [" ".join(cond.group(1).split())] if cond else []
            stack.append((chain if head.startswith("else") else []) + own)
        elif m.group() == "}":
            chain = stack.pop() if stack else []
        else:
            found.append((m.group(1), [c for conds in stack for c in conds if re.search(r"\bwarp\b", c)]))
        at = m.end()
    return found


def warpgroup(cond, names):
    """The bound, in warps, of a condition that keeps warpgroups together, else None."""
    m = re.fullmatch(r"warp (?:<|>=) (\w+)", cond)
    if not m:
        return None
    v = int(m.group(1)) if m.group(1).isdigit() else names.get(m.group(1))
    return v if v is not None and v % 4 == 0 else None


def test_the_reader_tells_them_apart():
    bad = 'if (warp == 0) {\n asm("setmaxnreg.dec 72;");\n } else if (warp == 1) {\n asm("setmaxnreg.dec 72;");\n } else {\n asm("setmaxnreg.inc 216;");\n }'
    assert splits(bad) == [("dec", ["warp == 0"]), ("dec", ["warp == 0", "warp == 1"]), ("inc", ["warp == 0", "warp == 1"])]
    good = 'if (warp < 4) {\n asm("setmaxnreg.dec 72;");\n if (warp == 0) {\n f();\n }\n } else {\n asm("setmaxnreg.inc 216;");\n }'
    assert splits(good) == [("dec", ["warp < 4"]), ("inc", ["warp < 4"])]


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_a_warpgroup_splits_as_one(path):
    text = open(path).read()
    names = {}
    for line in re.findall(r"constexpr int ([^;]*);", "\n".join(open(f).read() for f in glob.glob(os.path.join(CSRC, "*")))):
        for name, value in re.findall(r"(\w+) = (\d+)(?=,|$)", line):
            names[name] = int(value)
    got = splits(text)
    assert {kind for kind, _ in got} == {"dec", "inc"}
    for kind, conds in got:
        assert all(warpgroup(c, names) is not None for c in conds), (kind, conds)
    seen = [tuple(c) for kind, c in got if kind == "dec"]
    assert len(seen) == len(set(seen))
