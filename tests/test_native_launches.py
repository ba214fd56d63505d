"""Kernels that may start while the one before them still writes (programmatic launches), read as source.

What such a kernel reads of the one before it must not be promised constant (const with __restrict__ lets the compiler
load it ahead of the wait), and must be read behind the wait by loads that stay there. No run can show a load that was
moved for certain, so the source is what is tested."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna4-conv3d-wmma_b200", "csrc")
WRITTEN_BEFORE = ("part", "cpart", "gpart")       # the first pass's sums, in the second pass's arguments


def _functions(text):
    """(name, arguments, body) of every device function and kernel."""
    for m in re.finditer(r"^(?:template [^\n]*\n)?[^\n/]*__(?:global|device)__[^;{]*?(\w+)\(", text, re.M):
        at, depth = m.end(), 1
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        args, start = text[m.end():at - 1], text.find("{", at)
        end, depth = start + 1, 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield m.group(1), args, text[start:end]


def _sources():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = re.sub(r"//[^\n]*|__launch_bounds__\([^)]*\)", "", open(path).read())
        if "griddepcontrol" in text or "wait_for_previous" in text:
            yield os.path.basename(path), text


def test_sums_of_the_kernel_before_are_not_promised_constant():
    waiting = set()
    for path, text in _sources():
        found = list(_functions(text))
        reads = {n for n, a, b in found if "wait_for_previous()" in b}
        waiting |= reads
        for name, args, body in found:
            if name not in reads and name != "param_grads":          # (which kernels call behind their wait)
                continue
            for arg in args.split(","):
                words = arg.replace("*", " * ").split()
                if words and words[-1] in WRITTEN_BEFORE:
                    assert "__restrict__" not in words, f"{path}: {name}: {arg.strip()}"
    assert {"apply_kernel", "bwd_dx_kernel", "params_kernel"} <= waiting


def test_sums_of_the_kernel_before_are_read_behind_the_wait():
    for path, text in _sources():
        for name, args, body in _functions(text):
            if "wait_for_previous()" not in body and name != "param_grads":
                continue
            names = [w for w in WRITTEN_BEFORE if re.search(rf"\b{w}\b", args)]
            # a pointer into them counts as them
            names += [m.group(1) for w in list(names) for m in re.finditer(rf"\*\s*(\w+) = {w}\b", body)]
            for w in names:
                assert not re.search(rf"\b{w}\s*\[", body), f"{path}: {name} reads {w} with a plain load"
                first = body.find("wait_for_previous()")
                assert all(m.start() > first for m in re.finditer(rf"\b{w}\b", body)), f"{path}: {name}: {w}"
