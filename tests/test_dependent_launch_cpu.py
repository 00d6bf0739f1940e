"""Kernels that begin before the launch in front of them has ended: what they
read of its results stands behind the wait that the programming model asks for.
Read from the source, as no run can show a missing wait reliably."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zipmoe-icml26_b200", "csrc")


def _kernel(file, name):
    """Lines of a kernel, up to the closing brace in the first column."""
    text = open(os.path.join(CSRC, file)).read()
    m = re.search(r"__global__[^;{]*?\b" + name + r"\b", text)
    assert m, name
    return text[m.start():text.index("\n}", m.start())].splitlines()


def _waits(lines):
    return [i for i, line in enumerate(lines) if "griddepcontrol.wait" in line]


def test_adapter_gradient_waits_for_its_factors():
    # one wait in CTA (0, 0) keeps the launch from ending early; the other stands
    # in front of the loaders' loop, at most left out where nothing of the
    # launches in front is read (which: dB, whose factor is the caller's)
    lines = _kernel("lora_tc.cu", "lora_dw_kernel")
    waits = [i for i in _waits(lines) if "blockIdx" not in lines[i]]
    assert len(waits) == 1
    assert re.match(r'\s*(if \(!which\) )?asm volatile\("griddepcontrol.wait;"', lines[waits[0]])
    loop = next(i for i, line in enumerate(lines) if "for (int s0 = 0; s0 < ns" in line)
    assert waits[0] < loop


def test_other_dependents_wait_before_they_read():
    for file, name, read in (("permute.cu", "sort_first_kernel", r"wide_counts\("), ("permute.cu", "scatter_rows_kernel", r"row_of \+ t"),
                             ("lora_tc.cu", "lora_expand_kernel", r"a\.(split|second)\b")):
        lines = _kernel(file, name)
        at = next(i for i, line in enumerate(lines) if re.search(read, line))
        assert any(i < at and re.match(r"\s*asm volatile", lines[i]) for i in _waits(lines)), name
