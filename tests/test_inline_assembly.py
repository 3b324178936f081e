"""Inline assembly beside matrix products: the compiler puts the wait states that a result needs in front of the instructions that it knows, and
does not look into assembly.  A source that (with what it includes) has matrix products may have waits and barriers in assembly, nothing that
reads or writes a vector register."""
import os
import re

import pytest

from swifttransformer_amd.ops import library


def with_includes(path, seen):
    if path in seen:
        return ""
    seen.add(path)
    with open(path) as f:
        text = f.read()
    local = [os.path.join(library.CSRC, name) for name in re.findall(r'#include "([^"]+)"', text)]
    return text + "".join(with_includes(p, seen) for p in local if os.path.exists(p))


def instructions(text):
    """What the asm statements of a source hold."""
    code = re.sub(r"//[^\n]*", "", text)
    return [word for body in re.findall(r'\basm\b(?:\s+volatile)?\s*\(\s*"([^"]*)"', code)
            for word in re.findall(r"[a-z]\w*", re.sub(r"\\n|\\t", " ", body)) if re.match(r"[vsd][a-z]*_", word)]


@pytest.mark.parametrize("source", [os.path.basename(p) for p in library.sources()])
def test_no_vector_assembly_beside_matrix_products(source):
    text = with_includes(os.path.join(library.CSRC, source), set())
    if "__builtin_amdgcn_mfma" not in text:
        return
    assert set(instructions(text)) <= {"s_waitcnt", "s_barrier"}


def test_the_check_sees_assembly():
    assert instructions('asm("v_max_f32 %0, %1, %2" : "=v"(d) : "v"(a));  // asm("v_min_f32")') == ["v_max_f32"]
    assert instructions('asm volatile("s_waitcnt vmcnt(0)\\n\\ts_barrier" ::: "memory");') == ["s_waitcnt", "s_barrier"]
    assert instructions('asm volatile("" : "+v"(l));') == []
