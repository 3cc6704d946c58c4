"""Shared arrays that kernels read in wider pieces than their own type state the alignment of the piece (source text, no GPU)."""
import re

import pytest

from conftest import ROOT

SOURCES = sorted((ROOT / "fastmd_b200" / "csrc").glob("*.cu*"))
WIDTH = {"float4": 16, "uint4": 16, "int4": 16, "float2": 8, "uint2": 8, "double": 8, "uint64_t": 8}
SIZE = {"unsigned char": 1, "char": 1, "float": 4, "int": 4, "int32_t": 4, "uint32_t": 4, "float2": 8, "double": 8,
        "int64_t": 8, "uint64_t": 8}
DECLARED = re.compile(r"__shared__\s+(?P<align>(?:alignas|__align__)\((?P<bytes>\d+)\))?\s*(?P<type>unsigned char|\w+)\s+"
                      r"(?P<names>[^;=]+);")


def read_wider(text):
    """(name, alignment that is stated or that of its type, bytes of the widest piece it is cast to) of each shared array."""
    for m in DECLARED.finditer(text):
        if m["type"] not in SIZE:
            continue
        stated = int(m["bytes"] or 0) or SIZE[m["type"]]
        # the scope of a declaration: up to the end of the function, a brace in the first column
        scope = text[m.end():].split("\n}", 1)[0]
        for name in re.findall(r"(\w+)\s*\[", re.sub(r"\[[^\]]*\]", "[", m["names"])):
            casts = re.findall(r"reinterpret_cast<(?:const\s+)?(\w+)\s*(?:const\s*)?[*&]\s*>\(\s*&?" + name + r"\b", scope)
            # pointers that walk through the array: *x = name + .., and what those are cast to
            for walker in re.findall(r"\*\s*(\w+)\s*=\s*" + name + r"\b", scope):
                casts += re.findall(r"reinterpret_cast<(?:const\s+)?(\w+)\s*\*>\(\s*" + walker + r"\b", scope)
            yield name, stated, max([WIDTH.get(c, 0) for c in casts], default=0)


@pytest.mark.parametrize("source", SOURCES, ids=[s.name for s in SOURCES])
def test_alignment_is_stated(source):
    for name, stated, needed in read_wider(source.read_text()):
        assert stated >= needed, f"{source.name}: {name} is read in pieces of {needed} bytes, aligned to {stated}"


def test_the_search_finds_them():
    text = ("__global__ void f() {\n    __shared__ float q[8], v[4];\n    extern __shared__ float all[];\n"
            "    __shared__ alignas(16) float ok[8];\n    const float *x = all + 4, *w = x;\n"
            "    use(*reinterpret_cast<const float4*>(v + 4), *reinterpret_cast<float4*>(&ok[4]));\n"
            "    use(*reinterpret_cast<const float4*>(x + 8));\n}\n")
    assert list(read_wider(text)) == [("q", 4, 0), ("v", 4, 16), ("all", 4, 16), ("ok", 16, 16)]
