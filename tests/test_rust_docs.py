"""The Rust surface's documentation, on the CPU without a Rust toolchain."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_RS = os.path.join(ROOT, "crates", "headshot-hip", "src", "lib.rs")


def docs(text):
    """Public struct -> its doc comment."""
    out, doc = {}, []
    for line in text.splitlines():
        if line.startswith("///"):
            doc.append(line[3:].strip())
        elif not line.startswith("#["):
            m = re.match(r"pub (?:struct|enum) (\w+)", line)
            if m:
                out[m.group(1)] = " ".join(doc)
            doc = []
    return out


def test_public_types_are_documented():
    found = docs(open(LIB_RS).read())
    assert {"HipContext", "HipTensor", "PagedKv"} <= set(found)
    assert all(found.values()), [name for name, doc in found.items() if not doc]
    assert found["HipContext"].startswith("One device's op surface")
    assert found["PagedKv"].startswith("One layer's paged key-value cache")
