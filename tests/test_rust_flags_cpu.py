"""An engine flag that the Rust crate has is of use only with the functions that INTEGRATION.md names beside it: they are declared in the crate and in the copy
of its declarations that INTEGRATION.md prints, with the header's parameters."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
read = lambda *p: open(os.path.join(ROOT, *p)).read()  # noqa: E731


def params(text):
    text = re.sub(r"/\*.*?\*/|//[^\n]*", " ", text, flags=re.S)
    return {m[0]: len(m[1].split(",")) for m in re.findall(r"(dis_engine_\w+)\s*\(([^;()]*)\)", text)}


def test_functions_named_beside_a_flag_are_declared():
    doc, crate = read("INTEGRATION.md"), read("integration", "rust", "inference-sys", "src", "lib.rs")
    header = params(read("include", "dis_engine.h"))
    seen = 0
    for row in doc.splitlines():
        cell = row.split("|")[1] if row.startswith("| `DIS_FLAG_") else ""
        flags = re.findall(r"`(DIS_FLAG_\w+)`", cell)
        if not any(f"pub const {f}:" in crate for f in flags):
            continue
        for name in re.findall(r"`(dis_engine_\w+)`", cell):
            seen += 1
            for where in (crate, doc):
                decl = params("\n".join(re.findall(r"pub fn [^;]*;", where)))
                assert decl.get(name) == header[name], (name, flags)
    assert seen >= 2
