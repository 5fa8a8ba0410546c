"""How the 8-bit products' kernels read memory, from the sources.

They may start while the kernel in front still runs (programmatic dependent launch), so what it writes can change during their own lifetime: a load through the
read-only path, which `const __restrict__` allows the compiler to make of a plain one, is not made for that.  So whatever such a kernel reads it reads from
L2 (__ldcg), by TMA, or by a load that is written out."""
import os
import re

import pytest

from tests.test_kernel_order_cpu import CSRC


def kernels(name):
    s = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    for m in re.finditer(r"__global__", s):
        head = re.compile(r"(\w*kernel\w*)\s*\(([^{]*)\)\s*\{").search(s, m.start())
        at = start = head.end()
        depth = 1
        while depth:
            depth += {"{": 1, "}": -1}.get(s[at], 0)
            at += 1
        yield head.group(1), head.group(2), s[start:at]


@pytest.mark.parametrize("source", ["k_quant_f8.cu", "k_gemm_f8.cu"])
def test_what_an_overlapping_kernel_may_write_is_read_from_l2(source):
    seen = 0
    for name, params, body in kernels(source):
        if "pdl_wait();" not in body:
            continue
        seen += 1
        assert not re.search(r"\*\s*reinterpret_cast<const", body), name  # a vector load of the plain kind
        for p in re.findall(r"const \w+ ?\*\s*(?:__restrict__)?\s*(\w+)", params):
            assert not re.search(rf"(?<![.\w]){p}\[", body), (name, p)
    assert seen == {"k_quant_f8.cu": 3, "k_gemm_f8.cu": 2}[source]
