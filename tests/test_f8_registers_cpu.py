"""The pair kernel's warpgroups divide up the registers that a block is launched with (setmaxnreg): a compiler that gives a thread fewer makes every product in
pairs an error at run time.  Seen here when it is built."""
import os
import re
import subprocess

from distributed_inference_server_b200 import build as b


def test_the_pair_kernel_is_built_with_the_registers_that_it_divides_up(tmp_path):
    source = os.path.join(b.CSRC, "k_gemm_f8.cu")
    want = int(re.search(r"kF8PairRegs = (\d+)", open(source).read()).group(1))
    r = subprocess.run([b.NVCC, "-Xptxas=-v", *b.FLAGS, "-x", "cu", "-c", source, "-o", str(tmp_path / "o")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    used = re.findall(r"Compiling entry function '(\w*)'.*?Used (\d+) registers", r.stderr, flags=re.S)
    pairs = [int(n) for name, n in used if "gemm_f8_pair_kernel" in name]
    assert pairs == [want] * 5, used
