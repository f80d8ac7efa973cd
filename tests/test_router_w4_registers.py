"""What the router's and the 4-bit products' kernels keep on the stack, on the code the build actually generates (no GPU needed).

Values that do not fit a kernel's registers go to the stack without a word from the compiler.  The numbers are what was measured with:
none for rows of up to 512 experts; route and balance sums in one pass over rows of 513 to 1024 keep some 36 registers there, and the experts' products
with zero points up to seven, which 128 registers a lane (two workgroups to a CU) leave no room for."""

import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from deepep_amd import build


def _stack(source, out):
    """name -> (vector registers, bytes of stack) of every kernel of a source."""
    flags = [f for f in build.FLAGS if f != "-fPIC"] + list(build.FILE_FLAGS.get(source, ()))
    proc = subprocess.run([build._hipcc(), *flags, "--cuda-device-only", "-S", "-o", str(out), os.path.join(build.CSRC, source)], capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-2000:]
    found = {}
    for name, meta in re.findall(r"\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", out.read_text(), re.S):
        registers, stack = (int(re.search(rf"\.amdhsa_{field}\s+(\d+)", meta).group(1)) for field in ("next_free_vgpr", "private_segment_fixed_size"))
        found[name] = (registers, stack)
    return found


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    try:
        hipcc = build._hipcc()
        subprocess.run([hipcc, "--version"], capture_output=True, check=True)
    except (RuntimeError, OSError):
        pytest.skip("hipcc is not installed")
    folder = tmp_path_factory.mktemp("isa")
    with ThreadPoolExecutor(2) as pool:
        return dict(zip(("router", "w4"), pool.map(lambda name: _stack(name + ".hip", folder / (name + ".s")), ("router", "w4"))))


def test_router_kernels(kernels):
    rows = {name: re.search(r"router_(forward|backward)_kernelILi(\d+)E", name) for name in kernels["router"]}
    assert sum(match is not None for match in rows.values()) == 5 * 3 * 2 * (3 + 1)  # registers a lane, types, scores; three forward kernels and the gradient
    for name, (registers, stack) in kernels["router"].items():
        wide = rows[name] is not None and rows[name].group(2) == "16"
        assert stack <= (160 if wide and "forward" in name else 0), f"{name}: {registers} registers, {stack} bytes of stack"


def test_product_kernels(kernels):
    # kind, half, zero points, groups to an operand, blocks of rows, streamed
    products = {name: re.search(r"product_kernelIL\w*E(\d)ELb(\d)ELb(\d)ELi(\d)ELi(\d)ELb(\d)E", name) for name in kernels["w4"]}
    products = {name: match.groups() for name, match in products.items() if match is not None}
    assert len(products) == 3 * 2 * 2 * 3 * 3  # kinds, types, zero points or none, groups; one block (streamed or not) or four
    for name, (kind, _, zeros, _, blocks, _) in products.items():
        registers, stack = kernels["w4"][name]
        assert stack <= (32 if kind != "0" and zeros == "1" and blocks == "1" else 0), f"{name}: {registers} registers, {stack} bytes of stack"
