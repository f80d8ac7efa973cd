"""The norm's and the products' kernels on the code the build actually generates (no GPU needed): what they keep on the stack, and the waits that loads written by hand need.

Values that do not fit a kernel's registers go to the stack without a word from the compiler.  The numbers are what was measured with: none but for some
addresses of the tiles of 256 x 256 with turned operands, set aside outside the loop over k, and 30 registers of the gradient of FP32 rows of more than 8192 values, of which
1024 threads have 128 each.
The compiler puts no wait between a vector instruction that writes a scalar register and a load written by hand that reads it, which the machine asks five cycles for."""

import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from deepep_amd import build


def _assembly(source, out):
    flags = [f for f in build.FLAGS if f != "-fPIC"] + list(build.FILE_FLAGS.get(source, ()))
    proc = subprocess.run([build._hipcc(), *flags, "--cuda-device-only", "-S", "-o", str(out), os.path.join(build.CSRC, source)], capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-2000:]
    return out.read_text()


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    try:
        hipcc = build._hipcc()
        subprocess.run([hipcc, "--version"], capture_output=True, check=True)
    except (RuntimeError, OSError):
        pytest.skip("hipcc is not installed")
    folder = tmp_path_factory.mktemp("isa")
    with ThreadPoolExecutor(2) as pool:
        return dict(zip(("norm", "dense"), pool.map(lambda name: _assembly(name + ".hip", folder / (name + ".s")), ("norm", "dense"))))


def _stack(text):
    """name -> (vector registers, bytes of stack) of every kernel."""
    found = {}
    for name, meta in re.findall(r"\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", text, re.S):
        found[name] = tuple(int(re.search(rf"\.amdhsa_{field}\s+(\d+)", meta).group(1)) for field in ("next_free_vgpr", "private_segment_fixed_size"))
    return found


def test_norm_kernels(assembly):
    kernels = _stack(assembly["norm"])
    forward = [re.search(r"norm_kernelILi(\d+)ELi(\d)ELi(\d)E", name) for name in kernels]
    backward = [re.search(r"norm_backward_kernelILi(\d+)ELi(\d)ELi(\d)E", name) for name in kernels]
    assert sum(m is not None for m in forward) >= 3 and sum(m is not None for m in backward) >= 3
    for (name, (registers, stack)), match in zip(kernels.items(), backward):
        wide = match is not None and match.groups() == ("1024", "2", "0")
        assert stack <= (120 if wide else 0), f"{name}: {registers} registers, {stack} bytes of stack"


def test_product_kernels(assembly):
    kernels = _stack(assembly["dense"])
    ways = {name: re.search(r"(tile|products)_kernelI.*LNS0_3WayE(\d)E", name) for name in kernels}
    assert sum(m is not None for m in ways.values()) == 3 * (2 * 5 + 1 + 2)  # ways; of two types five tile kernels and the three products', of 8-bit integers one
    for name, (registers, stack) in kernels.items():
        large = ways[name] is not None and ways[name].group(2) == "3"
        assert stack <= (32 if large else 0), f"{name}: {registers} registers, {stack} bytes of stack"
        if ways[name] is not None and ways[name].group(2) == "2":
            assert registers <= 128, f"{name}: {registers} registers leave no room for a second workgroup"


def _scalars(text):
    found = set()
    for first, last in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        found |= set(range(int(first), int(last) + 1))
    return found | {int(n) for n in re.findall(r"\bs(\d+)\b", text)}


def test_loads_to_lds_wait_for_their_scalars(assembly):
    recent, loads = [], 0  # (cycles ago, registers, instruction) of vector instructions that write scalars
    for line in assembly["dense"].splitlines():
        instruction = line.split(";")[0].strip()
        if re.match(r"_Z\S+:", line):
            recent = []
        if not instruction or instruction.startswith(".") or instruction.endswith(":"):
            continue
        if re.match(r"buffer_load_dword.* lds", instruction):
            loads += 1
            reads = _scalars(instruction.split(",", 1)[1])
            assert not [i for ago, writes, i in recent if ago < 5 and writes & reads], instruction
        passed = int(instruction.split()[1]) + 1 if instruction.startswith("s_nop") else 1
        recent = [(ago + passed, writes, i) for ago, writes, i in recent if ago + passed < 8]
        if re.match(r"v_read|v_cmp", instruction):
            recent.append((0, _scalars(instruction.split(",")[0]), instruction))
    assert loads > 100
