"""The machine code of all that the operators around the 8-bit KV cache launch (CPU: read from the built library): no packed
fp32 vector instructions, some of whose forms have given wrong results on gfx950; and, in the kernel whose accumulators lie in
registers that only its asm statements touch, no other use of those."""
import os
import re
import subprocess
import sys

import pytest

import cabi
from test_kernel_resources import _code_objects

LLVM = "/opt/rocm/llvm/bin"
pytestmark = pytest.mark.skipif(not os.path.exists(LLVM + "/llvm-objdump"), reason="no llvm-objdump")


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    """kernel -> its instructions, of the library's kernels that have kv8 or qk_norm in their names"""
    found = {}
    for i, obj in enumerate(_code_objects(cabi.LIB_PATH)):
        f = tmp_path_factory.mktemp("co") / ("%d.co" % i)
        f.write_bytes(obj)
        names = subprocess.run([LLVM + "/llvm-readelf", "-sW", str(f)], capture_output=True, text=True, check=True).stdout
        if not re.search("kv8|qk_norm", names):
            continue
        name = None
        for line in subprocess.run([LLVM + "/llvm-objdump", "-d", "--no-show-raw-insn", str(f)], capture_output=True, text=True, check=True).stdout.splitlines():
            m = re.match(r"[0-9a-f]+ <(\S+)>:", line)
            if m:
                name = m.group(1)
                found[name] = []
            elif name and line.startswith("\t"):
                found[name].append(line.split("//")[0].strip())
    return found


def test_no_packed_fp32_instructions(code):
    kernels = [k for k in code if re.search("kv8|qk_norm", k)]
    for part in ("fwd_kv8_kernel", "kv8_combine", "kv8_prefill_kernel", "kv8_prefill_wide_kernel", "kv8_quantize", "kv8_dequantize", "qk_norm_fwd", "qk_norm_bwd"):
        assert any(part in k for k in kernels), part
    bad = {k: [x for x in lines if re.match(r"v_pk_(add|mul|fma)_f32", x)] for k, lines in code.items()}
    assert not {k: v[:3] for k, v in bad.items() if v}


def test_the_compiler_leaves_the_owned_accumulators_alone(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "vllm-flash-attention_amd")
    sys.path.insert(0, pkg)
    import build
    out = tmp_path / "k.s"
    src = "fwd_prefill_wide_kv8.hip"
    subprocess.check_call([build.HIPCC] + build.HIP_FLAGS + build.EXTRA_FLAGS[src] + ["-S", "--cuda-device-only", "-w", os.path.join(build.CSRC, src), "-o", str(out)])
    in_asm, bad, kernels = False, [], 0
    for line in open(out):
        if "#ASMSTART" in line:
            in_asm = True
        elif "#ASMEND" in line:
            in_asm = False
        elif not in_asm:
            kernels += bool(re.match(r"^_ZN3vfa23kv8_prefill_wide_kernel\S*:", line))
            for m in re.finditer(r"\ba(\d+)\b|\ba\[(\d+):(\d+)\]", line):
                if int(m.group(1) or m.group(2)) < 192 and not line.lstrip().startswith((";", ".")):
                    bad.append(line.strip())
    assert kernels >= 6 and not bad, bad[:10]
