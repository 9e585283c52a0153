"""No kernel of the built library has packed FP32 arithmetic (v_pk_add_f32, v_pk_mul_f32, v_pk_fma_f32), whatever its operands: the
library is built without the feature.  Read back from the gfx950 code objects, no GPU needed."""
import os
import re
import subprocess

import pytest

from closerlook3d_amd import build
from tests.test_isa_packed_operands import LIB, OBJDUMP, gfx950_code_objects

PACKED = re.compile(r"\bv_pk_(add|mul|fma)_f32\b")


def packed_arithmetic(lib, tmp_path):
    """{kernel: number of packed FP32 instructions}, and how many kernels there are."""
    found, kernels = {}, 0
    for n, blob in enumerate(gfx950_code_objects(lib)):
        co = tmp_path / f"obj{n}.co"
        co.write_bytes(blob)
        name = None
        for line in subprocess.run([OBJDUMP, "-d", str(co)], capture_output=True, text=True, check=True).stdout.splitlines():
            m = re.match(r"^[0-9a-f]{16} <([^>]+)>:", line)
            if m:
                name, kernels = m.group(1), kernels + 1
            elif PACKED.search(line):
                found[name] = found.get(name, 0) + 1
    return found, kernels


@pytest.mark.skipif(not os.path.exists(LIB), reason="libcl3d.so not built")
@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="llvm-objdump not available")
def test_the_library_has_no_packed_fp32_arithmetic(tmp_path):
    found, kernels = packed_arithmetic(LIB, tmp_path)
    assert kernels > 100, f"only {kernels} kernels disassembled: the code objects were not found"
    assert not found, found


@pytest.mark.skipif(not (os.path.exists(build.HIPCC) and os.path.exists(OBJDUMP)), reason="no compiler")
def test_the_build_flags_are_what_keeps_it_so(tmp_path):
    """A float pair, built with the library's flags and without the one."""
    src = tmp_path / "pair.hip"
    src.write_text("""#include <hip/hip_runtime.h>
typedef float f2 __attribute__((ext_vector_type(2)));
__global__ void pair(const f2 *a, const f2 *b, f2 *c) {
  c[threadIdx.x] = __builtin_elementwise_fma(a[threadIdx.x], b[threadIdx.x], c[threadIdx.x]);
}
""")
    flags = [f for f in build.FLAGS if f != "-shared"]
    at = flags.index("-packed-fp32-ops")
    assert flags[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"]
    for keep in (True, False):
        obj = tmp_path / f"pair{keep}.o"
        used = flags if keep else flags[:at - 3] + flags[at + 1:]
        subprocess.check_call([build.HIPCC, *used, "-c", str(src), "-o", str(obj)], stderr=subprocess.DEVNULL)
        found, kernels = packed_arithmetic(str(obj), tmp_path)
        assert kernels == 1 and bool(found) != keep, (keep, found)
