"""Wait states around inline assembly, read off the gfx950 assembly that the
build's own compiler writes for a small kernel.

A scalar register that a vector instruction wrote (v_readfirstlane, a compare)
may be read by a memory instruction five wait states later at the earliest.
The compiler keeps that distance for its own memory instructions; a load
inside inline assembly has to keep it by itself."""
import os
import re
import subprocess

import pytest

from text_guided_face_recognition_amd import build

WAIT = 5

# the base comes out of vector registers: its readfirstlanes stand right before
# the assembly
PROBE = {
    "dma16": ("tgfr_xattn.h", "tgfr::dma16(p[t], o[t], 0, tgfr::x_probe_lanes(o[t]));"),
    "glds16s": ("tgfr_common.h", "tgfr::glds16s(p[t], o[t], 0);"),
}


def compiled(tmp_path, header, call):
    src = tmp_path / "probe.hip"
    src.write_text(f'''#include "{header}"
namespace tgfr {{
__device__ uint64_t x_probe_lanes(unsigned o) {{ return __ballot(o != 0x80000000u); }}
}}
extern "C" __global__ void probe(const char* const* p, const unsigned* o, float* out) {{
  const int t = threadIdx.x;
  {call}
  out[t] = 0.f;
}}
''')
    out = tmp_path / "probe.s"
    subprocess.run([build.HIPCC, f"--offload-arch={build.ARCH}", "-O3", "-std=c++17",
                    "--offload-device-only", "-S", *build.NO_PACKED_FP32, "-I", build.CSRC,
                    str(src), "-o", str(out)], check=True, capture_output=True, timeout=300)
    return [s for s in (line.split(";")[0].strip() for line in out.read_text().splitlines())
            if re.match(r"[sv]_|global_|buffer_|ds_|flat_", s)]


def scalars(text):
    """Numbers of the scalar registers that an operand list names."""
    found = set()
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        found |= set(range(int(a), int(b) + 1))
    return found | {int(n) for n in re.findall(r"\bs(\d+)\b", text)}


def distance(lines, at):
    """Wait states between a memory instruction and the last vector
    instruction that wrote a scalar register it reads (None: there is none)."""
    reads, states = scalars(lines[at]), 0
    for line in reversed(lines[:at]):
        op, _, rest = line.partition(" ")
        written = scalars(rest.split(",")[0])
        if written & reads:
            if op.startswith("v_"):
                return states
            reads -= written
        states += int(rest, 0) + 1 if op == "s_nop" else op != "s_waitcnt"
    return None


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no compiler")
@pytest.mark.parametrize("name", sorted(PROBE))
def test_lds_dma_waits_for_its_scalar_base(tmp_path, name):
    lines = compiled(tmp_path, *PROBE[name])
    loads = [i for i, s in enumerate(lines) if s.startswith("global_load_lds") and "s[" in s]
    assert loads
    for i in loads:
        states = distance(lines, i)
        assert states is not None, "the base does not come from vector registers"
        assert states >= WAIT, f"{lines[i]}: {states} wait states\n" + "\n".join(lines[:i + 1])
