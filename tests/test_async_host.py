"""The asynchronous loads into LDS (trnrt_amd/csrc/dsa_async.h) as hipcc compiles them: a scalar write of m0, the LDS address,
must be followed by one wait state before the load that uses it, and the compiler does not look into an asm statement for
that. Compiles for gfx950 only, runs nothing."""

import re
import subprocess

from trnrt_amd import build

PROBE = r"""
#include "dsa_async.h"
namespace dsa {
__global__ void probe(const uint16_t* p, uint16_t* out, int at) {
  __shared__ uint16_t t[4096];
  const uint32_t lds = lds_address(t) + at;
#pragma unroll
  for (int i = 0; i < 4; ++i) load_lds16(p + 512 * i + 8 * threadIdx.x, lds + 1024 * i);
  wait_loads<0>();
  lds_barrier();
  out[threadIdx.x] = t[threadIdx.x];
}
}
"""


def instructions(asm: str) -> list[str]:
    lines = (ln.split(";")[0].strip() for ln in asm.splitlines())
    return [ln for ln in lines if ln and not ln.startswith(".") and not ln.endswith(":")]


def too_close(code: list[str]) -> list[str]:
    """The loads into LDS right behind a scalar write of m0, and those that no write comes before."""
    bad, since = [], None
    for ins in code:
        if re.match(r"(global_load_lds|buffer_load\w* .*\blds$)", ins):
            if not since:
                bad.append(ins)
        if re.match(r"s_\w+ m0,", ins):
            since = 0
        elif since is not None:
            since += 1
    return bad


def test_oracle():
    assert too_close(["s_mov_b32 m0, s0", "global_load_lds_dwordx4 v[0:1], off"])
    assert too_close(["s_nop 0", "global_load_lds_dwordx4 v[0:1], off"])
    assert not too_close(["s_mov_b32 m0, s0", "s_nop 0", "global_load_lds_dwordx4 v[0:1], off"])


def test_wait_state_behind_m0(tmp_path):
    src = tmp_path / "probe.hip"
    src.write_text(PROBE)
    r = subprocess.run([build.hipcc(), *build.CFLAGS, *build.DEVICE_FLAGS, "--offload-device-only", "-S", str(src), "-o", "-"],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    code = instructions(r.stdout)
    assert sum(ins.startswith("global_load_lds_dwordx4") for ins in code) == 4
    assert not too_close(code)


def test_no_other_statement_writes_m0():
    """One place brings m0, as an operand that the compiler knows of."""
    for src in sorted(build.CSRC.iterdir()):
        for asm in re.findall(r"asm volatile\((.*?)\);", src.read_text(), flags=re.S):
            assert not re.search(r"\bm0\s*,", asm), src.name
            assert '"{m0}"' not in asm or src.name == "dsa_async.h"
