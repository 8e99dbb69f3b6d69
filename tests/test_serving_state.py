"""What the batched serving calls leave of the host's HIP state and give their kernels, on a HIP
runtime without a device (tests/host_checks)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def state(tmp_path_factory):
    out = tmp_path_factory.mktemp("serving_state")
    here, runtime = os.path.join(ROOT, "tests", "host_checks"), os.path.join(ROOT, "ai-research_amd", "csrc", "runtime")
    sources = [os.path.join(runtime, s + ".cpp") for s in ("runtime", "engine", "model", "ring", "serving")]
    sources += [os.path.join(here, s) for s in ("fake_hip.cpp", "serving_state.cpp")]
    exe = str(out / "serving_state")
    objs = [str(out / ("%d.o" % i)) for i in range(len(sources))]
    jobs = [subprocess.Popen(["g++", "-O1", "-std=c++17", "-pthread", "-D__HIP_PLATFORM_AMD__", "-w",
                              "-I", os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"),
                              "-I", os.path.join(ROOT, "include"), "-I", os.path.dirname(runtime), "-I", here,
                              "-c", s, "-o", o]) for s, o in zip(sources, objs)]
    assert all(j.wait() == 0 for j in jobs)
    subprocess.run(["g++", "-pthread", *objs, "-ldl", "-Wl,--wrap=hipModuleGetFunction", "-Wl,--wrap=hipModuleLaunchKernel",
                    "-o", exe], check=True)
    for name in ("gh_gemv.hsaco", "gh_kv8.hsaco"):
        (out / name).write_bytes(b"")

    def ask(*args):
        r = subprocess.run([exe, str(out), *[str(a) for a in args]], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stderr
        return r.stdout.split()

    return ask


@pytest.mark.parametrize("before,after", [("none", "none"), ("not_found", "some"), ("invalid", "some")])
def test_errors_of_the_host_stay_pending_and_lookups_leave_none(state, before, after):
    assert state("error", before) == ["0", after]


@pytest.mark.parametrize("pages", [1, 40, 5000, 1 << 20, (1 << 24) + 1, 1 << 28, 1 << 31, 0xffffffff])
@pytest.mark.parametrize("tokens", [0, 1, 100000, 0xffffffff])
def test_parts_count_their_steps_in_32_bits(state, pages, tokens):
    # a token is a 32-bit number, so a table names at most 2^32 of them (a step has 32), whatever its size
    st, parts, chunk = map(int, state("split", pages, tokens))
    most = min(256 * pages, tokens or 1 << 40, (1 << 32) + 1)
    assert st == 0 and 1 <= parts <= 256
    assert chunk >= 1 and parts * chunk <= most // 32 + 1 + parts
