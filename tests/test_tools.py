"""What the measuring tools under tools/ must not do.  CPU only: the sources
are read, nothing of them is run."""
import glob
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOOLS = os.path.join(ROOT, "tools")
REGISTERS = re.compile(r"\b(?:hip|cuda)HostRegister\s*\(")


def sources(*patterns):
    return sorted(f for p in patterns for f in glob.glob(os.path.join(TOOLS, p)))


def text(path):
    with open(path) as f:
        return f.read()


def test_no_tool_disturbs_a_live_registration():
    """Five GPU faults of unproven cause followed the registration of memory
    that the runtime also copied as pageable, or that was freed and used again.
    No tool brings such a history about: none that registers existing memory
    copies other parts of it through the runtime, or moves its pages."""
    disturbs = re.compile(r"MADV_COLLAPSE|torch\.from_numpy")
    assert sources("*.py")
    found = [os.path.basename(f) for f in sources("*.py") if REGISTERS.search(text(f)) and disturbs.search(text(f))]
    assert found == []


def test_no_script_registers_existing_memory():
    """Page-locked memory is allocated (rs_host_alloc, torch's pin_memory);
    memory that exists already is never registered in place, not for a rate
    either: every recorded fault followed such a call."""
    assert [os.path.basename(f) for f in sources("*.py") if REGISTERS.search(text(f))] == []


def test_no_native_tool_registers_existing_memory():
    """The same for the compiled probes: hipHostMalloc is their only pinned memory."""
    native = sources("*.hip", "*.cpp", "*.c", "*.hpp")
    assert native
    assert [os.path.basename(f) for f in native if REGISTERS.search(text(f))] == []


def test_cpp_tools_compile_against_this_tree():
    """A C++ tool that no longer fits the library's sources is dead code."""
    csrc = os.path.join(ROOT, "java-reed-solomon-distributed-file-system_amd", "csrc")
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    assert sources("*.cpp")
    for f in sources("*.cpp"):
        p = subprocess.run(["g++", "-std=c++17", "-fsyntax-only", "-D__HIP_PLATFORM_AMD__", "-I", csrc,
                            "-I", os.path.join(rocm, "include"), f], capture_output=True, text=True)
        assert p.returncode == 0, f"{os.path.basename(f)}:\n{p.stderr[:2000]}"


def test_runner_leaves_no_progress_of_its_own():
    """gpu_run.sh's steps show their own progress; a loop beside them would
    make a hung step look alive."""
    for f in sources("*.sh"):
        assert not re.search(r"while\s+(true|:)|heartbeat", text(f)), os.path.basename(f)
