import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
try:
    import torch  # noqa: F401  must precede libshodh_hip.so: one HIP runtime per process
except ImportError:
    pass
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


def pytest_sessionstart(session):
    """libshodh_hip.so is (re)built before anything imports the package: importing shodh_memory_amd loads the library and fails loudly
    when it is missing or stale, which is the state of a fresh checkout. The build script is loaded by path for the same reason."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("_shodh_build", os.path.join(ROOT, "shodh_memory_amd", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    b.build()
    global BUILD_MODE
    BUILD_MODE = "libshodh_hip.so: %s" % b.LAST_BUILD_MODE
    # (with -q pytest prints no header: written here AND in the terminal summary, so that the driver's record of the run shows whether this box compiled
    # the library from source or reused the pushed one)
    sys.stderr.write("[conftest] %s\n" % BUILD_MODE)
    sys.stderr.flush()
    install_guard_allocator(b.LIB)


def install_guard_allocator(lib_path):
    """SHODH_GUARD=1|2|3 (csrc/guard.h): the library fences every allocation of its own; here torch's device allocator is replaced by the library's guard
    entry points, so that the tensors the tests hand to the *_device entry points (queries, rows, result buffers) are fenced mappings as well and a kernel
    over-reading a CALLER's buffer faults too. Must happen before the first device allocation of the process."""
    if os.environ.get("SHODH_GUARD", "0") in ("", "0"):
        return False
    import torch
    if not torch.cuda.is_available():
        return False
    alloc = torch.cuda.memory.CUDAPluggableAllocator(lib_path, "shodh_guard_torch_alloc", "shodh_guard_torch_free")
    torch.cuda.memory.change_current_allocator(alloc)
    sys.stderr.write("[conftest] SHODH_GUARD=%s: torch device tensors are fenced mappings too\n" % os.environ["SHODH_GUARD"])
    return True


# with that allocator torch cannot allocate while a stream is captured
needs_capture = pytest.mark.skipif(os.environ.get("SHODH_GUARD", "0") not in ("", "0"), reason="no capture under SHODH_GUARD")

BUILD_MODE = "build not run"


def pytest_report_header(config):
    return BUILD_MODE


def pytest_terminal_summary(terminalreporter, exitstatus, config):
    terminalreporter.write_line("[build] %s" % BUILD_MODE)


def has_gpu():
    try:
        import torch
        return torch.cuda.is_available()
    except Exception:
        return False


@pytest.fixture(scope="session")
def oracle():
    from oracle import oracle as o
    o.build()
    return o
