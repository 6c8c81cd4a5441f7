"""Shared pytest configuration.

Markers:
  gpu   - needs an MI355X (HIP device); the driver runs ``pytest -m gpu`` on a GPU box and ``-m "not gpu"`` on CPU.
  slow  - multi-second end-to-end scenarios (still part of the default CPU run).
"""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
os.environ.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
# a crash inside the library prints the faulting thread's native frames before Python's faulthandler runs (and
# SIGUSR2 dumps every thread of a hung test); the library reads this when it initialises
os.environ.setdefault("PCCL_DEBUG_BACKTRACE_SIGNAL", "1")
os.environ["PYTHONPATH"] = ROOT + os.pathsep + os.environ.get("PYTHONPATH", "")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: test needs an MI355X GPU (HIP backend)")
    config.addinivalue_line("markers", "slow: long-running end-to-end scenario")


@pytest.fixture(scope="session")
def hip():
    """Skips unless a HIP device is present *and* the HIP plugin is loaded (fails loudly if the plugin is missing)."""
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from pccl_amd.ops import kernels as K
    assert K.hip_device_count() > 0, "GPU present but libpccl_hip.so did not load"
    return torch.device("cuda:0")


# GPU tests whose subject is device memory that another process maps (the xGMI path between processes, the shared
# state's hand-off): by file, test, and the parameters of those cases where others do without
NEEDS_MAPPED_SHARES = {
    "test_benchmarks.py": {"test_basic_reduce": ["cuda:0"], "test_fault_tolerance": ["cuda:0-ipc"],
                           "test_py_latency": ["cuda:0"]},
    "test_fault_tolerance.py": {"test_gpu_ipc_sigkill_mid_op": None, "test_gpu_ipc_sigkill_after_local_success": None,
                                "test_gpu_ipc_sigkill_many_threads_restore_is_final": None,
                                "test_gpu_ipc_quarantine_reclaimed_on_unchanged_ring": None,
                                "test_gpu_shared_state_distributor_sigkill_mid_handoff": None},
    "test_gpu_allreduce.py": {"test_two_process_ipc": ["zero_copy-safe", "inplace-safe", "mixed-safe", "shareable-safe",
                                                       "shareable-fast", "shareable_inplace-safe",
                                                       "shareable_inplace-fast"],
                              "test_ipc_preflight_rehearsal": None, "test_two_process_ipc_large": None},
    "test_hierarchical.py": {"test_hierarchical_device": None, "test_hierarchical_inplace_mixed_bf16": None,
                             "test_hierarchical_quantized_inter_host": None,
                             "test_peer_crash_with_host_layout": ["cuda:0"]},
    "test_liveness.py": {"test_gpu_sigstopped_peer_ipc": None},
}
_mapping_refused = None


def mapping_refused() -> str:
    """What a joiner of another process says when it cannot map the device memory handed to it; "" where it can. Tried
    once a session, with the library's own shared state (which then arrives over TCP)."""
    global _mapping_refused
    if _mapping_refused is None:
        import subprocess
        import time

        from pccl_amd.utils import DIAG_SIGNALS, communicate_all, local_master, spawn_python
        worker = os.path.join(ROOT, "tests", "workers", "ss_peer.py")
        with local_master() as addr:
            ps = []
            for role in ("dist", "dist", "join"):
                if role == "join":  # the two that have the state are there first, and take the joiner in
                    time.sleep(2.0)
                ps.append(spawn_python([worker, addr, role, "--n", "5000", "--no-all-reduce"],
                                       env={"PCCL_LOG_LEVEL": "WARN"}, stdout=subprocess.PIPE, stderr=subprocess.PIPE,
                                       text=True))
            said = communicate_all(ps, 60, DIAG_SIGNALS)[2][1]
        _mapping_refused = next((line[line.index("cannot be mapped"):] for line in said.splitlines()
                                 if "cannot be mapped" in line), "")
    return _mapping_refused


def pytest_runtest_setup(item):
    cases = NEEDS_MAPPED_SHARES.get(os.path.basename(str(item.fspath)), {})
    name = getattr(item, "originalname", item.name)
    if item.get_closest_marker("gpu") is None or name not in cases:
        return
    if cases[name] is not None and item.callspec.id not in cases[name]:
        return
    import torch
    if torch.cuda.is_available() and mapping_refused():
        pytest.skip("device memory of another process " + mapping_refused())
