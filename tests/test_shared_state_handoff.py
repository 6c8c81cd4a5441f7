"""The same-host hand-off of the shared state between processes on the host-emulated device backend
(csrc/testing/hostdev_backend.cpp), whose shareable memory is a shared memory file (PCCL_HOSTDEV_VMM): entries arrive
through the joiner's mapping, and over TCP where the mapping is refused."""
import json
import os
import subprocess
import time

import pytest

from pccl_amd.utils import DIAG_SIGNALS, communicate_all, local_master, spawn_python

HERE = os.path.dirname(os.path.abspath(__file__))
HOSTDEV = os.environ.get("PCCL_TEST_HOSTDEV") or os.path.join(os.path.dirname(HERE), "pccl_amd", "lib",
                                                              "libpccl_hostdev.so")


@pytest.mark.parametrize("extra_tensors", [0, 40])
@pytest.mark.parametrize("importing", [True, False])
def test_handoff(importing, extra_tensors):
    if not os.path.exists(HOSTDEV) or os.environ.get("PCCL_DISABLE_HIP") == "1":
        pytest.skip("libpccl_hostdev.so not built, or device plugins disabled (PCCL_DISABLE_HIP)")
    worker, n = os.path.join(HERE, "workers", "ss_peer.py"), 300_001
    args = ["--device", "cpu", "--n", str(n), "--extra-tensors", str(extra_tensors), "--no-all-reduce"]
    env = {"PCCL_HIP_PLUGIN": HOSTDEV, "PCCL_HOSTDEV_ALL_DEVICE": "1", "PCCL_DISABLE_IPC": "1", "PCCL_HOSTDEV_VMM": "1",
           "PCCL_LOG_LEVEL": "WARN"}
    with local_master() as addr:
        ps = [spawn_python([worker, addr, "dist", *args], env=env, stdout=subprocess.PIPE, stderr=subprocess.PIPE,
                           text=True) for _ in range(2)]
        time.sleep(1.0)
        ps.append(spawn_python([worker, addr, "join", *args], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True,
                               env=env if importing else dict(env, PCCL_HOSTDEV_VMM="no_import")))
        outs = communicate_all(ps, 120, DIAG_SIGNALS)
    assert [p.returncode for p in ps] == [0, 0, 0], [o[1][-2000:] for o in outs]
    *given, got = (next(json.loads(x) for x in out.splitlines() if x.startswith("{")) for out, _ in outs)
    size = 4 * (n + sum(1 + (k * 997) % 50000 for k in range(extra_tensors)))
    assert "error" not in got, (got, outs[2][1][-2000:])
    assert got["lo"] == got["hi"] == 7.0 and got["extra_ok"] and got["revision"] == 5 and got["rx"] == size
    assert sum(g["tx"] for g in given) == size
    assert ("cannot be mapped (emulated refusal)" in outs[2][1]) == (not importing), outs[2][1][-2000:]
