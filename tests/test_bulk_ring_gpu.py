"""A ring whose wait runs out (bulk_ring_probe.cu, built here): the status word is set, nothing is copied afterwards, and the CTA
leaves within a bound and with the copies that were on their way in place. No fault is involved: the wait has a limit of 20 ms."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from cgpt_b200 import build

THREADS, STEPS = 64, 7


@pytest.mark.gpu
def test_a_wait_that_runs_out(tmp_path):
    so = tmp_path / "probe.so"
    source = Path(__file__).with_name("bulk_ring_probe.cu")
    made = subprocess.run([build._nvcc(), *build.ARCH_FLAGS, *build.COMMON, "-shared", "-o", str(so), str(source)], capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    probe = ctypes.CDLL(str(so))
    given = torch.arange(2 * 3 * THREADS, dtype=torch.int32, device="cuda")
    report = torch.zeros(probe.report_words(), dtype=torch.int32, device="cuda")
    assert probe.run_probe(ctypes.c_void_p(given.data_ptr()), ctypes.c_void_p(report.data_ptr()), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    status, armed, refused, failed, late, *rest = report.tolist()
    assert status == 5 and late == 0
    assert failed == THREADS                       # stage 2 is never filled: every thread gives up there
    assert armed == 4 and refused == STEPS - 2     # two stages at first, each refilled once; nothing after the failure
    assert rest[:STEPS] == [0, 0, 3, 1, 2, 3, 1]   # given up at stage 2; the stages still go round
    seen, landed = torch.tensor(rest[STEPS:STEPS * (1 + THREADS)]).view(STEPS, THREADS), torch.tensor(rest[STEPS * (1 + THREADS):]).view(2, THREADS)
    want = given.cpu().view(6, THREADS)
    assert torch.equal(seen[:2], want[:2].long()) and torch.equal(landed, want[2:4].long())
