"""The status word of the attention with changed scores: a wait that ran out is told once, and calls after it are as calls before it."""
import ctypes
import os
import subprocess
import sys
import time

import pytest
import torch

pytestmark = pytest.mark.gpu

from fsa import _lib

DEV = "cuda:0"


def read():
    st = ctypes.c_int(-1)
    assert _lib.lib().fsa_biased_read_status(ctypes.byref(st)) == 0
    return st.value


def seconds(stream=None):
    """A wait that runs out: how long it took."""
    torch.cuda.synchronize()
    t = time.perf_counter()
    assert _lib.lib().fsa_biased_debug_wait_timeout(stream.cuda_stream if stream else _lib.current_stream(torch.device(DEV))) == 0
    torch.cuda.synchronize()
    return time.perf_counter() - t


def test_reading_clears():
    torch.zeros(1, device=DEV)
    read()
    first, second = seconds(), seconds()        # 400e6 and 6.25e6 cycles: 0.2 s and 3 ms at 1.965 GHz
    assert first > 0.19 and second < 0.1, (first, second)
    assert read() == 1 and read() == 0
    assert seconds() > 0.19 and read() == 1 and read() == 0


def test_waits_are_as_long_as_ever_some_seconds_later():
    torch.zeros(1, device=DEV)
    read()
    assert seconds() > 0.19 and seconds() < 0.1
    time.sleep(2.5)                             # (two units of 2^30 ns)
    assert seconds() > 0.19
    assert read() == 1


def test_a_failure_on_another_stream_is_read():
    torch.zeros(1, device=DEV)
    read()
    side = torch.cuda.Stream()
    assert _lib.lib().fsa_biased_debug_wait_timeout(side.cuda_stream) == 0
    assert read() == 1                          # (waits for it)


SCRIPT = """
import torch
from fsa import _lib
from fsa.ops import biased_attention
from fsa_preview.ops import biased_decode_attention
x = [torch.randn(70, 2, 64, device="cuda").bfloat16().requires_grad_() for _ in range(3)]
cu = torch.tensor([0, 70], dtype=torch.int32, device="cuda")
n = torch.tensor([70], dtype=torch.int32, device="cuda")
def train():
    o, _ = biased_attention(*x, cu, softcap=5.0)
    torch.autograd.grad(o.float().sum(), x)
def decode():
    biased_decode_attention(x[0][-1:].detach(), x[1].detach(), x[2].detach(), n, n * 0, max_len=70, softcap=5.0)
for call in (train, decode):
    call()
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        assert _lib.lib().fsa_biased_debug_wait_timeout(stream.cuda_stream) == 0
        with torch.cuda.stream(stream):
            try:
                call()
                print("silent")
            except RuntimeError as e:
                print("raised", "status" in str(e))
            call()
            print("fine")
"""


def test_with_status_checks_a_failure_is_raised_once():
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "flash-sparse-attention_b200")
    r = subprocess.run([sys.executable, "-c", SCRIPT], env={**os.environ, "FSA_CHECK_STATUS": "1", "PYTHONPATH": root}, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.split("\n")[:-1] == ["raised True", "fine"] * 4, r.stdout + r.stderr[-2000:]
