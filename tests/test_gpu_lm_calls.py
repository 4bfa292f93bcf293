"""How the language-model operators are called: errors inside a backward pass, calls of several
host threads and from threads that have not used the device before."""
import ctypes
import os
import subprocess
import sys
import textwrap
import threading

import pytest
import torch

from conftest import REPO

pytestmark = pytest.mark.gpu


def _child(code, **env):
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], cwd=REPO, env=dict(os.environ, **env),
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, (r.returncode, r.stdout, r.stderr)


@pytest.mark.parametrize("call", ["gated_scan(a, a)[0]", "gated_ffn(a, w)"])
def test_an_error_in_a_backward_pass_raises(call, tmp_path):
    """The C call refuses (a library loaded in front of the package's own): autograd's thread, which does
    not hold Python's lock, hands the error on."""
    src, refuse = tmp_path / "refuse.c", tmp_path / "librefuse.so"
    src.write_text("int dg_gated_scan_backward(void) { return -2; }\nint dg_gated_ffn_backward(void) { return -2; }\n")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(refuse), str(src)], check=True)
    _child(f"""
        import torch
        from deltagrid_b200._lib import DeltaGridError
        from deltagrid_b200.ffn import gated_ffn
        from deltagrid_b200.recurrence import gated_scan
        a = torch.ones(2, 4, 8, device="cuda", requires_grad=True)
        w = torch.ones(16, 8, device="cuda")
        y = {call}
        torch.cuda.synchronize()
        for _ in range(3):
            try:
                y.sum().backward(retain_graph=True)
            except DeltaGridError as e:
                assert "backward failed: unsupported" in str(e), e
            else:
                raise SystemExit("no error")
        print("done")
        """, LD_PRELOAD=str(refuse))


def test_the_first_work_of_a_thread():
    """Tensor-core calls on threads that have made no CUDA call before: autograd's, in a backward pass, and a
    new one of the host's."""
    _child("""
        import threading
        import torch
        from deltagrid_b200.ffn import gated_ffn
        x = torch.randn(200, 64, device="cuda").bfloat16().requires_grad_(True)
        w = torch.randn(128, 64, device="cuda").bfloat16()
        dh = torch.randn(200, 64, device="cuda").bfloat16()
        h = gated_ffn(x, w)
        spare = [torch.empty(1 << 20, device="cuda") for _ in range(4)]      # memory the backward pass finds cached
        torch.cuda.synchronize()
        del spare
        torch.autograd.grad(h, [x], dh)
        got = []
        t = threading.Thread(target=lambda: got.append(gated_ffn(x.detach(), w)))
        t.start()
        t.join()
        assert len(got) == 1 and torch.equal(got[0], h)
        print("done")
        """)


def test_calls_of_two_host_threads():
    """Launches of one kernel that take little and much shared memory, from two threads through the C ABI."""
    from deltagrid_b200 import _lib
    L, F, bad = _lib.lib(), ctypes.c_float, []

    def worker(V, n):
        torch.cuda.set_device(0)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            logits, u = torch.zeros(1, V, device="cuda"), torch.zeros(1, device="cuda")
            token = torch.zeros(1, device="cuda", dtype=torch.int64)
            s.synchronize()
            for _ in range(n):
                rc = L.dg_sample(0, 1, V, logits.data_ptr(), V, u.data_ptr(), None, F(1.0), None, 0, None, F(1.0), None,
                                 F(0.0), token.data_ptr(), None, s.cuda_stream)
                if rc:
                    bad.append((V, rc, L.dg_last_cuda_error()))
            s.synchronize()

    ts = [threading.Thread(target=worker, args=(v, 4000)) for v in (8192, 200000)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad, (len(bad), bad[0])


def test_first_calls_of_many_threads():
    """Forward and backward passes of several threads at once, none of which has called the package before."""
    _child("""
        import threading
        import torch
        from deltagrid_b200.ffn import gated_ffn
        from deltagrid_b200.recurrence import gated_scan
        from deltagrid_b200 import hsru_delta_cuda as ext
        torch.zeros(1, device="cuda")
        gate, got = threading.Barrier(8), []

        def worker():
            torch.manual_seed(0)
            a = torch.randn(2, 40, 16, device="cuda", requires_grad=True)
            w = torch.randn(32, 16, device="cuda", requires_grad=True)
            torch.cuda.synchronize()
            gate.wait()
            for _ in range(20):
                g = torch.autograd.grad(gated_ffn(gated_scan(a, a)[0], w).sum(), [a, w])
            torch.cuda.synchronize()
            got.append([t.cpu() for t in g])

        ts = [threading.Thread(target=worker) for _ in range(8)]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
        assert len(got) == 8 and ext.device_status() == 0
        print("done")
        """)


def test_a_first_call_in_inference_mode():
    """The status word of a device is an ordinary tensor, whatever mode its first call was made in."""
    _child("""
        import torch
        from deltagrid_b200.ffn import gated_ffn
        from deltagrid_b200 import hsru_delta_cuda as ext
        with torch.inference_mode():
            gated_ffn(torch.ones(4, 8, device="cuda"), torch.ones(16, 8, device="cuda"))
        assert ext.device_status() == 0
        print("done")
        """)
