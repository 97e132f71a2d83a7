"""Calls of several host threads at a time, each on a stream of its own, in a process that has met none of the kernels before."""
import subprocess
import sys

import pytest

import conftest

pytestmark = pytest.mark.gpu

CODE = """
import sys; sys.path[:0] = ["tests", "."]
import threading
import torch, __graft_entry__ as e
from test_w4_gpu import make, reference, check
from test_block_norm_gpu import inputs, reference as norm_reference, check as norm_check
from pages_helpers import Device, Model
pkg = e.load_package()
sizes = [(r, d_in, d_out, g) for r, d_in, d_out, g in ((1, 4096, 512, 128), (12, 2048, 8192, 64), (64, 4096, 8192, 32), (30, 8192, 2048, 128), (8, 1024, 9600, 64), (48, 1024, 16500, 64))]
w4 = [make(*s[:3], s[3], True, i) for i, s in enumerate(sizes)]
norms = [(d, inputs(50, d, torch.float16, torch.float16, False, d)) for d in (64, 1000, 4096, 2049, 20000)]
torch.cuda.synchronize()
start, failed = threading.Barrier(4), []

def work(n):
    try:
        stream = torch.cuda.Stream()
        model = Model(200, 16, 9, 6)
        device = Device(pkg, 200, 16, 9, 6, seed=n)
        device.load(model)
        got = []
        outs = [(a[0].shape[0], torch.zeros(a[0].shape[0], a[1].shape[0], dtype=torch.float16, device="cuda")) for a in w4]
        news, gone = [[(3 * i + n) % 40 for i in range(9)], [1] * 9], [[0, 3], [1, n]]
        lists = [(device.starts(new), device.ints(*g)) for new, g in zip(news, gone)]
        torch.cuda.synchronize()
        start.wait()
        for i in range(len(w4)):
            k = (i + n) % len(w4)
            pkg.project_w4(w4[k][0], pkg.w4_weight(*w4[k][1:]), outs[k][1], outs[k][0], stream=stream)
        for k in range(len(norms)):
            d, (x, y, g, *w) = norms[(k + n) % len(norms)]
            bp = pkg.block_norm_params(d, post=True, gate=pkg.GATE_SIGMOID)
            x_out, h = torch.empty_like(x), torch.empty_like(x)
            stream.wait_stream(torch.cuda.current_stream())
            pkg.block_norm(x, y, x_out, h, 50, bp, g, *w, stream=stream)
            got.append((bp, (x, y, g, *w), x_out, h))
        for new, g, (starts, seqs) in zip(news, gone, lists):
            pkg.pages_take(device.pool, starts, device.ws, stream=stream)
            pkg.pages_free(device.pool, seqs, stream=stream)
            model.take(new); model.free(g)
        torch.cuda.synchronize()
        device.same(model)
        for a, (_, out) in zip(w4, outs):
            check(out, *reference(*a, torch.float16))
        for bp, args, x_out, h in got:
            r, tr, hr, th = norm_reference(pkg, bp, *args)
            norm_check(x_out, r, tr, "x_out"); norm_check(h, hr, th, "h")
    except BaseException as error:
        failed.append(repr(error))
        start.abort()
threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
[t.start() for t in threads]; [t.join() for t in threads]
assert not failed, failed
assert pkg.kernel_status()[0] == 0
"""


def test_threads_that_meet_the_kernels_together(torch_cuda):
    r = subprocess.run([sys.executable, "-c", CODE], cwd=conftest.ROOT, capture_output=True, text=True, timeout=250)
    assert r.returncode == 0, r.stderr[-2000:]
