"""Training operators called by two host threads at once, each on its own stream."""
import threading

import pytest
import torch

from opendde_b200 import _abi, kernels
from test_gpu_train_ops import _att, _rand
from train_ops_support import token_ids

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _attention(nk, dtype, device):
    q, k, v, do, bias, _ = _att(8, 33, nk, 2, 2, 32, dtype, device, "shared", dtype)
    o, saved = kernels.attention(q, k, v, bias, save=True)
    return lambda: kernels.attention_bwd(do, q, k, v, o, saved, bias, need=(True, False, False, True))[::3]


def _layernorm(c, dtype, device):
    x, dy = _rand((40, c), dtype, device, 1), _rand((40, c), dtype, device, 2)
    return lambda: kernels.layernorm_bwd(x, dy, None)


def _relpos(r_max, dtype, device):
    ids, g = token_ids(50, 2, device), _rand((4, 50, 50), dtype, device, 3)
    return lambda: (kernels.relpos_bias_bwd(g, ids, 0, 0, r_max, 2),)


class _Recorder:
    """The library, with the last call of each entry point kept."""

    def __init__(self, lib):
        self.lib, self.last = lib, None

    def __getattr__(self, name):
        def call(*args):
            self.last = getattr(self.lib, name), args
            return self.last[0](*args)
        return call


def _record(rec, call):
    got = call()
    return (*rec.last, got)


@pytest.mark.parametrize("make,dtype,sizes", [(_attention, BF16, (810, 30)), (_attention, F32, (500, 30)),
                                              (_layernorm, F32, (1021, 833)), (_layernorm, BF16, (1016, 800)),
                                              (_relpos, F32, (110, 70))])
def test_two_threads_with_different_sizes(make, dtype, sizes, cuda_device, monkeypatch):
    """The same kernels with much and little shared memory, launched from two threads as fast as they can: each call
    as the wrapper made it once, over buffers of its own."""
    kept, jobs = [], []
    lib, workspace = _abi.load(), kernels.workspace
    monkeypatch.setattr(kernels, "workspace", lambda *a: kept.append(workspace(*a)) or kept[-1])
    for n in sizes:
        call = make(n, dtype, cuda_device)
        want = call()
        torch.cuda.synchronize()
        rec = _Recorder(lib)
        with torch.cuda.stream(torch.cuda.Stream()), monkeypatch.context() as m:
            m.setattr(_abi, "load", lambda rec=rec: rec)
            jobs.append((*_record(rec, call), want, call))
    torch.cuda.synchronize()
    status = [set(), set()]

    def work(i):
        fn, args = jobs[i][:2]
        with torch.cuda.device(cuda_device):
            for _ in range(4000):
                status[i].add(fn(*args))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert status == [{0}, {0}]
    for _, _, got, want, _ in jobs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
