"""Two engines of different widths, each called from a host thread of its own.

The decode kernels take shared memory by the layer's widths, and the bound on it
belongs to the kernel, which both engines launch.  The threads take turns (one
call after the other, the GPU idle between them), so the order is fixed: a wide
layer, a narrow one, the wide one again."""
import threading

import numpy as np
import pytest

from oracle import oracle as O
from tests import helpers

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import doantotnghiepmoe_b200 as M  # noqa: E402
from doantotnghiepmoe_b200 import _lib  # noqa: E402


@pytest.mark.parametrize("path", [_lib.MOE_PATH_DIGITS, _lib.MOE_PATH_GEMV_FUSED,
                                  _lib.MOE_PATH_GEMV_PHASED, _lib.MOE_PATH_TENSOR])
@pytest.mark.parametrize("graphs", [True, False])
def test_wide_layer_after_a_narrow_one_of_another_thread(path, graphs):
    jobs = []
    for j, (H, I) in enumerate([(2048, 1024), (1536, 640)]):
        lw = O.synth_layer(700 + j, 0, H, I, 8, 2, True)
        eng = M.MoeLayerEngine(M.MoeConfig(H, I, 8, 2, True, 3, 1))
        dev = helpers.to_device(lw)
        eng.set_layer_packed(0, *dev)
        eng.set_path(path)
        eng.set_graphs(graphs)
        h = torch.from_numpy(O.synth_hidden(710 + j, 3, H)).cuda()
        ref = O.layer_forward(lw, h.cpu().numpy(), nthreads=8).out
        jobs.append(dict(eng=eng, h=h, out=torch.zeros_like(h), keep=dev, ref=ref))
    torch.cuda.synchronize()
    turns, errors = [threading.Semaphore(1), threading.Semaphore(0)], []

    def work(j, calls):
        for n in range(calls):
            turns[j].acquire()
            job = jobs[j]
            try:
                job["out"].zero_()
                torch.cuda.synchronize()
                job["eng"].forward(0, job["h"], job["out"])
                job["eng"].sync_status()
                if helpers.rel_err(job["out"].cpu().numpy(), job["ref"]) >= 1e-3:
                    errors.append((j, n, "differs"))
            except Exception as ex:
                errors.append((j, n, str(ex)))
            turns[1 - j].release()

    threads = [threading.Thread(target=work, args=a) for a in ((0, 3), (1, 2))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for job in jobs:
        job["eng"].close()
    assert errors == []
