"""Losses over more rows than a launch has workgroups of 1,024 threads for: rows that repeat, whose outputs then do too."""
import numpy as np
import pytest

import nlgpu
from test_gpu_loss import Case, check

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


def test_four_million_rows_of_many_targets():
    part, times = 4096, 1024
    c = Case(part, 300, 64, top=17, tau=2.0, per_row=True, bias=True)
    want = c.call()  # of the rows once
    check(c, want)
    rows = part * times
    d = {}
    for k in ("x", "index", "teacher", "dloss"):
        a = getattr(c, k)
        d[k] = nlgpu.DeviceArray(a.nbytes * times)
        for i in range(times):
            d[k].upload(a, i * a.nbytes)
    words, bias, beta = (nlgpu.to_device(a) for a in (c.words, c.bias, c.beta))
    loss, lse, dx = (nlgpu.to_device(np.full(rows * n, np.nan, F32)) for n in (1, 1, c.cols))
    need = nlgpu.ternary_distill_workspace(rows, c.vocab, c.cols, c.top, True)
    assert need
    print(f"[gpu] distillation: {rows} rows of {c.top} targets", flush=True)
    nlgpu.ternary_distill(d["x"], words, bias, beta, d["index"], d["teacher"], c.top, c.tau, loss, lse, rows, c.vocab, c.cols,
                          nlgpu.DeviceArray(need), dx=dx, dloss=d["dloss"], beta_per_row=True)
    nlgpu.sync()
    bits = lambda a: a.view(np.uint32)  # noqa: E731
    for got, w in ((loss, want[0]), (lse, want[1])):
        assert (got.download(np.uint32).reshape(times, part) == bits(w)).all()
    for i in (0, 1, times // 2, times - 1):
        # (more parts of the vocabulary may be summed where there are few rows: two bounds apart at most)
        got = dx.download(F32, part * c.cols, 4 * i * part * c.cols).reshape(part, c.cols)
        check(c, (None, None, got))
