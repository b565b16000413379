"""The ternary linear with adapters over more rows than a grid has in y, where its columns leave the projection to the
kernels that take a row as one."""
import numpy as np
import pytest

import lora_ref as ref
import nlgpu
from test_gpu_lora import Case, close, up

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


@pytest.mark.parametrize("lengths,cols", [([30000, 35535], 8), ([30000, 35536], 8), ([65535, 40, 65535], 72)])
def test_rows_past_65535(lengths, cols):
    c = Case(lengths, list(range(len(lengths))), len(lengths), 8, out=3, cols=cols)
    w = up(nlgpu.pack_ternary(nlgpu.trits(c.out, (c.out, c.cols))))
    x, beta, y = up(c.x), up(np.array([0.03], F32)), up(np.full((c.seq, c.out), np.nan, F32))
    ws = nlgpu.DeviceArray(nlgpu.ternary_linear_lora_workspace(c.seq, c.out, c.cols, c.rmax, len(c.adapter)))
    print(f"[gpu] ternary linear with adapters: {c.seq} rows of {c.cols}", flush=True)
    nlgpu.ternary_linear_lora(x, w, None, beta, up(c.a16), up(c.b16), up(c.scale), up(c.adapter), y, c.seq, c.out, c.cols,
                              c.n, c.rmax, len(c.adapter), ws, start=up(c.start), rank=up(c.rank), fmt=c.fmt)
    nlgpu.sync()
    base = []
    for r in range(0, c.seq, 10000):  # the projection alone, of fewer rows at a time
        part = c.x[r:r + 10000]
        b = nlgpu.DeviceArray(4 * len(part) * c.out)
        nlgpu.ternary_linear(up(part), w, None, beta, b, len(part), c.out, c.cols,
                             workspace=nlgpu.DeviceArray(nlgpu.ternary_linear_workspace(len(part), c.cols)))
        nlgpu.sync()
        base.append(b.download(F32).reshape(-1, c.out))
    want = ref.forward(c.x.astype(float), c.a, c.b, c.scale.astype(float), c.rank, c.of,
                       ref.Sums(np.concatenate(base).astype(float)))[0]
    close(y.download(F32), want, "y")
