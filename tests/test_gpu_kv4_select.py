"""Choosing pages where the bounds cannot be told apart in fp32: ties and near ties among more
pages than the kernel has threads, queries and summaries at the ends of fp32."""

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as kv4
from tests.test_gpu_kv4 import Case, dev, host, no_device_error, ops  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,grp", [(64, 5), (128, 1), (256, 8)])
@pytest.mark.parametrize("kind", ["equal", "block", "tiny", "subnormal", "huge", "mixed"])
def test_select_among_many_close_pages(ops, dim, grp, kind):
    """More pages about the border than there are threads: equal bounds, a block of equal ones
    across the border, queries too small and summaries too large for the bounds in fp32."""
    rng = np.random.default_rng(dim)
    c = Case(rng, [16 * 600, 16 * 258, 16 * 257 - 3, 16 * 300], 2, dim, 16, garbage=False)
    near, b, hq = c.cache.summary, 4, grp * 2
    q = rng.standard_normal((b, hq * dim)).astype(np.float32)
    if kind == "equal":
        near[:] = near[0]
    elif kind == "block":
        for t in c.table:
            near[t[50:450]] = near[t[50]]
    elif kind == "tiny":
        q *= 1e-35
    elif kind == "subnormal":
        q[:, ::3] *= 1e-42
    elif kind == "huge":
        near[:] = kv4.bf16(np.sort(3e38 * rng.uniform(-1, 1, near.shape), 2))
    else:  # some pages' sums overflow fp32, the others are ordinary
        near[c.table[:, 1:40:3]] *= 1e38
    c.summary = dev(near, torch.bfloat16)
    near[:] = host(c.summary)
    for n_sel in (2, 200, 256, 257, 290):
        for theta in (None, 10000.0):
            want = c.cache.select(q.reshape(b, hq, dim), c.table, c.lens - 1, n_sel, theta)
            got = ops.kv4_select(dev(q), c.summary, c.dtable, c.pos, n_q_heads=hq, page=16, n_sel=n_sel, theta=theta,
                                 **c.heads)
            assert np.array_equal(host(got), want), (n_sel, theta)
