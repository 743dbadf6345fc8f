"""Attention over the 4-bit paged cache where a sum or a scale can go wrong: long sequences of
equal scores, groups of 64 dims of unlike size, values far from zero."""

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as kv4
from tests.test_gpu_kv4 import dev, host, no_device_error, ops  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("steps", ["two", "any"])
def test_long_sequences_of_equal_scores(ops, steps):
    """32768 tokens of equal weight, whose values are around zero: what a sum loses each time adds
    up (steps of any size), or a weight's rounding that is the same for many tokens (steps of 1
    and 137 / 128: the fp16 weight of the former is 0.46 of a unit off).

    Neighbours have one step e and the codes n and 15 - n, so that the roundings of their weights
    cancel.  Bounds, in the largest e and per token: a tensor-core sum of 16 products is off by
    2^-22 of its terms' sizes (16 x 255 / 16 and half as much carried in, for the sums of two
    codes; a sixteenth for those of one): 25 x 2^-22.  The fp32 sums of offsets add 4 terms per
    tile and lane, each rounded by 2^-24 of a running sum of up to 16 + 256 in the 256 tiles of a
    warp (f = -8 e, half a step from the middle): 272 x 2^-24.  Weights and their sum are off by
    2^-22 and 512 x 2^-24 of that half step: 260 x 2^-24."""
    n, page, hkv, batch = 32768, 64, 2, 128
    rng = np.random.default_rng(1)
    c = kv4.Cache(n // page, hkv, 64, page)
    c.code[:] = rng.integers(0, 16, c.code.shape)
    c.code[..., 1::2, :] = 15 - c.code[..., 0::2, :]
    step = np.ones(c.meta.shape[:-2] + (8,))
    if steps == "two":
        step[..., 1::2] = 137 / 128
    else:
        step *= rng.integers(128, 256, step.shape) / 128
    step = step.repeat(2, -1)
    c.meta[..., 0], c.meta[..., 1] = step, -8 * step
    tol = step.max() * (4 * 25 + 272 + 260) * 2.0 ** -24
    want = c.values(1, np.arange(n // page)).mean(1).reshape(-1)
    table = np.tile(np.arange(n // page, dtype=np.int32), (batch, 1))
    got = ops.kv4_decode(torch.zeros(batch, hkv * 64, device="cuda"), dev(c.pool()), dev(table),
                         dev(np.full(batch, n - 1, np.int32)), n_q_heads=hkv, n_kv_heads=hkv, head_dim=64, theta=None,
                         out_f32=True)
    off = np.abs(host(got) - want).max()
    assert off <= tol, f"{off:.3g} > {tol:.3g}"
