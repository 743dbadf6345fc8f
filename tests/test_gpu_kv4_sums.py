"""Attention over the 4-bit paged cache where a sum or a scale can go wrong: long sequences of
equal scores, groups of 64 dims of unlike size, values far from zero."""

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as kv4
from tests.test_gpu_kv4 import F32_TOL, Case, close, dev, host, no_device_error, ops  # noqa: F401  (fixtures)

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


@pytest.mark.parametrize("batch", [1, 70])
def test_positions_past_the_planned_length(ops, batch):
    """max_len bounds pos + 1 to the token, not to its tile or page: a position past it is reported
    and left alone, one below it is not touched by that; in a cluster and with tiles dealt out."""
    rng = np.random.default_rng(batch)
    c = Case(rng, [100] * batch, 8, 64, 64)
    q = dev(rng.standard_normal((batch, 8 * 64)))
    call = dict(n_q_heads=8, theta=None, max_len=99)
    for last, bad in ((98, False), (99, True)):
        pos = np.full(batch, 98, np.int32)
        pos[0] = last
        out = torch.full((batch, 512), 3.0, device="cuda")
        ops.kv4_decode(q, c.pool, c.dtable, dev(pos), out=out, out_f32=True, **call, **c.heads)
        assert ops.device_error() == (5 if bad else 0)
        want = c.cache.decode(host(q).reshape(batch, 8, 64), c.table, pos).reshape(batch, -1)
        rest = slice(1 if bad else 0, None)
        close(host(out)[rest], want[rest], F32_TOL)
        assert (out[0] == 3.0).all() or not bad
        sel = ops.kv4_select(q, c.summary, c.dtable, dev(pos), page=64, n_sel=2, **call, **c.heads)
        assert ops.device_error() == (5 if bad else 0)
        assert (sel[0] == -1).all() or not bad


def by_group(x, dim):
    return np.linalg.norm(np.asarray(x, np.float64).reshape(-1, dim // 64, 64), axis=-1)


def decode_by_group(ops, c, grp, seed, tol):
    """Every head's 64 dims on their own: off by tol of their 2-norm at most."""
    b, hq = len(c.lens), grp * c.hkv
    q = np.random.default_rng(seed).standard_normal((b, hq * c.dim)).astype(np.float32)
    ref = c.cache.decode(q.reshape(b, hq, c.dim), c.table, c.lens - 1, 10000.0)
    got = host(ops.kv4_decode(dev(q), c.pool, c.dtable, c.pos, n_q_heads=hq, out_f32=True, **c.heads))
    assert np.isfinite(got).all()
    off, size = by_group(got.reshape(ref.shape) - ref, c.dim), by_group(ref, c.dim)
    worst = (off / np.maximum(size, 1e-300))[size > 0].max()
    assert worst <= tol, f"{worst:.3g} > {tol:.3g}"


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("power", [0, -9, -12, -20, -30])
def test_groups_of_unlike_size(ops, dim, power):
    """V's groups of 64 dims 2^power of one another: each of them as near as one alone is (3
    roundings of 2^-11: q's, the weights', and both in the sum that they are divided by)."""
    rng = np.random.default_rng(dim - power)
    c = Case(rng, [1, 17, 64, 100, 33], 2, dim, 32)
    size = 2.0 ** (power * (np.arange(dim // 64) % 2))
    size[-1] = 2.0 ** power
    c.cache.meta[..., 1, :, :] *= size[:, None, None]
    c.pool = dev(c.cache.pool())
    decode_by_group(ops, c, 4, 1, F32_TOL)


@pytest.mark.parametrize("dim", [128, 256])
def test_groups_whose_size_changes(ops, dim):
    """Groups that are small at first and large later, or the other way round, or in one page
    alone, in sequences that one warp reads whole and that many share."""
    rng = np.random.default_rng(dim)
    c = Case(rng, [900, 64, 16, 500], 2, dim, 16, garbage=False)
    for b, n in enumerate(c.lens):
        pages = -(-int(n) // 16)
        for i, at in enumerate(c.table[b, :pages]):
            for g in range(dim // 64):
                power = [(-25, 0), (0, -25), (0, 0), (-25, 12)][(b + g) % 4][int(2 * i >= pages)]
                c.cache.meta[at, :, :, g, 1] *= 2.0 ** power
    c.pool = dev(c.cache.pool())
    decode_by_group(ops, c, 3, 2, F32_TOL)


@pytest.mark.parametrize("dim", [64, 128])
def test_constant_values(ops, dim):
    """Tokens whose values are all alike have the least step, 2^-40, however large they are."""
    rng = np.random.default_rng(dim)
    c = Case(rng, [40, 17, 300], 2, dim, 16, garbage=False)
    c.cache.meta[..., 0, 1, :, 0] = 2.0 ** -40
    c.cache.meta[..., 0, 1, :, 1] = kv4.bf16(1e17 * (1 + rng.random(c.cache.meta.shape[:3] + (16,))))
    c.pool = dev(c.cache.pool())
    decode_by_group(ops, c, 2, 3, F32_TOL)


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("each", ["group", "page"])
def test_groups_of_unlike_size_in_shared_pairs(ops, dim, each):
    """The same with every pair's tiles dealt over several CTAs, in full stages, whose parts are
    joined; one group small throughout, or every page's groups of a size of their own."""
    rng = np.random.default_rng(dim + 1)
    c = Case(rng, rng.integers(1, 700, 150), 2, dim, 64, garbage=False)
    if each == "group":
        power = -18.0 * (np.arange(dim // 64) % 2)
    else:
        power = rng.choice([0, -18, -30, 10], (len(c.cache.meta), 1, 1, dim // 64))
    c.cache.meta[..., 1, :, :] *= 2.0 ** power[..., None, None]
    c.pool = dev(c.cache.pool())
    decode_by_group(ops, c, 2, 4, F32_TOL)


@pytest.mark.parametrize("power", [0, -20])
def test_nan_with_groups(ops, power):
    """A NaN key spoils its own sequence and kv head, a NaN value its own 64 dims; nothing else."""
    rng = np.random.default_rng(power + 30)
    c = Case(rng, [70, 70, 70], 2, 128, 16)
    c.cache.meta[..., 1, 1, :, :] *= 2.0 ** power
    c.cache.meta[c.table[0, 1], 0, 0, 1, 0, 3, 1] = np.nan
    c.cache.meta[c.table[1, 3], 1, 0, 1, 1, 9, 1] = np.nan
    c.pool = dev(c.cache.pool())
    q = rng.standard_normal((3, 4 * 128)).astype(np.float32)
    ref = c.cache.decode(q.reshape(3, 4, 128), c.table, c.lens - 1).reshape(3, 2, 2, 2, 64)
    got = host(ops.kv4_decode(dev(q), c.pool, c.dtable, c.pos, n_q_heads=4, theta=None, out_f32=True,
                              **c.heads)).reshape(ref.shape)
    assert np.isnan(got[0, 0]).all() and np.isnan(got[1, 1, :, 1]).all()
    ok = np.isfinite(ref)
    assert np.isfinite(got[ok]).all() and ok.sum() == ref.size - 2 * 128 - 2 * 64
    off, size = by_group(np.where(ok, got - ref, 0.0), 64), by_group(np.where(ok, ref, 0.0), 64)
    assert (off <= F32_TOL * size).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_scores_that_jump(ops, dim):
    """Scores of thousands that rise and fall between pages while the groups' sizes change: only the
    page of the largest score counts, whatever was summed before it."""
    rng = np.random.default_rng(dim)
    c = Case(rng, [16 * 40, 16 * 40], 1, dim, 16, garbage=False)
    c.cache.meta[..., 0, :, 0] = 2.0 ** -40
    for b in range(2):
        for i, at in enumerate(c.table[b, :40]):
            c.cache.meta[at, ..., 0, :, 1] = [-4.0, 0.5, 2.0, 1.0][i % 4] * (1 + (i == (37 if b else 4)))
            c.cache.meta[at, :, :, :, 1] *= 2.0 ** rng.choice([0, -25, 20, -35], (1, 1, dim // 64, 1, 1))
    c.pool = dev(c.cache.pool())
    q = 1 + np.abs(np.random.default_rng(1).standard_normal((2, 2 * dim))).astype(np.float32)
    for scale in (100.0, -100.0):
        ref = c.cache.decode(q.reshape(2, 2, dim), c.table, c.lens - 1, None, scale)
        got = host(ops.kv4_decode(dev(q), c.pool, c.dtable, c.pos, n_q_heads=2, theta=None, scale=scale, out_f32=True,
                                  **c.heads))
        off, size = by_group(got.reshape(ref.shape) - ref, dim), by_group(ref, dim)
        assert (off <= F32_TOL * size).all(), (scale, (off / size).max())
