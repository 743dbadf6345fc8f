"""Q4Decoder with its K and V in 4-bit pages, and Kv4Cache, on the GPU: the cache and the
attention of a step against the oracle on the step's own projections, GEMV and GEMM batches,
captured steps, and rows that fork and end."""

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as kv4
from tests.test_gpu_kv4 import BF16_TOL, F32_TOL, close, dev, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mod():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from llmnputest_b200 import decode, kv4 as kv4_mod, ops
    return decode, kv4_mod, ops


@pytest.mark.parametrize("batch,page", [(1, 16), (3, 64), (12, 32)])
def test_decoder_step(mod, batch, page):
    decode, _, ops = mod
    cfg = decode.DecoderConfig(n_layers=1, hidden=512, n_heads=8, n_kv_heads=2, intermediate=512, vocab=1024)
    ctx = 100
    dec = decode.Q4Decoder(cfg, batch, ctx, seed=5, kv_cache="kv4", kv_page=page)
    rng = np.random.default_rng(batch)
    start = rng.integers(0, ctx - 4, batch)
    ref = kv4.Cache.of(host(dec.cache.pool[0]), 64)
    table = host(dec.cache.table)
    assert sorted(table.reshape(-1)) == list(range(batch * -(-ctx // page)))
    graph = None
    for step in range(4):
        pos = start + step
        dec.x_in.copy_(dev(rng.standard_normal((batch, cfg.hidden))))
        dec.pos.copy_(dev(pos.astype(np.int32)))
        if step < 2:
            dec.step()
        else:  # the same step captured
            if graph is None:
                graph = dec.capture()
            graph.replay()
        qkv = host(dec.qkv)
        ref.append(qkv[:, 512:640], qkv[:, 640:], table, pos, None, cfg.rope_theta)
        assert np.array_equal(host(dec.cache.pool[0]), ref.pool()), step
        want = ref.decode(qkv[:, :512].reshape(batch, 8, 64), table, pos, cfg.rope_theta)
        close(host(dec.attn), want.reshape(batch, -1), BF16_TOL, f"step {step}")
        assert torch.isfinite(dec.logits).all()
    assert ops.device_error() == 0
    assert dec.bytes_per_step([10]) - dec.bytes_per_step([0]) == 10 * 2 * 64 * 9 // 8
    del graph


def test_decoder_near_the_dense_one(mod):
    """Two layers, the same weights: the logits of the 4-bit cache lie near the dense cache's.
    A value is off by half a step at most, 1/30 of its 64's range, and so are scores of a few
    units by a tenth: logits within a fifth of their size in the 2-norm."""
    decode, _, ops = mod
    cfg = decode.DecoderConfig(n_layers=2, hidden=512, n_heads=8, n_kv_heads=2, intermediate=512, vocab=1024)
    a = decode.Q4Decoder(cfg, 2, 64, seed=9)
    b = decode.Q4Decoder(cfg, 2, 64, weights=a.w, kv_cache="kv4", kv_page=16)
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    for i in range(6):
        x = torch.randn(2, cfg.hidden, device="cuda", generator=g)
        for d in (a, b):
            d.x_in.copy_(x)
            d.pos.fill_(i)
            d.step()
        off = (a.logits - b.logits).norm() / a.logits.norm()
        assert off < 0.2 and off > 0, float(off)
    assert ops.device_error() == 0


def test_cache_kept_by_a_server(mod):
    """Requests of unlike lengths, steps, a fork, an end, compaction; attention after each."""
    _, kv4_mod, ops = mod
    rng = np.random.default_rng(3)
    hkv, dim, page, n_pages = 2, 128, 16, 40
    c = kv4_mod.Kv4Cache(2, n_pages, hkv, dim, 3, 8, page, summaries=True)
    ref = [kv4.Cache(n_pages, hkv, dim, page) for _ in range(2)]

    def append(new):
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        pos, table = host(c.lens), host(c.table)
        for l in range(2):
            k, v = (rng.standard_normal((int(cu[-1]), hkv * dim)).astype(np.float32) for _ in range(2))
            c.append(l, dev(k), dev(v), c.lens, cu=dev(cu))
            ref[l].append(k, v, table, np.where(np.array(new) > 0, pos, -1), cu, 10000.0)
        c.advance(dev(np.array(new, np.int32)))

    def attend():
        q = rng.standard_normal((3, 4 * dim)).astype(np.float32)
        pos, table = host(c.lens) - 1, host(c.table)
        for l in range(2):
            got = c.decode(l, dev(q), c.lens - 1, n_q_heads=4, out_f32=True)
            want = ref[l].decode(q.reshape(3, 4, dim), table, pos, 10000.0)
            close(host(got), want.reshape(3, -1), F32_TOL, f"layer {l}")
            near = c.decode(l, dev(q), c.lens - 1, n_q_heads=4, n_sel=2, out_f32=True)
            sel = ref[l].select(q.reshape(3, 4, dim), table, pos, 2, 10000.0)
            want = ref[l].decode(q.reshape(3, 4, dim), table, pos, 10000.0, None, sel)
            close(host(near), want.reshape(3, -1), F32_TOL, f"layer {l}, two pages")

    def same_pages():
        for l in range(2):  # the pages moved or copied: the device's bytes are what the rows hold
            ref[l] = kv4.Cache.of(host(c.pool[l]), dim, host(c.summary[l]))

    c.reserve(dev(np.array([50, 20, 33], np.int32)))
    assert host(c.info).tolist() == [n_pages - 4 - 2 - 3, 0, 0, 0]
    append([50, 20, 33])
    attend()
    info = c.reorder(dev(np.array([0, 0, 2], np.int32)), dev(np.array([1, 1, 1], np.int32)))
    assert host(info).tolist() == [n_pages - 8, 1, 0, 0] and host(c.lens).tolist() == [50, 50, 33]
    same_pages()
    k0, _ = c.gather(1, torch.zeros(3, dtype=torch.int32, device="cuda"), 150,
                     cu=dev(np.array([0, 50, 100, 150], np.int32)), dtype=torch.float32)
    assert torch.equal(k0[:50], k0[50:100])  # the fork holds what its parent holds
    assert ops.device_error() == 5  # row 2 has no page for its tokens 48 and 49
    append([1, 1, 1])
    attend()
    c.reorder(dev(np.array([-1, 1, 2], np.int32)))
    c.compact()
    assert host(c.info).tolist()[0] == 4 + 3 and host(c.table).max() == 6
    same_pages()
    assert host(c.lens).tolist() == [0, 51, 34]
    attend()
    assert ops.device_error() == 0


def test_cache_refusals(mod):
    _, kv4_mod, _ = mod
    for bad in (dict(n_layers=0), dict(page=20), dict(head_dim=96), dict(max_pages=0)):
        args = dict(n_layers=1, n_pages=4, n_kv_heads=1, head_dim=64, batch=1, max_pages=2) | bad
        with pytest.raises(ValueError):
            kv4_mod.Kv4Cache(**args)
    c = kv4_mod.Kv4Cache(1, 4, 1, 64, 1, 2)
    with pytest.raises(ValueError, match="summaries"):
        c.decode(0, torch.zeros(1, 64, device="cuda"), c.lens, n_q_heads=1, n_sel=2)
    from llmnputest_b200.decode import DecoderConfig, Q4Decoder
    with pytest.raises(ValueError, match="kv_cache"):
        Q4Decoder(DecoderConfig(n_layers=1, vocab=1024), 1, 16, kv_cache="int8")
