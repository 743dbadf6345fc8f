"""Rows of a 4-bit paged cache that end, fork and begin again while steps go on (Kv4Cache), and a
decoder's (Q4Decoder.reorder)."""

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as kv4
from tests.test_gpu_kv4 import BF16_TOL, F32_TOL, close, dev, host, no_device_error, ops  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


class Served:
    """A cache and what its rows hold, as a server's loop calls it."""

    def __init__(self, n_pages=40, hkv=2, dim=64, batch=3, max_pages=6, page=16):
        from llmnputest_b200.kv4 import Kv4Cache
        self.c = Kv4Cache(1, n_pages, hkv, dim, batch, max_pages, page)
        self.rng, self.width = np.random.default_rng(0), hkv * dim
        self.rows = [[] for _ in range(batch)]  # the (k, v) of every row's tokens

    def prompts(self, new):
        new = np.asarray(new, np.int32)
        self.c.reserve(dev(new))
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        k, v = (self.rng.standard_normal((int(cu[-1]), self.width)).astype(np.float32) for _ in range(2))
        self.c.append(0, dev(k), dev(v), self.c.lens, cu=dev(cu))
        self.c.advance(dev(new))
        for b, row in enumerate(self.rows):
            row += [(k[i], v[i]) for i in range(cu[b], cu[b + 1])]

    def step(self, alive):
        """One token for every row in use, and the attention of all rows."""
        c, batch = self.c, len(self.rows)
        c.reserve(1)
        pos = c.positions()
        k, v = (self.rng.standard_normal((batch, self.width)).astype(np.float32) for _ in range(2))
        q = self.rng.standard_normal((batch, 2 * self.width)).astype(np.float32)
        c.append(0, dev(k), dev(v), pos)
        got = host(c.decode(0, dev(q), pos, n_q_heads=2 * c.n_kv_heads, out_f32=True))
        c.advance(1)
        for b in range(batch):
            if b in alive:
                self.rows[b].append((k[b], v[b]))
        lens = np.array([len(r) for r in self.rows], np.int32)
        assert host(c.lens).tolist() == lens.tolist()
        assert host(pos).tolist() == [n - 1 if b in alive else -1 for b, n in enumerate(lens)]
        for b, row in enumerate(self.rows):
            if b not in alive:
                assert (got[b] == 0).all()
                continue
            n = len(row)
            pages = -(-n // c.page)
            ref, table = kv4.Cache(pages, c.n_kv_heads, c.head_dim, c.page), np.arange(pages)[None]
            ref.append(*(np.stack(x) for x in zip(*row)), table, [0], [0, n], 10000.0)
            want = ref.decode(q[b].reshape(1, -1, c.head_dim), table, [n - 1], 10000.0)
            close(got[b:b + 1], want.reshape(1, -1), F32_TOL, f"row {b} of {n} tokens")

    def reorder(self, parent, reserve=None):
        self.c.reorder(dev(np.array(parent, np.int32)), None if reserve is None else dev(np.array(reserve, np.int32)))
        self.rows = [list(self.rows[p]) if p >= 0 else [] for p in parent]

    def pages(self):
        return int((host(self.c.refs) > 0).sum()), [int((t >= 0).sum()) for t in host(self.c.table)]


def test_a_row_that_ended_stays_empty(ops):
    """Steps go on with a row emptied: it takes no page and no token; then a request begins in it
    and attends to its own tokens alone."""
    s = Served()
    s.prompts([20, 15, 33])
    s.step({0, 1, 2})
    s.reorder([0, -1, 2])
    for _ in range(18):  # over a page's end in every row
        s.step({0, 2})
    assert s.pages()[1][1] == 0 and s.c.used.tolist() == [1, 0, 1]
    s.prompts([0, 7, 0])
    assert s.c.used.tolist() == [1, 1, 1]
    for _ in range(11):
        s.step({0, 1, 2})
    live, held = s.pages()
    assert held == [-(-len(r) // 16) for r in s.rows] and live == sum(held)


def test_rows_in_use_follow_their_parents(ops):
    """A row that forks an unused one is unused; a reserve above 0 begins a row; a parent outside
    the batch empties it, and is reported."""
    s = Served()
    s.prompts([5, 5, 5])
    s.reorder([-1, 1, 1])
    s.reorder([1, 0, 2])
    assert s.c.used.tolist() == [1, 0, 1] and s.c.positions().tolist() == [5, -1, 5]
    s.step({0, 2})
    s.reorder([0, -1, -1], [0, 9, 0])
    assert s.c.used.tolist() == [1, 1, 0] and s.c.positions().tolist() == [6, 0, -1]
    s.step({0, 1})
    s.c.reorder(dev(np.array([0, 3, -7], np.int32)))
    assert ops.device_error() == 5
    assert s.c.used.tolist() == [1, 0, 0] and s.c.lens.tolist() == [7, 0, 0]


def test_captured_steps_of_a_served_cache(ops):
    """reserve, positions, append, decode and advance in one graph, replayed over a page's end and
    over a row that ends between two replays."""
    s = Served(batch=2)
    s.prompts([14, 30])
    kv, q = torch.zeros(2, 2, s.width, device="cuda"), torch.zeros(2, 2 * s.width, device="cuda")
    out = torch.zeros(2, 2 * s.width, device="cuda")

    def step():
        s.c.reserve(1)
        pos = s.c.positions()
        s.c.append(0, kv[0], kv[1], pos)
        s.c.decode(0, q, pos, n_q_heads=4, out=out, out_f32=True)
        s.c.advance(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for b in range(2):  # the first run's token: zeros
        s.rows[b].append((np.zeros(s.width, np.float32),) * 2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(5):
        x = s.rng.standard_normal((2, 2, s.width)).astype(np.float32)
        y = s.rng.standard_normal((2, 2 * s.width)).astype(np.float32)
        kv.copy_(dev(x))
        q.copy_(dev(y))
        g.replay()
        alive = [0, 1] if i < 3 else [1]
        for b in alive:
            s.rows[b].append((x[0, b], x[1, b]))
            n = len(s.rows[b])
            pages = -(-n // 16)
            ref, table = kv4.Cache(pages, 2, 64, 16), np.arange(pages)[None]
            ref.append(*(np.stack(r) for r in zip(*s.rows[b])), table, [0], [0, n], 10000.0)
            want = ref.decode(y[b].reshape(1, 4, 64), table, [n - 1], 10000.0)
            close(host(out)[b:b + 1], want.reshape(1, -1), F32_TOL, f"replay {i} row {b}")
        assert s.c.lens.tolist() == [len(r) for r in s.rows]
        if i == 2:
            s.reorder([-1, 1])
    assert (out[0] == 0).all()
    del g


@pytest.mark.parametrize("batch,captured", [(3, False), (3, True), (12, True)])
def test_decoder_forks_and_ends(ops, batch, captured):
    """A decoder's sequences fork in the middle of a page and at its end, end and begin anew, and
    step on to ctx_max: the cache and the attention of every step against the oracle's, on the
    step's own projections."""
    from llmnputest_b200 import decode
    cfg = decode.DecoderConfig(n_layers=1, hidden=512, n_heads=8, n_kv_heads=2, intermediate=512, vocab=1024)
    ctx, page = 50, 16
    dec = decode.Q4Decoder(cfg, batch, ctx, seed=5, kv_cache="kv4", kv_page=page)
    rng = np.random.default_rng(batch)
    graph = dec.capture() if captured else None
    rows = [[] for _ in range(batch)]
    pos = np.zeros(batch, np.int32)
    pos[-1] = -1  # a padded sequence at first
    forks = {20: [0, 0, -1], 31: [1, 0, 0], 40: [0, -1, 2]}  # (page ends at 16, 32, 48)
    for t in range(ctx):
        dec.pos.copy_(dev(pos))
        dec.x_in.copy_(dev(rng.standard_normal((batch, cfg.hidden))))
        graph.replay() if captured else dec.step()
        qkv, got = host(dec.qkv), host(dec.attn)
        for b in range(batch):
            if pos[b] < 0:
                assert (got[b] == 0).all()
                continue
            rows[b].append(qkv[b, 512:])
            n = len(rows[b])
            assert n == pos[b] + 1
            kv, pages = np.stack(rows[b]), -(-n // page)
            ref, table = kv4.Cache(pages, 2, 64, page), np.arange(pages)[None]
            ref.append(kv[:, :128], kv[:, 128:], table, [0], [0, n], cfg.rope_theta)
            want = ref.decode(qkv[b, :512].reshape(1, 8, 64), table, [n - 1], cfg.rope_theta)
            close(got[b:b + 1], want.reshape(1, -1), BF16_TOL, f"step {t} sequence {b}")
        if t in forks:
            parent = np.array((forks[t] + list(range(3, batch)))[:batch], np.int32)
            dec.reorder(dev(parent))
            assert host(dec.cache.info)[2] == 0
            rows = [list(rows[p]) if p >= 0 else [] for p in parent]
            assert host(dec.pos).tolist() == [len(r) - 1 for r in rows] == (host(dec.cache.lens) - 1).tolist()
        pos = np.minimum(np.array([len(r) for r in rows]), ctx - 1).astype(np.int32)
        pos[[len(r) == ctx for r in rows]] = -1
        if t < 45:
            pos[-1] = -1 if batch > 3 or t < 20 else pos[-1]
    del graph


def test_decoder_reorder_is_refused_without_pages(ops):
    from llmnputest_b200 import decode
    cfg = decode.DecoderConfig(n_layers=1, hidden=512, n_heads=8, n_kv_heads=2, intermediate=512, vocab=1024)
    with pytest.raises(ValueError, match="kv4"):
        decode.Q4Decoder(cfg, 1, 16).reorder(dev(np.zeros(1, np.int32)))


def test_captured_reorders(ops):
    """A reorder and a reserve captured once and replayed with other parents."""
    s = Served(batch=3)
    s.prompts([20, 5, 33])
    parent, more = dev(np.array([0, 1, 2], np.int32)), dev(np.zeros(3, np.int32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.c.reorder(parent, more)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.c.reorder(parent, more)
    for new, reserve in (([0, 0, -1], [0, 3, 0]), ([1, -1, 0], [1, 0, 1]), ([0, 2, 2], [0, 0, 0])):
        parent.copy_(dev(np.array(new, np.int32)))
        more.copy_(dev(np.array(reserve, np.int32)))
        g.replay()
        s.rows = [list(s.rows[p]) if p >= 0 else [] for p in new]
        alive = {b for b, r in enumerate(s.rows) if r}
        assert s.c.used.tolist() == [int(b in alive) for b in range(3)]
        s.step(alive)
    del g


def test_a_row_without_a_first_request(ops):
    """A batch that begins with a free row: it stays free until a request begins in it.  A cache
    that begins by one number has all its rows in use."""
    s = Served()
    s.prompts([20, 0, 3])
    for _ in range(17):
        s.step({0, 2})
    assert s.pages()[1][1] == 0
    s.prompts([0, 30, 0])
    s.step({0, 1, 2})
    s = Served()
    s.c.reserve(0)
    for _ in range(17):
        s.step({0, 1, 2})
    s = Served()
    s.reorder([-1, -1, -1], [4, 0, 0])
    s.step({0})
