"""The 4-bit paged KV cache on the GPU against its definition in 64 bits (oracle/kv4_oracle.py).

Codes, steps, page choices, tables and counts are whole numbers: equal bit for bit.
Attention: q enters as fp16 (off by 2^-11 of itself at most), which moves a score by no more
than its own size times 2^-11, about 2^-11 in the natural log's units at the scores of these
cases (scale * |q| |k| ~ 1); the weights are rounded to fp16 once, 2^-11 again; numerator and
denominator together: 3 * 2^-11 < 2^-9 of the output's 2-norm.  A bf16 output adds 2^-8."""

import numpy as np
import pytest
import torch
from ml_dtypes import bfloat16

from oracle import kv4_oracle as kv4

pytestmark = pytest.mark.gpu
F32_TOL, BF16_TOL = 2.0 ** -9, 2.0 ** -9 + 2.0 ** -8


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from llmnputest_b200 import ops as _ops
    return _ops


@pytest.fixture(autouse=True)
def no_device_error(ops):
    ops.device_error()
    yield
    torch.cuda.synchronize()
    assert ops.device_error() == 0


def dev(a, dtype=None):
    a = np.ascontiguousarray(a)
    if a.dtype == np.float64:
        a = a.astype(np.float32)
    t = torch.from_numpy(a).cuda()
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.float().cpu().numpy().astype(np.float64) if t.is_floating_point() else t.cpu().numpy()


class Case:
    """A cache on both sides: random pages, a table that scatters them, lengths."""

    def __init__(self, rng, lens, hkv, dim, page, spare=2, extra=1, garbage=True):
        self.lens, self.hkv, self.dim, self.page = np.asarray(lens, np.int32), hkv, dim, page
        need = [-(-int(n) // page) for n in lens]
        most, total = max(1, max(need)) + extra, sum(need) + spare
        ids = rng.permutation(total)
        self.table = np.full((len(need), most), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.cache = kv4.Cache(total, hkv, dim, page)
        self.cache.code[:] = rng.integers(0, 16, self.cache.code.shape)
        m = -np.abs(rng.standard_normal(self.cache.meta.shape[:-1]))
        self.cache.meta[:] = kv4.bf16(np.stack([(0.1 + np.abs(m)) / 7.5, m], -1))
        near = np.sort(rng.standard_normal(self.cache.summary.shape), 2)
        self.cache.summary[:] = kv4.bf16(near)
        if garbage:  # what no token holds may be anything, NaN and infinity among it
            live = np.zeros((total, page), bool)
            for b, n in enumerate(lens):
                for t in range(int(n)):
                    live[self.table[b, t // page], t % page] = True
            dead = ~live.reshape(total, 1, page // 16, 1, 1, 16)
            odd = rng.choice([np.nan, np.inf, -np.inf, 3e38, 0.0], self.cache.meta.shape)
            self.cache.meta[:] = np.where(np.broadcast_to(dead[..., None], odd.shape), odd, self.cache.meta)
        self.pool = dev(self.cache.pool())
        self.summary = dev(self.cache.summary, torch.bfloat16)
        self.dtable, self.pos = dev(self.table), dev(self.lens - 1)
        self.heads = dict(n_kv_heads=hkv, head_dim=dim)


def close(got, ref, tol, what=""):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    for b in range(len(ref)):
        off, size = np.linalg.norm(got[b] - ref[b]), np.linalg.norm(ref[b])
        assert off <= tol * size, f"{what} row {b}: {off / max(size, 1e-300):.3g} > {tol:.3g}"


# ---------------------------------------------------------------- append and gather

@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,dtype,theta", [(16, torch.float32, 10000.0), (64, torch.bfloat16, None),
                                              (48, torch.float32, None), (128, torch.bfloat16, 1e7)])
def test_append_rows(ops, dim, page, dtype, theta):
    """Ragged rows that begin and end inside tiles and pages, a sequence with none, one that is
    not there, slices of a wider projection: every byte of the pool and every summary."""
    rng = np.random.default_rng(dim + page)
    start = np.array([0, 5, page - 1, 17, -1, 3 * page, 0], np.int32)
    new = np.array([1, 30, 2, 0, 4, page + 7, 2 * page + 16])
    c = Case(rng, np.maximum(start, 0) + new, 3, dim, page)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) + 2  # rows before and behind
    rows = int(cu[-1]) + 3
    kv = rng.standard_normal((rows, 2 * 3 * dim + 8)) * np.exp(rng.standard_normal(2 * 3 * dim + 8))
    kv = dev(kv, dtype)
    k, v = kv[:, :3 * dim], kv[:, 3 * dim:6 * dim]
    c.cache.append(host(k), host(v), c.table, start, cu, theta)
    ops.kv4_append(k, v, c.pool, c.dtable, dev(start), cu=dev(cu), theta=theta, summary=c.summary, **c.heads)
    want = c.cache.pool()
    got = host(c.pool)
    for i in range(len(new)):  # name the sequence first
        if start[i] >= 0 and new[i]:
            pages = c.table[i, start[i] // page:(start[i] + new[i] - 1) // page + 1]
            assert np.array_equal(got[pages], want[pages]), f"sequence {i}"
    assert np.array_equal(got, want)
    assert np.array_equal(host(c.summary), c.cache.summary)
    # read back, into rows of a wider buffer; rows without tokens stay
    for odt in (torch.float32, torch.bfloat16):
        buf = torch.full((2, rows, 3 * dim + 8), 77.0, dtype=odt, device="cuda")
        ops.kv4_gather(c.pool, c.dtable, dev(start), rows, cu=dev(cu), dtype=odt,
                       out=(buf[0, :, :3 * dim], buf[1, :, :3 * dim]), **c.heads)
        ref = np.full((2, rows, 3 * dim + 8), 77.0)
        for i in range(len(new)):
            if start[i] >= 0 and new[i]:
                ref[:, cu[i]:cu[i + 1], :3 * dim] = c.cache.gather(c.table[i], start[i], new[i])
        ref = ref.astype(np.float32)
        ref = ref if odt == torch.float32 else ref.astype(bfloat16)
        assert np.array_equal(host(buf), ref.astype(np.float64))


@pytest.mark.parametrize("dim,theta", [(64, 10000.0), (256, None)])
def test_append_step(ops, dim, theta):
    """One new token per sequence (a decode step), positions up to far ones, a padded row."""
    rng = np.random.default_rng(7)
    lens = np.array([1, 16, 17, 64, 65, 0, 5000, 100])
    c = Case(rng, lens, 8, dim, 64)
    k, v = (rng.standard_normal((8, 8 * dim)).astype(np.float32) for _ in range(2))
    c.cache.append(k, v, c.table, lens - 1, None, theta)
    ops.kv4_append(dev(k), dev(v), c.pool, c.dtable, c.pos, theta=theta, summary=c.summary, **c.heads)
    assert np.array_equal(host(c.pool), c.cache.pool())
    assert np.array_equal(host(c.summary), c.cache.summary)
    gk, gv = ops.kv4_gather(c.pool, c.dtable, c.pos, 8, dtype=torch.float32, **c.heads)
    for b, n in enumerate(lens):
        if n:
            rk, rv = c.cache.gather(c.table[b], n - 1, 1)
            assert np.array_equal(host(gk)[b], rk[0].astype(np.float32)), b
            assert np.array_equal(host(gv)[b], rv[0].astype(np.float32)), b


def test_append_special_values(ops):
    """Constant groups, zeros, values at the border of two codes, huge, tiny and unlike values,
    and values that are not finite."""
    rng = np.random.default_rng(3)
    rows = np.zeros((10, 64))
    rows[1] = -2.5
    rows[2] = (np.arange(64) % 31) * 0.5          # every other value between two codes
    rows[3] = np.linspace(-1e30, 1e30, 64)
    rows[4] = rng.standard_normal(64) * 1e-20
    rows[5, 9] = 1e4
    rows[6] = rng.standard_normal(64)
    rows[6, 3] = np.nan
    rows[7] = rng.standard_normal(64)
    rows[7, 63] = np.inf
    rows[8] = np.round(rng.standard_normal(64) * 8) / 16
    rows[9] = -0.0
    rows = rows.astype(np.float32)
    c = Case(rng, [10], 1, 64, 16)
    c.cache.append(rows, rows[::-1], c.table, [0], [0, 10], None)
    ops.kv4_append(dev(rows), dev(rows[::-1]), c.pool, c.dtable, dev(np.zeros(1, np.int32)),
                   cu=dev(np.array([0, 10], np.int32)), theta=None, **c.heads)
    code, meta = kv4.unpack(host(c.pool).reshape(c.cache.code.shape[:4] + (kv4.CELL,)))
    at = c.table[0, 0]
    assert np.array_equal(code[at, 0, 0, 0, :, :10], c.cache.code[at, 0, 0, 0, :, :10])
    assert np.array_equal(meta[at, 0, 0, 0, :, :10], c.cache.meta[at, 0, 0, 0, :, :10], equal_nan=True)
    k, _ = ops.kv4_gather(c.pool, c.dtable, dev(np.zeros(1, np.int32)), 10, cu=dev(np.array([0, 10], np.int32)),
                          dtype=torch.float32, **c.heads)
    assert np.isnan(host(k)[6:8]).all() and np.isfinite(host(k)[:6]).all()


def test_bad_positions_are_reported(ops):
    """Positions outside the table and pages outside the pool: device error 5, nothing written."""
    rng = np.random.default_rng(1)
    c = Case(rng, [40, 40, 40], 2, 64, 16, garbage=False)
    x = dev(rng.standard_normal((3, 256)))
    for pos, entry in (([5, -2, 7], None), ([5, 16 * c.table.shape[1], 7], None), ([5, 33, 7], 99999)):
        pool, table = c.pool.clone(), c.dtable.clone()
        if entry is not None:
            table[1, 2] = entry
        p = dev(np.array(pos, np.int32))
        ops.kv4_append(x[:, :128], x[:, 128:], pool, table, p, theta=None, **c.heads)
        assert ops.device_error() == 5
        before = kv4.Cache.of(host(c.pool), 64)
        before.append(host(x[:, :128]), host(x[:, 128:]), c.table, [pos[0], -1, pos[2]], None, None)
        assert np.array_equal(host(pool), before.pool())
        out = torch.full((3, 128), 9.0, device="cuda")
        ops.kv4_decode(x[:, :128], c.pool, table, p, n_q_heads=2, out=out, out_f32=True, theta=None, **c.heads)
        assert ops.device_error() == 5
        assert torch.isfinite(out).all() and (entry is not None or (out[1] == 9.0).all())
        sel = ops.kv4_select(x[:, :128], c.summary, table, p, n_q_heads=2, page=16, n_sel=2, theta=None, **c.heads)
        assert ops.device_error() == 5
        assert (sel[0] >= 0).any() and (entry is not None or (sel[1] == -1).all())


# ---------------------------------------------------------------- decode

def run_decode(ops, c, grp, rng, theta=10000.0, scale=None, **kw):
    b, hq = len(c.lens), grp * c.hkv
    wide = dev(rng.standard_normal((b, (hq + 2 * c.hkv) * c.dim)))
    q = wide[:, :hq * c.dim]
    ref = c.cache.decode(host(q).reshape(b, hq, c.dim), c.table, c.lens - 1, theta, scale,
                         None if kw.get("select") is None else host(kw["select"]))
    got = ops.kv4_decode(q, c.pool, c.dtable, c.pos, n_q_heads=hq, theta=theta, scale=scale, **c.heads, **kw)
    return got, ref.reshape(b, -1)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,grp", [(16, 5), (64, 4), (48, 1), (128, 8)])
def test_decode(ops, dim, page, grp):
    rng = np.random.default_rng(dim + page + grp)
    lens = [1, 2, 15, 16, 17, 0, 31, 33, page, page + 1, 3 * page - 1, 300, 0]
    c = Case(rng, lens, 2, dim, page)
    got, ref = run_decode(ops, c, grp, rng, out_f32=True)
    close(host(got), ref, F32_TOL, "fp32")
    assert (host(got)[[5, 12]] == 0).all()
    got, ref = run_decode(ops, c, grp, rng)
    assert got.dtype == torch.bfloat16
    close(host(got), ref, BF16_TOL, "bf16")


@pytest.mark.parametrize("lens,hkv,dim,page", [([5000], 8, 64, 64), ([9000, 1, 4097], 2, 256, 16),
                                               ([700] * 70, 8, 64, 32), ([2049, 100], 1, 128, 128)])
def test_decode_long_and_split(ops, lens, hkv, dim, page):
    rng = np.random.default_rng(len(lens))
    c = Case(rng, lens, hkv, dim, page)
    got, ref = run_decode(ops, c, 5 if dim == 64 else 4, rng, out_f32=True)
    close(host(got), ref, F32_TOL)


def test_decode_options(ops):
    """theta None, another scale, a strided out buffer, a given workspace, a max_len of its own."""
    rng = np.random.default_rng(2)
    c = Case(rng, [70, 200, 0, 129], 2, 64, 16)
    got, ref = run_decode(ops, c, 3, rng, theta=None, scale=0.5, out_f32=True)
    close(host(got), ref, 4 * F32_TOL)  # scores four times as large
    buf = torch.full((4, 400), 5.0, dtype=torch.bfloat16, device="cuda")
    need = ops.kv4_decode_workspace_bytes(4, 6, 2, 64, 16, 200)
    ws = torch.empty(need + 64, dtype=torch.uint8, device="cuda")
    got, ref = run_decode(ops, c, 3, rng, out=buf[:, :384], max_len=200, workspace=ws)
    close(host(got), ref, BF16_TOL)
    assert (buf[:, 384:] == 5.0).all()


def test_decode_unlike_scales(ops):
    """Values of very unlike size between tokens, sequences and heads, a dominating key, equal keys."""
    rng = np.random.default_rng(4)
    c = Case(rng, [257, 300, 128, 64], 2, 64, 32, garbage=False)
    size = np.exp(6 * rng.standard_normal(c.cache.meta.shape[:4] + (1, 16, 1)))
    c.cache.meta[..., 1, :, :] = kv4.bf16((c.cache.meta[..., 1, :, :] * size[..., 0, :, :]))
    c.cache.meta[c.table[2, 0], :, 0, :, 0, 3] = kv4.bf16(c.cache.meta[c.table[2, 0], :, 0, :, 0, 3] * 20)
    c.cache.meta[c.table[3, :2], :, :, :, 0, :, 0] = 2.0 ** -40
    c.cache.meta[c.table[3, :2], :, :, :, 0, :, 1] = 1.0
    c.cache.meta[c.table[1, :4], :, :, :, 1] *= 1e-12
    c.cache.meta[:] = kv4.bf16(c.cache.meta)
    c.cache.meta[..., 0] = np.maximum(c.cache.meta[..., 0], 2.0 ** -40)
    c.pool = dev(c.cache.pool())
    got, ref = run_decode(ops, c, 2, rng, out_f32=True)
    close(host(got), ref, 4 * F32_TOL)  # scores up to four times as large


def test_decode_nan_and_infinity(ops):
    """A key or value that is NaN reaches its own sequence and kv head, no other; a score of
    -inf counts for nothing."""
    rng = np.random.default_rng(5)
    c = Case(rng, [40, 40, 40], 2, 64, 16)
    c.cache.meta[c.table[0, 1], 0, 0, 0, 0, 3, 1] = np.nan
    c.cache.meta[c.table[1, 0], 1, 0, 0, 1, 9, 1] = np.nan
    c.pool = dev(c.cache.pool())
    got, ref = run_decode(ops, c, 2, rng, out_f32=True)
    got = host(got).reshape(3, 2, -1)
    ref = ref.reshape(3, 2, -1)
    assert np.isnan(got[0, 0]).all() and np.isnan(got[1, 1]).all()
    for b, h in ((0, 1), (1, 0), (2, 0), (2, 1)):
        close(got[b:b + 1, h], ref[b:b + 1, h], F32_TOL)


def test_decode_of_empty_pages(ops):
    """Zeroed pages attended as they are: their values are zero."""
    pool = torch.zeros(4, 2, ops.kv4_page_bytes(16, 64), dtype=torch.uint8, device="cuda")
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    out = ops.kv4_decode(torch.randn(1, 512, device="cuda"), pool, table, dev(np.array([50], np.int32)), n_q_heads=8,
                         n_kv_heads=2, head_dim=64)
    assert (out == 0).all()


# ---------------------------------------------------------------- select

@pytest.mark.parametrize("dim,page,n_sel,grp", [(64, 16, 5, 5), (128, 32, 1, 4), (256, 16, 7, 8), (64, 64, 300, 1),
                                                (64, 16, 64, 3)])
def test_select(ops, dim, page, n_sel, grp):
    rng = np.random.default_rng(dim + n_sel)
    lens = [1, page, 40 * page, 41 * page + 3, 0, 300 * page - 5, 17 * page]
    c = Case(rng, lens, 2, dim, page)
    b, hq = len(lens), grp * 2
    q = rng.standard_normal((b, hq * dim)).astype(np.float32)
    for theta in (10000.0, None):
        want = c.cache.select(q.reshape(b, hq, dim), c.table, c.lens - 1, n_sel, theta)
        got = ops.kv4_select(dev(q), c.summary, c.dtable, c.pos, n_q_heads=hq, page=page, n_sel=n_sel, theta=theta,
                             **c.heads)
        assert np.array_equal(host(got), want)
    got, ref = run_decode(ops, c, grp, rng, select=dev(want), out_f32=True)
    close(host(got), ref, F32_TOL)


@pytest.mark.parametrize("dim,ctx", [(64, 40), (256, 700)])
def test_more_pages_asked_for_than_there_are(ops, dim, ctx):
    """n_sel above the pages of the row, and of the whole table: all of them, -1 behind."""
    rng = np.random.default_rng(ctx)
    c = Case(rng, [ctx, 3], 2, dim, 16, extra=0)
    q = rng.standard_normal((2, 4 * dim)).astype(np.float32)
    sel = ops.kv4_select(dev(q), c.summary, c.dtable, c.pos, n_q_heads=4, page=16, n_sel=64, theta=None, **c.heads)
    assert np.array_equal(host(sel), c.cache.select(q.reshape(2, 4, dim), c.table, c.lens - 1, 64, None))
    got, ref = run_decode(ops, c, 2, rng, select=sel, out_f32=True)
    close(host(got), ref, F32_TOL)


def test_select_ties_go_to_the_lower_page(ops):
    rng = np.random.default_rng(9)
    c = Case(rng, [16 * 100], 1, 64, 16)
    near = c.cache.summary
    near[:] = near[0]
    near[c.table[0, 40:50]] *= 2  # ten pages above the rest, alike among themselves
    c.summary = dev(near, torch.bfloat16)
    q = rng.standard_normal((1, 128)).astype(np.float32)
    for n_sel in (1, 4, 11, 20):
        want = c.cache.select(q.reshape(1, 2, 64), c.table, c.lens - 1, n_sel, None)
        got = ops.kv4_select(dev(q), c.summary, c.dtable, c.pos, n_q_heads=2, page=16, n_sel=n_sel, theta=None,
                             **c.heads)
        assert np.array_equal(host(got), want), n_sel


def test_decode_odd_selections(ops):
    """Entries of -1, behind the query, twice the same or falling count for nothing."""
    rng = np.random.default_rng(11)
    c = Case(rng, [100, 100], 1, 64, 16)
    sel = np.array([[[1, 1, 3, 2, -1, 6, 7, 5]], [[-1] * 8]], np.int32)
    sel = np.pad(sel[..., :c.table.shape[1]], ((0, 0), (0, 0), (0, max(0, 0))))
    q = rng.standard_normal((2, 128)).astype(np.float32)
    seen = sel.copy()
    last = np.maximum.accumulate(np.pad(sel, ((0, 0), (0, 0), (1, 0)), constant_values=-1)[..., :-1], -1)
    falls = np.zeros(sel.shape, bool)
    falls[..., 1:] = sel[..., 1:] <= sel[..., :-1]
    seen[falls] = -1
    assert last.shape == sel.shape
    ref = c.cache.decode(q.reshape(2, 2, 64), c.table, c.lens - 1, None, None, seen)
    got = ops.kv4_decode(dev(q), c.pool, c.dtable, c.pos, n_q_heads=2, theta=None, select=dev(sel), out_f32=True,
                         **c.heads)
    close(host(got)[:1], ref.reshape(2, -1)[:1], F32_TOL)
    assert (host(got)[1] == 0).all()


# ---------------------------------------------------------------- pages

def pages_case(rng, b, layers, page, most, n_pages, hkv=2, dim=64):
    lens = rng.integers(0, most * page + 1, b).astype(np.int32)
    lens[::4] = lens[::4] // page * page
    need = -(-lens // page)
    while need.sum() > n_pages * 3 // 4:
        i = int(np.argmax(need))
        lens[i], need[i] = lens[i] // 2, -(-(lens[i] // 2) // page)
    ids = rng.permutation(n_pages)
    table, refs, at = np.full((b, most), -1, np.int32), np.zeros(n_pages, np.int32), 0
    for i in range(b):
        table[i, :need[i]] = ids[at:at + need[i]]
        at += need[i]
    np.add.at(refs, table[table >= 0], 1)
    pool = rng.integers(0, 256, (layers, n_pages, hkv, page // 16 * (dim // 64) * kv4.CELL)).astype(np.uint8)
    summary = kv4.bf16(rng.standard_normal((layers, n_pages, hkv, 2, dim)))
    return table, lens, refs, pool, summary


@pytest.mark.parametrize("seed", range(8))
def test_reorder(ops, seed):
    rng = np.random.default_rng(seed)
    b, page = int(rng.integers(1, 40)), int(rng.choice([16, 32, 48]))
    most, n_pages = int(rng.integers(1, 9)), int(rng.integers(20, 5000 if seed == 3 else 300))
    table, lens, refs, pool, summary = pages_case(rng, b, int(rng.integers(1, 4)), page, most, n_pages)
    refs[rng.integers(0, n_pages, 3)] += 1  # pages that something else holds too
    parent = rng.integers(-1, b, b).astype(np.int32)
    reserve = rng.integers(-3, 2 * page, b).astype(np.int32) if seed % 2 else None
    dpool, dsum = dev(pool), dev(summary, torch.bfloat16)
    for step in range(3):  # the outcome of one step is the next one's start
        want = kv4.reorder(table, lens, refs, parent, page, reserve)
        for src, dst in want[3]:
            pool[:, dst], summary[:, dst] = pool[:, src], summary[:, src]
        got = ops.kv4_reorder(dpool, dev(table), dev(lens), dev(refs), dev(parent), head_dim=64,
                              reserve=None if reserve is None else dev(reserve), summary=dsum)
        for g, w, name in zip(got, (*want[:3], want[4]), ("table", "lens", "refs", "info")):
            assert np.array_equal(host(g), w), (step, name)
        assert np.array_equal(host(dpool), pool) and np.array_equal(host(dsum), summary)
        assert ops.device_error() == (7 if want[4][2] else 0)
        table, lens, refs = want[:3]
        parent = rng.integers(-1, b, b).astype(np.int32)


def test_reorder_when_pages_run_out(ops):
    """Four rows go on with one row, one free page: one copy, the others cut to their full pages."""
    table = np.array([[0, 1], [2, -1], [-1, -1], [-1, -1]], np.int32)
    lens, refs = np.array([20, 3, 0, 0], np.int32), np.array([1, 1, 1], np.int32)
    pool = dev(np.arange(3 * 2 * 1152).reshape(1, 3, 2, 1152).astype(np.uint8))
    parent, reserve = np.zeros(4, np.int32), np.array([0, 0, 0, 40], np.int32)
    want = kv4.reorder(table, lens, refs, parent, 16, reserve)
    got = ops.kv4_reorder(pool, dev(table), dev(lens), dev(refs), dev(parent), head_dim=64, reserve=dev(reserve))
    for g, w in zip(got, (*want[:3], want[4])):
        assert np.array_equal(host(g), w)
    assert host(got[1]).tolist() == [20, 20, 16, 16] and host(got[3]).tolist() == [0, 1, 4, 0]
    assert ops.device_error() == 7
    assert torch.equal(pool[0, 2], pool[0, 1])


def test_reorder_odd_parents(ops):
    """A parent outside the batch frees the row and is reported."""
    table, lens, refs = np.array([[0], [1]], np.int32), np.array([4, 4], np.int32), np.array([1, 1], np.int32)
    pool = torch.zeros(1, 2, 1, 1152, dtype=torch.uint8, device="cuda")
    got = ops.kv4_reorder(pool, dev(table), dev(lens), dev(refs), dev(np.array([0, 2], np.int32)), head_dim=64)
    assert ops.device_error() == 5
    assert [host(g).tolist() for g in got] == [[[0], [-1]], [4, 0], [1, 0], [1, 0, 0, 0]]


@pytest.mark.parametrize("seed", range(6))
def test_compact(ops, seed):
    rng = np.random.default_rng(100 + seed)
    b, page, most = int(rng.integers(1, 40)), 16, int(rng.integers(1, 9))
    n_pages = [1, 2, 37, 300, 1025, 5000][seed]
    table, lens, refs, pool, summary = pages_case(rng, b, int(rng.integers(1, 4)), page, most, n_pages)
    refs[rng.integers(0, n_pages, 2)] += 1
    dpool, dsum = dev(pool), dev(summary, torch.bfloat16)
    t, r, moves, info = kv4.compact(table, refs)
    for src, dst in moves:
        pool[:, dst], summary[:, dst] = pool[:, src], summary[:, src]
    got = ops.kv4_compact(dpool, dev(table), dev(refs), summary=dsum)
    for g, w in zip(got, (t, r, info)):
        assert np.array_equal(host(g), w)
    assert np.array_equal(host(dpool), pool) and np.array_equal(host(dsum), summary)


def test_copy_pages(ops):
    rng = np.random.default_rng(0)
    pool = rng.integers(0, 256, (3, 20, 2, 1152)).astype(np.uint8)
    src, dst = np.array([3, -1, 5, 7, 3], np.int32), np.array([0, 1, 5, -4, 19], np.int32)
    dpool = dev(pool)
    ops.kv4_copy_pages(dpool, dev(src), dev(dst))
    pool[:, 0], pool[:, 19] = pool[:, 3], pool[:, 3]
    assert np.array_equal(host(dpool), pool)
    ops.kv4_copy_pages(dpool, dev(src[:0]), dev(dst[:0]))
    ops.kv4_copy_pages(dpool, dev(np.array([20], np.int32)), dev(np.array([1], np.int32)))
    assert ops.device_error() == 5
    assert np.array_equal(host(dpool), pool)


# ---------------------------------------------------------------- together

def test_a_run_of_all(ops):
    """Prompts, steps over chosen pages, a fork, steps of the forked rows, compaction: the cache
    and the attention after each, against the oracle's."""
    rng = np.random.default_rng(42)
    hkv, dim, page, n_pages, most, grp = 2, 64, 16, 60, 12, 5
    hq = hkv * grp
    heads = dict(n_kv_heads=hkv, head_dim=dim)
    pool = torch.zeros(1, n_pages, hkv, ops.kv4_page_bytes(page, dim), dtype=torch.uint8, device="cuda")
    summary = torch.zeros(1, n_pages, hkv, 2, dim, dtype=torch.bfloat16, device="cuda")
    cache = kv4.Cache(n_pages, hkv, dim, page)
    table, lens, refs = np.full((3, most), -1, np.int32), np.zeros(3, np.int32), np.zeros(n_pages, np.int32)

    def rows(parent, reserve):
        nonlocal table, lens, refs
        want = kv4.reorder(table, lens, refs, np.array(parent), page, np.array(reserve))
        got = ops.kv4_reorder(pool, dev(table), dev(lens), dev(refs), dev(np.array(parent, np.int32)), head_dim=dim,
                              reserve=dev(np.array(reserve, np.int32)), summary=summary)
        for g, w in zip(got, (*want[:3], want[4])):
            assert np.array_equal(host(g), w)
        for src, dst in want[3]:
            cache.code[dst], cache.meta[dst], cache.summary[dst] = cache.code[src], cache.meta[src], cache.summary[src]
        table, lens, refs = want[:3]

    def append(new):
        nonlocal lens
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        k, v = (rng.standard_normal((int(cu[-1]), hkv * dim)).astype(np.float32) for _ in range(2))
        cache.append(k, v, table, lens, cu, 10000.0)
        ops.kv4_append(dev(k), dev(v), pool[0], dev(table), dev(lens), cu=dev(cu), summary=summary[0], **heads)
        lens = lens + np.array(new, np.int32)
        assert np.array_equal(host(pool[0]), cache.pool())
        assert np.array_equal(host(summary[0]), cache.summary)

    def attend(n_sel):
        q = rng.standard_normal((3, hq * dim)).astype(np.float32)
        pos = lens - 1
        want = cache.select(q.reshape(3, hq, dim), table, pos, n_sel, 10000.0)
        sel = ops.kv4_select(dev(q), summary[0], dev(table), dev(pos), n_q_heads=hq, page=page, n_sel=n_sel, **heads)
        assert np.array_equal(host(sel), want)
        for s in (None, sel):
            got = ops.kv4_decode(dev(q), pool[0], dev(table), dev(pos), n_q_heads=hq, select=s, out_f32=True, **heads)
            ref = cache.decode(q.reshape(3, hq, dim), table, pos, 10000.0, None, None if s is None else want)
            close(host(got), ref.reshape(3, -1), F32_TOL)

    rows([-1, -1, -1], [100, 33, 16])
    append([100, 33, 16])
    attend(3)
    for _ in range(3):
        rows([0, 1, 2], [1, 1, 1])
        append([1, 1, 1])
        attend(4)
    rows([0, 0, 2], [1, 1, 1])  # row 1 ends, row 0 forks
    append([1, 1, 1])
    attend(5)
    rows([1, -1, 1], [20, 50, 1])
    append([20, 50, 1])
    attend(2)
    t, r, moves, info = kv4.compact(table, refs)
    got = ops.kv4_compact(pool, dev(table), dev(refs), summary=summary)
    for g, w in zip(got, (t, r, info)):
        assert np.array_equal(host(g), w)
    for src, dst in moves:
        cache.code[dst], cache.meta[dst], cache.summary[dst] = cache.code[src], cache.meta[src], cache.summary[src]
    table, refs = t, r
    attend(4)


def test_captured_step_and_other_streams(ops):
    """Append, select and decode captured once and replayed as the positions advance, on a stream
    of its own; the same calls on two streams at once."""
    rng = np.random.default_rng(8)
    c = Case(rng, [60, 33], 2, 64, 16, extra=3, garbage=False)
    for b, n in enumerate([60, 33]):  # pages for the steps to come
        free = [p for p in range(c.cache.code.shape[0]) if p not in set(c.table[c.table >= 0])]
        c.table[b, -(-n // 16)] = free[0]
    c.dtable = dev(c.table)
    kv = torch.zeros(2, 2 * 128, device="cuda")
    q = torch.zeros(2, 640, device="cuda")
    out = torch.zeros(2, 640, device="cuda")
    pos = dev(np.array([60, 33], np.int32))
    sel = torch.zeros(2, 2, 3, dtype=torch.int32, device="cuda")
    need = ops.kv4_decode_workspace_bytes(2, 10, 2, 64, 16, 16 * c.table.shape[1], 3)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")

    def step():
        ops.kv4_append(kv[:, :128], kv[:, 128:], c.pool, c.dtable, pos, summary=c.summary, **c.heads)
        ops.kv4_select(q, c.summary, c.dtable, pos, n_q_heads=10, page=16, n_sel=3, out=sel, **c.heads)
        ops.kv4_decode(q, c.pool, c.dtable, pos, n_q_heads=10, select=sel, out=out, out_f32=True, workspace=ws,
                       **c.heads)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    keep = c.pool.clone(), c.summary.clone()
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    c.pool.copy_(keep[0])
    c.summary.copy_(keep[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(4):
        x, y = rng.standard_normal((2, 256)).astype(np.float32), rng.standard_normal((2, 640)).astype(np.float32)
        kv.copy_(dev(x))
        q.copy_(dev(y))
        at = np.array([60 + i, 33 + i], np.int32)
        pos.copy_(dev(at))
        g.replay()
        c.cache.append(x[:, :128], x[:, 128:], c.table, at, None, 10000.0)
        assert np.array_equal(host(c.pool), c.cache.pool()), i
        want = c.cache.select(y.reshape(2, 10, 64), c.table, at, 3, 10000.0)
        assert np.array_equal(host(sel), want)
        close(host(out), c.cache.decode(y.reshape(2, 10, 64), c.table, at, 10000.0, None, want).reshape(2, -1), F32_TOL)
    del g
    # two streams at once, each with its own workspace
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [dev(rng.standard_normal((2, 640))) for _ in streams]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(ops.kv4_decode(qs[i], c.pool, c.dtable, pos, n_q_heads=10, out_f32=True, **c.heads))
    torch.cuda.synchronize()
    for i in range(2):
        ref = c.cache.decode(host(qs[i]).reshape(2, 10, 64), c.table, at, 10000.0).reshape(2, -1)
        for o in outs[i]:
            close(host(o), ref, F32_TOL)


def test_refusals(ops):
    rng = np.random.default_rng(0)
    c = Case(rng, [40, 20], 2, 64, 16)
    x = torch.zeros(2, 512, device="cuda")
    k = x[:, :128]
    ok = dict(n_kv_heads=2, head_dim=64)
    from llmnputest_b200._native import B2Error
    bad = [
        (TypeError, lambda: ops.kv4_append(k.half(), k.half(), c.pool, c.dtable, c.pos, **ok)),
        (TypeError, lambda: ops.kv4_append(k, k.bfloat16(), c.pool, c.dtable, c.pos, **ok)),
        (ValueError, lambda: ops.kv4_append(x[:, :100], k, c.pool, c.dtable, c.pos, **ok)),
        (ValueError, lambda: ops.kv4_append(x[:1, :128], x[:1, :128], c.pool, c.dtable, c.pos, **ok)),
        (ValueError, lambda: ops.kv4_append(k, x[:1, :128], c.pool, c.dtable, c.pos, **ok)),
        (ValueError, lambda: ops.kv4_append(k, k, c.pool, c.dtable, c.pos, cu=c.pos, **ok)),
        (ValueError, lambda: ops.kv4_append(k, k, c.pool[:, :, :1000], c.dtable, c.pos, **ok)),
        (ValueError, lambda: ops.kv4_append(k, k, c.pool, c.dtable, c.pos[:1], **ok)),
        (ValueError, lambda: ops.kv4_append(k, k, c.pool, c.dtable, c.pos, summary=c.summary[:1], **ok)),
        (TypeError, lambda: ops.kv4_append(k, k, c.pool, c.dtable.long(), c.pos, **ok)),
        (ValueError, lambda: ops.kv4_append(k, k, c.pool, c.dtable, c.pos, n_kv_heads=2, head_dim=96)),
        (B2Error, lambda: ops.kv4_append(k, k, c.pool, c.dtable, c.pos, theta=-1.0, **ok)),
        (B2Error, lambda: ops.kv4_append(k[:1].expand(2, 128), k, c.pool, c.dtable, c.pos, **ok)),
        (TypeError, lambda: ops.kv4_gather(c.pool, c.dtable, c.pos, 2, dtype=torch.float16, **ok)),
        (ValueError, lambda: ops.kv4_gather(c.pool, c.dtable, c.pos, 3, **ok)),
        (B2Error, lambda: ops.kv4_gather(c.pool, c.dtable, c.pos, 2, out=(x[:, 1:129], x[:, 1:129]),
                                         dtype=torch.float32, **ok)),
        (TypeError, lambda: ops.kv4_decode(x.bfloat16(), c.pool, c.dtable, c.pos, n_q_heads=8, **ok)),
        (B2Error, lambda: ops.kv4_decode(x, c.pool, c.dtable, c.pos, n_q_heads=3, **ok)),
        (ValueError, lambda: ops.kv4_decode(x, c.pool, c.dtable, c.pos, n_q_heads=18, **ok)),
        (B2Error, lambda: ops.kv4_decode(x, c.pool, c.dtable, c.pos, n_q_heads=4, max_len=10**6, **ok)),
        (ValueError, lambda: ops.kv4_decode(x, c.pool, c.dtable, c.pos, n_q_heads=4, select=c.dtable, **ok)),
        (ValueError, lambda: ops.kv4_decode(x, c.pool, c.dtable, c.pos, n_q_heads=4,
                                            select=torch.zeros(2, 2, 0, dtype=torch.int32, device="cuda"), **ok)),
        (ValueError, lambda: ops.kv4_select(x, c.summary, c.dtable, c.pos, n_q_heads=4, page=16, n_sel=0, **ok)),
        (B2Error, lambda: ops.kv4_select(x, c.summary, c.dtable, c.pos, n_q_heads=4, page=20, n_sel=1, **ok)),
        (ValueError, lambda: ops.kv4_copy_pages(c.pool, c.pos, c.pos)),
        (ValueError, lambda: ops.kv4_copy_pages(c.pool[None], c.pos, c.pos[:1])),
        (ValueError, lambda: ops.kv4_reorder(c.pool[None], c.dtable, c.pos, c.pos, c.pos, head_dim=64)),
        (ValueError, lambda: ops.kv4_compact(c.pool[None], c.dtable, c.pos)),
    ]
    before = c.pool.clone()
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {i} was not refused")
    assert torch.equal(before, c.pool)


# ---------------------------------------------------------------- the ends of the ranges

@pytest.mark.parametrize("scale", [1e9, 1e20, 1e30])
def test_decode_scores_of_any_size(ops, scale):
    """Scores far beyond what exp can take, above and below zero: the largest one's value.  One
    token's key is 2 in every dim, one's -2, the others' below 1 in size, so that no rounding of
    q (2^-11 of itself) comes near to changing which is largest; beside it the rest is e^-10^8."""
    rng = np.random.default_rng(3)
    c = Case(rng, [1, 20, 500, 3], 2, 64, 16, garbage=False)
    c.cache.meta[:, :, :, :, 0, :, 0] = 2.0 ** -40
    c.cache.meta[:, :, :, :, 0, :, 1] = kv4.bf16(rng.uniform(-1, 1, c.cache.meta.shape[:4] + (16,)))
    for b, (hi, lo) in enumerate([(0, 0), (17, 3), (444, 30), (2, 0)]):
        for t, m in ((lo, -2.0), (hi, 2.0)):
            c.cache.meta[c.table[b, t // 16], :, 0, :, 0, t % 16, 1] = m
    c.pool = dev(c.cache.pool())
    q = 1 + np.abs(rng.standard_normal((4, 4 * 64))).astype(np.float32)
    for sign in (1, -1):
        ref = c.cache.decode((sign * q).reshape(4, 4, 64), c.table, c.lens - 1, None, scale).reshape(4, -1)
        got = ops.kv4_decode(dev(sign * q), c.pool, c.dtable, c.pos, n_q_heads=4, theta=None, scale=scale, out_f32=True,
                             **c.heads)
        close(host(got), ref, F32_TOL, f"sign {sign}")


def test_decode_of_many_sequences(ops):
    """More sequences than one launch deals out, some without tokens."""
    rng = np.random.default_rng(4)
    lens = rng.integers(0, 40, 2100)
    lens[[0, 1023, 1024, 2047, 2099]] = [0, 33, 0, 17, 1]
    c = Case(rng, lens, 2, 64, 16, garbage=False)
    got, ref = run_decode(ops, c, 1, rng, out_f32=True, theta=None)
    close(host(got), ref, F32_TOL)
    assert (host(got)[lens == 0] == 0).all()


@pytest.mark.parametrize("dim", [64, 256])
def test_longest_page(ops, dim):
    """Pages of 4096 tokens: appended across a border, chosen and attended."""
    rng = np.random.default_rng(dim)
    start, new = np.array([4000, 0, 4095], np.int32), np.array([200, 3, 1])
    c = Case(rng, start + new, 1, dim, 4096, garbage=False)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    k, v = (rng.standard_normal((204, dim)).astype(np.float32) for _ in range(2))
    c.cache.append(k, v, c.table, start, cu, 10000.0)
    ops.kv4_append(dev(k), dev(v), c.pool, c.dtable, dev(start), cu=dev(cu), summary=c.summary, **c.heads)
    assert np.array_equal(host(c.pool), c.cache.pool())
    assert np.array_equal(host(c.summary), c.cache.summary)
    got, ref = run_decode(ops, c, 4, rng, out_f32=True)
    close(host(got), ref, F32_TOL)
    got, ref = run_decode(ops, c, 4, rng, out_f32=True, select=dev(np.array([[[0]], [[0]], [[0]]], np.int32)))
    close(host(got), ref, F32_TOL)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_rows_of_any_alignment(ops, dtype):
    """Rows that begin at an odd element and follow one another at an odd distance."""
    rng = np.random.default_rng(6)
    start, new = np.array([3, 0], np.int32), np.array([30, 9])
    c = Case(rng, start + new, 2, 64, 16)
    cu = np.array([0, 30, 39], np.int32)
    kv = dev(rng.standard_normal((39, 2 * 128 + 3)), dtype)
    k, v = kv[:, 1:129], kv[:, 130:258]
    c.cache.append(host(k), host(v), c.table, start, cu, 10000.0)
    ops.kv4_append(k, v, c.pool, c.dtable, dev(start), cu=dev(cu), summary=c.summary, **c.heads)
    assert np.array_equal(host(c.pool), c.cache.pool())
    assert np.array_equal(host(c.summary), c.cache.summary)


def test_append_offsets_outside_the_rows(ops):
    """Row offsets that fall, or lie outside the rows, are kept inside them: nothing is read
    or written beyond, and the sequences beside them have their tokens."""
    rng = np.random.default_rng(11)
    c = Case(rng, [20, 20, 20, 20], 2, 64, 16)
    k, v = (rng.standard_normal((10, 128)).astype(np.float32) for _ in range(2))
    cu = np.array([-5, 4, 2, 6, 900], np.int32)  # 0..4, none, 2..6, 6..10
    start = np.array([1, 2, 3, 4], np.int32)
    for b, (lo, hi) in enumerate([(0, 4), (0, 0), (2, 6), (6, 10)]):
        c.cache.append(k[lo:hi], v[lo:hi], c.table[b:b + 1], start[b:b + 1], np.array([0, hi - lo]), 10000.0)
    ops.kv4_append(dev(k), dev(v), c.pool, c.dtable, dev(start), cu=dev(cu), summary=c.summary, **c.heads)
    assert np.array_equal(host(c.pool), c.cache.pool())
    assert np.array_equal(host(c.summary), c.cache.summary)


@pytest.mark.parametrize("dim,pages,n_sel", [(64, 16384, 200), (256, 16384, 16383), (128, 4097, 1000)])
def test_select_among_the_most_pages(ops, dim, pages, n_sel):
    rng = np.random.default_rng(pages + n_sel)
    summary = np.sort(rng.standard_normal((pages, 1, 2, dim)), 2)
    cache = kv4.Cache(1, 1, dim, 16)
    cache.summary = kv4.bf16(summary)
    table = rng.permutation(pages).astype(np.int32)[None]
    q = rng.standard_normal((1, 3 * dim)).astype(np.float32)
    for pos in (16 * pages - 1, 16 * pages - 17):
        want = cache.select(q.reshape(1, 3, dim), table, np.array([pos]), n_sel, None)
        got = ops.kv4_select(dev(q), dev(cache.summary, torch.bfloat16), dev(table), dev(np.array([pos], np.int32)),
                             n_q_heads=3, n_kv_heads=1, head_dim=dim, page=16, n_sel=n_sel, theta=None)
        assert np.array_equal(host(got), want)


def test_a_pool_past_four_gigabytes(ops):
    """The same pages at the far end of a pool whose offsets pass 2^32 bytes: appended, gathered,
    attended, copied by a fork and moved down by a compaction as at its beginning."""
    rng = np.random.default_rng(12)
    c = Case(rng, [200, 65], 8, 64, 64, garbage=False)
    n = c.cache.code.shape[0]
    page_bytes = c.pool.shape[1] * c.pool.shape[2]
    total = (1 << 32) // page_bytes + 3 * n
    far = total - n - 1  # a free page behind them
    pool = torch.empty(total, 8, c.pool.shape[2], dtype=torch.uint8, device="cuda")
    pool[far:far + n] = c.pool
    table = np.where(c.table >= 0, c.table + far, -1).astype(np.int32)
    k, v = (rng.standard_normal((2, 512)).astype(np.float32) for _ in range(2))
    at = np.array([199, 64], np.int32)
    c.cache.append(k, v, c.table, at, None, 10000.0)
    ops.kv4_append(dev(k), dev(v), pool, dev(table), dev(at), **c.heads)
    assert np.array_equal(host(pool[far:far + n]), c.cache.pool())
    got = ops.kv4_gather(pool, dev(table), dev(at), 2, dtype=torch.float32, **c.heads)
    for i in range(2):
        want = c.cache.gather(c.table[i], int(at[i]), 1)
        for a, w in zip(got, want):
            assert np.array_equal(host(a[i]), w[0].astype(np.float32).astype(np.float64))
    q = dev(rng.standard_normal((2, 8 * 64)))
    ref = c.cache.decode(host(q).reshape(2, 8, 64), c.table, at, 10000.0).reshape(2, -1)

    def attend(p, t, rows):
        got = ops.kv4_decode(q, p, t, dev(at[rows]), n_q_heads=8, out_f32=True, **c.heads)
        close(host(got), ref[rows], F32_TOL)

    attend(pool, dev(table), [0, 1])
    refs = torch.ones(total, dtype=torch.int32, device="cuda")  # every page below is held elsewhere
    refs[far:] = 0
    live = table[table >= 0]
    refs[dev(live.astype(np.int64))] = 1
    # both rows go on with row 0: its last page is copied to a far free page
    t2, lens, refs2, info = ops.kv4_reorder(pool[None], dev(table), dev((at + 1).astype(np.int32)), refs,
                                            dev(np.array([0, 0], np.int32)), head_dim=64)
    assert host(info)[1] == 1 and host(info)[2] == 0 and host(t2)[1, 3] >= far
    q[1] = q[0]
    attend(pool, t2, [0, 0])
    # only these rows' pages are held: they move down to the beginning
    held = torch.zeros_like(refs2)
    held[far:] = refs2[far:]
    t3, refs3, info = ops.kv4_compact(pool[None], t2, held)
    assert host(t3).max() < host(info)[0] == int((held > 0).sum())
    attend(pool, t3, [0, 0])


@pytest.mark.parametrize("dim", [64, 256])
def test_decode_of_one_far_longer_sequence(ops, dim):
    """A pair shared by hundreds of CTAs, its parts joined by several threads an output."""
    rng = np.random.default_rng(dim + 1)
    c = Case(rng, [20000, 5, 0, 17], 2, dim, 64, garbage=False)
    for grp in (1, 8):
        got, ref = run_decode(ops, c, grp, rng, out_f32=True)
        close(host(got), ref, F32_TOL)


@pytest.mark.parametrize("dim", [64, 128])
def test_append_values_of_any_size(ops, dim):
    """Rows from fp32's subnormals to its largest, spreads far smaller than the values' own size,
    and values on the very borders between codes."""
    rng = np.random.default_rng(dim + 2)
    n = 160
    c = Case(rng, [n], 1, dim, 16, garbage=False)
    size = 10.0 ** np.linspace(-44, 38, n)[:, None]
    x = rng.uniform(-1, 1, (2, n, dim)) * size
    x[:, 1::4] = size[1::4] * (1 + 1e-6 * rng.uniform(0, 1, (2, n // 4, dim)))
    x[:, 2::4] = size[2::4] * rng.integers(0, 31, (2, n // 4, dim)) / 30
    k, v = x.astype(np.float32)
    c.cache.append(k, v, c.table, np.array([0]), np.array([0, n]), None)
    ops.kv4_append(dev(k), dev(v), c.pool, c.dtable, dev(np.array([0], np.int32)),
                   cu=dev(np.array([0, n], np.int32)), theta=None, summary=c.summary, **c.heads)
    assert np.array_equal(host(c.pool), c.cache.pool())
    assert np.array_equal(host(c.summary), c.cache.summary)


def test_two_graphs_of_one_pool(ops):
    """Two captured calls that allocate their own workspaces, replayed in turn as positions and
    queries change; tiles dealt over the grid, with pairs that several CTAs share."""
    rng = np.random.default_rng(21)
    lens = np.array([2500] * 20 + [1, 0, 777], np.int32)
    c = Case(rng, lens, 8, 64, 64, garbage=False)
    qs = [torch.zeros(len(lens), 8 * 64 * g, device="cuda") for g in (1, 5)]
    graphs, outs = [], []

    def call(i):
        return ops.kv4_decode(qs[i], c.pool, c.dtable, c.pos, n_q_heads=qs[i].shape[1] // 64, out_f32=True, **c.heads)

    for i in range(2):
        call(i)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(i))
        graphs.append(g)
    for turn in range(2):
        at = np.maximum(lens - 1 - 300 * turn, np.minimum(lens - 1, 0)).astype(np.int32)
        c.pos.copy_(dev(at))
        x = [rng.standard_normal(tuple(q.shape)).astype(np.float32) for q in qs]
        for q, y in zip(qs, x):
            q.copy_(dev(y))
        for i in (0, 1, 0):
            graphs[i].replay()
        for i in range(2):
            want = c.cache.decode(x[i].reshape(len(lens), -1, 64), c.table, at, 10000.0).reshape(len(lens), -1)
            close(host(outs[i]), want, F32_TOL, f"turn {turn} graph {i}")
