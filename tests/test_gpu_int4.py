"""The 4-bit cache on the GPU: writing bit-exact against the oracle's quantiser and record,
attention against 64 bits within the bound derived in oracle/int4_oracle.py, the cache class
through a decode step, captured and eager."""

import numpy as np
import pytest
import torch

from latentserve_b200 import cache as lc
from latentserve_b200 import decode_step as ds
from latentserve_b200 import int4_write as i4
from latentserve_b200 import paged_decode as pd
from latentserve_b200 import paged_decode_cuda as pdc
from oracle import int4_oracle as orc
from tests.gpu_util import device

pytestmark = pytest.mark.gpu


def make_pool(lens, heads, group, seed, spare=3, scale=1.0, shift=0.5):
    """Random pages under shuffled tables; rows past a sequence's end hold 0xff bytes (codes 15,
    scales NaN), and so do pages nobody owns."""
    rng = np.random.default_rng(seed)
    pages = [-(-n // 16) for n in lens]
    nb = sum(pages) + spare
    pool = np.full((nb, heads, orc.record_bytes(group)), 0xFF, np.uint8)
    order = rng.permutation(nb).astype(np.int32)
    tables = np.full((len(lens), max(1, max(pages))), order[-1], np.int32)
    mean = rng.standard_normal((2, heads, 128)) * shift
    at = 0
    for b, n in enumerate(lens):
        for p in range(pages[b]):
            blk = order[at]
            at += 1
            tables[b, p] = blk
            m = min(16, n - 16 * p)
            for h in range(heads):
                parts = []
                for side in range(2):
                    x = ((rng.standard_normal((16, 128)) + mean[side, h]) * scale).astype(np.float16)
                    code, step, lo = orc.quantize(x, group)
                    code[m:], step[m:], lo[m:] = 15, np.nan, np.nan
                    parts.append((code, step, lo))
                pool[blk, h] = orc.pack(*parts)
    return pool, tables


def attend(q, pool, tables, lens, **kw):
    dev = device()
    return pd.paged_decode_attention_int4(torch.from_numpy(q).to(dev), torch.from_numpy(pool).to(dev),
                                          torch.from_numpy(tables).to(dev),
                                          torch.tensor(lens, dtype=torch.int32, device=dev), **kw)


def check(got, q, pool, tables, lens, scale=None):
    got = got.float().cpu().numpy().astype(np.float64)
    want, bound = orc.attention(q, pool, tables, np.asarray(lens), scale)
    err = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (err <= bound).all(), f"max err {err.max():.3e}, worst {(err / bound).max():.2f} of its bound"
    # Each element's rounding is within 2^-11 of it; computing may add an eighth of that on the whole.
    norm = np.linalg.norm(want)
    if norm > 0:
        assert np.linalg.norm(err) <= 1.125 * 2.0 ** -11 * norm + 2.0 ** -25 * np.sqrt(err.size)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("lens", [[1], [16], [17], [15, 0, 33, 1], [300, 5, 128, 1000, 0], [2049, 4000]])
def test_attention_lengths(group, lens):
    rng = np.random.default_rng(len(lens) * 7 + group)
    q = rng.standard_normal((len(lens), 2, 6, 128)).astype(np.float16)
    pool, tables = make_pool(lens, 2, group, seed=sum(lens) + group)
    got = attend(q, pool, tables, lens)
    check(got, q, pool, tables, lens)
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all()


@pytest.mark.parametrize("heads,rep", [(1, 1), (1, 8), (3, 5), (8, 4), (5, 2), (2, 7)])
def test_attention_head_layouts(heads, rep):
    lens = [77, 200, 16]
    q = np.random.default_rng(heads * 10 + rep).standard_normal((3, heads, rep, 128)).astype(np.float16)
    pool, tables = make_pool(lens, heads, 64, seed=rep)
    check(attend(q, pool, tables, lens), q, pool, tables, lens)


@pytest.mark.parametrize("qs,vs", [(1e-6, 1.0), (60000.0, 1e-3), (1.0, 3000.0), (8.0, 0.02), (0.0, 1.0)])
def test_attention_magnitudes(qs, vs):
    """Queries from subnormal to the largest, values from small ones to those whose steps would
    overflow a product with a weight above 4."""
    lens = [700, 31]
    rng = np.random.default_rng(3)
    q = np.clip(rng.standard_normal((2, 2, 6, 128)) * qs, -65000, 65000).astype(np.float16)
    pool, tables = make_pool(lens, 2, 32, seed=9, scale=vs)
    check(attend(q, pool, tables, lens, softmax_scale=0.088 / max(qs * vs, 1.0)), q, pool, tables, lens,
          0.088 / max(qs * vs, 1.0))


def test_attention_largest_steps():
    """V rows that span all of fp16: steps of 8734, the largest the writer stores."""
    lens = [40]
    rng = np.random.default_rng(5)
    q = rng.standard_normal((1, 1, 4, 128)).astype(np.float16)
    pool, tables = make_pool(lens, 1, 32, seed=2)
    for p in range(3):
        rec = pool[tables[0, p], 0]
        k, _ = orc.unpack(rec)
        x = np.where(rng.random((16, 128)) < 0.5, -1, 1) * 65504.0
        v = orc.quantize(x.astype(np.float16), 32)
        assert v[1].max() == np.float16(8734)
        pool[tables[0, p], 0] = orc.pack(k, v)
    got = attend(q, pool, tables, lens).float().cpu().numpy()
    want, bound = orc.attention(q, pool, tables, np.asarray(lens))
    assert (np.abs(got - want) <= bound).all()


def test_attention_needles():
    """One token far above the rest, first, last or in between: the reference of the online softmax
    moves late or early."""
    lens = [500, 500, 500]
    rng = np.random.default_rng(6)
    q = np.abs(rng.standard_normal((3, 1, 6, 128))).astype(np.float16)
    pool, tables = make_pool(lens, 1, 32, seed=4)
    for b, t in enumerate([0, 250, 499]):
        rec = pool[tables[b, t // 16], 0]
        (code, step, lo), v = orc.unpack(rec)
        code[t % 16], step[t % 16], lo[t % 16] = 8, 0.125, 1.0          # every channel 2: a score of 18 or so
        pool[tables[b, t // 16], 0] = orc.pack((code, step, lo), v)
    check(attend(q, pool, tables, lens), q, pool, tables, lens)


def test_attention_strides_and_out():
    """q and out as views with rows between theirs, the pool a slice of one with more heads, the
    tables a slice of wider ones."""
    dev = device()
    lens = [100, 37]
    rng = np.random.default_rng(8)
    q = rng.standard_normal((2, 2, 6, 128)).astype(np.float16)
    pool, tables = make_pool(lens, 4, 32, seed=12)
    big = torch.from_numpy(pool).to(dev)
    wide_t = torch.full((2, 40), 10 ** 6, dtype=torch.int32, device=dev)
    wide_t[:, :tables.shape[1]] = torch.from_numpy(tables).to(dev)
    qw = torch.zeros(2, 3, 9, 128, dtype=torch.float16, device=dev)
    qw[:, 1:, 1:7] = torch.from_numpy(q).to(dev)
    outw = torch.full((2, 3, 9, 128), 7.0, dtype=torch.float16, device=dev)
    out = outw[:, 1:, 1:7]
    got = pd.paged_decode_attention_int4(qw[:, 1:, 1:7], big[:, 1:3], wide_t[:, :tables.shape[1]],
                                         torch.tensor(lens, dtype=torch.int32, device=dev), out=out)
    assert got is out
    check(out.contiguous(), q, np.ascontiguousarray(pool[:, 1:3]), tables, lens)
    assert (outw[:, 0] == 7).all() and (outw[:, :, 0] == 7).all() and (outw[:, :, 7:] == 7).all()


def test_attention_skips_blocks_outside_the_pool():
    lens = [64, 64]
    q = np.random.default_rng(1).standard_normal((2, 2, 6, 128)).astype(np.float16)
    pool, tables = make_pool(lens, 2, 64, seed=5)
    tables[1, 2], tables[0, 1] = 10 ** 7, -3
    work = pdc.DecodeWorkspace()
    got = attend(q, pool, tables, lens, workspace=work)
    check(got, q, pool, tables, lens)
    assert work.error_flag(device(), 2, 2) == 1


def test_attention_nothing_to_attend():
    """All lengths zero or negative, and sequences none of whose blocks lie in the pool: zeros."""
    q = np.random.default_rng(1).standard_normal((3, 2, 6, 128)).astype(np.float16)
    pool, tables = make_pool([64, 64, 64], 2, 32, seed=6)
    for lens in ([0, 0, 0], [-5, 0, -1]):
        assert (attend(q, pool, tables, lens) == 0).all()
    tables[1:] = 10 ** 6
    got = attend(q, pool, tables, [64, 64, 7])
    assert (got[1:] == 0).all()
    check(got[:1], q[:1], pool, tables[:1], [64])


@pytest.mark.parametrize("rep", [1, 4, 8])
def test_attention_one_long_sequence(rep):
    """More partial states than fit the merge's shared memory at once."""
    lens = [40001]
    q = np.random.default_rng(rep).standard_normal((1, 1, rep, 128)).astype(np.float16)
    pool, tables = make_pool(lens, 1, 128, seed=rep)
    check(attend(q, pool, tables, lens), q, pool, tables, lens)


@pytest.mark.parametrize("batch", [65, 300, 1024])
def test_attention_many_sequences(batch):
    """More sequences than chunks, than threads; empty ones among them; a workspace used at
    several batch sizes in turn."""
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, 90, batch).tolist()
    q = rng.standard_normal((batch, 2, 3, 128)).astype(np.float16)
    pool, tables = make_pool(lens, 2, 64, seed=batch)
    work = pdc.DecodeWorkspace()
    for n in (batch, 7, batch, batch // 2):
        check(attend(q[:n], pool, tables[:n], lens[:n], workspace=work), q[:n], pool, tables[:n], lens[:n])
    assert work.error_flag(device(), batch, 2) == 0


@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-6, 0.5])
def test_attention_scales(scale):
    lens = [200, 33]
    q = np.random.default_rng(2).standard_normal((2, 2, 5, 128)).astype(np.float16)
    pool, tables = make_pool(lens, 2, 32, seed=8)
    got = attend(q, pool, tables, lens, softmax_scale=scale).float().cpu().numpy()
    want, _ = orc.attention(q, pool, tables, np.asarray(lens), scale)
    _, bound = orc.attention(q, pool, tables, np.asarray(lens), abs(scale))
    wide, _ = orc.attention(-q if scale < 0 else q, pool, tables, np.asarray(lens), abs(scale))
    assert np.allclose(want, wide, rtol=1e-12, atol=1e-12)
    # The bound's terms are those of |scale|; its first one is the output's own.
    assert (np.abs(got - want) <= bound + 2.0 ** -11 * np.abs(want)).all()


def test_a_query_that_is_not_finite_spoils_its_own_row_only():
    lens = [100]
    q = np.random.default_rng(3).standard_normal((1, 2, 6, 128)).astype(np.float16)
    pool, tables = make_pool(lens, 2, 32, seed=9)
    want = attend(q, pool, tables, lens)
    q[0, 1, 2, 5] = np.nan
    got = attend(q, pool, tables, lens)
    assert got[0, 1, 2].isnan().all()
    keep = torch.ones(2, 6, dtype=torch.bool)
    keep[1, 2] = False
    assert torch.equal(got[0][keep.to(got.device)], want[0][keep.to(got.device)])


def test_attention_refusals():
    dev = device()
    q = torch.zeros(2, 2, 6, 128, dtype=torch.float16, device=dev)
    pool = torch.zeros(4, 2, 2560, dtype=torch.uint8, device=dev)
    tables = torch.zeros(2, 2, dtype=torch.int32, device=dev)
    lens = torch.ones(2, dtype=torch.int32, device=dev)
    for bad in [dict(q=q.float()), dict(q=q[..., :64]), dict(q=torch.zeros(2, 2, 9, 128, dtype=torch.float16, device=dev)),
                dict(pool=pool[:, :1]), dict(pool=pool[..., :2500]), dict(pool=pool.to(torch.int8)),
                dict(tables=tables.long()), dict(lens=lens.long()), dict(lens=lens.cpu()), dict(pool=pool.cpu()),
                dict(lens=lens[:1]), dict(out=torch.zeros(2, 2, 6, 128, device=dev))]:
        a = dict(q=q, pool=pool, tables=tables, lens=lens, out=None) | bad
        with pytest.raises(ValueError):
            pd.paged_decode_attention_int4(a["q"], a["pool"], a["tables"], a["lens"], out=a["out"])


def test_two_streams_and_two_graphs_do_not_share_bookkeeping():
    """Calls of one shape on two streams at once, and two captured calls replayed on two streams at
    once, give what they give alone, every time."""
    dev = device()
    cases = []
    for seed in range(2):
        lens = [3000 + 500 * seed, 777]
        q = np.random.default_rng(seed).standard_normal((2, 2, 6, 128)).astype(np.float16)
        pool, tables = make_pool(lens, 2, 128, seed=40 + seed)
        args = [torch.from_numpy(x).to(dev) for x in (q, pool, tables)] + [torch.tensor(lens, dtype=torch.int32, device=dev)]
        cases.append((args, pd.paged_decode_attention_int4(*args)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(pd.paged_decode_attention_int4(*cases[i][0]))
    graphs = []
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = pd.paged_decode_attention_int4(*cases[i][0])
        graphs.append((g, got))
    for _ in range(20):
        for (g, got), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, cases[i][1]) for o in outs[i])
        assert torch.equal(graphs[i][1], cases[i][1])


@pytest.mark.parametrize("programmatic", [False, True])
def test_programmatic_launch_gives_the_same(programmatic):
    lens = [900, 64, 1]
    q = np.random.default_rng(0).standard_normal((3, 2, 6, 128)).astype(np.float16)
    pool, tables = make_pool(lens, 2, 32, seed=77)
    try:
        pdc.set_programmatic_launch(programmatic)
        check(attend(q, pool, tables, lens), q, pool, tables, lens)
    finally:
        pdc.set_programmatic_launch(False)


# ---------------------------------------------------------------------------- writing


def written(k, v, lens, new, group, before=None, seed=0, start_pool=None):
    """Write through the library; returns (pool, tables) as numpy."""
    dev = device()
    heads = k.shape[1]
    rng = np.random.default_rng(seed)
    pages = [-(-max(n, 0) // 16) for n in lens]
    nb = sum(pages) + 2
    tables = np.zeros((len(lens), max(1, max(pages))), np.int32)
    order = rng.permutation(nb).astype(np.int32)
    at = 0
    for b, n in enumerate(pages):
        tables[b, :n] = order[at: at + n]
        at += n
    pool = rng.integers(0, 256, (nb, heads, orc.record_bytes(group))).astype(np.uint8)
    dpool = torch.from_numpy(pool).to(dev)
    i4.write(k, v, dpool, torch.from_numpy(tables).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
             None if new is None else torch.tensor(new, dtype=torch.int32, device=dev))
    return pool, dpool.cpu().numpy(), tables


def expect(pool, k, v, lens, new, tables, group):
    """The pool after the write, token by token: only the new tokens' own bytes change."""
    want = pool.copy()
    b, heads, n, _ = k.shape
    kq, vq = orc.quantize(k, group), orc.quantize(v, group)
    for i in range(b):
        m = n if new is None else min(max(new[i], 0), n)
        for t in range(m):
            pos = lens[i] - m + t
            if pos < 0 or pos // 16 >= tables.shape[1]:
                continue
            blk = tables[i, pos // 16]
            for h in range(heads):
                kk, vv = orc.unpack(want[blk, h])
                for part, new_part in ((kk, kq), (vv, vq)):
                    for a, x in zip(part, new_part):
                        a[pos % 16] = x[i, h, t]
                want[blk, h] = orc.pack(kk, vv)
    return want


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,lens,new", [
    (1, [1, 16, 17, 500], None), (5, [5, 18, 100], None), (40, [40, 47, 321], None), (16, [16, 32], None),
    (33, [33, 60, 90, 70], [33, 0, 1, 17]), (20, [7, 0, 20], None), (3, [50, 51], [9, -1])])
def test_write_is_bit_exact_and_touches_nothing_else(group, n, lens, new):
    rng = np.random.default_rng(n + group)
    shape = (len(lens), 2, n, 128)
    k = (rng.standard_normal(shape) * np.logspace(-4, 3, n)[None, None, :, None]).astype(np.float16)
    v = rng.standard_normal(shape).astype(np.float16)
    k[0, 0, 0], v[0, 1, 0] = 0, 3.0                          # groups of one value: step 0
    dev = device()
    before, after, tables = written(torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), lens, new, group, seed=n)
    assert np.array_equal(after, expect(before, k, v, lens, new, tables, group))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_write_rounds_ties_to_even_and_takes_any_range(group):
    """Rows on coarse lattices, where many quotients are exact halves, rows whose steps are subnormal,
    rows of one value, and rows with single far values."""
    rng = np.random.default_rng(group)
    n = 640
    k = rng.integers(0, 31, (2, 2, n, 128)) * np.float16(0.5) * 2.0 ** rng.integers(-12, 8, (2, 2, n, 1))
    v = rng.integers(-20, 20, (2, 2, n, 128)) * 2.0 ** -24 * 2.0 ** rng.integers(0, 6, (2, 2, n, 1))
    v[:, :, ::7] = 3.0
    k[:, :, 5::11, 17] = 60000.0
    k, v = k.astype(np.float16), v.astype(np.float16)
    step = orc.quantize(k, group)[1].astype(np.float64)
    left = (k.astype(np.float64) - k.astype(np.float64).reshape(2, 2, n, -1, group).min(-1).repeat(group, -1))
    assert ((left / step.repeat(group, -1)) % 1 == 0.5).mean() > 0.01            # ties there are
    dev = device()
    lens = [n, n + 9]
    before, after, tables = written(torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), lens, None, group)
    assert np.array_equal(after, expect(before, k, v, lens, None, tables, group))


def test_write_from_views_and_special_values():
    """K and V rows as interleaved views of one projection; infinities, NaN, -0, subnormals."""
    dev = device()
    rng = np.random.default_rng(2)
    proj = rng.standard_normal((3, 21, 4, 128)).astype(np.float16)
    proj[0, 0, 0, :6] = [np.inf, -np.inf, np.nan, -0.0, 6e-8, 65504]
    proj[1, 3, 2] = 6e-8
    proj[2, 20, 3] = np.nan
    t = torch.from_numpy(proj).to(dev)
    k, v = t[:, :, :2].transpose(1, 2), t[:, :, 2:].transpose(1, 2)
    assert not k.is_contiguous()
    lens = [21, 40, 23]
    before, after, tables = written(k, v, lens, None, 32)
    want = expect(before, proj[:, :, :2].transpose(0, 2, 1, 3), proj[:, :, 2:].transpose(0, 2, 1, 3), lens, None, tables, 32)
    # The sign of a zero low is the one bit the formula leaves open.
    for b, n in enumerate(lens):
        for h in range(2):
            for a, c in zip(orc.rows(after, tables[b], h, n), orc.rows(want, tables[b], h, n)):
                new = slice(n - 21, n)
                assert np.array_equal(a[new], c[new]) and np.isfinite(a[new]).all()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_read_gives_the_rounded_values(group):
    dev = device()
    lens, heads = [50, 0, 16, 33], 2
    pool, tables = make_pool(lens, heads, group, seed=3)
    tables[3, 1] = 999                                        # outside the pool: zeros
    tt = torch.from_numpy(tables).to(dev)
    ll = torch.tensor(lens, dtype=torch.int32, device=dev)
    for length, start in [(50, None), (64, None), (1, None), (20, [35, 0, 3, 15]), (7, [0, 5, 16, 30]), (0, None)]:
        st = None if start is None else torch.tensor(start, dtype=torch.int32, device=dev)
        k, v = i4.read(torch.from_numpy(pool).to(dev), tt, ll, length, st)
        want = np.zeros((2, len(lens), heads, length, 128), np.float16)
        for b, n in enumerate(lens):
            first = 0 if start is None else start[b]
            for p in range(first, min(n, first + length)):
                blk = tables[b, p // 16]
                if not 0 <= blk < pool.shape[0]:
                    continue
                for h in range(heads):
                    for side, part in enumerate(orc.unpack(pool[blk, h])):
                        # lo + step * code: the product is exact in fp32, the sum rounds there, then to fp16.
                        one = [x[p % 16: p % 16 + 1] for x in part]
                        want[side, b, h, p - first] = orc.dequantize(*one)[0].astype(np.float32).astype(np.float16)
        assert np.array_equal(k.cpu().numpy(), want[0]) and np.array_equal(v.cpu().numpy(), want[1])


def test_blocks_past_four_gigabytes():
    """A pool of 5.4 GB: write, copy, read and attend pages at its far end."""
    from latentserve_b200 import page_copy

    dev = device()
    nb = 1_050_000
    pool = torch.empty(nb, 2, 2560, dtype=torch.uint8, device=dev)
    rng = np.random.default_rng(4)
    k, v = (rng.standard_normal((1, 2, 40, 128)).astype(np.float16) for _ in range(2))
    tables = torch.tensor([[nb - 1, nb - 3, nb - 2]], dtype=torch.int32, device=dev)
    lens = torch.tensor([40], dtype=torch.int32, device=dev)
    i4.write(torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), pool, tables, lens)
    page_copy.copy_pages([pool], [nb - 2], [nb - 4])
    tables[0, 2] = nb - 4
    want = [orc.dequantize(*orc.quantize(x, 32)) for x in (k, v)]
    for got, x in zip(i4.read(pool, tables, lens, 40), want):
        assert np.array_equal(got.cpu().numpy(), x.astype(np.float32).astype(np.float16))
    q = rng.standard_normal((1, 2, 6, 128)).astype(np.float16)
    got = pd.paged_decode_attention_int4(torch.from_numpy(q).to(dev), pool, tables, lens)
    small = pool[nb - 4:].cpu().numpy()
    check(got, q, small, np.array([[3, 1, 0]], np.int32), [40])


def test_write_and_read_refusals():
    dev = device()
    k = torch.zeros(2, 2, 4, 128, dtype=torch.float16, device=dev)
    pool = torch.zeros(4, 2, 2560, dtype=torch.uint8, device=dev)
    tables = torch.zeros(2, 2, dtype=torch.int32, device=dev)
    lens = torch.full((2,), 4, dtype=torch.int32, device=dev)
    for bad in [dict(k=k.float()), dict(k=k[:, :1]), dict(v=k[:, :, :3]), dict(pool=pool[:, :1]), dict(pool=pool[..., :2432]),
                dict(new=lens.long()), dict(new=lens[:1]), dict(lens=lens[:1]), dict(k=k[..., :64]), dict(tables=tables.cpu()),
                dict(k=torch.zeros(2, 2, 4, 129, dtype=torch.float16, device=dev)[..., 1:])]:
        a = dict(k=k, v=k, pool=pool, tables=tables, lens=lens, new=None) | bad
        with pytest.raises(ValueError):
            i4.write(a["k"], a["v"], a["pool"], a["tables"], a["lens"], a["new"])
    with pytest.raises(ValueError):
        i4.read(pool, tables, lens, -1)
    with pytest.raises(ValueError):
        i4.read(pool, tables, lens, 4, start=lens.long())
    assert pool.count_nonzero() == 0


# ---------------------------------------------------------------------------- the cache


def spec(max_len=256, batch=4, layers=2, heads=2):
    return lc.KVCacheSpec(num_layers=layers, num_kv_heads=heads, head_dim=128, max_seq_len=max_len, max_batch_size=batch)


def fill(cache, n, seed, slots=None, batch=None):
    """Advance by n and write random rows into every layer; returns them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache.advance(n, batch, slots)
    b = len(cache.active_slots())
    rows = []
    for layer in range(cache.spec.num_layers):
        k, v = (torch.randn(b, cache.spec.num_kv_heads, n, 128, device="cuda", generator=g).half() for _ in range(2))
        cache.write(layer, k, v)
        rows.append((k, v))
    return rows


def test_cache_prompt_then_tokens_reads_back():
    cache = lc.Int4PagedKVCache(spec(), num_blocks=64)
    parts = [fill(cache, n, 10 + n, batch=3) for n in (21, 1, 1, 12)]
    for layer in range(2):
        k = torch.cat([p[layer][0] for p in parts], 2).cpu().numpy()
        v = torch.cat([p[layer][1] for p in parts], 2).cpu().numpy()
        for x, got in zip((k, v), cache.read(layer)):
            want = orc.dequantize(*orc.quantize(x, 32)).astype(np.float32).astype(np.float16)
            assert np.array_equal(got.cpu().numpy(), want)
    with pytest.raises(RuntimeError, match="advance"):
        cache.write(0, torch.zeros(3, 2, 2, 128, device="cuda").half(), torch.zeros(3, 2, 2, 128, device="cuda").half())


def test_rope_append_is_the_rotation_then_the_write():
    """The fused append gives the bytes that writing the fp16 cache's rotated rows gives."""
    dev = device()
    b, hq, h = 5, 12, 2
    fp16, c4 = lc.PagedKVCache(spec(batch=b), num_blocks=80), lc.Int4PagedKVCache(spec(batch=b), num_blocks=80, group=64)
    two = lc.Int4PagedKVCache(spec(batch=b), num_blocks=80, group=64)
    cos, sin = (t.half() for t in ds.rope_tables(ds.QwenShape(), 256, dev))
    g = torch.Generator(device="cuda").manual_seed(4)
    for step in range(19):
        qkv = torch.randn(b, (hq + 2 * h) * 128, device=dev, generator=g).half()
        pos = torch.full((b,), step, dtype=torch.int64, device=dev)
        q1, q2 = torch.empty(b, hq * 128, device=dev).half(), torch.empty(b, hq * 128, device=dev).half()
        for c in (fp16, c4, two):
            c.advance(1, b)
        fp16.rope_write(0, qkv, cos, sin, pos, q1, hq)
        c4.rope_write(0, qkv, cos, sin, pos, q2, hq)
        assert torch.equal(q1, q2)
        slot = torch.tensor([t.slot(step) for t in fp16.tables[:b]], device=dev)
        rows = [pool.view(-1, h, 128)[slot][:, :, None] for pool in (fp16.k_pool[0], fp16.v_pool[0])]
        two.write(0, *rows)
    assert torch.equal(c4.kv_pool[0], two.kv_pool[0])


@pytest.mark.parametrize("projections,fused", [("cublas", True), ("ls", True), ("cublas", False)])
@pytest.mark.parametrize("scaling", [None, {"type": "yarn", "factor": 4.0, "original_max_pos": 128}])
def test_decode_step_over_the_cache(projections, fused, scaling):
    """A small model's logits over the 4-bit cache against the same model in which each layer attends,
    in 64 bits, the values the cache holds; eager and captured."""
    dev = device()
    shape = ds.QwenShape(num_layers=2, hidden=256, q_heads=4, kv_heads=2, intermediate=512, vocab=320, rope_scaling=scaling)
    model = ds.DecodeModel(shape, dev, max_pos=512, fused=fused, projections=projections)
    b, prompt = 3, 37
    caches = [lc.Int4PagedKVCache(spec(batch=b), num_blocks=64) for _ in range(3)]
    for c in caches:
        fill(c, prompt, 5, batch=b)

    class Exact(ds.DecodeModel):
        def attend(self, cache, layer, q, batch, hint):
            pool, tables = cache.kv_pool[layer].cpu().numpy(), cache.block_tables_tensor(batch).cpu().numpy()
            out, _ = orc.attention(q.cpu().numpy(), pool, tables, cache.seq_lens_tensor(batch).cpu().numpy())
            return torch.from_numpy(out).to(q.device).half()

    exact = Exact(shape, dev, max_pos=512, fused=fused, projections=projections)
    step = ds.GraphedStep(model, caches[2], b, 256)
    tokens = torch.tensor([3, 200, 11], device=dev)
    step.tokens.copy_(tokens)
    captured = False
    for t in range(4):
        for c in caches:
            c.advance(1, b)
        if not captured:
            step.capture()
            captured = True
        pos = torch.full((b,), prompt + t, dtype=torch.int64, device=dev)
        got = model.forward(caches[0], tokens, pos, 256, return_logits=True).float()
        want = exact.forward(caches[1], tokens, pos, 256, return_logits=True).float()
        # The two attentions round to neighbouring fp16 numbers at worst (2^-10), in each of two
        # layers; what follows of a layer is linear up to the norms.
        assert (got - want).norm() <= 4 * 2.0 ** -10 * want.norm()
        step.tokens.copy_(tokens)
        picked = step.step(feed_back=False)
        assert torch.equal(picked, got.argmax(-1))
        assert torch.equal(caches[2]._kv_all, caches[0]._kv_all)
        tokens = picked.clone()


def test_rewind_then_grow():
    cache = lc.Int4PagedKVCache(spec(), num_blocks=40)
    rows = fill(cache, 40, 1, batch=2)
    cache.rewind(21)
    more = fill(cache, 30, 2, batch=2)
    for layer in range(2):
        for side in range(2):
            x = torch.cat([rows[layer][side][:, :, :21], more[layer][side]], 2).cpu().numpy()
            want = orc.dequantize(*orc.quantize(x, 32)).astype(np.float32).astype(np.float16)
            assert np.array_equal(cache.read(layer)[side].cpu().numpy(), want)
