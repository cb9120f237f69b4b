"""Page copies, forks and compaction: plain bytes, so everything is compared for equality."""

import numpy as np
import pytest
import torch

from latentserve_b200 import cache as lc
from latentserve_b200 import page_copy
from latentserve_b200 import paged_decode as pd
from tests.gpu_util import device
from tests.test_gpu_int4 import fill, spec

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,dtype", [
    ((9, 16, 2, 128), torch.float16), ((9, 16, 2, 128), torch.int8), ((9, 16, 3), torch.float32), ((9, 5), torch.float16),
    ((9, 7), torch.uint8), ((9,), torch.float32), ((9, 16, 8, 128), torch.float32), ((9, 2, 2560), torch.uint8),
    ((9, 33333), torch.uint8)])
def test_copy_any_page(shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    pool = torch.randint(-100, 100, shape, device="cuda", generator=g).to(dtype)
    want = pool.clone()
    src, dst = [3, 3, 0, 8], [1, 7, 4, 2]
    want[dst] = want[src]
    page_copy.copy_pages([pool], src, dst)
    assert torch.equal(pool, want)


def test_copy_many_pools_layers_and_views():
    """More pools than one launch takes, more pages than one launch takes, layers in front of the
    page axis, pools that are slices (their neighbours stay), unaligned ones."""
    g = torch.Generator(device="cuda").manual_seed(2)
    rng = np.random.default_rng(3)
    pools = [torch.randn(20, 24, device="cuda", generator=g) for _ in range(70)]
    want = [p.clone() for p in pools]
    page_copy.copy_pages(pools, [5, 6], [7, 8])
    for p, w in zip(pools, want):
        w[[7, 8]] = w[[5, 6]]
        assert torch.equal(p, w)
    order = rng.permutation(9000)
    big = torch.randint(0, 255, (3, 9000, 40), device="cuda", generator=g, dtype=torch.uint8)
    ref = big.clone()
    src, dst = order[:4100], order[4100:8200]
    ref[:, torch.from_numpy(dst).cuda()] = ref[:, torch.from_numpy(src).cuda()]
    page_copy.copy_pages([big], src, dst.tolist(), block_dim=1)
    assert torch.equal(big, ref)
    wide = torch.randn(2, 6, 11, device="cuda", generator=g)
    ref = wide.clone()
    ref[:, 4, 1:8] = ref[:, 2, 1:8]
    page_copy.copy_pages([wide[:, :, 1:8]], [2], [4], block_dim=1)
    assert torch.equal(wide, ref)
    page_copy.copy_pages([], [1], [2])
    page_copy.copy_pages([wide], [], [], block_dim=1)
    assert torch.equal(wide, ref)


def test_copy_is_captured_with_its_ids():
    pool = torch.arange(40, device="cuda", dtype=torch.float32).view(10, 4).contiguous()
    src, dst = [1], [9]
    page_copy.copy_pages([pool], [0], [8])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        page_copy.copy_pages([pool], src, dst)
    src[0], dst[0] = 2, 3                               # the lists may change after the call
    pool[1] = 77
    graph.replay()
    torch.cuda.synchronize()
    assert (pool[9] == 77).all() and pool[3, 0] == 12


def test_copy_refusals():
    pool = torch.zeros(8, 4, 6, device="cuda")
    with pytest.raises(ValueError, match="written twice"):
        page_copy.copy_pages([pool], [0, 1], [2, 2])
    with pytest.raises(ValueError, match="written twice|read and written"):
        page_copy.copy_pages([pool], [0, 2], [2, 3])
    with pytest.raises(ValueError, match="outside"):
        page_copy.copy_pages([pool], [0], [8])
    with pytest.raises(ValueError, match="source pages"):
        page_copy.copy_pages([pool], [0], [1, 2])
    with pytest.raises(ValueError, match="dense"):
        page_copy.copy_pages([pool[:, :, :3]], [0], [1])
    with pytest.raises(ValueError, match="one number of pages"):
        page_copy.copy_pages([pool, pool[:5]], [0], [1])
    with pytest.raises(ValueError, match="block_dim"):
        page_copy.copy_pages([pool], [0], [1], block_dim=2)
    with pytest.raises(ValueError):
        page_copy.copy_pages([pool[:1].expand(8, 4, 6)], [0], [1])


def make(kind):
    if kind == "int4":
        return lc.Int4PagedKVCache(spec(batch=6), num_blocks=40)
    if kind.startswith("int8"):
        cache = lc.Int8PagedKVCache(spec(batch=6), num_blocks=40, asymmetric=kind == "int8_asym")
        if kind == "int8_in_step":
            cache.enable_finalize_in_step()
        return cache
    cache = lc.PagedKVCache(spec(batch=6), num_blocks=40)
    if kind == "fp16_bounds":
        cache.enable_page_bounds()
    if kind == "fp16_fused":
        cache.enable_fused_append()
    return cache


KINDS = ["fp16", "fp16_bounds", "fp16_fused", "int8", "int8_asym", "int8_in_step", "int4"]


def attend(cache, layer, q):
    b = q.shape[0]
    tables, lens = cache.block_tables_tensor(b), cache.seq_lens_tensor(b)
    if hasattr(cache, "kv_pool"):
        return pd.paged_decode_attention_int4(q, cache.kv_pool[layer], tables, lens).clone()
    extra = {}
    if hasattr(cache, "k_scale_pool"):
        extra = dict(k_scale=cache.k_scale_pool[layer], v_scale=cache.v_scale_pool[layer],
                     k_residual=cache.residual(layer), res_rows=cache.residual_rows_tensor(b))
        if cache.asymmetric:
            extra.update(k_zero=cache.k_zero_pool[layer], v_zero=cache.v_zero_pool[layer])
    return pd.paged_decode_attention(q, cache.k_pool[layer], cache.v_pool[layer], tables, lens, **extra).clone()


def step(cache, slots, rows, q):
    """One decode step of `slots` with the given rows: outputs of every layer."""
    cache.advance(1, slots=slots)
    out = []
    for layer, (k, v) in enumerate(rows):
        cache.write(layer, k, v)
        out.append(attend(cache, layer, q))
    return torch.stack(out)


def row_set(n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = [tuple(torch.randn(n, 2, 1, 128, device="cuda", generator=g).half() for _ in range(2)) for _ in range(2)]
    return rows, torch.randn(n, 2, 6, 128, device="cuda", generator=g).half()


def pick(rows, i):
    return [tuple(x[i: i + 1].contiguous() for x in kv) for kv in rows]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("length", [1, 16, 20, 32, 47])
def test_forks_go_on_as_the_source_would(kind, length):
    """A sequence grown token by token, forked twice; all three then take different tokens. Each must
    equal a sequence of another cache that was given the same tokens from the start."""
    cache, alone = make(kind), [make(kind) for _ in range(3)]
    history = [row_set(1, 100 + t) for t in range(length)]
    for rows, q in history:
        step(cache, [2], rows, q)
        for c in alone:
            step(c, [0], rows, q)
    used = cache.allocator.num_used
    cache.fork(2, [0, 5])
    shared = cache.shareable_blocks(2)
    assert cache.tables[0].length == cache.tables[5].length == length
    assert cache.allocator.num_used == used + 2 * (-(-length // 16) - shared)
    assert all(cache.allocator.ref_count(b) == 3 for b in cache.tables[2].blocks[:shared])
    for t in range(20):
        rows, q = row_set(3, 500 + t)
        got = step(cache, [2, 0, 5], rows, q)
        for i in range(3):
            want = step(alone[i], [0], pick(rows, i), q[i: i + 1].contiguous())
            # The batch is cut into other pieces than a sequence alone: partial sums are added up in
            # another order (fp32), weights rounded about another maximum (fp16, 2^-11 each).
            err = (got[:, i].float() - want[:, 0].float()).abs().max()
            assert err <= 2.0 ** -9 * max(1.0, float(want.abs().max()))
    for i in (0, 2, 5):
        cache.free_sequence(i)
    assert cache.allocator.num_used == 0


@pytest.mark.parametrize("kind", KINDS)
def test_compaction_changes_nothing_but_ids(kind):
    cache, same = make(kind), make(kind)
    for c in (cache, same):
        for t in range(21):
            rows, q = row_set(4, 900 + t)
            step(c, [0, 1, 2, 3], rows, q)
        c.free_sequence(1)
        c.free_sequence(0)
        c.fork(2, [4])
    before = [list(t.blocks) for t in cache.tables]
    moves = cache.compact()
    assert moves and cache.allocator.compaction() == {}
    live = {b for t in cache.tables for b in t.blocks}
    assert live == set(range(cache.allocator.num_used))
    assert [list(t.blocks) for t in cache.tables] == [[moves.get(b, b) for b in old] for old in before]
    with pytest.raises(RuntimeError, match="advance"):
        cache.block_tables_tensor()
    for t in range(20):
        rows, q = row_set(3, 700 + t)
        assert torch.equal(step(cache, [2, 3, 4], rows, q), step(same, [2, 3, 4], rows, q))
    assert cache.compact() == {}


def test_fork_refusals_change_nothing():
    cache = make("int4")
    fill(cache, 20, 1, slots=[0, 1])
    state = [(list(t.blocks), t.length) for t in cache.tables]
    for source, targets in [(0, [0]), (0, [1]), (0, [2, 2]), (9, [2]), (0, [-1]), (0, [6])]:
        with pytest.raises(ValueError):
            cache.fork(source, targets)
    hold = cache.allocator.allocate(cache.allocator.num_free - 1)
    with pytest.raises(lc.OutOfBlocks):
        cache.fork(0, [2, 3])
    assert cache.allocator.num_free == 1 and state == [(list(t.blocks), t.length) for t in cache.tables]
    cache.allocator.free(hold)
    cache.fork(4, [5])                                  # an empty sequence
    assert cache.tables[5].length == 0


@pytest.mark.parametrize("kind", ["int4", "fp16"])
def test_rewinding_into_a_shared_page_is_refused(kind):
    cache = make(kind)
    fill(cache, 40, 1, slots=[0])
    cache.fork(0, [1])
    with pytest.raises(ValueError, match="shared"):
        cache.rewind(31, slots=[0])
    with pytest.raises(ValueError, match="shared"):
        cache.rewind(5, slots=[1])
    cache.rewind(33, slots=[0])                         # inside the page of its own
    cache.free_sequence(1)
    cache.rewind(31, slots=[0])
    assert cache.tables[0].length == 31


def test_fork_on_another_stream():
    dev = device()
    cache = make("int4")
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        rows = fill(cache, 23, 3, slots=[1])
        cache.fork(1, [0])
        cache.advance(1, slots=[0])
        k, _ = cache.read(0, 23)
    side.synchronize()
    src = lc.Int4PagedKVCache(spec(), num_blocks=8)
    src.advance(23, slots=[0])
    src.write(0, *rows[0])
    assert torch.equal(k, src.read(0, 23)[0])
