"""The 4-bit cache's operators without a GPU: the oracle's record, argument checks of the host
side and of the C ABI, the allocator's part of a compaction, rotary frequencies."""

import ctypes
import math

import numpy as np
import pytest
import torch

from latentserve_b200 import _lib, int4_write, page_copy, paged_decode, rotary
from latentserve_b200.cache import BlockAllocator, Int4PagedKVCache, KVCacheSpec
from oracle import int4_oracle as orc


@pytest.mark.parametrize("group", [32, 64, 128])
def test_oracle_record_holds_every_code_and_scale_once(group):
    rng = np.random.default_rng(group)
    k, v = rng.standard_normal((2, 16, 128)).astype(np.float16)
    parts = orc.quantize(k, group), orc.quantize(v, group)
    rec = orc.pack(*parts)
    assert rec.size == orc.record_bytes(group) == int4_write.record_bytes(group)
    for got, want in zip(orc.unpack(rec), parts):
        assert all(np.array_equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_oracle_quantiser_is_off_by_at_most_half_a_step(group):
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((64, 128)) * np.logspace(-2, 3, 64)[:, None]).astype(np.float16)
    code, step, lo = orc.quantize(x, group)
    err = np.abs(orc.dequantize(code, step, lo) - x.astype(np.float64))
    # Half a step, and what fifteen steps rounded to fp16 may miss of the group's range.
    s = np.repeat(step.astype(np.float64), group, -1)
    assert (err <= 0.5 * s + 15 * s * 2.0 ** -11 + 1e-12).all()


def test_refusals_without_a_gpu():
    q = torch.zeros(1, 2, 6, 128, dtype=torch.float16)
    pool = torch.zeros(4, 2, int4_write.record_bytes(32), dtype=torch.uint8)
    tables, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged_decode.paged_decode_attention_int4(q, pool, tables, lens)
    with pytest.raises(RuntimeError, match="no CPU path"):
        int4_write.write(q, q, pool, tables, lens)
    with pytest.raises(RuntimeError, match="no CPU path"):
        int4_write.read(pool, tables, lens, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        page_copy.copy_pages([pool], [0], [1])
    x = torch.zeros(3, 2, 128)
    with pytest.raises(RuntimeError, match="no CPU path"):
        rotary.apply_rotary(x, x, torch.zeros(4, 64), torch.zeros(4, 64), torch.arange(3))
    with pytest.raises(ValueError, match="group"):
        int4_write.record_bytes(16)
    spec = KVCacheSpec(1, 2, 128, 64, 2, device="cpu")
    with pytest.raises(RuntimeError, match="no CPU path"):
        Int4PagedKVCache(spec)
    with pytest.raises(ValueError, match="group"):
        Int4PagedKVCache(spec, group=48)
    with pytest.raises(ValueError, match="fp16"):
        Int4PagedKVCache(KVCacheSpec(1, 2, 128, 64, 2, dtype=torch.bfloat16, device="cpu"))


def test_pool_check():
    ok = torch.zeros(3, 2, 2304, dtype=torch.uint8)
    assert int4_write.pool_ok(ok) and int4_write.groups_of(ok) == 2
    assert not int4_write.pool_ok(ok.to(torch.int8))
    assert not int4_write.pool_ok(torch.zeros(3, 2, 2305, dtype=torch.uint8))
    assert not int4_write.pool_ok(torch.zeros(0, 2, 2304, dtype=torch.uint8))
    assert not int4_write.pool_ok(ok[:, :1].expand(3, 2, 2304))                # heads that overlap
    wide = torch.zeros(3, 2, 2306, dtype=torch.uint8)
    assert not int4_write.pool_ok(wide[:, :, :2304])                           # rows not 16-byte aligned


def test_table_checks():
    lens, tables = torch.ones(2, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    dev = lens.device
    assert int4_write.check_tables(tables, lens, 2, dev) is tables
    narrow = torch.zeros(2, 8, dtype=torch.int32)[:, :3]
    assert int4_write.check_tables(narrow, lens, 2, dev).is_contiguous()
    for bad_t, bad_l in [(tables.long(), lens), (tables, lens.long()), (tables[0], lens), (tables, lens[None]),
                         (tables[:1], lens), (tables, lens[:1]), (tables[:, :0], lens),
                         (tables, torch.ones(4, dtype=torch.int32)[::2])]:
        with pytest.raises(ValueError):
            int4_write.check_tables(bad_t, bad_l, 2, dev)


def test_c_abi_refusals_launch_nothing():
    lib = _lib.lib()
    p = 4096                                            # an aligned address that is never read
    decode = lambda pool=p, groups=4, sp_b=5120, sp_h=2560, r=6, b=1, flags=0, dim=128: lib.ls_paged_decode_int4(  # noqa: E731
        p, pool, p, p, p, p, p, b, 2, r, groups, dim, 16, 4, 8, 16, 8, flags, 1536, 768, 128, sp_b, sp_h, 1536,
        768, 128, 0.1, 0)
    assert decode(pool=0) == -1
    assert decode(b=0) == -2
    assert decode(sp_h=2544) == -3 and decode(pool=p + 8) == -4 and decode(sp_b=5121) == -4
    assert decode(b=1025) == -5
    assert decode(groups=3) == -6 and decode(r=9) == -6 and decode(dim=64) == -6 and decode(flags=0x400) == -6
    for call in (lambda k, groups, n, sk: lib.ls_int4_write(k, p, p, p, p, 0, 1, 2, n, groups, 128, 16, 4, 8, 256, 128, sk,
                                                            256, 128, 128, 5120, 2560, 0),
                 lambda k, groups, n, sk: lib.ls_int4_read(p, k, p, p, p, 0, 1, 2, n, groups, 128, 16, 4, 8, 256, 128, sk,
                                                           256, 128, 128, 5120, 2560, 0)):
        assert call(0, 4, 1, 128) == -1 and call(p, 4, 0, 128) == -2 and call(p, 4, 1, 132) == -4
        assert call(p, 5, 1, 128) == -6 and call(p, 4, (1 << 30) + 1, 128) == -5
    rope = lambda hq, groups: lib.ls_rope_append_int4(p, p, p, p, p, p, p, 1, hq, 2, groups, 128, 16, 64, 8, 2048, 128,  # noqa: E731
                                                      1536, 5120, 2560, 0)
    assert rope(0, 4) == -2 and rope(12, 0) == -6
    rot = lambda n=1, dim=128, r=128, dtype=0, q=p: lib.ls_rotary(q, p, p, p, p, p, p, n, 2, 1, dim, r, dtype, 0, 0, 64, 64,  # noqa: E731
                                                                  256, 128, 128, 128, 256, 128, 128, 128, 0)
    assert rot(q=0) == -1 and rot(n=0) == -2 and rot(r=130) == -2 and rot(r=63) == -2 and rot(dtype=3) == -6


def test_page_copy_refuses_what_would_race():
    lib = _lib.lib()
    pool = (page_copy._Pool * 1)(page_copy._Pool(4096, 0, 256, 256, 1))

    def call(src, dst, pools=pool, blocks=8):
        s, d = (ctypes.c_int32 * len(src))(*src), (ctypes.c_int32 * len(dst))(*dst)
        return lib.ls_copy_pages(pools, 1, s, d, len(src), blocks, 0)

    assert call([0, 1], [2, 2]) == -9                   # a page written twice
    assert call([0, 2], [2, 3]) == -9                   # read and written
    assert call([1], [1]) == -9
    assert call([0], [8]) == -10 and call([-1], [2]) == -10 and call([9], [1]) == -10
    assert call([], []) == 0
    assert call([0], [1], (page_copy._Pool * 1)(page_copy._Pool(4096, 0, 128, 256, 1))) == -3
    assert call([0], [1], (page_copy._Pool * 1)(page_copy._Pool(4096, 128, 256, 256, 2))) == -3
    assert call([0], [1], (page_copy._Pool * 1)(page_copy._Pool(0, 0, 256, 256, 1))) == -1
    assert call([0], [1], (page_copy._Pool * 1)(page_copy._Pool(4096, 0, 256, 256, 0))) == -2
    with pytest.raises(ValueError, match="whole numbers"):
        page_copy._ids([0.5], "src")
    with pytest.raises(ValueError, match="page ids"):
        page_copy._ids([2 ** 31], "src")
    with pytest.raises(ValueError, match="page ids"):
        page_copy._ids([[1, 2]], "src")


def test_allocator_compaction():
    a = BlockAllocator(10, 16)
    blocks = a.allocate(8)                              # 0 .. 7
    a.incref([7])
    a.free([1, 2, 5])
    moves = a.compaction()
    assert moves == {6: 1, 7: 2}                        # five live blocks: 0 1 2 3 4
    a.relocate(moves)
    assert [a.ref_count(b) for b in range(10)] == [1, 1, 2, 1, 1, 0, 0, 0, 0, 0]
    assert a.num_used == 5 and a.allocate(2) == [5, 6]
    assert a.compaction() == {}
    assert blocks == list(range(8))
    full = BlockAllocator(3, 16)
    full.allocate(3)
    assert full.compaction() == {} and BlockAllocator(3, 16).compaction() == {}


def test_rotary_frequencies():
    inv, mag = rotary.rotary_frequencies(64, 1e4)
    assert mag == 1.0 and inv.dtype == torch.float64
    assert torch.allclose(inv, torch.tensor([1e4 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-14)
    lin, _ = rotary.rotary_frequencies(64, 1e4, {"type": "linear", "factor": 4.0})
    assert torch.allclose(lin * 4, inv, rtol=1e-14)
    ntk, _ = rotary.rotary_frequencies(64, 1e4, {"type": "ntk", "factor": 4.0})
    assert math.isclose(ntk[0], 1.0) and math.isclose(ntk[-1] * 4, inv[-1], rel_tol=1e-12)     # the slowest by exactly 4
    yarn, mag = rotary.rotary_frequencies(64, 1e4, {"type": "yarn", "factor": 4.0, "original_max_pos": 4096})
    assert math.isclose(mag, 0.1 * math.log(4.0) + 1)
    turns = inv * 4096 / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], inv[turns > 40])
    assert torch.allclose(yarn[turns < 0.5] * 4, inv[turns < 0.5], rtol=1e-14)
    assert (yarn <= inv * (1 + 1e-15)).all() and (yarn >= inv / 4 * (1 - 1e-15)).all()
    for bad in [dict(type="spline"), dict(type="linear", factor=0.0), dict(type="yarn", factor=2.0),
                dict(type="ntk", factors=2.0)]:
        with pytest.raises(ValueError):
            rotary.rotary_frequencies(64, 1e4, bad)
    with pytest.raises(ValueError):
        rotary.rotary_frequencies(7)


def test_rotary_tables_keep_far_positions():
    cos, sin = rotary.rotary_tables(4, 1_000_001, 1e4, device="cpu")
    far = 1_000_000
    assert abs(float(cos[far, 0]) - math.cos(far)) < 2.0 ** -23 and abs(float(sin[far, 0]) - math.sin(far)) < 2.0 ** -23


def test_binding_declines_what_it_does_not_know():
    """Anything but CUDA tensors of the usual layout: None, no exception, nothing touched."""
    fast = _lib.binding()
    x = torch.zeros(2, 2, 3, 128, dtype=torch.float16)
    pool, tables = torch.zeros(4, 2, 2560, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.int32)
    lens = torch.ones(2, dtype=torch.int32)
    assert fast.decode(x, pool, tables, lens, None, 0.1, 0, 0, 1, 1, 0) is None
    assert fast.decode(x, pool) is None and fast.decode(1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11) is None
    assert fast.write(x, x, pool, tables, lens, None) is None and fast.write(None, x, pool, tables, lens, lens) is None
    assert fast.write(x, x, pool, tables, None, None) is None
    assert fast.read(pool, tables, lens, 4, None) is None and fast.read(pool, tables, lens, "4", None) is None
    assert fast.copy_pages([pool], [0], [1], 0) is None and fast.copy_pages([], [], [], 0) is None
    assert fast.copy_pages((pool,), [0], [1], 0) is None and fast.copy_pages([pool], [0], [1], 7) is None
    y = torch.zeros(3, 2, 64)
    assert fast.rotary(y, y, torch.zeros(4, 32), torch.zeros(4, 32), torch.arange(3), False, False, None, None) is None
    with pytest.raises(TypeError):
        fast.bind(1)
    with pytest.raises(ValueError):
        fast.bind(0, 0, 0, 0, 0)
