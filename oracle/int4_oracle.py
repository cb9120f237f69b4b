"""numpy restatement, in 64 bits, of the 4-bit cache: the quantiser, the page record and
attention over it. Test infrastructure; shares no code with the library.

The record's layout is stated in csrc/int4_page.cuh; here it is written down once more as the
address of each value (byte and shift of a code, index of a scale).
"""

import numpy as np

PAGE, DIM = 16, 128


def record_bytes(group):
    return 2048 + 128 * (DIM // group)


def quantize(x, group):
    """x [..., 128] -> codes int [..., 128], step, lo fp16 [..., G]."""
    x = np.nan_to_num(np.asarray(x, np.float64), nan=0.0, posinf=65504.0, neginf=-65504.0)
    y = x.reshape(*x.shape[:-1], DIM // group, group)
    lo, hi = y.min(-1), y.max(-1)
    step = ((hi - lo) / 15).astype(np.float16)
    s = step.astype(np.float64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(s > 0, np.rint((y - lo[..., None]) / s), 0.0)
    return np.clip(code, 0, 15).astype(np.int64).reshape(x.shape), step, lo.astype(np.float16)


def dequantize(code, step, lo):
    group = DIM // step.shape[-1]
    wide = lambda t: np.repeat(t.astype(np.float64), group, axis=-1)  # noqa: E731
    return wide(lo) + wide(step) * code


def _addresses(groups):
    t, c = np.meshgrid(np.arange(PAGE), np.arange(DIM), indexing="ij")
    k = (64 * t + 16 * (c % 32 // 8) + 4 * (c // 32) + c % 8 // 2, 4 * (c % 2))
    v = (1024 + 512 * (c // 64) + 16 * (4 * (c % 8) + t % 8 // 2) + 4 * (c % 64 // 16) + 2 * (t % 2) + t // 8,
         4 * (c % 16 // 8))
    t, g = np.meshgrid(np.arange(PAGE), np.arange(groups), indexing="ij")
    k_step = 1024 + t * 2 * groups + g
    v_step = 1024 + 32 * groups + (t % 8 // 2) * 4 * groups + 4 * g + 2 * (t // 8) + t % 2
    return k, v, (k_step, k_step + groups), (v_step, v_step + 16 * groups)


def pack(k_parts, v_parts):
    """(codes [16, 128], step, lo [16, G]) of K and of V -> one record, uint8."""
    groups = k_parts[1].shape[-1]
    (kb, ks), (vb, vs), (kst, klo), (vst, vlo) = _addresses(groups)
    rec = np.zeros(2048 + 128 * groups, np.uint8)
    np.add.at(rec, kb, (k_parts[0] << ks).astype(np.uint8))
    np.add.at(rec, vb, (v_parts[0] << vs).astype(np.uint8))
    half = rec.view(np.float16)
    half[kst], half[klo], half[vst], half[vlo] = k_parts[1], k_parts[2], v_parts[1], v_parts[2]
    return rec


def unpack(rec):
    """One record -> (codes, step, lo) of K and of V."""
    groups = (rec.size - 2048) // 128
    (kb, ks), (vb, vs), (kst, klo), (vst, vlo) = _addresses(groups)
    half = rec.view(np.float16)
    return ((rec[kb].astype(np.int64) >> ks) & 15, half[kst], half[klo]), (
        (rec[vb].astype(np.int64) >> vs) & 15, half[vst], half[vlo])


def rows(pool, table, head, length):
    """K and V [length, 128] of one sequence and head, as the cache holds them; a page whose
    block id lies outside the pool is left out, as the kernel leaves it."""
    ks, vs = [], []
    for page in range(-(-length // PAGE)):
        n = min(PAGE, length - page * PAGE)
        blk = int(table[page])
        if not 0 <= blk < pool.shape[0]:
            continue
        k, v = unpack(np.ascontiguousarray(pool[blk, head]))
        with np.errstate(invalid="ignore"):
            ks.append(dequantize(*k)[:n])
            vs.append(dequantize(*v)[:n])
    if not ks:
        return np.zeros((0, DIM)), np.zeros((0, DIM))
    return np.concatenate(ks), np.concatenate(vs)


def attention(q, pool, tables, lens, scale=None):
    """q [B, H, R, 128], pool uint8 [NB, H, record] -> (out [B, H, R, 128], bound): the output
    in 64 bits and how far an implementation may be from it, element by element:

      2^-11 |out| + 2^-25     rounding the output to fp16
      2 d max|v|              weights off by a factor 1 +- d: scores carry fp32 rounding errors of at most
                              2^-20 of the sum of their terms' magnitudes (about ten roundings of
                              2^-24 each, in accumulators of up to 2^1 times the final sum), exp2 2^-21
      16 N / W 2^-25 (1+step) a weight times a step is held in two fp16 halves, exact to 2^-24 or,
                              where the low half is subnormal, to 2^-25; codes reach 15; N tokens, W = the
                              sum of the weights relative to the largest
    """
    b, h, r, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    out = np.zeros(q.shape)
    bound = np.full(q.shape, 2.0 ** -25)
    for i in range(b):
        for j in range(h):
            k, v = rows(pool, tables[i], j, int(max(lens[i], 0)))
            if not len(k):
                continue
            x = q[i, j].astype(np.float64)
            s = x @ k.T * scale
            w = np.exp(s - s.max(-1, keepdims=True))
            total = w.sum(-1, keepdims=True)
            out[i, j] = (w / total) @ v
            # Magnitudes of the terms: |q| times the largest value that lo + step n is made of.
            terms = np.abs(x).sum(-1, keepdims=True) * 4 * np.abs(k).max() * scale
            delta = 2.0 ** -20 * terms + 2.0 ** -21
            top = np.abs(v).max()
            bound[i, j] += (2.0 ** -11 * np.abs(out[i, j]) + 2 * delta * top
                            + 16 * len(k) / total * 2.0 ** -25 * (1 + top))
    return out, bound
