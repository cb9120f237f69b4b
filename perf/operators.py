"""The operators around a cache held in 4 bits: what is timed, on which cases, in which plain form.

    decode   attention of one new token per sequence over a paged 4-bit cache
    write    quantising new K / V rows into the cache's pages, and reading them back
    copy     copying pages inside every layer's pools (forks, compaction)
    rotary   rotary positions of queries and keys, half or interleaved layout, part of the
             head, frequencies scaled for long contexts

A page of the 4-bit cache holds 16 tokens of one KV head (head_dim 128) as ONE record of bytes,
`kv_pool` uint8 [num_blocks, H, 2048 + 128 G], G = 128 / group scales per token and side. A
value stands for lo + step * code: lo and step fp16 per (token, head, group of channels), code
0..15.
    bytes 0..1023      K codes. Token t at 64 t: [j 4][q 4][byte 4], low nibble first; nibble i of
                       the word (q, j) is channel 32 q + 8 j + i.
    bytes 1024..2047   V codes, [c 2][g 8][j 4][i 4][e 2][f 2]: the byte holds token 8 f + 2 j + e,
                       channel 64 c + 16 i + g in its low nibble and that channel + 8 in its high one.
    then               K scales fp16 [16 tokens][step, lo][G]
    then               V steps fp16 [j 4][G][f 2][e 2], then V lows in the same order
"""

import math

import torch

own = False

PAGE, DIM = 16, 128
DEV = "cuda"


# ---------------------------------------------------------------------------- cases

def listed():
    return [
        # One short sequence: what a single user's first tokens cost, all latency.
        dict(name="decode_b1_1k", op="decode", batch=1, low=1000, high=1000, heads=2, rep=6, group=32),
        # The benchmark's dense batch, every sequence at 16 384 tokens.
        dict(name="decode_b16_16k", op="decode", batch=16, low=16384, high=16384, heads=2, rep=6, group=32),
        # The benchmark's ragged serving batch, at the coarsest scales.
        dict(name="decode_b64_1k_32k", op="decode", batch=64, low=1024, high=32768, heads=2, rep=6, group=128),
        # A model with more KV heads at long contexts: the largest cache read.
        dict(name="decode_b32_8k_32k_h8", op="decode", batch=32, low=8192, high=32768, heads=8, rep=4, group=64),
        # One decode step's append of a full serving batch.
        dict(name="write_b64_step", op="write", batch=64, tokens=1, even=True, before=4099, heads=2, group=32),
        # Ragged prompt chunks that start and end inside pages.
        dict(name="write_b4_chunk", op="write", batch=4, tokens=2048, even=False, before=5003, heads=2, group=64),
        # Whole prompts of a model with more heads.
        dict(name="write_b8_prompt_h8", op="write", batch=8, tokens=8197, even=True, before=0, heads=8, group=32),
        # Forking one sequence into three: the partly filled last page, in all 28 layers.
        dict(name="copy_fork3", op="copy", layers=28, blocks=64, pairs=3, same_source=True, heads=2),
        # Compacting a pool of 1024 blocks: half of them move.
        dict(name="copy_compact512", op="copy", layers=28, blocks=1024, pairs=512, same_source=False, heads=2),
        # A decode step's queries and keys far out in a scaled context.
        dict(name="rotary_b16_step", op="rotary", tokens=16, far=131072, q_heads=12, k_heads=2, dim=128, rotary=128,
             interleaved=False, dtype="float16", scaling="yarn", factor=4.0),
        # A prompt of odd length, half of each head rotated, in 32 bits.
        dict(name="rotary_8k_partial", op="rotary", tokens=8191, far=8191, q_heads=12, k_heads=2, dim=128, rotary=64,
             interleaved=True, dtype="float32", scaling="none", factor=1.0),
        # A long prompt of a wide model.
        dict(name="rotary_32k_wide", op="rotary", tokens=32768, far=32768, q_heads=32, k_heads=8, dim=128, rotary=128,
             interleaved=False, dtype="bfloat16", scaling="ntk", factor=2.0),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "write", "copy", "rotary"])
    if op == "decode":
        heads = rng.choice([1, 2, 4, 8])
        high = _log(rng, 1, 32768)
        # No more cells than the widest listed case has, padding included.
        batch = min(_log(rng, 1, 64), max(1, 64 * 32768 * 2 // (high * heads)))
        return dict(op=op, batch=batch, low=rng.randint(0, high), high=high, heads=heads, rep=rng.randint(1, 8),
                    group=rng.choice([32, 64, 128]))
    if op == "write":
        heads = rng.choice([1, 2, 4, 8])
        tokens = _log(rng, 1, 8197)
        batch = min(_log(rng, 1, 64), max(1, 8 * 8197 * 8 // (tokens * heads)))
        return dict(op=op, batch=batch, tokens=tokens, even=rng.random() < 0.5, before=rng.randint(0, 6000),
                    heads=heads, group=rng.choice([32, 64, 128]))
    if op == "copy":
        blocks = _log(rng, 8, 1024)
        return dict(op=op, layers=rng.randint(1, 28), blocks=blocks, pairs=_log(rng, 1, blocks // 2),
                    same_source=rng.random() < 0.3, heads=rng.choice([1, 2]))
    dim = rng.choice([64, 80, 96, 128])
    q_heads, k_heads = rng.choice([(12, 2), (32, 4), (20, 4), (5, 5), (7, 1)])
    tokens = _log(rng, 1, 16384)
    scaling = rng.choice(["none", "linear", "ntk", "yarn"])
    return dict(op=op, tokens=tokens, far=tokens + rng.randint(0, 100000), q_heads=q_heads, k_heads=k_heads, dim=dim,
                rotary=rng.choice([dim, dim // 2, 32]), interleaved=rng.random() < 0.5,
                dtype=rng.choice(["float16", "bfloat16", "float32"]), scaling=scaling,
                factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]))


# ---------------------------------------------------------------------------- the record, plainly

def _fit(x, group):
    """x fp16 [..., 128] -> codes uint8 [..., 128], step and lo fp16 [..., G]."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=65504.0, neginf=-65504.0)
    x = x.unflatten(-1, (DIM // group, group))
    lo, hi = x.amin(-1), x.amax(-1)
    step = ((hi - lo) / torch.full((), 15.0, device=x.device)).half()
    s = step.float().unsqueeze(-1)
    code = torch.round((x - lo.unsqueeze(-1)) / torch.where(s > 0, s, torch.ones_like(s))).clamp_(0, 15)
    code = torch.where(s > 0, code, torch.zeros_like(code))
    return code.to(torch.uint8).flatten(-2), step, lo.half()


def _offsets(tok, groups):
    """tok [N] -> byte offsets [N, 128 + 8 G] of one token's bytes inside its page's record:
    64 bytes of K codes, 64 of V codes, K steps and lows, V steps, V lows."""
    dev = tok.device
    f, j, e = tok // 8, tok % 8 // 2, tok % 2
    at = torch.arange(64, device=dev)
    kc = 64 * tok[:, None] + at
    vc = 1024 + 512 * (at // 32) + 64 * (at % 32 // 4) + 4 * (at % 4) + (16 * j + 2 * e + f)[:, None]
    ks = 2048 + 4 * groups * tok[:, None] + torch.arange(4 * groups, device=dev)
    two = torch.arange(2 * groups, device=dev)
    vs = 2048 + 64 * groups + 8 * groups * j[:, None] + 8 * (two // 2) + (4 * f + 2 * e)[:, None] + two % 2
    return torch.cat([kc, vc, ks, vs, vs + 32 * groups], dim=1)


def _image(kc, ks, kl, vc, vs, vl):
    """One token's bytes in the order of `_offsets`, [..., 128 + 8 G]."""
    k = kc.unflatten(-1, (4, 4, 4, 2)).transpose(-4, -3)          # [q][j][byte][nibble] -> [j][q][byte][nibble]
    k = (k[..., 0] | (k[..., 1] << 4)).flatten(-3)
    v = vc.unflatten(-1, (2, 4, 2, 8))                            # [c][i][nibble][g] -> [c][g][i]
    v = (v[..., 0, :] | (v[..., 1, :] << 4)).transpose(-1, -2).flatten(-3)
    def as_bytes(t):
        return t.contiguous().view(torch.uint8)
    return torch.cat([k, v, as_bytes(torch.cat([ks, kl], -1)), as_bytes(vs), as_bytes(vl)], dim=-1)


def _values(image, groups):
    """The inverse of `_image`: K and V in 32 bits, [..., 128] each."""
    k, v, ks, vs, vl = image.split([64, 64, 4 * groups, 2 * groups, 2 * groups], dim=-1)
    k = k.unflatten(-1, (4, 4, 4))
    k = torch.stack([k & 15, k >> 4], -1).transpose(-4, -3).flatten(-4).float()
    v = v.unflatten(-1, (2, 8, 4)).transpose(-1, -2)
    v = torch.stack([v & 15, v >> 4], -2).flatten(-4).float()
    ks, kl = ks.contiguous().view(torch.float16).float().split(groups, dim=-1)
    vs, vl = (t.contiguous().view(torch.float16).float() for t in (vs, vl))
    group = DIM // groups
    def wide(t):
        return t.repeat_interleave(group, dim=-1)
    return wide(kl) + wide(ks) * k, wide(vl) + wide(vs) * v


def _page_values(rec, groups):
    """Whole records uint8 [..., R] -> K, V in 32 bits, [..., 16, 128]."""
    lead = rec.dim() - 1
    k = rec[..., :1024].unflatten(-1, (16, 4, 4, 4))
    k = torch.stack([k & 15, k >> 4], -1).transpose(-4, -3).flatten(-4).float()
    v = rec[..., 1024:2048].unflatten(-1, (2, 8, 4, 4, 2, 2))
    v = torch.stack([v & 15, v >> 4], -1)                         # c g j i e f nibble
    c, g, j, i, e, f, s = range(lead, lead + 7)
    v = v.permute(*range(lead), f, j, e, c, i, s, g).flatten(-4).flatten(-4, -2).float()
    half = rec[..., 2048:].contiguous().view(torch.float16).float()
    ks, vs, vl = half.split([32 * groups, 16 * groups, 16 * groups], dim=-1)
    ks = ks.unflatten(-1, (16, 2, groups))
    def tokens(t):                                                # [j][G][f][e] -> [token][G]
        t = t.unflatten(-1, (4, groups, 2, 2))
        return t.permute(*range(lead), lead + 2, lead, lead + 3, lead + 1).flatten(-4, -2)
    group = DIM // groups
    def wide(t):
        return t.repeat_interleave(group, dim=-1)
    return wide(ks[..., 1, :]) + wide(ks[..., 0, :]) * k, wide(tokens(vl)) + wide(tokens(vs)) * v


# ---------------------------------------------------------------------------- inputs

def _lens(case, seed):
    g = torch.Generator().manual_seed(seed * 7919 + 13)
    low, high = case["low"], case["high"]
    u = torch.rand(case["batch"], generator=g, dtype=torch.float64)
    a, b = math.log(low + 1), math.log(high + 1)
    lens = torch.exp(a + u * (b - a)).sub(1).round().long().clamp(low, high)
    lens[0] = high
    return lens.tolist()


def _tables(lens, blocks, seed):
    """Shuffled block tables over a pool with room to spare."""
    g = torch.Generator().manual_seed(seed * 31 + 5)
    pages = [-(-n // PAGE) for n in lens]
    order = torch.randperm(blocks, generator=g, dtype=torch.int32)
    out = torch.zeros(len(lens), max(1, max(pages)), dtype=torch.int32)
    at = 0
    for row, n in enumerate(pages):
        out[row, :n] = order[at: at + n]
        at += n
    return out.to(DEV)


def _inv_freq(case):
    """Rotary frequencies fp64 [rotary / 2] and the factor on cos and sin."""
    n, theta, factor = case["rotary"], 1e6, case["factor"]
    if case["scaling"] == "ntk":
        theta = theta * factor ** (n / (n - 2))
    inv = theta ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    if case["scaling"] == "linear":
        inv = inv / factor
    if case["scaling"] != "yarn":
        return inv, 1.0
    # Dimensions that turn more than 32 times in the original window keep their frequency, those
    # that turn less than once are stretched, the ones between are blended.
    window = 32768
    def at(turns):
        return n * math.log(window / (turns * 2 * math.pi)) / (2 * math.log(theta))
    first, last = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), n - 1)
    ramp = ((torch.arange(n // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0, 1)
    return inv / factor * ramp + inv * (1 - ramp), 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, dtype=torch.float16):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)

    if case["op"] == "rotary":
        dtype = getattr(torch, case["dtype"])
        t, hq, hk, d = case["tokens"], case["q_heads"], case["k_heads"], case["dim"]
        # Queries and keys are views of the fused projection's rows, as a model has them.
        qkv = normal(t, (hq + 2 * hk) * d, dtype=dtype)
        first = case["far"] - t
        inv, mag = _inv_freq(case)
        angle = torch.arange(case["far"], dtype=torch.float64, device=DEV)[:, None] * inv.to(DEV)
        return dict(case=case, q=qkv[:, : hq * d].view(t, hq, d), k=qkv[:, hq * d: (hq + hk) * d].view(t, hk, d),
                    cos=(angle.cos() * mag).float(), sin=(angle.sin() * mag).float(),
                    positions=torch.arange(first, first + t, device=DEV))
    if case["op"] == "copy":
        pools = normal(2 * case["layers"], case["blocks"], PAGE, case["heads"], DIM)
        order = torch.randperm(case["blocks"], generator=torch.Generator().manual_seed(seed)).tolist()
        n = case["pairs"]
        src = [order[n]] * n if case["same_source"] else order[n: 2 * n]
        return dict(case=case, pools=pools, src=src, dst=order[:n])
    heads, groups = case["heads"], DIM // case["group"]
    if case["op"] == "write":
        b, n = case["batch"], case["tokens"]
        new = [n] * b
        if not case["even"]:
            new = torch.randint(0, n + 1, (b,), generator=torch.Generator().manual_seed(seed + 1)).tolist()
            new[0] = n
        lens = [case["before"] + 3 * i + m for i, m in enumerate(new)]
        blocks = int(1.2 * sum(-(-m // PAGE) for m in lens)) + 8
        kv = normal(b, n, 2 * heads, DIM)                        # the projection's K and V rows
        return dict(case=case, k=kv[:, :, :heads].transpose(1, 2), v=kv[:, :, heads:].transpose(1, 2),
                    kv_pool=torch.zeros(blocks, heads, 2048 + 128 * groups, dtype=torch.uint8, device=DEV),
                    tables=_tables(lens, blocks, seed),
                    lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                    new=torch.tensor(new, dtype=torch.int32, device=DEV),
                    start=torch.tensor([m - x for m, x in zip(lens, new)], dtype=torch.int32, device=DEV))
    lens = _lens(case, seed)
    blocks = int(1.2 * sum(-(-m // PAGE) for m in lens)) + 8
    pool = torch.empty(blocks, heads, 2048 + 128 * groups, dtype=torch.uint8, device=DEV)
    flat = _offsets(torch.arange(PAGE, device=DEV), groups).reshape(-1)
    shift = normal(2, heads, DIM) * 0.5                           # channels' own means
    for at in range(0, blocks, 2048):                             # in pieces: the pool is large
        m = min(2048, blocks - at)
        k, v = normal(m, heads, PAGE, DIM) + shift[0][:, None], normal(m, heads, PAGE, DIM) + shift[1][:, None]
        image = _image(*_fit(k, case["group"]), *_fit(v, case["group"]))
        pool[at: at + m, :, flat] = image.flatten(-2)
    return dict(case=case, q=normal(case["batch"], heads, case["rep"], DIM), kv_pool=pool,
                tables=_tables(lens, blocks, seed), lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                max_len=max(lens))


# ---------------------------------------------------------------------------- one pass

def _run_decode(state):
    q, pool, tables, lens = state["q"], state["kv_pool"], state["tables"], state["lens"]
    if own:
        from latentserve_b200 import paged_decode as pd
        return pd.paged_decode_attention_int4(q, pool, tables, lens, max_seq_len=state["max_len"])
    groups = DIM // state["case"]["group"]
    k, v = _page_values(pool[tables.long()].transpose(1, 2), groups)      # [B, H, pages, 16, 128]
    k, v = k.flatten(2, 3), v.flatten(2, 3)
    s = (q.float() @ k.transpose(-1, -2)) * DIM ** -0.5
    gone = torch.arange(k.shape[2], device=q.device) >= lens[:, None]
    s = s.masked_fill(gone[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(top > float("-inf"), top, torch.zeros_like(top)))
    return ((w @ v) / w.sum(-1, keepdim=True).clamp(min=1e-20)).half()


def _run_write(state):
    k, v, pool, tables = state["k"], state["v"], state["kv_pool"], state["tables"]
    lens, new, start, n = state["lens"], state["new"], state["start"], state["case"]["tokens"]
    if own:
        from latentserve_b200 import int4_write
        int4_write.write(k, v, pool, tables, lens, None if state["case"]["even"] else new)
        return int4_write.read(pool, tables, lens, n, start=start)
    group = state["case"]["group"]
    groups = DIM // group
    image = _image(*_fit(k, group), *_fit(v, group)).transpose(1, 2)      # [B, n, H, bytes]
    row, col = (torch.arange(n, device=k.device) < new[:, None]).nonzero(as_tuple=True)
    pos = start.long()[row] + col
    block = tables[row, pos // PAGE].long()[:, None, None]
    head = torch.arange(k.shape[1], device=k.device)[:, None]
    offset = _offsets(pos % PAGE, groups)[:, None, :]
    pool[block, head, offset] = image[row, col]
    kk, vv = _values(pool[block, head, offset], groups)
    out_k, out_v = k.new_zeros(k.shape[0], n, k.shape[1], DIM), k.new_zeros(k.shape[0], n, k.shape[1], DIM)
    out_k[row, col], out_v[row, col] = kk.half(), vv.half()
    return out_k.transpose(1, 2).contiguous(), out_v.transpose(1, 2).contiguous()


def _run_copy(state):
    pools = state["pools"]
    if own:
        from latentserve_b200 import page_copy
        page_copy.copy_pages([pools], state["src"], state["dst"], block_dim=1)
        return pools
    src, dst = (torch.tensor(x, device=pools.device) for x in (state["src"], state["dst"]))
    pools[:, dst] = pools[:, src]
    return pools


def _run_rotary(state):
    q, k, cos, sin, positions = (state[x] for x in ("q", "k", "cos", "sin", "positions"))
    case = state["case"]
    if own:
        from latentserve_b200 import rotary
        return rotary.apply_rotary(q, k, cos, sin, positions, interleaved=case["interleaved"])
    c, s = cos[positions][:, None], sin[positions][:, None]

    def turn(x):
        y = x.float()
        r = y[..., : case["rotary"]]
        if case["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
        else:
            a, b = r.chunk(2, -1)
            r = torch.cat([a * c - b * s, b * c + a * s], -1)
        return torch.cat([r, y[..., case["rotary"]:]], -1).to(x.dtype)

    return turn(q), turn(k)


def run(state):
    return {"decode": _run_decode, "write": _run_write, "copy": _run_copy, "rotary": _run_rotary}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "copy":
        moved = 2 * case["layers"] * case["pairs"] * PAGE * case["heads"] * DIM * 2
        distinct = moved // case["pairs"] if case["same_source"] else moved
        return dict(bytes=distinct + moved, flops=0)
    if case["op"] == "rotary":
        size = 4 if case["dtype"] == "float32" else 2
        rows = case["tokens"] * (case["q_heads"] + case["k_heads"])
        return dict(bytes=2 * rows * case["dim"] * size + case["tokens"] * (case["rotary"] * 4 + 8),
                    flops=3 * rows * case["rotary"])
    token = case["heads"] * (128 + 8 * (DIM // case["group"]))    # bytes of one token, all heads, K and V
    if case["op"] == "write":
        # fp16 rows in, codes and scales out, and back: codes in, fp16 rows out.
        count = case["batch"] * case["tokens"] if case["even"] else case["batch"] * case["tokens"] // 2
        return dict(bytes=count * (2 * token + 2 * 2 * case["heads"] * DIM * 2), flops=count * case["heads"] * DIM * 16)
    low, high = case["low"] + 1, case["high"] + 1
    mean = high if low == high else (high - low) / math.log(high / low)
    tokens = int(case["batch"] * mean)
    rows = case["batch"] * case["heads"] * case["rep"] * DIM
    return dict(bytes=tokens * token + tokens // PAGE * 4 + 2 * 2 * rows, flops=4 * tokens * case["heads"] * case["rep"] * DIM)


# ---------------------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    if case["op"] == "copy":
        return None
    state = prepare(case, seed)
    if case["op"] == "rotary":
        inv, mag = _inv_freq(case)
        angle = state["positions"].double()[:, None] * inv.to(DEV)
        z = torch.polar(torch.full_like(angle, mag), angle)[:, None]

        def turn(x):
            y = x.double().clone()
            n = case["rotary"]
            even = slice(0, n, 2) if case["interleaved"] else slice(0, n // 2)
            odd = slice(1, n, 2) if case["interleaved"] else slice(n // 2, n)
            r = torch.complex(y[..., even].contiguous(), y[..., odd].contiguous()) * z
            y[..., even], y[..., odd] = r.real, r.imag
            return y

        return turn(state["q"]), turn(state["k"])
    group = case["group"]
    groups = DIM // group
    if case["op"] == "write":
        keep = (torch.arange(case["tokens"], device=DEV) < state["new"][:, None])[:, None, :, None]

        def held(x):
            out = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
            for at in range(0, DIM, group):
                y = x[..., at: at + group].double()
                lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
                step = ((hi - lo) / 15).half().double()
                code = torch.where(step > 0, torch.round((y - lo) / step), 0.0).clamp(0, 15)
                out[..., at: at + group] = lo + step * torch.nan_to_num(code)
            return out * keep

        return held(state["k"]), held(state["v"])
    # Attention, sequence by sequence, each value looked up by the record's own addresses.
    tok, ch = torch.arange(PAGE, device=DEV)[:, None], torch.arange(DIM, device=DEV)[None, :]
    k_byte = 64 * tok + 16 * (ch % 32 // 8) + 4 * (ch // 32) + ch % 8 // 2
    k_shift = (4 * (ch % 2)).expand(PAGE, DIM)
    v_byte = (1024 + 512 * (ch // 64) + 16 * (4 * (ch % 8) + tok % 8 // 2) + 4 * (ch % 64 // 16) + 2 * (tok % 2) + tok // 8)
    v_shift = (4 * (ch % 16 // 8)).expand(PAGE, DIM)
    grp = ch // group
    k_step = 1024 + tok * 2 * groups + grp
    v_step = 1024 + 32 * groups + (tok % 8 // 2) * 4 * groups + 4 * grp + 2 * (tok // 8) + tok % 2
    out = torch.zeros(case["batch"], case["heads"], case["rep"], DIM, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lens(case, seed)):
        if n == 0:
            continue
        rec = state["kv_pool"][state["tables"][b, : -(-n // PAGE)].long()].transpose(0, 1)      # [H, pages, R]
        half = rec.contiguous().view(torch.float16)

        def side(byte, shift, step, low):
            code = (rec[:, :, byte] >> shift) & 15
            return (half[:, :, low].double() + half[:, :, step].double() * code.double()).flatten(1, 2)[:, :n]

        k = side(k_byte, k_shift, k_step, k_step + groups)
        p = torch.softmax(torch.einsum("hrd,htd->hrt", state["q"][b].double(), k) / math.sqrt(DIM), -1)
        out[b] = torch.einsum("hrt,htd->hrd", p, side(v_byte, v_shift, v_step, v_step + 16 * groups))
    return out
