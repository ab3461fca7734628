"""Operators of the 8-bit KV cache: what is measured.

Three operators of one path.  ``write`` rotates the queries and keys of new tokens, quantises keys and values with one scale
per token and kv head as it writes them into the paged cache, and (so that what was stored can be compared) reads the
sequences back; ``read`` gives the pages of whole sequences back as fp16, which is what prefill attention reads;
``attend`` is attention of one or a few new tokens of every sequence over the 8-bit pages.

The cache of a layer: ``data`` uint8 [blocks, 2 (K, V), kv heads, block size, head dim] and ``scale`` fp32 [blocks, 2, kv heads,
block size]; the value of an element is (data - 128) * scale.  Block tables [sequences, width] int32, -1 where a block was
dropped.  ``own`` is set by whoever measures: False computes the operators from elementary torch operations, True calls the
framework's.
"""
import functools
import math

import torch

own = False


# ---- cases ------------------------------------------------------------------------------------------------------------------
def _case(name, kind, seqs, lo, hi, nh, nkv, hd, bs, chunk=(1, 1), rot=None, planes=0, bias=0, window=0, holes=0):
    """``seqs`` sequences of lo to hi cached tokens; ``chunk``: new tokens of a sequence, least and most; ``rot``: rotated
    dimensions of a head; ``planes``: fp32 split-K planes the projection comes in (0: fp16 rows); ``holes``: every so-manieth
    block of a sequence was dropped."""
    c = dict(kind=kind, seqs=seqs, lo=lo, hi=hi, nh=nh, nkv=nkv, hd=hd, bs=bs, chunk_lo=chunk[0], chunk_hi=chunk[1],
             rot=rot or hd, planes=planes, bias=bias, window=window, holes=holes)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one sequence decodes: its new token's keys and values, latency is all that counts
        _case("write_one_token", "write", 1, 37, 37, 28, 4, 128, 16),
        # a decode step of a full batch from the QKV product's split-K planes with a bias, short contexts
        _case("write_step_64", "write", 64, 1, 200, 40, 8, 128, 16, planes=4, bias=1),
        # a pass of prompt chunks of three sequences, two with earlier chunks in the cache
        _case("write_chunk", "write", 3, 0, 1500, 40, 8, 128, 16, chunk=(301, 1047)),
        # first chunks of eight prompts, heads of 64 of which 48 dimensions rotate
        _case("write_prompts_64", "write", 8, 0, 0, 32, 8, 64, 32, chunk=(700, 1301), rot=48),
        # a short context read back before the second chunk of a prompt
        _case("read_short", "read", 1, 517, 517, 28, 4, 128, 16),
        # long contexts of four sequences, some of their blocks evicted
        _case("read_long", "read", 4, 9001, 32765, 40, 8, 128, 16, holes=11),
        # a chat's first answer: one short sequence
        _case("attend_one_short", "attend", 1, 300, 300, 28, 4, 128, 16),
        # one sequence with a long document in its context
        _case("attend_one_long", "attend", 1, 32765, 32765, 28, 4, 128, 16),
        # the batch that a server decodes most of the time: 64 sequences of mixed length
        _case("attend_batch_64", "attend", 64, 128, 2300, 40, 8, 128, 16),
        # a full batch of long contexts, the largest work of the path
        _case("attend_long_64", "attend", 64, 6001, 8190, 64, 8, 128, 32),
        # speculative verification: up to five rows of 32 sequences
        _case("attend_verify_32", "attend", 32, 2001, 4094, 40, 8, 128, 16, chunk=(2, 5)),
        # as many kv heads as heads, head dimension 96, a sliding window whose older blocks were dropped
        _case("attend_window_96", "attend", 17, 101, 3999, 32, 32, 96, 16, window=2047),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) )))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend"])
    hd = rng.choice([64, 96, 128, 128, 256])
    nkv = rng.choice([1, 2, 4, 8, 8, 16])
    group = rng.choice([1, 2, 4, 5, 7, 8, 12, 16])
    bs = rng.choice([16, 32, 64])
    rot = rng.choice([hd, hd, hd // 2 // 16 * 16])
    room = {"write": 1 << 24, "read": 1 << 26, "attend": 1 << 28}[kind]     # cached elements of K
    per = nkv * hd
    tokens = _log(rng, 1, max(1, room // per))
    seqs = min(_log(rng, 1, 128), tokens)
    hi = max(1, min(32765, tokens // seqs))
    lo = max(1, int(hi * rng.uniform(0.02, 1.0)))
    if kind == "write":
        most = max(1, min(8192, (1 << 25) // ((group + 2) * per)) // seqs)
        chunk = (1, 1) if rng.random() < 0.4 else (max(1, most // 3), most)
        planes = rng.choice([0, 1, 3, 8]) if chunk[1] * seqs <= 256 else 0
        return _case("", kind, seqs, rng.choice([0, lo]), hi, group * nkv, nkv, hd, bs, chunk=chunk, rot=rot, planes=planes,
                     bias=int(planes > 0 and rng.random() < 0.5), holes=rng.choice([0, 0, 9]))
    if kind == "read":
        return _case("", kind, seqs, lo, hi, group * nkv, nkv, hd, bs, holes=rng.choice([0, 0, 5]))
    chunk = (1, 1) if rng.random() < 0.7 else (1, rng.randint(2, 8))
    return _case("", kind, seqs, lo, hi, group * nkv, nkv, hd, bs, chunk=chunk,
                 window=rng.choice([0, 0, 0, max(1, hi // 3)]), holes=rng.choice([0, 0, 0, 13]))


def _lens(case):
    """(tokens of a sequence cached before the pass, its new tokens), spread over the case's ranges in a fixed order."""
    spread = lambda lo, hi, turn: [lo + int((hi - lo) * ((i * turn + 0.999) % 1.0) + 0.5) for i in range(case["seqs"])]
    new = spread(case["chunk_lo"], case["chunk_hi"], 0.754877666)
    old = spread(case["lo"], case["hi"], 0.618033989)
    if case["kind"] != "write":                 # lo..hi counts all tokens there: what is attended to is in the cache already
        new = [min(n, t) for n, t in zip(new, old)]
        old = [t - n for n, t in zip(new, old)]
    return old, new


def _dropped(case, old, blocks):
    """Blocks of a sequence that are holes: every so-manieth, and what lies before the window of its oldest new row.  The block
    that its new tokens begin in stays."""
    bs, out = case["bs"], set()
    if case["holes"]:
        out |= set(range(case["holes"] // 2, blocks, case["holes"]))
    if case["window"]:
        out |= set(range(0, max(0, old + 1 - case["window"]) // bs))
    return {b for b in out if b < old // bs}


def work(case):
    old, new = _lens(case)
    nh, nkv, hd, bs = case["nh"], case["nkv"], case["hd"], case["bs"]
    row = nkv * 2 * (hd + 4)                    # a token in the cache
    rows, total = sum(new), sum(old) + sum(new)
    width = max(-(-(o + n) // bs) for o, n in zip(old, new))
    gone = sum(len(_dropped(case, o, -(-(o + n) // bs))) for o, n in zip(old, new)) * bs
    tables = case["seqs"] * width * 4
    if case["kind"] == "attend":
        seen = flops = 0
        for o, n in zip(old, new):
            holes = _dropped(case, o, -(-(o + n) // bs))
            first = max(0, o + 1 - case["window"]) if case["window"] else 0
            live = o + n - first - sum(min(bs, (b + 1) * bs - first) for b in holes if (b + 1) * bs > first)
            seen += live
            flops += 4 * nh * hd * n * live
        return {"bytes": seen * row + 2 * rows * nh * hd * 2 + tables + rows * 4, "flops": flops}
    back = (total - gone) * nkv * hd * 2 * 2    # fp16 K and V
    if case["kind"] == "read":
        return {"bytes": (total - gone) * row + back + 2 * tables, "flops": (total - gone) * nkv * hd * 2 * 2}
    width_in = (nh + 2 * nkv) * hd
    given = rows * width_in * (4 * case["planes"] if case["planes"] else 2)
    return {"bytes": given + rows * nh * hd * 2 + rows * row + (total - gone - rows) * row + back + 2 * tables,
            "flops": rows * (nh + nkv) * hd * 3 + (total - gone) * nkv * hd * 4}


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(int(seed) + 1)
    host = torch.Generator().manual_seed(int(seed) + 1)
    nh, nkv, hd, bs, S = case["nh"], case["nkv"], case["hd"], case["bs"], case["seqs"]
    old, new = _lens(case)
    blocks = [-(-(o + n) // bs) for o, n in zip(old, new)]
    width = max(blocks)
    pool = sum(blocks) + sum(blocks) // 16 + 2
    perm = torch.randperm(pool, generator=host, dtype=torch.int32)
    tables = torch.full((S, width), -1, dtype=torch.int32)
    at = 0
    for s in range(S):
        ids = perm[at: at + blocks[s]].clone()
        at += blocks[s]
        for b in _dropped(case, old[s], blocks[s]):
            ids[b] = -1
        tables[s, : blocks[s]] = ids
    # what earlier passes left in the cache: some channels of the keys are much larger than others, values differ by head
    data = torch.empty(pool, 2, nkv, bs, hd, dtype=torch.uint8, device=dev)
    scale = torch.empty(pool, 2, nkv, bs, device=dev)
    size = torch.ones(2, nkv, 1, hd, device=dev)
    size[0] = torch.exp(0.6 * torch.randn(nkv, 1, hd, device=dev, generator=g))
    size[1] = torch.exp(0.5 * torch.randn(nkv, 1, 1, device=dev, generator=g)) * 0.4
    step = max(1, (1 << 25) // (2 * nkv * bs * hd))
    for b in range(0, pool, step):
        x = torch.randn(min(step, pool - b), 2, nkv, bs, hd, device=dev, generator=g) * size
        top = x.abs().amax(-1)
        scale[b: b + step] = top / 127
        data[b: b + step] = torch.round(x * (127 / top)[..., None]) + 128
    st = {"case": case, "data": data, "scale": scale, "tables": tables.to(dev)}
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=dev)
    rows = sum(new)
    seq = [s for s in range(S) for _ in range(new[s])]
    pos = [old[s] + i for s in range(S) for i in range(new[s])]
    st["lens"] = ints([o + n for o, n in zip(old, new)])
    if case["kind"] == "attend":
        st["q"] = (torch.randn(rows, (nh + 2 * nkv) * hd, device=dev, generator=g) * 2).half()   # the QKV rows of the pass
        st["out"] = torch.zeros(rows, nh * hd, dtype=torch.float16, device=dev)
        if case["chunk_hi"] > 1:
            cu = [0]
            for n in new:
                cu.append(cu[-1] + n)
            st["cu_q"], st["pos0"], st["most"] = ints(cu), ints(old), max(new)
        st["row_seq"], st["row_pos"] = ints(seq, torch.int64), ints(pos, torch.int64)
        return st
    cu = [0]
    for n in blocks:
        cu.append(cu[-1] + n)
    st["cu_blocks"] = ints(cu)
    st["pages"] = torch.zeros(cu[-1], 2, nkv, bs, hd, dtype=torch.float16, device=dev)
    st["page_tables"] = torch.full((S, width), -1, dtype=torch.int32, device=dev)
    if case["kind"] == "write":
        cols = (nh + 2 * nkv) * hd
        spread = torch.cat([torch.ones(nh * hd, device=dev), size[0].reshape(-1), size[1].expand(nkv, 1, hd).reshape(-1)])
        if case["planes"]:
            st["planes"] = torch.randn(case["planes"], rows, cols, device=dev, generator=g) * spread / math.sqrt(case["planes"])
            st["bias"] = (torch.randn(cols, device=dev, generator=g) * 0.5).half() if case["bias"] else None
        else:
            st["qkv"] = (torch.randn(rows, cols, device=dev, generator=g) * spread).half()
        st["q_out"] = torch.zeros(rows, cols, dtype=torch.float16, device=dev)
        st["positions"] = ints(pos)
        st["slots"] = ints([int(tables[s, p // bs]) * bs + p % bs for s, p in zip(seq, pos)], torch.int64)
        st["freqs"] = (1e6 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])).float().to(dev)
    return st


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _write_plain(s):
    c = s["case"]
    nh, nkv, hd, bs, half = c["nh"], c["nkv"], c["hd"], c["bs"], c["rot"] // 2
    if c["planes"]:
        x = s["planes"].sum(0)
        if s["bias"] is not None:
            x = x + s["bias"].float()
    else:
        x = s["qkv"].float()
    x = x.view(x.shape[0], nh + 2 * nkv, hd)
    angle = s["positions"].double()[:, None, None] * s["freqs"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = x[:, : nh + nkv, :half], x[:, : nh + nkv, half: 2 * half]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin, x[:, : nh + nkv, 2 * half:]], -1)
    s["q_out"][:, : nh * hd] = turned[:, :nh].clamp(-65504, 65504).reshape(x.shape[0], nh * hd)
    kv = torch.stack([turned[:, nh:], x[:, nh + nkv:]], 1).clamp(-65504, 65504)            # [rows, 2, kv heads, hd]
    top = kv.abs().amax(-1)
    steps = torch.where(top > 1e-30, 127 / top, torch.zeros_like(top))
    block, offset = s["slots"] // bs, s["slots"] % bs
    s["data"][block, :, :, offset] = (torch.round(kv * steps[..., None]) + 128).to(torch.uint8)
    s["scale"][block, :, :, offset] = torch.where(top > 1e-30, top / 127, torch.zeros_like(top))


def _read_plain(s):
    bs, tables, lens = s["case"]["bs"], s["tables"], s["lens"]
    place = torch.arange(tables.shape[1], device=tables.device)
    live = (place < ((lens + bs - 1) // bs)[:, None]) & (tables >= 0)
    to = s["cu_blocks"][:-1, None] + place
    s["page_tables"].copy_(torch.where(live, to, -1))
    seq, at = torch.nonzero(live, as_tuple=True)
    block = tables[seq, at].long()
    x = (s["data"][block].float() - 128) * s["scale"][block][..., None]
    inside = (at[:, None] * bs + torch.arange(bs, device=at.device)) < lens[seq][:, None]
    s["pages"][to[seq, at].long()] = torch.where(inside[:, None, None, :, None], x, torch.zeros_like(x)).half()


def _attend_plain(s):
    c, tables = s["case"], s["tables"]
    nh, nkv, hd, bs = c["nh"], c["nkv"], c["hd"], c["bs"]
    S, width = tables.shape
    L = width * bs
    block = tables.long().clamp_min(0)

    def rows_of(half):
        x = (s["data"][block, half].float() - 128) * s["scale"][block, half][..., None]     # [S, width, kv heads, bs, hd]
        return x.transpose(1, 2).reshape(S, nkv, L, hd)

    # rows of a sequence side by side, padded to the longest
    seq, pos = s["row_seq"], s["row_pos"]
    first = torch.searchsorted(seq, torch.arange(S, device=seq.device))
    at = torch.arange(seq.numel(), device=seq.device) - first[seq]
    R = s["most"] if c["chunk_hi"] > 1 else 1
    q = torch.zeros(S, R, nkv, nh // nkv, hd, device=seq.device)
    q[seq, at] = s["q"][:, : nh * hd].float().view(-1, nkv, nh // nkv, hd)
    sees = torch.full((S, R), -1, dtype=torch.int64, device=seq.device)
    sees[seq, at] = pos
    score = q.permute(0, 2, 1, 3, 4).reshape(S, nkv, -1, hd) @ rows_of(0).transpose(2, 3) * (1 / math.sqrt(hd))
    place = torch.arange(L, device=seq.device)
    seen = (place <= sees[..., None]) & (tables >= 0).repeat_interleave(bs, 1)[:, None]
    if c["window"]:
        seen &= place > sees[..., None] - c["window"]
    seen = seen.repeat_interleave(nh // nkv, 1)[:, None]                                    # [S, 1, R * group, L]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == -math.inf, 0))
    total = p.sum(-1, keepdim=True)
    out = (p / total.masked_fill(total == 0, 1)) @ rows_of(1)
    s["out"].copy_(out.view(S, nkv, R, nh // nkv, hd).permute(0, 2, 1, 3, 4)[seq, at].reshape(-1, nh * hd))


# ---- the framework's operators ------------------------------------------------------------------------------------------------
@functools.lru_cache(None)
def _framework():
    from zse_b200.cache.quant_kv import QuantKV
    from zse_b200.ops.backend import make_ops
    return make_ops("cuda"), QuantKV


def run(state):
    s = state
    c = s["case"]
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    if own:
        ops, QuantKV = _framework()
        kv = QuantKV(s["data"], s["scale"])
        if c["kind"] == "attend":
            ops.attn_decode_q8(s["q"], kv, s["tables"], s["lens"], s["out"], c["seqs"], nh, nkv, hd, 1 / math.sqrt(hd),
                               window=c["window"], cu_q=s.get("cu_q"), q_pos0=s.get("pos0"), max_q=s.get("most", 1))
        else:
            if c["kind"] == "write":
                rows = s["positions"].shape[0]
                ops.rope_kv_write_q8(s.get("qkv"), kv, s["positions"], s["slots"], s["freqs"], rows, nh, nkv, hd,
                                     q_out=s["q_out"], planes=s.get("planes"), n_planes=c["planes"], bias=s.get("bias"))
            ops.kv_read_q8(kv, s["tables"], s["lens"], s["cu_blocks"], c["seqs"], s["pages"], s["page_tables"])
    elif c["kind"] == "attend":
        _attend_plain(s)
    else:
        if c["kind"] == "write":
            _write_plain(s)
        _read_plain(s)
    if c["kind"] == "attend":
        return s["out"]
    out = {"pages": s["pages"], "page_tables": s["page_tables"]}
    return dict(out, q=s["q_out"][:, : nh * hd]) if c["kind"] == "write" else out


# ---- the same in 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """From the definitions, sequence by sequence: rotation, quantisation of (k, v) to round(x / (max|x| / 127)), softmax."""
    s = prepare(case, seed)
    nh, nkv, hd, bs, S = case["nh"], case["nkv"], case["hd"], case["bs"], case["seqs"]
    old, new = _lens(case)
    dev, f64 = s["data"].device, torch.float64
    tables = s["tables"].tolist()
    group = nh // nkv

    def cached(i, count):
        """K and V [count, kv heads, hd] of sequence i, and which of its tokens are there."""
        ids = torch.tensor(tables[i][: -(-count // bs)], device=dev)
        there = (ids >= 0).repeat_interleave(bs)[:count]
        at = torch.arange(count, device=dev)
        b = ids.clamp_min(0)[at // bs]
        x = s["data"][b, :, :, at % bs].to(f64) - 128
        return x[:, 0] * s["scale"][b, 0, :, at % bs].to(f64)[..., None], x[:, 1] * s["scale"][b, 1, :, at % bs].to(f64)[..., None], there

    if case["kind"] == "attend":
        out, row = torch.zeros(sum(new), nh * hd, dtype=f64, device=dev), 0
        for i in range(S):
            count = old[i] + new[i]
            k, v, there = cached(i, count)
            at = torch.arange(count, device=dev)
            for r in range(new[i]):
                p = old[i] + r
                see = there & (at <= p)
                if case["window"]:
                    see &= at > p - case["window"]
                q = s["q"][row, : nh * hd].to(f64).view(nkv, group, hd)
                z = torch.einsum("hgd,thd->hgt", q, k[see]) / math.sqrt(hd)
                if z.shape[-1]:
                    out[row] = torch.einsum("hgt,thd->hgd", torch.softmax(z, -1), v[see]).reshape(-1)
                row += 1
        return out
    cu = s["cu_blocks"].tolist()
    pages = torch.zeros(cu[-1], 2, nkv, bs, hd, dtype=f64, device=dev)
    page_tables = torch.full(s["page_tables"].shape, -1, dtype=torch.int64)
    q_out, row = None, 0
    if case["kind"] == "write":
        x = s["planes"].to(f64).sum(0) if case["planes"] else s["qkv"].to(f64)
        if s.get("bias") is not None:
            x = x + s["bias"].to(f64)
        x = x.view(-1, nh + 2 * nkv, hd).clone()
        half = case["rot"] // 2
        turn = s["positions"].to(f64)[:, None] * s["freqs"].to(f64)
        z = torch.complex(x[:, : nh + nkv, :half], x[:, : nh + nkv, half: 2 * half]) * torch.polar(torch.ones_like(turn), turn)[:, None]
        x[:, : nh + nkv, :half], x[:, : nh + nkv, half: 2 * half] = z.real, z.imag
        q_out = x[:, :nh].reshape(-1, nh * hd)
        x = x[:, nh:].reshape(-1, 2, nkv, hd)
        unit = x.abs().amax(-1, keepdim=True) / 127
        x = torch.round(x / unit) * unit
    for i in range(S):
        count = old[i] + new[i]
        k, v, there = cached(i, count)
        if case["kind"] == "write":
            k[old[i]:], v[old[i]:] = x[row: row + new[i], 0], x[row: row + new[i], 1]
            row += new[i]
        at = torch.arange(count, device=dev)[there]
        for half_, y in ((0, k), (1, v)):
            pages[cu[i] + at // bs, half_, :, at % bs] = y[there]
        for b in range(-(-count // bs)):
            if tables[i][b] >= 0:
                page_tables[i, b] = cu[i] + b
    out = {"pages": pages, "page_tables": page_tables.int().to(dev)}
    return dict(out, q=q_out) if case["kind"] == "write" else out
