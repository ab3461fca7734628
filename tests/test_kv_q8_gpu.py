"""Kernels of the 8-bit KV cache (csrc/kv_q8.cu, csrc/attention_q8.cu) against 64 bits: sizes, masks and contents where they can go
wrong, and the three of them together as a layer uses them."""
import pytest
import torch

from tests.helpers.kv_q8_oracle import attention, check_write, make_cache, make_tables, scale_of
from zse_b200.cache.quant_kv import QuantKV

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from zse_b200.ops.backend import make_ops
    return make_ops(DEV)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def freqs_of(rot, theta=1e6):
    return (theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).float().to(DEV)


# ---- write ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 16), (96, 96), (96, 48), (128, 128), (128, 96), (256, 256), (128, 0)])
@pytest.mark.parametrize("nh,nkv,M", [(4, 2, 1), (7, 1, 5), (40, 8, 33), (16, 16, 200)])
@pytest.mark.parametrize("planes,bias", [(0, False), (1, False), (3, True), (9, True)])
def test_write(ops, hd, rot, nh, nkv, M, planes, bias):
    g = gen(hd * 1000 + rot * 10 + M + planes)
    bs, blocks, cols = 16, M // 16 + 3, (nh + 2 * nkv) * hd
    pos = torch.randint(0, 40000, (M,), generator=g, dtype=torch.int32)
    pos[0] = 2 ** 31 - 1
    pos[-1] = 131071 if M > 1 else 2 ** 31 - 1
    slots = torch.randperm(blocks * bs, generator=g)[:M]
    slots[M // 2] = -1 if M > 1 else slots[0]
    kv = QuantKV(torch.full((blocks, 2, nkv, bs, hd), 77, dtype=torch.uint8, device=DEV),
                 torch.full((blocks, 2, nkv, bs), 7.0, device=DEV))
    qkv = torch.randn(M, cols + 24, generator=g).half().to(DEV)           # rows further apart than they are wide
    before = qkv.clone()
    p = b = None
    x = qkv[:, :cols].double()
    if planes:
        p = torch.randn(planes, M, cols, generator=g).to(DEV)
        b = torch.randn(cols, generator=g).half().to(DEV) if bias else None
        # the kernel's own sum: the bias, then plane by plane, in fp32
        acc = b.float().expand(M, cols) if bias else torch.zeros(M, cols, device=DEV)
        for i in range(planes):
            acc = acc + p[i]
        x = acc.double()
    ops.rope_kv_write_q8(qkv, kv, pos.to(DEV), slots.to(DEV), freqs_of(rot), M, nh, nkv, hd, planes=p, n_planes=planes, bias=b)
    torch.cuda.synchronize()
    ops.check()
    assert torch.equal(qkv[:, nh * hd:], before[:, nh * hd:])
    kept = slots >= 0
    blk, off = (slots.clamp_min(0) // bs).to(DEV), (slots.clamp_min(0) % bs).to(DEV)
    u, sc = kv.data[blk, :, :, off], kv.scale[blk, :, :, off]
    k = kept.to(DEV)
    check_write(x[k], pos.to(DEV)[k], freqs_of(rot), nh, nkv, hd, qkv[k, : nh * hd], u[k], sc[k])
    if not kept.all():                                                     # q of rows that are not stored is rotated too
        i = int((~kept).nonzero()[0])
        from tests.helpers.kv_q8_oracle import rotated
        h, pair = rotated(x[i: i + 1], pos[i: i + 1].to(DEV), freqs_of(rot), nh, nkv, hd)
        want, wide = h[0, :nh].reshape(-1), pair[0, :nh].reshape(-1)
        assert ((qkv[i, : nh * hd].double() - want).abs() <= want.abs() * 2.0 ** -11 + wide * 2.0 ** -21 + 2.0 ** -25).all()
    free = torch.ones(blocks * bs, dtype=torch.bool)
    free[slots[kept]] = False
    flat = lambda t: t.transpose(1, 3).reshape(blocks * bs, -1)
    assert (flat(kv.data)[free.to(DEV)] == 77).all() and (kv.scale.permute(0, 3, 1, 2).reshape(blocks * bs, -1)[free.to(DEV)] == 7).all()


def test_write_to_a_place_of_its_own(ops):
    nh, nkv, hd, M = 6, 2, 64, 19
    g = gen(3)
    qkv = torch.randn(M, (nh + 2 * nkv) * hd, generator=g).half().to(DEV)
    before, q = qkv.clone(), torch.full((M + 1, nh * hd + 8), 5.0, dtype=torch.float16, device=DEV)
    kv, kv2 = (QuantKV.zeros((2, 2, nkv, 16, hd), DEV) for _ in range(2))
    args = (ints(list(range(M))), ints(list(range(M)), torch.int64), freqs_of(hd), M, nh, nkv, hd)
    ops.rope_kv_write_q8(qkv, kv, *args, q_out=q)
    assert torch.equal(qkv, before) and (q[M] == 5).all() and (q[:, nh * hd:] == 5).all()
    ops.rope_kv_write_q8(qkv, kv2, *args)
    assert torch.equal(qkv[:, : nh * hd], q[:M, : nh * hd]) and torch.equal(kv.data, kv2.data) and torch.equal(kv.scale, kv2.scale)


def test_rows_of_zeros_infinities_and_nan(ops):
    nh, nkv, hd, M = 2, 2, 64, 4
    x = torch.randn(M, (nh + 2 * nkv) * hd, generator=gen(5)).half()
    k, v = slice(nh * hd, (nh + 1) * hd), slice((nh + nkv) * hd, (nh + nkv + 1) * hd)
    x[0, k] = 0
    x[1, v] = 0
    x[1, v.start + 5] = float("inf")
    x[2, v.start + 7] = float("-inf")
    x[3, v.start + 9] = float("nan")
    kv = QuantKV.zeros((1, 2, nkv, 16, hd), DEV)
    ops.rope_kv_write_q8(x.to(DEV), kv, ints([0] * M), ints([0, 1, 2, 3], torch.int64), freqs_of(hd), M, nh, nkv, hd)
    data, scale = kv.data.cpu(), kv.scale.cpu()
    assert (data[0, 0, 0, 0] == 128).all() and scale[0, 0, 0, 0] == 0
    one = torch.full((hd,), 128, dtype=torch.uint8)
    one[5] = 255
    assert torch.equal(data[0, 1, 0, 1], one) and abs(float(scale[0, 1, 0, 1]) * 127 / 65504 - 1) < 2.0 ** -22
    assert data[0, 1, 0, 2, 7] == 1 and abs(float(scale[0, 1, 0, 2]) * 127 / 65504 - 1) < 2.0 ** -22
    assert scale[0, 1, 0, 3].isnan() and not scale[0, 1, 1].isnan().any() and not scale[0, 0].isnan().any()


# ---- read back --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("nkv,bs", [(1, 16), (2, 48), (8, 32)])
@pytest.mark.parametrize("lens", [[1], [0, 16, 17, 0, 31, 500], [3] * 40, [2049]])
def test_read(ops, hd, nkv, bs, lens):
    g = gen(hd + nkv + len(lens))
    need = [-(-n // bs) for n in lens]
    blocks = sum(need) + 3
    data, scale = make_cache(g, blocks, nkv, bs, hd, DEV)
    kv = QuantKV(data, scale)
    holes = [(s, j) for s, n in enumerate(need) for j in range(1, n - 1, 3)]
    tables = make_tables(g, lens, bs, blocks, DEV, width=max(need) + 2, holes=holes)
    for s, n in enumerate(lens):                                           # what lies behind a sequence is anything
        if n % bs and tables[s, need[s] - 1] >= 0:
            scale[tables[s, need[s] - 1].long(), :, :, n % bs:] = float("nan")
    cu = [1]                                                               # a page that no sequence has, before and behind
    for n in need:
        cu.append(cu[-1] + n)
    out = torch.full((cu[-1] + 1, 2, nkv, bs, hd), 9.0, dtype=torch.float16, device=DEV)
    places = torch.full((len(lens) + 1, max(need) + 3), 55, dtype=torch.int32, device=DEV)
    ops.kv_read_q8(kv, tables, ints(lens), ints(cu), len(lens), out, places)
    torch.cuda.synchronize()
    ops.check()
    want = torch.full(out.shape, 9.0, dtype=torch.float64, device=DEV)
    want_places = torch.full(places.shape, -1, dtype=torch.int32, device=DEV)
    want_places[len(lens)] = 55
    for s, n in enumerate(lens):
        for j in range(need[s]):
            b = int(tables[s, j])
            if b < 0:
                continue
            want_places[s, j] = cu[s] + j
            y = (data[b].double() - 128) * scale[b].double()[..., None]
            y[:, :, max(0, n - j * bs):] = 0
            want[cu[s] + j] = y
    assert torch.equal(places, want_places)
    # one product in fp32, one rounding to fp16
    assert ((out.double() - want).abs() <= want.abs() * 2.0 ** -11 * 1.001 + 2.0 ** -25).all()


# ---- attention --------------------------------------------------------------------------------------------------------------
def attend(ops, lens, nh, nkv, hd, bs=16, window=0, holes=(), rows=None, splits=0, seed=0, cache=None, width=None, wide=16):
    """Runs the operator over sequences of ``lens`` tokens (``rows``: new rows of each) and compares with 64 bits."""
    g = gen(seed + hd + 7 * nkv + len(lens))
    blocks = sum(-(-n // bs) for n in lens) + 2
    data, scale = cache(g, blocks) if cache else make_cache(g, blocks, nkv, bs, hd, DEV)
    tables = make_tables(g, lens, bs, blocks, DEV, width=width, holes=holes)
    for s, n in enumerate(lens):
        if n % bs and tables[s, n // bs] >= 0:
            scale[tables[s, n // bs].long(), :, :, n % bs:] = float("nan")
    seen = [(s, n) for s, n in enumerate(lens)] if rows is None else [(s, n - r + 1 + i) for s, (n, r) in enumerate(zip(lens, rows))
                                                                   for i in range(r)]
    R = len(seen)
    q = (torch.randn(max(R, 1), nh * hd + wide, generator=g) * 2).half().to(DEV)
    out = torch.full((R + 2, nh * hd + wide), 3.0, dtype=torch.float16, device=DEV)
    kw = {}
    if rows is not None:
        cu = [0]
        for r in rows:
            cu.append(cu[-1] + r)
        kw = dict(cu_q=ints(cu), q_pos0=ints([n - r for n, r in zip(lens, rows)]), max_q=max(rows + [1]))
        seen = [(s, n - r + i + 1) for s, (n, r) in enumerate(zip(lens, rows)) for i in range(r)]
    call = lambda: ops.attn_decode_q8(q, QuantKV(data, scale), tables, ints(lens) if rows is None else None, out, len(lens), nh,
                                      nkv, hd, scale_of(hd), num_splits=splits, window=window, **kw)
    call()
    torch.cuda.synchronize()
    ops.check()
    want, tol = attention(q, data, scale, tables, seen, nh, scale_of(hd), window)
    got = out[:R, : nh * hd].double()
    assert (out[R:] == 3).all() and (out[:, nh * hd:] == 3).all()
    assert not got.isnan().any()
    bad = (got - want).abs() - tol
    assert (bad <= 0).all(), f"{float(bad.max())} over {float(tol.max())} at {tuple(int(i) for i in torch.nonzero(bad == bad.max())[0])}"
    first = out.clone()
    call()
    assert torch.equal(first, out)                                         # the same call gives the same bits
    return out


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("nh,nkv", [(1, 1), (8, 8), (7, 1), (40, 8), (16, 1), (24, 2)])
@pytest.mark.parametrize("lens", [[1], [0, 1, 15, 16, 17, 33, 0, 300], [2100]])
def test_attention_shapes(ops, hd, nh, nkv, lens):
    attend(ops, lens, nh, nkv, hd)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("bs", [16, 32, 48, 64])
@pytest.mark.parametrize("window", [0, 1, 17, 100])
def test_windows_and_holes(ops, hd, bs, window):
    lens = [1, 18, 130, 400, 0, 77]
    holes = [(s, j) for s, n in enumerate(lens) for j in range(0, -(-n // bs), 3)]        # the first block, and the only one
    attend(ops, lens, 8, 2, hd, bs=bs, window=window, holes=holes, width=40)


@pytest.mark.parametrize("splits", [0, 1, 2, 3, 5, 8, 16, 17, 40, 64])
@pytest.mark.parametrize("lens", [[5], [0], [700, 0, 31, 2000, 1], [0, 0, 16, 16, 900, 0]])
def test_pieces(ops, splits, lens):
    attend(ops, lens, 14, 2, 128, splits=splits)
    attend(ops, lens, 4, 4, 64, splits=splits, window=333)
    attend(ops, lens, 10, 2, 96, splits=splits, rows=[min(n, 1 + 2 * i) for i, n in enumerate(lens)], holes=[(len(lens) - 2, 1)] if len(lens) > 1 else ())


@pytest.mark.parametrize("splits", [0, 2, 32])
@pytest.mark.parametrize("hd,nh,nkv", [(64, 32, 8), (96, 4, 4), (128, 16, 1), (256, 16, 8)])
def test_mixed_lengths(ops, splits, hd, nh, nkv):
    lens = [(97 * i * i) % 400 for i in range(70)]
    attend(ops, lens, nh, nkv, hd, splits=splits)
    attend(ops, lens, nh, nkv, hd, splits=splits, rows=[min(n, 1 + i % 5) for i, n in enumerate(lens)], window=90)


@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 16), (96, 48), (128, 128), (256, 256), (128, 0)])
@pytest.mark.parametrize("M", [888, 1801, 7777])
def test_write_of_many_rows(ops, hd, rot, M):
    nh, nkv, bs = 6, 2, 16
    g = gen(hd + M)
    pos, slots = torch.arange(M, dtype=torch.int32, device=DEV) * 3, torch.randperm(M + 7, generator=g)[:M].to(DEV)
    slots[M // 3] = -1
    kv = QuantKV.zeros(((M + 7) // bs + 1, 2, nkv, bs, hd), DEV)
    qkv = torch.randn(M, (nh + 2 * nkv) * hd, generator=g).half().to(DEV)
    x, q = qkv.double(), torch.zeros(M, nh * hd, dtype=torch.float16, device=DEV)
    ops.rope_kv_write_q8(qkv, kv, pos, slots, freqs_of(rot), M, nh, nkv, hd, q_out=q)
    k = slots >= 0
    blk, off = slots[k] // bs, slots[k] % bs
    check_write(x[k], pos[k], freqs_of(rot), nh, nkv, hd, q[k], kv.data[blk, :, :, off], kv.scale[blk, :, :, off])
    assert int((kv.data != 0).any(-1).sum()) == 2 * nkv * (M - 1)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("nh,nkv", [(8, 8), (7, 1), (40, 8), (16, 1)])
@pytest.mark.parametrize("rows", [[5, 1, 3, 5], [2, 2, 2, 2], [1, 17, 4, 9]])
@pytest.mark.parametrize("window", [0, 50])
def test_rows_of_a_draft(ops, hd, nh, nkv, rows, window):
    attend(ops, [400, 1, 77, 18], nh, nkv, hd, rows=[min(r, n) for r, n in zip(rows, [400, 1, 77, 18])], window=window,
           holes=[(0, 3), (2, 0)])


def test_many_sequences(ops):
    attend(ops, [(37 * i) % 200 for i in range(300)], 8, 2, 64)
    attend(ops, [1 + (53 * i) % 90 for i in range(130)], 8, 8, 128, rows=[1 + i % 2 if (53 * i) % 90 else 1 for i in range(130)])


@pytest.mark.parametrize("nh,nkv,rows", [(16, 16, 1), (64, 16, 1), (40, 8, 5), (32, 16, 3)])
def test_more_pieces_than_fit_at_a_time(ops, nh, nkv, rows):
    """Up to 64 sequences are then taken the longest first: alike ones, empty ones, ones that windows make alike."""
    lens = [300, 0, 17, 300, 2, 64, 64, 1] * 8
    draft = None if rows == 1 else [min(n, 1 + i % rows) for i, n in enumerate(lens)]
    for S in (64, 63, 33):
        for window in (0, 40):
            attend(ops, lens[:S], nh, nkv, 64, rows=draft and draft[:S], window=window, splits=4)
    attend(ops, list(range(1, 64)), nh, nkv, 128, rows=draft and [min(n, 2) for n in range(1, 64)], splits=8)


def test_tables_inside_wider_ones(ops):
    g = gen(21)
    nh, nkv, hd, bs, lens = 8, 2, 64, 16, [40, 100, 5]
    data, scale = make_cache(g, 12, nkv, bs, hd, DEV)
    wide = torch.full((3, 20), 10 ** 6, dtype=torch.int32, device=DEV)           # what stands beside is no block
    wide[:, 3:10] = make_tables(g, lens, bs, 12, DEV, width=7)
    tables = wide[:, 3:10]
    q = torch.randn(3, nh * hd, generator=g).half().to(DEV)
    out = torch.zeros(3, nh * hd, dtype=torch.float16, device=DEV)
    ops.attn_decode_q8(q, QuantKV(data, scale), tables, ints(lens), out, 3, nh, nkv, hd, scale_of(hd))
    want, tol = attention(q, data, scale, tables, list(enumerate(lens)), nh, scale_of(hd))
    assert ((out.double() - want).abs() <= tol).all()
    pages, places = torch.zeros(11, 2, nkv, bs, hd, dtype=torch.float16, device=DEV), torch.full((3, 30), 5, dtype=torch.int32, device=DEV)
    ops.kv_read_q8(QuantKV(data, scale), tables, ints(lens), ints([0, 3, 10, 11]), 3, pages, places[:, 4:12])
    assert places[:, 4:12].tolist() == [[0, 1, 2] + [-1] * 5, [3, 4, 5, 6, 7, 8, 9, -1], [10] + [-1] * 7]
    assert (places[:, :4] == 5).all() and (places[:, 12:] == 5).all()
    torch.cuda.synchronize()
    ops.check()


def test_calls_of_nothing(ops):
    nh, nkv, hd = 4, 2, 64
    kv = QuantKV(*make_cache(gen(1), 2, nkv, 16, hd, DEV))
    before = kv.data.clone(), kv.scale.clone()
    e16, e32, e64 = (torch.zeros(0, 8 * hd, dtype=torch.float16, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV),
                     torch.zeros(0, dtype=torch.int64, device=DEV))
    ops.rope_kv_write_q8(e16, kv, e32, e64, freqs_of(hd), 0, nh, nkv, hd)
    ops.attn_decode_q8(e16, kv, torch.zeros(0, 1, dtype=torch.int32, device=DEV), e32, e16, 0, nh, nkv, hd, scale_of(hd))
    places = torch.zeros(0, 1, dtype=torch.int32, device=DEV)
    ops.kv_read_q8(kv, places, e32, ints([0]), 0, torch.zeros(1, 2, nkv, 16, hd, dtype=torch.float16, device=DEV), places)
    out = torch.full((2, nh * hd), 7.0, dtype=torch.float16, device=DEV)                     # tables without columns: nothing is seen
    ops.attn_decode_q8(out.clone(), kv, torch.zeros(2, 0, dtype=torch.int32, device=DEV), ints([0, 0]), out, 2, nh, nkv, hd, scale_of(hd))
    torch.cuda.synchronize()
    ops.check()
    assert (out == 0).all() and torch.equal(before[0], kv.data) and torch.equal(before[1], kv.scale)


def test_results_over_the_queries(ops):
    """The result may go where the queries were."""
    nh, nkv, hd, lens = 14, 2, 128, [700, 31, 2000]
    g = gen(8)
    data, scale = make_cache(g, 180, nkv, 16, hd, DEV)
    tables = make_tables(g, lens, 16, 180, DEV)
    q = torch.randn(3, nh * hd, generator=g).half().to(DEV)
    for splits in (0, 1, 8, 64):
        out, inplace = torch.zeros_like(q), q.clone()
        for to, src in ((out, q), (inplace, inplace)):
            ops.attn_decode_q8(src, QuantKV(data, scale), tables, ints(lens), to, 3, nh, nkv, hd, scale_of(hd), num_splits=splits)
        assert torch.equal(out, inplace)


def test_long_sequence(ops):
    attend(ops, [40001], 7, 1, 128)
    attend(ops, [20011, 3], 8, 1, 128, rows=[4, 1])


def test_scales_of_every_size(ops):
    """Values of one token a thousand times those of the next, and values of 1e-6."""
    def cache(g, blocks):
        data, scale = make_cache(g, blocks, 2, 16, 128, DEV)
        factor = torch.exp(torch.randn(blocks, 2, 16, generator=g) * 3.5).to(DEV)
        scale[:, 1] *= factor
        return data, scale

    def small(g, blocks):
        data, scale = make_cache(g, blocks, 2, 16, 128, DEV)
        scale[:, 1] *= 1e-6
        scale[:, 0] *= 3.0
        return data, scale
    attend(ops, [1000, 20], 8, 2, 128, cache=cache)
    out = attend(ops, [600, 3], 8, 2, 128, cache=small)
    assert out[:2, : 8 * 128].float().abs().max() > 0


@pytest.mark.parametrize("nh,nkv,rows", [(2, 2, None), (14, 2, None), (32, 2, None), (8, 2, [5, 1, 2])])
@pytest.mark.parametrize("behind,factor", [(2200.0, 1e6), (16.0, 1e6), (-8.0, 1e-6), (-8.0, 0.0), (-40.0, 1e-6)])
@pytest.mark.parametrize("window", [0, 250])
def test_tokens_of_another_size(ops, nh, nkv, rows, behind, factor, window):
    """A few tokens' values are a million times the others' and their weight zero or about a millionth of theirs, or the other way
    round; some of them lie before the window."""
    bs, hd, lens, g = 16, 128, [300, 17, 700], gen(nh + abs(int(behind)))
    data, scale = make_cache(g, 70, nkv, bs, hd, DEV)
    tables = make_tables(g, lens, bs, 70, DEV)
    for s, n in enumerate(lens):
        for t in {0, n // 2, n - 3, max(0, n - 252)}:
            b = tables[s, t // bs].long()
            scale[b, 1, :, t % bs] *= factor                               # its values
            data[b, 0, :, t % bs] = 1 if behind > 0 else 255               # its key: +-127 times the scale, against q of about 1.5
            scale[b, 0, :, t % bs] = abs(behind) / (127 * 1.5 * hd * scale_of(hd))
    seen = [(s, n) for s, n in enumerate(lens)] if rows is None else [(s, n - r + i + 1) for s, (n, r) in enumerate(zip(lens, rows))
                                                                   for i in range(r)]
    q = (torch.rand(len(seen), nh * hd, generator=g) + 1).half().to(DEV)
    out = torch.zeros_like(q)
    kw = {}
    if rows is not None:
        kw = dict(cu_q=ints([0, 5, 6, 8]), q_pos0=ints([n - r for n, r in zip(lens, rows)]), max_q=5)
    want, tol = attention(q, data, scale, tables, seen, nh, scale_of(hd), window)
    for splits in (0, 1, 4, 32):
        ops.attn_decode_q8(q, QuantKV(data, scale), tables, None if rows else ints(lens), out, 3, nh, nkv, hd, scale_of(hd),
                           num_splits=splits, window=window, **kw)
        bad = (out.double() - want).abs() - tol
        assert (bad <= 0).all(), f"{splits} pieces: {float(bad.max())} over {float(tol.max())}, results up to {float(want.abs().max())}"


def test_nan_is_seen_and_not_hidden(ops):
    nh, nkv, hd, bs = 4, 2, 64, 16
    g = gen(11)
    data, scale = make_cache(g, 4, nkv, bs, hd, DEV)
    tables = ints([[0, 1], [2, 3]])
    q = torch.randn(2, nh * hd, generator=g).half().to(DEV)
    scale[0, 1, 0, 3] = float("nan")                                       # sequence 0, value of token 3, kv head 0
    out = torch.zeros(2, nh * hd, dtype=torch.float16, device=DEV)
    ops.attn_decode_q8(q, QuantKV(data, scale), tables, ints([20, 20]), out, 2, nh, nkv, hd, scale_of(hd))
    nan = out.isnan().view(2, nkv, -1).all(-1).tolist()
    assert nan == [[True, False], [False, False]] and not out[1].isnan().any() and not out[0, nh * hd // 2:].isnan().any()
    scale[0, 1, 0, 3] = 0.01
    scale[2, 0, 1, 19 % bs] = float("nan")                                 # a key
    ops.attn_decode_q8(q, QuantKV(data, scale), tables, ints([20, 20]), out, 2, nh, nkv, hd, scale_of(hd))
    assert out.isnan().view(2, nkv, -1).all(-1).tolist() == [[False, False], [False, True]]


def test_cache_of_more_than_four_gigabytes(ops):
    nkv, bs, hd = 8, 64, 128
    blocks = 5 * 2 ** 30 // (2 * nkv * bs * hd)
    data = torch.empty(blocks, 2, nkv, bs, hd, dtype=torch.uint8, device=DEV)
    scale = torch.empty(blocks, 2, nkv, bs, device=DEV)
    g = gen(2)
    ids = [blocks - 1, 0, blocks - 2, blocks // 2]
    small, small_scale = make_cache(g, 4, nkv, bs, hd, DEV)
    data[ids], scale[ids] = small, small_scale
    q = torch.randn(1, 8 * hd, generator=g).half().to(DEV)
    out = torch.zeros(1, 8 * hd, dtype=torch.float16, device=DEV)
    tables = ints([ids])
    ops.attn_decode_q8(q, QuantKV(data, scale), tables, ints([4 * bs - 3]), out, 1, 8, nkv, hd, scale_of(hd))
    want, tol = attention(q, data, scale, tables, [(0, 4 * bs - 3)], 8, scale_of(hd))
    assert ((out.double() - want).abs() <= tol).all()
    qkv = torch.randn(1, (8 + 2 * nkv) * hd, generator=g).half().to(DEV)
    slot = blocks * bs - 2
    ops.rope_kv_write_q8(qkv, QuantKV(data, scale), ints([4]), ints([slot], torch.int64), freqs_of(hd), 1, 8, nkv, hd)
    pages, places = torch.zeros(4, 2, nkv, bs, hd, dtype=torch.float16, device=DEV), torch.zeros(1, 4, dtype=torch.int32, device=DEV)
    ops.kv_read_q8(QuantKV(data, scale), tables, ints([4 * bs]), ints([0, 4]), 1, pages, places)
    v = qkv[0, 16 * hd:].view(nkv, hd).double()
    step = v.abs().amax(-1, keepdim=True) / 127
    # half a step of the bytes, the fp16 of the page and 1e-3 of a step for fp32
    assert ((pages[0, 1, :, bs - 2].double() - v).abs() <= step * 0.501 + v.abs() * 2.0 ** -10).all()


# ---- what is reported -------------------------------------------------------------------------------------------------------
def test_ids_outside_the_cache_are_reported_and_not_followed(ops):
    from zse_b200.ops.native import DeviceStatusError
    nh, nkv, hd, bs = 4, 2, 64, 16
    data, scale = make_cache(gen(1), 3, nkv, bs, hd, DEV)
    kv = QuantKV(data, scale)
    q = torch.randn(1, nh * hd, generator=gen(2)).half().to(DEV)
    out = torch.zeros(1, nh * hd, dtype=torch.float16, device=DEV)
    ops.attn_decode_q8(q, kv, ints([[1, 3]]), ints([20]), out, 1, nh, nkv, hd, scale_of(hd))
    with pytest.raises(DeviceStatusError):
        ops.check()
    want, tol = attention(q, data, scale, ints([[1, -1]]), [(0, 20)], nh, scale_of(hd))
    assert ((out.double() - want).abs() <= tol).all()
    ops.attn_decode_q8(q, kv, ints([[1, 2]]), ints([33]), out, 1, nh, nkv, hd, scale_of(hd))     # more tokens than the table holds
    with pytest.raises(DeviceStatusError):
        ops.check()
    pages, places = torch.zeros(2, 2, nkv, bs, hd, dtype=torch.float16, device=DEV), torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    ops.kv_read_q8(kv, ints([[1, 7]]), ints([20]), ints([0, 2]), 1, pages, places)
    with pytest.raises(DeviceStatusError):
        ops.check()
    assert places.tolist() == [[0, -1]] and (pages[1] == 0).all() and (pages[0] != 0).any()
    ops.kv_read_q8(kv, ints([[1, 2]]), ints([20]), ints([0, 1]), 1, pages.zero_(), places)          # one page for two blocks
    with pytest.raises(DeviceStatusError):
        ops.check()
    assert (pages == 0).all() and places.tolist() == [[-1, -1]]
    x = torch.randn(2, (nh + 2 * nkv) * hd, generator=gen(4)).half().to(DEV)
    before = data.clone()
    ops.rope_kv_write_q8(x, kv, ints([0, 1]), ints([3 * bs, -5], torch.int64), freqs_of(hd), 2, nh, nkv, hd)
    with pytest.raises(DeviceStatusError):
        ops.check()
    assert torch.equal(before, data)
    ops.check()


@pytest.mark.parametrize("splits", [0, 8, 32])
def test_two_streams_and_two_graphs(ops, splits):
    """Calls that run at once share nothing; graphs of them keep their own scratch, whatever runs between their replays."""
    nh, nkv, hd, lens, g = 14, 2, 128, [[3000, 17], [900, 2222]], gen(31)
    data, scale = make_cache(g, 420, nkv, 16, hd, DEV)
    kv, qs, outs, args = QuantKV(data, scale), [], [], []
    for n in lens:
        qs.append(torch.randn(2, nh * hd, generator=g).half().to(DEV))
        outs.append(torch.zeros_like(qs[-1]))
        args.append((make_tables(g, n, 16, 420, DEV), ints(n)))
    call = lambda i: ops.attn_decode_q8(qs[i], kv, *args[i], outs[i], 2, nh, nkv, hd, scale_of(hd), num_splits=splits)
    want = []
    for i in range(2):
        call(i)
        want.append(outs[i].clone())
    streams, graphs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].zero_()
                call(i)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            call(i)
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].zero_()
                graphs[i].replay()
    call(0)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    ops.check()


def test_scratch_of_another_kind_and_another_device_are_refused(ops, monkeypatch):
    from zse_b200.ops.native import NativeError, attn_decode_q8_plan
    q = torch.zeros(1, 4 * 64, dtype=torch.float16, device=DEV)
    kv = QuantKV.zeros((64, 2, 2, 16, 64), DEV)
    tables, need = ints([list(range(64))]), attn_decode_q8_plan(1, 1, 4, 2, 64, 16, 64, num_splits=16)[1]
    call = lambda scratch: ops.attn_decode_q8(q, kv, tables, ints([1000]), q.clone(), 1, 4, 2, 64, 0.125, scratch, num_splits=16)
    assert need > 0
    call(torch.zeros(need, device=DEV))
    for scratch in (torch.zeros(need, device=DEV, dtype=torch.float16), torch.zeros(need), torch.zeros(2 * need, device=DEV)[::2],
                    torch.zeros(1, need, device=DEV)):
        with pytest.raises(ValueError, match="scratch"):
            call(scratch)
    with pytest.raises(NativeError, match="scratch"):
        call(torch.zeros(need - 1, device=DEV))
    monkeypatch.setattr(ops, "home", 1)
    with pytest.raises(NativeError, match="device"):
        call(None)


def test_refusals_of_the_library(ops):
    from zse_b200.ops.native import NativeError
    kv = QuantKV.zeros((2, 2, 2, 16, 80), DEV)                              # a head dimension without kernels
    q = torch.zeros(1, 4 * 80, dtype=torch.float16, device=DEV)
    with pytest.raises(NativeError, match="shape"):
        ops.attn_decode_q8(q, kv, ints([[0]]), ints([1]), q.clone(), 1, 4, 2, 80, 0.1)
    kv = QuantKV.zeros((2, 2, 2, 8, 64), DEV)                               # blocks of 8
    q = torch.zeros(1, 4 * 64, dtype=torch.float16, device=DEV)
    with pytest.raises(NativeError, match="shape"):
        ops.attn_decode_q8(q, kv, ints([[0]]), ints([1]), q.clone(), 1, 4, 2, 64, 0.1)
    kv = QuantKV.zeros((2, 2, 2, 16, 64), DEV)
    x = torch.zeros(1, 8 * 64 + 1, dtype=torch.float16, device=DEV)
    with pytest.raises(NativeError, match="aligned|stride"):
        ops.rope_kv_write_q8(x[:, 1:], kv, ints([0]), ints([0], torch.int64), freqs_of(64), 1, 4, 2, 64)
    with pytest.raises(NativeError, match="contiguous"):
        ops.attn_decode_q8(q, QuantKV(torch.zeros(4, 2, 2, 16, 64, dtype=torch.uint8, device=DEV)[::2],
                                      torch.zeros(4, 2, 2, 16, device=DEV)[::2]), ints([[0]]), ints([1]), q.clone(), 1, 4, 2, 64, 0.1)


# ---- together ---------------------------------------------------------------------------------------------------------------
def _step_inputs(g, lens, nh, nkv, hd, bs):
    blocks = sum(n // bs + 1 for n in lens) + 1
    data, scale = make_cache(g, blocks, nkv, bs, hd, DEV)
    tables = make_tables(g, [n + 1 for n in lens], bs, blocks, DEV)
    slots = ints([int(tables[s, n // bs]) * bs + n % bs for s, n in enumerate(lens)], torch.int64)
    qkv = torch.randn(len(lens), (nh + 2 * nkv) * hd, generator=g).half().to(DEV)
    return QuantKV(data, scale), tables, slots, qkv, ints(lens), ints([n + 1 for n in lens])


def _step(ops, kv, tables, slots, qkv, pos, lens, nh, nkv, hd, q, out):
    S = qkv.shape[0]
    ops.rope_kv_write_q8(qkv, kv, pos, slots, freqs_of_cached(hd), S, nh, nkv, hd, q_out=q)
    ops.attn_decode_q8(q, kv, tables, lens, out, S, nh, nkv, hd, scale_of(hd))


_FREQS = {}


def freqs_of_cached(hd):
    if hd not in _FREQS:
        _FREQS[hd] = freqs_of(hd)
    return _FREQS[hd]


@pytest.mark.parametrize("hd,nh,nkv", [(64, 8, 2), (128, 14, 2)])
def test_decode_step_then_prefill_read(ops, hd, nh, nkv):
    """A step writes and attends; then the same cache, read back, goes through the framework's prefill attention."""
    lens, bs, S = [31, 0, 200, 16], 16, 4
    kv, tables, slots, qkv, pos, now = _step_inputs(gen(hd), lens, nh, nkv, hd, bs)
    q = torch.zeros(S, nh * hd, dtype=torch.float16, device=DEV)
    out = torch.zeros(S, nh * hd, dtype=torch.float16, device=DEV)
    _step(ops, kv, tables, slots, qkv, pos, now, nh, nkv, hd, q, out)
    want, tol = attention(q, kv.data, kv.scale, tables, [(s, n + 1) for s, n in enumerate(lens)], nh, scale_of(hd))
    assert ((out.double() - want).abs() <= tol).all()
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n // bs + 1)
    pages = torch.zeros(cu[-1], 2, nkv, bs, hd, dtype=torch.float16, device=DEV)
    places = torch.zeros(S, tables.shape[1], dtype=torch.int32, device=DEV)
    ops.kv_read_q8(kv, tables, now, ints(cu), S, pages, places)
    again = torch.zeros(S, nh * hd, dtype=torch.float16, device=DEV)
    ops.attn_prefill(q, pages, places, ints(list(range(S + 1))), pos, again, S, S, 1, nh, nkv, hd, bs, scale_of(hd))
    torch.cuda.synchronize()
    ops.check()
    # the pages are rounded to fp16 once more: 2^-11 of every key and value; a key's share in the exponent is |q.k| * scale * 2^-11
    most = (q.double().view(S, nkv, nh // nkv, hd).abs().sum(-1).amax((1, 2))[:, None]
            * (kv.scale[:, 0].nan_to_num(0).double().max() * 127) * scale_of(hd) * 2.0 ** -11)
    size = (kv.scale[:, 1].double().max() * 127)
    assert ((again.double() - want).abs() <= 2 * tol + (2 * most + 2.0 ** -10) * size).all()


def test_graph_of_a_step(ops):
    """Captured, replayed with other lengths and tables in place, and beside a second graph on another stream."""
    nh, nkv, hd, bs = 14, 2, 128, 16
    made = []
    for seed, lens in ((1, [40, 300, 7]), (2, [900, 1, 64])):
        kv, tables, slots, qkv, pos, now = _step_inputs(gen(seed), lens, nh, nkv, hd, bs)
        wide = torch.full((3, 70), -1, dtype=torch.int32, device=DEV)
        wide[:, : tables.shape[1]] = tables
        q, out = (torch.zeros(3, nh * hd, dtype=torch.float16, device=DEV) for _ in range(2))
        args = (ops, kv, wide, slots, qkv, pos, now, nh, nkv, hd, q, out)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            _step(*args)
        made.append((graph, side, kv, wide, now, q, out, args))      # a graph's tensors live as long as it does
    for _ in range(3):
        for m in made:
            m[6].zero_()
        torch.cuda.synchronize()
        for graph, side, *_ in made:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, kv, wide, now, q, out, _ in made:
            want, tol = attention(q, kv.data, kv.scale, wide, [(s, int(n)) for s, n in enumerate(now)], nh, scale_of(hd))
            assert ((out.double() - want).abs() <= tol).all()
            now.sub_(1)                                                    # shorter sequences for the next replay
            now.clamp_(min=0)
    ops.check()


@pytest.mark.parametrize("stale", [-1, 0])
@pytest.mark.parametrize("groups", [
    # sequences' tokens in all, new rows of each, dropped blocks; a pass over more context than the pages hold is several groups
    [([300, 40, 129], [33, 40, 9], [(0, 2), (2, 0)])],
    [([130, 33], [130, 12], [(0, 0)]), ([50], [50], []), ([400, 16], [200, 16], [(0, 3), (0, 7)])],
])
def test_prefill_right_behind_the_read_back(ops, stale, groups):
    """Everything queued behind a long product, so that each kernel's CTAs are there before the one in front of it has written: the
    pages and tables of the read-back, not what stood there, are what attention sees.  ``stale``: the tables' contents before (dropped
    blocks everywhere; page 0 everywhere, over the dropped ones too); later groups find those of the groups before."""
    nh, nkv, hd, bs, g = 8, 2, 128, 16, gen(len(groups))
    most = max(sum(-(-n // bs) for n in lens) for lens, _, _ in groups)
    pages = torch.zeros(most, 2, nkv, bs, hd, dtype=torch.float16, device=DEV)
    places = torch.zeros(3, 26, dtype=torch.int32, device=DEV)
    made = []
    for lens, new, holes in groups:
        blocks = sum(-(-n // bs) for n in lens) + 1
        kv = QuantKV(*make_cache(g, blocks, nkv, bs, hd, DEV))
        full = make_tables(g, lens, bs, blocks, "cpu")
        pos = [p for n, r in zip(lens, new) for p in range(n - r, n)]
        slots = [int(full[s, p // bs]) * bs + p % bs for s, (n, r) in enumerate(zip(lens, new)) for p in range(n - r, n)]
        for s, b in holes:
            full[s, b] = -1
        cu, first = [0], [0]
        for n, r in zip(lens, new):
            cu.append(cu[-1] + -(-n // bs))
            first.append(first[-1] + r)
        x = torch.randn(first[-1], (nh + 2 * nkv) * hd, generator=g).half().to(DEV)
        made.append((kv, full.to(DEV), ints(lens), ints(cu), ints(first), ints([n - r for n, r in zip(lens, new)]), ints(pos),
                     ints(slots, torch.int64), x, x.clone(), torch.zeros(first[-1], nh * hd, dtype=torch.float16, device=DEV), max(new)))
    freqs, filler = freqs_of(hd), torch.randn(8192, 8192, device=DEV).half()

    def run(wait):
        places.fill_(stale)
        for m in made:
            m[9].copy_(m[8])
            m[10].zero_()
        if not wait:
            for _ in range(3):
                torch.mm(filler, filler)
        for kv, tables, lens, cu, first, pos0, pos, slots, _, q, out, max_q in made:
            S, M = lens.shape[0], pos.shape[0]
            ops.rope_kv_write_q8(q, kv, pos, slots, freqs, M, nh, nkv, hd)
            wait and torch.cuda.synchronize()
            ops.kv_read_q8(kv, tables, lens, cu, S, pages, places[:S])
            wait and torch.cuda.synchronize()
            ops.attn_prefill(q, pages, places[:S], first, pos0, out, S, M, max_q, nh, nkv, hd, bs, scale_of(hd))
            wait and torch.cuda.synchronize()
        return [m[10].clone() for m in made]

    want = run(True)
    for (lens, new, _), m, got in zip(groups, made, want):
        seen = [(s, n - r + 1 + i) for s, (n, r) in enumerate(zip(lens, new)) for i in range(r)]
        exact, tol = attention(m[9], m[0].data, m[0].scale, m[1], seen, nh, scale_of(hd))
        # keys and values rounded to fp16 once more, 2^-11 of each (of a key in the exponent), and weights that are fp16 numbers
        off = (m[9][:, : nh * hd].double().abs().view(-1, nh, hd).sum(-1).amax(1)[:, None] * m[0].scale[:, 0].double().max() * 127
               * scale_of(hd) * 2 + 2) * 2.0 ** -11 * m[0].scale[:, 1].double().max() * 127
        assert ((got.double() - exact).abs() <= 2 * tol + off).all()
    for _ in range(20):
        for got, right in zip(run(False), want):
            assert torch.equal(got, right)
    torch.cuda.synchronize()
    ops.check()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("group,draft", [(3, False), (5, False), (7, False), (11, False), (5, True), (1, True), (2, True)])
@pytest.mark.parametrize("window", [0, 90])
def test_what_lies_behind_a_sequence_changes_no_bit(ops, hd, group, draft, window):
    """Columns of the products that stand for no head or no row (groups of 5 or 7, drafts of fewer rows than the longest) see nothing
    either: scales left behind the last token, however large, move no reference of the columns beside them."""
    nkv, bs, lens, g = 2, 16, [2 + (29 * i) % 330 for i in range(24)], gen(hd + group)
    nh, blocks = group * nkv, sum(-(-n // bs) for n in lens)
    data, scale = make_cache(g, blocks, nkv, bs, hd, DEV)
    tables = make_tables(g, lens, bs, blocks, DEV)
    rows = [min(n, 1 + i % 5) for i, n in enumerate(lens)] if draft else [1] * len(lens)
    seen = [(s, n - r + 1 + i) for s, (n, r) in enumerate(zip(lens, rows)) for i in range(r)]
    q = (torch.randn(len(seen), nh * hd, generator=g) * 2).half().to(DEV)
    kw = {}
    if draft:
        cu = [0]
        for r in rows:
            cu.append(cu[-1] + r)
        kw = dict(cu_q=ints(cu), q_pos0=ints([n - r for n, r in zip(lens, rows)]), max_q=5)
    out = torch.zeros_like(q)
    for splits in (0, 1):
        first = None
        for keys, values in ((0.0, 0.0), (0.0, 1e30), (0.01, float("inf")), (1e30, 1e30), (float("inf"), 1e20), (float("nan"), 1e30), (0.0, -1e30)):
            for s, n in enumerate(lens):
                if n % bs:
                    scale[tables[s, n // bs].long(), 0, :, n % bs:] = keys
                    scale[tables[s, n // bs].long(), 1, :, n % bs:] = values
            ops.attn_decode_q8(q, QuantKV(data, scale), tables, None if draft else ints(lens), out, len(lens), nh, nkv, hd, scale_of(hd),
                               num_splits=splits, window=window, **kw)
            if first is None:
                first = out.clone()
                want, tol = attention(q, data, scale, tables, seen, nh, scale_of(hd), window)
                assert ((out.double() - want).abs() <= tol).all()
            assert torch.equal(out, first), (splits, keys, values)
    ops.check()


@pytest.mark.parametrize("pos", [2 ** 31 - 1, 2 ** 31 - 4, 2 ** 31 - 200, 33, 28, -1, -2 ** 31])
@pytest.mark.parametrize("nh,window", [(4, 0), (32, 0), (4, 9)])
def test_positions_outside_the_table_are_reported(ops, pos, nh, window):
    """The last of five rows is behind a table of 32 tokens, or the first before it; the sequence beside it gets its result."""
    from zse_b200.ops.native import DeviceStatusError
    nkv, hd, bs = 2, 64, 16
    data, scale = make_cache(gen(3), 4, nkv, bs, hd, DEV)
    tables = ints([[0, 1], [2, 3]])
    q = torch.randn(10, nh * hd, generator=gen(4)).half().to(DEV)
    out = torch.zeros_like(q)
    for p in (27, pos):
        ops.attn_decode_q8(q, QuantKV(data, scale), tables, None, out, 2, nh, nkv, hd, scale_of(hd), window=window, cu_q=ints([0, 5, 10]),
                           q_pos0=ints([p, 20]), max_q=5)
        want, tol = attention(q, data, scale, tables, [(s, n + i) for s, n in ((0, 28), (1, 21)) for i in range(5)], nh, scale_of(hd), window)
        assert ((out.double() - want).abs() <= tol)[0 if p == 27 else 5:].all()
        if p == 27:
            ops.check()
    with pytest.raises(DeviceStatusError):
        ops.check()
    ops.check()
