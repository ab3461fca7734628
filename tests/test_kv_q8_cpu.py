"""The 8-bit KV cache without a GPU: the torch forms of its operators against 64 bits, what they refuse, and the cache object."""
import pytest
import torch

from tests.helpers.kv_q8_oracle import attention, check_write, make_cache, make_tables, scale_of
from zse_b200.cache.quant_kv import QuantKV
from zse_b200.ops.backend import TorchOps


@pytest.fixture()
def ops():
    return TorchOps("cpu")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(v):
    return torch.tensor(v, dtype=torch.int32)


def i64(v):
    return torch.tensor(v, dtype=torch.int64)


def freqs_of(rot):
    return (1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).float()


# ---- the operators ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd,rot", [(64, 64), (96, 48), (128, 96), (80, 80)])
@pytest.mark.parametrize("planes,bias", [(0, False), (2, True)])
def test_write(ops, hd, rot, planes, bias):
    nh, nkv, M, bs = 6, 2, 21, 16
    g, cols = gen(hd + rot), (6 + 4) * hd
    pos = torch.randint(0, 100000, (M,), generator=g, dtype=torch.int32)
    pos[0] = 2 ** 31 - 1
    slots = torch.randperm(3 * bs, generator=g)[:M]
    slots[4] = -1
    kv = QuantKV.zeros((3, 2, nkv, bs, hd))
    qkv = torch.randn(M, cols + 8, generator=g).half()
    x, p, b = qkv[:, :cols].double(), None, None
    if planes:
        p, b = torch.randn(planes, M, cols, generator=g), torch.randn(cols, generator=g).half() if bias else None
        x = (p.sum(0) + b.float()).double()
    before = qkv.clone()
    ops.rope_kv_write_q8(qkv, kv, pos, slots, freqs_of(rot), M, nh, nkv, hd, planes=p, n_planes=planes, bias=b)
    assert torch.equal(qkv[:, nh * hd:], before[:, nh * hd:])
    k = slots >= 0
    blk, off = slots[k] // bs, slots[k] % bs
    check_write(x[k], pos[k], freqs_of(rot), nh, nkv, hd, qkv[k, : nh * hd], kv.data[blk, :, :, off], kv.scale[blk, :, :, off])
    assert int((kv.data != 0).any(-1).sum()) == 2 * nkv * (M - 1)          # nothing else was written


@pytest.mark.parametrize("nh,nkv,hd", [(4, 4, 64), (14, 2, 96)])
@pytest.mark.parametrize("window", [0, 1, 20])
def test_attention(ops, nh, nkv, hd, window):
    bs, lens, rows = 16, [0, 1, 40, 130], [0, 1, 3, 5]
    g = gen(nh + window)
    data, scale = make_cache(g, 16, nkv, bs, hd, "cpu")
    tables = make_tables(g, lens, bs, 16, "cpu", holes=[(3, 2), (2, 2)])
    scale[tables[1, 0].long(), :, :, 1:] = float("nan")                    # behind the sequence
    kv = QuantKV(data, scale)
    q = torch.randn(9, nh * hd, generator=g).half()
    out = torch.full((9, nh * hd), 3.0, dtype=torch.float16)
    ops.attn_decode_q8(q, kv, tables, i32(lens), out, 4, nh, nkv, hd, scale_of(hd), window=window)
    want, tol = attention(q, data, scale, tables, list(enumerate(lens)), nh, scale_of(hd), window)
    assert ((out[:4].double() - want).abs() <= tol).all() and (out[4:] == 3).all()
    ops.attn_decode_q8(q, kv, tables, None, out, 4, nh, nkv, hd, scale_of(hd), window=window, cu_q=i32([0, 0, 1, 4, 9]),
                       q_pos0=i32([0, 0, 37, 125]), max_q=5)
    seen = [(s, n - r + 1 + i) for s, (n, r) in enumerate(zip(lens, rows)) for i in range(r)]
    want, tol = attention(q, data, scale, tables, seen, nh, scale_of(hd), window)
    assert ((out.double() - want).abs() <= tol).all()


def test_read_gives_what_the_kernels_of_fp16_take(ops):
    """Attention over the pages read back is attention over the 8-bit cache, up to the rounding of the pages."""
    nh, nkv, hd, bs, lens = 4, 2, 64, 16, [17, 0, 48, 5]
    g = gen(1)
    data, scale = make_cache(g, 9, nkv, bs, hd, "cpu")
    tables = make_tables(g, lens, bs, 9, "cpu", holes=[(2, 1)])
    scale[tables[3, 0].long(), :, :, 5:] = float("nan")
    kv = QuantKV(data, scale)
    cu = i32([0, 2, 2, 5, 6])
    pages, places = torch.zeros(7, 2, nkv, bs, hd, dtype=torch.float16), torch.full((4, 4), 9, dtype=torch.int32)
    pages[6] = 4
    ops.kv_read_q8(kv, tables, i32(lens), cu, 4, pages, places)
    assert places.tolist() == [[0, 1, -1, -1], [-1] * 4, [2, -1, 4, -1], [5, -1, -1, -1]]
    assert (pages[6] == 4).all() and (pages[3] == 0).all() and (pages[5, :, :, 5:] == 0).all() and not pages.isnan().any()
    q = torch.randn(4, nh * hd, generator=g).half()
    a, b = torch.zeros(4, nh * hd, dtype=torch.float16), torch.zeros(4, nh * hd, dtype=torch.float16)
    ops.attn_decode_q8(q, kv, tables, i32(lens), a, 4, nh, nkv, hd, scale_of(hd))
    ops.attn_decode(q, pages, places, i32(lens), b, 4, nh, nkv, hd, bs, scale_of(hd))
    want, tol = attention(q, data, scale, tables, list(enumerate(lens)), nh, scale_of(hd))
    # keys and values rounded to fp16: 2^-11 of a value, and of a key in the exponent
    most = q.double().view(4, nkv, nh // nkv, hd).abs().sum(-1).amax((1, 2))[:, None] * scale[:, 0].nan_to_num(0).double().max() * 127 * scale_of(hd)
    size = scale[:, 1].nan_to_num(0).double().max() * 127
    assert ((a.double() - want).abs() <= tol).all()
    assert ((b.double() - want).abs() <= 2 * tol + (2 * most + 2) * 2.0 ** -11 * size).all()


def test_zeros_infinities_and_nan(ops):
    nh, nkv, hd = 2, 1, 64
    x = torch.randn(3, 4 * hd, generator=gen(0)).half()
    x[0, 2 * hd: 3 * hd] = 0
    x[1, 3 * hd + 4], x[2, 3 * hd + 4] = float("-inf"), float("nan")
    kv = QuantKV.zeros((1, 2, 1, 16, hd))
    ops.rope_kv_write_q8(x, kv, i32([0, 0, 0]), i64([0, 1, 2]), freqs_of(hd), 3, nh, nkv, hd)
    assert (kv.data[0, 0, 0, 0] == 128).all() and kv.scale[0, 0, 0, 0] == 0
    assert kv.data[0, 1, 0, 1, 4] == 1 and abs(float(kv.scale[0, 1, 0, 1]) * 127 / 65504 - 1) < 2.0 ** -22
    assert kv.scale[0, 1, 0, 2].isnan() and not kv.scale[0, 0].isnan().any()
    out = torch.zeros(2, nh * hd, dtype=torch.float16)
    ops.attn_decode_q8(x[:2], kv, i32([[0], [0]]), i32([3, 2]), out, 2, nh, nkv, hd, scale_of(hd))
    assert out[0].isnan().all() and not out[1].isnan().any()


# ---- refusals ---------------------------------------------------------------------------------------------------------------
def _write_args(M=2, nh=4, nkv=2, hd=64):
    return dict(qkv=torch.zeros(M, (nh + 2 * nkv) * hd, dtype=torch.float16), kv=QuantKV.zeros((2, 2, nkv, 16, hd)), positions=i32([0] * M),
                slots=i64(list(range(M))), inv_freq=freqs_of(hd), M=M, nh=nh, nkv=nkv, hd=hd)


@pytest.mark.parametrize("change", [
    dict(qkv=torch.zeros(2, 8 * 64)), dict(qkv=torch.zeros(2, 7 * 64, dtype=torch.float16)), dict(qkv=torch.zeros(1, 8 * 64, dtype=torch.float16)),
    dict(qkv=torch.zeros(8 * 64, 2, dtype=torch.float16).T), dict(qkv=None), dict(positions=i64([0, 0])), dict(positions=i32([0])),
    dict(slots=i32([0, 1])), dict(slots=i64([0])), dict(slots=i64([0, 32])), dict(inv_freq=freqs_of(64)[:12]), dict(inv_freq=freqs_of(80)), dict(inv_freq=freqs_of(64).double()),
    dict(nkv=4), dict(hd=32), dict(nh=5), dict(M=3), dict(M=-1), dict(bias=torch.zeros(512, dtype=torch.float16)),
    dict(planes=torch.zeros(2, 2, 8 * 64), n_planes=0), dict(planes=torch.zeros(2, 2, 8 * 64), n_planes=3),
    dict(planes=torch.zeros(1, 2, 8 * 64), n_planes=1, bias=torch.zeros(8, dtype=torch.float16)),
    dict(q_out=torch.zeros(2, 255, dtype=torch.float16)), dict(q_out=torch.zeros(2, 256)),
])
def test_write_refuses(ops, change):
    args = _write_args()
    ops.rope_kv_write_q8(**args)
    before = args["kv"].data.clone()
    with pytest.raises((ValueError, AttributeError)):
        ops.rope_kv_write_q8(**{**args, **change})
    assert torch.equal(before, args["kv"].data)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 256)), dict(q=torch.zeros(2, 255, dtype=torch.float16)), dict(q=torch.zeros(1, 256, dtype=torch.float16)),
    dict(out=torch.zeros(2, 255, dtype=torch.float16)), dict(out=torch.zeros(1, 256, dtype=torch.float16)), dict(out=torch.zeros(2, 256)),
    dict(block_tables=i64([[0], [1]])), dict(block_tables=i32([[0]])), dict(block_tables=i32([[0], [2]])), dict(seq_lens=None),
    dict(seq_lens=i32([1])), dict(seq_lens=i32([1, 17])), dict(seq_lens=i32([1, -1])), dict(S=3), dict(S=-1), dict(nh=3), dict(nkv=1), dict(hd=128), dict(window=-1),
    dict(max_q=2), dict(max_q=0), dict(cu_q=i32([0, 1, 2])), dict(cu_q=i32([0, 1]), q_pos0=i32([0, 0])),
    dict(cu_q=i32([0, 1, 2]), q_pos0=i32([0])), dict(cu_q=i32([0, 1, 2]), q_pos0=i32([0, 0]), max_q=65),
    dict(cu_q=i64([0, 1, 2]), q_pos0=i32([0, 0])), dict(scratch=torch.zeros(4096, dtype=torch.float16)),
    dict(cu_q=i32([0, 2, 2]), q_pos0=i32([0, 0])), dict(cu_q=i32([0, 1, 3]), q_pos0=i32([0, 0]), max_q=2), dict(scratch=torch.zeros(64, 64)), dict(scratch=torch.zeros(4096)[::2]),
])
def test_attention_refuses(ops, change):
    args = dict(q=torch.zeros(2, 256, dtype=torch.float16), kv=QuantKV.zeros((2, 2, 2, 16, 64)), block_tables=i32([[0], [1]]),
                seq_lens=i32([3, 16]), out=torch.zeros(2, 256, dtype=torch.float16), S=2, nh=4, nkv=2, hd=64, scale=0.125)
    ops.attn_decode_q8(**args)
    with pytest.raises(ValueError):
        ops.attn_decode_q8(**{**args, **change})


def test_too_many_heads_per_kv_head_are_refused(ops):
    z = torch.zeros(1, 17 * 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="16"):
        ops.attn_decode_q8(z, QuantKV.zeros((1, 2, 1, 16, 64)), i32([[0]]), i32([1]), z.clone(), 1, 17, 1, 64, 0.125)


@pytest.mark.parametrize("change", [
    dict(out=torch.zeros(3, 2, 2, 16, 64)), dict(out=torch.zeros(3, 2, 2, 16, 32, dtype=torch.float16)),
    dict(out=torch.zeros(3, 2, 2, 16, 128, dtype=torch.float16)[..., :64]), dict(out_tables=torch.zeros(2, 2, dtype=torch.int64)),
    dict(out_tables=torch.zeros(1, 2, dtype=torch.int32)), dict(cu_blocks=i32([0, 1])), dict(cu_blocks=i64([0, 1, 3])), dict(cu_blocks=i32([0, 1, 2])),
    dict(cu_blocks=i32([0, 2, 4])), dict(seq_lens=i32([3])), dict(seq_lens=i32([3, 33])), dict(seq_lens=i32([-3, 20])), dict(S=3), dict(S=-1), dict(block_tables=i32([[0, -1], [1, 4]])),
])
def test_read_refuses(ops, change):
    args = dict(kv=QuantKV.zeros((4, 2, 2, 16, 64)), block_tables=i32([[0, -1], [1, 3]]), seq_lens=i32([3, 20]), cu_blocks=i32([0, 1, 3]),
                S=2, out=torch.zeros(3, 2, 2, 16, 64, dtype=torch.float16), out_tables=torch.zeros(2, 2, dtype=torch.int32))
    ops.kv_read_q8(**args)
    with pytest.raises(ValueError):
        ops.kv_read_q8(**{**args, **change})


def test_cache_object():
    with pytest.raises(TypeError):
        QuantKV(torch.zeros(1, 2, 1, 16, 64, dtype=torch.int8), torch.zeros(1, 2, 1, 16))
    with pytest.raises(TypeError):
        QuantKV(torch.zeros(1, 2, 1, 16, 64, dtype=torch.uint8), torch.zeros(1, 2, 1, 16).half())
    with pytest.raises(ValueError):
        QuantKV(torch.zeros(1, 2, 1, 16, 64, dtype=torch.uint8), torch.zeros(1, 2, 1, 8))
    with pytest.raises(ValueError):
        QuantKV(torch.zeros(1, 1, 1, 16, 64, dtype=torch.uint8), torch.zeros(1, 1, 1, 16))
    kv = QuantKV.zeros((3, 4, 2, 1, 16, 64))
    kv.data[:, 1], kv.scale[:, 1] = 5, 0.5
    kv.copy_block(1, 3)
    assert (kv.data[:, 3] == 5).all() and (kv.scale[:, 3] == 0.5).all() and (kv.data[:, 2] == 0).all()
    layer = kv[2]
    assert (layer.num_blocks, layer.kv_heads, layer.block_size, layer.head_dim) == (4, 1, 16, 64)
    assert layer.data.data_ptr() == kv.data[2].data_ptr()


@pytest.mark.parametrize("pos", [-1, -4, -2 ** 31, 28, 33, 2 ** 31 - 1])
@pytest.mark.parametrize("window", [0, 9])
def test_positions_outside_the_table_are_refused(ops, pos, window):
    """Five rows, of which the first is before a table of 32 tokens or the last behind it."""
    q, kv = torch.ones(5, 256, dtype=torch.float16), QuantKV.zeros((2, 2, 2, 16, 64))
    call = lambda p: ops.attn_decode_q8(q, kv, i32([[0, 1]]), None, q.clone(), 1, 4, 2, 64, 0.125, window=window, cu_q=i32([0, 5]),
                                        q_pos0=i32([p]), max_q=5)
    call(27)
    with pytest.raises(ValueError):
        call(pos)
