"""The 8-bit products in pairs of CTAs, form by form: K whole and in parts, rows written 32 bytes at a time and by way of shared memory, each
output type with and without a bias.  Every case says which form it is for, and that is checked against the plan (on a GPU of 148 SMs)."""
import pytest
import torch

from tests.helpers.fp8_oracle import blocks, check_out, check_rows, gated, make_rows, make_weight, product, values, weight
from zse_b200.ops.fp8 import Fp8Rows, Fp8Weight

pytestmark = pytest.mark.gpu
DEV, F8, U8 = "cuda", torch.float8_e4m3fn, torch.uint8
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from zse_b200.ops.backend import make_ops
    return make_ops(DEV)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def planned(form, M, N, K, glu=False):
    """``form``: (token columns or 0 for pairs, parts of K, None for any number above one)."""
    from zse_b200.ops.native import gemm_fp8_plan
    got = gemm_fp8_plan(M, N, K, glu=glu)
    if form[0] == 0 and form[1] is None:
        assert got[0] == 0
    elif torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert got == form if form[1] is not None else got[0] == form[0] and got[1] > 1, (got, form)


def wide(out, N):
    """Whether rows are written 32 bytes at a time: addresses, row distances and widths are multiples of that."""
    item = out.element_size()
    return (out.data_ptr() | out.stride(0) * item | N * item) % 32 == 0


# parts of K, tokens, weight rows, columns of K: one round of units and several, the last of them not full; rows and columns behind the last
FORMS = [(1, 600, 2544, 528), (1, 2100, 9472, 144), (2, 600, 2544, 4112), (2, 2048, 3312, 8192), (4, 600, 1264, 4112), (4, 2100, 2288, 4096)]


@pytest.mark.parametrize("parts,M,N,K", FORMS)
@pytest.mark.parametrize("dtype,bias", [(t, b) for t in (F16, BF16, F32) for b in (None, F16, BF16, F32)])
@pytest.mark.parametrize("extra", [16, 3])                                  # between the rows: wide stores, or not
def test_linear(ops, parts, M, N, K, dtype, bias, extra):
    planned((0, parts), M, N, K)
    g = gen(M + N + K)
    if dtype is F32:
        N -= 8                                                              # (a multiple of eight, not of sixteen: the last store is half of one)
    x, w = make_rows(g, M + 1, K, DEV), make_weight(g, N, K, DEV, bias)
    x.scale[:, M:] = float("nan")
    whole = torch.full((M + 1, N + extra), 5.0, dtype=dtype, device=DEV)
    out = whole[:, :N]
    assert wide(out, N) == (extra == 16)
    ops.linear_fp8(w, x, M, out)
    torch.cuda.synchronize()
    ops.check()
    y, off = product(values(x, M), weight(w)[0])
    if bias is not None:
        y = y + w.bias.double()
        off = off + 2.0 ** -24 * y.abs()
    check_out(y, off, out[:M])
    assert (whole[M:] == 5).all() and (whole[:, N:] == 5).all()


def test_128_token_columns_with_k_whole(ops):
    for M, N, K in ((128, 10240, 1024), (100, 10232, 1040)):
        planned((128, 1), M, N, K)
        g = gen(M)
        x, w, out = make_rows(g, M, K, DEV), make_weight(g, N, K, DEV), torch.empty(M, N, dtype=F16, device=DEV)
        ops.linear_fp8(w, x, M, out)
        ops.check()
        check_out(*product(values(x, M), weight(w)[0]), out)


# ---- sums of whole numbers: no rounding anywhere, so not a unit may be missing ------------------------------------------------------------
def whole_numbers(g, M, N, K, glu=False):
    """Numbers 1 .. 16 (exact in e4m3) with scales 1, 2, 4 and 1, 2: a block's sum is at most 2^15, all of them 8 * 256 K <= 2^24."""
    assert K <= 8192
    ints = lambda *shape: torch.randint(1, 17, shape, generator=g).float().to(F8)             # noqa: E731
    parts = 2 if glu else 1
    x = Fp8Rows(ints(M, K).to(DEV), torch.exp2(torch.randint(0, 3, (blocks(K), M), generator=g).float()).to(DEV))
    s = torch.exp2(torch.randint(0, 2, (parts * blocks(N), blocks(K)), generator=g).float())
    return x, Fp8Weight(ints(parts * N, K).to(DEV), s.to(DEV), None, glu)


@pytest.mark.parametrize("form,M,N,K", [
    ((16, 1), 1, 19200, 272), ((16, None), 9, 5120, 2048), ((32, 1), 31, 20000, 144), ((32, None), 20, 1000, 4096), ((64, 1), 64, 19210, 400),
    ((64, None), 50, 5110, 4096), ((128, 1), 128, 10240, 1024), ((128, None), 120, 5120, 8192)] + [((0, p), *c) for p, *c in FORMS])
def test_whole_numbers(ops, form, M, N, K):
    planned(form, M, N, K)
    x, w = whole_numbers(gen(K), M, N, K)
    out = torch.empty(M, N, device=DEV)
    ops.linear_fp8(w, x, M, out)
    ops.check()
    assert torch.equal(out.double(), values(x, M) @ weight(w)[0].t())


GATED_FORMS = [((16, 1), 1, 19200, 144), ((16, None), 7, 5120, 2048), ((32, 1), 32, 13808, 400), ((32, None), 18, 4096, 2048), ((64, 1), 33, 9600, 272),
               ((64, None), 60, 5120, 4096), ((0, 1), 1300, 1936, 528), ((0, 2), 1300, 640, 4096), ((0, 2), 2048, 1648, 8192), ((0, 4), 300, 400, 8192),
               ((0, 4), 1100, 1936, 4096)]


@pytest.mark.parametrize("form,M,N,K", GATED_FORMS)
def test_gated_whole_numbers(ops, form, M, N, K):
    """The gates are so large that silu leaves them as they are: sums exact, then a sigmoid within 10 2^-24 and two products."""
    planned(form, M, N, K, glu=True)
    x, w = whole_numbers(gen(K), M, N, K, glu=True)
    out = Fp8Rows.empty(M, N, DEV)
    ops.linear_swiglu_fp8(w, x, M, out)
    ops.check()
    gate, up = (values(x, M) @ p.t() for p in weight(w))
    check_rows(gate * up, 12 * 2.0 ** -24, out, M)


# ---- numbers that are none, and none at all -----------------------------------------------------------------------------------------------
def same_bits(a, b):
    return torch.equal(a.contiguous().view(U8), b.contiguous().view(U8))


@pytest.mark.parametrize("parts,M,N,K", FORMS)
@pytest.mark.parametrize("dtype,extra", [(F16, 16), (F16, 3), (BF16, 16), (F32, 16), (F32, 1)])
def test_a_nan_stays_in_its_row_or_column(ops, parts, M, N, K, dtype, extra):
    planned((0, parts), M, N, K)
    g = gen(5)
    x, w = make_rows(g, M, K, DEV, hot=False), make_weight(g, N, K, DEV)
    clean, out = (torch.empty(M, N + extra, dtype=dtype, device=DEV)[:, :N] for _ in range(2))
    assert wide(out, N) == (extra == 16)
    ops.linear_fp8(w, x, M, clean)
    rows, last = (3, 130, 257, M - 1), blocks(K) - 1
    x.data.view(U8)[rows[0], K - 1] = 0x7F
    x.scale[last, rows[1]] = float("inf")
    x.scale[0, rows[2]] = float("nan")
    x.scale[:, rows[3]] = 0
    w.data.view(U8)[N - 1, 0] = 0x7F
    ops.linear_fp8(w, x, M, out)
    ops.check()
    assert out[rows[0]].isnan().all() and out[rows[2]].isnan().all() and out[:, N - 1].isnan().all()
    last_block = values(Fp8Rows(x.data[:, last * 128:], torch.ones(1, M, device=DEV)), M)[rows[1]] @ weight(w)[0][:, last * 128:].t()
    hit = out[rows[1], : N - 1]
    over = 65504 if dtype is F16 else float("inf")                          # (fp16 is held within its largest)
    assert (hit.isnan() | (hit.abs() == over)).all() and (hit[last_block[: N - 1] != 0].double() == torch.sign(last_block[: N - 1][last_block[: N - 1] != 0]) * over).all()
    assert (out[rows[3], : N - 1] == 0).all()
    keep = torch.ones(M, dtype=torch.bool, device=DEV)
    keep[list(rows)] = False
    assert same_bits(out[keep][:, : N - 1], clean[keep][:, : N - 1])


@pytest.mark.parametrize("parts,M,N,K", [FORMS[0], FORMS[3], FORMS[4]])
@pytest.mark.parametrize("extra", [16, 3])
def test_fp16_is_held_within_its_largest(ops, parts, M, N, K, extra):
    planned((0, parts), M, N, K)
    x, w = make_rows(gen(7), M, K, DEV, hot=False), make_weight(gen(8), N, K, DEV, F32)
    x.scale *= 1e7
    out = torch.empty(M, N + extra, dtype=F16, device=DEV)[:, :N]
    ops.linear_fp8(w, x, M, out)
    ops.check()
    y, off = product(values(x, M), weight(w)[0])
    y = y + w.bias.double()
    check_out(y, off + 2.0 ** -24 * y.abs(), out)
    assert out.isfinite().all() and (out.abs() == 65504).sum() > M * N // 2


@pytest.mark.parametrize("form,M,N,K", GATED_FORMS)
@pytest.mark.parametrize("gelu", [False, True])
def test_gated_a_nan_stays_in_its_row_or_block(ops, form, M, N, K, gelu):
    """A NaN or an infinity of a row reaches that row; one of a weight row reaches the block of 128 outputs that it is in; rows of scale 0
    are zeros with scale 0."""
    planned(form, M, N, K, glu=True)
    g = gen(6)
    x, w = make_rows(g, M, K, DEV, hot=False), make_weight(g, N, K, DEV, glu=True)
    clean, out = Fp8Rows.empty(M, N, DEV), Fp8Rows.empty(M, N, DEV)
    ops.linear_swiglu_fp8(w, x, M, clean, gelu=gelu)
    bad, none, last = sorted({0, M // 2}), M - 1, blocks(K) - 1
    if M > 2:
        x.data.view(U8)[0, K - 1] = 0x7F
        x.scale[last, M // 2] = float("inf")
        x.scale[:, none] = 0
    else:
        bad, none = [], None
    w.data.view(U8)[N + 5, K - 2] = 0x7F                                     # an up row of the first block, a gate row of the last
    w.data.view(U8)[N - 1, 1] = 0x7F
    ops.linear_swiglu_fp8(w, x, M, out, gelu=gelu)
    ops.check()
    y = out.dequant()
    for row in bad:
        assert not y[row].isfinite().any() and not out.scale[:, row].isfinite().any()
    first, rest = slice(0, 128), slice((N - 1) // 128 * 128, N)
    assert y[:, first].isnan().all() and y[:, rest].isnan().all()
    keep = torch.ones(M, dtype=torch.bool, device=DEV)
    keep[bad] = False
    inner = slice(128, rest.start)
    if none is not None:
        keep[none] = False
        assert (out.data[none, inner].float() == 0).all() and (out.scale[1: blocks(N) - 1, none] == 0).all()
    assert torch.equal(out.data.view(U8)[keep][:, inner], clean.data.view(U8)[keep][:, inner])
    assert torch.equal(out.scale[1: blocks(N) - 1, keep], clean.scale[1: blocks(N) - 1, keep])


# ---- rows more than 2^31 bytes from the first -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shift", [0, 1])
def test_offsets_past_2_31(ops, shift):
    M, N, K, ld = 520, 256, 4096, (1 << 22) + 16
    planned((0, None), M, N, K)
    g = gen(10)
    x, w = make_rows(g, M, K, DEV), make_weight(g, N, K, DEV)
    far = torch.empty(ld * M, dtype=U8, device=DEV).view(F8).as_strided((M, K), (ld, 1))       # rows that are read
    far.view(U8).copy_(x.data.view(U8))
    out = torch.empty(ld * M + 1, dtype=BF16, device=DEV)[shift:].as_strided((M, N), (ld, 1))
    assert wide(out, N) == (shift == 0) and (M - 1) * ld > 1 << 31
    ops.linear_fp8(w, Fp8Rows(far, x.scale), M, out)
    ops.check()
    check_out(*product(values(x, M), weight(w)[0]), out)


@pytest.mark.parametrize("M,ld", [(2, (1 << 31) + 16), (520, (1 << 22) + 16)])
def test_rows_in_8_bits_past_2_31(ops, M, ld):
    N, K = 272, 1024
    if M > 256:
        planned((0, None), M, N, K, glu=True)
    g = gen(11)
    x, w = make_rows(g, M, K, DEV, hot=False), make_weight(g, N, K, DEV, glu=True)
    data = torch.empty(ld * (M - 1) + N, dtype=U8, device=DEV).view(F8).as_strided((M, N), (ld, 1))
    out = Fp8Rows(data, torch.empty(blocks(N), M, device=DEV))
    ops.linear_swiglu_fp8(w, x, M, out)
    ops.check()
    (gate, g_off), (up, u_off) = (product(values(x, M), p) for p in weight(w))
    check_rows(*gated(gate, up, g_off, u_off, False), out, M)
    r = torch.randn(M, N, generator=g).to(DEV)
    ops.add_rmsnorm_fp8(r, None, 0, None, torch.ones(N, device=DEV).half(), out, M, 1e-6)
    one = Fp8Rows.empty(M, N, DEV)
    ops.add_rmsnorm_fp8(r, None, 0, None, torch.ones(N, device=DEV).half(), one, M, 1e-6)
    assert torch.equal(out.data.view(U8), one.data.view(U8)) and torch.equal(out.scale, one.scale)


# ---- how they are called ------------------------------------------------------------------------------------------------------------------------
def layer(seed, M, H, ff):
    g = gen(seed)
    return dict(r=torch.randn(M, H, generator=g).to(DEV), w16=(1 + torch.randn(H, generator=g) * 0.1).half().to(DEV),
                up=make_weight(g, ff, H, DEV, glu=True), down=make_weight(g, H, ff, DEV), x=Fp8Rows.empty(M, H, DEV),
                h=Fp8Rows.empty(M, ff, DEV), plane=torch.empty(1, M, H, device=DEV), M=M)


def feed_forward(ops, r, w16, up, down, x, h, plane, M):
    ops.add_rmsnorm_fp8(r, None, 0, None, w16, x, M, 1e-6)
    ops.linear_swiglu_fp8(up, x, M, h)
    ops.linear_fp8(down, h, M, plane[0])
    ops.add_rmsnorm_fp8(r, plane, 1, None, w16, x, M, 1e-6)


def bits(s):
    return [t.clone() for t in (s["r"], s["plane"], s["x"].data.view(U8), s["x"].scale, s["h"].data.view(U8), s["h"].scale)]


# seed, tokens, hidden and feed-forward columns, parts of K of the gated product and of the other
LAYERS = [(1, 600, 4096, 640, 4, 1), (2, 2100, 4096, 1280, 2, 1), (3, 600, 1280, 4096, 1, 4)]


def runs_of_pairs():
    for _, M, H, ff, up, down in LAYERS:
        planned((0, up), M, ff, H, glu=True)
        planned((0, down), M, H, ff)
    return [layer(*c[:4]) for c in LAYERS]


def wanted(ops, runs):
    start, want = [s["r"].clone() for s in runs], []
    for s in runs:
        feed_forward(ops, **s)
        want.append(bits(s))
    torch.cuda.synchronize()
    return start, want


def reset(runs, start):
    for s, r in zip(runs, start):
        s["r"].copy_(r)
        s["plane"].zero_()
        for t in (s["x"], s["h"]):
            t.scale.zero_()
            t.data.view(U8).zero_()
    torch.cuda.synchronize()


def same(runs, want):
    torch.cuda.synchronize()
    return all(torch.equal(a, b) for s, w in zip(runs, want) for a, b in zip(bits(s), w))


def test_streams_and_graphs(ops):
    runs = runs_of_pairs()
    start, want = wanted(ops, runs)
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(5):
        reset(runs, start)
        for s, stream in zip(runs, streams):
            with torch.cuda.stream(stream):
                feed_forward(ops, **s)
        assert same(runs, want)
    graphs = []
    for s, stream in zip(runs, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            feed_forward(ops, **s)
        graphs.append(graph)
    for _ in range(5):
        reset(runs, start)
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        assert same(runs, want)
    ops.check()


def test_a_weight_written_just_before(ops):
    M, N, K = 600, 2048, 2048
    planned((0, None), M, N, K)
    planned((0, None), M, N, K, glu=True)
    g = gen(M)
    x = make_rows(g, M, K, DEV, hot=False)
    for glu in (False, True):
        ws, want = [make_weight(g, N, K, DEV, glu=glu) for _ in range(2)], []

        def call(w, out):
            ops.linear_swiglu_fp8(w, x, M, out) if glu else ops.linear_fp8(w, x, M, out)

        def empty():
            return Fp8Rows.empty(M, N, DEV) if glu else torch.empty(M, N, device=DEV)

        def all_bits(out):
            return torch.cat([out.data.view(U8).flatten(), out.scale.view(U8).flatten()]) if glu else out.view(U8).flatten().clone()
        for w in ws:
            out = empty()
            call(w, out)
            want.append(all_bits(out))
        w, out = Fp8Weight(ws[0].data.clone(), ws[0].scale.clone(), None, glu), empty()
        for i in range(20):
            w.data.view(U8).copy_(ws[i % 2].data.view(U8))
            w.scale.copy_(ws[i % 2].scale)
            call(w, out)
            assert torch.equal(all_bits(out), want[i % 2])


def test_two_threads(ops):
    """Two Python threads, each on a stream of its own, with calls of both kinds of products at once."""
    import threading
    runs = runs_of_pairs() + [layer(4, 40, 1024, 2048), layer(5, 1, 2048, 1024)]
    start, want = wanted(ops, runs)
    for _ in range(3):
        reset(runs, start)
        wrong, gate = [], threading.Barrier(2)

        def work(mine):
            try:
                stream = torch.cuda.Stream()
                gate.wait(60)
                with torch.cuda.stream(stream):
                    for s in mine:
                        feed_forward(ops, **s)
                stream.synchronize()
            except Exception as e:                                          # noqa: BLE001
                wrong.append(e)
        threads = [threading.Thread(target=work, args=(runs[i::2],)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(120)
        assert not wrong and same(runs, want)
    ops.check()


def test_first_calls_from_two_threads():
    """What a kind of call sets up for itself the first time may be set up by two threads at once."""
    import subprocess
    import sys
    code = """
import threading, torch
from tests.helpers.fp8_oracle import make_rows, make_weight
from zse_b200.ops.backend import make_ops
from zse_b200.ops.fp8 import Fp8Rows
ops, g = make_ops("cuda"), torch.Generator().manual_seed(1)
sizes = (1, 20, 40, 120, 600, 2100)
x = {M: make_rows(g, M, 4096, "cuda", hot=False) for M in sizes}
w, up = make_weight(g, 2544, 4096, "cuda"), make_weight(g, 1680, 4096, "cuda", glu=True)
def outs():
    return {M: (torch.zeros(M, 2544, device="cuda"), Fp8Rows.empty(M, 1680, "cuda")) for M in sizes}
both, gate, wrong = [outs(), outs()], threading.Barrier(2), []
torch.cuda.synchronize()
def work(out):
    try:
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for M in sizes:
                gate.wait(60)
                ops.linear_fp8(w, x[M], M, out[M][0])
                ops.linear_swiglu_fp8(up, x[M], M, out[M][1])
        stream.synchronize()
    except Exception as e:
        wrong.append(e)
threads = [threading.Thread(target=work, args=(o,)) for o in both]
[t.start() for t in threads]
[t.join(120) for t in threads]
assert not wrong, wrong
again = outs()
for M in sizes:
    ops.linear_fp8(w, x[M], M, again[M][0])
    ops.linear_swiglu_fp8(up, x[M], M, again[M][1])
    for o in both:
        assert torch.equal(o[M][0], again[M][0]) and torch.equal(o[M][1].scale, again[M][1].scale)
        assert torch.equal(o[M][1].data.view(torch.uint8), again[M][1].data.view(torch.uint8))
ops.check()
print("FINE")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert "FINE" in done.stdout, done.stderr[-2000:]
