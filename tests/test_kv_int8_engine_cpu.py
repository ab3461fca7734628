"""Engines that keep their KV cache in 8 bits, on the CPU path: every way of getting tokens into the cache and out of it again."""
import random

import pytest
import torch

from zse_b200.cache.block_pool import BlockPool, row_bytes
from zse_b200.cache.quant_kv import QuantKV, refuses
from zse_b200.config import EngineConfig
from zse_b200.engine import ZStreamerEngine
from zse_b200.format import synth
from zse_b200.sched.request import FinishReason


@pytest.fixture(scope="module")
def model_path(tmp_path_factory):
    p = str(tmp_path_factory.mktemp("m") / "tiny.zse")
    synth.write_random_model(p, synth.shape_config("tiny"), seed=3)
    return p


def engine(path, **kw):
    return ZStreamerEngine(path, config=EngineConfig(**{**dict(device="cpu", max_batch_seqs=8, max_seq_len=256, kv_dtype="int8"), **kw}))


def prompts(n, lo, hi, seed=0):
    rng = random.Random(seed)
    return [[rng.randrange(1024) for _ in range(rng.randint(lo, hi))] for _ in range(n)]


def run(eng, ps, n):
    ids = [eng.add_request_tokens(p, max_tokens=n, temperature=0.0, stop_tokens=[]) for p in ps]
    eng.run_until_done()
    outs = [eng.get_result(i) for i in ids]
    assert all(o.finish_reason == FinishReason.LENGTH for o in outs)
    return [o.output_tokens for o in outs]


def logits_after(eng, toks, cuts, sid=77):
    """fp32 logits after the last of ``toks``, passed in portions that end at ``cuts`` (single tokens are decode steps)."""
    r = eng.runner
    r.cache.allocate_sequence(sid, num_tokens=0)
    try:
        at = 0
        for cut in list(cuts) + [len(toks)]:
            r.cache.extend_sequence(sid, cut - at)
            if cut - at == 1 and at > 0:
                r.decode([sid], [toks[at]])
            else:
                r.prefill([(sid, toks[at:cut], at)])
            at = cut
        return r.buf.logits[0].float().clone()
    finally:
        r.cache.free_sequence(sid)


def test_logits_do_not_depend_on_how_the_prompt_is_cut(model_path):
    """The cache is what attention reads, whatever the pass: one prefill, chunks, chunks of a few rows, single steps.  They differ in
    roundings to fp16 (the pages that long chunks read, the rows' activations): some tens of 2^-11 through two layers, within 2^-5 of
    the largest logit; a wrong page, place or scale changes them by their own size."""
    eng = engine(model_path)
    toks = prompts(1, 60, 60, seed=5)[0]
    whole = logits_after(eng, toks, [])
    size = whole.abs().max()
    for cuts in ([17], [16, 32, 48], [3, 9, 12, 40], [30, 34, 38, 55], list(range(50, 60)), list(range(1, 60))):
        assert (logits_after(eng, toks, cuts) - whole).abs().max() <= size * 2.0 ** -5, cuts
    plain = ZStreamerEngine(model_path, config=EngineConfig(device="cpu", max_batch_seqs=8, max_seq_len=256))
    # bytes are within 1/254 of a row's largest value: a few per cent after two layers, and not nothing
    off = (logits_after(plain, toks, []) - whole).abs().max()
    assert 0 < off <= size / 8
    eng.destroy(); plain.destroy()


def test_batches_chunks_sharing_and_preemption_give_the_tokens_of_single_runs(model_path):
    one = engine(model_path, max_batch_seqs=1, enable_prefix_cache=False)
    shared = prompts(1, 40, 40, seed=2)[0]
    ps = prompts(4, 3, 40, seed=1) + [shared + p for p in prompts(3, 3, 9, seed=3)]
    want = [run(one, [p], 10)[0] for p in ps]
    one.destroy()

    def agree(got):
        # (argmax of a random model: a rounding may turn a tie, after which the rest of that sequence differs)
        same = sum(g[0] == w[0] for g, w in zip(got, want))
        return same == len(want) and sum(a == b for g, w in zip(got, want) for a, b in zip(g, w)) >= 0.6 * 10 * len(want)
    for kw in (dict(), dict(prefill_chunk_size=16), dict(kv_blocks=24, max_batch_seqs=4), dict(prefill_chunk_size=5, max_batch_tokens=32)):
        eng = engine(model_path, **kw)
        assert agree(run(eng, ps, 10)), kw
        assert eng.kv_cache.num_sequences == 0
        eng.destroy()


@pytest.mark.parametrize("mode", ["ngram", "self"])
def test_speculative_decoding(model_path, mode):
    ps = [p * 3 for p in prompts(3, 6, 12, seed=4)]
    plain, spec = engine(model_path), engine(model_path, speculative_k=4, speculative_mode=mode)
    a, b = run(plain, ps, 12), run(spec, ps, 12)
    assert [x[0] for x in a] == [x[0] for x in b] and sum(x == y for p, q in zip(a, b) for x, y in zip(p, q)) >= 0.6 * 36
    plain.destroy(); spec.destroy()


def test_prefill_passes_larger_than_the_pages_run_in_groups(model_path):
    """Pages hold one sequence of the longest kind; a pass over more context is read back group by group."""
    eng = engine(model_path, max_seq_len=64, max_batch_tokens=400)
    r = eng.runner
    ps = prompts(6, 20, 60, seed=8)
    assert sum(-(-len(p) // r.cache.block_size) for p in ps) > r.buf.pages.shape[0]
    single = [logits_after(eng, p, []) for p in ps]
    for i, p in enumerate(ps):
        r.cache.allocate_sequence(i, prompt_tokens=p)
    r.prefill([(i, p, 0) for i, p in enumerate(ps)])
    assert len(r.buf.page_groups) > 1
    for i, want in enumerate(single):
        assert (r.buf.logits[i].float() - want).abs().max() <= want.abs().max() * 2.0 ** -5
    eng.destroy()


def test_forked_sequences_copy_bytes_and_scales(model_path):
    eng = engine(model_path)
    r, toks = eng.runner, prompts(1, 21, 21, seed=9)[0]
    r.cache.allocate_sequence(1, prompt_tokens=toks)
    r.prefill([(1, toks, 0)])
    r.cache.fork_sequence(1, 2)
    for sid in (1, 2):
        r.cache.extend_sequence(sid, 1)
    r.decode([1, 2], [5, 6])
    la = r.buf.logits[:2].float().clone()
    want = [logits_after(eng, toks + [t], [21], sid=50 + t) for t in (5, 6)]
    for i in (0, 1):
        assert (la[i] - want[i]).abs().max() <= want[i].abs().max() * 2.0 ** -5
    eng.destroy()


def test_window_and_partial_rotation(tmp_path):
    for name, over in (("phi3", dict(arch="phi3", sliding_window=24)), ("mistral", dict(arch="mistral", sliding_window=17)),
                       ("qwen2", dict(arch="qwen2", partial_rotary_factor=0.5))):
        path = str(tmp_path / f"{name}.zse")
        synth.write_random_model(path, synth.shape_config("tiny", **over), seed=4)
        eng, plain = engine(path), ZStreamerEngine(path, config=EngineConfig(device="cpu", max_batch_seqs=8, max_seq_len=256))
        toks = prompts(1, 70, 70, seed=6)[0]
        whole = logits_after(eng, toks, [])
        assert (logits_after(eng, toks, [33, 40, 41, 42]) - whole).abs().max() <= whole.abs().max() * 2.0 ** -5
        assert (logits_after(plain, toks, []) - whole).abs().max() <= whole.abs().max() / 8
        eng.destroy(); plain.destroy()


def test_adapters_beside_it(model_path, tmp_path):
    """Requests of one batch keep their own adapter, its keys and values their own blocks."""
    from zse_b200.lora.weights import random_adapter_file
    eng = engine(model_path, max_batch_seqs=4)
    for name, seed in (("a", 1), ("b", 2)):
        random_adapter_file(str(tmp_path / name), eng.model_config, rank=4, alpha=8.0, seed=seed, std=0.2)
        eng.lora_manager.load_adapter(name, str(tmp_path / name))
    prompt = prompts(1, 40, 40, seed=9)[0]

    def gen(*adapters):
        ids = [eng.add_request_tokens(prompt, max_tokens=8, temperature=0.0, stop_tokens=[], lora_id=x) for x in adapters]
        eng.run_until_done()
        return [eng.get_result(i).output_tokens for i in ids]
    alone = [gen(x)[0] for x in ("a", None, "b")]
    assert gen("a", None, "b") == alone and len({tuple(x) for x in alone}) > 1
    eng.destroy()


@pytest.mark.timeout(600)
def test_heads_over_two_ranks(tmp_path):
    from zse_b200.parallel.tp_engine import TPEngine
    path = str(tmp_path / "m.zse")
    synth.write_random_model(path, synth.shape_config("tiny-aligned"), seed=0)
    cfg = EngineConfig(device="cpu", kv_blocks=64, max_batch_seqs=4, max_batch_tokens=64, max_seq_len=256, kv_dtype="int8")
    ps = prompts(3, 12, 80, seed=5)
    want = run(ZStreamerEngine(path, config=cfg), ps, 6)
    e = TPEngine(path, tp_size=2, config=cfg, start_timeout_s=180)
    try:
        ids = [e.add_request_tokens(x, max_tokens=6, temperature=0.0, stop_tokens=[]) for x in ps]
        e.run_until_done(120)
        assert e.healthy and [e.get_result(i).output_tokens for i in ids] == want
    finally:
        e.stop()


def test_memory_is_counted(model_path):
    a, b = engine(model_path, kv_blocks=40), ZStreamerEngine(model_path, config=EngineConfig(device="cpu", kv_blocks=40, max_seq_len=256))
    hd = a.model_config.head_dim
    assert isinstance(a.kv_cache.slab, QuantKV) and a.kv_cache.slab.head_dim == hd
    assert a.kv_cache.stats().block_bytes * 2 * hd == b.kv_cache.stats().block_bytes * (hd + 4)
    assert row_bytes(hd, torch.uint8) == hd + 4 and row_bytes(hd, torch.float16) == 2 * hd
    a.destroy(); b.destroy()
    p = BlockPool.from_budget(10 * 16 * 2 * 3 * 2 * (64 + 4) + 5, 16, 3, 2, 64, device="cpu", dtype=torch.uint8)
    assert p.num_blocks == 10 and p.slab.shape == (3, 10, 2, 2, 16, 64) and p.total_bytes == 10 * 16 * 2 * 3 * 2 * 68
    blk = p.alloc()
    assert p.gpu_ptr_for_kv(blk, 2, True) == p.slab.data[2, blk.block_id, 1].data_ptr()


def test_what_is_refused(tmp_path, model_path):
    with pytest.raises(ValueError, match="int4"):
        engine(model_path, kv_dtype="int4")
    path = str(tmp_path / "gemma.zse")
    synth.write_random_model(path, synth.shape_config("tiny-gemma2"), seed=1)
    with pytest.raises(ValueError, match="gemma2"):
        engine(path)
    assert "nimelorn" in refuses(synth.shape_config("tiny-nimelorn")) and refuses(synth.shape_config("tiny")) is None
    assert "17 query heads" in refuses(synth.shape_config("tiny", num_heads=17, num_kv_heads=1))
    assert "24 rotated" in refuses(synth.shape_config("tiny", partial_rotary_factor=0.375))
    path = str(tmp_path / "hd80.zse")
    synth.write_random_model(path, synth.shape_config("tiny", head_dim=80), seed=1)
    with pytest.raises(ValueError, match="head dimension 80"):
        engine(path)
    plain = engine(model_path, kv_dtype="float16")
    assert not isinstance(plain.kv_cache.slab, QuantKV)
    plain.destroy()


def test_the_command_line_and_the_environment_reach_it(monkeypatch):
    from zse_b200 import cli
    seen = {}

    class Server:
        def __init__(self, *args, **kwargs):
            seen.update(kwargs)
            raise SystemExit

    monkeypatch.setattr("zse_b200.server.app.ZSEServer", Server)
    monkeypatch.setattr("os.path.exists", lambda p: True)
    with pytest.raises(SystemExit):
        cli.main(["serve", "m.zse", "--kv-dtype", "int8", "--cpu", "-q", "--admin-key", "k"])
    assert seen["engine_config"].kv_dtype == "int8"
    monkeypatch.setenv("ZSE_KV_DTYPE", "int8")
    assert EngineConfig.from_env().kv_dtype == "int8"
