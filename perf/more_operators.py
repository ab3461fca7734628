"""Operators of 8-bit floating point layers: what is measured.

Four operators of one path, a transformer's feed-forward and its projections with weights and activations in e4m3.  ``norm`` adds
split-K planes and a 16-bit row to the fp32 residual and writes its root-mean-square norm in 8 bits; ``quant`` writes rows, or
the gated product of their halves, in 8 bits; ``linear`` is the matrix product of such rows with an 8-bit weight; ``up`` is the
product with the gate and up weights whose gated activation leaves in 8 bits again.

Rows in 8 bits: ``data`` e4m3 [rows, columns] and ``scale`` fp32 [blocks of 128 columns, rows]; an element stands for data * scale
with scale = max|x| / 448 over its block.  Weights: ``data`` e4m3 [N, K] and ``scale`` fp32 [blocks of 128 rows, blocks of 128
columns]; gate and up weights are stacked, and each of the two begins its own blocks.  ``own`` is set by whoever measures: False
computes the operators from elementary torch operations, True calls the framework's.
"""
import functools
import math

import torch

own = False

BLOCK, TOP = 128, 448.0
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------------------------------
def _norm(name, M, H, planes, add=1, keep=0, dtype="f16"):
    """``planes``: fp32 planes that join the residual; ``add``: a 16-bit row joins it; ``keep``: the norm is wanted in 16 bits too."""
    return _case(name, "norm", M=M, H=H, planes=planes, add=add, keep=keep, dtype=dtype)


def _quant(name, M, C, act="none", dtype="f16"):
    """``act``: none, or which activation gates the second half of the rows with the first ("silu", "gelu")."""
    return _case(name, "quant", M=M, C=C, act=act, dtype=dtype)


def _linear(name, M, N, K, bias=0, dtype="f16"):
    return _case(name, "linear", M=M, N=N, K=K, bias=bias, dtype=dtype)


def _up(name, M, ff, K, act="silu"):
    return _case(name, "up", M=M, ff=ff, K=K, act=act)


def _case(name, kind, **c):
    return dict(c, kind=kind, name=name) if name else dict(c, kind=kind)


def listed():
    return [
        # one sequence decodes: the norm between two layers, all launch and latency
        _norm("norm_one_token", 1, 3584, planes=1, add=0),
        # a decode step of a full batch whose projection left split-K planes
        _norm("norm_step_64", 64, 5120, planes=4, add=0),
        # a pass of prompt chunks, the projection's output in 16 bits; adapters want the norm in 16 bits too
        _norm("norm_prompts", 8192, 5120, planes=0, keep=1, dtype="bf16"),
        # a decode step's attention output before the output projection
        _quant("quant_step_33", 33, 8192, dtype="bf16"),
        # gate and up products of a prompt chunk, changed by adapters before the activation
        _quant("quant_gated_prompts", 4099, 27648, act="silu"),
        # one sequence decodes: query, key and value projections with their bias, bound by the weights' bytes
        _linear("linear_one_token", 1, 4608, 3584, bias=1),
        # a decode step of a full batch, the deep projection back to the residual
        _linear("linear_step_64", 64, 5120, 13824, dtype="f32"),
        # one chunk of a prompt, a ragged number of tokens
        _linear("linear_chunk_777", 777, 10240, 8192, dtype="bf16"),
        # prompts of several sequences in one pass
        _linear("linear_prompts", 8192, 5120, 13824),
        # a decode step of a few sequences through the wide half of the feed-forward
        _up("up_step_5", 5, 18944, 3584),
        # speculative verification: four drafted tokens and one more of 32 sequences
        _up("up_verify_160", 160, 13824, 5120),
        # the largest work of the path: a long prompt through the wide half of the feed-forward
        _up("up_prompts", 4096, 13824, 5120),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["norm", "quant", "linear", "linear", "up", "up"])
    M = _log(rng, 1, 8192)
    wide = lambda most: 16 * _log(rng, 4, most // 16)          # columns: a multiple of 16, often no multiple of 128
    if rng.random() < 0.5:
        wide = lambda most: 128 * _log(rng, 2, most // 128)    # noqa: E731
    if kind == "norm":
        H = wide(16384)
        planes = rng.choice([0, 0, 1, 1, 2, 3, 8]) if M <= 256 else rng.choice([0, 1])
        return _norm("", min(M, max(1, (1 << 26) // (H * (planes + 2)))), H, planes, add=int(planes == 0 or rng.random() < 0.3),
                     keep=int(rng.random() < 0.3), dtype=rng.choice(["f16", "bf16"]))
    if kind == "quant":
        C = wide(29568)
        return _quant("", min(M, max(1, (1 << 27) // C)), C * rng.choice([1, 2]) // 32 * 32 or 32,
                      act=rng.choice(["none", "silu", "silu", "gelu"]), dtype=rng.choice(["f16", "bf16", "f32"]))
    K = wide(16384)
    N = rng.choice([rng.randint(1, 300), _log(rng, 128, 28000), 128 * _log(rng, 2, 220)])
    N = min(N, (1 << 27) // K)
    M = min(M, max(1, (1 << 38) // (N * K)))
    if kind == "linear":
        return _linear("", M, N, K, bias=int(rng.random() < 0.3), dtype=rng.choice(["f16", "bf16", "f32"]))
    return _up("", M, max(16, N // 2 // 16 * 16), K, act=rng.choice(["silu", "silu", "gelu"]))


def _blocks(n):
    return -(-n // BLOCK)


def _bytes8(M, C):
    return M * (C + 4 * _blocks(C))


def work(case):
    c, kind, M = case, case["kind"], case["M"]
    if kind == "norm":
        H, item = c["H"], 2
        moved = 4 * (1 + c["planes"]) + item * c["add"] + item * c["keep"] + (4 if c["planes"] or c["add"] else 0)
        return {"bytes": M * H * moved + item * H + _bytes8(M, H), "flops": M * H * (c["planes"] + c["add"] + 6)}
    item = TYPES[c["dtype"]].itemsize if "dtype" in c else 1
    if kind == "quant":
        C = c["C"] if c["act"] == "none" else c["C"] // 2
        return {"bytes": M * c["C"] * item + _bytes8(M, C), "flops": M * C * (3 if c["act"] == "none" else 9)}
    if kind == "linear":
        N, K = c["N"], c["K"]
        return {"bytes": _bytes8(M, K) + N * K + 4 * _blocks(N) * _blocks(K) + M * N * item + N * item * c["bias"], "flops": 2 * M * N * K}
    ff, K = c["ff"], c["K"]
    return {"bytes": _bytes8(M, K) + 2 * ff * K + 8 * _blocks(ff) * _blocks(K) + _bytes8(M, ff), "flops": 4 * M * ff * K}


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _rows8(rand, M, C, dev):
    return {"data": torch.empty(M, C, dtype=torch.float8_e4m3fn, device=dev), "scale": torch.empty(_blocks(C), M, device=dev)} if rand is None else {
        "data": (rand(M, C) * (TOP / 2.7)).clamp_(-TOP, TOP).to(torch.float8_e4m3fn),      # a block's largest is near 448
        "scale": (rand(_blocks(C), M) * 0.4 - 5).exp_()}


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device=dev, generator=g)       # noqa: E731
    M, s = c["M"], {"case": c}
    if c["kind"] == "norm":
        H, t = c["H"], TYPES[c["dtype"]]
        hot = torch.where(rand(H).abs() > 2.8, 20.0, 1.0)                    # a few channels of a residual stream are far larger
        s["residual"] = rand(M, H) * hot
        s["planes"] = rand(c["planes"], M, H).mul_(0.3) if c["planes"] else None
        s["add"] = (rand(M, H) * 0.5).to(t) if c["add"] else None
        s["weight"] = (1 + 0.2 * rand(H)).to(t)
        s["normed"] = torch.empty(M, H, dtype=t, device=dev) if c["keep"] else None
        s["out"] = _rows8(None, M, H, dev)
    elif c["kind"] == "quant":
        C = c["C"] if c["act"] == "none" else c["C"] // 2
        s["x"] = (rand(M, c["C"]) * 1.5).to(TYPES[c["dtype"]])
        s["out"] = _rows8(None, M, C, dev)
    else:
        K, parts = c["K"], 1 if c["kind"] == "linear" else 2
        N = c["N"] if parts == 1 else c["ff"]
        s["x"] = _rows8(rand, M, K, dev)
        s["w"] = (rand(parts * N, K) * (TOP / 4)).clamp_(-TOP, TOP).to(torch.float8_e4m3fn)
        s["w_scale"] = (rand(parts * _blocks(N), _blocks(K)) * 0.3).exp_() * (4 / TOP * (1.0 if parts == 1 else 4.0) / math.sqrt(K))
        if parts == 1:
            t = TYPES[c["dtype"]]
            s["bias"] = rand(N).to(t) if c["bias"] else None
            s["out"] = torch.empty(M, N, dtype=t, device=dev)
        else:
            s["out"] = _rows8(None, M, N, dev)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _put8(y, out):
    """Rows y in fp32 to 8 bits: scale = max|y| / 448 of each block of 128 columns, data = y * (448 / max|y|)."""
    M, C = y.shape
    y = torch.nn.functional.pad(y, (0, _blocks(C) * BLOCK - C)).view(M, -1, BLOCK)
    top = y.abs().amax(-1)
    there = top > 1e-30
    steps = torch.where(there, TOP / top, torch.zeros_like(top))
    out["data"].copy_((y * steps[..., None]).view(M, -1)[:, :C])
    out["scale"].copy_(torch.where(there, top / TOP, torch.zeros_like(top)).t())


def _rounded(y, t):
    return (y.clamp(-65504, 65504) if t is torch.float16 else y).to(t)


def _gated(act, g, u):
    z = g if act == "silu" else 1.5957691216057308 * (g + 0.044715 * g * g * g)      # gelu's tanh form is g sigmoid(2 z)
    return g / (1 + torch.exp(-z)) * u


def _norm_plain(s):
    r = s["residual"]
    if s["planes"] is not None or s["add"] is not None:
        total = r.double()
        if s["planes"] is not None:
            total = total + s["planes"].double().sum(0)
        if s["add"] is not None:
            total = total + s["add"].double()
        r.copy_(total)
    inv = torch.rsqrt(r.double().square().mean(-1, keepdim=True) + 1e-6).float()
    y = r * inv * s["weight"].float()
    _put8(y, s["out"])
    if s["normed"] is not None:
        s["normed"].copy_(_rounded(y, s["normed"].dtype))


def _values(x, scale):
    """Rows in 8 bits as fp32."""
    return x.float() * scale.t().repeat_interleave(BLOCK, 1)[:, : x.shape[1]]


def _weight(w, scale):
    return w.float() * scale.repeat_interleave(BLOCK, 0)[: w.shape[0]].repeat_interleave(BLOCK, 1)[:, : w.shape[1]]


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "norm":
        _norm_plain(s)
    elif c["kind"] == "quant":
        x = s["x"].float()
        half = c["C"] // 2
        _put8(x if c["act"] == "none" else _gated(c["act"], x[:, :half], x[:, half:]), s["out"])
    elif c["kind"] == "linear":
        y = _values(**_named(s["x"])) @ _weight(s["w"], s["w_scale"]).t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        s["out"].copy_(_rounded(y, s["out"].dtype))
    else:
        x, ff, nb = _values(**_named(s["x"])), c["ff"], _blocks(c["ff"])
        gate = x @ _weight(s["w"][:ff], s["w_scale"][:nb]).t()
        up = x @ _weight(s["w"][ff:], s["w_scale"][nb:]).t()
        _put8(_gated(c["act"], gate, up), s["out"])


def _named(rows):
    return {"x": rows["data"], "scale": rows["scale"]}


# ---- the framework's operators ------------------------------------------------------------------------------------------------
@functools.lru_cache(None)
def _framework():
    from zse_b200.ops import fp8
    from zse_b200.ops.backend import make_ops
    return make_ops("cuda"), fp8


def _run_own(s):
    ops, fp8 = _framework()
    c, M = s["case"], s["case"]["M"]
    out = s["out"] if c["kind"] == "linear" else fp8.Fp8Rows(s["out"]["data"], s["out"]["scale"])
    if c["kind"] == "norm":
        ops.add_rmsnorm_fp8(s["residual"], s["planes"], c["planes"], s["add"], s["weight"], out, M, 1e-6, normed=s["normed"])
    elif c["kind"] == "quant":
        if c["act"] == "none":
            ops.quant_fp8(s["x"], M, out)
        else:
            ops.swiglu_fp8(s["x"], M, out, gelu=c["act"] == "gelu")
    else:
        x = fp8.Fp8Rows(s["x"]["data"], s["x"]["scale"])
        w = fp8.Fp8Weight(s["w"], s["w_scale"], bias=s.get("bias"), glu=c["kind"] == "up")
        if c["kind"] == "linear":
            ops.linear_fp8(w, x, M, out)
        else:
            ops.linear_swiglu_fp8(w, x, M, out, gelu=c["act"] == "gelu")


def run(state):
    if own:
        _run_own(state)
    else:
        _run_plain(state)
    if state["case"]["kind"] == "linear":
        return state["out"]
    out = dict(state["out"])
    if state["case"]["kind"] == "norm":
        out["residual"] = state["residual"]
        if state["normed"] is not None:
            out["normed"] = state["normed"]
    return out


# ---- the same in 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)

    def e4m3(v):
        """The nearest number with three bits behind the leading one, of 2^-6 and more, or multiple of 2^-9 below, in 64 bits."""
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
        return torch.round(v / step) * step

    def blockwise(y):
        data, scale = torch.empty_like(y), torch.empty(_blocks(y.shape[1]), y.shape[0], dtype=y.dtype, device=y.device)
        for b in range(scale.shape[0]):
            part = y[:, b * BLOCK: (b + 1) * BLOCK]
            scale[b] = part.abs().max(1).values / TOP
            data[:, b * BLOCK: (b + 1) * BLOCK] = e4m3(torch.nan_to_num(part / scale[b][:, None], 0.0))
        return {"data": data, "scale": scale}

    def product(x, w, w_scale):
        """Sum over blocks of 128 columns of (row's scale x weight block's scale) x product of the 8-bit numbers."""
        M, K = x["data"].shape
        total = torch.zeros(M, w.shape[0], dtype=torch.float64, device=w.device)
        of_row = torch.arange(w.shape[0], device=w.device) // BLOCK
        for b in range(_blocks(K)):
            at = slice(b * BLOCK, (b + 1) * BLOCK)
            part = x["data"][:, at].to(torch.float64) @ w[:, at].to(torch.float64).t()
            total.addcmul_(part.mul_(x["scale"][b].double()[:, None]), w_scale[of_row, b].double()[None])
        return total

    def activation(g):
        if c["act"] == "silu":
            return g * torch.sigmoid(g)
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))

    if c["kind"] == "norm":
        r = s["residual"].to(torch.float64)
        for p in s["planes"] if c["planes"] else []:
            r += p
        if c["add"]:
            r += s["add"]
        y = r / torch.linalg.vector_norm(r, dim=1, keepdim=True).square().div(c["H"]).add(1e-6).sqrt() * s["weight"].to(torch.float64)
        out = dict(blockwise(y), residual=r)
        return dict(out, normed=y) if c["keep"] else out
    if c["kind"] == "quant":
        x = s["x"].to(torch.float64)
        return blockwise(x if c["act"] == "none" else activation(x[:, : c["C"] // 2]) * x[:, c["C"] // 2:])
    if c["kind"] == "linear":
        y = product(s["x"], s["w"], s["w_scale"])
        return y if s["bias"] is None else y + s["bias"].to(torch.float64)
    ff, nb = c["ff"], _blocks(c["ff"])
    return blockwise(activation(product(s["x"], s["w"][:ff], s["w_scale"][:nb])) * product(s["x"], s["w"][ff:], s["w_scale"][nb:]))
