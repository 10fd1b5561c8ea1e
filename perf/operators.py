"""Cases of the 4-bit block operators: microscaled quantisation and product, the norms around a
transformer block, and attention over packed sequences.

Each case names the operator it measures ("op") and its sizes and types:

  quantize   a matrix to microscaled 4-bit values (MXFP4: E2M1 codes, one power-of-two scale for 32
             values) and back
  product    act(A B^T + bias) of two matrices held in that form
  norm       x' = resid_scale x + gate * post(y), h = pre(x'): the norms after one block and before
             the next, with the gate and the residual between them
  mlp_in     the same with h in microscaled 4-bit form, and the product that reads it
  attention  softmax(scale Q K^T) V over packed sequences of different lengths, heads in groups that
             share keys and values, causal or not

With `own` false the plain form in elementary torch operations runs; with `own` true the calls of
librfdetr.so.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGUF = {"f32": 0, "f16": 1, "bf16": 30}  # the type ids that the library's entry points take
ACTS = {"none": 0, "gelu": 1, "relu": 2, "silu": 3}
NORMS = {"none": 0, "layer": 1, "rms": 2}
EPS = 1e-5


def listed():
    return [
        # one token's activations on their way into a 4-bit product: launch latency
        {"name": "quantize_token", "op": "quantize", "rows": 1, "k": 4096, "type": "bf16", "pad": 0},
        # the MLP's hidden layer of the Base model, 32 images of 1616 tokens, f16 like the engine's
        {"name": "quantize_batch", "op": "quantize", "rows": 51712, "k": 1536, "type": "f16", "pad": 0},
        # one token through a square projection: every weight read once
        {"name": "product_token", "op": "product", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "act": "none",
         "bias": False},
        # a few sequences' tokens through a gate projection, rows odd in number
        {"name": "product_few", "op": "product", "m": 13, "n": 11008, "k": 4096, "type": "bf16", "act": "silu",
         "bias": False},
        # the Base model's qkv linear on one image: short K, ragged rows
        {"name": "product_image", "op": "product", "m": 1616, "n": 1152, "k": 384, "type": "f16", "act": "none",
         "bias": True},
        # a long prompt through a wide layer: the tensor cores' own limit
        {"name": "product_large", "op": "product", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "act": "none",
         "bias": False},
        # one token between two blocks, both norms, 16-bit residual stream
        {"name": "norm_token", "op": "norm", "rows": 1, "dim": 4096, "type": "bf16", "resid": "bf16", "post": "rms",
         "pre": "rms", "gate": "none", "scale": 1.0},
        # the Base backbone between attention and MLP: layer scale, f32 residual stream, LayerNorm
        {"name": "norm_batch", "op": "norm", "rows": 51712, "dim": 384, "type": "f16", "resid": "f32", "post": "none",
         "pre": "layer", "gate": "channel", "scale": 1.0},
        # norms, gate and residual of a prompt, then the MLP's first product in 4 bits
        {"name": "mlp_in_prompt", "op": "mlp_in", "rows": 4097, "dim": 2048, "n": 8192, "type": "bf16",
         "resid": "bf16", "post": "rms", "pre": "rms", "gate": "group", "scale": 0.75, "act": "gelu"},
        # images of mixed sizes in one batch: bidirectional, short, every length different
        {"name": "attention_images", "op": "attention", "seqs": 24, "longest": 577, "heads": 6, "kv_heads": 6,
         "dim": 64, "causal": False, "type": "f16"},
        # prompts of very different lengths, grouped heads
        {"name": "attention_prompts", "op": "attention", "seqs": 7, "longest": 2049, "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True, "type": "bf16"},
        # one long document
        {"name": "attention_long", "op": "attention", "seqs": 1, "longest": 8192, "heads": 16, "kv_heads": 2,
         "dim": 128, "causal": True, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "norm", "mlp_in", "attention", "attention"])
    if op == "quantize":
        k = _log(rng, 1, 16384)
        return {"op": op, "rows": _log(rng, 1, min(65536, 79_000_000 // k)), "k": k,
                "type": rng.choice(["f32", "f16", "bf16"]), "pad": rng.choice([0, 0, 3, 8])}
    if op == "product":
        n, k = _log(rng, 16, 16384), _log(rng, 32, 16384)
        return {"op": op, "m": _log(rng, 1, min(16384, 8192 ** 3 // (n * k))), "n": n, "k": k,
                "type": rng.choice(["f16", "bf16"]), "act": rng.choice(["none", "gelu", "relu", "silu"]),
                "bias": rng.random() < 0.5}
    around = {"type": rng.choice(["f16", "bf16"]), "post": rng.choice(["none", "layer", "rms"]),
              "pre": rng.choice(["layer", "rms"]), "gate": rng.choice(["none", "channel", "group"]),
              "scale": rng.choice([1.0, 0.75])}
    around["resid"] = rng.choice([around["type"], "f32"])
    if op == "norm":
        dim = _log(rng, 32, 16384)
        around["type"] = rng.choice([around["type"], around["type"], "f32"])
        around["resid"] = "f32" if around["type"] == "f32" else around["resid"]
        return {"op": op, "rows": _log(rng, 1, min(65536, 19_800_000 // dim)), "dim": dim, **around}
    if op == "mlp_in":
        dim, n = _log(rng, 32, 8192), _log(rng, 64, 16384)
        return {"op": op, "rows": _log(rng, 1, min(8192, 8192 ** 3 // (dim * n))), "dim": dim, "n": n, **around,
                "act": rng.choice(["none", "gelu", "silu"])}
    kv, group, seqs = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8]), _log(rng, 1, 64)
    most = int(math.sqrt(8192 ** 2 * 16 / (kv * group * seqs)))  # the plain form's scores are padded
    return {"op": op, "seqs": seqs, "longest": _log(rng, 1, min(8192, most)), "heads": kv * group, "kv_heads": kv,
            "dim": rng.choice([64, 128]), "causal": rng.random() < 0.6, "type": rng.choice(["f16", "bf16"])}


def _lengths(c):
    """The sequences' lengths: the first the longest, the others anything down to none at all."""
    rng = random.Random("%d %d %d" % (c["seqs"], c["longest"], c["heads"]))
    return [c["longest"]] + [rng.choice([rng.randint(0, c["longest"]), _log(rng, 1, c["longest"])])
                             for _ in range(c["seqs"] - 1)]


def _size(t):
    return 4 if t == "f32" else 2


def work(c):
    """Every input read once, every output written once; 4-bit operands take 17 bytes for 32 values."""
    def mx(r, k):
        return r * -(-k // 32) * 17

    if c["op"] == "quantize":
        n = c["rows"] * c["k"]
        return {"bytes": 2 * n * _size(c["type"]) + 2 * mx(c["rows"], c["k"]), "flops": 4 * n}
    if c["op"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": mx(m, k) + mx(n, k) + 2 * m * n + (4 * n if c["bias"] else 0), "flops": 2 * m * n * k}
    if c["op"] in ("norm", "mlp_in"):
        r, d = c["rows"], c["dim"]
        small = 4 * d * ((c["post"] != "none") + (c["post"] == "layer") + 1 + (c["pre"] == "layer"))
        small += 4 * d * {"none": 0, "channel": 1, "group": -(-r // _period(c))}[c["gate"]]
        b = r * d * (_size(c["type"]) + 2 * _size(c["resid"])) + small
        if c["op"] == "norm":
            return {"bytes": b + r * d * _size(c["type"]), "flops": 12 * r * d}
        # the 4-bit rows between the two calls are written and read
        return {"bytes": b + 2 * mx(r, d) + mx(c["n"], d) + 2 * r * c["n"] + 4 * c["n"],
                "flops": 2 * r * d * c["n"] + 12 * r * d}
    lens, h, kv, d = _lengths(c), c["heads"], c["kv_heads"], c["dim"]
    pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in lens)
    return {"bytes": sum(lens) * d * 2 * (2 * h + 2 * kv), "flops": 4 * pairs * h * d}


def _period(c):
    """Rows that share a row of the gate: a sequence's or an image's."""
    return max(1, -(-c["rows"] // 5))


# ---- microscaled form -------------------------------------------------------


def _blocks(x):
    """x [rows][k] in 32 bits as [rows][blocks][32], zeros behind the last value."""
    rows, k = x.shape
    return torch.nn.functional.pad(x, (0, -k % 32)).view(rows, -1, 32)


def _exponents(b):
    """The biased exponent of each block's scale: that of its largest value, less E2M1's own 2."""
    amax = b.abs().amax(-1).contiguous()
    return ((amax.view(torch.int32) >> 23) - 2).clamp_min(0)


def _pow2(e):
    """2^(e - 127) in 32 bits."""
    return (e.to(torch.int32) << 23).view(torch.float32)


def _round_e2m1(r):
    """To the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code), the sign kept."""
    a = r.abs()
    step = 0.5 + 0.5 * (a >= 2) + 1.0 * (a >= 4)
    return torch.copysign((torch.round(a / step) * step).clamp_max(6.0), r)


def _mx_values(x):
    """What x [rows][k] (32 bits) stands for once it is held in microscaled 4-bit form."""
    b = _blocks(x)
    e = _exponents(b)[..., None]
    return (_round_e2m1(b * _pow2(254 - e)) * _pow2(e)).view(x.shape[0], -1)[:, :x.shape[1]]


def _mx_pack(x):
    """(codes uint8 [rows][blocks * 16], two to a byte, the lower first; exponents uint8 [rows][blocks])."""
    b = _blocks(x)
    e = _exponents(b)
    r = b * _pow2(254 - e)[..., None]
    a = r.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    code = (code + 8 * torch.signbit(r)).to(torch.uint8).view(x.shape[0], -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), e.to(torch.uint8)


def _mx_tiles(e):
    """The exponents in the order of the library's scale operand: tiles of 128 rows x 4 blocks, in a
    tile the rows 32 apart side by side."""
    rows, blocks = e.shape
    p = torch.nn.functional.pad(e, (0, -blocks % 4, 0, -rows % 128))
    t = p.view(p.shape[0] // 128, 4, 32, p.shape[1] // 4, 4)
    return t.permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _mx_unpack(codes, e):
    """The values in 32 bits, [rows][blocks * 32]."""
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1).view(codes.shape[0], -1, 32)
    return (v * _pow2(e)[..., None]).view(codes.shape[0], -1)


# ---- inputs -----------------------------------------------------------------


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _activations(g, rows, k):
    """Activations: a few channels much larger than the others, as transformers have them."""
    channel = torch.exp(0.7 * _randn(g, k))
    return _randn(g, rows, k) * channel


def _weights(g, n, k):
    return _randn(g, n, k) * (torch.exp(0.3 * _randn(g, n, 1)) / math.sqrt(k))


def _out(rows, cols, t):
    return torch.zeros(rows, cols, dtype=t, device="cuda")


def prepare(c, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "quantize":
        rows, k, t = c["rows"], c["k"], TYPES[c["type"]]
        s["x"] = torch.zeros(rows, k + c["pad"], dtype=t, device="cuda")[:, :k]
        s["x"].copy_(_activations(g, rows, k))
        s["codes"] = _out(rows, -(-k // 32) * 16, torch.uint8)
        s["scales"] = _out(1, -(-rows // 128) * -(-k // 128) * 512, torch.uint8)
        s["back"] = _out(rows, k, t)
    elif c["op"] == "product":
        for name, rows in (("a", c["m"]), ("b", c["n"])):
            x = _activations(g, rows, c["k"]) if name == "a" else _weights(g, rows, c["k"])
            s[name], s[name + "_exp"] = _mx_pack(x)
            s[name + "_scales"] = _mx_tiles(s[name + "_exp"])
        s["bias"] = _randn(g, c["n"]) * 0.1 if c["bias"] else None
        s["out"] = _out(c["m"], c["n"], TYPES[c["type"]])
    elif c["op"] in ("norm", "mlp_in"):
        rows, dim, t, tr = c["rows"], c["dim"], TYPES[c["type"]], TYPES[c["resid"]]
        s["y"] = _activations(g, rows, dim).to(t)
        s["x"] = (_randn(g, rows, dim) * 2 + 0.3).to(tr)
        for name, kind in (("post", c["post"]), ("pre", c["pre"])):
            s[name + "_w"] = 1 + 0.2 * _randn(g, dim) if kind != "none" else None
            s[name + "_b"] = 0.1 * _randn(g, dim) if kind == "layer" else None
        gates = {"none": 0, "channel": 1, "group": -(-rows // _period(c))}[c["gate"]]
        s["gate"] = 0.5 * _randn(g, gates, dim) if gates else None
        s["x_out"] = _out(rows, dim, tr)
        if c["op"] == "norm":
            s["h"] = _out(rows, dim, t)
        else:
            s["codes"] = _out(rows, -(-dim // 32) * 16, torch.uint8)
            s["scales"] = _out(1, -(-rows // 128) * -(-dim // 128) * 512, torch.uint8)
            s["w"], s["w_exp"] = _mx_pack(_weights(g, c["n"], dim))
            s["w_scales"] = _mx_tiles(s["w_exp"])
            s["bias"] = _randn(g, c["n"]) * 0.1
            s["out"] = _out(rows, c["n"], t)
    else:
        lens, h, kv, d = _lengths(c), c["heads"], c["kv_heads"], c["dim"]
        total = sum(lens)
        s["qkv"] = _randn(g, total, (h + 2 * kv) * d).to(TYPES[c["type"]])
        s["cu"] = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device="cuda")
        s["longest"] = max(lens)
        s["out"] = _out(total, h * d, TYPES[c["type"]])
    return s


# ---- plain forms ------------------------------------------------------------


def _act(v, act):
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "relu":
        return v.clamp_min(0)
    return v / (1 + torch.exp(-v)) if act == "silu" else v


def _norm(v, kind, w, b):
    if kind == "none":
        return v
    if kind == "rms":
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * w
    v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * w + b


def _plain_norms(s):
    c = s["case"]
    branch = _norm(s["y"].float(), c["post"], s["post_w"], s["post_b"])
    if c["gate"] == "channel":
        branch = branch * s["gate"]
    elif c["gate"] == "group":
        branch = branch * s["gate"].repeat_interleave(_period(c), 0)[:c["rows"]]
    x = c["scale"] * s["x"].float() + branch
    return x, _norm(x, c["pre"], s["pre_w"], s["pre_b"])


def _plain_attention(s):
    c = s["case"]
    h, kv, d, n = c["heads"], c["kv_heads"], c["dim"], s["longest"]
    cu, qkv = s["cu"].long(), s["qkv"]
    start, lens = cu[:-1], cu[1:] - cu[:-1]
    at = torch.arange(n, device="cuda")
    here = at < lens[:, None]                                             # [seqs][n]
    rows = torch.where(here, start[:, None] + at, 0)
    x = qkv[rows].float() * here[..., None]                               # [seqs][n][...]
    q = x[..., :h * d].view(len(lens), n, kv, h // kv, d).permute(0, 2, 3, 1, 4)
    k = x[..., h * d:(h + kv) * d].view(len(lens), n, kv, 1, d).permute(0, 2, 3, 4, 1)
    v = x[..., (h + kv) * d:].view(len(lens), n, kv, 1, d).permute(0, 2, 3, 1, 4)
    p = torch.matmul(q, k)
    keep = here[:, None, :]
    if c["causal"]:
        keep = keep & (at[None, :, None] >= at[None, None, :])
    p.mul_(d ** -0.5).masked_fill_(~keep[:, None, None], -torch.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    token = torch.arange(qkv.shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:], token, right=True)
    return o.permute(0, 3, 1, 2, 4).reshape(len(lens), n, h * d)[seq, token - start[seq]].to(qkv.dtype)


def _plain(s):
    c = s["case"]
    if c["op"] == "quantize":
        return _mx_values(s["x"].float()).to(TYPES[c["type"]])
    if c["op"] == "product":
        v = _mx_unpack(s["a"], s["a_exp"]) @ _mx_unpack(s["b"], s["b_exp"]).T
        return _act(v if s["bias"] is None else v + s["bias"], c["act"]).to(TYPES[c["type"]])
    if c["op"] == "attention":
        return _plain_attention(s)
    x, h = _plain_norms(s)
    if c["op"] == "norm":
        return {"x": x.to(TYPES[c["resid"]]), "h": h.to(TYPES[c["type"]])}
    v = _mx_values(h) @ _mx_unpack(s["w"], s["w_exp"])[:, :c["dim"]].T + s["bias"]
    return {"x": x.to(TYPES[c["resid"]]), "out": _act(v, c["act"]).to(TYPES[c["type"]])}


# ---- the library's calls ----------------------------------------------------


def _library():
    import os
    import sys
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rf-detr.cpp_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from rfdetr_b200 import lib
    return lib, lib.lib()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _done(status):
    if status != 0:
        raise RuntimeError("the library returned %d" % status)


def _own_norms(s, lib, L, stream):
    c = s["case"]
    a = lib.BlockNorm(
        y=_ptr(s["y"]), resid=_ptr(s["x"]), post_w=_ptr(s["post_w"]), post_b=_ptr(s["post_b"]), gate=_ptr(s["gate"]),
        pre_w=_ptr(s["pre_w"]), pre_b=_ptr(s["pre_b"]), out_resid=_ptr(s["x_out"]), out=_ptr(s.get("h")),
        mx_codes=_ptr(s.get("codes")), mx_scales=_ptr(s.get("scales")),
        rows=c["rows"], dim=c["dim"], type=GGUF[c["type"]], resid_type=GGUF[c["resid"]], post=NORMS[c["post"]],
        pre=NORMS[c["pre"]], ldy=c["dim"], ld_resid=c["dim"], ld_out_resid=c["dim"], ld_out=c["dim"],
        ld_mx=s["codes"].shape[1] if "codes" in s else 0, ld_gate=c["dim"],
        gate_period=_period(c) if c["gate"] == "group" else 0, resid_scale=c["scale"], post_eps=EPS, pre_eps=EPS)
    _done(L.rfdetr_b200_op_block_norm(a, stream))


def _own(s):
    lib, L = _library()
    c = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "quantize":
        t, rows, k = GGUF[c["type"]], c["rows"], c["k"]
        codes, scales, ld = _ptr(s["codes"]), _ptr(s["scales"]), s["codes"].shape[1]
        _done(L.rfdetr_b200_op_mx_quantize(_ptr(s["x"]), t, s["x"].stride(0), rows, k, codes, ld, scales, stream))
        _done(L.rfdetr_b200_op_mx_dequantize(codes, ld, scales, rows, k, _ptr(s["back"]), t, k, stream))
        return s["back"]
    if c["op"] == "product":
        _done(L.rfdetr_b200_op_mx_gemm(
            _ptr(s["a"]), s["a"].shape[1], _ptr(s["a_scales"]), _ptr(s["b"]), s["b"].shape[1], _ptr(s["b_scales"]),
            c["m"], c["n"], c["k"], ACTS[c["act"]], _ptr(s["bias"]), _ptr(s["out"]), GGUF[c["type"]], c["n"], stream))
        return s["out"]
    if c["op"] == "attention":
        h, kv, d, q = c["heads"], c["kv_heads"], c["dim"], _ptr(s["qkv"])
        ld = (h + 2 * kv) * d
        _done(L.rfdetr_b200_op_attention_packed(
            q, q + 2 * h * d, q + 2 * (h + kv) * d, ld, ld, ld, _ptr(s["out"]), h * d, GGUF[c["type"]], _ptr(s["cu"]),
            c["seqs"], s["qkv"].shape[0], s["longest"], h, kv, d, int(c["causal"]), d ** -0.5, stream))
        return s["out"]
    _own_norms(s, lib, L, stream)
    if c["op"] == "norm":
        return {"x": s["x_out"], "h": s["h"]}
    _done(L.rfdetr_b200_op_mx_gemm(
        _ptr(s["codes"]), s["codes"].shape[1], _ptr(s["scales"]), _ptr(s["w"]), s["w"].shape[1], _ptr(s["w_scales"]),
        c["rows"], c["n"], c["dim"], ACTS[c["act"]], _ptr(s["bias"]), _ptr(s["out"]), GGUF[c["type"]], c["n"], stream))
    return {"x": s["x_out"], "out": s["out"]}


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits ---------------------------------------------


def _exact_mx(x):
    """Microscaled 4-bit values of x [rows][k] in 64 bits: each value to the nearer of its neighbours on
    the grid, at a tie to the one whose code is even."""
    rows, k = x.shape
    out = torch.zeros_like(x)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    for c0 in range(0, k, 32 * 64):  # some blocks of every row at a time
        part = torch.nn.functional.pad(x[:, c0:c0 + 2048], (0, -min(2048, k - c0) % 32)).view(rows, -1, 32)
        amax = part.abs().amax(-1, keepdim=True)
        _, e = torch.frexp(amax)  # amax = m 2^e, 0.5 <= m < 1
        scale = torch.ldexp(torch.ones_like(amax), e - 3)
        a = part.abs() / scale
        hi = torch.searchsorted(grid, a.contiguous()).clamp(1, 7)
        below, above = a - grid[hi - 1], grid[hi] - a
        up = (above < below) | ((above == below) & (hi % 2 == 0))
        value = torch.where(up, grid[hi], grid[hi - 1]) * scale * torch.sign(part)
        out[:, c0:c0 + 2048] = value.view(rows, -1)[:, :min(2048, k - c0)]
    return out


def _exact_decode(codes, e):
    """Sign, exponent and mantissa bits of every code, read one by one."""
    both = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1).to(torch.int64)
    sign, exponent, mantissa = both >> 3, (both >> 1) & 3, (both & 1).double()
    v = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * torch.pow(2.0, (exponent - 1).double()))
    v = torch.where(sign == 1, -v, v)
    return v * torch.pow(2.0, e.double() - 127).repeat_interleave(32, 1)


def _exact_act(v, act):
    if act == "gelu":
        return torch.special.ndtr(v) * v
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    return v * torch.special.expit(v) if act == "silu" else v


def _exact_norm(v, kind, w, b):
    if kind == "none":
        return v
    w = w.double()
    if kind == "rms":
        return v * w * torch.rsqrt(v.square().sum(1, keepdim=True) / v.shape[1] + EPS)
    var, mean = torch.var_mean(v, 1, unbiased=False, keepdim=True)
    return torch.addcmul(b.double(), (v - mean) * torch.rsqrt(var + EPS), w)


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "quantize":
        return _exact_mx(s["x"].double())
    if c["op"] == "product":
        v = torch.mm(_exact_decode(s["a"], s["a_exp"]), _exact_decode(s["b"], s["b_exp"]).t())
        return _exact_act(v + s["bias"].double() if c["bias"] else v, c["act"])
    if c["op"] == "attention":
        h, kv, d = c["heads"], c["kv_heads"], c["dim"]
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        at = 0
        for n in _lengths(c):
            x = s["qkv"][at:at + n].double()
            future = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1) if c["causal"] else None
            for i in range(h if n else 0):
                j = i // (h // kv)
                z = x[:, i * d:(i + 1) * d] @ x[:, (h + j) * d:(h + j + 1) * d].t() / math.sqrt(d)
                if c["causal"]:
                    z.masked_fill_(future, -torch.inf)
                z = torch.softmax(z, 1) @ x[:, (h + kv + j) * d:(h + kv + j + 1) * d]
                out[at:at + n, i * d:(i + 1) * d] = z
            at += n
        return out
    branch = _exact_norm(s["y"].double(), c["post"], s["post_w"], s["post_b"])
    if s["gate"] is not None:
        row = torch.arange(c["rows"], device="cuda")
        branch *= s["gate"].double()[row // _period(c) if c["gate"] == "group" else row * 0]
    x = s["x"].double() * c["scale"] + branch
    h = _exact_norm(x, c["pre"], s["pre_w"], s["pre_b"])
    if c["op"] == "norm":
        return {"x": x, "h": h}
    v = torch.mm(_exact_mx(h), _exact_decode(s["w"], s["w_exp"])[:, :c["dim"]].t()) + s["bias"].double()
    return {"x": x, "out": _exact_act(v, c["act"])}
