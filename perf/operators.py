"""Timing cases of the layer operators of nemo_ops.h that serve a transformer layer beside the fixed-shape encoder:
the residual RMSNorm with an 8-bit output, the rotary embedding, the 4-bit group-quantised matrix-vector product and
the attention with a sliding window and first tokens that stay visible.

A case is a dict of sizes and choices, `prepare` makes its inputs from a seed, `run` does one pass: the plain torch
form, or the library's entry points where `own` is true. `exact` is the same result in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn,
          "i8": torch.int8}
CODES = {"f16": 0, "bf16": 1, "f32": 2, "e4m3": 3, "i8": 4}  # NEMO_DTYPE_*
TOP = {"e4m3": 448.0, "i8": 127.0}  # largest code of the 8-bit types
EPS = 1e-5


def listed():
    return [
        # The norm in front of a projection while one token is served: latency.
        {"name": "norm 1x2048", "op": "norm", "dtype": "f16", "rows": 1, "width": 2048, "residual": True, "out": "e4m3",
         "group": 0},
        # A ragged batch of short requests, integer activations; the width is no power of two.
        {"name": "norm 1171x5120 i8", "op": "norm", "dtype": "f16", "rows": 1171, "width": 5120, "residual": False,
         "out": "i8", "group": 0},
        # 16 requests of 1500 tokens, one scale for each 128 columns: bandwidth.
        {"name": "norm 24000x2048", "op": "norm", "dtype": "bf16", "rows": 24000, "width": 2048, "residual": True,
         "out": "e4m3", "group": 128},
        # One served token at a late position.
        {"name": "rope 1", "op": "rope", "dtype": "f16", "tokens": 1, "q_heads": 24, "k_heads": 8, "head_dim": 128,
         "rotary": 128, "layout": "pairs", "far": 32768},
        # A ragged batch whose heads are rotated in part, halves layout.
        {"name": "rope 1171 part", "op": "rope", "dtype": "bf16", "tokens": 1171, "q_heads": 24, "k_heads": 8,
         "head_dim": 128, "rotary": 64, "layout": "halves", "far": 5000},
        # 16 requests of 1500 tokens of a long-context model.
        {"name": "rope 24000", "op": "rope", "dtype": "f16", "tokens": 24000, "q_heads": 24, "k_heads": 8,
         "head_dim": 128, "rotary": 128, "layout": "pairs", "far": 1000000},
        # The fused QKV projection of one token.
        {"name": "w4 1x5120x2048", "op": "w4", "x": "f16", "m": 1, "n": 5120, "k": 2048, "group": 128, "zeros": False,
         "scale": "f16", "y": "f16", "x_group": 0},
        # The down projection of thirteen tokens in 8 bits, with zero points.
        {"name": "w4 13x2048x6144 e4m3", "op": "w4", "x": "e4m3", "m": 13, "n": 2048, "k": 6144, "group": 64,
         "zeros": True, "scale": "bf16", "y": "bf16", "x_group": 128},
        # One row against a matrix of the token table's size: bandwidth.
        {"name": "w4 1x131072x2048", "op": "w4", "x": "bf16", "m": 1, "n": 131072, "k": 2048, "group": 128,
         "zeros": True, "scale": "f16", "y": "f32", "x_group": 0},
        # One new token for each of 16 requests against caches of up to 5000 keys.
        {"name": "attention 16x1 of 5000", "op": "attention", "dtype": "f16", "batch": 16, "q_len": 1, "k_len": 5000,
         "ragged": True, "left": 1023, "right": 0, "sinks": 4, "q_heads": 24, "kv_heads": 8, "head_dim": 128},
        # A batch of documents through a local layer of an encoder, the first token seen by all.
        {"name": "attention 16x1500 local", "op": "attention", "dtype": "f16", "batch": 16, "q_len": 1500,
         "k_len": 1500, "ragged": True, "left": 128, "right": 128, "sinks": 1, "q_heads": 24, "kv_heads": 8,
         "head_dim": 128},
        # A long prompt through a causal layer with a window.
        {"name": "attention 8192 window", "op": "attention", "dtype": "bf16", "batch": 1, "q_len": 8192,
         "k_len": 8192, "ragged": False, "left": 2047, "right": 0, "sinks": 4, "q_heads": 24, "kv_heads": 8,
         "head_dim": 128},
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["norm", "rope", "w4", "attention", "attention"])
    if op == "norm":
        width = rng.choice([2048, 5120, 6144, 8 * _spread(rng, 8, 1536), _spread(rng, 65, 12288)])
        return {"op": op, "dtype": rng.choice(["f16", "bf16"]), "rows": _spread(rng, 1, 24000 * 2048 // width),
                "width": width, "residual": rng.random() < 0.6, "out": rng.choice(["e4m3", "i8"]),
                "group": rng.choice([0, 32, 64, 128])}
    if op == "rope":
        head_dim = rng.choice([64, 80, 128, 256])
        k_heads = rng.choice([1, 2, 4, 8])
        q_heads = k_heads * rng.choice([1, 2, 3, 4])
        return {"op": op, "dtype": rng.choice(["f16", "bf16"]),
                "tokens": _spread(rng, 1, 24000 * 4096 // ((q_heads + k_heads) * head_dim)), "q_heads": q_heads,
                "k_heads": k_heads, "head_dim": head_dim, "rotary": rng.choice([head_dim, head_dim // 2]),
                "layout": rng.choice(["pairs", "halves"]), "far": _spread(rng, 64, 1000000)}
    if op == "w4":
        group = rng.choice([32, 64, 128])
        k = group * _spread(rng, max(1, 256 // group), 8192 // group)
        x = rng.choice(["f16", "bf16", "e4m3", "i8"])
        return {"op": op, "x": x, "m": _spread(rng, 1, 16), "n": _spread(rng, 100, 131072 * 2048 // k), "k": k,
                "group": group, "zeros": rng.random() < 0.5, "scale": rng.choice(["f16", "bf16"]),
                "y": rng.choice(["f16", "bf16", "f32"]), "x_group": rng.choice([0, 32, 64, 128])}
    kv_heads = rng.choice([1, 2, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4])
    batch = _spread(rng, 1, 16)
    if rng.random() < 0.5:  # a few new tokens against a cache
        q_len, k_len = _spread(rng, 1, 16), _spread(rng, 16, 32768)
        left, right = rng.choice([-1, _spread(rng, 16, 8191)]), 0
    else:  # whole prompts or documents
        k_len = _spread(rng, 17, int(math.sqrt(8192 * 8192 * 24 / (batch * q_heads))) if batch * q_heads > 24 else 8192)
        q_len = k_len if rng.random() < 0.7 else max(1, k_len // 2)
        left = rng.choice([-1, _spread(rng, 16, 4095)])
        right = rng.choice([0, 0, -1, _spread(rng, 1, 512)])
    return {"op": "attention", "dtype": rng.choice(["f16", "bf16"]), "batch": batch, "q_len": q_len, "k_len": k_len,
            "ragged": batch > 1 and rng.random() < 0.7, "left": left, "right": right, "sinks": rng.choice([0, 1, 4, 64]),
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": rng.choice([64, 128])}


def _lengths(case):
    """(query length, key length) of each request: equal ones, or spread from a tenth up to the case's own. They
    belong to the case, not to the seed, so that every state of a case has the same work."""
    b, q, k = case["batch"], case["q_len"], case["k_len"]
    if not case["ragged"]:
        return [q] * b, [k] * b
    part = [1.0 - 0.9 * ((7 * i) % b) / b for i in range(b)]
    ks = [max(1, round(k * p)) for p in part]
    qs = [min(max(1, round(q * p)) if q > 16 else q, x) for p, x in zip(part, ks)]
    return qs, ks


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def whole(low, high, *shape, dtype=torch.int32):
        return torch.randint(low, high, shape, generator=g, device="cuda", dtype=dtype)

    s = {"case": case}
    if case["op"] == "norm":
        rows, width, t = case["rows"], case["width"], DTYPES[case["dtype"]]
        # a residual stream has a few columns that stand out
        loud = 1 + 15 * (torch.rand(width, generator=g, device="cuda") < 0.01).float()
        s["x"] = (2 * normal(rows, width) * loud).to(t)
        s["r"] = normal(rows, width).to(t) if case["residual"] else None
        s["w"] = 1 + 0.1 * normal(width)
        s["sum"] = torch.empty_like(s["x"]) if case["residual"] else None
        s["q"] = torch.empty((rows, width), dtype=DTYPES[case["out"]], device="cuda")
        s["scales"] = torch.empty((rows, -(-width // (case["group"] or width))), device="cuda")
    elif case["op"] == "rope":
        n, d, t = case["tokens"], case["head_dim"], DTYPES[case["dtype"]]
        s["q"] = normal(n, case["q_heads"], d).to(t)
        s["k"] = normal(n, case["k_heads"], d).to(t)
        s["pos"] = whole(0, case["far"], n)
        half = case["rotary"] // 2
        s["freq"] = 1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["magnitude"] = 1.0
        s["qo"], s["ko"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
    elif case["op"] == "w4":
        m, n, k, gr = case["m"], case["n"], case["k"], case["group"]
        s["w"] = whole(0, 256, n, k // 2, dtype=torch.uint8)
        s["s"] = (0.002 + 0.004 * torch.rand((n, k // gr), generator=g, device="cuda")).to(DTYPES[case["scale"]])
        s["z"] = whole(0, 256, n, (k // gr + 1) // 2, dtype=torch.uint8) if case["zeros"] else None
        s["xs"] = None
        if case["x"] in TOP:
            xg = case["x_group"] or k
            s["x"] = (normal(m, k).clamp(-3.9, 3.9) * (TOP[case["x"]] / 4)).to(DTYPES[case["x"]])
            s["xs"] = 0.005 + 0.01 * torch.rand((m, -(-k // xg)), generator=g, device="cuda")
        else:
            s["x"] = normal(m, k).to(DTYPES[case["x"]])
        s["y"] = torch.empty((m, n), dtype=DTYPES[case["y"]], device="cuda")
    else:
        qs, ks = _lengths(case)
        t, d, hq, hk = DTYPES[case["dtype"]], case["head_dim"], case["q_heads"], case["kv_heads"]
        s["q"] = normal(sum(qs), hq, d).to(t)
        s["k"] = normal(sum(ks), hk, d).to(t)
        s["v"] = normal(sum(ks), hk, d).to(t)
        s["q_off"] = torch.tensor([0] + list(np.cumsum(qs)), device="cuda", dtype=torch.int32)
        s["k_start"] = torch.tensor([0] + list(np.cumsum(ks))[:-1], device="cuda", dtype=torch.int32)
        s["k_len"] = torch.tensor(ks, device="cuda", dtype=torch.int32)
        s["max_q"], s["max_k"] = max(qs), max(ks)
        s["out"] = torch.empty_like(s["q"])
        s["err"] = torch.zeros(1, device="cuda", dtype=torch.int32)
    return s


def run(s):
    return {"norm": _norm, "rope": _rope, "w4": _w4, "attention": _attention}[s["case"]["op"]](s)


_library = None


def _lib():
    """The library's entry points, and the check of their status."""
    global _library
    if _library is None:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nemotron-3-embed-webgpu_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        from nemo_b200 import runtime
        _library = (runtime.load_library(), runtime.check)
    return _library


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _at(t):
    return None if t is None else t.data_ptr()


def _norm(s):
    c, x, r, w = s["case"], s["x"], s["r"], s["w"]
    rows, width = x.shape
    group = c["group"] or width
    if own:
        lib, check = _lib()
        check(lib.nemo_op_rmsnorm_q8(CODES[c["dtype"]], x.data_ptr(), width, _at(r), width, w.data_ptr(), rows, width,
                                     EPS, _at(s["sum"]), width, CODES[c["out"]], c["group"], s["q"].data_ptr(), width,
                                     s["scales"].data_ptr(), _stream()))
        return {"sum": s["sum"], "q": s["q"], "scales": s["scales"]}
    h = x.float()
    if r is not None:
        h = h + r.float()
    # codes from u = h * w and its largest value: the norm's factor is the same in both and falls out
    u = h * w
    pad = -width % group
    ug = torch.nn.functional.pad(u, (0, pad)).view(rows, -1, group)
    top = ug.abs().amax(-1)
    # a division of tensors rounds once (a number over a tensor is a reciprocal and a product)
    to = torch.where(top > 1e-30, torch.full_like(top, TOP[c["out"]]).div(top), 0.0)
    q = (ug * to.unsqueeze(-1)).view(rows, -1)[:, :width]
    q = q.round().to(torch.int8) if c["out"] == "i8" else q.to(torch.float8_e4m3fn)
    inv = (h.double().square().mean(-1, keepdim=True) + EPS).rsqrt()
    return {"sum": None if r is None else h.to(x.dtype), "q": q.contiguous(),
            "scales": (top.double() * inv / TOP[c["out"]]).float()}


def _rope(s):
    c, q, k = s["case"], s["q"], s["k"]
    rot, d = c["rotary"], c["head_dim"]
    if own:
        lib, check = _lib()
        check(lib.nemo_op_rope_apply(CODES[c["dtype"]], 1 if c["layout"] == "halves" else 0, q.data_ptr(),
                                     c["q_heads"] * d, c["q_heads"], k.data_ptr(), c["k_heads"] * d, c["k_heads"], d,
                                     rot, s["freq"].data_ptr(), s["magnitude"], s["pos"].data_ptr(), c["tokens"],
                                     s["qo"].data_ptr(), c["q_heads"] * d, s["ko"].data_ptr(), c["k_heads"] * d,
                                     _stream()))
        return {"q": s["qo"], "k": s["ko"]}
    angle = s["pos"].double().unsqueeze(-1) * s["freq"]  # positions reach a million: 64 bits
    cos, sin = ((f(angle) * s["magnitude"]).float().unsqueeze(1) for f in (torch.cos, torch.sin))
    return {"q": _turned(q, cos, sin, rot, c["layout"]), "k": _turned(k, cos, sin, rot, c["layout"])}


def _turned(x, cos, sin, rot, layout):
    f = x.float()
    if layout == "pairs":
        a, b = f[..., 0:rot:2], f[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = f[..., :rot // 2], f[..., rot // 2:rot]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, f[..., rot:]), -1).to(x.dtype)


def _nibbles(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _w4(s):
    c, x = s["case"], s["x"]
    m, n, k, group = c["m"], c["n"], c["k"], c["group"]
    if own:
        lib, check = _lib()
        check(lib.nemo_op_w4_matvec(CODES[c["x"]], x.data_ptr(), k, _at(s["xs"]), c["x_group"] or k, s["w"].data_ptr(),
                                    CODES[c["scale"]], s["s"].data_ptr(), _at(s["z"]), group, m, n, k, CODES[c["y"]],
                                    s["y"].data_ptr(), n, _stream()))
        return s["y"]
    q = _nibbles(s["w"]).float().view(n, k // group, group)
    z = 8.0 if s["z"] is None else _nibbles(s["z"])[:, :k // group].float().unsqueeze(-1)
    w = ((q - z) * s["s"].float().unsqueeze(-1)).view(n, k)
    f = x.float()
    if s["xs"] is not None:
        f = f * s["xs"].repeat_interleave(c["x_group"] or k, 1)[:, :k]
    return (f @ w.t()).to(DTYPES[c["y"]])


def _attention(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    b, hq, hk, d = c["batch"], c["q_heads"], c["kv_heads"], c["head_dim"]
    if own:
        lib, check = _lib()
        check(lib.nemo_op_attention_window(CODES[c["dtype"]], q.data_ptr(), hq * d, k.data_ptr(), hk * d, v.data_ptr(),
                                           hk * d, hq, hk, d, s["q_off"].data_ptr(), s["k_start"].data_ptr(),
                                           s["k_len"].data_ptr(), b, q.shape[0], k.shape[0], s["max_q"], s["max_k"],
                                           c["left"], c["right"], c["sinks"], d ** -0.5, s["out"].data_ptr(), hq * d,
                                           s["err"].data_ptr(), _stream()))
        return s["out"]
    mq, mk = s["max_q"], s["max_k"]
    i, j = torch.arange(mq, device=q.device), torch.arange(mk, device=q.device)
    q_len = (s["q_off"][1:] - s["q_off"][:-1]).view(b, 1)
    k_len = s["k_len"].view(b, 1)
    rows = (s["q_off"][:-1].view(b, 1) + i).clamp(max=q.shape[0] - 1)
    cols = (s["k_start"].view(b, 1) + j).clamp(max=k.shape[0] - 1)
    fq = q[rows].float().view(b, mq, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    fk = k[cols].float().permute(0, 2, 3, 1)
    fv = v[cols].float().permute(0, 2, 1, 3)
    p = (i + k_len - q_len).view(b, mq, 1)
    seen = (j < k_len).view(b, 1, mk).expand(b, mq, mk)
    if c["right"] >= 0:
        seen = seen & (j <= p + c["right"])
    if c["left"] >= 0:
        seen = seen & ((j >= p - c["left"]) | (j < c["sinks"]))
    score = (fq @ fk).view(b, hk, hq // hk, mq, mk).mul_(d ** -0.5)
    score.masked_fill_(~seen.view(b, 1, 1, mq, mk), -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = score.sum(-1, keepdim=True)
    o = (score.view(b, hk, -1, mk) @ fv).view(b, hk, hq // hk, mq, d) / total.clamp_(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, mq, hq, d)
    at = torch.arange(q.shape[0], device=q.device, dtype=torch.int32)
    of = torch.searchsorted(s["q_off"], at, right=True) - 1
    return o[of, at - s["q_off"][of]].to(q.dtype)


def _pairs(case):
    """Visible (query, key) pairs of a case, and the key rows that some query sees."""
    pairs = keys = 0
    for nq, nk in zip(*_lengths(case)):
        p = np.arange(nq) + nk - nq
        end = np.full(nq, nk) if case["right"] < 0 else np.minimum(nk, p + case["right"] + 1)
        begin = np.zeros(nq, dtype=int) if case["left"] < 0 else np.clip(p - case["left"], 0, None)
        first = np.minimum(np.minimum(case["sinks"], begin), end)  # sinks in front of the window
        pairs += int(np.clip(end - begin, 0, None).sum() + np.clip(first, 0, None).sum())
        keys += int(end.max() - min(begin.min(), end.max()) + min(case["sinks"], begin.min()))
    return pairs, keys


def work(case):
    if case["op"] == "norm":
        n, groups = case["rows"] * case["width"], -(-case["width"] // (case["group"] or case["width"]))
        return {"bytes": n * (7 if case["residual"] else 3) + 4 * case["width"] + 4 * case["rows"] * groups,
                "flops": 8 * n}
    if case["op"] == "rope":
        heads = case["tokens"] * (case["q_heads"] + case["k_heads"])
        return {"bytes": heads * case["head_dim"] * 4 + case["tokens"] * 4 + case["rotary"] * 4,
                "flops": heads * case["rotary"] * 3}
    if case["op"] == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        groups = n * (k // case["group"])
        x = m * k * (1 if case["x"] in TOP else 2)
        return {"bytes": n * k // 2 + groups * 2 + (groups // 2 if case["zeros"] else 0) + x
                + m * n * (4 if case["y"] == "f32" else 2), "flops": 2 * m * n * k}
    pairs, keys = _pairs(case)
    row = case["head_dim"] * 2
    return {"bytes": 2 * sum(_lengths(case)[0]) * case["q_heads"] * row + 2 * keys * case["kv_heads"] * row,
            "flops": 4 * pairs * case["q_heads"] * case["head_dim"]}


def exact(case, seed):
    """run()'s outputs in 64 bits. 8-bit codes are given as the numbers that they round; integer ones have none."""
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() + (s["r"].double() if case["residual"] else 0.0)
        y = h * s["w"].double() / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
        group = case["group"] or case["width"]
        scales = torch.stack([part.abs().max(1).values for part in y.split(group, 1)], 1) / TOP[case["out"]]
        each = scales.gather(1, (torch.arange(case["width"], device="cuda") // group).expand(case["rows"], -1))
        return {"sum": h if case["residual"] else None, "q": None if case["out"] == "i8" else y / each,
                "scales": scales}
    if case["op"] == "rope":
        half = case["rotary"] // 2
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double()[:, None] * s["freq"])
        out = {}
        for name in ("q", "k"):
            x = s[name].double()
            part = x[..., :2 * half]
            if case["layout"] == "pairs":
                z = torch.view_as_complex(part.unflatten(-1, (half, 2)).contiguous()) * turn[:, None]
                y = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * turn[:, None]
                y = torch.cat((z.real, z.imag), -1)
            out[name] = torch.cat((y, x[..., 2 * half:]), -1)
        return out
    if case["op"] == "w4":
        group, k = case["group"], case["k"]
        x = s["x"].double()
        if s["xs"] is not None:
            at = torch.arange(k, device="cuda") // (case["x_group"] or k)
            x = x * s["xs"].double()[:, at]
        y = torch.empty((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for r in range(0, case["n"], 8192):
            b = s["w"][r:r + 8192].to(torch.int16)
            w = torch.empty((b.shape[0], k), dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = (b % 16).double(), (b // 16).double()
            w = w.unflatten(1, (k // group, group))
            if s["z"] is None:
                w -= 8
            else:
                zb = s["z"][r:r + 8192].to(torch.int16)
                zero = torch.empty((b.shape[0], 2 * zb.shape[1]), dtype=torch.float64, device="cuda")
                zero[:, 0::2], zero[:, 1::2] = (zb % 16).double(), (zb // 16).double()
                w -= zero[:, :k // group, None]
            w *= s["s"][r:r + 8192].double()[..., None]
            y[:, r:r + 8192] = x @ w.flatten(1).t()
        return y
    ratio = case["q_heads"] // case["kv_heads"]
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    q0 = k0 = 0
    for nq, nk in zip(*_lengths(case)):
        p = torch.arange(nk - nq, nk, device="cuda")[:, None]
        j = torch.arange(nk, device="cuda")[None]
        hidden = torch.zeros((nq, nk), dtype=torch.bool, device="cuda")
        if case["right"] >= 0:
            hidden |= j - p > case["right"]
        if case["left"] >= 0:
            hidden |= (p - j > case["left"]) & (j >= case["sinks"])
        for h in range(case["kv_heads"]):
            kh, vh = s["k"][k0:k0 + nk, h].double(), s["v"][k0:k0 + nk, h].double()
            for e in range(h * ratio, (h + 1) * ratio):
                a = (s["q"][q0:q0 + nq, e].double() @ kh.t()) / math.sqrt(case["head_dim"])
                a = a.masked_fill(hidden, -math.inf).softmax(1).nan_to_num(0.0)
                out[q0:q0 + nq, e] = a @ vh
        q0, k0 = q0 + nq, k0 + nk
    return out
