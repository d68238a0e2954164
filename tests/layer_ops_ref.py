"""Plain 64-bit forms of the layer operators (include/nemo_ops.h), the error each may make, and call helpers."""
import math

import numpy as np
import torch

from nemo_b200.runtime import check, load_library

F16, BF16, F32, E4M3, I8 = range(5)  # NEMO_DTYPE_*
TORCH = {F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32, E4M3: torch.float8_e4m3fn, I8: torch.int8}
TOP = {E4M3: 448.0, I8: 127.0}
HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}  # largest relative rounding error
U32 = 2.0 ** -24


def lib():
    return load_library()


def at(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def close(got, want, bound):
    """|got - want| <= bound element by element (all finite)."""
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - bound
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0, f"{int((over > 0).sum())} of {over.numel()} values are off, by up to {worst:.3g} over the bound"


# --- rmsnorm_q8 ------------------------------------------------------------------

def rmsnorm_q8(x, r, w, eps, out, group, total=None, q=None, ldq=None):
    rows, width = x.shape
    dt = F16 if x.dtype == torch.float16 else BF16
    groups = -(-width // (group or width))
    if r is not None and total is None:
        total = torch.empty((rows, width), dtype=x.dtype, device="cuda")
    if q is None:
        q = torch.full((rows, width), 77, dtype=torch.uint8, device="cuda").view(TORCH[out])
    scales = torch.full((rows, groups), -1.0, device="cuda")
    check(lib().nemo_op_rmsnorm_q8(dt, x.data_ptr(), x.stride(0), at(r), r.stride(0) if r is not None else 0,
                                   w.data_ptr(), rows, width, eps, at(total), total.stride(0) if r is not None else 0,
                                   out, group, q.data_ptr(), q.stride(0), scales.data_ptr(), stream()))
    return total, q, scales


def check_rmsnorm_q8(x, r, w, eps, out, group, got):
    """sum: one rounding (of an f32 sum that is off by one f32 rounding). Codes: bit for bit, from the f32 products
    u = s * w and u * (Q / top). scale: the row's sum of squares has at most 32 + 5 + 32 additions in a chain, which
    is half of that in its root, and 8 more roundings: 48 f32 half steps."""
    total, q, scales = got
    rows, width = x.shape
    dt = F16 if x.dtype == torch.float16 else BF16
    s = x.float() if r is None else x.float() + r.float()
    if r is not None:
        s64 = x.double() + r.double()
        close(total, s64, HALF[dt] * s64.abs() * (1 + 1e-3) + 2.0 ** -25)
    u = s * w
    n = group or width
    ug = torch.nn.functional.pad(u, (0, -width % n)).view(rows, -1, n)
    top = ug.abs().amax(-1)
    to = torch.where(top > 1e-30, torch.full_like(top, TOP[out]).div(top), 0.0)  # TOP / top would be a reciprocal
    p = (ug * to.unsqueeze(-1)).view(rows, -1)[:, :width]
    want = p.round().to(torch.int8) if out == I8 else p.to(torch.float8_e4m3fn)
    assert torch.equal(q.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))
    s64 = x.double() + (r.double() if r is not None else 0.0)
    inv = 1 / torch.sqrt((s64 * s64).mean(1, keepdim=True) + eps)
    y = s64 * w.double() * inv
    yg = torch.nn.functional.pad(y, (0, -width % n)).view(rows, -1, n).abs().amax(-1) / TOP[out]
    close(scales, yg, 48 * U32 * yg)


# --- rope ------------------------------------------------------------------------

def rope_apply(q, k, inv_freq, magnitude, pos, rotary, layout, qo=None, ko=None):
    dt = F16 if q.dtype == torch.float16 else BF16
    tokens, hq, d = q.shape
    hk = 0 if k is None else k.shape[1]
    qo = torch.full((tokens, hq, d), float("nan"), dtype=q.dtype, device="cuda") if qo is None else qo
    if k is not None and ko is None:
        ko = torch.full((tokens, hk, d), float("nan"), dtype=q.dtype, device="cuda")
    check(lib().nemo_op_rope_apply(dt, layout, q.data_ptr(), q.stride(0), hq, at(k), k.stride(0) if hk else 0, hk, d,
                                   rotary, inv_freq.data_ptr(), magnitude, pos.data_ptr(), tokens, qo.data_ptr(),
                                   qo.stride(0), at(ko), ko.stride(0) if hk else 0, stream()))
    return qo, ko


def check_rope(x, inv_freq, magnitude, pos, rotary, layout, got):
    """One rounding to the type; cos and sin are off by at most 3 * 2^-23 (the f32 fraction of a turn and sincospi),
    the products and their sum by 3 more f32 roundings: 2^-21 of |a| + |b|. Copied columns are equal."""
    dt = F16 if x.dtype == torch.float16 else BF16
    half = rotary // 2
    t = pos.double()[:, None] * inv_freq
    cos, sin = magnitude * torch.cos(t)[:, None], magnitude * torch.sin(t)[:, None]
    v = x.double()
    a, b = (v[..., 0:rotary:2], v[..., 1:rotary:2]) if layout == 0 else (v[..., :half], v[..., half:rotary])
    g = got.double()
    ga, gb = (g[..., 0:rotary:2], g[..., 1:rotary:2]) if layout == 0 else (g[..., :half], g[..., half:rotary])
    slack = 2.0 ** -21 * abs(magnitude) * (a.abs() + b.abs()) + 2.0 ** -25
    for have, want in ((ga, a * cos - b * sin), (gb, a * sin + b * cos)):
        close(have, want, HALF[dt] * (want.abs() + slack) + slack)
    assert torch.equal(got[..., rotary:], x[..., rotary:])


# --- w4 --------------------------------------------------------------------------

def pack4(v):
    """Two values of 0..15 per byte, the even column in the low bits; an odd last column alone."""
    if v.shape[1] % 2:
        v = torch.nn.functional.pad(v, (0, 1))
    return (v[:, 0::2] | (v[:, 1::2] << 4)).to(torch.uint8).contiguous()


def w4_matvec(x, xs, x_group, w4, scales, zeros, group, n, y_dtype, y=None):
    dt = {v: k for k, v in TORCH.items()}
    m, k = x.shape
    y = torch.full((m, n), float("nan"), dtype=TORCH[y_dtype], device="cuda") if y is None else y
    check(lib().nemo_op_w4_matvec(dt[x.dtype], x.data_ptr(), x.stride(0), at(xs), x_group, w4.data_ptr(),
                                  dt[scales.dtype], scales.data_ptr(), at(zeros), group, m, n, k, y_dtype,
                                  y.data_ptr(), y.stride(0), stream()))
    return y


def check_w4(x, xs, x_group, q, scales, z, group, y, y_dtype):
    """One rounding to the type of y. The f32 sums: at most 8 instructions in a segment's chain, each good to two f32
    steps of its largest term, then one product and one addition for each of a warp's segments and 16 additions over
    warps and panels: (40 + segments / 4) steps of sum |x w|."""
    k = x.shape[1]
    f = x.double()
    if xs is not None:
        f = f * xs.double().repeat_interleave(min(x_group, k), 1)[:, :k]
    zz = 8.0 if z is None else z.double().repeat_interleave(group, 1)
    w = (q.double() - zz) * scales.double().repeat_interleave(group, 1)
    want = f @ w.t()
    mag = f.abs() @ w.abs().t()
    segments = k / min(group, x_group if xs is not None else group)
    slack = (40 + segments / 4) * 2 * U32 * mag
    close(y, want, HALF[y_dtype] * (want.abs() + slack) + slack + 2.0 ** -25)


# --- attention -------------------------------------------------------------------

def attention(q, k, v, q_off, k_start, k_len, left, right, sinks, scale=None, out=None, max_q=None, max_k=None,
              err=None):
    dt = F16 if q.dtype == torch.float16 else BF16
    hq, d = q.shape[1:]
    hk = k.shape[1]
    dev = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in (q_off, k_start, k_len)]
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") if out is None else out
    mine = err is None
    err = torch.zeros(1, dtype=torch.int32, device="cuda") if mine else err
    max_q = max(np.diff(q_off)) if max_q is None else max_q
    check(lib().nemo_op_attention_window(
        dt, q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), hq, hk, d,
        dev[0].data_ptr(), dev[1].data_ptr(), dev[2].data_ptr(), len(k_len), q.shape[0], k.shape[0], int(max_q),
        int(max(k_len) if max_k is None else max_k), left, right, sinks, d ** -0.5 if scale is None else scale,
        out.data_ptr(), out.stride(0), err.data_ptr(), stream()))
    torch.cuda.synchronize()  # the offsets above live until here
    if mine:
        assert int(err) == 0
    return out


def seen(nq, nk, left, right, sinks):
    """[nq x nk] truth of which query sees which key."""
    p = torch.arange(nk - nq, nk, device="cuda")[:, None]
    j = torch.arange(nk, device="cuda")[None]
    ok = torch.ones((nq, nk), dtype=torch.bool, device="cuda")
    if right >= 0:
        ok &= j <= p + right
    if left >= 0:
        ok &= (j >= p - left) | (j < sinks)
    return ok


def check_attention(q, k, v, q_off, k_start, k_len, left, right, sinks, got, scale=None):
    """Per request and head against a 64-bit softmax. The weights are rounded to the type (half a step each, and an
    absolute 2^-25 of the largest where an f16 weight is subnormal), the result once more; scores and exponentials in
    f32 are off by under 2^-15 of a weight."""
    dt = F16 if q.dtype == torch.float16 else BF16
    hq, d = q.shape[1:]
    ratio = hq // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    for b, nk in enumerate(k_len):
        q0, q1 = q_off[b], q_off[b + 1]
        ok = seen(q1 - q0, nk, left, right, sinks)
        for h in range(hq):
            kh = k[k_start[b]:k_start[b] + nk, h // ratio].double()
            vh = v[k_start[b]:k_start[b] + nk, h // ratio].double()
            s = (q[q0:q1, h].double() @ kh.t()) * scale
            s = s.masked_fill(~ok, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, 1), nan=0.0) if nk else s
            want, mag = p @ vh, p @ vh.abs()
            tiny = ok.sum(1, keepdim=True) * 2.0 ** -25 * (vh.abs().max() if nk else 0.0) + 2.0 ** -25
            slack = (HALF[dt] + 2.0 ** -15) * mag + tiny
            close(got[q0:q1, h], want, HALF[dt] * (want.abs() + slack) + slack)
