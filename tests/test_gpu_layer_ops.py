"""The layer operators of include/nemo_ops.h on the GPU against 64-bit forms (layer_ops_ref.py), where they can go
wrong: sizes around the tiles, strides, groups, windows that leave a row empty, garbage where nothing may look, streams
and graphs, and one layer's run of them together."""
import ctypes
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

import layer_ops_ref as ref
from layer_ops_ref import BF16, E4M3, F16, F32, I8, TORCH
from nemo_b200.runtime import NemoError, check, load_library

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("dt", [F16, BF16], ids=["f16", "bf16"])


@pytest.fixture
def gen():
    g = torch.Generator(device="cuda")
    g.manual_seed(77)
    return g


def normal(gen, *shape, dt=F32):
    return torch.randn(shape, generator=gen, device="cuda").to(TORCH[dt])


# --- rmsnorm_q8 ------------------------------------------------------------------

@TYPES
@pytest.mark.parametrize("out", [E4M3, I8], ids=["e4m3", "i8"])
@pytest.mark.parametrize("rows,width", [(1, 2048), (3, 1), (5, 7), (300, 64), (33, 129), (9, 5120), (2, 12296),
                                        (2, 32768), (700, 1000)])
def test_rmsnorm_q8(gen, dt, out, rows, width):
    x = normal(gen, rows, width, dt=dt) * 3
    w = 1 + 0.2 * normal(gen, width)
    r = normal(gen, rows, width, dt=dt)
    for group in (0, 32, 64, 128):
        for res in (None, r):
            got = ref.rmsnorm_q8(x, res, w, 1e-5, out, group)
            ref.check_rmsnorm_q8(x, res, w, 1e-5, out, group, got)


def test_rmsnorm_q8_strides_and_in_place(gen):
    rows, width = 37, 256
    for ld in (width + 3, width + 8):  # rows that are not, and that are, 16 bytes apart
        x, r = normal(gen, rows, ld, dt=F16), normal(gen, rows, ld, dt=F16)
        w = normal(gen, width)
        q = torch.full((rows, ld), 5, dtype=torch.int8, device="cuda")
        want = ref.rmsnorm_q8(x[:, :width].contiguous(), r[:, :width].contiguous(), w, 1e-5, I8, 64)
        before = x.clone()
        total, _, scales = ref.rmsnorm_q8(x[:, :width], r[:, :width], w, 1e-5, I8, 64, total=x[:, :width],
                                          q=q[:, :width])
        assert torch.equal(total, want[0]) and torch.equal(q[:, :width], want[1]) and torch.equal(scales, want[2])
        assert torch.equal(x[:, width:], before[:, width:]) and (q[:, width:] == 5).all()  # the gaps stay


def test_rmsnorm_q8_zeros_infinities_and_nan(gen):
    x = normal(gen, 4, 256, dt=BF16)
    w = torch.ones(256, device="cuda")
    x[0] = 0
    x[1, 130] = float("nan")
    x[2, 10] = float("inf")
    x[3, 64:128] = 0
    _, q, s = ref.rmsnorm_q8(x, None, w, 1e-5, E4M3, 64)
    q = q.view(torch.uint8)
    assert (q[0] == 0).all() and (s[0] == 0).all()
    assert torch.isnan(s[1]).all() and (q[1, 128:192] == 0).all()
    assert torch.isnan(s[2, 0]) and (s[2, 1:] == 0).all() and (q[2, :64] == 0).all()
    assert (q[3, 64:128] == 0).all() and s[3, 1] == 0 and (s[3, [0, 2, 3]] > 0).all()
    _, q, s = ref.rmsnorm_q8(torch.zeros_like(x), None, w, 0.0, I8, 0)  # 0 / 0 without eps
    assert (q == 0).all()


# --- rope ------------------------------------------------------------------------

def inv_freq(scaling, theta, rotary, *rest):
    out, mag = np.zeros(rotary // 2), ctypes.c_float()
    check(load_library().nemo_rope_inv_freq(scaling, theta, rotary, *rest, out.ctypes.data_as(ctypes.c_void_p),
                                            ctypes.byref(mag)))
    return torch.from_numpy(out).cuda(), mag.value


@TYPES
@pytest.mark.parametrize("layout", [0, 1], ids=["pairs", "halves"])
@pytest.mark.parametrize("tokens,hq,hk,d,rotary", [
    (1, 24, 8, 128, 128), (5, 3, 1, 128, 64), (77, 4, 4, 64, 64), (3, 2, 1, 80, 40), (2, 5, 0, 96, 2), (4, 1, 1, 6, 4),
    (3, 2, 2, 256, 256), (2, 1, 1, 512, 512), (2, 1, 1, 511, 510), (600, 24, 8, 128, 32)])
def test_rope_apply(gen, dt, layout, tokens, hq, hk, d, rotary):
    q = normal(gen, tokens, hq, d, dt=dt)
    k = normal(gen, tokens, hk, d, dt=dt) if hk else None
    freq, mag = inv_freq(3, 1e6, rotary, 16.0, 4096.0, 1.0, 32.0)
    pos = torch.randint(0, 40000, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    qo, ko = ref.rope_apply(q, k, freq, mag, pos, rotary, layout)
    ref.check_rope(q, freq, mag, pos, rotary, layout, qo)
    if hk:
        ref.check_rope(k, freq, mag, pos, rotary, layout, ko)


@pytest.mark.parametrize("layout", [0, 1], ids=["pairs", "halves"])
@pytest.mark.parametrize("pad", [8, 3])
def test_rope_apply_in_a_qkv_buffer_in_place(gen, layout, pad):
    tokens, hq, hk, d, rotary = 19, 6, 2, 64, 32
    ld = (hq + 2 * hk) * d + pad
    buf = normal(gen, tokens, ld, dt=F16)
    before = buf.clone()
    q = torch.as_strided(buf, (tokens, hq, d), (ld, d, 1))
    k = torch.as_strided(buf, (tokens, hk, d), (ld, d, 1), hq * d)
    freq, mag = inv_freq(0, 1e4, rotary, 1.0, 0.0, 0.0, 0.0)
    pos = torch.arange(tokens, device="cuda", dtype=torch.int32)
    wq, wk = q.clone(), k.clone()
    ref.rope_apply(q, k, freq, mag, pos, rotary, layout, qo=q, ko=k)
    ref.check_rope(wq, freq, mag, pos, rotary, layout, q)
    ref.check_rope(wk, freq, mag, pos, rotary, layout, k)
    assert torch.equal(buf[:, (hq + hk) * d:], before[:, (hq + hk) * d:])


def test_rope_apply_far_positions_keep_their_angle(gen):
    q = normal(gen, 4, 1, 64, dt=F16)
    freq, mag = inv_freq(0, 1e6, 64, 1.0, 0.0, 0.0, 0.0)
    pos = torch.tensor([0, 1, 999999, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
    qo, _ = ref.rope_apply(q, None, freq, mag, pos, 64, 0)
    ref.check_rope(q[:3], freq, mag, pos[:3], 64, 0, qo[:3])
    # the 64-bit product of the farthest position is itself off by 2^-23 of a turn
    t = pos[3:].double()[:, None] * freq
    a, b = q[3:, 0, 0::2].double(), q[3:, 0, 1::2].double()
    ref.close(qo[3:, 0, 0::2], a * torch.cos(t) - b * torch.sin(t), 2.0 ** -10 * (a.abs() + b.abs()))


# --- w4 --------------------------------------------------------------------------

def w4_inputs(gen, xt, m, n, k, group, zeros, st, x_group):
    q = torch.randint(0, 16, (n, k), generator=gen, device="cuda")
    z = torch.randint(0, 16, (n, k // group), generator=gen, device="cuda") if zeros else None
    s = (0.01 * normal(gen, n, k // group)).to(TORCH[st])
    xs = None
    if xt in (E4M3, I8):
        x = (normal(gen, m, k) * (100 if xt == E4M3 else 40)).clamp(-127, 127)
        x = (x.round() if xt == I8 else x).to(TORCH[xt])
        xs = 0.01 + 0.02 * torch.rand((m, -(-k // x_group)), generator=gen, device="cuda")
    else:
        x = normal(gen, m, k, dt=xt)
    return x, xs, q, s, z


@pytest.mark.parametrize("xt", [F16, BF16, E4M3, I8], ids=["f16", "bf16", "e4m3", "i8"])
@pytest.mark.parametrize("group,x_group", [(128, 128), (64, 32), (32, 10 ** 6), (128, 64), (32, 128)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 128), (1, 2048, 2048), (2, 17, 384), (3, 100, 1024), (5, 5120, 256),
                                   (8, 33, 2176), (9, 64, 6144), (16, 4800, 640), (16, 16, 8192), (1, 40, 20480)])
def test_w4_matvec(gen, xt, group, x_group, m, n, k):
    zeros, st, yt = (m + n) % 2 == 1, (F16, BF16)[m % 2], (F32, F16, BF16)[(m + k // 128) % 3]
    x, xs, q, s, z = w4_inputs(gen, xt, m, n, k, group, zeros, st, x_group)
    y = ref.w4_matvec(x, xs, x_group, ref.pack4(q), s, ref.pack4(z) if zeros else None, group, n, yt)
    ref.check_w4(x, xs, x_group, q, s, z, group, y, yt)


@pytest.mark.parametrize("xt,group,x_group,m,n,k", [
    (F16, 128, 0, 16, 50, 20480), (E4M3, 32, 64, 12, 9000, 14336), (BF16, 64, 0, 1, 40, 262144),
    (I8, 128, 32, 3, 2000, 65536), (F16, 32, 0, 16, 3, 12320)])
def test_w4_matvec_rows_longer_than_a_cluster_holds(gen, xt, group, x_group, m, n, k):
    """x of a row fills more panels of shared memory than a cluster has blocks: each block takes several in turn."""
    x, xs, q, s, z = w4_inputs(gen, xt, m, n, k, group, True, F16, x_group or k)
    y = ref.w4_matvec(x, xs, x_group, ref.pack4(q), s, ref.pack4(z), group, n, F32)
    ref.check_w4(x, xs, x_group, q, s, z, group, y, F32)


@pytest.mark.parametrize("xt,group,x_group,m,n,k", [
    (F16, 128, 0, 1, 20000, 1024), (BF16, 128, 0, 2, 60000, 640), (E4M3, 128, 128, 1, 30000, 2176),
    (F16, 64, 0, 1, 90000, 576), (F16, 32, 0, 1, 90000, 288), (E4M3, 128, 32, 2, 70000, 512), (I8, 128, 128, 1, 9001, 1024),
    (I8, 128, 0, 5, 40000, 384), (I8, 64, 32, 16, 60000, 256), (I8, 32, 10 ** 6, 3, 50000, 160),
    (F16, 128, 0, 1, 4000, 65536)])
def test_w4_matvec_many_rows(gen, xt, group, x_group, m, n, k):
    x, xs, q, s, z = w4_inputs(gen, xt, m, n, k, group, True, F16, x_group or k)
    y = ref.w4_matvec(x, xs, x_group or k, ref.pack4(q), s, ref.pack4(z), group, n, F32)
    ref.check_w4(x, xs, x_group or k, q, s, z, group, y, F32)


@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("xt,shift", [(F16, 0), (BF16, 0), (BF16, 100), (BF16, -70), (E4M3, 0)])
def test_w4_matvec_many_rows_of_uneven_values(gen, xt, shift, m):
    """Elements of a row whose magnitudes differ by 2^20 or more, whole groups of zeros and lone elements."""
    n, k, group = 50000, 1024, 128
    x, xs, q, s, z = w4_inputs(gen, xt, m, n, k, group, True, F16, k)
    spread = torch.randint(-10, 11, (m, k), generator=gen, device="cuda").double()
    if xt == E4M3:
        x = (x.float() * 2.0 ** (spread.float() - 10)).clamp(-448, 448).to(TORCH[xt])
    else:
        x = (x.double() * 2.0 ** (spread + shift)).clamp(-60000 * 2.0 ** shift, 60000 * 2.0 ** shift).to(TORCH[xt])
    x.view(torch.uint8 if xt == E4M3 else torch.int16)[:, 128:256] = 0
    x.view(torch.uint8 if xt == E4M3 else torch.int16)[:, 300:384] = 0
    y = ref.w4_matvec(x, xs, k, ref.pack4(q), s, ref.pack4(z), group, n, F32)
    ref.check_w4(x, xs, k, q, s, z, group, y, F32)


def test_w4_matvec_many_rows_do_not_mix(gen):
    m, n, k = 2, 50000, 512
    for bad in (float("nan"), float("inf"), -float("inf")):
        x, _, q, s, _ = w4_inputs(gen, BF16, m, n, k, 128, False, F16, k)
        x[1, 300] = bad
        s[7, 0] = float("inf")
        y = ref.w4_matvec(x, None, 0, ref.pack4(q), s, None, 128, n, F32)
        want = torch.zeros((m, n), dtype=torch.bool, device="cuda")
        want[1], want[:, 7] = True, True
        assert torch.equal(~torch.isfinite(y), want)


def test_w4_matvec_strides_and_odd_addresses(gen):
    m, n, k = 6, 50, 512
    x, _, q, s, z = w4_inputs(gen, F16, m, n, k, 64, True, F16, k)
    wide = torch.full((m, k + 5), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, 1:k + 1] = x  # rows two bytes past a 16-byte boundary and odd bytes apart
    y = torch.full((m, n + 7), 9.0, device="cuda")
    ref.w4_matvec(wide[:, 1:k + 1], None, 0, ref.pack4(q), s, ref.pack4(z), 64, n, F32, y=y[:, :n])
    ref.check_w4(x, None, k, q, s, z, 64, y[:, :n], F32)
    assert (y[:, n:] == 9.0).all()
    bytes_x = torch.randint(-127, 128, (m, k + 3), generator=gen, device="cuda", dtype=torch.int8)
    xs = torch.rand((m, 4), generator=gen, device="cuda")
    y = ref.w4_matvec(bytes_x[:, 1:k + 1], xs, 128, ref.pack4(q), s, ref.pack4(z), 64, n, F32)
    ref.check_w4(bytes_x[:, 1:k + 1], xs, 128, q, s, z, 64, y, F32)


@pytest.mark.parametrize("xt,m", [(F16, 2), (E4M3, 1), (I8, 3)])
def test_w4_matvec_many_rows_from_odd_addresses(gen, xt, m):
    n, k = 40000, 512
    x, xs, q, s, z = w4_inputs(gen, xt, m, n, k, 128, True, F16, k)
    wide = torch.zeros((m, k + 5), dtype=TORCH[xt], device="cuda")
    wide[:, 3:k + 3] = x
    y = torch.full((m, n + 3), 9.0, device="cuda")
    ref.w4_matvec(wide[:, 3:k + 3], xs, k, ref.pack4(q), s, ref.pack4(z), 128, n, F32, y=y[:, :n])
    ref.check_w4(x, xs, k, q, s, z, 128, y[:, :n], F32)
    assert (y[:, n:] == 9.0).all()


def test_w4_matvec_rows_do_not_mix(gen):
    """A NaN in one row of x and an infinite scale in one row of W stay in theirs."""
    m, n, k = 4, 64, 256
    x, _, q, s, _ = w4_inputs(gen, F16, m, n, k, 128, False, F16, k)
    x[2, 5] = float("nan")
    s[7, 0] = float("inf")
    y = ref.w4_matvec(x, None, 0, ref.pack4(q), s, None, 128, n, F32)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[2], want[:, 7] = True, True
    assert torch.equal(bad, want)


# --- attention -------------------------------------------------------------------

def packed(gen, dt, qs, ks, hq, hk, d):
    q = normal(gen, sum(qs), hq, d, dt=dt)
    k, v = normal(gen, sum(ks), hk, d, dt=dt), normal(gen, sum(ks), hk, d, dt=dt)
    q_off = [0] + np.cumsum(qs).tolist()
    return q, k, v, q_off, [0] + np.cumsum(ks).tolist()[:-1], list(ks)


WINDOWS = [(-1, -1, 0), (-1, 0, 0), (0, 0, 0), (5, 0, 3), (40, 17, 1), (200, 0, 130), (3, 300, 0), (-1, 6, 2),
           (2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1)]


@TYPES
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", WINDOWS, ids=lambda w: "l%d_r%d_s%d" % w)
@pytest.mark.parametrize("qs,ks", [([1], [1]), ([1, 1, 1], [1, 700, 33]), ([3], [3]), ([17, 0, 2, 40], [17, 9, 64, 40]),
                                   ([130, 1], [130, 300]), ([300, 257], [300, 600]), ([20, 4], [7, 0]),
                                   ([1400, 0, 513, 1], [1400, 5, 901, 1]), ([1300, 700], [90, 0])],
                         ids=["1", "tokens", "3", "ragged", "130", "long", "fewer_keys", "documents",
                              "documents_fewer_keys"])
def test_attention_window(gen, dt, d, window, qs, ks):
    hq, hk = (6, 2) if d == 128 else (5, 1)
    args = packed(gen, dt, qs, ks, hq, hk, d)
    got = ref.attention(*args, *window)
    ref.check_attention(*args, *window, got)


@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 8), (24, 8), (32, 2), (40, 1)])
def test_attention_window_head_layouts(gen, hq, hk):
    for qs, ks in (([2, 1], [900, 5000]), ([150], [333]), ([1100, 700], [1300, 700])):
        args = packed(gen, F16, qs, ks, hq, hk, 128)
        got = ref.attention(*args, 257, 0, 4)
        ref.check_attention(*args, 257, 0, 4, got)


def test_attention_window_more_requests_than_one_launch_takes(gen):
    qs = [1 + (37 * i) % 130 for i in range(1100)]
    args = packed(gen, F16, qs, [n + i % 3 for i, n in enumerate(qs)], 2, 1, 64)
    got = ref.attention(*args, 40, 3, 2)
    ref.check_attention(*args, 40, 3, 2, got)


def test_attention_window_more_work_than_a_block_lists(gen):
    """Over 50 pairs of 128-row tiles for each SM."""
    args = packed(gen, BF16, [1000 + i for i in range(64)], [1000 + i for i in range(64)], 32, 4, 64)
    got = ref.attention(*args, 100, 20, 1)
    ref.check_attention(*args, 100, 20, 1, got)


def test_attention_window_rows_without_keys_are_zeros(gen):
    args = packed(gen, F16, [200, 5], [40, 0], 4, 2, 64)
    got = ref.attention(*args, -1, 0, 0)
    assert (got[:160] == 0).all() and (got[200:] == 0).all()
    ref.check_attention(*args, -1, 0, 0, got)


def test_attention_window_cache_with_room_and_untouched_rows(gen):
    """Keys in a cache [request][capacity] whose unused rows hold NaN, inside a QKV-like row stride; rows of q and out
    behind the last request stay as they were."""
    cap, hq, hk, d = 700, 6, 2, 128
    for q_len, lens in ((1, [0, 1, 333, 700]), (90, [90, 130, 333, 700]), (600, [600, 611, 677, 700])):
        cache = torch.full((4 * cap, 3 * hk * d), float("nan"), dtype=torch.float16, device="cuda")
        for b, n in enumerate(lens):
            cache[b * cap:b * cap + n] = normal(gen, n, 3 * hk * d, dt=F16)
        k = torch.as_strided(cache, (4 * cap, hk, d), (3 * hk * d, d, 1), hk * d)
        v = torch.as_strided(cache, (4 * cap, hk, d), (3 * hk * d, d, 1), 2 * hk * d)
        rows = 4 * q_len + 3
        q = torch.full((rows, hq, d), float("nan"), dtype=torch.float16, device="cuda")
        q[:4 * q_len] = normal(gen, 4 * q_len, hq, d, dt=F16)
        q_off, start = [i * q_len for i in range(5)], [b * cap for b in range(4)]
        for window in ((-1, 0, 0), (100, 0, 2)):
            got = ref.attention(q, k, v, q_off, start, lens, *window)
            assert (got[4 * q_len:] == 7.0).all()
            ref.check_attention(q, k, v, q_off, start, lens, *window, got)


@TYPES
@pytest.mark.parametrize("q_len,nk", [(1, 420), (4, 420), (70, 420), (300, 420), (3000, 3200)])
def test_attention_window_garbage_in_unseen_keys(gen, dt, q_len, nk):
    """Infinities and NaN in keys and values reach the rows that see them, as NaN or infinity, and no other row."""
    hq, hk, d = 4, 2, 64
    args = packed(gen, dt, [q_len], [nk], hq, hk, d)
    q, k, v = args[:3]
    clean = [t.clone() for t in (k, v)]
    left, sinks = 30, 2
    at = nk - q_len + q_len // 2  # in the window of some queries where there are several
    k[at, 0], v[at, 0, 3] = float("nan"), float("inf")
    v[at, 1] = float("nan")
    k[5], v[6] = float("inf"), float("nan")  # between the sinks and every window of a short query
    got = ref.attention(*args, left, 0, sinks)
    ok = ref.seen(q_len, nk, left, 0, sinks)
    dirty = (ok[:, at] | ok[:, 5] | ok[:, 6]).cpu().numpy()
    assert not torch.isfinite(got[dirty]).all(-1).any()
    fine = ~dirty
    want = torch.full_like(got, 0)
    want[fine] = got[fine]
    ref_got = ref.attention(q, *clean, *args[3:], left, 0, sinks)
    ref.check_attention(q, *clean, *args[3:], left, 0, sinks, ref_got)
    # clean rows agree with the run on clean keys to two roundings of the weights
    assert torch.isfinite(got[fine]).all()
    ref.close(got[fine], ref_got[fine].double(), 4 * ref.HALF[dt] * clean[1].abs().max().double())


@TYPES
@pytest.mark.parametrize("q_len", [3, 260])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_attention_window_bad_keys_in_the_open(gen, dt, q_len, bad):
    """One key that every query sees, at each place of a 64-key tile in turn (one kv head each): NaN and infinite
    scores make every row of that head NaN or, for a score of -inf, count for nothing; the clean head stays clean."""
    hk, nk = 65, 700
    args = packed(gen, dt, [q_len], [nk], hk, hk, 64)
    q, k, v = args[:3]
    q.abs_()
    for h in range(64):
        k[128 + h, h] = bad
    got = ref.attention(*args, -1, -1, 0)
    if bad == -float("inf"):
        assert torch.isfinite(got).all()
        k[:, :64] = torch.where(torch.isinf(k[:, :64]), -1000.0, k[:, :64])  # no weight either
        ref.check_attention(*args, -1, -1, 0, got)
    else:
        assert not torch.isfinite(got[:, :64]).any()
        one = (q[:, 64:].contiguous(), k[:, 64:].contiguous(), v[:, 64:].contiguous(), *args[3:])
        ref.check_attention(*one, -1, -1, 0, got[:, 64:])


@TYPES
@pytest.mark.parametrize("q_len,hq", [(1, 2), (200, 2), (1200, 8)])
def test_attention_window_nothing_but_bad_values(gen, dt, q_len, hq):
    """Keys of NaN make every row NaN, values of NaN too; scores that are all -infinity count for nothing."""
    args = packed(gen, dt, [q_len], [1200], hq, 1, 64)
    q, k, v = args[:3]
    q.abs_().add_(0.5)
    for keys, values in ((float("nan"), None), (None, float("nan")), (-float("inf"), None)):
        kk = k if keys is None else torch.full_like(k, keys)
        vv = v if values is None else torch.full_like(v, values)
        got = ref.attention(q, kk, vv, *args[3:], 300, 0, 2)
        assert (got == 0).all() if keys == -float("inf") else torch.isnan(got).all()


@pytest.mark.parametrize("q_len,hq", [(1, 2), (200, 2), (1200, 8)])
def test_attention_window_nan_values_of_keys_without_weight(gen, q_len, hq):
    """A score of -infinity is a weight of 0, and 0 times a NaN is a NaN, wherever among the keys it stands."""
    for at in (0, 1199):
        args = packed(gen, F16, [q_len], [1200], hq, 1, 64)
        q, k, v = args[:3]
        q.abs_().add_(0.5)
        k[at], v[at] = -float("inf"), float("nan")
        assert torch.isnan(ref.attention(*args, -1, -1, 0)).all()


@pytest.mark.parametrize("longest", [40, 900])
def test_attention_window_lengths_that_steer(gen, longest):
    """max_k changes no result beyond the weights' roundings; rows past max_q are not written; requests share keys."""
    args = packed(gen, F16, [longest, 3, longest - 7], [1000, 0, 0], 4, 2, 64)
    args = (*args[:4], [0, 0, 100], [1000, 1000, 900])
    for max_k in (0, 1, 10 ** 9):
        got = ref.attention(*args, 200, 0, 4, max_k=max_k)
        ref.check_attention(*args, 200, 0, 4, got)
    cut = ref.attention(*args, 200, 0, 4, max_q=30)
    for b, (q0, q1) in enumerate(zip(args[3], args[3][1:])):
        n = min(30, q1 - q0)
        assert (cut[q0 + n:q1] == 7.0).all()
        ref.close(cut[q0:q0 + n], got[q0:q0 + n].double(), 4 * ref.HALF[F16] * args[2].abs().max().double())


@pytest.mark.parametrize("q_len,hq", [(1, 2), (200, 2), (900, 8)])
def test_attention_window_large_scores(gen, q_len, hq):
    """Scores of several thousand: the largest key takes all the weight, nothing overflows."""
    args = packed(gen, F16, [q_len], [500 if q_len < 500 else 1200], hq, 1, 128)
    args[0].mul_(30), args[1].mul_(30)
    got = ref.attention(*args, -1, -1, 0, scale=1.0)
    # scores reach 2^17, where an f32 sum of 128 products is good to about 2^-6: compare with the best key where it
    # leads by more
    s = torch.einsum("qhd,khd->hqk", args[0].double(), args[1].double().expand(-1, hq, -1))
    top = s.topk(2, -1)
    clear = (top.values[..., 0] - top.values[..., 1]) > 20
    assert clear.any()
    want = args[2][:, 0].double()[top.indices[..., 0]]
    ref.close(got.permute(1, 0, 2)[clear], want[clear], 2.0 ** -10 * want[clear].abs() + 2.0 ** -16)


@pytest.mark.parametrize("q_len", [1, 130, 800])
def test_attention_window_offsets_past_32_bits(q_len):
    """A cache whose later rows lie more than 2^32 bytes in."""
    rows, hk, d = 1_300_000, 8, 128
    cache = torch.empty((rows, 2 * hk * d), dtype=torch.float16, device="cuda")
    assert cache.numel() > 2 ** 31
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    n, start = 900, rows - 901
    cache[start:start + n] = torch.randn((n, 2 * hk * d), generator=g, device="cuda").half()
    k = torch.as_strided(cache, (rows, hk, d), (2 * hk * d, d, 1))
    v = torch.as_strided(cache, (rows, hk, d), (2 * hk * d, d, 1), hk * d)
    q = torch.randn((q_len, hk, d), generator=g, device="cuda").half()
    got = ref.attention(q, k, v, [0, q_len], [start], [n], 300, 0, 4)
    ref.check_attention(q, k, v, [0, q_len], [start], [n], 300, 0, 4, got)


# --- how they are called ---------------------------------------------------------

def test_repeats_streams_and_graphs_give_the_same_bits(gen):
    x, r, w = normal(gen, 50, 2048, dt=F16), normal(gen, 50, 2048, dt=F16), normal(gen, 2048)
    wx, xs, wq, s, z = w4_inputs(gen, E4M3, 3, 1024, 4096, 64, True, F16, 128)
    w4, z4 = ref.pack4(wq), ref.pack4(z)
    q, k, v = (normal(gen, n, 8, 128, dt=F16) for n in (1300, 2000, 2000))
    q1 = q[:2].contiguous()
    offs = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, 1300], [0], [2000], [0, 2])]
    pos = torch.arange(1300, device="cuda", dtype=torch.int32)
    freq, mag = inv_freq(0, 1e6, 128, 1.0, 0.0, 0.0, 0.0)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def buffers():
        return {"sum": torch.zeros_like(x), "q8": torch.zeros((50, 2048), dtype=torch.int8, device="cuda"),
                "sc": torch.zeros((50, 16), device="cuda"), "y": torch.zeros((3, 1024), device="cuda"),
                "ro": torch.zeros_like(q), "at": torch.zeros_like(q), "a1": torch.zeros_like(q1)}

    def all_of(b):
        L, st = load_library(), ref.stream()
        check(L.nemo_op_rmsnorm_q8(F16, x.data_ptr(), 2048, r.data_ptr(), 2048, w.data_ptr(), 50, 2048, 1e-5,
                                   b["sum"].data_ptr(), 2048, I8, 128, b["q8"].data_ptr(), 2048, b["sc"].data_ptr(), st))
        check(L.nemo_op_w4_matvec(E4M3, wx.data_ptr(), 4096, xs.data_ptr(), 128, w4.data_ptr(), F16, s.data_ptr(),
                                  z4.data_ptr(), 64, 3, 1024, 4096, F32, b["y"].data_ptr(), 1024, st))
        check(L.nemo_op_rope_apply(F16, 0, q.data_ptr(), 1024, 8, None, 0, 0, 128, 128, freq.data_ptr(), mag,
                                   pos.data_ptr(), 1300, b["ro"].data_ptr(), 1024, None, 0, st))
        for qq, off, n, o in ((b["ro"], offs[0], 1300, b["at"]), (q1, offs[3], 2, b["a1"])):
            check(L.nemo_op_attention_window(F16, qq.data_ptr(), 1024, k.data_ptr(), 1024, v.data_ptr(), 1024, 8, 8,
                                             128, off.data_ptr(), offs[1].data_ptr(), offs[2].data_ptr(), 1, n, 2000,
                                             n, 2000, 700, 0, 4, 0.08, o.data_ptr(), 1024, err.data_ptr(), st))

    want = buffers()
    all_of(want)
    torch.cuda.synchronize()
    a, b = buffers(), buffers()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):  # two calls at once
        for side, buf in zip(streams, (a, b)):
            with torch.cuda.stream(side):
                all_of(buf)
    torch.cuda.synchronize()
    graphs, bufs = [], [buffers(), buffers()]
    for buf in bufs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            all_of(buf)
        graphs.append(graph)
    for side, graph in zip(streams, graphs):  # two captured runs at once
        with torch.cuda.stream(side):
            graph.replay()
    torch.cuda.synchronize()
    for got in (a, b, *bufs):
        for name in want:
            assert torch.equal(got[name], want[name]), name
    assert int(err) == 0


def test_first_calls_inside_a_capture():
    """A process whose first calls are captured, which is when the kernels are loaded and given their shared memory."""
    program = """
import torch, layer_ops_ref as ref
from nemo_b200.runtime import check, load_library
L = load_library()
f = lambda *n: torch.ones(n, dtype=torch.float16, device="cuda")
x, w, y, o = f(2, 256), torch.ones(256, device="cuda"), f(2, 256), f(700, 256)
q8, sc = torch.zeros((2, 256), dtype=torch.int8, device="cuda"), torch.zeros((2, 2), device="cuda")
w4, s = torch.full((256, 128), 0x99, dtype=torch.uint8, device="cuda"), f(256, 2)
kv, off, i = f(700, 256), [torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, 2], [0, 700])], 0
pos, freq = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda")
start, n = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), 700, dtype=torch.int32, device="cuda")
err = torch.zeros(1, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    st = ref.stream()
    check(L.nemo_op_rmsnorm_q8(0, x.data_ptr(), 256, None, 0, w.data_ptr(), 2, 256, 0.0, None, 0, 4, 128, q8.data_ptr(),
                               256, sc.data_ptr(), st))
    check(L.nemo_op_w4_matvec(4, q8.data_ptr(), 256, sc.data_ptr(), 128, w4.data_ptr(), 0, s.data_ptr(), None, 128, 2,
                              256, 256, 0, y.data_ptr(), 256, st))
    check(L.nemo_op_rope_apply(0, 0, y.data_ptr(), 256, 4, None, 0, 0, 64, 64, freq.data_ptr(), 1.0, pos.data_ptr(), 2,
                               y.data_ptr(), 256, None, 0, st))
    for qq, rows, qo in ((y, 2, off[0]), (kv, 700, off[1])):
        check(L.nemo_op_attention_window(0, qq.data_ptr(), 256, kv.data_ptr(), 256, kv.data_ptr(), 256, 4, 4, 64,
                                         qo.data_ptr(), start.data_ptr(), n.data_ptr(), 1, rows, 700, rows, 700, -1, 0,
                                         0, 0.125, o.data_ptr(), 256, err.data_ptr(), st))
g.replay()
torch.cuda.synchronize()
assert (q8 == 127).all() and int(err) == 0 and (o == 1).all()
# 256 columns of 127 * (1 / 127) * (9 - 8)
assert ((y.float() - 256).abs() <= 256 * 2.0 ** -11).all()
print("captured")
"""
    run = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300,
                         env={**os.environ, "PYTHONPATH": ":".join(p for p in sys.path if p)})
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]


def test_two_host_threads_at_once(gen):
    """Calls from two threads on their own streams, refused ones among them: each gets its results and its message."""
    args = packed(gen, F16, [5, 300], [400, 300], 4, 2, 64)
    x, w = normal(gen, 40, 1000, dt=F16), normal(gen, 1000)
    want = ref.attention(*args, 50, 0, 1), ref.rmsnorm_q8(x, None, w, 1e-5, I8, 128)[1]
    wrong = []

    def work(first):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(20):
                    if (i + first) % 2:
                        if not torch.equal(ref.attention(*args, 50, 0, 1), want[0]):
                            wrong.append("attention")
                        with pytest.raises(NemoError, match="head_dim"):
                            ref.attention(*[t[..., :32] for t in args[:3]], *args[3:], 50, 0, 1)
                    else:
                        if not torch.equal(ref.rmsnorm_q8(x, None, w, 1e-5, I8, 128)[1], want[1]):
                            wrong.append("norm")
                        with pytest.raises(NemoError, match="group"):
                            ref.rmsnorm_q8(x, None, w, 1e-5, I8, 48)
        except BaseException as e:  # a failed check of this thread
            wrong.append(repr(e))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_host_memory_is_refused(gen):
    host = np.zeros(4096, np.float16)
    x, w = normal(gen, 1, 64, dt=F16), normal(gen, 64)
    q, sc = torch.zeros((1, 64), dtype=torch.int8, device="cuda"), torch.zeros((1, 1), device="cuda")
    with pytest.raises(NemoError, match="not device memory"):
        check(load_library().nemo_op_rmsnorm_q8(F16, host.ctypes.data, 64, None, 0, w.data_ptr(), 1, 64, 1e-5, None, 0,
                                                I8, 0, q.data_ptr(), 64, sc.data_ptr(), None))
    _, got, _ = ref.rmsnorm_q8(x, None, w, 1e-5, I8, 0)  # and the next call is served
    assert got.any()


@pytest.mark.parametrize("captured", [False, True], ids=["eager", "graph"])
def test_one_layer_step(gen, captured):
    """The operators as a layer of a served model runs them, each checked against its 64-bit form on the inputs that
    it had: residual norm to 8 bits, QKV projection, rotation into the cache, windowed attention, output projection."""
    tokens, width, hq, hk, d, cap = 3, 1024, 8, 2, 128, 600
    lens = [600, 1, 250]  # keys of each request with its new token
    qkv_w = (hq + 2 * hk) * d
    x, r, w = normal(gen, tokens, width, dt=BF16), normal(gen, tokens, width, dt=BF16), 1 + 0.1 * normal(gen, width)
    pq = torch.randint(0, 16, (qkv_w, width), generator=gen, device="cuda")
    ps = (0.02 * normal(gen, qkv_w, width // 64)).bfloat16()
    oq = torch.randint(0, 16, (width, hq * d), generator=gen, device="cuda")
    os_ = (0.02 * normal(gen, width, hq * d // 128)).bfloat16()
    pw, ow = ref.pack4(pq), ref.pack4(oq)
    cache_k, cache_v = (normal(gen, tokens * cap, hk, d, dt=BF16) for _ in range(2))
    freq, mag = inv_freq(1, 1e6, d, 4.0, 0.0, 0.0, 0.0)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")
    q_off = torch.arange(tokens + 1, dtype=torch.int32, device="cuda")
    start = torch.arange(tokens, dtype=torch.int32, device="cuda") * cap
    k_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
    rows = (start + pos).long()
    total, q8 = torch.empty_like(x), torch.empty((tokens, width), dtype=torch.float8_e4m3fn, device="cuda")
    sc = torch.empty((tokens, width // 128), device="cuda")
    qkv = torch.empty((tokens, qkv_w), dtype=torch.bfloat16, device="cuda")
    turned = torch.empty((tokens, (hq + hk) * d), dtype=torch.bfloat16, device="cuda")
    att = torch.empty((tokens, hq * d), dtype=torch.bfloat16, device="cuda")
    y = torch.empty((tokens, width), dtype=torch.bfloat16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def step():
        L, st = load_library(), ref.stream()
        check(L.nemo_op_rmsnorm_q8(BF16, x.data_ptr(), width, r.data_ptr(), width, w.data_ptr(), tokens, width, 1e-5,
                                   total.data_ptr(), width, E4M3, 128, q8.data_ptr(), width, sc.data_ptr(), st))
        check(L.nemo_op_w4_matvec(E4M3, q8.data_ptr(), width, sc.data_ptr(), 128, pw.data_ptr(), BF16, ps.data_ptr(),
                                  None, 64, tokens, qkv_w, width, BF16, qkv.data_ptr(), qkv_w, st))
        check(L.nemo_op_rope_apply(BF16, 1, qkv.data_ptr(), qkv_w, hq, qkv.data_ptr() + 2 * hq * d, qkv_w, hk, d, d,
                                   freq.data_ptr(), mag, pos.data_ptr(), tokens, turned.data_ptr(), (hq + hk) * d,
                                   turned.data_ptr() + 2 * hq * d, (hq + hk) * d, st))
        cache_k[rows] = turned[:, hq * d:].view(tokens, hk, d)
        cache_v[rows] = qkv[:, (hq + hk) * d:].view(tokens, hk, d)
        check(L.nemo_op_attention_window(BF16, turned.data_ptr(), (hq + hk) * d, cache_k.data_ptr(), hk * d,
                                         cache_v.data_ptr(), hk * d, hq, hk, d, q_off.data_ptr(), start.data_ptr(),
                                         k_len.data_ptr(), tokens, tokens, tokens * cap, 1, cap, 255, 0, 4, d ** -0.5,
                                         att.data_ptr(), hq * d, err.data_ptr(), st))
        check(L.nemo_op_w4_matvec(BF16, att.data_ptr(), hq * d, None, 0, ow.data_ptr(), BF16, os_.data_ptr(), None,
                                  128, tokens, width, hq * d, BF16, y.data_ptr(), width, st))

    step()
    if captured:
        first = y.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, first)
    torch.cuda.synchronize()
    ref.check_rmsnorm_q8(x, r, w, 1e-5, E4M3, 128, (total, q8, sc))
    ref.check_w4(q8, sc, 128, pq, ps, None, 64, qkv, BF16)
    ref.check_rope(qkv[:, :hq * d].view(tokens, hq, d), freq, mag, pos, d, 1, turned[:, :hq * d].view(tokens, hq, d))
    ref.check_rope(qkv[:, hq * d:(hq + hk) * d].view(tokens, hk, d), freq, mag, pos, d, 1,
                   turned[:, hq * d:].view(tokens, hk, d))
    ref.check_attention(turned[:, :hq * d].view(tokens, hq, d), cache_k, cache_v, [0, 1, 2, 3], start.tolist(), lens,
                        255, 0, 4, att.view(tokens, hq, d))
    ref.check_w4(att, None, 0, oq, os_, None, 128, y, BF16)
    assert int(err) == 0
