"""The layer operators of include/nemo_ops.h at the ends of their ranges: the smallest and largest values of a type,
infinities in long prompts, long caches, and launch shapes between those of test_gpu_layer_ops.py."""
import ctypes
import math

import numpy as np
import pytest
import torch

import layer_ops_ref as ref
from layer_ops_ref import BF16, E4M3, F16, F32, I8, TORCH
from nemo_b200.runtime import check, load_library

pytestmark = pytest.mark.gpu


@pytest.fixture
def gen():
    g = torch.Generator(device="cuda")
    g.manual_seed(78)
    return g


# --- rmsnorm_q8, rope_apply ------------------------------------------------------

@pytest.mark.parametrize("dt,out", [(F16, I8), (BF16, E4M3)], ids=["f16_i8", "bf16_e4m3"])
@pytest.mark.parametrize("rows,width", [(3, 264), (7, 512), (5, 765), (9, 768), (301, 1536), (151, 1100), (150, 20000)])
def test_rmsnorm_q8_of_two_three_and_more_warps_a_row(gen, dt, out, rows, width):
    """Blocks of several rows with a row missing at the end, and two or four vectors a thread."""
    x, r = ((3 * torch.randn((rows, width), generator=gen, device="cuda")).to(TORCH[dt]) for _ in range(2))
    w = 1 + 0.2 * torch.randn(width, generator=gen, device="cuda")
    for group in (0, 32, 128):
        ref.check_rmsnorm_q8(x, r, w, 1e-5, out, group, ref.rmsnorm_q8(x, r, w, 1e-5, out, group))


@pytest.mark.parametrize("layout", [0, 1], ids=["pairs", "halves"])
@pytest.mark.parametrize("pad", [0, 8, 1])
@pytest.mark.parametrize("tokens", [1184, 1185, 2500])
def test_rope_apply_of_many_tokens(gen, layout, pad, tokens):
    """From eight tokens an SM on a block has fewer threads; rows that are 16 bytes apart or not."""
    hq, hk, d, rotary = 6, 2, 64, 32
    rows = torch.randn((tokens, (hq + hk) * d + pad), generator=gen, device="cuda").half()
    ld = rows.stride(0)
    q = torch.as_strided(rows, (tokens, hq, d), (ld, d, 1))
    k = torch.as_strided(rows, (tokens, hk, d), (ld, d, 1), hq * d)
    freq = torch.from_numpy(1e6 ** (-np.arange(0, rotary, 2) / rotary)).cuda()
    pos = torch.randint(0, 40000, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    qo, ko = ref.rope_apply(q, k, freq, 1.0, pos, rotary, layout)
    ref.check_rope(q, freq, 1.0, pos, rotary, layout, qo)
    ref.check_rope(k, freq, 1.0, pos, rotary, layout, ko)


# --- w4_matvec -------------------------------------------------------------------

@pytest.mark.parametrize("m,n", [(1, 50000), (2, 50000), (3, 500)])
@pytest.mark.parametrize("shift", [-96, -110, -122])
def test_w4_matvec_of_the_smallest_bf16_values(gen, shift, m, n):
    """Rows whose largest element is near 2^shift, down to subnormal ones. As check_w4, but without an absolute term
    other than that of subnormal f32 sums: 2^-150 for each of at most 4 products a segment and 64 more additions."""
    k, group = 1024, 128
    x = torch.randn((m, k), generator=gen, device="cuda", dtype=torch.float64)
    x = (x * 2.0 ** (shift + torch.randint(-10, 1, (m, k), generator=gen, device="cuda"))).bfloat16()
    q = torch.randint(0, 16, (n, k), generator=gen, device="cuda")
    z = torch.randint(0, 16, (n, k // group), generator=gen, device="cuda")
    s = (4 * torch.randn((n, k // group), generator=gen, device="cuda")).half()
    y = ref.w4_matvec(x, None, 0, ref.pack4(q), s, ref.pack4(z), group, n, F32)
    w = (q.double() - z.double().repeat_interleave(group, 1)) * s.double().repeat_interleave(group, 1)
    want, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    segments = k // group
    slack = (40 + segments / 4) * 2 * ref.U32 * mag + (64 + 4 * segments) * 2.0 ** -150
    ref.close(y, want, ref.U32 * want.abs() + slack)


# --- attention_window ------------------------------------------------------------

def milliseconds(call):
    """The shortest of five, so that a pause of the host between the events does not count."""
    call()
    times = []
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("q_len", [4, 8192])
def test_attention_window_one_bad_value_does_not_stall_a_long_call(gen, q_len, bad):
    """One infinite or NaN element in the first value row, which every query sees: its column is lost, the other
    columns keep their values, and the call takes a few times as long as on clean values (a warp that walked key by
    key over every row took several hundred times)."""
    n, hq, hk, d = 8192, 24, 8, 128
    q = torch.randn((q_len, hq, d), generator=gen, device="cuda").half()
    k, v = (torch.randn((n, hk, d), generator=gen, device="cuda").half() for _ in range(2))
    v[7000] = 0
    args = (q, k, v, [0, q_len], [0], [n], -1, 0, 0)
    clean = ref.attention(*args)
    usual = milliseconds(lambda: ref.attention(*args))
    v[0, 3, 77] = bad
    got = ref.attention(*args)
    took = milliseconds(lambda: ref.attention(*args))
    lost = torch.zeros((hq, d), dtype=torch.bool, device="cuda")
    lost[9:12, 77] = True
    print(f"clean {usual:.3f} ms, with one bad value {took:.3f} ms")
    assert torch.equal(~torch.isfinite(got), lost.expand_as(got))
    assert torch.equal(got[:, ~lost], clean[:, ~lost])
    assert took < 20 * usual


@pytest.mark.parametrize("q_len", [4, 8192])
def test_attention_window_one_bad_key_does_not_stall_a_long_call(gen, q_len):
    n, hq, hk, d = 8192, 24, 8, 128
    q = torch.randn((q_len, hq, d), generator=gen, device="cuda").half()
    k, v = (torch.randn((n, hk, d), generator=gen, device="cuda").half() for _ in range(2))
    args = (q, k, v, [0, q_len], [0], [n], -1, -1, 0)
    clean = ref.attention(*args)
    usual = milliseconds(lambda: ref.attention(*args))
    k[n - 1, 5, 0] = math.nan
    got = ref.attention(*args)
    took = milliseconds(lambda: ref.attention(*args))
    print(f"clean {usual:.3f} ms, with one bad key {took:.3f} ms")
    assert torch.isnan(got[:, 15:18]).all()
    assert torch.equal(got[:, :15], clean[:, :15]) and torch.equal(got[:, 18:], clean[:, 18:])
    assert took < 20 * usual


@pytest.mark.parametrize("dt", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("q_len", [3, 1500])
def test_attention_window_infinities_and_nan_where_rows_see_them_and_not(gen, dt, q_len):
    """Bad values of some columns, of either sign, near one another, some of them out of the sight of some queries or
    of all: each result is what the sum of the visible keys' terms is, and clean columns are those of clean values."""
    n, hq, hk, d = 1500, 4, 2, 64
    q = torch.randn((q_len, hq, d), generator=gen, device="cuda").to(TORCH[dt])
    k, v = (torch.randn((n, hk, d), generator=gen, device="cuda").to(TORCH[dt]) for _ in range(2))
    left, right, sinks = 60, 3, 2
    args = (q, k, v, [0, q_len], [0], [n], left, right, sinks)
    clean = ref.attention(*args)
    for j, h, c, x in ((0, 0, 1, math.inf), (1, 0, 2, math.nan), (5, 0, 3, math.inf), (700, 1, 4, -math.inf),
                       (700, 1, 5, math.nan), (703, 1, 4, math.inf), (710, 1, 6, math.inf), (1498, 0, 63, -math.inf),
                       (1499, 1, 62, math.nan), (1497, 1, slice(None), math.inf)):
        v[j, h, c] = x
    got = ref.attention(*args)
    ok = ref.seen(q_len, n, left, right, sinks).double()
    for h in range(hq):
        # counts of the +infinite, -infinite and NaN terms that each result has
        up, down, nan = (ok @ (f(v[:, h // 2])).double() for f in (torch.isposinf, torch.isneginf, torch.isnan))
        want = torch.where(nan + up * down > 0, math.nan, torch.where(up > 0, math.inf, -math.inf))
        want = torch.where(nan + up + down > 0, want, 0.0).to(got.dtype)
        have = torch.where(torch.isfinite(got[:, h]), 0, got[:, h])
        assert torch.equal(torch.nan_to_num(have, nan=7.0), torch.nan_to_num(want, nan=7.0))
        fine = torch.isfinite(got[:, h])
        ref.close(got[:, h][fine], clean[:, h][fine].double(), 4 * ref.HALF[dt] * 5)


@pytest.mark.parametrize("q_len,heads", [(1, 2), (200, 2), (1200, 8)])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_attention_window_rows_without_any_weight_are_zeros_over_bad_values(gen, q_len, heads, bad):
    n, d = 1200, 64
    q = torch.rand((q_len, heads, d), generator=gen, device="cuda").half() + 0.5
    k = torch.full((n, 1, d), -math.inf, dtype=torch.float16, device="cuda")
    v = torch.randn((n, 1, d), generator=gen, device="cuda").half()
    v[::7, :, 3] = bad
    got = ref.attention(q, k, v, [0, q_len], [0], [n], 300, 0, 2)
    assert (got == 0).all()


@pytest.mark.parametrize("dt", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("q_len,nk,heads", [(1, 300, 1), (1, 5000, 1), (300, 1200, 1), (1200, 1200, 8)])
def test_attention_window_of_the_largest_values(gen, dt, q_len, nk, heads):
    """Values at the end of the type: a weighted mean of them is no larger, so it stays finite however the weights
    round. Here 15 of 16 weights round up by nearly half a step."""
    d, top = 64, torch.finfo(TORCH[dt]).max
    q = torch.zeros((q_len, heads, d), dtype=TORCH[dt], device="cuda")
    k = torch.zeros((nk, heads, d), dtype=TORCH[dt], device="cuda")
    q[..., 0] = 1
    k[..., 0] = -1
    k[::16, :, 0] = 0
    v = torch.full((nk, heads, d), top, dtype=TORCH[dt], device="cuda")
    v[..., 1::2] *= -1
    weight = 0.5 + 0.55 * (2.0 ** -11 if dt == F16 else 2.0 ** -8)  # the type's step there is 2^-11 or 2^-8
    args = (q, k, v, [0, q_len], [0], [nk], -1, -1, 0)
    got = ref.attention(*args, scale=-math.log(weight))
    ref.check_attention(*args, got, scale=-math.log(weight))


@pytest.mark.parametrize("batch,q_len,nk,heads,warps,share", [
    (1, 1, 500000, 1, 64, 1.03), (100, 1, 400000, 8, 4, 1.02645), (1, 2048, 131072, 8, 1, 1.03)])
def test_attention_window_many_small_weights(gen, batch, q_len, nk, heads, warps, share):
    """Some first keys with half of the weight and a long cache that shares the other half: each small weight keeps
    the type's relative precision (half a step of f16 for the weights, as much for the result; and each of the
    nk / warps / 16 instructions of a chain of sums may cut off one f32 step). `warps` of the 16-row kernel share the
    keys, 16 at a time each, and begin with a large one each."""
    d = 64
    q = torch.zeros((batch * q_len, heads, d), dtype=torch.float16, device="cuda")
    k = torch.zeros((nk, heads, d), dtype=torch.float16, device="cuda")
    q[..., 0] = 1
    k[..., 0] = -1
    v = 1 + torch.rand((nk, heads, d), generator=gen, device="cuda").half()
    first = range(0, 16 * warps, 16)
    for j in first:
        k[j], v[j] = 0, 0
    args = (q, k, v, [b * q_len for b in range(batch + 1)], [0] * batch, [nk] * batch, -1, -1, 0)
    scale = math.log(share * nk / len(first))
    got = ref.attention(*args, scale=scale).double()
    w = torch.full((nk,), math.exp(-scale), dtype=torch.float64, device="cuda")
    w[list(first)] = 1
    want = torch.stack([w @ v[:, h].double() for h in range(heads)]) / w.sum()
    error = float(((got - want) / want).abs().max())
    print(f"relative error {error:.2e}")
    assert error <= 2 * 2.0 ** -11 + 2.0 ** -15 + nk / warps / 16 * 2.0 ** -23


@pytest.mark.parametrize("qs,ks", [([512, 1, 1, 1], [512, 3000, 1, 777]), ([1, 1, 2048, 0, 1], [64, 900, 2048, 5, 4000])])
def test_attention_window_of_a_prompt_among_single_tokens(gen, qs, ks):
    hq, hk, d = 24, 8, 128
    q = torch.randn((sum(qs), hq, d), generator=gen, device="cuda").half()
    k, v = (torch.randn((sum(ks), hk, d), generator=gen, device="cuda").half() for _ in range(2))
    q_off, start = [0] + np.cumsum(qs).tolist(), [0] + np.cumsum(ks).tolist()[:-1]
    got = ref.attention(q, k, v, q_off, start, ks, 1023, 0, 4)
    ref.check_attention(q, k, v, q_off, start, ks, 1023, 0, 4, got)


def window_form(hq, hk, d, batch, q_rows, k_rows, max_q, max_k, left, right, sinks):
    tiles, splits = ctypes.c_int(), ctypes.c_int()
    check(load_library().nemo_op_attention_window_form(hq, hk, d, batch, q_rows, k_rows, max_q, max_k, left, right, sinks,
                                                       148, 16, ctypes.byref(tiles), ctypes.byref(splits)))
    return tiles.value, splits.value


@pytest.mark.parametrize("dt", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [(-1, -1, 0), (-1, 0, 0), (70, 0, 3), (40, 130, 65), (100, 33, 0)],
                         ids=lambda w: "l%d_r%d_s%d" % w)
def test_attention_window_around_the_edges_of_the_tiles(gen, dt, d, window):
    """Lengths beside multiples of the 128 queries and 64 keys of a tile, one to three heads a kv head, each on the
    128-query tiles."""
    for hq, hk in ((24, 8), (8, 8)):
        qs = [127, 1, 128, 129, 0, 255, 257, 64, 320, 700, 700, 700]
        ks = [127, 64, 129, 65, 9, 256, 511, 700, 321, 700, 701, 763]
        q = torch.randn((sum(qs), hq, d), generator=gen, device="cuda").to(TORCH[dt])
        k, v = (torch.randn((sum(ks), hk, d), generator=gen, device="cuda").to(TORCH[dt]) for _ in range(2))
        assert window_form(hq, hk, d, len(qs), sum(qs), sum(ks), max(qs), max(ks), *window)[0] == 1
        q_off, start = [0] + np.cumsum(qs).tolist(), [0] + np.cumsum(ks).tolist()[:-1]
        got = ref.attention(q, k, v, q_off, start, ks, *window)
        ref.check_attention(q, k, v, q_off, start, ks, *window, got)


# --- memory ----------------------------------------------------------------------

def test_managed_memory_is_served(gen):
    rt = ctypes.CDLL("libcudart.so.12")
    x, w = torch.randn((4, 256), generator=gen, device="cuda").half(), torch.ones(256, device="cuda")
    _, want, scales = ref.rmsnorm_q8(x, None, w, 1e-5, I8, 0)
    p = ctypes.c_void_p()
    assert rt.cudaMallocManaged(ctypes.byref(p), ctypes.c_size_t(4 * 256), ctypes.c_uint(1)) == 0
    try:
        sc = torch.zeros((4, 1), device="cuda")
        check(load_library().nemo_op_rmsnorm_q8(F16, x.data_ptr(), 256, None, 0, w.data_ptr(), 4, 256, 1e-5, None, 0, I8,
                                                0, p.value, 256, sc.data_ptr(), ref.stream()))
        torch.cuda.synchronize()
        got = np.ctypeslib.as_array(ctypes.cast(p, ctypes.POINTER(ctypes.c_int8)), (4, 256)).copy()
    finally:
        torch.cuda.synchronize()
        assert rt.cudaFree(p) == 0
    assert np.array_equal(got, want.cpu().numpy()) and torch.equal(sc, scales)
