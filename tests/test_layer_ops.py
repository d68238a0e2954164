"""The layer operators' host side (include/nemo_ops.h): every refusal happens before a device is touched, and the
frequencies of nemo_rope_inv_freq are the formulas'. Runs without a GPU."""
import ctypes
import math

import numpy as np
import pytest

import oracle
from nemo_b200.runtime import load_library

P = 4096  # an address that no refused call reads
ERR_ARGS = -1


def refused(name, args, change, message):
    call = dict(args)
    call.update(change)
    L = load_library()
    assert getattr(L, name)(*call.values()) == ERR_ARGS, change
    text = L.nemo_last_error().decode()
    assert text.startswith(name) and message in text, (change, text)


NORM = dict(dtype=0, x=P, ldx=64, residual=P, ldr=64, w=P, rows=2, width=64, eps=1e-5, sum=P, lds=64, out=3, group=0,
            q=P, ldq=64, scales=P, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=2), "f16 or bf16"), (dict(out=0), "e4m3 or i8"), (dict(rows=-1), "rows"), (dict(width=0), "width"),
    (dict(width=40000, ldx=40000), "width"), (dict(group=16), "group"), (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"), (dict(x=None), "null"), (dict(scales=None), "null"), (dict(sum=None), "d_sum"),
    (dict(residual=None), "d_sum"), (dict(ldx=63), "leading"), (dict(lds=1), "leading"), (dict(ldq=63), "leading"),
    (dict(lds=72), "in place"), (dict(x=P + 1, sum=P + 64), "aligned"), (dict(w=P + 2), "aligned")])
def test_rmsnorm_q8_refuses(change, message):
    refused("nemo_op_rmsnorm_q8", NORM, change, message)


ROPE = dict(dtype=0, layout=0, q=P, ldq=128, q_heads=2, k=P, ldk=64, k_heads=1, head_dim=64, rotary=64, freq=P,
            magnitude=1.0, pos=P, tokens=3, qo=P, ldqo=128, ko=P, ldko=64, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=3), "f16 or bf16"), (dict(layout=2), "layout"), (dict(q_heads=0), "q_heads"),
    (dict(tokens=-1), "tokens"), (dict(rotary=63), "rotary_dim"), (dict(rotary=66), "rotary_dim"),
    (dict(head_dim=514, ldq=2000), "head_dim"), (dict(magnitude=math.inf), "magnitude"), (dict(k=None), "null"),
    (dict(pos=None), "null"), (dict(ldq=127), "leading"), (dict(ldko=63), "leading"), (dict(ldqo=136), "in place"),
    (dict(freq=P + 4), "aligned")])
def test_rope_apply_refuses(change, message):
    refused("nemo_op_rope_apply", ROPE, change, message)


W4 = dict(x_dtype=0, x=P, ldx=256, xs=None, x_group=0, w=P, scale_dtype=0, scales=P, zeros=None, group=128, m=1, n=5,
          k=256, y_dtype=0, y=P, ldy=5, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(x_dtype=2), "x must be"), (dict(scale_dtype=2), "scales must be"), (dict(y_dtype=3), "y must be"),
    (dict(m=17), "m must be"), (dict(m=-1), "m must be"), (dict(n=0), "positive"), (dict(group=96), "group must be"),
    (dict(k=320, ldx=320), "divide"), (dict(xs=P), "d_x_scales"), (dict(x_dtype=4), "d_x_scales"),
    (dict(x_dtype=3, xs=P, x_group=48), "x_group"), (dict(w=None), "null"), (dict(ldx=255), "leading"),
    (dict(ldy=4), "leading"), (dict(w=P + 8), "16-byte"), (dict(y_dtype=2, y=P + 2), "aligned")])
def test_w4_matvec_refuses(change, message):
    refused("nemo_op_w4_matvec", W4, change, message)


ATTN = dict(dtype=0, q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, q_heads=4, kv_heads=2, head_dim=128, q_off=P,
            k_start=P, k_len=P, batch=1, q_rows=4, k_rows=4, max_q=4, max_k=4, left=-1, right=-1, sinks=0, scale=1.0,
            out=P, ldo=512, err=P, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=2), "f16 or bf16"), (dict(head_dim=96), "head_dim"), (dict(q_heads=3), "multiple of kv_heads"),
    (dict(batch=-1), "batch"), (dict(batch=70000), "batch"), (dict(q_rows=-1), "row counts"),
    (dict(left=-2), "left"), (dict(sinks=-1), "sinks"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(q=None), "null"), (dict(err=None), "null"), (dict(v=None), "null"), (dict(ldk=248), "leading"),
    (dict(ldq=516), "multiples of 8"), (dict(out=P + 8), "16-byte"), (dict(k_len=P + 2), "aligned")])
def test_attention_window_refuses(change, message):
    refused("nemo_op_attention_window", ATTN, change, message)


def test_empty_calls_do_nothing():
    L = load_library()
    assert L.nemo_op_rmsnorm_q8(*dict(NORM, rows=0).values()) == 0
    assert L.nemo_op_rope_apply(*dict(ROPE, tokens=0).values()) == 0
    assert L.nemo_op_w4_matvec(*dict(W4, m=0).values()) == 0
    assert L.nemo_op_attention_window(*dict(ATTN, batch=0).values()) == 0
    assert L.nemo_op_attention_window(*dict(ATTN, max_q=0).values()) == 0


def frequencies(scaling, theta, rotary, factor=1.0, original=0.0, slow=0.0, fast=0.0):
    out, mag = np.zeros(rotary // 2), ctypes.c_float()
    rc = load_library().nemo_rope_inv_freq(scaling, theta, rotary, factor, original, slow, fast,
                                           out.ctypes.data_as(ctypes.c_void_p), ctypes.byref(mag))
    assert rc == 0, load_library().nemo_last_error()
    return out, mag.value


def test_inv_freq_formulas():
    theta, r = 10000.0, 64
    f = theta ** (-np.arange(0, r, 2) / r)
    got, mag = frequencies(0, theta, r)
    np.testing.assert_allclose(got, f, rtol=1e-14)
    assert mag == 1.0
    np.testing.assert_allclose(frequencies(1, theta, r, 4.0)[0], f / 4, rtol=1e-14)
    # the scaled base slows the last pair by exactly the factor and leaves the first one
    ntk, _ = frequencies(2, theta, r, 8.0)
    np.testing.assert_allclose([ntk[0], ntk[-1]], [f[0], f[-1] / 8], rtol=1e-12)
    ramp, mag = frequencies(4, 500000.0, 128, 8.0, 8192.0, 1.0, 4.0)
    f = 500000.0 ** (-np.arange(0, 128, 2) / 128)
    turns = 8192 * f / (2 * np.pi)
    assert mag == 1.0
    np.testing.assert_allclose(ramp[turns >= 4], f[turns >= 4], rtol=1e-13)
    np.testing.assert_allclose(ramp[turns <= 1], f[turns <= 1] / 8, rtol=1e-13)
    mid = (turns > 1) & (turns < 4)
    assert mid.any()
    share = (turns[mid] - 1) / 3
    np.testing.assert_allclose(ramp[mid], share * f[mid] + (1 - share) * f[mid] / 8, rtol=1e-13)


def test_inv_freq_yarn_is_the_models_table():
    got, mag = frequencies(3, 1e6, 128, 16.0, 16384.0, 1.0, 32.0)
    assert mag == pytest.approx(0.1 * math.log(16.0) + 1)
    n = 600
    table = oracle.rope_table(n)
    angle = np.arange(n)[:, None] * got
    # the table holds f32 values of the same angles
    np.testing.assert_allclose(table[..., 0], np.cos(angle), atol=2.0 ** -24 + 1e-9)
    np.testing.assert_allclose(table[..., 1], np.sin(angle), atol=2.0 ** -24 + 1e-9)


@pytest.mark.parametrize("args", [
    (5, 1e4, 64, 1.0, 1.0, 1.0, 2.0), (0, 1.0, 64, 1.0, 1.0, 1.0, 2.0), (0, 1e4, 63, 1.0, 1.0, 1.0, 2.0),
    (1, 1e4, 64, 0.5, 1.0, 1.0, 2.0), (2, 1e4, 2, 2.0, 1.0, 1.0, 2.0), (3, 1e4, 64, 2.0, 0.0, 1.0, 2.0),
    (4, 1e4, 64, 2.0, 10.0, 2.0, 2.0)])
def test_inv_freq_refuses(args):
    out, mag = np.zeros(64), ctypes.c_float()
    L = load_library()
    assert L.nemo_rope_inv_freq(*args, out.ctypes.data_as(ctypes.c_void_p), ctypes.byref(mag)) == ERR_ARGS
    assert L.nemo_last_error().startswith(b"nemo_rope_inv_freq")
    assert L.nemo_rope_inv_freq(0, 1e4, 64, 1.0, 1.0, 1.0, 2.0, None, ctypes.byref(mag)) == ERR_ARGS


def test_w4_matvec_sends_larger_batches_to_no_entry_of_other_formats():
    """nemo_op_qmatmul takes Q4_K, Q6_K, Q4_0 and tile32 weights and f16 x, none of these."""
    L = load_library()
    assert L.nemo_op_w4_matvec(*dict(W4, m=17).values()) == ERR_ARGS
    text = L.nemo_last_error().decode()
    assert "qmatmul" not in text and "each 16" in text


@pytest.mark.parametrize("theta,rotary,factor", [(1e300, 64, 1e10), (1e4, 4, 1e200)])
def test_inv_freq_refuses_a_scaled_base_that_overflows(theta, rotary, factor):
    """theta * factor^(r / (r - 2)) past the largest double: every frequency but the first would be 0."""
    out, mag = np.zeros(64), ctypes.c_float()
    L = load_library()
    assert L.nemo_rope_inv_freq(2, theta, rotary, factor, 0.0, 0.0, 0.0, out.ctypes.data_as(ctypes.c_void_p),
                                ctypes.byref(mag)) == ERR_ARGS
    assert b"scaled" in L.nemo_last_error()


def window_form(q_heads=24, kv_heads=8, head_dim=128, batch=1, q_rows=1, k_rows=8192, max_q=1, max_k=8192, left=-1,
                right=0, sinks=0, sms=148, max_cluster=16):
    tiles, splits = ctypes.c_int(), ctypes.c_int()
    rc = load_library().nemo_op_attention_window_form(q_heads, kv_heads, head_dim, batch, q_rows, k_rows, max_q, max_k,
                                                      left, right, sinks, sms, max_cluster, ctypes.byref(tiles),
                                                      ctypes.byref(splits))
    assert rc == 0, load_library().nemo_last_error()
    return tiles.value, splits.value


def test_attention_window_forms():
    """Few queries on 16-row tiles whose keys up to 16 blocks share, prompts on 128-query ones."""
    assert window_form() == (0, 16)
    assert window_form(max_k=100) == (0, 1)
    assert window_form(batch=16, q_rows=16, max_k=32768, k_rows=16 * 32768) == (0, 8)
    assert window_form(q_rows=8192, max_q=8192)[0] == 1
    assert window_form(q_rows=8192, max_q=8192, k_rows=0, max_k=0)[0] == 0


def test_attention_window_splits_fit_the_device():
    """A device that cannot place a cluster of 16, or with few SMs, gets fewer blocks a tile."""
    for cluster in (1, 2, 4, 8, 16):
        assert window_form(max_cluster=cluster) == (0, cluster)
    assert window_form(max_cluster=11) == (0, 8)
    # one tile a kv head: 8 blocks, as many again for each doubling up to two an SM, then 8 an SM of long keys
    assert window_form(max_k=1024, sms=8) == (0, 2)
    assert window_form(max_k=32768, k_rows=32768, sms=8) == (0, 8)
    L = load_library()
    assert L.nemo_op_attention_window_form(3, 2, 128, 1, 1, 1, 1, 1, -1, -1, 0, 148, 16, None, None) == ERR_ARGS


def w4_form(x_dtype, x_group, group, m, n, k, sms=148):
    out = [ctypes.c_int() for _ in range(6)]
    rc = load_library().nemo_op_w4_matvec_form(x_dtype, x_group, group, m, n, k, sms, *[ctypes.byref(v) for v in out])
    assert rc == 0, load_library().nemo_last_error()
    return dict(zip(("digits", "rows", "slices", "panels", "blocks", "shared"), [v.value for v in out]))


def test_w4_matvec_forms():
    """Up to two rows of 16-bit or e4m3 x, and i8 codes, as digits where there are many weight rows."""
    assert w4_form(0, 0, 128, 1, 131072, 2048)["digits"] == 1
    assert w4_form(1, 0, 128, 2, 50000, 1024)["digits"] == 1
    assert w4_form(0, 0, 128, 3, 131072, 2048)["digits"] == 0
    assert w4_form(4, 128, 128, 16, 131072, 2048)["digits"] == 1
    assert w4_form(0, 0, 32, 16, 3, 12320)["panels"] > 1
    L = load_library()
    assert L.nemo_op_w4_matvec_form(2, 0, 128, 1, 1, 128, 148, None, None, None, None, None, None) == ERR_ARGS


@pytest.mark.parametrize("x_dtype,x_group", [(0, 0), (3, 10 ** 9), (3, 32), (4, 64)])
def test_w4_matvec_plans_two_blocks_an_sm_only_where_two_fit(x_dtype, x_group):
    """An SM has 228 KB, of which every block takes 1 KB more than it asks for."""
    for group in (32, 64, 128):
        for m in range(1, 17):
            for k in range(group, 12000, group):
                form = w4_form(x_dtype, x_group, group, m, 200000, k)
                if form["blocks"] > 148:
                    assert 2 * (form["shared"] + 1024) <= 228 * 1024, (group, m, k, form)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("batch,q_len,k_len,tiles", [
    (16, 8, 1500, 0), (16, 32, 1500, 1), (4, 64, 4096, 1), (1, 64, 16384, 0), (1, 128, 16384, 0), (1, 256, 16384, 1),
    (8, 2, 56, 0)])
def test_attention_window_takes_the_form_that_measures_faster(head_dim, batch, q_len, k_len, tiles):
    """128 queries on 16384 keys: 206 us in 16-row tiles and 239 in 128-query ones (128 columns), 135 and 224 (64); eight
    requests of 2 on 56 keys 4.0 and 6.6."""
    form = window_form(head_dim=head_dim, batch=batch, q_rows=batch * q_len, max_q=q_len, k_rows=batch * k_len,
                       max_k=k_len)
    assert form[0] == tiles
