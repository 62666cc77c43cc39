"""Refusals, sizes and tables of the token-model operators (no GPU: every call
here ends before any device work), and the integer restatement against a
float64 recurrence."""
import ctypes

import numpy as np
import pytest

from tests import token_ref as R

ARG = 1


def q4(ddg, K=64, N=8, group=32, q=256, step=256, b=None):
    return ddg.Q4Weights(K, N, group, q, step, b)


def la(ddg, batch=1, heads=2, tokens=5, dk=4, dv=3, chunk=4, pow_n=5):
    return ddg.LinattnShape(batch, heads, tokens, dk, dv, chunk, pow_n)


@pytest.mark.parametrize("kw", [dict(K=-1), dict(N=-1), dict(group=0), dict(group=48), dict(q=None), dict(step=None),
                                dict(q=264), dict(step=257)])
def test_fc_q4_refuses_bad_weights(ddg, kw):
    assert ddg.lib().ddg_fc_q4_share(32, 0, 2, q4(ddg, **kw), 256, 64, 256, 256, None) == ARG


@pytest.mark.parametrize("bw,party,M,ldx,x,c,out", [(16, 0, 2, 64, 256, 256, 256), (32, 2, 2, 64, 256, 256, 256),
                                                    (32, 0, -1, 64, 256, 256, 256), (32, 0, 2, 63, 256, 256, 256),
                                                    (32, 0, 2, 64, None, 256, 256), (32, 0, 2, 64, 256, None, 256),
                                                    (64, 1, 2, 64, 256, 256, None)])
def test_fc_q4_refuses_bad_arguments(ddg, bw, party, M, ldx, x, c, out):
    assert ddg.lib().ddg_fc_q4_share(bw, party, M, q4(ddg), x, ldx, c, out, None) == ARG


def test_fc_q4_null_weights_and_empty_calls(ddg):
    L = ddg.lib()
    assert L.ddg_fc_q4_share(32, 0, 2, None, 256, 64, 256, 256, None) == ARG
    assert L.ddg_fc_q4_share(32, 0, 0, q4(ddg), None, 64, None, None, None) == 0
    assert L.ddg_fc_q4_share(32, 0, 4, q4(ddg, N=0, q=None, step=None), None, 64, None, None, None) == 0
    assert L.ddg_q4_quantize(64, 8, 31, 256, 256, 256, None) == ARG
    assert L.ddg_q4_quantize(64, 8, 32, None, 256, 256, None) == ARG
    assert [int(L.ddg_q4_row_bytes(k)) for k in (-1, 0, 1, 32, 33)] == [0, 0, 16, 16, 32]


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(heads=0), dict(tokens=-1), dict(dk=0), dict(dk=129), dict(dv=0),
                                dict(dv=129), dict(chunk=0), dict(chunk=129), dict(pow_n=4),
                                dict(tokens=0, pow_n=0), dict(tokens=8193, pow_n=8193), dict(tokens=2049, pow_n=2049, chunk=1), dict(batch=1 << 30, heads=1 << 20, tokens=1 << 30,
                                                              pow_n=1 << 30)])
def test_linattn_refuses_bad_shapes(ddg, kw):
    L, s = ddg.lib(), la(ddg, **kw)
    p = [256] * 12
    assert L.ddg_linattn_sizes(s, (ctypes.c_int64 * 6)()) == ARG
    assert L.ddg_linattn_decay(32, s, 1 << 40, *p[:3], None) == ARG
    assert L.ddg_linattn_carry(32, s, *p[:4], None) == ARG
    assert L.ddg_linattn_chunk_share(32, 0, s, 1 << 40, *p[:6], None) == ARG
    assert L.ddg_linattn_output_share(32, 0, s, 1 << 40, *p[:10], None) == ARG
    assert L.ddg_linattn_step_share(32, 0, s, 1 << 40, *p[:7], None) == ARG
    assert L.ddg_linattn_key_bytes(32, 12, s, 0) == 0


def test_linattn_refuses_bad_arguments(ddg):
    L, s = ddg.lib(), la(ddg)
    w = 2 * (4 + 4 + 3)
    p = [256] * 12
    assert L.ddg_linattn_chunk_share(32, 0, s, w - 1, *p[:6], None) == ARG  # rows overlap
    assert L.ddg_linattn_chunk_share(48, 0, s, w, *p[:6], None) == ARG
    assert L.ddg_linattn_chunk_share(32, 2, s, w, *p[:6], None) == ARG
    for i in range(6):
        a = p[:6]
        a[i] = None
        assert L.ddg_linattn_chunk_share(32, 0, s, w, *a, None) == ARG
    assert L.ddg_linattn_output_share(32, 0, s, w, *p[:6], 256, None, 256, 256, None) == ARG  # s0 without its mask share
    assert L.ddg_linattn_output_share(32, 0, s, w, *p[:6], None, 256, 256, 256, None) == ARG
    for fn in (L.ddg_linattn_step_share, L.ddg_linattn_step_output_share):
        n = len(fn.argtypes) - 5
        assert fn(32, 0, s, w, *p[:n], None) == ARG  # five tokens
        one = la(ddg, tokens=1)
        for i in range(n):
            a = p[:n]
            a[i] = None
            assert fn(32, 0, one, w, *a, None) == ARG
    assert L.ddg_linattn_decay(32, s, w, None, 256, 256, None) == ARG
    assert L.ddg_linattn_carry(32, s, 256, None, None, 256, None) == ARG
    # nothing to do: no pointer is looked at
    for empty in (la(ddg, batch=0), la(ddg, tokens=0)):
        assert L.ddg_linattn_chunk_share(32, 0, empty, w, *([None] * 6), None) == 0
        assert L.ddg_linattn_output_share(64, 1, empty, w, *([None] * 10), None) == 0
        assert L.ddg_linattn_decay(64, empty, w, None, None, None, None) == 0
        assert L.ddg_linattn_carry(64, empty, None, None, None, None, None) == 0


def test_misaligned_arrays_are_refused(ddg):
    """A ring array off its element boundary would fault in a kernel: refused on the host, pointer by pointer."""
    L, s, one, w = ddg.lib(), la(ddg), la(ddg, tokens=1), 22
    for bw, off in ((32, 2), (64, 4)):
        bad = 256 + off
        for i in range(3):
            a = [256, 256, 256]
            a[i] = bad
            assert L.ddg_fc_q4_share(bw, 0, 2, q4(ddg), a[0], 64, a[1], a[2], None) == ARG
        assert L.ddg_fc_q4_share(bw, 0, 2, q4(ddg, b=bad), 256, 64, 256, 256, None) == ARG
        calls = ((L.ddg_linattn_chunk_share, 6, s), (L.ddg_linattn_output_share, 10, s),
                 (L.ddg_linattn_step_share, 7, one), (L.ddg_linattn_step_output_share, 7, one))
        for fn, n, shape in calls:
            for i in range(n):
                a = [256] * n
                a[i] = bad
                assert fn(bw, 0, shape, w, *a, None) == ARG, (fn, i)
        for i in range(3):
            a = [256, 256, 256]
            a[i] = bad
            assert L.ddg_linattn_decay(bw, s, w, *a, None) == ARG
        for i in range(4):
            a = [256] * 4
            a[i] = bad
            assert L.ddg_linattn_carry(bw, s, *a, None) == ARG
    assert L.ddg_q4_quantize(64, 8, 32, 260, 256, 256, None) == ARG


def test_linattn_sizes(ddg):
    s = R.Shape(2, 3, 11, 5, 7, 4)
    got = ddg.linattn_sizes(ddg.LinattnShape(2, 3, 11, 5, 7, 4, 11))
    assert got == {"qkv": 2 * 11 * s.width, "qkd": 2 * s.n_decayed, "ps": s.n_ps, "state": s.n_state,
                   "step": s.n_state + 6 * 8, "out": 2 * 11 * 3 * 7}


@pytest.mark.parametrize("bw", [32, 64])
def test_decay_table(ddg, bw):
    lam = [0.0, 0.5, 0.96875, 1.0, 1 / 3]
    t = ddg.decay_table(bw, 12, lam, 40)
    assert t.shape == (5, 41) and t.dtype == (np.uint32 if bw == 32 else np.uint64)
    want = np.array([[1.0 * l ** i for i in range(41)] for l in lam]) * 4096
    # rounded to nearest (half a unit) of powers whose 40 products err far less than that
    assert np.all(np.abs(t.astype(np.float64) - want) <= 0.5 + 1e-9)
    assert t[0].tolist() == [4096] + [0] * 40 and set(t[3].tolist()) == {4096}
    L = ddg.lib()
    buf = (ctypes.c_uint64 * 8)()
    for bad in (-0.1, 1.5, float("nan")):
        assert L.ddg_decay_table(32, 12, 1, 3, (ctypes.c_double * 1)(bad), buf) == ARG
    assert L.ddg_decay_table(32, 31, 1, 3, (ctypes.c_double * 1)(0.5), buf) == ARG
    assert L.ddg_decay_table(32, 12, 1, -1, (ctypes.c_double * 1)(0.5), buf) == ARG
    assert L.ddg_decay_table(32, 12, 1, 3, None, buf) == ARG


def test_wire_calls_refuse_without_a_gpu(ddg):
    L, c = ddg.lib(), ddg.Cursor()
    w, m = ddg.Wire(None, 0, None), ddg.MaskWire(None, 0, None, None)
    assert L.ddg_op_fc_q4_eval(None, c, q4(ddg), 1, 0, w, w) == ARG
    assert L.ddg_op_fc_q4_keygen(None, c, q4(ddg), 1, 0, m, m) == ARG
    assert L.ddg_linattn_eval(None, c, la(ddg), 256, w, None, w, w) == ARG
    assert L.ddg_linattn_keygen(None, c, la(ddg), 256, m, None, m, m) == ARG
    assert L.ddg_linattn_step_eval(None, c, la(ddg), 256, w, w, w, w) == ARG
    assert L.ddg_linattn_step_keygen(None, c, la(ddg), 256, m, m, m, m) == ARG
    assert L.ddg_op_fc_q4_key_bytes(32, 12, 64, 8, 2, ddg.ACT_NONE) == 256
    assert L.ddg_op_fc_q4_key_bytes(32, 12, 64, 8, 2, 4) == 0
    assert L.ddg_op_fc_q4_key_bytes(32, 30, 64, 8, 2, ddg.ACT_FLOOR) == 0
    assert L.ddg_op_fc_q4_key_bytes(48, 12, 64, 8, 2, ddg.ACT_NONE) == 0
    floor, trunc = (L.ddg_op_fc_q4_key_bytes(32, 12, 64, 1000, 2, a) for a in (ddg.ACT_FLOOR, ddg.ACT_TRUNC))
    assert 0 < floor < trunc / 5
    assert L.ddg_linattn_step_key_bytes(32, 12, la(ddg)) == 0  # five tokens
    assert L.ddg_linattn_step_key_bytes(32, 12, la(ddg, tokens=1)) > 0
    assert L.ddg_linattn_key_bytes(32, 12, la(ddg), 1) > L.ddg_linattn_key_bytes(32, 12, la(ddg), 0) > 0


def test_restatement_follows_the_recurrence(ddg):
    """The integer prompt and steps track S_t = lambda S + k v^T, o = q S in float64.  Every floor
    errs by at most one unit of 2^-scale, every table entry by half a unit, and |q|, |k|, |v| <= 1:
    P, S' and the carried state are sums of at most `chunk` (4) or 3 chunk terms, so no output has
    taken more than (dk + 16) x 8 x 4 units of error in these sizes."""
    scale, bw = 20, 64
    s = R.Shape(1, 2, 11, 5, 3, 4)
    rng = np.random.default_rng(0)
    lam = np.array([0.9, 0.75])
    x = rng.uniform(-1, 1, (1, 11, s.width))
    xi = np.round(x * 2**scale).astype(np.int64)
    pow_ = ddg.decay_table(bw, scale, lam, 11)
    o, S = R.clear_prompt(s, pow_, xi.view(np.uint64), None, scale, bw)
    one = R.Shape(1, 2, 1, 5, 3, 4)
    q, k, v = (i.view(np.int64) / 2**scale for i in s.heads(xi.view(np.uint64)))
    Sf, want = np.zeros((1, 2, 5, 3)), []
    Si, steps = np.zeros(one.n_state, np.uint64), []
    for t in range(11):
        Sf = lam[None, :, None, None] * Sf + k[:, :, t, :, None] * v[:, :, t, None, :]
        want.append((q[:, :, t, None] @ Sf)[:, :, 0])
        oi, Si = R.clear_step(one, pow_[:, 1], xi.view(np.uint64)[:, t:t + 1], Si, scale, bw)
        steps.append(oi.view(np.int64).reshape(1, 2, 3) / 2**scale)
    tol = (5 + 16) * 8 * 4 / 2**scale
    assert np.max(np.abs(o.view(np.int64).reshape(1, 11, 2, 3).transpose(0, 2, 1, 3) / 2**scale
                         - np.stack(want, 2))) < tol
    assert np.max(np.abs(np.stack(steps, 2) - np.stack(want, 2))) < tol
    for got in (S, Si):
        assert np.max(np.abs(got.view(np.int64).reshape(Sf.shape) / 2**scale - Sf)) < tol


@pytest.mark.parametrize("party", [0, 1])
@pytest.mark.parametrize("bw,M,K", [(32, 2, (1 << 18) + 1), (64, 2, (1 << 18) + 1), (32, 65535 * 64 + 1, 64),
                                    (64, 65535 * 32 + 1, 64)])
def test_fc_q4_overlong_calls_are_refused_alike(ddg, party, bw, M, K):
    # party 1 multiplies nothing, but has to give its peer's answer
    L = ddg.lib()
    assert L.ddg_fc_q4_share(bw, party, M, q4(ddg, K=K), 256, K, 256, 256, None) == ARG
    assert L.ddg_op_fc_q4_key_bytes(bw, 12, K, 8, M, ddg.ACT_NONE) == 0
