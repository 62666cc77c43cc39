"""Token-model operators on the GPU, bit for bit against the integer
definitions in tests/token_ref.py: fully connected layers with 4-bit weights
and linear attention with a decay per head, share by share and as wires."""
import numpy as np
import pytest

from tests import token_ref as R
from tests.gpu_util import dev_bytes, from_dev, ptr, ring_dt, to_dev
from tests.test_layers_gpu import Bufs, run_both, wire_host

pytestmark = pytest.mark.gpu
S = 12


def rnd(rng, bw, *shape):
    dt = ring_dt(bw)
    return rng.integers(0, np.iinfo(dt).max, size=shape, dtype=dt, endpoint=True)


def guarded(n, bw, before=0):
    """device buffer of n ring elements with 64 guard words behind, its fill and a checker"""
    dt = ring_dt(bw)
    host = np.full(n + 64, 0xA5A5A5A5, dtype=dt)
    d = to_dev(host)

    def read():
        got = from_dev(d, dt, n + 64)
        assert np.all(got[n:] == host[n:]), "wrote behind the output"
        return got[:n]

    return d, read


# ---------------------------------------------------------------- 4-bit weights

def fc_case(ddg, bw, M, K, N, group, *, seed=0, ldx=None, bias=True, alias=False, x=None, edge=False):
    rng = np.random.default_rng(1000 * M + 10 * K + N + group + bw + seed)
    ldx = K if ldx is None else ldx
    X = rnd(rng, bw, M, max(ldx, 1)) if x is None else x
    code = rng.integers(0, 16, size=(K, N), dtype=np.uint8)
    step = rng.integers(0, 4096, size=((K + group - 1) // group, N)).astype(np.uint16)
    if edge:
        code[:], step[:] = (0 if edge == "low" else 15), 4095
    C, b = rnd(rng, bw, M, N), rnd(rng, bw, N)
    want = R.mm(X[:, :K].astype(np.uint64), R.q4_weights(code, step, group).view(np.uint64)) + C
    if bias:
        want = want + b.astype(np.uint64)
    dq, ds, dx, dc, db = to_dev(R.q4_pack(code)), to_dev(step), to_dev(X), to_dev(C), to_dev(b)
    w = ddg.Q4Weights(K, N, group, ptr(dq), ptr(ds), ptr(db) if bias else None)
    if alias:
        ddg.fc_q4_share(bw, 0, M, w, ptr(dx), ldx, ptr(dc), ptr(dc))
        got = from_dev(dc, ring_dt(bw), M * N)
    else:
        out, read = guarded(M * N, bw)
        ddg.fc_q4_share(bw, 0, M, w, ptr(dx), ldx, ptr(dc), ptr(out))
        got = read()
    assert ddg.lib().ddg_gemm_status() == 0
    assert np.array_equal(got.reshape(M, N), R.ring(want, bw))


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("M,K,N,group", [(1, 1, 1, 32), (1, 31, 5, 32), (1, 32, 128, 32), (1, 376, 1024, 32),
                                         (2, 33, 7, 64), (3, 129, 130, 128), (4, 1000, 77, 96), (5, 64, 1, 32),
                                         (8, 500, 300, 128), (16, 1024, 129, 32), (17, 257, 255, 64),
                                         (33, 96, 640, 32), (64, 320, 256, 128), (65, 47, 131, 32),
                                         (130, 200, 200, 64), (300, 94, 188, 32)])
def test_fc_q4(ddg, cuda, bw, M, K, N, group):
    fc_case(ddg, bw, M, K, N, group)


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("M,K,N", [(1, 4096, 300), (7, 9000, 40), (40, 9000, 130)])
def test_fc_q4_long_reductions(ddg, cuda, bw, M, K, N):
    fc_case(ddg, bw, M, K, N, 128)


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("M,K,N", [(1, 4096, 9000), (1, 1023, 20001), (1, 2500, 2403), (2, 1500, 3001), (2, 2100, 7),
                                   (1, 20000, 600), (1, 30000, 50)])
def test_fc_q4_few_rows(ddg, cuda, bw, M, K, N):
    # one or two rows: every way of sharing K between the warps, several rounds of outputs
    fc_case(ddg, bw, M, K, N, 64)


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("M", [1, 6, 70])
def test_fc_q4_strided_rows_no_bias_and_in_place(ddg, cuda, bw, M):
    fc_case(ddg, bw, M, 100, 60, 32, ldx=103)
    fc_case(ddg, bw, M, 100, 60, 32, ldx=108, bias=False)
    fc_case(ddg, bw, M, 100, 60, 32, alias=True)


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("M,K", [(1, 20000), (9, 20000), (33, 20000)])
@pytest.mark.parametrize("edge", ["low", "high"])
def test_fc_q4_largest_sums(ddg, cuda, bw, M, K, edge):
    """every byte of x 255 and every weight the largest of its sign: the sums that a narrow accumulator loses"""
    fc_case(ddg, bw, M, K, 33, 32, x=np.full((M, K), np.iinfo(ring_dt(bw)).max, dtype=ring_dt(bw)), edge=edge)


@pytest.mark.parametrize("bw", [32, 64])
def test_fc_q4_empty_reduction_and_party_one(ddg, cuda, bw):
    rng = np.random.default_rng(3)
    C, b = rnd(rng, bw, 5, 9), rnd(rng, bw, 9)
    dc, db, dq = to_dev(C), to_dev(b), dev_bytes(256)
    out, read = guarded(45, bw)
    ddg.fc_q4_share(bw, 0, 5, ddg.Q4Weights(0, 9, 32, ptr(dq), ptr(dq), ptr(db)), None, 0, ptr(dc), ptr(out))
    assert np.array_equal(read().reshape(5, 9), (C + b).astype(C.dtype))
    out, read = guarded(45, bw)
    ddg.fc_q4_share(bw, 1, 5, ddg.Q4Weights(64, 9, 32, ptr(dq), ptr(dq), ptr(db)), None, 64, ptr(dc), ptr(out))
    assert np.array_equal(read().reshape(5, 9), C)


@pytest.mark.parametrize("K,N,group", [(1, 1, 32), (64, 5, 32), (100, 33, 64), (33, 200, 32)])
def test_q4_quantize(ddg, cuda, K, N, group):
    rng = np.random.default_rng(K + N)
    w = rng.integers(-4000, 4001, size=(K, N)).astype(np.int64)
    w[:, 0] = 0
    if N > 4:
        w[:, 1] = rng.integers(-60000, 60001, size=K)   # saturates
        w[0, 2], w[-1, 3] = -(1 << 63), (1 << 63) - 1
        w[:, 4] = 7
    code, step = R.q4_quantize(w, group)
    dw, dq, ds = to_dev(w), dev_bytes(N * 16 * ((K + 31) // 32)), dev_bytes(step.size * 2)
    ddg.q4_quantize(K, N, group, ptr(dw), ptr(dq), ptr(ds))
    assert np.array_equal(from_dev(ds, np.uint16, step.size).reshape(step.shape), step)
    assert np.array_equal(from_dev(dq, np.uint8, N * 16 * ((K + 31) // 32)).reshape(N, -1), R.q4_pack(code))
    inside = np.abs(w[:, 5:]).max(initial=0) <= 7 * 4095
    assert inside and np.all(2 * np.abs(R.q4_weights(code, step, group)[:, 5:] - w[:, 5:])
                             <= np.repeat(step.astype(np.int64), group, axis=0)[:K, 5:])


# ---------------------------------------------------------------- linear attention, share by share

SHAPES = [(1, 1, 1, 1, 1, 1), (1, 2, 5, 3, 2, 2), (2, 3, 130, 47, 47, 128), (1, 2, 257, 64, 64, 128),
          (1, 1, 128, 128, 128, 128), (2, 1, 300, 33, 65, 100), (1, 3, 40, 128, 17, 16), (1, 2, 127, 20, 128, 64),
          (3, 1, 7, 8, 12, 128), (1, 1, 700, 16, 16, 33)]


def la_inputs(ddg, rng, bw, shape, pad=0, extra_pow=0):
    B, H, T, dk, dv, C = shape
    s = R.Shape(*shape)
    sh = ddg.LinattnShape(B, H, T, dk, dv, C, T + extra_pow)
    pow_ = rnd(rng, bw, H, T + extra_pow + 1)
    ld = s.width + pad
    return s, sh, ld, pow_


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("shape", SHAPES)
def test_linattn_decay_and_carry(ddg, cuda, bw, shape):
    rng = np.random.default_rng(sum(shape) + bw)
    s, sh, ld, pow_ = la_inputs(ddg, rng, bw, shape, pad=5, extra_pow=3)
    x, ps, s0 = rnd(rng, bw, s.B, s.T, ld), rnd(rng, bw, s.n_ps), rnd(rng, bw, s.n_state)
    dp, dx, dps, ds0 = (to_dev(i) for i in (pow_, x, ps, s0))
    out, read = guarded(2 * s.n_decayed, bw)
    ddg.linattn_decay(bw, sh, ld, ptr(dp), ptr(dx), ptr(out))
    assert np.array_equal(read(), R.ring(R.decay(s, pow_, x), bw))
    for start, dstart in ((s0, ptr(ds0)), (None, None)):
        out, read = guarded(s.n_ps, bw)
        ddg.linattn_carry(bw, sh, ptr(dp), ptr(dps), dstart, ptr(out))
        assert np.array_equal(read(), R.ring(R.carry(s, pow_, ps, start), bw))


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("party", [0, 1])
@pytest.mark.parametrize("shape", SHAPES)
def test_linattn_chunk_and_output_shares(ddg, cuda, bw, party, shape):
    rng = np.random.default_rng(sum(shape) + bw + party)
    for pad in (0, 3):
        s, sh, ld, _ = la_inputs(ddg, rng, bw, shape, pad=pad)
        x, rx = rnd(rng, bw, s.B, s.T, ld), rnd(rng, bw, s.B, s.T, ld)
        kd, rkd = rnd(rng, bw, s.n_decayed), rnd(rng, bw, s.n_decayed)
        z = rnd(rng, bw, s.n_ps)
        dx, drx, dkd, drkd, dz = (to_dev(i) for i in (x, rx, kd, rkd, z))
        out, read = guarded(s.n_ps, bw)
        ddg.linattn_chunk_share(bw, party, sh, ld, ptr(dx), ptr(drx), ptr(dkd), ptr(drkd), ptr(dz), ptr(out))
        assert np.array_equal(read(), R.ring(R.chunk_share(s, party, x, rx, kd, rkd) + z, bw))
        ps, rps, s0, rs0 = (rnd(rng, bw, n) for n in (s.n_ps, s.n_ps, s.n_state, s.n_state))
        z = rnd(rng, bw, s.B * s.T * s.H * s.dv)
        dps, drps, ds0, drs0, dz = (to_dev(i) for i in (ps, rps, s0, rs0, z))
        for use in (True, False):
            out, read = guarded(z.size, bw)
            ddg.linattn_output_share(bw, party, sh, ld, ptr(dx), ptr(drx), ptr(dkd), ptr(drkd), ptr(dps), ptr(drps),
                                     ptr(ds0) if use else None, ptr(drs0) if use else None, ptr(dz), ptr(out))
            want = R.output_share(s, party, x, rx, kd, rkd, ps, rps, s0 if use else None, rs0 if use else None)
            assert np.array_equal(read(), R.ring(want + z, bw))
        assert ddg.lib().ddg_gemm_status() == 0


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("party", [0, 1])
@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 1, 1), (1, 4, 47, 47), (3, 2, 64, 64), (2, 3, 128, 128), (5, 1, 128, 33),
                                       (1, 7, 9, 128), (33, 5, 20, 12)])
def test_linattn_step_shares(ddg, cuda, bw, party, B, H, dk, dv):
    rng = np.random.default_rng(B + H + dk + dv + bw + party)
    for pad in (0, 1):
        s, sh, ld, pow_ = la_inputs(ddg, rng, bw, (B, H, 1, dk, dv, 128), pad=pad, extra_pow=2 * pad)
        x, rx = rnd(rng, bw, B, 1, ld), rnd(rng, bw, B, 1, ld)
        st, rst = rnd(rng, bw, s.n_state), rnd(rng, bw, s.n_state)
        nyw = B * H * (dv + 1)
        z = rnd(rng, bw, s.n_state + nyw)
        dp, dx, drx, ds, drs, dz = (to_dev(i) for i in (pow_, x, rx, st, rst, z))
        out, read = guarded(z.size, bw)
        ddg.linattn_step_share(bw, party, sh, ld, ptr(dp), ptr(dx), ptr(drx), ptr(ds), ptr(drs), ptr(dz), ptr(out))
        assert np.array_equal(read(), R.ring(R.step_share(s, party, pow_[:, 1], x, rx, st, rst) + z, bw))
        yw, ryw, z = rnd(rng, bw, nyw), rnd(rng, bw, nyw), rnd(rng, bw, B * H * dv)
        dyw, dryw, dz = (to_dev(i) for i in (yw, ryw, z))
        out, read = guarded(z.size, bw)
        ddg.linattn_step_output_share(bw, party, sh, ld, ptr(dp), ptr(dx), ptr(drx), ptr(dyw), ptr(dryw), ptr(dz),
                                      ptr(out))
        assert np.array_equal(read(), R.ring(R.step_output_share(s, party, pow_[:, 1], x, rx, yw, ryw) + z, bw))


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("BH,T", [(2, 40), (40, 256)])  # the CUDA-core tiles and the tensor cores
def test_linattn_products_in_place_of_the_dealers_word(ddg, cuda, bw, BH, T):
    """d_out may be d_z: every word is read before its place is written."""
    rng = np.random.default_rng(BH + T + bw)
    s, sh, ld, pow_ = la_inputs(ddg, rng, bw, (1, BH, T, 32, 48, 128))
    x, rx, kd, rkd = (rnd(rng, bw, *n) for n in ((1, T, ld), (1, T, ld), (s.n_decayed,), (s.n_decayed,)))
    ps, rps, z, z2 = (rnd(rng, bw, n) for n in (s.n_ps, s.n_ps, s.n_ps, T * BH * 48))
    dx, drx, dkd, drkd, dps, drps, dz, dz2 = (to_dev(i) for i in (x, rx, kd, rkd, ps, rps, z, z2))
    ddg.linattn_chunk_share(bw, 1, sh, ld, ptr(dx), ptr(drx), ptr(dkd), ptr(drkd), ptr(dz), ptr(dz))
    ddg.linattn_output_share(bw, 0, sh, ld, ptr(dx), ptr(drx), ptr(dkd), ptr(drkd), ptr(dps), ptr(drps), None, None,
                             ptr(dz2), ptr(dz2))
    assert np.array_equal(from_dev(dz, z.dtype, z.size), R.ring(R.chunk_share(s, 1, x, rx, kd, rkd) + z, bw))
    want = R.output_share(s, 0, x, rx, kd, rkd, ps, rps, None, None)
    assert np.array_equal(from_dev(dz2, z.dtype, z2.size), R.ring(want + z2, bw))
    s1, sh1, ld1, pow1 = la_inputs(ddg, rng, bw, (T, 2, 1, 64, 48, 128))
    x, rx, st, rst = (rnd(rng, bw, *n) for n in ((T, 1, ld1), (T, 1, ld1), (s1.n_state,), (s1.n_state,)))
    z = rnd(rng, bw, s1.n_state + T * 2 * 49)
    dp, dx, drx, ds, drs, dz = (to_dev(i) for i in (pow1, x, rx, st, rst, z))
    ddg.linattn_step_share(bw, 0, sh1, ld1, ptr(dp), ptr(dx), ptr(drx), ptr(ds), ptr(drs), ptr(dz), ptr(dz))
    assert np.array_equal(from_dev(dz, z.dtype, z.size), R.ring(R.step_share(s1, 0, pow1[:, 1], x, rx, st, rst) + z, bw))


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("shape", [(1, 12, 520, 64, 64, 128), (1, 20, 300, 48, 96, 100), (1, 30, 200, 47, 33, 64),
                                   (2, 16, 129, 32, 128, 128)])
def test_linattn_many_heads(ddg, cuda, bw, shape):
    """enough tiles for the tensor-core path, several per CTA: whole and ragged chunks, aligned and odd widths"""
    rng = np.random.default_rng(sum(shape) + bw)
    s, sh, ld, _ = la_inputs(ddg, rng, bw, shape)
    x, rx = rnd(rng, bw, s.B, s.T, ld), rnd(rng, bw, s.B, s.T, ld)
    kd, rkd, ps, rps = (rnd(rng, bw, n) for n in (s.n_decayed, s.n_decayed, s.n_ps, s.n_ps))
    s0, rs0, z, z2 = (rnd(rng, bw, n) for n in (s.n_state, s.n_state, s.n_ps, s.B * s.T * s.H * s.dv))
    d = [to_dev(i) for i in (x, rx, kd, rkd, ps, rps, s0, rs0, z, z2)]
    for party in (0, 1):
        out, read = guarded(s.n_ps, bw)
        ddg.linattn_chunk_share(bw, party, sh, ld, *[ptr(i) for i in d[:4]], ptr(d[8]), ptr(out))
        assert np.array_equal(read(), R.ring(R.chunk_share(s, party, x, rx, kd, rkd) + z, bw))
        out, read = guarded(z2.size, bw)
        ddg.linattn_output_share(bw, party, sh, ld, *[ptr(i) for i in d[:8]], ptr(d[9]), ptr(out))
        assert np.array_equal(read(), R.ring(R.output_share(s, party, x, rx, kd, rkd, ps, rps, s0, rs0) + z2, bw))
    assert ddg.lib().ddg_gemm_status() == 0


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("M,K,N,group", [(600, 1100, 2000, 128), (1030, 130, 5000, 32), (260, 2050, 4100, 160),
                                         (3, 40000, 260, 32), (20, 70000, 130, 64), (2, 5000, 4000, 96)])
def test_fc_q4_large(ddg, cuda, bw, M, K, N, group):
    """every tile, K split over clusters, two weight tiles per CTA, sums past one CTA's range, against float64 limbs"""
    import torch

    g = torch.Generator(device="cuda").manual_seed(M + K + N)
    dt = torch.int32 if bw == 32 else torch.int64
    rand = lambda *n: torch.randint(-(1 << (bw - 1)), (1 << (bw - 1)) - 1, n, dtype=dt, device="cuda", generator=g)  # noqa: E731
    row = 16 * ((K + 31) // 32)
    q = torch.randint(0, 256, (N, row), device="cuda", generator=g).to(torch.uint8)
    st = torch.randint(0, 4096, ((K + group - 1) // group, N), device="cuda", generator=g).to(torch.int16)
    x, C, b = rand(M, K), rand(M, N), rand(N)
    out = torch.empty(M, N, dtype=dt, device="cuda")
    torch.cuda.synchronize()
    w = ddg.Q4Weights(K, N, group, ptr(q), ptr(st), ptr(b))
    ddg.fc_q4_share(bw, 0, M, w, ptr(x), K, ptr(C), ptr(out))
    code = torch.stack((q & 15, q >> 4), 2).reshape(N, -1)[:, :K].double() - 8
    W = (code.t() * st.double().repeat_interleave(group, 0)[:K])
    want = C.long() + b.long()
    for i in range(bw // 16):  # 2^16 x 2^15 x K < 2^53: exact
        want = want + (torch.matmul(((x.long() >> (16 * i)) & 0xFFFF).double(), W).long() << (16 * i))
    assert torch.equal(out, want.to(dt))
    assert ddg.lib().ddg_gemm_status() == 0


def test_fc_q4_refuses_too_long_a_reduction(ddg, cuda):
    d = dev_bytes(4096)
    w = ddg.Q4Weights((1 << 18) + 1, 8, 32, ptr(d), ptr(d), None)
    assert ddg.lib().ddg_fc_q4_share(32, 0, 4, w, ptr(d), (1 << 18) + 1, ptr(d), ptr(d), None) == 1


@pytest.mark.parametrize("bw", [32, 64])
def test_share_calls_on_a_stream_and_in_a_graph(ddg, cuda, bw):
    """The share calls run on the stream they are given and can be captured; a replay reads the inputs anew."""
    import torch

    rng = np.random.default_rng(7)
    M, K, N = 20, 200, 150
    code = rng.integers(0, 16, size=(K, N), dtype=np.uint8)
    step = rng.integers(1, 4096, size=(K // 32 + 1, N)).astype(np.uint16)
    W = R.q4_weights(code, step, 32).view(np.uint64)
    s, sh, ld, _ = la_inputs(ddg, rng, bw, (1, 2, 200, 32, 32, 128))
    dq, ds = to_dev(R.q4_pack(code)), to_dev(step)
    w = ddg.Q4Weights(K, N, 32, ptr(dq), ptr(ds), None)
    new = lambda: (rnd(rng, bw, M, K), rnd(rng, bw, 1, 200, ld), rnd(rng, bw, s.n_decayed))  # noqa: E731
    X, x, kd = new()
    C, rx, rkd, z = rnd(rng, bw, M, N), rnd(rng, bw, 1, 200, ld), rnd(rng, bw, s.n_decayed), rnd(rng, bw, s.n_ps)
    dX, dx, dkd, dC, drx, drkd, dz = (to_dev(i) for i in (X, x, kd, C, rx, rkd, z))
    o1, o2 = dev_bytes(M * N * bw // 8), dev_bytes(s.n_ps * bw // 8)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()

    def call():
        ddg.fc_q4_share(bw, 0, M, w, ptr(dX), K, ptr(dC), ptr(o1), st.cuda_stream)
        ddg.linattn_chunk_share(bw, 0, sh, ld, ptr(dx), ptr(drx), ptr(dkd), ptr(drkd), ptr(dz), ptr(o2), st.cuda_stream)

    def check():
        torch.cuda.synchronize()
        assert np.array_equal(from_dev(o1, ring_dt(bw), M * N).reshape(M, N), R.ring(R.mm(X, W) + C, bw))
        assert np.array_equal(from_dev(o2, ring_dt(bw), s.n_ps), R.ring(R.chunk_share(s, 0, x, rx, kd, rkd) + z, bw))

    call()
    check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        call()
    for _ in range(2):
        X, x, kd = new()
        for d, h in ((dX, X), (dx, x), (dkd, kd)):
            d.copy_(to_dev(h))
        o1.zero_(), o2.zero_()
        torch.cuda.synchronize()
        g.replay()
        check()


# ---------------------------------------------------------------- as wires: a secure token model

class Model:
    """One attention block: x -> q|k|v (4-bit weights) -> linear attention -> output projection (4-bit weights)"""

    def __init__(self, ddg, bw, B, H, T, dk, dv, C, D, seed):
        self.bw, self.D, self.ddg = bw, D, ddg
        self.s, self.one = R.Shape(B, H, T, dk, dv, C), R.Shape(B, H, 1, dk, dv, C)
        rng = np.random.default_rng(seed)
        n = 3  # decoded tokens
        self.pow = ddg.decay_table(bw, S, np.linspace(0.8, 0.99, H), max(T, 1))
        self.sh = ddg.LinattnShape(B, H, T, dk, dv, C, self.pow.shape[1] - 1)
        self.sh1 = ddg.LinattnShape(B, H, 1, dk, dv, C, self.pow.shape[1] - 1)
        self.w, self.d = [], []
        for K, N, act in ((D, self.s.width, ddg.ACT_FLOOR), (H * dv, D, ddg.ACT_FLOOR), (D, D, ddg.ACT_RELU),
                          (D, 9, ddg.ACT_NONE)):
            real = rng.normal(0, 0.5 / np.sqrt(K), (K, N)) * (1 << S)
            w = np.round(real).astype(np.int64)
            dw, dq = to_dev(w), dev_bytes(N * 16 * ((K + 31) // 32))
            dst = dev_bytes(((K + 31) // 32) * N * 2)
            ddg.q4_quantize(K, N, 32, ptr(dw), ptr(dq), ptr(dst))
            b = rnd(rng, 32, N).astype(np.int64) % 4096 << S
            db = to_dev(b.astype(ring_dt(bw)))
            self.w.append((R.q4_weights(*R.q4_quantize(w, 32), 32), b))
            self.d.append((ddg.Q4Weights(K, N, 32, ptr(dq), ptr(dst), ptr(db)), act, (dw, dq, dst, db)))
        self.dpow = to_dev(self.pow)
        tok = lambda t: np.round(rng.uniform(-1, 1, (B, t, D)) * (1 << S)).astype(np.int64).view(np.uint64)  # noqa: E731
        self.x = [tok(T)] + [tok(1) for _ in range(n)]

    def fc(self, i, x):
        w, b = self.w[i]
        y = R.mm(x, w.view(np.uint64)) + b.view(np.uint64)
        act = self.d[i][1]
        if act == self.ddg.ACT_NONE:
            return y
        y = R.floor_shift(y, S, self.bw)
        return np.where(y.view(np.int64) < 0, 0, y) if act == self.ddg.ACT_RELU else y

    def clear(self):
        outs, st = [], None
        for t, x in enumerate(self.x):
            qkv = self.fc(0, x)
            if t == 0:
                o, st = R.clear_prompt(self.s, self.pow, qkv, None, S, self.bw)
            else:
                o, st = R.clear_step(self.one, self.pow[:, 1], qkv, st, S, self.bw)
            outs += [o, self.fc(3, self.fc(2, self.fc(1, o))), st]
        # the last tokens once more, as a prompt that continues from the state
        o, st = R.clear_prompt(self.s, self.pow, self.fc(0, self.x[0]), st, S, self.bw)
        return [i.reshape(-1) for i in outs + [o, st]]

    def key_bytes(self):
        L, n = self.ddg.lib(), 0
        s, up = self.s, lambda v: -(-int(v) // 256) * 256
        for t in [s.T] + [1] * (len(self.x) - 1) + [s.T]:
            n += up(s.B * t * self.D * self.bw // 8)
            for w, act, _ in self.d:
                n += L.ddg_op_fc_q4_key_bytes(self.bw, S, w.K, w.N, s.B * t, act)
        n += 2 * L.ddg_linattn_key_bytes(self.bw, S, self.sh, 1)
        return n + (len(self.x) - 1) * L.ddg_linattn_step_key_bytes(self.bw, S, self.sh1)

    def walk(self, h, kind, new, inputs):
        """the same calls for the dealer (keygen) and a party (eval); every output wire, in the order of clear()"""
        L, chk, s, c = self.ddg.lib(), self.ddg.check, self.s, self.ddg.Cursor()
        fcs, pr, st = (getattr(L, f"ddg_{n}_{kind}") for n in ("op_fc_q4", "linattn", "linattn_step"))
        outs, state = [], None

        def fc(i, x, rows):
            w, act, _ = self.d[i]
            y = new(rows * w.N)
            chk(fcs(h, c, w, rows, act, x, y))
            return y

        for t, x in enumerate(list(self.x) + [self.x[0]]):
            n = x.shape[1]
            xin = new(x.size)
            if kind == "eval":
                chk(L.ddg_op_input_eval(h, c, x.size, inputs[t], xin))
            else:
                chk(L.ddg_op_input_keygen(h, c, x.size, xin))
            qkv, o, after = fc(0, xin, s.B * n), new(s.B * n * s.H * s.dv), new(s.n_state)
            if t == 0 or t == len(self.x):
                chk(pr(h, c, self.sh, ptr(self.dpow), qkv, state, o, after))
            else:
                chk(st(h, c, self.sh1, ptr(self.dpow), qkv, state, o, state))
                after = new(s.n_state)
                import torch
                self.copy(after, state, torch)
            if t == 0:
                state = after
                after = new(s.n_state)
                import torch
                self.copy(after, state, torch)
            outs.append(o)
            if t < len(self.x):
                outs.append(fc(3, fc(2, fc(1, o, s.B * n), s.B * n), s.B * n))
            outs.append(after)
        return outs, c.offset

    def copy(self, dst, src, torch):
        from tests.test_layers_gpu import _cudart

        f = "d_value" if hasattr(src, "d_value") else "d_mask"
        torch.cuda.synchronize()
        assert _cudart().cudaMemcpy(getattr(dst, f), getattr(src, f), src.n * self.bw // 8, 3) == 0
        torch.cuda.synchronize()


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("backend", ["RELU_TT", "RELU_OT", "RELU_DCF"])
def test_secure_token_model(ddg, synth, cuda, bw, backend):
    """A prompt in chunks, three decoded tokens and a second prompt from their state, every layer's
    outputs unmasked with the dealer's masks against the cleartext integers, on both parties."""
    import torch

    m = Model(ddg, bw, 2, 3, 11, 5, 6, 4, 40, seed=bw)
    want = m.clear()
    dt = ring_dt(bw)
    blob = synth.weights_blob(synth.quantize_weights(synth.affinity_weights(5), S))
    ddg.relu_backend(getattr(ddg, backend))
    try:
        kb = m.key_bytes()
        keys = [dev_bytes(kb) for _ in range(2)]
        torch.cuda.synchronize()
        d = ddg.Dealer(bw, S, 0, 99, blob)
        d.bind_keys(ptr(keys[0]), ptr(keys[1]), kb)
        bufs = [Bufs(bw // 8) for _ in range(3)]
        masks, used = m.walk(d.h, "keygen", lambda n: bufs[2].mask_wire(ddg, n), None)
        assert 0 < used <= kb
        rng = np.random.default_rng(1)
        sh0 = [rnd(rng, bw, x.size) for x in list(m.x) + [m.x[0]]]
        sh1 = [(R.ring(x, bw).reshape(-1) - a).astype(dt) for x, a in zip(list(m.x) + [m.x[0]], sh0)]
        dev = [[to_dev(i) for i in sh] for sh in (sh0, sh1)]
        torch.cuda.synchronize()
        ps = [ddg.Party(p, bw, S, 0) for p in (0, 1)]
        for p, k in zip(ps, keys):
            p.bind_keys(ptr(k), kb)
        ddg.pair_local(ps[0], ps[1])
        got = [None, None]

        def side(p):
            got[p] = m.walk(ps[p].h, "eval", lambda n: bufs[p].wire(ddg, n), [ptr(i) for i in dev[p]])

        run_both(lambda: side(0), lambda: side(1))
        for i, (w, mask) in enumerate(zip(want, masks)):
            r = wire_host(mask.d_mask, mask.n, dt)
            for p in (0, 1):
                v = wire_host(got[p][0][i].d_value, mask.n, dt)
                assert np.array_equal((v - r).astype(dt), R.ring(w, bw)), (i, p)
        assert got[0][1] == got[1][1] == used
        for p in ps:
            p.close()
        d.close()
    finally:
        ddg.relu_backend(ddg.RELU_TT)


def test_wire_calls_refuse_wrong_wires(ddg, synth, cuda):
    """Sizes, nulls and the floors' scale are refused before any key is read; the cursor stays."""
    L = ddg.lib()
    blob = synth.weights_blob(synth.quantize_weights(synth.affinity_weights(5), S))
    d = ddg.Dealer(32, S, 0, 1, blob)
    keys = dev_bytes(1 << 16)
    d.bind_keys(ptr(keys), ptr(keys), 1 << 16)
    b, c = Bufs(4), ddg.Cursor()
    q = dev_bytes(4096)
    w = ddg.Q4Weights(32, 8, 32, ptr(q), ptr(q), None)
    sh = ddg.LinattnShape(1, 2, 3, 4, 5, 2, 3)
    mw = lambda n: b.mask_wire(ddg, n)  # noqa: E731
    assert L.ddg_op_fc_q4_keygen(d.h, c, w, 2, 0, mw(63), mw(16)) == 1
    assert L.ddg_op_fc_q4_keygen(d.h, c, w, 0, 0, mw(64), mw(16)) == 1
    assert L.ddg_op_fc_q4_keygen(d.h, c, w, 2, 7, mw(64), mw(16)) == 1
    assert L.ddg_op_fc_q4_keygen(d.h, c, w, 2, 0, ddg.MaskWire(None, 64, None, None), mw(16)) == 1
    assert L.ddg_linattn_keygen(d.h, c, sh, ptr(q), mw(77), None, mw(30), mw(40)) == 1
    assert L.ddg_linattn_keygen(d.h, c, sh, ptr(q), mw(78), mw(39), mw(30), mw(40)) == 1
    assert L.ddg_linattn_keygen(d.h, c, sh, None, mw(78), None, mw(30), mw(40)) == 1
    assert L.ddg_linattn_step_keygen(d.h, c, sh, ptr(q), mw(78), mw(40), mw(30), mw(40)) == 1
    # more key bytes than are bound: refused, the cursor unmoved
    assert L.ddg_op_fc_q4_keygen(d.h, c, ddg.Q4Weights(32, 8, 32, ptr(q), ptr(q), None), 1000, 0, mw(32000),
                                 mw(8000)) == 0
    big = c.offset
    assert L.ddg_op_fc_q4_keygen(d.h, c, w, 2000, 0, mw(64000), mw(16000)) == 3
    assert c.offset == big
    d.close()
    p = ddg.Party(0, 32, S, 0)
    assert L.ddg_op_fc_q4_eval(p.h, ddg.Cursor(), w, 1, 0, b.wire(ddg, 32), b.wire(ddg, 8)) == 5  # no channel
    p.close()
