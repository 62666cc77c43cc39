"""Token-model operators on the GPU at the ends of what their arguments allow,
bit for bit against the integer definitions in tests/token_ref.py."""
import numpy as np
import pytest

from tests import token_ref as R
from tests.gpu_util import dev_bytes, from_dev, ptr, ring_dt, to_dev

pytestmark = pytest.mark.gpu
S = 12


def rnd(rng, bw, *shape):
    dt = ring_dt(bw)
    return rng.integers(0, np.iinfo(dt).max, size=shape, dtype=dt, endpoint=True)


@pytest.fixture
def room(cuda):
    """the allocator's cache of a large test, given back for the library's own allocations of the next one"""
    yield
    cuda.cuda.synchronize()
    cuda.cuda.empty_cache()


# ---------------------------------------------------------------- 4-bit weights

LONGEST_GROUP = (1 << 31) - 32


@pytest.mark.parametrize("K,group", [(1, LONGEST_GROUP), (64, LONGEST_GROUP), (1000, LONGEST_GROUP), (70, 1 << 30)])
def test_one_step_per_output_as_a_group_beyond_K(ddg, cuda, K, group):
    """A group may be any multiple of 32: one far above K is one step per output."""
    rng = np.random.default_rng(K)
    N = 40
    w = rng.integers(-20000, 20001, size=(K, N)).astype(np.int64)
    code, step = R.q4_quantize(w, group)
    assert step.shape == (1, N)
    dw, dq, ds = to_dev(w), dev_bytes(N * 16 * ((K + 31) // 32)), dev_bytes(N * 2)
    ddg.q4_quantize(K, N, group, ptr(dw), ptr(dq), ptr(ds))
    assert np.array_equal(from_dev(ds, np.uint16, N).reshape(1, N), step)
    assert np.array_equal(from_dev(dq, np.uint8, N * 16 * ((K + 31) // 32)).reshape(N, -1), R.q4_pack(code))
    W = ((code.astype(np.int64) - 8) * step.astype(np.int64)).view(np.uint64)
    for bw in (32, 64):
        for M in (1, 5):
            X, C = rnd(rng, bw, M, K), rnd(rng, bw, M, N)
            dx, dc, out = to_dev(X), to_dev(C), dev_bytes(M * N * bw // 8)
            ddg.fc_q4_share(bw, 0, M, ddg.Q4Weights(K, N, group, ptr(dq), ptr(ds), None), ptr(dx), K, ptr(dc), ptr(out))
            assert np.array_equal(from_dev(out, ring_dt(bw), M * N).reshape(M, N), R.ring(R.mm(X, W) + C, bw))


def test_q4_quantize_of_the_longest_column(ddg, cuda, room):
    """K = 2^31 - 1: the row's last byte, half of it padding, and the last group's step are written."""
    import torch

    K = (1 << 31) - 1
    w = torch.zeros(K, dtype=torch.int64, device="cuda")
    w[-2], w[-1] = -21, 9  # step 3: codes 8 - 7 and 8 + 3
    row, groups = 1 << 30, 1 << 26
    q = torch.full((row,), 0xEE, dtype=torch.uint8, device="cuda")
    step = torch.full((groups,), -1, dtype=torch.int16, device="cuda")
    torch.cuda.synchronize()
    ddg.q4_quantize(K, 1, 32, ptr(w), ptr(q), ptr(step))
    torch.cuda.synchronize()
    # counted before the asserts, which would iterate over whole tensors to explain a failure
    other_codes, other_steps = int((q[:-2] != 0x88).sum()), int((step[:-1] != 1).sum())
    last, tail = int(step[-1]), q[-2:].tolist()
    assert (other_codes, other_steps, last) == (0, 0, 3)
    assert tail == [0x18, 0x8B]


@pytest.mark.parametrize("bw,K,N", [(32, 100, 60), (64, 100, 60), (64, 4100, 4200), (32, 130000, 70)])
def test_stride_of_a_single_row_is_not_used(ddg, cuda, bw, K, N):
    """With one row nothing lies a stride away: any ldx >= K gives the same product (CUDA and tensor cores)."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(K)
    dt = torch.int32 if bw == 32 else torch.int64
    row = 16 * ((K + 31) // 32)
    q = torch.randint(0, 256, (N, row), device="cuda", generator=g).to(torch.uint8)
    st = torch.randint(0, 4096, ((K + 31) // 32, N), device="cuda", generator=g).to(torch.int16)
    x = torch.randint(-(1 << (bw - 1)), (1 << (bw - 1)) - 1, (1, K), dtype=dt, device="cuda", generator=g)
    C = torch.zeros(1, N, dtype=dt, device="cuda")
    outs = []
    for ldx in (K, K + 1, 1 << 40, (1 << 62) + 1, (1 << 63) - 1):
        out = torch.empty(1, N, dtype=dt, device="cuda")
        torch.cuda.synchronize()
        ddg.fc_q4_share(bw, 0, 1, ddg.Q4Weights(K, N, 32, ptr(q), ptr(st), None), ptr(x), ldx, ptr(C), ptr(out))
        outs.append(out)
    code = torch.stack((q & 15, q >> 4), 2).reshape(N, -1)[:, :K].double() - 8
    W = code.t() * st.double().repeat_interleave(32, 0)[:K]
    want = torch.zeros(1, N, dtype=torch.int64, device="cuda")
    for i in range(bw // 16):  # 2^16 x 2^15 x K < 2^53: exact
        want = want + (torch.matmul(((x.long() >> (16 * i)) & 0xFFFF).double(), W).long() << (16 * i))
    same = [bool(torch.equal(out, want.to(dt))) for out in outs]
    assert all(same)
    assert ddg.lib().ddg_gemm_status() == 0


# every kernel and split of K that the choice (csrc/q4_plan.cuh) can make, by ring width:
# (tile, CTAs along K) -> (M, K, N); tile -2 is the CUDA-core kernel
FC_TILES = {
    32: {(-2, 1): (2, 700, 130), (0, 1): (5, 90, 130), (0, 2): (5, 700, 130), (0, 4): (5, 1030, 130),
         (0, 8): (5, 132010, 130), (1, 1): (299, 90, 130), (1, 2): (161, 700, 130), (1, 4): (79, 1030, 130),
         (1, 8): (47, 132010, 130), (2, 1): (33, 700, 5000), (2, 2): (299, 700, 130), (2, 4): (161, 1030, 130),
         (2, 8): (79, 132010, 130), (3, 1): (65, 700, 5000), (3, 2): (65, 700, 2403), (3, 4): (299, 1030, 130),
         (3, 8): (161, 132010, 130), (4, 1): (100, 90, 5000), (4, 2): (1501, 700, 130), (4, 4): (601, 700, 130),
         (4, 8): (601, 132010, 3), (5, 1): (199, 90, 5000)},
    64: {(-2, 1): (1, 700, 130), (0, 1): (3, 90, 130), (0, 2): (3, 700, 130), (0, 4): (3, 1030, 130),
         (0, 8): (3, 132010, 130), (1, 1): (161, 90, 130), (1, 2): (79, 700, 130), (1, 4): (47, 1030, 130),
         (1, 8): (21, 132010, 130), (2, 1): (17, 700, 5000), (2, 2): (161, 700, 130), (2, 4): (79, 1030, 130),
         (2, 8): (47, 132010, 130), (3, 1): (33, 700, 5000), (3, 2): (33, 700, 2403), (3, 4): (161, 1030, 130),
         (3, 8): (79, 132010, 130), (4, 1): (1501, 700, 130), (4, 2): (601, 700, 130), (4, 4): (299, 700, 130),
         (4, 8): (161, 132010, 130), (5, 1): (100, 90, 5000)},
}


@pytest.mark.parametrize("bw,tile", [(bw, tile) for bw in FC_TILES for tile in FC_TILES[bw]])
def test_fc_q4_every_tile_and_split(ddg, cuda, bw, tile):
    """rows on 16-byte boundaries (tensor maps) and off them (element copies), against float64 limbs"""
    import torch

    M, K, N = FC_TILES[bw][tile]
    g = torch.Generator(device="cuda").manual_seed(M + K + N + bw)
    dt, group = (torch.int32 if bw == 32 else torch.int64), 96
    rand = lambda *n: torch.randint(-(1 << (bw - 1)), (1 << (bw - 1)) - 1, n, dtype=dt, device="cuda", generator=g)  # noqa: E731
    q = torch.randint(0, 256, (N, 16 * ((K + 31) // 32)), device="cuda", generator=g).to(torch.uint8)
    st = torch.randint(0, 4096, ((K + group - 1) // group, N), device="cuda", generator=g).to(torch.int16)
    code = torch.stack((q & 15, q >> 4), 2).reshape(N, -1)[:, :K].double() - 8
    W = code.t() * st.double().repeat_interleave(group, 0)[:K]
    C, b = rand(M, N), rand(N)
    w = ddg.Q4Weights(K, N, group, ptr(q), ptr(st), ptr(b))
    for ldx in ((K + 3) // 4 * 4, K | 1):
        x = rand(M, ldx)
        out = torch.zeros(M * N + 64, dtype=dt, device="cuda")
        torch.cuda.synchronize()
        ddg.fc_q4_share(bw, 0, M, w, ptr(x), ldx, ptr(C), ptr(out))
        want = C.long() + b.long()
        for i in range(bw // 16):  # 2^16 x 2^15 x K < 2^53: exact
            want = want + (torch.matmul(((x[:, :K].long() >> (16 * i)) & 0xFFFF).double(), W).long() << (16 * i))
        same, behind = bool(torch.equal(out[:M * N].view(M, N), want.to(dt))), int(out[M * N:].count_nonzero())
        assert same and behind == 0
    assert ddg.lib().ddg_gemm_status() == 0


# (M, K, N) whose CTAs on the tensor cores add up the most k that one may: 32,768
FC_LONGEST = [(3, 32768, 10300), (40, 32768, 10300), (600, 32768, 9000), (1, 262144, 140), (5, 262144, 130),
              (90, 262144, 70)]


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("M,K,N", FC_LONGEST)
def test_fc_q4_sums_beyond_31_bits(ddg, cuda, room, bw, M, K, N):
    """Every byte of x 255, so that x is -1, and the two bytes of W + 2^15 up to 253 and 238: a column of byte products
    reaches 491 x 255 x 32768 = 0.955 x 2^32, beyond a signed accumulator's range."""
    import torch

    dt = torch.int32 if bw == 32 else torch.int64
    code = torch.tensor([15, 15, 0, 15, 8], device="cuda").repeat(N // 5 + 1)[:N]
    step = torch.tensor([4059, 4095, 4095, 4022, 1], device="cuda").repeat(N // 5 + 1)[:N]
    q = (code * 17).to(torch.uint8).view(N, 1).expand(N, 16 * ((K + 31) // 32)).contiguous()
    st = step.to(torch.int16).expand((K + 31) // 32, N).contiguous()
    x = torch.full((M, K), -1, dtype=dt, device="cuda")
    C = torch.arange(M * N, dtype=dt, device="cuda").view(M, N)
    out = torch.empty(M, N, dtype=dt, device="cuda")
    torch.cuda.synchronize()
    ddg.fc_q4_share(bw, 0, M, ddg.Q4Weights(K, N, 32, ptr(q), ptr(st), None), ptr(x), K, ptr(C), ptr(out))
    want = (C.long() - K * step * (code - 8)).to(dt)
    same = bool(torch.equal(out, want))
    assert same and ddg.lib().ddg_gemm_status() == 0


# ---------------------------------------------------------------- linear attention

def test_linattn_longest_table_of_powers(ddg, cuda, room):
    """pow_n = 2^31 - 1: the second head's powers start 2^31 elements into the table."""
    import torch

    T, dk, dv = 5, 4, 8
    table = torch.zeros(1 << 32, dtype=torch.int32, device="cuda")
    for bw, width in ((32, 4), (64, 8)):  # over Z_2^64 one head's table is what fits here
        H = 2 if bw == 32 else 1
        rng = np.random.default_rng(bw)
        few = rnd(rng, bw, H, T + 1)
        view = table.view(torch.uint8).view(H, -1)
        for h in range(H):
            view[h, :few[h].nbytes] = to_dev(few[h])
        s, one = R.Shape(1, H, T, dk, dv, 2), R.Shape(1, H, 1, dk, dv, 2)
        sh, sh1 = (ddg.LinattnShape(1, H, t, dk, dv, 2, (1 << 31) - 1) for t in (T, 1))
        x, ps, s0 = rnd(rng, bw, 1, T, s.width), rnd(rng, bw, s.n_ps), rnd(rng, bw, s.n_state)
        dx, dps, ds0 = to_dev(x), to_dev(ps), to_dev(s0)
        o1, o2 = dev_bytes(2 * s.n_decayed * width), dev_bytes(s.n_ps * width)
        torch.cuda.synchronize()
        ddg.linattn_decay(bw, sh, s.width, ptr(table), ptr(dx), ptr(o1))
        ddg.linattn_carry(bw, sh, ptr(table), ptr(dps), ptr(ds0), ptr(o2))
        assert np.array_equal(from_dev(o1, ring_dt(bw), 2 * s.n_decayed), R.ring(R.decay(s, few, x), bw))
        assert np.array_equal(from_dev(o2, ring_dt(bw), s.n_ps), R.ring(R.carry(s, few, ps, s0), bw))
        x, rx, rs, nyw = rnd(rng, bw, 1, 1, s.width), rnd(rng, bw, 1, 1, s.width), rnd(rng, bw, s.n_state), H * (dv + 1)
        z, yw, ryw, zo = (rnd(rng, bw, n) for n in (s.n_state + nyw, nyw, nyw, H * dv))
        dx, drx, drs, dz, dyw, dryw, dzo = (to_dev(i) for i in (x, rx, rs, z, yw, ryw, zo))
        torch.cuda.synchronize()
        ddg.linattn_step_share(bw, 0, sh1, s.width, ptr(table), ptr(dx), ptr(drx), ptr(ds0), ptr(drs), ptr(dz), ptr(dz))
        ddg.linattn_step_output_share(bw, 0, sh1, s.width, ptr(table), ptr(dx), ptr(drx), ptr(dyw), ptr(dryw), ptr(dzo),
                                      ptr(dzo))
        assert np.array_equal(from_dev(dz, z.dtype, z.size),
                              R.ring(R.step_share(one, 0, few[:, 1], x, rx, s0, rs) + z, bw))
        assert np.array_equal(from_dev(dzo, z.dtype, zo.size),
                              R.ring(R.step_output_share(one, 0, few[:, 1], x, rx, yw, ryw) + zo, bw))


# ---------------------------------------------------------------- as wires

@pytest.mark.parametrize("bw", [32, 64])
def test_token_model_result_is_read_without_affinity_weights(ddg, synth, cuda, bw):
    """Input -> 4-bit layer -> gate -> product of wires -> output on parties that hold no affinity weights; the calls
    that read those weights still refuse."""
    from tests.test_layers_gpu import Bufs, run_both

    L, dt, n = ddg.lib(), ring_dt(bw), 24
    rng = np.random.default_rng(bw)
    K, N, rows = 40, 12, 2
    one = 1 << S
    w = np.round(rng.normal(0, 0.3, (K, N)) * one).astype(np.int64)
    x = np.round(rng.uniform(-1, 1, (rows, K)) * one).astype(np.int64)
    y = np.round(rng.uniform(0, 6, (rows, N)) * one).astype(np.int64)
    code, step = R.q4_quantize(w, 32)
    act = np.maximum((x @ R.q4_weights(code, step, 32)) >> S, 0)
    want = ((act * y) >> S).reshape(-1)
    assert np.abs(act * y).max() < 1 << (bw - 2) and want.any()
    dw, dq, ds = to_dev(w), dev_bytes(N * 16 * ((K + 31) // 32)), dev_bytes(step.size * 2)
    ddg.q4_quantize(K, N, 32, ptr(dw), ptr(dq), ptr(ds))
    q4 = ddg.Q4Weights(K, N, 32, ptr(dq), ptr(ds), None)

    kb = 1 << 20
    keys = [dev_bytes(kb) for _ in range(2)]
    d = ddg.Dealer(bw, S, 0, 5, synth.weights_blob(synth.quantize_weights(synth.affinity_weights(5), S)))
    d.bind_keys(ptr(keys[0]), ptr(keys[1]), kb)
    bufs = [Bufs(bw // 8) for _ in range(3)]
    c, mw = ddg.Cursor(), lambda k: bufs[2].mask_wire(ddg, k)
    X, Y, Z, A, P = mw(x.size), mw(n), mw(n), mw(n), mw(n)
    for st in (L.ddg_op_input_keygen(d.h, c, x.size, X), L.ddg_op_input_keygen(d.h, c, n, Y),
               L.ddg_op_fc_q4_keygen(d.h, c, q4, rows, ddg.ACT_NONE, X, Z),
               L.ddg_op_gate_keygen(d.h, c, ddg.GATE_RELU_ARS, Z, A),
               L.ddg_op_mul_keygen(d.h, c, 0, 0, 0, A, Y, 0, P), L.ddg_op_output_keygen(d.h, c, P)):
        ddg.check(st)
    end = c.offset

    def split(v):
        a = rnd(rng, bw, v.size)
        return to_dev(a), to_dev((R.ring(v.reshape(-1).view(np.uint64), bw) - a).astype(dt))

    sx, sy = split(x), split(y)
    ps = [ddg.Party(p, bw, S, 0) for p in (0, 1)]
    for p, k in zip(ps, keys):
        p.bind_keys(ptr(k), kb)
    ddg.pair_local(ps[0], ps[1])
    got = [None, None]

    def side(p):
        c, wi, h = ddg.Cursor(), lambda k: bufs[p].wire(ddg, k), ps[p].h
        X, Y, Z, A, P = wi(x.size), wi(n), wi(n), wi(n), wi(n)
        ddg.check(L.ddg_op_input_eval(h, c, x.size, ptr(sx[p]), X))
        ddg.check(L.ddg_op_input_eval(h, c, n, ptr(sy[p]), Y))
        ddg.check(L.ddg_op_fc_q4_eval(h, c, q4, rows, ddg.ACT_NONE, X, Z))
        ddg.check(L.ddg_op_gate_eval(h, c, ddg.GATE_RELU_ARS, Z, A))
        ddg.check(L.ddg_op_mul_eval(h, c, 0, 0, 0, A, Y, 0, P))
        raw = np.zeros(n, np.int64)
        ddg.check(L.ddg_op_output_eval(h, c, n, P, raw.ctypes.data, None))
        assert c.offset == end
        # what reads the affinity weights
        big = wi(138 * 376)
        assert L.ddg_adjnorm_eval(h, c, 1, ptr(sx[p]), big) == 5
        assert L.ddg_op_fc_eval(h, c, 8, 1, 0, wi(256), wi(1)) == 5
        assert L.ddg_gcn_layer_eval(h, c, 0, 1, wi(138 * 138), wi(138 * 94), big) == 5
        got[p] = raw

    run_both(lambda: side(0), lambda: side(1))
    for p in (0, 1):
        assert np.array_equal(got[p], want)
        ps[p].close()
    d.close()


@pytest.mark.parametrize("bw,off", [(32, 2), (64, 4)])
def test_wire_calls_refuse_misaligned_arrays(ddg, synth, cuda, bw, off):
    """A wire, bias or table of powers off its element boundary would fault in a kernel: refused before any work, on
    the dealer and on a party, the cursors unmoved."""
    from tests.test_layers_gpu import Bufs

    L, kb = ddg.lib(), 1 << 18
    keys = [dev_bytes(kb) for _ in range(2)]
    d = ddg.Dealer(bw, S, 0, 1, synth.weights_blob(synth.quantize_weights(synth.affinity_weights(5), S)))
    d.bind_keys(ptr(keys[0]), ptr(keys[1]), kb)
    ps = [ddg.Party(p, bw, S, 0) for p in (0, 1)]
    for p, k in zip(ps, keys):
        p.bind_keys(ptr(k), kb)
    ddg.pair_local(ps[0], ps[1])
    b, q = Bufs(bw // 8), dev_bytes(1 << 16)
    sh, sh1, nq, ns = ddg.LinattnShape(1, 2, 3, 4, 5, 2, 3), ddg.LinattnShape(1, 2, 1, 4, 5, 2, 3), 78, 40
    good = ddg.Q4Weights(32, 8, 32, ptr(q), ptr(q), ptr(q))
    bad_bias = ddg.Q4Weights(32, 8, 32, ptr(q), ptr(q), ptr(q) + off)
    p, bad = ptr(q), ptr(q) + off

    def calls(h, c, kind, new, wire):
        fc, pr, st = (getattr(L, f"ddg_{n}_{kind}") for n in ("op_fc_q4", "linattn", "linattn_step"))
        yield fc(h, c, bad_bias, 2, 0, new(64), new(16))
        for x in wire(64):
            yield fc(h, c, good, 2, 0, x, new(16))
        yield pr(h, c, sh, bad, new(nq), None, new(30), new(ns))
        yield st(h, c, sh1, bad, new(nq // 3), new(ns), new(10), new(ns))
        for x in wire(nq):
            yield pr(h, c, sh, p, x, None, new(30), new(ns))
        for x in wire(nq // 3):
            yield st(h, c, sh1, p, x, new(ns), new(10), new(ns))
        for x in wire(ns):
            yield pr(h, c, sh, p, new(nq), x, new(30), new(ns))
            yield st(h, c, sh1, p, new(nq // 3), x, new(10), new(ns))

    c = ddg.Cursor()
    masks = lambda n: [ddg.MaskWire(*a) for a in ((bad, n, None, None), (p, n, bad, p), (p, n, p, bad))]  # noqa: E731
    said = lambda it: {(st, L.ddg_last_error()) for st in it}  # noqa: E731
    refused = {(1, b"misaligned ring array")}
    assert said(calls(d.h, c, "keygen", lambda n: b.mask_wire(ddg, n), masks)) == refused
    assert (c.offset, c.ops) == (0, 0)
    values = lambda n: [ddg.Wire(bad, n, None), ddg.Wire(p, n, bad)]  # noqa: E731
    for party in ps:
        assert said(calls(party.h, c, "eval", lambda n: b.wire(ddg, n), values)) == refused and c.offset == 0
    for party in ps:
        party.close()
    d.close()


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("shape", [(1, 12, 520, 64, 64, 128), (1, 30, 200, 47, 33, 64)])
def test_linattn_on_wires_with_many_heads(ddg, synth, cuda, bw, shape):
    """Prompt, a prompt from its state, a token: enough heads that the dealer's words and both parties' shares come from
    the tensor cores in the chunk and output stages; rows on and off 16-byte boundaries."""
    import torch

    from tests.test_layers_gpu import Bufs, run_both, wire_host

    L, dt = ddg.lib(), ring_dt(bw)
    s, one = R.Shape(*shape), R.Shape(*shape[:2], 1, *shape[3:])
    B, H, T, dk, dv, C = shape
    rng = np.random.default_rng(bw + T)
    pow_ = ddg.decay_table(bw, S, np.linspace(0.8, 0.99, H), T)
    sh, sh1 = ddg.LinattnShape(B, H, T, dk, dv, C, T), ddg.LinattnShape(B, H, 1, dk, dv, C, T)
    new_x = lambda t: np.round(rng.uniform(-0.5, 0.5, (B, t, s.width)) * (1 << S)).astype(np.int64).view(np.uint64)  # noqa: E731
    x = [new_x(T), new_x(T), new_x(1)]
    o0, st0 = R.clear_prompt(s, pow_, x[0], None, S, bw)
    o1, st1 = R.clear_prompt(s, pow_, x[1], st0, S, bw)
    o2, st2 = R.clear_step(one, pow_[:, 1], x[2], st1, S, bw)
    want = [o0, st0, o1, st1, o2, st2]

    up = lambda n: -(-n * bw // 8 // 256) * 256  # noqa: E731
    kb = sum(up(i.size) for i in x) + 2 * L.ddg_linattn_key_bytes(bw, S, sh, 1) + L.ddg_linattn_step_key_bytes(bw, S, sh1)
    keys, dpow = [dev_bytes(kb) for _ in range(2)], to_dev(pow_)
    torch.cuda.synchronize()
    d = ddg.Dealer(bw, S, 0, 17, synth.weights_blob(synth.quantize_weights(synth.affinity_weights(5), S)))
    d.bind_keys(ptr(keys[0]), ptr(keys[1]), kb)
    bufs = [Bufs(bw // 8) for _ in range(3)]

    def walk(h, kind, new, inputs):
        prompt, step = getattr(L, f"ddg_linattn_{kind}"), getattr(L, f"ddg_linattn_step_{kind}")
        c, X, outs = ddg.Cursor(), [], []
        for i, v in enumerate(x):
            X.append(new(v.size))
            ddg.check(L.ddg_op_input_keygen(h, c, v.size, X[-1]) if inputs is None
                      else L.ddg_op_input_eval(h, c, v.size, inputs[i], X[-1]))
        for call, shp, xi, t in ((prompt, sh, X[0], T), (prompt, sh, X[1], T), (step, sh1, X[2], 1)):
            o, st = new(B * t * H * dv), new(s.n_state)
            ddg.check(call(h, c, shp, ptr(dpow), xi, outs[-1] if outs else None, o, st))
            outs += [o, st]
        return outs, c.offset

    masks, used = walk(d.h, "keygen", lambda n: bufs[2].mask_wire(ddg, n), None)
    assert 0 < used <= kb
    sh0 = [rnd(rng, bw, i.size) for i in x]
    dev = [[to_dev(i) for i in sh0], [to_dev((R.ring(v, bw).reshape(-1) - a).astype(dt)) for v, a in zip(x, sh0)]]
    torch.cuda.synchronize()
    ps = [ddg.Party(p, bw, S, 0) for p in (0, 1)]
    for p, k in zip(ps, keys):
        p.bind_keys(ptr(k), kb)
    ddg.pair_local(ps[0], ps[1])
    got = [None, None]

    def side(p):
        got[p] = walk(ps[p].h, "eval", lambda n: bufs[p].wire(ddg, n), [ptr(i) for i in dev[p]])

    run_both(lambda: side(0), lambda: side(1))
    for i, (w, mask) in enumerate(zip(want, masks)):
        r = wire_host(mask.d_mask, mask.n, dt)
        for p in (0, 1):
            v = wire_host(got[p][0][i].d_value, mask.n, dt)
            assert np.array_equal((v - r).astype(dt), R.ring(w, bw).reshape(-1)), (i, p)
    assert got[0][1] == got[1][1] == used
    for p in ps:
        p.close()
    d.close()


@pytest.mark.parametrize("bw", [32, 64])
def test_share_calls_of_two_threads_and_two_graphs_at_once(ddg, cuda, bw):
    """Two host threads on two streams, then two captured graphs replayed at the same time: no call keeps anything that
    the other one uses."""
    import threading

    import torch

    M, K, N, T, H = 33, 700, 2403, 300, 20
    rng = np.random.default_rng(bw)
    code, step = rng.integers(0, 16, (K, N), dtype=np.uint8), rng.integers(0, 4096, ((K + 31) // 32, N)).astype(np.uint16)
    W = R.q4_weights(code, step, 32).view(np.uint64)
    dq, ds = to_dev(R.q4_pack(code)), to_dev(step)
    s, sh = R.Shape(1, H, T, 48, 96, 100), ddg.LinattnShape(1, H, T, 48, 96, 100, T)
    w = ddg.Q4Weights(K, N, 32, ptr(dq), ptr(ds), None)

    class Side:
        def __init__(self):
            self.st = torch.cuda.Stream()
            X, C = rnd(rng, bw, M, K), rnd(rng, bw, M, N)
            x, rx, kd, rkd, z = (rnd(rng, bw, *n) for n in ((1, T, s.width), (1, T, s.width), (s.n_decayed,),
                                                            (s.n_decayed,), (s.n_ps,)))
            self.want = (R.ring(R.mm(X, W) + C, bw).reshape(-1), R.ring(R.chunk_share(s, 0, x, rx, kd, rkd) + z, bw))
            self.d = [to_dev(i) for i in (X, C, x, rx, kd, rkd, z)]
            self.out = [dev_bytes(i.nbytes) for i in self.want]

        def call(self):
            X, C, x, rx, kd, rkd, z = (ptr(i) for i in self.d)
            ddg.fc_q4_share(bw, 0, M, w, X, K, C, ptr(self.out[0]), self.st.cuda_stream)
            ddg.linattn_chunk_share(bw, 0, sh, s.width, x, rx, kd, rkd, z, ptr(self.out[1]), self.st.cuda_stream)

        def check(self):
            for o, v in zip(self.out, self.want):
                assert np.array_equal(from_dev(o, v.dtype, v.size), v)
                o.zero_()
            torch.cuda.synchronize()

    sides, errs = [Side(), Side()], []
    torch.cuda.synchronize()

    def run(side):
        try:
            for _ in range(20):
                side.call()
        except Exception as e:  # raised below
            errs.append(e)

    ts = [threading.Thread(target=run, args=(i,)) for i in sides]
    for t in ts:
        t.start()
    for t in ts:
        t.join(timeout=60)
    assert not errs
    torch.cuda.synchronize()
    for side in sides:
        side.check()
    graphs = []
    for side in sides:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side.st):
            side.call()
    for side in sides:  # capturing ran nothing
        assert all(int(o.count_nonzero()) == 0 for o in side.out)
    torch.cuda.synchronize()
    for _ in range(10):
        for g, side in zip(graphs, sides):
            with torch.cuda.stream(side.st):
                g.replay()
    torch.cuda.synchronize()
    for side in sides:
        side.check()
    assert ddg.lib().ddg_gemm_status() == 0


# ---------------------------------------------------------------- long calls

def big(bw, *n, seed=0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed + sum(n))
    dt = torch.int32 if bw == 32 else torch.int64
    return torch.randint(-(1 << 31), (1 << 31) - 1, n, dtype=dt, device="cuda", generator=g)


def host(t):
    return t.cpu().numpy().astype(np.int64).view(np.uint64)


@pytest.mark.parametrize("bw", [32, 64])
@pytest.mark.parametrize("T,C", [(2048, 1), (262144, 128), (262100, 128)])
def test_linattn_most_chunks(ddg, cuda, bw, T, C):
    """2048 chunks: the longest prompt of one call, and as many chunks of one token"""
    rng = np.random.default_rng(T + C + bw)
    B, H, dk, dv, nc = 1, 2, 2, 3, 2048
    s, sh = R.Shape(B, H, T, dk, dv, C), ddg.LinattnShape(B, H, T, dk, dv, C, T)
    pow_, x, rx = rnd(rng, bw, H, T + 1), rnd(rng, bw, B, T, s.width), rnd(rng, bw, B, T, s.width)
    kd, rkd, ps, rps = (rnd(rng, bw, n) for n in (s.n_decayed, s.n_decayed, s.n_ps, s.n_ps))
    s0, rs0, z, z2 = (rnd(rng, bw, n) for n in (s.n_state, s.n_state, s.n_ps, T * H * dv))
    d = [to_dev(i) for i in (pow_, x, rx, kd, rkd, ps, rps, s0, rs0, z, z2)]
    dp, dx, drx, dkd, drkd, dps, drps, ds0, drs0, dz, dz2 = (ptr(i) for i in d)
    o1, o2 = dev_bytes(2 * s.n_decayed * bw // 8), dev_bytes(s.n_ps * bw // 8)
    ddg.linattn_decay(bw, sh, s.width, dp, dx, ptr(o1))
    ddg.linattn_carry(bw, sh, dp, dps, ds0, ptr(o2))
    ddg.linattn_chunk_share(bw, 0, sh, s.width, dx, drx, dkd, drkd, dz, dz)
    ddg.linattn_output_share(bw, 1, sh, s.width, dx, drx, dkd, drkd, dps, drps, ds0, drs0, dz2, dz2)
    assert np.array_equal(from_dev(o1, ring_dt(bw), 2 * s.n_decayed), R.ring(R.decay(s, pow_, x), bw))
    assert np.array_equal(from_dev(d[9], z.dtype, z.size), R.ring(R.chunk_share(s, 0, x, rx, kd, rkd) + z, bw))
    assert np.array_equal(from_dev(d[10], z.dtype, z2.size),
                          R.ring(R.output_share(s, 1, x, rx, kd, rkd, ps, rps, s0, rs0) + z2, bw))
    # the carry: every chunk's state as one product with the decays from chunk to chunk
    got, p64, U = from_dev(o2, ring_dt(bw), s.n_ps), pow_.astype(np.uint64), np.uint64
    full, st = s.split_ps(ps)
    ends = np.array([e for _, e in s.spans])
    gap = ends[:, None] - ends[None, :]
    for h in range(H):
        w = np.where(gap >= 0, p64[h][np.maximum(gap, 0)], U(0))
        want = R.mm(w, st[:, 0, h].reshape(nc, -1))
        want += p64[h][ends][:, None] * s0.astype(np.uint64).reshape(H, -1)[h][None, :]
        assert np.array_equal(got[s.n_scores:].reshape(nc, H, -1)[:, h], R.ring(want, bw))
    i, j = np.tril_indices(C)
    gaps = np.concatenate([(i - j)[:m * (m + 1) // 2] for m in np.diff(np.concatenate([[0], ends]))])
    want = ps[:s.n_scores].astype(np.uint64).reshape(H, -1) * p64[:, gaps]
    assert np.array_equal(got[:s.n_scores].reshape(H, -1), R.ring(want, bw))
    assert ddg.lib().ddg_gemm_status() == 0


def test_fc_q4_offsets_beyond_32_bits(ddg, cuda, room):
    """4.9 GB of codes under one row; 2.9 G outputs, in place"""
    import torch

    for M, K, N in ((1, 16384, 600001), (700001, 64, 4100)):
        q = torch.randint(0, 256, (N, K // 2), device="cuda", dtype=torch.uint8)
        st = torch.randint(0, 4096, (K // 32, N), device="cuda", dtype=torch.int16)
        x, C, m, n = big(32, M, K), big(32, M, N), min(M, 300), min(N, 300)
        was = C[-m:, -n:].clone()
        torch.cuda.synchronize()
        ddg.fc_q4_share(32, 0, M, ddg.Q4Weights(K, N, 32, ptr(q), ptr(st), None), ptr(x), K, ptr(C), ptr(C))
        code = torch.stack((q[-n:] & 15, q[-n:] >> 4), 2).reshape(n, K).double() - 8
        W, want = code.t() * st[:, -n:].double().repeat_interleave(32, 0), was.long()
        for i in range(2):  # 2^16 x 2^15 x K < 2^53: exact
            want = want + (torch.matmul(((x[-m:].long() >> (16 * i)) & 0xFFFF).double(), W).long() << (16 * i))
        same = bool(torch.equal(C[-m:, -n:], want.to(torch.int32)))
        assert same
        del q, st, x, C
        torch.cuda.empty_cache()
    assert ddg.lib().ddg_gemm_status() == 0


def test_linattn_offsets_beyond_32_bits(ddg, cuda, room):
    """128 x 16 heads x 16,384 tokens: 3.2 G elements of q|k|v, 2.4 G of scores and states; the last head's last chunk"""
    import torch

    B, H, T, dk, dv, C = 128, 16, 16384, 32, 32, 128
    s = R.Shape(1, 1, C, dk, dv, C)  # what is compared
    sh = ddg.LinattnShape(B, H, T, dk, dv, C, T)
    size = ddg.linattn_sizes(sh)
    assert size["qkv"] > 1 << 31 and size["ps"] > 1 << 31
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 90 GB of device memory")
    width, tri, bh = H * 96, (T // C) * (C * (C + 1) // 2), B * H
    pow_ = rnd(np.random.default_rng(2), 32, H, T + 1)
    dp, x, rx = to_dev(pow_), big(32, B * T, width), big(32, B * T, width, seed=1)
    kd, rkd = big(32, 2, bh, T, dk), big(32, 2, bh, T, dk, seed=1)
    ps, rps, z = big(32, size["ps"]), big(32, size["ps"], seed=1), big(32, size["ps"], seed=2)

    def last(t):  # [the last head's last chunk of scores | its state, and the one before]
        a, n = bh * tri, bh * dk * dv
        return [host(t[a - C * (C + 1) // 2:a])] + [host(t[a + c * n - dk * dv:a + c * n]) for c in (T // C, T // C - 1)]

    def tail(t):  # q, k, v of that chunk, as one head's rows
        r = host(t[-C:])
        return np.concatenate([r[:, (o + 1) * H * 32 - 32:(o + 1) * H * 32] for o in range(3)], 1)[None]

    lx, lrx, (p, s_end, s_in), (rp, rs_end, rs_in), z0 = tail(x), tail(rx), last(ps), last(rps), last(z)
    lkd, lrkd = (host(t[:, -1, -C:]) for t in (kd, rkd))
    torch.cuda.synchronize()
    ddg.linattn_chunk_share(32, 0, sh, width, ptr(x), ptr(rx), ptr(kd[1]), ptr(rkd[1]), ptr(z), ptr(z))
    got, want = last(z), R.chunk_share(s, 0, lx, lrx, lkd[1], lrkd[1])
    assert np.array_equal(R.ring(got[0], 32), R.ring(want[:s.n_scores] + z0[0], 32))
    assert np.array_equal(R.ring(got[1], 32), R.ring(want[s.n_scores:] + z0[1], 32))
    ddg.linattn_carry(32, sh, ptr(dp), ptr(ps), None, ptr(z))
    got = last(z)
    i, j = np.tril_indices(C)
    lam = pow_[-1].astype(np.uint64)
    assert np.array_equal(R.ring(got[0], 32), R.ring(p * lam[i - j], 32))
    n, nc = bh * dk * dv, T // C
    st = np.stack([host(ps[bh * tri + (c + 1) * n - dk * dv:bh * tri + (c + 1) * n]) for c in range(nc)])
    assert np.array_equal(R.ring(got[1], 32), R.ring(R.mm(lam[T - C * (1 + np.arange(nc))][None], st)[0], 32))
    out = big(32, B * T, H * dv, seed=3)
    o0 = host(out[-C:, -dv:])
    torch.cuda.synchronize()
    ddg.linattn_output_share(32, 0, sh, width, ptr(x), ptr(rx), ptr(kd), ptr(rkd), ptr(ps), ptr(rps), None, None,
                             ptr(out), ptr(out))
    join = lambda a, b: np.concatenate([a, b])  # noqa: E731
    want = R.output_share(s, 0, lx, lrx, lkd[0], lrkd[0], join(p, s_in), join(rp, rs_in), s_in, rs_in)
    assert np.array_equal(R.ring(host(out[-C:, -dv:]), 32).reshape(-1), R.ring(want + o0.reshape(-1), 32))
    ddg.linattn_decay(32, sh, width, ptr(dp), ptr(x), ptr(kd))
    w2 = lx.copy()
    w2[0, :, :dk] *= lam[1:C + 1, None]
    w2[0, :, dk:2 * dk] *= lam[C - 1::-1, None][:C]
    for half in (0, 1):
        assert np.array_equal(R.ring(host(kd[half, -1, -C:]), 32), R.ring(w2[0, :, half * dk:(half + 1) * dk], 32))
    assert ddg.lib().ddg_gemm_status() == 0
