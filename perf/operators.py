"""Workloads of the share-level operators for a secure token model: fully connected layers with 4-bit
public weights, and linear attention with a decay per head, for prompts and for single tokens.

Everything is arithmetic over Z_2^bw (bw 32 or 64; held in int32 / int64).  A wire x is held as its
masked value x + r, uniform over the ring, and each party's additive share of r.  One pass is one
party's local computation between two openings, as a party runs it; ring results have to be equal
bit for bit.

Sizes: 376 -> 1024 and 1024 -> 512 are layers of the affinity model's head, 138 its longest node
sequence, 47 its first hidden width over four heads; the others are generic transformer widths.
"""
import importlib
import math

import torch

own = False

SCALE = 12   # fixed-point bits of the affinity model
CHUNK = 128  # tokens of one attention chunk


# ---------------------------------------------------------------- cases

def listed():
    fc, pr, st = "fc_q4", "prompt", "step"
    return [
        # one sample through the drug head's first layer: a single launch, latency only
        _fc("fc_q4 head layer, 1 row", 32, 1, 376, 1024, 32),
        # one token's projection in a wide layer: reading the weights is all of it
        _fc("fc_q4 wide, 1 row, Z_2^64", 64, 1, 4096, 4096, 128),
        # a few requests decoded together
        _fc("fc_q4 wide, 16 rows", 32, 16, 4096, 8192, 128),
        # the fusion head at the batch of the headline benchmark
        _fc("fc_q4 fusion layer, 256 rows", 32, 256, 1024, 512, 64),
        # odd sizes: a last group that is cut short, rows that end inside a vector
        _fc("fc_q4 ragged, 37 rows, Z_2^64", 64, 37, 1003, 777, 32),
        # a prompt's projection
        _fc("fc_q4 prompt, 2048 rows", 32, 2048, 4096, 4096, 128),
        # one token, one request, a small model: latency
        _la("step, 1 x 4 heads", st, 32, 0, 1, 4, 1, 47, 47),
        # a batch of requests decoded together
        _la("step, 64 x 16 heads", st, 32, 0, 64, 16, 1, 128, 128),
        _la("step, 32 x 16 heads, Z_2^64", st, 64, 1, 32, 16, 1, 64, 128),
        # the node sequence of one sample
        _la("prompt, 1 x 4 x 138", pr, 32, 0, 1, 4, 138, 47, 47),
        # a batch of long prompts
        _la("prompt, 4 x 16 x 2048", pr, 32, 1, 4, 16, 2048, 64, 64),
        # the wide ring, a last chunk that is cut short
        _la("prompt, 2 x 8 x 1111, Z_2^64", pr, 64, 0, 2, 8, 1111, 128, 64),
    ]


def _fc(name, bw, rows, k, n, group):
    return {"name": name, "op": "fc_q4", "bw": bw, "rows": rows, "k": k, "n": n, "group": group}


def _la(name, op, bw, party, batch, heads, tokens, dk, dv):
    return {"name": name, "op": op, "bw": bw, "party": party, "batch": batch, "heads": heads, "tokens": tokens,
            "dk": dk, "dv": dv}


def _spread(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    bw = rng.choice((32, 32, 64))
    op = rng.choice(("fc_q4", "fc_q4", "step", "prompt"))
    if op == "fc_q4":
        c = _fc("", bw, _spread(rng, 1, 1024), _spread(rng, 64, 4096), _spread(rng, 64, 4096),
                rng.choice((32, 64, 128)))
    elif op == "step":
        dk, dv = rng.choice((32, 47, 64, 94, 128)), rng.choice((32, 47, 64, 94, 128))
        c = _la("", op, bw, rng.randrange(2), _spread(rng, 1, 32), _spread(rng, 1, 16), 1, dk, dv)
    else:
        dk, dv = rng.choice((32, 47, 64, 94, 128)), rng.choice((32, 47, 64, 94, 128))
        tokens = _spread(rng, 2, 1024)
        c = _la("", op, bw, rng.randrange(2), rng.randint(1, 2), rng.randint(1, 12), tokens, dk, dv)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs

def _dtype(case):
    return torch.int32 if case["bw"] == 32 else torch.int64


def _ring(gen, case, *shape):
    """uniform ring elements"""
    lim = 1 << (case["bw"] - 1)
    return torch.randint(-lim, lim - 1, shape, dtype=_dtype(case), device="cuda", generator=gen)


def _chunks(case):
    t = case["tokens"]
    return [(a, min(a + CHUNK, t)) for a in range(0, t, CHUNK)]


def _tri(case):
    """entries of the causal score triangles of one head"""
    return sum((b - a) * (b - a + 1) // 2 for a, b in _chunks(case))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "fc_q4":
        k, n, g, m = case["k"], case["n"], case["group"], case["rows"]
        row = 16 * ((k + 31) // 32)  # bytes of one output's weights: 2 per byte, 32 per 16 bytes
        q = torch.randint(0, 256, (n, row), dtype=torch.int32, device="cuda", generator=gen).to(torch.uint8)
        ng = (k + g - 1) // g
        sc = torch.randint(8, 400, (ng, n), dtype=torch.int32, device="cuda", generator=gen)
        sc[:, ::61] = 4095  # outliers: the largest step that a group can have
        s.update(q=q, scale=sc.to(torch.int16), bias=_ring(gen, case, n), x=_ring(gen, case, m, k),
                 c=_ring(gen, case, m, n), out=torch.empty(m, n, dtype=_dtype(case), device="cuda"))
        return s
    b, h, t, dk, dv = (case[i] for i in ("batch", "heads", "tokens", "dk", "dv"))
    lam = 1.0 - torch.pow(2.0, -5.0 - 3.0 * torch.rand(h, dtype=torch.float64, device="cuda", generator=gen))
    e = torch.arange(t + 1, dtype=torch.float64, device="cuda")
    s["pow"] = torch.round(torch.pow(lam[:, None], e) * (1 << SCALE)).to(_dtype(case)).contiguous()
    width = h * (2 * dk + dv)
    s["qkv"], s["qkv_ms"] = _ring(gen, case, b, t, width), _ring(gen, case, b, t, width)
    s["s0"], s["s0_ms"] = _ring(gen, case, b, h, dk, dv), _ring(gen, case, b, h, dk, dv)
    empty = lambda n: torch.empty(n, dtype=_dtype(case), device="cuda")  # noqa: E731
    if case["op"] == "step":
        n1, n2 = b * h * (dk * dv + dv + 1), b * h * dv
        s["yw"], s["yw_ms"] = _ring(gen, case, b * h * (dv + 1)), _ring(gen, case, b * h * (dv + 1))
        s["z1"], s["z2"], s["out1"], s["out2"] = _ring(gen, case, n1), _ring(gen, case, n2), empty(n1), empty(n2)
        return s
    nd, ns = b * h * t * dk, b * h * (_tri(case) + len(_chunks(case)) * dk * dv)
    s["qkd"], s["qkd_ms"] = _ring(gen, case, 2 * nd), _ring(gen, case, 2 * nd)      # decayed q | decayed k
    s["pds"] = _ring(gen, case, ns)                                                # scores | chunk states, opened
    s["ps"], s["ps_ms"] = _ring(gen, case, ns), _ring(gen, case, ns)               # decayed scores | carried states
    s["z1"], s["z2"] = _ring(gen, case, ns), _ring(gen, case, b * t * h * dv)
    s["out0"], s["out1"], s["out2"], s["out3"] = empty(2 * nd), empty(ns), empty(ns), empty(b * t * h * dv)
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"fc_q4": _own_fc, "step": _own_step, "prompt": _own_prompt}[op](state)
    return {"fc_q4": _plain_fc, "step": _plain_step, "prompt": _plain_prompt}[op](state)


_ddg = None


def _lib():
    global _ddg
    if _ddg is None:
        _ddg = importlib.import_module("idash26-track3_b200")
    return _ddg


def _own_fc(s):
    d, c = _lib(), s["case"]
    w = d.Q4Weights(c["k"], c["n"], c["group"], s["q"].data_ptr(), s["scale"].data_ptr(), s["bias"].data_ptr())
    d.fc_q4_share(c["bw"], 0, c["rows"], w, s["x"].data_ptr(), c["k"], s["c"].data_ptr(), s["out"].data_ptr())
    return s["out"]


def _shape(d, c):
    return d.LinattnShape(c["batch"], c["heads"], c["tokens"], c["dk"], c["dv"], CHUNK, c["tokens"])


def _own_step(s):
    d, c = _lib(), s["case"]
    sh, ld, p = _shape(d, c), s["qkv"].shape[-1], c["party"]
    d.linattn_step_share(c["bw"], p, sh, ld, s["pow"].data_ptr(), s["qkv"].data_ptr(), s["qkv_ms"].data_ptr(),
                         s["s0"].data_ptr(), s["s0_ms"].data_ptr(), s["z1"].data_ptr(), s["out1"].data_ptr())
    d.linattn_step_output_share(c["bw"], p, sh, ld, s["pow"].data_ptr(), s["qkv"].data_ptr(),
                                s["qkv_ms"].data_ptr(), s["yw"].data_ptr(), s["yw_ms"].data_ptr(),
                                s["z2"].data_ptr(), s["out2"].data_ptr())
    return s["out1"], s["out2"]


def _own_prompt(s):
    d, c = _lib(), s["case"]
    sh, ld, p = _shape(d, c), s["qkv"].shape[-1], c["party"]
    half = s["qkd"].numel() // 2 * s["qkd"].element_size()
    qd, qd_ms = s["qkd"].data_ptr(), s["qkd_ms"].data_ptr()
    d.linattn_decay(c["bw"], sh, ld, s["pow"].data_ptr(), s["qkv"].data_ptr(), s["out0"].data_ptr())
    d.linattn_chunk_share(c["bw"], p, sh, ld, s["qkv"].data_ptr(), s["qkv_ms"].data_ptr(), qd + half, qd_ms + half,
                          s["z1"].data_ptr(), s["out1"].data_ptr())
    d.linattn_carry(c["bw"], sh, s["pow"].data_ptr(), s["pds"].data_ptr(), s["s0"].data_ptr(), s["out2"].data_ptr())
    d.linattn_output_share(c["bw"], p, sh, ld, s["qkv"].data_ptr(), s["qkv_ms"].data_ptr(), qd, qd_ms,
                           s["ps"].data_ptr(), s["ps_ms"].data_ptr(), s["s0"].data_ptr(), s["s0_ms"].data_ptr(),
                           s["z2"].data_ptr(), s["out3"].data_ptr())
    return s["out0"], s["out1"], s["out2"], s["out3"]


# ---------------------------------------------------------------- plain form
#
# Ring products from 16-bit limbs: the limb products are exact in float64 (sums below 2^53), and
# their shifted sum in int64 wraps modulo 2^64, so the low bw bits are the ring's.

def _limbs(a, count):
    return [((a.to(torch.int64) >> (16 * i)) & 0xffff).to(torch.float64) for i in range(count)]


def _mm(a, b, bw):
    """a . b modulo 2^64, exact in its low bw bits"""
    count = bw // 16
    x, y = _limbs(a, count), _limbs(b, count)
    return sum(torch.matmul(x[i], y[j]).to(torch.int64) << (16 * (i + j))
               for i in range(count) for j in range(count - i))


def _beaver(a, ra, b, rb, party, bw):
    """one party's share of (a - r_a) . (b - r_b), without the dealer's word"""
    left = b - rb if party == 0 else -rb
    return _mm(a, left, bw) - _mm(ra, b, bw)


def _plain_fc(s):
    c = s["case"]
    k, n, g = c["k"], c["n"], c["group"]
    q = torch.stack((s["q"] & 15, s["q"] >> 4), dim=2).reshape(n, -1)[:, :k].to(torch.float64) - 8
    step = s["scale"].to(torch.float64).repeat_interleave(g, dim=0)[:k]
    w = q.t() * step
    x = _limbs(s["x"], c["bw"] // 16)
    y = sum(torch.matmul(v, w).to(torch.int64) << (16 * i) for i, v in enumerate(x))
    return (y + s["bias"].to(torch.int64) + s["c"].to(torch.int64)).to(_dtype(c))


def _split_qkv(x, c):
    """(b, t, width) -> q, k (b, h, t, dk) and v (b, h, t, dv), in 64 bits"""
    b, t, h, dk, dv = x.shape[0], x.shape[1], c["heads"], c["dk"], c["dv"]
    q, k, v = x.to(torch.int64).split((h * dk, h * dk, h * dv), dim=2)
    return tuple(y.reshape(b, t, h, -1).transpose(1, 2) for y in (q, k, v))


def _plain_step(s):
    c = s["case"]
    b, h, dk, dv, party = c["batch"], c["heads"], c["dk"], c["dv"], c["party"]
    q, k, v = (y[:, :, 0] for y in _split_qkv(s["qkv"], c))
    rq, rk, rv = (y[:, :, 0] for y in _split_qkv(s["qkv_ms"], c))
    st, rs = s["s0"].to(torch.int64), s["s0_ms"].to(torch.int64)
    lam = s["pow"][:, 1].to(torch.int64)
    p0 = 1 if party == 0 else 0
    u = (k[..., None] * (p0 * v - rv)[..., None, :] - rk[..., None] * v[..., None, :]
         + p0 * lam[:, None, None] * st)
    y = (q[..., None] * (p0 * st - rs) - rq[..., None] * st).sum(2)
    w = (q * (p0 * k - rk) - rq * k).sum(2)
    one = torch.cat([i.reshape(-1) for i in (u, y, w)]) + s["z1"]
    ny = b * h * dv
    yv = s["yw"][:ny].reshape(b, h, dv).to(torch.int64)
    wv, wr = (i[ny:].reshape(b, h, 1).to(torch.int64) for i in (s["yw"], s["yw_ms"]))
    two = p0 * lam[:, None] * yv + wv * (p0 * v - rv) - wr * v
    return one.to(_dtype(c)), (two.reshape(-1) + s["z2"]).to(_dtype(c))


def _chunked(x, c):
    """(b, h, t, d) -> (b, h, chunks, CHUNK, d), zeros behind the last token"""
    nc = len(_chunks(c))
    x = torch.nn.functional.pad(x, (0, 0, 0, nc * CHUNK - x.shape[2]))
    return x.reshape(x.shape[0], x.shape[1], nc, CHUNK, x.shape[3])


def _plain_prompt(s):
    c = s["case"]
    b, h, t, dk, dv, party, bw = (c[i] for i in ("batch", "heads", "tokens", "dk", "dv", "party", "bw"))
    nc, dt = len(_chunks(c)), _dtype(c)
    pw = s["pow"].to(torch.int64)
    at = torch.arange(t, device="cuda")
    within, last = at % CHUNK, torch.clamp((at // CHUNK + 1) * CHUNK, max=t)
    q, k, v = _split_qkv(s["qkv"], c)
    rq, rk, rv = _split_qkv(s["qkv_ms"], c)
    out0 = torch.cat([(q * pw[:, within + 1][..., None]).reshape(-1), (k * pw[:, last - 1 - at][..., None]).reshape(-1)])

    qd, kd = (_chunked(y.reshape(b, h, t, dk).to(torch.int64), c) for y in s["qkd"].split(b * h * t * dk))
    rqd, rkd = (_chunked(y.reshape(b, h, t, dk).to(torch.int64), c) for y in s["qkd_ms"].split(b * h * t * dk))
    qc, kc, vc, rqc, rkc, rvc = (_chunked(y, c) for y in (q, k, v, rq, rk, rv))
    i = torch.arange(CHUNK, device="cuda")
    token = torch.arange(nc * CHUNK, device="cuda").reshape(nc, CHUNK)
    keep = (i[None, :, None] >= i[None, None, :]) & (token < t)[:, :, None]
    scores = _beaver(qc, rqc, kc.transpose(3, 4), rkc.transpose(3, 4), party, bw)[:, :, keep]
    states = _beaver(kd.transpose(3, 4), rkd.transpose(3, 4), vc, rvc, party, bw)
    out1 = torch.cat((scores.reshape(-1), states.permute(2, 0, 1, 3, 4).reshape(-1))) + s["z1"]

    nt = b * h * _tri(c)
    gap = (i[:, None] - i[None, :]).clamp(min=0, max=t)
    decay = pw[:, gap][:, None].expand(h, nc, CHUNK, CHUNK)[:, keep]
    pd = s["pds"][:nt].reshape(b, h, -1).to(torch.int64) * decay
    ends = torch.tensor([e for _, e in _chunks(c)], device="cuda")
    between = ends[:, None] - ends[None, :]
    coef = torch.where(between >= 0, pw[:, between.clamp(min=0)], 0)  # (h, nc, nc)
    ds = s["pds"][nt:].reshape(nc, b, h, dk * dv).permute(1, 2, 0, 3)
    s0 = s["s0"].reshape(b, h, 1, dk * dv).to(torch.int64)
    carried = _mm(coef, ds, bw) + pw[:, ends][..., None] * s0
    out2 = torch.cat((pd.reshape(-1), carried.permute(2, 0, 1, 3).reshape(-1)))

    full, rfull = (torch.zeros(b, h, nc, CHUNK, CHUNK, dtype=torch.int64, device="cuda") for _ in range(2))
    full[:, :, keep] = s["ps"][:nt].reshape(b, h, -1).to(torch.int64)
    rfull[:, :, keep] = s["ps_ms"][:nt].reshape(b, h, -1).to(torch.int64)
    st, rst = (torch.cat((a[None], y[nt:].reshape(nc, b, h, dk, dv)[:-1])).permute(1, 2, 0, 3, 4)
               for a, y in ((s["s0"], s["ps"]), (s["s0_ms"], s["ps_ms"])))
    o = _beaver(full, rfull, vc, rvc, party, bw) + _beaver(qd, rqd, st, rst, party, bw)
    o = o.reshape(b, h, nc * CHUNK, dv)[:, :, :t].transpose(1, 2).reshape(-1)
    return out0.to(dt), out1.to(dt), out2.to(dt), (o + s["z2"]).to(dt)


# ---------------------------------------------------------------- the definition, apart from the plain form
#
# Integer products and sums in int64, which wraps modulo 2^64, one sequence piece at a time.

def _dot(a, b):
    """(..., m, x) . (..., n, x) -> (..., m, n) by products and sums, a few rows at a time"""
    rows = max(1, (1 << 27) // max(1, b.numel()))
    return torch.cat([(a[..., i:i + rows, None, :] * b[..., None, :, :]).sum(-1)
                      for i in range(0, a.shape[-2], rows)], dim=-2)


def _share(a, ra, b, rb, party):
    r = -_dot(a, rb) - _dot(ra, b)
    return r + _dot(a, b) if party == 0 else r


def exact(case, seed):
    s, c = prepare(case, seed), case
    dt = _dtype(c)
    wide = {i: v.to(torch.int64) for i, v in s.items() if torch.is_tensor(v) and not i.startswith("out")}
    if c["op"] == "fc_q4":
        k, n = c["k"], c["n"]
        at = torch.arange(k, device="cuda")
        nibble = (wide["q"][:, at // 2] >> (4 * (at % 2))) & 15
        w = (nibble - 8) * wide["scale"][at // c["group"], :].t()  # (n, k)
        y = torch.cat([_dot(wide["x"], w[i:i + 128]) for i in range(0, n, 128)], dim=1)
        return (y + wide["bias"] + wide["c"]).to(dt)

    b, h, t, dk, dv, p = (c[i] for i in ("batch", "heads", "tokens", "dk", "dv", "party"))
    head = lambda x, o, d: x[:, :, o:o + h * d].reshape(b, t, h, d).permute(0, 2, 1, 3)  # noqa: E731
    q, k, v = (head(wide["qkv"], o, d) for o, d in ((0, dk), (h * dk, dk), (2 * h * dk, dv)))
    rq, rk, rv = (head(wide["qkv_ms"], o, d) for o, d in ((0, dk), (h * dk, dk), (2 * h * dk, dv)))
    pw, s0, rs0 = wide["pow"], wide["s0"], wide["s0_ms"]
    tr = lambda x: x.transpose(-1, -2)  # noqa: E731
    if c["op"] == "step":
        lam = pw[:, 1].reshape(1, h, 1, 1)
        u = _share(tr(k), tr(rk), tr(v), tr(rv), p) + (lam * s0 if p == 0 else 0)
        y = _share(q, rq, tr(s0), tr(rs0), p)
        w = _share(q, rq, k, rk, p)
        one = torch.cat([i.reshape(-1) for i in (u, y, w)]) + wide["z1"]
        y1, w1 = wide["yw"].split((b * h * dv, b * h))
        w1, rw = (i.reshape(b, h, 1, 1) for i in (w1, wide["yw_ms"][b * h * dv:]))
        two = _share(w1, rw, tr(v), tr(rv), p) + (lam * y1.reshape(b, h, 1, dv) if p == 0 else 0)
        return one.to(dt), (two.reshape(-1) + wide["z2"]).to(dt)

    nd, nt = b * h * t * dk, b * h * _tri(c)
    qd, kd, rqd, rkd = (wide[i][a * nd:(a + 1) * nd].reshape(b, h, t, dk) for i in ("qkd", "qkd_ms") for a in (0, 1))
    pds_p, ps_p, ps_pm = (wide[i][:nt].reshape(b, h, -1) for i in ("pds", "ps", "ps_ms"))
    pds_s, ps_s, ps_sm = (wide[i][nt:].reshape(-1, b, h, dk, dv) for i in ("pds", "ps", "ps_ms"))
    dq, dk_, sc, ss, dec, car, outs, pos = [], [], [], [], [], [], [], 0
    run_coef = []
    for n, (a, e) in enumerate(_chunks(c)):
        m = e - a
        i = torch.arange(m, device="cuda")
        dq.append(q[:, :, a:e] * pw[:, 1:m + 1].reshape(1, h, m, 1))
        dk_.append(k[:, :, a:e] * pw[:, :m].flip(1).reshape(1, h, m, 1))
        low = torch.tril_indices(m, m, device="cuda")
        sc.append(_share(q[:, :, a:e], rq[:, :, a:e], k[:, :, a:e], rk[:, :, a:e], p)[:, :, low[0], low[1]])
        ss.append(_share(tr(kd[:, :, a:e]), tr(rkd[:, :, a:e]), tr(v[:, :, a:e]), tr(rv[:, :, a:e]), p))
        size = m * (m + 1) // 2
        dec.append(pds_p[:, :, pos:pos + size] * pw[:, low[0] - low[1]])
        total = pw[:, e].reshape(1, h, 1, 1) * s0
        run_coef.append(e)
        for j, end in enumerate(run_coef):
            total = total + pw[:, e - end].reshape(1, h, 1, 1) * pds_s[j]
        car.append(total)
        full, rfull = (torch.zeros(b, h, m, m, dtype=torch.int64, device="cuda") for _ in range(2))
        full[:, :, low[0], low[1]] = ps_p[:, :, pos:pos + size]
        rfull[:, :, low[0], low[1]] = ps_pm[:, :, pos:pos + size]
        before, rbefore = (s0, rs0) if n == 0 else (ps_s[n - 1], ps_sm[n - 1])
        outs.append(_share(full, rfull, tr(v[:, :, a:e]), tr(rv[:, :, a:e]), p)
                    + _share(qd[:, :, a:e], rqd[:, :, a:e], tr(before), tr(rbefore), p))
        pos += size
    flat = lambda x, d: torch.cat(x, dim=d).reshape(-1)  # noqa: E731
    stack = lambda x: torch.stack(x).reshape(-1)  # noqa: E731
    out0 = torch.cat((flat(dq, 2), flat(dk_, 2)))
    out1 = torch.cat((flat(sc, 2), stack(ss))) + wide["z1"]
    out2 = torch.cat((flat(dec, 2), stack(car)))
    out3 = torch.cat(outs, dim=2).permute(0, 2, 1, 3).reshape(-1) + wide["z2"]
    return out0.to(dt), out1.to(dt), out2.to(dt), out3.to(dt)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    """bytes: each input read once, each output written once; flops: two for each ring multiply-add"""
    c, word = case, case["bw"] // 8
    if c["op"] == "fc_q4":
        m, k, n = c["rows"], c["k"], c["n"]
        weights = n * k / 2 + 2 * n * ((k + c["group"] - 1) // c["group"])
        return {"bytes": weights + word * (m * k + 2 * m * n + n), "flops": 2 * m * k * n}
    b, h, t, dk, dv = (c[i] for i in ("batch", "heads", "tokens", "dk", "dv"))
    qkv, state = b * t * h * (2 * dk + dv), b * h * dk * dv
    p = 1 if c["party"] == 0 else 0
    if c["op"] == "step":
        words = 2 * qkv + 2 * state + 2 * (state + b * h * (dv + 1)) + b * h * (3 * dv + 2)
        return {"bytes": word * words, "flops": 2 * state * (4 + 2 * p)}
    nc, nt = len(_chunks(c)), b * h * _tri(c)
    nd, ns = b * h * t * dk, nt + nc * state
    carry = nt + state * (nc * (nc + 1) // 2 + nc)
    macs = 2 * nd + (2 + p) * (nt * dk + nd * dv) + carry + (2 + p) * (nt * dv + nd * dv)
    # qkv and its mask shares, both decayed operands (written, and read with their shares), the two score
    # and state arrays, the dealer's words, the outputs
    words = 2 * qkv + 2 * nd + 4 * nd + 2 * ns + 2 * ns + 2 * ns + 2 * state + 2 * b * t * h * dv
    return {"bytes": word * words, "flops": 2 * macs}
