"""Integer definitions of the token model's operators in numpy, modulo 2^64.

uint64 arithmetic wraps, and the low 32 bits of a product or sum are those of
the ring Z_2^32, so one restatement serves both rings; `ring` narrows it.
Shapes as in include/ddg_fss.h."""
import numpy as np

U = np.uint64


def ring(a, bw):
    return np.asarray(a, dtype=U).astype(np.uint32 if bw == 32 else np.uint64)


def signed(a, bw):
    return np.asarray(a).astype(np.uint32).view(np.int32).astype(np.int64) if bw == 32 else \
        np.asarray(a, dtype=U).view(np.int64)


def mm(a, b):
    with np.errstate(over="ignore"):
        return np.matmul(np.asarray(a, U), np.asarray(b, U))


def beaver(a, ra, b, rb, party):
    """a . (p0 b - r_b) - r_a . b"""
    right = (np.asarray(b, U) if party == 0 else U(0)) - np.asarray(rb, U)
    return mm(a, right) - mm(ra, b)


# ---------------------------------------------------------------- 4-bit weights

def q4_pack(code):
    """(K, N) codes 0..15 -> (N, row_bytes) uint8, padded with 8 (a zero weight)"""
    K, N = code.shape
    rows = np.full((N, 32 * ((K + 31) // 32)), 8, dtype=np.uint8)
    rows[:, :K] = code.T
    return rows[:, 0::2] | (rows[:, 1::2] << 4)


def q4_weights(code, step, group):
    """int64 weights (K, N)"""
    return (code.astype(np.int64) - 8) * np.repeat(step.astype(np.int64) & 4095, group, axis=0)[:code.shape[0]]


def q4_quantize(w, group):
    """(codes, steps) of an int64 matrix, in Python integers"""
    K, N = w.shape
    ng = (K + group - 1) // group
    code, step = np.zeros((K, N), np.uint8), np.zeros((ng, N), np.uint16)
    for g in range(ng):
        for n in range(N):
            col = [int(v) for v in w[g * group:(g + 1) * group, n]]
            s = min(4095, max(1, -(-max(abs(v) for v in col) // 7)))
            step[g, n] = s
            for i, v in enumerate(col):
                r = (2 * abs(v) + s) // (2 * s)
                code[g * group + i, n] = 8 + max(-8, min(7, r if v >= 0 else -r))
    return code, step


# ---------------------------------------------------------------- linear attention

class Shape:
    def __init__(self, B, H, T, dk, dv, C):
        self.B, self.H, self.T, self.dk, self.dv, self.C = B, H, T, dk, dv, C
        self.spans = [(a, min(a + C, T)) for a in range(0, T, C)]
        self.tri = sum((e - a) * (e - a + 1) // 2 for a, e in self.spans)
        self.width = H * (2 * dk + dv)
        self.n_decayed, self.n_state = B * H * T * dk, B * H * dk * dv
        self.n_scores = B * H * self.tri
        self.n_ps = self.n_scores + len(self.spans) * self.n_state

    def heads(self, x):
        """(B, T, >= width) -> q, k (B, H, T, dk), v (B, H, T, dv)"""
        x = np.asarray(x, U)
        out, o = [], 0
        for d in (self.dk, self.dk, self.dv):
            out.append(x[:, :, o:o + self.H * d].reshape(self.B, -1, self.H, d).transpose(0, 2, 1, 3))
            o += self.H * d
        return out

    def split_ps(self, x):
        """triangles per chunk as full (B, H, m, m) matrices, and states (chunks, B, H, dk, dv)"""
        x = np.asarray(x, U)
        tri, full, pos = x[:self.n_scores].reshape(self.B, self.H, self.tri), [], 0
        for a, e in self.spans:
            m = e - a
            i, j = np.tril_indices(m)
            f = np.zeros((self.B, self.H, m, m), U)
            f[:, :, i, j] = tri[:, :, pos:pos + i.size]
            full.append(f)
            pos += i.size
        return full, x[self.n_scores:].reshape(-1, self.B, self.H, self.dk, self.dv)

    def join_ps(self, full, states):
        tri = [f[:, :, np.tril_indices(f.shape[2])[0], np.tril_indices(f.shape[2])[1]] for f in full]
        return np.concatenate([np.concatenate(tri, axis=2).reshape(-1), np.stack(states).reshape(-1)])


def decay(s, pow_, x):
    q, k, _ = s.heads(x)
    pow_ = np.asarray(pow_, U)
    qd, kd = q.copy(), k.copy()
    for a, e in s.spans:
        qd[:, :, a:e] *= pow_[None, :, 1:e - a + 1, None]
        kd[:, :, a:e] *= pow_[None, :, :e - a][:, :, ::-1, None]
    return np.concatenate([qd.reshape(-1), kd.reshape(-1)])


def chunk_share(s, party, x, rx, kd, rkd):
    """without the dealer's word"""
    (q, k, v), (rq, rk, rv) = s.heads(x), s.heads(rx)
    kd, rkd = (np.asarray(i, U).reshape(s.B, s.H, s.T, s.dk) for i in (kd, rkd))
    t = lambda i: i.swapaxes(-1, -2)  # noqa: E731
    full = [beaver(q[:, :, a:e], rq[:, :, a:e], t(k[:, :, a:e]), t(rk[:, :, a:e]), party) for a, e in s.spans]
    st = [beaver(t(kd[:, :, a:e]), t(rkd[:, :, a:e]), v[:, :, a:e], rv[:, :, a:e], party) for a, e in s.spans]
    return s.join_ps(full, st)


def carry(s, pow_, ps, s0):
    pow_ = np.asarray(pow_, U)
    full, st = s.split_ps(ps)
    out = []
    for f in full:
        m = f.shape[2]
        gap = np.maximum(np.arange(m)[:, None] - np.arange(m)[None, :], 0)
        out.append(f * pow_[:, gap][None])
    states = []
    for c, (_, e) in enumerate(s.spans):
        tot = np.zeros((s.B, s.H, s.dk, s.dv), U)
        if s0 is not None:
            tot += pow_[None, :, e, None, None] * np.asarray(s0, U).reshape(tot.shape)
        for j in range(c + 1):
            tot += pow_[None, :, e - s.spans[j][1], None, None] * st[j]
        states.append(tot)
    return s.join_ps(out, states)


def output_share(s, party, x, rx, qd, rqd, ps, rps, s0, rs0):
    """(B, T, H, dv), without the dealer's word"""
    v, rv = s.heads(x)[2], s.heads(rx)[2]
    qd, rqd = (np.asarray(i, U).reshape(s.B, s.H, s.T, s.dk) for i in (qd, rqd))
    (full, st), (rfull, rst) = s.split_ps(ps), s.split_ps(rps)
    out = np.zeros((s.B, s.H, s.T, s.dv), U)
    for c, (a, e) in enumerate(s.spans):
        out[:, :, a:e] = beaver(full[c], rfull[c], v[:, :, a:e], rv[:, :, a:e], party)
        if c or s0 is not None:
            S, rS = (st[c - 1], rst[c - 1]) if c else (np.asarray(i, U).reshape(s.B, s.H, s.dk, s.dv)
                                                       for i in (s0, rs0))
            out[:, :, a:e] += beaver(qd[:, :, a:e], rqd[:, :, a:e], S, rS, party)
    return out.transpose(0, 2, 1, 3).reshape(-1)


def step_share(s, party, lam, x, rx, S, rS):
    (q, k, v), (rq, rk, rv) = s.heads(x), s.heads(rx)
    S, rS = (np.asarray(i, U).reshape(s.B, s.H, s.dk, s.dv) for i in (S, rS))
    t = lambda i: i.swapaxes(-1, -2)  # noqa: E731
    u = beaver(t(k), t(rk), v, rv, party)
    if party == 0:
        u = u + np.asarray(lam, U)[None, :, None, None] * S
    return np.concatenate([u.reshape(-1), beaver(q, rq, S, rS, party).reshape(-1),
                           beaver(q, rq, t(k), t(rk), party).reshape(-1)])


def step_output_share(s, party, lam, x, rx, yw, ryw):
    v, rv = s.heads(x)[2], s.heads(rx)[2]
    ny = s.B * s.H * s.dv
    yw, ryw = np.asarray(yw, U), np.asarray(ryw, U)
    w, rw = (i[ny:].reshape(s.B, s.H, 1, 1) for i in (yw, ryw))
    o = beaver(w, rw, v, rv, party)
    if party == 0:
        o = o + np.asarray(lam, U)[None, :, None, None] * yw[:ny].reshape(s.B, s.H, 1, s.dv)
    return o.reshape(-1)


# ---------------------------------------------------------------- on cleartext values (signed floors)

def floor_shift(a, scale, bw):
    """floor(a / 2^scale) as ring elements; a within the floors' range"""
    v = signed(ring(a, bw), bw)
    assert np.all(v >= -(1 << (bw - 2))) and np.all(v < (1 << (bw - 2))), "test values leave the floors' range"
    return (v >> scale).astype(np.int64).view(U)


def clear_prompt(s, pow_, x, s0, scale, bw):
    """(out (B, T, H * dv), final state), both at the scale"""
    f = lambda a: floor_shift(a, scale, bw)  # noqa: E731
    z = lambda a: np.zeros(np.asarray(a).shape, U)  # noqa: E731
    x = np.asarray(x, U)
    qkd = f(decay(s, pow_, x))
    qd, kd = qkd[:s.n_decayed], qkd[s.n_decayed:]
    ps = f(carry(s, pow_, f(chunk_share(s, 0, x, z(x), kd, z(kd))), s0))
    o = f(output_share(s, 0, x, z(x), qd, z(qd), ps, z(ps), s0, None if s0 is None else z(s0)))
    return o.reshape(s.B, s.T, s.H * s.dv), ps[s.n_ps - s.n_state:]


def clear_step(s, lam, x, S, scale, bw):
    f = lambda a: floor_shift(a, scale, bw)  # noqa: E731
    z = lambda a: np.zeros(np.asarray(a).shape, U)  # noqa: E731
    x = np.asarray(x, U)
    syw = f(step_share(s, 0, lam, x, z(x), S, z(S)))
    yw = syw[s.n_state:]
    o = f(step_output_share(s, 0, lam, x, z(x), yw, z(yw)))
    return o.reshape(s.B, s.T, s.H * s.dv), syw[:s.n_state]
