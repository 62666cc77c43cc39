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


def test_q4_quantize_of_the_longest_column(ddg, cuda):
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
