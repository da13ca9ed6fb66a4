"""GPU tests of decode attention behind a prefix that a kernel of its own reads (more than 32 rows, a row being one
query head of one sequence per key head) while k_decode runs beside it: what surrounds such a call."""
import numpy as np
import pytest

import sptmm_b200 as sp

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import NAN, TYPES, Batch, attend, check, i32, randn      # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()


def batch(lengths, prefix, H, Hk, D, dtype, page, **kw):
    b = Batch(lengths, prefix, H, Hk, D, dtype, page, **kw)
    assert prefix and b.B * (H // Hk) > 32, "the prefix's own kernel"
    return b


def test_steps_with_other_lengths_pages_and_queries():
    """rotate -> decode with SPTMM_LAUNCH_PDL, many steps in a row over the same buffers, whose lengths, page tables and
    queries change from step to step: every step sees its own."""
    H, Hk, D, page, dtype, B, prefix, rounds = 8, 2, 128, 16, sp.F16, 20, 600, 12
    rng = np.random.default_rng(3)
    most = rng.integers(1, 300, size=B)
    steps = [np.maximum(1, (most * rng.random(B)).astype(int)) for _ in range(rounds)]
    orders = [rng.permutation(B) for _ in range(rounds)]                 # whose pages a row of the table names
    side = torch.cuda.Stream()
    xs = [randn(50 + r, B, (H + 2 * Hk) * D, dtype=sp.F32) for r in range(rounds)]
    inv, pos = np.array([10000.0 ** (-i / 64) for i in range(64)]), i32(list(range(600, 600 + B)))

    def program(flags, wait):
        b = batch(most.tolist(), prefix, H, Hk, D, dtype, page, seed=5)
        for t in (b.k, b.v):
            t.nan_to_num_(nan=0.25)                              # a row may be shorter than the sequence whose pages it names, or longer
        rows, lens = [b.table[torch.from_numpy(o).cuda()].contiguous() for o in orders], [i32(s.tolist()) for s in steps]
        spare_k, spare_v = torch.zeros((2, B, Hk * D), dtype=torch.float16, device="cuda")
        keep = torch.zeros((rounds,) + tuple(b.out.shape), dtype=b.out.dtype, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for r in range(rounds):
                b.len.copy_(lens[r])
                b.table.copy_(rows[r])
                sp.rotate_heads(xs[r], B, H, Hk, D, pos, inv, b.q, dtype=dtype, K=spare_k, V=spare_v, flags=flags, stream=side.cuda_stream)
                if wait:
                    torch.cuda.synchronize()
                b.call(side.cuda_stream, flags)
                if wait:
                    torch.cuda.synchronize()
                keep[r].copy_(b.out)
        torch.cuda.synchronize()
        return keep

    want = program(0, True)
    assert torch.isfinite(want).all() and not torch.equal(want[0], want[1])
    for flags in (0, sp.LAUNCH_PDL):
        for _ in range(3):
            assert torch.equal(program(flags, False), want)
