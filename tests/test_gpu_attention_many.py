"""GPU tests of prompt attention over many sequences in one call."""
import numpy as np
import pytest

import sptmm_b200 as sp

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import attend, check, i32, offsets, randn      # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()


def case(lengths, context, H, Hk, D, start=0, extra=0):
    qo, ko = offsets(lengths, start), offsets([n + c for n, c in zip(lengths, context)])
    T, Tk = qo[-1] + extra, ko[-1]
    return dict(lengths=lengths, context=context, H=H, Hk=Hk, D=D, qo=qo, ko=ko, T=T, Tk=Tk, q=randn(1, T, H, D, scale=1.5), k=randn(2, Tk, Hk, D),
                v=randn(3, Tk, Hk, D), out=torch.full((T, H, D), 11.0, dtype=torch.float16, device="cuda"), dq=i32(qo), dk=i32(ko))


def run(c, causal=True, stream=0):
    sp.attention_prompt(c["q"], c["k"], c["v"], c["out"], c["dq"], c["dk"], len(c["lengths"]), c["T"], c["Tk"], c["H"], c["Hk"], c["D"],
                        causal=causal, stream=stream)


def verify(c, seqs, causal=True):
    lo, hi = c["qo"][0], c["qo"][-1]
    assert (c["out"][lo:hi] != 11).any(-1).all() and (c["out"][:lo] == 11).all() and (c["out"][hi:] == 11).all()
    for s in seqs:
        n, m, a, k0 = c["lengths"][s], c["lengths"][s] + c["context"][s], c["qo"][s], c["ko"][s]
        for i in sorted({0, n // 3, n - 1}) if n else []:
            top = m - n + i + 1 if causal else m
            check(c["out"][a + i:a + i + 1], *attend(c["q"][a + i:a + i + 1], c["k"][k0:k0 + top], c["v"][k0:k0 + top], sp.F16, c["D"] ** -0.5, False))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n_seqs", [2, 31, 32, 33, 34, 1024, 1025, 1100])
def test_numbers_of_sequences(n_seqs, causal):
    """Either side of the number up to which items are ordered, and of powers of 32; sequences of no token at the
    front, in a row and at the end; rows before the first and behind the last sequence stay as they were."""
    rng = np.random.default_rng(n_seqs)
    lengths = rng.integers(0, 40, size=n_seqs)
    lengths[rng.random(n_seqs) < 0.3] = 0
    lengths[rng.integers(0, n_seqs, size=3)] = [300, 129, 64]
    lengths[[0, -1]] = 0 if n_seqs > 2 else 70
    context = [int(x) for x in rng.integers(0, 200, size=n_seqs) * (rng.random(n_seqs) < 0.2)]
    c = case(lengths.tolist(), context, 4, 2, 64, start=5, extra=7)
    run(c, causal)
    torch.cuda.synchronize()
    longest = int(np.argmax(lengths))
    verify(c, sorted({0, 1, longest, n_seqs // 2, n_seqs - 2, n_seqs - 1} | set(range(0, n_seqs, max(1, n_seqs // 12)))), causal)


def test_65536_sequences():
    """The most that a call takes, in time that grows with their number: one token each, and only one that has any."""
    n = 65536
    c = case([1] * n, [0] * n, 2, 1, 64)
    run(c)
    torch.cuda.synchronize()
    assert torch.equal(c["out"].view(n, 2, 64), c["v"].expand(n, 2, 64))          # a query that sees one key: its value
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    run(c, stream=torch.cuda.current_stream().cuda_stream)
    b.record()
    torch.cuda.synchronize()
    assert a.elapsed_time(b) < 500                               # a few milliseconds; seconds if every CTA looked at all sequences
    lengths = [0] * n
    lengths[50001] = 130
    c = case(lengths, [0] * n, 2, 1, 64, start=3, extra=2)
    run(c)
    torch.cuda.synchronize()
    verify(c, [0, 50000, 50001, 50002, n - 1])


def test_offsets_that_fall_stay_within_the_buffers():
    """Offsets that are not what the call asks for name no row outside Q and K: whatever else is left out, nothing
    beyond the rows is written."""
    rng = np.random.default_rng(1)
    T, H, Hk, D = 500, 2, 1, 64
    wide = torch.full((T + 200, H, D), 11.0, dtype=torch.float16, device="cuda")
    q, k, v = randn(1, T, H, D), randn(2, T, Hk, D), randn(3, T, Hk, D)
    for n_seqs in (5, 60, 1100):
        for _ in range(4):
            off = i32(rng.integers(-100, 800, size=n_seqs + 1).tolist())
            sp.attention_prompt(q, k, v, wide, off, off, n_seqs, T, T, H, Hk, D)
            torch.cuda.synchronize()
            assert (wide[T:] == 11).all()
