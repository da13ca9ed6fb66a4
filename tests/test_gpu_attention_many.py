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


def test_no_keys_at_all_and_only_empty_sequences():
    T, H, Hk, D = 37, 4, 2, 64
    q, out = randn(1, T, H, D), torch.full((T, H, D), 11.0, dtype=torch.float16, device="cuda")
    for causal in (True, False):
        out.fill_(11.0)
        sp.attention_prompt(q, None, None, out, i32([0, 30, 30, 33]), i32([0, 0, 0, 0]), 3, T, 0, H, Hk, D, causal=causal)
        torch.cuda.synchronize()
        assert (out[:33] == 0).all() and (out[33:] == 11).all()
    out.fill_(11.0)
    k = randn(2, T, Hk, D)
    for n in (1, 7, 40):
        sp.attention_prompt(q, k, k, out, i32([5] * (n + 1)), i32([9] * (n + 1)), n, T, T, H, Hk, D)
    torch.cuda.synchronize()
    assert (out == 11).all()


def test_rows_beyond_32_bit_offsets():
    """Q, K, V and O as column ranges of one buffer whose rows lie so far apart that the last ones pass 2^32 elements;
    a value that is not finite among the last keys, so that the rows that do not see it go one by one."""
    T, ld, H, Hk, D = 70000, 65536, 2, 1, 128
    buf = torch.empty((T, ld), dtype=torch.float16, device="cuda")               # 9.2 GB, of which a hundredth is looked at
    q, k, v, o = (buf[:, a:a + n * D] for a, n in ((0, H), (256, Hk), (512, Hk), (1024, H)))
    for i, t in enumerate((q, k, v)):
        t.copy_(randn(i, T, t.shape[1]))
    starts = [0, 69000, T]
    off = i32(starts)
    v[T - 3, 5] = float("inf")
    o.fill_(11.0)
    sp.attention_prompt(q, k, v, o, off, off, 2, T, T, H, Hk, D, ldq=ld, ldk=ld, ldv=ld, ldo=ld)
    torch.cuda.synchronize()
    for i in (68999, 69000, 69500, T - 200, T - 4):
        a = max(s for s in starts if s <= i)
        check(o[i:i + 1].reshape(1, H, D), *attend(q[i:i + 1].reshape(1, H, D), k[a:i + 1].reshape(-1, Hk, D), v[a:i + 1].reshape(-1, Hk, D), sp.F16, D ** -0.5, False))
    assert not torch.isfinite(o[T - 3:].reshape(3, H, D)[..., 5]).any()
    # few queries: CTAs of a cluster share the far keys
    sp.attention_prompt(q[T - 40:], k, v, o[T - 40:], i32([0, 40]), i32([0, T]), 1, 40, T, H, Hk, D, ldq=ld, ldk=ld, ldv=ld, ldo=ld)
    torch.cuda.synchronize()
    for i in (T - 40, T - 4):
        check(o[i:i + 1].reshape(1, H, D), *attend(q[i:i + 1].reshape(1, H, D), k[:i + 1].reshape(-1, Hk, D), v[:i + 1].reshape(-1, Hk, D), sp.F16, D ** -0.5, False))
    del buf, q, k, v, o
    torch.cuda.empty_cache()
