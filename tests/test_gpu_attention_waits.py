"""What an attention call does when a wait inside it runs out: it ends by itself, the status word says so once, and the
next call is right.  No load or product is made to fail: with a limit of one look a CTA's time has run out before its
first tile has come from memory (sptmm_attention_set_wait_limit)."""
import pytest

import sptmm_b200 as sp

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import TYPES, Batch, attend, check, i32, offsets, randn      # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()


@pytest.fixture
def one_look():
    def limited(call):
        assert sp.attention_status() == 0
        sp.attention_set_wait_limit(1)
        try:
            call()
        finally:
            sp.attention_set_wait_limit(0)
        assert sp.attention_status() == 1                        # waits for the device: the call came back by itself
        assert sp.attention_status() == 0                        # read once
    yield limited
    sp.attention_set_wait_limit(0)


@TYPES
@pytest.mark.parametrize("lengths,context,H,Hk,D", [
    ([100] * 40, [], 4, 2, 128),                                 # an item to a CTA, one block of keys
    ([300] * 40, [700] * 40, 4, 2, 64),                          # many blocks
    ([300] * 40, [700] * 40, 4, 2, 128),
    ([40], [3000], 4, 2, 128),                                   # CTAs of a cluster share the keys
    ([300], [2000], 2, 1, 64),
])
def test_prompt_ends_by_itself(lengths, context, H, Hk, D, dtype, one_look):
    qo, ko = offsets(lengths), offsets([n + c for n, c in zip(lengths, context or [0] * len(lengths))])
    T, Tk = qo[-1], ko[-1]
    wide = torch.full((T + 64, H, D), 11.0, dtype=torch.float16, device="cuda").to(randn(0, 1, dtype=dtype).dtype)
    q, k, v, out = randn(1, T, H, D, dtype=dtype), randn(2, Tk, Hk, D, dtype=dtype), randn(3, Tk, Hk, D, dtype=dtype), wide[:T]
    dq, dk = i32(qo), i32(ko)
    call = lambda: sp.attention_prompt(q, k, v, out, dq, dk, len(lengths), T, Tk, H, Hk, D, dtype=dtype)
    for _ in range(2):
        one_look(call)
        out.fill_(11.0)
        call()
        torch.cuda.synchronize()
        for s in (0, len(lengths) - 1):
            for i in (0, lengths[s] // 2, lengths[s] - 1):
                a, c, top = qo[s] + i, ko[s], ko[s + 1] - ko[s] - lengths[s] + i + 1
                check(out[a:a + 1], *attend(q[a:a + 1], k[c:c + top], v[c:c + top], dtype, D ** -0.5, False))
        assert (wide[T:] == 11).all() and sp.attention_status() == 0


@TYPES
def test_decode_behind_a_prefix_ends_by_itself(dtype, one_look):
    for prefix, D in ((100, 128), (3000, 128), (3000, 64)):
        b = Batch([30, 0, 200] * 5, prefix, 8, 2, D, dtype, 16)
        for _ in range(2):
            one_look(b.call)
            b.workspace.fill_(255)
            b.call()
            b.verify()
            assert sp.attention_status() == 0


def test_limits_that_run_out_here_and_there():
    """Limits of about a CTA's time: some give up, wherever they are by then, with loads and products on their way, and
    others do not.  Results are right where no limit ran out, and the next call is right."""
    q, k, v = randn(1, 5000, 4, 128), randn(2, 5000, 2, 128), randn(3, 5000, 2, 128)
    off = i32(offsets([500] * 10))
    out, few, long = torch.zeros_like(q), torch.zeros_like(q[:40]), i32([0, 5000])
    b = Batch([30, 0, 200] * 5, 2000, 8, 2, 128, sp.F16, 16)
    calls = [(out, lambda: sp.attention_prompt(q, k, v, out, off, off, 10, 5000, 5000, 4, 2, 128)),
             (few, lambda: sp.attention_prompt(q, k, v, few, i32([0, 40]), long, 1, 40, 5000, 4, 2, 128)), (b.out, b.call)]
    for result, call in calls:
        call()
        assert sp.attention_status() == 0
        want, ran_out = result.clone(), []
        for polls in (1, 3, 10, 20, 30, 45, 60, 80, 100, 130, 160, 200, 250, 300, 400, 600, 1000, 2000, 10000000):
            sp.attention_set_wait_limit(polls)
            try:
                call()
            finally:
                sp.attention_set_wait_limit(0)
            status = sp.attention_status()
            assert status in (0, 1) and (status or torch.equal(result, want)), polls
            ran_out.append(status)
            result.zero_()
            call()
            assert sp.attention_status() == 0 and torch.equal(result, want), polls
        assert ran_out[0] == 1 and ran_out[-1] == 0


def test_a_captured_call_keeps_its_limit(one_look):
    T, H, Hk, D = 500, 2, 1, 128
    q, k, v = randn(1, T, H, D), randn(2, T, Hk, D), randn(3, T, Hk, D)
    out, off, graph, side = torch.zeros_like(q), i32([0, T]), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    call = lambda stream=0: sp.attention_prompt(q, k, v, out, off, off, 1, T, T, H, Hk, D, stream=stream)
    call()
    torch.cuda.synchronize()
    want = out.clone()
    with torch.cuda.graph(graph, stream=side):
        call(torch.cuda.current_stream().cuda_stream)
    sp.attention_set_wait_limit(1)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert sp.attention_status() == 0 and torch.equal(out, want)
