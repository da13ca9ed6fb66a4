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


@TYPES
def test_joint_pages_query_stride_and_scale(dtype):
    b = batch([100, 17, 260, 0, 5] * 3, 290, 8, 2, 128, dtype, 32, joint=True, ldq=8 * 128 + 64)
    b.scale = 0.21
    b.call()
    b.verify()


@TYPES
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (8, 4, 64)])
def test_repeat_side_stream_and_graph(H, Hk, D, dtype):
    """Same bits from call to call, on another stream and from a graph; a replay follows other lengths."""
    lengths = [700, 20, 333, 1, 0, 90] * 3
    b = batch(lengths, 300, H, Hk, D, dtype, 16)
    b.call()
    b.verify()
    want = b.out.clone()
    side = torch.cuda.Stream()
    for flags in (0, sp.LAUNCH_PDL):
        b.out.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            b.call(side.cuda_stream, flags)
        torch.cuda.synchronize()
        assert torch.equal(b.out, want)
    for flags in (0, sp.LAUNCH_PDL):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            for _ in range(3):
                b.call(torch.cuda.current_stream().cuda_stream, flags)
        b.out.zero_()
        b.workspace.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b.out, want)
        b.lengths = [100, 20, 0, 1, 0, 3] * 3
        b.len.copy_(i32(b.lengths))
        graph.replay()
        b.verify()
        b.lengths = lengths
        b.len.copy_(i32(lengths))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b.out, want)
        del graph


def test_two_streams_at_once():
    """Calls on two streams, each with a workspace of its own, do not disturb one another."""
    jobs = [batch([900, 3, 50] * 4, 500, 8, 2, 128, sp.F16, 16, seed=1), batch([20, 1200, 7, 64] * 5, 2100, 8, 2, 64, sp.BF16, 32, seed=2)]
    want = []
    for j in jobs:
        j.call()
        j.verify()
        want.append(j.out.clone())
        j.out.zero_()
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for i in range(20):
        for s, j in zip(streams, jobs):
            j.call(s.cuda_stream, sp.LAUNCH_PDL if i % 3 else 0)
    torch.cuda.synchronize()
    for j, w in zip(jobs, want):
        assert torch.equal(j.out, w)


@TYPES
def test_a_row_that_is_not_finite_stays_alone(dtype):
    for D in (64, 128):
        b = batch([100, 33, 70] * 5, 200, 4, 1, D, dtype, 16)
        b.call()
        torch.cuda.synchronize()
        clean = b.out.clone()
        b.q[7, D:2 * D] = NAN                                    # head 1 of sequence 7
        b.q[11, 0] = float("inf")                                # head 0 of sequence 11
        b.call()
        torch.cuda.synchronize()
        assert torch.isnan(b.out[7, 1]).all() and not torch.isfinite(b.out[11, 0]).any()
        b.out[7, 1], b.out[11, 0] = clean[7, 1], clean[11, 0]
        assert torch.equal(b.out, clean)


@TYPES
def test_rising_scores_across_parts(dtype):
    """Scores that rise, or fall, from the prefix's first key to a sequence's last."""
    for sign in (1.0, -1.0):
        b = batch([1000, 40] + [0] * 8, 600, 4, 1, 128, dtype, 16)
        b.q[:] = 1.0
        for pages, n, start in ((b.prefix_pages, 600, 0), (b.rows[0], 1000, 600), (b.rows[1], 40, 600)):
            for i, pg in enumerate(pages):
                m = max(0, min(16, n - 16 * i))
                b.k[pg, :, :m] = 0
                b.k[pg, :, :m, 0] = (sign * 0.5 * (start + 16 * i + torch.arange(m, device="cuda"))).to(b.k.dtype)
        b.call()
        b.verify()


def test_cache_beyond_32_bit_offsets():
    """Element offsets above 2^32: pages very far apart, for the prefix and for the sequences."""
    B, H, Hk, D, page, stride, n_pages = 9, 8, 2, 128, 16, 1 << 27, 35
    buf = torch.empty(stride * (n_pages - 1) + 2 * Hk * page * D, dtype=torch.float16, device="cuda")     # 9.1 GB
    each = Hk * page * D
    pages, q = [0, 33, 31, 34], randn(3, B, H, D)
    kk, vv = randn(1, 4, Hk, page, D), randn(2, 4, Hk, page, D)
    for i, pg in enumerate(pages):
        buf[pg * stride:pg * stride + each] = kk[i].flatten()
        buf[pg * stride + each:pg * stride + 2 * each] = vv[i].flatten()
    cache = sp.KVCache(buf, buf.data_ptr() + 2 * each, n_pages, page, Hk, D, sp.F16, stride)
    k, v = kk.transpose(1, 2).reshape(64, Hk, D), vv.transpose(1, 2).reshape(64, Hk, D)
    want, tol = attend(q, k[:60], v[:60], sp.F16, D ** -0.5, False)
    for prefix, own in ((32, 28), (60, 0)):
        table = i32([pages[2:]] * B)
        out = torch.zeros((B, H, D), dtype=torch.float16, device="cuda")
        ws = torch.empty(sp.attention_decode_workspace(B, H, Hk, D, prefix), dtype=torch.uint8, device="cuda")
        sp.attention_decode(q, out, B, H, cache, i32([own] * B), table, 2, prefix_table=i32(pages), prefix_len=prefix,
                            workspace=ws, workspace_bytes=ws.numel())
        torch.cuda.synchronize()
        check(out, want, tol)
    del buf, cache
    torch.cuda.empty_cache()


def late_schedule(lengths, prefix, H, Hk, D):
    """k_decode's division beside the prefix's kernel, restated (for up to 16 query heads per key head): CTAs that
    find an SM at once, blocks they take more than the late ones, and whether the late ones get any."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    ctas, group = min(2 * sms, 384), H // Hk
    pairs = -(-len(lengths) // (2 * (128 // group)))
    splits = min(max(74 // (pairs * Hk), 1), -(-prefix // 128))
    busy = pairs * Hk * splits
    if busy >= sms:
        return 0, 0, False
    early, lead = min(2 * (sms - busy), ctas), (8 + -(-prefix // (128 * splits)) * 12 // 5) * (1 if D > 64 else 2)
    total = sum((-(-n // 64) + 2) * Hk for n in lengths if n > 0)
    return early, lead, total >= early * lead + ctas


@TYPES
@pytest.mark.parametrize("lengths,prefix,H,Hk,D,late", [
    ([4000] * 36, 1024, 8, 2, 128, True),
    ([9000, 1, 0, 4097] * 12, 500, 8, 2, 64, False),
    ([12000, 1, 0, 6000] * 12, 500, 8, 2, 64, True),
    ([2500] * 34, 8192, 4, 4, 128, True),
    ([4000] * 4 + [10] * 32, 1024, 8, 2, 128, False),
])
def test_uneven_runs_beside_a_long_prefix(lengths, prefix, H, Hk, D, late, dtype):
    """Enough keys of the sequences' own that the CTAs which start when the prefix's kernel ends get some, too, and
    not enough."""
    assert late_schedule(lengths, prefix, H, Hk, D)[2] == late
    b = batch(lengths, prefix, H, Hk, D, dtype, 64)
    b.call()
    torch.cuda.synchronize()
    for i in list(range(0, b.B, 5)) + [b.B - 1]:
        check(b.out[i:i + 1], *b.want(i))
    want = b.out.clone()
    for flags in (0, sp.LAUNCH_PDL):
        b.out.zero_()
        b.workspace.fill_(255)
        b.call(flags=flags)
        torch.cuda.synchronize()
        assert torch.equal(b.out, want)
