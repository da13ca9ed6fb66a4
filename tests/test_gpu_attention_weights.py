"""GPU tests of the attention operators where softmax weights are very unequal, not finite or all zero.

The bound of test_gpu_attention.attend holds where every weight has a type's full precision.  fp16 weights
are kept as 2^(x - m + 9), m the running maximum and x the score in powers of two (csrc/attention.cuh, WeightRange),
so one below 2^-14 there is off by at most half of fp16's smallest step, 2^-25.  m is at most the row's true maximum,
so relative to the largest weight that is at most 2^-25 / 2^9 = 2^-34, and an output may be off by 2^-34 sum |v| / L more,
with L = sum of 2^(x - largest x), at least 1.  bf16 rounds weights of any size alike.  An fp16 output below 2^-14 is
off by 2^-25 at most."""
import pytest

import sptmm_b200 as sp

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import NAN, TYPES, Batch, attend, check, i32, offsets, randn      # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()


def attend_wide(q, k, v, dtype):
    """attend() of rows that see all keys, with the bound for weights below fp16's full precision."""
    want, tol = attend(q, k, v, dtype, q.shape[2] ** -0.5, False)
    if dtype == sp.F16:
        g = q.shape[1] // k.shape[1]
        kk, vv = k.double().repeat_interleave(g, 1), v.double().abs().repeat_interleave(g, 1)
        s = torch.einsum("nhd,mhd->nhm", q.double(), kk) * q.shape[2] ** -0.5
        L = (s - s.max(-1, keepdim=True).values).exp().sum(-1, keepdim=True)
        tol = tol + 2.0 ** -34 * vv.sum(0)[None] / L + 2.0 ** -25
    return want, tol


def sink(q, k, v, at, gap, spread):
    """Key `at` scores `gap` nats above the others, which score about the same (`spread`), and has a value of zero."""
    D = q.shape[-1]
    q *= spread
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[at] = 0.0
    k[at, :, 0] = gap * D ** 0.5 / 8
    v *= 20.0
    v += 30.0
    v[at] = 0.0


GAPS = pytest.mark.parametrize("gap,spread", [(10.0, 0.3), (13.0, 0.0), (15.0, 0.3), (17.5, 0.0), (17.5, 0.3)])


@TYPES
@GAPS
def test_prompt_attention_sink(gap, spread, dtype):
    """The largest weight's value is zero: the output is carried by thousands of weights far below it."""
    for H, Hk, D, lengths, context in ((4, 2, 128, [3], [6000]), (4, 4, 64, [2], [6000]), (4, 4, 128, [1] * 40, [1500] * 40), (6, 3, 64, [1] * 60, [900] * 60)):
        qo, ko = offsets(lengths), offsets([n + c for n, c in zip(lengths, context)])
        q, k, v = randn(1, qo[-1], H, D, dtype=dtype), randn(2, ko[-1], Hk, D, dtype=dtype), randn(3, ko[-1], Hk, D, dtype=dtype)
        sink(q, k, v, torch.tensor(ko[:-1], device="cuda") + 5, gap, spread)
        out = torch.full_like(q, 11.0)
        sp.attention_prompt(q, k, v, out, i32(qo), i32(ko), len(lengths), qo[-1], ko[-1], H, Hk, D, dtype=dtype)
        torch.cuda.synchronize()
        for s in range(0, len(lengths), 13):
            for i in range(lengths[s]):
                a, c = qo[s] + i, ko[s]
                top = context[s] + i + 1
                check(out[a:a + 1], *attend_wide(q[a:a + 1], k[c:c + top], v[c:c + top], dtype))


@TYPES
@GAPS
@pytest.mark.parametrize("lengths,prefix,H,Hk,D", [
    ([6000, 70], 0, 4, 1, 128),
    ([40, 3], 4000, 8, 2, 128),                                  # the prefix beside the sequences
    ([40, 3] * 12, 4000, 8, 2, 64),                              # the prefix by its own kernel
    ([300] * 12, 1500, 8, 2, 128),
])
def test_decode_attention_sink(lengths, prefix, H, Hk, D, gap, spread, dtype):
    b = Batch(lengths, prefix, H, Hk, D, dtype, 16)
    q, pages = b.q.view(b.B, H, D), [(b.prefix_pages[0] if prefix else rows[0]) for rows in b.rows]
    flat_k, flat_v = b.k.permute(0, 2, 1, 3), b.v.permute(0, 2, 1, 3)            # [page][slot][head][channel]
    q *= spread
    q[..., 0] = 8.0
    flat_k[..., 0] = 0.0
    flat_v *= 20.0
    flat_v += 30.0
    for p in set(pages):
        flat_k[p, 5] = 0.0
        flat_k[p, 5, :, 0] = gap * D ** 0.5 / 8
        flat_v[p, 5] = 0.0
    b.call()
    torch.cuda.synchronize()
    for i in range(0, b.B, 7):
        pk, pv = b.keys(b.prefix_pages, prefix)
        k, v = b.keys(b.rows[i], lengths[i])
        check(b.out[i:i + 1], *attend_wide(q[i:i + 1], torch.cat((pk, k)), torch.cat((pv, v)), dtype))


def far_value(q, k, v, at, high, value, D):
    """Key `high` scores 200 nats above the others, whose weights beside it are zero in 32 bits; key `at` has a
    value that is not finite in channel 3."""
    q[..., 0], k[..., 0] = 16.0, 0.0
    k[high][..., 0] = 200 * D ** 0.5 / 16
    v[at][..., 3] = value


@TYPES
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("at,high", [(2, 3), (20, 40), (10, 2900), (2900, 10), (1500, 1400)])
def test_a_value_that_is_not_finite_is_seen_whatever_its_weight(at, high, value, dtype):
    """0 times infinity, as in 32 bits: the same wherever the row's keys are divided -- within a tile, between warps,
    between CTAs and between the prefix and a sequence's own keys."""
    H, Hk, D, m = 4, 2, 128, 3000
    for lengths, context in (([2], [m - 2]), ([2] * 40, [m - 2] * 40)):           # clusters share the keys; one CTA has them all
        qo, ko = offsets(lengths), offsets([n + c for n, c in zip(lengths, context)])
        q, k, v = randn(1, qo[-1], H, D, dtype=dtype), randn(2, ko[-1], Hk, D, dtype=dtype), randn(3, ko[-1], Hk, D, dtype=dtype)
        for s in range(len(lengths)):
            far_value(q[qo[s]:qo[s + 1]], k[ko[s]:ko[s + 1]], v[ko[s]:ko[s + 1]], at, high, value, D)
        out = torch.full_like(q, 11.0)
        sp.attention_prompt(q, k, v, out, i32(qo), i32(ko), len(lengths), qo[-1], ko[-1], H, Hk, D, dtype=dtype)
        torch.cuda.synchronize()
        assert not torch.isfinite(out[..., 3]).any()
        out[..., 3] = 0
        assert torch.isfinite(out).all()
    for B, prefix in ((1, 0), (5, 1000), (20, 1000)):
        b = Batch([m - prefix] * B, prefix, H, Hk, D, dtype, 16)
        for i in range(B):
            (pa, sa), (ph, sh) = [((b.prefix_pages if j < prefix else b.rows[i])[(j if j < prefix else j - prefix) // 16],
                                   (j if j < prefix else j - prefix) % 16) for j in (at, high)]
            if i == 0:
                b.q.view(B, H, D)[..., 0], b.k[..., 0] = 16.0, 0.0
            b.k[ph, :, sh, 0] = 200 * D ** 0.5 / 16
            b.v[pa, :, sa, 3] = value
        b.call()
        torch.cuda.synchronize()
        assert not torch.isfinite(b.out[..., 3]).any(), (B, prefix)
        b.out[..., 3] = 0
        assert torch.isfinite(b.out).all()


@TYPES
def test_rows_whose_scores_are_all_minus_infinity_are_zero(dtype):
    """Wherever the row is computed: by one CTA or several, or by itself because a value behind it is not finite."""
    ninf = float("-inf")
    for H, Hk, D, n, m in ((4, 2, 128, 3, 3000), (4, 4, 64, 2, 1500), (4, 2, 128, 40, 90), (2, 1, 64, 300, 300)):
        q, k, v = torch.zeros((n, H, D)), torch.zeros((m, Hk, D)), randn(3, m, Hk, D, dtype=dtype)
        q[..., 0], k[..., 0] = 1.0, ninf
        q, k = q.to(v), k.to(v)
        for last in (1.0, NAN):
            v[m - 1] = last
            out = torch.full_like(q, 11.0)
            sp.attention_prompt(q, k, v, out, i32([0, n]), i32([0, m]), 1, n, m, H, Hk, D, dtype=dtype)
            torch.cuda.synchronize()
            assert (out[:n - 1] == 0).all()
            assert torch.isnan(out[n - 1]).all() if last != last else (out[n - 1] == 0).all()
    for lengths, prefix, H, Hk, D in (([300], 0, 4, 2, 128), ([3000, 20], 0, 4, 2, 64), ([5, 70], 400, 8, 2, 128), ([5, 70] * 9, 400, 8, 2, 128)):
        b = Batch(lengths, prefix, H, Hk, D, dtype, 16)
        b.q.zero_()
        b.q.view(b.B, H, D)[..., 0] = 1.0
        keep = torch.isnan(b.k)
        b.k.zero_()
        b.k[..., 0] = ninf
        b.k[keep] = NAN
        b.call()
        torch.cuda.synchronize()
        assert (b.out == 0).all()
