"""GPU tests of the attention operators (sptmm_rotate_heads, sptmm_attention_prompt,
sptmm_attention_decode) through the C ABI, against plain float64 forms of the same formulas.

Tolerances.  u = eps / 2 of the 16-bit type (a rounding is off by at most that, relative to the value).
Attention, per output element: with p the exact softmax weights and A = sum p |v|,
  * the output is rounded once:                                      u |o|
  * every weight is rounded to the type before it multiplies v:      u A
  * a score is a sum of D products of 16-bit numbers in fp32, then scaled; with S the largest
    scale * sum |q_i k_i| of the row its error is at most (D + 3) 2^-23 S, and an error d of a score
    changes weight and normaliser by a factor of at most e^d each:   2 (D + 3) 2^-23 S A
  * exp2 is good to 2^-16, in weight and normaliser:                 2 2^-16 A
  * sums over n keys in fp32, products and normaliser:               2 n 2^-23 A
Rotation: fp32 with a handful of roundings of values of the pair's size r = |a| + |b|, then one to
the type: u |y| + 2^-18 r (the mean of at most 128 squares, rsqrt and the weight: below 2^-19 relative;
cosine and sine of an angle good to 2^-22)."""
import numpy as np
import pytest

import oracle_lib as O
import sptmm_b200 as sp

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {sp.F16: torch.float16, sp.BF16: torch.bfloat16, sp.F32: torch.float32}
TYPES = pytest.mark.parametrize("dtype", [sp.F16, sp.BF16], ids=["f16", "bf16"])
NAN = float("nan")


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(seed, *shape, dtype=sp.F16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(DT[dtype])


def attend(q, k, v, dtype, scale, causal):
    """q (n, H, D), k and v (m, Hk, D) -> exact output and the tolerance of every element."""
    n, H, D = q.shape
    m, g = k.shape[0], H // k.shape[1]
    u = torch.finfo(DT[dtype]).eps / 2
    out = torch.zeros((n, H, D), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for i in range(n):
        top = max(0, min(m, i + m - n + 1)) if causal else m
        if top == 0:
            continue
        for h in range(H):
            kk, vv, qq = k[:top, h // g].double(), v[:top, h // g].double(), q[i, h].double()
            s = kk @ qq * scale
            S = (kk.abs() @ qq.abs()).max() * scale
            w = torch.softmax(s, 0)
            o, A = w @ vv, w @ vv.abs()
            out[i, h] = o
            tol[i, h] = u * o.abs() + A * (u + 2 * (D + 3) * 2.0 ** -23 * S + 2.0 ** -15 + 2 * top * 2.0 ** -23)
    return out, tol + 1e-30


def check(got, want, tol):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), "%d of %d outside; worst %.3g of its tolerance, at %s" % (
        int(bad.sum()), bad.numel(), float((err / tol).nan_to_num(1e9).max()), bad.nonzero()[0].tolist())


# ---- rotation --------------------------------------------------------------------------------------

def rotate_exact(x, H, Hk, D, pos, inv, qn, kn, eps, interleaved):
    T, r = x.shape[0], 2 * len(inv)
    x = x.double().reshape(T, H + 2 * Hk, D).clone()
    for lo, hi, w in ((0, H, qn), (H, H + Hk, kn)):
        if w is not None:
            x[:, lo:hi] *= w.double() / (x[:, lo:hi].square().mean(-1, keepdim=True) + eps).sqrt()
    size = x.abs()
    if r:
        t = torch.from_numpy(np.outer(pos.cpu().numpy().astype(np.float64), inv)).cuda()[:, None]
        ia, ib = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
        y = x[:, :H + Hk]
        a, b = y[..., ia].clone(), y[..., ib].clone()
        y[..., ia], y[..., ib] = a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()
        size[:, :H + Hk][..., ia] = size[:, :H + Hk][..., ib] = a.abs() + b.abs()
    return x, size


def run_rotate(T, H, Hk, D, src, dtype, rot, interleaved, norm, packed, page, pos=None, pad=0, seed=0, stream=0, T_slots=None):
    width = (H + 2 * Hk) * D
    x = randn(seed, T, width + pad, dtype=src, scale=1.3)
    pos = pos if pos is not None else i32(list(range(T)))
    inv = np.array([10000.0 ** (-2.0 * i / max(rot, 1)) for i in range(rot // 2)])
    qn = (randn(seed + 1, D, dtype=sp.F32) * 0.3 + 1) if norm else None
    kn = (randn(seed + 2, D, dtype=sp.F32) * 0.3 + 1) if norm else None
    q = torch.full((T, H, D + 0), 7.0, dtype=DT[dtype], device="cuda")
    k = torch.full((T, Hk, D), 7.0, dtype=DT[dtype], device="cuda") if packed else None
    v = torch.full((T, Hk, D), 7.0, dtype=DT[dtype], device="cuda") if packed else None
    cache = slots = kp = vp = None
    if page:
        n_pages = (T + page - 1) // page + 2
        perm = np.random.default_rng(seed).permutation(n_pages * page)[:T]
        slot_list = perm.tolist()
        if T > 2:
            slot_list[1] = -1
            slot_list[2] = n_pages * page                       # past the cache
        slots = i32(slot_list)
        kp = torch.full((n_pages, Hk, page, D), 3.0, dtype=DT[dtype], device="cuda")
        vp = torch.full_like(kp, 5.0)
        cache = sp.KVCache(kp, vp, n_pages, page, Hk, D, dtype)
    sp.rotate_heads(x, T, H, Hk, D, pos, inv if rot else None, q, in_dtype=src, dtype=dtype, q_norm=qn, k_norm=kn, eps=1e-5,
                    interleaved=interleaved, K=k, V=v, cache=cache, slots=slots, ldqkv=width + pad if pad else 0, stream=stream)
    torch.cuda.synchronize()
    want, size = rotate_exact(x[:, :width], H, Hk, D, pos, inv if rot else inv[:0], qn, kn, 1e-5, interleaved)
    tol = torch.finfo(DT[dtype]).eps / 2 * want.abs() + 2.0 ** -18 * size + (2.0 ** -25 if dtype == sp.F16 else 0)   # fp16 subnormals: half of 2^-24
    check(q, want[:, :H], tol[:, :H])
    if packed:
        check(k, want[:, H:H + Hk], tol[:, H:H + Hk])
        check(v, want[:, H + Hk:], tol[:, H + Hk:])
    if page:
        for pages, part, fill in ((kp, slice(H, H + Hk), 3.0), (vp, slice(H + Hk, H + 2 * Hk), 5.0)):
            flat = pages.permute(0, 2, 1, 3).reshape(n_pages * page, Hk, D)
            keep = [i for i, s in enumerate(slot_list) if 0 <= s < n_pages * page]
            at = [slot_list[i] for i in keep]
            check(flat[at], want[keep][:, part], tol[keep][:, part])
            rest = torch.ones(n_pages * page, dtype=torch.bool, device="cuda")
            rest[at] = False
            assert (flat[rest] == fill).all()                    # nothing else was touched
    return q


@TYPES
@pytest.mark.parametrize("T,H,Hk,D,src,rot,interleaved,norm,packed,page", [
    (1, 20, 5, 128, sp.F32, 128, False, True, False, 16),
    (37, 20, 5, 128, sp.F32, 128, False, True, True, 32),
    (5, 16, 16, 64, sp.F16, 32, True, False, True, 0),
    (9, 3, 3, 64, sp.BF16, 64, False, True, True, 64),
    (7, 4, 1, 72, sp.F32, 24, False, True, False, 128),
    (6, 12, 4, 80, sp.F16, 80, True, True, True, 16),
    (3, 2, 1, 8, sp.F32, 8, False, True, True, 16),
    (3, 1, 1, 16, sp.F32, 8, True, False, True, 0),
    (4, 7, 7, 120, sp.F32, 112, False, True, True, 0),
    (2, 100, 10, 128, sp.F32, 64, False, True, True, 0),
    (5, 6, 2, 96, sp.BF16, 0, False, True, True, 0),
    (5, 6, 2, 96, sp.F32, 0, False, False, True, 0),
])
def test_rotate(T, H, Hk, D, src, rot, interleaved, norm, packed, page, dtype):
    run_rotate(T, H, Hk, D, src, dtype, rot, interleaved, norm, packed, page)


def test_rotate_far_and_negative_positions():
    pos = i32([0, 1, 131071, 1048575, 16777217, 2147483647, -5])
    run_rotate(7, 4, 2, 128, sp.F32, sp.F16, 128, False, False, True, 0, pos=pos)


@pytest.mark.parametrize("src", [sp.F32, sp.F16])
def test_rotate_row_strides(src):
    run_rotate(11, 4, 2, 64, src, sp.F16, 64, False, True, True, 16, pad=24)
    # outputs as column ranges of one wider row; what lies between stays
    T, H, Hk, D = 6, 4, 2, 64
    x = randn(3, T, (H + 2 * Hk) * D, dtype=src)
    wide = torch.full((T, 1024), 9.0, dtype=torch.float16, device="cuda")
    tight = [torch.zeros((T, n * D), dtype=torch.float16, device="cuda") for n in (H, Hk, Hk)]
    inv = np.array([0.5 ** i for i in range(32)])
    pos = i32([3, 1, 4, 1, 5, 9])
    sp.rotate_heads(x, T, H, Hk, D, pos, inv, tight[0], in_dtype=src, K=tight[1], V=tight[2])
    sp.rotate_heads(x, T, H, Hk, D, pos, inv, wide, in_dtype=src, K=wide[:, 264:], V=wide[:, 400:], ldq=1024, ldk=1024, ldv=1024)
    torch.cuda.synchronize()
    for lo, t in ((0, tight[0]), (264, tight[1]), (400, tight[2])):
        assert torch.equal(wide[:, lo:lo + t.shape[1]], t)
    assert (wide[:, 256:264] == 9).all() and (wide[:, 392:400] == 9).all() and (wide[:, 528:] == 9).all()


def test_rotate_many_tokens():
    run_rotate(4099, 20, 5, 128, sp.F32, sp.BF16, 128, False, True, True, 64, seed=4)


# ---- prompts ----------------------------------------------------------------------------------------

def offsets(lengths, start=0):
    return (np.concatenate([[0], np.cumsum(lengths)]) + start).tolist()


def run_prompt(lengths, context, H, Hk, D, dtype, causal=True, scale=0.0, extra=3, seed=0, fused=False, stream=0, flags=0, poison=True):
    qo = offsets(lengths)
    ko = offsets([n + c for n, c in zip(lengths, context)] if context else lengths)
    T, Tk = qo[-1] + extra, ko[-1] + extra
    if fused:                                                    # column ranges of one fused row (self attention only)
        row = randn(seed, T, (H + 2 * Hk) * D, dtype=dtype, scale=1.2)
        q, k, v = row[:, :H * D], row[:, H * D:(H + Hk) * D], row[:, (H + Hk) * D:]
        ld = dict(ldq=row.shape[1], ldk=row.shape[1], ldv=row.shape[1])
    else:
        q, k, v = randn(seed, T, H * D, dtype=dtype, scale=1.5), randn(seed + 1, Tk, Hk * D, dtype=dtype), randn(seed + 2, Tk, Hk * D, dtype=dtype)
        ld = {}
    if poison and extra:                                         # rows behind the last sequence are not looked at
        q[qo[-1]:], k[ko[-1]:], v[ko[-1]:] = NAN, NAN, NAN
    out = torch.full((T, H * D), 11.0, dtype=DT[dtype], device="cuda")
    sp.attention_prompt(q, k, v, out, i32(qo), i32(ko), len(lengths), T, Tk, H, Hk, D, dtype=dtype, causal=causal, scale=scale,
                        stream=stream, flags=flags, **ld)
    torch.cuda.synchronize()
    for a, b, c, e in zip(qo, qo[1:], ko, ko[1:]):
        if b > a:
            want, tol = attend(q[a:b].reshape(b - a, H, D), k[c:e].reshape(e - c, Hk, D), v[c:e].reshape(e - c, Hk, D), dtype,
                               scale or D ** -0.5, causal)
            check(out[a:b].reshape(b - a, H, D), want, tol)
    assert (out[qo[-1]:] == 11).all()                            # left as they were
    return out


@TYPES
@pytest.mark.parametrize("lengths,context,H,Hk,D", [
    ([1], [], 1, 1, 128),
    ([0, 5, 0, 1, 33, 0], [], 4, 1, 128),
    ([31, 32, 33, 64, 65], [], 4, 1, 128),
    ([127, 128, 129], [], 2, 2, 64),
    ([200], [], 20, 5, 128),
    ([150], [], 7, 1, 128),
    ([70, 3], [], 12, 4, 80),
    ([90], [], 3, 1, 8),
    ([40], [], 2, 1, 72),
    ([65, 2], [], 32, 2, 64),
    ([20], [], 40, 1, 128),
    ([5, 9], [], 128, 1, 64),
    ([3], [], 100, 1, 128),
    ([4, 70, 1], [300, 1, 127], 4, 2, 128),
    ([1, 1, 1], [0, 128, 511], 8, 1, 64),
    ([300], [], 2, 1, 128),
])
def test_prompt(lengths, context, H, Hk, D, dtype):
    run_prompt(lengths, context, H, Hk, D, dtype)


@TYPES
@pytest.mark.parametrize("lengths,context", [([130, 1, 64], []), ([7, 0, 200], [250, 9, 0]), ([12], [700])])
def test_prompt_not_causal(lengths, context, dtype):
    run_prompt(lengths, context, 4, 2, 128, dtype, causal=False)


@TYPES
def test_prompt_more_queries_than_keys(dtype):
    """Queries before the first key see nothing: zeros.  Sequences without keys: all zeros."""
    run_prompt([10, 140, 6], [-3, -60, -6], 4, 2, 64, dtype)
    run_prompt([10, 140, 6], [-3, -60, -6], 4, 2, 128, dtype, causal=False)
    out = run_prompt([5, 300], [-5, -300], 2, 1, 128, dtype)
    assert (out[:305] == 0).all()


@TYPES
def test_prompt_fused_rows_and_scale(dtype):
    run_prompt([77, 130], [], 8, 2, 64, dtype, fused=True, scale=0.3)
    run_prompt([150], [], 4, 4, 128, dtype, fused=True, scale=0.02)


@TYPES
def test_prompt_large_and_equal_scores(dtype):
    """Scores far above and below one another, running maxima that keep rising, constant rows."""
    T, H, Hk, D = 300, 4, 2, 128
    for kind in range(3):
        q, k, v = randn(1, T, H, D, dtype=dtype), randn(2, T, Hk, D, dtype=dtype), randn(3, T, Hk, D, dtype=dtype)
        if kind == 0:                                            # key j has score ~ j / 4 for every query
            q[:], k[:] = 1.0, 0.0
            k[..., 0] = (torch.arange(T, device="cuda", dtype=torch.float32) * 2.75).to(DT[dtype])[:, None]
        elif kind == 1:                                          # falling
            q[:], k[:] = 1.0, 0.0
            k[..., 0] = (-torch.arange(T, device="cuda", dtype=torch.float32) * 2.75).to(DT[dtype])[:, None]
        else:
            q[:] = 0.0
        out = torch.zeros_like(q)
        sp.attention_prompt(q, k, v, out, i32([0, T]), i32([0, T]), 1, T, T, H, Hk, D, dtype=dtype)
        torch.cuda.synchronize()
        check(out, *attend(q, k, v, dtype, D ** -0.5, True))


@TYPES
def test_prompt_hidden_values_do_not_count(dtype):
    """NaN and infinity in another sequence's keys and values, and in a sequence's later ones, do not
    reach the rows that do not see them; the rows that do see them are not finite."""
    H, Hk, D = 4, 2, 128
    lengths = [50, 70, 140]
    off = offsets(lengths)
    T = off[-1]
    base = [randn(s, T, n, D, dtype=dtype) for s, n in ((1, H), (2, Hk), (3, Hk))]
    off_d = i32(off)

    def go(q, k, v):
        out = torch.zeros((T, H, D), dtype=DT[dtype], device="cuda")
        sp.attention_prompt(q, k, v, out, off_d, off_d, 3, T, T, H, Hk, D, dtype=dtype)
        torch.cuda.synchronize()
        return out

    clean = go(*base)
    for value in (NAN, float("inf")):
        k, v = base[1].clone(), base[2].clone()
        k[off[1]:off[2]] = value
        v[off[1]:off[2]] = value
        out = go(base[0], k, v)
        assert torch.equal(out[:off[1]], clean[:off[1]]) and torch.equal(out[off[2]:], clean[off[2]:])
        assert not torch.isfinite(out[off[1]:off[2]]).any()
        at = off[2] + 100                                        # row 100 of the last sequence
        v = base[2].clone()
        v[at, 0, 5] = value
        out = go(base[0], base[1], v)
        want = clean.clone()
        seen = out[at:, :2, 5].clone()
        out[at:, :2, 5] = want[at:, :2, 5] = 0
        assert not torch.isfinite(seen).any()
        g, tol = attend(base[0][off[2]:], base[1][off[2]:], base[2][off[2]:], dtype, D ** -0.5, True)
        g[100:, :2, 5] = 0
        check(out[off[2]:], g, tol)
        assert torch.equal(out[:off[2]], clean[:off[2]])
        k = base[1].clone()
        k[at, 1, 3] = NAN
        out = go(base[0], k, base[2])
        assert torch.equal(out[:at], clean[:at]) and torch.equal(out[at:, :2], clean[at:, :2])
        assert torch.isnan(out[at:, 2:]).all()


def test_prompt_offsets_outside_the_buffers_are_cut():
    H, Hk, D, T = 2, 1, 64, 40
    q, k, v = randn(1, T, H, D), randn(2, T, Hk, D), randn(3, T, Hk, D)
    out = torch.full((T, H, D), 11.0, dtype=torch.float16, device="cuda")
    sp.attention_prompt(q, k, v, out, i32([0, 30, 1 << 20]), i32([-7, 30, 2147483647]), 2, T, T, H, Hk, D)
    torch.cuda.synchronize()
    check(out[:30], *attend(q[:30], k[:30], v[:30], sp.F16, D ** -0.5, True))
    check(out[30:], *attend(q[30:], k[30:], v[30:], sp.F16, D ** -0.5, True))


def test_prompt_many_sequences():
    rng = np.random.default_rng(0)
    lengths = rng.integers(0, 4, size=700).tolist()
    run_prompt(lengths, [], 2, 1, 64, sp.F16)
    run_prompt(lengths[:300], rng.integers(0, 9, size=300).tolist(), 2, 1, 64, sp.F16)


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_many_sequences_of_many_tiles(causal):
    """More sequences than a warp has lanes, of zero to seven tiles, some with context: every row is written, and
    the first and last sequences, the longest and one with context are right."""
    rng = np.random.default_rng(7)
    lengths = rng.integers(0, 600, size=75).tolist()
    lengths[3], lengths[40], lengths[74] = 0, 700, 130
    context = [int(c) for c in rng.integers(0, 900, size=75) * (rng.random(75) < 0.3)]
    context[74] = 300
    H, Hk, D = 3, 3, 64
    qo, ko = offsets(lengths), offsets([n + c for n, c in zip(lengths, context)])
    q, k, v = randn(1, qo[-1], H, D, scale=1.5), randn(2, ko[-1], Hk, D), randn(3, ko[-1], Hk, D)
    out = torch.full_like(q, 11.0)
    sp.attention_prompt(q, k, v, out, i32(qo), i32(ko), 75, qo[-1], ko[-1], H, Hk, D, causal=causal)
    torch.cuda.synchronize()
    assert (out != 11).any(-1).all()
    for s in (0, 31, 32, 40, 74):
        rows = sorted({0, lengths[s] // 3, lengths[s] - 1}) if lengths[s] else []
        for i in rows:
            m = lengths[s] + context[s]
            top = context[s] + i + 1 if causal else m
            a, c = qo[s] + i, ko[s]
            check(out[a:a + 1], *attend(q[a:a + 1], k[c:c + top], v[c:c + top], sp.F16, D ** -0.5, False))


def test_prompt_side_stream_repeat_and_graph():
    """Same bits on another stream, from call to call and from a graph; a replay follows new offsets."""
    H, Hk, D, dtype = 8, 2, 128, sp.BF16
    T = 500
    q, k, v = randn(1, T, H, D, dtype=dtype), randn(2, T, Hk, D, dtype=dtype), randn(3, T, Hk, D, dtype=dtype)
    first, second = [0, 100, 500, 500], [0, 333, 334, 490]
    off = i32(first)
    out = torch.zeros((T, H, D), dtype=DT[dtype], device="cuda")

    def call(stream=0, flags=0):
        sp.attention_prompt(q, k, v, out, off, off, 3, T, T, H, Hk, D, dtype=dtype, stream=stream, flags=flags)

    call()
    torch.cuda.synchronize()
    want = out.clone()
    side = torch.cuda.Stream()
    for flags in (0, sp.LAUNCH_PDL):
        out.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            call(side.cuda_stream, flags)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(torch.cuda.current_stream().cuda_stream)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    off.copy_(i32(second))
    out.fill_(11.0)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(second, second[1:]):
        check(out[a:b], *attend(q[a:b], k[a:b], v[a:b], dtype, D ** -0.5, True))
    assert (out[490:] == 11).all()


# ---- decode -----------------------------------------------------------------------------------------

class Batch:
    def __init__(self, lengths, prefix, H, Hk, D, dtype, page, seed=0, max_pages=None, joint=False, ldq=0):
        rng = np.random.default_rng(seed)
        self.lengths, self.prefix, self.H, self.Hk, self.D, self.dtype, self.page = lengths, prefix, H, Hk, D, dtype, page
        self.B = len(lengths)
        need = [(n + page - 1) // page for n in lengths]
        self.max_pages = max_pages if max_pages is not None else max(need + [1])
        n_prefix = (prefix + page - 1) // page
        self.n_pages = sum(need) + n_prefix + 2
        order = rng.permutation(self.n_pages).tolist()
        self.prefix_pages, order = order[:n_prefix], order[n_prefix:]
        table, self.rows = np.full((self.B, max(self.max_pages, 1)), -1), []
        for b, n in enumerate(need):
            self.rows.append(order[:n])
            table[b, :n], order = order[:n], order[n:]
        self.table = i32(table.tolist())
        self.prefix_table = i32(self.prefix_pages) if prefix else None
        if joint:                                                # k and v of a page side by side in one buffer
            both = randn(seed, self.n_pages, 2, Hk, page, D, dtype=dtype)
            self.k, self.v, stride = both[:, 0], both[:, 1], 2 * Hk * page * D
        else:
            self.k, self.v, stride = randn(seed + 1, self.n_pages, Hk, page, D, dtype=dtype), randn(seed + 2, self.n_pages, Hk, page, D, dtype=dtype), 0
        used = torch.zeros((self.n_pages, page), dtype=torch.bool, device="cuda")
        for pages, n in zip(self.rows + [self.prefix_pages], list(lengths) + [prefix]):
            for i, pg in enumerate(pages):
                used[pg, :max(0, min(page, n - i * page))] = True
        for t in (self.k, self.v):                               # slots nobody owns hold NaN
            t.permute(0, 2, 1, 3)[~used] = NAN
        self.cache = sp.KVCache(self.k, self.v, self.n_pages, page, Hk, D, dtype, stride)
        self.q = randn(seed + 3, self.B, max(ldq, H * D), dtype=dtype, scale=1.5)
        self.ldq = ldq
        self.workspace = torch.full((sp.attention_decode_workspace(self.B, H, Hk, D, prefix),), 255, dtype=torch.uint8, device="cuda")
        self.out = torch.full((self.B, H, D), 11.0, dtype=DT[dtype], device="cuda")
        self.len = i32(lengths)
        self.scale = 0.0

    def call(self, stream=0, flags=0):
        sp.attention_decode(self.q, self.out, self.B, self.H, self.cache, self.len, self.table, self.max_pages,
                            prefix_table=self.prefix_table, prefix_len=self.prefix, workspace=self.workspace,
                            workspace_bytes=self.workspace.numel(), scale=self.scale, ldq=self.ldq, stream=stream, flags=flags)

    def keys(self, pages, n, drop=()):
        out = []
        for t in (self.k, self.v):
            rows = [t[pg].transpose(0, 1)[:max(0, min(self.page, n - i * self.page))] for i, pg in enumerate(pages) if pg not in drop]
            out.append(torch.cat(rows) if rows else t.new_zeros((0, self.Hk, self.D)))
        return out

    def want(self, b, drop=()):
        pk, pv = self.keys(self.prefix_pages, self.prefix, drop)
        k, v = self.keys(self.rows[b], self.lengths[b], drop)
        q = self.q[b, :self.H * self.D].view(1, self.H, self.D)
        return attend(q, torch.cat((pk, k)), torch.cat((pv, v)), self.dtype, self.scale or self.D ** -0.5, False)

    def verify(self, drop=()):
        torch.cuda.synchronize()
        for b in range(self.B):
            want, tol = self.want(b, drop)
            check(self.out[b:b + 1], want, tol)


@TYPES
@pytest.mark.parametrize("lengths,prefix,H,Hk,D,page", [
    ([1], 0, 4, 1, 128, 16),
    ([0, 1, 2, 15, 16, 17], 0, 4, 2, 128, 16),
    ([300], 0, 20, 5, 128, 16),
    ([5000, 3, 0, 700], 0, 4, 1, 128, 32),
    ([63, 64, 65, 129], 0, 16, 16, 64, 64),
    ([127, 128, 129, 1000], 0, 7, 1, 80, 128),
    ([33, 100], 0, 2, 1, 8, 16),
    ([40], 0, 3, 3, 72, 16),
    ([90, 200], 0, 20, 1, 128, 16),
    ([90, 200], 0, 128, 1, 64, 32),
    ([50] * 40, 0, 8, 2, 128, 16),
    ([0], 1, 4, 1, 128, 16),
    ([10, 0, 37], 300, 20, 5, 128, 16),
    ([3, 130], 128, 4, 2, 128, 64),
    ([5, 70, 0], 1000, 16, 16, 64, 32),
    ([9], 2000, 7, 1, 80, 128),
    ([1, 2], 129, 40, 1, 128, 16),
    ([4, 8], 513, 100, 1, 96, 16),
    ([20] * 70, 260, 8, 2, 128, 16),
    ([0, 0], 77, 8, 8, 72, 32),
])
def test_decode(lengths, prefix, H, Hk, D, page, dtype):
    b = Batch(lengths, prefix, H, Hk, D, dtype, page)
    b.call()
    b.verify()


@TYPES
@pytest.mark.parametrize("B,own,prefix,H,Hk,D,page", [
    (1, [5], 1000, 16, 1, 128, 16),                              # one tile of 16 rows
    (17, [0, 20, 70], 130, 1, 1, 64, 32),                        # seventeen rows: two tiles
    (8, [33], 700, 8, 2, 128, 64),                               # 32 rows
    (33, [0, 1, 40], 300, 2, 2, 64, 32),                         # more rows: the prefix's own kernel
    (16, [33], 700, 8, 2, 128, 64),
    (33, [7, 0], 129, 4, 2, 64, 64),
    (70, [3], 1, 4, 4, 8, 128),
    (20, [100, 2], 4000, 28, 4, 128, 16),
    (40, [1, 30], 900, 6, 2, 72, 128),
    (5, [64], 640, 64, 2, 128, 64),
])
def test_decode_prefix_for_few_and_many_rows(B, own, prefix, H, Hk, D, page, dtype):
    b = Batch([own[i % len(own)] for i in range(B)], prefix, H, Hk, D, dtype, page)
    b.call()
    b.verify()
    if prefix > 2 * page:                                        # pages outside the cache, in the middle and at the end
        drop = [b.prefix_pages[1], b.prefix_pages[-1]]
        t = b.prefix_table.cpu()
        t[1], t[-1] = -1, b.n_pages
        b.prefix_table = t.cuda()
        b.call()
        b.verify(drop)


@TYPES
def test_decode_joint_pages_query_stride_and_scale(dtype):
    b = Batch([100, 17, 260], 90, 8, 2, 128, dtype, 32, joint=True, ldq=8 * 128 + 64)
    b.scale = 0.21
    b.call()
    b.verify()


@TYPES
@pytest.mark.parametrize("prefix", [0, 150])
def test_decode_nothing_to_see_is_zero(prefix, dtype):
    b = Batch([0, 0, 5], prefix, 4, 2, 128, dtype, 16)
    b.len = i32([0, -3, 5])
    b.call()
    b.verify()
    if not prefix:
        assert (b.out[:2] == 0).all()
        c = Batch([0, 0], 0, 4, 2, 128, dtype, 16, max_pages=0)
        c.len = i32([9, 1])                                      # no pages at all: cut to nothing
        c.call()
        torch.cuda.synchronize()
        assert (c.out == 0).all()


@TYPES
def test_decode_pages_outside_the_cache_are_left_out(dtype):
    b = Batch([100, 64, 33], 80, 4, 2, 128, dtype, 16)
    b.call()
    b.verify()
    drop = [b.rows[0][2], b.rows[1][0], b.rows[1][1], b.rows[1][2], b.rows[1][3], b.prefix_pages[1]]
    t, pt = b.table.cpu(), b.prefix_table.cpu()
    t[0, 2], t[1, 0], t[1, 1], t[1, 2], t[1, 3] = -1, b.n_pages, 2 ** 31 - 1, -2 ** 31, b.n_pages + 5
    pt[1] = -7
    b.table, b.prefix_table = t.cuda(), pt.cuda()
    b.call()
    b.verify(drop)


def test_decode_lengths_are_cut_to_the_table():
    b = Batch([64, 32], 0, 4, 2, 128, sp.F16, 16)
    b.len = i32([2 ** 31 - 1, 32])
    b.call()
    b.verify()


@TYPES
def test_decode_one_page_for_many_sequences(dtype):
    """The same page in several rows of the table, and twice in one row."""
    b = Batch([48, 48, 48], 0, 4, 2, 64, dtype, 16)
    r = b.rows[0]
    b.rows = [[r[0], r[1], r[2]], [r[0], r[1], r[1]], [r[2], r[0], r[1]]]
    b.table = i32(b.rows)
    b.call()
    b.verify()


@TYPES
def test_decode_rising_scores_across_splits(dtype):
    for sign in (1.0, -1.0):
        b = Batch([3000, 40], 600, 4, 1, 128, dtype, 16)
        b.q[:] = 1.0
        for pages, n, start in ((b.prefix_pages, 600, 0), (b.rows[0], 3000, 600), (b.rows[1], 40, 600)):
            for i, pg in enumerate(pages):
                m = max(0, min(16, n - 16 * i))
                b.k[pg, :, :m] = 0
                b.k[pg, :, :m, 0] = (sign * 0.5 * (start + 16 * i + torch.arange(m, device="cuda"))).to(DT[dtype])
        b.call()
        b.verify()


def test_decode_repeat_side_stream_and_graph():
    for prefix in (0, 300):
        b = Batch([700, 20, 333, 1], prefix, 8, 2, 128, sp.BF16, 16)
        b.call()
        b.verify()
        want = b.out.clone()
        side = torch.cuda.Stream()
        for flags in (0, sp.LAUNCH_PDL):
            b.out.zero_()
            torch.cuda.synchronize()
            for _ in range(4):
                b.call(side.cuda_stream, flags)
            torch.cuda.synchronize()
            assert torch.equal(b.out, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            b.call(torch.cuda.current_stream().cuda_stream)
        b.out.zero_()
        b.workspace.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b.out, want)
        b.lengths = [100, 20, 0, 1]
        b.len.copy_(i32(b.lengths))
        graph.replay()
        b.verify()


def test_decode_cache_beyond_32_bit_offsets():
    """Element offsets above 2^32 and 2^33 bytes: a few pages very far apart."""
    Hk, D, page, stride, n_pages = 2, 128, 16, 1 << 27, 35
    buf = torch.empty(stride * (n_pages - 1) + 2 * Hk * page * D, dtype=torch.float16, device="cuda")     # 9.1 GB
    each = Hk * page * D
    pages, q = [0, 33, 31, 34], randn(3, 1, 4, D)
    kk, vv = randn(1, 4, Hk, page, D), randn(2, 4, Hk, page, D)
    for i, pg in enumerate(pages):
        buf[pg * stride:pg * stride + each] = kk[i].flatten()
        buf[pg * stride + each:pg * stride + 2 * each] = vv[i].flatten()
    cache = sp.KVCache(buf, buf.data_ptr() + 2 * each, n_pages, page, Hk, D, sp.F16, stride)
    k, v = kk.transpose(1, 2).reshape(64, Hk, D), vv.transpose(1, 2).reshape(64, Hk, D)
    want, tol = attend(q, k[:60], v[:60], sp.F16, D ** -0.5, False)
    table = i32([pages])
    for prefix, own in ((0, 60), (32, 28), (60, 0)):
        out = torch.zeros((1, 4, D), dtype=torch.float16, device="cuda")
        ws = torch.empty(sp.attention_decode_workspace(1, 4, Hk, D, prefix), dtype=torch.uint8, device="cuda")
        sp.attention_decode(q, out, 1, 4, cache, i32([own]), table[:, prefix // 16:].contiguous() if own else table, 4 - prefix // 16,
                            prefix_table=table if prefix else None, prefix_len=prefix, workspace=ws, workspace_bytes=ws.numel())
        torch.cuda.synchronize()
        check(out, want, tol)
    # the rotation's stores reach the far pages too
    x = randn(5, 2, (4 + 2 * Hk) * D, dtype=sp.F32)
    qq = torch.zeros((2, 4, D), dtype=torch.float16, device="cuda")
    sp.rotate_heads(x, 2, 4, Hk, D, None, None, qq, cache=cache, slots=i32([33 * page + 5, 34 * page + 15]))
    torch.cuda.synchronize()
    for t, (pg, s) in enumerate(((33, 5), (34, 15))):
        for h in range(Hk):
            at = pg * stride + (h * page + s) * D
            assert torch.equal(buf[at:at + D], x[t, (4 + h) * D:(5 + h) * D].half())
            assert torch.equal(buf[at + each:at + each + D], x[t, (4 + Hk + h) * D:(5 + Hk + h) * D].half())
    del buf, cache
    torch.cuda.empty_cache()


# ---- the operators together -------------------------------------------------------------------------

def test_attention_between_the_ternary_products_of_a_layer():
    """qkv product -> rotation into packed rows and cache -> prompt attention -> o product; then decode
    steps over that cache give what the prompt gives when it holds the new token too."""
    H, Hk, D, hidden, page = 4, 1, 64, 256, 16
    N = (H + 2 * Hk) * D
    wqkv = sp.Weights(sp.gen_ternary_iid(hidden, N, 0.5, 1)).upload()
    wo = sp.Weights(sp.gen_ternary_iid(H * D, hidden, 0.5, 2)).upload()
    lengths, steps = [19, 40], 3
    total = [n + steps for n in lengths]
    inv = np.array([10000.0 ** (-2.0 * i / D) for i in range(D // 2)])
    qn, kn = randn(8, D, dtype=sp.F32) * 0.1 + 1, randn(9, D, dtype=sp.F32) * 0.1 + 1
    x = [randn(20 + s, n, hidden) for s, n in enumerate(total)]           # every sequence with its later tokens
    n_pages = 10
    kp = torch.full((n_pages, Hk, page, D), NAN, dtype=torch.float16, device="cuda")
    vp = torch.full_like(kp, NAN)
    cache = sp.KVCache(kp, vp, n_pages, page, Hk, D, sp.F16)
    table = [[7, 2, 5], [1, 9, 0]]
    slot = lambda s, i: table[s][i // page] * page + i % page

    def layer(rows, pos, slots, attention):
        T = rows.shape[0]
        qkv = torch.zeros((T, N), dtype=torch.float32, device="cuda")
        wqkv.gemv(rows.contiguous(), T, qkv, sp.F16)
        q = torch.zeros((T, H * D), dtype=torch.float16, device="cuda")
        k, v = torch.zeros((T, Hk * D), dtype=torch.float16, device="cuda"), torch.zeros((T, Hk * D), dtype=torch.float16, device="cuda")
        with_cache = dict(cache=cache, slots=i32(slots)) if slots else {}
        sp.rotate_heads(qkv, T, H, Hk, D, i32(pos), inv, q, q_norm=qn, k_norm=kn, K=k, V=v, **with_cache)
        att = torch.zeros((T, H * D), dtype=torch.float16, device="cuda")
        attention(q, k, v, att)
        out = torch.zeros((T, hidden), dtype=torch.float32, device="cuda")
        wo.gemv(att, T, out, sp.F16)
        torch.cuda.synchronize()
        return qkv, q, k, v, att, out

    def prompt(lens):
        off = i32(offsets(lens))
        T = sum(lens)
        return lambda q, k, v, att: sp.attention_prompt(q, k, v, att, off, off, len(lens), T, T, H, Hk, D)

    rows = torch.cat([x[s][:n] for s, n in enumerate(lengths)])
    pos = [i for n in lengths for i in range(n)]
    slots = [slot(s, i) for s, n in enumerate(lengths) for i in range(n)]
    qkv, q, k, v, att, out = layer(rows, pos, slots, prompt(lengths))
    W = sp.gen_ternary_iid(hidden, N, 0.5, 1)
    plain = rows.double() @ torch.from_numpy(W).cuda().double().T
    assert (qkv.double() - plain).abs().max() < 1e-3
    a = 0
    for n in lengths:
        check(att[a:a + n].view(n, H, D), *attend(q[a:a + n].view(n, H, D), k[a:a + n].view(n, Hk, D), v[a:a + n].view(n, Hk, D), sp.F16, D ** -0.5, True))
        a += n
    Wo = sp.gen_ternary_iid(H * D, hidden, 0.5, 2)
    assert (out.double() - att.double() @ torch.from_numpy(Wo).cuda().double().T).abs().max() < 1e-3

    ws = torch.empty(sp.attention_decode_workspace(2, H, Hk, D), dtype=torch.uint8, device="cuda")
    for step in range(steps):
        lens = [n + step + 1 for n in lengths]
        decode = lambda q, k, v, att: sp.attention_decode(q, att, 2, H, cache, i32(lens), i32(table), 3, workspace=ws, workspace_bytes=ws.numel())
        new = torch.stack([x[s][lens[s] - 1] for s in range(2)])
        got = layer(new, [n - 1 for n in lens], [slot(s, lens[s] - 1) for s in range(2)], decode)
        whole = layer(torch.cat([x[s][:n] for s, n in enumerate(lens)]), [i for n in lens for i in range(n)], None, prompt(lens))
        last = [lens[0] - 1, lens[0] + lens[1] - 1]
        q, k, v = whole[1], whole[2], whole[3]
        for s in range(2):
            a = 0 if s == 0 else lens[0]
            want, tol = attend(q[last[s]].view(1, H, D), k[a:a + lens[s]].view(-1, Hk, D), v[a:a + lens[s]].view(-1, Hk, D), sp.F16, D ** -0.5, False)
            check(got[4][s].view(1, H, D), want, tol)
            check(whole[4][last[s]].view(1, H, D), want, tol)


def test_programmatic_launches_in_a_row():
    """rotate -> decode behind a prefix, and rotate -> prompt, with SPTMM_LAUNCH_PDL on one stream: every call
    reads what the one before it wrote, over and over into the same buffers."""
    H, Hk, D, page, B, dtype = 8, 2, 128, 16, 6, sp.F16
    lengths, prefix = [5, 40, 1, 300, 17, 64], 270
    side = torch.cuda.Stream()

    def program(flags, rounds):
        b = Batch(lengths, prefix, H, Hk, D, dtype, page, seed=5)
        new = [b.rows[i][(n - 1) // page] * page + (n - 1) % page for i, n in enumerate(lengths)]       # the slot of every sequence's last key
        slots, pos = i32(new), i32([n + prefix - 1 for n in lengths])
        inv = np.array([10000.0 ** (-i / 64) for i in range(64)])
        off, pq = i32([0, 2, 6]), torch.zeros((B, H * D), dtype=torch.float16, device="cuda")
        pk, pv, po = (torch.zeros((B, n * D), dtype=torch.float16, device="cuda") for n in (Hk, Hk, H))
        outs = []
        xs = [randn(50 + r, B, (H + 2 * Hk) * D, dtype=sp.F32) for r in range(rounds)]
        keep = [(torch.zeros_like(b.out), torch.zeros_like(po)) for _ in range(rounds)]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for r in range(rounds):
                s = side.cuda_stream
                sp.rotate_heads(xs[r], B, H, Hk, D, pos, inv, b.q, dtype=dtype, K=pk, V=pv, cache=b.cache, slots=slots, flags=flags, stream=s)
                b.call(s, flags)
                keep[r][0].copy_(b.out)
                sp.rotate_heads(xs[r], B, H, Hk, D, pos, inv, pq, dtype=dtype, K=pk, V=pv, flags=flags, stream=s)
                sp.attention_prompt(pq, pk, pv, po, off, off, 2, B, B, H, Hk, D, dtype=dtype, flags=flags, stream=s)
                keep[r][1].copy_(po)
        torch.cuda.synchronize()
        return keep

    plain, pdl = program(0, 12), program(sp.LAUNCH_PDL, 12)
    for a, b in zip(plain, pdl):
        assert torch.isfinite(a[0]).all() and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert not torch.equal(plain[0][0], plain[1][0])


def test_two_streams_at_once():
    """Calls on two streams, each with a workspace of its own, do not disturb one another."""
    jobs = [Batch([900, 3, 50], 500, 8, 2, 128, sp.F16, 16, seed=1), Batch([20, 1200, 7, 64], 0, 8, 2, 128, sp.F16, 32, seed=2)]
    want = []
    for j in jobs:
        j.call()
        torch.cuda.synchronize()
        want.append(j.out.clone())
        j.verify()
    T = 700
    q, k, v = randn(1, T, 8, 128), randn(2, T, 2, 128), randn(3, T, 2, 128)
    o, off = torch.zeros_like(q), i32([0, 300, 700])
    prompt = lambda stream: sp.attention_prompt(q, k, v, o, off, off, 2, T, T, 8, 2, 128, stream=stream)
    prompt(0)
    torch.cuda.synchronize()
    first = o.clone()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for s, j in zip(streams, jobs):
            j.call(s.cuda_stream)
        prompt(streams[2].cuda_stream)
    torch.cuda.synchronize()
    for j, w in zip(jobs, want):
        assert torch.equal(j.out, w)
    assert torch.equal(o, first)


def test_decode_many_sequences():
    rng = np.random.default_rng(1)
    lengths = rng.integers(0, 40, size=1500).tolist()
    for prefix in (0, 64):
        b = Batch(lengths, prefix, 2, 1, 64, sp.F16, 16)
        b.call()
        torch.cuda.synchronize()
        for i in list(range(0, 1500, 97)) + [1499]:
            check(b.out[i:i + 1], *b.want(i))


@TYPES
def test_decode_a_row_that_is_not_finite_stays_alone(dtype):
    for prefix in (0, 200):
        b = Batch([100, 33, 70], prefix, 4, 1, 128, dtype, 16)
        b.call()
        torch.cuda.synchronize()
        clean = b.out.clone()
        b.q[1, 128:256] = NAN                                    # head 1 of sequence 1
        b.call()
        torch.cuda.synchronize()
        assert torch.isnan(b.out[1, 1]).all()
        b.out[1, 1] = clean[1, 1]
        want = [b.want(i) for i in (0, 2)]
        check(b.out[0:1], *want[0])
        check(b.out[2:3], *want[1])
        assert torch.isfinite(b.out).all()


def test_prompt_clusters_and_long_keys():
    """Few queries over many keys, so that CTAs of a cluster share them: the same rows as query by query."""
    for H, Hk, D, n, m in ((4, 1, 128, 70, 3000), (20, 5, 128, 33, 2100), (2, 2, 64, 300, 1500), (7, 1, 80, 40, 2500)):
        q, k, v = randn(1, n, H, D, scale=1.5), randn(2, m, Hk, D), randn(3, m, Hk, D)
        out = torch.zeros_like(q)
        sp.attention_prompt(q, k, v, out, i32([0, n]), i32([0, m]), 1, n, m, H, Hk, D)
        torch.cuda.synchronize()
        for i in (0, 1, n // 2, n - 1):
            top = i + m - n + 1
            want, tol = attend(q[i:i + 1], k[:top], v[:top], sp.F16, D ** -0.5, False)
            check(out[i:i + 1], want, tol)
        v[m - n + 20, 0, 3] = NAN                                # a key that the queries from 20 on see
        sp.attention_prompt(q, k, v, out, i32([0, n]), i32([0, m]), 1, n, m, H, Hk, D)
        torch.cuda.synchronize()
        g = H // Hk
        assert torch.isfinite(out[:20]).all() and torch.isnan(out[20:, :g, 3]).all() and torch.isfinite(out[20:, :, 4:]).all()
        for i in (0, 19):
            top = i + m - n + 1
            check(out[i:i + 1], *attend(q[i:i + 1], k[:top], v[:top], sp.F16, D ** -0.5, False))


def test_no_wait_ran_out():
    assert sp.attention_status() == 0
