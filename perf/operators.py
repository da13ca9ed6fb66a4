"""What the attention operators of sptmm_b200 are measured on: their inputs, their plain forms in
elementary torch operations, the calls a user makes of them, and the same results in 64 bits.

Three operators stand between the qkv projection and the output projection of a quantised layer:

  rotate   the fused qkv row of every token -> norms of its query and key heads, position rotation,
           16-bit rounding, and the keys and values put where attention reads them (packed rows of a
           prompt, slots of a paged cache)
  prompt   attention over whole prompts: packed sequences of different lengths, grouped heads, causal
           with the last query on the last key
  decode   one new token per sequence over a paged cache, optionally behind a prefix that the whole
           batch shares

The head shapes are 20 query heads over 5 key heads of 128 channels (hidden 2560, kv 640) and generic
ones.  Lists (sequence lengths, contexts) are comma-separated texts.
"""
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def ints(text):
    return [int(x) for x in text.split(",")] if text else []


def _sp():
    import sptmm_b200 as sp
    return sp, {"f32": sp.F32, "f16": sp.F16, "bf16": sp.BF16}


# ---- cases ---------------------------------------------------------------------------------------

def rotate_case(tokens, heads, kv_heads, head_dim, src, dtype, rot_dim, interleaved, norm, packed, page, max_pos):
    return {"op": "rotate", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "src": src,
            "dtype": dtype, "rot_dim": rot_dim, "interleaved": interleaved, "norm": norm, "packed": packed, "page": page,
            "max_pos": max_pos}


def prompt_case(lengths, context, heads, kv_heads, head_dim, dtype, causal=True):
    return {"op": "prompt", "lengths": lengths, "context": context, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "causal": causal}


def decode_case(lengths, prefix, heads, kv_heads, head_dim, dtype, page):
    return {"op": "decode", "lengths": lengths, "prefix": prefix, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "page": page}


def listed():
    ragged = random.Random(5)
    cases = [
        # a decode step of sixteen requests: one token each, far positions, straight into the cache
        ("rotate_step16", rotate_case(16, 20, 5, 128, "f32", "f16", 128, False, True, False, 16, 131072)),
        # a prompt of 8192 tokens from the float results of the qkv projection
        ("rotate_prompt8192", rotate_case(8192, 20, 5, 128, "f32", "bf16", 128, False, True, True, 64, 8192)),
        # an odd number of tokens from 16-bit rows: adjacent pairs, half of the channels rotated, no norms
        ("rotate_odd1021", rotate_case(1021, 16, 16, 64, "f16", "f16", 32, True, False, True, 0, 4096)),
        # a handful of short chat turns packed into one call
        ("prompt_short", prompt_case("37,128,5,300,1,211,64", "", 20, 5, 128, "f16")),
        # one long document
        ("prompt_8192", prompt_case("8192", "", 20, 5, 128, "bf16")),
        # mixed traffic: one very long prompt beside others down to a single token
        ("prompt_mixed", prompt_case("233,16384,64,9001,1,4001,1777", "", 20, 5, 128, "f16")),
        # a head of 64 channels for each query head, odd lengths
        ("prompt_heads64", prompt_case("1023,2049,515", "", 16, 16, 64, "bf16")),
        # the last 512 tokens of a prompt whose first 7680 were done before
        ("prompt_chunk", prompt_case("512", "7680", 20, 5, 128, "bf16")),
        # one request with a short history: latency
        ("decode_one", decode_case("300", 0, 20, 5, 128, "f16", 16)),
        # a batch of 64 requests of very different ages
        ("decode_ragged64", decode_case(",".join(str(int(8192 ** ragged.random())) for _ in range(64)), 0, 20, 5, 128, "bf16", 16)),
        # 64 requests behind one system prompt of 8192 tokens
        ("decode_prefix64", decode_case(",".join(str(ragged.randint(1, 700)) for _ in range(64)), 8192, 20, 5, 128, "f16", 16)),
        # two requests with 128k tokens of history
        ("decode_long", decode_case("131072,130001", 0, 20, 5, 128, "bf16", 64)),
    ]
    return [dict(case, name=name) for name, case in cases]


HEADS = ((20, 5, 128), (16, 16, 64), (32, 8, 128), (28, 4, 128), (8, 1, 128), (12, 4, 80), (16, 2, 96), (14, 2, 64))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    most = {}
    for case in listed():
        w = work(case)
        b, f = most.get(case["op"], (0, 0))
        most[case["op"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        op = rng.choice(("rotate", "prompt", "decode"))
        heads, kv_heads, head_dim = rng.choice(HEADS)
        dtype = rng.choice(("f16", "bf16"))
        page = rng.choice((16, 32, 64, 128))
        if op == "rotate":
            packed = rng.random() < 0.6
            case = rotate_case(_log(rng, 1, 8192), heads, kv_heads, head_dim, rng.choice(("f32", "f32", dtype)), dtype,
                               rng.choice((head_dim, head_dim, head_dim // 16 * 8)), rng.random() < 0.3, rng.random() < 0.6, packed,
                               page if not packed or rng.random() < 0.5 else 0, _log(rng, 1000, 131072))
        elif op == "prompt":
            lengths = [_log(rng, 1, 16384) for _ in range(rng.choice((1, 1, 2, 3, 5, 8, 13)))]
            context = [_log(rng, 1, 8192) for _ in lengths] if rng.random() < 0.3 else []
            case = prompt_case(",".join(map(str, lengths)), ",".join(map(str, context)), heads, kv_heads, head_dim, dtype,
                               rng.random() < 0.85)
        else:
            batch, top = _log(rng, 1, 128), _log(rng, 64, 131072)
            lengths = [_log(rng, 1, top) for _ in range(batch)]
            case = decode_case(",".join(map(str, lengths)), rng.choice((0, _log(rng, 100, 16384))), heads, kv_heads, head_dim, dtype, page)
        w = work(case)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1]:
            return case


def work(case):
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rotate":
        t, out = case["tokens"], SIZE[case["dtype"]]
        copies = (1 if case["packed"] else 0) + (1 if case["page"] else 0)
        values = t * (h + 2 * hk) * d
        return {"bytes": values * SIZE[case["src"]] + t * h * d * out + copies * t * 2 * hk * d * out + 4 * t,
                "flops": t * (h + hk) * d * (7 if case["norm"] else 3)}
    if case["op"] == "prompt":
        lengths = ints(case["lengths"])
        context = ints(case["context"]) or [0] * len(lengths)
        keys = sum(lengths) + sum(context)
        pairs = sum(n * c + (n * (n + 1) // 2 if case["causal"] else n * n) for n, c in zip(lengths, context))
        return {"bytes": 2 * d * (2 * sum(lengths) * h + 2 * keys * hk), "flops": 4 * d * h * pairs}
    lengths = ints(case["lengths"])
    keys = sum(lengths) + case["prefix"]                      # the shared prefix is read once
    return {"bytes": 2 * d * (2 * len(lengths) * h + 2 * keys * hk),
            "flops": 4 * d * h * (sum(lengths) + len(lengths) * case["prefix"])}


# ---- inputs --------------------------------------------------------------------------------------

def _randn(gen, shape, dtype, scale=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    if out.numel():
        out.normal_(0.0, scale, generator=gen)
    return out


def _offsets(lengths):
    return [0] + list(np.cumsum(lengths, dtype=np.int64).tolist())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dev = dict(device="cuda")
    st = dict(case)
    h, hk, d, dt = case["heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    if case["op"] == "rotate":
        t, page = case["tokens"], case["page"]
        st["x"] = _randn(gen, (t, (h + 2 * hk) * d), DTYPES[case["src"]], 1.7)
        if t > 8 or not case["packed"]:
            pos = [rng.randrange(case["max_pos"]) for _ in range(t)] if t <= 128 else [i % case["max_pos"] for i in range(t)]
        else:
            pos = list(range(t))
        st["positions"] = torch.tensor(pos, dtype=torch.int32, **dev)
        r = case["rot_dim"]
        st["inv_freq"] = np.array([500000.0 ** (-2.0 * i / r) for i in range(r // 2)], dtype=np.float64)
        st["q_norm"] = 1.0 + 0.2 * _randn(gen, (d,), torch.float32) if case["norm"] else None
        st["k_norm"] = 1.0 + 0.2 * _randn(gen, (d,), torch.float32) if case["norm"] else None
        st["q"] = torch.zeros((t, h, d), dtype=dt, **dev)
        st["k"] = torch.zeros((t, hk, d), dtype=dt, **dev) if case["packed"] else None
        st["v"] = torch.zeros((t, hk, d), dtype=dt, **dev) if case["packed"] else None
        st["cache"] = st["slots"] = None
        if page:
            n_pages = (t + page - 1) // page + 3
            order = list(range(n_pages))
            rng.shuffle(order)
            slots = [order[i // page] * page + i % page for i in range(t)]
            if t >= 8:
                slots[t // 2] = -1                            # a padded row of the batch: not stored
            st["slots"] = torch.tensor(slots, dtype=torch.int32, **dev)
            st["k_pages"] = torch.zeros((n_pages, hk, page, d), dtype=dt, **dev)
            st["v_pages"] = torch.zeros((n_pages, hk, page, d), dtype=dt, **dev)
            if own:
                sp, names = _sp()
                st["cache"] = sp.KVCache(st["k_pages"], st["v_pages"], n_pages, page, hk, d, names[case["dtype"]])
        return st
    lengths = ints(case["lengths"])
    if case["op"] == "prompt":
        context = ints(case["context"]) or [0] * len(lengths)
        st["q_off"] = _offsets(lengths)
        st["k_off"] = _offsets([n + c for n, c in zip(lengths, context)])
        st["q_offsets"] = torch.tensor(st["q_off"], dtype=torch.int32, **dev)
        st["k_offsets"] = torch.tensor(st["k_off"], dtype=torch.int32, **dev)
        st["q"] = _randn(gen, (st["q_off"][-1], h, d), dt, 1.6)
        st["k"] = _randn(gen, (st["k_off"][-1], hk, d), dt)
        st["v"] = _randn(gen, (st["k_off"][-1], hk, d), dt)
        st["out"] = torch.zeros((st["q_off"][-1], h, d), dtype=dt, **dev)
        return st
    page, prefix, batch = case["page"], case["prefix"], len(lengths)
    counts = [(n + page - 1) // page for n in lengths]
    prefix_count = (prefix + page - 1) // page
    n_pages = sum(counts) + prefix_count + 1
    order = list(range(n_pages))
    rng.shuffle(order)
    st["prefix_list"] = order[:prefix_count]
    rows, at = [], prefix_count
    for c in counts:
        rows.append(order[at:at + c])
        at += c
    st["pages"] = rows
    st["max_pages"] = max(counts)
    st["table"] = torch.tensor([r + [0] * (st["max_pages"] - len(r)) for r in rows], dtype=torch.int32, **dev)
    st["prefix_table"] = torch.tensor(st["prefix_list"], dtype=torch.int32, **dev) if prefix else None
    st["seq_lengths"] = torch.tensor(lengths, dtype=torch.int32, **dev)
    st["k_pages"] = _randn(gen, (n_pages, hk, page, d), dt)
    st["v_pages"] = _randn(gen, (n_pages, hk, page, d), dt)
    st["q"] = _randn(gen, (batch, h, d), dt, 1.6)
    st["out"] = torch.zeros((batch, h, d), dtype=dt, **dev)
    if own:
        sp, names = _sp()
        st["cache"] = sp.KVCache(st["k_pages"], st["v_pages"], n_pages, page, hk, d, names[case["dtype"]])
        nbytes = sp.attention_decode_workspace(batch, h, hk, d, prefix)
        st["workspace"] = torch.empty(nbytes, dtype=torch.uint8, **dev)
    return st


# ---- one pass ------------------------------------------------------------------------------------

def run(st):
    return {"rotate": _rotate, "prompt": _prompt, "decode": _decode}[st["op"]](st)


def _rotate(st):
    h, hk, d, t, r = st["heads"], st["kv_heads"], st["head_dim"], st["tokens"], st["rot_dim"]
    if own:
        sp, names = _sp()
        sp.rotate_heads(st["x"], t, h, hk, d, st["positions"], st["inv_freq"], st["q"], in_dtype=names[st["src"]],
                        dtype=names[st["dtype"]], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=1e-5,
                        interleaved=st["interleaved"], K=st["k"], V=st["v"], cache=st["cache"], slots=st["slots"],
                        stream=torch.cuda.current_stream().cuda_stream)
        return [x for x in (st["q"], st["k"], st["v"], st.get("k_pages"), st.get("v_pages")) if x is not None]
    dt = DTYPES[st["dtype"]]
    x = st["x"].float().view(t, h + 2 * hk, d)
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    if st["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-5) * st["q_norm"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-5) * st["k_norm"]
    inv = torch.from_numpy(st["inv_freq"]).to("cuda", non_blocking=True)
    angle = st["positions"].double()[:, None] * inv[None, :]                    # far positions need 64 bits
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]

    def turn(y):
        rot = y[..., :r]
        a, b = (rot[..., 0::2], rot[..., 1::2]) if st["interleaved"] else (rot[..., :r // 2], rot[..., r // 2:])
        a, b = a * cos - b * sin, a * sin + b * cos
        rot = torch.stack((a, b), -1).flatten(-2) if st["interleaved"] else torch.cat((a, b), -1)
        return torch.cat((rot, y[..., r:]), -1).to(dt)

    q, k, v = turn(q), turn(k), v.to(dt)
    out = [q]
    if st["packed"]:
        out += [k, v]
    if st["page"]:
        page = st["page"]
        keep = st["slots"] >= 0
        slot = st["slots"][keep].long()
        st["k_pages"][slot // page, :, slot % page] = k[keep]
        st["v_pages"][slot // page, :, slot % page] = v[keep]
        out += [st["k_pages"], st["v_pages"]]
    return out


def _plain_attention(q, k, v, dt, causal):
    """q (n, heads, d) over k, v (m, kv_heads, d); with `causal` the last query sees the last key."""
    n, h, d = q.shape
    m, hk, _ = k.shape
    g = h // hk
    if m == 0 or n == 0:
        return torch.zeros((n, h, d), dtype=dt, device=q.device)
    q = q.float().view(n, hk, g, d).permute(1, 2, 0, 3) * d ** -0.5             # hk, g, n, d
    k = k.float().permute(1, 2, 0)[:, None]                                     # hk, 1, d, m
    v = v.float().permute(1, 0, 2)[:, None]                                     # hk, 1, m, d
    out = torch.empty((n, h, d), dtype=dt, device=q.device)
    rows = max(1, min(n, (1 << 28) // (h * m)))
    for r0 in range(0, n, rows):
        r1 = min(n, r0 + rows)
        top = min(m, m - n + r1) if causal else m
        s = torch.matmul(q[:, :, r0:r1], k[..., :top])
        if causal:
            last = torch.arange(r0, r1, device=q.device) + (m - n)
            s = s.masked_fill(torch.arange(top, device=q.device)[None, :] > last[:, None], float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p, v[:, :, :top]) / p.sum(-1, keepdim=True)
        out[r0:r1] = o.permute(2, 0, 1, 3).reshape(r1 - r0, h, d).to(dt)
    return out


def _prompt(st):
    h, hk, d, n = st["heads"], st["kv_heads"], st["head_dim"], len(st["q_off"]) - 1
    if own:
        sp, names = _sp()
        sp.attention_prompt(st["q"], st["k"], st["v"], st["out"], st["q_offsets"], st["k_offsets"], n, st["q_off"][-1],
                            st["k_off"][-1], h, hk, d, dtype=names[st["dtype"]], causal=st["causal"],
                            stream=torch.cuda.current_stream().cuda_stream)
        return st["out"]
    dt = DTYPES[st["dtype"]]
    return torch.cat([_plain_attention(st["q"][a:b], st["k"][c:e], st["v"][c:e], dt, st["causal"])
                      for a, b, c, e in zip(st["q_off"], st["q_off"][1:], st["k_off"], st["k_off"][1:])])


def _rows_of(pages, index, count):
    """The first `count` keys or values of the listed pages as (count, kv_heads, d)."""
    x = pages[index].permute(0, 2, 1, 3)
    return x.reshape(-1, x.shape[2], x.shape[3])[:count]


def _decode(st):
    h, hk, d, lengths = st["heads"], st["kv_heads"], st["head_dim"], ints(st["lengths"])
    if own:
        sp, _ = _sp()
        sp.attention_decode(st["q"], st["out"], len(lengths), h, st["cache"], st["seq_lengths"], st["table"], st["max_pages"],
                            prefix_table=st["prefix_table"], prefix_len=st["prefix"], workspace=st["workspace"],
                            workspace_bytes=st["workspace"].numel(), stream=torch.cuda.current_stream().cuda_stream)
        return st["out"]
    dt, b, g, prefix = DTYPES[st["dtype"]], len(lengths), h // hk, st["prefix"]
    q = st["q"].float().view(b, hk, g, d) * d ** -0.5
    out = torch.empty((b, h, d), dtype=dt, device="cuda")
    if prefix:                                                # one product for the whole batch
        pk = _rows_of(st["k_pages"], st["prefix_table"], prefix).float().permute(1, 2, 0)
        pv = _rows_of(st["v_pages"], st["prefix_table"], prefix).float().permute(1, 0, 2)
        ps = torch.matmul(q.permute(1, 0, 2, 3).reshape(hk, b * g, d), pk)      # hk, b*g, prefix
        pm = ps.amax(-1, keepdim=True)
        pe = torch.exp(ps - pm)
        pl = pe.sum(-1, keepdim=True).view(hk, b, g, 1)
        po = torch.matmul(pe, pv).view(hk, b, g, d)
        pm = pm.view(hk, b, g, 1)
    for i, n in enumerate(lengths):
        index = st["table"][i, :(n + st["page"] - 1) // st["page"]]
        k = _rows_of(st["k_pages"], index, n).float().permute(1, 2, 0)
        v = _rows_of(st["v_pages"], index, n).float().permute(1, 0, 2)
        s = torch.matmul(q[i], k)
        m = s.amax(-1, keepdim=True)
        if prefix:
            m = torch.maximum(m, pm[:, i])
        e = torch.exp(s - m)
        l, o = e.sum(-1, keepdim=True), torch.matmul(e, v)
        if prefix:
            w = torch.exp(pm[:, i] - m)
            l, o = l + pl[:, i] * w, o + po[:, i] * w
        out[i] = (o / l).reshape(h, d).to(dt)
    return out


# ---- the same in 64 bits, head by head from the definitions ------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(st)
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "prompt":
        out = torch.zeros((st["q_off"][-1], h, d), dtype=torch.float64, device="cuda")
        for i in range(len(st["q_off"]) - 1):
            a, b, c, e = st["q_off"][i], st["q_off"][i + 1], st["k_off"][i], st["k_off"][i + 1]
            for head in range(h):
                k, v = st["k"][c:e, head // (h // hk)].double(), st["v"][c:e, head // (h // hk)].double()
                for r0 in range(a, b, 4096):
                    r1 = min(b, r0 + 4096)
                    logits = torch.einsum("nd,md->nm", st["q"][r0:r1, head].double(), k) / d ** 0.5
                    if case["causal"]:
                        hidden = torch.ones_like(logits, dtype=torch.bool).triu((e - c) - (b - a) + (r0 - a) + 1)
                        logits[hidden] = -float("inf")
                    out[r0:r1, head] = torch.exp(logits - torch.logsumexp(logits, 1)[:, None]) @ v
        return out
    lengths = ints(case["lengths"])
    out = torch.zeros((len(lengths), h, d), dtype=torch.float64, device="cuda")

    def rows(pages, index, count, head):
        return torch.cat([pages[p, head] for p in index], 0)[:count].double() if index else pages.new_zeros((0, d)).double()

    for j in range(hk):
        pk, pv = (rows(st[x], st["prefix_list"], case["prefix"], j) for x in ("k_pages", "v_pages"))
        for i, n in enumerate(lengths):
            k = torch.cat((pk, rows(st["k_pages"], st["pages"][i], n, j)))
            v = torch.cat((pv, rows(st["v_pages"], st["pages"][i], n, j)))
            g = slice(j * (h // hk), (j + 1) * (h // hk))
            logits = st["q"][i, g].double() @ k.T / d ** 0.5
            out[i, g] = torch.exp(logits - torch.logsumexp(logits, 1)[:, None]) @ v
    return out


def _exact_rotate(st):
    h, hk, d, r, t = st["heads"], st["kv_heads"], st["head_dim"], st["rot_dim"], st["tokens"]
    x = st["x"].double().view(t, h + 2 * hk, d).clone()
    if st["norm"]:
        weights = [st["q_norm"]] * h + [st["k_norm"]] * hk
        for i, w in enumerate(weights):
            x[:, i] *= w.double() / torch.sqrt(x[:, i].square().sum(-1, keepdim=True) / d + 1e-5)
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                    torch.outer(st["positions"].double(), torch.from_numpy(st["inv_freq"]).cuda()))
    first = torch.arange(r // 2, device="cuda") * (2 if st["interleaved"] else 1)
    second = first + (1 if st["interleaved"] else r // 2)
    for i in range(h + hk):                                   # a pair of channels is one complex number
        pair = torch.complex(x[:, i, first], x[:, i, second]) * z
        x[:, i, first], x[:, i, second] = pair.real, pair.imag
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    out = [q]
    if st["packed"]:
        out += [k, v]
    if st["page"]:
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        slots = st["slots"].tolist()
        keep = [i for i, s in enumerate(slots) if s >= 0]
        page = torch.tensor([slots[i] // st["page"] for i in keep], device="cuda")
        slot = torch.tensor([slots[i] % st["page"] for i in keep], device="cuda")
        kp[page, :, slot], vp[page, :, slot] = k[keep], v[keep]
        out += [kp, vp]
    return out
