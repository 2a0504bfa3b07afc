"""Packed-sequence attention and rotary positions on several axes, as timed cases.

Each case is one pass through ``packed_attention`` or ``rotary_embed`` as a program calls it: over
packed prompts and images of different lengths (inference, and training with the three gradients),
over the keys of a cache with one or some new tokens a sequence, and the rotation of queries and
keys by their positions. ``lengths`` are the sequences' numbers of queries, ``keys`` their numbers
of keys, ``room`` the rows that a cache holds for each sequence (0: the keys are packed too).
:func:`draw` gives further cases of the same ranges.

Where ``own`` is false, :func:`run` computes the same from elementary torch operations in 32 bits.
"""

import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _package():
    path = os.path.join(os.getcwd(), "rf-detr-jax_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import rfdetr_jax_amd

    return rfdetr_jax_amd


def _ragged(count, lo, hi):
    """`count` lengths between lo and hi, spread over their logarithm in no order."""
    return ",".join(str(round(lo * (hi / lo) ** ((i * 0.6180339887498949) % 1.0))) for i in range(count))


def _attention(name, lengths, heads, kv_heads, head_dim, dtype="bf16", keys="", room=0, causal=True, train=False):
    return {"name": name, "op": "attention", "lengths": lengths, "keys": keys or lengths, "room": room, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "causal": causal, "train": train}


def _rotary(name, tokens, heads, kv_heads, head_dim, sections, positions, dtype, shared, interleaved, train):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "sections": sections, "positions": positions, "dtype": dtype, "shared": shared, "interleaved": interleaved, "train": train}


def listed():
    return [
        # One new token of one sequence over a short cache: the smallest call, launch latency.
        _attention("one_token_bf16", "1", 8, 2, 64, keys="517", room=1024),
        # Serving 64 sequences, one new token each, over caches filled to different lengths: the
        # bytes of the keys and values.
        _attention("tokens_cache_bf16", ",".join(["1"] * 64), 32, 8, 128, keys=_ragged(64, 129, 8000), room=8192),
        # New tokens of a few sequences (a chunk of a prompt, the end of one, a single token) over
        # long caches: few query rows, many keys.
        _attention("chunk_cache_bf16", "256,77,1", 16, 4, 128, keys="16001,5021,9000", room=16384),
        # A batch of packed prompts: the largest call, bound by its products.
        _attention("prompt_bf16", "7001,4096,2900,1500,503", 32, 8, 128),
        # The same kind in f32 at a small size, as many key heads as query heads.
        _attention("prompt_f32", "1500,400,33", 8, 8, 64, dtype="f32"),
        # Training on packed prompts down to one token, four query heads to a key head.
        _attention("train_prompt_bf16", "4096,2048,1531,777,300,95,1", 16, 4, 128, train=True),
        # Training a vision transformer on packed images of different sizes: 24 x 24 to 36 x 36
        # patches, every patch sees its whole image.
        _attention("train_images_bf16", "576,1296,768,400,1024,576,900,1296", 12, 12, 64, causal=False, train=True),
        # Training the decoder's self-attention (8 heads of 32 channels) on packed sets of at most 300
        # queries, f32.
        _attention("train_queries_f32", _ragged(26, 100, 300), 8, 8, 32, dtype="f32", causal=False, train=True),
        # Positions of one new token each of 64 sequences, far into them: launch latency.
        _rotary("rotary_tokens_bf16", 64, 32, 8, 128, "16,24,24", "far", "bf16", True, False, False),
        # Queries and keys of a packed batch with images and video in it, three axes, in training:
        # the bytes of the rows.
        _rotary("rotary_train_bf16", 16000, 32, 8, 128, "16,24,24", "text", "bf16", True, False, True),
        # Two axes with frequencies of their own over 8 images of 24 x 24 patches, neighbouring
        # channels paired, fractional positions, f32 training.
        _rotary("rotary_images_f32", 4608, 8, 8, 32, "8,8", "grid", "f32", False, True, True),
    ]


def _between(rng, lo, hi):
    """A whole number, its logarithm uniform."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


_MOST = 2 * 10 ** 11  # products of a drawn attention case: no more than the largest listed one's


def draw(rng):
    if rng.random() < 0.3:
        d = rng.choice([32, 64, 64, 80, 128])
        axes = rng.choice([1, 2, 3])
        pairs = d // 2 if rng.random() < 0.7 else d // 4
        cut = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = [b - a for a, b in zip([0, *cut], [*cut, pairs])]
        kv = rng.choice([1, 2, 4, 8])
        return {"op": "rotary", "tokens": _between(rng, 1, 16000), "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "head_dim": d,
                "sections": ",".join(str(s) for s in sections), "positions": rng.choice(["far", "text", "grid"]),
                "dtype": rng.choice(["f32", "bf16", "bf16"]), "shared": rng.random() < 0.5, "interleaved": rng.random() < 0.5,
                "train": rng.random() < 0.5}
    kind = rng.choice(["tokens", "chunk", "prompt", "train", "train"])
    kv = rng.choice([1, 2, 4, 8])
    case = {"op": "attention", "heads": kv * rng.choice([1, 1, 2, 3, 4, 8]), "kv_heads": kv,
            "head_dim": rng.choice([32, 40, 64, 64, 80, 96, 128, 128]), "dtype": rng.choice(["f32", "bf16", "bf16", "bf16"]),
            "causal": kind in ("tokens", "chunk") or rng.random() < 0.6, "train": kind == "train", "room": 0}
    if kind in ("tokens", "chunk"):
        count = _between(rng, 1, 64 if kind == "tokens" else 8)
        case["room"] = _between(rng, 128, 16384)
        keys = [_between(rng, 1, case["room"]) for _ in range(count)]
        lengths = [1 if kind == "tokens" else min(m, _between(rng, 1, 300)) for m in keys]
    else:
        lengths = [_between(rng, 1, 4096) for _ in range(_between(rng, 1, 16))]
        keys = list(lengths)
        if rng.random() < 0.2:  # a sequence without tokens, and rows that see no key
            lengths.insert(rng.randrange(len(lengths) + 1), 0)
            keys = [n if rng.random() < 0.7 else n // 2 for n in lengths]
    while case["heads"] * sum(n * m for n, m in zip(lengths, keys)) * case["head_dim"] > _MOST:
        i = lengths.index(max(lengths))
        lengths[i], keys[i] = lengths[i] // 2, keys[i] // 2
    case["lengths"], case["keys"] = (",".join(str(x) for x in t) for t in (lengths, keys))
    return case


def _numbers(text):
    return [int(x) for x in text.split(",")]


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rotary":
        rows, pairs = case["tokens"] * (h + hk), sum(_numbers(case["sections"]))
        passes = 2 if case["train"] else 1
        return {"bytes": 2 * rows * d * size * passes + case["tokens"] * 4 * len(_numbers(case["sections"])),
                "flops": 6 * rows * pairs * passes}
    lengths, keys = _numbers(case["lengths"]), _numbers(case["keys"])
    pairs = 0
    for n, m in zip(lengths, keys):
        if not case["causal"]:
            pairs += n * m
        else:  # query t sees keys 0 .. t + m - n
            first = max(1, m - n + 1)
            pairs += max(0, (first + m) * (m - first + 1) // 2)
    q, kv = sum(lengths) * h * d * size, sum(keys) * hk * d * size
    if not case["train"]:
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * h * d}
    return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * h * d}


# -- inputs -------------------------------------------------------------------------------------


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    dt, h, hk, d = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["head_dim"]
    state = {"case": case}
    if case["op"] == "rotary":
        t, axes = case["tokens"], len(_numbers(case["sections"]))
        qkv = normal(t, h + 2 * hk, d).to(dt)  # one projection's rows; q and k are slices of them
        state["inputs"] = [x.detach().requires_grad_(case["train"]) for x in (qkv[:, :h], qkv[:, h:h + hk])]
        if case["positions"] == "grid":  # fractional coordinates
            state["positions"] = torch.rand((t, axes), generator=g, device="cuda") * 36
        else:
            far = 1_000_000 if case["positions"] == "far" else 16_000
            start = torch.randint(0, far, (t, 1), generator=g, device="cuda")
            state["positions"] = (start + torch.randint(0, 64, (t, axes), generator=g, device="cuda")).to(torch.int32)
        if case["train"]:
            state["grads"] = [normal(t, n, d).to(dt) for n in (h, hk)]
        return state
    lengths, keys, room = _numbers(case["lengths"]), _numbers(case["keys"]), case["room"]
    state["lengths"], state["keys"] = lengths, keys
    starts = _starts(lengths)
    key_starts = [i * room for i in range(len(keys) + 1)] if room else _starts(keys)
    state["starts"], state["key_starts"] = starts, key_starts
    state["offsets"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    state["key_offsets"] = state["offsets"] if key_starts == starts else torch.tensor(key_starts, dtype=torch.int32, device="cuda")
    state["key_lengths"] = torch.tensor(keys, dtype=torch.int32, device="cuda") if room else None
    if key_starts == starts:  # one projection's rows
        qkv = normal(starts[-1], h + 2 * hk, d).to(dt)
        inputs = [1.5 * qkv[:, :h] if not case["train"] else qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]]
    else:
        inputs = [1.5 * normal(starts[-1], h, d).to(dt), normal(key_starts[-1], hk, d).to(dt), normal(key_starts[-1], hk, d).to(dt)]
    state["inputs"] = [x.detach().requires_grad_(case["train"]) for x in inputs]
    if case["train"]:
        state["grad"] = normal(starts[-1], h, d).to(dt)
    return state


# -- one pass -----------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        if not own:
            return _plain_rotary(state)
        q, k = state["inputs"]
        out = _package().rotary_embed(q, k, state["positions"], tuple(_numbers(case["sections"])),
                                      shared_frequencies=case["shared"], interleaved=case["interleaved"])
        if not case["train"]:
            return {"q": out[0], "k": out[1]}
        grads = torch.autograd.grad(out, (q, k), state["grads"])
        return {"q": out[0], "k": out[1], "grad_q": grads[0], "grad_k": grads[1]}
    if not own:
        return _plain_attention(state)
    inputs = state["inputs"]
    out = _package().packed_attention(*inputs, state["offsets"], state["key_offsets"], state["key_lengths"], causal=case["causal"])
    if not case["train"]:
        return {"out": out}
    grads = torch.autograd.grad(out, inputs, state["grad"])
    return {"out": out, "grad_q": grads[0], "grad_k": grads[1], "grad_v": grads[2]}


# -- the plain form -----------------------------------------------------------------------------


def _turn(x, cos, sin, interleaved):
    """Rotates the pairs of x [T, heads, D] by angles [T, n]; channels from 2 n on stay."""
    n = cos.shape[1]
    x = x.float()
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _angles(case, positions):
    sections = _numbers(case["sections"])
    n, columns = sum(sections), []
    start = 0
    for a, s in enumerate(sections):
        p = torch.arange(s, dtype=torch.float64, device="cuda")
        e = (p + start) / n if case["shared"] else p / s
        columns.append(positions[:, a:a + 1].double() * torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"), -e))
        start += s
    return torch.cat(columns, 1)


def _plain_rotary(state):
    case = state["case"]
    angle = _angles(case, state["positions"])  # 64 bits: positions are far from 0
    cos, sin = angle.cos().float(), angle.sin().float()
    dt = DTYPES[case["dtype"]]
    out = {n: _turn(x.detach(), cos, sin, case["interleaved"]).to(dt) for n, x in zip("qk", state["inputs"])}
    if case["train"]:
        out.update({f"grad_{n}": _turn(g, cos, -sin, case["interleaved"]).to(dt) for n, g in zip("qk", state["grads"])})
    return out


def _plain_attention(state):
    case = state["case"]
    dt, hk, d, train = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"], case["train"]
    q, k, v = (x.detach() for x in state["inputs"])
    group = case["heads"] // hk
    scale = d ** -0.5
    out = torch.zeros(q.shape, dtype=dt, device="cuda")
    if train:
        gq, gk, gv = (torch.zeros(x.shape, dtype=dt, device="cuda") for x in (q, k, v))
    for i, (n, m) in enumerate(zip(state["lengths"], state["keys"])):
        if n == 0 or m == 0:
            continue
        rows, cols = slice(state["starts"][i], state["starts"][i] + n), slice(state["key_starts"][i], state["key_starts"][i] + m)
        # [key heads, tokens, group, D]
        qi = q[rows].float().view(n, hk, group, d).transpose(0, 1)
        ki, vi = (x[cols].float().transpose(0, 1).contiguous() for x in (k, v))
        if train:
            gi = state["grad"][rows].float().view(n, hk, group, d).transpose(0, 1)
            dk, dv = torch.zeros_like(ki), torch.zeros_like(vi)
        step = max(1, (1 << 28) // (m * hk * group))  # some rows at a time bound the memory
        for t in range(0, n, step):
            e = min(n, t + step)
            qs = qi[:, t:e].reshape(hk, -1, d)
            s = torch.bmm(qs, ki.transpose(1, 2)) * scale
            if case["causal"]:
                seen = torch.arange(m, device="cuda")[None, :] <= torch.arange(t, e, device="cuda")[:, None] + (m - n)
                seen = seen.repeat_interleave(group, 0)
                s = torch.where(seen, s, -torch.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, 1.0, total)
            del s
            o = torch.bmm(p, vi)
            out[rows][t:e] = o.view(hk, e - t, group, d).transpose(0, 1).reshape(e - t, -1, d).to(dt)
            if train:
                gs = gi[:, t:e].reshape(hk, -1, d)
                dv += torch.bmm(p.transpose(1, 2), gs)
                dp = torch.bmm(gs, vi.transpose(1, 2))
                ds = p * (dp - (gs * o).sum(-1, keepdim=True)) * scale
                gq[rows][t:e] = torch.bmm(ds, ki).view(hk, e - t, group, d).transpose(0, 1).reshape(e - t, -1, d).to(dt)
                dk += torch.bmm(ds.transpose(1, 2), qs)
        if train:
            gk[cols], gv[cols] = dk.transpose(0, 1).to(dt), dv.transpose(0, 1).to(dt)
    if not train:
        return {"out": out}
    return {"out": out, "grad_q": gq, "grad_k": gk, "grad_v": gv}


# -- the same in 64 bits ------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        # as complex numbers: a pair times exp(i angle), its gradient times exp(-i angle)
        sections = _numbers(case["sections"])
        n = sum(sections)
        axis = torch.tensor([a for a, s in enumerate(sections) for _ in range(s)], device="cuda")
        local = torch.tensor([j / s for s in sections for j in range(s)], dtype=torch.float64, device="cuda")
        power = torch.arange(n, dtype=torch.float64, device="cuda") / n if case["shared"] else local
        angle = state["positions"].double()[:, axis] * torch.exp(-power * torch.log(torch.tensor(10000.0, dtype=torch.float64)).item())

        def turned(x, sign):
            x = x.detach().double().clone()
            even, odd = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if case["interleaved"] else (slice(0, n), slice(n, 2 * n))
            z = torch.complex(x[..., even].contiguous(), x[..., odd].contiguous()) * torch.polar(torch.ones_like(angle), sign * angle)[:, None]
            x[..., even], x[..., odd] = z.real, z.imag
            return x

        out = {name: turned(x, 1.0) for name, x in zip("qk", state["inputs"])}
        if case["train"]:
            out.update({f"grad_{name}": turned(g, -1.0) for name, g in zip("qk", state["grads"])})
        return out
    q, k, v = (x.detach() for x in state["inputs"])
    group, train = case["heads"] // case["kv_heads"], case["train"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (q, k, v)] if train else []
    for i, (n, m) in enumerate(zip(state["lengths"], state["keys"])):
        if n == 0 or m == 0:
            continue
        a, b = state["starts"][i], state["key_starts"][i]
        seen = torch.ones((n, m), dtype=torch.bool, device="cuda")
        if case["causal"]:
            seen = seen.tril(m - n)
        for head in range(case["heads"]):
            at = [x[s:s + c, j].double().requires_grad_(train) for x, s, c, j in ((q, a, n, head), (k, b, m, head // group), (v, b, m, head // group))]
            w = (at[0] @ at[1].T / case["head_dim"] ** 0.5).masked_fill(~seen, float("-inf"))
            blind = ~seen.any(1, keepdim=True)
            w = torch.softmax(w.masked_fill(blind, 0.0), -1).masked_fill(blind, 0.0)
            o = w @ at[2]
            out[a:a + n, head] = o.detach()
            if train:
                for total, j, s, c, x in zip(grads, (head, head // group, head // group), (a, b, b), (n, m, m),
                                             torch.autograd.grad(o, at, state["grad"][a:a + n, head].double())):
                    total[s:s + c, j] += x
    if not train:
        return {"out": out}
    return {"out": out, "grad_q": grads[0], "grad_k": grads[1], "grad_v": grads[2]}
