"""Norms with rotary positions, packed attention with shaped scores, and a cache in 4 bits, as timed cases.

Each case is one pass through ``norm_rotary_embed``, ``packed_attention`` with a cap, a bias by distance, a window or a
prefix, ``cache4_attention``, or ``cache4_write`` and ``cache4_read`` of what was written, as a program calls them.
``lengths`` are the sequences' numbers of queries, ``keys`` their numbers of keys, ``room`` the rows that a cache holds
for each sequence (0: the keys are packed too). :func:`draw` gives further cases of the same ranges.

Where ``own`` is false, :func:`run` computes the same from elementary torch operations in 32 bits.
"""

import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6
BLOCK = 32  # channels of a cache row that share one scale


def _package():
    path = os.path.join(os.getcwd(), "rf-detr-jax_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import rfdetr_jax_amd

    return rfdetr_jax_amd


def _ragged(count, lo, hi):
    """`count` lengths between lo and hi, spread over their logarithm in no order."""
    return ",".join(str(round(lo * (hi / lo) ** ((i * 0.6180339887498949) % 1.0))) for i in range(count))


def _norm(name, tokens, heads, kv_heads, head_dim, sections, positions, dtype, interleaved=False, weights=True, train=False):
    return {"name": name, "op": "norm_rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "sections": sections, "positions": positions, "dtype": dtype, "interleaved": interleaved, "weights": weights, "train": train}


def _attention(name, lengths, heads, kv_heads, head_dim, dtype="bf16", keys="", room=0, causal=True, train=False, cap=0.0, slopes=False,
               window=0, prefixes=""):
    return {"name": name, "op": "attention", "lengths": lengths, "keys": keys or lengths, "room": room, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "causal": causal, "train": train, "cap": cap,
            "slopes": slopes, "window": window, "prefixes": prefixes}


def _cache(name, lengths, heads, kv_heads, head_dim, keys, room, dtype="bf16", cap=0.0, slopes=False, window=0):
    return {"name": name, "op": "cache_attention", "lengths": lengths, "keys": keys, "room": room, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "causal": True, "train": False, "cap": cap, "slopes": slopes, "window": window, "prefixes": ""}


def _write(name, lengths, kv_heads, head_dim, keys, room, dtype="bf16"):
    return {"name": name, "op": "cache_write", "lengths": lengths, "keys": keys, "room": room, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype}


def listed():
    return [
        # Queries and keys of one new token each of 64 sequences, far into them: launch latency.
        _norm("norm_rotary_tokens_bf16", 64, 32, 8, 128, "64", "far", "bf16"),
        # Queries and keys of a packed batch in training, three axes: the bytes of the rows, and the weights' gradients,
        # which are sums over all tokens and heads.
        _norm("norm_rotary_train_bf16", 16000, 32, 8, 128, "16,24,24", "text", "bf16", train=True),
        # A batch of packed prompts whose scores are capped: the largest call.
        _attention("capped_prompt_bf16", "6001,4500,3100,1700,601", 32, 8, 128, cap=50.0),
        # Training with a bias that falls with the distance, a slope for each of 16 heads, down to one token.
        _attention("sloped_train_bf16", "4001,2100,1531,777,300,95,1", 16, 16, 64, train=True, slopes=True),
        # Training on long sequences, scores capped, every token sees the last 1024.
        _attention("capped_window_train_bf16", "8192,3001,900", 16, 8, 128, train=True, cap=50.0, window=1024),
        # Training on packed pairs of an image (24 x 24 patches that see each other) and a text behind it, f32.
        _attention("prefix_train_f32", "833,640,577,1210", 8, 8, 32, dtype="f32", train=True, prefixes="576,576,576,576"),
        # Serving 64 sequences, one new token each, the last 4096 keys of caches filled to different lengths, scores capped.
        _attention("capped_tokens_bf16", ",".join(["1"] * 64), 32, 8, 128, keys=_ragged(64, 129, 8000), room=8192, cap=30.0, window=4096),
        # One new token of one sequence over a short cache in 4 bits: the smallest call.
        _cache("cache_one_token_bf16", "1", 8, 2, 64, keys="700", room=1024),
        # Serving 64 sequences, one new token each, over caches in 4 bits: their bytes.
        _cache("cache_tokens_bf16", ",".join(["1"] * 64), 32, 8, 128, keys=_ragged(64, 129, 8000), room=8192),
        # New tokens of a few sequences (a chunk of a prompt, the end of one, a single token) over long caches in 4 bits.
        _cache("cache_chunk_bf16", "200,61,1", 16, 4, 128, keys="15001,6021,9000", room=16384),
        # The keys and values of one new token each of 64 sequences into the cache, and back as a check of a store would.
        _write("cache_write_tokens_bf16", ",".join(["1"] * 64), 8, 128, keys=_ragged(64, 129, 8000), room=8192),
        # Those of whole prompts, f32.
        _write("cache_write_prompt_f32", "6001,4500,1333,97", 8, 128, keys="6001,4500,1400,97", room=8192, dtype="f32"),
    ]


def _between(rng, lo, hi):
    """A whole number, its logarithm uniform."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


_MOST = 5.6 * 10 ** 11  # operations of a drawn attention case: no more than the largest listed one's


def draw(rng):
    kind = rng.choice(["norm", "norm", "write", "cache", "cache", "cache", "tokens", "prompt", "train", "train", "train"])
    kv, d = rng.choice([1, 2, 4, 8]), rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    dtype = rng.choice(["f32", "bf16", "bf16", "bf16"])
    if kind == "norm":
        axes = rng.choice([1, 1, 2, 3])
        pairs = d // 2 if rng.random() < 0.7 else d // 4
        cut = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = [b - a for a, b in zip([0, *cut], [*cut, pairs])]
        return {"op": "norm_rotary", "tokens": _between(rng, 1, 16000), "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "head_dim": d,
                "sections": ",".join(str(s) for s in sections), "positions": rng.choice(["far", "text", "grid"]), "dtype": dtype,
                "interleaved": rng.random() < 0.5, "weights": rng.random() < 0.8, "train": rng.random() < 0.6}
    if kind in ("write", "cache", "tokens"):
        single = rng.random() < 0.6
        count = _between(rng, 1, 64 if single else 8)
        room = _between(rng, 128, 16384)
        keys = [_between(rng, 1, room) for _ in range(count)]
        lengths = [1 if single else min(m, _between(rng, 1, 300)) for m in keys]
        if rng.random() < 0.2:  # a sequence without new tokens
            lengths[rng.randrange(count)] = 0
            lengths[0] = max(lengths[0], 1)
        if kind == "write":
            return {"op": "cache_write", "lengths": _text(lengths), "keys": _text(keys), "room": room, "kv_heads": kv, "head_dim": d, "dtype": dtype}
        case = {"op": "attention" if kind == "tokens" else "cache_attention", "causal": True, "train": False, "room": room, "prefixes": ""}
    else:
        lengths = [_between(rng, 1, 4096) for _ in range(_between(rng, 1, 16))]
        if rng.random() < 0.2:  # a sequence without tokens, and rows that see no key
            lengths.insert(rng.randrange(len(lengths) + 1), 0)
        keys = [n if rng.random() < 0.9 else n // 2 for n in lengths]
        case = {"op": "attention", "causal": rng.random() < 0.8, "train": kind == "train", "room": 0, "prefixes": ""}
    case.update({"heads": kv * rng.choice([1, 1, 2, 3, 4, 8]), "kv_heads": kv, "head_dim": d, "dtype": dtype,
                 "cap": rng.choice([0.0, 20.0, 30.0, 50.0]), "slopes": rng.random() < 0.4,
                 "window": _between(rng, 1, 4096) if rng.random() < 0.4 else 0})
    while (14 if case["train"] else 4) * case["heads"] * sum(n * m for n, m in zip(lengths, keys)) * d > _MOST:
        i = lengths.index(max(lengths))
        lengths[i], keys[i] = lengths[i] // 2, keys[i] // 2 if case["room"] == 0 else keys[i]
    if case["room"] == 0 and case["causal"] and rng.random() < 0.4:
        case["prefixes"] = _text(rng.randint(0, m) for m in keys)
    if case["op"] == "attention" and not (case["cap"] or case["slopes"] or case["window"] or case["prefixes"]):
        case["cap"] = 50.0
    case["lengths"], case["keys"] = _text(lengths), _text(keys)
    return case


def _text(numbers):
    return ",".join(str(x) for x in numbers)


def _numbers(text):
    return [int(x) for x in text.split(",")]


def _seen(case, n, m, prefix, device):
    """Which of m keys the n queries see, and their distances: [n, m] each."""
    place = torch.arange(m - n, m, device=device)[:, None]
    key = torch.arange(m, device=device)[None, :]
    distance = (place - key).abs()
    seen = torch.ones((n, m), dtype=torch.bool, device=device)
    if case["causal"]:
        seen = (key <= place) | (key < prefix)
    if case["window"]:
        seen = seen & (distance < case["window"])
    return seen, distance


def _pairs(case):
    """Pairs of query and key that are seen, and keys that some query sees, over all sequences."""
    pairs = keys = 0
    lengths, counts = _numbers(case["lengths"]), _numbers(case["keys"])
    prefixes = _numbers(case["prefixes"]) if case["prefixes"] else [0] * len(lengths)
    for n, m, prefix in zip(lengths, counts, prefixes):
        if n == 0 or m == 0:
            continue
        place = torch.arange(m - n, m)
        lo, hi = torch.zeros_like(place), torch.full_like(place, m)
        if case["causal"]:
            hi = torch.clamp(place + 1, min=prefix, max=m)
        if case["window"]:
            lo = torch.clamp(place - case["window"] + 1, min=0)
            hi = torch.minimum(hi, place + case["window"])
        count = torch.clamp(hi - lo, min=0)
        pairs += int(count.sum())
        some = count > 0
        if bool(some.any()):
            keys += int(hi[some].max() - lo[some].min())
    return pairs, keys


def work(case):
    size, hk, d = 2 if case["dtype"] == "bf16" else 4, case["kv_heads"], case["head_dim"]
    if case["op"] == "norm_rotary":
        rows = case["tokens"] * (case["heads"] + hk)
        moved = rows * d * size
        return {"bytes": (4 if case["train"] else 2) * moved + case["tokens"] * 4 * len(_numbers(case["sections"])),
                "flops": (20 if case["train"] else 7) * rows * d}
    packed = d // 2 + (d + BLOCK - 1) // BLOCK  # bytes of a cache row: codes and scales
    lengths = _numbers(case["lengths"])
    if case["op"] == "cache_write":
        rows = 2 * sum(lengths) * hk
        return {"bytes": rows * (d * size + packed + d * size), "flops": 4 * rows * d}
    pairs, keys = _pairs(case)
    h = case["heads"]
    q = sum(lengths) * h * d * size
    kv = keys * hk * (packed if case["op"] == "cache_attention" else d * size)
    if not case["train"]:
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * h * d}
    return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * h * d}


# -- a cache row in 4 bits ----------------------------------------------------------------------
#
# 32 channels share a power of two 2^e, held as the byte e + 127; a channel is a sign and 3 bits, which stand for
# 0, 1/2, 1, 3/2, 2, 3, 4 and 6 of it. e is the least with all magnitudes within 7 * 2^e (from -120 to 125); a channel
# is rounded to the nearest, to the even code between two. Two channels make a byte, the first in its lower half.

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # between them; of these an odd code's own neighbours go to the even one


def _blocks(x):
    """[..., D] with zeros behind, as [..., blocks, 32] in 32 bits."""
    x = x.float()
    short = -x.shape[-1] % BLOCK
    if short:
        x = torch.cat([x, x.new_zeros((*x.shape[:-1], short))], -1)
    return x.unflatten(-1, (-1, BLOCK))


def _encode(x):
    """(codes [..., D / 2], scales [..., D / 32]), bytes, of rows [..., D]."""
    x = _blocks(x)
    most = x.abs().amax(-1)
    # 7 * 2^e of every e: the number of those below the maximum is e's place
    e = torch.arange(-120, 126, device=x.device)
    steps = (torch.ldexp(torch.tensor(7.0, dtype=torch.float64, device=x.device), e)).float()
    at = torch.searchsorted(steps, most.contiguous()).clamp(max=len(e) - 1)
    exponent = e[at]
    y = torch.ldexp(x.abs().double(), -exponent[..., None]).float()
    code = torch.zeros(x.shape, dtype=torch.uint8, device=x.device)
    for i, border in enumerate(BORDERS):
        code += (y >= border) if i % 2 else (y > border)
    code = code + 8 * torch.signbit(x).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (exponent + 127).to(torch.uint8)


def _decode(codes, scales, d):
    """The rows' values in 32 bits."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    value = torch.tensor([*MAGNITUDES, *(-v for v in MAGNITUDES)], device=codes.device)[code.int()]
    scale = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    return (value.unflatten(-1, (-1, BLOCK)) * scale[..., None]).flatten(-2)[..., :d]


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

    dt, hk, d = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"]
    state = {"case": case}
    if case["op"] == "norm_rotary":
        h, t, axes, train = case["heads"], case["tokens"], len(_numbers(case["sections"])), case["train"]
        qkv = (2.0 * normal(t, h + 2 * hk, d)).to(dt)  # one projection's rows; q and k are slices of them
        state["inputs"] = [x.detach().requires_grad_(train) for x in (qkv[:, :h], qkv[:, h:h + hk])]
        state["weights"] = [(1.0 + 0.2 * normal(d)).requires_grad_(train) for _ in range(2)] if case["weights"] else [None, None]
        if case["positions"] == "grid":  # fractional coordinates
            state["positions"] = torch.rand((t, axes), generator=g, device="cuda") * 36
        else:
            far = 1_000_000 if case["positions"] == "far" else 16_000
            start = torch.randint(0, far, (t, 1), generator=g, device="cuda")
            state["positions"] = (start + torch.randint(0, 64, (t, axes), generator=g, device="cuda")).to(torch.int32)
        if train:
            state["grads"] = [normal(t, n, d).to(dt) for n in (h, hk)]
        return state
    lengths, keys, room = _numbers(case["lengths"]), _numbers(case["keys"]), case["room"]
    starts = _starts(lengths)
    key_starts = [i * room for i in range(len(keys) + 1)] if room else _starts(keys)
    state.update({"lengths": lengths, "keys": keys, "starts": starts, "key_starts": key_starts})
    state["offsets"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    state["key_offsets"] = state["offsets"] if key_starts == starts else torch.tensor(key_starts, dtype=torch.int32, device="cuda")
    state["key_lengths"] = torch.tensor(keys, dtype=torch.int32, device="cuda") if room else None
    if case["op"].startswith("cache"):
        rows, blocks = key_starts[-1], (d + BLOCK - 1) // BLOCK
        cache = [torch.empty((hk, rows, n), dtype=torch.uint8, device="cuda") for n in (16 * blocks, blocks) * 2]
        for i in (0, 2):
            spread = torch.exp(0.5 * normal(d))  # some channels are larger than others
            for head in range(hk):
                cache[i][head], cache[i + 1][head] = _encode(normal(rows, d) * spread)
        state["cache"] = cache
    if case["op"] == "cache_write":
        state["new"] = [(normal(starts[-1], hk, d) * torch.exp(normal(starts[-1], hk, 1))).to(dt) for _ in range(2)]
        return state
    h, train = case["heads"], case["train"]
    state["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda") / h) if case["slopes"] else None
    prefixes = _numbers(case["prefixes"]) if case["prefixes"] else None
    state["prefixes"] = prefixes or [0] * len(lengths)
    state["prefix_lengths"] = torch.tensor(prefixes, dtype=torch.int32, device="cuda") if prefixes else None
    wide = 4.0 if case["cap"] else 1.5 if not train else 1.0  # capped scores are those that grew
    if case["op"] == "cache_attention":
        state["inputs"] = [(wide * normal(starts[-1], h, d)).to(dt)]
        return state
    if key_starts == starts:  # one projection's rows
        qkv = normal(starts[-1], h + 2 * hk, d)
        qkv[:, :h] *= wide
        qkv = qkv.to(dt)
        inputs = [qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]]
    else:
        inputs = [(wide * normal(starts[-1], h, d)).to(dt), normal(key_starts[-1], hk, d).to(dt), normal(key_starts[-1], hk, d).to(dt)]
    state["inputs"] = [x.detach().requires_grad_(train) for x in inputs]
    if train:
        state["grad"] = normal(starts[-1], h, d).to(dt)
    return state


# -- one pass -----------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if not own:
        return {"norm_rotary": _plain_norm, "attention": _plain_attention, "cache_attention": _plain_attention,
                "cache_write": _plain_write}[case["op"]](state)
    if case["op"] == "norm_rotary":
        (q, k), weights = state["inputs"], state["weights"]
        out = _package().norm_rotary_embed(q, k, *weights, state["positions"], tuple(_numbers(case["sections"])), eps=EPS,
                                           interleaved=case["interleaved"])
        if not case["train"]:
            return {"q": out[0], "k": out[1]}
        leaves = [x for x in (q, k, *weights) if x is not None]
        grads = torch.autograd.grad(out, leaves, state["grads"])
        return {"q": out[0], "k": out[1], **dict(zip(("grad_q", "grad_k", "grad_q_weight", "grad_k_weight"), grads))}
    places = (state["offsets"], state["key_offsets"], state["key_lengths"])
    if case["op"] == "cache_write":
        cache = _package().Cache4(*state["cache"], case["head_dim"])
        _package().cache4_write(cache, *state["new"], *places)
        return dict(zip(("keys", "values"), _package().cache4_read(cache, state["starts"][-1], *places, dtype=DTYPES[case["dtype"]])))
    shape = {"cap": case["cap"] or None, "slopes": state["slopes"], "window": case["window"] or None}
    if case["op"] == "cache_attention":
        cache = _package().Cache4(*state["cache"], case["head_dim"])
        return {"out": _package().cache4_attention(*state["inputs"], cache, *places, **shape)}
    inputs = state["inputs"]
    out = _package().packed_attention(*inputs, *places, causal=case["causal"], prefix_lengths=state["prefix_lengths"], **shape)
    if not case["train"]:
        return {"out": out}
    grads = torch.autograd.grad(out, inputs, state["grad"])
    return {"out": out, "grad_q": grads[0], "grad_k": grads[1], "grad_v": grads[2]}


# -- the plain form -----------------------------------------------------------------------------


def _turn(x, cos, sin, interleaved):
    """Rotates the pairs of x [T, heads, D] by angles [T, n]; channels from 2 n on stay."""
    n = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_norm(state):
    case = state["case"]
    dt, columns = DTYPES[case["dtype"]], []
    for a, s in enumerate(_numbers(case["sections"])):
        e = torch.arange(s, dtype=torch.float64, device="cuda") / s
        columns.append(state["positions"][:, a:a + 1].double() * torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"), -e))
    angle = torch.cat(columns, 1)  # 64 bits: positions are far from 0
    cos, sin = angle.cos().float(), angle.sin().float()
    out = {}
    for name, x, w in zip("qk", state["inputs"], state["weights"]):
        x, w = x.detach().float(), 1.0 if w is None else w.detach()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        out[name] = _turn(x * r * w, cos, sin, case["interleaved"]).to(dt)
    if case["train"]:
        sums = {}
        for name, x, w, g in zip("qk", state["inputs"], state["weights"], state["grads"]):
            x, w = x.detach().float(), None if w is None else w.detach()
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            g = _turn(g.float(), cos, -sin, case["interleaved"])
            u = g if w is None else g * w
            out[f"grad_{name}"] = (r * (u - x * r * r * (u * x).mean(-1, keepdim=True))).to(dt)
            if w is not None:
                sums[f"grad_{name}_weight"] = (g * x * r).double().sum((0, 1)).float()
        out.update(sums)
    return out


def _plain_write(state):
    case = state["case"]
    codes = state["cache"]
    out = {}
    for name, at, x in (("keys", 0, state["new"][0]), ("values", 2, state["new"][1])):
        back = torch.empty(x.shape, dtype=x.dtype, device="cuda")
        for i, n in enumerate(state["lengths"]):
            if n == 0:
                continue
            first = state["key_starts"][i] + state["keys"][i] - n
            rows = slice(state["starts"][i], state["starts"][i] + n)
            code, scale = _encode(x[rows].transpose(0, 1))
            codes[at][:, first:first + n], codes[at + 1][:, first:first + n] = code, scale
            back[rows] = _decode(codes[at][:, first:first + n], codes[at + 1][:, first:first + n], case["head_dim"]).transpose(0, 1).to(x.dtype)
        out[name] = back
    return out


def _keys_values(state, cols):
    """Keys and values of some rows, [key heads, rows, D] in 32 bits."""
    if state["case"]["op"] == "cache_attention":
        c = state["cache"]
        return [_decode(c[i][:, cols], c[i + 1][:, cols], state["case"]["head_dim"]) for i in (0, 2)]
    return [x.detach()[cols].float().transpose(0, 1).contiguous() for x in state["inputs"][1:]]


def _plain_attention(state):
    case = state["case"]
    dt, hk, d, train, cap = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"], case["train"], case["cap"]
    q = state["inputs"][0].detach()
    group = case["heads"] // hk
    scale = d ** -0.5
    out = torch.zeros(q.shape, dtype=dt, device="cuda")
    if train:
        gq, gk, gv = (torch.zeros(x.shape, dtype=dt, device="cuda") for x in state["inputs"])
    for i, (n, m) in enumerate(zip(state["lengths"], state["keys"])):
        if n == 0 or m == 0:
            continue
        rows, cols = slice(state["starts"][i], state["starts"][i] + n), slice(state["key_starts"][i], state["key_starts"][i] + m)
        qi = q[rows].float().view(n, hk, group, d).transpose(0, 1)  # [key heads, tokens, group, D]
        ki, vi = _keys_values(state, cols)
        if train:
            gi = state["grad"][rows].float().view(n, hk, group, d).transpose(0, 1)
            dk, dv = torch.zeros_like(ki), torch.zeros_like(vi)
        all_seen, all_distance = _seen(case, n, m, state["prefixes"][i], "cuda")
        step = max(1, (1 << 28) // (m * hk * group))  # some rows at a time bound the memory
        for t in range(0, n, step):
            e = min(n, t + step)
            qs = qi[:, t:e].reshape(hk, -1, d)
            x = torch.bmm(qs, ki.transpose(1, 2)) * scale
            if cap:
                bent = torch.tanh(x / cap)
                x = cap * bent
            if case["slopes"]:
                distance = all_distance[t:e].float()[None, :, None, :]
                x = (x.view(hk, e - t, group, m) - state["slopes"].view(hk, 1, group, 1) * distance).view(hk, -1, m)
            x = torch.where(all_seen[t:e].repeat_interleave(group, 0), x, -torch.inf)
            top = x.amax(-1, keepdim=True)
            p = torch.exp(x - torch.where(top == -torch.inf, 0.0, top))
            del x
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, 1.0, total)
            o = torch.bmm(p, vi)
            out[rows][t:e] = o.view(hk, e - t, group, d).transpose(0, 1).reshape(e - t, -1, d).to(dt)
            if train:
                gs = gi[:, t:e].reshape(hk, -1, d)
                dv += torch.bmm(p.transpose(1, 2), gs)
                dp = torch.bmm(gs, vi.transpose(1, 2))
                ds = p * (dp - (gs * o).sum(-1, keepdim=True)) * scale
                if cap:
                    ds = ds * (1 - bent * bent)
                gq[rows][t:e] = torch.bmm(ds, ki).view(hk, e - t, group, d).transpose(0, 1).reshape(e - t, -1, d).to(dt)
                dk += torch.bmm(ds.transpose(1, 2), qs)
        if train:
            gk[cols], gv[cols] = dk.transpose(0, 1).to(dt), dv.transpose(0, 1).to(dt)
    if not train:
        return {"out": out}
    return {"out": out, "grad_q": gq, "grad_k": gk, "grad_v": gv}


# -- the same in 64 bits ------------------------------------------------------------------------


def _nearest(x):
    """The values that rows [..., D] have in 4 bits, in 64 bits, by the distance to each of the eight."""
    d = x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -d % BLOCK)).unflatten(-1, (-1, BLOCK))
    most = x.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(most / 7)  # most / 7 = mantissa 2^exponent, mantissa in [1/2, 1)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent)
    exponent = torch.where(most == 0, -120, exponent).clamp(-120, 125)
    unit = torch.ldexp(torch.ones_like(most), exponent)
    levels = [(v, 0.0 if i % 2 == 0 else 1e-9) for i, v in enumerate(MAGNITUDES)]  # even codes win ties
    best = torch.full_like(x, torch.inf)
    value = torch.zeros_like(x)
    for v, handicap in levels:
        away = (x.abs() / unit - v).abs() + handicap
        value = torch.where(away < best, v, value)
        best = torch.minimum(away, best)
    return (torch.sign(x) * value * unit).flatten(-2)[..., :d]


def _held(codes, scales, d):
    """A cache's rows in 64 bits, from the definition of its two bytes."""
    half = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
    bits = half % 8
    # 0 and 1 stand for 0 and 1/2, the others for (1 or 3/2) 2^(bits / 2 - 1)
    size = torch.where(bits < 2, bits.double() / 2, (1 + (bits % 2).double() / 2) * torch.exp2((bits // 2 - 1).double()))
    size = torch.where(half >= 8, -size, size)
    return (size.unflatten(-1, (-1, BLOCK)) * torch.exp2(scales.double() - 127)[..., None]).flatten(-2)[..., :d]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "cache_write":
        return {name: _nearest(x) for name, x in zip(("keys", "values"), state["new"])}
    if case["op"] == "norm_rotary":
        # as complex numbers: a pair times exp(i angle); gradients by differentiation
        sections = _numbers(case["sections"])
        n = sum(sections)
        axis = torch.tensor([a for a, s in enumerate(sections) for _ in range(s)], device="cuda")
        power = torch.tensor([j / s for s in sections for j in range(s)], dtype=torch.float64, device="cuda")
        angle = state["positions"].double()[:, axis] * torch.exp(-power * torch.log(torch.tensor(10000.0, dtype=torch.float64)).item())
        phase = torch.polar(torch.ones_like(angle), angle)[:, None]
        even, odd = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if case["interleaved"] else (slice(0, n), slice(n, 2 * n))
        out, grads = {}, {}
        for i, name in enumerate("qk"):
            x = state["inputs"][i].detach().double().requires_grad_(case["train"])
            w = None if state["weights"][i] is None else state["weights"][i].detach().double().requires_grad_(case["train"])
            y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
            y = y if w is None else y * w
            z = torch.complex(y[..., even], y[..., odd]) * phase
            pairs = torch.stack([z.real, z.imag], -1).flatten(-2) if case["interleaved"] else torch.cat([z.real, z.imag], -1)
            y = torch.cat([pairs, y[..., 2 * n:]], -1)
            out[name] = y.detach()
            if case["train"]:
                got = torch.autograd.grad(y, [x] if w is None else [x, w], state["grads"][i].double())
                out[f"grad_{name}"] = got[0]
                if w is not None:
                    grads[f"grad_{name}_weight"] = got[1]
        order = ("q", "k", "grad_q", "grad_k", "grad_q_weight", "grad_k_weight")
        out.update(grads)
        return {name: out[name] for name in order if name in out}
    q = state["inputs"][0].detach()
    hk, d, train = case["kv_heads"], case["head_dim"], case["train"]
    group = case["heads"] // hk
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in state["inputs"]] if train else []
    for i, (n, m) in enumerate(zip(state["lengths"], state["keys"])):
        if n == 0 or m == 0:
            continue
        a, b = state["starts"][i], state["key_starts"][i]
        seen, distance = _seen(case, n, m, state["prefixes"][i], "cuda")
        blind = ~seen.any(1, keepdim=True)
        for kv in range(hk):
            if case["op"] == "cache_attention":
                c = state["cache"]
                rows = [_held(c[j][kv, b:b + m], c[j + 1][kv, b:b + m], d) for j in (0, 2)]
            else:
                rows = [x.detach()[b:b + m, kv].double() for x in state["inputs"][1:]]
            for head in range(kv * group, kv * group + group):
                at = [x.detach().requires_grad_(train) for x in (q[a:a + n, head].double(), *rows)]
                x = at[0] @ at[1].T / d ** 0.5
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["slopes"]:
                    x = x - state["slopes"][head].double() * distance
                w = torch.softmax(x.masked_fill(~seen, float("-inf")).masked_fill(blind, 0.0), -1).masked_fill(blind, 0.0)
                o = w @ at[2]
                out[a:a + n, head] = o.detach()
                if train:
                    for total, j, s, c, x in zip(grads, (head, kv, kv), (a, b, b), (n, m, m),
                                                 torch.autograd.grad(o, at, state["grad"][a:a + n, head].double())):
                        total[s:s + c, j] += x
    if not train:
        return {"out": out}
    return {"out": out, "grad_q": grads[0], "grad_k": grads[1], "grad_v": grads[2]}
