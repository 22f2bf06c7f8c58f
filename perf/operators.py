"""What is measured of the packed-batch operators: attention of packed queries
(whole prompts, chunks of prompts and single tokens of many sequences at once),
attention of a batch that shares a long prefix, and the pass that norms and
rotates new queries and keys and appends the keys and values to their slots.

Each case names its geometry and the lengths of its sequences; ``run`` makes
one call, in plain torch operations (32 bits, 64 for angles) or, with ``own``,
through the package's entry points.
"""

import functools
import math
import os
import sys

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
DEVICE = "cuda"


# ---- cases -------------------------------------------------------------------


def _attend(name, dtype, heads, kv_heads, dim, q_lens, kv_lens, layout, causal=True):
    return {"name": name, "op": "packed", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "q_lens": q_lens, "kv_lens": kv_lens, "layout": layout, "causal": causal}


def _shared(name, dtype, heads, kv_heads, dim, prefix, q_lens, kv_lens):
    return {"name": name, "op": "shared", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "prefix": prefix, "q_lens": q_lens, "kv_lens": kv_lens}


def _append(name, dtype, heads, kv_heads, dim, rotary, q_lens, kv_lens, interleaved=False, norm=True):
    return {"name": name, "op": "append", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "q_lens": q_lens, "kv_lens": kv_lens, "interleaved": interleaved, "norm": norm}


def _text(lens):
    return ",".join(str(n) for n in lens)


def listed():
    return [
        # one 16K prompt of the benchmark's geometry: the largest compute-bound call
        _attend("prompt_16k", "bf16", 32, 8, 128, "16384", "16384", "packed"),
        # prompts of very different lengths admitted together, odd and ragged ones among them
        _attend("prompts_ragged", "bf16", 32, 8, 128, "1,17,129,777,1024,2049,3001,128", "1,17,129,777,1024,2049,3001,128",
                "packed"),
        # one 1K prompt of the small benchmark model (head dim 64, 8 query heads a group)
        _attend("prompt_1k_d64", "f16", 32, 4, 64, "1024", "1024", "packed"),
        # chunked prefill next to decoding: two chunks of 512 behind long histories, six single tokens
        _attend("chunks_and_tokens", "bf16", 32, 8, 128, "512,1,1,512,1,1,1,1", "8192,5000,77,4611,16000,1,12345,9000",
                "slots"),
        # one decode step of the benchmark batch on exact tiers: 8 sequences at 16K, one query each
        _attend("tokens_16k", "bf16", 32, 8, 128, _text([1] * 8), _text([16384] * 8), "slots"),
        # the smallest call: one token of one short sequence
        _attend("token_short", "f16", 32, 4, 64, "1", "130", "slots"),
        # 64 samples of one 8K prompt, each some hundred tokens on
        _shared("shared_8k_64", "bf16", 32, 8, 128, 8192, _text([1] * 64), _text([1 + (37 * i) % 509 for i in range(64)])),
        # four samples of a 32K document, head dim 64
        _shared("shared_32k_4", "f16", 32, 4, 64, 32768, "1,1,1,1", "40,1,257,128"),
        # a short system prompt in front of two sequences, three drafted tokens each: latency
        _shared("shared_short", "bf16", 32, 8, 128, 200, "3,3", "90,11"),
        # the new tokens of a 16K prompt: norm, rotation, append
        _append("append_16k", "bf16", 32, 8, 128, 128, "16384", "0"),
        # ragged prompts behind histories, pair-wise rotation of half the dims, no norms
        _append("append_ragged_d64", "f16", 32, 4, 64, 32, "1,300,77,1025", "9000,0,12,515", interleaved=True, norm=False),
        # one decode step of 8 sequences: latency
        _append("append_tokens", "bf16", 32, 8, 128, 128, _text([1] * 8), "2000,100,0,1999,1024,777,5,1500"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _geometry(rng):
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    return rng.choice(["bf16", "f16"]), kv_heads * group, kv_heads, rng.choice([64, 96, 128])


def _draw_once(rng):
    dtype, heads, kv_heads, dim = _geometry(rng)
    kind = rng.choice(["prompts", "chunks", "tokens", "shared", "shared", "append", "append"])
    if kind == "prompts":
        lens = [_log_int(rng, 1, 8192) for _ in range(rng.randint(1, 12))]
        return _attend("", dtype, heads, kv_heads, dim, _text(lens), _text(lens), "packed", rng.random() < 0.85)
    if kind == "chunks":
        kv = [_log_int(rng, 1, 16384) for _ in range(rng.randint(1, 12))]
        q = [min(n, rng.choice([1, 1, _log_int(rng, 1, 1024)])) for n in kv]
        return _attend("", dtype, heads, kv_heads, dim, _text(q), _text(kv), rng.choice(["slots", "packed"]))
    if kind == "tokens":
        n = _log_int(rng, 1, 64)
        top = 16384 if n <= 16 else 4096
        return _attend("", dtype, heads, kv_heads, dim, _text([1] * n), _text([_log_int(rng, 1, top) for _ in range(n)]),
                       "slots")
    if kind == "shared":
        n = _log_int(rng, 1, 64)
        kv = [_log_int(rng, 1, 600) for _ in range(n)]
        most = rng.choice([1, 1, 4])
        q = [min(k, rng.randint(1, most)) for k in kv]
        return _shared("", dtype, heads, kv_heads, dim, _log_int(rng, 16, 32768), _text(q), _text(kv))
    n = rng.randint(1, 12)
    lens = [rng.choice([1, _log_int(rng, 1, 2048)]) for _ in range(n)]
    rotary = rng.choice([dim, dim, dim // 2])
    return _append("", dtype, heads, kv_heads, dim, rotary, _text(lens),
                   _text([rng.choice([0, _log_int(rng, 1, 4096)]) for _ in range(n)]), rng.random() < 0.4, rng.random() < 0.7)


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def _scores(case):
    """Score elements the plain form holds at once (padded to the longest sequences)."""
    if case["op"] == "append":
        return 0
    q, kv = _lens(case["q_lens"]), _lens(case["kv_lens"])
    n = case["heads"] * len(q) * max(q) * max(kv)
    return max(n, case["heads"] * sum(q) * case["prefix"]) if case["op"] == "shared" else n


def draw(rng):
    most = max(_cost(c) for c in listed())
    for _ in range(1000):
        case = _draw_once(rng)
        if _cost(case) <= most and _scores(case) <= 4 << 30:
            break
    del case["name"]
    return case


# ---- work ----------------------------------------------------------------------


def _lens(text):
    return [int(n) for n in text.split(",")]


def _visible(q, kv, causal):
    """Query-key pairs of one sequence: query i sits at position kv - q + i."""
    return sum(max(0, min(kv, kv - q + i + 1)) for i in range(q)) if causal else q * kv


def work(case):
    q, kv = _lens(case["q_lens"]), _lens(case["kv_lens"])
    tokens, heads, kv_heads, dim = sum(q), case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        moved = tokens * (heads + 2 * kv_heads) * dim * 2 * 2
        flops = tokens * (heads + kv_heads) * (4 * dim * case["norm"] + 3 * case["rotary"])
        return {"bytes": moved, "flops": flops}
    pairs = sum(_visible(a, b, case["op"] == "shared" or case["causal"]) for a, b in zip(q, kv))
    keys = sum(kv)
    if case["op"] == "shared":
        pairs += tokens * case["prefix"]
        keys += case["prefix"]
    return {"bytes": 2 * (2 * tokens * heads * dim + 2 * keys * kv_heads * dim), "flops": 4 * dim * heads * pairs}


# ---- inputs ----------------------------------------------------------------------


def _int32(values):
    return torch.tensor(values, dtype=torch.int32).to(DEVICE)


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed) * 7919 + 17)
    dtype = DTYPES[case["dtype"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    q_lens, kv_lens = _lens(case["q_lens"]), _lens(case["kv_lens"])
    n, tokens = len(q_lens), sum(q_lens)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)

    def keys(*shape):
        """Keys as caches hold them: the channels of a head have scales of their own."""
        scale = torch.rand((dim,), generator=gen, device=DEVICE) * 1.5 + 0.5
        return normal(*shape, dim).mul_(scale.to(dtype))

    state = {"case": case, "q_lens": q_lens, "kv_lens": kv_lens, "cu_q": _int32(_starts(q_lens)), "scale": dim ** -0.5,
             "sequence": torch.repeat_interleave(torch.arange(n), torch.tensor(q_lens)).to(DEVICE),
             "offset": torch.cat([torch.arange(m) for m in q_lens]).to(DEVICE)}
    if case["op"] == "append":
        # one projection holds a token's queries, keys and values side by side
        qkv = normal(tokens, heads + 2 * kv_heads, dim)
        capacity = -(-max(a + b for a, b in zip(q_lens, kv_lens)) // 16) * 16
        half = case["rotary"] // 2
        state.update(
            query=qkv[:, :heads], key=qkv[:, heads:heads + kv_heads], value=qkv[:, heads + kv_heads:],
            key_slots=torch.zeros((n, kv_heads, capacity, dim), dtype=dtype, device=DEVICE),
            value_slots=torch.zeros((n, kv_heads, capacity, dim), dtype=dtype, device=DEVICE),
            kv_len=_int32(kv_lens),
            inv_freq=(500000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).float().to(DEVICE),
            q_weight=(1 + 0.2 * normal(dim)) if case["norm"] else None,
            k_weight=(1 + 0.2 * normal(dim)) if case["norm"] else None)
        return state
    state["query"] = normal(tokens, heads, dim)
    if case["op"] == "shared" or case["layout"] == "slots":
        # slots as a store holds them, longer than what is valid; stale rows behind the lengths
        capacity = -(-(max(kv_lens) + 1) // 16) * 16
        state.update(key=keys(n, kv_heads, capacity), value=normal(n, kv_heads, capacity, dim), kv_len=_int32(kv_lens))
    else:
        state.update(key=keys(sum(kv_lens), kv_heads), value=normal(sum(kv_lens), kv_heads, dim),
                     cu_k=_int32(_starts(kv_lens)))
    if case["op"] == "shared":
        state.update(prefix_key=keys(kv_heads, case["prefix"]), prefix_value=normal(kv_heads, case["prefix"], dim))
    return state


# ---- one pass ----------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _package():
    """The package's entry points."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "helix-online-kv_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.rotary import norm_rotate_append
    from helix_online_kv.shared_prefix import shared_prefix_attention
    return packed_attention, shared_prefix_attention, norm_rotate_append


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "append":
        return _plain_append(state)
    return _plain_shared(state) if op == "shared" else _plain_packed(state)


def _run_own(s):
    packed_attention, shared_prefix_attention, norm_rotate_append = _package()
    case = s["case"]
    if case["op"] == "append":
        query = norm_rotate_append(s["query"], s["key"], s["value"], s["key_slots"], s["value_slots"], s["cu_q"],
                                   s["kv_len"], s["inv_freq"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS,
                                   interleaved=case["interleaved"])
        return query, s["key_slots"], s["value_slots"]
    if case["op"] == "shared":
        return shared_prefix_attention(s["query"], s["prefix_key"], s["prefix_value"], s["key"], s["value"], s["kv_len"],
                                       cu_seqlens_q=s["cu_q"], scaling=s["scale"])
    if case["layout"] == "slots":
        return packed_attention(s["query"], s["key"], s["value"], s["cu_q"], kv_len=s["kv_len"], scaling=s["scale"],
                                is_causal=case["causal"])
    return packed_attention(s["query"], s["key"], s["value"], s["cu_q"], s["cu_k"], scaling=s["scale"],
                            is_causal=case["causal"])


def _padded(s):
    """The queries [n, kv_heads, group * longest, dim] and the keys and values
    [n, kv_heads, longest, dim] of every sequence, padded, in 32 bits, and which keys a query sees."""
    case = s["case"]
    kv_heads, dim = case["kv_heads"], case["dim"]
    group, most_q, most_kv = case["heads"] // kv_heads, max(s["q_lens"]), max(s["kv_lens"])
    n = len(s["q_lens"])
    at_q, at_kv = torch.arange(most_q, device=DEVICE), torch.arange(most_kv, device=DEVICE)
    start, q_len = s["cu_q"][:-1].long(), s["cu_q"].long().diff()
    query = s["query"][(start[:, None] + at_q).clamp(max=sum(s["q_lens"]) - 1)].float()
    query = query.view(n, most_q, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, group * most_q, dim)
    if "cu_k" in s:
        kv_len = s["cu_k"].long().diff()
        rows = (s["cu_k"][:-1].long()[:, None] + at_kv).clamp(max=sum(s["kv_lens"]) - 1)
        key, value = (s[name][rows].float().transpose(1, 2) for name in ("key", "value"))
    else:
        kv_len = s["kv_len"].long()
        key, value = (s[name][:, :, :most_kv].float() for name in ("key", "value"))
    seen = (at_kv < kv_len[:, None])[:, None, :].expand(n, most_q, most_kv)
    if case["op"] == "shared" or case["causal"]:
        seen = seen & (at_kv <= ((kv_len - q_len)[:, None] + at_q)[:, :, None])
    return query, key, value, seen[:, None, None]


def _unpadded(s, padded):
    """[n, kv_heads, group * longest, dim] -> [tokens, heads, dim]."""
    case = s["case"]
    n, kv_heads, rows, width = padded.shape
    group = case["heads"] // kv_heads
    by_token = padded.view(n, kv_heads, group, rows // group, width).permute(0, 3, 1, 2, 4)
    return by_token[s["sequence"], s["offset"]].reshape(-1, case["heads"], width)


def _plain_packed(s):
    query, key, value, seen = _padded(s)
    n, kv_heads, rows, _ = query.shape
    score = (query * s["scale"]) @ key.transpose(-1, -2)
    masked = score.view(n, kv_heads, -1, seen.shape[-2], seen.shape[-1]).masked_fill_(~seen, float("-inf"))
    top = masked.amax(-1, keepdim=True).clamp_(min=-1e30)
    weight = masked.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = (weight.view(score.shape) @ value) / total.view(n, kv_heads, rows, 1).clamp_(min=1e-30)
    return _unpadded(s, out).to(s["query"].dtype)


def _plain_shared(s):
    query, key, value, seen = _padded(s)
    case = s["case"]
    n, kv_heads, rows, dim = query.shape
    tokens, group = s["query"].shape[0], case["heads"] // kv_heads
    # the shared prefix, once for all queries
    flat = s["query"].float().view(tokens, kv_heads, group, dim).transpose(0, 1).reshape(kv_heads, tokens * group, dim)
    front = ((flat * s["scale"]) @ s["prefix_key"].float().transpose(-1, -2))
    front_top = front.amax(-1, keepdim=True)
    front_weight = front.sub_(front_top).exp_()

    def by_token(x):
        return x.view(kv_heads, tokens, group, -1).transpose(0, 1).reshape(tokens, kv_heads * group, -1)

    front_total, front_sum = by_token(front_weight.sum(-1)), by_token(front_weight @ s["prefix_value"].float())
    front_top = by_token(front_top)
    # each sequence's own rows
    score = (query * s["scale"]) @ key.transpose(-1, -2)
    masked = score.view(n, kv_heads, group, -1, score.shape[-1]).masked_fill(~seen, float("-inf"))
    back_top = masked.amax(-1, keepdim=True).clamp(min=-1e30)
    weight = (masked - back_top).exp().view(score.shape)
    back_total, back_sum = _unpadded(s, weight.sum(-1, keepdim=True)), _unpadded(s, weight @ value)
    back_top = _unpadded(s, back_top.view(n, kv_heads, rows, 1))
    top = torch.maximum(front_top, back_top)
    a, b = (front_top - top).exp(), (back_top - top).exp()
    out = (front_sum * a + back_sum * b) / (front_total * a + back_total * b)
    return out.to(s["query"].dtype)


def _plain_append(s):
    case = s["case"]
    rotary = case["rotary"]
    place = s["kv_len"].long()[s["sequence"]] + s["offset"]
    angle = place.double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
        head, rest = x[..., :rotary], x[..., rotary:]
        if case["interleaved"]:
            a, b = head[..., 0::2], head[..., 1::2]
            head = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = head[..., :rotary // 2], head[..., rotary // 2:]
            head = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((head, rest), -1).to(s["query"].dtype)

    s["key_slots"][s["sequence"], :, place] = turned(s["key"], s["k_weight"])
    s["value_slots"][s["sequence"], :, place] = s["value"]
    return turned(s["query"], s["q_weight"]), s["key_slots"], s["value_slots"]


# ---- 64 bits ----------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group = heads // kv_heads
    out = torch.zeros((sum(s["q_lens"]), heads, dim), dtype=torch.float64, device=DEVICE)
    causal = case["op"] == "shared" or case["causal"]
    q0 = k0 = 0
    for b, (nq, nk) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        for h in range(heads):
            kh = h // group
            if "cu_k" in s:
                k, v = s["key"][k0:k0 + nk, kh], s["value"][k0:k0 + nk, kh]
            else:
                k, v = s["key"][b, kh, :nk], s["value"][b, kh, :nk]
            far = 0
            if case["op"] == "shared":
                far = case["prefix"]
                k, v = torch.cat((s["prefix_key"][kh], k)), torch.cat((s["prefix_value"][kh], v))
            z = s["query"][q0:q0 + nq, h].double() @ k.double().T * s["scale"]
            if causal:
                last = torch.arange(nq, device=DEVICE) + (far + nk - nq)
                z.masked_fill_(torch.arange(far + nk, device=DEVICE)[None] > last[:, None], -math.inf)
            out[q0:q0 + nq, h] = torch.softmax(z, -1).nan_to_num_(0.0) @ v.double()
        q0, k0 = q0 + nq, k0 + nk
    return out


def _exact_append(s):
    case = s["case"]
    half = case["rotary"] // 2
    at = s["key_slots"].double(), s["value_slots"].double()
    place = torch.tensor([n + i for n, m in zip(s["kv_lens"], s["q_lens"]) for i in range(m)], device=DEVICE)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE), place.double()[:, None] * s["inv_freq"].double())

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = x / ((x ** 2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
        if case["interleaved"]:
            first, second = torch.arange(half) * 2, torch.arange(half) * 2 + 1
        else:
            first, second = torch.arange(half), torch.arange(half) + half
        z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
        x[..., first], x[..., second] = z.real, z.imag
        return x

    query, key, t = turned(s["query"].clone(), s["q_weight"]), turned(s["key"].clone(), s["k_weight"]), 0
    for b, (n, m) in enumerate(zip(s["kv_lens"], s["q_lens"])):
        at[0][b, :, n:n + m] = key[t:t + m].transpose(0, 1)
        at[1][b, :, n:n + m] = s["value"][t:t + m].double().transpose(0, 1)
        t += m
    return query, at[0], at[1]
