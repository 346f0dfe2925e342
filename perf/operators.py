"""What a prompt and a shared prefix add to the work that cases.py measures, as measurable cases.

Three kinds, all through the public entry points:

* ``prompt``      ``prompt_attention``: causal attention over whole prompts, packed one behind another; the keys may reach further back than
                  the queries (a chunk of a prompt behind its ``history``) and begin with a prefix that all sequences share.
* ``importance``  ``prompt_importance``: the head-summed probabilities of each sequence's last queries, which seed the importance ring.
* ``prefix``      ``qkv_matmul_hqe_prefix``: one decode step of a batch that shares a dense prefix, each sequence with a tiered cache
                  of its own behind it.

Shapes are those of ``hqekv_b200.configs`` and of the model harness (128 channels a head, 32 query heads over 8 kv heads, or a GPU's share of
them), data is N(0, 1) with a few K channels x10 where the configurations have such outliers.
"""
import math

import torch

own = False

D = 128
F16, BF16 = "float16", "bfloat16"


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _prompt(name, sequences, longest, kv=8, rep=4, dtype=F16, history=0, prefix=0, outliers=False):
    return {"name": name, "kind": "prompt", "sequences": sequences, "longest": longest, "kv_heads": kv, "rep": rep, "dtype": dtype,
            "history": history, "prefix": prefix, "outliers": outliers}


def _importance(name, sequences, longest, rows=20, kv=8, rep=4, dtype=F16, history=0):
    return {"name": name, "kind": "importance", "sequences": sequences, "longest": longest, "kv_heads": kv, "rep": rep, "dtype": dtype,
            "history": history, "rows": rows}


def _prefix(name, batch, prefix, four, two, residual, group=32, kv=8, rep=4):
    return {"name": name, "kind": "prefix", "batch": batch, "prefix": prefix, "four": four, "two": two, "residual": residual, "group": group,
            "kv_heads": kv, "rep": rep}


def listed():
    return [
        # a chat turn of a few words: the smallest call, bound by its launch
        _prompt("prompt-17", 1, 17),
        # one long document, the context of the headline configuration (configuration 1): the largest call
        _prompt("prompt-32k", 1, 32768),
        # eight requests of different lengths taken in one pass
        _prompt("prompt-b8-ragged-5k", 8, 5151, outliers=True),
        # four prompts in bf16, eight query heads per kv head (a GPU's half of the heads)
        _prompt("prompt-b4-4k-bf16-rep8", 4, 4096, kv=4, rep=8, dtype=BF16),
        # a chunk of each of four prompts behind what is cached of them: few rows, many keys
        _prompt("prompt-chunk-b4-16k", 4, 96, history=16257),
        # sixteen short questions behind the same long instructions
        _prompt("prompt-b16-prefix-8k", 16, 411, prefix=8179),
        # ring rows of the long document
        _importance("importance-32k", 1, 32768),
        # ring rows of the eight requests
        _importance("importance-b8-ragged-5k", 8, 5151),
        # a handful of chats behind a short system prompt, nothing quantised yet: the smallest decode step
        _prefix("prefix-b4-2k", 4, 2048, 0, 0, 37),
        # a batch of chats behind long instructions, a thousand tokens of its own in the tiers of each
        _prefix("prefix-b32-32k", 32, 32768, 512, 512, 45),
        # many chats, groups of 64, two query heads per kv head, a prefix of odd length
        _prefix("prefix-b61-8k-g64-rep2", 61, 8179, 192, 448, 109, group=64, kv=4, rep=2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "prompt", "importance", "prefix", "prefix"))
    kv = rng.choice((8, 8, 4, 2, 1))
    rep = rng.choice((4, 4, 4, 8, 2, 1))
    if kind == "prefix":
        batch, prefix, group = _log(rng, 2, 64), _log(rng, 200, 60000), rng.choice((32, 64, 128))
        own_tokens = min(2048, prefix // 4)        # behind a prefix that is long beside what each sequence adds
        four, two = (rng.randint(0, own_tokens // 2) // group * group for _ in range(2))
        return _unnamed(_prefix("", batch, prefix, four, two, rng.randint(1, 130), group, kv, rep))
    sequences = _log(rng, 1, 32)
    dtype = rng.choice((F16, F16, BF16))
    if kind == "importance":
        longest = min(_log(rng, 10, 60000), 200000 // sequences)
        return _unnamed(_importance("", sequences, longest, rng.choice((20, 20, 20, 1, 7, 32)), kv, rep, dtype, rng.choice((0, 0, 300))))
    shape = rng.choice(("plain", "plain", "chunk", "prefix"))
    longest = _log(rng, 1, 2000) if shape != "plain" else _log(rng, 1, 32000)
    history = _log(rng, 100, 20000) if shape == "chunk" else 0
    prefix = _log(rng, 100, 20000) if shape == "prefix" else 0
    case = _prompt("", sequences, longest, kv, rep, dtype, history, prefix, rng.random() < 0.3)
    while work(case)["flops"] > 5e12:
        if case["sequences"] > 1:
            case["sequences"] = (case["sequences"] + 1) // 2
        else:
            case["longest"] = case["longest"] * 3 // 4
    return _unnamed(case)


def _lengths(count, longest):
    """Lengths of ``count`` sequences, spread over 1 ... ``longest``; the first is the longest."""
    return [max(1, round(longest * (1 - (0.6180339887 * i) % 1))) for i in range(count)]


def _shape(case):
    """Query and key lengths of the sequences."""
    q = _lengths(case["sequences"], case["longest"])
    h = _lengths(case["sequences"], case["history"]) if case["history"] else [0] * len(q)
    return q, [a + b for a, b in zip(q, h)]


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _randn(gen, *shape, dtype=torch.float16):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _outliers(gen, k):
    """Four channels of every K head, x10."""
    heads = k.shape[-2]
    channels = torch.rand(heads, D, generator=gen, device="cuda").argsort(-1)[:, :4]
    return k.mul_(torch.ones(heads, D, device="cuda", dtype=k.dtype).scatter_(1, channels, 10.0))


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _tier(gen, batch, heads, n, bits, group):
    """``n`` tokens of a sequence's cache in one tier: K along tokens per channel, V along channels per token; data of about
    N(0, 1), a group's levels spread over what its values span."""
    def codes(*shape):
        return torch.randint(-2 ** 31, 2 ** 31, shape, generator=gen, device="cuda", dtype=torch.int64).int()

    def scales(*shape):
        reach = 2.2 + 0.4 * torch.rand(*shape, generator=gen, device="cuda")
        return (2 * reach / (2 ** bits - 1)).half(), (-reach).half()

    k, v = codes(batch, heads, D, n * bits // 32), codes(batch, heads, n, D * bits // 32)
    return k, scales(batch, heads, D, n // group), v, scales(batch, heads, n, D // group)


def _places(gen, n, group):
    """Blocks of ``group`` tokens in some order: the logical position of every token of a side."""
    blocks = torch.randperm(n // group, generator=gen, device="cuda")
    return (blocks.unsqueeze(1) * group + torch.arange(group, device="cuda")).reshape(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kv, nh = case["kv_heads"], case["kv_heads"] * case["rep"]
    state = {"case": case}
    if case["kind"] == "prefix":
        B, P, g = case["batch"], case["prefix"], case["group"]
        state["prefix"] = (_randn(gen, P, kv, D), _randn(gen, P, kv, D))
        cache = [None] * 42
        k_at, v_at = _places(gen, case["four"] + case["two"], g), _places(gen, case["four"] + case["two"], g)
        begin = 0
        for bits, slot, n in ((4, 12, case["four"]), (2, 20, case["two"])):
            if n:
                k, (ks, kz), v, (vs, vz) = _tier(gen, B, kv, n, bits, g)
                cache[slot:slot + 8] = [k, k_at[begin:begin + n].clone(), ks, kz, v, v_at[begin:begin + n].clone(), vs, vz]
                begin += n
        cache[39], cache[40] = _randn(gen, B, kv, case["residual"], D), _randn(gen, B, kv, case["residual"], D)
        cache[41] = begin + case["residual"]
        state["cache"], state["q"] = tuple(cache), _randn(gen, B, nh, 1, D)
        return state
    dtype = getattr(torch, case["dtype"])
    lq, lk = _shape(case)
    state["lengths"] = lq, lk
    state["q_starts"], state["k_starts"] = _starts(lq), _starts(lk)
    state["q"] = _randn(gen, sum(lq), nh, D, dtype=dtype)
    state["k"] = _randn(gen, sum(lk), kv, D, dtype=dtype)
    if case["kind"] == "importance":
        # the log-sum-exp that the prompt's attention has left; only the last queries' is read
        state["lse"] = torch.zeros(nh, sum(lq), device="cuda")
        tq, tk = 0, 0
        for n, m in zip(lq, lk):
            t = min(case["rows"], n)
            s = _scores(state["q"][tq + n - t:tq + n], state["k"][tk:tk + m])
            state["lse"][:, tq + n - t:tq + n] = _hide(s, t, m).logsumexp(-1).view(nh, t)
            tq, tk = tq + n, tk + m
        return state
    if case["outliers"]:
        _outliers(gen, state["k"])
    state["v"] = _randn(gen, sum(lk), kv, D, dtype=dtype)
    if case["prefix"]:
        state["prefix"] = (_randn(gen, case["prefix"], kv, D, dtype=dtype), _randn(gen, case["prefix"], kv, D, dtype=dtype))
    return state


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------
def _scores(q, k):
    """q [n, nh, D], k [m, kv, D] -> [kv, rep, n, m] in 32 bits, scaled."""
    n, nh, m, kv = q.shape[0], q.shape[1], k.shape[0], k.shape[1]
    rows = q.float().view(n, kv, nh // kv, D).permute(1, 2, 0, 3).reshape(kv, -1, D)
    return (torch.matmul(rows, k.float().permute(1, 2, 0)) * D ** -0.5).view(kv, nh // kv, n, m)


def _hide(s, n, visible):
    """The last of the n queries sees the first ``visible`` keys, the one before it one less, ..."""
    i = torch.arange(n, device=s.device).unsqueeze(1)
    return s.masked_fill_(torch.arange(s.shape[-1], device=s.device) > i + (visible - n), -math.inf)


def _plain_sequence(q, k, v, out, lse, history):
    """Attention of one sequence's queries, a block of rows at a time, over the keys that the block sees."""
    n, nh, kv = q.shape[0], q.shape[1], k.shape[1]
    block = max(1, min(n, int(5e8 / (nh * k.shape[0]))))
    for i in range(0, n, block):
        e = min(i + block, n)
        seen = history + e
        s = _hide(_scores(q[i:e], k[:seen]), e - i, seen)
        top = s.amax(-1, keepdim=True)
        p = s.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(kv, -1, seen), v[:seen].float().transpose(0, 1)).view(kv, nh // kv, e - i, D) / total
        out[i:e] = o.permute(2, 0, 1, 3).reshape(e - i, nh, D)
        lse[:, i:e] = (top + total.log()).view(nh, e - i)


def _plain_prompt(state):
    q, k, v = state["q"], state["k"], state["v"]
    out, lse = torch.empty_like(q), torch.empty(q.shape[1], q.shape[0], device="cuda")
    tq, tk = 0, 0
    for n, m in zip(*state["lengths"]):
        ks, vs = k[tk:tk + m], v[tk:tk + m]
        if "prefix" in state:
            ks, vs = torch.cat((state["prefix"][0], ks)), torch.cat((state["prefix"][1], vs))
        _plain_sequence(q[tq:tq + n], ks, vs, out[tq:tq + n], lse[:, tq:tq + n], ks.shape[0] - n)
        tq, tk = tq + n, tk + m
    return out, lse


def _plain_importance(state):
    q, k, rows = state["q"], state["k"], state["case"]["rows"]
    out = torch.zeros(rows, k.shape[0], dtype=torch.float16, device="cuda")
    tq, tk = 0, 0
    for n, m in zip(*state["lengths"]):
        t = min(rows, n)
        s = _scores(q[tq + n - t:tq + n], k[tk:tk + m])
        s -= state["lse"][:, tq + n - t:tq + n].reshape(s.shape[0], s.shape[1], t, 1)
        out[:t, tk:tk + m] = _hide(s, t, m).exp_().sum((0, 1))
        tq, tk = tq + n, tk + m
    return out


def _values(words, scale, zero, bits, group):
    """Codes along the last axis, 32 / bits to a word, as what they stand for: code * scale + zero of their group."""
    code = (words.unsqueeze(-1) >> torch.arange(0, 32, bits, device=words.device)) & (2 ** bits - 1)
    return code.flatten(-2).float() * scale.float().repeat_interleave(group, -1) + zero.float().repeat_interleave(group, -1)


def _dense(cache, group):
    """A sequence's own K and V [B, kv, L, D] in 32 bits, tokens at their logical positions."""
    new_k, new_v = cache[39], cache[40]
    B, H, _, _ = new_k.shape
    k, v = (torch.empty(B, H, cache[41], D, device="cuda") for _ in range(2))
    k[:, :, cache[41] - new_k.shape[2]:], v[:, :, cache[41] - new_k.shape[2]:] = new_k, new_v
    for bits, slot in ((4, 12), (2, 20)):
        if cache[slot] is not None:
            kc, k_at, ks, kz, vc, v_at, vs, vz = cache[slot:slot + 8]
            k[:, :, k_at] = _values(kc, ks, kz, bits, group).transpose(2, 3)
            v[:, :, v_at] = _values(vc, vs, vz, bits, group)
    return k, v


def _plain_prefix(state):
    q, (pk, pv), g = state["q"], state["prefix"], state["case"]["group"]
    k, v = _dense(state["cache"], g)
    B, kv, L, _ = k.shape
    rows = q.float().view(B, kv, -1, D)
    before = torch.matmul(rows.transpose(0, 1).reshape(kv, -1, D), pk.float().permute(1, 2, 0)) * D ** -0.5
    s = torch.matmul(rows, k.transpose(2, 3)) * D ** -0.5
    before = before.view(kv, B, -1, pk.shape[0]).transpose(0, 1)
    top = torch.maximum(before.amax(-1, keepdim=True), s.amax(-1, keepdim=True))
    before, s = (before - top).exp_(), (s - top).exp_()
    total = before.sum(-1, keepdim=True) + s.sum(-1, keepdim=True)
    o = torch.matmul(before.transpose(0, 1).reshape(kv, -1, pk.shape[0]), pv.float().transpose(0, 1))
    o = o.view(kv, B, -1, D).transpose(0, 1) + torch.matmul(s, v)
    return (s / total).reshape(B, -1, 1, L).half(), (o / total).reshape(q.shape).half()


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        if kind == "prefix":
            from hqekv_b200.quant.hqe_matmul import qkv_matmul_hqe_prefix
            g = state["case"]["group"]
            return qkv_matmul_hqe_prefix(state["q"], state["cache"], state["prefix"], D, "uniform_group", g, g)
        from hqekv_b200.prompt import prompt_attention, prompt_importance
        if kind == "importance":
            return prompt_importance(state["q"], state["k"], state["lse"], state["q_starts"], state["k_starts"], rows=state["case"]["rows"])
        return prompt_attention(state["q"], state["k"], state["v"], state["q_starts"], state["k_starts"], prefix=state.get("prefix"))
    if kind == "prefix":
        return _plain_prefix(state)
    return _plain_importance(state) if kind == "importance" else _plain_prompt(state)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    kv, nh = case["kv_heads"], case["kv_heads"] * case["rep"]
    if case["kind"] == "prefix":
        B, P, g = case["batch"], case["prefix"], case["group"]
        L = case["four"] + case["two"] + case["residual"]
        cached = 2 * (case["four"] * (D / 2 + 4 * D / g) + case["two"] * (D / 4 + 4 * D / g) + case["residual"] * 2 * D)   # K and V of a kv head
        return {"bytes": 4.0 * P * kv * D + B * kv * cached + 16 * (L - case["residual"]) + B * nh * (4 * D + 2 * L),
                "flops": 4.0 * D * B * nh * (P + L)}
    lq, lk = _shape(case)
    tq, tk = sum(lq), sum(lk)
    if case["kind"] == "importance":
        rows = sum(min(case["rows"], n) for n in lq)
        pairs = sum(t * m - t * (t - 1) / 2 for t, m in ((min(case["rows"], n), m) for n, m in zip(lq, lk)))
        return {"bytes": 2.0 * tk * kv * D + rows * nh * (2 * D + 4) + 2 * case["rows"] * tk, "flops": 2.0 * D * nh * pairs}
    pairs = sum(n * (m + case["prefix"]) - n * (n - 1) / 2 for n, m in zip(lq, lk))
    return {"bytes": 4.0 * tq * nh * D + 4 * tq * nh + 4.0 * (tk + case["prefix"]) * kv * D, "flops": 4.0 * D * nh * pairs}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_rows(q, k, v, first):
    """softmax(q k^T / sqrt(D)) v and the log of its denominator; q [n, D] are queries ``first``, ``first`` + 1, ... of the sequence,
    each of which sees the keys up to its own number."""
    z = torch.einsum("nd,md->nm", q, k) / math.sqrt(D)
    late = torch.ones_like(z, dtype=torch.bool).triu(first + 1)
    z[late] = -math.inf
    lse = torch.logsumexp(z, 1)
    return torch.einsum("nm,md->nd", torch.exp(z - lse[:, None]), v), lse


def exact(case, seed):
    state = prepare(case, seed)
    rep = case["rep"]
    if case["kind"] == "prefix":
        return _exact_prefix(state)
    q, k = state["q"].double(), state["k"].double()
    bounds = list(zip(state["q_starts"].tolist(), state["q_starts"].tolist()[1:], state["k_starts"].tolist(), state["k_starts"].tolist()[1:]))
    if case["kind"] == "importance":
        out = torch.zeros(case["rows"], k.shape[0], dtype=torch.float64, device="cuda")
        for q0, q1, k0, k1 in bounds:
            for r, i in enumerate(range(max(q0, q1 - case["rows"]), q1)):
                seen = k1 - (q1 - 1 - i)
                z = torch.einsum("hd,mhd->hm", q[i], k[k0:seen].repeat_interleave(rep, 1)) / math.sqrt(D)
                out[r, k0:seen] = torch.exp(z - state["lse"][:, i, None].double()).sum(0)
        return out
    v, out = state["v"].double(), torch.empty_like(q)
    lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float64, device="cuda")
    for q0, q1, k0, k1 in bounds:
        for h in range(q.shape[1]):
            kh, vh = k[k0:k1, h // rep], v[k0:k1, h // rep]
            if "prefix" in state:
                kh = torch.cat((state["prefix"][0][:, h // rep].double(), kh))
                vh = torch.cat((state["prefix"][1][:, h // rep].double(), vh))
            step = 4096
            for i in range(q0, q1, step):
                e = min(i + step, q1)
                first = kh.shape[0] - (q1 - i)
                out[i:e, h], lse[h, i:e] = _exact_rows(q[i:e, h], kh[:first + e - i], vh[:first + e - i], first)
    return out, lse


def _exact_prefix(state):
    """A sequence and kv head at a time, every word of the cache taken apart for itself."""
    cache, q, case = state["cache"], state["q"].double(), state["case"]
    g, rep, L = case["group"], case["rep"], cache[41]
    weights = torch.empty(q.shape[0], q.shape[1], 1, L, dtype=torch.float64, device="cuda")
    out = torch.empty_like(q)

    def spread(words, levels, lowest, bits):
        parts = [torch.bitwise_and(torch.bitwise_right_shift(words, s), 2 ** bits - 1) for s in range(0, 32, bits)]
        code = torch.stack(parts, -1).reshape(words.shape[0], words.shape[1], -1, g).double()
        return (code * levels.double()[..., None] + lowest.double()[..., None]).flatten(2)

    for b in range(q.shape[0]):
        k = torch.empty(case["kv_heads"], L, D, dtype=torch.float64, device="cuda")
        v = torch.empty_like(k)
        for bits, s in ((4, 12), (2, 20)):
            if cache[s] is not None:
                k[:, cache[s + 1]] = spread(cache[s][b], cache[s + 2][b], cache[s + 3][b], bits).mT
                v[:, cache[s + 5]] = spread(cache[s + 4][b], cache[s + 6][b], cache[s + 7][b], bits)
        k[:, L - case["residual"]:], v[:, L - case["residual"]:] = cache[39][b], cache[40][b]
        for h in range(case["kv_heads"]):
            keys = torch.cat((state["prefix"][0][:, h].double(), k[h]))
            values = torch.cat((state["prefix"][1][:, h].double(), v[h]))
            p = torch.softmax(q[b, h * rep:(h + 1) * rep, 0] @ keys.T / math.sqrt(D), -1)
            out[b, h * rep:(h + 1) * rep, 0] = p @ values
            weights[b, h * rep:(h + 1) * rep, 0] = p[:, case["prefix"]:]
    return weights, out
