"""Operators of a server whose cache is long, timed by themselves:

* rows of keys and values rotated, rounded to eight bits with a scale per row on their way into a paged cache, and read back;
* attention of single tokens over such a cache;
* attention of prompts over such a cache;
* attention of single tokens whose sequences hold their first positions in common (the same pages), over a cache in eight bits
  or in bfloat16.

A case is a set of sizes; lengths follow from the case alone, pages, values and their order from the seed.  With `own` false all
run in elementary torch operations, sums in 32 bits; with `own` true they are the calls that a user makes of
`inferllm_b200.kernels.ops`.

A row x of eight bits: s = max |x| / 127, u = 128 + round(x / s), and it stands for (u - 128) s.
"""
import math

import torch

own = False

# query heads, key/value heads, head size: the benchmark's models, the tests' small ones and groups of odd sizes
HEADS = ((32, 8, 128), (32, 32, 128), (40, 40, 128), (4, 2, 64), (14, 2, 64), (12, 4, 128), (16, 1, 128), (24, 8, 64))
PAGE = 64
THETA = 10000.0


def listed():
    def cache(name, seqs, tokens, past, heads):
        return dict(name=name, kind="cache", seqs=seqs, tokens=tokens, past=past, heads=heads[0], kv_heads=heads[1], head_dim=heads[2])

    def decode(name, seqs, longest, heads, window=0):
        return dict(name=name, kind="decode", seqs=seqs, longest=longest, heads=heads[0], kv_heads=heads[1], head_dim=heads[2], window=window)

    def prompts(name, seqs, tokens, past, heads, window=0):
        return dict(name=name, kind="prompts", seqs=seqs, tokens=tokens, past=past, heads=heads[0], kv_heads=heads[1], head_dim=heads[2], window=window)

    def shared(name, bits, seqs, groups, prefix, rest, heads):
        return dict(name=name, kind="shared", bits=bits, seqs=seqs, groups=groups, prefix=prefix, rest=rest, heads=heads[0], kv_heads=heads[1],
                    head_dim=heads[2])

    return [
        # eight answers, one token each, on their way into the cache of a 7B layer
        cache("cache-8", 8, 8, 4000, (32, 32, 128)),
        # sixteen unequal prompts in one step at the 8B size
        cache("cache-prompts", 16, 4096, 100, (32, 8, 128)),
        # one user's answer behind an ordinary conversation
        decode("decode-1", 1, 1777, (32, 8, 128)),
        # a small model's two answers, odd group of heads
        decode("decode-small", 2, 333, (14, 2, 64)),
        # the benchmark's batch at the end of its context, 7B
        decode("decode-8", 8, 4096, (32, 32, 128)),
        # a full server, unequal conversations, 8B
        decode("decode-64", 64, 8192, (32, 8, 128)),
        # one prompt of a chat turn
        prompts("prompt-200", 1, 200, 0, (32, 8, 128)),
        # sixteen unequal questions behind conversations that are there already
        prompts("prompts-16", 16, 2048, 1500, (32, 8, 128)),
        # a long document's second half, 7B
        prompts("prompt-long", 1, 4096, 2001, (32, 32, 128)),
        # eight questions about one document, 7B, the cache as the model makes it
        shared("shared-8", 16, 8, 1, 2048, 150, (32, 32, 128)),
        # three system prompts of unequal length, some sequences with none
        shared("shared-groups", 16, 40, 3, 4096, 500, (32, 8, 128)),
        # a full server behind one long system prompt, in eight bits
        shared("shared-64", 8, 64, 1, 8192, 700, (32, 8, 128)),
    ]


LARGEST_KEYS = 64 * 8192 * 8 * 128             # of decode-64: key elements
LARGEST_PAIRS = 4096 * (2001 + 2048) * 32 * 128       # of prompt-long


def draw(rng):
    def between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("cache", "decode", "decode", "prompts", "prompts", "shared", "shared"))
    nh, nkv, d = rng.choice(HEADS)
    sizes = dict(heads=nh, kv_heads=nkv, head_dim=d)
    if kind == "cache":
        tokens = min(between(1, 8192), 4096 * 6144 // ((nh + 2 * nkv) * d))
        return dict(kind=kind, seqs=min(tokens, between(1, 64)), tokens=tokens, past=between(1, 4000), **sizes)
    if kind == "decode":
        seqs = between(1, 96)
        longest = between(1, max(1, min(32768, LARGEST_KEYS // (seqs * nkv * d))))
        return dict(kind=kind, seqs=seqs, longest=longest, window=rng.choice((0, 0, 0, 100, 1000)), **sizes)
    if kind == "prompts":
        seqs, tokens = between(1, 24), between(2, 4096)
        seqs = min(seqs, tokens)
        most = LARGEST_PAIRS * 2 // 3 // (tokens * nh * d)       # positions before the prompts, on an average
        past = rng.choice((0, between(1, max(1, min(8000, most - tokens // seqs)))))
        return dict(kind=kind, seqs=seqs, tokens=tokens, past=past, window=rng.choice((0, 0, 0, 100, 1000)), **sizes)
    seqs = between(2, 96)
    rest = between(1, min(1500, LARGEST_KEYS // (seqs * nkv * d) // 2))
    prefix = max(1, between(64, max(64, min(16384, LARGEST_KEYS // (seqs * nkv * d) - rest))) // PAGE) * PAGE
    return dict(kind=kind, bits=rng.choice((8, 16)), seqs=seqs, groups=rng.choice((1, 1, 2, 4)), prefix=prefix, rest=rest, **sizes)


# ---------------------------------------------------------------- what a case says


def spread(n, total):
    """n unequal whole numbers, each at least 1, with the sum `total`."""
    out, left = [], total
    for i in range(n):
        share = left // (n - i)
        out.append(left if i == n - 1 else max(1, min(left - (n - 1 - i), int(share * (0.5 + (i * 0.6180339887498949) % 1.0)))))
        left -= out[-1]
    return out


def uneven(n, most):
    """n unequal lengths of at most `most`, the first of them the longest."""
    return [max(1, int(most * (1.0 - 0.8 * ((i * 0.6180339887498949) % 1.0)))) for i in range(n)]


def layout(case):
    """Per sequence the tokens of the step, the positions after it, its group (-1: none) and the positions it has in common with it."""
    n = case["seqs"]
    if case["kind"] in ("cache", "prompts"):
        new = spread(n, case["tokens"])
        past = uneven(n, case["past"]) if case["past"] else [0] * n
        return new, [p + q for p, q in zip(past, new)], [-1] * n, [0] * n
    if case["kind"] == "decode":
        return [1] * n, uneven(n, case["longest"]), [-1] * n, [0] * n
    # one group: all sequences; several: they take turns with sequences that have no prefix in common with any
    g = case["groups"]
    group = [0] * n if g == 1 else [i % (g + 1) if i % (g + 1) < g else -1 for i in range(n)]
    common = [max(PAGE, case["prefix"] // (a + 1) // PAGE * PAGE) if a >= 0 else 0 for a in group]
    return [1] * n, [c + r for c, r in zip(common, uneven(n, case["rest"]))], group, common


def visible(case):
    """(query, key) pairs of one query head, over the whole step."""
    new, lens, _, _ = layout(case)
    w, pairs = case.get("window", 0), 0
    for q, n in zip(new, lens):
        first = n - q + 1                  # keys of the first token of the step
        if w and w < first:
            pairs += q * w
        elif w and w < n:
            pairs += (first + w) * (w - first + 1) // 2 + (n - w) * w
        else:
            pairs += (first + n) * q // 2
    return pairs


def work(case):
    nh, nkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    new, lens, group, common = layout(case)
    T = sum(new)
    if case["kind"] == "cache":
        # the projection once; queries, rows of eight bits with their scales, and what they stand for
        return dict(bytes=2 * T * (nh + 2 * nkv) * d + 2 * T * nh * d + 2 * T * nkv * (d + 4) + 2 * T * nkv * 2 * d, flops=T * d * (6 * nh + 12 * nkv))
    if case["kind"] == "shared":
        held = sum({a: c for a, c in zip(group, common) if a >= 0}.values()) + sum(n - c for n, c in zip(lens, common))
    else:
        w = case["window"]
        held = sum(min(n, w + q - 1) if w else n for q, n in zip(new, lens))
    row = 2 * d if case.get("bits", 8) == 16 else d + 4
    return dict(bytes=2 * held * nkv * row + 2 * 2 * T * nh * d, flops=4 * visible(case) * nh * d)


# ---------------------------------------------------------------- inputs


def to_eight_bits(x):
    """Rows of the last axis -> (u, s)."""
    s = x.abs().amax(-1) / 127.0
    u = torch.round(x / torch.where(s > 0, s, torch.ones_like(s))[..., None]) + 128.0
    return u.to(torch.uint8), s


def rows_of(u, s):
    return (u.to(s.dtype) - 128.0) * s[..., None]


def inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    nh, nkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    new, lens, group, common = layout(case)
    T, n = sum(new), len(lens)
    width = -(-max(lens) // PAGE)
    shared_pages = {a: c // PAGE for a, c in zip(group, common) if a >= 0}
    own_pages = [-(-l // PAGE) - c // PAGE for l, c in zip(lens, common)]
    pages = sum(shared_pages.values()) + sum(own_pages) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table, at = torch.full((n, width), -1, dtype=torch.int32, device="cuda"), 0
    of_group = {}
    for a, c in shared_pages.items():
        of_group[a] = order[at:at + c]
        at += c
    for i in range(n):
        c = common[i] // PAGE
        if c:
            table[i, :c] = of_group[group[i]]
        table[i, c:c + own_pages[i]] = order[at:at + own_pages[i]]
        at += own_pages[i]
    seq = torch.tensor([i for i, q in enumerate(new) for _ in range(q)], dtype=torch.int32, device="cuda")
    pos = torch.tensor([l - q + j for q, l in zip(new, lens) for j in range(q)], dtype=torch.int32, device="cuda")
    cu = [0]
    for q in new:
        cu.append(cu[-1] + q)
    given = dict(table=table, seq=seq, pos=pos, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"),
                 lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), pages=pages)
    # a few channels of the keys stand out, as they do in trained models
    loud = torch.ones((nkv, d), device="cuda")
    loud.scatter_(1, torch.randint(0, d, (nkv, 3), generator=g, device="cuda"), 5.0)
    if case["kind"] == "cache":
        # rows before the rotation, as the projection leaves them
        qkv = torch.randn((T, (nh + 2 * nkv) * d), generator=g, device="cuda")
        qkv[:, nh * d:(nh + nkv) * d] *= loud.reshape(-1)
        angle = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None] * THETA ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        given.update(qkv=qkv.bfloat16(), cos_sin=torch.stack([angle.cos(), angle.sin()], -1).float())
        return given
    k = torch.randn((pages, nkv, PAGE, d), generator=g, device="cuda") * loud[:, None]
    v = torch.randn((pages, nkv, PAGE, d), generator=g, device="cuda")
    # queries with scores of some spread: part of the keys carries the weight
    given["q"] = (torch.randn((T, nh * d), generator=g, device="cuda") * 1.5).bfloat16()
    if case.get("bits", 8) == 16:
        given.update(k=k.bfloat16(), v=v.bfloat16())
    else:
        (ku, ks), (vu, vs) = to_eight_bits(k), to_eight_bits(v)
        given.update(k=ku, v=vu, k_scale=ks, v_scale=vs)
    return given


def prepare(case, seed):
    state = dict(inputs(case, seed), case=case, own=own)
    new, lens, group, common = layout(case)
    state.update(longest=max(lens), max_q=max(new))
    if not own:
        return state
    from inferllm_b200.kernels import ops
    if case["kind"] == "cache":
        state.update(cache=ops.CacheInt8.empty(state["pages"], case["kv_heads"], PAGE, case["head_dim"]), err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    elif "k_scale" in state:
        state["cache"] = ops.CacheInt8(state["k"], state["v"], state["k_scale"], state["v_scale"])
    else:
        state["cache"] = (state["k"], state["v"])
    if case["kind"] == "shared":
        members = {}
        for t, a in enumerate(group):
            members.setdefault(a, []).append(t)
        state["plan"] = ops.SharedPrefixes([(common[m[0]], m) for a, m in members.items() if a >= 0], lens, case["heads"] // case["kv_heads"])
    return state


# ---------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    nh, nkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    if state["own"]:
        from inferllm_b200.kernels import ops
        if case["kind"] == "cache":
            q = ops.kv_write_int8(state["qkv"], state["cos_sin"], d, state["pos"], state["seq"], state["table"], state["cache"], nh, state["err"])
            return (q,) + ops.kv_read_int8(state["cache"], state["pos"], state["seq"], state["table"])
        if case["kind"] == "decode":
            return ops.attention_decode_int8(state["q"], state["cache"], state["table"], state["pos"], state["seq"], nh, case["window"], d ** -0.5,
                                             state["longest"])
        if case["kind"] == "prompts":
            return ops.attention_prompts_int8(state["q"], state["cache"], state["table"], state["cu"], state["lens"], state["max_q"], nh, case["window"],
                                              d ** -0.5)
        return ops.attention_decode_shared(state["q"], state["cache"], state["table"], state["pos"], state["seq"], state["plan"], nh, d ** -0.5,
                                           state["longest"])
    if case["kind"] == "cache":
        return plain_cache(state, nh, nkv, d)
    return plain_attention(state, nh, nkv, d, case.get("window", 0))


def plain_cache(state, nh, nkv, d):
    T = state["qkv"].shape[0]
    x = state["qkv"].float().reshape(T, nh + 2 * nkv, d)
    at = state["cos_sin"][state["pos"].long()][:, None]
    cos, sin, lo, hi = at[..., 0], at[..., 1], x[:, :nh + nkv, :d // 2], x[:, :nh + nkv, d // 2:]
    turned = torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1)
    rows = torch.cat([turned[:, nh:], x[:, nh + nkv:]], 1)
    back = rows_of(*to_eight_bits(rows)).bfloat16()
    return turned[:, :nh].reshape(T, nh * d).bfloat16(), back[:, :nkv], back[:, nkv:]


def plain_attention(state, nh, nkv, d, window):
    # sequences side by side, padded to the longest: [n, longest, kv heads, d]
    n, longest, most = state["table"].shape[0], state["longest"], state["max_q"]
    place = torch.arange(longest, device="cuda")
    page = state["table"].long().clamp_min(0)[:, place // PAGE]

    def gather(x):
        return x[page, :, place % PAGE]

    if "k_scale" in state:
        k, v = rows_of(gather(state["k"]), gather(state["k_scale"])), rows_of(gather(state["v"]), gather(state["v_scale"]))
    else:
        k, v = gather(state["k"]).float(), gather(state["v"]).float()
    # queries side by side: [n, most, heads, d]
    seq, pos = state["seq"].long(), state["pos"].long()
    nth = pos - (state["lens"].long() - (state["cu"][1:] - state["cu"][:-1]).long())[seq]
    q = torch.zeros((n, most, nh, d), device="cuda")
    q[seq, nth] = state["q"].float().reshape(-1, nh, d)
    at = torch.zeros((n, most), dtype=torch.long, device="cuda")
    at[seq, nth] = pos
    s = torch.matmul(q.reshape(n, most, nkv, nh // nkv, d).permute(0, 2, 3, 1, 4), k.permute(0, 2, 3, 1)[:, :, None]) * d ** -0.5
    hidden = place > at[..., None]
    if window:
        hidden = hidden | (place <= at[..., None] - window)
    s = s.masked_fill_(hidden[:, None, None], float("-inf"))
    s = torch.exp(s.sub_(s.amax(-1, keepdim=True)))
    o = torch.matmul(s, v.permute(0, 2, 1, 3)[:, :, None]) / s.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(n, most, nh * d)[seq, nth].bfloat16()


# ---------------------------------------------------------------- the same in 64 bits, from the definitions


def exact(case, seed):
    given = inputs(case, seed)
    nh, nkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    new, lens, _, _ = layout(case)
    if case["kind"] == "cache":
        return exact_cache(given, nh, nkv, d)
    out, at, w, G = [], 0, case.get("window", 0), nh // nkv
    for i, (q_len, n) in enumerate(zip(new, lens)):
        pages = given["table"][i, :-(-n // PAGE)].long()

        def sequence(name):
            x = given[name][pages].double()
            if name + "_scale" in given:
                x = (x - 128.0) * given[name + "_scale"][pages].double()[..., None]
            return x.transpose(1, 2).reshape(-1, nkv, d)[:n]

        k, v = sequence("k"), sequence("v")
        q = given["q"][at:at + q_len].double().reshape(q_len, nh, d)
        at += q_len
        heads = []
        for h in range(nh):
            s = q[:, h] @ k[:, h // G].t() / math.sqrt(d)
            p, j = torch.arange(n - q_len, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
            s[(j > p) | ((j <= p - w) if w else (j > p))] = -math.inf
            heads.append(torch.softmax(s, -1) @ v[:, h // G])
        out.append(torch.stack(heads, 1).reshape(q_len, nh * d))
    return torch.cat(out)


def exact_cache(given, nh, nkv, d):
    x = given["qkv"].double().reshape(-1, nh + 2 * nkv, d)
    angle = given["pos"].double()[:, None] * torch.exp(torch.arange(d // 2, device="cuda", dtype=torch.float64) * (-2.0 * math.log(THETA) / d))
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    z = torch.complex(x[:, :nh + nkv, :d // 2], x[:, :nh + nkv, d // 2:]) * turn
    turned = torch.cat([z.real, z.imag], -1)

    def stands_for(rows):
        step = rows.abs().max(-1, keepdim=True).values / 127.0
        return torch.where(step > 0, (rows / step).round() * step, torch.zeros_like(rows))

    return turned[:, :nh].reshape(-1, nh * d), stands_for(turned[:, nh:]), stands_for(x[:, nh + nkv:])
