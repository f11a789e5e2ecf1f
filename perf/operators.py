"""Two operators of a server whose requests differ from one another, timed by themselves:

* the product of a shared projection with a low-rank adapter per token beside it,
  y[t] = x[t] W^T + s_a (x[t] A_a^T) B_a^T with a = the adapter of token t's request, or none;
* the choice of the next token from given random numbers with a temperature, top-k, top-p and min-p per row.

A case is a set of sizes; inputs come from a seed.  With `own` false both run in elementary torch operations, products in
32 bits and the choice in 64 (a cumulative sum over a vocabulary has neighbours closer than 32 bits tell apart); with `own`
true they are the calls that a user makes of `inferllm_b200.kernels.ops`.

Which adapter a request has, and each adapter's rank, follow from the case alone; weights, activations, logits, settings and
random numbers follow from the seed.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
# inner size and outputs of a projection: the widths, packed projections and feed-forwards of the benchmark's models and the tests
SHAPES = ((64, 192), (144, 240), (1024, 1536), (1024, 5632), (2816, 1024), (2048, 2048), (4096, 4096), (4096, 6144), (4096, 12288),
          (4096, 22016), (11008, 4096), (5120, 5120), (4096, 1001), (2048, 32001))
VOCABULARIES = (256, 512, 1000, 32000, 32001, 50257, 65521, 128256)
LARGEST_PRODUCT = 2 * 4096 * 4096 * 22016          # of the largest listed case
LARGEST_LOGITS = 64 * 128256


def listed():
    def adapter(name, dtype, tokens, requests, n_in, n_out, pool, used, rank, mixed=False, bare=0):
        return dict(name=name, kind="adapter", dtype=dtype, tokens=tokens, requests=requests, n_in=n_in, n_out=n_out, pool=pool, used=used, rank=rank,
                    mixed=mixed, bare=bare)

    def sample(name, dtype, rows, words, settings, masked=False):
        return dict(name=name, kind="sample", dtype=dtype, rows=rows, words=words, settings=settings, masked=masked)

    return [
        # one user's answer, token by token: the output projection of a 7B layer with that user's adapter
        adapter("adapter-1", "bfloat16", 1, 1, 4096, 4096, 8, 1, 16),
        # eight users with eight adapters, one token each: the packed query, key and value projection
        adapter("adapter-8", "bfloat16", 8, 8, 4096, 12288, 32, 8, 16),
        # a full server: sixty-four single tokens, adapters of several ranks, every fourth request without one, the down projection
        adapter("adapter-64", "bfloat16", 64, 64, 11008, 4096, 64, 48, 64, mixed=True, bare=4),
        # one prompt of a chat turn at the 8B size
        adapter("adapter-200", "bfloat16", 200, 1, 4096, 6144, 8, 1, 16),
        # sixteen unequal prompts in one step, twelve adapters among them, odd ranks
        adapter("adapter-prompts", "bfloat16", 2048, 16, 4096, 4096, 16, 12, 24, mixed=True, bare=5),
        # long prompts through the packed gate and up projection with adapters of a large rank
        adapter("adapter-long", "bfloat16", 4096, 3, 4096, 22016, 4, 2, 64),
        # the checking mode in true float32
        adapter("adapter-float32", "float32", 257, 4, 1024, 5632, 4, 3, 8, mixed=True),
        # a test's model: three rows of a small vocabulary
        sample("sample-small", "float32", 3, 512, "mixed"),
        # one chat at the settings most programs start with
        sample("sample-1", "float32", 1, 32000, "chat"),
        # a full server of requests that each bring settings of their own, some of the words forbidden
        sample("sample-64", "float32", 64, 128256, "mixed", masked=True),
        # many requests, logits in 16 bits (many of them equal)
        sample("sample-256", "bfloat16", 256, 32000, "mixed"),
        # temperature alone, nothing cut off: every word of a large vocabulary can come
        sample("sample-free", "float32", 16, 128256, "free"),
    ]


def draw(rng):
    def between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    if rng.random() < 0.5:
        words = rng.choice(VOCABULARIES + (between(33, 128256),))
        rows = min(between(1, 256), max(1, LARGEST_LOGITS // words))
        return dict(kind="sample", dtype=rng.choice(("float32", "float32", "bfloat16")), rows=rows, words=words,
                    settings=rng.choice(("mixed", "mixed", "chat", "free")), masked=rng.random() < 0.3)
    n_in, n_out = rng.choice(SHAPES)
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    most = min(4096, LARGEST_PRODUCT // (2 * n_in * n_out)) if dtype == "bfloat16" else max(1, min(600, 12000000000 // (2 * n_in * n_out)))
    tokens = between(1, max(1, most))
    # single tokens of many requests, or prompts of a few
    requests = tokens if tokens <= 128 and rng.random() < 0.6 else min(tokens, between(1, 24))
    pool = between(1, 64)
    return dict(kind="adapter", dtype=dtype, tokens=tokens, requests=requests, n_in=n_in, n_out=n_out, pool=pool, used=rng.randint(1, pool),
                rank=rng.choice((4, 8, 16, 16, 24, 32, 64)), mixed=rng.random() < 0.5, bare=rng.choice((0, 0, 2, 3, 5)))


# ---------------------------------------------------------------- what a case says


def ranks_of(case):
    r = case["rank"]
    return [(r, max(1, r // 2), max(1, r * 3 // 4), max(1, r // 4))[i % 4] if case["mixed"] else r for i in range(case["pool"])]


def index_of(case):
    """The adapter of every token, -1 for none: requests one after another, of unequal lengths, adapters in no order."""
    n, left, index = case["requests"], case["tokens"], []
    for i in range(n):
        share = left // (n - i)
        length = left if i == n - 1 else max(1, min(left - (n - 1 - i), int(share * (0.5 + (i * 0.6180339887498949) % 1.0))))
        bare = case["bare"] and i % case["bare"] == case["bare"] - 1
        index += [-1 if bare else (i * 7 + 3) % case["used"]] * length
        left -= length
    return index


def work(case):
    """Inputs and weights once, of the adapters only those that the tokens name, results once."""
    if case["kind"] == "sample":
        n = case["rows"] * case["words"]
        return dict(bytes=n * DTYPES[case["dtype"]].itemsize + case["rows"] * 24, flops=4 * n)
    size, K, N, T = DTYPES[case["dtype"]].itemsize, case["n_in"], case["n_out"], case["tokens"]
    index, ranks = index_of(case), ranks_of(case)
    low = sum(ranks[a] for a in set(index) if a >= 0)
    return dict(bytes=size * (T * K + N * K + T * N + low * (K + N)), flops=2 * T * N * K + 2 * (K + N) * sum(ranks[a] for a in index if a >= 0))


# ---------------------------------------------------------------- inputs


def inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    if case["kind"] == "adapter":
        K, N, ranks = case["n_in"], case["n_out"], ranks_of(case)
        # rows as a norm leaves them; adapters as training leaves them: both factors at work, scale alpha / rank
        return dict(x=normal(case["tokens"], K), w=normal(N, K, std=0.02), a=[normal(r, K, std=K ** -0.5) for r in ranks],
                    b=[normal(N, r, std=0.1) for r in ranks], scale=[(16.0, 32.0, 24.0)[i % 3] / r for i, r in enumerate(ranks)])
    R, V = case["rows"], case["words"]
    logits = torch.randn((R, V), generator=g, device="cuda") * 2.0
    # a handful of words stand out, as after most contexts
    top = torch.randint(0, V, (R, 12), generator=g, device="cuda")
    logits.scatter_(1, top, torch.rand((R, 12), generator=g, device="cuda") * 7.0 + 4.0)
    if case["masked"]:
        logits.masked_fill_(torch.rand((R, V), generator=g, device="cuda") < 0.3, float("-inf"))
        logits[:, V // 2] = 1.0

    def pick(values, kind=torch.float32):
        t = torch.tensor(values, dtype=kind, device="cuda")
        return t[torch.randint(0, len(values), (R,), generator=g, device="cuda")]

    settings = case["settings"]
    if settings == "mixed":
        temp, top_k = pick([0.0, 0.3, 0.7, 1.0, 1.0, 1.3]), pick([0, 0, 1, 20, 50, 1000], torch.int32)
        top_p, min_p = pick([1.0, 1.0, 0.95, 0.9, 0.5]), pick([0.0, 0.0, 0.02, 0.1])
    else:
        free = settings == "free"
        temp, top_k = pick([1.0 if free else 0.8]), pick([0 if free else 40], torch.int32)
        top_p, min_p = pick([1.0 if free else 0.95]), pick([0.0 if free else 0.05])
    return dict(logits=logits.to(dtype), u=torch.rand((R,), generator=g, device="cuda"), temp=temp, top_k=top_k, top_p=top_p, min_p=min_p)


def prepare(case, seed):
    state = dict(inputs(case, seed), kind=case["kind"], own=own)
    if case["kind"] == "sample":
        return state
    index, ranks = index_of(case), ranks_of(case)
    if not own:
        # per adapter in use the rows of its tokens: one look at the step's requests serves all its projections
        at = {}
        for t, a in enumerate(index):
            if a >= 0:
                at.setdefault(a, []).append(t)
        state["at"] = {a: torch.tensor(t, device="cuda") for a, t in sorted(at.items())}
        return state
    from inferllm_b200.kernels import ops
    adapters = ops.Adapters(case["pool"], case["rank"], case["n_out"], case["n_in"], DTYPES[case["dtype"]])
    for i in range(case["pool"]):
        adapters.put(i, state["a"][i], state["b"][i], state["scale"][i])
    state.update(adapters=adapters, rows=ops.AdapterRows(index, adapters.ranks))
    return state


# ---------------------------------------------------------------- one pass


def run(state):
    if state["own"]:
        from inferllm_b200.kernels import ops
        if state["kind"] == "adapter":
            return ops.linear_adapters(state["x"], state["w"], state["adapters"], state["rows"])
        return ops.sample_rows(state["logits"], state["u"], state["temp"], state["top_k"], state["top_p"], state["min_p"])
    if state["kind"] == "adapter":
        return plain_adapters(state)
    return plain_sample(state)


def plain_adapters(state):
    x = state["x"].float()
    y = x @ state["w"].float().t()
    for a, rows in state["at"].items():
        y[rows] += state["scale"][a] * ((x[rows] @ state["a"][a].float().t()) @ state["b"][a].float().t())
    return y.to(state["x"].dtype)


def plain_sample(state):
    """Per row: words in descending order of their logit (equal ones in ascending order of their id) are kept up to the
    top_k-th, up to the first at which the kept ones' probability reaches top_p, and as long as a word is at least min_p times
    as likely as the first; of these the first, in ascending order of the id, at which the probability exceeds u.  Temperature
    0: the lowest id among the largest.  -1 where nothing may come."""
    logits, u = state["logits"].double(), state["u"].double()
    temp, top_k, top_p, min_p = state["temp"].double(), state["top_k"].long(), state["top_p"].double(), state["min_p"].double()
    words = logits.shape[1]
    largest = logits.max(1, keepdim=True).values
    greedy = temp <= 0
    distance = torch.where(logits == largest, torch.zeros_like(logits), logits - largest)
    weight = torch.exp(distance / torch.where(greedy, torch.ones_like(temp), temp)[:, None])
    sorted_logits, order = torch.sort(logits, dim=1, descending=True, stable=True)
    ranked = weight.gather(1, order)
    place = torch.arange(words, device=logits.device)[None]
    keep = place < torch.where(top_k > 0, top_k, torch.full_like(top_k, words))[:, None]
    ranked = torch.where(keep, ranked, torch.zeros_like(ranked))
    reached = torch.cumsum(ranked, 1)
    before = torch.cat([torch.zeros_like(reached[:, :1]), reached[:, :-1]], 1)
    keep &= (top_p >= 1)[:, None] | (before < top_p[:, None] * reached[:, -1:])
    keep &= ranked >= min_p[:, None]
    keep = torch.zeros_like(keep).scatter(1, order, keep)
    weight = torch.where(keep, weight, torch.zeros_like(weight))
    reached = torch.cumsum(weight, 1)
    above = (reached > (u * reached[:, -1])[:, None]) & (weight > 0)
    token = torch.where(greedy, (logits == largest).int().argmax(1), above.int().argmax(1))
    return torch.where(torch.isneginf(largest[:, 0]), torch.full_like(token, -1), token).int()


# ---------------------------------------------------------------- the same in 64 bits, from the definitions


def exact(case, seed):
    given = inputs(case, seed)
    if case["kind"] == "sample":
        return exact_sample(given)
    x, w, index = given["x"].double(), given["w"].double(), torch.tensor(index_of(case), device="cuda")
    y = torch.empty((x.shape[0], w.shape[0]), dtype=torch.float64, device="cuda")
    for a in sorted(set(index.tolist())):
        # the adapter's tokens see the projection with the adapter merged into it
        merged = w if a < 0 else torch.addmm(w, given["b"][a].double(), given["a"][a].double(), alpha=given["scale"][a])
        rows = (index == a).nonzero()[:, 0]
        y[rows] = x[rows] @ merged.t()
    return y


def exact_sample(given):
    out = []
    host = {k: v.double().cpu().numpy() for k, v in given.items()}
    for row in range(len(host["u"])):
        z, temp, k = host["logits"][row], host["temp"][row], int(host["top_k"][row])
        best = z.max()
        if best == -np.inf:
            out.append(-1)
            continue
        if temp <= 0:
            out.append(int(np.flatnonzero(z == best)[0]))
            continue
        order = np.argsort(-z, kind="stable")[:k if k > 0 else None]
        p = np.exp((z[order] - best) / temp)
        if host["top_p"][row] < 1:
            sums = np.cumsum(p)
            order = order[:int(np.searchsorted(sums, host["top_p"][row] * sums[-1], side="left")) + 1]
            p = p[:len(order)]
        order = np.sort(order[p >= host["min_p"][row]])
        sums = np.cumsum(np.exp((z[order] - best) / temp))
        out.append(int(order[min(int(np.searchsorted(sums, host["u"][row] * sums[-1], side="right")), len(order) - 1)]))
    return torch.tensor(out, dtype=torch.int32)
