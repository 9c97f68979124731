"""What the operators of a batch of many requests are timed on.

Three operators of one serving step whose requests differ in what they bring along, and share what they have in common:

``adapters``  low-rank adapters of many requests beside a shared projection: row t of the projection's output gets
              ``scale[i] * (x[t] down[i]^T) up[i]^T`` of its own adapter ``i = ids[t]``, or nothing (``ids[t]`` = -1).
``shared``    attention of a batch over pages, whose sequences share a long prefix: the prefix' pages are read once for all of them.
``controls``  what a request lays on its logits before a token is chosen: penalties for repeated tokens, a bias per token and the mask
              of a grammar.

Sizes are those of the architectures that the framework serves (widths 768 to 8192, 12 to 64 heads, vocabularies of 32000 and 50272), or
generic. Lengths within a batch are spread evenly by arithmetic, so that a case says what it has to read; values come from the seed.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---- the cases -------------------------------------------------------------------------------------------------------
def _adapters(name, tokens, requests, width, outputs, rank, dtype="bf16", used=None, bare=0):
    """`tokens` rows of `requests` requests; `used` adapters among them (each at least once), `bare` requests without one."""
    c = {"op": "adapters", "tokens": tokens, "requests": requests, "width": width, "outputs": outputs, "rank": rank, "dtype": dtype,
         "used": requests - bare if used is None else used, "bare": bare}
    return dict(c, name=name) if name else c


def _shared(name, sequences, heads, kv_heads, dim, prefix, own_keys, dtype="bf16", block=64, groups=1, lone=0, tokens=1):
    """`sequences` in `groups` groups with a prefix each (the last group's is half as long), `lone` sequences with none; up to `own_keys`
    keys and up to `tokens` new tokens of their own."""
    c = {"op": "shared", "sequences": sequences, "heads": heads, "kv_heads": kv_heads, "dim": dim, "prefix": prefix, "own_keys": own_keys,
         "dtype": dtype, "block": block, "groups": groups, "lone": lone, "tokens": tokens}
    return dict(c, name=name) if name else c


def _controls(name, rows, vocab, history, bias, grammar, dtype="bf16"):
    """`rows` requests with up to `history` tokens so far, `bias` biased tokens each, every second one under a grammar if there is one."""
    c = {"op": "controls", "rows": rows, "vocab": vocab, "history": history, "bias": bias, "grammar": grammar, "dtype": dtype}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user of a server decodes with an adapter: latency
        _adapters("adapters-one", 1, 1, 4096, 4096, 16),
        # a decode step of a full batch, every request with an adapter of its own, some with none
        _adapters("adapters-decode", 64, 64, 4096, 11008, 16, bare=3),
        # the same for a wide model with large adapters, in speculative steps of five tokens: an odd number of requests share nine adapters
        _adapters("adapters-steps", 215, 43, 8192, 8192, 64, used=9),
        # prompts of seven requests enter together, one of them without an adapter
        _adapters("adapters-prompts", 4099, 7, 4096, 4096, 32, dtype="fp16", bare=1),
        # a small model answers a few requests behind a common instruction: latency
        _shared("shared-small", 4, 12, 12, 64, 512, 90, dtype="fp16", block=16),
        # a server of a 7B model: an instruction with examples ahead of every request
        _shared("shared-heads", 32, 32, 32, 128, 4096, 300),
        # grouped queries: one long document, questions by many users
        _shared("shared-groups", 64, 64, 8, 128, 8192, 600),
        # two instructions and requests with none, drafts of up to three tokens, an odd number of sequences
        _shared("shared-drafts", 77, 32, 8, 128, 2048, 500, block=32, groups=2, lone=9, tokens=3),
        # a few users ask about a whole book
        _shared("shared-book", 9, 64, 8, 128, 65536, 1500, block=128),
        # one user of the small model, penalties only: latency
        _controls("controls-one", 1, 50272, 700, 0, False, dtype="fp16"),
        # a full batch, everything set
        _controls("controls-batch", 64, 32000, 4096, 300, True),
        # the largest batch, a large vocabulary whose rows start on odd addresses, fp32 logits
        _controls("controls-large", 256, 131071, 8192, 64, True, dtype="fp32"),
    ]


def draw(rng):
    """Any of the three operators, from one row to the largest batch, up to the cost of the largest listed case."""
    over = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["adapters", "shared", "controls"])
        if op == "adapters":
            requests = over(1, 96)
            tokens = requests * (1 if rng.random() < 0.5 else over(1, 200)) + rng.randint(0, 3)
            bare = rng.randint(0, requests // 4)
            c = _adapters(None, tokens, requests, 8 * over(64, 1024), 8 * over(64, 1376), 8 * over(1, 8), rng.choice(["bf16", "bf16", "fp16"]),
                          rng.choice([requests - bare, over(1, requests - bare)]), bare)
        elif op == "shared":
            sequences = over(1, 96)
            heads, kv_heads, dim = rng.choice([(12, 12, 64), (32, 32, 128), (32, 8, 128), (64, 8, 128), (16, 4, 128), (28, 4, 128), (40, 40, 128), (20, 2, 64)])
            block = rng.choice([16, 32, 64, 128])
            groups = rng.randint(1, min(3, sequences))
            lone = rng.choice([0, 0, rng.randint(0, sequences - groups)])
            c = _shared(None, sequences, heads, kv_heads, dim, 2 * block * over(1, 32768 // block), over(4, 2000), rng.choice(["bf16", "bf16", "fp16"]), block,
                        groups, lone, rng.choice([1, 1, rng.randint(2, 4)]))
        else:
            c = _controls(None, over(1, 256), over(1000, 131072), over(1, 8192), rng.choice([0, over(1, 300)]), rng.random() < 0.6,
                          rng.choice(["bf16", "fp16", "fp32"]))
        if _cost(c) <= most:
            return c


def _cost(case):
    """Seconds on a card of 6.5 TB/s and 1600 TFLOP/s, roughly; the plain attention reads every sequence's prefix."""
    w = work(case)
    more = 0.0
    if case["op"] == "shared":
        more = case["sequences"] * case["prefix"] * case["kv_heads"] * case["dim"] * 4 / 6.5e12
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15 + more


# ---- lengths ---------------------------------------------------------------------------------------------------------
def _spread(i, most):
    """1 ... most, every length about as often."""
    return 1 + (i * 7919 + 13) % most


def _lengths(case):
    """Shared attention: (new tokens, keys, prefix) of every sequence and the groups as (first sequence, sequences, prefix)."""
    S, grouped = case["sequences"], case["sequences"] - case["lone"]
    groups, at = [], 0
    for g in range(case["groups"]):
        n = grouped // case["groups"] + (1 if g < grouped % case["groups"] else 0)
        prefix = case["prefix"] // 2 if g and g == case["groups"] - 1 else case["prefix"]
        groups.append((at, n, prefix // case["block"] * case["block"]))
        at += n
    shared = [0] * S
    for first, n, prefix in groups:
        shared[first:first + n] = [prefix] * n
    new = [1 + i % case["tokens"] for i in range(S)]
    keys = [shared[i] + max(new[i], _spread(i, case["own_keys"])) for i in range(S)]
    return new, keys, shared, groups


def _request_lengths(case):
    """Adapters: tokens of every request, longer and shorter ones in turn."""
    n, T = case["requests"], case["tokens"]
    weights = [1 + (i * 5) % 7 if T > 8 * n else 1 for i in range(n)]
    total = sum(weights)
    cuts = [T * sum(weights[:i]) // total for i in range(n + 1)]
    cuts[n] = T
    return [cuts[i + 1] - cuts[i] for i in range(n)]


def _history_lengths(case):
    return [_spread(i, case["history"]) for i in range(case["rows"])]


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "adapters":
        T, R, K, N = case["tokens"], case["rank"], case["width"], case["outputs"]
        with_one = sum(_request_lengths(case)[case["bare"]:])
        return {"bytes": e * (case["used"] * R * (K + N) + with_one * K + 2 * T * N), "flops": 2 * with_one * R * (K + N)}
    if case["op"] == "shared":
        new, keys, shared, groups = _lengths(case)
        rows = sum(new)
        read = sum(p for _, _, p in groups) + sum(k - s for k, s in zip(keys, shared))
        seen = sum(n * k - n * (n - 1) // 2 for n, k in zip(new, keys))
        return {"bytes": e * (2 * read * case["kv_heads"] * case["dim"] + 2 * rows * case["heads"] * case["dim"]),
                "flops": 4 * seen * case["heads"] * case["dim"]}
    n, V = case["rows"], case["vocab"]
    masks = (n // 2 * 4 * -(-V // 32)) if case["grammar"] else 0
    return {"bytes": 2 * e * n * V + 4 * sum(_history_lengths(case)) + 8 * n * case["bias"] + masks + 20 * n, "flops": 6 * n * V}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return {"adapters": _prepare_adapters, "shared": _prepare_shared, "controls": _prepare_controls}[case["op"]](case, g)


def _normal(g, shape, dtype, std=1.0):
    """Normal values of a type, filled piece by piece: a cache may be gigabytes."""
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 26):
        part = flat[at:at + (1 << 26)]
        part.copy_(torch.randn(part.numel(), generator=g, device=DEV) * std)
    return out


def _prepare_adapters(case, g):
    T, R, K, N, n = case["tokens"], case["rank"], case["width"], case["outputs"], case["requests"]
    dt = DTYPES[case["dtype"]]
    bank = case["used"] + 1                       # one more than the batch uses, as in a server
    names = torch.randperm(bank, generator=g, device=DEV).tolist()[:case["used"]]
    adapter = [-1] * case["bare"] + [names[i % case["used"]] for i in range(n - case["bare"])]
    per = [[adapter[i]] * t for i, t in enumerate(_request_lengths(case))]
    st = {"case": case, "ids": sum(per, []), "x": _normal(g, (T, K), dt), "base": _normal(g, (T, N), dt, 1.0),
          "down": _normal(g, (bank, R, K), dt, K**-0.5), "up": _normal(g, (bank, N, R), dt, R**-0.5),
          "scales": 0.5 + torch.rand(bank, generator=g, device=DEV)}
    st["ids_dev"] = torch.tensor(st["ids"], device=DEV)
    if own:
        from hcache_deepspeed_b200.ops import kernels
        st["plan"] = kernels.AdapterPlan(st["ids"], bank, device=DEV)
    return st


def _prepare_shared(case, g):
    new, keys, shared, groups = _lengths(case)
    S, bs, d = case["sequences"], case["block"], case["dim"]
    dt = DTYPES[case["dtype"]]
    own_blocks = [-(-(k - s) // bs) for k, s in zip(keys, shared)]
    total = sum(p // bs for _, _, p in groups) + sum(own_blocks) + 3
    order = torch.randperm(total, generator=g, device=DEV).cpu().to(torch.int32)
    tables, at = torch.zeros(S, max(s // bs + o for s, o in zip(shared, own_blocks)) + 2, dtype=torch.int32), 0
    for first, n, prefix in groups:
        tables[first:first + n, :prefix // bs] = order[at:at + prefix // bs]
        at += prefix // bs
    for i in range(S):
        tables[i, shared[i] // bs:shared[i] // bs + own_blocks[i]] = order[at:at + own_blocks[i]]
        at += own_blocks[i]
    rows = sum(new)
    st = {"case": case, "new": new, "keys": keys, "shared": shared, "groups": groups, "tables": tables.to(DEV), "scale": d**-0.5,
          "q": _normal(g, (rows, case["heads"] * d), dt, 2.0), "cache": _normal(g, (total, 2, case["kv_heads"], bs, d), dt),
          "out": torch.zeros(rows, case["heads"] * d, dtype=dt, device=DEV)}
    if own:
        from hcache_deepspeed_b200.ops import kernels
        st["plan"] = kernels.SharedPrefixPlan(new, keys, groups, case["heads"], case["kv_heads"], d, bs, device=DEV)
    return st


def _prepare_controls(case, g):
    n, V, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    lengths = _history_lengths(case)
    cap = case["history"]
    rand = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    st = {"case": case, "logits": _normal(g, (n, V), dt, 4.0),
          # few tokens make up most of a text
          "history": (rand(n, cap) ** 3 * V).to(torch.int32).clamp_(max=V - 1), "history_len": torch.tensor(lengths, dtype=torch.int32, device=DEV),
          "prompt_len": torch.tensor([x * (i % 3) // 3 for i, x in enumerate(lengths)], dtype=torch.int32, device=DEV),
          "repetition": 1.0 + 0.3 * rand(n), "presence": rand(n) - 0.2, "frequency": 0.5 * rand(n) - 0.1, "bias_ids": None, "bias": None,
          "mask": None, "mask_rows": None}
    if case["bias"]:
        # tokens of a row's list are all different: places of an even spread, moved at random
        step = V // case["bias"]
        st["bias_ids"] = (torch.arange(case["bias"], device=DEV) * step + (rand(n, case["bias"]) * step).long().clamp_(max=step - 1)).to(torch.int32)
        st["bias"] = 10.0 * rand(n, case["bias"]) - 5.0
    if case["grammar"]:
        words = -(-V // 32)
        bits = torch.randint(0, 1 << 32, (max(1, n // 2), words), generator=g, device=DEV)
        st["mask"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
        st["mask_rows"] = torch.tensor([i // 2 if i % 2 and i // 2 < n // 2 else -1 for i in range(n)], dtype=torch.int32, device=DEV)
    return st


# ---- a pass ----------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    return {"adapters": _plain_adapters, "shared": _plain_shared, "controls": _plain_controls}[state["case"]["op"]](state)


def _own(st):
    from hcache_deepspeed_b200.ops import kernels
    op = st["case"]["op"]
    if op == "adapters":
        return kernels.adapter_add(st["base"], st["x"], st["down"], st["up"], st["scales"], st["plan"])
    if op == "shared":
        kernels.paged_attention_shared(st["q"], st["out"], st["cache"], st["tables"], st["plan"], st["scale"])
        return st["out"]
    return kernels.logit_controls(st["logits"], history=st["history"], history_len=st["history_len"], prompt_len=st["prompt_len"],
                                  repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"], bias_ids=st["bias_ids"],
                                  bias=st["bias"], mask=st["mask"], mask_rows=st["mask_rows"])


def _plain_adapters(st):
    y = st["base"].float()
    x = st["x"].float()
    for i in sorted(set(st["ids"])):
        if i >= 0:
            rows = (st["ids_dev"] == i).nonzero()[:, 0]
            y[rows] += st["scales"][i] * (x[rows] @ st["down"][i].float().t() @ st["up"][i].float().t())
    return y.to(st["base"].dtype)


def _plain_shared(st):
    case = st["case"]
    kvh, d, bs = case["kv_heads"], case["dim"], case["block"]
    G, row = case["heads"] // kvh, 0
    out = torch.empty_like(st["out"])
    for i, (n, keys) in enumerate(zip(st["new"], st["keys"])):
        pages = st["cache"][st["tables"][i, :-(-keys // bs)].long()].float()                  # [pages, 2, kvh, bs, d]
        k, v = pages.permute(1, 2, 0, 3, 4).reshape(2, kvh, -1, d)[:, :, :keys]
        q = st["q"][row:row + n].float().view(n, kvh, G, d).permute(1, 0, 2, 3).reshape(kvh, n * G, d)
        s = (q @ k.transpose(1, 2)).view(kvh, n, G, keys) * st["scale"]
        hidden = torch.arange(keys, device=DEV)[None] > torch.arange(keys - n, keys, device=DEV)[:, None]
        s = s.masked_fill(hidden[None, :, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = (p / p.sum(-1, keepdim=True)).view(kvh, n * G, keys) @ v
        out[row:row + n] = o.view(kvh, n, G, d).permute(1, 0, 2, 3).reshape(n, -1).to(out.dtype)
        row += n
    return out


def _plain_controls(st):
    x = st["logits"].float()
    n, V = x.shape
    place = torch.arange(st["history"].shape[1], device=DEV)[None]
    live, answer = place < st["history_len"][:, None], place >= st["prompt_len"][:, None]
    ids = st["history"].long()
    seen = torch.zeros_like(x).scatter_add_(1, ids, live.float()) > 0
    count = torch.zeros_like(x).scatter_add_(1, ids, (live & answer).float())
    r = st["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None] * count - st["presence"][:, None] * (count > 0)
    if st["bias"] is not None:
        x = x.scatter_add(1, st["bias_ids"].long(), st["bias"])
    if st["mask"] is not None:
        token = torch.arange(V, device=DEV)
        allowed = (st["mask"][st["mask_rows"].clamp(min=0).long()][:, token // 32] >> (token % 32)) & 1
        x = x.masked_fill((allowed == 0) & (st["mask_rows"] >= 0)[:, None], -math.inf)
    return x.to(st["logits"].dtype)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"adapters": _exact_adapters, "shared": _exact_shared, "controls": _exact_controls}[case["op"]](st)


def _exact_adapters(st):
    out = st["base"].double()
    start, ids = 0, st["ids"]
    while start < len(ids):                       # runs of rows with the same adapter
        stop = start
        while stop < len(ids) and ids[stop] == ids[start]:
            stop += 1
        if ids[start] >= 0:
            down, up = st["down"][ids[start]].double(), st["up"][ids[start]].double()
            hidden = torch.einsum("tk,rk->tr", st["x"][start:stop].double(), down)
            out[start:stop] += st["scales"][ids[start]].double() * torch.einsum("tr,nr->tn", hidden, up)
        start = stop
    return out


def _exact_shared(st):
    """Token by token and KV head by KV head, over the keys that the token sees."""
    case = st["case"]
    kvh, d, bs = case["kv_heads"], case["dim"], case["block"]
    G = case["heads"] // kvh
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for i, (n, keys) in enumerate(zip(st["new"], st["keys"])):
        ids = st["tables"][i, :(keys + bs - 1) // bs].long()
        for h in range(kvh):
            k = st["cache"][ids, 0, h].reshape(-1, d).double()
            v = st["cache"][ids, 1, h].reshape(-1, d).double()
            for t in range(n):
                sees = keys - n + t + 1
                q = st["q"][row + t, h * G * d:(h + 1) * G * d].view(G, d).double()
                w = torch.softmax(torch.einsum("gd,kd->gk", q, k[:sees]) * st["scale"], dim=1)
                out[row + t, h * G * d:(h + 1) * G * d] = torch.einsum("gk,kd->gd", w, v[:sees]).reshape(-1)
        row += n
    return out


def _exact_controls(st):
    """Row by row."""
    out = st["logits"].double()
    V = out.shape[1]
    lengths, prompts = st["history_len"].tolist(), st["prompt_len"].tolist()
    for i in range(out.shape[0]):
        x = out[i]
        told = st["history"][i, :lengths[i]].long()
        both = torch.bincount(told, minlength=V)
        answer = torch.bincount(told[prompts[i]:], minlength=V)
        rep = st["repetition"][i].double()
        seen = both > 0
        x[seen] = torch.where(x[seen] > 0, x[seen] / rep, x[seen] * rep)
        x -= st["frequency"][i].double() * answer
        x -= st["presence"][i].double() * (answer > 0)
        if st["bias"] is not None:
            x.index_add_(0, st["bias_ids"][i].long(), st["bias"][i].double())
        if st["mask"] is not None and int(st["mask_rows"][i]) >= 0:
            words = st["mask"][int(st["mask_rows"][i])]
            bits = torch.stack([(words >> b) & 1 for b in range(32)], dim=1).reshape(-1)[:V]
            x[bits == 0] = -math.inf
    return out
