"""The operators of a paged serving step, as cases that can be timed and compared.

Four operators of one step that serves many requests of different lengths at once:

  batch      block table, slot map and token positions of the step, from the requests' lengths
  scatter    the fused QKV product into q rows and K/V pages, with the per-head norms and RoPE
  attention  a chunk of new tokens (or a single one) per request over the paged cache
  sample     the next token from logits, by temperature, top-k, top-p, min-p and a given random number

`run` computes each in its plain form with elementary torch operations; where `own` is true it makes the calls
that a user makes of `popcorn_b200.Kernels`. Head layouts and vocabularies are those of this repository's own
decode configurations (8 / 4 and 16 / 8 heads of 256, vocabulary 256000) or generic ones.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- cases -----------------------------------------------------------------

def listed():
    return [
        # a decode step of a small server: every request adds one token; latency counts
        {"name": "batch decode", "op": "batch", "requests": 32, "chunk": 1, "context": 8192, "page": 16, "mix": 1},
        # a large step that admits many prompts beside running requests
        {"name": "batch prompts", "op": "batch", "requests": 509, "chunk": 700, "context": 8192, "page": 64, "mix": 2},
        # the decode step of a batch of 32 with per-head norms and RoPE
        {"name": "scatter decode", "op": "scatter", "tokens": 32, "q_heads": 16, "kv_heads": 8, "head_dim": 256,
         "page": 16, "dtype": "bf16", "norm": True, "rope": True},
        # a step of long prompt chunks, RoPE alone
        {"name": "scatter chunk", "op": "scatter", "tokens": 8191, "q_heads": 8, "kv_heads": 4, "head_dim": 256,
         "page": 64, "dtype": "f16", "norm": False, "rope": True},
        # one user decoding at a context of 4096
        {"name": "decode one", "op": "attention", "requests": 1, "chunk": 1, "context": 4096, "q_heads": 8,
         "kv_heads": 4, "head_dim": 256, "page": 16, "dtype": "f16", "window": 0, "sinks": 0, "mix": 0},
        # a batch of 32 decoding at contexts up to 8192
        {"name": "decode batch", "op": "attention", "requests": 32, "chunk": 1, "context": 8192, "q_heads": 16,
         "kv_heads": 8, "head_dim": 256, "page": 64, "dtype": "bf16", "window": 0, "sinks": 0, "mix": 3},
        # four whole prompts of 2048 tokens
        {"name": "prompts", "op": "attention", "requests": 4, "chunk": 2048, "context": 2048, "q_heads": 8,
         "kv_heads": 4, "head_dim": 256, "page": 64, "dtype": "bf16", "window": 0, "sinks": 0, "mix": 0},
        # a chunk of a long document: sliding window with a few first tokens kept
        {"name": "long chunk, window, sinks", "op": "attention", "requests": 1, "chunk": 2000, "context": 40001,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "dtype": "f16", "window": 4096, "sinks": 4,
         "mix": 0},
        # running requests and prompt chunks in one step, odd lengths
        {"name": "mixed step", "op": "attention", "requests": 13, "chunk": 515, "context": 6001, "q_heads": 16,
         "kv_heads": 2, "head_dim": 128, "page": 32, "dtype": "bf16", "window": 0, "sinks": 0, "mix": 5},
        # one user's next token, every filter on
        {"name": "sample one", "op": "sample", "rows": 1, "vocab": 256000, "dtype": "bf16", "top_k": 64, "top_p": 0.95,
         "min_p": 0.02},
        # a batch drawing from the nucleus alone
        {"name": "sample nucleus", "op": "sample", "rows": 48, "vocab": 256000, "dtype": "f32", "top_k": 0,
         "top_p": 0.9, "min_p": 0.0},
        # a smaller, odd vocabulary, top-k alone
        {"name": "sample odd vocabulary", "op": "sample", "rows": 131, "vocab": 50257, "dtype": "f16", "top_k": 200,
         "top_p": 1.0, "min_p": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["batch", "scatter", "attention", "attention", "sample"])
    mix = rng.randrange(1, 1 << 20)
    page = rng.choice([8, 16, 24, 32, 64, 128])
    if op == "batch":
        return {"op": op, "requests": _log(rng, 1, 400), "chunk": rng.choice([1, _log(rng, 2, 600)]),
                "context": _log(rng, 1, 8192), "page": rng.choice([1, 7, page]), "mix": mix}
    q_heads, kv_heads = rng.choice([(8, 4), (16, 8), (16, 2), (4, 4), (12, 4), (8, 1)])
    head_dim = rng.choice([64, 128, 256])
    dtype = rng.choice(["bf16", "f16"])
    if op == "scatter":
        row = (q_heads + 2 * kv_heads) * head_dim
        return {"op": op, "tokens": _log(rng, 1, 33000000 // row), "q_heads": q_heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "page": page, "dtype": dtype, "norm": rng.random() < 0.5,
                "rope": rng.random() < 0.7}
    if op == "sample":
        rows = _log(rng, 1, 128)
        return {"op": op, "rows": rows, "vocab": _log(rng, 1000, min(256000, 12000000 // rows)),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "top_k": rng.choice([0, 1, _log(rng, 2, 1000)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                "min_p": rng.choice([0.0, round(rng.uniform(0.001, 0.2), 4)])}
    if rng.random() < 0.5:  # single tokens
        requests, chunk = _log(rng, 1, 64), 1
        context = _log(rng, 1, min(32768, 196608 // requests))
    else:
        requests = _log(rng, 1, 16)
        chunk = _log(rng, 2, min(2048, 8192 // requests))
        most = int(6e10 / (4 * q_heads * head_dim * requests * chunk))  # as much work as the largest listed case
        context = chunk + _log(rng, 1, max(2, min(16384, most) - chunk))
    window = rng.choice([0, 0, _log(rng, 64, 4096)])
    return {"op": op, "requests": requests, "chunk": chunk, "context": context, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype, "window": window,
            "sinks": rng.choice([0, 1, 4, 130]) if window else 0, "mix": mix}


def _lengths(case):
    """(new tokens, keys in the cache after them) of each request. With a mix of 0 every request has the case's
    own; else they are ragged: contexts from a single key to the whole, and, where there are chunks, half of the
    requests add a single token."""
    r, n, s = case["requests"], case["chunk"], case["context"]
    if not case["mix"]:
        return [n] * r, [s] * r
    rng = random.Random(case["mix"])
    new, keys = [], []
    for i in range(r):
        k = s if i == 0 else max(1, int(s * rng.random()))
        m = n if i == 0 else (1 if n == 1 or rng.random() < 0.5 else rng.randint(1, n))
        new.append(min(m, k))
        keys.append(k)
    return new, keys


def _pages(keys, page):
    return [-(-k // page) for k in keys]


# ---- inputs ----------------------------------------------------------------

def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)
    state = {"case": dict(case), "device": device}
    {"batch": _prepare_batch, "scatter": _prepare_scatter, "attention": _prepare_attention,
     "sample": _prepare_sample}[case["op"]](case, state, g)
    return state


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _ramp(lengths):
    """0..n-1 for each n of `lengths`, one after the other, and the index of the n each belongs to."""
    owner = torch.repeat_interleave(torch.arange(lengths.numel(), device=lengths.device), lengths)
    return torch.arange(owner.numel(), device=lengths.device) - (lengths.cumsum(0) - lengths)[owner], owner


def _fill_table(table, counts, ids):
    """The first counts[r] entries of each row from the front of `ids`, one after the other."""
    column, row = _ramp(counts)
    table[row, column] = ids[:row.numel()].to(table.dtype)


def _prepare_batch(case, s, g):
    dev, page = s["device"], case["page"]
    new, keys = _lengths(case)
    cached = [k - n for n, k in zip(new, keys)]
    before, after = _pages(cached, page), _pages(keys, page)
    total = sum(after)
    ids = torch.randperm(total + 64, generator=g, device=dev)
    # as wide as the longest request may get, and room for the tokens of the step as a server pads them
    width = max(after) + 3
    s["page"] = page
    s["cached"], s["new"] = _i32(cached, dev), _i32(new, dev)
    s["table"] = torch.full((case["requests"], width), -1, dtype=torch.int32, device=dev)
    _fill_table(s["table"], torch.tensor(before, device=dev), ids)
    s["free"] = ids[sum(before):].to(torch.int32).contiguous()
    # the head of the free list differs by seed, as after earlier steps
    s["head"] = torch.randint(0, 60, (1,), generator=g, device=dev, dtype=torch.int32)
    tokens = sum(new) + (-sum(new)) % 64 + 64
    for name, n in (("seq_lens", case["requests"]), ("query_start", case["requests"] + 1), ("positions", tokens),
                    ("slots", tokens), ("last_rows", case["requests"]), ("head_out", 1), ("admitted", 1)):
        s[name] = torch.zeros(n, dtype=torch.int32, device=dev)


def _prepare_scatter(case, s, g):
    dev, dt, hd = s["device"], DTYPES[case["dtype"]], case["head_dim"]
    t, nq, nkv, page = case["tokens"], case["q_heads"], case["kv_heads"], case["page"]
    pages = -(-t // page) + 8
    s["qkv"] = torch.randn(t, (nq + 2 * nkv) * hd, generator=g, device=dev).to(dt)
    slots = torch.randperm(pages * page, generator=g, device=dev)[:t]
    slots[t - t // 32:] = -1  # the rows that pad a step
    s["slots"] = slots.to(torch.int32)
    s["k_pages"] = torch.randn(pages, nkv, page, hd, generator=g, device=dev).to(dt)
    s["v_pages"] = torch.randn(pages, nkv, page, hd, generator=g, device=dev).to(dt)
    s["q_out"] = torch.zeros(t, nq, hd, dtype=dt, device=dev)
    s["cos"] = s["sin"] = s["q_norm"] = s["k_norm"] = None
    if case["rope"]:
        position = torch.randint(0, 32768, (t, 1), generator=g, device=dev).double()
        angle = position * 10000.0 ** (-torch.arange(0, hd, 2, device=dev).double() / hd)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    if case["norm"]:
        s["q_norm"] = 0.1 * torch.randn(hd, generator=g, device=dev)
        s["k_norm"] = 0.1 * torch.randn(hd, generator=g, device=dev)


def _prepare_attention(case, s, g):
    dev, dt, hd = s["device"], DTYPES[case["dtype"]], case["head_dim"]
    nq, nkv, page = case["q_heads"], case["kv_heads"], case["page"]
    new, keys = _lengths(case)
    counts = _pages(keys, page)
    pages = sum(counts) + 5
    s["table"] = torch.full((case["requests"], max(counts) + 2), -1, dtype=torch.int32, device=dev)
    _fill_table(s["table"], torch.tensor(counts, device=dev), torch.randperm(pages, generator=g, device=dev))
    s["seq_lens"] = _i32(keys, dev)
    s["query_start"] = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
    s["q"] = (1.5 * torch.randn(sum(new), nq, hd, generator=g, device=dev)).to(dt)
    s["k_pages"] = torch.randn(pages, nkv, page, hd, generator=g, device=dev, dtype=dt)
    s["v_pages"] = torch.randn(pages, nkv, page, hd, generator=g, device=dev, dtype=dt)
    s["out"] = torch.zeros_like(s["q"])
    s["scale"] = hd ** -0.5


def _prepare_sample(case, s, g):
    dev, rows, vocab = s["device"], case["rows"], case["vocab"]
    # a language model's logits: a wide bell, and a few likely tokens above it
    logits = 2.0 * torch.randn(rows, vocab, generator=g, device=dev)
    logits += 3.0 * torch.randn(rows, vocab, generator=g, device=dev).clamp_(min=3.0).sub_(3.0)
    s["logits"] = logits.to(DTYPES[case["dtype"]])
    s["uniform"] = torch.rand(rows, generator=g, device=dev)
    s["temperature"] = 0.5 + torch.rand(rows, generator=g, device=dev)
    s["temperature"][rows // 2::7] = 0.0  # requests that ask for the most likely token
    if rows == 1:
        s["temperature"].fill_(0.8)
    s["top_k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device=dev)
    s["top_p"] = torch.full((rows,), case["top_p"], device=dev)
    s["min_p"] = torch.full((rows,), case["min_p"], device=dev)
    s["tokens"] = torch.zeros(rows, dtype=torch.int32, device=dev)


# ---- one pass --------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        if "encoder" not in state:  # a user's program builds its kernels once, over its own buffers
            _build(state)
        state["encoder"].encode(state["kernel"])
    else:
        {"batch": _batch, "scatter": _scatter, "attention": _attention, "sample": _sample}[op](state)
    return _outputs(state)


def _outputs(s):
    names = {"batch": ("seq_lens", "query_start", "positions", "slots", "last_rows", "head_out", "admitted", "table"),
             "scatter": ("q_out", "k_pages", "v_pages"), "attention": ("out",), "sample": ("tokens",)}
    return {n: s[n] for n in names[s["case"]["op"]]}


_library = {}


def _build(s):
    import popcorn_b200 as pc
    index = s["device"].index
    if index not in _library:
        _library[index] = (pc.KernelLibrary(index), pc.ScratchPool(index))
    library, scratch = _library[index]
    K, op = pc.Kernels, s["case"]["op"]
    if op == "batch":
        kernel = K.PagedBatchBuild(s["cached"], s["new"], s["free"], s["head"], s["table"], s["page"],
                                   seq_lens=s["seq_lens"], query_start=s["query_start"], positions=s["positions"],
                                   slots=s["slots"], last_rows=s["last_rows"], free_head_out=s["head_out"],
                                   admitted=s["admitted"])
    elif op == "scatter":
        kernel = K.PagedQKVScatter(s["qkv"], s["slots"], s["q_out"], s["k_pages"], s["v_pages"], cos=s["cos"],
                                   sin=s["sin"], qk_norm=s["case"]["norm"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                                   norm_v=s["case"]["norm"], add_one_to_weight=True)
    elif op == "attention":
        window = s["case"]["window"]
        mask = pc.AttentionMask.causal_sliding_window(window) if window else pc.AttentionMask.causal
        kernel = K.PagedAttention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["seq_lens"], s["query_start"],
                                  into=s["out"], scale=s["scale"], mask=mask, sinks=s["case"]["sinks"])
    else:
        kernel = K.Sample(s["logits"], s["uniform"], s["tokens"], temperature=s["temperature"], top_k=s["top_k"],
                          top_p=s["top_p"], min_p=s["min_p"])
    s["kernel"] = kernel
    s["encoder"] = pc.KernelCommandEncoder(library, scratch=scratch)


def _batch(s):
    page, table = s["page"], s["table"]
    cached, new = s["cached"].long().clamp(min=0), s["new"].long().clamp(min=0)
    before, after = (cached + page - 1) // page, (cached + new + page - 1) // page
    head, tokens = s["head"].long(), s["positions"].numel()
    need = after - before
    # in the order of the requests: the first that does not fit, and all after it, wait
    fits = (new.cumsum(0) <= tokens) & (head + need.cumsum(0) <= s["free"].numel()) & (after <= table.shape[1])
    admitted = fits.long().cumprod(0)
    new, need = new * admitted, need * admitted
    page_start = need.cumsum(0) - need
    column, row = _ramp(need)
    table[row, before[row] + column] = s["free"][head + page_start[row] + column]
    offset, owner = _ramp(new)
    position = cached[owner] + offset
    n = position.numel()
    s["positions"][:n], s["positions"][n:] = position.to(torch.int32), 0
    s["slots"][:n] = table[owner, position // page] * page + (position % page).to(torch.int32)
    s["slots"][n:] = -1
    s["seq_lens"].copy_(cached + new)
    s["query_start"][1:] = new.cumsum(0)
    s["last_rows"].copy_((new.cumsum(0) - 1).clamp(min=0))
    s["head_out"].copy_(head + need.sum())
    s["admitted"].copy_(admitted.sum())


def _scatter(s):
    case = s["case"]
    nq, nkv, hd, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    x = s["qkv"].view(-1, nq + 2 * nkv, hd).float()
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    if case["norm"]:
        def norm(y):
            return y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)
        q, k, v = norm(q) * (1.0 + s["q_norm"]), norm(k) * (1.0 + s["k_norm"]), norm(v)
    if case["rope"]:
        c, n = s["cos"][:, None], s["sin"][:, None]

        def rope(y):
            a, b = y[..., :hd // 2], y[..., hd // 2:]
            return torch.cat([a * c - b * n, b * c + a * n], -1)
        q, k = rope(q), rope(k)
    dt = s["q_out"].dtype
    s["q_out"].copy_(q)
    rows = (s["slots"] >= 0).nonzero()[:, 0]
    slot = s["slots"][rows].long()
    s["k_pages"][slot // page, :, slot % page] = k[rows].to(dt)
    s["v_pages"][slot // page, :, slot % page] = v[rows].to(dt)


def _padded(s):
    """Rows [R, L] of q per request, their positions, and which of them are there; likewise slots [R, S] of keys."""
    page = s["case"]["page"]
    start, length = s["query_start"].long(), s["seq_lens"].long()
    new = start[1:] - start[:-1]
    column = torch.arange(s["case"]["chunk"], device=s["device"])
    there = column < new[:, None]
    row = (start[:-1, None] + column).clamp(max=s["q"].shape[0] - 1)
    position = (length - new)[:, None] + column
    key = torch.arange(s["case"]["context"], device=s["device"])
    slot = s["table"].long().clamp(min=0)[:, key // page] * page + key % page
    return row, position, there, key, slot, length


def _attention(s):
    case = s["case"]
    nq, nkv, hd, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    row, position, there, key, slot, length = _padded(s)
    q = s["q"][row].float().view(*row.shape, nkv, nq // nkv, hd).permute(0, 2, 3, 1, 4)  # [R, Nkv, G, L, Hd]
    r, _, grp, n, _ = q.shape
    k = s["k_pages"][slot // page, :, slot % page].float().permute(0, 2, 3, 1)  # [R, Nkv, Hd, S]
    v = s["v_pages"][slot // page, :, slot % page].float().permute(0, 2, 1, 3)  # [R, Nkv, S, Hd]
    score = (q.reshape(r, nkv, grp * n, hd) @ k).mul_(s["scale"])
    seen = key <= position[..., None]
    if case["window"]:
        seen = seen & ((position[..., None] - key < case["window"]) | (key < case["sinks"]))
    score = score.view(r, nkv, grp, n, -1).masked_fill_(~seen[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(r, nkv, grp * n, -1) @ v).view(r, nkv, grp, n, hd) / total.clamp(min=1e-37)
    out = out.permute(0, 3, 1, 2, 4).reshape(r, n, nq, hd)
    s["out"][row[there]] = out[there].to(s["out"].dtype)


def _sample(s):
    # in 64 bits: a sum that is a little off moves the border between two tokens
    logits = s["logits"].double()
    logits = torch.where(logits.isnan(), -math.inf, logits)
    vocab = logits.shape[1]
    temperature = s["temperature"].double()[:, None]
    greedy = ~(temperature > 0)
    value, index = torch.sort(logits, dim=1, descending=True, stable=True)
    weight = torch.where(value == value[:, :1], 1.0, torch.exp((value - value[:, :1]) / torch.where(greedy, 1.0, temperature)))
    rank = torch.arange(vocab, device=s["device"])
    top_k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    weight = weight * (rank < top_k)
    mass = weight.cumsum(1)
    top_p = s["top_p"].double()[:, None]
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], 1)
    keep = (before < top_p * mass[:, -1:]) | (top_p >= 1) | (rank == 0)
    keep &= weight >= s["min_p"].double()[:, None]
    keep = torch.where(greedy, rank == 0, keep)
    kept = torch.zeros_like(weight).scatter_(1, index, weight * keep)
    mass = kept.cumsum(1)
    token = (mass <= s["uniform"].double()[:, None] * mass[:, -1:]).sum(1)
    s["tokens"].copy_(torch.where(greedy[:, 0], index[:, 0], token))


# ---- what a pass cannot do without -----------------------------------------

def _visible(case):
    """(rows x keys that they see, keys that some row sees) summed over the requests, one query head."""
    pairs = union = 0
    w, sinks = case["window"], case["sinks"]
    for n, k in zip(*_lengths(case)):
        p = np.arange(k - n, k, dtype=np.int64)
        if w:
            first = np.maximum(0, p - w + 1)
            pairs += int((p + 1 - first + np.minimum(first, sinks)).sum())
            first = max(0, k - n - w + 1)
            union += k - first + min(first, sinks)
        else:
            pairs += int((p + 1).sum())
            union += k
    return pairs, union


def work(case):
    op = case["op"]
    if op == "batch":
        new, keys = _lengths(case)
        need = sum(a - b for a, b in zip(_pages(keys, case["page"]),
                                         _pages([k - n for n, k in zip(new, keys)], case["page"])))
        return {"bytes": 4 * (5 * case["requests"] + 2 * sum(new) + 2 * need), "flops": 0}
    if op == "scatter":
        row = (case["q_heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        tables = 4 * case["head_dim"] * case["tokens"] if case["rope"] else 0
        return {"bytes": 2 * 2 * row * case["tokens"] + tables + 4 * case["tokens"],
                "flops": (6 if case["norm"] else 3) * row * case["tokens"]}
    if op == "attention":
        pairs, union = _visible(case)
        new, _ = _lengths(case)
        hd = case["head_dim"]
        return {"bytes": 2 * (2 * union * case["kv_heads"] * hd + 2 * sum(new) * case["q_heads"] * hd),
                "flops": 4 * pairs * case["q_heads"] * hd}
    size = 4 if case["dtype"] == "f32" else 2
    return {"bytes": size * case["rows"] * case["vocab"], "flops": 2 * case["rows"] * case["vocab"]}


# ---- the definition in 64 bits ---------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"batch": _exact_batch, "scatter": _exact_scatter, "attention": _exact_attention,
            "sample": _exact_sample}[case["op"]](s)


def _exact_batch(s):
    page, cap, width = s["page"], s["positions"].numel(), s["table"].shape[1]
    cached, new, free = s["cached"].tolist(), s["new"].tolist(), s["free"].tolist()
    table, head = s["table"].cpu().numpy().copy(), int(s["head"])
    seq, start, position, slot, last, waits, admitted = [], [0], [], [], [], False, 0
    for r, (c, n) in enumerate(zip(cached, new)):
        first, end = -(-c // page), -(-(c + n) // page)
        waits = waits or len(slot) + n > cap or head + end - first > len(free) or end > width
        if waits:
            n = 0
        else:
            admitted += 1
            table[r, first:end] = free[head:head + end - first]
            head += end - first
        for p in range(c, c + n):
            position.append(p)
            slot.append(int(table[r, p // page]) * page + p % page)
        seq.append(c + n)
        start.append(len(slot))
        last.append(max(0, len(slot) - 1))
    pad = cap - len(slot)
    out = {"seq_lens": seq, "query_start": start, "positions": position + [0] * pad, "slots": slot + [-1] * pad,
           "last_rows": last, "head_out": [head], "admitted": [admitted], "table": table}
    return {k: torch.tensor(np.asarray(v), dtype=torch.int32) for k, v in out.items()}


def _exact_scatter(s):
    case = s["case"]
    nq, nkv, hd, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    x = s["qkv"].double().view(-1, nq + 2 * nkv, hd)
    if case["norm"]:
        x = x / (x.pow(2).sum(-1, keepdim=True) / hd + 1e-6).sqrt()
        gain = torch.ones(nq + 2 * nkv, hd, dtype=torch.float64, device=x.device)
        gain[:nq] += s["q_norm"]
        gain[nq:nq + nkv] += s["k_norm"]
        x = x * gain
    if case["rope"]:
        turn = torch.complex(s["cos"].double(), s["sin"].double())[:, None]
        y = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * turn
        turned = torch.cat([y.real, y.imag], -1)
        x = torch.cat([turned[:, :nq + nkv], x[:, nq + nkv:]], 1)
    out = {"q_out": x[:, :nq].contiguous()}
    there = s["slots"] >= 0
    slot = s["slots"][there].long()
    for name, first in (("k_pages", nq), ("v_pages", nq + nkv)):
        flat = s[name].double().transpose(1, 2).reshape(-1, nkv, hd)  # [slot, Nkv, Hd]
        flat = flat.index_copy(0, slot, x[there][:, first:first + nkv])
        out[name] = flat.view(-1, page, nkv, hd).transpose(1, 2).contiguous()
    return out


def _exact_attention(s):
    case = s["case"]
    pairs, _ = _visible(case)
    if pairs * case["q_heads"] * case["head_dim"] > 4e12:
        return None
    nq, nkv, hd, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    group = nq // nkv
    start, lengths = s["query_start"].tolist(), s["seq_lens"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["device"])
    for r, length in enumerate(lengths):
        pages = s["table"][r, :-(-length // page)].long()
        k = s["k_pages"][pages].transpose(1, 2).reshape(-1, nkv, hd)[:length].double()
        v = s["v_pages"][pages].transpose(1, 2).reshape(-1, nkv, hd)[:length].double()
        n = start[r + 1] - start[r]
        key = torch.arange(length, device=s["device"])
        for first in range(0, n, 512):
            last = min(n, first + 512)
            p = torch.arange(length - n + first, length - n + last, device=s["device"])[:, None]
            hidden = key > p
            if case["window"]:
                hidden = hidden | ((p - key >= case["window"]) & (key >= case["sinks"]))
            for h in range(nq):
                logit = s["q"][start[r] + first:start[r] + last, h].double() @ k[:, h // group].T * s["scale"]
                out[start[r] + first:start[r] + last, h] = logit.masked_fill(hidden, -math.inf).softmax(1) @ v[:, h // group]
    return {"out": out}


def _exact_sample(s):
    tokens = []
    for r in range(s["case"]["rows"]):
        x = s["logits"][r].double().cpu().numpy()
        t, u = float(s["temperature"][r]), float(s["uniform"][r])
        order = np.lexsort((np.arange(x.size), -x))
        if not t > 0:
            tokens.append(int(order[0]))
            continue
        k, p, m = int(s["top_k"][r]), float(s["top_p"][r]), float(s["min_p"][r])
        order = order[:k] if k > 0 else order
        w = np.exp((x[order] - x[order[0]]) / t)
        if p < 1:
            c = np.cumsum(w)
            n = int(np.searchsorted(c, p * c[-1], side="left")) + 1
            order, w = order[:n], w[:n]
        order = order[w >= m]
        order.sort()
        c = np.cumsum(np.exp((x[order] - x.max()) / t))
        tokens.append(int(order[np.searchsorted(c, u * c[-1], side="right")]))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32)}
