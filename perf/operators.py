"""Cases of the cache and scoring operators: attention with a sliding window and
sinks, attention over a prefix that the batch shares, page copies of the KV
cache, and log probabilities of given tokens.

``run`` computes each in plain f32 tensor arithmetic, or (``own``) through the
package's entry points.  Head layouts and vocabulary sizes are those of the
decoder shapes in ``ie_tpq/stack.py`` and ``ie_tpq/model.py``.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

PACKAGE_ROOT = str(Path(__file__).resolve().parent.parent / "inference-engine_b200")
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ITEMSIZE = {"bf16": 2, "f16": 2, "f32": 4}
# (query heads, kv heads, head dim)
LAYOUTS = ((32, 8, 128), (64, 8, 128), (14, 2, 64))


# ---- the cases -------------------------------------------------------------
def listed():
    return [
        # one user's next token on a streaming model: the latency of a decode step
        {"name": "window_decode_one", "kind": "window", "dtype": "bf16", "heads": 32, "kv_heads": 8,
         "head_dim": 128, "seqs": 1, "queries": 1, "context": 2048, "window": 1024, "sinks": 4,
         "block": 16},
        # a full serving batch decoding over contexts far longer than the window
        {"name": "window_decode_batch", "kind": "window", "dtype": "bf16", "heads": 32,
         "kv_heads": 8, "head_dim": 128, "seqs": 64, "queries": 1, "context": 32768,
         "window": 4096, "sinks": 4, "block": 16},
        # chunked prefill of a mixed batch: odd query lengths, earlier context, odd pages
        {"name": "window_prefill_mixed", "kind": "window", "dtype": "f16", "heads": 14,
         "kv_heads": 2, "head_dim": 64, "seqs": 7, "queries": 777, "context": 3989,
         "window": 1000, "sinks": 3, "block": 48},
        # two long prompts prefilled whole
        {"name": "window_prefill_long", "kind": "window", "dtype": "bf16", "heads": 32,
         "kv_heads": 8, "head_dim": 128, "seqs": 2, "queries": 8192, "context": 8192,
         "window": 2048, "sinks": 4, "block": 256},
        # four samples of one short prompt
        {"name": "prefix_decode_four", "kind": "prefix", "dtype": "bf16", "heads": 32,
         "kv_heads": 8, "head_dim": 128, "seqs": 4, "queries": 1, "prefix": 1024, "context": 1100,
         "block": 16},
        # a batch behind one long system prompt, each with a few hundred tokens of its own
        {"name": "prefix_decode_batch", "kind": "prefix", "dtype": "bf16", "heads": 32,
         "kv_heads": 8, "head_dim": 128, "seqs": 64, "queries": 1, "prefix": 8192,
         "context": 8700, "block": 16},
        # many sequences on one document with the larger model's heads
        {"name": "prefix_decode_many", "kind": "prefix", "dtype": "f16", "heads": 64,
         "kv_heads": 8, "head_dim": 128, "seqs": 128, "queries": 1, "prefix": 16384,
         "context": 17400, "block": 64},
        # best-of-16 forks one prompt: the last, partly filled page of every layer is copied
        {"name": "pages_fork", "kind": "pages", "dtype": "bf16", "layers": 32, "kv_heads": 8,
         "head_dim": 128, "block": 16, "pages": 192, "moves": 16, "pattern": "fork"},
        # a fragmented cache is compacted: high live pages move into holes
        {"name": "pages_compact", "kind": "pages", "dtype": "bf16", "layers": 32, "kv_heads": 8,
         "head_dim": 128, "block": 16, "pages": 601, "moves": 220, "pattern": "compact"},
        # the log probability of one sampled token and its five best alternatives
        {"name": "logprobs_one", "kind": "logprobs", "dtype": "f32", "rows": 1, "vocab": 128256,
         "top": 5, "masked": False},
        # a decode batch under a vocabulary mask, twenty alternatives each
        {"name": "logprobs_batch", "kind": "logprobs", "dtype": "f32", "rows": 64,
         "vocab": 128256, "top": 20, "masked": True},
        # scoring a whole prompt
        {"name": "logprobs_prompt", "kind": "logprobs", "dtype": "bf16", "rows": 4095,
         "vocab": 128256, "top": 1, "masked": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("window", "window", "prefix", "pages", "logprobs"))
    if kind == "pages":
        layers = rng.choice((2, 24, 32))
        moves = _log_int(rng, 1, 220)
        return {"kind": kind, "dtype": rng.choice(("bf16", "f16")), "layers": layers,
                "kv_heads": rng.choice((2, 8)), "head_dim": rng.choice((64, 128)),
                "block": rng.choice((1, 7, 16)), "pages": 2 * moves + rng.randint(2, 160),
                "moves": moves, "pattern": rng.choice(("fork", "compact"))}
    if kind == "logprobs":
        dtype = rng.choice(("f32", "bf16", "f16"))
        return {"kind": kind, "dtype": dtype,
                "rows": _log_int(rng, 1, 4095 if dtype != "f32" else 2047),
                "vocab": rng.choice((_log_int(rng, 64, 128256), 128256)),
                "top": rng.randint(0, 20), "masked": rng.random() < 0.5}
    heads, kv_heads, head_dim = rng.choice(LAYOUTS)
    dtype = rng.choice(("bf16", "f16"))
    block = rng.choice((16, 16, 48, 64, 256, 5))
    case = {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim}
    if kind == "window":
        sinks = rng.choice((0, 1, 4, 17, 128))
        if rng.random() < 0.5:    # decode
            case.update(seqs=_log_int(rng, 1, 48), queries=1, context=_log_int(rng, 1, 24000),
                        window=_log_int(rng, 16, 4096))
            if case["context"] <= 4096 and rng.random() < 0.3:
                case["window"] = 0
            if rng.random() < 0.25:   # the f32 model
                case.update(dtype="f32", seqs=min(case["seqs"], 8), heads=14, kv_heads=2,
                            head_dim=64)
        else:                     # prefill: the whole prompt, or a chunk of it
            queries = _log_int(rng, 2, 4096)
            context = queries if rng.random() < 0.5 else queries + _log_int(rng, 1, 2048)
            case.update(seqs=rng.randint(1, 2) if heads < 64 else 1, queries=queries,
                        context=context, window=rng.choice((_log_int(rng, 16, 2048), 0)))
        case.update(sinks=sinks, block=block)
        return case
    prefix = _log_int(rng, 64, 16384)
    queries = 1 if rng.random() < 0.7 else _log_int(rng, 2, 32)
    case.update(seqs=_log_int(rng, 2, 96 if queries == 1 else 12), queries=queries, prefix=prefix,
                context=prefix + queries + _log_int(rng, 1, 900), block=block)
    return case


def _lens(case):
    """(context lengths, query lengths) of an attention case: spread over the batch,
    the longest first, with an empty sequence where the batch is large enough."""
    n, ctx, que = case["seqs"], case["context"], case["queries"]
    spread = [1.0] + [((i * 0.6180339887) % 1.0) for i in range(1, n)]
    floor = case.get("prefix", 0)
    if que == 1:
        context = [max(floor + 1, int(floor + (ctx - floor) * f)) for f in spread]
        if n >= 16 and not floor:
            context[-1] = 0       # a padded row of a fixed-size batch
        return context, [1] * n
    query = [max(1, int(que * f)) for f in spread]
    context = [q + int((ctx - que - floor) * f) + floor for q, f in zip(query, spread)]
    return context, query


def _visible(context, query, window, sinks):
    """(visible (query, key) pairs, keys seen by any query) of one sequence."""
    pairs = 0
    for pos in range(max(context - query, 0), context):
        low = max(0, pos - window + 1) if window else 0
        pairs += pos + 1 - low + min(sinks, low)
    first = max(context - query, 0)
    low = max(0, first - window + 1) if window else 0
    return pairs, (context - low + min(sinks, low) if context > 0 and query > 0 else 0)


def work(case):
    size = ITEMSIZE[case["dtype"]]
    if case["kind"] == "pages":
        page = case["block"] * case["kv_heads"] * case["head_dim"] * size
        read = 1 if case["pattern"] == "fork" else case["moves"]
        return {"bytes": 2 * case["layers"] * (read + case["moves"]) * page, "flops": 0}
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 6 * n}
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    context, query = _lens(case)
    tokens = sum(query)
    pairs = keys = 0
    for c, q in zip(context, query):
        p, k = _visible(c, q, case.get("window", 0), case.get("sinks", 0))
        pairs += p
        keys += k - case.get("prefix", 0)
    keys += case.get("prefix", 0)
    return {"bytes": 2 * tokens * heads * hd * size + 2 * keys * kv * hd * size,
            "flops": 4 * hd * heads * pairs}


# ---- inputs ------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)

    if case["kind"] == "pages":
        return _prepare_pages(case, gen, dtype)
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.empty((rows, vocab), device="cuda", dtype=dtype)
        logits.normal_(0.0, 2.5, generator=gen)
        if case["masked"]:        # the tokens a grammar forbids
            block = torch.rand((rows, vocab), generator=gen, device="cuda") < 0.6
            block[:, 0] = False
            logits.masked_fill_(block, -math.inf)
        tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        return {"case": case, "logits": logits, "tokens": tokens}
    heads, kv, hd, block = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    context, query = _lens(case)
    tables, pages = _tables(case, context, query, gen)
    cu = [0]
    for q in query:
        cu.append(cu[-1] + q)
    i32 = dict(device="cuda", dtype=torch.int32)
    state = {
        "case": case,
        # scores of a trained layer are wider than those of unit normal vectors
        "q": normal(cu[-1], heads, hd, std=1.5),
        "k": normal(pages * block, kv, hd), "v": normal(pages * block, kv, hd),
        "tables": tables, "context": torch.tensor(context, **i32),
        "cu": torch.tensor(cu, **i32), "max_context": max(context), "max_query": max(query),
    }
    return state


def _tables(case, context, query, gen):
    """Block tables over scattered pages.  Pages that no query sees any more (behind
    the window) have been given back and read -1, as do entries past the context."""
    block, prefix = case["block"], case.get("prefix", 0)
    width = max(1, -(-max(context) // block))
    shared = prefix // block      # whole pages; a partial one is every sequence's own copy
    n = len(context)
    ctx, que = torch.tensor(context), torch.tensor(query)
    page = torch.arange(width)[None, :]
    live = page * block < ctx[:, None]
    window = case.get("window", 0)
    if window:
        low = (ctx - que - window + 1).clamp_min(0)[:, None]
        live &= ((page + 1) * block > low) | (page * block < case["sinks"])
    private = live & (page >= shared)
    private[0] = live[0]
    count = int(private.sum())
    order = torch.randperm(count, generator=gen, device="cuda").to(torch.int32)
    tables = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    tables[private.cuda()] = order
    tables[:, :shared] = tables[:1, :shared]
    return tables, max(count, 1)


def _prepare_pages(case, gen, dtype):
    shape = (case["layers"], case["pages"] * case["block"], case["kv_heads"], case["head_dim"])
    k = torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, 1.0, generator=gen)
    v = torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, 1.0, generator=gen)
    moves, pages = case["moves"], case["pages"]
    order = torch.randperm(pages, generator=gen, device="cuda").cpu()
    if case["pattern"] == "fork":     # one parent page, a copy for every child
        src, dst = order[:1].expand(moves), order[1:1 + moves]
    else:                             # the highest pages move into holes below
        src = torch.arange(pages - moves, pages)
        dst = order[order < pages - moves][:moves].sort().values
    state = {"case": case, "k": k, "v": v, "src": src.numpy().astype("int32"),
             "dst": dst.numpy().astype("int32")}
    if own:   # the pool is made once, with the cache
        state["pool"] = _package("kv_pages").KVPagePool(list(k.unbind(0)), list(v.unbind(0)),
                                                        case["block"])
    return state


# ---- one pass ------------------------------------------------------------------
_MODULES: dict = {}


def _package(name):
    if name not in _MODULES:
        import importlib

        if PACKAGE_ROOT not in sys.path:
            sys.path.insert(0, PACKAGE_ROOT)
        _MODULES[name] = importlib.import_module("ie_tpq." + name)
    return _MODULES[name]


def run(state):
    kind = state["case"]["kind"]
    return (_RUN_OWN if own else _RUN_PLAIN)[kind](state)


def _own_window(s):
    c = s["case"]
    return _package("kv_attention").window_attention(
        s["q"], s["k"], s["v"], s["tables"], s["context"], c["block"], window=c["window"],
        sinks=c["sinks"], cu_seqlens_q=s["cu"] if s["max_query"] > 1 else None,
        max_query_len=s["max_query"], max_context_len=s["max_context"])


def _own_prefix(s):
    c = s["case"]
    return _package("kv_attention").shared_prefix_attention(
        s["q"], s["k"], s["v"], s["tables"], s["context"], c["prefix"], c["block"],
        cu_seqlens_q=s["cu"] if s["max_query"] > 1 else None, max_query_len=s["max_query"],
        max_context_len=s["max_context"])


def _own_pages(s):
    s["pool"].copy_pages(s["src"], s["dst"])
    return s["k"], s["v"]


def _own_logprobs(s):
    r = _package("scoring").token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    return r.logprobs, r.entropy, r.top_logprobs, r.top_tokens


# ---- plain forms ---------------------------------------------------------------
def _gather(cache, tables, rows, key, block):
    """f32 keys or values at positions ``key`` of the sequences ``rows``."""
    page = tables[rows, (key // block).clamp_max(tables.shape[1] - 1)].long().clamp_min(0)
    return cache[page * block + key % block].float()


def _softmax_sum(scores, seen, v):
    """Rows of ``softmax(scores) @ v`` over the keys that are seen; 0 where none is."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, p @ v / total, torch.zeros((), device=v.device))


def _positions(s):
    """(sequence, position) of every query token."""
    cu, ctx = s["cu"].long(), s["context"].long()
    token = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(cu, token, right=True) - 1
    return seq, ctx[seq] - (cu[seq + 1] - cu[seq]) + token - cu[seq]


def _plain_window(s):
    c, q = s["case"], s["q"]
    heads, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    group = heads // kv
    window, sinks = c["window"] or c["context"], c["sinks"]
    seq, pos = _positions(s)
    tokens = q.shape[0]
    if s["max_query"] == 1:           # each query gathers just the keys it sees
        n = min(s["max_context"], window + sinks)
        low = (pos - window + 1).clamp_min(0)[:, None]
        ns = low.clamp_max(sinks)
        v = torch.arange(n, device="cuda")[None, :]
        key = torch.where(v < ns, v, low + v - ns)
        seen = (key <= pos[:, None])
        key = key.clamp_max(max(s["max_context"] - 1, 0))
        k = _gather(s["k"], s["tables"], seq[:, None], key, c["block"])
        val = _gather(s["v"], s["tables"], seq[:, None], key, c["block"])
        scores = q.float().view(tokens, kv, group, hd) @ k.permute(0, 2, 3, 1) * hd ** -0.5
        o = _softmax_sum(scores, seen[:, None, None], val.transpose(1, 2))
        return o.reshape(tokens, heads, hd).to(q.dtype)
    seqs, most = c["seqs"], s["max_context"]
    every = torch.arange(most, device="cuda")[None, :].expand(seqs, most)
    row = torch.arange(seqs, device="cuda")[:, None]
    k = _gather(s["k"], s["tables"], row, every, c["block"]).permute(0, 2, 3, 1)
    val = _gather(s["v"], s["tables"], row, every, c["block"]).transpose(1, 2)
    slot = torch.arange(tokens, device="cuda") - s["cu"].long()[seq]
    padded = torch.zeros((seqs, s["max_query"], heads, hd), device="cuda")
    padded[seq, slot] = q.float()
    at = torch.full((seqs, s["max_query"]), -1, device="cuda")
    at[seq, slot] = pos
    rows = padded.view(seqs, -1, kv, group, hd).permute(0, 2, 3, 1, 4)
    scores = (rows.reshape(seqs, kv, -1, hd) @ k).mul_(hd ** -0.5)
    scores = scores.view(seqs, kv, group, s["max_query"], most)
    at = at[:, :, None]
    seen = (every[:, None] <= at) & ((every[:, None] > at - window) | (every[:, None] < sinks))
    o = _softmax_sum(scores, seen[:, None, None], val[:, :, None])
    return o.permute(0, 3, 1, 2, 4)[seq, slot].reshape(tokens, heads, hd).to(q.dtype)


def _plain_prefix(s):
    c, q = s["case"], s["q"]
    heads, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    group, prefix = heads // kv, c["prefix"]
    seq, pos = _positions(s)
    tokens = q.shape[0]
    key = torch.arange(prefix, device="cuda")
    k = _gather(s["k"], s["tables"], 0, key, c["block"])          # [prefix, kv, hd], once
    v = _gather(s["v"], s["tables"], 0, key, c["block"])
    rows = q.float().view(tokens, kv, group, hd).permute(1, 0, 2, 3).reshape(kv, -1, hd)
    first = (rows @ k.permute(1, 2, 0)).view(kv, tokens, group, prefix).permute(1, 0, 2, 3)
    tail = torch.arange(prefix, s["max_context"], device="cuda")[None, :]
    own_k = _gather(s["k"], s["tables"], torch.arange(c["seqs"], device="cuda")[:, None],
                    tail, c["block"]).permute(0, 2, 3, 1)
    own_v = _gather(s["v"], s["tables"], torch.arange(c["seqs"], device="cuda")[:, None],
                    tail, c["block"]).transpose(1, 2)
    second = q.float().view(tokens, kv, group, hd) @ own_k[seq]
    scores = torch.cat((first, second), -1) * hd ** -0.5
    seen = torch.arange(s["max_context"], device="cuda")[None, :] <= pos[:, None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    a = p[..., :prefix].permute(1, 0, 2, 3).reshape(kv, -1, prefix) @ v.transpose(0, 1)
    o = a.view(kv, tokens, group, hd).permute(1, 0, 2, 3) + p[..., prefix:] @ own_v[seq]
    return (o / total).reshape(tokens, heads, hd).to(q.dtype)


def _plain_pages(s):
    c = s["case"]
    src, dst = (torch.from_numpy(s[n]).cuda().long() for n in ("src", "dst"))
    k = s["k"].view(c["layers"], c["pages"], -1)
    v = s["v"].view(c["layers"], c["pages"], -1)
    k[:, dst] = k[:, src]
    v[:, dst] = v[:, src]
    return s["k"], s["v"]


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    given = x.gather(1, s["tokens"][:, None]) - lse
    p /= total
    entropy = -(p * (x - lse).clamp_min(-3e38)).sum(-1)
    # unique whole keys: the value's order first, then the lower index
    bits = (x + 0.0).view(torch.int32)
    bits = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    index = torch.arange(c["vocab"], device="cuda")
    best = torch.topk(bits * 2 ** 32 + (2 ** 32 - 1 - index), min(c["top"], c["vocab"]), dim=-1)
    tokens = 2 ** 32 - 1 - best.values % 2 ** 32
    return given[:, 0], entropy, x.gather(1, tokens) - lse, tokens


_RUN_PLAIN = {"window": _plain_window, "prefix": _plain_prefix, "pages": _plain_pages,
              "logprobs": _plain_logprobs}
_RUN_OWN = {"window": _own_window, "prefix": _own_prefix, "pages": _own_pages,
            "logprobs": _own_logprobs}


# ---- in 64 bits ----------------------------------------------------------------
def exact(case, seed):
    """The definitions in f64, sequence by sequence and head by head."""
    s = prepare(case, seed)
    if case["kind"] == "pages":
        return None
    if case["kind"] == "logprobs":
        given, entropy, best = [], [], []
        for x, t in zip(s["logits"], s["tokens"]):
            x = x.double()
            logp = x - torch.logsumexp(x, 0)
            given.append(logp[t])
            p = logp.exp()
            entropy.append(-torch.where(p > 0, p * logp, torch.zeros_like(p)).sum())
            best.append(logp.sort(descending=True).values[:case["top"]])
        return torch.stack(given), torch.stack(entropy), torch.stack(best), None
    heads, kv, hd, block = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    context, query = _lens(case)
    out = torch.zeros((sum(query), heads, hd), dtype=torch.float64, device="cuda")
    window, sinks, start = case.get("window", 0), case.get("sinks", 0), 0
    for i, (ctx, n) in enumerate(zip(context, query)):
        key = torch.arange(ctx, device="cuda")
        pos = torch.arange(ctx - n, ctx, device="cuda")[:, None]
        if n == 1 and window:             # only the keys that the one query sees
            key = key[(key > ctx - 1 - window) | (key < sinks)]
        page = s["tables"][i, key // block].long()
        page[key < case.get("prefix", 0)] = s["tables"][0, key[key < case.get("prefix", 0)] // block].long()
        slot = page.clamp_min(0) * block + key % block
        hidden = key[None] > pos
        if window:
            hidden |= (key[None] <= pos - window) & (key[None] >= sinks)
        for h in range(kv if ctx > 0 else 0):
            group = slice(h * (heads // kv), (h + 1) * (heads // kv))
            rows = s["q"][start:start + n, group].double().transpose(0, 1)
            scores = (rows @ s["k"][slot, h].double().T).div_(math.sqrt(hd))
            scores.masked_fill_(hidden, -math.inf)
            out[start:start + n, group] = (
                torch.softmax(scores, -1) @ s["v"][slot, h].double()).transpose(0, 1)
        start += n
    return out
