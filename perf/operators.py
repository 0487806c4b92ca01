"""Cases and plain forms of the paged decode operators.

Four operators serve one token-VLA decode step and what follows it:

  append    new tokens' K and V rows go into a paged key-value cache (bf16,
            fp16, or e4m3 with one scale per row);
  decode    attention of one new token per sequence over that cache, with
            grouped query heads; on request every key's attention weight is
            added to the sequence's accumulated weights;
  evict     a sequence is cut to a budget of tokens per KV head: the most
            recent ones and those of the greatest accumulated weight, moved in
            order to the pages of another page table;
  logprobs  log probability of given tokens, entropy, and the top alternatives
            of every row of logits.

``run`` with ``own`` false is the definition in elementary torch operations in
32 bits; with ``own`` true it is the call a user makes of this package.
"""

from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}


# ------------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # One decode step of 64 candidates: one row per sequence and head, nothing but latency.
        dict(name="append_step", op="append", batch=64, short=512, long=520, new=1, kv_heads=32, head_dim=128,
             page=16, kv="bf16", layout="bhsd"),
        # The prompts of a batch of requests enter an e4m3 cache at once: quantizing at memory speed.
        dict(name="append_prompts_e4m3", op="append", batch=48, short=0, long=0, new=4099, kv_heads=8, head_dim=128,
             page=64, kv="e4m3", layout="bhsd"),
        # One robot, one candidate: the smallest call, a 512-token prompt and a few action tokens.
        dict(name="decode_one", op="decode", batch=1, short=519, long=519, q_heads=32, kv_heads=32, head_dim=128,
             page=16, kv="bf16", layout="bhsd", weights=False),
        # 64 candidates of 8 tokens behind a 512-token prompt each, weights kept for a later eviction.
        dict(name="decode_candidates", op="decode", batch=64, short=512, long=520, q_heads=32, kv_heads=32,
             head_dim=128, page=16, kv="bf16", layout="bhsd", weights=True),
        # Two long episodes: few rows, the work has to be split over the cache's length.
        dict(name="decode_long", op="decode", batch=2, short=99991, long=131071, q_heads=32, kv_heads=8, head_dim=128,
             page=64, kv="fp16", layout="bshd", weights=False),
        # A serving batch of ragged lengths on an e4m3 cache, grouped heads, weights kept.
        dict(name="decode_batch_e4m3", op="decode", batch=128, short=1, long=8191, q_heads=32, kv_heads=8,
             head_dim=128, page=32, kv="e4m3", layout="bhsd", weights=True),
        # One sequence passes its budget: latency of the selection and of a small move.
        dict(name="evict_one", op="evict", batch=1, short=1100, long=1100, budget=512, recent=64, kv_heads=32,
             head_dim=128, page=16, kv="bf16", layout="bhsd"),
        # A batch of episodes of unequal length, some still below the budget.
        dict(name="evict_batch", op="evict", batch=16, short=1001, long=16385, budget=4096, recent=256, kv_heads=8,
             head_dim=128, page=64, kv="bf16", layout="bshd"),
        # Few long episodes on an e4m3 cache: the selection runs over a long row of weights.
        dict(name="evict_long_e4m3", op="evict", batch=2, short=70001, long=98303, budget=16000, recent=1000,
             kv_heads=8, head_dim=128, page=32, kv="e4m3", layout="bhsd"),
        # The score of one sampled token.
        dict(name="logprobs_one", op="logprobs", rows=1, vocab=32000, dtype="bf16", top=5),
        # 64 candidates of 8 action tokens, ranked by their log probability.
        dict(name="logprobs_candidates", op="logprobs", rows=512, vocab=32000, dtype="bf16", top=8),
        # Prompt scoring of a batch with a large odd vocabulary: rows start at odd addresses.
        dict(name="logprobs_prompts", op="logprobs", rows=4095, vocab=100003, dtype="fp32", top=20),
    ]


def _log_uniform(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    op = rng.choice(("append", "decode", "decode", "evict", "logprobs"))
    if op == "logprobs":
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        vocab = _log_uniform(rng, 500, 160000)
        rows = _log_uniform(rng, 1, max(1, min(16384, 4095 * 100003 // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, top=rng.randint(0, 32))
    kv = rng.choice(("bf16", "fp16", "e4m3"))
    head_dim = rng.choice((64, 128, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8, 32))
    common = dict(kv_heads=kv_heads, head_dim=head_dim, page=rng.choice((16, 32, 48, 64, 128)), kv=kv,
                  layout=rng.choice(("bhsd", "bshd")))
    tokens = int(2e9 / (kv_heads * head_dim * 8))  # cached tokens of all sequences, at the listed cases' size
    if op == "append":
        batch = _log_uniform(rng, 1, 128)
        new = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, max(2, min(4096, tokens // (4 * batch))))
        short = rng.randint(0, 300)
        return dict(op=op, batch=batch, short=short, long=short + rng.randint(0, 400), new=new, **common)
    if op == "decode":
        batch = _log_uniform(rng, 1, 128)
        long = _log_uniform(rng, 16, max(17, min(131071, tokens // batch)))
        group = rng.choice((1, 2, 4, 6, 8, 16))
        return dict(op=op, batch=batch, short=rng.randint(0, long), long=long,
                    q_heads=kv_heads * (group if kv_heads < 32 else 1), weights=rng.random() < 0.5, **common)
    batch = _log_uniform(rng, 1, 16)
    long = _log_uniform(rng, 300, max(301, min(98303, tokens // (2 * batch))))
    budget = rng.randint(max(1, long // 8), max(2, long // 2))
    return dict(op=op, batch=batch, short=rng.randint(1, long), long=long, budget=budget,
                recent=rng.randint(0, budget), **common)


def _lengths(case: dict) -> list[int]:
    """Lengths spread over [short, long]; the longest is ``long``."""
    n, short, long = case["batch"], case["short"], case["long"]
    return [long - round((long - short) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _new_tokens(case: dict) -> list[int]:
    """New tokens of each sequence: one each, or between an eighth of ``new`` and ``new``."""
    n, new = case["batch"], case["new"]
    return [new - round((new - max(1, new // 8)) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def work(case: dict) -> dict:
    """Each input read once and each output written once."""
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # exp, two sums and two products of each logit
        return {"bytes": rows * (vocab * _SIZE[case["dtype"]] + 16 + 12 * case["top"]), "flops": 6 * rows * vocab}
    H, D, size = case["kv_heads"], case["head_dim"], _SIZE[case["kv"]]
    row = 2 * (D * size + (4 if case["kv"] == "e4m3" else 0))  # one token's K and V of one head
    if case["op"] == "append":
        n = sum(_new_tokens(case)) * H
        return {"bytes": n * (4 * D + row), "flops": (6 if case["kv"] == "e4m3" else 0) * n * D}
    lens = _lengths(case)
    if case["op"] == "decode":
        n, q = sum(lens) * H, case["batch"] * case["q_heads"]
        return {"bytes": n * (row + (8 if case["weights"] else 0)) + q * (4 * D + 4),
                "flops": 4 * D * sum(lens) * case["q_heads"]}
    read = sum(lens) * H
    kept = sum(min(x, case["budget"]) for x in lens) * H
    return {"bytes": 4 * read + kept * (2 * row + 4 + 4), "flops": read}


# ------------------------------------------------------------------ inputs
def _pages(n: int, page: int) -> int:
    return (n + page - 1) // page


def _tables(counts: list[int], width: int, first: int, perm: torch.Tensor) -> torch.Tensor:
    """(batch, width) int32 page tables from a shuffled pool; -1 past a sequence's pages."""
    table = torch.full((len(counts), width), -1, dtype=torch.int32)
    for b, n in enumerate(counts):
        table[b, :n] = perm[first : first + n]
        first += n
    return table


def _rows_e4m3(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 rows and one scale per row (last dimension): the amax, floored at
    the input type's value nearest 1e-6, over 425.6 rounded to the input type;
    the values times its reciprocal, clamped to +-448, rounded once."""
    f = x.float()
    floor = torch.full((), 1e-6, dtype=x.dtype, device=x.device).float()
    scale = (torch.maximum(f.abs().amax(-1), floor) / 425.6).to(x.dtype).float()
    return (f * (1.0 / scale).unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    s: dict = {"op": case["op"]}
    if case["op"] == "logprobs":
        rows, vocab, dtype = case["rows"], case["vocab"], _TYPES[case["dtype"]]
        x = torch.randn((rows, vocab), generator=gen, device="cuda")
        x.mul_(2.0)
        # one confident logit a row, and the padding at the vocabulary's end masked off
        peak = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        x[torch.arange(rows, device="cuda"), peak] += 8.0
        x[:, vocab - vocab // 500 :] = float("-inf")
        usual = torch.randint(0, vocab - vocab // 500, (rows,), generator=gen, device="cuda")
        s["logits"] = x.to(dtype)
        s["tokens"] = torch.where(torch.rand((rows,), generator=gen, device="cuda") < 0.5, peak, usual)
        s["top"] = case["top"]
        return s

    H, D, page, layout = case["kv_heads"], case["head_dim"], case["page"], case["layout"]
    lens = _lengths(case)
    order = torch.randperm(case["batch"], generator=host).tolist()
    lens = [lens[i] for i in order]
    new = [_new_tokens(case)[i] for i in order] if case["op"] == "append" else [0] * len(lens)
    after = [a + b for a, b in zip(lens, new)]
    kept = [_pages(min(n, case["budget"]), page) for n in lens] if case["op"] == "evict" else []
    counts = [_pages(n, page) for n in after]
    pool = sum(counts) + sum(kept) + 3
    perm = torch.randperm(pool, generator=host).to(torch.int32)
    s["page_table"] = _tables(counts, max(1, max(counts)), 0, perm).cuda()
    s["lengths"] = torch.tensor(lens, dtype=torch.int32).cuda()
    kv = _TYPES[case["kv"]]
    shape = (pool, H, page, D) if layout == "bhsd" else (pool, page, H, D)
    s["layout"] = layout
    half = torch.bfloat16 if case["kv"] == "e4m3" else kv
    s["k_scales"] = s["v_scales"] = None
    for name in ("k", "v"):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(half)
        if case["kv"] == "e4m3":
            x, scale = _rows_e4m3(x)
            s[name + "_scales"] = (scale if layout == "bhsd" else scale.transpose(1, 2)).contiguous()
        s[name] = x
    if case["op"] == "append":
        starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
        total = int(starts[-1])
        s["starts"] = None if case["new"] == 1 else starts.cuda()
        s["new"] = [torch.randn((total, H, D), generator=gen, device="cuda").to(half) for _ in range(2)]
    elif case["op"] == "decode":
        s["q"] = torch.randn((case["batch"], case["q_heads"], D), generator=gen, device="cuda").to(half)
        s["weights"] = None
        if case["weights"]:
            s["weights"] = torch.rand((case["batch"], H, s["page_table"].shape[1] * page), generator=gen, device="cuda")
    else:
        # accumulated weights are spread over orders of magnitude; some keys never had any
        shape = (case["batch"], H, s["page_table"].shape[1] * page)
        w = torch.exp(2.0 * torch.randn(shape, generator=gen, device="cuda") - 4.0)
        s["weights"] = torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.1, torch.zeros_like(w), w)
        s["out_table"] = _tables(kept, _pages(case["budget"], page), sum(counts), perm).cuda()
        s["budget"], s["recent"] = case["budget"], case["recent"]
    if own:
        from repercep_runtime_b200 import paged

        s["cache"] = paged.PagedKV(s["k"], s["v"], s["k_scales"], s["v_scales"], layout)
    return s


# ------------------------------------------------------------- plain forms
def _raw(x: torch.Tensor) -> torch.Tensor:
    """e4m3 as bytes, for indexing."""
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _slots(s: dict, table: torch.Tensor, seq: torch.Tensor, pos: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Page and slot of positions ``pos`` of sequences ``seq``."""
    page = s["k"].shape[2 if s["layout"] == "bhsd" else 1]
    return table[seq, (pos // page).clamp(max=table.shape[1] - 1)].long(), pos % page


def _heads_first(s: dict, name: str) -> torch.Tensor:
    """(pages, heads, page, D) view of a pool."""
    return _raw(s[name]) if s["layout"] == "bhsd" else _raw(s[name]).transpose(1, 2)


def _plain_append(s: dict) -> dict:
    total = s["new"][0].shape[0]
    t = torch.arange(total, device="cuda")
    if s["starts"] is None:
        seq, pos, counts = t, s["lengths"].long(), torch.ones_like(s["lengths"])
    else:
        starts = s["starts"].long()
        seq = torch.searchsorted(starts, t, right=True) - 1
        pos = s["lengths"].long()[seq] + t - starts[seq]
        counts = s["starts"][1:] - s["starts"][:-1]
    page, slot = _slots(s, s["page_table"], seq, pos)
    out = {}
    for name, x in zip(("k", "v"), s["new"]):
        if s[name].dtype == torch.float8_e4m3fn:
            x, scale = _rows_e4m3(x)
            s[name + "_scales"][page, :, slot] = scale
            out[name + "_scales"] = s[name + "_scales"]
        _heads_first(s, name)[page, :, slot] = _raw(x)
        out[name] = s[name]
    out["lengths"] = s["lengths"] + counts
    return out


def _gathered(s: dict, name: str) -> torch.Tensor:
    """(batch, heads, capacity, D) fp32 K or V of every sequence."""
    table = s["page_table"].clamp(min=0).long()
    x = _heads_first(s, name)[table]  # batch, pages, heads, page, D
    B, P, H, page, D = x.shape
    x = x.permute(0, 2, 1, 3, 4).reshape(B, H, P * page, D)
    if s[name].dtype == torch.float8_e4m3fn:
        scale = s[name + "_scales"][table].permute(0, 2, 1, 3).reshape(B, H, P * page, 1)
        return x.view(torch.float8_e4m3fn).float() * scale
    return x.float()


def _plain_decode(s: dict) -> dict:
    k, v = _gathered(s, "k"), _gathered(s, "v")
    B, H, L, D = k.shape
    q = s["q"].float().view(B, H, -1, D)
    x = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    gone = torch.arange(L, device="cuda") >= s["lengths"].view(B, 1, 1, 1)
    x = x.masked_fill(gone, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == float("-inf"), 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0.0, 1.0)
    out = {"out": torch.matmul(p, v).reshape(B, -1, D).to(s["q"].dtype), "lse": (top + torch.log(total)).reshape(B, -1)}
    if s["weights"] is not None:
        s["weights"].add_(p.sum(2))
        out["weights"] = s["weights"]
    return out


def _plain_evict(s: dict) -> dict:
    w, budget, recent = s["weights"], s["budget"], s["recent"]
    B, H, L = w.shape
    n = s["lengths"].view(B, 1, 1)
    pos = torch.arange(L, device="cuda").view(1, 1, L)
    older = pos < n - recent
    rank = torch.empty((B, H, L), dtype=torch.int64, device="cuda")
    order = torch.sort(w.masked_fill(~older, float("-inf")), dim=-1, descending=True, stable=True).indices
    rank.scatter_(2, order, pos.expand(B, H, L))
    keep = torch.where(n <= budget, pos < n, torch.where(older, rank < budget - recent, pos < n))
    kept = torch.sort(torch.where(keep, pos, L), dim=-1).values[:, :, :budget]
    if kept.shape[2] < budget:
        kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[2]), value=L)
    lengths = s["lengths"].clamp(max=budget)
    valid = kept < L
    # the move: a place past the new length repeats the sequence's last row
    place = torch.minimum(torch.arange(budget, device="cuda"), lengths.long().view(B, 1, 1) - 1).expand(B, H, budget)
    seq = torch.arange(B, device="cuda").view(B, 1, 1).expand(B, H, budget)
    head = torch.arange(H, device="cuda").view(1, H, 1).expand(B, H, budget)
    to_page, to_slot = _slots(s, s["out_table"], seq, place)
    page, slot = _slots(s, s["page_table"], seq, kept.gather(2, place))
    out = {}
    for name in ("k", "v"):
        rows = _heads_first(s, name)
        rows[to_page, head, to_slot] = rows[page, head, slot]
        out[name] = s[name]
        if s[name + "_scales"] is not None:
            scales = s[name + "_scales"]
            scales[to_page, head, to_slot] = scales[page, head, slot]
            out[name + "_scales"] = scales
    cut = torch.zeros((B, H, s["out_table"].shape[1] * s["k"].shape[2 if s["layout"] == "bhsd" else 1]), device="cuda")
    cut[:, :, :budget] = torch.where(valid, w.gather(2, kept.clamp(max=L - 1)), 0.0)
    out.update(kept=torch.where(valid, kept, -1).to(torch.int32), lengths=lengths, weights=cut)
    return out


def _plain_logprobs(s: dict) -> dict:
    x = s["logits"].float()
    rows, vocab = x.shape
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    logp = x - lse
    p = torch.exp(logp)
    out = {"entropy": -(p * logp.masked_fill(p == 0.0, 0.0)).sum(-1),
           "logprobs": logp.gather(1, s["tokens"].view(-1, 1)).view(-1)}
    # ties go to the lowest index: whole-number keys of value first, then index
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 31) + (vocab - 1 - torch.arange(vocab, device="cuda"))
    ids = vocab - 1 - (torch.topk(key, s["top"], dim=-1).values & ((1 << 31) - 1))
    out.update(top_ids=ids, top_logprobs=logp.gather(1, ids))
    return out


def _own_call(s: dict) -> dict:
    from repercep_runtime_b200 import paged, scoring

    if s["op"] == "logprobs":
        got = scoring.token_logprobs(s["logits"], s["tokens"], top=s["top"])
        return {"entropy": got.entropy, "logprobs": got.logprobs, "top_ids": got.top_ids,
                "top_logprobs": got.top_logprobs}
    c = s["cache"]
    scales = {} if c.k_scales is None else {"k_scales": c.k_scales, "v_scales": c.v_scales}
    if s["op"] == "append":
        lengths = paged.append(c, *s["new"], s["page_table"], s["lengths"], starts=s["starts"])
        return {"k": c.k, "v": c.v, "lengths": lengths, **scales}
    if s["op"] == "decode":
        out, lse = paged.decode(s["q"], c, s["page_table"], s["lengths"], weights=s["weights"], return_lse=True)
        return {"out": out, "lse": lse} | ({} if s["weights"] is None else {"weights": s["weights"]})
    got = paged.evict(c, s["page_table"], s["lengths"], s["weights"], s["out_table"], budget=s["budget"],
                      recent=s["recent"])
    return {"k": c.k, "v": c.v, "kept": got.kept, "lengths": got.lengths, "weights": got.weights, **scales}


_PLAIN = {"append": _plain_append, "decode": _plain_decode, "evict": _plain_evict, "logprobs": _plain_logprobs}


def run(state: dict) -> dict:
    return _own_call(state) if own else _PLAIN[state["op"]](state)


# ---------------------------------------------------------- in 64 bits
def _exact_decode(case: dict, s: dict) -> dict:
    B, Hq, D = s["q"].shape
    H, page = case["kv_heads"], case["page"]
    out = torch.zeros((B, Hq, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq), float("-inf"), dtype=torch.float64, device="cuda")
    weights = None if s["weights"] is None else s["weights"].double()
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        pages = s["page_table"][b, : _pages(n, page)].long()
        rows = []
        for name in ("k", "v"):
            x = s[name].view(torch.int8)[pages].view(s[name].dtype)  # by bytes: the e4m3 type has no indexing
            x = x.double() if s["layout"] == "bhsd" else x.double().transpose(1, 2)
            if s[name + "_scales"] is not None:
                x = x * s[name + "_scales"][pages].double().unsqueeze(-1)
            rows.append(x.transpose(0, 1).reshape(H, -1, D)[:, :n])
        score = torch.einsum("hgd,hnd->hgn", s["q"][b].double().view(H, -1, D), rows[0]) / math.sqrt(D)
        lse[b] = torch.logsumexp(score, -1).view(-1)
        share = torch.softmax(score, -1)
        out[b] = torch.einsum("hgn,hnd->hgd", share, rows[1]).reshape(Hq, D)
        if weights is not None:
            weights[b, :, :n] += share.sum(1)
    return {"out": out, "lse": lse} | ({} if weights is None else {"weights": weights})


def _exact_logprobs(s: dict) -> dict:
    got: dict = {"entropy": [], "logprobs": [], "top_ids": None, "top_logprobs": []}
    for x, t in zip(s["logits"].split(256), s["tokens"].split(256)):
        logp = torch.log_softmax(x.double(), -1)
        got["logprobs"].append(logp.gather(1, t.view(-1, 1)).view(-1))
        got["entropy"].append(torch.special.entr(logp.exp()).sum(-1))
        got["top_logprobs"].append(torch.topk(logp, s["top"], dim=-1).values)
    return {k: None if v is None else torch.cat(v) for k, v in got.items()}


def exact(case: dict, seed: int):
    """What ``run`` computes from numbers, from its definition in 64 bits;
    rows that are only moved, bytes of e4m3 rows and whole numbers have no
    value of their own here."""
    s = prepare(case, seed)
    if case["op"] == "decode":
        return _exact_decode(case, s)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    if case["op"] == "append" and case["kv"] == "e4m3":
        out: dict = {"k": None, "v": None, "lengths": None}
        table, lens = s["page_table"].tolist(), s["lengths"].tolist()
        starts = s["starts"].tolist() if s["starts"] is not None else list(range(case["batch"] + 1))
        for name, x in zip(("k_scales", "v_scales"), s["new"]):
            scale = (x.double().abs().amax(-1).clamp(min=1e-6) / 425.6).to(x.dtype).double()
            pool = s[name].double()
            for b, n in enumerate(lens):
                rows = scale[starts[b] : starts[b + 1]]
                at = 0
                while at < rows.shape[0]:  # a page at a time
                    pos = n + at
                    take = min(rows.shape[0] - at, case["page"] - pos % case["page"])
                    first = pos % case["page"]
                    pool[table[b][pos // case["page"]], :, first : first + take] = rows[at : at + take].T
                    at += take
            out[name] = pool
        return out
    return None
