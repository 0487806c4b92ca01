"""Candidate decoding of a token-VLA over a paged key-value cache.

The planner of the reference (``VLAEngine.plan``, src/repercep/models/vla.py:
229-258) samples N candidate action chunks that share one prompt and ranks
them.  This example runs that loop on the paged operators, on a decoder of
random weights:

  1. the prompt's K and V go into pages once (``paged.append``), and the prompt
     is attended to with the FP8 kernel (``ops.fp8_attention``);
  2. a long prompt is cut to a budget (``paged.evict``) by the attention weights
     that its last tokens gave it;
  3. every candidate's page table starts with the prompt's full pages, which
     all candidates share; each adds pages of its own for its action tokens;
  4. per step and layer: one row per candidate is appended, attended to
     (``paged.decode``), and the sampled tokens are scored
     (``scoring.token_logprobs``); the candidate of greatest total log
     probability wins.

    python examples/token_vla_decode.py [--candidates 64] [--tokens 8] [--prompt 512] [--kv e4m3]
"""

from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from repercep_runtime_b200 import ops, paged, scoring  # noqa: E402


@dataclass
class Config:
    layers: int = 2
    heads: int = 32
    kv_heads: int = 32
    head_dim: int = 128
    hidden: int = 512
    vocab: int = 32000
    page: int = 16


class Decoder:
    """A decoder of random weights: per layer a QKV and an output projection
    around the attention (bf16, residual), then the head."""

    def __init__(self, cfg: Config, seed: int = 0) -> None:
        self.cfg = cfg
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(rows: int, cols: int, scale: float = 1.0) -> torch.Tensor:
            return (torch.randn((rows, cols), generator=g, device="cuda") * (scale / rows**0.5)).bfloat16()

        width, kv = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim
        self.embed = torch.randn((cfg.vocab, cfg.hidden), generator=g, device="cuda").bfloat16()
        self.qkv = [weight(cfg.hidden, width + 2 * kv) for _ in range(cfg.layers)]
        self.out = [weight(width, cfg.hidden) for _ in range(cfg.layers)]
        self.head = weight(cfg.hidden, cfg.vocab, 2.0)

    def project(self, layer: int, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(tokens, heads, D) q and (tokens, kv_heads, D) k, v: views of one product."""
        c = self.cfg
        y = (x @ self.qkv[layer]).view(x.shape[0], c.heads + 2 * c.kv_heads, c.head_dim)
        return y[:, : c.heads], y[:, c.heads : c.heads + c.kv_heads], y[:, c.heads + c.kv_heads :]


class Pages:
    """The free pages of a pool; a page may belong to several tables."""

    def __init__(self, count: int) -> None:
        self.free = list(range(count))

    def take(self, n: int) -> list[int]:
        if n > len(self.free):
            raise RuntimeError(f"{n} pages wanted, {len(self.free)} free")
        got, self.free = self.free[:n], self.free[n:]
        return got

    def give(self, pages: list[int]) -> None:
        self.free.extend(pages)


def table_of(rows: list[list[int]]) -> torch.Tensor:
    width = max(len(r) for r in rows)
    return torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32).cuda()


@dataclass
class Plan:
    tokens: torch.Tensor  # (candidates, steps) sampled tokens
    logprobs: torch.Tensor  # (candidates, steps)
    entropy: torch.Tensor  # (candidates, steps)
    best: int  # the candidate of greatest total log probability
    kept: torch.Tensor | None  # prompt positions that the cut left, of the first layer


def plan(
    model: Decoder,
    prompt: torch.Tensor,
    candidates: int,
    steps: int,
    *,
    kv: torch.dtype = torch.bfloat16,
    budget: int | None = None,
    observe: int = 8,
    seed: int = 0,
) -> Plan:
    """Decodes ``candidates`` chunks of ``steps`` tokens after ``prompt`` (ids).

    ``budget``: at most that many prompt tokens stay per head, chosen by the
    attention weights of the prompt's last ``observe`` tokens; it and an uncut
    prompt have to fill whole pages, since all candidates share them."""
    c = model.cfg
    P = int(prompt.shape[0])
    stay = P if budget is None else min(P, budget)
    if stay % c.page:
        raise ValueError(f"{stay} prompt tokens do not fill pages of {c.page}")
    own = -(-steps // c.page)  # pages of a candidate's own
    prompt_pages = -(-P // c.page)
    x = model.embed[prompt]
    upto = torch.arange(1, P + 1, dtype=torch.int32, device="cuda")  # tokens of the prompt up to each
    kept = None
    caches, tables = [], []
    for layer in range(c.layers):
        pages = Pages(prompt_pages + stay // c.page + candidates * own)
        cache = paged.alloc(prompt_pages + stay // c.page + candidates * own, c.kv_heads, c.page, c.head_dim, kv)
        table_rows = pages.take(prompt_pages)
        table = table_of([table_rows])
        q, k, v = model.project(layer, x)
        lengths = torch.zeros(1, dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, P], dtype=torch.int32, device="cuda")
        lengths = paged.append(cache, k, v, table, lengths, starts=starts)
        group = c.heads // c.kv_heads
        rows = [t.transpose(0, 1).unsqueeze(0) for t in (q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1))]
        attended = ops.fp8_attention(*(t.contiguous() for t in rows), causal=True, scale_mode=ops.SCALE_PER_BLOCK128)
        if stay < P:
            # weights of the last tokens' queries: one call each, over the prompt up to its own token
            weights = torch.zeros((1, c.kv_heads, table.shape[1] * c.page), device="cuda")
            for t in range(max(0, P - observe), P):
                paged.decode(q[t : t + 1], cache, table, upto[t : t + 1], weights=weights)
            new_rows = pages.take(stay // c.page)
            cut = paged.evict(cache, table, lengths, weights, table_of([new_rows]), budget=stay, recent=observe)
            pages.give(table_rows)
            table_rows = new_rows
            kept = cut.kept if kept is None else kept
        x = x + attended[0].transpose(0, 1).reshape(P, -1) @ model.out[layer]
        caches.append(cache)
        tables.append(table_of([table_rows + pages.take(own) for _ in range(candidates)]))

    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = (x[-1:] @ model.head).expand(candidates, -1)
    lengths = torch.full((candidates,), stay, dtype=torch.int32, device="cuda")
    tokens, logprobs, entropy = [], [], []
    for _ in range(steps):
        token = torch.multinomial(torch.softmax(logits.float(), -1), 1, generator=gen)[:, 0]
        score = scoring.token_logprobs(logits.contiguous(), token, top=1)
        tokens.append(token)
        logprobs.append(score.logprobs)
        entropy.append(score.entropy)
        h = model.embed[token]
        after = lengths
        for layer in range(c.layers):
            q, k, v = model.project(layer, h)
            after = paged.append(caches[layer], k, v, tables[layer], lengths)
            out = paged.decode(q, caches[layer], tables[layer], after)
            h = h + out.view(candidates, -1) @ model.out[layer]
        lengths = after
        logits = h @ model.head
    total = torch.stack(logprobs, 1)
    return Plan(torch.stack(tokens, 1), total, torch.stack(entropy, 1), int(total.sum(1).argmax()), kept)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--candidates", type=int, default=64)
    ap.add_argument("--tokens", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--budget", type=int, default=None, help="prompt tokens to keep per head")
    ap.add_argument("--kv", choices=("bf16", "e4m3"), default="bf16", help="type of the cache")
    args = ap.parse_args()
    model = Decoder(Config())
    prompt = torch.randint(0, model.cfg.vocab, (args.prompt,), generator=torch.Generator().manual_seed(1)).cuda()
    kv = torch.bfloat16 if args.kv == "bf16" else paged.FP8
    got = plan(model, prompt, args.candidates, args.tokens, kv=kv, budget=args.budget)
    total = got.logprobs.sum(1)
    print(f"best candidate {got.best}: log probability {float(total[got.best]):.3f} "
          f"(mean {float(total.mean()):.3f}, mean entropy {float(got.entropy.mean()):.3f})")
    print("tokens", got.tokens[got.best].tolist())


if __name__ == "__main__":
    main()
