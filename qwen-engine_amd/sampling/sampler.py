"""Choice of the next token: greedy (the reference's only rule,
src/engine/executor.py:51-54: argmax, lowest index on ties) and temperature
sampling (not in the reference).

Temperature sampling draws by inverse CDF from softmax(logits / temperature) with
one uniform number per request and output position.  The number comes from a hash
of (seed, request, position), so a request's tokens do not depend on what else is
in the batch, on the order of requests or on preemption.

Drafted tokens (not in the reference either) are verified against the logits behind them:
each is kept with the probability that makes the tokens distributed as if drawn one by one.
"""
from __future__ import annotations

import hashlib
import struct
from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch

from ..kernels import ops


@dataclass
class SamplingParams:
    max_new_tokens: int = 16
    temperature: float = 0.0     # 0: greedy
    seed: int = 0
    ignore_eos: bool = False

    def validate(self) -> None:
        if self.max_new_tokens <= 0:
            raise ValueError("max_new_tokens must be positive")
        if self.temperature < 0:
            raise ValueError("temperature must not be negative")


def uniform_for(seed: int, request_key: int, position: int, purpose: str = "") -> float:
    """A number in [0, 1) with 24 random bits, fixed by (seed, request, output position) and what it is for
    (at most 16 bytes of text): a position whose token was drafted needs one for the draft, one for accepting
    it and one for the token in its place, which must not hang together."""
    digest = hashlib.blake2b(struct.pack("<qqq", int(seed), int(request_key), int(position)),
                             digest_size=8, person=purpose.encode()).digest()
    return (int.from_bytes(digest, "little") >> 40) / float(1 << 24)


class Sampler:
    """Runs the sampling kernels on the logits of one step."""

    def sample(self, logits: torch.Tensor, temperatures: Sequence[float], uniforms: Sequence[float]) -> List[int]:
        """logits float32 [R, V] on the device; one temperature and one uniform per row."""
        R = logits.shape[0]
        if R == 0:
            return []
        if len(temperatures) != R or len(uniforms) != R:
            raise ValueError("one temperature and one uniform number per row are needed")
        greedy = ops.argmax(logits)
        if all(t <= 0 for t in temperatures):
            return [int(v) for v in greedy.tolist()]
        temps = torch.tensor([t if t > 0 else 1.0 for t in temperatures], dtype=torch.float32).to(logits.device)
        us = torch.tensor(list(uniforms), dtype=torch.float32).to(logits.device)
        drawn = ops.sample(logits, temps, us)
        g, d = greedy.tolist(), drawn.tolist()
        return [int(d[i]) if temperatures[i] > 0 else int(g[i]) for i in range(R)]

    def verify(self, logits: torch.Tensor, drafts: Sequence[Sequence[int]], draft_logits: Optional[torch.Tensor],
               temperatures: Sequence[float], accept_uniforms: Sequence[Sequence[float]],
               draw_uniforms: Sequence[float]) -> List[List[int]]:
        """The tokens that every request gets from one step over its drafts: those that stand, and one more.  logits float32
        on the device, for each request one row more than it has drafts (row j: behind j of them), the requests one after
        another; draft_logits float32, a row a draft in the same order: what the drafts were drawn from at the same
        temperatures (None: looked up, not drawn).  One number in [0, 1) a draft, and one a request."""
        R, rows = len(drafts), sum(len(d) + 1 for d in drafts)
        if R == 0:
            return []
        if len(temperatures) != R or len(accept_uniforms) != R or len(draw_uniforms) != R or \
                any(len(d) != len(u) for d, u in zip(drafts, accept_uniforms)):
            raise ValueError("one temperature and one uniform number per request and one per draft are needed")
        if logits.shape[0] != rows:
            raise ValueError(f"{rows} rows of logits are needed, one more per request than it has drafts")
        if any(not -2 ** 31 <= t < 2 ** 31 for d in drafts for t in d):
            raise ValueError("a draft is no token id")
        first = [0]
        for d in drafts:
            first.append(first[-1] + len(d) + 1)
        flat = [t for d in drafts for t in d]
        # (two copies to the device: the whole numbers, and the others)
        whole = torch.tensor(first + flat, dtype=torch.int32).to(logits.device)
        other = torch.tensor(list(temperatures) + list(draw_uniforms) + [u for us in accept_uniforms for u in us],
                             dtype=torch.float32).to(logits.device)
        tokens, accepted = ops.verify_drafts(logits, whole[:R + 1], whole[R + 1:], draft_logits, other[:R], other[2 * R:], other[R:2 * R])
        got, kept = tokens.tolist(), accepted.tolist()
        return [got[first[r]:first[r] + kept[r] + 1] for r in range(R)]
