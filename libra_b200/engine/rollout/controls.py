"""What a rollout engine keeps to run ``ops.control_logits`` on its batches:
token histories on the device, biases and grammar masks on the host.

A request that uses a penalty owns a row of one int32 table [rows, width] for
as long as it runs.  Its prompt goes up once and every step adds the tokens
since the last one, so a step moves a few bytes a request whatever the
history's length; the kernel counts the occurrences itself.  Masks and biases
are small and go up with the step that uses them, through pinned memory.
"""

from __future__ import annotations

from typing import Dict, List, Optional, Protocol, Sequence

import torch

from libra_b200 import ops


class Grammar(Protocol):
    """Restricts a request's next token (``SamplingParams.grammar``)."""

    def fill_mask(self, output_tokens: List[int], words: torch.Tensor) -> None:
        """Set, in the zeroed int32 ``words`` [ceil(V / 32)], bit v % 32 of word
        v // 32 for every token v that may follow ``output_tokens``
        (``allow_tokens`` does it for a list of ids).  Setting none ends the
        request with finish reason "grammar"."""


def allow_tokens(words: torch.Tensor, ids: Sequence[int], vocab_size: int) -> None:
    """Set the bits of ``ids`` (those inside the vocabulary) in a mask row."""
    allowed = torch.zeros(words.numel() * 32, dtype=torch.int64)
    try:
        t = torch.as_tensor(list(ids), dtype=torch.int64)
    except (RuntimeError, ValueError, OverflowError):  # an id beyond 64 bits is outside every vocabulary
        t = torch.as_tensor([int(i) for i in ids if 0 <= i < vocab_size], dtype=torch.int64)
    allowed[t[(t >= 0) & (t < vocab_size)]] = 1
    bits = (allowed.view(-1, 32) << torch.arange(32)).sum(1)
    words |= torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)


class LogitControls:
    """The controls of one engine's requests (any object with ``request_id``,
    ``params``, ``out``, ``prompt``, ``n_tokens`` and ``token_slice``)."""

    def __init__(self, vocab_size: int, max_rows: int, device):
        self.V, self.max_rows, self.device = int(vocab_size), int(max_rows), torch.device(device)
        self.words = (self.V + 31) // 32
        self.table: Optional[torch.Tensor] = None
        self._row: Dict[str, int] = {}      # request id -> table row
        self._sent: Dict[str, int] = {}     # tokens of it that are in the table
        self._free: List[int] = list(range(self.max_rows))
        self._static: Dict[str, torch.Tensor] = {}   # masks of allowed_token_ids
        self._mask: Dict[str, torch.Tensor] = {}     # this step's mask of every masked request
        self.h2d = 0

    def release(self, request_id: str) -> None:
        row = self._row.pop(request_id, None)
        if row is not None:
            self._free.append(row)
        for d in (self._sent, self._static, self._mask):
            d.pop(request_id, None)

    # ------------------------------------------------------------------ masks
    def prepare(self, req) -> str:
        """The mask of a request's next token, on the host before the step runs.
        Returns the finish reason if there is none to take ("grammar", or
        "grammar_error" where building it raised), else ""."""
        try:
            words = self._build_mask(req)
        except Exception as exc:  # noqa: BLE001 - the caller's code and values; only its own request ends
            print(f"request {req.request_id}: grammar failed: {exc}")
            return "grammar_error"
        if words is None:
            return ""
        self._mask[req.request_id] = words
        return "" if bool(words.any()) else "grammar"

    def _build_mask(self, req) -> Optional[torch.Tensor]:
        p, rid = req.params, req.request_id
        words = None
        if p.grammar is not None:
            words = torch.zeros(self.words, dtype=torch.int32)
            p.grammar.fill_mask(list(req.out), words)
            if self.V % 32:
                words[-1] &= (1 << (self.V % 32)) - 1
        if p.allowed_token_ids is not None:
            if rid not in self._static:
                static = torch.zeros(self.words, dtype=torch.int32)
                allow_tokens(static, p.allowed_token_ids, self.V)
                self._static[rid] = static
            words = self._static[rid] if words is None else words & self._static[rid]
        return words

    # ------------------------------------------------------------------ histories
    def _up(self, t: torch.Tensor) -> torch.Tensor:
        if self.device.type != "cuda":
            return t.to(self.device)
        self.h2d += t.numel() * t.element_size()
        return t.pin_memory().to(self.device, non_blocking=True)

    def _grow(self, need: int) -> None:
        width = 4096 if self.table is None else self.table.shape[1]
        while width < need:
            width *= 2
        if 16384 < need <= 32760:
            width = 32760  # the kernel counts histories below 32768 in 16 bits
        if self.table is None or width != self.table.shape[1]:
            new = torch.zeros(self.max_rows, width, dtype=torch.int32, device=self.device)
            if self.table is not None:
                new[:, :self.table.shape[1]] = self.table
            self.table = new

    def _send_histories(self, reqs) -> None:
        need = max(r.n_tokens for r in reqs)
        if self.table is None or need > self.table.shape[1]:
            self._grow(need)
        at, vals = [], []
        for r in reqs:
            rid = r.request_id
            if rid not in self._row:
                self._row[rid], self._sent[rid] = self._free.pop(), 0
            row, sent, n = self._row[rid], self._sent[rid], r.n_tokens
            new = r.token_slice(sent, n)
            if len(new) > 256:
                self.table[row, sent:n].copy_(self._up(torch.tensor(new, dtype=torch.int32)))
            else:
                at.extend(range(row * self.table.shape[1] + sent, row * self.table.shape[1] + n))
                vals.extend(new)
            self._sent[rid] = n
        if at:
            self.table.view(-1)[self._up(torch.tensor(at, dtype=torch.long))] = self._up(
                torch.tensor(vals, dtype=torch.int32))

    # ------------------------------------------------------------------ one step
    def apply(self, logits: torch.Tensor, reqs) -> torch.Tensor:
        """``logits`` [B, V] of ``reqs`` with their controls, fp32 (rows padded
        to a multiple of 8 for the samplers' aligned loads).  ``prepare`` must
        have run for every request of the batch."""
        B = len(reqs)
        ps = [r.params for r in reqs]
        kw = {}
        pen = [r for r in reqs if r.params.penalized]
        if pen:
            self._send_histories(pen)
            f = self._up(torch.tensor([[p.repetition_penalty for p in ps], [p.presence_penalty for p in ps],
                                       [p.frequency_penalty for p in ps]], dtype=torch.float32))
            i = self._up(torch.tensor([[self._row.get(r.request_id, 0) for r in reqs],
                                       [r.n_tokens if r.params.penalized else 0 for r in reqs],
                                       [len(r.prompt) for r in reqs]], dtype=torch.int32))
            # the table as wide as this batch needs it: the kernel takes smaller counters for short histories, and the
            # table keeps the width of the longest request it ever held
            kw.update(history=self.table[:, :max(r.n_tokens for r in pen)], history_rows=i[0], history_lens=i[1], prompt_lens=i[2], repetition=f[0],
                      presence=f[1], frequency=f[2])
        if any(p.logit_bias for p in ps):
            offs, ids, vals = [0], [], []
            for p in ps:
                ids.extend(p.logit_bias or ())
                vals.extend((p.logit_bias or {}).values())
                offs.append(len(ids))
            kw.update(bias_offsets=self._up(torch.tensor(offs, dtype=torch.int32)),
                      bias_ids=self._up(torch.tensor(ids, dtype=torch.int32)),
                      bias_values=self._up(torch.tensor(vals, dtype=torch.float32)))
        masked = [r.request_id for r in reqs if r.request_id in self._mask]
        if masked:
            rows = {rid: n for n, rid in enumerate(masked)}
            kw.update(mask=self._up(torch.stack([self._mask[rid] for rid in masked])),
                      mask_rows=self._up(torch.tensor([rows.get(r.request_id, -1) for r in reqs], dtype=torch.int32)))
        out = torch.empty(B, -(-self.V // 8) * 8, dtype=torch.float32, device=logits.device)[:, :self.V]
        return ops.control_logits(logits, out=out, **kw)
