"""Token constraints: structured output by masking the logits before sampling.

``response_format = {"type": "json_object"}`` (or ``json_schema``, which is held to "a JSON object") makes the engine
keep a grammar state per row.  Before every step the state's allowed-token mask (computed natively over a byte trie of
the vocabulary, ``native/src/json_constraint.cpp``) becomes a row of bit words; where its bit is not set, a logit turns into a large
negative number ahead of the sampler, inside the captured graph of the step's processed variant, beside biases and penalties
(:class:`LogitTables`, ``ops.process_logits``); after the step the sampled token advances the state.  The end-of-sequence tokens
are allowed exactly when the document is complete, so a constrained request stops by itself on valid JSON.

Reference: engine token constraints + the tokenizer's grammar (``cpp_runtime/engine/include``: token constraints;
``cpp_runtime/components/tokenizer``: grammar), and ``response_format`` in the OpenAI-compatible request parser
(``mfq/server/api/openai_compat.py:125``).
"""

from __future__ import annotations

import math

import numpy as np
import torch

from .. import ops

PLACES_KEPT = 1024  # biases a row that tables keep room for: 64 rows of 128256 take 7.5 us with 8 places on a B200, 16.8 with 1024, 722 with 65536
NEG = -1.0e30  # representable in bf16; exp() of it is 0 and an arg-max never picks it


class JsonTokenConstraint:
    def __init__(self, vocabulary, stop_ids, need_object: bool = True) -> None:
        from .. import native
        self.vocabulary = vocabulary
        self.stop_ids = tuple(int(t) for t in stop_ids if t is not None and 0 <= int(t) < vocabulary.size)
        self.state = native.JsonState(vocabulary, need_object)
        self.finished = False

    def allowed(self) -> np.ndarray:
        mask = self.state.mask()
        if self.state.complete or not mask.any():  # complete, or a dead end (depth limit): let the request end
            mask[list(self.stop_ids)] = True
        return mask

    def biases(self, width: int) -> dict:
        return {}

    def words(self, width: int) -> torch.Tensor:
        """Bit words ``[ceil(width / 32)]`` int32: set where a token may come next (ids past the vocabulary, e.g. padding columns
        of the output projection, are never allowed)."""
        cache = self.vocabulary.__dict__.setdefault("_words_cache", {})
        key = (self.state.key, self.state.complete, self.stop_ids, width)
        hit = cache.get(key)
        if hit is not None:  # e.g. every step inside a string value: same state, same row
            return hit
        out = np.zeros((width + 31) // 32 * 32, dtype=np.uint8)
        mask = self.allowed()
        n = min(width, mask.size)
        out[:n] = mask[:n]
        row = torch.from_numpy(np.packbits(out, bitorder="little").view(np.int32).copy())
        if len(cache) >= 128:
            cache.pop(next(iter(cache)))
        cache[key] = row
        return row

    def advance(self, token: int) -> None:
        if self.finished:
            return
        if token in self.stop_ids or not self.state.feed_token(int(token)):
            self.finished = True


class LogitBias:
    """OpenAI ``logit_bias``: a fixed additive bias on chosen token ids for the whole request (values are clamped to
    +-100 as the API defines them); optionally on top of a grammar constraint."""

    def __init__(self, bias: dict, inner=None) -> None:
        self.table = {int(t): max(-100.0, min(100.0, float(v))) for t, v in bias.items()}
        self.inner = inner
        self.finished = False
        self._inside: dict[int, dict] = {}  # columns -> the biases of tokens that there are

    def biases(self, width: int) -> dict:
        """Token -> bias of the ids below ``width``, one dict for all steps: a request may name any id, what is no token has no logit."""
        if width not in self._inside:
            self._inside[width] = {t: v for t, v in self.table.items() if 0 <= t < width}
        return self._inside[width]

    def words(self, width: int) -> torch.Tensor | None:
        return self.inner.words(width) if self.inner is not None else None

    def advance(self, token: int) -> None:
        if self.inner is not None:
            self.inner.advance(token)
            self.finished = self.inner.finished


def make_constraint(response_format, vocabulary, stop_ids):
    """``response_format`` as the request carried it (a dict, a type string or None) -> a constraint or None."""
    if not response_format or vocabulary is None:
        return None
    kind = response_format.get("type") if isinstance(response_format, dict) else str(response_format)
    if kind in ("json_object", "json_schema", "json"):
        return JsonTokenConstraint(vocabulary, stop_ids, need_object=True)
    return None


def penalties(params) -> tuple[float, float, float]:
    """Presence, frequency and repetition penalty of a request.  What is no number, or no factor, penalizes nothing; what fp32 would make an infinity
    stays below it, so that no logit turns into a NaN."""
    def held(x: float, neutral: float) -> float:
        return neutral if math.isnan(x) else max(-1e30, min(1e30, x))

    repetition = held(params.repetition_penalty, 1.0)
    return held(params.presence_penalty, 0.0), held(params.frequency_penalty, 0.0), max(1e-30, repetition) if repetition > 0.0 else 1.0


def penalized(params) -> bool:
    """Whether a request penalizes tokens that it has already."""
    return params is not None and penalties(params) != (0.0, 0.0, 1.0)


class LogitTables:
    """What ``ops.process_logits`` reads beside the sampling records, a row per batch row: token counts, biases and allowed tokens."""

    def __init__(self, rows: int, width: int, device: torch.device) -> None:
        self.width = width
        self.counts = torch.zeros((rows, width), dtype=torch.int16, device=device)
        self.counted = torch.full((rows,), -1, dtype=torch.int32, device=device)  # the rows whose token a step counts
        self.allowed = torch.full((rows, (width + 31) // 32), -1, dtype=torch.int32, device=device)
        self._held: dict[int, tuple] = {}  # row -> the host's words and biases that its rows hold (None: no limit)
        self.make_places(8)

    def make_places(self, places: int, tables: int = 1) -> None:
        """Room for ``places`` biases a row in each of ``tables`` tables; the biases are written again by the next :meth:`limit`."""
        most = 8
        while most < places:
            most *= 2
        if most > ops.MAX_BIASES:
            raise ValueError(f"a table has at most {ops.MAX_BIASES} biases a row, got {places}")
        rows, dev = self.counts.shape[0], self.counts.device
        self.biases = [(torch.full((rows, most), -1, dtype=torch.int32, device=dev), torch.zeros((rows, most), dtype=torch.float32, device=dev))
                       for _ in range(tables)]
        self._held = {r: (w, None) for r, (w, _) in self._held.items()}

    @property
    def bias_ids(self) -> torch.Tensor:
        return self.biases[0][0]

    def make_room(self, places: int) -> bool:
        """Room for ``places`` biases a row, in several tables where one is not allowed as many; whether the tables are other ones now.  Many places are given
        back once a quarter is enough: the kernel goes over all of them in every row."""
        have = sum(ids.shape[1] for ids, _ in self.biases)
        if places <= have and (have <= PLACES_KEPT or places > have // 4):
            return False
        tables = max(1, -(-places // ops.MAX_BIASES))
        self.make_places(places if tables == 1 else ops.MAX_BIASES, tables)
        return True

    def limit(self, row: int, constraint) -> None:
        """Bring row ``row`` in line with a constraint (None: no limits)."""
        words, table = (None, {}) if constraint is None else (constraint.words(self.width), constraint.biases(self.width))
        held_words, held_table = self._held.get(row, (None, {}))
        parts = None
        if table is not held_table and not (held_table == {} and not table):
            parts, at = [], 0
            for ids, _ in self.biases:
                part = list(table.items())[at : at + ids.shape[1]]
                at += len(part)
                # held as the bf16 numbers that logits had added before there was a kernel for it
                parts.append((torch.tensor([t for t, _ in part], dtype=torch.int32), torch.tensor([v for _, v in part], dtype=torch.float32).to(torch.bfloat16).float()))
        self._held[row] = (self, None)  # neither is what the row holds, should a write fail
        if words is not held_words:  # the words of a grammar state are one tensor: within a string, say, the device has them already
            if words is None:
                self.allowed[row].fill_(-1)
            else:
                self.allowed[row].copy_(words, non_blocking=True)
        for (ids, values), (tokens, biases) in zip(self.biases, parts or ()):
            ids[row].fill_(-1)
            if tokens.numel():
                ids[row, : tokens.numel()] = tokens.to(ids.device)
                values[row, : tokens.numel()] = biases.to(values.device)
        self._held[row] = (words, table)
