"""Offline perplexity of a checkpoint over local text: no server, no network, no external harness.

Documents (strings) are tokenised, packed by the training packer into ``[rows, seq_len]`` batches with ``cu_seqlens``
(documents never attend across their borders, the first token of a document is not a target) and run through the model's
own loss head; the result is the token-weighted mean negative log-likelihood and its exponential. Works under tensor
parallelism as well (every rank calls it with the same documents). The reference evaluates through an external harness
over its HTTP server only (``scripts/eval.py:67-357``)."""
from __future__ import annotations

import json
import math
from typing import Dict, Iterable, Iterator, List, Optional, Tuple

import torch

from ..data.packing import pack_chunk_aligned


def iter_documents(files: Iterable[str], text_field: str = "content") -> Iterator[str]:
    """Documents of local files: ``.jsonl`` (one object per line, text under ``text_field`` or ``text``), ``.parquet``
    (same fields) and anything else as plain text (documents separated by blank lines)."""
    for f in files:
        f = str(f)
        if f.endswith(".parquet"):
            from ..data.streaming import iter_parquet_rows
            for row in iter_parquet_rows(f):
                t = row.get(text_field) or row.get("text")
                if t:
                    yield t
        elif f.endswith(".jsonl") or f.endswith(".json"):
            with open(f) as fh:
                for line in fh:
                    if line.strip():
                        row = json.loads(line)
                        t = row.get(text_field) or row.get("text")
                        if t:
                            yield t
        else:
            with open(f, errors="replace") as fh:
                for doc in fh.read().split("\n\n"):
                    if doc.strip():
                        yield doc


def piece_length(cfg, seq_len: int) -> int:
    """Tokens of a whole piece of a document: ``seq_len`` in whole chunks of the packer, one chunk at least."""
    return max(cfg.pack_chunk_size, seq_len // cfg.pack_chunk_size * cfg.pack_chunk_size)


@torch.no_grad()
def evaluate_perplexity(model, tokenizer, documents: Iterable[str], seq_len: int = 1024, batch_rows: int = 4,
                        max_tokens: Optional[int] = None) -> Dict[str, float]:
    """``{"nll", "perplexity", "tokens", "documents"}`` over ``documents``. Documents longer than ``seq_len`` are cut into
    pieces of ``seq_len`` tokens (each piece is scored on its own context)."""
    cfg = model.cfg
    dev = next(model.parameters()).device
    eos = getattr(tokenizer, "eos_token_id", None)
    chunk = cfg.pack_chunk_size
    seq_len = piece_length(cfg, seq_len)
    was_training = model.training
    model.eval()
    total_nll, total_tok, n_docs = 0.0, 0, 0
    pending: List[List[int]] = []

    def flush(final: bool):
        nonlocal total_nll, total_tok, pending
        while pending and (final or len(pending) >= 4 * batch_rows):
            take, pending = pending[:4 * batch_rows], pending[4 * batch_rows:]
            while take:
                # documents are placed largest first; whatever did not fit goes into the next batch
                ids, labels, cu, fitted = pack_chunk_aligned(take, seq_len, chunk, batch_rows, pad_id=0, eos_id=None,
                                                             return_placed=True)
                out = model(ids.to(dev), labels=labels.to(dev), cu_seqlens=cu.to(device=dev, dtype=torch.int32))
                n = int(out["n_valid"])
                if n > 0:
                    total_nll += float(out["loss"]) * n
                    total_tok += n
                fitted = set(fitted)
                take = [d for i, d in enumerate(take) if i not in fitted]
        return

    for text in documents:
        toks = tokenizer.encode(text, add_special_tokens=False)
        if eos is not None:
            toks = toks + [eos]
        if len(toks) < 2:
            continue
        n_docs += 1
        for s in range(0, len(toks), seq_len):
            piece = toks[s:s + seq_len]
            if len(piece) >= 2:
                pending.append(piece)
        flush(False)
        if max_tokens is not None and total_tok >= max_tokens:
            pending = []
            break
    flush(True)
    model.train(was_training)
    nll = total_nll / max(1, total_tok)
    return {"nll": nll, "perplexity": math.exp(min(nll, 700.0)), "tokens": total_tok, "documents": n_docs}


@torch.no_grad()
def score_documents(model, tokenizer, documents: Iterable[str], seq_len: int = 1024, batch_tokens: int = 8192,
                    top_logprobs: int = 0, max_tokens: Optional[int] = None) -> Iterator[Dict[str, object]]:
    """Scores of every token, a row for each piece of a document (cut at the same places as in ``evaluate_perplexity``, each piece
    on its own context): ``{"document", "tokens", "logprobs", "entropy"}`` and, with ``top_logprobs``, ``"top_tokens"`` /
    ``"top_logprobs"``. The first token of a piece has no score (null). Pieces run packed; a pass holds fewer than
    ``batch_tokens`` tokens and one piece. ``max_tokens``: ends with the piece that brings so many scores."""
    dev = next(model.parameters()).device
    eos = getattr(tokenizer, "eos_token_id", None)
    seq_len = piece_length(model.cfg, seq_len)
    w = model.mesh.tp
    was_training = model.training
    model.eval()
    pending: List[Tuple[int, List[int]]] = []
    seen = waiting = 0                                     # tokens scored or about to be, tokens in `pending`

    def flush() -> Iterator[Dict[str, object]]:
        nonlocal pending
        take, pending = pending, []
        if not take:
            return
        flat = [t for _, p in take for t in p]
        ends = [0]
        for _, p in take:
            ends.append(ends[-1] + len(p))
        pad = -len(flat) % w                               # a dummy document fills the stream up to even shards
        cu = ends + ([ends[-1] + pad] if pad else [])
        got = model.token_logprobs(torch.tensor(flat + [0] * pad, dtype=torch.long, device=dev),
                                   cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev), top_k=top_logprobs)
        cols = [x.tolist() if x is not None else None for x in got]
        for (doc, p), s, e in zip(take, ends, ends[1:]):
            row: Dict[str, object] = {"document": doc, "tokens": p, "logprobs": [None] + cols[0][s + 1:e], "entropy": [None] + cols[1][s + 1:e]}
            if top_logprobs:
                row["top_logprobs"], row["top_tokens"] = [None] + cols[2][s + 1:e], [None] + cols[3][s + 1:e]
            yield row

    try:
        for d, text in enumerate(documents):
            toks = tokenizer.encode(text, add_special_tokens=False)
            if eos is not None:
                toks = toks + [eos]
            for s in range(0, len(toks), seq_len):
                piece = toks[s:s + seq_len]
                if len(piece) >= 2:
                    pending.append((d, piece))
                    seen += len(piece) - 1
                    waiting += len(piece)
                    if waiting >= batch_tokens:
                        yield from flush()
                        waiting = 0
                if max_tokens is not None and seen >= max_tokens:
                    break
            if max_tokens is not None and seen >= max_tokens:
                break
        yield from flush()
    finally:                                               # (also of a caller that reads some of the rows only)
        model.train(was_training)
