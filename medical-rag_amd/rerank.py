"""Re-ranking of retrieved pages by query likelihood: the pages after which a causal
language model finds the query most likely come first.

The reference re-ranks with an engine that returns the log probabilities of answer
tokens (pipeline/utils/reranker.py, pipeline/utils/vllm_handler.py:109-144).  Here the
decoder's body is a PyTorch(-ROCm) forward, as the encoder's is; its last steps run in
the library's kernels: the final norm into microscaled 8-bit rows, the product with the
vocabulary matrix held in microscaled 4-bit (a quarter of its bfloat16 bytes), the log
probabilities of the query's tokens.  Only the positions that predict a query token go
through them.  There is no CPU form.

    rerank_pages(query, hits, pages, model_name, device) -> (positions, scores), best first
    rerank_hits(hits_by_keyword, pages, model_name, ...) -> the same dict, every list re-ordered
    ScoringHead.from_model(model)                        the last steps of a loaded model
"""
from __future__ import annotations

import logging
import threading

import numpy as np
import torch

from . import scoring

__all__ = ["ScoringHead", "page_scores", "rerank_pages", "rerank_hits"]

MAX_LENGTH = 8192       # tokens of a page and a query together, where the model takes as many: what the index builder truncates pages to
SEPARATOR = "\n\n"      # between the page and the query


_FORWARD = threading.Lock()     # one forward of a model at a time: the hook sees every one of them


class ScoringHead:
    """The last steps of a causal language model on one GPU: root-mean-square norm with
    `norm_weight` and `eps`, then logits against `vocabulary` (MxRows in mxfp4, one row
    a token).  Calls take (n, d) rows of the decoder's last hidden states BEFORE the
    final norm, with `residual` added first if given."""

    def __init__(self, norm_weight, eps: float, vocabulary: "scoring.MxRows"):
        if vocabulary.format != "mxfp4" or norm_weight.shape != (vocabulary.d,) or norm_weight.device != vocabulary.device:
            raise ValueError("ScoringHead wants a vocabulary in mxfp4 and a norm weight of its width on its GPU")
        self.norm_weight, self.eps, self.vocabulary = norm_weight.detach(), float(eps), vocabulary

    @classmethod
    def from_model(cls, model):
        """Of a Hugging Face causal language model on a GPU: its body's `norm` and its
        output embeddings, quantised once.  ValueError for heads that compute something
        else: a norm that is not a plain root-mean-square norm, a bias, scaled or capped
        logits."""
        norm, out = _body(model).norm, model.get_output_embeddings()
        config = model.config
        if out is None or getattr(out, "bias", None) is not None:
            raise ValueError("the model's output embeddings are missing or have a bias")
        if getattr(config, "final_logit_softcapping", None) or getattr(config, "logits_scaling", 1.0) != 1.0 \
                or getattr(config, "logit_scale", None) not in (None, 1.0):
            raise ValueError("the model scales or caps its logits")
        weight = getattr(norm, "weight", None)
        eps = getattr(norm, "variance_epsilon", getattr(norm, "eps", None))
        if weight is None or eps is None or weight.dim() != 1:
            raise ValueError("the model's final norm is no root-mean-square norm")
        with torch.no_grad():
            x = torch.linspace(-2, 3, weight.numel(), device=weight.device).to(weight.dtype)[None]
            want = x.double() / (x.double().square().mean() + eps).sqrt() * weight.double()
            if not torch.allclose(norm(x).double(), want, rtol=2e-2, atol=2e-2):
                raise ValueError("the model's final norm is no plain root-mean-square norm")
            # its logits of a few tokens against the same steps on the states in front of its norm: 2e-2 of the largest
            # one is what roundings to 16 bits leave
            ids = torch.arange(min(8, out.weight.shape[0]), device=weight.device)[None]
            states, result = _states(model, model, ids)
            logits = (result.logits if hasattr(result, "logits") else result[0])[0, -1].double()
            want = torch.nn.functional.linear(norm(states[0, -1:]), out.weight)[0].double()
            if logits.shape != want.shape or not bool(((logits - want).abs() <= 2e-2 * want.abs().max()).all()):
                raise ValueError("the model's logits are not its final norm times its output embeddings")
            return cls(weight, eps, scoring.mx_quantize(out.weight.detach(), "mxfp4"))

    def logits(self, hidden, residual=None, dtype=torch.float32):
        """(n, vocabulary) logits of `dtype` (float32 or bfloat16)."""
        rows, _ = scoring.rms_norm_mx(hidden, self.norm_weight, self.eps, residual)
        return scoring.mx_matmul(rows, self.vocabulary, dtype)

    def token_logprobs(self, hidden, tokens, top_k: int = 0, residual=None) -> "scoring.TokenLogprobs":
        """Log probabilities of `tokens`, entropy and the top_k alternatives for each
        row, the logits in float32 and never more than about 2 GB of them at a time."""
        step = max(1, (2 << 30) // (4 * len(self.vocabulary)))
        if len(hidden) <= step:
            return scoring.token_logprobs(self.logits(hidden, residual), tokens, top_k)
        cut = lambda t, lo: None if t is None else t[lo:lo + step]  # noqa: E731
        parts = [scoring.token_logprobs(self.logits(cut(hidden, lo), cut(residual, lo)), cut(tokens, lo), top_k)
                 for lo in range(0, len(hidden), step)]
        return scoring.TokenLogprobs(*(torch.cat(p) for p in zip(*parts)))


def _body(model):
    """The decoder under a causal language model's head, which ends with `norm`."""
    body = getattr(model, "model", None)
    if body is None or not hasattr(body, "norm"):
        raise ValueError(f"{type(model).__name__} has no decoder body that ends with a norm")
    return body


def _states(model, module, ids, **inputs):
    """What goes into the norm that ends the decoder's body, (rows, tokens, width), and what `module` (the model
    or its body) returns."""
    captured = []
    with _FORWARD, torch.no_grad():
        hook = _body(model).norm.register_forward_pre_hook(lambda _, args: captured.append(args[0]))
        try:
            result = module(input_ids=ids, use_cache=False, **inputs)
        finally:
            hook.remove()
    if not captured:
        raise ValueError(f"{type(model).__name__} does not go through its body's norm")
    return captured[-1], result


def _context(model) -> int | None:
    """How many positions the model was made for; None where its configuration does not say."""
    config = model.config.get_text_config() if hasattr(model.config, "get_text_config") else model.config
    limit = getattr(config, "max_position_embeddings", None)
    return limit if isinstance(limit, int) and limit > 0 else None


def _sequences(page_ids: list, query_ids: list, separator_ids: list, start_ids: list, max_length: int):
    """Token lists [start, page, separator, query], the page cut so that the whole is at
    most max_length long, and where each one's query begins."""
    room = max_length - len(start_ids) - len(separator_ids) - len(query_ids)
    if room < 0:
        raise ValueError(f"the query has {len(query_ids)} tokens, more than fit {max_length}")
    rows = [start_ids + ids[:room] + separator_ids + query_ids for ids in page_ids]
    return rows, [len(r) - len(query_ids) for r in rows]


def page_scores(query: str, texts: list, model, tokenizer, head: ScoringHead, batch_size: int = 8, max_length: int = MAX_LENGTH) -> list:
    """Mean log probability of the query's tokens after each text, in nats.  Texts are
    cut so that they and the query fit max_length tokens and the model's positions; NaN
    for all of them where the query alone does not."""
    encode = lambda t: list(tokenizer(t, add_special_tokens=False)["input_ids"])  # noqa: E731
    query_ids = encode(query)
    if not query_ids or not texts:
        return [0.0] * len(texts)
    start = tokenizer.bos_token_id if tokenizer.bos_token_id is not None else tokenizer.cls_token_id
    if start is None:
        start = tokenizer.eos_token_id
    # without any such token an empty page leaves nothing before the query's first one
    start_ids = [start] if start is not None else query_ids[:1]
    separator_ids, limit = encode(SEPARATOR), min(max_length, _context(model) or max_length)
    if len(start_ids) + len(separator_ids) + len(query_ids) > limit:
        logging.error(f"A query of {len(query_ids)} tokens does not fit the {limit} of the re-ranking model: its pages keep their order.")
        return [float("nan")] * len(texts)
    rows, begins = _sequences([encode(t) for t in texts], query_ids, separator_ids, start_ids, limit)
    body, q = _body(model), len(query_ids)
    device = head.vocabulary.device
    scores = []
    with torch.no_grad():
        tokens = torch.tensor(query_ids, device=device)
        for lo in range(0, len(rows), batch_size):
            part, at = rows[lo:lo + batch_size], begins[lo:lo + batch_size]
            longest = max(map(len, part))
            ids = torch.zeros((len(part), longest), dtype=torch.int64)
            mask = torch.zeros((len(part), longest), dtype=torch.int64)
            for i, r in enumerate(part):
                ids[i, :len(r)], mask[i, :len(r)] = torch.tensor(r), 1
            hidden, _ = _states(model, body, ids.to(device), attention_mask=mask.to(device))
            # the state at a position predicts the next token: from the one before the query to its last but one
            where = (torch.tensor(at)[:, None] - 1 + torch.arange(q)[None]).to(device)
            picked = hidden.gather(1, where[:, :, None].expand(-1, -1, hidden.shape[2])).reshape(-1, hidden.shape[2])
            lp = head.token_logprobs(picked, tokens.repeat(len(part))).logprobs
            scores.append(lp.reshape(len(part), q).mean(dim=1))
    return torch.cat(scores).tolist()


_MODEL = {"key": None, "model": None, "tokenizer": None, "head": None, "refused": None}
_LOADING = threading.Lock()


def _model_for(model_name: str, device: str):
    with _LOADING:
        return _load(model_name, device)


def _load(model_name: str, device: str):
    key = (model_name, device)
    if _MODEL["key"] == key:
        if _MODEL["refused"]:
            raise ValueError(_MODEL["refused"])
        return _MODEL["model"], _MODEL["tokenizer"], _MODEL["head"]
    from transformers import AutoModelForCausalLM, AutoTokenizer
    logging.info(f"Loading re-ranking model '{model_name}' onto device '{device}'.")
    try:
        tokenizer = AutoTokenizer.from_pretrained(model_name)
        model = AutoModelForCausalLM.from_pretrained(model_name).to(device).eval()
    except Exception as exc:  # the encoder's soft failure (pipeline/utils/local_rag.py:34-37)
        logging.error(f"Failed to load re-ranking model '{model_name}': {exc}", exc_info=True)
        _MODEL.update(key=None, model=None, tokenizer=None, head=None, refused=None)
        return None, None, None
    try:
        head = ScoringHead.from_model(model)
    except ValueError as exc:       # remembered: loading the same model again would end here again
        _MODEL.update(key=key, model=None, tokenizer=None, head=None, refused=str(exc))
        raise
    _MODEL.update(key=key, model=model, tokenizer=tokenizer, head=head, refused=None)
    return model, tokenizer, head


def rerank_pages(query: str, hits, pages, model_name: str, device: str = "cuda", batch_size: int = 8):
    """List positions `hits` of `pages` in the order of how likely the model finds the
    query after each page, and those scores (mean log probability a query token), both
    numpy arrays; equal scores keep their order, padding (position -1) is dropped.
    When the model cannot be loaded, or the query has more tokens than it takes, the hits
    come back as they are, with NaN scores."""
    hits = [int(h) for h in np.asarray(hits).reshape(-1) if 0 <= int(h) < len(pages)]
    if not hits:
        return np.empty(0, np.int64), np.empty(0, np.float32)
    if not str(device).startswith("cuda"):
        raise ValueError("re-ranking runs on a GPU only")
    model, tokenizer, head = _model_for(model_name, device)
    if model is None:
        return np.array(hits, np.int64), np.full(len(hits), np.nan, np.float32)
    scores = np.array(page_scores(query, [pages[h].get("text", "") for h in hits], model, tokenizer, head, batch_size), np.float32)
    order = np.argsort(-scores, kind="stable")
    return np.array(hits, np.int64)[order], scores[order]


def rerank_hits(hits: dict, pages, model_name: str, device: str = "cuda", top_k: int | None = None, batch_size: int = 8) -> dict:
    """What caller.top_pages_for_keywords or top_pages_for_texts returns -- keyword ->
    (positions, scores) -- with every keyword's positions re-ranked and the best top_k
    kept (all of them unless given)."""
    out = {}
    for keyword, (idx, _) in hits.items():
        idx, scores = rerank_pages(keyword, idx, pages, model_name, device, batch_size)
        out[keyword] = (idx[:top_k], scores[:top_k])
    return out
