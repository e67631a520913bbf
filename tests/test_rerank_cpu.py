"""Re-ranking: what needs no GPU (token arrangement, conventions, refusals)."""
import logging
from types import SimpleNamespace

import numpy as np
import pytest
import torch


def test_sequences_cut_the_page_and_never_the_query():
    from medical_rag_amd.rerank import _sequences
    rows, begins = _sequences([[1, 2, 3], [], [4] * 50], [7, 8], [9], [0], 10)
    assert rows == [[0, 1, 2, 3, 9, 7, 8], [0, 9, 7, 8], [0] + [4] * 6 + [9, 7, 8]]
    assert begins == [5, 2, 8] and all(len(r) <= 10 and r[b:] == [7, 8] for r, b in zip(rows, begins))
    with pytest.raises(ValueError):
        _sequences([[1]], [7] * 10, [9], [0], 10)


def test_no_hits_and_no_model():
    from medical_rag_amd import rerank
    pages = [{"index": i, "text": f"page {i}"} for i in range(4)]
    for hits in ([], np.array([-1, -1]), [9]):
        idx, scores = rerank.rerank_pages("q", hits, pages, "unused")
        assert idx.shape == (0,) and scores.shape == (0,)
    with pytest.raises(ValueError):
        rerank.rerank_pages("q", [1, 2], pages, "unused", device="cpu")
    logging.disable(logging.CRITICAL)
    try:
        idx, scores = rerank.rerank_pages("q", [2, -1, 0], pages, "/nonexistent/model/dir")
    finally:
        logging.disable(logging.NOTSET)
    assert idx.tolist() == [2, 0] and np.isnan(scores).all()
    assert rerank.rerank_hits({}, pages, "unused") == {}


def tiny_llama(**extra):
    from transformers import LlamaConfig, LlamaForCausalLM
    return LlamaForCausalLM(LlamaConfig(vocab_size=64, hidden_size=32, intermediate_size=48, num_hidden_layers=1, num_attention_heads=2,
                                        num_key_value_heads=2, max_position_embeddings=64, **extra)).eval()


def test_heads_that_compute_something_else_are_refused():
    from medical_rag_amd.rerank import ScoringHead

    class Centred(torch.nn.Module):
        def __init__(self, weight):
            super().__init__()
            self.weight, self.eps = weight, 1e-6

        def forward(self, x):
            return torch.nn.functional.layer_norm(x, x.shape[-1:], self.weight)

    for change in (lambda m: setattr(m.model, "norm", Centred(m.model.norm.weight)), lambda m: setattr(m.config, "final_logit_softcapping", 30.0),
                   lambda m: setattr(m.config, "logit_scale", 0.5), lambda m: setattr(m.model, "norm", torch.nn.Identity()),
                   lambda m: setattr(m, "lm_head", torch.nn.Linear(32, 64, bias=True)), lambda m: delattr(m.model, "norm")):
        model = tiny_llama()
        change(model)
        with pytest.raises(ValueError):
            ScoringHead.from_model(model)
    with pytest.raises(ValueError):     # a plain head, but not on a GPU
        ScoringHead.from_model(tiny_llama())


class Characters:
    """A tokenizer of one token a character."""
    bos_token_id, cls_token_id, eos_token_id = 1, None, None

    def __call__(self, text, add_special_tokens):
        return {"input_ids": [2 + ord(c) % 60 for c in text]}


class PlainHead:
    """What ScoringHead does, in torch on any device."""

    def __init__(self, model):
        self.model = model
        self.vocabulary = model.get_output_embeddings().weight

    def token_logprobs(self, hidden, tokens):
        from medical_rag_amd.scoring import TokenLogprobs
        logits = self.model.get_output_embeddings()(self.model.model.norm(hidden))
        return TokenLogprobs(torch.log_softmax(logits.double(), 1).gather(1, tokens[:, None]), None, None, None)


def test_pages_are_cut_to_the_models_positions():
    """The tiny model has 64: a longer page is scored as its beginning that fits, and no forward is longer."""
    from medical_rag_amd import rerank
    torch.manual_seed(0)
    model = tiny_llama()
    seen = []
    model.model.register_forward_pre_hook(lambda module, args, kwargs: seen.append(kwargs["input_ids"].shape[1]), with_kwargs=True)
    page, query = "".join(chr(97 + i * 7 % 26) for i in range(500)), "a query"
    room = 64 - 1 - len(rerank.SEPARATOR) - len(query)
    head = PlainHead(model)
    long, cut, short = rerank.page_scores(query, [page, page[:room], page[:room - 20]], model, Characters(), head)
    assert max(seen) == 64 and long == cut and cut != short
    assert rerank.page_scores(query, [page], model, Characters(), head, max_length=40) == pytest.approx(
        rerank.page_scores(query, [page[:room - 24]], model, Characters(), head))
    bare = lambda **settings: SimpleNamespace(config=SimpleNamespace(**settings))  # noqa: E731
    assert rerank._context(model) == 64 and rerank._context(bare(max_position_embeddings=9)) == 9
    assert rerank._context(bare()) is None and rerank._context(bare(max_position_embeddings=None)) is None     # not every configuration says


def test_a_query_that_does_not_fit_keeps_its_own_order_and_the_others_theirs(monkeypatch):
    from medical_rag_amd import rerank
    torch.manual_seed(0)
    model = tiny_llama()
    monkeypatch.setattr(rerank, "_model_for", lambda name, device: (model, Characters(), PlainHead(model)))
    pages = [{"index": i, "text": "page %d about it" % i} for i in range(5)]
    long, fits = "x" * 64, "y" * (64 - 1 - len(rerank.SEPARATOR))
    hits = {"first": ([0, 1, 2], None), long: ([4, -1, 2, 3], None), fits: ([1, 0], None), "last": ([3, 4], None)}
    logging.disable(logging.CRITICAL)
    try:
        out = rerank.rerank_hits(hits, pages, "unused")
    finally:
        logging.disable(logging.NOTSET)
    assert list(out) == list(hits)
    assert out[long][0].tolist() == [4, 2, 3] and np.isnan(out[long][1]).all() and out[long][1].dtype == np.float32
    for keyword in ("first", fits, "last"):
        idx, scores = out[keyword]
        want = dict(zip(hits[keyword][0], rerank.page_scores(keyword, [pages[i]["text"] for i in hits[keyword][0]], model, Characters(), PlainHead(model))))
        assert [want[i] for i in idx.tolist()] == pytest.approx(scores.tolist()) and (np.diff(scores) <= 0).all()


def test_a_refused_head_is_remembered(monkeypatch):
    """The second call raises like the first and loads nothing; another model is loaded as ever."""
    import transformers

    from medical_rag_amd import rerank
    loads = []

    def load(name):
        loads.append(name)
        model = tiny_llama()
        model.lm_head = torch.nn.Linear(32, 64, bias=True)
        return model
    monkeypatch.setattr(rerank, "_MODEL", dict.fromkeys(rerank._MODEL))
    monkeypatch.setattr(transformers.AutoTokenizer, "from_pretrained", lambda name: Characters())
    monkeypatch.setattr(transformers.AutoModelForCausalLM, "from_pretrained", load)
    for name, so_far in (("one", 1), ("one", 1), ("two", 2), ("two", 2), ("one", 3)):
        with pytest.raises(ValueError, match="bias"):
            rerank._model_for(name, "cpu")
        assert len(loads) == so_far
    assert rerank._MODEL["model"] is None


def test_heads_are_compared_with_the_models_own_logits():
    """Whatever a model does to its logits, named in its configuration or not."""
    from transformers import LlamaForCausalLM

    from medical_rag_amd.rerank import ScoringHead
    torch.manual_seed(0)

    def changed(change):
        model = tiny_llama()
        whole = LlamaForCausalLM.forward

        def forward(*args, **kwargs):
            result = whole(model, *args, **kwargs)
            result.logits = change(result.logits)
            return result
        model.forward = forward
        return model
    for change in (lambda x: x / 2, lambda x: x * 1.1, lambda x: x[..., :40], lambda x: x + 0.1, lambda x: x * float("nan")):
        with pytest.raises(ValueError, match="times its output embeddings"):
            ScoringHead.from_model(changed(change))
    for plain in (tiny_llama(), tiny_llama().to(torch.bfloat16), changed(lambda x: x.float())):     # then it is only not on a GPU
        with pytest.raises(ValueError, match="GPU"):
            ScoringHead.from_model(plain)


def test_heads_of_models_that_return_tuples_or_pass_their_norm_by():
    from types import MethodType

    from medical_rag_amd.rerank import ScoringHead
    whole = tiny_llama()
    inner = whole.forward
    whole.forward = lambda *args, **kwargs: (inner(*args, **kwargs).logits,)
    with pytest.raises(ValueError, match="GPU"):        # a plain head, but not on a GPU
        ScoringHead.from_model(whole)
    around = tiny_llama()
    around.forward = MethodType(lambda self, input_ids, use_cache: SimpleNamespace(logits=self.lm_head(self.model.embed_tokens(input_ids))), around)
    with pytest.raises(ValueError, match="norm"):
        ScoringHead.from_model(around)
