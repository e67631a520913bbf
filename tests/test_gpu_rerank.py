"""Re-ranking on the GPU: a tiny randomly initialised decoder, its scoring head in the
library's kernels, against the same steps in 64 bits."""
import os

import numpy as np
import pytest

from oracle import scoring_oracle as orc

pytestmark = pytest.mark.gpu
TINY = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "tiny_encoder")
PAGES = ["pulmonary edema with kerley b lines", "", "absent lung markings beyond a visible pleural line", "pleural effusion " * 40, "x"]


@pytest.fixture(scope="module")
def decoder_dir(tmp_path_factory):
    import shutil

    import torch
    from transformers import AutoTokenizer, LlamaConfig, LlamaForCausalLM
    path = tmp_path_factory.mktemp("decoder")
    for f in ("tokenizer.json", "tokenizer_config.json", "vocab.txt"):
        shutil.copy(os.path.join(TINY, f), path / f)
    vocab = len(AutoTokenizer.from_pretrained(TINY))
    torch.manual_seed(3)
    model = LlamaForCausalLM(LlamaConfig(vocab_size=vocab + 5, hidden_size=96, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
                                         num_key_value_heads=2, max_position_embeddings=512, initializer_range=0.3))
    with torch.no_grad():
        model.model.norm.weight.copy_(1 + 0.2 * torch.randn(96))
    model.save_pretrained(path)         # float32: a padded batch's states are then those of the single pages to 1e-5
    return str(path)


@pytest.fixture(scope="module")
def loaded(decoder_dir):
    from medical_rag_amd import rerank
    model, tok, head = rerank._model_for(decoder_dir, "cuda")
    assert model is not None
    return rerank, model, tok, head


def plain_score(model, tok, text, query):
    """One page at a time, nothing padded, everything after the body in 64 bits on the
    quantised operands: (score, what the 8-bit rounding may move it)."""
    import torch
    enc = lambda t: tok(t, add_special_tokens=False)["input_ids"]  # noqa: E731
    q = enc(query)
    start = tok.bos_token_id if tok.bos_token_id is not None else tok.cls_token_id
    ids = [start] + enc(text) + enc("\n\n") + q
    kept = []
    hook = model.model.norm.register_forward_pre_hook(lambda m, a: kept.append(a[0]))
    with torch.no_grad():
        model.model(input_ids=torch.tensor([ids], device="cuda"))
    hook.remove()
    h = kept[0][0, len(ids) - len(q) - 1:-1].double().cpu().numpy()
    norm = model.model.norm
    y = orc.rms_norm(h, norm.weight.detach().double().cpu().numpy(), norm.variance_epsilon)
    w = model.get_output_embeddings().weight.detach().double().cpu().numpy()
    wq = orc.mx_values(*orc.mx_quantize(w, "mxfp4"), "mxfp4", w.shape[1])
    # e4m3 rounds to half a step: 2^-4 of a value, or of the lowest step 2^-9 times the block's scale, which is at most amax 2^-7
    amax = np.repeat(np.abs(np.pad(y, ((0, 0), (0, 0)))).reshape(len(y), -1, 32).max(2), 32, axis=1)
    move = (np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -17 * amax) @ np.abs(wq).T).max(axis=1)
    lp, _, _, _ = orc.token_logprobs(y @ wq.T, np.array(q)[:, None], 0)
    return lp.mean(), 2 * move.mean()


def test_page_scores_against_64_bits(loaded):
    rerank, model, tok, head = loaded
    query = "pleural line"
    together = rerank.page_scores(query, PAGES, model, tok, head, batch_size=5)
    alone = [rerank.page_scores(query, [p], model, tok, head)[0] for p in PAGES]
    for got, one, page in zip(together, alone, PAGES):
        want, move = plain_score(model, tok, page, query)
        # the body's float32 states differ by their rounding between a padded batch and a single page: 1e-3 covers what
        # that and the sums of the head move, the rest is the rounding to 8 bits
        assert abs(one - want) <= move + 1e-3
        assert abs(got - want) <= move + 1e-3
    assert rerank.page_scores("", PAGES, model, tok, head) == [0.0] * len(PAGES)
    assert rerank.page_scores(query, [], model, tok, head) == []


def test_head_is_its_operators_and_is_cut_without_a_trace(loaded, monkeypatch):
    import torch

    from medical_rag_amd import scoring
    rerank, model, tok, head = loaded
    g = torch.Generator().manual_seed(1)
    hidden = torch.randn(37, 96, generator=g).to(torch.bfloat16).cuda()
    residual = torch.randn(37, 96, generator=g).to(torch.bfloat16).cuda()
    tokens = torch.randint(0, len(head.vocabulary), (37, 2), generator=g).cuda()
    for res in (None, residual):
        rows, _ = scoring.rms_norm_mx(hidden, model.model.norm.weight.detach(), model.model.norm.variance_epsilon, res)
        want = scoring.token_logprobs(scoring.mx_matmul(rows, head.vocabulary), tokens, 4)
        got = head.token_logprobs(hidden, tokens, 4, res)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(head.logits(hidden, res, torch.bfloat16), scoring.mx_matmul(rows, head.vocabulary, torch.bfloat16))


def test_rows_taken_in_parts(loaded):
    """More logits than are held at a time: the same results, with and without tokens and a residual."""
    import torch

    from medical_rag_amd import scoring
    rerank, model, tok, head = loaded

    class Few(rerank.ScoringHead):      # a vocabulary that counts as half a gigabyte of logits a row: four rows a part
        class vocabulary_(scoring.MxRows):
            __slots__ = ()

            def __len__(self):
                return 1 << 27

    v = head.vocabulary
    few = Few(head.norm_weight, head.eps, Few.vocabulary_(v.values, v.scales, v.d, v.format))
    g = torch.Generator().manual_seed(1)
    hidden, residual = (torch.randn(11, 96, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    tokens = torch.randint(0, len(v), (11, 2), generator=g).cuda()
    for tk in (None, tokens):
        for res in (None, residual):
            for a, b in zip(few.token_logprobs(hidden, tk, 4, res), head.token_logprobs(hidden, tk, 4, res)):
                assert torch.equal(a, b)


def test_rerank_pages_and_hits(loaded, decoder_dir):
    rerank, model, tok, head = loaded
    pages = [{"index": i, "text": t} for i, t in enumerate(PAGES)]
    idx, scores = rerank.rerank_pages("pleural line", [3, 0, -1, 2, 1, 4], pages, decoder_dir)
    assert sorted(idx.tolist()) == [0, 1, 2, 3, 4] and (np.diff(scores) <= 0).all()
    plain = dict(zip([3, 0, 2, 1, 4], rerank.page_scores("pleural line", [PAGES[i] for i in [3, 0, 2, 1, 4]], model, tok, head)))
    assert [plain[i] for i in idx.tolist()] == pytest.approx(scores.tolist(), abs=1e-6)
    out = rerank.rerank_hits({"pleural line": (np.array([3, 0, 2]), None), "x": (np.array([-1]), None)}, pages, decoder_dir, top_k=2)
    assert len(out["pleural line"][0]) == 2 and len(out["x"][0]) == 0


def test_caller_re_ranks_its_candidates(decoder_dir):
    from medical_rag_amd import caller, index_builder
    from medical_rag_amd import local_rag as rag
    pages = [{"index": i, "text": t} for i, t in enumerate(PAGES)]
    embedded = index_builder.generate_embeddings_hf(pages, TINY, "cuda", batch_size=4)
    index = rag.PageIndex.from_pages(embedded)
    plain = caller.top_pages_for_texts(["pleural line"], TINY, "cuda", index, top_k=5)
    got = caller.top_pages_for_texts(["pleural line"], TINY, "cuda", index, top_k=3, rerank_model=decoder_dir, candidates=5)
    idx, scores = got["pleural line"]
    assert len(idx) == 3 and set(idx.tolist()) <= set(plain["pleural line"][0].tolist()) and (np.diff(scores) <= 0).all()
    index.close()


def test_two_threads_score_with_one_model(loaded):
    """Each gets its own pages' scores, the ones it gets alone."""
    from concurrent.futures import ThreadPoolExecutor
    rerank, model, tok, head = loaded
    lists = [PAGES[:3] * 8, PAGES[2:] * 8]
    score = lambda pages: rerank.page_scores("pleural line", pages, model, tok, head, batch_size=3)  # noqa: E731
    want = [score(p) for p in lists]
    with ThreadPoolExecutor(2) as pool:
        got = list(pool.map(score, lists * 3))
    for i, g in enumerate(got):
        assert g == want[i % 2]
